"""The operators of a key/value cache that is held in 8 bits, as cases that can be timed and compared.

A cache row of a head is int8 with a scale, a power of two, for each block of rows and head.  ``write`` cases append the tokens of
a step to their sequences and read the blocks that this touched back, as the attention of a continued prompt does; ``read`` cases read
whole prefixes; ``attend`` cases are the attention of a step's tokens over the cached rows.  Head counts and sizes are those of the
7B, 13B and 70B presets and of the serving benchmark, lengths those between a short question and a long document.

``own`` False: plain torch in 32 bits; True: the calls of ``easyllm_b200.ops.infer``.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
GROW = 256                                        # rows a cache grows by


def listed():
    return [
        # one chat, a few turns old: the latency of a layer's attention
        {"name": "attend_one", "op": "attend", "seqs": 1, "longest": 203, "new": 1, "heads": 32, "groups": 8, "dim": 128, "vdim": 128,
         "block": 16, "dtype": "bf16", "alibi": False, "sink": False, "window": 0},
        # a full batch of unequal age, grouped heads
        {"name": "attend_batch", "op": "attend", "seqs": 64, "longest": 8192, "new": 1, "heads": 32, "groups": 8, "dim": 128, "vdim": 128,
         "block": 16, "dtype": "bf16", "alibi": False, "sink": False, "window": 0},
        # the 7B preset: every query head has keys of its own
        {"name": "attend_7b", "op": "attend", "seqs": 24, "longest": 4096, "new": 1, "heads": 32, "groups": 32, "dim": 128, "vdim": 128,
         "block": 16, "dtype": "bf16", "alibi": False, "sink": False, "window": 0},
        # the 70B preset on one long document
        {"name": "attend_long", "op": "attend", "seqs": 1, "longest": 131071, "new": 1, "heads": 64, "groups": 8, "dim": 128, "vdim": 128,
         "block": 64, "dtype": "bf16", "alibi": False, "sink": False, "window": 0},
        # the 13B ALiBi heads, drafted tokens that are looked over together, a scale for every row
        {"name": "attend_drafts", "op": "attend", "seqs": 6, "longest": 1900, "new": 5, "heads": 40, "groups": 40, "dim": 128, "vdim": 128,
         "block": 1, "dtype": "bf16", "alibi": True, "sink": False, "window": 0},
        # hybrid layers in fp32: sinks, odd head sizes, values narrower than keys, a window
        {"name": "attend_hybrid_fp32", "op": "attend", "seqs": 9, "longest": 1031, "new": 1, "heads": 15, "groups": 3, "dim": 72, "vdim": 40,
         "block": 8, "dtype": "fp32", "alibi": False, "sink": True, "window": 500},
        # prompts that go on: the next turns of two conversations
        {"name": "attend_prompts", "op": "attend", "seqs": 2, "longest": 4096, "new": 512, "heads": 32, "groups": 8, "dim": 128, "vdim": 128,
         "block": 16, "dtype": "bf16", "alibi": False, "sink": False, "window": 0},
        # a decode step's tokens, most of them in the middle of a block
        {"name": "write_step", "op": "write", "seqs": 64, "longest": 4096, "new": 1, "groups": 8, "dim": 128, "vdim": 128, "block": 16,
         "dtype": "bf16"},
        # a long prompt of the 7B preset
        {"name": "write_prompt", "op": "write", "seqs": 1, "longest": 4096, "new": 4096, "groups": 32, "dim": 128, "vdim": 128, "block": 16,
         "dtype": "bf16"},
        # turns of unequal length that go on in the middle of blocks, odd heads, fp32
        {"name": "write_turns_fp32", "op": "write", "seqs": 7, "longest": 1500, "new": 333, "groups": 5, "dim": 72, "vdim": 40, "block": 32,
         "dtype": "fp32"},
        # the prefixes of a batch, for layers that take 16 bits
        {"name": "read_prefixes", "op": "read", "seqs": 8, "longest": 4096, "groups": 8, "dim": 128, "vdim": 128, "block": 16, "dtype": "bf16"},
        # one short prefix
        {"name": "read_short", "op": "read", "seqs": 1, "longest": 77, "groups": 4, "dim": 80, "vdim": 64, "block": 4, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    op = rng.choice(["attend", "attend", "attend", "write", "read"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    groups = rng.choice([1, 2, 3, 4, 5, 8, 8, 16, 32])
    dim, vdim = rng.choice([(128, 128), (128, 128), (64, 64), (80, 80), (96, 96), (72, 40), (16, 24), (56, 128), (120, 100)])
    case = {"op": op, "seqs": _spread(rng, 1, 64), "longest": _spread(rng, 1, 60000), "groups": groups, "dim": dim, "vdim": vdim,
            "block": rng.choice([1, 2, 4, 8, 16, 16, 32, 64, 128]), "dtype": dtype}
    bound = 24 * 4096 * 32 * 256 if op == "attend" else 8 * 4096 * 8 * 256
    while case["seqs"] * case["longest"] * groups * (dim + vdim) > bound:
        case["seqs"], case["longest"] = max(1, case["seqs"] // 2), max(1, case["longest"] * 3 // 4)
    if op != "read":
        case["new"] = rng.choice([1, 1, _spread(rng, 1, 16), _spread(rng, 1, 1024)])
        case["new"] = min(case["new"], case["longest"])
    if op == "attend":
        case["heads"] = groups * rng.choice([1, 1, 2, 4, 4, 5, 8, 16, 20] if groups <= 8 else [1, 1, 2, 3])
        while case["new"] > 1 and case["seqs"] * case["new"] * case["longest"] * case["heads"] > 2 * 512 * 4096 * 32:
            case["new"] = max(1, case["new"] // 2)
        case.update(alibi=rng.random() < 0.25, sink=rng.random() < 0.25,
                    window=_spread(rng, 1, 4096) if rng.random() < 0.2 else 0)
    return case


# ---- lengths -----------------------------------------------------------------------------------
def lengths(case):
    """(rows of each sequence behind the step, the step's tokens of each), spread unevenly below the longest."""
    n, longest, new = case["seqs"], case["longest"], case.get("new", 0)
    total, fresh = [], []
    for i in range(n):
        last = i == n - 1
        c = new if last or new <= 1 else 1 + int((new - 1) * ((i + 1) * 0.7548776662 % 1.0))
        t = longest if last else 1 + int((longest - 1) * ((i + 1) * 0.6180339887 % 1.0))
        total.append(max(t, c))
        fresh.append(c)
    return total, fresh


def work(case):
    G, d, dv, e = case["groups"], case["dim"], case["vdim"], 2 if case["dtype"] == "bf16" else 4
    total, fresh = lengths(case)
    rows, new = sum(total), sum(fresh)
    if case["op"] == "read":
        return {"bytes": rows * G * (d + dv) * (1 + e) + 8 * G * (rows // case["block"] + 1), "flops": rows * G * (d + dv)}
    if case["op"] == "write":
        back = sum(t - (t - c) // case["block"] * case["block"] for t, c in zip(total, fresh))
        return {"bytes": (new * (e + 1) + back * (1 + e)) * G * (d + dv) + 16 * G * (back // case["block"] + 1),
                "flops": (3 * new + back) * G * (d + dv)}
    H, w = case["heads"], case["window"] or 1 << 60
    read = sum(min(t, w + c - 1) for t, c in zip(total, fresh))
    pairs = sum(sum(min(t - i, w) for i in range(c)) for t, c in zip(total, fresh))
    return {"bytes": read * G * (d + dv) + 8 * G * (read // case["block"] + 1) + new * H * (d + dv) * e,
            "flops": 2 * pairs * H * (d + dv)}


# ---- inputs ------------------------------------------------------------------------------------
def _round16(n):
    return -(-n // 16) * 16


def _pow2_scale(amax):
    """The least power of two, 2^-126 or more, of which 127 times is ``amax`` or more; NaN where that is not finite."""
    m, e = torch.frexp(amax)                       # amax = m 2^e, m in [1/2, 1)
    e = torch.where(m <= 127 / 128, e - 7, e - 6).clamp(min=-126)
    e = torch.where(amax == 0, torch.full_like(e, -126), e)
    power = ((e.int() + 127) << 23).view(torch.float32)                # pow() is not exact everywhere
    return torch.where(torch.isfinite(amax), power, torch.full_like(amax, float("nan")))


def _filled(case, slots, capacity, used, width, g):
    """An 8-bit cache whose slots hold ``used[s]`` rows (and, behind their last block, what former sequences left)."""
    G, block = case["groups"], case["block"]
    q = torch.zeros(slots, capacity, G, _round16(width), dtype=torch.int8, device="cuda")
    scale = torch.zeros(slots, capacity // block, G, device="cuda")
    channel = torch.exp(0.5 * torch.randn(G, width, device="cuda", generator=g))
    for s in range(slots):
        x = torch.randn(capacity, G, width, device="cuda", generator=g) * channel
        x[used[s]:-(-used[s] // block) * block] = 0
        amax = x.abs().view(capacity // block, block, G, width).amax((1, 3))
        scale[s] = _pow2_scale(amax)
        q[s, :, :, :width] = torch.round(x / scale[s].repeat_interleave(block, 0).unsqueeze(-1)).clamp(-127, 127).to(torch.int8)
    return q.view(-1, G, q.shape[-1]), scale.view(-1, G)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    G, d, dv, block, dt = case["groups"], case["dim"], case["vdim"], case["block"], TYPES[case["dtype"]]
    total, fresh = lengths(case)
    n = case["seqs"]
    capacity = -(-max(total) // GROW) * GROW
    order = random.Random(seed).sample(range(n), n)                     # the slot of each sequence
    before = [t - c for t, c in zip(total, fresh)]
    used = [0] * n
    for i, s in enumerate(order):
        used[s] = before[i] if case["op"] == "write" else total[i]
    st = {"case": case, "dim": d, "vdim": dv, "block": block}
    st["k"], st["k_scale"] = _filled(case, n, capacity, used, d, g)
    st["v"], st["v_scale"] = _filled(case, n, capacity, used, dv, g)
    base = [s * capacity for s in order]
    if case["op"] == "read":
        st.update(base=_ints(base), length=_ints(total), longest=max(total))
        return st
    cu = [0]
    for c in fresh:
        cu.append(cu[-1] + c)
    T = cu[-1]
    st["kv_base"] = _ints([base[i] for i in range(n) for _ in range(fresh[i])])
    st["kv_len"] = _ints([before[i] + j + 1 for i in range(n) for j in range(fresh[i])])
    st["cu_seqlens"], st["max_seqlen"], st["longest"] = _ints(cu), max(fresh), max(total)
    if case["op"] == "write":
        # keys and values are columns of the projection's rows
        wide = torch.randn(T, G * (d + dv) + 64, device="cuda", generator=g).to(dt)
        st["new_k"] = wide[:, 64:64 + G * d].view(T, G, d)
        st["new_v"] = wide[:, 64 + G * d:].view(T, G, dv)
        first = [p // block * block for p in before]
        st["back_base"] = _ints([b + f for b, f in zip(base, first)])
        st["back_len"] = _ints([t - f for t, f in zip(total, first)])
        st["back_longest"] = max(t - f for t, f in zip(total, first))
        return st
    H = case["heads"]
    st["q"] = torch.randn(T, H, d, device="cuda", generator=g).to(dt)
    st["sink"] = torch.randn(H, device="cuda", generator=g) if case["sink"] else None
    st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda") if case["alibi"] else None
    st["scale"] = d ** -0.5
    return st


# ---- one pass ------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else {"attend": _attend, "write": _write, "read": _read}[state["case"]["op"]](state)


def _run_own(st):
    from easyllm_b200.ops import infer
    case = st["case"]
    cache = infer.KV8(st["k"], st["v"], st["k_scale"], st["v_scale"], st["dim"], st["vdim"])
    if case["op"] == "read":
        return infer.kv8_read(cache, st["base"], st["length"], st["longest"], TYPES[case["dtype"]])
    if case["op"] == "write":
        infer.kv8_append(cache, st["new_k"], st["new_v"], st)
        return infer.kv8_read(cache, st["back_base"], st["back_len"], st["back_longest"], TYPES[case["dtype"]])
    several = st["max_seqlen"] > 1
    return infer.attention_kv8(st["q"], cache, st["kv_base"], st["kv_len"], st["longest"], st["scale"], st["sink"], st["slopes"],
                               case["window"] or None, st["cu_seqlens"] if several else None, st["max_seqlen"])


def _values(q, scale, base, longest, width, block):
    """fp32 ``[n, longest, G, width]`` of the rows from ``base`` on (rows behind the cache repeat its last)."""
    at = (base.long().unsqueeze(1) + torch.arange(longest, device=q.device)).clamp(max=q.shape[0] - 1)
    return q[at][..., :width].float() * scale[at // block].unsqueeze(-1)


def _read_rows(st, base, length, longest):
    keep = torch.arange(longest, device=length.device) < length.unsqueeze(1)
    dt = TYPES[st["case"]["dtype"]]
    out = []
    for name, width in (("k", st["dim"]), ("v", st["vdim"])):
        x = _values(st[name], st[name + "_scale"], base, longest, width, st["block"])
        out.append(torch.where(keep.view(*keep.shape, 1, 1), x, torch.zeros_like(x)).to(dt))
    return tuple(out)


def _read(st):
    return _read_rows(st, st["base"], st["length"], st["longest"])


def _write(st):
    block = st["block"]
    cu = st["cu_seqlens"].long()
    row = st["kv_base"].long() + st["kv_len"].long() - 1                # of every new token
    start = row[cu[:-1]]                                                # of every sequence's first
    inside = torch.arange(block, device=row.device)
    for name in ("k", "v"):
        q, scale, x = st[name], st[name + "_scale"], st["new_" + name].float()
        G, width = x.shape[1:]
        amax = torch.zeros_like(scale).scatter_reduce(0, (row // block).unsqueeze(1).expand(-1, G), x.abs().amax(-1), "amax")
        need = _pow2_scale(amax)
        old = scale[start // block]                                     # [sequences, G]: of the block a sequence goes on in
        goes_on = (start % block != 0).unsqueeze(1)
        first = torch.where(goes_on, torch.maximum(old, need[start // block]), need[start // block])
        new = need.index_copy(0, start // block, first)
        touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=row.device).index_fill(0, row // block, True)
        # rows that were in the block already take its new scale
        there = (start // block * block).unsqueeze(1) + inside
        had = q[there].float()
        again = torch.round(had * (old / first).view(-1, 1, G, 1)).to(torch.int8)
        stay = (there < start.unsqueeze(1)).view(-1, block, 1, 1)
        q[there] = torch.where(stay, again, q[there])
        scale.copy_(torch.where(touched.unsqueeze(1), new, scale))
        q[row, :, :width] = torch.round(x / new[row // block].unsqueeze(-1)).to(torch.int8)
    return _read_rows(st, st["back_base"], st["back_len"], st["back_longest"])


def _attend(st):
    q, cu, longest, window = st["q"], st["cu_seqlens"].long(), st["longest"], st["case"]["window"]
    T, H, d = q.shape
    n, most, G, dv = cu.numel() - 1, st["max_seqlen"], st["k"].shape[1], st["vdim"]
    seq = torch.repeat_interleave(torch.arange(n, device=q.device), cu[1:] - cu[:-1], output_size=T)
    place = torch.arange(T, device=q.device) - cu[seq]
    base = st["kv_base"][cu[:-1]]
    k = _values(st["k"], st["k_scale"], base, longest, d, st["block"]).permute(0, 2, 3, 1)            # [n, G, d, longest]
    v = _values(st["v"], st["v_scale"], base, longest, dv, st["block"]).permute(0, 2, 1, 3)           # [n, G, longest, dv]
    rows = torch.zeros(n, most, H, d, device=q.device)
    rows[seq, place] = q.float()
    end = torch.ones(n, most, dtype=torch.long, device=q.device)
    end[seq, place] = st["kv_len"].long()
    rows = rows.view(n, most, G, H // G, d).permute(0, 2, 3, 1, 4).reshape(n, G, H // G * most, d)
    s = (torch.matmul(rows, k) * st["scale"]).view(n, H, most, longest)
    key = torch.arange(longest, device=q.device)
    if st["slopes"] is not None:
        s = s + st["slopes"].view(1, H, 1, 1) * (key - (end.unsqueeze(-1) - 1)).float().unsqueeze(1)
    hidden = key >= end.unsqueeze(-1)
    if window:
        hidden = hidden | (key < end.unsqueeze(-1) - window)
    s = s.masked_fill(hidden.unsqueeze(1), float("-inf"))
    top = s.amax(-1, keepdim=True)
    if st["sink"] is not None:
        top = torch.maximum(top, st["sink"].view(1, H, 1, 1))
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if st["sink"] is not None:
        total = total + torch.exp(st["sink"].view(1, H, 1, 1) - top)
    o = torch.matmul((p / total).view(n, G, H // G * most, longest), v).view(n, H, most, dv)
    return o.permute(0, 2, 1, 3)[seq, place].to(q.dtype)


# ---- the definition in 64 bits -------------------------------------------------------------------
def _least_power(amax):
    """2^e in 64 bits: the least e >= -126 with amax <= 127 2^e."""
    s = torch.full_like(amax, 2.0 ** -126)
    while bool((amax > 127 * s).any()):
        s = torch.where(amax > 127 * s, 2 * s, s)
    return s


def exact(case, seed):
    st = prepare(case, seed)
    block = case["block"]
    wide = {name: st[name].double()[..., :st[w]] for name, w in (("k", "dim"), ("v", "vdim"))} if case["op"] != "attend" else {}
    if case["op"] == "attend":
        q, cu = st["q"].double(), st["cu_seqlens"].tolist()
        base, length = st["kv_base"].tolist(), st["kv_len"].tolist()
        H, G = case["heads"], case["groups"]
        out = torch.zeros(q.shape[0], H, st["vdim"], dtype=torch.float64, device=q.device)
        for a, b in zip(cu[:-1], cu[1:]):
            end = length[b - 1]
            low = max(0, length[a] - case["window"]) if case["window"] else 0
            at = torch.arange(base[a] + low, base[a] + end, device=q.device)
            of = at // block
            pos, key = torch.arange(length[a], end + 1, device=q.device), at - base[a]
            for g in range(G):
                k = st["k"][at, g, :st["dim"]].double() * st["k_scale"][of, g].double().unsqueeze(1)
                v = st["v"][at, g, :st["vdim"]].double() * st["v_scale"][of, g].double().unsqueeze(1)
                hs = range(g * (H // G), (g + 1) * (H // G))
                for h in hs:
                    s = q[a:b, h] @ k.t() * st["scale"]
                    if st["slopes"] is not None:
                        s = s + st["slopes"][h].double() * (key.unsqueeze(0) - (pos.unsqueeze(1) - 1))
                    see = key.unsqueeze(0) < pos.unsqueeze(1)
                    if case["window"]:
                        see = see & (key.unsqueeze(0) >= pos.unsqueeze(1) - case["window"])
                    s = torch.where(see, s, torch.full_like(s, -math.inf))
                    if st["sink"] is not None:
                        s = torch.cat((s, st["sink"][h].double().expand(b - a, 1)), 1)
                    out[a:b, h] = torch.softmax(s, -1)[:, :len(at)] @ v
        return out
    if case["op"] == "write":
        first, cu = (st["kv_base"] + st["kv_len"] - 1).tolist(), st["cu_seqlens"].tolist()
        for name in ("k", "v"):
            q, scale, x = wide[name], st[name + "_scale"], st["new_" + name].double()
            for a, b in zip(cu[:-1], cu[1:]):
                r0, r1 = first[a], first[a] + b - a
                lo = r0 // block * block
                at = torch.arange(lo, r1, device=q.device)
                blocks = at // block - lo // block
                amax = torch.zeros(int(blocks[-1]) + 1, x.shape[1], dtype=torch.float64, device=q.device)
                amax.scatter_reduce_(0, blocks[r0 - lo:].unsqueeze(1).expand(-1, x.shape[1]), x[a:b].abs().amax(-1), "amax")
                s = _least_power(amax)
                if r0 > lo:
                    old = scale[lo // block].double()
                    s[0] = torch.maximum(s[0], old)
                    q[lo:r0] = torch.round(q[lo:r0] * (old / s[0]).unsqueeze(1))
                q[r0:r1] = torch.round(x[a:b] / s[blocks[r0 - lo:]].unsqueeze(-1))
                scale[lo // block:lo // block + s.shape[0]] = s.float()
        base, length, longest = st["back_base"].tolist(), st["back_len"].tolist(), st["back_longest"]
    else:
        base, length, longest = st["base"].tolist(), st["length"].tolist(), st["longest"]
    out = []
    for name in ("k", "v"):
        q, scale = wide[name], st[name + "_scale"].double()
        o = torch.zeros(len(base), longest, *q.shape[1:], dtype=torch.float64, device=q.device)
        for i, (b, n) in enumerate(zip(base, length)):
            at = torch.arange(b, b + n, device=q.device)
            o[i, :n] = q[at] * scale[at // block].unsqueeze(-1)
        out.append(o)
    return tuple(out)
