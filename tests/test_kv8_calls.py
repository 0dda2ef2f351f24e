"""Calls of the 8-bit key/value cache at the edges of what they take: which of them run, by which way, and what is refused."""
import pytest
import torch

from easyllm_b200.ops import infer as iops
from test_kv8 import (BF16, DEVICES, F32, _device, _no_kernel_gave_up, check_attention, filled, ints, near, plain_attention, rand,  # noqa: F401
                      step)


class NoKernel:
    """In the place of the launchers: a call of any of them is a failure."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


# ---- borders without a sequence ---------------------------------------------------------------------
@pytest.mark.parametrize("max_len,max_q", [(64, 1), (64, 3), (5000, 3), (5000, 300)])
def test_rows_without_a_sequence_reach_no_kernel(monkeypatch, max_len, max_q):
    cache = iops.kv8_empty(64, 2, 32, 16, 16)
    monkeypatch.setattr(iops, "_kern", lambda x: True)
    monkeypatch.setattr(iops, "_cu", NoKernel)
    q, places = torch.ones(5, 4, 32, dtype=BF16), ints([999] * 5)
    got = iops.attention_kv8(q, cache, places, places, max_len, 1.0, cu_seqlens=ints([0]), max_q=max_q)
    assert got.shape == (5, 4, 16) and got.dtype == BF16 and not bool(got.any())


def test_the_entry_refuses_borders_without_a_sequence():
    """Before it looks at anything on the device, so this needs none."""
    import ctypes
    from easyllm_b200.ops import cuda, cuda_infer
    at = 1 << 20                                                  # an address that nobody looks at
    words = (at, at, at, at, 2, 32, 16, 16, 64)
    for n_seq in (0, -1):
        call = cuda_infer._KV8_CALLS["ell_attn_kv8"](*words, at, at, 0, 0, at, at, 0, 0, at, 5, n_seq, 1, 4, 128, 64, 0, 1, at, 1.0)
        assert cuda.lib().ell_attn_kv8(ctypes.c_char_p(call), ctypes.c_void_p(0)) == -2


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("max_len,max_q,H", [(64, 1, 4), (64, 3, 4), (5000, 3, 4), (5000, 300, 4), (5000, 2, 512)])
def test_rows_without_a_sequence_are_zero(device, dtype, max_len, max_q, H):
    dev = _device(device)
    cache, _ = filled(64, 2, 32, 32, 16, dev)
    places = ints([0, 999, -1, 1 << 30, 16], dev)
    got = iops.attention_kv8(torch.ones(5, H, 32, dtype=dtype, device=dev), cache, places, places, max_len, 1.0, cu_seqlens=ints([0], dev), max_q=max_q)
    assert got.shape == (5, H, 32) and got.dtype == dtype and not bool(got.any())


# ---- rows read back -----------------------------------------------------------------------------------
def way(monkeypatch, T, H, cache, max_len, cu_seqlens, max_q, window=None, dtype=BF16):
    """Which way a call takes on a GPU: "bytes" (integer products on the cache) or "back" (rows read back).  Nothing is launched."""
    from easyllm_b200.ops import cuda_infer as ci
    taken = []
    monkeypatch.setattr(ci, "_attention_read_back", lambda *a: taken.append("back"))
    monkeypatch.setattr(ci, "_kv8_call", lambda name, *a: taken.append("bytes"))
    monkeypatch.setattr(ci, "_err_word", lambda device: 0)
    places = ints([0] * T)
    q = torch.empty(T, H, cache.dim, dtype=dtype)
    words = iops._kv8_check(cache, places)[:-1] + (1 << 30,)      # as of a cache with any number of rows
    ci.attention_kv8.__wrapped__(q, words, places, places, max_len, 1.0, None, None, window, cu_seqlens, max_q)
    assert len(taken) == 1
    return taken[0]


def test_single_tokens_stay_on_the_bytes_whatever_their_heads(monkeypatch):
    """The kernel behind the other way goes by borders of sequences of several tokens: without them, or with one token each, it takes every
    row by its own place, also rows behind the last border, which have none."""
    cache = iops.kv8_empty(64, 1, 128, 128, 16)
    for H in (256, 512, 1024):
        for max_len in (64, 5000):
            assert way(monkeypatch, 3, H, cache, max_len, None, None) == "bytes"
            assert way(monkeypatch, 3, H, cache, max_len, ints([0, 1, 2]), 1) == "bytes"
    for T, want in ((5, "bytes"), (6, "back")):                   # 16 heads of each token fill a tile
        assert way(monkeypatch, T, 1024, cache, 5000, ints([0, T]), T) == want


def test_more_sequences_than_are_read_back_stay_on_the_bytes(monkeypatch):
    cache = iops.kv8_empty(64, 1, 16, 16, 16)
    for n, want in ((65535, "back"), (65536, "bytes")):
        cu = torch.arange(n + 1, dtype=torch.int32)
        assert way(monkeypatch, 6 * n, 16, cache, 64, 6 * cu, 6) == want


def test_the_way_goes_by_the_work_and_by_what_a_sequence_reads(monkeypatch):
    cache = iops.kv8_empty(64, 8, 128, 128, 16)

    def of(new, H, max_len, **kw):
        cu = ints([0] + new).cumsum(0).int()
        return way(monkeypatch, sum(new), H, cache, max_len, cu, kw.pop("max_q", max(new)), **kw)
    assert of([512], 32, 4096) == of([512, 1], 32, 4096) == of([64], 32, 4096) == "back"
    assert of([512], 32, 4096, dtype=F32) == "bytes"              # the kernel takes bf16
    assert of([23], 32, 30000) == "bytes"                         # 92 rows of a tile of 128
    assert of([24], 32, 30000) == "back"
    assert of([128], 8, 1000) == "bytes"                          # little to do
    assert of([512] + [1] * 30, 32, 4096) == "bytes"              # 30 prefixes of which every row serves one token
    assert of([512] * 16, 32, 8192) == of([512] * 32, 32, 8192) == "back"
    assert of([512] * 33, 32, 8192) == "bytes"                    # past the memory
    assert of([5], 32, 30000, max_q=2048) == "bytes"              # a bound that the rows do not reach


def test_the_way_goes_by_what_a_window_leaves_to_do(monkeypatch):
    """A whole prefix is not written out in 16 bits for rows that see the end of it."""
    cache = iops.kv8_empty(64, 8, 128, 128, 16)

    def of(new, max_len, window):
        return way(monkeypatch, new, 32, cache, max_len, ints([0, new]), new, window)
    assert of(512, 30000, 64) == of(512, 30000, 256) == of(128, 30000, 1024) == of(128, 30000, 4096) == "bytes"
    assert of(512, 30000, 1024) == of(128, 30000, 16384) == of(512, 4096, 64) == of(2048, 30000, 64) == "back"
    assert of(512, 30000, 1 << 40) == of(512, 30000, None) == "back"


@pytest.mark.parametrize("window", [(1 << 31) + 3, (1 << 32) + 5, 1 << 70])
def test_windows_past_32_bits_are_not_cut_to_them(monkeypatch, window):
    """Both ways get a window that hides nothing, in the words that they have for it."""
    from easyllm_b200.ops import cuda_infer as ci
    cache, seen = iops.kv8_empty(64, 8, 128, 128, 16), []
    monkeypatch.setattr(ci, "_attention_read_back", lambda q, words, base, length, max_len, scale, sink, slopes, window, *a: seen.append(window))
    monkeypatch.setattr(ci, "_kv8_call", lambda name, label, n, *words: seen.append(ci._KV8_CALLS[name](*words) and words[24]))
    monkeypatch.setattr(ci, "_err_word", lambda device: 0)
    for new, max_len in ((512, 4096), (2, 64)):
        places = ints([0] * new)
        ci.attention_kv8.__wrapped__(torch.empty(new, 32, 128, dtype=BF16), iops._kv8_check(cache, places)[:-1] + (1 << 30,), places, places, max_len,
                                     1.0, None, None, window, ints([0, new]), new)
    assert len(seen) == 2 and all(4096 <= w < 1 << 31 for w in seen)


@pytest.mark.gpu
@pytest.mark.parametrize("device", ["cuda"])
def test_attention_of_more_sequences_than_are_read_back(device):
    """65536 sequences, of 32 tokens the first and the last, the others of none."""
    dev = _device(device)
    cache, plain = filled(128, 1, 16, 16, 16, dev)
    q = rand(64, 16, 16, seed=1).to(BF16).to(dev)
    base, length = ints([0] * 32 + [64] * 32, dev), ints(list(range(20, 52)) + list(range(1, 33)), dev)
    cu = ints([0] + [32] * 65535 + [64], dev)
    got = iops.attention_kv8(q, cache, base, length, 64, 0.3, cu_seqlens=cu, max_q=32)
    for r, (b, n) in enumerate(zip(base.tolist(), length.tolist())):
        near(got[r], *plain_attention(q[r], *(p.values(b, n) for p in plain), 0.3))


@pytest.mark.gpu
@pytest.mark.parametrize("device", ["cuda"])
@pytest.mark.parametrize("H,longest,block", [(512, 90, 16), (256, 4200, 64), (512, 4200, 16), (258, 4200, 16)])
def test_single_tokens_of_many_heads(device, H, longest, block):
    """One key head for hundreds of query heads, as tokens of their own and as sequences of one, with rows behind the last border."""
    dev = _device(device)
    n, d, cap = 3, 32, -(-longest // 128) * 128
    cache, plain = filled(n * cap, 1, d, d, block, dev)
    q = rand(n + 2, H, d, seed=1).to(BF16).to(dev)
    total = [longest, 1, longest // 2]
    base, length = ints([0, cap, 2 * cap, 1 << 30, -7], dev), ints(total + [99, 1 << 30], dev)
    alone = iops.attention_kv8(q[:n], cache, base[:n], length[:n], longest, 0.2)
    bordered = iops.attention_kv8(q, cache, base, length, longest, 0.2, cu_seqlens=ints([0, 1, 2, 3], dev), max_q=1)
    assert torch.equal(bordered[:n], alone) and not bool(bordered[n:].any())
    for r, t in enumerate(total):
        near(alone[r], *plain_attention(q[r], *(p.values(r * cap, t) for p in plain), 0.2))


@pytest.mark.gpu
def test_rows_behind_the_last_border_have_no_place_among_rows_read_back():
    """What the attention over rows read back is told of them: place 0, length 0."""
    from easyllm_b200.ops import cuda_infer as ci
    dev = _device("cuda")
    cache, _ = filled(512, 2, 32, 32, 16, dev)
    for cu, rows in (([0, 3, 5], 9), ([0, 5, 5], 9), ([0, 5], 300), ([0, 0], 4), ([0, 9], 9)):
        cu, max_len, n = ints(cu, dev), 64, len(cu) - 1
        length, base = ints([40 + r for r in range(rows)], dev).clamp(max=64), ints([0] * rows, dev)
        k, v = (torch.empty(n * max_len, 2, 32, dtype=BF16, device=dev) for _ in "kv")
        place = torch.full((2, rows), -1, dtype=torch.int32, device=dev)
        ci._kv8_call("ell_kv8_read", "kv8_read", 1, *iops._kv8_check(cache, cu), k.data_ptr(), v.data_ptr(), base.data_ptr(), length.data_ptr(),
                     cu.data_ptr(), place.data_ptr(), n, rows, max_len, 1, ci._err_word(dev))
        border = cu.tolist()
        want = [[i * max_len for i in range(n) for _ in range(border[i + 1] - border[i])], length.tolist()[:border[-1]]]
        assert place.tolist() == [w + [0] * (rows - border[-1]) for w in want]


# ---- where the cache starts -----------------------------------------------------------------------------
def shifted(cache, name, by):
    """``cache`` with one of its tensors starting ``by`` bytes behind a 16-byte boundary, contiguous as before."""
    t = getattr(cache, name)
    room = torch.zeros(t.numel() * t.element_size() + 32, dtype=torch.uint8, device=t.device)
    start = -room.data_ptr() % 16 + by
    moved = room[start:start + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
    assert moved.data_ptr() % 16 == by and moved.is_contiguous()
    moved.copy_(t)
    return cache._replace(**{name: moved})


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name,by", [("k", 1), ("k", 4), ("v", 8), ("v", 15)])
def test_rows_that_start_off_a_boundary_are_refused(device, name, by):
    dev = _device(device)
    cache, one = shifted(iops.kv8_empty(64, 2, 32, 16, 16, dev), name, by), ints([0], dev)
    with pytest.raises(ValueError, match="16-byte"):
        iops.kv8_append(cache, torch.zeros(1, 2, 32, device=dev), torch.zeros(1, 2, 16, device=dev), step([1], [0], [0], 64, dev))
    with pytest.raises(ValueError, match="16-byte"):
        iops.kv8_read(cache, one, one, 4)
    for dtype in (F32, BF16):
        with pytest.raises(ValueError, match="16-byte"):
            iops.attention_kv8(torch.zeros(1, 4, 32, dtype=dtype, device=dev), cache, one, one, 4, 1.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("d,dv", [(32, 16), (40, 9)])
def test_scales_and_inputs_may_start_anywhere(device, d, dv):
    """Scales behind a 4-byte boundary, new rows and queries behind that of their type: the rows of an aligned cache, to the bit, and attention
    over them within the bound of 32-bit sums (on the CPU a library's product, whose order of sums goes by where its operands start)."""
    dev = _device(device)
    T, G, H, cap = 37, 2, 4, 64
    for dtype in (F32, BF16):
        k, v, q = (rand(T * n * w + 1, seed=w + n).to(dtype).to(dev) for n, w in ((G, d), (G, dv), (H, d)))
        results = []
        for at in (0, 1):
            cache = iops.kv8_empty(cap, G, d, dv, 16, dev)
            if at:
                cache = shifted(shifted(cache, "k_scale", 4), "v_scale", 12)
            meta = step([T], [0], [0], cap, dev)
            kk, vv, qq = (t[1:].view(T, n, w) if at else t[1:].clone().view(T, n, w) for t, n, w in ((k, G, d), (v, G, dv), (q, H, d)))
            iops.kv8_append(cache, kk, vv, meta)
            results.append(iops.kv8_read(cache, ints([0], dev), ints([T], dev), T, dtype))
            got = iops.attention_kv8(qq, cache, meta["kv_base"], meta["kv_len"], T, 0.2, cu_seqlens=meta["cu_seqlens"], max_q=T)
            rows = [x[0].double().cpu() for x in results[-1]]
            for r in range(T):
                near(got[r], *plain_attention(qq[r], *(x[:r + 1] for x in rows), 0.2))
        for a, b in zip(*results):
            assert torch.equal(a, b)


def test_the_entries_refuse_rows_off_a_boundary():
    """Before they look at anything on the device, so this needs none."""
    import ctypes
    from easyllm_b200.ops import cuda, cuda_infer
    at = 1 << 20
    rest = {"ell_kv8_append": (at, at, at, at, at, 1, 1, 1, 64, 32, 1, at), "ell_kv8_read": (at, at, at, at, 0, 0, 1, 1, 4, 1, at),
            "ell_attn_kv8": (at, at, 0, 0, at, at, 0, 0, 0, 1, 0, 1, 4, 128, 4, 0, 1, at, 1.0)}
    for name, words in rest.items():
        for k, v in ((at + 1, at), (at, at + 8)):
            call = cuda_infer._KV8_CALLS[name](k, v, at, at, 2, 32, 16, 16, 64, *words)
            assert getattr(cuda.lib(), name)(ctypes.c_char_p(call), ctypes.c_void_p(0)) == -2, name


# ---- bounds that do not hold --------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bound", [0, -3])
@pytest.mark.parametrize("n,start", [(40, 0), (17, 16), (30, 9)])
def test_rows_beyond_a_bound_of_none_are_reported(bound, n, start):
    """``max_seqlen`` below 1 with a sequence that brings more rows than a block takes: the error word is set, as with any other bound
    that does not hold, and what was written before the bound is a whole block."""
    from easyllm_b200.ops import cuda
    dev = _device("cuda")
    cache, plain = filled(128, 2, 32, 32, 16, dev)
    x = rand(n, 2, 32, seed=1).to(dev)
    iops.kv8_append(cache, x, x, dict(step([n], [start], [0], 128, dev), max_seqlen=bound))
    with pytest.raises(cuda.KernelError, match="51"):
        cuda.check_err_flag()
    for p in plain:
        p.append(0, start, x[:16 - start % 16])
    for got, p in zip(iops.kv8_read(cache, ints([0], dev), ints([128], dev), 128, F32), plain):
        assert torch.equal(got[0].double().cpu(), p.values(0, 128))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("max_len,total,new", [(10, 40, 1), (0, 1, 1), (-5, 7, 3), (64, 65, 1), (1100, 1300, 2)])
def test_lengths_beyond_their_bound_are_reported(dtype, max_len, total, new):
    """By the attention on the cache's bytes as by that on rows read back; there the answers are those of the true lengths."""
    from easyllm_b200.ops import cuda
    dev = _device("cuda")
    cache, plain = filled(1408, 2, 32, 32, 16, dev)
    meta = step([new], [total - new], [0], 1408, dev)
    q = rand(new, 4, 32, seed=3).to(dtype).to(dev)
    kw = dict(cu_seqlens=meta["cu_seqlens"], max_q=new) if new > 1 else {}
    for bound, fine in ((total, True), (max_len, False)):
        got = iops.attention_kv8(q, cache, meta["kv_base"], meta["kv_len"], bound, 0.2, **kw)
        if fine:
            cuda.check_err_flag()
        else:
            with pytest.raises(cuda.KernelError, match="51"):
                cuda.check_err_flag()
        for r in range(new):
            near(got[r], *plain_attention(q[r], *(p.values(0, total - new + 1 + r) for p in plain), 0.2))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("block", [1, 16])
def test_bounds_that_are_far_off(device, dtype, block):
    """``max_seqlen``, ``max_q`` and ``max_len`` say "at most": of a call's rows, or of the cache, there are never more."""
    dev = _device(device)
    cache, plain = filled(256, 2, 32, 16, block, dev)
    T, far = 9, 1 << 40
    k, v, q = (rand(T, n, w, seed=n + w).to(dtype).to(dev) for n, w in ((2, 32), (2, 16), (4, 32)))
    meta = step([5, 4], [40, 0], [1, 0], 128, dev)
    iops.kv8_append(cache, k, v, dict(meta, max_seqlen=far))
    for p, x in zip(plain, (k, v)):
        p.append(128, 40, x[:5])
        p.append(0, 0, x[5:])
    for x, p in zip(iops.kv8_read(cache, ints([0], dev), ints([256], dev), 256, F32), plain):
        assert torch.equal(x[0].double().cpu(), p.values(0, 256))
    for kw in (dict(cu_seqlens=meta["cu_seqlens"], max_q=far), {}):
        got = iops.attention_kv8(q, cache, meta["kv_base"], meta["kv_len"], far, 0.2, **kw)
        for r, (b, n) in enumerate(zip(meta["kv_base"].tolist(), meta["kv_len"].tolist())):
            near(got[r], *plain_attention(q[r], *(p.values(b, n) for p in plain), 0.2))


@pytest.mark.parametrize("device", DEVICES)
def test_a_bound_of_none_with_no_rows(device):
    dev = _device(device)
    cache, plain = filled(128, 2, 32, 32, 16, dev)
    x = rand(3, 2, 32, seed=1).to(dev)
    iops.kv8_append(cache, x, x, {"kv_base": ints([0] * 3, dev), "kv_len": ints([5, 6, 7], dev), "cu_seqlens": ints([0, 0, 0], dev), "max_seqlen": 0})
    for got, p in zip(iops.kv8_read(cache, ints([0], dev), ints([128], dev), 128, F32), plain):
        assert torch.equal(got[0].double().cpu(), p.values(0, 128))


# ---- models -----------------------------------------------------------------------------------------------
def test_latent_attention_refuses_the_cache_however_it_is_asked_for(tmp_path):
    from easyllm_b200.models.hf_models import CausalLM, arch_from_hf_config
    from megozen_models import CONFIGS
    arch = arch_from_hf_config(CONFIGS["odd"])
    CausalLM(arch).save_pretrained(str(tmp_path))
    assert CausalLM.from_pretrained(str(tmp_path), arch_overrides={"bos_token_id": 1}).arch.bos_token_id == 1
    with pytest.raises(ValueError, match="kv_cache_block"):
        CausalLM.from_pretrained(str(tmp_path), arch_overrides={"kv_cache_block": 16})
    arch.kv_cache_block = 16
    with pytest.raises(ValueError, match="kv_cache_block"):
        CausalLM(arch)


def test_a_config_that_leaves_the_cache_empty():
    """``null``, as tools write what is not set."""
    from easyllm_b200.models.hf_models import arch_from_hf_config
    from pafodra_models import CONFIGS
    for cfg in ({"model_type": "llama"}, CONFIGS["odd"]):
        assert arch_from_hf_config(dict(cfg, kv_cache_block=None)).kv_cache_block == 0
        assert arch_from_hf_config(dict(cfg, kv_cache_block=8)).kv_cache_block == 8


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,block,dtype", [(21, 16, F32), (40, 8, BF16), (1, 128, BF16), (0, 16, F32)])
def test_a_prefix_is_held_as_the_definition_says(monkeypatch, device, n, block, dtype):
    """Prefixes in any order of memory, into slots in any order: the rows of the definition, the other slots as they were; a step that goes
    on inside the prefix's last block joins it."""
    from easyllm_b200.models.hf_models.state import KV8Rows
    from easyllm_b200.ops import cuda_infer as ci
    dev = _device(device)
    append = iops.kv8_append

    def packed(cache, k, v, meta):                                # what the kernel takes, on the CPU too
        ci._packed(k, "k"), ci._packed(v, "v")
        append(cache, k, v, meta)
    monkeypatch.setattr(iops, "kv8_append", packed)
    slots, cap, G, d, dv = 4, 256, 3, 40, 24
    rows = KV8Rows(slots, cap, G, d, dv, block, dev)
    had, plain = filled(slots * cap, G, d, dv, block, dev)
    rows.cache = had
    k = rand(G, n, d, seed=1).to(dtype).to(dev).transpose(0, 1)   # heads first in memory
    v = rand(n, dv, G, seed=2).to(dtype).to(dev).transpose(1, 2)
    rows.load_prefix([3, 1], k, v)
    more = [rand(2, G, w, seed=w).to(dtype).to(dev) for w in (d, dv)]
    append(rows.cache, *more, step([1, 1], [n, n], [1, 3], cap, dev))
    for s, r in ((1, 0), (3, 1)):
        for p, x, y in zip(plain, (k, v), more):
            p.append(s * cap, 0, x) if n else None
            p.append(s * cap, n, y[r:r + 1])
    for x, p in zip(iops.kv8_read(rows.cache, ints([0], dev), ints([slots * cap], dev), slots * cap, F32), plain):
        assert torch.equal(x[0].double().cpu(), p.values(0, slots * cap))


@pytest.mark.gpu
def test_a_captured_step_is_not_replayed_once_the_state_has_grown():
    """A state without a free slot grows by a new sequence: its caches are elsewhere then, whatever their kind."""
    from easyllm_b200.models.hf_models.state import DecodeGraph
    from test_kv8 import _model
    dev = _device("cuda")
    for block in (0, 16):
        m = _model("llama", dev, BF16, kv_cache_block=block)
        state = m.new_state(1, 40)
        slot = state.open()
        m.step(state, [slot], [list(range(20))])
        ids = torch.tensor([7], device=dev)
        m.logits(m.step(state, [slot], ids)[0])
        graph = DecodeGraph(m, state, [slot])
        graph.step(ids)
        state.open()
        with pytest.raises(RuntimeError, match="capture"):
            graph.step(ids)


def test_growth_in_slots_and_in_positions_ends_a_graph():
    from types import SimpleNamespace
    from easyllm_b200.models.hf_models.state import DecodeGraph
    replays = []
    graph = DecodeGraph.__new__(DecodeGraph)
    graph.slots, graph.capacity, graph.state_slots, graph.ids, graph.logits = [1], 256, 2, torch.zeros(1, dtype=torch.long), None
    graph.graph = SimpleNamespace(replay=lambda: replays.append(1))
    for capacity, lengths, fine in ((256, [3, 9], True), (256, [3, 9, 0, 0], False), (512, [3, 9], False), (256, [3, 256], False)):
        graph.state = SimpleNamespace(capacity=capacity, slots=len(lengths), lengths=lengths)
        if fine:
            graph.step(torch.ones(1, dtype=torch.long))
        else:
            with pytest.raises(RuntimeError, match="capture"):
                graph.step(torch.ones(1, dtype=torch.long))
    assert len(replays) == 1


def _hybrid(name, dev, dtype, **kw):
    from easyllm_b200.models.hf_models import CausalLM, arch_from_hf_config
    from pafodra_models import CONFIGS
    torch.manual_seed(0)
    m = CausalLM(arch_from_hf_config(dict(CONFIGS[name], **kw)), dtype)
    for n, p in m.named_parameters():                             # states that neither vanish nor blow up, sinks that count
        if n.endswith("sink"):
            p.data.normal_(1.0)
    return m.to(dev).eval()


class Watch:
    """Looks over the calls that a model makes of the cache: keeps, for each layer and sequence, what a cache should hold by the test's own
    count of positions, and holds every answer of the attention against it."""

    def __init__(self, monkeypatch, block):
        self.block, self.held, self.rows, self.appended, self.attended, self.calls = block, {}, [], 0, 0, []
        self.append, self.attend = iops.kv8_append, iops.attention_kv8
        monkeypatch.setattr(iops, "kv8_append", self.on_append)
        monkeypatch.setattr(iops, "attention_kv8", self.on_attend)

    def begin(self, rows):
        """``rows``: (sequence, positions it has, tokens) of the step, in the order of its rows."""
        self.rows, self.layer = rows, -1

    def on_append(self, cache, k, v, meta):
        from test_kv8 import Plain
        self.layer += 1
        self.appended += 1
        self.calls.append((self.layer, k.clone(), v.clone()))
        self.append(cache, k, v, meta)
        r = 0
        for seq, start, n in self.rows:
            held = self.held.setdefault((self.layer, seq), [Plain(384, x.shape[1], x.shape[2], self.block) for x in (k, v)])
            for p, x in zip(held, (k, v)):
                p.append(0, start, x[r:r + n])
            r += n
        assert r == k.shape[0]

    def on_attend(self, q, cache, base, length, max_len, scale, sink=None, slopes=None, **kw):
        got = self.attend(q, cache, base, length, max_len, scale, sink, slopes, **kw)
        self.attended += 1
        r = 0
        for seq, start, n in self.rows:
            for j in range(n):
                if j in (0, 1, n // 2, n - 1):                    # of a prompt some rows
                    keys, values = (p.values(0, start + j + 1) for p in self.held[self.layer, seq])
                    near(got[r + j], *plain_attention(q[r + j], keys, values, scale, sink, slopes))
            r += n
        return got


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["llama", "alibi", "qwen", "aligned", "odd"])
def test_every_layer_attends_to_what_its_cache_should_hold(monkeypatch, device, dtype, kind):
    """Ragged prompts, a state that grows in slots and in positions, decoding, a prompt beside decoding sequences, a slot used again: in
    every layer that attends, hybrid models' too, each answer is that of the rows which a cache kept by the test's own count would hold."""
    from test_kv8 import _model
    dev = _device(device)
    hybrid = kind in ("aligned", "odd")
    m = _hybrid(kind, dev, dtype, kv_cache_block=8) if hybrid else _model(kind, dev, dtype, kv_cache_block=8)
    attending = sum(l.type == "attention" for l in m.arch.layers) if hybrid else 2
    watch = Watch(monkeypatch, 8)
    state = m.new_state(1, 10)
    ids = torch.randint(0, 80, (400,), generator=torch.Generator().manual_seed(1))
    lengths, slots, at, steps = {}, {}, 0, 0
    for step_ in ([("a", 250), ("b", 9)], [("a", 1), ("b", 1)], [("b", 1), ("a", 1)], [("a", 1), ("c", 13), ("b", 2)], [("a", 3)],
                  [("c", 1), ("b", 1), ("a", 1)], ["close b"], [("a", 1), ("d", 21)], [("d", 1), ("c", 1), ("a", 1)]):
        if step_ == ["close b"]:
            state.close(slots["b"])
            continue
        for s, _ in step_:
            if s not in slots:
                slots[s], lengths[s] = state.open(), 0
        watch.begin([(s, lengths[s], n) for s, n in step_])
        m.step(state, [slots[s] for s, _ in step_], [ids[at + i:at + i + n] for i, (_, n) in enumerate(step_)])
        for s, n in step_:
            lengths[s] += n
        at, steps = at + 7, steps + 1
        assert watch.layer == attending - 1
    assert slots["d"] == slots["b"] and state.capacity > 256 and state.slots > 2
    # a step of prompts alone may attend to its own keys, every other one looks into the cache
    assert watch.appended == steps * attending and watch.attended >= (steps - 1) * attending


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["llama", "qwen", "aligned"])
def test_what_a_layer_writes_is_what_it_would_write_in_full(monkeypatch, device, kind):
    """The first attending layer's keys and values of a prompt, as the model without the 8-bit cache hands them to its own."""
    from test_kv8 import _model
    dev = _device(device)
    wrote = {}
    for block in (8, 0):
        m = _hybrid(kind, dev, F32, kv_cache_block=block) if kind == "aligned" else _model(kind, dev, F32, kv_cache_block=block)
        with monkeypatch.context() as patch:
            patch.setattr(iops, "kv8_append", lambda cache, k, v, meta: wrote.setdefault(8, (k.clone(), v.clone())))
            patch.setattr(iops, "attention_kv8", lambda q, cache, *a, **kw: q.new_zeros(*q.shape[:2], cache.vdim))
            patch.setattr(iops, "kv_append", lambda kc, vc, k, v, meta: wrote.setdefault(0, (k.clone(), v.clone())))
            state = m.new_state(2, 40)
            m.step(state, [state.open(), state.open()], [list(range(30)), list(range(5, 16))])
    assert all(torch.equal(a, b) for a, b in zip(wrote[8], wrote[0]))


@pytest.mark.parametrize("device", DEVICES)
def test_a_hybrid_model_generates_from_8_bits(device):
    """Rows of unequal length give the tokens that each gives alone; on a GPU through the captured step as without it."""
    dev = _device(device)
    m = _hybrid("aligned", dev, F32, kv_cache_block=16)
    ids = torch.randint(0, 264, (3, 12), generator=torch.Generator().manual_seed(2)).to(dev)
    mask = torch.ones_like(ids)
    mask[1, :5] = 0
    out = m.generate(ids, attention_mask=mask, max_new_tokens=9)
    assert torch.equal(out[1, 12:], m.generate(ids[1:2, 5:], max_new_tokens=9)[0, 7:])
    assert torch.equal(out, m.generate(ids, attention_mask=mask, max_new_tokens=9, cuda_graph=False))


# ---- rows read back, whatever the rule says ---------------------------------------------------------------------
def read_back(monkeypatch):
    """Calls that can be go to rows read back; the list that is given back gets an entry for each."""
    from easyllm_b200.ops import cuda_infer as ci
    taken, back = [], ci._attention_read_back
    monkeypatch.setattr(ci, "_kv8_reads_back", lambda *a: True)
    monkeypatch.setattr(ci, "_attention_read_back", lambda *a: (taken.append(1), back(*a))[1])
    return taken


@pytest.mark.gpu
@pytest.mark.parametrize("device", ["cuda"])
@pytest.mark.parametrize("H,G,d,dv,new,kind", [(8, 2, 128, 128, [150, 1, 300], None), (8, 1, 64, 32, [70, 131], "sink"), (4, 4, 128, 128, [1, 530], "alibi"),
                                               (12, 2, 48, 128, [90, 1, 1, 200], "window"), (16, 16, 16, 16, [40, 51, 1], None), (64, 2, 96, 80, [3, 2], "sink"),
                                               (40, 1, 112, 128, [33, 5], "window")])
def test_attention_over_rows_read_back(monkeypatch, device, H, G, d, dv, new, kind):
    dev = _device(device)
    taken = read_back(monkeypatch)
    check_attention(dev, BF16, H, G, d, dv, 16, [601 + 77 * i for i in range(len(new))], new, sink=kind == "sink", alibi=kind == "alibi",
                    window=150 if kind == "window" else None)
    check_attention(dev, BF16, H, G, d, dv, 4, [max(new) + 3] + [1] * (len(new) - 1), new, sink=kind == "sink")
    assert len(taken) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("device", ["cuda"])
def test_rows_read_back_keep_what_is_not_finite_and_what_sees_nothing(monkeypatch, device):
    """The cases of such rows, and of rows past two gigabytes, by this way."""
    import test_kv8 as cases
    taken = read_back(monkeypatch)
    cases.test_long_prompts_beside_rows_that_see_nothing(device, BF16)
    cases.test_what_is_not_finite_reaches_the_rows_that_see_it(device, BF16, 60)
    cases.test_rows_that_see_nothing_are_zero(device, BF16, True)
    cases.test_rows_past_two_gigabytes()
    cases.test_steps_of_a_conversation(device, BF16)
    assert len(taken) >= 5


# ---- memory that nobody wrote ---------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("window,kind", [(None, None), (90, None), (None, "sink"), (None, "alibi")])
@pytest.mark.parametrize("H,G,d,dv", [(8, 2, 128, 128), (16, 1, 48, 64)])
def test_rows_read_back_do_not_depend_on_what_lay_behind_them(monkeypatch, H, G, d, dv, window, kind):
    """Long continued prompts of unequal length, a sequence without rows, one whose rows see nothing, rows behind the last border: the bits
    are the same when all memory that the call allocates held NaN before."""
    dev = _device("cuda")
    cap, total, new = 1024, [700, 65, 64, 330], [150, 1, 64, 129]
    cache, plain = filled(4 * cap, G, d, dv, 16, dev)
    meta = step(new, [t - c for t, c in zip(total, new)], [3, 0, 2, 1], cap, dev)
    T, dead = sum(new), 7
    base = torch.cat((meta["kv_base"], ints([5] * dead, dev)))
    length = torch.cat((meta["kv_len"], ints([0, 0, 0, 900, 901, 902, 903], dev)))
    cu = ints(meta["cu_seqlens"].tolist()[:2] + meta["cu_seqlens"].tolist()[1:] + [T + 3], dev)         # the second sequence is empty, the last sees nothing
    q = rand(T + dead, H, d, seed=1).to(BF16).to(dev)
    sink = rand(H, seed=4).to(dev) if kind == "sink" else None
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]).to(dev) if kind == "alibi" else None
    taken = read_back(monkeypatch)

    def call():
        return iops.attention_kv8(q, cache, base, length, 720, 0.1, sink, slopes, window, cu, 160)
    want = call()
    empty, poisoned = torch.empty, []

    def held_nan(*a, **kw):
        t = empty(*a, **kw)
        if t.is_cuda and t.is_floating_point():
            t.fill_(float("nan"))
            poisoned.append(t.numel())
        return t
    with monkeypatch.context() as patch:
        patch.setattr(torch, "empty", held_nan)
        got = call()
    assert len(taken) == 2 and len(poisoned) >= 3 and torch.equal(got, want) and not bool(got[T:].any())
    assert bool(got.isfinite().all())
    r = 0
    for t, n, s in zip(total, new, (3, 0, 2, 1)):
        for j in sorted({0, n // 2, n - 1}):
            end = t - n + j + 1
            low = max(0, end - window) if window else 0
            near(got[r + j], *plain_attention(q[r + j], *(p.values(s * cap + low, end - low) for p in plain), 0.1, sink, slopes))
        r += n


# ---- padded batches ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("G,dv,longest,pad", [(2, 64, 90, 1000), (1, 7, 90, 1000), (2, 12, 1500, 333), (1, 9, 1500, 1), (4, 16, 1500, 2000)])
def test_rows_of_a_padded_batch_are_zero(device, dtype, G, dv, longest, pad):
    """Few tokens in front of many rows behind the last border: every one of those is zero, in memory that held NaN, and no other is."""
    dev = _device(device)
    cap, H, d = 1536, 4, 32
    cache, plain = filled(2 * cap, G, d, dv, 16, dev)
    total, new = [longest, 40], [3, 2]
    meta = step(new, [t - c for t, c in zip(total, new)], [1, 0], cap, dev)
    T = sum(new)
    q = rand(T + pad, H, d, seed=1).to(dtype).to(dev)
    base, length = (torch.cat((meta[n], ints([-1] * pad, dev))) for n in ("kv_base", "kv_len"))
    for _ in range(3):
        held = [torch.full((T + pad, H, dv), float("nan"), dtype=dtype, device=dev) for _ in range(3)]
        del held                                                  # the allocator hands this memory out again
        got = iops.attention_kv8(q, cache, base, length, longest, 0.2, cu_seqlens=meta["cu_seqlens"], max_q=3)
        assert not bool(got[T:].any())
        r = 0
        for t, c, s in zip(total, new, (1, 0)):
            for j in range(c):
                near(got[r], *plain_attention(q[r], *(p.values(s * cap, t - c + j + 1) for p in plain), 0.2))
                r += 1


@pytest.mark.gpu
@pytest.mark.parametrize("back", [False, True])
def test_a_captured_step_takes_any_batch_that_fits_it(monkeypatch, back):
    """A step of a fixed number of rows and sequences, captured once: its replays write and attend for whatever tokens the borders name then,
    the rows behind them are zero, and the bits are those of eager calls."""
    from easyllm_b200.ops import cuda
    dev = _device("cuda")
    G, H, d, cap, T, slots = 2, 8, 64, 1536, 300, 3
    taken = read_back(monkeypatch) if back else []
    cache, plain = filled(slots * cap, G, d, d, 16, dev)
    had, before = [t.clone() for t in cache[:4]], [(p.q.clone(), p.s.clone()) for p in plain]
    k, v, q = (torch.zeros(T, n, d, dtype=BF16, device=dev) for n in (G, G, H))
    meta = {"kv_base": ints([0] * T, dev), "kv_len": ints([0] * T, dev), "cu_seqlens": ints([0] * (slots + 1), dev), "max_seqlen": 200}

    def run():
        iops.kv8_append(cache, k, v, meta)
        return iops.attention_kv8(q, cache, meta["kv_base"], meta["kv_len"], cap, 0.15, cu_seqlens=meta["cu_seqlens"], max_q=200)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i, (counts, start, order) in enumerate([([200, 1, 99], [0, 1300, 40], [2, 0, 1]), ([1, 1, 1], [1535, 0, 17], [0, 1, 2]), ([0, 0, 0], [0, 0, 0], [0, 1, 2]),
                                                ([0, 120, 2], [0, 1400, 999], [1, 2, 0]), ([100, 100, 100], [5, 600, 1234], [0, 2, 1])]):
        m = step(counts, start, order, cap, dev)
        n = sum(counts)
        for name, pad in (("kv_base", -5), ("kv_len", 1 << 30)):  # rows behind the last border say anything
            meta[name].fill_(pad)
            meta[name][:n] = m[name]
        meta["cu_seqlens"].copy_(m["cu_seqlens"])
        for j, t in enumerate((k, v, q)):
            t.copy_(rand(*t.shape, seed=10 * i + j).to(BF16))
        results = []
        for call in (graph.replay, run):
            for t, h in zip(cache[:4], had):
                t.copy_(h)
            got = call()
            results.append([t.clone() for t in cache[:4]] + [(out if got is None else got).clone()])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        got = results[0][-1]
        assert not bool(got[n:].any())
        r = 0
        for c, p0, s in zip(counts, start, order):
            for p, (q0, s0), x in zip(plain, before, (k, v)):     # each step starts from the same cache
                p.q.copy_(q0), p.s.copy_(s0)
                if c:
                    p.append(s * cap, p0, x[r:r + c])
            for j in sorted({0, c // 2, c - 1} if c else ()):
                near(got[r + j], *plain_attention(q[r + j], *(p.values(s * cap, p0 + j + 1) for p in plain), 0.15))
            r += c
    cuda.check_err_flag()
    assert not back or len(taken) >= 7
