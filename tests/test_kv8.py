"""The key/value cache in 8 bits: writing, reading back, attention over it, and models that serve from it, against plain statements
in 64 bits; on the CPU and, marked gpu, the kernels."""
import math

import pytest
import torch

from easyllm_b200.ops import infer as iops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(autouse=True)
def _no_kernel_gave_up(request):
    yield
    if "cuda" in request.node.callspec.params.values() if hasattr(request.node, "callspec") else False:
        from easyllm_b200.ops import cuda
        cuda.check_err_flag()


def _device(name):
    if name == "cuda":
        if not torch.cuda.is_available():
            pytest.skip("no GPU")
        from easyllm_b200.ops import cuda
        cuda.lib()
    return torch.device(name)


def rand(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


def ints(values, dev="cpu"):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def step(counts, start, slots, capacity, dev="cpu"):
    """Index of a step that appends ``counts[i]`` rows to the sequence of ``slots[i]`` that has ``start[i]``."""
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    return {"kv_base": ints([s * capacity for s, c in zip(slots, counts) for _ in range(c)], dev),
            "kv_len": ints([p + j + 1 for p, c in zip(start, counts) for j in range(c)], dev),
            "cu_seqlens": ints(cu, dev), "max_seqlen": max(counts)}


# ---- plain statements in 64 bits ------------------------------------------------------------------
def least_power(amax):
    """Python float ``amax`` → the scale of its block."""
    if not math.isfinite(amax):
        return math.nan
    s = 2.0 ** -126
    while 127 * s < amax and s < 2.0 ** 121:
        s *= 2
    return s


class Plain:
    """A cache as lists of exact numbers: q and scale in 64 bits."""

    def __init__(self, rows, heads, dim, block):
        self.q, self.s, self.block = torch.zeros(rows, heads, dim, dtype=torch.float64), torch.zeros(rows // block, heads, dtype=torch.float64), block

    def append(self, base, start, x):
        x = x.double().cpu()
        B = self.block
        for g in range(x.shape[1]):
            p = start
            while p < start + x.shape[0]:
                b0 = p // B * B
                end = min(b0 + B, start + x.shape[0])
                y = x[p - start:end - start, g]
                s = least_power(float(y.abs().max()) if bool(torch.isfinite(y).all()) else math.nan)
                at = (base + b0) // B
                if p > b0:
                    old = float(self.s[at, g])
                    s = math.nan if math.isnan(old) or math.isnan(s) else max(s, old)
                    self.q[base + b0:base + p, g] = torch.round(self.q[base + b0:base + p, g] * (old / s))
                self.s[at, g] = s
                self.q[base + p:base + end, g] = torch.round(y / s).clamp(-127, 127)
                p = end

    def values(self, first, n):
        at = torch.arange(first, first + n)
        return self.q[at] * self.s[at // self.block].unsqueeze(-1)


def plain_attention(q, k, v, scale, sink=None, slope=None):
    """One query row ``[H, d]`` at the last of the rows k ``[n, G, d]``, v ``[n, G, dv]``: output ``[H, dv]`` and a bound of what 32-bit
    sums may be off by.  A score of d products is off by (d + 16) 2^-24 of its terms' magnitudes, where q is cut to 22 bits of the largest of
    a head by 2^-22 of that besides; a weight by twice the scores' error; the sums of n weights, which may be cut to 22 bits of the largest,
    by (n + 16) 2^-22."""
    q, k, v = q.double().cpu(), k.double(), v.double()
    H, d = q.shape
    n, G = k.shape[:2]
    out, err = torch.zeros(H, v.shape[2], dtype=torch.float64), torch.zeros(H, 1, dtype=torch.float64)
    for h in range(H if n else 0):
        kk, vv = k[:, h // (H // G)], v[:, h // (H // G)]
        s = kk @ q[h] * scale
        terms = (kk.abs() @ q[h].abs()) * scale
        cut = q[h].abs().max() * kk.abs().sum(1) * scale
        if slope is not None:
            bias = float(slope[h]) * (torch.arange(n) - (n - 1)).double()
            s, terms = s + bias, terms + bias.abs()
        t = s if sink is None else torch.cat((s, sink[h].double().cpu().view(1)))
        out[h] = torch.softmax(t, 0)[:n] @ vv
        err[h] = (2 * ((d + 16) * 2.0 ** -24 * terms.max() + 2.0 ** -22 * cut.max()) + (n + 16) * 2.0 ** -22) * vv.abs().max()
    return out, err


def near(got, want, err):
    """Equal but for ``err`` and one rounding to the type of ``got``."""
    bound = err + torch.finfo(got.dtype).eps / 2 * (want.abs() + err)
    d = (got.double().cpu() - want).abs()
    assert got.shape == want.shape and bool((d <= bound).all()), float((d / bound).max())


def filled(rows, heads, dim, vdim, block, dev, seed=0, dtype=F32):
    """A cache of random values of unequal size, and its exact values."""
    cache = iops.kv8_empty(rows, heads, dim, vdim, block)
    plain = []
    x = [rand(rows, heads, w, seed=seed + i) * torch.exp(rand(rows, heads, 1, seed=seed + 9 + i)) for i, w in enumerate((dim, vdim))]
    for q, s, y in ((cache.k, cache.k_scale, x[0]), (cache.v, cache.v_scale, x[1])):
        p = Plain(rows, heads, y.shape[2], block)
        p.append(0, 0, y)
        q[..., :y.shape[2]] = p.q.to(torch.int8)
        s.copy_(p.s.float())
        plain.append(p)
    return cache._replace(**{n: getattr(cache, n).to(dev) for n in ("k", "v", "k_scale", "v_scale")}), plain


# ---- scales ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
def test_scale_is_the_least_power_of_two_that_serves(device):
    dev = _device(device)
    amax = [0.0, 1e-45, 2.0 ** -126, 127 * 2.0 ** -126, 127.0001 * 2.0 ** -126, 1.0, 126.99999, 127.0, 127.00001, 254.0, 255.0, 3.3e38,
            3.4028234e38, math.inf, math.nan]
    x = torch.tensor(amax).view(-1, 1, 1)
    cache = iops.kv8_empty(len(amax), 1, 1, 1, 1, dev)
    n = len(amax)
    iops.kv8_append(cache, x.to(dev), -x.to(dev), step([n], [0], [0], n, dev))
    want = torch.tensor([least_power(float(a)) for a in x.view(-1)])
    for s in (cache.k_scale, cache.v_scale):
        torch.testing.assert_close(s.cpu().view(-1), want.float(), rtol=0, atol=0, equal_nan=True)
    back = iops.kv8_read(cache, ints([0], dev), ints([n], dev), n, F32)[0].view(-1).cpu()
    fine = torch.isfinite(x.view(-1))
    off = (back - x.view(-1)).abs() / want
    top = x.view(-1) > 127 * 2.0 ** 121
    assert bool((off <= 0.5)[fine & ~top].all()) and bool((off <= 1)[fine & top].all()) and bool(back[~fine].isnan().all())


# ---- writing and reading -----------------------------------------------------------------------------
SHAPES = [(1, 1, 16, 16), (2, 16, 128, 128), (3, 8, 72, 40), (1, 128, 7, 100), (5, 4, 24, 128), (8, 32, 128, 64), (2, 64, 80, 16), (1, 2, 3, 1)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("G,block,d,dv", SHAPES)
def test_writes_and_reads_are_exact(device, dtype, G, block, d, dv):
    """Prompts, tokens one by one and turns that go on inside blocks, over slots in any order: every row reads as the definition says,
    to the bit, and rows of slots that the steps leave out stay as they were."""
    dev = _device(device)
    capacity, slots = 256, 5
    cache, plain = filled(slots * capacity, G, d, dv, block, dev, seed=d)
    start = [0, 0, 3, 131, 60]
    steps = [([1, 2, 7], [2, 0, 4]), ([5, 1, 1, 1], [1, 0, 2, 3]), ([1, 1, 1], [0, 2, 4]), ([70, 33, 1, 90], [0, 3, 2, 1]), ([1, 64], [4, 3])]
    for i, (counts, which) in enumerate(steps):
        T = sum(counts)
        wide = (rand(T, G * (d + dv) + 3, seed=i) * torch.exp(2 * rand(T, 1, seed=50 + i))).to(dtype).to(dev)
        k, v = wide[:, 3:3 + G * d].view(T, G, d), wide[:, 3 + G * d:].view(T, G, dv)
        meta = step(counts, [start[s] for s in which], which, capacity, dev)
        iops.kv8_append(cache, k, v, meta)
        at = 0
        for c, s in zip(counts, which):
            for p, x in zip(plain, (k, v)):
                p.append(s * capacity, start[s], x[at:at + c])
            start[s] += c
            at += c
    for out in (F32, BF16):
        got = iops.kv8_read(cache, ints([s * capacity for s in range(slots)], dev), ints([capacity] * slots, dev), capacity, out)
        for x, p in zip(got, plain):
            assert x.dtype == out and torch.equal(x.double().cpu().view(-1, G, x.shape[3]), p.values(0, slots * capacity))
    assert bool((cache.k[..., d:] == 0).all()) and bool((cache.v[..., dv:] == 0).all())


@pytest.mark.parametrize("device", DEVICES)
def test_a_block_filled_row_by_row_is_off_by_less_than_its_scale(device):
    dev = _device(device)
    n = 128
    x = rand(n, 2, 32, seed=3) * torch.exp2(torch.arange(n).view(-1, 1, 1) / 8.0)       # sixteen times the scale grows
    cache = iops.kv8_empty(n, 2, 32, 32, n, dev)
    for p in range(n):
        iops.kv8_append(cache, x[p:p + 1].to(dev), x[p:p + 1].to(dev), step([1], [p], [0], n, dev))
    back = iops.kv8_read(cache, ints([0], dev), ints([n], dev), n, F32)[0][0].cpu()
    assert bool(((back - x).abs() < cache.k_scale.cpu().view(1, 2, 1)).all())


@pytest.mark.parametrize("device", DEVICES)
def test_what_is_not_finite_marks_its_block_and_no_other(device):
    dev = _device(device)
    G, d, B, cap = 3, 32, 8, 256
    cache = iops.kv8_empty(2 * cap, G, d, d, B, dev)
    x = rand(20, G, d, seed=1)
    bad = x.clone()
    bad[10, 1, 5], bad[17, 2, 0], bad[18, 0, 3] = math.nan, math.inf, -math.inf
    iops.kv8_append(cache, bad.to(dev), x.to(dev), step([20], [0], [1], cap, dev))
    iops.kv8_append(cache, x[:5].to(dev), x[:5].to(dev), step([5], [20], [1], cap, dev))       # joins the marked block
    k, v = (t.cpu()[0] for t in iops.kv8_read(cache, ints([cap], dev), ints([25], dev), 25, F32))
    want = torch.zeros(25, G, dtype=torch.bool)
    want[8:16, 1] = want[16:24, 2] = want[16:24, 0] = True
    assert torch.equal(k.isnan().all(-1), want) and torch.equal(k.isnan().any(-1), want) and not bool(v.isnan().any())
    iops.kv8_append(cache, x.to(dev), x.to(dev), step([20], [0], [1], cap, dev))               # the slot's next sequence
    assert not bool(iops.kv8_read(cache, ints([cap], dev), ints([20], dev), 20, F32)[0].isnan().any())


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_are_padding_write_nothing(device):
    """Rows behind the last border, sequences without rows, and sequences of length 0."""
    dev = _device(device)
    cache, plain = filled(512, 2, 32, 16, 16, dev)
    k, v = rand(9, 2, 32, seed=5).to(dev), rand(9, 2, 16, seed=6).to(dev)
    meta = {"kv_base": ints([0, 0, 256, 256, -5, 7, 7, 7, 7], dev), "kv_len": ints([20, 21, 0, 0, 9, 9, 9, 9, 9], dev),
            "cu_seqlens": ints([0, 2, 2, 4, 4], dev), "max_seqlen": 6}
    iops.kv8_append(cache, k, v, meta)
    for p, x in zip(plain, (k, v)):
        p.append(0, 19, x[:2])
    for x, p in zip(iops.kv8_read(cache, ints([0], dev), ints([512], dev), 512, F32), plain):
        assert torch.equal(x[0].double().cpu(), p.values(0, 512))
    iops.kv8_append(cache, k[:0], v[:0], {"kv_base": ints([], dev), "kv_len": ints([], dev), "cu_seqlens": ints([0], dev), "max_seqlen": 0})


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("d,dv", [(128, 128), (40, 24), (9, 3)])
def test_reads_end_with_zeros(device, d, dv):
    dev = _device(device)
    cache, plain = filled(768, 3, d, dv, 16, dev)
    cache.k_scale[-1] = math.nan                                  # nobody reads there
    base, length, most = [256, 0, 512, 16, 752], [0, 1, 37, 60, -3], 37
    for out in (F32, BF16):
        for x, p in zip(iops.kv8_read(cache, ints(base, dev), ints(length, dev), most, out), plain):
            assert x.shape[:2] == (5, most)
            for i, (b, n) in enumerate(zip(base, length)):
                n = min(max(n, 0), most)
                assert torch.equal(x[i, :n].double().cpu(), p.values(b, n)) and not bool(x[i, n:].any())
    assert iops.kv8_read(cache, ints([], dev), ints([], dev), 4)[0].shape == (0, 4, 3, d)
    assert iops.kv8_read(cache, ints([0], dev), ints([1], dev), 0)[0].shape == (1, 0, 3, d)


# ---- attention -----------------------------------------------------------------------------------------
def check_attention(dev, dtype, H, G, d, dv, block, total, new, sink=False, alibi=False, window=None, several=None, qscale=1.0):
    """Sequences of ``total[i]`` rows of which the last ``new[i]`` ask, in slots in reverse order, over rows that hold other things behind
    the ends, NaN among them."""
    n, total = len(total), [max(t, c) for t, c in zip(total, new)]
    capacity = -(-max(total) // 128) * 128
    cache, plain = filled(n * capacity, G, d, dv, block, dev, seed=H + d)
    slots = list(range(n))[::-1]
    for t, s in zip(total, slots):                                # blocks behind the end
        for scale in (cache.k_scale, cache.v_scale):
            scale[(s * capacity + t + block - 1) // block:(s + 1) * capacity // block] = math.nan
    meta = step(new, [t - c for t, c in zip(total, new)], slots, capacity, dev)
    T = sum(new)
    q = (rand(T, H * d + 8, seed=3, scale=qscale).to(dtype).to(dev))[:, 8:].view(T, H, d)
    sk = rand(H, seed=4).to(dev) if sink else None
    sl = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]).to(dev) if alibi else None
    several = max(new) > 1 if several is None else several
    got = iops.attention_kv8(q, cache, meta["kv_base"], meta["kv_len"], max(total), d ** -0.5, sk, sl, window,
                             meta["cu_seqlens"] if several else None, max(new) if several else None)
    assert got.dtype == dtype
    r = 0
    for t, c, s in zip(total, new, slots):
        for j in range(c):
            end = t - c + j + 1
            low = max(0, end - window) if window else 0
            if T > 100 and r % 7 and j not in (0, c - 1):         # of long prompts some rows
                r += 1
                continue
            want, err = plain_attention(q[r], *(p.values(s * capacity + low, end - low) for p in plain), d ** -0.5, sk, sl)
            near(got[r], want, err)
            r += 1


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,G,d,dv,block", [(1, 1, 16, 16, 1), (4, 4, 128, 128, 16), (8, 2, 128, 128, 16), (16, 2, 64, 64, 64), (10, 2, 72, 40, 8),
                                            (20, 1, 24, 128, 32), (3, 3, 100, 7, 2), (34, 2, 128, 96, 128), (5, 5, 1, 1, 4), (16, 1, 96, 128, 16)])
def test_attention_of_single_tokens(device, dtype, H, G, d, dv, block):
    dev = _device(device)
    check_attention(dev, dtype, H, G, d, dv, block, [1, 2, 31, 32, 33, 128, 300, 129, 64], [1] * 9)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,G,d,dv,block", [(4, 4, 128, 128, 16), (8, 2, 128, 128, 1), (20, 1, 24, 128, 32), (34, 2, 128, 96, 128), (3, 3, 100, 7, 2)])
def test_attention_over_lengths_that_shares_cut(device, dtype, H, G, d, dv, block):
    """One sequence beyond 1024 keys among short ones: CTAs take shares of all keys, whose ends cut the sequences anywhere."""
    dev = _device(device)
    check_attention(dev, dtype, H, G, d, dv, block, [1, 1500, 256, 257, 31, 1100], [1] * 6, sink=True)
    check_attention(dev, dtype, H, G, d, dv, block, [1300, 3, 5, 700], [3, 1, 5, 2], window=1200, alibi=True)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["sink", "alibi", "window", "all"])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [3, 1, 2, 5], [40, 1, 77, 130]])
def test_attention_with_sinks_slopes_and_windows(device, dtype, kind, new):
    dev = _device(device)
    check_attention(dev, dtype, 6, 3, 64, 48, 16, [700, 1, 77, 263], new, sink=kind in ("sink", "all"), alibi=kind in ("alibi", "all"),
                    window={"window": 37, "all": 100}.get(kind))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,G,new", [(4, 4, [2, 1, 7]), (8, 1, [2, 2, 2]), (32, 8, [4, 1, 3]), (12, 4, [6, 16, 17]), (40, 2, [3, 1, 1]), (8, 2, [50, 3, 129]),
                                     (8, 8, [64, 1, 200])])
def test_attention_of_several_tokens(device, dtype, H, G, new):
    dev = _device(device)
    check_attention(dev, dtype, H, G, 128, 128, 16, [300, 3, 201], new)
    check_attention(dev, dtype, H, G, 40, 72, 4, [50, 16, 201], new)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_over_many_ranges(device, dtype):
    """Few rows over many keys, with weights that a far key dominates: the ranges are joined."""
    dev = _device(device)
    check_attention(dev, dtype, 4, 2, 128, 128, 64, [9001], [1], qscale=4.0)
    check_attention(dev, dtype, 8, 2, 64, 128, 16, [5003], [3], qscale=0.01)
    check_attention(dev, dtype, 2, 2, 64, 64, 16, [5003, 40], [1, 1], window=4000)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("several", [False, True])
def test_rows_that_see_nothing_are_zero(device, dtype, several):
    """Length 0 with and without a sink, whatever the places; rows behind the last border; sequences without rows."""
    dev = _device(device)
    cache, plain = filled(256, 2, 32, 32, 16, dev)
    cache.v_scale[8:] = math.nan
    q = rand(7, 4, 32, seed=1).to(dtype).to(dev)
    base, length = ints([0, 0, 128, 999, -16, 0, 0], dev), ints([0, 1, 0, 0, 0, 40, 41], dev)
    cu = ints([0, 1, 2, 2, 3, 4, 5], dev) if several else None
    for sink in (None, torch.zeros(4, device=dev)):
        got = iops.attention_kv8(q, cache, base, length, 64, 0.2, sink, None, None, cu, 1 if several else None)
        assert not bool(got[[0, 2, 3, 4]].any())
        near(got[1], *plain_attention(q[1], *(p.values(0, 1) for p in plain), 0.2, sink))
        if several:
            assert not bool(got[5:].any())
        else:
            near(got[6], *plain_attention(q[6], *(p.values(0, 41) for p in plain), 0.2, sink))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 3, 60])
def test_what_is_not_finite_reaches_the_rows_that_see_it(device, dtype, new):
    """A marked block of keys or values makes NaN of the rows that see it, of its head; queries that are not finite are NaN themselves."""
    dev = _device(device)
    n = 100
    cache, _ = filled(256, 2, 64, 64, 16, dev)
    q = rand(2 * new, 4, 64, seed=1).to(dtype).to(dev)
    q[0, 3, 5] = math.inf
    base, cu = ints([0] * new + [128] * new, dev), ints([0, new, 2 * new], dev)
    length = ints(list(range(n - new + 1, n + 1)) * 2, dev)
    cache.k_scale[(128 + 80) // 16, 0] = math.nan                 # keys 80 .. 96 of the second sequence
    cache.v_scale[16 // 16, 1] = math.nan                         # values 16 .. 32 of the first
    got = iops.attention_kv8(q, cache, base, length, n, 0.125, cu_seqlens=cu, max_q=new).float().cpu().isnan().all(-1)
    sees = length.cpu()[:new] > 80
    want = torch.zeros(2 * new, 4, dtype=torch.bool)
    want[:new, 2:] = True
    want[new:, :2] = sees.view(-1, 1)
    want[0, 3] = True
    assert torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_scores_and_values_of_any_size(device):
    """Values near both ends of the range, weights of values of unequal blocks, one key that takes all the weight."""
    dev = _device(device)
    d, n = 32, 96
    for k_size, v_size, q_size in ((1.0, 1e30, 1.0), (1.0, 1e-30, 1.0), (1e18, 1.0, 1e-18), (1e-18, 1.0, 1e18), (20.0, 1.0, 20.0), (0.0, 1.0, 1.0)):
        k, v = rand(n, 1, d, seed=1) * k_size, rand(n, 1, d, seed=2) * v_size
        v[:16] *= 2.0 ** -20                                      # a block of small values
        cache, meta = iops.kv8_empty(128, 1, d, d, 16, dev), step([n], [0], [0], 128, dev)
        iops.kv8_append(cache, k.to(dev), v.to(dev), meta)
        k, v = (t[0].double().cpu() for t in iops.kv8_read(cache, ints([0], dev), ints([n], dev), n, F32))
        q = rand(1, 2, d, seed=3).to(dev) * q_size
        got = iops.attention_kv8(q, cache, ints([0], dev), ints([n], dev), n, 0.2)
        near(got[0], *plain_attention(q[0], k, v, 0.2))


# ---- refusals ------------------------------------------------------------------------------------------
def test_refusals():
    cache = iops.kv8_empty(64, 2, 32, 16, 16)
    for bad in ((64, 2, 129, 16, 16), (64, 2, 32, 0, 16), (64, 2, 32, 16, 3), (64, 2, 32, 16, 256), (60, 2, 32, 16, 16), (64, 2, 32, 16, 0)):
        with pytest.raises(ValueError):
            iops.kv8_empty(*bad)
    one = ints([0])
    q, k, v = torch.zeros(1, 4, 32), torch.zeros(1, 2, 32), torch.zeros(1, 2, 16)
    meta = step([1], [0], [0], 64)
    bad_caches = [cache._replace(k=cache.k[:, :, :16]), cache._replace(k_scale=cache.k_scale[:3]), cache._replace(k_scale=cache.k_scale.double()),
                  cache._replace(v=cache.v.to(torch.uint8)), cache._replace(dim=31 - 16), cache._replace(k=cache.k.transpose(0, 1).contiguous().transpose(0, 1)),
                  cache._replace(k_scale=cache.k_scale[:0], v_scale=cache.v_scale[:0])]
    for c in bad_caches:
        with pytest.raises(ValueError):
            iops.attention_kv8(q, c, one, one, 4, 1.0)
        with pytest.raises(ValueError):
            iops.kv8_append(c, k, v, meta)
        with pytest.raises(ValueError):
            iops.kv8_read(c, one, one, 4)
    for args in ((k[..., :16], v), (k, v.double()), (k[:, :1], v), (torch.zeros(2, 2, 32), torch.zeros(2, 2, 16))):
        with pytest.raises(ValueError):
            iops.kv8_append(cache, *args, meta)
    for name in ("kv_base", "kv_len", "cu_seqlens"):
        with pytest.raises(ValueError):
            iops.kv8_append(cache, k, v, dict(meta, **{name: meta[name].long()}))
    ok = dict(q=q, cache=cache, kv_base=one, kv_len=one, max_len=4, scale=1.0)
    for change in (dict(q=torch.zeros(1, 4, 16)), dict(q=torch.zeros(1, 3, 32)), dict(kv_len=ints([1, 2])), dict(kv_len=one.long()), dict(window=0),
                   dict(sink=torch.zeros(3)), dict(alibi_slopes=torch.zeros(2)), dict(cu_seqlens=ints([0, 1])), dict(cu_seqlens=ints([]), max_q=1)):
        with pytest.raises(ValueError):
            iops.attention_kv8(**{**ok, **change})
    with pytest.raises(ValueError):
        iops.kv8_append(cache, k, v, dict(meta, cu_seqlens=ints([])))
    with pytest.raises(ValueError):
        iops.kv8_append(cache, k, v, dict(meta, cu_seqlens=torch.ones(65537, dtype=torch.int32)))
    with pytest.raises(ValueError):
        iops.kv8_read(cache, torch.zeros(65536, dtype=torch.int32), torch.zeros(65536, dtype=torch.int32), 4)
    with pytest.raises(ValueError):
        iops.kv8_read(cache, one, one, 4, torch.float16)
    with pytest.raises(RuntimeError):
        iops.attention_kv8(**{**ok, "q": q.clone().requires_grad_()})
    with pytest.raises(RuntimeError):
        iops.kv8_append(cache, k.clone().requires_grad_(), v, meta)
    # places outside the cache, or inside a block
    for base, n in ((-16, 1), (8, 1), (48, 17), (64, 1)):
        b, l = ints([base]), ints([n])
        with pytest.raises(ValueError):
            iops.attention_kv8(q, cache, b, l, 64, 1.0)
        with pytest.raises(ValueError):
            iops.kv8_read(cache, b, l, 64)
        with pytest.raises(ValueError):
            iops.kv8_append(cache, k, v, {"kv_base": b, "kv_len": l, "cu_seqlens": ints([0, 1]), "max_seqlen": 1})


@pytest.mark.gpu
@pytest.mark.parametrize("base,n", [(-16, 1), (8, 1), (48, 17), (64, 1), (0x7ffffff0, 16)])
def test_places_outside_the_cache_are_reported(base, n):
    """The kernels look at every place before they touch it: nothing is read or written there, and the error word says so."""
    from easyllm_b200.ops import cuda
    dev = _device("cuda")
    cache, plain = filled(64, 2, 32, 16, 16, dev)
    b, l = ints([base], dev), ints([n], dev)
    calls = [lambda: iops.attention_kv8(torch.ones(1, 4, 32, device=dev), cache, b, l, 64, 1.0),
             lambda: iops.attention_kv8(torch.ones(1, 4, 32, device=dev, dtype=BF16), cache, b, l, 64, 1.0, cu_seqlens=ints([0, 1], dev), max_q=1),
             lambda: iops.kv8_read(cache, b, l, 64)[0],
             lambda: iops.kv8_append(cache, torch.ones(1, 2, 32, device=dev), torch.ones(1, 2, 16, device=dev),
                                     {"kv_base": b, "kv_len": l, "cu_seqlens": ints([0, 1], dev), "max_seqlen": 1})]
    for call in calls:
        out = call()
        with pytest.raises(cuda.KernelError, match="51"):
            cuda.check_err_flag()
        assert out is None or not bool(out.any())
    for x, p in zip(iops.kv8_read(cache, ints([0], dev), ints([64], dev), 64, F32), plain):
        assert torch.equal(x[0].double().cpu(), p.values(0, 64))


@pytest.mark.gpu
def test_bounds_that_are_exceeded_are_reported():
    """More rows of a sequence, or longer ones, than the call was told: the error word is set, and nothing outside is touched."""
    from easyllm_b200.ops import cuda
    dev = _device("cuda")
    cache, plain = filled(1024, 2, 32, 32, 16, dev)
    k, v = rand(70, 2, 32, seed=1).to(dev), rand(70, 2, 32, seed=2).to(dev)
    meta = step([70], [0], [0], 1024, dev)
    iops.kv8_append(cache, k, v, dict(meta, max_seqlen=3))
    with pytest.raises(cuda.KernelError, match="51"):
        cuda.check_err_flag()
    q = rand(300, 4, 32, seed=3).to(BF16).to(dev)
    meta = step([300], [500], [0], 1024, dev)
    cache, plain = filled(1024, 2, 32, 32, 16, dev)
    for max_q, max_len in ((8, 800), (300, 600)):                 # the second through rows read back, whose kernels stop at an error
        got = iops.attention_kv8(q, cache, meta["kv_base"], meta["kv_len"], max_len, 0.2, cu_seqlens=meta["cu_seqlens"], max_q=max_q)
        with pytest.raises(cuda.KernelError, match="51"):
            cuda.check_err_flag()
        for r in range(8 if max_q == 8 else 0):
            near(got[r], *plain_attention(q[r], *(p.values(0, 501 + r) for p in plain), 0.2))


# ---- a run of them together -------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps_of_a_conversation(device, dtype):
    """Prompt, tokens, the next turn, tokens: every step appends and attends, and each row's answer is that of the rows the cache holds
    then."""
    dev = _device(device)
    H, G, d, B, cap = 8, 2, 64, 16, 256
    cache = iops.kv8_empty(2 * cap, G, d, d, B, dev)
    plain = [Plain(2 * cap, G, d, B) for _ in range(2)]
    start = [0, 0]
    for i, counts in enumerate([[45, 7], [1, 1], [1, 1], [1, 30], [60, 1], [1, 1]]):
        T = sum(counts)
        qkv = rand(T, (H + 2 * G) * d, seed=i).to(dtype).to(dev)
        q, k, v = qkv[:, :H * d].view(T, H, d), qkv[:, H * d:(H + G) * d].view(T, G, d), qkv[:, (H + G) * d:].view(T, G, d)
        meta = step(counts, start, [1, 0], cap, dev)
        iops.kv8_append(cache, k, v, meta)
        one = max(counts) == 1
        got = iops.attention_kv8(q, cache, meta["kv_base"], meta["kv_len"], 256, d ** -0.5, cu_seqlens=None if one else meta["cu_seqlens"],
                                 max_q=max(counts))
        r = 0
        for j, (c, s) in enumerate(zip(counts, (1, 0))):
            for p, x in zip(plain, (k, v)):
                p.append(s * cap, start[j], x[r:r + c])
            for e in range(c):
                want, err = plain_attention(q[r + e], *(p.values(s * cap, start[j] + e + 1) for p in plain), d ** -0.5)
                near(got[r + e], want, err)
            r += c
            start[j] += c


def _model(kind, dev, dtype=F32, **kw):
    from easyllm_b200.models.hf_models.modeling import CausalLM, HFArch
    torch.manual_seed(0)
    a = dict(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, eos_token_id=None)
    a.update({"alibi": dict(position="alibi"), "qwen": dict(family="qwen", qkv_bias=True, use_logn_attn=True, seq_length=16)}.get(kind, {}))
    a.update(kw)
    m = CausalLM(HFArch(**a), dtype)
    for p in m.parameters():
        p.data.mul_(3)                                            # scores that differ
    return m.to(dev).eval()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["llama", "alibi", "qwen"])
def test_a_model_that_serves_from_8_bits(device, kind):
    """Ragged prompts and decoding steps: what layers attend to in a model without the cache, with keys and values replaced by what an
    8-bit cache makes of them, gives the same logits; the cache grows, and slots are used again."""
    dev = _device(device)
    m = _model(kind, dev, kv_cache_block=8)
    from easyllm_b200.models.hf_models.state import KV8Rows
    state = m.new_state(1, 10)
    assert all(isinstance(c, KV8Rows) for c in state.layers)
    a, b = state.open(), state.open()                             # the second one makes the state grow
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 97, (300,), generator=g)
    h, meta = m.step(state, [a, b], [ids[:250], ids[:9]])
    for t in range(250, 270):                                     # past the first 256 positions
        h, _ = m.step(state, [a, b], ids[[t, t - 241]].to(dev))
    got = m.logits(h)
    full = _model(kind, dev)
    full.load_state_dict(m.state_dict())
    ref_state = full.new_state(2, 300)
    s = [ref_state.open(), ref_state.open()]
    full.step(ref_state, s, [ids[:250], ids[:9]])
    for t in range(250, 270):
        h, _ = full.step(ref_state, s, ids[[t, t - 241]].to(dev))
    want = full.logits(h)
    # 8 bits of a block's largest: a relative error of up to 2^-7 in keys and values, through two layers
    assert float((got - want).abs().max()) < 0.1 * float(want.abs().max()) and float((got - want).abs().max()) > 0
    state.close(b)
    c = state.open()
    h1, _ = m.step(state, [c], [ids[:30]])
    state2 = m.new_state(1, 30)
    h2, _ = m.step(state2, [state2.open()], [ids[:30]])
    assert torch.equal(h1, h2)


@pytest.mark.parametrize("device", DEVICES)
def test_generation_from_8_bits(device):
    dev = _device(device)
    m = _model("llama", dev, kv_cache_block=16)
    ids = torch.randint(0, 97, (3, 12), generator=torch.Generator().manual_seed(2)).to(dev)
    mask = torch.ones_like(ids)
    mask[1, :5] = 0                                               # rows of unequal length
    out = m.generate(ids, attention_mask=mask, max_new_tokens=9)
    assert out.shape == (3, 21)
    alone = m.generate(ids[1:2, 5:], max_new_tokens=9)
    assert torch.equal(out[1, 12:], alone[0, 7:])
    prefix = {"kv": rand(2, 2, 5, 2, 16, seed=3).to(dev)}
    assert m.generate(ids, max_new_tokens=4, soft_prefix=prefix).shape == (3, 16)


def test_the_cache_is_asked_for_in_the_config():
    from easyllm_b200.models.hf_models.io import export_config
    from easyllm_b200.models.hf_models.modeling import HFArch, arch_from_hf_config
    a = arch_from_hf_config({"model_type": "llama", "kv_cache_block": 16})
    assert a.kv_cache_block == 16 and arch_from_hf_config(export_config(a)).kv_cache_block == 16
    assert "kv_cache_block" not in export_config(HFArch()) and arch_from_hf_config({"model_type": "llama"}).kv_cache_block == 0
    for wrong in (3, 256, -1):
        with pytest.raises(ValueError):
            _model("llama", "cpu", kv_cache_block=wrong).new_state(1, 16)
    with pytest.raises(ValueError):                               # heads of 256
        _model("llama", "cpu", kv_cache_block=16, hidden_size=512, num_attention_heads=2).new_state(1, 16)
    from megozen_models import CONFIGS
    with pytest.raises(ValueError):
        arch_from_hf_config(dict(CONFIGS["odd"], kv_cache_block=16))


# ---- long continued prompts ---------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("device", ["cuda"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,G,d,dv,new,kind", [(8, 2, 128, 128, [150, 1, 300], None), (8, 1, 64, 32, [70, 131], "sink"), (4, 4, 128, 128, [1, 530], "alibi"),
                                               (12, 2, 48, 128, [90, 1, 1, 200], "window"), (16, 2, 72, 128, [100, 20], None)])
def test_attention_of_long_continued_prompts(device, dtype, H, G, d, dv, new, kind):
    """Enough rows for the path through rows read back (bf16), and the same in fp32."""
    dev = _device(device)
    check_attention(dev, dtype, H, G, d, dv, 16, [601 + 77 * i for i in range(len(new))], new, sink=kind == "sink", alibi=kind == "alibi",
                    window=150 if kind == "window" else None)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_prompts_beside_rows_that_see_nothing(device, dtype):
    """A sequence without rows, one whose rows have length 0, rows behind the last border, a marked block."""
    dev = _device(device)
    H, G, d, n, cap = 8, 2, 64, 200, 512
    cache, plain = filled(3 * cap, G, d, d, 16, dev)
    cache.v_scale[(cap + 48) // 16, 1] = math.nan                 # values 48 .. 64 of the second sequence, head 1
    q = rand(2 * n + 9, H, d, seed=1).to(dtype).to(dev)
    base = ints([0] * n + [cap] * n + [3, -1, 777, 1 << 30, 0, 0, 0, 0, 0], dev)
    length = ints(list(range(201, 201 + n)) + list(range(1, n + 1)) + [0, 0, 0, 99, 5, 6, 7, 8, 9], dev)
    cu = ints([0, n, n, 2 * n, 2 * n + 3], dev)
    got = iops.attention_kv8(q, cache, base, length, 401, 0.125, cu_seqlens=cu, max_q=n)
    assert not bool(got[2 * n:].any())
    nan = got.isnan().all(-1).cpu()
    want_nan = torch.zeros(2 * n + 9, H, dtype=torch.bool)
    want_nan[n + 48:2 * n, 4:] = True
    assert torch.equal(nan, want_nan) and torch.equal(got.isnan().any(-1).cpu(), want_nan)
    for r in (0, 1, 77, n - 1, n, n + 1, n + 47):
        seq, end = r // n, 201 + r if r < n else r - n + 1
        near(got[r], *plain_attention(q[r], *(p.values(seq * cap, end) for p in plain), 0.125))


# ---- streams, graphs, devices, places past 32 bits ------------------------------------------------------------
def _calls(dev, seed, dtype=BF16):
    """A step of three sequences as closures over its own buffers: append, attend (in shares, which are joined), read."""
    H, G, d, cap = 8, 2, 128, 2048
    cache, _ = filled(3 * cap, G, d, d, 16, dev, seed=seed)
    meta = step([1, 1, 1], [1300, 17, 2047], [2, 0, 1], cap, dev)
    k, v, q = (rand(3, n, d, seed=seed + i).to(dtype).to(dev) for i, n in enumerate((G, G, H)))
    base, length = meta["kv_base"], meta["kv_len"]

    def run():
        iops.kv8_append(cache, k, v, meta)
        o = iops.attention_kv8(q, cache, base, length, cap, d ** -0.5)
        return (o,) + iops.kv8_read(cache, base, length, cap)
    return run, (k, v, q), cache


@pytest.mark.gpu
def test_two_captured_steps_replay_beside_each_other():
    """Two graphs of steps that share nothing but the library, replayed on two streams at once with new inputs: the bits of eager steps."""
    dev = _device("cuda")
    runs = [_calls(dev, 1), _calls(dev, 100)]
    for run, _, _ in runs:
        run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for run, _, _ in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in runs]
    for i in range(5):
        for j, (_, inputs, _) in enumerate(runs):
            for t in inputs:
                t.copy_(rand(*t.shape, seed=7 * i + j).to(t.dtype))
        torch.cuda.synchronize()
        kept = [tuple(t.clone() for t in cache[:4]) for _, _, cache in runs]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        got = [tuple(t.clone() for t in o) for o in outs]
        for (run, _, cache), before, g in zip(runs, kept, got):
            for t, b in zip(cache[:4], before):
                t.copy_(b)
            for a, b in zip(g, run()):
                assert torch.equal(a, b)
    from easyllm_b200.ops import cuda
    cuda.check_err_flag()


@pytest.mark.gpu
def test_on_another_stream_and_again_on_the_same_inputs():
    dev = _device("cuda")
    run, _, _ = _calls(dev, 5)
    want = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [run() for _ in range(20)]
    s.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.gpu
def test_rows_past_two_gigabytes():
    """A cache of more than 2^31 bytes: the places of its last rows."""
    dev = _device("cuda")
    G, d, B, rows = 16, 128, 16, (1 << 20) + 4096
    cache = iops.kv8_empty(rows, G, d, d, B, dev)
    assert cache.k.numel() > 1 << 31
    n, base = 301, rows - 512
    k, v, q = (rand(n, h, d, seed=h + i).to(BF16).to(dev) for i, h in enumerate((G, G, 2 * G)))
    meta = {"kv_base": ints([base] * n, dev), "kv_len": ints(list(range(1, n + 1)), dev), "cu_seqlens": ints([0, n], dev), "max_seqlen": n}
    iops.kv8_append(cache, k, v, meta)
    plain = [Plain(512, G, d, B) for _ in range(2)]
    for p, x in zip(plain, (k, v)):
        p.append(0, 0, x)
    for x, p in zip(iops.kv8_read(cache, ints([base], dev), ints([n], dev), n, F32), plain):
        assert torch.equal(x[0].double().cpu(), p.values(0, n))
    near(iops.attention_kv8(q[-1:], cache, ints([base], dev), ints([n], dev), n, 0.1)[0], *plain_attention(q[-1], *(p.values(0, n) for p in plain), 0.1))
    got = iops.attention_kv8(q, cache, meta["kv_base"], meta["kv_len"], n, 0.1, cu_seqlens=meta["cu_seqlens"], max_q=n)
    near(got[-1], *plain_attention(q[-1], *(p.values(0, n) for p in plain), 0.1))


@pytest.mark.gpu
def test_a_decoding_model_replays_its_graph():
    """Generation with and without the captured decode step gives the same tokens, in bf16, and so does a state that is used again."""
    dev = _device("cuda")
    m = _model("llama", dev, BF16, kv_cache_block=16, hidden_size=512, num_attention_heads=4, num_key_value_heads=2)
    ids = torch.randint(0, 97, (3, 40), generator=torch.Generator().manual_seed(3)).to(dev)
    a = m.generate(ids, max_new_tokens=24)
    b = m.generate(ids, max_new_tokens=24, cuda_graph=False)
    assert a.shape == (3, 64) and torch.equal(a, b) and torch.equal(a, m.generate(ids, max_new_tokens=24))


@pytest.mark.gpu
def test_arguments_are_looked_over_on_a_gpu_too():
    dev = _device("cuda")
    cache = iops.kv8_empty(64, 2, 32, 16, 16, dev)
    one = ints([0], dev)
    with pytest.raises(ValueError):                               # an index on the host
        iops.attention_kv8(torch.zeros(1, 4, 32, device=dev), cache, ints([0]), one, 4, 1.0)
    with pytest.raises(ValueError):                               # queries on the host
        iops.attention_kv8(torch.zeros(1, 4, 32), cache, one, one, 4, 1.0)
    with pytest.raises(ValueError):                               # heads that are not packed
        iops.attention_kv8(torch.zeros(2, 32, 4, device=dev).transpose(1, 2), cache, ints([0, 0], dev), ints([1, 1], dev), 4, 1.0)
    with pytest.raises(ValueError):
        iops.attention_kv8(torch.zeros(1, 4, 32, device=dev), cache, one, one, 4, 1.0, sink=torch.zeros(4))
    with pytest.raises(ValueError):
        iops.kv8_append(cache, torch.zeros(1, 2, 32), torch.zeros(1, 2, 16), step([1], [0], [0], 64, dev))
