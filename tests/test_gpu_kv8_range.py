"""pi05_kv8_attention over caches whose rows differ widely in size, against 64 bits.

The bound is a sum over the keys that a row sees: each weight is off by its logit's error (the fp32 sum of head_dim products,
the base-2 exponent's rounding), 2^-22 of the exponential, the fp32 sums over the keys, and one rounding of the weight:
fp16, 2^-11 of it or 2^-25 of the largest weight where it is subnormal.  A key that a row does not see, or whose weight is 0, adds
nothing, whatever its size."""
import math

import pytest
import torch
from launched import assert_launches
from test_gpu_fp8 import BF, decode, gen, i32, new_cache, randn

pytestmark = pytest.mark.gpu

FP16, BF16 = 2.0**-11, 2.0**-8  # half a step of a weight


@pytest.fixture(autouse=True)
def _check_device(pn):
    yield
    pn.fp8_status()  # no bounded wait gave up


def bounded(got, q, cache, lens, slots=None, causal=False, scale=None, weight=FP16, floor=2.0**-110):
    """asserts got against the definition; returns nothing"""
    B, T, H, hd = q.shape
    N, cap, kvh, _ = cache[0].shape
    scale = hd**-0.5 if scale is None else scale
    for b in range(B):
        sl = int(slots[b]) if slots is not None else b
        n = min(max(int(lens[b]), 0), cap)
        if n == 0:
            assert (got[b] == 0).all()
            continue
        k, v = decode(cache[0][sl, :n], cache[1][sl, :n].long()), decode(cache[2][sl, :n], cache[3][sl, :n].long())
        seen = torch.ones(T, n, dtype=torch.bool, device="cuda")
        if causal:
            seen = torch.arange(n, device="cuda")[None] < (n - T + 1 + torch.arange(T, device="cuda"))[:, None]
        for h in range(H):
            kh, vh, qh = k[:, h // (H // kvh)], v[:, h // (H // kvh)], q[b, :, h].double()
            s = (qh @ kh.t() * scale).masked_fill(~seen, -math.inf)
            mag = torch.where(seen, qh.abs() @ kh.abs().t() * abs(scale), 0).amax(-1, keepdim=True)
            top = torch.where(seen, s.abs(), 0).amax(-1, keepdim=True)
            p = torch.softmax(s, -1)
            p[~seen.any(-1)] = 0
            dl = mag * (hd + 8) * 2.0**-23 + top * 2.0**-22
            dp = p * (2 * dl + 2.0**-22 + weight + (n + 16) * 2.0**-23) + p.clamp(max=2.0**-25)
            ref, tol = p @ vh, dp @ vh.abs()
            tol = tol + 2.0**-8 * (ref.abs() + tol) + floor
            off = (got[b, :, h].double() - ref).abs()
            worst = (off / tol).nan_to_num(nan=1e9).max().item()
            assert worst <= 1, f"sample {b}, head {h}: {worst:.3g} of the tolerance"


# (batch, T, heads, kv_heads, head_dim, capacity) that reach each kernel
ROWS = [(1, 40, 8, 2, 128, 64), (2, 1, 8, 1, 256, 300), (3, 7, 6, 2, 64, 150)]
ROWS_SPLIT = [(1, 1, 8, 1, 256, 20000), (1, 3, 8, 2, 64, 40000)]
KERNELS = {"rows": "kv8_attn_rows_kernel", "tc": "kv8_attn_tc_kernel"}


def run(pn, kernel, q, cache, lens, **kw):
    call = lambda: pn.kv8_attention(q, *cache, lens=lens, **kw)  # noqa: E731
    got = call()
    assert_launches(call, *([KERNELS[kernel]] if isinstance(kernel, str) else kernel))
    return got


def written(pn, k, v):
    B, n, kvh, hd = k.shape
    cache = new_cache(B, n, kvh, hd)
    pn.kv8_write(k.to(BF), v.to(BF), *cache)
    return cache


def one_large_hidden_value(pn, kernel, shape, large):
    """V rows of 1 and a last one that only the last token sees: all others give the mean of ones"""
    B, T, H, kvh, hd, n = shape
    k = torch.zeros(B, n, kvh, hd, device="cuda")
    v = torch.ones(B, n, kvh, hd, device="cuda")
    v[:, n - 1] = large
    q = torch.zeros(B, T, H, hd, device="cuda", dtype=BF)
    got = run(pn, kernel, q, written(pn, k, v), torch.full((B,), n, device="cuda", dtype=torch.int32), causal=True).float()
    first = max(T - n, 0)  # the first token that sees a key
    assert (got[:, :first] == 0).all() and ((got[:, first:-1] - 1).abs() <= 2.0**-8).all()
    last = (n - 1 + float(v[0, -1, 0, 0].to(BF).double())) / n
    assert ((got[:, -1].double() - last).abs() <= 2.0**-4 * last).all()  # the value itself is rounded to e4m3


def far_apart(pn, kernel, shape, causal, seed, spread, weight=FP16, floor=2.0**-110):
    """every V row of its own size, 2^-spread to 2^spread; some rows of zeros"""
    B, T, H, kvh, hd, n = shape
    g = gen(seed)
    k = randn(g, B, n, kvh, hd)
    v = randn(g, B, n, kvh, hd) * torch.exp2(torch.randint(-spread, spread + 1, (B, n, kvh, 1), device="cuda", generator=g).float())
    v[:, 3::7] = 0
    q = randn(g, B, T, H, hd, dtype=BF)
    cache = written(pn, k, v)
    lens = torch.arange(n, n - B, -1, device="cuda").int()
    bounded(run(pn, kernel, q, cache, lens, causal=causal), q, cache, lens, causal=causal, weight=weight, floor=floor)


@pytest.mark.parametrize("large", [2.0**9, 2.0**16, 2.0**30, 2.0**90, 3.3e38])
@pytest.mark.parametrize("shape", [ROWS[0], (2, 5, 8, 1, 256, 300), (3, 9, 6, 2, 64, 150)])
def test_rows_kernel_large_hidden_value(pn, shape, large):
    one_large_hidden_value(pn, "rows", shape, large)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("spread", [4, 8, 40])
@pytest.mark.parametrize("shape", ROWS + ROWS_SPLIT)
def test_rows_kernel_values_far_apart(pn, shape, spread, causal):
    far_apart(pn, "rows", shape, causal, 41, spread)


def test_rows_kernel_values_growing_and_shrinking(pn):
    """sizes that wander over 2^-60 .. 2^60 and back along the cache: the window of exponents has to follow both ways"""
    g = gen(42)
    B, T, H, kvh, hd, n = 1, 2, 8, 1, 128, 4000
    e = 60 * torch.sin(torch.arange(n, device="cuda") / 150.0)
    v = randn(g, B, n, kvh, hd) * torch.exp2(e)[None, :, None, None]
    k = randn(g, B, n, kvh, hd)
    q = randn(g, B, T, H, hd, dtype=BF)
    cache = written(pn, k, v)
    for lens in (i32(n), i32(471), i32(940)):
        bounded(run(pn, "rows", q, cache, lens), q, cache, lens)


def test_rows_kernel_tiny_values(pn):
    """V rows next to the smallest exponent"""
    g = gen(43)
    v = randn(g, 1, 200, 1, 128) * 2.0**-115
    k = randn(g, 1, 200, 1, 128)
    q = randn(g, 1, 1, 8, 128, dtype=BF)
    cache = written(pn, k, v)
    bounded(run(pn, "rows", q, cache, i32(200)), q, cache, i32(200), floor=2.0**-126)


# ---- the tcgen05 kernel: weights of a tile whose scales span more than 2^22 are bf16
TC = [(2, 130, 8, 1, 256, 150), (8, 200, 8, 2, 128, 64), (4, 200, 8, 1, 128, 150), (8, 400, 8, 1, 64, 300)]
TC_SPLIT = [(1, 968, 8, 1, 256, 968)]


@pytest.mark.parametrize("large", [2.0**9, 2.0**16, 2.0**30, 2.0**90, 3.3e38])
@pytest.mark.parametrize("shape", TC)
def test_tcgen05_kernel_large_hidden_value(pn, shape, large):
    one_large_hidden_value(pn, "tc", shape, large)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("spread", [4, 8, 40])
@pytest.mark.parametrize("shape", TC + TC_SPLIT)
def test_tcgen05_kernel_values_far_apart(pn, shape, spread, causal):
    far_apart(pn, "tc", shape, causal, 44, spread, weight=BF16 if spread > 8 else FP16)


def test_tcgen05_kernel_values_growing_and_shrinking(pn):
    g = gen(45)
    B, T, H, kvh, hd, n = 2, 150, 8, 1, 128, 4000
    e = 60 * torch.sin(torch.arange(n, device="cuda") / 400.0)
    v = randn(g, B, n, kvh, hd) * torch.exp2(e)[None, :, None, None]
    k = randn(g, B, n, kvh, hd)
    q = randn(g, B, T, H, hd, dtype=BF)
    cache = written(pn, k, v)
    for lens in (i32(n, 1256), i32(471, 940)):
        bounded(run(pn, "tc", q, cache, lens), q, cache, lens, weight=BF16)


def test_tcgen05_kernel_wide_tiles_among_others(pn):
    """tiles of 64 keys by turns of one size, far apart, and of another size: the weights' type changes from tile to tile"""
    g = gen(46)
    B, T, H, kvh, hd, n = 4, 200, 8, 1, 128, 64 * 9 + 5
    v = randn(g, B, n, kvh, hd)
    e = torch.zeros(n, device="cuda")
    e[64:128] = torch.randint(-30, 30, (64,), device="cuda", generator=g).float()
    e[256:320] = 40
    e[384:448] = torch.randint(-60, 60, (64,), device="cuda", generator=g).float()
    e[576] = 100
    v *= torch.exp2(e)[None, :, None, None]
    k = randn(g, B, n, kvh, hd)
    q = randn(g, B, T, H, hd, dtype=BF)
    cache = written(pn, k, v)
    for causal in (False, True):
        lens = i32(n, 577, 380, 250)
        bounded(run(pn, "tc", q, cache, lens, causal=causal), q, cache, lens, causal=causal, weight=BF16)


def test_tcgen05_kernel_tiny_values(pn):
    g = gen(47)
    v = randn(g, 4, 150, 1, 128) * 2.0**-115
    k = randn(g, 4, 150, 1, 128)
    q = randn(g, 4, 200, 8, 128, dtype=BF)
    cache = written(pn, k, v)
    lens = i32(150, 100, 64, 3)
    bounded(run(pn, "tc", q, cache, lens), q, cache, lens, weight=BF16, floor=2.0**-126)


# ---- key splits joined through a workspace
@pytest.mark.parametrize("shape,kernel", [(ROWS_SPLIT[0], ["kv8_attn_rows", "kv8_attn_combine"]), (TC_SPLIT[0], ["kv8_attn_tc", "kv8_attn_combine"])])
@pytest.mark.parametrize("size", [1.0, 2.0**120, 3.0e38])
def test_partials_of_the_largest_values_are_finite(pn, shape, kernel, size):
    """V next to the largest finite number: no weighted average of it is larger"""
    B, T, H, kvh, hd, n = shape
    g = gen(48)
    v = (0.5 + 0.5 * torch.rand(B, n, kvh, hd, device="cuda", generator=g)) * size
    k = randn(g, B, n, kvh, hd)
    q = randn(g, B, T, H, hd, dtype=BF)
    cache = written(pn, k, v)
    got = run(pn, kernel, q, cache, i32(n))
    assert torch.isfinite(got).all()
    bounded(got / size, q, (cache[0], cache[1], cache[2], (cache[3].int() - int(math.log2(size))).to(torch.uint8)), i32(n)) if size < 3e38 else None


@pytest.mark.parametrize("large", [2.0**30, 3.3e38])
def test_large_hidden_value_with_splits(pn, large):
    one_large_hidden_value(pn, "tc", TC_SPLIT[0], large)


# ---- logits of ordinary size from very large and very small factors
@pytest.mark.parametrize("qe,ke", [(116, -114), (-114, 116), (-60, 62), (62, -60), (100, -100), (-100, 100)])
@pytest.mark.parametrize("kernel,shape", [("rows", ROWS[0]), ("rows", ROWS[1]), ("tc", TC[0]), ("tc", TC[2]), ("tc", TC[3])])
def test_large_keys_and_small_queries_or_the_reverse(pn, kernel, shape, qe, ke):
    B, T, H, kvh, hd, n = shape
    g = gen(49)
    q = (randn(g, B, T, H, hd) * 2.0**qe).to(BF)
    k = randn(g, B, n, kvh, hd) * 2.0**ke
    k[:, 5::9] *= 2.0**-8  # smaller rows beside them
    v = randn(g, B, n, kvh, hd)
    cache = written(pn, k, v)
    lens = torch.arange(n, n - B, -1, device="cuda").int()
    bounded(run(pn, kernel, q, cache, lens, causal=True), q, cache, lens, causal=True)


@pytest.mark.parametrize("kernel,shape", [("rows", ROWS[1]), ("tc", TC[0])])
def test_queries_and_keys_both_large_but_orthogonal(pn, kernel, shape):
    """products of zeros: the weights are equal however large the factors"""
    B, T, H, kvh, hd, n = shape
    g = gen(50)
    q, k = torch.zeros(B, T, H, hd, device="cuda"), torch.zeros(B, n, kvh, hd, device="cuda")
    q[..., : hd // 2] = randn(g, B, T, H, hd // 2) * 2.0**100
    k[..., hd // 2 :] = randn(g, B, n, kvh, hd // 2) * 2.0**100
    v = randn(g, B, n, kvh, hd)
    cache = written(pn, k, v)
    lens = torch.full((B,), n, device="cuda", dtype=torch.int32)
    q = q.to(BF)
    bounded(run(pn, kernel, q, cache, lens), q, cache, lens)


@pytest.mark.parametrize("kernel,shape", [("rows", ROWS[0]), ("rows", (2, 5, 8, 1, 256, 300)), ("tc", TC[0]), ("tc", TC[2]), ("tc", TC[3]), ("tc", TC_SPLIT[0])])
def test_values_2_to_the_180_apart(pn, kernel, shape):
    """the range that the header names: V near 2^-54 beside one row of 2^126 that only the last token sees"""
    B, T, H, kvh, hd, n = shape
    g = gen(51)
    k = randn(g, B, n, kvh, hd)
    v = (1 + torch.rand(B, n, kvh, hd, device="cuda", generator=g)) * 2.0**-54
    v[:, n - 1] = 2.0**126
    q = randn(g, B, T, H, hd, dtype=BF)
    cache, lens = written(pn, k, v), torch.full((B,), n, device="cuda", dtype=torch.int32)
    got = run(pn, kernel, q, cache, lens, causal=True)
    bounded(got, q, cache, lens, causal=True, weight=FP16 if kernel == "rows" else BF16, floor=2.0**-85)


# one key behind whole steps of 32 and tiles of 64, so that it has a step, a warp, a tile, a CTA of a cluster or a split to itself
ALONE = [("rows", (1, 40, 8, 2, 128, 65)), ("rows", (1, 3, 8, 1, 256, 129)), ("rows", (1, 3, 8, 1, 256, 33)), ("rows", (1, 2, 8, 1, 256, 2049)),
         ("rows", (1, 2, 8, 2, 64, 1025)), ("rows", (1, 2, 8, 1, 256, 20001)), ("tc", (2, 130, 8, 1, 256, 129)), ("tc", (4, 200, 8, 1, 128, 193)),
         ("tc", (8, 400, 8, 1, 64, 257)), ("tc", (1, 968, 8, 1, 256, 961)), ("tc", (2, 300, 8, 1, 128, 1025))]


@pytest.mark.parametrize("large", [2.0**30, 2.0**70, 2.0**100, 3.3e38])
@pytest.mark.parametrize("kernel,shape", ALONE)
def test_large_hidden_value_alone_in_its_step(pn, kernel, shape, large):
    one_large_hidden_value(pn, kernel, shape, large)


@pytest.mark.parametrize("where", ["first", "middle", "last", "a tile"])
@pytest.mark.parametrize("kernel,shape", ALONE)
def test_large_values_without_weight(pn, kernel, shape, where):
    """keys whose logits are e^-900 below the others, with V of 3e38: they count for nothing, before, among and behind the rest"""
    B, T, H, kvh, hd, n = shape
    g = gen(52)
    k, v = randn(g, B, n, kvh, hd), randn(g, B, n, kvh, hd)
    q = randn(g, B, T, H, hd)
    q[..., 0] = 30.0
    at = {"first": [0], "middle": [n // 2], "last": [n - 1], "a tile": list(range(min(64, n - 2)))}[where]
    k[:, at] = 0
    k[:, at, :, 0] = -30.0 * math.sqrt(hd)
    v[:, at] = 2.0**126
    cache, lens = written(pn, k, v), torch.full((B,), n, device="cuda", dtype=torch.int32)
    q = q.to(BF)
    got = run(pn, kernel, q, cache, lens)
    bounded(got, q, cache, lens, weight=FP16 if kernel == "rows" else BF16, floor=2.0**-60)


@pytest.mark.parametrize("qe,ke,scale", [(-100, 118, 1e-30), (-126, 118, 1e-30), (100, -100, 0.1), (10, 20, 1e-38)])
@pytest.mark.parametrize("kernel,shape", [("rows", ROWS[0]), ("tc", TC[0]), ("tc", TC[2]), ("tc", TC[3])])
def test_factors_at_the_ends_of_the_float_range(pn, kernel, shape, qe, ke, scale):
    """logits that vanish though a factor of theirs is next to the largest, and keys of ordinary logits beside a hidden huge one"""
    B, T, H, kvh, hd, n = shape
    g = gen(53)
    q = (randn(g, B, T, H, hd) * 2.0**qe).to(BF)
    k = randn(g, B, n, kvh, hd) * 2.0**ke
    if ke < 0:
        k[:, n - 1] = randn(g, B, kvh, hd) * 2.0**116
        q[:, T - 1] = 0  # the token that sees it
    v = randn(g, B, n, kvh, hd)
    cache, lens = written(pn, k, v), torch.full((B,), n, device="cuda", dtype=torch.int32)
    bounded(run(pn, kernel, q, cache, lens, causal=True, scale=scale), q, cache, lens, causal=True, scale=scale)


@pytest.mark.parametrize("kernel,shape", [("rows", ROWS[0]), ("rows", ROWS_SPLIT[0]), ("tc", TC[1]), ("tc", TC_SPLIT[0])])
def test_far_apart_values_again_on_streams_and_from_a_graph(pn, kernel, shape):
    """the bf16 products too give the same bits each time: twice at once, and replayed on a cache that has changed between wide and
    narrow"""
    B, T, H, kvh, hd, n = shape
    g = gen(54)
    k = randn(g, B, n, kvh, hd)
    wide = randn(g, B, n, kvh, hd) * torch.exp2(torch.randint(-40, 41, (B, n, kvh, 1), device="cuda", generator=g).float())
    caches = [written(pn, k, wide), written(pn, k, randn(g, B, n, kvh, hd))]
    q, lens = randn(g, B, T, H, hd, dtype=BF), torch.full((B,), n, device="cuda", dtype=torch.int32)
    want = [run(pn, kernel, q, c, lens) for c in caches]
    side = [torch.cuda.Stream() for _ in caches]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for c, s in zip(caches, side):
            with torch.cuda.stream(s):
                got.append(pn.kv8_attention(q, *c, lens=lens))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))
    live = [t.clone() for t in caches[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pn.kv8_attention(q, *live, lens=lens)
    for i in (0, 1, 0, 1, 1, 0):
        for a, b in zip(live, caches[i]):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, want[i])
