"""The special cases of pi05_kv8_attention on both of its kernels, held to the bound over the keys that a row sees
(test_gpu_kv8_range.py); each test asserts which kernel ran."""
import math

import pytest
import torch
from test_gpu_fp8 import BF, E4M3, filled, gen, i32, randn
from test_gpu_kv8_range import bounded, run, written

pytestmark = pytest.mark.gpu

# kernel, (batch, T, heads, kv_heads, head_dim, capacity)
BOTH = [("rows", (2, 2, 8, 1, 256, 150)), ("rows", (2, 20, 8, 2, 128, 150)), ("rows", (2, 9, 6, 2, 64, 150)),
        ("tc", (2, 130, 8, 1, 256, 150)), ("tc", (4, 200, 8, 1, 128, 150)), ("tc", (8, 400, 8, 1, 64, 300))]


@pytest.fixture(autouse=True)
def _check_device(pn):
    yield
    pn.fp8_status()  # no bounded wait gave up


def inputs(pn, seed, shape, spread=1.0):
    B, T, H, kvh, hd, n = shape
    g = gen(seed)
    return g, randn(g, B, T, H, hd, dtype=BF), filled(pn, g, B, n, kvh, hd, spread), torch.arange(n, n - B, -1, device="cuda").int()


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 1e-12, -1e-30, 1e30])
@pytest.mark.parametrize("kernel,shape", BOTH)
def test_scales_and_small_queries(pn, kernel, shape, scale):
    _, q, cache, lens = inputs(pn, 81, shape)
    q *= 0.3 if abs(scale) <= 1 else 2.0**-100
    q[:, :, 3] = 0
    q[:, :, 4] *= 2.0**-20 if abs(scale) > 1 else 2.0**-120
    bounded(run(pn, kernel, q, cache, lens, scale=scale, causal=True), q, cache, lens, scale=scale, causal=True)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kernel,shape", BOTH)
def test_what_lies_behind_the_length(pn, kernel, shape, causal):
    """NaN codes and NaN scales in positions that no row sees, in whole slots and behind lengths inside a tile"""
    B, T, H, kvh, hd, n = shape
    _, q, cache, _ = inputs(pn, 82, shape)
    lens = torch.arange(n - 5, n - 5 - 9 * B, -9, device="cuda").int()
    for c in cache:
        for b in range(B):
            c.view(torch.uint8)[b, int(lens[b]) :] = 0x7F if c.dtype == E4M3 else 255
    bounded(run(pn, kernel, q, cache, lens, causal=causal), q, cache, lens, causal=causal)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("kernel,shape", BOTH)
def test_a_nan_row_of_the_cache(pn, kernel, shape, which):
    """NaN for the tokens that see it, under the causal limit, and nothing for the others"""
    B, T, H, kvh, hd, n = shape
    g = gen(83)
    k, v = randn(g, B, n, kvh, hd, dtype=BF), randn(g, B, n, kvh, hd, dtype=BF)
    q = randn(g, B, T, H, hd, dtype=BF)
    clean = written(pn, k, v)
    lens = torch.full((B,), n, device="cuda", dtype=torch.int32)
    want = pn.kv8_attention(q, *clean, lens=lens, causal=True)
    at = n - max(1, T // 3) - 1
    (k if which == "k" else v)[:, at, 0, 5] = math.nan
    got = run(pn, kernel, q, written(pn, k, v), lens, causal=True)
    sees = (n - T + 1 + torch.arange(T, device="cuda") > at)[None, :, None].expand(B, T, H).clone()
    sees[:, :, H // kvh :] = False  # the other K/V heads
    assert torch.equal(torch.isnan(got).all(-1), sees) and torch.equal(torch.isnan(got).any(-1), sees)
    # the running maximum and the V window may move at other keys: equal to the rounding of the output and of the weights
    off = (got.float() - want.float()).abs()[~sees]
    assert (off <= 2.0**-7 * want.float().abs()[~sees] + 2.0**-9).all()


@pytest.mark.parametrize("kernel,shape", BOTH)
def test_logits_far_apart(pn, kernel, shape):
    """growing keys, so that the running maximum moves often; large, tiny and lopsided queries"""
    B, T, H, kvh, hd, n = shape
    g = gen(84)
    k = randn(g, B, n, kvh, hd) * torch.linspace(0.01, 30, n, device="cuda")[None, :, None, None]
    v = randn(g, B, n, kvh, hd)
    q = randn(g, B, T, H, hd)
    q[:, :, 0] *= 100
    q[:, :, 1] *= 2.0**-100
    q[:, :, 2] = 0
    q[:, :, 3, 1:] *= 2.0**-20
    q = q.to(BF)
    cache, lens = written(pn, k, v), torch.arange(n, n - B, -1, device="cuda").int()
    for causal in (False, True):
        bounded(run(pn, kernel, q, cache, lens, causal=causal), q, cache, lens, causal=causal)


LENGTHS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kernel,T", [("rows", 1), ("tc", 60)])
def test_lengths_next_to_tiles(pn, kernel, T, hd, causal):
    g = gen(85)
    B, cap = len(LENGTHS), 260
    cache = filled(pn, g, B, cap, 1, hd)
    q = randn(g, B, T, 8, hd, dtype=BF)
    lens = i32(*LENGTHS)
    bounded(run(pn, kernel, q, cache, lens, causal=causal), q, cache, lens, causal=causal)


@pytest.mark.parametrize("kernel,shape", BOTH)
def test_strided_query_and_out(pn, kernel, shape):
    B, T, H, kvh, hd, n = shape
    g, _, cache, lens = inputs(pn, 86, shape)
    wide = randn(g, B, T + 3, (H + 2) * hd, dtype=BF)
    q = wide[:, :T, : H * hd].unflatten(2, (H, hd))
    big = torch.full((B, T + 1, (H + 1) * hd), 3.0, device="cuda", dtype=BF)
    out = big[:, :T, : H * hd].unflatten(2, (H, hd))
    got = run(pn, kernel, q, cache, lens, out=out)
    assert torch.equal(got, pn.kv8_attention(q.contiguous(), *cache, lens=lens))
    assert (big[:, T:] == 3).all() and (big[..., H * hd :] == 3).all()
    bounded(got, q, cache, lens)


@pytest.mark.parametrize("kernel,shape", BOTH)
def test_out_may_be_the_query(pn, kernel, shape):
    _, q, cache, lens = inputs(pn, 87, shape)
    want = run(pn, kernel, q, cache, lens, causal=True)
    assert torch.equal(pn.kv8_attention(q, *cache, lens=lens, causal=True, out=q), want)


@pytest.mark.parametrize("heads,kvh,hd,B,T,cap", [(8, 1, 256, 1, 1, 20000), (8, 1, 256, 2, 50, 1018), (8, 1, 256, 1, 968, 968),
                                                  (16, 4, 128, 1, 300, 3001), (8, 8, 64, 2, 257, 700), (4, 1, 128, 1, 129, 4097),
                                                  (8, 2, 64, 1, 1, 70001)])
@pytest.mark.parametrize("causal", [False, True])
def test_long_caches_key_by_key(pn, heads, kvh, hd, B, T, cap, causal):
    """the sum over seen keys of each weight's own error, at lengths where a bound by the largest |v| would let zeros pass"""
    g = gen(88 + cap + T)
    cache = filled(pn, g, B, cap, kvh, hd)
    q = randn(g, B, T, heads, hd, dtype=BF)
    lens = torch.arange(cap, cap - B, -1, device="cuda").int()
    bounded(pn.kv8_attention(q, *cache, lens=lens, causal=causal), q, cache, lens, causal=causal)


@pytest.mark.parametrize("kernel,T", [("rows", 1), ("tc", 140)])
def test_small_weights_add_up(pn, kernel, T):
    """one key with most of the weight and 60,000 near 2^-21 of it, V of one sign: their sum keeps a weight's 2^-25"""
    cap, hd = 60001, 64
    k, v = torch.zeros(1, cap, 1, hd, device="cuda"), torch.ones(1, cap, 1, hd, device="cuda")
    k[0, 0, 0, 0], v[0, 0] = 1.0, 0.0
    cache = written(pn, k, v)
    q = torch.zeros(1, T, 8, hd, device="cuda", dtype=BF)
    q[..., 0] = 14.5
    got = run(pn, kernel, q, cache, i32(cap), scale=1.0)
    w = (cap - 1) * math.exp(-14.5)
    ref = w / (1 + w)
    # weights of 2^-20.9: fp16 with V's window 2^9 above it, or 2^7 p, is normal from 2^-23 or 2^-21 on, so each is off by at
    # most 2^-11 of itself, or 2^-25 / 2^7 (subnormal); the fp32 sums by 60,000 * 2^-23
    rel = 2.0**-11 + 2.0**-32 / math.exp(-14.5) + cap * 2.0**-23 + 2.0**-20 + 14.5 * 1.45 * 2.0**-22
    assert (got.double() - ref).abs().max() <= (rel + 2.0**-8) * ref


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kernel,shape", [("tc", (8, 400, 8, 1, 64, 5)), ("tc", (8, 200, 8, 1, 128, 3)), ("tc", (8, 200, 8, 1, 256, 1)),
                                          ("rows", (3, 1, 40, 8, 128, 1)), ("rows", (2, 3, 71, 1, 64, 300)), ("tc", (16, 2, 96, 1, 128, 700)),
                                          ("tc", (8, 30, 71, 1, 128, 400)), ("tc", (64, 3, 71, 1, 256, 300))])
def test_caches_smaller_than_a_tile_and_odd_groups(pn, kernel, shape, causal):
    """capacities of 1 to 5 positions; 71 and 96 query heads on one, so that tokens straddle the row tiles"""
    B, T, H, kvh, hd, n = shape
    g = gen(89)
    q, cache = randn(g, B, T, H, hd, dtype=BF), filled(pn, g, B, n, kvh, hd)
    lens = torch.randint(0, n + 2, (B,), device="cuda", generator=g).int()
    lens[0] = n
    bounded(run(pn, kernel, q, cache, lens, causal=causal), q, cache, lens, causal=causal)
