"""pi05_fp8_linear at sizes that reach the CTA-pair kernel with several tiles a cluster (74 clusters on 148 SMs), and the
128-token tiles of the few-token kernel in clusters along K.  Each test asserts which kernel ran."""
import math

import pytest
import torch
from launched import assert_launches
from test_gpu_fp8 import BF, E4M3, _saved, check_linear, gen, operand, randn

pytestmark = pytest.mark.gpu

# tokens, features, K: 144 tiles of 240 features (rows of no 16-byte multiple, K of five blocks); 207 of 192; 144 of 144 with a
# K that ends 8 into a block; 144 with a K of 34 blocks (scale words of three pieces a tile)
PAIR = [(1800, 4306, 640), (2100, 4304, 1152), (2000, 2570, 1160), (2100, 2304, 4304)]
FEW = [(768, 1152, 4304), (700, 1170, 6000), (601, 1158, 4008)]


@pytest.fixture(autouse=True)
def _check_device(pn):
    yield
    pn.fp8_status()  # no bounded wait gave up


def reaches(pn, kernel, x, xs, w, ws, epi="store", **kw):
    assert_launches(lambda: pn.fp8_linear(x, xs, w, ws, epi=epi, **kw), kernel)


def case(pn, seed, T, F, K, epi, with_bias, spread=0.5):
    g = gen(seed)
    x, w = operand(pn, g, T, K, spread), operand(pn, g, F, K, spread)
    bias = randn(g, F, dtype=BF) if with_bias else None
    res = randn(g, T, F, dtype=BF) if epi in ("resid", "gated") else None
    gate = randn(g, F, dtype=BF) if epi == "gated" else None
    return x, w, bias, res, gate


@pytest.mark.parametrize("epi", ["store", "gelu", "resid", "gated", "geglu", "f32"])
@pytest.mark.parametrize("T,F,K", PAIR)
def test_pair_epilogues(pn, T, F, K, epi):
    x, w, bias, res, gate = case(pn, T + F + K, T, F, K, epi, (F + K) % 3 != 0)
    check_linear(pn, *x, *w, epi, bias, res, gate)
    reaches(pn, "fp8_pair_kernel", *x, *w, epi=epi, bias=bias, res=res, gate=gate)


@pytest.mark.parametrize("epi", ["store", "gelu", "resid", "gated", "geglu", "f32"])
@pytest.mark.parametrize("T,F,K", FEW)
def test_128_token_clusters(pn, T, F, K, epi):
    x, w, bias, res, gate = case(pn, T + F + K + 1, T, F, K, epi, epi != "store")
    check_linear(pn, *x, *w, epi, bias, res, gate)
    reaches(pn, "fp8_few_kernelILi128E", *x, *w, epi=epi, bias=bias, res=res, gate=gate)


@pytest.mark.parametrize("T,F,K", PAIR)
def test_pair_residual_in_place(pn, T, F, K):
    x, w, bias, res, _ = case(pn, 61, T, F, K, "resid", True)
    _saved["res"] = res.clone()
    check_linear(pn, *x, *w, "resid", bias, res=res, out=res)


@pytest.mark.parametrize("T,F,K,kernel", [(1801, 4306, 648, "fp8_pair_kernel"), (2000, 2570, 1160, "fp8_pair_kernel"),
                                          (601, 1158, 4008, "fp8_few_kernelILi128E")])
def test_strided_operands_and_rows_behind(pn, T, F, K, kernel):
    g = gen(62)
    (xq, xs), (wq, ws) = operand(pn, g, T, K), operand(pn, g, F, K)

    def spread(q, s, pad):  # inside larger buffers whose other bytes are NaN codes and NaN scales
        big = torch.full((q.shape[0] + 2, -(-q.shape[1] // 16) * 16 + pad), 0x7F, device="cuda", dtype=torch.uint8)
        sb = torch.full((q.shape[0] + 2, -(-s.shape[1] // 4) * 4 + 4), 255, device="cuda", dtype=torch.uint8)
        big[: q.shape[0], : q.shape[1]] = q.view(torch.uint8)
        sb[: q.shape[0], : s.shape[1]] = s
        return big.view(E4M3)[: q.shape[0], : q.shape[1]], sb[: q.shape[0], : s.shape[1]]

    x, w = spread(xq, xs, 16), spread(wq, ws, 48)
    want = pn.fp8_linear(xq, xs, wq, ws)
    out = torch.full((T + 3, F), 5.0, device="cuda", dtype=BF)
    got = check_linear(pn, *x, *w, "store", out=out[:T])
    reaches(pn, kernel, *x, *w)
    assert torch.equal(got, want) and (out[T:] == 5).all()


@pytest.mark.parametrize("T,F,K,kernel", [(1800, 4306, 640, "fp8_pair_kernel"), (2100, 2304, 4304, "fp8_pair_kernel"),
                                          (601, 1158, 4008, "fp8_few_kernelILi128E")])
def test_nan_rows_stay_their_own(pn, T, F, K, kernel):
    g = gen(63)
    x, w = randn(g, T, K), randn(g, F, K)
    rows, feats = [0, T // 2, T - 1], [17, F - 1]
    for i, r in enumerate(rows):
        x[r, (i * 301) % K] = math.nan
    for f in feats:
        w[f, K - 1] = math.inf
    xq, wq = pn.fp8_quantize(x), pn.fp8_quantize(w)
    y = pn.fp8_linear(*xq, *wq, epi="f32")
    reaches(pn, kernel, *xq, *wq, epi="f32")
    bad = torch.zeros(T, F, dtype=torch.bool, device="cuda")
    bad[rows], bad[:, feats] = True, True
    assert torch.equal(torch.isnan(y), bad)


@pytest.mark.parametrize("T,F,K,kernel", [(1800, 4306, 640, "fp8_pair_kernel"), (2100, 2304, 4304, "fp8_pair_kernel"),
                                          (768, 1152, 4304, "fp8_few_kernelILi128E")])
def test_scales_far_apart(pn, T, F, K, kernel):
    """scales from 2^-60 to 2^60 within a row: a scale word read for the wrong row, block or tile would show"""
    g = gen(64)
    blocks = -(-K // 128)
    e = torch.randint(-60, 60, (T, blocks), device="cuda", generator=g).float().repeat_interleave(128, 1)[:, :K]
    x, w = pn.fp8_quantize(randn(g, T, K) * torch.exp2(e)), operand(pn, g, F, K)
    check_linear(pn, *x, *w, "f32")
    reaches(pn, kernel, *x, *w, epi="f32")


@pytest.mark.parametrize("ex,ew", [(118, -118), (-118, 118), (60, 60), (-60, -60)])
@pytest.mark.parametrize("T,F,K", [(4, 136, 256), (2100, 4304, 1152)])
def test_scales_at_the_ends_of_their_range(pn, T, F, K, ex, ew):
    """the two scales of a product may each be far outside what their sum is"""
    g = gen(65)
    x = pn.fp8_quantize(randn(g, T, K) * 2.0**ex)
    w = pn.fp8_quantize(randn(g, F, K) * 2.0**ew)
    check_linear(pn, *x, *w, "f32")


@pytest.mark.parametrize("T,F,K", PAIR)
def test_pair_reruns_are_identical(pn, T, F, K):
    g = gen(66)
    x, w = operand(pn, g, T, K), operand(pn, g, F, K)
    a = pn.fp8_linear(*x, *w, epi="f32")
    for _ in range(20):
        assert torch.equal(a, pn.fp8_linear(*x, *w, epi="f32"))


@pytest.mark.parametrize("T,F,K", [PAIR[0], FEW[0]])
def test_two_streams_and_a_graph(pn, T, F, K):
    """two calls at once, and one replayed, give the eager bits"""
    g = gen(67)
    runs = [(operand(pn, g, T, K), operand(pn, g, F, K)) for _ in range(2)]
    want = [pn.fp8_linear(*x, *w) for x, w in runs]
    side = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for (x, w), s in zip(runs, side):
            with torch.cuda.stream(s):
                got.append(pn.fp8_linear(*x, *w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = pn.fp8_linear(*runs[0][0], *runs[0][1])
    y.fill_(-1)
    gr.replay()
    assert torch.equal(y, want[0])


@pytest.mark.parametrize("T", [1793, 1799, 1823, 1825, 1855])
def test_pair_with_warps_across_the_last_token(pn, T):
    """the last token inside a warp's 32: its lanes behind it sit out the epilogue's arithmetic and no more"""
    F, K = 4306, 640
    for epi in ("gelu", "f32"):
        x, w, bias, _, _ = case(pn, 68 + T, T, F, K, epi, True)
        check_linear(pn, *x, *w, epi, bias)
        reaches(pn, "fp8_pair_kernel", *x, *w, epi=epi, bias=bias)
