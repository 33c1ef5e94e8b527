"""The 8-bit operators against plain 64-bit restatements.

Tolerances come from the formats.  Quantisation, writing and reading are exact by definition (a power-of-two scale, one
rounding to e4m3 or bf16): equality.  The products are held to: one rounding of the result (bf16: 2^-8 of it; fp32: 2^-24) plus
the fp32 sums, at most (number of terms) * 2^-23 of the sum of magnitudes, plus what the epilogue or the softmax adds,
written where it is used."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3, BF = torch.float8_e4m3fn, torch.bfloat16


@pytest.fixture(autouse=True)
def _check_device(pn):
    yield
    pn.fp8_status()  # no bounded wait gave up


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


# ---------------------------------------------------------------- the format, in 64 bits
def encode(x):
    """(codes as values, exponent bytes) of the last axis"""
    x = x.double()
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], 0.0, x)
    top = x.abs().amax(-1)
    e = torch.full_like(top, -127)
    for cand in range(127, -128, -1):  # the smallest e that holds the largest magnitude
        e = torch.where(top <= 448 * 2.0**cand, float(cand), e)
    e = torch.where(top == 0, -127.0, e)
    y = x / torch.exp2(e)[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0**-6))) - 3)
    codes = torch.round(y / step) * step
    return codes, torch.where(bad, 255, e + 127).long()


def decode(codes, byte):
    s = torch.where(byte == 255, math.nan, torch.exp2(byte.double() - 127))
    return codes.double() * s[..., None]


def blocks_of(x):
    n, c = x.shape
    nb = -(-c // 128)
    full = torch.zeros(n, nb * 128, device=x.device, dtype=x.dtype)
    full[:, :c] = x
    return full.view(n, nb, 128)


def values(q, s):
    return decode(blocks_of(q.float()), s.long()).flatten(1)[:, : q.shape[1]]


# ---------------------------------------------------------------- quantise
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 17), (50, 1024), (7, 1152), (129, 4304), (33, 200), (2, 2056),
                                       (1000, 72), (5, 8)])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_quantize(pn, rows, cols, dtype):
    g = gen(rows * 31 + cols)
    x = (randn(g, rows, cols) * torch.exp2(20 * randn(g, rows, 1))).to(dtype)
    q, s = pn.fp8_quantize(x)
    codes, byte = encode(blocks_of(x))
    assert q.dtype == E4M3 and q.shape == x.shape and torch.equal(s.long(), byte)
    assert torch.equal(q.double(), codes.flatten(1)[:, :cols])


def test_quantize_special_values(pn):
    x = torch.zeros(12, 256, device="cuda")
    x[1, 5] = 448.0
    x[2, 5] = math.nextafter(448.0, 1e9)
    x[2, 5] = x[2, 5] + 2**-15 * 448
    x[3, 130] = math.nan
    x[4, 0] = math.inf
    x[5, 1] = -math.inf
    x[6, 3], x[6, 4] = 2.0**-149, -(2.0**-130)  # subnormal
    x[7, 9], x[7, 10] = 3.4e38, 1.0
    x[8, :128] = torch.linspace(-448, 448, 128, device="cuda")
    x[9, :16] = torch.tensor([1.0625, 1.1875, 1.3125, 17, 19, 21, 2**-9, 2**-10, 3 * 2**-10, 2**-10 * 1.001, 0.5, -0.0, 448, 432, 440, 424],
                             device="cuda")  # ties and the smallest codes
    q, s = pn.fp8_quantize(x)
    codes, byte = encode(blocks_of(x))
    assert torch.equal(s.long(), byte) and torch.equal(q.double(), codes.flatten(1))
    assert s[3].tolist() == [0, 255] and s[4, 0] == 255 and s[0].tolist() == [0, 0]
    b, _ = pn.fp8_quantize(x.to(BF))
    assert torch.isfinite(b.float()).all()


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_quantize_strided_rows_and_untouched_padding(pn, dtype):
    g = gen(5)
    wide = randn(g, 37, 311).to(dtype)
    for x in (wide[:, 3:203], wide[::2, :136], wide[:, 8:264]):  # misaligned, strided, aligned for no type
        rows, cols = x.shape
        nb = -(-cols // 128)
        qs = torch.full((rows, 320), 3, device="cuda", dtype=torch.uint8)
        ss = torch.full((rows, 8), 77, device="cuda", dtype=torch.uint8)
        pn.fp8_quantize(x, out=(qs.view(E4M3)[:, :cols], ss[:, :nb]))
        codes, byte = encode(blocks_of(x.contiguous()))
        assert torch.equal(qs.view(E4M3)[:, :cols].double(), codes.flatten(1)[:, :cols])
        assert torch.equal(ss[:, :nb].long(), byte)
        assert (qs[:, cols:] == 3).all() and (ss[:, nb:] == 77).all()


# ---------------------------------------------------------------- linear
def operand(pn, g, rows, k, spread=2.0):
    return pn.fp8_quantize(randn(g, rows, k) * torch.exp2(spread * randn(g, rows, 1)))


def gelu(z):
    return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))


def check_linear(pn, x, xs, w, ws, epi, bias=None, res=None, gate=None, out=None):
    got = pn.fp8_linear(x, xs, w, ws, epi=epi, bias=bias, res=res.clone() if res is not None and out is None else res, gate=gate, out=out)
    X, W = values(x, xs), values(w, ws)
    y, mag = X @ W.t(), X.abs() @ W.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    err = (x.shape[1] + 8) * 2.0**-23 * mag  # the sum in fp32
    if epi == "gelu":
        err = 1.13 * err + 2.0**-19 * y.abs()  # |gelu'| <= 1.13; its exponential and quotient
        y = gelu(y)
    elif epi == "geglu":
        a, u, ea, eu = y[:, 0::2], y[:, 1::2], err[:, 0::2], err[:, 1::2]
        ga = gelu(a)
        ea = 1.13 * ea + 2.0**-19 * a.abs()
        y, err = ga * u, ea * u.abs() + ga.abs() * eu + ea * eu
    elif epi == "resid":
        y = res0(res, out) + y
    elif epi == "gated":
        y, err = res0(res, out) + y * gate.double(), err * gate.double().abs()
    assert got.shape == y.shape and got.dtype == (torch.float32 if epi == "f32" else BF)
    tol = err + (2.0**-24 if epi == "f32" else 2.0**-8) * (y.abs() + err) + 2.0**-126
    off = (got.double() - y).abs()
    assert (off <= tol).all(), f"{(off / tol).max().item():.3g} of the tolerance"
    return got


_saved = {}


def res0(res, out):
    return _saved["res"].double() if out is not None and out is res else res.double()


SHAPES = [(1, 8, 16), (1, 1, 1), (3, 130, 72), (16, 256, 128), (50, 1024, 1024), (50, 8192, 1024), (64, 2560, 2048), (65, 66, 129),
          (127, 384, 640), (128, 128, 512), (129, 257, 513), (200, 4304, 1152), (256, 1152, 4304), (300, 96, 2064), (777, 1000, 336),
          (968, 2560, 2048), (1031, 520, 4096)]


@pytest.mark.parametrize("T,F,K", SHAPES)
def test_linear_store(pn, T, F, K):
    g = gen(T + F + K)
    check_linear(pn, *operand(pn, g, T, K), *operand(pn, g, F, K), "store")


@pytest.mark.parametrize("epi", ["gelu", "resid", "gated", "geglu", "f32"])
@pytest.mark.parametrize("T,F,K", [(1, 2, 16), (50, 1024, 1024), (50, 8192, 1024), (33, 130, 200), (129, 258, 272), (512, 512, 2048),
                                   (700, 1158, 1152)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear_epilogues(pn, T, F, K, epi, with_bias):
    g = gen(T * 7 + F + K)
    x, w = operand(pn, g, T, K, 0.5), operand(pn, g, F, K, 0.5)
    bias = randn(g, F, dtype=BF) if with_bias else None
    res = randn(g, T, F, dtype=BF) if epi in ("resid", "gated") else None
    gate = randn(g, F, dtype=BF) if epi == "gated" else None
    check_linear(pn, *x, *w, epi, bias, res, gate)


@pytest.mark.parametrize("T", [20, 300])
def test_linear_residual_in_place(pn, T):
    g = gen(3)
    x, w = operand(pn, g, T, 256), operand(pn, g, 264, 256)
    res = randn(g, T, 264, dtype=BF)
    _saved["res"] = res.clone()
    check_linear(pn, *x, *w, "resid", res=res, out=res)


@pytest.mark.parametrize("T", [9, 150, 520])
def test_linear_strided_operands_and_rows_behind(pn, T):
    g = gen(11)
    F, K = 200, 300
    xq, xs = operand(pn, g, T, K)
    wq, ws = operand(pn, g, F, K)

    def spread(q, s, pad):  # inside larger buffers whose other bytes are NaN codes and NaN scales
        big = torch.full((q.shape[0] + 2, 320 + pad), 0x7F, device="cuda", dtype=torch.uint8)
        sb = torch.full((q.shape[0] + 2, 8), 255, device="cuda", dtype=torch.uint8)
        big[: q.shape[0], : q.shape[1]] = q.view(torch.uint8)
        sb[: q.shape[0], : s.shape[1]] = s
        return big.view(E4M3)[: q.shape[0], : q.shape[1]], sb[: q.shape[0], : s.shape[1]]

    want = pn.fp8_linear(xq, xs, wq, ws)
    out = torch.full((T + 3, F), 5.0, device="cuda", dtype=BF)
    got = check_linear(pn, *spread(xq, xs, 16), *spread(wq, ws, 48), "store", out=out[:T])
    assert torch.equal(got, want) and (out[T:] == 5).all()


@pytest.mark.parametrize("T", [5, 140, 600])
def test_linear_nan_rows_stay_their_own(pn, T):
    g = gen(13)
    x = randn(g, T, 384)
    x[T // 2, 200] = math.nan
    xq, xs = pn.fp8_quantize(x)
    w = randn(g, 264, 384)
    w[17, 0] = math.inf
    wq, ws = pn.fp8_quantize(w)
    y = pn.fp8_linear(xq, xs, wq, ws, epi="f32")
    bad = torch.zeros(T, 264, dtype=torch.bool, device="cuda")
    bad[T // 2], bad[:, 17] = True, True
    assert torch.equal(torch.isnan(y), bad)


@pytest.mark.parametrize("T", [4, 200, 600])
def test_linear_scales_far_apart(pn, T):
    """scales from 2^-60 to 2^60 within one row: the largest blocks decide, as in the fp32 sum of the definition"""
    g = gen(17)
    x = randn(g, T, 1024) * torch.exp2(torch.randint(-60, 60, (T, 8), device="cuda", generator=g).float()).repeat_interleave(128, 1)
    check_linear(pn, *pn.fp8_quantize(x), *operand(pn, g, 136, 1024), "f32")


@pytest.mark.parametrize("T,F,K", [(50, 2048, 2048), (500, 1024, 1024)])
def test_linear_reruns_are_identical(pn, T, F, K):
    g = gen(19)
    x, w = operand(pn, g, T, K), operand(pn, g, F, K)
    a = pn.fp8_linear(*x, *w, epi="f32")
    for _ in range(5):
        assert torch.equal(a, pn.fp8_linear(*x, *w, epi="f32"))


# ---------------------------------------------------------------- the cache
def new_cache(n, cap, kvh, hd, fill=0x7F, scale=255):
    k8 = torch.full((n, cap, kvh, hd), fill, device="cuda", dtype=torch.uint8).view(E4M3)
    ks = torch.full((n, cap, kvh), scale, device="cuda", dtype=torch.uint8)
    return k8, ks, k8.clone(), ks.clone()


def i32(*v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


LAYOUTS = [(1, 256), (2, 128), (8, 64), (3, 256), (1, 64)]


@pytest.mark.parametrize("kvh,hd", LAYOUTS)
@pytest.mark.parametrize("B,T", [(1, 1), (3, 50), (5, 131)])
def test_write_and_read(pn, kvh, hd, B, T):
    g = gen(B * T + hd)
    n, cap = B + 2, T + 20
    k = randn(g, B, T, kvh, hd, dtype=BF) * torch.exp2(4 * randn(g, B, T, 1, 1)).to(BF)
    v = randn(g, B, T, kvh, hd, dtype=BF)
    k[0, 0, 0] = 0
    slots = torch.randperm(n, device="cuda", generator=g)[:B].int()
    start = torch.randint(0, 21, (B,), device="cuda", generator=g).int()
    count = torch.randint(0, T + 1, (B,), device="cuda", generator=g).int()
    count[0] = T
    cache = new_cache(n, cap, kvh, hd)
    want = [t.clone() for t in cache]
    pn.kv8_write(k, v, *cache, start=start, count=count, slots=slots)
    for x, c, s in ((k, want[0], want[1]), (v, want[2], want[3])):
        codes, byte = encode(x)
        for b in range(B):
            sl, p, m = int(slots[b]), int(start[b]), int(count[b])
            c[sl, p : p + m] = codes[b, :m].float().to(E4M3)
            s[sl, p : p + m] = byte[b, :m].to(torch.uint8)
    for got, ref in zip(cache, want):
        assert torch.equal(got.view(torch.uint8) & 0x7F if got.dtype == E4M3 else got, ref.view(torch.uint8) & 0x7F if ref.dtype == E4M3 else ref)
        if got.dtype == E4M3:  # signs of codes that are not zero
            assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(ref.float()))
    ko, vo = torch.full_like(k, 7), torch.full_like(v, 7)
    pn.kv8_read(*cache, start=start, T=T, count=count, slots=slots, out=(ko, vo))
    for o, x in ((ko, k), (vo, v)):
        ref = decode(*encode(x)).to(BF)
        for b in range(B):
            m = int(count[b])
            assert torch.equal(o[b, :m], ref[b, :m]) and (o[b, m:] == 7).all()


def test_write_defaults_and_read_of_whole_slots(pn):
    g = gen(2)
    k, v = randn(g, 3, 10, 1, 256, dtype=BF), randn(g, 3, 10, 1, 256, dtype=BF)
    cache = new_cache(3, 10, 1, 256)
    pn.kv8_write(k, v, *cache)
    ko, vo = pn.kv8_read(*cache)
    assert torch.equal(ko, decode(*encode(k)).to(BF)) and torch.equal(vo, decode(*encode(v)).to(BF))


def test_rows_outside_the_cache_are_passed_over(pn):
    g = gen(4)
    k = randn(g, 6, 8, 2, 128, dtype=BF)
    cache = new_cache(4, 16, 2, 128, fill=1, scale=9)
    before = [t.clone() for t in cache]
    # a negative slot, one too large, positions before the cache, behind it, far behind it, and a count above T
    pn.kv8_write(k, k, *cache, start=i32(0, 0, -3, 12, 2**31 - 1, 4), count=i32(8, 8, 8, 8, 8, 99), slots=i32(-1, 4, 0, 1, 2, 3))
    codes, byte = encode(k)
    for i, (c, s) in enumerate(((0, 1), (2, 3))):
        w8, ws = before[c].clone(), before[s].clone()
        w8[0, 0:5], ws[0, 0:5] = codes[2, 3:].float().to(E4M3), byte[2, 3:].to(torch.uint8)
        w8[1, 12:16], ws[1, 12:16] = codes[3, :4].float().to(E4M3), byte[3, :4].to(torch.uint8)
        w8[3, 4:12], ws[3, 4:12] = codes[5].float().to(E4M3), byte[5].to(torch.uint8)
        assert torch.equal(cache[c].float(), w8.float()) and torch.equal(cache[s], ws)
    ko = torch.full_like(k, 7)
    vo = ko.clone()
    pn.kv8_read(*cache, start=i32(0, 0, -3, 12, 2**31 - 1, 4), T=8, slots=i32(-1, 4, 0, 1, 2, 3), out=(ko, vo))
    assert (ko[:2] == 7).all() and (ko[2, :3] == 7).all() and (ko[3, 4:] == 7).all() and (ko[4] == 7).all()
    ref = decode(codes, byte).to(BF)
    assert torch.equal(vo[2, 3:], ref[2, 3:]) and torch.equal(vo[3, :4], ref[3, :4]) and torch.equal(vo[5], ref[5])


def test_write_the_same_place_twice_keeps_the_later_sample(pn):
    g = gen(6)
    k = randn(g, 4, 40, 1, 256, dtype=BF)
    for _ in range(5):
        cache = new_cache(2, 64, 1, 256)
        pn.kv8_write(k, k, *cache, start=i32(0, 10, 0, 20), count=i32(40, 40, 5, 40), slots=i32(1, 1, 0, 1))
        ko, _ = pn.kv8_read(*cache)
        ref = decode(*encode(k)).to(BF)
        assert torch.equal(ko[1, :10], ref[0, :10]) and torch.equal(ko[1, 10:20], ref[1, :10]) and torch.equal(ko[1, 20:60], ref[3])
        assert torch.equal(ko[0, :5], ref[2, :5])


def test_write_strided_rows_of_a_fused_projection(pn):
    g = gen(8)
    qkv = randn(g, 2, 20, 2560, dtype=BF)  # 8 query heads, k, v of 256
    k, v = qkv[..., 2048:2304].unflatten(2, (1, 256)), qkv[..., 2304:].unflatten(2, (1, 256))
    cache, ref = new_cache(2, 32, 1, 256), new_cache(2, 32, 1, 256)
    pn.kv8_write(k, v, *cache)
    pn.kv8_write(k.contiguous(), v.contiguous(), *ref)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, ref))


def test_a_row_with_nan_or_infinity_reads_as_nan(pn):
    k = torch.ones(1, 4, 2, 128, device="cuda", dtype=BF)
    v = k.clone()
    k[0, 1, 0, 3], v[0, 2, 1, 0] = math.nan, -math.inf
    cache = new_cache(1, 4, 2, 128)
    pn.kv8_write(k, v, *cache)
    ko, vo = pn.kv8_read(*cache)
    for o, x in ((ko, k), (vo, v)):
        bad = ~torch.isfinite(x).all(-1)
        assert torch.equal(torch.isnan(o).all(-1), bad) and torch.equal(torch.isnan(o).any(-1), bad)


# ---------------------------------------------------------------- attention
def check_attention(pn, q, cache, lens, slots=None, causal=False, scale=None, out=None):
    got = pn.kv8_attention(q, *cache, lens=lens, slots=slots, causal=causal, scale=scale, out=out)
    B, T, H, hd = q.shape
    N, cap, kvh, _ = cache[0].shape
    G = H // kvh
    scale = hd**-0.5 if scale is None else scale
    worst = 0.0
    for b in range(B):
        sl = int(slots[b]) if slots is not None else b
        n = min(max(int(lens[b]), 0), cap) if 0 <= sl < N else 0
        if n == 0:
            assert (got[b] == 0).all()
            continue
        k, v = decode(cache[0][sl, :n], cache[1][sl, :n].long()), decode(cache[2][sl, :n], cache[3][sl, :n].long())
        k, v = (t.repeat_interleave(G, 1).transpose(0, 1) for t in (k, v))  # [H][n][hd]
        qq = q[b].double().transpose(0, 1)
        s = qq @ k.transpose(1, 2) * scale
        mag = qq.abs() @ k.abs().transpose(1, 2) * abs(scale)
        if causal:
            seen = torch.arange(n, device="cuda")[None] < (n - T + 1 + torch.arange(T, device="cuda"))[:, None]
        else:
            seen = torch.ones(T, n, dtype=torch.bool, device="cuda")
        s = s.masked_fill(~seen, -math.inf)
        empty = ~seen.any(-1)
        p = torch.softmax(s, -1)
        p[:, empty] = 0
        ref, a = p @ v, p @ v.abs()
        # a weight's relative error: its logit's (fp32 sum of hd products, and the base-2 exponent's own
        # rounding), 2^-22 of the exponential, one fp16 rounding; the sums over n keys; weights below the
        # smallest normal fp16 (2^-14, where the largest is 1 or more) are off by 2^-25 of the largest |v|
        top_logit = torch.where(seen, s.abs(), 0).amax(-1)
        dl = torch.where(seen, mag, 0).amax(-1) * (hd + 8) * 2.0**-23 + top_logit * 2.0**-22
        rel = (2 * dl + 2.0**-22 + 2.0**-11 + (n + 16) * 2.0**-23)[..., None]
        tol = rel * a + n * 2.0**-24 * v.abs().amax((1, 2))[:, None, None] + 2.0**-8 * ref.abs() + 2.0**-126
        ref, tol = ref.transpose(0, 1), tol.transpose(0, 1)
        off = (got[b].double() - ref).abs()
        worst = max(worst, (off / tol).nan_to_num(nan=1e9).max().item())
    assert worst <= 1, f"{worst:.3g} of the tolerance"
    return got


def filled(pn, g, n, cap, kvh, hd, spread=1.0):
    k = randn(g, n, cap, kvh, hd) * torch.exp2(spread * randn(g, n, cap, kvh, 1))
    v = randn(g, n, cap, kvh, hd) * torch.exp2(spread * randn(g, n, cap, kvh, 1))
    cache = new_cache(n, cap, kvh, hd)
    pn.kv8_write(k.to(BF), v.to(BF), *cache)
    return cache


@pytest.mark.parametrize("heads,kvh,hd", [(8, 1, 256), (8, 2, 128), (16, 16, 64), (32, 8, 128), (6, 2, 64), (20, 1, 128), (3, 3, 256)])
@pytest.mark.parametrize("T", [1, 2, 7, 50])
@pytest.mark.parametrize("causal", [False, True])
def test_attention(pn, heads, kvh, hd, T, causal):
    g = gen(heads * T + hd)
    cap = 333
    cache = filled(pn, g, 6, cap, kvh, hd)
    q = randn(g, 5, T, heads, hd, dtype=BF)
    check_attention(pn, q, cache, i32(333, 0, 1, 17, 200), slots=i32(3, 0, 5, 1, 2), causal=causal)


@pytest.mark.parametrize("heads,kvh,hd,B,T,cap", [(8, 1, 256, 1, 1, 20000), (8, 1, 256, 2, 50, 1018), (8, 1, 256, 1, 968, 968),
                                                  (16, 4, 128, 1, 300, 3001), (8, 8, 64, 2, 257, 700), (4, 1, 128, 1, 129, 4097),
                                                  (8, 2, 64, 1, 1, 70001)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_long(pn, heads, kvh, hd, B, T, cap, causal):
    g = gen(cap + T)
    cache = filled(pn, g, B, cap, kvh, hd)
    q = randn(g, B, T, heads, hd, dtype=BF)
    check_attention(pn, q, cache, torch.arange(cap, cap - B, -1, device="cuda").int(), causal=causal)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_lengths_next_to_tiles(pn, n, T, hd):
    g = gen(n)
    cache = filled(pn, g, 1, 300, 1, hd)
    q = randn(g, 1, T, 8, hd, dtype=BF)
    check_attention(pn, q, cache, i32(n), causal=True)
    check_attention(pn, q, cache, i32(n))


@pytest.mark.parametrize("T", [1, 4, 60])
def test_attention_ignores_what_lies_behind_the_length(pn, T):
    """NaN codes and NaN scales in positions that no row sees, other samples' slots among them"""
    g = gen(21)
    cache = filled(pn, g, 2, 200, 2, 128)
    q = randn(g, 1, T, 8, 128, dtype=BF)
    for c in cache:
        c.view(torch.uint8)[1, 77:] = 0x7F if c.dtype == E4M3 else 255
        c.view(torch.uint8)[0] = 0x7F if c.dtype == E4M3 else 255
    check_attention(pn, q, cache, i32(77), slots=i32(1))
    check_attention(pn, q, cache, i32(77), slots=i32(1), causal=True)


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("which", ["k", "v"])
def test_attention_nan_row_reaches_only_those_that_see_it(pn, T, which):
    g = gen(22)
    cap = 150
    k, v = randn(g, 1, cap, 1, 256, dtype=BF), randn(g, 1, cap, 1, 256, dtype=BF)
    (k if which == "k" else v)[0, cap - 2, 0, 5] = math.nan
    cache = new_cache(1, cap, 1, 256)
    pn.kv8_write(k, v, *cache)
    q = randn(g, 1, T, 8, 256, dtype=BF)
    out = pn.kv8_attention(q, *cache, lens=i32(cap), causal=True)
    assert torch.isnan(out[0, -2:]).all() and torch.isfinite(out[0, :-2]).all()
    clean = pn.kv8_attention(q[:, : T - 2].contiguous(), *cache, lens=i32(cap - 2), causal=True)
    tol = 2.0**-7 * clean.float().abs() + 2.0**-9
    assert ((out[:, :-2].float() - clean.float()).abs() <= tol).all()


@pytest.mark.parametrize("T", [1, 50])
def test_attention_bad_slots_and_lengths_give_zero(pn, T):
    g = gen(23)
    cache = filled(pn, g, 3, 64, 1, 256)
    q = randn(g, 4, T, 8, 256, dtype=BF)
    check_attention(pn, q, cache, i32(64, 64, -5, 1000), slots=i32(-1, 3, 0, 1))


@pytest.mark.parametrize("T", [1, 33])
def test_attention_logits_far_apart(pn, T):
    """one key far above the rest (its weight is 1), keys far below (0), large and tiny queries, growing logits"""
    g = gen(24)
    cap = 600
    k = randn(g, 1, cap, 1, 128) * torch.linspace(0.01, 30, cap, device="cuda")[None, :, None, None]
    v = randn(g, 1, cap, 1, 128) * torch.exp2(torch.linspace(-20, 20, cap, device="cuda"))[None, :, None, None]
    cache = new_cache(1, cap, 1, 128)
    pn.kv8_write(k.to(BF), v.to(BF), *cache)
    q = randn(g, 1, T, 8, 128)
    q[:, :, 0] *= 100
    q[:, :, 1] *= 2.0**-100
    q[:, :, 2] = 0
    q[:, :, 3, 1:] *= 2.0**-20
    check_attention(pn, q.to(BF), cache, i32(cap))


def test_attention_small_weights_add_up(pn):
    """one key with most of the weight and 60,000 whose weights are near 2^-21 of it each, V of one sign"""
    cap, hd = 60001, 64
    k = torch.zeros(1, cap, 1, hd, device="cuda", dtype=BF)
    k[0, 0, 0, 0] = 1.0
    v = torch.ones(1, cap, 1, hd, device="cuda", dtype=BF)
    v[0, 0] = 0.0
    cache = new_cache(1, cap, 1, hd)
    pn.kv8_write(k, v, *cache)
    for T in (1, 40):
        q = torch.zeros(1, T, 2, hd, device="cuda", dtype=BF)
        q[..., 0] = 14.5
        got = pn.kv8_attention(q, *cache, lens=i32(cap), scale=1.0)
        w = (cap - 1) * math.exp(-14.5)
        ref = w / (1 + w)
        # fp16 weights of 2^-21 or more of the largest: at worst 2^-25 / 2^-21 = 2^-4 of themselves off where
        # the largest is 1 (subnormal); these are the same number in every key
        assert (got.float() - ref).abs().max() <= (2.0**-4 + 2.0**-8) * ref


@pytest.mark.parametrize("T", [2, 40, 130])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_query_with_nan_or_infinity(pn, T, hd):
    """its rows are NaN where they see a key and 0 where they see none; all others are as without it"""
    g = gen(27)
    cache = filled(pn, g, 2, 90, 1, hd)
    q = randn(g, 2, T, 8, hd, dtype=BF)
    lens = i32(90, T - 1)  # causal: the second sample's first token sees nothing
    want = pn.kv8_attention(q, *cache, lens=lens, causal=True)
    bad = q.clone()
    bad[0, 1, 2, 5], bad[0, T - 1, 7, 0] = math.nan, math.inf
    bad[1, 0, 1, 3], bad[1, T - 1, 0, 9] = -math.inf, math.nan
    got = pn.kv8_attention(bad, *cache, lens=lens, causal=True)
    sees = (lens[:, None] - T + 1 + torch.arange(T, device="cuda")) > 0
    isbad = ~torch.isfinite(bad).all(-1) & sees[..., None]
    assert torch.equal(torch.isnan(got).all(-1), isbad) and torch.equal(torch.isnan(got).any(-1), isbad)
    assert torch.equal(got[~isbad], want[~isbad]) and (got[~sees] == 0).all() and isbad.any()


@pytest.mark.parametrize("heads,kvh,hd", [(8, 1, 256), (8, 2, 64), (6, 2, 128)])
@pytest.mark.parametrize("T,cap", [(3, 200), (50, 300), (150, 260), (40, 30000)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_a_padded_batch(pn, heads, kvh, hd, T, cap, causal):
    """samples with fewer query tokens than T: their tokens give what they give alone, rows behind stay as they were"""
    g = gen(34)
    cache = filled(pn, g, 5, cap, kvh, hd)
    q = randn(g, 5, T, heads, hd, dtype=BF)
    q[:, T // 2 + 1 :, 0] = math.nan  # in padding too
    counts, lens = [T, T // 2 + 1, 0, 1, T + 7], [cap, cap - 5, 100, 1, T // 2]
    q[0] = q[4] = randn(g, T, heads, hd, dtype=BF)
    out = torch.full_like(q, 3)
    got = pn.kv8_attention(q, *cache, lens=i32(*lens), count=i32(*counts), causal=causal, out=out)
    assert got is out
    for b, n in enumerate(counts):
        n = min(n, T)
        assert (out[b, n:] == 3).all()
        if n:
            alone = check_attention(pn, q[b : b + 1, :n].contiguous(), cache, i32(lens[b]), slots=i32(b), causal=causal)
            assert ((out[b, :n].float() - alone[0].float()).abs() <= 2.0**-7 * alone[0].float().abs() + 2.0**-8).all()
    assert (pn.kv8_attention(q, *cache, lens=i32(*lens), count=i32(*counts), causal=causal)[2] == 0).all()


@pytest.mark.parametrize("T", [1, 60])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 1e-12, -1e-30])
def test_attention_other_scales(pn, T, scale):
    g = gen(28)
    cache = filled(pn, g, 2, 150, 1, 256)
    q = randn(g, 2, T, 8, 256, dtype=BF) * 0.3
    q[:, :, 3] = 0
    q[:, :, 4] *= 2.0**-120
    check_attention(pn, q, cache, i32(150, 70), scale=scale, causal=True)


def test_attention_one_query_for_all_samples(pn):
    """a query broadcast over the batch (sample stride 0)"""
    g = gen(29)
    cache = filled(pn, g, 4, 100, 2, 128)
    for T in (1, 40):
        q = randn(g, 1, T, 8, 128, dtype=BF).expand(4, -1, -1, -1)
        got = pn.kv8_attention(q, *cache, lens=i32(100, 5, 64, 0))
        assert torch.equal(got, pn.kv8_attention(q.contiguous(), *cache, lens=i32(100, 5, 64, 0)))


@pytest.mark.parametrize("T", [1, 40])
def test_attention_with_workspaces_on_two_streams_and_in_graphs(pn, T):
    g = gen(30)
    cap = 40000
    assert pn.lib.pi05_kv8_attention_workspace(1, T, 8, 1, 256, cap) > 0
    runs = []
    for i in range(2):
        runs.append((randn(g, 1, T, 8, 256, dtype=BF), filled(pn, g, 1, cap, 1, 256), i32(cap - 3 * i)))
    want = [pn.kv8_attention(q, *c, lens=n) for q, c, n in runs]
    side = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for (q, c, n), s in zip(runs, side):
            with torch.cuda.stream(s):
                got.append(pn.kv8_attention(q, *c, lens=n))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))
    graphs, outs = [], []
    for q, c, n in runs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(pn.kv8_attention(q, *c, lens=n))
        graphs.append(gr)
    for _ in range(3):
        for gr, s in zip(graphs, side):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("T", [1, 50])
def test_attention_strided_query_and_out(pn, T):
    g = gen(25)
    cache = filled(pn, g, 2, 100, 1, 256)
    qkv = randn(g, 2, T + 3, 2560, dtype=BF)
    q = qkv[:, :T, :2048].unflatten(2, (8, 256))
    big = torch.full((2, T + 1, 2560), 3.0, device="cuda", dtype=BF)
    got = check_attention(pn, q, cache, i32(100, 60), out=big[:, :T, :2048].unflatten(2, (8, 256)))
    assert torch.equal(got, pn.kv8_attention(q.contiguous(), *cache, lens=i32(100, 60)))
    assert (big[:, T:] == 3).all() and (big[..., 2048:] == 3).all()


@pytest.mark.parametrize("T,cap", [(1, 9000), (50, 1018), (300, 900)])
def test_attention_reruns_are_identical(pn, T, cap):
    g = gen(26)
    cache = filled(pn, g, 1, cap, 1, 256)
    q = randn(g, 1, T, 8, 256, dtype=BF)
    a = pn.kv8_attention(q, *cache, lens=i32(cap))
    for _ in range(5):
        assert torch.equal(a, pn.kv8_attention(q, *cache, lens=i32(cap)))


# ---------------------------------------------------------------- together, streams, graphs
def layer(pn, h, weights, cache, start, lens, slots):
    """One attention layer as a server runs it: 8 query heads of 256 on one K/V head, 8-bit weights and cache."""
    B, T, D = h.shape
    wqkv, wo, wgu, wd = weights
    qkv = pn.fp8_linear(*pn.fp8_quantize(h.flatten(0, 1)), *wqkv).view(B, T, 2560)
    q = qkv[..., :2048].unflatten(2, (8, 256))
    k, v = qkv[..., 2048:2304].unflatten(2, (1, 256)), qkv[..., 2304:].unflatten(2, (1, 256))
    pn.kv8_write(k, v, *cache, start=start, slots=slots)
    a = pn.kv8_attention(q, *cache, lens=lens, slots=slots, causal=True)
    h = pn.fp8_linear(*pn.fp8_quantize(a.view(B * T, 2048)), *wo, epi="resid", res=h.flatten(0, 1))
    u = pn.fp8_linear(*pn.fp8_quantize(h), *wgu, epi="geglu")
    return pn.fp8_linear(*pn.fp8_quantize(u), *wd, epi="resid", res=h).view(B, T, D)


def layer_weights(pn, g, D=1024, M=2048):
    w = lambda f, k: pn.fp8_quantize(randn(g, f, k) * k**-0.5)  # noqa: E731
    return w(2560, D), w(D, 2048), w(2 * M, D), w(D, M)


def layer_plain(pn, h, weights, past, T):
    """the same layer in 64 bits on the values that the codes stand for, rounded where the operators round"""
    wqkv, wo, wgu, wd = (values(*w) for w in weights)
    quant = lambda x: decode(*encode(blocks_of(x))).flatten(1)[:, : x.shape[1]]  # noqa: E731
    bf = lambda x: x.to(BF).double()  # noqa: E731
    qkv = bf(quant(h) @ wqkv.t())
    k = torch.cat([past[0], decode(*encode(qkv[:, 2048:2304]))])
    v = torch.cat([past[1], decode(*encode(qkv[:, 2304:]))])
    q = qkv[:, :2048].view(T, 8, 256).transpose(0, 1)
    s = q @ k.t() / 16
    n = k.shape[0]
    s = s.masked_fill(torch.arange(n, device="cuda")[None] > (n - T + torch.arange(T, device="cuda"))[:, None], -math.inf)
    a = bf((torch.softmax(s, -1) @ v).transpose(0, 1).reshape(T, 2048))
    h = bf(h + quant(a) @ wo.t())
    gu = quant(h) @ wgu.t()
    u = bf(gelu(gu[:, 0::2]) * gu[:, 1::2])
    return bf(h + quant(u) @ wd.t()), (k, v)


def test_prompt_then_tokens_through_a_layer(pn):
    """a prompt of 200 and two single tokens for three samples of different slots, step by step against 64 bits.
    A rounding that falls the other way (bf16 2^-8 of a value, then an e4m3 code by a step, 2^-3 of it) moves a later product
    by one term; the bound is 3 % of the output's norm, a tenth of what one operator left out changes."""
    g = gen(31)
    weights = layer_weights(pn, g)
    cache = new_cache(5, 256, 1, 256)
    slots = i32(4, 0, 2)
    past = [(torch.zeros(0, 256, device="cuda", dtype=torch.float64),) * 2 for _ in range(3)]
    done = 0
    for T in (200, 1, 1):
        h = randn(g, 3, T, 1024, dtype=BF)
        start = torch.full((3,), done, device="cuda", dtype=torch.int32)
        y = layer(pn, h, weights, cache, start, start + T, slots)
        for b in range(3):
            ref, past[b] = layer_plain(pn, h[b].double(), weights, past[b], T)
            assert (y[b].double() - ref).norm() <= 0.03 * ref.norm()
        done += T


def test_side_stream_and_captured_graph(pn):
    """the layer on a side stream and replayed from graphs, two of which run at the same time, gives the eager bits"""
    g = gen(32)
    weights = layer_weights(pn, g)
    runs = []
    for i in range(2):
        h = randn(g, 2, 50, 1024, dtype=BF)
        runs.append(dict(h=h, cache=new_cache(2, 2048, 1, 256, fill=1, scale=120), start=i32(900 + i, 1500), lens=i32(950 + i, 1550)))
    step = lambda r: layer(pn, r["h"], weights, r["cache"], r["start"], r["lens"], None)  # noqa: E731
    want = [step(r).clone() for r in runs]
    side = [torch.cuda.Stream() for _ in runs]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for r, s in zip(runs, side):
        with torch.cuda.stream(s):
            got.append(step(r))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for r in runs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            r["y"] = step(r)
        graphs.append(gr)
    for _ in range(3):
        for r in runs:
            r["y"].fill_(-1)
        torch.cuda.synchronize()
        for gr, s in zip(graphs, side):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(r["y"], w) for r, w in zip(runs, want))
    # new inputs in the captured buffers
    runs[0]["h"].copy_(randn(g, 2, 50, 1024, dtype=BF))
    runs[0]["lens"].copy_(i32(40, 1550))
    runs[0]["start"].copy_(i32(0, 1500))
    graphs[0].replay()
    y = runs[0]["y"].clone()
    torch.cuda.synchronize()
    assert torch.equal(y, step(runs[0]))


def test_offsets_past_32_bits(pn):
    """a cache of 4.5 GB codes and queries into its last slot; a quantised matrix of 2.2 G values"""
    g = gen(33)
    n, cap, kvh, hd = 9, 1 << 20, 2, 256
    k8 = torch.zeros(n, cap, kvh, hd, device="cuda", dtype=torch.uint8).view(E4M3)
    ks = torch.full((n, cap, kvh), 127, device="cuda", dtype=torch.uint8)
    cache = (k8, ks, k8.clone(), ks.clone())
    k, v = randn(g, 1, 70, kvh, hd, dtype=BF), randn(g, 1, 70, kvh, hd, dtype=BF)
    pn.kv8_write(k, v, *cache, start=i32(cap - 70), slots=i32(8))
    ko, vo = pn.kv8_read(*cache, start=i32(cap - 70), T=70, slots=i32(8))
    assert torch.equal(ko, decode(*encode(k)).to(BF)) and torch.equal(vo, decode(*encode(v)).to(BF))
    q = 40 * k[:, -2:].repeat_interleave(4, 2)
    got = pn.kv8_attention(q, *cache, lens=i32(cap), slots=i32(8), causal=True)
    small = pn.kv8_attention(q, *(c[8:, cap - 70 :].contiguous() for c in cache), lens=i32(70), causal=True)
    assert ((got.float() - small.float()).abs() <= 2.0**-7 * small.float().abs() + 1e-6).all()  # keys of zeros weigh e^-100s
    q = (40 * k[:, -60:].repeat_interleave(4, 2)).contiguous()
    got = pn.kv8_attention(q, *cache, lens=i32(cap), slots=i32(8), causal=True)
    small = pn.kv8_attention(q, *(c[8:, cap - 70 :].contiguous() for c in cache), lens=i32(70), causal=True)
    assert ((got.float() - small.float()).abs() <= 2.0**-7 * small.float().abs() + 1e-6).all()
    del cache, k8, ks
    x = torch.zeros(1 << 17, 17000, device="cuda", dtype=BF)
    x[-1] = randn(g, 17000, dtype=BF)
    q, s = pn.fp8_quantize(x)
    codes, byte = encode(blocks_of(x[-1:]))
    assert torch.equal(q[-1:].double(), codes.flatten(1)[:, :17000]) and torch.equal(s[-1:].long(), byte)
