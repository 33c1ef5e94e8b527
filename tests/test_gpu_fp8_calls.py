"""The Python calls of the 8-bit operators: what they refuse, layouts, devices."""
import pytest
import torch
from test_gpu_fp8 import BF, E4M3, filled, gen, i32, new_cache, randn

pytestmark = pytest.mark.gpu


def test_a_tensor_that_needs_a_gradient_is_refused(pn):
    g = gen(71)
    x = randn(g, 8, 256, dtype=BF)
    xq, w = pn.fp8_quantize(x), pn.fp8_quantize(randn(g, 16, 256, dtype=BF))
    bias, gate, res = randn(g, 16, dtype=BF), randn(g, 16, dtype=BF), randn(g, 8, 16, dtype=BF)
    cache = filled(pn, g, 2, 20, 1, 256)
    k, q = randn(g, 2, 3, 1, 256, dtype=BF), randn(g, 2, 3, 8, 256, dtype=BF)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda f: pn.fp8_quantize(f(x)), lambda f: pn.fp8_linear(*xq, *w, bias=f(bias)),
             lambda f: pn.fp8_linear(*xq, *w, epi="resid", res=f(res)),
             lambda f: pn.fp8_linear(*xq, *w, epi="gated", res=res, gate=f(gate)), lambda f: pn.kv8_write(f(k), k, *cache),
             lambda f: pn.kv8_write(k, f(k), *cache), lambda f: pn.kv8_attention(f(q), *cache, lens=i32(20, 10))]
    for call in calls:
        with pytest.raises(pn.Pi05Error, match="no backward"):
            call(grad)
        call(lambda t: t)
        with torch.no_grad():
            call(grad)


@pytest.mark.parametrize("T,B,kvh,hd", [(5, 3, 2, 128), (140, 4, 1, 256), (40, 8, 2, 64)])
def test_outputs_with_tokens_outside_samples(pn, T, B, kvh, hd):
    """[T][batch][heads][head_dim] buffers seen as [batch][T]...: no two rows share an element"""
    g = gen(72)
    cache = filled(pn, g, B, T + 7, kvh, hd)
    lens = torch.arange(T + 7, T + 7 - B, -1, device="cuda").int()
    q = randn(g, T, B, 4 * kvh, hd, dtype=BF).transpose(0, 1)
    out = torch.full((T, B, 4 * kvh, hd), 3.0, device="cuda", dtype=BF).transpose(0, 1)
    got = pn.kv8_attention(q, *cache, lens=lens, causal=True, out=out)
    assert got is out and torch.equal(got, pn.kv8_attention(q.contiguous(), *cache, lens=lens, causal=True))
    k, v = (torch.zeros(T, B, kvh, hd, device="cuda", dtype=BF).transpose(0, 1) for _ in range(2))
    pn.kv8_read(*cache, T=T, start=i32(*range(B)), out=(k, v))
    want = pn.kv8_read(*cache, T=T, start=i32(*range(B)))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    twice = new_cache(B, T, kvh, hd, fill=0, scale=0)
    pn.kv8_write(k, v, *twice)
    assert all(torch.equal(a, b) for a, b in zip(pn.kv8_read(*twice), want))


def test_reading_into_the_two_halves_of_a_buffer(pn):
    g = gen(73)
    cache = filled(pn, g, 2, 30, 2, 128)
    both = torch.zeros(2, 30, 4, 128, device="cuda", dtype=BF)
    k, v = pn.kv8_read(*cache, out=(both[:, :, :2], both[:, :, 2:]))
    want = pn.kv8_read(*cache)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    with pytest.raises(pn.Pi05Error, match="overlaps"):
        pn.kv8_read(*cache, out=(want[0], want[0]))
    with pytest.raises(pn.Pi05Error, match="overlaps"):
        pn.kv8_write(*want, cache[0], cache[1], cache[0], cache[3])


@pytest.mark.parametrize("shape", [(1, 8, 0, 256), (0, 8, 1, 256), (1, 0, 1, 256)])
def test_empty_caches_are_refused(pn, shape):
    """with the library's own error, before anything is divided or allocated"""
    k8, ks = torch.zeros(shape, device="cuda").to(E4M3), torch.zeros(shape[:3], device="cuda", dtype=torch.uint8)
    cache = (k8, ks, k8.clone(), ks.clone())
    q, k = torch.zeros(1, 1, 8, 256, device="cuda", dtype=BF), torch.zeros(1, 1, 1, 256, device="cuda", dtype=BF)
    for call in (lambda: pn.kv8_attention(q, *cache, lens=i32(1)), lambda: pn.kv8_read(*cache), lambda: pn.kv8_write(k, k, *cache)):
        with pytest.raises(pn.Pi05Error):
            call()


def test_an_index_that_is_no_vector_is_refused(pn):
    cache = new_cache(2, 8, 1, 256, fill=0, scale=0)
    with pytest.raises(pn.Pi05Error):
        pn.kv8_read(*cache, start=torch.tensor(0, device="cuda", dtype=torch.int32))
    with pytest.raises(pn.Pi05Error):
        pn.kv8_read(*cache, slots=torch.zeros(1, 1, device="cuda", dtype=torch.int32))
