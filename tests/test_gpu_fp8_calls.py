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


def test_the_engines_prefixes_held_in_8_bits(pn):
    """a server's path: prefixes of two samples out of the engine into slots of an 8-bit cache, later back into the engine, all by
    device pointers.  What the engine then holds is the quantised prefix bit for bit, and it denoises as from the same
    values installed from the host."""
    import ctypes

    import numpy as np
    from test_gpu_fp8 import decode, encode

    layers, n = 2, 2
    eng = pn.Engine(pn.Config.make(siglip_layers=1, gemma_layers=layers, num_steps=2), max_batch=n)
    eng.init_random_weights(3)
    imgs = np.stack([pn.synth_images(3, i) for i in range(n)])
    toks = np.stack([pn.synth_tokens(3, i) for i in range(n)])
    noise = np.stack([pn.synth_noise(3, i) for i in range(n)])
    plain = eng.infer(imgs, toks, noise)
    P = eng.prefix_len
    k, v = (torch.empty(n, layers, P, 256, device="cuda", dtype=BF) for _ in range(2))
    for i in range(n):
        for layer in range(layers):
            assert pn.lib.pi05_get_prefix_cache(eng._h, i, layer, ctypes.c_void_p(k[i, layer].data_ptr()), ctypes.c_void_p(v[i, layer].data_ptr())) == 0
    cache = new_cache(7, P, 1, 256)
    slots = i32(5, 0, 3, 6)
    pn.kv8_write(k.view(n * layers, P, 1, 256), v.view(n * layers, P, 1, 256), *cache, slots=slots)
    k2, v2 = pn.kv8_read(*cache, T=P, slots=slots)
    torch.cuda.synchronize()
    assert pn.lib.pi05_set_prefix_cache(eng._h, n, ctypes.c_void_p(k2.data_ptr()), ctypes.c_void_p(v2.data_ptr())) == 0
    got = eng.denoise(noise)
    host = [decode(*encode(t)).to(BF).cpu() for t in (k, v)]
    assert torch.equal(k2.view_as(k).cpu(), host[0]) and torch.equal(v2.view_as(v).cpu(), host[1])
    eng.set_prefix_cache(*(t.view(torch.int16).numpy().view(np.uint16) for t in host))
    want = eng.denoise(noise)
    assert np.array_equal(got, want) and np.isfinite(got).all() and not np.array_equal(got, plain)
