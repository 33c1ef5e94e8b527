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
