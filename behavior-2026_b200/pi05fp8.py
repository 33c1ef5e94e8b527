"""The 8-bit operators of libpi05.so (pi05_fp8_*, pi05_kv8_* in include/pi05.h) on torch CUDA tensors.

Reached as pi05native.fp8_quantize and so on.  Each call runs on torch's current stream of its tensors' device, allocates
its outputs (and attention's workspace) from torch's allocator, may be captured into a torch.cuda.CUDAGraph, and raises
Pi05Error where the shapes, types or devices do not fit, or where autograd would want a gradient (there is no backward pass).  float8_e4m3fn codes and uint8 exponent bytes: a block's values are
codes * 2^(byte - 127); byte 255 stands for NaN.

The checks are written for a few microseconds a call: a single-token step makes several hundred of these calls.
"""
import ctypes
import threading

import torch

from pi05native import ERR_ARG, OK, Engine, Pi05Error, lib

E4M3, U8, BF, F32, I32 = torch.float8_e4m3fn, torch.uint8, torch.bfloat16, torch.float32, torch.int32
EPI = Engine.EPI
_raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_empty, _empty_strided, _grad_enabled = torch.empty, torch.empty_strided, torch.is_grad_enabled
_tls = threading.local()


def _bad(what):
    raise Pi05Error(ERR_ARG, what)


def _no_grad(what, *tensors):
    """these operators have no backward pass, so a result that autograd expects to follow is refused, not returned without a graph"""
    if _grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _bad(f"{what}: no backward pass: call it under torch.no_grad(), or with tensors that need no gradient")


def _err():
    try:
        return _tls.err
    except AttributeError:
        _tls.err = ctypes.create_string_buffer(512)
        return _tls.err


def _call(fn, dev, *args):
    """one call with device `dev` (an index) current, on its current torch stream"""
    err = _err()
    if dev == _device():
        rc = fn(*args, _raw_stream(dev), err, 512)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev), err, 512)
    if rc != OK:
        raise Pi05Error(rc, err.value.decode())


def _pitch(t, rows, cols):
    """elements between rows of t; of a single row any pitch will do, so one that every check takes"""
    r, c = t.stride()
    if c != 1 and cols > 1:
        _bad("rows must be contiguous")
    return r if rows > 1 else (cols + 15) // 16 * 16


def fp8_quantize(x, out=None):
    """pi05_fp8_quantize: x [rows][cols] bf16 or fp32 (rows may be strided) -> (q, scales): q float8_e4m3fn [rows][cols]
    and scales uint8 [rows][ceil(cols / 128)], both with padded rows as fp8_linear loads them best; x ~ q * 2^(scales - 127)
    block by block.  `out` = (q, scales) to write into."""
    dt, shape, dev = x.dtype, x.shape, x.get_device()
    if dev < 0 or len(shape) != 2 or (dt != BF and dt != F32) or x.numel() == 0:
        _bad("fp8_quantize: x must be a CUDA tensor [rows][cols], bf16 or fp32, not empty")
    _no_grad("fp8_quantize", x)
    rows, cols = shape
    blocks = (cols + 127) // 128
    if out is None:
        # rows of whole 128-byte lines and scale rows of 16 bytes, which fp8_linear loads best
        ldq, lds = blocks * 128 if cols > 64 else 64, (blocks + 15) // 16 * 16
        device = x.device
        q = _empty_strided((rows, cols), (ldq, 1), dtype=E4M3, device=device)
        s = _empty_strided((rows, blocks), (lds, 1), dtype=U8, device=device)
    else:
        q, s = out
        if q.dtype != E4M3 or s.dtype != U8 or q.shape != shape or s.shape != (rows, blocks) or q.get_device() != dev or s.get_device() != dev:
            _bad("fp8_quantize: out must be (float8_e4m3fn [rows][cols], uint8 [rows][ceil(cols / 128)]) on x's device")
        ldq, lds = _pitch(q, rows, cols), _pitch(s, rows, blocks)
    _call(lib.pi05_fp8_quantize, dev, rows, cols, x.data_ptr(), 1 if dt == F32 else 0, _pitch(x, rows, cols),
          q.data_ptr(), ldq, s.data_ptr(), lds)
    return q, s


def _vector(t, shape, dev, what):
    if t.dtype != BF or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        _bad(f"fp8_linear: {what} must be contiguous bf16 on x's device")
    return t.data_ptr()


def fp8_linear(x, x_scales, w, w_scales, epi="store", bias=None, res=None, gate=None, out=None):
    """pi05_fp8_linear: epilogue(x . w^T) of two quantised operands (fp8_quantize's outputs: x [T][K], w [F][K]); epi
    "store", "gelu", "resid", "gated", "geglu" (w rows interleaved gate/up) or "f32"; bias, gate [F], res [T][F] bf16.
    Returns bf16 [T][F] ([T][F/2] for geglu, fp32 for f32); `out` may be given, and may be res."""
    dev = x.get_device()
    if dev < 0 or x.dtype != E4M3 or w.dtype != E4M3 or x_scales.dtype != U8 or w_scales.dtype != U8:
        _bad("fp8_linear: x, w must be CUDA float8_e4m3fn tensors, their scales uint8")
    if x.dim() != 2 or w.dim() != 2 or x.numel() == 0 or w.numel() == 0:
        _bad("fp8_linear: x [T][K] and w [F][K] must not be empty")
    T, K = x.shape
    F, Kw = w.shape
    blocks = (K + 127) // 128
    if Kw != K or x_scales.shape != (T, blocks) or w_scales.shape != (F, blocks):
        _bad("fp8_linear: x [T][K] and w [F][K] must agree in K, scales must be [rows][ceil(K / 128)]")
    if w.get_device() != dev or x_scales.get_device() != dev or w_scales.get_device() != dev:
        _bad("fp8_linear: operands on different devices")
    _no_grad("fp8_linear", bias, res, gate, out)
    code = EPI.get(epi)
    if code is None or (code == 4 and F % 2):
        _bad(f"fp8_linear: unknown epilogue {epi!r}, or geglu with an odd F")
    b = _vector(bias, (F,), dev, "bias [F]") if bias is not None else None
    r = _vector(res, (T, F), dev, "res [T][F]") if res is not None else None
    g = _vector(gate, (F,), dev, "gate [F]") if gate is not None else None
    shape, dtype = (T, F // 2 if code == 4 else F), F32 if code == 5 else BF
    if out is None:
        out = _empty(shape, dtype=dtype, device=x.device)
    elif out.dtype != dtype or out.shape != shape or out.get_device() != dev or not out.is_contiguous():
        _bad(f"fp8_linear: out must be contiguous {dtype} {list(shape)} on x's device")
    _call(lib.pi05_fp8_linear, dev, T, F, K, x.data_ptr(), _pitch(x, T, K), x_scales.data_ptr(), _pitch(x_scales, T, blocks),
          w.data_ptr(), _pitch(w, F, K), w_scales.data_ptr(), _pitch(w_scales, F, blocks), b, r, g, code, out.data_ptr())
    return out


def fp8_status(device=None):
    """pi05_fp8_status: waits for the current torch stream of `device`; raises Pi05Error(ERR_DEVICE) if a device-side wait of
    an 8-bit operator there has given up since the last call."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index
    _call(lib.pi05_fp8_status, torch.cuda.current_device() if dev is None else dev)


def _index(t, batch, dev, what):
    if t is None:
        return None
    if t.dtype != I32 or t.shape != (batch,) or t.get_device() != dev or not t.is_contiguous():
        _bad(f"{what} must be a contiguous int32 tensor [batch] on the cache's device")
    return t.data_ptr()


def _cache(what, dev, k8, k_scales, v8, v_scales):
    """(slots, capacity, kv_heads, head_dim) and the four addresses"""
    shape = k8.shape
    if len(shape) != 4 or v8.shape != shape or k_scales.shape != shape[:3] or v_scales.shape != shape[:3] or 0 in shape:
        _bad(f"{what}: codes must be [slots][capacity][kv_heads][head_dim], not empty, scales [slots][capacity][kv_heads]")
    if k8.dtype != E4M3 or v8.dtype != E4M3 or k_scales.dtype != U8 or v_scales.dtype != U8:
        _bad(f"{what}: codes must be float8_e4m3fn, scales uint8")
    if not (k8.is_contiguous() and v8.is_contiguous() and k_scales.is_contiguous() and v_scales.is_contiguous()):
        _bad(f"{what}: the cache must be contiguous")
    if dev < 0 or k8.get_device() != dev or v8.get_device() != dev or k_scales.get_device() != dev or v_scales.get_device() != dev:
        _bad(f"{what}: all tensors must be on one CUDA device")
    return shape, (k8.data_ptr(), k_scales.data_ptr(), v8.data_ptr(), v_scales.data_ptr())


def _strides(what, t, shape):
    """(sample, token) strides of [batch][T][heads][head_dim] with contiguous heads; along an axis of length 1 any will do"""
    batch, T, h, d = shape
    sb, st, sh, sd = t.stride()
    if sd != 1 or (h > 1 and sh != d):
        _bad(f"{what}: the heads of a token must be contiguous")
    if T == 1:
        st = h * d
    return (sb if batch > 1 else T * st), st


def _rows(what, k, v, h, d, dev):
    shape = k.shape
    if k.dtype != BF or v.dtype != BF or len(shape) != 4 or v.shape != shape or shape[2] != h or shape[3] != d or k.numel() == 0 \
            or k.get_device() != dev or v.get_device() != dev:
        _bad(f"{what}: k, v must be CUDA bf16 tensors [batch][T][kv_heads][head_dim] of the cache's heads and device, not empty")
    _no_grad(what, k, v)
    strides = _strides(what, k, shape)
    if v.stride() != k.stride() and _strides(what, v, shape) != strides:
        _bad(f"{what}: k and v must be strided alike")
    return shape, strides


def kv8_write(k, v, k8, k_scales, v8, v_scales, start=None, count=None, slots=None):
    """pi05_kv8_write: quantises k, v (bf16 [batch][T][kv_heads][head_dim]) into the cache (k8, v8 float8_e4m3fn
    [slots][capacity][kv_heads][head_dim], scales uint8 [slots][capacity][kv_heads]): sample b's rows t < count[b] go to
    positions start[b] + t of slot slots[b].  start, count, slots: int32 CUDA tensors [batch] or None."""
    dev = k.get_device()
    (n, cap, h, d), at = _cache("kv8_write", dev, k8, k_scales, v8, v_scales)
    (batch, T, _, _), (sb, st) = _rows("kv8_write", k, v, h, d, dev)
    _call(lib.pi05_kv8_write, dev, batch, T, h, d, k.data_ptr(), v.data_ptr(), sb, st, n, cap, *at,
          _index(start, batch, dev, "kv8_write: start"), _index(count, batch, dev, "kv8_write: count"),
          _index(slots, batch, dev, "kv8_write: slots"))


def kv8_read(k8, k_scales, v8, v_scales, start=None, T=None, count=None, slots=None, out=None):
    """pi05_kv8_read: positions start[b] + t, t < count[b] <= T, of slot slots[b] back as bf16 (k, v) [batch][T][kv_heads]
    [head_dim].  The batch is that of start, count or slots (else every slot), T defaults to the capacity.  Rows that are not
    read keep what `out` = (k, v) held (0 in new tensors)."""
    dev = k8.get_device()
    (n, cap, h, d), at = _cache("kv8_read", dev, k8, k_scales, v8, v_scales)
    first = start if start is not None else count if count is not None else slots
    if first is not None and first.dim() != 1:
        _bad("kv8_read: start, count and slots must be int32 tensors [batch]")
    batch = n if first is None else first.shape[0]
    T = cap if T is None else T
    if out is None:
        out = tuple(torch.zeros((batch, T, h, d), dtype=BF, device=k8.device) for _ in range(2))
    k, v = out
    shape, (sb, st) = _rows("kv8_read", k, v, h, d, dev)
    if shape[0] != batch or shape[1] != T:
        _bad("kv8_read: out must be [batch][T][kv_heads][head_dim]")
    _call(lib.pi05_kv8_read, dev, batch, T, h, d, k.data_ptr(), v.data_ptr(), sb, st, n, cap, *at,
          _index(start, batch, dev, "kv8_read: start"), _index(count, batch, dev, "kv8_read: count"),
          _index(slots, batch, dev, "kv8_read: slots"))
    return k, v


def kv8_attention(q, k8, k_scales, v8, v_scales, lens, slots=None, causal=False, scale=None, out=None, count=None):
    """pi05_kv8_attention: attention of q (bf16 [batch][T][heads][head_dim], samples and tokens may be strided) over the
    first lens[b] positions of slot slots[b]; causal: token t sees lens[b] - n + t + 1 of them, n = count[b] (T without counts).
    Rows t >= n keep what `out` held (0 in a new tensor).  scale defaults to head_dim^-0.5.  Returns bf16 [batch][T][heads]
    [head_dim]."""
    dev = q.get_device()
    (n, cap, kvh, d), at = _cache("kv8_attention", dev, k8, k_scales, v8, v_scales)
    shape = q.shape
    if dev < 0 or q.dtype != BF or len(shape) != 4 or shape[3] != d or shape[2] % kvh or q.numel() == 0:
        _bad("kv8_attention: q must be a CUDA bf16 tensor [batch][T][heads][head_dim], heads a multiple of the cache's, not empty")
    _no_grad("kv8_attention", q, out)
    batch, T, heads, _ = shape
    qb, qt = _strides("kv8_attention", q, shape)
    if out is None:
        out = (_empty if count is None else torch.zeros)(shape, dtype=BF, device=q.device)
        ob, ot = T * heads * d, heads * d
    else:
        if out.dtype != BF or out.shape != shape or out.get_device() != dev:
            _bad("kv8_attention: out must be bf16 of q's shape on its device")
        ob, ot = _strides("kv8_attention", out, shape)
    if lens is None:
        _bad("kv8_attention: lens is required")
    lens, slots = _index(lens, batch, dev, "kv8_attention: lens"), _index(slots, batch, dev, "kv8_attention: slots")
    count = _index(count, batch, dev, "kv8_attention: count")
    if dev == _device():
        need = lib.pi05_kv8_attention_workspace(batch, T, heads, kvh, d, cap)
    else:
        with torch.cuda.device(dev):
            need = lib.pi05_kv8_attention_workspace(batch, T, heads, kvh, d, cap)
    if need > 0:
        ws = _empty(need, dtype=U8, device=q.device)
        ws_at = ws.data_ptr()
    else:
        need = ws_at = 0
    _call(lib.pi05_kv8_attention, dev, batch, T, heads, kvh, d, q.data_ptr(), qb, qt, n, cap, *at, lens, count, slots, 1 if causal else 0,
          d**-0.5 if scale is None else scale, out.data_ptr(), ob, ot, ws_at, need)
    return out
