"""The 8-bit serving operators on real work: quantisation in blocks of 128, the linear layer on its output, writing a
quantised K/V cache, reading it back, and attention over it.

A value is stored as an e4m3 code times a power of two.  The exponent belongs to a block: 128 consecutive values of a
row for activations and weights, one head of one position for the cache.  It is the smallest e with
max|x| <= 448 * 2^e, held as the byte e + 127, so scaling is exact and only the rounding to e4m3 loses anything.

Sizes are those of the pi0.5 model this repository serves: widths 1024 (action expert), 1152 / 4304 (SigLIP),
2048 / 16384 / 32768 (Gemma-2B), 8 query heads on one K/V head of 256, prefixes of 968 positions (three images and 200
prompt tokens), action chunks of 50, 1 to 64 environments; beside them generic head layouts and long caches.
"""
import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
BLOCK = 128


def listed():
    return [
        # one action chunk's activations before an expert projection: a latency
        {"name": "quantize chunk 50x1024", "op": "quantize", "rows": 50, "cols": 1024, "f32": False},
        # the prefix activations of 64 environments
        {"name": "quantize prefix 61952x2048", "op": "quantize", "rows": 61952, "cols": 2048, "f32": False},
        # the expert's gate/up projection for one chunk: few tokens, the weights are streamed
        {"name": "linear chunk geglu", "op": "linear", "T": 50, "F": 8192, "K": 1024, "epi": "geglu", "bias": False},
        # SigLIP's second MLP layer for three images: a K that is no multiple of the block, bias and residual
        {"name": "linear siglip fc2", "op": "linear", "T": 768, "F": 1152, "K": 4304, "epi": "resid", "bias": True},
        # Gemma's gate/up projection for the prefixes of eight environments
        {"name": "linear prefix geglu", "op": "linear", "T": 7744, "F": 32768, "K": 2048, "epi": "geglu", "bias": False},
        # an action chunk's K/V appended behind one environment's prefix
        {"name": "write chunk", "op": "write", "batch": 1, "slots": 4, "T": 50, "kv_heads": 1, "head_dim": 256,
         "capacity": 1024, "ragged": False},
        # the prefixes of 64 environments, prompts of different lengths
        {"name": "write 64 prefixes", "op": "write", "batch": 64, "slots": 64, "T": 968, "kv_heads": 1, "head_dim": 256,
         "capacity": 1024, "ragged": True},
        # one environment's prefix copied out
        {"name": "read one prefix", "op": "read", "batch": 1, "slots": 4, "T": 968, "kv_heads": 1, "head_dim": 256,
         "capacity": 1024, "ragged": False},
        # grouped heads, long histories of different lengths
        {"name": "read 16 histories", "op": "read", "batch": 16, "slots": 20, "T": 4099, "kv_heads": 8, "head_dim": 128,
         "capacity": 4200, "ragged": True},
        # one new token for each of 16 long histories
        {"name": "attend 1 token", "op": "attention", "batch": 16, "slots": 16, "T": 1, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "capacity": 16400, "min_len": 4000, "max_len": 16387, "causal": True},
        # the action chunks of 64 environments over prefix and chunk
        {"name": "attend 64 chunks", "op": "attention", "batch": 64, "slots": 64, "T": 50, "heads": 8, "kv_heads": 1,
         "head_dim": 256, "capacity": 1024, "min_len": 900, "max_len": 1018, "causal": False},
        # a long prompt's last part over what is cached before it
        {"name": "attend prompt part", "op": "attention", "batch": 2, "slots": 4, "T": 2049, "heads": 16, "kv_heads": 4,
         "head_dim": 128, "capacity": 8200, "min_len": 6001, "max_len": 8192, "causal": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "write", "read", "attention", "attention"])
    if op == "quantize":
        cols = rng.choice([1024, 1152, 2048, 4304, 16384, _log(rng, 16, 20000)])
        return {"op": op, "rows": min(_log(rng, 1, 62000), 120_000_000 // cols), "cols": cols, "f32": rng.random() < 0.3}
    if op == "linear":
        F = rng.choice([1024, 1152, 2048, 2560, 4304, 16384, 2 * _log(rng, 8, 10000)])
        K = rng.choice([1024, 1152, 2048, 4096, 4304, _log(rng, 16, 17000)])
        T = min(_log(rng, 1, 8000), max(1, 500_000_000_000 // (F * K)))
        return {"op": op, "T": T, "F": F, "K": K, "epi": rng.choice(["store", "gelu", "resid", "gated", "geglu", "f32"]),
                "bias": rng.random() < 0.4}
    kvh, hd = rng.choice([(1, 256), (1, 256), (8, 128), (4, 128), (2, 64), (16, 64)])
    slots = _log(rng, 1, 64)
    batch = rng.randint(1, slots)
    if op == "attention":
        T = rng.choice([1, 1, rng.randint(2, 16), 50, _log(rng, 17, 2100)])
        group = rng.choice([1, 2, 4, 8]) if kvh > 1 else 8
        cap = _log(rng, 64, 20000) + T
        batch = max(1, min(batch, 1_000_000_000 // (T * cap * group * kvh)))
        cap = min(cap, 300_000_000 // (slots * kvh * hd) + T)
        top = rng.randint(T, cap)
        return {"op": op, "batch": batch, "slots": slots, "T": T, "heads": group * kvh, "kv_heads": kvh, "head_dim": hd,
                "capacity": cap, "min_len": rng.randint(0, top), "max_len": top, "causal": rng.random() < 0.5}
    T = min(_log(rng, 1, 8000), max(1, 60_000_000 // (slots * kvh * hd)))
    return {"op": op, "batch": batch, "slots": slots, "T": T, "kv_heads": kvh, "head_dim": hd,
            "capacity": T + rng.randint(0, 100), "ragged": rng.random() < 0.7}


# ---- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(g, n, cols, spread=1.5):
    """activations: rows of different size, a few channels far above the rest, one block that is all zero"""
    x = torch.randn(n, cols, device="cuda", generator=g)
    x *= torch.exp2(spread * torch.randn(n, 1, device="cuda", generator=g))
    x *= 1 + 30 * (torch.rand(cols, device="cuda", generator=g) > 0.995)
    if n > 2 and cols > BLOCK:
        x[n // 2, :BLOCK] = 0
    return x


def _codes(shape, g):
    """cache contents: codes of N(0, 1) values under random scales"""
    raw = torch.randn(shape, device="cuda", generator=g, dtype=torch.bfloat16).mul_(100).clamp_(-448, 448).to(E4M3)
    return raw, torch.randint(118, 123, shape[:-1], device="cuda", generator=g, dtype=torch.int32).to(torch.uint8)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "quantize":
        s["x"] = _rows(g, case["rows"], case["cols"]).to(torch.float32 if case["f32"] else torch.bfloat16)
        return s
    if case["op"] == "linear":
        T, F, K = case["T"], case["F"], case["K"]
        s["xq"], s["xs"] = _plain_quantize(_rows(g, T, K))
        s["wq"], s["ws"] = _plain_quantize(torch.randn(F, K, device="cuda", generator=g) * K**-0.5)
        vec = lambda *n: torch.randn(*n, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
        s["biasv"] = vec(F) if case["bias"] else None
        s["res"] = vec(T, F) if case["epi"] in ("resid", "gated") else None
        s["gate"] = vec(F) if case["epi"] == "gated" else None
        return s
    B, N, T = case["batch"], case["slots"], case["T"]
    kvh, hd, cap = case["kv_heads"], case["head_dim"], case["capacity"]
    s["k8"], s["ks"] = _codes((N, cap, kvh, hd), g)
    s["v8"], s["vs"] = _codes((N, cap, kvh, hd), g)
    s["slot"] = torch.randperm(N, device="cuda", generator=g)[:B].to(torch.int32)
    if case["op"] == "attention":
        s["q"] = torch.randn(B, T, case["heads"], hd, device="cuda", generator=g).mul_(1.5).to(torch.bfloat16)
        n = torch.randint(case["min_len"], case["max_len"] + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        n[0] = case["max_len"]
        s["lens"] = n
        return s
    s["start"] = torch.randint(0, cap - T + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    s["count"] = None
    if case["ragged"]:
        s["count"] = torch.randint(T - T // 4, T + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    if case["op"] == "write":
        s["k"] = _rows(g, B * T * kvh, hd).to(torch.bfloat16).view(B, T, kvh, hd)
        s["v"] = _rows(g, B * T * kvh, hd).to(torch.bfloat16).view(B, T, kvh, hd)
    else:
        s["k"] = torch.zeros(B, T, kvh, hd, device="cuda", dtype=torch.bfloat16)
        s["v"] = torch.zeros(B, T, kvh, hd, device="cuda", dtype=torch.bfloat16)
    return s


# ---- the plain forms, in 32 bits

def _pow2(b):
    """2^(b - 127) for integers b in [0, 254], from its bits"""
    b = b.int()
    return torch.where(b > 0, b << 23, 1 << 22).view(torch.float32)


def _encode(x):
    """codes and exponent bytes of the last axis of x (one block)"""
    top = x.abs().amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(m <= 0.875, e - 9, e - 8)  # 448 = 0.875 * 2^9
    e = torch.where(top == 0, -127, e).clamp(-127, 127)
    return (x * _pow2(127 - e).unsqueeze(-1)).to(E4M3), (e + 127).to(torch.uint8)


def _decode(q, s):
    return q.float() * _pow2(s).unsqueeze(-1)


def _plain_quantize(x):
    """codes [rows][cols] with rows 16 bytes apart (or a multiple), exponents [rows][blocks], 4 bytes likewise"""
    n, cols = x.shape
    blocks = -(-cols // BLOCK)
    full = torch.zeros(n, blocks * BLOCK, device=x.device)
    full[:, :cols] = x
    q, s = _encode(full.view(n, blocks, BLOCK))
    sp = torch.zeros(n, -(-blocks // 4) * 4, device=x.device, dtype=torch.uint8)
    sp[:, :blocks] = s
    return q.view(n, -1)[:, :cols], sp[:, :blocks]


def _plain_dequantize(q, s):
    n, cols = q.shape
    full = torch.zeros(n, s.shape[1] * BLOCK, device=q.device)
    full[:, :cols] = q.float()
    return (full.view(n, -1, BLOCK) * _pow2(s).unsqueeze(-1)).view(n, -1)[:, :cols]


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))


def _plain_linear(s):
    y = _plain_dequantize(s["xq"], s["xs"]) @ _plain_dequantize(s["wq"], s["ws"]).t()
    if s["biasv"] is not None:
        y += s["biasv"].float()
    if s["epi"] == "f32":
        return y
    if s["epi"] == "gelu":
        y = _gelu(y)
    elif s["epi"] == "geglu":
        y = _gelu(y[:, 0::2]) * y[:, 1::2]
    elif s["epi"] == "resid":
        y = s["res"].float() + y
    elif s["epi"] == "gated":
        y = s["res"].float() + y * s["gate"].float()
    return y.to(torch.bfloat16)


def _places(s):
    """flat cache rows of every (sample, t), and which of them count"""
    t = torch.arange(s["T"], device="cuda")
    at = s["slot"].long()[:, None] * s["capacity"] + s["start"].long()[:, None] + t
    if s["count"] is None:
        return at, None
    return at, (t < s["count"][:, None])[..., None]


def _write_rows(x, codes, scales, at, valid):
    q, e = _encode(x.float())
    codes, scales, q = codes.view(torch.uint8).flatten(0, 1), scales.flatten(0, 1), q.view(torch.uint8)
    if valid is not None:
        q, e = torch.where(valid[..., None], q, codes[at]), torch.where(valid, e, scales[at])
    codes[at] = q
    scales[at] = e


def _plain_write(s):
    at, valid = _places(s)
    _write_rows(s["k"], s["k8"], s["ks"], at, valid)
    _write_rows(s["v"], s["v8"], s["vs"], at, valid)
    return s["k8"], s["ks"], s["v8"], s["vs"]


def _read_rows(x, codes, scales, at, valid):
    codes = codes.view(torch.uint8).flatten(0, 1)[at].view(E4M3)
    y = _decode(codes, scales.flatten(0, 1)[at]).to(torch.bfloat16)
    x.copy_(y if valid is None else torch.where(valid[..., None], y, x))


def _plain_read(s):
    at, valid = _places(s)
    _read_rows(s["k"], s["k8"], s["ks"], at, valid)
    _read_rows(s["v"], s["v8"], s["vs"], at, valid)
    return s["k"], s["v"]


def _plain_attention(s):
    B, T, kvh, hd, cap = s["batch"], s["T"], s["kv_heads"], s["head_dim"], s["capacity"]
    slot = s["slot"].long()
    k = _decode(s["k8"].view(torch.uint8)[slot].view(E4M3), s["ks"][slot]).transpose(1, 2)  # [B][kvh][cap][hd]
    v = _decode(s["v8"].view(torch.uint8)[slot].view(E4M3), s["vs"][slot]).transpose(1, 2)
    q = s["q"].float().view(B, T, kvh, -1, hd).transpose(1, 2).reshape(B, kvh, -1, hd)  # rows t * group + g
    logits = (q @ k.transpose(2, 3)).view(B, kvh, T, -1, cap) * hd**-0.5
    limit = s["lens"].long()[:, None].expand(B, T)
    if s["causal"]:
        limit = limit - T + 1 + torch.arange(T, device="cuda")
    seen = (torch.arange(cap, device="cuda") < limit[..., None])[:, None, :, None]
    logits = logits.masked_fill(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, 0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    y = p.view(B, kvh, -1, cap) @ v
    return y.view(B, kvh, T, -1, hd).transpose(1, 2).reshape(B, T, s["heads"], hd).to(torch.bfloat16)


# ---- one pass

if os.path.isdir("behavior-2026_b200") and os.path.abspath("behavior-2026_b200") not in sys.path:
    sys.path.append(os.path.abspath("behavior-2026_b200"))


def run(s):
    op = s["op"]
    if not own:
        if op == "quantize":
            return _plain_quantize(s["x"].float())
        return {"linear": _plain_linear, "write": _plain_write, "read": _plain_read, "attention": _plain_attention}[op](s)
    import pi05native as pn

    if op == "quantize":
        return pn.fp8_quantize(s["x"])
    if op == "linear":
        return pn.fp8_linear(s["xq"], s["xs"], s["wq"], s["ws"], epi=s["epi"], bias=s["biasv"], res=s["res"], gate=s["gate"])
    cache = (s["k8"], s["ks"], s["v8"], s["vs"])
    if op == "write":
        pn.kv8_write(s["k"], s["v"], *cache, start=s["start"], count=s["count"], slots=s["slot"])
        return cache
    if op == "read":
        return pn.kv8_read(*cache, start=s["start"], T=s["T"], count=s["count"], slots=s["slot"], out=(s["k"], s["v"]))
    return pn.kv8_attention(s["q"], *cache, lens=s["lens"], slots=s["slot"], causal=s["causal"])


def work(case):
    if case["op"] == "quantize":
        n, cols = case["rows"], case["cols"]
        return {"bytes": n * cols * (5 if case["f32"] else 3) + n * -(-cols // BLOCK), "flops": 3 * n * cols}
    if case["op"] == "linear":
        T, F, K, epi = case["T"], case["F"], case["K"], case["epi"]
        out = T * F * {"f32": 4, "geglu": 1, "resid": 4, "gated": 4}.get(epi, 2)
        return {"bytes": (T + F) * (K + -(-K // BLOCK)) + out, "flops": 2 * T * F * K}
    kvh, hd = case["kv_heads"], case["head_dim"]
    if case["op"] == "attention":
        B, T, H = case["batch"], case["T"], case["heads"]
        keys = case["max_len"] + (B - 1) * (case["min_len"] + case["max_len"]) / 2  # of all samples together
        seen = max(keys - (B * (T - 1) / 2 if case["causal"] else 0), keys / 2)
        return {"bytes": 2 * keys * kvh * (hd + 1) + 4 * B * T * H * hd, "flops": 4 * T * H * hd * seen}
    rows = case["batch"] * case["T"] * (7 / 8 if case["ragged"] else 1) * kvh * 2
    return {"bytes": rows * (3 * hd + 1), "flops": 2 * rows * hd}


# ---- the definitions in 64 bits

def _exact_block(x):
    """(code values, e + 127) of the last axis of x, both from their definitions"""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448))
    e = e + (top > 448 * torch.exp2(e)).double() - (top <= 448 * torch.exp2(e - 1)).double()  # log2 may be off next to a power of two
    e = torch.where(top > 0, e, -127.0).clamp(-127, 127)
    y = x / torch.exp2(e)
    bottom = torch.log2(y.abs().clamp_min(2.0**-6))  # at least the smallest normal
    step = torch.floor(bottom)
    step = step + (y.abs() >= torch.exp2(step + 1)).double() - (y.abs().clamp_min(2.0**-6) < torch.exp2(step)).double()
    step = torch.exp2(step - 3)
    return torch.round(y / step) * step, (e.squeeze(-1) + 127).long()


def _exact_values(q, s):
    rep = torch.exp2(s.double() - 127).repeat_interleave(BLOCK, 1)[:, : q.shape[1]]
    return q.double() * rep


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        qs, es = zip(*(_exact_block(b) for b in s["x"].double().split(BLOCK, 1)))
        return torch.cat(qs, 1), torch.stack(es, 1)
    if op == "linear":
        y = _exact_values(s["xq"], s["xs"]) @ _exact_values(s["wq"], s["ws"]).t()
        if s["biasv"] is not None:
            y = y + s["biasv"].double()
        act = lambda z: z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))  # noqa: E731
        if case["epi"] == "gelu":
            return act(y)
        if case["epi"] == "geglu":
            return act(y[:, 0::2]) * y[:, 1::2]
        if case["epi"] == "gated":
            y = y * s["gate"].double()
        return y if s["res"] is None else y + s["res"].double()
    count = s.get("count")
    if op == "write":
        k8, v8, ks, vs = s["k8"].double(), s["v8"].double(), s["ks"].long(), s["vs"].long()
        for b in range(case["batch"]):
            n = case["T"] if count is None else int(count[b])
            c, p = int(s["slot"][b]), int(s["start"][b])
            k8[c, p : p + n], ks[c, p : p + n] = _exact_block(s["k"][b, :n].double())
            v8[c, p : p + n], vs[c, p : p + n] = _exact_block(s["v"][b, :n].double())
        return k8, ks, v8, vs
    if op == "read":
        k, v = s["k"].double(), s["v"].double()
        for b in range(case["batch"]):
            n = case["T"] if count is None else int(count[b])
            c, p = int(s["slot"][b]), int(s["start"][b])
            k[b, :n] = s["k8"][c, p : p + n].double() * torch.exp2(s["ks"][c, p : p + n, :, None].double() - 127)
            v[b, :n] = s["v8"][c, p : p + n].double() * torch.exp2(s["vs"][c, p : p + n, :, None].double() - 127)
        return k, v
    T, H, hd, group = case["T"], case["heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(case["batch"], T, H, hd, device="cuda", dtype=torch.float64)
    for b in range(case["batch"]):
        c, n = int(s["slot"][b]), int(s["lens"][b])
        k = s["k8"][c, :n].double() * torch.exp2(s["ks"][c, :n, :, None].double() - 127)
        v = s["v8"][c, :n].double() * torch.exp2(s["vs"][c, :n, :, None].double() - 127)
        hidden = torch.zeros(T, n, device="cuda", dtype=torch.bool)
        if case["causal"]:
            hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - T, n, device="cuda")[:, None]
        for h in range(H):
            z = (s["q"][b, :, h].double() @ k[:, h // group].t()) / math.sqrt(hd)
            z[hidden] = -math.inf
            w = torch.softmax(z, -1) if n else z
            out[b, :, h] = torch.nan_to_num(w, nan=0.0) @ v[:, h // group]
    return out
