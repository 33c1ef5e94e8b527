"""What the 8-bit operators refuse, checked on the host before any launch: no GPU is touched here."""
import ctypes

import pytest

ERR_ARG = -1


def call(pn, name, *args):
    err = ctypes.create_string_buffer(512)
    rc = getattr(pn.lib, name)(*args, None, err, 512)
    return rc, err.value.decode()


A = 1 << 20  # an aligned address that nothing reads: every call below is refused on the host


def quantize_args(**kw):
    a = dict(rows=4, cols=256, x=A, x_type=0, ldx=256, q=A, ldq=256, scales=A, lds=4)
    a.update(kw)
    return list(a.values())


def linear_args(**kw):
    a = dict(T=4, F=64, K=256, x=A, ldx=256, xs=A, ld_xs=4, w=A, ldw=256, ws=A, ld_ws=4, bias=None, res=None, gate=None, epi=0,
             out=A)
    a.update(kw)
    return list(a.values())


def rows_args(**kw):
    a = dict(batch=2, T=4, kvh=2, hd=128, k=A, v=A, sb=1024, st=256, n_slots=4, capacity=16, k8=A, ks=A, v8=A, vs=A, start=A,
             count=A, slots=A)
    a.update(kw)
    return list(a.values())


def attention_args(**kw):
    a = dict(batch=2, T=1, heads=8, kvh=2, hd=128, q=A, qb=1024, qt=1024, n_slots=4, capacity=16, k8=A, ks=A, v8=A, vs=A, lens=A,
             count=A, slots=A, causal=0, scale=1.0, out=A, ob=1024, ot=1024, ws=A, ws_bytes=1 << 40)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw", [dict(rows=0), dict(cols=0), dict(rows=1 << 31), dict(rows=1 << 28, cols=1024, ldx=1024, ldq=1024),
                                dict(x_type=2), dict(x=None), dict(q=None), dict(scales=None), dict(x=A + 1), dict(q=A + 8),
                                dict(ldq=264), dict(ldx=255), dict(ldq=240), dict(lds=1), dict(x_type=1, x=A + 2)])
def test_quantize_refuses(pn, kw):
    rc, msg = call(pn, "pi05_fp8_quantize", *quantize_args(**kw))
    assert rc == ERR_ARG and msg.startswith("pi05_fp8_quantize:")


@pytest.mark.parametrize("kw", [dict(T=0), dict(F=0), dict(K=0), dict(T=(1 << 24) + 1), dict(F=(1 << 24) + 1), dict(K=(1 << 24) + 1),
                                dict(epi=-1), dict(epi=6), dict(epi=4, F=63), dict(x=None), dict(w=None), dict(xs=None),
                                dict(ws=None), dict(out=None), dict(epi=2), dict(epi=3, res=A), dict(epi=3, gate=A), dict(x=A + 8),
                                dict(w=A + 4), dict(ldx=264), dict(ldw=248), dict(ldx=240), dict(ldw=240), dict(xs=A + 2),
                                dict(ws=A + 1), dict(ld_xs=6), dict(ld_ws=1), dict(ld_ws=2), dict(out=A + 8), dict(bias=A + 2),
                                dict(epi=2, res=A + 2), dict(epi=3, res=A, gate=A + 2), dict(ldx=1 << 40)])
def test_linear_refuses(pn, kw):
    rc, msg = call(pn, "pi05_fp8_linear", *linear_args(**kw))
    assert rc == ERR_ARG and msg.startswith("pi05_fp8_linear:")


@pytest.mark.parametrize("name", ["pi05_kv8_write", "pi05_kv8_read"])
@pytest.mark.parametrize("kw", [dict(batch=0), dict(batch=65536), dict(T=0), dict(kvh=0), dict(hd=96), dict(n_slots=0),
                                dict(capacity=0), dict(k=None), dict(v=None), dict(k8=None), dict(ks=None), dict(v8=None),
                                dict(vs=None), dict(k=A + 8), dict(v=A + 2), dict(k8=A + 4), dict(v8=A + 8), dict(sb=1020),
                                dict(st=252), dict(st=128), dict(sb=-8), dict(batch=5, slots=None),
                                dict(T=0x7fffffff, kvh=64, st=64 * 128)])
def test_cache_rows_refuse(pn, name, kw):
    rc, msg = call(pn, name, *rows_args(**kw))
    assert rc == ERR_ARG and msg.startswith(name + ":")


def test_reading_into_overlapping_samples_is_refused(pn):
    rc, msg = call(pn, "pi05_kv8_read", *rows_args(sb=768))
    assert rc == ERR_ARG and "overlap" in msg


@pytest.mark.parametrize("kw", [dict(batch=0), dict(T=0), dict(heads=0), dict(kvh=0), dict(heads=7), dict(hd=80), dict(n_slots=0),
                                dict(capacity=0), dict(batch=40000), dict(q=None), dict(k8=None), dict(ks=None), dict(v8=None),
                                dict(vs=None), dict(lens=None), dict(out=None), dict(q=A + 8), dict(k8=A + 8), dict(v8=A + 8),
                                dict(out=A + 8), dict(qb=1020), dict(qt=1020), dict(qt=1016), dict(ot=1016), dict(ob=1020),
                                dict(ob=512), dict(T=2, ob=1024), dict(batch=5, slots=None), dict(scale=float("inf")),
                                dict(scale=float("nan")), dict(T=1 << 24, heads=512, ob=1 << 62)])
def test_attention_refuses(pn, kw):
    rc, msg = call(pn, "pi05_kv8_attention", *attention_args(**kw))
    assert rc == ERR_ARG and msg.startswith("pi05_kv8_attention:")


@pytest.mark.parametrize("kw", [dict(ws=None), dict(ws_bytes=16), dict(ws=A + 8)])
def test_attention_refuses_a_workspace_too_small(pn, kw):
    kw = dict(batch=1, capacity=1 << 20, **kw)
    assert pn.lib.pi05_kv8_attention_workspace(1, 1, 8, 2, 128, 1 << 20) > 16  # this shape needs one
    rc, msg = call(pn, "pi05_kv8_attention", *attention_args(**kw))
    assert rc == ERR_ARG and "workspace" in msg


def test_workspace_of_a_bad_shape_is_an_error(pn):
    ok = pn.lib.pi05_kv8_attention_workspace
    assert ok(1, 1, 8, 1, 256, 1 << 20) > 0
    for bad in ((0, 1, 8, 1, 256, 64), (1, 0, 8, 1, 256, 64), (1, 1, 8, 3, 256, 64), (1, 1, 8, 1, 256, 0), (1, 1, 8, 1, 96, 64)):
        assert ok(*bad) == ERR_ARG


def test_a_refusal_without_a_message_buffer(pn):
    assert pn.lib.pi05_fp8_quantize(*quantize_args(rows=0), None, None, 0) == ERR_ARG
    assert pn.lib.pi05_fp8_linear(*linear_args(T=0), None, None, 0) == ERR_ARG


def test_python_refuses_host_tensors_and_wrong_types(pn):
    import torch

    with pytest.raises(pn.Pi05Error):
        pn.fp8_quantize(torch.zeros(4, 128, dtype=torch.bfloat16))
    q, s = torch.zeros(4, 128, dtype=torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8)
    with pytest.raises(pn.Pi05Error):
        pn.fp8_linear(q, s, q, s)
    k = torch.zeros(1, 4, 1, 256, dtype=torch.bfloat16)
    k8, ks = torch.zeros(1, 8, 1, 256, dtype=torch.float8_e4m3fn), torch.zeros(1, 8, 1, dtype=torch.uint8)
    with pytest.raises(pn.Pi05Error):
        pn.kv8_write(k, k, k8, ks, k8, ks)
    with pytest.raises(pn.Pi05Error):
        pn.kv8_read(k8, ks, k8, ks)
    with pytest.raises(pn.Pi05Error):
        pn.kv8_attention(k, k8, ks, k8, ks, lens=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("kw", [dict(T=4, sb=256, st=256), dict(T=4, sb=128, st=1024), dict(T=4, sb=264, st=512), dict(batch=3, T=4, sb=256, st=512)])
def test_reading_into_rows_that_share_elements_is_refused(pn, kw):
    """neither the samples' nor the tokens' rows clear of each other (256 elements a row)"""
    rc, msg = call(pn, "pi05_kv8_read", *rows_args(**kw))
    assert rc == ERR_ARG and "overlap" in msg


@pytest.mark.parametrize("kw", [dict(T=2, ob=1024, ot=1024), dict(T=3, ob=512, ot=4096), dict(batch=3, T=2, ob=1024, ot=2048)])
def test_attention_into_rows_that_share_elements_is_refused(pn, kw):
    rc, msg = call(pn, "pi05_kv8_attention", *attention_args(**kw))
    assert rc == ERR_ARG and "overlapping" in msg


@pytest.mark.parametrize("bad", [(40000, 1, 8, 2, 128, 64), (1, 1 << 30, 8, 2, 128, 64), (1 << 12, 1 << 12, 512, 1, 64, 64),
                                 (1, 1, 8, 2, 128, 0x7fffffff), (-1, 1, 8, 1, 256, 64), (1, 1, 8, 0, 256, 64)])
def test_workspace_is_asked_for_the_shapes_that_attention_takes(pn, bad):
    """a size is never given for a call that would then be refused"""
    b, t, h, kvh, hd, cap = bad
    if (kvh, cap) != (2, 0x7fffffff):  # 2^39 bytes a slot: taken
        assert pn.lib.pi05_kv8_attention_workspace(*bad) == ERR_ARG
        rc, _ = call(pn, "pi05_kv8_attention", *attention_args(batch=b, T=t, heads=h, kvh=kvh, hd=hd, capacity=cap, n_slots=1 << 20))
        assert rc == ERR_ARG
    else:
        assert pn.lib.pi05_kv8_attention_workspace(*bad) >= 0
        assert pn.lib.pi05_kv8_attention_workspace(b, t, h, 8, 128, cap) == ERR_ARG


def test_workspaces_are_not_monotone_and_each_is_enough_for_its_own_shape(pn):
    need = [pn.lib.pi05_kv8_attention_workspace(n, 50, 8, 1, 256, 1024) for n in (2, 8, 64)]
    assert need[2] == 0 and need[0] > 0 and need[1] > 0
    for n, bytes_ in zip((2, 8), need):
        rc, msg = call(pn, "pi05_kv8_attention", *attention_args(batch=n, T=50, heads=8, kvh=1, hd=256, qb=50 * 2048, qt=2048, ob=50 * 2048,
                                                                ot=2048, n_slots=64, capacity=1024, ws_bytes=bytes_ - 1))
        assert rc == ERR_ARG and "workspace" in msg


@pytest.mark.parametrize("name,kw", [("pi05_kv8_read", dict()), ("pi05_kv8_read", dict(v=A + 496)), ("pi05_kv8_read", dict(k=A + 16)),
                                     ("pi05_kv8_write", dict()), ("pi05_kv8_write", dict(v8=A + 4 * 16 * 256 - 16, vs=A - 4096)),
                                     ("pi05_kv8_write", dict(v8=A + (1 << 19), vs=A + 127)), ("pi05_kv8_write", dict(k8=A + (1 << 19), ks=A + 1))])
def test_k_and_v_written_to_one_place_is_refused(pn, name, kw):
    a = dict(batch=2, T=4, kvh=2, hd=128, sb=1024, st=256, n_slots=4, capacity=16)
    a.update(kw)
    rc, msg = call(pn, name, *rows_args(**a))
    assert rc == ERR_ARG and "overlaps" in msg
