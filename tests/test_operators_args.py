"""Refusals of add_rmsnorm, the 4-bit products and verify_drafts: argument errors come before any device work, so these run without a GPU."""
import ctypes as C

import numpy as np
import pytest

import bebelm_b200 as bb

F = (C.c_float * 4096)()
P = C.addressof(F)


def norm(x=P, xs=64, res=None, rs=64, dtype=bb.F32, rows=2, n=64, gain=P, sum_out=None, ss=64, y=P + 8192, yd=bb.F32, ysc=None,
         group=0, mem=bb.MEM_HOST):
    return bb.load_library().bebelm_add_rmsnorm(x, xs, res, rs, dtype, rows, n, gain, 1e-5, sum_out, ss, y, yd, ysc, group, mem, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=bb.INT8), bb.ERR_UNSUPPORTED), (dict(yd=bb.FP8), bb.ERR_UNSUPPORTED), (dict(n=0), bb.ERR_UNSUPPORTED),
    (dict(n=32769, xs=32769), bb.ERR_UNSUPPORTED), (dict(rows=1 << 31), bb.ERR_INVALID), (dict(x=None), bb.ERR_INVALID),
    (dict(gain=None), bb.ERR_INVALID), (dict(y=None), bb.ERR_INVALID), (dict(yd=bb.INT8), bb.ERR_INVALID),
    (dict(yd=bb.INT8, ysc=P, group=48), bb.ERR_UNSUPPORTED), (dict(yd=bb.INT8, ysc=P, group=128), bb.ERR_INVALID),
    (dict(group=32), bb.ERR_INVALID), (dict(xs=63), bb.ERR_INVALID), (dict(res=P, rs=10), bb.ERR_INVALID),
    (dict(xs=80), bb.ERR_INVALID), (dict(sum_out=P + 8192, res=P), bb.ERR_INVALID), (dict(mem=2), bb.ERR_INVALID),
])
def test_add_rmsnorm_refuses(kw, code):
    assert norm(**kw) == code and bb.last_error()


def test_no_rows_is_no_work():
    assert norm(rows=0) == bb.OK


@pytest.mark.parametrize("kw,code", [
    (dict(out=None), bb.ERR_INVALID), (dict(codes=None), bb.ERR_INVALID), (dict(scales=None), bb.ERR_INVALID),
    (dict(sd=bb.F32), bb.ERR_UNSUPPORTED), (dict(group=0), bb.ERR_UNSUPPORTED), (dict(group=96), bb.ERR_UNSUPPORTED),
    (dict(n_in=100), bb.ERR_INVALID), (dict(n_in=0), bb.ERR_INVALID), (dict(n_out=0), bb.ERR_INVALID),
    (dict(n_out=1 << 31), bb.ERR_INVALID), (dict(mem=7), bb.ERR_INVALID),
])
def test_w4_create_refuses(kw, code):
    h = C.c_void_p()
    a = dict(n_in=128, n_out=2, group=32, codes=P, scales=P, sd=bb.F16, mem=bb.MEM_HOST, out=C.byref(h)) | kw
    assert bb.load_library().bebelm_w4_create(0, a["n_in"], a["n_out"], a["group"], a["codes"], a["scales"], a["sd"], None,
                                              a["mem"], a["out"]) == code
    assert bb.last_error()


def test_w4_needs_a_handle():
    L, n = bb.load_library(), C.c_size_t()
    assert L.bebelm_w4_matmul(None, P, bb.F32, 128, None, 0, 1, P, bb.F32, None, 0, bb.MEM_HOST, None) == bb.ERR_INVALID
    assert L.bebelm_w4_workspace(None, P, bb.F32, 128, 0, 1, C.byref(n)) == bb.ERR_INVALID
    assert L.bebelm_w4_destroy(None) == bb.OK


def verify(target=P, ts=8, draft=None, ds=8, b=1, d=2, v=8, probs=0, temp=1.0, tokens=(1, 2), n=None, u=P, us=P, out=P, acc=P,
           mem=bb.MEM_HOST):
    tok = None if tokens is None else (C.c_int32 * len(tokens))(*tokens)
    nn = None if n is None else (C.c_int32 * len(n))(*n)
    return bb.load_library().bebelm_verify_drafts(target, ts, draft, ds, b, d, v, probs, temp, tok, nn, u, us, out, acc, None, 0,
                                                  mem, None)


@pytest.mark.parametrize("kw", [
    dict(target=None), dict(out=None), dict(acc=None), dict(tokens=None), dict(u=None), dict(us=None), dict(ts=7),
    dict(draft=P, ds=7), dict(ts=9), dict(draft=P, ds=9), dict(v=0), dict(v=1 << 31), dict(b=1 << 20), dict(d=1 << 10),
    dict(temp=-1.0), dict(temp=float("nan")), dict(temp=1e-9), dict(temp=1e9), dict(probs=1, temp=0.5), dict(tokens=(1, 8)),
    dict(tokens=(-1, 2)), dict(n=(3,)), dict(n=(-1,)), dict(mem=5),
])
def test_verify_refuses(kw):
    assert verify(**kw) == bb.ERR_INVALID and bb.last_error()


def test_verify_without_sequences():
    assert verify(b=0) == bb.OK
    n = C.c_size_t(5)
    assert bb.load_library().bebelm_verify_workspace(1, 1, 0, 1, 0, 1.0, C.byref(n)) == bb.ERR_INVALID


def test_python_shapes_are_checked():
    x = np.zeros((2, 64), np.float32)
    with pytest.raises(ValueError):
        bb.add_rmsnorm(x, np.ones(63, np.float32))
    with pytest.raises(ValueError):
        bb.add_rmsnorm(x, np.ones(64, np.float32), residual=np.zeros((2, 63), np.float32))
    with pytest.raises(ValueError):
        bb.add_rmsnorm(x, np.ones(64, np.float32), out_dtype=bb.BF16)
    with pytest.raises(ValueError):
        bb.W4Weights(np.zeros((4, 64), np.uint8), np.zeros((4, 3), np.float16), group=32)
    with pytest.raises(ValueError):
        bb.W4Weights(np.zeros((4, 64), np.uint8), np.zeros((4, 4), np.float32), group=32)
    with pytest.raises(ValueError):
        bb.W4Weights(np.zeros((4, 64), np.int32), np.zeros((4, 4), np.float16), group=32)
    with pytest.raises(ValueError):
        bb.verify_drafts(np.zeros((2, 3, 5), np.float32), np.zeros((2, 3), np.int32), None, None)


def test_w4_check_needs_a_handle():
    assert bb.load_library().bebelm_w4_check(None, None) == bb.ERR_INVALID and bb.last_error()


def no_weights(n_in=512, n_out=4):
    """W4Weights without a handle: what is checked before the library is called."""
    w = object.__new__(bb.W4Weights)
    w.n_in, w.n_out, w.group, w.device, w._h = n_in, n_out, 64, 0, C.c_void_p()
    return w


@pytest.mark.parametrize("shape,lead,group", [
    ((3, 4), (3,), 128), ((3, 1), (3,), 0), ((3,), (3,), 0), ((4,), (), 128), ((1, 4), (), 128), ((), (), 0), ((1,), (), 0),
    ((2, 3, 4), (2, 3), 128), ((6, 4), (2, 3), 128), ((2, 3), (2, 3), 0), ((6,), (2, 3), 0), ((0, 4), (0,), 128), ((4, 4), (4,), 128),
    ((4, 3), (3,), None), ((12,), (3,), None), ((1, 3, 4), (3,), None), ((3, 2, 2), (3,), None), ((3, 0), (3,), None), ((3, 5), (3,), None),
    ((4, 1), (3,), None), ((8,), (4,), None), ((3, 2, 4), (2, 3), None), ((4, 2, 3), (2, 3), None),
])
def test_the_shape_of_x_scales(shape, lead, group):
    w = no_weights()
    if group is not None:
        assert w._x_group(shape, lead) == group
        return
    with pytest.raises(ValueError):
        w._x_group(shape, lead)


def test_w4_host_activations_are_checked():
    """int8 activations without scales (one token too, which was taken as a token with a scale of NaN), scales of other shapes,
    and scales beside float activations."""
    w = no_weights()
    q, x = np.ones((3, 512), np.int8), np.ones((3, 512), np.float32)
    for args in ((q[:1], None), (q[0], None), (q, None), (q, np.ones((4, 3), np.float32)), (q, np.ones((3, 5), np.float32)),
                 (x, np.ones((3, 4), np.float32)), (x[0], np.ones(4, np.float32))):
        with pytest.raises(ValueError):
            w.matmul(*args)
