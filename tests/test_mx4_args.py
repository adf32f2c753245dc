"""Refusals of the MX4 entry points, on the CPU: every one of these calls has to end before
any device work."""
import numpy as np
import pytest

import simplang_amd as sa

F, U = np.float32, np.uint8


def _q(m=4, k=64):
    return dict(x=np.zeros((m, k), F), codes=np.zeros((m, (k + 1) // 2), U), scales=np.zeros((m, -(-k // 32)), U))


def _d(m=4, k=64):
    a = _q(m, k)
    return dict(codes=a["codes"], scales=a["scales"], out=a["x"])


def _rows(n, kb):
    return np.zeros((n, kb), U), np.zeros((n, -(-kb // 16)), U)


def _mm(m=4, n=8, kb=32):
    (a, s), (b, t) = _rows(m, kb), _rows(n, kb)
    return dict(a=a, a_scales=s, b=b, b_scales=t, out=np.zeros((m, n), F))


def _gate(m=4, n=8, kb=32):
    (a, s), (b, t), (c, u) = _rows(m, kb), _rows(n, kb), _rows(n, kb)
    return dict(a=a, a_scales=s, w1=b, s1=t, w3=c, s3=u, out=np.zeros((m, n), F))


CALLS = [(sa.quantize_mx4, _q), (sa.dequantize_mx4, _d), (sa.matmul_mx4, _mm), (sa.swiglu_mx4, _gate)]


@pytest.mark.parametrize("f, make, change", [
    (sa.quantize_mx4, _q, dict(codes=np.zeros((4, 31), U))),
    (sa.quantize_mx4, _q, dict(codes=np.zeros((3, 32), U))),
    (sa.quantize_mx4, _q, dict(scales=np.zeros((4, 3), U))),
    (sa.quantize_mx4, _q, dict(x=np.zeros((4, 65), F))),
    (sa.dequantize_mx4, _d, dict(out=np.zeros((4, 62), F))),
    (sa.dequantize_mx4, _d, dict(out=np.zeros((5, 64), F))),
    (sa.dequantize_mx4, _d, dict(scales=np.zeros((4, 1), U))),
    (sa.matmul_mx4, _mm, dict(a=np.zeros((4, 31), U))),
    (sa.matmul_mx4, _mm, dict(a_scales=np.zeros((4, 3), U))),
    (sa.matmul_mx4, _mm, dict(a_scales=np.zeros((3, 2), U))),
    (sa.matmul_mx4, _mm, dict(b_scales=np.zeros((8, 1), U))),
    (sa.matmul_mx4, _mm, dict(b=np.zeros((7, 32), U))),
    (sa.matmul_mx4, _mm, dict(zip(("b", "b_scales"), _rows(8, 48)))),
    (sa.matmul_mx4, _mm, dict(out=np.zeros((4, 7), F))),
    (sa.matmul_mx4, _mm, dict(out=np.zeros((8, 4), F))),
    (sa.swiglu_mx4, _gate, dict(zip(("w3", "s3"), _rows(9, 32)))),
    (sa.swiglu_mx4, _gate, dict(zip(("w1", "s1"), _rows(8, 16)))),
    (sa.swiglu_mx4, _gate, dict(s3=np.zeros((8, 3), U))),
])
def test_refuses_shapes(f, make, change):
    with pytest.raises(sa.SimpRTError, match="shape mismatch"):
        f(**{**make(), **change})


@pytest.mark.parametrize("f, make", CALLS)
def test_refuses_types_ranks_and_strides(f, make):
    for name, x in make().items():
        with pytest.raises(TypeError, match=f"{name} must be"):
            f(**{**make(), name: x.astype(np.int32)})
        with pytest.raises(ValueError, match="rank-2"):
            f(**{**make(), name: x.reshape(-1)})
        with pytest.raises(sa.SimpRTError, match="inner stride"):
            f(**{**make(), name: np.zeros((x.shape[0], 2 * x.shape[1]), x.dtype)[:, ::2]})
        with pytest.raises(sa.SimpRTError, match="stride"):
            one = np.zeros((1, x.shape[1]), x.dtype)
            f(**{**make(), name: np.broadcast_to(one, x.shape)})


def test_refuses_null_pointers_and_overflowing_extents():
    a = np.zeros((4, 64), np.uint8)
    p = a.ctypes.data
    good = [p, p, 0, 4, 32, 32, 1]
    s = [p, p, 0, 4, 2, 2, 1]
    o = [p, p, 0, 4, 4, 4, 1]
    f = sa.lib.simp_rt_matmul_mx4
    assert f(None, None, 0, 4, 32, 32, 1, *s, *good, *s, *o) == -1
    assert b"null" in sa.lib.simp_rt_last_error()
    assert f(*good, *s, p, p, 0, 4, 32, 1 << 62, 1, *s, *o) == -1
    assert b"overflow" in sa.lib.simp_rt_last_error()
    assert f(p, p, -1, 4, 32, 32, 1, *s, *good, *s, *o) == -1
    assert f(*good, *s, *good, *s, p, p, 0, -4, 4, 4, 1) == -1
    big = (1 << 31) - 1
    assert f(p, p, 0, big, 32, 32, 1, p, p, 0, big, 2, 2, 1, *good, *s, p, p, 0, big, 4, 4, 1) == -4


def _views(dtype, shape, at, buf, stride):
    return np.ndarray(shape, dtype, buf, at, (stride, np.dtype(dtype).itemsize))


def test_refuses_shared_memory():
    buf = np.zeros(1 << 16, U)
    match = "share"
    a = _mm()
    with pytest.raises(sa.SimpRTError, match=match):          # out over a row of b
        sa.matmul_mx4(**{**a, "b": _views(U, (8, 32), 0, buf, 32), "out": _views(F, (4, 8), 64, buf, 32)})
    with pytest.raises(sa.SimpRTError, match=match):          # rows between rows, one byte too long
        sa.matmul_mx4(**{**a, "a_scales": _views(U, (4, 2), 32, buf, 64), "out": _views(F, (4, 8), 0, buf, 64)[:, :],
                         "a": _views(U, (4, 32), 31, buf, 64)})
    g = _gate()
    with pytest.raises(sa.SimpRTError, match=match):
        sa.swiglu_mx4(**{**g, "s3": _views(U, (8, 2), 100, buf, 2), "out": _views(F, (4, 8), 0, buf, 32)})
    q = _q()
    with pytest.raises(sa.SimpRTError, match=match):          # codes over x
        sa.quantize_mx4(**{**q, "x": _views(F, (4, 64), 0, buf, 256), "codes": _views(U, (4, 32), 992, buf, 32)})
    with pytest.raises(sa.SimpRTError, match=match):          # scales inside the codes' rows
        sa.quantize_mx4(**{**q, "codes": _views(U, (4, 32), 0, buf, 40), "scales": _views(U, (4, 2), 31, buf, 40)})
    with pytest.raises(sa.SimpRTError, match=match):          # another stride
        sa.quantize_mx4(**{**q, "codes": _views(U, (4, 32), 0, buf, 40), "scales": _views(U, (4, 2), 32, buf, 80)})
    d = _d()
    with pytest.raises(sa.SimpRTError, match=match):
        sa.dequantize_mx4(**{**d, "scales": _views(U, (4, 2), 0, buf, 2), "out": _views(F, (4, 64), 0, buf, 256)})


def test_nothing_to_do_is_no_error():
    sa.quantize_mx4(**_q(m=0))
    sa.quantize_mx4(**_q(k=0))
    sa.dequantize_mx4(**_d(m=0))
    sa.dequantize_mx4(**_d(k=0))
    sa.matmul_mx4(**_mm(m=0))
    sa.matmul_mx4(**_mm(n=0))
    sa.swiglu_mx4(**_gate(m=0, kb=0))
    sa.swiglu_mx4(**_gate(n=0))
