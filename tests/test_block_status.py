"""Status codes of the operators of a residual block on a handle without a device: every parameter check answers, nothing is
launched, and a call that passes them all stops where it would launch."""
import ctypes
import os

import pytest

os.environ.setdefault("MLUOP_LOG_PRINT", "0")

import mluop_hip as m  # noqa: E402

OK, BAD, FAILED, UNSUPPORTED = 0, m.STATUS_BAD_PARAM, m.STATUS_EXECUTION_FAILED, m.STATUS_NOT_SUPPORTED
SOME = 1 << 12  # an address that is never looked at
F, H, B, I32, I64, U8 = m.DTYPE_FLOAT, m.DTYPE_HALF, m.DTYPE_BFLOAT16, m.DTYPE_INT32, m.DTYPE_INT64, m.DTYPE_UINT8
BIG = 1 << 60


@pytest.fixture
def handle(monkeypatch):
    monkeypatch.setenv("MLUOP_HOST_ONLY_HANDLE", "1")
    h = m.Handle()
    yield h
    h.close()


def call(name, args, **changed):
    values = dict(args, **changed)
    return getattr(m.lib(), name)(*values.values())


def check(name, args, refused):
    """(`args` in order pass every check) `refused`: [(changed arguments, status)]"""
    assert call(name, args) == FAILED
    for changed, status in refused:
        assert call(name, args, **changed) == status, changed


def test_layer_norm(handle):
    size = ctypes.c_size_t()
    query = m.lib().mluOpExtGetLayerNormBackwardWorkspaceSize
    assert query(100, 8, ctypes.byref(size)) == OK and size.value > 0
    assert query(100, 8, None) == BAD and query(-1, 8, ctypes.byref(size)) == BAD and query(100, 0, ctypes.byref(size)) == BAD
    assert query(100, 1 << 16, ctypes.byref(size)) == UNSUPPORTED and query(1 << 45, 8, ctypes.byref(size)) == UNSUPPORTED
    args = dict(handle=handle.ptr, type=H, x=SOME, stride=8, rows=100, channels=8, param=F, weight=SOME, bias=SOME, eps=1e-5,
                out=SOME, mean=SOME, rstd=SOME)
    both = [(dict(handle=None), BAD), (dict(type=U8), BAD), (dict(param=B), BAD), (dict(rows=-1), BAD), (dict(channels=0), BAD),
            (dict(x=None), BAD), (dict(mean=None), BAD), (dict(rstd=None), BAD), (dict(stride=7), BAD), (dict(stride=1 << 45), BAD),
            (dict(channels=1 << 16, stride=1 << 16), UNSUPPORTED)]
    check("mluOpExtLayerNormForward", args, both + [(dict(out=None), BAD), (dict(eps=-1.0), BAD), (dict(eps=float("nan")), BAD)])
    assert call("mluOpExtLayerNormForward", args, weight=None, bias=None) == FAILED
    args = dict(handle=handle.ptr, type=H, dy=SOME, dy_stride=8, x=SOME, stride=8, rows=100, channels=8, param=F, weight=SOME,
                mean=SOME, rstd=SOME, workspace=SOME, size=size.value, dx=SOME, dw=SOME, db=SOME)
    check("mluOpExtLayerNormBackward", args, both + [(dict(dy=None), BAD), (dict(dy_stride=7), BAD), (dict(dx=None), BAD),
                                                     (dict(workspace=None), BAD), (dict(size=size.value - 1), BAD)])
    assert call("mluOpExtLayerNormBackward", args, dw=None, db=None) == FAILED


def test_gated_scan(handle):
    carries, size = ctypes.c_size_t(), ctypes.c_size_t()
    query = m.lib().mluOpExtGetGatedScanSizes
    assert query(1000, 8, 3, ctypes.byref(carries), ctypes.byref(size)) == OK and carries.value > 0 and size.value > 0
    assert query(0, 8, 3, ctypes.byref(carries), ctypes.byref(size)) == OK
    for bad in ((-1, 8, 3), (10, 0, 3), (10, 8, 0)):
        assert query(*bad, ctypes.byref(carries), ctypes.byref(size)) == BAD
    for large in ((1 << 31, 8, 3), (10, 1 << 21, 3), (10, 8, 1 << 21)):
        assert query(*large, ctypes.byref(carries), ctypes.byref(size)) == UNSUPPORTED
    assert query(10, 8, 3, None, ctypes.byref(size)) == BAD and query(10, 8, 3, ctypes.byref(carries), None) == BAD
    assert query(1000, 8, 3, ctypes.byref(carries), ctypes.byref(size)) == OK
    shape = dict(x=SOME, x_stride=8, g=SOME, g_stride=8, rows=1000, channels=8, starts=SOME, samples=3)
    args = dict(handle=handle.ptr, type=B, **shape, initial=None, kind=1, reverse=0, workspace=SOME, size=size.value, out=SOME,
                final=SOME, carries=SOME)
    both = [(dict(handle=None), BAD), (dict(type=I32), BAD), (dict(x=None), BAD), (dict(g=None), BAD), (dict(x_stride=7), BAD),
            (dict(g_stride=1 << 45), BAD), (dict(starts=None), BAD), (dict(samples=0), BAD), (dict(kind=2), BAD),
            (dict(carries=None), BAD), (dict(workspace=None), BAD), (dict(size=size.value - 1), BAD),
            (dict(rows=1 << 31), UNSUPPORTED)]
    check("mluOpExtGatedScanForward", args, both + [(dict(out=None), BAD), (dict(final=None), BAD)])
    assert call("mluOpExtGatedScanForward", args, starts=None, samples=1) == FAILED
    args = dict(handle=handle.ptr, type=B, dh=SOME, dh_stride=8, df=None, **shape, carries=SOME, kind=0, reverse=1,
                workspace=SOME, size=size.value, dx=SOME, dg=SOME, di=None)
    check("mluOpExtGatedScanBackward", args, both + [(dict(dh=None), BAD), (dict(dh_stride=7), BAD), (dict(dx=None), BAD),
                                                     (dict(dg=None), BAD)])


def test_expert_rows(handle):
    size = ctypes.c_size_t()
    query = m.lib().mluOpExtGetExpertOrderWorkspaceSize
    assert query(100, 2, 8, ctypes.byref(size)) == OK and size.value > 0
    for bad in ((-1, 2, 8), (100, 0, 8), (100, 2, 0)):
        assert query(*bad, ctypes.byref(size)) == BAD
    for large in ((1 << 30, 2, 8), (100, 1 << 32, 8), (100, 2, 2048)):
        assert query(*large, ctypes.byref(size)) == UNSUPPORTED
    assert query(100, 2, 8, None) == BAD and query(100, 2, 8, ctypes.byref(size)) == OK
    args = dict(handle=handle.ptr, type=I64, chosen=SOME, rows=100, choices=2, experts=8, workspace=SOME, size=size.value,
                ordered=SOME, starts=SOME, places=SOME)
    check("mluOpExtExpertOrder", args, [
        (dict(handle=None), BAD), (dict(type=F), BAD), (dict(chosen=None), BAD), (dict(rows=-1), BAD), (dict(choices=0), BAD),
        (dict(experts=0), BAD), (dict(workspace=None), BAD), (dict(size=size.value - 1), BAD), (dict(ordered=None), BAD),
        (dict(starts=None), BAD), (dict(places=None), BAD), (dict(experts=4000), UNSUPPORTED)])
    args = dict(handle=handle.ptr, type=H, x=SOME, stride=16, rows=100, channels=16, choices=2, places=SOME, starts=SOME,
                experts=8, out=SOME)
    check("mluOpExtExpertDispatch", args, [
        (dict(handle=None), BAD), (dict(type=I32), BAD), (dict(x=None), BAD), (dict(stride=15), BAD), (dict(rows=-1), BAD),
        (dict(channels=0), BAD), (dict(choices=0), BAD), (dict(places=None), BAD), (dict(starts=None), BAD),
        (dict(experts=0), BAD), (dict(out=None), BAD), (dict(channels=1 << 21, stride=1 << 21), UNSUPPORTED),
        (dict(rows=1 << 30), UNSUPPORTED)])
    args = dict(handle=handle.ptr, type=H, y=SOME, stride=16, rows=100, channels=16, choices=2, places=SOME, weight=F, w=SOME,
                out=SOME)
    check("mluOpExtExpertCombine", args, [
        (dict(handle=None), BAD), (dict(type=U8), BAD), (dict(weight=B), BAD), (dict(y=None), BAD), (dict(stride=15), BAD),
        (dict(places=None), BAD), (dict(out=None), BAD), (dict(choices=0), BAD)])
    assert call("mluOpExtExpertCombine", args, w=None) == FAILED
    args = dict(handle=handle.ptr, type=H, dy=SOME, dy_stride=16, y=SOME, stride=16, rows=100, channels=16, choices=2,
                places=SOME, starts=SOME, experts=8, weight=H, w=SOME, dr=SOME, dw=SOME)
    check("mluOpExtExpertCombineBackward", args, [
        (dict(handle=None), BAD), (dict(weight=B), BAD), (dict(dy=None), BAD), (dict(dy_stride=15), BAD), (dict(y=None), BAD),
        (dict(stride=15), BAD), (dict(places=None), BAD), (dict(starts=None), BAD), (dict(experts=0), BAD), (dict(dr=None), BAD)])
    assert call("mluOpExtExpertCombineBackward", args, y=None, dw=None) == FAILED


def test_dropout(handle):
    args = dict(handle=handle.ptr, type=F, x=SOME, residual=None, count=100, p=0.5, state=SOME, out=SOME)
    check("mluOpExtDropoutAdd", args, [
        (dict(handle=None), BAD), (dict(type=I32), BAD), (dict(x=None), BAD), (dict(out=None), BAD), (dict(state=None), BAD),
        (dict(state=SOME + 4), BAD), (dict(count=-1), BAD), (dict(p=-0.1), BAD), (dict(p=1.1), BAD), (dict(p=float("nan")), BAD),
        (dict(count=1 << 47), UNSUPPORTED)])
