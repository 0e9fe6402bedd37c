"""Status codes of the operators of a training step on a handle without a device: every parameter check answers, nothing is
launched, and a call that passes them all stops where it would launch."""
import ctypes
import os

import pytest

os.environ.setdefault("MLUOP_LOG_PRINT", "0")

import mluop_hip as m  # noqa: E402

OK, BAD, FAILED, UNSUPPORTED = 0, m.STATUS_BAD_PARAM, m.STATUS_EXECUTION_FAILED, m.STATUS_NOT_SUPPORTED
SOME = 1 << 12  # an address that is never looked at
F, H, B, I32, I64, U8 = m.DTYPE_FLOAT, m.DTYPE_HALF, m.DTYPE_BFLOAT16, m.DTYPE_INT32, m.DTYPE_INT64, m.DTYPE_UINT8
BIG = 1 << 40


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


def test_embedding(handle):
    args = dict(handle=handle.ptr, type=F, table=SOME, rows=10, channels=8, stride=8, token_type=I32, tokens=SOME, n=5,
                scale=1.0, out=SOME)
    check("mluOpExtEmbeddingForward", args, [
        (dict(handle=None), BAD), (dict(type=I32), BAD), (dict(token_type=F), BAD), (dict(rows=0), BAD),
        (dict(channels=0), BAD), (dict(stride=7), BAD), (dict(n=-1), BAD), (dict(table=None), BAD), (dict(tokens=None), BAD),
        (dict(out=None), BAD), (dict(rows=1 << 31), UNSUPPORTED), (dict(n=1 << 31), UNSUPPORTED),
        (dict(channels=1 << 21, stride=1 << 21), UNSUPPORTED), (dict(stride=1 << 45), BAD)])
    size = ctypes.c_size_t()
    query = m.lib().mluOpExtGetEmbeddingBackwardWorkspaceSize
    assert query(5, 10, 8, ctypes.byref(size)) == OK and size.value > 0
    assert query(5, 10, 8, None) == BAD and query(5, 0, 8, ctypes.byref(size)) == BAD
    assert query(1 << 31, 10, 8, ctypes.byref(size)) == UNSUPPORTED
    args = dict(handle=handle.ptr, type=B, grad=SOME, stride=8, token_type=I64, tokens=SOME, n=5, rows=10, channels=8,
                scale=1.0, workspace=SOME, size=size.value, out=SOME)
    check("mluOpExtEmbeddingBackward", args, [
        (dict(handle=None), BAD), (dict(type=I32), BAD), (dict(token_type=H), BAD), (dict(grad=None), BAD),
        (dict(tokens=None), BAD), (dict(stride=7), BAD), (dict(workspace=None), BAD), (dict(size=size.value - 1), BAD),
        (dict(out=None), BAD), (dict(rows=-1), BAD)])


def test_group_norm(handle):
    size = ctypes.c_size_t()
    query = m.lib().mluOpExtGetGroupNormWorkspaceSize
    assert query(100, 8, 2, 3, ctypes.byref(size)) == OK and size.value > 0
    for bad in ((-1, 8, 2, 3), (100, 8, 3, 3), (100, 0, 1, 3), (100, 8, 0, 3), (100, 8, 2, 0)):
        assert query(*bad, ctypes.byref(size)) == BAD
    assert query(1 << 31, 8, 2, 1, ctypes.byref(size)) == UNSUPPORTED and query(100, 8, 2, 3, None) == BAD
    assert query(100, 8, 2, 3, ctypes.byref(size)) == OK
    shape = dict(rows=100, channels=8, groups=2, starts=SOME, samples=3, param=F, weight=SOME, bias=SOME)
    args = dict(handle=handle.ptr, type=H, x=SOME, **shape, eps=1e-5, act=2, workspace=SOME, size=size.value, out=SOME,
                mean=SOME, rstd=SOME)
    both = [(dict(handle=None), BAD), (dict(type=U8), BAD), (dict(param=B), BAD), (dict(groups=3), BAD), (dict(starts=None), BAD),
            (dict(act=3), BAD), (dict(workspace=None), BAD), (dict(size=size.value - 1), BAD),
            (dict(mean=None), BAD), (dict(rstd=None), BAD), (dict(x=None), BAD), (dict(channels=1 << 21, groups=1), UNSUPPORTED)]
    check("mluOpExtGroupNormForward", args, both + [(dict(eps=-1.0), BAD), (dict(eps=float("nan")), BAD), (dict(out=None), BAD)])
    assert call("mluOpExtGroupNormForward", args, weight=None, bias=None) == FAILED
    args = dict(handle=handle.ptr, type=H, dy=SOME, x=SOME, **shape, mean=SOME, rstd=SOME, act=2, workspace=SOME,
                size=size.value, dx=SOME, dw=SOME, db=SOME)
    check("mluOpExtGroupNormBackward", args, both + [(dict(dy=None), BAD), (dict(dx=None), BAD)])
    assert call("mluOpExtGroupNormBackward", args, dw=None, db=None) == FAILED


def test_grouped_matmul(handle):
    size = ctypes.c_size_t(1)
    query = m.lib().mluOpExtGetGroupedMatmulWorkspaceSize
    for which in (0, 1, 2):
        assert query(handle.ptr, which, H, 100, 4, 8, 16, ctypes.byref(size)) == OK
    for bad in ((3, H, 100, 4, 8, 16), (0, I32, 100, 4, 8, 16), (0, H, -1, 4, 8, 16), (0, H, 100, 0, 8, 16),
                (0, H, 100, 4, 0, 16), (0, H, 100, 4, 8, 0)):
        assert query(handle.ptr, *bad, ctypes.byref(size)) == BAD
    for large in ((0, H, 1 << 31, 4, 8, 16), (0, H, 100, 65536, 8, 16), (0, H, 100, 4, 1 << 16, 1 << 16)):
        assert query(handle.ptr, *large, ctypes.byref(size)) == UNSUPPORTED
    assert query(None, 0, H, 100, 4, 8, 16, ctypes.byref(size)) == BAD and query(handle.ptr, 0, H, 100, 4, 8, 16, None) == BAD
    shape = dict(rows=100, starts=SOME, groups=4, ci=8, co=16)
    for name, stride in (("Forward", 8), ("BackwardData", 16)):
        args = dict(handle=handle.ptr, type=H, x=SOME, stride=stride, **shape, filters=SOME, workspace=SOME, size=BIG, out=SOME)
        check("mluOpExtGroupedMatmul" + name, args, [
            (dict(handle=None), BAD), (dict(type=U8), BAD), (dict(x=None), BAD), (dict(stride=stride - 1), BAD),
            (dict(stride=1 << 45), BAD), (dict(starts=None), BAD), (dict(groups=0), BAD), (dict(filters=None), BAD),
            (dict(out=None), BAD), (dict(rows=1 << 31), UNSUPPORTED)])
    args = dict(handle=handle.ptr, type=B, x=SOME, x_stride=8, dy=SOME, dy_stride=16, **shape, workspace=SOME, size=BIG, out=SOME)
    check("mluOpExtGroupedMatmulBackwardFilter", args, [
        (dict(handle=None), BAD), (dict(x=None), BAD), (dict(dy=None), BAD), (dict(x_stride=7), BAD), (dict(dy_stride=15), BAD),
        (dict(starts=None), BAD), (dict(out=None), BAD), (dict(co=0), BAD)])


class Tensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "m", "v", "master", "m_scale", "v_scale")] + [("count", ctypes.c_int64)]


def test_adamw(handle):
    def tensors(*all_of):
        return (Tensor * len(all_of))(*all_of)
    plain = Tensor(SOME, SOME, SOME, SOME, None, None, None, 10)
    one = tensors(plain)
    args = dict(handle=handle.ptr, tensors=one, n=1, param=F, grad=F, state=F, step=1, lr=1e-3, beta1=0.9, beta2=0.99,
                eps=1e-8, decay=0.0, scale=1.0)
    nan = float("nan")
    check("mluOpExtAdamWStep", args, [
        (dict(handle=None), BAD), (dict(tensors=None), BAD), (dict(n=-1), BAD), (dict(param=I32), BAD), (dict(grad=H), BAD),
        (dict(state=H), BAD), (dict(step=0), BAD), (dict(lr=nan), BAD), (dict(beta1=1.0), BAD), (dict(beta2=-0.1), BAD),
        (dict(eps=-1.0), BAD), (dict(decay=nan), BAD), (dict(scale=float("inf")), BAD),
        (dict(state=U8), BAD),                                                     # no scales
        (dict(tensors=tensors(Tensor(SOME, SOME, SOME, SOME, SOME, None, None, 10))), BAD),   # fp32 params with a master
        (dict(tensors=tensors(Tensor(SOME, None, SOME, SOME, None, None, None, 10))), BAD),
        (dict(tensors=tensors(Tensor(SOME, SOME, None, SOME, None, None, None, 10))), BAD),
        (dict(tensors=tensors(Tensor(SOME, SOME, SOME, SOME, None, None, None, -1))), BAD)])
    mixed = tensors(plain, Tensor(SOME, SOME, SOME, SOME, SOME, None, None, 10))
    assert call("mluOpExtAdamWStep", args, tensors=mixed, n=2, param=H, grad=H) == BAD
    # tensors of nothing have no addresses
    assert call("mluOpExtAdamWStep", args, tensors=tensors(Tensor(None, None, None, None, None, None, None, 0), plain), n=2) == FAILED
