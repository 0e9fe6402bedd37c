"""Tables without rows on a handle without a device: taken where there are no tokens, refused where there are."""
import ctypes
import os

import pytest

os.environ.setdefault("MLUOP_LOG_PRINT", "0")

import mluop_hip as m  # noqa: E402

SOME = 1 << 12  # an address that is never looked at


@pytest.fixture
def handle(monkeypatch):
    monkeypatch.setenv("MLUOP_HOST_ONLY_HANDLE", "1")
    h = m.Handle()
    yield h
    h.close()


def test_embedding(handle):
    lib, size = m.lib(), ctypes.c_size_t()
    # (a call that passes every check stops where it would need the device)
    forward, backward = lib.mluOpExtEmbeddingForward, lib.mluOpExtEmbeddingBackward
    for tokens, status in ((0, m.STATUS_EXECUTION_FAILED), (1, m.STATUS_BAD_PARAM)):
        assert forward(handle.ptr, m.DTYPE_FLOAT, None, 0, 8, 8, m.DTYPE_INT32, SOME, tokens, 1.0, SOME) == status
        queried = lib.mluOpExtGetEmbeddingBackwardWorkspaceSize(tokens, 0, 8, ctypes.byref(size))
        assert queried == (0 if tokens == 0 else m.STATUS_BAD_PARAM)
        assert backward(handle.ptr, m.DTYPE_FLOAT, SOME, 8, m.DTYPE_INT32, SOME, tokens, 0, 8, 1.0, SOME, size.value,
                        None) == status
    assert forward(handle.ptr, m.DTYPE_FLOAT, SOME, -1, 8, 8, m.DTYPE_INT32, SOME, 0, 1.0, SOME) == m.STATUS_BAD_PARAM
