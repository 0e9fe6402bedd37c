"""Sizes that the operators of a training step refuse because no launch holds them (queries: no GPU)."""
import ctypes
import os

os.environ.setdefault("MLUOP_LOG_PRINT", "0")

import mluop_hip as m  # noqa: E402


def test_group_norm_pairs_of_a_sample_and_a_group():
    """a workgroup of 256 threads for each of them, and for every four channels, in one grid of fewer than 2^32 threads"""
    size = ctypes.c_size_t()
    query = m.lib().mluOpExtGetGroupNormWorkspaceSize
    most = 15 << 20
    assert query(100, 32, 32, most // 32, ctypes.byref(size)) == 0
    assert query(100, 32, 16, 15 << 16, ctypes.byref(size)) == 0
    for channels, groups, samples in ((32, 32, most // 32 + 1), (32, 32, 1 << 20), (16, 16, 1 << 20), (1 << 10, 1 << 8, 1 << 20)):
        assert query(100, channels, groups, samples, ctypes.byref(size)) == m.STATUS_NOT_SUPPORTED
