"""Operators a network over ragged rows of features needs next to its convolutions (mlu_op_ext.h): each function makes one
call of the C API on a `Handle` and returns new tensors; all are names of the package itself."""
import ctypes

__all__ = ["AdamWTensors"]

_vp = ctypes.c_void_p
_int, _i64, _float, _double, _size = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_double, ctypes.c_size_t

SIGNATURES = {
    "mluOpExtAdamWStep": (_int, [_vp, _vp, _int, _int, _int, _int, _i64] + [_double] * 6),
}


def _native():
    from . import native
    return native()


class AdamWTensors:
    """Parameters and optimizer states of an AdamW step over many tensors (mluOpExtAdamWStep), checked once and kept.

    `params` are float32, float16 or bfloat16, all of one type; `masters` fp32 copies of 16-bit params.  States are float32
    of the params' sizes, or, with `exp_avg_scales` and `exp_avg_sq_scales` (float32, one for each 256 elements),
    torch.float8_e4m3fn (or uint8 codes): exp_avgs hold m, exp_avg_sqs the root of v, both in units of their scales.
    `step` updates them in place; a param whose gradient is None is left alone."""

    def __init__(self, params, exp_avgs, exp_avg_sqs, masters=None, exp_avg_scales=None, exp_avg_sq_scales=None):
        self._tensors = _native().AdamWTensors(list(params), list(exp_avgs), list(exp_avg_sqs), masters, exp_avg_scales,
                                              exp_avg_sq_scales)

    def step(self, handle, grads, step, lr, betas, eps, weight_decay, grad_scale=1.0):
        """`step` counts from 1.  `grad_scale` multiplies the gradients (the reciprocal of a loss scale)."""
        self._tensors.step(handle.ptr.value, grads, step, lr, betas[0], betas[1], eps, weight_decay, grad_scale)
