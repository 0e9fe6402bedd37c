"""Operators a network over ragged rows of features needs next to its convolutions (mlu_op_ext.h): each function makes one
call of the C API on a `Handle` and returns new tensors; all are names of the package itself."""
import ctypes

__all__ = ["AdamWTensors", "embedding_forward", "embedding_backward", "group_norm_forward", "group_norm_backward",
           "grouped_matmul_forward", "grouped_matmul_backward_data", "grouped_matmul_backward_filter"]

_vp = ctypes.c_void_p
_int, _i64, _float, _double, _size = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_double, ctypes.c_size_t

SIGNATURES = {
    "mluOpExtAdamWStep": (_int, [_vp, _vp, _int, _int, _int, _int, _i64] + [_double] * 6),
    "mluOpExtGetGroupNormWorkspaceSize": (_int, [_i64, _i64, _i64, _i64, ctypes.POINTER(_size)]),
    "mluOpExtGroupNormForward": (_int, [_vp, _int, _vp, _i64, _i64, _i64, _vp, _i64, _int, _vp, _vp, _float, _int, _vp,
                                        _size, _vp, _vp, _vp]),
    "mluOpExtGroupNormBackward": (_int, [_vp, _int, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _int, _vp, _vp, _vp, _vp, _int,
                                         _vp, _size, _vp, _vp, _vp]),
    "mluOpExtEmbeddingForward": (_int, [_vp, _int, _vp, _i64, _i64, _i64, _int, _vp, _i64, _float, _vp]),
    "mluOpExtGetEmbeddingBackwardWorkspaceSize": (_int, [_i64, _i64, _i64, ctypes.POINTER(_size)]),
    "mluOpExtEmbeddingBackward": (_int, [_vp, _int, _vp, _i64, _int, _vp, _i64, _i64, _i64, _float, _vp, _size, _vp]),
    "mluOpExtGetGroupedMatmulWorkspaceSize": (_int, [_vp, _int, _int, _i64, _i64, _i64, _i64, ctypes.POINTER(_size)]),
    "mluOpExtGroupedMatmulForward": (_int, [_vp, _int, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _size, _vp]),
    "mluOpExtGroupedMatmulBackwardData": (_int, [_vp, _int, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _size, _vp]),
    "mluOpExtGroupedMatmulBackwardFilter": (_int, [_vp, _int, _vp, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _i64, _vp,
                                                   _size, _vp]),
}

# mluOpExtActivation_t
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2}


def _native():
    from . import native
    return native()


def _guarded():
    from . import _guarded
    return _guarded()


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


def group_norm_forward(handle, features, weight, bias, groups, row_starts=None, eps=1e-5, activation="none"):
    """Group norm with an activation over `features` [rows, channels].

    `row_starts` int32 [samples + 1] on the device, ascending: sample s has the rows row_starts[s] to row_starts[s + 1] - 1
    (None: all rows are one sample).  `weight`, `bias` [channels] of the features' type or float32, or None.
    Returns (out, mean, rstd), the last two float32 [samples, groups]."""
    return _native().group_norm_forward(handle.ptr.value, _guarded(), features, weight, bias, groups, row_starts, eps,
                                        ACTIVATIONS[activation])


def group_norm_backward(handle, output_grad, features, weight, bias, mean, rstd, groups, row_starts=None,
                        activation="none"):
    """Gradients (features, weight, bias) of `group_norm_forward`, whose mean and rstd it takes."""
    return _native().group_norm_backward(handle.ptr.value, _guarded(), output_grad, features, weight, bias, mean, rstd,
                                         groups, row_starts, ACTIVATIONS[activation])


def embedding_forward(handle, table, tokens, scale=1.0):
    """scale * table[tokens]: [*tokens.shape, channels] of the table's type.  `tokens` are int32 or int64; one outside
    [0, rows) names no row, and its result is zero.  The table's rows may lie apart."""
    return _native().embedding_forward(handle.ptr.value, _guarded(), table, tokens, scale)


def embedding_backward(handle, output_grad, tokens, rows, scale=1.0):
    """Gradient [rows, channels] of the table of `embedding_forward`: each row adds up the gradients of the tokens that
    name it, in fp32 and in an order that the tokens alone decide."""
    return _native().embedding_backward(handle.ptr.value, _guarded(), output_grad, tokens, rows, scale)


def grouped_matmul_forward(handle, features, filters, group_starts):
    """Rows group_starts[g] to group_starts[g + 1] - 1 of `features` [rows, ci] times filters[g] of [groups, ci, co]:
    [rows, co].  `group_starts` int32 [groups + 1] on the device, ascending, any group empty; rows of no group give zeros.
    The features' rows may lie apart."""
    return _native().grouped_matmul_rows(handle.ptr.value, _guarded(), features, filters, group_starts, True)


def grouped_matmul_backward_data(handle, output_grad, filters, group_starts):
    """Gradient [rows, ci] of the features of `grouped_matmul_forward`."""
    return _native().grouped_matmul_rows(handle.ptr.value, _guarded(), output_grad, filters, group_starts, False)


def grouped_matmul_backward_filter(handle, features, output_grad, group_starts):
    """Gradient [groups, ci, co] of the filters of `grouped_matmul_forward`; zero for a group without rows."""
    return _native().grouped_matmul_backward_filter(handle.ptr.value, _guarded(), features, output_grad, group_starts)
