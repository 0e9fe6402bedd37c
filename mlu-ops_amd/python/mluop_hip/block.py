"""Operators of a residual block over ragged rows (mlu_op_ext.h): layer norm, a gated recurrence along the rows of every sample,
rows by expert and back, dropout onto a residual.  Each function makes one call of the C API on a `Handle` and returns new tensors; all
are names of the package itself."""
import ctypes

from .training import _double, _float, _guarded, _i64, _int, _native, _size, _vp

__all__ = ["layer_norm_forward", "layer_norm_backward", "gated_scan_forward", "gated_scan_backward", "expert_order",
           "expert_dispatch", "expert_combine", "expert_combine_backward", "dropout_add_forward", "dropout_add_backward"]

SIGNATURES = {
    "mluOpExtLayerNormForward": (_int, [_vp, _int, _vp, _i64, _i64, _i64, _int, _vp, _vp, _float, _vp, _vp, _vp]),
    "mluOpExtGetLayerNormBackwardWorkspaceSize": (_int, [_i64, _i64, ctypes.POINTER(_size)]),
    "mluOpExtLayerNormBackward": (_int, [_vp, _int, _vp, _i64, _vp, _i64, _i64, _i64, _int, _vp, _vp, _vp, _vp, _size, _vp,
                                         _vp, _vp]),
    "mluOpExtGetGatedScanSizes": (_int, [_i64, _i64, _i64, ctypes.POINTER(_size), ctypes.POINTER(_size)]),
    "mluOpExtGatedScanForward": (_int, [_vp, _int, _vp, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _vp, _int, _int, _vp, _size,
                                        _vp, _vp, _vp]),
    "mluOpExtGatedScanBackward": (_int, [_vp, _int, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _vp, _int,
                                         _int, _vp, _size, _vp, _vp, _vp]),
    "mluOpExtGetExpertOrderWorkspaceSize": (_int, [_i64, _i64, _i64, ctypes.POINTER(_size)]),
    "mluOpExtExpertOrder": (_int, [_vp, _int, _vp, _i64, _i64, _i64, _vp, _size, _vp, _vp, _vp]),
    "mluOpExtExpertDispatch": (_int, [_vp, _int, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _i64, _vp]),
    "mluOpExtExpertCombine": (_int, [_vp, _int, _vp, _i64, _i64, _i64, _i64, _vp, _int, _vp, _vp]),
    "mluOpExtExpertCombineBackward": (_int, [_vp, _int, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _i64, _int, _vp,
                                             _vp, _vp]),
    "mluOpExtDropoutAdd": (_int, [_vp, _int, _vp, _vp, _i64, _double, _vp, _vp]),
}

# mluOpExtGate_t
GATES = {"sigmoid": 0, "exp": 1}


def layer_norm_forward(handle, features, weight, bias, eps=1e-5):
    """Layer norm of every row of `features` [rows, channels], whose rows may lie apart.  `weight`, `bias` [channels] of the
    features' type or float32, or None.  Returns (out, mean, rstd), the last two float32 [rows]."""
    return _native().layer_norm_forward(handle.ptr.value, _guarded(), features, weight, bias, eps)


def layer_norm_backward(handle, output_grad, features, weight, bias, mean, rstd):
    """Gradients (features, weight, bias) of `layer_norm_forward`, whose mean and rstd it takes."""
    return _native().layer_norm_backward(handle.ptr.value, _guarded(), output_grad, features, weight, bias, mean, rstd)


def gated_scan_forward(handle, features, gates, row_starts=None, initial=None, kind="sigmoid", reverse=False):
    """h_t = a h_(t-1) + (1 - a) x_t with a = sigmoid(gate_t), or ("exp") h_t = a h_(t-1) + x_t with a = exp(gate_t), for every
    channel of `features` and `gates` [rows, channels], whose rows may lie apart.

    `row_starts` int32 [samples + 1] on the device, ascending: sample s has the rows row_starts[s] to row_starts[s + 1] - 1
    (None: all rows are one sample); rows of no sample give zeros.  `initial` float32 [samples, channels]: the states in front
    (None: zero).  `reverse`: from each sample's last row to its first.  Returns (out, final, carries): the states behind every
    row, those behind each sample's last, float32, and what `gated_scan_backward` takes."""
    return _native().gated_scan_forward(handle.ptr.value, _guarded(), features, gates, row_starts, initial, GATES[kind],
                                        reverse)


def gated_scan_backward(handle, output_grad, final_grad, features, gates, carries, row_starts=None, kind="sigmoid",
                        reverse=False):
    """Gradients (features, gates, initial) of `gated_scan_forward`, whose carries it takes; `final_grad` may be None."""
    return _native().gated_scan_backward(handle.ptr.value, _guarded(), output_grad, final_grad, features, gates, carries,
                                         row_starts, GATES[kind], reverse)


def expert_order(handle, experts_of_rows, experts):
    """(rows, group_starts, places) of a routing [rows, choices], int32 or int64: the row at every place when all choices are
    ordered by expert (equal experts by row and choice), -1 behind the last expert's; where each expert's places begin, int32
    [experts + 1]; and the place of every choice, int32 [rows, choices].  A number outside [0, experts) is no expert, and its
    choice has place -1.  At most 2047 experts."""
    return _native().expert_order(handle.ptr.value, _guarded(), experts_of_rows, experts)


def expert_dispatch(handle, features, places, group_starts):
    """The rows of `features` [rows, channels] at the places of their choices: [rows * choices, channels], zeros from
    group_starts[-1] on.  `places` and `group_starts` are those of `expert_order`."""
    return _native().expert_dispatch_rows(handle.ptr.value, _guarded(), features, places, group_starts)


def expert_combine(handle, results, places, weights=None):
    """out[r] = sum over k of weights[r, k] * results[places[r, k]]: [rows, channels].  `weights` [rows, choices] of the results'
    type or float32 (None: one); a choice with place -1 adds nothing.  Without weights it is the gradient of the features of
    `expert_dispatch`."""
    return _native().expert_combine_rows(handle.ptr.value, _guarded(), results, places, weights)


def expert_combine_backward(handle, output_grad, results, places, weights, group_starts):
    """Gradients (results, weights) of `expert_combine`; the second is None without weights."""
    return _native().expert_combine_backward(handle.ptr.value, _guarded(), output_grad, results, places, weights, group_starts)


def dropout_add_forward(handle, features, residual, p, state):
    """residual + features / (1 - p), where each element of `features` is dropped with probability p (taken to a multiple of
    2^-16).  `residual` may be None.  `state` int64 [2] on the device: a seed and the number of the call, which with an element's
    number decide whether it is kept."""
    return _native().dropout_add_rows(handle.ptr.value, _guarded(), features, residual, p, state)


def dropout_add_backward(handle, output_grad, p, state):
    """Gradient of the features of `dropout_add_forward`, for the same p and state (that of the residual is output_grad)."""
    return _native().dropout_add_rows(handle.ptr.value, _guarded(), output_grad, None, p, state)
