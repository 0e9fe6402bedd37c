"""PyTorch caller layer over the C API: the call sequence mmcv's sparse-conv ops run against
mlu-ops (descriptor -> workspace size -> mluOpGetIndicePairs -> num_act_out -> device-to-host
copy of indice_num -> the three indice-convolution operators), wrapped in an autograd function and
the modules `SubMConv3d`, `SparseConv3d` and `SparseInverseConv3d` (the last one through the
library's extended modes, which the reference does not have).

A `SparseTensor` carries features [L, C], int32 indices [L, 4] = (n, d, h, w), the spatial shape
and the batch size, plus a cache of rulebooks keyed by `indice_key`, so that stacked submanifold
layers with the same key build the rulebook once (the reference design's layer chain,
docs/design_docs/indice_convolution_forward/indice_convolution_forward.md:229-234).

torch is used for device memory, the stream and the autograd graph only; every number is computed
by libmluops.so.  Weights are stored [kd, kh, kw, Ci, Co] (LAYOUT_ARRAY), the one layout all three
operators accept (indice_convolution_backward_filter.cpp:227-242 in the reference)."""
import math

import torch

from . import Handle, _capturing, _guarded, get_indice_pairs, native, regular_output_space, rulebook_counts
from .training import ACTIVATIONS

_handles = {}


def _handle():
    """The library handle of the current device and stream (made by the native path, which keeps one for
    each: a handle is used from one stream at a time)."""
    address = native().stream_handle()
    if address not in _handles:
        _handles[address] = Handle.borrowed(address)
    return _handles[address]


_share_row_maps = False


def share_row_maps(enable):
    """Layers and passes that use one rulebook share its row maps (built once per rulebook, direction
    and stream, without the verifying count since the coordinates are known to be distinct)
    instead of rebuilding them in every operator call or reading the pair lists.  Pays a little when a
    rulebook serves many calls (a fixed scene: the forward of a 64 -> 64 layer on 120 000 rows takes
    30.2 us with a kept map and 30.7 to 31.8 us on the pair lists); with a new rulebook per step and two
    layers per stage the pair lists are faster (the 11-layer encoder: 2.93 ms a step, 3.14 ms with
    shared maps), and the maps hold K x rows x 8 bytes per rulebook,
    hence off by default."""
    global _share_row_maps
    _share_row_maps = bool(enable)


# How many rulebooks of a plan may have their pair counts outstanding, and of how many offsets: a handle has those of 32
# rulebooks of up to 343 on file, and others are copied, behind whatever convolutions are enqueued by then (40 layers:
# the device was drained eight times).
_PENDING, _COUNTED = 16, 343


class Rulebook:
    """indice_pairs [K,2,L] (device; -1 behind an offset's indice_num pairs, with `tails` off only once `pairs` has
    been asked for: the operators read no further than the pairs), indice_num as host ints (where
    `indice_num_host` is the device tensor, those that the handle `built_on` has on file, waited for when first
    asked for), out_indices, num_act_out."""

    def __init__(self, pairs, out_indices, indice_num_host, num_act_out, filter_space, sub_m, out_space,
                 in_indices=None, in_space=None, distinct=False, built_on=None, tails=True, single=False, in_ordered=None,
                 out_ordered=None):
        # the input coordinates were distinct: no offset names a result row twice, and the
        # operators may skip their check for such pairs (mluOpExtSetDistinctPairsPromise)
        self.distinct = distinct
        # no input row is in two pairs: a kernel that reaches no further than its stride (the gradient of such a
        # layer's input, and its inverse, multiply full tiles of pairs: mluOpExtSetSinglePairsPromise)
        self.single = single
        self.in_indices = in_indices  # what an inverse convolution over this rulebook gives back
        # whether their rows, and those of out_indices, lie sample after sample (None: nobody knows)
        self.in_ordered, self.out_ordered = in_ordered, out_ordered
        self.in_space = None if in_space is None else tuple(in_space)
        self._pairs = pairs
        self._tails = tails
        self.out_indices = out_indices
        self._indice_num = indice_num_host
        self._built_on = built_on
        self.num_act_out = num_act_out
        self.filter_space = tuple(filter_space)
        self.counts_are_copied = math.prod(self.filter_space) > _COUNTED
        self.sub_m = sub_m
        self.out_space = tuple(out_space)
        self._for_operators = None

    @property
    def pairs(self):
        if not self._tails:
            with torch.inference_mode(self._pairs.is_inference()):
                for of_offset, n in zip(self._pairs, self.indice_num):
                    of_offset[:, n:].fill_(-1)
            self._tails = not _capturing()   # (what is captured has not run)
        return self._pairs

    @pairs.setter
    def pairs(self, value):
        self._pairs, self._tails = value, True

    @property
    def indice_num(self):
        num = self._indice_num
        if isinstance(num, torch.Tensor):
            # (an operator may have taken them: the handle need not have them on file any more)
            self._indice_num = num = (rulebook_counts(self._built_on, self._pairs, num) if self._for_operators is None
                                      else self._for_operators.counts())
        return num

    @indice_num.setter
    def indice_num(self, value):
        self._indice_num = value

    def for_operators(self):
        """What the native operators take of this rulebook; it holds the row maps they share, and waits for the pair counts
        itself when the first of them needs them."""
        if self._for_operators is None:
            num = self._indice_num
            pending = (num, self._built_on.ptr.value) if isinstance(num, torch.Tensor) else (None, 0)
            self._for_operators = native().LayerRulebook(self._pairs, None if pending[1] else num, self.num_act_out,
                                                         list(self.filter_space), self.sub_m, self.distinct,
                                                         self.single, *pending)
        return self._for_operators

    @property
    def _row_maps(self):
        """{(handle address, pair column that names the result rows): True} of the row maps built so far (with
        `share_row_maps` on, for coordinates known to be distinct; on first use, one per handle and direction)."""
        return {} if self._for_operators is None else dict.fromkeys(self._for_operators.row_maps(), True)


def _in_sample_order(samples):
    return samples.shape[0] < 2 or bool((samples[1:] >= samples[:-1]).all())


class SparseTensor:
    """`distinct=True` is the caller's word that no coordinate occurs twice (the output of a
    voxelizer, or of a strided layer, never repeats one); the convolution operators then skip
    their check for pairs of one offset that share a result row.

    `ordered=True` is the caller's word that rows lie sample after sample (a strided layer's do, whatever its input's).  With
    None the first layer that takes statistics by sample looks, once for all layers on these coordinates, and waits for the
    answer; rows in no order are put into one for it.  (Behind guard bands the word is checked.)"""

    def __init__(self, features, indices, spatial_shape, batch_size, rulebooks=None, distinct=False, ordered=None):
        assert indices.dtype == torch.int32 and indices.dim() == 2 and indices.shape[1] == 4
        assert features.shape[0] == indices.shape[0]
        self.features = features
        self.indices = indices.contiguous()
        self.spatial_shape = tuple(int(s) for s in spatial_shape)
        self.batch_size = int(batch_size)
        self.rulebooks = {} if rulebooks is None else rulebooks
        self.distinct = bool(distinct)
        self.ordered = ordered

    def replace_features(self, features):
        return SparseTensor(features, self.indices, self.spatial_shape, self.batch_size, self.rulebooks,
                            self.distinct, self.ordered)

    def _rows_of_samples(self):
        """(order, places, starts), None for one sample: the rows sample after sample and the place of every row among them
        (int32, None where they lie so), and where every sample's begin (int32 [batch_size + 1]).  Kept with the rulebooks."""
        if self.batch_size == 1:
            return None, None, None
        kept = self.rulebooks.get(("samples", id(self.indices)))
        if kept is not None and kept[0] is self.indices:
            return kept[1:]
        if _capturing() and not self.ordered:
            raise RuntimeError("whether a SparseTensor's rows are ordered by sample cannot be waited for while a graph is "
                               "captured: say so (ordered=True), or run a layer on it before")
        with torch.no_grad(), torch.inference_mode(False):
            samples, order, places = self.indices[:, 0].contiguous(), None, None
            if self.ordered and _guarded() and not _capturing() and not _in_sample_order(samples):
                raise ValueError("a SparseTensor's rows were said to be ordered by sample, and are not")
            if not self.ordered and not (self.ordered is None and _in_sample_order(samples)):
                samples, order = torch.sort(samples, stable=True)
                places = torch.empty_like(order, dtype=torch.int32)
                places[order] = torch.arange(order.shape[0], device=order.device, dtype=torch.int32)
                order = order.to(torch.int32)
            numbers = torch.arange(self.batch_size + 1, device=samples.device, dtype=torch.int32)
            starts = torch.searchsorted(samples, numbers, out_int32=True)
        if not _capturing():   # (what is captured has not run)
            self.rulebooks[("samples", id(self.indices))] = (self.indices, order, places, starts)
        return order, places, starts

    def row_starts(self):
        """int32 [batch_size + 1]: where every sample's rows begin; None for one sample.  Of rows that are ordered by sample
        only: others raise a ValueError."""
        order, _, starts = self._rows_of_samples()
        if order is not None:
            raise ValueError("the rows are not ordered by sample")
        return starts

    def dense(self):
        """[N, C, D, H, W] dense tensor (for inspection and tests)."""
        d, h, w = self.spatial_shape
        out = torch.zeros((self.batch_size, d, h, w, self.features.shape[1]), dtype=self.features.dtype,
                          device=self.features.device)
        i = self.indices.long()
        out[i[:, 0], i[:, 1], i[:, 2], i[:, 3]] = self.features
        return out.permute(0, 4, 1, 2, 3).contiguous()


class _IndiceConv:
    """The layers' differentiable convolution; its autograd node is native (csrc/python/native.cpp)."""

    @staticmethod
    def apply(features, weight, rulebook, inverse=False, relu=False):
        return native().indice_conv(features, weight, rulebook.for_operators(), inverse, _share_row_maps,
                                    _guarded(), relu)


def _triple(v):
    return [int(v)] * 3 if isinstance(v, int) else [int(x) for x in v]


class _ConvBase(torch.nn.Module):
    inverse = False

    def __init__(self, in_channels, out_channels, kernel_size, stride, padding, dilation, sub_m, bias,
                 indice_key):
        super().__init__()
        self.in_channels, self.out_channels = in_channels, out_channels
        self.kernel_size = _triple(kernel_size)
        self.stride, self.padding, self.dilation = _triple(stride), _triple(padding), _triple(dilation)
        self.sub_m = sub_m
        self.indice_key = indice_key
        k = self.kernel_size[0] * self.kernel_size[1] * self.kernel_size[2]
        bound = 1.0 / math.sqrt(k * in_channels)
        self.weight = torch.nn.Parameter(
            torch.empty(*self.kernel_size, in_channels, out_channels).uniform_(-bound, bound))
        self.bias = torch.nn.Parameter(torch.zeros(out_channels)) if bias else None

    def _rulebook(self, x, wait_counts=True):
        if self.indice_key is not None and self.indice_key in x.rulebooks:
            rb = x.rulebooks[self.indice_key]
            assert rb.filter_space == tuple(self.kernel_size) and rb.sub_m == self.sub_m
            return rb
        # a rulebook planned for this layer and these very coordinates (SparseSequential)
        planned = x.rulebooks.get(("planned", id(self)))
        if planned is not None and planned.in_indices is x.indices and planned.in_space == x.spatial_shape:
            return planned
        if self.sub_m:
            out_space = list(x.spatial_shape)
        else:
            out_space = regular_output_space(x.spatial_shape, self.kernel_size, self.padding, self.stride,
                                             self.dilation)
        # the operators take indice_num as host ints: one wait per rulebook, here or in the first of them
        handle = _handle()
        pairs, out_indices, num, n_out = get_indice_pairs(
            handle, x.indices, x.batch_size, x.spatial_shape, self.kernel_size, out_space, self.padding,
            self.stride, self.dilation, self.sub_m, for_layer=True, tails=False, wait_counts=wait_counts)
        rb = Rulebook(pairs, out_indices, num, n_out, self.kernel_size, self.sub_m,
                      out_space, in_indices=x.indices, in_space=x.spatial_shape, distinct=x.distinct,
                      built_on=handle, tails=False, in_ordered=x.ordered,
                      # (a regular rulebook numbers its output cells in their linear order)
                      out_ordered=x.ordered if self.sub_m else True,
                      single=not self.sub_m and all((k - 1) * d < s for k, d, s in
                                                    zip(self.kernel_size, self.dilation, self.stride)))
        if self.indice_key is not None:
            x.rulebooks[self.indice_key] = rb
        else:
            x.rulebooks[("planned", id(self))] = rb
        return rb

    def _plain_rulebook(self):
        """Whether `_rulebook` takes `wait_counts`: it is the library's, and not one put in its place."""
        return getattr(self._rulebook, "__func__", None) in (_ConvBase._rulebook, SparseInverseConv3d._rulebook)

    def _cells_after(self, x, rb):
        """(indices, spatial shape, distinct) of this layer's result on `x`, from the rulebook alone."""
        if self.sub_m:
            return x.indices, x.spatial_shape, x.distinct
        if self.inverse:
            return rb.in_indices, rb.in_space, rb.distinct
        return rb.out_indices.contiguous(), rb.out_space, True

    def _order_after(self, x, rb):
        """What is known about the order of this layer's result on `x`, by sample."""
        return x.ordered if self.sub_m else getattr(rb, "in_ordered" if self.inverse else "out_ordered", None)

    def _result(self, x, rb, feats):
        if self.sub_m:
            return x.replace_features(feats)
        # the cache travels on, so that an inverse layer downstream finds this rulebook by its key;
        # the active output cells of a regular convolution are distinct by construction
        return SparseTensor(feats, rb.out_indices.contiguous(), rb.out_space, x.batch_size, x.rulebooks,
                            distinct=True, ordered=self._order_after(x, rb))

    def forward(self, x):
        return self._convolve(x)

    def _convolve(self, x, **store):
        # (the counts are waited for in the operator, behind what the host has to do there: 60 000 rows, 48 -> 48
        # channels 53 -> 48 us, a training step of 3001 rows 109 -> 99)
        rb = self._rulebook(x, wait_counts=False) if self._plain_rulebook() else self._rulebook(x)
        feats, weight = x.features, self.weight.to(x.features.dtype)
        feats = _IndiceConv.apply(feats, weight, rb, self.inverse, **store)
        if self.bias is not None:
            feats = feats + self.bias.to(feats.dtype)
        return self._result(x, rb, feats)


class SubMConv3d(_ConvBase):
    """Submanifold 3-D sparse convolution: outputs live on the input's active cells."""

    def __init__(self, in_channels, out_channels, kernel_size, dilation=1, bias=False, indice_key=None):
        ks = _triple(kernel_size)
        dil = _triple(dilation)
        pad = [d * (k // 2) for k, d in zip(ks, dil)]
        super().__init__(in_channels, out_channels, ks, 1, pad, dil, True, bias, indice_key)


class SparseConv3d(_ConvBase):
    """Regular (strided / dilated) 3-D sparse convolution: every cell an active input reaches is active."""

    def __init__(self, in_channels, out_channels, kernel_size, stride=1, padding=0, dilation=1, bias=False,
                 indice_key=None):
        super().__init__(in_channels, out_channels, kernel_size, stride, padding, dilation, False, bias,
                         indice_key)


class SparseInverseConv3d(_ConvBase):
    """Inverse of the `SparseConv3d` that cached its rulebook under `indice_key`: takes a tensor on that
    layer's output cells back to its input cells (spconv / mmcv SparseInverseConv3d).  The rulebook
    is read backwards; the filter is this layer's own [kd, kh, kw, Ci, Co]."""

    inverse = True

    def __init__(self, in_channels, out_channels, kernel_size, indice_key, bias=False):
        super().__init__(in_channels, out_channels, kernel_size, 1, 0, 1, False, bias, indice_key)

    def _rulebook(self, x, wait_counts=True):
        rb = x.rulebooks.get(self.indice_key)
        assert rb is not None, "no layer has cached a rulebook under indice_key %r" % (self.indice_key,)
        assert rb.filter_space == tuple(self.kernel_size) and not rb.sub_m
        assert rb.num_act_out == x.features.shape[0], "the input does not live on the partner layer's output"
        return rb

    def _result(self, x, rb, feats):
        return SparseTensor(feats, rb.in_indices, rb.in_space, x.batch_size, x.rulebooks, distinct=rb.distinct,
                            ordered=self._order_after(x, rb))


def _unwatched():
    """Whether torch's calls are made by themselves: no tracing, no transform, no mode that sees them."""
    return not (torch.jit.is_tracing() or torch.compiler.is_compiling() or
                torch._C._len_torch_function_stack() or torch._C._len_torch_dispatch_stack() or
                torch._C._functorch.peek_interpreter_stack() is not None)


_MODULE_CALL, _CONV_FORWARD, _RELU_FORWARD = torch.nn.Module.__call__, _ConvBase.forward, torch.nn.ReLU.forward


def _plain_call(m, forward):
    """Whether calling module `m` comes to the function `forward` and nothing else."""
    return (type(m).forward is forward and type(m).__call__ is _MODULE_CALL and m._compiled_call_impl is None and
            not ("forward" in m.__dict__ or m._forward_hooks or m._forward_pre_hooks or
                 m._backward_hooks or m._backward_pre_hooks or
                 torch.nn.modules.module._has_any_global_hook()))


def _relu_in_store(conv, relu):
    """Whether the convolution `conv` can store what the module `relu` behind it would make of its result.
    Only where the layers' own calls would run and nobody could see the result in between: the library's
    layer types without a bias, exactly torch.nn.ReLU, no hook, nothing compiled or put in a method's place, no
    mode that watches torch's calls."""
    return (type(conv) in (SubMConv3d, SparseConv3d, SparseInverseConv3d) and type(relu) is torch.nn.ReLU and
            conv.bias is None and _plain_call(conv, _CONV_FORWARD) and _plain_call(relu, _RELU_FORWARD) and
            # (behind guard bands a result is a view, which autograd does not let a ReLU overwrite)
            not (relu.inplace and _guarded()) and
            _unwatched())


def embedding(table, tokens, scale=1.0):
    """scale * table[tokens] on the current device, with autograd: [*tokens.shape, channels] of the table's type.  A token
    outside the table (-1, say) gives zeros and no gradient.  With a list of rows as tokens it puts the rows of a tensor
    into another order, any of them several times or never."""
    return native().embedding(table, tokens, scale, _guarded())


class Embedding(torch.nn.Module):
    """A table of `rows` learned rows, looked up by int32 or int64 tokens and multiplied with `scale`."""

    def __init__(self, rows, channels, scale=1.0):
        super().__init__()
        self.scale = float(scale)
        self.weight = torch.nn.Parameter(torch.randn(rows, channels))

    def forward(self, tokens):
        return embedding(self.weight, tokens, self.scale)


def grouped_matmul(features, filters, group_starts):
    """Rows of groups times the filters of their groups on the current device, with autograd: features [rows, ci] in
    group order, filters [groups, ci, co], group_starts int32 [groups + 1] on the device -> [rows, co]."""
    return native().grouped_matmul(features, filters, group_starts, _guarded())


class ExpertLinear(torch.nn.Module):
    """A linear map for each expert, over rows that are ordered by expert (`expert_order`)."""

    def __init__(self, experts, in_channels, out_channels):
        super().__init__()
        bound = 1.0 / math.sqrt(in_channels)
        self.weight = torch.nn.Parameter(torch.empty(experts, in_channels, out_channels).uniform_(-bound, bound))

    def forward(self, features, group_starts):
        return grouped_matmul(features, self.weight.to(features.dtype), group_starts)


def expert_order(experts_of_rows, experts):
    """(rows, group_starts, places) of a routing [rows, choices] of integers in [0, experts): the source row of every place
    when all choices are ordered by expert (equal experts by row), int32 [rows * choices]; where each expert's
    places begin, int32 [experts + 1]; and the place of every row's choices, int32 [rows, choices].
    `embedding(features, rows)` puts rows into that order, and its gradient adds the copies of a row up again;
    `embedding(results, places)` brings the results back."""
    flat = experts_of_rows.reshape(experts_of_rows.shape[0], math.prod(experts_of_rows.shape[1:]))
    ordered, order = torch.sort(flat.reshape(-1), stable=True)
    starts = torch.searchsorted(ordered, torch.arange(experts + 1, device=flat.device, dtype=ordered.dtype), out_int32=True)
    places = torch.empty_like(order, dtype=torch.int32)
    places[order] = torch.arange(order.shape[0], device=flat.device, dtype=torch.int32)
    rows = torch.div(order, max(flat.shape[1], 1), rounding_mode="floor").to(torch.int32)
    return rows, starts, places.view(flat.shape)


class ExpertMLP(torch.nn.Module):
    """Two expert layers with SiLU in between; every row of features [rows, channels] goes to `choices` of `experts`, the
    largest of a learned linear map, and its results are added up with the softmax of their scores as weights.  One row (a
    step of a program that answers) takes the same way as a batch."""

    def __init__(self, channels, hidden, experts, choices):
        super().__init__()
        self.experts, self.choices = int(experts), int(choices)
        self.gate = torch.nn.Linear(channels, experts, bias=False)
        self.up = ExpertLinear(experts, channels, hidden)
        self.down = ExpertLinear(experts, hidden, channels)

    def forward(self, features):
        scores, chosen = torch.topk(self.gate(features.to(self.gate.weight.dtype)), self.choices, dim=1)
        rows, starts, places = expert_order(chosen, self.experts)
        hidden = torch.nn.functional.silu(self.up(embedding(features, rows), starts))
        results = embedding(self.down(hidden, starts), places)
        # (weights, products and sums in 32 bits whatever the rows' type, and one rounding)
        weights = torch.softmax(scores.float(), dim=1)
        return (results * weights.unsqueeze(2)).sum(dim=1).to(results.dtype)


def group_norm(features, weight, bias, groups, row_starts=None, eps=1e-5, activation="none"):
    """Group norm with an activation ("none", "relu" or "silu") over `features` [rows, channels] on the current device, with
    autograd.  Rows row_starts[s] to row_starts[s + 1] - 1 are sample s (int32 on the device; None: one sample of all
    rows).  `weight` and `bias` [channels] are of the features' type or float32, or None."""
    return native().group_norm(features, weight, bias, groups, row_starts, eps, ACTIVATIONS[activation], _guarded())


class GroupNormAct(torch.nn.Module):
    """Group norm over the channels of every sample, with an activation ("none", "relu", "silu") in the same pass.

    Takes a SparseTensor (the statistics are those of each sample's rows; rows that are not ordered by sample are put into
    that order and back, two passes more), or a tensor [rows, channels] with `row_starts`.
    The parameters may be float32 whatever the features are."""

    def __init__(self, groups, channels, eps=1e-5, activation="none", affine=True):
        super().__init__()
        if channels % groups != 0:
            raise ValueError("channels are a multiple of groups")
        self.groups, self.channels, self.eps = int(groups), int(channels), float(eps)
        self.activation = activation
        ACTIVATIONS[activation]
        self.weight = torch.nn.Parameter(torch.ones(channels)) if affine else None
        self.bias = torch.nn.Parameter(torch.zeros(channels)) if affine else None

    def forward(self, x, row_starts=None):
        if not isinstance(x, SparseTensor):
            return group_norm(x, self.weight, self.bias, self.groups, row_starts, self.eps, self.activation)
        order, places, starts = x._rows_of_samples()
        rows = x.features if order is None else embedding(x.features, order)
        rows = group_norm(rows, self.weight, self.bias, self.groups, starts, self.eps, self.activation)
        return x.replace_features(rows if order is None else embedding(rows, places))


class SparseSequential(torch.nn.Sequential):
    """Layers applied in order to a SparseTensor (spconv's SparseSequential): sparse convolutions
    take and return the tensor, any other module is applied to its features.

    Before the first layer runs, the rulebooks of all its convolutions are built, one after the
    other: a rulebook needs coordinates only, and the operators take its pair counts on the host.
    Built layer by layer inside the network, every wait for these drains the queue in front of the
    convolutions that follow; built up front, the host runs ahead through all convolutions and the
    device stays busy.  While they are built, only a strided layer's number of output rows is waited for (waiting
    for each rulebook's counts before the next left the device idle some 30 us a rulebook: seven of them;
    voxelizer and 11-layer encoder 865 -> 817 us); `plan` by itself waits for the counts behind the last
    rulebook, a call lets every layer take those of its own when it runs (encoder's training step 2765 -> 2743)."""

    def plan(self, x):
        built = []
        try:
            return self._plan(x, built)
        finally:
            for rb in built:
                rb.indice_num

    def _plan(self, x, built):
        cells = x
        for m in self:
            if isinstance(m, SparseSequential):
                # (a plan of the network's own is asked for as it is)
                own = type(m).plan is not _SEQUENTIAL_PLAN or "plan" in m.__dict__
                if own:  # (it may build any number)
                    for rb in built:
                        rb.indice_num
                cells = m.plan(cells) if own else m._plan(cells, built)
            elif isinstance(m, _ConvBase):
                if type(m) in (SubMConv3d, SparseConv3d) and m._plain_rulebook():
                    rb = m._rulebook(cells, wait_counts=False)
                else:
                    rb = m._rulebook(cells)
                if isinstance(rb, Rulebook) and rb not in built:
                    built.append(rb)
                    if len(built) > _PENDING:
                        built[-1 - _PENDING].indice_num
                indices, space, distinct = m._cells_after(cells, rb)
                if indices is not cells.indices:
                    # (features are not looked at while planning: a view of the right height)
                    cells = SparseTensor(indices.new_empty((indices.shape[0], 0)), indices, space,
                                         cells.batch_size, cells.rulebooks, distinct, m._order_after(cells, rb))
            elif isinstance(m, GroupNormAct) and type(m).forward is GroupNormAct.forward:
                # (what is waited for is waited for here, too)
                cells._rows_of_samples()
        return cells

    def forward(self, x):
        if type(self).plan is not _SEQUENTIAL_PLAN or "plan" in self.__dict__:
            self.plan(x)
        else:
            built = []
            try:
                self._plan(x, built)
                for rb in built:
                    if rb.counts_are_copied:
                        rb.indice_num
            except BaseException:
                for rb in built:
                    rb.indice_num
                raise
        layers = list(self)
        stored = None  # the ReLU that the convolution in front of it has already applied
        for m, following in zip(layers, layers[1:] + [None]):
            if m is stored:
                stored = None
            elif following is not None and _relu_in_store(m, following):
                # a launch and a pass over the result less each: voxelizer and 11-layer encoder 1085 -> 1007 us,
                # the encoder's training step 3231 -> 3095 us
                x, stored = m._convolve(x, relu=True), following
            elif isinstance(m, (_ConvBase, SparseSequential, GroupNormAct)):
                x = m(x)
            else:
                x = x.replace_features(m(x.features))
        return x


_SEQUENTIAL_PLAN = SparseSequential.plan


class Voxelization(torch.nn.Module):
    """Hard voxelization of one point cloud [N, F] (x, y, z first), the module mmcv puts in front of
    its sparse encoder: returns (voxels [V, max_num_points, F], coors [V, 3] as (z, y, x),
    num_points_per_voxel [V]) cut to the V voxels found (the host waits for V, not for the voxels)."""

    def __init__(self, voxel_size, point_cloud_range, max_num_points, max_voxels):
        super().__init__()
        self.register_buffer("voxel_size", torch.tensor(voxel_size, dtype=torch.float32))
        self.register_buffer("point_cloud_range", torch.tensor(point_cloud_range, dtype=torch.float32))
        self.max_num_points = int(max_num_points)
        self.max_voxels = int(max_voxels)

    def grid_shape(self):
        """(D, H, W) = cells along (z, y, x), the spatial shape of the sparse tensor."""
        r, s = self.point_cloud_range.tolist(), self.voxel_size.tolist()
        return tuple(int(math.floor((r[3 + a] - r[a]) / s[a] + 0.5)) for a in (2, 1, 0))

    @torch.no_grad()
    def forward(self, points):
        return native().voxelization_cut(_guarded(), points.contiguous().float(), self.voxel_size,
                                         self.point_cloud_range, self.max_num_points, self.max_voxels)


def mean_voxel_features(voxels, num_points_per_voxel):
    """Mean of the points of every voxel (mmcv's HardSimpleVFE): [V, max_points, F] -> [V, F]."""
    if _mean_by_library(voxels, num_points_per_voxel):
        return native().mean_voxel_points(_guarded(), voxels, num_points_per_voxel)
    return voxels.sum(dim=1) / num_points_per_voxel.clamp(min=1).to(voxels.dtype).unsqueeze(1)


def _mean_by_library(voxels, counts):
    """Whether the library's kernel takes the means (one launch in place of four; voxelizer and 11-layer encoder, 120 000
    voxels: 746 -> 713 us): what it accepts, on the current device, without a gradient to record and no mode that
    watches torch's calls.  It sums a voxel's points one after the other, torch's reduction of many points side by
    side.  us, torch / the library: 1000 voxels of 64 features, 100 points 22/8, 200 points 24/34, 400 34/66; 10 000 of 4
    features, 100 points 22/9, 128 20/16, 200 23/30; 30 of 16 features, 1000 points 26/61, 4000 35/635."""
    return (type(voxels) is torch.Tensor and type(counts) is torch.Tensor and voxels.is_cuda and counts.is_cuda and
            voxels.dtype == torch.float32 and counts.dtype == torch.int32 and voxels.dim() == 3 and counts.dim() == 1 and
            voxels.shape[1] <= 128 and counts.shape[0] == voxels.shape[0] and 0 < voxels.numel() < 1 << 31 and
            voxels.is_contiguous() and counts.is_contiguous() and not voxels.is_conj() and not voxels.is_neg() and
            voxels.device.index == torch.cuda.current_device() and counts.device == voxels.device and
            not (torch.is_grad_enabled() and voxels.requires_grad) and
            torch.autograd.forward_ad.unpack_dual(voxels).tangent is None and _unwatched())


def _ordered_by_library(coors, spatial_shape, batch_index):
    """Whether the library's kernels order these voxels (six launches in place of some 20 of a sort and the
    steps around it; voxelizer and 11-layer encoder, 120 000 voxels: 986 -> 865 us): what they accept, on
    the current device, and no mode that watches torch's calls."""
    return (coors.is_cuda and coors.dim() == 2 and coors.shape[1] == 3 and 1 < coors.shape[0] <= 1 << 20 and
            coors.device.index == torch.cuda.current_device() and len(spatial_shape) == 3 and
            all(0 < int(v) < 1 << 20 for v in spatial_shape) and -(1 << 31) <= int(batch_index) < 1 << 31 and
            _unwatched())


def sparse_tensor_from_voxels(features, coors, spatial_shape, batch_index=0, batch_size=1, order_by_cell=True):
    """SparseTensor of one cloud's voxels: indices (n, z, y, x) with n = batch_index.

    A voxelizer numbers its voxels by their first point, not by their place in the grid.  With
    `order_by_cell` (the default) the voxels are put in ascending order of their linear cell
    index here, once: every rulebook built from them, and from the outputs of the layers that
    follow, then sees rows in cell order, which mluOpGetIndicePairs resolves without its hash
    table and the convolutions read as pair lists without a row map.  The rows of the returned
    tensor are a permutation of the voxelizer's; `order_by_cell=False` keeps its order."""
    coors = coors.to(torch.int32)
    if order_by_cell and _ordered_by_library(coors, spatial_shape, batch_index):
        order, indices = native().order_voxels(_guarded(), coors.contiguous(), [int(v) for v in spatial_shape],
                                               int(batch_index))
        return SparseTensor(features[order], indices, spatial_shape, batch_size, distinct=True, ordered=True)
    if order_by_cell and coors.shape[0] > 1:
        d, h, w = (int(v) for v in spatial_shape)
        key = (coors[:, 0].to(torch.int64) * h + coors[:, 1].to(torch.int64)) * w + coors[:, 2].to(torch.int64)
        order = torch.argsort(key)
        coors = coors[order]
        features = features[order]
    n = torch.full((coors.shape[0], 1), int(batch_index), dtype=torch.int32, device=coors.device)
    # a voxelizer emits every voxel once
    return SparseTensor(features, torch.cat([n, coors], dim=1).contiguous(), spatial_shape, batch_size,
                        distinct=True, ordered=True)
