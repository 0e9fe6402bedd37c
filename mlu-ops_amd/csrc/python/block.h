// The operators of a residual block over ragged rows (mlu_op_ext.h): layer norm, the gated recurrence, rows by expert and back,
// dropout onto a residual.  Tensors in, tensors out, and their autograd nodes.  A part of native.cpp, behind training.h.

// Rows [rows, channels] of floats on the GPU, whose channels lie side by side.
inline at::Tensor floatRows(const at::Tensor &t, const char *what) {
  require(t.is_cuda() && t.dim() == 2 && t.size(1) > 0 && isFeatureType(t.scalar_type()), what);
  return channelsTogether(t);
}
inline at::Tensor floatRowsLike(const at::Tensor &t, const at::Tensor &like, const char *what) {
  require(t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.sizes() == like.sizes(), what);
  return channelsTogether(t);
}
template <typename T>
T *addressOf(const at::Tensor &t) {
  return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}

// ---- layer norm ----------------------------------------------------------------------------

struct RowNormArguments {
  at::Tensor x, weight, bias;
  int64_t rows, channels;
  mluOpDataType_t type, param_type;
  at::ScalarType param_scalar;

  RowNormArguments(const at::Tensor &features, const MaybeTensor &w, const MaybeTensor &b) {
    x = floatRows(features, "features are [rows, channels] of float32, float16 or bfloat16 on the GPU");
    rows = x.size(0);
    channels = x.size(1);
    param_scalar = x.scalar_type();
    auto param = [&](const MaybeTensor &t) {
      if (!t || !t->defined()) return at::Tensor();
      require(t->device() == x.device() && t->dim() == 1 && t->size(0) == channels &&
                  (t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat),
              "weight and bias are [channels] of the features' type or float32");
      param_scalar = t->scalar_type();
      return t->contiguous();
    };
    weight = param(w);
    bias = param(b);
    require(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
            "weight and bias have one type");
    type = dtypeCode(x.scalar_type());
    param_type = dtypeCode(param_scalar);
  }
};

std::vector<at::Tensor> layerNormForward(mluOpHandle_t handle, bool guarded, const at::Tensor &features,
                                         const MaybeTensor &weight, const MaybeTensor &bias, double eps) {
  const RowNormArguments a(features, weight, bias);
  const Buffers buffers(guarded, a.x.device());
  const at::Tensor out = buffers.output({a.rows, a.channels}, a.x.scalar_type(), "out");
  const at::Tensor mean = buffers.output({a.rows}, at::kFloat, "mean");
  const at::Tensor rstd = buffers.output({a.rows}, at::kFloat, "rstd");
  check(api.mluOpExtLayerNormForward(handle, a.type, a.x.data_ptr(), rowStride(a.x), a.rows, a.channels, a.param_type,
                                     addressOf<void>(a.weight), addressOf<void>(a.bias), static_cast<float>(eps),
                                     out.data_ptr(), addressOf<float>(mean), addressOf<float>(rstd)),
        "mluOpExtLayerNormForward");
  buffers.done("mluOpExtLayerNormForward");
  return {out, mean, rstd};
}

// (want: gradients of features, weight and bias)
std::vector<at::Tensor> layerNormBackward(mluOpHandle_t handle, bool guarded, const at::Tensor &output_grad,
                                          const at::Tensor &features, const MaybeTensor &weight, const MaybeTensor &bias,
                                          const at::Tensor &mean, const at::Tensor &rstd, bool want_weight, bool want_bias) {
  const RowNormArguments a(features, weight, bias);
  const at::Tensor dy = floatRowsLike(output_grad, a.x, "output_grad has the features' shape and type, on their GPU");
  for (const at::Tensor *t : {&mean, &rstd})
    require(t->device() == a.x.device() && t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 1 &&
                t->size(0) == a.rows,
            "mean and rstd are float32 [rows], as the forward call returned them");
  const Buffers buffers(guarded, a.x.device());
  const at::Tensor dx = buffers.output({a.rows, a.channels}, a.x.scalar_type(), "input_grad");
  const at::Tensor dw = want_weight ? buffers.output({a.channels}, a.param_scalar, "weight_grad") : at::Tensor();
  const at::Tensor db = want_bias ? buffers.output({a.channels}, a.param_scalar, "bias_grad") : at::Tensor();
  size_t bytes = 0;
  check(api.mluOpExtGetLayerNormBackwardWorkspaceSize(a.rows, a.channels, &bytes),
        "mluOpExtGetLayerNormBackwardWorkspaceSize");
  const at::Tensor ws = buffers.workspace(bytes);
  check(api.mluOpExtLayerNormBackward(handle, a.type, dy.data_ptr(), rowStride(dy), a.x.data_ptr(), rowStride(a.x), a.rows,
                                      a.channels, a.param_type, addressOf<void>(a.weight), addressOf<float>(mean),
                                      addressOf<float>(rstd), ws.data_ptr(), bytes, dx.data_ptr(), addressOf<void>(dw),
                                      addressOf<void>(db)),
        "mluOpExtLayerNormBackward");
  buffers.done("mluOpExtLayerNormBackward");
  return {dx, dw, db};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &features, const MaybeTensor &weight,
                            const MaybeTensor &bias, double eps, bool guarded) {
    StreamHandle &h = handleFor(features);
    const OperatorLock lock(h);
    const std::vector<at::Tensor> r = layerNormForward(h.handle, guarded, features, weight, bias, eps);
    ctx->save_for_backward({features, orNone(weight), orNone(bias), r[1], r[2]});
    ctx->saved_data["guarded"] = guarded;
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(5);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    StreamHandle &h = handleFor(saved[0]);
    const OperatorLock lock(h);
    const std::vector<at::Tensor> r = layerNormBackward(
        h.handle, ctx->saved_data["guarded"].toBool(), grads[0], saved[0], saved[1], saved[2], saved[3], saved[4],
        saved[1].defined() && ctx->needs_input_grad(1),
        saved[2].defined() && ctx->needs_input_grad(saved[1].defined() ? 2 : 1));
    if (ctx->needs_input_grad(0)) out[0] = r[0];
    out[1] = r[1];
    out[2] = r[2];
    return differentiableOnce(std::move(out), {grads[0], saved[0], saved[1], saved[2]});
  }
};

// ---- gated recurrence ----------------------------------------------------------------------

struct ScanArguments {
  at::Tensor x, gates, starts;
  int64_t rows, channels, samples;
  size_t carries = 0, workspace = 0;
  mluOpDataType_t type;
  mluOpExtGate_t kind;

  ScanArguments(const at::Tensor &features, const at::Tensor &g, const MaybeTensor &row_starts, int kind_code)
      : kind(static_cast<mluOpExtGate_t>(kind_code)) {
    x = near(floatRows(features, "features are [rows, channels] of float32, float16 or bfloat16 on the GPU"));
    gates = near(floatRowsLike(g, x, "gates have the features' shape and type, on their GPU"));
    rows = x.size(0);
    channels = x.size(1);
    samples = 1;
    if (row_starts && row_starts->defined()) {
      starts = startsOn(*row_starts, x, "row_starts are int32 [samples + 1] on the features' GPU");
      samples = starts.size(0) - 1;
    }
    type = dtypeCode(x.scalar_type());
    check(api.mluOpExtGetGatedScanSizes(rows, channels, samples, &carries, &workspace), "mluOpExtGetGatedScanSizes");
  }
  // (rows that lie further apart than the operator takes are laid out anew)
  static at::Tensor near(const at::Tensor &t) { return rowStride(t) > MLUOP_EXT_GATED_SCAN_MOST_STRIDE ? t.contiguous() : t; }
  // States [samples, channels], or nothing.
  at::Tensor states(const MaybeTensor &t, const char *what) const {
    if (!t || !t->defined()) return at::Tensor();
    require(t->device() == x.device() && t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == samples &&
                t->size(1) == channels,
            what);
    return t->contiguous();
  }
};

std::vector<at::Tensor> gatedScanForward(mluOpHandle_t handle, bool guarded, const at::Tensor &features,
                                         const at::Tensor &gates, const MaybeTensor &row_starts, const MaybeTensor &initial,
                                         int kind, bool reverse) {
  const ScanArguments a(features, gates, row_starts, kind);
  const at::Tensor h0 = a.states(initial, "initial states are float32 [samples, channels] on the features' GPU");
  const Buffers buffers(guarded, a.x.device());
  const at::Tensor out = buffers.output({a.rows, a.channels}, a.x.scalar_type(), "out");
  const at::Tensor final = buffers.output({a.samples, a.channels}, at::kFloat, "final");
  const at::Tensor carries = buffers.output({static_cast<int64_t>(a.carries), a.channels}, at::kFloat, "carries");
  const at::Tensor ws = buffers.workspace(a.workspace);
  check(api.mluOpExtGatedScanForward(handle, a.type, a.x.data_ptr(), rowStride(a.x), a.gates.data_ptr(), rowStride(a.gates),
                                     a.rows, a.channels, addressOf<const int32_t>(a.starts), a.samples,
                                     addressOf<const float>(h0), a.kind, reverse ? 1 : 0, ws.data_ptr(), a.workspace,
                                     out.data_ptr(), addressOf<float>(final), addressOf<float>(carries)),
        "mluOpExtGatedScanForward");
  buffers.done("mluOpExtGatedScanForward");
  return {out, final, carries};
}

std::vector<at::Tensor> gatedScanBackward(mluOpHandle_t handle, bool guarded, const at::Tensor &output_grad,
                                          const MaybeTensor &final_grad, const at::Tensor &features, const at::Tensor &gates,
                                          const at::Tensor &carries, const MaybeTensor &row_starts, int kind, bool reverse,
                                          bool want_initial) {
  const ScanArguments a(features, gates, row_starts, kind);
  const at::Tensor dh = a.near(floatRowsLike(output_grad, a.x, "output_grad has the features' shape and type, on their GPU"));
  const at::Tensor df = a.states(final_grad, "final_grad is float32 [samples, channels] on the features' GPU");
  require(carries.device() == a.x.device() && carries.scalar_type() == at::kFloat && carries.dim() == 2 &&
              carries.size(0) == static_cast<int64_t>(a.carries) && carries.size(1) == a.channels && carries.is_contiguous(),
          "carries are what the forward call returned");
  const Buffers buffers(guarded, a.x.device());
  const at::Tensor dx = buffers.output({a.rows, a.channels}, a.x.scalar_type(), "features_grad");
  const at::Tensor dg = buffers.output({a.rows, a.channels}, a.x.scalar_type(), "gates_grad");
  const at::Tensor di = want_initial ? buffers.output({a.samples, a.channels}, at::kFloat, "initial_grad") : at::Tensor();
  const at::Tensor ws = buffers.workspace(a.workspace);
  check(api.mluOpExtGatedScanBackward(handle, a.type, dh.data_ptr(), rowStride(dh), addressOf<const float>(df),
                                      a.x.data_ptr(), rowStride(a.x), a.gates.data_ptr(), rowStride(a.gates), a.rows,
                                      a.channels, addressOf<const int32_t>(a.starts), a.samples,
                                      addressOf<const float>(carries), a.kind, reverse ? 1 : 0, ws.data_ptr(), a.workspace,
                                      dx.data_ptr(), dg.data_ptr(), addressOf<float>(di)),
        "mluOpExtGatedScanBackward");
  buffers.done("mluOpExtGatedScanBackward");
  return {dx, dg, di};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const at::Tensor &features,
                                                const at::Tensor &gates, const MaybeTensor &initial,
                                                const MaybeTensor &row_starts, int64_t kind, bool reverse, bool guarded) {
    StreamHandle &h = handleFor(features);
    const OperatorLock lock(h);
    const std::vector<at::Tensor> r = gatedScanForward(h.handle, guarded, features, gates, row_starts, initial,
                                                       static_cast<int>(kind), reverse);
    ctx->save_for_backward({features, gates, orNone(initial), orNone(row_starts), r[2]});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["guarded"] = guarded;
    ctx->set_materialize_grads(false);
    return {r[0], r[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(7);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    StreamHandle &h = handleFor(saved[0]);
    const OperatorLock lock(h);
    const std::vector<at::Tensor> r = gatedScanBackward(
        h.handle, ctx->saved_data["guarded"].toBool(), grads[0].defined() ? grads[0] : at::zeros_like(saved[0]), grads[1],
        saved[0], saved[1], saved[4], saved[3], static_cast<int>(ctx->saved_data["kind"].toInt()),
        ctx->saved_data["reverse"].toBool(), saved[2].defined() && ctx->needs_input_grad(2));
    if (ctx->needs_input_grad(0)) out[0] = r[0];
    if (ctx->needs_input_grad(1)) out[1] = r[1];
    out[2] = r[2];
    return differentiableOnce(std::move(out), {grads[0], grads[1], saved[0], saved[1], saved[2]});
  }
};

// ---- rows by expert and back ---------------------------------------------------------------

std::vector<at::Tensor> expertOrder(mluOpHandle_t handle, bool guarded, const at::Tensor &experts_of_rows, int64_t experts) {
  require(experts_of_rows.is_cuda() && experts_of_rows.dim() == 2 && experts_of_rows.size(1) > 0,
          "experts of rows are [rows, choices] on the GPU");
  const mluOpDataType_t type = tokenType(experts_of_rows);
  const at::Tensor chosen = experts_of_rows.contiguous();
  const int64_t rows = chosen.size(0), choices = chosen.size(1);
  size_t bytes = 0;
  check(api.mluOpExtGetExpertOrderWorkspaceSize(rows, choices, experts, &bytes), "mluOpExtGetExpertOrderWorkspaceSize");
  const Buffers buffers(guarded, chosen.device());
  const at::Tensor ordered = buffers.output({rows * choices}, at::kInt, "ordered_rows");
  const at::Tensor starts = buffers.output({experts + 1}, at::kInt, "group_starts");
  const at::Tensor places = buffers.output({rows, choices}, at::kInt, "places");
  const at::Tensor ws = buffers.workspace(bytes);
  check(api.mluOpExtExpertOrder(handle, type, chosen.data_ptr(), rows, choices, experts, ws.data_ptr(), bytes,
                                addressOf<int32_t>(ordered), addressOf<int32_t>(starts), addressOf<int32_t>(places)),
        "mluOpExtExpertOrder");
  buffers.done("mluOpExtExpertOrder");
  return {ordered, starts, places};
}

inline at::Tensor placesOn(const at::Tensor &t, const at::Tensor &like) {
  require(t.device() == like.device() && t.dim() == 2 && t.size(1) > 0 && t.scalar_type() == at::kInt,
          "places are int32 [rows, choices] on the rows' GPU");
  return t.contiguous();
}

at::Tensor expertDispatch(mluOpHandle_t handle, bool guarded, const at::Tensor &features, const at::Tensor &places,
                          const at::Tensor &group_starts) {
  const at::Tensor x = floatRows(features, "features are [rows, channels] of float32, float16 or bfloat16 on the GPU");
  const at::Tensor to = placesOn(places, x);
  require(to.size(0) == x.size(0), "every row has its places");
  const at::Tensor starts = startsOn(group_starts, x, "group_starts are int32 [experts + 1] on the features' GPU");
  const Buffers buffers(guarded, x.device());
  const at::Tensor out = buffers.output({to.numel(), x.size(1)}, x.scalar_type(), "out");
  check(api.mluOpExtExpertDispatch(handle, dtypeCode(x.scalar_type()), x.data_ptr(), rowStride(x), x.size(0), x.size(1),
                                   to.size(1), addressOf<const int32_t>(to), addressOf<const int32_t>(starts),
                                   starts.size(0) - 1, out.data_ptr()),
        "mluOpExtExpertDispatch");
  buffers.done("mluOpExtExpertDispatch");
  return out;
}

// Weights of the choices, or nothing; the code of their type.
inline at::Tensor weightsOn(const MaybeTensor &t, const at::Tensor &rows, const at::Tensor &places, mluOpDataType_t *type) {
  *type = dtypeCode(rows.scalar_type());
  if (!t || !t->defined()) return at::Tensor();
  require(t->device() == rows.device() && t->sizes() == places.sizes() &&
              (t->scalar_type() == rows.scalar_type() || t->scalar_type() == at::kFloat),
          "weights are [rows, choices] of the results' type or float32");
  *type = dtypeCode(t->scalar_type());
  return t->contiguous();
}

at::Tensor expertCombine(mluOpHandle_t handle, bool guarded, const at::Tensor &results, const at::Tensor &places,
                         const MaybeTensor &weights) {
  const at::Tensor y = floatRows(results, "results are [rows, channels] of float32, float16 or bfloat16 on the GPU");
  const at::Tensor from = placesOn(places, y);
  require(y.size(0) == from.numel(), "there are as many results as places");
  mluOpDataType_t weight_type;
  const at::Tensor w = weightsOn(weights, y, from, &weight_type);
  const Buffers buffers(guarded, y.device());
  const at::Tensor out = buffers.output({from.size(0), y.size(1)}, y.scalar_type(), "out");
  check(api.mluOpExtExpertCombine(handle, dtypeCode(y.scalar_type()), y.data_ptr(), rowStride(y), from.size(0), y.size(1),
                                  from.size(1), addressOf<const int32_t>(from), weight_type, addressOf<void>(w),
                                  out.data_ptr()),
        "mluOpExtExpertCombine");
  buffers.done("mluOpExtExpertCombine");
  return out;
}

std::vector<at::Tensor> expertCombineBackward(mluOpHandle_t handle, bool guarded, const at::Tensor &output_grad,
                                              const at::Tensor &results, const at::Tensor &places,
                                              const MaybeTensor &weights, const at::Tensor &group_starts, bool want_weights) {
  const at::Tensor y = floatRows(results, "results are [rows, channels] of float32, float16 or bfloat16 on the GPU");
  const at::Tensor from = placesOn(places, y);
  require(y.size(0) == from.numel(), "there are as many results as places");
  require(output_grad.device() == y.device() && output_grad.scalar_type() == y.scalar_type() && output_grad.dim() == 2 &&
              output_grad.size(0) == from.size(0) && output_grad.size(1) == y.size(1),
          "output_grad is [rows, channels] of the results' type, on their GPU");
  const at::Tensor dout = channelsTogether(output_grad);
  const at::Tensor starts = startsOn(group_starts, y, "group_starts are int32 [experts + 1] on the results' GPU");
  mluOpDataType_t weight_type;
  const at::Tensor w = weightsOn(weights, y, from, &weight_type);
  const Buffers buffers(guarded, y.device());
  const at::Tensor dy = buffers.output({y.size(0), y.size(1)}, y.scalar_type(), "results_grad");
  const at::Tensor dw =
      want_weights && w.defined() ? buffers.output({from.size(0), from.size(1)}, w.scalar_type(), "weights_grad") : at::Tensor();
  check(api.mluOpExtExpertCombineBackward(handle, dtypeCode(y.scalar_type()), dout.data_ptr(), rowStride(dout), y.data_ptr(),
                                          rowStride(y), from.size(0), y.size(1), from.size(1),
                                          addressOf<const int32_t>(from), addressOf<const int32_t>(starts),
                                          starts.size(0) - 1, weight_type, addressOf<void>(w), dy.data_ptr(),
                                          addressOf<void>(dw)),
        "mluOpExtExpertCombineBackward");
  buffers.done("mluOpExtExpertCombineBackward");
  return {dy, dw};
}

struct ExpertDispatch : torch::autograd::Function<ExpertDispatch> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &features, const at::Tensor &places,
                            const at::Tensor &group_starts, bool guarded) {
    StreamHandle &h = handleFor(features);
    const OperatorLock lock(h);
    ctx->save_for_backward({places});
    ctx->saved_data["guarded"] = guarded;
    return expertDispatch(h.handle, guarded, features, places, group_starts);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(4);
    if (!grads[0].defined() || !ctx->needs_input_grad(0)) return out;
    const auto saved = ctx->get_saved_variables();
    StreamHandle &h = handleFor(grads[0]);
    const OperatorLock lock(h);
    out[0] = expertCombine(h.handle, ctx->saved_data["guarded"].toBool(), grads[0], saved[0], std::nullopt);
    return differentiableOnce(std::move(out), {grads[0]});
  }
};

struct ExpertCombine : torch::autograd::Function<ExpertCombine> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &results, const MaybeTensor &weights,
                            const at::Tensor &places, const at::Tensor &group_starts, bool guarded) {
    StreamHandle &h = handleFor(results);
    const OperatorLock lock(h);
    ctx->save_for_backward({results, orNone(weights), places, group_starts});
    ctx->saved_data["guarded"] = guarded;
    return expertCombine(h.handle, guarded, results, places, weights);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(5);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    StreamHandle &h = handleFor(saved[0]);
    const OperatorLock lock(h);
    const std::vector<at::Tensor> r =
        expertCombineBackward(h.handle, ctx->saved_data["guarded"].toBool(), grads[0], saved[0], saved[2], saved[1], saved[3],
                              saved[1].defined() && ctx->needs_input_grad(1));
    if (ctx->needs_input_grad(0)) out[0] = r[0];
    out[1] = r[1];
    return differentiableOnce(std::move(out), {grads[0], saved[0], saved[1]});
  }
};

// ---- dropout -------------------------------------------------------------------------------

at::Tensor dropoutAdd(mluOpHandle_t handle, bool guarded, const at::Tensor &features, const MaybeTensor &residual, double p,
                      const at::Tensor &state) {
  require(features.is_cuda() && isFeatureType(features.scalar_type()),
          "features are float32, float16 or bfloat16 on the GPU");
  require(state.device() == features.device() && state.scalar_type() == at::kLong && state.dim() == 1 && state.size(0) == 2,
          "state is int64 [2] on the features' GPU: a seed and the number of the call");
  require(p >= 0.0 && p <= 1.0, "p lies in [0, 1]");
  const at::Tensor x = features.contiguous(), seed = state.contiguous();
  at::Tensor r;
  if (residual && residual->defined()) {
    require(residual->device() == x.device() && residual->scalar_type() == x.scalar_type() && residual->sizes() == x.sizes(),
            "residual has the features' shape and type, on their GPU");
    r = residual->contiguous();
  }
  const Buffers buffers(guarded, x.device());
  const at::Tensor out = buffers.output(x.sizes(), x.scalar_type(), "out");
  check(api.mluOpExtDropoutAdd(handle, dtypeCode(x.scalar_type()), x.data_ptr(), addressOf<void>(r), x.numel(), p,
                               addressOf<const int64_t>(seed), out.data_ptr()),
        "mluOpExtDropoutAdd");
  buffers.done("mluOpExtDropoutAdd");
  return out;
}

struct DropoutAdd : torch::autograd::Function<DropoutAdd> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &features, const MaybeTensor &residual,
                            double p, const at::Tensor &state, bool guarded) {
    StreamHandle &h = handleFor(features);
    const OperatorLock lock(h);
    ctx->save_for_backward({state});
    ctx->saved_data["p"] = p;
    ctx->saved_data["added"] = residual && residual->defined();
    ctx->saved_data["guarded"] = guarded;
    return dropoutAdd(h.handle, guarded, features, residual, p, state);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(5);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    if (ctx->needs_input_grad(0)) {
      StreamHandle &h = handleFor(grads[0]);
      const OperatorLock lock(h);
      out[0] = dropoutAdd(h.handle, ctx->saved_data["guarded"].toBool(), grads[0], std::nullopt,
                          ctx->saved_data["p"].toDouble(), saved[0]);
    }
    if (ctx->saved_data["added"].toBool() && ctx->needs_input_grad(1)) out[1] = grads[0];
    return differentiableOnce(std::move(out), {grads[0]});
  }
};

void defineBlock(py::module_ &m) {
  using NoGil = py::gil_scoped_release;
  auto optional = [](const at::Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
  m.def("layer_norm_forward", [](uintptr_t handle, bool guarded, const at::Tensor &features, const MaybeTensor &weight,
                                 const MaybeTensor &bias, double eps) {
    std::vector<at::Tensor> r;
    {
      NoGil released;
      const OperatorLock lock(asHandle(handle));
      r = layerNormForward(asHandle(handle), guarded, features, weight, bias, eps);
    }
    return py::make_tuple(r[0], r[1], r[2]);
  });
  m.def("layer_norm_backward", [](uintptr_t handle, bool guarded, const at::Tensor &output_grad, const at::Tensor &features,
                                  const MaybeTensor &weight, const MaybeTensor &bias, const at::Tensor &mean,
                                  const at::Tensor &rstd) {
    std::vector<at::Tensor> r;
    {
      NoGil released;
      const OperatorLock lock(asHandle(handle));
      r = layerNormBackward(asHandle(handle), guarded, output_grad, features, weight, bias, mean, rstd, true, true);
    }
    return py::make_tuple(r[0], r[1], r[2]);
  });
  m.def("layer_norm", [](const at::Tensor &features, const MaybeTensor &weight, const MaybeTensor &bias, double eps,
                         bool guarded) {
    NoGil released;
    return LayerNorm::apply(features, weight, bias, eps, guarded);
  });
  m.def("gated_scan_forward", [](uintptr_t handle, bool guarded, const at::Tensor &features, const at::Tensor &gates,
                                 const MaybeTensor &row_starts, const MaybeTensor &initial, int kind, bool reverse) {
    std::vector<at::Tensor> r;
    {
      NoGil released;
      const OperatorLock lock(asHandle(handle));
      r = gatedScanForward(asHandle(handle), guarded, features, gates, row_starts, initial, kind, reverse);
    }
    return py::make_tuple(r[0], r[1], r[2]);
  });
  m.def("gated_scan_backward",
        [](uintptr_t handle, bool guarded, const at::Tensor &output_grad, const MaybeTensor &final_grad,
           const at::Tensor &features, const at::Tensor &gates, const at::Tensor &carries, const MaybeTensor &row_starts,
           int kind, bool reverse) {
          std::vector<at::Tensor> r;
          {
            NoGil released;
            const OperatorLock lock(asHandle(handle));
            r = gatedScanBackward(asHandle(handle), guarded, output_grad, final_grad, features, gates, carries, row_starts,
                                  kind, reverse, true);
          }
          return py::make_tuple(r[0], r[1], r[2]);
        });
  m.def("gated_scan", [](const at::Tensor &features, const at::Tensor &gates, const MaybeTensor &row_starts,
                         const MaybeTensor &initial, int64_t kind, bool reverse, bool guarded) {
    torch::autograd::variable_list r;
    {
      NoGil released;
      r = GatedScan::apply(features, gates, initial, row_starts, kind, reverse, guarded);
    }
    return py::make_tuple(r[0], r[1]);
  });
  m.def("expert_order", [](uintptr_t handle, bool guarded, const at::Tensor &experts_of_rows, int64_t experts) {
    std::vector<at::Tensor> r;
    {
      NoGil released;
      const OperatorLock lock(asHandle(handle));
      r = expertOrder(asHandle(handle), guarded, experts_of_rows, experts);
    }
    return py::make_tuple(r[0], r[1], r[2]);
  });
  m.def("expert_dispatch_rows", [](uintptr_t handle, bool guarded, const at::Tensor &features, const at::Tensor &places,
                                   const at::Tensor &group_starts) {
    NoGil released;
    const OperatorLock lock(asHandle(handle));
    return expertDispatch(asHandle(handle), guarded, features, places, group_starts);
  });
  m.def("expert_combine_rows", [](uintptr_t handle, bool guarded, const at::Tensor &results, const at::Tensor &places,
                                  const MaybeTensor &weights) {
    NoGil released;
    const OperatorLock lock(asHandle(handle));
    return expertCombine(asHandle(handle), guarded, results, places, weights);
  });
  m.def("expert_combine_backward",
        [optional](uintptr_t handle, bool guarded, const at::Tensor &output_grad, const at::Tensor &results,
                   const at::Tensor &places, const MaybeTensor &weights, const at::Tensor &group_starts) {
          std::vector<at::Tensor> r;
          {
            NoGil released;
            const OperatorLock lock(asHandle(handle));
            r = expertCombineBackward(asHandle(handle), guarded, output_grad, results, places, weights, group_starts, true);
          }
          return py::make_tuple(r[0], optional(r[1]));
        });
  m.def("expert_dispatch", [](const at::Tensor &features, const at::Tensor &places, const at::Tensor &group_starts,
                              bool guarded) {
    NoGil released;
    return ExpertDispatch::apply(features, places, group_starts, guarded);
  });
  m.def("expert_combine", [](const at::Tensor &results, const MaybeTensor &weights, const at::Tensor &places,
                             const at::Tensor &group_starts, bool guarded) {
    NoGil released;
    return ExpertCombine::apply(results, weights, places, group_starts, guarded);
  });
  m.def("dropout_add_rows", [](uintptr_t handle, bool guarded, const at::Tensor &features, const MaybeTensor &residual,
                               double p, const at::Tensor &state) {
    NoGil released;
    const OperatorLock lock(asHandle(handle));
    return dropoutAdd(asHandle(handle), guarded, features, residual, p, state);
  });
  m.def("dropout_add", [](const at::Tensor &features, const MaybeTensor &residual, double p, const at::Tensor &state,
                          bool guarded) {
    NoGil released;
    return DropoutAdd::apply(features, residual, p, state, guarded);
  });
}
