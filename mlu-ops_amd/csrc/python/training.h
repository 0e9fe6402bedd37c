// The operators of the rest of a training step (mlu_op_ext.h): tensors in, tensors out, and their autograd nodes.  A part of
// native.cpp, included inside its namespace.

// What these operators take is checked here, since the C API sees addresses and sizes only.
inline void require(bool met, const char *what) {
  if (!met) throw py::value_error(what);
}

inline bool isFeatureType(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

// The tensors of an AdamW step: checked once and kept, so that a step looks at its gradients only.
class AdamWTensors {
 public:
  using Tensors = std::vector<at::Tensor>;
  AdamWTensors(Tensors params, Tensors exp_avgs, Tensors exp_avg_sqs, std::optional<Tensors> masters,
               std::optional<Tensors> exp_avg_scales, std::optional<Tensors> exp_avg_sq_scales) {
    const size_t n = params.size();
    require(exp_avgs.size() == n && exp_avg_sqs.size() == n && (!masters || masters->size() == n),
            "params, states and masters are lists of one length");
    require(exp_avg_scales.has_value() == exp_avg_sq_scales.has_value(), "both states have scales or neither");
    eight_ = exp_avg_scales.has_value();
    require(!eight_ || (exp_avg_scales->size() == n && exp_avg_sq_scales->size() == n),
            "scales are lists of the params' length");
    raw_.resize(n);
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor &p = params[i];
      const int64_t count = p.numel();
      if (i == 0) {
        type_ = p.scalar_type();
        device_ = p.device();
        require(device_.is_cuda(), "params are on the GPU");
        require(isFeatureType(type_), "params are float32, float16 or bfloat16");
        require(!masters || type_ != at::kFloat, "float32 params have no masters");
      }
      require(p.scalar_type() == type_, "params have one type");
      require(p.device() == device_ && p.is_non_overlapping_and_dense(), "params are dense, on one device");
      auto state = [&](const at::Tensor &t, int64_t length) {
        require(t.device() == device_ && t.numel() == length, "states have their parameter's device and size");
        // (an element's state lies where the element does)
        require(t.strides() == p.strides() || (p.is_contiguous() && t.is_contiguous()),
                "states lie in memory as their parameter does");
        if (!eight_) return;
        require(t.scalar_type() == at::kByte || t.scalar_type() == at::kFloat8_e4m3fn,
                "8-bit states are float8_e4m3fn or uint8");
      };
      state(exp_avgs[i], count);
      state(exp_avg_sqs[i], count);
      require(eight_ || (exp_avgs[i].scalar_type() == at::kFloat && exp_avg_sqs[i].scalar_type() == at::kFloat),
              "states without scales are float32");
      mluOpExtAdamWTensor_t &r = raw_[i];
      r = {p.data_ptr(), nullptr, exp_avgs[i].data_ptr(), exp_avg_sqs[i].data_ptr(), nullptr, nullptr, nullptr, count};
      if (masters) {
        const at::Tensor &m = (*masters)[i];
        require(m.scalar_type() == at::kFloat && m.device() == device_ && m.numel() == count &&
                    (m.strides() == p.strides() || (p.is_contiguous() && m.is_contiguous())),
                "masters are float32 and lie as their parameter does");
        r.master = static_cast<float *>(m.data_ptr());
      }
      if (eight_) {
        const int64_t blocks = (count + MLUOP_EXT_ADAMW_BLOCK - 1) / MLUOP_EXT_ADAMW_BLOCK;
        auto scale = [&](const at::Tensor &t) {
          require(t.scalar_type() == at::kFloat && t.device() == device_ && t.numel() == blocks && t.is_contiguous(),
                  "scales are float32, one for each 256 elements");
          return static_cast<float *>(t.data_ptr());
        };
        r.exp_avg_scale = scale((*exp_avg_scales)[i]);
        r.exp_avg_sq_scale = scale((*exp_avg_sq_scales)[i]);
      }
    }
    params_ = std::move(params);
    for (auto *list : {&exp_avgs, &exp_avg_sqs}) kept_.insert(kept_.end(), list->begin(), list->end());
    for (auto *list : {&masters, &exp_avg_scales, &exp_avg_sq_scales})
      if (*list) kept_.insert(kept_.end(), (*list)->begin(), (*list)->end());
  }

  // Gradients: one for each param, undefined (None) where a param has none and is left alone.
  void step(mluOpHandle_t handle, const std::vector<std::optional<at::Tensor>> &grads, int64_t step, double lr,
            double beta1, double beta2, double eps, double weight_decay, double grad_scale) {
    require(grads.size() == raw_.size(), "a gradient (or None) for each param");
    std::vector<mluOpExtAdamWTensor_t> own, wide;  // gradients of the params' type, and float32 ones
    own.reserve(raw_.size());
    std::vector<at::Tensor> laid_out;  // alive until the launches are enqueued
    for (size_t i = 0; i < raw_.size(); ++i) {
      if (!grads[i] || !grads[i]->defined()) continue;
      at::Tensor g = *grads[i];
      const at::Tensor &p = params_[i];
      require(g.device() == device_ && g.numel() == raw_[i].count, "gradients have their parameter's device and size");
      require(g.scalar_type() == type_ || g.scalar_type() == at::kFloat,
              "gradients are of the params' type or float32");
      if (g.strides() != p.strides() && !(p.is_contiguous() && g.is_contiguous())) {
        require(g.sizes() == p.sizes(), "gradients have their parameter's shape");
        at::Tensor same = at::empty_strided(p.sizes(), p.strides(), g.options());
        same.copy_(g);
        laid_out.push_back(same);
        g = same;
      }
      mluOpExtAdamWTensor_t r = raw_[i];
      r.grad = g.data_ptr();
      (g.scalar_type() == type_ ? own : wide).push_back(r);
    }
    auto run = [&](const std::vector<mluOpExtAdamWTensor_t> &list, mluOpDataType_t grad_type) {
      if (list.empty()) return;
      check(api.mluOpExtAdamWStep(handle, list.data(), static_cast<int>(list.size()), dtypeCode(type_), grad_type,
                                  eight_ ? MLUOP_DTYPE_UINT8 : MLUOP_DTYPE_FLOAT, step, lr, beta1, beta2, eps,
                                  weight_decay, grad_scale),
            "mluOpExtAdamWStep");
    };
    run(own, own.empty() ? MLUOP_DTYPE_FLOAT : dtypeCode(type_));
    run(wide, MLUOP_DTYPE_FLOAT);
    // Autograd's record of what has been written: a backward pass that needs a value from before the step says so.
    // (A tensor that was made without a record has none; states are no part of a graph.)
    for (size_t i = 0; i < raw_.size(); ++i)
      if (grads[i] && grads[i]->defined() && !params_[i].is_inference()) params_[i].unsafeGetTensorImpl()->bump_version();
  }

 private:
  std::vector<mluOpExtAdamWTensor_t> raw_;
  Tensors params_, kept_;
  at::ScalarType type_ = at::kFloat;
  at::Device device_ = at::kCPU;
  bool eight_ = false;
};

// ---- group norm ----------------------------------------------------------------------------

// A tensor of floats on the GPU of `like`, laid out row by row.
inline at::Tensor rowsOn(const at::Tensor &t, const at::Tensor &like, int64_t dim, const char *what) {
  require(t.device() == like.device() && t.device().is_cuda() && t.dim() == dim && t.scalar_type() == like.scalar_type(),
          what);
  return t.contiguous();
}

// int32 starts of segments, one more than there are.
inline at::Tensor startsOn(const at::Tensor &t, const at::Tensor &like, const char *what) {
  require(t.device() == like.device() && t.dim() == 1 && t.size(0) >= 2 && t.scalar_type() == at::kInt, what);
  return t.contiguous();
}

using MaybeTensor = std::optional<at::Tensor>;

struct NormArguments {
  at::Tensor x, weight, bias, starts;
  int64_t rows, channels, samples;
  mluOpDataType_t type, param_type;

  NormArguments(const at::Tensor &features, const MaybeTensor &w, const MaybeTensor &b, int64_t groups,
                const MaybeTensor &row_starts) {
    require(features.is_cuda() && features.dim() == 2 && isFeatureType(features.scalar_type()),
            "features are [rows, channels] of float32, float16 or bfloat16 on the GPU");
    x = features.contiguous();
    rows = x.size(0);
    channels = x.size(1);
    require(groups > 0 && channels > 0 && channels % groups == 0, "channels are a multiple of groups");
    type = dtypeCode(x.scalar_type());
    param_type = type;
    auto param = [&](const MaybeTensor &t) {
      if (!t || !t->defined()) return at::Tensor();
      require(t->device() == x.device() && t->dim() == 1 && t->size(0) == channels &&
                  (t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat),
              "weight and bias are [channels] of the features' type or float32");
      param_type = dtypeCode(t->scalar_type());
      return t->contiguous();
    };
    weight = param(w);
    bias = param(b);
    require(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
            "weight and bias have one type");
    samples = 1;
    if (row_starts && row_starts->defined()) {
      starts = startsOn(*row_starts, x, "row_starts are int32 [samples + 1] on the features' GPU");
      samples = starts.size(0) - 1;
    }
  }
  static void *at(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
  at::Tensor workspace(const Buffers &buffers, int64_t groups, size_t *bytes) const {
    check(api.mluOpExtGetGroupNormWorkspaceSize(rows, channels, groups, samples, bytes),
          "mluOpExtGetGroupNormWorkspaceSize");
    return buffers.workspace(*bytes);
  }
};

std::vector<at::Tensor> groupNormForward(mluOpHandle_t handle, bool guarded, const at::Tensor &features,
                                         const MaybeTensor &weight, const MaybeTensor &bias, int64_t groups,
                                         const MaybeTensor &row_starts, double eps, int activation) {
  const NormArguments a(features, weight, bias, groups, row_starts);
  const Buffers buffers(guarded, a.x.device());
  const at::Tensor out = buffers.output({a.rows, a.channels}, a.x.scalar_type(), "out");
  const at::Tensor mean = buffers.output({a.samples, groups}, at::kFloat, "mean");
  const at::Tensor rstd = buffers.output({a.samples, groups}, at::kFloat, "rstd");
  size_t bytes = 0;
  const at::Tensor ws = a.workspace(buffers, groups, &bytes);
  check(api.mluOpExtGroupNormForward(handle, a.type, a.x.data_ptr(), a.rows, a.channels, groups,
                                     static_cast<const int32_t *>(a.at(a.starts)), a.samples, a.param_type,
                                     a.at(a.weight), a.at(a.bias), static_cast<float>(eps),
                                     static_cast<mluOpExtActivation_t>(activation), ws.data_ptr(), bytes,
                                     out.data_ptr(), static_cast<float *>(mean.data_ptr()),
                                     static_cast<float *>(rstd.data_ptr())),
        "mluOpExtGroupNormForward");
  buffers.done("mluOpExtGroupNormForward");
  return {out, mean, rstd};
}

std::vector<at::Tensor> groupNormBackward(mluOpHandle_t handle, bool guarded, const at::Tensor &output_grad,
                                          const at::Tensor &features, const MaybeTensor &weight,
                                          const MaybeTensor &bias, const at::Tensor &mean, const at::Tensor &rstd,
                                          int64_t groups, const MaybeTensor &row_starts, int activation) {
  const NormArguments a(features, weight, bias, groups, row_starts);
  const Buffers buffers(guarded, a.x.device());
  const at::Tensor dy = rowsOn(output_grad, a.x, 2, "output_grad is of the features' type, on their GPU");
  require(dy.sizes() == a.x.sizes(), "output_grad has the features' shape");
  for (const at::Tensor *t : {&mean, &rstd})
    require(t->device() == a.x.device() && t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 2 &&
                t->size(0) == a.samples && t->size(1) == groups,
            "mean and rstd are float32 [samples, groups], as the forward call returned them");
  const at::ScalarType param = a.weight.defined() ? a.weight.scalar_type()
                               : a.bias.defined() ? a.bias.scalar_type()
                                                  : a.x.scalar_type();
  const at::Tensor dx = buffers.output({a.rows, a.channels}, a.x.scalar_type(), "input_grad");
  const at::Tensor dw = buffers.output({a.channels}, param, "weight_grad");
  const at::Tensor db = buffers.output({a.channels}, param, "bias_grad");
  size_t bytes = 0;
  const at::Tensor ws = a.workspace(buffers, groups, &bytes);
  check(api.mluOpExtGroupNormBackward(handle, a.type, dy.data_ptr(), a.x.data_ptr(), a.rows, a.channels, groups,
                                      static_cast<const int32_t *>(a.at(a.starts)), a.samples, a.param_type,
                                      a.at(a.weight), a.at(a.bias), static_cast<const float *>(mean.data_ptr()),
                                      static_cast<const float *>(rstd.data_ptr()),
                                      static_cast<mluOpExtActivation_t>(activation), ws.data_ptr(), bytes,
                                      dx.data_ptr(), dw.data_ptr(), db.data_ptr()),
        "mluOpExtGroupNormBackward");
  buffers.done("mluOpExtGroupNormBackward");
  return {dx, dw, db};
}

// The handle of the current stream, for tensors of the current device.
StreamHandle &handleFor(const at::Tensor &t) {
  require(t.is_cuda() && t.device().index() == c10::hip::current_device(), "tensors lie on the current GPU");
  return streamHandle();
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &features, const at::Tensor &weight,
                            const at::Tensor &bias, int64_t groups, const MaybeTensor &row_starts, double eps,
                            int64_t activation, bool guarded) {
    StreamHandle &h = handleFor(features);
    const OperatorLock lock(h);
    const std::vector<at::Tensor> r = groupNormForward(h.handle, guarded, features, weight, bias, groups, row_starts, eps,
                                                       static_cast<int>(activation));
    ctx->save_for_backward({features, weight, bias, row_starts ? *row_starts : at::Tensor(), r[1], r[2]});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["guarded"] = guarded;
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(8);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    StreamHandle &h = handleFor(saved[0]);
    const OperatorLock lock(h);
    const std::vector<at::Tensor> r = groupNormBackward(
        h.handle, ctx->saved_data["guarded"].toBool(), grads[0], saved[0], saved[1], saved[2], saved[4], saved[5],
        ctx->saved_data["groups"].toInt(), saved[3], static_cast<int>(ctx->saved_data["activation"].toInt()));
    if (ctx->needs_input_grad(0)) out[0] = r[0];
    if (saved[1].defined() && ctx->needs_input_grad(1)) out[1] = r[1];
    if (saved[2].defined() && ctx->needs_input_grad(2)) out[2] = r[2];
    return differentiableOnce(std::move(out), {grads[0], saved[0], saved[1], saved[2]});
  }
};

// ---- embedding -----------------------------------------------------------------------------

// A tensor [rows, channels] whose channels lie side by side: as it is, or laid out anew.
inline at::Tensor channelsTogether(const at::Tensor &t) {
  const bool together = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
  return together ? t : t.contiguous();
}
inline int64_t rowStride(const at::Tensor &t) { return t.size(0) <= 1 ? std::max<int64_t>(t.size(1), 1) : t.stride(0); }

inline mluOpDataType_t tokenType(const at::Tensor &tokens) {
  require(tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong, "tokens are int32 or int64");
  return tokens.scalar_type() == at::kInt ? MLUOP_DTYPE_INT32 : MLUOP_DTYPE_INT64;
}

at::Tensor embeddingForward(mluOpHandle_t handle, bool guarded, const at::Tensor &table, const at::Tensor &tokens,
                            double scale) {
  require(table.is_cuda() && table.dim() == 2 && isFeatureType(table.scalar_type()),
          "a table is [rows, channels] of float32, float16 or bfloat16 on the GPU");
  require(tokens.device() == table.device(), "tokens lie on the table's GPU");
  const mluOpDataType_t token_type = tokenType(tokens);
  const at::Tensor w = channelsTogether(table), t = tokens.contiguous();
  const Buffers buffers(guarded, w.device());
  std::vector<int64_t> shape = t.sizes().vec();
  shape.push_back(w.size(1));
  const at::Tensor out = buffers.output(shape, w.scalar_type(), "out");
  check(api.mluOpExtEmbeddingForward(handle, dtypeCode(w.scalar_type()), w.data_ptr(), w.size(0), w.size(1), rowStride(w),
                                     token_type, t.data_ptr(), t.numel(), static_cast<float>(scale), out.data_ptr()),
        "mluOpExtEmbeddingForward");
  buffers.done("mluOpExtEmbeddingForward");
  return out;
}

at::Tensor embeddingBackward(mluOpHandle_t handle, bool guarded, const at::Tensor &output_grad, const at::Tensor &tokens,
                             int64_t rows, double scale) {
  require(output_grad.is_cuda() && output_grad.dim() >= 1 && isFeatureType(output_grad.scalar_type()),
          "output_grad is float32, float16 or bfloat16 on the GPU");
  require(tokens.device() == output_grad.device(), "tokens lie on the gradient's GPU");
  require(output_grad.sizes().slice(0, output_grad.dim() - 1) == tokens.sizes(), "output_grad is [*tokens.shape, channels]");
  const mluOpDataType_t token_type = tokenType(tokens);
  const int64_t channels = output_grad.size(-1), n = tokens.numel();
  const at::Tensor g = output_grad.dim() == 2 ? channelsTogether(output_grad) : output_grad.contiguous().view({n, channels});
  const at::Tensor t = tokens.contiguous();
  const Buffers buffers(guarded, g.device());
  size_t bytes = 0;
  check(api.mluOpExtGetEmbeddingBackwardWorkspaceSize(n, rows, channels, &bytes),
        "mluOpExtGetEmbeddingBackwardWorkspaceSize");
  const at::Tensor grad_table = buffers.output({rows, channels}, g.scalar_type(), "grad_table");
  const at::Tensor ws = buffers.workspace(bytes);
  check(api.mluOpExtEmbeddingBackward(handle, dtypeCode(g.scalar_type()), g.data_ptr(), rowStride(g), token_type,
                                      t.data_ptr(), n, rows, channels, static_cast<float>(scale), ws.data_ptr(), bytes,
                                      grad_table.data_ptr()),
        "mluOpExtEmbeddingBackward");
  buffers.done("mluOpExtEmbeddingBackward");
  return grad_table;
}

struct EmbeddingRows : torch::autograd::Function<EmbeddingRows> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &table, const at::Tensor &tokens,
                            double scale, bool guarded) {
    StreamHandle &h = handleFor(table);
    const OperatorLock lock(h);
    ctx->save_for_backward({tokens});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["guarded"] = guarded;
    return embeddingForward(h.handle, guarded, table, tokens, scale);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(4);
    if (!grads[0].defined() || !ctx->needs_input_grad(0)) return out;
    const auto saved = ctx->get_saved_variables();
    StreamHandle &h = handleFor(grads[0]);
    const OperatorLock lock(h);
    out[0] = embeddingBackward(h.handle, ctx->saved_data["guarded"].toBool(), grads[0], saved[0],
                               ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble());
    return differentiableOnce(std::move(out), {grads[0]});
  }
};

// ---- products grouped by expert ------------------------------------------------------------

inline at::Tensor rowsOfProduct(const at::Tensor &t, const char *what) {
  require(t.is_cuda() && t.dim() == 2 && isFeatureType(t.scalar_type()), what);
  return channelsTogether(t);
}

inline at::Tensor groupedWorkspace(mluOpHandle_t handle, const Buffers &buffers, mluOpExtGroupedMatmul_t which,
                                   mluOpDataType_t type, int64_t rows, int64_t groups, int64_t ci, int64_t co,
                                   size_t *bytes) {
  check(api.mluOpExtGetGroupedMatmulWorkspaceSize(handle, which, type, rows, groups, ci, co, bytes),
        "mluOpExtGetGroupedMatmulWorkspaceSize");
  return *bytes > 0 ? buffers.workspace(*bytes) : at::Tensor();
}

// rows [rows, reduction] times the filters of their groups (or their transposes).
at::Tensor groupedRows(mluOpHandle_t handle, bool guarded, const at::Tensor &rows_in, const at::Tensor &filters,
                       const at::Tensor &group_starts, bool forward) {
  const at::Tensor x = rowsOfProduct(rows_in, "rows are [rows, channels] of float32, float16 or bfloat16 on the GPU");
  const at::Tensor w = rowsOn(filters, x, 3, "filters are [groups, ci, co] of the rows' type, on their GPU");
  const at::Tensor starts = startsOn(group_starts, x, "group_starts are int32 [groups + 1] on the rows' GPU");
  const int64_t groups = w.size(0), ci = w.size(1), co = w.size(2), rows = x.size(0);
  require(starts.size(0) == groups + 1, "group_starts are one more than the filters");
  require(x.size(1) == (forward ? ci : co), "rows have the filters' channels");
  const Buffers buffers(guarded, x.device());
  const mluOpDataType_t type = dtypeCode(x.scalar_type());
  const at::Tensor out = buffers.output({rows, forward ? co : ci}, x.scalar_type(), forward ? "out" : "input_grad");
  size_t bytes = 0;
  const at::Tensor ws = groupedWorkspace(handle, buffers, forward ? MLUOP_EXT_GROUPED_FORWARD : MLUOP_EXT_GROUPED_BACKWARD_DATA,
                                         type, rows, groups, ci, co, &bytes);
  void *at = ws.defined() ? ws.data_ptr() : nullptr;
  const auto *s = static_cast<const int32_t *>(starts.data_ptr());
  if (forward)
    check(api.mluOpExtGroupedMatmulForward(handle, type, x.data_ptr(), rowStride(x), rows, s, groups, ci, co, w.data_ptr(),
                                           at, bytes, out.data_ptr()),
          "mluOpExtGroupedMatmulForward");
  else
    check(api.mluOpExtGroupedMatmulBackwardData(handle, type, x.data_ptr(), rowStride(x), rows, s, groups, ci, co,
                                                w.data_ptr(), at, bytes, out.data_ptr()),
          "mluOpExtGroupedMatmulBackwardData");
  buffers.done(forward ? "mluOpExtGroupedMatmulForward" : "mluOpExtGroupedMatmulBackwardData");
  return out;
}

at::Tensor groupedFilter(mluOpHandle_t handle, bool guarded, const at::Tensor &features, const at::Tensor &output_grad,
                         const at::Tensor &group_starts) {
  const at::Tensor x = rowsOfProduct(features, "features are [rows, ci] of float32, float16 or bfloat16 on the GPU");
  require(output_grad.device() == x.device() && output_grad.dim() == 2 && output_grad.scalar_type() == x.scalar_type() &&
              output_grad.size(0) == x.size(0),
          "output_grad is [rows, co] of the features' type, on their GPU");
  const at::Tensor dy = channelsTogether(output_grad);
  const at::Tensor starts = startsOn(group_starts, x, "group_starts are int32 [groups + 1] on the features' GPU");
  const int64_t rows = x.size(0), groups = starts.size(0) - 1, ci = x.size(1), co = dy.size(1);
  const Buffers buffers(guarded, x.device());
  const mluOpDataType_t type = dtypeCode(x.scalar_type());
  const at::Tensor out = buffers.output({groups, ci, co}, x.scalar_type(), "filters_grad");
  size_t bytes = 0;
  const at::Tensor ws =
      groupedWorkspace(handle, buffers, MLUOP_EXT_GROUPED_BACKWARD_FILTER, type, rows, groups, ci, co, &bytes);
  check(api.mluOpExtGroupedMatmulBackwardFilter(handle, type, x.data_ptr(), rowStride(x), dy.data_ptr(), rowStride(dy),
                                                rows, static_cast<const int32_t *>(starts.data_ptr()), groups, ci, co,
                                                ws.defined() ? ws.data_ptr() : nullptr, bytes, out.data_ptr()),
        "mluOpExtGroupedMatmulBackwardFilter");
  buffers.done("mluOpExtGroupedMatmulBackwardFilter");
  return out;
}

struct GroupedMatmul : torch::autograd::Function<GroupedMatmul> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &features, const at::Tensor &filters,
                            const at::Tensor &group_starts, bool guarded) {
    StreamHandle &h = handleFor(features);
    const OperatorLock lock(h);
    ctx->save_for_backward({features, filters, group_starts});
    ctx->saved_data["guarded"] = guarded;
    return groupedRows(h.handle, guarded, features, filters, group_starts, true);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(4);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const bool guarded = ctx->saved_data["guarded"].toBool();
    StreamHandle &h = handleFor(saved[0]);
    const OperatorLock lock(h);
    if (ctx->needs_input_grad(0)) out[0] = groupedRows(h.handle, guarded, grads[0], saved[1], saved[2], false);
    if (ctx->needs_input_grad(1)) out[1] = groupedFilter(h.handle, guarded, saved[0], grads[0], saved[2]);
    return differentiableOnce(std::move(out), {grads[0], saved[0], saved[1]});
  }
};

void defineTraining(py::module_ &m) {
  using NoGil = py::gil_scoped_release;
  py::class_<AdamWTensors>(m, "AdamWTensors")
      .def(py::init<AdamWTensors::Tensors, AdamWTensors::Tensors, AdamWTensors::Tensors,
                    std::optional<AdamWTensors::Tensors>, std::optional<AdamWTensors::Tensors>,
                    std::optional<AdamWTensors::Tensors>>())
      .def("step", [](AdamWTensors &tensors, uintptr_t handle, const std::vector<std::optional<at::Tensor>> &grads,
                      int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay,
                      double grad_scale) {
        NoGil released;
        const OperatorLock lock(asHandle(handle));
        tensors.step(asHandle(handle), grads, step, lr, beta1, beta2, eps, weight_decay, grad_scale);
      });
  m.def("group_norm_forward",
        [](uintptr_t handle, bool guarded, const at::Tensor &features, const MaybeTensor &weight, const MaybeTensor &bias,
           int64_t groups, const MaybeTensor &row_starts, double eps, int activation) {
          std::vector<at::Tensor> r;
          {
            NoGil released;
            const OperatorLock lock(asHandle(handle));
            r = groupNormForward(asHandle(handle), guarded, features, weight, bias, groups, row_starts, eps, activation);
          }
          return py::make_tuple(r[0], r[1], r[2]);
        });
  m.def("group_norm_backward",
        [](uintptr_t handle, bool guarded, const at::Tensor &output_grad, const at::Tensor &features,
           const MaybeTensor &weight, const MaybeTensor &bias, const at::Tensor &mean, const at::Tensor &rstd,
           int64_t groups, const MaybeTensor &row_starts, int activation) {
          std::vector<at::Tensor> r;
          {
            NoGil released;
            const OperatorLock lock(asHandle(handle));
            r = groupNormBackward(asHandle(handle), guarded, output_grad, features, weight, bias, mean, rstd, groups,
                                  row_starts, activation);
          }
          return py::make_tuple(r[0], r[1], r[2]);
        });
  m.def("group_norm", [](const at::Tensor &features, const MaybeTensor &weight, const MaybeTensor &bias, int64_t groups,
                         const MaybeTensor &row_starts, double eps, int64_t activation, bool guarded) {
    NoGil released;
    return GroupNorm::apply(features, weight ? *weight : at::Tensor(), bias ? *bias : at::Tensor(), groups, row_starts,
                            eps, activation, guarded);
  });
  m.def("embedding_forward", [](uintptr_t handle, bool guarded, const at::Tensor &table, const at::Tensor &tokens,
                                double scale) {
    NoGil released;
    const OperatorLock lock(asHandle(handle));
    return embeddingForward(asHandle(handle), guarded, table, tokens, scale);
  });
  m.def("embedding_backward", [](uintptr_t handle, bool guarded, const at::Tensor &output_grad, const at::Tensor &tokens,
                                 int64_t rows, double scale) {
    NoGil released;
    const OperatorLock lock(asHandle(handle));
    return embeddingBackward(asHandle(handle), guarded, output_grad, tokens, rows, scale);
  });
  m.def("embedding", [](const at::Tensor &table, const at::Tensor &tokens, double scale, bool guarded) {
    NoGil released;
    return EmbeddingRows::apply(table, tokens, scale, guarded);
  });
  m.def("grouped_matmul_rows", [](uintptr_t handle, bool guarded, const at::Tensor &rows, const at::Tensor &filters,
                                  const at::Tensor &group_starts, bool forward) {
    NoGil released;
    const OperatorLock lock(asHandle(handle));
    return groupedRows(asHandle(handle), guarded, rows, filters, group_starts, forward);
  });
  m.def("grouped_matmul_backward_filter", [](uintptr_t handle, bool guarded, const at::Tensor &features,
                                             const at::Tensor &output_grad, const at::Tensor &group_starts) {
    NoGil released;
    const OperatorLock lock(asHandle(handle));
    return groupedFilter(asHandle(handle), guarded, features, output_grad, group_starts);
  });
  m.def("grouped_matmul", [](const at::Tensor &features, const at::Tensor &filters, const at::Tensor &group_starts,
                             bool guarded) {
    NoGil released;
    return GroupedMatmul::apply(features, filters, group_starts, guarded);
  });
}
