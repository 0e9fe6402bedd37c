/*
 * mlu_op_ext.h -- small extensions of the MI355X library that the reference
 * API does not have.  Nothing here is needed to use the operators.
 */
#ifndef MLUOP_AMD_MLU_OP_EXT_H_
#define MLUOP_AMD_MLU_OP_EXT_H_

#include "mlu_op.h"

#if defined(__cplusplus)
extern "C" {
#endif

/* Per-kernel device timing.  The reference offers kernel tracing through
 * environment switches that wrap every kernel invocation
 * (core/kernel_tracing.cpp:41-120, core/mlu_op_trace.cpp:50-100); here the
 * handle records a HIP event pair around every kernel it enqueues while timing
 * is enabled.  Enabling (or re-enabling) clears earlier records.  Recording
 * costs two event records per launch, so leave it off in production. */
mluOpStatus_t MLUOP_WIN_API mluOpExtSetKernelTiming(mluOpHandle_t handle, int enable);

/* Kernel choices of the sparse convolution operators.  Where two kernels compute the same
 * result the shape decides between them; the parity tests switch each one on and off through
 * this call and compare.  value: -1 the shape decides (the default), 0 never, 1 whenever the
 * kernel can run the shape.  The choice belongs to the handle and holds until changed.  (The
 * reference selects kernels by shape only; its test-time switches are environment variables
 * of the test runner, pb_gtest/src/runtime.cpp.) */
typedef enum {
  MLUOP_EXT_KERNEL_GATHER_SIMT = 0,    /* plain SIMT kernels instead of the MFMA ones */
  MLUOP_EXT_KERNEL_DENSE_TILES = 1,    /* register-accumulating gather kernel */
  MLUOP_EXT_KERNEL_WAVE_PER_TILE = 2,  /* one-wavefront-per-tile gather kernel */
  MLUOP_EXT_KERNEL_FLAT_SLICE_SUM = 3, /* backward filter: partial tiles summed on a flat grid */
  MLUOP_EXT_KERNEL_FLAT_SCATTER = 4,   /* row maps built on a flat grid */
  MLUOP_EXT_KERNEL_SMALL_MAP_CHUNKS = 5, /* 1: row maps cover 2048 result rows at a time instead of
                                            as many as 64 MiB hold (runs the chunked path on small inputs) */
  MLUOP_EXT_KERNEL_FILTER_STORES = 6,   /* 1: backward filter transposes its operands with element-sized
                                           LDS stores also for 2-byte types of 32 to 128 channels, where
                                           transposing LDS reads are the default */
  MLUOP_EXT_KERNEL_LISTS_ON_TRUST = 7,  /* forward on a rulebook of this handle whose report (were the input
                                           rows in cell order?) has not reached the host yet, as under graph
                                           capture or without any wait between the two calls.  -1: start on
                                           the pair lists and enqueue the row-map kernels behind them; the
                                           first kernel's check decides on the device which of the two do the
                                           work, the others return at once.  0: build the row map.  1: a test
                                           switch: the pair lists only; a call whose lists fail the check
                                           leaves its output as it was */
  MLUOP_EXT_KERNEL_TALL_TILES = 16,     /* gather kernel with tall tiles of result rows (8 is refused, as it always was) */
  MLUOP_EXT_KERNEL_SMALL_RULEBOOK = 17 /* submanifold rulebooks of up to 4096 rows in one launch */
} mluOpExtKernelChoice_t;

mluOpStatus_t MLUOP_WIN_API mluOpExtSetKernelChoice(mluOpHandle_t handle,
                                                    mluOpExtKernelChoice_t which, int value);

/* Waits for the handle's queue, then reports how many launches were recorded. */
mluOpStatus_t MLUOP_WIN_API mluOpExtGetKernelTimingCount(mluOpHandle_t handle, int *count);

/* Name and duration in milliseconds of recorded launch `index` (launch order).
 * The name points at a string literal owned by the library. */
mluOpStatus_t MLUOP_WIN_API mluOpExtGetKernelTiming(mluOpHandle_t handle, int index,
                                                    const char **name, float *milliseconds);

/* Modes of the indice-convolution operators that the reference rejects
 * (kernels/sparse_conv/indice_convolution_forward/indice_convolution_forward.cpp:74-78,
 * indice_convolution_backward_data.cpp:129-132, indice_convolution_backward_filter.cpp:185).
 * Off by default: a fresh handle answers them with the reference's status codes.
 * With `enable` non-zero the three operators accept
 *   - inverse = 1: the sparse inverse convolution of the PyTorch sparse-convolution
 *     stacks (spconv / mmcv SparseInverseConv3d).  The operator runs the rulebook of
 *     its partner layer backwards: input-side rows (features, input_grad) are taken
 *     through pair column 1, output-side rows (features_out, output_grad) through
 *     column 0, so indice_pairs.dim[2] must equal the row count of the output-side
 *     tensor (num_act_out for the forward operator) and the filter stays
 *     W(k, ci, co) of this layer;
 *   - a filters_grad descriptor tagged NHWC / NDHWC ([Co, (kd,) kh, kw, Ci]) or
 *     NCHW / NCDHW ([Co, Ci, (kd,) kh, kw]) in mluOpIndiceConvolutionBackwardFilter,
 *     written in that layout (the reference reads the dimensions positionally as
 *     (kd,) kh, kw, Ci, Co whatever the tag says). */
mluOpStatus_t MLUOP_WIN_API mluOpExtSetSparseConvExtendedModes(mluOpHandle_t handle, int enable);

/* mluOpIndiceConvolutionForward and mluOpIndiceConvolutionBackwardData add every pair of
 * indice_pairs, as the reference does, also when several pairs of one offset name the same
 * result row (which mluOpGetIndicePairs produces for repeated input coordinates, and made-up
 * pair tensors can hold anywhere).  Finding out costs one small kernel behind every call.  A
 * caller whose coordinates are distinct (voxelized point clouds are) can promise so: with
 * `promised` non-zero that kernel is not launched, and a rulebook that breaks the promise loses
 * all but one of such pairs.  Off by default. */
mluOpStatus_t MLUOP_WIN_API mluOpExtSetDistinctPairsPromise(mluOpHandle_t handle, int promised);

/* A caller can promise that one pair column (0 or 1) names rows of the result only and none of them twice, over all
 * offsets together: the input rows of a strided layer whose kernel reaches no further than its stride are in
 * one pair each.  mluOpIndiceConvolutionForward and mluOpIndiceConvolutionBackwardData calls whose result rows
 * that column names then multiply full tiles of pairs and store the products, with nothing to add up.  Rows in no pair
 * are zero, and so is the row of a pair whose other column names no row.  Where a rulebook breaks the promise, a row
 * named twice may hold any mixture of its pairs' products, from run to run another, and a row in no pair may keep what
 * the memory held before.  -1, the value of a new handle: no promise.  Holds until changed; the second call
 * says which is in force. */
mluOpStatus_t MLUOP_WIN_API mluOpExtSetSinglePairsPromise(mluOpHandle_t handle, int column);
mluOpStatus_t MLUOP_WIN_API mluOpExtGetSinglePairsPromise(mluOpHandle_t handle, int *column);

/* Whether mluOpGetIndicePairs sets the slots of indice_pairs behind each offset's indice_num pairs to -1 (the
 * default, and what the reference does).  0: it leaves them as they are, which saves most of a sparse
 * rulebook's writes; for callers who, like the indice-convolution operators, read no further than
 * indice_num.  Holds for the handle until changed.  The second call says which of the two is in force, for
 * callers who change it for a while. */
mluOpStatus_t MLUOP_WIN_API mluOpExtSetPairTails(mluOpHandle_t handle, int fill);
mluOpStatus_t MLUOP_WIN_API mluOpExtGetPairTails(mluOpHandle_t handle, int *fill);

/* mluOpIndiceConvolutionForward stores negative results as zero (NaN stays NaN) while this is on: the ReLU
 * behind a layer without a pass of its own over the result.  Off for a new handle; holds until changed. */
mluOpStatus_t MLUOP_WIN_API mluOpExtSetForwardRelu(mluOpHandle_t handle, int enable);
mluOpStatus_t MLUOP_WIN_API mluOpExtGetForwardRelu(mluOpHandle_t handle, int *enable);

/* The pair counts of a rulebook on the host.  The convolution operators take indice_num as a host
 * array, so a caller has to bring the counts mluOpGetIndicePairs left in device memory over; a copy
 * waits for the whole queue.  The last kernel of a rulebook also stores them into pinned memory of
 * the handle: this call waits for them there and fills indice_num[0 .. kernel_volume).  For the last
 * 32 rulebooks of the handle.  `indice_pairs` names a rulebook by its address: the answer is for the
 * one this handle last built there.  NOT_SUPPORTED if it built none with so many offsets there, built
 * it under graph capture or with more than 343 offsets, or if an operator of this handle has written
 * into the tensor since (copy the counts then).  What others write there, or that the memory was
 * freed and given out again, the handle cannot see: ask while the tensor is the rulebook, as for the
 * operators that take both.  No counterpart in the reference. */
mluOpStatus_t MLUOP_WIN_API mluOpExtGetIndicePairsHostCounts(mluOpHandle_t handle, const void *indice_pairs,
                                                             int kernel_volume, int64_t indice_num[]);

/* The number of voxels of the handle's last mluOpVoxelization on the host.  Its last kernel stores the
 * number into pinned memory of the handle while it writes the voxels: this call waits for it there,
 * where a copy of voxel_num waits for the whole queue.  NOT_SUPPORTED if `voxel_num` is not the address
 * that call was given, an operator of this handle has written there since, or the call was captured
 * into a graph (copy the number then).  The answer is what that call found, whatever others have
 * written to the address since.  No counterpart in the reference. */
mluOpStatus_t MLUOP_WIN_API mluOpExtGetVoxelizationHostCount(mluOpHandle_t handle, const void *voxel_num,
                                                             int32_t *count);

/* The order of voxels by their linear cell index (z * space[1] + y) * space[2] + x, and their cells in that
 * order.  coors [voxels, 3] int32 (z, y, x) as mluOpVoxelization writes them; order [voxels] int64, the
 * voxel at each place; indices [voxels, 4] int32 (batch_index, z, y, x) in order.  Equal cells are ordered
 * by voxel; coordinates outside the space are ordered by their index all the same.  1 to 2^20 voxels
 * (NOT_SUPPORTED above), workspace of the queried size.  No counterpart in the reference. */
mluOpStatus_t MLUOP_WIN_API mluOpExtGetOrderVoxelsWorkspaceSize(int64_t voxels, const int64_t space[3],
                                                                size_t *size);
mluOpStatus_t MLUOP_WIN_API mluOpExtOrderVoxels(mluOpHandle_t handle, const void *coors, int64_t voxels,
                                                const int64_t space[3], int32_t batch_index, void *workspace,
                                                size_t workspace_size, void *order, void *indices);

/* The mean of every voxel's points: voxels [num_voxels, max_points, features] fp32, contiguous, as mluOpVoxelization
 * writes them (all slots are summed: those behind a voxel's points hold zeros), num_points_per_voxel
 * [num_voxels] int32, below one taken as one; mean [num_voxels, features] fp32.  One launch, no workspace, no
 * wait.  No counterpart in the reference. */
mluOpStatus_t MLUOP_WIN_API mluOpExtMeanVoxelPoints(mluOpHandle_t handle, const void *voxels,
                                                    const void *num_points_per_voxel, int64_t num_voxels,
                                                    int32_t max_points, int32_t features, void *mean);

/* Row maps kept across calls.  mluOpIndiceConvolutionForward and ...BackwardData turn the pair
 * lists into a [K, rows] map (partner row of every result row at every offset, or -1) on every
 * call: the reference API (mlu_op.h:10321-10448, :9625-9773) hands them nothing else to keep.
 * Layers that share a rulebook, and the forward and backward pass of each, can build the map
 * once.  No counterpart in the reference.
 *
 *   mluOpExtGetRowMapSize  bytes of a map buffer for `rows` result rows.
 *   mluOpExtBuildRowMap    fills `row_map` (device memory of that size, owned by the caller) on
 *                          the handle's queue and waits for the queue once.  `row_column` is the
 *                          pair column that names the result rows: 1 for a forward convolution
 *                          (and an inverse layer's backward data), 0 for backward data (and an
 *                          inverse layer's forward); `rows` / `source_rows` are the row counts
 *                          of the result and of the gathered tensor, the one that column 0
 *                          indexes being indice_pairs.dim[2].  `*lost_pairs` returns how many
 *                          pairs found no slot of their own (several pairs of one offset naming
 *                          one result row, or rows outside their tensors): such a map is not
 *                          recorded and cannot be used; call the operators without it.
 *                          With mluOpExtSetDistinctPairsPromise in force `lost_pairs` may be
 *                          NULL: the build then neither counts nor waits, and the promise
 *                          stands in for the verdict.
 *   mluOpExtUseRowMap      announces a recorded map for the next mluOpIndiceConvolutionForward
 *                          or ...BackwardData call on this handle, which must be given the same
 *                          indice_pairs pointer, shapes and direction the map was built for
 *                          (BAD_PARAM otherwise) and then launches neither the map kernels nor
 *                          the check for colliding pairs.  The announcement ends with that call,
 *                          whatever it returns.  The pair tensor must not have changed since the
 *                          map was built.  NULL withdraws an announcement.
 *   mluOpExtForgetRowMap   drops the record of a buffer about to be freed (NULL: all records). */
mluOpStatus_t MLUOP_WIN_API mluOpExtGetRowMapSize(const mluOpTensorDescriptor_t indice_pairs_desc,
                                                  int64_t rows, size_t *size);
mluOpStatus_t MLUOP_WIN_API mluOpExtBuildRowMap(mluOpHandle_t handle,
                                                const mluOpTensorDescriptor_t indice_pairs_desc,
                                                const void *indice_pairs, const int64_t indice_num[],
                                                int64_t rows, int64_t source_rows, int row_column,
                                                void *row_map, size_t size, int64_t *lost_pairs);
mluOpStatus_t MLUOP_WIN_API mluOpExtUseRowMap(mluOpHandle_t handle, const void *row_map);
mluOpStatus_t MLUOP_WIN_API mluOpExtForgetRowMap(mluOpHandle_t handle, const void *row_map);

/* mluOpIndiceConvolutionBackwardFilter for callers that cannot allocate device memory (code
 * under HIP graph capture, serving loops, harnesses that forbid hipMalloc) and therefore have
 * no workspace to hand over.  No counterpart in the reference.  Same arguments and checks as
 * mluOpIndiceConvolutionBackwardFilter (mlu_op.h), without `workspace` and `workspace_size`:
 * the partial sums live in an array of MLUOP_EXT_NO_ALLOC_SCRATCH_BYTES that the library
 * holds on every GPU it runs on until the process ends.  The call allocates and frees nothing,
 * does not wait for the queue, follows the handle's kernel choices and is left out of its
 * per-kernel timing (which creates events).  Shapes of the matrix-core kernels (16 to 128
 * channels) whose usual number of partial tiles exceeds the array are cut into fewer, longer
 * slices: the result then agrees with the workspace entry point within the accuracy standard
 * (the additions are grouped differently), and bit for bit otherwise (up to 64 x 64 channels at
 * 27 offsets).  MLUOP_STATUS_NOT_SUPPORTED when the array is too small all the same (the generic
 * kernels' tiles at large channel counts) or with more than 128 kernel offsets.  All calls on
 * one GPU share the array:
 * calls that can overlap there (different queues, different handles) race and must be ordered
 * by the caller. */
#define MLUOP_EXT_NO_ALLOC_SCRATCH_BYTES (16 * 1024 * 1024)
mluOpStatus_t MLUOP_WIN_API mluOpExtIndiceConvolutionBackwardFilterNoAlloc(
    mluOpHandle_t handle, const mluOpTensorDescriptor_t features_desc, const void *features,
    const mluOpTensorDescriptor_t output_grad_desc, const void *output_grad,
    const mluOpTensorDescriptor_t indice_pairs_desc, const void *indice_pairs,
    const int64_t indice_num[], const int64_t inverse, const int64_t subm,
    const mluOpTensorDescriptor_t filters_grad_desc, void *filters_grad);

/* ---- the rest of a training step --------------------------------------------------------------
 * Operators a network over ragged rows of features needs next to its convolutions: none of them has a counterpart in the
 * reference.  All pointers are device memory unless said otherwise; types are MLUOP_DTYPE_FLOAT, _HALF or _BFLOAT16 for
 * features, and every sum is held in fp32 and rounded once.  They enqueue kernels on the handle's queue and return: no
 * wait, no allocation, nothing that a graph capture refuses.  No float atomics: results repeat bit by bit. */

/* One AdamW step (decoupled weight decay) over many tensors in as few launches as they fit in:
 *   g = grad_scale * grad;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2;
 *   p = p (1 - lr weight_decay) - lr / (1 - beta1^step) * m / (sqrt(v / (1 - beta2^step)) + eps)
 * in fp32.  `tensors` is host memory, read before the call returns.  param_type: of all params; grad_type: the same or
 * FLOAT.  master: fp32 copies of 16-bit params, from which a step starts and which it updates together with the params;
 * for all tensors or for none.  state_type FLOAT: exp_avg (m) and exp_avg_sq (v) are fp32 [count], the scales are not looked
 * at.  UINT8: they are OCP e4m3 codes [count] of m and of sqrt(v), and every block of MLUOP_EXT_ADAMW_BLOCK consecutive
 * elements has an fp32 scale [ceil(count / block)] that its codes' values are multiplied by (largest magnitude / 448).
 * step counts from 1; 0 <= beta1, beta2 < 1; eps >= 0.  Tensors of no elements are passed over.  A NaN or an infinity in a
 * gradient stays in its element, but for an infinity with 8-bit states, which is its block's scale. */
#define MLUOP_EXT_ADAMW_BLOCK 256
typedef struct {
  void *param;
  const void *grad;
  void *exp_avg;
  void *exp_avg_sq;
  float *master;
  float *exp_avg_scale;
  float *exp_avg_sq_scale;
  int64_t count;
} mluOpExtAdamWTensor_t;
mluOpStatus_t MLUOP_WIN_API mluOpExtAdamWStep(mluOpHandle_t handle, const mluOpExtAdamWTensor_t tensors[],
                                              int num_tensors, mluOpDataType_t param_type, mluOpDataType_t grad_type,
                                              mluOpDataType_t state_type, int64_t step, double lr, double beta1,
                                              double beta2, double eps, double weight_decay, double grad_scale);

/* Group norm with an activation over rows [rows, channels] whose channels lie side by side.  Rows belong to samples: sample
 * s has the rows row_starts[s] to row_starts[s + 1] - 1 (int32 [samples + 1], ascending; NULL: one sample of all rows).
 * Mean and variance (of the population) are taken over a sample's rows and the channels / groups channels of each group;
 *   out = activation((x - mean) * rstd * weight + bias),  rstd = 1 / sqrt(variance + eps).
 * weight and bias [channels] of param_type, FLOAT or `type`; NULL: one and zero.  mean and rstd fp32 [samples, groups] are
 * results that the backward pass takes (0 and 1 / sqrt(eps) for a sample without rows).  Rows of no sample are zero in
 * every result.  Backward: input_grad [rows, channels], weight_grad and bias_grad [channels] of param_type (NULL where not
 * wanted).  One workspace size serves both.  At most 2^20 channels and samples, and 15 * 2^20 pairs of a sample and a group. */
typedef enum {
  MLUOP_EXT_ACTIVATION_NONE = 0,
  MLUOP_EXT_ACTIVATION_RELU = 1,
  MLUOP_EXT_ACTIVATION_SILU = 2
} mluOpExtActivation_t;
mluOpStatus_t MLUOP_WIN_API mluOpExtGetGroupNormWorkspaceSize(int64_t rows, int64_t channels, int64_t groups,
                                                              int64_t samples, size_t *size);
mluOpStatus_t MLUOP_WIN_API mluOpExtGroupNormForward(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                                     int64_t rows, int64_t channels, int64_t groups,
                                                     const int32_t *row_starts, int64_t samples,
                                                     mluOpDataType_t param_type, const void *weight, const void *bias,
                                                     float eps, mluOpExtActivation_t activation, void *workspace,
                                                     size_t workspace_size, void *out, float *mean, float *rstd);
mluOpStatus_t MLUOP_WIN_API mluOpExtGroupNormBackward(mluOpHandle_t handle, mluOpDataType_t type,
                                                      const void *output_grad, const void *features, int64_t rows,
                                                      int64_t channels, int64_t groups, const int32_t *row_starts,
                                                      int64_t samples, mluOpDataType_t param_type, const void *weight,
                                                      const void *bias, const float *mean, const float *rstd,
                                                      mluOpExtActivation_t activation, void *workspace,
                                                      size_t workspace_size, void *input_grad, void *weight_grad,
                                                      void *bias_grad);

/* Rows of a table by their numbers: out[t, :] = scale * table[tokens[t], :], for num_tokens tokens (token_type INT32 or
 * INT64) of a table [rows, channels] whose rows lie row_stride elements apart (at least channels); out [num_tokens,
 * channels].  A token outside [0, rows) names no row: its result is zero.  A table may have no rows where there are no tokens.
 * The gradient of the table: grad_table[v, :] = scale * sum of output_grad[t, :] over the tokens that name v, added up in
 * an order that the tokens alone decide; zero for a row that none names.  The tokens are sorted in the workspace.  rows,
 * num_tokens below 2^31. */
mluOpStatus_t MLUOP_WIN_API mluOpExtEmbeddingForward(mluOpHandle_t handle, mluOpDataType_t type, const void *table,
                                                     int64_t rows, int64_t channels, int64_t row_stride,
                                                     mluOpDataType_t token_type, const void *tokens, int64_t num_tokens,
                                                     float scale, void *out);
mluOpStatus_t MLUOP_WIN_API mluOpExtGetEmbeddingBackwardWorkspaceSize(int64_t num_tokens, int64_t rows,
                                                                      int64_t channels, size_t *size);
mluOpStatus_t MLUOP_WIN_API mluOpExtEmbeddingBackward(mluOpHandle_t handle, mluOpDataType_t type,
                                                      const void *output_grad, int64_t row_stride,
                                                      mluOpDataType_t token_type, const void *tokens, int64_t num_tokens,
                                                      int64_t rows, int64_t channels, float scale, void *workspace,
                                                      size_t workspace_size, void *grad_table);

/* Products grouped by expert: rows group_starts[g] to group_starts[g + 1] - 1 (int32 [groups + 1] on the device, ascending,
 * any of them empty) are multiplied with the filter of group g, filters [groups, ci, co]:
 *   forward          out[r, :]         = features[r, :] . filters[g]            [rows, co]
 *   backward data    input_grad[r, :]  = output_grad[r, :] . filters[g]^T       [rows, ci]
 *   backward filter  filters_grad[g]   = features_g^T . output_grad_g           [groups, ci, co]
 * features_stride, output_grad_stride: elements from row to row.  Rows of no group are zero in the results, a group without
 * rows has a gradient of zero, and a filter without rows is not read.  The workspace of the queried size (which may be 0)
 * belongs to one of the three. */
typedef enum {
  MLUOP_EXT_GROUPED_FORWARD = 0,
  MLUOP_EXT_GROUPED_BACKWARD_DATA = 1,
  MLUOP_EXT_GROUPED_BACKWARD_FILTER = 2
} mluOpExtGroupedMatmul_t;
mluOpStatus_t MLUOP_WIN_API mluOpExtGetGroupedMatmulWorkspaceSize(mluOpHandle_t handle, mluOpExtGroupedMatmul_t which,
                                                                  mluOpDataType_t type, int64_t rows, int64_t groups,
                                                                  int64_t ci, int64_t co, size_t *size);
mluOpStatus_t MLUOP_WIN_API mluOpExtGroupedMatmulForward(mluOpHandle_t handle, mluOpDataType_t type,
                                                         const void *features, int64_t features_stride, int64_t rows,
                                                         const int32_t *group_starts, int64_t groups, int64_t ci,
                                                         int64_t co, const void *filters, void *workspace,
                                                         size_t workspace_size, void *out);
mluOpStatus_t MLUOP_WIN_API mluOpExtGroupedMatmulBackwardData(mluOpHandle_t handle, mluOpDataType_t type,
                                                              const void *output_grad, int64_t output_grad_stride,
                                                              int64_t rows, const int32_t *group_starts, int64_t groups,
                                                              int64_t ci, int64_t co, const void *filters,
                                                              void *workspace, size_t workspace_size, void *input_grad);
mluOpStatus_t MLUOP_WIN_API mluOpExtGroupedMatmulBackwardFilter(mluOpHandle_t handle, mluOpDataType_t type,
                                                                const void *features, int64_t features_stride,
                                                                const void *output_grad, int64_t output_grad_stride,
                                                                int64_t rows, const int32_t *group_starts,
                                                                int64_t groups, int64_t ci, int64_t co, void *workspace,
                                                                size_t workspace_size, void *filters_grad);

/* Layer norm: every row [channels] of features [rows, channels] (features_stride elements from row to row) by itself:
 *   out = (x - mean) * rstd * weight + bias,  rstd = 1 / sqrt(variance + eps),  variance of the population.
 * weight and bias [channels] of param_type, FLOAT or `type`; NULL: one and zero.  mean and rstd fp32 [rows] are results that the
 * backward pass takes.  Backward: input_grad [rows, channels], weight_grad and bias_grad [channels] of param_type (NULL where
 * not wanted; zero where there are no rows).  Statistics are fp32: where squares of differences from the mean leave its range,
 * rstd is zero.  At most 2^15 channels. */
mluOpStatus_t MLUOP_WIN_API mluOpExtLayerNormForward(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                                     int64_t features_stride, int64_t rows, int64_t channels,
                                                     mluOpDataType_t param_type, const void *weight, const void *bias,
                                                     float eps, void *out, float *mean, float *rstd);
mluOpStatus_t MLUOP_WIN_API mluOpExtGetLayerNormBackwardWorkspaceSize(int64_t rows, int64_t channels, size_t *size);
mluOpStatus_t MLUOP_WIN_API mluOpExtLayerNormBackward(mluOpHandle_t handle, mluOpDataType_t type, const void *output_grad,
                                                      int64_t output_grad_stride, const void *features,
                                                      int64_t features_stride, int64_t rows, int64_t channels,
                                                      mluOpDataType_t param_type, const void *weight, const float *mean,
                                                      const float *rstd, void *workspace, size_t workspace_size,
                                                      void *input_grad, void *weight_grad, void *bias_grad);

/* A gated linear recurrence along the rows of every sample, each channel by itself:
 *   SIGMOID  h_t = a h_(t-1) + (1 - a) x_t,  a = 1 / (1 + exp(-gate_t))
 *   EXP      h_t = a h_(t-1) + x_t,          a = exp(gate_t)
 * features and gates [rows, channels]; samples and row_starts as for the group norm; `initial` fp32 [samples, channels] (NULL:
 * zero) is the state in front of a sample's first row, `final` fp32 [samples, channels] that behind its last (the initial one of a
 * sample without rows).  reverse: from the last row of a sample to its first.  out [rows, channels]; rows of no sample are not
 * read, and zero in every result.  carries fp32 [carries of the sizes query, channels] is a result that the backward pass takes,
 * with the same row_starts, kind and direction.  Backward: final_grad fp32 [samples, channels] (NULL: zero), features_grad and
 * gates_grad [rows, channels], initial_grad fp32 [samples, channels] (NULL where not wanted).  One workspace size serves
 * both.  Rows are joined by composing their steps: a value that is not finite is one in the rows behind it (an infinity may be a
 * NaN there), and in no row in front of it; and with EXP gates above zero, products of a along a sample that leave fp32's range may
 * make NaNs of states that are finite.  At most 2^20 channels and samples, and MLUOP_EXT_GATED_SCAN_MOST_STRIDE elements from
 * row to row. */
#define MLUOP_EXT_GATED_SCAN_MOST_STRIDE (1 << 23)
typedef enum {
  MLUOP_EXT_GATE_SIGMOID = 0,
  MLUOP_EXT_GATE_EXP = 1
} mluOpExtGate_t;
mluOpStatus_t MLUOP_WIN_API mluOpExtGetGatedScanSizes(int64_t rows, int64_t channels, int64_t samples, size_t *carries,
                                                      size_t *workspace_size);
mluOpStatus_t MLUOP_WIN_API mluOpExtGatedScanForward(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                                     int64_t features_stride, const void *gates, int64_t gates_stride,
                                                     int64_t rows, int64_t channels, const int32_t *row_starts,
                                                     int64_t samples, const float *initial, mluOpExtGate_t kind,
                                                     int reverse, void *workspace, size_t workspace_size, void *out,
                                                     float *final, float *carries);
mluOpStatus_t MLUOP_WIN_API mluOpExtGatedScanBackward(mluOpHandle_t handle, mluOpDataType_t type, const void *output_grad,
                                                      int64_t output_grad_stride, const float *final_grad,
                                                      const void *features, int64_t features_stride, const void *gates,
                                                      int64_t gates_stride, int64_t rows, int64_t channels,
                                                      const int32_t *row_starts, int64_t samples, const float *carries,
                                                      mluOpExtGate_t kind, int reverse, void *workspace,
                                                      size_t workspace_size, void *features_grad, void *gates_grad,
                                                      float *initial_grad);

/* Rows into the order of the experts they are sent to, for the grouped products, and the results back.
 * Order: experts_of_rows [rows, choices] (index_type INT32 or INT64; a number outside [0, experts) is no expert) gives, with the
 * choices ordered by expert and equal experts by row and choice: ordered_rows int32 [rows * choices], the row at every place
 * (-1 behind the last expert's); group_starts int32 [experts + 1], where every expert's places begin; places int32 [rows,
 * choices], the place of every choice (-1 of one without an expert).  At most 2047 experts.
 * Dispatch: out[places[r, k], :] = features[r, :], out [rows * choices, channels]; places from group_starts[experts] on are zero.
 * `places` names every place in front of it once, as the order does; an entry outside of out is passed over.
 * Combine: out[r, :] = sum over k of weights[r, k] * results[places[r, k], :] in the choices' order, nothing for an entry outside
 * [0, rows * choices); weights [rows, choices] of weight_type, FLOAT or `type`; NULL: one.  Without weights it is the gradient
 * of the dispatched rows.
 * Its gradients: results_grad [rows * choices, channels], zero behind the experts' places, and weights_grad [rows, choices] of
 * weight_type (NULL where not wanted; results are read for it only). */
mluOpStatus_t MLUOP_WIN_API mluOpExtGetExpertOrderWorkspaceSize(int64_t rows, int64_t choices, int64_t experts,
                                                                size_t *size);
mluOpStatus_t MLUOP_WIN_API mluOpExtExpertOrder(mluOpHandle_t handle, mluOpDataType_t index_type,
                                                const void *experts_of_rows, int64_t rows, int64_t choices,
                                                int64_t experts, void *workspace, size_t workspace_size,
                                                int32_t *ordered_rows, int32_t *group_starts, int32_t *places);
mluOpStatus_t MLUOP_WIN_API mluOpExtExpertDispatch(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                                   int64_t features_stride, int64_t rows, int64_t channels,
                                                   int64_t choices, const int32_t *places, const int32_t *group_starts,
                                                   int64_t experts, void *out);
mluOpStatus_t MLUOP_WIN_API mluOpExtExpertCombine(mluOpHandle_t handle, mluOpDataType_t type, const void *results,
                                                  int64_t results_stride, int64_t rows, int64_t channels, int64_t choices,
                                                  const int32_t *places, mluOpDataType_t weight_type, const void *weights,
                                                  void *out);
mluOpStatus_t MLUOP_WIN_API mluOpExtExpertCombineBackward(mluOpHandle_t handle, mluOpDataType_t type,
                                                          const void *output_grad, int64_t output_grad_stride,
                                                          const void *results, int64_t results_stride, int64_t rows,
                                                          int64_t channels, int64_t choices, const int32_t *places,
                                                          const int32_t *group_starts, int64_t experts,
                                                          mluOpDataType_t weight_type, const void *weights,
                                                          void *results_grad, void *weights_grad);

/* Dropout onto a residual: out = residual + (kept ? scale * features : 0), `count` values that lie one after the other (residual
 * NULL: none).  Its gradient for the features is the same call on the output's gradient without a residual.  The probability
 * of dropping is p in [0, 1], rounded to a multiple of 2^-16, and scale is 1 / (1 - that) (at 1 nothing is kept).  state int64
 * [2], on the device: the seed and the number of the call.  Eight elements share the four 32-bit words of Philox4x32-10 with
 * the counter (element / 8 in 64 bits, number of the call in 64 bits) and the seed as key: element 8 g + i has the lower half of
 * word i / 2 for an even i, the upper for an odd one, and is kept where that is not below p * 2^16.  A value that is dropped does
 * not count, whatever it is. */
mluOpStatus_t MLUOP_WIN_API mluOpExtDropoutAdd(mluOpHandle_t handle, mluOpDataType_t type, const void *features,
                                               const void *residual, int64_t count, double p, const int64_t *state,
                                               void *out);

#if defined(__cplusplus)
}
#endif

#endif /* MLUOP_AMD_MLU_OP_EXT_H_ */
