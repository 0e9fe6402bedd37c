// mluOpExtGroupedMatmulForward / BackwardData / BackwardFilter and their workspace query (no counterpart in the reference).
#include "grouped_matmul/grouped_matmul.h"

#include "core/core.h"
#include "core/elements.h"

namespace {

using mluop::grouped_matmul::Problem;

mluOpStatus_t checkShape(const char *api, mluOpDataType_t type, int64_t rows, int64_t groups, int64_t ci, int64_t co) {
  PARAM_CHECK(api, mluop::isFloating(type));
  PARAM_CHECK(api, rows >= 0);
  PARAM_CHECK(api, groups > 0);
  PARAM_CHECK(api, ci > 0);
  PARAM_CHECK(api, co > 0);
  if (rows > INT32_MAX - 4096 || groups > 65535 || ci > (1 << 20) || co > (1 << 20) || ci * co > ((int64_t)1 << 30) ||
      groups * ci * co > ((int64_t)1 << 44)) {
    MLUOP_LOG(ERROR) << api << " At most 2^31 - 4097 rows, 65 535 groups, 2^20 channels and 2^30 elements of a filter are "
                     << "supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  return MLUOP_STATUS_SUCCESS;
}

Problem problemOf(mluOpExtGroupedMatmul_t which, mluOpDataType_t type, int64_t rows, int64_t groups, int64_t ci,
                  int64_t co) {
  Problem p = {};
  p.which = which;
  p.type = type;
  p.rows = (int)rows;
  p.groups = (int)groups;
  p.ci = (int)ci;
  p.co = (int)co;
  return p;
}

size_t wantedBytes(const Problem &p, int cu_count) {
  const size_t bytes = mluop::grouped_matmul::workspaceBytes(p, cu_count);
  return bytes == 0 ? 0 : bytes + 256;  // (the caller's memory need not be aligned)
}

mluOpStatus_t run(const char *api, mluOpHandle_t handle, Problem p, const void *left, int64_t left_stride,
                  int64_t left_channels, const void *right, int64_t right_stride, const int32_t *starts,
                  void *workspace, size_t workspace_size, void *out, int64_t out_elements) {
  PARAM_CHECK(api, starts != NULL);
  PARAM_CHECK(api, p.rows == 0 || left != NULL);
  PARAM_CHECK(api, p.rows == 0 || left_stride >= left_channels);
  PARAM_CHECK(api, p.rows == 0 || left_stride <= ((int64_t)1 << 46) / p.rows);
  PARAM_CHECK(api, out_elements == 0 || out != NULL);
  DEVICE_HANDLE_CHECK(api, handle);
  const size_t wanted = wantedBytes(p, handle->cu_count);
  PARAM_CHECK(api, workspace_size >= wanted);
  PARAM_CHECK(api, wanted == 0 || workspace != NULL);
  if (out_elements == 0) return MLUOP_STATUS_SUCCESS;
  HIP_CHECK_RETURN(api, hipSetDevice(handle->device));
  if (handle->hasNotes()) {
    handle->forgetNotesIn(out, (size_t)out_elements * mluop::elementBytes(p.type));
    if (wanted > 0) handle->forgetNotesIn(workspace, workspace_size);
  }
  p.starts = starts;
  p.left = left;
  p.right = right;
  p.left_stride = left_stride;
  p.right_stride = right_stride;
  p.out = out;
  void *aligned = reinterpret_cast<void *>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~(uintptr_t)255);
  HIP_CHECK_RETURN(api, mluop::grouped_matmul::launch(handle->launchCtx(), p, handle->cu_count, aligned));
  return MLUOP_STATUS_SUCCESS;
}

}  // namespace

mluOpStatus_t MLUOP_WIN_API mluOpExtGetGroupedMatmulWorkspaceSize(mluOpHandle_t handle, mluOpExtGroupedMatmul_t which,
                                                                  mluOpDataType_t type, int64_t rows, int64_t groups,
                                                                  int64_t ci, int64_t co, size_t *size) {
  const char *api = "[mluOpExtGetGroupedMatmulWorkspaceSize]";
  PARAM_CHECK(api, handle != NULL);
  PARAM_CHECK(api, size != NULL);
  PARAM_CHECK(api, which >= MLUOP_EXT_GROUPED_FORWARD && which <= MLUOP_EXT_GROUPED_BACKWARD_FILTER);
  const mluOpStatus_t status = checkShape(api, type, rows, groups, ci, co);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  *size = wantedBytes(problemOf(which, type, rows, groups, ci, co), handle->cu_count);
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpExtGroupedMatmulForward(mluOpHandle_t handle, mluOpDataType_t type,
                                                         const void *features, int64_t features_stride, int64_t rows,
                                                         const int32_t *group_starts, int64_t groups, int64_t ci,
                                                         int64_t co, const void *filters, void *workspace,
                                                         size_t workspace_size, void *out) {
  const char *api = "[mluOpExtGroupedMatmulForward]";
  PARAM_CHECK(api, handle != NULL);
  const mluOpStatus_t status = checkShape(api, type, rows, groups, ci, co);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, filters != NULL);
  return run(api, handle, problemOf(MLUOP_EXT_GROUPED_FORWARD, type, rows, groups, ci, co), features, features_stride, ci,
             filters, co, group_starts, workspace, workspace_size, out, rows * co);
}

mluOpStatus_t MLUOP_WIN_API mluOpExtGroupedMatmulBackwardData(mluOpHandle_t handle, mluOpDataType_t type,
                                                              const void *output_grad, int64_t output_grad_stride,
                                                              int64_t rows, const int32_t *group_starts, int64_t groups,
                                                              int64_t ci, int64_t co, const void *filters,
                                                              void *workspace, size_t workspace_size, void *input_grad) {
  const char *api = "[mluOpExtGroupedMatmulBackwardData]";
  PARAM_CHECK(api, handle != NULL);
  const mluOpStatus_t status = checkShape(api, type, rows, groups, ci, co);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, filters != NULL);
  return run(api, handle, problemOf(MLUOP_EXT_GROUPED_BACKWARD_DATA, type, rows, groups, ci, co), output_grad,
             output_grad_stride, co, filters, co, group_starts, workspace, workspace_size, input_grad, rows * ci);
}

mluOpStatus_t MLUOP_WIN_API mluOpExtGroupedMatmulBackwardFilter(mluOpHandle_t handle, mluOpDataType_t type,
                                                                const void *features, int64_t features_stride,
                                                                const void *output_grad, int64_t output_grad_stride,
                                                                int64_t rows, const int32_t *group_starts,
                                                                int64_t groups, int64_t ci, int64_t co, void *workspace,
                                                                size_t workspace_size, void *filters_grad) {
  const char *api = "[mluOpExtGroupedMatmulBackwardFilter]";
  PARAM_CHECK(api, handle != NULL);
  const mluOpStatus_t status = checkShape(api, type, rows, groups, ci, co);
  if (status != MLUOP_STATUS_SUCCESS) return status;
  PARAM_CHECK(api, rows == 0 || output_grad != NULL);
  PARAM_CHECK(api, rows == 0 || output_grad_stride >= co);
  PARAM_CHECK(api, rows == 0 || output_grad_stride <= ((int64_t)1 << 46) / rows);
  return run(api, handle, problemOf(MLUOP_EXT_GROUPED_BACKWARD_FILTER, type, rows, groups, ci, co), features,
             features_stride, ci, output_grad, output_grad_stride, group_starts, workspace, workspace_size, filters_grad,
             groups * ci * co);
}
