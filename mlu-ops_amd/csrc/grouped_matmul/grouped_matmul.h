// Products grouped by expert: the problem as host and kernels see it.
#ifndef MLUOP_AMD_GROUPED_MATMUL_H_
#define MLUOP_AMD_GROUPED_MATMUL_H_

#include <cstddef>
#include <cstdint>

#include "core/launch.h"
#include "mlu_op_ext.h"

namespace mluop {
namespace grouped_matmul {

// out = left . right over a reduction, one product for every group:
//   forward          rows x co: features [rows, ci] . filters [ci, co]
//   backward data    rows x ci: output_grad [rows, co] . filters^T
//   backward filter  ci x co:   features^T . output_grad, the reduction over the group's rows
struct Problem {
  mluOpExtGroupedMatmul_t which;
  mluOpDataType_t type;
  int rows, groups, ci, co;
  const int32_t *starts;
  const void *left;   // features, or output_grad of backward data
  const void *right;  // filters, or output_grad of backward filter
  void *out;
  int64_t left_stride, right_stride;  // elements from row to row
};

// Bytes of workspace (aligned by the caller to 256).
size_t workspaceBytes(const Problem &p, int cu_count);

hipError_t launch(const LaunchCtx &lc, const Problem &p, int cu_count, void *workspace);

}  // namespace grouped_matmul
}  // namespace mluop

#endif  // MLUOP_AMD_GROUPED_MATMUL_H_
