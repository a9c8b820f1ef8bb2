// bell_mx_gemm.h — host-side pieces shared by the MXFP4 product kernels.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/bell.h"

namespace bell {
namespace mx {

// The rows of a product: quantised chunks, or the caller's rows (bf16 or f32).
struct RowSource {
  const void* chunks;
  const void* src;
  int64_t ld;
  int32_t f32;
};

// Argument checks of rows [T, features], ld elements apart (bell_mx_quant.cu).
int check_rows(int64_t T, int32_t features, int32_t B, int32_t dtype, const void* rows, const void* chunks, int64_t ld);

// T <= BELL_MX_FEW_ROWS (bell_mx_few.cu): one launch each.
int few_linear(int64_t T, const RowSource& x, const BellMxEll& w, const void* residual, void* out, int32_t out_f32,
               int32_t max_ctas, cudaStream_t s);
int few_swiglu(int64_t T, const RowSource& x, const BellMxEll& g, const BellMxEll& u, const BellMxEll& w, void* h,
               void* gate_pre, void* up_out, const void* residual, void* out, int32_t out_f32, int32_t max_ctas,
               cudaStream_t s);

}  // namespace mx
}  // namespace bell
