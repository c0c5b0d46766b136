// few_rows.h -- the learned layers' products for a few rows (few_rows.cu).
#pragma once

#include "af2_internal.h"

namespace af2 {

// Whether a product is small enough for the CUDA-core kernel, which starts and ends sooner than the
// tensor-core one and reads f32 as it is.  Measured on whole transitions, us (few rows | tensor cores):
// bf16, 512 -> 2048: 8 rows 9.8 | 15, 16 rows 15.0 | 15.1; 1024 -> 4096: 4 rows 13 | 20, 8 rows 25 | 20;
// f32, 512 -> 2048: 48 rows 39.1 | 39.0; 1024 -> 4096: 16 rows 46 | 80, 24 rows 70 | 72.
inline bool few_rows(int64_t rows, int64_t inner, int64_t columns, int dtype) {
  const int64_t most = dtype == AF2_F32 ? 3 << 24 : 1 << 24;  // products of two elements
  return rows <= 256 && rows * inner * columns <= most;
}

struct FewRows {
  int64_t rows = 0, inner = 0, columns = 0;
  int dtype = 0, activation = 0;
  const void *x = nullptr;  // [rows][x_stride] of dtype
  int64_t x_stride = 0;
  // weight[1] NULL: out = act(x weight[0] + bias[0]) (+ residual);
  // else out = act(x weight[0] + bias[0]) * (x weight[1] + bias[1])
  const void *weight[2] = {nullptr, nullptr}, *bias[2] = {nullptr, nullptr};
  const void *residual = nullptr;
  int64_t residual_stride = 0;
  void *out = nullptr;
  int64_t out_stride = 0;
  bool follows = false;  // x is written by the launch before on the stream, which touches no weight
};
af2_status few_rows_launch(af2_ctx *ctx, const FewRows &f, cudaStream_t stream);

}  // namespace af2
