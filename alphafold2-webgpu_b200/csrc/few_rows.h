// few_rows.h -- the learned layers' products for a few rows (few_rows.cu).
#pragma once

#include "af2_internal.h"

namespace af2 {

// Up to this many rows the layers are bound by the read of the weights and by latency, and the
// CUDA-core kernel is used.
constexpr int kFewRows = 8;

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
