// few_rows.h -- the learned layers' products for a few rows (few_rows.cu).
#pragma once

#include "af2_internal.h"

namespace af2 {

// Whether a product (`gated`: the transition's first, of two weights) is small enough for the CUDA-core
// kernel, which starts and ends sooner than the tensor-core ones and reads f32 as it is.  Its time grows
// with rows x weight, theirs hardly with the rows: they meet at some rows for any weight and more for
// small ones.  Measured, us (few rows | tensor cores), whole transitions or one dense layer:
//   bf16 gated  256 -> 1024: 32 rows 10.4 | 12.9, 48 rows 15.6 | 13.2;  512 -> 2048: 8 rows 11.3 | 14.4,
//               16 rows 15.2 | 14.6;  1024 -> 4096: 4 rows 12.8 | 19.1, 8 rows 22.3 | 19.1
//   bf16 dense  512 -> 512: 64 rows 5.1 | 6.2, 96 rows 8.0 | 6.2;  1024 -> 4096: 4 rows 5.0 | 8.7, 8 rows 9.3 | 8.6
//   f32 gated   256 -> 1024: 96 rows 19.9 | 21.2, 128 rows 23.6 | 22.3;  1024 -> 4096: 16 rows 45 | 64, 24 rows 69 | 55
//   f32 dense   512 -> 512: 128 rows 9.3 | 11.3, 192 rows 13.0 | 11.7;  1024 -> 4096: 16 rows 17 | 26, 24 rows 24 | 21
// Weight rows that are not 16-byte pieces are read one element at a time (293 -> 893, gated: bf16 24 rows
// 13.7 | 15.5, 32 rows 17.5 | 15.7; f32 48 rows 21.3 | 21.7, 96 rows 27.6 | 22.7).
// A dense layer's times part where the kernel's blocks (four rows by 32 columns) are more than the SMs hold
// at a time, two each, or one where the weight is large; the f32 products take twice and four times that.
inline bool few_rows(int64_t rows, int64_t inner, int64_t columns, int dtype, bool gated) {
  const bool f32 = dtype == AF2_F32, pieces = columns % (f32 ? 4 : 8) == 0;
  if (rows > 256) return false;
  if (gated) {
    const int64_t always = f32 ? 16 : 4, most = f32 ? 24 << 20 : 8 << 20;
    return (rows - always) * inner * columns <= (pieces ? most : most / 4 * 3);
  }
  const int64_t held = f32 ? 592 : inner * columns >= 1 << 21 ? 148 : 296;
  return rows <= 4 || (rows + 3) / 4 * ((columns + 31) / 32) <= (pieces ? held : held / 4 * 3);
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
