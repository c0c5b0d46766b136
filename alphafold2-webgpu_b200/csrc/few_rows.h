// few_rows.h -- the learned layers' products for a few rows (few_rows.cu).
#pragma once

#include "af2_internal.h"

namespace af2 {

// Over how many blocks a cluster shares the depth: while the SMs are not all busy and each block keeps
// 128 weight rows.  blocks: four rows by 32 columns each.
inline int few_rows_splits(int64_t blocks, int64_t inner, int sms) {
  int splits = 1;
  while (splits < 8 && blocks * splits * 2 <= sms && inner / (splits * 2) >= 128) splits *= 2;
  return splits;
}

// Whether a product (`gated`: the transition's first, of two weights) is small enough for the CUDA-core
// kernel, which starts and ends sooner than the tensor-core ones and reads f32 as it is.  Measured, us
// (few rows | tensor cores), whole transitions or one dense layer:
//   bf16 gated  256 -> 1024: 32 rows 10.4 | 12.9, 48 rows 15.6 | 13.2;  512 -> 2048: 8 rows 11.3 | 14.4,
//               16 rows 15.2 | 14.6;  1024 -> 4096: 4 rows 12.8 | 19.1, 8 rows 22.3 | 19.1
//   f32 gated   256 -> 1024: 96 rows 19.9 | 21.2, 128 rows 23.6 | 22.3;  1024 -> 4096: 16 rows 45 | 64, 24 rows 69 | 55
//   bf16 dense  512 -> 512: 64 rows 5.2 | 6.2, 96 rows 8.2 | 6.2;  1024 -> 4096: 4 rows 5.1 | 8.4, 8 rows 9.4 | 8.7;
//               4096 -> 1024: 8 rows 8.9 | 9.6, 16 rows 14.2 | 9.1;  32768 -> 512: 2 rows 15.1 | 13.5, 32 rows 100 | 14
//   f32 dense   512 -> 512: 128 rows 9.4 | 11.4, 192 rows 13.1 | 11.7;  4096 -> 1024: 16 rows 14.0 | 20.8, 48 rows
//               39.2 | 21.8;  65536 -> 128: 8 rows 26 | 37, 96 rows 189 | 52
// A transition's time grows with rows x weight, the tensor cores' hardly with the rows.  A dense layer takes as
// long as an SM's blocks one after the other, each its share of the depth and a fixed part worth 512 of it
// (half of that for one or two rows); the tensor cores' time grows with the weight in f32, whose terms they
// need.  Weight rows that are not 16-byte pieces are read one element at a time, which counts half as much
// again (293 -> 893, gated: bf16 24 rows 13.7 | 15.5, 32 rows 17.5 | 15.7).  Over 34 dense shapes of 64 to
// 65536 deep, 32 to 65536 wide, and 1 to 256 rows in either type, what this takes is 0.5 % above the faster
// kernel's time in the mean, 47 % at most.
inline bool few_rows(int64_t rows, int64_t inner, int64_t columns, int dtype, bool gated) {
  const bool f32 = dtype == AF2_F32, pieces = columns % (f32 ? 4 : 8) == 0;
  if (rows > 256) return false;
  if (gated) {
    const int64_t always = f32 ? 16 : 4, most = f32 ? 24 << 20 : 8 << 20;
    return (rows - always) * inner * columns <= (pieces ? most : most / 4 * 3);
  }
  constexpr int kSms = 148;
  const int64_t blocks = (rows + 3) / 4 * ((columns + 31) / 32);
  const int splits = few_rows_splits(blocks, inner, kSms);
  const int64_t depth = (inner + splits - 1) / splits, turns = (blocks * splits + kSms - 1) / kSms;
  const int64_t cost = turns * ((pieces ? depth : depth + depth / 2) + 512);
  return (rows <= 2 ? cost / 2 : cost) <= (f32 ? 4096 + inner * columns / 1024 : 2560);
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
