// layer_gemm.h -- the products behind the layers with learned weights.
#pragma once

#include "af2_internal.h"

namespace af2 {

// One 16-bit operand as TMA reads it: rows of `pitch` elements (a multiple of 8, 16-byte aligned).
// K-major: [outer][pitch] with k contiguous; MN-major: [k][pitch] with the outer index contiguous.
// pieces > 1: an f32 operand as that many bf16 terms (high to low), `piece_stride` elements apart.
struct GemmOperand {
  const void *ptr = nullptr;
  int64_t pitch = 0;
  bool mn_major = false;
  int64_t piece_stride = 0;
};

// How a tile leaves the accumulators.
enum GemmEpilogue {
  kEpilogueOut = 0,       // out = act(acc + bias) (+ residual), saved = act'(acc + bias)
  kEpilogueGate = 1,      // b[0], b[1] are the gate's and the value's weights: out = act(g) v,
                          // saved = v act'(g) and act(g): what the backward pass multiplies dh by (f32: g and v)
  kEpilogueGateBackward,  // acc = dh: out = dh times each of the two saved factors (dg and dv)
};

// Factors kept for the backward pass, rows of `pitch` elements; the second factor's plane `stride`
// elements after the first's.  f32 and f16 tensors keep f32 in `f32`.  bf16 ones keep 16 bits
// (layer_factor.cuh) in `half`; the gated transition's factors, of any size, with an exponent byte for
// every 16 columns of a row, four of them (two factors x two halves) as a word per row and 32 columns in
// `scale` [pitch / 32][scale_rows].
struct SavedPlanes {
  uint16_t *half = nullptr;
  uint32_t *scale = nullptr;
  float *f32 = nullptr;
  int64_t pitch = 0, stride = 0, scale_rows = 0;
};

struct LayerGemm {
  int64_t m = 0, n = 0, k = 0;  // n: of one batch entry (the gate: hidden channels)
  int segments = 1;             // sums over a[s] b[s], s < segments, each of depth k
  int batch = 1;                // products a[0] b[z] -> out[z], z < batch
  GemmOperand a[2], b[2];
  bool bf16 = false;            // the operands' type
  int pieces = 1;               // 1, or 3: f32 operands in bf16 terms
  GemmEpilogue epilogue = kEpilogueOut;
  int activation = 0;
  int out_dtype = 0;
  void *out[2] = {nullptr, nullptr};
  int64_t out_stride = 0;
  int64_t out_piece_stride = 0;              // f32 gate: out[0] is an operand of three terms this far apart
  const void *bias[2] = {nullptr, nullptr};  // of out_dtype, or NULL
  const void *residual = nullptr;            // of out_dtype
  int64_t residual_stride = 0;
  SavedPlanes saved;                         // written by Out and Gate, read by GateBackward
  float *column_partial = nullptr;           // GateBackward: [ceil(m / 32)][2 * saved.pitch] column sums, or NULL
  // layer_gemm_plan: the tile's width, the parts the depth is cut into and the split sums' bytes
  int tile_n = 0, splits = 0;
  int given = 0;  // which of the products given this is, or is rows of, from first_row on
  int64_t first_row = 0;
  uint64_t scratch_bytes = 0;
  uint8_t *scratch = nullptr;
};

// Row pitch (elements) of a 16-bit operand of `width` (rows begin on a 32-byte sector), and of the saved planes.
inline int64_t operand_pitch(int64_t width) { return align_up(width, 16); }
inline int64_t saved_pitch(int64_t width) { return align_up(width, 32); }

// Up to this many products of one type in a launch (more than one: kEpilogueOut with no bias, activation
// or residual).
constexpr int kMaxProducts = 4;  // three, and what is cut from one
// Fills in the plan, in which a product may have become two, in another order: g has room for
// kMaxProducts; returns how many there are.  Then each product with scratch_bytes needs scratch.
int layer_gemm_plan(LayerGemm *g, int count);
af2_status layer_gemm_launch(af2_ctx *ctx, const LayerGemm *g, int count, cudaStream_t stream);

// out[c] of the call's type = the sum over the chunks of partial[chunk * stride + c], f32, or with `rows`
// the rows of a tensor of the call's type.
struct ColumnSums {
  const void *partial = nullptr;
  int64_t chunks = 0, stride = 0, columns = 0;
  void *out = nullptr;
  bool rows = false;
};
constexpr int kMaxSums = 3;
// What is left after layer_gemm_launch, in one launch (none where there is nothing): the sums of the
// products that were split, and column sums.
af2_status layer_finish_launch(af2_ctx *ctx, int dtype, const LayerGemm *g, int count, const ColumnSums *sums,
                               int sum_count, cudaStream_t stream);

}  // namespace af2
