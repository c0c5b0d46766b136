// gated_fused.h -- the gated transition in one kernel (gated_fused.cu).
#pragma once

#include "layer_gemm.h"

namespace af2 {

// y = (act(x Wg + bg) (x Wv + bv)) Wo + bo (+ r) for 16-bit tensors that TMA can address.
struct GatedFused {
  int64_t rows = 0, channels = 0, hidden = 0;
  int dtype = 0, activation = 0;
  GemmOperand x, gate, value, output;  // x [rows][pitch], gate and value [channels][pitch], output [hidden][pitch]
  const void *gate_bias = nullptr, *value_bias = nullptr, *output_bias = nullptr, *residual = nullptr;
  int64_t residual_stride = 0, out_stride = 0;
  void *out = nullptr;
};
// Whether the kernel covers the call, and is the faster one for it.
bool gated_fused_fits(const GatedFused &f);    // its sizes and type
bool gated_fused_covers(const GatedFused &f);  // and its output and residual
af2_status gated_fused_launch(af2_ctx *ctx, const GatedFused &f, cudaStream_t stream);

}  // namespace af2
