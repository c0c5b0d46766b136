// dense.cu -- the dense layer and the gated transition, forward and backward.
//
//   dense:  z = x W + b, y = act(z) (+ r);   dz = dy act'(z), dx = dz W^T,
//           dW = x^T dz, db = column sums of dz
//   gated:  g = x Wg + bg, v = x Wv + bv, h = act(g) v, y = h Wo + bo (+ r);
//           dh = dy Wo^T, dv = dh act(g), dg = dh v act'(g),
//           dx = dg Wg^T + dv Wv^T, dWg = x^T dg, dWv = x^T dv, dWo = h^T dy
//
// Simplest form: one tiled product in f32 on the CUDA cores for every operand
// order, its sums kept in f32 in the scratch, and one elementwise pass for
// each of the rest.
#include <type_traits>

#include "af2_internal.h"
#include "layer_math.cuh"

namespace af2 {
namespace {

// C[m][n] (+)= sum_k A(m, k) B(k, n); A(m, k) = a[m * a_m + k * a_k], B(k, n) = b[k * b_k + n * b_n].
struct Product {
  const void *a, *b;
  int64_t a_m, a_k, b_k, b_n;
  int64_t m, n, k;
  float *c;  // [m][n]
  int accumulate;
};

constexpr int kTile = 64, kDepth = 16;

template <typename TA, typename TB>
__global__ void __launch_bounds__(256) product_kernel(const Product p) {
  __shared__ float sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kTile;
  const int64_t n0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const TA *a = static_cast<const TA *>(p.a);
  const TB *b = static_cast<const TB *>(p.b);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kDepth) {
    for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
      // the contiguous index of each operand runs fastest over the threads
      const int am = p.a_k == 1 ? i / kDepth : i % kTile, ak = p.a_k == 1 ? i % kDepth : i / kTile;
      const int64_t m = m0 + am, ka = k0 + ak;
      sa[ak][am] = m < p.m && ka < p.k ? to_f32<TA>(a[m * p.a_m + ka * p.a_k]) : 0.f;
      const int bn = p.b_k == 1 ? i / kDepth : i % kTile, bk = p.b_k == 1 ? i % kDepth : i / kTile;
      const int64_t n = n0 + bn, kb = k0 + bk;
      sb[bk][bn] = n < p.n && kb < p.k ? to_f32<TB>(b[kb * p.b_k + n * p.b_n]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty + 16 * i], sb[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m >= p.m || n >= p.n) continue;
      float *c = p.c + m * p.n + n;
      *c = p.accumulate ? *c + acc[i][j] : acc[i][j];
    }
}

__device__ __forceinline__ int64_t grid_index() {
  return static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
}
__device__ __forceinline__ int64_t grid_stride() { return static_cast<int64_t>(gridDim.x) * blockDim.x; }

// out = act(acc + bias) (+ residual); saved = acc + bias
template <typename T, int ACT>
__global__ void dense_finish_kernel(const float *acc, int64_t rows, int64_t cols, const T *bias, const T *residual,
                                    int64_t residual_stride, T *out, int64_t out_stride, float *saved) {
  for (int64_t i = grid_index(); i < rows * cols; i += grid_stride()) {
    const int64_t r = i / cols, c = i - r * cols;
    const float z = acc[i] + (bias ? to_f32<T>(bias[c]) : 0.f);
    if (saved) saved[i] = z;
    float y = activate<ACT>(z);
    if (residual) y += to_f32<T>(residual[r * residual_stride + c]);
    out[r * out_stride + c] = from_f32<T>(y);
  }
}

// dz = dy act'(z), in f32
template <typename T, int ACT>
__global__ void dense_slope_kernel(const T *dy, int64_t dy_stride, const float *z, int64_t rows, int64_t cols,
                                   float *dz) {
  for (int64_t i = grid_index(); i < rows * cols; i += grid_stride()) {
    const int64_t r = i / cols, c = i - r * cols;
    float value, slope = 1.f;
    if (ACT != AF2_ACTIVATION_NONE) activate_slope<ACT>(z[i], value, slope);
    dz[i] = to_f32<T>(dy[r * dy_stride + c]) * slope;
  }
}

// saved [rows][2 cols] = the biased pre-activations (gate, value); h = act(gate) value
template <typename T, int ACT>
__global__ void gate_kernel(const float *g, const float *v, int64_t rows, int64_t cols, const T *bg, const T *bv,
                            T *h, float *saved) {
  for (int64_t i = grid_index(); i < rows * cols; i += grid_stride()) {
    const int64_t r = i / cols, c = i - r * cols;
    const float gate = g[i] + (bg ? to_f32<T>(bg[c]) : 0.f), value = v[i] + (bv ? to_f32<T>(bv[c]) : 0.f);
    if (saved) {
      saved[r * 2 * cols + c] = gate;
      saved[r * 2 * cols + cols + c] = value;
    }
    h[i] = from_f32<T>(activate<ACT>(gate) * value);
  }
}

// dh [rows][cols] and saved [rows][2 cols] -> dgv [rows][2 cols] (dg, dv) and h
template <typename T, int ACT>
__global__ void gate_backward_kernel(const float *dh, const float *saved, int64_t rows, int64_t cols, float *dgv,
                                     T *h) {
  for (int64_t i = grid_index(); i < rows * cols; i += grid_stride()) {
    const int64_t r = i / cols, c = i - r * cols;
    const float g = saved[r * 2 * cols + c], v = saved[r * 2 * cols + cols + c];
    float value, slope;
    activate_slope<ACT>(g, value, slope);
    dgv[r * 2 * cols + c] = dh[i] * v * slope;
    dgv[r * 2 * cols + cols + c] = dh[i] * value;
    h[i] = from_f32<T>(value * v);
  }
}

// rounds rows of f32 sums to T
template <typename T>
__global__ void round_kernel(const float *src, int64_t rows, int64_t cols, T *dst, int64_t dst_stride) {
  for (int64_t i = grid_index(); i < rows * cols; i += grid_stride()) {
    const int64_t r = i / cols, c = i - r * cols;
    dst[r * dst_stride + c] = from_f32<T>(src[i]);
  }
}

// dst[c] = sum over the rows of src; one block per 32 columns, rows strided over its 32 warps
template <typename TS, typename T>
__global__ void __launch_bounds__(1024) column_sum_kernel(const TS *src, int64_t stride, int64_t rows, int64_t cols,
                                                          T *dst) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum = 0.f;
  if (c < cols)
    for (int64_t r = warp; r < rows; r += 32) sum += to_f32<TS>(src[r * stride + c]);
  part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < cols) {
    float total = 0.f;
    for (int w = 0; w < 32; ++w) total += part[w][lane];
    dst[c] = from_f32<T>(total);
  }
}

struct Launcher {
  af2_ctx *ctx;
  cudaStream_t stream;
  af2_status status = AF2_OK;

  void check(const char *what) {
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess && status == AF2_OK) status = cuda_fail(ctx, e, what);
  }
  int blocks(int64_t elements) const {
    return static_cast<int>(std::min<int64_t>((elements + 255) / 256, 16 * ctx->sm_count));
  }
  template <typename TA, typename TB>
  void product(const Product &p) {
    LaunchScope scope(ctx, stream, kProfLayerGemm);
    const dim3 grid(static_cast<unsigned>((p.m + kTile - 1) / kTile), static_cast<unsigned>((p.n + kTile - 1) / kTile));
    product_kernel<TA, TB><<<grid, 256, 0, stream>>>(p);
    check("layer product");
  }
  template <typename F>
  void elementwise(F &&f) {
    LaunchScope scope(ctx, stream, kProfLayerElementwise);
    f();
    check("layer elementwise kernel");
  }
  void zero(void *ptr, size_t bytes) {
    if (!ptr || status != AF2_OK) return;
    if (cudaError_t e = cudaMemsetAsync(ptr, 0, bytes, stream); e != cudaSuccess) status = cuda_fail(ctx, e, "zero");
  }
};

size_t element_size(int dtype) { return dtype == AF2_F32 ? 4 : 2; }
uint64_t part(uint64_t bytes) { return align_up(bytes, 256); }

}  // namespace

uint64_t dense_saved_bytes(int64_t rows, int64_t columns, int dtype, int activation) {
  return activation == AF2_ACTIVATION_NONE ? 0 : 4ull * rows * columns;
}
uint64_t dense_workspace_bytes(int64_t rows, int64_t inner, int64_t columns, int dtype, int activation,
                               bool backward) {
  if (!backward) return part(4ull * rows * columns);
  return part(4ull * rows * columns) + part(4ull * rows * inner) + part(4ull * inner * columns);
}
uint64_t gated_saved_bytes(int64_t rows, int64_t hidden, int dtype) { return 8ull * rows * hidden; }
uint64_t gated_workspace_bytes(int64_t rows, int64_t channels, int64_t hidden, int dtype, bool backward) {
  const uint64_t h = part(element_size(dtype) * rows * hidden);
  if (!backward) return h + 2 * part(4ull * rows * hidden) + part(4ull * rows * channels);
  return h + part(4ull * rows * hidden) + part(8ull * rows * hidden) + part(4ull * rows * channels) +
         part(4ull * channels * hidden);
}

af2_status dense_forward_launch(af2_ctx *ctx, const DenseForward &p, void *workspace, cudaStream_t stream) {
  Launcher l{ctx, stream};
  float *acc = static_cast<float *>(workspace);
  with_element(p.dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    l.product<T, T>({p.x, p.weight, p.x_stride, 1, p.columns, 1, p.rows, p.columns, p.inner, acc, 0});
    with_activation(p.activation, [&](auto act) {
      l.elementwise([&] {
        dense_finish_kernel<T, act.value><<<l.blocks(p.rows * p.columns), 256, 0, stream>>>(
            acc, p.rows, p.columns, static_cast<const T *>(p.bias), static_cast<const T *>(p.residual),
            p.residual_stride, static_cast<T *>(p.out), p.out_stride,
            act.value == AF2_ACTIVATION_NONE ? nullptr : static_cast<float *>(p.saved));
      });
    });
  });
  return l.status;
}

af2_status dense_backward_launch(af2_ctx *ctx, const DenseBackward &p, void *workspace, cudaStream_t stream) {
  Launcher l{ctx, stream};
  const size_t e = element_size(p.dtype);
  if (p.rows == 0) {
    l.zero(p.d_weight, e * p.inner * p.columns);
    l.zero(p.d_bias, e * p.columns);
    return l.status;
  }
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  float *dz = reinterpret_cast<float *>(ws);
  float *dx = reinterpret_cast<float *>(ws + part(4ull * p.rows * p.columns));
  float *dw = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(dx) + part(4ull * p.rows * p.inner));
  with_element(p.dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    with_activation(p.activation, [&](auto act) {
      l.elementwise([&] {
        dense_slope_kernel<T, act.value><<<l.blocks(p.rows * p.columns), 256, 0, stream>>>(
            static_cast<const T *>(p.d_out), p.d_out_stride, static_cast<const float *>(p.saved), p.rows, p.columns,
            dz);
      });
    });
    if (p.d_x) {
      l.product<float, T>({dz, p.weight, p.columns, 1, 1, p.columns, p.rows, p.inner, p.columns, dx, 0});
      l.elementwise([&] {
        round_kernel<T><<<l.blocks(p.rows * p.inner), 256, 0, stream>>>(dx, p.rows, p.inner, static_cast<T *>(p.d_x),
                                                                        p.d_x_stride);
      });
    }
    if (p.d_weight) {
      l.product<T, float>({p.x, dz, 1, p.x_stride, p.columns, 1, p.inner, p.columns, p.rows, dw, 0});
      l.elementwise([&] {
        round_kernel<T><<<l.blocks(p.inner * p.columns), 256, 0, stream>>>(dw, p.inner, p.columns,
                                                                           static_cast<T *>(p.d_weight), p.columns);
      });
    }
    if (p.d_bias)
      l.elementwise([&] {
        column_sum_kernel<float, T><<<static_cast<unsigned>((p.columns + 31) / 32), 1024, 0, stream>>>(
            dz, p.columns, p.rows, p.columns, static_cast<T *>(p.d_bias));
      });
  });
  return l.status;
}

af2_status gated_forward_launch(af2_ctx *ctx, const GatedForward &p, void *workspace, cudaStream_t stream) {
  Launcher l{ctx, stream};
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  float *g = reinterpret_cast<float *>(ws + part(element_size(p.dtype) * p.rows * p.hidden));
  float *v = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(g) + part(4ull * p.rows * p.hidden));
  float *y = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(v) + part(4ull * p.rows * p.hidden));
  with_element(p.dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    T *h = reinterpret_cast<T *>(ws);
    l.product<T, T>({p.x, p.w.gate_weight, p.x_stride, 1, p.hidden, 1, p.rows, p.hidden, p.channels, g, 0});
    l.product<T, T>({p.x, p.w.value_weight, p.x_stride, 1, p.hidden, 1, p.rows, p.hidden, p.channels, v, 0});
    with_activation(p.activation, [&](auto act) {
      l.elementwise([&] {
        gate_kernel<T, act.value><<<l.blocks(p.rows * p.hidden), 256, 0, stream>>>(
            g, v, p.rows, p.hidden, static_cast<const T *>(p.w.gate_bias), static_cast<const T *>(p.w.value_bias), h,
            static_cast<float *>(p.saved));
      });
    });
    l.product<T, T>({h, p.w.output_weight, p.hidden, 1, p.channels, 1, p.rows, p.channels, p.hidden, y, 0});
    l.elementwise([&] {
      dense_finish_kernel<T, AF2_ACTIVATION_NONE><<<l.blocks(p.rows * p.channels), 256, 0, stream>>>(
          y, p.rows, p.channels, static_cast<const T *>(p.w.output_bias), static_cast<const T *>(p.residual),
          p.residual_stride, static_cast<T *>(p.out), p.out_stride, nullptr);
    });
  });
  return l.status;
}

af2_status gated_backward_launch(af2_ctx *ctx, const GatedBackward &p, void *workspace, cudaStream_t stream) {
  Launcher l{ctx, stream};
  const size_t e = element_size(p.dtype);
  if (p.rows == 0) {
    const size_t w = e * p.channels * p.hidden;
    l.zero(p.g.gate_weight, w);
    l.zero(p.g.value_weight, w);
    l.zero(p.g.output_weight, w);
    l.zero(p.g.gate_bias, e * p.hidden);
    l.zero(p.g.value_bias, e * p.hidden);
    l.zero(p.g.output_bias, e * p.channels);
    return l.status;
  }
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  float *dh = reinterpret_cast<float *>(ws + part(e * p.rows * p.hidden));
  float *dgv = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(dh) + part(4ull * p.rows * p.hidden));
  float *dx = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(dgv) + part(8ull * p.rows * p.hidden));
  float *dw = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(dx) + part(4ull * p.rows * p.channels));
  const int64_t c = p.channels, hid = p.hidden;
  with_element(p.dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    T *h = reinterpret_cast<T *>(ws);
    auto round_to = [&](const float *src, int64_t rows, int64_t cols, void *dst, int64_t stride) {
      l.elementwise([&] {
        round_kernel<T><<<l.blocks(rows * cols), 256, 0, stream>>>(src, rows, cols, static_cast<T *>(dst), stride);
      });
    };
    l.product<T, T>({p.d_out, p.w.output_weight, p.d_out_stride, 1, 1, c, p.rows, hid, c, dh, 0});
    with_activation(p.activation, [&](auto act) {
      l.elementwise([&] {
        gate_backward_kernel<T, act.value><<<l.blocks(p.rows * hid), 256, 0, stream>>>(
            dh, static_cast<const float *>(p.saved), p.rows, hid, dgv, h);
      });
    });
    if (p.g.x) {
      l.product<float, T>({dgv, p.w.gate_weight, 2 * hid, 1, 1, hid, p.rows, c, hid, dx, 0});
      l.product<float, T>({dgv + hid, p.w.value_weight, 2 * hid, 1, 1, hid, p.rows, c, hid, dx, 1});
      round_to(dx, p.rows, c, p.g.x, p.d_x_stride);
    }
    for (int i = 0; i < 2; ++i) {
      void *dst = i ? p.g.value_weight : p.g.gate_weight, *bias = i ? p.g.value_bias : p.g.gate_bias;
      if (dst) {
        l.product<T, float>({p.x, dgv + i * hid, 1, p.x_stride, 2 * hid, 1, c, hid, p.rows, dw, 0});
        round_to(dw, c, hid, dst, hid);
      }
      if (bias)
        l.elementwise([&] {
          column_sum_kernel<float, T><<<static_cast<unsigned>((hid + 31) / 32), 1024, 0, stream>>>(
              dgv + i * hid, 2 * hid, p.rows, hid, static_cast<T *>(bias));
        });
    }
    if (p.g.output_weight) {
      l.product<T, T>({h, p.d_out, 1, hid, p.d_out_stride, 1, hid, c, p.rows, dw, 0});
      round_to(dw, hid, c, p.g.output_weight, c);
    }
    if (p.g.output_bias)
      l.elementwise([&] {
        column_sum_kernel<T, T><<<static_cast<unsigned>((c + 31) / 32), 1024, 0, stream>>>(
            static_cast<const T *>(p.d_out), p.d_out_stride, p.rows, c, static_cast<T *>(p.g.output_bias));
      });
  });
  return l.status;
}

}  // namespace af2
