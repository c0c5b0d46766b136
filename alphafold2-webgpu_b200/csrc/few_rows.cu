// few_rows.cu -- y = act(x W + b) (+ r), or act(x Wg + bg) (x Wv + bv), for a
// few rows: one token, or one position of a small batch.
//
// Each weight is read once for four rows, so the read bounds it: 25 MB of a
// 1024 -> 4096 -> 1024 transition take 3.9 us at the copy rate.  More rows are
// further groups of four beside the first, whose reads find the weights in L2.  A block
// has 32 columns and sixteen warps over the depth; a lane reads 16 bytes of a
// weight row and keeps several such reads in flight.  With few columns a cluster
// of blocks shares the depth and adds up through distributed shared memory, in
// rank order.  The launch that follows another (the transition's second
// product) reads its first weights before it waits for the one before it.  One row of
// that transition: 11.1 us for both launches; 1024 -> 1024 alone 4.8, with the call.
#include <algorithm>
#include <type_traits>

#include "few_rows.h"
#include "layer_math.cuh"

namespace af2 {
namespace {

constexpr int COLS = 32, WARPS = 16, THREADS = 32 * WARPS;
constexpr int CHUNK = 1024;  // depth of x in shared memory at a time

struct Args {
  const void *x, *weight[2], *bias[2], *residual;
  void *out;
  int64_t x_stride, residual_stride, out_stride;
  int rows, inner, columns, activation, splits, follows;
};

// V consecutive weights of a row; zeros past the columns.
template <typename T, int V>
struct Piece {
  using Word = std::conditional_t<V == 1, T, uint4>;
  static __device__ __forceinline__ Word load(const T *p) {
    if constexpr (V == 1)
      return *p;
    else
      return __ldg(reinterpret_cast<const uint4 *>(p));
  }
  static __device__ __forceinline__ void values(const Word &w, float (&v)[V]) {
    if constexpr (V == 1) {
      v[0] = to_f32<T>(w);
    } else {
      const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = to_f32<T>(e[i]);
    }
  }
};

// A group of R rows per blockIdx.y (those past p.rows are zero in x), V weights per read; GATE: warps 0-7 have the gate, 8-15 the value.
// Two blocks fit an SM, so the second product's blocks stand ready, their reads issued, while the
// first's still run; that leaves a lane 64 registers: eight reads in flight, or four beside four rows'
// sums.  DEEP: one block, and eight reads with four rows too, which large weights need more (four rows
// of 512 -> 2048 -> 512: two blocks 9.9 us, one 13.2; of 1024 -> 4096 -> 1024: 19.3 and 13.4).
template <typename T, int V, int R, bool GATE, bool DEEP>
__global__ void __launch_bounds__(THREADS, DEEP ? 1 : 2) few_rows_kernel(const Args p) {
  constexpr int FLIGHT = R <= 2 || DEEP ? 8 : 4;
  constexpr int SETS = GATE ? 2 : 1, SET_WARPS = WARPS / SETS;
  constexpr int LANES = COLS / V;  // lanes on one weight row
  constexpr int DEPTH = 32 / LANES;  // weight rows of one read of a warp (= V)
  __shared__ float work[CHUNK * R];  // x, then the warps' sums
  __shared__ float total[SETS * R * COLS];
  __shared__ float others[7 * SETS * R * COLS];  // the cluster's other blocks' sums, in rank 0's memory
  static_assert(CHUNK >= WARPS * COLS, "the warps' sums fit where x was");
  float *const xs = work, *const part = work;
  using P = Piece<T, V>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = p.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int row0 = static_cast<int>(blockIdx.y) * R, rows = min(R, p.rows - row0);
  const int c_block = static_cast<int>(blockIdx.x) / p.splits * COLS;
  const int k0 = static_cast<int>(static_cast<int64_t>(p.inner) * rank / p.splits);
  const int k1 = static_cast<int>(static_cast<int64_t>(p.inner) * (rank + 1) / p.splits);
  const int set = GATE ? warp / SET_WARPS : 0, w = GATE ? warp % SET_WARPS : warp;
  const int col = c_block + (lane % LANES) * V;
  const bool in = col < p.columns;  // V > 1: the columns are a multiple of V
  const T *weight = static_cast<const T *>(set ? p.weight[1] : p.weight[0]) + col;
  const int first = k0 + w * DEPTH + lane / LANES;
  if (p.splits > 1) cluster_started();
  constexpr int STEP = SET_WARPS * DEPTH;  // from one read of a lane to its next

  typename P::Word buf[FLIGHT];
  auto fetch = [&](int k, int end) {
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i)
      if (in && k + i * STEP < end) buf[i] = P::load(weight + static_cast<int64_t>(k + i * STEP) * p.columns);
  };
  // chunks are CHUNK deep and the first read of each warp starts at its own place in the chunk
  if (p.follows) {
    // the launch before this one writes no weight, and waited itself for those before it
    fetch(first, min(k1, k0 + CHUNK));
    dependency_wait();
  } else {
    dependency_wait();
    fetch(first, min(k1, k0 + CHUNK));
  }

  float acc[R][V] = {};
  const T *x = static_cast<const T *>(p.x) + static_cast<int64_t>(row0) * p.x_stride;
  for (int c0 = k0; c0 < k1; c0 += CHUNK) {
    const int end = min(k1, c0 + CHUNK);
    if (c0 != k0) __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
      for (int k = threadIdx.x; k < end - c0; k += THREADS)
        xs[k * R + r] = r < rows ? to_f32<T>(x[r * p.x_stride + c0 + k]) : 0.f;
    __syncthreads();
    for (int k = first + (c0 - k0); k < end; k += FLIGHT * STEP) {
      if (k != first) fetch(k, end);
#pragma unroll
      for (int i = 0; i < FLIGHT; ++i) {
        const int ki = k + i * STEP;
        if (!in || ki >= end) break;
        float wv[V], xv[R];
        P::values(buf[i], wv);
#pragma unroll
        for (int r = 0; r < R; ++r) xv[r] = xs[(ki - c0) * R + r];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int v = 0; v < V; ++v) acc[r][v] = fmaf(xv[r], wv[v], acc[r][v]);
      }
    }
  }

  // over the warp's weight rows: halving the columns at each exchange leaves one column a lane
#pragma unroll
  for (int o = 16, half = V / 2; half >= 1; o >>= 1, half >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < half; ++v) {
        const float keep = upper ? acc[r][v + half] : acc[r][v], send = upper ? acc[r][v] : acc[r][v + half];
        acc[r][v] = keep + __shfl_xor_sync(kFull, send, o);
      }
  }
  // the column: bit i of lane / LANES (from the top) chose the upper half of what was left
  const int mine = (lane % LANES) * V + lane / LANES;
  __syncthreads();  // every warp is done with x
#pragma unroll
  for (int r = 0; r < R; ++r) part[(warp * R + r) * COLS + mine] = acc[r][0];
  __syncthreads();
  // blocks of a cluster are scheduled together, but one may be here before rank 0 has begun
  if (p.splits > 1) cluster_wait_started();
  for (int i = threadIdx.x; i < SETS * R * COLS; i += THREADS) {
    const int s = i / (R * COLS), at = i - s * (R * COLS);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < SET_WARPS; ++j) sum += part[(s * SET_WARPS + j) * R * COLS + at];
    if (rank == 0) {
      total[i] = sum;
    } else {
      uint32_t there;
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;"
                   : "=r"(there)
                   : "r"(smem_u32(&others[(rank - 1) * SETS * R * COLS + i])));
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(sum) : "memory");
    }
  }
  if (p.splits > 1) {
    cluster_sync_all();  // the others' sums have arrived
    if (rank != 0) return;
    for (int i = threadIdx.x; i < SETS * R * COLS; i += THREADS) {
      float sum = total[i];  // (written by this thread)
      for (int s = 1; s < p.splits; ++s) sum += others[(s - 1) * SETS * R * COLS + i];
      total[i] = sum;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * COLS; i += THREADS) {
    const int r = i / COLS, c = c_block + (i - r * COLS);
    if (r >= rows || c >= p.columns) continue;
    float y = total[i];
    if (p.bias[0]) y += to_f32<T>(static_cast<const T *>(p.bias[0])[c]);
    with_activation(p.activation, [&](auto act) { y = activate2<decltype(act)::value, sizeof(T) == 2>(f2(y)).x; });
    if constexpr (GATE) {
      float v = total[R * COLS + i];
      if (p.bias[1]) v += to_f32<T>(static_cast<const T *>(p.bias[1])[c]);
      y *= v;
    }
    const int64_t row = row0 + r;
    if (p.residual) y += to_f32<T>(static_cast<const T *>(p.residual)[row * p.residual_stride + c]);
    static_cast<T *>(p.out)[row * p.out_stride + c] = from_f32<T>(y);
  }
}

template <typename T, int V, int R, bool GATE, bool DEEP = false>
cudaError_t launch(const Args &p, int blocks, cudaStream_t stream) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(blocks * p.splits), static_cast<unsigned>((p.rows + R - 1) / R));
  config.blockDim = dim3(THREADS);
  config.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(p.splits), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, few_rows_kernel<T, V, R, GATE, DEEP>, p);
}

template <typename T, int V, bool GATE>
cudaError_t launch_rows(const Args &p, int blocks, cudaStream_t stream) {
  if (p.rows == 1) return launch<T, V, 1, GATE>(p, blocks, stream);
  if (p.rows == 2) return launch<T, V, 2, GATE>(p, blocks, stream);
  if (static_cast<int64_t>(p.inner) * p.columns >= 1 << 21) return launch<T, V, 4, GATE, true>(p, blocks, stream);
  return launch<T, V, 4, GATE>(p, blocks, stream);
}

}  // namespace

af2_status few_rows_launch(af2_ctx *ctx, const FewRows &f, cudaStream_t stream) {
  const bool gate = f.weight[1] != nullptr;
  Args p{f.x, {f.weight[0], f.weight[1]}, {f.bias[0], f.bias[1]}, f.residual, f.out, f.x_stride, f.residual_stride,
         f.out_stride, static_cast<int>(f.rows), static_cast<int>(f.inner), static_cast<int>(f.columns), f.activation, 1,
         f.follows};
  const int blocks = (p.columns + COLS - 1) / COLS;
  p.splits = few_rows_splits((f.rows + 3) / 4 * blocks, f.inner, ctx->sm_count);
  LaunchScope scope(ctx, stream, kProfLayerGemm);
  cudaError_t e = cudaSuccess;
  with_element(f.dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr int V = 16 / sizeof(T);
    bool wide = p.columns % V == 0;
    for (int i = 0; i < (gate ? 2 : 1); ++i) wide &= reinterpret_cast<uintptr_t>(f.weight[i]) % 16 == 0;
    if (wide)
      e = gate ? launch_rows<T, V, true>(p, blocks, stream) : launch_rows<T, V, false>(p, blocks, stream);
    else
      e = gate ? launch_rows<T, 1, true>(p, blocks, stream) : launch_rows<T, 1, false>(p, blocks, stream);
  });
  if (e != cudaSuccess) return cuda_fail(ctx, e, "layer product of a few rows");
  return AF2_OK;
}

}  // namespace af2
