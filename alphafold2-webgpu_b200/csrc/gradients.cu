// gradients.cu -- the global norm of a set of tensors, and their clipping.
//
//   norm = sqrt(sum of squares), factor = min(1, limit / (norm + 1e-6)),
//   out = factor * in
//
// The set's table goes to the device inside kernel arguments (no host buffer
// outlives the call).  The elements are cut into chunks, each block takes a
// contiguous range of chunks and sums their squares in f64, and one block adds
// the blocks' sums in order: no atomics, so the result depends on the sizes
// alone.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "af2_internal.h"
#include "layer_math.cuh"

namespace af2 {
namespace {

constexpr int kChunk = 8192;        // elements
constexpr int kNormThreads = 512;
constexpr int kMaxBlocks = 1024;
constexpr int kUpload = 64;         // table entries per upload launch

struct SetEntry {
  const void *in;
  void *out;
  int64_t count;
  int64_t first_chunk;  // chunks of the tensors before this one
  int64_t dtype;
};

struct Upload {
  SetEntry entry[kUpload];
  SetEntry *table;
  int count;
};

__global__ void upload_kernel(const __grid_constant__ Upload u) {
  if (threadIdx.x < u.count) u.table[threadIdx.x] = u.entry[threadIdx.x];
}

// Calls f(entry, first element, elements) for this block's chunks, in order.
template <typename F>
__device__ __forceinline__ void for_chunks(const SetEntry *table, int tensors, int64_t chunks, F &&f) {
  const int64_t begin = chunks * blockIdx.x / gridDim.x, end = chunks * (blockIdx.x + 1) / gridDim.x;
  if (begin == end) return;
  int lo = 0, hi = tensors - 1;  // the last tensor whose first chunk is at or before `begin`
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (table[mid].first_chunk <= begin)
      lo = mid;
    else
      hi = mid - 1;
  }
  for (int64_t c = begin; c < end; ++c) {
    while (lo + 1 < tensors && table[lo + 1].first_chunk <= c) ++lo;
    const int64_t first = (c - table[lo].first_chunk) * kChunk;
    f(table[lo], first, static_cast<int>(min(static_cast<int64_t>(kChunk), table[lo].count - first)));
  }
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T *p, int n) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += kNormThreads) {
    const double v = static_cast<double>(to_f32<T>(p[i]));
    sum = fma(v, v, sum);
  }
  return sum;
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double warps[kNormThreads / 32];
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  double total = 0.0;
  for (int w = 0; w < kNormThreads / 32; ++w) total += warps[w];
  return total;
}

__global__ void __launch_bounds__(kNormThreads) squares_kernel(const SetEntry *table, int tensors, int64_t chunks,
                                                                double *partial) {
  double sum = 0.0;
  for_chunks(table, tensors, chunks, [&](const SetEntry &e, int64_t first, int n) {
    if (e.dtype == AF2_F32)
      sum += chunk_squares(static_cast<const float *>(e.in) + first, n);
    else if (e.dtype == AF2_F16)
      sum += chunk_squares(static_cast<const __half *>(e.in) + first, n);
    else
      sum += chunk_squares(static_cast<const __nv_bfloat16 *>(e.in) + first, n);
  });
  const double total = block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

__global__ void __launch_bounds__(kNormThreads) finish_kernel(const double *partial, int blocks, float limit,
                                                               float *norm, float *factor) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < blocks; i += kNormThreads) sum += partial[i];
  const double total = block_sum(sum);
  if (threadIdx.x == 0) {
    const float n = static_cast<float>(sqrt(total));
    *norm = n;
    const float f = limit / (n + 1e-6f);
    *factor = f > 1.f ? 1.f : f;  // a NaN stays one
  }
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T *in, T *out, int n, float factor) {
  for (int i = threadIdx.x; i < n; i += kNormThreads) out[i] = from_f32<T>(to_f32<T>(in[i]) * factor);
}

__global__ void __launch_bounds__(kNormThreads) scale_kernel(const SetEntry *table, int tensors, int64_t chunks,
                                                              const float *factor) {
  const float f = *factor;
  for_chunks(table, tensors, chunks, [&](const SetEntry &e, int64_t first, int n) {
    if (e.in == e.out && f == 1.f) return;
    if (e.dtype == AF2_F32)
      chunk_scale(static_cast<const float *>(e.in) + first, static_cast<float *>(e.out) + first, n, f);
    else if (e.dtype == AF2_F16)
      chunk_scale(static_cast<const __half *>(e.in) + first, static_cast<__half *>(e.out) + first, n, f);
    else
      chunk_scale(static_cast<const __nv_bfloat16 *>(e.in) + first, static_cast<__nv_bfloat16 *>(e.out) + first, n,
                  f);
  });
}

constexpr size_t kOffFactor = 0, kOffPartial = 256, kOffTable = kOffPartial + 8 * kMaxBlocks;

}  // namespace

uint64_t gradient_norm_workspace_bytes(int64_t count) { return align_up(kOffTable + sizeof(SetEntry) * count, 256); }

af2_status gradient_norm_launch(af2_ctx *ctx, const af2_tensor_ref *tensors, const af2_tensor_ref *outputs,
                                int64_t count, bool clip, float max_norm, float *norm, void *workspace,
                                cudaStream_t stream) {
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  float *factor = reinterpret_cast<float *>(ws + kOffFactor);
  double *partial = reinterpret_cast<double *>(ws + kOffPartial);
  SetEntry *table = reinterpret_cast<SetEntry *>(ws + kOffTable);
  auto failed = [&](const char *what, af2_status *st) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) *st = cuda_fail(ctx, e, what);
    return e != cudaSuccess;
  };
  af2_status st = AF2_OK;
  int64_t chunks = 0;
  int used = 0;
  Upload u;
  auto flush = [&](int n) {
    u.table = table + (used - n);
    u.count = n;
    LaunchScope scope(ctx, stream, kProfGradientNorm);
    upload_kernel<<<1, kUpload, 0, stream>>>(u);
    return !failed("gradient table", &st);
  };
  int pending = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (tensors[i].count == 0) continue;
    u.entry[pending++] = {tensors[i].data, outputs ? outputs[i].data : tensors[i].data, tensors[i].count, chunks,
                          tensors[i].dtype};
    chunks += (tensors[i].count + kChunk - 1) / kChunk;
    ++used;
    if (pending == kUpload) {
      if (!flush(pending)) return st;
      pending = 0;
    }
  }
  if (pending && !flush(pending)) return st;
  const int blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({chunks, 4 * ctx->sm_count, kMaxBlocks})));
  {
    LaunchScope scope(ctx, stream, kProfGradientNorm);
    squares_kernel<<<blocks, kNormThreads, 0, stream>>>(table, used, chunks, partial);
    if (failed("gradient squares", &st)) return st;
  }
  {
    LaunchScope scope(ctx, stream, kProfGradientNorm);
    finish_kernel<<<1, kNormThreads, 0, stream>>>(partial, blocks, std::min(max_norm, FLT_MAX), norm, factor);
    if (failed("gradient norm", &st)) return st;
  }
  if (clip && chunks) {
    LaunchScope scope(ctx, stream, kProfGradientNorm);
    scale_kernel<<<blocks, kNormThreads, 0, stream>>>(table, used, chunks, factor);
    if (failed("gradient scaling", &st)) return st;
  }
  return st;
}

}  // namespace af2
