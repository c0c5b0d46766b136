// gradients.cu -- the global norm of a set of tensors, and their clipping.
//
//   norm = sqrt(sum of squares), factor = min(1, limit / (norm + 1e-6)),
//   out = factor * in
//
// One cooperative launch.  The set is cut into chunks of 16 KB, and each block
// takes a contiguous range of them: it sums their squares, the grid meets, every
// block adds all blocks' sums in the same order (no atomics: the result depends
// on the sizes alone) and scales its own chunks, the last read first, because
// those are still in L2.  A set is read once for the norm, and again, as far as it
// has left the 126 MB of L2, for the scaling: 201 MB of bf16 take 107 us, 93 in a
// launch alone, whose 452 MB of DRAM traffic are 59 % of that memory's rate (69 us),
// so that memory is not all that bounds it; the norm of 0.8 MB 6.2 us, a launch and
// the grid's meeting.
//
// Squares are summed in f64.  Eight elements at a time are first summed in f32,
// whose rounding (2^-24 of the eight) is far below f32's own once the sums of
// many are added; where that sum overflows or is so small that squares may
// have vanished, the eight are squared in f64.
//
// The set's table goes to the device inside the kernel's arguments (no host
// buffer outlives the call), or, when it is longer than those can hold, through
// the scratch.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "af2_internal.h"
#include "layer_math.cuh"

namespace af2 {
namespace {

constexpr int kThreads = 256, kBlocksPerSm = 6;
constexpr int kChunkBytes = 16384;
constexpr int kVectors = kChunkBytes / 16 / kThreads;  // 16-byte loads of a thread per chunk
constexpr int kInline = 960;                           // table entries in the kernel's arguments

struct SetEntry {
  const void *in;
  void *out;
  int64_t count;
  uint32_t first_chunk;  // chunks of the tensors before this one
  uint32_t dtype;
};
static_assert(sizeof(SetEntry) == 32, "");

template <int N>
struct Table {
  SetEntry entry[N];
};
struct Set {
  const SetEntry *table;  // NULL: the entries are in the arguments
  double *partial;        // one per block
  float *norm;
  uint32_t tensors, chunks;
  float limit;
  int clip;
};

template <int N>
__global__ void upload_kernel(const __grid_constant__ Table<N> t, SetEntry *dst, int count) {
  for (int i = threadIdx.x; i < count; i += blockDim.x) dst[i] = t.entry[i];
}

// The tensor that chunk c belongs to: the last whose first chunk is at or before it.
__device__ __forceinline__ uint32_t find(const SetEntry *table, uint32_t tensors, uint32_t c) {
  uint32_t lo = 0, hi = tensors - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) / 2;
    if (table[mid].first_chunk <= c)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ double square(T v) {
  const double d = static_cast<double>(to_f32<T>(v));
  return d * d;
}

// The squares of 16 bytes.
template <typename T>
__device__ __forceinline__ double squares16(const uint4 &u) {
  constexpr int N = 16 / sizeof(T);
  const T *e = reinterpret_cast<const T *>(&u);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s = fmaf(to_f32<T>(e[i]), to_f32<T>(e[i]), s);
  if (s >= 0x1p-100f && s <= FLT_MAX) return static_cast<double>(s);
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) d += square(e[i]);
  return d;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T *p, int n) {
  constexpr int N = 16 / sizeof(T);
  double sum = 0.0;
  if (reinterpret_cast<uintptr_t>(p) % 16 == 0) {
    const uint4 *v = reinterpret_cast<const uint4 *>(p);
    if (n == kChunkBytes / static_cast<int>(sizeof(T))) {
      uint4 u[kVectors];
#pragma unroll
      for (int i = 0; i < kVectors; ++i) u[i] = v[threadIdx.x + i * kThreads];
#pragma unroll
      for (int i = 0; i < kVectors; ++i) sum += squares16<T>(u[i]);
    } else {
      for (int i = threadIdx.x; i < n / N; i += kThreads) sum += squares16<T>(v[i]);
      for (int i = n / N * N + threadIdx.x; i < n; i += kThreads) sum += square(p[i]);
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kThreads) sum += square(p[i]);
  }
  return sum;
}

template <typename T>
__device__ __forceinline__ uint4 scale16(const uint4 &u, float f) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(__uint_as_float(u.x) * f), __float_as_uint(__uint_as_float(u.y) * f),
                      __float_as_uint(__uint_as_float(u.z) * f), __float_as_uint(__uint_as_float(u.w) * f));
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = f2mul(unpack2<T>(w[i]), f2(f));
      r[i] = pack2_t<T>(x.x, x.y);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T *in, T *out, int n, float f) {
  constexpr int N = 16 / sizeof(T);
  if ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) % 16 == 0) {
    const uint4 *v = reinterpret_cast<const uint4 *>(in);
    uint4 *o = reinterpret_cast<uint4 *>(out);
    if (n == kChunkBytes / static_cast<int>(sizeof(T))) {
      uint4 u[kVectors];
#pragma unroll
      for (int i = 0; i < kVectors; ++i) u[i] = v[threadIdx.x + i * kThreads];
#pragma unroll
      for (int i = 0; i < kVectors; ++i) __stcs(o + threadIdx.x + i * kThreads, scale16<T>(u[i], f));
    } else {
      for (int i = threadIdx.x; i < n / N; i += kThreads) o[i] = scale16<T>(v[i], f);
      for (int i = n / N * N + threadIdx.x; i < n; i += kThreads) out[i] = from_f32<T>(to_f32<T>(in[i]) * f);
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kThreads) out[i] = from_f32<T>(to_f32<T>(in[i]) * f);
  }
}

// Calls f with the element type's null pointer, the chunk's first element and its elements.
template <typename F>
__device__ __forceinline__ void with_chunk(const SetEntry &e, uint32_t c, F &&f) {
  const int size = e.dtype == AF2_F32 ? 4 : 2;
  const int64_t per = kChunkBytes / size, first = static_cast<int64_t>(c - e.first_chunk) * per;
  const int n = static_cast<int>(min(per, e.count - first));
  if (e.dtype == AF2_F32)
    f(static_cast<float *>(nullptr), first, n);
  else if (e.dtype == AF2_F16)
    f(static_cast<__half *>(nullptr), first, n);
  else
    f(static_cast<__nv_bfloat16 *>(nullptr), first, n);
}

// The sum over the block, to every thread.
__device__ __forceinline__ double block_sum(double v, double (&warps)[kThreads / 32]) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += warps[w];
  return total;
}

template <int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    gradient_kernel(const __grid_constant__ Table<N> inlined, const Set s) {
  __shared__ double warps[kThreads / 32];
  const SetEntry *table = s.table ? s.table : inlined.entry;
  const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(s.chunks) * blockIdx.x / gridDim.x);
  const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(s.chunks) * (blockIdx.x + 1) / gridDim.x);
  double sum = 0.0;
  uint32_t at = begin < end ? find(table, s.tensors, begin) : 0;
  for (uint32_t c = begin; c < end; ++c) {
    while (at + 1 < s.tensors && table[at + 1].first_chunk <= c) ++at;
    with_chunk(table[at], c, [&](auto *tag, int64_t first, int n) {
      using T = std::remove_pointer_t<decltype(tag)>;
      sum += chunk_squares(static_cast<const T *>(table[at].in) + first, n);
    });
  }
  sum = block_sum(sum, warps);
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) s.partial[blockIdx.x] = sum;
    cooperative_groups::this_grid().sync();
    if (!s.clip && blockIdx.x != 0) return;
    sum = 0.0;
    for (uint32_t i = threadIdx.x; i < gridDim.x; i += kThreads) sum += __ldcg(s.partial + i);
    sum = block_sum(sum, warps);
  }
  const float norm = static_cast<float>(sqrt(sum));
  if (blockIdx.x == 0 && threadIdx.x == 0) *s.norm = norm;
  if (!s.clip) return;
  float f = s.limit / (norm + 1e-6f);
  f = f > 1.f ? 1.f : f;  // a NaN stays one
  for (uint32_t c = end; c-- > begin;) {
    while (table[at].first_chunk > c) --at;
    if (table[at].in == table[at].out && f == 1.f) continue;
    with_chunk(table[at], c, [&](auto *tag, int64_t first, int n) {
      using T = std::remove_pointer_t<decltype(tag)>;
      chunk_scale(static_cast<const T *>(table[at].in) + first, static_cast<T *>(table[at].out) + first, n, f);
    });
  }
}

constexpr size_t kOffTable = 16384;  // behind the blocks' sums
static_assert(kOffTable >= 8 * 256 * kBlocksPerSm, "");

template <int N>
cudaError_t launch_upload(const SetEntry *entries, int count, SetEntry *dst, cudaStream_t stream) {
  Table<N> t;
  std::copy(entries, entries + count, t.entry);
  upload_kernel<N><<<1, 256, 0, stream>>>(t, dst, count);
  return cudaGetLastError();
}

template <int N>
cudaError_t launch_set(const SetEntry *entries, const Set &set, int blocks, cudaStream_t stream) {
  Table<N> t;  // entries past the set's are not read
  if (!set.table) std::copy(entries, entries + set.tensors, t.entry);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(kThreads);
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  config.attrs = attr;
  config.numAttrs = blocks > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&config, gradient_kernel<N>, t, set);
}

}  // namespace

uint64_t gradient_norm_workspace_bytes(int64_t count) {
  return kOffTable + (count > kInline ? align_up(sizeof(SetEntry) * count, 256) : 0);
}

af2_status gradient_norm_launch(af2_ctx *ctx, const af2_tensor_ref *tensors, const af2_tensor_ref *outputs,
                                int64_t count, bool clip, float max_norm, float *norm, void *workspace,
                                cudaStream_t stream) {
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  SetEntry *table = reinterpret_cast<SetEntry *>(ws + kOffTable);
  std::vector<SetEntry> entries;
  entries.reserve(count);
  uint64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (tensors[i].count == 0) continue;
    const uint64_t bytes = static_cast<uint64_t>(tensors[i].count) * (tensors[i].dtype == AF2_F32 ? 4 : 2);
    entries.push_back({tensors[i].data, outputs ? outputs[i].data : tensors[i].data, tensors[i].count,
                       static_cast<uint32_t>(chunks), static_cast<uint32_t>(tensors[i].dtype)});
    chunks += (bytes + kChunkBytes - 1) / kChunkBytes;
    if (chunks > 0x7fffffff) return fail(ctx, AF2_ERR_UNSUPPORTED, "the set has more than 2^31 chunks of 16 KB");
  }
  const int used = static_cast<int>(entries.size());
  Set set{};
  set.partial = reinterpret_cast<double *>(ws);
  set.norm = norm;
  set.tensors = used;
  set.chunks = static_cast<uint32_t>(chunks);
  set.limit = std::min(max_norm, FLT_MAX);
  set.clip = clip;
  const int sms = std::min(ctx->sm_count, 256);
  const int blocks = static_cast<int>(std::max<uint64_t>(1, std::min<uint64_t>(chunks, kBlocksPerSm * sms)));
  cudaError_t e = cudaSuccess;
  if (used > kInline) {
    set.table = table;
    for (int i = 0; i < used && e == cudaSuccess; i += kInline) {
      LaunchScope scope(ctx, stream, kProfGradientNorm);
      e = launch_upload<kInline>(entries.data() + i, std::min(kInline, used - i), table + i, stream);
    }
    if (e != cudaSuccess) return cuda_fail(ctx, e, "gradient table");
  }
  LaunchScope scope(ctx, stream, kProfGradientNorm);
  // the arguments are copied for each launch (30 KB of them take some 10 us): no longer than needed
  if (used <= 64 || set.table)
    e = launch_set<64>(entries.data(), set, blocks, stream);
  else if (used <= 224)
    e = launch_set<224>(entries.data(), set, blocks, stream);
  else if (used <= 480)
    e = launch_set<480>(entries.data(), set, blocks, stream);
  else
    e = launch_set<kInline>(entries.data(), set, blocks, stream);
  if (e != cudaSuccess) return cuda_fail(ctx, e, "gradient norm");
  return AF2_OK;
}

}  // namespace af2
