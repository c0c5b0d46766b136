// dense.cu -- the dense layer and the gated transition, forward and backward.
//
//   dense:  z = x W + b, y = act(z) (+ r);   dz = dy act'(z), dx = dz W^T,
//           dW = x^T dz, db = column sums of dz
//   gated:  g = x Wg + bg, v = x Wv + bv, h = act(g) v, y = h Wo + bo (+ r);
//           dh = dy Wo^T, dv = dh act(g), dg = dh v act'(g),
//           dx = dg Wg^T + dv Wv^T, dWg = x^T dg, dWv = x^T dv, dWo = h^T dy
//
// Every product is a layer_gemm launch on the operands as they are stored, the
// activations, slopes and gates in its epilogues.  Tensors that TMA cannot read
// (rows not in 16-byte pieces) are copied to padded rows first, and f32 ones are
// split into bf16 terms by the same pass (22117 x 263 f32: 9 us, 6 TB/s).  What is
// left are passes over rows, which memory bounds: dz and its column sums of 16384 x
// 4096 bf16 80 us, 5.0 TB/s.
//
// What a forward pass saves: the factors that the backward pass multiplies by
// (dense: act'(z); gated: v act'(g) and act(g); the f32 gated transition g and v
// themselves), and the gated transition's h, an operand already.
#include <algorithm>
#include <type_traits>

#include "few_rows.h"
#include "gated_fused.h"
#include "layer_factor.cuh"
#include "layer_gemm.h"
#include "layer_math.cuh"

namespace af2 {
namespace {

size_t element_size(int dtype) { return dtype == AF2_F32 ? 4 : 2; }
uint64_t part(uint64_t bytes) { return align_up(bytes, 256); }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- copies to operands ---------------------------------------------------------

constexpr int kMaxPackJobs = 6;
struct PackJob {
  const void *src;
  int64_t stride;  // elements
  int64_t rows, width;
  void *dst;       // [pieces][rows][pitch] of 16 bits
  int64_t pitch, piece_stride;
  int64_t first;   // 8-column groups of the jobs before this one
};
struct PackArgs {
  PackJob job[kMaxPackJobs];
  int count;
  int64_t groups;
};

// Eight values of a row as they are in memory (nothing is computed from them yet, so that a thread's
// loads need not wait for one another), and as f32; zeros past the first n.
template <typename T>
struct Raw8 {
  uint32_t w[2 * sizeof(T)];
};
template <typename T>
__device__ __forceinline__ void load_raw8(const T *p, int n, Raw8<T> &x) {
  constexpr int WORDS = 2 * sizeof(T);
  if (n >= 8 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const uint4 u = reinterpret_cast<const uint4 *>(p)[i / 4];
      x.w[i] = u.x, x.w[i + 1] = u.y, x.w[i + 2] = u.z, x.w[i + 3] = u.w;
    }
  } else if (n >= 8 && reinterpret_cast<uintptr_t>(p) % (2 * sizeof(T)) == 0) {  // rows of an even length
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        const uint2 u = reinterpret_cast<const uint2 *>(p)[i];
        x.w[2 * i] = u.x, x.w[2 * i + 1] = u.y;
      } else {
        x.w[i] = reinterpret_cast<const uint32_t *>(p)[i];
      }
    }
  } else {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x.w[i] = i < n ? reinterpret_cast<const uint32_t *>(p)[i] : 0u;
    } else {
      const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = 2 * i < n ? q[2 * i] : 0u, hi = 2 * i + 1 < n ? q[2 * i + 1] : 0u;
        x.w[i] = lo | (hi << 16);
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ void values8(const Raw8<T> &r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 v;
    if constexpr (sizeof(T) == 4)
      v = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    else
      v = unpack2<T>(r.w[i]);
    x[2 * i] = v.x;
    x[2 * i + 1] = v.y;
  }
}

// Eight values as an operand: rounded to T, or f32 as three bf16 terms `piece_stride` elements apart.
template <typename T>
__device__ __forceinline__ void store_operand8(void *dst, int64_t at, int64_t piece_stride, const float (&x)[8]) {
  uint16_t *d = static_cast<uint16_t *>(dst) + at;
  if constexpr (sizeof(T) == 4) {
    uint4 t[3];
    split8(x, t);
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4 *>(d + k * piece_stride) = t[k];
  } else {
    *reinterpret_cast<uint4 *>(d) = make_uint4(pack2_t<T>(x[0], x[1]), pack2_t<T>(x[2], x[3]),
                                               pack2_t<T>(x[4], x[5]), pack2_t<T>(x[6], x[7]));
  }
}

// The copies, by block `block` of `blocks`.
template <typename T>
__device__ __forceinline__ void pack_groups(const PackArgs &p, unsigned block, unsigned blocks) {
  for (int64_t g = static_cast<int64_t>(block) * 256 + threadIdx.x; g < p.groups;
       g += static_cast<int64_t>(blocks) * 256) {
    int j = 0;
    while (j + 1 < p.count && g >= p.job[j + 1].first) ++j;
    const PackJob &job = p.job[j];
    const int64_t per_row = job.pitch / 8, at = g - job.first, r = at / per_row, c = (at - r * per_row) * 8;
    Raw8<T> raw;
    load_raw8<T>(static_cast<const T *>(job.src) + r * job.stride + c,
                 static_cast<int>(min(static_cast<int64_t>(8), job.width - c)), raw);
    float x[8];
    values8<T>(raw, x);
    store_operand8<T>(job.dst, r * job.pitch + c, job.piece_stride, x);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackArgs p) {
  dependency_wait();
  pack_groups<T>(p, blockIdx.x, gridDim.x);
}

// ---- passes over rows, with column sums --------------------------------------------

// How a pass covers its rows: `lanes` threads of eight columns each along a row and `at_once` rows side
// by side in a block of 256 threads, `group` rows a block, `across` blocks along the width.  Few threads
// are left without work (at a width of 320, 40 lanes and six rows instead of 64 lanes of which 24 would
// idle), and among the splits of the width that are within 1/16 of the best the narrowest is taken:
// blocks of more rows have fewer sums to write and to join (16384 x 4096 bf16 in two blocks of 256 lanes
// took 117 us, in 16 of 32 lanes 80).  A thread has eight rows, fewer where that would leave SMs without
// a block.
struct RowGrid {
  int lanes, at_once, group;
  unsigned across;
  unsigned down = 0;  // blocks along the rows
};
inline RowGrid row_grid(int64_t rows, int64_t width) {
  const int64_t pieces = ceil_div(width, 8), least = ceil_div(pieces, 256);
  RowGrid g{};
  int64_t best = 0;
  for (int pass = 0; pass < 2; ++pass)
    for (int64_t n = least; n < least + 16; ++n) {
      const int64_t lanes = ceil_div(pieces, n), at_once = 256 / lanes;
      if (n > least && lanes < 32) break;
      const int64_t use = (pieces * at_once << 16) / n;  // threads with work of each block
      if (pass == 0)
        best = std::max(best, use);
      else if (use >= best - best / 16)
        g = {static_cast<int>(lanes), static_cast<int>(at_once), 0, static_cast<unsigned>(n), 0};
    }
  int each = 8;
  while (each > 1 && ceil_div(rows, g.at_once * each) * g.across < 296) each /= 2;
  g.group = g.at_once * each;
  g.down = static_cast<unsigned>(ceil_div(rows, g.group));
  return g;
}

// load(row, column, in) for DEPTH rows a thread, then use(row, column, in, sums) for them: the loads of
// one are held up neither by the other's stores nor by its arithmetic.  Then sums[s] over the block's rows
// go to partial[x][s][pitch], in a fixed order.
template <typename In, int SETS, int DEPTH, typename Load, typename Use>
__device__ __forceinline__ void for_row_groups(int64_t rows, int64_t width, const RowGrid &grid, float *partial,
                                               int64_t pitch, Load &&load, Use &&use) {
  const unsigned y = blockIdx.x / grid.down, x = blockIdx.x - y * grid.down;
  const int ty = threadIdx.x / grid.lanes, tx = threadIdx.x - ty * grid.lanes;
  const int64_t c = (static_cast<int64_t>(y) * grid.lanes + tx) * 8;
  const int64_t r0 = static_cast<int64_t>(x) * grid.group;
  float sums[SETS][8] = {};
  if (c < width && ty < grid.at_once) {
    const int end = static_cast<int>(min(rows - r0, static_cast<int64_t>(grid.group)));
    for (int r = ty; r < end; r += DEPTH * grid.at_once) {
      In in[DEPTH];
#pragma unroll
      for (int i = 0; i < DEPTH; ++i)
        if (r + i * grid.at_once < end) load(r0 + r + i * grid.at_once, c, in[i]);
#pragma unroll
      for (int i = 0; i < DEPTH; ++i)
        if (r + i * grid.at_once < end) use(r0 + r + i * grid.at_once, c, in[i], sums);
    }
  }
  if (!partial) return;
  __shared__ float all[256][9];
#pragma unroll
  for (int s = 0; s < SETS; ++s) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) all[threadIdx.x][i] = sums[s][i];
    __syncthreads();
    for (int k = threadIdx.x; k < grid.lanes * 8; k += 256) {
      float total = 0.f;
      for (int w = 0; w < grid.at_once; ++w) total += all[w * grid.lanes + (k >> 3)][k & 7];
      const int64_t col = static_cast<int64_t>(y) * grid.lanes * 8 + k;
      if (col < pitch) partial[(static_cast<int64_t>(x) * SETS + s) * pitch + col] = total;
    }
  }
}

__device__ __forceinline__ int columns_of(int64_t width, int64_t c) {
  return static_cast<int>(min(static_cast<int64_t>(8), width - c));
}

template <typename T>
__global__ void __launch_bounds__(256) column_sum_kernel(const T *src, int64_t stride, int64_t rows, int64_t width,
                                                         const RowGrid grid, float *partial, int64_t pitch) {
  dependency_wait();
  for_row_groups<Raw8<T>, 1, 4>(
      rows, width, grid, partial, pitch,
      [&](int64_t r, int64_t c, Raw8<T> &in) { load_raw8<T>(src + r * stride + c, columns_of(width, c), in); },
      [&](int64_t, int64_t, const Raw8<T> &in, float (&sums)[1][8]) {
        float x[8];
        values8<T>(in, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[0][i] += x[i];
      });
}

// What a slope is kept in (SavedPlanes).
template <typename T>
using Kept = std::conditional_t<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat16, float>;
// Eight saved slopes.
template <typename T>
__device__ __forceinline__ void load_slopes8(const SavedPlanes &s, int64_t r, int64_t c, Raw8<Kept<T>> &x) {
  const int64_t at = r * s.pitch + c;
  if constexpr (sizeof(Kept<T>) == 4)
    load_raw8<float>(s.f32 + at, 8, x);
  else
    load_raw8<T>(reinterpret_cast<const T *>(s.half + at), 8, x);
}
template <typename T>
__device__ __forceinline__ void slopes8(const Raw8<Kept<T>> &r, float (&x)[8]) {
  if constexpr (sizeof(Kept<T>) == 4) {
    values8<float>(r, x);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = slope_values(r.w[i]);
      x[2 * i] = v.x;
      x[2 * i + 1] = v.y;
    }
  }
}

// dz = dy act'(z), the slope saved (without SLOPE dy itself), as an operand, with its column sums; the
// blocks past these make the copies of other operands.
template <typename T, bool SLOPE>
__global__ void __launch_bounds__(256) dense_slope_kernel(const T *dy, int64_t dy_stride, const SavedPlanes saved,
                                                          int64_t rows, int64_t width, const RowGrid grid, void *dz,
                                                          int64_t dz_pitch, int64_t dz_piece, float *partial,
                                                          int64_t pitch, const __grid_constant__ PackArgs copies) {
  dependency_wait();
  const unsigned own = grid.down * grid.across;
  if (blockIdx.x >= own) return pack_groups<T>(copies, blockIdx.x - own, gridDim.x - own);
  constexpr int DEPTH = sizeof(T) == 4 ? 2 : 4;
  struct In {
    Raw8<T> dy;
    Raw8<Kept<T>> slope;
  };
  for_row_groups<In, 1, DEPTH>(
      rows, width, grid, partial, pitch,
      [&](int64_t r, int64_t c, In &in) {
        load_raw8<T>(dy + r * dy_stride + c, columns_of(width, c), in.dy);
        if constexpr (SLOPE) load_slopes8<T>(saved, r, c, in.slope);
      },
      [&](int64_t r, int64_t c, const In &in, float (&sums)[1][8]) {
        float d[8];
        values8<T>(in.dy, d);
        if constexpr (SLOPE) {
          float z[8];
          slopes8<T>(in.slope, z);
          const int n = columns_of(width, c);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = i < n ? d[i] * z[i] : 0.f;  // (past the width nothing was saved)
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[0][i] += d[i];
        store_operand8<T>(dz, r * dz_pitch + c, dz_piece, d);
      });
}

// ---- one pass of a layer --------------------------------------------------------------

// Lays the scratch out and launches; without a context it only counts the scratch.
class Pass {
 public:
  Pass(af2_ctx *ctx, int dtype, void *scratch, cudaStream_t stream)
      : ctx_(ctx), dtype_(dtype), base_(static_cast<uint8_t *>(scratch)), stream_(stream) {}

  af2_status status = AF2_OK;
  uint64_t used = 0;

  bool live() const { return ctx_ && status == AF2_OK; }
  bool f32() const { return dtype_ == AF2_F32; }
  int pieces() const { return f32() ? 3 : 1; }

  uint8_t *take(uint64_t bytes) {
    uint8_t *p = base_ + used;
    used += part(bytes);
    return p;
  }
  // Room for an operand of this width made by a kernel.
  GemmOperand make_operand(int64_t rows, int64_t width) {
    GemmOperand o;
    o.pitch = operand_pitch(width);
    o.piece_stride = rows * o.pitch;
    o.ptr = take(2ull * pieces() * rows * o.pitch);
    return o;
  }
  // Whether a tensor of the call's type is an operand as it is.
  bool in_place(const void *src, int64_t stride) const {
    return !f32() && reinterpret_cast<uintptr_t>(src) % 16 == 0 && stride % 8 == 0 && stride < (int64_t(1) << 38);
  }
  // The tensor as an operand: itself, or a copy (pack() launches the copies).
  GemmOperand operand(const void *src, int64_t stride, int64_t rows, int64_t width) {
    if (in_place(src, stride)) {
      GemmOperand o;
      o.ptr = src;
      o.pitch = stride;
      return o;
    }
    const GemmOperand o = make_operand(rows, width);
    jobs_.job[jobs_.count++] = {src, stride, rows, width, const_cast<void *>(o.ptr), o.pitch, o.piece_stride,
                                jobs_.groups};
    jobs_.groups += rows * (o.pitch / 8);
    return o;
  }
  unsigned pack_blocks() const {
    return static_cast<unsigned>(std::min<int64_t>(ceil_div(jobs_.groups, 256), 16 * ctx_->sm_count));
  }
  void pack() {
    if (live() && jobs_.count) {
      const unsigned blocks = pack_blocks();
      LaunchScope scope(ctx_, stream_, kProfLayerElementwise);
      with_element(dtype_, [&](auto *tag) {
        check(launch_early(pack_kernel<std::remove_pointer_t<decltype(tag)>>, dim3(blocks), 256, 0, stream_, jobs_),
              "layer operand copies");
      });
    }
    jobs_ = PackArgs{};
  }

  LayerGemm product(int64_t m, int64_t n, int64_t k) const {
    LayerGemm g;
    g.m = m;
    g.n = n;
    g.k = k;
    g.bf16 = dtype_ != AF2_F16;
    g.pieces = pieces();
    g.out_dtype = dtype_;
    return g;
  }
  static GemmOperand mn(GemmOperand o) {
    o.mn_major = true;
    return o;
  }
  void run(const LayerGemm &g) {
    LayerGemm one[kMaxProducts];
    one[0] = g;
    run(one, 1);
  }
  // Independent products in one launch: their tiles fill the SMs together.  g: room for kMaxProducts.
  // With the last ones go the column sums asked for so far.
  void run(LayerGemm *g, int count, bool last = false) {
    const uint64_t mark = used;
    if (count) count = layer_gemm_plan(g, count);
    for (int i = 0; i < count; ++i) g[i].scratch = take(g[i].scratch_bytes);
    if (live() && count) status = layer_gemm_launch(ctx_, g, count, stream_);
    if (live()) status = layer_finish_launch(ctx_, dtype_, g, count, sums_, last ? sum_count_ : 0, stream_);
    peak_ = std::max(peak_, used);
    used = mark;  // launches follow one another on the stream: the next may use the same place
  }
  uint64_t total() const { return std::max(peak_, used); }

  SavedPlanes planes(void *saved, int64_t rows, int64_t width, int count) const {
    SavedPlanes s;
    s.pitch = saved_pitch(width);
    s.stride = rows * s.pitch;
    if (dtype_ != AF2_BF16) {
      s.f32 = static_cast<float *>(saved);
    } else {
      s.half = static_cast<uint16_t *>(saved);
      s.scale = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(saved) + part(2ull * count * s.stride));
      s.scale_rows = align_up(rows, 32);
    }
    return s;
  }

  // launch(blocks, grid) for a kernel of for_row_groups
  template <typename F>
  void rows_kernel(int64_t rows, int64_t width, F &&launch) {
    if (!live()) return;
    const RowGrid grid = row_grid(rows, width);
    LaunchScope scope(ctx_, stream_, kProfLayerElementwise);
    check(launch(dim3(grid.down * grid.across), grid), "layer row pass");
  }
  // The column sums of a tensor: the blocks' sums, `sets` of them, and how many blocks there are.
  static int64_t sum_chunks(int64_t rows, int64_t width) { return ceil_div(rows, row_grid(rows, width).group); }
  float *sum_room(int64_t rows, int64_t width, int sets) {
    return reinterpret_cast<float *>(take(4ull * sets * sum_chunks(rows, width) * saved_pitch(width)));
  }
  // Sums of chunks, one set of a row of `sets`, to go out with the last products.
  void finish_sums(const float *partial, int64_t chunks, int64_t width, void *dst, int set = 0, int sets = 1) {
    if (!dst) return;
    const int64_t pitch = saved_pitch(width);
    sums_[sum_count_++] = {partial + set * pitch, chunks, sets * pitch, width, dst, false};
  }
  void column_sums(const void *src, int64_t stride, int64_t rows, int64_t width, void *dst) {
    if (!dst) return;
    if (rows <= 1024) {  // four reads one after the other in the last launch are less than a launch more
      sums_[sum_count_++] = {src, rows, stride, width, dst, true};
      return;
    }
    float *partial = sum_room(rows, width, 1);
    rows_kernel(rows, width, [&](dim3 blocks, const RowGrid &grid) {
      cudaError_t e = cudaSuccess;
      with_element(dtype_, [&](auto *tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        e = launch_early(column_sum_kernel<T>, blocks, 256, 0, stream_, static_cast<const T *>(src), stride, rows,
                         width, grid, partial, saved_pitch(width));
      });
      return e;
    });
    finish_sums(partial, sum_chunks(rows, width), width, dst);
  }
  // dz = dy act'(z) (without SLOPE dy) into an operand, and its column sums; with it the operands taken
  // so far are copied
  template <bool SLOPE>
  void slope(const void *dy, int64_t stride, const SavedPlanes &saved, int64_t rows, int64_t width,
             const GemmOperand &dz, void *d_bias) {
    float *partial = d_bias ? sum_room(rows, width, 1) : nullptr;
    rows_kernel(rows, width, [&](dim3 blocks, const RowGrid &grid) {
      cudaError_t e = cudaSuccess;
      with_element(dtype_, [&](auto *tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        e = launch_early(dense_slope_kernel<T, SLOPE>, dim3(blocks.x + pack_blocks()), 256, 0, stream_,
                         static_cast<const T *>(dy), stride, saved, rows, width, grid, const_cast<void *>(dz.ptr),
                         dz.pitch, dz.piece_stride, partial, saved_pitch(width), jobs_);
      });
      return e;
    });
    jobs_ = PackArgs{};
    finish_sums(partial, sum_chunks(rows, width), width, d_bias);
  }
  // The operands taken so far copied, and a gradient as an operand (where one is wanted) with its
  // column sums: one pass for both where the operand is a copy.
  GemmOperand operand_and_sums(const void *dy, int64_t stride, int64_t rows, int64_t width, bool wanted, void *d_bias) {
    if (wanted && d_bias && !in_place(dy, stride)) {
      const GemmOperand o = make_operand(rows, width);
      slope<false>(dy, stride, SavedPlanes{}, rows, width, o, d_bias);
      return o;
    }
    const GemmOperand o = wanted ? operand(dy, stride, rows, width) : GemmOperand{};
    pack();
    column_sums(dy, stride, rows, width, d_bias);
    return o;
  }
  void zero(void *ptr, size_t bytes) {
    if (!ptr || !live()) return;
    if (cudaError_t e = cudaMemsetAsync(ptr, 0, bytes, stream_); e != cudaSuccess)
      status = cuda_fail(ctx_, e, "zero a gradient");
  }
  void check(cudaError_t e, const char *what) {
    if (e != cudaSuccess && status == AF2_OK) status = cuda_fail(ctx_, e, what);
  }

 private:
  af2_ctx *ctx_;
  int dtype_;
  uint8_t *base_;
  cudaStream_t stream_;
  PackArgs jobs_{};
  ColumnSums sums_[kMaxSums];
  int sum_count_ = 0;
  uint64_t peak_ = 0;
};

uint64_t planes_bytes(int64_t rows, int64_t width, int dtype, int count) {
  const uint64_t n = static_cast<uint64_t>(count) * rows * saved_pitch(width);
  if (dtype != AF2_BF16) return part(4 * n);
  return part(2 * n) + (count > 1 ? part(align_up(rows, 32) * saved_pitch(width) / 8) : 0);
}
uint64_t hidden_bytes(int64_t rows, int64_t hidden, int dtype) {
  return part(2ull * (dtype == AF2_F32 ? 3 : 1) * rows * operand_pitch(hidden));
}

}  // namespace

uint64_t dense_saved_bytes(int64_t rows, int64_t columns, int dtype, int activation) {
  return activation == AF2_ACTIVATION_NONE ? 0 : planes_bytes(rows, columns, dtype, 1);
}
uint64_t gated_saved_bytes(int64_t rows, int64_t hidden, int dtype) {
  return hidden_bytes(rows, hidden, dtype) + planes_bytes(rows, hidden, dtype, 2);
}

af2_status dense_forward(af2_ctx *ctx, const DenseForward &p, void *scratch, uint64_t *bytes, cudaStream_t stream) {
  Pass l(ctx, p.dtype, scratch, stream);
  if (few_rows(p.rows, p.inner, p.columns, p.dtype, false) && !(p.saved && p.activation != AF2_ACTIVATION_NONE)) {
    *bytes = 0;
    if (!ctx) return AF2_OK;
    FewRows f;
    f.rows = p.rows, f.inner = p.inner, f.columns = p.columns;
    f.dtype = p.dtype, f.activation = p.activation;
    f.x = p.x, f.x_stride = p.x_stride;
    f.weight[0] = p.weight, f.bias[0] = p.bias;
    f.residual = p.residual, f.residual_stride = p.residual_stride;
    f.out = p.out, f.out_stride = p.out_stride;
    return few_rows_launch(ctx, f, stream);
  }
  LayerGemm g = l.product(p.rows, p.columns, p.inner);
  g.a[0] = l.operand(p.x, p.x_stride, p.rows, p.inner);
  g.b[0] = Pass::mn(l.operand(p.weight, p.columns, p.inner, p.columns));
  l.pack();
  g.activation = p.activation;
  g.bias[0] = p.bias;
  g.residual = p.residual;
  g.residual_stride = p.residual_stride;
  g.out[0] = p.out;
  g.out_stride = p.out_stride;
  if (p.saved && p.activation != AF2_ACTIVATION_NONE) g.saved = l.planes(p.saved, p.rows, p.columns, 1);
  l.run(g);
  *bytes = l.total();
  return l.status;
}

af2_status dense_backward(af2_ctx *ctx, const DenseBackward &p, void *scratch, uint64_t *bytes, cudaStream_t stream) {
  Pass l(ctx, p.dtype, scratch, stream);
  const size_t e = element_size(p.dtype);
  if (p.rows == 0) {
    l.zero(p.d_weight, e * p.inner * p.columns);
    l.zero(p.d_bias, e * p.columns);
    *bytes = 0;
    return l.status;
  }
  GemmOperand dz, x, w;
  if (p.d_weight) x = l.operand(p.x, p.x_stride, p.rows, p.inner);
  if (p.d_x) w = l.operand(p.weight, p.columns, p.inner, p.columns);
  if (p.activation == AF2_ACTIVATION_NONE) {
    dz = l.operand_and_sums(p.d_out, p.d_out_stride, p.rows, p.columns, p.d_x || p.d_weight, p.d_bias);
  } else {
    dz = l.make_operand(p.rows, p.columns);
    const SavedPlanes saved = l.planes(const_cast<void *>(p.saved), p.rows, p.columns, 1);
    l.slope<true>(p.d_out, p.d_out_stride, saved, p.rows, p.columns, dz, p.d_bias);
  }
  LayerGemm products[kMaxProducts];
  int count = 0;
  if (p.d_x) {
    LayerGemm &g = products[count++] = l.product(p.rows, p.inner, p.columns);
    g.a[0] = dz;
    g.b[0] = w;
    g.out[0] = p.d_x;
    g.out_stride = p.d_x_stride;
  }
  if (p.d_weight) {
    LayerGemm &g = products[count++] = l.product(p.inner, p.columns, p.rows);
    g.a[0] = Pass::mn(x);
    g.b[0] = Pass::mn(dz);
    g.out[0] = p.d_weight;
    g.out_stride = p.columns;
  }
  l.run(products, count, true);
  *bytes = l.total();
  return l.status;
}

af2_status gated_forward(af2_ctx *ctx, const GatedForward &p, void *scratch, uint64_t *bytes, cudaStream_t stream) {
  Pass l(ctx, p.dtype, scratch, stream);
  GatedFused fused;
  fused.rows = p.rows, fused.channels = p.channels, fused.hidden = p.hidden;
  fused.dtype = p.dtype, fused.activation = p.activation;
  fused.residual = p.residual, fused.residual_stride = p.residual_stride;
  fused.out = p.out, fused.out_stride = p.out_stride;
  const bool one_kernel = !p.saved && gated_fused_covers(fused);
  const bool few = !p.saved && few_rows(p.rows, p.channels, p.hidden, p.dtype, true);
  // One kernel for both products takes 8.1 us at 128 -> 512 up to 256 rows, few rows 8.0 at 4 and 19 at 256.
  // Which of them runs depends on addresses too, so the scratch is counted for both.
  const bool fits = p.rows > 4 && gated_fused_fits(fused);
  if (few && (!fits || (ctx && !one_kernel))) {
    void *h = l.take(element_size(p.dtype) * p.rows * p.hidden);
    *bytes = l.total();
    if (!ctx) return AF2_OK;
    FewRows f;
    f.rows = p.rows, f.inner = p.channels, f.columns = p.hidden;
    f.dtype = p.dtype, f.activation = p.activation;
    f.x = p.x, f.x_stride = p.x_stride;
    f.weight[0] = p.w.gate_weight, f.weight[1] = p.w.value_weight;
    f.bias[0] = p.w.gate_bias, f.bias[1] = p.w.value_bias;
    f.out = h, f.out_stride = p.hidden;
    if (af2_status st = few_rows_launch(ctx, f, stream); st != AF2_OK) return st;
    FewRows y;
    y.rows = p.rows, y.inner = p.hidden, y.columns = p.channels;
    y.dtype = p.dtype;
    y.x = h, y.x_stride = p.hidden;
    y.weight[0] = p.w.output_weight, y.bias[0] = p.w.output_bias;
    y.residual = p.residual, y.residual_stride = p.residual_stride;
    y.out = p.out, y.out_stride = p.out_stride;
    y.follows = true;
    return few_rows_launch(ctx, y, stream);
  }
  const uint64_t few_bytes = few ? part(element_size(p.dtype) * p.rows * p.hidden) : 0;
  const GemmOperand x = l.operand(p.x, p.x_stride, p.rows, p.channels);
  const GemmOperand wg = l.operand(p.w.gate_weight, p.hidden, p.channels, p.hidden);
  const GemmOperand wv = l.operand(p.w.value_weight, p.hidden, p.channels, p.hidden);
  const GemmOperand wo = l.operand(p.w.output_weight, p.channels, p.hidden, p.channels);
  l.pack();
  fused.x = x, fused.gate = wg, fused.value = wv, fused.output = wo;
  fused.gate_bias = p.w.gate_bias, fused.value_bias = p.w.value_bias, fused.output_bias = p.w.output_bias;
  if (one_kernel) {
    *bytes = std::max(l.total(), few_bytes);
    return l.live() ? gated_fused_launch(ctx, fused, stream) : l.status;
  }
  GemmOperand h;
  if (p.saved) {
    h.ptr = p.saved;
    h.pitch = operand_pitch(p.hidden);
    h.piece_stride = p.rows * h.pitch;
  } else {
    h = l.make_operand(p.rows, p.hidden);
  }
  LayerGemm g = l.product(p.rows, p.hidden, p.channels);
  g.a[0] = x;
  g.b[0] = Pass::mn(wg);
  g.b[1] = Pass::mn(wv);
  g.bias[0] = p.w.gate_bias;
  g.bias[1] = p.w.value_bias;
  g.epilogue = kEpilogueGate;
  g.activation = p.activation;
  g.out[0] = const_cast<void *>(h.ptr);
  g.out_stride = h.pitch;
  g.out_piece_stride = h.piece_stride;
  if (p.saved)
    g.saved = l.planes(static_cast<uint8_t *>(p.saved) + hidden_bytes(p.rows, p.hidden, p.dtype), p.rows, p.hidden, 2);
  l.run(g);
  LayerGemm y = l.product(p.rows, p.channels, p.hidden);
  y.a[0] = h;
  y.b[0] = Pass::mn(wo);
  y.bias[0] = p.w.output_bias;
  y.residual = p.residual;
  y.residual_stride = p.residual_stride;
  y.out[0] = p.out;
  y.out_stride = p.out_stride;
  l.run(y);
  *bytes = std::max(l.total(), few_bytes);
  return l.status;
}

af2_status gated_backward(af2_ctx *ctx, const GatedBackward &p, void *scratch, uint64_t *bytes, cudaStream_t stream) {
  Pass l(ctx, p.dtype, scratch, stream);
  const int64_t c = p.channels, hid = p.hidden;
  if (p.rows == 0) {
    const size_t e = element_size(p.dtype);
    for (void *w : {p.g.gate_weight, p.g.value_weight, p.g.output_weight}) l.zero(w, e * c * hid);
    for (void *b : {p.g.gate_bias, p.g.value_bias}) l.zero(b, e * hid);
    l.zero(p.g.output_bias, e * c);
    *bytes = 0;
    return l.status;
  }
  const bool gradients_at_hidden = p.g.x || p.g.gate_weight || p.g.gate_bias || p.g.value_weight || p.g.value_bias;
  GemmOperand x, wg, wv, wo, dgv[2];
  if (p.g.gate_weight || p.g.value_weight) x = l.operand(p.x, p.x_stride, p.rows, c);
  if (p.g.x) {
    wg = l.operand(p.w.gate_weight, hid, c, hid);
    wv = l.operand(p.w.value_weight, hid, c, hid);
  }
  if (gradients_at_hidden) wo = l.operand(p.w.output_weight, c, hid, c);
  const GemmOperand dy = l.operand_and_sums(p.d_out, p.d_out_stride, p.rows, c,
                                            gradients_at_hidden || p.g.output_weight, p.g.output_bias);
  GemmOperand h;
  h.ptr = p.saved;
  h.pitch = operand_pitch(hid);
  h.piece_stride = p.rows * h.pitch;
  uint8_t *planes_at = static_cast<uint8_t *>(const_cast<void *>(p.saved)) + hidden_bytes(p.rows, hid, p.dtype);
  const SavedPlanes saved = l.planes(planes_at, p.rows, hid, 2);

  if (gradients_at_hidden) {
    dgv[0] = l.make_operand(p.rows, hid);
    dgv[1] = l.make_operand(p.rows, hid);
    const bool sums = p.g.gate_bias || p.g.value_bias;
    LayerGemm g = l.product(p.rows, hid, c);
    g.a[0] = dy;
    g.b[0] = wo;
    const int64_t chunks = ceil_div(p.rows, 32);
    float *partial = sums ? reinterpret_cast<float *>(l.take(8ull * chunks * saved.pitch)) : nullptr;
    g.epilogue = kEpilogueGateBackward;
    g.activation = p.activation;
    g.saved = saved;
    g.out[0] = const_cast<void *>(dgv[0].ptr);
    g.out[1] = const_cast<void *>(dgv[1].ptr);
    g.out_stride = dgv[0].pitch;
    g.out_piece_stride = dgv[0].piece_stride;
    g.column_partial = partial;
    l.run(g);
    l.finish_sums(partial, chunks, hid, p.g.gate_bias, 0, 2);
    l.finish_sums(partial, chunks, hid, p.g.value_bias, 1, 2);
  }
  LayerGemm products[kMaxProducts];
  int count = 0;
  if (p.g.x) {
    LayerGemm &g = products[count++] = l.product(p.rows, c, hid);
    g.segments = 2;
    g.a[0] = dgv[0];
    g.a[1] = dgv[1];
    g.b[0] = wg;
    g.b[1] = wv;
    g.out[0] = p.g.x;
    g.out_stride = p.d_x_stride;
  }
  if (p.g.gate_weight || p.g.value_weight) {
    LayerGemm &g = products[count++] = l.product(c, hid, p.rows);
    g.a[0] = Pass::mn(x);
    int n = 0;
    if (p.g.gate_weight) g.b[n] = Pass::mn(dgv[0]), g.out[n++] = p.g.gate_weight;
    if (p.g.value_weight) g.b[n] = Pass::mn(dgv[1]), g.out[n++] = p.g.value_weight;
    g.batch = n;
    g.out_stride = hid;
  }
  if (p.g.output_weight) {
    LayerGemm &g = products[count++] = l.product(hid, c, p.rows);
    g.a[0] = Pass::mn(h);
    g.b[0] = Pass::mn(dy);
    g.out[0] = p.g.output_weight;
    g.out_stride = c;
  }
  l.run(products, count, true);
  *bytes = l.total();
  return l.status;
}

}  // namespace af2
