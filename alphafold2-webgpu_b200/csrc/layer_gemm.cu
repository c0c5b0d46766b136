// layer_gemm.cu -- the product of the layers with learned weights on tcgen05:
// D = sum_s A_s B_s^T over 16-bit operands in either order each, f32 sums in
// TMEM, and the layers' epilogues.
//
// A cluster of two CTAs computes a 256 x BN tile with M = 256 MMAs
// (cta_group::2): CTA r holds rows 128 r .. of A's tile and half of B's rows,
// so each SM reads half of the B tile that it multiplies by.  Warp 0 of each
// CTA issues TMA loads, warp 1 of the even CTA the MMAs, warps 2-17 drain the
// two accumulators, together, or in two groups of eight (two per TMEM lane
// quarter) that take tiles in turn where a tile is too narrow for all.  One
// tile's epilogue overlaps the next tile's MMAs.  Operands are taken as they are stored: K-major rows as one
// 128-byte-swizzled block per K step of 64, MN-major ones as 64-wide blocks of
// 64 k each (the tensor core's transposed order), so no weight and no
// activation is ever transposed in memory.  What an epilogue reads (residual,
// saved factors) comes by TMA into the same block of shared memory that its
// result leaves from.
//
// Measured: 16384 x 1024 -> 4096 in bf16 96 us, 1.43 PFLOP/s, bound by the tensor
// core (with gelu 108, its slopes kept 119); the gate with factors of 32768 x 256
// -> 1024 in bf16 55 us for 226 MB, its backward product 61 us for 293 MB: epilogues
// whose phases overlap in part (f16, whose factors are f32: the forward pass 115 us
// for bf16's 95, the backward pass 162 to 168 for 167 to 175); the gradients' products of 8192 x 1024 -> 4096 258 us,
// 0.80 of cuBLAS's rate.  Small products take some 7 us whatever their size.
//
// f32 tensors are multiplied as three bf16 terms each, x = x0 + x1 + x2, and
// the six products whose weight is at least 2^-16 of the largest are summed:
// what is left out is below 2^-24 of |x||y|, f32's own rounding.  A K step's
// three terms of both operands are in shared memory together, so each is read
// once for its products (one read for each product took 900 SM clocks a product
// and step of 64 against 256 of work), and a step is 32 deep, so that the ring
// holds four (with 64 it held two, and waited for each load).  The
// tensor core cuts its sums where f32 rounds them (some 2^-27 of the sum lost
// at each step of 16: sums of one sign over a depth of 4096 came out 2e-6 low),
// so the five small products have an accumulator of their own, and a tile is
// summed over 256 of the depth at a time and these sums are added in registers.
// (An infinite f32 element makes its sums NaN or infinite.)  18944 x 1024 -> 768:
// 121 us, the depth at 1.69 PFLOP/s of its six products.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "layer_factor.cuh"
#include "layer_gemm.h"
#include "layer_math.cuh"

namespace af2 {
namespace {

constexpr int BM = 128, PAIR_M = 256, BK = 64;
constexpr int EPI_WARPS = 16, THREADS = 64 + 32 * EPI_WARPS;
constexpr int kPairs = 74;  // CTA pairs of a B200; only the choice of tiles and splits depends on it

// The kernels behind the epilogues: Out, the same with the slopes kept and (with or without them) where
// TMA cannot address the rows of what is written or of the residual (their code costs Out registers:
// 163578 x 112 -> 40 took 27 us with both in it, 22 without), Out for several products with nothing but their sums
// (whose arguments are no longer operands from the constant bank but loads), and Gate with and
// without what the backward pass needs.
enum Kind { kOut, kOutSave, kOutRows, kProducts, kGate, kGateSave, kGateBackward };

// Stages of the operand ring and bytes of one epilogue warp's staging: 32 x 32 blocks of 16 bits
// (2 KB), two of them (GateBackward: one of each factor); three where h and two bf16 factors leave
// together, paid for with a stage.
// f32: a stage has a step's three terms, A's [3][128 x 32] and B's behind them; the staged blocks
// are 32 x 16.
template <typename T>
constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
template <int KIND, int BN, typename OT>
struct Shape {
  static constexpr bool F32 = sizeof(OT) == 4;
  static constexpr int STEP = F32 ? 32 : BK;
  static constexpr uint32_t A_TERM = BM * STEP * 2, B_TERM = (BN / 2) * STEP * 2;
  static constexpr uint32_t OFF_B = (F32 ? 3 : 1) * A_TERM;
  static constexpr uint32_t STAGE_BYTES = OFF_B + (F32 ? 3 : 1) * B_TERM;
  static constexpr uint32_t SLOT_BYTES = KIND == kGateSave && kBf16<OT> ? 6144 : 4096;
  static constexpr int STAGES = (229376 - EPI_WARPS * SLOT_BYTES) / STAGE_BYTES;
  static constexpr uint32_t OFF_STAGE = STAGES * STAGE_BYTES;
  static constexpr uint32_t OFF_BAR = OFF_STAGE + EPI_WARPS * SLOT_BYTES;
  static constexpr uint32_t BYTES = OFF_BAR + 512 + 1024;
};

struct Maps {
  CUtensorMap a[2], b[2], out[2], residual, half;
};

// n / d and n % d for n below 2^30, d fixed for a launch: the quotient by a multiply-high with
// ceil(2^(32 + s) / d), 2^s >= d, whose error stays below 1 / d there.
struct Divisor {
  uint32_t d = 1, mul = 0, shift = 0;
  Divisor() = default;
  explicit Divisor(uint32_t divisor) : d(divisor) {
    while ((1u << shift) < d) ++shift;
    // 2^32 < 2^(32 + s) / d < 2^33: the leading 2^32 is added by the quotient itself
    mul = static_cast<uint32_t>(((uint64_t(1) << (32 + shift)) + d - 1) / d - (uint64_t(1) << 32));
  }
  __device__ __forceinline__ int split(int &n) const {  // n becomes the quotient; returns the remainder
    const uint32_t q = (__umulhi(static_cast<uint32_t>(n), mul) + static_cast<uint32_t>(n)) >> shift;
    const int r = n - static_cast<int>(q * d);
    n = static_cast<int>(q);
    return r;
  }
};

struct Args {
  void *out[2];
  int64_t out_stride, out_piece_stride;
  const void *bias[2];
  const void *residual;
  int64_t residual_stride;
  uint32_t *saved_scale;
  float *saved_f32;
  int64_t saved_pitch, saved_stride, scale_rows;
  float *column_partial;
  int64_t m;
  int n, k_blocks, splits, segments;
  Divisor tiles_m, tiles_n, batches;
  int a_mn, b_mn, bf16, activation;
  int tma_out;       // out rows are 16-byte aligned: whole blocks leave by TMA
  int tma_residual;  // the residual's blocks come by TMA
  int vector_bias;   // 16-byte aligned
  int save;          // Out: the slopes are kept
  int partial;       // out[0] is [split][batch][m][n] of f32 sums (no bias, activation or residual)
  int first_tile;    // the tiles of the products before this one
};

// What a launch computes: products whose tiles follow one another.  One product's tiles go to the pairs
// in turn.  Several products' tiles differ in length, and the pairs that have a long one take fewer of the
// short: each wave is a run of pairs that take `repeats` tiles each, from `first` on.
struct Product {
  Maps maps;
  Args args;
};
struct Wave {
  int first, repeats;
  int at, pairs;
};
constexpr int kMaxWaves = 24;
struct Waves {
  Wave wave[kMaxWaves];
  int count;
};
struct NoWaves {};
template <int N>
struct Launch {
  Product product[N];
  std::conditional_t<(N > 1), Waves, NoWaves> waves;
  int products, total_tiles;
  int alternate;  // the two groups of epilogue warps take tiles in turn
  unsigned int *err;
};
template <int N>
__device__ __forceinline__ const Product &product_of(const Launch<N> &l, int t) {
  int i = 0;
  if constexpr (N > 1)
    while (i + 1 < l.products && t >= l.product[i + 1].args.first_tile) ++i;
  return l.product[i];
}

// The tiles of a pair, one after the other.
template <int N>
struct Walk {
  const Launch<N> &launch;
  int pair, pairs;
  int at = 0, turn = 0;  // one product: turns taken; several: the wave, and the turns in it
  __device__ __forceinline__ bool next(int &t) {
    if constexpr (N == 1) {
      t = pair + turn++ * pairs;
      return t < launch.total_tiles;
    } else {
      for (; at < launch.waves.count; ++at, turn = 0) {
        const Wave &w = launch.waves.wave[at];
        const int i = pair - w.at;
        if (i >= 0 && i < w.pairs && turn < w.repeats) {
          t = w.first + turn++ * w.pairs + i;
          return true;
        }
      }
      return false;
    }
  }
};

// The terms (of A, of B) of the six products of an f32 operand pair, the largest last.
constexpr int kProductsF32 = 6;
__device__ constexpr int term_a(int c) { return c == 0 ? 2 : c == 2 || c == 3 ? 1 : 0; }
__device__ constexpr int term_b(int c) { return c == 1 ? 2 : c == 2 || c == 4 ? 1 : 0; }

struct Tile {
  int split, z, mi, ni;
};
__device__ __forceinline__ Tile tile_at(const Args &p, int t) {
  Tile r;
  t -= p.first_tile;
  r.ni = p.tiles_n.split(t);
  r.mi = p.tiles_m.split(t);
  r.z = p.batches.split(t);
  r.split = t;
  return r;
}
constexpr int kPromote = 8;  // K steps (of 32) of an f32 tile, and segment, before its sums go to registers

// The tile's range of K steps.
__device__ __forceinline__ int k_begin(const Args &p, int split) {
  return static_cast<int>(static_cast<int64_t>(p.k_blocks) * split / p.splits);
}

// 16 values of a row as raw 16-bit pairs; zeros past `cols`.  `vector`: row + c0 is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load_raw16(const T *row, int c0, int cols, bool vector, uint32_t (&w)[8]) {
  if (vector && c0 + 16 <= cols) {
    const uint4 *p = reinterpret_cast<const uint4 *>(row + c0);
    const uint4 u = __ldg(p), x = __ldg(p + 1);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w, w[4] = x.x, w[5] = x.y, w[6] = x.z, w[7] = x.w;
  } else {
    const uint16_t *p = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = c0 + 2 * i < cols ? p[c0 + 2 * i] : 0, b = c0 + 2 * i + 1 < cols ? p[c0 + 2 * i + 1] : 0;
      w[i] = a | (b << 16);
    }
  }
}

// 16-byte piece c of row `row` of a 32 x 32 block of 16 bits (64B-swizzled).
__device__ __forceinline__ uint4 *piece16(uint8_t *block, int row, int c) {
  return reinterpret_cast<uint4 *>(block + row * 64 + ((c ^ ((row >> 1) & 3)) << 4));
}
// 16-byte piece c of a 32 x 32 block of f32 (128B-swizzled, 4 KB).
__device__ __forceinline__ float4 *piece32(uint8_t *block, int row, int c) {
  return reinterpret_cast<float4 *>(block + sw128_offset(row, c));
}

// Rows that TMA cannot address, moved between memory and a block with the lanes along each row (f32: 16
// lanes, two rows at a time): BATCH loads, then their stores.  (One after the other each store waits for
// its load; with the block's swizzled addresses worked out for each element instead of four times, 34
// instructions a row made an unaligned 60690 x 424 -> 737 product 91 us instead of 55.)
template <typename T, bool IN, int BATCH = 8>
__device__ __forceinline__ void move_rows(uint8_t *block, T *at, int64_t stride, int rows, int cols, int lane) {
  constexpr int SIDE = sizeof(T) == 4 ? 2 : 1, EACH = 16 / sizeof(T), SPAN = BATCH * SIDE;  // rows at a time
  static_assert(SPAN % 8 == 0 && 32 % SPAN == 0);
  const int c = SIDE == 2 ? lane & 15 : lane, side = SIDE == 2 ? lane >> 4 : 0;
  if (c >= cols) return;
  // where the column lies in a row whose number / 2 leaves k to 4
  uint8_t *column[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    column[k] = block + side * 64 + (((c / EACH) ^ k) << 4) + (c % EACH) * static_cast<int>(sizeof(T));
  T *g = at + c;
  auto element = [&](int r0, int i) { return reinterpret_cast<T *>(column[(SIDE * i >> 1) & 3] + (r0 + SIDE * i) * 64); };
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += SPAN) {
    T v[BATCH];
    if constexpr (IN) {
#pragma unroll
      for (int i = 0; i < BATCH; ++i)  // (the last row again instead of one past it: a condition would part the loads)
        v[i] = g[min(r0 + SIDE * i + side, rows - 1) * stride];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) *element(r0, i) = v[i];
    } else {
      T *to = g + (r0 + side) * stride;
#pragma unroll
      for (int i = 0; i < BATCH; ++i) v[i] = *element(r0, i);
      if (r0 + SPAN <= rows) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i, to += SIDE * stride) *to = v[i];
      } else {
#pragma unroll
        for (int i = 0; i < BATCH; ++i, to += SIDE * stride)
          if (r0 + SIDE * i + side < rows) *to = v[i];
      }
    }
  }
}

// 32 aligned bytes (a sector): a TMA store of 16 columns of terms, rows of 32 bytes, takes two clocks a row,
// 12,000 for the six that a tile of the f32 gate's backward pass writes.
__device__ __forceinline__ void store_sector(void *at, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// The three terms of 16 f32, `piece` elements apart.
__device__ __forceinline__ void store_terms16(uint16_t *at, int64_t piece, const float (&x)[16]) {
  uint4 t[2][3];
  split8(reinterpret_cast<const float(&)[8]>(x[0]), t[0]);
  split8(reinterpret_cast<const float(&)[8]>(x[8]), t[1]);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const uint32_t w[8] = {t[0][k].x, t[0][k].y, t[0][k].z, t[0][k].w, t[1][k].x, t[1][k].y, t[1][k].z, t[1][k].w};
    store_sector(at + k * piece, w);
  }
}

// x[i] of lane l becomes, in x[0] of lane i, the sum over the lanes: 31 exchanges for 32 columns.
__device__ __forceinline__ float lane_sums(float (&x)[32], int lane) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = upper ? x[i + o] : x[i], send = upper ? x[i] : x[i + o];
      x[i] = keep + __shfl_xor_sync(kFull, send, o);
    }
  }
  return x[0];
}

template <int KIND, typename OT, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    layer_gemm_kernel(const __grid_constant__ Launch<KIND == kProducts ? kMaxProducts : 1> launch) {
  constexpr int LIMIT = KIND == kProducts ? kMaxProducts : 1;
  using S = Shape<KIND, BN, OT>;
  constexpr bool GATE = KIND == kGate || KIND == kGateSave;
  constexpr bool F32 = sizeof(OT) == 4;
  constexpr int STAGES = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = align1024(smem_raw);
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + S::OFF_BAR;
  // full: the leader's only (both CTAs' loads complete on it); empty, acc_full: both CTAs
  // (multicast commits); acc_empty: the leader's, one arrival per epilogue warp of the pair;
  // load: one per epilogue warp and block, for what it reads
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * STAGES + 2 + b); };
  const uint32_t drain = bar0 + 8u * (2 * STAGES + 4);
  auto load = [&](int w, int b) { return bar0 + 8u * (2 * STAGES + 5 + 2 * w + b); };
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + S::OFF_BAR + 488);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + S::OFF_BAR + 496);
  const int warp = warp_index_uniform(), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), launch.alternate ? EPI_WARPS : 2 * EPI_WARPS);  // both CTAs' warps on a tile
    }
    mbar_init(drain, 1);
    for (int w = 0; w < EPI_WARPS; ++w)
      for (int b = 0; b < 2; ++b) mbar_init(load(w, b), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane < launch.products) {  // (the maps are the launch's own: nothing to wait for)
    const Maps &maps = launch.product[lane].maps;
    tma_prefetch_map(&maps.a[0]);
    tma_prefetch_map(&maps.b[0]);
    tma_prefetch_map(&maps.out[0]);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers exist before any arrival crosses the pair
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0, s = 0;
      uint32_t ph = 1;
      bool ok = true;
      Walk<LIMIT> walk{launch, pair, npairs};
      for (int t; ok && walk.next(t);) {
        const Product &product = product_of(launch, t);
        const Maps &maps = product.maps;
        const Args &p = product.args;
        const Tile tile = tile_at(p, t);
        const int kb0 = p.splits > 1 ? k_begin(p, tile.split) : 0;
        const int kb1 = p.splits > 1 ? k_begin(p, tile.split + 1) : p.k_blocks;
        const int arow = tile.mi * PAIR_M + rank * BM;
        const int brow = GATE ? tile.ni * (BN / 2) : tile.ni * BN + rank * (BN / 2);
        const int segments = p.segments, a_mn = p.a_mn, b_mn = p.b_mn, part = F32 ? kPromote : kb1 - kb0;
        // K steps of a part, segment by segment
        for (int from = kb0; from < kb1 && ok; from += part) {
          for (int seg = 0; seg < segments && ok; ++seg) {
            const CUtensorMap *am = &maps.a[seg];
            const CUtensorMap *bm = &maps.b[GATE ? rank : seg + tile.z];
            for (int kb = from; kb < min(from + part, kb1) && ok; ++kb) {
              // the stage is free in this CTA once the pair's MMAs have read it (multicast commit)
              if (!mbar_wait(empty(s), ph, abort_flag, launch.err, kErrWaitProducer)) {
                ok = false;
                break;
              }
              const uint32_t stage = sbase + s * S::STAGE_BYTES;
              if (leader) mbar_arrive_expect_tx(full(s), 2 * S::STAGE_BYTES);
#pragma unroll
              for (int term = 0; term < (F32 ? 3 : 1); ++term) {
                const uint32_t dst = stage + term * S::A_TERM, dst_b = stage + S::OFF_B + term * S::B_TERM;
                if (a_mn) {
                  tma_load_3d_pair(dst, am, full(s), arow, kb * S::STEP, term);
                  tma_load_3d_pair(dst + S::STEP * 128, am, full(s), arow + 64, kb * S::STEP, term);
                } else {
                  tma_load_3d_pair(dst, am, full(s), kb * S::STEP, arow, term);
                }
                if (b_mn) {
#pragma unroll
                  for (int j = 0; j < BN / 128; ++j)
                    tma_load_3d_pair(dst_b + j * S::STEP * 128, bm, full(s), brow + 64 * j, kb * S::STEP, term);
                } else {
                  tma_load_3d_pair(dst_b, bm, full(s), kb * S::STEP, brow, term);
                }
              }
              ++it;
              if (++s == STAGES) {
                s = 0;
                ph ^= 1;
              }
            }
          }
        }
      }
      // every load issued has landed before the pair exits (the leader's barriers count
      // both CTAs' bytes; the peer waits for the leader at the final cluster barrier)
      if (leader)
        for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j)
          mbar_wait_drain(full(j % STAGES), (j / STAGES) & 1, launch.err);
    }
  } else if (warp == 1) {
    if (leader) {
      // the whole warp runs the issue loop (uniform waits, running descriptors); one elected lane issues
      int s = 0, buf = 0;
      uint32_t ph = 0, bph = 0;
      bool ok = true;
      Walk<LIMIT> walk{launch, pair, npairs};
      for (int t; ok && walk.next(t);) {
        const Args &p = product_of(launch, t).args;
        const uint32_t idesc = idesc_16_f32(PAIR_M, BN, p.bf16, p.a_mn, p.b_mn);
        auto k_major = [](uint32_t at) { return F32 ? sdesc_k_sw64(at) : sdesc_k_sw128(at); };
        const uint64_t a_base = p.a_mn ? sdesc_mn_sw128(sbase, S::STEP * 128, 1024) : k_major(sbase);
        const uint64_t b_base = p.b_mn ? sdesc_mn_sw128(sbase + S::OFF_B, S::STEP * 128, 1024) : k_major(sbase + S::OFF_B);
        // bytes >> 4 from one K step of 16 to the next
        const uint32_t a_step = p.a_mn ? 2048 >> 4 : 32 >> 4, b_step = p.b_mn ? 2048 >> 4 : 32 >> 4;
        uint64_t ad = desc_add(a_base, s * S::STAGE_BYTES), bd = desc_add(b_base, s * S::STAGE_BYTES);
        int steps = p.k_blocks;
        if (p.splits > 1) {
          const int split = tile_at(p, t).split;
          steps = k_begin(p, split + 1) - k_begin(p, split);
        }
        const int part = F32 ? kPromote : steps;
        for (int from = 0; from < steps && ok; from += part) {
          const int iters = min(part, steps - from) * p.segments;
          if (!warp_wait(acc_empty(buf), bph ^ 1, abort_flag, launch.err, kErrWaitMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + buf * 256;
          for (int i = 0; i < iters; ++i) {
            if (!warp_wait(full(s), ph, abort_flag, launch.err, kErrWaitMma)) {
              ok = false;
              break;
            }
            tc_fence_after();
            if constexpr (F32) {
#pragma unroll
              for (int c = 0; c < kProductsF32; ++c)
#pragma unroll
                for (int ks = 0; ks < S::STEP / 16; ++ks)
                  umma_pair(d + (c < kProductsF32 - 1 ? 128 : 0), desc_add(ad, term_a(c) * S::A_TERM) + ks * a_step,
                            desc_add(bd, term_b(c) * S::B_TERM) + ks * b_step, idesc,
                            (i | ks | (c < kProductsF32 - 1 ? c : 0)) != 0);
            } else {
#pragma unroll
              for (int ks = 0; ks < BK / 16; ++ks)
                umma_pair(d, ad + ks * a_step, bd + ks * b_step, idesc, (i | ks) != 0);
            }
            umma_commit_pair_both(empty(s));
            ad += S::STAGE_BYTES >> 4;
            bd += S::STAGE_BYTES >> 4;
            if (++s == STAGES) {
              s = 0;
              ph ^= 1;
              ad = a_base;
              bd = b_base;
            }
          }
          if (!ok) break;
          umma_commit_pair_both(acc_full(buf));
          buf ^= 1;
          if (buf == 0) bph ^= 1;
        }
      }
      // Every MMA has completed before TMEM is freed, whether or not a consumer gave up.
      umma_commit_pair(drain);
      mbar_wait_drain(drain, 0, launch.err);
    }
  } else {
    // Each warp: its lane quarter's 32 rows, every second (one of the two warps of its group and
    // quarter) or fourth block of 32 columns.
    const int q = warp & 3, ew = warp - 2, group = ew >> 3;
    const int first = launch.alternate ? (ew >> 2) & 1 : ew >> 2, step = launch.alternate ? 2 : 4;
    constexpr int WIDTH = GATE ? BN / 2 : BN;  // output columns of a tile
    uint8_t *const block = smem + S::OFF_STAGE + ew * S::SLOT_BYTES;
    const uint32_t block_addr = sbase + S::OFF_STAGE + ew * S::SLOT_BYTES;
    int acc_it = 0, stores = 0, loads = 0;  // stores, loads: through the two blocks in turn
    Walk<LIMIT> walk{launch, pair, npairs};
    for (int t; walk.next(t); ++acc_it) {
      if (launch.alternate && (acc_it & 1) != group) continue;
      const Product &product = product_of(launch, t);
      const Maps &maps = product.maps;
      const Args &p = product.args;
      const Tile tile = tile_at(p, t);
      const int r0 = tile.mi * PAIR_M + rank * BM + q * 32;  // the warp's first row
      const int64_t m = static_cast<int64_t>(r0) + lane;
      const int n0 = tile.ni * WIDTH;
      // this warp's blocks of the tile: first, first + step, ... below `end`
      // (the f32 gate's are 16 columns wide: a warp has those of the gate and of the value)
      constexpr int SHIFT = F32 && GATE ? 4 : 5;
      const int end = r0 < p.m ? min(WIDTH >> SHIFT, (p.n - n0 + (1 << SHIFT) - 1) >> SHIFT) : 0;
      bool ok = true;
      // f32: the sums of each part of the depth, into registers (each warp has one block: BN is 128)
      [[maybe_unused]] float sums[32];
      auto add_part = [&](int b) {
        const uint32_t at0 = tmem + (static_cast<uint32_t>(q * 32) << 16) + b * 256 + (first << SHIFT);
#pragma unroll
        for (int c = 0; c < 32; c += 16) {  // (all at once takes more registers than there are)
          uint32_t r[16], small[16];
          const uint32_t at = at0 + (GATE && c ? WIDTH : c);
          tmem_ld16(at, r);
          tmem_ld16(at + 128, small);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) sums[c + i] += __uint_as_float(r[i]) + __uint_as_float(small[i]);
        }
      };
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) sums[i] = 0.f;
        int steps = p.k_blocks;
        if (p.splits > 1) steps = k_begin(p, tile.split + 1) - k_begin(p, tile.split);
        for (int from = kPromote; from < steps; from += kPromote, ++acc_it) {  // (the last part below)
          const int b = acc_it & 1;
          ok = warp_wait(acc_full(b), (acc_it >> 1) & 1, abort_flag, launch.err, kErrWaitEpilogue);
          if (!ok) break;
          tc_fence_after();
          if (first < end) add_part(b);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader_relaxed(acc_empty(b));
        }
        if (!ok) break;
      }
      const int buf = acc_it & 1;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + buf * 256;
      const uint32_t acc_phase = (acc_it >> 1) & 1;

      if constexpr (KIND == kGateBackward && F32) {
        // dg = dh v act'(g) and dv = dh act(g) from the saved g and v, 16 columns at a time: g and v come
        // into the warp's blocks, the terms of dg and dv leave from each lane along its row.
        const int blocks = first < end ? min(2, (p.n - n0 - first * 32 + 15) >> 4) : 0;
        auto fetch = [&](int c) {
          if (lane == 0) {
            mbar_arrive_expect_tx(load(ew, 0), 4096);
            tma_load_3d(block_addr, &maps.half, load(ew, 0), c, r0, 0);
            tma_load_3d(block_addr + 2048, &maps.half, load(ew, 0), c, r0, 1);
          }
        };
        if (blocks) fetch(n0 + first * 32);
        if (!warp_wait(acc_full(buf), acc_phase, abort_flag, launch.err, kErrWaitEpilogue)) {
          if (blocks && lane == 0) mbar_wait_drain(load(ew, 0), loads & 1, launch.err);
          break;
        }
        tc_fence_after();
        if (blocks) add_part(buf);
        // (rolled, the second half's sums moved to the first's place: a small launch runs this code once,
        // and reading it takes longer than running it)
#pragma unroll 1
        for (int half = 0; half < blocks; ++half) {
          const int c0 = n0 + first * 32 + 16 * half;
          ok = warp_wait(load(ew, 0), loads & 1, abort_flag, launch.err, kErrWaitEpilogue);
          if (!ok) {
            if (lane == 0) mbar_wait_drain(load(ew, 0), loads & 1, launch.err);
            break;
          }
          ++loads;
          float d[32];  // g and v, then dg and dv
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float4 u = *reinterpret_cast<const float4 *>(piece16(block + (c >> 2) * 2048, lane, c & 3));
            d[4 * c] = u.x, d[4 * c + 1] = u.y, d[4 * c + 2] = u.z, d[4 * c + 3] = u.w;
          }
          fence_async_smem();
          __syncwarp();  // every lane has read g and v
          if (half + 1 < blocks) fetch(c0 + 16);
          with_activation(p.activation, [&](auto act) {
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float2 dh = make_float2(sums[i], sums[i + 1]);
              const float2 v = make_float2(d[16 + i], d[16 + i + 1]);
              float2 value, slope;
              activate_slope2<decltype(act)::value, false>(make_float2(d[i], d[i + 1]), value, slope);
              const float2 dg = f2mul(f2mul(dh, v), slope), dv = f2mul(dh, value);
              d[i] = dg.x, d[i + 1] = dg.y;
              d[16 + i] = dv.x, d[16 + i + 1] = dv.y;
            }
          });
          if (m < p.m)
#pragma unroll
            for (int set = 0; set < 2; ++set)
              store_terms16(static_cast<uint16_t *>(p.out[set]) + m * p.out_stride + c0, p.out_piece_stride,
                            reinterpret_cast<const float(&)[16]>(d[16 * set]));
          if (p.column_partial) {
            const float sum = lane_sums(d, lane);
            p.column_partial[(static_cast<int64_t>(r0 >> 5) * 2 + (lane >> 4)) * p.saved_pitch + c0 + (lane & 15)] = sum;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) sums[i] = sums[16 + i];
        }
        if (!ok) break;
      } else if constexpr (KIND == kGateBackward && !kBf16<OT>) {
        // f16: dg = dh p and dv = dh a with the saved factors p = v act'(g) and a = act(g) in f32, 16 columns at
        // a time: the factors come into the warp's blocks, dg and dv leave from each lane along its row.
        auto fetch = [&](int c) {
          if (lane == 0) {
            mbar_arrive_expect_tx(load(ew, 0), 4096);
            tma_load_3d(block_addr, &maps.half, load(ew, 0), c, r0, 0);
            tma_load_3d(block_addr + 2048, &maps.half, load(ew, 0), c, r0, 1);
          }
        };
        if (first < end) fetch(n0 + first * 32);
        if (!warp_wait(acc_full(buf), acc_phase, abort_flag, launch.err, kErrWaitEpilogue)) {
          if (first < end && lane == 0) mbar_wait_drain(load(ew, 0), loads & 1, launch.err);
          break;
        }
        tc_fence_after();
        int half = 0;
#pragma unroll 1
        for (int b = first; b < end;) {
          const int at = b * 32 + 16 * half, c0 = n0 + at;
          uint32_t dh[16];
          tmem_ld16(taddr + at, dh);
          ok = warp_wait(load(ew, 0), loads & 1, abort_flag, launch.err, kErrWaitEpilogue);
          if (!ok) {
            if (lane == 0) mbar_wait_drain(load(ew, 0), loads & 1, launch.err);
            break;
          }
          ++loads;
          float d[32];  // p and a, then dg and dv
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float4 u = *reinterpret_cast<const float4 *>(piece16(block + (c >> 2) * 2048, lane, c & 3));
            d[4 * c] = u.x, d[4 * c + 1] = u.y, d[4 * c + 2] = u.z, d[4 * c + 3] = u.w;
          }
          fence_async_smem();
          __syncwarp();  // every lane has read p and a
          if (half == 0 && c0 + 16 < p.n) {
            half = 1;
          } else {
            half = 0;
            b += step;
          }
          if (b < end) fetch(n0 + b * 32 + 16 * half);
          tmem_ld_wait();
#pragma unroll
          for (int set = 0; set < 2; ++set) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float *x = d + 16 * set + 2 * i;
              const float2 f = f2mul(make_float2(x[0], x[1]),
                                     make_float2(__uint_as_float(dh[2 * i]), __uint_as_float(dh[2 * i + 1])));
              x[0] = f.x, x[1] = f.y;
              w[i] = pack2_t<OT>(f.x, f.y);
            }
            if (m < p.m) store_sector(static_cast<OT *>(p.out[set]) + m * p.out_stride + c0, w);
          }
          if (p.column_partial) {
            const float sum = lane_sums(d, lane);
            p.column_partial[(static_cast<int64_t>(r0 >> 5) * 2 + (lane >> 4)) * p.saved_pitch + c0 + (lane & 15)] = sum;
          }
        }
        if (!ok) break;
      } else if constexpr (KIND == kGateBackward) {
        // dg = dh p and dv = dh a with the saved factors p = v act'(g) and a = act(g).  A block's
        // factors come into the warp's two blocks and the products leave from the same place.
        auto fetch = [&](int b) {
          if (lane == 0) {
            bulk_wait_read_all();  // the products before them have left
            mbar_arrive_expect_tx(load(ew, 0), 4096);
            tma_load_3d(block_addr, &maps.half, load(ew, 0), n0 + b * 32, r0, 0);
            tma_load_3d(block_addr + 2048, &maps.half, load(ew, 0), n0 + b * 32, r0, 1);
          }
        };
        if (first < end) fetch(first);
        if (!warp_wait(acc_full(buf), acc_phase, abort_flag, launch.err, kErrWaitEpilogue)) {
          if (first < end && lane == 0) mbar_wait_drain(load(ew, 0), loads & 1, launch.err);
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int b = first; b < end; b += step) {
          const int c0 = n0 + b * 32;
          if (b != first) fetch(b);
          uint32_t v[32];
          tmem_ld32(taddr + b * 32, v);
          const uint32_t scales = p.saved_scale[(c0 >> 5) * p.scale_rows + m];
          ok = warp_wait(load(ew, 0), loads & 1, abort_flag, launch.err, kErrWaitEpilogue);
          tmem_ld_wait();
          if (!ok) {
            if (lane == 0) mbar_wait_drain(load(ew, 0), loads & 1, launch.err);
            break;
          }
          ++loads;
#pragma unroll
          for (int plane = 0; plane < 2; ++plane) {
            float d[32];
#pragma unroll
            for (int c = 0; c < 4; ++c) {  // 8 columns each
              const float scale = factor_scale((scales >> (16 * plane + 8 * (c >> 1))) & 0xffu);
              uint4 *piece = piece16(block + plane * 2048, lane, c);
              const uint4 u = *piece;
              uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 dh = make_float2(__uint_as_float(v[8 * c + 2 * i]), __uint_as_float(v[8 * c + 2 * i + 1]));
                const float2 f = f2mul(factor_values(w[i], scale), dh);
                w[i] = pack2_t<OT>(f.x, f.y);
                d[8 * c + 2 * i] = f.x;
                d[8 * c + 2 * i + 1] = f.y;
              }
              *piece = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (p.column_partial) {
              // the bias gradients' sums, of the products before they are rounded
              const float sum = lane_sums(d, lane);
              p.column_partial[(static_cast<int64_t>(r0 >> 5) * 2 + plane) * p.saved_pitch + c0 + lane] = sum;
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&maps.out[0], block_addr, c0, r0, 0);
            tma_store_3d(&maps.out[1], block_addr + 2048, c0, r0, 0);
            bulk_commit();
          }
        }
        if (!ok) break;
      } else if constexpr (GATE) {
        // h = act(g) v; columns [0, BN / 2) of the accumulator are g, the others v
        constexpr bool CODES = KIND == kGateSave && kBf16<OT>;  // factors leave through blocks of their own
        if (!warp_wait(acc_full(buf), acc_phase, abort_flag, launch.err, kErrWaitEpilogue)) break;
        tc_fence_after();
        if constexpr (F32) {
          if (first < end) {
            add_part(buf);
            const int c0 = n0 + first * 16, cols = min(16, p.n - c0);
#pragma unroll
            for (int set = 0; set < 2; ++set) {
              const float *bias = static_cast<const float *>(p.bias[set]);
              float *z = sums + 16 * set;
              if (bias && p.vector_bias && cols == 16) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float4 u = __ldg(reinterpret_cast<const float4 *>(bias + c0) + i);
                  z[4 * i] += u.x, z[4 * i + 1] += u.y, z[4 * i + 2] += u.z, z[4 * i + 3] += u.w;
                }
              } else if (bias) {
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] += i < cols ? __ldg(bias + c0 + i) : 0.f;
              }
            }
            // h as three terms, g and v, from each lane along its row
            if (m < p.m) {
              with_activation(p.activation, [&](auto act) {
                float h[16];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                  const float2 a = activate2<decltype(act)::value, false>(make_float2(sums[i], sums[i + 1]));
                  h[i] = a.x * sums[16 + i];
                  h[i + 1] = a.y * sums[16 + i + 1];
                }
                store_terms16(static_cast<uint16_t *>(p.out[0]) + m * p.out_stride + c0, p.out_piece_stride, h);
              });
              if constexpr (KIND == kGateSave) {
#pragma unroll
                for (int set = 0; set < 2; ++set)
#pragma unroll
                  for (int c = 0; c < 16; c += 8) {
                    const float *z = sums + 16 * set + c;
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(z[i]);
                    store_sector(p.saved_f32 + set * p.saved_stride + m * p.saved_pitch + c0 + c, w);
                  }
              }
            }
          }
        } else
#pragma unroll 1
        for (int b = first; b < end; b += step) {
          const int c0 = n0 + b * 32;
          const uint32_t at = CODES ? 0 : (stores++ & 1) * 2048;
          uint32_t scales = 0;
#pragma unroll
          for (int part = 0; part < 2; ++part) {  // 16 columns each
            uint32_t g[16], v[16], bg[8] = {}, bv[8] = {};
            tmem_ld16(taddr + b * 32 + part * 16, g);
            tmem_ld16(taddr + WIDTH + b * 32 + part * 16, v);
            if (p.bias[0]) load_raw16(static_cast<const OT *>(p.bias[0]), c0 + part * 16, p.n, p.vector_bias, bg);
            if (p.bias[1]) load_raw16(static_cast<const OT *>(p.bias[1]), c0 + part * 16, p.n, p.vector_bias, bv);
            tmem_ld_wait();
            uint32_t h[8], pw[8], aw[8];
            with_activation(p.activation, [&](auto act) {
              constexpr int ACT = decltype(act)::value;
              float2 pf[8], af[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 gz = f2add(make_float2(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1])),
                                        unpack2<OT>(bg[i]));
                const float2 vz = f2add(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])),
                                        unpack2<OT>(bv[i]));
                if constexpr (KIND == kGateSave) {
                  activate_slope2<ACT, true>(gz, af[i], pf[i]);
                  pf[i] = f2mul(pf[i], vz);
                } else {
                  af[i] = activate2<ACT, true>(gz);
                }
                const float2 hz = f2mul(af[i], vz);
                h[i] = pack2_t<OT>(hz.x, hz.y);
              }
              if constexpr (CODES) {
                scales |= factor_block(pf, pw) << (8 * part) | factor_block(af, aw) << (16 + 8 * part);
              } else if constexpr (KIND == kGateSave) {  // f32, from each lane along its row
                if (m < p.m)
#pragma unroll
                  for (int set = 0; set < 2; ++set)
#pragma unroll
                    for (int c = 0; c < 8; c += 4) {
                      const float2 *f = (set ? af : pf) + c;
                      uint32_t w[8];
#pragma unroll
                      for (int i = 0; i < 4; ++i) w[2 * i] = __float_as_uint(f[i].x), w[2 * i + 1] = __float_as_uint(f[i].y);
                      store_sector(p.saved_f32 + set * p.saved_stride + m * p.saved_pitch + c0 + part * 16 + 2 * c, w);
                    }
              }
            });
            if (part == 0) {
              // the blocks are free once what left from them before has been read
              if (lane == 0) {
                if (CODES)
                  bulk_wait_read_all();
                else
                  bulk_wait_read_but_one();
              }
              __syncwarp();
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int pc = part * 2 + c;
              *piece16(block + at, lane, pc) = make_uint4(h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
              if constexpr (CODES) {
                *piece16(block + 2048, lane, pc) = make_uint4(pw[4 * c], pw[4 * c + 1], pw[4 * c + 2], pw[4 * c + 3]);
                *piece16(block + 4096, lane, pc) = make_uint4(aw[4 * c], aw[4 * c + 1], aw[4 * c + 2], aw[4 * c + 3]);
              }
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&maps.out[0], block_addr + at, c0, r0, 0);
            if constexpr (CODES) {
              tma_store_3d(&maps.half, block_addr + 2048, c0, r0, 0);
              tma_store_3d(&maps.half, block_addr + 4096, c0, r0, 1);
            }
            bulk_commit();
          }
          if constexpr (CODES) p.saved_scale[(c0 >> 5) * p.scale_rows + m] = scales;
        }
      } else {
        // out = act(acc + bias) (+ residual)
        constexpr bool PLAIN = KIND == kProducts, LANES = KIND == kOutRows || PLAIN;
        const int partial = p.partial;
        const bool tma_residual = !PLAIN && p.tma_residual;
        const OT *residual = PLAIN ? nullptr : static_cast<const OT *>(p.residual);
        const int z = partial ? tile.split * static_cast<int>(p.batches.d) + tile.z : 0;
        const CUtensorMap *omap = &maps.out[partial ? 0 : tile.z];
        // The residual's blocks come ahead, each into the block that its result leaves from: the two in
        // turn, the second where the first holds slopes (f32: the two halves of the warp's only block of
        // columns).
        const bool keep = (KIND == kOutSave || KIND == kOutRows) && p.save;
        const bool staged = keep && kBf16<OT>;  // (f32 slopes leave from each lane)
        auto fetch = [&](int b, int at) {
          if (lane == 0) {
            bulk_wait_read_all();
            mbar_arrive_expect_tx(load(ew, at & 1), F32 ? 4096 : 2048);
            const uint32_t to = block_addr + (F32 ? 0 : 2048 * (staged ? 1 : at & 1));
            tma_load_3d(to, &maps.residual, load(ew, at & 1), n0 + b * 32, r0, 0);
            if (F32) tma_load_3d(to + 2048, &maps.residual, load(ew, at & 1), n0 + b * 32 + 16, r0, 0);
          }
        };
        const int rows = static_cast<int>(min(static_cast<int64_t>(32), p.m - r0));
        if (tma_residual && first < end) fetch(first, loads);
        // ... or by the lanes, into the second block
        const bool lane_residual = KIND == kOutRows && residual && !tma_residual;
        [[maybe_unused]] auto bring = [&](int b) {
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
          const int c = n0 + b * 32;
          move_rows<OT, true, 16>(block + 2048, const_cast<OT *>(residual) + static_cast<int64_t>(r0) * p.residual_stride + c,
                                  p.residual_stride, rows, min(32, p.n - c), lane);
          __syncwarp();
        };
        if constexpr (!F32) {
          if (lane_residual && first < end) bring(first);
        } else {
          if (lane_residual && first < end) {
            if (lane == 0) bulk_wait_read_all();
            __syncwarp();
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              const int c = n0 + first * 32 + 16 * h;
              move_rows<OT, true>(block + 2048 * h, const_cast<OT *>(residual) + static_cast<int64_t>(r0) * p.residual_stride + c,
                                  p.residual_stride, rows, min(16, p.n - c), lane);
            }
            __syncwarp();
          }
        }
        if (!warp_wait(acc_full(buf), acc_phase, abort_flag, launch.err, kErrWaitEpilogue)) {
          if (tma_residual && first < end && lane == 0) mbar_wait_drain(load(ew, loads & 1), (loads >> 1) & 1, launch.err);
          break;
        }
        tc_fence_after();
        if constexpr (F32) {
          if (first < end) {
            if (tma_residual) {
              ok = warp_wait(load(ew, loads & 1), (loads >> 1) & 1, abort_flag, launch.err, kErrWaitEpilogue);
              if (!ok) {
                if (lane == 0) mbar_wait_drain(load(ew, loads & 1), (loads >> 1) & 1, launch.err);
                break;
              }
              ++loads;
            }
            const float *bias = PLAIN || partial ? nullptr : static_cast<const float *>(p.bias[tile.z]);
            add_part(buf);
            // (rolled, the second half's sums moved to the first's place: a small launch runs this code
            // once, and reading it takes longer than running it)
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              const int c0 = n0 + first * 32 + 16 * h;
              if (c0 >= p.n) break;
              float *y = sums;
              const int cols = min(16, p.n - c0);
              if (bias) {
                if (p.vector_bias && cols == 16) {
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const float4 u = __ldg(reinterpret_cast<const float4 *>(bias + c0) + i);
                    y[4 * i] += u.x, y[4 * i + 1] += u.y, y[4 * i + 2] += u.z, y[4 * i + 3] += u.w;
                  }
                } else {
#pragma unroll
                  for (int i = 0; i < 16; ++i) y[i] += i < cols ? __ldg(bias + c0 + i) : 0.f;
                }
              }
              if (!PLAIN && !partial && p.activation != AF2_ACTIVATION_NONE)
                with_activation(p.activation, [&](auto act) {
                  constexpr int ACT = decltype(act)::value;
                  if (keep) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                      float2 value[2], s[2];
#pragma unroll
                      for (int i = 0; i < 2; ++i)
                        activate_slope2<ACT, false>(make_float2(y[4 * c + 2 * i], y[4 * c + 2 * i + 1]), value[i], s[i]);
                      y[4 * c] = value[0].x, y[4 * c + 1] = value[0].y, y[4 * c + 2] = value[1].x, y[4 * c + 3] = value[1].y;
                      if (m < p.m)
                        *reinterpret_cast<float4 *>(p.saved_f32 + m * p.saved_pitch + c0 + 4 * c) =
                            make_float4(s[0].x, s[0].y, s[1].x, s[1].y);
                    }
                  } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                      const float2 v2 = activate2<ACT, false>(make_float2(y[2 * i], y[2 * i + 1]));
                      y[2 * i] = v2.x;
                      y[2 * i + 1] = v2.y;
                    }
                  }
                });
              // out of the half's own block where the residual is in it, else of the two in turn
              const uint32_t at = 2048u * (residual ? h : stores++ & 1);
              uint8_t *const dst = block + at;
              if (!residual) {
                if (lane == 0) bulk_wait_read_but_one();
                __syncwarp();
              }
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                float4 o = make_float4(y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]);
                float4 *piece = reinterpret_cast<float4 *>(piece16(dst, lane, c));
                if (residual) {
                  const float4 res = *piece;
                  o.x += res.x, o.y += res.y, o.z += res.z, o.w += res.w;
                }
                *piece = o;
              }
              if (!LANES || p.tma_out) {
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                  tma_store_3d(omap, block_addr + at, c0, r0, z);
                  bulk_commit();
                }
              } else {
                __syncwarp();
                move_rows<OT, false>(dst, static_cast<OT *>(p.out[tile.z]) + static_cast<int64_t>(r0) * p.out_stride + c0,
                                     p.out_stride, rows, cols, lane);
                __syncwarp();
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) sums[i] = sums[16 + i];
            }
          }
        } else {
#pragma unroll 1
        for (int b = first; b < end; b += step) {
          const int c0 = n0 + b * 32;
          uint32_t r[32];
          tmem_ld32(taddr + b * 32, r);
          if (tma_residual && !staged && b + step < end) fetch(b + step, loads + 1);
          float(&y)[32] = reinterpret_cast<float(&)[32]>(r);
          const int cols = min(32, p.n - c0);
          const OT *bias = PLAIN || partial ? nullptr : static_cast<const OT *>(p.bias[tile.z]);
          uint32_t bw[2][8] = {};
          if (bias) {
            load_raw16(bias, c0, p.n, p.vector_bias, bw[0]);
            load_raw16(bias, c0 + 16, p.n, p.vector_bias, bw[1]);
          }
          tmem_ld_wait();
          if (bias) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 s2 = f2add(make_float2(y[2 * i], y[2 * i + 1]), unpack2<OT>(bw[i >> 3][i & 7]));
              y[2 * i] = s2.x;
              y[2 * i + 1] = s2.y;
            }
          }
          if (!PLAIN && !partial && p.activation != AF2_ACTIVATION_NONE) {
            if (keep) {  // the slopes: f32 along each lane's row, or 16 bits through the first block
              if (staged) {
                if (lane == 0) bulk_wait_read_all();
                __syncwarp();
              }
              with_activation(p.activation, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  float2 s[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    float2 v2;
                    activate_slope2<ACT, true>(make_float2(y[8 * c + 2 * i], y[8 * c + 2 * i + 1]), v2, s[i]);
                    y[8 * c + 2 * i] = v2.x;
                    y[8 * c + 2 * i + 1] = v2.y;
                  }
                  if constexpr (kBf16<OT>) {
                    *piece16(block, lane, c) = make_uint4(slope_codes(s[0]), slope_codes(s[1]),
                                                          slope_codes(s[2]), slope_codes(s[3]));
                  } else if (m < p.m) {
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[2 * i] = __float_as_uint(s[i].x), w[2 * i + 1] = __float_as_uint(s[i].y);
                    store_sector(p.saved_f32 + m * p.saved_pitch + c0 + 8 * c, w);
                  }
                }
              });
              if (staged) {
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                  tma_store_3d(&maps.half, block_addr, c0, r0, 0);
                  bulk_commit();
                }
              }
            } else {
              with_activation(p.activation, [&](auto act) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float2 v2 = activate2<decltype(act)::value, true>(make_float2(y[2 * i], y[2 * i + 1]));
                  y[2 * i] = v2.x;
                  y[2 * i + 1] = v2.y;
                }
              });
            }
          }
          if (partial) {  // the f32 sums, through both blocks
            if (lane == 0) bulk_wait_read_all();
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *piece32(block, lane, c) = make_float4(y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(omap, block_addr, c0, r0, z);
              bulk_commit();
            }
            continue;
          }
          // the block that the result leaves from, with the residual in it where there is one
          const uint32_t at = 2048u * (staged || lane_residual ? 1 : tma_residual ? loads & 1 : stores++ & 1);
          uint8_t *const dst = block + at;
          if (tma_residual) {
            ok = warp_wait(load(ew, loads & 1), (loads >> 1) & 1, abort_flag, launch.err, kErrWaitEpilogue);
            if (!ok) {
              if (lane == 0) {
                mbar_wait_drain(load(ew, loads & 1), (loads >> 1) & 1, launch.err);
                ++loads;
                if (!staged && b + step < end) mbar_wait_drain(load(ew, loads & 1), (loads >> 1) & 1, launch.err);
              }
              break;
            }
            ++loads;
          } else if (!lane_residual) {
            if (lane == 0) {
              if (PLAIN)
                bulk_wait_read_all();  // (f32 sums of another product may be leaving both blocks)
              else
                bulk_wait_read_but_one();
            }
            __syncwarp();
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint4 *piece = piece16(dst, lane, c);
            uint32_t w[4];
            if (residual) {
              const uint4 u = *piece;
              w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float2 o = make_float2(y[8 * c + 2 * i], y[8 * c + 2 * i + 1]);
              if (residual) o = f2add(o, unpack2<OT>(w[i]));
              w[i] = pack2_t<OT>(o.x, o.y);
            }
            *piece = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (!LANES || p.tma_out) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(omap, block_addr + at, c0, r0, z);
              bulk_commit();
            }
          } else {
            __syncwarp();
            move_rows<OT, false>(dst, static_cast<OT *>(p.out[tile.z]) + static_cast<int64_t>(r0) * p.out_stride + c0,
                                 p.out_stride, rows, cols, lane);
            __syncwarp();
          }
          if (tma_residual && staged && b + step < end) fetch(b + step, loads);
          if (lane_residual && b + step < end) bring(b + step);
        }
        }
        if (!ok) break;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader_relaxed(acc_empty(buf));
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  cluster_sync_all();  // the pair's MMAs and loads are done before either CTA releases TMEM or exits
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---- what follows the products ---------------------------------------------------

// out = act(sum of the splits' partial sums + bias) (+ residual), saved = the slope.
struct ReduceArgs {
  const float *partial;  // [split][batch][m][pitch]
  int splits, batch, activation;
  int64_t m, n, pitch;
  void *out[2];
  int64_t out_stride;
  const void *bias[2];
  const void *residual;
  int64_t residual_stride;
  uint16_t *saved_half;
  float *saved_f32;
  int64_t saved_pitch;
};

// The column sums (blockIdx.y below `sum_count`), whose few blocks run longest, then the split products'
// sums: one launch for both.
struct FinishLaunch {
  ReduceArgs product[kMaxProducts];
  ColumnSums sums[kMaxSums];
  int products, sum_count;
};

// A thread has four columns of a row; latency bounds it, so all that it reads is asked for at once (some
// 3 us for a small layer's sums).
template <typename OT>
__device__ __forceinline__ void reduce(const ReduceArgs &p) {
  // (a product is only split while it has few tiles: its elements count in 32 bits)
  const uint32_t quads = static_cast<uint32_t>(p.pitch / 4), rows = static_cast<uint32_t>(p.m);
  const uint32_t total = p.batch * rows * quads;
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
    const uint32_t row = i / quads, c0 = (i - row * quads) * 4, z = row / rows;
    const int64_t m = row - z * rows;
    const int cols = static_cast<int>(min(static_cast<int64_t>(4), p.n - c0));
    const OT *bias = static_cast<const OT *>(p.bias[z]);
    OT *out = static_cast<OT *>(p.out[z]) + m * p.out_stride + c0;
    float b[4] = {}, r[4] = {};
    if (bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < cols) b[j] = to_f32<OT>(bias[c0 + j]);
    }
    if (p.residual) {
      const OT *res = static_cast<const OT *>(p.residual) + m * p.residual_stride + c0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < cols) r[j] = to_f32<OT>(res[j]);
    }
    const float4 *src = reinterpret_cast<const float4 *>(p.partial) + i;
    float y[4] = {};
    for (int s0 = 0; s0 < p.splits; s0 += 8) {
      float4 part[8];
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s0 + s < p.splits) part[s] = src[static_cast<int64_t>(s0 + s) * total];
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s0 + s < p.splits) {
          y[0] += part[s].x;
          y[1] += part[s].y;
          y[2] += part[s].z;
          y[3] += part[s].w;
        }
    }
    float slope[4];
    with_activation(p.activation, [&](auto act) {
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        float2 value, slopes;
        activate_slope2<decltype(act)::value, sizeof(OT) == 2>(make_float2(y[j] + b[j], y[j + 1] + b[j + 1]), value, slopes);
        y[j] = value.x, y[j + 1] = value.y;
        slope[j] = slopes.x, slope[j + 1] = slopes.y;
      }
    });
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= cols) break;
      if constexpr (kBf16<OT>) {
        if (p.saved_half)
          p.saved_half[m * p.saved_pitch + c0 + j] = static_cast<uint16_t>(slope_codes(f2(slope[j])));
      } else {
        if (p.saved_f32) p.saved_f32[m * p.saved_pitch + c0 + j] = slope[j];
      }
      out[j] = from_f32<OT>(y[j] + r[j]);
    }
  }
}

// dst[c] = the sum over the chunks of partial[chunk][c]: eight columns a block, 32 threads a column with
// sixteen reads in flight each, joined in a fixed order.
template <typename OT, typename ST>
__device__ __forceinline__ void column_sums(const ColumnSums &p) {
  __shared__ float all[8][8];
  const int c = threadIdx.x & 7, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t c0 = static_cast<int64_t>(blockIdx.x) * 8; c0 < p.columns; c0 += static_cast<int64_t>(gridDim.x) * 8) {
    float sum = 0.f;
    if (c0 + c < p.columns) {
      const ST *src = static_cast<const ST *>(p.partial) + c0 + c;
      for (int64_t k0 = threadIdx.x >> 3; k0 < p.chunks; k0 += 16 * 32) {
        ST x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = src[min(k0 + 32 * i, p.chunks - 1) * p.stride];
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += k0 + 32 * i < p.chunks ? to_f32<ST>(x[i]) : 0.f;
      }
    }
    sum += __shfl_xor_sync(kFull, sum, 8);
    sum += __shfl_xor_sync(kFull, sum, 16);
    if (lane < 8) all[warp][lane] = sum;
    __syncthreads();
    if (threadIdx.x < 8 && c0 + c < p.columns) {
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) total += all[w][c];
      static_cast<OT *>(p.out)[c0 + c] = from_f32<OT>(total);
    }
    __syncthreads();
  }
}

template <typename OT>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ FinishLaunch launch) {
  dependency_wait();
  const int y = blockIdx.y;
  if (y >= launch.sum_count)
    reduce<OT>(launch.product[y - launch.sum_count]);
  else if (launch.sums[y].rows)
    column_sums<OT, OT>(launch.sums[y]);
  else
    column_sums<OT, float>(launch.sums[y]);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool aligned16(const void *ptr, int64_t stride, int element) {
  return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && (stride * element) % 16 == 0 &&
         stride * element < (int64_t(1) << 40);
}

bool operand_map(af2_ctx *ctx, CUtensorMap *map, const GemmOperand &o, int64_t outer, int64_t k, bool bf16, int pieces,
                 int box_outer) {
  const CUtensorMapDataType t = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t row = o.pitch * 2, piece = pieces > 1 ? o.piece_stride * 2 : row;  // (one piece: no step)
  const int step = pieces > 1 ? 32 : BK;
  if (o.mn_major)
    return layer_map_3d(ctx, map, t, o.ptr, outer, k, pieces, row, piece, 64, step, 1, CU_TENSOR_MAP_SWIZZLE_128B);
  return layer_map_3d(ctx, map, t, o.ptr, k, outer, pieces, row, piece, step, box_outer, 1,
                       pieces > 1 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

int launch_pairs(const af2_ctx *ctx, int tiles) { return std::min(tiles, std::max(1, ctx->sm_count / 2)); }

template <int KIND, typename OT, int BN>
af2_status launch(af2_ctx *ctx, Launch<KIND == kProducts ? kMaxProducts : 1> &l, cudaStream_t stream) {
  constexpr uint32_t smem = Shape<KIND, BN, OT>::BYTES;
  auto kernel = layer_gemm_kernel<KIND, OT, BN>;
  static std::atomic<uint64_t> allowed{0};  // devices on which this kernel has its shared memory
  const uint64_t bit = uint64_t(1) << (ctx->device & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit) || ctx->device > 63) {
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        e != cudaSuccess)
      return cuda_fail(ctx, e, "layer product shared memory");
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const int pairs = launch_pairs(ctx, l.total_tiles);
  // Two groups of eight warps take tiles in turn where a tile has at most four blocks of columns, so that
  // some warps would have none of it; otherwise all take each tile, whose accumulator is then free sooner
  // (60690 x 424 -> 736: 60.5 us in turn, 54.1 together; 163578 x 112 -> 40: 22.4 and 29.4).
  const int width = std::min(KIND == kGate || KIND == kGateSave ? BN / 2 : BN, l.product[0].args.n);
  l.alternate = l.total_tiles > pairs && sizeof(OT) == 2 && width <= 128;
  LaunchScope scope(ctx, stream, kProfLayerGemm);
  if (cudaError_t e = launch_early(kernel, dim3(2 * pairs), THREADS, smem, stream, l); e != cudaSuccess)
    return cuda_fail(ctx, e, "layer product");
  return AF2_OK;
}

template <int KIND, typename OT, int N>
af2_status launch_bn(af2_ctx *ctx, int bn, Launch<N> &l, cudaStream_t stream) {
  // f32 tiles are 128 wide: a warp holds the sums of one block of 32 columns
  if constexpr (sizeof(OT) == 4)
    return launch<KIND, OT, 128>(ctx, l, stream);
  else
    return bn == 256 ? launch<KIND, OT, 256>(ctx, l, stream) : launch<KIND, OT, 128>(ctx, l, stream);
}
// A 16-bit output type.
template <int KIND, int N>
af2_status launch_16(af2_ctx *ctx, int dtype, int bn, Launch<N> &l, cudaStream_t stream) {
  return dtype == AF2_F16 ? launch_bn<KIND, __half>(ctx, bn, l, stream)
                          : launch_bn<KIND, __nv_bfloat16>(ctx, bn, l, stream);
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == AF2_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : dtype == AF2_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                            : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

}  // namespace

namespace {

// Tiles of one length.
struct TileClass {
  int64_t tiles;
  double clocks;  // of each
};

// Tiles of several lengths, the longest first, dealt out to `pairs`: always to the pairs that have the
// least to do, neighbours within half a tile of one another together.  Returns the clocks of the pair that
// has the most; fills in the waves.
double deal(const TileClass *classes, int count, int pairs, Waves *waves) {
  struct Run { int at, pairs; double load; } run[kMaxWaves];
  int runs = 1, n = 0, first = 0;
  run[0] = {0, pairs, 0};
  bool fits = true;
  for (int j = 0; j < count && fits; ++j) {
    const double cost = classes[j].clocks;
    for (int64_t left = classes[j].tiles; left > 0 && fits;) {
      int lo = 0;
      for (int i = 1; i < runs; ++i)
        if (run[i].load < run[lo].load) lo = i;
      const double least = run[lo].load + cost / 2;
      int hi = lo;
      while (lo > 0 && run[lo - 1].load <= least) --lo;
      while (hi + 1 < runs && run[hi + 1].load <= least) ++hi;
      for (int i = lo + 1; i <= hi; ++i) {
        run[lo].pairs += run[i].pairs;
        run[lo].load = std::max(run[lo].load, run[i].load);
      }
      std::copy(run + hi + 1, run + runs, run + lo + 1);
      runs -= hi - lo;
      Run &r = run[lo];
      int64_t turns = left / r.pairs;
      for (int i = 0; i < runs; ++i)
        if (i != lo) turns = std::min(turns, std::max<int64_t>(1, std::llround((run[i].load - r.load) / cost)));
      if (n == kMaxWaves || (turns == 0 && runs == kMaxWaves)) {
        fits = false;
      } else if (turns > 0) {
        if (waves) waves->wave[n] = {first, static_cast<int>(turns), r.at, r.pairs};
        r.load += turns * cost;
        first += static_cast<int>(turns * r.pairs);
        left -= turns * r.pairs;
      } else {  // fewer tiles than pairs
        std::copy_backward(run + lo + 1, run + runs, run + runs + 1);
        ++runs;
        run[lo + 1] = {r.at + static_cast<int>(left), r.pairs - static_cast<int>(left), r.load};
        if (waves) waves->wave[n] = {first, 1, r.at, static_cast<int>(left)};
        run[lo].pairs = static_cast<int>(left);
        run[lo].load += cost;
        first += static_cast<int>(left);
        left = 0;
      }
      ++n;
    }
  }
  double most = 0;
  if (fits) {
    for (int i = 0; i < runs; ++i) most = std::max(most, run[i].load);
  } else {  // too many waves: every product's tiles to all pairs in turn
    n = first = 0;
    for (int j = 0; j < count; ++j) {
      const int turns = static_cast<int>(classes[j].tiles / pairs), rest = static_cast<int>(classes[j].tiles % pairs);
      if (waves) {
        if (turns) waves->wave[n++] = {first, turns, 0, pairs};
        if (rest) waves->wave[n++] = {first + turns * pairs, 1, 0, rest};
      }
      first += static_cast<int>(classes[j].tiles);
      most += (turns + (rest ? 1 : 0)) * classes[j].clocks;
    }
  }
  if (waves) waves->count = n;
  return most;
}

// What a launch costs in SM clocks: a K step of 64 takes 512 (BN = 256) or 420 (BN = 128; the ring's
// latency) clocks, in f32 900 for 32, a tile's hand-over 800.
double step_clocks(bool f32, int bn) { return f32 ? 900 : bn == 256 ? 512 : 420; }
TileClass tile_class(const LayerGemm &g, int bn, int splits) {
  const bool f32 = g.pieces > 1;
  const int64_t k_blocks = ceil_div(g.k, f32 ? 32 : BK);
  const int width = g.epilogue == kEpilogueGate ? bn / 2 : bn;
  return {splits * g.batch * ceil_div(g.m, PAIR_M) * ceil_div(g.n, width),
          ceil_div(k_blocks, splits) * g.segments * step_clocks(f32, bn) + 800};
}
int split_limit(const LayerGemm &g) {
  if (g.batch * g.m * align_up(g.n, 4) >= int64_t(1) << 31) return 1;
  return static_cast<int>(std::min<int64_t>((ceil_div(g.k, g.pieces > 1 ? 32 : BK) + 1) / 2, 64));
}
// Split sums are written, read and reduced by another launch.
double split_clocks(double bytes) { return bytes > 0 ? 4000 + bytes / 2500 : 0; }
double split_bytes(const LayerGemm &g, int splits) {
  return splits > 1 ? 8.0 * splits * g.batch * g.m * align_up(g.n, 4) : 0;
}
double launch_clocks(TileClass *classes, int count, double bytes) {
  std::sort(classes, classes + count, [](const TileClass &a, const TileClass &b) { return a.clocks > b.clocks; });
  return 2500 + split_clocks(bytes) + deal(classes, count, kPairs, nullptr);
}

// The rows of g from `row` on (a multiple of 8) as a product of their own; g keeps those before.
LayerGemm cut_rows(LayerGemm &g, int64_t row) {
  LayerGemm tail = g;
  auto past = [&](const void *p, int64_t elements, int size) {
    return static_cast<const uint8_t *>(p) + elements * size;
  };
  for (int i = 0; i < g.segments; ++i)
    tail.a[i].ptr = past(g.a[i].ptr, g.a[i].mn_major ? row : row * g.a[i].pitch, 2);
  for (int i = 0; i < g.batch; ++i)
    tail.out[i] = const_cast<uint8_t *>(past(g.out[i], row * g.out_stride, g.out_dtype == AF2_F32 ? 4 : 2));
  tail.m = g.m - row;
  tail.first_row = row;
  g.m = row;
  return tail;
}

// Launches this long (SM clocks) are worth the host's search for a cut, some 20 us.
constexpr double kCutFrom = 200000;

// Tile width and the parts that each depth is cut into, by the clocks that the launch costs.  Where the
// tiles of long products leave pairs without work at the end, the last rows of one become a product of its
// own whose depth is cut: at 8192 x 1024 -> 4096 the gradients' 320 tiles fill 74 pairs 4.3 times, and
// 24 of them cut in three end all pairs together.
int search_plan(LayerGemm *g, int count) {
  const bool f32 = g[0].pieces > 1;
  TileClass classes[kMaxProducts];
  double best = 0;
  int64_t longest = 0;
  for (int i = 0; i < count; ++i) longest = std::max(longest, ceil_div(g[i].k, f32 ? 32 : BK) * g[i].segments);
  for (int bn : {256, 128}) {
    if (f32 && bn == 256) continue;
    // `most`: K steps that a tile may have before its depth is cut
    for (int64_t most : {int64_t(1) << 40, int64_t(512), int64_t(384), int64_t(256), int64_t(192), int64_t(128),
                         int64_t(96), int64_t(64), int64_t(48), int64_t(32), int64_t(24), int64_t(16), int64_t(12),
                         int64_t(8), int64_t(6), int64_t(4), int64_t(2)}) {
      if (most < int64_t(1) << 40 && (most >= longest || g[0].epilogue != kEpilogueOut)) continue;
      int splits[kMaxProducts];
      double bytes = 0;
      for (int i = 0; i < count; ++i) {
        const int64_t all = ceil_div(g[i].k, f32 ? 32 : BK) * g[i].segments;
        splits[i] = std::max(1, static_cast<int>(std::min<int64_t>(ceil_div(all, most), split_limit(g[i]))));
        classes[i] = tile_class(g[i], bn, splits[i]);
        bytes += split_bytes(g[i], splits[i]);
      }
      const double clocks = launch_clocks(classes, count, bytes);
      if (best == 0 || clocks < best) {
        best = clocks;
        for (int i = 0; i < count; ++i) {
          g[i].tile_n = bn;
          g[i].splits = splits[i];
        }
      }
    }
  }
  if (count > 1 && count < kMaxProducts && best > kCutFrom) {
    const int bn = g[0].tile_n;
    double whole = 0;
    for (int i = 0; i < count; ++i) whole += split_bytes(g[i], g[i].splits);
    int cut = -1, cut_splits = 0;
    int64_t cut_row = 0;
    for (int i = 0; i < count; ++i) {
      const int64_t tile_rows = ceil_div(g[i].m, PAIR_M), in_row = g[i].batch * ceil_div(g[i].n, bn);
      if (g[i].splits > 1) continue;
      for (int64_t rows = 1; rows < tile_rows && rows * in_row <= kPairs; ++rows)
        for (int splits = 2; splits <= std::min(8, split_limit(g[i])); ++splits) {
          LayerGemm head = g[i];
          const int64_t row = (tile_rows - rows) * PAIR_M;
          const LayerGemm tail = cut_rows(head, row);
          for (int j = 0; j < count; ++j) classes[j] = tile_class(j == i ? head : g[j], bn, g[j].splits);
          classes[count] = tile_class(tail, bn, splits);
          const double clocks = launch_clocks(classes, count + 1, whole + split_bytes(tail, splits));
          if (clocks < best) {
            best = clocks;
            cut = i;
            cut_splits = splits;
            cut_row = row;
          }
        }
    }
    if (cut >= 0) {
      g[count] = cut_rows(g[cut], cut_row);
      g[count++].splits = cut_splits;
    }
  }
  if (count > 1)  // (the waves take the longest tiles first)
    std::stable_sort(g, g + count, [&](const LayerGemm &a, const LayerGemm &b) {
      return tile_class(a, a.tile_n, a.splits).clocks > tile_class(b, b.tile_n, b.splits).clocks;
    });
  return count;
}

// A plan by the shapes that it was made for: it is asked for twice a call (to size the scratch, and to
// launch), and costs 2 us to 50.
struct KeptPlan {
  static constexpr int kGiven = kMaxProducts - 1, kWords = 1 + 6 * kGiven;
  int64_t shapes[kWords];
  int count;
  struct { int64_t first_row, m; int given, tile_n, splits; } product[kMaxProducts];
};

}  // namespace

int layer_gemm_plan(LayerGemm *g, int count) {
  static thread_local KeptPlan plans[64];
  int64_t shapes[KeptPlan::kWords] = {count};
  uint64_t hash = count;
  for (int i = 0; i < count; ++i) {
    const int64_t words[6] = {g[i].m, g[i].n, g[i].k, g[i].segments, g[i].batch | static_cast<int64_t>(g[i].pieces) << 32,
                              g[i].epilogue};
    for (int w = 0; w < 6; ++w) {
      shapes[1 + 6 * i + w] = words[w];
      hash = (hash ^ static_cast<uint64_t>(words[w])) * 0x9e3779b97f4a7c15ull;
    }
    g[i].given = i;
    g[i].first_row = 0;
  }
  KeptPlan &kept = plans[hash >> 58];
  if (!std::equal(shapes, shapes + KeptPlan::kWords, kept.shapes)) {
    LayerGemm made[kMaxProducts];
    std::copy(g, g + count, made);
    kept.count = search_plan(made, count);
    for (int i = 0; i < kept.count; ++i)
      kept.product[i] = {made[i].first_row, made[i].m, made[i].given, made[i].tile_n, made[i].splits};
    std::copy(shapes, shapes + KeptPlan::kWords, kept.shapes);
  }
  LayerGemm given[KeptPlan::kGiven];
  std::copy(g, g + count, given);
  for (int i = 0; i < kept.count; ++i) {
    const auto &k = kept.product[i];
    LayerGemm &q = g[i] = given[k.given];
    if (k.first_row) q = cut_rows(q, k.first_row);
    q.m = k.m;
    q.tile_n = k.tile_n;
    q.splits = k.splits;
    q.scratch_bytes = q.splits > 1 ? align_up(4ull * q.splits * q.batch * q.m * align_up(q.n, 4), 256) : 0;
  }
  return kept.count;
}

namespace {

// One product's maps and arguments; its tiles follow `first_tile`.
af2_status describe(af2_ctx *ctx, const LayerGemm &g, int64_t first_tile, Product *product, int64_t *tiles) {
  const bool gate = g.epilogue == kEpilogueGate;
  Maps &maps = product->maps;
  Args &p = product->args;
  p.m = g.m;
  p.n = static_cast<int>(g.n);
  p.k_blocks = static_cast<int>(ceil_div(g.k, g.pieces > 1 ? 32 : BK));
  p.splits = g.splits;
  p.segments = g.segments;
  p.batches = Divisor(g.batch);
  p.tiles_m = Divisor(static_cast<uint32_t>(ceil_div(g.m, PAIR_M)));
  p.tiles_n = Divisor(static_cast<uint32_t>(ceil_div(g.n, gate ? g.tile_n / 2 : g.tile_n)));
  *tiles = static_cast<int64_t>(p.splits) * g.batch * p.tiles_m.d * p.tiles_n.d;
  if (first_tile + *tiles > 0x3fffffff) return fail(ctx, AF2_ERR_UNSUPPORTED, "the product has too many tiles");
  p.first_tile = static_cast<int>(first_tile);
  p.a_mn = g.a[0].mn_major;
  p.b_mn = g.b[0].mn_major;
  p.bf16 = g.bf16;
  const int bsets = gate ? 2 : std::max(g.segments, g.batch);
  bool maps_ok = true;
  for (int i = 0; i < g.segments; ++i)
    maps_ok &= operand_map(ctx, &maps.a[i], g.a[i], g.m, g.k, g.bf16, g.pieces, BM);
  for (int i = 0; i < bsets; ++i)
    maps_ok &= operand_map(ctx, &maps.b[i], g.b[i], g.n, g.k, g.bf16, g.pieces, g.tile_n / 2);

  const int out_bytes = g.out_dtype == AF2_F32 ? 4 : 2;
  const int64_t pitch = align_up(g.n, 4);
  const int outs = g.epilogue == kEpilogueGateBackward ? 2 : g.batch;
  if (g.splits > 1) {
    p.partial = 1;
    p.tma_out = 1;
    maps_ok &= layer_map_3d(ctx, &maps.out[0], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, g.scratch, g.n, g.m, g.splits * g.batch,
                             pitch * 4, g.m * pitch * 4, g.pieces > 1 ? 16 : 32, 32, 1,
                             g.pieces > 1 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
  } else {
    p.activation = g.activation;
    p.residual = g.residual;
    p.residual_stride = g.residual_stride;
    if (g.residual && aligned16(g.residual, g.residual_stride, out_bytes)) {
      p.tma_residual = 1;
      const int64_t row = g.residual_stride * out_bytes;
      maps_ok &= layer_map_3d(ctx, &maps.residual, map_type(g.out_dtype), g.residual, g.n, g.m, 1, row, row,
                               out_bytes == 4 ? 16 : 32, 32, 1, CU_TENSOR_MAP_SWIZZLE_64B);
    }
    p.out_stride = g.out_stride;
    p.out_piece_stride = g.out_piece_stride;
    p.vector_bias = 1;
    p.tma_out = 1;
    for (int i = 0; i < 2; ++i) {
      p.out[i] = g.out[i];
      p.bias[i] = g.bias[i];
      if (g.bias[i] && reinterpret_cast<uintptr_t>(g.bias[i]) % 16 != 0) p.vector_bias = 0;
      if (i < outs && !aligned16(g.out[i], g.out_stride, out_bytes)) p.tma_out = 0;
    }
    const bool by_lanes = g.epilogue == kEpilogueGateBackward ? g.saved.f32 != nullptr
                                                               : g.epilogue == kEpilogueGate && out_bytes == 4;
    if (p.tma_out && !by_lanes)
      for (int i = 0; i < outs; ++i)
        maps_ok &= layer_map_3d(ctx, &maps.out[i], map_type(g.out_dtype), g.out[i], g.n, g.m, 1, g.out_stride * out_bytes,
                                 g.out_stride * out_bytes, out_bytes == 4 ? 16 : 32, 32, 1, CU_TENSOR_MAP_SWIZZLE_64B);
    p.save = g.saved.half || g.saved.f32;
    p.saved_f32 = g.saved.f32;
    p.saved_scale = g.saved.scale;
    p.saved_pitch = g.saved.pitch;
    p.saved_stride = g.saved.stride;
    p.scale_rows = g.saved.scale_rows;
    if (g.saved.half)
      maps_ok &= layer_map_3d(ctx, &maps.half, CU_TENSOR_MAP_DATA_TYPE_UINT16, g.saved.half, g.saved.pitch, g.m,
                               g.epilogue == kEpilogueOut ? 1 : 2, g.saved.pitch * 2, g.saved.stride * 2, 32, 32, 1,
                               CU_TENSOR_MAP_SWIZZLE_64B);
    if (g.epilogue == kEpilogueGateBackward && g.saved.f32)
      maps_ok &= layer_map_3d(ctx, &maps.half, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, g.saved.f32, g.n, g.m, 2, g.saved.pitch * 4,
                               g.saved.stride * 4, 16, 32, 1, CU_TENSOR_MAP_SWIZZLE_64B);
    p.column_partial = g.column_partial;
  }
  if (!maps_ok) return fail(ctx, AF2_ERR_CUDA, "cannot describe the layer's tensors to the TMA unit");
  return AF2_OK;
}

}  // namespace

namespace {

// Describes and launches the products; run(launch) picks the kernel.
template <int N, typename F>
af2_status describe_and_run(af2_ctx *ctx, const LayerGemm *g, int count, F &&run) {
  Launch<N> l{};
  l.products = count;
  l.err = ctx->err_word;
  int64_t total = 0;
  for (int j = 0; j < count; ++j) {
    int64_t tiles = 0;
    if (af2_status st = describe(ctx, g[j], total, &l.product[j], &tiles); st != AF2_OK) return st;
    total += tiles;
  }
  l.total_tiles = static_cast<int>(total);
  if constexpr (N > 1) {
    TileClass classes[N];
    for (int j = 0; j < count; ++j) classes[j] = tile_class(g[j], g[j].tile_n, g[j].splits);
    deal(classes, count, launch_pairs(ctx, l.total_tiles), &l.waves);
  }
  return run(l);
}

}  // namespace

af2_status layer_gemm_launch(af2_ctx *ctx, const LayerGemm *g, int count, cudaStream_t stream) {
  const int bn = g[0].tile_n, dtype = g[0].out_dtype;
  af2_status st;
  if (count > 1)
    st = describe_and_run<kMaxProducts>(ctx, g, count, [&](auto &l) {
      return dtype == AF2_F32 ? launch_bn<kProducts, float>(ctx, bn, l, stream)
                              : launch_16<kProducts>(ctx, dtype, bn, l, stream);
    });
  else
    st = describe_and_run<1>(ctx, g, 1, [&](auto &l) {
      if (g->epilogue == kEpilogueGateBackward)
        return dtype == AF2_F32 ? launch_bn<kGateBackward, float>(ctx, bn, l, stream)
                                : launch_16<kGateBackward>(ctx, dtype, bn, l, stream);
      if (g->epilogue == kEpilogueGate) {
        const bool save = l.product[0].args.save;
        return dtype == AF2_F32 ? (save ? launch_bn<kGateSave, float>(ctx, bn, l, stream)
                                        : launch_bn<kGate, float>(ctx, bn, l, stream))
               : save ? launch_16<kGateSave>(ctx, dtype, bn, l, stream)
                      : launch_16<kGate>(ctx, dtype, bn, l, stream);
      }
      const Args &p = l.product[0].args;
      auto out = [&](auto kind) {
        constexpr int KIND = decltype(kind)::value;
        return dtype == AF2_F32 ? launch_bn<KIND, float>(ctx, bn, l, stream) : launch_16<KIND>(ctx, dtype, bn, l, stream);
      };
      if (!p.tma_out || (p.residual && !p.tma_residual)) return out(std::integral_constant<int, kOutRows>());
      return p.save ? out(std::integral_constant<int, kOutSave>()) : out(std::integral_constant<int, kOut>());
    });
  return st;
}

af2_status layer_finish_launch(af2_ctx *ctx, int dtype, const LayerGemm *g, int count, const ColumnSums *sums,
                               int sum_count, cudaStream_t stream) {
  FinishLaunch l{};
  int64_t blocks = 0;
  for (int j = 0; j < count; ++j) {
    const LayerGemm &q = g[j];
    if (q.splits == 1) continue;
    ReduceArgs &r = l.product[l.products++];
    r.partial = reinterpret_cast<const float *>(q.scratch);
    r.splits = q.splits;
    r.batch = q.batch;
    r.activation = q.activation;
    r.m = q.m;
    r.n = q.n;
    r.pitch = align_up(q.n, 4);
    for (int i = 0; i < 2; ++i) {
      r.out[i] = q.out[i];
      r.bias[i] = q.bias[i];
    }
    r.out_stride = q.out_stride;
    r.residual = q.residual;
    r.residual_stride = q.residual_stride;
    r.saved_half = q.saved.half;
    r.saved_f32 = q.saved.f32;
    r.saved_pitch = q.saved.pitch;
    blocks = std::max(blocks, ceil_div(q.batch * q.m * r.pitch / 4, 256));
  }
  l.sum_count = sum_count;
  for (int j = 0; j < sum_count; ++j) {
    l.sums[j] = sums[j];
    blocks = std::max(blocks, ceil_div(sums[j].columns, 8));
  }
  if (blocks == 0) return AF2_OK;
  blocks = std::min<int64_t>(blocks, 8 * ctx->sm_count);
  LaunchScope scope(ctx, stream, kProfLayerElementwise);
  cudaError_t e = cudaSuccess;
  with_element(dtype, [&](auto *tag) {
    e = launch_early(finish_kernel<std::remove_pointer_t<decltype(tag)>>,
                     dim3(static_cast<unsigned>(blocks), l.products + sum_count), 256, 0, stream, l);
  });
  if (e != cudaSuccess) return cuda_fail(ctx, e, "layer sums");
  return AF2_OK;
}

}  // namespace af2
