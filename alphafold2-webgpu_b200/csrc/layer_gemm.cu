// layer_gemm.cu -- the product of the layers with learned weights on tcgen05:
// D = sum_s A_s B_s^T over 16-bit operands in either order each, f32 sums in
// TMEM, and the layers' epilogues.
//
// A cluster of two CTAs computes a 256 x BN tile with M = 256 MMAs
// (cta_group::2): CTA r holds rows 128 r .. of A's tile and half of B's rows,
// so each SM reads half of the B tile that it multiplies by.  Warp 0 of each
// CTA issues TMA loads, warp 1 of the even CTA the MMAs, warps 2-9 drain the
// accumulators (two warps per TMEM lane quarter, half of the columns each);
// two accumulators, so one tile's epilogue overlaps the next tile's MMAs.
// Operands are taken as they are stored: K-major rows as one 128-byte-swizzled
// block per K step of 64, MN-major ones as 64-wide blocks of 64 k each (the
// tensor core's transposed order), so no weight and no activation is ever
// transposed in memory.
//
// f32 tensors are multiplied as three bf16 terms each, x = x0 + x1 + x2, and
// the six products whose weight is at least 2^-16 of the largest are summed,
// the small ones first: what is left out is below 2^-24 of |x||y|, f32's own
// rounding.
#include <algorithm>
#include <type_traits>

#include "layer_gemm.h"
#include "layer_math.cuh"

namespace af2 {
namespace {

constexpr int BM = 128, PAIR_M = 256, BK = 64;
constexpr int EPI_WARPS = 8, THREADS = 64 + 32 * EPI_WARPS;
constexpr uint32_t A_BYTES = BM * 128;
constexpr int kPairs = 74;  // CTA pairs of a B200; only the choice of tiles and splits depends on it

// Stages of the operand ring and bytes of one epilogue warp's staging.
template <int EPI, int BN>
struct Shape {
  static constexpr uint32_t B_BYTES = (BN / 2) * 128;
  static constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = EPI == kEpilogueGateBackward ? 4 : BN == 256 ? 6 : 8;
  // Out, Gate: two 32 x 32 blocks of 16 bits (or one of 32); GateBackward: two slots of the four
  // planes' blocks (g and v: 2 KB of upper halves, 1 KB of lower bytes), the results written over them
  static constexpr uint32_t SLOT_BYTES = EPI == kEpilogueGateBackward ? 6144 : 2048;
  static constexpr uint32_t OFF_STAGE = STAGES * STAGE_BYTES;
  static constexpr uint32_t OFF_BAR = OFF_STAGE + EPI_WARPS * 2 * SLOT_BYTES;
  static constexpr uint32_t BYTES = OFF_BAR + 512 + 1024;
};

struct Maps {
  CUtensorMap a[2], b[2], out[2], hi, lo;
};

struct Args {
  void *out[2];
  int64_t out_stride;
  const void *bias[2];
  const void *residual;
  int64_t residual_stride;
  uint16_t *saved_hi;
  uint8_t *saved_lo;
  float *saved_f32;
  int64_t saved_pitch, saved_stride;
  float *column_partial;
  int64_t m;
  int n, k_blocks, splits, combos, segments, batch;
  int tiles_m, tiles_n, total_tiles;
  int a_mn, b_mn, bf16, activation;
  int tma_out;     // out rows are 16-byte aligned: whole blocks leave by TMA
  int vector_res;  // residual rows are 16-byte aligned
  int vector_bias;
  int partial;     // out[0] is [split][batch][m][n] of f32 sums (no bias, activation or residual)
  unsigned int *err;
};

// The terms (of A, of B) of the six products of an f32 operand pair, small ones first.
__constant__ const int8_t kTermA[6] = {2, 0, 1, 1, 0, 0};
__constant__ const int8_t kTermB[6] = {0, 2, 1, 0, 1, 0};

struct Tile {
  int split, z, mi, ni, kb0, kb1;
};
__device__ __forceinline__ Tile tile_at(const Args &p, int t) {
  Tile r;
  r.ni = t % p.tiles_n;
  t /= p.tiles_n;
  r.mi = t % p.tiles_m;
  t /= p.tiles_m;
  r.z = t % p.batch;
  r.split = t / p.batch;
  r.kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * r.split / p.splits);
  r.kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (r.split + 1) / p.splits);
  return r;
}

template <typename F>
__device__ __forceinline__ void activation_switch(int activation, F &&f) {
  switch (activation) {
    case AF2_ACTIVATION_RELU: f(std::integral_constant<int, AF2_ACTIVATION_RELU>()); break;
    case AF2_ACTIVATION_SIGMOID: f(std::integral_constant<int, AF2_ACTIVATION_SIGMOID>()); break;
    case AF2_ACTIVATION_SILU: f(std::integral_constant<int, AF2_ACTIVATION_SILU>()); break;
    case AF2_ACTIVATION_GELU: f(std::integral_constant<int, AF2_ACTIVATION_GELU>()); break;
    default: f(std::integral_constant<int, AF2_ACTIVATION_NONE>()); break;
  }
}

// x[i] += row[c0 + i] for the columns below `cols`; `vector`: row + c0 is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void add_row32(const T *row, int c0, int cols, bool vector, float (&x)[32]) {
  if (vector && c0 + 32 <= cols) {
    constexpr int PER = 16 / sizeof(T);
    const uint4 *p = reinterpret_cast<const uint4 *>(row + c0);
#pragma unroll
    for (int w = 0; w < 32 / PER; ++w) {
      const uint4 u = p[w];
      const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
      for (int i = 0; i < PER; ++i) x[w * PER + i] += to_f32<T>(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (c0 + i < cols) x[i] += to_f32<T>(row[c0 + i]);
  }
}

// The upper 16 bits of two f32 as one word (the first in its lower half), and the third bytes of four.
__device__ __forceinline__ uint32_t upper_halves(float a, float b) {
  return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
}
__device__ __forceinline__ uint32_t third_bytes(float a, float b, float c, float d) {
  return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0051),
                     __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0051), 0x5410);
}
// The f32 whose upper half is half `i` of `hi` and whose third byte is byte `j` of `lo`.
template <int I, int J>
__device__ __forceinline__ float from_planes(uint32_t hi, uint32_t lo) {
  // bytes (low to high): 0, lo[J], hi[2I], hi[2I + 1]; byte_perm sources 0-3 = hi, 4-7 = lo
  constexpr uint32_t sel = ((2 * I + 1) << 12) | ((2 * I) << 8) | ((4 + J) << 4);
  return __uint_as_float(__byte_perm(hi, lo, sel) & 0xffffff00u);
}

// One row (`lane`) of a 32 x 32 block of 16-bit values in a 64B-swizzled slot: its four 16-byte pieces.
__device__ __forceinline__ uint4 *slot_piece(uint8_t *slot, int lane, int c) {
  return reinterpret_cast<uint4 *>(slot + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
}
__device__ __forceinline__ void slot_write(uint8_t *slot, int lane, const uint32_t (&w)[16]) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *slot_piece(slot, lane, c) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
}

// An epilogue warp's ring of two 2 KB blocks on their way out.
struct StoreRing {
  uint8_t *ptr;
  uint32_t addr;
  int next = 0;

  // The next block, free for writing.
  __device__ __forceinline__ int take(int lane) {
    if (lane == 0) bulk_wait_read_but_one();
    __syncwarp();
    return next;
  }
  __device__ __forceinline__ void store16(const CUtensorMap *map, int lane, const uint32_t (&w)[16], int c0, int r0,
                                          int z, bool inside) {
    const int b = take(lane);
    slot_write(ptr + b * 2048, lane, w);
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (inside) tma_store_3d(map, addr + b * 2048, c0, r0, z);
      bulk_commit();
    }
    next ^= 1;
  }
  // A 32 x 32 block of f32 over both blocks (128B-swizzled rows).
  __device__ __forceinline__ void store32(const CUtensorMap *map, int lane, const float (&y)[32], int c0, int r0,
                                          int z, bool inside) {
    if (lane == 0) bulk_wait_read_all();
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *reinterpret_cast<float4 *>(ptr + sw128_offset(lane, c)) =
          make_float4(y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]);
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (inside) tma_store_3d(map, addr, c0, r0, z);
      bulk_commit();
    }
  }
};

// The planes of 32 saved pre-activations of one row: upper halves through the ring, third bytes directly.
__device__ __forceinline__ void save_planes(const Maps &maps, const Args &p, StoreRing &ring, int lane,
                                            const float (&z)[32], int c0, int r0, int plane, int64_t m, bool inside) {
  uint32_t hi[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) hi[i] = upper_halves(z[2 * i], z[2 * i + 1]);
  ring.store16(&maps.hi, lane, hi, c0, r0, plane, inside);
  if (inside && m < p.m) {
    uint4 *dst = reinterpret_cast<uint4 *>(p.saved_lo + plane * p.saved_stride + m * p.saved_pitch + c0);
    uint32_t lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = third_bytes(z[4 * i], z[4 * i + 1], z[4 * i + 2], z[4 * i + 3]);
    dst[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    dst[1] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
  }
}

template <typename T>
__device__ __forceinline__ void pack_row(const float (&y)[32], uint32_t (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack2_t<T>(y[2 * i], y[2 * i + 1]);
}

template <int EPI, typename OT, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    layer_gemm_kernel(const __grid_constant__ Maps maps, const Args p) {
  using S = Shape<EPI, BN>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = align1024(smem_raw);
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + S::OFF_BAR;
  // full: the leader's only (both CTAs' loads complete on it); empty, acc_full: both CTAs
  // (multicast commits); acc_empty: the leader's, one arrival per epilogue warp of the pair;
  // load: one per epilogue warp and slot, for the planes it reads
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
      mbar_init(acc_empty(b), 2 * EPI_WARPS);
    }
    mbar_init(drain, 1);
    if (EPI == kEpilogueGateBackward)
      for (int w = 0; w < EPI_WARPS; ++w)
        for (int b = 0; b < 2; ++b) mbar_init(load(w, b), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers exist before any arrival crosses the pair
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_map(&maps.a[0]);
      tma_prefetch_map(&maps.b[0]);
      int it = 0, s = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int t = pair; t < p.total_tiles && ok; t += npairs) {
        const Tile tile = tile_at(p, t);
        const int arow = tile.mi * PAIR_M + rank * BM;
        const int brow = EPI == kEpilogueGate ? tile.ni * (BN / 2) : tile.ni * BN + rank * (BN / 2);
        for (int c = 0; c < p.combos && ok; ++c) {
          const int ta = p.combos > 1 ? kTermA[c] : 0, tb = p.combos > 1 ? kTermB[c] : 0;
          for (int seg = 0; seg < p.segments && ok; ++seg) {
            const CUtensorMap *am = &maps.a[seg];
            const CUtensorMap *bm = &maps.b[EPI == kEpilogueGate ? rank : seg + tile.z];
            for (int kb = tile.kb0; kb < tile.kb1; ++kb, ++it) {
              // the stage is free in this CTA once the pair's MMAs have read it (multicast commit)
              if (!mbar_wait(empty(s), ph, abort_flag, p.err, kErrWaitProducer)) {
                ok = false;
                break;
              }
              const uint32_t dst = sbase + s * S::STAGE_BYTES;
              if (leader) mbar_arrive_expect_tx(full(s), 2 * S::STAGE_BYTES);
              if (p.a_mn) {
                tma_load_3d_pair(dst, am, full(s), arow, kb * BK, ta);
                tma_load_3d_pair(dst + 8192, am, full(s), arow + 64, kb * BK, ta);
              } else {
                tma_load_3d_pair(dst, am, full(s), kb * BK, arow, ta);
              }
              if (p.b_mn) {
#pragma unroll
                for (int j = 0; j < BN / 128; ++j)
                  tma_load_3d_pair(dst + A_BYTES + j * 8192, bm, full(s), brow + 64 * j, kb * BK, tb);
              } else {
                tma_load_3d_pair(dst + A_BYTES, bm, full(s), kb * BK, brow, tb);
              }
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
          mbar_wait_drain(full(j % STAGES), (j / STAGES) & 1, p.err);
    }
  } else if (warp == 1) {
    if (leader) {
      // the whole warp runs the issue loop (uniform waits, running descriptors); one elected lane issues
      const uint32_t idesc = idesc_16_f32(PAIR_M, BN, p.bf16, p.a_mn, p.b_mn);
      const uint64_t a_base = p.a_mn ? sdesc_mn_sw128(sbase, 8192, 1024) : sdesc_k_sw128(sbase);
      const uint64_t b_base =
          p.b_mn ? sdesc_mn_sw128(sbase + A_BYTES, 8192, 1024) : sdesc_k_sw128(sbase + A_BYTES);
      // bytes >> 4 from one K step of 16 to the next
      const uint32_t a_step = p.a_mn ? 2048 >> 4 : 32 >> 4, b_step = p.b_mn ? 2048 >> 4 : 32 >> 4;
      uint64_t ad = a_base, bd = b_base;
      int s = 0, buf = 0;
      uint32_t ph = 0, bph = 0;
      bool ok = true;
      for (int t = pair; t < p.total_tiles && ok; t += npairs) {
        const Tile tile = tile_at(p, t);
        const int iters = (tile.kb1 - tile.kb0) * p.segments * p.combos;
        if (!warp_wait(acc_empty(buf), bph ^ 1, abort_flag, p.err, kErrWaitMma)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * 256;
        for (int i = 0; i < iters; ++i) {
          if (!warp_wait(full(s), ph, abort_flag, p.err, kErrWaitMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < BK / 16; ++ks)
            umma_pair(d, ad + ks * a_step, bd + ks * b_step, idesc, (i | ks) != 0);
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
      // Every MMA has completed before TMEM is freed, whether or not a consumer gave up.
      umma_commit_pair(drain);
      mbar_wait_drain(drain, 0, p.err);
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2, ew = warp - 2;
    StoreRing ring{smem + S::OFF_STAGE + ew * 2 * S::SLOT_BYTES, sbase + S::OFF_STAGE + ew * 2 * S::SLOT_BYTES};
    int tile_it = 0, loads = 0;
    for (int t = pair; t < p.total_tiles; t += npairs, ++tile_it) {
      const Tile tile = tile_at(p, t);
      const int buf = tile_it & 1;
      const int r0 = tile.mi * PAIR_M + rank * BM + q * 32;  // the warp's first row
      const int64_t m = static_cast<int64_t>(r0) + lane;
      const bool rows_ok = r0 < p.m, row_ok = m < p.m;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + buf * 256;

      if constexpr (EPI == kEpilogueGateBackward) {
        // planes of the chunk that starts at column c0, into slot loads & 1
        auto fetch = [&](int c0, int slot) {
          if (lane == 0) {
            bulk_wait_read_all();  // the results of the chunk that used this slot have left it
            const uint32_t dst = ring.addr + slot * S::SLOT_BYTES, bar = load(ew, slot);
            mbar_arrive_expect_tx(bar, 6144);
            tma_load_3d(dst, &maps.hi, bar, c0, r0, 0);
            tma_load_3d(dst + 2048, &maps.hi, bar, c0, r0, 1);
            tma_load_3d(dst + 4096, &maps.lo, bar, c0, r0, 0);
            tma_load_3d(dst + 5120, &maps.lo, bar, c0, r0, 1);
          }
        };
        constexpr int CHUNKS = BN / 64;
        const int col0 = tile.ni * BN + half * (BN / 2);
        const int chunks = rows_ok ? min(CHUNKS, max(0, (p.n - col0 + 31) / 32)) : 0;
        if (chunks > 0) fetch(col0, loads & 1);
        if (!warp_wait(acc_full(buf), (tile_it >> 1) & 1, abort_flag, p.err, kErrWaitEpilogue)) {
          if (chunks > 0 && lane == 0) mbar_wait_drain(load(ew, loads & 1), (loads >> 1) & 1, p.err);
          break;
        }
        tc_fence_after();
        bool ok = true;
        for (int chunk = 0; chunk < chunks; ++chunk, ++loads) {
          const int slot = loads & 1, c0 = col0 + chunk * 32;
          if (chunk + 1 < chunks) fetch(c0 + 32, slot ^ 1);
          uint32_t v[32];
          tmem_ld32(taddr + half * (BN / 2) + chunk * 32, v);
          ok = warp_wait(load(ew, slot), (loads >> 1) & 1, abort_flag, p.err, kErrWaitEpilogue);
          tmem_ld_wait();
          if (!ok) {
            if (chunk + 1 < chunks && lane == 0) mbar_wait_drain(load(ew, slot ^ 1), ((loads + 1) >> 1) & 1, p.err);
            break;
          }
          uint8_t *sl = ring.ptr + slot * S::SLOT_BYTES;
          uint32_t dg[16], dv[16];
          activation_switch(p.activation, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
#pragma unroll
            for (int c = 0; c < 4; ++c) {  // 8 columns each
              const uint4 gh = *slot_piece(sl, lane, c), vh = *slot_piece(sl + 2048, lane, c);
              const uint2 gl = *reinterpret_cast<const uint2 *>(sl + 4096 + lane * 32 + c * 8);
              const uint2 vl = *reinterpret_cast<const uint2 *>(sl + 5120 + lane * 32 + c * 8);
              const uint32_t ghw[4] = {gh.x, gh.y, gh.z, gh.w}, vhw[4] = {vh.x, vh.y, vh.z, vh.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t glw = i < 2 ? gl.x : gl.y, vlw = i < 2 ? vl.x : vl.y;
                float g0, g1, v0, v1;
                if (i & 1) {
                  g0 = from_planes<0, 2>(ghw[i], glw), g1 = from_planes<1, 3>(ghw[i], glw);
                  v0 = from_planes<0, 2>(vhw[i], vlw), v1 = from_planes<1, 3>(vhw[i], vlw);
                } else {
                  g0 = from_planes<0, 0>(ghw[i], glw), g1 = from_planes<1, 1>(ghw[i], glw);
                  v0 = from_planes<0, 0>(vhw[i], vlw), v1 = from_planes<1, 1>(vhw[i], vlw);
                }
                float a0, s0, a1, s1;
                activate_slope<ACT>(g0, a0, s0);
                activate_slope<ACT>(g1, a1, s1);
                const float d0 = __uint_as_float(v[8 * c + 2 * i]), d1 = __uint_as_float(v[8 * c + 2 * i + 1]);
                dg[4 * c + i] = pack2_t<OT>(d0 * v0 * s0, d1 * v1 * s1);
                dv[4 * c + i] = pack2_t<OT>(d0 * a0, d1 * a1);
              }
            }
          });
          __syncwarp();
          slot_write(sl, lane, dg);
          slot_write(sl + 2048, lane, dv);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            const uint32_t src = ring.addr + slot * S::SLOT_BYTES;
            tma_store_3d(&maps.out[0], src, c0, r0, 0);
            tma_store_3d(&maps.out[1], src + 2048, c0, r0, 0);
            bulk_commit();
          }
          if (p.column_partial) {
            // the block's column sums: lane l takes columns 2 (l % 16), + 1 of rows l / 16, + 2, ...
            const int pc = lane & 15, par = lane >> 4;
#pragma unroll
            for (int plane = 0; plane < 2; ++plane) {
              float2 sum = make_float2(0.f, 0.f);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int row = 2 * i + par;
                const uint32_t w = *reinterpret_cast<const uint32_t *>(
                    sl + plane * 2048 + row * 64 + (((pc >> 2) ^ ((row >> 1) & 3)) << 4) + (pc & 3) * 4);
                sum = f2add(sum, unpack2<OT>(w));
              }
              sum.x += __shfl_xor_sync(kFull, sum.x, 16);
              sum.y += __shfl_xor_sync(kFull, sum.y, 16);
              if (par == 0)
                *reinterpret_cast<float2 *>(p.column_partial + (static_cast<int64_t>(r0 >> 5) * 2 + plane) *
                                                                   p.saved_pitch + c0 + 2 * pc) = sum;
            }
          }
        }
        if (!ok) break;
      } else {
        if (!warp_wait(acc_full(buf), (tile_it >> 1) & 1, abort_flag, p.err, kErrWaitEpilogue)) break;
        tc_fence_after();
        if constexpr (EPI == kEpilogueGate) {
#pragma unroll 1
          for (int chunk = 0; chunk < BN / 128; ++chunk) {
            const int cc = half * (BN / 4) + chunk * 32, c0 = tile.ni * (BN / 2) + cc;
            uint32_t gr[32], vr[32];
            tmem_ld32(taddr + cc, gr);
            tmem_ld32(taddr + BN / 2 + cc, vr);
            tmem_ld_wait();
            const bool inside = rows_ok && c0 < p.n;
            float(&g)[32] = reinterpret_cast<float(&)[32]>(gr);
            float(&v)[32] = reinterpret_cast<float(&)[32]>(vr);
            if (p.bias[0]) add_row32(static_cast<const OT *>(p.bias[0]), c0, p.n, p.vector_bias, g);
            if (p.bias[1]) add_row32(static_cast<const OT *>(p.bias[1]), c0, p.n, p.vector_bias, v);
            if (p.saved_hi) {
              save_planes(maps, p, ring, lane, g, c0, r0, 0, m, inside);
              save_planes(maps, p, ring, lane, v, c0, r0, 1, m, inside);
            }
            activation_switch(p.activation, [&](auto act) {
#pragma unroll
              for (int i = 0; i < 32; ++i) g[i] = activate<decltype(act)::value>(g[i]) * v[i];
            });
            uint32_t w[16];
            pack_row<OT>(g, w);
            ring.store16(&maps.out[0], lane, w, c0, r0, 0, inside);
          }
        } else {
          const int z = p.partial ? tile.split * p.batch + tile.z : 0;
          const CUtensorMap *omap = &maps.out[p.partial ? 0 : tile.z];
#pragma unroll 1
          for (int chunk = 0; chunk < BN / 64; ++chunk) {
            const int cc = half * (BN / 2) + chunk * 32, c0 = tile.ni * BN + cc;
            if (c0 >= p.n || !rows_ok) break;
            uint32_t r[32];
            tmem_ld32(taddr + cc, r);
            tmem_ld_wait();
            float(&y)[32] = reinterpret_cast<float(&)[32]>(r);
            if (!p.partial) {
              if (p.bias[tile.z]) add_row32(static_cast<const OT *>(p.bias[tile.z]), c0, p.n, p.vector_bias, y);
              if (p.saved_hi) save_planes(maps, p, ring, lane, y, c0, r0, 0, m, true);
              if (p.saved_f32 && row_ok) {
                float4 *dst = reinterpret_cast<float4 *>(p.saved_f32 + m * p.saved_pitch + c0);
#pragma unroll
                for (int i = 0; i < 8; ++i) dst[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
              }
              activation_switch(p.activation, [&](auto act) {
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = activate<decltype(act)::value>(y[i]);
              });
              if (p.residual && row_ok)
                add_row32(static_cast<const OT *>(p.residual) + m * p.residual_stride, c0, p.n, p.vector_res, y);
            }
            if (p.tma_out) {
              if constexpr (sizeof(OT) == 4) {
                ring.store32(omap, lane, y, c0, r0, z, true);
              } else {
                uint32_t w[16];
                pack_row<OT>(y, w);
                ring.store16(omap, lane, w, c0, r0, z, true);
              }
            } else if (row_ok) {
              OT *orow = static_cast<OT *>(p.out[tile.z]) + m * p.out_stride;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c0 + i < p.n) orow[c0 + i] = from_f32<OT>(y[i]);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(acc_empty(buf));
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

// out = act(sum of the splits' partial sums + bias) (+ residual), saved = the pre-activation.  One
// thread per four columns.
struct ReduceArgs {
  const float *partial;  // [split][batch][m][pitch]
  int splits, batch, activation;
  int64_t m, n, pitch;
  void *out[2];
  int64_t out_stride;
  const void *bias[2];
  const void *residual;
  int64_t residual_stride;
  uint16_t *saved_hi;
  uint8_t *saved_lo;
  float *saved_f32;
  int64_t saved_pitch;
};

template <typename OT>
__global__ void __launch_bounds__(256) reduce_kernel(const ReduceArgs p) {
  const int64_t quads = p.pitch / 4, total = p.batch * p.m * quads;
  const int64_t split_stride = p.batch * p.m * quads;  // float4s
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const float4 *src = reinterpret_cast<const float4 *>(p.partial) + i;
    float4 a = src[0];
    for (int s = 1; s < p.splits; ++s) {
      const float4 b = src[s * split_stride];
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    const int64_t row = i / quads, z = row / p.m, m = row - z * p.m, c0 = (i - row * quads) * 4;
    float y[4] = {a.x, a.y, a.z, a.w};
    const OT *bias = static_cast<const OT *>(p.bias[z]);
    OT *out = static_cast<OT *>(p.out[z]) + m * p.out_stride;
    const OT *res = p.residual ? static_cast<const OT *>(p.residual) + m * p.residual_stride : nullptr;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = c0 + j;
      if (c >= p.n) break;
      if (bias) y[j] += to_f32<OT>(bias[c]);
      if (p.saved_hi) {
        const uint32_t bits = __float_as_uint(y[j]);
        p.saved_hi[m * p.saved_pitch + c] = static_cast<uint16_t>(bits >> 16);
        p.saved_lo[m * p.saved_pitch + c] = static_cast<uint8_t>(bits >> 8);
      }
      if (p.saved_f32) p.saved_f32[m * p.saved_pitch + c] = y[j];
      activation_switch(p.activation, [&](auto act) { y[j] = activate<decltype(act)::value>(y[j]); });
      if (res) y[j] += to_f32<OT>(res[c]);
      out[c] = from_f32<OT>(y[j]);
    }
  }
}

// Tile width and number of splits of the depth, from what a launch costs in SM clocks: a K step of
// 64 takes 512 (BN = 256) or about 300 (BN = 128) clocks, a tile's start and its last epilogue about
// 2500, and split sums are written, read and reduced by another kernel.
struct Plan {
  int bn = 256, splits = 1;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

Plan make_plan(const LayerGemm &g) {
  Plan best;
  double best_cost = 0;
  const int64_t k_blocks = ceil_div(g.k, BK), combos = g.pieces > 1 ? 6 : 1;
  const bool gate = g.epilogue == kEpilogueGate, may_split = g.epilogue == kEpilogueOut;
  for (int bn : {256, 128}) {
    if (g.epilogue == kEpilogueGateBackward && bn == 128) continue;
    const int64_t tiles = g.batch * ceil_div(g.m, PAIR_M) * ceil_div(g.n, gate ? bn / 2 : bn);
    const int64_t max_splits = may_split ? std::min<int64_t>({ceil_div(k_blocks, 4), ceil_div(2 * kPairs, tiles), 64}) : 1;
    for (int64_t s = 1; s <= std::max<int64_t>(max_splits, 1); ++s) {
      const double waves = static_cast<double>(ceil_div(tiles * s, kPairs));
      const double steps = static_cast<double>(ceil_div(k_blocks, s) * g.segments * combos);
      double cost = waves * steps * (bn == 256 ? 512 : 300) + waves * 800 + 2500;
      if (s > 1) cost += 5000 + 8.0 * s * g.batch * g.m * align_up(g.n, 4) / 2500;
      if (best_cost == 0 || cost < best_cost) {
        best_cost = cost;
        best = {bn, static_cast<int>(s)};
      }
    }
  }
  return best;
}

bool aligned16(const void *ptr, int64_t stride, int element) {
  return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && (stride * element) % 16 == 0 &&
         stride * element < (int64_t(1) << 40);
}

bool operand_map(CUtensorMap *map, const GemmOperand &o, int64_t outer, int64_t k, bool bf16, int pieces,
                 int box_outer) {
  const CUtensorMapDataType t = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t row = o.pitch * 2, piece = pieces > 1 ? o.piece_stride * 2 : row;  // (one piece: no step)
  if (o.mn_major)
    return encode_map_3d(map, t, o.ptr, outer, k, pieces, row, piece, 64, BK, 1, CU_TENSOR_MAP_SWIZZLE_128B);
  return encode_map_3d(map, t, o.ptr, k, outer, pieces, row, piece, BK, box_outer, 1, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int EPI, typename OT, int BN>
af2_status launch(af2_ctx *ctx, const Maps &maps, const Args &p, cudaStream_t stream) {
  constexpr uint32_t smem = Shape<EPI, BN>::BYTES;
  auto kernel = layer_gemm_kernel<EPI, OT, BN>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      e != cudaSuccess)
    return cuda_fail(ctx, e, "layer product shared memory");
  const int pairs = std::min(p.total_tiles, std::max(1, ctx->sm_count / 2));
  LaunchScope scope(ctx, stream, kProfLayerGemm);
  kernel<<<2 * pairs, THREADS, smem, stream>>>(maps, p);
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return cuda_fail(ctx, e, "layer product");
  return AF2_OK;
}

template <typename OT>
af2_status launch_out(af2_ctx *ctx, int bn, const Maps &maps, const Args &p, cudaStream_t stream) {
  return bn == 256 ? launch<kEpilogueOut, OT, 256>(ctx, maps, p, stream)
                   : launch<kEpilogueOut, OT, 128>(ctx, maps, p, stream);
}
template <typename OT>
af2_status launch_gate(af2_ctx *ctx, int bn, const Maps &maps, const Args &p, cudaStream_t stream) {
  return bn == 256 ? launch<kEpilogueGate, OT, 256>(ctx, maps, p, stream)
                   : launch<kEpilogueGate, OT, 128>(ctx, maps, p, stream);
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == AF2_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : dtype == AF2_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                            : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

}  // namespace

uint64_t layer_gemm_scratch(const LayerGemm &g) {
  const Plan plan = make_plan(g);
  return plan.splits > 1 ? align_up(4ull * plan.splits * g.batch * g.m * align_up(g.n, 4), 256) : 0;
}

af2_status layer_gemm_launch(af2_ctx *ctx, const LayerGemm &g, cudaStream_t stream) {
  const Plan plan = make_plan(g);
  const bool gate = g.epilogue == kEpilogueGate;
  Maps maps{};
  Args p{};
  p.m = g.m;
  p.n = static_cast<int>(g.n);
  p.k_blocks = static_cast<int>(ceil_div(g.k, BK));
  p.splits = plan.splits;
  p.combos = g.pieces > 1 ? 6 : 1;
  p.segments = g.segments;
  p.batch = g.batch;
  p.tiles_m = static_cast<int>(ceil_div(g.m, PAIR_M));
  p.tiles_n = static_cast<int>(ceil_div(g.n, gate ? plan.bn / 2 : plan.bn));
  const int64_t total = static_cast<int64_t>(p.splits) * p.batch * p.tiles_m * p.tiles_n;
  if (total > 0x3fffffff) return fail(ctx, AF2_ERR_UNSUPPORTED, "the product has too many tiles");
  p.total_tiles = static_cast<int>(total);
  p.a_mn = g.a[0].mn_major;
  p.b_mn = g.b[0].mn_major;
  p.bf16 = g.bf16;
  p.err = ctx->err_word;
  const int bsets = gate ? 2 : std::max(g.segments, g.batch);
  bool maps_ok = true;
  for (int i = 0; i < g.segments; ++i)
    maps_ok &= operand_map(&maps.a[i], g.a[i], g.m, g.k, g.bf16, g.pieces, BM);
  for (int i = 0; i < bsets; ++i)
    maps_ok &= operand_map(&maps.b[i], g.b[i], g.n, g.k, g.bf16, g.pieces, plan.bn / 2);

  const int out_bytes = g.out_dtype == AF2_F32 ? 4 : 2;
  const int64_t pitch = align_up(g.n, 4);
  const int outs = g.epilogue == kEpilogueGateBackward ? 2 : g.batch;
  if (plan.splits > 1) {
    p.partial = 1;
    p.tma_out = 1;
    maps_ok &= encode_map_3d(&maps.out[0], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, g.scratch, g.n, g.m,
                             plan.splits * g.batch, pitch * 4, g.m * pitch * 4, 32, 32, 1,
                             CU_TENSOR_MAP_SWIZZLE_128B);
  } else {
    p.activation = g.activation;
    p.residual = g.residual;
    p.residual_stride = g.residual_stride;
    p.vector_res = aligned16(g.residual, g.residual_stride, out_bytes);
    p.out_stride = g.out_stride;
    p.vector_bias = 1;
    p.tma_out = 1;
    for (int i = 0; i < 2; ++i) {
      p.out[i] = g.out[i];
      p.bias[i] = g.bias[i];
      if (g.bias[i] && reinterpret_cast<uintptr_t>(g.bias[i]) % 16 != 0) p.vector_bias = 0;
      if (i < outs && !aligned16(g.out[i], g.out_stride, out_bytes)) p.tma_out = 0;
    }
    if (p.tma_out)
      for (int i = 0; i < outs; ++i)
        maps_ok &= encode_map_3d(&maps.out[i], map_type(g.out_dtype), g.out[i], g.n, g.m, 1, g.out_stride * out_bytes,
                                 g.out_stride * out_bytes, 32, 32, 1,
                                 out_bytes == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
    p.saved_f32 = g.saved.f32;
    p.saved_hi = g.saved.hi;
    p.saved_lo = g.saved.lo;
    p.saved_pitch = g.saved.pitch;
    p.saved_stride = g.saved.stride;
    if (g.saved.hi) {
      const int planes = g.epilogue == kEpilogueOut ? 1 : 2;
      maps_ok &= encode_map_3d(&maps.hi, CU_TENSOR_MAP_DATA_TYPE_UINT16, g.saved.hi, g.saved.pitch, g.m, planes,
                               g.saved.pitch * 2, g.saved.stride * 2, 32, 32, 1, CU_TENSOR_MAP_SWIZZLE_64B);
      if (g.epilogue == kEpilogueGateBackward)
        maps_ok &= encode_map_3d(&maps.lo, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.saved.lo, g.saved.pitch, g.m, planes,
                                 g.saved.pitch, g.saved.stride, 32, 32, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
    }
    p.column_partial = g.column_partial;
  }
  if (!maps_ok) return fail(ctx, AF2_ERR_CUDA, "cannot describe the layer's tensors to the TMA unit");

  af2_status st = AF2_OK;
  if (g.epilogue == kEpilogueGateBackward)
    st = g.out_dtype == AF2_F16 ? launch<kEpilogueGateBackward, __half, 256>(ctx, maps, p, stream)
                                : launch<kEpilogueGateBackward, __nv_bfloat16, 256>(ctx, maps, p, stream);
  else if (gate)
    st = g.out_dtype == AF2_F16 ? launch_gate<__half>(ctx, plan.bn, maps, p, stream)
                                : launch_gate<__nv_bfloat16>(ctx, plan.bn, maps, p, stream);
  else if (p.partial || g.out_dtype == AF2_F32)
    st = launch_out<float>(ctx, plan.bn, maps, p, stream);
  else
    st = g.out_dtype == AF2_F16 ? launch_out<__half>(ctx, plan.bn, maps, p, stream)
                                : launch_out<__nv_bfloat16>(ctx, plan.bn, maps, p, stream);
  if (st != AF2_OK || plan.splits == 1) return st;

  ReduceArgs r{};
  r.partial = reinterpret_cast<const float *>(g.scratch);
  r.splits = plan.splits;
  r.batch = g.batch;
  r.activation = g.activation;
  r.m = g.m;
  r.n = g.n;
  r.pitch = pitch;
  for (int i = 0; i < 2; ++i) {
    r.out[i] = g.out[i];
    r.bias[i] = g.bias[i];
  }
  r.out_stride = g.out_stride;
  r.residual = g.residual;
  r.residual_stride = g.residual_stride;
  r.saved_hi = g.saved.hi;
  r.saved_lo = g.saved.lo;
  r.saved_f32 = g.saved.f32;
  r.saved_pitch = g.saved.pitch;
  const int blocks = static_cast<int>(std::min<int64_t>(ceil_div(g.batch * g.m * pitch / 4, 256), 8 * ctx->sm_count));
  LaunchScope scope(ctx, stream, kProfLayerElementwise);
  with_element(g.out_dtype, [&](auto *tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    reduce_kernel<T><<<blocks, 256, 0, stream>>>(r);
  });
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return cuda_fail(ctx, e, "layer split sums");
  return AF2_OK;
}

}  // namespace af2
