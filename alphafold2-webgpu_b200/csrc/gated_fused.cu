// gated_fused.cu -- the gated transition in one kernel, for up to 128 channels:
// y = (act(x Wg + bg) (x Wv + bv)) Wo + bo (+ r), the hidden activations never
// leaving the chip.
//
// A CTA takes 128 rows at a time and the hidden channels in chunks of 64: the
// first product's N = 128 accumulator holds a chunk's gate and value side by
// side, sixteen warps (two groups of eight, chunks in turn) make h of it and
// write it to TMEM as the second product's A operand, and that product sums all
// chunks of the row tile in its own accumulator, drained by eight warps.  x is
// read once, y written once; the weights stream from L2 through two rings, a warp
// for each, read as they are stored (MN-major).
//
// What bounds it.  Per chunk and SM the tensor core takes 768 clocks (512 + 256)
// and the activations 8192 values: with one exponential and half a reciprocal each
// the multi-function unit takes 768 clocks too, beside it; neither is full (tensor
// 49 %, that unit 51 %, issue slots 59 % on 75776 rows), and what the gate warps wait
// for most is their accumulator.  (Every second pair's
// exponentials as a polynomial on the FMA pipe: 119 us where this takes 114, every
// fourth 115.  silu as z / 2 (1 + tanh(z / 2)), one instruction of that unit a value:
// 110, but tanh.approx's 2^-11 is up to 1 % of silu at z = -4 and 10 % at -6.)
// 262144 rows of 128 -> 512 -> 128 in bf16: 94 us in a burst, 62 of them at cuBLAS's
// rate for the products (98 to 114 repeated, as the power cap has it; f16 102).
#include <algorithm>
#include <type_traits>

#include "gated_fused.h"
#include "layer_math.cuh"

namespace af2 {
namespace {

constexpr int TILE = 128, HC = 64;             // rows of a tile, hidden channels of a chunk
constexpr int X_BUFS = 2, W1_STAGES = 5, W2_STAGES = 2, D1_BUFS = 2, H_BUFS = 4;
constexpr int MOST_HIDDEN = 2048;              // the gate's and the value's biases in shared memory
constexpr int GATE_WARPS = 16, OUT_WARPS = 8;  // warps 2-17 and 18-25
constexpr int SECOND_WARP = 2 + GATE_WARPS + OUT_WARPS;  // issues the second products
constexpr int W2_WARP = SECOND_WARP + 1;                // loads their weights
constexpr int THREADS = 32 * (W2_WARP + 1);
// TMEM columns: D1 2 x 128, D2 128, H 4 x 32 (64 16-bit values each)
constexpr uint32_t COL_D2 = D1_BUFS * 128, COL_H = COL_D2 + 128;

template <int KB>
struct Layout {
  static constexpr uint32_t X = KB * 16384u;   // [KB][128 rows][128 B]
  static constexpr uint32_t W1 = 16384u;       // a stage holds one of a chunk's KB parts: [gate, value][64 k][128 B]
  static constexpr uint32_t W2 = KB * 8192u;   // [KB][64 k][128 B]
  static constexpr uint32_t OFF_W1 = X_BUFS * X, OFF_W2 = OFF_W1 + W1_STAGES * W1;
  static constexpr uint32_t OUT = KB * 2048u;  // per out warp a 2 KB block for every 32 of its columns
  static constexpr uint32_t OFF_OUT = OFF_W2 + W2_STAGES * W2;
  static constexpr uint32_t OFF_BIAS = OFF_OUT + OUT_WARPS * OUT;  // the output bias in f32
  static constexpr uint32_t OFF_GATE_BIAS = OFF_BIAS + KB * 256u;  // gate and value biases in f32
  static constexpr uint32_t OFF_BAR = OFF_GATE_BIAS + 2 * 4 * MOST_HIDDEN;
  static constexpr uint32_t BYTES = OFF_BAR + 512 + 1024;
};

struct Maps {
  CUtensorMap x, gate, value, output, out, residual;
};
struct Args {
  const void *gate_bias, *value_bias, *output_bias;
  int64_t rows;
  int channels, hidden, chunks, tiles, activation, has_residual;
  unsigned int *err;
};

// The chunks of a CTA's tiles in order; a tile starts at chunk (tile mod chunks), so that the CTAs do
// not all read the same weights at once.
struct Cursor {
  int it = 0, step = 0, chunk;
  __device__ __forceinline__ explicit Cursor(int chunks) : chunk(static_cast<int>(blockIdx.x) % chunks) {}
  __device__ __forceinline__ void advance(int chunks) {
    if (++step == chunks) {
      step = 0;
      ++it;
      chunk = static_cast<int>(blockIdx.x + it * gridDim.x) % chunks;
    } else if (++chunk == chunks) {
      chunk = 0;
    }
  }
};

template <typename T, int KB, int ACT>
__global__ void __launch_bounds__(THREADS, 1) gated_fused_kernel(const __grid_constant__ Maps maps, const Args p) {
  using L = Layout<KB>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = align1024(smem_raw);
  const uint32_t sbase = smem_u32(smem), bar0 = sbase + L::OFF_BAR;
  auto x_full = [&](int b) { return bar0 + 8u * b; };
  auto x_empty = [&](int b) { return bar0 + 8u * (2 + b); };
  auto w1_full = [&](int s) { return bar0 + 8u * (4 + s); };
  auto w1_empty = [&](int s) { return bar0 + 8u * (9 + s); };
  auto w2_full = [&](int s) { return bar0 + 8u * (14 + s); };
  auto w2_empty = [&](int s) { return bar0 + 8u * (16 + s); };
  auto d1_full = [&](int b) { return bar0 + 8u * (18 + b); };
  auto d1_empty = [&](int b) { return bar0 + 8u * (20 + b); };
  auto h_full = [&](int b) { return bar0 + 8u * (22 + b); };
  auto h_empty = [&](int b) { return bar0 + 8u * (26 + b); };
  const uint32_t d2_full = bar0 + 8u * 30, d2_empty = bar0 + 8u * 31;
  auto load = [&](int w) { return bar0 + 8u * (32 + w); };  // an out warp's residual (8 of them)
  auto drain = [&](int i) { return bar0 + 8u * (40 + i); };
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::OFF_BAR + 480);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::OFF_BAR + 488);
  const int warp = warp_index_uniform(), lane = threadIdx.x & 31;
  const int my_tiles = (p.tiles - 1 - static_cast<int>(blockIdx.x)) / static_cast<int>(gridDim.x) + 1;
  const int total = my_tiles * p.chunks;  // chunks of this CTA

  if (threadIdx.x == 0) {
    for (int b = 0; b < X_BUFS; ++b) {
      mbar_init(x_full(b), 1);
      mbar_init(x_empty(b), 1);
    }
    for (int s = 0; s < W1_STAGES; ++s) {
      mbar_init(w1_full(s), 1);
      mbar_init(w1_empty(s), 1);
    }
    for (int s = 0; s < W2_STAGES; ++s) {
      mbar_init(w2_full(s), 1);
      mbar_init(w2_empty(s), 1);
    }
    for (int b = 0; b < D1_BUFS; ++b) {
      mbar_init(d1_full(b), 1);
      mbar_init(d1_empty(b), GATE_WARPS / 2);
    }
    for (int b = 0; b < H_BUFS; ++b) {
      mbar_init(h_full(b), GATE_WARPS / 2);
      mbar_init(h_empty(b), 1);
    }
    mbar_init(d2_full, 1);
    mbar_init(d2_empty, OUT_WARPS);
    mbar_init(drain(0), 1);
    mbar_init(drain(1), 1);
    for (int w = 0; w < OUT_WARPS; ++w) mbar_init(load(w), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  dependency_wait();
  float *const bias_out = reinterpret_cast<float *>(smem + L::OFF_BIAS);

  if (warp == 0) {
    // ---- loads of x and of the first products' weights, in their order ----
    if (lane == 0) {
      tma_prefetch_map(&maps.x);
      tma_prefetch_map(&maps.gate);
      tma_prefetch_map(&maps.value);
      int x_issued = 0, n = 0;
      auto issue_x = [&]() {
        const int b = x_issued % X_BUFS;
        if (!mbar_wait(x_empty(b), ((x_issued / X_BUFS) & 1) ^ 1, abort_flag, p.err, kErrWaitProducer)) return false;
        mbar_arrive_expect_tx(x_full(b), L::X);
        const int row0 = static_cast<int>(blockIdx.x + x_issued * gridDim.x) * TILE;
#pragma unroll
        for (int k = 0; k < KB; ++k) tma_load_3d(sbase + b * L::X + k * 16384, &maps.x, x_full(b), k * 64, row0, 0);
        ++x_issued;
        return true;
      };
      bool ok = issue_x();
      const int early = p.chunks > 1 ? 1 : 0;  // the next tile's x follows this step's weights
      Cursor c(p.chunks);
      for (int j = 0; ok && j < total; ++j) {
        for (int k = 0; k < KB; ++k, ++n) {
          const int s = n % W1_STAGES;
          ok = mbar_wait(w1_empty(s), ((n / W1_STAGES) & 1) ^ 1, abort_flag, p.err, kErrWaitProducer);
          if (!ok) break;
          mbar_arrive_expect_tx(w1_full(s), L::W1);
          const uint32_t dst = sbase + L::OFF_W1 + s * L::W1;
          tma_load_3d(dst, &maps.gate, w1_full(s), c.chunk * HC, k * 64, 0);
          tma_load_3d(dst + 8192, &maps.value, w1_full(s), c.chunk * HC, k * 64, 0);
        }
        if (ok && c.step == early && c.it + 1 < my_tiles) ok = issue_x();
        c.advance(p.chunks);
      }
      // every load issued has landed before the CTA exits
      for (int i = std::max(0, n - W1_STAGES); i < n; ++i)
        mbar_wait_drain(w1_full(i % W1_STAGES), (i / W1_STAGES) & 1, p.err);
      for (int i = std::max(0, x_issued - X_BUFS); i < x_issued; ++i)
        mbar_wait_drain(x_full(i % X_BUFS), (i / X_BUFS) & 1, p.err);
    }
  } else if (warp == W2_WARP) {
    // ---- loads of the second products' weights (in one thread with the others they came late) ----
    if (lane == 0) {
      tma_prefetch_map(&maps.output);
      int n = 0;
      Cursor c(p.chunks);
      for (; n < total; ++n, c.advance(p.chunks)) {
        const int s = n % W2_STAGES;
        if (!mbar_wait(w2_empty(s), ((n / W2_STAGES) & 1) ^ 1, abort_flag, p.err, kErrWaitProducer)) break;
        mbar_arrive_expect_tx(w2_full(s), L::W2);
#pragma unroll
        for (int k = 0; k < KB; ++k)
          tma_load_3d(sbase + L::OFF_W2 + s * L::W2 + k * 8192, &maps.output, w2_full(s), k * 64, c.chunk * HC, 0);
      }
      for (int i = std::max(0, n - W2_STAGES); i < n; ++i)
        mbar_wait_drain(w2_full(i % W2_STAGES), (i / W2_STAGES) & 1, p.err);
    }
  } else if (warp == 1) {
    // ---- first products: D1[j % 2] = x [Wg, Wv] of chunk j.  The second products have a warp of
    //      their own: with one warp for both, the tensor core ran dry while it waited for either ----
    constexpr uint32_t idesc = idesc_16_f32(TILE, 2 * HC, BF16, false, true);
    const uint64_t x_desc = sdesc_k_sw128(sbase);
    const uint64_t w_desc = sdesc_mn_sw128(sbase + L::OFF_W1, 8192, 1024);
    for (int j = 0, it = 0, step = 0, n = 0; j < total; ++j) {
      const int xb = it % X_BUFS, b = j % D1_BUFS;
      if ((step == 0 && !warp_wait(x_full(xb), (it / X_BUFS) & 1, abort_flag, p.err, kErrWaitMma)) ||
          !warp_wait(d1_empty(b), ((j / D1_BUFS) & 1) ^ 1, abort_flag, p.err, kErrWaitMma))
        break;
      const uint32_t d = tmem + b * 128;
      bool ok = true;
#pragma unroll
      for (int k = 0; k < KB; ++k, ++n) {
        const int s = n % W1_STAGES;
        ok = warp_wait(w1_full(s), (n / W1_STAGES) & 1, abort_flag, p.err, kErrWaitMma);
        if (!ok) break;
        tc_fence_after();
        const uint64_t xd = desc_add(x_desc, xb * L::X + k * 16384), wd = desc_add(w_desc, s * L::W1);
        if (k == 0)
          umma_first(d, xd, wd, idesc);
        else
          umma_acc(d, xd, wd, idesc);
#pragma unroll
        for (int ks = 1; ks < 4; ++ks) umma_acc(d, desc_add(xd, ks * 32), desc_add(wd, ks * 2048), idesc);
        umma_commit(w1_empty(s));
      }
      if (!ok) break;
      umma_commit(d1_full(b));
      if (step == p.chunks - 1) umma_commit(x_empty(xb));
      if (++step == p.chunks) {
        step = 0;
        ++it;
      }
    }
    // Every MMA has completed before TMEM is freed, whether or not a consumer gave up.
    umma_commit(drain(0));
    mbar_wait_drain(drain(0), 0, p.err);
  } else if (warp == SECOND_WARP) {
    // ---- second products: D2 += h Wo of chunk j ----
    constexpr uint32_t idesc = idesc_16_f32(TILE, KB * 64, BF16, false, true);
    const uint64_t w_desc = sdesc_mn_sw128(sbase + L::OFF_W2, 8192, 1024);
    const uint32_t d = tmem + COL_D2;
    for (int j = 0, it = 0, step = 0; j < total; ++j) {
      const int s = j % W2_STAGES, hb = j % H_BUFS;
      if ((step == 0 && !warp_wait(d2_empty, (it & 1) ^ 1, abort_flag, p.err, kErrWaitMma)) ||
          !warp_wait(w2_full(s), (j / W2_STAGES) & 1, abort_flag, p.err, kErrWaitMma) ||
          !warp_wait(h_full(hb), (j / H_BUFS) & 1, abort_flag, p.err, kErrWaitMma))
        break;
      tc_fence_after();
      const uint32_t h = tmem + COL_H + hb * 32;
      const uint64_t wd = desc_add(w_desc, s * L::W2);
      if (step == 0)
        umma_ts_first(d, h, wd, idesc);
      else
        umma_ts_acc(d, h, wd, idesc);
#pragma unroll
      for (int ks = 1; ks < HC / 16; ++ks) umma_ts_acc(d, h + ks * 8, desc_add(wd, ks * 2048), idesc);
      umma_commit(w2_empty(s));
      umma_commit(h_empty(hb));
      if (step == p.chunks - 1) umma_commit(d2_full);
      if (++step == p.chunks) {
        step = 0;
        ++it;
      }
    }
    umma_commit(drain(1));
    mbar_wait_drain(drain(1), 0, p.err);
  } else if (warp < 2 + GATE_WARPS) {
    // ---- h = act(g) v: group (warp - 2) / 8 takes every second chunk; a warp 32 rows and 32 of the
    //      chunk's 64 hidden channels ----
    const int group = (warp - 2) >> 3, q = warp & 3, half = ((warp - 2) >> 2) & 1;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const bool biased = p.gate_bias || p.value_bias;
    float *const gate_bias = reinterpret_cast<float *>(smem + L::OFF_GATE_BIAS);
    if (biased) {
      for (int i = threadIdx.x - 64; i < p.chunks * HC; i += 32 * GATE_WARPS) {
        gate_bias[i] = p.gate_bias && i < p.hidden ? to_f32<T>(static_cast<const T *>(p.gate_bias)[i]) : 0.f;
        gate_bias[MOST_HIDDEN + i] =
            p.value_bias && i < p.hidden ? to_f32<T>(static_cast<const T *>(p.value_bias)[i]) : 0.f;
      }
      named_barrier(2, 32 * GATE_WARPS);  // the gate warps only
    }
    Cursor c(p.chunks);
    for (int j = 0; j < total; ++j, c.advance(p.chunks)) {
      if ((j & 1) != group) continue;
      const int b = j % D1_BUFS, hb = j % H_BUFS, c0 = c.chunk * HC + half * 32;
      if (!warp_wait(d1_full(b), (j / D1_BUFS) & 1, abort_flag, p.err, kErrWaitEpilogue)) break;
      tc_fence_after();
      bool ok = true;
#pragma unroll
      for (int part = 0; part < 2; ++part) {  // 16 columns each
        uint32_t g[16], v[16], h[8];
        tmem_ld16(lanes + b * 128 + half * 32 + part * 16, g);
        tmem_ld16(lanes + b * 128 + HC + half * 32 + part * 16, v);
        tmem_ld_wait();
        if (part == 1) {  // the accumulator is in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(d1_empty(b));
        }
        const float4 *bg = reinterpret_cast<const float4 *>(gate_bias + c0 + part * 16);
        const float4 *bv = reinterpret_cast<const float4 *>(gate_bias + MOST_HIDDEN + c0 + part * 16);
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          float2 gz[2], vz[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int at = 4 * i4 + 2 * i;
            gz[i] = make_float2(__uint_as_float(g[at]), __uint_as_float(g[at + 1]));
            vz[i] = make_float2(__uint_as_float(v[at]), __uint_as_float(v[at + 1]));
          }
          if (biased) {
            const float4 g4 = bg[i4], v4 = bv[i4];
            gz[0] = f2add(gz[0], make_float2(g4.x, g4.y));
            gz[1] = f2add(gz[1], make_float2(g4.z, g4.w));
            vz[0] = f2add(vz[0], make_float2(v4.x, v4.y));
            vz[1] = f2add(vz[1], make_float2(v4.z, v4.w));
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 a = f2mul(activate2<ACT, true>(gz[i]), vz[i]);
            h[2 * i4 + i] = pack2_t<T>(a.x, a.y);
          }
        }
        if (part == 0) {
          // the second product is done with what this buffer held
          ok = warp_wait(h_empty(hb), ((j / H_BUFS) & 1) ^ 1, abort_flag, p.err, kErrWaitEpilogue);
          if (!ok) break;
          tc_fence_after();
        }
        tmem_st8(lanes + COL_H + hb * 32 + half * 16 + part * 8, h);
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(h_full(hb));
    }
  } else {
    // ---- y = D2 + bo (+ r): two warps per lane quarter, each half of the columns ----
    const int q = warp & 3, ow = warp - 2 - GATE_WARPS, col0 = (ow >> 2) * KB * 32;
    uint8_t *const block = smem + L::OFF_OUT + ow * L::OUT;
    const uint32_t block_addr = sbase + L::OFF_OUT + ow * L::OUT;
    const int blocks = max(0, min(KB, (p.channels - col0 + 31) / 32));
    for (int i = threadIdx.x - 32 * (2 + GATE_WARPS); i < KB * 64; i += 32 * OUT_WARPS)
      bias_out[i] =
          p.output_bias && i < p.channels ? to_f32<T>(static_cast<const T *>(p.output_bias)[i]) : 0.f;
    named_barrier(1, 32 * OUT_WARPS);  // the out warps only
    for (int it = 0, loads = 0; it < my_tiles; ++it) {
      const int r0 = static_cast<int>(blockIdx.x + it * gridDim.x) * TILE + q * 32;
      const bool rows_ok = r0 < p.rows, res = p.has_residual && rows_ok && blocks > 0;
      // the blocks are free once the last tile's results have left them; the residual's come ahead,
      // each into the block that its result leaves from
      if (lane == 0) {
        bulk_wait_read_all();
        if (res) {
          mbar_arrive_expect_tx(load(ow), blocks * 2048);
          for (int c = 0; c < blocks; ++c) tma_load_3d(block_addr + c * 2048, &maps.residual, load(ow), col0 + c * 32, r0, 0);
        }
      }
      __syncwarp();
      if (!warp_wait(d2_full, it & 1, abort_flag, p.err, kErrWaitEpilogue)) {
        if (res && lane == 0) mbar_wait_drain(load(ow), loads & 1, p.err);
        break;
      }
      tc_fence_after();
      if (res && !warp_wait(load(ow), loads & 1, abort_flag, p.err, kErrWaitEpilogue)) {
        if (lane == 0) mbar_wait_drain(load(ow), loads & 1, p.err);
        break;
      }
      loads += res;
      // the next tile's second products wait for this read: all blocks first, then the stores
      const uint32_t d2 = tmem + (static_cast<uint32_t>(q * 32) << 16) + COL_D2 + col0;
      uint32_t v[2][16];
      tmem_ld16(d2, v[0]);
#pragma unroll
      for (int h = 0; h < KB * 2; ++h) {  // 16 columns each
        tmem_ld_wait();
        if (h + 1 < KB * 2) {
          tmem_ld16(d2 + (h + 1) * 16, v[(h + 1) & 1]);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(d2_empty);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint4 *piece = reinterpret_cast<uint4 *>(block + (h >> 1) * 2048 + lane * 64 +
                                                   ((((h & 1) * 2 + k) ^ ((lane >> 1) & 3)) << 4));
          uint32_t w[4] = {};
          if (res) {
            const uint4 u = *piece;
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
          }
          const float2 *bias = reinterpret_cast<const float2 *>(bias_out + col0 + h * 16 + k * 8);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 y = f2add(make_float2(__uint_as_float(v[h & 1][8 * k + 2 * i]),
                                         __uint_as_float(v[h & 1][8 * k + 2 * i + 1])),
                             bias[i]);
            if (res) y = f2add(y, unpack2<T>(w[i]));
            w[i] = pack2_t<T>(y.x, y.y);
          }
          *piece = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0 && rows_ok) {
        for (int c = 0; c < blocks; ++c) tma_store_3d(&maps.out, block_addr + c * 2048, col0 + c * 32, r0, 0);
        bulk_commit();
      }
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

bool addressable(const void *ptr, int64_t stride) {
  return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && stride % 8 == 0 && stride < (int64_t(1) << 38);
}

template <typename T, int KB>
af2_status launch(af2_ctx *ctx, const Maps &maps, const Args &p, cudaStream_t stream) {
  constexpr uint32_t smem = Layout<KB>::BYTES;
  const dim3 grid(static_cast<unsigned>(std::min(p.tiles, ctx->sm_count)));
  LaunchScope scope(ctx, stream, kProfLayerGemm);
  cudaError_t e = cudaSuccess;
  with_activation(p.activation, [&](auto act) {
    auto kernel = gated_fused_kernel<T, KB, decltype(act)::value>;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = launch_early(kernel, grid, THREADS, smem, stream, maps, p);
  });
  if (e != cudaSuccess) return cuda_fail(ctx, e, "gated transition");
  return AF2_OK;
}

}  // namespace

bool gated_fused_fits(const GatedFused &f) { return f.dtype != AF2_F32 && f.channels <= 128 && f.hidden <= MOST_HIDDEN; }
bool gated_fused_covers(const GatedFused &f) {
  return gated_fused_fits(f) && addressable(f.out, f.out_stride) && (!f.residual || addressable(f.residual, f.residual_stride));
}

af2_status gated_fused_launch(af2_ctx *ctx, const GatedFused &f, cudaStream_t stream) {
  const bool bf16 = f.dtype == AF2_BF16;
  const CUtensorMapDataType t = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUtensorMapSwizzle wide = CU_TENSOR_MAP_SWIZZLE_128B, narrow = CU_TENSOR_MAP_SWIZZLE_64B;
  Maps maps{};
  auto map = [&](CUtensorMap *m, const void *ptr, int64_t width, int64_t rows, int64_t pitch, int box_rows, int box_cols,
                 CUtensorMapSwizzle swizzle) {
    return layer_map_3d(ctx, m, t, ptr, width, rows, 1, pitch * 2, pitch * 2, box_cols, box_rows, 1, swizzle);
  };
  bool ok = map(&maps.x, f.x.ptr, f.channels, f.rows, f.x.pitch, TILE, 64, wide) &&
            map(&maps.gate, f.gate.ptr, f.hidden, f.channels, f.gate.pitch, 64, 64, wide) &&
            map(&maps.value, f.value.ptr, f.hidden, f.channels, f.value.pitch, 64, 64, wide) &&
            map(&maps.output, f.output.ptr, f.channels, f.hidden, f.output.pitch, 64, 64, wide) &&
            map(&maps.out, f.out, f.channels, f.rows, f.out_stride, 32, 32, narrow);
  if (f.residual) ok = ok && map(&maps.residual, f.residual, f.channels, f.rows, f.residual_stride, 32, 32, narrow);
  if (!ok) return fail(ctx, AF2_ERR_CUDA, "cannot describe the transition's tensors to the TMA unit");
  Args p{};
  p.gate_bias = f.gate_bias;
  p.value_bias = f.value_bias;
  p.output_bias = f.output_bias;
  p.rows = f.rows;
  p.channels = static_cast<int>(f.channels);
  p.hidden = static_cast<int>(f.hidden);
  p.chunks = static_cast<int>((f.hidden + HC - 1) / HC);
  p.tiles = static_cast<int>((f.rows + TILE - 1) / TILE);
  p.activation = f.activation;
  p.has_residual = f.residual != nullptr;
  p.err = ctx->err_word;
  if (f.channels <= 64)
    return bf16 ? launch<__nv_bfloat16, 1>(ctx, maps, p, stream) : launch<__half, 1>(ctx, maps, p, stream);
  return bf16 ? launch<__nv_bfloat16, 2>(ctx, maps, p, stream) : launch<__half, 2>(ctx, maps, p, stream);
}

}  // namespace af2
