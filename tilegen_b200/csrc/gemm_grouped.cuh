// INT8 GEMM with one weight per expert over ragged groups of rows (sm_100a):
//
//   out[r,n] = ((float(sum_k xq[a(r),k] * wq[e,n,k]) * xscale[a(r)]) * wscale[e,n]) + bias[e,n]
//
// for the rows r in [offsets[e], offsets[e+1]) of each expert e, with
// a(r) = rows[r] (a gather of the activation rows) or r.  The arithmetic of
// each row is gemm_i8.cuh's, so a group's rows are bit-identical to
// tg_int8_gemm_dequant on that expert's weight.
//
// Structure (persistent, one CTA per SM, 192 threads; roles as in gemm_i8.cuh):
//  * The operands swap roles, as in gemm_splitk.cuh: a 128-row tile of an
//    expert's WEIGHT is the UMMA M operand and up to TN of its activation rows
//    are UMMA N.  N is set per tile (a multiple of 16), so a group of three
//    rows costs a 16-column product and three rows' loads, not a 128-row
//    tile's, and nothing of a neighbouring group is ever computed.
//  * The offsets stay on the device: each CTA turns them into a prefix sum of
//    tiles per expert in shared memory, and its roles walk the tiles
//    blockIdx.x, blockIdx.x + gridDim.x, ... by it.  An expert's rows are cut
//    into equal token tiles, which run fastest, so tiles in flight share
//    their weight rows in L2; an expert without rows has no tile.
//  * Activation rows come by TMA, 16 rows a box, or with `rows` by
//    tile::gather4 (box one row high): each lane of the producer warp
//    holds the row numbers of its gathers and issues them.
//  * The epilogue holds one output channel per lane and stores column by
//    column (32 neighbouring channels of a row per warp and store).
// What bounds it: few rows per expert, the used experts' weight bytes (HBM);
// hundreds of rows, the int8 tensor rate.
#pragma once

#include "common.cuh"
#include "gemm_i8.cuh"
#include "gemv_i4.cuh"

namespace tg {

namespace grouped {
constexpr int THREADS = 192;
constexpr int BNW = 128;                 // weight rows per tile (UMMA M)
constexpr int BK = 128;                  // bytes of K per k-block
constexpr int UK = 32;                   // K per tcgen05.mma kind::i8
constexpr uint32_t W_BYTES = BNW * BK;   // 16 KB
constexpr int XBOX = 16;                 // activation rows per TMA box
constexpr int MAX_E = TG_MAX_EXPERTS;
__host__ __device__ constexpr uint32_t stage_bytes(int tn) { return W_BYTES + uint32_t(tn) * BK; }
__host__ __device__ constexpr int stages(int tn) {
  return int(208u * 1024u / stage_bytes(tn)) > 10 ? 10 : int(208u * 1024u / stage_bytes(tn));
}
__host__ __device__ constexpr uint32_t smem_bytes(int tn) { return uint32_t(stages(tn)) * stage_bytes(tn) + 1024; }
__host__ __device__ constexpr int tmem_cols(int tn) { return 2 * tn < 32 ? 32 : 2 * tn; }
}  // namespace grouped

struct GroupedParams {
  const float* xscale;
  const float* wscale;
  const void* bias;
  const int32_t* rows;
  const int32_t* offsets;
  int bias_dtype;
  int wscale_mode;  // elements: 0 one, 1 one per expert, 2 one per expert and output channel
  int M;            // rows of xq
  int R, E, N, K;
  int n_tiles, k_blocks;
  void* out;        // [R, N] of OUT
};

// cp.async.bulk.tensor tile::gather4: four rows (row numbers r0..r3) of one
// 128-byte column box to 512 bytes of shared memory.
__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int4 r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(r.x), "r"(r.y),
      "r"(r.z), "r"(r.w)
      : "memory");
}

// A named barrier that tells every thread whether all of them passed `ok`.
__device__ __forceinline__ bool named_barrier_and(int id, int nthreads, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %3, 0;\n\tbarrier.cta.red.and.pred q, %1, %2, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(nthreads), "r"(uint32_t(ok))
      : "memory");
  return r != 0;
}

// One tile: expert, its weight row, its output rows.
struct GroupedTile {
  int e, n0, r0, rows;  // rows <= TN
};

// The tiles of a CTA in order: a cursor over the prefix sums of tiles per expert.
template <int TN>
struct GroupedWalk {
  const int* cum;     // [E + 1] tiles before expert e
  const int* start;   // [E] first output row of expert e
  const int* count;   // [E] its rows
  int E, n_tiles, e;
  __device__ __forceinline__ GroupedWalk(const int* c, const int* s, const int* k, int E_, int nt)
      : cum(c), start(s), count(k), E(E_), n_tiles(nt), e(0) {}
  __device__ __forceinline__ GroupedTile at(int t) {
    while (e + 1 < E && t >= cum[e + 1]) ++e;
    const int local = t - cum[e];
    const int tok = (count[e] + TN - 1) / TN;       // token tiles of this expert
    const int per = ((count[e] + tok - 1) / tok + 15) & ~15;
    GroupedTile g;
    g.e = e;
    g.n0 = (local / tok) * grouped::BNW;
    const int j = (local % tok) * per;
    g.r0 = start[e] + j;
    g.rows = min(per, count[e] - j);
    return g;
  }
};

// TN: activation rows per tile at most (UMMA N); OUT: tg_dtype; GATHER: rows given.
template <int TN, int OUT, bool GATHER>
__global__ void __launch_bounds__(grouped::THREADS, 1)
    gemm_i8_grouped_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x,
                           const GroupedParams p) {
  using namespace grouped;
  constexpr int S = stages(TN);
  constexpr uint32_t STAGE = stage_bytes(TN);
  constexpr uint32_t TMEM_COLS = tmem_cols(TN);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);

  __shared__ __align__(8) uint64_t full_bar[S];
  __shared__ __align__(8) uint64_t empty_bar[S];
  __shared__ __align__(8) uint64_t tfull_bar[2];
  __shared__ __align__(8) uint64_t tempty_bar[2];
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_flag;
  __shared__ int issued;  // ring slots the producer filled
  __shared__ int cum[MAX_E + 1], start[MAX_E], count[MAX_E];
  __shared__ __align__(16) float col_xs[2][TN];

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tma_w);
    prefetch_tmap(&tma_x);
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], 4);
    }
    fence_mbar_init();
    abort_flag = 0;
    issued = 0;
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, TMEM_COLS);
    tmem_relinquish();
  }
  // The offsets, xq and xscale are the previous kernel's.
  pdl_wait();
  for (int e = threadIdx.x; e < p.E; e += THREADS) {
    const int a = min(max(p.offsets[e], 0), p.R);
    const int b = min(max(p.offsets[e + 1], a), p.R);
    start[e] = a;
    count[e] = b - a;
  }
  __syncthreads();
  if (warp == 0) {  // prefix sum of tiles, 32 experts at a time
    int sum = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      int v = e0 + lane < p.E ? (count[e0 + lane] + TN - 1) / TN * p.n_tiles : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (e0 + lane < p.E) cum[e0 + lane + 1] = sum + v;
      sum += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) cum[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;
  const int tiles = cum[p.E];
  GroupedWalk<TN> walk(cum, start, count, p.E, p.n_tiles);

  // Bounded wait that also gives up as soon as another role has given up.
  auto wait = [&](uint64_t* bar, uint32_t parity, unsigned int err) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    for (;;) {
      for (int i = 0; i < 32; ++i)
        if (mbar_try_wait(bar, parity)) return true;
      if (abort_flag) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        atomicOr(&g_device_status, err);
        abort_flag = 1;
        return false;
      }
    }
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int stage = 0, n_issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const GroupedTile g = walk.at(t);
      const int nt = (g.rows + 15) & ~15;
      // Lane l gathers rows 4 l .. 4 l + 3 of each 128; a row number outside
      // xq reads row 0 (its scale is taken as 0).
      constexpr int GL = (TN + 127) / 128;
      int4 idx[GL];
      if (GATHER) {
#pragma unroll
        for (int i = 0; i < GL; ++i) {
          int v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = i * 128 + lane * 4 + j;
            v[j] = r < g.rows ? p.rows[g.r0 + r] : 0;
            if (v[j] < 0 || v[j] >= p.M) v[j] = 0;
          }
          idx[i] = make_int4(v[0], v[1], v[2], v[3]);
        }
      }
      const int wrow = g.e * p.N + g.n0;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        ok = __all_sync(0xffffffffu, wait(&empty_bar[stage], phase ^ 1u, DEVERR_PIPE_TIMEOUT));
        if (!ok) break;
        uint8_t* sw = smem + stage * STAGE;
        uint8_t* sx = sw + W_BYTES;
        if (lane == 0) {
          mbar_arrive_expect_tx(&full_bar[stage], W_BYTES + uint32_t(nt) * BK);
          tma_load_2d(sw, &tma_w, &full_bar[stage], kb * BK, wrow);
        }
        __syncwarp();
        if (GATHER) {
#pragma unroll
          for (int i = 0; i < GL; ++i) {
            const int r = i * 128 + lane * 4;
            if (r < nt) tma_gather4(sx + r * BK, &tma_x, &full_bar[stage], kb * BK, idx[i]);
          }
        } else if (lane * XBOX < nt) {
          tma_load_2d(sx + lane * XBOX * BK, &tma_x, &full_bar[stage], kb * BK, g.r0 + lane * XBOX);
        }
        ++n_issued;
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (lane == 0) issued = n_issued;
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++local) {
        const GroupedTile g = walk.at(t);
        const uint32_t idesc = gemm::idesc(BNW, (g.rows + 15) & ~15);
        const int ab = local & 1;
        ok = wait(&tempty_bar[ab], (uint32_t(local >> 1) & 1u) ^ 1u, DEVERR_PIPE_TIMEOUT);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + uint32_t(ab * TN);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          ok = wait(&full_bar[stage], phase, DEVERR_TMA_TIMEOUT);
          if (!ok) break;
          tc_fence_after();
          const uint32_t w_addr = smem_u32(smem + stage * STAGE);
#pragma unroll
          for (int k = 0; k < BK / UK; ++k)
            mma_i8(d_tmem, gemm::kmajor_sw128_desc(w_addr + k * UK),
                   gemm::kmajor_sw128_desc(w_addr + W_BYTES + k * UK), idesc, (kb | k) != 0 ? 1u : 0u);
          mma_commit(&empty_bar[stage]);
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) mma_commit(&tfull_bar[ab]);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int et = threadIdx.x - 64;  // 0..127
    const int quarter = warp & 3;     // TMEM lanes [32*quarter, +32)
    int local = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++local) {
      const GroupedTile g = walk.at(t);
      const int ab = local & 1;
      const int n = g.n0 + quarter * 32 + lane;
      // This tile's row scales (two buffers: the warps may be a tile apart).
      for (int c = et; c < g.rows; c += 128) {
        int a = GATHER ? p.rows[g.r0 + c] : g.r0 + c;
        col_xs[ab][c] = a >= 0 && a < p.M ? p.xscale[a] : 0.0f;
      }
      float ws = 0.0f, bs = 0.0f;
      if (n < p.N) {
        const size_t en = size_t(g.e) * size_t(p.N) + size_t(n);
        ws = p.wscale[p.wscale_mode == 0 ? 0 : (p.wscale_mode == 1 ? size_t(g.e) : en)];
        if (p.bias) bs = load_as_f32(p.bias, p.bias_dtype, en);
      }
      const bool hb = p.bias != nullptr;
      // All four warps go on or none; the barrier also shows them the scales.
      if (!named_barrier_and(1, 128, wait(&tfull_bar[ab], uint32_t(local >> 1) & 1u, DEVERR_MMA_TIMEOUT))) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(ab * TN);
      const size_t esz = OUT == 0 ? 4 : 2;
      char* o = static_cast<char*>(p.out) + (size_t(g.r0) * size_t(p.N) + size_t(n)) * esz;
#pragma unroll 1
      for (int c0 = 0; c0 < g.rows; c0 += 16) {
        uint32_t acc[16];
        tmem_ld_32x32b_x16(t_row + uint32_t(c0), acc);
        tmem_wait_ld();
        reg_after_wait(acc);
        if (n < p.N) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (c0 + j < g.rows) {
              char* oj = o + size_t(c0 + j) * size_t(p.N) * esz;
              if (hb) store_dequant<OUT, true>(oj, int32_t(acc[j]), col_xs[ab][c0 + j], ws, bs);
              else store_dequant<OUT, false>(oj, int32_t(acc[j]), col_xs[ab][c0 + j], ws, bs);
            }
          }
        }
      }
      // This warp is done reading the accumulator: hand it back to the MMA.
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty_bar[ab]);
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // A wait gave up: let the loads still in flight (at most the last S slots)
  // land before the CTA exits.
  if (abort_flag && threadIdx.x == 0) {
    for (int i = max(0, issued - S); i < issued; ++i)
      mbar_wait(&full_bar[i % S], uint32_t(i / S) & 1u, DEVERR_TMA_TIMEOUT);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

}  // namespace tg
