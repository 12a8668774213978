// INT8 GEMM with one weight per expert over ragged groups of rows (sm_100a):
//
//   out[r,n] = ((float(sum_k xq[a(r),k] * wq[e,n,k]) * xscale[a(r)]) * wscale[e,n]) + bias[e,n]
//
// for the rows r in [offsets[e], offsets[e+1]) of each expert e, with
// a(r) = rows[r] (a gather of the activation rows) or r.  The arithmetic of
// each row is gemm_i8.cuh's, so a group's rows are bit-identical to
// tg_int8_gemm_dequant on that expert's weight.
//
// Structure (persistent, one CTA per SM; roles as in gemm_i8.cuh: warp 0 TMA
// producer, warp 1 MMA issuer, warps 2-5 epilogue; with gathered rows warps 6-12
// are producers too):
//  * The operands swap roles, as in gemm_splitk.cuh: a 256-row tile of an
//    expert's WEIGHT is the UMMA M operand and up to TN of its activation rows
//    are UMMA N.  N is set per tile (a multiple of 32), so a group of three rows
//    costs a 32-column product and as many rows' loads, not a 128-row tile's.
//  * The two CTAs of a cluster share a tile by the pair MMA: each loads its
//    128 weight rows and half of the activation rows.
//  * The offsets stay on the device: each CTA turns them into a prefix sum of
//    tiles per expert in shared memory, and its roles walk the tiles unit,
//    unit + units, ... by it.  An expert's rows are cut into tiles of TN
//    and a rest (a tile's loads, 256 + N rows, bound it as much as its product,
//    so fewer tiles are cheaper than equal ones); these run fastest, so tiles in
//    flight share their weight rows in L2.  An expert without rows has no tile.
//  * Activation rows come by TMA, XBOX rows a box, or with `rows` by
//    tile::gather4 (box one row high).  One lane issuing a gather takes about 50
//    cycles, so seven warps share them.
//  * The epilogue holds one output channel per lane and a row per column: it
//    stages 32 rows x 32 channels a warp in shared memory for one TMA store, and
//    stores the part-filled last chunk of a group directly, row by row.
// What bounds it: few rows per expert, the used experts' weight bytes (HBM);
// hundreds of rows, the int8 tensor rate.
#pragma once

#include "common.cuh"
#include "gemm_i8.cuh"
#include "gemv_i4.cuh"

namespace tg {

namespace grouped {
constexpr int BNW = 128;                 // weight rows per CTA
constexpr int TILE_N = 2 * BNW;          // weight rows per pair (UMMA M)
constexpr int STEP = 32;                 // granularity of the pair MMA's N
constexpr int BK = 128;                  // bytes of K per k-block
constexpr int UK = 32;                   // K per tcgen05.mma kind::i8
constexpr uint32_t W_BYTES = BNW * BK;   // 16 KB
constexpr int GATHERERS = 7;             // warps that gather rows, beside warp 0 (the weights)
constexpr int STAGE_OUT = 4096;          // epilogue staging bytes per warp
constexpr int MAX_E = TG_MAX_EXPERTS;
__host__ __device__ constexpr int threads(bool gather) { return 192 + (gather ? 32 * GATHERERS : 0); }
constexpr int XBOX = 32;                 // activation rows per TMA box
// 128-byte K sub-blocks per ring slot (two, as gemm_i8.cuh's pairs), bytes of a
// sub-block's activation rows in each CTA (half of the tile's), of a slot, ring depth.
constexpr int KS = 2;
__host__ __device__ constexpr uint32_t x_bytes(int tn) { return uint32_t(tn / 2) * BK; }
__host__ __device__ constexpr uint32_t stage_bytes(int tn) { return uint32_t(KS) * (W_BYTES + x_bytes(tn)); }
__host__ __device__ constexpr int stages(int tn) { return int(198u * 1024u / stage_bytes(tn)); }
__host__ __device__ constexpr uint32_t smem_bytes(int tn) {
  return uint32_t(stages(tn)) * stage_bytes(tn) + 4u * STAGE_OUT + 1024u;
}
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

// cp.async.bulk.tensor tile::gather4: four rows (row numbers r) of one 128-byte
// column box to 512 bytes of shared memory; completion on the mbarrier at the
// shared::cluster address `mbar`, which may be the peer CTA's.
__device__ __forceinline__ void tma_gather4_pair(void* dst, const CUtensorMap* m, uint32_t mbar, int c0, int4 r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(mbar), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z),
      "r"(r.w)
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

// One tile: expert, its first weight row (of the CTA or pair), its output rows.
struct GroupedTile {
  int e, n0, r0, rows;  // rows <= TN
};

// The tiles of a unit in order: a cursor over the prefix sums of tiles per expert.
template <int TN>
struct GroupedWalk {
  const int* cum;     // [E + 1] tiles before expert e
  const int* start;   // [E] first output row of expert e
  const int* count;   // [E] its rows
  int E, e;
  __device__ __forceinline__ GroupedWalk(const int* c, const int* s, const int* k, int E_)
      : cum(c), start(s), count(k), E(E_), e(0) {}
  __device__ __forceinline__ GroupedTile at(int t) {
    while (e + 1 < E && t >= cum[e + 1]) ++e;
    const int local = t - cum[e];
    const int tok = (count[e] + TN - 1) / TN;       // token tiles of this expert
    GroupedTile g;
    g.e = e;
    g.n0 = (local / tok) * grouped::TILE_N;
    const int j = (local % tok) * TN;
    g.r0 = start[e] + j;
    g.rows = min(TN, count[e] - j);
    return g;
  }
};

// TN: activation rows per tile at most (UMMA N); OUT: tg_dtype; GATHER: rows given.
// Launched with clusters of 2 CTAs.
template <int TN, int OUT, bool GATHER>
__global__ void __launch_bounds__(grouped::threads(GATHER), 1)
    gemm_i8_grouped_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x,
                           const __grid_constant__ CUtensorMap tma_out, const GroupedParams p) {
  using namespace grouped;
  constexpr int S = stages(TN);
  constexpr uint32_t X_BYTES = x_bytes(TN);
  constexpr uint32_t STAGE = stage_bytes(TN);
  constexpr uint32_t TMEM_COLS = 2 * TN;
  constexpr int THREADS = threads(GATHER);
  constexpr int ESZ = OUT == 0 ? 4 : 2;
  constexpr int CHUNK = 32 * 32 * ESZ;      // a staged chunk: 32 rows x 32 channels
  constexpr int NBUF = STAGE_OUT / CHUNK;
  static_assert(TN % 32 == 0 && 2 * TN >= 32 && 2 * TN <= 512, "token tile");

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);

  __shared__ __align__(8) uint64_t full_bar[S];
  __shared__ __align__(8) uint64_t empty_bar[S];
  __shared__ __align__(8) uint64_t tfull_bar[2];
  __shared__ __align__(8) uint64_t tempty_bar[2];
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_flag;
  __shared__ int cum[MAX_E + 1], start[MAX_E], count[MAX_E];
  __shared__ __align__(16) float col_xs[2][TN];

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int unit = int(blockIdx.x >> 1);
  const int units = int(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    prefetch_tmap(&tma_w);
    prefetch_tmap(&tma_x);
    prefetch_tmap(&tma_out);
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], 8);
    }
    fence_mbar_init();
    abort_flag = 0;
  }
  if (warp == 1) {
    tmem_alloc_pair(&tmem_base_sh, TMEM_COLS);
    tmem_relinquish_pair();
  }
  // The kernel after this one may start its prologue on SMs that are done here.
  pdl_launch_dependents();
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
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;
  const int tiles = cum[p.E];
  GroupedWalk<TN> walk(cum, start, count, p.E);

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

  if (warp == 0 || warp >= 6) {
    // ------------------------------------------------------------ producers
    // Warp 0 loads the weight rows and announces the bytes; it also loads the
    // activation rows in boxes.  Gathered ones are the other warps', so that the
    // weights' loads never wait for row numbers.
    static_assert(int(X_BYTES) / BK / 4 <= 32 * GATHERERS, "one gather per lane");
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = unit; t < tiles && ok; t += units) {
      const GroupedTile g = walk.at(t);
      const int nt = (g.rows + STEP - 1) / STEP * STEP;
      const int mine = nt / 2;                        // activation rows this CTA loads
      const int first = int(rank) * mine;             // the first of them in the tile
      const int loaded = GATHER ? mine : (mine + XBOX - 1) / XBOX * XBOX;
      const uint32_t tx = 2u * uint32_t(KS) * (W_BYTES + uint32_t(loaded) * BK);
      // This lane's gather: rows 4 (warp - 6 + GATHERERS lane) + 0..3 of this CTA's.
      // A row number outside xq reads row 0 (its scale is taken as 0).
      const int gr = GATHER && warp != 0 ? 4 * (warp - 6 + GATHERERS * lane) : mine;
      int4 idx = make_int4(0, 0, 0, 0);
      if (gr < mine) {
        int v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = first + gr + j;
          v[j] = r < g.rows ? p.rows[g.r0 + r] : 0;
          if (v[j] < 0 || v[j] >= p.M) v[j] = 0;
        }
        idx = make_int4(v[0], v[1], v[2], v[3]);
      }
      const int wrow = g.e * p.N + g.n0 + int(rank) * BNW;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        ok = __all_sync(0xffffffffu, wait(&empty_bar[stage], phase ^ 1u, DEVERR_PIPE_TIMEOUT));
        if (!ok) break;
        uint8_t* sw = smem + stage * STAGE;
        uint8_t* sx = sw + KS * W_BYTES;
        // Both CTAs' copies land on the even CTA's barrier, which expects
        // the bytes of both.
        const uint32_t fb = mapa_shared(smem_u32(&full_bar[stage]), 0);
        if (warp == 0 && elect_one_lane()) {
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], tx);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const int kx = (kb * KS + ks) * BK;
            tma_load_2d_pair(sw + ks * W_BYTES, &tma_w, fb, kx, wrow);
            if (!GATHER) {
              for (int r = 0; r < loaded; r += XBOX)
                tma_load_2d_pair(sx + ks * X_BYTES + r * BK, &tma_x, fb, kx, g.r0 + first + r);
            }
          }
        }
        __syncwarp();
        if (gr < mine) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            tma_gather4_pair(sx + ks * X_BYTES + gr * BK, &tma_x, fb, (kb * KS + ks) * BK, idx);
        }
        __syncwarp();
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && leader) {
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = unit; t < tiles && ok; t += units, ++local) {
        const GroupedTile g = walk.at(t);
        const uint32_t idesc = gemm::idesc(TILE_N, (g.rows + STEP - 1) / STEP * STEP);
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
          const uint32_t x_addr = w_addr + KS * W_BYTES;
#pragma unroll
          for (int k = 0; k < KS * (BK / UK); ++k) {
            const int ks = k / (BK / UK), kk = k % (BK / UK);
            const uint64_t wd = gemm::kmajor_sw128_desc(w_addr + ks * W_BYTES + kk * UK);
            const uint64_t xd = gemm::kmajor_sw128_desc(x_addr + ks * X_BYTES + kk * UK);
            const uint32_t acc = (kb | k) != 0 ? 1u : 0u;
            mma_i8_pair(d_tmem, wd, xd, idesc, acc);
          }
          mma_commit_pair(&empty_bar[stage], 0x3);
          if (++stage == S) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) mma_commit_pair(&tfull_bar[ab], 0x3);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int et = threadIdx.x - 64;  // 0..127
    const int quarter = warp & 3;     // TMEM lanes [32*quarter, +32)
    uint8_t* const sbufs = smem + S * STAGE + (warp - 2) * STAGE_OUT;
    const uint32_t tempty0 = mapa_shared(smem_u32(&tempty_bar[0]), 0);
    const uint32_t tempty1 = mapa_shared(smem_u32(&tempty_bar[1]), 0);
    const bool hb = p.bias != nullptr;
    int local = 0, chunk_seq = 0;  // chunk_seq: chunks this warp has staged, one bulk group each
    for (int t = unit; t < tiles; t += units, ++local) {
      const GroupedTile g = walk.at(t);
      const int ab = local & 1;
      const int n_warp = g.n0 + int(rank) * BNW + quarter * 32;
      const int n = n_warp + lane;
      // This tile's row scales (two buffers: the warps may be a tile apart).
      for (int c = et; c < g.rows; c += 128) {
        const int a = GATHER ? p.rows[g.r0 + c] : g.r0 + c;
        col_xs[ab][c] = a >= 0 && a < p.M ? p.xscale[a] : 0.0f;
      }
      float ws = 0.0f, bs = 0.0f;
      if (n < p.N) {
        const size_t en = size_t(g.e) * size_t(p.N) + size_t(n);
        ws = p.wscale[p.wscale_mode == 0 ? 0 : (p.wscale_mode == 1 ? size_t(g.e) : en)];
        if (hb) bs = load_as_f32(p.bias, p.bias_dtype, en);
      }
      // All four warps go on or none; the barrier also shows them the scales.
      if (!named_barrier_and(1, 128, wait(&tfull_bar[ab], uint32_t(local >> 1) & 1u, DEVERR_MMA_TIMEOUT))) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(ab * TN);
#pragma unroll 1
      for (int c0 = 0; c0 < g.rows; c0 += 32) {
        uint32_t acc[32];
        tmem_ld_32x32b_x32(t_row + uint32_t(c0), acc);
        tmem_wait_ld();
        reg_after_wait(acc);
        if (c0 + 32 <= g.rows) {
          uint8_t* const sbuf = sbufs + (chunk_seq % NBUF) * CHUNK;
          ++chunk_seq;
          // The store that last used this buffer must have finished reading it.
          if (lane == 0) bulk_wait_read<NBUF - 1>();
          __syncwarp();
          char* o = reinterpret_cast<char*>(sbuf) + lane * ESZ;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (hb) store_dequant<OUT, true>(o + j * 32 * ESZ, int32_t(acc[j]), col_xs[ab][c0 + j], ws, bs);
            else store_dequant<OUT, false>(o + j * 32 * ESZ, int32_t(acc[j]), col_xs[ab][c0 + j], ws, bs);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (n_warp < p.N) tma_store_2d(&tma_out, sbuf, n_warp, g.r0 + c0);
            bulk_commit();
          }
        } else if (n < p.N) {
          char* o = static_cast<char*>(p.out) + (size_t(g.r0 + c0) * size_t(p.N) + size_t(n)) * ESZ;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (c0 + j < g.rows) {
              char* oj = o + size_t(j) * size_t(p.N) * ESZ;
              if (hb) store_dequant<OUT, true>(oj, int32_t(acc[j]), col_xs[ab][c0 + j], ws, bs);
              else store_dequant<OUT, false>(oj, int32_t(acc[j]), col_xs[ab][c0 + j], ws, bs);
            }
          }
        }
      }
      // This warp is done reading the accumulator: hand it back to the MMA.
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(ab ? tempty1 : tempty0);
    }
    if (lane == 0) bulk_wait<0>();
  }

  __syncwarp();
  // Every role is done; one that gave up has set the flag.  Loads (the odd CTA's land
  // on the even one's barriers, a gather's perhaps on one that warp 0 did not announce)
  // and products may then still be in flight.  A CTA whose roles all finished has
  // none: its epilogue saw every product of the pair.
  __syncthreads();
  if (abort_flag && threadIdx.x == 0) wait_out();
  __syncwarp();
  tc_fence_before();
  // Neither CTA of a pair may leave while the other can still touch its shared
  // memory or tensor memory.
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// The gather as a pass of its own, for groups large enough that the tensor cores
// are the bound: the TMA unit takes gathered rows at a quarter of the rate of
// whole boxes, and a tile's rows would be gathered again for every 256 output
// channels.  A warp copies a row (and its scale); a row number outside xq gives
// zeros.
struct GatherRowsParams {
  const int8_t* xq;      // [M, K]
  const float* xscale;   // [M]
  const int32_t* rows;   // [R]
  int8_t* q;             // [R, K] out
  float* scale;          // [R] out
  int M, R, K;
};

__global__ void __launch_bounds__(256) gather_rows_kernel(const GatherRowsParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= p.R) return;
  const int a = p.rows[r];
  const bool ok = a >= 0 && a < p.M;
  const int4* src = reinterpret_cast<const int4*>(p.xq + size_t(ok ? a : 0) * p.K);
  int4* dst = reinterpret_cast<int4*>(p.q + size_t(r) * p.K);
  if (lane == 0) p.scale[r] = ok ? p.xscale[a] : 0.0f;
#pragma unroll 4
  for (int i = lane; i < p.K / 16; i += 32) dst[i] = ok ? src[i] : make_int4(0, 0, 0, 0);
}

}  // namespace tg
