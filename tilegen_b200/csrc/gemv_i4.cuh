// Few-row products with a 4-bit weight and group scales (sm_100a), for M <= 64
// activation rows:
//
//   out[m,n] = (sum_g wscale[n,g] * float(sum_{k in g} xq[m,k] * w4[n,k])) * xscale[m] + bias[n]
//
// xq are the quantiser's int8 codes, w4 signed 4-bit codes (-8..7), g runs over
// groups of 32, 64, 128 or 256 consecutive input channels.  The sum over a group
// (each half of a group of 256) is exact (int32); these sums are added in fp32.
// (With one row: the sums over a group's 8, 16 or 32 codes in 16 bytes of weight.)
//
// Weight layout (K a multiple of 128; K/2 bytes a row): of each block of 128
// codes, byte 16 t + 4 j + b (t, j, b in 0..3) holds code 32 j + 8 t + b in its
// low half and code 32 j + 8 t + 4 + b in its high half, in two's complement.
// Chunk t of a block (16 bytes) is then what lane t of a quad needs of one row
// for the four m16n8k32 products of the block, word j for product j, and a word
// splits into the two int8x4 operands with three logical operations:
// (w << 4) & 0xf0f0f0f0 and w & 0xf0f0f0f0 are 16 times the codes (the sign bit
// of the 4-bit code lands on the byte's); the factor 16 goes into the epilogue.
//
// What bounds it: the weight's bytes, while the rows are few.  The weight comes
// through a ring of shared memory by TMA, which keeps tens of KB in flight per SM
// without a register, and is the products' M operand; the activations are the N
// operand, 8 rows a product.  Legacy mma.sync, because tcgen05 needs the unpacked
// weight written back to shared memory: at the weight's HBM rate 16 rows take 420 of
// its measured 1140 TOP/s, 44 rows all of them and 64 rows 1680, so that from there
// on the products are the floor (64 x 5120 x 15360: 8.8 us, the bytes 6.2).  33 rows
// pay for 64 columns, 17 for 32, 9 for 16.
//  * A CTA has WR * RT * 16 weight rows and all of K.  A step is one or two blocks
//    of 128 codes for each of the four warps along K, so the activations of a
//    step are read once per CTA.  The order of all additions depends on K alone: a
//    row's bits depend neither on M (from two rows up) nor on the other rows.
//  * Both come in boxes of 128 bytes a row with the 128-byte swizzle (narrower
//    rows, laid out for the reads, made the TMA unit the bound: it takes rows
//    at a fixed rate); a step's activations are one copy, by a
//    three-dimensional map.  A quad reads 64 bytes of a weight row and 32 of an
//    activation row; lane g's row is picked (w_row, x_row) so that the rows one
//    shared-memory pass reads lie in different banks.  Blocks past K and rows
//    past N arrive as zeros, so the loop has no edges.
//  * The rows' scales, one contiguous stretch, come by one bulk copy at the start.
//  * The int32 accumulators start at the bits of 1.5 * 2^23, so that the finished
//    sum v is the fp32 number 1.5 * 2^23 + v (|v| <= 2^21): one paired
//    subtraction and one paired fma per two outputs and group, no conversion.
//    With 64 columns and several groups a block the conversions, on another
//    pipe than the fmas, are the faster way (61 rows, groups of 32: 29 us, not 39).
//
// One activation row has a kernel of its own (gemv_i4_one_kernel): the matrix
// instructions would use an eighth of their columns, and the ring's start-up and
// steps are much of so short a launch.  Four weight rows per warp with plain
// 128-bit loads and dp4a, as gemv_i8_kernel.  Lane l takes the 16-byte chunks l,
// l + 32, ... of its part of K; a chunk holds 8 codes of each 32 of a block, so the
// CTA first lays the row out in shared memory as [half][chunk][16 bytes], two
// 128-bit reads a chunk that serve the four rows.  K x N, this form / the ring (us):
// 2048 x 1536 2.2 / 2.9, 5120 x 15360 8.3 / 9.4, 5120 x 5120 5.3 / 5.3, 13824 x 5120
// 8.6 / 11.5.  It is bound by the loads' latency: the launch is about one wave, and
// what it reads per us depends on the loads its resident warps have under way.
// Written for more rows it took, with two rows, 13.1 us on 5120 x 15360 and 11.8 on
// 13824 x 5120 (the ring 8.9 and 11.4), and with four 16.3 and 20.7 (the ring as
// with two).
#pragma once

#include "common.cuh"
#include "gemv_i8.cuh"

namespace tg {

namespace gemv4 {
constexpr int WK = 4;                 // warps along K
constexpr int MAX_STAGES = 16;
__host__ __device__ constexpr int threads(int wr) { return 32 * (WK * wr + 1); }
__host__ __device__ constexpr int rows(int rt, int wr) { return 16 * rt * wr; }
// Bytes of a ring slot's weights ([two blocks][row][128]) and activations
// ([block][row][128]) with kb blocks a warp, and of the scales of the CTA's rows.
__host__ __device__ constexpr uint32_t w_bytes(int kb, int rows) { return uint32_t(kb * rows) * WK * 64; }
__host__ __device__ constexpr uint32_t x_bytes(int kb, int m) { return (uint32_t(kb * m) * WK * 128 + 1023u) & ~1023u; }
__host__ __device__ constexpr uint32_t scale_bytes(int rows, int groups, bool s4) {
  return (uint32_t(rows) * uint32_t(groups) * (s4 ? 4u : 2u) + 15u) & ~15u;
}
// The weight row and the activation row, of eight, that lanes 4 g .. 4 g + 3 hold.
// Swizzled, byte chunk c of row r lies at c ^ r: a pass of eight lanes reads 64
// bytes of w_row 2i and 2i + 1, which differ in bit 2 (other halves of the 128
// bytes); a pass of sixteen reads 32 bytes of four x_rows, which differ in bits 1-2.
__device__ __forceinline__ int w_row(int g) { return (g >> 1) | ((g & 1) << 2); }
__device__ __forceinline__ int x_row(int g) { return ((g & 3) << 1) | (g >> 2); }
}  // namespace gemv4

struct GemvI4Params {
  const float* xscale;
  const void* wscale;   // [N, groups] of wscale_dtype
  const void* bias;
  int wscale_dtype;
  int bias_dtype;
  int out_dtype;
  int groups;           // K / group
  int scale_shift;      // groups of 256: 1 (two blocks share a scale), else 0
  int M, N, K;
  int stages;           // ring slots
  int prefetch;         // slots' weights asked into L2 before the dependent wait
  void* out;            // [M, N] of out_dtype
};

// Element i of a vector of a tg_dtype, as fp32.  Plain loads: the 16-bit __ldg
// is an asm statement that the compiler may move, and it was moved out of a loop
// past the `if (bias)` that guards it.
__device__ __forceinline__ float load_as_f32(const void* p, int dtype, size_t i) {
  if (dtype == TG_DT_F32) return static_cast<const float*>(p)[i];
  if (dtype == TG_DT_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// fp32 to element i of a vector of a tg_dtype, rounded to nearest even.
__device__ __forceinline__ void store_f32_as(void* out, int dtype, size_t i, float r) {
  if (dtype == TG_DT_F32) static_cast<float*>(out)[i] = r;
  else if (dtype == TG_DT_F16) static_cast<__half*>(out)[i] = __float2half_rn(r);
  else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(r);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// An untiled copy of `bytes` (a multiple of 16) to shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// One block's scales of a row: SV of them, as stored.
template <int SV, bool S4>
struct RawScale {
  uint32_t v[S4 ? SV : (SV + 1) / 2];
  __device__ __forceinline__ void load(const uint8_t* q) {  // from shared or global memory
    constexpr int BYTES = SV * (S4 ? 4 : 2);
    if constexpr (BYTES == 2) {
      v[0] = *reinterpret_cast<const unsigned short*>(q);
    } else if constexpr (BYTES == 4) {
      v[0] = *reinterpret_cast<const uint32_t*>(q);
    } else if constexpr (BYTES == 8) {
      const uint2 a = *reinterpret_cast<const uint2*>(q);
      v[0] = a.x;
      v[1] = a.y;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(q);
      v[0] = a.x;
      v[1] = a.y;
      v[2] = a.z;
      v[3] = a.w;
    }
  }
  __device__ __forceinline__ float get(int i, bool f16) const {
    if constexpr (S4) {
      return __uint_as_float(v[i]);
    } else {
      const uint32_t h = (i & 1) ? v[i / 2] >> 16 : v[i / 2] & 0xffffu;
      return f16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(h))) : __uint_as_float(h << 16);
    }
  }
};

// d = a (16 x 32, rows) * b (32 x 8, columns) + c, int8 -> int32.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b,
                                       const int (&c)[4]) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

// MT: activation rows padded to 8 MT; RT: row tiles of 16 weights per warp; WR:
// warps along N; KB: blocks of 128 codes a warp takes per step; SV: scales per block
// (groups of 32: 4, 64: 2, 128 and 256: 1); S4: fp32 scales.
template <int MT, int RT, int WR, int KB, int SV, bool S4>
__global__ void __launch_bounds__(gemv4::threads(WR), 1)
    gemv_i4_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x,
                   const GemvI4Params p) {
  using namespace gemv4;
  constexpr int THREADS = threads(WR);
  constexpr int ROWS = rows(RT, WR), COLS = MT * 8;
  constexpr int STEP = KB * WK;  // blocks per step
  constexpr uint32_t W_BYTES = w_bytes(KB, ROWS);
  constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23
  constexpr bool CONVERT = MT == 8 && SV >= 2;
  // Ring slots [weights | activations], then the scales; the partial tiles of the
  // end lie over the ring.
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem4 = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ __align__(8) uint64_t full_bar[MAX_STAGES];
  __shared__ __align__(8) uint64_t empty_bar[MAX_STAGES];
  __shared__ __align__(8) uint64_t scale_bar;
  __shared__ volatile int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * ROWS;
  const int blocks = p.K / 128;
  const int steps = (blocks + STEP - 1) / STEP;
  const uint32_t slot_bytes = W_BYTES + x_bytes(KB, p.M);
  // The scales of this CTA's rows are one stretch of wscale (16-byte aligned: n0 is
  // a multiple of 16); its last bytes may not fill 16.
  constexpr uint32_t SSZ = S4 ? 4 : 2;
  uint8_t* const scale = smem4 + uint32_t(p.stages) * slot_bytes;
  const uint8_t* const scale_src = static_cast<const uint8_t*>(p.wscale) + size_t(n0) * size_t(p.groups) * SSZ;
  const uint32_t scale_len = uint32_t(min(ROWS, p.N - n0)) * uint32_t(p.groups) * SSZ;
  const uint32_t scale_bulk = scale_len & ~15u;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    prefetch_tmap(&tma_w);
    prefetch_tmap(&tma_x);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], WK * WR);
    }
    mbar_init(&scale_bar, 1);
    fence_mbar_init();
    abort_flag = 0;
    // Only into L2: the kernel before may be the one that wrote the weight.
    for (int s = 0; s < (STEP / 2) * p.prefetch; ++s) tma_prefetch_l2_2d(&tma_w, s * 128, n0);
  }
  __syncthreads();
  pdl_wait();

  // Bounded wait that also gives up as soon as another warp has given up.
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

  float2 acc[RT][MT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[r][i][0] = acc[r][i][1] = make_float2(0.0f, 0.0f);
  const int kw = warp % WK, wr = warp / WK;   // of a computing warp
  const int g = lane >> 2, t = lane & 3;

  if (warp == WK * WR) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int slot = 0, filled = 0;
      uint32_t phase = 0;
      mbar_arrive_expect_tx(&scale_bar, scale_bulk);
      if (scale_bulk) bulk_load(scale, scale_src, scale_bulk, &scale_bar);
      for (int s = 0; s < steps; ++s) {
        if (!wait(&empty_bar[slot], phase ^ 1u, DEVERR_PIPE_TIMEOUT)) break;
        uint8_t* dst = smem4 + uint32_t(slot) * slot_bytes;
        mbar_arrive_expect_tx(&full_bar[slot], W_BYTES + uint32_t(p.M) * (STEP * 128));
#pragma unroll
        for (int b = 0; b < STEP / 2; ++b)
          tma_load_2d(dst + b * (ROWS * 128), &tma_w, &full_bar[slot], (s * (STEP / 2) + b) * 128, n0);
        tma_load_3d(dst + W_BYTES, &tma_x, &full_bar[slot], 0, 0, s * STEP);
        ++filled;
        if (++slot == p.stages) {
          slot = 0;
          phase ^= 1u;
        }
      }
      // The loads in flight land before the CTA can exit or reuse the ring (after
      // a wait gave up too: these waits do not heed the flag).
      ring_drain(full_bar, filled, p.stages, DEVERR_TMA_TIMEOUT);
      mbar_wait(&scale_bar, 0u, DEVERR_TMA_TIMEOUT);
    }
  } else {
    if (scale_bulk != scale_len) {  // (the same for all warps)
      if (threadIdx.x < 16 && scale_bulk + threadIdx.x < scale_len)
        scale[scale_bulk + threadIdx.x] = scale_src[scale_bulk + threadIdx.x];
      named_barrier(1, WK * WR * 32);
    }
    // ------------------------------------------------------------ products
    const uint32_t w_off = uint32_t(((kw >> 1) * ROWS + wr * RT * 16 + w_row(g)) * 128 +
                                    ((((kw & 1) * 4 + t) ^ w_row(g)) << 4));
    // (Rows from M up are whatever lies behind: their columns are dropped.)  A row's
    // swizzle follows from its place in the slot.
    uint32_t x_off[KB][4];
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const int xr = (k * WK + kw) * p.M + x_row(g);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x_off[k][j] = W_BYTES + uint32_t(xr * 128 + (((2 * j + (t >> 1)) ^ (xr & 7)) << 4) + (t & 1) * 8);
    }
    // (The rows past N read whatever lies behind the scales: they are dropped.)
    const uint32_t spitch = uint32_t(p.groups) * SSZ;
    const uint8_t* srow = scale + uint32_t(wr * RT * 16 + w_row(g)) * spitch;
    const bool f16 = p.wscale_dtype == TG_DT_F16;
    const int start = CONVERT ? 0 : __float_as_int(MAGIC);
    const int magic[4] = {start, start, start, start};
    auto sums = [](int a, int b) {  // two finished accumulators as fp32
      return CONVERT ? make_float2(__int2float_rn(a), __int2float_rn(b))
                     : sub2(make_float2(__int_as_float(a), __int_as_float(b)), make_float2(MAGIC, MAGIC));
    };
    int slot = 0;
    uint32_t phase = 0;
    const bool go = __all_sync(0xffffffffu, wait(&scale_bar, 0u, DEVERR_TMA_TIMEOUT));
    for (int s = 0; go && s < steps; ++s) {
      if (!__all_sync(0xffffffffu, wait(&full_bar[slot], phase, DEVERR_TMA_TIMEOUT))) break;
      const uint8_t* base = smem4 + uint32_t(slot) * slot_bytes;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const int b = s * STEP + k * WK + kw;
        if (b < blocks) {
          uint4 w[RT][2];
          float sc[RT][2][SV];
          const uint32_t si = uint32_t(b >> p.scale_shift) * (SV * SSZ);
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              w[r][h] = *reinterpret_cast<const uint4*>(base + w_off + (k * (WK / 2) * ROWS + r * 16 + h * 8) * 128);
              RawScale<SV, S4> raw;
              raw.load(srow + (r * 16 + h * 8) * spitch + si);
#pragma unroll
              for (int i = 0; i < SV; ++i) sc[r][h][i] = raw.get(i, f16);
            }
          uint32_t lo[RT][2][4], hi[RT][2][4];
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t v[4] = {w[r][h].x, w[r][h].y, w[r][h].z, w[r][h].w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                lo[r][h][j] = (v[j] << 4) & 0xf0f0f0f0u;
                hi[r][h][j] = v[j] & 0xf0f0f0f0u;
              }
            }
          // IB column tiles at a time, all their products first: a product's result
          // takes about 35 cycles, so neighbouring ones must not wait for each other.
          constexpr int IB = MT >= 2 && SV <= 2 ? 2 : 1;
          constexpr int MM = 4 / SV;  // products per scale
#pragma unroll
          for (int i0 = 0; i0 < MT; i0 += IB) {
            uint2 x[IB][4];
#pragma unroll
            for (int i = 0; i < IB; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                x[i][j] = *reinterpret_cast<const uint2*>(base + x_off[k][j] + (i0 + i) * 1024);
            int v[IB][RT][SV][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int i = 0; i < IB; ++i)
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                  int(&d)[4] = v[i][r][j / MM];
                  if (j % MM == 0) mma_s8(d, lo[r][0][j], lo[r][1][j], hi[r][0][j], hi[r][1][j], x[i][j], magic);
                  else mma_s8(d, lo[r][0][j], lo[r][1][j], hi[r][0][j], hi[r][1][j], x[i][j], d);
                }
#pragma unroll
            for (int q = 0; q < SV; ++q)
#pragma unroll
              for (int i = 0; i < IB; ++i)
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                  const int(&d)[4] = v[i][r][q];
                  float2(&o)[2] = acc[r][i0 + i];
                  o[0] = fma2(sums(d[0], d[1]), make_float2(sc[r][0][q], sc[r][0][q]), o[0]);
                  o[1] = fma2(sums(d[2], d[3]), make_float2(sc[r][1][q], sc[r][1][q]), o[1]);
                }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[slot]);
      if (++slot == p.stages) {
        slot = 0;
        phase ^= 1u;
      }
    }
  }

  // The warps' partial tiles [warp along K][column][row] over the ring, which
  // every load has landed in and every warp has left; added in order.
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem4);
  if (warp < WK * WR) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float* o = red + (kw * COLS + i * 8) * ROWS + (wr * RT + r) * 16 + h * 8 + w_row(g);
          o[x_row(2 * t) * ROWS] = acc[r][i][h].x;
          o[x_row(2 * t + 1) * ROWS] = acc[r][i][h].y;
        }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.M * ROWS; i += THREADS) {
    const int m = i / ROWS, r = i % ROWS;
    const int n = n0 + r;
    if (n >= p.N) continue;
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < WK; ++k) v += red[(k * COLS + m) * ROWS + r];
    v = v * 0.0625f * p.xscale[m];
    if (p.bias) v += load_as_f32(p.bias, p.bias_dtype, size_t(n));
    store_f32_as(p.out, p.out_dtype, size_t(m) * p.N + n, v);
  }
}

// One row on the CUDA cores (the header says why and what it measured).
namespace gemv4one {
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int R = 4;  // weight rows per warp
}  // namespace gemv4one

struct GemvI4OneParams {
  const int8_t* xq;
  const float* xscale;
  const uint8_t* w4;
  const void* wscale;   // [N, groups] of wscale_dtype
  const void* bias;
  int wscale_dtype;
  int bias_dtype;
  int out_dtype;
  int groups;           // K / group
  int scale_shift;      // groups of 256: 1 (two blocks share a scale), else 0
  int N, K;
  int kp;               // K parts per row group = warps per group (1, 2, 4 or 8)
  int part_chunks;      // 16-byte chunks of a row per part
  int prefetch;         // 1: prefetch a quarter of each warp's weight rows into L2 first
  void* out;            // [1, N] of out_dtype
};

// U: chunks of each row that a lane has under way; SV, S4 as in gemv_i4_kernel.
template <int U, int SV, bool S4>
__global__ void __launch_bounds__(gemv4one::THREADS, U == 1 ? 4 : 3) gemv_i4_one_kernel(const GemvI4OneParams p) {
  using namespace gemv4one;
  constexpr int SSZ = S4 ? 4 : 2;
  extern __shared__ __align__(16) uint8_t sx[];  // [2][chunks][16]
  __shared__ float partial[WARPS][R];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kp = p.kp;
  const int groups_per_cta = WARPS / kp;
  const int g_local = warp / kp, part = warp - g_local * kp;
  const uint32_t N = uint32_t(p.N);  // rows past the last one pass 2^31
  const uint32_t n0 = (blockIdx.x * uint32_t(groups_per_cta) + uint32_t(g_local)) * R;
  const int nch = p.K >> 5;
  const int c0 = part * p.part_chunks;
  const int c1 = min(c0 + p.part_chunks, nch);
  const bool live = n0 < N && c0 < c1;
  pdl_launch_dependents();
  if (live && p.prefetch && lane < R && n0 + lane < N)
    prefetch_l2_bulk(p.w4 + (size_t(n0 + lane) * size_t(nch) + size_t(c0)) * 16u, uint32_t(c1 - c0 + 3) / 4u * 16u);
  pdl_wait();

  // U chunks of the four rows and their scales (a row past N reads the last one's
  // and is dropped; a chunk past the part's end its last one's).
  const uint32_t first = min(n0, N - 1);
  const uint8_t* const wbase = p.w4 + size_t(first) * (size_t(nch) * 16u);
  const uint8_t* const sbase = static_cast<const uint8_t*>(p.wscale) + size_t(first) * (size_t(p.groups) * SSZ);
  uint32_t wrow[R], srow[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t n = min(uint32_t(r), N - 1 - first);
    wrow[r] = n * uint32_t(nch) * 16u;
    srow[r] = n * uint32_t(p.groups) * SSZ;
  }
  int4 w[U][R];
  RawScale<SV, S4> sc[U][R];
  auto load = [&](int c) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int cc = min(c + 32 * u, c1 - 1);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        w[u][r] = ld_stream_v4(reinterpret_cast<const int4*>(wbase + (wrow[r] + uint32_t(cc) * 16u)));
        sc[u][r].load(sbase + (srow[r] + uint32_t((cc >> 2) >> p.scale_shift) * uint32_t(SV * SSZ)));
      }
    }
  };
  if (live) load(c0 + lane);  // under way while the activations are laid out
  for (int q = threadIdx.x; q < p.K >> 4; q += THREADS) {  // 16 codes: two pieces
    const int4 v = *reinterpret_cast<const int4*>(p.xq + q * 16);
    const int j = (q >> 1) & 3, chunk = (q >> 3) * 4 + (q & 1) * 2;
    int2* d = reinterpret_cast<int2*>(sx + uint32_t((j >> 1) * nch + chunk) * 16u + (j & 1) * 8);
    d[0] = make_int2(v.x, v.y);
    d[2] = make_int2(v.z, v.w);  // the next chunk's
  }
  __syncthreads();

  float acc[R] = {};
  const bool f16 = p.wscale_dtype == TG_DT_F16;
  if (live) {
    for (int c = c0 + lane; c < c1; c += 32 * U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int cc = c + 32 * u;
        if (cc >= c1) break;
        const uint4 a = *reinterpret_cast<const uint4*>(sx + uint32_t(cc) * 16u);
        const uint4 b = *reinterpret_cast<const uint4*>(sx + uint32_t(nch + cc) * 16u);
        const uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint32_t v[4] = {uint32_t(w[u][r].x), uint32_t(w[u][r].y), uint32_t(w[u][r].z), uint32_t(w[u][r].w)};
#pragma unroll
          for (int q = 0; q < SV; ++q) {
            int sum = 0;
#pragma unroll
            for (int j = q * (4 / SV); j < (q + 1) * (4 / SV); ++j) {
              sum = __dp4a(int(v[j] & 0xf0f0f0f0u), int(x[2 * j + 1]), sum);
              sum = __dp4a(int((v[j] << 4) & 0xf0f0f0f0u), int(x[2 * j]), sum);
            }
            acc[r] = fmaf(__int2float_rn(sum), sc[u][r].get(q, f16), acc[r]);
          }
        }
      }
      if (c + 32 * U < c1) load(c + 32 * U);  // the other warps' products cover it
    }
  }

  // Sum over the warp's lanes, then over the K parts of each row group.
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float v = acc[r];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == r) partial[warp][r] = v;
  }
  __syncthreads();
  const int i = threadIdx.x;
  if (i < groups_per_cta * R) {
    const int g = i / R, r = i - g * R;
    const uint32_t n = (blockIdx.x * uint32_t(groups_per_cta) + uint32_t(g)) * R + uint32_t(r);
    if (n < N) {
      float v = 0.0f;
      for (int k = 0; k < kp; ++k) v += partial[g * kp + k][r];
      v = v * 0.0625f * p.xscale[0];
      if (p.bias) v += load_as_f32(p.bias, p.bias_dtype, size_t(n));
      store_f32_as(p.out, p.out_dtype, size_t(n), v);
    }
  }
}

}  // namespace tg
