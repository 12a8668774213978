// Few-row products with a 4-bit weight and group scales (sm_100a), for M <= 64
// activation rows:
//
//   out[m,n] = (sum_g wscale[n,g] * float(sum_{k in g} xq[m,k] * w4[n,k])) * xscale[m] + bias[n]
//
// xq are the quantiser's int8 codes, w4 signed 4-bit codes (-8..7), g runs over
// groups of 32, 64, 128 or 256 consecutive input channels.  The sum over a group
// (each half of a group of 256) is exact (int32); these sums are added in fp32.
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
// What bounds it: the weight's bytes.  A row tile of 16 weights is the products'
// M operand, straight from registers: each lane loads its 16 bytes of the rows
// lane/4 and lane/4 + 8 (no shared memory for the weight), DEPTH blocks ahead.
// The legacy mma.sync is enough here: at 64 rows the products are 20 % of its
// measured 1140 TOP/s at the weight's HBM rate, while tcgen05 would need the
// unpacked weight written to shared memory.  The activations are the N operand,
// 8 rows a product, from shared memory (row pitch = 32 mod 128 bytes, so a
// half-warp's 8-byte reads of four rows meet no bank twice).
//  * A CTA is WK warps over the same RT * 16 weight rows; warp w takes the blocks
//    w, w + WK, ...: neighbouring blocks are in flight together, and the
//    activations' next KC columns come in by cp.async while the present ones
//    are used.
//  * The int32 accumulators start at the bits of 1.5 * 2^23, so that the finished
//    sum v is the fp32 number 1.5 * 2^23 + v (|v| <= 2^21): one paired
//    subtraction and one paired fma per two outputs and group, no conversion.
//  * The warps' fp32 sums are added in order at the end.  WK follows from N
//    alone, so the order of all additions, and with it a row's bits, does not
//    depend on M.
#pragma once

#include "common.cuh"
#include "gemv_i8.cuh"

namespace tg {

namespace gemv4 {
// Activation columns per buffer (two buffers): PER steps of the WK warps' blocks.
__host__ __device__ constexpr int per(int mt, int wk) { return mt == 1 && wk == 4 ? 2 : 1; }
__host__ __device__ constexpr int kc(int mt, int wk) { return per(mt, wk) * wk * 128; }
__host__ __device__ constexpr int pitch(int mt, int wk) { return kc(mt, wk) + 32; }
// Shared memory for m activation rows (m <= 8 mt): the buffers, later the warps'
// partial tiles.
__host__ __device__ constexpr uint32_t smem_bytes(int m, int mt, int rt, int wk) {
  return uint32_t(2 * m * pitch(mt, wk)) > uint32_t(wk * rt * 16 * mt * 8 * 4)
             ? uint32_t(2 * m * pitch(mt, wk)) : uint32_t(wk * rt * 16 * mt * 8 * 4);
}
// CTAs per SM the registers are held to, and weight blocks a lane loads ahead.
__host__ __device__ constexpr int ctas(int mt, int wk) { return mt == 1 ? (wk == 4 ? 7 : 3) : (mt == 2 ? 2 : 1); }
__host__ __device__ constexpr int depth(int rt) { return rt == 1 ? 3 : 2; }
}  // namespace gemv4

struct GemvI4Params {
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
  int M, N, K;
  int prefetch;         // bytes of each weight row asked into L2 before the dependent wait
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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// d += a (16 x 32, rows) * b (32 x 8, columns), int8 -> int32.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One block's scales of a row: SV of them (one per 128 / SV codes), as loaded.
template <int SV, bool S4>
struct RawScale {
  uint32_t v[S4 ? SV : (SV + 1) / 2];
  __device__ __forceinline__ void load(const void* p) {
    constexpr int BYTES = SV * (S4 ? 4 : 2);
    if constexpr (BYTES == 2) {
      v[0] = __ldg(static_cast<const unsigned short*>(p));
    } else if constexpr (BYTES == 4) {
      v[0] = __ldg(static_cast<const uint32_t*>(p));
    } else if constexpr (BYTES == 8) {
      const uint2 a = __ldg(static_cast<const uint2*>(p));
      v[0] = a.x;
      v[1] = a.y;
    } else {
      const uint4 a = __ldg(static_cast<const uint4*>(p));
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

// MT: activation rows padded to 8 MT; RT: row tiles of 16 weights per CTA; WK: warps
// along K; SV: scales per block of 128 codes (groups of 32: 4, 64: 2, 128 and 256:
// 1); S4: fp32 scales.
template <int MT, int RT, int WK, int SV, bool S4>
__global__ void __launch_bounds__(WK * 32, gemv4::ctas(MT, WK)) gemv_i4_kernel(const GemvI4Params p) {
  using namespace gemv4;
  constexpr int THREADS = WK * 32;
  constexpr int KC = kc(MT, WK), PITCH = pitch(MT, WK), PER = per(MT, WK);
  constexpr int DEPTH = depth(RT);
  constexpr int ROWS = RT * 16, COLS = MT * 8;
  constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23
  extern __shared__ __align__(16) uint8_t smem4[];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * ROWS;
  const int blocks = p.K >> 7;
  const int steps = (blocks + WK - 1) / WK;
  const size_t row_bytes = size_t(p.K) >> 1;
  const uint32_t buf_bytes = uint32_t(p.M * PITCH);
  pdl_launch_dependents();
  if (p.prefetch > 0 && lane < 4) {
    const int r = warp * 4 + lane;
    if (r < ROWS && n0 + r < p.N) prefetch_l2_bulk(p.w4 + size_t(n0 + r) * row_bytes, uint32_t(p.prefetch));
  }
  pdl_wait();

  // Activation columns [c KC, c KC + KC) into buffer c & 1.
  auto fetch = [&](int c) {
    const int k0 = c * KC, width = min(KC, p.K - k0) >> 4;
    const uint32_t dst = smem_u32(smem4) + uint32_t(c & 1) * buf_bytes;
    for (int i = threadIdx.x; i < p.M * (KC / 16); i += THREADS) {
      const int m = i / (KC / 16), k = i % (KC / 16);
      if (k < width) cp_async16(dst + uint32_t(m * PITCH + k * 16), p.xq + size_t(m) * p.K + k0 + k * 16);
    }
    cp_async_commit();
  };

  // This lane's weight rows (clamped: the rows past N are computed and dropped).
  // As 32-bit offsets from the first row of the CTA (K is below 2^24).
  const uint8_t* const wbase = p.w4 + size_t(n0) * row_bytes;
  constexpr int SSZ = S4 ? 4 : 2;
  const char* const sbase = static_cast<const char*>(p.wscale) + size_t(n0) * size_t(p.groups) * SSZ;
  uint32_t wrow[RT][2], srow[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t n = uint32_t(min(r * 16 + h * 8 + g, p.N - 1 - n0));
      wrow[r][h] = n * uint32_t(row_bytes) + t * 16;
      srow[r][h] = n * uint32_t(p.groups * SSZ);
    }
  int4 wbuf[DEPTH][RT][2];
  RawScale<SV, S4> sbuf[DEPTH][RT][2];
  auto load = [&](int slot, int step) {
    const int b = min(step * WK + warp, blocks - 1);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        wbuf[slot][r][h] = ld_stream_v4(reinterpret_cast<const int4*>(wbase + (wrow[r][h] + uint32_t(b) * 64u)));
        sbuf[slot][r][h].load(sbase + (srow[r][h] + uint32_t(b >> p.scale_shift) * uint32_t(SV * SSZ)));
      }
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (d < steps) load(d, d);
  fetch(0);

  // Activation row of this lane in each 8-row tile (clamped: the columns past M
  // are computed and dropped).
  uint32_t xrow[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xrow[i] = uint32_t(min(i * 8 + g, p.M - 1) * PITCH + warp * 128 + t * 8);
  float2 acc[RT][MT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[r][i][0] = acc[r][i][1] = make_float2(0.0f, 0.0f);
  const bool f16 = p.wscale_dtype == TG_DT_F16;

  for (int s0 = 0; s0 < steps; s0 += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int s = s0 + d;
      if (s >= steps) break;
      if (s % PER == 0) {
        cp_async_wait_all();
        __syncthreads();  // this buffer is in, and nobody reads the other one any more
        if ((s / PER + 1) * KC < p.K) fetch(s / PER + 1);
      }
      if (s * WK + warp < blocks) {
        const uint8_t* xs = smem4 + ((s / PER) & 1) * buf_bytes + (s % PER) * (WK * 128);
        uint32_t lo[RT][2][4], hi[RT][2][4];
        float sc[RT][2][SV];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int4 w = wbuf[d][r][h];
            const uint32_t v[4] = {uint32_t(w.x), uint32_t(w.y), uint32_t(w.z), uint32_t(w.w)};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              lo[r][h][j] = (v[j] << 4) & 0xf0f0f0f0u;
              hi[r][h][j] = v[j] & 0xf0f0f0f0u;
            }
#pragma unroll
            for (int i = 0; i < SV; ++i) sc[r][h][i] = sbuf[d][r][h].get(i, f16);
          }
        if (s + DEPTH < steps) load(d, s + DEPTH);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint2 x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const uint2*>(xs + xrow[i] + j * 32);
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int q = 0; q < SV; ++q) {
              constexpr int MM = 4 / SV;  // products per scale
              int v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = __float_as_int(MAGIC);
#pragma unroll
              for (int j = q * MM; j < q * MM + MM; ++j)
                mma_s8(v, lo[r][0][j], lo[r][1][j], hi[r][0][j], hi[r][1][j], x[j].x, x[j].y);
              const float2 m2 = make_float2(MAGIC, MAGIC);
              acc[r][i][0] = fma2(sub2(make_float2(__int_as_float(v[0]), __int_as_float(v[1])), m2),
                                  make_float2(sc[r][0][q], sc[r][0][q]), acc[r][i][0]);
              acc[r][i][1] = fma2(sub2(make_float2(__int_as_float(v[2]), __int_as_float(v[3])), m2),
                                  make_float2(sc[r][1][q], sc[r][1][q]), acc[r][i][1]);
            }
        }
      }
    }
  }

  // The warps' partial tiles [warp][column][row] into shared memory, added in order.
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem4);
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* o = red + (warp * COLS + i * 8 + 2 * t) * ROWS + r * 16 + h * 8 + g;
        o[0] = acc[r][i][h].x;
        o[ROWS] = acc[r][i][h].y;
      }
  __syncthreads();
  for (int i = threadIdx.x; i < p.M * ROWS; i += THREADS) {
    const int m = i / ROWS, r = i % ROWS;
    const int n = n0 + r;
    if (n >= p.N) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < WK; ++w) v += red[(w * COLS + m) * ROWS + r];
    v = v * 0.0625f * p.xscale[m];
    if (p.bias) v += load_as_f32(p.bias, p.bias_dtype, size_t(n));
    store_f32_as(p.out, p.out_dtype, size_t(m) * p.N + n, v);
  }
}

}  // namespace tg
