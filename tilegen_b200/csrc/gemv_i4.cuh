// Few-row products with a 4-bit weight and group scales (sm_100a), for M <= 64
// activation rows:
//
//   out[m,n] = (sum_g wscale[n,g] * float(sum_{k in g} xq[m,k] * w4[n,k])) * xscale[m] + bias[n]
//
// xq are the quantiser's int8 codes, w4 signed 4-bit codes (-8..7), g runs over
// groups of 32, 64, 128 or 256 consecutive input channels.  The sum inside a
// group is exact (int32); the groups are added in fp32.
//
// Weight layout (K a multiple of 128; K/2 bytes a row): of each block of 128
// codes, byte 16 t + 4 j + b (t, j, b in 0..3) holds code 32 j + 8 t + b in its
// low half and code 32 j + 8 t + 4 + b in its high half, in two's complement.
// A 16-byte chunk t is then four words, word j inside the j-th 32 codes, and
// each word splits into two int8x4 words of consecutive codes with three
// logical operations:  (w << 4) & 0xf0f0f0f0 and w & 0xf0f0f0f0 are 16 times
// the codes (the sign bit of the 4-bit code lands on the byte's), and the
// factor 16 goes into the epilogue's scale, exactly.
#pragma once

#include "common.cuh"

namespace tg {

namespace gemv4 {
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MB = 8;  // activation rows per pass
}  // namespace gemv4

struct GemvI4Params {
  const int8_t* xq;
  const float* xscale;
  const uint8_t* w4;
  const void* wscale;   // [N, K / group] of wscale_dtype
  const void* bias;
  int wscale_dtype;
  int bias_dtype;
  int group;
  int M, N, K;
  void* out;            // [M, N] of OUT
};

// Element i of a vector of a tg_dtype, as fp32.
__device__ __forceinline__ float load_as_f32(const void* p, int dtype, size_t i) {
  if (dtype == TG_DT_F32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == TG_DT_F16) return __half2float(__ldg(static_cast<const __half*>(p) + i));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
}

template <int OUT>
__device__ __forceinline__ void store_f32_as(void* out, size_t i, float r) {
  if (OUT == 0) static_cast<float*>(out)[i] = r;
  else if (OUT == 1) static_cast<__half*>(out)[i] = __float2half_rn(r);
  else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(r);
}

// One warp per weight row; its lanes take the row's 16-byte chunks in turn.
template <int OUT>
__global__ void __launch_bounds__(gemv4::THREADS) gemv_i4_kernel(const GemvI4Params p) {
  using namespace gemv4;
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * WARPS + (threadIdx.x >> 5);
  pdl_wait();
  if (n >= p.N) return;
  const int chunks = p.K / 32;
  const int groups = p.K / p.group;
  const int4* w = reinterpret_cast<const int4*>(p.w4) + size_t(n) * chunks;
  for (int m0 = 0; m0 < p.M; m0 += MB) {
    float acc[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[m] = 0.0f;
    for (int c = lane; c < chunks; c += 32) {
      const int4 v = __ldg(w + c);
      const uint32_t word[4] = {uint32_t(v.x), uint32_t(v.y), uint32_t(v.z), uint32_t(v.w)};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = (c >> 2) * 128 + j * 32 + (c & 3) * 8;
        const float ws = load_as_f32(p.wscale, p.wscale_dtype, size_t(n) * groups + k / p.group);
        const int lo = int((word[j] << 4) & 0xf0f0f0f0u), hi = int(word[j] & 0xf0f0f0f0u);
#pragma unroll
        for (int m = 0; m < MB; ++m) {
          if (m0 + m < p.M) {
            const int2 x = __ldg(reinterpret_cast<const int2*>(p.xq + size_t(m0 + m) * p.K + k));
            acc[m] = fmaf(float(__dp4a(lo, x.x, __dp4a(hi, x.y, 0))), ws, acc[m]);
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      for (int o = 16; o; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
      if (lane == 0 && m0 + m < p.M) {
        float r = acc[m] * 0.0625f * p.xscale[m0 + m];
        if (p.bias) r += load_as_f32(p.bias, p.bias_dtype, n);
        store_f32_as<OUT>(p.out, size_t(m0 + m) * p.N + n, r);
      }
    }
  }
}

}  // namespace tg
