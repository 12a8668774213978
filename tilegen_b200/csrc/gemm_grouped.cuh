// INT8 GEMM with one weight per expert over ragged groups of rows (sm_100a):
//
//   out[r,n] = ((float(sum_k xq[a(r),k] * wq[e,n,k]) * xscale[a(r)]) * wscale[e,n]) + bias[e,n]
//
// for the rows r in [offsets[e], offsets[e+1]) of each expert e, with
// a(r) = rows[r] (a gather of the activation rows) or r.  The arithmetic of
// each row is gemm_i8.cuh's, so a group's rows are bit-identical to
// tg_int8_gemm_dequant on that expert's weight.  The offsets stay on the
// device: the grid covers the most tiles the R rows can make (every expert may
// leave one tile part-filled) and CTAs without a tile return.
#pragma once

#include "common.cuh"
#include "gemv_i4.cuh"

namespace tg {

namespace grouped {
constexpr int THREADS = 256;
constexpr int BM = 64, BN = 64, BK = 64;
}  // namespace grouped

struct GroupedParams {
  const int8_t* xq;
  const float* xscale;
  const int8_t* wq;
  const float* wscale;
  const void* bias;
  const int32_t* rows;
  const int32_t* offsets;
  int bias_dtype;
  int wscale_mode;  // elements: 0 one, 1 one per expert, 2 one per expert and output channel
  int64_t M;        // rows of xq
  int R, E, N, K;
  void* out;        // [R, N] of OUT
};

template <int OUT>
__global__ void __launch_bounds__(grouped::THREADS) grouped_simple_kernel(const GroupedParams p) {
  using namespace grouped;
  __shared__ int32_t sx[BM][BK / 4 + 1];
  __shared__ int32_t sw[BN][BK / 4 + 1];
  __shared__ int32_t srow[BM];
  pdl_wait();
  int tile = blockIdx.y, e = 0, r0 = 0, r1 = 0;
  for (; e < p.E; ++e) {
    r0 = min(max(p.offsets[e], 0), p.R);
    r1 = min(max(p.offsets[e + 1], r0), p.R);
    const int tiles = (r1 - r0 + BM - 1) / BM;
    if (tile < tiles) break;
    tile -= tiles;
  }
  if (e == p.E) return;
  r0 += tile * BM;
  const int n0 = blockIdx.x * BN;
  for (int i = threadIdx.x; i < BM; i += THREADS) {
    int64_t a = -1;
    if (r0 + i < r1) a = p.rows ? p.rows[r0 + i] : r0 + i;
    srow[i] = a < p.M ? int32_t(a) : -1;
  }
  __syncthreads();
  int32_t acc[4][4] = {};
  const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  for (int k0 = 0; k0 < p.K; k0 += BK) {
    for (int i = threadIdx.x; i < BM * BK / 4; i += THREADS) {
      const int m = i / (BK / 4), k = k0 + i % (BK / 4) * 4;
      sx[m][i % (BK / 4)] = srow[m] >= 0 && k < p.K
                                ? *reinterpret_cast<const int32_t*>(p.xq + int64_t(srow[m]) * p.K + k) : 0;
      sw[m][i % (BK / 4)] = n0 + m < p.N && k < p.K
                                ? *reinterpret_cast<const int32_t*>(p.wq + (int64_t(e) * p.N + n0 + m) * p.K + k) : 0;
    }
    __syncthreads();
    for (int k = 0; k < BK / 4; ++k)
      for (int a = 0; a < 4; ++a)
        for (int b = 0; b < 4; ++b) acc[a][b] = __dp4a(sx[tm + 16 * a][k], sw[tn + 16 * b][k], acc[a][b]);
    __syncthreads();
  }
  for (int a = 0; a < 4; ++a) {
    const int r = r0 + tm + 16 * a;
    if (r >= r1) continue;
    const int src = srow[tm + 16 * a];
    const float xs = src >= 0 ? p.xscale[src] : 0.0f;
    for (int b = 0; b < 4; ++b) {
      const int n = n0 + tn + 16 * b;
      if (n >= p.N) continue;
      const size_t en = size_t(e) * p.N + n;
      const float ws = p.wscale[p.wscale_mode == 0 ? 0 : (p.wscale_mode == 1 ? size_t(e) : en)];
      float v = __fmul_rn(__fmul_rn(__int2float_rn(acc[a][b]), xs), ws);
      if (p.bias) v = __fadd_rn(v, load_as_f32(p.bias, p.bias_dtype, en));
      store_f32_as(p.out, OUT, size_t(r) * p.N + n, v);
    }
  }
}

}  // namespace tg
