// The two ends of a routed feed-forward layer (sm_100a): the router, which picks
// each token's experts and sorts the (token, expert) slots by expert, and the
// combine, which adds each token's expert rows back together.
//
// Router.  For token t, the top_k experts by logit (descending; equal logits by
// ascending index; NaN above everything, as torch's sort has it), and
//   weights[t,j] = exp(l_j - l_max) / sum exp(l - l_max)
// over the chosen experts (renormalize) or over all.  A slot whose logit is
// -inf is left out: weight 0, id and place -1; a token whose logits are all
// -inf (padding) takes no part at all.
// The slots (t, j) that are left, in order of (expert, t, j), are the rows of the
// grouped products: offsets[e] .. offsets[e+1] are expert e's, rows[r] is row
// r's token, place[t,j] slot (t, j)'s row; rows behind offsets[E] are -1.
#pragma once

#include "common.cuh"
#include "gemv_i4.cuh"

namespace tg {

namespace route {
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_E = TG_MAX_EXPERTS;
constexpr int MAX_K = TG_MAX_TOP_K;
}  // namespace route

struct RouteParams {
  const void* logits;  // [T, E]
  int dtype;
  int T, E, top_k, renormalize;
  int per_block;       // tokens per CTA
  int blocks;          // ceil(T / per_block)
  float* weights;      // [T, top_k]
  int32_t* ids;        // [T, top_k]
  int32_t* offsets;    // [E + 1]
  int32_t* rows;       // [T * top_k]
  int32_t* place;      // [T, top_k]
  int32_t* counts;     // [blocks, E]: slots of each expert in each CTA's tokens
};

// Order-preserving key of an fp32 logit; 0 is below every key.  -0 counts as
// +0; NaN is above +inf.
__device__ __forceinline__ uint32_t logit_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The chosen experts and weights of every token, and each CTA's counts.
// A warp per token; lane l holds the logits l, l + 32, ...
__global__ void __launch_bounds__(route::THREADS) route_topk_kernel(const RouteParams p) {
  using namespace route;
  __shared__ int32_t count[MAX_E];
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < p.E; e += THREADS) count[e] = 0;
  __syncthreads();
  pdl_wait();
  const int t0 = blockIdx.x * p.per_block;
  const int t1 = min(t0 + p.per_block, p.T);
  for (int t = t0 + warp; t < t1; t += WARPS) {
    uint32_t used = 0;  // bit i: logit lane + 32 i is taken
    float top = 0.0f, sum = 0.0f, mine = 0.0f;
    int id = -1;
    for (int j = 0; j < p.top_k; ++j) {
      uint32_t best = 0;
      int at = 0x7fffffff;
      for (int i = 0, e = lane; e < p.E; e += 32, ++i) {
        if (used >> i & 1u) continue;
        const uint32_t key = logit_key(load_as_f32(p.logits, p.dtype, size_t(t) * p.E + e));
        if (key > best) {
          best = key;
          at = e;
        }
      }
      const uint32_t win = __reduce_max_sync(0xffffffffu, best);
      const int e = __reduce_min_sync(0xffffffffu, best == win ? at : 0x7fffffff);
      if ((e & 31) == lane) used |= 1u << (e >> 5);
      const float v = load_as_f32(p.logits, p.dtype, size_t(t) * p.E + e);
      if (j == 0) top = v == -INFINITY ? 0.0f : v;
      const float w = expf(v - top);
      if (p.renormalize) sum += w;
      if (lane == j) {
        mine = w;
        id = v == -INFINITY ? -1 : e;
      }
      if (lane == 0 && v != -INFINITY) atomicAdd(&count[e], 1);
    }
    if (!p.renormalize) {
      for (int e = lane; e < p.E; e += 32) sum += expf(load_as_f32(p.logits, p.dtype, size_t(t) * p.E + e) - top);
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane < p.top_k) {
      p.ids[size_t(t) * p.top_k + lane] = id;
      p.weights[size_t(t) * p.top_k + lane] = id < 0 ? 0.0f : mine / sum;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += THREADS) p.counts[size_t(blockIdx.x) * p.E + e] = count[e];
}

// The slots' rows.  Each CTA adds up the counts of the CTAs before it (and all
// of them, for the offsets), then places its own slots in order.
__global__ void __launch_bounds__(route::THREADS) route_place_kernel(const RouteParams p) {
  using namespace route;
  __shared__ int32_t next[MAX_E];
  __shared__ int32_t total[MAX_E];
  pdl_wait();
  for (int e = threadIdx.x; e < p.E; e += THREADS) {
    int32_t before = 0, all = 0;
    for (int b = 0; b < p.blocks; ++b) {
      const int32_t c = p.counts[size_t(b) * p.E + e];
      if (b < int(blockIdx.x)) before += c;
      all += c;
    }
    next[e] = before;
    total[e] = all;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int32_t sum = 0;
    for (int e = 0; e < p.E; ++e) {
      next[e] += sum;
      if (blockIdx.x == 0) p.offsets[e] = sum;
      sum += total[e];
    }
    if (blockIdx.x == 0) p.offsets[p.E] = sum;
    total[0] = sum;
  }
  __syncthreads();
  const int slots = p.T * p.top_k;
  for (int r = total[0] + int(blockIdx.x * THREADS + threadIdx.x); r < slots; r += int(gridDim.x) * THREADS)
    p.rows[r] = -1;
  if (threadIdx.x == 0) {
    const int t0 = blockIdx.x * p.per_block;
    const int t1 = min(t0 + p.per_block, p.T);
    for (int s = t0 * p.top_k; s < t1 * p.top_k; ++s) {
      const int e = p.ids[s];
      const int r = e < 0 ? -1 : next[e]++;
      p.place[s] = r;
      if (r >= 0) p.rows[r] = s / p.top_k;
    }
  }
}

// out[t,:] = (residual[t,:] +) sum_j weights[t,j] * y[place[t,j],:], in fp32, j
// ascending, rounded once.  A place outside [0, R) adds nothing.
struct CombineParams {
  const void* y;          // [R, N] of DT
  const int32_t* place;   // [T, top_k]
  const float* weights;   // [T, top_k]
  const void* residual;   // [T, N] of DT or NULL
  void* out;              // [T, N] of DT
  int64_t R, T, N;
  int top_k;
};

template <int DT>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
  pdl_wait();
  const int64_t t = blockIdx.x;
  for (int64_t n = threadIdx.x; n < p.N; n += 256) {
    float acc = 0.0f;
    for (int j = 0; j < p.top_k; ++j) {
      const int64_t r = p.place[t * p.top_k + j];
      if (r < 0 || r >= p.R) continue;
      acc = fmaf(p.weights[t * p.top_k + j], load_as_f32(p.y, DT, size_t(r) * p.N + n), acc);
    }
    if (p.residual) acc += load_as_f32(p.residual, DT, size_t(t) * p.N + n);
    store_f32_as(p.out, DT, size_t(t) * p.N + n, acc);
  }
}

}  // namespace tg
