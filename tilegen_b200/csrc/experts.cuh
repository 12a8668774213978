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
//
// A warp takes a token: lane l holds the logits l, l + 32, ... as order-preserving
// 32-bit keys, and each of the top_k rounds is a maximum over the lane's keys
// and two warp reductions (the key, then the lowest index that has it).  A token
// has an expert at most once, so a CTA's slots of one expert are a bit mask over
// its tokens: a slot's rank among them is a population count of the bits
// before it, and no atomic's order decides anything.  Up to SINGLE tokens one CTA
// does everything; above, a first kernel writes the choices and each CTA's
// counts, a second one adds up the counts of the CTAs before it and places the
// slots.  Measured (us, top 8 of 64 / 256 / 1024 experts): one CTA, 1 token 2.9 / 4.0
// / 9.2, 32 tokens 4.0 / 7.4 / 20.5, 64 6.3 / 12.2 / 34.8, 256 20.2 / 40.7 / 117; two
// kernels, 257 tokens 5.9 / 9.3 / 23.3: the one CTA is the faster up to about 32 to 60
// tokens, and one launch up to SINGLE.  The launches and a few dependent memory
// latencies bound the two kernels, one SM's issue rate the one CTA.  Neither of
// the two lets the kernel after it start early: CTAs that wait on SMs which are
// done first leave the later ones unevenly placed (4096 tokens: 12.9 us, not 9.2).
#pragma once

#include <type_traits>

#include "common.cuh"
#include "gemv_i4.cuh"

namespace tg {

namespace route {
constexpr int THREADS = 1024;                 // of the placing kernel
// Of the choosing kernel: sixteen or more keys a lane leave 512 threads' registers.
__host__ __device__ constexpr int threads(int epl) { return epl >= 16 ? 512 : 1024; }
constexpr int MAX_E = TG_MAX_EXPERTS;
constexpr int MAX_K = TG_MAX_TOP_K;
constexpr int ROW_THREADS = 256;              // of the thread-per-token chooser,
constexpr int ROW_MAX_E = 128;                // its most experts
constexpr int ROW_MAX_K = 8;                  // and choices
constexpr int ROW_MIN_T = 16384;              // and fewest tokens (512 warps)
constexpr int SINGLE = 256;                   // most tokens of the one-CTA form
constexpr int MAX_WORDS = 8;                  // mask words of an expert in shared memory
constexpr int PASS = 32 * MAX_WORDS;          // tokens whose masks are held at once
constexpr int SLOTS = PASS * MAX_K / THREADS;  // their slots per thread at most
}  // namespace route

struct RouteParams {
  const void* logits;  // [T, E]
  int dtype;
  int T, E, top_k, renormalize;
  int per_block;       // tokens per CTA, a multiple of 32
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
// The logit of a key (of NaN, a NaN).
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// v[i] = element from + step i of the logits for the i with first + step i < end: all
// loads in flight at once (the branch on the type is outside of them).
template <int N>
__device__ __forceinline__ void load_logits(const RouteParams& p, size_t from, int step, int first, int end,
                                            float (&v)[N]) {
  auto load = [&](auto dt) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = first + step * i < end ? load_as_f32(p.logits, decltype(dt)::value, from + size_t(step) * i) : 0.0f;
  };
  if (p.dtype == TG_DT_F32) load(std::integral_constant<int, TG_DT_F32>());
  else if (p.dtype == TG_DT_F16) load(std::integral_constant<int, TG_DT_F16>());
  else load(std::integral_constant<int, TG_DT_BF16>());
}

// Token t's logits as keys: lane l's i-th is expert l + 32 i (0 past E).
template <int EPL>
__device__ __forceinline__ void route_load(const RouteParams& p, int t, int lane, uint32_t (&key)[EPL]) {
  float v[EPL];
  load_logits<EPL>(p, size_t(t) * p.E + lane, 32, lane, p.E, v);
#pragma unroll
  for (int i = 0; i < EPL; ++i) key[i] = lane + 32 * i < p.E ? logit_key(v[i]) : 0u;
}

// The token's choices: lane j < top_k gets slot j's expert (-1: left out) and weight.
template <int EPL>
__device__ __forceinline__ void route_token(const RouteParams& p, int lane, uint32_t (&key)[EPL], int& id,
                                            float& weight) {
  id = -1;
  uint32_t mine = 0;  // slot `lane`'s key
  float all = 0.0f;   // sum over all experts, relative to the first choice
  float top = 0.0f;
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) best = max(best, key[i]);
    const uint32_t win = __reduce_max_sync(0xffffffffu, best);
    int at = 0x7fffffff;
#pragma unroll
    for (int i = EPL - 1; i >= 0; --i) at = key[i] == win ? lane + 32 * i : at;
    const int e = EPL == 1 ? __ffs(__ballot_sync(0xffffffffu, key[0] == win)) - 1
                           : int(__reduce_min_sync(0xffffffffu, at));
    if (j == 0) {
      const float v = key_logit(win);
      top = v == -INFINITY ? 0.0f : v;
      if (!p.renormalize) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) s += key[i] != 0u ? expf(key_logit(key[i]) - top) : 0.0f;
        all = warp_sum(s);
      }
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane + 32 * i == e) key[i] = 0u;
    if (lane == j) {
      mine = win;
      id = e;
    }
  }
  const float v = key_logit(mine);
  const float w = lane < p.top_k ? expf(v - top) : 0.0f;
  if (p.renormalize) all = warp_sum(w);
  const bool live = lane < p.top_k && v != -INFINITY;
  if (!live) id = -1;
  weight = live ? w / all : 0.0f;
}

// Exclusive prefix sum of total[0, E) into base (E + 1 values), by warp 0.
__device__ __forceinline__ void route_scan(const int32_t* total, int32_t* base, int E, int lane) {
  int sum = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    int v = e0 + lane < E ? total[e0 + lane] : 0;
    const int own = v;
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (e0 + lane < E) base[e0 + lane] = sum + v - own;
    sum += __shfl_sync(0xffffffffu, v, 31);
  }
  if (lane == 0) base[E] = sum;
}

// MULTI: the choices and each CTA's counts only; otherwise (one CTA) everything.
template <int EPL, bool MULTI>
__global__ void __launch_bounds__(route::threads(EPL)) route_topk_kernel(const RouteParams p) {
  using namespace route;
  constexpr int THREADS = threads(EPL);
  constexpr int WARPS = THREADS / 32;
  // MULTI counts with integer atomics; the one-CTA form keeps the masks.
  __shared__ uint32_t mask[MULTI ? 1 : MAX_WORDS][MULTI ? 1 : EPL * 32];
  __shared__ int32_t count[EPL * 32];
  __shared__ int32_t base[MULTI ? 1 : EPL * 32 + 1];
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  if (!MULTI) pdl_launch_dependents();
  for (int e = threadIdx.x; e < p.E; e += THREADS) {
    count[e] = 0;
    if (!MULTI)
      for (int w = 0; w < MAX_WORDS; ++w) mask[w][e] = 0u;
  }
  __syncthreads();
  pdl_wait();
  const int t0 = blockIdx.x * p.per_block;
  const int t1 = min(t0 + p.per_block, p.T);
  uint32_t key[EPL];
  if (t0 + warp < t1) route_load<EPL>(p, t0 + warp, lane, key);
  for (int t = t0 + warp; t < t1; t += WARPS) {
    uint32_t next[EPL];
    if (t + WARPS < t1) route_load<EPL>(p, t + WARPS, lane, next);
    int id;
    float w;
    route_token<EPL>(p, lane, key, id, w);
    if (lane < p.top_k) {
      p.ids[size_t(t) * p.top_k + lane] = id;
      p.weights[size_t(t) * p.top_k + lane] = w;
      if (id >= 0) {
        if (MULTI) atomicAdd(&count[id], 1);
        else atomicOr(&mask[(t - t0) >> 5][id], 1u << ((t - t0) & 31));
      }
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = next[i];
  }
  __syncthreads();
  if (MULTI) {
    for (int e = threadIdx.x; e < p.E; e += THREADS) p.counts[size_t(blockIdx.x) * p.E + e] = count[e];
    return;
  }
  for (int e = threadIdx.x; e < p.E; e += THREADS) {
    int c = 0;
    for (int w = 0; w < MAX_WORDS; ++w) c += __popc(mask[w][e]);
    count[e] = c;
  }
  __syncthreads();
  if (warp == 0) route_scan(count, base, p.E, lane);
  __syncthreads();
  for (int e = threadIdx.x; e <= p.E; e += THREADS) p.offsets[e] = base[e];
  const int slots = p.T * p.top_k;
  for (int s = threadIdx.x; s < slots; s += THREADS) {
    const int t = s / p.top_k;
    const int e = p.ids[s];  // this CTA's own stores, behind the barriers above
    int r = -1;
    if (e >= 0) {
      r = base[e] + __popc(mask[t >> 5][e] & ((1u << (t & 31)) - 1u));
      for (int w = 0; w < (t >> 5); ++w) r += __popc(mask[w][e]);
      p.rows[r] = t;
    }
    p.place[s] = r;
    if (s >= base[p.E]) p.rows[s] = -1;
  }
}

// The choices and each CTA's counts where the tokens are many and the experts
// few: a thread takes a token.  A warp brings the 32 tokens' logits, one
// contiguous stretch, into shared memory (an odd pitch), and each lane scans its
// row once, keeping the K best in order; an equal logit does not displace an
// earlier one.  About E (5 + 3 K) instructions for 32 tokens where the warp per
// token takes about 250 for one: 65520 tokens, 31 experts, 2 chosen, 22 us
// (issue bound) against 4.
template <int K>
__global__ void __launch_bounds__(route::ROW_THREADS) route_rows_kernel(const RouteParams p) {
  using namespace route;
  extern __shared__ float tile[];  // [warps][32][pitch]
  __shared__ int32_t count[ROW_MAX_E];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pitch = p.E | 1;
  float* const mine = tile + (warp * 32 + lane) * pitch;
  for (int e = threadIdx.x; e < p.E; e += ROW_THREADS) count[e] = 0;
  __syncthreads();
  pdl_wait();
  const int t0 = blockIdx.x * p.per_block;
  const int t1 = min(t0 + p.per_block, p.T);
  for (int u = t0 + warp * 32; u < t1; u += ROW_THREADS) {
    const int n = min(32, t1 - u) * p.E;
    __syncwarp();
    {
      const size_t from = size_t(u) * p.E;
      int r = lane / p.E, c = lane - r * p.E;  // of element `lane`, then 32 on
      const int rs = 32 / p.E, cs = 32 - rs * p.E;
      float* w = tile + warp * 32 * pitch;
      for (int i = lane; i < n; i += 32 * 16) {
        float v[16];
        load_logits<16>(p, from + i, 32, i, n, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (i + 32 * j < n) w[r * pitch + c] = v[j];
          r += rs;
          c += cs;
          if (c >= p.E) {
            c -= p.E;
            ++r;
          }
        }
      }
    }
    __syncwarp();
    const int t = u + lane;
    if (t < t1) {
      uint32_t key[K];
      int id[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        key[k] = 0u;
        id[k] = -1;
      }
#pragma unroll 8
      for (int e = 0; e < p.E; ++e) {
        uint32_t x = logit_key(mine[e]);
        int xi = e;
        bool up = false;
#pragma unroll
        for (int k = 0; k < K; ++k) {  // sink to its place, then all behind it move one on
          up = up || x > key[k];
          const uint32_t y = key[k];
          const int yi = id[k];
          key[k] = up ? x : y;
          id[k] = up ? xi : yi;
          x = up ? y : x;
          xi = up ? yi : xi;
        }
      }
      const float first = key_logit(key[0]);
      const float top = first == -INFINITY ? 0.0f : first;
      float w[K], all = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        w[k] = k < p.top_k ? expf(key_logit(key[k]) - top) : 0.0f;
        all += w[k];
      }
      if (!p.renormalize) {
        all = 0.0f;
#pragma unroll 8
        for (int e = 0; e < p.E; ++e) all += expf(mine[e] - top);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (k < p.top_k) {
          const bool live = key_logit(key[k]) != -INFINITY;
          p.ids[size_t(t) * p.top_k + k] = live ? id[k] : -1;
          p.weights[size_t(t) * p.top_k + k] = live ? w[k] / all : 0.0f;
          if (live) atomicAdd(&count[id[k]], 1);
        }
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += ROW_THREADS) p.counts[size_t(blockIdx.x) * p.E + e] = count[e];
}

// The slots' rows.  Each CTA adds up the counts of the CTAs before it (and all
// of them, for the offsets), then places its own slots in order.
__global__ void __launch_bounds__(route::THREADS) route_place_kernel(const RouteParams p) {
  using namespace route;
  __shared__ uint32_t mask[MAX_WORDS][MAX_E];
  __shared__ int32_t before[MAX_E], total[MAX_E];
  __shared__ int32_t base[MAX_E + 1];
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < p.E; e += THREADS) {
    before[e] = total[e] = 0;
    for (int w = 0; w < MAX_WORDS; ++w) mask[w][e] = 0u;
  }
  __syncthreads();
  pdl_wait();
  // This CTA's slots of the first PASS tokens: on their way while the counts are added.
  const int t0 = blockIdx.x * p.per_block;
  const int t1 = min(t0 + p.per_block, p.T);
  int id[SLOTS];
  auto load_ids = [&](int u0) {
    const int s1 = min(u0 + PASS, t1) * p.top_k;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int s = u0 * p.top_k + int(threadIdx.x) + i * THREADS;
      id[i] = s < s1 ? p.ids[s] : -1;
    }
  };
  load_ids(t0);
  // Neighbouring threads take neighbouring experts; the CTAs' counts are shared
  // out over the groups of `span` threads.
  const int span = min((p.E + 31) & ~31, THREADS);
  const int groups = THREADS / span;
  const int grp = threadIdx.x / span;
  if (grp < groups) {
    for (int e = threadIdx.x - grp * span; e < p.E; e += span) {
      int32_t b = 0, a = 0;
#pragma unroll 8
      for (int i = grp; i < p.blocks; i += groups) {
        const int32_t c = p.counts[size_t(i) * p.E + e];
        a += c;
        b += i < int(blockIdx.x) ? c : 0;
      }
      atomicAdd(&total[e], a);
      atomicAdd(&before[e], b);
    }
  }
  __syncthreads();
  if (warp == 0) route_scan(total, base, p.E, lane);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= p.E; e += THREADS) p.offsets[e] = base[e];
  const int live = base[p.E], slots = p.T * p.top_k;
  for (int r = live + int(blockIdx.x * THREADS + threadIdx.x); r < slots; r += int(gridDim.x) * THREADS)
    p.rows[r] = -1;
  for (int u0 = t0; u0 < t1; u0 += PASS) {  // PASS tokens at a time
    const int u1 = min(u0 + PASS, t1);
    const int words = (u1 - u0 + 31) >> 5;
    const int s1 = u1 * p.top_k;
    if (u0 != t0) {
      load_ids(u0);
      for (int e = threadIdx.x; e < p.E; e += THREADS)
        for (int w = 0; w < words; ++w) mask[w][e] = 0u;
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      if (u0 * p.top_k + i * THREADS >= s1) break;
      if (id[i] >= 0) {
        const int u = (u0 * p.top_k + int(threadIdx.x) + i * THREADS) / p.top_k - u0;
        atomicOr(&mask[u >> 5][id[i]], 1u << (u & 31));
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int s = u0 * p.top_k + int(threadIdx.x) + i * THREADS;
      if (u0 * p.top_k + i * THREADS >= s1) break;
      if (s < s1) {
        const int t = s / p.top_k, u = t - u0, e = id[i];
        int r = -1;
        if (e >= 0) {
          r = base[e] + before[e] + __popc(mask[u >> 5][e] & ((1u << (u & 31)) - 1u));
          for (int w = 0; w < (u >> 5); ++w) r += __popc(mask[w][e]);
          p.rows[r] = t;
        }
        p.place[s] = r;
      }
    }
    if (u1 < t1) {
      __syncthreads();
      for (int e = threadIdx.x; e < p.E; e += THREADS) {
        int c = 0;
        for (int w = 0; w < words; ++w) c += __popc(mask[w][e]);
        before[e] += c;
      }
      __syncthreads();
    }
  }
}

// out[t,:] = sum_j weights[t,j] * y[place[t,j],:] (+ residual[t,:]), in fp32, j
// ascending, rounded once.  A place outside [0, R) adds nothing.
struct CombineParams {
  const void* y;          // [R, N] of DT
  const int32_t* place;   // [T, top_k]
  const float* weights;   // [T, top_k]
  const void* residual;   // [T, N] of DT or NULL; may be out
  void* out;              // [T, N] of DT
  int64_t R, T, N;
  int top_k;
  uint32_t per_row;       // vectors (or elements) of a row
};

// VEC elements of a row per thread (16 bytes, or one where a row or an address
// is not a multiple of 16 bytes).  One pass over the rows, HBM bound: a thread's
// residual and two slots' loads are in flight together, and 42 registers keep six
// CTAs of 256 threads on an SM.  4096 tokens, top 2, fp32 / 16-bit: 73 / 34 us at N =
// 5120 (the bytes: 51 / 26), 121 / 166 at N = 5119, where one element a thread keeps
// too few bytes in flight.
template <int DT, int VEC>
__global__ void __launch_bounds__(256, 6) combine_kernel(const CombineParams p) {
  constexpr int ESZ = DT == TG_DT_F32 ? 4 : 2;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  // A 32-bit division wherever the index fits.
  const int64_t t = (i >> 32) == 0 ? int64_t(uint32_t(i) / p.per_row) : i / int64_t(p.per_row);
  if (t >= p.T) return;
  const int64_t n = (i - t * p.per_row) * VEC;
  struct __align__(VEC * ESZ) Raw {
    char b[VEC * ESZ];
  };
  const int64_t o = (t * p.N + n) * ESZ;
  Raw res;
  if (p.residual) res = *reinterpret_cast<const Raw*>(static_cast<const char*>(p.residual) + o);
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
  const char* y = static_cast<const char*>(p.y) + n * ESZ;
  const int64_t pitch = p.N * ESZ;
  const int32_t* place = p.place + t * p.top_k;
  const float* weight = p.weights + t * p.top_k;
  for (int j = 0; j < p.top_k; j += 2) {
    const int64_t r0 = place[j], r1 = j + 1 < p.top_k ? place[j + 1] : -1;
    const bool ok0 = r0 >= 0 && r0 < p.R, ok1 = r1 >= 0 && r1 < p.R;
    Raw a, b;
    if (ok0) a = *reinterpret_cast<const Raw*>(y + r0 * pitch);
    if (ok1) b = *reinterpret_cast<const Raw*>(y + r1 * pitch);
    if (ok0) {
      const float w = weight[j];
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v] = fmaf(w, load_as_f32(&a, DT, v), acc[v]);
    }
    if (ok1) {
      const float w = weight[j + 1];
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v] = fmaf(w, load_as_f32(&b, DT, v), acc[v]);
    }
  }
  if (p.residual) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] += load_as_f32(&res, DT, v);
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) store_f32_as(&res, DT, v, acc[v]);
  *reinterpret_cast<Raw*>(static_cast<char*>(p.out) + o) = res;
}

}  // namespace tg
