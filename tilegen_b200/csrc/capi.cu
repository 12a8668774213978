// Host side of the tilegen_b200 C ABI (include/tilegen_b200.h): argument
// checks, launch-shape selection, TMA descriptor encoding and the launches.
// One translation unit holds every kernel so they share the device status word.
#include <cstdio>
#include <cstring>
#include <atomic>
#include <mutex>

#include "common.cuh"
#include "experts.cuh"
#include "gemm_grouped.cuh"
#include "gemm_i8.cuh"
#include "gemm_splitk.cuh"
#include "gemv_i4.cuh"
#include "gemv_i8.cuh"
#include "rotquant.cuh"

namespace {

constexpr int kMaxDevices = 64;
constexpr int64_t kRotQuantMaxK = 32768;
// Most rows that kernels with tiles of up to 256 rows and 32-bit row numbers take:
// the numbers of a last tile's absent rows stay below 2^31 too.
constexpr int64_t kMaxTiledRows = (int64_t(1) << 31) - 256;

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

struct DeviceInfo {
  int sms = 0;       // SMs the persistent kernels may use (the SM budget applied)
  int sms_all = 0;   // SMs of the device
};

// Process-wide cap on the SMs the persistent kernels (rotate+quant, the tiled
// GEMM) size their grids for; 0 = every SM (tg_set_sm_budget).
std::atomic<int> g_sm_budget{0};

bool current_device(int* dev, DeviceInfo* info) {
  static std::atomic<int> known[kMaxDevices];  // SMs; 0: not asked yet.  Threads may make their first calls together.
  if (cudaGetDevice(dev) != cudaSuccess || *dev < 0 || *dev >= kMaxDevices) return false;
  int v = known[*dev].load(std::memory_order_relaxed);
  if (v == 0) {
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, *dev) != cudaSuccess || v <= 0) return false;
    known[*dev].store(v, std::memory_order_relaxed);
  }
  info->sms = info->sms_all = v;
  const int budget = g_sm_budget.load(std::memory_order_relaxed);
  if (budget > 0 && budget < info->sms) info->sms = budget;
  return true;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// 2-D tiled tensor map, innermost dimension first.
bool make_tmap_2d(CUtensorMap* m, CUtensorMapDataType dt, const void* base, uint64_t inner, uint64_t outer,
                  uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle swz) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {row_bytes};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, dt, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Per-(kernel, device) one-time attribute setup.
template <typename K>
bool ensure_smem_attr(K kernel, int dev, uint32_t bytes, uint32_t* done_bytes) {
  if (done_bytes[dev] >= bytes) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)) != cudaSuccess)
    return false;
  done_bytes[dev] = bytes;
  return true;
}

// ------------------------------------------------------------------ rotate+quant
// Dynamic shared memory of a launch: alignment slack, the ring of `stages`
// slots, their mbarriers, the row maxima and NaN flags ([3][R] each), and for
// the LayerNorm prologue its partial sums (the CTA has stage_bytes / 128 threads).
uint32_t rotquant_smem(int stages, uint32_t stage_bytes, int R, bool ln) {
  const uint32_t ln_bytes = ln ? uint32_t(tg::ln_words(int(stage_bytes / 128u), R)) * 4u : 0u;
  return 1024u + uint32_t(stages) * stage_bytes + uint32_t(stages) * 8u + uint32_t(6 * R) * 4u + ln_bytes;
}

constexpr uint32_t kSmemPerCtaMax = 232448u;  // 227 KB: the opt-in maximum of one CTA
constexpr uint32_t kSmemPerSm = 233472u;      // 228 KB per SM, 1 KB of it reserved per resident CTA

// CTAs per SM that a rotquant variant's registers allow (with the shallowest
// ring), and the deepest ring (2 to 4 slots) that that many CTAs fit.
template <int NST, bool BF16, int ACT, bool EXACT, int REGS>
bool rotquant_shape(int dev, int threads, uint32_t stage_bytes, int R, int* occ_out, int* stages_out) {
  static uint32_t attr_done[kMaxDevices];
  static uint32_t static_smem = ~0u;
  // (occ | stages << 8) per device, CTA width in warps and rows per batch; 0 = not known yet.
  static int known[kMaxDevices][17][9];
  const int tw = threads / 32;
  if (tw <= 16 && R <= 8 && known[dev][tw][R] != 0) {
    *occ_out = known[dev][tw][R] & 0xff;
    *stages_out = known[dev][tw][R] >> 8;
    return true;
  }
  auto kern = tg::rotquant_kernel<NST, BF16, ACT, EXACT, REGS>;
  if (static_smem == ~0u) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess) return false;
    static_smem = uint32_t(fa.sharedSizeBytes);
  }
  const uint32_t dyn_max = kSmemPerCtaMax - static_smem;  // static + dynamic <= the per-CTA maximum
  if (!ensure_smem_attr(kern, dev, dyn_max, attr_done)) return false;
  int occ = 0;
  constexpr bool kLn = ACT == tg::kActLnMod;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, threads, rotquant_smem(2, stage_bytes, R, kLn)) !=
          cudaSuccess ||
      occ < 1)
    return false;
  int stages = 4;
  while (stages > 2 && (rotquant_smem(stages, stage_bytes, R, kLn) > dyn_max ||
                        uint64_t(occ) * (rotquant_smem(stages, stage_bytes, R, kLn) + static_smem + 1024u) >
                            kSmemPerSm))
    --stages;
  *occ_out = occ;
  *stages_out = stages;
  if (tw <= 16 && R <= 8) known[dev][tw][R] = occ | (stages << 8);
  return true;
}

template <int NST, bool BF16, int ACT, bool EXACT, int REGS>
int launch_rotquant_t(const CUtensorMap& tm, tg::RotQuantParams p, int threads, int occ, int dev, int sms,
                      cudaStream_t st) {
  auto kern = tg::rotquant_kernel<NST, BF16, ACT, EXACT, REGS>;
  const uint32_t smem = rotquant_smem(p.stages, p.stage_bytes, p.rows_per_batch, ACT == tg::kActLnMod);
  const int64_t grid64 = std::min<int64_t>(p.nbatches, int64_t(sms) * occ);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(unsigned(grid64));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, tm, p) != cudaSuccess) return TG_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? TG_OK : TG_ERR_CUDA;
}

// The register budget.  96 registers a thread by default; the hot form (G=256,
// short order, no activation) also has an 80-register build, taken when it
// keeps more warps resident: a CTA of seven warps (K=13824: 216 lines a row)
// fits twice per SM at 96 registers (five warps' registers per SM
// sub-partition) but three times at 80.
template <int NST, bool BF16, int ACT, bool EXACT>
int launch_rotquant_regs(const CUtensorMap& tm, tg::RotQuantParams p, int threads, int dev, int sms,
                         cudaStream_t st) {
  int occ = 0, stages = 0;
  if (!rotquant_shape<NST, BF16, ACT, EXACT, 96>(dev, threads, p.stage_bytes, p.rows_per_batch, &occ, &stages))
    return TG_ERR_CUDA;
  if constexpr (NST == 4 && ACT == tg::kActNone && !EXACT) {
    int occ80 = 0, stages80 = 0;
    if (!rotquant_shape<NST, BF16, ACT, EXACT, 80>(dev, threads, p.stage_bytes, p.rows_per_batch, &occ80,
                                                   &stages80))
      return TG_ERR_CUDA;
    if (occ80 > occ) {
      p.stages = stages80;
      return launch_rotquant_t<NST, BF16, ACT, EXACT, 80>(tm, p, threads, occ80, dev, sms, st);
    }
  }
  p.stages = stages;
  return launch_rotquant_t<NST, BF16, ACT, EXACT, 96>(tm, p, threads, occ, dev, sms, st);
}

// Internal code of the LayerNorm + modulation prologue (tg_quantize_ln_mod),
// beside the public TG_ACT_* codes.
constexpr int kLnModCode = 3;

template <int NST, bool BF16, bool EXACT>
int launch_rotquant_act(int act, const CUtensorMap& tm, const tg::RotQuantParams& p, int threads, int dev, int sms,
                        cudaStream_t st) {
  switch (act) {
    case TG_ACT_GELU_TANH:
      return launch_rotquant_regs<NST, BF16, tg::kActGeluTanh, EXACT>(tm, p, threads, dev, sms, st);
    case TG_ACT_GELU: return launch_rotquant_regs<NST, BF16, tg::kActGelu, EXACT>(tm, p, threads, dev, sms, st);
    case kLnModCode:
      // Built for the rotated groups in the short order only.
      if constexpr (NST > 0 && !EXACT) {
        return launch_rotquant_regs<NST, BF16, tg::kActLnMod, EXACT>(tm, p, threads, dev, sms, st);
      } else {
        return TG_ERR_UNSUPPORTED;
      }
    default: return launch_rotquant_regs<NST, BF16, tg::kActNone, EXACT>(tm, p, threads, dev, sms, st);
  }
}

// The butterfly order: the reference kernel's (bit-identical to it) or the
// short one (the default).  The rotation-free form has no butterflies.
template <int NST, bool BF16>
int launch_rotquant_order(bool exact, int act, const CUtensorMap& tm, const tg::RotQuantParams& p, int threads,
                          int dev, int sms, cudaStream_t st) {
  if constexpr (NST == 0) {
    return launch_rotquant_act<NST, BF16, true>(act, tm, p, threads, dev, sms, st);
  } else {
    if (exact) return launch_rotquant_act<NST, BF16, true>(act, tm, p, threads, dev, sms, st);
    return launch_rotquant_act<NST, BF16, false>(act, tm, p, threads, dev, sms, st);
  }
}

int gcd_int(int a, int b) {
  while (b) {
    const int t = a % b;
    a = b;
    b = t;
  }
  return a;
}

// The LayerNorm + modulation prologue's arguments (tg_quantize_ln_mod).
struct LnModArgs {
  const void* scale;
  const void* shift;
  int64_t rows;
  float eps;
};

// The shared body of tg_quantize_act and tg_quantize_ln_mod: shape checks,
// launch shape, tensor map, launch.
int quantize_launch(const void* x, int x_dtype, int64_t M, int64_t K, int group, int act, bool exact,
                    const LnModArgs* ln, int8_t* q, float* scale, void* stream);

}  // namespace

extern "C" {

int tg_version(void) { return (0 << 16) | 1; }

const char* tg_status_string(int s) {
  switch (s) {
    case TG_OK: return "ok";
    case TG_ERR_INVALID_ARG: return "invalid argument";
    case TG_ERR_UNSUPPORTED: return "unsupported shape or group size";
    case TG_ERR_MISALIGNED: return "pointer not 16-byte aligned";
    case TG_ERR_CUDA: return "CUDA call failed";
    case TG_ERR_DEVICE_TIMEOUT: return "a kernel's bounded wait expired";
    default: return "unknown status";
  }
}

int64_t tg_rotate_quant_max_k(void) { return kRotQuantMaxK; }

int tg_rotate_quant(const void* x, int x_dtype, int64_t M, int64_t K, int group, int8_t* q, float* scale,
                    void* stream) {
  if (group == 1) {  // the rotation-free branch is tg_quantize_act's
    if (M < 0 || K <= 0 || (x_dtype != TG_DT_F16 && x_dtype != TG_DT_BF16)) return TG_ERR_INVALID_ARG;
    return TG_ERR_UNSUPPORTED;
  }
  return tg_quantize_act(x, x_dtype, M, K, group, TG_ACT_NONE, q, scale, stream);
}

int tg_quantize_act(const void* x, int x_dtype, int64_t M, int64_t K, int group, int act, int8_t* q, float* scale,
                    void* stream) {
  if (M < 0 || K <= 0) return TG_ERR_INVALID_ARG;
  if (x_dtype != TG_DT_F16 && x_dtype != TG_DT_BF16) return TG_ERR_INVALID_ARG;
  const bool exact = (act & TG_QUANT_REFERENCE_ORDER) != 0;
  act &= ~TG_QUANT_REFERENCE_ORDER;
  if (act != TG_ACT_NONE && act != TG_ACT_GELU_TANH && act != TG_ACT_GELU) return TG_ERR_INVALID_ARG;
  return quantize_launch(x, x_dtype, M, K, group, act, exact, nullptr, q, scale, stream);
}

int tg_quantize_ln_mod(const void* x, int x_dtype, int64_t M, int64_t K, int group, float eps, const void* mod_scale,
                       const void* mod_shift, int64_t mod_rows, int8_t* q, float* scale, void* stream) {
  if (M < 0 || K <= 0 || mod_rows < 1) return TG_ERR_INVALID_ARG;
  if (x_dtype != TG_DT_F16 && x_dtype != TG_DT_BF16) return TG_ERR_INVALID_ARG;
  if (!(eps >= 0.0f) || eps > 3.0e38f) return TG_ERR_INVALID_ARG;  // also rejects NaN
  if (group == 1) return TG_ERR_UNSUPPORTED;                         // rotated groups only
  if (M > 0) {
    if (!mod_scale || !mod_shift) return TG_ERR_INVALID_ARG;
    if (!aligned16(mod_scale) || !aligned16(mod_shift)) return TG_ERR_MISALIGNED;
  }
  const LnModArgs ln{mod_scale, mod_shift, mod_rows, eps};
  return quantize_launch(x, x_dtype, M, K, group, kLnModCode, false, &ln, q, scale, stream);
}

}  // extern "C"

namespace {

int quantize_launch(const void* x, int x_dtype, int64_t M, int64_t K, int group, int act, bool exact,
                    const LnModArgs* ln, int8_t* q, float* scale, void* stream) {
  int nst;
  switch (group) {
    case 1: nst = 0; break;
    case 4: nst = 1; break;
    case 16: nst = 2; break;
    case 64: nst = 3; break;
    case 256: nst = 4; break;
    default: return TG_ERR_UNSUPPORTED;
  }
  // Rotated: K % 256 as the reference launcher requires (int8_convrot.py:196-230).
  // Row-wise: whole 64-element lines (one thread owns one).
  if (K % (nst == 0 ? 64 : 256) != 0 || K > kRotQuantMaxK) return TG_ERR_UNSUPPORTED;
  if (M == 0) return TG_OK;
  if (!x || !q || !scale) return TG_ERR_INVALID_ARG;
  if (!aligned16(x) || !aligned16(q) || (reinterpret_cast<uintptr_t>(scale) & 3u)) return TG_ERR_MISALIGNED;
  const int cpr = int(K / 64);
  // 32-bit line and batch indices in the kernel (with up to 8 rows of slack).
  if ((M + 8) * int64_t(cpr) >= (int64_t(1) << 31)) return TG_ERR_UNSUPPORTED;

  // Rows per batch: the fewest that fill whole warps to within 5 %.
  int R = 1;
  for (int r = 1; r <= 8; ++r) {
    const int lines = r * cpr;
    const int thr = (lines + 31) / 32 * 32;
    if (thr > 512) break;
    if ((thr - lines) * 20 <= lines) {
      R = r;
      break;
    }
  }
  const int active = R * cpr;
  const int threads = (active + 31) / 32 * 32;
  if (threads > 512) return TG_ERR_UNSUPPORTED;
  int box = active;
  if (box > 256) {
    box = 4;
    for (int d = 256; d >= 4; --d)
      if (active % d == 0) {
        box = d;
        break;
      }
  }
  // The ring's depth (2 to 4 slots) is chosen at launch from the kernel's
  // occupancy (launch_rotquant_regs).
  const uint32_t stage_bytes = uint32_t(threads) * 128u;

  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;

  CUtensorMap tm;
  if (!make_tmap_2d(&tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, x, 64, uint64_t(M) * uint64_t(cpr), 128, 64,
                    uint32_t(box), CU_TENSOR_MAP_SWIZZLE_128B))
    return TG_ERR_CUDA;

  tg::RotQuantParams p;
  p.q = q;
  p.scale = scale;
  p.M = M;
  p.K = int(K);
  p.cpr = cpr;
  p.rows_per_batch = R;
  p.active = active;
  p.box_lines = box;
  p.boxes = active / box;
  p.nbatches = (M + R - 1) / R;
  p.stages = 2;
  p.stage_bytes = stage_bytes;
  p.seg = gcd_int(cpr, 32);
  p.mod_scale = ln ? ln->scale : nullptr;
  p.mod_shift = ln ? ln->shift : nullptr;
  p.mod_rows = ln ? ln->rows : 1;
  p.ln_eps = ln ? ln->eps : 0.0f;
  p.ln_inv_k = 1.0f / float(K);

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = x_dtype == TG_DT_BF16;
#define TG_RQ_CASE(N)                                                                           \
  case N:                                                                                       \
    return bf ? launch_rotquant_order<N, true>(exact, act, tm, p, threads, dev, info.sms, st) \
              : launch_rotquant_order<N, false>(exact, act, tm, p, threads, dev, info.sms, st);
  switch (nst) {
    TG_RQ_CASE(0)
    TG_RQ_CASE(1)
    TG_RQ_CASE(2)
    TG_RQ_CASE(3)
    default:
      return bf ? launch_rotquant_order<4, true>(exact, act, tm, p, threads, dev, info.sms, st)
                : launch_rotquant_order<4, false>(exact, act, tm, p, threads, dev, info.sms, st);
  }
#undef TG_RQ_CASE
}

}  // namespace

namespace {

template <int BN, int OUT, bool HAS_BIAS, bool PAIR>
int launch_gemm_t(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& to, const tg::GemmParams& p,
                  int dev, int units, cudaStream_t st) {
  static uint32_t attr_done[kMaxDevices];
  constexpr uint32_t smem = tg::gemm::smem_bytes(BN, PAIR);
  auto kern = tg::gemm_i8_dequant_kernel<BN, OUT, HAS_BIAS, PAIR>;
  if (!ensure_smem_attr(kern, dev, smem, attr_done)) return TG_ERR_CUDA;
  const int tiles = p.m_tiles * p.n_tiles;
  const int grid_units = tiles < units ? tiles : units;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(unsigned(grid_units * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(tg::gemm::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  // Programmatic dependent launch: the prologue overlaps the previous kernel
  // (the quantiser), the kernel waits for it before reading xq/xscale.
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, ta, tb, to, p) != cudaSuccess) return TG_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? TG_OK : TG_ERR_CUDA;
}

template <int BN, bool PAIR>
int launch_gemm_bn(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& to, const tg::GemmParams& p,
                   int out_dtype, bool has_bias, int dev, int units, cudaStream_t st) {
  switch (out_dtype) {
    case TG_DT_F32: return has_bias ? launch_gemm_t<BN, 0, true, PAIR>(ta, tb, to, p, dev, units, st)
                                    : launch_gemm_t<BN, 0, false, PAIR>(ta, tb, to, p, dev, units, st);
    case TG_DT_F16: return has_bias ? launch_gemm_t<BN, 1, true, PAIR>(ta, tb, to, p, dev, units, st)
                                    : launch_gemm_t<BN, 1, false, PAIR>(ta, tb, to, p, dev, units, st);
    default: return has_bias ? launch_gemm_t<BN, 2, true, PAIR>(ta, tb, to, p, dev, units, st)
                             : launch_gemm_t<BN, 2, false, PAIR>(ta, tb, to, p, dev, units, st);
  }
}

template <bool PAIR>
int launch_gemm_mode(int bn, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& to,
                     const tg::GemmParams& p, int out_dtype, bool hb, int dev, int units, cudaStream_t st) {
  switch (bn) {
    case 224: return launch_gemm_bn<224, PAIR>(ta, tb, to, p, out_dtype, hb, dev, units, st);
    case 192: return launch_gemm_bn<192, PAIR>(ta, tb, to, p, out_dtype, hb, dev, units, st);
    case 160: return launch_gemm_bn<160, PAIR>(ta, tb, to, p, out_dtype, hb, dev, units, st);
    case 128: return launch_gemm_bn<128, PAIR>(ta, tb, to, p, out_dtype, hb, dev, units, st);
    default: return launch_gemm_bn<256, PAIR>(ta, tb, to, p, out_dtype, hb, dev, units, st);
  }
}

// Tile-processing units that can be resident at once: SMs for single-CTA
// tiles, co-resident clusters of 2 for pair tiles (queried once per device).
int gemm_units(int dev, int sms, bool pair) {
  static int cache[kMaxDevices];
  if (!pair) return sms;
  if (cache[dev] > 0) return cache[dev] < sms / 2 ? cache[dev] : sms / 2;
  int all = sms;
  if (cudaDeviceGetAttribute(&all, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) all = sms;
  auto kern = tg::gemm_i8_dequant_kernel<256, 1, false, true>;
  constexpr uint32_t smem = tg::gemm::smem_bytes(256, true);
  static uint32_t attr_done[kMaxDevices];
  int n = 0;
  if (ensure_smem_attr(kern, dev, smem, attr_done)) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(unsigned(all));
    cfg.blockDim = dim3(tg::gemm::THREADS);
    cfg.dynamicSmemBytes = smem;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) n = 0;
  }
  cache[dev] = n > 0 ? n : all / 2;
  return cache[dev] < sms / 2 ? cache[dev] : sms / 2;
}

// Tile shape for an M x N problem.  The persistent grid runs
// ceil(tiles / units) waves of tiles costing about (BN + kTileOverhead) column
// steps each; pick the width minimising waves * (BN + overhead).  Pair tiles
// (256 rows on two SMs) are used whenever M has more than one 128-row block.
constexpr int kGemmWidths[] = {256, 224, 192, 160, 128};
constexpr int kTileOverhead = 32;
int g_forced_bn = 0;     // tg_set_gemm_config(): 0 = cost model
int g_forced_pair = -1;  // -1 = by M

void pick_gemm_config(int64_t M, int64_t N, int dev, int sms, int* bn_out, int* pair_out) {
  const bool pair = g_forced_pair >= 0 ? g_forced_pair != 0 : M > tg::gemm::BM;
  const int units = gemm_units(dev, sms, pair);
  const int64_t tm = pair ? 2 * tg::gemm::BM : tg::gemm::BM;
  const int64_t mt = (M + tm - 1) / tm;
  int best = 256;
  int64_t best_cost = -1;
  for (int bn : kGemmWidths) {
    const int64_t tiles = mt * ((N + bn - 1) / bn);
    const int64_t waves = (tiles + units - 1) / units;
    const int64_t cost = waves * (bn + kTileOverhead);
    if (best_cost < 0 || cost < best_cost) {
      best_cost = cost;
      best = bn;
    }
  }
  *bn_out = g_forced_bn ? g_forced_bn : best;
  *pair_out = pair ? 1 : 0;
}

}  // namespace

extern "C" {

int tg_int8_gemm_dequant(const int8_t* xq, const float* xscale, const int8_t* wq, const float* wscale,
                         int64_t wscale_numel, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K,
                         int out_dtype, void* out, void* stream) {
  using namespace tg::gemm;
  if (M < 0 || N <= 0 || K <= 0) return TG_ERR_INVALID_ARG;
  if (out_dtype != TG_DT_F32 && out_dtype != TG_DT_F16 && out_dtype != TG_DT_BF16) return TG_ERR_INVALID_ARG;
  if (bias && bias_dtype != TG_DT_F32 && bias_dtype != TG_DT_F16 && bias_dtype != TG_DT_BF16)
    return TG_ERR_INVALID_ARG;
  if (wscale_numel != 1 && wscale_numel != N) return TG_ERR_INVALID_ARG;
  const int esz = out_dtype == TG_DT_F32 ? 4 : 2;
  if (K % 16 != 0 || (N * esz) % 16 != 0) return TG_ERR_UNSUPPORTED;
  if (M >= (int64_t(1) << 31) || N >= (int64_t(1) << 31) || K >= (int64_t(1) << 31)) return TG_ERR_UNSUPPORTED;
  if (M == 0) return TG_OK;
  if (!xq || !xscale || !wq || !wscale || !out) return TG_ERR_INVALID_ARG;
  if (!aligned16(xq) || !aligned16(wq) || !aligned16(out)) return TG_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(xscale) & 3u) || (reinterpret_cast<uintptr_t>(wscale) & 3u))
    return TG_ERR_MISALIGNED;

  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;

  int bn, pair;
  pick_gemm_config(M, N, dev, info.sms, &bn, &pair);
  const int ch_bytes = (bn * esz) % 128 == 0 ? 128 : 64;  // epilogue chunk row bytes (kernel's CH_BYTES)

  CUtensorMap ta, tb, to;
  if (!make_tmap_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, xq, uint64_t(K), uint64_t(M), uint64_t(K), BK, BM,
                    CU_TENSOR_MAP_SWIZZLE_128B))
    return TG_ERR_CUDA;
  if (!make_tmap_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, wq, uint64_t(K), uint64_t(N), uint64_t(K), BK,
                    uint32_t(tg::gemm::b_rows(bn, pair != 0)), CU_TENSOR_MAP_SWIZZLE_128B))
    return TG_ERR_CUDA;
  const CUtensorMapDataType odt = out_dtype == TG_DT_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : out_dtype == TG_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (!make_tmap_2d(&to, odt, out, uint64_t(N), uint64_t(M), uint64_t(N) * esz, uint32_t(ch_bytes / esz), 32,
                    ch_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
    return TG_ERR_CUDA;

  tg::GemmParams p;
  p.xscale = xscale;
  p.wscale = wscale;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.wscale_bcast = wscale_numel == 1 ? 1 : 0;
  p.M = int(M);
  p.N = int(N);
  p.K = int(K);
  p.m_tiles = int((M + (pair ? 2 * BM : BM) - 1) / (pair ? 2 * BM : BM));
  p.n_tiles = int((N + bn - 1) / bn);
  p.k_blocks = int((K + int64_t(BK) * tg::gemm::ksub(pair != 0) - 1) / (int64_t(BK) * tg::gemm::ksub(pair != 0)));

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool hb = bias != nullptr;
  const int units = gemm_units(dev, info.sms, pair != 0);
  return pair ? launch_gemm_mode<true>(bn, ta, tb, to, p, out_dtype, hb, dev, units, st)
              : launch_gemm_mode<false>(bn, ta, tb, to, p, out_dtype, hb, dev, units, st);
}

int tg_set_sm_budget(int sms) {
  if (sms < 0) return TG_ERR_INVALID_ARG;
  g_sm_budget.store(sms, std::memory_order_relaxed);
  return TG_OK;
}

int tg_sm_budget(void) { return g_sm_budget.load(std::memory_order_relaxed); }

int tg_set_gemm_config(int bn, int pair) {
  if (pair < -1 || pair > 1) return TG_ERR_INVALID_ARG;
  bool ok = bn == 0;
  for (int w : kGemmWidths) ok = ok || w == bn;
  if (!ok) return TG_ERR_INVALID_ARG;
  g_forced_bn = bn;
  g_forced_pair = pair;
  return TG_OK;
}

int tg_gemm_config(int64_t M, int64_t N, int* bn, int* pair) {
  if (!bn || !pair) return TG_ERR_INVALID_ARG;
  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;
  pick_gemm_config(M, N, dev, info.sms, bn, pair);
  return TG_OK;
}

int tg_device_status(int device, uint32_t* bits, int clear) {
  if (!bits) return TG_ERR_INVALID_ARG;
  int prev;
  if (cudaGetDevice(&prev) != cudaSuccess) return TG_ERR_CUDA;
  if (device != prev && cudaSetDevice(device) != cudaSuccess) return TG_ERR_CUDA;
  unsigned int v = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, tg::g_device_status, sizeof(v));
  if (e == cudaSuccess && clear) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbol(tg::g_device_status, &zero, sizeof(zero));
  }
  if (device != prev) cudaSetDevice(prev);
  if (e != cudaSuccess) return TG_ERR_CUDA;
  *bits = v;
  return v ? TG_ERR_DEVICE_TIMEOUT : TG_OK;
}

}  // extern "C"

// ------------------------------------------------------------ small-M GEMM
namespace {

size_t round256(size_t v) { return (v + 255) & ~size_t(255); }

// The argument checks of tg_int8_gemm_dequant (M == 0 passes).
int check_gemm_args(const int8_t* xq, const float* xscale, const int8_t* wq, const float* wscale,
                    int64_t wscale_numel, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K,
                    int out_dtype, const void* out) {
  if (M < 0 || N <= 0 || K <= 0) return TG_ERR_INVALID_ARG;
  if (out_dtype != TG_DT_F32 && out_dtype != TG_DT_F16 && out_dtype != TG_DT_BF16) return TG_ERR_INVALID_ARG;
  if (bias && bias_dtype != TG_DT_F32 && bias_dtype != TG_DT_F16 && bias_dtype != TG_DT_BF16)
    return TG_ERR_INVALID_ARG;
  if (wscale_numel != 1 && wscale_numel != N) return TG_ERR_INVALID_ARG;
  const int esz = out_dtype == TG_DT_F32 ? 4 : 2;
  if (K % 16 != 0 || (N * esz) % 16 != 0) return TG_ERR_UNSUPPORTED;
  if (M >= (int64_t(1) << 31) || N >= (int64_t(1) << 31) || K >= (int64_t(1) << 31)) return TG_ERR_UNSUPPORTED;
  if (M == 0) return TG_OK;
  if (!xq || !xscale || !wq || !wscale || !out) return TG_ERR_INVALID_ARG;
  if (!aligned16(xq) || !aligned16(wq) || !aligned16(out)) return TG_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(xscale) & 3u) || (reinterpret_cast<uintptr_t>(wscale) & 3u))
    return TG_ERR_MISALIGNED;
  return TG_OK;
}

// Workspace of the split-K GEMM: [count: ceil(N/128) u32 | acc: M x N int32],
// each part 256-byte aligned.
struct SplitKWs {
  size_t count, acc, total;
};
SplitKWs splitk_ws(int64_t M, int64_t N) {
  SplitKWs w;
  const int64_t tiles = (N + tg::splitk::BNW - 1) / tg::splitk::BNW;
  w.count = 0;
  w.acc = round256(size_t(tiles) * 4);
  w.total = w.acc + round256(size_t(M) * size_t(N) * 4);
  return w;
}

// Whether the cluster form of the split-K kernel runs with `slices` CTAs per
// cluster on device `dev`: at most 8, and the occupancy calculator schedules at
// least one such cluster (cached per device and size).
template <int MPAD, int OUT, bool HAS_BIAS>
bool splitk_cluster_ok(int slices, int dev) {
  static uint32_t attr_done[kMaxDevices];
  static uint8_t ok_cache[kMaxDevices][9];  // 0 unknown, 1 yes, 2 no
  if (slices < 1 || slices > 8) return false;
  constexpr uint32_t smem = tg::splitk::smem_bytes(MPAD);
  auto kcl = tg::gemm_i8_splitk_kernel<MPAD, OUT, HAS_BIAS, true>;
  if (!ensure_smem_attr(kcl, dev, smem, attr_done)) {
    cudaGetLastError();
    return false;
  }
  uint8_t& ok = ok_cache[dev][slices];
  if (ok == 0) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(unsigned(slices), 1);
    cfg.blockDim = dim3(tg::splitk::THREADS);
    cfg.dynamicSmemBytes = smem;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(slices);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    ok = (cudaOccupancyMaxActiveClusters(&n, kcl, &cfg) == cudaSuccess && n > 0) ? 1 : 2;
    cudaGetLastError();  // a refusal here only selects the other form
  }
  return ok == 1;
}

template <int MPAD, int OUT, bool HAS_BIAS>
int launch_splitk_t(const CUtensorMap& tw, const CUtensorMap& tx, const tg::SplitKParams& p, int tiles, int dev,
                    cudaStream_t st) {
  static uint32_t attr_done[kMaxDevices];
  constexpr uint32_t smem = tg::splitk::smem_bytes(MPAD);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(unsigned(p.slices), unsigned(tiles));
  cfg.blockDim = dim3(tg::splitk::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(p.slices);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  // The slices of a column tile as one cluster, reduced in shared memory,
  // when K is split at most 8 ways and such a cluster fits on the device.
  if (splitk_cluster_ok<MPAD, OUT, HAS_BIAS>(p.slices, dev)) {
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, tg::gemm_i8_splitk_kernel<MPAD, OUT, HAS_BIAS, true>, tw, tx, p) != cudaSuccess)
      return TG_ERR_CUDA;
    return cudaGetLastError() == cudaSuccess ? TG_OK : TG_ERR_CUDA;
  }
  auto kern = tg::gemm_i8_splitk_kernel<MPAD, OUT, HAS_BIAS, false>;
  if (!ensure_smem_attr(kern, dev, smem, attr_done)) return TG_ERR_CUDA;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, tw, tx, p) != cudaSuccess) return TG_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? TG_OK : TG_ERR_CUDA;
}

template <int MPAD>
int launch_splitk_m(const CUtensorMap& tw, const CUtensorMap& tx, const tg::SplitKParams& p, int tiles,
                    int out_dtype, bool hb, int dev, cudaStream_t st) {
  switch (out_dtype) {
    case TG_DT_F32: return hb ? launch_splitk_t<MPAD, 0, true>(tw, tx, p, tiles, dev, st)
                              : launch_splitk_t<MPAD, 0, false>(tw, tx, p, tiles, dev, st);
    case TG_DT_F16: return hb ? launch_splitk_t<MPAD, 1, true>(tw, tx, p, tiles, dev, st)
                              : launch_splitk_t<MPAD, 1, false>(tw, tx, p, tiles, dev, st);
    default: return hb ? launch_splitk_t<MPAD, 2, true>(tw, tx, p, tiles, dev, st)
                       : launch_splitk_t<MPAD, 2, false>(tw, tx, p, tiles, dev, st);
  }
}

// K split of the small-M GEMM: about 1.6 CTAs per SM stream the weight
// (measured at M=1 on the DiT shapes: more in flight costs DRAM efficiency,
// fewer leaves bandwidth unused), so K is split until tiles x slices is nearest
// that, every slice non-empty.  Returns the slice count; *kb_per = k-blocks each.
int splitk_slices(int64_t N, int64_t K, int sms, int* kb_per) {
  using namespace tg::splitk;
  const int tiles = int((N + BNW - 1) / BNW);
  const int k_blocks = int((K + BK - 1) / BK);
  int slices = (16 * sms / 10 + tiles / 2) / tiles;
  slices = slices < 1 ? 1 : (slices > k_blocks ? k_blocks : slices);
  *kb_per = (k_blocks + slices - 1) / slices;
  return (k_blocks + *kb_per - 1) / *kb_per;
}

// The split-K launch over a zero-initialised scratch (count, acc), shared by
// the workspace entry point and any other caller that owns such scratch.
int splitk_launch(const int8_t* xq, const float* xscale, const int8_t* wq, const float* wscale,
                  int64_t wscale_numel, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K,
                  int out_dtype, void* out, uint32_t* count, int32_t* acc, void* stream) {
  using namespace tg::splitk;
  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;
  const int mpad = M <= 16 ? 16 : (M <= 32 ? 32 : (M <= 64 ? 64 : 128));
  const int tiles = int((N + BNW - 1) / BNW);
  const int k_blocks = int((K + BK - 1) / BK);
  int kb_per;
  const int slices = splitk_slices(N, K, info.sms, &kb_per);

  CUtensorMap tw, tx;
  if (!make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, wq, uint64_t(K), uint64_t(N), uint64_t(K), BK, BNW,
                    CU_TENSOR_MAP_SWIZZLE_128B))
    return TG_ERR_CUDA;
  if (!make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, xq, uint64_t(K), uint64_t(M), uint64_t(K), BK,
                    uint32_t(mpad), CU_TENSOR_MAP_SWIZZLE_128B))
    return TG_ERR_CUDA;
  tg::SplitKParams p;
  p.xscale = xscale;
  p.wscale = wscale;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.wscale_bcast = wscale_numel == 1 ? 1 : 0;
  p.M = int(M);
  p.N = int(N);
  p.K = int(K);
  p.k_blocks = k_blocks;
  p.kb_per_slice = kb_per;
  p.slices = slices;
  p.acc = acc;
  p.count = count;
  p.out = out;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool hb = bias != nullptr;
  switch (mpad) {
    case 16: return launch_splitk_m<16>(tw, tx, p, tiles, out_dtype, hb, dev, st);
    case 32: return launch_splitk_m<32>(tw, tx, p, tiles, out_dtype, hb, dev, st);
    case 64: return launch_splitk_m<64>(tw, tx, p, tiles, out_dtype, hb, dev, st);
    default: return launch_splitk_m<128>(tw, tx, p, tiles, out_dtype, hb, dev, st);
  }
}

}  // namespace

extern "C" {

size_t tg_int8_gemm_dequant_splitk_workspace(int64_t M, int64_t N) {
  if (M < 0 || N < 0) return 0;
  return splitk_ws(M, N).total;
}

int tg_int8_gemm_dequant_splitk(const int8_t* xq, const float* xscale, const int8_t* wq, const float* wscale,
                                int64_t wscale_numel, const void* bias, int bias_dtype, int64_t M, int64_t N,
                                int64_t K, int out_dtype, void* out, void* workspace, size_t workspace_bytes,
                                void* stream) {
  const int chk = check_gemm_args(xq, xscale, wq, wscale, wscale_numel, bias, bias_dtype, M, N, K, out_dtype, out);
  if (chk != TG_OK || M == 0) return chk;
  if (M > tg::splitk::M_MAX) return TG_ERR_UNSUPPORTED;
  if (!workspace) return TG_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return TG_ERR_MISALIGNED;
  const SplitKWs L = splitk_ws(M, N);
  if (workspace_bytes < L.total) return TG_ERR_INVALID_ARG;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return splitk_launch(xq, xscale, wq, wscale, wscale_numel, bias, bias_dtype, M, N, K, out_dtype, out,
                       reinterpret_cast<uint32_t*>(ws + L.count), reinterpret_cast<int32_t*>(ws + L.acc), stream);
}

int64_t tg_int8_gemm_dequant_splitk_max_m(void) { return tg::splitk::M_MAX; }

int tg_int8_gemm_dequant_splitk_config(int64_t M, int64_t N, int64_t K, int out_dtype, int has_bias, int* slices,
                                       int* cluster) {
  if (M < 1 || M > tg::splitk::M_MAX || N < 1 || K < 1 || !slices || !cluster) return TG_ERR_INVALID_ARG;
  if (out_dtype != TG_DT_F32 && out_dtype != TG_DT_F16 && out_dtype != TG_DT_BF16) return TG_ERR_INVALID_ARG;
  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;
  int kb_per;
  const int s = splitk_slices(N, K, info.sms, &kb_per);
  const int mpad = M <= 16 ? 16 : (M <= 32 ? 32 : (M <= 64 ? 64 : 128));
  const bool hb = has_bias != 0;
#define TG_SK_OK(MP, O) (hb ? splitk_cluster_ok<MP, O, true>(s, dev) : splitk_cluster_ok<MP, O, false>(s, dev))
#define TG_SK_OUT(MP) (out_dtype == TG_DT_F32 ? TG_SK_OK(MP, 0) : out_dtype == TG_DT_F16 ? TG_SK_OK(MP, 1) : TG_SK_OK(MP, 2))
  const bool cl = mpad == 16 ? TG_SK_OUT(16) : mpad == 32 ? TG_SK_OUT(32) : mpad == 64 ? TG_SK_OUT(64) : TG_SK_OUT(128);
#undef TG_SK_OUT
#undef TG_SK_OK
  *slices = s;
  *cluster = cl ? 1 : 0;
  return TG_OK;
}

}  // extern "C"

// ------------------------------------------------------------ few-row GEMV
namespace {

template <int MR, int OUT, bool HAS_BIAS>
int launch_gemv_t(const tg::GemvParams& p, int ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(tg::gemv::THREADS);
  cfg.dynamicSmemBytes = 0;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, tg::gemv_i8_kernel<MR, OUT, HAS_BIAS>, p) != cudaSuccess) return TG_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? TG_OK : TG_ERR_CUDA;
}

template <int MR>
int launch_gemv_m(const tg::GemvParams& p, int ctas, int out_dtype, bool hb, cudaStream_t st) {
  switch (out_dtype) {
    case TG_DT_F32: return hb ? launch_gemv_t<MR, 0, true>(p, ctas, st) : launch_gemv_t<MR, 0, false>(p, ctas, st);
    case TG_DT_F16: return hb ? launch_gemv_t<MR, 1, true>(p, ctas, st) : launch_gemv_t<MR, 1, false>(p, ctas, st);
    default: return hb ? launch_gemv_t<MR, 2, true>(p, ctas, st) : launch_gemv_t<MR, 2, false>(p, ctas, st);
  }
}

// K parts per group of 4 weight rows: the fewest of 1, 2, 4, 8 that put at
// least two CTAs (16 warps) per SM on the weight stream, each part keeping
// at least one 16-byte chunk per lane.
int gemv_parts(int64_t N, int64_t K, int sms) {
  using namespace tg::gemv;
  const int64_t groups = N / R;
  const int64_t nch = K / 16;
  int kp = 1;
  while (kp < WARPS && (groups * kp + WARPS - 1) / WARPS < 2 * int64_t(sms) && nch >= int64_t(64) * kp) kp *= 2;
  return kp;
}

// Weights up to this size have a quarter asked into L2 before the wait (the
// L2 holds 126 MB, so the quarter stays there until it is read); larger ones
// stream without the prefetch.
constexpr int64_t kGemvPrefetchMaxBytes = int64_t(256) << 20;

}  // namespace

extern "C" {

int tg_int8_gemv_dequant(const int8_t* xq, const float* xscale, const int8_t* wq, const float* wscale,
                         int64_t wscale_numel, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K,
                         int out_dtype, void* out, void* stream) {
  const int chk = check_gemm_args(xq, xscale, wq, wscale, wscale_numel, bias, bias_dtype, M, N, K, out_dtype, out);
  if (chk != TG_OK || M == 0) return chk;
  if (M > TG_GEMV_MAX_M) return TG_ERR_UNSUPPORTED;
  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;
  using namespace tg::gemv;
  const int kp = gemv_parts(N, K, info.sms_all);
  const int64_t nch = K / 16;
  const int64_t groups = N / R;  // N is a multiple of 4 (16-byte output rows)
  const int64_t per_cta = WARPS / kp;
  const int64_t ctas = (groups + per_cta - 1) / per_cta;
  if (ctas > 0x7fffffff) return TG_ERR_UNSUPPORTED;
  tg::GemvParams p;
  p.xq = xq;
  p.xscale = xscale;
  p.wq = wq;
  p.wscale = wscale;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.wscale_bcast = wscale_numel == 1 ? 1 : 0;
  p.M = int(M);
  p.N = int(N);
  p.K = int(K);
  p.kp = kp;
  p.part_chunks = int((nch + kp - 1) / kp);
  p.prefetch = N * K <= kGemvPrefetchMaxBytes ? 1 : 0;
  p.out = out;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool hb = bias != nullptr;
  switch (M) {
    case 1: return launch_gemv_m<1>(p, int(ctas), out_dtype, hb, st);
    case 2: return launch_gemv_m<2>(p, int(ctas), out_dtype, hb, st);
    default: return launch_gemv_m<4>(p, int(ctas), out_dtype, hb, st);
  }
}

int tg_int8_gemv_dequant_config(int64_t N, int64_t K, int* parts, int* ctas) {
  if (N < 1 || K < 16 || !parts || !ctas) return TG_ERR_INVALID_ARG;
  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;
  const int kp = gemv_parts(N, K, info.sms_all);
  const int64_t per_cta = tg::gemv::WARPS / kp;
  *parts = kp;
  *ctas = int((N / tg::gemv::R + per_cta - 1) / per_cta);
  return TG_OK;
}

}  // extern "C"

// ------------------------------------------------------------ no-allocation variant
// The split-K GEMM for callers that must not allocate device memory.  Its
// scratch is this file-scope array, sized for at most 2^20 accumulator
// elements (M x N, 4 MiB) and N <= 65536 (2 KiB of tile counters): 4 MiB + 2 KiB
// that every GPU which loads the library keeps until the process exits.
namespace {

constexpr int64_t kNoAllocMaxM = 64;
constexpr int64_t kNoAllocMaxN = 65536;
constexpr int64_t kNoAllocMaxAcc = int64_t(1) << 20;
constexpr size_t kNoAllocCountBytes = size_t(kNoAllocMaxN / tg::splitk::BNW) * 4;  // 256-byte multiple
constexpr size_t kNoAllocBytes = kNoAllocCountBytes + size_t(kNoAllocMaxAcc) * 4;

static __device__ __align__(256) unsigned char g_splitk_scratch[kNoAllocBytes];

// Device address of g_splitk_scratch on `dev` (the current device).  In host
// code the array's name only stands in for the symbol; its address on a
// device comes from the runtime, once per device.
bool noalloc_scratch(int dev, uint8_t** out) {
  static std::mutex mu;
  static void* addr[kMaxDevices];
  std::lock_guard<std::mutex> lock(mu);
  if (!addr[dev]) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_splitk_scratch) != cudaSuccess || p == nullptr) return false;
    addr[dev] = p;
  }
  *out = static_cast<uint8_t*>(addr[dev]);
  return true;
}

}  // namespace

extern "C" {

int tg_int8_gemm_dequant_splitk_noalloc(const int8_t* xq, const float* xscale, const int8_t* wq,
                                        const float* wscale, int64_t wscale_numel, const void* bias, int bias_dtype,
                                        int64_t M, int64_t N, int64_t K, int out_dtype, void* out, void* stream) {
  const int chk = check_gemm_args(xq, xscale, wq, wscale, wscale_numel, bias, bias_dtype, M, N, K, out_dtype, out);
  if (chk != TG_OK || M == 0) return chk;
  if (M > kNoAllocMaxM || N > kNoAllocMaxN || M * N > kNoAllocMaxAcc) return TG_ERR_UNSUPPORTED;
  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;
  uint8_t* scratch = nullptr;
  if (!noalloc_scratch(dev, &scratch)) return TG_ERR_CUDA;
  // Every call shares the array: when the sums go through it (K split more
  // than a cluster holds), zero the counters and this call's part of the
  // accumulator first, in stream order (a memset, not an allocation).  The
  // cluster form sums in shared memory and never touches the array.
  int slices = 0, cluster = 0;
  const int cfg = tg_int8_gemm_dequant_splitk_config(M, N, K, out_dtype, bias != nullptr, &slices, &cluster);
  if (cfg != TG_OK) return cfg;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!cluster && cudaMemsetAsync(scratch, 0, kNoAllocCountBytes + size_t(M) * size_t(N) * 4, st) != cudaSuccess)
    return TG_ERR_CUDA;
  return splitk_launch(xq, xscale, wq, wscale, wscale_numel, bias, bias_dtype, M, N, K, out_dtype, out,
                       reinterpret_cast<uint32_t*>(scratch), reinterpret_cast<int32_t*>(scratch + kNoAllocCountBytes),
                       stream);
}

}  // extern "C"

// ------------------------------------------------------------------ peer memory
// Buffers that other processes on this node (one per GPU) can map, and copies
// between mapped buffers on a stream.  cudaMemcpyAsync between this device and
// a peer's mapped memory runs on a copy engine over NVLink, using no SMs.
extern "C" {

size_t tg_peer_handle_bytes(void) { return sizeof(cudaIpcMemHandle_t); }

int tg_peer_alloc(size_t bytes, void** ptr, void* handle) {
  if (!ptr || !handle || bytes == 0) return TG_ERR_INVALID_ARG;
  *ptr = nullptr;
  void* p = nullptr;
  if (cudaMalloc(&p, bytes) != cudaSuccess) return TG_ERR_CUDA;
  if (cudaIpcGetMemHandle(static_cast<cudaIpcMemHandle_t*>(handle), p) != cudaSuccess) {
    cudaFree(p);
    return TG_ERR_CUDA;
  }
  *ptr = p;
  return TG_OK;
}

int tg_peer_free(void* ptr) {
  if (!ptr) return TG_ERR_INVALID_ARG;
  return cudaFree(ptr) == cudaSuccess ? TG_OK : TG_ERR_CUDA;
}

int tg_peer_open(const void* handle, void** ptr) {
  if (!handle || !ptr) return TG_ERR_INVALID_ARG;
  *ptr = nullptr;
  cudaIpcMemHandle_t h;
  memcpy(&h, handle, sizeof(h));
  void* p = nullptr;
  if (cudaIpcOpenMemHandle(&p, h, cudaIpcMemLazyEnablePeerAccess) != cudaSuccess) return TG_ERR_CUDA;
  *ptr = p;
  return TG_OK;
}

int tg_peer_close(void* ptr) {
  if (!ptr) return TG_ERR_INVALID_ARG;
  return cudaIpcCloseMemHandle(ptr) == cudaSuccess ? TG_OK : TG_ERR_CUDA;
}

int tg_copy_async(void* dst, const void* src, size_t bytes, void* stream) {
  if (bytes == 0) return TG_OK;
  if (!dst || !src) return TG_ERR_INVALID_ARG;
  return cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDeviceToDevice, static_cast<cudaStream_t>(stream)) ==
                 cudaSuccess
             ? TG_OK
             : TG_ERR_CUDA;
}

}  // extern "C"

// ------------------------------------------------------------ 4-bit weights, few rows
namespace {

bool is_dtype(int d) { return d == TG_DT_F32 || d == TG_DT_F16 || d == TG_DT_BF16; }

size_t dtype_bytes(int d) { return d == TG_DT_F32 ? 4 : 2; }

bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Whether two buffers share a byte.
bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
  const uint64_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x <= y ? y - x < a_bytes : x - y < b_bytes;
}

// A launch as the programmatic dependent of the kernel before it.
template <typename P>
int launch_dependent(void (*kern)(const P), const P& p, dim3 grid, int threads, uint32_t smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) return TG_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? TG_OK : TG_ERR_CUDA;
}

// 3-D tiled tensor map over rows of bytes (a multiple of 128) cut into 128-byte
// blocks: (byte of the block, row, block), 128-byte swizzle.  What lies behind the
// last block reads as zero.
bool make_tmap_blocks(CUtensorMap* m, const void* base, uint64_t row_bytes, uint64_t rows, uint32_t box_rows,
                      uint32_t box_blocks) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[3] = {128, rows, row_bytes / 128};
  cuuint64_t strides[2] = {row_bytes, 128};
  cuuint32_t box[3] = {128, box_rows, box_blocks};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Shared memory of a launch with `stages` ring slots: the ring (or the partial
// tiles) and the scales.
constexpr uint32_t gemv4_smem(int m, int mt, int rows, int kb, int groups, bool s4, int stages) {
  using namespace tg::gemv4;
  const uint32_t ring = uint32_t(stages) * (w_bytes(kb, rows) + x_bytes(kb, m));
  return std::max(ring + scale_bytes(rows, groups, s4), uint32_t(WK * 8 * mt * rows) * 4u) +
         1024u + uint32_t(8 * mt - m) * 128u;  // alignment, and the rows past m that are read and dropped
}

constexpr uint32_t kGemv4Static = 512;  // barriers and the abort flag, rounded up

// The form with 32 weight rows a CTA fits an SM at every documented size: two ring
// slots beside the scales of the longest rows in the finest groups (and the dropped
// rows of any m, which need less of the ring).  64 or 96 rows' scales may not.
constexpr bool gemv4_always_fits(int mt, int kb) {
  return gemv4_smem(8 * mt, mt, 32, kb, int(kRotQuantMaxK / 32), true, 2) + 8u * uint32_t(mt) * 128u + kGemv4Static +
             1024u <= kSmemPerSm;
}
static_assert(gemv4_always_fits(1, 1) && gemv4_always_fits(1, 2) && gemv4_always_fits(2, 2) &&
              gemv4_always_fits(4, 1) && gemv4_always_fits(8, 1), "a form for every size");

// K parts per group of four weight rows, as gemv_parts: the fewest that put two
// CTAs on every SM, each part keeping at least one 16-byte chunk a lane.
int gemv4_parts(int64_t N, int64_t K, int sms) {
  using namespace tg::gemv4one;
  const int64_t row_groups = (N + R - 1) / R, nch = K / 32;
  int kp = 1;
  while (kp < WARPS && (row_groups * kp + WARPS - 1) / WARPS < 2 * int64_t(sms) && nch >= int64_t(64) * kp) kp *= 2;
  return kp;
}

template <int U, int SV, bool S4>
int launch_gemv4_one_t(const tg::GemvI4OneParams& p, int64_t ctas, cudaStream_t st) {
  static_assert(kRotQuantMaxK <= 48 * 1024 - 256, "a row fits the shared memory of any launch");
  return launch_dependent(tg::gemv_i4_one_kernel<U, SV, S4>, p, dim3(unsigned(ctas)), tg::gemv4one::THREADS,
                          uint32_t(p.K), st);
}

// Two chunks of a row under way at once need registers that leave three CTAs per
// SM, and help where the launch is one wave of those and a lane has more than two
// chunks; otherwise four CTAs per SM with one chunk each carry more.  Measured (K x
// N, two / one, us): 13824 x 5120 8.6 / 9.6, 5120 x 5120 5.2 / 5.35; 5120 x 15360
// (480 CTAs) 11.4 / 8.0, 2048 x 1536 (one chunk a lane) 2.3 / 2.15.  Groups of 32
// with fp32 scales are 16 more registers a chunk and spilled: 12.7 / 11.2.
template <int SV, bool S4>
int launch_gemv4_one_sv(const tg::GemvI4OneParams& p, int sms, cudaStream_t st) {
  using namespace tg::gemv4one;
  const int64_t row_groups = (int64_t(p.N) + R - 1) / R, per_cta = WARPS / p.kp;
  const int64_t ctas = (row_groups + per_cta - 1) / per_cta;
  if constexpr (SV < 4 || !S4) {
    if (ctas <= 3 * int64_t(sms) && p.part_chunks > 64) return launch_gemv4_one_t<2, SV, S4>(p, ctas, st);
  }
  return launch_gemv4_one_t<1, SV, S4>(p, ctas, st);
}

int launch_gemv4_one(const tg::GemvI4OneParams& p, int sv, int sms, cudaStream_t st) {
  const bool s4 = p.wscale_dtype == TG_DT_F32;
  switch (sv) {
    case 4: return s4 ? launch_gemv4_one_sv<4, true>(p, sms, st) : launch_gemv4_one_sv<4, false>(p, sms, st);
    case 2: return s4 ? launch_gemv4_one_sv<2, true>(p, sms, st) : launch_gemv4_one_sv<2, false>(p, sms, st);
    default: return s4 ? launch_gemv4_one_sv<1, true>(p, sms, st) : launch_gemv4_one_sv<1, false>(p, sms, st);
  }
}

// want: CTAs per SM to make room for; as many ring slots as then fit (two at least).
template <int MT, int RT, int WR, int KB, int SV, bool S4>
int launch_gemv4_t(const int8_t* xq, const uint8_t* w4, tg::GemvI4Params p, int want, int dev, cudaStream_t st) {
  using namespace tg::gemv4;
  static uint32_t attr_done[kMaxDevices];
  auto kern = tg::gemv_i4_kernel<MT, RT, WR, KB, SV, S4>;
  if (!ensure_smem_attr(kern, dev, kSmemPerCtaMax - kGemv4Static, attr_done)) return TG_ERR_CUDA;
  constexpr int kRows = rows(RT, WR);
  const int steps = (p.K / 128 + KB * WK - 1) / (KB * WK);
  int stages = std::min(MAX_STAGES, std::max(2, steps));
  auto fits = [&](int s, int ctas) {
    return uint64_t(ctas) * (gemv4_smem(p.M, MT, kRows, KB, p.groups, S4, s) + kGemv4Static + 1024u) <= kSmemPerSm;
  };
  while (want > 1 && !fits(std::min(3, stages), want)) --want;
  while (stages > 2 && !fits(stages, want)) --stages;
  if (!fits(stages, 1)) return TG_ERR_UNSUPPORTED;
  p.stages = stages;
  p.prefetch = std::min(stages, steps);
  CUtensorMap tw, tx;
  if (!make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w4, uint64_t(p.K) / 2, uint64_t(p.N), uint64_t(p.K) / 2, 128,
                    uint32_t(kRows), CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_blocks(&tx, xq, uint64_t(p.K), uint64_t(p.M), uint32_t(p.M), uint32_t(KB * WK)))
    return TG_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(unsigned((int64_t(p.N) + kRows - 1) / kRows));
  cfg.blockDim = dim3(threads(WR));
  cfg.dynamicSmemBytes = gemv4_smem(p.M, MT, kRows, KB, p.groups, S4, stages);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, tw, tx, p) != cudaSuccess) return TG_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? TG_OK : TG_ERR_CUDA;
}

template <int MT, int RT, int WR, int KB>
int launch_gemv4(const int8_t* xq, const uint8_t* w4, const tg::GemvI4Params& p, int sv, int want, int dev,
                 cudaStream_t st) {
  const bool s4 = p.wscale_dtype == TG_DT_F32;
  switch (sv) {
    case 4: return s4 ? launch_gemv4_t<MT, RT, WR, KB, 4, true>(xq, w4, p, want, dev, st)
                      : launch_gemv4_t<MT, RT, WR, KB, 4, false>(xq, w4, p, want, dev, st);
    case 2: return s4 ? launch_gemv4_t<MT, RT, WR, KB, 2, true>(xq, w4, p, want, dev, st)
                      : launch_gemv4_t<MT, RT, WR, KB, 2, false>(xq, w4, p, want, dev, st);
    default: return s4 ? launch_gemv4_t<MT, RT, WR, KB, 1, true>(xq, w4, p, want, dev, st)
                       : launch_gemv4_t<MT, RT, WR, KB, 1, false>(xq, w4, p, want, dev, st);
  }
}

}  // namespace

extern "C" {

int tg_int4_gemv_dequant(const int8_t* xq, const float* xscale, const uint8_t* w4, const void* wscale,
                         int wscale_dtype, int group, const void* bias, int bias_dtype, int64_t M, int64_t N,
                         int64_t K, int out_dtype, void* out, void* stream) {
  if (M < 0 || N <= 0 || K <= 0) return TG_ERR_INVALID_ARG;
  if (!is_dtype(out_dtype) || !is_dtype(wscale_dtype) || (bias && !is_dtype(bias_dtype))) return TG_ERR_INVALID_ARG;
  if (group != 32 && group != 64 && group != 128 && group != 256) return TG_ERR_UNSUPPORTED;
  if (M > TG_INT4_MAX_M || K % 128 != 0 || K % group != 0) return TG_ERR_UNSUPPORTED;
  if (N > kMaxTiledRows || K > kRotQuantMaxK) return TG_ERR_UNSUPPORTED;
  if (M == 0) return TG_OK;
  if (!xq || !xscale || !w4 || !wscale || !out) return TG_ERR_INVALID_ARG;
  if (!aligned16(xq) || !aligned16(w4) || !aligned16(wscale)) return TG_ERR_MISALIGNED;
  if (!aligned_to(xscale, 4) || !aligned_to(out, dtype_bytes(out_dtype)) ||
      (bias && !aligned_to(bias, dtype_bytes(bias_dtype))))
    return TG_ERR_MISALIGNED;
  tg::GemvI4Params p;
  p.xscale = xscale;
  p.wscale = wscale;
  p.bias = bias;
  p.wscale_dtype = wscale_dtype;
  p.bias_dtype = bias_dtype;
  p.out_dtype = out_dtype;
  p.groups = int(K / group);
  p.scale_shift = group == 256 ? 1 : 0;
  p.M = int(M);
  p.N = int(N);
  p.K = int(K);
  p.out = out;
  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sv = group == 32 ? 4 : (group == 64 ? 2 : 1);
  if (M == 1) {
    tg::GemvI4OneParams q;
    q.xq = xq;
    q.xscale = xscale;
    q.w4 = w4;
    q.wscale = wscale;
    q.bias = bias;
    q.wscale_dtype = wscale_dtype;
    q.bias_dtype = bias_dtype;
    q.out_dtype = out_dtype;
    q.groups = p.groups;
    q.scale_shift = p.scale_shift;
    q.N = p.N;
    q.K = p.K;
    q.kp = gemv4_parts(N, K, info.sms_all);
    q.part_chunks = int((K / 32 + q.kp - 1) / q.kp);
    q.prefetch = N * K / 2 <= kGemvPrefetchMaxBytes ? 1 : 0;
    q.out = out;
    return launch_gemv4_one(q, sv, info.sms_all, st);
  }
  // 16-row tiles an SM gets.  Where they are few, a CTA's steps are what takes the
  // time, and two blocks a step halve them; where they are many, one block a step
  // leaves room for the rings of more CTAs.  Measured (K x N, two blocks / one, us):
  // 8 rows, 5120 x 5120 5.3 / 6.5, 13824 x 5120 11.3 / 12.5, 5120 x 15360 12.6 / 8.8;
  // 16 rows, 5120 x 5120 6.2 / 8.7, 13824 x 5120 12.0 / 18.5, 5120 x 15360 13.5 / 10.4.
  const int64_t tiles = (N + 15) / 16, sms = info.sms_all;
  const int want = int(std::max<int64_t>(1, std::min<int64_t>(8, (tiles + sms - 1) / sms)));
  const bool few = want <= 3;
  if (M <= 8) return few ? launch_gemv4<1, 2, 1, 2>(xq, w4, p, sv, (want + 1) / 2, dev, st)
                         : launch_gemv4<1, 2, 1, 1>(xq, w4, p, sv, (want + 1) / 2, dev, st);
  if (M <= 16) {
    const int rc = few ? launch_gemv4<2, 1, 2, 2>(xq, w4, p, sv, (want + 1) / 2, dev, st)
                       : launch_gemv4<2, 2, 2, 1>(xq, w4, p, sv, 2, dev, st);
    // Very long rows of fine fp32 scales leave no room for 64 rows of them.
    return rc == TG_ERR_UNSUPPORTED ? launch_gemv4<2, 1, 2, 2>(xq, w4, p, sv, 1, dev, st) : rc;
  }
  if (M <= 32) return launch_gemv4<4, 2, 1, 1>(xq, w4, p, sv, std::min(2, (want + 1) / 2), dev, st);
  // 64 or 96 rows a CTA, one CTA per SM: whichever takes the fewer rows of them in all.
  const int64_t t32 = (N + 31) / 32;
  const int64_t cost2 = (t32 + 2 * sms - 1) / (2 * sms) * 2, cost3 = (t32 + 3 * sms - 1) / (3 * sms) * 3;
  const int rc = cost3 < cost2 ? launch_gemv4<8, 2, 3, 1>(xq, w4, p, sv, 1, dev, st)
                               : launch_gemv4<8, 2, 2, 1>(xq, w4, p, sv, 1, dev, st);
  // As above.
  return rc == TG_ERR_UNSUPPORTED ? launch_gemv4<8, 2, 1, 1>(xq, w4, p, sv, 2, dev, st) : rc;
}

}  // extern "C"

// ------------------------------------------------------------ routed experts
namespace {

// Most (token, expert) slots: 32-bit slot numbers, with room for a grid's stride.
constexpr int64_t kMaxRouteSlots = int64_t(1) << 30;

// Tokens per CTA of the router's two-kernel form, a multiple of 32: a warp a
// token and 32 warps, more where that would make more than 256 CTAs, whose
// counts every CTA of the second kernel reads.
int route_per_block(int64_t T) {
  const int64_t per = (T + 256 * 32 - 1) / (256 * 32) * 32;
  return int(per);
}

template <int K>
int launch_route_rows(const tg::RouteParams& p, int dev, cudaStream_t st) {
  using namespace tg::route;
  static uint32_t attr_done[kMaxDevices];
  auto kern = tg::route_rows_kernel<K>;
  if (!ensure_smem_attr(kern, dev, uint32_t(ROW_THREADS * (ROW_MAX_E | 1) * 4), attr_done)) return TG_ERR_CUDA;
  return launch_dependent(kern, p, dim3(unsigned(p.blocks)), ROW_THREADS, uint32_t(ROW_THREADS * (p.E | 1) * 4), st);
}

template <int EPL>
int launch_route(const tg::RouteParams& p, int dev, cudaStream_t st) {
  using namespace tg::route;
  const dim3 grid{unsigned(p.blocks)};
  if (p.T <= SINGLE) return launch_dependent(tg::route_topk_kernel<EPL, false>, p, grid, threads(EPL), 0, st);
  // A thread per token where there are tokens for every SM and a row is short.
  const bool rows = p.T >= ROW_MIN_T && p.E <= ROW_MAX_E && p.top_k <= ROW_MAX_K;
  const int rc = !rows ? launch_dependent(tg::route_topk_kernel<EPL, true>, p, grid, threads(EPL), 0, st)
                 : p.top_k <= 2 ? launch_route_rows<2>(p, dev, st)
                 : p.top_k <= 4 ? launch_route_rows<4>(p, dev, st)
                                : launch_route_rows<8>(p, dev, st);
  if (rc != TG_OK) return rc;
  return launch_dependent(tg::route_place_kernel, p, grid, THREADS, 0, st);
}

template <int DT>
int launch_combine(tg::CombineParams p, cudaStream_t st) {
  constexpr int ESZ = DT == TG_DT_F32 ? 4 : 2;
  constexpr int VEC = 16 / ESZ;
  const bool vec = p.N % VEC == 0 && aligned16(p.y) && aligned16(p.residual) && aligned16(p.out);
  p.per_row = uint32_t(vec ? p.N / VEC : p.N);
  const int64_t ctas = (p.T * int64_t(p.per_row) + 255) / 256;
  if (ctas > 0x7fffffff) return TG_ERR_UNSUPPORTED;
  const dim3 grid{unsigned(ctas)};
  return vec ? launch_dependent(tg::combine_kernel<DT, VEC>, p, grid, 256, 0, st)
             : launch_dependent(tg::combine_kernel<DT, 1>, p, grid, 256, 0, st);
}

}  // namespace

extern "C" {

size_t tg_route_experts_workspace(int64_t T, int64_t E) {
  if (T <= tg::route::SINGLE || T > kMaxRouteSlots || E <= 0 || E > tg::route::MAX_E) return 0;
  const int per = route_per_block(T);
  return size_t((T + per - 1) / per) * size_t(E) * 4;
}

int tg_route_experts(const void* logits, int dtype, int64_t T, int64_t E, int top_k, int renormalize,
                     float* weights, int32_t* ids, int32_t* offsets, int32_t* rows, int32_t* place, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (T < 0 || E <= 0 || top_k <= 0 || top_k > E || !is_dtype(dtype)) return TG_ERR_INVALID_ARG;
  if (E > tg::route::MAX_E || top_k > tg::route::MAX_K) return TG_ERR_UNSUPPORTED;
  if (T > kMaxRouteSlots / top_k) return TG_ERR_UNSUPPORTED;
  if (!offsets || !aligned_to(offsets, 4)) return offsets ? TG_ERR_MISALIGNED : TG_ERR_INVALID_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0)
    return cudaMemsetAsync(offsets, 0, size_t(E + 1) * 4, st) == cudaSuccess ? TG_OK : TG_ERR_CUDA;
  const size_t need = tg_route_experts_workspace(T, E);
  if (!logits || !weights || !ids || !rows || !place || (need > 0 && !workspace)) return TG_ERR_INVALID_ARG;
  if (!aligned_to(logits, dtype_bytes(dtype)) || !aligned_to(weights, 4) || !aligned_to(ids, 4) ||
      !aligned_to(rows, 4) || !aligned_to(place, 4) || !aligned_to(workspace, 4))
    return TG_ERR_MISALIGNED;
  if (workspace_bytes < need) return TG_ERR_INVALID_ARG;
  tg::RouteParams p;
  p.logits = logits;
  p.dtype = dtype;
  p.T = int(T);
  p.E = int(E);
  p.top_k = top_k;
  p.renormalize = renormalize != 0;
  p.per_block = T <= tg::route::SINGLE ? tg::route::SINGLE : route_per_block(T);
  p.blocks = int((T + p.per_block - 1) / p.per_block);
  p.weights = weights;
  p.ids = ids;
  p.offsets = offsets;
  p.rows = rows;
  p.place = place;
  p.counts = static_cast<int32_t*>(workspace);
  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;
  if (E <= 32) return launch_route<1>(p, dev, st);
  if (E <= 64) return launch_route<2>(p, dev, st);
  if (E <= 128) return launch_route<4>(p, dev, st);
  if (E <= 256) return launch_route<8>(p, dev, st);
  if (E <= 512) return launch_route<16>(p, dev, st);
  return launch_route<32>(p, dev, st);
}

int tg_combine_experts(const void* y, int dtype, int64_t R, const int32_t* place, const float* weights, int64_t T,
                       int top_k, const void* residual, int64_t N, void* out, void* stream) {
  if (T < 0 || R < 0 || N <= 0 || top_k <= 0 || !is_dtype(dtype)) return TG_ERR_INVALID_ARG;
  if (top_k > tg::route::MAX_K || T >= (int64_t(1) << 31) || N >= (int64_t(1) << 31) || R >= (int64_t(1) << 31))
    return TG_ERR_UNSUPPORTED;
  if (T == 0) return TG_OK;
  if ((!y && R > 0) || !place || !weights || !out) return TG_ERR_INVALID_ARG;
  const size_t esz = dtype_bytes(dtype);
  if (!aligned_to(y, esz) || !aligned_to(out, esz) || !aligned_to(residual, esz) || !aligned_to(place, 4) ||
      !aligned_to(weights, 4))
    return TG_ERR_MISALIGNED;
  // A row of out is written while others are still to be read.
  const uint64_t out_bytes = uint64_t(T) * uint64_t(N) * esz, slot_bytes = uint64_t(T) * uint64_t(top_k) * 4u;
  if ((R > 0 && overlap(out, out_bytes, y, uint64_t(R) * uint64_t(N) * esz)) ||
      (residual && residual != out && overlap(out, out_bytes, residual, out_bytes)) ||
      overlap(out, out_bytes, place, slot_bytes) || overlap(out, out_bytes, weights, slot_bytes))
    return TG_ERR_INVALID_ARG;
  tg::CombineParams p;
  p.y = y;
  p.place = place;
  p.weights = weights;
  p.residual = residual;
  p.out = out;
  p.R = R;
  p.T = T;
  p.N = N;
  p.top_k = top_k;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TG_DT_F32: return launch_combine<TG_DT_F32>(p, st);
    case TG_DT_F16: return launch_combine<TG_DT_F16>(p, st);
    default: return launch_combine<TG_DT_BF16>(p, st);
  }
}

}  // extern "C"

namespace {

// A pass of its own gathers the rows where an expert has 256 of them or more and
// the products are 1.25e11 multiply-adds or more, about 100 us: measured (in the
// kernel / in a pass, us) 455 / 420 at 8192 x 13824 x 5120 over 8 experts, 295 / 284
// and 178 / 171 at 32768 and 16384 x 4096 x 2048 over 64; below, the pass costs
// what it saves: 63 / 65 at 2048 x 5120 x 5120 over 8, 17.6 / 18.9 at 4096 x 1024 x
// 1024 over 8, 124 / 123 at 128 rows an expert.
constexpr int64_t kGatherPassMinRows = 256;
constexpr double kGatherPassMinWork = 1.25e11;

// Sizes whose row numbers have 32 bits (E * N within 64 bits).
bool grouped_in_range(int64_t R, int64_t E, int64_t N, int64_t K) {
  return E <= tg::route::MAX_E && R <= kMaxTiledRows && K < (int64_t(1) << 31) && N <= kMaxTiledRows &&
         E * N <= kMaxTiledRows;
}

// Rows an expert has on average, if every expert has some.
int64_t grouped_avg(int64_t R, int64_t E) { return R / std::max<int64_t>(1, std::min(E, R)); }

// The output's tensor map has to match the kernel's chunk (32 rows x 32 channels).
template <int TN, int OUT, bool GATHER>
int launch_grouped_t(const CUtensorMap& tw, const CUtensorMap& tx, const CUtensorMap& to, tg::GroupedParams p, int dev,
                     int sms, cudaStream_t st) {
  static uint32_t attr_done[kMaxDevices];
  using namespace tg::grouped;
  constexpr uint32_t smem = smem_bytes(TN);
  auto kern = tg::gemm_i8_grouped_kernel<TN, OUT, GATHER>;
  if (!ensure_smem_attr(kern, dev, smem, attr_done)) return TG_ERR_CUDA;
  constexpr int64_t kKBlock = int64_t(BK) * KS;
  p.n_tiles = int((int64_t(p.N) + TILE_N - 1) / TILE_N);
  p.k_blocks = int((int64_t(p.K) + kKBlock - 1) / kKBlock);
  // No more tiles than the full ones and a part-filled one for each expert.
  const int64_t most = (int64_t(p.R) / TN + std::min<int64_t>(p.E, p.R)) * p.n_tiles;
  // The pair GEMM's clusters of two take as much shared memory: as many fit.
  const int units = int(std::min<int64_t>(std::max(gemm_units(dev, sms, true), 1), most));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(unsigned(2 * units));
  cfg.blockDim = dim3(threads(GATHER));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, tw, tx, to, p) != cudaSuccess) return TG_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? TG_OK : TG_ERR_CUDA;
}

template <int TN>
int launch_grouped_tn(const int8_t* xq, const CUtensorMap& tw, const CUtensorMap& to, const tg::GroupedParams& p,
                      int out_dtype, int dev, int sms, cudaStream_t st) {
  const bool g = p.rows != nullptr;
  CUtensorMap tx;
  if (!make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, xq, uint64_t(p.K), uint64_t(p.M), uint64_t(p.K),
                    tg::grouped::BK, g ? 1u : uint32_t(tg::grouped::XBOX), CU_TENSOR_MAP_SWIZZLE_128B))
    return TG_ERR_CUDA;
  switch (out_dtype) {
    case TG_DT_F32: return g ? launch_grouped_t<TN, 0, true>(tw, tx, to, p, dev, sms, st)
                             : launch_grouped_t<TN, 0, false>(tw, tx, to, p, dev, sms, st);
    case TG_DT_F16: return g ? launch_grouped_t<TN, 1, true>(tw, tx, to, p, dev, sms, st)
                             : launch_grouped_t<TN, 1, false>(tw, tx, to, p, dev, sms, st);
    default: return g ? launch_grouped_t<TN, 2, true>(tw, tx, to, p, dev, sms, st)
                      : launch_grouped_t<TN, 2, false>(tw, tx, to, p, dev, sms, st);
  }
}

}  // namespace

extern "C" {

size_t tg_int8_grouped_gemm_dequant_workspace(int64_t R, int64_t E, int64_t N, int64_t K) {
  if (R <= 0 || E <= 0 || N <= 0 || K <= 0 || !grouped_in_range(R, E, N, K) || grouped_avg(R, E) < kGatherPassMinRows ||
      double(R) * double(N) * double(K) < kGatherPassMinWork)
    return 0;
  return size_t(R) * size_t(K + 4);
}

int tg_int8_grouped_gemm_dequant(const int8_t* xq, const float* xscale, int64_t M, const int8_t* wq,
                                 const float* wscale, int64_t wscale_numel, const void* bias, int bias_dtype,
                                 const int32_t* rows, const int32_t* offsets, int64_t R, int64_t E, int64_t N,
                                 int64_t K, int out_dtype, void* out, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (M < 0 || R < 0 || E <= 0 || N <= 0 || K <= 0) return TG_ERR_INVALID_ARG;
  if (!is_dtype(out_dtype) || (bias && !is_dtype(bias_dtype))) return TG_ERR_INVALID_ARG;
  if ((!rows && R > M) || (R > 0 && M == 0)) return TG_ERR_INVALID_ARG;
  if (M > kMaxTiledRows || !grouped_in_range(R, E, N, K)) return TG_ERR_UNSUPPORTED;
  if (wscale_numel != 1 && wscale_numel != E && wscale_numel != E * N) return TG_ERR_INVALID_ARG;
  if (K % 16 != 0 || (N * int64_t(dtype_bytes(out_dtype))) % 16 != 0) return TG_ERR_UNSUPPORTED;
  if (R == 0) return TG_OK;
  if (!xq || !xscale || !wq || !wscale || !offsets || !out) return TG_ERR_INVALID_ARG;
  if (!aligned16(xq) || !aligned16(wq) || !aligned16(out)) return TG_ERR_MISALIGNED;
  if (!aligned_to(xscale, 4) || !aligned_to(wscale, 4) || !aligned_to(rows, 4) || !aligned_to(offsets, 4) ||
      (bias && !aligned_to(bias, dtype_bytes(bias_dtype))))
    return TG_ERR_MISALIGNED;
  int dev;
  DeviceInfo info;
  if (!current_device(&dev, &info)) return TG_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t need = rows ? tg_int8_grouped_gemm_dequant_workspace(R, E, N, K) : 0;
  if (need > 0 && workspace && workspace_bytes >= need) {
    if (!aligned16(workspace)) return TG_ERR_MISALIGNED;
    tg::GatherRowsParams g;
    g.xq = xq;
    g.xscale = xscale;
    g.rows = rows;
    g.q = static_cast<int8_t*>(workspace);
    g.scale = reinterpret_cast<float*>(g.q + R * K);
    g.M = int(M);
    g.R = int(R);
    g.K = int(K);
    const int rc = launch_dependent(tg::gather_rows_kernel, g, dim3(unsigned((R + 7) / 8)), 256, 0, st);
    if (rc != TG_OK) return rc;
    xq = g.q;
    xscale = g.scale;
    rows = nullptr;
    M = R;
  }
  using namespace tg::grouped;
  CUtensorMap tw, to;
  if (!make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, wq, uint64_t(K), uint64_t(E * N), uint64_t(K), BK, BNW,
                    CU_TENSOR_MAP_SWIZZLE_128B))
    return TG_ERR_CUDA;
  const CUtensorMapDataType odt = out_dtype == TG_DT_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : out_dtype == TG_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (!make_tmap_2d(&to, odt, out, uint64_t(N), uint64_t(R), uint64_t(N) * dtype_bytes(out_dtype), 32, 32,
                    CU_TENSOR_MAP_SWIZZLE_NONE))
    return TG_ERR_CUDA;
  tg::GroupedParams p;
  p.xscale = xscale;
  p.wscale = wscale;
  p.bias = bias;
  p.rows = rows;
  p.offsets = offsets;
  p.bias_dtype = bias_dtype;
  p.wscale_mode = wscale_numel == 1 ? 0 : (wscale_numel == E * N ? 2 : 1);
  p.M = int(M);
  p.R = int(R);
  p.E = int(E);
  p.N = int(N);
  p.K = int(K);
  p.out = out;
  const int64_t avg = grouped_avg(R, E);
  if (avg <= 24) return launch_grouped_tn<64>(xq, tw, to, p, out_dtype, dev, info.sms, st);
  if (avg <= 64) return launch_grouped_tn<128>(xq, tw, to, p, out_dtype, dev, info.sms, st);
  return launch_grouped_tn<256>(xq, tw, to, p, out_dtype, dev, info.sms, st);
}

}  // extern "C"
