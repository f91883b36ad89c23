// C ABI of the dense projection, the expert router and the mixture-of-experts layer
// (declarations in include/ffn_b200.h).
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <mutex>
#include <new>

#include "../../include/ffn_b200.h"
#include "gemm_kernel.cuh"
#include "pack_kernel.cuh"
#include "router_kernel.cuh"
#include "stream_kernel.cuh"

namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t pitch_of(int64_t cols) { return (cols + 7) / 8 * 8; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool bad_rows(const void* p, int64_t ld, int64_t cols) { return !aligned16(p) || ld % 8 != 0 || ld < cols; }
constexpr int64_t kMaxDim = 65535;
constexpr uint64_t kMaxWaitNs = 3600ull * 1000000000ull;  // an hour: a negative number taken for an unsigned one is refused

// Makes `device` current for one call and puts the caller's device back.
struct DeviceScope {
  int before = -1;
  bool ok = true;
  explicit DeviceScope(int device) {
    int cur = 0;
    ok = cudaGetDevice(&cur) == cudaSuccess;
    if (ok && cur != device) {
      ok = cudaSetDevice(device) == cudaSuccess;
      if (ok) before = cur;
    }
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
};

int device_sms(int given, int* sms) {
  *sms = given;
  if (given > 0) return FFN_B200_OK;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return FFN_B200_ERR_DEVICE;
  }
  int maj = 0, min = 0;
  return ffn_b200_device_info(dev, sms, &maj, &min);
}

int check_device(int device) {
  int sms = 0, maj = 0, min = 0;
  const int rc = ffn_b200_device_info(device, &sms, &maj, &min);
  if (rc) return rc;
  return maj == 10 && min == 0 ? FFN_B200_OK : FFN_B200_ERR_DEVICE;
}

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

int get_encode() {
  static std::once_flag once;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult st;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &st) == cudaSuccess &&
        st == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  return g_encode ? FFN_B200_OK : FFN_B200_ERR_CUDA;
}

// 128B-swizzled tensor map of 16-bit elements; `strides` in elements, one per dimension but the first.
int encode(CUtensorMap* tm, const void* base, int dtype, int rank, const int64_t* dims, const int64_t* strides,
           const uint32_t* box) {
  cuuint64_t gdim[4], gstr[3];
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) gdim[i] = static_cast<cuuint64_t>(dims[i]);
  for (int i = 0; i + 1 < rank; ++i) gstr[i] = static_cast<cuuint64_t>(strides[i]) * 2;
  const CUresult r = g_encode(tm, dtype == FFN_B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                              static_cast<cuuint32_t>(rank), const_cast<void*>(base), gdim, gstr, box, ones,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FFN_B200_OK : FFN_B200_ERR_CUDA;
}
// Weights [experts][halves][rows][cols] in boxes of `box_rows` rows of every half.
int encode_weights(CUtensorMap* tm, const void* base, int dtype, int64_t cols, int64_t rows, int64_t halves,
                   int64_t experts, int64_t ld, int64_t stride, int box_rows) {
  const int64_t dims[4] = {cols, rows, halves, experts};
  const int64_t strides[3] = {ld, rows * ld, stride};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_rows), static_cast<uint32_t>(halves), 1};
  return encode(tm, base, dtype, 4, dims, strides, box);
}
// Rows [rows][cols] in boxes of `box_rows` (1: gathered loads).
int encode_rows(CUtensorMap* tm, const void* base, int dtype, int64_t cols, int64_t rows, int64_t ld, int box_rows) {
  const int64_t dims[2] = {cols, rows};
  const uint32_t box[2] = {64, static_cast<uint32_t>(box_rows)};
  return encode(tm, base, dtype, 2, dims, &ld, box);
}

constexpr int kMaxSmem = 232448;
// Tokens up to which the experts' first product gathers its token rows itself (a gather of four rows
// takes the TMA about 200 clocks, so a step's weights hide three); above, they are copied into
// the pairs' order first.  Gathered / copied, us: 16 tokens of K 2048, 6 of 64 experts 116 / 121, of K 4096, 4 of
// 32 214 / 227; 20 tokens 135 / 125 and 249 / 248; 32 tokens 140 / 141 and 261 / 259.
constexpr int64_t kMoeGather = 16;

// Token columns of a tile: a multiple of the MMA's 16, at most 128.
int stream_chunk(int64_t tokens) { return static_cast<int>(std::min<int64_t>(128, cdiv(tokens, 16) * 16)); }
// The ring beside `list_bytes` of lists: K steps per slot (of `slab` weight bytes and `chunk` token
// rows each), slots, and the dynamic shared memory they add up to.  Up to 60 KB and 8 steps: longer
// stretches of each weight row at a time and fewer waits, against fewer slots (1x4096x4096: 15.9 us
// with 2 steps, 11.3 with 4, 9.9 with 8, 10.2 with 12; 16 tokens, 4 of 32 experts: 229 us with 2,
// 226 with 3, 225 with 4).
// (The MMA reads 128 rows from a slab's start.)
struct StreamRing {
  int blocks, stages;
  int64_t smem;
  StreamRing(int slab, int chunk, int list_bytes) {
    const int step = slab + chunk * 128;
    blocks = std::max(1, std::min(8, 61440 / step));
    const int fixed = 1024 + ffnb200::kStreamBarBytes + list_bytes +
                      std::max(0, ffnb200::kABytes - slab - blocks * chunk * 128);
    stages = std::min(ffnb200::kStreamMaxStages, (kMaxSmem - fixed) / (blocks * step));
    smem = static_cast<int64_t>(stages) * blocks * step + fixed;
  }
};

using GemmFn = void (*)(const ffnb200::GemmParams);
// A tile family of the dense projection.
struct GemmTile {
  int rows, cols, box_rows, smem, stages;  // box_rows: rows of a weight load
  GemmFn fn[2];                            // fp16, bf16
};
template <int BN, bool PAIR>
GemmTile gemm_tile() {
  using LY = ffnb200::GemmLayout<BN, PAIR>;
  return {PAIR ? 256 : 128, BN, LY::kBRows, LY::kSmem, LY::kStages,
          {ffnb200::gemm_kernel<false, BN, PAIR>, ffnb200::gemm_kernel<true, BN, PAIR>}};
}
GemmTile gemm_tile(int tile) {
  if (tile == FFN_B200_LINEAR_PAIR256) return gemm_tile<256, true>();
  return tile == FFN_B200_LINEAR_CTA128 ? gemm_tile<128, false>() : gemm_tile<64, false>();
}

using StreamFn = void (*)(const ffnb200::StreamParams);

int launch_stream(StreamFn fn, const ffnb200::StreamParams& params, int grid, int64_t smem, bool cooperative,
                  void* stream) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(ffnb200::kStreamThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  if (cooperative) {  // CTAs wait on one another: all resident at once
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
  } else {  // no waits between CTAs: set-up overlaps the previous kernel's end
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, fn, params) == cudaSuccess) return FFN_B200_OK;
  cudaGetLastError();
  return FFN_B200_ERR_CUDA;
}

using RouteFn = void (*)(const ffnb200::RouteParams);

ffnb200::RouteParams route_params(const ffn_b200_router_problem& pr, const void* w, int64_t ldw, const float* cbias,
                                  double* logits, int parts, uint32_t* counters) {
  ffnb200::RouteParams P;
  std::memset(&P, 0, sizeof(P));
  P.w = w;
  P.ldw = ldw;
  P.choice_bias = cbias;
  P.logits = logits;
  P.sums = reinterpret_cast<float*>(logits + parts * pr.m * pr.experts);
  P.parts = parts;
  P.counters = counters;
  P.M = static_cast<int>(pr.m);
  P.K = static_cast<int>(pr.k);
  P.E = pr.experts;
  P.top = pr.top_k;
  P.weight_f32 = pr.weight_f32;
  P.sigmoid = pr.sigmoid;
  P.renormalize = pr.renormalize;
  P.scale = pr.scale;
  return P;
}

struct RouteFns {
  RouteFn few, few32, many32, logits, choose;
};
template <bool BF16, int PER>
constexpr RouteFns route_fns() {
  return {ffnb200::route_kernel<BF16, false, 1, 1, PER>, ffnb200::route_kernel<BF16, true, 1, 1, PER>,
          ffnb200::route_kernel<BF16, true, 2, 4, PER>, ffnb200::route_logits_kernel<BF16>,
          ffnb200::route_choose_kernel<BF16, PER>};
}
const RouteFns kRouteFns[3][2] = {{route_fns<false, 2>(), route_fns<true, 2>()},
                                  {route_fns<false, 8>(), route_fns<true, 8>()},
                                  {route_fns<false, 16>(), route_fns<true, 16>()}};

// Tokens from which the router runs as two kernels (16-bit weights), and the parts of K of its first.  One / two
// kernels, us: 64 experts of K 2048 at 64 tokens 16.1 / 15.1, 128 18.5 / 17.9, 256 18.9 / 17.9; 256 experts of K 4096
// 64: 37 / 24, 128: 37 / 31, 512: 78 / 34; 8 experts of K 1000 128: 9.9 / 14.2, 512: 9.9 / 15.9.  (So many
// experts would gain from two kernels sooner, and a few lose by them.)
constexpr int64_t kRouteMany = 128;
bool route_many(const ffn_b200_router_problem& p) { return p.m >= kRouteMany && !p.weight_f32; }
int route_parts(const ffn_b200_router_problem& p) {
  if (!route_many(p)) return 1;
  const int64_t tiles = cdiv(p.m, ffnb200::kLogitTile) * cdiv(p.experts, ffnb200::kLogitTile);
  const int64_t steps = cdiv(p.k, ffnb200::kRouteStep);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({8, 296 / tiles, steps / 8})));  // two CTAs per SM
}

int launch_route(RouteFn fn, const ffnb200::RouteParams& P, dim3 grid, int smem, void* stream) {
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return FFN_B200_ERR_CUDA;
  }
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(ffnb200::kRouteThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, fn, P) == cudaSuccess) return FFN_B200_OK;
  cudaGetLastError();
  return FFN_B200_ERR_CUDA;
}
// One kernel of 16 mt x 8 nt tiles; shared memory: the warps' parts of K, then logits and scores.
int launch_route(RouteFn fn, const ffnb200::RouteParams& P, int mt, int nt, void* stream) {
  const dim3 grid(static_cast<unsigned>(cdiv(P.E, 8 * nt) * cdiv(P.M, 16 * mt)), 1, 1);
  return launch_route(fn, P, grid, std::max(ffnb200::kRouteWarps * 128 * mt * nt * 12, ffnb200::route_space<ffnb200::kRouteWarps>(P.E)),
                      stream);
}

int set_smem(const void* fn, int64_t smem) {
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) == cudaSuccess)
    return FFN_B200_OK;
  cudaGetLastError();
  return FFN_B200_ERR_CUDA;
}

int check_linear(const ffn_b200_linear_problem& p) {
  if (p.m <= 0 || p.k <= 0 || p.n <= 0 || p.k > kMaxDim || p.n > kMaxDim || p.m > (int64_t(1) << 31) - 16)
    return FFN_B200_ERR_INVALID;
  if (p.dtype != FFN_B200_F16 && p.dtype != FFN_B200_BF16) return FFN_B200_ERR_INVALID;
  if (p.activation < 0 || p.activation > FFN_B200_IDENTITY || p.activation == FFN_B200_SWIGLU)
    return FFN_B200_ERR_INVALID;
  if (p.block_num < 0 || p.reserved || p.tile < 0 || p.tile > FFN_B200_LINEAR_CTA64) return FFN_B200_ERR_INVALID;
  return FFN_B200_OK;
}

int check_router(const ffn_b200_router_problem& p) {
  if (p.m <= 0 || p.k <= 0 || p.k > kMaxDim || p.m > (int64_t(1) << 31) - 16) return FFN_B200_ERR_INVALID;
  if (p.experts < 1 || p.experts > FFN_B200_MAX_EXPERTS || p.top_k < 1 || p.top_k > FFN_B200_MAX_TOP_K ||
      p.top_k > p.experts)
    return FFN_B200_ERR_INVALID;
  if (p.dtype != FFN_B200_F16 && p.dtype != FFN_B200_BF16) return FFN_B200_ERR_INVALID;
  if ((p.weight_f32 | p.sigmoid | p.renormalize) & ~1 || p.reserved) return FFN_B200_ERR_INVALID;
  return FFN_B200_OK;
}

int check_moe(const ffn_b200_moe_problem& p) {
  if (p.m <= 0 || p.k <= 0 || p.h <= 0 || p.n <= 0 || p.k > kMaxDim || p.h > kMaxDim || p.n > kMaxDim)
    return FFN_B200_ERR_INVALID;
  if (p.m > FFN_B200_MOE_MAX_TOKENS) return FFN_B200_ERR_TOO_LARGE;
  if (p.experts < 1 || p.experts > FFN_B200_MAX_EXPERTS || p.top_k < 1 || p.top_k > FFN_B200_MAX_TOP_K ||
      p.top_k > p.experts)
    return FFN_B200_ERR_INVALID;
  if (p.dtype != FFN_B200_F16 && p.dtype != FFN_B200_BF16) return FFN_B200_ERR_INVALID;
  if (p.activation < 0 || p.activation > FFN_B200_SWIGLU || p.block_num < 0) return FFN_B200_ERR_INVALID;
  return FFN_B200_OK;
}

}  // namespace

struct ffn_b200_linear {
  ffn_b200_linear_problem prob;
  ffn_b200_linear_plan plan;
  int device;
  const void* w;
  int64_t ldw;
  const void* bias;
  int32_t* status;
  ffnb200::StreamParams params;  // tile FFN_B200_LINEAR_STREAM
  StreamFn fn;
  ffnb200::GemmParams gemm;      // the other tiles
};

struct ffn_b200_moe {
  ffn_b200_moe_problem prob;
  ffn_b200_moe_plan plan;
  ffn_b200_moe_buffers buf;
  int device;
  ffnb200::StreamParams params;
  StreamFn fn;
  uint32_t* route_counters;
};

// ---- dense projection ----------------------------------------------------------------------
// Measured on 148 SMs, us.  Streaming kernel (tokens are its MMAs' columns, 128 at most) / 64- and 128-column tiles:
//   rows   K 4096, N 4096     K 4096, N 16384    K 2048, N 512      K 1024, N 8192
//     16   10.8 / 12.1 13.4   26.0 / 29.3 27.4    6.8 / 7.0 8.4      7.2 / 10.3 11.0
//     32   12.3 / 12.2 13.4   27.4 / 29.6 27.5    8.0 / 6.7 8.4      8.5 /  9.7 10.7
//     64   16.6 / 12.3 13.5   30.2 / 30.0 27.9   10.5 / 6.7 8.4     10.9 /  7.4  9.9
//    128   25.2 / 12.5 13.7   37.1 / 30.7 28.6   17.1 / 6.7 8.5     16.1 /  7.6 10.1
// so the streaming kernel up to 32 rows.
// Pairs of CTAs / 128 columns: K 4096 with 64, 72, 80 tiles of 256 x 256 27.7 / 31.6, 28.5 / 32.8, 44.8 / 40.1 (six
// tiles of a second wave), K 2048 with 128 28.3 / 32.5; many tiles of 8, 7, 4 K steps 19.1 / 19.4, 18.6 / 18.2, 15.8 / 13.1.
// 128 / 64 columns, K 2048: 64, 72, 80, 96 tiles of 128 x 128 10.9 / 9.0, 11.1 / 9.0, 11.1 / 13.4, 11.1 / 13.6.
constexpr int64_t kLinearStream = 32;
static int linear_tile(const ffn_b200_linear_problem& p, int grid) {
  if (p.m <= kLinearStream) return FFN_B200_LINEAR_STREAM;
  const int64_t pairs = cdiv(p.m, 256) * cdiv(p.n, 256), steps = cdiv(p.k, 64);
  if (grid >= 2 && pairs >= grid / 2 && steps >= 8) return FFN_B200_LINEAR_PAIR256;
  return cdiv(p.m, 128) * cdiv(p.n, 128) >= grid / 2 ? FFN_B200_LINEAR_CTA128 : FFN_B200_LINEAR_CTA64;
}

extern "C" {

int ffn_b200_linear_make_plan(const ffn_b200_linear_problem* pr, ffn_b200_linear_plan* out) {
  if (!pr || !out) return FFN_B200_ERR_INVALID;
  int rc = check_linear(*pr);
  if (rc) return rc;
  int sms = 0;
  rc = device_sms(pr->sm_count, &sms);
  if (rc) return rc;
  std::memset(out, 0, sizeof(*out));
  const int grid = pr->block_num ? pr->block_num : sms;
  out->block_num = grid;
  out->split = 1;
  if (pr->tile == FFN_B200_LINEAR_STREAM && pr->m > 128) return FFN_B200_ERR_INVALID;
  out->status_words = 4;
  out->tile = pr->tile ? pr->tile : linear_tile(*pr, grid);
  if (out->tile == FFN_B200_LINEAR_STREAM) {
    // Equal numbers of weight rows per CTA, in tiles of at most 128.
    const int64_t per_cta = cdiv(pr->n, static_cast<int64_t>(grid) * 128);
    out->tile_m = static_cast<int32_t>(cdiv(pr->n, grid * per_cta));
    out->tile_n = stream_chunk(pr->m);
    const StreamRing ring(static_cast<int>(cdiv(out->tile_m, 8)) * 1024, out->tile_n, 0);
    out->stages = ring.stages;
    out->smem_bytes = ring.smem;
    return FFN_B200_OK;
  }
  const GemmTile tile = gemm_tile(out->tile);
  const int64_t tiles = cdiv(pr->m, tile.rows) * cdiv(pr->n, tile.cols), steps = cdiv(pr->k, 64);
  if (tiles >= (int64_t(1) << 31)) return FFN_B200_ERR_TOO_LARGE;
  out->tile_m = tile.rows;
  out->tile_n = tile.cols;
  out->stages = tile.stages;
  out->smem_bytes = tile.smem;
  if (out->tile == FFN_B200_LINEAR_PAIR256) {
    if (grid < 2) return FFN_B200_ERR_INVALID;
    out->block_num = static_cast<int32_t>(2 * std::min<int64_t>(tiles, grid / 2));
  } else {
    // Few tiles: clusters of up to 8 CTAs split K while each keeps at least 4 steps.
    while (out->split < 8 && tiles * out->split * 2 <= grid && steps >= out->split * 2 * 4) out->split *= 2;
    out->block_num = static_cast<int32_t>(std::min<int64_t>(tiles, grid / out->split) * out->split);
  }
  return FFN_B200_OK;
}

int ffn_b200_linear_prepare(const ffn_b200_linear_problem* pr, const void* w, int64_t ldw, const void* bias,
                            int32_t* status, int device, ffn_b200_linear** out) {
  if (!pr || !w || !out) return FFN_B200_ERR_INVALID;
  *out = nullptr;
  ffn_b200_linear_plan plan;
  int rc = check_device(device);
  if (!rc) rc = ffn_b200_linear_make_plan(pr, &plan);
  if (rc) return rc;
  if (bad_rows(w, ldw, pr->k)) return FFN_B200_ERR_ALIGNMENT;
  if (bias && !aligned16(bias)) return FFN_B200_ERR_ALIGNMENT;
  if (!status) return FFN_B200_ERR_INVALID;
  int sms = 0, maj = 0, min = 0;
  rc = ffn_b200_device_info(device, &sms, &maj, &min);
  if (rc) return rc;
  if (plan.block_num > sms) return FFN_B200_ERR_DEVICE;
  rc = get_encode();
  if (rc) return rc;
  DeviceScope scope(device);
  if (!scope.ok) return FFN_B200_ERR_DEVICE;
  auto* h = new (std::nothrow) ffn_b200_linear();
  if (!h) return FFN_B200_ERR_INVALID;
  h->prob = *pr;
  h->plan = plan;
  h->device = device;
  h->w = w;
  h->ldw = ldw;
  h->bias = bias;
  h->status = status;
  if (plan.tile == FFN_B200_LINEAR_STREAM) {
    ffnb200::StreamParams& P = h->params;
    std::memset(&P, 0, sizeof(P));
    const int rows = plan.tile_m;
    rc = encode_weights(&P.tm_w1, w, pr->dtype, pr->k, pr->n, 1, 1, ldw, pr->n * ldw, rows);
    P.tokens = static_cast<int>(pr->m);
    P.groups1 = static_cast<int>(cdiv(pr->n, rows));
    P.group_rows = P.group_feats = rows;
    P.unit_groups = 1;
    P.steps1 = static_cast<int>(cdiv(pr->k, 64));
    P.feat1 = static_cast<int>(pr->n);
    P.slab = static_cast<int>(cdiv(rows, 8)) * 1024;
    P.chunk = plan.tile_n;
    const StreamRing ring(P.slab, P.chunk, 0);
    P.blocks = ring.blocks;
    P.stages = ring.stages;
    P.act = pr->activation;
    P.bias = static_cast<const uint16_t*>(bias);
    P.status = status;
    P.wait_limit_ns = 4000000000ull;
    h->fn = pr->dtype == FFN_B200_BF16 ? ffnb200::stream_kernel<true, false> : ffnb200::stream_kernel<false, false>;
    if (!rc) rc = set_smem(reinterpret_cast<const void*>(h->fn), kMaxSmem);
  } else {
    const GemmTile tile = gemm_tile(plan.tile);
    ffnb200::GemmParams& G = h->gemm;
    std::memset(&G, 0, sizeof(G));
    rc = encode_rows(&G.tm_w, w, pr->dtype, pr->k, pr->n, ldw, tile.box_rows);
    G.M = static_cast<int>(pr->m);
    G.N = static_cast<int>(pr->n);
    G.steps = static_cast<int>(cdiv(pr->k, 64));
    G.tiles_m = static_cast<int>(cdiv(pr->m, tile.rows));
    G.tiles_n = static_cast<int>(cdiv(pr->n, tile.cols));
    G.group = std::min(G.tiles_m, 8);
    G.split = plan.split;
    G.act = pr->activation;
    G.bias = static_cast<const uint16_t*>(bias);
    G.status = status;
    G.wait_limit_ns = 4000000000ull;
    if (!rc) rc = set_smem(reinterpret_cast<const void*>(tile.fn[pr->dtype == FFN_B200_BF16]), tile.smem);
  }
  if (rc) {
    delete h;
    return rc;
  }
  *out = h;
  return FFN_B200_OK;
}

int ffn_b200_linear_run(ffn_b200_linear* h, const void* x, int64_t ldx, const void* res, int64_t ldr, void* y,
                        int64_t ldy, void* stream) {
  if (!h || !x || !y) return FFN_B200_ERR_INVALID;
  const ffn_b200_linear_problem& p = h->prob;
  if (bad_rows(x, ldx, p.k) || bad_rows(y, ldy, p.n) || (res && bad_rows(res, ldr, p.n))) return FFN_B200_ERR_ALIGNMENT;
  DeviceScope scope(h->device);
  if (!scope.ok) return FFN_B200_ERR_DEVICE;
  if (h->plan.tile == FFN_B200_LINEAR_STREAM) {
    ffnb200::StreamParams P = h->params;
    const int rc = encode_rows(&P.tm_x, x, p.dtype, p.k, p.m, ldx, P.chunk);
    if (rc) return rc;
    P.residual = static_cast<const uint16_t*>(res);
    P.ldr = ldr;
    P.y = static_cast<uint16_t*>(y);
    P.ldy = ldy;
    return launch_stream(h->fn, P, h->plan.block_num, h->plan.smem_bytes, false, stream);
  }
  ffnb200::GemmParams G = h->gemm;
  int rc = encode_rows(&G.tm_x, x, p.dtype, p.k, p.m, ldx, 128);
  if (!rc) rc = encode_rows(&G.tm_y, y, p.dtype, p.n, p.m, ldy, 32);
  if (rc) return rc;
  G.residual = static_cast<const uint16_t*>(res);
  G.ldr = ldr;
  G.y = static_cast<uint16_t*>(y);
  G.ldy = ldy;
  const GemmTile tile = gemm_tile(h->plan.tile);
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(h->plan.block_num), 1, 1);
  cfg.blockDim = dim3(ffnb200::kGemmThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(tile.smem);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int cluster = h->plan.tile == FFN_B200_LINEAR_PAIR256 ? 2 : h->plan.split;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  if (cudaLaunchKernelEx(&cfg, tile.fn[p.dtype == FFN_B200_BF16], G) == cudaSuccess) return FFN_B200_OK;
  cudaGetLastError();
  return FFN_B200_ERR_CUDA;
}

int ffn_b200_linear_reset(ffn_b200_linear* h, void* stream) {
  if (!h) return FFN_B200_ERR_INVALID;
  DeviceScope scope(h->device);  // (a null stream is the current device's)
  if (!scope.ok) return FFN_B200_ERR_DEVICE;
  if (cudaMemsetAsync(h->status, 0, 4 * h->plan.status_words, static_cast<cudaStream_t>(stream)) == cudaSuccess)
    return FFN_B200_OK;
  cudaGetLastError();
  return FFN_B200_ERR_CUDA;
}

int ffn_b200_linear_destroy(ffn_b200_linear* h) {
  delete h;
  return FFN_B200_OK;
}

// ---- expert router -------------------------------------------------------------------------
int ffn_b200_router_scratch(const ffn_b200_router_problem* pr, int64_t* logit_doubles, int64_t* counter_words) {
  if (!pr || !logit_doubles || !counter_words) return FFN_B200_ERR_INVALID;
  const int rc = check_router(*pr);
  if (rc) return rc;
  // fp64 logits, then fp32: sums of |x w|, or of many tokens the squared norms of their rows and the weights'
  // (more of them than logits when there is one expert).
  const int64_t parts = route_parts(*pr), cells = parts * pr->m * pr->experts;
  const int64_t floats = route_many(*pr) ? std::max(cells, parts * (pr->m + pr->experts)) : cells;
  *logit_doubles = cells + (floats + 1) / 2;
  *counter_words = cdiv(pr->m, 16);
  return FFN_B200_OK;
}

int ffn_b200_router_run(const ffn_b200_router_problem* pr, const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const float* cbias, const uint8_t* mask, int32_t* ids, float* weights, double* logits,
                        uint32_t* counters, void* stream) {
  if (!pr || !x || !w || !ids || !weights || !logits || !counters) return FFN_B200_ERR_INVALID;
  const int rc = check_router(*pr);
  if (rc) return rc;
  if (bad_rows(x, ldx, pr->k) || bad_rows(w, ldw, pr->k)) return FFN_B200_ERR_ALIGNMENT;
  ffnb200::RouteParams P = route_params(*pr, w, ldw, cbias, logits, route_parts(*pr), counters);
  P.x = x;
  P.ldx = ldx;
  P.mask = mask;
  P.ids = ids;
  P.weights = weights;
  // Experts per lane of a warp: as few registers and as little code as the number of experts needs.
  const int per = pr->experts <= 64 ? 0 : (pr->experts <= 256 ? 1 : 2);
  const RouteFns& fns = pr->dtype == FFN_B200_BF16 ? kRouteFns[per][1] : kRouteFns[per][0];
  if (pr->m < kRouteMany) return launch_route(pr->weight_f32 ? fns.few32 : fns.few, P, 1, 1, stream);  // small tiles: more CTAs
  if (!route_many(*pr)) return launch_route(fns.many32, P, 2, 4, stream);
  P.many = 1;
  const dim3 tiles(static_cast<unsigned>(cdiv(P.E, ffnb200::kLogitTile) * cdiv(P.M, ffnb200::kLogitTile)),
                   static_cast<unsigned>(P.parts), 1);
  const int rc2 = launch_route(fns.logits, P, tiles, ffnb200::kLogitSmem, stream);
  if (rc2) return rc2;
  return launch_route(fns.choose, P, dim3(static_cast<unsigned>(cdiv(P.M, ffnb200::kRouteWarps)), 1, 1),
                      ffnb200::route_space<ffnb200::kRouteWarps>(P.E), stream);
}

// ---- mixture-of-experts layer --------------------------------------------------------------
// Parts of K of the router's logits, so that its tiles of 16 tokens x 8 experts fill the CTAs.
static int moe_route_parts(const ffn_b200_moe_problem& p, int grid) {
  const int64_t tiles = cdiv(p.m, 16) * cdiv(p.experts, 8), steps = cdiv(p.k, ffnb200::kRouteStep);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({8, grid / tiles, cdiv(steps, 16)})));
}

int ffn_b200_moe_make_plan(const ffn_b200_moe_problem* pr, ffn_b200_moe_plan* out) {
  if (!pr || !out) return FFN_B200_ERR_INVALID;
  int rc = check_moe(*pr);
  if (rc) return rc;
  int sms = 0;
  rc = device_sms(pr->sm_count, &sms);
  if (rc) return rc;
  std::memset(out, 0, sizeof(*out));
  const int grid = pr->block_num ? pr->block_num : sms;
  const int tokens = static_cast<int>(pr->m);
  out->block_num = grid;
  // Tokens of one item: an expert's even share and three times its spread, so that few experts need a
  // second item (and their weights a second trip) while the ring keeps its room for weights (64
  // tokens, 6 of 64 experts: 168 us with slots of 64 token rows, 150 us with 16).
  const double share = static_cast<double>(pr->m) * pr->top_k / pr->experts;
  out->chunk = stream_chunk(std::min<int64_t>(pr->m, static_cast<int64_t>(std::ceil(share + 3.0 * std::sqrt(share)))));
  const ffnb200::StreamLists lists(tokens, pr->experts, pr->top_k, out->chunk);
  const StreamRing ring(ffnb200::kABytes, out->chunk, lists.bytes);
  out->stages = ring.stages;
  out->smem_bytes = ring.smem;
  out->hidden_rows = pr->m * pr->top_k;
  out->hidden_pitch = pitch_of(pr->h);
  out->sorted_pitch = pr->m > kMoeGather ? pitch_of(pr->k) : 0;
  const int64_t slots = 2ll * grid * out->chunk * 128;
  const int64_t items = ffnb200::StreamLists::most_items(tokens, pr->experts, pr->top_k, out->chunk);
  const int64_t down = cdiv(pr->n, 128);
  if (items * down * cdiv(pr->h, 64) >= (int64_t(1) << 31)) return FFN_B200_ERR_TOO_LARGE;
  out->workspace_floats = slots + out->hidden_rows * down * 128;
  out->counter_words = ffnb200::kStreamSync + items + cdiv(pr->m, 16) + 1;
  out->route_doubles = (pr->m * pr->experts * moe_route_parts(*pr, grid) * 3 + 1) / 2;  // fp64 logits, fp32 sums
  out->status_words = 4;
  return FFN_B200_OK;
}

int ffn_b200_moe_prepare(const ffn_b200_moe_problem* pr, const ffn_b200_moe_buffers* b, int device,
                         ffn_b200_moe** out) {
  if (!pr || !b || !out) return FFN_B200_ERR_INVALID;
  *out = nullptr;
  ffn_b200_moe_plan plan;
  int rc = check_device(device);
  if (!rc) rc = ffn_b200_moe_make_plan(pr, &plan);
  if (rc) return rc;
  int sms = 0, maj = 0, min = 0;
  rc = ffn_b200_device_info(device, &sms, &maj, &min);
  if (rc) return rc;
  if (plan.block_num > sms) return FFN_B200_ERR_DEVICE;  // the CTAs wait on one another
  if (!b->w1 || !b->w2 || !b->hidden || !b->workspace || !b->counters || !b->status) return FFN_B200_ERR_INVALID;
  if (plan.sorted_pitch && !b->sorted) return FFN_B200_ERR_INVALID;
  if (bad_rows(b->w1, b->ldw1, pr->k) || bad_rows(b->w2, b->ldw2, pr->h) || b->stride1 % 8 || b->stride2 % 8 ||
      b->stride1 <= 0 || b->stride2 <= 0 || !aligned16(b->hidden) || !aligned16(b->sorted) || !aligned16(b->workspace))
    return FFN_B200_ERR_ALIGNMENT;
  rc = get_encode();
  if (rc) return rc;
  DeviceScope scope(device);
  if (!scope.ok) return FFN_B200_ERR_DEVICE;
  auto* h = new (std::nothrow) ffn_b200_moe();
  if (!h) return FFN_B200_ERR_INVALID;
  h->prob = *pr;
  h->plan = plan;
  h->buf = *b;
  h->device = device;
  ffnb200::StreamParams& P = h->params;
  std::memset(&P, 0, sizeof(P));
  const bool glu = pr->activation == FFN_B200_SWIGLU;
  // Groups of 16 weight rows: 16 hidden features, or gate and up rows of 8.
  P.group_rows = 16;
  P.group_feats = glu ? 8 : 16;
  P.unit_groups = 8;
  P.slab = ffnb200::kABytes;
  rc = encode_weights(&P.tm_w1, b->w1, pr->dtype, pr->k, pr->h, glu ? 2 : 1, pr->experts, b->ldw1, b->stride1,
                      P.group_feats);
  if (!rc)
    rc = encode_weights(&P.tm_w2, b->w2, pr->dtype, pr->h, pr->n, 1, pr->experts, b->ldw2, b->stride2, 128);
  if (!rc) rc = encode_rows(&P.tm_h8, b->hidden, pr->dtype, pr->h, plan.hidden_rows, plan.hidden_pitch, 8);
  if (!rc) rc = encode_rows(&P.tm_h64, b->hidden, pr->dtype, pr->h, plan.hidden_rows, plan.hidden_pitch, 64);
  if (plan.sorted_pitch) {
    if (!rc) rc = encode_rows(&P.tm_x8, b->sorted, pr->dtype, pr->k, plan.hidden_rows, plan.sorted_pitch, 8);
    if (!rc) rc = encode_rows(&P.tm_x64, b->sorted, pr->dtype, pr->k, plan.hidden_rows, plan.sorted_pitch, 64);
    P.sorted = static_cast<uint16_t*>(b->sorted);
    P.lds = plan.sorted_pitch;
  }
  P.tokens = static_cast<int>(pr->m);
  P.groups1 = static_cast<int>(cdiv(pr->h, P.group_feats));
  P.steps1 = static_cast<int>(cdiv(pr->k, 64));
  P.feat1 = static_cast<int>(pr->h);
  P.tiles2 = static_cast<int>(cdiv(pr->n, 128));
  P.steps2 = static_cast<int>(cdiv(pr->h, 64));
  P.feat2 = static_cast<int>(pr->n);
  P.chunk = plan.chunk;
  const StreamRing ring(P.slab, P.chunk, ffnb200::StreamLists(P.tokens, pr->experts, pr->top_k, P.chunk).bytes);
  P.blocks = ring.blocks;
  P.stages = ring.stages;
  P.act = pr->activation;
  P.hidden = static_cast<uint16_t*>(b->hidden);
  P.ldh = plan.hidden_pitch;
  const int64_t slots = 2ll * plan.block_num * plan.chunk * 128;
  P.pieces = b->workspace;
  P.whole = b->workspace + slots;
  P.counters = b->counters;
  h->route_counters = b->counters + plan.counter_words - cdiv(pr->m, 16) - 1;
  P.status = b->status;
  P.experts = pr->experts;
  P.top = pr->top_k;
  P.wait_limit_ns = 4000000000ull;
  h->fn = pr->dtype == FFN_B200_BF16 ? ffnb200::stream_kernel<true, true> : ffnb200::stream_kernel<false, true>;
  if (!rc) rc = set_smem(reinterpret_cast<const void*>(h->fn), kMaxSmem);
  if (rc) {
    delete h;
    return rc;
  }
  *out = h;
  return FFN_B200_OK;
}

// The router's part of a run's arguments: set once per handle, before its first routed run.
int ffn_b200_moe_set_router(ffn_b200_moe* h, const ffn_b200_router_problem* pr, const void* w, int64_t ldw,
                            const float* choice_bias, double* logits) {
  if (!h || !pr || !w || !logits) return FFN_B200_ERR_INVALID;
  const int rc = check_router(*pr);
  if (rc) return rc;
  const ffn_b200_moe_problem& p = h->prob;
  if (pr->m != p.m || pr->k != p.k || pr->experts != p.experts || pr->top_k != p.top_k || pr->dtype != p.dtype)
    return FFN_B200_ERR_INVALID;
  if (bad_rows(w, ldw, pr->k)) return FFN_B200_ERR_ALIGNMENT;
  h->params.route = route_params(*pr, w, ldw, choice_bias, logits, moe_route_parts(p, h->plan.block_num), h->route_counters);
  return FFN_B200_OK;
}

static int moe_launch(ffn_b200_moe* h, ffnb200::StreamParams& P, const void* x, int64_t ldx, const void* res, int64_t ldr,
                      void* y, int64_t ldy, void* stream) {
  const ffn_b200_moe_problem& p = h->prob;
  if (bad_rows(x, ldx, p.k) || bad_rows(y, ldy, p.n) || (res && bad_rows(res, ldr, p.n))) return FFN_B200_ERR_ALIGNMENT;
  DeviceScope scope(h->device);
  if (!scope.ok) return FFN_B200_ERR_DEVICE;
  const int rc = P.sorted ? FFN_B200_OK : encode_rows(&P.tm_x, x, p.dtype, p.k, p.m, ldx, 1);
  if (rc) return rc;
  P.x = static_cast<const uint16_t*>(x);
  P.ldx = ldx;
  P.residual = static_cast<const uint16_t*>(res);
  P.ldr = ldr;
  P.y = static_cast<uint16_t*>(y);
  P.ldy = ldy;
  return launch_stream(h->fn, P, h->plan.block_num, h->plan.smem_bytes, true, stream);
}

int ffn_b200_moe_run(ffn_b200_moe* h, const void* x, int64_t ldx, const uint8_t* mask, int32_t* ids, float* weights,
                     const void* res, int64_t ldr, void* y, int64_t ldy, void* stream) {
  if (!h || !x || !ids || !weights || !y || !h->params.route.w) return FFN_B200_ERR_INVALID;
  ffnb200::StreamParams P = h->params;
  P.routed = 1;
  P.route.x = x;
  P.route.ldx = ldx;
  P.route.mask = mask;
  P.route.ids = ids;
  P.route.weights = weights;
  P.ids = ids;
  P.weights = weights;
  return moe_launch(h, P, x, ldx, res, ldr, y, ldy, stream);
}

int ffn_b200_moe_run_routed(ffn_b200_moe* h, const void* x, int64_t ldx, const int32_t* ids, const float* weights,
                            const void* res, int64_t ldr, void* y, int64_t ldy, void* stream) {
  if (!h || !x || !ids || !weights || !y) return FFN_B200_ERR_INVALID;
  ffnb200::StreamParams P = h->params;
  P.ids = ids;
  P.weights = weights;
  return moe_launch(h, P, x, ldx, res, ldr, y, ldy, stream);
}

int ffn_b200_moe_reset(ffn_b200_moe* h, void* stream) {
  if (!h) return FFN_B200_ERR_INVALID;
  DeviceScope scope(h->device);
  if (!scope.ok) return FFN_B200_ERR_DEVICE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cudaMemsetAsync(h->buf.counters, 0, 4 * h->plan.counter_words, st) != cudaSuccess ||
      cudaMemsetAsync(h->buf.status, 0, 4 * h->plan.status_words, st) != cudaSuccess) {
    cudaGetLastError();
    return FFN_B200_ERR_CUDA;
  }
  return FFN_B200_OK;
}

int ffn_b200_moe_set_wait_limit(ffn_b200_moe* h, uint64_t ns) {
  if (!h || ns == 0 || ns > kMaxWaitNs) return FFN_B200_ERR_INVALID;
  h->params.wait_limit_ns = ns;
  return FFN_B200_OK;
}

int ffn_b200_moe_set_fault_injection(ffn_b200_moe* h, int mode) {
  if (!h || mode < 0 || mode > 1) return FFN_B200_ERR_INVALID;
  h->params.inject = mode;
  return FFN_B200_OK;
}

int ffn_b200_moe_destroy(ffn_b200_moe* h) {
  delete h;
  return FFN_B200_OK;
}

// ---- operand packing -----------------------------------------------------------------------
int ffn_b200_pack_rows(const void* src, int64_t row_stride, int64_t col_stride, int64_t rows, int64_t cols, void* dst,
                       int64_t ld, int device, void* stream) {
  if (!src || !dst || rows <= 0 || cols <= 0 || cols > kMaxDim || row_stride < 0 || col_stride < 0 || ld < cols)
    return FFN_B200_ERR_INVALID;
  const int64_t tiles = cdiv(rows, ffnb200::kPackTile);
  if (tiles >= (int64_t(1) << 31)) return FFN_B200_ERR_TOO_LARGE;
  DeviceScope scope(device);
  if (!scope.ok) return FFN_B200_ERR_DEVICE;
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(cdiv(cols, ffnb200::kPackTile)), 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, ffnb200::pack_rows_kernel, static_cast<const uint16_t*>(src), static_cast<long long>(row_stride),
                         static_cast<long long>(col_stride), static_cast<long long>(rows), static_cast<int>(cols),
                         static_cast<uint16_t*>(dst), static_cast<long long>(ld)) == cudaSuccess)
    return FFN_B200_OK;
  cudaGetLastError();
  return FFN_B200_ERR_CUDA;
}

}  // extern "C"
