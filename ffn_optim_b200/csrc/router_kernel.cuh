// Expert router: logits = X . W^T, scores, top-k and weights in one launch.
//
// The ids must be those of 64-bit logits, whatever the order of the sums, at the cost of tensor
// cores rather than of fp64 arithmetic (64 multiply-adds per clock and SM):
//   * 16-bit weights: products on mma.sync (m16n8k16, fp32 accumulation) in chains of 64 of K; each
//     chain's fp32 result is added in fp64.  A chain of four MMAs loses at most 4 * 2^-22 of the
//     sum of its |x w|, so a logit is off by at most 2^-20 S, S = sum |x w|, which a second set
//     of MMAs over the operands with their signs cleared gives.
//   * The finishing warp picks the top k + 1 keys; experts whose key lies closer to one of them
//     than those errors allow (and logits that left fp32's range) are summed again in fp64, by the
//     whole warp, and the choice is made again.  For normally distributed logits that is a
//     few tokens in a thousand.
//   * fp32 weights are summed in fp64 outright (S = 0: nothing is summed twice).
//
// A CTA takes 16 MT tokens x 8 NT experts; its 8 warps split K in steps of 64 (operands straight
// from L2 to registers: a lane reads 16 bytes of a row, and since A and B use the same order of
// K inside a step, no shuffle is needed).  The CTA that arrives last at its tokens finishes
// them, a warp per token.  What bounds it: for a few tokens the launch and three dependent L2
// trips; for many the L2 reads of the operand tiles.
#pragma once

#include "ffn_kernel.cuh"

namespace ffnb200 {

constexpr int kRouteWarps = 8;
constexpr int kRouteThreads = 32 * kRouteWarps;
constexpr int kRouteStep = 64;                 // K per chain
constexpr double kRouteLoss = 1.0 / (1 << 20); // error of a logit over the sum of its |x w|

struct RouteParams {
  const void* x;
  long long ldx;
  const void* w;
  long long ldw;
  const float* choice_bias;
  const uint8_t* mask;
  int* ids;
  float* weights;
  double* logits;   // [M][E]
  float* sums;      // [M][E]: sum |x w|
  unsigned* counters;
  int M, K, E, top;
  int sigmoid, renormalize;
  float scale;
};

template <bool BF16>
__device__ __forceinline__ void mma_16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 consecutive 16-bit values of a row from column k (a multiple of 8), zero from column K on.
// (A 16-byte aligned read that holds at least one column of the row stays inside its allocation.)
__device__ __forceinline__ uint4 row_chunk(const void* base, long long off, int k, int K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k < K) {
    v = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + off + k));
    if (k + 8 > K) {
      uint32_t* r = &v.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (k + 2 * i >= K) r[i] = 0;
        else if (k + 2 * i + 1 >= K) r[i] &= 0xFFFFu;
      }
    }
  }
  return v;
}
// sum x w of 8 values in fp64
template <bool BF16>
__device__ __forceinline__ double dot8(const uint4& a, const uint4& b, double s) {
  const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fma(static_cast<double>(unpack_lo<BF16>(av[i])), static_cast<double>(unpack_lo<BF16>(bv[i])), s);
    s = fma(static_cast<double>(unpack_hi<BF16>(av[i])), static_cast<double>(unpack_hi<BF16>(bv[i])), s);
  }
  return s;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A double as an unsigned integer of the same order (no NaN).
__device__ __forceinline__ unsigned long long ordered(double v) {
  const long long b = __double_as_longlong(v + 0.0);  // (+ 0.0: one zero)
  return static_cast<unsigned long long>(b ^ (b < 0 ? -1ll : static_cast<long long>(1ull << 63)));
}
// The key of expert e: its score, with the choice bias; NaN ranks last.
__device__ __forceinline__ double route_key(const RouteParams& p, double score, int e) {
  const double key = p.choice_bias ? score + static_cast<double>(__ldg(p.choice_bias + e)) : score;
  return key == key ? key : -INFINITY;
}

// One token's choice by a warp; z and q: this warp's logits and scores in shared memory [E].
// (Loops are kept rolled: the code runs once per token, and fetching it costs more than running it.)
template <bool BF16, bool W32>
__device__ __forceinline__ void route_token(const RouteParams& p, int t, int lane, double* z, double* q) {
  int* ids = p.ids + static_cast<size_t>(t) * p.top;
  float* weights = p.weights + static_cast<size_t>(t) * p.top;
  if (p.mask && !p.mask[t]) {
    for (int j = lane; j < p.top; j += 32) ids[j] = -1, weights[j] = 0.f;
    return;
  }
  float s = 0.f;
  bool odd = false;  // a logit left fp32's range
#pragma unroll 2
  for (int e = lane; e < p.E; e += 32) {
    const double v = __ldcg(p.logits + static_cast<size_t>(t) * p.E + e);
    if (!W32) {
      s = fmaxf(s, __ldcg(p.sums + static_cast<size_t>(t) * p.E + e));
      odd |= !isfinite(v);
    }
    z[e] = v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, o));
  const double loss = kRouteLoss * static_cast<double>(s);
  int chosen = -1;     // lane j < top: the j-th choice,
  double score = 0.0;  // its score
#pragma unroll 1
  for (int pass = 0;; ++pass) {
    // Scores.  A NaN logit makes every softmax score NaN.
    double scale = 1.0;
    if (!p.sigmoid) {
      double top = -INFINITY, sum = 0.0;
      bool nan = false;
#pragma unroll 1
      for (int e = lane; e < p.E; e += 32) top = fmax(top, z[e]), nan |= z[e] != z[e];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (__any_sync(0xffffffffu, nan)) top = NAN;
#pragma unroll 1
      for (int e = lane; e < p.E; e += 32) sum += q[e] = exp(z[e] - top);
      scale = 1.0 / warp_sum(sum);
    }
    // This lane's best expert not yet chosen.
    unsigned used = 0;  // bit i: expert lane + 32 i
    int at = -1;
    double best = 0.0;
    unsigned long long order = 0;
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32) {
      const double v = p.sigmoid ? 1.0 / (1.0 + exp(-z[e])) : q[e] * scale;
      q[e] = v;
      const double key = route_key(p, v, e);
      if (at < 0 || key > best) best = key, at = e;
    }
    order = at < 0 ? 0 : ordered(best);
    // The k largest keys and the next one, equal ones by index.
    double key = 0.0, rest = 0.0;  // lane j: the j-th key; the key after the last choice
    const int want = W32 || pass || p.top == p.E ? p.top : p.top + 1;
#pragma unroll 1
    for (int j = 0; j < want; ++j) {
      const unsigned hi = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(order >> 32));
      bool mine = static_cast<unsigned>(order >> 32) == hi;
      const unsigned lo = __reduce_max_sync(0xffffffffu, mine ? static_cast<unsigned>(order) : 0u);
      mine = mine && static_cast<unsigned>(order) == lo;
      const unsigned e = __reduce_min_sync(0xffffffffu, mine && at >= 0 ? static_cast<unsigned>(at) : 0xffffffffu);
      const double kj = __shfl_sync(0xffffffffu, best, static_cast<int>(e & 31u));
      if (j == p.top) {
        rest = kj;
        break;
      }
      if (lane == j) chosen = static_cast<int>(e), key = kj, score = q[e];
      if (lane == static_cast<int>(e & 31u)) {
        used |= 1u << (e >> 5);
        at = -1;
#pragma unroll 1
        for (int f = lane; f < p.E; f += 32)
          if (!(used >> (f >> 5) & 1u)) {
            const double v = route_key(p, q[f], f);
            if (at < 0 || v > best) best = v, at = f;
          }
        order = at < 0 ? 0 : ordered(best);
      }
      __syncwarp();
    }
    if (W32 || pass) break;
    // Could the errors of two logits have swapped neighbours?  A score moves by at most its slope
    // times a logit's error: p (1 - p) for the sigmoid, 2 p with softmax's normaliser.
    const double after = __shfl_down_sync(0xffffffffu, key, 1);
    const double next = lane == p.top - 1 ? rest : after;
    const double slope = p.sigmoid ? 0.25 : 2.0 * score;
    const bool last = lane == p.top - 1 && p.top == p.E;
    const bool near = lane < p.top && !last && key - next <= 2.0 * loss * slope && loss > 0.0;
    if (!__any_sync(0xffffffffu, near || odd)) break;
    // Sums again in fp64, unless the token itself is not finite.
    const long long xo = static_cast<long long>(t) * p.ldx;
    bool finite = true;
#pragma unroll 1
    for (int k = 8 * lane; k < p.K; k += 256) {
      const uint4 v = row_chunk(p.x, xo, k, p.K);
      const uint32_t r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) finite = finite && isfinite(unpack_lo<BF16>(r[i])) && isfinite(unpack_hi<BF16>(r[i]));
    }
    if (!__all_sync(0xffffffffu, finite)) break;
    // Which: logits out of range, and experts whose key is as close to a chosen one's or to the
    // next one's.  (Of two scores within reach of one another the chosen one's slope is the larger.)
#pragma unroll 1
    for (int base = 0; base < p.E; base += 32) {
      const int e = base + lane;
      const double ke = e < p.E ? route_key(p, q[e], e) : 0.0;
      bool again = e < p.E && !isfinite(z[e]);
#pragma unroll 1
      for (int j = 0; j < p.top; ++j) {
        const double kj = __shfl_sync(0xffffffffu, key, j), sj = __shfl_sync(0xffffffffu, slope, j);
        const int cj = __shfl_sync(0xffffffffu, chosen, j);
        again |= e < p.E && e != cj && fabs(ke - kj) <= 2.0 * loss * sj;
        // (the chosen one itself, when its neighbour is that close)
        const bool nj = __shfl_sync(0xffffffffu, near, j) || (j > 0 && __shfl_sync(0xffffffffu, near, j > 0 ? j - 1 : 0));
        again |= e == cj && nj;
      }
      unsigned todo = __ballot_sync(0xffffffffu, again);
#pragma unroll 1
      while (todo) {
        const int src = __ffs(todo) - 1;
        todo &= todo - 1;
        const long long wo = static_cast<long long>(base + src) * p.ldw;
        double a = 0.0, b = 0.0;
#pragma unroll 1
        for (int k = 8 * lane; k < p.K; k += 512) {
          const uint4 xa = row_chunk(p.x, xo, k, p.K), wa = row_chunk(p.w, wo, k, p.K);
          const uint4 xb = row_chunk(p.x, xo, k + 256, p.K), wb = row_chunk(p.w, wo, k + 256, p.K);
          a = dot8<BF16>(xa, wa, a);
          b = dot8<BF16>(xb, wb, b);
        }
        a = warp_sum(a + b);
        if (lane == src) z[base + src] = a;
      }
    }
    __syncwarp();
  }
  const double total = warp_sum(lane < p.top ? score : 0.0);
  if (lane < p.top) {
    ids[lane] = chosen;
    weights[lane] = static_cast<float>((p.renormalize ? score / total : score) * static_cast<double>(p.scale));
  }
}

template <bool BF16, bool W32, int MT, int NT>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const RouteParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  double* part = reinterpret_cast<double*>(smem);  // [warps][16 MT][8 NT], then the |x w| sums
  float* part_s = reinterpret_cast<float*>(part + kRouteWarps * 128 * MT * NT);
  __shared__ int last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int t0 = blockIdx.y * 16 * MT, e0 = blockIdx.x * 8 * NT;
  if (threadIdx.x == 0) grid_dep_launch();
  grid_dep_wait();

  double z[MT][NT][4] = {};
  float sa[MT][NT][4] = {};
  if constexpr (!W32) {
    long long xo[2 * MT], wo[NT];  // rows past the last token or expert repeat it; nobody reads their sums
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) xo[i] = static_cast<long long>(min(t0 + 8 * i + g, p.M - 1)) * p.ldx;
#pragma unroll
    for (int j = 0; j < NT; ++j) wo[j] = static_cast<long long>(min(e0 + 8 * j + g, p.E - 1)) * p.ldw;
#pragma unroll(MT == 1 ? 4 : 1)
    for (int k0 = warp * kRouteStep; k0 < p.K; k0 += kRouteWarps * kRouteStep) {
      uint4 xv[2][2 * MT], wv[2][NT];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) xv[h][i] = row_chunk(p.x, xo[i], k0 + 32 * h + 8 * q, p.K);
#pragma unroll
        for (int j = 0; j < NT; ++j) wv[h][j] = row_chunk(p.w, wo[j], k0 + 32 * h + 8 * q, p.K);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          constexpr uint32_t kAbs = 0x7FFF7FFFu;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 &a = xv[h][2 * i], &b = xv[h][2 * i + 1], &w = wv[h][j];
            mma_16816<BF16>(d, a.x, b.x, a.y, b.y, w.x, w.y);
            mma_16816<BF16>(d, a.z, b.z, a.w, b.w, w.z, w.w);
            mma_16816<BF16>(sa[i][j], a.x & kAbs, b.x & kAbs, a.y & kAbs, b.y & kAbs, w.x & kAbs, w.y & kAbs);
            mma_16816<BF16>(sa[i][j], a.z & kAbs, b.z & kAbs, a.w & kAbs, b.w & kAbs, w.z & kAbs, w.w & kAbs);
          }
#pragma unroll
          for (int v = 0; v < 4; ++v) z[i][j][v] += static_cast<double>(d[v]);
        }
    }
  } else {
    const float* w = static_cast<const float*>(p.w);
    for (int k0 = warp * kRouteStep; k0 < p.K; k0 += kRouteWarps * kRouteStep)
      for (int k = k0; k < min(k0 + kRouteStep, p.K); ++k) {
        double xd[2 * MT], wd[2 * NT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)
          xd[i] = static_cast<double>(unpack_lo<BF16>(static_cast<uint32_t>(
              __ldg(static_cast<const uint16_t*>(p.x) + static_cast<long long>(min(t0 + 8 * i + g, p.M - 1)) * p.ldx + k))));
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j)
          wd[j] = static_cast<double>(__ldg(w + static_cast<long long>(min(e0 + 8 * (j / 2) + 2 * q + j % 2, p.E - 1)) * p.ldw + k));
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) z[i][j][v] = fma(xd[2 * i + v / 2], wd[2 * j + v % 2], z[i][j][v]);
      }
  }
  // The warps' parts of K, added in warp order.
  constexpr int kCols = 8 * NT, kCells = 128 * MT * NT;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int cell = (16 * i + 8 * (v / 2) + g) * kCols + 8 * j + 2 * q + v % 2;
        part[warp * kCells + cell] = z[i][j][v];
        if (!W32) part_s[warp * kCells + cell] = sa[i][j][v];
      }
  __syncthreads();
  for (int cell = threadIdx.x; cell < kCells; cell += kRouteThreads) {
    const int t = t0 + cell / kCols, e = e0 + cell % kCols;
    double sum = 0.0;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) {
      sum += part[w * kCells + cell];
      if (!W32) s += part_s[w * kCells + cell];
    }
    if (t < p.M && e < p.E) {
      __stcg(p.logits + static_cast<size_t>(t) * p.E + e, sum);
      if (!W32) __stcg(p.sums + static_cast<size_t>(t) * p.E + e, s);
    }
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned old;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(p.counters + blockIdx.y) : "memory");
    last = old == gridDim.x - 1;
    if (last) p.counters[blockIdx.y] = 0;  // for the next launch
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double* z_of = reinterpret_cast<double*>(smem) + 2 * warp * p.E;  // (the parts have been added up)
#pragma unroll 1
  for (int t = t0 + warp; t < min(t0 + 16 * MT, p.M); t += kRouteWarps) {
    route_token<BF16, W32>(p, t, lane, z_of, z_of + p.E);
    __syncwarp();
  }
}

}  // namespace ffnb200
