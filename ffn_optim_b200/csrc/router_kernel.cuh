// Expert router: logits = X . W^T, scores, top-k and weights, in one kernel for few tokens and in two for many.
//
// The ids must be those of 64-bit logits, whatever the order of the sums, at the cost of tensor
// cores rather than of fp64 arithmetic (64 multiply-adds per clock and SM):
//   * 16-bit weights: products on mma.sync (m16n8k16, fp32 accumulation) in chains of 64 of K; each
//     chain's fp32 result is added in fp64.  An MMA cuts its addends (16 products, the accumulator) off
//     at 2^-25 of the largest one's power of two, and its result to 24 bits: it loses at most
//     16 * 2^-25 + 2^-23 = 2.5 * 2^-22 of the sum of their sizes (measured with operands made for
//     it: 2.25), and a chain of four 10 * 2^-22 (8.2) of the sum of its |x w|.  So a logit is off by at most
//     2.5 * 2^-20 S, S = sum |x w|.  For few tokens a second set of MMAs over the operands with their
//     signs cleared gives S (short by the same rule: K / 16 MMAs lose 0.25 % at most); for many, where that
//     cost most (1000 tokens of 256 experts of 4096: 29 us for the logits), the norms of the two
//     rows bound it.
//   * The finishing warp picks the top k keys; chosen experts whose key another one's may meet within
//     those errors, those others, and logits that left fp32's range are summed again in fp64 by the
//     whole CTA, and the choice is made again.  For normally distributed operands that is less
//     than one token in a hundred of 64 experts, two to five of 256 in the many-token form.
//     (Softmax with a choice bias: all logits of such a token, since its denominator moves two keys
//     of different scores apart.)
//   * fp32 weights are summed in fp64 outright (S = 0: nothing is summed twice).
//
// Fewer than 128 tokens, and fp32 weights (route_kernel): a CTA takes 16 MT tokens x 8 NT experts;
// its 8 warps split K in steps of 64 (operands straight from L2 to registers: a lane reads 16
// bytes of a row, and since A and B use the same order of K inside a step, no shuffle is needed).
// The CTA that arrives last at its tokens finishes them, a warp per token.  Bound by the launch
// and three dependent L2 trips.
// More tokens (route_logits_kernel, route_choose_kernel): 64 x 64 tiles with K split over CTAs,
// operands through shared memory (the first form's L2 reads took 60 us for 1000 tokens and 256
// experts of 4096), then a warp per token over all SMs.
#pragma once

#include "ffn_kernel.cuh"

namespace ffnb200 {

constexpr int kRouteWarps = 8;
constexpr int kRouteThreads = 32 * kRouteWarps;
constexpr int kRouteStep = 64;                 // K per chain
constexpr double kRouteLoss = 2.51 / (1 << 20);  // error of a logit over the sum of its |x w|

struct RouteParams {
  const void* x;
  long long ldx;
  const void* w;
  long long ldw;
  const float* choice_bias;
  const uint8_t* mask;
  int* ids;
  float* weights;
  double* logits;   // [parts][M][E]: sums over a part of K
  float* sums;      // [parts][M][E]: sum |x w|; of many tokens [parts][M + E]: sum x^2, then sum w^2
  int parts, many;
  unsigned* counters;
  int M, K, E, top;
  int weight_f32, sigmoid, renormalize;
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
__device__ __forceinline__ double unordered(unsigned long long k) {
  const long long b = static_cast<long long>(k);
  return __longlong_as_double(b < 0 ? b ^ static_cast<long long>(1ull << 63) : ~b);
}

// The choice for one token per warp by a CTA's WARPS warps together (token t of this warp; t >= M: none):
// lane l holds experts l, l + 32, ... (PER of them) in registers.  smem: RouteSpace bytes.  Only
// sums taken again need the whole CTA: each is split over its warps, since one warp's trips through
// K would keep all the others waiting.  (Code that runs once per token is fetched more slowly than
// it runs: only the short loops over a lane's own experts are unrolled.)
constexpr int kAgainSlots = 4;  // sums again that a warp asks for at a time
template <int WARPS>
__host__ __device__ constexpr int route_space(int experts) {
  return WARPS * experts * 8 + WARPS * kAgainSlots * (WARPS * 8 + 4);
}
template <bool BF16, int PER, int WARPS>
__device__ __forceinline__ void route_tokens(const RouteParams& p, int t, uint8_t* smem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double* q = reinterpret_cast<double*>(smem) + warp * p.E;  // this warp's scores
  double* part = reinterpret_cast<double*>(smem) + WARPS * p.E;  // [warp][slot][part of K]
  int* slots = reinterpret_cast<int*>(part + WARPS * kAgainSlots * WARPS);  // [warp][slot]: expert, or -1
  int* ids = p.ids + static_cast<size_t>(t) * p.top;
  float* weights = p.weights + static_cast<size_t>(t) * p.top;
  const bool live = t < p.M && (!p.mask || p.mask[t]);
  if (!live && t < p.M)
    for (int j = lane; j < p.top; j += 32) ids[j] = -1, weights[j] = 0.f;
  double z[PER], bias[PER], v[PER];
  float s = 0.f;
  bool odd = false;  // a logit left fp32's range
  int chosen = 0;               // lane j < top: the j-th choice,
  double score = 0.0;           // its score
  unsigned long long mine = 0;  // and its key
  double loss = 0.0;    // a logit's error at most
  unsigned again = 0;  // bit i: expert lane + 32 i has to be summed again
  if (live) {
    // All of a part's loads are in flight together.
    const size_t cells = static_cast<size_t>(p.M) * p.E, pitch = p.many ? p.M + p.E : cells;
    const size_t at = static_cast<size_t>(t) * p.E + lane;
    const float* sum = p.sums + (p.many ? p.M + lane : at);
    float size[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) z[i] = 0.0, size[i] = 0.f, bias[i] = 0.0;
#pragma unroll 1
    for (int c = 0; c < p.parts; ++c) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < p.E) {
          z[i] += __ldcg(p.logits + c * cells + at + 32 * i);
          size[i] += __ldcg(sum + c * pitch + 32 * i);
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (lane + 32 * i < p.E) {
        if (p.choice_bias) bias[i] = static_cast<double>(__ldg(p.choice_bias + lane + 32 * i));
        s = fmaxf(s, size[i]);
        odd |= !p.weight_f32 && !isfinite(z[i]);
      } else {
        z[i] = -INFINITY;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, o));
    if (p.many) {  // |x| |w| of the longest w
      float x2 = 0.f;
      for (int c = 0; c < p.parts; ++c) x2 += __ldcg(p.sums + static_cast<size_t>(c) * (p.M + p.E) + t);
      // (The sums of squares are fp32, and zero only of zeros.  Below 2^-100 squares may be missing: such a
      // token's logits are summed again.)
      s = x2 == 0.f || s == 0.f ? 0.f : x2 < 0x1p-100f || s < 0x1p-100f ? INFINITY : sqrtf(x2) * sqrtf(s) * 1.001f;
    }
    loss = p.weight_f32 ? 0.0 : kRouteLoss * static_cast<double>(s);
  }
  // A key moves by at most a logit's error times the steepest slope on the way: p (1 - p) for the sigmoid,
  // whose slope moves by less than the error; p_i (e^(2 loss) - 1), at most 1/2 loss, for the softmax.
  double other = -INFINITY;
  const double steep = 2.0 + 3.0 * loss;
  auto reach = [&](double v) {
    return loss * (p.sigmoid ? v * (1.0 - v) + loss : loss > 0.5 ? 0.5 : fmin(0.5, steep * v));
  };
  // Once, and again where sums changed: one loop, so that the code is there once (few tokens wait for
  // instruction fetches more than for arithmetic; 1000 tokens of 256 experts 42.9 -> 41.0 us).
  bool first = true, changed = false;
#pragma unroll 1
  while (true) {
    if (live) {
      // Scores.  A NaN logit makes every softmax score NaN.
      if (p.sigmoid) {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = 1.0 / (1.0 + exp(-z[i]));
      } else {
        double top = -INFINITY, sum = 0.0;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) top = fmax(top, z[i]), nan |= z[i] != z[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (__any_sync(0xffffffffu, nan)) top = NAN;
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += v[i] = lane + 32 * i < p.E ? exp(z[i] - top) : 0.0;
        const double scale = 1.0 / warp_sum(sum);
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] *= scale;
      }
      // Keys as integers; 1, NaN, ranks below all numbers, and 0 below that: no expert, or one already chosen.
      unsigned long long key[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        const double k = v[i] + bias[i];
        key[i] = e < p.E ? (k == k ? ordered(k) : 1ull) : 0ull;
        if (e < p.E) q[e] = v[i];
      }
      __syncwarp();
      // The k largest keys, equal ones by index.
#pragma unroll 1
      for (int j = 0; j < p.top; ++j) {
        unsigned long long best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < PER; ++i)
          if (key[i] > best) best = key[i], at = i;
        const unsigned hi = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(best >> 32));
        const bool high = static_cast<unsigned>(best >> 32) == hi;
        const unsigned lo = __reduce_max_sync(0xffffffffu, high ? static_cast<unsigned>(best) : 0u);
        const bool top = high && static_cast<unsigned>(best) == lo;
        const int e = static_cast<int>(__reduce_min_sync(0xffffffffu, top ? static_cast<unsigned>(lane + 32 * at) : 0xffffffffu));
        const unsigned long long k = static_cast<unsigned long long>(hi) << 32 | lo;
        if (lane == j) chosen = e, mine = k;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (e == lane + 32 * i) key[i] = 0;
      }
      if (lane < p.top) score = q[chosen];
      // The key that another expert may have at most.
      if (first && loss > 0.0) {
        other = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (key[i]) other = fmax(other, unordered(key[i]) + reach(v[i]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) other = fmax(other, __shfl_xor_sync(0xffffffffu, other, o));
      }
    }
    if (!first) break;
    first = false;
    if (live) {
      // Could errors have changed the choice, or its order?  (Keys of infinite size do not move.)
      const double here = unordered(mine), far = reach(score);
      bool close = false;
      if (loss > 0.0) {
        double later = lane < p.top ? here + far : -INFINITY;  // at most, from this choice on
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) later = fmax(later, __shfl_down_sync(0xffffffffu, later, o));
        later = __shfl_down_sync(0xffffffffu, later, 1);
        close = lane < p.top && isfinite(here) && fmax(lane == p.top - 1 ? -INFINITY : later, other) >= here - far;
      }
      const bool nears = __any_sync(0xffffffffu, close);
      const bool odds = __any_sync(0xffffffffu, odd);
      if (nears || odds) {
        // Every logit of a token that holds a NaN is NaN, as the first sums are.
        bool nan = false;
#pragma unroll 1
        for (int k = odds ? 8 * lane : p.K; k < p.K; k += 256) {
          const uint4 c = row_chunk(p.x, static_cast<long long>(t) * p.ldx, k, p.K);
          const uint32_t r[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) nan = nan || isnan(unpack_lo<BF16>(r[i])) || isnan(unpack_hi<BF16>(r[i]));
        }
        if (!__any_sync(0xffffffffu, nan)) {
          // Logits out of range, chosen experts whose key another one's may meet, and those others.  Beside a
          // bias the softmax's denominator does not cancel between two keys, and every expert is part of it.
          const bool all = nears && !p.sigmoid && p.choice_bias;
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (lane + 32 * i < p.E && (all || !isfinite(z[i]))) again |= 1u << i;
#pragma unroll 1
          for (int j = 0; j < (all ? 0 : p.top); ++j) {
            const double kj = __shfl_sync(0xffffffffu, here, j), rj = __shfl_sync(0xffffffffu, far, j);
            const int cj = __shfl_sync(0xffffffffu, chosen, j);
            bool met = false;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const int e = lane + 32 * i;
              if (loss > 0.0 && e < p.E && e != cj && fabs(v[i] + bias[i] - kj) <= rj + reach(v[i])) met = true, again |= 1u << i;
            }
            if (__any_sync(0xffffffffu, met) && lane == cj % 32) again |= 1u << (cj / 32);
          }
        }
      }
    }
    // Sums again in fp64, a few of every warp's at a time, by all warps.
#pragma unroll 1
    while (__syncthreads_or(again != 0)) {
      int asked[kAgainSlots];
#pragma unroll
      for (int c = 0; c < kAgainSlots; ++c) {
        const unsigned who = __ballot_sync(0xffffffffu, again != 0);
        const int src = __ffs(who) - 1;
        asked[c] = who ? src + 32 * (__ffs(__shfl_sync(0xffffffffu, again, max(src, 0))) - 1) : -1;
        if (lane == src) again &= again - 1;
        if (lane == 0) slots[warp * kAgainSlots + c] = asked[c];
      }
      __syncthreads();
#pragma unroll 1
      for (int lot = 0; lot < WARPS * kAgainSlots; lot += 32)
#pragma unroll 1
        for (unsigned todo = __ballot_sync(0xffffffffu, slots[lot + lane] >= 0); todo; todo &= todo - 1) {
          const int i = lot + __ffs(todo) - 1;
          const long long xo = static_cast<long long>(t - warp + i / kAgainSlots) * p.ldx;
          const long long wo = static_cast<long long>(slots[i]) * p.ldw;
          double a = 0.0;
#pragma unroll 2
          for (int k = 8 * threadIdx.x; k < p.K; k += 256 * WARPS)
            a = dot8<BF16>(row_chunk(p.x, xo, k, p.K), row_chunk(p.w, wo, k, p.K), a);
          a = warp_sum(a);
          if (lane == 0) part[i * WARPS + warp] = a;
        }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < kAgainSlots; ++c)
        if (asked[c] >= 0) {
          changed = true;
          double a = 0.0;
#pragma unroll 1
          for (int w = 0; w < WARPS; ++w) a += part[(warp * kAgainSlots + c) * WARPS + w];
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (asked[c] == lane + 32 * i) z[i] = a;
        }
    }
    if (!changed) break;
  }
  if (!live) return;
  const double total = warp_sum(lane < p.top ? score : 0.0);
  if (lane < p.top) {
    ids[lane] = chosen;
    weights[lane] = static_cast<float>((p.renormalize ? score / total : score) * static_cast<double>(p.scale));
  }
}

// K steps first, first + stride, ... below `end` of 16 MT x 8 NT logits (and of their sums |x w|), in
// the MMA's lane layout: value v of tile (i, j) is token 16 i + 8 (v / 2) + g, expert 8 j + 2 q + v % 2.
template <bool BF16, bool W32, int MT, int NT>
__device__ __forceinline__ void route_sums(const RouteParams& p, int t0, int e0, int first, int stride, int end, int lane,
                                           double (&z)[MT][NT][4], float (&sa)[MT][NT][4]) {
  const int g = lane >> 2, q = lane & 3;
  if constexpr (!W32) {
    long long xo[2 * MT], wo[NT];  // rows past the last token or expert repeat it; nobody reads their sums
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) xo[i] = static_cast<long long>(min(t0 + 8 * i + g, p.M - 1)) * p.ldx;
#pragma unroll
    for (int j = 0; j < NT; ++j) wo[j] = static_cast<long long>(min(e0 + 8 * j + g, p.E - 1)) * p.ldw;
#pragma unroll(MT == 1 ? 4 : 1)
    for (int s = first; s < end; s += stride) {
      const int k0 = s * kRouteStep;
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
#pragma unroll 1
    for (int s = first; s < end; s += stride)
#pragma unroll 4
      for (int k = s * kRouteStep; k < min((s + 1) * kRouteStep, p.K); ++k) {
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
}

// Part `kp` of `parts` of K of a tile by a CTA of WARPS warps: each takes every WARPS-th step, their
// sums are added in warp order and go to part kp of the scratch.
template <bool BF16, bool W32, int MT, int NT, int WARPS>
__device__ __forceinline__ void route_tile(const RouteParams& p, int t0, int e0, int kp, int parts, uint8_t* smem) {
  double* part = reinterpret_cast<double*>(smem);  // [warps][16 MT][8 NT], then the |x w| sums
  float* part_s = reinterpret_cast<float*>(part + WARPS * 128 * MT * NT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int steps = (p.K + kRouteStep - 1) / kRouteStep;
  double z[MT][NT][4] = {};
  float sa[MT][NT][4] = {};
  route_sums<BF16, W32, MT, NT>(p, t0, e0, steps * kp / parts + warp, WARPS, steps * (kp + 1) / parts, lane, z, sa);
  constexpr int kCols = 8 * NT, kCells = 128 * MT * NT;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int cell = (16 * i + 8 * (v / 2) + g) * kCols + 8 * j + 2 * q + v % 2;
        part[warp * kCells + cell] = z[i][j][v];
        part_s[warp * kCells + cell] = sa[i][j][v];
      }
  __syncthreads();
  for (int cell = threadIdx.x; cell < kCells; cell += 32 * WARPS) {
    const int t = t0 + cell / kCols, e = e0 + cell % kCols;
    double sum = 0.0;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      sum += part[w * kCells + cell];
      s += part_s[w * kCells + cell];
    }
    if (t < p.M && e < p.E) {
      const size_t at = (static_cast<size_t>(kp) * p.M + t) * p.E + e;
      __stcg(p.logits + at, sum);
      __stcg(p.sums + at, s);
    }
  }
  __syncthreads();
}

template <bool BF16, bool W32, int MT, int NT, int PER>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const RouteParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int last;
  const int warp = threadIdx.x >> 5;
  // Tiles in one grid dimension, which takes any number of tokens, neighbours with the same tokens.
  const unsigned groups = (p.E + 8 * NT - 1) / (8 * NT), tile = blockIdx.x / groups, group = blockIdx.x - tile * groups;
  const int t0 = static_cast<int>(tile) * 16 * MT;
  if (threadIdx.x == 0) grid_dep_launch();
  grid_dep_wait();
  route_tile<BF16, W32, MT, NT, kRouteWarps>(p, t0, static_cast<int>(group) * 8 * NT, 0, 1, smem);
  if (threadIdx.x == 0) {
    unsigned old;  // (releases what the whole CTA wrote: the barrier above)
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(p.counters + tile) : "memory");
    last = old == groups - 1;
    if (last) p.counters[tile] = 0;  // for the next launch
  }
  __syncthreads();
  if (!last) return;
#pragma unroll 1
  for (int t = t0; t < min(t0 + 16 * MT, p.M); t += kRouteWarps) {  // (the parts have been added up)
    route_tokens<BF16, PER, kRouteWarps>(p, t + warp, smem);
    __syncthreads();
  }
}

// ---- many tokens -----------------------------------------------------------------------------
constexpr int kLogitTile = 64;                            // tokens and experts of a tile
constexpr int kLogitStages = 3;
constexpr int kLogitChains = 2;                           // K steps of 64 in a stage (one per barrier: 37.8 us, two 36.3)
constexpr int kLogitPart = kLogitTile * kRouteStep * 2;   // bytes: 64 x 64 of x or of w
constexpr int kLogitStage = 2 * kLogitChains * kLogitPart;
constexpr int kLogitSmem = kLogitStages * kLogitStage;

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, int bytes) {  // the rest is zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_u4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Part blockIdx.y of K of a 64 x 64 tile of logits (blockIdx.x, as in route_kernel): warps 2 x 4, each 32
// tokens x 16 experts (warps 0 and 1 the first 16 experts, even warps the first 32 tokens).
template <bool BF16>
__global__ void __launch_bounds__(kRouteThreads, 2) route_logits_kernel(const RouteParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const unsigned groups = (p.E + kLogitTile - 1) / kLogitTile, tile = blockIdx.x / groups, group = blockIdx.x - tile * groups;
  const int t0 = static_cast<int>(tile) * kLogitTile, e0 = static_cast<int>(group) * kLogitTile;
  const int steps = (p.K + kLogitChains * kRouteStep - 1) / (kLogitChains * kRouteStep);
  const int s0 = steps * blockIdx.y / gridDim.y, s1 = steps * (blockIdx.y + 1) / gridDim.y;
  if (threadIdx.x == 0) grid_dep_launch();
  grid_dep_wait();
  // Thread i copies 16-byte chunk i % 8 of rows i / 8 and i / 8 + 32 of both operands; rows past the
  // last repeat it.  Chunk c of row r lies at c ^ 4 (r % 2): eight lanes read the same half of two rows.
  const int row = threadIdx.x >> 3, chunk = threadIdx.x & 7;
  auto load = [&](int step, int slot) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row + 32 * h;
      const long long x = static_cast<long long>(min(t0 + r, p.M - 1)) * p.ldx, w = static_cast<long long>(min(e0 + r, p.E - 1)) * p.ldw;
#pragma unroll
      for (int c = 0; c < kLogitChains; ++c) {
        const int k = (step * kLogitChains + c) * kRouteStep + 8 * chunk;
        const int bytes = max(0, min(16, 2 * (p.K - k)));
        const uint32_t dst = base + slot * kLogitStage + 2 * c * kLogitPart + r * 128 + ((chunk ^ (4 * (r & 1))) << 4);
        copy_async16(dst, static_cast<const uint16_t*>(p.x) + x + (bytes ? k : 0), bytes);
        copy_async16(dst + kLogitPart, static_cast<const uint16_t*>(p.w) + w + (bytes ? k : 0), bytes);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kLogitStages - 1; ++i) {
    if (s0 + i < s1) load(s0 + i, i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const int m0 = (warp & 1) * 32, n0 = (warp >> 1) * 16;  // of the tile
  // Squares of the rows this warp has in hand anyway: tokens in the first column of tiles, experts in the first row.
  const bool x_norm = group == 0 && warp < 2, w_norm = tile == 0 && (warp & 1) == 0;
  float x2[4] = {}, w2[2] = {};
  uint32_t xb[4] = {}, wb[2] = {};  // the bits that their values have set: squares of small ones vanish
  auto squares = [](const uint4& v, float s, uint32_t& bits) {
    const uint32_t r[4] = {v.x, v.y, v.z, v.w};
    bits |= (v.x | v.y | v.z | v.w) & 0x7FFF7FFFu;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s = fmaf(unpack_lo<BF16>(r[i]), unpack_lo<BF16>(r[i]), s);
      s = fmaf(unpack_hi<BF16>(r[i]), unpack_hi<BF16>(r[i]), s);
    }
    return s;
  };
  double z[2][2][4] = {};
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kLogitStages - 2) : "memory");
    __syncthreads();
    if (s + kLogitStages - 1 < s1) load(s + kLogitStages - 1, (s - s0 + kLogitStages - 1) % kLogitStages);
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
    for (int c = 0; c < kLogitChains; ++c) {
      const uint32_t sx = base + (s - s0) % kLogitStages * kLogitStage + 2 * c * kLogitPart, sw = sx + kLogitPart;
      float d[2][2][4] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 xv[4], wv[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[i] = ld_shared_u4(sx + (m0 + 8 * i + g) * 128 + (((4 * h + q) ^ (4 * (g & 1))) << 4));
#pragma unroll
        for (int j = 0; j < 2; ++j) wv[j] = ld_shared_u4(sw + (n0 + 8 * j + g) * 128 + (((4 * h + q) ^ (4 * (g & 1))) << 4));
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 &a = xv[2 * i], &b = xv[2 * i + 1], &w = wv[j];
            mma_16816<BF16>(d[i][j], a.x, b.x, a.y, b.y, w.x, w.y);
            mma_16816<BF16>(d[i][j], a.z, b.z, a.w, b.w, w.z, w.w);
          }
        if (x_norm) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x2[i] = squares(xv[i], x2[i], xb[i]);
        }
        if (w_norm) {
#pragma unroll
          for (int j = 0; j < 2; ++j) w2[j] = squares(wv[j], w2[j], wb[j]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) z[i][j][v] += static_cast<double>(d[i][j][v]);
    }
  }
  const size_t part = static_cast<size_t>(blockIdx.y) * p.M * p.E;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int t = t0 + m0 + 16 * i + 8 * (v / 2) + g, e = e0 + n0 + 8 * j + 2 * q + v % 2;
        if (t < p.M && e < p.E) p.logits[part + static_cast<size_t>(t) * p.E + e] = z[i][j][v];
      }
  // A row's squares lie with the four lanes of its group; 2^-120 stands for those that vanished.
  float* norms = p.sums + static_cast<size_t>(blockIdx.y) * (p.M + p.E);
  auto put = [&](float s, uint32_t bits, int at, int end, float* to) {
    if (bits && s < 0x1p-120f) s = 0x1p-120f;
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    if (q == 0 && at < end) to[at] = s;
  };
  if (x_norm) {
#pragma unroll
    for (int i = 0; i < 4; ++i) put(x2[i], xb[i], t0 + m0 + 8 * i + g, p.M, norms);
  }
  if (w_norm) {
#pragma unroll
    for (int j = 0; j < 2; ++j) put(w2[j], wb[j], e0 + n0 + 8 * j + g, p.E, norms + p.M);
  }
}

template <bool BF16, int PER>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  if (threadIdx.x == 0) grid_dep_launch();
  grid_dep_wait();
  route_tokens<BF16, PER, kRouteWarps>(p, blockIdx.x * kRouteWarps + (threadIdx.x >> 5), smem);
}

}  // namespace ffnb200
