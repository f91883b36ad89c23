// Weight-streaming kernel for few tokens: the dense projection's small inputs and the routed
// experts of the mixture-of-experts layer.
//
//   projection   Y = act(X . W^T + b) + R
//   experts      hidden_p = act(X_t . W1_e^T) for every (token t, expert e) chosen,
//                Y_t = R_t + sum_j w_tj hidden_p . W2_e^T
//
// With few tokens every weight is used a few times only, so the floor is the weights' bytes over
// HBM bandwidth.  The weight rows are the MMA's A operand (up to 128 rows) and the tokens its N
// columns (a multiple of 16, at most 128); a K step is 64 columns of both, and a ring slot holds
// `blocks` of them (a wait on a barrier costs its thread about 150 clocks, which small slots would
// spend per step).
//
// Routing (experts, if asked for): all CTAs share the router's logits, cut by tokens, experts and K;
// the CTA that arrives last at 16 tokens chooses for them, a warp per token, and everyone waits
// for all choices.  (A launch of its own took 17 to 32 us with cold weights, most of it waiting.
// Every CTA choosing for itself saves two trips to L2, but all read the same lines: 1 token 0.2 us
// less, 7 tokens 2.8 us more.)
// First product (the only one of the projection): the weight rows are dealt out evenly over the
// CTAs (one per SM) in groups -- the projection's rows / CTAs, or 16 rows of an expert -- and a
// CTA takes each of its tiles over the whole of K, so no sum is ever split between CTAs.
// Second product (experts): a line of items x tiles of 128 rows x K steps of 64 is cut into equal
// stretches.  An uncut tile goes to memory whole; of a cut one every CTA leaves its fp32 piece, and
// the final combination over the token's experts adds the pieces in ascending CTA order, which
// keeps results the same from run to run.  It starts when all CTAs have counted (the one
// grid-wide wait; cooperative launch).  A second-product step waits for its item's hidden
// rows; the weight half of the ring (A) runs ahead of that wait, so HBM stays busy across the
// change of product.
//
// Roles: warp 0 weight loads (TMA), warp 1 MMA issue (tcgen05, accumulators in two TMEM halves),
// warp 2 token rows (TMA; the experts' first product gathers four per instruction), warps 4-7
// epilogue.  Each of the first three is one thread that its warp elects: TMA and MMA instructions
// then issue every 12 to 35 clocks, where they took 45 behind a test of the lane number.  Every
// wait is bounded as in ffn_kernel.cuh.
#pragma once

#include "router_kernel.cuh"

namespace ffnb200 {

constexpr int kStreamThreads = 512;  // 8 warps with roles, 8 more for the lists and the combination
constexpr int kStreamMaxStages = 40;
constexpr int kStreamMinSteps = 4;   // fewest K steps of the second product worth a CTA of their own
constexpr int kStreamBarBytes = 1024;

struct StreamParams {
  CUtensorMap tm_w1, tm_w2;  // weights [E][halves][rows][K]: a box is one group's rows (SwiGLU: 8 of
                             // both halves), or 128 rows of the second product
  CUtensorMap tm_x;          // token rows: the projection's in one box, the experts' in boxes of one row
  CUtensorMap tm_x8, tm_x64; // experts, `sorted` not null: its rows in boxes of 8 and 64
  CUtensorMap tm_h8, tm_h64; // hidden rows
  int tokens;
  int groups1, group_rows, group_feats, unit_groups;  // first product: row groups per item, weight rows and
                             // output features of a group, groups of one tile at most
  int steps1, feat1;         // K steps; output features
  int tiles2, steps2, feat2; // second product (experts)
  int slab;                  // bytes of a step's weights in a ring slot (a multiple of 1024)
  int chunk;                 // tokens per item at most (a multiple of 16 up to 128)
  int blocks, stages;        // K steps per ring slot; ring slots
  int act;                   // ffn_b200_gelu
  const uint16_t* bias;      // projection, optional [N]
  const uint16_t* residual;  // optional
  long long ldr;
  uint16_t* y;
  long long ldy;
  const uint16_t* x;         // experts with `sorted`: the token rows, copied to [pair][ldx] in its order
  long long ldx;
  uint16_t* sorted;
  long long lds;
  uint16_t* hidden;          // experts: [pair][ldh], pairs ordered by expert, then token
  long long ldh;
  float* pieces;             // [2 C][chunk][128] pieces of cut tiles of the second product
  float* whole;              // [pair][tiles2 * 128] its uncut tiles
  unsigned* counters;        // kStreamSync words, then the items' finished groups
  int* status;
  const int* ids;            // experts: [tokens][top]
  const float* weights;
  int experts, top;
  int routed;                // 1: the kernel chooses the experts itself (into ids and weights)
  RouteParams route;         // counters: of 16 tokens each, then the choices made
  unsigned long long wait_limit_ns;
  int inject;
};
constexpr int kStreamSync = 3;  // CTAs done with the second product; CTAs done with the counters; CTAs done with `sorted`

// Shared memory behind the ring and barriers for the experts' lists.
struct StreamLists {
  int words;          // u32 words of an expert's token set
  int sets, first, offset, item, token, bytes;  // byte offsets
  __host__ __device__ StreamLists(int tokens, int experts, int top, int chunk) {
    words = (tokens + 31) / 32;
    const int pairs = tokens * top;
    sets = 0;
    offset = sets + experts * words * 4;      // u16 [E + 1]: pairs before expert e
    first = offset + (experts + 1) * 2;       // u16 [E + 1]: items before expert e
    item = (first + (experts + 1) * 2 + 7) & ~7;  // uint2 per item: expert | count << 16, first pair
    token = item + 8 * most_items(tokens, experts, top, chunk);  // u16 per pair: its token
    bytes = (token + pairs * 2 + 15) & ~15;
  }
  // Items at most: one per chosen expert, and one more for each full chunk of pairs.
  __host__ __device__ static int most_items(int tokens, int experts, int top, int chunk) {
    const int pairs = tokens * top;
    return (experts < pairs ? experts : pairs) + pairs / chunk;
  }
};

// `total` things in a line dealt out over at most `grid` CTAs in stretches that differ by one at most, of at
// least `least` each.  (32-bit divisions: every role does this before its first load or wait.)
struct StreamSplit {
  unsigned ctas, each, more;  // the first `more` CTAs take each + 1
  __device__ StreamSplit(unsigned total, unsigned grid, unsigned least) {
    const unsigned most = total / least;
    ctas = most < 1u ? 1u : (most < grid ? most : grid);
    each = total / ctas;
    more = total - each * ctas;
  }
  __device__ int begin(unsigned c) const {
    c = min(c, ctas);
    return static_cast<int>(c * each + min(c, more));
  }
  __device__ int cta_of(unsigned i) const {
    const unsigned big = more * (each + 1);
    return static_cast<int>(i < big ? i / (each + 1) : more + (i - big) / each);
  }
};

// Four gathered rows (64 columns from c0) into 512 consecutive bytes of a 128B-swizzled tile.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* tm, int c0, int r0, int r1, int r2, int r3,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, int c3,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_hint(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, int c3,
                                                 uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar), "l"(policy)
      : "memory");
}
// One lane of a converged warp, as the compiler knows a single one.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r != 0;
}
// All 128 epilogue threads meet; true when every one brought true.
__device__ __forceinline__ int epilogue_all(int ok) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 q, %1, 0;\n\t"
      "barrier.cta.red.and.pred p, 1, 128, q;\n\t"
      "selp.s32 %0, 1, 0, p;\n\t}\n"
      : "=r"(r)
      : "r"(ok)
      : "memory");
  return r;
}
__device__ __forceinline__ unsigned atom_add_acq_rel(unsigned* p, unsigned v) {
  unsigned old;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}
template <int W>
__device__ __forceinline__ void apply_act(float* v, int act) {
  if (act == 0) {
#pragma unroll
    for (int j = 0; j < W; j += 2) gelu_rational2(v[j], v[j + 1]);
  } else if (act == 1) {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = gelu_erf(v[j]);
  } else if (act == 2) {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = silu(v[j]);
  }
}
__device__ __forceinline__ bool stream_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                            const StreamParams& p, int aux) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = gtimer();
  uint32_t n = 0;
#pragma unroll 1
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++n & 15u) == 0) {
      if (*abort_flag) return false;
      if (gtimer() - t0 > 2 * p.wait_limit_ns) {  // twice the cross-CTA limit: the cause reports first
        if (p.status && atomicCAS(p.status, 0, 1) == 0) p.status[1] = blockIdx.x, p.status[2] = aux;
        *abort_flag = 1;
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool stream_wait_word(const unsigned* word, unsigned target, volatile int* abort_flag,
                                                 const StreamParams& p, int code, int aux) {
  if (ld_acquire(word) >= target) return true;
  const uint64_t t0 = gtimer();
#pragma unroll 1
  while (true) {
    __nanosleep(32);
    if (ld_acquire(word) >= target) return true;
    if (*abort_flag) return false;
    if (gtimer() - t0 > p.wait_limit_ns) {
      if (p.status && atomicCAS(p.status, 0, code) == 0) p.status[1] = blockIdx.x, p.status[2] = aux;
      *abort_flag = 1;
      return false;
    }
  }
}

template <bool BF16, bool MOE>
__global__ void __launch_bounds__(kStreamThreads, 1) stream_kernel(const __grid_constant__ StreamParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const int ST = p.stages;
  const uint32_t slab = static_cast<uint32_t>(p.slab);
  const uint32_t token_bytes = static_cast<uint32_t>(p.chunk) * 128u;
  const int KS = p.blocks;
  const uint32_t stage_bytes = KS * (slab + token_bytes);
  const uint32_t sBar = base + ST * stage_bytes;
  uint8_t* ctrl = gbase + ST * stage_bytes;
  auto full_bar = [&](int s) { return sBar + 8u * s; };
  auto empty_bar = [&](int s) { return sBar + 8u * (kStreamMaxStages + s); };
  auto acc_full = [&](int b) { return sBar + 8u * (2 * kStreamMaxStages + b); };
  auto acc_empty = [&](int b) { return sBar + 8u * (2 * kStreamMaxStages + 2 + b); };
  const uint32_t drain_bar = sBar + 8u * (2 * kStreamMaxStages + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 8 * (2 * kStreamMaxStages + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* last_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);
  int* n_items = reinterpret_cast<int*>(tmem_slot + 3);
  int* n_pairs = n_items + 1;
  int* warp_sums = n_items + 2;  // [16] x 2
  const StreamLists lists(p.tokens, MOE ? p.experts : 0, MOE ? p.top : 0, p.chunk);
  uint8_t* lbase = ctrl + kStreamBarBytes;
  unsigned* sets = reinterpret_cast<unsigned*>(lbase + lists.sets);
  uint16_t* offset = reinterpret_cast<uint16_t*>(lbase + lists.offset);
  uint16_t* first = reinterpret_cast<uint16_t*>(lbase + lists.first);
  uint2* item_list = reinterpret_cast<uint2*>(lbase + lists.item);
  uint16_t* token_of = reinterpret_cast<uint16_t*>(lbase + lists.token);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int c = blockIdx.x;
  const int C = gridDim.x;
  const uint32_t tmem_cols = p.chunk <= 16 ? 32u : (p.chunk <= 32 ? 64u : (p.chunk <= 64 ? 128u : 256u));  // two accumulators

  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int s = 0; s < ST; ++s) {
      mbar_init(full_bar(s), 2);  // the weight load's and the token rows' arrivals
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 4);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    *n_items = 1;
    fence_barrier_init();
    fence_async_shared();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&p.tm_w1);
    prefetch_tmap(MOE && p.sorted ? &p.tm_x8 : &p.tm_x);
    if (MOE) {
      prefetch_tmap(&p.tm_w2);
      prefetch_tmap(&p.tm_h8);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), tmem_cols);
    tmem_relinquish();
  }
  if (MOE)
    for (int i = threadIdx.x; i < p.experts * lists.words; i += kStreamThreads) sets[i] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (threadIdx.x == 0) grid_dep_launch();
  grid_dep_wait();

  if constexpr (MOE) {
    if (p.routed) {
      const RouteParams& r = p.route;
      constexpr int kWarps = kStreamThreads / 32;
      static_assert(kWarps == 16, "a warp per token of a tile");
      const int groups = (p.experts + 7) / 8, tiles = (p.tokens + 15) / 16;
      const int units = groups * tiles * r.parts;
#pragma unroll 1
      for (int u = c; u < units; u += C) {  // (token tile fastest: its CTAs share weights)
        const int tile = u % tiles, v = u / tiles, group = v % groups, kp = v / groups;
        if (r.weight_f32) route_tile<BF16, true, 1, 1, kWarps>(r, tile * 16, group * 8, kp, r.parts, gbase);
        else route_tile<BF16, false, 1, 1, kWarps>(r, tile * 16, group * 8, kp, r.parts, gbase);
        if (threadIdx.x == 0)  // (releases what the whole CTA wrote: the barrier above)
          *last_flag = atom_add_acq_rel(r.counters + tile, 1u) == static_cast<unsigned>(groups * r.parts - 1);
        __syncthreads();
        if (*last_flag) {
          const int t = tile * 16 + warp;
          if (p.experts <= 64) route_tokens<BF16, 2, kWarps>(r, t, gbase);
          else if (p.experts <= 256) route_tokens<BF16, 8, kWarps>(r, t, gbase);
          else route_tokens<BF16, 16, kWarps>(r, t, gbase);
          __syncthreads();
          if (threadIdx.x == 0) red_release_add(r.counters + tiles, 1u);
        }
        __syncthreads();
      }
      if (threadIdx.x == 0) stream_wait_word(r.counters + tiles, static_cast<unsigned>(tiles), abort_flag, p, 2, -2);
      fence_async_shared();  // the ring's bytes were used above; TMA writes them next
      __syncthreads();
    }
    // Pairs (token, expert) ordered by expert, then token: each expert's tokens as a bit set, so
    // that every CTA finds the same order whatever order its threads run in.  A token that names
    // an expert twice is one pair; an id outside [0, experts) is none.
    const int pairs = p.tokens * p.top;
    for (int i = threadIdx.x; i < pairs; i += kStreamThreads) {
      const int e = __ldcg(p.ids + i);
      const int t = i / p.top;
      if (static_cast<unsigned>(e) < static_cast<unsigned>(p.experts))
        atomicOr(&sets[e * lists.words + (t >> 5)], 1u << (t & 31));
    }
    __syncthreads();
    // Exclusive sums over the experts of pairs and items; thread i takes expert i.
    static_assert(kStreamThreads >= 512, "one thread per expert");
    const int e = threadIdx.x;
    int cnt = 0;
    if (e < p.experts)
      for (int w = 0; w < lists.words; ++w) cnt += __popc(sets[e * lists.words + w]);
    const int itm = (cnt + p.chunk - 1) / p.chunk;
    int a = cnt, b = itm;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) a += ua, b += ub;
    }
    if (lane == 31) warp_sums[warp] = a, warp_sums[16 + warp] = b;
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < warp; ++w) a += warp_sums[w], b += warp_sums[16 + w];
    if (e < p.experts) {
      offset[e] = static_cast<uint16_t>(a - cnt);
      first[e] = static_cast<uint16_t>(b - itm);
      for (int i = 0; i < itm; ++i)
        item_list[b - itm + i] = make_uint2(static_cast<unsigned>(e) | static_cast<unsigned>(min(p.chunk, cnt - i * p.chunk)) << 16,
                                            static_cast<unsigned>(a - cnt + i * p.chunk));
    }
    if (threadIdx.x == kStreamThreads - 1) *n_items = b, *n_pairs = a;
    __syncthreads();
    for (int i = threadIdx.x; i < p.experts * lists.words; i += kStreamThreads) {
      const int e = i / lists.words, w = i - e * lists.words;
      int at = offset[e];
      for (int v = 0; v < w; ++v) at += __popc(sets[e * lists.words + v]);
      for (unsigned bits = sets[i]; bits; bits &= bits - 1) token_of[at++] = static_cast<uint16_t>(32 * w + __ffs(bits) - 1);
    }
    __syncthreads();
  }

  const int items = *n_items;
  unsigned* sync_words = p.counters;
  unsigned* item_done = sync_words + kStreamSync;
  const bool glu = MOE && p.act == 3;
  auto item_of = [&](int it, int& expert, int& start, int& count) {
    if constexpr (MOE) {
      const uint2 v = item_list[it];
      expert = static_cast<int>(v.x & 0xFFFFu);
      count = static_cast<int>(v.x >> 16);
      start = static_cast<int>(v.y);
    } else {
      expert = 0, start = 0, count = p.tokens;
    }
  };
  // Experts, first product: C / items CTAs per item, or an even deal of all groups, whichever leaves the
  // busiest CTA less to load: its groups (2 KB a step) and, for every tile, the tokens (`chunk` rows
  // of 128 bytes a step); by an even deal a CTA that crosses from one item to the next has a tile
  // more.  (One token, 6 of 64 experts: CTAs per item end 6 us earlier; 64 tokens: 12 us later.)
  const int per_item = max(1, MOE && items ? C / items : 1);
  const int most_whole = (p.groups1 + per_item - 1) / per_item, most_even = (items * p.groups1 + C - 1) / C;
  const int row_cost = (p.chunk + 15) / 16;
  const bool whole_items = items > 0 && items <= C &&
                           most_whole + row_cost * ((most_whole + p.unit_groups - 1) / p.unit_groups) <=
                               most_even + row_cost * ((most_even + p.unit_groups - 1) / p.unit_groups + 1);
  // Projection with at most 64 weight rows per CTA: MMAs of 64 rows, 25 clocks each instead of 42 (1 x
  // 4096 x 4096: 28 rows).  Row r of them lies in TMEM lane 32 (r / 16) + r % 16.
  const bool half_tile = !MOE && p.group_rows <= 64;
  // This CTA's tiles, in the same order for every role: tile(ph, item, g0, groups, k0, k1) returns
  // false to stop.  First product: groups [g0, g0 + groups) of the item over all of K.  Second:
  // tile g0, K steps [k0, k1).
  auto for_tiles = [&](auto&& tile) {
    if (items == 0) return;
    const StreamSplit rows(items * p.groups1, C, 1);
    int g = rows.begin(c), end = rows.begin(c + 1);
    if (MOE && whole_items) {
      // Few items: each gets CTAs of its own, so that none has two short tiles instead of one.
      const int it = c / per_item;
      const StreamSplit one(p.groups1, per_item, 1);
      g = end = 0;
      if (it < items) {
        g = it * p.groups1 + one.begin(c - it * per_item);
        end = it * p.groups1 + one.begin(c - it * per_item + 1);
      }
    }
    while (g < end) {
      const int it = g / p.groups1, g0 = g - it * p.groups1;
      const int n = min(min(p.unit_groups, p.groups1 - g0), end - g);
      if (!tile(0, it, g0, n, 0, p.steps1)) return;
      g += n;
    }
    if constexpr (MOE) {
      const StreamSplit line(items * p.tiles2 * p.steps2, C, kStreamMinSteps);
      for (int s = line.begin(c), end = line.begin(c + 1); s < end;) {
        const int u = s / p.steps2, k0 = s - u * p.steps2, k1 = min(p.steps2, k0 + end - s);
        const int it = u / p.tiles2;
        if (!tile(1, it, u - it * p.tiles2, 1, k0, k1)) return;
        s += k1 - k0;
      }
    }
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ weight loads
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      const uint32_t box_bytes = static_cast<uint32_t>(p.group_rows) * 128u;
      // Experts' weights leave L2 first: another call chooses others (229 -> 225 us for 16 tokens, 4 of 32
      // experts).  A projection's may stay until its next call (11.5 us with the hint, 11.3 without).
      const uint64_t policy = policy_evict_first();
      for_tiles([&](int ph, int it, int g0, int n, int k0, int k1) {
        int expert, start, count;
        item_of(it, expert, start, count);
        const uint32_t bytes = ph ? static_cast<uint32_t>(kABytes) : box_bytes * n;
#pragma unroll 1
        for (int kb = k0; kb < k1; kb += KS) {
          const int nb = min(KS, k1 - kb);
          if (!stream_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, 100 + stage)) return false;
          const uint32_t dst = base + stage * stage_bytes;
          mbar_expect_tx(full_bar(stage), bytes * nb);
#pragma unroll 1
          for (int i = 0; i < nb; ++i) {
            if (MOE && ph) {
              tma_load_4d_hint(dst + i * slab, &p.tm_w2, (kb + i) * kBK, g0 * kBM, 0, expert, full_bar(stage), policy);
            } else if (MOE) {
#pragma unroll 1
              for (int j = 0; j < n; ++j)
                tma_load_4d_hint(dst + i * slab + j * box_bytes, &p.tm_w1, (kb + i) * kBK, (g0 + j) * p.group_feats, 0, expert,
                                 full_bar(stage), policy);
            } else {
#pragma unroll 1
              for (int j = 0; j < n; ++j)
                tma_load_4d(dst + i * slab + j * box_bytes, &p.tm_w1, (kb + i) * kBK, (g0 + j) * p.group_feats, 0, expert,
                            full_bar(stage));
            }
          }
          ++issued;
          if (++stage == ST) { stage = 0; phase ^= 1u; }
        }
        return true;
      });
      // Every load lands before the CTA may leave.  After an abort the token rows of a slot may
      // never have been asked for and its barrier never completes: a millisecond then.
      const uint64_t t0 = gtimer();
      bool late = false;
      for (long long i = issued > ST ? issued - ST : 0; i < issued && !late; ++i)
        while (!mbar_try_wait(full_bar(static_cast<int>(i % ST)), static_cast<uint32_t>((i / ST) & 1)))
          if (gtimer() - t0 > p.wait_limit_ns || (*abort_flag && gtimer() - t0 > 1000000ull)) { late = true; break; }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      int n_acc = 0;
      for_tiles([&](int, int it, int, int, int k0, int k1) {
        int expert, start, count;
        item_of(it, expert, start, count);
        const uint32_t idesc =
            (half_tile ? make_idesc<BF16, 0, 64>() : make_idesc<BF16, 0, kBM>()) | static_cast<uint32_t>((count + 15) / 16 * 2) << 17;
        const int b = n_acc & 1;
        if (!stream_wait(acc_empty(b), ((n_acc >> 1) & 1) ^ 1u, abort_flag, p, 200 + b)) return false;
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(b * p.chunk);
#pragma unroll 1
        for (int kb = k0; kb < k1; kb += KS) {
          const int nb = min(KS, k1 - kb);
          if (!stream_wait(full_bar(stage), phase, abort_flag, p, 300 + stage)) return false;
          tc_fence_after();
          // (A tile of fewer than 128 rows reads on into what lies behind: its TMEM lanes are not used.)
          uint64_t da = sw128_desc(base + stage * stage_bytes);
          uint64_t db = sw128_desc(base + stage * stage_bytes + KS * slab);
#pragma unroll 1
          for (int i = 0; i < nb; ++i) {
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k)
              umma_f16(d, da + 2 * k, db + 2 * k, idesc, kb > k0 || i > 0 || k > 0 ? 1u : 0u);
            da += slab >> 4;
            db += token_bytes >> 4;
          }
          umma_commit(empty_bar(stage));
          if (++stage == ST) { stage = 0; phase ^= 1u; }
        }
        umma_commit(acc_full(b));
        ++n_acc;
        return true;
      });
      umma_commit(drain_bar);
      const uint64_t t0 = gtimer();
      while (!mbar_try_wait(drain_bar, 0))
        if (gtimer() - t0 > p.wait_limit_ns) break;
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ token rows
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for_tiles([&](int ph, int it, int, int, int k0, int k1) {
        int expert, start, count;
        item_of(it, expert, start, count);
        if (MOE && (ph || p.sorted)) {
          ok = ph ? stream_wait_word(item_done + it, static_cast<unsigned>(p.groups1 + (p.inject ? 1 : 0)), abort_flag, p, 2, it)
                  : stream_wait_word(p.counters + 2, static_cast<unsigned>(C), abort_flag, p, 2, -1);
          if (!ok) return false;
          fence_async_global();  // rows written by other CTAs' threads, read by this one's TMA
        }
        const bool gathered = MOE && ph == 0 && !p.sorted;
        // Boxes of 64 rows, of 8 for a remainder of up to 24.  (Rows behind the item's last belong to
        // columns nobody reads.)
        const int wide = count / 64 + (count % 64 > 24 && (count / 64 + 1) * 64 <= p.chunk ? 1 : 0);
        const int narrow = max(0, count - wide * 64 + 7) / 8;
        const uint32_t bytes =
            !MOE ? token_bytes : (gathered ? (count + 3) / 4 * 512u : static_cast<uint32_t>(wide) * 8192u + narrow * 1024u);
        const CUtensorMap* tm8 = ph ? &p.tm_h8 : &p.tm_x8;
        const CUtensorMap* tm64 = ph ? &p.tm_h64 : &p.tm_x64;
#pragma unroll 1
        for (int kb = k0; kb < k1; kb += KS) {
          const int nb = min(KS, k1 - kb);
          ok = stream_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, 150 + stage);
          if (!ok) return false;
          const uint32_t bar = full_bar(stage);
          const uint32_t dst = base + stage * stage_bytes + KS * slab;
          mbar_expect_tx(bar, bytes * nb);
          if (!MOE) {
#pragma unroll 1
            for (int i = 0; i < nb; ++i) tma_load_2d(dst + i * token_bytes, &p.tm_x, (kb + i) * kBK, 0, bar);
          } else if (!gathered) {
#pragma unroll 1
            for (int i = 0; i < nb; ++i) {
#pragma unroll 1
              for (int r = 0; r < wide; ++r)
                tma_load_2d(dst + i * token_bytes + r * 8192, tm64, (kb + i) * kBK, start + 64 * r, bar);
#pragma unroll 1
              for (int r = 0; r < narrow; ++r)
                tma_load_2d(dst + i * token_bytes + wide * 8192 + r * 1024, tm8, (kb + i) * kBK, start + 64 * wide + 8 * r, bar);
            }
          } else {
#pragma unroll 1
            for (int r = 0; r < count; r += 4) {  // (a group that runs past the item repeats its last row)
              const int last = count - 1;
              const int r0 = token_of[start + r], r1 = token_of[start + min(r + 1, last)];
              const int r2 = token_of[start + min(r + 2, last)], r3 = token_of[start + min(r + 3, last)];
#pragma unroll 1
              for (int i = 0; i < nb; ++i)
                tma_gather4(dst + i * token_bytes + r * 128, &p.tm_x, (kb + i) * kBK, r0, r1, r2, r3, bar);
            }
          }
          if (++stage == ST) { stage = 0; phase ^= 1u; }
        }
        return true;
      });
      if (!ok) {  // (token rows asked for before the abort land before the CTA leaves)
        const uint64_t t0 = gtimer();
        while (gtimer() - t0 < 1000000ull) {
        }
      }
    }
  } else if (warp >= 4 && warp < 8) {
    // ------------------------------------------------------------------ epilogue
    const int sub = warp - 4;  // TMEM lane sub-partition
    const uint32_t lane_off = static_cast<uint32_t>(sub * 32) << 16;
    const int row = half_tile ? (lane < 16 ? sub * 16 + lane : kBM) : sub * 32 + lane;  // weight row of the tile
    int n_acc = 0;
    for_tiles([&](int ph, int it, int g0, int n, int k0, int k1) {
      int expert, start, count;
      item_of(it, expert, start, count);
      const int b = n_acc & 1;
      int ok = 1;
      if (lane == 0) ok = stream_wait(acc_full(b), (n_acc >> 1) & 1, abort_flag, p, 400 + b) ? 1 : 0;
      if (!epilogue_all(lane != 0 || ok)) return false;
      tc_fence_after();
      const uint32_t acc = tmem_base + lane_off + static_cast<uint32_t>(b * p.chunk);
      if (MOE && ph == 1) {
        // fp32 sums [token][128 rows]: a piece, or a whole tile.
        size_t pitch = kBM;
        float* dst;
        if (k0 > 0 || k1 < p.steps2) {
          dst = p.pieces + (2 * static_cast<size_t>(c) + (k0 == 0 ? 1 : 0)) * static_cast<size_t>(p.chunk) * kBM;
        } else {
          pitch = static_cast<size_t>(p.tiles2) * kBM;
          dst = p.whole + static_cast<size_t>(start) * pitch + static_cast<size_t>(g0) * kBM;
        }
#pragma unroll 1
        for (int c0 = 0; c0 < count; c0 += 16) {
          float v[16];
          tmem_ld16(acc + c0, v);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < count) __stcg(dst + static_cast<size_t>(c0 + j) * pitch + row, v[j]);
        }
      } else {
        // SwiGLU: of a group's 16 rows the first 8 are gates, the others the matching up rows.
        const int feature = glu ? (g0 + (row >> 4)) * p.group_feats + (row & 7) : g0 * p.group_feats + row;
        const bool live = row < n * p.group_rows && feature < p.feat1;
        const float bias = !MOE && p.bias && live ? unpack_lo<BF16>(static_cast<uint32_t>(__ldg(p.bias + feature))) : 0.f;
        // 8 columns at a time: for few tokens fetching the code costs more than running it.
        uint32_t r[8];
        auto read_ahead = [&](int c0) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            r[j] = p.residual && live && c0 + j < count
                       ? static_cast<uint32_t>(__ldg(p.residual + static_cast<long long>(c0 + j) * p.ldr + feature))
                       : 0u;
        };
        if constexpr (!MOE) read_ahead(0);
#pragma unroll 1
        for (int c0 = 0; c0 < count; c0 += 8) {
          float v[8];
          tmem_ld8(acc + c0, v);
          if constexpr (MOE) {
            if (glu) {
              // Lane l holds a gate row, lane l + 8 the matching up row: of each column pair the
              // lower lane finishes the first, the upper lane the second.
              const bool low = (lane & 8) == 0;
#pragma unroll
              for (int j = 0; j < 8; j += 2) {
                const float got = __shfl_xor_sync(0xffffffffu, low ? v[j + 1] : v[j], 8);
                const float gate = low ? v[j] : got, up = low ? got : v[j + 1];
                const int col = c0 + j + (low ? 0 : 1);
                if (live && col < count)
                  p.hidden[static_cast<long long>(start + col) * p.ldh + feature] = cvt1<BF16>(silu(gate) * up);
              }
            } else {
              apply_act<8>(v, p.act);
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (live && c0 + j < count)
                  p.hidden[static_cast<long long>(start + c0 + j) * p.ldh + feature] = cvt1<BF16>(v[j]);
            }
          } else {
            uint32_t now[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              now[j] = r[j];
              v[j] += bias;
            }
            if (c0 + 8 < count) read_ahead(c0 + 8);
            apply_act<8>(v, p.act);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (live && c0 + j < count)
                p.y[static_cast<long long>(c0 + j) * p.ldy + feature] = cvt1<BF16>(v[j] + unpack_lo<BF16>(now[j]));
          }
        }
        if constexpr (MOE) {
          fence_async_global();  // hidden: written here, read through other CTAs' TMA
          epilogue_all(1);       // (the release below covers what all 128 threads wrote before it)
          if (threadIdx.x == 128) red_release_add(item_done + it, static_cast<unsigned>(n));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty(b));
      ++n_acc;
      return true;
    });
  }

  else if (MOE && warp >= 8 && p.sorted) {
    // ------------------------------------------------------------------ token rows in the pairs' order
    // Dealt out over the CTAs, a warp taking 512 bytes of a row at a time.  The weights, already on
    // their way, hide the grid-wide wait for them.
    const int vecs = static_cast<int>(p.lds / 8), strips = (vecs + 31) / 32;
#pragma unroll 4
    for (int i = (warp - 8) * C + c; i < *n_pairs * strips; i += C * (kStreamThreads / 32 - 8)) {
      const int pair = i / strips, v = (i - pair * strips) * 32 + lane;
      if (v < vecs)
        reinterpret_cast<uint4*>(p.sorted + static_cast<long long>(pair) * p.lds)[v] =
            __ldg(reinterpret_cast<const uint4*>(p.x + static_cast<long long>(token_of[pair]) * p.ldx) + v);
    }
    fence_async_global();  // written here, read through every CTA's TMA
    asm volatile("barrier.cta.sync 2, %0;" ::"n"(kStreamThreads - 256) : "memory");
    if (threadIdx.x == 256) red_release_add(p.counters + 2, 1u);
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, tmem_cols);

  if constexpr (MOE) {
    // Combination: when every CTA's second-product sums are in memory, each warp takes
    // (token, 128 output features) and adds the token's experts in order, each expert's pieces in
    // ascending CTA order, with the fp32 weights, then the residual; rounded once.
    // What the sums do not depend on is looked up before the wait.
    const StreamSplit line(items * p.tiles2 * p.steps2, C, kStreamMinSteps);
    const size_t pitch = static_cast<size_t>(p.tiles2) * kBM;
    const size_t slot = static_cast<size_t>(p.chunk) * kBM;
    const int n_units = p.tokens * p.tiles2;
    // Lane j < top knows choice j: its weight, its pieces and where the first one lies; every lane
    // its four features of the residual.
    struct Share {
      const float* src;
      int pieces, t, f0;
      float wt;
      uint2 res;
    };
    auto look_up = [&](int unit) {
      Share u{nullptr, 0, unit / p.tiles2, 0, 0.f, make_uint2(0u, 0u)};
      if (unit >= n_units) return u;
      const int t = u.t, tile = unit - t * p.tiles2;
      u.f0 = tile * kBM + 4 * lane;
      if (p.residual) {  // (rows are 16-byte aligned and padded to 8 elements: four at a time stay inside)
        const uint16_t* r = p.residual + static_cast<long long>(t) * p.ldr + u.f0;
        if (u.f0 + 4 <= p.feat2) {
          u.res = __ldg(reinterpret_cast<const uint2*>(r));
        } else {
          for (int q = 0; u.f0 + q < p.feat2; ++q)
            (q < 2 ? u.res.x : u.res.y) |= static_cast<uint32_t>(__ldg(r + q)) << (16 * (q & 1));
        }
      }
      if (lane < p.top) {
        const int at = t * p.top + lane;
        const int e = __ldcg(p.ids + at);
        if (static_cast<unsigned>(e) < static_cast<unsigned>(p.experts)) {
          u.wt = __ldcg(p.weights + at);
          int rank = 0;
          for (int w = 0; w < (t >> 5); ++w) rank += __popc(sets[e * lists.words + w]);
          rank += __popc(sets[e * lists.words + (t >> 5)] & ((1u << (t & 31)) - 1u));
          const int chunk_of = rank / p.chunk;
          const int s = ((first[e] + chunk_of) * p.tiles2 + tile) * p.steps2;
          const int c_first = line.cta_of(s);
          u.pieces = line.cta_of(s + p.steps2 - 1) - c_first + 1;
          u.src = u.pieces == 1
                      ? p.whole + static_cast<size_t>(offset[e] + rank) * pitch + static_cast<size_t>(tile) * kBM
                      : p.pieces + (2 * static_cast<size_t>(c_first) + 1) * slot + static_cast<size_t>(rank - chunk_of * p.chunk) * kBM;
        }
      }
      return u;
    };
    if (threadIdx.x == 0) red_release_add(sync_words, 1u);  // (covers the whole CTA's sums: the barrier above)
    int unit = warp * C + c;
    Share now = look_up(unit);
    if (threadIdx.x == 0) {
      if (!*abort_flag) stream_wait_word(sync_words, static_cast<unsigned>(C), abort_flag, p, 3, -1);
      // From here on this CTA reads no counter; the last to say so clears them for the next launch.
      *last_flag = atom_add_acq_rel(sync_words + 1, 1u) == static_cast<unsigned>(C - 1);
    }
    __syncthreads();
    if (!*abort_flag) {
#pragma unroll 1
      for (; unit < n_units; unit += C * (kStreamThreads / 32)) {
        // Four experts' first two pieces in flight at a time, and the next unit's look-up under the
        // first four.  (Piece q > 0 of a cut tile lies in the first slot of CTA c_first + q: 2 q - 1
        // slots behind piece 0.)
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        Share next{};
#pragma unroll 1
        for (int j0 = 0; j0 < p.top; j0 += 4) {
          float4 z[4], z1[4];
          int n[4];
          const float4* at[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = (j0 + i) & 31;  // (lanes from `top` on bring no pieces)
            n[i] = __shfl_sync(0xffffffffu, now.pieces, j);
            at[i] = reinterpret_cast<const float4*>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(now.src), j)) + lane;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            z[i] = n[i] > 0 ? __ldcg(at[i]) : make_float4(0.f, 0.f, 0.f, 0.f);
            z1[i] = n[i] > 1 ? __ldcg(at[i] + slot / 4) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
          if (j0 == 0) next = look_up(unit + C * (kStreamThreads / 32));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            z[i].x += z1[i].x, z[i].y += z1[i].y, z[i].z += z1[i].z, z[i].w += z1[i].w;
#pragma unroll 4
            for (int q = 2; q < n[i]; ++q) {
              const float4 v = __ldcg(at[i] + static_cast<size_t>(2 * q - 1) * (slot / 4));
              z[i].x += v.x, z[i].y += v.y, z[i].z += v.z, z[i].w += v.w;
            }
            const float wj = __shfl_sync(0xffffffffu, now.wt, (j0 + i) & 31);
            if (n[i] > 0) {
              sum.x = fmaf(wj, z[i].x, sum.x), sum.y = fmaf(wj, z[i].y, sum.y);
              sum.z = fmaf(wj, z[i].z, sum.z), sum.w = fmaf(wj, z[i].w, sum.w);
            }
          }
        }
        if (p.residual) {
          sum.x += unpack_lo<BF16>(now.res.x), sum.y += unpack_hi<BF16>(now.res.x);
          sum.z += unpack_lo<BF16>(now.res.y), sum.w += unpack_hi<BF16>(now.res.y);
        }
        uint16_t* y = p.y + static_cast<long long>(now.t) * p.ldy + now.f0;
        const uint2 out = make_uint2(pack2<BF16>(sum.x, sum.y), pack2<BF16>(sum.z, sum.w));
        if (now.f0 + 4 <= p.feat2) {
          *reinterpret_cast<uint2*>(y) = out;
        } else {
          for (int q = 0; now.f0 + q < p.feat2; ++q)
            y[q] = static_cast<uint16_t>((q < 2 ? out.x : out.y) >> (16 * (q & 1)));
        }
        now = next;
      }
    }
    if (*last_flag) {
      for (int i = threadIdx.x; i < items; i += kStreamThreads) item_done[i] = 0;
      if (threadIdx.x < kStreamSync) sync_words[threadIdx.x] = 0;
      if (p.routed && threadIdx.x <= (p.tokens + 15) / 16) p.route.counters[threadIdx.x] = 0;
    }
  }
}

}  // namespace ffnb200
