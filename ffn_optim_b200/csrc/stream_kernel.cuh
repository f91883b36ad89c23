// Weight-streaming kernel for few tokens: the dense projection's small inputs and the routed
// experts of the mixture-of-experts layer.
//
//   projection   Y = act(X . W^T + b) + R
//   experts      hidden_p = act(X_t . W1_e^T) for every (token t, expert e) chosen,
//                Y_t = R_t + sum_j w_tj hidden_p . W2_e^T
//
// With few tokens every weight is used a few times only, so the floor is the weights' bytes over
// HBM bandwidth.  The weight rows are the MMA's 128-row A operand and the tokens its N columns
// (a multiple of 16, at most 128), so one K step of 64 moves 16 KB of weights for one
// 128 x N x 64 product.  All CTAs (one per SM) read equal stretches of the weights:
//
//   A phase is `items` x `tiles` x L steps (item: an expert's tokens, or a chunk of the
//   projection's; tile: 128 weight rows; step: 64 of K) in one line; CTA c takes the stretch
//   [T c / C, T (c+1) / C).  A stretch that covers a tile's whole K goes straight to the epilogue;
//   a tile cut by a stretch's end is summed from fp32 partials in ascending CTA order, which
//   keeps results the same from run to run.
//
//   Projection and experts' first product: every CTA that shares a tile writes its partial and
//   counts up; the one that counts last adds them all and finishes the tile, so nobody waits.
//   Experts' second product: partials are added in the final combination over the token's
//   experts, which starts when all CTAs have counted (the one grid-wide wait; cooperative launch).
//   A second-product step waits for its item's hidden rows; the weight half of the ring (A) runs
//   ahead of that wait, so HBM stays busy across the change of phase.
//
// Roles: warp 0 weight loads (TMA), warp 1 MMA issue (tcgen05, accumulators in two TMEM halves),
// warp 2 token rows (TMA gather of four rows per instruction), warps 4-7 epilogue.  Every wait is
// bounded as in ffn_kernel.cuh.
#pragma once

#include "ffn_kernel.cuh"

namespace ffnb200 {

constexpr int kStreamThreads = 256;
constexpr int kStreamMaxStages = 12;
constexpr int kStreamMinSteps = 4;   // fewest K steps worth a CTA of their own
constexpr int kStreamBarBytes = 512;

struct StreamParams {
  CUtensorMap tm_w1, tm_w2;  // weights [E][halves][rows][K]: box 64 x 128 rows, or 64 x 16 x 2 halves (SwiGLU)
  CUtensorMap tm_x, tm_h;    // token rows, box 64 x 1 (gathered)
  int tokens, items;         // items: the projection's token chunks (experts: found on the device)
  int tiles1, steps1, feat1; // first product: tiles per item, K steps per tile, output features
  int tiles2, steps2, feat2; // second product (experts)
  int chunk, stages;         // tokens per item at most (16, 32, 64 or 128); ring slots
  int act;                   // ffn_b200_gelu
  const uint16_t* bias;      // projection, optional [N]
  const uint16_t* residual;  // optional
  long long ldr;
  uint16_t* y;
  long long ldy;
  uint16_t* hidden;          // experts: [pair][ldh], pairs ordered by expert, then token
  long long ldh;
  float* partial1;           // [2 C][chunk][128] partial tiles of the first product
  float* partial2;           // same for the second
  float* whole2;             // [pair][tiles2 * 128] uncut tiles of the second product
  unsigned* counters;        // [C] arrivals at cut tiles, then kStreamSync words, then items' finished tiles
  int* status;
  const int* ids;            // experts: [tokens][top]
  const float* weights;
  int experts, top;
  unsigned long long wait_limit_ns;
  int inject;
};
constexpr int kStreamSync = 2;  // CTAs done with the second product; CTAs leaving

// Shared memory behind the ring and barriers for the experts' lists.
struct StreamLists {
  int words;          // u32 words of an expert's token set
  int sets, first, offset, item, token, bytes;  // byte offsets
  __host__ __device__ StreamLists(int tokens, int experts, int top) {
    words = (tokens + 31) / 32;
    const int pairs = tokens * top;
    sets = 0;
    offset = sets + experts * words * 4;      // u16 [E + 1]: pairs before expert e
    first = offset + (experts + 1) * 2;       // u16 [E + 1]: items before expert e
    item = (first + (experts + 1) * 2 + 7) & ~7;  // uint2 per item: expert | count << 16, first pair
    token = item + 8 * stream_items(tokens, experts, top);  // u16 per pair: its token
    bytes = (token + pairs * 2 + 15) & ~15;
  }
  // Items at most: one per chosen expert, and one more for each full 128 pairs.
  __host__ __device__ static int stream_items(int tokens, int experts, int top) {
    const int pairs = tokens * top;
    return (experts < pairs ? experts : pairs) + pairs / 128;
  }
};

// One row stretch [s0, s1) of a phase with T steps over `ctas` CTAs, and the CTA of a step.
struct StreamSplit {
  long long T;
  int ctas;
  __device__ StreamSplit(long long total, int grid) : T(total) {
    const long long most = total / kStreamMinSteps;
    ctas = most < 1 ? 1 : (most < grid ? static_cast<int>(most) : grid);
  }
  __device__ int begin(int c) const { return c >= ctas ? static_cast<int>(T) : static_cast<int>(T * c / ctas); }
  __device__ int cta_of(int step) const {
    return static_cast<int>(((static_cast<long long>(step) + 1) * ctas - 1) / T);
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
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == 0) return gelu_rational(z);
  if (act == 1) return gelu_erf(z);
  if (act == 2) return silu(z);
  return z;
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
  const uint32_t stage_bytes = kABytes + static_cast<uint32_t>(p.chunk) * 128u;
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
  int* warp_sums = reinterpret_cast<int*>(tmem_slot + 4);  // [8] x 2
  const StreamLists lists(p.tokens, MOE ? p.experts : 0, MOE ? p.top : 0);
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
  const uint32_t tmem_cols = p.chunk <= 16 ? 32u : 2u * static_cast<uint32_t>(p.chunk);

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
    *n_items = p.items;
    fence_barrier_init();
    fence_async_shared();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&p.tm_w1);
    prefetch_tmap(&p.tm_x);
    if (MOE) {
      prefetch_tmap(&p.tm_w2);
      prefetch_tmap(&p.tm_h);
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
    // Pairs (token, expert) ordered by expert, then token: each expert's tokens as a bit set, so
    // that every CTA finds the same order whatever order its threads run in.  A token that names
    // an expert twice is one pair; an id outside [0, experts) is none.
    const int pairs = p.tokens * p.top;
    for (int i = threadIdx.x; i < pairs; i += kStreamThreads) {
      const int e = __ldg(p.ids + i);
      const int t = i / p.top;
      if (static_cast<unsigned>(e) < static_cast<unsigned>(p.experts))
        atomicOr(&sets[e * lists.words + (t >> 5)], 1u << (t & 31));
    }
    __syncthreads();
    // Exclusive sums over the experts of pairs and items; thread i takes experts 2i and 2i + 1.
    int cnt[2], itm[2];
    for (int q = 0; q < 2; ++q) {
      const int e = 2 * threadIdx.x + q;
      cnt[q] = 0;
      if (e < p.experts)
        for (int w = 0; w < lists.words; ++w) cnt[q] += __popc(sets[e * lists.words + w]);
      itm[q] = (cnt[q] + p.chunk - 1) / p.chunk;
    }
    int a = cnt[0] + cnt[1], b = itm[0] + itm[1];
    const int mine_a = a, mine_b = b;
    for (int o = 1; o < 32; o <<= 1) {
      const int ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) a += ua, b += ub;
    }
    if (lane == 31) warp_sums[warp] = a, warp_sums[8 + warp] = b;
    __syncthreads();
    for (int w = 0; w < warp; ++w) a += warp_sums[w], b += warp_sums[8 + w];
    int pa = a - mine_a, pb = b - mine_b;
    for (int q = 0; q < 2; ++q) {
      const int e = 2 * threadIdx.x + q;
      if (e < p.experts) {
        offset[e] = static_cast<uint16_t>(pa);
        first[e] = static_cast<uint16_t>(pb);
        for (int i = 0; i < itm[q]; ++i)
          item_list[pb + i] = make_uint2(static_cast<unsigned>(e) |
                                             static_cast<unsigned>(min(p.chunk, cnt[q] - i * p.chunk)) << 16,
                                         static_cast<unsigned>(pa + i * p.chunk));
      }
      pa += cnt[q], pb += itm[q];
    }
    if (threadIdx.x == kStreamThreads - 1) *n_items = pb;
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
  unsigned* arrivals = p.counters;
  unsigned* sync_words = p.counters + C;
  unsigned* item_done = sync_words + kStreamSync;
  const int phases = MOE ? 2 : 1;
  // Unit u of a phase: the projection takes its token chunks innermost, so that CTAs next to one
  // another share a weight tile; the experts' units are item-major.
  auto unit_item = [&](int u, int tiles) { return MOE ? u / tiles : u % items; };
  auto unit_tile = [&](int u, int tiles) { return MOE ? u % tiles : u / items; };
  auto item_of = [&](int it, int& expert, int& start, int& count) {
    if constexpr (MOE) {
      const uint2 v = item_list[it];
      expert = static_cast<int>(v.x & 0xFFFFu);
      count = static_cast<int>(v.x >> 16);
      start = static_cast<int>(v.y);
    } else {
      expert = 0;
      start = it * p.chunk;
      count = min(p.chunk, p.tokens - start);
    }
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ weight loads
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
#pragma unroll 1
      for (int ph = 0; ph < phases && ok; ++ph) {
        const int tiles = ph ? p.tiles2 : p.tiles1, L = ph ? p.steps2 : p.steps1;
        const StreamSplit split(static_cast<long long>(items) * tiles * L, C);
        const int end = items ? split.begin(c + 1) : 0;
        int s = items ? split.begin(c) : 0;
        const CUtensorMap* tm = ph ? &p.tm_w2 : &p.tm_w1;
        const bool glu = ph == 0 && p.act == 3;
#pragma unroll 1
        while (s < end && ok) {
          const int u = s / L, k0 = s - u * L, k1 = min(L, k0 + end - s);
          int expert, start, count;
          item_of(unit_item(u, tiles), expert, start, count);
          const int tile = unit_tile(u, tiles);
#pragma unroll 1
          for (int kb = k0; kb < k1; ++kb) {
            if (!stream_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, 100 + stage)) { ok = false; break; }
            const uint32_t dst = base + stage * stage_bytes;
            mbar_expect_tx(full_bar(stage), kABytes);
            if (glu) {  // rows 32 w + (0..15) gate, (16..31) up: a warp's TMEM lanes hold both
#pragma unroll
              for (int w = 0; w < 4; ++w)
                tma_load_4d(dst + w * 4096, tm, kb * kBK, tile * 64 + 16 * w, 0, expert, full_bar(stage));
            } else {
              tma_load_4d(dst, tm, kb * kBK, tile * kBM, 0, expert, full_bar(stage));
            }
            ++issued;
            if (++stage == ST) { stage = 0; phase ^= 1u; }
          }
          s += k1 - k0;
        }
      }
      // Every load lands before the CTA may leave.  After an abort the token rows of a slot may
      // never have been asked for and its barrier never completes: wait for the limit then.
      const uint64_t t0 = gtimer();
      bool late = false;
      for (long long i = issued > ST ? issued - ST : 0; i < issued && !late; ++i)
        while (!mbar_try_wait(full_bar(static_cast<int>(i % ST)), static_cast<uint32_t>((i / ST) & 1)))
          if (gtimer() - t0 > p.wait_limit_ns || (*abort_flag && gtimer() - t0 > 1000000ull)) { late = true; break; }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int n_acc = 0;
      bool ok = true;
#pragma unroll 1
      for (int ph = 0; ph < phases && ok; ++ph) {
        const int tiles = ph ? p.tiles2 : p.tiles1, L = ph ? p.steps2 : p.steps1;
        const StreamSplit split(static_cast<long long>(items) * tiles * L, C);
        const int end = items ? split.begin(c + 1) : 0;
        int s = items ? split.begin(c) : 0;
#pragma unroll 1
        while (s < end && ok) {
          const int u = s / L, k0 = s - u * L, k1 = min(L, k0 + end - s);
          int expert, start, count;
          item_of(unit_item(u, tiles), expert, start, count);
          const uint32_t idesc = make_idesc<BF16, 0, kBM>() | static_cast<uint32_t>((count + 15) / 16 * 2) << 17;
          const int b = n_acc & 1;
          if (!stream_wait(acc_empty(b), ((n_acc >> 1) & 1) ^ 1u, abort_flag, p, 200 + b)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + static_cast<uint32_t>(b * p.chunk);
#pragma unroll 1
          for (int kb = k0; kb < k1; ++kb) {
            if (!stream_wait(full_bar(stage), phase, abort_flag, p, 300 + stage)) { ok = false; break; }
            tc_fence_after();
            const uint64_t da = sw128_desc(base + stage * stage_bytes);
            const uint64_t db = sw128_desc(base + stage * stage_bytes + kABytes);
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) umma_f16(d, da + 2 * k, db + 2 * k, idesc, kb > k0 || k > 0 ? 1u : 0u);
            umma_commit(empty_bar(stage));
            if (++stage == ST) { stage = 0; phase ^= 1u; }
          }
          if (!ok) break;
          umma_commit(acc_full(b));
          ++n_acc;
          s += k1 - k0;
        }
      }
      umma_commit(drain_bar);
      const uint64_t t0 = gtimer();
      while (!mbar_try_wait(drain_bar, 0))
        if (gtimer() - t0 > p.wait_limit_ns) break;
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ token rows
    int stage = 0;
    uint32_t phase = 0;
    int ok = 1;
#pragma unroll 1
    for (int ph = 0; ph < phases && ok; ++ph) {
      const int tiles = ph ? p.tiles2 : p.tiles1, L = ph ? p.steps2 : p.steps1;
      const StreamSplit split(static_cast<long long>(items) * tiles * L, C);
      const int end = items ? split.begin(c + 1) : 0;
      int s = items ? split.begin(c) : 0;
      const CUtensorMap* tm = ph ? &p.tm_h : &p.tm_x;
#pragma unroll 1
      while (s < end && ok) {
        const int u = s / L, k0 = s - u * L, k1 = min(L, k0 + end - s);
        int expert, start, count;
        const int it = unit_item(u, tiles);
        item_of(it, expert, start, count);
        const int groups = (count + 3) / 4;
        int r[4];  // this lane's four rows; a group that runs past the item repeats its last row
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = start + min(4 * lane + j, count - 1);
          r[j] = MOE && ph == 0 ? token_of[at] : at;
        }
        if (MOE && ph == 1) {
          if (lane == 0)
            ok = stream_wait_word(item_done + it, static_cast<unsigned>(p.tiles1 + (p.inject ? 1 : 0)), abort_flag, p, 2, it);
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          fence_async_global();  // hidden rows written by other CTAs' threads, read by this one's TMA
        }
#pragma unroll 1
        for (int kb = k0; kb < k1; ++kb) {
          if (lane == 0) ok = stream_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, 120 + stage) ? 1 : 0;
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(full_bar(stage), static_cast<uint32_t>(groups) * 512u);
          __syncwarp();
          if (lane < groups)
            tma_gather4(base + stage * stage_bytes + kABytes + lane * 512u, tm, kb * kBK, r[0], r[1], r[2], r[3],
                        full_bar(stage));
          if (++stage == ST) { stage = 0; phase ^= 1u; }
        }
        s += k1 - k0;
      }
    }
    if (!ok) {  // (token rows asked for before the abort land before the CTA leaves)
      const uint64_t t0 = gtimer();
      while (gtimer() - t0 < 1000000ull) {
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue
    const int sub = warp - 4;  // TMEM lane sub-partition
    const uint32_t lane_off = static_cast<uint32_t>(sub * 32) << 16;
    const int row = sub * 32 + lane;  // weight row of the tile
    int n_acc = 0;
    int ok = 1;
#pragma unroll 1
    for (int ph = 0; ph < phases && ok; ++ph) {
      const int tiles = ph ? p.tiles2 : p.tiles1, L = ph ? p.steps2 : p.steps1;
      const StreamSplit split(static_cast<long long>(items) * tiles * L, C);
      const int end = items ? split.begin(c + 1) : 0;
      int s = items ? split.begin(c) : 0;
#pragma unroll 1
      while (s < end && ok) {
        const int u = s / L, k0 = s - u * L, k1 = min(L, k0 + end - s);
        int expert, start, count;
        const int it = unit_item(u, tiles), tile = unit_tile(u, tiles);
        item_of(it, expert, start, count);
        const int b = n_acc & 1;
        if (lane == 0) ok = stream_wait(acc_full(b), (n_acc >> 1) & 1, abort_flag, p, 400 + b) ? 1 : 0;
        ok = epilogue_all(lane != 0 || ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tmem_base + lane_off + static_cast<uint32_t>(b * p.chunk);
        const bool cut = k0 > 0 || k1 < L;
        if (cut || (MOE && ph == 1)) {
          // Partial sums, or an uncut tile of the experts' second product: [token][128 rows] fp32.
          float* dst;
          size_t pitch = kBM;
          if (cut) {
            dst = (ph ? p.partial2 : p.partial1) +
                  (2 * static_cast<size_t>(c) + (k0 == 0 ? 1 : 0)) * static_cast<size_t>(p.chunk) * kBM;
          } else {
            pitch = static_cast<size_t>(p.tiles2) * kBM;
            dst = p.whole2 + static_cast<size_t>(start) * pitch + static_cast<size_t>(tile) * kBM;
          }
#pragma unroll 1
          for (int c0 = 0; c0 < count; c0 += 16) {
            float v[16];
            tmem_ld16(acc + c0, v);
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (c0 + j < count) __stcg(dst + static_cast<size_t>(c0 + j) * pitch + row, v[j]);
          }
        }
        int finish = !cut && !(MOE && ph == 1);
        int c_first = c, c_last = c;
        if (cut && !(MOE && ph == 1)) {
          // The CTA that arrives last at this tile finishes it.
          c_first = split.cta_of(u * L);
          c_last = split.cta_of(u * L + L - 1);
          __threadfence();
          epilogue_all(1);
          if (threadIdx.x == 128) {
            const unsigned old = atom_add_acq_rel(arrivals + c_first, 1u);
            const int last = old == static_cast<unsigned>(c_last - c_first);
            if (last) arrivals[c_first] = 0;  // for the next launch
            *last_flag = last;
          }
          epilogue_all(1);
          finish = *last_flag;
          __threadfence();
        }
        if (finish) {
          const bool glu = MOE && p.act == 3;
          const int feature = glu ? tile * 64 + sub * 16 + (lane & 15) : tile * kBM + row;
          const bool live = feature < p.feat1;
          const float bias = !MOE && p.bias && live ? unpack_lo<BF16>(static_cast<uint32_t>(__ldg(p.bias + feature))) : 0.f;
#pragma unroll 1
          for (int c0 = 0; c0 < count; c0 += 16) {
            float v[16];
            if (!cut) {
              tmem_ld16(acc + c0, v);
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = 0.f;
#pragma unroll 1
              for (int q = c_first; q <= c_last; ++q) {
                // (the first CTA's stretch begins the tile: its second slot)
                const float* src = p.partial1 +
                                   (2 * static_cast<size_t>(q) + (q == c_first ? 1 : 0)) * static_cast<size_t>(p.chunk) * kBM +
                                   row;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (c0 + j < count) v[j] += __ldcg(src + static_cast<size_t>(c0 + j) * kBM);
              }
            }
            if constexpr (MOE) {
              if (glu) {
                // Lane l < 16 holds gate row l, lane l + 16 the matching up row: of each column
                // pair the lower lane finishes the first, the upper lane the second.
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                  const float got = __shfl_xor_sync(0xffffffffu, lane < 16 ? v[j + 1] : v[j], 16);
                  const float gate = lane < 16 ? v[j] : got, up = lane < 16 ? got : v[j + 1];
                  const int col = c0 + j + (lane < 16 ? 0 : 1);
                  if (live && col < count)
                    p.hidden[static_cast<long long>(start + col) * p.ldh + feature] = cvt1<BF16>(silu(gate) * up);
                }
              } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (live && c0 + j < count)
                    p.hidden[static_cast<long long>(start + c0 + j) * p.ldh + feature] = cvt1<BF16>(act_value(v[j], p.act));
              }
            } else {
              float r[16];
#pragma unroll
              for (int j = 0; j < 16; ++j)
                r[j] = p.residual && live && c0 + j < count
                           ? unpack_lo<BF16>(static_cast<uint32_t>(
                                 __ldg(p.residual + static_cast<long long>(start + c0 + j) * p.ldr + feature)))
                           : 0.f;
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (live && c0 + j < count)
                  p.y[static_cast<long long>(start + c0 + j) * p.ldy + feature] =
                      cvt1<BF16>(act_value(v[j] + bias, p.act) + r[j]);
            }
          }
          if constexpr (MOE) {
            fence_async_global();  // hidden: written here, read through other CTAs' TMA
            __threadfence();
            epilogue_all(1);
            if (threadIdx.x == 128) red_release_add(item_done + it, 1u);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty(b));
        ++n_acc;
        s += k1 - k0;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, tmem_cols);

  if constexpr (MOE) {
    // Combination: when every CTA's second-product sums are in memory, each warp takes
    // (token, 128 output features) and adds the token's experts in order, each expert's pieces in
    // ascending CTA order, with the fp32 weights, then the residual; rounded once.
    if (threadIdx.x == 0) {
      __threadfence();
      red_release_add(sync_words, 1u);
      if (!*abort_flag) stream_wait_word(sync_words, static_cast<unsigned>(C), abort_flag, p, 3, -1);
    }
    __syncthreads();
    if (!*abort_flag) {
      __threadfence();
      const StreamSplit split(static_cast<long long>(items) * p.tiles2 * p.steps2, C);
      const int L = p.steps2;
      const size_t whole_pitch = static_cast<size_t>(p.tiles2) * kBM;
      for (long long unit = static_cast<long long>(warp) * C + c; unit < static_cast<long long>(p.tokens) * p.tiles2;
           unit += static_cast<long long>(C) * (kStreamThreads / 32)) {
        const int t = static_cast<int>(unit / p.tiles2), tile = static_cast<int>(unit % p.tiles2);
        // Lane j knows choice j: its weight, the first piece's address and the pieces' count.
        const float* src = nullptr;
        int pieces = 0, c_first = 0;
        float wt = 0.f;
        if (lane < p.top) {
          const int e = __ldg(p.ids + t * p.top + lane);
          if (static_cast<unsigned>(e) < static_cast<unsigned>(p.experts)) {
            wt = __ldg(p.weights + t * p.top + lane);
            int rank = 0;
            for (int w = 0; w < (t >> 5); ++w) rank += __popc(sets[e * lists.words + w]);
            rank += __popc(sets[e * lists.words + (t >> 5)] & ((1u << (t & 31)) - 1u));
            const int it = first[e] + rank / p.chunk;
            const int u = it * p.tiles2 + tile;
            c_first = split.cta_of(u * L);
            pieces = split.cta_of(u * L + L - 1) - c_first + 1;
            if (pieces == 1)
              src = p.whole2 + static_cast<size_t>(offset[e] + rank) * whole_pitch + static_cast<size_t>(tile) * kBM;
            else
              src = p.partial2 + static_cast<size_t>(rank % p.chunk) * kBM;
          }
        }
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        const size_t slot = static_cast<size_t>(p.chunk) * kBM;
        for (int j = 0; j < p.top; ++j) {
          const int n = __shfl_sync(0xffffffffu, pieces, j);
          const int cf = __shfl_sync(0xffffffffu, c_first, j);
          const float wj = __shfl_sync(0xffffffffu, wt, j);
          const float* sj = reinterpret_cast<const float*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), j));
          if (n == 0) continue;
          float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int q = 0; q < n; ++q) {
            const float* at = n == 1 ? sj : sj + (2 * static_cast<size_t>(cf + q) + (q == 0 ? 1 : 0)) * slot;
            const float4 v = __ldcg(reinterpret_cast<const float4*>(at) + lane);
            z.x += v.x, z.y += v.y, z.z += v.z, z.w += v.w;
          }
          sum.x = fmaf(wj, z.x, sum.x), sum.y = fmaf(wj, z.y, sum.y);
          sum.z = fmaf(wj, z.z, sum.z), sum.w = fmaf(wj, z.w, sum.w);
        }
        const float s4[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int f = tile * kBM + 4 * lane + q;
          if (f < p.feat2) {
            const float r = p.residual ? unpack_lo<BF16>(static_cast<uint32_t>(p.residual[static_cast<long long>(t) * p.ldr + f])) : 0.f;
            p.y[static_cast<long long>(t) * p.ldy + f] = cvt1<BF16>(s4[q] + r);
          }
        }
      }
    }
    // The last CTA to leave clears the counters for the next launch.
    __syncthreads();
    if (threadIdx.x == 0) *last_flag = atom_add_acq_rel(sync_words + 1, 1u) == static_cast<unsigned>(C - 1);
    __syncthreads();
    if (*last_flag) {
      for (int i = threadIdx.x; i < items; i += kStreamThreads) item_done[i] = 0;
      if (threadIdx.x < kStreamSync) sync_words[threadIdx.x] = 0;
    }
  }
}

}  // namespace ffnb200
