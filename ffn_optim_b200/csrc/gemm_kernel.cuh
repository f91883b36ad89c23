// Dense projection for more than a few tokens:  Y = act(X . W^T + b) + R,  tcgen05 tiles.
//
// Bound by the tensor cores when K is long, by the bytes of X, R and Y when it is short, by
// latency when the tiles are fewer than the SMs.  Three tiles:
//   256 x 256 by a CTA pair (cta_group::2): each SM loads half of both operands, so a K step of 64
//     feeds 512 MMA clocks with 32 KB per SM -- long runs of tiles with long K;
//   128 x 128 and 128 x 64 by one CTA; for few tiles a cluster of up to 8 CTAs splits a tile's K,
//     each CTA finishing its share of the columns from the fp32 parts that its peers store into
//     its shared memory, added in rank order.
// Persistent grid; TMA producer (warp 0), MMA issuer (warp 1), 8 epilogue warps (4..11, two per
// TMEM sub-partition, halves of the columns) over two TMEM accumulators, so a tile's epilogue runs
// under the next tile's MMAs.  Residual and bias are read ahead of the accumulator (6993 x 100 x 1000, SiLU: residual
// a row per lane and bias when needed 18.6 us, whole lines and both ahead 17.0 us); results leave through swizzled staging and TMA stores, which clip ragged edges.
#pragma once

#include "stream_kernel.cuh"

namespace ffnb200 {

constexpr int kGemmThreads = 384;
constexpr int kGemmEpiWarps = 8;

struct GemmParams {
  CUtensorMap tm_x, tm_w, tm_y;  // boxes 64 x 128 rows, 64 x (BN; pair: 128) rows, 64 x 32 rows (store)
  int M, N, steps;               // K steps of 64
  int tiles_m, tiles_n, group;   // tile grid; tile rows walked together before the next column
  int split;                     // CTAs (a cluster) per tile's K; pair tiles: 1
  int act;                       // ffn_b200_gelu
  const uint16_t* bias;
  const uint16_t* residual;
  long long ldr;
  uint16_t* y;
  long long ldy;
  int* status;
  unsigned long long wait_limit_ns;
};

template <int BN, bool PAIR>
struct GemmLayout {
  static constexpr int kBRows = PAIR ? BN / 2 : BN;
  static constexpr int kStage = kABytes + kBRows * 128;
  static constexpr int kStages = 196608 / kStage;
  static constexpr int kStaging = kGemmEpiWarps * kStageBufBytes;
  static constexpr int kSmem = 1024 + kStages * kStage + kStaging + 256;
  static constexpr int kTmemCols = 2 * BN;
  static_assert(kSmem <= 232448 && (2 * kStages + 6) * 8 <= 256 && kTmemCols <= 512, "sizes");
};

__device__ __forceinline__ void st_cluster_f4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
// 16 bytes to this CTA's shared memory.
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// W residual values of one row (two per word) from column c0; zero outside the matrix.
template <int W>
__device__ __forceinline__ void load_row(uint32_t* r, const uint16_t* base, long long ld, int row, int rows, int c0, int cols) {
  if (row < rows && c0 + W <= cols) {
    const uint4* src = reinterpret_cast<const uint4*>(base + static_cast<long long>(row) * ld + c0);
#pragma unroll
    for (int q = 0; q < W / 8; ++q) {
      const uint4 w = __ldg(src + q);
      r[4 * q] = w.x, r[4 * q + 1] = w.y, r[4 * q + 2] = w.z, r[4 * q + 3] = w.w;
    }
  } else {
#pragma unroll
    for (int q = 0; q < W / 2; ++q) {
      const uint16_t* src = base + static_cast<long long>(row) * ld + c0 + 2 * q;
      const uint32_t lo = row < rows && c0 + 2 * q < cols ? __ldg(src) : 0;
      const uint32_t hi = row < rows && c0 + 2 * q + 1 < cols ? __ldg(src + 1) : 0;
      r[q] = lo | hi << 16;
    }
  }
}

// The first `count` (at most W) of W values to a 16-byte aligned row.
template <bool BF16, int W>
__device__ __forceinline__ void store_row(uint16_t* y, const float* v, int count) {
#pragma unroll
  for (int q = 0; q < W; q += 8) {
    if (q + 8 <= count) {
      *reinterpret_cast<uint4*>(y + q) = make_uint4(pack2<BF16>(v[q], v[q + 1]), pack2<BF16>(v[q + 2], v[q + 3]),
                                                    pack2<BF16>(v[q + 4], v[q + 5]), pack2<BF16>(v[q + 6], v[q + 7]));
    } else {
#pragma unroll
      for (int j = q; j < q + 8; ++j)
        if (j < count) y[j] = cvt1<BF16>(v[j]);
    }
  }
}

__device__ __forceinline__ bool gemm_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, const GemmParams& p,
                                          int aux) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = gtimer();
  uint32_t n = 0;
#pragma unroll 1
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++n & 15u) == 0) {
      if (*abort_flag) return false;
      if (gtimer() - t0 > p.wait_limit_ns) {
        if (atomicCAS(p.status, 0, 1) == 0) p.status[1] = blockIdx.x, p.status[2] = aux;
        *abort_flag = 1;
        return false;
      }
    }
  }
}

template <bool BF16, int BN, bool PAIR>
__global__ void __launch_bounds__(kGemmThreads, 1) gemm_kernel(const __grid_constant__ GemmParams p) {
  using LY = GemmLayout<BN, PAIR>;
  constexpr int ST = LY::kStages;
  constexpr int kTileM = PAIR ? 256 : 128;
  constexpr uint32_t kIdesc = make_idesc<BF16, BN, kTileM>();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t sStage = base + ST * LY::kStage;
  const uint32_t sBar = sStage + LY::kStaging;
  auto full_bar = [&](int s) { return sBar + 8u * s; };
  auto empty_bar = [&](int s) { return sBar + 8u * (ST + s); };
  auto tfull_bar = [&](int a) { return sBar + 8u * (2 * ST + a); };
  auto tempty_bar = [&](int a) { return sBar + 8u * (2 * ST + 2 + a); };
  const uint32_t drain_bar = sBar + 8u * (2 * ST + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + (sBar - base) + 8 * (2 * ST + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int S = PAIR ? 2 : p.split;  // CTAs of the cluster
  const uint32_t rank = S > 1 ? cluster_rank() : 0u;
  const int owner = static_cast<int>(blockIdx.x) / S, owners = static_cast<int>(gridDim.x) / S;
  const int tiles = p.tiles_m * p.tiles_n;
  // K steps of this CTA (all of them unless the tile's K is split).
  const int k0 = PAIR ? 0 : p.steps * static_cast<int>(rank) / S;
  const int k1 = PAIR ? p.steps : p.steps * (static_cast<int>(rank) + 1) / S;

  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int s = 0; s < ST; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), kGemmEpiWarps * (PAIR ? 2 : 1));
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_async_shared();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&p.tm_x);
    prefetch_tmap(&p.tm_w);
    prefetch_tmap(&p.tm_y);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), LY::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), LY::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (S > 1) cluster_sync();  // the peers' barriers are there before anything arrives on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (threadIdx.x == 0) grid_dep_launch();
  grid_dep_wait();

  auto coords = [&](int t, int& tm, int& tn) {
    const int per_group = p.group * p.tiles_n;
    const int g = t / per_group, rem = t - g * per_group;
    const int rows = min(p.group, p.tiles_m - g * p.group);
    tm = g * p.group + rem % rows;
    tn = rem / rows;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
#pragma unroll 1
      for (int t = owner; t < tiles && ok; t += owners) {
        int tm, tn;
        coords(t, tm, tn);
        const int arow = tm * kTileM + (PAIR ? static_cast<int>(rank) * kBM : 0);
        const int brow = tn * BN + (PAIR ? static_cast<int>(rank) * LY::kBRows : 0);
#pragma unroll 1
        for (int kb = k0; kb < k1; ++kb) {
          if (!gemm_wait(empty_bar(stage), phase ^ 1u, abort_flag, p, 100 + stage)) { ok = false; break; }
          const uint32_t dst = base + stage * LY::kStage;
          if constexpr (PAIR) {
            const uint32_t fb = map_to_rank(full_bar(stage), 0);
            if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * LY::kStage);
            tma_load_2d_pair(dst, &p.tm_x, kb * kBK, arow, fb);
            tma_load_2d_pair(dst + kABytes, &p.tm_w, kb * kBK, brow, fb);
          } else {
            mbar_expect_tx(full_bar(stage), LY::kStage);
            tma_load_2d(dst, &p.tm_x, kb * kBK, arow, full_bar(stage));
            tma_load_2d(dst + kABytes, &p.tm_w, kb * kBK, brow, full_bar(stage));
          }
          ++issued;
          if (++stage == ST) { stage = 0; phase ^= 1u; }
        }
      }
      // Every load lands before the CTA may leave: a slot's reuse was waited for, the last
      // ST are waited for here by their consumption (empty barriers; bounded).
      const uint64_t t0 = gtimer();
      bool late = false;
      for (long long i = issued > ST ? issued - ST : 0; i < issued && !late; ++i)
        while (!mbar_try_wait(empty_bar(static_cast<int>(i % ST)), static_cast<uint32_t>((i / ST) & 1)))
          if (gtimer() - t0 > p.wait_limit_ns || (*abort_flag && gtimer() - t0 > 1000000ull)) { late = true; break; }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue (pair: the leader)
    if ((!PAIR || rank == 0) && elect_one()) {
      int stage = 0, n_acc = 0;
      uint32_t phase = 0;
      bool ok = true;
#pragma unroll 1
      for (int t = owner; t < tiles && ok; t += owners, ++n_acc) {
        const int a = n_acc & 1;
        if (!gemm_wait(tempty_bar(a), ((n_acc >> 1) & 1) ^ 1u, abort_flag, p, 200 + a)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(a * BN);
#pragma unroll 1
        for (int kb = k0; kb < k1; ++kb) {
          if (!gemm_wait(full_bar(stage), phase, abort_flag, p, 300 + stage)) { ok = false; break; }
          tc_fence_after();
          const uint64_t da = sw128_desc(base + stage * LY::kStage), db = sw128_desc(base + stage * LY::kStage + kABytes);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            const uint32_t accum = kb > k0 || k > 0 ? 1u : 0u;
            if constexpr (PAIR) umma_f16_pair(d, da + 2 * k, db + 2 * k, kIdesc, accum);
            else umma_f16(d, da + 2 * k, db + 2 * k, kIdesc, accum);
          }
          if constexpr (PAIR) umma_commit_pair_both(empty_bar(stage));
          else umma_commit(empty_bar(stage));
          if (++stage == ST) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if constexpr (PAIR) umma_commit_pair_both(tfull_bar(a));
        else umma_commit(tfull_bar(a));
      }
      if constexpr (PAIR) umma_commit_pair(drain_bar);
      else umma_commit(drain_bar);
      const uint64_t t0 = gtimer();
      while (!mbar_try_wait(drain_bar, 0))
        if (gtimer() - t0 > p.wait_limit_ns) break;
    }
  } else if (warp >= 4 && (PAIR || S == 1)) {
    // ------------------------------------------------------------------ epilogue
    constexpr int kChunks = BN / 64;                       // 64-column chunks of a tile
    constexpr int kMine = kChunks >= 2 ? kChunks / 2 : 1;  // chunks of one warp
    const int sub = warp & 3, half = (warp - 4) >> 2;
    const bool works = kChunks >= 2 || half == 0;
    const uint32_t stg = sStage + static_cast<uint32_t>((warp - 4) * kStageBufBytes);
    int n_acc = 0;
    uint32_t r[32], b[32];  // the next chunk's residual (16-byte piece lane % 8 of rows lane / 8 + 4 q) and bias
    auto read = [&](int row0, int col0) {
      if (p.residual) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          load_row<8>(r + 4 * q, p.residual, p.ldr, row0 + 4 * q + (lane >> 3), p.M, col0 + 8 * (lane & 7), p.N);
      }
      if (p.bias) load_row<64>(b, p.bias, 0, 0, 1, col0, p.N);
    };
    auto place = [&](int t, int& row0, int& first) {
      int tm, tn;
      coords(t, tm, tn);
      row0 = tm * kTileM + (PAIR ? static_cast<int>(rank) * kBM : 0) + sub * 32;
      first = tn * BN + half * kMine * 64;
    };
    int row0 = 0, first = 0;
    if (owner < tiles) place(owner, row0, first);
    if (works && owner < tiles) read(row0, first);
#pragma unroll 1
    for (int t = owner; t < tiles; t += owners, ++n_acc) {
      const int a = n_acc & 1;
      int next_row0 = 0, next_first = 0;
      const bool more = t + owners < tiles;
      if (more) place(t + owners, next_row0, next_first);
      int ok = 1;
      if (lane == 0) ok = gemm_wait(tfull_bar(a), (n_acc >> 1) & 1, abort_flag, p, 400 + a) ? 1 : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem_base + (static_cast<uint32_t>(sub * 32) << 16) + static_cast<uint32_t>(a * BN);
#pragma unroll 1
      for (int c = 0; c < kMine; ++c) {
        const int col0 = first + 64 * c;
        float v[64];
        if (works) tmem_ld64(acc + static_cast<uint32_t>((half * kMine + c) * 64), v);
        if (c == kMine - 1) {  // the accumulator is read: free for the tile after next
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR) mbar_arrive_cluster(map_to_rank(tempty_bar(a), 0));
            else mbar_arrive(tempty_bar(a));
          }
        }
        // The chunk after this one (of the next tile, if it is the last).
        auto read_ahead = [&]() {
          if (!works) return;
          if (c + 1 < kMine) read(row0, col0 + 64);
          else if (more) read(next_row0, next_first);
        };
        if (!works || col0 >= p.N || row0 >= p.M) {
          read_ahead();
          continue;
        }
        if (lane == 0) bulk_wait_read0();  // the staging's previous store has been read
        __syncwarp();
        if (p.residual) {  // to rows through the staging: whole lines asked for, a row per lane used
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int row = 4 * q + (lane >> 3);
            st_shared_v4(stg + static_cast<uint32_t>(row * 128 + (((lane ^ row) & 7) << 4)), r[4 * q], r[4 * q + 1], r[4 * q + 2],
                         r[4 * q + 3]);
          }
        }
        if (p.bias) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            v[2 * j] += unpack_lo<BF16>(b[j]);
            v[2 * j + 1] += unpack_hi<BF16>(b[j]);
          }
        }
        read_ahead();
        apply_act<64>(v, p.act);
        if (p.residual) {
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const uint4 w = ld_shared_u4(stg + static_cast<uint32_t>(lane * 128 + ((q ^ (lane & 7)) << 4)));
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              v[8 * q + 2 * j] += unpack_lo<BF16>(u[j]);
              v[8 * q + 2 * j + 1] += unpack_hi<BF16>(u[j]);
            }
          }
        }
        if (col0 + 64 > p.N && (p.N & 7) != 0) {
          // (A TMA store clips rows, but columns only to 16 bytes: the last columns go out one by one.)
          if (row0 + lane < p.M) store_row<BF16, 64>(p.y + static_cast<long long>(row0 + lane) * p.ldy + col0, v, p.N - col0);
          continue;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q)
          st_shared_v4(stg + static_cast<uint32_t>(lane * 128 + ((q ^ (lane & 7)) << 4)), pack2<BF16>(v[8 * q], v[8 * q + 1]),
                       pack2<BF16>(v[8 * q + 2], v[8 * q + 3]), pack2<BF16>(v[8 * q + 4], v[8 * q + 5]),
                       pack2<BF16>(v[8 * q + 6], v[8 * q + 7]));
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&p.tm_y, stg, col0, row0);
          bulk_commit();
        }
      }
      row0 = next_row0, first = next_first;
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }

  if (!PAIR && S > 1) {
    // ------------------------------------------------------------------ split K: one tile per cluster
    const int sub = warp & 3, half = (warp - 4) >> 2;
    const int row = sub * 32 + lane;
    const int share = BN / S;  // columns that each CTA finishes (8 at least)
    int tm, tn;
    coords(owner, tm, tn);
    int ok = 1;
    uint32_t r[4];  // the next 8 columns' residual, asked for before anything is waited for
    auto read_ahead = [&](int c0) {
      if (p.residual && c0 < share)
        load_row<8>(r, p.residual, p.ldr, tm * kBM + row, p.M, tn * BN + static_cast<int>(rank) * share + c0, p.N);
    };
    if (warp >= 4) {
      read_ahead(8 * half);
      if (lane == 0) ok = gemm_wait(tfull_bar(0), 0, abort_flag, p, 400) ? 1 : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      tc_fence_after();
    }
    __syncthreads();
    cluster_sync();  // every CTA's loads and MMAs are done: the rings are free
    const uint32_t acc = tmem_base + (static_cast<uint32_t>(sub * 32) << 16);
    // Buffer in a finisher's ring: [sender][share / 4][128 rows] float4.
    auto cell = [&](int sender, int quad) { return base + static_cast<uint32_t>(((sender * (share / 4) + quad) * kBM + row) * 16); };
    if (warp >= 4) {
#pragma unroll 1
      for (int c0 = 8 * half; c0 < BN; c0 += 16) {  // the two warps of a sub-partition take columns in turn
        const int to = c0 / share;
        if (to == static_cast<int>(rank)) continue;
        float v[8];
        tmem_ld8(acc + static_cast<uint32_t>(c0), v);
        const uint32_t dst = map_to_rank(cell(static_cast<int>(rank), (c0 - to * share) / 4), static_cast<uint32_t>(to));
        st_cluster_f4(dst, v[0], v[1], v[2], v[3]);
        st_cluster_f4(dst + kBM * 16, v[4], v[5], v[6], v[7]);
      }
    }
    cluster_sync();
    if (warp >= 4) {
      const int grow = tm * kBM + row;
#pragma unroll 1
      for (int c0 = 8 * half; c0 < share; c0 += 16) {
        const int col = tn * BN + static_cast<int>(rank) * share + c0;
        float own[8], v[8];
        __syncwarp();
        tmem_ld8(acc + static_cast<uint32_t>(static_cast<int>(rank) * share + c0), own);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll 1
        for (int s = 0; s < S; ++s) {
          if (s == static_cast<int>(rank)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += own[j];
          } else {
            const float4 lo = ld_shared_f4(cell(s, c0 / 4)), hi = ld_shared_f4(cell(s, c0 / 4 + 1));
            v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
            v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
          }
        }
        const bool write = grow < p.M && col < p.N && !*abort_flag;
        if (write && p.bias) add_bias<BF16, 8>(v, p.bias, col, p.N);
        apply_act<8>(v, p.act);
        if (p.residual) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[2 * j] += unpack_lo<BF16>(r[j]), v[2 * j + 1] += unpack_hi<BF16>(r[j]);
          read_ahead(c0 + 16);
        }
        if (!write) continue;
        store_row<BF16, 8>(p.y + static_cast<long long>(grow) * p.ldy + col, v, p.N - col);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // no CTA leaves while its peer may still signal it
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, LY::kTmemCols);
    else tmem_dealloc(tmem_base, LY::kTmemCols);
  }
}

}  // namespace ffnb200
