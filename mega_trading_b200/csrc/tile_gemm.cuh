// One persistent tcgen05 matrix product for operators that differ in element
// type, operand layout and epilogue:  C[M, N] = A B^T over K, where A's and
// B's rows (M and N) are the strided dimension (K-major) or the contiguous
// one (MN-major, 16-bit types only).
//
// Layout of one CTA: EW epilogue warps in warpgroups that take the column steps
// of a tile in turn (thread = row = TMEM lane), then a TMA producer warp (which
// also allocates TMEM) and an MMA issuer warp.  EW = 16 puts four epilogue
// warps on a scheduler to cover each other's TMEM, fence and staging latencies,
// for products whose epilogue outlasts a tile's main loop with 8 (8-bit, K of
// about 1,000: 65,537 x 5,632 x 1,024 in 0.42 ms with 8, 0.37 ms with 16); 8
// leave room for one more stage and poll less.  Tiles are 128 x BN with one
// CTA, or 256 x BN with a CTA pair (tcgen05 cta_group::2): each CTA of a pair
// stages its own 128 rows of A and half of B's rows, which takes a third off
// the shared-memory traffic per product.  A stage of the TMA ring holds 128
// bytes of K (64 16-bit or 128 8-bit elements) of both operands in 128-byte
// swizzle; two BN-column fp32 / int32 accumulators alternate in TMEM, so a
// tile's epilogue runs under the next tile's products.
//
// The pair's stage loads complete on the even CTA's barrier, which expects
// both CTAs' bytes; the even CTA issues the MMAs and commits to both CTAs'
// barriers.  Before teardown the odd CTA waits (bounded) for the release of
// every stage it loaded.  Every wait is bounded; on a timeout the status word
// is set, copies in flight are drained and TMEM is freed.
//
// Epilogue steps cover one 128-byte row segment of the output (64 16-bit or 32
// fp32 columns) of a warp's 32 rows.  They leave through the warp's own
// 4 KB staging box and a TMA store (or TMA fp32 add), so no barrier spans
// warps (32-byte stores straight from registers were 9 % slower, copying the box
// out with 16-byte stores 17-30 %); outputs whose row stride or base is not a
// multiple of 16 bytes are copied out of the box with plain coalesced stores.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace mt {

enum { kKindBf16 = 0, kKindF16 = 1, kKindI8 = 2 };

// D[tmem] (+)= A[smem] * B[smem] on signed 8-bit integers, 32-bit accumulators.
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Bounded waits whose try_wait may suspend the thread for up to 10 ms before it
// looks again: the epilogue warps wait through a tile's whole main loop, and
// polling costs issue slots and power (the distillation step of 32,768 rows runs
// at the power limit and went from 4.24 to 4.14 ms).
__device__ __forceinline__ bool try_wait_long(uint64_t* bar, uint32_t parity, bool cluster) {
  uint32_t ok;
  if (cluster)
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, 0x989680;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 0x989680;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
  return ok != 0;
}
template <bool CLUSTER>
__device__ __forceinline__ bool wait_bounded_long(const WaitCtx& ctx, uint64_t* bar, uint32_t parity, uint32_t site) {
  if (try_wait_long(bar, parity, CLUSTER)) return true;
  long long t0 = clock64();
  while (true) {
    if (*ctx.abort_flag) return false;
    if (try_wait_long(bar, parity, CLUSTER)) return true;
    if (clock64() - t0 > ctx.limit) {
      atomicCAS(ctx.status, 0u, (ctx.kernel_id << 16) | site);
      *ctx.abort_flag = 1;
      return false;
    }
  }
}

// Instruction descriptor, kind::i8: signed 8-bit A and B (K-major), int32 accumulator.
__host__ __device__ constexpr uint32_t make_idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

// EW: epilogue warps, 8 or 16.
template <int KIND_, bool A_MN_, bool B_MN_, int BN_, bool PAIR_, int EW_>
struct TileCfg {
  static constexpr int EW = EW_;
  static constexpr int kThreads = (EW + 2) * 32;
  static constexpr int KIND = KIND_, BN = BN_;
  static constexpr bool A_MN = A_MN_, B_MN = B_MN_, PAIR = PAIR_;
  static_assert(KIND != kKindI8 || (!A_MN && !B_MN), "8-bit operands are K-major");
  static constexpr int ESZ = KIND == kKindI8 ? 1 : 2;
  static constexpr int BK = 128 / ESZ;  // K elements per stage
  static constexpr int TM = PAIR ? 256 : 128;
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;  // rows of B one CTA stages
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = B_ROWS * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int BOX = 4096;  // a warp's staging box: 32 rows x 128 bytes
  static constexpr int OUT_BYTES = EW * BOX;
  static constexpr int COL_BYTES = EW * 256;  // a warp's 64 per-column values
  static constexpr int kMaxStages = (226 * 1024 - OUT_BYTES - COL_BYTES) / STAGE;
  static constexpr int NST = kMaxStages < 8 ? kMaxStages : 8;
  static constexpr int OFF_OUT = NST * STAGE;
  static constexpr int OFF_COL = OFF_OUT + OUT_BYTES;
  static constexpr int OFF_BAR = OFF_COL + COL_BYTES;
  static constexpr int SMEM = OFF_BAR + 256;
  static_assert(SMEM <= 227 * 1024, "more shared memory than one sm_100 CTA may use");
  static_assert(2 * NST + 5 <= 28, "mbarriers overlap the TMEM slot");
};

template <class EP>
struct TileParams {
  CUtensorMap tm_a, tm_b, tm_out;
  int M, N;                  // output rows and columns
  int n_mt, n_nt, n_tiles;   // n_tiles = n_mt * n_nt * splits, columns fastest, splits slowest
  int n_k, k_per_split;      // stages of K in total and per split
  int per_unit;              // > 0: a CTA (pair) takes this many consecutive tiles; 0: every n-th
  FastDiv div_nt, div_split;  // by n_nt and by n_mt * n_nt
  int64_t split_rows;        // rows of the output map between two splits
  void* out;                 // direct stores only
  int64_t ld_out;
  uint32_t* status;
  EP ep;
};

// byte offset of 16-byte chunk j of row r in a 128-byte-swizzled box
__device__ __forceinline__ int box128_off(int r, int j) { return r * 128 + ((j ^ (r & 7)) << 4); }

// One 32-bit TMEM column of the warp's 32 lanes.
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(v)
               : "r"(taddr)
               : "memory");
  return v;
}

// Element-wise fp32 add of a staging box into global memory.
__device__ __forceinline__ void tma_out(const CUtensorMap* map, const void* src, int c0, int c1, bool add) {
  if (add)
    tma_reduce_add_2d(map, src, c0, c1);
  else
    tma_store_2d(map, src, c0, c1);
}

// EP (epilogue) provides
//   static constexpr uint32_t kKernelId;
//   static constexpr int OUT_SIZE;          2 or 4 bytes per output element
//   struct Row;                             per-row values of a tile
//   Row row(int m, bool live)               loads them
//   static constexpr bool kCols;            whether per-column values are used
//   float col(int n)                        loads one (0 past the last column)
//   void pack(const uint32_t (&z)[32], const Row&, const float* cols, uint32_t* words)
//       32 accumulator columns and their column values (shared memory) -> 16
//       (OUT_SIZE 2) or 32 (4) packed words
//   bool add, direct                        TMA add instead of store; plain stores
//   static constexpr bool kAltB;            whether B may come from another tensor:
//   const CUtensorMap* b_map(const CUtensorMap*) const    decides (device memory may say)
// or, with `static constexpr bool kStats = true` (per_unit > 0), nothing is
// written per tile and a thread keeps its row's state over consecutive tiles:
//   struct State;
//   void begin(State&, int m, bool live, int mt, int unit, int group)
//   int next(const State&)                  next column whose value is asked for
//   void take(State&, uint32_t z)           gets it and moves on
//   void skip(State&)                       moves on without it
//   void add(State&, const uint32_t (&z)[32], int n0)
//   void end(const State&)                  the row's last tile of this CTA is done
template <class C, class EP>
__global__ void __launch_bounds__(C::kThreads, 1) tile_gemm_kernel(const __grid_constant__ TileParams<EP> p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr bool PAIR = C::PAIR;
  constexpr uint32_t kId = EP::kKernelId;
  const int warp = warp_id();
  const int lane = lane_id();
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0u, (kId << 16) | 0xFFFFu);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* full = bars;                   // [NST]
  uint64_t* empty = bars + C::NST;         // [NST]
  uint64_t* acc_full = bars + 2 * C::NST;  // [2]
  uint64_t* acc_empty = acc_full + 2;      // [2]
  uint64_t* fin = acc_full + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 28);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 29);

  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int n_units = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const int row_off = (int)rank * 128;
  const int per_split = p.n_mt * p.n_nt;
  const int t_begin = p.per_unit > 0 ? unit * p.per_unit : unit;
  const int t_end = p.per_unit > 0 ? min(t_begin + p.per_unit, p.n_tiles) : p.n_tiles;
  const int t_step = p.per_unit > 0 ? 1 : n_units;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::NST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], (PAIR ? 2 : 1) * C::EW);  // one arrival per epilogue warp (of both CTAs)
    }
    mbar_init(fin, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == C::EW) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, 2 * C::BN);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 2 * C::BN);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (PAIR)
    cluster_sync_all();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const WaitCtx wc{p.status, abort_flag, kId};
  auto wait_x = [&](uint64_t* bar, uint32_t parity, uint32_t site) {
    return wait_bounded_long<PAIR>(wc, bar, parity, site);
  };
  struct Tile {
    int m0, n0, k0, k1, split, mt;
  };
  auto tile_at = [&](int t) {
    const int split = (int)p.div_split.div((uint32_t)t), u = t - split * per_split;
    const int mt = (int)p.div_nt.div((uint32_t)u), nt = u - mt * p.n_nt;
    const int k0 = split * p.k_per_split;
    return Tile{mt * C::TM + row_off, nt * C::BN, k0, min(k0 + p.k_per_split, p.n_k), split, mt};
  };

  if (warp == C::EW) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const CUtensorMap* tm_b = &p.tm_b;
      if constexpr (EP::kAltB) tm_b = p.ep.b_map(tm_b);
      tma_prefetch_desc(&p.tm_a);
      tma_prefetch_desc(tm_b);
      int it = 0;
      bool ok = true;
      for (int t = t_begin; ok && t < t_end; t += t_step) {
        const Tile w = tile_at(t);
        const int b0 = w.n0 + (int)rank * C::B_ROWS;
        for (int kc = w.k0; kc < w.k1; ++kc, ++it) {
          const int st = it % C::NST;
          if (it >= C::NST && !wait_x(&empty[st], ((it / C::NST) & 1) ^ 1, 1)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + st * C::STAGE;
          uint8_t* sb = sa + C::A_BYTES;
          const int k = kc * C::BK;
          const uint32_t bar = PAIR ? leader_addr(&full[st]) : 0u;
          if (leader) mbar_arrive_expect_tx(&full[st], (PAIR ? 2 : 1) * C::STAGE);
          auto load = [&](void* dst, const CUtensorMap* map, int c0, int c1) {
            if constexpr (PAIR)
              tma_load_2d_pair(dst, map, bar, c0, c1);
            else
              tma_load_2d(dst, map, &full[st], c0, c1);
          };
          if constexpr (C::A_MN) {
            load(sa, &p.tm_a, w.m0, k);
            load(sa + 8192, &p.tm_a, w.m0 + 64, k);
          } else {
            load(sa, &p.tm_a, k, w.m0);
          }
          if constexpr (C::B_MN) {
#pragma unroll
            for (int j = 0; j < C::B_ROWS / 64; ++j) load(sb + j * 8192, tm_b, b0 + j * 64, k);
          } else {
            load(sb, tm_b, k, b0);
          }
        }
      }
      if (PAIR && !leader) {
        // the odd CTA's loads complete on the leader's barrier: wait until the
        // leader's MMAs released every stage loaded here (bounded)
        for (int j = (it > C::NST ? it - C::NST : 0); j < it; ++j)
          wait_drain(wc, &empty[j % C::NST], (j / C::NST) & 1, 15);
      }
      if (*abort_flag) {
        for (int j = (it > C::NST ? it - C::NST : 0); j < it; ++j)
          wait_drain(wc, &full[j % C::NST], (j / C::NST) & 1, 11);
      }
    }
  } else if (warp == C::EW + 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA of a pair)
    if (lane == 0 && leader) {
      constexpr uint32_t idesc = C::KIND == kKindI8
                                     ? make_idesc_i8(C::TM, C::BN)
                                     : make_idesc(C::TM, C::BN, C::KIND == kKindBf16 ? 1 : 0, C::A_MN, C::B_MN);
      // one MMA takes 32 bytes of K: inside the swizzled row (K-major), or 16 rows (MN-major)
      constexpr uint32_t a_step = C::A_MN ? 16 * 128 / 16 : 2, b_step = C::B_MN ? 16 * 128 / 16 : 2;
      const uint32_t base = smem_u32(smem);
      int it = 0, lt = 0;
      bool ok = true;
      for (int t = t_begin; ok && t < t_end; t += t_step, ++lt) {
        const Tile w = tile_at(t);
        const int buf = lt & 1;
        if (lt >= 2 && !wait_x(&acc_empty[buf], ((lt >> 1) & 1) ^ 1, 2)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * C::BN;
        for (int kc = w.k0; kc < w.k1; ++kc, ++it) {
          const int st = it % C::NST;
          if (!wait_x(&full[st], (it / C::NST) & 1, 3)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = base + st * C::STAGE;
          const uint32_t b = a + C::A_BYTES;
          const uint64_t ad = make_sdesc(a, C::A_MN ? 8192 : 16, 1024, kSwizzle128);
          const uint64_t bd = make_sdesc(b, C::B_MN ? 8192 : 16, 1024, kSwizzle128);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t acc = (kc > w.k0 || kk > 0) ? 1u : 0u;
            if constexpr (C::KIND == kKindI8) {
              if constexpr (PAIR)
                umma_i8_pair(d, ad + a_step * kk, bd + b_step * kk, idesc, acc);
              else
                umma_i8(d, ad + a_step * kk, bd + b_step * kk, idesc, acc);
            } else {
              if constexpr (PAIR)
                umma_ss_pair(d, ad + a_step * kk, bd + b_step * kk, idesc, acc);
              else
                umma_ss(d, ad + a_step * kk, bd + b_step * kk, idesc, acc);
            }
          }
          if constexpr (PAIR)
            umma_commit_pair_mc(&empty[st], 3);
          else
            umma_commit(&empty[st]);
        }
        if (ok) {
          if constexpr (PAIR)
            umma_commit_pair_mc(&acc_full[buf], 3);
          else
            umma_commit(&acc_full[buf]);
        }
      }
      if constexpr (PAIR)
        umma_commit_pair(fin);
      else
        umma_commit(fin);
      wait_drain(wc, fin, 0, 13);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    constexpr int kGroups = C::EW / 4;
    const int wg = warp >> 2;
    const int r = threadIdx.x & 127;  // row within the tile = TMEM lane
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t acc_empty_x[2] = {PAIR ? cluster_addr(&acc_empty[0], 0) : 0u,
                                     PAIR ? cluster_addr(&acc_empty[1], 0) : 0u};
    auto release = [&](int buf) {
      // this warp's last read of the accumulator
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          mbar_arrive_remote(acc_empty_x[buf]);
        else
          mbar_arrive(&acc_empty[buf]);
      }
    };
    if constexpr (EP::kStats) {
      // a warpgroup takes BN / kGroups consecutive columns of every tile
      constexpr int kSpan = C::BN / kGroups;
      typename EP::State st;
      int lt = 0, mt = -1;
      for (int t = t_begin; t < t_end; t += t_step, ++lt) {
        const Tile w = tile_at(t);
        const int buf = lt & 1;
        if (w.mt != mt) {
          if (mt >= 0) p.ep.end(st);
          mt = w.mt;
          p.ep.begin(st, w.m0 + r, w.m0 + r < p.M, mt, unit, wg);
        }
        if (!__all_sync(0xffffffffu, wait_x(&acc_full[buf], (lt >> 1) & 1, 8))) break;
        tc_fence_after();
        const uint32_t acc = tmem + lane_off + buf * C::BN;
#pragma unroll 1
        for (int c = wg * kSpan; c < (wg + 1) * kSpan; c += 32) {
          uint32_t z[32];
          __syncwarp();  // the TMEM loads want the whole warp
          tmem_ld32(acc + c, z);
          tmem_ld_wait();
          const int n0 = w.n0 + c;
          while (__any_sync(0xffffffffu, p.ep.next(st) < n0))
            if (p.ep.next(st) < n0) p.ep.skip(st);
          while (true) {
            // one asked-for column at a time, read again out of TMEM (registers cannot be indexed)
            const int want = p.ep.next(st);
            const uint32_t asking = __ballot_sync(0xffffffffu, want < n0 + 32);
            if (asking == 0) break;
            const int col = __shfl_sync(0xffffffffu, want, __ffs(asking) - 1);
            __syncwarp();
            const uint32_t v = tmem_ld1(acc + (col - w.n0));
            if (want == col) p.ep.take(st, v);
          }
          if (c + 32 >= (wg + 1) * kSpan) release(buf);
          p.ep.add(st, z, n0);
        }
      }
      if (mt >= 0) p.ep.end(st);
    } else {
      constexpr int kCols = 128 / EP::OUT_SIZE;  // columns of a step
      constexpr int kSub = kCols / 32;
      constexpr int kSteps = C::BN / kCols;
      // a warpgroup takes the column steps c with c % kGroups == wg
      uint8_t* box = smem + C::OFF_OUT + warp * C::BOX;
      float* cols = reinterpret_cast<float*>(smem + C::OFF_COL) + warp * 64;
      int lt = 0;
      for (int t = t_begin; t < t_end; t += t_step, ++lt) {
        const Tile w = tile_at(t);
        const int buf = lt & 1;
        const int m = w.m0 + r;
        const auto rv = p.ep.row(m, m < p.M);
        auto fetch_cols = [&](int c) {
          // this step's per-column values, one or two per lane
          if constexpr (EP::kCols) {
            __syncwarp();
#pragma unroll
            for (int h = 0; h < kSub; ++h) cols[h * 32 + lane] = p.ep.col(w.n0 + c * kCols + h * 32 + lane);
            __syncwarp();
          }
        };
        if (wg < kSteps) fetch_cols(wg);
        if (!__all_sync(0xffffffffu, wait_x(&acc_full[buf], (lt >> 1) & 1, 8))) break;
        tc_fence_after();
        const uint32_t acc = tmem + lane_off + buf * C::BN;
        const int warp_row = w.m0 + (warp & 3) * 32;
        if (wg >= kSteps) release(buf);
#pragma unroll 1
        for (int c = wg; c < kSteps; c += kGroups) {
          uint32_t z[kSub][32];
          __syncwarp();  // the TMEM loads want the whole warp
#pragma unroll
          for (int h = 0; h < kSub; ++h) tmem_ld32(acc + c * kCols + h * 32, z[h]);
          tmem_ld_wait();
          if (c + kGroups >= kSteps) release(buf);
          const int n0 = w.n0 + c * kCols;
          if (n0 >= p.N) continue;  // nothing of this step exists (warp-uniform)
          if (c != wg) fetch_cols(c);
          uint32_t words[32];
#pragma unroll
          for (int h = 0; h < kSub; ++h) p.ep.pack(z[h], rv, cols + h * 32, words + h * 16);
          if (lane == 0) bulk_wait_group_read0();  // the box's previous store has left it
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(box + box128_off(lane, j)) =
                make_uint4(words[4 * j], words[4 * j + 1], words[4 * j + 2], words[4 * j + 3]);
          if (p.ep.direct) {
            __syncwarp();
            using W = typename std::conditional<EP::OUT_SIZE == 2, uint16_t, uint32_t>::type;
            const int rows = min(32, p.M - warp_row);
            for (int i = 0; i < rows; ++i) {
              W* dst = static_cast<W*>(p.out) + (w.split * p.split_rows + warp_row + i) * p.ld_out + n0;
#pragma unroll
              for (int e = lane; e < kCols; e += 32)
                if (n0 + e < p.N)
                  dst[e] = *reinterpret_cast<const W*>(box + box128_off(i, e * EP::OUT_SIZE / 16) +
                                                       (e * EP::OUT_SIZE) % 16);
            }
            __syncwarp();
          } else {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_out(&p.tm_out, box, n0, (int)(w.split * p.split_rows) + warp_row, p.ep.add);
              bulk_commit_group();
            }
          }
        }
      }
      if (lane == 0) bulk_wait_group0();  // stores done before the CTA exits
    }
  }

  __syncwarp();
  tc_fence_before();
  if constexpr (PAIR)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == C::EW) {
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem, 2 * C::BN);
    else
      tmem_dealloc(tmem, 2 * C::BN);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
inline CUtensorMapDataType tile_dtype(int kind) {
  return kind == kKindI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                         : (kind == kKindBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
}

// Operand of `rows` (M or N) by `k` elements, ld elements between consecutive
// values of the strided dimension.  box_rows: rows one CTA stages (K-major).
template <class C>
int tile_operand_map(CUtensorMap* m, const void* base, bool mn_major, int64_t rows, int64_t k, int64_t ld,
                     int box_rows) {
  uint64_t dims[2] = {(uint64_t)(mn_major ? rows : k), (uint64_t)(mn_major ? k : rows)};
  uint64_t str[1] = {(uint64_t)ld * C::ESZ};
  uint32_t box[2] = {(uint32_t)(mn_major ? 64 : C::BK), (uint32_t)(mn_major ? C::BK : box_rows)};
  return encode_tensor_map(m, tile_dtype(C::KIND), 2, const_cast<void*>(base), dims, str, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
}

// Output of `rows` x `cols` in dtype (MT_F32, MT_F16 or MT_BF16), boxes of 32 rows x 128 bytes.
inline int tile_output_map(CUtensorMap* m, void* base, int dtype, int64_t rows, int64_t cols, int64_t ld) {
  const int sz = dtype == MT_F32 ? 4 : 2;
  uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows};
  uint64_t str[1] = {(uint64_t)ld * sz};
  uint32_t box[2] = {(uint32_t)(128 / sz), 32};
  const CUtensorMapDataType dt = dtype == MT_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : dtype == MT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return encode_tensor_map(m, dt, 2, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <class C, class EP>
int launch_tile_gemm(TileParams<EP>& prm, int splits, const char* name, cudaStream_t stream) {
  static_assert(std::is_trivially_copyable<EP>::value, "kernel parameter");
  prm.n_mt = (prm.M + C::TM - 1) / C::TM;
  prm.n_nt = (prm.N + C::BN - 1) / C::BN;
  const int64_t tiles = int64_t(prm.n_mt) * prm.n_nt * splits;
  if (tiles > 0x7fffffffLL) return MT_ERR_INVALID_ARGUMENT;
  prm.n_tiles = (int)tiles;
  prm.div_nt.init((uint32_t)prm.n_nt);
  prm.div_split.init((uint32_t)(prm.n_mt * prm.n_nt));
  constexpr int per_unit = C::PAIR ? 2 : 1;
  int units = (int)std::min<int64_t>(tiles, get_sm_count() / per_unit);
  if (prm.per_unit > 0) units = (int)((tiles + prm.per_unit - 1) / prm.per_unit);
  auto kern = tile_gemm_kernel<C, EP>;
  int st = set_smem_limit((const void*)kern, C::SMEM);
  if (st != MT_OK) return st;
  if constexpr (C::PAIR) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * 2));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t err = cudaLaunchKernelEx(&cfg, kern, prm);
    if (err != cudaSuccess) {
      set_last_error(name, err);
      return MT_ERR_LAUNCH;
    }
  } else {
    kern<<<units, C::kThreads, C::SMEM, stream>>>(prm);
  }
  return check_launch(name);
}

}  // namespace mt
