// Token embedding lookup with a scale, and its gradient by sorted tokens.
//
//   forward   y[n, :] = round(scale * W[id[n], :])
//   gradient  dW[v, :] = round(scale * sum_{n: id[n] = v} dy[n, :])   (dense, every row written)
//
// Reference: nn.Embedding of TradingModel (duoan/mega-trading
// src/mega_trading/model.py:20-147), whose gradient PyTorch computes.
//
// Forward: bound by HBM (N * dim elements written; the table stays in L2 at
// 16-bit sizes of this model).  One warp per token, 16-byte streaming stores:
// 262,144 x 768 in 158 us fp32 (7.2 TB/s of DRAM traffic, the 66 MB table missing
// one die's half of L2) and 74 us bf16.
//
// Gradient: bound by reading dy once.  The token ids are sorted with their
// positions (stable least-significant-digit radix sort, 8 bits a pass, written
// here: one block for up to 2,048 tokens, otherwise a histogram launch and one
// scatter launch per pass), so that the rows of dy which meet in one row of dW
// are neighbours in the sorted order.  The sorted order is cut into ranges of
// equal length, so a token that makes up a large share of the stream costs no
// more than any other, and runs of equal ids are summed in fp32 registers:
//   embed_reduce_bulk_kernel  two blocks per SM, one range each; a producer
//       warp gathers whole rows with bulk copies (cp.async.bulk) into a 96 KB
//       ring, so the loads in flight do not depend on registers or on where
//       runs end (rows of a multiple of 16 bytes): 262,144 x 768 fp32 in 146 us,
//       6.0 TB/s with dW's rows.  Every 64 rows of a run meet in a second fp32
//       accumulator, so the error of a long run does not grow with its range
//   embed_reduce_kernel       any width and alignment: a warp walks a chunk of
//       32 or 64 positions for one slab of columns
// A run that lies inside its range goes straight to dW; a run cut by a border
// leaves fp32 partial sums, at most two per range, which embed_join_kernel adds
// up (it also zeroes the rows no token chose).  Every sum has a fixed order (no
// atomics on values): results are the same each time.  Up to 256 tokens take one
// launch that looks each row's tokens up instead (no sort, no workspace).
//
// Ids outside [0, V) read nothing: their output row is zero, they add to no
// gradient and the status word is set.  Places holding padding_idx look up
// their row like any other and add to no gradient.
#include <algorithm>

#include "common.cuh"

namespace mt {
namespace {

constexpr uint32_t kKernelId = 7;
constexpr int kRounds = 4;  // 32-token rounds a warp ranks at a time
// Warps of a sort block: 16 halve the tiles whose histograms every block sums
// (whole gradient of 262,144 tokens x 768: 169 us, 8 warps 178), 8 start sooner
// (5,000 tokens: 35.8 us, 16 warps 40.4).
int sort_warps(int64_t n) { return n >= 65536 ? 16 : 8; }
constexpr int kOneRounds = 2;
constexpr int kOneBlock = 1024 * kOneRounds;  // tokens the single-block sort takes (whole gradient of 1,000
                                              // tokens x 768: 34.7 us, tiled 38.9; of 4,096: 41.6 / 36.5)
constexpr int kMaxTiles = 512;   // blocks of a sort pass (a block then takes several sub-tiles)

__device__ __forceinline__ int64_t load_id(const void* ids, int i64, int64_t n) {
  return i64 ? __ldg(static_cast<const int64_t*>(ids) + n) : (int64_t)__ldg(static_cast<const int32_t*>(ids) + n);
}

// ---------------------------------------------------------------------------
// vectors of E elements: 16 bytes of the wider of two types, or single
// elements 32 apart when a width or an address does not allow vectors
// ---------------------------------------------------------------------------
template <typename T, int E>
__device__ __forceinline__ void load_n(const T* p, float (&v)[E]) {
  constexpr int kPer = 16 / sizeof(T);
  if constexpr (E * sizeof(T) == 8) {
    const uint2 raw = __ldg(reinterpret_cast<const uint2*>(p));
    unpack2<T>(raw.x, v[0], v[1]);
    unpack2<T>(raw.y, v[2], v[3]);
  } else {
    static_assert(E % kPer == 0, "whole 16-byte words");
#pragma unroll
    for (int i = 0; i < E; i += kPer) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p + i));
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i + e] = __uint_as_float(w[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) unpack2<T>(w[e], v[i + 2 * e], v[i + 2 * e + 1]);
      }
    }
  }
}
// STREAM: written once and not read soon (leaves the cache to what is)
template <typename T, int E, bool STREAM = false>
__device__ __forceinline__ void store_n(T* p, const float (&v)[E]) {
  constexpr int kPer = 16 / sizeof(T);
  if constexpr (E * sizeof(T) == 8) {
    const uint2 q = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    if constexpr (STREAM)
      __stcs(reinterpret_cast<uint2*>(p), q);
    else
      *reinterpret_cast<uint2*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < E; i += kPer) {
      uint4 q;
      if constexpr (sizeof(T) == 4)
        q = make_uint4(__float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]),
                       __float_as_uint(v[i + 3]));
      else
        q = make_uint4(pack2<T>(v[i], v[i + 1]), pack2<T>(v[i + 2], v[i + 3]), pack2<T>(v[i + 4], v[i + 5]),
                       pack2<T>(v[i + 6], v[i + 7]));
      if constexpr (STREAM)
        __stcs(reinterpret_cast<uint4*>(p + i), q);
      else
        *reinterpret_cast<uint4*>(p + i) = q;
    }
  }
}

// A lane's E columns of a slab that starts at column c0.
template <int E, bool VEC>
struct Cols {
  static constexpr int kSlab = 32 * E;
  template <typename T>
  static __device__ __forceinline__ void load(const T* row, int c0, int dim, float (&v)[E]) {
    const int lane = lane_id();
    if constexpr (VEC) {
      if (c0 + lane * E < dim) {
        load_n<T, E>(row + c0 + lane * E, v);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = c0 + e * 32 + lane;
        v[e] = c < dim ? to_f32<T>(row[c]) : 0.f;
      }
    }
  }
  template <typename T, bool STREAM = false>
  static __device__ __forceinline__ void store(T* row, int c0, int dim, const float (&v)[E]) {
    const int lane = lane_id();
    if constexpr (VEC) {
      if (c0 + lane * E < dim) store_n<T, E, STREAM>(row + c0 + lane * E, v);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = c0 + e * 32 + lane;
        if (c < dim) row[c] = from_f32<T>(v[e]);
      }
    }
  }
};

// Elements per lane: 4 when either type is 32 bits wide, else 8.
template <typename A, typename B>
constexpr int lane_elems() {
  return sizeof(A) == 4 || sizeof(B) == 4 ? 4 : 8;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// TPW tokens per warp, one after the other: 4 keep the loads of 16-bit rows coming
// while a row is written, 1 spreads few tokens over more warps.  bf16 from a cold L2,
// us with 4 / 1: 8,000 tokens x 256 5.6 / 4.5, x 768 11.3 / 8.1; 18,944 (where 4
// begin) x 256 6.5 / 7.0, x 768 13.5 / 12.8; 131,072 x 256 22.5 / 29.7, x 768
// 51.5 / 54.7, x 1,024 70.1 / 70.8, x 2,048 150 / 141.  fp32 rows take 1.
template <typename TW, typename TO, bool VEC, int TPW>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const void* __restrict__ ids, int i64, int64_t n_tokens,
                                                        const TW* __restrict__ w, int64_t vocab, int dim, float scale,
                                                        TO* __restrict__ y, uint32_t* status) {
  constexpr int E = lane_elems<TW, TO>();
  using C = Cols<E, VEC>;
  // 768 columns in flight.  us with 768 / 1,024 / 512: 131,072 bf16 rows of 768 51.5 /
  // 58.2 / 48.3, of 1,024 70.1 / 76.4 / 62.9; 2,000 fp32 rows of 768 3.1 / 3.1 / 3.7,
  // 131,072 of 1,024 112.2 / 111.8 / 112.8
  constexpr int kSlabs = 24 / E;
  const int64_t n0 = (int64_t(blockIdx.x) * 8 + warp_id()) * TPW;
  int64_t mine = 0;
  if (lane_id() < TPW && n0 + lane_id() < n_tokens) mine = load_id(ids, i64, n0 + lane_id());
#pragma unroll
  for (int t = 0; t < TPW; ++t) {
    if (n0 + t >= n_tokens) return;
    const int64_t id = __shfl_sync(0xffffffffu, mine, t);
    TO* row = y + (n0 + t) * dim;
    if (id < 0 || id >= vocab) {
      if (lane_id() == 0) atomicCAS(status, 0u, (kKernelId << 16) | 0xEEEEu);
      const float zero[E] = {};
      for (int c0 = 0; c0 < dim; c0 += C::kSlab) C::store(row, c0, dim, zero);
      continue;
    }
    const TW* src = w + id * dim;
    for (int c0 = 0; c0 < dim; c0 += kSlabs * C::kSlab) {
      float v[kSlabs][E];
#pragma unroll
      for (int s = 0; s < kSlabs; ++s)
        if (c0 + s * C::kSlab < dim) C::load(src, c0 + s * C::kSlab, dim, v[s]);
#pragma unroll
      for (int s = 0; s < kSlabs; ++s)
        if (c0 + s * C::kSlab < dim) {
#pragma unroll
          for (int e = 0; e < E; ++e) v[s][e] *= scale;
          C::template store<TO, true>(row, c0 + s * C::kSlab, dim, v[s]);
        }
    }
  }
}

// ---------------------------------------------------------------------------
// stable radix sort of (id, position); places that add to no gradient carry
// the key V and end up last
// ---------------------------------------------------------------------------
struct SortIn {
  const void* ids;
  int i64;
  int64_t vocab, pad;  // pad < 0: none
  uint32_t* status;
};

__device__ __forceinline__ uint32_t key_of(const SortIn& in, int64_t id) {
  if (id < 0 || id >= in.vocab || id == in.pad) return (uint32_t)in.vocab;
  return (uint32_t)id;
}
// The first kernel of a gradient also reports ids outside the vocabulary.
__device__ __forceinline__ void report_id(const SortIn& in, int64_t id) {
  if (id < 0 || id >= in.vocab) atomicCAS(in.status, 0u, (kKernelId << 16) | 0xEEEEu);
}

// Rank of each of the tile's items among the items of its digit (in the order
// warp, round, lane), and the number of items per digit.  Items of warp w in
// round i are the i-th 32 of its R * 32 consecutive items.
template <int NW, int R>
__device__ __forceinline__ void rank_tile(const uint32_t (&digit)[R], uint32_t (&rank)[R], uint32_t (*cnt)[256],
                                          uint32_t* total) {
  const int w = warp_id(), lane = lane_id();
  for (int i = lane; i < 256; i += 32) cnt[w][i] = 0;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint32_t d = digit[i];  // 256: no item
    const uint32_t peers = __match_any_sync(0xffffffffu, d);
    const uint32_t before = d < 256 ? cnt[w][d] : 0u;
    rank[i] = before + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (d < 256 && lane == __ffs(peers) - 1) cnt[w][d] = before + __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  if (threadIdx.x < 256) {
    uint32_t sum = 0;
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      const uint32_t c = cnt[q][threadIdx.x];
      cnt[q][threadIdx.x] = sum;
      sum += c;
    }
    total[threadIdx.x] = sum;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (digit[i] < 256) rank[i] += cnt[w][digit[i]];
}

// Exclusive prefix sums of 256 values by the first 256 threads (8 warps);
// every thread of the block calls it.
__device__ __forceinline__ void scan256(const uint32_t* in, uint32_t* out, uint32_t* warp_tot) {
  uint32_t v = 0, x = 0;
  const int t = threadIdx.x;
  if (t < 256) {
    v = x = in[t];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane_id() >= o) x += y;
    }
    if (lane_id() == 31) warp_tot[warp_id()] = x;
  }
  __syncthreads();
  if (t < 256) {
    uint32_t base = 0;
    for (int q = 0; q < warp_id(); ++q) base += warp_tot[q];
    out[t] = base + x - v;
  }
  __syncthreads();
}

// One block: the whole sort in shared memory.
__global__ void __launch_bounds__(1024) embed_sort_small_kernel(SortIn in, int n_tokens, int bits, uint2* out,
                                                                uint2* seg) {
  __shared__ uint32_t cnt[32][256];
  __shared__ uint32_t total[256], base[256], warp_tot[8];
  __shared__ uint16_t pos_s[kOneBlock];
  uint32_t key[kOneRounds], pos[kOneRounds], digit[kOneRounds], rank[kOneRounds];
  // the id ranges start out empty
  for (int64_t v = threadIdx.x; v <= in.vocab; v += 1024) seg[v] = make_uint2(0u, 0u);
  const int first = warp_id() * (32 * kOneRounds) + lane_id();
#pragma unroll
  for (int i = 0; i < kOneRounds; ++i) {
    pos[i] = first + i * 32;
    const int64_t id = (int)pos[i] < n_tokens ? load_id(in.ids, in.i64, pos[i]) : 0;
    key[i] = key_of(in, id);
    report_id(in, id);
  }
  for (int shift = 0; shift < bits; shift += 8) {
#pragma unroll
    for (int i = 0; i < kOneRounds; ++i) digit[i] = first + i * 32 < n_tokens ? (key[i] >> shift) & 255u : 256u;
    rank_tile<32, kOneRounds>(digit, rank, cnt, total);
    scan256(total, base, warp_tot);
    const bool last = shift + 8 >= bits;
    // the order of this pass: the place of each item (pos_s holds the permutation)
#pragma unroll
    for (int i = 0; i < kOneRounds; ++i)
      if (digit[i] < 256) {
        const uint32_t dst = base[digit[i]] + rank[i];
        if (last)
          out[dst] = make_uint2(key[i], pos[i]);
        else
          pos_s[dst] = (uint16_t)pos[i];
      }
    __syncthreads();
    if (!last) {
#pragma unroll
      for (int i = 0; i < kOneRounds; ++i)
        if (first + i * 32 < n_tokens) {
          pos[i] = pos_s[first + i * 32];
          key[i] = key_of(in, load_id(in.ids, in.i64, pos[i]));
        }
      __syncthreads();
    }
  }
}

// Histogram of the first digit per tile; clears the later passes' histograms
// and the id ranges.
template <int NW>
__global__ void __launch_bounds__(NW * 32) embed_hist_kernel(SortIn in, int64_t n_tokens, int64_t tile,
                                                         uint32_t* __restrict__ hist, int64_t hist_words, uint2* seg) {
  constexpr int kSortThreads = NW * 32, kSubTile = kSortThreads * kRounds;
  __shared__ uint32_t h[256];
  if (threadIdx.x < 256) h[threadIdx.x] = 0;
  const int64_t gid = int64_t(blockIdx.x) * kSortThreads + threadIdx.x, gsz = int64_t(gridDim.x) * kSortThreads;
  const int64_t own = int64_t(gridDim.x) * 256;  // this pass's histograms
  for (int64_t i = own + gid; i < hist_words; i += gsz) hist[i] = 0;
  for (int64_t v = gid; v <= in.vocab; v += gsz) seg[v] = make_uint2(0u, 0u);
  __syncthreads();
  const int64_t lo = blockIdx.x * tile, hi = min(lo + tile, n_tokens);
  for (int64_t s0 = lo; s0 < hi; s0 += kSubTile) {
    int64_t id[kRounds];
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int64_t n = s0 + i * kSortThreads + threadIdx.x;
      id[i] = n < hi ? load_id(in.ids, in.i64, n) : -1;
    }
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const bool live = s0 + i * kSortThreads + threadIdx.x < hi;
      const uint32_t d = live ? key_of(in, id[i]) & 255u : 256u;
      if (live) report_id(in, id[i]);
      const uint32_t peers = __match_any_sync(0xffffffffu, d);
      if (d < 256 && lane_id() == __ffs(peers) - 1) atomicAdd(&h[d], (uint32_t)__popc(peers));
    }
  }
  __syncthreads();
  if (threadIdx.x < 256) hist[int64_t(blockIdx.x) * 256 + threadIdx.x] = h[threadIdx.x];
}

// One stable pass: items move to (items of smaller digits) + (items of the same
// digit in earlier tiles) + (rank inside the tile).  FIRST reads the ids, later
// passes the pairs.  next != NULL: counts the next digit per destination tile
// (integer atomics: the counts do not depend on their order).
template <bool FIRST, int NW>
__global__ void __launch_bounds__(NW * 32) embed_scatter_kernel(SortIn in, const uint2* __restrict__ src, int64_t n_tokens,
                                                            int64_t tile, int shift, const uint32_t* __restrict__ hist,
                                                            uint32_t* __restrict__ next, uint2* __restrict__ dst) {
  constexpr int kSubTile = NW * 32 * kRounds;
  __shared__ __align__(16) uint32_t cnt[NW][256];
  __shared__ uint32_t total[256], base[256], warp_tot[8];
  // this block's items of the first sub-tile, on their way while the places are summed
  const int64_t lo = blockIdx.x * tile, hi = min(lo + tile, n_tokens);
  uint32_t key[kRounds], pos[kRounds];
  auto fetch = [&](int64_t s0) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int64_t n = s0 + warp_id() * (32 * kRounds) + i * 32 + lane_id();
      if constexpr (FIRST) {
        key[i] = key_of(in, n < hi ? load_id(in.ids, in.i64, n) : 0);
        pos[i] = (uint32_t)n;
      } else {
        const uint2 q = n < hi ? src[n] : make_uint2(0u, 0u);
        key[i] = q.x;
        pos[i] = q.y;
      }
    }
  };
  fetch(lo);
  {
    // this tile's first place for every digit: kParts threads share a column of
    // four digits, each takes every kParts-th tile
    constexpr int kParts = NW / 2;
    const int quad = threadIdx.x & 63, part = threadIdx.x >> 6;
    const uint4* col = reinterpret_cast<const uint4*>(hist) + quad;
    const int tiles = gridDim.x, me = blockIdx.x;
    uint4 all = make_uint4(0u, 0u, 0u, 0u), before = all;
#pragma unroll 8
    for (int b = part; b < tiles; b += kParts) {
      const uint4 c = __ldg(col + int64_t(b) * 64);
      const uint32_t m = b < me ? 0xffffffffu : 0u;
      all.x += c.x; all.y += c.y; all.z += c.z; all.w += c.w;
      before.x += c.x & m; before.y += c.y & m; before.z += c.z & m; before.w += c.w & m;
    }
    *reinterpret_cast<uint4*>(&cnt[part][quad * 4]) = all;
    *reinterpret_cast<uint4*>(&cnt[kParts + part][quad * 4]) = before;
    __syncthreads();
    const int d = threadIdx.x;
    uint32_t mine = 0;
    if (d < 256) {
      uint32_t sum = 0;
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        sum += cnt[i][d];
        mine += cnt[kParts + i][d];
      }
      total[d] = sum;
    }
    __syncthreads();
    scan256(total, base, warp_tot);
    if (d < 256) base[d] += mine;
    __syncthreads();
  }
  for (int64_t s0 = lo; s0 < hi; s0 += kSubTile) {
    if (s0 > lo) fetch(s0);
    uint32_t digit[kRounds], rank[kRounds];
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int64_t n = s0 + warp_id() * (32 * kRounds) + i * 32 + lane_id();
      digit[i] = n < hi ? (key[i] >> shift) & 255u : 256u;
    }
    rank_tile<NW, kRounds>(digit, rank, cnt, total);
#pragma unroll
    for (int i = 0; i < kRounds; ++i)
      if (digit[i] < 256) {
        const uint32_t at = base[digit[i]] + rank[i];
        dst[at] = make_uint2(key[i], pos[i]);
        if (next != nullptr)
          atomicAdd(&next[int64_t(at / (uint32_t)tile) * 256 + ((key[i] >> (shift + 8)) & 255u)], 1u);
      }
    __syncthreads();
    if (threadIdx.x < 256) base[threadIdx.x] += total[threadIdx.x];
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// sums of equal ids
// ---------------------------------------------------------------------------
// One warp: one chunk of the sorted order, one slab of columns.  Runs cut by a
// chunk border leave partial sums: slot 0 for a run that began in an earlier
// chunk, slot 1 for one that begins here and goes on.
template <typename TG, typename TD, bool VEC>
__global__ void __launch_bounds__(256) embed_reduce_kernel(const uint2* __restrict__ sorted, int64_t n_tokens,
                                                           int chunk, int slabs, const TG* __restrict__ dy,
                                                           uint32_t vocab, int dim, float scale, TD* __restrict__ dw,
                                                           float* __restrict__ partial, uint2* __restrict__ seg) {
  constexpr int E = lane_elems<TG, TD>();
  using C = Cols<E, VEC>;
  const int lane = lane_id();
  const int64_t unit = int64_t(blockIdx.x) * 8 + warp_id();
  const int64_t ch = unit / slabs;
  const int slab = int(unit - ch * slabs), c0 = slab * C::kSlab;
  const int64_t lo = ch * chunk, hi = min(lo + chunk, n_tokens);
  if (lo >= hi) return;
  // 0xffffffff: no neighbour (ids are below 2^31)
  uint32_t prev = lo > 0 ? sorted[lo - 1].x : 0xffffffffu;
  bool begins = true;  // the current run begins in this chunk
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  bool first = true;
  for (int64_t b0 = lo; b0 < hi; b0 += 32) {
    const int nb = (int)min((int64_t)32, hi - b0);
    uint2 mine = make_uint2(0xffffffffu, 0u);
    if (lane < nb) mine = __ldg(sorted + b0 + lane);
    // key of the item after this batch
    uint32_t after = b0 + nb < n_tokens ? __ldg(&sorted[b0 + nb].x) : 0xffffffffu;
#pragma unroll 1
    for (int j0 = 0; j0 < nb; j0 += 8) {
      float v[8][E];
      uint32_t key[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        key[j] = __shfl_sync(0xffffffffu, mine.x, j0 + j);
        const uint32_t pos = __shfl_sync(0xffffffffu, mine.y, j0 + j);
        if (j0 + j < nb && key[j] < vocab) C::load(dy + int64_t(pos) * dim, c0, dim, v[j]);
      }
      const uint32_t beyond = j0 + 8 < 32 ? __shfl_sync(0xffffffffu, mine.x, (j0 + 8) & 31) : 0xffffffffu;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j0 + j >= nb || key[j] >= vocab) continue;
        const int64_t at = b0 + j0 + j;
        if (first || key[j] != prev) {
          // a run starts here, unless it came in from the previous chunk
          begins = key[j] != prev;
          if (begins && slab == 0 && lane == 0) seg[key[j]].x = (uint32_t)at;
        }
        first = false;
        prev = key[j];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += v[j][e];
        const uint32_t next = j0 + j + 1 >= nb ? after : (j < 7 ? key[j < 7 ? j + 1 : 7] : beyond);
        const bool ends = next != key[j];
        if (ends && slab == 0 && lane == 0) seg[key[j]].y = (uint32_t)at + 1u;
        if (ends || at + 1 == hi) {
          if (begins && ends) {
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = acc[e] * scale;
            C::store(dw + int64_t(key[j]) * dim, c0, dim, o);
          } else {
            C::store(partial + (ch * 2 + (begins ? 1 : 0)) * dim, c0, dim, acc);
          }
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = 0.f;
        }
      }
    }
  }
}

// The same sums for rows of a multiple of 16 bytes.  A block owns one range of
// the sorted order for one slab of columns (up to 4 KB of a row); warps 0-7 add
// (thread = 16 bytes of the row), warp 8 gathers.  A ring stage holds 16 KB:
// `rp` rows with the ids they belong to.
constexpr int kBulkStage = 16384;
constexpr int kBulkStages = 6;
constexpr int kBulkThreads = 9 * 32;
constexpr int kBulkSlab = 4096;  // bytes
enum : uint32_t { kRunStarts = 1, kRunEnds = 2, kNoRow = 4 };

struct BulkSmem {
  uint8_t ring[kBulkStages][kBulkStage];
  uint2 meta[kBulkStages][32];  // {id, flags}
  uint64_t full[kBulkStages], empty[kBulkStages];
  int abort_flag;
};

// 16-byte aligned copy of `bytes` (a multiple of 16) from global to this CTA's
// shared memory, completing on its mbarrier.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <typename TG, typename TD>
__global__ void __launch_bounds__(kBulkThreads) embed_reduce_bulk_kernel(
    const uint2* __restrict__ sorted, int64_t n_tokens, int64_t range, int rp, const TG* __restrict__ dy,
    uint32_t vocab, int dim, float scale, TD* __restrict__ dw, float* __restrict__ partial, uint2* __restrict__ seg,
    uint32_t* status) {
  constexpr int E = 16 / sizeof(TG);
  extern __shared__ __align__(128) uint8_t raw[];
  BulkSmem& sm = *reinterpret_cast<BulkSmem*>(raw);
  const int64_t lo = int64_t(blockIdx.x) * range, hi = min(lo + range, n_tokens);
  const int c0 = blockIdx.y * (kBulkSlab / (int)sizeof(TG));
  const int cols = min(dim - c0, kBulkSlab / (int)sizeof(TG));
  const uint32_t bytes = cols * (uint32_t)sizeof(TG);
  const int adders = (int)(bytes + 511) / 512;  // warps that own columns
  const int lane = lane_id(), warp = warp_id();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBulkStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], adders);
    }
    sm.abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  const WaitCtx wc{status, &sm.abort_flag, kKernelId};
  if (warp == 8) {
    // ------------------------------------------------------------ gather
    uint32_t prev = lo > 0 ? __ldg(&sorted[lo - 1].x) : 0xffffffffu;  // ids are below 2^31
    uint2 mine = lo + lane < hi ? __ldg(sorted + lo + lane) : make_uint2(0xffffffffu, 0u);
    int it = 0;
    bool ok = true;
    for (int64_t b0 = lo; ok && b0 < hi; b0 += 32) {
      // the pair after this batch's last one decides where its run ends
      uint2 later = b0 + 32 + lane < n_tokens ? __ldg(sorted + b0 + 32 + lane) : make_uint2(0xffffffffu, 0u);
      const bool in = b0 + lane < hi;
      uint32_t before = __shfl_up_sync(0xffffffffu, mine.x, 1);
      if (lane == 0) before = prev;
      uint32_t after = __shfl_down_sync(0xffffffffu, mine.x, 1);
      const uint32_t beyond = __shfl_sync(0xffffffffu, later.x, 0);
      if (lane == 31) after = beyond;
      if (b0 + lane + 1 == hi && hi < n_tokens) after = __ldg(&sorted[hi].x);
      const bool row = in && mine.x < vocab;
      const uint32_t flags = (mine.x != before ? kRunStarts : 0u) | (mine.x != after ? kRunEnds : 0u) |
                             (row ? 0u : kNoRow);
      prev = __shfl_sync(0xffffffffu, mine.x, 31);
      for (int g = 0; g < 32 && b0 + g < hi; g += rp, ++it) {
        const int st = it % kBulkStages;
        // every lane waits, and the warp leaves together when one of them gives up
        if (it >= kBulkStages &&
            !__all_sync(0xffffffffu, wait_bounded(wc, &sm.empty[st], ((it / kBulkStages) & 1) ^ 1, 1))) {
          ok = false;
          break;
        }
        const bool here = lane >= g && lane < g + rp;
        if (here) sm.meta[st][lane - g] = make_uint2(mine.x, flags);
        const uint32_t n = __popc(__ballot_sync(0xffffffffu, here && row));
        // lane 0's arrival releases the other lanes' entries too (a stage without
        // rows is complete with it)
        __syncwarp();
        if (lane == 0) {
          if (n > 0)
            mbar_arrive_expect_tx(&sm.full[st], n * bytes);
          else
            mbar_arrive(&sm.full[st]);
        }
        __syncwarp();
        if (here && row)
          bulk_load(&sm.ring[st][(lane - g) * bytes], dy + int64_t(mine.y) * dim + c0, bytes, &sm.full[st]);
      }
      mine = b0 + 32 + lane < hi ? later : make_uint2(0xffffffffu, 0u);
    }
    if (!ok || sm.abort_flag) {
      for (int j = (it > kBulkStages ? it - kBulkStages : 0); j < it; ++j)
        wait_drain(wc, &sm.full[j % kBulkStages], (j / kBulkStages) & 1, 11);
    }
  } else if (warp < adders) {
    // ------------------------------------------------------------ add
    const bool own = threadIdx.x * 16 < (int)bytes;
    const int col = c0 + threadIdx.x * E;
    // a run's latest rows, 64 at most, and the sum of those before them: a long run
    // carries about 64 + rows / 64 roundings instead of one per row
    float acc[E], sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = sum[e] = 0.f;
    int held = 0;        // rows in acc, or more
    bool begins = true;  // the current run begins in this range
    int64_t at = lo;
    for (int it = 0; at < hi; ++it) {
      const int st = it % kBulkStages;
      if (held + rp > 64) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          sum[e] += acc[e];
          acc[e] = 0.f;
        }
        held = 0;
      }
      held += rp;
      if (!__all_sync(0xffffffffu, wait_bounded(wc, &sm.full[st], (it / kBulkStages) & 1, 2))) break;
      const int rows = (int)min((int64_t)rp, hi - at);
      // four rows at a time: their values and run flags are fetched together
      for (int i0 = 0; i0 < rows; i0 += 4) {
        uint2 m[4];
        uint4 q[4];
        uint32_t any = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m[j] = sm.meta[st][i0 + j];
          if (i0 + j >= rows) m[j].y = kNoRow;
          any |= m[j].y;
          q[j] = *reinterpret_cast<const uint4*>(&sm.ring[st][own ? (i0 + j) * bytes + threadIdx.x * 16 : 0]);
        }
        auto add = [&](const uint4& v) {
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
          if constexpr (sizeof(TG) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += __uint_as_float(w[e]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float a, b;
              unpack2<TG>(w[e], a, b);
              acc[2 * e] += a;
              acc[2 * e + 1] += b;
            }
          }
        };
        if (any == 0 && at > lo && at + 4 < hi) {  // inside one run
#pragma unroll
          for (int j = 0; j < 4; ++j) add(q[j]);
          at += 4;
          continue;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (i0 + j >= rows) break;
          const int64_t here = at++;
          if (m[j].y & kNoRow) continue;
          if (m[j].y & kRunStarts) {
            begins = true;
            if (blockIdx.y == 0 && threadIdx.x == 0) seg[m[j].x].x = (uint32_t)here;
          } else if (here == lo) {
            begins = false;
          }
          add(q[j]);
          const bool ends = m[j].y & kRunEnds;
          if (ends && blockIdx.y == 0 && threadIdx.x == 0) seg[m[j].x].y = (uint32_t)here + 1u;
          if (ends || here + 1 == hi) {
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += sum[e];
            if (own) {
              if (begins && ends) {
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] *= scale;
                store_n<TD, E>(dw + int64_t(m[j].x) * dim + col, acc);
              } else {
                store_n<float, E>(partial + (int64_t(blockIdx.x) * 2 + (begins ? 1 : 0)) * dim + col, acc);
              }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = sum[e] = 0.f;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[st]);
    }
  }
  __syncthreads();
}

// Rows no token chose become zero; runs cut by range borders become the sum of
// their partial sums.  A warp takes 32 ids and one slab of columns; a run of
// more than kWide partial sums is shared by the block's warps.
template <typename TD, int E, bool VEC>
__global__ void __launch_bounds__(256) embed_join_kernel(const uint2* __restrict__ seg, int64_t vocab, int64_t range,
                                                         const float* __restrict__ partial, int dim, float scale,
                                                         TD* __restrict__ dw) {
  using C = Cols<E, VEC>;
  constexpr int kWide = 16, kBatch = 32 / E;
  __shared__ float red[8][32 * E];
  __shared__ uint32_t wide[256];
  __shared__ int n_wide;
  if (threadIdx.x == 0) n_wide = 0;
  __syncthreads();
  const int c0 = blockIdx.y * C::kSlab;
  const int lane = lane_id(), w = warp_id();
  const int64_t v0 = int64_t(blockIdx.x) * 256 + w * 32;
  const uint2 mine = v0 + lane < vocab ? __ldg(seg + v0 + lane) : make_uint2(0u, 1u);
  // ranges the run touches; a run inside one range was written by the reduction
  const int64_t a = mine.x / (uint64_t)range, b = (mine.y - (mine.y > 0 ? 1 : 0)) / (uint64_t)range;
  const bool none = mine.x == mine.y;
  uint32_t todo = __ballot_sync(0xffffffffu, none);
  float zero[E];
#pragma unroll
  for (int e = 0; e < E; ++e) zero[e] = 0.f;
  for (; todo != 0; todo &= todo - 1) C::store(dw + (v0 + __ffs(todo) - 1) * dim, c0, dim, zero);
  // partial sums lo .. hi - 1 of a run whose first one is `head` (slot 1)
  auto sum = [&](int64_t lo, int64_t hi, int64_t head, float(&acc)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int64_t q = lo; q < hi; q += kBatch) {
      float v[kBatch][E];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (q + j < hi) C::load(partial + ((q + j) * 2 + (q + j == head ? 1 : 0)) * dim, c0, dim, v[j]);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (q + j < hi)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += v[j][e];
    }
  };
  const bool cut = !none && a != b;
  if (cut && b - a >= kWide) wide[atomicAdd(&n_wide, 1)] = (uint32_t)(w * 32 + lane);
  for (todo = __ballot_sync(0xffffffffu, cut && b - a < kWide); todo != 0; todo &= todo - 1) {
    const int i = __ffs(todo) - 1;
    const int64_t ra = __shfl_sync(0xffffffffu, a, i), rb = __shfl_sync(0xffffffffu, b, i);
    float acc[E];
    sum(ra, rb + 1, ra, acc);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= scale;
    C::store(dw + (v0 + i) * dim, c0, dim, acc);
  }
  __syncthreads();
  for (int k = 0; k < n_wide; ++k) {  // in any order: each run is its own sum
    const int64_t v = int64_t(blockIdx.x) * 256 + wide[k];
    const uint2 run = __ldg(seg + v);
    const int64_t ra = run.x / (uint64_t)range, rb = (run.y - 1) / (uint64_t)range;
    const int64_t per = (rb + 1 - ra + 7) / 8;
    float acc[E];
    sum(ra + w * per, min(ra + (w + 1) * per, rb + 1), ra, acc);
#pragma unroll
    for (int e = 0; e < E; ++e) red[w][e * 32 + lane] = acc[e];
    __syncthreads();
    if (w == 0) {
#pragma unroll
      for (int q = 1; q < 8; ++q)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += red[q][e * 32 + lane];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= scale;
      C::store(dw + v * dim, c0, dim, acc);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// a few tokens: one launch, no workspace
// ---------------------------------------------------------------------------
// A block writes 32 rows of dW and a warp four of them: it looks its ids up in
// the token list (in shared memory) and adds the rows of dy that name them, in
// the order of their positions, eight at a time.  For up to kFew tokens the
// whole list is 256 compares per row and the longest sum 32 steps.
constexpr int kFew = 256;

template <typename TG, typename TD, bool VEC>
__global__ void __launch_bounds__(256) embed_few_kernel(SortIn in, int n_tokens, const TG* __restrict__ dy, int dim,
                                                        float scale, TD* __restrict__ dw) {
  constexpr int E = lane_elems<TG, TD>();
  using C = Cols<E, VEC>;
  __shared__ uint32_t keys[kFew];
  __shared__ uint16_t found[8][kFew];
  const int lane = lane_id(), w = warp_id();
  {
    const int i = threadIdx.x;
    const int64_t id = i < n_tokens ? load_id(in.ids, in.i64, i) : 0;
    keys[i] = i < n_tokens ? key_of(in, id) : 0xffffffffu;
    if (blockIdx.x == 0 && i < n_tokens) report_id(in, id);
  }
  __syncthreads();
  for (int r = 0; r < 4; ++r) {
    const int64_t v = int64_t(blockIdx.x) * 32 + w * 4 + r;
    if (v >= in.vocab) break;
    int count = 0;
    for (int i0 = 0; i0 < n_tokens; i0 += 32) {
      const uint32_t hits = __ballot_sync(0xffffffffu, keys[i0 + lane] == (uint32_t)v);
      if (hits >> lane & 1u) found[w][count + __popc(hits & ((1u << lane) - 1u))] = (uint16_t)(i0 + lane);
      count += __popc(hits);
    }
    __syncwarp();
    for (int c0 = 0; c0 < dim; c0 += C::kSlab) {
      float acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      for (int q = 0; q < count; q += 8) {
        float x[8][E];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (q + j < count) {
            C::load(dy + int64_t(found[w][q + j]) * dim, c0, dim, x[j]);
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[j][e] = 0.f;
          }
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
          acc[e] += ((x[0][e] + x[1][e]) + (x[2][e] + x[3][e])) + ((x[4][e] + x[5][e]) + (x[6][e] + x[7][e]));
      }
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= scale;
      C::store(dw + v * dim, c0, dim, acc);
    }
    __syncwarp();
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename F>
int with_type(int code, F&& f) {
  switch (code) {
    case MT_F32: return f(float{});
    case MT_F16: return f(__half{});
    case MT_BF16: return f(__nv_bfloat16{});
    default: return MT_ERR_UNSUPPORTED_DTYPE;
  }
}
bool known(int code) { return code == MT_F32 || code == MT_F16 || code == MT_BF16; }

struct EmbedPlan {
  int bits, passes, chunk;
  int64_t tile, tiles, chunks;
  int64_t off_pairs[2], off_hist, hist_words, off_seg, off_part, bytes;
};

EmbedPlan plan_embed(int64_t n, int64_t vocab, int64_t dim) {
  EmbedPlan pl;
  pl.bits = 1;
  while ((int64_t(1) << pl.bits) < vocab + 1) ++pl.bits;
  pl.passes = (pl.bits + 7) / 8;
  const int64_t sub_tile = sort_warps(n) * 32 * kRounds;
  pl.tile = sub_tile;
  while ((n + pl.tile - 1) / pl.tile > kMaxTiles) pl.tile += sub_tile;
  pl.tiles = (n + pl.tile - 1) / pl.tile;
  pl.chunk = n <= 32768 ? 32 : 64;
  pl.chunks = (n + pl.chunk - 1) / pl.chunk;
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  int64_t at = 0;
  for (int i = 0; i < 2; ++i) {
    pl.off_pairs[i] = at;
    at += up(n * 8);
  }
  pl.off_hist = at;
  pl.hist_words = pl.passes * pl.tiles * 256;
  at += up(pl.hist_words * 4);
  pl.off_seg = at;
  at += up((vocab + 1) * 8);
  pl.off_part = at;
  at += up(pl.chunks * 2 * dim * 4);
  pl.bytes = at;
  return pl;
}

// Sort of more than kOneBlock tokens; pass p ends in pairs[p & 1].
template <int NW>
int sort_tiled(const SortIn& in, int64_t n, const EmbedPlan& pl, uint32_t* hist, uint2* seg, uint2* const (&pairs)[2],
               cudaStream_t s) {
  const unsigned grid = (unsigned)pl.tiles;
  embed_hist_kernel<NW><<<grid, NW * 32, 0, s>>>(in, n, pl.tile, hist, pl.hist_words, seg);
  int st = check_launch("embedding_bwd_hist");
  for (int p = 0; st == MT_OK && p < pl.passes; ++p) {
    const uint32_t* h = hist + int64_t(p) * pl.tiles * 256;
    uint32_t* next = p + 1 < pl.passes ? hist + int64_t(p + 1) * pl.tiles * 256 : nullptr;
    if (p == 0)
      embed_scatter_kernel<true, NW><<<grid, NW * 32, 0, s>>>(in, nullptr, n, pl.tile, 0, h, next, pairs[0]);
    else
      embed_scatter_kernel<false, NW><<<grid, NW * 32, 0, s>>>(in, pairs[(p - 1) & 1], n, pl.tile, 8 * p, h, next,
                                                               pairs[p & 1]);
    st = check_launch("embedding_bwd_scatter");
  }
  return st;
}

int check_embed(int64_t n, int64_t vocab, int64_t dim) {
  if (n < 0 || vocab <= 0 || dim <= 0) return MT_ERR_INVALID_ARGUMENT;
  // positions and ids are 32-bit, a launch covers 8 tokens per block
  if (n > 0x7fffffffLL || vocab >= 0x7fffffffLL || dim > 0x7fffffffLL / 8) return MT_ERR_INVALID_ARGUMENT;
  return MT_OK;
}

}  // namespace
}  // namespace mt

using namespace mt;

extern "C" int mt_embedding_fwd(const void* ids, int ids_i64, int64_t n, const void* weight, int w_dtype,
                                int64_t vocab, int64_t dim, float scale, void* out, int out_dtype, uint32_t* status,
                                void* stream) {
  int st = check_embed(n, vocab, dim);
  if (st != MT_OK) return st;
  if (!known(w_dtype) || !known(out_dtype)) return MT_ERR_UNSUPPORTED_DTYPE;
  if (n == 0) return MT_OK;
  if (ids == nullptr || weight == nullptr || out == nullptr || status == nullptr) return MT_ERR_INVALID_ARGUMENT;
  if ((st = bind_device_of(weight)) != MT_OK) return st;
  auto s = static_cast<cudaStream_t>(stream);
  return with_type(w_dtype, [&](auto wv) {
    return with_type(out_dtype, [&](auto ov) {
      using TW = decltype(wv);
      using TO = decltype(ov);
      const bool vec = on16(weight) && on16(out) && dim % lane_elems<TW, TO>() == 0;
      const bool four = sizeof(TO) == 2 && n >= 128 * int64_t(get_sm_count());
      auto kern = four ? (vec ? embed_fwd_kernel<TW, TO, true, 4> : embed_fwd_kernel<TW, TO, false, 4>)
                       : (vec ? embed_fwd_kernel<TW, TO, true, 1> : embed_fwd_kernel<TW, TO, false, 1>);
      const int64_t per_block = four ? 32 : 8;
      kern<<<(unsigned)((n + per_block - 1) / per_block), 256, 0, s>>>(
          ids, ids_i64, n, static_cast<const TW*>(weight), vocab, (int)dim, scale, static_cast<TO*>(out), status);
      return check_launch("embedding_fwd");
    });
  });
}

extern "C" int64_t mt_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t dim) {
  if (n <= kFew || check_embed(n, vocab, dim) != MT_OK) return 0;
  return plan_embed(n, vocab, dim).bytes;
}

extern "C" int mt_embedding_bwd(const void* ids, int ids_i64, int64_t n, const void* dout, int dout_dtype,
                                int64_t vocab, int64_t dim, float scale, int64_t padding_idx, void* dweight,
                                int dw_dtype, void* workspace, int64_t workspace_bytes, uint32_t* status,
                                void* stream) {
  int st = check_embed(n, vocab, dim);
  if (st != MT_OK) return st;
  if (!known(dout_dtype) || !known(dw_dtype)) return MT_ERR_UNSUPPORTED_DTYPE;
  if (padding_idx >= vocab) return MT_ERR_INVALID_ARGUMENT;
  if (dweight == nullptr) return MT_ERR_INVALID_ARGUMENT;
  auto s = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    cudaError_t e = cudaMemsetAsync(dweight, 0, size_t(vocab) * dim * (dw_dtype == MT_F32 ? 4 : 2), s);
    if (e != cudaSuccess) {
      set_last_error("cudaMemsetAsync(dweight)", e);
      return MT_ERR_LAUNCH;
    }
    return MT_OK;
  }
  if (ids == nullptr || dout == nullptr || status == nullptr) return MT_ERR_INVALID_ARGUMENT;
  if (n <= kFew) {
    if ((st = bind_device_of(dweight)) != MT_OK) return st;
    const SortIn few{ids, ids_i64, vocab, padding_idx < 0 ? int64_t(-1) : padding_idx, status};
    return with_type(dout_dtype, [&](auto gv) {
      return with_type(dw_dtype, [&](auto dv) {
        using TG = decltype(gv);
        using TD = decltype(dv);
        const bool vec = on16(dout) && on16(dweight) && dim % lane_elems<TG, TD>() == 0;
        auto kern = vec ? embed_few_kernel<TG, TD, true> : embed_few_kernel<TG, TD, false>;
        kern<<<(unsigned)((vocab + 31) / 32), 256, 0, s>>>(few, (int)n, static_cast<const TG*>(dout), (int)dim, scale,
                                                           static_cast<TD*>(dweight));
        return check_launch("embedding_bwd_few");
      });
    });
  }
  const EmbedPlan pl = plan_embed(n, vocab, dim);
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0 || workspace_bytes < pl.bytes)
    return MT_ERR_WORKSPACE;
  if ((st = bind_device_of(dweight)) != MT_OK) return st;
  char* ws = static_cast<char*>(workspace);
  uint2* pairs[2] = {reinterpret_cast<uint2*>(ws + pl.off_pairs[0]), reinterpret_cast<uint2*>(ws + pl.off_pairs[1])};
  uint32_t* hist = reinterpret_cast<uint32_t*>(ws + pl.off_hist);
  uint2* seg = reinterpret_cast<uint2*>(ws + pl.off_seg);
  float* partial = reinterpret_cast<float*>(ws + pl.off_part);
  const SortIn in{ids, ids_i64, vocab, padding_idx < 0 ? int64_t(-1) : padding_idx, status};
  uint2* sorted = pairs[0];
  if (n <= kOneBlock) {
    embed_sort_small_kernel<<<1, 1024, 0, s>>>(in, (int)n, pl.bits, sorted, seg);
    if ((st = check_launch("embedding_bwd_sort")) != MT_OK) return st;
  } else {
    st = sort_warps(n) == 16 ? sort_tiled<16>(in, n, pl, hist, seg, pairs, s) : sort_tiled<8>(in, n, pl, hist, seg, pairs, s);
    if (st != MT_OK) return st;
    sorted = pairs[(pl.passes - 1) & 1];
  }
  return with_type(dout_dtype, [&](auto gv) {
    return with_type(dw_dtype, [&](auto dv) {
      using TG = decltype(gv);
      using TD = decltype(dv);
      constexpr int E = lane_elems<TG, TD>();
      const bool vec = on16(dout) && on16(dweight) && dim % E == 0 && dim % 4 == 0;
      const int slabs = (int)((dim + 32 * E - 1) / (32 * E));
      int64_t range = pl.chunk;
      int rc;
      if (on16(dout) && on16(dweight) && (dim * sizeof(TG)) % 16 == 0) {
        // two blocks per SM, each with an equal part of the sorted order
        const int64_t row = dim * sizeof(TG);
        const int64_t bslabs = (row + kBulkSlab - 1) / kBulkSlab;
        if (bslabs > 65535) return (int)MT_ERR_INVALID_ARGUMENT;
        const int64_t want = std::max<int64_t>(1, 2 * get_sm_count() / bslabs);
        range = std::max<int64_t>(pl.chunk, ((n + want - 1) / want + 31) / 32 * 32);
        int rp = 32;
        while (rp * std::min<int64_t>(row, kBulkSlab) > kBulkStage) rp /= 2;
        auto kern = embed_reduce_bulk_kernel<TG, TD>;
        if ((rc = set_smem_limit((const void*)kern, sizeof(BulkSmem))) != MT_OK) return rc;
        kern<<<dim3((unsigned)((n + range - 1) / range), (unsigned)bslabs), kBulkThreads, sizeof(BulkSmem), s>>>(
            sorted, n, range, rp, static_cast<const TG*>(dout), (uint32_t)vocab, (int)dim, scale,
            static_cast<TD*>(dweight), partial, seg, status);
      } else {
        const int64_t units = pl.chunks * slabs;
        if ((units + 7) / 8 > 0x7fffffffLL || slabs > 65535) return (int)MT_ERR_INVALID_ARGUMENT;
        auto red = vec ? embed_reduce_kernel<TG, TD, true> : embed_reduce_kernel<TG, TD, false>;
        red<<<(unsigned)((units + 7) / 8), 256, 0, s>>>(sorted, n, pl.chunk, slabs, static_cast<const TG*>(dout),
                                                        (uint32_t)vocab, (int)dim, scale, static_cast<TD*>(dweight),
                                                        partial, seg);
      }
      if ((rc = check_launch("embedding_bwd_reduce")) != MT_OK) return rc;
      auto join = vec ? embed_join_kernel<TD, E, true> : embed_join_kernel<TD, E, false>;
      join<<<dim3((unsigned)((vocab + 255) / 256), (unsigned)slabs), 256, 0, s>>>(
          seg, vocab, range, partial, (int)dim, scale, static_cast<TD*>(dweight));
      return check_launch("embedding_bwd_join");
    });
  });
}
