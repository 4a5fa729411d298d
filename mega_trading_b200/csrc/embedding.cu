// Token embedding lookup with a scale, and its gradient by sorted tokens.
//
//   forward   y[n, :] = round(scale * W[id[n], :])
//   gradient  dW[v, :] = round(scale * sum_{n: id[n] = v} dy[n, :])   (dense, every row written)
//
// Reference: nn.Embedding of TradingModel (duoan/mega-trading
// src/mega_trading/model.py:20-147), whose gradient PyTorch computes.
//
// Forward: bound by HBM (N * dim elements written; the table stays in L2 at
// this model's sizes).  One warp per token, 16-byte stores.
//
// Gradient: bound by reading dy once.  The token ids are sorted with their
// positions (stable least-significant-digit radix sort, 8 bits a pass, written
// here: one block for up to 4,096 tokens, otherwise a histogram launch and one
// scatter launch per pass), so that the rows of dy which meet in one row of dW
// are neighbours in the sorted order.  embed_reduce_kernel cuts the sorted
// order into chunks of equal length, so a token that makes up a large share of
// the stream costs no more than any other: a warp walks one chunk for one slab
// of columns and sums runs of equal ids in fp32 registers, eight rows in
// flight.  A run that lies inside its chunk goes straight to dW; a run cut by a
// chunk border leaves fp32 partial sums, at most two per chunk, which
// embed_join_kernel adds up (it also zeroes the rows no token chose).  Every
// sum has a fixed order (no atomics on values): results are the same each time.
//
// Ids outside [0, V) read nothing: their output row is zero, they add to no
// gradient and the status word is set.  Places holding padding_idx look up
// their row like any other and add to no gradient.
#include <algorithm>

#include "common.cuh"

namespace mt {
namespace {

constexpr uint32_t kKernelId = 7;
constexpr int kSubTile = 2048;   // tokens one sort block ranks at a time (8 warps x 8 x 32)
constexpr int kOneBlock = 4096;  // tokens the single-block sort takes (32 warps x 4 x 32)
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
template <typename T, int E>
__device__ __forceinline__ void store_n(T* p, const float (&v)[E]) {
  constexpr int kPer = 16 / sizeof(T);
  if constexpr (E * sizeof(T) == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
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
  template <typename T>
  static __device__ __forceinline__ void store(T* row, int c0, int dim, const float (&v)[E]) {
    const int lane = lane_id();
    if constexpr (VEC) {
      if (c0 + lane * E < dim) store_n<T, E>(row + c0 + lane * E, v);
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
template <typename TW, typename TO, bool VEC>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const void* __restrict__ ids, int i64, int64_t n_tokens,
                                                        const TW* __restrict__ w, int64_t vocab, int dim, float scale,
                                                        TO* __restrict__ y, uint32_t* status) {
  constexpr int E = lane_elems<TW, TO>();
  using C = Cols<E, VEC>;
  const int64_t n = int64_t(blockIdx.x) * 8 + warp_id();
  if (n >= n_tokens) return;
  const int64_t id = load_id(ids, i64, n);
  TO* row = y + n * dim;
  if (id < 0 || id >= vocab) {
    if (lane_id() == 0) atomicCAS(status, 0u, (kKernelId << 16) | 0xEEEEu);
    const float zero[E] = {};
    for (int c0 = 0; c0 < dim; c0 += C::kSlab) C::store(row, c0, dim, zero);
    return;
  }
  const TW* src = w + id * dim;
  for (int c0 = 0; c0 < dim; c0 += 4 * C::kSlab) {
    float v[4][E];
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (c0 + s * C::kSlab < dim) C::load(src, c0 + s * C::kSlab, dim, v[s]);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (c0 + s * C::kSlab < dim) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[s][e] *= scale;
        C::store(row, c0 + s * C::kSlab, dim, v[s]);
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

__device__ __forceinline__ uint32_t key_of(const SortIn& in, int64_t n) {
  const int64_t id = load_id(in.ids, in.i64, n);
  if (id < 0 || id >= in.vocab) {
    atomicCAS(in.status, 0u, (kKernelId << 16) | 0xEEEEu);
    return (uint32_t)in.vocab;
  }
  return id == in.pad ? (uint32_t)in.vocab : (uint32_t)id;
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
  uint32_t key[4], pos[4], digit[4], rank[4];
  // the id ranges start out empty
  for (int64_t v = threadIdx.x; v <= in.vocab; v += 1024) seg[v] = make_uint2(0u, 0u);
  const int first = warp_id() * 128 + lane_id();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    pos[i] = first + i * 32;
    key[i] = (int)pos[i] < n_tokens ? key_of(in, pos[i]) : 0u;
  }
  for (int shift = 0; shift < bits; shift += 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) digit[i] = first + i * 32 < n_tokens ? (key[i] >> shift) & 255u : 256u;
    rank_tile<32, 4>(digit, rank, cnt, total);
    scan256(total, base, warp_tot);
    const bool last = shift + 8 >= bits;
    // the order of this pass: the place of each item (pos_s holds the permutation)
#pragma unroll
    for (int i = 0; i < 4; ++i)
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
      for (int i = 0; i < 4; ++i)
        if (first + i * 32 < n_tokens) {
          pos[i] = pos_s[first + i * 32];
          key[i] = key_of(in, pos[i]);
        }
      __syncthreads();
    }
  }
}

// Histogram of the first digit per tile; clears the later passes' histograms
// and the id ranges.
__global__ void __launch_bounds__(256) embed_hist_kernel(SortIn in, int64_t n_tokens, int64_t tile,
                                                         uint32_t* __restrict__ hist, int64_t hist_words, uint2* seg) {
  __shared__ uint32_t h[256];
  h[threadIdx.x] = 0;
  const int64_t gid = int64_t(blockIdx.x) * 256 + threadIdx.x, gsz = int64_t(gridDim.x) * 256;
  const int64_t own = int64_t(gridDim.x) * 256;  // this pass's histograms
  for (int64_t i = own + gid; i < hist_words; i += gsz) hist[i] = 0;
  for (int64_t v = gid; v <= in.vocab; v += gsz) seg[v] = make_uint2(0u, 0u);
  __syncthreads();
  const int64_t lo = blockIdx.x * tile, hi = min(lo + tile, n_tokens);
  for (int64_t i = lo + threadIdx.x; i < hi + 255; i += 256) {
    if (i - threadIdx.x >= hi) break;
    const uint32_t d = i < hi ? key_of(in, i) & 255u : 256u;
    const uint32_t peers = __match_any_sync(0xffffffffu, d);
    if (d < 256 && lane_id() == __ffs(peers) - 1) atomicAdd(&h[d], (uint32_t)__popc(peers));
  }
  __syncthreads();
  hist[int64_t(blockIdx.x) * 256 + threadIdx.x] = h[threadIdx.x];
}

// One stable pass: items move to (items of smaller digits) + (items of the same
// digit in earlier tiles) + (rank inside the tile).  FIRST reads the ids, later
// passes the pairs.  next != NULL: counts the next digit per destination tile
// (integer atomics: the counts do not depend on their order).
template <bool FIRST>
__global__ void __launch_bounds__(256) embed_scatter_kernel(SortIn in, const uint2* __restrict__ src, int64_t n_tokens,
                                                            int64_t tile, int shift, const uint32_t* __restrict__ hist,
                                                            uint32_t* __restrict__ next, uint2* __restrict__ dst) {
  __shared__ uint32_t cnt[8][256];
  __shared__ uint32_t total[256], base[256], warp_tot[8];
  {
    // this tile's first place for every digit
    uint32_t before = 0, all = 0;
    const uint32_t* col = hist + threadIdx.x;
    const int tiles = gridDim.x, me = blockIdx.x;
#pragma unroll 16
    for (int b = 0; b < tiles; ++b) {
      const uint32_t c = __ldg(col + int64_t(b) * 256);
      all += c;
      before += b < me ? c : 0u;
    }
    total[threadIdx.x] = all;
    __syncthreads();
    scan256(total, base, warp_tot);
    base[threadIdx.x] += before;
    __syncthreads();
  }
  const int64_t lo = blockIdx.x * tile, hi = min(lo + tile, n_tokens);
  for (int64_t s0 = lo; s0 < hi; s0 += kSubTile) {
    uint32_t key[8], pos[8], digit[8], rank[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t n = s0 + warp_id() * 256 + i * 32 + lane_id();
      digit[i] = 256u;
      if (n < hi) {
        if constexpr (FIRST) {
          key[i] = key_of(in, n);
          pos[i] = (uint32_t)n;
        } else {
          const uint2 q = src[n];
          key[i] = q.x;
          pos[i] = q.y;
        }
        digit[i] = (key[i] >> shift) & 255u;
      }
    }
    rank_tile<8, 8>(digit, rank, cnt, total);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (digit[i] < 256) {
        const uint32_t at = base[digit[i]] + rank[i];
        dst[at] = make_uint2(key[i], pos[i]);
        if (next != nullptr) atomicAdd(&next[int64_t(at / (uint32_t)tile) * 256 + ((key[i] >> (shift + 8)) & 255u)], 1u);
      }
    __syncthreads();
    base[threadIdx.x] += total[threadIdx.x];
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

// Rows no token chose become zero; runs cut by chunk borders become the sum of
// their partial sums.  A block takes 32 ids and one slab of columns; a run of
// more than kWide partials is shared by the block's warps.
template <typename TD, int E, bool VEC>
__global__ void __launch_bounds__(256) embed_join_kernel(const uint2* __restrict__ seg, int64_t vocab, int chunk,
                                                         const float* __restrict__ partial, int dim, float scale,
                                                         TD* __restrict__ dw) {
  using C = Cols<E, VEC>;
  constexpr int kWide = 64;
  __shared__ float red[8][32 * E];
  const int c0 = blockIdx.y * C::kSlab;
  const int lane = lane_id(), w = warp_id();
  const int64_t v0 = int64_t(blockIdx.x) * 32;
  const uint2 mine = v0 + lane < vocab ? __ldg(seg + v0 + lane) : make_uint2(0u, 0u);
  auto sum = [&](int64_t lo, int64_t hi, int64_t head, float(&acc)[E]) {
    // partials lo .. hi of a run whose first one is `head` (slot 1), eight rows in flight
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int64_t q = lo; q < hi; q += 8) {
      float v[8][E];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (q + j < hi) C::load(partial + ((q + j) * 2 + (q + j == head ? 1 : 0)) * dim, c0, dim, v[j]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (q + j < hi)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += v[j][e];
    }
  };
  for (int i = 0; i < 32; ++i) {
    const uint32_t start = __shfl_sync(0xffffffffu, mine.x, i), end = __shfl_sync(0xffffffffu, mine.y, i);
    if (v0 + i >= vocab) break;
    TD* row = dw + (v0 + i) * dim;
    float acc[E];
    if (start == end) {
      if ((i & 7) != w) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      C::store(row, c0, dim, acc);
      continue;
    }
    const int64_t a = start / (uint32_t)chunk, b = (end - 1) / (uint32_t)chunk;
    if (a == b) continue;  // written by the reduction
    if (b - a < kWide) {
      if ((i & 7) != w) continue;
      sum(a, b + 1, a, acc);
    } else {
      const int64_t per = (b + 1 - a + 7) / 8;
      sum(a + w * per, min(a + (w + 1) * per, b + 1), a, acc);
#pragma unroll
      for (int e = 0; e < E; ++e) red[w][e * 32 + lane] = acc[e];
      __syncthreads();
      if (w == 0) {
#pragma unroll
        for (int q = 1; q < 8; ++q)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += red[q][e * 32 + lane];
      }
      __syncthreads();
      if (w != 0) continue;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= scale;
    C::store(row, c0, dim, acc);
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
  pl.tile = kSubTile;
  while ((n + pl.tile - 1) / pl.tile > kMaxTiles) pl.tile += kSubTile;
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
      auto kern = vec ? embed_fwd_kernel<TW, TO, true> : embed_fwd_kernel<TW, TO, false>;
      kern<<<(unsigned)((n + 7) / 8), 256, 0, s>>>(ids, ids_i64, n, static_cast<const TW*>(weight), vocab, (int)dim,
                                                   scale, static_cast<TO*>(out), status);
      return check_launch("embedding_fwd");
    });
  });
}

extern "C" int64_t mt_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t dim) {
  if (n <= 0 || check_embed(n, vocab, dim) != MT_OK) return 256;
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
    const unsigned grid = (unsigned)pl.tiles;
    embed_hist_kernel<<<grid, 256, 0, s>>>(in, n, pl.tile, hist, pl.hist_words, seg);
    if ((st = check_launch("embedding_bwd_hist")) != MT_OK) return st;
    for (int p = 0; p < pl.passes; ++p) {
      const uint32_t* h = hist + int64_t(p) * pl.tiles * 256;
      uint32_t* next = p + 1 < pl.passes ? hist + int64_t(p + 1) * pl.tiles * 256 : nullptr;
      uint2* dst = pairs[p & 1];
      if (p == 0)
        embed_scatter_kernel<true><<<grid, 256, 0, s>>>(in, nullptr, n, pl.tile, 0, h, next, dst);
      else
        embed_scatter_kernel<false><<<grid, 256, 0, s>>>(in, sorted, n, pl.tile, 8 * p, h, next, dst);
      if ((st = check_launch("embedding_bwd_scatter")) != MT_OK) return st;
      sorted = dst;
    }
  }
  return with_type(dout_dtype, [&](auto gv) {
    return with_type(dw_dtype, [&](auto dv) {
      using TG = decltype(gv);
      using TD = decltype(dv);
      constexpr int E = lane_elems<TG, TD>();
      const bool vec = on16(dout) && on16(dweight) && dim % E == 0 && dim % 4 == 0;
      const int slabs = (int)((dim + 32 * E - 1) / (32 * E));
      const int64_t units = pl.chunks * slabs;
      if ((units + 7) / 8 > 0x7fffffffLL || slabs > 65535) return (int)MT_ERR_INVALID_ARGUMENT;
      auto red = vec ? embed_reduce_kernel<TG, TD, true> : embed_reduce_kernel<TG, TD, false>;
      red<<<(unsigned)((units + 7) / 8), 256, 0, s>>>(sorted, n, pl.chunk, slabs, static_cast<const TG*>(dout),
                                                      (uint32_t)vocab, (int)dim, scale, static_cast<TD*>(dweight),
                                                      partial, seg);
      int rc = check_launch("embedding_bwd_reduce");
      if (rc != MT_OK) return rc;
      auto join = vec ? embed_join_kernel<TD, E, true> : embed_join_kernel<TD, E, false>;
      join<<<dim3((unsigned)((vocab + 31) / 32), (unsigned)slabs), 256, 0, s>>>(
          seg, vocab, pl.chunk, partial, (int)dim, scale, static_cast<TD*>(dweight));
      return check_launch("embedding_bwd_join");
    });
  });
}
