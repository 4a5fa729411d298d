// Distillation loss of an output projection against a teacher's top logits.
//
//   p_r = softmax(t_r / T) over the row's listed entries that are not masked
//   q_r = softmax(h_r W^T / T) over the whole vocabulary
//   loss = T^2 * mean over rows with an entry of  sum_j p_rj (log p_rj - log q_r[id_rj])
//   dz_r = (q_r - scatter(p_r)) * T / n_rows,   dh = dz W,   dW = dz^T h
//
// No counterpart in the reference, which trains against labels only.
//
// Forward: distill_prep_kernel turns a row's list into its probabilities, sorted
// by id with equal ids merged.  The tile product keeps a running maximum and sum
// per row over the vocabulary tiles a CTA pair takes (consecutive ones, so a row
// is cut over few pairs) and, walking the sorted list along, picks the listed
// logits out of TMEM: the logits never reach memory.  distill_row_kernel joins
// the pieces and forms the loss.
//
// Backward: dz is needed by two products with different reductions (dh over
// the vocabulary, dW over the rows).  Recomputing the logits once per product
// on chip costs 8 N V K operations; writing dz out once costs 6 N V K and
// 2 bytes per logit, so rows are taken in chunks whose 16-bit dz fits in a
// bounded workspace:
//   1. dz chunk = round(2^(z log2e / T - lse)) (tile product, epilogue)
//   2. listed entries are overwritten with round(q - p) from the forward's
//      fp32 logits: the difference is rounded once, not its parts
//   3. dh chunk = dz W        (W read along its rows, no transposed copy)
//   4. dW      += dz^T h      (fp32, both operands read along their rows; rows
//      without an entry as zeros whatever they hold: 0 * inf is NaN)
// q - p is kept without the factor T * grad / n, which the epilogues apply in
// fp32: it would push 16-bit values of a mean over many rows out of range.
// fp16 values are held times 2^15 for the same reason (|q - p| <= 1).  The rounding of
// dz to 16 bits (half a step of its own magnitude) is the tensor cores' operand
// type and the one rounding between the fp32 logits and the fp32 sums.  One or
// two rows take a path without tiles or that rounding.
//
// Bound by the tensor pipe and, in a steady stream, by the power limit: 32,768
// rows x 768 against 21,504 entries, forward and backward, 3.70-3.89 ms (8 NVK
// operations at 1.11-1.17 PFLOP/s).  Alone: statistics 745-759 us (tensor pipe
// 81-82 % busy), per 6,144-row chunk dz 148 us (82 %), dh 128-130 us (93 %), dW
// 138-144 us (81-85 %: 252 tiles in two splits on 74 CTA pairs, 6.8 of 7 waves,
// each chunk added to two 66 MB sets of fp32 sums).
#include <cmath>

#include "tile_gemm.cuh"

namespace mt {
namespace {

constexpr uint32_t kKernelId = 8;
constexpr int kMaxTop = 256;
constexpr int kNone = 0x7fffffff;  // id of an unused list slot
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994530942f;

// ---------------------------------------------------------------------------
// the teacher's lists
// ---------------------------------------------------------------------------
struct PrepParams {
  const void* ids;
  int ids_i64;
  const void* logits;
  int64_t ignore_index;
  int N, V, top;
  float temp;
  int* tid;      // [N, top] ids in rising order, kNone past the last
  float* tp;     // [N, top] their probabilities (0 past the last)
  float* ent;    // [N] sum p log p; NaN-free for empty rows (0)
  float* mass;   // [N] 1 for a row with an entry, else 0
  uint32_t* status;
};

// One warp per row, kPer list entries per lane.
template <typename TL, int kPer>
__global__ void __launch_bounds__(256) distill_prep_kernel(const PrepParams p) {
  __shared__ int s_id[8][kPer * 32];
  __shared__ int o_id[8][kPer * 32];
  __shared__ float o_p[8][kPer * 32];
  const int lane = lane_id(), w = warp_id();
  const int64_t row = int64_t(blockIdx.x) * 8 + w;
  if (row >= p.N) return;
  const int top = p.top;
  float a[kPer];
  int id[kPer];
  float mx = -INFINITY;
  bool odd = false;  // an id outside the vocabulary
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = i * 32 + lane;
    id[i] = kNone;
    a[i] = -INFINITY;
    if (j < top) {
      const int64_t at = row * top + j;
      const int64_t v = p.ids_i64 ? static_cast<const int64_t*>(p.ids)[at]
                                  : (int64_t) static_cast<const int32_t*>(p.ids)[at];
      if (v >= 0 && v < p.V && v != p.ignore_index) {
        id[i] = (int)v;
        a[i] = __fdiv_rn(to_f32<TL>(static_cast<const TL*>(p.logits)[at]), p.temp);
        mx = fmaxf(mx, a[i]);
      } else if (v != p.ignore_index) {
        odd = true;
      }
      s_id[w][j] = id[i];
    }
  }
  if (odd) atomicCAS(p.status, 0u, (kKernelId << 16) | 0xEEEEu);
  mx = warp_max(mx);
  // a list of -inf only has no mass: the row counts as empty.  (A NaN logit
  // keeps mx finite or -inf and makes the sum NaN.)
  float e[kPer], sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    e[i] = id[i] != kNone ? expf(a[i] - mx) : 0.f;
    sum += e[i];
  }
  sum = warp_sum(sum);
  const bool nan_row = __any_sync(0xffffffffu, [&] {
    bool b = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) b |= id[i] != kNone && isnan(a[i]);
    return b;
  }());
  const bool live = mx > -INFINITY || nan_row;
  const float lse = logf(sum);
  float ent = 0.f;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = i * 32 + lane;
    if (i * 32 >= top) break;
    const float pr = live && id[i] != kNone ? __fdiv_rn(e[i], sum) : 0.f;
    if (pr != 0.f) ent += pr * (a[i] - mx - lse);
    if (j < top) {
      // place in the order of (id, position)
      int rank = 0;
      const int mine = id[i];
      for (int q = 0; q < top; ++q) {
        const int other = s_id[w][q];
        rank += other < mine || (other == mine && q < j);
      }
      o_id[w][rank] = live ? mine : kNone;
      o_p[w][rank] = pr;
    }
  }
  ent = warp_sum(ent);
  __syncwarp();
  // merge equal ids into the first of them and close the gaps
  int kept = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (i * 32 >= top) break;
    const int j = i * 32 + lane;
    const int mine = j < top ? o_id[w][j] : kNone;
    const bool head = mine != kNone && (j == 0 || o_id[w][j - 1] != mine);
    const uint32_t heads = __ballot_sync(0xffffffffu, head);
    if (head) {
      float s = o_p[w][j];
      for (int q = j + 1; q < top && o_id[w][q] == mine; ++q) s += o_p[w][q];
      const int at = kept + __popc(heads & ((1u << lane) - 1u));
      p.tid[row * top + at] = mine;
      p.tp[row * top + at] = s;
    }
    kept += __popc(heads);
  }
  for (int j = kept + lane; j < top; j += 32) {
    p.tid[row * top + j] = kNone;
    p.tp[row * top + j] = 0.f;
  }
  if (lane == 0) {
    p.ent[row] = live ? ent : 0.f;
    p.mass[row] = live ? 1.f : 0.f;
  }
}

// ---------------------------------------------------------------------------
// row statistics of the logits, and the listed logits
// ---------------------------------------------------------------------------
struct StatsEpilogue {
  static constexpr uint32_t kKernelId = mt::kKernelId;
  static constexpr int OUT_SIZE = 4;
  static constexpr bool kStats = true;
  static constexpr bool kAltB = false;
  const int* tid;
  float* zt;
  float* part_m;  // [N, pieces]: pieces = slots * groups
  float* part_s;
  int V, top, pieces, groups, n_nt, per_unit;
  float zscale;

  struct State {
    float m, s;          // running maximum (times zscale) and sum of 2^(z zscale - m)
    int64_t at, end;     // place in the row's list
    int want, later;     // ids at `at` and after it
    int64_t piece;       // where the row's statistics go, -1: no such row
  };
  __device__ __forceinline__ int id_at(int64_t i, int64_t end) const { return i < end ? __ldg(tid + i) : kNone; }

  __device__ __forceinline__ void begin(State& st, int m, bool live, int mt, int unit, int group) const {
    st.m = -INFINITY;
    st.s = 0.f;
    st.at = int64_t(m) * top;
    st.end = live ? st.at + top : st.at;
    st.want = id_at(st.at, st.end);
    st.later = id_at(st.at + 1, st.end);
    const int slot = unit - int(int64_t(mt) * n_nt / per_unit);
    st.piece = live ? int64_t(m) * pieces + slot * groups + group : -1;
  }
  __device__ __forceinline__ int next(const State& st) const { return st.want; }
  __device__ __forceinline__ void skip(State& st) const {
    ++st.at;
    st.want = st.later;
    st.later = id_at(st.at + 1, st.end);
  }
  __device__ __forceinline__ void take(State& st, uint32_t z) const {
    zt[st.at] = __uint_as_float(z);
    skip(st);
  }
  __device__ __forceinline__ void add(State& st, const uint32_t (&z)[32], int n0) const {
    if (n0 >= V) return;
    float x[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = n0 + i < V ? __uint_as_float(z[i]) : -INFINITY;
    float cm = fmaxf(x[0], x[1]);
#pragma unroll
    for (int i = 2; i < 32; i += 2) cm = fmax3(cm, x[i], x[i + 1]);
    const float mn = fmaxf(st.m, cm * zscale);  // zscale > 0
    // a maximum of -inf means nothing but -inf (which adds 0) or NaN (which has to stay) so far
    const float base = mn == -INFINITY ? 0.f : mn;
    const float2 zs = make_float2(zscale, zscale), sh = make_float2(-base, -base);
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float2 e = fma2(make_float2(x[i], x[i + 1]), zs, sh);
      sum = add2(sum, make_float2(fast_exp2(e.x), fast_exp2(e.y)));
    }
    st.s = st.s * fast_exp2(st.m - base) + (sum.x + sum.y);
    st.m = mn;
  }
  __device__ __forceinline__ void end(const State& st) const {
    if (st.piece >= 0) {
      part_m[st.piece] = st.m;
      part_s[st.piece] = st.s;
    }
  }
};

// ---------------------------------------------------------------------------
// per-row loss
// ---------------------------------------------------------------------------
struct RowParams {
  int N, top, pieces, groups, n_nt, per_unit;
  const float* part_m;
  const float* part_s;
  const float* tp;
  const float* zt;
  const float* ent;
  const float* mass;
  float inv_temp;
  float* lse2;   // [N] log2 of the row's sum, +inf for rows without an entry
  float* part;   // [blocks, 2] sums of loss and of rows
};

// One warp per row; the block's partial sums in a fixed order.
__global__ void __launch_bounds__(256) distill_row_kernel(const RowParams p) {
  __shared__ float red[2][8];
  const int lane = lane_id(), w = warp_id();
  const int64_t row = int64_t(blockIdx.x) * 8 + w;
  float loss = 0.f, count = 0.f;
  if (row < p.N) {
    // pieces that exist: the CTA pairs whose tiles cover this row's 256-row tile
    const int64_t t0 = row / 256 * p.n_nt;
    const int used = int((t0 + p.n_nt - 1) / p.per_unit - t0 / p.per_unit + 1) * p.groups;
    const float* pm = p.part_m + row * p.pieces;
    const float* ps = p.part_s + row * p.pieces;
    float M = -INFINITY;
    for (int i = lane; i < used; i += 32) M = fmaxf(M, pm[i]);
    M = warp_max(M);
    const float base = M == -INFINITY ? 0.f : M;
    float S = 0.f;
    for (int i = lane; i < used; i += 32) S += ps[i] * exp2f(pm[i] - base);  // pm -inf: ps is 0 or NaN
    const float l2 = base + log2f(warp_sum(S));
    const bool live = p.mass[row] != 0.f;
    if (live) {
      float cross = 0.f;
      for (int j = lane; j < p.top; j += 32) {
        const int64_t at = row * p.top + j;
        const float pr = p.tp[at];  // 0 past the list's end
        if (pr != 0.f) cross += pr * (p.zt[at] * p.inv_temp - l2 * kLn2);
      }
      loss = p.ent[row] - warp_sum(cross);
      count = 1.f;
    }
    if (lane == 0) p.lse2[row] = live ? l2 : INFINITY;
  }
  if (lane == 0) {
    red[0][w] = loss;
    red[1][w] = count;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += red[threadIdx.x][i];
    p.part[int64_t(blockIdx.x) * 2 + threadIdx.x] = s;
  }
}

// loss = T^2 * sum / rows (0 without rows); scal = {loss, rows, 1 / rows}
__global__ void __launch_bounds__(1024) distill_loss_kernel(const float* __restrict__ part, int n, float temp,
                                                            float* __restrict__ scal, float* __restrict__ loss) {
  __shared__ float sl[32], sv[32];
  float l = 0.f, v = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 1024) {
    const float2 q = __ldg(reinterpret_cast<const float2*>(part) + i);
    l += q.x;
    v += q.y;
  }
  l = warp_sum(l);
  v = warp_sum(v);
  if (lane_id() == 0) {
    sl[warp_id()] = l;
    sv[warp_id()] = v;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    l = warp_sum(sl[threadIdx.x]);
    v = warp_sum(sv[threadIdx.x]);
    if (threadIdx.x == 0) {
      const float inv = v > 0.f ? 1.f / v : 0.f;
      const float r = v > 0.f ? temp * temp * l * inv : 0.f;
      scal[0] = r;
      scal[1] = v;
      scal[2] = inv;
      loss[0] = r;
    }
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// 16-bit q times `up` (a power of two), columns past the vocabulary zero.
template <typename T>
struct SoftmaxEpilogue {
  static constexpr uint32_t kKernelId = mt::kKernelId;
  static constexpr int OUT_SIZE = 2;
  static constexpr bool kStats = false;
  static constexpr bool kAltB = false;
  const float* lse2;
  float zscale;
  float log2_up;
  bool add, direct;

  struct Row {
    float shift;  // log2(up) - lse2, or -inf for a row without an entry
  };
  __device__ __forceinline__ Row row(int m, bool live) const {
    return Row{live ? log2_up - __ldg(lse2 + m) : -INFINITY};
  }
  static constexpr bool kCols = false;
  __device__ __forceinline__ void pack(const uint32_t (&z)[32], const Row& r, const float*, uint32_t* words) const {
    const bool some = r.shift != -INFINITY;  // NaN logits of a row without an entry stay out
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float a = fast_exp2(fmaf(__uint_as_float(z[i]), zscale, r.shift));
      const float b = fast_exp2(fmaf(__uint_as_float(z[i + 1]), zscale, r.shift));
      words[i >> 1] = some ? pack2<T>(a, b) : 0u;
    }
  }
};

// The hidden states that dW's product reads: rows without an entry have dz = 0,
// but 0 times an infinity or a NaN is NaN, so where such rows exist the product
// reads a copy of the chunk in which they are zero.
struct LiveHidden {
  CUtensorMap copy;
  const float* live;  // rows with an entry in the whole batch
  float rows;         // fewer than this many: read the copy
};
struct NoOther {};

// accumulator * temp * grad_out / rows / up
template <typename TO, bool DW>
struct GradEpilogue {
  static constexpr uint32_t kKernelId = mt::kKernelId;
  static constexpr int OUT_SIZE = sizeof(TO);
  static constexpr bool kStats = false;
  static constexpr bool kAltB = DW;
  const float* inv_rows;
  const float* grad_out;
  float factor;  // temp / up
  bool add, direct;
  typename std::conditional<DW, LiveHidden, NoOther>::type hidden;

  __device__ __forceinline__ const CUtensorMap* b_map(const CUtensorMap* all) const {
    return __ldg(hidden.live) < hidden.rows ? &hidden.copy : all;
  }

  struct Row {
    float g;
  };
  __device__ __forceinline__ Row row(int, bool) const { return Row{factor * __ldg(grad_out) * __ldg(inv_rows)}; }
  static constexpr bool kCols = false;
  __device__ __forceinline__ void pack(const uint32_t (&z)[32], const Row& r, const float*, uint32_t* words) const {
    if constexpr (sizeof(TO) == 4) {
#pragma unroll
      for (int i = 0; i < 32; ++i) words[i] = __float_as_uint(__uint_as_float(z[i]) * r.g);
    } else {
#pragma unroll
      for (int i = 0; i < 32; i += 2)
        words[i >> 1] = pack2<TO>(__uint_as_float(z[i]) * r.g, __uint_as_float(z[i + 1]) * r.g);
    }
  }
};

// Listed entries of a chunk of rows: dz = round((q - p) * up); and, in the blocks
// after those, the chunk's hidden states with zero rows where there is no entry
// (none to write when every row of the batch has one).
struct ListedParams {
  const int* tid;
  const float *tp, *zt, *lse2;
  uint32_t n, top;        // entries in all, per row
  unsigned entry_blocks;  // blocks for them
  float zscale, up;
  void* dz;
  int64_t ld;
  const uint4* hidden;
  uint4* copy;
  int rows, words;        // of the chunk, 16-byte words of a row
  const float* live;      // as in LiveHidden
  float all_rows;
};

template <typename T>
__global__ void __launch_bounds__(256) distill_listed_kernel(const ListedParams p) {
  if (blockIdx.x >= p.entry_blocks) {
    if (!(__ldg(p.live) < p.all_rows)) return;
    // a warp per row
    const int step = (gridDim.x - p.entry_blocks) * 8;
    for (int r = (blockIdx.x - p.entry_blocks) * 8 + warp_id(); r < p.rows; r += step) {
      const bool none = __ldg(p.lse2 + r) == INFINITY;
      const int64_t at = int64_t(r) * p.words;
#pragma unroll 4
      for (int i = lane_id(); i < p.words; i += 32)
        p.copy[at + i] = none ? make_uint4(0u, 0u, 0u, 0u) : __ldg(p.hidden + at + i);
    }
    return;
  }
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.n) return;
  const int id = p.tid[i];
  if (id == kNone) return;
  const uint32_t row = i / p.top;
  const float q = fast_exp2(fmaf(p.zt[i], p.zscale, -p.lse2[row]));
  static_cast<T*>(p.dz)[int64_t(row) * p.ld + id] = from_f32<T>((q - p.tp[i]) * p.up);
}

// out = sum over splits of part (fixed order), cast to out's dtype; 4 columns a thread.
template <typename TO>
__global__ void __launch_bounds__(256) sum_splits_kernel(const float* __restrict__ part, int splits,
                                                         int64_t split_elems, int64_t n4, TO* __restrict__ out) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n4; i += int64_t(gridDim.x) * 256) {
    float4 a = __ldg(reinterpret_cast<const float4*>(part) + i);
    for (int s = 1; s < splits; ++s) {
      const float4 b = __ldg(reinterpret_cast<const float4*>(part + s * split_elems) + i);
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    if constexpr (sizeof(TO) == 4)
      reinterpret_cast<float4*>(out)[i] = a;
    else
      reinterpret_cast<uint2*>(out)[i] = make_uint2(pack2<TO>(a.x, a.y), pack2<TO>(a.z, a.w));
  }
}

// ---------------------------------------------------------------------------
// backward of a few rows: everything in fp32, no tiles
// ---------------------------------------------------------------------------
// With up to kFewRows rows a 256-row tile would be nearly empty and W is what
// there is to read, so two passes over it do: one warp per vocabulary entry v
// forms the rows' z_v by dot products, dz_v = q - p and dW_v = sum_r dz_rv h_r at
// once; then dh = dz W in strips of v, joined in a fixed order.  dz stays in fp32
// (a single row's error would otherwise be one rounding of its largest entry).
// Measured against the tiles, backward alone, cold cache: 21,504 x 768, 1 row 31
// against 49 us and 2 rows 39 against 51; 2,048 columns, 68 against 92 and 84
// against 94; 2,000 x 256, 12 against 29.  Past the L2 the second pass over W pays
// HBM again: 100,000 x 1,024, 178 against 158.  The dot products of more rows cost
// instructions (an earlier form: 4 rows of 2,048 columns 109 against 88).
constexpr int kFewRows = 2;
constexpr int kFewK = 2048;  // and the rows' hidden states in 8 KB of shared memory
constexpr int64_t kFewWeight = 64 << 20;  // V * K: 128 MB, about the L2
constexpr int kFewStrips = 512;

struct FewParams {
  const void* hidden;
  const void* weight;
  int N, V, K, top;
  float zscale, factor;  // log2(e) / temperature, temperature
  const int* tid;
  const float* tp;
  const float* lse2;
  const float* inv_rows;
  const float* grad_out;
  float* dz;  // [N, V] fp32
  void* dw;   // may be NULL
};

// p of id v in a row's list (rising ids, kNone past the last).
__device__ __forceinline__ float listed_prob(const int* tid, const float* tp, int top, int v) {
  int lo = 0, hi = top;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(tid + mid) < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo < top && __ldg(tid + lo) == v ? __ldg(tp + lo) : 0.f;
}

template <typename T, typename TO, int MT>
__global__ void __launch_bounds__(256) distill_few_dw_kernel(const FewParams p) {
  extern __shared__ __align__(16) uint8_t raw[];
  T* h = reinterpret_cast<T*>(raw);  // [N, K]
  const int lane = lane_id();
  for (int i = threadIdx.x * 8; i < p.N * p.K; i += 256 * 8)
    *reinterpret_cast<uint4*>(h + i) = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.hidden) + i));
  __syncthreads();
  const float lse2 = lane < p.N ? __ldg(p.lse2 + lane) : INFINITY;
  const float g = p.factor * __ldg(p.grad_out) * __ldg(p.inv_rows);
  const int warps = gridDim.x * 8;
  for (int v = blockIdx.x * 8 + warp_id(); v < p.V; v += warps) {
    const T* wv = static_cast<const T*>(p.weight) + int64_t(v) * p.K;
    float z[MT];
#pragma unroll
    for (int r = 0; r < MT; ++r) z[r] = 0.f;
#pragma unroll 4
    for (int k = lane * 8; k < p.K; k += 256) {
      float x[8];
      load_vec<T, 8>(wv + k, x);
#pragma unroll
      for (int r = 0; r < MT; ++r)
        if (r < p.N) {
          float y[8];
          load_vec<T, 8>(h + r * p.K + k, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) z[r] = fmaf(x[e], y[e], z[r]);
        }
    }
    float mine = 0.f;  // lane r: row r's logit
#pragma unroll
    for (int r = 0; r < MT; ++r) {
      const float t = warp_sum(z[r]);
      if (lane == r) mine = t;
    }
    float d = 0.f;
    if (lane < p.N && lse2 != INFINITY) {  // rows without an entry stay out
      d = exp2f(fmaf(mine, p.zscale, -lse2)) - listed_prob(p.tid + lane * p.top, p.tp + lane * p.top, p.top, v);
    }
    if (lane < p.N) p.dz[int64_t(lane) * p.V + v] = d;
    if (p.dw != nullptr) {
      TO* out = static_cast<TO*>(p.dw) + int64_t(v) * p.K;
      for (int k0 = 0; k0 < p.K; k0 += 256) {
        const int k = k0 + lane * 8;
        float acc[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
        for (int r = 0; r < p.N; ++r) {
          const float dr = __shfl_sync(0xffffffffu, d, r);
          if (dr != 0.f && k < p.K) {
            float y[8];
            load_vec<T, 8>(h + r * p.K + k, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(dr, y[e], acc[e]);
          }
        }
        if (k < p.K) {
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] *= g;
          if constexpr (sizeof(TO) == 2) {
            store_vec<TO, 8>(out + k, acc);
          } else {
            store_vec<TO, 4>(out + k, {acc[0], acc[1], acc[2], acc[3]});
            store_vec<TO, 4>(out + k + 4, {acc[4], acc[5], acc[6], acc[7]});
          }
        }
      }
    }
  }
}

// A strip of vocabulary entries for 256 columns (two per thread): partial sums
// part[strip, r, k] of dz W.
template <typename T, int MT>
__global__ void __launch_bounds__(128) distill_few_dh_kernel(const float* __restrict__ dz, const T* __restrict__ w,
                                                             int N, int V, int K, int strip,
                                                             float* __restrict__ part) {
  __shared__ float s[MT][64];
  const int k = blockIdx.y * 256 + threadIdx.x * 2;
  const int lo = blockIdx.x * strip, hi = min(lo + strip, V);
  float2 acc[MT];
#pragma unroll
  for (int r = 0; r < MT; ++r) acc[r] = make_float2(0.f, 0.f);
  for (int v0 = lo; v0 < hi; v0 += 64) {
    const int nv = min(64, hi - v0);
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 64; i += 128) {
      const int r = i >> 6, j = i & 63;
      s[r][j] = r < N && j < nv ? dz[int64_t(r) * V + v0 + j] : 0.f;
    }
    __syncthreads();
    if (k >= K) continue;
    const T* wp = w + int64_t(v0) * K + k;
    for (int j0 = 0; j0 < nv; j0 += 8) {
      uint32_t x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[j] = j0 + j < nv ? __ldg(reinterpret_cast<const uint32_t*>(wp + int64_t(j0 + j) * K)) : 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float a, b;
        unpack2<T>(x[j], a, b);
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          acc[r].x = fmaf(s[r][j0 + j], a, acc[r].x);
          acc[r].y = fmaf(s[r][j0 + j], b, acc[r].y);
        }
      }
    }
  }
  if (k >= K) return;
#pragma unroll
  for (int r = 0; r < MT; ++r)
    if (r < N) *reinterpret_cast<float2*>(part + (int64_t(blockIdx.x) * N + r) * K + k) = acc[r];
}

// dh = factor * sum over strips (8 lanes of strips per element, then in order).
template <typename TO>
__global__ void __launch_bounds__(256) distill_few_join_kernel(const float* __restrict__ part, int strips, int n,
                                                               float factor, const float* __restrict__ inv_rows,
                                                               const float* __restrict__ grad_out,
                                                               TO* __restrict__ out) {
  __shared__ float s[8][32];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + x;
  float a = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int q = y; q < strips; q += 8) a += part[int64_t(q) * n + i];
  }
  s[y][x] = a;
  __syncthreads();
  if (y == 0 && i < n) {
    float t = s[0][x];
#pragma unroll
    for (int q = 1; q < 8; ++q) t += s[q][x];
    out[i] = from_f32<TO>(t * (factor * __ldg(grad_out) * __ldg(inv_rows)));
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

constexpr int kStatsWarps = 16;
constexpr int kGroups = kStatsWarps / 4;  // warpgroups that share a row's statistics
template <int KIND>
struct Cfgs {
  using S = TileCfg<KIND, false, false, 256, true, kStatsWarps>;  // row statistics of H W^T
  using Z = TileCfg<KIND, false, false, 256, true, 8>;   // dz from H W^T
  using H = TileCfg<KIND, false, true, 256, true, 8>;    // dh = dz W
  using W = TileCfg<KIND, true, true, 256, true, 8>;     // dW = dz^T H
};

struct FwdPlan {
  int n_nt, per_unit, pieces;
  int64_t blocks, off_m, off_s, off_ent, off_mass, off_part, bytes;
};
FwdPlan plan_fwd(int64_t N, int64_t V) {
  FwdPlan pl;
  const int64_t units = std::max<int64_t>(1, get_sm_count() / 2);
  pl.n_nt = (int)((V + 255) / 256);
  const int64_t tiles = (N + 255) / 256 * pl.n_nt;
  pl.per_unit = (int)((tiles + units - 1) / units);
  // consecutive tiles of one row tile meet at most this many pairs
  pl.pieces = ((pl.n_nt - 1) / pl.per_unit + 2) * kGroups;
  pl.blocks = (N + 7) / 8;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up256(bytes);
    return o;
  };
  pl.off_m = take(N * pl.pieces * 4);
  pl.off_s = take(N * pl.pieces * 4);
  pl.off_ent = take(N * 4);
  pl.off_mass = take(N * 4);
  pl.off_part = take(pl.blocks * 8);
  pl.bytes = at;
  return pl;
}

// No split without a stage: every partial sum that is read was written.
int even_splits(int64_t k_stages, int64_t splits) {
  const int64_t per = (k_stages + splits - 1) / splits;
  return (int)((k_stages + per - 1) / per);
}

// Splits of the inner dimension (k_stages stages of 64): the split that ends
// soonest counted in stages over whole waves of CTA pairs, where a tile costs
// about 4 stages of pipeline fill and drain and every split's partial sums are
// written and read again.
int choose_k_splits(int64_t tiles, int64_t k_stages) {
  const int64_t units = std::max<int64_t>(1, get_sm_count() / 2);
  int best = 1;
  double best_cost = 1e30;
  const int64_t most = std::min<int64_t>(64, std::max<int64_t>(1, k_stages / 4));
  for (int64_t s = 1; s <= most; ++s) {
    const int64_t per = (k_stages + s - 1) / s;
    const int64_t waves = (tiles * s + units - 1) / units;
    const double cost = double(waves) * double(per + 4) + (s > 1 ? 4.0 + 0.15 * double(s) : 0.0);
    if (cost < best_cost * 0.98) {
      best_cost = cost;
      best = (int)s;
    }
  }
  return even_splits(k_stages, best);
}

// One chunk's dz takes at most this (256 rows, the fewest of a chunk, take more
// from a vocabulary of 524,288 on).
constexpr int64_t kDzBytes = int64_t(256) << 20;

struct BwdPlan {
  int64_t ld;          // dz row stride (elements)
  int64_t rows;        // rows per chunk
  int chunks, h_splits, h_last, w_splits;
  int64_t h_pad, w_pad;  // rows of one split's partials
  int64_t off_dz, off_copy, off_h, off_w, bytes;
};
BwdPlan plan_bwd(int64_t N, int64_t V, int64_t K) {
  BwdPlan pl;
  pl.ld = (V + 7) / 8 * 8;
  const int64_t units = std::max<int64_t>(1, get_sm_count() / 2);
  const int64_t nt = (K + 255) / 256;
  // a chunk's dh tiles fill the GPU once, as far as the workspace bound allows
  int64_t mt = std::max<int64_t>(1, units / nt);
  mt = std::max<int64_t>(1, std::min<int64_t>(mt, kDzBytes / (pl.ld * 2 * 256)));
  pl.rows = std::min<int64_t>(N, mt * 256);
  pl.chunks = (int)((N + pl.rows - 1) / pl.rows);
  const int64_t h_tiles = (pl.rows + 255) / 256 * nt, w_tiles = (V + 255) / 256 * nt;
  pl.h_splits = choose_k_splits(h_tiles, (V + 63) / 64);
  // a shorter last chunk has fewer tiles and takes more splits
  const int64_t last = N - (pl.chunks - 1) * pl.rows;
  pl.h_last = choose_k_splits((last + 255) / 256 * nt, (V + 63) / 64);
  pl.w_splits = choose_k_splits(w_tiles, (pl.rows + 63) / 64);
  pl.h_pad = (pl.rows + 255) / 256 * 256;
  pl.w_pad = (V + 255) / 256 * 256;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up256(bytes);
    return o;
  };
  pl.off_dz = take(pl.rows * pl.ld * 2);
  pl.off_copy = take(pl.rows * K * 2);
  const int64_t last_pad = (last + 255) / 256 * 256;
  pl.off_h = take(std::max(pl.h_splits > 1 ? pl.h_splits * pl.h_pad : 0,
                           pl.h_last > 1 ? pl.h_last * last_pad : 0) * K * 4);
  // fp32 sums of dW: several splits, or several chunks (of a 16-bit gradient; the
  // size does not know the type).  One split of one chunk goes straight to its place.
  pl.off_w = take(pl.w_splits > 1 || pl.chunks > 1 ? pl.w_splits * pl.w_pad * K * 4 : 0);
  pl.bytes = at;
  return pl;
}

int sum_splits(const float* part, int splits, int64_t split_elems, int64_t n, void* out, int dtype, cudaStream_t s) {
  const int64_t n4 = n / 4;  // K is a multiple of 8
  const int blocks = (int)std::min<int64_t>((n4 + 255) / 256, int64_t(get_sm_count()) * 64);
  if (dtype == MT_F32)
    sum_splits_kernel<float><<<blocks, 256, 0, s>>>(part, splits, split_elems, n4, static_cast<float*>(out));
  else if (dtype == MT_BF16)
    sum_splits_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(part, splits, split_elems, n4,
                                                             static_cast<__nv_bfloat16*>(out));
  else
    sum_splits_kernel<__half><<<blocks, 256, 0, s>>>(part, splits, split_elems, n4, static_cast<__half*>(out));
  return check_launch("distill_bwd_sum");
}

// A gradient product's launch with `dtype` outputs of rows x K; `live` for dW.
template <class C, typename TO, bool DW>
int grad_product(const CUtensorMap& a, const CUtensorMap& b, int64_t rows, int64_t K, int64_t k_elems, int splits,
                 int64_t split_rows, void* out, int dtype, bool add, const float* inv_rows, const float* grad_out,
                 float factor, const LiveHidden* live, uint32_t* status, const char* name, cudaStream_t s) {
  TileParams<GradEpilogue<TO, DW>> prm;
  prm.tm_a = a;
  prm.tm_b = b;
  const int64_t map_rows = splits > 1 ? splits * split_rows : rows;
  const int64_t stages = (k_elems + C::BK - 1) / C::BK;
  // a last chunk with fewer stages leaves the later splits' sums as they are (add)
  splits = even_splits(stages, splits);
  int st = tile_output_map(&prm.tm_out, out, dtype, map_rows, K, K);
  if (st != MT_OK) return st;
  prm.M = (int)rows;
  prm.N = (int)K;
  prm.n_k = (int)stages;
  prm.k_per_split = (prm.n_k + splits - 1) / splits;
  prm.per_unit = 0;
  prm.split_rows = split_rows;
  prm.out = out;
  prm.ld_out = K;
  prm.status = status;
  prm.ep.inv_rows = inv_rows;
  prm.ep.grad_out = grad_out;
  prm.ep.factor = factor;
  prm.ep.add = add;
  prm.ep.direct = false;
  if constexpr (DW) prm.ep.hidden = *live;
  return launch_tile_gemm<C>(prm, splits, name, s);
}

template <class C, bool DW>
int grad_product_as(int dtype, const CUtensorMap& a, const CUtensorMap& b, int64_t rows, int64_t K, int64_t k_elems,
                    int splits, int64_t split_rows, void* out, bool add, const float* inv_rows, const float* grad_out,
                    float factor, const LiveHidden* live, uint32_t* status, const char* name, cudaStream_t s) {
  if (dtype == MT_F32)
    return grad_product<C, float, DW>(a, b, rows, K, k_elems, splits, split_rows, out, dtype, add, inv_rows, grad_out,
                                      factor, live, status, name, s);
  if (dtype == MT_BF16)
    return grad_product<C, __nv_bfloat16, DW>(a, b, rows, K, k_elems, splits, split_rows, out, dtype, add, inv_rows,
                                              grad_out, factor, live, status, name, s);
  return grad_product<C, __half, DW>(a, b, rows, K, k_elems, splits, split_rows, out, dtype, add, inv_rows, grad_out,
                                     factor, live, status, name, s);
}

template <typename TL>
int launch_prep(const PrepParams& p, unsigned blocks, cudaStream_t s) {
  if (p.top <= 32)
    distill_prep_kernel<TL, 1><<<blocks, 256, 0, s>>>(p);
  else if (p.top <= 64)
    distill_prep_kernel<TL, 2><<<blocks, 256, 0, s>>>(p);
  else
    distill_prep_kernel<TL, kMaxTop / 32><<<blocks, 256, 0, s>>>(p);
  return check_launch("distill_prep");
}

template <int KIND>
int run_stats(const void* hidden, const void* weight, int64_t N, int64_t V, int64_t K, const StatsEpilogue& ep,
              uint32_t* status, cudaStream_t s) {
  using C = typename Cfgs<KIND>::S;
  TileParams<StatsEpilogue> prm;
  int st = tile_operand_map<C>(&prm.tm_a, hidden, false, N, K, K, 128);
  if (st != MT_OK) return st;
  if ((st = tile_operand_map<C>(&prm.tm_b, weight, false, V, K, K, C::B_ROWS)) != MT_OK) return st;
  prm.tm_out = prm.tm_a;  // not used
  prm.M = (int)N;
  prm.N = (int)V;
  prm.n_k = (int)((K + C::BK - 1) / C::BK);
  prm.k_per_split = prm.n_k;
  prm.per_unit = ep.per_unit;
  prm.split_rows = 0;
  prm.out = nullptr;
  prm.ld_out = 0;
  prm.status = status;
  prm.ep = ep;
  return launch_tile_gemm<C>(prm, 1, "distill_stats", s);
}

struct BwdArgs {
  const void *hidden, *weight;
  int64_t N, V, K;
  int top;
  float temp;
  const int* tid;
  const float *tp, *zt, *lse2, *live_rows, *inv_rows, *grad_out;
  void* dh;
  int dh_dtype;
  void* dw;
  int dw_dtype;
  char* ws;
  uint32_t* status;
  cudaStream_t s;
};

template <typename T, int KIND>
int run_bwd(const BwdArgs& a, const BwdPlan& pl) {
  using Z = typename Cfgs<KIND>::Z;
  using H = typename Cfgs<KIND>::H;
  using W = typename Cfgs<KIND>::W;
  const float zscale = kLog2e / a.temp;
  const float log2_up = KIND == kKindF16 ? 15.f : 0.f, up = KIND == kKindF16 ? 32768.f : 1.f;
  const float factor = a.temp / up;
  T* dz = reinterpret_cast<T*>(a.ws + pl.off_dz);
  T* h_copy = reinterpret_cast<T*>(a.ws + pl.off_copy);
  float* h_part = reinterpret_cast<float*>(a.ws + pl.off_h);
  float* w_part = reinterpret_cast<float*>(a.ws + pl.off_w);
  // dW goes straight to its place when one fp32 tensor or one chunk takes it
  const bool w_direct = pl.w_splits == 1 && (a.dw_dtype == MT_F32 || pl.chunks == 1);
  // live rows are counted in fp32, exact up to 2^24: past that the copy is always made
  const float all_rows = a.N <= (1 << 24) ? float(a.N) : INFINITY;
  int st;
  for (int c = 0; c < pl.chunks; ++c) {
    const int64_t r0 = c * pl.rows, rows = std::min(pl.rows, a.N - r0);
    const T* h = static_cast<const T*>(a.hidden) + r0 * a.K;
    // 1. q
    TileParams<SoftmaxEpilogue<T>> zp;
    if ((st = tile_operand_map<Z>(&zp.tm_a, h, false, rows, a.K, a.K, 128)) != MT_OK) return st;
    if ((st = tile_operand_map<Z>(&zp.tm_b, a.weight, false, a.V, a.K, a.K, Z::B_ROWS)) != MT_OK) return st;
    if ((st = tile_output_map(&zp.tm_out, dz, KIND == kKindBf16 ? MT_BF16 : MT_F16, rows, a.V, pl.ld)) != MT_OK)
      return st;
    zp.M = (int)rows;
    zp.N = (int)a.V;
    zp.n_k = (int)((a.K + Z::BK - 1) / Z::BK);
    zp.k_per_split = zp.n_k;
    zp.per_unit = 0;
    zp.split_rows = 0;
    zp.out = dz;
    zp.ld_out = pl.ld;
    zp.status = a.status;
    zp.ep = SoftmaxEpilogue<T>{a.lse2 + r0, zscale, log2_up, false, false};
    if ((st = launch_tile_gemm<Z>(zp, 1, "distill_bwd_dz", a.s)) != MT_OK) return st;
    // 2. q - p where the teacher lists an entry
    const int64_t n = rows * a.top;
    const ListedParams lp{a.tid + r0 * a.top, a.tp + r0 * a.top, a.zt + r0 * a.top, a.lse2 + r0, (uint32_t)n,
                          (uint32_t)a.top, (unsigned)((n + 255) / 256), zscale, up, dz, pl.ld,
                          reinterpret_cast<const uint4*>(h), reinterpret_cast<uint4*>(h_copy), (int)rows,
                          (int)(a.K / 8), a.live_rows, all_rows};
    const unsigned copy_blocks =
        a.dw != nullptr ? (unsigned)std::min<int64_t>((rows + 7) / 8, int64_t(get_sm_count()) * 8) : 0u;
    distill_listed_kernel<T><<<lp.entry_blocks + copy_blocks, 256, 0, a.s>>>(lp);
    if ((st = check_launch("distill_bwd_listed")) != MT_OK) return st;
    // 3. dh = dz W
    if (a.dh != nullptr) {
      char* out = static_cast<char*>(a.dh) + r0 * a.K * (a.dh_dtype == MT_F32 ? 4 : 2);
      CUtensorMap ma, mb;
      if ((st = tile_operand_map<H>(&ma, dz, false, rows, a.V, pl.ld, 128)) != MT_OK) return st;
      if ((st = tile_operand_map<H>(&mb, a.weight, true, a.K, a.V, a.K, 0)) != MT_OK) return st;
      const int splits = c + 1 == pl.chunks ? pl.h_last : pl.h_splits;
      if (splits > 1) {
        const int64_t pad = (rows + 255) / 256 * 256;
        if ((st = grad_product_as<H, false>(MT_F32, ma, mb, rows, a.K, a.V, splits, pad, h_part, false, a.inv_rows,
                                            a.grad_out, factor, nullptr, a.status, "distill_bwd_dh", a.s)) != MT_OK)
          return st;
        if ((st = sum_splits(h_part, splits, pad * a.K, rows * a.K, out, a.dh_dtype, a.s)) != MT_OK) return st;
      } else if ((st = grad_product_as<H, false>(a.dh_dtype, ma, mb, rows, a.K, a.V, 1, 0, out, false, a.inv_rows,
                                                 a.grad_out, factor, nullptr, a.status, "distill_bwd_dh", a.s)) != MT_OK) {
        return st;
      }
    }
    // 4. dW += dz^T h
    if (a.dw != nullptr) {
      CUtensorMap ma, mb;
      if ((st = tile_operand_map<W>(&ma, dz, true, a.V, rows, pl.ld, 0)) != MT_OK) return st;
      if ((st = tile_operand_map<W>(&mb, h, true, a.K, rows, a.K, 0)) != MT_OK) return st;
      LiveHidden live{{}, a.live_rows, all_rows};
      if ((st = tile_operand_map<W>(&live.copy, h_copy, true, a.K, rows, a.K, 0)) != MT_OK) return st;
      if ((st = grad_product_as<W, true>(w_direct ? a.dw_dtype : MT_F32, ma, mb, a.V, a.K, rows, pl.w_splits, pl.w_pad,
                                         w_direct ? a.dw : w_part, c > 0, a.inv_rows, a.grad_out, factor, &live,
                                         a.status, "distill_bwd_dw", a.s)) != MT_OK)
        return st;
    }
  }
  if (a.dw != nullptr && !w_direct)
    return sum_splits(w_part, pl.w_splits, pl.w_pad * a.K, a.V * a.K, a.dw, a.dw_dtype, a.s);
  return MT_OK;
}

bool few_rows(int64_t N, int64_t V, int64_t K) { return N <= kFewRows && K <= kFewK && V * K <= kFewWeight; }
int64_t few_part_off(int64_t N, int64_t V) { return up256(N * V * 4); }
int64_t few_bytes(int64_t N, int64_t V, int64_t K) { return few_part_off(N, V) + up256(kFewStrips * N * K * 4); }

template <typename T, typename TO, int MT>
int launch_few_dw(const FewParams& p, cudaStream_t s) {
  auto kern = distill_few_dw_kernel<T, TO, MT>;
  const int smem = p.N * p.K * (int)sizeof(T);
  const int grid = (int)std::min<int64_t>((int64_t(p.V) + 7) / 8, int64_t(get_sm_count()) * 8);
  kern<<<grid, 256, smem, s>>>(p);
  return check_launch("distill_bwd_few_dw");
}

template <typename T, int MT>
int run_few_rows(const BwdArgs& a) {
  float* dz = reinterpret_cast<float*>(a.ws);
  float* part = reinterpret_cast<float*>(a.ws + few_part_off(a.N, a.V));
  const FewParams p{a.hidden, a.weight, (int)a.N, (int)a.V, (int)a.K, a.top, kLog2e / a.temp, a.temp, a.tid, a.tp,
                    a.lse2, a.inv_rows, a.grad_out, dz, a.dw};
  int st = a.dw_dtype == MT_F32    ? launch_few_dw<T, float, MT>(p, a.s)
           : a.dw_dtype == MT_BF16 ? launch_few_dw<T, __nv_bfloat16, MT>(p, a.s)
                                   : launch_few_dw<T, __half, MT>(p, a.s);
  if (st != MT_OK || a.dh == nullptr) return st;
  const int strip = std::max(16, (int)((a.V + kFewStrips - 1) / kFewStrips)), strips = (int)((a.V + strip - 1) / strip);
  distill_few_dh_kernel<T, MT><<<dim3((unsigned)strips, (unsigned)((a.K + 255) / 256)), 128, 0, a.s>>>(
      dz, static_cast<const T*>(a.weight), (int)a.N, (int)a.V, (int)a.K, strip, part);
  if ((st = check_launch("distill_bwd_few_dh")) != MT_OK) return st;
  const int n = (int)(a.N * a.K);
  const unsigned grid = (unsigned)((n + 31) / 32);
  if (a.dh_dtype == MT_F32)
    distill_few_join_kernel<float><<<grid, 256, 0, a.s>>>(part, strips, n, a.temp, a.inv_rows, a.grad_out,
                                                          static_cast<float*>(a.dh));
  else if (a.dh_dtype == MT_BF16)
    distill_few_join_kernel<__nv_bfloat16><<<grid, 256, 0, a.s>>>(part, strips, n, a.temp, a.inv_rows, a.grad_out,
                                                                  static_cast<__nv_bfloat16*>(a.dh));
  else
    distill_few_join_kernel<__half><<<grid, 256, 0, a.s>>>(part, strips, n, a.temp, a.inv_rows, a.grad_out,
                                                           static_cast<__half*>(a.dh));
  return check_launch("distill_bwd_few_join");
}

template <typename T>
int run_few(const BwdArgs& a) {
  if (a.N == 1) return run_few_rows<T, 1>(a);
  return run_few_rows<T, kFewRows>(a);
}

int check_args(const void* hidden, const void* weight, int dtype, int64_t N, int64_t V, int64_t K, int64_t top,
               float temp) {
  if (dtype != MT_BF16 && dtype != MT_F16) return MT_ERR_UNSUPPORTED_DTYPE;
  if (N < 0 || V <= 0 || K <= 0 || top <= 0) return MT_ERR_INVALID_ARGUMENT;
  if (top > kMaxTop) {
    set_last_error_text("distillation: at most 256 listed entries per row");
    return MT_ERR_INVALID_ARGUMENT;
  }
  if (!(temp > 0.f) || !std::isfinite(temp)) return MT_ERR_INVALID_ARGUMENT;
  if (N > 0x7fffffffLL - 256 || V > 0x7fffffffLL - 256 || K > 0x7fffffffLL / 4 - 256) return MT_ERR_INVALID_ARGUMENT;
  if (N > 0 && (hidden == nullptr || weight == nullptr)) return MT_ERR_INVALID_ARGUMENT;
  if (K % 8 != 0) return MT_ERR_UNSUPPORTED_LAYOUT;
  if ((reinterpret_cast<uintptr_t>(hidden) & 15u) || (reinterpret_cast<uintptr_t>(weight) & 15u))
    return MT_ERR_UNSUPPORTED_LAYOUT;
  return MT_OK;
}

bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace
}  // namespace mt

using namespace mt;

extern "C" int64_t mt_distill_workspace_bytes(int64_t N, int64_t V) {
  if (N <= 0 || V <= 0) return 256;
  return plan_fwd(N, V).bytes;
}

extern "C" int mt_distill_fwd(const void* hidden, const void* weight, int dtype, const void* teacher_ids, int ids_i64,
                              int64_t ignore_index, const void* teacher_logits, int logits_dtype, int64_t N,
                              int64_t V, int64_t K, int64_t top, float temperature, float* loss, int* list_ids,
                              float* list_probs, float* list_logits, float* row_stats, void* workspace,
                              int64_t workspace_bytes, uint32_t* status, void* stream) {
  int st = check_args(hidden, weight, dtype, N, V, K, top, temperature);
  if (st != MT_OK) return st;
  if (logits_dtype != MT_F32 && logits_dtype != MT_F16 && logits_dtype != MT_BF16) return MT_ERR_UNSUPPORTED_DTYPE;
  if (loss == nullptr || row_stats == nullptr) return MT_ERR_INVALID_ARGUMENT;
  auto s = static_cast<cudaStream_t>(stream);
  if (N == 0) {
    cudaError_t e = cudaMemsetAsync(loss, 0, 4, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(row_stats, 0, 12, s);
    return e == cudaSuccess ? MT_OK : MT_ERR_LAUNCH;
  }
  if (teacher_ids == nullptr || teacher_logits == nullptr || list_ids == nullptr || list_probs == nullptr ||
      list_logits == nullptr || status == nullptr)
    return MT_ERR_INVALID_ARGUMENT;
  const FwdPlan pl = plan_fwd(N, V);
  if (workspace == nullptr || !aligned_to(workspace, 256) || workspace_bytes < pl.bytes) return MT_ERR_WORKSPACE;
  if ((st = bind_device_of(hidden)) != MT_OK) return st;
  if ((st = check_arch()) != MT_OK) return st;
  char* ws = static_cast<char*>(workspace);
  float* pm = reinterpret_cast<float*>(ws + pl.off_m);
  float* ps = reinterpret_cast<float*>(ws + pl.off_s);
  float* ent = reinterpret_cast<float*>(ws + pl.off_ent);
  float* mass = reinterpret_cast<float*>(ws + pl.off_mass);
  float* part = reinterpret_cast<float*>(ws + pl.off_part);
  const PrepParams pp{teacher_ids, ids_i64, teacher_logits, ignore_index, (int)N, (int)V, (int)top, temperature,
                      list_ids, list_probs, ent, mass, status};
  const unsigned blocks = (unsigned)pl.blocks;
  st = logits_dtype == MT_F32    ? launch_prep<float>(pp, blocks, s)
       : logits_dtype == MT_BF16 ? launch_prep<__nv_bfloat16>(pp, blocks, s)
                                 : launch_prep<__half>(pp, blocks, s);
  if (st != MT_OK) return st;
  const StatsEpilogue ep{list_ids, list_logits, pm, ps, (int)V, (int)top, pl.pieces, kGroups, pl.n_nt, pl.per_unit,
                         kLog2e / temperature};
  st = dtype == MT_BF16 ? run_stats<kKindBf16>(hidden, weight, N, V, K, ep, status, s)
                        : run_stats<kKindF16>(hidden, weight, N, V, K, ep, status, s);
  if (st != MT_OK) return st;
  const RowParams rp{(int)N, (int)top, pl.pieces, kGroups, pl.n_nt, pl.per_unit, pm, ps, list_probs, list_logits,
                     ent, mass, 1.f / temperature, row_stats, part};
  distill_row_kernel<<<blocks, 256, 0, s>>>(rp);
  if ((st = check_launch("distill_row")) != MT_OK) return st;
  distill_loss_kernel<<<1, 1024, 0, s>>>(part, (int)pl.blocks, temperature, row_stats + N, loss);
  return check_launch("distill_loss");
}

extern "C" int64_t mt_distill_bwd_workspace_bytes(int64_t N, int64_t V, int64_t K) {
  if (N <= 0 || V <= 0 || K <= 0) return 256;
  return few_rows(N, V, K) ? few_bytes(N, V, K) : plan_bwd(N, V, K).bytes;
}

extern "C" int mt_distill_bwd(const void* hidden, const void* weight, int dtype, int64_t N, int64_t V, int64_t K,
                              int64_t top, float temperature, const int* list_ids, const float* list_probs,
                              const float* list_logits, const float* row_stats, const float* grad_out, void* dhidden,
                              int dh_dtype, void* dweight, int dw_dtype, void* workspace, int64_t workspace_bytes,
                              uint32_t* status, void* stream) {
  int st = check_args(hidden, weight, dtype, N, V, K, top, temperature);
  if (st != MT_OK) return st;
  for (int d : {dh_dtype, dw_dtype})
    if (d != MT_F32 && d != MT_F16 && d != MT_BF16) return MT_ERR_UNSUPPORTED_DTYPE;
  if (!aligned_to(dhidden, 16) || !aligned_to(dweight, 16)) return MT_ERR_UNSUPPORTED_LAYOUT;
  auto s = static_cast<cudaStream_t>(stream);
  if (N == 0) {
    if (dweight != nullptr &&
        cudaMemsetAsync(dweight, 0, size_t(V) * K * (dw_dtype == MT_F32 ? 4 : 2), s) != cudaSuccess)
      return MT_ERR_LAUNCH;
    return MT_OK;
  }
  if (list_ids == nullptr || list_probs == nullptr || list_logits == nullptr || row_stats == nullptr ||
      grad_out == nullptr || status == nullptr)
    return MT_ERR_INVALID_ARGUMENT;
  const bool few = few_rows(N, V, K);
  const BwdPlan pl = plan_bwd(N, V, K);
  if (workspace == nullptr || !aligned_to(workspace, 256) || workspace_bytes < mt_distill_bwd_workspace_bytes(N, V, K))
    return MT_ERR_WORKSPACE;
  if (std::max(pl.h_splits, pl.h_last) * pl.h_pad > 0x7fffffffLL || pl.w_splits * pl.w_pad > 0x7fffffffLL) return MT_ERR_INVALID_ARGUMENT;
  if ((st = bind_device_of(hidden)) != MT_OK) return st;
  if ((st = check_arch()) != MT_OK) return st;
  const BwdArgs a{hidden, weight, N, V, K, (int)top, temperature, list_ids, list_probs, list_logits, row_stats,
                  row_stats + N + 1, row_stats + N + 2, grad_out, dhidden, dh_dtype, dweight, dw_dtype, static_cast<char*>(workspace),
                  status, s};
  if (few) return dtype == MT_BF16 ? run_few<__nv_bfloat16>(a) : run_few<__half>(a);
  return dtype == MT_BF16 ? run_bwd<__nv_bfloat16, kKindBf16>(a, pl) : run_bwd<__half, kKindF16>(a, pl);
}
