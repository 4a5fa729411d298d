// 8-bit outputs with one scale per row: RMSNorm (with the residual add fused
// in front) and plain row quantisation.  No counterpart in the reference,
// which runs every projection in bf16; these feed mt_int8_gemm.
//
//   s = round(h + r)                      (ADD; else s = x)
//   v_i = s_i * w_i                       (NORM; else v = s)
//   a = max_i |v_i|,  q_i = rint(v_i * (127 / a)),  scale = a / 127 * rstd
//   rstd = rsqrt(mean(s^2) + eps)         (NORM; else 1)
//
// The normalised row is rstd * v, so rstd cancels out of q: q depends on exact
// products and an exact maximum only, never on the order in which the sum of
// squares was taken, and is the same integer for any grouping of threads.  A
// row whose a is below 2^-119 (127 / a would overflow) gives q = 0, scale = 0;
// a row with an infinity or a NaN gives a NaN scale, so whatever is computed
// from it is NaN too (its q means nothing).  Squares past fp32's range are summed
// again, scaled: a row of the type's lowest value has its scale.
//
// Bound by HBM: each element is read once (plus the residual read and written)
// and leaves as one byte (131,072 x 1,024, bf16 branch and fp32 residual: 235
// us, 0.96 of the measured copy rate; 30,011 x 2,816 bf16 without a norm: 41-43
// us, 0.91-0.95).  The row stays in registers between the reduction and the
// quantisation.  One warp owns a row of up to 1024 elements; wider
// rows take 128, 256 or 1024 threads (their statistics meet in shared memory).
// Accesses are 16-byte vectors when the width and every address allow it,
// single elements (consecutive lanes on consecutive elements) otherwise.
#include <cmath>

#include "common.cuh"

namespace mt {
namespace {

constexpr float kTinyAmax = 1.504632769052528e-36f;  // 2^-119
constexpr int kMaxDim = 32768;

template <typename T>
__device__ __forceinline__ void load8f(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    load_vec<T, 8>(p, v);
  } else {
    float a[4], b[4];
    load_vec<T, 4>(p, a);
    load_vec<T, 4>(p + 4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[i + 4] = b[i];
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8f(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    store_vec<T, 8>(p, v);
  } else {
    store_vec<T, 4>(p, {v[0], v[1], v[2], v[3]});
    store_vec<T, 4>(p + 4, {v[4], v[5], v[6], v[7]});
  }
}

// max(a, |b|) that is NaN if either is.
__device__ __forceinline__ float amax_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(fabsf(b)));
  return d;
}

// rint(v) for |v| <= 127 in the low byte: adding 1.5 * 2^23 leaves the integer,
// rounded to even, in the low mantissa bits (FMA pipe instead of conversions).
__device__ __forceinline__ uint32_t int8_bits(float v) { return __float_as_uint(__fadd_rn(v, 12582912.f)); }
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Sum of squares of a row times `factor` squared, by one warp.
template <typename T>
__device__ __forceinline__ float scaled_squares(const T* s, int dim, float factor) {
  float a = 0.f;
#pragma unroll 1
  for (int i = lane_id(); i < dim; i += 32) {
    const float v = to_f32<T>(s[i]) * factor;
    a = fmaf(v, v, a);
  }
  return warp_sum(a);
}

struct QParams {
  const void* x;
  const void* res;   // ADD
  const void* w;     // NORM
  int w_f32;         // weight in fp32 (else in x's dtype)
  void* new_res;     // ADD
  int8_t* q;
  float* scale;
  int64_t rows;
  int dim;
  float eps;
};

enum { kPlain = 0, kNorm = 1, kAddNorm = 2 };

// Two 16-bit maxima of magnitudes at a time, NaN if either is.
template <typename T> struct Pair16;
template <> struct Pair16<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair16<__half> { using type = __half2; };
template <typename T>
__device__ __forceinline__ uint32_t amax2_nan(uint32_t a, uint32_t b) {
  using P = typename Pair16<T>::type;
  P r = __hmax2_nan(*reinterpret_cast<P*>(&a), __habs2(*reinterpret_cast<P*>(&b)));
  return *reinterpret_cast<uint32_t*>(&r);
}

// Plain rows of 16-bit values in 16-byte words: the maximum is exact in 16
// bits, so the row is kept packed (half the registers of the general kernel,
// more rows in flight) and widened once, when it is quantised.
template <typename T, int TPR, int NC>
__global__ void __launch_bounds__(256, 8) quant8_packed_kernel(const __grid_constant__ QParams p) {
  static_assert(TPR <= 256, "one block's threads");
  constexpr int kRows = 256 / TPR;
  __shared__ float red[8];
  const int t = threadIdx.x % TPR;
  const int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / TPR;
  const bool live = row < p.rows;
  const T* x = static_cast<const T*>(p.x) + row * p.dim;
  uint4 r[NC];
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + t) * 8;
    r[c] = live && col < p.dim ? __ldg(reinterpret_cast<const uint4*>(x + col)) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int c = 0; c < NC; ++c)
    m = amax2_nan<T>(amax2_nan<T>(amax2_nan<T>(amax2_nan<T>(m, r[c].x), r[c].y), r[c].z), r[c].w);
  float lo, hi;
  unpack2<T>(m, lo, hi);
  float amax = amax_nan(lo, hi);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = amax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    if (lane_id() == 0) red[warp_id()] = amax;
    __syncthreads();
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) amax = amax_nan(amax, red[threadIdx.x / TPR * kWarps + i]);
  }
  if (!live) return;
  const bool finite = amax < INFINITY;
  const float inv = finite && amax >= kTinyAmax ? __fdiv_rn(127.f, amax) : 0.f;
  if (t == 0) p.scale[row] = !finite ? NAN : (amax >= kTinyAmax ? amax / 127.f : 0.f);
  int8_t* q = p.q + row * p.dim;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * TPR + t) * 8;
    const uint32_t w[4] = {r[c].x, r[c].y, r[c].z, r[c].w};
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v0, v1;
      unpack2<T>(w[e], v0, v1);
      b[2 * e] = int8_bits(__fmul_rn(v0, inv));
      b[2 * e + 1] = int8_bits(__fmul_rn(v1, inv));
    }
    if (col < p.dim)
      *reinterpret_cast<uint2*>(q + col) = make_uint2(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]));
  }
}

// TPR threads own a row; each holds NC chunks of 8 elements.
template <typename TX, typename TR, int MODE, int TPR, int NC, bool VEC>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) quant8_kernel(const __grid_constant__ QParams p) {
  constexpr int kBlock = TPR < 256 ? 256 : TPR;
  constexpr int kRows = kBlock / TPR;
  __shared__ float red[2][kBlock / 32];
  const int t = threadIdx.x % TPR;
  const int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / TPR;
  const bool live = row < p.rows;
  const int dim = p.dim;
  const TX* x = static_cast<const TX*>(p.x) + row * dim;
  const TR* r = static_cast<const TR*>(p.res) + row * dim;
  TR* nr = static_cast<TR*>(p.new_res) + row * dim;
  float v[NC][8];
  float ss = 0.f;
  // element e of chunk c: VEC 8 consecutive, else strided by the row's threads
  auto col_of = [&](int c, int e) { return VEC ? (c * TPR + t) * 8 + e : (c * 8 + e) * TPR + t; };
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if constexpr (VEC) {
      const int col = col_of(c, 0);
      if (live && col < dim) {
        load8f<TX>(x + col, v[c]);
        if constexpr (MODE == kAddNorm) {
          float rv[8];
          load8f<TR>(r + col, rv);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[c][e] = round_to<TR>(v[c][e] + rv[e]);
          store8f<TR>(nr + col, v[c]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = col_of(c, e);
        v[c][e] = 0.f;
        if (live && col < dim) {
          v[c][e] = to_f32<TX>(x[col]);
          if constexpr (MODE == kAddNorm) v[c][e] = round_to<TR>(v[c][e] + to_f32<TR>(r[col]));
        }
      }
      if constexpr (MODE == kAddNorm) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (live && col_of(c, e) < dim) nr[col_of(c, e)] = from_f32<TR>(v[c][e]);
      }
    }
  }
  float amax = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if constexpr (MODE != kPlain) {
      float wv[8];
      if constexpr (VEC) {
        const int col = col_of(c, 0);
        if (col < dim) {
          if (p.w_f32)
            load8f<float>(static_cast<const float*>(p.w) + col, wv);
          else
            load8f<TX>(static_cast<const TX*>(p.w) + col, wv);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) wv[e] = 0.f;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int col = col_of(c, e);
          wv[e] = 0.f;
          if (col < dim)
            wv[e] = p.w_f32 ? static_cast<const float*>(p.w)[col] : to_f32<TX>(static_cast<const TX*>(p.w)[col]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss = fmaf(v[c][e], v[c][e], ss);
        v[c][e] = __fmul_rn(v[c][e], wv[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = amax_nan(amax, v[c][e]);
  }
  if constexpr (MODE != kPlain) ss = warp_sum(ss);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = amax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int base = (threadIdx.x / TPR) * kWarps;
    if (lane_id() == 0) {
      red[0][warp_id()] = ss;
      red[1][warp_id()] = amax;
    }
    __syncthreads();
    ss = 0.f;
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      ss += red[0][base + i];
      amax = amax_nan(amax, red[1][base + i]);
    }
  }
  if (!live) return;
  // an infinity or a NaN anywhere in the row: the scale is NaN
  const bool finite = amax < INFINITY;
  const float inv = finite && amax >= kTinyAmax ? __fdiv_rn(127.f, amax) : 0.f;
  int8_t* q = p.q + row * dim;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = int8_bits(__fmul_rn(v[c][e], inv));
    if constexpr (VEC) {
      const int col = col_of(c, 0);
      if (col < dim)
        *reinterpret_cast<uint2*>(q + col) = make_uint2(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col_of(c, e) < dim) q[col_of(c, e)] = (int8_t)(b[e] & 0xFFu);
    }
  }
  if (t >= 32) return;
  float rs = 1.f;
  if constexpr (MODE != kPlain) {
    rs = rsqrtf(ss / float(dim) + p.eps);
    // Squares outside fp32's range (values of about 2^59 and more, or below 2^-50
    // with next to no eps): the row's first warp sums them again from memory, scaled.
    const bool over = ss == INFINITY, under = ss < 0x1p-100f && p.eps < 0x1p-80f;
    if (finite && amax >= kTinyAmax && (over || under)) {
      const float f = over ? 0x1p-80f : 0x1p80f;
      __syncwarp();  // new_res is read across the lanes that wrote it (wider rows met at the barrier above)
      const float sq = MODE == kAddNorm ? scaled_squares<TR>(nr, dim, f) : scaled_squares<TX>(x, dim, f);
      rs = rsqrtf(sq / float(dim) + p.eps * f * f) * f;
    }
  }
  if (t == 0) p.scale[row] = !finite ? NAN : (amax >= kTinyAmax || isnan(rs) ? amax * rs / 127.f : 0.f);
}

bool al(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <typename TX, typename TR, int MODE, int TPR, int NC>
int launch_q(const QParams& p, bool vec, cudaStream_t s) {
  constexpr int kBlock = TPR < 256 ? 256 : TPR;
  const int64_t grid = (p.rows + kBlock / TPR - 1) / (kBlock / TPR);
  if (grid > 0x7fffffffLL) return MT_ERR_INVALID_ARGUMENT;
  if (vec) {
    if constexpr (MODE == kPlain && sizeof(TX) == 2 && TPR <= 256)
      quant8_packed_kernel<TX, TPR, NC><<<(unsigned)grid, kBlock, 0, s>>>(p);
    else
      quant8_kernel<TX, TR, MODE, TPR, NC, true><<<(unsigned)grid, kBlock, 0, s>>>(p);
  } else
    quant8_kernel<TX, TR, MODE, TPR, NC, false><<<(unsigned)grid, kBlock, 0, s>>>(p);
  return check_launch(MODE == kPlain ? "quantize_rows_int8" : "rms_norm_int8");
}

template <typename TX, typename TR, int MODE>
int dispatch(const QParams& p, cudaStream_t s) {
  const bool vec = p.dim % 8 == 0 && al(p.x, 16) && al(p.q, 8) && (MODE == kPlain || al(p.w, 16)) &&
                   (MODE != kAddNorm || (al(p.res, 16) && al(p.new_res, 16)));
  const int chunks = (p.dim + 7) / 8;
  if (chunks <= 32) return launch_q<TX, TR, MODE, 32, 1>(p, vec, s);
  // Few rows: four warps per row shorten the one wave there is (8 x 1,024, norm:
  // 2.2 us, one warp 3.9); many rows want no exchange between warps (65,536 x
  // 1,024 without a norm: 34.7 us, four warps 45.4).  Between them, four warps / one:
  // 592 x 512 without a norm 1.84 / 1.74 us, 592 x 1,024 with the add and the norm 3.6 /
  // 5.7, 2,368 x 1,024 6.8 / 7.8, 4,736 x 1,024 11.7 / 11.2.
  if (chunks <= 128 && p.rows <= 4 * int64_t(get_sm_count())) return launch_q<TX, TR, MODE, 128, 1>(p, vec, s);
  if (chunks <= 64) return launch_q<TX, TR, MODE, 32, 2>(p, vec, s);
  if (chunks <= 96) return launch_q<TX, TR, MODE, 32, 3>(p, vec, s);
  if (chunks <= 128) return launch_q<TX, TR, MODE, 32, 4>(p, vec, s);
  // 128 threads up to 384 chunks (32,768 x 2,048: 33.6 us, 256 threads 46.5), then
  // 256 (16,384 x 4,096: 32.8 us, 128 threads 34.9)
  if (chunks <= 256) return launch_q<TX, TR, MODE, 128, 2>(p, vec, s);
  if (chunks <= 384) return launch_q<TX, TR, MODE, 128, 3>(p, vec, s);
  if (chunks <= 512) return launch_q<TX, TR, MODE, 256, 2>(p, vec, s);
  if (chunks <= 1024) return launch_q<TX, TR, MODE, 256, 4>(p, vec, s);
  return launch_q<TX, TR, MODE, 1024, 4>(p, vec, s);
}

int check_shape(int64_t rows, int64_t dim) {
  if (rows < 0 || dim <= 0) return MT_ERR_INVALID_ARGUMENT;
  if (dim > kMaxDim) {
    set_last_error_text("8-bit rows: dim must be at most 32768");
    return MT_ERR_INVALID_ARGUMENT;
  }
  return MT_OK;
}

}  // namespace
}  // namespace mt

using namespace mt;

extern "C" int mt_rms_norm_int8(const void* hidden, int act_dtype, const void* residual, int res_dtype, const void* w,
                                int w_dtype, void* new_residual, int8_t* q, float* scale, int64_t rows, int64_t dim,
                                float eps, void* stream) {
  int st = check_shape(rows, dim);
  if (st != MT_OK) return st;
  const bool add = residual != nullptr;
  if (w_dtype != MT_F32 && w_dtype != act_dtype) return MT_ERR_UNSUPPORTED_DTYPE;
  if (add && res_dtype != act_dtype && res_dtype != MT_F32) return MT_ERR_UNSUPPORTED_DTYPE;
  if (act_dtype != MT_F32 && act_dtype != MT_F16 && act_dtype != MT_BF16) return MT_ERR_UNSUPPORTED_DTYPE;
  if (rows == 0) return MT_OK;
  if (hidden == nullptr || w == nullptr || q == nullptr || scale == nullptr || (add && new_residual == nullptr))
    return MT_ERR_INVALID_ARGUMENT;
  if ((st = bind_device_of(hidden)) != MT_OK) return st;
  QParams p{hidden, residual, w, w_dtype == MT_F32, new_residual, q, scale, rows, (int)dim, eps};
  auto s = static_cast<cudaStream_t>(stream);
  const bool wide = add && res_dtype == MT_F32;
  switch (act_dtype) {
    case MT_F32: return add ? dispatch<float, float, kAddNorm>(p, s) : dispatch<float, float, kNorm>(p, s);
    case MT_F16:
      if (!add) return dispatch<__half, __half, kNorm>(p, s);
      return wide ? dispatch<__half, float, kAddNorm>(p, s) : dispatch<__half, __half, kAddNorm>(p, s);
    default:
      if (!add) return dispatch<__nv_bfloat16, __nv_bfloat16, kNorm>(p, s);
      return wide ? dispatch<__nv_bfloat16, float, kAddNorm>(p, s)
                  : dispatch<__nv_bfloat16, __nv_bfloat16, kAddNorm>(p, s);
  }
}

extern "C" int mt_quantize_rows_int8(const void* x, int dtype, int8_t* q, float* scale, int64_t rows, int64_t dim,
                                     void* stream) {
  int st = check_shape(rows, dim);
  if (st != MT_OK) return st;
  if (dtype != MT_F32 && dtype != MT_F16 && dtype != MT_BF16) return MT_ERR_UNSUPPORTED_DTYPE;
  if (rows == 0) return MT_OK;
  if (x == nullptr || q == nullptr || scale == nullptr) return MT_ERR_INVALID_ARGUMENT;
  if ((st = bind_device_of(x)) != MT_OK) return st;
  QParams p{x, nullptr, nullptr, 0, nullptr, q, scale, rows, (int)dim, 0.f};
  auto s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case MT_F32: return dispatch<float, float, kPlain>(p, s);
    case MT_F16: return dispatch<__half, __half, kPlain>(p, s);
    default: return dispatch<__nv_bfloat16, __nv_bfloat16, kPlain>(p, s);
  }
}
