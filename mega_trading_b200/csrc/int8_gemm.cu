// 8-bit matrix product with a scale per token and per channel:
//   y[m, n] = round( (sum_k x[m, k] w[n, k]) * xs[m] * ws[n] )
// x [M, K] and w [N, K] int8 row-major, the sum exact in int32 (K < 131,072
// keeps 128 * 128 * K below 2^31), the scales applied in fp32, one rounding to
// the output type.  No counterpart in the reference (bf16 projections).
//
// Many tokens: the tcgen05 product of tile_gemm.cuh with kind::i8 (twice the
// rate of 16-bit operands), scales in the epilogue: 65,537 x 5,632 x 1,024 to
// bf16 in 0.37 ms (2.0 POP/s; at K = 8,192 2.95 POP/s).  Few tokens (M <= 8): the
// product is bound by reading w once and by latency, and a 128-row MMA tile
// would be almost empty, so a dot-product kernel reads w straight into
// registers (16 bytes per lane, 8 lanes per channel) and multiplies with dp4a.
#include "tile_gemm.cuh"

namespace mt {
namespace {

constexpr uint32_t kKernelId = 9;
constexpr int kMaxK = 131056;
// us, dot products / 128 x 128 tiles.  From a cold L2, 21,504 channels: K = 768 with
// 4 tokens 7.8 / 10.0, 8 tokens 10.2 / 10.1; K = 1,024 9.1 / 11.8, 12.3 / 11.8; K =
// 2,816 18.0 / 25.2, 25.0 / 24.9; 1,280 channels, K = 2,816, 8 tokens 9.1 / 10.8.
// With w in the L2: 21,504 x 768 with 4 tokens 5.1 / 8.2, 8
// tokens 8.0 / 8.9, 16 tokens 13.8 / 8.8; 1,280 x 768 2.3 / 4.9, 3.2 / 4.8, 4.5 / 4.8
constexpr int kFewTokens = 8;

template <typename TO>
struct Int8Epilogue {
  static constexpr uint32_t kKernelId = mt::kKernelId;
  static constexpr int OUT_SIZE = sizeof(TO);
  static constexpr bool kStats = false;
  static constexpr bool kAltB = false;
  const float* xs;
  const float* ws;
  int n;
  bool add, direct;

  struct Row {
    float xs;
  };
  __device__ __forceinline__ Row row(int m, bool live) const { return Row{live ? __ldg(xs + m) : 0.f}; }

  static constexpr bool kCols = true;
  __device__ __forceinline__ float col(int i) const { return i < n ? __ldg(ws + i) : 0.f; }

  __device__ __forceinline__ void pack(const uint32_t (&z)[32], const Row& r, const float* cols,
                                       uint32_t* words) const {
    const float2 xs2 = make_float2(r.xs, r.xs);
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 s = *reinterpret_cast<const float4*>(cols + j);
      const float2 a = mul2(mul2(make_float2(__int2float_rn((int)z[j]), __int2float_rn((int)z[j + 1])), xs2),
                            make_float2(s.x, s.y));
      const float2 b = mul2(mul2(make_float2(__int2float_rn((int)z[j + 2]), __int2float_rn((int)z[j + 3])), xs2),
                            make_float2(s.z, s.w));
      if constexpr (sizeof(TO) == 4) {
        words[j] = __float_as_uint(a.x);
        words[j + 1] = __float_as_uint(a.y);
        words[j + 2] = __float_as_uint(b.x);
        words[j + 3] = __float_as_uint(b.y);
      } else {
        words[j / 2] = pack2<TO>(a.x, a.y);
        words[j / 2 + 1] = pack2<TO>(b.x, b.y);
      }
    }
  }
};

// 8 lanes per channel, 4 channels per warp, 32 channels per block; MT tokens
// (rows past M are zero).  Blocks of 1,024 of K: a lane's 8 x 16 bytes of w are on
// their way to registers before the tokens' part of x is staged, so all of a
// resident block's w is in flight at once (21,504 x 768 has 672 blocks: all of them
// with one token, 592 with two to four, 444 with up to eight).
template <typename TO, int MT>
__global__ void __launch_bounds__(256) int8_few_kernel(const int8_t* __restrict__ x, const float* __restrict__ xs,
                                                       const int8_t* __restrict__ w, const float* __restrict__ ws,
                                                       TO* __restrict__ y, int M, int N, int K) {
  constexpr int kBlockK = 1024;
  __shared__ __align__(16) int8_t sx[MT][kBlockK];
  const int sub = threadIdx.x & 7;
  const int n = (blockIdx.x * 256 + threadIdx.x) >> 3;
  const bool live = n < N;
  const int8_t* wr = w + int64_t(live ? n : N - 1) * K;
  int acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = 0;
  for (int k0 = 0; k0 < K; k0 += kBlockK) {
    int4 b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k0 + i * 128 + sub * 16;
      b[i] = k < K ? __ldg(reinterpret_cast<const int4*>(wr + k)) : make_int4(0, 0, 0, 0);
    }
    if (k0 > 0) __syncthreads();
    for (int i = threadIdx.x; i < MT * (kBlockK / 16); i += 256) {
      const int m = i / (kBlockK / 16), k = k0 + i % (kBlockK / 16) * 16;
      *reinterpret_cast<int4*>(&sx[m][k - k0]) = m < M && k < K
                                                     ? __ldg(reinterpret_cast<const int4*>(x + int64_t(m) * K + k))
                                                     : make_int4(0, 0, 0, 0);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (k0 + i * 128 >= K) break;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int4 a = *reinterpret_cast<const int4*>(&sx[m][i * 128 + sub * 16]);
        acc[m] = __dp4a(a.x, b[i].x, acc[m]);
        acc[m] = __dp4a(a.y, b[i].y, acc[m]);
        acc[m] = __dp4a(a.z, b[i].z, acc[m]);
        acc[m] = __dp4a(a.w, b[i].w, acc[m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
  if (!live) return;
  const float s = ws[n];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    if ((m & 7) == sub && m < M) y[int64_t(m) * N + n] = from_f32<TO>(__int2float_rn(acc[m]) * xs[m] * s);
}

template <typename TO>
int launch_few(const int8_t* x, const float* xs, const int8_t* w, const float* ws, TO* y, int M, int N, int K,
               cudaStream_t s) {
  const unsigned grid = (unsigned)((int64_t(N) * 8 + 255) / 256);
  if (M == 1)
    int8_few_kernel<TO, 1><<<grid, 256, 0, s>>>(x, xs, w, ws, y, M, N, K);
  else if (M == 2)
    int8_few_kernel<TO, 2><<<grid, 256, 0, s>>>(x, xs, w, ws, y, M, N, K);
  else if (M <= 4)
    int8_few_kernel<TO, 4><<<grid, 256, 0, s>>>(x, xs, w, ws, y, M, N, K);
  else
    int8_few_kernel<TO, 8><<<grid, 256, 0, s>>>(x, xs, w, ws, y, M, N, K);
  return check_launch("int8_gemm_few");
}

template <class C, typename TO>
int launch_tiles(const int8_t* x, const float* xs, const int8_t* w, const float* ws, TO* y, int out_dtype, int M,
                 int N, int K, uint32_t* status, cudaStream_t s) {
  TileParams<Int8Epilogue<TO>> prm;
  int st = tile_operand_map<C>(&prm.tm_a, x, false, M, K, K, 128);
  if (st != MT_OK) return st;
  if ((st = tile_operand_map<C>(&prm.tm_b, w, false, N, K, K, C::B_ROWS)) != MT_OK) return st;
  const bool direct = (reinterpret_cast<uintptr_t>(y) & 15u) != 0 || (int64_t(N) * sizeof(TO)) % 16 != 0;
  if (direct)
    prm.tm_out = prm.tm_a;  // not used
  else if ((st = tile_output_map(&prm.tm_out, y, out_dtype, M, N, N)) != MT_OK)
    return st;
  prm.M = M;
  prm.N = N;
  prm.n_k = (K + C::BK - 1) / C::BK;
  prm.k_per_split = prm.n_k;
  prm.per_unit = 0;
  prm.split_rows = 0;
  prm.out = y;
  prm.ld_out = N;
  prm.status = status;
  prm.ep = Int8Epilogue<TO>{xs, ws, N, false, direct};
  return launch_tile_gemm<C>(prm, 1, "int8_gemm", s);
}

template <typename TO>
int run_int8(const int8_t* x, const float* xs, const int8_t* w, const float* ws, void* out, int out_dtype, int M,
             int N, int K, uint32_t* status, cudaStream_t s) {
  TO* y = static_cast<TO*>(out);
  if (M <= kFewTokens) return launch_few<TO>(x, xs, w, ws, y, M, N, K, s);
  // CTA pairs from one and a half 256 x 256 tiles per pair on; smaller products
  // take 128 x 128 tiles, four times as many.  us, pairs / single, by tiles of
  // a pair: 80 (4,096 x 1,280 x 768) 12.4 / 10.1, 64 (1,024 x 4,096 x 1,024) 10.3 / 9.2,
  // 128 (2,048 x 4,096 x 1,024) 13.8 / 14.8, 336 (1,024 x 21,504 x 768) 22.6 / 25.4
  const int64_t pair_tiles = int64_t((M + 255) / 256) * ((N + 255) / 256);
  if (4 * pair_tiles >= 3 * get_sm_count())
    return launch_tiles<TileCfg<kKindI8, false, false, 256, true, 16>, TO>(x, xs, w, ws, y, out_dtype, M, N, K, status, s);
  return launch_tiles<TileCfg<kKindI8, false, false, 128, false, 16>, TO>(x, xs, w, ws, y, out_dtype, M, N, K, status, s);
}

}  // namespace
}  // namespace mt

using namespace mt;

extern "C" int mt_int8_gemm(const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale, void* out,
                            int out_dtype, int64_t M, int64_t N, int64_t K, uint32_t* status, void* stream) {
  if (M < 0 || N <= 0 || K <= 0) return MT_ERR_INVALID_ARGUMENT;
  if (out_dtype != MT_F32 && out_dtype != MT_F16 && out_dtype != MT_BF16) return MT_ERR_UNSUPPORTED_DTYPE;
  if (M > 0x7fffffffLL - 256 || N > 0x7fffffffLL / 8 - 256 || K > kMaxK) return MT_ERR_INVALID_ARGUMENT;
  if (K % 16 != 0) return MT_ERR_UNSUPPORTED_LAYOUT;  // 16-byte rows
  if (M == 0) return MT_OK;
  if (x_scale == nullptr || out == nullptr || status == nullptr) return MT_ERR_INVALID_ARGUMENT;
  for (const void* q : {static_cast<const void*>(x), static_cast<const void*>(w), static_cast<const void*>(w_scale)})
    if (q == nullptr || (reinterpret_cast<uintptr_t>(q) & 15u) != 0) return MT_ERR_UNSUPPORTED_LAYOUT;
  int st = bind_device_of(x);
  if (st != MT_OK) return st;
  if ((st = check_arch()) != MT_OK) return st;
  auto s = static_cast<cudaStream_t>(stream);
  switch (out_dtype) {
    case MT_F32: return run_int8<float>(x, x_scale, w, w_scale, out, out_dtype, (int)M, (int)N, (int)K, status, s);
    case MT_F16: return run_int8<__half>(x, x_scale, w, w_scale, out, out_dtype, (int)M, (int)N, (int)K, status, s);
    default: return run_int8<__nv_bfloat16>(x, x_scale, w, w_scale, out, out_dtype, (int)M, (int)N, (int)K, status, s);
  }
}
