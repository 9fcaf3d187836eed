// Matrix product in 8-bit integers with a scale for each token and channel:
//   C[m,n] = act(a_scale[m] * b_scale[n] * sum_k A[m,k] B[n,k] + bias[n]).
// |A * B| <= 2^14, so 32-bit sums are exact up to K = 131071.
#include "nplk_device.cuh"
#include "nplk_host.h"
#include "typed_io.cuh"

namespace nplk {
namespace {

struct I8Args {
  int64_t M, N, K, lda, ldb, ldc;
  const int8_t *A, *B;
  const float *a_scale, *b_scale, *bias;
  int act;
  float alpha;
};

// Any pitch and alignment: 64 x 64 tiles, 64 bytes of K at a time gathered by
// bytes into shared memory, four products an instruction (dp4a). 256 threads,
// 4 x 4 results each.
constexpr int kTile = 64, kPitch = 17;  // words a row: 16, and one against bank conflicts

template <typename T>
__global__ void __launch_bounds__(256) gemm_i8_bytes_kernel(I8Args p, T *C) {
  __shared__ int sa[kTile * kPitch], sb[kTile * kPitch];
  const int64_t m_tiles = (p.M + kTile - 1) / kTile;
  const int64_t m0 = blockIdx.x % m_tiles * kTile, n0 = blockIdx.x / m_tiles * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.K; k0 += 64) {
    for (int i = threadIdx.x; i < kTile * 64; i += 256) {
      const int r = i >> 6, k = i & 63;
      const bool in_k = k0 + k < p.K;
      reinterpret_cast<int8_t *>(sa + r * kPitch)[k] =
          in_k && m0 + r < p.M ? p.A[(m0 + r) * p.lda + k0 + k] : int8_t(0);
      reinterpret_cast<int8_t *>(sb + r * kPitch)[k] =
          in_k && n0 + r < p.N ? p.B[(n0 + r) * p.ldb + k0 + k] : int8_t(0);
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      int a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = sa[(ty + 16 * i) * kPitch + w];
        b[i] = sb[(tx + 16 * i) * kPitch + w];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (m < p.M && n < p.N) {
        const float v = fmaf(static_cast<float>(acc[i][j]) * p.a_scale[m], p.b_scale[n],
                             p.bias ? p.bias[n] : 0.0f);
        C[m * p.ldc + n] = from_float<T>(apply_act(v, p.act, p.alpha));
      }
    }
  }
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_gemm_i8(void *stream, int64_t M, int64_t N, int64_t K, const int8_t *A,
                            int64_t lda, const float *a_scale, const int8_t *B, int64_t ldb,
                            const float *b_scale, const float *bias, int act, float act_alpha,
                            int c_dtype, void *C, int64_t ldc, int *status) {
  const int size = dtype_bytes(c_dtype);
  if (M < 1 || N < 1 || K < 1 || !A || !B || !a_scale || !b_scale || !C || !size || lda < K ||
      ldb < K || ldc < N || act < 0 || act > 10)
    return kErrInvalidArg;
  if (reinterpret_cast<uintptr_t>(C) % size) return kErrInvalidArg;
  if (M > (int64_t(1) << 30) || N > (int64_t(1) << 30) || K > 131071) return kErrUnsupported;
  (void)status;
  I8Args p{M, N, K, lda, ldb, ldc, A, B, a_scale, b_scale, bias, act, act_alpha};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t tiles = ceil_div(M, kTile) * ceil_div(N, kTile);
  if (tiles >= (int64_t(1) << 31)) return kErrUnsupported;
  auto go = [&](auto zero) {
    using T = decltype(zero);
    gemm_i8_bytes_kernel<T><<<static_cast<unsigned>(tiles), 256, 0, s>>>(p, static_cast<T *>(C));
  };
  if (c_dtype == NPLK_DTYPE_FP32) go(float{});
  else if (c_dtype == NPLK_DTYPE_FP16) go(__half{});
  else go(__nv_bfloat16{});
  count_launch();
  return launch_result();
}
