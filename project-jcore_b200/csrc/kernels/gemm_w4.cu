// Product with weights in 4 bits:
//   C[m,n] = act(sum_k x[m,k] * scale[n, k / group] * (nibble[n,k] - zero[n, k / group]) + bias[n]).
// nibble - zero is a whole number of at most 15, exact in fp16 and bf16, and so are its
// products with x in the tensor cores' fp32 sums: only those sums, the groups' products
// with their scales and the result round. (x in fp32 enters as three bf16 parts that add
// up to it exactly.)
//
//   rows    (gemm_w4_rows.cu) few tokens: warps stream the weights into mma.sync fragments;
//   mma     (gemm_w4_mma.cu) more tokens: tcgen05 tiles;
//   tiles   (below) weights that are not 16-byte aligned.
#include "gemm_w4.cuh"
#include "ptx_sm100.cuh"

namespace nplk {
namespace {

// ---------------------------------------------------------------------------
// tiles: 64 x 64 results a CTA, 32 of K at a time as fp32 in shared memory, all of one group.
// 256 threads, 4 x 4 results each: the group's sums, which its scales multiply at its end, and
// the results'; four CTAs an SM (three, which the registers of both would leave, took 1388 us at 512 x
// 4096 x 4096 bf16, now 1030; single bytes and values are loaded, 1 x 4096 x 4096 takes 390).
// ---------------------------------------------------------------------------
constexpr int kTile = 64, kTileK = 32, kTilePitch = kTileK + 1;

template <typename X, typename T>
__global__ void __launch_bounds__(256, 4) gemm_w4_tiles_kernel(W4Args p, const X *x, T *C) {
  __shared__ float sx[kTile * kTilePitch], sw[kTile * kTilePitch], scales[kTile];
  const int64_t m_tiles = (static_cast<int64_t>(p.M) + kTile - 1) / kTile;
  const int64_t m0 = blockIdx.x % m_tiles * kTile, n0 = blockIdx.x / m_tiles * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int group_bits = __ffs(p.group) - 1;
  float acc[4][4] = {}, part[4][4] = {};
  griddep_wait();
  griddep_launch_dependents();
  for (int k0 = 0; k0 < p.K; k0 += kTileK) {
    for (int i = threadIdx.x; i < kTile * kTileK; i += 256) {
      const int r = i / kTileK, k = k0 + i % kTileK;
      float v = 0.0f, w = 0.0f;
      if (k < p.K && m0 + r < p.M) v = to_float(x[(m0 + r) * p.ldx + k]);
      if (k < p.K && n0 + r < p.N) {
        const int64_t n = n0 + r;
        const int nibble = p.q[n * p.ldq + k / 2] >> (k % 2 * 4) & 15;
        const int zero = p.zero ? p.zero[n * p.ldz + (k0 >> group_bits)] & 15 : 8;
        w = static_cast<float>(nibble - zero);
      }
      sx[r * kTilePitch + i % kTileK] = v;
      sw[r * kTilePitch + i % kTileK] = w;
    }
    if ((k0 & (p.group - 1)) == 0 && threadIdx.x < kTile) {
      const int64_t n = min(n0 + threadIdx.x, static_cast<int64_t>(p.N) - 1);
      scales[threadIdx.x] = load_scale(p.scale, p.scale_type, n * p.lds + (k0 >> group_bits));
    }
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < kTileK; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = sx[(ty + 16 * i) * kTilePitch + k];
        b[i] = sw[(tx + 16 * i) * kTilePitch + k];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = fmaf(a[i], b[j], part[i][j]);
    }
    if (((k0 + kTileK) & (p.group - 1)) == 0 || k0 + kTileK >= p.K) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = scales[tx + 16 * j];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[i][j] = fmaf(s, part[i][j], acc[i][j]);
          part[i][j] = 0.0f;
        }
      }
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      v[j] = acc[i][j] + (p.bias && n < p.N ? p.bias[n] : 0.0f);
    }
    act_array<T, false>(v, p.act, p.alpha);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (m < p.M && n < p.N) C[m * p.ldc + n] = from_float<T>(v[j]);
    }
  }
}

template <typename X, typename T>
int run_tiles(cudaStream_t s, const W4Args &p) {
  const int64_t tiles = ceil_div(p.M, kTile) * ceil_div(p.N, kTile);
  if (tiles >= (int64_t(1) << 31)) return kErrUnsupported;
  return launch_programmatic(gemm_w4_tiles_kernel<X, T>, dim3(static_cast<unsigned>(tiles)),
                             dim3(256), 0, s, p, static_cast<const X *>(p.x),
                             static_cast<T *>(p.C));
}

template <typename X>
int run_tiles(cudaStream_t s, const W4Args &p) {
  if (p.c_type == NPLK_DTYPE_FP32) return run_tiles<X, float>(s, p);
  if (p.c_type == NPLK_DTYPE_FP16) return run_tiles<X, __half>(s, p);
  return run_tiles<X, __nv_bfloat16>(s, p);
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_gemm_w4(void *stream, int64_t M, int64_t N, int64_t K, int64_t group,
                            int x_dtype, const void *x, int64_t ldx, const uint8_t *q, int64_t ldq,
                            int scale_dtype, const void *scale, int64_t lds, const uint8_t *zero,
                            int64_t ldz, const float *bias, int act, float act_alpha, int c_dtype,
                            void *C, int64_t ldc, int *status) {
  const int xs = dtype_bytes(x_dtype), ss = dtype_bytes(scale_dtype), cs = dtype_bytes(c_dtype);
  if (M < 1 || N < 1 || K < 1 || group < 1 || !xs || !ss || !cs || !x || !q || !scale || !C ||
      ldx < K || ldq < ceil_div(K, 2) || lds < ceil_div(K, group) ||
      (zero && ldz < ceil_div(K, group)) || ldc < N || act < 0 || act > 10)
    return kErrInvalidArg;
  if (reinterpret_cast<uintptr_t>(x) % xs || reinterpret_cast<uintptr_t>(scale) % ss ||
      reinterpret_cast<uintptr_t>(C) % cs || reinterpret_cast<uintptr_t>(bias) % 4 ||
      reinterpret_cast<uintptr_t>(status) % 4)
    return kErrInvalidArg;
  if (!w4_group_ok(group) || M > (int64_t(1) << 30) || N > (int64_t(1) << 30) ||
      K > (int64_t(1) << 30))
    return kErrUnsupported;
  const W4Args p{ldx, ldq, lds, ldz, ldc, x, q, zero, scale, bias, C, static_cast<int>(M),
                 static_cast<int>(N), static_cast<int>(K), static_cast<int>(group),
                 static_cast<int>(ceil_div(K, group)), x_dtype, scale_dtype, c_dtype, act,
                 act_alpha, status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (gemm_w4_rows_fits(p)) return gemm_w4_rows(s, p);
  if (gemm_w4_mma_fits(p)) return gemm_w4_mma(s, p);
  if (x_dtype == NPLK_DTYPE_FP32) return run_tiles<float>(s, p);
  if (x_dtype == NPLK_DTYPE_FP16) return run_tiles<__half>(s, p);
  return run_tiles<__nv_bfloat16>(s, p);
}
