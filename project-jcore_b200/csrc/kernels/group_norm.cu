// Group norm with an activation, channels last, and its gradient.
//
// For image i and group g (cg = c / groups channels, M = hw * cg values):
//   mean, M2 = sum (x - mean)^2, rstd = 1/sqrt(M2 / M + eps),
//   y = act(gamma * (x - mean) * rstd + beta).
// Gradient, with xh = (x - mean) * rstd, z = gamma * xh + beta, dz = dy * act'(z):
//   dx = rstd * (gamma * dz - (A + xh * B) / M), A = sum gamma dz, B = sum gamma dz xh,
//   dgamma = sum dz * xh, dbeta = sum dz over images and pixels.
#include "activation_grad.cuh"
#include "nplk_host.h"
#include "typed_io.cuh"

namespace nplk {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // red may still be read from the previous sum
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
  for (int w = 0; w < kThreads / 32; ++w) t += red[w];
  return t;
}

struct NormArgs {
  int64_t n, hw, c, groups, ldx, ldy, lddy;
  const float *gamma, *beta;
  float eps, alpha;
  int act;
};

// One block per image and group, three passes over the group.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_kernel(NormArgs p, const T *x, T *y, float *mean_out,
                                                        float *rstd_out) {
  __shared__ float red[kThreads / 32];
  const int64_t img = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
  const int64_t cg = p.c / p.groups, m = p.hw * cg;
  const T *xi = x + img * p.hw * p.ldx + g * cg;
  float s = 0.0f;
  for (int64_t i = threadIdx.x; i < m; i += kThreads) s += to_float(xi[i / cg * p.ldx + i % cg]);
  const float mean = block_sum(s, red) / static_cast<float>(m);
  float q = 0.0f;
  for (int64_t i = threadIdx.x; i < m; i += kThreads) {
    const float d = to_float(xi[i / cg * p.ldx + i % cg]) - mean;
    q += d * d;
  }
  const float rstd = 1.0f / sqrtf(block_sum(q, red) / static_cast<float>(m) + p.eps);
  if (threadIdx.x == 0) {
    if (mean_out) mean_out[blockIdx.x] = mean;
    if (rstd_out) rstd_out[blockIdx.x] = rstd;
  }
  T *yi = y + img * p.hw * p.ldy + g * cg;
  for (int64_t i = threadIdx.x; i < m; i += kThreads) {
    const int64_t ch = g * cg + i % cg;
    const float xh = (to_float(xi[i / cg * p.ldx + i % cg]) - mean) * rstd;
    const float z = (p.gamma ? p.gamma[ch] : 1.0f) * xh + (p.beta ? p.beta[ch] : 0.0f);
    yi[i / cg * p.ldy + i % cg] = from_float<T>(apply_act(z, p.act, p.alpha));
  }
}

// One block per image and group: per-channel sums of the image into
// part[img][2][c], then dx.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_grad_kernel(NormArgs p, const T *dy, const T *x, const float *mean_in,
                     const float *rstd_in, T *dx, float *part) {
  __shared__ float red[kThreads / 32];
  const int64_t img = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
  const int64_t cg = p.c / p.groups;
  const float mean = mean_in[blockIdx.x], rstd = rstd_in[blockIdx.x];
  const T *xi = x + img * p.hw * p.ldx + g * cg;
  const T *di = dy + img * p.hw * p.lddy + g * cg;
  T *oi = dx + img * p.hw * p.ldy + g * cg;
  float a = 0.0f, b = 0.0f;
  for (int64_t ch = 0; ch < cg; ++ch) {
    const float ga = p.gamma ? p.gamma[g * cg + ch] : 1.0f;
    const float be = p.beta ? p.beta[g * cg + ch] : 0.0f;
    float sp = 0.0f, sq = 0.0f;
    for (int64_t r = threadIdx.x; r < p.hw; r += kThreads) {
      const float xh = (to_float(xi[r * p.ldx + ch]) - mean) * rstd;
      const float dz = to_float(di[r * p.lddy + ch]) * act_slope(ga * xh + be, p.act, p.alpha);
      sp += dz;
      sq += dz * xh;
    }
    sp = block_sum(sp, red);
    sq = block_sum(sq, red);
    a += ga * sp;
    b += ga * sq;
    if (threadIdx.x == 0) {
      part[(img * 2 + 0) * p.c + g * cg + ch] = sq;
      part[(img * 2 + 1) * p.c + g * cg + ch] = sp;
    }
  }
  const float inv = 1.0f / static_cast<float>(p.hw * cg);
  for (int64_t i = threadIdx.x; i < p.hw * cg; i += kThreads) {
    const int64_t r = i / cg, ch = i % cg;
    const float ga = p.gamma ? p.gamma[g * cg + ch] : 1.0f;
    const float be = p.beta ? p.beta[g * cg + ch] : 0.0f;
    const float xh = (to_float(xi[r * p.ldx + ch]) - mean) * rstd;
    const float dz = to_float(di[r * p.lddy + ch]) * act_slope(ga * xh + be, p.act, p.alpha);
    oi[r * p.ldy + ch] = from_float<T>(rstd * (ga * dz - (a + xh * b) * inv));
  }
}

__global__ void param_grad_kernel(int64_t rows, int64_t c, const float *part, float *dgamma,
                                  float *dbeta) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= 2 * c) return;
  float *out = i < c ? dgamma : dbeta;
  if (!out) return;
  float s = 0.0f;
  for (int64_t r = 0; r < rows; ++r) s += part[r * 2 * c + i];
  out[i < c ? i : i - c] = s;
}

// 0, or why the sizes are refused.
int check_sizes(int64_t n, int64_t hw, int64_t c, int64_t groups) {
  if (n < 1 || hw < 1 || c < 1 || groups < 1 || c % groups != 0) return kErrInvalidArg;
  if (n >= (int64_t(1) << 31) || hw >= (int64_t(1) << 31) || c / groups > 8192)
    return kErrUnsupported;
  if (n > ((int64_t(1) << 31) - 1) / groups) return kErrUnsupported;
  return kOk;
}

bool element_aligned(const void *p, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" size_t nplk_group_norm_workspace_size(int64_t n, int64_t hw, int64_t c,
                                                 int64_t groups) {
  if (check_sizes(n, hw, c, groups) != kOk) return 0;
  return align_up(static_cast<size_t>(n) * 2 * c * sizeof(float), 256);
}

extern "C" int nplk_group_norm_act(void *stream, int64_t n, int64_t hw, int64_t c, int64_t groups,
                                   int dtype, const void *x, int64_t ldx, const float *gamma,
                                   const float *beta, float eps, int act, float act_alpha, void *y,
                                   int64_t ldy, float *mean, float *rstd, void *workspace,
                                   size_t workspace_bytes) {
  const int size = dtype_bytes(dtype);
  if (!size || !x || !y || ldx < c || ldy < c || act < 0 || act > 10) return kErrInvalidArg;
  if (int rc = check_sizes(n, hw, c, groups)) return rc;
  if (!element_aligned(x, size) || !element_aligned(y, size) || (x == y && ldx != ldy))
    return kErrInvalidArg;
  if (!workspace || !element_aligned(workspace, 256) ||
      workspace_bytes < nplk_group_norm_workspace_size(n, hw, c, groups))
    return kErrInvalidArg;
  NormArgs p{n, hw, c, groups, ldx, ldy, 0, gamma, beta, eps, act_alpha, act};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(n * groups);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    norm_kernel<T><<<grid, kThreads, 0, s>>>(p, static_cast<const T *>(x), static_cast<T *>(y),
                                             mean, rstd);
  };
  if (dtype == NPLK_DTYPE_FP32) go(float{});
  else if (dtype == NPLK_DTYPE_FP16) go(__half{});
  else go(__nv_bfloat16{});
  count_launch();
  return launch_result();
}

extern "C" int nplk_group_norm_act_backward(void *stream, int64_t n, int64_t hw, int64_t c,
                                            int64_t groups, int dtype, const void *dy,
                                            int64_t lddy, const void *x, int64_t ldx,
                                            const float *mean, const float *rstd,
                                            const float *gamma, const float *beta, int act,
                                            float act_alpha, void *dx, int64_t lddx,
                                            float *dgamma, float *dbeta, void *workspace,
                                            size_t workspace_bytes) {
  const int size = dtype_bytes(dtype);
  if (!size || !dy || !x || !mean || !rstd || !dx || lddy < c || ldx < c || lddx < c || act < 0 ||
      act > 10)
    return kErrInvalidArg;
  if (int rc = check_sizes(n, hw, c, groups)) return rc;
  if (!element_aligned(dy, size) || !element_aligned(x, size) || !element_aligned(dx, size) ||
      (dx == dy && lddx != lddy) || (dx == x && lddx != ldx))
    return kErrInvalidArg;
  if (!workspace || !element_aligned(workspace, 256) ||
      workspace_bytes < nplk_group_norm_workspace_size(n, hw, c, groups))
    return kErrInvalidArg;
  NormArgs p{n, hw, c, groups, ldx, lddx, lddy, gamma, beta, 0.0f, act_alpha, act};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(n * groups);
  float *part = static_cast<float *>(workspace);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    norm_grad_kernel<T><<<grid, kThreads, 0, s>>>(p, static_cast<const T *>(dy),
                                                  static_cast<const T *>(x), mean, rstd,
                                                  static_cast<T *>(dx), part);
  };
  if (dtype == NPLK_DTYPE_FP32) go(float{});
  else if (dtype == NPLK_DTYPE_FP16) go(__half{});
  else go(__nv_bfloat16{});
  count_launch();
  if (int rc = launch_result()) return rc;
  if (dgamma || dbeta) {
    param_grad_kernel<<<static_cast<unsigned>(ceil_div(2 * c, kThreads)), kThreads, 0, s>>>(
        n, c, part, dgamma, dbeta);
    count_launch();
  }
  return launch_result();
}
