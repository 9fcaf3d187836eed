// 8-bit operands of nplk_gemm_i8: a scale for each row (token) or column
// (output channel) and the rounded quotients.
//
//   scale = max(max|x| / 127, 2^-126), q = rint(x / scale).
//
// The lower limit keeps the quotient finite where max|x| / 127 is denormal.
// q is the rounding of the correctly rounded fp32 quotient: it depends on x
// alone, not on how a kernel forms it.
#include <math_constants.h>

#include <algorithm>

#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "typed_io.cuh"

namespace nplk {
namespace {

// Magnitudes are compared as bits: for non-negative values the order of the
// bits is the values', infinity is above every number and a NaN above both
// (fmaxf would drop it).
__device__ __forceinline__ float scale_of(uint32_t top_bits) {
  if (top_bits > 0x7f800000u) return CUDART_NAN_F;
  return fmaxf(__uint_as_float(top_bits) / 127.0f, 1.17549435e-38f);  // +infinity stays
}

// Largest magnitude of a pack, as fp32 bits.
template <typename T, int V>
__device__ __forceinline__ uint32_t top_of(const Pack<T, V> &p) {
  uint32_t top = 0;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    // two 16-bit magnitudes at a time
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&p);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) top = __vmaxu2(top, w[j] & 0x7fff7fffu);
    const uint16_t h = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
    return __float_as_uint(to_float(reinterpret_cast<const T &>(h)));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(to_float(p.e[j])) & 0x7fffffffu);
    return top;
  }
}

struct Scale {
  float value;             // as stored
  float divisor, inverse;  // value, or value * 2^64 where `lifted`, and 1 / divisor
  bool finite, lifted;
};

constexpr float kLift = 18446744073709551616.0f;  // 2^64

__device__ __forceinline__ Scale make_scale(uint32_t top_bits) {
  Scale s;
  s.value = scale_of(top_bits);
  s.finite = s.value < CUDART_INF_F;
  s.lifted = s.value < 7.8886091e-31f;  // 2^-100
  s.divisor = s.lifted ? s.value * kLift : s.value;
  s.inverse = 1.0f / s.divisor;
  return s;
}

constexpr float kToInt = 12582912.0f;  // 1.5 * 2^23: a sum's low bits are the rounded integer

// q of a pack, in the low byte of each word: the fp32 quotient x / scale, then
// its rounding to the nearest integer.
//
// The quotient by P. Markstein's method ("Computation of elementary functions on
// the IBM RISC System/6000 processor", 1990): with y the correctly rounded
// 1 / scale and q within one step of x / scale, q + y (x - q scale), the
// remainder exact in one fused step, is x / scale correctly rounded. x * y may be
// 1.5 steps off; one such correction brings it within one, the second is the
// theorem's. The remainder's last bit is at least 2^-48 of the scale where the
// quotient is above 1/4 (below, it rounds to 0 whatever its error): exact for
// scales from 2^-100 on; under that, x and the scale are both lifted by 2^64.
// Correcting only the products near a half instead is no faster: the coarse
// grids of 16-bit types make exact halves common, nearly every warp has one, and
// 8192 x 4096 bf16 took 23 us that way against 21.
template <typename T, int V>
__device__ __forceinline__ void quotients(const Pack<T, V> &p, const Scale &s, uint32_t (&b)[V]) {
  if (!s.finite) {
#pragma unroll
    for (int j = 0; j < V; ++j) b[j] = 0u;
    return;
  }
  float x[V];
  unpack(p, x);
  if (s.lifted) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] *= kLift;
  }
  if constexpr (V % 2 == 0) {
    const float2 y = make_float2(s.inverse, s.inverse), d = make_float2(-s.divisor, -s.divisor);
    const float2 one = make_float2(1.0f, 1.0f), to_int = make_float2(kToInt, kToInt);
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 v = make_float2(x[j], x[j + 1]);
      float2 q = mul2(v, y);
      q = fma2(fma2(q, d, v), y, q);
      q = fma2(fma2(q, d, v), y, q);
      q = fma2(q, one, to_int);
      b[j] = __float_as_uint(q.x);
      b[j + 1] = __float_as_uint(q.y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float q = x[j] * s.inverse;
      q = fmaf(fmaf(q, -s.divisor, x[j]), s.inverse, q);
      q = fmaf(fmaf(q, -s.divisor, x[j]), s.inverse, q);
      b[j] = __float_as_uint(q + kToInt);
    }
  }
}

// The q of a pack to `q`, `count` of them.
template <typename T, int V>
__device__ __forceinline__ void store_quotients(const Pack<T, V> &p, const Scale &s, int8_t *q,
                                                int count, bool whole) {
  uint32_t b[V];
  quotients(p, s, b);
  if constexpr (V >= 4) {
    if (whole && count >= V) {
      uint32_t w[V / 4];
#pragma unroll
      for (int j = 0; j < V / 4; ++j)
        w[j] = __byte_perm(__byte_perm(b[4 * j], b[4 * j + 1], 0x0040),
                           __byte_perm(b[4 * j + 2], b[4 * j + 3], 0x0040), 0x5410);
      if constexpr (V == 8) *reinterpret_cast<uint2 *>(q) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t *>(q) = w[0];
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (j < count) q[j] = static_cast<int8_t>(b[j]);
}

// One row per block, or per warp (kWarpRows), held in registers between the
// two passes: each byte is read once. Thread t of the row's `threads` takes
// packs t, t + threads, ... V: 16-byte packs, or single elements where rows
// are not 16-byte aligned. Bound by memory: 8192 x 4096 bf16 MEASURED.
template <typename T, int V, int NV, bool kWarpRows>
__global__ void __launch_bounds__(kWarpRows ? 128 : 1024)
    quantize_rows_kernel(int64_t rows, int cols, const T *x, int64_t ldx, int8_t *q,
                                     int64_t ldq, float *scale_out, bool whole) {
  __shared__ uint32_t red[32];
  griddep_wait();
  griddep_launch_dependents();
  const int threads = kWarpRows ? 32 : static_cast<int>(blockDim.x);
  const int t = kWarpRows ? static_cast<int>(threadIdx.x) & 31 : static_cast<int>(threadIdx.x);
  const int64_t row = kWarpRows ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) +
                                      (threadIdx.x >> 5)
                                : static_cast<int64_t>(blockIdx.x);
  if (kWarpRows && row >= rows) return;
  const T *xr = x + row * ldx;
  Pack<T, V> v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * threads) * V;
    if (c + V <= cols) {
      v[i] = load_pack<T, V>(xr + c);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i].e[j] = c + j < cols ? xr[c + j] : from_float<T>(0.0f);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) top = max(top, top_of(v[i]));
  top = __reduce_max_sync(0xffffffffu, top);
  if (!kWarpRows) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    const int warps = static_cast<int>(blockDim.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
    top = __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
  }
  const Scale scale = make_scale(top);
  if (t == 0) scale_out[row] = scale.value;
  int8_t *qr = q + row * ldq;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * threads) * V;
    if (c < cols) store_quotients(v[i], scale, qr + c, cols - c, whole);
  }
}

// Rows longer than the registers of a block: read twice.
constexpr int kLongThreads = 1024;

template <typename T>
__global__ void __launch_bounds__(kLongThreads)
    quantize_long_rows_kernel(int64_t cols, const T *x, int64_t ldx, int8_t *q, int64_t ldq,
                              float *scale_out) {
  __shared__ uint32_t red[kLongThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const T *xr = x + static_cast<int64_t>(blockIdx.x) * ldx;
  uint32_t top = 0;
  for (int64_t j = threadIdx.x; j < cols; j += kLongThreads)
    top = max(top, __float_as_uint(to_float(xr[j])) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, red[threadIdx.x & 31]);
  const Scale scale = make_scale(top);
  if (threadIdx.x == 0) scale_out[blockIdx.x] = scale.value;
  int8_t *qr = q + static_cast<int64_t>(blockIdx.x) * ldq;
  for (int64_t j = threadIdx.x; j < cols; j += kLongThreads)
    store_quotients(Pack<T, 1>{{xr[j]}}, scale, qr + j, 1, false);
}

// Columns: a cluster of S CTAs takes 32 columns, its CTAs equal runs of rows
// (multiples of 128). First the columns' largest magnitudes, a lane per column,
// joined over the cluster; then, from L2, the quotients, 128 rows at a time
// through shared memory so that each column's 128 bytes leave together.
constexpr int kColThreads = 256, kColRows = 128;

template <typename T>
__global__ void __launch_bounds__(kColThreads)
    quantize_cols_kernel(int64_t rows, int64_t cols, const T *x, int64_t ldx, int8_t *q,
                         int64_t ldq, float *scale_out, int slices, int64_t rows_each, bool words) {
  __shared__ uint32_t tile[32][kColRows / 4 + 1];
  __shared__ uint32_t red[kColThreads / 32][32];
  __shared__ uint32_t tops[32];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % slices;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) / slices * 32;
  const int64_t col = c0 + lane;
  const bool in = col < cols;
  const int64_t r0 = rank * rows_each;
  const int64_t r1 = r0 + rows_each < rows ? r0 + rows_each : rows;
  uint32_t top = 0;
  if (in) {
#pragma unroll 8
    for (int64_t r = r0 + warp; r < r1; r += kColThreads / 32)
      top = max(top, __float_as_uint(to_float(x[r * ldx + col])) & 0x7fffffffu);
  }
  red[warp][lane] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kColThreads / 32; ++w) top = max(top, red[w][lane]);
  if (slices > 1) {
    if (warp == 0) tops[lane] = top;
    __syncthreads();
    cluster_sync();
    for (int s = 0; s < slices; ++s)
      top = max(top, ld_shared_cluster_u32(mapa_shared(smem_u32(&tops[lane]), s)));
    cluster_sync_relaxed();  // no CTA leaves while another reads its maxima
  }
  const Scale scale = make_scale(top);
  if (rank == 0 && warp == 0 && in) scale_out[col] = scale.value;
  for (int64_t r = r0; r < r1; r += kColRows) {
    __syncthreads();  // the previous tile has been stored
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // this warp's 16 rows, four to a word
      Pack<T, 4> v;
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t rr = r + warp * 16 + i * 4 + j;
        v.e[j] = in && rr < r1 ? x[rr * ldx + col] : from_float<T>(0.0f);
      }
      quotients(v, scale, b);
      tile[lane][warp * 4 + i] =
          __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t c = c0 + warp * 4 + i;
      if (c >= cols) continue;
      const uint32_t w = tile[warp * 4 + i][lane];
      const int64_t rr = r + 4 * lane;
      int8_t *out = q + c * ldq + rr;
      if (words && rr + 4 <= r1) {
        *reinterpret_cast<uint32_t *>(out) = w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (rr + j < r1) out[j] = static_cast<int8_t>(w >> (8 * j));
      }
    }
  }
}

template <typename T, int V>
int run_rows(cudaStream_t s, int64_t rows, int64_t cols, const T *x, int64_t ldx, int8_t *q,
             int64_t ldq, float *scale) {
  constexpr int kNV = V == 1 ? 16 : 4;  // packs of a thread in a block
  const bool whole = V > 1 && reinterpret_cast<uintptr_t>(q) % V == 0 && ldq % V == 0;
  const int64_t packs = ceil_div(cols, V);
  if (packs > 1024 * kNV) {
    return launch_programmatic(quantize_long_rows_kernel<T>, dim3(static_cast<unsigned>(rows)),
                               dim3(kLongThreads), 0, s, cols, x, ldx, q, ldq, scale);
  }
  auto go = [&](auto *fn, int64_t blocks, int threads) {
    return launch_programmatic(fn, dim3(static_cast<unsigned>(blocks)),
                               dim3(static_cast<unsigned>(threads)), 0, s, rows,
                               static_cast<int>(cols), x, ldx, q, ldq, scale, whole);
  };
  // A warp per row, without a barrier, while few registers hold the row.
  if (packs <= 32 * 4) return go(quantize_rows_kernel<T, V, 4, true>, ceil_div(rows, 4), 128);
  if (packs <= 32 * 8)
    return go(quantize_rows_kernel<T, V, 8, true>, ceil_div(rows, 4), 128);
  const int threads = static_cast<int>(ceil_div(ceil_div(packs, kNV), 32) * 32);
  return go(quantize_rows_kernel<T, V, kNV, false>, rows, threads);
}

template <typename T>
int run_quantize(cudaStream_t s, int64_t rows, int64_t cols, const T *x, int64_t ldx, int8_t *q,
                 int64_t ldq, float *scale, bool by_rows) {
  if (by_rows) {
    const bool aligned =
        reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * sizeof(T) % 16 == 0;
    return aligned ? run_rows<T, 16 / sizeof(T)>(s, rows, cols, x, ldx, q, ldq, scale)
                   : run_rows<T, 1>(s, rows, cols, x, ldx, q, ldq, scale);
  }
  int slices = 8;
  while (slices > 1 && static_cast<int64_t>(slices) * kColRows > rows) slices /= 2;
  const int64_t each = ceil_div(ceil_div(rows, slices), kColRows) * kColRows;
  const int64_t ctas = ceil_div(cols, 32) * slices;
  const bool words = reinterpret_cast<uintptr_t>(q) % 4 == 0 && ldq % 4 == 0;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(slices);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = slices > 1 ? 2 : 1;
  cfg.stream = s;
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kColThreads);
  count_launch();
  return map_cuda_error(cudaLaunchKernelEx(&cfg, quantize_cols_kernel<T>, rows, cols, x, ldx, q,
                                           ldq, scale, slices, each, words));
}

int quantize_lines(void *stream, int64_t rows, int64_t cols, int dtype, const void *x,
                   int64_t ldx, int8_t *q, int64_t ldq, float *scale, bool by_rows) {
  const int size = dtype_bytes(dtype);
  if (rows < 1 || cols < 1 || !size || !x || !q || !scale || ldx < cols ||
      ldq < (by_rows ? cols : rows))
    return kErrInvalidArg;
  if (reinterpret_cast<uintptr_t>(x) % size) return kErrInvalidArg;
  if (rows >= (int64_t(1) << 31) || cols >= (int64_t(1) << 31)) return kErrUnsupported;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == NPLK_DTYPE_FP32)
    return run_quantize(s, rows, cols, static_cast<const float *>(x), ldx, q, ldq, scale, by_rows);
  if (dtype == NPLK_DTYPE_FP16)
    return run_quantize(s, rows, cols, static_cast<const __half *>(x), ldx, q, ldq, scale, by_rows);
  return run_quantize(s, rows, cols, static_cast<const __nv_bfloat16 *>(x), ldx, q, ldq, scale,
                      by_rows);
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_quantize_rows(void *stream, int64_t rows, int64_t cols, int dtype,
                                  const void *x, int64_t ldx, int8_t *q, int64_t ldq,
                                  float *scale) {
  return quantize_lines(stream, rows, cols, dtype, x, ldx, q, ldq, scale, true);
}

extern "C" int nplk_quantize_cols(void *stream, int64_t rows, int64_t cols, int dtype,
                                  const void *x, int64_t ldx, int8_t *q, int64_t ldq,
                                  float *scale) {
  return quantize_lines(stream, rows, cols, dtype, x, ldx, q, ldq, scale, false);
}
