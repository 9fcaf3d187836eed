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

__device__ __forceinline__ Scale split_scale(float value) {
  Scale s;
  s.value = value;
  s.finite = s.value < CUDART_INF_F;
  s.lifted = s.value < 7.8886091e-31f;  // 2^-100
  s.divisor = s.lifted ? s.value * kLift : s.value;
  s.inverse = 1.0f / s.divisor;
  return s;
}
__device__ __forceinline__ Scale make_scale(uint32_t top_bits) {
  return split_scale(scale_of(top_bits));
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

// Four low bytes as one word.
__device__ __forceinline__ uint32_t low_bytes(const uint32_t *b) {
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// One row per block, or per kLanes lanes of a warp, held in registers between the
// two passes: each byte is read once. Thread t of the row's `threads` takes the
// 16-byte packs t, t + threads, ... Bound by memory: 8192 x 4096 bf16 takes 20.1 us,
// 5.0 TB/s, fp32 29 us, 5.7 TB/s.
// kShift: rows that are not 16-byte aligned (odd widths), or whose q is not. The
// packs are those of aligned addresses, so the first holds `head` places that
// belong to the row before; the q pass through shared memory and leave as the
// aligned words of their own row. 8192 x 4095 bf16 takes 30 us so; a thread per
// element took 50 us.
// The bounds of 1024 threads are for 64 registers: two blocks of 512 on an SM.
template <typename T, int NV, int kLanes, bool kShift>
__global__ void __launch_bounds__(kLanes ? 128 : 1024)
    quantize_rows_kernel(int64_t rows, int cols, const T *x, int64_t ldx, int8_t *q, int64_t ldq,
                         float *scale_out) {
  constexpr int V = 16 / sizeof(T);
  // Whether packs past the row are told apart: warps have many (16384 x 320 fp16 with
  // four a lane: 7.2 us against 8.4), blocks of aligned rows next to none (8192 x 4096
  // bf16: 20.5 against 19.9).
  constexpr bool kSkip = kLanes || kShift;
  extern __shared__ __align__(16) uint32_t bytes[];  // kShift: V bytes for each pack
  __shared__ uint32_t red[32];
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kRow = kLanes ? kLanes : 128;
  const int threads = kLanes ? kLanes : static_cast<int>(blockDim.x);
  const int t = kLanes ? static_cast<int>(threadIdx.x) % kRow : static_cast<int>(threadIdx.x);
  const int part = kLanes ? static_cast<int>(threadIdx.x) / kRow : 0;
  int64_t row = static_cast<int64_t>(blockIdx.x) * (128 / kRow) + part;
  const bool live = !kLanes || row < rows;
  if (!live) {  // beside the last rows: an empty one
    row = 0;
    cols = 0;
  }
  const T *xr = x + row * ldx;
  const int head =
      kShift ? static_cast<int>(reinterpret_cast<uintptr_t>(xr) % 16 / sizeof(T)) : 0;
  Pack<T, V> v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * threads) * V - head;
    if (c >= 0 && c + V <= cols) {
      v[i] = load_pack<T, V>(xr + c);
    } else if (!kSkip || c < cols) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        v[i].e[j] = c + j >= 0 && c + j < cols ? xr[c + j] : from_float<T>(0.0f);
    } else {
      v[i] = {};
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) top = max(top, top_of(v[i]));
  if constexpr (kLanes % 32 == 0) {
    top = __reduce_max_sync(0xffffffffu, top);
  } else {
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (!kLanes) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    const int warps = static_cast<int>(blockDim.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
    top = __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
  }
  const Scale scale = make_scale(top);
  if (t == 0 && live) scale_out[row] = scale.value;
  int8_t *qr = q + row * ldq;
  uint32_t *line = bytes + (kLanes ? part * (kLanes * NV * V / 4) : 0);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = t + i * threads, c = at * V - head;
    if (c >= cols) continue;
    uint32_t b[V], w[V / 4];
    quotients(v[i], scale, b);
#pragma unroll
    for (int j = 0; j < V; j += 4) w[j / 4] = low_bytes(b + j);
    if (kShift || c + V <= cols) {
      void *to = kShift ? static_cast<void *>(line + at * (V / 4)) : static_cast<void *>(qr + c);
      if constexpr (V == 8) *static_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
      else *static_cast<uint32_t *>(to) = w[0];
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < cols) qr[c + j] = static_cast<int8_t>(b[j]);
    }
  }
  if constexpr (kShift) {
    if (kLanes) __syncwarp();
    else __syncthreads();
    const int8_t *byte = reinterpret_cast<const int8_t *>(line);
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(qr) % 4);
    const int words = (mis + cols + 3) / 4, by = head - mis;  // byte of element c: c + head
    for (int k = t; k < words; k += threads) {
      const int c = 4 * k - mis, at = 4 * k + by;
      if (c >= 0 && c + 4 <= cols) {
        const uint32_t low = line[at >> 2], high = line[(at + 3) >> 2];
        *reinterpret_cast<uint32_t *>(qr + c) = __funnelshift_r(low, high, (at & 3) * 8);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j >= 0 && c + j < cols) qr[c + j] = byte[at + j];
      }
    }
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
  for (int64_t j = threadIdx.x; j < cols; j += kLongThreads) {
    uint32_t b[1];
    quotients(Pack<T, 1>{{xr[j]}}, scale, b);
    qr[j] = static_cast<int8_t>(b[0]);
  }
}

// Columns, in two kernels. The first takes the columns' largest magnitudes: a
// warp reads 32 * V columns of a row at a time, a CTA joins its run of rows, and
// the CTAs join in scale_out itself: the scale is a monotone function of the
// magnitude, so the largest of the runs' scales is the scale (all are positive,
// their bits ordered like their values), whatever the order of the atomics.
constexpr int kColThreads = 256, kColWarps = kColThreads / 32;

template <typename T, int V>
__global__ void __launch_bounds__(kColThreads, 4)
    column_scales_kernel(int64_t rows, int64_t cols, const T *x, int64_t ldx, float *scale_out,
                         unsigned strips, int64_t rows_each) {
  __shared__ uint32_t red[kColWarps][32 * V];
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x % strips) * (32 * V);
  const int64_t r0 = blockIdx.x / strips * rows_each;
  const int64_t r1 = r0 + rows_each < rows ? r0 + rows_each : rows;
  const int64_t col = c0 + lane * V;
  uint32_t top[V] = {};
  if (col + V <= cols) {
    constexpr int kWords = sizeof(T) == 2 && V > 1 ? V / 2 : V;
    uint32_t most[kWords] = {};
    const T *from = x + (r0 + warp) * ldx + col;
    const int64_t step = kColWarps * ldx;
    for (int64_t r = r0 + warp; r < r1; r += 8 * kColWarps) {
      Pack<T, V> v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r + i * kColWarps < r1) v[i] = load_pack<T, V>(from + i * step);
        else v[i] = {};
      from += 8 * step;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kWords < V) {
          // two 16-bit magnitudes at a time
          const uint32_t *w = reinterpret_cast<const uint32_t *>(&v[i]);
#pragma unroll
          for (int j = 0; j < kWords; ++j) most[j] = __vmaxu2(most[j], w[j] & 0x7fff7fffu);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            most[j] = max(most[j], __float_as_uint(to_float(v[i].e[j])) & 0x7fffffffu);
        }
      }
    }
    if constexpr (kWords < V) {
      const T *m = reinterpret_cast<const T *>(most);
#pragma unroll
      for (int j = 0; j < V; ++j) top[j] = __float_as_uint(to_float(m[j]));
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) top[j] = most[j];
    }
  } else {
    for (int64_t r = r0 + warp; r < r1; r += kColWarps)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (col + j < cols)
          top[j] = max(top[j], __float_as_uint(to_float(x[r * ldx + col + j])) & 0x7fffffffu);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) red[warp][j * 32 + lane] = top[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += kColThreads) {
    uint32_t most = 0;
#pragma unroll
    for (int w = 0; w < kColWarps; ++w) most = max(most, red[w][i]);
    const int64_t c = c0 + i % 32 * V + i / 32;
    if (c >= cols) continue;
    if (rows_each >= rows) scale_out[c] = scale_of(most);
    else atomicMax(reinterpret_cast<unsigned *>(scale_out + c), __float_as_uint(scale_of(most)));
  }
}

// The second: a tile of 256 rows and 32 columns per CTA, a lane per column, which
// finds x in L2 where that holds it; the q pass through shared memory so that
// each column's 256 bytes leave together. 4096 x 4096 fp32 takes 30 us in both
// kernels, 8192 x 4096 fp16 44 us; the second, two thirds of it, is bound by its
// instructions (16 per value). One kernel instead, with clusters over the rows of
// a strip of columns that kept in shared memory what fits there, read x once but
// took 40 and 61 us: its CTAs load and compute in step.
constexpr int kColRows = 256, kColEach = kColRows / kColWarps;  // rows: of a tile, of a lane

template <typename T>
__global__ void __launch_bounds__(kColThreads, 4)
    quantize_cols_kernel(int64_t rows, int64_t cols, const T *x, int64_t ldx, int8_t *q,
                         int64_t ldq, const float *scales, unsigned strips, bool words) {
  __shared__ uint32_t tile[32][kColRows / 4 + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x % strips) * 32;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x / strips) * kColRows;
  const bool in = c0 + lane < cols;
  const int left = static_cast<int>(rows - r0 < kColRows ? rows - r0 : kColRows);
  const T *from = x + (r0 + warp * kColEach) * ldx + c0 + lane;
  Pack<T, kColEach> v;
  if (left == kColRows && in) {
#pragma unroll
    for (int i = 0; i < kColEach; ++i, from += ldx) v.e[i] = *from;
  } else {
#pragma unroll
    for (int i = 0; i < kColEach; ++i, from += ldx)
      v.e[i] = in && warp * kColEach + i < left ? *from : from_float<T>(0.0f);
  }
  griddep_wait();
  griddep_launch_dependents();
  uint32_t b[kColEach];
  quotients(v, split_scale(in ? scales[c0 + lane] : 1.0f), b);
#pragma unroll
  for (int i = 0; i < kColEach; i += 4) tile[lane][(warp * kColEach + i) / 4] = low_bytes(b + i);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = c0 + warp * 4 + i;
    if (c >= cols) continue;
    int8_t *out = q + c * ldq + r0;
#pragma unroll
    for (int r = 4 * lane; r < kColRows; r += 128) {
      const uint32_t w = tile[warp * 4 + i][r / 4];
      if (words && r + 4 <= left) {
        *reinterpret_cast<uint32_t *>(out + r) = w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r + j < left) out[r + j] = static_cast<int8_t>(w >> (8 * j));
      }
    }
  }
}

template <typename T, bool kShift>
int run_rows(cudaStream_t s, int64_t rows, int64_t cols, const T *x, int64_t ldx, int8_t *q,
             int64_t ldq, float *scale) {
  // Packs of a thread in a block: four (and one for the first pack's head), or eight
  // where that took more than 512 threads.
  constexpr int V = 16 / sizeof(T), kFew = kShift ? 5 : 4, kMany = kShift ? 9 : 8;
  const int64_t packs = ceil_div(cols + (kShift ? V - 1 : 0), V);
  if (packs > 512 * kMany) {
    return launch_programmatic(quantize_long_rows_kernel<T>, dim3(static_cast<unsigned>(rows)),
                               dim3(kLongThreads), 0, s, cols, x, ldx, q, ldq, scale);
  }
  auto go = [&](auto *fn, int64_t blocks, int threads, int each) {
    return launch_programmatic(fn, dim3(static_cast<unsigned>(blocks)),
                               dim3(static_cast<unsigned>(threads)),
                               kShift ? static_cast<size_t>(threads) * each * V : 0, s, rows,
                               static_cast<int>(cols), x, ldx, q, ldq, scale);
  };
  // A warp per row, without a barrier, while few registers hold the row; two packs a
  // lane where they do (16384 x 320 fp16: 6.3 us against 7.3 with four), then of a part
  // of the warp (65536 x 64 bf16: 5.5 us against 17.7).
  auto lanes = [&](auto *fn, int each, int per_row) {
    return go(fn, ceil_div(rows, 128 / per_row), 128, each);
  };
  if (packs <= 8 * 2) return lanes(quantize_rows_kernel<T, 2, 8, kShift>, 2, 8);
  if (packs <= 16 * 2) return lanes(quantize_rows_kernel<T, 2, 16, kShift>, 2, 16);
  if (packs <= 32 * 2) return lanes(quantize_rows_kernel<T, 2, 32, kShift>, 2, 32);
  if (packs <= 32 * 4) return lanes(quantize_rows_kernel<T, 4, 32, kShift>, 4, 32);
  if (packs <= 32 * 8) return lanes(quantize_rows_kernel<T, 8, 32, kShift>, 8, 32);
  // A block of 1024 threads has an SM to itself: 4096 x 16384 fp32 took 78.5 us with
  // four packs a thread, 57.0 with eight. Up to 512 threads four are faster (8192 x
  // 4096 bf16: 20.0 us against 21.4).
  auto block = [&](int each) {
    return static_cast<int>(ceil_div(ceil_div(packs, each), 32) * 32);
  };
  if (packs <= 512 * kFew)
    return go(quantize_rows_kernel<T, kFew, 0, kShift>, rows, block(kFew), kFew);
  return go(quantize_rows_kernel<T, kMany, 0, kShift>, rows, block(kMany), kMany);
}

template <typename T>
int run_quantize(cudaStream_t s, int64_t rows, int64_t cols, const T *x, int64_t ldx, int8_t *q,
                 int64_t ldq, float *scale, bool by_rows) {
  if (by_rows) {
    constexpr int V = 16 / sizeof(T);
    const bool aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % V == 0 &&
                         reinterpret_cast<uintptr_t>(q) % V == 0 && ldq % V == 0;
    return aligned ? run_rows<T, false>(s, rows, cols, x, ldx, q, ldq, scale)
                   : run_rows<T, true>(s, rows, cols, x, ldx, q, ldq, scale);
  }
  constexpr int V = 16 / sizeof(T);
  const bool packs = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % V == 0;
  const int64_t strips = ceil_div(cols, 32), tiles = strips * ceil_div(rows, kColRows);
  if (tiles >= (int64_t(1) << 31)) return kErrUnsupported;
  // As many runs of rows as fill the GPU, of 64 rows or more: 512 x 320 takes 8.3 us
  // with eight runs, 13.5 us with one, although that needs no zeros to start from.
  const int64_t wide = ceil_div(cols, packs ? 32 * V : 32);
  const int64_t most = std::min(ceil_div(rows, 64), ceil_div(148 * 8, wide));
  const int64_t each = ceil_div(rows, most);
  int rc = 0;
  if (most > 1)
    rc = map_cuda_error(cudaMemsetAsync(scale, 0, static_cast<size_t>(cols) * sizeof(float), s));
  if (rc) return rc;
  auto *fn = packs ? column_scales_kernel<T, V> : column_scales_kernel<T, 1>;
  count_launch();
  fn<<<static_cast<unsigned>(wide * ceil_div(rows, each)), kColThreads, 0, s>>>(
      rows, cols, x, ldx, scale, static_cast<unsigned>(wide), each);
  rc = launch_result();
  if (rc) return rc;
  const bool words = reinterpret_cast<uintptr_t>(q) % 4 == 0 && ldq % 4 == 0;
  return launch_programmatic(quantize_cols_kernel<T>, dim3(static_cast<unsigned>(tiles)),
                             dim3(kColThreads), 0, s, rows, cols, x, ldx, q, ldq, scale,
                             static_cast<unsigned>(strips), words);
}

int quantize_lines(void *stream, int64_t rows, int64_t cols, int dtype, const void *x,
                   int64_t ldx, int8_t *q, int64_t ldq, float *scale, bool by_rows) {
  const int size = dtype_bytes(dtype);
  if (rows < 1 || cols < 1 || !size || !x || !q || !scale || ldx < cols ||
      ldq < (by_rows ? cols : rows))
    return kErrInvalidArg;
  if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(scale) % 4)
    return kErrInvalidArg;
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
