// Dropout from a counter-based generator: the mask is recomputed from (seed,
// position) wherever it is needed and never stored.
//
// Eight consecutive positions j (a block, j / 8) share one Philox4x32-10
// output (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", 2011): four 32-bit words, two 16-bit numbers each. 16 bits
// make the keep probability exact to 2^-17; the scale is the inverse of the
// probability that results, so the expected value is x exactly. With 32 bits a
// number the generator's multiplications, not memory, would bound the kernel
// in 16-bit types.
#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "typed_io.cuh"

namespace nplk {
namespace {

constexpr int kThreads = 256;

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t block, uint32_t k0, uint32_t k1) {
  // positions are modulo 2^64, their blocks modulo 2^61
  uint32_t c0 = static_cast<uint32_t>(block),
           c1 = static_cast<uint32_t>(block >> 32) & 0x1fffffffu, c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u;
    const uint64_t b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

__device__ __forceinline__ uint32_t bits16(const Words &w, uint32_t k) {
  const uint32_t v = k < 4 ? (k < 2 ? w.w[0] : w.w[1]) : (k < 6 ? w.w[2] : w.w[3]);
  return (k & 1) ? v >> 16 : v & 0xffffu;
}

struct DropoutArgs {
  int64_t n;
  uint32_t threshold;  // t < 65536
  float scale;
  uint64_t seed, offset;
  const uint64_t *device_offset;
};

// One element by itself: the ends of a vector, and misaligned pointers.
template <typename T>
__device__ __forceinline__ void drop_one(const DropoutArgs &p, uint64_t offset, const T *x, T *y,
                                         int64_t i) {
  const uint64_t j = offset + static_cast<uint64_t>(i);
  const Words w = philox(j >> 3, static_cast<uint32_t>(p.seed),
                         static_cast<uint32_t>(p.seed >> 32));
  const float v = to_float(x[i]) * p.scale;
  y[i] = from_float<T>(bits16(w, static_cast<uint32_t>(j & 7)) >= p.threshold ? v : 0.0f);
}

// Pointers aligned differently: a thread per generator block, elements one at
// a time.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    dropout_elements_kernel(DropoutArgs p, const T *x, T *y) {
  griddep_wait();
  griddep_launch_dependents();
  uint64_t offset = p.offset;
  if (p.device_offset) offset += *p.device_offset;
  const int64_t lead = static_cast<int64_t>(offset & 7);
  const int64_t block = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const Words w = philox((offset >> 3) + static_cast<uint64_t>(block),
                         static_cast<uint32_t>(p.seed), static_cast<uint32_t>(p.seed >> 32));
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int64_t i = block * 8 - lead + k;
    if (i >= 0 && i < p.n) {
      const float v = to_float(x[i]) * p.scale;
      y[i] = from_float<T>(bits16(w, k) >= p.threshold ? v : 0.0f);
    }
  }
}

// Groups of eight elements from element `head` on, whose addresses are aligned
// to 16 bytes; a warp takes kUnroll * 32 consecutive groups. Where positions
// and groups are out of step by `lead`, a group needs its own generator block
// and the next one, which the next lane has (for lane 31: lane 0's of the next
// step), so each lane computes kUnroll + 1 blocks instead of two per group.
// Memory bounds it in fp32: 25.7 M values take 33 us, 6.2 TB/s; in bf16 18.5 us, 5.6
// TB/s, the generator's integer products (4 a round and block, ten rounds) beside it.
constexpr int kUnroll = 4;

template <typename T>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(DropoutArgs p, const T *x, T *y, int head, int64_t groups) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T)), kPacks = 8 / kPer;
  griddep_wait();
  griddep_launch_dependents();
  uint64_t offset = p.offset;
  if (p.device_offset) offset += *p.device_offset;
  if (blockIdx.x == 0) {
    if (static_cast<int>(threadIdx.x) < head) drop_one(p, offset, x, y, threadIdx.x);
    const int64_t i = head + 8 * groups + threadIdx.x;
    if (i < p.n) drop_one(p, offset, x, y, i);  // fewer than eight are left
  }
  const int lane = threadIdx.x & 31;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t first = warp * (kUnroll * 32);
  if (first >= groups) return;
  Pack<T, kPer> v[kUnroll][kPacks];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t g = first + u * 32 + lane;
    if (g < groups)
#pragma unroll
      for (int q = 0; q < kPacks; ++q) v[u][q] = load_pack<T, kPer>(x + head + 8 * g + kPer * q);
  }
  const uint64_t at = offset + static_cast<uint64_t>(head);
  const uint64_t block = (at >> 3) + static_cast<uint64_t>(first + lane);
  const uint32_t lead = static_cast<uint32_t>(at & 7);
  const uint32_t k0 = static_cast<uint32_t>(p.seed), k1 = static_cast<uint32_t>(p.seed >> 32);
  const uint32_t limit = p.threshold << 16;
  Words now = philox(block, k0, k1);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    Words r = now;
    if (u + 1 < kUnroll || lead) now = philox(block + 32u * (u + 1), k0, k1);
    if (lead) {
      uint32_t w[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        w[q] = r.w[q];
        w[4 + q] = __shfl_sync(0xffffffffu, lane == 0 ? now.w[q] : r.w[q], (lane + 1) & 31);
      }
      if (lead & 4) {
#pragma unroll
        for (int q = 0; q < 6; ++q) w[q] = w[q + 2];
      }
      if (lead & 2) {
#pragma unroll
        for (int q = 0; q < 5; ++q) w[q] = w[q + 1];
      }
      if (lead & 1) {
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = __funnelshift_r(w[q], w[q + 1], 16);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) r.w[q] = w[q];
    }
    const int64_t g = first + u * 32 + lane;
    if (g < groups) {
#pragma unroll
      for (int q = 0; q < kPacks; ++q) {
        float f[kPer];
        unpack(v[u][q], f);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const uint32_t word = r.w[(q * kPer + k) >> 1];
          // number >= threshold, compared in the upper half of a word
          const bool keep = ((k & 1) ? word : word << 16) >= limit;
          f[k] = keep ? f[k] * p.scale : 0.0f;
        }
        store_pack(y + head + 8 * g + kPer * q, pack<T, kPer>(f));
      }
    }
  }
}

template <typename T>
int run_dropout(cudaStream_t s, const DropoutArgs &p, const T *x, T *y) {
  const uintptr_t ax = reinterpret_cast<uintptr_t>(x) % 16,
                  ay = reinterpret_cast<uintptr_t>(y) % 16;
  if (ax != ay) {
    const int64_t blocks = ceil_div(p.n + 7, 8);
    return launch_programmatic(dropout_elements_kernel<T>,
                               dim3(static_cast<unsigned>(ceil_div(blocks, kThreads))),
                               dim3(kThreads), 0, s, p, x, y);
  }
  int64_t head = ax ? static_cast<int64_t>((16u - ax) / sizeof(T)) : 0;
  if (head > p.n) head = p.n;
  const int64_t groups = (p.n - head) / 8;
  const int64_t per_cta = kThreads * kUnroll;
  const int64_t grid = groups > 0 ? ceil_div(groups, per_cta) : 1;
  return launch_programmatic(dropout_kernel<T>, dim3(static_cast<unsigned>(grid)), dim3(kThreads),
                             0, s, p, x, y, static_cast<int>(head), groups);
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_dropout(void *stream, int64_t n, int dtype, const void *x, void *y, float p,
                            uint64_t seed, uint64_t offset, const uint64_t *device_offset) {
  const int size = dtype_bytes(dtype);
  if (n < 1 || !size || !x || !y || !(p >= 0.0f && p <= 1.0f)) return kErrInvalidArg;
  if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(y) % size ||
      reinterpret_cast<uintptr_t>(device_offset) % 8)
    return kErrInvalidArg;
  if (n > (int64_t(1) << 40)) return kErrUnsupported;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t threshold = static_cast<uint32_t>(static_cast<double>(p) * 65536.0 + 0.5);
  if (threshold == 65536u)  // nothing is kept
    return map_cuda_error(cudaMemsetAsync(y, 0, static_cast<size_t>(n) * size, s));
  const float scale = 65536.0f / static_cast<float>(65536u - threshold);
  const DropoutArgs a{n, threshold, scale, seed, offset, device_offset};
  if (dtype == NPLK_DTYPE_FP32)
    return run_dropout(s, a, static_cast<const float *>(x), static_cast<float *>(y));
  if (dtype == NPLK_DTYPE_FP16)
    return run_dropout(s, a, static_cast<const __half *>(x), static_cast<__half *>(y));
  return run_dropout(s, a, static_cast<const __nv_bfloat16 *>(x), static_cast<__nv_bfloat16 *>(y));
}
