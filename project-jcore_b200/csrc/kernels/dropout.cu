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
#include "typed_io.cuh"

namespace nplk {
namespace {

constexpr int kThreads = 256;

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t block, uint32_t k0, uint32_t k1) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = 0,
           c3 = 0;
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

__device__ __forceinline__ uint32_t bits16(const Words &w, int k) {
  const uint32_t v = k < 4 ? (k < 2 ? w.w[0] : w.w[1]) : (k < 6 ? w.w[2] : w.w[3]);
  return (k & 1) ? v >> 16 : v & 0xffffu;
}

// One thread per element.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(int64_t n, const T *x, T *y, uint32_t threshold, float scale, uint64_t seed,
                   uint64_t offset, const uint64_t *device_offset) {
  if (device_offset) offset += *device_offset;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const uint64_t j = offset + static_cast<uint64_t>(i);
    const Words w = philox(j >> 3, static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32));
    const float v = to_float(x[i]) * scale;
    y[i] = from_float<T>(bits16(w, static_cast<int>(j & 7)) >= threshold ? v : 0.0f);
  }
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
  const uint32_t threshold = static_cast<uint32_t>(static_cast<double>(p) * 65536.0 + 0.5);
  const float scale =
      threshold == 65536u ? 0.0f : 65536.0f / static_cast<float>(65536u - threshold);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t blocks = ceil_div(n, kThreads);
  const int64_t most = static_cast<int64_t>(sm_count()) * 8;
  const unsigned grid = static_cast<unsigned>(blocks < most ? blocks : most);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    dropout_kernel<T><<<grid, kThreads, 0, s>>>(n, static_cast<const T *>(x),
                                                static_cast<T *>(y), threshold, scale, seed,
                                                offset, device_offset);
  };
  if (dtype == NPLK_DTYPE_FP32) go(float{});
  else if (dtype == NPLK_DTYPE_FP16) go(__half{});
  else go(__nv_bfloat16{});
  count_launch();
  return launch_result();
}
