// Weights to 4 bits with a scale (and a zero point) for each group of a row:
//   symmetric:  s = max(round(max|w| / 7), least),           nibble = rint(w / s) + 8;
//   with zeros: s = max(round((high - low) / 15), least),    zero = rint(-low / s),
//               nibble = rint(w / s) + zero,  low <= 0 <= high,
// clamped to 0..15. The scale is rounded to its stored type first: the quotients are by
// what the product will multiply with. `least` is the type's smallest normal number.
#include <algorithm>

#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "w4_format.cuh"

namespace nplk {
namespace {

constexpr float kInf = __builtin_huge_valf();

struct QuantArgs {
  int64_t ldw, ldq, lds, ldz;
  int n, k, groups;
  int scale_type;
  uint8_t *q, *zero;
  void *scale;
};

// Rounded to the stored type, as stored; the value that reads back.
__device__ __forceinline__ float round_scale(float s, int type) {
  if (type == NPLK_DTYPE_FP16) {
    s = __half2float(__float2half_rn(s));
    return s < 6.103515625e-5f ? 6.103515625e-5f : s;
  }
  if (type == NPLK_DTYPE_BF16) s = __bfloat162float(__float2bfloat16_rn(s));
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}
__device__ __forceinline__ void store_scale(void *to, int type, int64_t at, float s) {
  if (type == NPLK_DTYPE_FP32) static_cast<float *>(to)[at] = s;
  else if (type == NPLK_DTYPE_FP16) static_cast<__half *>(to)[at] = __float2half_rn(s);
  else static_cast<__nv_bfloat16 *>(to)[at] = __float2bfloat16_rn(s);
}

// A larger magnitude, with NaN above all.
__device__ __forceinline__ float most_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A group belongs to group / 8 neighbouring lanes, eight values each. kPacks: w in whole
// 16-byte pieces and q in whole words; otherwise value by value.
template <typename T, int kGroup, bool kZeros, bool kPacks>
__global__ void __launch_bounds__(256)
    quantize_w4_kernel(QuantArgs p, const T *w, int64_t items) {
  constexpr int kLanes = kGroup / 8;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  const int per_row = p.groups * kLanes;
  // whole warps go round together: a group's lanes shuffle
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * 256 + (threadIdx.x & ~31); i0 < items;
       i0 += step) {
    const int64_t item = i0 + (threadIdx.x & 31);
    const bool live = item < items;
    const int64_t row = live ? item / per_row : 0;
    const int part = live ? static_cast<int>(item - row * per_row) : 0;
    const int c = part * 8;
    const int here = live ? min(8, p.k - c) : 0;  // may be none or negative
    const T *x = w + row * p.ldw + c;
    float v[8];
    if (kPacks && here == 8) {
      if constexpr (sizeof(T) == 2) {
        unpack(load_pack<T, 8>(x), v);
      } else {
        const Pack<T, 4> a = load_pack<T, 4>(x), b = load_pack<T, 4>(x + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = to_float(a.e[j]);
          v[4 + j] = to_float(b.e[j]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < here ? to_float(x[j]) : 0.0f;
    }
    float high = 0.0f, low = 0.0f;  // low as the largest of -w
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      high = most_nan(high, kZeros ? v[j] : fabsf(v[j]));
      if (kZeros) low = most_nan(low, -v[j]);
    }
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) {
      high = most_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
      if (kZeros) low = most_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    const float s = round_scale(kZeros ? (high + low) / 15.0f : high / 7.0f, p.scale_type);
    const bool finite = s < kInf;
    float zero = 8.0f;
    if (kZeros) zero = finite ? fminf(fmaxf(rintf(low / s), 0.0f), 15.0f) : 0.0f;
    if (here > 0 && part % kLanes == 0) {
      const int64_t g = part / kLanes;
      store_scale(p.scale, p.scale_type, row * p.lds + g, s);
      if (kZeros) p.zero[row * p.ldz + g] = static_cast<uint8_t>(zero);
    }
    if (here <= 0) continue;
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q = finite ? rintf(v[j] / s) + zero : zero;
      // values behind the row's end are 0 bits
      const uint32_t nibble =
          j < here ? static_cast<uint32_t>(fminf(fmaxf(q, 0.0f), 15.0f)) : 0u;
      word |= nibble << (4 * j);
    }
    uint8_t *to = p.q + row * p.ldq + c / 2;
    if (kPacks && here == 8) {
      *reinterpret_cast<uint32_t *>(to) = word;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (2 * j < here) to[j] = static_cast<uint8_t>(word >> (8 * j));
    }
  }
}

template <typename T, int kGroup>
int launch(cudaStream_t s, const QuantArgs &p, const T *w) {
  const bool packs = reinterpret_cast<uintptr_t>(w) % 16 == 0 && p.ldw * sizeof(T) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(p.q) % 4 == 0 && p.ldq % 4 == 0;
  const int64_t items = static_cast<int64_t>(p.n) * p.groups * (kGroup / 8);
  const int64_t ctas = std::min<int64_t>(ceil_div(items, 256), static_cast<int64_t>(sm_count()) * 64);
  auto *fn = p.zero ? (packs ? quantize_w4_kernel<T, kGroup, true, true>
                             : quantize_w4_kernel<T, kGroup, true, false>)
                    : (packs ? quantize_w4_kernel<T, kGroup, false, true>
                             : quantize_w4_kernel<T, kGroup, false, false>);
  return launch_programmatic(fn, dim3(static_cast<unsigned>(ctas)), dim3(256), 0, s, p, w, items);
}

template <typename T>
int run(cudaStream_t s, const QuantArgs &p, const T *w, int64_t group) {
  return group == 32 ? launch<T, 32>(s, p, w) : group == 64 ? launch<T, 64>(s, p, w)
                                                            : launch<T, 128>(s, p, w);
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_quantize_w4(void *stream, int64_t N, int64_t K, int64_t group, int dtype,
                                const void *w, int64_t ldw, uint8_t *q, int64_t ldq,
                                int scale_dtype, void *scale, int64_t lds, uint8_t *zero,
                                int64_t ldz) {
  const int size = dtype_bytes(dtype), scale_size = dtype_bytes(scale_dtype);
  if (N < 1 || K < 1 || group < 1 || !size || !scale_size || !w || !q || !scale || ldw < K ||
      ldq < ceil_div(K, 2) || lds < ceil_div(K, group) || (zero && ldz < ceil_div(K, group)) ||
      reinterpret_cast<uintptr_t>(w) % size || reinterpret_cast<uintptr_t>(scale) % scale_size)
    return kErrInvalidArg;
  if (!w4_group_ok(group) || N > (int64_t(1) << 30) || K > (int64_t(1) << 30))
    return kErrUnsupported;
  const QuantArgs p{ldw, ldq, lds, ldz, static_cast<int>(N), static_cast<int>(K),
                    static_cast<int>(ceil_div(K, group)), scale_dtype, q, zero, scale};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == NPLK_DTYPE_FP32) return run(s, p, static_cast<const float *>(w), group);
  if (dtype == NPLK_DTYPE_FP16) return run(s, p, static_cast<const __half *>(w), group);
  return run(s, p, static_cast<const __nv_bfloat16 *>(w), group);
}
