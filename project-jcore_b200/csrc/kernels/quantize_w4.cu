// Weights to 4 bits with a scale (and a zero point) for each group of a row:
//   symmetric:  s = max(round(max|w| / 7), least),           nibble = rint(w / s) + 8;
//   with zeros: s = max(round((high - low) / 15), least),    zero = rint(-low / s),
//               nibble = rint(w / s) + zero,  low <= 0 <= high,
// clamped to 0..15. The scale is rounded to its stored type first: the quotients are by
// what the product will multiply with. `least` is the type's smallest normal number.
#include <algorithm>
#include <type_traits>

#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "quotient.cuh"
#include "w4_format.cuh"

namespace nplk {
namespace {

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

// Eight values' limits: high the largest magnitude, or with zeros the largest of w and 0, and
// low then the largest of -w and 0. 16-bit types two at a time; NaN stays.
template <typename T, bool kZeros>
__device__ __forceinline__ void limits(const Pack<T, 8> &v, float &high, float &low) {
  if constexpr (std::is_same<T, float>::value) {
    high = low = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      high = most_nan(high, kZeros ? v.e[j] : fabsf(v.e[j]));
      if (kZeros) low = most_nan(low, -v.e[j]);
    }
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 h{}, l{};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const T2 w = reinterpret_cast<const T2 *>(&v)[j];
      h = __hmax2_nan(h, kZeros ? w : __habs2(w));
      if (kZeros) l = __hmax2_nan(l, __hneg2(w));
    }
    high = most_nan(to_float(h.x), to_float(h.y));
    low = most_nan(to_float(l.x), to_float(l.y));
  }
}

// Eight 4-bit numbers, in the low bytes of b, as a word.
__device__ __forceinline__ uint32_t pack_nibbles(const uint32_t (&b)[8]) {
  const uint32_t even = low_bytes(b) & 0x0f0f0f0fu, odd = low_bytes(b + 4) & 0x0f0f0f0fu;
  return __byte_perm(even | even >> 4, odd | odd >> 4, 0x6420);
}

// Eight values an item, a group to group / 8 neighbouring lanes, a row to `lanes` threads (a
// power of two, 32 to 256), kItems items of a thread at a time: their loads come first.
// Bound by memory: 16384 x 4096 bf16 in groups of 128 takes 30 us, 5.6 TB/s (a thread an item
// with a division for each value and one for its place took 91 us). kPacks: w in whole
// 16-byte pieces and q in whole words; otherwise value by value.
constexpr int kThreads = 256, kItems = 4;

template <typename T, int kGroup, bool kZeros, bool kPacks>
__global__ void __launch_bounds__(kThreads)
    quantize_w4_kernel(const QuantArgs p, const T *w, int lanes) {
  constexpr int kLanes = kGroup / 8;
  griddep_wait();
  griddep_launch_dependents();
  const int t = static_cast<int>(threadIdx.x) & (lanes - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / lanes) +
                      static_cast<int>(threadIdx.x) / lanes;
  const bool live = row < p.n;
  const T *x = w + (live ? row : p.n - 1) * p.ldw;
  uint8_t *q = p.q + row * p.ldq;
  const int items = p.groups * kLanes;
  // whole warps go round together: a group's lanes shuffle
  for (int base = 0; base < items; base += lanes * kItems) {
    Pack<T, 8> v[kItems];
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const int c = (base + u * lanes + t) * 8;
      if (kPacks && c + 8 <= p.k) {
        if constexpr (sizeof(T) == 2) {
          v[u] = load_pack<T, 8>(x + c);
        } else {
          *reinterpret_cast<Pack<T, 4> *>(&v[u].e[0]) = load_pack<T, 4>(x + c);
          *reinterpret_cast<Pack<T, 4> *>(&v[u].e[4]) = load_pack<T, 4>(x + c + 4);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[u].e[j] = c + j < p.k ? x[c + j] : from_float<T>(0.0f);
      }
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const int item = base + u * lanes + t, c = item * 8;
      if (base + u * lanes >= items) break;
      float high, low;
      limits<T, kZeros>(v[u], high, low);
#pragma unroll
      for (int o = kLanes / 2; o; o >>= 1) {
        high = most_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
        if (kZeros) low = most_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
      }
      const Scale s =
          split_scale(round_scale(kZeros ? (high + low) / 15.0f : high / 7.0f, p.scale_type));
      int zero = 8;
      if (kZeros) {
        uint32_t z[1];
        quotients(Pack<float, 1>{{low}}, s, z);
        zero = min(static_cast<int>(z[0] & 0xffu), 15);
      }
      if (!live || c >= p.k) continue;
      if (item % kLanes == 0) {
        const int64_t g = item / kLanes;
        store_scale(p.scale, p.scale_type, row * p.lds + g, s.value);
        if (kZeros) p.zero[row * p.ldz + g] = static_cast<uint8_t>(zero);
      }
      uint32_t b[8];
      quotients(v[u], s, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        b[j] += zero;
        if (kZeros) b[j] = static_cast<uint32_t>(max(0, min(15, static_cast<int>(b[j] << 24) >> 24)));
      }
      uint32_t word = pack_nibbles(b);
      uint8_t *to = q + c / 2;
      if (kPacks && c + 8 <= p.k) {
        *reinterpret_cast<uint32_t *>(to) = word;
      } else {
        const int here = min(8, p.k - c);
        if (here < 8) word &= (1u << (4 * here)) - 1u;  // the half byte behind an odd row is 0
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (2 * j < here) to[j] = static_cast<uint8_t>(word >> (8 * j));
      }
    }
  }
}

template <typename T, int kGroup>
int launch(cudaStream_t s, const QuantArgs &p, const T *w) {
  const bool packs = reinterpret_cast<uintptr_t>(w) % 16 == 0 &&
                     (p.ldw * sizeof(T) % 16 == 0 || p.n == 1) &&
                     reinterpret_cast<uintptr_t>(p.q) % 4 == 0 && (p.ldq % 4 == 0 || p.n == 1);
  const int64_t items = static_cast<int64_t>(p.groups) * (kGroup / 8);
  int lanes = 32;
  while (lanes < kThreads && lanes * kItems < items) lanes *= 2;
  const int64_t ctas = ceil_div(p.n, kThreads / lanes);
  auto *fn = p.zero ? (packs ? quantize_w4_kernel<T, kGroup, true, true>
                             : quantize_w4_kernel<T, kGroup, true, false>)
                    : (packs ? quantize_w4_kernel<T, kGroup, false, true>
                             : quantize_w4_kernel<T, kGroup, false, false>);
  return launch_programmatic(fn, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, s, p, w,
                             lanes);
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
