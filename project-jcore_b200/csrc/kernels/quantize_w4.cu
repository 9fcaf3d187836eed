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

// Two values in one register: two rows of 16-bit types, one of fp32 in each.
template <typename T>
struct Two {
  using type = float2;
};
template <>
struct Two<__half> {
  using type = __half2;
};
template <>
struct Two<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
__device__ __forceinline__ float2 most2(float2 a, float2 b) {
  return make_float2(most_nan(a.x, b.x), most_nan(a.y, b.y));
}
__device__ __forceinline__ __half2 most2(__half2 a, __half2 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 most2(__nv_bfloat162 a, __nv_bfloat162 b) {
  return __hmax2_nan(a, b);
}
__device__ __forceinline__ float2 shuffle2(float2 a, int o) {
  return make_float2(__shfl_xor_sync(0xffffffffu, a.x, o), __shfl_xor_sync(0xffffffffu, a.y, o));
}
__device__ __forceinline__ __half2 shuffle2(__half2 a, int o) {
  return __shfl_xor_sync(0xffffffffu, a, o);
}
__device__ __forceinline__ __nv_bfloat162 shuffle2(__nv_bfloat162 a, int o) {
  return __shfl_xor_sync(0xffffffffu, a, o);
}

// Eight values' limits, NaN above all: high the largest magnitude, or with zeros the largest
// of w and 0, and low then the largest of -w and 0.
template <typename T, bool kZeros>
__device__ __forceinline__ void limits(const Pack<T, 8> &v, T &high, T &low) {
  if constexpr (std::is_same<T, float>::value) {
    high = low = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      high = most_nan(high, kZeros ? v.e[j] : fabsf(v.e[j]));
      if (kZeros) low = most_nan(low, -v.e[j]);
    }
  } else {
    using T2 = typename Two<T>::type;
    T2 h{}, l{};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const T2 w = reinterpret_cast<const T2 *>(&v)[j];
      h = most2(h, kZeros ? w : __habs2(w));
      if (kZeros) l = most2(l, __hneg2(w));
    }
    high = __hmax_nan(h.x, h.y);
    if (kZeros) low = __hmax_nan(l.x, l.y);
  }
}

// Eight 4-bit numbers, in the low bytes of b, as a word.
__device__ __forceinline__ uint32_t pack_nibbles(const uint32_t (&b)[8]) {
  const uint32_t even = low_bytes(b) & 0x0f0f0f0fu, odd = low_bytes(b + 4) & 0x0f0f0f0fu;
  return __byte_perm(even | even >> 4, odd | odd >> 4, 0x6420);
}

// Eight values an item, a group to group / 8 neighbouring lanes, a row to `lanes` threads (a
// power of two, 32 to 256), four items of a thread at a time: their loads come first, and of
// four lanes each works out the scale of another item (two divisions each).
// 16384 x 4096 bf16 in groups of 128 takes 41 us, of 26 for its bytes; issue is at 71% (a
// thread an item with a division for each value and one for its place took 91 us). kPacks:
// w in whole 16-byte pieces and q in whole words; otherwise value by value.
constexpr int kThreads = 256, kItems = 4;

template <typename T, int kGroup, bool kZeros, bool kPacks>
__global__ void __launch_bounds__(kThreads)
    quantize_w4_kernel(const QuantArgs p, const T *w, int lanes) {
  constexpr int kLanes = kGroup / 8;
  using T2 = typename Two<T>::type;
  griddep_wait();
  griddep_launch_dependents();
  const int t = static_cast<int>(threadIdx.x) & (lanes - 1), lane = static_cast<int>(threadIdx.x) & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / lanes) +
                      static_cast<int>(threadIdx.x) / lanes;
  const bool live = row < p.n;
  const T *x = w + (live ? row : p.n - 1) * p.ldw;
  uint8_t *q = p.q + row * p.ldq;
  // One time round. `whole`: every item lies in the row.
  const auto go = [&](int base, auto tag) {
    constexpr bool whole = decltype(tag)::value;
    Pack<T, 8> v[kItems];
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const int c = (base + u * lanes + t) * 8;
      if (kPacks && (whole || c + 8 <= p.k)) {
        if constexpr (sizeof(T) == 2) {
          v[u] = load_pack<T, 8>(x + c);
        } else {
          *reinterpret_cast<Pack<T, 4> *>(&v[u].e[0]) = load_pack<T, 4>(x + c);
          *reinterpret_cast<Pack<T, 4> *>(&v[u].e[4]) = load_pack<T, 4>(x + c + 4);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[u].e[j] = whole || c + j < p.k ? x[c + j] : from_float<T>(0.0f);
      }
    }
    // limits of the four items' groups, two of them together
    T2 high[2], low[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      limits<T, kZeros>(v[2 * u], high[u].x, low[u].x);
      limits<T, kZeros>(v[2 * u + 1], high[u].y, low[u].y);
#pragma unroll
      for (int o = kLanes / 2; o; o >>= 1) {
        high[u] = most2(high[u], shuffle2(high[u], o));
        if (kZeros) low[u] = most2(low[u], shuffle2(low[u], o));
      }
    }
    // item lane % 4's
    const auto mine = [&](const T2 (&of)[2]) {
      const T2 pair = lane & 2 ? of[1] : of[0];
      return to_float(lane & 1 ? pair.y : pair.x);
    };
    const float h = mine(high), l = kZeros ? mine(low) : 0.0f;
    const Scale s = split_scale(round_scale(kZeros ? (h + l) / 15.0f : h / 7.0f, p.scale_type));
    int zero = 8;
    if (kZeros) {
      uint32_t z[1];
      quotients(Pack<float, 1>{{l}}, s, z);
      zero = static_cast<int>(z[0] & 0xffu);  // at most 15: l is at most 15 scales and a rounding
    }
    // the group's first four lanes store their items' scales
    const int g = (base + (lane & 3) * lanes + t) / kLanes;
    if (lane % kLanes < 4 && live && (whole || g < p.groups)) {
      store_scale(p.scale, p.scale_type, row * p.lds + g, s.value);
      if (kZeros) p.zero[row * p.ldz + g] = static_cast<uint8_t>(zero);
    }
    const bool rare = __any_sync(0xffffffffu, s.lifted);
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const int c = (base + u * lanes + t) * 8;
      const int from = (lane & ~3) + u;
      Scale of;
      of.value = of.divisor = __shfl_sync(0xffffffffu, s.value, from);
      of.inverse = __shfl_sync(0xffffffffu, s.inverse, from);
      of.finite = of.value < CUDART_INF_F;
      of.lifted = false;
      const int z = kZeros ? __shfl_sync(0xffffffffu, zero, from) : 8;
      uint32_t b[8], word;
      if (rare) {
        of = split_scale(of.value);
        quotients(v[u], of, b);
      } else {
        finite_quotients(v[u], of, b);
      }
      if (kZeros) {
        // rounded apart, the largest value and the zero may come to 16
#pragma unroll
        for (int j = 0; j < 8; ++j)
          b[j] = static_cast<uint32_t>(min((static_cast<int>(b[j] << 24) >> 24) + z, 15));
        word = pack_nibbles(b);
      } else {
        word = pack_nibbles(b) ^ 0x88888888u;  // plus 8 in 4 bits
      }
      if (!of.finite) word = kZeros ? 0u : 0x88888888u;
      uint8_t *to = q + c / 2;
      if (kPacks && (whole || c + 8 <= p.k)) {
        if (live) *reinterpret_cast<uint32_t *>(to) = word;
      } else if (live) {
        const int here = min(8, p.k - c);  // may be none or negative
        if (here < 8) word &= (1u << (4 * max(here, 0))) - 1u;  // the half byte behind an odd row is 0
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (2 * j < here) to[j] = static_cast<uint8_t>(word >> (8 * j));
      }
    }
  };
  // whole warps go round together: a group's lanes shuffle
  const int each = lanes * kItems;
  int base = 0;
  for (; (base + each) * 8 <= p.k; base += each) go(base, std::true_type());
  for (; base < p.groups * kLanes; base += each) go(base, std::false_type());
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
