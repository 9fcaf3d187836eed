// Element types of the kernels that take fp32, fp16 and bf16 tensors: values
// are read in packs of up to 16 bytes, computed in fp32 and rounded once
// (to nearest even) on the way out.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "npl_kernels.h"

namespace nplk {

inline int dtype_bytes(int dtype) {
  return dtype == NPLK_DTYPE_FP32 ? 4
         : dtype == NPLK_DTYPE_FP16 || dtype == NPLK_DTYPE_BF16 ? 2
                                                                : 0;
}

// V consecutive elements, moved by one load or store of sizeof(T) * V bytes.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T e[V];
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V> &p, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = to_float(p.e[j]);
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> pack(const float (&v)[V]) {
  Pack<T, V> p;
#pragma unroll
  for (int j = 0; j < V; ++j) p.e[j] = from_float<T>(v[j]);
  return p;
}

// Two values rounded to 16 bits, `a` in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t &>(h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return reinterpret_cast<const uint32_t &>(h);
}

// (a0, a1) * (b0, b1) and (a0, a1) * (b0, b1) + (c0, c1), two fp32 products an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)));
  return reinterpret_cast<const float2 &>(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)),
        "l"(reinterpret_cast<const uint64_t &>(c)));
  return reinterpret_cast<const float2 &>(r);
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)));
  return reinterpret_cast<const float2 &>(r);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The pack's values two by two (a lone one as both halves of one pair).
template <typename T, int V>
__device__ __forceinline__ void unpack_pairs(const Pack<T, V> &p, float2 (&v)[(V + 1) / 2]) {
  if constexpr (V == 1) {
    v[0] = both(to_float(p.e[0]));
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) v[j / 2] = make_float2(to_float(p.e[j]), to_float(p.e[j + 1]));
  }
}

// Loads with no reuse in L1 (each value is read once by one thread). Not the
// non-coherent path: the destination may be the source.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p) {
  Pack<T, V> r;
  if constexpr (sizeof(T) * V == 16) {
    uint4 &u = reinterpret_cast<uint4 &>(r);
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "l"(p));
  } else if constexpr (sizeof(T) * V == 8) {
    uint2 &u = reinterpret_cast<uint2 &>(r);
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
                 : "=r"(u.x), "=r"(u.y)
                 : "l"(p));
  } else {
    r = *reinterpret_cast<const Pack<T, V> *>(p);
  }
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, V> &v) {
  *reinterpret_cast<Pack<T, V> *>(p) = v;
}

// Copies one pack from global to shared memory without passing through
// registers where the hardware can (4, 8 and 16 bytes), counted in the
// thread's cp.async groups; a 2-byte pack is copied at once.
template <typename T, int V>
__device__ __forceinline__ void copy_pack_async(Pack<T, V> *dst, const T *src) {
  constexpr int kBytes = sizeof(T) * V;
  if constexpr (kBytes == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src)
                 : "memory");
  } else if constexpr (kBytes == 4 || kBytes == 8) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src), "n"(kBytes)
                 : "memory");
  } else {
    *dst = *reinterpret_cast<const Pack<T, V> *>(src);
  }
}
__device__ __forceinline__ void copy_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace nplk
