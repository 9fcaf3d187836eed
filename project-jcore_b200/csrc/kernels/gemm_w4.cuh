// Shared by the kernels of nplk_gemm_w4: arguments, 4-bit numbers as fp16 and bf16 pairs,
// the parts of fp32 inputs, the results' types.
#pragma once

#include "act_epilogue.cuh"
#include "nplk_host.h"
#include "w4_format.cuh"

namespace nplk {

struct W4Args {
  int64_t ldx, ldq, lds, ldz, ldc;
  const void *x;
  const uint8_t *q, *zero;
  const void *scale;
  const float *bias;
  void *C;
  int M, N, K;
  int group, groups;
  int x_type, scale_type, c_type;
  int act;
  float alpha;
  int *status;
};

// Few tokens; whether the call suits the kernel, and the call.
bool gemm_w4_rows_fits(const W4Args &p);
int gemm_w4_rows(cudaStream_t s, const W4Args &p);
// Tiles of the tensor cores' accumulators.
bool gemm_w4_mma_fits(const W4Args &p);
int gemm_w4_mma(cudaStream_t s, const W4Args &p);

// fp16 and bf16. Two nibbles in the low bits of a pair of 16-bit values become the
// numbers 1024 + n (fp16) or 128 + n (bf16) by setting the exponent; subtracting
// 1024 + zero or 128 + zero is then exact.
struct W4Half {
  static constexpr uint32_t kBias = 0x64006400u;
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r =
        __hsub2(reinterpret_cast<const __half2 &>(a), reinterpret_cast<const __half2 &>(b));
    return reinterpret_cast<const uint32_t &>(r);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
struct W4Bfloat {
  static constexpr uint32_t kBias = 0x43004300u;
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(reinterpret_cast<const __nv_bfloat162 &>(a),
                                     reinterpret_cast<const __nv_bfloat162 &>(b));
    return reinterpret_cast<const uint32_t &>(r);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// The matrix instructions' type for inputs of type X, and the parts that X enters in.
template <typename X>
struct W4Type {
  using Frag = W4Bfloat;
  static constexpr int kParts = 1;
};
template <>
struct W4Type<__half> {
  using Frag = W4Half;
  static constexpr int kParts = 1;
};
template <>
struct W4Type<float> {
  using Frag = W4Bfloat;
  static constexpr int kParts = 3;
};

// 1024 + zero (128 + zero) in both halves.
template <typename F>
__device__ __forceinline__ uint32_t w4_offset(int zero) {
  return F::kBias + static_cast<uint32_t>(zero) * 0x00010001u;
}

// Eight weights less their zero as four pairs (0, 4), (1, 5), (2, 6), (3, 7).
template <typename F>
__device__ __forceinline__ void w4_widen(uint32_t word, uint32_t offset, uint32_t (&pair)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    pair[i] = F::sub((word >> (4 * i) & 0x000f000fu) | F::kBias, offset);
}

// fp32 as three bf16 parts by truncation: 8 bits of the significand each, so the last
// remainder fits (but for bits below the least denormal). An infinity or NaN is its first
// part alone.
__device__ __forceinline__ void w4_split3(float x, uint32_t (&part)[3]) {
  const uint32_t bits = __float_as_uint(x);
  part[0] = bits >> 16;
  if ((bits & 0x7f800000u) == 0x7f800000u) {
    if (bits & 0x007fffffu) part[0] |= 0x40u;  // a NaN whose set bits are all cut off
    part[1] = part[2] = 0u;
    return;
  }
  const float r = x - __uint_as_float(bits & 0xffff0000u);
  const uint32_t rb = __float_as_uint(r);
  part[1] = rb >> 16;
  part[2] = __float_as_uint(r - __uint_as_float(rb & 0xffff0000u)) >> 16;
}

// Activation and store of V results of consecutive channels (`whole`: as one pack).
template <int V>
__device__ __forceinline__ void w4_store(const W4Args &p, int64_t at, float (&v)[V], int count,
                                         bool whole) {
  const auto put = [&](auto *c, auto tag) {
    using T = decltype(tag);
    act_array<T, false>(v, p.act, p.alpha);
    if (whole && count >= V) {
      store_pack(c + at, pack<T, V>(v));
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < count) c[at + j] = from_float<T>(v[j]);
    }
  };
  if (p.c_type == NPLK_DTYPE_FP32) put(static_cast<float *>(p.C), float());
  else if (p.c_type == NPLK_DTYPE_FP16) put(static_cast<__half *>(p.C), __half());
  else put(static_cast<__nv_bfloat16 *>(p.C), __nv_bfloat16());
}

}  // namespace nplk
