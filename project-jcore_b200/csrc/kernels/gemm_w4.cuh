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

// (a & b) | c, one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// Nibbles as fp16 or bf16 pairs, less their zero, exactly, without a shift for each:
// a nibble in bits 0-3 of 16 ("low") or in bits 4-7 ("high") is masked where it is, an
// exponent set beside it, and one fused multiply-add brings it to its value.
//   fp16: low 1024 + n, times 1; high 1024 + 16 n, times 1/16.
//   bf16 has 7 bits of significand: low 128 + n, times 1/4; high without an exponent is
//   the number 16 n 2^-133 (bit 7 is the lowest exponent bit, and exponents 0 and 1 have the
//   same step), times 2^127. So bf16 weights are quarters, kUnit the factor left for the end.
// Masks, shifts and permutations issue every second cycle; a shift and a subtraction for each pair
// took 14 of those cycles a word against 10, 16 for adjacent pairs.
struct W4Half {
  static constexpr float kUnit = 1.0f;
  static constexpr uint32_t kLowBias = 0x6400u, kHighBias = 0x6400u;
  static constexpr uint32_t kLowScale = 0x3c00u, kHighScale = 0x2c00u;  // 1, 1/16
  static __device__ __forceinline__ uint32_t low_offset(int z) {  // -(1024 + z)
    return 0xe400u + static_cast<uint32_t>(z);
  }
  static __device__ __forceinline__ uint32_t high_offset(int z) {  // -(64 + z)
    return 0xd400u + static_cast<uint32_t>(z << 4);
  }
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const float (&c)[4], uint32_t a0,
                                             uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
          "f"(c[3]));
  }
};
struct W4Bfloat {
  static constexpr float kUnit = 4.0f;
  static constexpr uint32_t kLowBias = 0x4300u, kHighBias = 0u;
  static constexpr uint32_t kLowScale = 0x3e80u, kHighScale = 0x7f00u;  // 1/4, 2^127
  static __device__ __forceinline__ uint32_t low_offset(int z) {  // -(32 + z / 4)
    return 0xc200u + static_cast<uint32_t>(z);
  }
  static __device__ __forceinline__ uint32_t high_offset(int z) {  // -z / 4
    return __float_as_uint(-0.25f * static_cast<float>(z)) >> 16;
  }
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const float (&c)[4], uint32_t a0,
                                             uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
          "f"(c[3]));
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

__device__ __forceinline__ constexpr uint32_t twice(uint32_t half) { return half * 0x00010001u; }

// What the fused multiply-adds add, for one zero: to both halves of low and high pairs.
struct W4Offsets {
  uint32_t low, high;
};
template <typename F>
__device__ __forceinline__ W4Offsets w4_offsets(int zero) {
  return {twice(F::low_offset(zero)), twice(F::high_offset(zero))};
}

// Eight weights less their zero as four pairs (0, 4), (1, 5), (2, 6), (3, 7).
template <typename F>
__device__ __forceinline__ void w4_widen(uint32_t word, const W4Offsets &off, uint32_t (&pair)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint32_t w = i ? word >> 8 : word;
    pair[i] = F::fma(and_or(w, 0x000f000fu, twice(F::kLowBias)), twice(F::kLowScale), off.low);
    pair[i + 1] =
        F::fma(and_or(w, 0x00f000f0u, twice(F::kHighBias)), twice(F::kHighScale), off.high);
  }
}

// The same as adjacent pairs (0, 1), (2, 3), (4, 5), (6, 7): byte i to both halves, its low
// nibble taken from the low half, its high one from the high half. `off`: low_offset in
// the low half, high_offset in the high one.
template <typename F>
__device__ __forceinline__ uint32_t w4_adjacent_offset(int zero) {
  return F::low_offset(zero) | F::high_offset(zero) << 16;
}
template <typename F>
__device__ __forceinline__ uint4 w4_widen_adjacent(uint32_t word, uint32_t off) {
  uint32_t pair[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    pair[i] = F::fma(and_or(__byte_perm(word, 0u, 0x4040u + static_cast<uint32_t>(i) * 0x0101u),
                            0x00f0000fu, F::kLowBias | F::kHighBias << 16),
                     F::kLowScale | F::kHighScale << 16, off);
  return make_uint4(pair[0], pair[1], pair[2], pair[3]);
}

// fp32 as three bf16 parts by truncation: 8 bits of the significand each, so the last
// remainder fits (but for bits below the least denormal). Infinity is its first part
// alone; of a NaN, the remainders are NaN. Two values at a time, the first in the low halves.
__device__ __forceinline__ void w4_split3(float a, float b, uint32_t (&part)[3]) {
  const float inf = __builtin_huge_valf();
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    part[q] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    if (q == 2) break;
    const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u),
                rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    a = q == 0 && fabsf(a) == inf ? 0.0f : ra;
    b = q == 0 && fabsf(b) == inf ? 0.0f : rb;
  }
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
