// Product with weights in 4 bits:
//   C[m,n] = act(sum_k x[m,k] * scale[n, k / group] * (nibble[n,k] - zero[n, k / group]) + bias[n]).
// nibble - zero is a whole number of at most 15, exact in fp16 and bf16, and so are its
// products with x in the tensor cores' fp32 sums: only those sums, the groups' products
// with their scales and the result round. (x in fp32 enters as three bf16 parts that add
// up to it exactly.)
//
//   rows    few tokens: the weights' bytes. Warps stream 16 channels at a time into
//           mma.sync fragments and share K.
//   tiles   everything else: any pitch, alignment and size.
#include <algorithm>

#include "act_epilogue.cuh"
#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "w4_format.cuh"

namespace nplk {
namespace {

struct W4Args {
  int64_t ldx, ldq, lds, ldz, ldc;
  const uint8_t *q, *zero;
  const void *scale;
  const float *bias;
  int M, N, K;
  int group, groups;
  int scale_type;
  int act;
  float alpha;
  int *status;
};

// ---------------------------------------------------------------------------
// tiles: 64 x 64 results a CTA, 32 of K at a time as fp32 in shared memory. 256 threads,
// 4 x 4 results each.
// ---------------------------------------------------------------------------
constexpr int kTile = 64, kTileK = 32, kTilePitch = kTileK + 1;

template <typename X, typename T>
__global__ void __launch_bounds__(256) gemm_w4_tiles_kernel(W4Args p, const X *x, T *C) {
  __shared__ float sx[kTile * kTilePitch], sw[kTile * kTilePitch];
  const int64_t m_tiles = (static_cast<int64_t>(p.M) + kTile - 1) / kTile;
  const int64_t m0 = blockIdx.x % m_tiles * kTile, n0 = blockIdx.x / m_tiles * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += kTileK) {
    for (int i = threadIdx.x; i < kTile * kTileK; i += 256) {
      const int r = i / kTileK, k = k0 + i % kTileK;
      float v = 0.0f, w = 0.0f;
      if (k < p.K && m0 + r < p.M) v = to_float(x[(m0 + r) * p.ldx + k]);
      if (k < p.K && n0 + r < p.N) {
        const int64_t n = n0 + r;
        const int g = k / p.group;
        const int nibble = p.q[n * p.ldq + k / 2] >> (k % 2 * 4) & 15;
        const int zero = p.zero ? p.zero[n * p.ldz + g] & 15 : 8;
        w = load_scale(p.scale, p.scale_type, n * p.lds + g) * static_cast<float>(nibble - zero);
      }
      sx[r * kTilePitch + i % kTileK] = v;
      sw[r * kTilePitch + i % kTileK] = w;
    }
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < kTileK; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = sx[(ty + 16 * i) * kTilePitch + k];
        b[i] = sw[(tx + 16 * i) * kTilePitch + k];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      v[j] = acc[i][j] + (p.bias && n < p.N ? p.bias[n] : 0.0f);
    }
    act_array<T, false>(v, p.act, p.alpha);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (m < p.M && n < p.N) C[m * p.ldc + n] = from_float<T>(v[j]);
    }
  }
}

// ---------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------
// fp16 and bf16 fragments. Two nibbles in the low bits of a 16-bit pair become the
// numbers 1024 + n (fp16) or 128 + n (bf16) by setting the exponent; the subtraction
// of 1024 + zero or 128 + zero is then exact.
struct Half {
  static constexpr uint32_t kBias = 0x64006400u;
  __device__ static uint32_t offset(int zero) {
    return kBias + static_cast<uint32_t>(zero) * 0x00010001u;
  }
  __device__ static uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(reinterpret_cast<const __half2 &>(a), reinterpret_cast<const __half2 &>(b));
    return reinterpret_cast<const uint32_t &>(r);
  }
  __device__ static void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
struct Bfloat {
  static constexpr uint32_t kBias = 0x43004300u;
  __device__ static uint32_t offset(int zero) {
    return kBias + static_cast<uint32_t>(zero) * 0x00010001u;
  }
  __device__ static uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(reinterpret_cast<const __nv_bfloat162 &>(a),
                                     reinterpret_cast<const __nv_bfloat162 &>(b));
    return reinterpret_cast<const uint32_t &>(r);
  }
  __device__ static void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <typename X>
struct RowsType {
  using Frag = Bfloat;
  static constexpr int kParts = 1;
};
template <>
struct RowsType<__half> {
  using Frag = Half;
  static constexpr int kParts = 1;
};
template <>
struct RowsType<float> {
  using Frag = Bfloat;
  static constexpr int kParts = 3;
};

// Eight weights as four pairs (0, 4), (1, 5), (2, 6), (3, 7).
template <typename F>
__device__ __forceinline__ void widen(uint32_t word, uint32_t offset, uint32_t (&pair)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    pair[i] = F::sub((word >> (4 * i) & 0x000f000fu) | F::kBias, offset);
}

// fp32 as three bf16 parts by truncation: 8 bits of the significand each, so the last
// remainder fits. An infinity or NaN is its first part alone.
__device__ __forceinline__ void split3(float x, uint32_t (&part)[3]) {
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

constexpr int kRowsStageK = 256;                    // values of K a warp takes at a time
constexpr int kRowsPitch = kRowsStageK / 2 + 16;    // bytes: 16 lanes' words on 16 banks apart
constexpr int kRowsStageBytes = 16 * kRowsPitch;
constexpr int kRowsDepth = 3;                       // stages in flight and at work
constexpr int kRowsMostWarps = 16;

struct RowsPlan {
  int slices, teams;  // warps that share K, and such teams (16 channels each) in a CTA
  int steps;          // stages of K a warp takes for 16 channels
  int tiles;          // of 16 channels
  int x_units;        // 16-byte units of x in shared memory
  int smem;
};

// A CTA's `teams` teams of `slices` warps take 16 channels each at a time, CTA after CTA
// round the tiles. Warp s of a team takes K from s * steps * 256 on. Lane (g, t) of mma
// m16n8k16 holds channels g and g + 8 and token g: word t of every group of 32 nibbles
// (8 values) gives it the pairs (0, 4), (1, 5) for one mma and (2, 6), (3, 7) for the next,
// with x in shared memory in the same order -- a sum does not mind. Weights go by
// cp.async through a ring of each warp's own, across the ends of tiles.
template <typename X, typename T, int NT, bool kZeros>
__global__ void __launch_bounds__(kRowsMostWarps * 32)
    gemm_w4_rows_kernel(const W4Args p, const X *x, T *C, const RowsPlan plan) {
  using F = typename RowsType<X>::Frag;
  constexpr int P = RowsType<X>::kParts;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warps = plan.slices * plan.teams;
  uint4 *sx = reinterpret_cast<uint4 *>(smem);
  uint8_t *ring = smem + static_cast<size_t>(plan.x_units) * 16 ;
  float *red = reinterpret_cast<float *>(ring + warps * kRowsDepth * kRowsStageBytes);
  griddep_wait();
  griddep_launch_dependents();

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int slice = warp % plan.slices, team = warp / plan.slices;
  const int k_begin = slice * plan.steps * kRowsStageK;
  const int steps = max(0, min(plan.steps, (p.K - k_begin + kRowsStageK - 1) / kRowsStageK));
  const int row_bytes = (p.K + 1) >> 1;
  const int stride = static_cast<int>(gridDim.x) * plan.teams;
  const int tile0 = static_cast<int>(blockIdx.x) * plan.teams + team;
  uint8_t *mine = ring + warp * (kRowsDepth * kRowsStageBytes);

  // rounds of the CTA: the same for all its warps, which meet after each
  const int rounds = (plan.tiles - static_cast<int>(blockIdx.x) * plan.teams + stride - 1) / stride;
  const int total = steps * rounds;
  const auto issue = [&](int i) {
    if (i < total) {
      const int tile = tile0 + i / steps * stride, step = i % steps;
      uint8_t *to = mine + i % kRowsDepth * kRowsStageBytes;
      const int byte0 = (k_begin + step * kRowsStageK) / 2;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = j * 4 + (lane >> 3), piece = lane & 7;
        const int64_t n = min(static_cast<int64_t>(tile) * 16 + r, static_cast<int64_t>(p.N) - 1);
        const int b = byte0 + piece * 16;
        const int valid = max(0, min(16, row_bytes - b));
        const uint8_t *from = p.q + n * p.ldq + (valid ? b : 0);
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(
                         smem_u32(to + r * kRowsPitch + piece * 16)),
                     "l"(from), "r"(valid)
                     : "memory");
      }
    }
    copy_async_commit();
  };
  // scales (and zeros) of a stage's 16 channels, lane l: channel l % 16, groups of half l / 16
  const int per_stage = kRowsStageK / p.group;  // 2, 4 or 8
  const int per_half = per_stage >> 1;
  float sc[4];
  int ze[4];
  const auto fetch_scales = [&](int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sc[j] = 0.0f;
      ze[j] = 8;
    }
    if (i >= total) return;
    const int tile = tile0 + i / steps * stride, step = i % steps;
    const int64_t n = min(static_cast<int64_t>(tile) * 16 + (lane & 15), static_cast<int64_t>(p.N) - 1);
    const int g0 = (k_begin + step * kRowsStageK) / p.group + (lane >> 4) * per_half;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < per_half && g0 + j < p.groups) {
        sc[j] = load_scale(p.scale, p.scale_type, n * p.lds + g0 + j);
        if (kZeros) ze[j] = __ldg(p.zero + n * p.ldz + g0 + j) & 15;
      }
    }
  };

#pragma unroll
  for (int i = 0; i < kRowsDepth - 1; ++i) issue(i);
  fetch_scales(0);

  // x into shared memory, in the fragments' order, zeros behind K
  {
    const int blocks = (p.K + 31) >> 5;
    for (int u = threadIdx.x; u < blocks * p.M * 4; u += blockDim.x) {
      const int kb = u / (p.M * 4), m = u / 4 % p.M, k = kb * 32 + (u & 3) * 8;
      const X *from = x + m * p.ldx + k;
      uint32_t h[P][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (P == 3) {
          uint32_t parts[3];
          split3(k + j < p.K ? from[j] : 0.0f, parts);
          for (int q = 0; q < 3; ++q) h[q][j] = parts[q];
        } else {
          h[0][j] = k + j < p.K ? reinterpret_cast<const uint16_t *>(from)[j] : 0u;
        }
      }
#pragma unroll
      for (int q = 0; q < P; ++q)
        sx[(kb * P + q) * p.M * 4 + m * 4 + (u & 3)] =
            make_uint4(h[q][0] | h[q][4] << 16, h[q][1] | h[q][5] << 16, h[q][2] | h[q][6] << 16,
                       h[q][3] | h[q][7] << 16);
    }
  }
  __syncthreads();

  float acc[NT][4] = {};
  int at = 0;  // stage of this warp's ring
  for (int round = 0; round < rounds; ++round) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[j][r] = 0.0f;
    for (int step = 0; step < steps; ++step, ++at) {
      issue(at + kRowsDepth - 1);
      float scale[4];
      int zero[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        scale[j] = sc[j];
        zero[j] = ze[j];
      }
      fetch_scales(at + 1);
      copy_async_wait<kRowsDepth - 1>();
      __syncwarp();
      const uint8_t *st = mine + at % kRowsDepth * kRowsStageBytes + g * kRowsPitch + t * 4;
      const int kb0 = (k_begin + step * kRowsStageK) >> 5;
      const int kb_most = (p.K + 31) >> 5;
      float part[NT][4];
      uint32_t off0 = 0, off1 = 0;
      float s0 = 0.0f, s1 = 0.0f;
      const int mask = (p.group >> 5) - 1;
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        if ((b & mask) == 0) {
          // group b / (group / 32) of the stage: held by lanes of half (b >= 4)
          const int j = (b & 3) >> (p.group == 32 ? 0 : p.group == 64 ? 1 : 2);
          const float v = j == 0 ? scale[0] : j == 1 ? scale[1] : j == 2 ? scale[2] : scale[3];
          s0 = __shfl_sync(0xffffffffu, v, (b >> 2) * 16 + g);
          s1 = __shfl_sync(0xffffffffu, v, (b >> 2) * 16 + g + 8);
          if (kZeros) {
            const int z = j == 0 ? zero[0] : j == 1 ? zero[1] : j == 2 ? zero[2] : zero[3];
            off0 = F::offset(__shfl_sync(0xffffffffu, z, (b >> 2) * 16 + g));
            off1 = F::offset(__shfl_sync(0xffffffffu, z, (b >> 2) * 16 + g + 8));
          } else {
            off0 = off1 = F::offset(8);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[n][r] = 0.0f;
        }
        if (kb0 + b < kb_most) {
          uint32_t w0[4], w1[4];
          widen<F>(*reinterpret_cast<const uint32_t *>(st + b * 16), off0, w0);
          widen<F>(*reinterpret_cast<const uint32_t *>(st + 8 * kRowsPitch + b * 16), off1, w1);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int q = 0; q < P; ++q) {
              uint4 v = make_uint4(0, 0, 0, 0);
              if (n * 8 + g < p.M) v = sx[((kb0 + b) * P + q) * p.M * 4 + (n * 8 + g) * 4 + t];
              F::mma(part[n], w0[0], w1[0], w0[1], w1[1], v.x, v.y);
              F::mma(part[n], w0[2], w1[2], w0[3], w1[3], v.z, v.w);
            }
          }
        }
        if ((b & mask) == mask) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[n][0] = fmaf(s0, part[n][0], acc[n][0]);
            acc[n][1] = fmaf(s0, part[n][1], acc[n][1]);
            acc[n][2] = fmaf(s1, part[n][2], acc[n][2]);
            acc[n][3] = fmaf(s1, part[n][3], acc[n][3]);
          }
        }
      }
      __syncwarp();  // the stage has been read: the next issue writes over it
    }
    // the team's sums: [buffer][warp][token][channel]
    float *mine_red = red + ((round & 1) * warps + warp) * (NT * 128);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float *r = mine_red + (8 * n + 2 * t) * 16 + g;
      r[0] = acc[n][0];
      r[16] = acc[n][1];
      r[8] = acc[n][2];
      r[24] = acc[n][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < plan.teams * p.M * 16; i += blockDim.x) {
      const int ch = i & 15, m = i / 16 % p.M, tm = i / (16 * p.M);
      const int tile = (static_cast<int>(blockIdx.x) * plan.teams + tm) + round * stride;
      const int64_t n = static_cast<int64_t>(tile) * 16 + ch;
      if (tile >= plan.tiles || n >= p.N) continue;
      const float *from = red + ((round & 1) * warps + tm * plan.slices) * (NT * 128) + m * 16 + ch;
      float v[1] = {0.0f};
      for (int s = 0; s < plan.slices; ++s) v[0] += from[s * (NT * 128)];
      if (p.bias) v[0] += p.bias[n];
      act_array<T, false>(v, p.act, p.alpha);
      C[m * p.ldc + n] = from_float<T>(v[0]);
    }
  }
  copy_async_wait<0>();
}

constexpr int kRowsMostX = 96 * 1024;  // bytes of x in shared memory

template <typename X>
bool rows_fits(const W4Args &p) {
  return p.M <= 16 &&
         ceil_div(p.K, 32) * 64 * p.M * RowsType<X>::kParts <= kRowsMostX &&
         reinterpret_cast<uintptr_t>(p.q) % 16 == 0 && p.ldq % 16 == 0;
}

template <typename X, typename T>
int launch_rows(cudaStream_t s, const W4Args &p, const X *x, T *C) {
  RowsPlan plan;
  const int64_t sms = sm_count(), stages = ceil_div(p.K, kRowsStageK);
  plan.tiles = static_cast<int>(ceil_div(p.N, 16));
  plan.slices = static_cast<int>(std::min<int64_t>(stages, kRowsMostWarps));
  plan.steps = static_cast<int>(ceil_div(stages, plan.slices));
  plan.slices = static_cast<int>(ceil_div(stages, plan.steps));
  plan.teams = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(kRowsMostWarps / plan.slices, plan.tiles / (2 * sms))));
  plan.x_units = static_cast<int>(ceil_div(p.K, 32)) * 4 * p.M * RowsType<X>::kParts;
  const int warps = plan.slices * plan.teams, nt = p.M <= 8 ? 1 : 2;
  plan.smem = plan.x_units * 16 + warps * kRowsDepth * kRowsStageBytes + 2 * warps * nt * 512;
  auto *fn = nt == 1 ? (p.zero ? gemm_w4_rows_kernel<X, T, 1, true> : gemm_w4_rows_kernel<X, T, 1, false>)
                     : (p.zero ? gemm_w4_rows_kernel<X, T, 2, true> : gemm_w4_rows_kernel<X, T, 2, false>);
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(fn), plan.smem);
  if (rc) return rc;
  const int fit = std::max(1, std::min(2048 / (warps * 32), (228 * 1024) / (plan.smem + 1024)));
  const int64_t grid = std::min<int64_t>(ceil_div(plan.tiles, plan.teams), sms * std::min(fit, 2));
  return launch_programmatic(fn, dim3(static_cast<unsigned>(grid)),
                             dim3(static_cast<unsigned>(warps * 32)),
                             static_cast<size_t>(plan.smem), s, p, x, C, plan);
}

template <typename X, typename T>
int run(cudaStream_t s, const W4Args &p, const void *x, void *C) {
  if (rows_fits<X>(p)) return launch_rows(s, p, static_cast<const X *>(x), static_cast<T *>(C));
  const int64_t tiles = ceil_div(p.M, kTile) * ceil_div(p.N, kTile);
  if (tiles >= (int64_t(1) << 31)) return kErrUnsupported;
  gemm_w4_tiles_kernel<X, T><<<static_cast<unsigned>(tiles), 256, 0, s>>>(
      p, static_cast<const X *>(x), static_cast<T *>(C));
  count_launch();
  return launch_result();
}

template <typename X>
int run_to(cudaStream_t s, const W4Args &p, const void *x, void *C, int c_dtype) {
  if (c_dtype == NPLK_DTYPE_FP32) return run<X, float>(s, p, x, C);
  if (c_dtype == NPLK_DTYPE_FP16) return run<X, __half>(s, p, x, C);
  return run<X, __nv_bfloat16>(s, p, x, C);
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_gemm_w4(void *stream, int64_t M, int64_t N, int64_t K, int64_t group,
                            int x_dtype, const void *x, int64_t ldx, const uint8_t *q, int64_t ldq,
                            int scale_dtype, const void *scale, int64_t lds, const uint8_t *zero,
                            int64_t ldz, const float *bias, int act, float act_alpha, int c_dtype,
                            void *C, int64_t ldc, int *status) {
  const int xs = dtype_bytes(x_dtype), ss = dtype_bytes(scale_dtype), cs = dtype_bytes(c_dtype);
  if (M < 1 || N < 1 || K < 1 || group < 1 || !xs || !ss || !cs || !x || !q || !scale || !C ||
      ldx < K || ldq < ceil_div(K, 2) || lds < ceil_div(K, group) ||
      (zero && ldz < ceil_div(K, group)) || ldc < N || act < 0 || act > 10)
    return kErrInvalidArg;
  if (reinterpret_cast<uintptr_t>(x) % xs || reinterpret_cast<uintptr_t>(scale) % ss ||
      reinterpret_cast<uintptr_t>(C) % cs || reinterpret_cast<uintptr_t>(bias) % 4 ||
      reinterpret_cast<uintptr_t>(status) % 4)
    return kErrInvalidArg;
  if (!w4_group_ok(group) || M > (int64_t(1) << 30) || N > (int64_t(1) << 30) ||
      K > (int64_t(1) << 30))
    return kErrUnsupported;
  const W4Args p{ldx, ldq, lds, ldz, ldc, q, zero, scale, bias, static_cast<int>(M),
                 static_cast<int>(N), static_cast<int>(K), static_cast<int>(group),
                 static_cast<int>(ceil_div(K, group)), scale_dtype, act, act_alpha, status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_dtype == NPLK_DTYPE_FP32) return run_to<float>(s, p, x, C, c_dtype);
  if (x_dtype == NPLK_DTYPE_FP16) return run_to<__half>(s, p, x, C, c_dtype);
  return run_to<__nv_bfloat16>(s, p, x, C, c_dtype);
}
