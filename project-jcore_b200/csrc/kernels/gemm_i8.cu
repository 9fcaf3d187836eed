// Matrix product in 8-bit integers with a scale for each token and channel:
//   C[m,n] = act((sum_k A[m,k] B[n,k]) * a_scale[m] * b_scale[n] + bias[n]).
// |A * B| <= 2^14, so 32-bit sums are exact up to K = 131071 in any order, and every
// kernel rounds the same steps: a token's results do not depend on its batch.
//
// Four kernels, by what bounds the product (choose_plan):
//   rows    few tokens: the weights' bytes. Each warp streams 16 channels with
//           plain 16-byte loads into mma.sync fragments, warps share K;
//   split   middle sizes: tcgen05 tiles of 128 channels x MT tokens, K shared
//           by a cluster of up to 8 CTAs that add their sums over distributed
//           shared memory;
//   pair    large sizes: persistent CTA pairs, 256 channels x 256 tokens;
//   bytes   operands that TMA and 16-byte loads cannot read.
// In all tcgen05 tiles the channels are the accumulator's 128 lanes and the
// tokens its columns: a warp then holds 32 consecutive channels of one token,
// which are consecutive in C, so its stores are whole 64- or 128-byte pieces
// without a transpose, and b_scale and bias are one register each.
#include <algorithm>

#include "act_epilogue.cuh"
#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "typed_io.cuh"

namespace nplk {
namespace {

struct I8Args {
  int64_t lda, ldb, ldc;
  const int8_t *A, *B;
  const float *a_scale, *b_scale, *bias;
  int M, N, K;
  int act;
  float alpha;
  uint32_t stall_us;  // fault injection: 0 except on an armed launch (injected_stall)
  int *status;
};

// ---------------------------------------------------------------------------
// bytes: 64 x 64 tiles, 64 bytes of K at a time gathered by bytes into shared
// memory, four products an instruction (dp4a). 256 threads, 4 x 4 results each.
// ---------------------------------------------------------------------------
constexpr int kTile = 64, kPitch = 17;  // words a row: 16, and one against bank conflicts

template <typename T>
__global__ void __launch_bounds__(256) gemm_i8_bytes_kernel(I8Args p, T *C) {
  __shared__ int sa[kTile * kPitch], sb[kTile * kPitch];
  const int64_t m_tiles = (static_cast<int64_t>(p.M) + kTile - 1) / kTile;
  const int64_t m0 = blockIdx.x % m_tiles * kTile, n0 = blockIdx.x / m_tiles * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 64) {
    for (int i = threadIdx.x; i < kTile * 64; i += 256) {
      const int r = i >> 6, k = i & 63;
      const bool in_k = k0 + k < p.K;
      reinterpret_cast<int8_t *>(sa + r * kPitch)[k] =
          in_k && m0 + r < p.M ? p.A[(m0 + r) * p.lda + k0 + k] : int8_t(0);
      reinterpret_cast<int8_t *>(sb + r * kPitch)[k] =
          in_k && n0 + r < p.N ? p.B[(n0 + r) * p.ldb + k0 + k] : int8_t(0);
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      int a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = sa[(ty + 16 * i) * kPitch + w];
        b[i] = sb[(tx + 16 * i) * kPitch + w];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      v[j] = m < p.M && n < p.N ? fmaf(static_cast<float>(acc[i][j]) * p.a_scale[m], p.b_scale[n],
                                       p.bias ? p.bias[n] : 0.0f)
                                : 0.0f;
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
// rows: up to 8 * NT tokens. A CTA takes 16 channels; its 16 warps take every
// 16th 64-byte piece of K. mma.sync m16n8k32 with the channels as its rows:
// lane (g, t) loads the 16 bytes at 64 c + 16 t of channels g and g + 8 and of
// token g, and uses words 0, 1 and then 2, 3 as its two fragments -- K in the
// same other order on both sides, which a sum does not mind. The warps' sums
// meet in shared memory.
// ---------------------------------------------------------------------------
constexpr int kRowsWarps = 16, kRowsUnroll = 4;

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load16(const int8_t *p) {
  return __ldg(reinterpret_cast<const uint4 *>(p));
}

// Weights: each byte is read once, and the bytes after it soon by other warps.
__device__ __forceinline__ uint4 load16_stream(const int8_t *p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// The first `count` (1..15) of 16 bytes, then zeros.
__device__ __forceinline__ uint4 load_bytes(const int8_t *p, int count) {
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; ++i)
    if (i < count) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(p[i])) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int NT, typename T>
__global__ void __launch_bounds__(kRowsWarps * 32) gemm_i8_rows_kernel(I8Args p, T *C) {
  __shared__ int red[kRowsWarps][NT * 8][16];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  // rows past the last are read as the last, their results dropped
  const int8_t *b0 = p.B + (n0 + g < p.N ? n0 + g : p.N - 1) * p.ldb + 16 * t;
  const int8_t *b1 = p.B + (n0 + g + 8 < p.N ? n0 + g + 8 : p.N - 1) * p.ldb + 16 * t;
  const int8_t *a[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
    a[j] = p.A + static_cast<int64_t>(8 * j + g < p.M ? 8 * j + g : p.M - 1) * p.lda + 16 * t;
  int acc[NT][4] = {};
  auto step = [&](const uint4 &x, const uint4 &y, const uint4 (&z)[NT]) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      mma_s8(acc[j], x.x, y.x, x.y, y.y, z[j].x, z[j].y);
      mma_s8(acc[j], x.z, y.z, x.w, y.w, z[j].z, z[j].w);
    }
  };
  const int full = p.K >> 6;
  int c = warp;
  for (; c + (kRowsUnroll - 1) * kRowsWarps < full; c += kRowsUnroll * kRowsWarps) {
    uint4 x[kRowsUnroll], y[kRowsUnroll], z[kRowsUnroll][NT];
#pragma unroll
    for (int u = 0; u < kRowsUnroll; ++u) {
      const int64_t o = static_cast<int64_t>(c + u * kRowsWarps) * 64;
      x[u] = load16_stream(b0 + o);
      y[u] = load16_stream(b1 + o);
#pragma unroll
      for (int j = 0; j < NT; ++j) z[u][j] = load16(a[j] + o);
    }
#pragma unroll
    for (int u = 0; u < kRowsUnroll; ++u) step(x[u], y[u], z[u]);
  }
  for (; c < full; c += kRowsWarps) {
    const int64_t o = static_cast<int64_t>(c) * 64;
    uint4 z[NT];
    const uint4 x = load16(b0 + o), y = load16(b1 + o);
#pragma unroll
    for (int j = 0; j < NT; ++j) z[j] = load16(a[j] + o);
    step(x, y, z);
  }
  if ((p.K & 63) && warp == full % kRowsWarps) {  // the last, shorter piece
    const int64_t o = static_cast<int64_t>(full) * 64;
    const int left = (p.K & 63) - 16 * t;  // bytes of this lane's 16 inside K
    uint4 x = make_uint4(0, 0, 0, 0), y = x, z[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) z[j] = x;
    if (left >= 16) {
      x = load16(b0 + o);
      y = load16(b1 + o);
#pragma unroll
      for (int j = 0; j < NT; ++j) z[j] = load16(a[j] + o);
    } else if (left > 0) {
      x = load_bytes(b0 + o, left);
      y = load_bytes(b1 + o, left);
#pragma unroll
      for (int j = 0; j < NT; ++j) z[j] = load_bytes(a[j] + o, left);
    }
    step(x, y, z);
  }
  // accumulator: channels g, g + 8 (rows), tokens 2t, 2t + 1 (columns)
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    red[warp][8 * j + 2 * t][g] = acc[j][0];
    red[warp][8 * j + 2 * t + 1][g] = acc[j][1];
    red[warp][8 * j + 2 * t][g + 8] = acc[j][2];
    red[warp][8 * j + 2 * t + 1][g + 8] = acc[j][3];
  }
  __syncthreads();
  if (threadIdx.x < NT * 128) {
    const int ch = threadIdx.x & 15, m = threadIdx.x >> 4;
    const int64_t n = n0 + ch;
    if (m < p.M && n < p.N) {
      int s = 0;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) s += red[w][m][ch];
      float v[1] = {fmaf(static_cast<float>(s) * p.a_scale[m], p.b_scale[n],
                         p.bias ? p.bias[n] : 0.0f)};
      act_array<T, false>(v, p.act, p.alpha);
      C[m * p.ldc + n] = from_float<T>(v[0]);
    }
  }
}

// ---------------------------------------------------------------------------
// The tcgen05 kernels' common parts. A stage holds 128 bytes of K of 128
// channels and of the tile's tokens (or this CTA's half of them), as TMA's
// 128-byte swizzle lays them out; one MMA takes 32 bytes of K.
// ---------------------------------------------------------------------------
constexpr int kI8BK = 128, kI8Channels = 128, kI8WeightBytes = kI8Channels * kI8BK;

// Where an epilogue warp takes its results: a 32-token x 32-channel box of C,
// staged in shared memory (2 KB for 16-bit results, 4 KB for fp32) and handed
// to the TMA unit, which clips it at C's edges; or, where C or its pitch is not
// 16-byte aligned, stores of single values. Staging takes the addresses and
// edge checks off the warps: with a store per value an epilogue warp issued
// about 250 instructions a box, and their issue bound the kernels at small K.
template <typename T>
struct I8Out {
  const CUtensorMap *map;  // null: stores of single values
  uint8_t *box;
  T *C;
};

// One warp's box: TMEM columns t_cols.. (tokens m0..) of its 32 lanes (channels
// n0..). `scales`: the tokens' a_scale, in shared memory. b_scale and bias of
// the lane's channels: sb, bias [k] of channel n0 + lane / 4 + 8 k in the mma
// layout (16-bit box), [0] of channel n0 + lane otherwise. `release` runs once
// the columns have been read.
template <typename T, typename Release>
__device__ __forceinline__ void i8_finish_box(const I8Args &p, const I8Out<T> &out,
                                              uint32_t t_cols, int m0, int n0,
                                              const float (&sb)[4], const float (&bias)[4],
                                              const float *scales, Release release) {
  const int lane = threadIdx.x & 31;
  const bool staged = sizeof(T) == 2 && out.map;
  if constexpr (sizeof(T) == 2) {
    if (staged) {
      // mma layout: packed pairs of tokens go to shared memory transposed
      uint32_t r[2][16];
      tmem_ld_frag32(t_cols, r[0]);
      tmem_ld_frag32(t_cols + (16u << 16), r[1]);
      tmem_wait_ld16x2(r[0], r[1]);
      release();
      if (m0 >= p.M) return;
      float v[32];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 s = *reinterpret_cast<const float2 *>(scales + 8 * i + 2 * (lane & 3));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t *q = &r[k >> 1][4 * i + 2 * (k & 1)];
          const float2 x = make_float2(static_cast<float>(static_cast<int>(q[0])),
                                       static_cast<float>(static_cast<int>(q[1])));
          const float2 y = fma2(mul2(x, s), both(sb[k]), both(bias[k]));
          v[8 * i + 2 * k] = y.x;
          v[8 * i + 2 * k + 1] = y.y;
        }
      }
      act_array<T, false>(v, p.act, p.alpha);
      if (lane == 0) bulk_wait_group_read<0>();  // the previous box has been read
      __syncwarp();
      // lane l addresses row l % 8 of matrix l / 8: token 8 (i + matrix / 2) + row,
      // 16-byte piece 2 h + matrix % 2, swizzled as the map's 64-byte swizzle
      const uint32_t base = smem_u32(out.box);
      const uint32_t row = 8u * (lane >> 4) + (lane & 7), piece = (lane >> 3) & 1u;
#pragma unroll
      for (int i = 0; i < 4; i += 2)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t token = 8u * i + row;
          const uint32_t at = base + token * 64u + (((2u * h + piece) ^ ((token >> 1) & 3u)) << 4);
          stmatrix_x4_trans(at, pack2<T>(v[8 * i + 4 * h], v[8 * i + 4 * h + 1]),
                            pack2<T>(v[8 * i + 4 * h + 2], v[8 * i + 4 * h + 3]),
                            pack2<T>(v[8 * i + 8 + 4 * h], v[8 * i + 8 + 4 * h + 1]),
                            pack2<T>(v[8 * i + 8 + 4 * h + 2], v[8 * i + 8 + 4 * h + 3]));
        }
    }
  }
  if (!staged) {
    uint32_t r[32];
    tmem_ld32(t_cols, r);
    tmem_wait_ld(r);
    release();
    if (m0 >= p.M) return;
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const float2 x = make_float2(static_cast<float>(static_cast<int>(r[j])),
                                   static_cast<float>(static_cast<int>(r[j + 1])));
      const float2 y = fma2(mul2(x, *reinterpret_cast<const float2 *>(scales + j)),
                            make_float2(sb[0], sb[0]), make_float2(bias[0], bias[0]));
      v[j] = y.x;
      v[j + 1] = y.y;
    }
    act_array<T, false>(v, p.act, p.alpha);
    if (!out.map) {
      const int64_t n = static_cast<int64_t>(n0) + lane;
      const int rows = p.M - m0;
      T *c = out.C + static_cast<int64_t>(m0) * p.ldc + n;
      if (n >= p.N) return;
      if (rows >= 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) c[j * p.ldc] = from_float<T>(v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < rows) c[j * p.ldc] = from_float<T>(v[j]);
      }
      return;
    }
    if (lane == 0) bulk_wait_group_read<0>();
    __syncwarp();
    float *box = reinterpret_cast<float *>(out.box);
#pragma unroll
    for (int j = 0; j < 32; ++j) box[32 * j + lane] = v[j];
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (n0 < p.N) tma_store_2d(out.map, out.box, n0, m0);
    bulk_commit_group();
  }
}

// b_scale and bias of a lane's channels as i8_finish_box takes them.
template <typename T>
__device__ __forceinline__ void i8_channel_scales(const I8Args &p, bool boxes, int n0,
                                                  float (&sb)[4], float (&bias)[4]) {
  const int lane = threadIdx.x & 31;
  const bool frag = sizeof(T) == 2 && boxes;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t n = static_cast<int64_t>(n0) + (frag ? (lane >> 2) + 8 * k : lane);
    const bool in = n < p.N && (frag || k == 0);
    sb[k] = in ? p.b_scale[n] : 0.0f;
    bias[k] = in && p.bias ? p.bias[n] : 0.0f;
  }
}

// ---------------------------------------------------------------------------
// split: one 128-channel x MT-token tile per cluster of S CTAs, CTA r taking
// its share of the K blocks. TMA producer, MMA issuer, 8 epilogue warps
// (two per lane quadrant, every second 32 tokens each: one warp per scheduler
// alone would wait out every latency of the epilogue; 16 warps took 1 us more a
// launch, since two CTAs of successive launches no longer fit one SM). With S > 1
// each CTA lays its partial sums in its own shared memory ([token][channel], over
// the stages, which are read out by then), and CTA r adds tokens
// [r MT / S, (r + 1) MT / S) of all S CTAs.
// TMEM: a CTA of a cluster must not wait for columns that another cluster holds.
// With S > 1, MT is at most 128, and those that shared memory and threads let onto
// an SM together (3 x 128, or 6 smaller) ask for at most 384 of its 512 columns; the
// kernels of CTA pairs, which take all 512, leave too little shared memory for one
// (kTmemClusterSmem); CTAs without a cluster give theirs back by themselves.
// ---------------------------------------------------------------------------
constexpr int kSplitEpiWarps = 8;
constexpr int kSplitThreads = 64 + kSplitEpiWarps * 32;

template <int MT>
struct SplitTraits {
  static constexpr int kStageBytes = kI8WeightBytes + MT * kI8BK;
  static constexpr int kMostStages = MT >= 256 ? 4 : MT >= 128 ? 6 : MT >= 64 ? 8 : 10;
  static constexpr int kTmemCols = MT;
  static constexpr int kPartialBytes = MT * kI8Channels * 4;  // over the stages
  // Shared memory after the stages: barriers, then the epilogue warps' scales.
  static constexpr int kTailBytes = 256 + MT * 4;
  static constexpr int kBoxBytes = kSplitEpiWarps * 4096;  // over the stages
  static constexpr int smem_bytes(int stages, bool partials) {
    const int area = stages * kStageBytes;
    const int least = partials && kPartialBytes > kBoxBytes ? kPartialBytes : kBoxBytes;
    return 1024 + (area < least ? least : area) + kTailBytes;
  }
  static_assert(1024 + kBoxBytes + kTailBytes >= kTmemClusterSmem, "no CTA pair beside a cluster");
  static_assert(1024 + kMostStages * kStageBytes + kTailBytes <= 232448, "shared memory budget");
};

// This CTA's share of the cluster's tokens: the sums of all S CTAs' partial
// sums, a token per warp at a time, four channels per lane.
template <int MT, int S, typename T>
__device__ __forceinline__ void i8_add_slices(const I8Args &p, const uint8_t *part, int rank,
                                              int n0, int m0, T *C) {
  constexpr int kPer = MT / S, kEach = kPer / kSplitEpiWarps,
                kBatch = kEach < 1 ? 1 : kEach < 4 ? kEach : 4;
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) - 2;
  const int64_t n = static_cast<int64_t>(n0) + 4 * lane;
  float sb[4], bias[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sb[j] = n + j < p.N ? p.b_scale[n + j] : 0.0f;
    bias[j] = p.bias && n + j < p.N ? p.bias[n + j] : 0.0f;
  }
  const bool whole = n + 4 <= p.N && p.ldc % 4 == 0 &&
                     reinterpret_cast<uintptr_t>(C) % (4 * sizeof(T)) == 0;
#pragma unroll 1
  for (int i = w * kBatch; i < kPer; i += kSplitEpiWarps * kBatch) {
    const int tok = rank * kPer + i;
    const int here = min(kBatch, p.M - m0 - tok);  // of the batch; the others lie past M
    if (here <= 0) break;
    // All loads first: a round trip to another SM each. None that no sum below waits for:
    // it could still be under way when that SM's CTA ends.
    uint4 v[kBatch][S];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (b < here)
#pragma unroll
        for (int r = 0; r < S; ++r)
          v[b][r] = ld_shared_cluster_v4(mapa_shared(
              smem_u32(part) + static_cast<uint32_t>((tok + b) * kI8Channels + 4 * lane) * 4u,
              static_cast<uint32_t>(r)));
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t m = static_cast<int64_t>(m0) + tok + b;
      if (b >= here) break;
      int s[4] = {};
#pragma unroll
      for (int r = 0; r < S; ++r) {
        s[0] += static_cast<int>(v[b][r].x);
        s[1] += static_cast<int>(v[b][r].y);
        s[2] += static_cast<int>(v[b][r].z);
        s[3] += static_cast<int>(v[b][r].w);
      }
      const float sa = p.a_scale[m];
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf(static_cast<float>(s[j]) * sa, sb[j], bias[j]);
      act_array<T, false>(o, p.act, p.alpha);
      T *c = C + m * p.ldc + n;
      if (whole) {
        store_pack(c, pack<T, 4>(o));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) c[j] = from_float<T>(o[j]);
      }
    }
  }
}

template <int MT, typename T>
__global__ void __launch_bounds__(kSplitThreads, 2)
    gemm_i8_split_kernel(const __grid_constant__ CUtensorMap map_w,
                         const __grid_constant__ CUtensorMap map_x,
                         const __grid_constant__ CUtensorMap map_c, const I8Args p, T *C,
                         int boxes, int slices, int n_tiles, int stages, int area) {
  using S = SplitTraits<MT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = align_smem_1024(smem_raw);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + area);
  uint64_t *empty = full + S::kMostStages;
  uint64_t *acc_full = empty + S::kMostStages;
  uint64_t *never = acc_full + 1;  // never arrived on (injected_stall)
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(never + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  float *scales = reinterpret_cast<float *>(smem + area + 256);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % slices;
  const int tile = static_cast<int>(blockIdx.x) / slices;
  const int n0 = tile % n_tiles * kI8Channels, m0 = tile / n_tiles * MT;
  const int blocks = (p.K + kI8BK - 1) / kI8BK;
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * blocks / slices);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * blocks / slices);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(never, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  bool have = false;  // epilogue threads: the accumulator is complete
  const int quad = warp & 3;
  const int ch = quad * 32 + lane;
  const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, pending = 0, pending_phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer))
          break;
        uint8_t *st = smem + stage * S::kStageBytes;
        mbar_arrive_expect_tx(&full[stage], S::kStageBytes);
        tma_load_2d(&map_w, &full[stage], st, kb * kI8BK, n0);
        tma_load_2d(&map_x, &full[stage], st + kI8WeightBytes, kb * kI8BK, m0);
        pending |= 1u << stage;
        pending_phase = (pending_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // the last copy into each stage lands before the CTA can exit
      for (int s = 0; s < stages; ++s)
        if ((pending >> s) & 1u) mbar_drain(&full[s], (pending_phase >> s) & 1u);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_s8(kI8Channels, MT);
      int stage = 0;
      uint32_t phase = 0;
      bool go = injected_stall(never, p.stall_us, abort_flag, p.status);
      for (int kb = kb0; go && kb < kb1; ++kb) {
        go = mbar_wait(&full[stage], phase, abort_flag, p.status, kStatusTimeoutMma);
        if (!go) break;
        tc_fence_after_sync();
        const uint32_t st = smem_u32(smem + stage * S::kStageBytes);
        const uint64_t w = umma_desc_sw128(st), x = umma_desc_sw128(st + kI8WeightBytes);
#pragma unroll
        for (int kk = 0; kk < kI8BK / 32; ++kk)
          mma_i8_ss(tmem_base, w + 2 * kk, x + 2 * kk, idesc, kb > kb0 || kk > 0 ? 1u : 0u);
        mma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (go) mma_commit(acc_full);
    }
    __syncwarp();
  } else {
    const int c_first = (warp - 2) / 4 * 32;
    float sb[4], bias[4];
    if (slices == 1) {
      i8_channel_scales<T>(p, boxes, n0 + quad * 32, sb, bias);
      for (int i = threadIdx.x - 64; i < MT; i += kSplitEpiWarps * 32)
        scales[i] = m0 + i < p.M ? p.a_scale[m0 + i] : 0.0f;
      asm volatile("bar.sync 1, %0;" ::"n"(kSplitEpiWarps * 32) : "memory");  // epilogue warps
    }
    // by the whole warp or not at all: TMEM loads are for whole warps
    have = __all_sync(0xffffffffu, mbar_wait(acc_full, 0u, abort_flag, p.status,
                                             kStatusTimeoutEpilogue));
    tc_fence_after_sync();
    if (have && slices == 1) {
      // boxes over the stages, which the MMAs have read out
      const I8Out<T> out{boxes ? &map_c : nullptr, smem + (warp - 2) * 4096, C};
#pragma unroll 1
      for (int c0 = c_first; c0 < MT && m0 + c0 < p.M; c0 += kSplitEpiWarps * 8)
        i8_finish_box<T>(p, out, t_row + c0, m0 + c0, n0 + quad * 32, sb, bias, scales + c0, [] {});
      if (boxes && lane == 0) bulk_wait_group_read<0>();  // the boxes outlive their stores
      __syncwarp();
    } else if (have) {
      int *part = reinterpret_cast<int *>(smem);
#pragma unroll 1
      for (int c0 = c_first; c0 < MT; c0 += kSplitEpiWarps * 8) {
        uint32_t acc[32];
        tmem_ld32(t_row + c0, acc);
        tmem_wait_ld(acc);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          part[(c0 + j) * kI8Channels + ch] = static_cast<int>(acc[j]);
      }
    }
    tc_fence_before_sync();
  }
  if (slices > 1) {
    cluster_sync();  // every CTA's partial sums are in its shared memory
    if (warp >= 2 && have) {
      if (slices == 2) i8_add_slices<MT, 2, T>(p, smem, rank, n0, m0, C);
      else if (slices == 4) i8_add_slices<MT, 4, T>(p, smem, rank, n0, m0, C);
      else i8_add_slices<MT, 8, T>(p, smem, rank, n0, m0, C);
    }
    __syncwarp();
    // No CTA leaves while another reads its shared memory. Ordering: the relaxed form
    // says nothing of loads issued before it. Its release waits for the stores of C too,
    // 0.2 to 0.5 us; arriving before those stores is no better in sum (333 x 1000 x 1280
    // fp32 5.6 us against 5.4, 256 x 4096 x 4096 10.4 against 10.1, 77 x 1280 x 1024 4.9
    // against 5.3).
    cluster_sync();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// pair: persistent clusters of two CTAs (tcgen05 cta_group::2), tiles of 256
// channels x 256 tokens. Each CTA loads its 128 channels and 128 of the tokens
// (32 KB a stage), so a K block's bytes serve twice the products of a one-SM
// 128 x 256 tile's. Two accumulators of 256 columns: the epilogue of one tile
// runs under the next tile's MMAs. 8 epilogue warps, two per lane quadrant.
//   full (leader)       the leader's expect_tx for both CTAs' copies
//   empty, acc_full     in each CTA, by the leader's commit to both
//   acc_empty (leader)  16 arrivals: the 8 epilogue warps of each CTA
// ---------------------------------------------------------------------------
constexpr int kPairTokens = 256, kPairEpiWarps = 8;
constexpr int kPairSpan = kPairTokens / (kPairEpiWarps / 4);  // tokens of an epilogue warp
constexpr int kPairStage = kI8WeightBytes + kPairTokens / 2 * kI8BK;
constexpr int kPairThreads = 64 + kPairEpiWarps * 32;
// After the stages: the epilogue warps' boxes and scales, the barriers.
template <typename T>
struct PairTraits {
  static constexpr int kStages = sizeof(T) == 2 ? 6 : 5;
  static constexpr int kBox = 32 * 32 * static_cast<int>(sizeof(T));
  static constexpr int kScaleBytes = kPairEpiWarps * kPairSpan * 4;
  static constexpr int kSmemBytes =
      1024 + kStages * kPairStage + kPairEpiWarps * kBox + kScaleBytes + 256;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
  static_assert(tmem_excludes_clusters(kSmemBytes), "no other cluster's TMEM beside a pair");
};

// Tile order: groups of 8 channel tiles sweep all token tiles, so that the
// pairs at work at one time share operand rows in L2.
struct PairOrder {
  int tiles, full_tiles;  // all; those of the groups of 8
  FastDiv per_group;      // 8 * token tiles
  FastDiv rest;           // channel tiles of the last, smaller group
};

PairOrder pair_order(int n_tiles, int m_tiles) {
  PairOrder o;
  o.tiles = n_tiles * m_tiles;
  o.full_tiles = n_tiles / 8 * 8 * m_tiles;
  o.per_group = make_fastdiv(static_cast<uint32_t>(8 * m_tiles));
  o.rest = make_fastdiv(static_cast<uint32_t>(n_tiles % 8 ? n_tiles % 8 : 1));
  return o;
}

__device__ __forceinline__ void pair_tile(const PairOrder &o, int tile, int &nt, int &mt) {
  const uint32_t group = fdiv(static_cast<uint32_t>(tile), o.per_group);
  const uint32_t local = static_cast<uint32_t>(tile) - group * o.per_group.d;
  const uint32_t m = tile < o.full_tiles ? local >> 3 : fdiv(local, o.rest);
  mt = static_cast<int>(m);
  nt = static_cast<int>(8 * group + local - m * (tile < o.full_tiles ? 8u : o.rest.d));
}

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
    gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap map_w,
                        const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_c, const I8Args p, T *C,
                        int boxes, const PairOrder order) {
  using Tr = PairTraits<T>;
  constexpr int kPairStages = Tr::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = align_smem_1024(smem_raw);
  uint8_t *box_area = smem + kPairStages * kPairStage;
  float *scales = reinterpret_cast<float *>(box_area + kPairEpiWarps * Tr::kBox);
  uint64_t *full = reinterpret_cast<uint64_t *>(scales + kPairEpiWarps * kPairSpan);
  uint64_t *empty = full + kPairStages;
  uint64_t *acc_full = empty + kPairStages;
  uint64_t *acc_empty = acc_full + 2;
  uint64_t *never = acc_empty + 2;  // never arrived on (injected_stall)
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(never + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t peer_abort = mapa_shared(smem_u32(const_cast<int *>(abort_flag)), rank ^ 1u);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kPairEpiWarps);
    }
    mbar_init(never, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before any remote arrival
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  const int tiles = order.tiles;
  const int pairs = static_cast<int>(gridDim.x >> 1), pair = static_cast<int>(blockIdx.x >> 1);
  const int blocks = (p.K + kI8BK - 1) / kI8BK;

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, issued_phase = 0;
      bool aborted = false;
      for (int tile = pair; tile < tiles && !aborted; tile += pairs) {
        int nt, mt;
        pair_tile(order, tile, nt, mt);
        const int row_w = nt * 2 * kI8Channels + static_cast<int>(rank) * kI8Channels;
        const int row_x = mt * kPairTokens + static_cast<int>(rank) * (kPairTokens / 2);
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait_pair_async(&empty[stage], phase ^ 1u, abort_flag, peer_abort, p.status,
                              kStatusTimeoutProducer)) {
            aborted = true;
            break;
          }
          uint8_t *st = smem + stage * kPairStage;
          const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0u);
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * kPairStage);
          tma_load_2d_pair(&map_w, bar, st, kb * kI8BK, row_w);
          tma_load_2d_pair(&map_x, bar, st + kI8WeightBytes, kb * kI8BK, row_x);
          issued |= 1u << stage;
          issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
          if (++stage == kPairStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // the MMAs' last commits have arrived here too, in both CTAs
      for (int s = 0; s < kPairStages && !aborted; ++s)
        if ((issued >> s) & 1u)
          aborted = !mbar_wait_pair_async(&empty[s], (issued_phase >> s) & 1u, abort_flag,
                                          peer_abort, p.status, kStatusTimeoutProducer);
      if (rank == 0) {
        // both CTAs' copies complete on the leader's barriers: every issued
        // phase lands before the pair can exit
        for (int s = 0; s < kPairStages; ++s)
          if ((issued >> s) & 1u) mbar_drain(&full[s], (issued_phase >> s) & 1u);
      } else if (aborted && issued) {
        // this CTA cannot observe its own copies: give those in flight time to land
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader) ----------------
    if (rank == 0 && lane == 0) {
      const uint32_t idesc = umma_idesc_s8(2 * kI8Channels, kPairTokens);
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool go = injected_stall(never, p.stall_us, abort_flag, p.status);
      if (!go) pair_raise_abort(peer_abort);
      for (int tile = pair; go && tile < tiles; tile += pairs, ++local) {
        const int acc = local & 1;
        go = mbar_wait_pair_async(&acc_empty[acc], ((local >> 1) & 1) ^ 1u, abort_flag, peer_abort,
                            p.status, kStatusTimeoutAccFree);
        if (!go) break;
        tc_fence_after_sync();
        const uint32_t d = tmem_base + acc * kPairTokens;
        for (int kb = 0; kb < blocks; ++kb) {
          go = mbar_wait_pair_async(&full[stage], phase, abort_flag, peer_abort, p.status,
                              kStatusTimeoutMma);
          if (!go) break;
          tc_fence_after_sync();
          const uint32_t st = smem_u32(smem + stage * kPairStage);
          const uint64_t w = umma_desc_sw128(st), x = umma_desc_sw128(st + kI8WeightBytes);
#pragma unroll
          for (int kk = 0; kk < kI8BK / 32; ++kk)
            mma_i8_ss_pair(d, w + 2 * kk, x + 2 * kk, idesc, kb > 0 || kk > 0 ? 1u : 0u);
          mma_commit_pair_both(&empty[stage]);
          if (++stage == kPairStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (go) mma_commit_pair_both(&acc_full[acc]);
      }
    }
  } else {
    // ---------------- epilogue: the two warps of a lane quadrant share the tokens ----------------
    const int quad = warp & 3, part = (warp - 2) >> 2;
    float *mine = scales + (warp - 2) * kPairSpan;
    const I8Out<T> out{boxes ? &map_c : nullptr, box_area + (warp - 2) * Tr::kBox, C};
    int local = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++local) {
      int nt, mt;
      pair_tile(order, tile, nt, mt);
      const int n0 = nt * 2 * kI8Channels + static_cast<int>(rank) * kI8Channels + quad * 32;
      const int acc = local & 1, m0 = mt * kPairTokens + part * kPairSpan;
      float sb[4], bias[4];
      i8_channel_scales<T>(p, boxes, n0, sb, bias);
      __syncwarp();  // the previous tile's scales have been read
#pragma unroll
      for (int i = 0; i < kPairSpan; i += 32)
        mine[i + lane] = m0 + i + lane < p.M ? p.a_scale[m0 + i + lane] : 0.0f;
      __syncwarp();
      // by the whole warp or not at all: TMEM loads are for whole warps
      if (!__all_sync(0xffffffffu,
                      mbar_wait_pair_async(&acc_full[acc], (local >> 1) & 1, abort_flag,
                                           peer_abort, p.status, kStatusTimeoutEpilogue)))
        break;
      tc_fence_after_sync();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                             static_cast<uint32_t>(acc * kPairTokens + part * kPairSpan);
#pragma unroll 1
      for (int c0 = 0; c0 < kPairSpan; c0 += 32)
        i8_finish_box<T>(p, out, t_row + c0, m0 + c0, n0, sb, bias, mine + c0, [&] {
          if (c0 + 32 == kPairSpan) {  // the accumulator has been read: hand it back
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_tmem_read(mapa_shared(smem_u32(&acc_empty[acc]), 0u));
          }
        });
    }
    if (boxes && lane == 0) bulk_wait_group_read<0>();  // the boxes outlive their stores
  }
  __syncthreads();
  cluster_sync();  // no remote arrival, copy or MMA into either CTA is left
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------
// Choice and launch
// ---------------------------------------------------------------------------
enum class I8Kernel { kBytes, kRows, kSplit, kPair };

struct I8Plan {
  I8Kernel kernel;
  int mt, slices;
};

template <int MT>
constexpr int split_smem(int stages, bool partials) {
  return SplitTraits<MT>::smem_bytes(stages, partials);
}

int split_smem(int mt, int stages, bool partials) {
  return mt == 32    ? split_smem<32>(stages, partials)
         : mt == 64  ? split_smem<64>(stages, partials)
         : mt == 128 ? split_smem<128>(stages, partials)
                     : split_smem<256>(stages, partials);
}

int split_stages(int mt, int64_t blocks) {
  const int most = mt >= 256 ? SplitTraits<256>::kMostStages
                   : mt >= 128 ? SplitTraits<128>::kMostStages
                   : mt >= 64  ? SplitTraits<64>::kMostStages
                               : SplitTraits<32>::kMostStages;
  return static_cast<int>(std::min<int64_t>(blocks, most));
}

// The rows kernel up to 8 tokens, and up to 16 while all its CTAs (two per SM)
// are at work at once: 16 tokens, N = K = 4096: 6.2 us against 7.0 (split); N =
// 11008: 13.4 against 11.2. Otherwise the tile and K split of least estimated
// time. The estimates (microseconds on 148 SMs) are a fit to 777 timings of 114
// sizes, 1 to 8192 tokens, 45 to 16384 channels, K from 67 to 16384 (rms error
// 17%); the choice they make took 2% longer than the best one on average and
// 34% at worst (77 x 1280 x 1024: 5.0 us against 3.8). The clusters' last barrier has
// become up to 0.5 us longer since the fit.
//   split: waves * (start and end + K blocks * (latency or the bytes that the
//          CTAs of an SM share) + results) + adding the slices
//   pair:  start + rounds * max(K blocks, epilogue) + the shorter of the two
I8Plan choose_plan(int64_t M, int64_t N, int64_t K, bool aligned) {
  if (!aligned) return {I8Kernel::kBytes, 0, 0};
  const int64_t sms = sm_count(), blocks = ceil_div(K, kI8BK);
  if (M <= 8 || (M <= 16 && ceil_div(N, 16) <= 2 * sms)) return {I8Kernel::kRows, 0, 0};
  const double main_us = 0.31 * static_cast<double>(blocks), end_us = 3.3;
  const int64_t rounds = ceil_div(ceil_div(N, 256) * ceil_div(M, kPairTokens), sms / 2);
  I8Plan best{I8Kernel::kPair, 0, 0};
  double least = 1.1 + static_cast<double>(rounds) * std::max(main_us, end_us) +
                 std::min(main_us, end_us);
  for (int mt : {32, 64, 128, 256}) {
    for (int s : {1, 2, 4, 8}) {
      if (s > blocks || (mt == 256 && s > 1)) continue;
      const int64_t each = ceil_div(blocks, s);
      const int64_t ctas = ceil_div(N, kI8Channels) * ceil_div(M, mt) * s;
      const int smem = split_smem(mt, split_stages(mt, each), s > 1) + 1024;
      const int fit = 2 * smem <= 228 * 1024 ? 2 : 1;
      const double per_sm = static_cast<double>(ctas) / static_cast<double>(sms);
      const double share = std::min<double>(fit, std::max(1.0, per_sm));
      const double block_us = std::max(0.25, share * (kI8Channels + mt) * kI8BK * 9.2e-6);
      const double us = static_cast<double>(ceil_div(ctas, sms * fit)) *
                            (2.6 + static_cast<double>(each) * block_us + 0.0096 * mt * share) +
                        (s > 1 ? 0.1 + 0.015 * mt : 0.0);
      if (us < least) {
        least = us;
        best = {I8Kernel::kSplit, mt, s};
      }
    }
  }
  return best;
}

// Launch attributes: programmatic serialization, and clusters of `cluster` CTAs.
void set_launch(cudaLaunchConfig_t &cfg, cudaLaunchAttribute (&attr)[2], cudaStream_t s,
                unsigned cluster) {
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cfg.stream = s;
}

// Whether the TMA unit can store into C.
template <typename T>
bool i8_boxes(const I8Args &p, const T *C) {
  return reinterpret_cast<uintptr_t>(C) % 16 == 0 && p.ldc * sizeof(T) % 16 == 0;
}

template <int MT, typename T>
int launch_split(cudaStream_t s, const I8Args &p, T *C, int slices) {
  using Tr = SplitTraits<MT>;
  CUtensorMap mw, mx, mc = {};
  int rc = encode_tmap_2d_u8_sw128(&mw, p.B, p.K, p.N, p.ldb, kI8Channels);
  if (rc) return rc;
  rc = encode_tmap_2d_u8_sw128(&mx, p.A, p.K, p.M, p.lda, MT);
  if (rc) return rc;
  const bool boxes = slices == 1 && i8_boxes(p, C);
  if (boxes) rc = encode_tmap_2d_box32(&mc, C, p.N, p.M, p.ldc * sizeof(T), sizeof(T));
  if (rc) return rc;
  auto *fn = gemm_i8_split_kernel<MT, T>;
  // As many stages as a CTA has K blocks, up to the limit: with a short K
  // several CTAs share an SM, and one's loads run under another's stores.
  const int stages = split_stages(MT, ceil_div(ceil_div(p.K, kI8BK), slices));
  const int smem = Tr::smem_bytes(stages, slices > 1);
  rc = ensure_dynamic_smem(reinterpret_cast<const void *>(fn), smem);
  if (rc) return rc;
  const int n_tiles = static_cast<int>(ceil_div(p.N, kI8Channels));
  const int64_t ctas = static_cast<int64_t>(n_tiles) * ceil_div(p.M, MT) * slices;
  if (ctas >= (int64_t(1) << 31)) return kErrUnsupported;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = smem;
  set_launch(cfg, attr, s, static_cast<unsigned>(slices));
  count_launch();
  return map_cuda_error(cudaLaunchKernelEx(&cfg, fn, mw, mx, mc, p, C, boxes ? 1 : 0, slices,
                                           n_tiles, stages, smem - 1024 - Tr::kTailBytes));
}

template <typename T>
int launch_pair(cudaStream_t s, const I8Args &p, T *C) {
  CUtensorMap mw, mx, mc = {};
  int rc = encode_tmap_2d_u8_sw128(&mw, p.B, p.K, p.N, p.ldb, kI8Channels);
  if (rc) return rc;
  rc = encode_tmap_2d_u8_sw128(&mx, p.A, p.K, p.M, p.lda, kPairTokens / 2);
  if (rc) return rc;
  const bool boxes = i8_boxes(p, C);
  if (boxes) rc = encode_tmap_2d_box32(&mc, C, p.N, p.M, p.ldc * sizeof(T), sizeof(T));
  if (rc) return rc;
  auto *fn = gemm_i8_pair_kernel<T>;
  rc = ensure_dynamic_smem(reinterpret_cast<const void *>(fn), PairTraits<T>::kSmemBytes);
  if (rc) return rc;
  const int64_t n_tiles = ceil_div(p.N, 2 * kI8Channels), m_tiles = ceil_div(p.M, kPairTokens);
  if (n_tiles * m_tiles >= (int64_t(1) << 27)) return kErrUnsupported;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = PairTraits<T>::kSmemBytes;
  set_launch(cfg, attr, s, 2);
  // A grid beyond the pairs that fit at once would still be right (no pair
  // waits for another); all of them at once is what the tile order counts on.
  const int64_t fit = sm_count() / 2;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<int64_t>(n_tiles * m_tiles, fit)));
  count_launch();
  return map_cuda_error(cudaLaunchKernelEx(&cfg, fn, mw, mx, mc, p, C, boxes ? 1 : 0,
                                           pair_order(static_cast<int>(n_tiles),
                                                      static_cast<int>(m_tiles))));
}

template <typename T>
int run(cudaStream_t s, I8Args p, T *C, const I8Plan &plan) {
  if (plan.kernel == I8Kernel::kBytes) {
    const int64_t tiles = ceil_div(p.M, kTile) * ceil_div(p.N, kTile);
    if (tiles >= (int64_t(1) << 31)) return kErrUnsupported;
    gemm_i8_bytes_kernel<T><<<static_cast<unsigned>(tiles), 256, 0, s>>>(p, C);
    count_launch();
    return launch_result();
  }
  if (plan.kernel == I8Kernel::kRows) {
    const dim3 grid(static_cast<unsigned>(ceil_div(p.N, 16))), block(kRowsWarps * 32);
    return p.M <= 8 ? launch_programmatic(gemm_i8_rows_kernel<1, T>, grid, block, 0, s, p, C)
                    : launch_programmatic(gemm_i8_rows_kernel<2, T>, grid, block, 0, s, p, C);
  }
  if (!p.status) p.status = device_status_word();
  if (!p.status) return kErrInternal;
  p.stall_us = take_armed_stall(NPLK_DEBUG_GEMM);
  if (plan.kernel == I8Kernel::kPair) return launch_pair<T>(s, p, C);
  switch (plan.mt) {
    case 32:
      return launch_split<32, T>(s, p, C, plan.slices);
    case 64:
      return launch_split<64, T>(s, p, C, plan.slices);
    case 128:
      return launch_split<128, T>(s, p, C, plan.slices);
    default:
      return launch_split<256, T>(s, p, C, plan.slices);
  }
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_gemm_i8(void *stream, int64_t M, int64_t N, int64_t K, const int8_t *A,
                            int64_t lda, const float *a_scale, const int8_t *B, int64_t ldb,
                            const float *b_scale, const float *bias, int act, float act_alpha,
                            int c_dtype, void *C, int64_t ldc, int *status) {
  const int size = dtype_bytes(c_dtype);
  if (M < 1 || N < 1 || K < 1 || !A || !B || !a_scale || !b_scale || !C || !size || lda < K ||
      ldb < K || ldc < N || act < 0 || act > 10)
    return kErrInvalidArg;
  if (reinterpret_cast<uintptr_t>(C) % size) return kErrInvalidArg;
  for (const void *v : {static_cast<const void *>(a_scale), static_cast<const void *>(b_scale),
                        static_cast<const void *>(bias), static_cast<const void *>(status)})
    if (reinterpret_cast<uintptr_t>(v) % 4) return kErrInvalidArg;
  if (M > (int64_t(1) << 30) || N > (int64_t(1) << 30) || K > 131071) return kErrUnsupported;
  const bool aligned = reinterpret_cast<uintptr_t>(A) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(B) % 16 == 0 && lda % 16 == 0 &&
                       ldb % 16 == 0;
  const I8Args p{lda, ldb, ldc, A, B, a_scale, b_scale, bias, static_cast<int>(M),
                 static_cast<int>(N), static_cast<int>(K), act, act_alpha, 0u, status};
  const I8Plan plan = choose_plan(M, N, K, aligned);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c_dtype == NPLK_DTYPE_FP32) return run(s, p, static_cast<float *>(C), plan);
  if (c_dtype == NPLK_DTYPE_FP16) return run(s, p, static_cast<__half *>(C), plan);
  return run(s, p, static_cast<__nv_bfloat16 *>(C), plan);
}
