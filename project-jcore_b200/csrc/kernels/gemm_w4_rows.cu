// 4-bit product for few tokens: the weights' bytes are what there is to do.
//
// A team of `slices` warps takes 32 channels at a time and shares K; a CTA holds `teams` of
// them and goes round the channels with the other CTAs, one CTA to an SM. mma.sync m16n8k16
// with the channels as its rows: lane (g, t) holds channels g, g + 8, g + 16 and g + 24 (two
// products) and token g. Which values of K a lane takes is free as long as weights and x
// agree, so a lane takes whole 32-bit words of eight nibbles, which come apart as the pairs
// (0, 4), (1, 5) for one mma and (2, 6), (3, 7) for the next; x lies in shared memory in that
// order. All lanes of one mma must lie in one group: for groups of 32, 64, 128 lane t takes
// 1, 2, 4 words in a row of each (its "run"), one load of shared memory each.
//
// Weights go by cp.async through a ring of each warp's own, across the ends of tiles: no
// barrier but the team's own, once per 32 channels, to add its sums. What bounds it: the
// widening's instructions as much as the bytes where there are many channels (16 channels a
// tile, with twice the loads of x and of scales to a weight, took 82 us where 32 take 67), and
// the latencies of a start, a stage and a meeting where there are few.
//
// Measured (group 128, cold weights): 1 x 4096 x 4096 bf16 6.7 us, 8 tokens 8.2;
// 4 x 128000 x 4096 fp16 67 us, of which the bytes are 43; 8 x 128000 x 4096 bf16 with groups
// of 32 78 us.
#include <algorithm>
#include <cmath>

#include "gemm_w4.cuh"
#include "ptx_sm100.cuh"

namespace nplk {
namespace {

constexpr int kRows = 32;                 // channels of a tile
constexpr int kStageK = 256;              // values of K a warp takes at a time
constexpr int kStagePitch = kStageK / 2;  // bytes
constexpr int kStageBytes = kRows * kStagePitch;
constexpr int kDepth = 2;                 // stages in flight and at work
constexpr int kMostWarps = 16;
// Bytes of x in shared memory, for up to eight tokens and for more; the first leave room for
// twelve warps.
constexpr int kMostX = 100 * 1024, kMostX16 = 64 * 1024;
constexpr int kRedBytes = kRows * 8 * 4;  // sums of a warp and eight tokens
constexpr int kWarpBytes = kDepth * kStageBytes + 2 * kRedBytes, kSmem = 232448;
static_assert(kMostX + 12 * kWarpBytes <= kSmem && kMostX16 + kMostWarps * kWarpBytes <= kSmem,
              "shared memory");

struct RowsPlan {
  int slices, teams;
  int steps;    // stages of K a warp takes for a tile
  int tiles;
  FastDiv words;  // eights of a token's values, padded to whole groups
  int x_bytes;  // room of x, whole 128 bytes: the ring behind it is swizzled by address
  int packed;   // a stage's scales of a channel as one aligned piece
};

__device__ __forceinline__ void team_sync(int team, int threads) {
  if (threads == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(threads) : "memory");
}

template <int kWords>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[kWords]) {
  if constexpr (kWords == 4) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (kWords == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  }
}

// Zeros where there is nothing. No branch: the compiler waits for a load where its branch
// joins, and one latency per load was half of a small call of eight tokens.
__device__ __forceinline__ uint4 load_if(const void *p, bool there) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  asm volatile(
      "{\n\t.reg .pred there;\n\tsetp.ne.u32 there, %5, 0;\n\t"
      "@there ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
      : "l"(p), "r"(static_cast<uint32_t>(there)));
  return v;
}

// NT: tokens in eights. Sums of a team have two buffers where NT is 1, so that one barrier a
// round keeps the next round's sums off this round's readers; else two barriers.
template <typename X, int NT, bool kZeros, int kGroup>
__global__ void __launch_bounds__(kMostWarps * 32, 1)
    gemm_w4_rows_kernel(const W4Args p, const RowsPlan plan) {
  using F = typename W4Type<X>::Frag;
  constexpr int P = W4Type<X>::kParts;
  constexpr int kRun = kGroup / 32;          // words of a lane in a group
  constexpr int kGroups = kStageK / kGroup;  // groups of a stage
  extern __shared__ __align__(128) uint8_t smem[];
  const int warps = plan.slices * plan.teams;
  uint4 *sx = reinterpret_cast<uint4 *>(smem);
  uint8_t *ring = smem + plan.x_bytes;
  float *red = reinterpret_cast<float *>(ring + warps * kDepth * kStageBytes);
  griddep_wait();
  griddep_launch_dependents();

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int slice = warp % plan.slices, team = warp / plan.slices;
  const int k_begin = slice * plan.steps * kStageK;
  const int steps = max(0, min(plan.steps, (p.K - k_begin + kStageK - 1) / kStageK));
  const int row_bytes = (p.K + 1) >> 1;
  const int stride = static_cast<int>(gridDim.x) * plan.teams;
  const int tile0 = static_cast<int>(blockIdx.x) * plan.teams + team;
  const int rounds = tile0 < plan.tiles ? (plan.tiles - tile0 + stride - 1) / stride : 0;
  uint8_t *mine = ring + warp * (kDepth * kStageBytes);

  // What is copied next: a stage of a tile, into a slot of the ring. Lane l copies the
  // 16 bytes l % 8 of rows l / 8, + 4, ... + 28; those are swizzled within their row.
  const int piece = lane & 7, c_r = lane >> 3;
  const uint32_t c_to = smem_u32(mine + c_r * kStagePitch + ((piece ^ (c_r * kRun & 7)) << 4));
  const int byte0 = k_begin / 2 + piece * 16;
  const bool no_tail = (k_begin + steps * kStageK) / 2 <= row_bytes;
  int c_round = steps ? 0 : rounds, c_step = 0, c_slot = 0;
  const uint8_t *c_row;  // of row c_r
  int64_t c_four;        // bytes from one of the lane's rows to the next
  int c_most;            // rows of the lane in the weights, less one
  const auto aim = [&](int round) {
    const int64_t n = static_cast<int64_t>(tile0 + round * stride) * kRows + c_r;
    // rows past the last are read as the lane's last, or the tile's first, their results dropped
    const int64_t left = p.N - 1 - n;
    c_most = left < 0 ? 0 : static_cast<int>(left < 28 ? left >> 2 : 7);
    c_row = p.q + (n < p.N ? n : p.N - 1) * p.ldq;
  };
  c_four = 4 * p.ldq;
  aim(0);
  const auto issue = [&] {
    if (c_round < rounds) {
      const int at = byte0 + c_step * (kStageK / 2);
      // of the 16 bytes; zeros for the rest
      const int valid = no_tail ? 16 : max(0, min(16, row_bytes - at));
      const uint8_t *from = c_row + (valid ? at : 0);
      const uint32_t to = c_to + static_cast<uint32_t>(c_slot * kStageBytes);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // (rows 4 apart differ in their swizzle where a row's step of it is 1)
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(
                         (kRun == 1 && (j & 1) ? to ^ 64u : to) + j * 4 * kStagePitch),
                     "l"(from), "r"(valid)
                     : "memory");
        if (j < c_most) from += c_four;
      }
      if (++c_step == steps) {
        c_step = 0;
        ++c_round;
        aim(c_round);
      }
    }
    c_slot = c_slot + 1 == kDepth ? 0 : c_slot + 1;
    copy_async_commit();
  };

  // Scales (and zeros) of a stage, loaded one stage ahead: lane l holds those of channel l.
  uint32_t sc_next[kGroups];  // as loaded: packed pairs in the first half, or one each
  uint32_t ze_next[kGroups];
  int64_t s_row = 0, z_row = 0;
  bool pairs = false;
  const auto aim_scales = [&](int round) {
    // past the last channel or group: the last one's, for results that are dropped and
    // inputs that are 0
    const int64_t at = static_cast<int64_t>(tile0 + round * stride) * kRows + lane;
    const int64_t n = at < p.N ? at : p.N - 1;
    s_row = n * p.lds;
    if (kZeros) z_row = n * p.ldz;
  };
  const auto fetch = [&](int step) {
    const int g0 = (k_begin + step * kStageK) / kGroup;
    if (plan.packed && g0 + kGroups <= p.groups) {  // 16-bit scales, whole pieces of 2 kGroups bytes
      const unsigned short *from = static_cast<const unsigned short *>(p.scale) + s_row + g0;
      pairs = true;
      if constexpr (kGroups == 2) {
        sc_next[0] = __ldg(reinterpret_cast<const unsigned int *>(from));
      } else if constexpr (kGroups == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(from));
        sc_next[0] = v.x, sc_next[1] = v.y;
      } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(from));
        sc_next[0] = v.x, sc_next[1] = v.y, sc_next[2] = v.z, sc_next[3] = v.w;
      }
    } else {
      pairs = false;
#pragma unroll
      for (int j = 0; j < kGroups; ++j)
        sc_next[j] = load_scale_bits(p.scale, p.scale_type, s_row + min(g0 + j, p.groups - 1));
    }
    if (kZeros) {
#pragma unroll
      for (int j = 0; j < kGroups; ++j)
        ze_next[j] = load_zero_bits(p.zero, z_row + min(g0 + j, p.groups - 1));
    }
  };

  // x into shared memory: unit w of a token holds the pairs of its eight values from 8 w on,
  // zeros behind K, each part by itself. In a chunk of 4 kRun units lane t of a quad takes units
  // t kRun + r, r = 0 .. kRun - 1; (chunk, r, part, token, t) lies at
  // (((chunk kRun + r) P + part) M + token) 4 + t.
  const X *x = static_cast<const X *>(p.x);
  const bool packs = reinterpret_cast<uintptr_t>(x) % 16 == 0 && p.ldx * sizeof(X) % 16 == 0 &&
                     p.K % p.group == 0;
  const int words = static_cast<int>(plan.words.d), all_words = words * p.M;
  struct Unit {
    uint4 v[sizeof(X) / 2];
  };
  const auto load_unit = [&](int u) {
    Unit unit;
    const int m = static_cast<int>(fdiv(u, plan.words));
    const X *from = x + m * p.ldx + (u - m * words) * 8;
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(X)) / 2; ++j)
      unit.v[j] = load_if(from + j * (16 / sizeof(X)), u < all_words);
    return unit;
  };
  const auto load_ragged = [&](int u) {
    Unit unit{};
    const int m = static_cast<int>(fdiv(u, plan.words)), k = (u - m * words) * 8;
    const X *from = x + m * p.ldx + k;
    X *v = reinterpret_cast<X *>(&unit);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < p.K) v[j] = from[j];
    return unit;
  };
  const auto store_unit = [&](int u, const Unit &unit) {
    const int m = static_cast<int>(fdiv(u, plan.words)), w = u - m * words;
    const int chunk = w / (4 * kRun), in = w % (4 * kRun), lane_t = in / kRun, r = in % kRun;
    const X *v = reinterpret_cast<const X *>(&unit);
    uint32_t h[P][4];  // pairs (0, 4), (1, 5), ... of each part
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (P == 3) {
        uint32_t parts[3];
        w4_split3(v[j], v[j + 4], parts);
#pragma unroll
        for (int q = 0; q < 3; ++q) h[q][j] = parts[q];
      } else {
        h[0][j] = reinterpret_cast<const uint16_t &>(v[j]) |
                  static_cast<uint32_t>(reinterpret_cast<const uint16_t &>(v[j + 4])) << 16;
      }
    }
#pragma unroll
    for (int q = 0; q < P; ++q)
      sx[(((chunk * kRun + r) * P + q) * p.M + m) * 4 + lane_t] =
          make_uint4(h[q][0], h[q][1], h[q][2], h[q][3]);
  };

  // all of the first loads before any of them is waited for: weights, x, scales
  constexpr int kUnits = 16 / sizeof(X);
  const int threads = static_cast<int>(blockDim.x), first = static_cast<int>(threadIdx.x);
  Unit units[kUnits];
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) issue();
  if (packs) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) units[i] = load_unit(first + i * threads);
  }
  aim_scales(0);
  fetch(0);
  if (packs) {
    for (int u = first;;) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
        if (u + i * threads < all_words) store_unit(u + i * threads, units[i]);
      u += kUnits * threads;
      if (u >= all_words) break;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) units[i] = load_unit(u + i * threads);
    }
  } else {
    for (int u = first; u < all_words; u += threads) store_unit(u, load_ragged(u));
  }
  __syncthreads();

  int slot = 0;
  const int swizzle = (g * kRun & 7) << 4;
  const int x_part = p.M * 4, x_chunk = kRun * P * x_part;
  int x_at[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x_at[n] = min(n * 8 + g, p.M - 1) * 4 + t;
  const int chunks_all = (p.K + kGroup - 1) / kGroup;
  for (int round = 0; round < rounds; ++round) {
    const int64_t n_out = static_cast<int64_t>(tile0 + round * stride) * kRows + lane;
    const float bias = p.bias && n_out < p.N ? __ldg(p.bias + n_out) : 0.0f;
    float acc[2][NT][4] = {};
    for (int step = 0; step < steps; ++step) {
      issue();
      float sc[kGroups];
      uint32_t offs[kGroups];  // low and high offset of the zero, a half each
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        const uint32_t pair = sc_next[j / 2];
        sc[j] = scale_value(!pairs ? sc_next[j] : j & 1 ? pair >> 16 : pair & 0xffffu, p.scale_type);
        if (kZeros) offs[j] = w4_adjacent_offset<F>(static_cast<int>(ze_next[j] & 15u));
      }
      if (step + 1 < steps) {
        fetch(step + 1);
      } else {
        aim_scales(round + 1);
        fetch(0);
      }
      copy_async_wait<kDepth - 1>();
      __syncwarp();
      const uint8_t *st = mine + slot * kStageBytes + g * kStagePitch;
      slot = slot + 1 == kDepth ? 0 : slot + 1;
      const int chunk0 = (k_begin + step * kStageK) / kGroup;
      const uint4 *xs = sx + chunk0 * x_chunk;
#pragma unroll
      for (int c = 0; c < kGroups; ++c, xs += x_chunk) {
        if (chunk0 + c >= chunks_all) break;
        uint32_t w[4][kRun];
        // rows are swizzled by 16-byte pieces, so that the 8 rows of a load miss each other's banks
        const int at = (c * (kGroup / 2) + t * (4 * kRun)) ^ swizzle;
#pragma unroll
        for (int h = 0; h < 4; ++h) load_words<kRun>(st + h * (8 * kStagePitch) + at, w[h]);
        W4Offsets off[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          if (kZeros) {
            const uint32_t both_of = __shfl_sync(0xffffffffu, offs[c], h * 8 + g);
            off[h] = {__byte_perm(both_of, 0u, 0x1010), __byte_perm(both_of, 0u, 0x3232)};
          } else {
            off[h] = w4_offsets<F>(8);
          }
        }
        float part[2][NT][4];
#pragma unroll
        for (int r = 0; r < kRun; ++r) {
          uint32_t wide[4][4];
#pragma unroll
          for (int h = 0; h < 4; ++h) w4_widen<F>(w[h][r], off[h], wide[h]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < P; ++q) {
              // tokens past the last are read as the last, their results dropped
              const uint4 v = xs[(r * P + q) * x_part + x_at[n]];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const auto &a = wide[2 * h], &b = wide[2 * h + 1];
                if (r == 0 && q == 0) {
                  const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                  F::mma(part[h][n], none, a[0], b[0], a[1], b[1], v.x, v.y);
                } else {
                  F::mma(part[h][n], part[h][n], a[0], b[0], a[1], b[1], v.x, v.y);
                }
                F::mma(part[h][n], part[h][n], a[2], b[2], a[3], b[3], v.z, v.w);
              }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float s0 = __shfl_sync(0xffffffffu, sc[c], h * 16 + g);
          const float s1 = __shfl_sync(0xffffffffu, sc[c], h * 16 + 8 + g);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[h][n][0] = fmaf(s0, part[h][n][0], acc[h][n][0]);
            acc[h][n][1] = fmaf(s0, part[h][n][1], acc[h][n][1]);
            acc[h][n][2] = fmaf(s1, part[h][n][2], acc[h][n][2]);
            acc[h][n][3] = fmaf(s1, part[h][n][3], acc[h][n][3]);
          }
        }
      }
      __syncwarp();  // the stage has been read: the next issue writes over it
    }
    // the team's sums meet, [token][channel]
    constexpr int kSums = NT * 8 * kRows;
    if (NT > 1) team_sync(team, plan.slices * 32);
    float *buffer = red + (NT == 1 ? (round & 1) * warps * kSums : 0);
    float *to = buffer + warp * kSums;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float *r = to + (8 * n + 2 * t) * kRows + h * 16 + g;
        r[0] = acc[h][n][0];
        r[kRows] = acc[h][n][1];
        r[8] = acc[h][n][2];
        r[kRows + 8] = acc[h][n][3];
      }
    team_sync(team, plan.slices * 32);
    const float *sums = buffer + team * plan.slices * kSums + lane;
    for (int m = slice; m < p.M; m += plan.slices) {
      float v[1] = {0.0f};
#pragma unroll 4
      for (int s = 0; s < plan.slices; ++s) v[0] += sums[s * kSums + m * kRows];
      v[0] = fmaf(v[0], F::kUnit, bias);
      if (n_out < p.N) w4_store<1>(p, m * p.ldc + n_out, v, 1, false);
    }
  }
  copy_async_wait<0>();
}

int parts_of(const W4Args &p) { return p.x_type == NPLK_DTYPE_FP32 ? 3 : 1; }
int64_t x_units(const W4Args &p) {
  return ceil_div(p.K, p.group) * (p.group / 8) * p.M * parts_of(p);
}

template <typename X, int NT>
auto pick(const W4Args &p) {
  switch (p.group) {
    case 32:
      return p.zero ? gemm_w4_rows_kernel<X, NT, true, 32> : gemm_w4_rows_kernel<X, NT, false, 32>;
    case 64:
      return p.zero ? gemm_w4_rows_kernel<X, NT, true, 64> : gemm_w4_rows_kernel<X, NT, false, 64>;
    default:
      return p.zero ? gemm_w4_rows_kernel<X, NT, true, 128>
                    : gemm_w4_rows_kernel<X, NT, false, 128>;
  }
}

}  // namespace

// Up to 16 tokens, as far as x fits, this way is the faster or even, against the tensor cores'
// tiles of 32 tokens: 1 and 8 x 4096 x 4096 bf16 6.7 and 8.2 us (9.1, 9.2), 1 x 16384 x 4096
// 12 (17), 16 x 128000 x 2048 52 (77), 16 x 4096 x 2048 7.9 (7.6). With more of x than leaves
// room for sixteen warps: 4 x 4096 x 11008 12.3 (14.6), 3 x 4096 x 16384 15.7 (18.5), 4 x 4096 x
// 4096 fp32 10.3 (16.1), 12 x 16384 x 4096 17.7 (17.3), 8 x 4096 x 8192, where ten are left,
// 13.4 (12.1).
bool gemm_w4_rows_fits(const W4Args &p) {
  return p.M <= 16 && x_units(p) * 16 <= (p.M <= 8 ? kMostX : kMostX16) &&
         reinterpret_cast<uintptr_t>(p.q) % 16 == 0 && (p.ldq % 16 == 0 || p.N == 1);
}

// Slices and teams of least estimated time: rounds of (stages of K, 1.5 us each for 16
// warps at the memory's rate and hardly less for few, and the sums' meeting), and x's way into
// shared memory.
int gemm_w4_rows(cudaStream_t s, const W4Args &p) {
  RowsPlan plan{};
  const int64_t sms = sm_count(), stages = ceil_div(p.K, kStageK);
  plan.tiles = static_cast<int>(ceil_div(p.N, kRows));
  plan.x_bytes = static_cast<int>(align_up(static_cast<size_t>(x_units(p)) * 16, 128));
  const int64_t most = std::min(kMostWarps, (kSmem - plan.x_bytes) / kWarpBytes);
  double least = 1e30;
  for (int64_t want = 1; want <= std::min(stages, most); ++want) {
    const int64_t steps = ceil_div(stages, want), slices = ceil_div(stages, steps);
    const int64_t teams = std::min<int64_t>(most / slices, std::max<int64_t>(1, ceil_div(plan.tiles, sms)));
    const int64_t rounds = ceil_div(plan.tiles, teams * sms);
    const double warps = static_cast<double>(slices * teams);
    const double us =
        static_cast<double>(rounds) *
            (std::max(0.093 * static_cast<double>(steps) * warps, 0.5 * static_cast<double>(steps)) +
             0.3) +
        0.15 * std::ceil(static_cast<double>(ceil_div(p.K, 8) * p.M) / (32.0 * warps));
    if (us < least) {
      least = us;
      plan.steps = static_cast<int>(steps);
      plan.slices = static_cast<int>(slices);
      plan.teams = static_cast<int>(teams);
    }
  }
  plan.words = make_fastdiv(static_cast<uint32_t>(ceil_div(p.K, p.group) * (p.group / 8)));
  // pieces of 2 (256 / group) bytes
  const int64_t piece = kStageK / p.group;
  plan.packed = p.scale_type != NPLK_DTYPE_FP32 && p.lds % piece == 0 &&
                reinterpret_cast<uintptr_t>(p.scale) % (2 * piece) == 0;
  const int warps = plan.slices * plan.teams, nt = p.M <= 8 ? 1 : 2;
  const int smem = plan.x_bytes + warps * kWarpBytes;
  auto *fn = p.x_type == NPLK_DTYPE_FP32   ? (nt == 1 ? pick<float, 1>(p) : pick<float, 2>(p))
             : p.x_type == NPLK_DTYPE_FP16 ? (nt == 1 ? pick<__half, 1>(p) : pick<__half, 2>(p))
                                           : (nt == 1 ? pick<__nv_bfloat16, 1>(p)
                                                      : pick<__nv_bfloat16, 2>(p));
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(fn), smem);
  if (rc) return rc;
  const int64_t grid = std::min<int64_t>(ceil_div(plan.tiles, plan.teams), sms);
  return launch_programmatic(fn, dim3(static_cast<unsigned>(grid)),
                             dim3(static_cast<unsigned>(warps * 32)), static_cast<size_t>(smem), s,
                             p, plan);
}

}  // namespace nplk
