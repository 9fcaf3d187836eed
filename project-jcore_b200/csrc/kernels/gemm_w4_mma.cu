// 4-bit product for more tokens, on the tensor cores' own accumulators (tcgen05).
//
// A tile is 128 channels (the accumulator's lanes) x NTOK tokens (its columns); K may be
// shared by a cluster of up to 8 CTAs. Weights arrive packed by TMA, eight warps widen
// them to whole numbers in fp16 or bf16 (exact), into TMEM, where the matrix
// instructions take them from. A scale belongs to a channel and a group, so the
// sums of one group go to an accumulator of their own, and eight other warps add
// scale * accumulator to fp32 registers while the next group runs: a lane is a
// channel, so the scale is one register. Scaling the weights before the product would
// round them once more (2^-9 for bf16).
//
// x comes by TMA where it can (16-bit, 16-byte aligned rows); otherwise, and for fp32, whose
// three bf16 parts each take a product of their own, eight more warps bring it.
//
// Measured (group 128, cold weights): 512 x 4096 x 4096 bf16 22.3 us, 512 x 16384 x 4096 89,
// 48 x 16384 x 4096 with zeros 18.5, 256 x 4096 x 4096 fp32 47. What bounds it are the roles'
// waits for one another: without loads, widening, products and sums they alone take 15 us of
// the 48 tokens' time and 20 of the 512's (issue is at 59%, three instructions to a pair of
// weights and some 70 to an epilogue warp's group; the tensor cores are at 40%). Groups of 64
// and 32 have two and four times the sums to add: 512 x 4096 x 4096 41 and 69 us.
#include <algorithm>

#include "gemm_w4.cuh"
#include "ptx_sm100.cuh"

namespace nplk {
namespace {

constexpr int kChannels = 128, kBK = 128;  // of a tile; values of K a stage
constexpr int kRawBytes = kChannels * (kBK / 2);
constexpr int kACols = kBK / 2;            // TMEM columns of a stage's widened weights
// Warpgroups: TMA and MMA issue; epilogue; widening (two); x where it does not come by TMA
// (two). A stage's chain of waits, loads and stores is long against its products, so roles
// come in two teams that take every second stage or group: MMA issue, widening and, up to 64
// tokens, the epilogue.
//
// Epilogue: sixteen warps where groups' sums are many, 128 tokens or short groups (512 x 4096 x
// 4096 23.6 us, 25.3 with eight; 48 x 16384 x 4096 with groups of 32 37 and 42); eight otherwise
// (48 x 16384 x 4096 21.1 us, 22.0 with sixteen; 17 x 4096 x 4096 9.3 and 10.1; all before
// halves were read under sums, which took another 4%).
//
// Warps, threads, and registers a thread: at launch, and as the warpgroups share them.
template <int NTOK, int kGroup, bool kTma>
struct MmaThreads {
  static constexpr bool kMany = kTma && (NTOK == 128 || kGroup < 128);
  static constexpr int kEpiFirst = 4, kEpiWarps = kMany ? 16 : 8,
                       kWideFirst = kEpiFirst + kEpiWarps, kWideWarps = 8,
                       kXFirst = kWideFirst + kWideWarps, kXWarps = kTma ? 0 : 8;
  static constexpr int kThreads = 32 * (kXFirst + kXWarps);
  static constexpr int kLaunch = kTma && !kMany ? 96 : 72;
  static constexpr int kIssue = kTma && !kMany ? 48 : 40,
                       kEpi = !kTma ? 88 : kMany ? 80 : 136, kWide = kTma && !kMany ? 80 : 64,
                       kX = 72;
  static_assert(kIssue * 128 + kEpi * 32 * kEpiWarps + kWide * 32 * kWideWarps +
                        kX * 32 * kXWarps <=
                    kLaunch * kThreads,
                "register shares");
  static_assert(kLaunch * kThreads <= 65536 && (kLaunch + 8) * kThreads > 65536,
                "what the launch bounds give a thread");
};

// P parts of x.
template <int NTOK, int P, int kGroup, bool kTma>
struct MmaTraits {
  // Epilogue teams, and the tokens of one of their warps, whose sums it holds.
  static constexpr int kTeams = NTOK <= 64 && kTma ? 2 : 1;
  static constexpr int kParts = MmaThreads<NTOK, kGroup, kTma>::kEpiWarps / 4 / kTeams;
  static constexpr int kCols = NTOK / kParts;
  static constexpr int kAccCols = NTOK == 48 ? 64 : NTOK;  // from one accumulator to the next
  static constexpr int kXAtom = NTOK * 128;  // NTOK rows x 64 values
  static constexpr int kXBytes = 2 * kXAtom * P;
  // Rings: widened weights in TMEM, x (its loads take some 2000 cycles, a stage about
  // 600) and packed weights in shared memory.
  static constexpr int kA = 4, kX = kXBytes <= 16 * 1024 ? 8 : 4;
  static constexpr int kRaw =
      208 * 1024 - kX * kXBytes > 8 * kRawBytes ? 8 : (208 * 1024 - kX * kXBytes) / kRawBytes;
  static constexpr int kAcc = NTOK == 128 ? 2 : 4;
  static constexpr int kTmemCols = 512;
  static constexpr int kRings = kX * kXBytes + kRaw * kRawBytes;
  static constexpr int kBarriers = 2 * (kA + kX + kRaw + kAcc) + 1;
  // at least what keeps other clusters' TMEM off this SM
  static constexpr int kNeeded = 1024 + kRings + 8 * kBarriers + 64;
  static constexpr int kSmem = kNeeded > 200 * 1024 ? kNeeded : 200 * 1024;
  static_assert(kAcc * kAccCols + kA * kACols <= kTmemCols, "TMEM columns");
  static_assert(kRaw >= 2 && kRaw % 2 == 0 && kA % 2 == 0 && kX % 2 == 0 && kAcc % 2 == 0,
                "a slot belongs to one of two teams");
  static_assert(kTeams * NTOK * kChannels * 4 <= kRings, "partial sums over the rings");
  static_assert(kSmem <= 232448, "shared memory budget");
  static_assert(tmem_excludes_clusters(kSmem), "no other cluster's TMEM beside this one's");
};

// Accumulators belong to issuer teams, kAcc / 2 each, taken in turn: a team's l-th group uses
// its slot l mod (kAcc / 2) for the l / (kAcc / 2)-th time. Waits are by parity, so whoever
// waits on a slot has to see each of its uses; the epilogue's teams are the issuers' for that.
template <int kAcc>
struct AccSlot {
  int at;
  uint32_t phase;
  __device__ __forceinline__ AccSlot(int team, int l)
      : at(team * (kAcc / 2) + l % (kAcc / 2)), phase(l / (kAcc / 2) & 1) {}
};

struct MmaPlan {
  int slices, n_tiles;
  uint32_t stall_us;  // fault injection: 0 except on an armed launch
};

// A wait's outcome for the whole warp: TMEM accesses and warp barriers are for whole warps.
__device__ __forceinline__ bool all(bool done) { return __all_sync(0xffffffffu, done); }

// A slot of a ring and the phase of its barriers.
struct Slot {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int count) {
    if (++at == count) {
      at = 0;
      phase ^= 1u;
    }
  }
};

// kCols consecutive TMEM columns of this thread's lane, and the wait for them.
template <int kCols>
__device__ __forceinline__ void tmem_ld(uint32_t from, uint32_t (&v)[kCols]) {
  if constexpr (kCols == 16) tmem_ld16(from, v);
  else tmem_ld32(from, v);
}
template <int kCols>
__device__ __forceinline__ void tmem_landed(uint32_t (&v)[kCols]) {
  if constexpr (kCols == 16) tmem_wait_ld16(v);
  else tmem_wait_ld(v);
}

template <typename X, int NTOK, int kGroup, bool kTma>
__global__ void __launch_bounds__(MmaThreads<NTOK, kGroup, kTma>::kThreads, 1)
    gemm_w4_mma_kernel(const __grid_constant__ CUtensorMap map_w,
                       const __grid_constant__ CUtensorMap map_x, const W4Args p,
                       const MmaPlan plan) {
  using F = typename W4Type<X>::Frag;
  constexpr int P = W4Type<X>::kParts;
  using Tr = MmaTraits<NTOK, P, kGroup, kTma>;
  using Th = MmaThreads<NTOK, kGroup, kTma>;
  constexpr int kPer = kBK / kGroup;  // groups a stage
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = align_smem_1024(smem_raw);
  uint8_t *ring_x = smem, *ring_raw = ring_x + Tr::kX * Tr::kXBytes;
  uint64_t *a_full = reinterpret_cast<uint64_t *>(smem + Tr::kRings);
  uint64_t *a_empty = a_full + Tr::kA, *x_full = a_empty + Tr::kA, *x_empty = x_full + Tr::kX,
           *raw_full = x_empty + Tr::kX, *raw_empty = raw_full + Tr::kRaw,
           *acc_full = raw_empty + Tr::kRaw, *acc_empty = acc_full + Tr::kAcc,
           *never = acc_empty + Tr::kAcc;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(never + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % plan.slices;
  const int tile = static_cast<int>(blockIdx.x) / plan.slices;
  const int n0 = tile % plan.n_tiles * kChannels, m0 = tile / plan.n_tiles * NTOK;
  const int blocks = (p.K + kBK - 1) / kBK;
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * blocks / plan.slices);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * blocks / plan.slices);
  const int g_begin = kb0 * kPer, g_end = min(p.groups, kb1 * kPer);

  if (threadIdx.x == 0) {
    for (int i = 0; i < Tr::kA; ++i) {
      mbar_init(&a_full[i], Th::kWideWarps / 2);
      mbar_init(&a_empty[i], 1);
    }
    for (int i = 0; i < Tr::kX; ++i) {
      mbar_init(&x_full[i], kTma ? 1 : Th::kXWarps);
      mbar_init(&x_empty[i], 1);
    }
    for (int i = 0; i < Tr::kRaw; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], Th::kWideWarps / 2);
    }
    for (int i = 0; i < Tr::kAcc; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], Th::kEpiWarps / Tr::kTeams);
    }
    mbar_init(never, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_w);
    if (kTma) tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Tr::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot, tmem_a = tmem_base + Tr::kAcc * Tr::kAccCols;
  griddep_wait();
  griddep_launch_dependents();

  bool have = false;  // epilogue warps: the sums are whole
  if (warp < Th::kEpiFirst) {
    registers_down<Th::kIssue>();
    if (warp == 0 && lane == 0) {
      // ---------------- TMA: packed weights ----------------
      Slot r;
      uint32_t used = 0, last = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&raw_empty[r.at], r.phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer))
          break;
        mbar_arrive_expect_tx(&raw_full[r.at], kRawBytes);
        tma_load_2d(&map_w, &raw_full[r.at], ring_raw + r.at * kRawBytes, kb * (kBK / 2), n0);
        used |= 1u << r.at;
        last = (last & ~(1u << r.at)) | (r.phase << r.at);
        r.next(Tr::kRaw);
      }
      // the last copy into each slot lands before the CTA can exit
      for (int i = 0; i < Tr::kRaw; ++i)
        if ((used >> i) & 1u) mbar_drain(&raw_full[i], (last >> i) & 1u);
    } else if (kTma && warp == 3 && lane == 0) {
      // ---------------- TMA: x ----------------
      Slot x;
      uint32_t used = 0, last = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&x_empty[x.at], x.phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer))
          break;
        mbar_arrive_expect_tx(&x_full[x.at], Tr::kXBytes);
        uint8_t *to = ring_x + x.at * Tr::kXBytes;
        tma_load_2d(&map_x, &x_full[x.at], to, kb * (kBK * 2), m0);
        tma_load_2d(&map_x, &x_full[x.at], to + Tr::kXAtom, kb * (kBK * 2) + 128, m0);
        used |= 1u << x.at;
        last = (last & ~(1u << x.at)) | (x.phase << x.at);
        x.next(Tr::kX);
      }
      for (int i = 0; i < Tr::kX; ++i)
        if ((used >> i) & 1u) mbar_drain(&x_full[i], (last >> i) & 1u);
    } else if (warp == 1 || warp == 2) {
      // ---------------- MMA issuers ----------------
      // The whole warp goes round, one lane issues: addresses and descriptors then stay in
      // uniform registers (one lane alone took 75 cycles an instruction). Groups have
      // accumulators of their own, so the two warps' products need no order.
      const int team = warp - 1;
      const uint32_t idesc = umma_idesc_f16(std::is_same<F, W4Bfloat>::value, kChannels, NTOK);
      const uint64_t desc0 = umma_desc_sw128(smem_u32(ring_x));
      Slot st, x;
      if (team) {
        st.next(Tr::kA);
        x.next(Tr::kX);
      }
      bool go = team || all(injected_stall(never, plan.stall_us, abort_flag, p.status));
      for (int kb = kb0 + team; go && kb < kb1; kb += 2) {
        const bool a_ready = mbar_test(&a_full[st.at], st.phase),
                   x_ready = mbar_test(&x_full[x.at], x.phase);
        if (!all(a_ready && x_ready))
          go = all(mbar_wait(&a_full[st.at], st.phase, abort_flag, p.status, kStatusTimeoutMma) &&
                   mbar_wait(&x_full[x.at], x.phase, abort_flag, p.status, kStatusTimeoutMma));
        if (!go) break;
        const uint64_t desc = desc0 + static_cast<uint64_t>(x.at * (Tr::kXBytes >> 4));
        const uint32_t a = tmem_a + static_cast<uint32_t>(st.at * kACols);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (kb * kPer + i >= g_end) break;
          const AccSlot<Tr::kAcc> acc(team, (kb - kb0) / 2 * kPer + i);
          const uint32_t free = acc.phase ^ 1u;
          if (!all(mbar_test(&acc_empty[acc.at], free)))
            go = all(mbar_wait(&acc_empty[acc.at], free, abort_flag, p.status,
                               kStatusTimeoutAccFree));
          if (!go) break;
          tc_fence_after_sync();
          const uint32_t d = tmem_base + static_cast<uint32_t>(acc.at * Tr::kAccCols);
          if (elect_lane()) {
#pragma unroll
            for (int kk = 0; kk < kGroup / 16; ++kk) {
              const int k = i * kGroup + kk * 16;  // of the stage
#pragma unroll
              for (int q = 0; q < P; ++q)
                mma_f16_ts(d, a + k / 2,
                           desc + static_cast<uint64_t>(((2 * q + k / 64) * Tr::kXAtom >> 4) +
                                                        k % 64 / 8),
                           idesc, kk > 0 || q > 0 ? 1u : 0u);
            }
            mma_commit(&acc_full[acc.at]);
          }
          __syncwarp();
        }
        if (!go) break;
        if (elect_lane()) {  // slots that are to be filled again
          if (kb + Tr::kA < kb1) mma_commit(&a_empty[st.at]);
          if (kb + Tr::kX < kb1) mma_commit(&x_empty[x.at]);
        }
        __syncwarp();
        st.next(Tr::kA);
        st.next(Tr::kA);
        x.next(Tr::kX);
        x.next(Tr::kX);
      }
    }
    __syncwarp();
  } else if (warp < Th::kWideFirst) {
    // ---------------- groups' sums: scaled and added in registers ----------------
    registers_up<Th::kEpi>();
    constexpr int kCols = Tr::kCols;
    const int quad = warp & 3, of = (warp - Th::kEpiFirst) >> 2;
    const int team = of / Tr::kParts, first = of % Tr::kParts * kCols;  // tokens from here on
    const int64_t n = static_cast<int64_t>(n0) + quad * 32 + lane;
    const uint32_t row =
        tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(first);
    float2 sum[kCols / 2] = {};
    // channels past the last take its scales, their results are dropped
    const int64_t scale_row = (n < p.N ? n : p.N - 1) * p.lds;
    const auto scale_at = [&](int g) {
      return load_scale_bits(p.scale, p.scale_type, scale_row + min(g, g_end - 1));
    };
    // this team's j-th group, and its accumulator
    const auto group_of = [&](int j) {
      return Tr::kTeams == 2 ? (kb0 + team + j / kPer * 2) * kPer + j % kPer : g_begin + j;
    };
    const auto slot_of = [&](int j) {
      return Tr::kTeams == 2
                 ? AccSlot<Tr::kAcc>(team, j)
                 : AccSlot<Tr::kAcc>(j / kPer % 2, j / (2 * kPer) * kPer + j % kPer);
    };
    uint32_t s_next = scale_at(group_of(0)), s_after = scale_at(group_of(1));
    have = true;
    // A group's chain -- the wait, the read, the sums -- is what bounds short groups: the next
    // group's barrier is asked for and the scale brought along under this one's sums. More
    // than 32 columns are read in two parts, under each other's sums.
    constexpr int kRead = kCols < 32 ? kCols : 32, kRest = kCols > 32 ? kCols - 32 : 16;
    const auto add = [&](const auto &v, int at, float s) {
#pragma unroll
      for (int c = 0; c < static_cast<int>(sizeof(v) / 8); ++c)
        sum[at / 2 + c] = fma2(make_float2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])),
                               both(s), sum[at / 2 + c]);
    };
    uint32_t va[kRead], vb[kRest];
    bool ready = false;  // the next group; where columns are more than 32, read as far as va
    AccSlot<Tr::kAcc> acc = slot_of(0);
    for (int j = 0; group_of(j) < g_end; ++j) {
      const AccSlot<Tr::kAcc> next = slot_of(j + 1);
      const uint32_t from = row + static_cast<uint32_t>(acc.at * Tr::kAccCols);
      if (!all(ready)) {
        have = all(mbar_wait(&acc_full[acc.at], acc.phase, abort_flag, p.status,
                             kStatusTimeoutEpilogue));
        if (!have) break;
      }
      if (kCols <= 32 || !ready) {
        tc_fence_after_sync();
        tmem_ld<kRead>(from, va);
      }
      const float s = scale_value(s_next, p.scale_type);
      s_next = s_after;
      s_after = scale_at(group_of(j + 2));
      tmem_landed<kRead>(va);
      if constexpr (kCols > 32) {
        tmem_ld<kRest>(from + kRead, vb);
        add(va, 0, s);
        tmem_landed<kRest>(vb);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc.at]);  // all read: it is free again
      ready = mbar_test(&acc_full[next.at], next.phase);
      if constexpr (kCols > 32) {
        ready = group_of(j + 1) < g_end && all(ready);
        if (ready) {
          tc_fence_after_sync();
          tmem_ld<kRead>(row + static_cast<uint32_t>(next.at * Tr::kAccCols), va);
        }
        add(vb, kRead, s);
      } else {
        add(va, 0, s);
      }
      acc = next;
    }
    // [team][token][channel], over the rings. Another team's groups may still be at work on
    // them: all their MMAs have read the rings once the whole epilogue is here.
    asm volatile("bar.sync 1, %0;" ::"n"(Th::kEpiWarps * 32) : "memory");
    if (have) {
      float *part = reinterpret_cast<float *>(smem) +
                    (team * NTOK + first) * kChannels + quad * 32 + lane;
#pragma unroll
      for (int j = 0; j < kCols; ++j)
        part[j * kChannels] = (j & 1 ? sum[j / 2].y : sum[j / 2].x) * F::kUnit;
    }
    __syncwarp();
    if (plan.slices == 1)
      asm volatile("bar.sync 1, %0;" ::"n"(Th::kEpiWarps * 32) : "memory");  // these warps
  } else if (warp < Th::kXFirst) {
    // ---------------- widening: packed rows to TMEM, every second stage ----------------
    registers_down<Th::kWide>();
    const int quad = warp & 3, team = (warp - Th::kWideFirst) >> 2;
    const int row = quad * 32 + lane;  // a channel: its lane of TMEM
    const int64_t n = static_cast<int64_t>(n0) + row;
    const uint32_t t_row = tmem_a + (static_cast<uint32_t>(quad * 32) << 16);
    const int64_t zero_row = (n < p.N ? n : p.N - 1) * p.ldz;
    const auto zero_at = [&](int kb, int i) {
      return p.zero ? load_zero_bits(p.zero, zero_row + min(kb * kPer + i, p.groups - 1)) : 8u;
    };
    uint32_t z_next[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) z_next[i] = zero_at(kb0 + team, i);
    Slot st, r;
    if (team) {
      st.next(Tr::kA);
      r.next(Tr::kRaw);
    }
    for (int kb = kb0 + team; kb < kb1; kb += 2) {
      uint32_t off[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        off[i] = w4_adjacent_offset<F>(static_cast<int>(z_next[i] & 15u));
        z_next[i] = zero_at(kb + 2, i);
      }
      const bool raw_ready = mbar_test(&raw_full[r.at], r.phase),
                 a_free = mbar_test(&a_empty[st.at], st.phase ^ 1u);
      if (!all(raw_ready && a_free) &&
          !all(mbar_wait(&raw_full[r.at], r.phase, abort_flag, p.status, kStatusTimeoutStage) &&
               mbar_wait(&a_empty[st.at], st.phase ^ 1u, abort_flag, p.status,
                         kStatusTimeoutStage)))
        break;
      tc_fence_after_sync();
      const uint8_t *from = ring_raw + r.at * kRawBytes + row * 64;
      const int sw = (row >> 1) & 3;
      const uint32_t to = t_row + static_cast<uint32_t>(st.at * kACols);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const uint4 lo = *reinterpret_cast<const uint4 *>(from + ((i ^ sw) << 4));
        const uint4 hi = *reinterpret_cast<const uint4 *>(from + (((i + 1) ^ sw) << 4));
        if (i == 2) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&raw_empty[r.at]);
        }
        uint32_t v[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint4 &q = j < 4 ? lo : hi;
          const uint32_t word = j % 4 == 0 ? q.x : j % 4 == 1 ? q.y : j % 4 == 2 ? q.z : q.w;
          const uint4 w = w4_widen_adjacent<F>(word, off[(i * 32 + j * 8) / kGroup]);
          v[4 * j] = w.x;
          v[4 * j + 1] = w.y;
          v[4 * j + 2] = w.z;
          v[4 * j + 3] = w.w;
        }
        tmem_st32(to + i * 16, v);
      }
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full[st.at]);
      st.next(Tr::kA);
      st.next(Tr::kA);
      r.next(Tr::kRaw);
      r.next(Tr::kRaw);
    }
    __syncwarp();
  } else {
    // ---------------- x without TMA ----------------
    if constexpr (!kTma) {
      registers_up<Th::kX>();
      const X *src = static_cast<const X *>(p.x);
      const int tid = static_cast<int>(threadIdx.x) - Th::kXFirst * 32;
      const bool packs = reinterpret_cast<uintptr_t>(src) % 16 == 0 && p.ldx * sizeof(X) % 16 == 0;
      constexpr int E = 16 / sizeof(X), kPieces = NTOK * 16 / (Th::kXWarps * 32);
      Slot x;
      for (int kb = kb0; kb < kb1; ++kb) {
        // pieces of eight values, 16 to a token's row of the stage; all loads first, ahead of
        // the slot
        alignas(16) X v[kPieces][8];
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          const int i = tid + c * (Th::kXWarps * 32), token = i >> 4, k = kb * kBK + (i & 15) * 8;
          const X *from = src + static_cast<int64_t>(m0 + token) * p.ldx + k;
          if (packs && m0 + token < p.M && k + 8 <= p.K) {
#pragma unroll
            for (int j = 0; j < 8; j += E)
              *reinterpret_cast<Pack<X, E> *>(v[c] + j) = load_pack<X, E>(from + j);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              v[c][j] = m0 + token < p.M && k + j < p.K ? from[j] : from_float<X>(0.0f);
          }
        }
        if (!all(mbar_wait(&x_empty[x.at], x.phase ^ 1u, abort_flag, p.status, kStatusTimeoutStage)))
          break;
        uint8_t *xs = ring_x + x.at * Tr::kXBytes;
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          const int i = tid + c * (Th::kXWarps * 32), token = i >> 4, piece = i & 15;
          uint32_t h[P][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (P == 3) {
              uint32_t parts[3];
              w4_split3(v[c][2 * j], v[c][2 * j + 1], parts);
#pragma unroll
              for (int q = 0; q < 3; ++q) h[q][j] = parts[q];
            } else {
              h[0][j] = reinterpret_cast<const uint32_t &>(v[c][2 * j]);
            }
          }
#pragma unroll
          for (int q = 0; q < P; ++q)
            *reinterpret_cast<uint4 *>(xs + (2 * q + (piece >> 3)) * Tr::kXAtom +
                                       sw128_offset(static_cast<uint32_t>(token), piece & 7)) =
                make_uint4(h[q][0], h[q][1], h[q][2], h[q][3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&x_full[x.at]);
        x.next(Tr::kX);
      }
    }
    __syncwarp();
  }

  if (plan.slices > 1) cluster_sync();  // every CTA's sums are in its shared memory
  if (warp >= Th::kEpiFirst && warp < Th::kWideFirst && have) {
    // this CTA's share of the cluster's tokens: a token per warp at a time, four channels a lane
    const int each = NTOK / plan.slices;
    const int64_t n = static_cast<int64_t>(n0) + 4 * lane;
    float bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) bias[j] = p.bias && n + j < p.N ? p.bias[n + j] : 0.0f;
    const int size = p.c_type == NPLK_DTYPE_FP32 ? 4 : 2;
    const bool whole = p.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(p.C) % (4 * size) == 0;
    const int count = n < p.N ? static_cast<int>(p.N - n < 4 ? p.N - n : 4) : 0;
    for (int i = warp - Th::kEpiFirst; i < each; i += Th::kEpiWarps) {
      const int token = rank * each + i;
      // (a load from another CTA that no store waits for could be under way when that CTA ends)
      if (m0 + token >= p.M || count == 0) break;
      const uint32_t at = smem_u32(smem) + static_cast<uint32_t>(token * kChannels + 4 * lane) * 4u;
      float v[4] = {};
      for (int i = 0; i < plan.slices * Tr::kTeams; ++i) {
        const int team = i % Tr::kTeams * (NTOK * kChannels * 4);
        const uint4 q = plan.slices == 1
                            ? *reinterpret_cast<const uint4 *>(smem + team + (token * kChannels + 4 * lane) * 4)
                            : ld_shared_cluster_v4(mapa_shared(at + team, static_cast<uint32_t>(i / Tr::kTeams)));
        v[0] += __uint_as_float(q.x);
        v[1] += __uint_as_float(q.y);
        v[2] += __uint_as_float(q.z);
        v[3] += __uint_as_float(q.w);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += bias[j];
      w4_store<4>(p, static_cast<int64_t>(m0 + token) * p.ldc + n, v, count, whole);
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  if (plan.slices > 1) cluster_sync();  // no CTA leaves while another reads its shared memory
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, Tr::kTmemCols);
  }
}

template <typename X, int NTOK, int kGroup, bool kTma>
int launch(cudaStream_t s, const W4Args &p, MmaPlan plan) {
  using Tr = MmaTraits<NTOK, W4Type<X>::kParts, kGroup, kTma>;
  CUtensorMap mw, mx = {};
  int rc = encode_tmap_2d_u8_sw64(&mw, p.q, ceil_div(p.K, 2), p.N, p.ldq, kChannels);
  if (!rc && kTma) rc = encode_tmap_2d_u8_sw128(&mx, p.x, 2 * static_cast<int64_t>(p.K), p.M, 2 * p.ldx, NTOK);
  if (rc) return rc;
  auto *fn = gemm_w4_mma_kernel<X, NTOK, kGroup, kTma>;
  rc = ensure_dynamic_smem(reinterpret_cast<const void *>(fn), Tr::kSmem);
  if (rc) return rc;
  plan.n_tiles = static_cast<int>(ceil_div(p.N, kChannels));
  const int64_t ctas = static_cast<int64_t>(plan.n_tiles) * ceil_div(p.M, NTOK) * plan.slices;
  if (ctas >= (int64_t(1) << 31)) return kErrUnsupported;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(plan.slices);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(MmaThreads<NTOK, kGroup, kTma>::kThreads);
  cfg.dynamicSmemBytes = Tr::kSmem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = plan.slices > 1 ? 2 : 1;
  count_launch();
  return map_cuda_error(cudaLaunchKernelEx(&cfg, fn, mw, mx, p, plan));
}

template <typename X, int NTOK, bool kTma>
int by_group(cudaStream_t s, const W4Args &p, const MmaPlan &plan) {
  return p.group == 32   ? launch<X, NTOK, 32, kTma>(s, p, plan)
         : p.group == 64 ? launch<X, NTOK, 64, kTma>(s, p, plan)
                         : launch<X, NTOK, 128, kTma>(s, p, plan);
}

template <typename X>
int by_tokens(cudaStream_t s, const W4Args &p, const MmaPlan &plan, int tokens, bool tma) {
  if (!tma) return by_group<X, 64, false>(s, p, plan);
  if (tokens == 48) return launch<X, 48, 128, true>(s, p, plan);
  return tokens == 32   ? by_group<X, 32, true>(s, p, plan)
         : tokens == 64 ? by_group<X, 64, true>(s, p, plan)
                        : by_group<X, 128, true>(s, p, plan);
}

}  // namespace

bool gemm_w4_mma_fits(const W4Args &p) {
  return reinterpret_cast<uintptr_t>(p.q) % 16 == 0 && (p.ldq % 16 == 0 || p.N == 1);
}

int gemm_w4_mma(cudaStream_t s, const W4Args &args) {
  W4Args p = args;
  if (p.N == 1) p.ldq = static_cast<int64_t>(align_up(ceil_div(p.K, 2), 16));  // a pitch that leads nowhere
  const bool tma = p.x_type != NPLK_DTYPE_FP32 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 &&
                   (p.ldx % 8 == 0 || p.M == 1);
  if (p.M == 1) p.ldx = static_cast<int64_t>(align_up(p.K, 8));
  // tiles of 48 tokens where there are eight epilogue warps (48 x 16384 x 4096 with zeros 19.6 us,
  // as 64 columns 20.4)
  const int tokens = !tma                               ? 64
                     : p.M <= 32                        ? 32
                     : p.M <= 48 && p.group == kBK ? 48
                     : p.M <= 64                        ? 64
                                                        : 128;
  const int64_t sms = sm_count(), blocks = ceil_div(p.K, kBK);
  const int64_t tiles = ceil_div(p.N, kChannels) * ceil_div(p.M, tokens);
  MmaPlan plan{1, 0, 0};
  // waves of (start and end, stages of a slice), and the slices' meeting, as measured for groups of 128
  // in 16 bits. Shorter groups' and fp32 tokens' stages take two to four times as long, which moves
  // the choice little; it is the best of the four for them too (us for 1, 2, 4, 8 slices: 64 x 4096 x 4096 18.7,
  // 13.3, 11.7, 30.2; with groups of 32 34.1, 20.9, 15.9, 39.2; 256 tokens with groups of 32 69, 38.6, 46,
  // 78; 512 69, 77, 91, 141; 40 x 4096 x 4096 fp32 52, 29.8, 17.5, 36; 64 x 1000 x 16384 bf16 58, 33, 20, 15.1).
  double least = 1e30;
  for (int slices : {1, 2, 4, 8}) {
    if (slices > blocks) break;
    const double us = static_cast<double>(ceil_div(tiles * slices, sms)) *
                          (4.5 + 0.55 * static_cast<double>(ceil_div(blocks, slices))) +
                      (slices > 1 ? 0.5 : 0.0);
    if (us < least) {
      least = us;
      plan.slices = slices;
    }
  }
  if (!p.status) p.status = device_status_word();
  if (!p.status) return kErrInternal;
  plan.stall_us = take_armed_stall(NPLK_DEBUG_GEMM);
  if (p.x_type == NPLK_DTYPE_FP32) return by_group<float, 64, false>(s, p, plan);
  if (p.x_type == NPLK_DTYPE_FP16) return by_tokens<__half>(s, p, plan, tokens, tma);
  return by_tokens<__nv_bfloat16>(s, p, plan, tokens, tma);
}

}  // namespace nplk
