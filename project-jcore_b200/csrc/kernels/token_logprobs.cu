// Log probabilities of given tokens with the entropy and the likeliest
// alternatives of each row of logits, and their gradient into the logits.
//
// With m = max l, d = scale (l - m), S = sum e^d, L = log S and t the target:
//   logprob = d[t] - L,  entropy = L - (sum e^d d) / S,
//   p = e^(d - L),  dl = scale (g ([v = t] - p) - h p (d - L + H)).
// Differences to m come first: scale * l alone may leave fp32 (masks of the type's
// lowest value) or lose the last bits of d, and m with L keeps both for the gradient.
#include <algorithm>
#include <type_traits>

#include "act_epilogue.cuh"
#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "typed_io.cuh"

namespace nplk {
namespace {

constexpr float kInf = __builtin_huge_valf(), kLowest = -3.402823466e38f;
constexpr float kMostScale = 0x1p126f;  // times log2 e still finite
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
constexpr unsigned kAll = 0xffffffffu;
constexpr int kMostTop = 32;      // alternatives: one a lane
constexpr int kMostCluster = 8;
constexpr int kCandidates = 512;  // keys put in order at a time
constexpr int kTidBits = 9;       // of a batch's key: order of the maximum, complemented batch, thread

// ---------------------------------------------------------------------------
// Forward: one pass over the logits. A row belongs to a CTA, or to a cluster of up to
// 8 where there are fewer rows than SMs; a thread takes every (threads)-th 16-byte
// pack and keeps its own maximum and sums, which it rescales when the maximum
// grows: with t = scale (l - m) log2 e (its own m) s = sum 2^t, w = sum 2^t t.
//
// The alternatives: a thread's batch is 64 (32) values, whose largest the softmax needs
// anyway; the loop only leaves it in shared memory. The n best elements lie in the n
// batches of largest maxima (of equal ones, those further left), so at the row's end
// those batches are found, read again, and their elements put in order as keys: the
// logit's order in the high half, the complemented index in the low one, so that the larger
// key is the larger logit or, of equal ones, the lower index. (Elements put in order on the way took
// 30 to 70 us more than no alternatives, 43 us, at 2048 x 50021 fp16; batches noted on
// the way against a rising floor 20 to 70.)
// ---------------------------------------------------------------------------
struct LogprobArgs {
  int64_t rows, ld;
  int vocab;
  float scale;
  const int64_t *targets;
  float *logprob, *entropy, *stats;
  int top;
  int64_t *top_ids;
  float *top_logprobs;
};

// Sums relative to a maximum.
struct Part {
  float m, s, w;
};

// Exponents are scale log2 e (l - m), as c (f l - f m): f is 1/2 for scales below 1, under which a
// distance beyond fp32 may count (above, its exponential is 0 and its logarithm -infinity). f is a
// power of two, so nothing else changes.
struct Factors {
  float f, scale, c;  // f; scale / f, and that times log2 e
  __device__ __forceinline__ explicit Factors(float of)
      : f(of < 1.0f ? 0.5f : 1.0f), scale(of < 1.0f ? 2.0f * of : of), c(scale * kLog2e) {}
  // -f m; 0 where there is nothing but -infinity
  __device__ __forceinline__ float origin(float m) const { return m == -kInf ? 0.0f : -f * m; }
  // Kept finite: 0 times a masked logit's would be NaN. Not before the product with c, which may
  // bring any finite number back to 0.
  __device__ __forceinline__ float exponent(float l, float origin) const {
    return at_least(fmaf(l, f, origin) * c, kLowest);
  }
  // scale (l - m) - log_sum
  __device__ __forceinline__ float log_p(float l, float m, float log_sum) const {
    return fmaf(fmaf(l, f, -f * m), scale, -log_sum);
  }
};

// The part relative to `m`, not below its own maximum.
__device__ __forceinline__ Part rebase(const Part &a, float m, const Factors &k) {
  const float d = k.exponent(a.m, k.origin(m)), e = exp2_approx(d);
  // d e first: d s may leave fp32 where e is 0
  return {m, a.s * e, a.w * e + d * e * a.s};
}

// The parts of the 2 * `half` lanes of a group joined, in all of them.
template <int half>
__device__ __forceinline__ Part join_lanes(Part a, const Factors &k) {
  float m = a.m;
#pragma unroll
  for (int o = half; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
  a = rebase(a, m, k);
#pragma unroll
  for (int o = half; o; o >>= 1) {
    a.s += __shfl_xor_sync(kAll, a.s, o);
    a.w += __shfl_xor_sync(kAll, a.w, o);
  }
  return a;
}

// fp32 values (no NaN) in the order of unsigned integers; -0 counts as 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t bits = __float_as_uint(v + 0.0f);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
  return static_cast<uint64_t>(order_of(v)) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_order(uint64_t key) {
  return static_cast<uint32_t>(key >> 32);
}
__device__ __forceinline__ int64_t key_index(uint64_t key) {
  return 0xffffffffu - static_cast<uint32_t>(key);
}

// The rank-th largest (0 the largest) of the lanes' values.
__device__ __forceinline__ uint32_t ranked(uint32_t v, int rank, int lane) {
  uint32_t most = __reduce_max_sync(kAll, v);
  for (; rank > 0; --rank) {
    if (lane == __ffs(__ballot_sync(kAll, v == most)) - 1) v = 0;  // one of them out
    most = __reduce_max_sync(kAll, v);
  }
  return most;
}

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

template <typename T>
struct Batch {
  static constexpr int E = 16 / sizeof(T), U = 8;
  Pack<T, E> p[U];
};

// Largest value of a pack, NaNs left out: 16-bit types two at a time.
template <typename T, int E>
__device__ __forceinline__ float most_of(const Pack<T, E> &p) {
  if constexpr (std::is_same<T, float>::value) {
    return fmaxf(fmaxf(p.e[0], p.e[1]), fmaxf(p.e[2], p.e[3]));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2 *v = reinterpret_cast<const T2 *>(&p);
    const T2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
    return fmaxf(to_float(m.x), to_float(m.y));
  }
}

template <int kThreads>
struct Shelf {
  // maxima of thread batches, kept until they are looked through
  static constexpr int kMaxima = kThreads < 128 ? 32 * kThreads : 4096;
  uint64_t candidates[kCandidates], best[kMostTop];
  uint64_t carried[kMostTop];             // the best of what came before
  float maxima[kMaxima];
  static constexpr int kBatches = kMostTop + kThreads;
  uint32_t batches[kBatches];             // those to be read again
  uint32_t floors[kThreads / 32];
  int found;
};

// Keys that reach a bound come together, and each takes the place that the number above
// it gives. Where they are too many (long runs of equal logits), the n-th of some of them
// is a better bound, and they come together again.
template <int kThreads, typename Gather>
__device__ __forceinline__ void in_order(Shelf<kThreads> &shelf, int top, uint64_t bound,
                                         Gather gather) {
  const int tid = static_cast<int>(threadIdx.x);
  for (;;) {
    if (tid == 0) shelf.found = 0;
    if (tid < kMostTop) shelf.best[tid] = 0;
    __syncthreads();
    gather([&](uint64_t key) {
      if (key < bound) return;
      const int at = atomicAdd(&shelf.found, 1);
      if (at < kCandidates) shelf.candidates[at] = key;
    });
    __syncthreads();
    const int all = shelf.found, n = min(all, kCandidates);
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t key = shelf.candidates[i];
      int place = 0;
#pragma unroll 8
      for (int k = 0; k < n; ++k) place += shelf.candidates[k] > key;
      if (place < top) shelf.best[place] = key;
    }
    __syncthreads();
    if (all <= kCandidates) return;
    bound = shelf.best[top - 1];
    __syncthreads();
  }
}

// The n best of what came before, the lone values and the packs [from, end), whose batches'
// maxima are in the shelf: in order in shelf.best, and carried. Out of line: the loop
// keeps its registers.
template <typename T, int kWarps>
__device__ __noinline__ void collect(const T *xp, int from, int end, int lead, float lone_value,
                                     int lone_index, int top, Shelf<kWarps * 32> &shelf) {
  constexpr int E = Batch<T>::E, U = Batch<T>::U, kThreads = kWarps * 32;
  static_assert(U == 8, "a batch's packs");
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int batches = (end - from + U * kThreads - 1) / (U * kThreads);
  // n batches reach the least of the warps' ceil(n / warps)-th largest of a maximum a lane
  float most = -kInf;
  for (int b = 0; b < batches; ++b) most = fmaxf(most, shelf.maxima[b * kThreads + tid]);
  const uint32_t reach = ranked(order_of(most), (top + kWarps - 1) / kWarps - 1, lane);
  if (lane == 0) shelf.floors[warp] = reach;
  if (tid == 0) shelf.found = 0;
  __syncthreads();
  uint32_t floor = shelf.floors[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) floor = min(floor, shelf.floors[i]);
  float least = fmaxf(value_of(floor), kLowest);
  // two or three times n of them, in general
  if (most >= least)
    for (int b = 0; b < batches; ++b)
      if (shelf.maxima[b * kThreads + tid] >= least) {
        const int at = atomicAdd(&shelf.found, 1);
        if (at < shelf.kBatches) shelf.batches[at] = b * kThreads + tid;
      }
  __syncthreads();
  int count = shelf.found;
  __syncthreads();
  if (count > shelf.kBatches) {  // runs of equal logits
    const auto key_at = [&](int b) -> uint64_t {
      const float m = shelf.maxima[b * kThreads + tid];
      return m == -kInf ? 0
                        : static_cast<uint64_t>(order_of(m)) << 32 |
                              (0x7fffffu - static_cast<uint32_t>(b)) << kTidBits |
                              static_cast<uint32_t>(tid);
    };
    in_order<kThreads>(shelf, top, static_cast<uint64_t>(order_of(least)) << 32, [&](auto take) {
      for (int b = 0; b < batches; ++b) take(key_at(b));
    });
    // the n-th batch; all of its threads' batches with an equal maximum count, their
    // elements lie between one another's
    const uint64_t nth = shelf.best[top - 1] >> kTidBits;
    least = value_of(static_cast<uint32_t>(nth >> (32 - kTidBits)));
    __syncthreads();
    if (tid == 0) shelf.found = 0;
    __syncthreads();
    for (int b = 0; b < batches; ++b)
      if (key_at(b) >> kTidBits >= nth)
        shelf.batches[atomicAdd(&shelf.found, 1)] = b * kThreads + tid;
    __syncthreads();
    count = shelf.found;
    __syncthreads();
  }
  in_order<kThreads>(shelf, top, static_cast<uint64_t>(order_of(least)) << 32, [&](auto take) {
    if (lone_value >= least) take(key_of(lone_value, lone_index));
    if (tid < top && shelf.carried[tid]) take(shelf.carried[tid]);
    // eight lanes to a batch, a pack each
    for (int i = tid >> 3; i < count; i += kThreads / 8) {
      const int batch = static_cast<int>(shelf.batches[i]) / kThreads,
                thread = static_cast<int>(shelf.batches[i]) % kThreads;
      const int at = from + batch * (U * kThreads) + (lane & 7) * kThreads + thread;
      if (at >= end) continue;
      const Pack<T, E> v = load_pack<T, E>(xp + static_cast<int64_t>(at) * E);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float f = to_float(v.e[e]);
        if (f >= least) take(key_of(f, static_cast<uint32_t>(lead + at * E + e)));
      }
    }
  });
  if (tid < kMostTop) shelf.carried[tid] = shelf.best[tid];
  __syncthreads();
}

// kTop: with alternatives. The launch's CTAs are whole clusters of `cluster`. A row's end is a
// third of a CTA's time then, under which others load: 28 warps an SM (2048 x 50021 fp16 with
// five 50.8 us; 24 warps 55.4, 32, which spill, 58.9; 1024 x 128000 bf16 with 20 60, 73, 68).
template <typename T, bool kTop, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps == 16 ? 1 : (kTop ? 28 : 32) / kWarps)
    token_logprobs_kernel(LogprobArgs p, const T *logits, int cluster) {
  using B = Batch<T>;
  constexpr int E = B::E, U = B::U, kThreads = kWarps * 32;
  static_assert(kThreads <= 1 << kTidBits && kMostCluster * kMostTop <= kCandidates, "keys");
  constexpr int kLook = Shelf<kThreads>::kMaxima / kThreads;  // batches after which the maxima are looked through
  __shared__ Part warp_part[kWarps];
  // what the cluster's CTAs hand to its first: two rows' worth, so that one barrier a
  // row keeps the next row's writes off this row's reads
  __shared__ Part cta_part[2][kMostCluster];
  __shared__ uint64_t cta_list[2][kTop ? kMostCluster * kMostTop : 1];
  __shared__ __align__(16) uint8_t shelf_room[kTop ? sizeof(Shelf<kThreads>) : 16];
  Shelf<kThreads> &shelf = *reinterpret_cast<Shelf<kThreads> *>(shelf_room);
  griddep_wait();
  griddep_launch_dependents();

  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(blockIdx.x) % cluster;
  const Factors k(p.scale);
  if (cluster > 1) {  // the first CTA has started before anything is stored into it
    cluster_arrive_relaxed();
    cluster_wait();
  }

  int parity = 0;
  for (int64_t row = blockIdx.x / cluster; row < p.rows; row += gridDim.x / cluster, parity ^= 1) {
    const T *x = logits + row * p.ld;
    // up to E - 1 values before the first whole pack, and behind the last
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    const int lead = min(mis ? E - mis : 0, p.vocab);
    const int packs = (p.vocab - lead) / E, tail = lead + packs * E;
    const int j0 = static_cast<int>(static_cast<int64_t>(packs) * rank / cluster);
    const int j1 = static_cast<int>(static_cast<int64_t>(packs) * (rank + 1) / cluster);
    const T *xp = x + lead;

    Part mine{-kInf, 0.0f, 0.0f};
    const auto load = [&](B &b, int j, int here) {
      const T *from = xp + static_cast<int64_t>(j + tid) * E;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < here) b.p[u] = load_pack<T, E>(from + u * (kThreads * E));
    };

    // the target's logit, long before it is needed
    int64_t target = -1;
    float target_logit = 0.0f;
    if (p.logprob && rank == 0 && tid == 0) {
      target = p.targets[row];
      if (target >= 0 && target < p.vocab) target_logit = to_float(x[target]);
      else target = -1;
    }
    // the lone values, by the first CTA's first warp
    const int lone_index = lane < lead ? lane : tail + lane - lead;
    const bool lone = rank == 0 && warp == 0 && lane < lead + p.vocab - tail;
    const float lone_value = lone ? to_float(x[lone_index]) : -kInf;
    if (lone) {
      mine.m = fmaxf(lone_value, -kInf);  // the maximum of a NaN and nothing
      const float d = k.exponent(lone_value, k.origin(mine.m));
      mine.s = exp2_approx(d);
      mine.w = mine.s * d;
    }

    if (kTop && tid < kMostTop) shelf.carried[tid] = 0;  // (seen by collect past its barriers)
    int from = j0;  // of the maxima held
    for (int j = j0; j < j1; j += U * kThreads) {
      B now;
      const bool whole = j + U * kThreads <= j1;
      const int here = min(U, (j1 - j - tid + kThreads - 1) / kThreads);  // packs of this thread
      load(now, j, whole ? U : here);
      float most = -kInf;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (whole || u < here) most = fmaxf(most, most_of(now.p[u]));
      if (most > mine.m) mine = rebase(mine, most, k);
      const float origin = k.origin(mine.m);
      float ss[2] = {}, ww[2] = {};
      const auto add = [&](const Pack<T, E> &p) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float t = k.exponent(to_float(p.e[e]), origin);
          const float r = exp2_approx(t);
          ss[e & 1] += r;
          ww[e & 1] = fmaf(r, t, ww[e & 1]);
        }
      };
      if (whole) {
#pragma unroll
        for (int u = 0; u < U; ++u) add(now.p[u]);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u < here) add(now.p[u]);
      }
      mine.s += ss[0] + ss[1];
      mine.w += ww[0] + ww[1];
      if constexpr (kTop) {
        const int batch = (j - from) / (U * kThreads);
        shelf.maxima[batch * kThreads + tid] = most;
        if (batch == kLook - 1 && j + U * kThreads < j1) {
          collect<T, kWarps>(xp, from, j + U * kThreads, lead, -kInf, 0, p.top, shelf);
          from = j + U * kThreads;
        }
      }
    }

    // the warp's, then the CTA's, then the cluster's sums
    mine = join_lanes<16>(mine, k);
    if (lane == 0) warp_part[warp] = mine;
    __syncthreads();
    if constexpr (kTop)
      collect<T, kWarps>(xp, from, j1, lead, lone ? lone_value : -kInf, lone_index, p.top, shelf);
    Part total{-kInf, 0.0f, 0.0f};
    if (warp == 0) {
      if (lane < kWarps) total = warp_part[lane];
      total = join_lanes<kWarps / 2>(total, k);
    }
    if (cluster > 1) {
      if (tid == 0) {
        const uint32_t to = mapa_shared(smem_u32(&cta_part[parity][rank]), 0u);
        st_shared_cluster_f32(to, total.m);
        st_shared_cluster_f32(to + 4, total.s);
        st_shared_cluster_f32(to + 8, total.w);
      }
      if (kTop && tid < kMostTop)
        st_cluster_u64(mapa_shared(smem_u32(&cta_list[parity][rank * kMostTop + tid]), 0u),
                       shelf.best[tid]);
      cluster_sync();
      if (rank != 0) continue;
      if (warp == 0) {
        total = lane < cluster ? cta_part[parity][lane] : Part{-kInf, 0.0f, 0.0f};
        total = join_lanes<kMostCluster / 2>(total, k);
      }
      if constexpr (kTop) {
        uint64_t most = 0;  // n keys reach any CTA's n-th
        for (int i = 0; i < cluster; ++i)
          most = max(most, cta_list[parity][i * kMostTop + p.top - 1]);
        in_order<kThreads>(shelf, p.top, max(most, uint64_t(1)), [&](auto take) {
          for (int i = tid; i < cluster * kMostTop; i += kThreads) take(cta_list[parity][i]);
        });
      }
    }
    if (warp == 0) {
      if (kWarps < 32) {  // what lane 0 has
        total.m = __shfl_sync(kAll, total.m, 0);
        total.s = __shfl_sync(kAll, total.s, 0);
        total.w = __shfl_sync(kAll, total.w, 0);
      }
      const float log_sum = logf(total.s);
      const bool bad = total.s != total.s;  // a NaN or +infinity in the row
      if (lane == 0) {
        if (p.stats) {
          p.stats[2 * row] = bad ? log_sum : total.m;  // (the maximum has left out NaNs)
          p.stats[2 * row + 1] = log_sum;
        }
        if (p.entropy)
          p.entropy[row] = total.s == 0.0f ? 0.0f : log_sum - kLn2 * (total.w / total.s);
        if (p.logprob) {
          p.logprob[row] = target < 0              ? 0.0f
                           : bad                   ? log_sum
                           : target_logit == -kInf ? -kInf
                                                   : k.log_p(target_logit, total.m, log_sum);
        }
      }
      if (kTop && lane < p.top) {
        const uint64_t key = shelf.best[lane];
        const int64_t to = row * p.top + lane;
        p.top_ids[to] = key && !bad ? key_index(key) : -1;
        p.top_logprobs[to] = bad ? log_sum
                             : key ? k.log_p(value_of(key_order(key)), total.m, log_sum)
                                   : -kInf;
      }
    }
    __syncthreads();  // the next row's floors, lists and best
  }
}

// ---------------------------------------------------------------------------
// Gradient: dl = p (A + B t) + [v = target] scale g with t = (d - L) log2 e, p = 2^t,
// A = -scale (g + h H), B = -scale h ln 2. Under scales above kMostInner (kLast) the scale comes
// last instead: where p is 0, or A p and scale g cancel, they must be finite (for every scale it
// would cost 2% at 4096 x 32000 bf16, 8% at 8192 x 500). CTAs go round runs of packs of a row; a run's
// logits load under the one before, and its row's numbers, which say whether they are
// needed at all, one run earlier still. Bound by memory: 4096 x 32000 bf16 takes 92 us, of 80
// for its bytes (121 us with a CTA a run, which waited for one and then for the other).
// Short rows go to CTAs of one warp.
// ---------------------------------------------------------------------------
struct LogprobGradArgs {
  int64_t ld, ldd;
  int vocab;
  float scale;
  const int64_t *targets;
  const float *stats, *entropy, *d_logprob, *d_entropy;
};

constexpr int kGradPacks = 4;
constexpr float kMostInner = 0x1p32f;  // A + B t and scale g are finite for g and h up to 2^85

// What a run needs to know of its row.
struct GradRow {
  int64_t row, target;
  float g, h, m, log_sum, entropy;
  int first;  // pack
};

template <typename T, int E, int kThreads, bool kLast>
__global__ void __launch_bounds__(kThreads, 3 * 256 / kThreads)
    token_logprobs_grad_kernel(LogprobGradArgs p, const T *logits, T *dlogits, uint32_t runs,
                               FastDiv per_row) {
  griddep_wait();
  griddep_launch_dependents();
  const int tid = static_cast<int>(threadIdx.x);
  const Factors k(p.scale);
  const auto row_of = [&](uint32_t run) {
    GradRow r{};
    if (run >= runs) return r;
    const uint32_t row = fdiv(run, per_row);
    r.row = row;
    r.first = static_cast<int>(run - row * per_row.d) * (kThreads * kGradPacks);
    r.target = p.targets ? p.targets[row] : -1;
    if (p.d_logprob) r.g = p.d_logprob[row];
    if (p.d_entropy) {
      r.h = p.d_entropy[row];
      r.entropy = p.entropy[row];
    }
    r.m = p.stats[2 * static_cast<int64_t>(row)];
    r.log_sum = p.stats[2 * static_cast<int64_t>(row) + 1];
    return r;
  };
  const auto asked = [&](const GradRow &r) { return r.target >= 0 && r.target < p.vocab; };
  // nothing asked of the row, or nothing in it
  const auto zeros = [&](const GradRow &r) {
    return ((r.g == 0.0f || !asked(r)) && r.h == 0.0f) || (r.m == -kInf && r.log_sum == -kInf);
  };
  const auto lead_of = [&](const T *x) {
    const int mis = E == 1 ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    return min(mis ? E - mis : 0, p.vocab);
  };
  struct Packs {
    Pack<T, E> v[kGradPacks];
  };
  const auto load = [&](const GradRow &r, uint32_t run) {
    Packs q;
    const T *x = logits + r.row * p.ld;
    const int lead = lead_of(x), packs = (p.vocab - lead) / E;
    if (run < runs && !zeros(r)) {
#pragma unroll
      for (int u = 0; u < kGradPacks; ++u) {
        const int at = r.first + u * kThreads + tid;
        if (at < packs) q.v[u] = load_pack<T, E>(x + lead + static_cast<int64_t>(at) * E);
      }
    }
    return q;
  };

  const uint32_t step = gridDim.x;
  uint32_t run = blockIdx.x;
  GradRow now = row_of(run), next = row_of(run + step);
  Packs in = load(now, run);
  for (; run < runs; run += step) {
    const Packs in_next = load(next, run + step);
    const GradRow after = row_of(run + 2 * step);
    const T *x = logits + now.row * p.ld;
    T *dx = dlogits + now.row * p.ldd;
    const bool none = zeros(now), hit_row = asked(now);
    const float g = hit_row ? now.g : 0.0f, h = now.h;
    const float inner = kLast ? 1.0f : p.scale;
    const float a = -inner * (h != 0.0f ? fmaf(h, now.entropy, g) : g);
    const float2 aa = both(a), bb = both(-inner * h * kLn2);
    const float2 f = both(k.f), c = both(k.c), base = both(-k.f * now.m),
                 ll = both(-now.log_sum * kLog2e);
    const float hot = inner * g;
    const int lead = lead_of(x), packs = (p.vocab - lead) / E, tail = lead + packs * E;
    const int hit = hit_row ? static_cast<int>(now.target) : -1;
    const auto pairs = [&](float2 v) {
      // (2^-1000 is 0, and 0 times a finite number too; a masked logit's t is -infinity up to here)
      const float2 t = at_least(fma2(fma2(v, f, base), c, ll), -1000.0f);
      const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
      return mul2(e, fma2(t, bb, aa));
    };
#pragma unroll
    for (int u = 0; u < kGradPacks; ++u) {
      const int at = now.first + u * kThreads + tid;
      if (at >= packs) break;
      const int index = lead + at * E;
      float v[E];
      if (none) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.0f;
      } else {
        float2 q[(E + 1) / 2];
        unpack_pairs(in.v[u], q);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 r = pairs(q[e / 2]);
          v[e] = r.x;
          if (E > 1) v[e + 1] = r.y;
        }
        if (hit >= index && hit < index + E) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (hit == index + e) v[e] += hot;
        }
        if constexpr (kLast) {
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] *= p.scale;
        }
      }
      store_pack(dx + index, pack<T, E>(v));
    }
    // the lone values beside the packs, by the row's first run
    if (now.first == 0 && tid < lead + p.vocab - tail) {
      const int index = tid < lead ? tid : tail + tid - lead;
      float v = 0.0f;
      if (!none) {
        v = pairs(both(to_float(x[index]))).x;
        if (index == hit) v += hot;
        if (kLast) v *= p.scale;
      }
      dx[index] = from_float<T>(v);
    }
    now = next;
    next = after;
    in = in_next;
  }
}

template <typename T>
auto pick_forward(bool top, int warps) {
  switch (warps) {
    case 1:
      return top ? token_logprobs_kernel<T, true, 1> : token_logprobs_kernel<T, false, 1>;
    case 4:
      return top ? token_logprobs_kernel<T, true, 4> : token_logprobs_kernel<T, false, 4>;
    default:
      return top ? token_logprobs_kernel<T, true, 16> : token_logprobs_kernel<T, false, 16>;
  }
}

// One warp for rows of up to four packs a lane (8192 x 1000 bf16 11.3 us, by four 25.9; 500 x 500 3.2,
// 3.4), else four, or 16 where rows do not fill the SMs (256 x 128000 bf16 22.0 us, by four 25.8;
// 297, where the rule takes four, 27.7, by 16 29.5, with five alternatives 30.7, 38.3); then clusters too,
// while each CTA has two packs a thread and the cluster's double takes up to 3/4 of the SMs (us at
// 128000 bf16 for clusters of 1, 2, 4, 8: one row 8.9, 6.4, 4.6, 4.0; 8 rows 9.2, 6.5, 4.8, 4.2; 16 10.6,
// 7.3, 5.4, 8.2; 37 11.1, 7.8, 10.1, 12.5; 55 11.2, 8.2, 10.7, 16.4; 111 11.7, 15.3, 19.7, 31.2). A cluster
// too many costs more than one too few, but short of these borders the next larger form would win: 28
// rows in fours 5.8 (in twos 7.6), 64 in twos 8.3 (11.3); so would fewer warps for shorter rows, 256 x
// 9000 with five by four 8.2 (13.7), 8192 x 1100 by one 12.3 (28.3). Eight warps a row instead of
// four were slower (measured with a slower loop: 2048 x 50021 fp16 48 us against 43, with five
// alternatives 65 against 51; 4096 x 32000 bf16 88 against 65; 1024 x 128000 bf16 with 20 73 against 61).
template <typename T>
int run_forward(cudaStream_t s, const LogprobArgs &p, const T *logits) {
  constexpr int E = 16 / sizeof(T);
  const int64_t packs = std::max(1, p.vocab / E), sms = sm_count();
  const int warps = packs <= 128 ? 1 : packs > 1024 && p.rows <= 2 * sms ? 16 : 4;
  int cluster = 1;
  while (warps == 16 && cluster < kMostCluster && p.rows * cluster * 8 <= sms * 3 &&
         packs >= 2 * cluster * 16 * 32 * 2)
    cluster *= 2;
  const int64_t rows = std::min<int64_t>(p.rows, sms * 128);
  auto *fn = pick_forward<T>(p.top > 0, warps);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster));
  cfg.blockDim = dim3(static_cast<unsigned>(warps * 32));
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  count_launch();
  return map_cuda_error(cudaLaunchKernelEx(&cfg, fn, p, logits, cluster));
}

template <typename T, int E, bool kLast>
auto pick_gradient(int threads) {
  return threads == 32 ? token_logprobs_grad_kernel<T, E, 32, kLast>
                       : token_logprobs_grad_kernel<T, E, 256, kLast>;
}

template <typename T>
int run_gradient(cudaStream_t s, int64_t rows, const LogprobGradArgs &p, const T *logits,
                 T *dlogits) {
  constexpr int E = 16 / sizeof(T);
  // Packs need rows of the same alignment on both sides. A pitch that changes it from row to
  // row changes it on both alike if the pitches differ by whole packs.
  const bool alike = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) %
                             16 == 0 &&
                     (rows == 1 || (p.ld - p.ldd) % E == 0);
  const int packs = p.vocab / (alike ? E : 1), threads = packs <= 32 * kGradPacks ? 32 : 256;
  const int64_t per_row = std::max<int64_t>(1, ceil_div(packs, threads * kGradPacks));
  auto *fn = p.scale > kMostInner
                 ? (alike ? pick_gradient<T, E, true>(threads) : pick_gradient<T, 1, true>(threads))
                 : (alike ? pick_gradient<T, E, false>(threads) : pick_gradient<T, 1, false>(threads));
  // rows of a launch: their runs are counted in 31 bits
  const int64_t most = std::max<int64_t>(1, (int64_t(1) << 30) / per_row);
  for (int64_t r = 0; r < rows; r += most) {
    LogprobGradArgs q = p;
    if (q.targets) q.targets += r;
    if (q.d_logprob) q.d_logprob += r;
    if (q.d_entropy) q.d_entropy += r;
    if (q.entropy) q.entropy += r;
    q.stats += 2 * r;
    const int64_t runs = std::min(most, rows - r) * per_row;
    const int64_t grid = std::min<int64_t>(runs, static_cast<int64_t>(sm_count()) * (3 * 256 / threads));
    const int rc = launch_programmatic(fn, dim3(static_cast<unsigned>(grid)), dim3(static_cast<unsigned>(threads)), 0, s,
                                       q, logits + r * p.ld, dlogits + r * p.ldd,
                                       static_cast<uint32_t>(runs),
                                       make_fastdiv(static_cast<uint32_t>(per_row)));
    if (rc) return rc;
  }
  return kOk;
}

// Checks shared by both directions.
int check(int64_t rows, int64_t vocab, int dtype, const void *logits, int64_t ld, float scale) {
  const int size = dtype_bytes(dtype);
  if (rows < 1 || vocab < 1 || !size || !logits || ld < vocab || !(scale > 0.0f) ||
      !(scale <= kMostScale) || reinterpret_cast<uintptr_t>(logits) % size)
    return kErrInvalidArg;
  if (vocab >= (int64_t(1) << 31) - 65536 || rows > (int64_t(1) << 40)) return kErrUnsupported;
  return kOk;
}

bool misaligned(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_token_logprobs(void *stream, int64_t rows, int64_t vocab, int dtype,
                                   const void *logits, int64_t ld, float scale,
                                   const int64_t *targets, float *logprob, float *entropy,
                                   float *stats, int n_top, int64_t *top_ids,
                                   float *top_logprobs) {
  const int rc = check(rows, vocab, dtype, logits, ld, scale);
  if (rc) return rc;
  if (n_top < 0 || (n_top > 0 && (!top_ids || !top_logprobs)) || (logprob && !targets) ||
      (!logprob && !entropy && !stats && n_top == 0))
    return kErrInvalidArg;
  if (misaligned(targets, 8) || misaligned(logprob, 4) || misaligned(entropy, 4) ||
      misaligned(stats, 4) || misaligned(top_ids, 8) || misaligned(top_logprobs, 4))
    return kErrInvalidArg;
  if (n_top > kMostTop) return kErrUnsupported;
  const LogprobArgs p{rows,    ld,    static_cast<int>(vocab), scale,   targets,     logprob,
                      entropy, stats, n_top,                   top_ids, top_logprobs};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == NPLK_DTYPE_FP32) return run_forward(s, p, static_cast<const float *>(logits));
  if (dtype == NPLK_DTYPE_FP16) return run_forward(s, p, static_cast<const __half *>(logits));
  return run_forward(s, p, static_cast<const __nv_bfloat16 *>(logits));
}

extern "C" int nplk_token_logprobs_backward(void *stream, int64_t rows, int64_t vocab, int dtype,
                                            const void *logits, int64_t ld, float scale,
                                            const int64_t *targets, const float *stats,
                                            const float *entropy, const float *d_logprob,
                                            const float *d_entropy, void *dlogits, int64_t ldd) {
  const int rc = check(rows, vocab, dtype, logits, ld, scale);
  if (rc) return rc;
  if (!stats || !dlogits || ldd < vocab || (!d_logprob && !d_entropy) || (d_logprob && !targets) ||
      (d_entropy && !entropy) || (logits == dlogits && ld != ldd && rows > 1))
    return kErrInvalidArg;
  if (misaligned(dlogits, dtype_bytes(dtype)) || misaligned(targets, 8) || misaligned(stats, 4) ||
      misaligned(entropy, 4) || misaligned(d_logprob, 4) || misaligned(d_entropy, 4))
    return kErrInvalidArg;
  const LogprobGradArgs p{ld,    ldd,     static_cast<int>(vocab), scale,    targets,
                          stats, entropy, d_logprob,               d_entropy};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == NPLK_DTYPE_FP32)
    return run_gradient(s, rows, p, static_cast<const float *>(logits), static_cast<float *>(dlogits));
  if (dtype == NPLK_DTYPE_FP16)
    return run_gradient(s, rows, p, static_cast<const __half *>(logits), static_cast<__half *>(dlogits));
  return run_gradient(s, rows, p, static_cast<const __nv_bfloat16 *>(logits),
                      static_cast<__nv_bfloat16 *>(dlogits));
}
