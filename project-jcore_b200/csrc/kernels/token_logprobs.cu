// Log probabilities of given tokens with the entropy and the likeliest
// alternatives of each row of logits, and their gradient into the logits.
//
// With m = max l, d = scale (l - m), S = sum e^d, L = log S and t the target:
//   logprob = d[t] - L,  entropy = L - (sum e^d d) / S,
//   p = e^(d - L),  dl = scale (g ([v = t] - p) - h p (d - L + H)).
// Differences to m come first: scale * l alone may leave fp32 (masks of the type's
// lowest value) or lose the last bits of d, and m with L keeps both for the gradient.
#include <algorithm>

#include "act_epilogue.cuh"
#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "typed_io.cuh"

namespace nplk {
namespace {

constexpr float kInf = __builtin_huge_valf(), kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
constexpr unsigned kAll = 0xffffffffu;
constexpr int kMostTop = 32;      // alternatives: one a lane
constexpr int kMostWarps = 16, kMostCluster = 8;

// ---------------------------------------------------------------------------
// Forward: one pass over the logits. A row belongs to a CTA, or to a cluster of up to
// 8 where there are fewer rows than SMs; a thread takes every (threads)-th 16-byte
// pack and keeps its own maximum and sums, which it rescales when the maximum
// grows: with u = l - m (its own m) s = sum e^(scale u), w = sum e^(scale u) u.
//
// The alternatives ride along. Each warp keeps the 32 best it has seen, one a lane,
// ordered by key: the logit's order in the high half, the complemented index in the
// low one, so that the larger key is the larger logit or, of equal ones, the lower
// index. What a logit must reach to be looked at is `floor`, the larger of the warp's own
// n-th key and the least of the warps' ceil(n / warps)-th keys (at least n elements of the
// row reach that one). It is compared with the largest of a thread's 32 (16) values,
// which the softmax needs anyway.
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

struct Part {
  float m, s, w;
};

// Both sums relative to the larger maximum. c = scale * log2 e.
__device__ __forceinline__ Part join(const Part &a, const Part &b, float c) {
  Part r;
  r.m = fmaxf(a.m, b.m);
  const float base = r.m == -kInf ? 0.0f : r.m;  // nothing but -infinity: u stays -infinity
  const float ua = at_least(a.m - base, kLowest), ub = at_least(b.m - base, kLowest);
  const float ea = exp2_approx(ua * c), eb = exp2_approx(ub * c);
  r.s = a.s * ea + b.s * eb;
  // u e first: u s may leave fp32 where e is 0
  r.w = (a.w * ea + ua * ea * a.s) + (b.w * eb + ub * eb * b.s);
  return r;
}

__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
  const uint32_t bits = __float_as_uint(v + 0.0f);  // -0 counts as 0
  const uint32_t order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  return static_cast<uint64_t>(order) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t order = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ int64_t key_index(uint64_t key) {
  return 0xffffffffu - static_cast<uint32_t>(key);
}

// Puts `key` (the same in all lanes) in its place of the warp's descending list.
__device__ __forceinline__ void insert(uint64_t &mine, uint64_t key, int lane) {
  const int at = __popc(__ballot_sync(kAll, mine > key));
  const uint64_t above = __shfl_up_sync(kAll, mine, 1);
  if (lane > at) mine = above;
  if (lane == at) mine = key;
}

// The rank-th largest (0 the largest) of the lanes' values, none of them NaN.
__device__ __forceinline__ float ranked(float v, int rank, int lane) {
  int before = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float other = __shfl_sync(kAll, v, j);
    before += other > v || (other == v && j < lane);
  }
  return __shfl_sync(kAll, v, __ffs(__ballot_sync(kAll, before == rank)) - 1);
}

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

template <typename T>
struct Batch {
  static constexpr int E = 16 / sizeof(T), U = 4, kValues = E * U;
  Pack<T, E> p[U];
};

// kTop: with alternatives. The launch's CTAs are whole clusters of `cluster`.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kMostWarps * 32)
    token_logprobs_kernel(LogprobArgs p, const T *logits, int cluster) {
  using B = Batch<T>;
  constexpr int E = B::E, U = B::U;
  __shared__ Part warp_part[kMostWarps];
  __shared__ uint64_t lists[kTop ? kMostWarps * kMostTop : 1];
  __shared__ uint64_t floors[kTop ? kMostWarps : 1];
  // what the cluster's CTAs hand to its first: two rows' worth, so that one barrier a
  // row keeps the next row's writes off this row's reads
  __shared__ Part cta_part[2][kMostCluster];
  __shared__ uint64_t cta_list[2][kTop ? kMostCluster * kMostTop : 1];
  __shared__ uint64_t best[kMostTop];
  griddep_wait();
  griddep_launch_dependents();

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int threads = blockDim.x, warps = threads >> 5;
  const int rank = static_cast<int>(blockIdx.x) % cluster;
  const float c = p.scale * kLog2e;
  const int share = kTop ? (p.top + warps - 1) / warps : 0;
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
    uint64_t list = 0, floor = key_of(kLowest, 0xffffffffu);  // lists hold no -infinity
    float floor_value = kLowest;
    const auto raise = [&](uint64_t to) {
      if (to > floor) {
        floor = to;
        floor_value = key_value(to);
      }
    };

    // one value, or none: lane's own
    const auto offer = [&](float v, int index, bool here) {
      uint64_t key = here && v >= floor_value ? key_of(v, index) : 0;
      unsigned want = __ballot_sync(kAll, key >= floor);
      while (want) {
        const int src = __ffs(want) - 1;
        want &= want - 1;
        const uint64_t k = __shfl_sync(kAll, key, src);
        if (k < floor) continue;
        insert(list, k, lane);
        raise(__shfl_sync(kAll, list, p.top - 1));
      }
    };

    bool first = true;
    const int last_batch = j0 + ((j1 - j0) + U * threads - 1) / (U * threads) * (U * threads);
    const auto load = [&](B &b, int j) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = j + u * threads + static_cast<int>(threadIdx.x);
        if (at < j1) b.p[u] = load_pack<T, E>(xp + static_cast<int64_t>(at) * E);
        else
#pragma unroll
          for (int e = 0; e < E; ++e) b.p[u].e[e] = from_float<T>(-kInf);
      }
    };
    B next;
    if (j0 < last_batch) load(next, j0);

    // the lone values, by the first CTA's first warp
    if (rank == 0 && warp == 0) {
      const bool here = lane < lead + p.vocab - tail;
      const int index = lane < lead ? lane : tail + lane - lead;
      const float v = here ? to_float(x[index]) : -kInf;
      if (here) {
        mine.m = v == v ? v : -kInf;  // the maximum of a NaN and nothing
        const float u = at_least(v - (mine.m == -kInf ? 0.0f : mine.m), kLowest);
        mine.s = exp2_approx(u * c);
        mine.w = mine.s * u;
      }
      if (kTop) offer(v, index, here);
    }

    for (int j = j0; j < last_batch; j += U * threads) {
      const B now = next;
      if (j + U * threads < last_batch) load(next, j + U * threads);
      float most = -kInf;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) most = fmaxf(most, to_float(now.p[u].e[e]));
      if (most > mine.m) {
        const float u = at_least(mine.m - most, kLowest), e = exp2_approx(u * c);
        mine.w = mine.w * e + u * e * mine.s;
        mine.s *= e;
        mine.m = most;
      }
      const float2 base = both(mine.m == -kInf ? 0.0f : -mine.m), cc = both(c);
      float2 s = make_float2(0.0f, 0.0f), w = s;
#pragma unroll
      for (int q = 0; q < U; ++q) {
        float2 v[E / 2];
        unpack_pairs(now.p[q], v);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          const float2 u = at_least(add2(v[e], base), kLowest);
          const float2 t = mul2(u, cc);
          const float2 r = make_float2(exp2_approx(t.x), exp2_approx(t.y));
          s = add2(s, r);
          w = fma2(r, u, w);
        }
      }
      mine.s += s.x + s.y;
      mine.w += w.x + w.y;
      if constexpr (kTop) {
        if (first) {
          // n elements reach the least of the warps' share-th largest: each is the
          // maximum of another thread's values
          const uint64_t reach = key_of(ranked(most, share - 1, lane), 0xffffffffu);
          if (lane == 0) floors[warp] = reach;
          __syncthreads();
          uint64_t least = floors[0];
          for (int i = 1; i < warps; ++i) least = min(least, floors[i]);
          raise(least);
          first = false;
        } else {
          uint64_t least = *reinterpret_cast<volatile uint64_t *>(&floors[0]);
          for (int i = 1; i < warps; ++i)
            least = min(least, *reinterpret_cast<volatile uint64_t *>(&floors[i]));
          raise(__shfl_sync(kAll, least, 0));  // the lanes may have read at different times
        }
        unsigned some = __ballot_sync(kAll, most >= floor_value);
        if (some) {
          // many at once (rising logits): the n-th of the lanes' maxima first
          if (__popc(some) > 8 && __popc(some) >= p.top) {
            raise(key_of(ranked(most, p.top - 1, lane), 0xffffffffu));
          }
          uint32_t mask = 0;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e)
              mask |= static_cast<uint32_t>(to_float(now.p[u].e[e]) >= floor_value) << (u * E + e);
          while (__any_sync(kAll, mask != 0)) {
            const int bit = __ffs(mask) - 1;
            const int at = j + bit / E * threads + static_cast<int>(threadIdx.x);
            const int index = lead + at * E + bit % E;
            offer(mask ? to_float(x[index]) : 0.0f, index, mask != 0);
            mask &= mask - 1;
          }
          const uint64_t reach = __shfl_sync(kAll, list, share - 1);
          if (lane == 0 && reach > floors[warp])
            *reinterpret_cast<volatile uint64_t *>(&floors[warp]) = reach;
        }
      }
    }

    // the warp's, then the CTA's, then the cluster's sums
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      Part other;
      other.m = __shfl_xor_sync(kAll, mine.m, o);
      other.s = __shfl_xor_sync(kAll, mine.s, o);
      other.w = __shfl_xor_sync(kAll, mine.w, o);
      mine = join(mine, other, c);
    }
    if (lane == 0) warp_part[warp] = mine;
    if (kTop) lists[warp * kMostTop + lane] = list;
    if (kTop && threadIdx.x < kMostTop) best[threadIdx.x] = 0;
    __syncthreads();
    // the place of each key among all: those above it in its own list, and in the others
    const auto merge = [&](const uint64_t *from, int count) {
      for (int i = threadIdx.x; i < count * kMostTop; i += threads) {
        const int own = i / kMostTop;
        const uint64_t key = from[i];
        int place = i % kMostTop;
        if (key == 0 || place >= p.top) continue;
        for (int l = 0; l < count && place < p.top; ++l) {
          if (l == own) continue;
          const uint64_t *other = from + l * kMostTop;
          for (int k = 0; k < p.top && other[k] > key; ++k) ++place;
        }
        if (place < p.top) best[place] = key;
      }
      __syncthreads();
    };
    if (kTop) merge(lists, warps);
    Part total = warp_part[0];
    for (int i = 1; i < warps; ++i) total = join(total, warp_part[i], c);
    if (cluster > 1) {
      if (threadIdx.x == 0) {
        const uint32_t to = mapa_shared(smem_u32(&cta_part[parity][rank]), 0u);
        st_shared_cluster_f32(to, total.m);
        st_shared_cluster_f32(to + 4, total.s);
        st_shared_cluster_f32(to + 8, total.w);
      }
      if (kTop && threadIdx.x < kMostTop)
        st_cluster_u64(mapa_shared(smem_u32(&cta_list[parity][rank * kMostTop + threadIdx.x]), 0u),
                       best[threadIdx.x]);
      cluster_sync();
      if (rank != 0) continue;
      total = cta_part[parity][0];
      for (int i = 1; i < cluster; ++i) total = join(total, cta_part[parity][i], c);
      if (kTop) {
        if (threadIdx.x < kMostTop) best[threadIdx.x] = 0;
        __syncthreads();
        merge(cta_list[parity], cluster);
      }
    }
    const float log_sum = logf(total.s);
    const bool bad = total.s != total.s;  // a NaN or +infinity in the row
    if (threadIdx.x == 0) {
      if (p.stats) {
        p.stats[2 * row] = total.m;
        p.stats[2 * row + 1] = log_sum;
      }
      if (p.entropy)
        p.entropy[row] = total.s == 0.0f ? 0.0f : log_sum - p.scale * (total.w / total.s);
      if (p.logprob) {
        const int64_t t = p.targets[row];
        float v = 0.0f;
        if (t >= 0 && t < p.vocab) {
          const float l = to_float(x[t]);
          v = bad ? log_sum : l == -kInf ? -kInf : fmaf(l - total.m, p.scale, -log_sum);
        }
        p.logprob[row] = v;
      }
    }
    if (kTop && static_cast<int>(threadIdx.x) < p.top) {
      const uint64_t key = best[threadIdx.x];
      const int64_t to = row * p.top + threadIdx.x;
      p.top_ids[to] = key && !bad ? key_index(key) : -1;
      p.top_logprobs[to] =
          bad ? log_sum : key ? fmaf(key_value(key) - total.m, p.scale, -log_sum) : -kInf;
    }
    __syncthreads();  // the next row's floors, lists and best
  }
}

// ---------------------------------------------------------------------------
// Gradient: dl = p (A + B t) + [v = target] scale g with t = (d - L) log2 e, p = 2^t,
// A = -scale (g + h H), B = -scale h ln 2. A CTA takes a run of packs of one row.
// ---------------------------------------------------------------------------
struct LogprobGradArgs {
  int64_t rows, ld, ldd;
  int vocab;
  float scale;
  const int64_t *targets;
  const float *stats, *entropy, *d_logprob, *d_entropy;
};

constexpr int kGradThreads = 256, kGradPacks = 4;

template <typename T, int E>
__global__ void __launch_bounds__(kGradThreads)
    token_logprobs_grad_kernel(LogprobGradArgs p, const T *logits, T *dlogits, int64_t runs,
                               int per_row) {
  griddep_wait();
  griddep_launch_dependents();
  for (int64_t run = blockIdx.x; run < runs; run += gridDim.x) {
    const int64_t row = run / per_row;
    const T *x = logits + row * p.ld;
    T *dx = dlogits + row * p.ldd;
    const int64_t target = p.targets ? p.targets[row] : -1;
    const bool asked = target >= 0 && target < p.vocab;
    const float g = asked && p.d_logprob ? p.d_logprob[row] : 0.0f;
    const float h = p.d_entropy ? p.d_entropy[row] : 0.0f;
    const float m = p.stats[2 * row], log_sum = p.stats[2 * row + 1];
    // nothing asked of the row, or nothing in it
    const bool zeros = (g == 0.0f && h == 0.0f) || (m == -kInf && log_sum == -kInf);
    const float a = -p.scale * (h != 0.0f ? fmaf(h, p.entropy[row], g) : g);
    const float2 aa = both(a), bb = both(-p.scale * h * kLn2);
    const float2 c = both(p.scale * kLog2e), base = both(-m), ll = both(-log_sum * kLog2e);
    const float hot = p.scale * g;
    const int mis = E == 1 ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    const int lead = min(mis ? E - mis : 0, p.vocab);
    const int packs = (p.vocab - lead) / E, tail = lead + packs * E;
    const int hit = asked ? static_cast<int>(target) : -1;
    const auto pairs = [&](float2 v) {
      const float2 u = at_least(add2(v, base), kLowest);
      // (2^-1000 is 0, and 0 times a finite number too)
      const float2 t = at_least(fma2(u, c, ll), -1000.0f);
      const float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
      return mul2(e, fma2(t, bb, aa));
    };
    const int first = static_cast<int>(run % per_row) * (kGradThreads * kGradPacks);
    Pack<T, E> in[kGradPacks];
    if (!zeros) {
#pragma unroll
      for (int u = 0; u < kGradPacks; ++u) {
        const int at = first + u * kGradThreads + static_cast<int>(threadIdx.x);
        if (at < packs) in[u] = load_pack<T, E>(x + lead + static_cast<int64_t>(at) * E);
      }
    }
#pragma unroll
    for (int u = 0; u < kGradPacks; ++u) {
      const int at = first + u * kGradThreads + static_cast<int>(threadIdx.x);
      if (at >= packs) break;
      const int index = lead + at * E;
      float v[E];
      if (zeros) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.0f;
      } else {
        float2 q[(E + 1) / 2];
        unpack_pairs(in[u], q);
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
      }
      store_pack(dx + index, pack<T, E>(v));
    }
    // the lone values beside the packs, by the row's first run
    const int lone = static_cast<int>(threadIdx.x);
    if (first == 0 && lone < lead + p.vocab - tail) {
      const int index = lone < lead ? lone : tail + lone - lead;
      float v = 0.0f;
      if (!zeros) {
        v = pairs(both(to_float(x[index]))).x;
        if (index == hit) v += hot;
      }
      dx[index] = from_float<T>(v);
    }
  }
}

template <typename T>
int run_forward(cudaStream_t s, const LogprobArgs &p, const T *logits) {
  constexpr int E = 16 / sizeof(T), U = Batch<T>::U;
  const int64_t packs = std::max(1, p.vocab / E), sms = sm_count();
  int cluster = 1;
  while (cluster < kMostCluster && p.rows * cluster * 2 <= sms &&
         packs >= 2 * cluster * 2 * 32 * U)
    cluster *= 2;
  int warps = 1;
  while (warps < (p.rows * cluster <= sms ? 16 : 8) && ceil_div(packs, cluster) > warps * 32)
    warps *= 2;
  const int64_t rows = std::min<int64_t>(p.rows, sms * 32);
  auto *fn = p.top > 0 ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>;
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

template <typename T>
int run_gradient(cudaStream_t s, const LogprobGradArgs &p, const T *logits, T *dlogits) {
  constexpr int E = 16 / sizeof(T);
  // Packs need rows of the same alignment on both sides. A pitch that changes it from row to
  // row changes it on both alike if the pitches differ by whole packs.
  const bool alike = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) %
                             16 == 0 &&
                     (p.rows == 1 || (p.ld - p.ldd) % E == 0);
  const int width = alike ? E : 1;
  const int64_t per_row = std::max<int64_t>(1, ceil_div(p.vocab / width, kGradThreads * kGradPacks));
  const int64_t runs = p.rows * per_row;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(runs, int64_t(1) << 30));
  return alike ? launch_programmatic(token_logprobs_grad_kernel<T, E>, dim3(grid),
                                     dim3(kGradThreads), 0, s, p, logits, dlogits, runs,
                                     static_cast<int>(per_row))
               : launch_programmatic(token_logprobs_grad_kernel<T, 1>, dim3(grid),
                                     dim3(kGradThreads), 0, s, p, logits, dlogits, runs,
                                     static_cast<int>(per_row));
}

// Checks shared by both directions.
int check(int64_t rows, int64_t vocab, int dtype, const void *logits, int64_t ld, float scale) {
  const int size = dtype_bytes(dtype);
  if (rows < 1 || vocab < 1 || !size || !logits || ld < vocab || !(scale > 0.0f) ||
      !(scale < kInf) || reinterpret_cast<uintptr_t>(logits) % size)
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
  const LogprobGradArgs p{rows,    ld,      ldd,       static_cast<int>(vocab), scale, targets,
                          stats,   entropy, d_logprob, d_entropy};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == NPLK_DTYPE_FP32)
    return run_gradient(s, p, static_cast<const float *>(logits), static_cast<float *>(dlogits));
  if (dtype == NPLK_DTYPE_FP16)
    return run_gradient(s, p, static_cast<const __half *>(logits), static_cast<__half *>(dlogits));
  return run_gradient(s, p, static_cast<const __nv_bfloat16 *>(logits),
                      static_cast<__nv_bfloat16 *>(dlogits));
}
