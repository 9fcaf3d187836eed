// What the group norm kernels share: the work split and its plan.
//
// An image's channels are cut into strips of whole groups; a cluster of CTAs
// takes one strip of one image (or a run of its rows), each CTA a run of rows.
// In a CTA, a row's strip is nv packs of V channels; thread t has pack t % nv
// of rows t / nv, t / nv + lanes, ... (lanes = threads / nv), so that a
// thread's channels never change and consecutive threads read consecutive
// memory. A strip of more packs than threads takes several turns (lanes = 1).
#pragma once

#include <algorithm>
#include <type_traits>

#include "nplk_device.cuh"
#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "typed_io.cuh"

namespace nplk {

struct NormGeom {
  int64_t ldx, ldy, lddy;  // pitches of x, of the output, of dy
  uint32_t hw;
  int c, groups, cg;
  int gs, strips;       // groups of a strip; strips of an image
  int slices;           // CTAs of a cluster
  int chunks;           // clusters that share a strip's rows
  uint32_t cta_rows;    // rows of a CTA
  FastDiv div_cg, div_slices, div_chunks, div_strips;
  FastDiv div_nv[2], div_lanes[2];  // packs and row lanes of a strip; of the last strip
  const float *gamma, *beta;
  float eps, alpha;
  int act;
};

struct NormPlan {
  NormGeom g;
  int v;            // elements of a pack
  bool keep;        // the strip stays in the cluster's shared memory
  int threads;
  int64_t batch;    // images of a launch
  int apply_chunks; // second pass: CTAs per image and strip
};

// Most threads of a CTA. A thread keeps its channels' constants and sums in
// registers (60 to 80 of them forward, up to 128 in the gradient), so an SM holds
// 24 and 16 warps.
constexpr int kNormMostThreads = 256;

// Workspace: per image and chunk, sums per channel and group.
constexpr int kNormMostChunks = 74;
inline int64_t norm_most_chunks(int64_t hw) {
  const int64_t by_rows = ceil_div(hw, 64);
  return by_rows < kNormMostChunks ? by_rows : kNormMostChunks;
}

// Bytes of shared memory beside the kept strips (norm_smem below).
inline int norm_tail_bytes(int threads, int v, int cw, int gs) {
  const int acc = threads * v > cw ? threads * v : cw;  // per row lane and channel
  const int teams = gs > 32 ? gs : 32;
  return 2 * acc * 4 + 2 * cw * 4 + teams * 16 + gs * 16 + 2 * gs * 4 + 64;
}

// Shared memory of a CTA of the kept form: two fit an SM.
constexpr int kNormKeepLimit = 112 * 1024;

// The divisions that the kernels do by multiplication, for the plan's split.
inline void norm_divisors(NormPlan &p) {
  NormGeom &g = p.g;
  g.div_slices = make_fastdiv(static_cast<uint32_t>(g.slices));
  g.div_chunks = make_fastdiv(static_cast<uint32_t>(g.chunks));
  g.div_strips = make_fastdiv(static_cast<uint32_t>(g.strips));
  for (int last = 0; last < 2; ++last) {
    const int gs = last ? g.groups - (g.strips - 1) * g.gs : g.gs;
    const int nv = gs * g.cg / p.v;
    g.div_nv[last] = make_fastdiv(static_cast<uint32_t>(nv));
    g.div_lanes[last] = make_fastdiv(static_cast<uint32_t>(nv <= p.threads ? p.threads / nv : 1));
  }
}

// `tensors`: strips that the kept form holds (x; or x and dy).
inline NormPlan plan_norm(int64_t n, int64_t hw, int64_t c, int64_t groups, int size, int v_fit,
                          int tensors) {
  NormPlan p{};
  const int cg = static_cast<int>(c / groups);
  auto gcd = [](int a, int b) {
    while (b) {
      const int t = a % b;
      a = b;
      b = t;
    }
    return a;
  };
  // The widest packs that the pointers allow and that fill whole groups within
  // 8192 channels (v divides c, so v / gcd(v, cg) divides the group count).
  int v = v_fit;
  while (v > 1 && (c % v != 0 || v / gcd(v, cg) * cg > 8192)) v /= 2;
  const int gs0 = v / gcd(v, cg);
  const int sms = sm_count();
  p.v = v;
  p.g.hw = static_cast<uint32_t>(hw);
  p.g.c = static_cast<int>(c);
  p.g.groups = static_cast<int>(groups);
  p.g.cg = cg;
  p.g.div_cg = make_fastdiv(static_cast<uint32_t>(cg));

  // Kept form: strips of at least 64 bytes a row; of those up to 512 bytes, the
  // narrowest in whole 32-byte sectors if 48 KB in each of 8 CTAs hold it, else the
  // narrowest.
  auto row = [&](int gs) { return static_cast<int64_t>(gs) * cg * size; };
  int gs = gs0;
  while (gs + gs0 <= groups && row(gs) < 64) gs += gs0;
  for (int m = gs; m <= groups && row(m) <= 512; m += gs0) {
    if (row(m) % 32 == 0 && ceil_div(hw, 8) * row(m) * tensors <= 48 * 1024) {
      gs = m;
      break;
    }
  }
  p.g.gs = gs;
  p.g.strips = static_cast<int>(ceil_div(groups, gs));
  p.g.chunks = 1;
  const int cw = gs * cg;
  const int64_t row_bytes = static_cast<int64_t>(cw) * size * tensors;
  int s = 1;
  auto slab = [&](int slices) { return ceil_div(hw, slices) * row_bytes; };
  // Up to 48 KB a CTA keeps four on an SM, so that one's loads run under another's
  // stores; more CTAs while they are few.
  const int64_t ctas = n * p.g.strips;
  while (s < 8 && (slab(s) > 48 * 1024 || (slab(s) > 16 * 1024 && ctas * s < 2 * sms))) s *= 2;
  p.g.slices = s;
  p.g.cta_rows = static_cast<uint32_t>(ceil_div(hw, s));
  constexpr int most = kNormMostThreads;
  // Six packs a thread: what a thread does once costs as much as 40 values.
  const int64_t packs = p.g.cta_rows * static_cast<int64_t>(cw / v);
  int64_t threads = ceil_div(ceil_div(packs, 6), 32) * 32;
  if (threads < cw / v) threads = ceil_div(cw / v, 32) * 32;
  p.threads = static_cast<int>(threads < 64 ? 64 : threads > most ? most : threads);
  p.keep = slab(s) + norm_tail_bytes(p.threads, v, cw, gs) <= kNormKeepLimit;
  if (p.keep) {
    norm_divisors(p);
    const int64_t most = ((int64_t(1) << 31) - 1) / (static_cast<int64_t>(p.g.strips) * s);
    p.batch = n < most ? n : most;
    return p;
  }

  // Two passes: whole rows where a CTA's threads hold one, else as many groups.
  gs = static_cast<int>(groups);
  if (c > most * v) gs = most * v / (gs0 * cg) * gs0;
  if (gs > 512) gs = 512 / gs0 * gs0;
  if (gs < gs0) gs = gs0;
  p.g.gs = gs;
  p.g.strips = static_cast<int>(ceil_div(groups, gs));
  p.threads = most;
  // Images whose tensors stay in L2 between the passes (a third of its 126 MB).
  const int64_t image = hw * c * size * tensors;
  int64_t batch = (40 << 20) / image;
  if (batch < 1) batch = 1;
  p.batch = n < batch ? n : batch;
  const int64_t wanted = static_cast<int64_t>(sms) * (tensors == 1 ? 3 : 2);
  int64_t chunks = wanted / (8 * p.g.strips * p.batch);
  if (chunks < 1) chunks = 1;
  if (chunks > norm_most_chunks(hw)) chunks = norm_most_chunks(hw);
  if (chunks > 1 && chunks * gs > 8192) chunks = 8192 / gs;  // 64 KB where they are joined
  p.g.slices = 8;
  p.g.chunks = static_cast<int>(chunks);
  p.g.cta_rows = static_cast<uint32_t>(ceil_div(hw, chunks * 8));
  int64_t apply = ceil_div(wanted, p.g.strips * p.batch);
  if (apply > hw) apply = hw;
  p.apply_chunks = static_cast<int>(apply);
  norm_divisors(p);
  return p;
}

// Elements of a pack that a pointer and pitch allow, at most 16 bytes.
inline int norm_pack_fit(const void *ptr, int64_t ld, int size) {
  int v = 16 / size;
  while (v > 1 && (reinterpret_cast<uintptr_t>(ptr) % (v * size) != 0 || ld % v != 0)) v /= 2;
  return v;
}

inline int norm_check(int64_t n, int64_t hw, int64_t c, int64_t groups) {
  if (n < 1 || hw < 1 || c < 1 || groups < 1 || c % groups != 0) return kErrInvalidArg;
  if (n >= (int64_t(1) << 31) || hw >= (int64_t(1) << 31) || c / groups > 8192 ||
      c > (int64_t(1) << 24))
    return kErrUnsupported;
  if (n > ((int64_t(1) << 31) - 1) / groups) return kErrUnsupported;
  return kOk;
}

inline size_t norm_workspace(int64_t n, int64_t hw, int64_t c, int64_t groups) {
  return align_up(static_cast<size_t>(n) * norm_most_chunks(hw) * (2 * c + 2 * groups) * sizeof(float),
                  256);
}

inline bool norm_aligned(const void *p, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

// Where a CTA of the first pass is: image, strip, rows.
struct NormPlace {
  int64_t image, chunk;
  int strip, rank, g0, gsl, cw, nv, lanes, col, lane;  // col, lane: of this thread
  uint32_t r0, rows, mine;  // the CTA's rows; how many are this thread's
  uint32_t base, rest;      // rows of a row lane: base, and one more in the first `rest`
  bool active;
};

__device__ __forceinline__ uint32_t lane_rows(const NormPlace &w, uint32_t lane) {
  return w.base + (lane < w.rest ? 1u : 0u);
}

template <int V>
__device__ __forceinline__ NormPlace norm_place(const NormGeom &p) {
  NormPlace w;
  const uint32_t cluster = fdiv(blockIdx.x, p.div_slices);
  w.rank = static_cast<int>(blockIdx.x - cluster * p.slices);
  const uint32_t at = fdiv(cluster, p.div_chunks);
  w.chunk = cluster - at * p.chunks;
  w.image = fdiv(at, p.div_strips);
  w.strip = static_cast<int>(at - static_cast<uint32_t>(w.image) * p.strips);
  w.g0 = w.strip * p.gs;
  w.gsl = min(p.gs, p.groups - w.g0);
  w.cw = w.gsl * p.cg;
  const int last = w.gsl < p.gs ? 1 : 0;
  w.nv = static_cast<int>(p.div_nv[last].d);
  w.lanes = static_cast<int>(p.div_lanes[last].d);
  const int threads = static_cast<int>(blockDim.x), t = static_cast<int>(threadIdx.x);
  w.lane = w.nv <= threads ? static_cast<int>(fdiv(t, p.div_nv[last])) : 0;
  w.col = t - w.lane * w.nv;
  w.active = w.lane < w.lanes && w.col < w.nv;
  const uint64_t first =
      (static_cast<uint64_t>(w.chunk) * p.slices + w.rank) * static_cast<uint64_t>(p.cta_rows);
  w.r0 = first < p.hw ? static_cast<uint32_t>(first) : p.hw;
  w.rows = min(p.cta_rows, p.hw - w.r0);
  w.base = fdiv(w.rows, p.div_lanes[last]);
  w.rest = w.rows - w.base * w.lanes;
  w.mine = w.active ? lane_rows(w, w.lane) : 0;
  return w;
}

// Calls f(pack size, activation) with both as std::integral_constant: 16-byte
// packs with the usual activations known to the compiler, everything else with
// the activation as an argument (-1). With it as an argument the kernels hold
// 118 registers across the calls of the rare ones instead of 40 to 80, which
// halves the loads in flight on an SM.
template <int kMost, typename F>
int norm_with_pack(int v, int act, F f) {
  using std::integral_constant;
  if (v == kMost) {
    constexpr integral_constant<int, kMost> pack{};
    switch (act) {
      case 0:
        return f(pack, integral_constant<int, 0>{});
      case 1:
        return f(pack, integral_constant<int, 1>{});
      case 5:
        return f(pack, integral_constant<int, 5>{});
      case 6:
        return f(pack, integral_constant<int, 6>{});
      default:
        return f(pack, integral_constant<int, -1>{});
    }
  }
  constexpr integral_constant<int, -1> any{};
  if constexpr (kMost > 4)
    if (v == 4) return f(integral_constant<int, 4>{}, any);
  if (v == 2) return f(integral_constant<int, 2>{}, any);
  return f(integral_constant<int, 1>{}, any);
}

template <typename... KArgs, typename... Args>
int norm_launch(void (*kernel)(KArgs...), int64_t grid, int threads, int smem, int cluster,
                cudaStream_t s, Args... args) {
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), smem)) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  count_launch();
  return map_cuda_error(cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...));
}

}  // namespace nplk
