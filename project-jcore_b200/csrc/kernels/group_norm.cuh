// What the group norm kernels share: the work split, its plan, and how a CTA's
// rows come into shared memory.
//
// An image's channels are cut into strips of whole groups; a cluster of CTAs
// takes a strip of an image (or of a run of its rows), each CTA a run of rows,
// which come into its shared memory as [row][pitch]. A row's strip is nv packs of
// V channels; thread t has pack t % nv of rows t / nv, t / nv + lanes, ... (lanes =
// threads / nv), so that a thread's channels never change and consecutive threads
// read consecutive memory. A strip of more packs than threads takes several turns
// (lanes = 1).
#pragma once

#include <algorithm>
#include <type_traits>

#include "nplk_device.cuh"
#include "nplk_host.h"
#include "ptx_sm100.cuh"
#include "typed_io.cuh"

namespace nplk {

constexpr int kNormThreads = 256;  // at most
constexpr int kNormStages = 4;     // steps in which a CTA's rows arrive

struct NormGeom {
  int64_t ldx, ldy, lddy;  // pitches of x, of the output, of dy
  uint32_t hw;
  int c, groups, cg;
  int gs, strips;      // groups of a strip; strips of an image
  int slices, chunks;  // CTAs of a cluster; runs of rows of a strip that is not kept
  uint32_t cta_rows;   // rows of a CTA
  int pitch;           // channels of a full strip: a row's elements in shared memory
  int box_rows, boxes; // rows of a TMA box and boxes of a stage; 0: copied by the threads
  uint32_t stage_rows;
  FastDiv div_cg, div_slices, div_chunks, div_strips;
  FastDiv div_nv[2], div_lanes[2];  // packs and row lanes of a strip; of the last strip
  const float *gamma, *beta;
  float eps, alpha;
  int act;
  int *status;
};

struct NormPlan {
  NormGeom g;
  int v;          // elements of a pack
  bool keep;      // a cluster holds the strip's rows: one launch
  int threads;
  int64_t batch;  // images of a launch
};

// Runs of rows of a strip that is not kept, at most.
inline int64_t norm_most_chunks(int64_t hw) {
  const int64_t by_rows = ceil_div(hw, 8);
  return by_rows < 448 ? by_rows : 448;
}

// The passes over memory keep a ring of three batches of four packs per thread and
// tensor in shared memory: while one batch is worked on the next two are on their way.
constexpr int kNormRing = 12;
inline int norm_ring_bytes(int v, int size) { return kNormRing * kNormThreads * v * size; }

// Bytes of shared memory beside the rows (the layouts of both kernels fit it);
// `shared`: in clusters, whose CTAs share out the channels' sums.
inline int norm_tail_bytes(int threads, int v, int cw, int gs, bool shared) {
  const int acc = threads * v > cw ? threads * v : cw;
  return 2 * acc * 4 + 2 * cw * 4 + (shared ? 2 * (cw + 8) * 4 : 0) + (gs > 32 ? gs : 32) * 16 +
         9 * gs * 16 + 2 * gs * 4 + 256;
}
// Of a CTA that keeps its rows: two fit an SM.
constexpr int kNormKeepLimit = 112 * 1024;

// The divisions that the kernels do by multiplication, and how rows arrive.
inline void norm_finish(NormPlan &p, int64_t n, int size) {
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
  g.pitch = g.gs * g.cg;
  // TMA boxes where packs are of 16 bytes (then pitches and strips are too), a row
  // fits a box and row numbers 32 bits; boxes of whole 8 rows start 128-byte aligned.
  const int64_t each = ceil_div(g.cta_rows, kNormStages);
  g.boxes = 0;
  g.stage_rows = static_cast<uint32_t>(each);
  if (p.v * size == 16 && g.pitch <= 256 && n * g.hw < (int64_t(1) << 31) - 1024) {
    g.boxes = static_cast<int>(ceil_div(each, 256));
    g.box_rows = static_cast<int>(ceil_div(ceil_div(each, g.boxes), 8) * 8);
    g.stage_rows = static_cast<uint32_t>(g.box_rows * g.boxes);
  }
}

// Bytes of a CTA's rows of one tensor.
inline int64_t norm_rows_bytes(const NormGeom &g, int size) {
  const int64_t rows = g.boxes ? static_cast<int64_t>(g.stage_rows) * kNormStages : g.cta_rows;
  return (rows * g.pitch * size + 127) / 128 * 128;
}

// What a plan is made from. `tensors`: what is read (x; or x and dy). v: elements of a
// pack; gs0: the fewest groups that fill whole packs.
struct NormSize {
  int64_t n, hw, c, groups;
  int size, tensors, cg, v, gs0;

  NormSize(int64_t n_, int64_t hw_, int64_t c_, int64_t groups_, int size_, int v_fit,
           int tensors_)
      : n(n_), hw(hw_), c(c_), groups(groups_), size(size_), tensors(tensors_),
        cg(static_cast<int>(c_ / groups_)), v(v_fit) {
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
    while (v > 1 && (c % v != 0 || v / gcd(v, cg) * cg > 8192)) v /= 2;
    gs0 = v / gcd(v, cg);
  }
  int64_t row(int gs) const { return static_cast<int64_t>(gs) * cg * size; }
  // Images whose tensors stay in L2 between two passes (72 of its 126 MB: 4 x 16384 x 512
  // bf16 took 43.8 us in one batch, 53.8 in two).
  int64_t l2_images() const {
    return std::max<int64_t>(1, (72 << 20) / (hw * c * size * tensors));
  }
  // CTAs of a pass over memory that the SMs hold at once.
  int64_t ctas_at_once() const { return static_cast<int64_t>(sm_count()) * (tensors == 1 ? 3 : 2); }
  // Runs of rows, where `images` images share the SMs.
  int64_t chunks(int strips, int64_t images) const {
    return std::max<int64_t>(1, std::min(ctas_at_once() / (strips * images), norm_most_chunks(hw)));
  }
};

inline NormPlan norm_plan_base(const NormSize &z) {
  NormPlan p{};
  p.v = z.v;
  p.g.hw = static_cast<uint32_t>(z.hw);
  p.g.c = static_cast<int>(z.c);
  p.g.groups = static_cast<int>(z.groups);
  p.g.cg = z.cg;
  p.g.div_cg = make_fastdiv(static_cast<uint32_t>(z.cg));
  return p;
}

// Kept form: strips of at least 64 bytes a row; of those up to 512 bytes, the
// narrowest in whole 32-byte sectors if 48 KB in each of 8 CTAs hold it, else the
// narrowest. Up to 48 KB a CTA keeps several on an SM, so that one's loads run
// under another's stores; more CTAs while they are few.
inline NormPlan plan_norm_kept(const NormSize &z) {
  NormPlan p = norm_plan_base(z);
  auto threads_for = [&](int64_t rows, int cw, int64_t ctas) {
    // What a thread does once costs as much as ten packs. Six packs a thread while
    // there are few CTAs (2 x 1024 x 640 bf16: 7.9 us, with 20 packs 9.7); where there
    // are many, 20 forward (8 x 4096 x 320: 18.5 us against 24.3 with six) and 12 in the
    // gradient (3 x 961 x 510 fp32: 12.6 against 18.4). From 223 CTAs on the better
    // choice changes with how they fill the SMs: six would be 12% faster at 384 CTAs (6 x
    // 1024 x 640 forward: 10.7 us against 12.1) and 11% at 768, 34% slower at 512 (8 x
    // 1024 x 640: 17.3 against 12.9) and 28% at 1024.
    const int each = 2 * ctas <= 3 * sm_count() ? 6 : z.tensors == 1 ? 20 : 12;
    int64_t t = ceil_div(ceil_div(rows * (cw / z.v), each), 32) * 32;
    t = std::max<int64_t>(t, ceil_div(cw / z.v, 32) * 32);
    return static_cast<int>(std::min<int64_t>(std::max<int64_t>(t, 64), kNormThreads));
  };
  int gs = z.gs0;
  while (gs + z.gs0 <= z.groups && z.row(gs) < 64) gs += z.gs0;
  for (int m = gs; m <= z.groups && z.row(m) <= 512; m += z.gs0) {
    if (z.row(m) % 32 == 0 && ceil_div(z.hw, 8) * z.row(m) * z.tensors <= 48 * 1024) {
      gs = m;
      break;
    }
  }
  p.g.gs = gs;
  p.g.strips = static_cast<int>(ceil_div(z.groups, gs));
  p.g.chunks = 1;
  int s = 1;
  auto slab = [&](int slices) { return ceil_div(z.hw, slices) * z.row(gs) * z.tensors; };
  const int64_t ctas = z.n * p.g.strips;
  while (s < 8 && (slab(s) > 48 * 1024 || (slab(s) > 16 * 1024 && ctas * s < 2 * sm_count())))
    s *= 2;
  p.g.slices = s;
  p.g.cta_rows = static_cast<uint32_t>(ceil_div(z.hw, s));
  p.threads = threads_for(p.g.cta_rows, gs * z.cg, ctas * s);
  const int64_t most = ((int64_t(1) << 31) - 1) / (static_cast<int64_t>(p.g.strips) * s);
  p.batch = std::min(z.n, most);
  p.keep = true;
  norm_finish(p, z.n, z.size);
  return p;
}
inline bool norm_fits(const NormPlan &p, const NormSize &z) {
  return z.tensors * norm_rows_bytes(p.g, z.size) +
             norm_tail_bytes(p.threads, z.v, p.g.gs * z.cg, p.g.gs, true) <=
         kNormKeepLimit;
}

// Passes over memory: strips as wide as a CTA, one long run of rows for each CTA
// that the SMs hold at once, images in batches whose tensors stay in L2.
inline NormPlan plan_norm_passes(const NormSize &z) {
  NormPlan p = norm_plan_base(z);
  int gs = z.gs0;
  while (gs + z.gs0 <= z.groups && gs + z.gs0 <= 256 && (gs + z.gs0) * z.cg <= kNormThreads * z.v)
    gs += z.gs0;
  p.g.gs = gs;
  p.g.strips = static_cast<int>(ceil_div(z.groups, gs));
  p.batch = std::min(z.n, z.l2_images());
  p.g.slices = 1;
  p.threads = kNormThreads;
  p.g.chunks = static_cast<int>(z.chunks(p.g.strips, p.batch));
  p.g.cta_rows = static_cast<uint32_t>(ceil_div(z.hw, p.g.chunks));
  norm_finish(p, z.n, z.size);
  return p;
}

inline NormPlan plan_norm(const NormSize &z) {
  const NormPlan kept = plan_norm_kept(z);
  return norm_fits(kept, z) ? kept : plan_norm_passes(z);
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

// The workspace, in floats. Forward, in passes over memory: [batch][groups] mean and
// rstd, [batch * chunks][groups] mean and M2. Gradient: in passes over memory
// [batch][groups] statistics of four and [batch * chunks][groups] A, B; then, in both
// forms, [n * chunks][2][c] channel sums.
struct NormWork {
  int64_t stats, partial, channels;
  size_t bytes() const { return static_cast<size_t>(stats + partial + channels) * sizeof(float); }
};
inline NormWork norm_work(const NormPlan &p, int64_t n, int tensors) {
  NormWork w{};
  if (!p.keep) {
    w.stats = p.batch * p.g.groups * (tensors == 1 ? 2 : 4);
    w.partial = p.batch * p.g.chunks * p.g.groups * 2;
  }
  if (tensors == 2) w.channels = n * p.g.chunks * 2 * p.g.c;
  return w;
}
constexpr size_t kNormWorkLeast = 256;

// What suffices for either direction, every type and alignment, and for fewer images.
inline size_t norm_workspace(int64_t n, int64_t hw, int64_t c, int64_t groups) {
  size_t most = kNormWorkLeast;
  for (int size : {2, 4}) {
    for (int v = 16 / size; v >= 1; v /= 2) {
      for (int tensors : {1, 2}) {
        const NormSize z(n, hw, c, groups, size, v, tensors);
        NormPlan p = plan_norm_kept(z);
        // Fewer images have as many slices or more, and so no more rows in a CTA, but
        // perhaps more threads, and boxes where the rows of all would not take them.
        p.threads = kNormThreads;
        norm_finish(p, 1, size);
        if (!norm_fits(p, z)) {
          // k images have max(1, min(T / (strips min(k, B)), most)) chunks each, B = l2_images(),
          // T = ctas_at_once(): k <= B of them max(k, min(k most, T / strips)) at most
          p = plan_norm_passes(z);
          const int64_t together =
              std::max(n, std::min(n * norm_most_chunks(hw), z.ctas_at_once() / p.g.strips));
          const int64_t runs = std::max(together, n * z.chunks(p.g.strips, z.l2_images()));
          const NormWork w{n * groups * 4, runs * groups * 2, tensors == 2 ? runs * 2 * c : 0};
          most = std::max(most, w.bytes());
        } else {
          most = std::max(most, norm_work(p, n, tensors).bytes());
        }
      }
    }
  }
  return align_up(most, 256);
}

inline bool norm_aligned(const void *p, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

// Where a CTA of the first pass is, and its thread.
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

__device__ __forceinline__ NormPlace norm_place(const NormGeom &p, uint32_t block) {
  NormPlace w;
  const uint32_t cluster = fdiv(block, p.div_slices);
  w.rank = static_cast<int>(block - cluster * p.slices);
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

// A CTA's rows of kTensors tensors on their way into shared memory: TMA boxes,
// a barrier per stage, or copies by the threads that read them (counted in
// cp.async groups, 2-byte packs at once).
template <typename T, int V, int kTensors>
struct RowLoads {
  uint64_t *bars;           // [kNormStages]
  volatile int *abort_flag;
  int arrived;              // stages this thread has waited for

  // Before griddep_wait; ends with a barrier.
  __device__ __forceinline__ void prepare(const NormGeom &p, uint8_t *at) {
    bars = reinterpret_cast<uint64_t *>(at);
    abort_flag = reinterpret_cast<volatile int *>(bars + kNormStages);
    arrived = 0;
    if (threadIdx.x == 0) {
      for (int s = 0; s < kNormStages; ++s) mbar_init(&bars[s], 1);
      *abort_flag = 0;
      fence_mbar_init();
    }
    __syncthreads();
  }
  __device__ __forceinline__ void start(const NormGeom &p, const NormPlace &w,
                                        const CUtensorMap *const (&maps)[kTensors],
                                        uint8_t *const (&to)[kTensors], int64_t first_image_row) {
    if (!p.boxes || threadIdx.x != 0) return;
    for (int s = 0; s < kNormStages; ++s) {
      const uint32_t from = s * p.stage_rows;
      if (from >= w.rows) break;
      mbar_arrive_expect_tx(&bars[s], kTensors * p.stage_rows * p.pitch * sizeof(T));
      for (int b = 0; b < p.boxes; ++b) {
        const uint32_t r = from + b * p.box_rows;
#pragma unroll
        for (int k = 0; k < kTensors; ++k)
          tma_load_2d(maps[k], &bars[s], to[k] + static_cast<size_t>(r) * p.pitch * sizeof(T),
                      w.g0 * p.cg, static_cast<int>(first_image_row + w.r0 + r));
      }
    }
  }
  // Row r (of the CTA) and those before it have arrived.
  __device__ __forceinline__ void wait(const NormGeom &p, uint32_t r) {
    while (arrived < kNormStages && r >= arrived * p.stage_rows) {
      mbar_wait(&bars[arrived], 0u, abort_flag, p.status, kStatusTimeoutStage);
      ++arrived;
    }
  }
  // Before the CTA's end: nothing is in flight (the threads have waited unless a
  // wait expired).
  __device__ __forceinline__ void drain(const NormGeom &p, const NormPlace &w) {
    if (!p.boxes || threadIdx.x != 0 || !*abort_flag) return;
    for (int s = 0; s < kNormStages; ++s)
      if (s * p.stage_rows < w.rows) mbar_drain(&bars[s], 0u);
  }
};

// Copies packs from + k * pitch to `to` + k * step, k < count, in cp.async groups;
// 2-byte packs, which cp.async does not take, by eight loads at a time.
template <typename T, int V>
__device__ __forceinline__ void copy_rows(Pack<T, V> *to, int step, const T *from, int64_t pitch,
                                          uint32_t count) {
  if constexpr (sizeof(Pack<T, V>) == 2) {
    for (uint32_t k = 0; k < count; k += 8) {
      Pack<T, V> v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < count) v[i] = load_pack<T, V>(from + (k + i) * pitch);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < count) to[(k + i) * step] = v[i];
    }
  } else {
#pragma unroll 4
    for (uint32_t k = 0; k < count; ++k) copy_pack_async<T, V>(to + k * step, from + k * pitch);
  }
}

// Calls work(batch of packs, how many) for a thread's rows k = 0, 1, ... of kTensors
// tensors, four at a time; from[i] + k * pitch[i] is row k. ring: the thread's own
// slots are ring[i * kNormThreads + threadIdx.x], so it waits for its own copies only.
template <typename T, int V, int kTensors, typename F>
__device__ __forceinline__ void stream_rows(uint32_t count, const T *const (&from)[kTensors],
                                            const int64_t (&pitch)[kTensors], Pack<T, V> *ring,
                                            F work) {
  auto ask = [&](uint32_t batch) {
    const uint32_t at = 4 * batch;
#pragma unroll
    for (int t = 0; t < kTensors; ++t)
      copy_rows(ring + ((t * kNormRing + batch % 3 * 4) * kNormThreads + threadIdx.x), kNormThreads,
                from[t] + at * pitch[t], pitch[t], at < count ? min(4u, count - at) : 0u);
    copy_async_commit();
  };
  ask(0);
  ask(1);
  for (uint32_t batch = 0; 4 * batch < count; ++batch) {
    ask(batch + 2);
    copy_async_wait<2>();
    const uint32_t slot = batch % 3 * 4;
    Pack<T, V> v[kTensors][4];
#pragma unroll
    for (int t = 0; t < kTensors; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[t][i] = ring[(t * kNormRing + slot + i) * kNormThreads + threadIdx.x];
    work(v, static_cast<int>(min(4u, count - 4 * batch)));
  }
  copy_async_wait<0>();
}

// Calls f(pack size, activation) with both as std::integral_constant: 16-byte
// packs with the usual activations known to the compiler, everything else with
// the activation as an argument (-1): the calls of the rare ones in the loops keep
// every constant of a thread's channels in registers that calls preserve, or spill.
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
int norm_launch(void (*kernel)(KArgs...), int64_t grid, int threads, int64_t smem, int cluster,
                cudaStream_t s, const Args &...args) {
  if (grid > INT32_MAX) return kErrUnsupported;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), static_cast<int>(smem)))
    return rc;
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
