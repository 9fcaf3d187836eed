// Group norm with an activation, channels last.
//
// For image i and group g (cg = c / groups channels, M = hw * cg values):
//   mean, M2 = sum (x - mean)^2, rstd = 1/sqrt(M2 / M + eps),
//   y = act(gamma * (x - mean) * rstd + beta).
//
// Statistics. Each thread keeps a mean and an M2 per channel and takes its rows
// in batches of four: the batch's own mean and M2 from the values in registers,
// then joined to the running ones (Chan, Golub and LeVeque, 1979: means differ by
// d, counts a and b: M2 = M2a + M2b + d^2 a b / (a + b)). Sums of squares are
// always taken about a mean of the same values, so a group whose mean is
// thousands of deviations from zero keeps its variance. Channels, threads, CTAs
// and chunks are joined the same way, by n-weighted mean and then
// M2 + n (mean_i - mean)^2.
//
// Kept form (norm_kernel<kKeep>): the strip of one image stays in the shared
// memory of a cluster of up to 8 CTAs: x is read once and y written once, in one
// launch. Otherwise three launches, image batch by image batch, so that the last
// one finds its x in L2: moments of chunks, their joining, normalising.
#include "act_epilogue.cuh"
#include "group_norm.cuh"

namespace nplk {
namespace {

struct Moments {
  float n, mean, m2;
};

// Weights of a join use the hardware's reciprocal as it is, within 2^-23: a weight is a
// factor of the difference of two means or of its square, and moves a mean by that much of
// the difference, which rounds by 2^-24 as it is; the variance by that much of itself. Only
// a whole mean is multiplied by a refined one (rcp_fine).

// 1 / x within a step of 2^-23 (one Newton step on the approximate reciprocal), x in
// the range of counts.
__device__ __forceinline__ float rcp_fine(float x) {
  const float r = rcp_approx(x);
  return fmaf(r, fmaf(-x, r, 1.0f), r);
}

// Of one pack's channels; the mean negated, pairs of channels together.
template <int V>
struct Running {
  static constexpr int kPairs = (V + 1) / 2;
  float n;
  float2 minus_mean[kPairs], m2[kPairs];
};

// Joins R rows, held as packs, to the running moments.
template <typename T, int V, int R>
__device__ __forceinline__ void join_rows(const Pack<T, V> (&p)[R], Running<V> &run) {
  const float total = run.n + static_cast<float>(R);
  const float share = static_cast<float>(R) * rcp_approx(total), cross = run.n * share;
  float2 x[R][Running<V>::kPairs];
#pragma unroll
  for (int r = 0; r < R; ++r) unpack_pairs(p[r], x[r]);
#pragma unroll
  for (int j = 0; j < Running<V>::kPairs; ++j) {
    float2 sum = x[0][j];
#pragma unroll
    for (int r = 1; r < R; ++r) sum = add2(sum, x[r][j]);
    const float2 minus = mul2(sum, both(-1.0f / static_cast<float>(R)));
    if (R > 1) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float2 e = add2(x[r][j], minus);
        run.m2[j] = fma2(e, e, run.m2[j]);
      }
    }
    const float2 d = fma2(run.minus_mean[j], both(-1.0f), minus);
    run.minus_mean[j] = fma2(d, both(share), run.minus_mean[j]);
    run.m2[j] = fma2(mul2(d, d), both(cross), run.m2[j]);
  }
  run.n = total;
}

// Joins one more to a list's moments.
__device__ __forceinline__ void join_one(Moments &t, const Moments &m) {
  if (m.n > 0.0f) {
    const float total = t.n + m.n, share = m.n * rcp_approx(total), d = m.mean - t.mean;
    t.m2 += fmaf(d * d, t.n * share, m.m2);
    t.mean = fmaf(d, share, t.mean);
    t.n = total;
  }
}

// Joins the moments of each aligned run of kWidth lanes; all of them get it.
template <int kWidth>
__device__ __forceinline__ Moments join_lanes(const Moments &m) {
  float n = m.n, s = m.n > 0.0f ? m.n * m.mean : 0.0f;
#pragma unroll
  for (int o = kWidth / 2; o; o >>= 1) {
    n += __shfl_xor_sync(0xffffffffu, n, o);
    s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  const float mean = n > 0.0f ? s * rcp_fine(n) : 0.0f, d = m.mean - mean;
  float q = m.n > 0.0f ? fmaf(m.n * d, d, m.m2) : 0.0f;
#pragma unroll
  for (int o = kWidth / 2; o; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
  return {n, mean, q};
}

struct Shared {  // the dynamic shared memory, after the kept rows
  float4 *team, *all;    // moments of the warps of a group; of the cluster's CTAs [8][gs]
  float *mean, *m2;      // per thread
  float *gamma, *beta;   // [cw]
  float *gmean, *grstd;  // [gs]
  uint8_t *bars;
};

template <int V>
__device__ __forceinline__ Shared norm_shared(uint8_t *at, const NormGeom &p) {
  const int acc = max(static_cast<int>(blockDim.x) * V, p.pitch);
  Shared s;
  s.bars = at;
  s.team = reinterpret_cast<float4 *>(at + 64);
  s.all = s.team + max(p.gs, 32);
  s.mean = reinterpret_cast<float *>(s.all + 8 * p.gs);
  s.m2 = s.mean + acc;
  s.gamma = s.m2 + acc;
  s.beta = s.gamma + p.pitch;
  s.gmean = s.beta + p.pitch;
  s.grstd = s.gmean + p.gs;
  return s;
}

// A thread's moments of one pack's channels into s.mean, s.m2: per channel, or,
// where a group has at least V channels, already joined over the pack's channels of
// its first group and of its second one.
template <int V>
__device__ __forceinline__ void put_moments(const NormGeom &p, const NormPlace &w, const Shared &s,
                                            const Running<V> &run, int col) {
  float mean[V], m2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    mean[j] = -((j & 1) ? run.minus_mean[j / 2].y : run.minus_mean[j / 2].x);
    m2[j] = (j & 1) ? run.m2[j / 2].y : run.m2[j / 2].x;
  }
  if (V > 1 && p.cg >= V) {
    const int ch = col * V;
    const int first = (static_cast<int>(fdiv(ch, p.div_cg)) + 1) * p.cg - ch;  // of its group
    float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sum0 += j < first ? mean[j] : 0.0f;
      sum1 += j < first ? 0.0f : mean[j];
    }
    const float k0 = static_cast<float>(first < V ? first : V), k1 = V - k0;
    const float mean0 = sum0 * rcp_fine(k0), mean1 = k1 > 0.0f ? sum1 * rcp_fine(k1) : 0.0f;
    float q0 = 0.0f, q1 = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = mean[j] - (j < first ? mean0 : mean1);
      const float q = fmaf(run.n * d, d, m2[j]);
      q0 += j < first ? q : 0.0f;
      q1 += j < first ? 0.0f : q;
    }
    const int at = 2 * (w.lane * w.nv + col);
    *reinterpret_cast<float2 *>(s.mean + at) = make_float2(mean0, mean1);
    *reinterpret_cast<float2 *>(s.m2 + at) = make_float2(q0, q1);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s.mean[w.lane * w.cw + col * V + j] = mean[j];
      s.m2[w.lane * w.cw + col * V + j] = m2[j];
    }
  }
}

// The moments of each of the CTA's groups, from what put_moments left, to
// s.all[rank] of every CTA of the cluster. kWidth lanes take a group, all lanes of
// several warps where there are warps to spare and more than 8 entries a lane.
template <int V, int kWidth>
__device__ __forceinline__ void cta_groups_by(const NormGeom &p, const NormPlace &w,
                                              const Shared &s, int each) {
  constexpr int kGroups = 32 / kWidth;  // of a warp at once
  const int warps = static_cast<int>(blockDim.x) >> 5, warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & (kWidth - 1), part = (threadIdx.x & 31) / kWidth;
  const bool joined = V > 1 && p.cg >= V;
  auto send = [&](int g, const Moments &t) {  // lane k to CTA k
    if (lane < p.slices && g < w.gsl)
      st_shared_cluster_f32x4(mapa_shared(smem_u32(&s.all[w.rank * p.gs + g]), lane),
                              make_float4(t.n, t.mean, t.m2, 0.0f));
  };
  const int teams = each == 1 ? warps : warps / each, team = each == 1 ? warp : warp / each;
  const int member = warp - team * each;
  for (int g0 = team * kGroups; g0 < w.gsl && team < teams; g0 += teams * kGroups) {
    const int g = g0 + part;
    Moments t{0.0f, 0.0f, 0.0f};
    if (g < w.gsl) {
      // per row lane: the group's channels, or the packs that hold some of them
      const int from = g * p.cg, to = from + p.cg;
      const int p0 = from / V, packs = joined ? (to - 1) / V - p0 + 1 : p.cg;
      const uint32_t magic = packs > 1 ? 0xffffffffu / static_cast<uint32_t>(packs) + 1 : 0u;
      const int entries = w.lanes * packs;
#pragma unroll 2
      for (int e = member * kWidth + lane; e < entries; e += each * kWidth) {
        const uint32_t l = packs == 1 ? e : __umulhi(static_cast<uint32_t>(e), magic);
        const int k = e - static_cast<int>(l) * packs;
        const float rows = static_cast<float>(lane_rows(w, l));
        if (joined) {
          const int c0 = (p0 + k) * V;
          const int at = 2 * (static_cast<int>(l) * w.nv + p0 + k) + (c0 < from ? 1 : 0);
          const int here = min(c0 + V, to) - max(c0, from);
          join_one(t, {rows * static_cast<float>(here), s.mean[at], s.m2[at]});
        } else {
          const int at = static_cast<int>(l) * w.cw + from + k;
          join_one(t, {rows, s.mean[at], s.m2[at]});
        }
      }
    }
    t = join_lanes<kWidth>(t);
    if (each == 1) send(g, t);
    else if (lane == 0) s.team[g * each + member] = make_float4(t.n, t.mean, t.m2, 0.0f);
  }
  if (each == 1) return;
  __syncthreads();
  for (int g = warp; g < w.gsl; g += warps) {
    const float4 v = lane < each ? s.team[g * each + lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    send(g, join_lanes<kWidth>({v.x, v.y, v.z}));
  }
}

template <int V>
__device__ __forceinline__ void cta_groups(const NormGeom &p, const NormPlace &w, const Shared &s) {
  const int warps = static_cast<int>(blockDim.x) >> 5;
  const int most = w.lanes * (V > 1 && p.cg >= V ? (p.cg + V - 1) / V + (p.cg % V ? 1 : 0) : p.cg);
  if (most <= 16) return cta_groups_by<V, 8>(p, w, s, 1);
  int each = 1;  // warps of a group
  while (2 * each * w.gsl <= warps && most > 256 * each) each *= 2;
  cta_groups_by<V, 32>(p, w, s, each);
}

// The normalised, scaled and activated values of one pack's channels.
template <typename T, int V, int kAct>
struct Affine {
  static constexpr int kPairs = (V + 1) / 2;
  float2 minus_mean[kPairs], scale[kPairs], shift[kPairs];

  // `stat(g)`: mean and rstd of group g of the strip; gamma, beta of channel ch on.
  template <typename F>
  __device__ __forceinline__ void set(const NormGeom &p, int ch, const float *gamma,
                                      const float *beta, F stat) {
    float m[V], a[V], b[V];
    const int g = static_cast<int>(fdiv(static_cast<uint32_t>(ch), p.div_cg));
    int left = (g + 1) * p.cg - ch;  // of the group, in this pack
    if (V > 1 && p.cg >= V) {
      const float2 s0 = stat(g), s1 = left < V ? stat(g + 1) : s0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        m[j] = -(j < left ? s0.x : s1.x);
        a[j] = j < left ? s0.y : s1.y;
      }
    } else {
      int k = g;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 v = stat(k);
        m[j] = -v.x;
        a[j] = v.y;
        if (--left == 0) {
          left = p.cg;
          if (j + 1 < V) ++k;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      a[j] *= gamma ? gamma[j] : 1.0f;
      b[j] = beta ? beta[j] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int k = V == 1 ? 0 : 2 * j + 1;
      minus_mean[j] = make_float2(m[2 * j], m[k]);
      scale[j] = make_float2(a[2 * j], a[k]);
      shift[j] = make_float2(b[2 * j], b[k]);
    }
  }
  __device__ __forceinline__ Pack<T, V> operator()(const Pack<T, V> &in, const NormGeom &p) const {
    float2 x[kPairs];
    unpack_pairs(in, x);
    float v[V];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const float2 z = fma2(add2(x[j], minus_mean[j]), scale[j], shift[j]);
      v[2 * j] = z.x;
      if (V > 1) v[2 * j + (V > 1 ? 1 : 0)] = z.y;
    }
    act_array<T, (V > 1)>(v, kAct >= 0 ? kAct : p.act, p.alpha);
    return pack<T, V>(v);
  }
};

// Moments of the strips, and with kKeep all of it.
template <typename T, int V, int kAct, bool kKeep>
__global__ void __launch_bounds__(kNormThreads, 3)
    norm_kernel(const __grid_constant__ CUtensorMap map, const NormGeom p, const T *x, T *y,
                float *mean_out, float *rstd_out, float2 *partial) {
  extern __shared__ __align__(128) uint8_t smem[];
  const NormPlace w = norm_place(p, blockIdx.x);
  Pack<T, V> *strip = reinterpret_cast<Pack<T, V> *>(smem);
  const int64_t held = p.boxes ? static_cast<int64_t>(p.stage_rows) * kNormStages : p.cta_rows;
  const size_t strip_bytes = kKeep ? (held * p.pitch * sizeof(T) + 127) / 128 * 128
                                   : kNormRing * kNormThreads * sizeof(Pack<T, V>);
  const Shared s = norm_shared<V>(smem + strip_bytes, p);
  const int c0 = w.g0 * p.cg;
  const int64_t row0 = w.image * p.hw + w.r0;
  const T *xs = x + row0 * p.ldx + c0;
  const uint32_t lanes = static_cast<uint32_t>(w.lanes);
  const int turn = w.lanes * (p.pitch / V);  // in packs, from one of the thread's rows to the next
  RowLoads<T, V, 1> loads;
  if (p.slices > 1) cluster_arrive_relaxed();
  if (kKeep) loads.prepare(p, s.bars);
  griddep_wait();
  griddep_launch_dependents();
  if (kKeep) {
    loads.start(p, w, {&map}, {smem}, w.image * p.hw);
    for (int i = threadIdx.x; i < w.cw; i += blockDim.x) {
      s.gamma[i] = p.gamma ? p.gamma[c0 + i] : 1.0f;
      s.beta[i] = p.beta ? p.beta[c0 + i] : 0.0f;
    }
  }
  for (int col = w.active ? w.col : w.nv; col < w.nv; col += blockDim.x) {
    Running<V> run;
    run.n = 0.0f;
#pragma unroll
    for (int j = 0; j < Running<V>::kPairs; ++j) run.minus_mean[j] = run.m2[j] = both(0.0f);
    const T *from = xs + static_cast<int64_t>(w.lane) * p.ldx + col * V;
    const int64_t pitch = static_cast<int64_t>(lanes) * p.ldx;
    if constexpr (kKeep) {
      Pack<T, V> *own = strip + w.lane * (p.pitch / V) + col;
      if (!p.boxes) {
        copy_rows(own, turn, from, pitch, w.mine);
        copy_async_commit();
        copy_async_wait<0>();  // its own copies are all that a thread reads: no barrier
      }
      uint32_t k = 0, r = w.lane;
      for (; k + 4 <= w.mine; k += 4, r += 4 * lanes) {
        if (p.boxes) loads.wait(p, r + 3 * lanes);
        const Pack<T, V> v[4] = {own[k * turn], own[(k + 1) * turn], own[(k + 2) * turn],
                                 own[(k + 3) * turn]};
        join_rows(v, run);
      }
      if (p.boxes && k < w.mine) loads.wait(p, w.lane + (w.mine - 1) * lanes);
      if (k + 2 <= w.mine) {
        const Pack<T, V> v[2] = {own[k * turn], own[(k + 1) * turn]};
        join_rows(v, run);
        k += 2;
      }
      if (k < w.mine) {
        const Pack<T, V> v[1] = {own[k * turn]};
        join_rows(v, run);
      }
    } else {
      stream_rows<T, V, 1>(w.mine, {from}, {pitch}, strip,
                           [&](const Pack<T, V>(&v)[1][4], int rows) {
        if (rows == 4) {
          join_rows(v[0], run);
        } else {
          const Pack<T, V> two[2] = {v[0][0], v[0][1]};
          const Pack<T, V> one[1] = {rows == 1 ? v[0][0] : v[0][2]};
          if (rows >= 2) join_rows(two, run);
          if (rows != 2) join_rows(one, run);
        }
      });
    }
    put_moments<V>(p, w, s, run, col);
  }
  __syncthreads();
  if (p.slices > 1) cluster_wait();  // every CTA of it has started and may be written to
  cta_groups<V>(p, w, s);
  if (p.slices > 1) cluster_sync();
  else __syncthreads();
  for (int i = threadIdx.x; i < (w.gsl * 8 + 31) / 32 * 32; i += blockDim.x) {
    const int g = i >> 3, k = i & 7;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (g < w.gsl && k < p.slices) v = s.all[k * p.gs + g];
    const Moments t = join_lanes<8>({v.x, v.y, v.z});
    if (g < w.gsl && k == 0) {
      if (kKeep) {
        const float rstd = 1.0f / sqrtf(t.m2 / t.n + p.eps);
        s.gmean[g] = t.mean;
        s.grstd[g] = rstd;
        const int64_t at = w.image * p.groups + w.g0 + g;
        if (w.rank == 0 && mean_out) mean_out[at] = t.mean;
        if (w.rank == 0 && rstd_out) rstd_out[at] = rstd;
      } else if (w.rank == 0) {
        partial[(w.image * p.chunks + w.chunk) * p.groups + w.g0 + g] = make_float2(t.mean, t.m2);
      }
    }
  }
  if constexpr (kKeep) {
    __syncthreads();
    for (int col = w.active ? w.col : w.nv; col < w.nv; col += blockDim.x) {
      Affine<T, V, kAct> f;
      f.set(p, col * V, s.gamma + col * V, s.beta + col * V,
            [&](int g) { return make_float2(s.gmean[g], s.grstd[g]); });
      const Pack<T, V> *own = strip + w.lane * (p.pitch / V) + col;
      T *to = y + (row0 + w.lane) * p.ldy + c0 + col * V;
      const int64_t pitch = static_cast<int64_t>(lanes) * p.ldy;
#pragma unroll 2
      for (uint32_t k = 0; k < w.mine; ++k, own += turn, to += pitch) store_pack(to, f(*own, p));
    }
    loads.drain(p, w);
  }
}

// Joins the chunks' moments: a CTA per image and group. mean and rstd to the
// caller and to stats.
__global__ void __launch_bounds__(128)
    norm_join_kernel(const NormGeom p, const float2 *partial, float *mean_out, float *rstd_out,
                     float2 *stats) {
  __shared__ float4 warps[4];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t at = blockIdx.x, image = at / p.groups;
  const float2 *from = partial + image * p.chunks * p.groups + (at - image * p.groups);
  Moments t{0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int k = threadIdx.x; k < p.chunks; k += 128) {
    const uint64_t first = static_cast<uint64_t>(k) * p.cta_rows;
    const uint64_t rows = first < p.hw ? min(static_cast<uint64_t>(p.cta_rows), p.hw - first) : 0;
    const float2 v = from[static_cast<int64_t>(k) * p.groups];
    join_one(t, {static_cast<float>(rows) * static_cast<float>(p.cg), v.x, v.y});
  }
  t = join_lanes<32>(t);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) warps[warp] = make_float4(t.n, t.mean, t.m2, 0.0f);
  __syncthreads();
  if (warp == 0) {
    const float4 v = lane < 4 ? warps[lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    t = join_lanes<32>({v.x, v.y, v.z});
    if (lane == 0) {
      const float rstd = 1.0f / sqrtf(t.m2 / t.n + p.eps);
      if (mean_out) mean_out[at] = t.mean;
      if (rstd_out) rstd_out[at] = rstd;
      stats[at] = make_float2(t.mean, rstd);
    }
  }
}

// Normalises: CTAs and threads as in the moments' pass, the images and rows in the
// other order, so that what that pass read last comes first, out of L2.
template <typename T, int V, int kAct>
__global__ void __launch_bounds__(kNormThreads, 3)
    norm_apply_kernel(const NormGeom p, const T *x, T *y, const float2 *stats) {
  extern __shared__ __align__(128) uint8_t smem[];
  NormPlace w = norm_place(p, gridDim.x - 1 - blockIdx.x);
  Pack<T, V> *ring = reinterpret_cast<Pack<T, V> *>(smem);
  griddep_wait();
  griddep_launch_dependents();
  if (w.mine == 0) return;
  // the thread's last row first
  const int64_t row = w.image * p.hw + w.r0 + w.lane + static_cast<int64_t>(w.mine - 1) * w.lanes;
  const int64_t xp = -static_cast<int64_t>(w.lanes) * p.ldx,
                yp = -static_cast<int64_t>(w.lanes) * p.ldy;
  const float2 *st = stats + w.image * p.groups + w.g0;
  for (int col = w.col; col < w.nv; col += blockDim.x) {
    const int ch = w.g0 * p.cg + col * V;
    T *to = y + row * p.ldy + ch;
    Affine<T, V, kAct> f;
    bool ready = false;
    stream_rows<T, V, 1>(w.mine, {x + row * p.ldx + ch}, {xp}, ring,
                         [&](const Pack<T, V>(&v)[1][4], int rows) {
      if (!ready) {  // the channels' constants arrive under the first rows
        f.set(p, col * V, p.gamma ? p.gamma + ch : nullptr, p.beta ? p.beta + ch : nullptr,
              [&](int g) { return st[g]; });
        ready = true;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < rows) store_pack(to + i * yp, f(v[0][i], p));
      to += 4 * yp;
    });
  }
}

template <typename T>
int run_norm(cudaStream_t s, int64_t n, const NormPlan &plan, const T *x, T *y, float *mean,
             float *rstd, float2 *work) {
  const NormGeom &g = plan.g;
  CUtensorMap map = {};
  if (plan.keep && g.boxes) {
    if (int rc = encode_tmap_2d_plain(&map, x, g.c, n * g.hw, g.ldx * sizeof(T), g.pitch,
                                      g.box_rows, sizeof(T)))
      return rc;
  }
  return norm_with_pack<16 / sizeof(T)>(plan.v, g.act, [&](auto pack_size, auto act) {
    constexpr int V = decltype(pack_size)::value, kAct = decltype(act)::value;
    const int tail = norm_tail_bytes(plan.threads, V, g.pitch, g.gs, plan.keep);
    float2 *stats = work, *partial = work + norm_work(plan, n, 1).stats / 2;
    for (int64_t i = 0; i < n; i += plan.batch) {
      const int64_t count = std::min(n - i, plan.batch);
      const T *xi = x + i * g.hw * g.ldx;
      T *yi = y + i * g.hw * g.ldy;
      float *mi = mean ? mean + i * g.groups : nullptr, *ri = rstd ? rstd + i * g.groups : nullptr;
      const int64_t ctas = count * g.strips * g.chunks * g.slices;
      if (plan.keep) {
        if (i > 0 && g.boxes) {
          if (int rc = encode_tmap_2d_plain(&map, xi, g.c, count * g.hw, g.ldx * sizeof(T), g.pitch,
                                            g.box_rows, sizeof(T)))
            return rc;
        }
        if (int rc = norm_launch(norm_kernel<T, V, kAct, true>, ctas, plan.threads,
                                 norm_rows_bytes(g, sizeof(T)) + tail, g.slices, s, map, g, xi, yi,
                                 mi, ri, nullptr))
          return rc;
        continue;
      }
      if (int rc = norm_launch(norm_kernel<T, V, 0, false>, ctas, plan.threads,
                               norm_ring_bytes(V, sizeof(T)) + tail, g.slices, s, map, g, xi, yi,
                               nullptr, nullptr, partial))
        return rc;
      if (int rc = norm_launch(norm_join_kernel, count * g.groups, 128, 0, 1, s, g, partial, mi, ri,
                               stats))
        return rc;
      if (int rc = norm_launch(norm_apply_kernel<T, V, kAct>, ctas, plan.threads,
                               norm_ring_bytes(V, sizeof(T)), 1, s, g, xi, yi, stats))
        return rc;
    }
    return kOk;
  });
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" size_t nplk_group_norm_workspace_size(int64_t n, int64_t hw, int64_t c,
                                                 int64_t groups) {
  if (norm_check(n, hw, c, groups) != kOk) return 0;
  return norm_workspace(n, hw, c, groups);
}

extern "C" int nplk_group_norm_act(void *stream, int64_t n, int64_t hw, int64_t c, int64_t groups,
                                   int dtype, const void *x, int64_t ldx, const float *gamma,
                                   const float *beta, float eps, int act, float act_alpha, void *y,
                                   int64_t ldy, float *mean, float *rstd, void *workspace,
                                   size_t workspace_bytes) {
  const int size = dtype_bytes(dtype);
  if (!size || !x || !y || ldx < c || ldy < c || act < 0 || act > 10) return kErrInvalidArg;
  if (int rc = norm_check(n, hw, c, groups)) return rc;
  if (!norm_aligned(x, size) || !norm_aligned(y, size) || (x == y && ldx != ldy))
    return kErrInvalidArg;
  for (const float *p : {gamma, beta, static_cast<const float *>(mean),
                         static_cast<const float *>(rstd)})
    if (!norm_aligned(p, 4)) return kErrInvalidArg;
  const int fx = norm_pack_fit(x, ldx, size), fy = norm_pack_fit(y, ldy, size);
  NormPlan plan = plan_norm({n, hw, c, groups, size, std::min(fx, fy), 1});
  if (!workspace || !norm_aligned(workspace, 256) ||
      workspace_bytes < std::max(kNormWorkLeast, norm_work(plan, n, 1).bytes()))
    return kErrInvalidArg;
  plan.g.ldx = ldx;
  plan.g.ldy = ldy;
  plan.g.gamma = gamma;
  plan.g.beta = beta;
  plan.g.eps = eps;
  plan.g.act = act;
  plan.g.alpha = act_alpha;
  plan.g.status = device_status_word();
  if (!plan.g.status) return kErrInternal;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float2 *work = static_cast<float2 *>(workspace);
  if (dtype == NPLK_DTYPE_FP32)
    return run_norm(s, n, plan, static_cast<const float *>(x), static_cast<float *>(y), mean, rstd,
                    work);
  if (dtype == NPLK_DTYPE_FP16)
    return run_norm(s, n, plan, static_cast<const __half *>(x), static_cast<__half *>(y), mean,
                    rstd, work);
  return run_norm(s, n, plan, static_cast<const __nv_bfloat16 *>(x),
                  static_cast<__nv_bfloat16 *>(y), mean, rstd, work);
}
