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
// thousands of deviations from zero keeps its variance, at about 6 instructions
// a value. Rows, channels, CTAs and chunks are joined the same way, by
// n-weighted mean and then M2 + n (mean_i - mean)^2.
//
// Kept form (norm_kernel<kKeep>): the strip of one image stays in the shared
// memory of a cluster of up to 8 CTAs: x is read once and y written once, in one
// launch. Otherwise two passes, image batch by image batch, so that the second
// pass finds its x in L2.
#include "act_epilogue.cuh"
#include "group_norm.cuh"

namespace nplk {
namespace {

struct Moments {
  float n, mean, m2;
};

// Of one pack's channels; the mean negated, pairs of channels together.
template <int V>
struct Running {
  static constexpr int kPairs = (V + 1) / 2;
  float n;
  float2 minus_mean[kPairs], m2[kPairs];
};

template <typename T, int V>
__device__ __forceinline__ void unpack_pairs(const Pack<T, V> &p, float2 (&v)[(V + 1) / 2]) {
  if constexpr (V == 1) {
    v[0] = both(to_float(p.e[0]));
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) v[j / 2] = make_float2(to_float(p.e[j]), to_float(p.e[j + 1]));
  }
}

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

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Joins the moments of each aligned run of kWidth lanes; all of them get it.
template <int kWidth>
__device__ __forceinline__ Moments join_lanes(Moments m) {
  float n = m.n, s = m.n > 0.0f ? m.n * m.mean : 0.0f;
#pragma unroll
  for (int o = kWidth / 2; o; o >>= 1) {
    n += __shfl_xor_sync(0xffffffffu, n, o);
    s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  const float mean = n > 0.0f ? s / n : 0.0f, d = m.mean - mean;
  float q = m.n > 0.0f ? fmaf(m.n * d, d, m.m2) : 0.0f;
#pragma unroll
  for (int o = kWidth / 2; o; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
  return {n, mean, q};
}

struct Shared {  // the dynamic shared memory, after the kept strip
  float *mean, *m2;       // [lanes][cw]
  float *gamma, *beta;    // [cw]
  float4 *team, *group;   // moments of the warps of a group; of the CTA's groups
  float *gmean, *grstd;   // [gs]
};

template <int V>
__device__ __forceinline__ Shared norm_shared(uint8_t *at, const NormGeom &p) {
  const int cw = p.gs * p.cg;
  const int acc = max(static_cast<int>(blockDim.x) * V, cw);
  Shared s;
  s.team = reinterpret_cast<float4 *>(at);
  s.group = s.team + max(p.gs, 32);
  s.mean = reinterpret_cast<float *>(s.group + p.gs);
  s.m2 = s.mean + acc;
  s.gamma = s.m2 + acc;
  s.beta = s.gamma + cw;
  s.gmean = s.beta + cw;
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
    const float mean0 = sum0 * rcp_approx(k0), mean1 = k1 > 0.0f ? sum1 * rcp_approx(k1) : 0.0f;
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

// The CTA's moments of each of its groups, from what put_moments left, to
// s.group. The warps are shared out over the groups.
template <int V>
__device__ __forceinline__ void cta_groups(const NormGeom &p, const NormPlace &w, const Shared &s) {
  const int warps = static_cast<int>(blockDim.x) >> 5, warp = threadIdx.x >> 5,
            lane = threadIdx.x & 31;
  const int each = w.gsl >= warps ? 1 : warps / w.gsl, teams = w.gsl >= warps ? warps : w.gsl;
  const bool joined = V > 1 && p.cg >= V;
  const int team = each == 1 ? warp : warp / each, member = warp - team * each;
  if (team < teams) {
    for (int g = team; g < w.gsl; g += teams) {
      // per row lane: the group's channels, or the packs that hold some of them
      const int from = g * p.cg, to = from + p.cg;
      const int p0 = from / V, packs = joined ? (to - 1) / V - p0 + 1 : p.cg;
      const uint32_t magic = 0xffffffffu / static_cast<uint32_t>(packs) + 1;  // packs > 1
      const int entries = w.lanes * packs;
      auto entry = [&](int e) {
        const uint32_t l = packs == 1 ? e : __umulhi(static_cast<uint32_t>(e), magic);
        const int k = e - static_cast<int>(l) * packs;
        const float rows = static_cast<float>(lane_rows(w, l));
        if (joined) {
          const int c0 = (p0 + k) * V;
          const int here = min(c0 + V, to) - max(c0, from);
          const int at = 2 * (static_cast<int>(l) * w.nv + p0 + k) + (c0 < from ? 1 : 0);
          return Moments{rows * static_cast<float>(here), s.mean[at], s.m2[at]};
        }
        const int at = static_cast<int>(l) * w.cw + from + k;
        return Moments{rows, s.mean[at], s.m2[at]};
      };
      float n = 0.0f, m = 0.0f, q = 0.0f;
      for (int e = member * 32 + lane; e < entries; e += each * 32) {
        const Moments v = entry(e);
        n += v.n;
        if (v.n > 0.0f) m = fmaf(v.n, v.mean, m);
      }
      n = warp_sum(n);
      m = warp_sum(m);
      const float mean = n > 0.0f ? m / n : 0.0f;
      for (int e = member * 32 + lane; e < entries; e += each * 32) {
        const Moments v = entry(e);
        const float d = v.mean - mean;
        if (v.n > 0.0f) q += fmaf(v.n * d, d, v.m2);
      }
      q = warp_sum(q);
      if (lane == 0) (each == 1 ? s.group[g] : s.team[g * each + member]) = make_float4(n, mean, q, 0.0f);
    }
  }
  __syncthreads();
  if (each == 1) return;
  for (int i = threadIdx.x; i < (w.gsl * 16 + 31) / 32 * 32; i += blockDim.x) {
    const int g = i >> 4, k = i & 15;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (g < w.gsl && k < each) v = s.team[g * each + k];
    const Moments t = join_lanes<16>({v.x, v.y, v.z});
    if (g < w.gsl && k == 0) s.group[g] = make_float4(t.n, t.mean, t.m2, 0.0f);
  }
  __syncthreads();
}

// The normalised, scaled and activated values of one pack's channels.
template <typename T, int V, int kAct>
struct Affine {
  static constexpr int kPairs = (V + 1) / 2;
  float2 minus_mean[kPairs], scale[kPairs], shift[kPairs];

  __device__ __forceinline__ void set(const NormGeom &p, int ch, const float *gmean,
                                      const float *grstd, const float *gamma, const float *beta) {
    float m[V], a[V], b[V];
    int g = static_cast<int>(fdiv(static_cast<uint32_t>(ch), p.div_cg)), left = (g + 1) * p.cg - ch;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      m[j] = -gmean[g];
      a[j] = grstd[g] * gamma[ch + j];
      b[j] = beta[ch + j];
      if (--left == 0) {
        left = p.cg;
        if (j + 1 < V) ++g;
      }
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
    act_array<T>(v, kAct >= 0 ? kAct : p.act, p.alpha);
    return pack<T, V>(v);
  }
};

// First pass, and with kKeep the whole of it.
template <typename T, int V, int kAct, bool kKeep>
__global__ void __launch_bounds__(kNormMostThreads, 3) norm_kernel(NormGeom p, const T *x, T *y, float *mean_out,
                                                   float *rstd_out, float2 *partial) {
  extern __shared__ __align__(16) uint8_t smem[];
  const NormPlace w = norm_place<V>(p);
  Pack<T, V> *strip = reinterpret_cast<Pack<T, V> *>(smem);
  const size_t strip_bytes =
      kKeep ? (static_cast<size_t>(p.cta_rows) * p.gs * p.cg * sizeof(T) + 15) / 16 * 16 : 0;
  const Shared s = norm_shared<V>(smem + strip_bytes, p);
  griddep_wait();
  griddep_launch_dependents();
  const int c0 = w.g0 * p.cg;
  const int64_t row0 = w.image * p.hw + w.r0;
  const T *xs = x + row0 * p.ldx + c0;
  const uint32_t lanes = static_cast<uint32_t>(w.lanes);

  if (kKeep) {
    for (int i = threadIdx.x; i < w.cw; i += blockDim.x) {
      if (p.gamma) copy_pack_async<float, 1>(reinterpret_cast<Pack<float, 1> *>(s.gamma + i), p.gamma + c0 + i);
      else s.gamma[i] = 1.0f;
      if (p.beta) copy_pack_async<float, 1>(reinterpret_cast<Pack<float, 1> *>(s.beta + i), p.beta + c0 + i);
      else s.beta[i] = 0.0f;
    }
    copy_async_commit();
  }
  for (int col = w.active ? w.col : w.nv; col < w.nv; col += blockDim.x) {
    Running<V> run;
    run.n = 0.0f;
#pragma unroll
    for (int j = 0; j < Running<V>::kPairs; ++j) run.minus_mean[j] = run.m2[j] = both(0.0f);
    const T *xc = xs + col * V;
    if constexpr (kKeep) {
      // All of the thread's rows are asked for at once, in four groups of
      // copies; it reads back only what it copied, so no barrier.
      const uint32_t mine = w.mine;
      const uint32_t step = (mine + 15) / 16 * 4;
      Pack<T, V> *own = strip + w.lane * w.nv + col;
      const int turn = w.lanes * w.nv;  // from one of the thread's rows to the next
      const T *from = xc + static_cast<int64_t>(w.lane) * p.ldx;
      const int64_t pitch = static_cast<int64_t>(lanes) * p.ldx;
#pragma unroll 1
      for (uint32_t q = 0; q < 4; ++q) {
        const uint32_t end = min((q + 1) * step, mine);
#pragma unroll 4
        for (uint32_t k = q * step; k < end; ++k)
          copy_pack_async<T, V>(own + k * turn, from + k * pitch);
        copy_async_commit();
      }
#pragma unroll 1
      for (uint32_t q = 0; q < 4; ++q) {
        if (q == 0) copy_async_wait<3>();
        else if (q == 1) copy_async_wait<2>();
        else if (q == 2) copy_async_wait<1>();
        else copy_async_wait<0>();
        const uint32_t end = min((q + 1) * step, mine);
        uint32_t k = q * step;
        for (; k + 4 <= end; k += 4) {
          Pack<T, V> v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = own[(k + i) * turn];
          join_rows(v, run);
        }
        if (k + 2 <= end) {
          const Pack<T, V> v[2] = {own[k * turn], own[(k + 1) * turn]};
          join_rows(v, run);
          k += 2;
        }
        if (k < end) {
          const Pack<T, V> v[1] = {own[k * turn]};
          join_rows(v, run);
        }
      }
    } else {
      // Eight rows asked for at a time, joined four by four.
      uint32_t r = w.lane;
      const int64_t pitch = static_cast<int64_t>(lanes) * p.ldx;
      const T *at = xc + static_cast<int64_t>(r) * p.ldx;
      for (; r + 7 * lanes < w.rows; r += 8 * lanes, at += 8 * pitch) {
        Pack<T, V> a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = load_pack<T, V>(at + i * pitch);
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = load_pack<T, V>(at + (4 + i) * pitch);
        join_rows(a, run);
        join_rows(b, run);
      }
      if (r < w.rows) {
        Pack<T, V> a[4], b[2], c[1];
        const uint32_t left = (w.mine & 7u);
        const bool four = left & 4u, two = left & 2u, one = left & 1u;
        if (four) {
#pragma unroll
          for (int i = 0; i < 4; ++i) a[i] = load_pack<T, V>(at + i * pitch);
          at += 4 * pitch;
        }
        if (two) {
#pragma unroll
          for (int i = 0; i < 2; ++i) b[i] = load_pack<T, V>(at + i * pitch);
          at += 2 * pitch;
        }
        if (one) c[0] = load_pack<T, V>(at);
        if (four) join_rows(a, run);
        if (two) join_rows(b, run);
        if (one) join_rows(c, run);
      }
    }
    put_moments<V>(p, w, s, run, col);
  }
  copy_async_wait<0>();
  __syncthreads();
  cta_groups<V>(p, w, s);
  // The cluster's groups, in every CTA of it.
  if (p.slices > 1) {
    cluster_sync();
    // 8 lanes a group: one round trip to all CTAs
    for (int i = threadIdx.x; i < (w.gsl * 8 + 31) / 32 * 32; i += blockDim.x) {
      const int g = i >> 3, k = i & 7;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (g < w.gsl && k < p.slices)
        v = ld_shared_cluster_v4(mapa_shared(smem_u32(&s.group[g]), static_cast<uint32_t>(k)));
      const Moments t =
          join_lanes<8>({__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z)});
      if (g < w.gsl && k == 0) {
        s.gmean[g] = t.mean;
        s.grstd[g] = kKeep ? 1.0f / sqrtf(t.m2 / t.n + p.eps) : t.m2;
      }
    }
    __syncthreads();
  } else {
    for (int g = threadIdx.x; g < w.gsl; g += blockDim.x) {
      const float4 t = s.group[g];
      s.gmean[g] = t.y;
      s.grstd[g] = kKeep ? 1.0f / sqrtf(t.z / t.x + p.eps) : t.z;
    }
  }
  if (w.rank == 0) {
    for (int g = threadIdx.x; g < w.gsl; g += blockDim.x) {
      if (kKeep) {
        if (mean_out) mean_out[w.image * p.groups + w.g0 + g] = s.gmean[g];
        if (rstd_out) rstd_out[w.image * p.groups + w.g0 + g] = s.grstd[g];
      } else {
        partial[(w.image * p.chunks + w.chunk) * p.groups + w.g0 + g] =
            make_float2(s.gmean[g], s.grstd[g]);
      }
    }
  }
  if constexpr (kKeep) {
    __syncthreads();
    T *ys = y + row0 * p.ldy + c0;
    for (int col = w.active ? w.col : w.nv; col < w.nv; col += blockDim.x) {
      Affine<T, V, kAct> f;
      f.set(p, col * V, s.gmean, s.grstd, s.gamma, s.beta);
      const Pack<T, V> *own = strip + w.lane * w.nv + col;
      const int turn = w.lanes * w.nv;
      T *to = ys + static_cast<int64_t>(w.lane) * p.ldy + col * V;
      const int64_t pitch = static_cast<int64_t>(lanes) * p.ldy;
#pragma unroll 2
      for (uint32_t r = w.lane; r < w.rows; r += lanes, own += turn, to += pitch)
        store_pack(to, f(*own, p));
    }
  }
  if (p.slices > 1) cluster_sync_relaxed();  // no CTA leaves while another reads its groups
}

// Second pass: joins the chunks' moments, then normalises. Rows are taken from
// the image's end, which the first pass read last; the first ones are asked for
// before the moments are joined.
template <typename T, int V, int kAct>
__global__ void __launch_bounds__(kNormMostThreads, 3)
    norm_apply_kernel(NormGeom p, const T *x, T *y, float *mean_out, float *rstd_out,
                      const float2 *partial, FastDiv apply_chunks, uint32_t apply_rows) {
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t at = gridDim.x - 1 - blockIdx.x;
  const uint32_t piece = fdiv(at, apply_chunks);
  const uint32_t chunk = at - piece * apply_chunks.d;
  const int64_t image = fdiv(piece, p.div_strips);
  const int g0 = static_cast<int>(piece - static_cast<uint32_t>(image) * p.strips) * p.gs;
  const int gsl = min(p.gs, p.groups - g0), cw = gsl * p.cg, c0 = g0 * p.cg;
  const int last = gsl < p.gs ? 1 : 0;
  const int nv = static_cast<int>(p.div_nv[last].d);
  const uint32_t lanes = p.div_lanes[last].d;
  float2 *chunks = reinterpret_cast<float2 *>(smem);  // [chunks][gsl]
  float *gmean = reinterpret_cast<float *>(chunks + p.chunks * p.gs), *grstd = gmean + p.gs;
  float *gamma = grstd + p.gs, *beta = gamma + p.gs * p.cg;
  const int threads = static_cast<int>(blockDim.x), t = static_cast<int>(threadIdx.x);
  const uint32_t rl = nv <= threads ? fdiv(t, p.div_nv[last]) : 0;
  int col = t - static_cast<int>(rl) * nv;
  const uint64_t begin = static_cast<uint64_t>(chunk) * apply_rows;
  const uint32_t r0 = begin < p.hw ? static_cast<uint32_t>(begin) : p.hw;
  const uint32_t rows = min(apply_rows, p.hw - r0);
  const int64_t xp = static_cast<int64_t>(lanes) * p.ldx, yp = static_cast<int64_t>(lanes) * p.ldy;
  const T *xc = x + (image * p.hw + r0 + rl) * p.ldx + c0 + col * V;
  T *yc = y + (image * p.hw + r0 + rl) * p.ldy + c0 + col * V;
  if (rl >= lanes) col = nv;
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kAsk = V == 8 ? 2 : 4;  // rows in registers, and as many on their way
  Pack<T, V> v[kAsk];
  auto ask = [&](const T *from, uint32_t r) {
#pragma unroll
    for (int i = 0; i < kAsk; ++i)
      if (r + i * lanes < rows) v[i] = load_pack<T, V>(from + i * xp);
  };
  if (col < nv) ask(xc, rl);
  for (int i = t; i < cw; i += threads) {
    gamma[i] = p.gamma ? p.gamma[c0 + i] : 1.0f;
    beta[i] = p.beta ? p.beta[c0 + i] : 0.0f;
  }
  const int warp = t >> 5, lane = t & 31, warps = threads >> 5;
  for (int k = warp; k < p.chunks; k += warps)
    for (int g = lane; g < gsl; g += 32)
      chunks[k * gsl + g] = partial[(image * p.chunks + k) * p.groups + g0 + g];
  __syncthreads();
  const uint32_t chunk_rows = p.cta_rows * p.slices;
  for (int g = warp; g < gsl; g += warps) {
    Moments m{0.0f, 0.0f, 0.0f};
    for (int k = lane; k < p.chunks; k += 32) {  // at most three
      const uint64_t first = static_cast<uint64_t>(k) * chunk_rows;
      if (first >= p.hw) break;
      const float n = static_cast<float>(min(chunk_rows, p.hw - static_cast<uint32_t>(first))) *
                      static_cast<float>(p.cg);
      const float2 c = chunks[k * gsl + g];
      const float total = m.n + n, d = c.x - m.mean, share = n / total;
      m.mean = fmaf(d, share, m.mean);
      m.m2 += fmaf(d * d, m.n * share, c.y);
      m.n = total;
    }
    m = join_lanes<32>(m);
    if (lane == 0) {
      gmean[g] = m.mean;
      grstd[g] = 1.0f / sqrtf(m.m2 / m.n + p.eps);
      if (chunk == 0) {
        if (mean_out) mean_out[image * p.groups + g0 + g] = m.mean;
        if (rstd_out) rstd_out[image * p.groups + g0 + g] = grstd[g];
      }
    }
  }
  __syncthreads();
  for (bool first = true; col < nv; col += threads, xc += threads * V, yc += threads * V, first = false) {
    Affine<T, V, kAct> f;
    f.set(p, col * V, gmean, grstd, gamma, beta);
    if (!first) ask(xc, rl);
    const T *from = xc;
    T *to = yc;
    for (uint32_t r = rl; r < rows; r += kAsk * lanes, to += kAsk * yp) {
      Pack<T, V> o[kAsk];
#pragma unroll
      for (int i = 0; i < kAsk; ++i) o[i] = v[i];
      from += kAsk * xp;
      if (r + kAsk * lanes < rows) ask(from, r + kAsk * lanes);  // the next ones, under these
#pragma unroll
      for (int i = 0; i < kAsk; ++i)
        if (r + i * lanes < rows) store_pack(to + i * yp, f(o[i], p));
    }
  }
}

template <typename T>
int run_norm(cudaStream_t s, int64_t n, const NormPlan &plan, const T *x, T *y, float *mean,
             float *rstd, float2 *partial) {
  const NormGeom &g = plan.g;
  return norm_with_pack<16 / sizeof(T)>(plan.v, g.act, [&](auto pack_size, auto act) {
    constexpr int V = decltype(pack_size)::value, kAct = decltype(act)::value;
    const int cw = g.gs * g.cg;
    const int tail = norm_tail_bytes(plan.threads, V, cw, g.gs);
    for (int64_t i = 0; i < n; i += plan.batch) {
      const int64_t count = n - i < plan.batch ? n - i : plan.batch;
      const T *xi = x + i * g.hw * g.ldx;
      T *yi = y + i * g.hw * g.ldy;
      float *mi = mean ? mean + i * g.groups : nullptr, *ri = rstd ? rstd + i * g.groups : nullptr;
      const int64_t ctas = count * g.strips * g.chunks * g.slices;
      if (plan.keep) {
        const int strip = static_cast<int>(
            align_up(static_cast<size_t>(g.cta_rows) * cw * sizeof(T), 16));
        if (int rc = norm_launch(norm_kernel<T, V, kAct, true>, ctas, plan.threads, strip + tail,
                                 g.slices, s, g, xi, yi, mi, ri, nullptr))
          return rc;
        continue;
      }
      if (int rc = norm_launch(norm_kernel<T, V, 0, false>, ctas, plan.threads, tail, g.slices, s, g,
                               xi, yi, mi, ri, partial))
        return rc;
      const uint32_t rows = static_cast<uint32_t>(ceil_div(g.hw, plan.apply_chunks));
      const int smem =
          (2 * g.chunks * g.gs + 2 * g.gs + 2 * cw) * static_cast<int>(sizeof(float));
      if (int rc = norm_launch(norm_apply_kernel<T, V, kAct>, count * g.strips * plan.apply_chunks,
                               plan.threads, smem, 1, s, g, xi, yi, mi, ri, partial,
                               make_fastdiv(static_cast<uint32_t>(plan.apply_chunks)), rows))
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
  if (!workspace || !norm_aligned(workspace, 256) ||
      workspace_bytes < norm_workspace(n, hw, c, groups))
    return kErrInvalidArg;
  const int fx = norm_pack_fit(x, ldx, size), fy = norm_pack_fit(y, ldy, size);
  NormPlan plan = plan_norm(n, hw, c, groups, size, fx < fy ? fx : fy, 1);
  plan.g.ldx = ldx;
  plan.g.ldy = ldy;
  plan.g.gamma = gamma;
  plan.g.beta = beta;
  plan.g.eps = eps;
  plan.g.act = act;
  plan.g.alpha = act_alpha;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float2 *partial = static_cast<float2 *>(workspace);
  if (dtype == NPLK_DTYPE_FP32)
    return run_norm(s, n, plan, static_cast<const float *>(x), static_cast<float *>(y), mean, rstd,
                    partial);
  if (dtype == NPLK_DTYPE_FP16)
    return run_norm(s, n, plan, static_cast<const __half *>(x), static_cast<__half *>(y), mean,
                    rstd, partial);
  return run_norm(s, n, plan, static_cast<const __nv_bfloat16 *>(x),
                  static_cast<__nv_bfloat16 *>(y), mean, rstd, partial);
}
