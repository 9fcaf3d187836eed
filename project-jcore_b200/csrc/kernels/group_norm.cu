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

template <int V>
struct Running {
  float n, mean[V], m2[V];
};

// Joins R rows, held as packs, to the running moments.
template <typename T, int V, int R>
__device__ __forceinline__ void join_rows(const Pack<T, V> (&p)[R], Running<V> &run) {
  const float total = run.n + static_cast<float>(R);
  const float share = static_cast<float>(R) * rcp_approx(total), cross = run.n * share;
  float x[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r) unpack(p[r], x[r]);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float mean = x[0][j], m2 = 0.0f;
    if (R > 1) {
#pragma unroll
      for (int r = 1; r < R; ++r) mean += x[r][j];
      mean *= 1.0f / static_cast<float>(R);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float e = x[r][j] - mean;
        m2 = fmaf(e, e, m2);
      }
    }
    const float d = mean - run.mean[j];
    run.mean[j] = fmaf(d, share, run.mean[j]);
    run.m2[j] = fmaf(d * d, cross, run.m2[j] + m2);
  }
  run.n = total;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Joins count moments that `at(i)` gives, in order.
template <typename F>
__device__ __forceinline__ Moments join_list(int count, F at) {
  Moments t{0.0f, 0.0f, 0.0f};
  for (int i = 0; i < count; ++i) {
    const Moments m = at(i);
    t.n += m.n;
    t.mean += m.n * m.mean;
  }
  t.mean = t.n > 0.0f ? t.mean / t.n : 0.0f;
  for (int i = 0; i < count; ++i) {
    const Moments m = at(i);
    const float d = m.mean - t.mean;
    if (m.n > 0.0f) t.m2 += m.m2 + m.n * d * d;
  }
  return t;
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

// The CTA's moments of each of its groups, from every thread's per-channel ones
// in s.mean, s.m2, to s.group. The warps are shared out over the groups.
__device__ __forceinline__ void cta_groups(const NormGeom &p, const NormPlace &w, const Shared &s) {
  const int warps = static_cast<int>(blockDim.x) >> 5, warp = threadIdx.x >> 5,
            lane = threadIdx.x & 31;
  const int each = max(1, warps / w.gsl), teams = warps / each;
  const int member = warp % each;
  const uint32_t base = w.rows / w.lanes, rest = w.rows - base * w.lanes;  // rows of a row lane
  for (int g = warp / each; g < w.gsl && warp < teams * each; g += teams) {
    const int entries = w.lanes * p.cg;
    float n = 0.0f, m = 0.0f, q = 0.0f;
    for (int e = member * 32 + lane; e < entries; e += each * 32) {
      const uint32_t l = fdiv(static_cast<uint32_t>(e), p.div_cg);
      const float k = static_cast<float>(base + (l < rest ? 1u : 0u));
      n += k;
      m += k * s.mean[l * w.cw + g * p.cg + (e - l * p.cg)];
    }
    n = warp_sum(n);
    m = warp_sum(m);
    const float mean = n > 0.0f ? m / n : 0.0f;
    for (int e = member * 32 + lane; e < entries; e += each * 32) {
      const uint32_t l = fdiv(static_cast<uint32_t>(e), p.div_cg);
      const float k = static_cast<float>(base + (l < rest ? 1u : 0u));
      const int i = l * w.cw + g * p.cg + (e - l * p.cg);
      const float d = s.mean[i] - mean;
      if (k > 0.0f) q += s.m2[i] + k * d * d;
    }
    q = warp_sum(q);
    if (lane == 0) s.team[g * each + member] = make_float4(n, mean, q, 0.0f);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < w.gsl; g += blockDim.x) {
    const Moments t = join_list(each, [&](int i) {
      const float4 v = s.team[g * each + i];
      return Moments{v.x, v.y, v.z};
    });
    s.group[g] = make_float4(t.n, t.mean, t.m2, 0.0f);
  }
}

// The normalised, scaled and activated values of one pack's channels.
template <typename T, int V, int kAct>
struct Affine {
  float mean[V], scale[V], shift[V];

  __device__ __forceinline__ void set(const NormGeom &p, int ch, const float *gmean,
                                      const float *grstd, const float *gamma, const float *beta) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t g = fdiv(static_cast<uint32_t>(ch + j), p.div_cg);
      mean[j] = gmean[g];
      scale[j] = grstd[g] * gamma[ch + j];
      shift[j] = beta[ch + j];
    }
  }
  __device__ __forceinline__ Pack<T, V> operator()(const Pack<T, V> &in, const NormGeom &p) const {
    float v[V];
    unpack(in, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = fmaf(v[j] - mean[j], scale[j], shift[j]);
    act_array<T>(v, kAct >= 0 ? kAct : p.act, p.alpha);
    return pack<T, V>(v);
  }
};

// First pass, and with kKeep the whole of it.
template <typename T, int V, int kAct, bool kKeep>
__global__ void __launch_bounds__(norm_most_threads(V), V == 8 ? 3 : 2) norm_kernel(NormGeom p, const T *x, T *y, float *mean_out,
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
    for (int j = 0; j < V; ++j) run.mean[j] = run.m2[j] = 0.0f;
    const T *xc = xs + col * V;
    if constexpr (kKeep) {
      // All of the thread's rows are asked for at once, in four groups of
      // copies; it reads back only what it copied, so no barrier.
      const uint32_t mine = w.rows > static_cast<uint32_t>(w.lane)
                                ? (w.rows - w.lane + lanes - 1) / lanes
                                : 0;
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
        for (; k < end; ++k) {
          const Pack<T, V> v[1] = {own[k * turn]};
          join_rows(v, run);
        }
      }
    } else {
      // Eight rows asked for at a time, joined four by four (the last ones singly).
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
        Pack<T, V> a[7];
#pragma unroll
        for (int i = 0; i < 7; ++i)
          if (r + i * lanes < w.rows) a[i] = load_pack<T, V>(at + i * pitch);
#pragma unroll
        for (int i = 0; i < 7; ++i)
          if (r + i * lanes < w.rows) {
            const Pack<T, V> one[1] = {a[i]};
            join_rows(one, run);
          }
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s.mean[w.lane * w.cw + col * V + j] = run.mean[j];
      s.m2[w.lane * w.cw + col * V + j] = run.m2[j];
    }
  }
  copy_async_wait<0>();
  __syncthreads();
  cta_groups(p, w, s);
  // The cluster's groups, in every CTA of it.
  if (p.slices > 1) {
    cluster_sync();
    for (int g = threadIdx.x; g < w.gsl; g += blockDim.x) {
      const uint32_t at = smem_u32(&s.group[g]);
      const Moments t = join_list(p.slices, [&](int i) {
        const uint4 v = ld_shared_cluster_v4(mapa_shared(at, static_cast<uint32_t>(i)));
        return Moments{__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z)};
      });
      s.gmean[g] = t.mean;
      s.grstd[g] = kKeep ? 1.0f / sqrtf(t.m2 / t.n + p.eps) : t.m2;
    }
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
// the image's end, which the first pass read last.
template <typename T, int V, int kAct>
__global__ void __launch_bounds__(norm_most_threads(V), V == 8 ? 3 : 2)
    norm_apply_kernel(NormGeom p, const T *x, T *y, float *mean_out, float *rstd_out,
                      const float2 *partial, int apply_chunks, uint32_t apply_rows) {
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t at = gridDim.x - 1 - blockIdx.x;
  const uint32_t piece = at / static_cast<uint32_t>(apply_chunks);
  const uint32_t chunk = at - piece * apply_chunks;
  const int64_t image = piece / static_cast<uint32_t>(p.strips);
  const int g0 = static_cast<int>(piece - image * p.strips) * p.gs;
  const int gsl = min(p.gs, p.groups - g0), cw = gsl * p.cg, nv = cw / V, c0 = g0 * p.cg;
  float *gmean = reinterpret_cast<float *>(smem), *grstd = gmean + p.gs;
  float *gamma = grstd + p.gs, *beta = gamma + p.gs * p.cg;
  griddep_wait();
  griddep_launch_dependents();
  for (int i = threadIdx.x; i < cw; i += blockDim.x) {
    gamma[i] = p.gamma ? p.gamma[c0 + i] : 1.0f;
    beta[i] = p.beta ? p.beta[c0 + i] : 0.0f;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t chunk_rows = p.cta_rows * p.slices;
  for (int g = warp; g < gsl; g += static_cast<int>(blockDim.x) >> 5) {
    float n = 0.0f, m = 0.0f, q = 0.0f;
    const float2 *from = partial + image * p.chunks * p.groups + g0 + g;
    auto count = [&](int i) {
      const uint64_t first = static_cast<uint64_t>(i) * chunk_rows;
      return first < p.hw ? static_cast<float>(min(chunk_rows, p.hw - static_cast<uint32_t>(first))) : 0.0f;
    };
    for (int i = lane; i < p.chunks; i += 32) {
      n += count(i);
      m += count(i) * from[static_cast<int64_t>(i) * p.groups].x;
    }
    n = warp_sum(n);
    const float mean = warp_sum(m) / n;
    for (int i = lane; i < p.chunks; i += 32) {
      const float2 v = from[static_cast<int64_t>(i) * p.groups];
      const float d = v.x - mean, k = count(i);
      if (k > 0.0f) q += v.y + k * static_cast<float>(p.cg) * d * d;
    }
    q = warp_sum(q);
    if (lane == 0) {
      gmean[g] = mean;
      grstd[g] = 1.0f / sqrtf(q / (n * static_cast<float>(p.cg)) + p.eps);
      if (chunk == 0) {
        if (mean_out) mean_out[image * p.groups + g0 + g] = mean;
        if (rstd_out) rstd_out[image * p.groups + g0 + g] = grstd[g];
      }
    }
  }
  __syncthreads();
  const int threads = static_cast<int>(blockDim.x), t = static_cast<int>(threadIdx.x);
  const uint32_t lanes = nv <= threads ? threads / nv : 1;
  const uint32_t rl = nv <= threads ? t / nv : 0;
  const int first_col = nv <= threads ? t - static_cast<int>(rl) * nv : t;
  const uint64_t begin = static_cast<uint64_t>(chunk) * apply_rows;
  if (begin >= p.hw || rl >= lanes) return;
  const uint32_t r0 = static_cast<uint32_t>(begin), rows = min(apply_rows, p.hw - r0);
  const T *xs = x + (image * p.hw + r0) * p.ldx + c0;
  T *ys = y + (image * p.hw + r0) * p.ldy + c0;
  for (int col = first_col; col < nv; col += threads) {
    Affine<T, V, kAct> f;
    f.set(p, col * V, gmean, grstd, gamma, beta);
    const T *xc = xs + col * V;
    T *yc = ys + col * V;
    const int64_t xp = static_cast<int64_t>(lanes) * p.ldx, yp = static_cast<int64_t>(lanes) * p.ldy;
    xc += static_cast<int64_t>(rl) * p.ldx;
    yc += static_cast<int64_t>(rl) * p.ldy;
    for (uint32_t r = rl; r < rows; r += 4 * lanes, xc += 4 * xp, yc += 4 * yp) {
      Pack<T, V> v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r + i * lanes < rows) v[i] = load_pack<T, V>(xc + i * xp);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r + i * lanes < rows) store_pack(yc + i * yp, f(v[i], p));
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
      const int smem = (2 * g.gs + 2 * cw) * static_cast<int>(sizeof(float));
      if (int rc = norm_launch(norm_apply_kernel<T, V, kAct>, count * g.strips * plan.apply_chunks,
                               plan.threads, smem, 1, s, g, xi, yi, mi, ri, partial,
                               plan.apply_chunks, rows))
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
