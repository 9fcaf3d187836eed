// Gradient of group norm with an activation, channels last.
//
// With xh = (x - mean) * rstd, z = gamma * xh + beta, dz = dy * act'(z), per image:
//   P[ch] = sum dz, Q[ch] = sum dz * xh over the pixels,
//   A = sum_ch gamma P, B = sum_ch gamma Q over the group,
//   dx = rstd * (gamma * dz - (A + xh * B) / M),
//   dgamma = sum Q, dbeta = sum P over the images.
//
// The first pass sums P and Q per thread and channel, then over the CTA's rows by
// halving, the cluster and the chunks, always in the same order. Kept form: x and
// dy of the strip stay in the cluster's shared memory (20 bytes of traffic a
// value less than reading them twice in fp32); otherwise two passes, image batch
// by image batch, as in the forward kernel.
#include "act_epilogue.cuh"
#include "group_norm.cuh"

namespace nplk {
namespace {

struct GradArgs {
  const float *mean, *rstd;  // [n][groups]
  float *channels;           // [n * chunks][2][c]: Q, P; or null
  float2 *groups;            // [n * chunks][groups]: A, B (two passes)
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

// xh and dz of one pack's channels, pairs of channels together.
template <typename T, int V, int kAct>
struct Chain {
  static constexpr int kPairs = (V + 1) / 2;
  float2 minus_mean[kPairs], rstd[kPairs], gamma[kPairs], beta[kPairs];

  // `each(j, group)` is called for the pack's channels with their groups.
  template <typename F>
  __device__ __forceinline__ void set(const NormGeom &p, int ch, const float *gmean,
                                      const float *grstd, const float *ga, const float *be,
                                      F each) {
    float m[V], r[V];
    int g = static_cast<int>(fdiv(static_cast<uint32_t>(ch), p.div_cg)), left = (g + 1) * p.cg - ch;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      m[j] = -gmean[g];
      r[j] = grstd[g];
      each(j, g);
      if (--left == 0) {
        left = p.cg;
        if (j + 1 < V) ++g;
      }
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int k = V == 1 ? 0 : 2 * j + 1;
      minus_mean[j] = make_float2(m[2 * j], m[k]);
      rstd[j] = make_float2(r[2 * j], r[k]);
      gamma[j] = make_float2(ga[ch + 2 * j], ga[ch + k]);
      beta[j] = make_float2(be[ch + 2 * j], be[ch + k]);
    }
  }
  __device__ __forceinline__ void operator()(const Pack<T, V> &x, const Pack<T, V> &dy,
                                             const NormGeom &p, float2 (&xh)[kPairs],
                                             float2 (&dz)[kPairs]) const {
    unpack_pairs(x, xh);
    float z[V];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      xh[j] = mul2(add2(xh[j], minus_mean[j]), rstd[j]);
      const float2 v = fma2(gamma[j], xh[j], beta[j]);
      z[2 * j] = v.x;
      if (V > 1) z[2 * j + (V > 1 ? 1 : 0)] = v.y;
    }
    act_slope_array<T>(z, kAct >= 0 ? kAct : p.act, p.alpha);
    unpack_pairs(dy, dz);
#pragma unroll
    for (int j = 0; j < kPairs; ++j)
      dz[j] = mul2(dz[j], make_float2(z[2 * j], z[V == 1 ? 0 : 2 * j + 1]));
  }
};

// dx of one pack from its chain and the group's sums over M:
// rstd gamma * dz - (rstd A + xh rstd B).
template <typename T, int V, int kAct>
struct Input {
  static constexpr int kPairs = (V + 1) / 2;
  Chain<T, V, kAct> chain;
  float2 a[kPairs], b[kPairs];  // -rstd A / M, -rstd B / M

  __device__ __forceinline__ void set(const NormGeom &p, int ch, const float *gmean,
                                      const float *grstd, const float *ga, const float *be,
                                      const float2 *ab) {
    float u[V], v[V];
    chain.set(p, ch, gmean, grstd, ga, be, [&](int j, int g) {
      u[j] = -grstd[g] * ab[g].x;
      v[j] = -grstd[g] * ab[g].y;
    });
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int k = V == 1 ? 0 : 2 * j + 1;
      a[j] = make_float2(u[2 * j], u[k]);
      b[j] = make_float2(v[2 * j], v[k]);
    }
  }
  __device__ __forceinline__ Pack<T, V> operator()(const Pack<T, V> &x, const Pack<T, V> &dy,
                                                   const NormGeom &p) const {
    float2 xh[kPairs], dz[kPairs];
    chain(x, dy, p, xh, dz);
    float o[V];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const float2 d =
          fma2(mul2(chain.rstd[j], chain.gamma[j]), dz[j], fma2(xh[j], b[j], a[j]));
      o[2 * j] = d.x;
      if (V > 1) o[2 * j + (V > 1 ? 1 : 0)] = d.y;
    }
    return pack<T, V>(o);
  }
};

struct GradShared {  // the dynamic shared memory, after the kept strips
  float *q, *p;          // [lanes][cw]
  float *gamma, *beta;   // [cw]
  float2 *group, *total; // A, B of the CTA's groups; of the cluster's, over M
  float *gmean, *grstd;  // [gs]
};

template <int V>
__device__ __forceinline__ GradShared grad_shared(uint8_t *at, const NormGeom &p) {
  const int cw = p.gs * p.cg;
  const int acc = max(static_cast<int>(blockDim.x) * V, cw);
  GradShared s;
  s.group = reinterpret_cast<float2 *>(at);
  s.total = s.group + p.gs;
  s.q = reinterpret_cast<float *>(s.total + p.gs);
  s.p = s.q + acc;
  s.gamma = s.p + acc;
  s.beta = s.gamma + cw;
  s.gmean = s.beta + cw;
  s.grstd = s.gmean + p.gs;
  return s;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int V, int kAct, bool kKeep>
__global__ void __launch_bounds__(kNormMostThreads, 2)
    norm_grad_kernel(NormGeom p, GradArgs g, const T *dy, const T *x, T *dx) {
  extern __shared__ __align__(16) uint8_t smem[];
  const NormPlace w = norm_place<V>(p);
  const size_t strip_bytes =
      kKeep ? (static_cast<size_t>(p.cta_rows) * p.gs * p.cg * sizeof(T) + 15) / 16 * 16 : 0;
  Pack<T, V> *xk = reinterpret_cast<Pack<T, V> *>(smem);
  Pack<T, V> *dk = reinterpret_cast<Pack<T, V> *>(smem + strip_bytes);
  const GradShared s = grad_shared<V>(smem + 2 * strip_bytes, p);
  griddep_wait();
  griddep_launch_dependents();
  const int c0 = w.g0 * p.cg;
  const int64_t row0 = w.image * p.hw + w.r0;
  const T *xs = x + row0 * p.ldx + c0, *ds = dy + row0 * p.lddy + c0;
  const uint32_t lanes = static_cast<uint32_t>(w.lanes);
  const uint32_t mine = w.mine;
  const uint32_t step = (mine + 3) / 4;
  // The thread's first row, and from one of its rows to the next.
  const int first = w.lane * w.nv, turn = w.lanes * w.nv;
  const T *xl = xs + static_cast<int64_t>(w.lane) * p.ldx;
  const T *dl = ds + static_cast<int64_t>(w.lane) * p.lddy;
  const int64_t xp = static_cast<int64_t>(lanes) * p.ldx, dp = static_cast<int64_t>(lanes) * p.lddy;
  auto ask = [&](int col) {  // the thread's rows of one pack, in four groups of copies
#pragma unroll 1
    for (uint32_t q = 0; q < 4; ++q) {
      const uint32_t end = min((q + 1) * step, mine);
#pragma unroll 2
      for (uint32_t k = q * step; k < end; ++k) {
        copy_pack_async<T, V>(xk + first + k * turn + col, xl + k * xp + col * V);
        copy_pack_async<T, V>(dk + first + k * turn + col, dl + k * dp + col * V);
      }
      copy_async_commit();
    }
  };
  if (kKeep && w.active) ask(w.col);  // the first turn's, under the loads below
  for (int i = threadIdx.x; i < w.cw; i += blockDim.x) {
    s.gamma[i] = p.gamma ? p.gamma[c0 + i] : 1.0f;
    s.beta[i] = p.beta ? p.beta[c0 + i] : 0.0f;
  }
  for (int i = threadIdx.x; i < w.gsl; i += blockDim.x) {
    s.gmean[i] = g.mean[w.image * p.groups + w.g0 + i];
    s.grstd[i] = g.rstd[w.image * p.groups + w.g0 + i];
  }
  __syncthreads();
  for (int col = w.active ? w.col : w.nv; col < w.nv; col += blockDim.x) {
    Chain<T, V, kAct> chain;
    chain.set(p, col * V, s.gmean, s.grstd, s.gamma, s.beta, [](int, int) {});
    constexpr int kPairs = (V + 1) / 2;
    float2 sp[kPairs], sq[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) sp[j] = sq[j] = both(0.0f);
    auto add = [&](const Pack<T, V> &a, const Pack<T, V> &b) {
      float2 xh[kPairs], dz[kPairs];
      chain(a, b, p, xh, dz);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        sp[j] = add2(sp[j], dz[j]);
        sq[j] = fma2(dz[j], xh[j], sq[j]);
      }
    };
    if constexpr (kKeep) {
      if (col != w.col) ask(col);
#pragma unroll 1
      for (uint32_t q = 0; q < 4; ++q) {
        if (q == 0) copy_async_wait<3>();
        else if (q == 1) copy_async_wait<2>();
        else if (q == 2) copy_async_wait<1>();
        else copy_async_wait<0>();
        const uint32_t end = min((q + 1) * step, mine);
#pragma unroll 2
        for (uint32_t k = q * step; k < end; ++k) {
          const int at = first + k * turn + col;
          add(xk[at], dk[at]);
        }
      }
    } else {
      const T *xc = xl + col * V, *dc = dl + col * V;
      for (uint32_t r = w.lane; r < w.rows; r += 4 * lanes, xc += 4 * xp, dc += 4 * dp) {
        Pack<T, V> a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r + i * lanes < w.rows) {
            a[i] = load_pack<T, V>(xc + i * xp);
            b[i] = load_pack<T, V>(dc + i * dp);
          }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r + i * lanes < w.rows) add(a[i], b[i]);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s.q[w.lane * w.cw + col * V + j] = (j & 1) ? sq[j / 2].y : sq[j / 2].x;
      s.p[w.lane * w.cw + col * V + j] = (j & 1) ? sp[j / 2].y : sp[j / 2].x;
    }
  }
  __syncthreads();
  // The CTA's sums per channel, by halving the row lanes.
  for (int n = w.lanes; n > 1;) {
    const int h = (n + 1) / 2;
    for (int i = threadIdx.x; i < (n - h) * w.cw; i += blockDim.x) {
      s.q[i] += s.q[i + h * w.cw];
      s.p[i] += s.p[i + h * w.cw];
    }
    n = h;
    __syncthreads();
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < w.gsl; i += static_cast<int>(blockDim.x) >> 5) {
    float a = 0.0f, b = 0.0f;
    for (int ch = i * p.cg + lane; ch < (i + 1) * p.cg; ch += 32) {
      a = fmaf(s.gamma[ch], s.p[ch], a);
      b = fmaf(s.gamma[ch], s.q[ch], b);
    }
    a = warp_sum(a);
    b = warp_sum(b);
    if (lane == 0) s.group[i] = make_float2(a, b);
  }
  if (p.slices > 1) cluster_sync();
  else __syncthreads();
  const float inv = 1.0f / (static_cast<float>(p.hw) * static_cast<float>(p.cg));
  // 8 lanes a group: one round trip to all CTAs of the cluster.
  for (int i = threadIdx.x; i < (w.gsl * 8 + 31) / 32 * 32; i += blockDim.x) {
    const int at = i >> 3, k = i & 7;
    float2 t = make_float2(0.0f, 0.0f);
    if (at < w.gsl && k < p.slices) {
      const uint32_t from = mapa_shared(smem_u32(&s.group[at]), static_cast<uint32_t>(k));
      t = make_float2(__uint_as_float(ld_shared_cluster_u32(from)),
                      __uint_as_float(ld_shared_cluster_u32(from + 4)));
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) {
      t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
      t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
    }
    if (at < w.gsl && k == 0) {
      if (kKeep) s.total[at] = make_float2(t.x * inv, t.y * inv);
      else if (w.rank == 0)
        g.groups[(w.image * p.chunks + w.chunk) * p.groups + w.g0 + at] = t;
    }
  }
  if (g.channels) {
    // Each CTA adds its share of the channels over the cluster.
    float *out = g.channels + (w.image * p.chunks + w.chunk) * 2 * p.c + c0;
    for (int ch = w.rank * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x); ch < w.cw;
         ch += p.slices * static_cast<int>(blockDim.x)) {
      float q[8], b[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = k < p.slices;
        const uint32_t r = in ? static_cast<uint32_t>(k) : 0u;
        q[k] = __uint_as_float(ld_shared_cluster_u32(mapa_shared(smem_u32(&s.q[ch]), r)));
        b[k] = __uint_as_float(ld_shared_cluster_u32(mapa_shared(smem_u32(&s.p[ch]), r)));
        if (!in) q[k] = b[k] = 0.0f;
      }
      out[ch] = ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
      out[p.c + ch] = ((b[0] + b[1]) + (b[2] + b[3])) + ((b[4] + b[5]) + (b[6] + b[7]));
    }
  }
  if constexpr (kKeep) {
    __syncthreads();
    T *os = dx + row0 * p.ldy + c0;
    for (int col = w.active ? w.col : w.nv; col < w.nv; col += blockDim.x) {
      Input<T, V, kAct> f;
      f.set(p, col * V, s.gmean, s.grstd, s.gamma, s.beta, s.total);
      const Pack<T, V> *xo = xk + first + col, *dn = dk + first + col;
      T *to = os + static_cast<int64_t>(w.lane) * p.ldy + col * V;
      const int64_t op = static_cast<int64_t>(lanes) * p.ldy;
#pragma unroll 2
      for (uint32_t r = w.lane; r < w.rows; r += lanes, xo += turn, dn += turn, to += op)
        store_pack(to, f(*xo, *dn, p));
    }
  }
  if (p.slices > 1) cluster_sync_relaxed();  // no CTA leaves while another reads its sums
}

// Second pass, rows from the image's end; the first ones are asked for before the
// chunks' sums are added.
template <typename T, int V, int kAct>
__global__ void __launch_bounds__(kNormMostThreads, 2)
    norm_grad_apply_kernel(NormGeom p, GradArgs g, const T *dy, const T *x, T *dx,
                           FastDiv apply_chunks, uint32_t apply_rows) {
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
  float2 *total = chunks + p.chunks * p.gs;
  float *gmean = reinterpret_cast<float *>(total + p.gs), *grstd = gmean + p.gs;
  float *gamma = grstd + p.gs, *beta = gamma + p.gs * p.cg;
  const int threads = static_cast<int>(blockDim.x), t = static_cast<int>(threadIdx.x);
  const uint32_t rl = nv <= threads ? fdiv(t, p.div_nv[last]) : 0;
  int col = t - static_cast<int>(rl) * nv;
  const uint64_t begin = static_cast<uint64_t>(chunk) * apply_rows;
  const uint32_t r0 = begin < p.hw ? static_cast<uint32_t>(begin) : p.hw;
  const uint32_t rows = min(apply_rows, p.hw - r0);
  const int64_t row = image * p.hw + r0 + rl;
  const int64_t xp = static_cast<int64_t>(lanes) * p.ldx, dp = static_cast<int64_t>(lanes) * p.lddy,
                op = static_cast<int64_t>(lanes) * p.ldy;
  const T *xc = x + row * p.ldx + c0 + col * V, *dc = dy + row * p.lddy + c0 + col * V;
  T *oc = dx + row * p.ldy + c0 + col * V;
  if (rl >= lanes) col = nv;
  griddep_wait();
  griddep_launch_dependents();
  Pack<T, V> xv[2], dv[2];
  auto ask = [&](const T *xf, const T *df, uint32_t r) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (r + i * lanes < rows) {
        xv[i] = load_pack<T, V>(xf + i * xp);
        dv[i] = load_pack<T, V>(df + i * dp);
      }
  };
  if (col < nv) ask(xc, dc, rl);
  for (int i = t; i < cw; i += threads) {
    gamma[i] = p.gamma ? p.gamma[c0 + i] : 1.0f;
    beta[i] = p.beta ? p.beta[c0 + i] : 0.0f;
  }
  for (int i = t; i < gsl; i += threads) {
    gmean[i] = g.mean[image * p.groups + g0 + i];
    grstd[i] = g.rstd[image * p.groups + g0 + i];
  }
  const int warp = t >> 5, lane = t & 31, warps = threads >> 5;
  for (int k = warp; k < p.chunks; k += warps)
    for (int i = lane; i < gsl; i += 32)
      chunks[k * gsl + i] = g.groups[(image * p.chunks + k) * p.groups + g0 + i];
  __syncthreads();
  const float inv = 1.0f / (static_cast<float>(p.hw) * static_cast<float>(p.cg));
  for (int i = warp; i < gsl; i += warps) {
    float a = 0.0f, b = 0.0f;
    for (int k = lane; k < p.chunks; k += 32) {
      a += chunks[k * gsl + i].x;
      b += chunks[k * gsl + i].y;
    }
    a = warp_sum(a);
    b = warp_sum(b);
    if (lane == 0) total[i] = make_float2(a * inv, b * inv);
  }
  __syncthreads();
  for (bool first = true; col < nv;
       col += threads, xc += threads * V, dc += threads * V, oc += threads * V, first = false) {
    Input<T, V, kAct> f;
    f.set(p, col * V, gmean, grstd, gamma, beta, total);
    if (!first) ask(xc, dc, rl);
    const T *xf = xc, *df = dc;
    T *to = oc;
    for (uint32_t r = rl; r < rows; r += 2 * lanes, to += 2 * op) {
      Pack<T, V> a[2], b[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[i] = xv[i];
        b[i] = dv[i];
      }
      xf += 2 * xp;
      df += 2 * dp;
      if (r + 2 * lanes < rows) ask(xf, df, r + 2 * lanes);  // the next ones, under these
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (r + i * lanes < rows) store_pack(to + i * op, f(a[i], b[i], p));
    }
  }
}

// dgamma and dbeta: the sums of `rows` rows [2][c]. A block takes 32 of the 2 c
// columns, its 8 warps every eighth row.
__global__ void __launch_bounds__(256)
    param_grad_kernel(int64_t rows, int c, const float *from, float *dgamma, float *dbeta) {
  __shared__ float part[8][32];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float s = 0.0f;
  if (i < 2 * static_cast<int64_t>(c)) {
#pragma unroll 4
    for (int64_t r = warp; r < rows; r += 8) s += from[r * 2 * c + i];
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && i < 2 * static_cast<int64_t>(c)) {
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += part[k][lane];
    float *out = i < c ? dgamma : dbeta;
    if (out) out[i < c ? i : i - c] = s;
  }
}

template <typename T>
int run_grad(cudaStream_t s, int64_t n, const NormPlan &plan, GradArgs args, const T *dy,
             const T *x, T *dx) {
  const NormGeom &g = plan.g;
  return norm_with_pack<16 / sizeof(T)>(plan.v, g.act, [&](auto pack_size, auto act) {
    constexpr int V = decltype(pack_size)::value, kAct = decltype(act)::value;
    const int cw = g.gs * g.cg;
    const int tail = norm_tail_bytes(plan.threads, V, cw, g.gs);
    for (int64_t i = 0; i < n; i += plan.batch) {
      const int64_t count = n - i < plan.batch ? n - i : plan.batch;
      GradArgs a = args;
      a.mean += i * g.groups;
      a.rstd += i * g.groups;
      if (a.channels) a.channels += i * g.chunks * 2 * g.c;
      const T *xi = x + i * g.hw * g.ldx, *di = dy + i * g.hw * g.lddy;
      T *oi = dx + i * g.hw * g.ldy;
      const int64_t ctas = count * g.strips * g.chunks * g.slices;
      if (plan.keep) {
        const int strip = static_cast<int>(
            align_up(static_cast<size_t>(g.cta_rows) * cw * sizeof(T), 16));
        if (int rc = norm_launch(norm_grad_kernel<T, V, kAct, true>, ctas, plan.threads,
                                 2 * strip + tail, g.slices, s, g, a, di, xi, oi))
          return rc;
        continue;
      }
      if (int rc = norm_launch(norm_grad_kernel<T, V, kAct, false>, ctas, plan.threads, tail,
                               g.slices, s, g, a, di, xi, oi))
        return rc;
      const uint32_t rows = static_cast<uint32_t>(ceil_div(g.hw, plan.apply_chunks));
      const int smem =
          (2 * g.chunks * g.gs + 4 * g.gs + 2 * cw) * static_cast<int>(sizeof(float));
      if (int rc = norm_launch(norm_grad_apply_kernel<T, V, kAct>,
                               count * g.strips * plan.apply_chunks, plan.threads, smem, 1, s, g, a,
                               di, xi, oi, make_fastdiv(static_cast<uint32_t>(plan.apply_chunks)), rows))
        return rc;
    }
    return kOk;
  });
}

}  // namespace
}  // namespace nplk

using namespace nplk;

extern "C" int nplk_group_norm_act_backward(void *stream, int64_t n, int64_t hw, int64_t c,
                                            int64_t groups, int dtype, const void *dy,
                                            int64_t lddy, const void *x, int64_t ldx,
                                            const float *mean, const float *rstd,
                                            const float *gamma, const float *beta, int act,
                                            float act_alpha, void *dx, int64_t lddx,
                                            float *dgamma, float *dbeta, void *workspace,
                                            size_t workspace_bytes) {
  const int size = dtype_bytes(dtype);
  if (!size || !dy || !x || !mean || !rstd || !dx || lddy < c || ldx < c || lddx < c || act < 0 ||
      act > 10)
    return kErrInvalidArg;
  if (int rc = norm_check(n, hw, c, groups)) return rc;
  if (!norm_aligned(dy, size) || !norm_aligned(x, size) || !norm_aligned(dx, size) ||
      (dx == dy && lddx != lddy) || (dx == x && lddx != ldx))
    return kErrInvalidArg;
  if (!workspace || !norm_aligned(workspace, 256) ||
      workspace_bytes < norm_workspace(n, hw, c, groups))
    return kErrInvalidArg;
  int fit = norm_pack_fit(x, ldx, size);
  fit = std::min(fit, norm_pack_fit(dy, lddy, size));
  fit = std::min(fit, norm_pack_fit(dx, lddx, size));
  NormPlan plan = plan_norm(n, hw, c, groups, size, fit, 2);
  plan.g.ldx = ldx;
  plan.g.ldy = lddx;
  plan.g.lddy = lddy;
  plan.g.gamma = gamma;
  plan.g.beta = beta;
  plan.g.act = act;
  plan.g.alpha = act_alpha;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // The workspace: [n * chunks][2][c] channel sums, then [n * chunks][groups] A, B.
  const int64_t rows = n * plan.g.chunks;
  GradArgs a{mean, rstd, nullptr, nullptr};
  float *channels = static_cast<float *>(workspace);
  a.channels = dgamma || dbeta ? channels : nullptr;
  a.groups = reinterpret_cast<float2 *>(channels + rows * 2 * c);
  int rc;
  if (dtype == NPLK_DTYPE_FP32)
    rc = run_grad(s, n, plan, a, static_cast<const float *>(dy), static_cast<const float *>(x),
                  static_cast<float *>(dx));
  else if (dtype == NPLK_DTYPE_FP16)
    rc = run_grad(s, n, plan, a, static_cast<const __half *>(dy), static_cast<const __half *>(x),
                  static_cast<__half *>(dx));
  else
    rc = run_grad(s, n, plan, a, static_cast<const __nv_bfloat16 *>(dy),
                  static_cast<const __nv_bfloat16 *>(x), static_cast<__nv_bfloat16 *>(dx));
  if (rc || !a.channels) return rc;
  return launch_programmatic(param_grad_kernel, dim3(static_cast<unsigned>(ceil_div(2 * c, 32))),
                             dim3(256), 0, s, rows, static_cast<int>(c), channels, dgamma, dbeta);
}
