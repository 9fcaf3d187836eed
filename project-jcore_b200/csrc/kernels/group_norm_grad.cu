// Gradient of group norm with an activation, channels last.
//
// With xh = (x - mean) * rstd, z = gamma * xh + beta, dz = dy * act'(z), per image:
//   P[ch] = sum dz, Q[ch] = sum dz * xh over the pixels,
//   A = sum_ch gamma P, B = sum_ch gamma Q over the group,
//   dx = rstd * (gamma * dz - (A + xh * B) / M),
//   dgamma = sum Q, dbeta = sum P over the images.
//
// P and Q are summed per thread and channel, then over the CTA's rows by halving,
// the cluster and the chunks, always in the same order. Kept form: x and dy of the
// strip stay in the cluster's shared memory, one launch for dx; otherwise sums of
// chunks, their joining, then dx, image batch by image batch so that the last
// launch finds x and dy in L2. The parameters' gradients are summed over the
// images by a last, small launch.
#include "act_epilogue.cuh"
#include "group_norm.cuh"

namespace nplk {
namespace {

struct GradArgs {
  const float *mean, *rstd;  // [n][groups]
  float *channels;           // [n * chunks][2][c]: Q, P; or null
  float2 *groups;            // [n * chunks][groups]: A, B (not kept)
};

// xh and dz of one pack's channels, pairs of channels together.
template <typename T, int V, int kAct>
struct Chain {
  static constexpr int kPairs = (V + 1) / 2;
  float2 minus_mean[kPairs], rstd[kPairs], gamma[kPairs], beta[kPairs];

  // `stat(g)`: mean, rstd and two values more of group g of the strip, the latter to
  // u and v per channel; ga, be of channel ch on (null: 1 and 0).
  template <typename F>
  __device__ __forceinline__ void set(const NormGeom &p, int ch, const float *ga, const float *be,
                                      float (&u)[V], float (&v)[V], F stat) {
    float m[V], r[V], w[V], b[V];
    int g = static_cast<int>(fdiv(static_cast<uint32_t>(ch), p.div_cg)), left = (g + 1) * p.cg - ch;
    float4 s0 = stat(g), s1 = s0;
    if (V > 1 && p.cg >= V && left < V) s1 = stat(g + 1);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (V > 1 && p.cg < V && j > 0 && left == 0) {
        s0 = stat(++g);
        left = p.cg;
      }
      const float4 s = V > 1 && p.cg >= V && j >= left ? s1 : s0;
      m[j] = -s.x;
      r[j] = s.y;
      u[j] = s.z;
      v[j] = s.w;
      w[j] = ga ? ga[j] : 1.0f;
      b[j] = be ? be[j] : 0.0f;
      if (V > 1 && p.cg < V) --left;
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int k = V == 1 ? 0 : 2 * j + 1;
      minus_mean[j] = make_float2(m[2 * j], m[k]);
      rstd[j] = make_float2(r[2 * j], r[k]);
      gamma[j] = make_float2(w[2 * j], w[k]);
      beta[j] = make_float2(b[2 * j], b[k]);
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

  // `stat(g)`: mean, rstd, A / M, B / M.
  template <typename F>
  __device__ __forceinline__ void set(const NormGeom &p, int ch, const float *ga, const float *be,
                                      F stat) {
    float u[V], v[V];
    chain.set(p, ch, ga, be, u, v, stat);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int k = V == 1 ? 0 : 2 * j + 1;
      const float2 r = chain.rstd[j];
      a[j] = make_float2(-r.x * u[2 * j], -r.y * u[k]);
      b[j] = make_float2(-r.x * v[2 * j], -r.y * v[k]);
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

struct GradShared {  // the dynamic shared memory, after the kept rows
  uint8_t *bars;
  float4 *stat;         // [gs]: mean, rstd, A / M, B / M
  float2 *all;          // [8][gs]: A, B of the cluster's CTAs
  float *q, *p;         // [lanes][pitch]
  float *gamma, *beta;  // [pitch]
  float *got;           // [slices][share][2], in clusters: Q, P of this CTA's share of the channels
};

template <int V>
__device__ __forceinline__ GradShared grad_shared(uint8_t *at, const NormGeom &p) {
  const int acc = max(static_cast<int>(blockDim.x) * V, p.pitch);
  GradShared s;
  s.bars = at;
  s.stat = reinterpret_cast<float4 *>(at + 64);
  s.all = reinterpret_cast<float2 *>(s.stat + p.gs);
  s.q = reinterpret_cast<float *>(s.all + 8 * p.gs);
  s.p = s.q + acc;
  s.gamma = s.p + acc;
  s.beta = s.gamma + p.pitch;
  s.got = s.beta + p.pitch;  // 2 * (pitch + 8) floats
  return s;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Kept rows are worked on four at a time: few warps fit beside them, and a value's
// chain of about twenty dependent instructions needs others to run under it
// (8 x 4096 x 320 bf16: 35.6 us against 37.8 with two rows; 64 x 196 x 512 fp32: 29.3
// against 31.4). 288 in its bounds means 112 registers: with 128, 4 x 1024 x 1920 took
// 31.3 us, with 112 25.7, with 80 27.2. Not kept it needs the 128 (4 x 16384 x 512: 99.9
// us, with 112 116).
constexpr int kGradBatch = 4;

template <typename T, int V, int kAct, bool kKeep>
__global__ void __launch_bounds__(kKeep ? 288 : kNormThreads, 2)
    norm_grad_kernel(const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ CUtensorMap map_dy, const NormGeom p,
                     const GradArgs g, const T *dy, const T *x, T *dx) {
  extern __shared__ __align__(128) uint8_t smem[];
  const NormPlace w = norm_place(p, blockIdx.x);
  const int64_t held = p.boxes ? static_cast<int64_t>(p.stage_rows) * kNormStages : p.cta_rows;
  const size_t strip_bytes = kKeep ? (held * p.pitch * sizeof(T) + 127) / 128 * 128
                                   : kNormRing * kNormThreads * sizeof(Pack<T, V>);
  Pack<T, V> *xk = reinterpret_cast<Pack<T, V> *>(smem);
  Pack<T, V> *dk = reinterpret_cast<Pack<T, V> *>(smem + strip_bytes);
  const GradShared s = grad_shared<V>(smem + 2 * strip_bytes, p);
  const int c0 = w.g0 * p.cg;
  const int64_t row0 = w.image * p.hw + w.r0;
  const uint32_t lanes = static_cast<uint32_t>(w.lanes);
  const int turn = w.lanes * (p.pitch / V);
  const int64_t xp = static_cast<int64_t>(lanes) * p.ldx, dp = static_cast<int64_t>(lanes) * p.lddy;
  const T *xl = x + (row0 + w.lane) * p.ldx + c0, *dl = dy + (row0 + w.lane) * p.lddy + c0;
  RowLoads<T, V, 2> loads;
  if (p.slices > 1) cluster_arrive_relaxed();
  if (kKeep) loads.prepare(p, s.bars);
  griddep_wait();
  griddep_launch_dependents();
  if (kKeep) loads.start(p, w, {&map_x, &map_dy}, {smem, smem + strip_bytes}, w.image * p.hw);
  for (int i = threadIdx.x; i < w.cw; i += blockDim.x) {
    s.gamma[i] = p.gamma ? p.gamma[c0 + i] : 1.0f;
    s.beta[i] = p.beta ? p.beta[c0 + i] : 0.0f;
  }
  for (int i = threadIdx.x; i < w.gsl; i += blockDim.x) {
    const int64_t at = w.image * p.groups + w.g0 + i;
    s.stat[i] = make_float4(g.mean[at], g.rstd[at], 0.0f, 0.0f);
  }
  __syncthreads();
  for (int col = w.active ? w.col : w.nv; col < w.nv; col += blockDim.x) {
    constexpr int kPairs = (V + 1) / 2;
    Chain<T, V, kAct> chain;
    float2 sp[kPairs], sq[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) sp[j] = sq[j] = both(0.0f);
    const int first = w.lane * (p.pitch / V) + col;
    const T *xc = xl + col * V, *dc = dl + col * V;
    if (kKeep && !p.boxes) {
      copy_rows(xk + first, turn, xc, xp, w.mine);
      copy_rows(dk + first, turn, dc, dp, w.mine);
      copy_async_commit();
    }
    {
      float none[V], more[V];
      chain.set(p, col * V, s.gamma + col * V, s.beta + col * V, none, more,
                [&](int k) { return s.stat[k]; });
    }
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
      if (!p.boxes) copy_async_wait<0>();
      const Pack<T, V> *xo = xk + first, *dn = dk + first;
      uint32_t k = 0;
      for (; k + kGradBatch <= w.mine; k += kGradBatch) {
        if (p.boxes) loads.wait(p, w.lane + (k + kGradBatch - 1) * lanes);
        Pack<T, V> a[kGradBatch], b[kGradBatch];
#pragma unroll
        for (int i = 0; i < kGradBatch; ++i) {
          a[i] = xo[i * turn];
          b[i] = dn[i * turn];
        }
#pragma unroll
        for (int i = 0; i < kGradBatch; ++i) add(a[i], b[i]);
        xo += kGradBatch * turn;
        dn += kGradBatch * turn;
      }
      if (p.boxes && k < w.mine) loads.wait(p, w.lane + (w.mine - 1) * lanes);
      for (; k < w.mine; ++k, xo += turn, dn += turn) add(*xo, *dn);
    } else {
      stream_rows<T, V, 2>(w.mine, {xc, dc}, {xp, dp}, xk,
                           [&](const Pack<T, V>(&v)[2][4], int rows) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < rows) add(v[0][i], v[1][i]);
      });
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
  if (p.slices > 1) cluster_wait();  // every CTA of it has started and may be written to
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < w.gsl; i += static_cast<int>(blockDim.x) >> 5) {
    float a = 0.0f, b = 0.0f;
    for (int ch = i * p.cg + lane; ch < (i + 1) * p.cg; ch += 32) {
      a = fmaf(s.gamma[ch], s.p[ch], a);
      b = fmaf(s.gamma[ch], s.q[ch], b);
    }
    a = warp_sum(a);
    b = warp_sum(b);
    if (lane < p.slices) {  // lane k to CTA k
      const uint32_t to = mapa_shared(smem_u32(&s.all[w.rank * p.gs + i]), lane);
      st_shared_cluster_f32(to, a);
      st_shared_cluster_f32(to + 4, b);
    }
  }
  const int share = (p.pitch + p.slices - 1) / p.slices;  // channels that a CTA adds up
  if (g.channels && p.slices > 1) {
    for (int ch = threadIdx.x; ch < w.cw; ch += blockDim.x) {
      const int owner = ch / share;
      const uint32_t to = mapa_shared(
          smem_u32(&s.got[2 * (w.rank * share + ch - owner * share)]), owner);
      st_shared_cluster_f32(to, s.q[ch]);
      st_shared_cluster_f32(to + 4, s.p[ch]);
    }
  }
  if (p.slices > 1) cluster_sync();
  else __syncthreads();
  const float inv = 1.0f / (static_cast<float>(p.hw) * static_cast<float>(p.cg));
  for (int i = threadIdx.x; i < (w.gsl * 8 + 31) / 32 * 32; i += blockDim.x) {
    const int at = i >> 3, k = i & 7;
    float2 t = at < w.gsl && k < p.slices ? s.all[k * p.gs + at] : make_float2(0.0f, 0.0f);
#pragma unroll
    for (int o = 4; o; o >>= 1) {
      t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
      t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
    }
    if (at < w.gsl && k == 0) {
      if (kKeep) {
        s.stat[at].z = t.x * inv;
        s.stat[at].w = t.y * inv;
      } else if (w.rank == 0) {
        g.groups[(w.image * p.chunks + w.chunk) * p.groups + w.g0 + at] = t;
      }
    }
  }
  if (g.channels) {
    float *out = g.channels + (w.image * p.chunks + w.chunk) * 2 * p.c + c0;
    for (int i = threadIdx.x; i < share && w.rank * share + i < w.cw; i += blockDim.x) {
      float q = s.q[i], b = s.p[i];  // of a CTA by itself
      if (p.slices > 1) q = b = 0.0f;
      for (int k = 0; p.slices > 1 && k < p.slices; ++k) {
        q += s.got[2 * (k * share + i)];
        b += s.got[2 * (k * share + i) + 1];
      }
      out[w.rank * share + i] = q;
      out[p.c + w.rank * share + i] = b;
    }
  }
  if constexpr (kKeep) {
    __syncthreads();
    for (int col = w.active ? w.col : w.nv; col < w.nv; col += blockDim.x) {
      Input<T, V, kAct> f;
      f.set(p, col * V, s.gamma + col * V, s.beta + col * V, [&](int k) { return s.stat[k]; });
      const int first = w.lane * (p.pitch / V) + col;
      const Pack<T, V> *xo = xk + first, *dn = dk + first;
      T *to = dx + (row0 + w.lane) * p.ldy + c0 + col * V;
      const int64_t op = static_cast<int64_t>(lanes) * p.ldy;
      uint32_t k = 0;
      for (; k + kGradBatch <= w.mine; k += kGradBatch) {
        Pack<T, V> v[kGradBatch];
#pragma unroll
        for (int i = 0; i < kGradBatch; ++i) v[i] = f(xo[i * turn], dn[i * turn], p);
#pragma unroll
        for (int i = 0; i < kGradBatch; ++i) store_pack(to + i * op, v[i]);
        xo += kGradBatch * turn;
        dn += kGradBatch * turn;
        to += kGradBatch * op;
      }
      for (; k < w.mine; ++k, xo += turn, dn += turn, to += op) store_pack(to, f(*xo, *dn, p));
    }
    loads.drain(p, w);
  }
}

// Adds the chunks' sums: a CTA per image and group; with its mean and rstd to stat.
__global__ void __launch_bounds__(128)
    norm_grad_join_kernel(const NormGeom p, const GradArgs g, float4 *stat) {
  __shared__ float2 warps[4];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t at = blockIdx.x, image = at / p.groups;
  const float2 *from = g.groups + image * p.chunks * p.groups + (at - image * p.groups);
  float a = 0.0f, b = 0.0f;
#pragma unroll 4
  for (int k = threadIdx.x; k < p.chunks; k += 128) {
    const float2 v = from[static_cast<int64_t>(k) * p.groups];
    a += v.x;
    b += v.y;
  }
  a = warp_sum(a);
  b = warp_sum(b);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  if (threadIdx.x == 0) {
    const float inv = 1.0f / (static_cast<float>(p.hw) * static_cast<float>(p.cg));
    a = (warps[0].x + warps[1].x) + (warps[2].x + warps[3].x);
    b = (warps[0].y + warps[1].y) + (warps[2].y + warps[3].y);
    stat[at] = make_float4(g.mean[at], g.rstd[at], a * inv, b * inv);
  }
}

// dx: CTAs and threads as in the sums' pass, the images and rows in the other
// order, so that what that pass read last comes first, out of L2.
template <typename T, int V, int kAct>
__global__ void __launch_bounds__(kNormThreads, 2)
    norm_grad_apply_kernel(const NormGeom p, const float4 *stat, const T *dy, const T *x, T *dx) {
  extern __shared__ __align__(128) uint8_t smem[];
  const NormPlace w = norm_place(p, gridDim.x - 1 - blockIdx.x);
  Pack<T, V> *ring = reinterpret_cast<Pack<T, V> *>(smem);
  griddep_wait();
  griddep_launch_dependents();
  if (w.mine == 0) return;
  // the thread's last row first
  const int64_t row = w.image * p.hw + w.r0 + w.lane + static_cast<int64_t>(w.mine - 1) * w.lanes;
  const int64_t xp = -static_cast<int64_t>(w.lanes) * p.ldx,
                dp = -static_cast<int64_t>(w.lanes) * p.lddy,
                op = -static_cast<int64_t>(w.lanes) * p.ldy;
  const float4 *st = stat + w.image * p.groups + w.g0;
  for (int col = w.col; col < w.nv; col += blockDim.x) {
    const int ch = w.g0 * p.cg + col * V;
    T *to = dx + row * p.ldy + ch;
    Input<T, V, kAct> f;
    bool ready = false;
    stream_rows<T, V, 2>(w.mine, {x + row * p.ldx + ch, dy + row * p.lddy + ch}, {xp, dp}, ring,
                         [&](const Pack<T, V>(&v)[2][4], int rows) {
      if (!ready) {  // the channels' constants arrive under the first rows
        f.set(p, col * V, p.gamma ? p.gamma + ch : nullptr, p.beta ? p.beta + ch : nullptr,
              [&](int k) { return st[k]; });
        ready = true;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < rows) store_pack(to + i * op, f(v[0][i], v[1][i], p));
      to += 4 * op;
    });
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
int run_grad(cudaStream_t s, int64_t n, const NormPlan &plan, const GradArgs &args, float4 *stat,
             const T *dy, const T *x, T *dx) {
  const NormGeom &g = plan.g;
  return norm_with_pack<4>(plan.v, g.act, [&](auto pack_size, auto act) {
    constexpr int V = decltype(pack_size)::value, kAct = decltype(act)::value;
    const int tail = norm_tail_bytes(plan.threads, V, g.pitch, g.gs, plan.keep);
    for (int64_t i = 0; i < n; i += plan.batch) {
      const int64_t count = std::min(n - i, plan.batch);
      GradArgs a = args;
      a.mean += i * g.groups;
      a.rstd += i * g.groups;
      if (a.channels) a.channels += i * g.chunks * 2 * g.c;
      const T *xi = x + i * g.hw * g.ldx, *di = dy + i * g.hw * g.lddy;
      T *oi = dx + i * g.hw * g.ldy;
      const int64_t ctas = count * g.strips * g.chunks * g.slices;
      CUtensorMap mx = {}, md = {};
      if (plan.keep) {
        int rc = kOk;
        if (g.boxes)
          rc = encode_tmap_2d_plain(&mx, xi, g.c, count * g.hw, g.ldx * sizeof(T), g.pitch,
                                    g.box_rows, sizeof(T));
        if (!rc && g.boxes)
          rc = encode_tmap_2d_plain(&md, di, g.c, count * g.hw, g.lddy * sizeof(T), g.pitch,
                                    g.box_rows, sizeof(T));
        if (!rc)
          rc = norm_launch(norm_grad_kernel<T, V, kAct, true>, ctas, plan.threads,
                           2 * norm_rows_bytes(g, sizeof(T)) + tail, g.slices, s, mx, md, g, a, di,
                           xi, oi);
        if (rc) return rc;
        continue;
      }
      if (int rc = norm_launch(norm_grad_kernel<T, V, kAct, false>, ctas, plan.threads,
                               2 * norm_ring_bytes(V, sizeof(T)) + tail, g.slices, s, mx, md, g,
                               a, di, xi, oi))
        return rc;
      if (int rc = norm_launch(norm_grad_join_kernel, count * g.groups, 128, 0, 1, s, g, a, stat))
        return rc;
      if (int rc = norm_launch(norm_grad_apply_kernel<T, V, kAct>, ctas, plan.threads,
                               2 * norm_ring_bytes(V, sizeof(T)), 1, s, g, stat, di, xi, oi))
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
  for (const float *p : {mean, rstd, gamma, beta, static_cast<const float *>(dgamma),
                         static_cast<const float *>(dbeta)})
    if (!norm_aligned(p, 4)) return kErrInvalidArg;
  int fit = norm_pack_fit(x, ldx, size);
  fit = std::min(fit, norm_pack_fit(dy, lddy, size));
  fit = std::min(fit, norm_pack_fit(dx, lddx, size));
  // Four values a pack also in 16-bit types: with eight, the constants and sums of a
  // pack's channels leave half as many warps on an SM (8 x 4096 x 320 bf16: 41.8 us
  // against 37.5; 1 x 64 x 1280: 9.9 against 7.0).
  fit = std::min(fit, 4);
  NormPlan plan = plan_norm({n, hw, c, groups, size, fit, 2});
  const NormWork room = norm_work(plan, n, 2);
  if (!workspace || !norm_aligned(workspace, 256) ||
      workspace_bytes < std::max(kNormWorkLeast, room.bytes()))
    return kErrInvalidArg;
  plan.g.ldx = ldx;
  plan.g.ldy = lddx;
  plan.g.lddy = lddy;
  plan.g.gamma = gamma;
  plan.g.beta = beta;
  plan.g.act = act;
  plan.g.alpha = act_alpha;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  plan.g.status = device_status_word();
  if (!plan.g.status) return kErrInternal;
  const int64_t rows = n * plan.g.chunks;
  GradArgs a{mean, rstd, nullptr, nullptr};
  float4 *stat = static_cast<float4 *>(workspace);
  a.groups = reinterpret_cast<float2 *>(static_cast<float *>(workspace) + room.stats);
  float *channels = static_cast<float *>(workspace) + room.stats + room.partial;
  a.channels = dgamma || dbeta ? channels : nullptr;
  int rc;
  if (dtype == NPLK_DTYPE_FP32)
    rc = run_grad(s, n, plan, a, stat, static_cast<const float *>(dy),
                  static_cast<const float *>(x), static_cast<float *>(dx));
  else if (dtype == NPLK_DTYPE_FP16)
    rc = run_grad(s, n, plan, a, stat, static_cast<const __half *>(dy),
                  static_cast<const __half *>(x), static_cast<__half *>(dx));
  else
    rc = run_grad(s, n, plan, a, stat, static_cast<const __nv_bfloat16 *>(dy),
                  static_cast<const __nv_bfloat16 *>(x), static_cast<__nv_bfloat16 *>(dx));
  if (rc || !a.channels) return rc;
  return launch_programmatic(param_grad_kernel, dim3(static_cast<unsigned>(ceil_div(2 * c, 32))),
                             dim3(256), 0, s, rows, static_cast<int>(c), channels, dgamma, dbeta);
}
