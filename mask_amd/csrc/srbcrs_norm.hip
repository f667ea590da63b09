// Group norm with an activation over channels-last features:
//   y = act((x - mean) * rstd * w + b), mean and rstd of a sample's rows and a
//   group's channels;  backward with du = dy act'(u):
//   dw = sum du xhat, db = sum du, dx = rstd (du w - mean(du w) - xhat mean(du w xhat)).
//
// Every thread keeps one vector of channels and walks rows, so nothing is
// divided per element, loads of a row are whole lines and a thread's channels
// may belong to several groups.  Three forms:
//  - samples of one row (nodes normalised by themselves): a group in adjacent lanes;
//  - a sample that fits the registers of one workgroup is read once, its
//    variance taken as the mean of squared differences from the mean;
//  - a longer one is split along its rows: partial statistics of each channel
//    (mean and squared differences, joined pairwise, so that a large mean costs no
//    digits), one small kernel that joins them, and a second pass.
// Partial sums are 32 bits, joined in 64 in a fixed order.
//
// relu's slope jumps at u = 0, so a rounding of u there switches whole
// gradient entries (one of 60 million channels of nodes is 5e-4 of its weight's gradient). Mean, rstd and rstd w are
// therefore kept as two floats each, and relu's u is summed from both, in the forward and the backward pass
// alike: what decides its sign is the statistics' own error.  Of float32 samples of one row, or of few (a thread has one),
// summed in 64 bits, that is about 1e-14.  In the others, and in 16 bits, a thread adds its values in 32 bits: the mean is off by up to
// 2^-24 of them and the variance by 2^-24 of itself a value that a thread adds, mostly far less, as the threads'
// errors are of either sign.  It costs no time: the passes wait for memory.
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/srbcrs.h"
#include "srbcrs_ops.h"

namespace srbcrs {
namespace {

constexpr float kLog2e = 1.44269504088896341f;

// The normal distribution's probability below u, and exp(-u^2 / 2).  Below -|u| it is exp(-u^2 / 2) t P(t) with
// t = 1 / (1 + 0.3 |u| / sqrt 2): P is fitted to it by least squares reweighted towards the least
// largest relative error, 2e-8 down to u = -14, so that gelu's negative tail, which is this alone, keeps its digits as
// far as exp does.  Four terms fewer lose 2e-3 of it at -5, more than a rounding to float16, and save 2 % at most (20000 x
// 13 x 1000, bfloat16, forward: 610 us for 621).
__device__ __forceinline__ float normal_cdf(float u, float& e) {
  e = __builtin_amdgcn_exp2f(u * u * (-0.5f * kLog2e));
  const float t = __builtin_amdgcn_rcpf(fmaf(0.212132034f, fabsf(u), 1.f));
  float p = -0.06476129575f;
  p = fmaf(p, t, 0.2427808618f), p = fmaf(p, t, -0.2561375458f);
  p = fmaf(p, t, 0.273858342f), p = fmaf(p, t, -0.04732423627f);
  p = fmaf(p, t, 0.1074625614f), p = fmaf(p, t, 0.07416970176f);
  p = fmaf(p, t, 0.08535759755f), p = fmaf(p, t, 0.08459400352f);
  const float q = p * t * e;
  return u < 0.f ? q : 1.f - q;
}
__device__ __forceinline__ float sigmoid(float u) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-u * kLog2e));
}

// NaN stays NaN under every activation; relu of it too
template <int V>
__device__ __forceinline__ void act_all(int act, float (&u)[V]) {
  switch (act) {
    case SRBCRS_ACT_RELU:
#pragma unroll
      for (int e = 0; e < V; ++e) u[e] = u[e] < 0.f ? 0.f : u[e];
      break;
    case SRBCRS_ACT_SILU:
#pragma unroll
      for (int e = 0; e < V; ++e) u[e] = u[e] == -INFINITY ? 0.f : u[e] * sigmoid(u[e]);
      break;
    case SRBCRS_ACT_GELU:
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float x;
        u[e] = u[e] == -INFINITY ? 0.f : u[e] * normal_cdf(u[e], x);
      }
      break;
    default: break;
  }
}
// d act / d u
template <int V>
__device__ __forceinline__ void slope_all(int act, float (&u)[V]) {
  switch (act) {
    case SRBCRS_ACT_RELU:
#pragma unroll
      for (int e = 0; e < V; ++e) u[e] = u[e] > 0.f ? 1.f : u[e] == u[e] ? 0.f : u[e];
      break;
    case SRBCRS_ACT_SILU:
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float s = sigmoid(u[e]);
        u[e] = s * fmaf(u[e], 1.f - s, 1.f);
      }
      break;
    case SRBCRS_ACT_GELU:
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float x;
        const float c = normal_cdf(u[e], x);
        u[e] = fmaf(u[e] * 0.39894228040143268f, x, c);
      }
      break;
    default:
#pragma unroll
      for (int e = 0; e < V; ++e) u[e] = 1.f;
  }
}

template <class T, int V>
struct VecOf { typedef T type __attribute__((ext_vector_type(V))); };
template <class T>
struct VecOf<T, 1> { typedef T type; };
template <class T, int V>
using Vec = typename VecOf<T, V>::type;
template <class T, int V>
__device__ __forceinline__ void widen(const Vec<T, V>& v, float (&f)[V]) {
  if constexpr (V == 1) f[0] = (float)v;
  else
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (float)v[e];
}
template <class T, int V>
__device__ __forceinline__ Vec<T, V> narrow(const float (&f)[V]) {
  Vec<T, V> v;
  if constexpr (V == 1) v = (T)f[0];
  else
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)f[e];
  return v;
}
__device__ __forceinline__ float param(const void* p, int dtype, int64_t i, float none) {
  if (!p) return none;
  return dtype == kF32T ? ((const float*)p)[i] : dtype == kBf16T ? (float)((const __bf16*)p)[i] : (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ void put_param(void* p, int dtype, int64_t i, float v) {
  if (dtype == kF32T) ((float*)p)[i] = v;
  else if (dtype == kBf16T) ((__bf16*)p)[i] = (__bf16)v;
  else ((_Float16*)p)[i] = (_Float16)v;
}

struct Shape {
  int64_t batch, length;
  int channels, groups, per_group;   // per_group: channels of a group
  int64_t ldx, batch_x, lddy, batch_dy;
  const void *weight, *bias;
  int param_dtype, act;
  float eps;
};

// mean, rstd and their low parts (stats, as the backward pass reads them)
__device__ __forceinline__ float4 pack_stats(double mean, double var, float eps) {
  const float m = (float)mean;
  const double v2 = var + (double)eps;
  const float v = (float)v2, vl = (float)(v2 - v), r = 1.f / sqrtf(v);
  // 1 - v r^2 to second order: what r lacks
  const float p = r * r, pl = fmaf(r, r, -p), e = fmaf(-v, p, 1.f) - fmaf(v, pl, vl * p);
  return make_float4(m, r, (float)(mean - m), 0.5f * r * e);
}

// A thread's channels: statistics of their groups, and a = rstd w in two parts.
template <int V>
struct Affine {
  float mean[V], rstd[V], a[V], b[V], mean_lo[V], a_lo[V], w[V];
  __device__ __forceinline__ void params(const Shape& sh, int c0) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[e] = param(sh.weight, sh.param_dtype, c0 + e, 1.f);
      b[e] = param(sh.bias, sh.param_dtype, c0 + e, 0.f);
    }
  }
  __device__ __forceinline__ void stats(int e, float4 st) {
    mean[e] = st.x, rstd[e] = st.y, mean_lo[e] = st.z;
    a[e] = st.y * w[e];
    a_lo[e] = fmaf(st.y, w[e], -a[e]) + st.w * w[e];
  }
  // f: x, becomes (x - mean) * rstd where the caller asks for it; u: x's place before the activation
  template <bool HAT>
  __device__ __forceinline__ void apply(int act, float (&f)[V], float (&u)[V]) const {
    if (act == SRBCRS_ACT_RELU) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = f[e] - mean[e], t = d - f[e];
        const float lost = (f[e] - (d - t)) - (mean[e] + t);   // f - mean = d + lost
        const float low = fmaf(d, a_lo[e], (lost - mean_lo[e]) * a[e]);
        u[e] = fmaf(d, a[e], b[e]) + low;
        f[e] = d;
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[e] -= mean[e];
        u[e] = fmaf(f[e], a[e], b[e]);
      }
    }
    if constexpr (HAT)
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] *= rstd[e];
  }
};

// ---- a sample in one workgroup's registers ----------------------------------
//
// x (and dy) are read once; what bounds it is the wait for the other threads, twice forward and once backward.
// 20000 x 5 x 96 in 8 groups, float32, relu: 31 us forward (2.5 TB/s), 37 backward (3.1).

struct Small {
  int row_threads;   // threads along a sample's rows
  int vectors;       // threads along its channels
  int samples;       // samples of a workgroup at a time
  int lanes;         // threads that join one group: a power of two, 64 at most
};

// Sums of `v` over each group of each of the workgroup's samples: end(i, sums) in one
// thread for i = sample * groups + group.  All threads of the workgroup call it, and
// what `end` leaves in LDS is there for all afterwards.
template <int V, int N, class R, class F>
__device__ __forceinline__ void group_sums(const Shape& sh, const Small& sm, bool on, int s, int rt, int cv,
                                           R (&v)[N][V], R* red, F&& end) {
  const bool whole = sh.per_group % V == 0;   // a vector lies in one group
  const int width = whole ? sm.vectors : sh.channels, per = whole ? sh.per_group / V : sh.per_group;
  const int slice = sm.samples * sm.row_threads * width, ns = sm.samples * sh.groups;
  if (on) {
    const int at = (s * sm.row_threads + rt) * width;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (whole) {
        R t = v[k][0];
#pragma unroll
        for (int e = 1; e < V; ++e) t += v[k][e];
        red[k * slice + at + cv] = t;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) red[k * slice + at + cv * V + e] = v[k][e];
      }
    }
  }
  __syncthreads();
  // a lane takes every sm.lanes-th entry (row, channel of the group)
  const int lane = threadIdx.x & (sm.lanes - 1), step = blockDim.x / sm.lanes;
  const int rows_on = sm.lanes / per, cols_on = sm.lanes - rows_on * per, r0 = lane / per, j0 = lane - r0 * per;
  for (int base = 0; base < ns; base += step) {
    const int i = base + threadIdx.x / sm.lanes;
    double t[N];
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = 0.;
    if (i < ns) {
      const int si = i / sh.groups, g = i - si * sh.groups;
      const R* in = red + si * sm.row_threads * width + g * per;
      for (int r = r0, j = j0; r < sm.row_threads;) {
#pragma unroll
        for (int k = 0; k < N; ++k) t[k] += in[k * slice + r * width + j];
        r += rows_on, j += cols_on;
        if (j >= per) j -= per, ++r;
      }
    }
    for (int d = sm.lanes / 2; d; d >>= 1)
#pragma unroll
      for (int k = 0; k < N; ++k) t[k] += __shfl_xor(t[k], d);
    if (i < ns && lane == 0) end(i, t);
  }
  __syncthreads();
}
// what a thread's channels have of their groups' values: one read where they lie in one group
template <int V, class P>
__device__ __forceinline__ void of_groups(P (&to)[V], const P* from, const int (&g)[V], bool whole) {
  if (whole) {
    const P v = from[g[0]];
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = v;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = from[g[e]];
  }
}

// threads of a workgroup at most: single channels a thread leave registers for twice as many
__host__ __device__ constexpr int small_threads(int v) { return v == 1 ? 1024 : 512; }

// A thread's sums of the statistics: 64 bits where a thread has one row of 32 bits, for relu's side
template <class T, int NR>
using SmallSum = std::conditional_t<sizeof(T) == 4 && NR == 1, double, float>;

template <class T, int V, int NR>
__global__ __launch_bounds__(small_threads(V)) void k_norm_small(Shape sh, Small sm, const T* __restrict__ x, T* __restrict__ y,
                                                     float4* __restrict__ stats) {
  extern __shared__ double sums[];   // of each group of each sample the mean and its statistics, then the threads' sums
  float4* st = (float4*)(sums + ((sm.samples * sh.groups + 1) & ~1));
  using R = SmallSum<T, NR>;
  R* red = (R*)(st + sm.samples * sh.groups);
  const int per_sample = sm.row_threads * sm.vectors;
  const int s = threadIdx.x / per_sample, u = threadIdx.x - s * per_sample, rt = u / sm.vectors, cv = u - rt * sm.vectors;
  const int c0 = cv * V;
  Affine<V> af;
  int g[V] = {};
  const bool whole = sh.per_group % V == 0;
  if (s < sm.samples) {
    af.params(sh, c0);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = s * sh.groups + (c0 + e) / sh.per_group;
  }
  const double inv = 1. / ((double)sh.length * sh.per_group);
  for (int64_t n0 = (int64_t)blockIdx.x * sm.samples; n0 < sh.batch; n0 += (int64_t)gridDim.x * sm.samples) {
    const bool on = s < sm.samples && n0 + s < sh.batch;
    const T* xs = x + (n0 + s) * sh.batch_x + c0;
    Vec<T, V> raw[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (on && rt + i * sm.row_threads < sh.length)
        raw[i] = *(const Vec<T, V>*)(xs + (rt + i * sm.row_threads) * sh.ldx);
    R t[1][V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[0][e] = 0;
    if (on)
#pragma unroll
      for (int i = 0; i < NR; ++i)
        if (rt + i * sm.row_threads < sh.length) {
          float f[V];
          widen<T, V>(raw[i], f);
#pragma unroll
          for (int e = 0; e < V; ++e) t[0][e] += f[e];
        }
    group_sums<V, 1>(sh, sm, on, s, rt, cv, t, red, [&](int i, const double(&v)[1]) { sums[i] = v[0] * inv; });
    if (on) {
      double mean64[V];
      of_groups<V>(mean64, sums, g, whole);
      R mean[V];
#pragma unroll
      for (int e = 0; e < V; ++e) mean[e] = (R)mean64[e], t[0][e] = 0;
#pragma unroll
      for (int i = 0; i < NR; ++i)
        if (rt + i * sm.row_threads < sh.length) {
          float f[V];
          widen<T, V>(raw[i], f);
#pragma unroll
          for (int e = 0; e < V; ++e) t[0][e] = fma(f[e] - mean[e], f[e] - mean[e], t[0][e]);
        }
    }
    group_sums<V, 1>(sh, sm, on, s, rt, cv, t, red, [&](int i, const double(&v)[1]) {
      const float4 p = pack_stats(sums[i], v[0] * inv, sh.eps);
      st[i] = p;
      if (n0 + i / sh.groups < sh.batch) stats[n0 * sh.groups + i] = p;
    });
    if (on) {
      float4 sv[V];
      of_groups<V>(sv, st, g, whole);
#pragma unroll
      for (int e = 0; e < V; ++e) af.stats(e, sv[e]);
      T* ys = y + ((n0 + s) * sh.length) * sh.channels + c0;
#pragma unroll
      for (int i = 0; i < NR; ++i)
        if (rt + i * sm.row_threads < sh.length) {
          float f[V], o[V];
          widen<T, V>(raw[i], f);
          af.template apply<false>(sh.act, f, o);
          act_all<V>(sh.act, o);
          *(Vec<T, V>*)(ys + (int64_t)(rt + i * sm.row_threads) * sh.channels) = narrow<T, V>(o);
        }
    }
  }
}

// This workgroup's part of the parameters' gradients: the sum of its `rows` threads
// of a channel, lds[row][channel].  All threads of the workgroup call both.
template <int V>
__device__ __forceinline__ void put_params(const Shape& sh, bool on, int row, int c0, const float (&dw)[V], const float (&db)[V],
                                           float2* lds) {
  if (on)
#pragma unroll
    for (int e = 0; e < V; ++e) lds[row * sh.channels + c0 + e] = make_float2(dw[e], db[e]);
}
__device__ __forceinline__ void join_params(const Shape& sh, int rows, const float2* lds, float2* __restrict__ part) {
  __syncthreads();
  for (int c = threadIdx.x; c < sh.channels; c += blockDim.x) {
    double2 a = make_double2(0., 0.);
    for (int r = 0; r < rows; ++r) {
      const float2 o = lds[r * sh.channels + c];
      a.x += o.x, a.y += o.y;
    }
    part[(int64_t)blockIdx.x * sh.channels + c] = make_float2((float)a.x, (float)a.y);
  }
}

template <class T, int V, int NR>
__global__ __launch_bounds__(small_threads(V)) void k_norm_small_bwd(Shape sh, Small sm, const T* __restrict__ x,
                                                         const T* __restrict__ dy, T* __restrict__ dx,
                                                         const float4* __restrict__ stats, float2* __restrict__ part) {
  extern __shared__ double sums[];   // of each group of each sample two means, then the threads' sums
  float2* means = (float2*)sums;
  float* red = (float*)(means + sm.samples * sh.groups);
  const int per_sample = sm.row_threads * sm.vectors;
  const int s = threadIdx.x / per_sample, u = threadIdx.x - s * per_sample, rt = u / sm.vectors, cv = u - rt * sm.vectors;
  const int c0 = cv * V;
  float dw[V], db[V];
  Affine<V> af;
  int g[V] = {};
  const bool whole = sh.per_group % V == 0;
#pragma unroll
  for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.f;
  if (s < sm.samples) {
    af.params(sh, c0);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = (c0 + e) / sh.per_group;
  }
  const double inv = 1. / ((double)sh.length * sh.per_group);
  for (int64_t n0 = (int64_t)blockIdx.x * sm.samples; n0 < sh.batch; n0 += (int64_t)gridDim.x * sm.samples) {
    const bool on = s < sm.samples && n0 + s < sh.batch;
    const T *xs = x + (n0 + s) * sh.batch_x + c0, *ds = dy + (n0 + s) * sh.batch_dy + c0;
    Vec<T, V> raw[NR], rd[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (on && rt + i * sm.row_threads < sh.length) {
        raw[i] = *(const Vec<T, V>*)(xs + (rt + i * sm.row_threads) * sh.ldx);
        rd[i] = *(const Vec<T, V>*)(ds + (rt + i * sm.row_threads) * sh.lddy);
      }
    float t[2][V], f[V], d[V], u2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[0][e] = t[1][e] = 0.f;
    if (on) {
      float4 sv[V];
      of_groups<V>(sv, stats + (n0 + s) * sh.groups, g, whole);
#pragma unroll
      for (int e = 0; e < V; ++e) af.stats(e, sv[e]);
#pragma unroll
      for (int i = 0; i < NR; ++i)
        if (rt + i * sm.row_threads < sh.length) {
          widen<T, V>(raw[i], f);
          widen<T, V>(rd[i], d);
          af.template apply<true>(sh.act, f, u2);
          slope_all<V>(sh.act, u2);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float du = d[e] * u2[e];
            db[e] += du;
            dw[e] = fmaf(du, f[e], dw[e]);
            t[0][e] = fmaf(du, af.w[e], t[0][e]);
            t[1][e] = fmaf(du * af.w[e], f[e], t[1][e]);
          }
        }
    }
    group_sums<V, 2>(sh, sm, on, s, rt, cv, t, red, [&](int i, const double(&v)[2]) {
      means[i] = make_float2((float)(v[0] * inv), (float)(v[1] * inv));
    });
    if (on) {
      T* os = dx + ((n0 + s) * sh.length) * sh.channels + c0;
      float2 m[V];
      of_groups<V>(m, means + s * sh.groups, g, whole);
#pragma unroll
      for (int i = 0; i < NR; ++i)
        if (rt + i * sm.row_threads < sh.length) {
          widen<T, V>(raw[i], f);
          widen<T, V>(rd[i], d);
          af.template apply<true>(sh.act, f, u2);
          slope_all<V>(sh.act, u2);
#pragma unroll
          for (int e = 0; e < V; ++e) d[e] = af.rstd[e] * (fmaf(d[e] * u2[e], af.w[e], -m[e].x) - f[e] * m[e].y);
          *(Vec<T, V>*)(os + (int64_t)(rt + i * sm.row_threads) * sh.channels) = narrow<T, V>(d);
        }
    }
  }
  if (!part) return;
  put_params<V>(sh, s < sm.samples, s * sm.row_threads + rt, c0, dw, db, (float2*)red);
  join_params(sh, sm.samples * sm.row_threads, (float2*)red, part);
}

// ---- samples of one row: a group in adjacent lanes of a wave ------------------

// v plus that of the lane at distance 1, 2, 4 ... in its group of `lanes`: sums of
// the same values in the same order in each of them.
template <int CTRL>
__device__ __forceinline__ float across(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double across(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true);
  return __hiloint2double(hi, lo);
}
template <class R>
__device__ __forceinline__ R lanes_sum(R v, int lanes) {
  if (lanes > 1) v += across<0xB1>(v);    // within pairs
  if (lanes > 2) v += across<0x4E>(v);    // pairs of a quad
  if (lanes > 4) v += across<0x141>(v);   // mirrored in 8 lanes: quads are uniform by now
  if (lanes > 8) v += across<0x140>(v);   // mirrored in 16
  if (lanes > 16) v += __shfl_xor(v, 16);
  if (lanes > 32) v += __shfl_xor(v, 32);
  return v;
}

// The place of a thread: of sm.samples x groups x sm.lanes threads; its W vectors of
// a group's channels are sm.lanes apart, those past the last channel idle along.
template <int V, int W>
struct RowPlace {
  int sample, group, c0[W];
  bool on[W], first;
  __device__ RowPlace(const Shape& sh, const Small& sm) {
    const int row = sh.groups * sm.lanes, u = threadIdx.x % row, lane = u % sm.lanes;
    sample = threadIdx.x / row;
    group = u / sm.lanes;
    first = lane == 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int j = (lane + w * sm.lanes) * V;
      on[w] = sample < sm.samples && j < sh.per_group;
      c0[w] = on[w] ? group * sh.per_group + j : 0;
    }
  }
};

// A thread keeps its channels and walks samples, 4 / W in flight; nothing is shared
// beyond the wave, so no wave waits for another.  Sums of 32-bit features are 64 bits
// from the start, as relu's side asks for; of 16-bit ones 32 bits.  Memory bounds it: 65536 x 512 in 8
// groups, float32, gelu: 66 us, 4080 GB/s; with the sums through LDS it took 133.
template <class T, int V, int W>
__global__ __launch_bounds__(512) void k_norm_rows(Shape sh, Small sm, const T* __restrict__ x, T* __restrict__ y,
                                                    float4* __restrict__ stats) {
  using R = std::conditional_t<sizeof(T) == 4, double, float>;
  const RowPlace<V, W> p(sh, sm);
  if (p.sample >= sm.samples) return;
  Affine<V> af[W];
#pragma unroll
  for (int w = 0; w < W; ++w) af[w].params(sh, p.c0[w]);
  const R inv = (R)1 / sh.per_group;
  const int64_t step = (int64_t)gridDim.x * sm.samples;
  constexpr int U = 4 / W;
  for (int64_t n = (int64_t)blockIdx.x * sm.samples + p.sample; n < sh.batch; n += U * step) {
    Vec<T, V> raw[U][W];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t at = n + i * step < sh.batch ? n + i * step : n;
#pragma unroll
      for (int w = 0; w < W; ++w) raw[i][w] = *(const Vec<T, V>*)(x + at * sh.batch_x + p.c0[w]);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t at = n + i * step;
      if (at >= sh.batch) break;
      float f[W][V], o[V];
      R sum = 0, sq = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        widen<T, V>(raw[i][w], f[w]);
        if (p.on[w])
#pragma unroll
          for (int e = 0; e < V; ++e) sum += f[w][e];
      }
      const R mean = lanes_sum(sum, sm.lanes) * inv;
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (p.on[w])
#pragma unroll
          for (int e = 0; e < V; ++e) sq += (f[w][e] - mean) * (f[w][e] - mean);
      const float4 st = pack_stats(mean, lanes_sum(sq, sm.lanes) * inv, sh.eps);
      if (p.first) stats[at * sh.groups + p.group] = st;
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int e = 0; e < V; ++e) af[w].stats(e, st);
        af[w].template apply<false>(sh.act, f[w], o);
        act_all<V>(sh.act, o);
        if (p.on[w]) *(Vec<T, V>*)(y + at * sh.channels + p.c0[w]) = narrow<T, V>(o);
      }
    }
  }
}

template <class T, int V, int W>
__global__ __launch_bounds__(512) void k_norm_rows_bwd(Shape sh, Small sm, const T* __restrict__ x, const T* __restrict__ dy,
                                                        T* __restrict__ dx, const float4* __restrict__ stats,
                                                        float2* __restrict__ part) {
  extern __shared__ double sums[];
  const RowPlace<V, W> p(sh, sm);
  float dw[W][V], db[W][V];
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[w][e] = db[w][e] = 0.f;
  if (p.sample < sm.samples) {
    Affine<V> af[W];
#pragma unroll
    for (int w = 0; w < W; ++w) af[w].params(sh, p.c0[w]);
    const float inv = 1.f / sh.per_group;
    const int64_t step = (int64_t)gridDim.x * sm.samples;
    constexpr int U = 4 / W;
    for (int64_t n = (int64_t)blockIdx.x * sm.samples + p.sample; n < sh.batch; n += U * step) {
      Vec<T, V> raw[U][W], rd[U][W];
      float4 st[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t at = n + i * step < sh.batch ? n + i * step : n;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          raw[i][w] = *(const Vec<T, V>*)(x + at * sh.batch_x + p.c0[w]);
          rd[i][w] = *(const Vec<T, V>*)(dy + at * sh.batch_dy + p.c0[w]);
        }
        st[i] = stats[at * sh.groups + p.group];
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t at = n + i * step;
        if (at >= sh.batch) break;
        float f[W][V], d[W][V], u[V], t0 = 0.f, t1 = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          widen<T, V>(raw[i][w], f[w]);
          widen<T, V>(rd[i][w], d[w]);
#pragma unroll
          for (int e = 0; e < V; ++e) af[w].stats(e, st[i]);
          af[w].template apply<true>(sh.act, f[w], u);
          slope_all<V>(sh.act, u);
          if (p.on[w])
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float du = d[w][e] * u[e];
              db[w][e] += du;
              dw[w][e] = fmaf(du, f[w][e], dw[w][e]);
              d[w][e] = du * af[w].w[e];
              t0 += d[w][e];
              t1 = fmaf(d[w][e], f[w][e], t1);
            }
        }
        const float m1 = lanes_sum(t0, sm.lanes) * inv, m2 = lanes_sum(t1, sm.lanes) * inv;
#pragma unroll
        for (int w = 0; w < W; ++w) {
#pragma unroll
          for (int e = 0; e < V; ++e) d[w][e] = st[i].y * (d[w][e] - m1 - f[w][e] * m2);
          if (p.on[w]) *(Vec<T, V>*)(dx + at * sh.channels + p.c0[w]) = narrow<T, V>(d[w]);
        }
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int w = 0; w < W; ++w) put_params<V>(sh, p.on[w], p.sample, p.c0[w], dw[w], db[w], (float2*)sums);
  join_params(sh, sm.samples, (float2*)sums, part);
}

// ---- a sample split along its rows ------------------------------------------
//
// Four passes over memory, which bounds each.  One sample of 232965 x 256 in 32 groups, float32, relu:
// statistics 48 us (5.0 TB/s), y 74 (6.4, some of x from the last-level cache), sums of the gradient 83 (5.8), dx 142 (5.0).

struct Chunks {
  int row_threads, vectors;   // threads of a workgroup along rows and channels
  int rows;                   // rows of a chunk
  int count;                  // chunks of a sample
  int tiles;                  // workgroups along the channels
};

// joins (n2 values of mean m2 and squared differences q2) into (n, m, q)
template <class R>
__device__ __forceinline__ void join(R& n, R& m, R& q, R n2, R m2, R q2) {
  const R all = n + n2;
  if (all == 0) return;
  const R f = n2 / all, d = m2 - m;
  m = fma(d, f, m);
  q += q2 + d * d * (n * f);
  n = all;
}
struct Share { double n, mean, squares; };

// A workgroup's row threads in pairs, pairs of pairs and so on: with(d) joins thread rt + d's values into its own.
// One after the other they are a chain of up to 256 steps for the few threads that have a channel: 220 x 10134 x 2 took 99 us
// for its statistics (the call 107 us, 18.7 in pairs).
template <class F>
__device__ __forceinline__ void join_rows(bool on, int rt, int row_threads, F&& with) {
  int d = 1;
  while (d < row_threads) d *= 2;
  __syncthreads();
  for (d /= 2; d; d /= 2) {
    if (on && rt < d && rt + d < row_threads) with(d);
    __syncthreads();
  }
}

// blockIdx: x chunk, y tile of the channels, z sample (the grid's z is bounded: a loop)
#define SRBCRS_CHUNK_PROLOGUE                                                                               \
  const int rt = threadIdx.x / ch.vectors, cv = blockIdx.y * ch.vectors + threadIdx.x - rt * ch.vectors;    \
  const int c0 = cv * V;                                                                                    \
  const bool on = rt < ch.row_threads && c0 < sh.channels;                                                  \
  const int64_t r0 = (int64_t)blockIdx.x * ch.rows, r1 = min(sh.length, r0 + ch.rows);

template <class T, int V>
__global__ __launch_bounds__(256) void k_norm_stats(Shape sh, Chunks ch, const T* __restrict__ x, float2* __restrict__ part) {
  __shared__ float2 red[V][256];
  __shared__ float rows[256];
  SRBCRS_CHUNK_PROLOGUE
  for (int64_t n = blockIdx.z; n < sh.batch; n += gridDim.z) {
    float mean[V], m2[V];
    float cnt = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.f;
    if (on) {
      const T* xs = x + n * sh.batch_x + c0;
      int64_t r = r0 + rt;
      const int64_t step = ch.row_threads;
      constexpr int U = 8;
      for (; r + (U - 1) * step < r1; r += U * step) {
        Vec<T, V> raw[U];
#pragma unroll
        for (int i = 0; i < U; ++i) raw[i] = *(const Vec<T, V>*)(xs + (r + i * step) * sh.ldx);
        float s[V], q[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = q[e] = 0.f;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          float f[V];
          widen<T, V>(raw[i], f);
#pragma unroll
          for (int e = 0; e < V; ++e) s[e] += f[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] *= 1.f / U;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          float f[V];
          widen<T, V>(raw[i], f);
#pragma unroll
          for (int e = 0; e < V; ++e) q[e] = fmaf(f[e] - s[e], f[e] - s[e], q[e]);
        }
        const float f = U / (cnt + U), g = cnt * f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = s[e] - mean[e];
          mean[e] = fmaf(d, f, mean[e]);
          m2[e] += fmaf(d * d, g, q[e]);
        }
        cnt += U;
      }
      for (; r < r1; r += step) {
        float f[V];
        widen<T, V>(*(const Vec<T, V>*)(xs + r * sh.ldx), f);
        cnt += 1.f;
        const float k = 1.f / cnt;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = f[e] - mean[e];
          mean[e] = fmaf(d, k, mean[e]);
          m2[e] = fmaf(d, f[e] - mean[e], m2[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) red[e][threadIdx.x] = make_float2(mean[e], m2[e]);
      rows[threadIdx.x] = cnt;
    }
    join_rows(on, rt, ch.row_threads, [&](int d) {
      const int from = threadIdx.x + d * ch.vectors;
      const float have = cnt;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 o = red[e][from];
        cnt = have;
        join(cnt, mean[e], m2[e], rows[from], o.x, o.y);
        red[e][threadIdx.x] = make_float2(mean[e], m2[e]);
      }
      rows[threadIdx.x] = cnt;
    });
    if (on && rt == 0)
#pragma unroll
      for (int e = 0; e < V; ++e) part[(n * ch.count + blockIdx.x) * sh.channels + c0 + e] = make_float2(mean[e], m2[e]);
  }
}

__device__ __forceinline__ float4 final_stats(const Shape& sh, double m, double q) {
  return pack_stats(m, q / ((double)sh.length * sh.per_group), sh.eps);
}

// Joins in two levels, so that few long samples still have many workgroups at
// it: 32 groups of 4096 parts took 63 us with a workgroup a group.
// First: blockIdx.x a group of a sample, blockIdx.y one of gridDim.y shares of its
// channels' parts of all chunks; one share is the end already.
constexpr int kJoinShare = 2048;   // parts of a share: 8 a thread

__global__ __launch_bounds__(256) void k_norm_stats_join(Shape sh, Chunks ch, const float2* __restrict__ part,
                                                         Share* __restrict__ shares, float4* __restrict__ stats) {
  __shared__ Share red[256];
  for (int64_t ng = blockIdx.x; ng < sh.batch * sh.groups; ng += gridDim.x) {
    const int64_t n = ng / sh.groups;
    const int g = (int)(ng - n * sh.groups);
    double a = 0., m = 0., q = 0.;
    const int all = ch.count * sh.per_group;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < all; i += gridDim.y * 256) {
      const int k = i / sh.per_group, c = g * sh.per_group + i - k * sh.per_group;
      const float2 o = part[(n * ch.count + k) * sh.channels + c];
      const int64_t rows = min((int64_t)ch.rows, sh.length - (int64_t)k * ch.rows);
      join(a, m, q, (double)rows, (double)o.x, (double)o.y);
    }
    red[threadIdx.x] = Share{a, m, q};
    __syncthreads();
    for (int d = 128; d; d >>= 1) {
      if ((int)threadIdx.x < d) {
        const Share o = red[threadIdx.x + d];
        join(a, m, q, o.n, o.mean, o.squares);
        red[threadIdx.x] = Share{a, m, q};
      }
      __syncthreads();
    }
    if (threadIdx.x == 0) {
      if (gridDim.y == 1) stats[ng] = final_stats(sh, m, q);
      else shares[ng * gridDim.y + blockIdx.y] = Share{a, m, q};
    }
    __syncthreads();
  }
}
__global__ __launch_bounds__(256) void k_norm_stats_end(Shape sh, int n_shares, const Share* __restrict__ shares,
                                                        float4* __restrict__ stats) {
  const int64_t ng = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (ng >= sh.batch * sh.groups) return;
  double a = 0., m = 0., q = 0.;
  for (int i = 0; i < n_shares; ++i) {
    const Share o = shares[ng * n_shares + i];
    join(a, m, q, o.n, o.mean, o.squares);
  }
  stats[ng] = final_stats(sh, m, q);
}

template <class T, int V>
__global__ __launch_bounds__(256) void k_norm_apply(Shape sh, Chunks ch, const T* __restrict__ x, T* __restrict__ y,
                                                    const float4* __restrict__ stats) {
  SRBCRS_CHUNK_PROLOGUE
  if (!on) return;
  Affine<V> af;
  af.params(sh, c0);
  int g[V];
#pragma unroll
  for (int e = 0; e < V; ++e) g[e] = (c0 + e) / sh.per_group;
  for (int64_t n = blockIdx.z; n < sh.batch; n += gridDim.z) {
#pragma unroll
    for (int e = 0; e < V; ++e) af.stats(e, stats[n * sh.groups + g[e]]);
    const T* xs = x + n * sh.batch_x + c0;
    T* ys = y + n * sh.length * sh.channels + c0;
    const int64_t step = ch.row_threads;
    auto one = [&](const Vec<T, V>& raw, int64_t r) {
      float f[V], u[V];
      widen<T, V>(raw, f);
      af.template apply<false>(sh.act, f, u);
      act_all<V>(sh.act, u);
      __builtin_nontemporal_store(narrow<T, V>(u), (Vec<T, V>*)(ys + r * sh.channels));
    };
    int64_t r = r0 + rt;
    constexpr int U = 4;
    for (; r + (U - 1) * step < r1; r += U * step) {
      Vec<T, V> raw[U];
#pragma unroll
      for (int i = 0; i < U; ++i) raw[i] = *(const Vec<T, V>*)(xs + (r + i * step) * sh.ldx);
#pragma unroll
      for (int i = 0; i < U; ++i) one(raw[i], r + i * step);
    }
    for (; r < r1; r += step) one(*(const Vec<T, V>*)(xs + r * sh.ldx), r);
  }
}

// Sums of du xhat and du of each channel over a chunk.
template <class T, int V>
__global__ __launch_bounds__(256) void k_norm_bwd_sums(Shape sh, Chunks ch, const T* __restrict__ x,
                                                       const T* __restrict__ dy, const float4* __restrict__ stats,
                                                       float2* __restrict__ part) {
  __shared__ double2 red[V][256];
  SRBCRS_CHUNK_PROLOGUE
  Affine<V> af;
  int g[V];
  if (on) {
    af.params(sh, c0);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = (c0 + e) / sh.per_group;
  }
  for (int64_t n = blockIdx.z; n < sh.batch; n += gridDim.z) {
    double2 sum[V];
    if (on) {
      float sw[V], sb[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        af.stats(e, stats[n * sh.groups + g[e]]);
        sw[e] = sb[e] = 0.f;
      }
      const T *xs = x + n * sh.batch_x + c0, *ds = dy + n * sh.batch_dy + c0;
      const int64_t step = ch.row_threads;
      auto one = [&](const Vec<T, V>& rx, const Vec<T, V>& rd) {
        float f[V], d[V], u[V];
        widen<T, V>(rx, f);
        widen<T, V>(rd, d);
        af.template apply<true>(sh.act, f, u);
        slope_all<V>(sh.act, u);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float du = d[e] * u[e];
          sb[e] += du;
          sw[e] = fmaf(du, f[e], sw[e]);
        }
      };
      int64_t r = r0 + rt;
      constexpr int U = 4;
      for (; r + (U - 1) * step < r1; r += U * step) {
        Vec<T, V> rx[U], rd[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          rx[i] = *(const Vec<T, V>*)(xs + (r + i * step) * sh.ldx);
          rd[i] = *(const Vec<T, V>*)(ds + (r + i * step) * sh.lddy);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) one(rx[i], rd[i]);
      }
      for (; r < r1; r += step) one(*(const Vec<T, V>*)(xs + r * sh.ldx), *(const Vec<T, V>*)(ds + r * sh.lddy));
#pragma unroll
      for (int e = 0; e < V; ++e) red[e][threadIdx.x] = sum[e] = make_double2(sw[e], sb[e]);
    }
    join_rows(on, rt, ch.row_threads, [&](int d) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double2 o = red[e][threadIdx.x + d * ch.vectors];
        sum[e].x += o.x, sum[e].y += o.y;
        red[e][threadIdx.x] = sum[e];
      }
    });
    if (on && rt == 0)
#pragma unroll
      for (int e = 0; e < V; ++e)
        part[(n * ch.count + blockIdx.x) * sh.channels + c0 + e] = make_float2((float)sum[e].x, (float)sum[e].y);
  }
}

// How a backward pass's parts are joined: one after the other in the grid, `groups` workgroups a share of the
// groups' sums, then `params` a share of the parameters'.  Each has as many shares as its own parts ask for:
// many short samples have few parts a group, and many of a parameter (8192 x 100 x 320 in 32 groups).
struct BackwardJoin {
  int groups, group_shares;
  int params, param_shares;
};

// Sums of du w and du w xhat of a group of a sample; of du xhat and du of 16 channels.
// One share is the end already.  Of up to 64 parts a wave joins a group, of more a workgroup.
__global__ __launch_bounds__(256) void k_norm_bwd_join(Shape sh, int chunks, const float2* __restrict__ part, int64_t parts,
                                                       BackwardJoin jn, double2* __restrict__ group_shares,
                                                       float2* __restrict__ means, double2* __restrict__ param_shares,
                                                       void* __restrict__ dweight, void* __restrict__ dbias) {
  __shared__ double2 red[256];
  const int group_blocks = jn.groups * jn.group_shares;
  if ((int)blockIdx.x < group_blocks) {
    const int all = chunks * sh.per_group;
    const double inv = 1. / ((double)sh.length * sh.per_group);
    auto mean = [&](double2 a) { return make_float2((float)(a.x * inv), (float)(a.y * inv)); };
    auto sum = [&](int64_t ng, int first, int step) {
      const int64_t n = ng / sh.groups;
      const int g = (int)(ng - n * sh.groups);
      double2 a = make_double2(0., 0.);
      for (int i = first; i < all; i += step) {
        const int k = i / sh.per_group, c = g * sh.per_group + i - k * sh.per_group;
        const float2 o = part[(n * chunks + k) * sh.channels + c];
        const double w = param(sh.weight, sh.param_dtype, c, 1.f);
        a.x = fma(w, (double)o.y, a.x), a.y = fma(w, (double)o.x, a.y);
      }
      return a;
    };
    if (all <= 64) {
      for (int64_t ng = blockIdx.x * 4 + (threadIdx.x >> 6); ng < sh.batch * sh.groups; ng += jn.groups * 4) {
        double2 a = sum(ng, threadIdx.x & 63, 64);
#pragma unroll
        for (int d = 32; d; d >>= 1) a.x += __shfl_xor(a.x, d), a.y += __shfl_xor(a.y, d);
        if ((threadIdx.x & 63) == 0) means[ng] = mean(a);
      }
      return;
    }
    const int share = (int)blockIdx.x / jn.groups;
    for (int64_t ng = (int)blockIdx.x - share * jn.groups; ng < sh.batch * sh.groups; ng += jn.groups) {
      red[threadIdx.x] = sum(ng, share * 256 + threadIdx.x, jn.group_shares * 256);
      __syncthreads();
      for (int d = 128; d; d >>= 1) {
        if ((int)threadIdx.x < d) red[threadIdx.x].x += red[threadIdx.x + d].x, red[threadIdx.x].y += red[threadIdx.x + d].y;
        __syncthreads();
      }
      if (threadIdx.x == 0) {
        if (jn.group_shares == 1) means[ng] = mean(red[0]);
        else group_shares[ng * jn.group_shares + share] = red[0];
      }
      __syncthreads();
    }
    return;
  }
  const int id = (int)blockIdx.x - group_blocks, share = id / jn.params;
  const int c = (id - share * jn.params) * 16 + (threadIdx.x & 15), sub = threadIdx.x >> 4;
  double2 a = make_double2(0., 0.);
  if (c < sh.channels) {
#pragma unroll 4
    for (int64_t p = share * 16 + sub; p < parts; p += jn.param_shares * 16) {
      const float2 o = part[p * sh.channels + c];
      a.x += o.x, a.y += o.y;
    }
  }
  red[threadIdx.x] = a;
  __syncthreads();
  for (int d = 8; d; d >>= 1) {
    if (sub < d) {
      const double2 o = red[threadIdx.x + 16 * d];
      a.x += o.x, a.y += o.y;
      red[threadIdx.x] = a;
    }
    __syncthreads();
  }
  if (sub || c >= sh.channels) return;
  if (jn.param_shares == 1) {
    if (dweight) put_param(dweight, sh.param_dtype, c, (float)a.x);
    if (dbias) put_param(dbias, sh.param_dtype, c, (float)a.y);
  } else {
    param_shares[(int64_t)share * sh.channels + c] = a;
  }
}
// The shares' sums: means of n_groups groups, gradients of the parameters (n_param 0: there is nothing to do for either).
__global__ __launch_bounds__(256) void k_norm_bwd_end(Shape sh, int64_t n_groups, int n_shares,
                                                      const double2* __restrict__ group_shares, float2* __restrict__ means,
                                                      int n_param, const double2* __restrict__ param_shares,
                                                      void* __restrict__ dweight, void* __restrict__ dbias) {
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  double2 a = make_double2(0., 0.);
  if (i < n_groups) {
    for (int k = 0; k < n_shares; ++k) {
      const double2 o = group_shares[i * n_shares + k];
      a.x += o.x, a.y += o.y;
    }
    const double inv = 1. / ((double)sh.length * sh.per_group);
    means[i] = make_float2((float)(a.x * inv), (float)(a.y * inv));
  } else if (i - n_groups < sh.channels && n_param) {
    i -= n_groups;
    for (int k = 0; k < n_param; ++k) {
      const double2 o = param_shares[(int64_t)k * sh.channels + i];
      a.x += o.x, a.y += o.y;
    }
    if (dweight) put_param(dweight, sh.param_dtype, i, (float)a.x);
    if (dbias) put_param(dbias, sh.param_dtype, i, (float)a.y);
  }
}

template <class T, int V>
__global__ __launch_bounds__(256) void k_norm_bwd_apply(Shape sh, Chunks ch, const T* __restrict__ x,
                                                        const T* __restrict__ dy, T* __restrict__ dx,
                                                        const float4* __restrict__ stats, const float2* __restrict__ means) {
  SRBCRS_CHUNK_PROLOGUE
  if (!on) return;
  Affine<V> af;
  af.params(sh, c0);
  int g[V];
#pragma unroll
  for (int e = 0; e < V; ++e) g[e] = (c0 + e) / sh.per_group;
  for (int64_t n = blockIdx.z; n < sh.batch; n += gridDim.z) {
    float m1[V], m2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      af.stats(e, stats[n * sh.groups + g[e]]);
      const float2 mm = means[n * sh.groups + g[e]];
      m1[e] = mm.x, m2[e] = mm.y;
    }
    const T *xs = x + n * sh.batch_x + c0, *ds = dy + n * sh.batch_dy + c0;
    T* os = dx + n * sh.length * sh.channels + c0;
    const int64_t step = ch.row_threads;
    auto one = [&](const Vec<T, V>& rx, const Vec<T, V>& rd, int64_t r) {
      float f[V], d[V], u[V];
      widen<T, V>(rx, f);
      widen<T, V>(rd, d);
      af.template apply<true>(sh.act, f, u);
      slope_all<V>(sh.act, u);
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = af.rstd[e] * (fmaf(d[e] * u[e], af.w[e], -m1[e]) - f[e] * m2[e]);
      __builtin_nontemporal_store(narrow<T, V>(d), (Vec<T, V>*)(os + r * sh.channels));
    };
    int64_t r = r0 + rt;
    constexpr int U = 4;
    for (; r + (U - 1) * step < r1; r += U * step) {
      Vec<T, V> rx[U], rd[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        rx[i] = *(const Vec<T, V>*)(xs + (r + i * step) * sh.ldx);
        rd[i] = *(const Vec<T, V>*)(ds + (r + i * step) * sh.lddy);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) one(rx[i], rd[i], r + i * step);
    }
    for (; r < r1; r += step) one(*(const Vec<T, V>*)(xs + r * sh.ldx), *(const Vec<T, V>*)(ds + r * sh.lddy), r);
  }
}

// ---- launches ----------------------------------------------------------------

Shape shape_of(const NormArgs& a, int64_t lddy, int64_t batch_dy) {
  Shape s;
  s.batch = a.batch, s.length = a.length;
  s.channels = (int)a.channels, s.groups = (int)a.groups, s.per_group = (int)(a.channels / a.groups);
  s.ldx = a.ldx, s.batch_x = a.batch_x, s.lddy = lddy, s.batch_dy = batch_dy;
  s.weight = a.weight, s.bias = a.bias, s.param_dtype = a.param_dtype, s.act = a.act, s.eps = a.eps;
  return s;
}

// Channels a thread takes at once: 16 bytes of them where every row starts at
// a multiple of that, else 2, else 1.  Of one row a sample: such that a vector lies in one
// group (60000 x 1000 in 4 groups, float32, forward and backward: 293 us with 2 for 461 with 4).
int vector_of(const NormArgs& a, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
  const int size = dtype_size(a.dtype);
  for (int v : {16 / size, 2}) {
    bool ok = (a.length == 1 ? a.channels / a.groups : a.channels) % v == 0;
    for (const void* p : ptrs) ok = ok && (uintptr_t)p % (v * size) == 0;
    for (int64_t s : strides) ok = ok && s % v == 0;
    if (ok) return v;
  }
  return 1;
}

struct SmallPlan {
  bool ok = false;
  int rows = 0;   // of the form of one row a sample: vectors of a thread
  int threads = 256, nr = 1;
  unsigned blocks = 1;
  Small sm{};
};

// A sample in one workgroup, up to 8 vectors a thread.  Few long samples
// would leave most CUs without work: they are split instead.  Split short samples are parts of one row each: 58809 rows
// of 728 channels in groups of 91, bfloat16, which have one channel a thread, took 1097 us so, and take 154 (training 16418 and 315).
SmallPlan small_plan(const NormArgs& a, int v) {
  SmallPlan p;
  const int64_t cv = a.channels / v, vectors = a.length * cv;
  if (a.batch < 64 && vectors > 1024 * 2) return p;
  const int64_t cg = a.channels / a.groups;
  if (a.length == 1 && cg % v == 0) {
    int lanes = 1, w = 1;
    while (lanes < 64 && lanes < cg / v) lanes *= 2;
    while (w * lanes < cg / v) w *= 2;
    const int64_t row = a.groups * lanes, t = row > 256 ? 512 : 256;
    if (row <= t && w <= 4 && w * v <= 16) {   // 16 channels a thread
      p.ok = true;
      p.rows = w;
      p.threads = (int)t;
      p.sm.vectors = (int)cv;
      p.sm.row_threads = 1;
      p.sm.lanes = lanes;
      p.sm.samples = (int)(t / row);
      const int64_t turns = (a.batch + p.sm.samples - 1) / p.sm.samples, most = 1024 * 256 / t;
      p.blocks = (unsigned)(turns < most ? turns : most);
      return p;
    }
  }
  for (int t = 256; t <= small_threads(v); t *= 2) {
    if (cv > t || (t == 1024 && cv <= 512)) continue;
    const int64_t rt = t / cv < a.length ? t / cv : a.length, nr = (a.length + rt - 1) / rt;
    int64_t samples = t / (rt * cv);
    if (samples > a.batch) samples = a.batch;
    // LDS: two sums a channel and thread, statistics of the groups
    if (nr > 8 || samples * (2 * rt * cv * v * 4 + 24 * a.groups) > 64 * 1024 - 8) continue;
    p.ok = true;
    p.threads = t;
    p.nr = nr <= 1 ? 1 : nr <= 4 ? 4 : 8;
    p.sm.row_threads = (int)rt;
    p.sm.vectors = (int)cv;
    p.sm.samples = (int)samples;
    const int64_t entries = rt * (cg % v == 0 ? cg / v : cg);
    int lanes = 1;
    while (lanes < 64 && 2 * lanes <= entries) lanes *= 2;
    p.sm.lanes = lanes;
    const int64_t turns = (a.batch + samples - 1) / samples, most = 2048 * 256 / t;
    p.blocks = (unsigned)(turns < most ? turns : most);
    return p;
  }
  return p;
}

Chunks chunks_of(const NormArgs& a, int v, int64_t z) {
  Chunks c;
  const int64_t cv = a.channels / v;
  c.vectors = (int)(cv < 256 ? cv : 256);
  c.row_threads = 256 / c.vectors;
  c.tiles = (int)((cv + c.vectors - 1) / c.vectors);
  int64_t count = 2048 / (z * c.tiles);   // one generation of resident workgroups
  const int64_t most = (a.length + c.row_threads * 8 - 1) / (c.row_threads * 8);
  if (count > most) count = most;
  if (count < 1) count = 1;
  const int64_t rows = (a.length + count - 1) / count;
  c.rows = (int)rows;
  c.count = (int)((a.length + rows - 1) / rows);
  return c;
}

template <class T, class F>
void by_vector(int v, F&& f) {
  constexpr int full = 16 / sizeof(T);
  if (v == full) f(std::integral_constant<int, full>{});
  else if (v == 2) f(std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 1>{});
}
// w vectors a thread; w V <= 16
template <class T, int V>
auto rows_kernel(int w) {
  if constexpr (V <= 4) {
    if (w == 4) return k_norm_rows<T, V, 4>;
  }
  return w == 2 ? k_norm_rows<T, V, 2> : k_norm_rows<T, V, 1>;
}
template <class T, int V>
auto rows_bwd_kernel(int w) {
  if constexpr (V <= 4) {
    if (w == 4) return k_norm_rows_bwd<T, V, 4>;
  }
  return w == 2 ? k_norm_rows_bwd<T, V, 2> : k_norm_rows_bwd<T, V, 1>;
}
template <class F>
void by_type(int dtype, F&& f) {
  if (dtype == kF32T) f((const float*)nullptr);
  else if (dtype == kBf16T) f((const __bf16*)nullptr);
  else f((const _Float16*)nullptr);
}
// shares of `parts` parts that are joined at once
int shares_of(int64_t parts, int64_t share) {
  const int64_t n = (parts + share - 1) / share;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
// of a backward pass in `count` chunks a sample
BackwardJoin backward_join(const NormArgs& a, int64_t count, bool params) {
  const int64_t parts = count * (a.channels / a.groups), all = a.batch * a.groups, blocks = parts <= 64 ? (all + 3) / 4 : all;
  return {(int)(blocks < 65536 ? blocks : 65536), shares_of(parts, kJoinShare), params ? (int)((a.channels + 15) / 16) : 0,
          shares_of(a.batch * count, 256)};
}
unsigned grid_z(int64_t batch) { return (unsigned)(batch < 65535 ? batch : 65535); }

__global__ __launch_bounds__(256) void k_fill_zero(char* p, size_t n) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0;
}

}  // namespace

void fill_zero(void* p, size_t bytes, hipStream_t s) {
  const size_t blocks = (bytes + 255) / 256;
  if (blocks) k_fill_zero<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>((char*)p, bytes);
}

size_t norm_workspace(const NormArgs& a, bool backward) {
  size_t most = 1;
  for (int v : {16 / dtype_size(a.dtype), 2, 1}) {
    if (a.channels % v) continue;
    const SmallPlan sp = small_plan(a, v);
    Carver c(nullptr);
    if (sp.ok) {
      if (backward) {
        c.take<float2>((size_t)sp.blocks * a.channels);
        c.take<double2>((size_t)shares_of(sp.blocks, 256) * a.channels);
      }
    } else {
      const int64_t count = chunks_of(a, v, grid_z(a.batch)).count;
      c.take<float2>(a.batch * count * a.channels);
      if (backward) {
        const BackwardJoin jn = backward_join(a, count, true);
        c.take<double2>(jn.group_shares > 1 ? a.batch * a.groups * jn.group_shares : 0);
        c.take<float2>(a.batch * a.groups);
        c.take<double2>((size_t)jn.param_shares * a.channels);
      } else {
        c.take<Share>(a.batch * a.groups * shares_of(count * (a.channels / a.groups), kJoinShare));
      }
    }
    if (c.used > most) most = c.used;
  }
  return most;
}

void norm_forward(const NormArgs& a, void* y, hipStream_t s) {
  const int v = vector_of(a, {a.x, y}, {a.ldx, a.batch_x});
  const SmallPlan sp = small_plan(a, v);
  const Shape sh = shape_of(a, 0, 0);
  Carver c(a.ws);
  if (sp.ok) {
    const size_t sum = a.dtype == kF32T && sp.nr == 1 ? sizeof(double) : sizeof(float);   // SmallSum
    const size_t lds = sp.sm.samples * (sp.sm.row_threads * sp.sm.vectors * v * sum + a.groups * (sizeof(float4) + sizeof(double))) + sizeof(double);
    by_type(a.dtype, [&](auto* t) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
      by_vector<T>(v, [&](auto vc) {
        constexpr int V = decltype(vc)::value;
        auto* k = sp.rows ? rows_kernel<T, V>(sp.rows) : sp.nr == 1 ? k_norm_small<T, V, 1> : sp.nr == 4 ? k_norm_small<T, V, 4> : k_norm_small<T, V, 8>;
        k<<<sp.blocks, sp.threads, lds, s>>>(sh, sp.sm, (const T*)a.x, (T*)y, (float4*)a.stats);
      });
    });
    return;
  }
  const unsigned z = grid_z(a.batch);
  const Chunks ch = chunks_of(a, v, z);
  float2* part = c.take<float2>(a.batch * ch.count * a.channels);
  const int n_shares = shares_of((int64_t)ch.count * sh.per_group, kJoinShare);
  Share* shares = c.take<Share>(a.batch * a.groups * n_shares);
  by_type(a.dtype, [&](auto* t) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    by_vector<T>(v, [&](auto vc) {
      constexpr int V = decltype(vc)::value;
      const dim3 grid(ch.count, ch.tiles, z);
      k_norm_stats<T, V><<<grid, 256, 0, s>>>(sh, ch, (const T*)a.x, part);
      const int64_t ng = a.batch * a.groups;
      k_norm_stats_join<<<dim3((unsigned)(ng < 65536 ? ng : 65536), n_shares), 256, 0, s>>>(sh, ch, part, shares, (float4*)a.stats);
      if (n_shares > 1) k_norm_stats_end<<<(unsigned)((ng + 255) / 256), 256, 0, s>>>(sh, n_shares, shares, (float4*)a.stats);
      k_norm_apply<T, V><<<grid, 256, 0, s>>>(sh, ch, (const T*)a.x, (T*)y, (const float4*)a.stats);
    });
  });
}

void norm_backward(const NormArgs& a, const void* dy, int64_t lddy, int64_t batch_dy, void* dx, void* dweight,
                     void* dbias, hipStream_t s) {
  const int v = vector_of(a, {a.x, dy, dx}, {a.ldx, a.batch_x, lddy, batch_dy});
  const SmallPlan sp = small_plan(a, v);
  const Shape sh = shape_of(a, lddy, batch_dy);
  const bool params = dweight || dbias;
  Carver c(a.ws);
  if (sp.ok) {
    float2* part = c.take<float2>((size_t)sp.blocks * a.channels);
    const int rows = sp.sm.samples * sp.sm.row_threads;
    const size_t lds = 2 * rows * sp.sm.vectors * v * sizeof(float) + sp.sm.samples * a.groups * sizeof(float2);
    by_type(a.dtype, [&](auto* t) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
      by_vector<T>(v, [&](auto vc) {
        constexpr int V = decltype(vc)::value;
        auto* k = sp.rows ? rows_bwd_kernel<T, V>(sp.rows) : sp.nr == 1 ? k_norm_small_bwd<T, V, 1> : sp.nr == 4 ? k_norm_small_bwd<T, V, 4> : k_norm_small_bwd<T, V, 8>;
        k<<<sp.blocks, sp.threads, lds, s>>>(sh, sp.sm, (const T*)a.x, (const T*)dy, (T*)dx, (const float4*)a.stats,
                                              params ? part : nullptr);
      });
    });
    if (params) {
      const int n = shares_of(sp.blocks, 256);
      const BackwardJoin jn{0, 0, (int)((a.channels + 15) / 16), n};
      double2* shares = c.take<double2>((size_t)n * a.channels);
      k_norm_bwd_join<<<(unsigned)(jn.params * n), 256, 0, s>>>(sh, 0, part, sp.blocks, jn, nullptr, nullptr, shares, dweight, dbias);
      if (n > 1)
        k_norm_bwd_end<<<(unsigned)((a.channels + 255) / 256), 256, 0, s>>>(sh, 0, 0, nullptr, nullptr, n, shares, dweight, dbias);
    }
    return;
  }
  const unsigned z = grid_z(a.batch);
  const Chunks ch = chunks_of(a, v, z);
  float2* part = c.take<float2>(a.batch * ch.count * a.channels);
  const BackwardJoin jn = backward_join(a, ch.count, params);
  double2* group_shares = c.take<double2>(jn.group_shares > 1 ? a.batch * a.groups * jn.group_shares : 0);
  float2* means = c.take<float2>(a.batch * a.groups);
  double2* param_shares = c.take<double2>((size_t)jn.param_shares * a.channels);
  by_type(a.dtype, [&](auto* t) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    by_vector<T>(v, [&](auto vc) {
      constexpr int V = decltype(vc)::value;
      const dim3 grid(ch.count, ch.tiles, z);
      k_norm_bwd_sums<T, V><<<grid, 256, 0, s>>>(sh, ch, (const T*)a.x, (const T*)dy, (const float4*)a.stats, part);
      k_norm_bwd_join<<<(unsigned)(jn.groups * jn.group_shares + jn.params * jn.param_shares), 256, 0, s>>>(
          sh, ch.count, part, a.batch * ch.count, jn, group_shares, means, param_shares, dweight, dbias);
      // what is not in shares is done
      const int64_t ng = jn.group_shares > 1 ? a.batch * a.groups : 0;
      const int np = params && jn.param_shares > 1 ? jn.param_shares : 0;
      if (ng || np)
        k_norm_bwd_end<<<(unsigned)((ng + (np ? a.channels : 0) + 255) / 256), 256, 0, s>>>(
            sh, ng, jn.group_shares, group_shares, means, np, param_shares, dweight, dbias);
      k_norm_bwd_apply<T, V><<<grid, 256, 0, s>>>(sh, ch, (const T*)a.x, (const T*)dy, (T*)dx, (const float4*)a.stats, means);
    });
  });
}

}  // namespace srbcrs
