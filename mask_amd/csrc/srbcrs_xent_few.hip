// Linear cross entropy where one of its two matrices has few rows: few classes
// (a graph network's classifier) or few rows of features (tokens to score
// against a large vocabulary).  The other matrix is read where it is, once a
// product, and that is what bounds it where it is long (streams, below).
//
// A wave holds the logits of its rows of the long matrix with all rows of the short one in
// registers.  The matrix instructions' operands of the long one come straight from memory: a
// lane's 8 values of a row are next to each other there.  The short matrix is laid
// out once a call in the order in which the lanes take it, and comes to LDS a line at a time for the workgroup.  dz
// leaves the logits' registers as the operand of the next product: the
// short dimension is summed in the order in which the registers hold it, on both sides.
//
//  forward   few classes: softmax and loss need no other wave.  Few rows: each wave leaves (max, sum)
//            of its classes for each row, joined afterwards
//  backward  logits again, dz -> the long matrix's gradient in the same kernel, dz^T to memory
//            (rows x classes, small); the short matrix's gradient = dz^T times the long one,
//            split over its rows, the parts joined in order
//
// 32-bit values are three bfloat16 (24 bits, no scale needed), six products; dz of
// 16-bit inputs is two of their type.  Sums are 32 bits.
//
// 232965 rows of 256 features against 64 classes, float32: loss 64 us (3.7 TB/s), dz and
// dh 143 (3.3 TB/s), dw 98 (3.0); the products take a third to a half of it and mostly run under the loads.
// Rows that are not aligned to 16 bytes are read and written at two thirds of that.
#include <hip/hip_runtime.h>

#include "srbcrs_xent.hpp"

namespace srbcrs {
namespace xent {
namespace few {

constexpr float kHalfScale = 16384.f;   // dz as float16: |dz| <= 1 to its upper end

template <class T>
struct Traits {              // 32 bits: bfloat16 x 3, times the same
  static constexpr int W = sizeof(T) == 4 ? 3 : 1;     // parts of a feature or weight
  static constexpr int Z = sizeof(T) == 4 ? 3 : 2;     // parts of dz
  static constexpr int KIND = __is_same(T, _Float16) ? kF16 : kBf16;
  static constexpr float SCALE = __is_same(T, _Float16) ? kHalfScale : 1.f;
  static constexpr int LINE = 128 / sizeof(T);         // features of a step: a row's whole line
  static constexpr int SUB = LINE / 32;                // matrix steps of it
  static constexpr int OUT = LINE / 16;                // 16-feature tiles of a step of the long gradient
};

// the first N parts of 8 values: each the rounded rest of the ones before
template <int KIND, int N>
__device__ __forceinline__ void parts_of(const float (&x)[8], float4v (&out)[N]) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
  for (int p = 0; p < N; ++p) {
    if constexpr (KIND == kF16) {
      half8 h;
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = (_Float16)r[e], r[e] -= (float)h[e];
      out[p] = __builtin_bit_cast(float4v, h);
    } else {
      bf8 h;
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = (__bf16)r[e], r[e] -= (float)h[e];
      out[p] = __builtin_bit_cast(float4v, h);
    }
  }
}
// c += a b to the last part that counts: parts (p, q) with p + q below the longer operand's
template <int KIND, int NA, int NB>
__device__ __forceinline__ float4v mma_parts(const float4v (&a)[NA], const float4v (&b)[NB], float4v c) {
  constexpr int MOST = NA > NB ? NA : NB;
#pragma unroll
  for (int s = MOST - 1; s >= 0; --s)   // small products first
#pragma unroll
    for (int p = 0; p <= s; ++p)
      if (p < NA && s - p < NB) c = mma<KIND>(a[p], b[s - p], c);
  return c;
}

// A lane's 32 bytes of a row's line from feature k on: SUB times 8 values, 32 apart;
// zeros past `dim`; any alignment.
template <class T>
struct Raw {
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  vec v[2];
};
template <class T, bool TAIL>
__device__ __forceinline__ void load_line(Raw<T>& r, const T* row, int k, int dim) {
  constexpr int V = 16 / sizeof(T), APART = Traits<T>::SUB == 1 ? V : 32;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (!TAIL) {
      r.v[i] = *(const typename Raw<T>::vec*)(row + k + i * APART);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) r.v[i][e] = k + i * APART + e < dim ? row[k + i * APART + e] : (T)0.f;
    }
  }
}
template <class T, int N>
__device__ __forceinline__ void operand(const Raw<T>& r, int sub, float4v (&out)[N]) {
  if constexpr (sizeof(T) == 2) {
    out[0] = __builtin_bit_cast(float4v, r.v[sub]);
  } else {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)r.v[i / 4][i % 4];
    parts_of<kBf16, N>(x, out);
  }
}
// matrix steps of z in the short matrix's layout, and groups of OUT tiles in the other
template <class T>
__host__ __device__ inline int z_steps(int dim) { return (dim + Traits<T>::LINE - 1) / Traits<T>::LINE * Traits<T>::SUB; }
template <class T>
__host__ __device__ inline int out_groups(int dim) { return (dim + Traits<T>::LINE - 1) / Traits<T>::LINE; }

// The short matrix f in the lanes' order.  Of z: [32 features][16 rows][part][lane],
// row lane % 16, features 8 (lane / 16)...  Of the long gradient: [line of features][tile of it]
// [32 rows][part][lane], rows 4 (lane / 16)... and 16 + 4 (lane / 16)..., features of tile o such
// that a lane's results of all OUT tiles are next to each other; there
// rows of factor 0 are zeros whatever they hold.
template <class T>
__global__ __launch_bounds__(256) void k_few_layout(const T* __restrict__ f, int64_t ld, int n_f, int dim, int vt,
                                                    const float* __restrict__ factor, float4v* __restrict__ fz,
                                                    float4v* __restrict__ fg) {
  constexpr int W = Traits<T>::W, OUT = Traits<T>::OUT;
  const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int nz = z_steps<T>(dim) * vt, ng = fg ? out_groups<T>(dim) * OUT * (vt / 2) : 0;
  if (id >= nz + ng) return;
  float x[8];
  const bool z = id < nz;
  const int r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    int v, d;
    if (z) v = id % vt * 16 + r, d = id / vt * 32 + 8 * q + e;
    else {
      const int i = id - nz, c = i % (vt / 2), t = i / (vt / 2), o = t % OUT;
      d = t / OUT * Traits<T>::LINE + 4 * OUT * (r >> 2) + 4 * o + (r & 3), v = 32 * c + (e < 4 ? 4 * q + e : 16 + 4 * q + e - 4);
    }
    const bool in = v < n_f && d < dim && (z || !factor || factor[v] != 0.f);
    x[e] = in ? (float)f[v * ld + d] : 0.f;
  }
  float4v p[W];
  parts_of<Traits<T>::KIND, W>(x, p);
  float4v* to = z ? fz + (int64_t)id * W * 64 : fg + (int64_t)(id - nz) * W * 64;
#pragma unroll
  for (int i = 0; i < W; ++i) to[i * 64 + lane] = p[i];
}

// The short matrix's layout a line at a time, for all waves of a workgroup: a wave would fetch VT W KB of it from L2 for each
// 2 TJ KB of its own rows, which bounded 65 and more short rows of 32 bits (60000 x 4096 against 100, float32: 702 us a
// loss; 4 waves that share it take 423).  Lines pass through registers (`stage`), loaded a step before they are written,
// to two places in LDS; one barrier a step.  Both layouts have as much a line.
template <class T, int VT>
struct Lines {
  static constexpr int UNITS = Traits<T>::SUB * VT * Traits<T>::W, PER_WAVE = (UNITS + 3) / 4;   // of 1 KB
  static_assert(UNITS == Traits<T>::OUT * (VT / 2) * Traits<T>::W, "the gradient's layout has the same lines");
  typedef float4v Place[UNITS][64];
  Place* lds;              // two
  const float4v* from;
  int count, lane, wave;
  float4v stage[PER_WAVE];

  __device__ __forceinline__ Lines(Place* lds_) : lds(lds_), lane(threadIdx.x & 63), wave(threadIdx.x >> 6) {}
  __device__ __forceinline__ int unit(int k) const { return min(wave + 4 * k, UNITS - 1); }   // the last ones of some waves twice
  __device__ __forceinline__ void fetch(int c) {
    const float4v* p = from + (int64_t)min(c, count - 1) * (UNITS * 64) + lane;
#pragma unroll
    for (int k = 0; k < PER_WAVE; ++k) stage[k] = p[unit(k) * 64];
  }
  __device__ __forceinline__ void put(int c) {
#pragma unroll
    for (int k = 0; k < PER_WAVE; ++k) lds[c & 1][unit(k)][lane] = stage[k];
  }
  // all waves are done with the places' last use
  __device__ __forceinline__ void begin(const float4v* layout, int lines) {
    from = layout, count = lines;
    fetch(0);
    put(0);
    fetch(1);
  }
  // Line c for all waves; its place is read until the next call.
  __device__ __forceinline__ const Place& next(int c) {
    barrier();
    put(c + 1);
    fetch(c + 2);
    return lds[c & 1];
  }
  // LDS reads and writes before it are complete; loads stay in flight
  static __device__ __forceinline__ void barrier() {
    wait_lgkmcnt0();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

// z[i][j][e]: row 16 i + 4 (lane / 16) + e of the short matrix with row[j] of the long one.
// All waves of the workgroup call it.
template <class T, int VT, int TJ>
__device__ __forceinline__ void logits(float4v (&z)[VT][TJ], const T* const (&row)[TJ], int dim, const float4v* fz,
                                       Lines<T, VT>& lines) {
  constexpr int W = Traits<T>::W, KIND = Traits<T>::KIND, SUB = Traits<T>::SUB, LINE = Traits<T>::LINE;
#pragma unroll
  for (int i = 0; i < VT; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) z[i][j] = float4v{0.f, 0.f, 0.f, 0.f};
  // lines of rows in flight: a wave of 16 rows alone takes four to fill its share of the memory's latency
  constexpr int PF = TJ == 1 ? 4 : 1;
  const int lane = lines.lane, q8 = 8 * (lane >> 4), whole = dim / LINE;
  Raw<T> next[PF][TJ];
  auto step = [&](int c, Raw<T> (&line)[TJ], bool more) {
    const auto& a_of = lines.next(c);
    Raw<T> cur[TJ];
#pragma unroll
    for (int j = 0; j < TJ; ++j) cur[j] = line[j];
    if (more)
#pragma unroll
      for (int j = 0; j < TJ; ++j) load_line<T, false>(line[j], row[j], (c + PF) * LINE + q8, dim);
    __builtin_amdgcn_sched_barrier(0);   // loads first: they run under the products
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      float4v b[TJ][W];
#pragma unroll
      for (int j = 0; j < TJ; ++j) operand<T, W>(cur[j], s, b[j]);
#pragma unroll
      for (int i = 0; i < VT; ++i) {
        float4v a[W];
#pragma unroll
        for (int k = 0; k < W; ++k) a[k] = a_of[(s * VT + i) * W + k][lane];
#pragma unroll
        for (int j = 0; j < TJ; ++j) z[i][j] = mma_parts<KIND, W, W>(a, b[j], z[i][j]);
      }
    }
  };
  lines.begin(fz, (dim + LINE - 1) / LINE);
#pragma unroll
  for (int u = 0; u < PF; ++u)
    if (u < whole)
#pragma unroll
      for (int j = 0; j < TJ; ++j) load_line<T, false>(next[u][j], row[j], u * LINE + q8, dim);
  for (int c = 0; c < whole; c += PF)
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (c + u < whole) step(c + u, next[u], c + u + PF < whole);
  if (dim % LINE) {
#pragma unroll
    for (int j = 0; j < TJ; ++j) load_line<T, true>(next[0][j], row[j], whole * LINE + q8, dim);
    step(whole, next[0], false);
  }
}

struct Args {
  const void* r;         // the long matrix
  int64_t ld;
  int n_r, n_f, dim;     // rows of the long and the short one, features
  int rows, classes;     // one of n_r and n_f each
  const int64_t* target;
  int64_t ignore;
  float2* lse;
};

template <class T, int TJ>
__device__ __forceinline__ void row_pointers(const T* (&row)[TJ], const Args& a, int r0, int lane) {
#pragma unroll
  for (int j = 0; j < TJ; ++j) row[j] = (const T*)a.r + min(r0 + 16 * j + (lane & 15), a.n_r - 1) * a.ld;
}

template <class T, int VT, int TJ>
__global__ __launch_bounds__(256) void k_few_loss(Args a, const float4v* __restrict__ wz, float* __restrict__ loss,
                                                  float2* __restrict__ wave_sum) {
  const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int t0 = wave * 16 * TJ;
  const T* row[TJ];
  row_pointers(row, a, t0, lane);
  float4v z[VT][TJ];
  __shared__ typename Lines<T, VT>::Place places[2];
  Lines<T, VT> lines(places);
  logits<T, VT, TJ>(z, row, a.dim, wz, lines);
  if (t0 >= a.n_r) return;
  const int q4 = 4 * (lane >> 4);
  float sum = 0.f, count = 0.f;
#pragma unroll
  for (int j = 0; j < TJ; ++j) {
    const int t = t0 + 16 * j + (lane & 15);
    const bool in = t < a.rows;
    const int64_t tg = in ? a.target[t] : a.ignore;
    float mx = -INFINITY, zt = 0.f, s = 0.f;
#pragma unroll
    for (int i = 0; i < VT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = 16 * i + q4 + e;
        if (v >= a.classes) z[i][j][e] = -INFINITY;
        mx = fmaxf(mx, z[i][j][e]);
        zt = v == tg ? z[i][j][e] : zt;
      }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int i = 0; i < VT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f((z[i][j][e] - ref) * kLog2e);
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    // one of the four lanes of a row holds the target's logit, the others 0
    zt += __shfl_xor(zt, 16);
    zt += __shfl_xor(zt, 32);
    if (lane < 16 && in) {
      a.lse[t] = make_float2(mx, 1.f / s);
      float l = 0.f;
      if (tg != a.ignore) {
        l = tg >= 0 && tg < a.classes ? (mx - zt) + logf(s) : NAN;
        count += 1.f;
      }
      sum += l;
      if (loss) loss[t] = l;
    }
  }
  if (wave_sum) {
#pragma unroll
    for (int d = 8; d; d >>= 1) sum += __shfl_xor(sum, d), count += __shfl_xor(count, d);
    if (lane == 0) wave_sum[wave] = make_float2(sum, count);
  }
}

// Few rows: (max, sum of exponentials) of the wave's classes for each row, and the target's logit.
template <class T, int VT, int TJ>
__global__ __launch_bounds__(256) void k_few_stats(Args a, const float4v* __restrict__ fz, float2* __restrict__ part,
                                                   float* __restrict__ zt) {
  const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int v0 = wave * 16 * TJ;
  const T* row[TJ];
  row_pointers(row, a, v0, lane);
  float4v z[VT][TJ];
  __shared__ typename Lines<T, VT>::Place places[2];
  Lines<T, VT> lines(places);
  logits<T, VT, TJ>(z, row, a.dim, fz, lines);
  if (v0 >= a.n_r) return;
#pragma unroll
  for (int i = 0; i < VT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = 16 * i + 4 * (lane >> 4) + e;
      const int64_t tg = t < a.rows ? a.target[t] : -1;
      float mx = -INFINITY, s = 0.f;
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        const int v = v0 + 16 * j + (lane & 15);
        if (v >= a.classes) z[i][j][e] = -INFINITY;
        else if (v == tg) zt[t] = z[i][j][e];
        mx = fmaxf(mx, z[i][j][e]);
      }
#pragma unroll
      for (int d = 8; d; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
      const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int j = 0; j < TJ; ++j) s += __builtin_amdgcn_exp2f((z[i][j][e] - ref) * kLog2e);
#pragma unroll
      for (int d = 8; d; d >>= 1) s += __shfl_xor(s, d);
      if ((lane & 15) == 0 && t < a.rows) part[(int64_t)wave * a.rows + t] = make_float2(mx, s);
    }
}

// dz of the wave's rows of the long matrix, times the feature row's factor over the
// largest one: to dzt [row of the short matrix][row of the long one], `pitch` of them (zeros past
// the last), and the long matrix's gradient = dz times the short matrix.
// ROWS: the short matrix is the features'.
template <class T, int VT, int TJ, bool ROWS>
__global__ __launch_bounds__(256, 2) void k_few_grad(Args a, const float4v* __restrict__ wz, const float4v* __restrict__ wh,
                                                  const float* __restrict__ factor, const unsigned* __restrict__ fmax,
                                                  float* __restrict__ dzt, int64_t pitch, T* __restrict__ dh) {
  constexpr int W = Traits<T>::W, Z = Traits<T>::Z, KIND = Traits<T>::KIND;
  const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int t0 = wave * 16 * TJ;
  const T* row[TJ];
  row_pointers(row, a, t0, lane);   // waves past the last row fill dzt up to `pitch`
  float4v z[VT][TJ];
  __shared__ typename Lines<T, VT>::Place places[2];
  Lines<T, VT> lines(places);
  logits<T, VT, TJ>(z, row, a.dim, wz, lines);
  const int q4 = 4 * (lane >> 4);
  const float unit = factor_unit(fmax);
  float4v b[VT / 2][TJ][Z];
  // what a feature row brings: factor, statistics, target
  struct Row { float f; float2 st; int64_t tg; };
  auto of = [&](int t) {
    Row r;
    r.f = t < a.rows ? factor[t] / unit : 0.f;
    r.st = r.f == 0.f ? make_float2(0.f, 0.f) : a.lse[t];
    r.tg = r.f == 0.f ? -1 : a.target[t];
    return r;
  };
  auto dz = [&](const Row& r, int v, float zv) {
    float p = __builtin_amdgcn_exp2f((zv - r.st.x) * kLog2e) * r.st.y;
    p = v == r.tg ? p - 1.f : p;
    return r.f == 0.f || v >= a.classes ? 0.f : p * r.f;
  };
#pragma unroll
  for (int c = 0; c < VT / 2; ++c) {
    float x[TJ][8];
    if constexpr (ROWS) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = 2 * c + (e >> 2), t = 16 * i + q4 + (e & 3);
        const Row r = of(t);
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          const int v = t0 + 16 * j + (lane & 15);
          x[j][e] = dz(r, v, z[i][j][e & 3]);
          if (dzt && t < a.rows && v < pitch) dzt[t * pitch + v] = x[j][e];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        const int t = t0 + 16 * j + (lane & 15);
        const Row r = of(t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = 2 * c + (e >> 2), v = 16 * i + q4 + (e & 3);
          x[j][e] = dz(r, v, z[i][j][e & 3]);
          if (dzt && v < a.classes && t < pitch) dzt[v * pitch + t] = x[j][e];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] *= Traits<T>::SCALE;
      parts_of<KIND, Z>(x[j], b[c][j]);
    }
  }
  if (!dh) return;
  const float out = unit / Traits<T>::SCALE;
  constexpr int OUT = Traits<T>::OUT, LINE = Traits<T>::LINE;
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  const int n_lines = out_groups<T>(a.dim);
  lines.barrier();   // the logits' last line is read
  lines.begin(wh, n_lines);
  for (int k = 0; k < n_lines; ++k) {
    const auto& w_of = lines.next(k);
    const int d = LINE * k + 4 * OUT * (lane >> 4);   // this lane's 4 OUT features, 32 bytes
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      float4v acc[OUT];
#pragma unroll
      for (int o = 0; o < OUT; ++o) acc[o] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < VT / 2; ++c)
#pragma unroll
        for (int o = 0; o < OUT; ++o) {
          float4v w[W];
#pragma unroll
          for (int i = 0; i < W; ++i) w[i] = w_of[(o * (VT / 2) + c) * W + i][lane];
          acc[o] = mma_parts<KIND, W, Z>(w, b[c][j], acc[o]);
        }
      const int t = t0 + 16 * j + (lane & 15);
      if (t >= a.n_r || d >= a.dim) continue;
      T* to = dh + (int64_t)t * a.dim + d;
      if (d + 4 * OUT <= a.dim) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          vec v;
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] = (T)(acc[(h * V + e) >> 2][e & 3] * out);
          *(vec*)(to + h * V) = v;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4 * OUT; ++e)
          if (d + e < a.dim) to[e] = (T)(acc[e >> 2][e & 3] * out);
      }
    }
  }
}

// Part of the short matrix's gradient: the long one's rows in steps of 32, dealt to the waves of all of
// a part's workgroups; 16 NJ features a workgroup.  A lane's features of tile j: d0 + APART j, in 16 bits next to each other
// and loaded together, in 32 each by itself: 16 bytes a lane of rows that are not aligned to them come at half the rate (81064 x
// 3126 against 10: 480 us for 265), and of rows that are no faster.  dz^T is read once for all of a workgroup's features: NJ is 8 where
// registers allow.  A long row of factor 0 (null: all are 1) counts as zeros whatever it holds.
template <class T, int VT, int NJ>
__global__ __launch_bounds__(256, VT * NJ >= 32 ? 1 : 2) void k_few_short(Args a, const float* __restrict__ factor, const float* __restrict__ dzt,
                                                     int64_t pitch, float* __restrict__ part) {
  constexpr int W = Traits<T>::W, Z = Traits<T>::Z, KIND = Traits<T>::KIND;
  __shared__ float sum[VT * 16 * 16 * NJ];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q8 = 8 * (lane >> 4);
  constexpr int APART = sizeof(T) == 4 ? 16 : 1;
  const int d0 = blockIdx.x * 16 * NJ + (APART == 1 ? NJ * r : r);
  typedef T vecn __attribute__((ext_vector_type(NJ), aligned(sizeof(T))));
  float4v acc[VT][NJ];
#pragma unroll
  for (int i = 0; i < VT; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};
  const int64_t steps = pitch / 32;
  const bool whole = d0 + APART * (NJ - 1) < a.dim;
  vecn raw[8];
  float4v f[2], zraw[VT][2];
  // a step's values; dzt and factor reach to whole steps, h is read at its last row past the end
  auto fetch = [&](int64_t s) {
    const int64_t t0 = s * 32 + q8;
    if (factor) {
      f[0] = *(const float4v*)(factor + t0);
      f[1] = *(const float4v*)(factor + t0 + 4);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e >> 2][e & 3] = t0 + e < a.n_r ? 1.f : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const T* p = (const T*)a.r + min(t0 + e, (int64_t)a.n_r - 1) * a.ld + d0;
      if (APART == 1 && whole) raw[e] = *(const vecn*)p;
      else
#pragma unroll
        for (int j = 0; j < NJ; ++j) raw[e][j] = whole || d0 + APART * j < a.dim ? p[APART * j] : (T)0.f;
    }
#pragma unroll
    for (int i = 0; i < VT; ++i) {
      const float4v* p = (const float4v*)(dzt + (int64_t)min(16 * i + r, a.n_f - 1) * pitch + t0);
      zraw[i][0] = p[0], zraw[i][1] = p[1];
    }
  };
  const int64_t stride = gridDim.y * 4;
  int64_t s = blockIdx.y * 4 + wave;
  if (s < steps) fetch(s);
  while (s < steps) {
    float4v b[NJ][W], z[VT][Z];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if constexpr (sizeof(T) == 2) {
        typedef T vec8 __attribute__((ext_vector_type(8)));
        vec8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = f[e >> 2][e & 3] == 0.f ? (T)0.f : raw[e][j];
        b[j][0] = __builtin_bit_cast(float4v, x);
      } else {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = f[e >> 2][e & 3] == 0.f ? 0.f : (float)raw[e][j];
        parts_of<KIND, W>(x, b[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < VT; ++i) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 16 * i + r < a.n_f ? zraw[i][e >> 2][e & 3] * Traits<T>::SCALE : 0.f;
      parts_of<KIND, Z>(x, z[i]);
    }
    s += stride;
    if (s < steps) fetch(s);   // the next step's loads run under this one's products
#pragma unroll
    for (int i = 0; i < VT; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = mma_parts<KIND, Z, W>(z[i], b[j], acc[i][j]);
  }
  // the waves' sums one after the other: always the same order
#pragma unroll 1
  for (int w = 0; w < 4; ++w) {
    if (wave == w)
#pragma unroll
      for (int i = 0; i < VT; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float* p = sum + (16 * i + 4 * (lane >> 4) + e) * (16 * NJ) + d0 - blockIdx.x * 16 * NJ + APART * j;
            *p = w ? *p + acc[i][j][e] : acc[i][j][e];
          }
    __syncthreads();
  }
  float* to = part + (int64_t)blockIdx.y * a.n_f * a.dim;
  for (int i = threadIdx.x; i < a.n_f * 16 * NJ; i += 256) {
    const int v = i / (16 * NJ), d = blockIdx.x * 16 * NJ + i % (16 * NJ);
    if (d < a.dim) to[(int64_t)v * a.dim + d] = sum[i];
  }
}

template <class F>
void by_type(int dtype, F&& f) {
  if (dtype == kF32T) f((const float*)nullptr);
  else if (dtype == kBf16T) f((const __bf16*)nullptr);
  else f((const _Float16*)nullptr);
}
// 16-row tiles of the short matrix: 2, 4 or 8
int short_tiles(int64_t n) { return n <= 32 ? 2 : n <= 64 ? 4 : 8; }
// and of the long one a wave: 4 (with 128 short rows' dz in registers 2), or 1 where the waves would be few.
// Training, float32, 2048 features: 120000 rows against 4 take 875 us for 1040 with one, 60000 532 for 510; 60000 against
// 64 take 598 for 640, against 100 804 for 906, 40000 against 64 489 for 428.
int long_tiles(int vt, int64_t n_r) { return n_r < (vt == 2 ? 64 : 48) * 1024 ? 1 : vt == 8 ? 2 : 4; }
// 16-feature tiles of a workgroup of the short gradient
template <class T>
constexpr int short_columns(int vt) { return sizeof(T) == 2 && vt == 2 ? 8 : 4; }
template <class F>
void by_tiles(int vt, F&& f) {
  if (vt == 2) f(std::integral_constant<int, 2>{});
  else if (vt == 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}
template <int VT, class F>
void by_long(int tj, F&& f) {
  if (tj == 1) f(std::integral_constant<int, 1>{});
  else f(std::integral_constant<int, VT == 8 ? 2 : 4>{});
}

struct Plan {
  Args args;
  const void* f;         // the short matrix
  int64_t ldf;
  bool by_rows;          // it is the features'
  int vt, tj, waves, n_layout;
  unsigned blocks;
  float4v *wz, *wh = nullptr;
  Plan(const XentArgs& a, Carver& c, bool gradient) {
    by_rows = a.classes > kFewClasses;
    const int64_t n_r = by_rows ? a.classes : a.rows, n_f = by_rows ? a.rows : a.classes;
    args = {by_rows ? a.w : a.h, by_rows ? a.ldw : a.ldh, (int)n_r, (int)n_f, (int)a.dim, (int)a.rows, (int)a.classes,
            a.target, a.ignore, (float2*)a.lse};
    f = by_rows ? a.h : a.w, ldf = by_rows ? a.ldh : a.ldw;
    vt = short_tiles(n_f);
    tj = long_tiles(vt, n_r);
    waves = (int)((n_r + 16 * tj - 1) / (16 * tj));
    blocks = (unsigned)((waves + 3) / 4);
    by_type(a.dtype, [&](auto* t) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
      const int z = z_steps<T>((int)a.dim) * vt, g = gradient ? out_groups<T>((int)a.dim) * Traits<T>::OUT * (vt / 2) : 0;
      n_layout = z + g;
      wz = c.take<float4v>((size_t)z * Traits<T>::W * 64);
      if (g) wh = c.take<float4v>((size_t)g * Traits<T>::W * 64);
    });
  }
  void layout(const XentArgs& a, const float* factor, hipStream_t s) const {
    by_type(a.dtype, [&](auto* t) {
      k_few_layout<<<(unsigned)((n_layout + 3) / 4), 256, 0, s>>>((decltype(t))f, ldf, args.n_f, args.dim, vt,
                                                                  by_rows ? factor : nullptr, wz, wh);
    });
  }
};

}  // namespace few

// Where this form is taken: it streams the long matrix, but each wave walks all features in turn, so a short long
// matrix is faster in tiles, whose sums are split.  Times of the tiles are in brackets.
namespace {
bool is_few(const XentArgs& a) { return a.classes <= kFewClasses || a.rows <= kFewRows; }
// Few classes or rows, and a long matrix that fills the chip.  Training, float32, 4096 features: 5000 rows against 4 classes
// take 254 us (264), 1500 245 (134); against 64 10000 335 (555), 5000 314 (295); against 100 20000 741 (1015), 10000 493 (598),
// 5000 460 (312).  Few features are few steps, and packing the operands counts: 1500 x 256 against 4, float32, 52 us
// (56), against 64 66 (61).
bool streams(const XentArgs& a) {
  const bool by_rows = a.classes > kFewClasses;
  const int vt = few::short_tiles(by_rows ? a.rows : a.classes);
  if (a.dim < (vt == 2 ? 512 : vt == 4 ? 256 : 0)) return true;
  return (by_rows ? a.classes : a.rows) >= (vt == 2 ? 4608 : vt == 4 ? 5632 : 12288);
}
}  // namespace
// 16 bits that the tiles' products can read where they are: the tiles copy nothing.  One row against 32000 classes of 2048
// features: 40 us (31); float16, 60000 rows of 2048 against 100 classes 74 (49), 10000 against 4 30 (22), 60000 against 4 48 (55);
// of up to 512 features both take a launch.
bool few_forwards(const XentArgs& a, bool readable) {
  if (!is_few(a)) return false;
  if (a.dtype == kF32T) return streams(a);
  if (!readable) return a.dim < 1024 || streams(a);
  return a.classes <= kFewClasses && (a.dim < 1024 || (a.classes <= 32 && a.rows >= 20000));
}
// In 16 bits this form's dz has two parts, the tiles' one.
bool few_backwards(const XentArgs& a) { return is_few(a) && (a.dtype != kF32T || streams(a)); }

size_t few_forward(const XentArgs& a, float* loss, hipStream_t s) {
  using namespace few;
  Carver c(a.ws);
  const Plan p(a, c, false);
  float2* part = p.by_rows ? c.take<float2>((int64_t)p.waves * a.rows) : nullptr;
  float* zt = p.by_rows ? c.take<float>(a.rows) : nullptr;
  const int n_sums = p.by_rows ? (int)a.rows : p.waves;
  float2* sums = a.reduction ? c.take<float2>(n_sums) : nullptr;
  if (!a.ws) return c.used;
  p.layout(a, nullptr, s);
  float* each = a.reduction ? nullptr : loss;
  by_type(a.dtype, [&](auto* t) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    by_tiles(p.vt, [&](auto vt) {
      constexpr int VT = decltype(vt)::value;
      by_long<VT>(p.tj, [&](auto tj) {
        constexpr int TJ = decltype(tj)::value;
        if (p.by_rows) k_few_stats<T, VT, TJ><<<p.blocks, 256, 0, s>>>(p.args, p.wz, part, zt);
        else k_few_loss<T, VT, TJ><<<p.blocks, 256, 0, s>>>(p.args, p.wz, each, sums);
      });
    });
  });
  if (p.by_rows) join_stats(part, p.waves, zt, a, each, sums, s);
  if (a.reduction) total(sums, n_sums, a, loss, s);
  return c.used;
}

size_t few_backward(const XentArgs& a, const float* dloss, void* dh, void* dw, hipStream_t s) {
  using namespace few;
  Carver c(a.ws);
  const bool by_rows = a.classes > kFewClasses;
  void *dlong = by_rows ? dw : dh, *dshort = by_rows ? dh : dw;
  const Plan p(a, c, dlong != nullptr);
  const int64_t pitch = round_up(p.args.n_r, 32), steps = pitch / 32;
  const int width = 16 * (a.dtype == kF32T ? short_columns<float>(p.vt) : short_columns<__bf16>(p.vt));
  const unsigned columns = (unsigned)((a.dim + width - 1) / width);
  // two workgroups a CU, and at least two steps a wave
  int64_t splits = 512 / columns;
  if (splits > (steps + 7) / 8) splits = (steps + 7) / 8;
  if (splits < 1) splits = 1;
  unsigned* fmax = c.take<unsigned>(1);
  float* factor = c.take<float>(round_up(a.rows, 32));
  float* dzt = dshort ? c.take<float>(p.args.n_f * pitch) : nullptr;
  float* part = dshort ? c.take<float>(splits * p.args.n_f * a.dim) : nullptr;
  if (!a.ws) return c.used;
  factors(a, dloss, factor, fmax, false, s);
  p.layout(a, factor, s);
  const float half = a.dtype == kF16T ? kHalfScale : 1.f;
  by_type(a.dtype, [&](auto* t) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    by_tiles(p.vt, [&](auto vt) {
      constexpr int VT = decltype(vt)::value;
      by_long<VT>(p.tj, [&](auto tj) {
        constexpr int TJ = decltype(tj)::value;
        auto* k = by_rows ? k_few_grad<T, VT, TJ, true> : k_few_grad<T, VT, TJ, false>;
        k<<<(unsigned)((pitch + 64 * TJ - 1) / (64 * TJ)), 256, 0, s>>>(p.args, p.wz, p.wh, factor, fmax, dzt, pitch, (T*)dlong);
      });
      if (dshort)
        k_few_short<T, VT, short_columns<T>(VT)><<<dim3(columns, (unsigned)splits), 256, 0, s>>>(p.args, by_rows ? nullptr : factor, dzt, pitch, part);
    });
  });
  if (dshort)
    join_parts(part, (int)splits, Out{dshort, a.dim, a.dtype, nullptr, nullptr, 1.f / half, nullptr, fmax, p.args.n_f, (int)a.dim}, s);
  return c.used;
}

}  // namespace xent
}  // namespace srbcrs
