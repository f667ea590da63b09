// Operand rows for the dense products (srbcrs_dense.hpp) from a caller's
// matrix, whole steps of 128 bytes with zeros past the last value.
//
// Its rows: 16 bits as they are; 32 bits each scaled by a power of two of its own, from its largest
// finite magnitude, so that no row's values cost another row's digits; its inverse's exponent
// goes to the product's end.
// Its columns: their sum runs over the rows, so one power of two scales all of them, from the largest finite magnitude
// of a row times the row's factor: rows that do not count (factor 0) have no say in it.
// What is all zeros, or has none finite, is scaled by 1.
//
// Maxima of many workgroups are joined by atomicMax on unsigned (of floats that are not negative the bits):
// the order does not matter.
#pragma once
#include "srbcrs_dense.hpp"
#include "srbcrs_ops.h"

namespace srbcrs {
namespace dense {

// 14 - exponent: scaled by 2 to its power, the largest magnitude lands in [2^14, 2^15).
// Clamped: the scale and its inverse are normal floats.
__device__ __forceinline__ int scale_exponent(unsigned max_bits) {
  return max_bits == 0 ? 0 : min(max(14 - ((int)(max_bits >> 23) - 127), -126), 126);
}
__device__ __forceinline__ float power_of_two(int e) { return __builtin_bit_cast(float, (unsigned)(e + 127) << 23); }

// The largest factor's magnitude, 1 where all are 0.
__device__ __forceinline__ float factor_unit(const unsigned* max_bits) {
  return *max_bits ? __builtin_bit_cast(float, *max_bits) : 1.f;
}
// A magnitude's exponent, biased: 0 only of 0.  Products of two floats neither overflow nor vanish in 64 bits.
__device__ __forceinline__ unsigned exponent_of(double v) { return v > 0. ? (unsigned)__double2hiint(v) >> 20 : 0u; }
// Of a matrix whose entries times their factors have `largest` as their largest exponent_of, for
// factors in units of the largest one (unit null: none): they land below 2^15.
__device__ __forceinline__ int scale_exponent(const unsigned* largest, const unsigned* unit) {
  const int u = unit ? (int)exponent_of(factor_unit(unit)) - 1023 : 0;
  return *largest == 0 ? 0 : min(max(14 - ((int)*largest - 1023 - u), -126), 126);
}

template <class T>
__global__ __launch_bounds__(64) void k_zero_words(T* p, int n) {
  if ((int)threadIdx.x < n) p[threadIdx.x] = 0;
}

// A workgroup's maximum to *out: one atomic each, and at most a workgroup a CU, since
// atomics on one word follow each other at about 10 ns (4096 of them cost 40 us).  A launch
// of one workgroup sets *out, more of them need a zero there first.
__device__ __forceinline__ void join_max(unsigned m, unsigned* out) {
  __shared__ unsigned all[16];
#pragma unroll
  for (int d = 32; d; d >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, d));
  __syncthreads();   // an earlier call's are read
  if ((threadIdx.x & 63) == 0) all[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < (int)(blockDim.x >> 6); ++i) m = max(m, all[i]);
    if (gridDim.x == 1) *out = m;
    else if (m) atomicMax(out, m);
  }
}

// A caller's matrix, and what becomes of it.  Kernels take two by blockIdx.y: launches of
// small matrices cost more than their work.
template <class T>
struct Source {
  const T* x;
  int64_t ld, rows, cols;
  char* dst;                     // operand rows
  int64_t ld_dst;
  int* exponent;                 // of each row, of its scale's inverse (k_pack_rows)
  float* row_max;                // of each row, its largest finite magnitude (k_row_max, k_pack_rows), null: not wanted
  // of k_pack_t
  const unsigned* largest;       // exponent_of its entries times their factors, null: not scaled
  const float* factor;           // of its rows, null: none
  const unsigned* factor_max;
};
template <class T>
struct Pair { Source<T> m[2]; };

// see(value) for each value of a matrix once, in a fixed order of the threads of
// gridDim.x workgroups: four loads of 16 bytes in flight where rows allow.
template <class T, class F>
__device__ __forceinline__ void walk(const T* x, int64_t ld, int64_t rows, int64_t cols, F&& see) {
  if (ld == cols) cols *= rows, rows = 1;
  constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V)));
  // a long row is walked by all workgroups, short ones by a wave each
  const bool lone = rows == 1;
  const int per_block = blockDim.x >> 6;
  const int64_t wave = (int64_t)blockIdx.x * per_block + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * per_block;
  const int64_t c0 = lone ? (int64_t)blockIdx.x * blockDim.x + threadIdx.x : threadIdx.x & 63;
  const int64_t step = lone ? (int64_t)gridDim.x * blockDim.x : 64;
  for (int64_t r = lone ? 0 : wave; r < rows; r += waves) {
    const T* row = x + r * ld;
    int64_t done = 0;
    if (((uintptr_t)row & 15) == 0) {
      const int64_t n = cols / V;
      int64_t i = c0;
      for (; i + 3 * step < n; i += 4 * step) {
        vec v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = *(const vec*)(row + (i + u * step) * V);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int q = 0; q < V; ++q) see((float)v[u][q]);
      }
      for (; i < n; i += step) {
        const vec v = *(const vec*)(row + i * V);
#pragma unroll
        for (int q = 0; q < V; ++q) see((float)v[q]);
      }
      done = n * V;
    }
#pragma unroll 4
    for (int64_t i = done + c0; i < cols; i += step) see((float)row[i]);
  }
}

// The largest finite |x[r][:]| of every row r, by `lanes` lanes a row (a power of two, a wave at most).
template <class T>
__global__ __launch_bounds__(256) void k_row_max(Pair<T> pair, int lanes) {
  const Source<T>& src = pair.m[blockIdx.y];
  const int cols = (int)src.cols, lane = threadIdx.x & (lanes - 1), per_block = 256 / lanes;
  typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  for (int64_t r = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes; r < src.rows; r += (int64_t)gridDim.x * per_block) {
    const T* x = src.x + r * src.ld;
    float m = 0.f;
    auto see = [&](float v) {
      v = fabsf(v);
      m = v < INFINITY ? fmaxf(m, v) : m;
    };
#pragma unroll 4
    for (int c = 8 * lane; c + 8 <= cols; c += 8 * lanes) {
      const vec v = *(const vec*)(x + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) see((float)v[e]);
    }
    for (int c = (cols & ~7) + lane; c < cols; c += lanes) see((float)x[c]);
    for (int d = lanes / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) src.row_max[r] = m;
  }
}

// Rows of 16 bits: dst row r holds x[r][:].  Four values a thread, four times in flight.
template <int KIND, class T>
__global__ __launch_bounds__(256) void k_pack(Pair<T> pair) {
  const Source<T>& src = pair.m[blockIdx.y];
  const T* x = src.x;
  const int64_t ld = src.ld, rows = src.rows, cols = src.cols, ld_dst = src.ld_dst;
  char* dst = src.dst;
  const int64_t quads = ld_dst / kStep * (step_values(KIND) / 4), n = rows * quads, all = (int64_t)gridDim.x * 256;
  const bool narrow = n < (1ll << 31);   // a 64-bit division takes longer than the copy
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  constexpr int U = 4;
  for (int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x; i0 < n; i0 += U * all) {
    int64_t r[U];
    int c[U];
    float4v v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * all < n ? i0 + u * all : i0;
      r[u] = narrow ? (int64_t)((unsigned)i / (unsigned)quads) : i / quads;
      c[u] = (int)(i - r[u] * quads) * 4;
      const T* at = x + r[u] * ld + c[u];
      if (c[u] + 4 <= cols) {
        const vec t = *(const vec*)at;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[u][q] = (float)t[q];
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[u][q] = c[u] + q < cols ? (float)at[q] : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * all < n) put4<KIND>(dst + r[u] * ld_dst, c[u], v[u]);
  }
}

// Rows of 32 bits, each with its own scale: `lanes` lanes a row, a power of two that is at most a wave, four quads of
// values a lane in flight.  Rows of up to 1024 values stay in registers between their maximum and
// their place; longer ones are read again, from the cache that they have just passed.
template <class T>
__global__ __launch_bounds__(256) void k_pack_rows(Pair<T> pair, int lanes) {
  const Source<T>& src = pair.m[blockIdx.y];
  const int cols = (int)src.cols, quads = (int)(src.ld_dst / kStep * (step_values(kSplit) / 4));
  const int lane = threadIdx.x & (lanes - 1), per_block = 256 / lanes;
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  constexpr int U = 4;
  for (int64_t r = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes; r < src.rows; r += (int64_t)gridDim.x * per_block) {
    const T* x = src.x + r * src.ld;
    char* to = src.dst + r * src.ld_dst;
    float4v v[U];
    auto load = [&](int q0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int q = q0 + u * lanes, c = 4 * q;
        v[u] = float4v{0.f, 0.f, 0.f, 0.f};
        if (c + 4 <= cols) {
          const vec t = *(const vec*)(x + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = (float)t[e];
        } else if (c < cols) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = c + e < cols ? (float)x[c + e] : 0.f;
        }
      }
    };
    float m = 0.f;
    for (int q0 = lane; q0 < quads; q0 += U * lanes) {
      load(q0);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = fabsf(v[u][e]);
          m = a < INFINITY ? fmaxf(m, a) : m;
        }
    }
    for (int d = lanes / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    const int e = scale_exponent(__builtin_bit_cast(unsigned, m));
    const float scale = power_of_two(e);
    if (lane == 0) src.exponent[r] = -e;
    if (lane == 0 && src.row_max) src.row_max[r] = m;
    const bool held = quads <= U * lanes;
    for (int q0 = lane; q0 < quads; q0 += U * lanes) {
      if (!held) load(q0);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q0 + u * lanes < quads) put4<kSplit>(to, 4 * (q0 + u * lanes), v[u] * scale);
    }
  }
}

// Columns: dst row c holds x[:][c] * scale (* factor[r] / the largest factor: exactly 1 where all
// are the same; a zero factor gives a zero whatever x holds).  A workgroup turns a 64 x 64 tile in LDS.
template <int KIND, class T>
__global__ __launch_bounds__(256) void k_pack_t(Pair<T> pair) {
  const Source<T>& src = pair.m[blockIdx.y];
  const T* x = src.x;
  const int64_t ld = src.ld, rows = src.rows, cols = src.cols, ld_dst = src.ld_dst;
  char* dst = src.dst;
  const unsigned* factor_max = src.factor_max;
  const float* factor = src.factor;
  __shared__ float tile[64][65];
  const float scale = src.largest ? power_of_two(scale_exponent(src.largest, factor_max)) : 1.f;
  const float unit = factor_max ? factor_unit(factor_max) : 1.f;
  const int64_t ct = (cols + 63) / 64, c0 = (blockIdx.x % ct) * 64, r0 = (blockIdx.x / ct) * 64;
  if (r0 >= rows) return;   // the other matrix has more tiles
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const int tx = 4 * (threadIdx.x & 15), ty = threadIdx.x >> 4;
  const int64_t c = c0 + tx;
  // all of a thread's loads before the first of them is used
  float v[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = r0 + ty + 16 * i;
    if (r < rows && c + 4 <= cols) {
      const vec t = *(const vec*)(x + r * ld + c);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[i][q] = (float)t[q];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[i][q] = r < rows && c + q < cols ? (float)x[r * ld + c + q] : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = r0 + ty + 16 * i;
    // the scale first with the factor: a large value of a small factor does not overflow
    const float f = factor && r < rows ? factor[r] / unit * scale : scale;
#pragma unroll
    for (int q = 0; q < 4; ++q) tile[ty + 16 * i][tx + q] = f == 0.f ? 0.f : v[i][q] * f;
  }
  __syncthreads();
  // 16 quads of 4 values along r for each of 64 columns
  const int64_t width = ld_dst / kStep * step_values(KIND);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = threadIdx.x & 15, c = (threadIdx.x >> 4) + 16 * i;
    const int64_t r = r0 + 4 * q;
    if (c0 + c < cols && r < width) {
      const float4v v = {tile[4 * q][c], tile[4 * q + 1][c], tile[4 * q + 2][c], tile[4 * q + 3][c]};
      put4<KIND>(dst + (c0 + c) * ld_dst, (int)r, v);
    }
  }
}

inline unsigned blocks_for(int64_t work, int64_t per_block, int64_t most = 4096) {
  const int64_t n = (work + per_block - 1) / per_block;
  return (unsigned)(n < 1 ? 1 : n > most ? most : n);
}

// lanes that share a row of `loads` loads
inline int lanes_for(int64_t loads) {
  int lanes = 1;
  while (lanes < 64 && lanes < loads) lanes *= 2;
  return lanes;
}
template <class T>
int64_t most_rows(const Pair<T>& p, int n) { return n > 1 && p.m[1].rows > p.m[0].rows ? p.m[1].rows : p.m[0].rows; }

// of n matrices (1 or 2) of one width
template <class T>
void row_maxima(const Pair<T>& p, int n, hipStream_t s) {
  const int lanes = lanes_for(p.m[0].cols / 8);
  k_row_max<T><<<dim3(blocks_for(most_rows(p, n), 256 / lanes, 8192), n), 256, 0, s>>>(p, lanes);
}
template <int KIND, class T>
void pack(const Pair<T>& p, int n, hipStream_t s) {
  int64_t most = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t quads = p.m[i].rows * (p.m[i].ld_dst / kStep * (step_values(KIND) / 4));
    most = most > quads ? most : quads;
  }
  k_pack<KIND, T><<<dim3(blocks_for(most, 256 * 4, 8192), n), 256, 0, s>>>(p);
}
// rows of one length
template <class T>
void pack_rows(const Pair<T>& p, int n, hipStream_t s) {
  const int lanes = lanes_for(p.m[0].ld_dst / kStep * (step_values(kSplit) / 4));
  k_pack_rows<T><<<dim3(blocks_for(most_rows(p, n), 256 / lanes, 8192), n), 256, 0, s>>>(p, lanes);
}
// the rows of dst reach to whole steps: tiles of 64 rows of x cover them
template <int KIND, class T>
void pack_t(const Pair<T>& p, int n, hipStream_t s) {
  int64_t most = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t tiles = ((p.m[i].cols + 63) / 64) * ((p.m[i].rows + 63) / 64);
    most = most > tiles ? most : tiles;
  }
  k_pack_t<KIND, T><<<dim3((unsigned)most, n), 256, 0, s>>>(p);
}

}  // namespace dense
}  // namespace srbcrs
