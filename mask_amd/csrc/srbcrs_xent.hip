// Softmax cross entropy of a linear classifier, z = h w^T, loss_t =
// log sum_v exp z_tv - z_t,target, without the logits in memory:
//
//  forward   one product over all classes whose epilogue leaves (max, sum of
//            exponentials) of every 128 (or 64, 32) classes a row, joined afterwards
//  backward  the classes in pieces: the piece's logits again, their epilogue
//            writes dz = softmax - onehot as float16 scaled by 2^14, by rows and
//            by columns; then dh += dz w and dw = dz^T (g h), where g is the
//            row's upstream gradient (1 / labelled rows for the mean)
//
// Statistics, sums and products' sums are 32 bits.  Roundings to fewer: 16-bit
// inputs are used as they are; dz keeps 11 bits (float16: 3 more than
// bfloat16 inputs have) or, for 32-bit inputs, 22 as two float16.  32-bit inputs keep 22 bits too, in the logits
// each row's values to its own largest; in the gradients' sums over rows and classes, which have one scale each,
// to the largest row times its factor and to the largest weight.
//
// The products bound it: 8192 rows of 2048 features, 65536 classes, bfloat16, forward and backward: 7.3 to 7.5 ms, four
// products at 1180 to 1200 TFLOP/s; statistics 1.72 ms, dz 2.23 (it writes 2.1 GB), dh and dw 1.76 each.
#include <hip/hip_runtime.h>

#include "srbcrs_xent.hpp"

namespace srbcrs {
namespace xent {   // named: its types are template arguments of kernels

constexpr float kDzScale = 16384.f;          // |softmax - onehot| <= 1 to float16's upper end
// dz of a piece of the classes, each of its two orders.  Half as much costs 17 % with 55732 x 2364 against 4377 classes and
// 21 % with 100000 x 256 against 1000, both float32; twice as much gains the first 8 % and nothing else, for twice the memory.
constexpr int64_t kPieceBytes = 512ll << 20;

// What the backward pass's operands are scaled by: exponents of the largest h times its row's
// factor and of the largest w (null: they are not scaled), and the largest factor.
struct Scalars { unsigned *h_largest, *w_largest, *gmax; };

// Exponents of what a product of scaled rows lacks, of every row of w and of h; null: rows are as they are.
// Both reach to a whole number of tiles (what is past the last row is not used).
struct Exponents {
  const int *w, *h;
  // of four rows of w
  __device__ __forceinline__ int4 of_w(int v) const { return w ? *(const int4*)(w + v) : make_int4(0, 0, 0, 0); }
  __device__ __forceinline__ int of_h(int t) const { return h ? h[t] : 0; }
};
__device__ __forceinline__ float4v logits_of(float4v sum, int4 ew, int eh) {
  return float4v{__builtin_amdgcn_ldexpf(sum[0], ew.x + eh), __builtin_amdgcn_ldexpf(sum[1], ew.y + eh),
                 __builtin_amdgcn_ldexpf(sum[2], ew.z + eh), __builtin_amdgcn_ldexpf(sum[3], ew.w + eh)};
}

// unnormalised row statistics: the largest logit and the sum of exp(z - it)
struct StatEpi : WaveEpi {
  Exponents ex;
  float2* part;                  // [parts][rows]
  float* zt;
  const int64_t* target;
  int rows, classes;
  template <int TI, int TJ>
  __device__ void store(float4v (&acc)[TI][TJ], const Where& w) const {
    int4 ew[TI];
#pragma unroll
    for (int i = 0; i < TI; ++i) ew[i] = ex.of_w(row_of(w, i));
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int t = col_of(w, j), eh = ex.of_h(t);
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        acc[i][j] = logits_of(acc[i][j], ew[i], eh);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z = row_of(w, i) + e < classes ? acc[i][j][e] : -INFINITY;
          acc[i][j][e] = z;
          mx = fmaxf(mx, z);
        }
      }
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float ref = mx == -INFINITY ? 0.f : mx;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f((acc[i][j][e] - ref) * kLog2e);
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if (t < rows) {
        if (w.lane < 16) part[(int64_t)w.m_part * rows + t] = make_float2(mx, s);
        const int64_t at = target[t] - w.m0;
        if (at >= 0 && at < 16 * TI && at + w.m0 < classes) {
#pragma unroll
          for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (row_of(w, i) + e - w.m0 == (int)at) zt[t] = acc[i][j][e];
        }
      }
    }
  }
};

template <int KIND>   // of dz
struct GradEpi : WaveEpi {
  Exponents ex;
  const float2* lse;             // row: largest logit, 1 / sum of exponentials
  const int64_t* target;
  const float* factor;           // a row of factor 0 has a dz of 0, whatever its logits
  char *dz, *dzt;                // [rows][classes of the piece], [classes of the piece][rows]
  int64_t ld, ldt;
  int rows, classes, first;      // first: the piece's first class
  template <int TI, int TJ>
  __device__ void store(float4v (&acc)[TI][TJ], const Where& w) const {
    constexpr int SV = step_values(KIND);
    const int classes_up = (classes + SV - 1) / SV * SV, rows_up = (rows + SV - 1) / SV * SV;
    // the statistics of this lane's columns: rows of h
    float2 st[TJ];
    int at[TJ];
    bool live[TJ];
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int t = col_of(w, j);
      live[j] = t < rows && factor[t] != 0.f;
      const int64_t tg = live[j] ? target[t] : -1;
      st[j] = live[j] ? lse[t] : make_float2(0.f, 0.f);
      at[j] = tg >= first && tg < (int64_t)first + classes ? (int)(tg - first) : -1;
    }
    if (ex.w)
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const int4 ew = ex.of_w(row_of(w, i));
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[i][j] = logits_of(acc[i][j], ew, ex.of_h(col_of(w, j)));
      }
    through_lds<TI, TJ>(
        acc, w,
        [&](int v, int t, float4v z) {
          const int j = (t - w.n0) >> 4;
          float4v d;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float p = __builtin_amdgcn_exp2f((z[e] - st[j].x) * kLog2e) * st[j].y;
            p = v + e == at[j] ? p - 1.f : p;
            d[e] = live[j] && v + e < classes ? p * kDzScale : 0.f;
          }
          return d;
        },
        [&](const float* b, int v0, int t0) {
          if (v0 < classes_up)
            put_block<KIND, true>(b, w.lane, [&](int i) { return t0 + i < rows ? dz + (t0 + i) * ld + offset32<KIND>(v0) : nullptr; });
          if (t0 < rows_up)
            put_block<KIND, false>(b, w.lane,
                                   [&](int i) { return v0 + i < classes ? dzt + (v0 + i) * ldt + offset32<KIND>(t0) : nullptr; });
        });
  }
};

struct OutEpi : WaveEpi {
  Out o;
  template <int TI, int TJ>
  __device__ void store(float4v (&acc)[TI][TJ], const Where& w) const {
    const float f = o.factor();
    through_lds<TI, TJ>(
        acc, w, [&](int, int, float4v x) { return x * f; },
        [&](const float* b, int r0, int c0) {
          // 32 consecutive lanes a row: whole lines of any alignment
#pragma unroll 4
          for (int k = 0; k < 16; ++k) {
            const int r = r0 + 2 * k + (w.lane >> 5), c = c0 + (w.lane & 31);
            if (r < o.m && c < o.n) o.put(r, c, o.finish(r, c, b[(w.lane & 31) * kBlockLd + 2 * k + (w.lane >> 5)]));
          }
        });
  }
};

__global__ __launch_bounds__(256) void k_join_parts(const float* __restrict__ part, int splits, Out o) {
  const int64_t n = (int64_t)o.m * o.n, all = (int64_t)gridDim.x * 256;
  const float f = o.factor();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += all) {
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < splits; ++k) s += part[k * n + i];
    const int r = (int)(i / o.n), c = (int)(i - (int64_t)r * o.n);
    o.put(r, c, o.finish(r, c, s * f));
  }
}

// Rows' statistics from their parts; SUB threads a row.
template <int SUB>
__global__ __launch_bounds__(256) void k_xent_join(const float2* __restrict__ part, int parts, int rows,
                                                   const float* __restrict__ zt, const int64_t* __restrict__ target,
                                                   int64_t ignore, int classes, float2* __restrict__ lse,
                                                   float* __restrict__ loss, float2* __restrict__ block_sum) {
  constexpr int TPB = 256 / SUB;
  __shared__ float2 red[256];
  const int sub = threadIdx.x / TPB, t = blockIdx.x * TPB + threadIdx.x % TPB;
  float m = -INFINITY, s = 0.f;
  auto join = [&](float2 o) {
    const float nm = fmaxf(m, o.x), ref = nm == -INFINITY ? 0.f : nm;
    s = s * __builtin_amdgcn_exp2f((m - ref) * kLog2e) + o.y * __builtin_amdgcn_exp2f((o.x - ref) * kLog2e);
    m = nm;
  };
  if (t < rows)
#pragma unroll 8
    for (int p = sub; p < parts; p += SUB) join(part[(int64_t)p * rows + t]);
  red[threadIdx.x] = make_float2(m, s);
  __syncthreads();
#pragma unroll
  for (int d = SUB / 2; d; d >>= 1) {
    if (sub < d) {
      join(red[threadIdx.x + d * TPB]);
      red[threadIdx.x] = make_float2(m, s);
    }
    __syncthreads();
  }
  float l = 0.f, n = 0.f;
  if (sub == 0 && t < rows) {
    lse[t] = make_float2(m, 1.f / s);
    const int64_t tg = target[t];
    if (tg != ignore) {
      // a target that names no class makes the loss NaN
      l = tg >= 0 && tg < classes ? (m - zt[t]) + logf(s) : NAN;
      n = 1.f;
    }
    if (loss) loss[t] = l;
  }
  if (block_sum) {
    red[threadIdx.x] = make_float2(l, n);
    __syncthreads();
#pragma unroll
    for (int d = TPB / 2; d; d >>= 1) {
      if ((int)threadIdx.x < d) {
        red[threadIdx.x].x += red[threadIdx.x + d].x;
        red[threadIdx.x].y += red[threadIdx.x + d].y;
      }
      __syncthreads();
    }
    if (threadIdx.x == 0) block_sum[blockIdx.x] = red[0];
  }
}

// The loss over all rows and the number of labelled ones (at least 1, so that no label at all is a loss of 0).
// Counts are summed as integers: a float would stop at 2^24.
__global__ __launch_bounds__(1024) void k_xent_total(const float2* __restrict__ block_sum, int n, int mean,
                                                     float* __restrict__ loss, float* __restrict__ count) {
  __shared__ float ls[1024];
  __shared__ long long ns[1024];
  float l = 0.f;
  long long c = 0;
  for (int i = threadIdx.x; i < n; i += 1024) {
    const float2 b = block_sum[i];
    l += b.x;
    c += (long long)b.y;
  }
  ls[threadIdx.x] = l;
  ns[threadIdx.x] = c;
  __syncthreads();
  for (int d = 512; d; d >>= 1) {
    if ((int)threadIdx.x < d) {
      ls[threadIdx.x] += ls[threadIdx.x + d];
      ns[threadIdx.x] += ns[threadIdx.x + d];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const float labelled = (float)(ns[0] > 0 ? ns[0] : 1);
    count[0] = labelled;
    if (loss) loss[0] = mean ? ls[0] / labelled : ls[0];
  }
}

// A row's factor: its upstream gradient, 0 where it is not labelled, NaN
// where its target names no class (as its loss is).
__global__ __launch_bounds__(256) void k_xent_factor(const float* __restrict__ dloss, const int64_t* __restrict__ target,
                                                     int64_t ignore, int classes, const float* __restrict__ count,
                                                     int reduction, int64_t rows, int64_t rows_up, float* __restrict__ factor,
                                                     unsigned* __restrict__ fmax, Magnitudes mag) {
  float m = 0.f;
  unsigned largest = 0;
  const int64_t all = (int64_t)gridDim.x * 256;
  if (blockIdx.y) {   // the weight's
    for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < classes; v += all) m = fmaxf(m, mag.w[v]);
    join_max(exponent_of(m), mag.w_largest);
    return;
  }
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < rows_up; t += all) {
    const int64_t tg = t < rows ? target[t] : ignore;
    float f = 0.f;
    if (tg != ignore) {
      f = reduction == 0 ? dloss[t] : reduction == 1 ? dloss[0] / count[0] : dloss[0];
      if (tg < 0 || tg >= classes) f = NAN;
    }
    factor[t] = f;
    const float af = fabsf(f);
    if (af < INFINITY) {
      m = fmaxf(m, af);
      if (mag.h && t < rows) largest = max(largest, exponent_of((double)mag.h[t] * af));
    }
  }
  join_max(__builtin_bit_cast(unsigned, m), fmax);
  if (mag.h) join_max(largest, mag.h_largest);
}

// Rows of 16-bit values that the products can read where they are.
bool usable(const void* p, int64_t ld, int64_t dim) {
  return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && dim % 64 == 0;
}

// Operands of the logits: the caller's own matrices, or copies in whole steps.
struct Logits {
  Operand w, h;
  int kind;
  Exponents ex{};
  // row_max_w, row_max_h: rows' largest magnitudes, written where 32-bit rows are packed; null: not wanted
  Logits(const XentArgs& a, Carver& c, hipStream_t s, float* row_max_w = nullptr, float* row_max_h = nullptr) {
    kind = a.dtype == kF32T ? kSplit : a.dtype == kBf16T ? kBf16 : kF16;
    const bool go = a.ws != nullptr;
    // {weight, features}: as they are, or copies
    const void* p[2] = {a.w, a.h};
    const int64_t ld[2] = {a.ldw, a.ldh}, rows[2] = {a.classes, a.rows}, rb = row_bytes(kind, a.dim);
    float* row_max[2] = {row_max_w, row_max_h};
    int* exponent[2] = {};
    if (kind == kSplit) {
      for (int i = 0; i < 2; ++i) exponent[i] = c.take<int>(round_up(rows[i], tile_size(kTile256)));
      ex = {exponent[0], exponent[1]};
    }
    Operand o[2];
    int copied[2], n = 0;
    for (int i = 0; i < 2; ++i) {
      if (kind != kSplit && usable(p[i], ld[i], a.dim)) {
        o[i] = Operand{p[i], ld[i] * 2, 0, (int)rows[i]};
      } else {
        o[i] = Operand{c.take<char>(rows[i] * rb), rb, 0, (int)rows[i]};
        copied[n++] = i;
      }
    }
    auto copy = [&](auto kind_c, auto* t) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
      Pair<T> pair{};
      for (int k = 0; k < n; ++k) {
        const int i = copied[k];
        pair.m[k] = {(const T*)p[i], ld[i], rows[i], a.dim, (char*)o[i].p, rb, exponent[i], row_max[i], nullptr, nullptr, nullptr};
      }
      if constexpr (decltype(kind_c)::value == kSplit) pack_rows(pair, n, s);
      else pack<decltype(kind_c)::value>(pair, n, s);
    };
    if (go && n) {
      if (kind == kSplit) copy(std::integral_constant<int, kSplit>{}, (const float*)nullptr);
      else if (kind == kBf16) copy(std::integral_constant<int, kBf16>{}, (const __bf16*)nullptr);
      else copy(std::integral_constant<int, kF16>{}, (const _Float16*)nullptr);
    }
    w = o[0], h = o[1];
  }
  template <bool SPLIT, bool JOIN, class Epi>
  void run(const Cut& cut, Operand rows_w, int64_t dim, const Epi& epi, float* scratch, hipStream_t s) const {
    if constexpr (SPLIT) launch<kSplit, false, JOIN>(cut, rows_w, h, dim, epi, scratch, s);
    else if (kind == kBf16) launch<kBf16, false, JOIN>(cut, rows_w, h, dim, epi, scratch, s);
    else launch<kF16, false, JOIN>(cut, rows_w, h, dim, epi, scratch, s);
  }
};

template <int KIND>
void product(const Operand& a, const Operand& b, int64_t k, const Out& o, Carver& c, hipStream_t s, bool go) {
  const Cut cut = cut_for(KIND, o.m, o.n, k, 1, false, true);
  float* scratch = c.take<float>(cut.floats());
  if (go) launch<KIND, false, true>(cut, a, b, k, OutEpi{{}, o}, scratch, s);
}

template <int KIND>   // of dz
void backward_pieces(const XentArgs& a, Carver& c, const Logits& lg, const Scalars& sc, const float* factor, void* dh,
                     void* dw, hipStream_t s, size_t& used) {
  const bool go = a.ws != nullptr;
  const int64_t value = KIND == kSplit ? 4 : 2;
  int64_t piece = kPieceBytes / value / (a.rows < 64 ? 64 : a.rows) / 256 * 256;
  if (piece < 256) piece = 256;
  if (piece > a.classes) piece = a.classes;
  const int64_t n_pieces = (a.classes + piece - 1) / piece;
  const int64_t ldw = row_bytes(KIND, a.classes), ldh = row_bytes(KIND, a.rows);
  char* wt = dh ? c.take<char>(a.dim * ldw) : nullptr;
  char* ht = dw ? c.take<char>(a.dim * ldh) : nullptr;
  const int64_t ldz = row_bytes(KIND, piece), ldzt = ldh;
  char* dz = c.take<char>(a.rows * ldz);
  char* dzt = c.take<char>(piece * ldzt);
  float* sum = dh && n_pieces > 1 ? c.take<float>((size_t)a.rows * a.dim) : nullptr;
  if (go) {
    auto turn = [&](auto* t) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
      Pair<T> pair{};
      int n = 0;
      if (dh) pair.m[n++] = {(const T*)a.w, a.ldw, a.classes, a.dim, wt, ldw, nullptr, nullptr, sc.w_largest, nullptr, nullptr};
      if (dw) pair.m[n++] = {(const T*)a.h, a.ldh, a.rows, a.dim, ht, ldh, nullptr, nullptr, sc.h_largest, factor, sc.gmax};
      pack_t<KIND>(pair, n, s);
    };
    if constexpr (KIND == kSplit) turn((const float*)nullptr);
    else if (a.dtype == kBf16T) turn((const __bf16*)nullptr);
    else turn((const _Float16*)nullptr);
  }
  for (int64_t p = 0, v0 = 0; v0 < a.classes; ++p, v0 += piece) {
    const int64_t n = a.classes - v0 < piece ? a.classes - v0 : piece;
    // the parts of split sums are used within one product: every product's start there
    const size_t mark = c.used;
    const Cut cut = cut_for(lg.kind, n, a.rows, a.dim, 1, false, true, KIND == kSplit);
    float* scratch = c.take<float>(cut.floats());
    used = used > c.used ? used : c.used;
    if (go) {
      Operand wp = lg.w;
      wp.p = (const char*)wp.p + v0 * wp.ld;
      wp.rows = (int)n;
      GradEpi<KIND> e{{}, {lg.ex.w ? lg.ex.w + v0 : nullptr, lg.ex.h}, (const float2*)a.lse, a.target, factor, dz, dzt, ldz, ldzt,
                      (int)a.rows, (int)n, (int)v0};
      lg.run<KIND == kSplit, true>(cut, wp, a.dim, e, scratch, s);
    }
    c.used = mark;
    if (dh) {
      const bool last = p + 1 == n_pieces;
      Out o{last ? dh : sum, a.dim, last ? a.dtype : kF32T, p ? sum : nullptr, sc.w_largest, 1.f / kDzScale,
            last ? factor : nullptr, nullptr, (int)a.rows, (int)a.dim};
      product<KIND>(Operand{dz, ldz, 0, (int)a.rows},
                    Operand{wt + v0 / step_values(KIND) * kStep, ldw, 0, (int)a.dim}, n, o, c, s, go);
      used = used > c.used ? used : c.used;
      c.used = mark;
    }
    if (dw) {
      Out o{(char*)dw + v0 * a.dim * dtype_size(a.dtype), a.dim, a.dtype, nullptr, sc.h_largest, 1.f / kDzScale,
            nullptr, sc.gmax, (int)n, (int)a.dim};
      product<KIND>(Operand{dzt, ldzt, 0, (int)n}, Operand{ht, ldh, 0, (int)a.dim}, a.rows, o, c, s, go);
      used = used > c.used ? used : c.used;
      c.used = mark;
    }
  }
  used = used > c.used ? used : c.used;
}

void join_parts(const float* part, int splits, const Out& o, hipStream_t s) {
  k_join_parts<<<blocks_for((int64_t)o.m * o.n, 256, 2048), 256, 0, s>>>(part, splits, o);
}
void join_stats(const float2* part, int parts, const float* zt, const XentArgs& a, float* loss, float2* block_sum,
                hipStream_t s) {
  k_xent_join<256><<<(unsigned)a.rows, 256, 0, s>>>(part, parts, (int)a.rows, zt, a.target, a.ignore, (int)a.classes,
                                                     (float2*)a.lse, loss, block_sum);
}
void total(const float2* block_sum, int n, const XentArgs& a, float* loss, hipStream_t s) {
  k_xent_total<<<1, 1024, 0, s>>>(block_sum, n, a.reduction == 1, loss, a.count);
}
void factors(const XentArgs& a, const float* dloss, float* factor, unsigned* fmax, bool zeroed, hipStream_t s,
             const Magnitudes& mag) {
  const unsigned blocks = blocks_for(mag.w && a.classes > a.rows ? a.classes : a.rows, 256 * 4, 256);
  if (blocks > 1 && !zeroed) k_zero_words<<<1, 64, 0, s>>>(fmax, 1);
  k_xent_factor<<<dim3(blocks, mag.w ? 2 : 1), 256, 0, s>>>(dloss, a.target, a.ignore, (int)a.classes, a.count, a.reduction,
                                                            a.rows, round_up(a.rows, 32), factor, fmax, mag);
}

}  // namespace xent

using namespace xent;

size_t xent_forward(const XentArgs& a, float* loss, hipStream_t s) {
  if (few_forwards(a, usable(a.h, a.ldh, a.dim) && usable(a.w, a.ldw, a.dim))) return few_forward(a, loss, s);
  const bool go = a.ws != nullptr;
  Carver c(a.ws);
  // statistics are per wave of a tile: no join from parts of the sum
  const Cut cut = cut_for(a.dtype == kF32T ? kSplit : kBf16, a.classes, a.rows, a.dim, 1, false, false);
  const int64_t parts = (a.classes + tile_size(cut.tile) - 1) / tile_size(cut.tile) * waves_m(cut.tile);
  float2* part = c.take<float2>(parts * a.rows);
  float* zt = c.take<float>(a.rows);
  // the fewer the rows, the more threads join one row's parts
  const bool wide = a.rows <= 256, some = a.rows <= 4096;
  const unsigned blocks = (unsigned)(wide ? a.rows : some ? (a.rows + 3) / 4 : (a.rows + 31) / 32);
  float2* bs = a.reduction ? c.take<float2>(blocks) : nullptr;
  const Logits lg(a, c, s);
  if (!go) return c.used;
  const StatEpi epi{{}, lg.ex, part, zt, a.target, (int)a.rows, (int)a.classes};
  if (lg.kind == kSplit) lg.run<true, false>(cut, lg.w, a.dim, epi, nullptr, s);
  else lg.run<false, false>(cut, lg.w, a.dim, epi, nullptr, s);
  float* each = a.reduction ? nullptr : loss;
  if (wide)
    join_stats(part, (int)parts, zt, a, each, bs, s);
  else if (some)
    k_xent_join<64><<<blocks, 256, 0, s>>>(part, (int)parts, (int)a.rows, zt, a.target, a.ignore, (int)a.classes,
                                           (float2*)a.lse, each, bs);
  else
    k_xent_join<8><<<blocks, 256, 0, s>>>(part, (int)parts, (int)a.rows, zt, a.target, a.ignore, (int)a.classes,
                                          (float2*)a.lse, each, bs);
  if (a.reduction) total(bs, (int)blocks, a, loss, s);
  return c.used;
}

size_t xent_backward(const XentArgs& a, const float* dloss, void* dh, void* dw, hipStream_t s) {
  if (few_backwards(a)) return few_backward(a, dloss, dh, dw, s);
  const bool go = a.ws != nullptr;
  Carver c(a.ws);
  const bool scaled = a.dtype != kF16T;   // float16 inputs are operands as they are
  unsigned* words = c.take<unsigned>(3);
  const Scalars sc{scaled ? words : nullptr, scaled ? words + 1 : nullptr, words + 2};
  float* factor = c.take<float>(round_up(a.rows, 32));
  float *max_h = scaled ? c.take<float>(a.rows) : nullptr, *max_w = scaled ? c.take<float>(a.classes) : nullptr;
  const Logits lg(a, c, s, max_w, max_h);
  if (go) {
    if (a.dtype == kBf16T) {
      Pair<__bf16> pair{};
      pair.m[0] = {(const __bf16*)a.w, a.ldw, a.classes, a.dim, nullptr, 0, nullptr, max_w, nullptr, nullptr, nullptr};
      pair.m[1] = {(const __bf16*)a.h, a.ldh, a.rows, a.dim, nullptr, 0, nullptr, max_h, nullptr, nullptr, nullptr};
      row_maxima(pair, 2, s);
    }
    k_zero_words<<<1, 64, 0, s>>>(words, 3);
    factors(a, dloss, factor, sc.gmax, true, s, {max_h, max_w, sc.h_largest, sc.w_largest});
  }
  size_t used = c.used;
  if (a.dtype == kF32T) backward_pieces<kSplit>(a, c, lg, sc, factor, dh, dw, s, used);
  else backward_pieces<kF16>(a, c, lg, sc, factor, dh, dw, s, used);
  return used;
}

}  // namespace srbcrs
