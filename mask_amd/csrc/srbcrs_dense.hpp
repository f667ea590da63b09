// Dense products D = A B^T for the training operators, both operands rows of
// 16-bit values along the summed dimension, on the 16x16x32 matrix
// instructions with 32-bit sums.
//
// Operand rows.  An operand is rows of 128-byte steps, 128-byte aligned or at
// least 16-byte aligned.  kF16 / kBf16: a step is 64 values.  kSplit: a step
// is 32 values of a 32-bit matrix, each as the sum of two float16, 64 bytes of
// high parts and then 64 bytes of low parts.  With a row, or the matrix, scaled by a
// power of two to a largest value in [2^14, 2^15), high + low hold 22 bits of every
// value down to 2^-29 of the largest, and an absolute error of 2^-40 of it
// below.  A product of two such matrices is
// high high + high low + low high; what is left out is 2^-22 of a term.  Three float16 products cost
// 3/16 of the 32-bit matrix instructions' time for the same product.
//
// A step is the unit of the whole pipeline: rows of both tiles go to LDS
// with direct-to-LDS loads of 16 bytes a lane, eight lanes a row.
// LDS holds rows of 128 bytes; chunk c of row r sits at chunk c ^ ((r / 2) & 7), so
// that the 16-byte reads of 16 rows at one chunk meet all 64 banks once.  The
// direct loads write LDS in lane order, so it is the lane's source address
// that is permuted.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "srbcrs_stream.hpp"   // xcd_remap

namespace srbcrs {
namespace dense {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

enum Kind { kF16 = 0, kBf16 = 1, kSplit = 2 };
constexpr int kStep = 128;                       // bytes of an operand row in one step
__host__ __device__ constexpr int step_values(int kind) { return kind == kSplit ? 32 : 64; }
inline int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
// bytes of an operand row of k values, whole steps
inline int64_t row_bytes(int kind, int64_t k) { return round_up(k, step_values(kind)) / step_values(kind) * kStep; }

struct Operand {
  const void* p;
  int64_t ld;      // bytes between rows
  int64_t batch;   // bytes between matrices of a batch
  int rows;        // rows past the last one are read as the last one
};

struct GemmArgs {
  Operand a, b;
  int steps;            // steps of 128 bytes along the summed dimension
  int split_steps;      // steps of one part where the sum is split (blockIdx.y), else steps
  int tiles_m, tiles_n;
  int tiles;            // of one matrix of the batch
  int first;            // the launch's first tile, counted through the batch
};

// The tile's rows and columns that a wave holds: acc[i][j][e] is the element
// (m0 + 16 i + 4 (lane / 16) + e, n0 + 16 j + lane % 16).
struct Where {
  int m0, n0;
  int lane;
  int batch;
  int m_part;      // index of this wave's rows among all waves' along m
  bool mirror;     // a symmetric product's tile whose transpose no workgroup computes
  float* lds;      // this wave's share of the tiles' LDS, free after the products
};

__device__ __forceinline__ int row_of(const Where& w, int i) { return w.m0 + 16 * i + 4 * (w.lane >> 4); }
__device__ __forceinline__ int col_of(const Where& w, int j) { return w.n0 + 16 * j + (w.lane & 15); }

// Tile `id` of a matrix.  Symmetric products: the tiles on and below the diagonal, by rows.
// Others: strips of 8 tile rows, whose A tiles and current B tiles stay in an XCD's L2.
template <bool SYM>
__device__ __forceinline__ void tile_at(const GemmArgs& g, int id, int& tm, int& tn) {
  if constexpr (SYM) {
    tm = (int)((sqrtf(8.f * id + 1.f) - 1.f) * 0.5f);
    while ((tm + 1) * (tm + 2) / 2 <= id) ++tm;
    while (tm * (tm + 1) / 2 > id) --tm;
    tn = id - tm * (tm + 1) / 2;
  } else {
    const int strip = id / (8 * g.tiles_n), in = id - strip * 8 * g.tiles_n;
    const int h = min(8, g.tiles_m - 8 * strip);
    tm = 8 * strip + in % h;
    tn = in / h;
  }
}

// Results leave through LDS, 32 x 32 at a time: the wave turns its registers
// (4 consecutive rows of one column each) into 16 bytes a lane,
// of a row or of a column, for stores of whole lines in either order, and the code
// behind it is there once for each 32 rows only.  LDS holds column c's rows at
// c * kBlockLd: 16-byte writes of 16 lanes meet all banks once.
constexpr int kBlockLd = 36;

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// value(row, column, x): the final values of four rows of a column from their sums x;
// block(t, r, c): the 32 x 32 block at t has its first element at (r, c).
template <int TI, int TJ, class V, class F>
__device__ __forceinline__ void through_lds(float4v (&acc)[TI][TJ], const Where& w, V&& value, F&& block) {
#pragma unroll
  for (int i = 0; i < TI; i += 2) {
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4v v = value(row_of(w, i + h), col_of(w, j), acc[i + h][j]);
        *(float4v*)(w.lds + (16 * j + (w.lane & 15)) * kBlockLd + 16 * h + 4 * (w.lane >> 4)) = v;
      }
    wave_fence();
#pragma unroll 1
    for (int j = 0; j < TJ / 2; ++j) block(w.lds + j * 32 * kBlockLd, w.m0 + 16 * i, w.n0 + 32 * j);
    wave_fence();
  }
}

// Four consecutive values of an operand row (k % 4 == 0).
template <int KIND>
__device__ __forceinline__ void put4(void* row, int k, float4v v) {
  if constexpr (KIND == kSplit) {
    char* s = (char*)row + (int64_t)(k >> 5) * kStep + 2 * (k & 31);
    half4 hi, lo;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      hi[q] = (_Float16)v[q];
      lo[q] = (_Float16)(v[q] - (float)hi[q]);
    }
    *(half4*)s = hi;
    *(half4*)(s + 64) = lo;
  } else if constexpr (KIND == kF16) {
    half4 h;
#pragma unroll
    for (int q = 0; q < 4; ++q) h[q] = (_Float16)v[q];
    *(half4*)((_Float16*)row + k) = h;
  } else {
    bf4 h;
#pragma unroll
    for (int q = 0; q < 4; ++q) h[q] = (__bf16)v[q];
    *(bf4*)((__bf16*)row + k) = h;
  }
}
// The rows (COLUMNS: the columns) of the 32 x 32 block at t as operand rows: a line of
// 128 bytes (one float16: 64) a row, 16 bytes a lane, whole lines a store; the
// block_stores() of them one by one.  place(i): where row i's values go, null: nowhere.
template <int KIND>
__device__ constexpr int block_stores() { return KIND == kSplit ? 4 : 2; }
template <int KIND, bool COLUMNS, class P>
__device__ __forceinline__ void put_block(const float* t, int lane, int store, P&& place) {
  constexpr int LANES = KIND == kSplit ? 8 : 4;
  const int c = lane % LANES, k = 8 * (c & 3), i = store * (64 / LANES) + lane / LANES;
  char* p = place(i);
  if (!p) return;
  float v[8];
  if constexpr (COLUMNS) {
    const float4v* s = (const float4v*)(t + i * kBlockLd + k);
    const float4v x = s[0], y = s[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = x[e], v[4 + e] = y[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = t[(k + e) * kBlockLd + i];
  }
  half8 h;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const _Float16 hi = (_Float16)v[e];
    h[e] = KIND == kSplit && c >= 4 ? (_Float16)(v[e] - (float)hi) : hi;
  }
  *(half8*)(p + 16 * c) = h;
}
template <int KIND, bool COLUMNS, class P>
__device__ __forceinline__ void put_block(const float* t, int lane, P&& place) {
#pragma unroll
  for (int i = 0; i < block_stores<KIND>(); ++i) put_block<KIND, COLUMNS>(t, lane, i, place);
}
// place of column k (a multiple of 32) in an operand row
template <int KIND>
__device__ __forceinline__ int64_t offset32(int k) { return KIND == kSplit ? (int64_t)(k >> 5) * kStep : 2 * (int64_t)k; }

template <int KIND>
__device__ __forceinline__ float4v mma(float4v a, float4v b, float4v c) {
  if constexpr (KIND == kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// 16 bytes a lane to LDS, in lane order from `to`, which the wave's lanes share.
__device__ __forceinline__ void load_lds(const char* from, char* to) {
  typedef __attribute__((address_space(3))) void lds_void;
  __builtin_amdgcn_global_load_lds(from, (lds_void*)to, 16, 0, 0);
}

// The order of MM matrix instructions, RD LDS reads and then LD direct loads
// that do not depend on each other: one of these after a matrix instruction, which leaves the
// wave 12 cycles to issue it in.  Reads come first, so that they arrive before the next group.
template <int MM, int RD, int LD>
__device__ __forceinline__ void mix() {
  constexpr int RSLOTS = (LD ? MM / 4 : MM / 2) > 0 ? (LD ? MM / 4 : MM / 2) : 1;
  constexpr int RPS = (RD + RSLOTS - 1) / RSLOTS, USED = RPS ? (RD + RPS - 1) / RPS : 0;
  constexpr int LSLOTS = MM > USED ? MM - USED : 1, LPS = (LD + LSLOTS - 1) / LSLOTS;
  constexpr int EVERY = LD && LSLOTS / LD > 1 ? LSLOTS / LD : 1;
#pragma unroll
  for (int n = 0; n < MM; ++n) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (n < USED) __builtin_amdgcn_sched_group_barrier(0x100, RPS, 0);
    else if (LPS && (n - USED) % EVERY == 0) __builtin_amdgcn_sched_group_barrier(0x020, LPS, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// The workgroup's barrier that leaves N of a wave's direct loads in flight (__syncthreads waits
// for all).  LDS reads before it are complete, LDS writes of the other loads visible.
template <int N>
__device__ __forceinline__ void step_barrier() {
  wait_vmcnt<N>();
  wait_lgkmcnt0();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// One workgroup: a BM x BN tile on WM x WN waves.  SYM: A = B, square tiles,
// the tiles with tm >= tn only.
//
// The loop.  The products run in phases, and while one runs, the operands of the next
// are read from LDS into registers that no running product uses.  Before a
// step's last phase the wave has read all of the step, so that after a barrier
// its place in LDS is free for loads.  LDS holds two steps of A and three of B, all of a
// CU's 160 KB with 256 x 256 tiles or twice 128 x 128: a step's A is loaded one step ahead,
// its B two, since half a step's rows arrive in time in one step and all of them do not.
// One barrier a step.  Phases: of 32 values each, two a step; kSplit: high low, high high, low
// high, so that each part is read once and four register sets do.
//
// The largest tile has eight waves of 128 x 64.  32x32x16 instructions move
// twice the accumulators for a multiply-add; with them the same loop took an eighth longer
// (a training step of 8192 rows, 65536 classes, 2048 features).  8192 x 65536 x 2048, bfloat16,
// takes 1.79 ms: 1230 TFLOP/s at the power limit, where clocks fall to 1.7 to 1.9 GHz.
template <int KIND, int BM, int BN, int WM, int WN, bool SYM, class Epi>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_gemm(GemmArgs g, Epi epi) {
  constexpr int NW = WM * WN, TI = BM / WM / 16, TJ = BN / WN / 16;
  constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW;   // 1 KB loads of a wave in a step
  constexpr int BUF_A = BM * kStep, BUF_B = BN * kStep, LDS = 2 * BUF_A + 3 * BUF_B;
  static_assert(LA * 8 * NW == BM && LB * 8 * NW == BN && TI * 16 * WM == BM && TJ * 16 * WN == BN, "tile shape");
  static_assert(TI % 2 == 0 && TJ % 2 == 0, "results leave in blocks of 32 x 32");
  __shared__ __attribute__((aligned(1024))) char lds[LDS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = g.first + (int)xcd_remap(blockIdx.x, gridDim.x), batch = id / g.tiles;
  int tm, tn;
  tile_at<SYM>(g, id - batch * g.tiles, tm, tn);
  const int first = blockIdx.y * g.split_steps;
  const int steps = min(g.split_steps, g.steps - first);

  // this lane's source address of each of its wave's loads
  const char *src_a[LA], *src_b[LB];
  {
    auto of = [&](const Operand& o, int tile_row, int r) {   // row r of the tile
      const int row = min(tile_row + r, o.rows - 1), c = (lane & 7) ^ ((r >> 1) & 7);
      return (const char*)o.p + batch * o.batch + row * o.ld + (int64_t)first * kStep + c * 16;
    };
#pragma unroll
    for (int i = 0; i < LA; ++i) src_a[i] = of(g.a, tm * BM, (wave * LA + i) * 8 + (lane >> 3));
#pragma unroll
    for (int i = 0; i < LB; ++i) src_b[i] = of(g.b, tn * BN, (wave * LB + i) * 8 + (lane >> 3));
  }
  // the next step to a buffer; past the last step it is loaded again, and never read
  auto load_a = [&](int buf, bool more) {
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      load_lds(src_a[i], lds + buf * BUF_A + (wave * LA + i) * 1024);
      src_a[i] += more ? kStep : 0;
    }
  };
  auto load_b = [&](int buf, bool more) {
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      load_lds(src_b[i], lds + 2 * BUF_A + buf * BUF_B + (wave * LB + i) * 1024);
      src_b[i] += more ? kStep : 0;
    }
  };

  const int wm = wave / WN, wn = wave % WN;
  float4v acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};

  const int a_row = (wm * TI * 16 + (lane & 15)) * kStep;
  const int b_row = 2 * BUF_A + (wn * TJ * 16 + (lane & 15)) * kStep;
  // chunk 4 half + lane / 16 of the rows; a half of a step is 32 values, or all values' high or low parts
  const int chunk0 = ((lane >> 4) ^ ((lane >> 1) & 7)) * 16;
  auto read_a = [&](float4v(&to)[TI], int buf, int half) {
    const char* t = lds + buf * BUF_A + a_row + (chunk0 ^ (half * 64));
#pragma unroll
    for (int i = 0; i < TI; ++i) to[i] = *(const float4v*)(t + i * 16 * kStep);
  };
  auto read_b = [&](float4v(&to)[TJ], int buf, int half) {
    const char* t = lds + buf * BUF_B + b_row + (chunk0 ^ (half * 64));
#pragma unroll
    for (int j = 0; j < TJ; ++j) to[j] = *(const float4v*)(t + j * 16 * kStep);
  };
  auto multiply = [&](const float4v(&a)[TI], const float4v(&b)[TJ]) {
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j] = mma<KIND>(a[i], b[j], acc[i][j]);
  };
  float4v a0[TI], b0[TJ], a1[TI], b1[TJ];
  constexpr int MM = TI * TJ;
  if (steps > 0) {
    load_a(0, steps > 1);
    load_b(0, steps > 1);
    load_a(1, steps > 2);
    load_b(1, steps > 2);
    load_b(2, steps > 3);
    step_barrier<LA + 2 * LB>();
    int pa = 0, pb = 0;   // the current step's buffers
    // a phase's end: all of the current step is in registers, the next step in LDS
    auto turn = [&] {
      step_barrier<LB>();
      pa ^= 1;
      pb = pb == 2 ? 0 : pb + 1;
    };
    // into the last step's buffers, after turn()
    auto loads = [&](int s) {
      load_a(pa ^ 1, s + 3 < steps);
      load_b(pb == 0 ? 2 : pb - 1, s + 4 < steps);
    };
    if constexpr (KIND == kSplit) {
      // a0, a1: high and low parts, b0, b1 likewise
      read_a(a0, 0, 0);
      read_b(b1, 0, 1);
      __builtin_amdgcn_sched_barrier(0);
      for (int s = 0; s < steps; ++s) {
        read_b(b0, pb, 0);
        multiply(a0, b1);
        mix<MM, TJ, 0>();
        read_a(a1, pa, 1);
        multiply(a0, b0);
        mix<MM, TI, 0>();
        turn();
        read_a(a0, pa, 0);
        read_b(b1, pb, 1);
        loads(s);
        multiply(a1, b0);
        mix<MM, TI + TJ, LA + LB>();
      }
    } else {
      read_a(a0, 0, 0);
      read_b(b0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      for (int s = 0; s < steps; ++s) {
        read_a(a1, pa, 1);
        read_b(b1, pb, 1);
        multiply(a0, b0);
        mix<MM, TI + TJ, 0>();
        turn();
        read_a(a0, pa, 0);
        read_b(b0, pb, 0);
        loads(s);
        multiply(a1, b1);
        mix<MM, TI + TJ, LA + LB>();
      }
    }
  }
  Where w;
  w.m0 = tm * BM + wm * TI * 16;
  w.n0 = tn * BN + wn * TJ * 16;
  w.lane = lane;
  w.batch = batch;
  w.m_part = tm * WM + wm;
  w.mirror = SYM && tm != tn;
  static_assert(TJ * 16 * kBlockLd * 4 * NW <= LDS && LDS / NW % 16 == 0, "the waves' blocks fit the tiles' LDS");
  w.lds = (float*)(lds + wave * (LDS / NW));
  wait_vmcnt<0>();   // loads past the last step still write LDS
  __syncthreads();
  epi.template store<TI, TJ>(acc, w);
}

// Sums of a part of the steps as they are, in the order of the registers:
// [part][tile of the launch][wave][32 x 32 block of it][fragment][lane].
struct PartEpi {
  float4v* part;
  template <int TI, int TJ>
  __device__ void store(float4v (&acc)[TI][TJ], const Where& w) const {
    const int64_t tile = (int64_t)blockIdx.y * gridDim.x + xcd_remap(blockIdx.x, gridDim.x);
    float4v* p = part + (tile * (blockDim.x >> 6) + (threadIdx.x >> 6)) * (TI * TJ * 64) + w.lane;
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j) p[(((i / 2) * (TJ / 2) + j / 2) * 4 + (i & 1) * 2 + (j & 1)) * 64] = acc[i][j];
  }
};

// The parts' sums, in order, and the product's own end.  A wave joins a 32 x 32 block.
template <int BM, int BN, int WM, int WN, bool SYM, class Epi>
__global__ __launch_bounds__(256) void k_join(GemmArgs g, const float4v* __restrict__ part, int n_tiles, int parts, Epi epi) {
  constexpr int TI = BM / WM / 16, TJ = BN / WN / 16, PER_WAVE = TI * TJ / 4, PER = WM * WN * PER_WAVE;
  __shared__ __attribute__((aligned(16))) float lds[4][32 * kBlockLd];
  const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int slot = id / PER, block = id - slot * PER, wave = block / PER_WAVE, bi = block - wave * PER_WAVE;
  if (slot >= n_tiles) return;
  const int tile = g.first + slot, batch = tile / g.tiles;
  int tm, tn;
  tile_at<SYM>(g, tile - batch * g.tiles, tm, tn);
  float4v acc[2][2];
#pragma unroll
  for (int f = 0; f < 4; ++f) acc[f >> 1][f & 1] = float4v{0.f, 0.f, 0.f, 0.f};
  const float4v* p = part + (int64_t)id * 256 + lane;
#pragma unroll 4
  for (int s = 0; s < parts; ++s)
#pragma unroll
    for (int f = 0; f < 4; ++f) acc[f >> 1][f & 1] += p[(int64_t)s * n_tiles * PER * 256 + f * 64];
  Where w;
  w.m0 = tm * BM + wave / WN * TI * 16 + bi / (TJ / 2) * 32;
  w.n0 = tn * BN + wave % WN * TJ * 16 + bi % (TJ / 2) * 32;
  w.lane = lane;
  w.batch = batch;
  w.m_part = 0;   // not for results by wave rows
  w.mirror = SYM && tm != tn;
  w.lds = lds[threadIdx.x >> 6];
  epi.template store<2, 2>(acc, w);
}

// Few tiles: a workgroup of 8 waves a 32 x 32 tile, the steps dealt to the waves,
// operands straight from memory to registers (a row's 16 bytes a lane), sums joined in LDS.
// Nothing is shared in the loop, so a short sum costs one load's latency.  Where the
// epilogue has parts (SHARED), four waves finish a quarter of the tile each, with what else they read
// on its way before the sums are, and all eight write it (512 x 256 orthogonalised: 93 us; by one wave 112).
template <int KIND, bool SYM, class Epi>
__global__ __launch_bounds__(512) void k_gemm_few(GemmArgs g, Epi epi) {
  __shared__ __attribute__((aligned(16))) float4v red[8][256];
  __shared__ __attribute__((aligned(16))) float block[32 * kBlockLd];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = (int)xcd_remap(blockIdx.x, gridDim.x), batch = id / g.tiles;
  int tm, tn;
  tile_at<SYM>(g, id - batch * g.tiles, tm, tn);
  const char *pa[2], *pb[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    pa[i] = (const char*)g.a.p + batch * g.a.batch + min(tm * 32 + 16 * i + (lane & 15), g.a.rows - 1) * g.a.ld + 16 * (lane >> 4);
    pb[i] = (const char*)g.b.p + batch * g.b.batch + min(tn * 32 + 16 * i + (lane & 15), g.b.rows - 1) * g.b.ld + 16 * (lane >> 4);
  }
  float4v acc[2][2], a[2][2], b[2][2];   // operands: [half of the step][tile]
#pragma unroll
  for (int f = 0; f < 4; ++f) acc[f >> 1][f & 1] = float4v{0.f, 0.f, 0.f, 0.f};
  auto fetch = [&](int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[h][i] = *(const float4v*)(pa[i] + (int64_t)s * kStep + 64 * h);
        b[h][i] = *(const float4v*)(pb[i] + (int64_t)s * kStep + 64 * h);
      }
  };
  if (wave < g.steps) fetch(wave);
  Where w;
  w.m0 = tm * 32;
  w.n0 = tn * 32;
  w.lane = lane;
  w.batch = batch;
  w.m_part = tm;
  w.mirror = SYM && tm != tn;
  w.lds = block;
  // this wave's quarter
  [[maybe_unused]] const int row = row_of(w, (wave >> 1) & 1), col = col_of(w, wave & 1);
  [[maybe_unused]] auto with = epi.before(w, row, col);
  for (int s = wave; s < g.steps; s += 8) {
    float4v x[2][2], y[2][2];
#pragma unroll
    for (int f = 0; f < 4; ++f) x[f >> 1][f & 1] = a[f >> 1][f & 1], y[f >> 1][f & 1] = b[f >> 1][f & 1];
    if (s + 8 < g.steps) fetch(s + 8);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (KIND == kSplit) {
          acc[i][j] = mma<KIND>(x[0][i], y[1][j], acc[i][j]);
          acc[i][j] = mma<KIND>(x[1][i], y[0][j], acc[i][j]);
        } else {
          acc[i][j] = mma<KIND>(x[1][i], y[1][j], acc[i][j]);
        }
        acc[i][j] = mma<KIND>(x[0][i], y[0][j], acc[i][j]);
      }
  }
#pragma unroll
  for (int f = 0; f < 4; ++f) red[wave][f * 64 + lane] = acc[f >> 1][f & 1];
  __syncthreads();
  if constexpr (Epi::SHARED) {
    if (wave < 4) {
      float4v t = red[0][threadIdx.x];
#pragma unroll
      for (int k = 1; k < 8; ++k) t += red[k][threadIdx.x];
      *(float4v*)(block + (col - w.n0) * kBlockLd + row - w.m0) = epi.value(with, row, col, t);
    }
    __syncthreads();
    epi.lines(w, block, w.m0, w.n0, wave);
  } else {
    if (threadIdx.x < 256) {
      float4v t = red[0][threadIdx.x];
#pragma unroll
      for (int k = 1; k < 8; ++k) t += red[k][threadIdx.x];
      red[0][threadIdx.x] = t;
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int f = 0; f < 4; ++f) acc[f >> 1][f & 1] = red[0][f * 64 + lane];
    epi.template store<2, 2>(acc, w);
  }
}

// An epilogue whose results leave in 32 x 32 blocks:
//  before(w, r, c)      what value() needs from memory for rows r... of column c;
//  value(that, r, c, x) the final values of four rows of a column from their sums;
//  lines(w, t, r, c, i) share i of 8 of the block at t to memory.
template <class E>
struct BlockEpi {
  static constexpr bool SHARED = true;
  template <int TI, int TJ>
  __device__ __forceinline__ void store(float4v (&acc)[TI][TJ], const Where& w) const {
    const E& e = static_cast<const E&>(*this);
    through_lds<TI, TJ>(
        acc, w, [&](int r, int c, float4v x) { return e.value(e.before(w, r, c), r, c, x); },
        [&](const float* t, int r, int c) {
#pragma unroll
          for (int i = 0; i < 8; ++i) e.lines(w, t, r, c, i);
        });
  }
};
// All of it by one wave.
struct WaveEpi {
  static constexpr bool SHARED = false;
  __device__ __forceinline__ int before(const Where&, int, int) const { return 0; }
};

// ---- tiles ------------------------------------------------------------------

enum Tile { kTile256 = 0, kTile128 = 1, kTile64 = 2, kTileFew = 3 };
__host__ constexpr int tile_size(int t) { return t == kTile256 ? 256 : t == kTile128 ? 128 : t == kTile64 ? 64 : 32; }
// rows of a wave's part of a tile, and such parts of a tile
__host__ constexpr int waves_m(int t) { return t == kTileFew ? 1 : 2; }

inline int64_t tile_count(int t, int64_t m, int64_t n, bool sym) {
  const int64_t a = (m + tile_size(t) - 1) / tile_size(t), b = (n + tile_size(t) - 1) / tile_size(t);
  return sym ? a * (a + 1) / 2 : a * b;
}

// How a product is cut: `whole` tiles (through the batch) with all their steps,
// then the rest's steps in `parts` parts that are joined afterwards.
struct Cut {
  int tile = kTile64;
  int64_t whole = 0, rest = 0;
  int parts = 1;
  // floats of the parts' sums
  size_t floats() const { return parts > 1 ? (size_t)parts * rest * tile_size(tile) * tile_size(tile) : 0; }
};

// The cut that takes the least time by what launches take here, in microseconds,
// measured over products of 64 to 4096 rows, sums of 64 to 8000 and batches of 1 to 12: the ends of a
// workgroup, then a step's time, which is that of the workgroups of a CU one after
// another but no less than one workgroup's latency (more of it the more CUs work).
// Examples, kSplit: 512 x 512 x 512 takes 8 us in few tiles, 11 in 64, 16 in 128, 39 in 256; 4096 x 4096 x
// 4096 takes 456 in 64, 322 in 128, 287 in 256; 300 x 300 x 8000 takes 96 in tiles of 64 and 24 in 8 parts of 128.
// join: whether the result can be joined from parts.  few: whether the tiles may
// reach to a multiple of 32 only, not 64 (rows of one float16 are filled to 64).
inline Cut cut_for(int kind, int64_t m, int64_t n, int64_t k, int64_t batch, bool sym, bool join, bool few = true) {
  struct Cost { int resident; double ends, step, alone, loaded; };
  // tiles of 256, 128, 64, few
  static const Cost two[4] = {{1, 12.0, 2.2, 1.4, 2.2}, {2, 5.0, 0.66, 0.47, 0.80}, {4, 4.0, 0.225, 0.37, 0.42}, {4, 3.7, 0.25, 0.09, 0.12}};
  static const Cost one[4] = {{1, 12.0, 1.72, 1.2, 1.72}, {2, 5.0, 0.53, 0.42, 0.68}, {4, 4.0, 0.19, 0.34, 0.38}, {4, 3.7, 0.20, 0.08, 0.10}};
  const int64_t steps = row_bytes(kind, k) / kStep;
  Cut best;
  double best_t = INFINITY;
  for (int t = 0; t < (few ? 4 : 3); ++t) {
    const Cost& c = (kind == kSplit ? two : one)[t];
    const int64_t total = tile_count(t, m, n, sym) * batch, slots = 256 * c.resident;
    // One operand of a single tile: the other is read once, and waves that share nothing read it faster
    // (32000 x 1 x 2048 takes 31 us for 36 in tiles of 64).
    if (few && t != kTileFew && (m <= 32 || n <= 32) && tile_count(kTileFew, m, n, sym) * batch >= 256) continue;
    auto time = [&](int64_t tiles, double s) {   // tiles <= slots, s steps each
      const double busy = (double)((tiles + 255) / 256) * c.step;
      const double latency = c.alone + (c.loaded - c.alone) * (tiles < 256 ? tiles / 256.0 : 1.0);
      return tiles ? c.ends + s * (busy > latency ? busy : latency) : 0.0;
    };
    const int64_t full = total / slots, rest = total % slots;
    const double whole = (double)full * time(slots, (double)steps);
    const double plain = whole + time(rest, (double)steps);
    if (plain < best_t) {
      best_t = plain;
      best = Cut();
      best.tile = t, best.whole = total;
    }
    if (!join || t == kTileFew || !rest) continue;
    // the rest in parts of its sums: whole generations of them where it takes long
    // (2073 x 2364, sums of 55732, float32: 90 tiles of 256 in 2 parts fill 180 CUs of 256, in 5 two generations)
    for (int64_t parts = 2; parts <= slots / rest || parts <= 8; ++parts) {
      if (parts > steps / 4) break;
      const int64_t each = (steps + parts - 1) / parts, left = rest * parts % slots;
      // the parts' sums go to memory and back
      const double bytes = 8.0 * parts * rest * tile_size(t) * tile_size(t);
      const double joined = whole + (double)(rest * parts / slots) * time(slots, (double)each) + time(left, (double)each) + 6.0 + bytes / 4e6;
      if (joined < best_t) {
        best_t = joined;
        best = Cut();
        best.tile = t, best.whole = total - rest, best.rest = rest, best.parts = (int)parts;
      }
    }
  }
  return best;
}

template <int KIND, int BM, int WN, bool SYM, bool JOIN, class Epi>
void launch_cut(const Cut& cut, GemmArgs g, const Epi& epi, float* scratch, hipStream_t stream) {
  constexpr int threads = 64 * 2 * WN;
  if (cut.whole) k_gemm<KIND, BM, BM, 2, WN, SYM><<<dim3((unsigned)cut.whole, 1), threads, 0, stream>>>(g, epi);
  if constexpr (JOIN) {
    if (!cut.rest) return;
    g.first = (int)cut.whole;
    const int steps = g.split_steps;
    g.split_steps = (steps + cut.parts - 1) / cut.parts;
    const int parts = (steps + g.split_steps - 1) / g.split_steps;
    k_gemm<KIND, BM, BM, 2, WN, SYM>
        <<<dim3((unsigned)cut.rest, (unsigned)parts), threads, 0, stream>>>(g, PartEpi{(float4v*)scratch});
    const unsigned waves = (unsigned)(cut.rest * (BM / 32) * (BM / 32));
    k_join<BM, BM, 2, WN, SYM><<<(waves + 3) / 4, 256, 0, stream>>>(g, (const float4v*)scratch, (int)cut.rest, parts, epi);
  }
}

// D = A B^T by the cut of (a.rows, b.rows, k, batch); scratch: cut.floats() floats.
// JOIN: as the cut was asked for.
template <int KIND, bool SYM, bool JOIN, class Epi>
void launch(const Cut& cut, const Operand& a, const Operand& b, int64_t k, const Epi& epi, float* scratch, hipStream_t stream) {
  GemmArgs g{};
  g.a = a, g.b = b;
  g.steps = g.split_steps = (int)(row_bytes(KIND, k) / kStep);
  const int ts = tile_size(cut.tile);
  g.tiles_m = (a.rows + ts - 1) / ts;
  g.tiles_n = (b.rows + ts - 1) / ts;
  g.tiles = (int)tile_count(cut.tile, a.rows, b.rows, SYM);
  if (cut.tile == kTile256) launch_cut<KIND, 256, 4, SYM, JOIN>(cut, g, epi, scratch, stream);
  else if (cut.tile == kTile128) launch_cut<KIND, 128, 2, SYM, JOIN>(cut, g, epi, scratch, stream);
  else if (cut.tile == kTile64) launch_cut<KIND, 64, 2, SYM, JOIN>(cut, g, epi, scratch, stream);
  else k_gemm_few<KIND, SYM><<<(unsigned)cut.whole, 512, 0, stream>>>(g, epi);
}

}  // namespace dense
}  // namespace srbcrs
