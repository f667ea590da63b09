// What the two forms of the linear cross entropy share: srbcrs_xent.hip
// (any number of classes) and srbcrs_xent_few.hip (few).
#pragma once
#include "srbcrs_operand.hpp"

namespace srbcrs {
namespace xent {
using namespace dense;

constexpr float kLog2e = 1.44269504088896341f;

// Output values: sum * alpha / (operand's scale) (* the unit of a factor folded into an
// operand) + what earlier pieces left, times the row's factor.
struct Out {
  void* p;
  int64_t ld;
  int dtype;
  const float* prev;        // null: none; [m][n] with n values a row
  const unsigned* largest;  // what the operand is scaled by (k_pack_t), null: it is not
  float alpha;
  const float* row;         // null: 1
  const unsigned* fmax;     // largest of the factors folded into an operand (k_pack_t), null: none
  int m, n;
  __device__ float factor() const {
    return alpha * (largest ? power_of_two(-scale_exponent(largest, fmax)) : 1.f) * (fmax ? factor_unit(fmax) : 1.f);
  }
  // v is already times factor()
  __device__ float finish(int r, int c, float v) const {
    if (prev) v += prev[(int64_t)r * n + c];
    if (row) {
      const float f = row[r];
      v = f == 0.f ? 0.f : v * f;
    }
    return v;
  }
  __device__ void put(int r, int c, float v) const {
    const int64_t at = (int64_t)r * ld + c;
    if (dtype == kF32T) ((float*)p)[at] = v;
    else if (dtype == kBf16T) ((__bf16*)p)[at] = (__bf16)v;
    else ((_Float16*)p)[at] = (_Float16)v;
  }
};

// Sums over `splits` parts [m][n] of 32-bit sums, in order, to o.
void join_parts(const float* part, int splits, const Out& o, hipStream_t s);
// The loss over all rows and the number of labelled ones from n workgroups' sums of both.
void total(const float2* block_sum, int n, const XentArgs& a, float* loss, hipStream_t s);
// Rows' largest magnitudes, and where the largest exponents of h times its rows' factors and of w go; null: not wanted.
struct Magnitudes {
  const float *h, *w;
  unsigned *h_largest, *w_largest;
};
// Rows' factors, zeros up to a multiple of 32 rows, and the largest of them
// (zeroed: that, and what else is joined, is 0 already).
void factors(const XentArgs& a, const float* dloss, float* factor, unsigned* fmax, bool zeroed, hipStream_t s,
             const Magnitudes& mag = {});

// Rows' statistics, losses (loss: each, may be null) and sums (block_sum: one a row, may be
// null) from `parts` parts [part][row] of few rows.
void join_stats(const float2* part, int parts, const float* zt, const XentArgs& a, float* loss, float2* block_sum,
                hipStream_t s);

// Few classes or few rows: waves hold logits with all of them in registers.
constexpr int64_t kFewClasses = 128, kFewRows = 128;
bool few_forwards(const XentArgs& a, bool readable);
bool few_backwards(const XentArgs& a);
size_t few_forward(const XentArgs& a, float* loss, hipStream_t s);
size_t few_backward(const XentArgs& a, const float* dloss, void* dh, void* dw, hipStream_t s);

}  // namespace xent
}  // namespace srbcrs
