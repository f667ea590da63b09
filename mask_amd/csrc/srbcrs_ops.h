// Internal launch interface of the training operators (group norm, linear
// cross entropy, orthogonalised updates).  Arguments are checked by the C ABI
// layer (srbcrs_ops_capi.cpp); launches report through hipGetLastError.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace srbcrs {

enum Dtype { kF32T = 0, kBf16T = 1, kF16T = 2 };   // SRBCRS_F32, _BF16, _F16
inline int dtype_size(int t) { return t == kF32T ? 4 : 2; }

// Pieces of one caller workspace, 256-byte aligned; base null: sizes only.
struct Carver {
  char* base;
  size_t used = 0;
  explicit Carver(void* p) : base((char*)p) {}
  template <class T>
  T* take(size_t n) {
    T* p = base ? (T*)(base + used) : nullptr;
    used += (n * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

// Zeros, by a kernel: a memset node of a captured graph is not replayed reliably.
void fill_zero(void* p, size_t bytes, hipStream_t stream);

struct XentArgs {
  const void *h, *w;
  int64_t ldh, ldw;          // values between rows
  int64_t rows, dim, classes;
  int dtype;
  const int64_t* target;
  int64_t ignore;
  int reduction;             // 0 none, 1 mean, 2 sum
  float* lse;                // rows: kept from the forward pass for the backward pass
  float* count;              // 1: max(labelled rows, 1), likewise
  void* ws;
};
// ws == null: nothing runs.  Returns the bytes of workspace that the call uses.
size_t xent_forward(const XentArgs& a, float* loss, hipStream_t stream);
size_t xent_backward(const XentArgs& a, const float* dloss, void* dh, void* dw, hipStream_t stream);

struct OrthoArgs {
  const void* g;
  void* out;
  int64_t batch, rows, cols, ldg, batch_g;   // values between rows and matrices of g; out is contiguous
  int dtype, steps;
  float a, b, c, eps;
  void* ws;
};
// out == null: nothing runs.  Returns the bytes of workspace that the call uses, maybe none.
size_t ortho(const OrthoArgs& a, hipStream_t stream);

struct NormArgs {
  const void *x, *weight, *bias;     // weight, bias: may be null
  int64_t batch, length, channels, groups;
  int64_t ldx, batch_x;              // values between rows and samples of x
  int dtype, param_dtype, act;
  float eps;
  float* stats;                      // batch x groups x 4: mean, 1 / sqrt(var + eps), their low parts
  void* ws;
};
// The workspace that any alignment of the arguments may use.
size_t norm_workspace(const NormArgs& a, bool backward);
void norm_forward(const NormArgs& a, void* y, hipStream_t stream);
void norm_backward(const NormArgs& a, const void* dy, int64_t lddy, int64_t batch_dy, void* dx, void* dweight,
                     void* dbias, hipStream_t stream);

}  // namespace srbcrs
