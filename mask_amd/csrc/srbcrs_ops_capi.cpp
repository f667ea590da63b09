// C ABI of the training operators: argument checks, then the launches.
// Declarations: include/srbcrs.h.
#include <hip/hip_runtime.h>
#include <math.h>

#include "srbcrs_error.h"
#include "srbcrs_ops.h"

namespace {

using namespace srbcrs;

constexpr int64_t kMostRows = INT32_MAX - 1024;   // 32-bit tile coordinates, rounded up to tiles
constexpr int64_t kMostValues = int64_t(1) << 46;

void check_dtype(int dtype, const char* name) {
  if (dtype != SRBCRS_F32 && dtype != SRBCRS_BF16 && dtype != SRBCRS_F16) fail(SRBCRS_EINVAL, "unknown %s %d", name, dtype);
}
void check_size(int64_t v, int64_t most, const char* name) {
  if (v < 0 || v > most) fail(SRBCRS_EINVAL, "%s out of range: %lld", name, (long long)v);
}
void check_ptr(const void* p, const char* name) {
  if (!p) fail(SRBCRS_EINVAL, "%s is NULL", name);
}
void check_aligned(const void* p, int dtype, const char* name) {
  if ((uintptr_t)p % dtype_size(dtype)) fail(SRBCRS_EINVAL, "%s is not aligned to its values", name);
}
// a need of 1: none is used
void check_ws(const void* ws, size_t have, size_t need) {
  if (need <= 1) return;
  if (!ws) fail(SRBCRS_EINVAL, "workspace is NULL");
  if ((uintptr_t)ws % 256) fail(SRBCRS_EINVAL, "workspace is not 256-byte aligned");
  if (have < need) fail(SRBCRS_EINVAL, "workspace of %zu bytes is too small: %zu are needed", have, need);
}
void check_launches(const char* what) { hip_check(hipGetLastError(), what); }

// ---- group norm ---------------------------------------------------------------

NormArgs norm_args(const srbcrs_norm_desc* d, bool backward) {
  check_ptr(d, "desc");
  check_dtype(d->dtype, "dtype");
  check_dtype(d->param_dtype, "param_dtype");
  check_size(d->batch, kMostRows, "batch");
  check_size(d->length, kMostRows, "length");
  check_size(d->channels, 1 << 20, "channels");
  if (d->groups < 1 || d->channels % d->groups) fail(SRBCRS_EINVAL, "channels must be a multiple of groups");
  if (d->batch && d->length && d->channels && (double)d->batch * d->length * d->channels > (double)kMostValues)
    fail(SRBCRS_EINVAL, "too many values");
  if (d->activation < SRBCRS_ACT_NONE || d->activation > SRBCRS_ACT_GELU)
    fail(SRBCRS_EINVAL, "unknown activation %d", d->activation);
  if (!(d->eps >= 0.f) || !isfinite(d->eps)) fail(SRBCRS_EINVAL, "eps must be finite and not negative");
  if (d->length > 1 && d->ld_x < 0) fail(SRBCRS_EINVAL, "ld_x must not be negative");
  if (d->batch > 1 && d->batch_x < 0) fail(SRBCRS_EINVAL, "batch_x must not be negative");
  if (backward && ((d->length > 1 && d->ld_dy < 0) || (d->batch > 1 && d->batch_dy < 0)))
    fail(SRBCRS_EINVAL, "strides of dy must not be negative");
  NormArgs a{};
  a.batch = d->batch, a.length = d->length, a.channels = d->channels, a.groups = d->groups;
  a.ldx = d->ld_x, a.batch_x = d->batch_x;
  a.dtype = d->dtype, a.param_dtype = d->param_dtype, a.act = d->activation, a.eps = d->eps;
  return a;
}
bool empty(const NormArgs& a) { return !a.batch || !a.length || !a.channels; }

// ---- cross entropy --------------------------------------------------------------

XentArgs xent_args(const srbcrs_xent_desc* d, const void* h, const void* w) {
  check_ptr(d, "desc");
  check_dtype(d->dtype, "dtype");
  check_size(d->rows, kMostRows, "rows");
  check_size(d->classes, kMostRows, "classes");
  check_size(d->dim, 1 << 24, "dim");
  if (d->classes < 1) fail(SRBCRS_EINVAL, "at least one class is needed");
  if (d->dim < 1) fail(SRBCRS_EINVAL, "at least one feature is needed");
  if (d->reduction < SRBCRS_REDUCE_NONE || d->reduction > SRBCRS_REDUCE_SUM)
    fail(SRBCRS_EINVAL, "unknown reduction %d", d->reduction);
  if (d->rows > 1 && d->ld_h < 0) fail(SRBCRS_EINVAL, "ld_h must not be negative");
  if (d->classes > 1 && d->ld_w < 0) fail(SRBCRS_EINVAL, "ld_w must not be negative");
  XentArgs a{};
  a.h = h, a.w = w;
  a.ldh = d->ld_h, a.ldw = d->ld_w;
  a.rows = d->rows, a.dim = d->dim, a.classes = d->classes;
  a.dtype = d->dtype, a.ignore = d->ignore_index, a.reduction = d->reduction;
  return a;
}

// ---- orthogonalised updates -------------------------------------------------------

OrthoArgs ortho_args(const srbcrs_ortho_desc* d) {
  check_ptr(d, "desc");
  check_dtype(d->dtype, "dtype");
  check_size(d->batch, 65535, "batch");
  check_size(d->rows, 1 << 24, "rows");
  check_size(d->cols, 1 << 24, "cols");
  if (d->steps < 1 || d->steps > 100) fail(SRBCRS_EINVAL, "steps must be 1 to 100: %d", d->steps);
  const float bound = fabsf(d->a) + 2 * fabsf(d->b) + 4 * fabsf(d->c);
  if (!(bound > 0.f && bound <= 1024.f)) fail(SRBCRS_EINVAL, "coefficients out of range");
  if (!(d->eps >= 0.f) || !isfinite(d->eps)) fail(SRBCRS_EINVAL, "eps must be finite and not negative");
  if ((d->rows > 1 && d->ld_g < 0) || (d->batch > 1 && d->batch_g < 0))
    fail(SRBCRS_EINVAL, "strides of g must not be negative");
  OrthoArgs a{};
  a.batch = d->batch, a.rows = d->rows, a.cols = d->cols, a.ldg = d->ld_g, a.batch_g = d->batch_g;
  a.dtype = d->dtype, a.steps = d->steps, a.a = d->a, a.b = d->b, a.c = d->c, a.eps = d->eps;
  return a;
}

size_t at_least_one(size_t n) { return n ? n : 1; }

}  // namespace

extern "C" {

int srbcrs_group_norm_workspace(const srbcrs_norm_desc* desc, int32_t backward, size_t* bytes) {
  return guarded([&] {
    const NormArgs a = norm_args(desc, backward != 0);
    check_ptr(bytes, "bytes");
    *bytes = empty(a) ? 1 : norm_workspace(a, backward != 0);
  });
}

int srbcrs_group_norm(const srbcrs_norm_desc* desc, const void* d_x, const void* d_weight, const void* d_bias, void* d_y,
                      float* d_stats, void* d_ws, size_t ws_bytes, void* stream) {
  return guarded([&] {
    NormArgs a = norm_args(desc, false);
    if (empty(a)) return;
    check_ptr(d_x, "x");
    check_ptr(d_y, "y");
    check_ptr(d_stats, "stats");
    if ((uintptr_t)d_stats % 16) fail(SRBCRS_EINVAL, "stats is not 16-byte aligned");
    check_aligned(d_x, a.dtype, "x");
    check_aligned(d_y, a.dtype, "y");
    check_aligned(d_weight, a.param_dtype, "weight");
    check_aligned(d_bias, a.param_dtype, "bias");
    check_ws(d_ws, ws_bytes, norm_workspace(a, false));
    a.x = d_x, a.weight = d_weight, a.bias = d_bias, a.stats = d_stats, a.ws = d_ws;
    norm_forward(a, d_y, (hipStream_t)stream);
    check_launches("group norm");
  });
}

int srbcrs_group_norm_backward(const srbcrs_norm_desc* desc, const void* d_dy, const void* d_x, const void* d_weight,
                               const void* d_bias, const float* d_stats, void* d_dx, void* d_dweight, void* d_dbias,
                               void* d_ws, size_t ws_bytes, void* stream) {
  return guarded([&] {
    NormArgs a = norm_args(desc, true);
    if (empty(a)) {
      // sums over nothing
      const size_t bytes = (size_t)a.channels * dtype_size(a.param_dtype);
      if (bytes && d_dweight) fill_zero(d_dweight, bytes, (hipStream_t)stream);
      if (bytes && d_dbias) fill_zero(d_dbias, bytes, (hipStream_t)stream);
      return;
    }
    check_ptr(d_dy, "dy");
    check_ptr(d_x, "x");
    check_ptr(d_stats, "stats");
    if ((uintptr_t)d_stats % 16) fail(SRBCRS_EINVAL, "stats is not 16-byte aligned");
    check_ptr(d_dx, "dx");
    check_aligned(d_x, a.dtype, "x");
    check_aligned(d_dy, a.dtype, "dy");
    check_aligned(d_dx, a.dtype, "dx");
    for (const void* p : {d_weight, d_bias, (const void*)d_dweight, (const void*)d_dbias})
      check_aligned(p, a.param_dtype, "a parameter or its gradient");
    check_ws(d_ws, ws_bytes, norm_workspace(a, true));
    a.x = d_x, a.weight = d_weight, a.bias = d_bias, a.stats = (float*)d_stats, a.ws = d_ws;
    norm_backward(a, d_dy, desc->ld_dy, desc->batch_dy, d_dx, d_dweight, d_dbias, (hipStream_t)stream);
    check_launches("group norm's backward pass");
  });
}

int srbcrs_linear_xent_workspace(const srbcrs_xent_desc* desc, const void* d_h, const void* d_weight, int32_t backward,
                                 size_t* bytes) {
  return guarded([&] {
    const XentArgs a = xent_args(desc, d_h, d_weight);
    check_ptr(bytes, "bytes");
    // any pointers: both gradients are wanted
    void* some = bytes;
    *bytes = !a.rows ? 1 : at_least_one(backward ? xent_backward(a, nullptr, some, some, nullptr) : xent_forward(a, nullptr, nullptr));
  });
}

int srbcrs_linear_xent(const srbcrs_xent_desc* desc, const void* d_h, const void* d_weight, const int64_t* d_target,
                       float* d_loss, float* d_state, void* d_ws, size_t ws_bytes, void* stream) {
  return guarded([&] {
    XentArgs a = xent_args(desc, d_h, d_weight);
    if (!a.rows) {
      if (a.reduction && d_loss) fill_zero(d_loss, sizeof(float), (hipStream_t)stream);
      return;
    }
    check_ptr(d_h, "h");
    check_ptr(d_weight, "weight");
    check_ptr(d_target, "target");
    check_ptr(d_loss, "loss");
    check_ptr(d_state, "state");
    if ((uintptr_t)d_state % 8) fail(SRBCRS_EINVAL, "state is not 8-byte aligned");
    check_aligned(d_h, a.dtype, "h");
    check_aligned(d_weight, a.dtype, "weight");
    check_ws(d_ws, ws_bytes, xent_forward(a, nullptr, nullptr));
    a.target = d_target, a.lse = d_state, a.count = d_state + 2 * a.rows, a.ws = d_ws;
    xent_forward(a, d_loss, (hipStream_t)stream);
    check_launches("linear cross entropy");
  });
}

int srbcrs_linear_xent_backward(const srbcrs_xent_desc* desc, const void* d_h, const void* d_weight,
                                const int64_t* d_target, const float* d_state, const float* d_dloss, void* d_dh,
                                void* d_dweight, void* d_ws, size_t ws_bytes, void* stream) {
  return guarded([&] {
    XentArgs a = xent_args(desc, d_h, d_weight);
    if (!d_dh && !d_dweight) return;
    if (!a.rows) {
      if (d_dweight)
        fill_zero(d_dweight, (size_t)a.classes * a.dim * dtype_size(a.dtype), (hipStream_t)stream);
      return;
    }
    check_ptr(d_h, "h");
    check_ptr(d_weight, "weight");
    check_ptr(d_target, "target");
    check_ptr(d_state, "state");
    if ((uintptr_t)d_state % 8) fail(SRBCRS_EINVAL, "state is not 8-byte aligned");
    check_ptr(d_dloss, "dloss");
    for (const void* p : {d_h, d_weight, (const void*)d_dh, (const void*)d_dweight}) check_aligned(p, a.dtype, "a matrix");
    check_ws(d_ws, ws_bytes, xent_backward(a, nullptr, d_dh, d_dweight, nullptr));
    a.target = d_target, a.lse = (float*)d_state, a.count = (float*)d_state + 2 * a.rows, a.ws = d_ws;
    xent_backward(a, d_dloss, d_dh, d_dweight, (hipStream_t)stream);
    check_launches("linear cross entropy's backward pass");
  });
}

int srbcrs_orthogonalize_workspace(const srbcrs_ortho_desc* desc, size_t* bytes) {
  return guarded([&] {
    const OrthoArgs a = ortho_args(desc);
    check_ptr(bytes, "bytes");
    *bytes = !a.batch || !a.rows || !a.cols ? 1 : at_least_one(ortho(a, nullptr));
  });
}

int srbcrs_orthogonalize(const srbcrs_ortho_desc* desc, const void* d_g, void* d_out, void* d_ws, size_t ws_bytes,
                         void* stream) {
  return guarded([&] {
    OrthoArgs a = ortho_args(desc);
    if (!a.batch || !a.rows || !a.cols) return;
    check_ptr(d_g, "g");
    check_ptr(d_out, "out");
    check_aligned(d_g, a.dtype, "g");
    check_aligned(d_out, a.dtype, "out");
    check_ws(d_ws, ws_bytes, ortho(a, nullptr));
    a.g = d_g, a.out = d_out, a.ws = d_ws;
    ortho(a, (hipStream_t)stream);
    check_launches("orthogonalised update");
  });
}

}  // extern "C"
