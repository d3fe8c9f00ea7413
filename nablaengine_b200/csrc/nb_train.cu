// libnabla_g1: the operators that train a policy through the control step, behind the C ABI of include/nabla_g1.h:
// layer norm (nb_layer_norm.cuh) and the global gradient norm with clipping (nb_grad_norm.cuh).
#include "../../include/nabla_g1.h"
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <new>
#include "nb_grad_norm.cuh"
#include "nb_layer_norm_call.h"

using namespace nbtrain;

namespace {

// ---- arguments ------------------------------------------------------------------------------------------------------
bool ln_args_ok(long long rows, long long cols, long long stride, int dtype, int wtype) {
  return rows >= 0 && cols >= 1 && cols <= INT_MAX / 4 && stride >= 0 && dtype_ok(dtype) &&
         (wtype == F32 || wtype == dtype);
}

bool aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % dtype_bytes(dtype) == 0; }

// ---- the gradient list ----------------------------------------------------------------------------------------------
bool grads_ok(int count, const void* const* in, const long long* sizes, const int* types) {
  if (count < 0) return false;
  if (count == 0) return true;
  if (!in || !sizes || !types) return false;
  for (int i = 0; i < count; i++)
    if (sizes[i] < 0 || !dtype_ok(types[i]) || (sizes[i] && (!in[i] || !aligned(in[i], types[i])))) return false;
  return true;
}

struct Span {
  uintptr_t lo, hi;
  bool written;
};

// The outputs are valid and none overlaps another output or another tensor's input; an output may be its own tensor's
// input (the same address and type: the tensor is scaled in place).
int outs_error(int count, const void* const* in, void* const* out, const long long* sizes, const int* types,
               const int* out_types) {
  if (count == 0) return cudaSuccess;
  if (!out_types) return cudaErrorInvalidValue;
  Span* spans = new (std::nothrow) Span[2 * (size_t)count];
  if (!spans) return cudaErrorMemoryAllocation;
  int n = 0, err = cudaSuccess;
  for (int i = 0; i < count && !err; i++) {
    if (!dtype_ok(out_types[i])) err = cudaErrorInvalidValue;
    if (err || sizes[i] == 0) continue;
    if (!out[i] || !aligned(out[i], out_types[i])) err = cudaErrorInvalidValue;
    const uintptr_t a = reinterpret_cast<uintptr_t>(in[i]), b = reinterpret_cast<uintptr_t>(out[i]);
    spans[n++] = {b, b + (uintptr_t)sizes[i] * dtype_bytes(out_types[i]), true};
    if (a != b || types[i] != out_types[i]) spans[n++] = {a, a + (uintptr_t)sizes[i] * dtype_bytes(types[i]), false};
  }
  std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.lo < b.lo; });
  uintptr_t written = 0, any = 0;
  for (int i = 0; i < n && !err; i++) {
    if (spans[i].lo < (spans[i].written ? any : written)) err = cudaErrorInvalidValue;
    any = std::max(any, spans[i].hi);
    if (spans[i].written) written = std::max(written, spans[i].hi);
  }
  delete[] spans;
  return err;
}

int grad_launches(int count) { return (count + GN_TENSORS - 1) / GN_TENSORS; }

// The table of tensors [i0, i0 + GN_TENSORS) and its launch's blocks.
int fill_table(GradTable& t, int i0, int count, const void* const* in, void* const* out, const long long* sizes,
               const int* types, const int* out_types) {
  t.count = 0;
  long long chunks = 0;
  for (int i = i0; i < count && i < i0 + GN_TENSORS; i++) {
    if (sizes[i] == 0) continue;
    GradEntry& e = t.t[t.count++];
    e = {in[i],       out ? out[i] : nullptr, sizes[i],
         (int)chunks, (short)types[i],        (short)(out ? out_types[i] : types[i])};
    chunks += (sizes[i] + GN_CHUNK - 1) / GN_CHUNK;
    if (chunks > INT_MAX / 2) return -1;
  }
  t.chunks = (int)chunks;
  return (int)std::min<long long>(chunks, GN_MAX_BLOCKS);
}

int grad_sumsq(cudaStream_t stream, int count, const void* const* grads, const long long* sizes, const int* types,
               int zero, double* part, double* stats) {
  GradTable t;
  int parts = 0;
  for (int i0 = 0; i0 < count; i0 += GN_TENSORS) {
    const int blocks = fill_table(t, i0, count, grads, nullptr, sizes, types, nullptr);
    if (blocks < 0) return cudaErrorInvalidValue;
    if (!blocks) continue;
    k_grad_sumsq<<<blocks, GN_THREADS, 0, stream>>>(t, zero, parts, part);
    parts += blocks;
  }
  k_grad_finish<<<1, GN_THREADS, 0, stream>>>(parts, part, stats);
  return (int)cudaGetLastError();
}

int grad_scale(cudaStream_t stream, int count, const void* const* grads, void* const* outs, const long long* sizes,
               const int* types, const int* out_types, int zero, double max_norm, double eps, const double* stats,
               float* norm, long long* bad) {
  GradTable t;
  if (outs)
    for (int i0 = 0; i0 < count; i0 += GN_TENSORS) {
      const int blocks = fill_table(t, i0, count, grads, outs, sizes, types, out_types);
      if (blocks < 0) return cudaErrorInvalidValue;
      if (blocks) k_grad_scale<<<blocks, GN_THREADS, 0, stream>>>(t, stats, max_norm, eps, zero);
    }
  if (norm || bad) k_grad_result<<<1, 1, 0, stream>>>(stats, norm, bad);
  return (int)cudaGetLastError();
}

}  // namespace

extern "C" {

long long nb_g1_layer_norm_work_bytes(long long rows, long long cols) {
  if (rows < 0 || cols < 1 || cols > INT_MAX / 4) return -1;
  return ln_max_parts(rows, (int)cols) * 2 * cols * 4;
}

int nb_g1_layer_norm_forward(cudaStream_t stream, long long rows, long long cols, long long stride, int dtype,
                             const void* x, int wtype, const void* weight, const void* bias, float eps, void* y,
                             float* mean, float* rstd) {
  if (!ln_args_ok(rows, cols, stride, dtype, wtype) || !(eps >= 0.f) || !std::isfinite(eps))
    return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  if (!x || !y || !mean || !rstd || !aligned(x, dtype) || !aligned(y, dtype) || !aligned(weight, wtype) ||
      !aligned(bias, wtype))
    return (int)cudaErrorInvalidValue;
  const LnForward a = {stream, rows, (int)cols, stride, x, wtype, weight, bias, eps, y, mean, rstd};
  return dtype == F32 ? ln_forward<float>(a) : dtype == BF16 ? ln_forward<__nv_bfloat16>(a) : ln_forward<__half>(a);
}

int nb_g1_layer_norm_backward(cudaStream_t stream, long long rows, long long cols, long long g_stride,
                              long long stride, int dtype, const void* g_y, const void* x, const float* mean,
                              const float* rstd, int wtype, const void* weight, void* g_x, void* g_weight,
                              void* g_bias, void* work) {
  if (!ln_args_ok(rows, cols, stride, dtype, wtype) || g_stride < 0) return (int)cudaErrorInvalidValue;
  if ((rows && (!g_y || !x || !mean || !rstd)) || !aligned(g_y, dtype) || !aligned(x, dtype) ||
      !aligned(g_x, dtype) || !aligned(weight, wtype) || !aligned(g_weight, wtype) || !aligned(g_bias, wtype))
    return (int)cudaErrorInvalidValue;
  if (rows && (g_weight || g_bias) && !work) return (int)cudaErrorInvalidValue;
  const LnBackward a = {stream, rows, (int)cols, g_stride, stride, g_y, x, mean, rstd,
                        wtype, weight, g_x, g_weight, g_bias, static_cast<float*>(work)};
  return dtype == F32 ? ln_backward<float>(a) : dtype == BF16 ? ln_backward<__nv_bfloat16>(a)
                                                              : ln_backward<__half>(a);
}

long long nb_g1_grad_work_bytes(int count) {
  if (count < 0) return -1;
  return 16ll + 16ll * GN_MAX_BLOCKS * grad_launches(count);
}

int nb_g1_grad_sumsq(cudaStream_t stream, int count, const void* const* grads, const long long* sizes,
                     const int* types, int zero_nonfinite, void* work, double* stats) {
  if (!grads_ok(count, grads, sizes, types) || !work || !stats) return (int)cudaErrorInvalidValue;
  return grad_sumsq(stream, count, grads, sizes, types, zero_nonfinite, static_cast<double*>(work) + 2, stats);
}

int nb_g1_grad_scale(cudaStream_t stream, int count, const void* const* grads, void* const* outs,
                     const long long* sizes, const int* types, const int* out_types, int zero_nonfinite,
                     double max_norm, double eps, const double* stats, float* norm, long long* bad) {
  if (!grads_ok(count, grads, sizes, types) || !stats || std::isnan(max_norm) || max_norm < 0 || std::isnan(eps) ||
      eps < 0)
    return (int)cudaErrorInvalidValue;
  if (outs) {
    const int e = outs_error(count, grads, outs, sizes, types, out_types);
    if (e) return e;
  }
  return grad_scale(stream, count, grads, outs, sizes, types, out_types, zero_nonfinite, max_norm, eps, stats, norm,
                    bad);
}

int nb_g1_grad_clip(cudaStream_t stream, int count, const void* const* grads, void* const* outs,
                    const long long* sizes, const int* types, const int* out_types, int zero_nonfinite,
                    double max_norm, double eps, void* work, float* norm, long long* bad) {
  if (!grads_ok(count, grads, sizes, types) || !work || std::isnan(max_norm) || max_norm < 0 || std::isnan(eps) ||
      eps < 0)
    return (int)cudaErrorInvalidValue;
  if (outs) {
    const int e = outs_error(count, grads, outs, sizes, types, out_types);
    if (e) return e;
  }
  double* stats = static_cast<double*>(work);
  const int e = grad_sumsq(stream, count, grads, sizes, types, zero_nonfinite, stats + 2, stats);
  if (e) return e;
  return grad_scale(stream, count, grads, outs, sizes, types, out_types, zero_nonfinite, max_norm, eps, stats, norm,
                    bad);
}

}  // extern "C"
