// libnabla_g1: the operators that train a policy through the control step, behind the C ABI of include/nabla_g1.h:
// layer norm (nb_layer_norm.cuh) and the global gradient norm with clipping (nb_grad_norm.cuh).
#include "../../include/nabla_g1.h"
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>
#include <new>
#include "nb_grad_norm.cuh"
#include "nb_launch.h"
#include "nb_layer_norm_call.h"

using namespace nbtrain;

namespace {

// ---- arguments ------------------------------------------------------------------------------------------------------
constexpr long long LONGEST = 1ll << 40;  // values of a tensor: more than any GPU holds

bool ln_size_ok(long long rows, long long cols) {
  return rows >= 0 && cols >= 1 && cols <= INT_MAX / 4 && rows <= LONGEST / cols;
}
bool ln_stride_ok(long long rows, long long stride) {
  return stride >= 0 && stride <= LONGEST / std::max(rows, 1ll);
}
bool ln_types_ok(int dtype, int wtype) { return dtype_ok(dtype) && (wtype == F32 || wtype == dtype); }

bool aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % dtype_bytes(dtype) == 0; }

// ---- the gradient list ----------------------------------------------------------------------------------------------
bool grads_ok(int count, const void* const* in, const long long* sizes, const int* types) {
  if (count < 0) return false;
  if (count == 0) return true;
  if (!in || !sizes || !types) return false;
  for (int i = 0; i < count; i++)
    if (sizes[i] < 0 || sizes[i] > LONGEST || !dtype_ok(types[i]) ||
        (sizes[i] && (!in[i] || !aligned(in[i], types[i]))))
      return false;
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

int grad_launches(int count) { return (count + GN_MANY - 1) / GN_MANY; }

// The table of the tensors from i0 on, as many as it takes; returns its launch's blocks.
template <int N>
int fill_table(GradTable<N>& t, int i0, int count, const void* const* in, void* const* out, const long long* sizes,
               const int* types, const int* out_types, int shortest = 2048, int takers = GN_BLOCKS) {
  const int i1 = std::min(count, i0 + N);
  long long total = 0, chunks = 0;
  for (int i = i0; i < i1; i++) total += sizes[i];
  // chunks of `shortest` to 16384 values: about one for each block (or warp) that takes them where there are few
  t.chunk = shortest;
  while (t.chunk < 16384 && total > (long long)t.chunk * takers) t.chunk *= 2;
  t.count = 0;
  for (int i = i0; i < i1; i++) {
    if (sizes[i] == 0) continue;
    GradEntry& e = t.t[t.count++];
    const int es = dtype_bytes(types[i]);
    const uintptr_t a = reinterpret_cast<uintptr_t>(in[i]);
    e.in = in[i];
    e.out = out ? out[i] : nullptr;
    e.n = sizes[i];
    e.first = (int)chunks;
    e.in_type = (unsigned char)types[i];
    e.out_type = (unsigned char)(out ? out_types[i] : types[i]);
    e.lead = (unsigned char)((16 - a % 16) % 16 / es);
    const int os = dtype_bytes(e.out_type);
    e.vectors = (reinterpret_cast<uintptr_t>(e.out) + (uintptr_t)e.lead * os) % std::min(16, 16 / es * os) == 0;
    chunks += std::max<long long>(1, (sizes[i] - e.lead + t.chunk - 1) / t.chunk);
    if (chunks > INT_MAX / 2) return -1;
  }
  t.chunks = (int)chunks;
  return (int)std::min<long long>(chunks, GN_BLOCKS);
}

struct GradList {
  int count;
  const void* const* in;
  void* const* out;
  const long long* sizes;
  const int *types, *out_types;
  int zero;
};

// The partial sums of the list into `part`; sets their number.
template <int N> int grad_sumsq(cudaStream_t stream, const GradList& g, double2* part, int* parts) {
  GradTable<N> t;
  *parts = 0;
  for (int i0 = 0; i0 < g.count; i0 += N) {
    const int blocks = fill_table(t, i0, g.count, g.in, nullptr, g.sizes, g.types, nullptr);
    if (blocks < 0) return cudaErrorInvalidValue;
    if (!blocks) continue;
    const int e = launch_after({stream, blocks, GN_THREADS}, k_grad_sumsq<N>, t, g.zero, *parts, part);
    if (e) return e;
    *parts += blocks;
  }
  return 0;
}
int grad_sumsq(cudaStream_t stream, const GradList& g, double2* part, int* parts) {
  return g.count <= GN_FEW ? grad_sumsq<GN_FEW>(stream, g, part, parts) : grad_sumsq<GN_MANY>(stream, g, part, parts);
}

// Every tensor times its coefficient, and the results, from the partial sums.
template <int N>
int grad_scale(cudaStream_t stream, const GradList& g, int parts, const double2* part, double max_norm, double eps,
               float* norm, long long* bad) {
  GradTable<N> t;
  bool first = true;
  for (int i0 = 0; g.out && i0 < g.count; i0 += N) {
    const int blocks = fill_table(t, i0, g.count, g.in, g.out, g.sizes, g.types, g.out_types);
    if (blocks < 0) return cudaErrorInvalidValue;
    if (!blocks) continue;
    const int e = launch_after({stream, blocks, GN_THREADS}, k_grad_scale<N>, t, parts, part, max_norm, eps, g.zero,
                               first ? norm : nullptr, first ? bad : nullptr);
    if (e) return e;
    first = false;
  }
  if (!first || (!norm && !bad)) return 0;
  return launch_after({stream, 1, GN_THREADS}, k_grad_finish, parts, part, nullptr, norm, bad);
}
int grad_scale(cudaStream_t stream, const GradList& g, int parts, const double2* part, double max_norm, double eps,
               float* norm, long long* bad) {
  return g.count <= GN_FEW ? grad_scale<GN_FEW>(stream, g, parts, part, max_norm, eps, norm, bad)
                           : grad_scale<GN_MANY>(stream, g, parts, part, max_norm, eps, norm, bad);
}

// A list that one cluster takes in one launch (measured: see k_grad_small).
bool grad_small(int count, const long long* sizes) {
  if (count > NB_G1_GRAD_SMALL_TENSORS) return false;
  long long total = 0;
  for (int i = 0; i < count; i++) total += sizes[i];
  return total <= NB_G1_GRAD_SMALL_VALUES;
}
template <int BLOCKS>
int grad_clip_small(cudaStream_t stream, const GradList& g, double max_norm, double eps, float* norm, long long* bad) {
  GradTable<GN_FEW> t;
  if (fill_table(t, 0, g.count, g.in, g.out, g.sizes, g.types, g.out_types, 512, BLOCKS * GN_SMALL_THREADS / 32) < 0)
    return cudaErrorInvalidValue;
  return launch_after({stream, BLOCKS, GN_SMALL_THREADS, 0, BLOCKS}, k_grad_small<BLOCKS>, t, g.out ? 1 : 0, max_norm,
                      eps, g.zero, norm, bad);
}
// Whether the current device holds a cluster of 16 blocks of k_grad_small (8 is what every device does), asked once.
bool cluster_of_16() {
  static std::atomic<int> known[64];  // 0: not asked, 1: no, 2: yes
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  int k = known[dev].load(std::memory_order_relaxed);
  if (k == 0) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 16, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(16);
    config.blockDim = dim3(GN_SMALL_THREADS);
    config.attrs = &attr;
    config.numAttrs = 1;
    int n = 0;
    const bool yes =
        cudaFuncSetAttribute(k_grad_small<16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&n, k_grad_small<16>, &config) == cudaSuccess && n > 0;
    if (!yes) (void)cudaGetLastError();
    k = yes ? 2 : 1;
    known[dev].store(k, std::memory_order_relaxed);
  }
  return k == 2;
}
static_assert(NB_G1_GRAD_SMALL_TENSORS <= GN_FEW, "a short list is one table");

bool limits_ok(double max_norm, double eps) { return max_norm >= 0 && eps >= 0 && std::isfinite(eps); }
bool results_ok(const float* norm, const long long* bad) {
  return aligned(norm, F32) && reinterpret_cast<uintptr_t>(bad) % 8 == 0;
}

}  // namespace

extern "C" {

long long nb_g1_layer_norm_work_bytes(long long rows, long long cols) {
  if (!ln_size_ok(rows, cols)) return -1;
  return ln_max_parts(rows, (int)cols) * 2 * cols * 4;
}

int nb_g1_layer_norm_forward(cudaStream_t stream, long long rows, long long cols, long long stride, int dtype,
                             const void* x, int wtype, const void* weight, const void* bias, float eps, void* y,
                             float* mean, float* rstd) {
  if (!ln_size_ok(rows, cols) || !ln_stride_ok(rows, stride) || !ln_types_ok(dtype, wtype) || !(eps >= 0.f) ||
      !std::isfinite(eps))
    return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  if (!x || !y || !mean || !rstd || !aligned(x, dtype) || !aligned(y, dtype) || !aligned(weight, wtype) ||
      !aligned(bias, wtype) || !aligned(mean, F32) || !aligned(rstd, F32))
    return (int)cudaErrorInvalidValue;
  const LnForward a = {stream, rows, (int)cols, stride, x, wtype, weight, bias, eps, y, mean, rstd};
  return dtype == F32 ? ln_forward<float>(a) : dtype == BF16 ? ln_forward<__nv_bfloat16>(a) : ln_forward<__half>(a);
}

int nb_g1_layer_norm_backward(cudaStream_t stream, long long rows, long long cols, long long g_stride,
                              long long stride, int dtype, const void* g_y, const void* x, const float* mean,
                              const float* rstd, int wtype, const void* weight, void* g_x, void* g_weight,
                              void* g_bias, void* work) {
  if (!ln_size_ok(rows, cols) || !ln_stride_ok(rows, stride) || !ln_stride_ok(rows, g_stride) ||
      !ln_types_ok(dtype, wtype))
    return (int)cudaErrorInvalidValue;
  if ((rows && (!g_y || !x || !mean || !rstd)) || !aligned(g_y, dtype) || !aligned(x, dtype) ||
      !aligned(g_x, dtype) || !aligned(weight, wtype) || !aligned(g_weight, wtype) || !aligned(g_bias, wtype) ||
      !aligned(mean, F32) || !aligned(rstd, F32))
    return (int)cudaErrorInvalidValue;
  if ((g_weight || g_bias) && ((rows && !work) || reinterpret_cast<uintptr_t>(work) % 16))
    return (int)cudaErrorInvalidValue;
  const LnBackward a = {stream, rows, (int)cols, g_stride, stride, g_y, x, mean, rstd,
                        wtype, weight, g_x, g_weight, g_bias, static_cast<float*>(work)};
  return dtype == F32 ? ln_backward<float>(a) : dtype == BF16 ? ln_backward<__nv_bfloat16>(a)
                                                              : ln_backward<__half>(a);
}

long long nb_g1_grad_work_bytes(int count) {
  if (count < 0) return -1;
  return 16ll * GN_BLOCKS * std::max(1, grad_launches(count));
}

int nb_g1_grad_sumsq(cudaStream_t stream, int count, const void* const* grads, const long long* sizes,
                     const int* types, int zero_nonfinite, void* work, double* stats) {
  if (!grads_ok(count, grads, sizes, types) || !work || !stats || reinterpret_cast<uintptr_t>(work) % 16 ||
      reinterpret_cast<uintptr_t>(stats) % 16)
    return (int)cudaErrorInvalidValue;
  double2* part = static_cast<double2*>(work);
  int parts = 0;
  const int e = grad_sumsq(stream, {count, grads, nullptr, sizes, types, nullptr, zero_nonfinite}, part, &parts);
  if (e) return e;
  return launch_after({stream, 1, GN_THREADS}, k_grad_finish, parts, part, reinterpret_cast<double2*>(stats), nullptr,
                      nullptr);
}

int nb_g1_grad_scale(cudaStream_t stream, int count, const void* const* grads, void* const* outs,
                     const long long* sizes, const int* types, const int* out_types, int zero_nonfinite,
                     double max_norm, double eps, const double* stats, float* norm, long long* bad) {
  if (!grads_ok(count, grads, sizes, types) || !stats || reinterpret_cast<uintptr_t>(stats) % 16 ||
      !limits_ok(max_norm, eps) || !results_ok(norm, bad))
    return (int)cudaErrorInvalidValue;
  if (outs) {
    const int e = outs_error(count, grads, outs, sizes, types, out_types);
    if (e) return e;
  }
  return grad_scale(stream, {count, grads, outs, sizes, types, out_types, zero_nonfinite}, 1,
                    reinterpret_cast<const double2*>(stats), max_norm, eps, norm, bad);
}

int nb_g1_grad_clip(cudaStream_t stream, int count, const void* const* grads, void* const* outs,
                    const long long* sizes, const int* types, const int* out_types, int zero_nonfinite,
                    double max_norm, double eps, void* work, float* norm, long long* bad) {
  if (!grads_ok(count, grads, sizes, types) || !limits_ok(max_norm, eps) || !results_ok(norm, bad))
    return (int)cudaErrorInvalidValue;
  const bool small = grad_small(count, sizes);
  if (!small && (!work || reinterpret_cast<uintptr_t>(work) % 16)) return (int)cudaErrorInvalidValue;
  if (outs) {
    const int e = outs_error(count, grads, outs, sizes, types, out_types);
    if (e) return e;
  }
  const GradList g = {count, grads, outs, sizes, types, out_types, zero_nonfinite};
  if (small) {
    const auto clip = cluster_of_16() ? grad_clip_small<16> : grad_clip_small<8>;
    return clip(stream, g, max_norm, eps, norm, bad);
  }
  double2* part = static_cast<double2*>(work);
  int parts = 0;
  const int e = grad_sumsq(stream, g, part, &parts);
  return e ? e : grad_scale(stream, g, parts, part, max_norm, eps, norm, bad);
}

}  // extern "C"
