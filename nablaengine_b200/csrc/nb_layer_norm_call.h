// The layer norm's calls: arguments (checked by the C entries) and the launches, one set per value type of x
// (nb_layer_norm_f32.cu, _bf16.cu, _f16.cu).
#pragma once
#include <cuda_runtime.h>

namespace nbtrain {

struct LnForward {
  cudaStream_t stream;
  long long rows;
  int cols;
  long long stride;
  const void* x;
  int wtype;
  const void *weight, *bias;
  float eps;
  void* y;
  float *mean, *rstd;
};
struct LnBackward {
  cudaStream_t stream;
  long long rows;
  int cols;
  long long g_stride, stride;
  const void *g, *x;
  const float *mean, *rstd;
  int wtype;
  const void* weight;
  void *gx, *gw, *gb;
  float* part;  // ln_max_parts(rows, cols) x 2 x cols
};
template <class T> int ln_forward(const LnForward& a);
template <class T> int ln_backward(const LnBackward& a);
long long ln_max_parts(long long rows, int cols);

}  // namespace nbtrain
