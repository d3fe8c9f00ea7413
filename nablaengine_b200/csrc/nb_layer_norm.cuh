// Layer norm over the last dimension (N columns, M rows), forward and backward.
//   mean = sum x / N, var = sum (x - mean)^2 / N, rstd = (var + eps)^(-1/2), xh = (x - mean) rstd, y = xh w + b
//   h = g w, c1 = sum h / N, c2 = sum h xh / N, gx = rstd (h - c1 - xh c2), gw = sum_rows g xh, gb = sum_rows g
// Sums are float32; the variance is taken from the deviations (a second pass), not from sum x^2.
#pragma once
#include "nb_values.cuh"

namespace nbtrain {

constexpr int LN_WARPS = 8;     // warps (rows) per block
constexpr int LN_PARTS = 256;   // partial column sums at most

// One warp per row, the row read three times (mean, variance, result).
template <class T, class W>
__global__ void __launch_bounds__(LN_WARPS * 32) k_ln_forward(long long rows, int cols, long long stride,
                                                              const T* __restrict__ x, const W* __restrict__ weight,
                                                              const W* __restrict__ bias, float eps,
                                                              T* __restrict__ y, float* __restrict__ mean_out,
                                                              float* __restrict__ rstd_out) {
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * LN_WARPS + (threadIdx.x >> 5);
  if (row >= rows) return;
  const T* xr = x + row * stride;
  float s = 0.f;
  for (int c = lane; c < cols; c += 32) s += to_f32(xr[c]);
  const float mean = warp_sum(s) / cols;
  s = 0.f;
  for (int c = lane; c < cols; c += 32) {
    const float d = to_f32(xr[c]) - mean;
    s = fmaf(d, d, s);
  }
  const float rstd = 1.f / sqrtf(warp_sum(s) / cols + eps);
  for (int c = lane; c < cols; c += 32) {
    float v = (to_f32(xr[c]) - mean) * rstd;
    if (weight) v *= to_f32(weight[c]);
    if (bias) v += to_f32(bias[c]);
    y[row * cols + c] = from_f32<T>(v);
  }
  if (lane == 0) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
}

// The input's gradient: one warp per row.
template <class T, class W>
__global__ void __launch_bounds__(LN_WARPS * 32) k_ln_backward_x(long long rows, int cols, long long gstride,
                                                                 long long stride, const T* __restrict__ g,
                                                                 const T* __restrict__ x,
                                                                 const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd,
                                                                 const W* __restrict__ weight, T* __restrict__ gx) {
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * LN_WARPS + (threadIdx.x >> 5);
  if (row >= rows) return;
  const T *xr = x + row * stride, *gr = g + row * gstride;
  const float m = mean[row], r = rstd[row];
  float c1 = 0.f, c2 = 0.f;
  for (int c = lane; c < cols; c += 32) {
    const float h = to_f32(gr[c]) * (weight ? to_f32(weight[c]) : 1.f);
    c1 += h;
    c2 = fmaf(h, (to_f32(xr[c]) - m) * r, c2);
  }
  c1 = warp_sum(c1) / cols;
  c2 = warp_sum(c2) / cols;
  for (int c = lane; c < cols; c += 32) {
    const float h = to_f32(gr[c]) * (weight ? to_f32(weight[c]) : 1.f);
    gx[row * cols + c] = from_f32<T>((h - c1 - (to_f32(xr[c]) - m) * r * c2) * r);
  }
}

// Column sums of g xh and g over part_rows rows per block row, one thread per column: part (parts, 2, cols).
template <class T>
__global__ void __launch_bounds__(128) k_ln_backward_part(long long rows, int cols, long long gstride,
                                                          long long stride, const T* __restrict__ g,
                                                          const T* __restrict__ x, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, long long part_rows,
                                                          float* __restrict__ part) {
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= cols) return;
  const long long r0 = blockIdx.y * part_rows, r1 = r0 + part_rows < rows ? r0 + part_rows : rows;
  float gw = 0.f, gb = 0.f;
  for (long long r = r0; r < r1; r++) {
    const float gv = to_f32(g[r * gstride + c]);
    gw = fmaf(gv, (to_f32(x[r * stride + c]) - mean[r]) * rstd[r], gw);
    gb += gv;
  }
  part[((long long)blockIdx.y * 2 + 0) * cols + c] = gw;
  part[((long long)blockIdx.y * 2 + 1) * cols + c] = gb;
}

template <class W>
__global__ void __launch_bounds__(128) k_ln_backward_sum(int parts, int cols, const float* __restrict__ part,
                                                         W* __restrict__ gw, W* __restrict__ gb) {
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= cols) return;
  float w = 0.f, b = 0.f;
  for (int p = 0; p < parts; p++) {
    w += part[((long long)p * 2 + 0) * cols + c];
    b += part[((long long)p * 2 + 1) * cols + c];
  }
  if (gw) gw[c] = from_f32<W>(w);
  if (gb) gb[c] = from_f32<W>(b);
}

}  // namespace nbtrain
