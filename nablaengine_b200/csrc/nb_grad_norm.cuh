// The global norm of a list of tensors and the list times the clip coefficient:
//   S = sum g^2 over every value of every tensor, norm = sqrt(S), c = min(1, max_norm / (norm + eps)), out = c g
// S is summed in 64 bits, so neither a gradient of 1e30 overflows it nor one of 1e-30 vanishes from it, and in a fixed
// order (one partial sum per block, no atomics), so results repeat bit for bit. Non-finite values are counted; with
// `zero` they count as 0 in S and in out.
#pragma once
#include "nb_values.cuh"

namespace nbtrain {

constexpr int GN_THREADS = 256;
constexpr int GN_CHUNK = 8192;     // values of one tensor that a block takes at a time
constexpr int GN_MAX_BLOCKS = 1184;  // partial sums of a launch (8 blocks for each of the 148 SMs)
constexpr int GN_TENSORS = 96;     // tensors of one launch (their table travels as a kernel argument)

struct GradEntry {
  const void* in;
  void* out;
  long long n;
  int first;  // the tensor's first chunk in the launch
  short in_type, out_type;
};
struct GradTable {
  int count, chunks;
  GradEntry t[GN_TENSORS];
};

__device__ __forceinline__ float load_value(const void* p, int type, long long i) {
  if (type == BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  if (type == F16) return to_f32(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_value(void* p, int type, long long i, float v) {
  if (type == BF16) static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
  else if (type == F16) static_cast<__half*>(p)[i] = from_f32<__half>(v);
  else static_cast<float*>(p)[i] = v;
}

// The tensor of chunk `c`: the last one whose first chunk is at most c.
__device__ __forceinline__ int tensor_of_chunk(const GradTable& t, int c) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.t[mid].first <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A block's sum of a double per thread (the result at thread 0).
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double s[GN_THREADS / 32];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < GN_THREADS / 32; w++) v += s[w];
  return v;
}

// part[2 (base + block)] = the block's sum of squares, [.. + 1] = its non-finite values
__global__ void __launch_bounds__(GN_THREADS) k_grad_sumsq(const __grid_constant__ GradTable t, int zero, int base,
                                                           double* __restrict__ part) {
  double s = 0.0, bad = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const GradEntry& e = t.t[tensor_of_chunk(t, c)];
    const long long i0 = (long long)(c - e.first) * GN_CHUNK;
    const int n = (int)(e.n - i0 < GN_CHUNK ? e.n - i0 : GN_CHUNK);
    for (int i = threadIdx.x; i < n; i += GN_THREADS) {
      const float v = load_value(e.in, e.in_type, i0 + i);
      const bool finite = isfinite(v);
      if (!finite) bad += 1.0;
      if (finite || !zero) s = fma((double)v, (double)v, s);
    }
  }
  s = block_sum(s);
  bad = block_sum(bad);
  if (threadIdx.x == 0) {
    part[2 * (base + blockIdx.x)] = s;
    part[2 * (base + blockIdx.x) + 1] = bad;
  }
}

// stats = the partial sums' sums (one block)
__global__ void __launch_bounds__(GN_THREADS) k_grad_finish(int parts, const double* __restrict__ part,
                                                            double* __restrict__ stats) {
  double s = 0.0, bad = 0.0;
  for (int i = threadIdx.x; i < parts; i += GN_THREADS) {
    s += part[2 * i];
    bad += part[2 * i + 1];
  }
  s = block_sum(s);
  bad = block_sum(bad);
  if (threadIdx.x == 0) {
    stats[0] = s;
    stats[1] = bad;
  }
}

__device__ __forceinline__ float clip_coefficient(double sumsq, double max_norm, double eps) {
  const double d = sqrt(sumsq) + eps;
  return d <= max_norm ? 1.f : (float)(max_norm / d);  // (a NaN norm gives NaN, an infinite one 0)
}

__global__ void k_grad_result(const double* __restrict__ stats, float* __restrict__ norm, long long* __restrict__ bad) {
  if (norm) *norm = (float)sqrt(stats[0]);
  if (bad) *bad = (long long)stats[1];
}

__global__ void __launch_bounds__(GN_THREADS) k_grad_scale(const __grid_constant__ GradTable t,
                                                           const double* __restrict__ stats, double max_norm,
                                                           double eps, int zero) {
  const float coef = clip_coefficient(stats[0], max_norm, eps);
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const GradEntry& e = t.t[tensor_of_chunk(t, c)];
    const long long i0 = (long long)(c - e.first) * GN_CHUNK;
    const int n = (int)(e.n - i0 < GN_CHUNK ? e.n - i0 : GN_CHUNK);
    for (int i = threadIdx.x; i < n; i += GN_THREADS) {
      float v = load_value(e.in, e.in_type, i0 + i);
      if (zero && !isfinite(v)) v = 0.f;
      store_value(e.out, e.out_type, i0 + i, v * coef);
    }
  }
}

}  // namespace nbtrain
