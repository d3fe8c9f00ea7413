// The global norm of a list of tensors and the list times the clip coefficient:
//   S = sum g^2 over every value of every tensor, norm = sqrt(S), out = c g,
//   c = 1 where norm + eps <= max_norm, else max_norm / (norm + eps)
// Non-finite values are counted; with `zero` they count as 0 in S and in out.
//
// S is held in 64 bits, so neither a gradient of 1e30 overflows it nor one of 1e-30 vanishes from it. Eight squares at
// a time are summed in float32 first; where that sum is not between 2^-100 and the largest float (an overflow, values
// that vanish, a non-finite one) the eight are taken again one by one in 64 bits. Every block writes one partial sum
// and the next kernel's blocks add them all up, each for itself, in the same order: no atomics, the same bits every
// time.
//
// Both passes are bound by memory. The tensors are cut into chunks that the blocks take in turn, in the first pass from
// the first chunk on and in the second from the last one back, so that the second finds in the second-level cache
// what the first read last (30.4M float32 values: 22 us, 5.5 TB/s, and 34 us, in which 54 MB are read from DRAM, 68 MB
// from the cache, and 122 MB written: 5.2 TB/s of DRAM's 6.55; a fill of 122 MB takes 22.5 us, so the writes alone do
// not bound it, but keeping 28 MB more on the chip changed nothing). 100M bfloat16 values: 98 us.
#pragma once
#include <cstdint>
#include "nb_values.cuh"

namespace nbtrain {

constexpr int GN_THREADS = 256;
constexpr int GN_BLOCKS = 8 * SMS;  // blocks of a launch at most, and its partial sums
constexpr int GN_FEW = 96, GN_MANY = 960;  // tensors of one launch (their table travels as a kernel argument)
constexpr int GN_UNROLL = 8;  // 16-byte loads in flight per thread
constexpr int GN_SMALL_THREADS = 512;  // of a block of k_grad_small

// One tensor: its values from the first 16-byte boundary on (`lead` values in) are cut into chunks.
struct GradEntry {
  const void* in;
  void* out;
  long long n;
  int first;  // the tensor's first chunk in the launch
  unsigned char in_type, out_type, lead, vectors;  // vectors: out takes whole pieces where in gives them
};
template <int N> struct GradTable {
  int count, chunks, chunk;  // chunk: values of a chunk
  GradEntry t[N];
};

// The values [first, first + n) of the tensor `e` that chunk c of a table is, without the lead.
struct GradPart {
  long long first;
  int n;
};
template <int N> __device__ __forceinline__ GradPart grad_part(const GradTable<N>& t, const GradEntry& e, int c) {
  const long long first = e.lead + (long long)(c - e.first) * t.chunk, left = e.n - first;
  return {first, (int)(left < t.chunk ? left : t.chunk)};
}

__device__ __forceinline__ void add_value(float v, int zero, double& s, double& bad) {
  const bool finite = isfinite(v);
  if (!finite) bad += 1.0;
  if (finite || !zero) s = fma((double)v, (double)v, s);
}
// eight values (four pairs)
__device__ __forceinline__ void add_eight(const float2* v, int zero, double& s, double& bad) {
  float2 q = mul2(v[0], v[0]);
  q = fma2(v[1], v[1], q);
  q = fma2(v[2], v[2], q);
  q = fma2(v[3], v[3], q);
  const float sum = q.x + q.y;
  if (sum >= 0x1p-100f && sum <= 3.4e38f) {
    s += (double)sum;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      add_value(v[i].x, zero, s, bad);
      add_value(v[i].y, zero, s, bad);
    }
  }
}

template <class T> __device__ __forceinline__ void unpack_piece(uint4 u, float2* v) {
  if constexpr (sizeof(T) == 4) {
    v[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    v[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  } else {
    v[0] = unpack2<T>(u.x), v[1] = unpack2<T>(u.y), v[2] = unpack2<T>(u.z), v[3] = unpack2<T>(u.w);
  }
}

// (tid of THREADS: the threads that share the part)
template <int THREADS, class T>
__device__ __forceinline__ void sumsq_part(const GradEntry& e, GradPart part, int tid, int zero, double& s,
                                           double& bad) {
  constexpr int P = 16 / sizeof(T), STEP = THREADS * GN_UNROLL;
  const T* base = static_cast<const T*>(e.in);
  if (part.first == e.lead)
    for (int i = tid; i < min((long long)e.lead, e.n); i += THREADS)
      add_value(to_f32(base[i]), zero, s, bad);
  if (part.n <= 0) return;
  const uint4* from = reinterpret_cast<const uint4*>(base + part.first);
  const int pieces = part.n / P;
  int i = tid;
  for (; i + STEP - THREADS < pieces; i += STEP) {
    uint4 u[GN_UNROLL];
#pragma unroll
    for (int k = 0; k < GN_UNROLL; k++) u[k] = from[i + k * THREADS];
#pragma unroll
    for (int k = 0; k < GN_UNROLL; k += P == 4 ? 2 : 1) {
      float2 v[4];
      unpack_piece<T>(u[k], v);
      if constexpr (P == 4) unpack_piece<T>(u[k + 1], v + 2);
      add_eight(v, zero, s, bad);
    }
  }
  for (; i < pieces; i += THREADS) {
    float2 v[4] = {both(0.f), both(0.f), both(0.f), both(0.f)};
    unpack_piece<T>(from[i], v);
    add_eight(v, zero, s, bad);
  }
  for (int k = pieces * P + tid; k < part.n; k += THREADS)
    add_value(to_f32(base[part.first + k]), zero, s, bad);
}

template <int THREADS>
__device__ __forceinline__ void sumsq_part(const GradEntry& e, GradPart p, int tid, int zero, double& s, double& bad) {
  if (e.in_type == F32) sumsq_part<THREADS, float>(e, p, tid, zero, s, bad);
  else if (e.in_type == BF16) sumsq_part<THREADS, __nv_bfloat16>(e, p, tid, zero, s, bad);
  else sumsq_part<THREADS, __half>(e, p, tid, zero, s, bad);
}

// Sums over the block of a double per thread (the result at thread 0).
__device__ __forceinline__ double2 block_sum(double2 v) {
  __shared__ double2 s[GN_THREADS / 32];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, m);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, m);
  }
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < GN_THREADS / 32; w++) v.x += s[w].x, v.y += s[w].y;
  return v;
}

// part[base + block] = the block's sum of squares and its non-finite values
template <int N>
__global__ void __launch_bounds__(GN_THREADS) k_grad_sumsq(const __grid_constant__ GradTable<N> t, int zero, int base,
                                                           double2* __restrict__ part) {
  let_next_start();
  wait_for_last();
  double s = 0.0, bad = 0.0;
  int i = 0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    while (i + 1 < t.count && t.t[i + 1].first <= c) i++;
    const GradEntry& e = t.t[i];
    sumsq_part<GN_THREADS>(e, grad_part(t, e, c), threadIdx.x, zero, s, bad);
  }
  const double2 r = block_sum(make_double2(s, bad));
  if (threadIdx.x == 0) part[base + blockIdx.x] = r;
}

// The sum of all partial sums, for every thread of the block.
__device__ __forceinline__ double2 sum_parts(int parts, const double2* part) {
  __shared__ double2 total;
  double2 v = make_double2(0.0, 0.0);
  for (int i = threadIdx.x; i < parts; i += GN_THREADS) v.x += part[i].x, v.y += part[i].y;
  v = block_sum(v);
  if (threadIdx.x == 0) total = v;
  __syncthreads();
  return total;
}

// The results alone (one block), each where wanted.
__global__ void __launch_bounds__(GN_THREADS) k_grad_finish(int parts, const double2* __restrict__ part,
                                                            double2* __restrict__ stats, float* __restrict__ norm,
                                                            long long* __restrict__ bad) {
  let_next_start();
  wait_for_last();
  const double2 v = sum_parts(parts, part);
  if (threadIdx.x) return;
  if (stats) *stats = v;
  if (norm) *norm = (float)sqrt(v.x);
  if (bad) *bad = (long long)v.y;
}

__device__ __forceinline__ double clip_coefficient(double sumsq, double max_norm, double eps) {
  const double d = sqrt(sumsq) + eps;
  return d <= max_norm ? 1.0 : max_norm / d;  // (a NaN norm gives NaN, an infinite one 0)
}

// c v; where non-finite values count as 0 and there are any, those are 0
__device__ __forceinline__ float clip_value(float v, float c, bool clean) {
  return clean && !isfinite(v) ? 0.f : v * c;
}

template <class O, int P> __device__ __forceinline__ void store_piece(O* p, const float2* v) {
  if constexpr (P * sizeof(O) == 32) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0].x, v[0].y, v[1].x, v[1].y));
    __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(v[2].x, v[2].y, v[3].x, v[3].y));
  } else if constexpr (sizeof(O) == 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0].x, v[0].y, v[1].x, v[1].y));
  } else if constexpr (P == 8) {
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack2<O>(v[0]), pack2<O>(v[1]), pack2<O>(v[2]), pack2<O>(v[3])));
  } else {
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack2<O>(v[0]), pack2<O>(v[1])));
  }
}

template <int THREADS, class T, class O>
__device__ __forceinline__ void scale_part(const GradEntry& e, GradPart part, int tid, double exact, bool clean) {
  // The coefficient is rounded to float32 (as exact as the products' own rounding) unless that is below float32's
  // normal range, where it has few bits left: then the values are scaled one by one in 64 bits.
  const float coef = (float)exact;
  const bool tiny = exact > 0.0 && exact < 0x1p-126;
  constexpr int P = 16 / sizeof(T), STEP = THREADS * GN_UNROLL;
  const T* base = static_cast<const T*>(e.in);
  O* out = static_cast<O*>(e.out);
  auto one = [&](long long i) {
    const float v = to_f32(base[i]);
    out[i] = from_f32<O>(tiny && isfinite(v) ? (float)((double)v * exact) : clip_value(v, coef, clean));
  };
  if (part.first == e.lead)
    for (int i = tid; i < min((long long)e.lead, e.n); i += THREADS) one(i);
  if (part.n <= 0) return;
  const uint4* from = reinterpret_cast<const uint4*>(base + part.first);
  O* to = out + part.first;
  const int pieces = e.vectors && !tiny ? part.n / P : 0;
  auto piece = [&](int at, uint4 u) {
    float2 v[P / 2];
    unpack_piece<T>(u, v);
#pragma unroll
    for (int k = 0; k < P / 2; k++) {
      if (clean) v[k] = make_float2(isfinite(v[k].x) ? v[k].x : 0.f, isfinite(v[k].y) ? v[k].y : 0.f);
      v[k] = mul2(v[k], both(coef));
    }
    store_piece<O, P>(to + (long long)at * P, v);
  };
  int i = tid;
  for (; i + STEP - THREADS < pieces; i += STEP) {
    uint4 u[GN_UNROLL];
#pragma unroll
    for (int k = 0; k < GN_UNROLL; k++) u[k] = __ldcs(from + i + k * THREADS);
#pragma unroll
    for (int k = 0; k < GN_UNROLL; k++) piece(i + k * THREADS, u[k]);
  }
  for (; i < pieces; i += THREADS) piece(i, __ldcs(from + i));
  for (int k = pieces * P + tid; k < part.n; k += THREADS) one(part.first + k);
}

template <int THREADS, class T>
__device__ __forceinline__ void scale_part(const GradEntry& e, GradPart part, int tid, double coef, bool clean) {
  if (e.out_type == F32) scale_part<THREADS, T, float>(e, part, tid, coef, clean);
  else if (e.out_type == BF16) scale_part<THREADS, T, __nv_bfloat16>(e, part, tid, coef, clean);
  else scale_part<THREADS, T, __half>(e, part, tid, coef, clean);
}
template <int THREADS>
__device__ __forceinline__ void scale_part(const GradEntry& e, GradPart part, int tid, double coef, bool clean) {
  if ((float)coef == 1.f && !clean && e.in == e.out) return;  // (in place, and every value stays as it is)
  if (e.in_type == F32) scale_part<THREADS, float>(e, part, tid, coef, clean);
  else if (e.in_type == BF16) scale_part<THREADS, __nv_bfloat16>(e, part, tid, coef, clean);
  else scale_part<THREADS, __half>(e, part, tid, coef, clean);
}

template <int N>
__global__ void __launch_bounds__(GN_THREADS) k_grad_scale(const __grid_constant__ GradTable<N> t, int parts,
                                                           const double2* __restrict__ part, double max_norm,
                                                           double eps, int zero, float* __restrict__ norm,
                                                           long long* __restrict__ bad) {
  let_next_start();
  wait_for_last();
  const double2 stats = sum_parts(parts, part);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (norm) *norm = (float)sqrt(stats.x);
    if (bad) *bad = (long long)stats.y;
  }
  const double coef = clip_coefficient(stats.x, max_norm, eps);
  const bool clean = zero && stats.y > 0.0;
  int i = t.count - 1;
  // (the chunks that this block had in the first pass, back from the last one)
  for (int c = blockIdx.x + (t.chunks - 1 - blockIdx.x) / gridDim.x * gridDim.x; c >= (int)blockIdx.x;
       c -= gridDim.x) {
    while (t.t[i].first > c) i--;
    const GradEntry& e = t.t[i];
    scale_part<GN_THREADS>(e, grad_part(t, e, c), threadIdx.x, coef, clean);
  }
}

// A short list in one launch: one cluster, whose blocks' warps take the chunks in turn, the blocks' sums exchanged
// through their shared memory under the cluster's barrier, the values read again from the caches. Two launches over all
// SMs wait for each other's start and end instead (a launch's time on the GPU, two launches / 16 blocks / 8 blocks: 34k
// float32 values 11 / 6.5 / 6.1 us, 438k bfloat16 to float32 11.7 / 9.0 / 13.1, 500k float32 10.8 / 7.1 / 10.4, 900k
// bfloat16 to float32 11.5 / 14.2 / 22.4).
template <int BLOCKS>
__global__ void __launch_bounds__(GN_SMALL_THREADS)
    k_grad_small(const __grid_constant__ GradTable<GN_FEW> t, int scale, double max_norm, double eps, int zero,
                 float* __restrict__ norm, long long* __restrict__ bad) {
  constexpr int WARPS = GN_SMALL_THREADS / 32;
  __shared__ double2 warp_sums[WARPS], block_sums[BLOCKS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x;  // (one cluster)
  let_next_start();
  cluster_arrive();
  wait_for_last();
  double2 v = make_double2(0.0, 0.0);
  auto entry = [&](int c) -> const GradEntry& {  // of chunk c: the last one whose first chunk is at most c
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t.t[mid].first <= c) lo = mid;
      else hi = mid - 1;
    }
    return t.t[lo];
  };
  // (a block's warps a chunk each, then the next block's, so that a few chunks are spread over all blocks' warps)
  const int first = warp * BLOCKS + rank, step = WARPS * BLOCKS;
  for (int c = first; c < t.chunks; c += step) {
    const GradEntry& e = entry(c);
    sumsq_part<32>(e, grad_part(t, e, c), lane, zero, v.x, v.y);
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, m);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, m);
  }
  if (lane == 0) warp_sums[warp] = v;
  __syncthreads();
  cluster_wait();  // (the other blocks are there)
  if (warp == 0) {
    v = lane < WARPS ? warp_sums[lane] : make_double2(0.0, 0.0);
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, m);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, m);
    }
    if (lane < BLOCKS) {  // lane k tells block k
      unsigned at = (unsigned)__cvta_generic_to_shared(&block_sums[rank]);
      asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(lane));
      asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(at), "d"(v.x), "d"(v.y) : "memory");
    }
    __syncwarp();
  }
  cluster_barrier();
  v = block_sums[0];
#pragma unroll
  for (int k = 1; k < BLOCKS; k++) v.x += block_sums[k].x, v.y += block_sums[k].y;
  if (rank == 0 && threadIdx.x == 0) {
    if (norm) *norm = (float)sqrt(v.x);
    if (bad) *bad = (long long)v.y;
  }
  if (!scale) return;
  const double coef = clip_coefficient(v.x, max_norm, eps);
  const bool clean = zero && v.y > 0.0;
  for (int c = first; c < t.chunks; c += step) {
    const GradEntry& e = entry(c);
    scale_part<32>(e, grad_part(t, e, c), lane, coef, clean);
  }
}

}  // namespace nbtrain
