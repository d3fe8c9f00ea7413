// The value types of the training operators (float32, bfloat16, float16), their conversions, and warp sums.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace nbtrain {

constexpr int SMS = 148;  // a B200's SMs (what grids and workspaces are sized by)

enum Dtype { F32 = 0, BF16 = 1, F16 = 2 };  // the C entries' type codes

inline int dtype_bytes(int d) { return d == F32 ? 4 : 2; }
inline bool dtype_ok(int d) { return d >= F32 && d <= F16; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
// (to 16 bits: the one rounding of a result, to nearest even)
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Two float32 operations in one instruction (each rounded to nearest, as the single ones).
__device__ __forceinline__ unsigned long long bits2(float2 v) { return *reinterpret_cast<unsigned long long*>(&v); }
__device__ __forceinline__ float2 pair2(unsigned long long b) { return *reinterpret_cast<float2*>(&b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return pair2(r);
}
// For kernels launched by launch_after: the next kernel may be set up from here on; and: the one before is complete and
// its memory seen (nothing is read or written earlier).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_barrier() {
  cluster_arrive();
  cluster_wait();
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The two values of a 32-bit word, and back.
template <class T> __device__ __forceinline__ float2 unpack2(unsigned w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(unsigned w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
template <class T> __device__ __forceinline__ unsigned pack2(float2 v);
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float2 v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <> __device__ __forceinline__ unsigned pack2<__half>(float2 v) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const unsigned*>(&h);
}

// V neighbouring values from one aligned access, as float32 pairs (zeros if they are not `there`), and back (V even).
template <class T, int V> __device__ __forceinline__ void load_pairs(const T* p, bool there, float2* out) {
  constexpr int W = V * sizeof(T) / 4;  // 32-bit words: 4 or 1
  unsigned w[W];
  if constexpr (W == 4) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (there) u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else {
    w[0] = there ? *reinterpret_cast<const unsigned*>(p) : 0u;
  }
#pragma unroll
  for (int i = 0; i < V / 2; i++) {
    if constexpr (sizeof(T) == 4) out[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else out[i] = unpack2<T>(w[i]);
  }
}
template <class T, int V> __device__ __forceinline__ void store_pairs(T* p, const float2* v) {
  constexpr int W = V * sizeof(T) / 4;
  unsigned w[W];
#pragma unroll
  for (int i = 0; i < V / 2; i++) {
    if constexpr (sizeof(T) == 4) w[2 * i] = __float_as_uint(v[i].x), w[2 * i + 1] = __float_as_uint(v[i].y);
    else w[i] = pack2<T>(v[i]);
  }
  if constexpr (W == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<unsigned*>(p) = w[0];
}

}  // namespace nbtrain
