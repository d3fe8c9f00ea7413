// The layer norm's launches: how a call is spread over blocks and tiles, and which kernel it takes.
#pragma once
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>
#include "nb_layer_norm.cuh"
#include "nb_launch.h"
#include "nb_layer_norm_call.h"

namespace nbtrain {

// How a layer norm of rows that a ring holds is spread: the tiles, and the blocks that take the tiles in turn.
constexpr int LN_SMEM = 226 * 1024, LN_SMEM_SM = 220 * 1024;
// bytes of a tile: 48 KB, or 32 where the backward's two tensors or two blocks an SM share the stages
constexpr int ln_tile(int lanes, bool backward) { return backward && lanes < 512 ? 32768 : backward ? 65536 : 49152; }
struct LnPlan {
  LnTiles t;
  int blocks, smem;
  bool fits;
};
// The lanes of a row and the values per lane.
inline void ln_spread(int cols, bool backward, int* lanes, int* ept) {
  // 8 for the narrowest rows, where 16 would leave half of the places empty (36 columns of float32: see k_ln_forward);
  // 32 for the widest of the forward, whose sums then meet in 8 warps instead of 16 (8192 x 8192 bfloat16: 49 us
  // against 59; the backward's two column sums leave no registers for it)
  *ept = cols <= 64 ? 8 : !backward && cols > 4096 ? 32 : 16;
  *lanes = 8;
  while (*lanes * *ept < cols) *lanes *= 2;
}
inline LnPlan ln_plan(long long rows, int cols, int e, bool backward) {
  LnPlan p = {};
  p.fits = cols <= LN_MAX_COLS;
  if (!p.fits) return p;
  ln_spread(cols, backward, &p.t.lanes, &p.t.ept);
  const int lanes = p.t.lanes, groups = ln_threads(lanes, e, backward) / lanes, row = cols * e;
  const int per_sm = ln_per_sm(lanes, e, backward), tensors = backward ? 2 : 1;
  const long long slots = (long long)SMS * per_sm, rounds = (rows + groups - 1) / groups;
  // a tile of about ln_tile bytes (of all tensors), but not so long that a block has no tile
  const int per_group = (int)std::max<long long>(
      1, std::min<long long>(ln_tile(lanes, backward) / (groups * row * tensors), (rounds + slots - 1) / slots));
  p.t.rows = rows, p.t.cols = cols, p.t.per_tile = groups * per_group;
  p.t.tile_bytes = (p.t.per_tile * row + 15) / 16 * 16 + 16;  // (16: a first row that starts inside a piece)
  p.t.stage_bytes = tensors * p.t.tile_bytes + (backward ? (8 * p.t.per_tile + 15) / 16 * 16 : 0);
  p.t.stages = std::min(4, LN_SMEM_SM / per_sm / p.t.stage_bytes);
  if (p.t.stages < 2) p.t.stages = std::min(4, LN_SMEM / p.t.stage_bytes);
  p.fits = p.t.stages >= 2;
  p.smem = p.t.stages * p.t.stage_bytes;
  p.blocks = (int)std::min<long long>((rounds + per_group - 1) / per_group, slots);
  return p;
}

// The partial column sums of the backward: one per block; with rows that no ring holds, one per block of rows.
constexpr int LN_WIDE_PARTS = 64;
inline int ln_wide_parts(long long rows) { return (int)std::min<long long>(LN_WIDE_PARTS, (rows + 15) / 16); }

inline int ln_kind(const void* p, long long rows, int cols, long long stride, int e) {
  if (rows == 1) stride = cols;
  const bool start = reinterpret_cast<uintptr_t>(p) % 16 == 0;
  if (start && stride == cols) return SPAN;
  return start && (long long)cols * e % 16 == 0 && stride * e % 16 == 0 ? PIECES : VALUES;
}

// The longest vector (16 bytes, 4 bytes or one value) that the rows' lengths and the result's start are multiples of.
inline int ln_vector(int e, int cols, const void* result) {
  const uintptr_t bits = (uintptr_t)cols * e | reinterpret_cast<uintptr_t>(result);
  return bits % 16 == 0 ? 16 / e : bits % 4 == 0 ? 4 / e : 1;
}

// calls f with the lanes of a row, the values per lane, the vector length and whether the lanes' places are all taken,
// as types
template <int N> using Int = std::integral_constant<int, N>;
template <class T, class F> int ln_vectors(const LnTiles& t, int vector, F f) {
  if (vector == (int)(16 / sizeof(T)))
    return t.cols == t.lanes * t.ept ? f(Int<16 / sizeof(T)>(), std::true_type())
                                     : f(Int<16 / sizeof(T)>(), std::false_type());
  if (sizeof(T) == 2 && vector == 2) return f(Int<4 / sizeof(T)>(), std::false_type());
  return f(Int<1>(), std::false_type());
}
template <class T, bool BACKWARD, class F> int ln_variant(const LnTiles& t, int vector, F f) {
  auto with = [&](auto lanes, auto ept) {
    return ln_vectors<T>(t, vector, [&](auto v, auto full) { return f(lanes, ept, v, full); });
  };
  switch (t.lanes) {
    case 8: return t.ept == 8 ? with(Int<8>(), Int<8>()) : with(Int<8>(), Int<16>());
    case 16: return with(Int<16>(), Int<16>());
    case 32: return with(Int<32>(), Int<16>());
    case 64: return with(Int<64>(), Int<16>());
    case 128: return with(Int<128>(), Int<16>());
    case 256:
      if constexpr (!BACKWARD)
        if (t.ept == 32) return with(Int<256>(), Int<32>());
      return with(Int<256>(), Int<16>());
    case 512: return with(Int<512>(), Int<BACKWARD ? 16 : 32>());
    default:
      if constexpr (BACKWARD) return with(Int<1024>(), Int<16>());
      else return (int)cudaErrorInvalidValue;
  }
}

// Lets a kernel use all of an SM's shared memory, once per device.
template <class K> int allow_smem(K kernel, std::atomic<bool>* done) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_relaxed)) return 0;
  const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LN_SMEM);
  if (rc == cudaSuccess && dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_relaxed);
  return (int)rc;
}

// calls f with the value type of the parameters
template <class T, class F> void ln_param_type(int wtype, F f) {
  if (wtype == F32) f(float());
  else f(T());
}

template <class T> int ln_forward(const LnForward& a) {
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  const LnPlan p = ln_plan(a.rows, a.cols, sizeof(T), false);
  if (!p.fits) {
    ln_param_type<T>(a.wtype, [&](auto w) {
      using W = decltype(w);
      k_ln_forward_wide<T, W><<<(unsigned)std::min<long long>(a.rows, 2 * SMS), 1024, 0, a.stream>>>(
          a.rows, a.cols, a.stride, x, static_cast<const W*>(a.weight), static_cast<const W*>(a.bias), a.eps, y,
          a.mean, a.rstd);
    });
    return (int)cudaGetLastError();
  }
  const int kind = ln_kind(a.x, a.rows, a.cols, a.stride, sizeof(T));
  return ln_variant<T, false>(p.t, ln_vector(sizeof(T), a.cols, y), [&](auto lanes, auto ept, auto v, auto full) {
    auto kernel = k_ln_forward<T, lanes.value, ept.value, v.value, full.value>;
    static std::atomic<bool> done[64];
    const int e = allow_smem(kernel, done);
    if (e) return e;
    return launch_after(a.stream, p.blocks, ln_threads(lanes.value, sizeof(T), false), p.smem, kernel, p.t, kind,
                        a.stride, x, a.wtype, a.weight, a.bias, a.eps, y, a.mean, a.rstd);
  });
}

template <class T> int ln_backward(const LnBackward& a) {
  const T *g = static_cast<const T*>(a.g), *x = static_cast<const T*>(a.x);
  T* gx = static_cast<T*>(a.gx);
  const bool sums = a.gw || a.gb;
  int parts = 0, e = 0;
  const LnPlan p = ln_plan(std::max(a.rows, 1ll), a.cols, sizeof(T), true);
  if (a.rows && !p.fits) {
    parts = ln_wide_parts(a.rows);
    if (gx)
      ln_param_type<T>(a.wtype, [&](auto w) {
        using W = decltype(w);
        k_ln_backward_wide<T, W><<<(unsigned)std::min<long long>(a.rows, 2 * SMS), 1024, 0, a.stream>>>(
            a.rows, a.cols, a.g_stride, a.stride, g, x, a.mean, a.rstd, static_cast<const W*>(a.weight), gx);
      });
    if (sums)
      k_ln_backward_wide_part<T><<<dim3((a.cols + 127) / 128, parts), 128, 0, a.stream>>>(
          a.rows, a.cols, a.g_stride, a.stride, g, x, a.mean, a.rstd, (a.rows + parts - 1) / parts, a.part);
    e = (int)cudaGetLastError();
  } else if (a.rows) {
    parts = p.blocks;
    const int gkind = ln_kind(a.g, a.rows, a.cols, a.g_stride, sizeof(T));
    const int kind = ln_kind(a.x, a.rows, a.cols, a.stride, sizeof(T));
    e = ln_variant<T, true>(p.t, ln_vector(sizeof(T), a.cols, gx), [&](auto lanes, auto ept, auto v, auto full) {
      auto kernel = k_ln_backward<T, lanes.value, ept.value, v.value, full.value>;
      static std::atomic<bool> done[64];
      const int rc = allow_smem(kernel, done);
      if (rc) return rc;
      return launch_after(a.stream, p.blocks, ln_threads(lanes.value, sizeof(T), true), p.smem, kernel, p.t, gkind,
                          a.g_stride, kind, a.stride, g, x, a.mean, a.rstd, a.wtype, a.weight, gx,
                          sums ? a.part : nullptr);
    });
  }
  if (e || !sums) return e;
  ln_param_type<T>(a.wtype, [&](auto w) {
    using W = decltype(w);
    // (many warps to a column where there are few columns, few where a block would wait for its place)
    auto sum = [&](auto warps) {
      return launch_after(a.stream, (2 * a.cols + 31) / 32, 32 * warps.value, 0, k_ln_backward_sum<W, warps.value>,
                          parts, a.cols, a.part, static_cast<W*>(a.gw), static_cast<W*>(a.gb));
    };
    e = a.cols <= 2048 ? sum(Int<32>()) : sum(Int<8>());
  });
  return e;
}

}  // namespace nbtrain
