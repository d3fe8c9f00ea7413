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

// How a layer norm of rows that a ring holds is spread: the tiles, and the blocks (clusters) that take them in turn.
constexpr int LN_SMEM = 224 * 1024, LN_SMEM_SM = 220 * 1024;
// bytes of a tile, of all tensors and the backward's two floats a row: 48 KB of rows, or 64, and room for the floats
// (backward, bfloat16 131072 x 512: 70 us with 48 KB, 76 with 32; 8192 x 8192, whose one block an SM waits at each
// tile: 81 us with 64 KB, 93 with 32)
constexpr int ln_tile(int lanes) { return lanes > LN_LANES ? 67 * 1024 : 50 * 1024; }
struct LnPlan {
  LnTiles t;
  int blocks, smem, per_sm;
  bool fits;
};
// The blocks and lanes of a row and the values per lane. 8 values for the narrowest rows, where 16 would leave half of
// the places empty; 32 for the widest of the forward, whose sums then meet in 8 warps instead of 16 (8192 x 8192
// bfloat16: 49 us against 59; the backward's column sums leave no registers for it, so it takes 512 lanes there).
// Beyond that a row is split over a cluster, evenly and in multiples of 16 columns, so that every part keeps the row's
// alignment.
inline bool ln_split_rows(int cols) { return cols > 16 * LN_SPLIT_LANES; }  // (in the backward)
inline void ln_spread(int cols, int e, bool backward, LnTiles* t) {
  const bool wide = cols > 16 * LN_LANES;
  const int most = backward && wide ? LN_SPLIT_LANES : LN_LANES;
  t->ept = cols <= 64 ? 8 : wide && !backward ? 32 : backward && ln_split_rows(cols) ? ln_split_ept(e) : 16;
  t->split = 1;
  while (t->split * most * t->ept < cols) t->split *= 2;
  t->width = t->split == 1 ? cols : ((cols + t->split - 1) / t->split + 15) / 16 * 16;
  t->lanes = wide ? most : 8;
  while (t->lanes * t->ept < t->width) t->lanes *= 2;
}
inline LnPlan ln_plan(long long rows, int cols, int e, bool backward) {
  LnPlan p = {};
  p.fits = cols <= LN_WIDEST;
  if (!p.fits) return p;
  ln_spread(cols, e, backward, &p.t);
  const int lanes = p.t.lanes, row = p.t.width * e, tensors = backward ? 2 : 1;
  const int groups = ln_threads(lanes, e, backward) / lanes;
  const bool split = backward && ln_split_rows(cols);  // (tiles of one row, and more of them)
  p.per_sm = ln_per_sm(lanes, e, backward, p.t.split > 1);
  const long long slots = (long long)SMS * p.per_sm / p.t.split, rounds = (rows + groups - 1) / groups;
  // Tiles of about ln_tile bytes; where a block has few of them, of the length that leaves the busiest block the least
  // rounds (a tile's own cost: a quarter of one).
  const int round = groups * (row * tensors + (backward ? 8 : 0));
  int per_group = 1;
  if (!split)
    per_group = (int)std::max<long long>(1, std::min<long long>(ln_tile(lanes) / round, (rounds + slots - 1) / slots));
  if (rounds < 8 * slots * per_group) {
    double least = 1e30;
    for (int k = per_group, longest = k; k >= 1 && k > longest / 2; k--) {
      const double tiles = (double)(((rounds + k - 1) / k + slots - 1) / slots), cost = tiles * (k + 0.25);
      if (cost < least) least = cost, per_group = k;
    }
  }
  p.t.rows = rows, p.t.cols = cols, p.t.per_tile = groups * per_group;
  p.t.tile_bytes = (p.t.per_tile * row + 15) / 16 * 16 + 16;  // (16: a first row that starts inside a piece)
  p.t.stage_bytes = tensors * p.t.tile_bytes + (backward ? (8 * p.t.per_tile + 15) / 16 * 16 : 0);
  p.t.stages = std::min(split ? 6 : 4, LN_SMEM_SM / p.per_sm / p.t.stage_bytes);
  p.fits = p.t.stages >= (split ? 4 : 2);
  p.smem = p.t.stages * p.t.stage_bytes;
  p.blocks = (int)std::min<long long>((rounds + per_group - 1) / per_group, slots) * p.t.split;
  return p;
}

// The partial column sums of the backward: one per block; with rows that no ring holds, one per block of rows.
constexpr int LN_WIDE_PARTS = 64;
inline int ln_wide_parts(long long rows) { return (int)std::min<long long>(LN_WIDE_PARTS, (rows + 15) / 16); }

inline int ln_kind(const void* p, const LnTiles& t, long long stride, int e) {
  const int cols = t.cols;
  if (t.rows == 1) stride = cols;
  const bool start = reinterpret_cast<uintptr_t>(p) % 16 == 0;
  if (start && stride == cols && t.split == 1) return SPAN;
  return start && (long long)cols * e % 16 == 0 && stride * e % 16 == 0 ? PIECES : VALUES;
}

// The longest vector (16 bytes, 4 bytes or one value) that the rows' lengths and the result's start are multiples of.
inline int ln_vector(int e, int cols, const void* result) {
  const uintptr_t bits = (uintptr_t)cols * e | reinterpret_cast<uintptr_t>(result);
  return bits % 16 == 0 ? 16 / e : bits % 4 == 0 ? 4 / e : 1;
}

// calls f with the lanes of a row, the values per lane, the vector length, whether the lanes' places are all taken and
// whether the row is split, as types
template <int N> using Int = std::integral_constant<int, N>;
template <class T, class F> int ln_vectors(const LnTiles& t, int vector, F f) {
  if (vector == (int)(16 / sizeof(T)))
    return t.cols == t.split * t.lanes * t.ept ? f(Int<16 / sizeof(T)>(), std::true_type())
                                               : f(Int<16 / sizeof(T)>(), std::false_type());
  if (sizeof(T) == 2 && vector == 2) return f(Int<4 / sizeof(T)>(), std::false_type());
  return f(Int<1>(), std::false_type());
}
template <class T, bool BACKWARD, class F> int ln_variant(const LnTiles& t, int vector, F f) {
  auto with = [&](auto lanes, auto ept, auto split) {
    return ln_vectors<T>(t, vector, [&](auto v, auto full) { return f(lanes, ept, v, full, split); });
  };
  const std::false_type one;
  if constexpr (!BACKWARD)
    if (t.split > 1) return with(Int<LN_LANES>(), Int<32>(), std::true_type());
  if (t.ept == 8) return with(Int<8>(), Int<8>(), one);
  if constexpr (!BACKWARD)
    if (t.ept == 32) return with(Int<LN_LANES>(), Int<32>(), one);
  switch (t.lanes) {
    case 8: return with(Int<8>(), Int<16>(), one);
    case 16: return with(Int<16>(), Int<16>(), one);
    case 32: return with(Int<32>(), Int<16>(), one);
    case 64: return with(Int<64>(), Int<16>(), one);
    case 128: return with(Int<128>(), Int<16>(), one);
    case LN_LANES: return with(Int<LN_LANES>(), Int<16>(), one);
    default:
      if constexpr (BACKWARD) return with(Int<LN_SPLIT_LANES>(), Int<16>(), one);
      else return (int)cudaErrorInvalidValue;
  }
}

// The blocks of a call whose rows are split over clusters: no more than the GPU holds at a time (asked once per kernel,
// cluster size and device).
template <auto KERNEL> int cluster_blocks(const LnPlan& p, int threads) {
  static std::atomic<int> known[64 * (LN_CLUSTER + 1)];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return p.blocks;
  std::atomic<int>& held = known[dev * (LN_CLUSTER + 1) + p.t.split];
  n = held.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = p.t.split, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(p.t.split * SMS);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = LN_SMEM_SM / p.per_sm;
    config.attrs = &attr;
    config.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, KERNEL, &config) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      return p.blocks;  // (they run one after the other)
    }
    held.store(n, std::memory_order_relaxed);
  }
  return std::min(p.blocks, n * p.t.split);
}

// Lets a kernel use all of an SM's shared memory, once per device.
template <auto KERNEL> int allow_smem() {
  static std::atomic<bool> done[64];
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_relaxed)) return 0;
  const cudaError_t rc = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, LN_SMEM);
  if (rc == cudaSuccess && dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_relaxed);
  return (int)rc;
}

// Prepares KERNEL and launches it as the plan has it (`blocks` is set to how many there are).
template <auto KERNEL, class... A>
int ln_launch(cudaStream_t stream, const LnPlan& p, int threads, int* blocks, A... args) {
  const int e = allow_smem<KERNEL>();
  if (e) return e;
  *blocks = p.t.split > 1 ? cluster_blocks<KERNEL>(p, threads) : p.blocks;
  return launch_after({stream, *blocks, threads, p.smem, p.t.split}, KERNEL, p.t, args...);
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
  const int kind = ln_kind(a.x, p.t, a.stride, sizeof(T));
  int blocks;
  return ln_variant<T, false>(p.t, ln_vector(sizeof(T), a.cols, y), [&](auto lanes, auto ept, auto v, auto full,
                                                                       auto split) {
    return ln_launch<k_ln_forward<T, lanes.value, ept.value, v.value, full.value, split.value>>(
        a.stream, p, ln_threads(lanes.value, sizeof(T), false), &blocks, kind, a.stride, x, a.wtype, a.weight, a.bias,
        a.eps, y, a.mean, a.rstd);
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
    const int gkind = ln_kind(a.g, p.t, a.g_stride, sizeof(T)), kind = ln_kind(a.x, p.t, a.stride, sizeof(T));
    const int vector = ln_vector(sizeof(T), a.cols, gx);
    float* part = sums ? a.part : nullptr;
    int blocks = 0;
    if (ln_split_rows(a.cols))
      e = ln_vectors<T>(p.t, vector, [&](auto v, auto full) {
        return ln_launch<k_ln_backward_split<T, LN_SPLIT_LANES, v.value, full.value>>(
            a.stream, p, LN_SPLIT_LANES, &blocks, gkind, a.g_stride, kind, a.stride, g, x, a.mean, a.rstd, a.wtype,
            a.weight, gx, part);
      });
    else
      e = ln_variant<T, true>(p.t, vector, [&](auto lanes, auto ept, auto v, auto full, auto) {
        return ln_launch<k_ln_backward<T, lanes.value, ept.value, v.value, full.value>>(
            a.stream, p, ln_threads(lanes.value, sizeof(T), true), &blocks, gkind, a.g_stride, kind, a.stride, g, x,
            a.mean, a.rstd, a.wtype, a.weight, gx, part);
      });
    parts = blocks / p.t.split;
  }
  if (e || !sums) return e;
  ln_param_type<T>(a.wtype, [&](auto w) {
    using W = decltype(w);
    // four columns to a thread where there are many (8192 x 8192 bfloat16 in all 80.6 us, 82.3 with one, 77.1 without
    // the sum)
    auto sum = [&](auto warps, auto v) {
      constexpr int WIDE = 32 * v.value;
      return launch_after({a.stream, (2 * a.cols + WIDE - 1) / WIDE, 32 * warps.value},
                          k_ln_backward_sum<W, warps.value, v.value>, parts, a.cols, a.part, static_cast<W*>(a.gw),
                          static_cast<W*>(a.gb));
    };
    e = a.cols <= 2048 ? sum(Int<32>(), Int<1>()) : a.cols % 4 ? sum(Int<8>(), Int<1>()) : sum(Int<32>(), Int<4>());
  });
  return e;
}

}  // namespace nbtrain
