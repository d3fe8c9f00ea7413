// Layer norm over the last dimension (N columns, M rows), forward and backward.
//   mean = sum x / N, var = sum (x - mean)^2 / N, rstd = (var + eps)^(-1/2), xh = (x - mean) rstd, y = xh w + b
//   h = g w, c1 = sum h / N, c2 = sum h xh / N, gx = rstd (h - c1 - xh c2), gw = sum_rows g xh, gb = sum_rows g
// Sums are float32; the variance is taken from the deviations (a second pass over registers), not from sum x^2. (Where
// the squares' sum is beyond float32 rstd is 0; where it vanishes and eps is 0, infinite.)
//
// A block takes tiles of rows in turn. The tiles come through a ring of up to four stages in shared memory, filled by
// asynchronous copies, so loads are in flight while a tile is worked on, and a dense x is copied in 16-byte pieces
// whatever its width: a tile is one span of memory, rounded out to whole pieces, and a row starts where it starts.
// From shared memory a row goes to the registers of `lanes` threads (8 to 512, a power of two), EPT values each. A
// thread keeps the same columns for every row it takes, so the weight, the bias and the two column sums of the backward
// stay in its registers too. Rows that do not fit take the row-in-memory kernels at the end.
//
// Memory bounds both directions (8 and 14 operations a value). 131072 x 512: forward bfloat16 50 us, 5.4 TB/s; backward
// float32 139 us, 5.8 TB/s with the sum of the column sums (a plain copy reaches 6.55). 16-bit rows of an odd width are
// bound by their instructions (values one by one: 65536 x 1001 float16 forward 74 us, backward 116), and the backward
// of rows of more than 4096 columns by one block an SM, whose 16 warps meet at each row (8192 x 8192 bfloat16: 83 us,
// 4.8 TB/s).
#pragma once
#include <cstdint>
#include "nb_values.cuh"

namespace nbtrain {

constexpr int LN_LANES = 256;        // lanes of a row in one block, two blocks an SM
constexpr int LN_SPLIT_LANES = 512;  // in the backward's widest rows: one block an SM
constexpr int LN_WIDEST = 32768;     // the widest row held in registers
constexpr int LN_CLUSTER = 8;        // blocks of a cluster at most
// values per lane there: 32 bytes of a row, so that four rows of both tensors fit the ring
__host__ __device__ constexpr int ln_split_ept(int e) { return 32 / e; }
// The threads of a block and the blocks per SM for rows of `lanes` lanes of e-byte values, as measured. Forward: one
// large block (131072 x 512 float32 88 us, 6100 GB/s, against 97 in two of half the size; 262144 x 512 bfloat16 88
// against 97), but two for 16-bit rows that are spread over several warps, where one computes while the other waits for
// its sums (131072 x 1024: 95 us against 108). Backward: one block for float32, which is bound by DRAM then
// (131072 x 512: 128 us, 6300 GB/s, against 142 in two), two for 16 bits, bound by its instructions (131072 x 1024:
// 133 us against 166).
__host__ __device__ constexpr int ln_threads(int lanes, int e, bool backward) {
  return lanes > LN_LANES || (!backward && lanes < LN_LANES && (e == 4 || lanes <= 32)) ? 512 : 256;
}
__host__ __device__ constexpr int ln_per_sm(int lanes, int e, bool backward, bool split) {
  return ln_threads(lanes, e, backward) == 256 && (split || !(backward && e == 4)) ? 2 : 1;
}

// How a tensor's rows lie: SPAN: dense rows from a 16-byte boundary; PIECES: every row a whole number of 16-byte
// pieces from a 16-byte boundary; VALUES: anything else.
enum LnRows { SPAN = 0, PIECES = 1, VALUES = 2 };

// The tiles of a call: rows of a tile, the tile's bytes in a stage (per tensor) and a stage's bytes. A row's columns
// are split over `split` blocks, `width` to each (the last has what is left).
struct LnTiles {
  long long rows;
  int cols, split, width, lanes, ept, per_tile, stages, tile_bytes, stage_bytes;
};

__device__ __forceinline__ void copy_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest n groups are complete (n: 0 to 3)
__device__ __forceinline__ void copy_wait(int n) {
  if (n == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (n == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// One tensor's rows on their way into the ring: a block's tiles one after the other.
template <class T, int THREADS> struct LnFeed {
  static constexpr int P = 16 / sizeof(T);
  const T* next;  // the first row of the next tile
  int kind, cols;
  long long stride, step;  // in values: between rows, between the block's tiles
  __device__ __forceinline__ LnFeed(const T* x, int kind, long long stride, const LnTiles& t, int team, int teams,
                                    int cols)
      : next(x + (long long)team * t.per_tile * stride),
        kind(kind),
        cols(cols),
        stride(stride),
        step((long long)teams * t.per_tile * stride) {}
  // The byte at which the first row of the tile at p starts in its stage.
  __device__ __forceinline__ int phase(const T* p) const {
    return kind == SPAN ? (int)(reinterpret_cast<uintptr_t>(p) & 15) : 0;
  }
  // Start copying the next tile's n rows into `dst` (16-byte aligned); `last`: the tensor ends with them.
  __device__ __forceinline__ void fill(unsigned char* dst, int n, bool last) {
    if (kind == SPAN) {
      const int lead = phase(next), bytes = lead + n * cols * (int)sizeof(T);
      const int pieces = last ? bytes >> 4 : (bytes + 15) >> 4;
      const unsigned char* from = reinterpret_cast<const unsigned char*>(next) - lead;
#pragma unroll 4
      for (int i = threadIdx.x; i < pieces; i += THREADS) copy_async16(dst + i * 16, from + i * 16);
      if (last && (bytes & 15))  // the tensor's last values, less than a piece
        for (int i = pieces * P + threadIdx.x; i < bytes / (int)sizeof(T); i += THREADS)
          reinterpret_cast<T*>(dst)[i] = reinterpret_cast<const T*>(from)[i];
    } else if (kind == PIECES) {
      const int per_row = cols / P;
      if (per_row >= THREADS) {
        for (int r = 0; r < n; r++)
          for (int i = threadIdx.x; i < per_row; i += THREADS)
            copy_async16(dst + (r * per_row + i) * 16, next + r * stride + i * P);
      } else {
        for (int i = threadIdx.x; i < per_row * n; i += THREADS) {
          const int r = i / per_row;
          copy_async16(dst + i * 16, next + r * stride + (i - r * per_row) * P);
        }
      }
    } else {
      for (int r = threadIdx.x >> 5; r < n; r += THREADS / 32) {
        const T* from = next + r * stride;
        T* to = reinterpret_cast<T*>(dst) + r * cols;
        if (sizeof(T) == 4) {
          for (int c = threadIdx.x & 31; c < cols; c += 32) copy_async4(to + c, from + c);
        } else {
#pragma unroll 8
          for (int c = threadIdx.x & 31; c < cols; c += 32) to[c] = from[c];
        }
      }
    }
    next += step;
  }
};

// A block's (or cluster's) tiles: the first row of the tile that is worked on, and of the one that is filled.
struct LnTurn {
  long long rows, row, fill_row, step;
  int per_tile;
  __device__ __forceinline__ LnTurn(const LnTiles& t, int team, int teams)
      : rows(t.rows),
        row((long long)team * t.per_tile),
        fill_row(row),
        step((long long)teams * t.per_tile),
        per_tile(t.per_tile) {}
  __device__ __forceinline__ int here(long long at) const {
    return rows - at < per_tile ? (int)(rows - at) : per_tile;
  }
};

// The LANES threads that share a row, and the sums of one or two floats over them: shuffles inside a warp, and for
// wider rows one exchange through `slots` (two sets in turn, so one barrier is enough): under the group's own named
// barrier, or, where the row is split over a cluster, with every warp's sum put into the slots of all its blocks, under
// the cluster's barrier. A thread holds the row's values i = 0 .. EPT - 1 at the columns (i / V * LANES + lane) * V +
// i % V, in pairs.
template <int LANES, bool SPLIT> struct LnGroup {
  static constexpr int WARPS = LANES / 32;
  int lane, index;  // lane: the thread's place in its row's group; index: the group in the block
  int rank, split;  // of the cluster
  float* slots;     // 2 x 64
  int turn;
  __device__ __forceinline__ void sum(float (&v)[1]) {
#pragma unroll
    for (int m = (LANES < 32 ? LANES : 32) / 2; m > 0; m >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
    if constexpr (SPLIT) {
      float* s = slots + (turn & 1) * 64;
      turn++;
      const int to = threadIdx.x & 31;  // lane k of each warp tells block k
      if (to < split) {
        unsigned at = (unsigned)__cvta_generic_to_shared(s + rank * WARPS + (lane >> 5));
        asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(to));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v[0]) : "memory");
      }
      cluster_barrier();
      const int all = split * WARPS;  // 16, 32 or 64
      v[0] = s[to & (all - 1)];
      if (all > 32) v[0] += s[32 + to];
      for (int m = (all < 32 ? all : 32) / 2; m > 0; m >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
    } else if constexpr (LANES > 32) {
      float* s = slots + (turn & 1) * 64 + index * WARPS;
      turn++;
      if ((threadIdx.x & 31) == 0) s[lane >> 5] = v[0];
      asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "n"(LANES) : "memory");
      v[0] = s[threadIdx.x & (WARPS - 1)];
#pragma unroll
      for (int m = WARPS / 2; m > 0; m >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
    }
  }
  // two sums: from the first step on half of a warp holds the one and half the other
  __device__ __forceinline__ void sum(float (&v)[2]) {
    static_assert(!SPLIT, "one sum at a time over a cluster");
    constexpr int HALF = (LANES < 32 ? LANES : 32) / 2;
    const bool upper = threadIdx.x & HALF;
    float mine = upper ? v[1] : v[0];
    mine += __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[1], HALF);
#pragma unroll
    for (int m = HALF / 2; m > 0; m >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, m);
    if constexpr (LANES > 32) {
      float* s = slots + (turn & 1) * 64 + index * 2 * WARPS + (upper ? WARPS : 0);
      turn++;
      if ((threadIdx.x & 15) == 0) s[lane >> 5] = mine;
      asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "n"(LANES) : "memory");
      mine = s[threadIdx.x & (WARPS - 1)];
#pragma unroll
      for (int m = WARPS / 2; m > 0; m >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, m);
    }
    const float other = __shfl_xor_sync(0xffffffffu, mine, HALF);
    v[0] = upper ? other : mine;
    v[1] = upper ? mine : other;
  }
};

template <int LANES, int V> __device__ __forceinline__ int ln_column(int lane, int i) {
  return (i / V * LANES + lane) * V + i % V;
}

// A thread's values of a parameter, `absent` where there is none.
template <int LANES, int EPT, int V>
__device__ __forceinline__ void load_param(const void* p, int wtype, int col0, float absent, int cols, int lane,
                                           float2* out) {
#pragma unroll
  for (int i = 0; i < EPT; i++) {
    const int c = ln_column<LANES, V>(lane, i);
    float v = absent;
    if (p && c < cols)
      v = wtype == F32 ? static_cast<const float*>(p)[col0 + c]
          : wtype == BF16 ? to_f32(static_cast<const __nv_bfloat16*>(p)[col0 + c])
                          : to_f32(static_cast<const __half*>(p)[col0 + c]);
    (i % 2 ? out[i / 2].y : out[i / 2].x) = v;
  }
}

// A thread's values of a row, 0 beyond the last column.
template <class T, int LANES, int EPT, int V, bool FULL>
__device__ __forceinline__ void load_row(const T* row, int cols, int lane, float2* out) {
  if constexpr (V == 1) {
#pragma unroll
    for (int i = 0; i < EPT; i++) {
      const int c = i * LANES + lane;
      (i % 2 ? out[i / 2].y : out[i / 2].x) = c < cols ? to_f32(row[c]) : 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPT / V; j++) {
      const int c = (j * LANES + lane) * V;
      load_pairs<T, V>(row + c, FULL || c < cols, out + j * V / 2);
    }
  }
}

template <class T, int LANES, int EPT, int V, bool FULL>
__device__ __forceinline__ void store_row(T* row, int cols, int lane, const float2* v) {
  if constexpr (V == 1) {
#pragma unroll
    for (int i = 0; i < EPT; i++) {
      const int c = i * LANES + lane;
      if (c < cols) row[c] = from_f32<T>(i % 2 ? v[i / 2].y : v[i / 2].x);
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPT / V; j++) {
      const int c = (j * LANES + lane) * V;
      if (FULL || c < cols) store_pairs<T, V>(row + c, v + j * V / 2);
    }
  }
}

// A thread's float32 values at its columns of `row` (any alignment of its start where V is 1 or 2).
template <int LANES, int EPT, int V, bool FULL>
__device__ __forceinline__ void store_sums(float* row, int cols, int lane, const float2* v) {
#pragma unroll
  for (int j = 0; j < EPT / V; j++) {
    const int c = (j * LANES + lane) * V;
    if (!FULL && c >= cols) continue;
    if constexpr (V >= 4) {
#pragma unroll
      for (int k = 0; k < V / 4; k++) store_pairs<float, 4>(row + c + 4 * k, v + (j * V + 4 * k) / 2);
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) row[c + k] = (j * V + k) % 2 ? v[(j * V + k) / 2].y : v[(j * V + k) / 2].x;
    }
  }
}

// Set the places beyond the last column to 0 (a vector is on one side of it).
template <int LANES, int EPT, int V>
__device__ __forceinline__ void clear_beyond(int cols, int lane, float2* v) {
#pragma unroll
  for (int j = 0; j < EPT / V; j++) {
    const bool beyond = (j * LANES + lane) * V >= cols;
#pragma unroll
    for (int k = j * V; k < (j + 1) * V; k++)
      if (beyond) (k % 2 ? v[k / 2].y : v[k / 2].x) = 0.f;
  }
}

// The forward: the row's mean, then the variance from the deviations in registers, each sum over the lanes; rstd by
// rsqrtf (2 units in the last place at most, below what the variance's sum leaves). FULL: every block has LANES * EPT
// columns (no thread has a place beyond the last); SPLIT: a row is split over the blocks of a cluster.
template <class T, int LANES, int EPT, int V, bool FULL, bool SPLIT>
__global__ void __launch_bounds__(ln_threads(LANES, sizeof(T), false), ln_per_sm(LANES, sizeof(T), false, SPLIT))
    k_ln_forward(LnTiles t, int kind, long long stride, const T* __restrict__ x, int wtype,
                 const void* __restrict__ weight, const void* __restrict__ bias, float eps, T* __restrict__ y,
                 float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float slots[128];
  constexpr int THREADS = ln_threads(LANES, sizeof(T), false), GROUPS = THREADS / LANES, N2 = EPT / 2;
  static_assert(!SPLIT || GROUPS == 1, "the blocks of a cluster share one row");
  // this block's place in its cluster, its columns, and its team's place among the teams that take the tiles in turn
  const int split = SPLIT ? t.split : 1, rank = SPLIT ? (int)(blockIdx.x % split) : 0, col0 = rank * t.width;
  const int cols = FULL ? LANES * EPT : SPLIT ? min(t.width, t.cols - col0) : t.cols, pitch = SPLIT ? t.cols : cols;
  const int team = SPLIT ? blockIdx.x / split : blockIdx.x, teams = SPLIT ? gridDim.x / split : gridDim.x;
  const int lane = threadIdx.x % LANES;
  let_next_start();
  if (SPLIT) cluster_barrier();  // (the other blocks' slots are there)
  LnGroup<LANES, SPLIT> g = {lane, (int)threadIdx.x / LANES, rank, split, slots, 0};
  const int shift = LANES < 32 ? (int)(threadIdx.x & 31) / LANES : 0;  // the group's place in its warp
  const float inv = 1.f / t.cols;
  LnFeed<T, THREADS> feed(x + col0, kind, stride, t, team, teams, cols);
  LnTurn turn(t, team, teams);
  auto fill = [&](int stage) {
    if (turn.fill_row < turn.rows) {
      const int n = turn.here(turn.fill_row);
      feed.fill(ring + stage * t.stage_bytes, n, turn.fill_row + n == turn.rows);
      turn.fill_row += turn.step;
    }
    copy_commit();
  };
  const T* at = feed.next;
  T* out = y + turn.row * pitch + col0;
  const long long out_step = turn.step * pitch;
  wait_for_last();
  for (int s = 0; s + 1 < t.stages; s++) fill(s);
  float2 w[N2], b[N2];
  load_param<LANES, EPT, V>(weight, wtype, col0, 1.f, cols, lane, w);
  load_param<LANES, EPT, V>(bias, wtype, col0, 0.f, cols, lane, b);
  int stage = 0, free_stage = t.stages - 1;
  for (; turn.row < turn.rows; turn.row += turn.step, at += feed.step, out += out_step) {
    copy_wait(t.stages - 2);
    __syncthreads();  // the tile is here, and nobody reads the stage of the tile before it any more
    fill(free_stage);
    const int n = turn.here(turn.row);
    const T* rows = reinterpret_cast<const T*>(ring + stage * t.stage_bytes + feed.phase(at));
    free_stage = stage;
    stage = stage + 1 == t.stages ? 0 : stage + 1;
    // (two rows' loops in one where it gains: 65536 x 1024 bfloat16 47.8 -> 45.6 us; not 131072 x 512 float32, 85 ->
    // 90, nor 65536 x 1001 bfloat16, 71 -> 80)
    constexpr int TOGETHER = sizeof(T) == 2 && LANES > 32 && V > 1 ? 2 : 1;
#pragma unroll TOGETHER
    for (int r0 = g.index - shift; r0 < n; r0 += GROUPS) {  // (r0: the warp's first row)
      const int r = r0 + shift;
      float2 v[N2];
      load_row<T, LANES, EPT, V, FULL>(rows + min(r, n - 1) * cols, cols, lane, v);
      float2 a = v[0];
#pragma unroll
      for (int i = 1; i < N2; i++) a = add2(a, v[i]);
      float s[1] = {a.x + a.y};
      g.sum(s);
      const float mean = s[0] * inv;
#pragma unroll
      for (int i = 0; i < N2; i++) v[i] = add2(v[i], both(-mean));
      if (!FULL) clear_beyond<LANES, EPT, V>(cols, lane, v);
      a = mul2(v[0], v[0]);
#pragma unroll
      for (int i = 1; i < N2; i++) a = fma2(v[i], v[i], a);
      s[0] = a.x + a.y;
      g.sum(s);
      const float rstd = rsqrtf(fmaf(s[0], inv, eps));
#pragma unroll
      for (int i = 0; i < N2; i++) v[i] = fma2(mul2(v[i], both(rstd)), w[i], b[i]);
      if (r < n) {
        store_row<T, LANES, EPT, V, FULL>(out + (long long)r * pitch, cols, lane, v);
        if (rank == 0 && lane < 2) (lane ? rstd_out : mean_out)[turn.row + r] = lane ? rstd : mean;
      }
    }
  }
  if (SPLIT) cluster_barrier();  // (nobody leaves while others put sums into its slots)
}

// The sum of N terms (a power of two) in a tree, so that none passes through more than log2 N additions.
template <int N, class F> __device__ __forceinline__ float tree_sum(F term) {
  if constexpr (N == 1) return term(0);
  else return tree_sum<N / 2>(term) + tree_sum<N / 2>([&](int k) { return term(k + N / 2); });
}

// The backward: both sums of a row (h and h xh) meet in one exchange; (x - mean) rstd is taken as written, not as one
// fused product, which would leave rounding where x is the mean. part (gridDim.x, 2, cols), if wanted: the block's
// column sums of g xh and g, which k_ln_backward_sum adds up in a fixed order.
template <class T, int LANES, int EPT, int V, bool FULL>
__global__ void __launch_bounds__(ln_threads(LANES, sizeof(T), true), ln_per_sm(LANES, sizeof(T), true, false))
    k_ln_backward(LnTiles t, int gkind, long long gstride, int kind, long long stride, const T* __restrict__ gy,
                  const T* __restrict__ x, const float* __restrict__ mean, const float* __restrict__ rstd, int wtype,
                  const void* __restrict__ weight, T* __restrict__ gx, float* __restrict__ part) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float slots[128];
  constexpr int THREADS = ln_threads(LANES, sizeof(T), true), GROUPS = THREADS / LANES, N2 = EPT / 2;
  const int cols = FULL ? LANES * EPT : t.cols, lane = threadIdx.x % LANES;
  let_next_start();
  LnGroup<LANES, false> g = {lane, (int)threadIdx.x / LANES, 0, 1, slots, 0};
  const int shift = LANES < 32 ? (int)(threadIdx.x & 31) / LANES : 0;
  const float inv = 1.f / t.cols;
  LnFeed<T, THREADS> xfeed(x, kind, stride, t, blockIdx.x, gridDim.x, cols);
  LnFeed<T, THREADS> gfeed(gy, gkind, gstride, t, blockIdx.x, gridDim.x, cols);
  LnTurn turn(t, blockIdx.x, gridDim.x);
  auto fill = [&](int stage) {
    if (turn.fill_row < turn.rows) {
      unsigned char* to = ring + stage * t.stage_bytes;
      const int n = turn.here(turn.fill_row);
      const bool last = turn.fill_row + n == turn.rows;
      xfeed.fill(to, n, last);
      gfeed.fill(to + t.tile_bytes, n, last);
      float* stats = reinterpret_cast<float*>(to + 2 * t.tile_bytes);
      for (int i = threadIdx.x; i < n; i += THREADS) {
        copy_async4(stats + i, mean + turn.fill_row + i);
        copy_async4(stats + t.per_tile + i, rstd + turn.fill_row + i);
      }
      turn.fill_row += turn.step;
    }
    copy_commit();
  };
  const T *xat = xfeed.next, *gat = gfeed.next;
  T* out = gx + turn.row * cols;
  const long long out_step = turn.step * cols;
  wait_for_last();
  for (int s = 0; s + 1 < t.stages; s++) fill(s);
  float2 w[N2], gw[N2], gb[N2];
  load_param<LANES, EPT, V>(weight, wtype, 0, 1.f, cols, lane, w);
#pragma unroll
  for (int i = 0; i < N2; i++) gw[i] = gb[i] = both(0.f);
  int stage = 0, free_stage = t.stages - 1;
  for (; turn.row < turn.rows; turn.row += turn.step, xat += xfeed.step, gat += gfeed.step, out += out_step) {
    copy_wait(t.stages - 2);
    __syncthreads();
    fill(free_stage);
    const int n = turn.here(turn.row);
    const unsigned char* base = ring + stage * t.stage_bytes;
    const T* xrows = reinterpret_cast<const T*>(base + xfeed.phase(xat));
    const T* grows = reinterpret_cast<const T*>(base + t.tile_bytes + gfeed.phase(gat));
    const float* stats = reinterpret_cast<const float*>(base + 2 * t.tile_bytes);
    free_stage = stage;
    stage = stage + 1 == t.stages ? 0 : stage + 1;
    // (as in the forward: 8192 x 8192 bfloat16 80.6 -> 76.8 us, 262144 x 36 float32 38.3 -> 30.5; 16384 x 4096 float32
    // 131 -> 135)
    constexpr int TOGETHER = LANES > LN_LANES || EPT == 8 ? 2 : 1;
#pragma unroll TOGETHER
    for (int r0 = g.index - shift; r0 < n; r0 += GROUPS) {
      const int r = r0 + shift, at = min(r, n - 1);
      float2 xh[N2], h[N2];
      load_row<T, LANES, EPT, V, FULL>(xrows + at * cols, cols, lane, xh);
      load_row<T, LANES, EPT, V, FULL>(grows + at * cols, cols, lane, h);
      const float m = stats[at], rs = stats[t.per_tile + at];
#pragma unroll
      for (int i = 0; i < N2; i++) xh[i] = mul2(add2(xh[i], both(-m)), both(rs));
      if (!FULL) clear_beyond<LANES, EPT, V>(cols, lane, xh);
      if (r < n) {
#pragma unroll
        for (int i = 0; i < N2; i++) {
          gw[i] = fma2(h[i], xh[i], gw[i]);
          gb[i] = add2(gb[i], h[i]);
        }
      }
      float2 c1 = both(0.f), c2 = both(0.f);
#pragma unroll
      for (int i = 0; i < N2; i++) {
        h[i] = mul2(h[i], w[i]);
        c1 = add2(c1, h[i]);
        c2 = fma2(h[i], xh[i], c2);
      }
      float c[2] = {c1.x + c1.y, c2.x + c2.y};
      g.sum(c);
      if (!gx || r >= n) continue;
      c1 = both(-c[0] * inv * rs);
      c2 = both(-c[1] * inv * rs);
#pragma unroll
      for (int i = 0; i < N2; i++) h[i] = fma2(xh[i], c2, fma2(h[i], both(rs), c1));
      store_row<T, LANES, EPT, V, FULL>(out + r * cols, cols, lane, h);
    }
  }
  if (!part) return;
  // the column sums of the block: of its one group, or of its groups, (GROUPS, 2, cols) over the ring
  float* sums = part + (long long)blockIdx.x * 2 * cols;
  float* mine = GROUPS == 1 ? sums : reinterpret_cast<float*>(ring) + g.index * 2 * cols;
  if (GROUPS > 1) {
    copy_wait(0);
    __syncthreads();
  }
  store_sums<LANES, EPT, V, FULL>(mine, cols, lane, gw);
  store_sums<LANES, EPT, V, FULL>(mine + cols, cols, lane, gb);
  if (GROUPS == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * cols; c += THREADS)
    sums[c] = tree_sum<GROUPS>([&](int k) { return reinterpret_cast<const float*>(ring)[k * 2 * cols + c]; });
}

// The backward of rows that one block does not take: a row to each team of t.split blocks (a cluster) of LANES threads,
// t.width columns to a block. The two sums of a row meet in the slots of all its blocks
// under the cluster's barrier, which is split: between arriving with row k's sums and waiting for the others' a thread
// finishes row k - 1, from shared memory again: nobody stands still for the exchange, for half as many instructions
// again (8192 x 8192 bfloat16, which needs no cluster, took 103 us here when k_ln_backward took 94; 4096 x 16384
// bfloat16: 113 us, 3.6 TB/s; 4096 x 12000 float32: 223 us, 2.6 TB/s: the exchange and the second load bound it). part
// (teams, 2, cols), if wanted.
template <class T, int LANES, int V, bool FULL>
__global__ void __launch_bounds__(LANES, 512 / LANES)
    k_ln_backward_split(LnTiles t, int gkind, long long gstride, int kind, long long stride, const T* __restrict__ gy,
                        const T* __restrict__ x, const float* __restrict__ mean, const float* __restrict__ rstd,
                        int wtype, const void* __restrict__ weight, T* __restrict__ gx, float* __restrict__ part) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float2 slots[2][128];
  constexpr int EPT = ln_split_ept(sizeof(T)), N2 = EPT / 2, WARPS = LANES / 32;
  const int split = t.split, rank = blockIdx.x % split, team = blockIdx.x / split, teams = gridDim.x / split;
  const int col0 = rank * t.width, cols = FULL ? LANES * EPT : min(t.width, t.cols - col0);
  const int lane = threadIdx.x, to = lane & 31, all = split * WARPS;
  let_next_start();
  LnFeed<T, LANES> xfeed(x + col0, kind, stride, t, team, teams, cols);
  LnFeed<T, LANES> gfeed(gy + col0, gkind, gstride, t, team, teams, cols);
  const float inv = 1.f / t.cols;
  long long fill_row = team;
  auto fill = [&](int stage) {
    if (fill_row < t.rows) {
      unsigned char* dst = ring + stage * t.stage_bytes;
      xfeed.fill(dst, 1, fill_row + 1 == t.rows);
      gfeed.fill(dst + t.tile_bytes, 1, fill_row + 1 == t.rows);
      float* stats = reinterpret_cast<float*>(dst + 2 * t.tile_bytes);
      if (lane < 2) copy_async4(stats + lane, (lane ? rstd : mean) + fill_row);
      fill_row += teams;
    }
    copy_commit();
  };
  const T *xat = xfeed.next, *gat = gfeed.next;
  cluster_arrive();
  wait_for_last();
  for (int s = 0; s + 2 < t.stages; s++) fill(s);
  float2 w[N2], gw[N2], gb[N2];
  load_param<LANES, EPT, V>(weight, wtype, col0, 1.f, cols, lane, w);
#pragma unroll
  for (int i = 0; i < N2; i++) gw[i] = gb[i] = both(0.f);
  copy_wait(t.stages - 3);  // row 0 is here
  __syncthreads();
  cluster_wait();  // (and the other blocks' slots are there)
  // a row of stage `stage`: its normalised values and its cotangent times the weight
  auto load = [&](int stage, const T* xp, const T* gp, float2* xh, float2* h) {
    const unsigned char* base = ring + stage * t.stage_bytes;
    load_row<T, LANES, EPT, V, FULL>(reinterpret_cast<const T*>(base + xfeed.phase(xp)), cols, lane, xh);
    load_row<T, LANES, EPT, V, FULL>(reinterpret_cast<const T*>(base + t.tile_bytes + gfeed.phase(gp)), cols, lane, h);
    const float* stats = reinterpret_cast<const float*>(base + 2 * t.tile_bytes);
    const float m = stats[0], rs = stats[1];
#pragma unroll
    for (int i = 0; i < N2; i++) xh[i] = mul2(add2(xh[i], both(-m)), both(rs));
    if (!FULL) clear_beyond<LANES, EPT, V>(cols, lane, xh);
    return rs;
  };
  int stage = 0, last = 0, next = t.stages - 2;  // of the row that is summed, of the one that is finished, to be filled
  float c1 = 0.f, c2 = 0.f;
  T* out = gx + (long long)team * t.cols + col0;  // of the row that is finished
  auto finish = [&](int at, const T* xp, const T* gp) {
    if (!gx) return;
    float2 xh[N2], h[N2];
    const float rs = load(at, xp, gp, xh, h);
    const float2 a = both(-c1 * inv * rs), b = both(-c2 * inv * rs);
#pragma unroll
    for (int i = 0; i < N2; i++) h[i] = fma2(xh[i], b, fma2(mul2(h[i], w[i]), both(rs), a));
    store_row<T, LANES, EPT, V, FULL>(out, cols, lane, h);
    out += (long long)teams * t.cols;
  };
  bool first = true;
  int turn = 0;
  for (long long row = team; row < t.rows; row += teams, turn ^= 1) {
    float s[2];
    {
      float2 xh[N2], h[N2], a = both(0.f), b = both(0.f);
      load(stage, xat, gat, xh, h);
#pragma unroll
      for (int i = 0; i < N2; i++) {
        gw[i] = fma2(h[i], xh[i], gw[i]);
        gb[i] = add2(gb[i], h[i]);
        h[i] = mul2(h[i], w[i]);
        a = add2(a, h[i]);
        b = fma2(h[i], xh[i], b);
      }
      s[0] = a.x + a.y;
      s[1] = b.x + b.y;
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
      s[0] += __shfl_xor_sync(0xffffffffu, s[0], m);
      s[1] += __shfl_xor_sync(0xffffffffu, s[1], m);
    }
    if (to < split) {  // lane k of each warp tells block k
      unsigned at = (unsigned)__cvta_generic_to_shared(&slots[turn][rank * WARPS + (lane >> 5)]);
      asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(to));
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(s[0]), "f"(s[1]) : "memory");
    }
    copy_wait(t.stages - 4);  // the next row is here once everybody has arrived
    __syncwarp();
    cluster_arrive();
    if (!first) finish(last, xat - xfeed.step, gat - gfeed.step);
    first = false;
    cluster_wait();
    // the sums of this row (read before the next arrival: the slots are the next but one row's), and the stage of the
    // row before the last, which everybody has finished
    float2 o = slots[turn][to & (all - 1)];
    for (int k = 32 + to; k < all; k += 32) o.x += slots[turn][k].x, o.y += slots[turn][k].y;
    for (int m = (all < 32 ? all : 32) / 2; m > 0; m >>= 1) {
      o.x += __shfl_xor_sync(0xffffffffu, o.x, m);
      o.y += __shfl_xor_sync(0xffffffffu, o.y, m);
    }
    c1 = o.x, c2 = o.y;
    fill(next);
    next = next + 1 == t.stages ? 0 : next + 1;
    last = stage;
    stage = stage + 1 == t.stages ? 0 : stage + 1;
    xat += xfeed.step, gat += gfeed.step;
  }
  if (!first) finish(last, xat - xfeed.step, gat - gfeed.step);
  copy_wait(0);
  if (!part) return;
  float* sums = part + (long long)team * 2 * t.cols + col0;
  store_sums<LANES, EPT, V, FULL>(sums, cols, lane, gw);
  store_sums<LANES, EPT, V, FULL>(sums + t.cols, cols, lane, gb);
}

// gw, gb = the sums of the blocks' column sums: 32 V columns a block, a warp for each WARPS-th of the parts
template <class W, int WARPS, int V>
__global__ void __launch_bounds__(32 * WARPS) k_ln_backward_sum(int parts, int cols, const float* __restrict__ part,
                                                                W* __restrict__ gw, W* __restrict__ gb) {
  __shared__ float s[WARPS][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + lane) * V;  // 0 .. 2 cols: gw's columns, then gb's (V divides both)
  let_next_start();
  wait_for_last();
  float v[V];
#pragma unroll
  for (int k = 0; k < V; k++) v[k] = 0.f;
  if (c < 2 * cols) {
#pragma unroll 10
    for (int p = warp; p < parts; p += WARPS) {
      const float* from = part + (long long)p * 2 * cols + c;
      if constexpr (V == 4) {
        const float4 u = *reinterpret_cast<const float4*>(from);
        v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
      } else {
        v[0] += *from;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < V; k++) s[warp][lane * V + k] = v[k];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 32 * WARPS) {
    const int at = blockIdx.x * 32 * V + i;
    if (at >= 2 * cols) continue;
    const float t = tree_sum<WARPS>([&](int k) { return s[k][i]; });
    if (at < cols) {
      if (gw) gw[at] = from_f32<W>(t);
    } else if (gb) {
      gb[at - cols] = from_f32<W>(t);
    }
  }
}

// ---- rows that no ring holds: a block per row, the row read again from memory in each pass ---------------------
__device__ __forceinline__ float wide_sum(float v) {
  __shared__ float s[32];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[threadIdx.x & 31];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

template <class T, class W>
__global__ void __launch_bounds__(1024) k_ln_forward_wide(long long rows, int cols, long long stride,
                                                          const T* __restrict__ x, const W* __restrict__ weight,
                                                          const W* __restrict__ bias, float eps, T* __restrict__ y,
                                                          float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * stride;
    float s = 0.f;
    for (int c = threadIdx.x; c < cols; c += 1024) s += to_f32(xr[c]);
    const float mean = wide_sum(s) / cols;
    s = 0.f;
    for (int c = threadIdx.x; c < cols; c += 1024) {
      const float d = to_f32(xr[c]) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = rsqrtf(wide_sum(s) / cols + eps);
    for (int c = threadIdx.x; c < cols; c += 1024) {
      float v = (to_f32(xr[c]) - mean) * rstd;
      if (weight) v *= to_f32(weight[c]);
      if (bias) v += to_f32(bias[c]);
      y[row * cols + c] = from_f32<T>(v);
    }
    if (threadIdx.x == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

template <class T, class W>
__global__ void __launch_bounds__(1024) k_ln_backward_wide(long long rows, int cols, long long gstride,
                                                           long long stride, const T* __restrict__ g,
                                                           const T* __restrict__ x, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd,
                                                           const W* __restrict__ weight, T* __restrict__ gx) {
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * stride, *gr = g + row * gstride;
    const float m = mean[row], r = rstd[row];
    float c1 = 0.f, c2 = 0.f;
    for (int c = threadIdx.x; c < cols; c += 1024) {
      const float h = to_f32(gr[c]) * (weight ? to_f32(weight[c]) : 1.f);
      c1 += h;
      c2 = fmaf(h, (to_f32(xr[c]) - m) * r, c2);
    }
    c1 = wide_sum(c1) / cols;
    c2 = wide_sum(c2) / cols;
    for (int c = threadIdx.x; c < cols; c += 1024) {
      const float h = to_f32(gr[c]) * (weight ? to_f32(weight[c]) : 1.f);
      gx[row * cols + c] = from_f32<T>((h - c1 - (to_f32(xr[c]) - m) * r * c2) * r);
    }
  }
}

// Column sums of g xh and g over part_rows rows per block row, one thread per column: part (parts, 2, cols).
template <class T>
__global__ void __launch_bounds__(128) k_ln_backward_wide_part(long long rows, int cols, long long gstride,
                                                               long long stride, const T* __restrict__ g,
                                                               const T* __restrict__ x,
                                                               const float* __restrict__ mean,
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

}  // namespace nbtrain
