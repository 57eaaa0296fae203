// Layer norm of rows, and its gradient.
//
//   mean = sum(x) / D    rstd = 1 / sqrt(sum((x - mean)^2) / D + eps)
//   xhat = (x - mean) * rstd        y = xhat * weight + bias
//
//   g  = dy * weight
//   dx = rstd * (g - sum(g) / D - xhat * sum(g * xhat) / D)
//   d_weight = sum over rows of dy * xhat        d_bias = sum over rows of dy
//
// Bound by HBM: the forward pass reads and writes every row once, the backward
// pass reads two and writes one.  A row stays in registers between its
// reduction and its use.  Statistics, sums and products are 32-bit floats, and
// every result is rounded once; the variance is the sum of squared distances
// from the mean (not of squares), so rows far from zero lose nothing.
//
// Rows are given by base and stride, or (the pointer form) by one address per
// row, as find* returns them: rows are then normalised straight from where the
// table keeps them, rows in pinned host memory included, and the output rows of
// misses (null addresses) are left as they are, as find leaves them.
//
// The reference has no such operator; what it hands to one are the rows of
// find (include/merlin_hashtable.cuh:2464-2577) and find* (2729-2787).
#include "hkv_norm.h"
#include "hkv_rows.cuh"

namespace hkv {

namespace {

constexpr uint32_t kFull = 0xFFFFFFFFu;
constexpr int kNormBlock = 256;       // forward; more where a row needs more
constexpr int kBackwardBlock = 512;

// Sum over the `group` threads of a row (a power of two: part of a warp, or
// whole warps of this block); every thread gets it.  scratch: two floats of each
// value per warp, used in turn, so that one barrier of the group's own (named
// 1 + its number in the block) is enough.
template <int N>
struct GroupSum {
  uint32_t group, warp, first_warp, barrier;
  float (*scratch)[2][N];   // [warps of the block]
  uint32_t turn = 0;

  __device__ __forceinline__ GroupSum(uint32_t group_, float (*scratch_)[2][N])
      : group(group_),
        warp(threadIdx.x >> 5),
        first_warp((threadIdx.x >> 5) & ~((group_ >> 5) - (group_ >> 5 ? 1u : 0u))),
        barrier(1u + threadIdx.x / group_),
        scratch(scratch_) {}

  __device__ __forceinline__ void operator()(float (&v)[N]) {
    const uint32_t width = group < 32u ? group : 32u;
    for (uint32_t d = width >> 1; d > 0; d >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kFull, v[i], d);
    }
    if (group <= 32u) return;
    if ((threadIdx.x & 31u) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) scratch[warp][turn][i] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(group) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    for (uint32_t w = first_warp; w < first_warp + (group >> 5); ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += scratch[w][turn][i];
    }
    turn ^= 1u;
  }
};

// Where a thread's chunks lie in its row: chunk c of the thread is
// first + c * width.  A warp of a group above 32 owns consecutive chunks, so that
// neighbouring chunks are in neighbouring lanes whatever the group.
struct ChunkMap {
  uint32_t first, width, lane;   // lane: within the width

  __device__ __forceinline__ ChunkMap(uint32_t group, int per_thread) {
    width = group < 32u ? group : 32u;
    lane = threadIdx.x & (width - 1u);
    const uint32_t warp_in_group = (threadIdx.x & (group - 1u)) >> 5;
    first = warp_in_group * 32u * uint32_t(per_thread) + lane;
  }
  __device__ __forceinline__ uint32_t operator()(int c) const { return first + uint32_t(c) * width; }
};

// The thread's chunks of a row; what is behind the row's end is zero.
template <typename T, int CHUNKS, bool WHOLE>
__device__ __forceinline__ void load_row(const uint8_t* row, uint64_t row_bytes, uint32_t chunks,
                                         const ChunkMap& map, const uint8_t* first,
                                         const uint8_t* last, Chunk<T> (&x)[CHUNKS]) {
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t at = map(c);
    x[c].raw = make_uint4(0, 0, 0, 0);
    if (row == nullptr || at >= chunks) continue;
    const uint8_t* p = row + uint64_t(at) * 16;
    if (WHOLE) {
      x[c].raw = __ldg(reinterpret_cast<const uint4*>(p));
    } else {
      x[c].raw = load_chunk<sizeof(T)>(p, p, row + row_bytes, first, last);
      if (p + 16 > row + row_bytes) {
        const int have = int(row + row_bytes - p) / int(sizeof(T));
#pragma unroll
        for (int e = 0; e < Chunk<T>::kElems; ++e) {
          if (e >= have) x[c].set(e, 0.f);
        }
      }
    }
  }
}

// Stores the thread's chunks of a row.  At an unaligned address every aligned 16
// bytes belong to two neighbouring chunks: a lane gets its left neighbour's and
// stores the joint; only the ends of the row, and of a warp's run of it, are
// stored element by element.  The whole warp calls; row == nullptr: nothing.
template <typename T, int CHUNKS, bool WHOLE>
__device__ __forceinline__ void store_row(uint8_t* row, uint64_t row_bytes, uint32_t chunks,
                                          const ChunkMap& map, const Chunk<T> (&y)[CHUNKS]) {
  if (WHOLE) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const uint32_t at = map(c);
      if (row != nullptr && at < chunks) *reinterpret_cast<uint4*>(row + uint64_t(at) * 16) = y[c].raw;
    }
    return;
  }
  const uint32_t s = uint32_t(reinterpret_cast<uintptr_t>(row)) & 15u;
  const uint8_t* end = row + row_bytes;
  const uint32_t left = (threadIdx.x & 31u & ~(map.width - 1u)) | ((map.lane - 1u) & (map.width - 1u));
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t at = map(c);
    const bool to_next = map.lane == map.width - 1u;   // its right neighbour is in the next round
    const uint4 mine = y[c].raw;
    const uint4 give = to_next && c > 0 ? y[c > 0 ? c - 1 : 0].raw : mine;
    uint4 prev;
    prev.x = __shfl_sync(kFull, give.x, left);
    prev.y = __shfl_sync(kFull, give.y, left);
    prev.z = __shfl_sync(kFull, give.z, left);
    prev.w = __shfl_sync(kFull, give.w, left);
    if (row == nullptr || at > chunks) continue;
    uint8_t* q = row + uint64_t(at) * 16;
    const bool joined = map.lane != 0 || c > 0;        // the left neighbour's bytes are here
    if (s == 0) {
      store_chunk<sizeof(T)>(q, mine, row, end);
      continue;
    }
    store_chunk<sizeof(T)>(q - s, shifted(prev, mine, 16u - s), joined ? row : q, end);
    if (c == CHUNKS - 1 && to_next) {
      // the end of the warp's run: nobody joins this chunk's last bytes
      const uint4 none = make_uint4(0, 0, 0, 0);
      const uint8_t* stop = q + 16 < end ? q + 16 : end;
      store_chunk<sizeof(T)>(q - s + 16, shifted(mine, none, 16u - s), row, stop);
    }
  }
}

// weight or bias of a chunk's columns; 1 or 0 where there is none or no column.
template <typename T, bool WHOLE, int N>
__device__ __forceinline__ void load_params(const void* p, bool f32, uint32_t column, uint32_t dim,
                                            float none, float (&out)[N]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = none;
  } else if (WHOLE) {
    // whole chunks of columns, and the launcher has checked the address
    if (f32) {
      const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + column);
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const float4 v = __ldg(s + e / 4);
        out[e] = v.x;
        out[e + 1] = v.y;
        out[e + 2] = v.z;
        out[e + 3] = v.w;
      }
    } else {
      Chunk<T> v;
      v.raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p) + column));
#pragma unroll
      for (int e = 0; e < N; ++e) out[e] = v.get(e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      out[e] = none;
      if (column + e < dim) {
        out[e] = f32 ? static_cast<const float*>(p)[column + e]
                     : to_float(static_cast<const T*>(p)[column + e]);
      }
    }
  }
}

// CHUNKS chunks per thread, `group` threads per row, one row per group.
template <typename T, int CHUNKS, bool WHOLE>
__global__ void __launch_bounds__(1024)
    norm_kernel(const NormArgs a, const uint32_t group, const uint32_t chunks, const RowsIn in) {
  using C = Chunk<T>;
  __shared__ float scratch[32][2][1];
  const uint64_t r = (uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) / group;
  const ChunkMap map(group, CHUNKS);
  const uint64_t row_bytes = a.dim * sizeof(T);
  const uint8_t *row = nullptr, *first = in.first, *last = in.last;
  if (r < a.n) {
    if (a.row_ptrs != nullptr) {
      row = first = static_cast<const uint8_t*>(a.row_ptrs[r]);
      last = row + row_bytes;
    } else {
      row = in.first + r * in.stride;
    }
  }
  C x[CHUNKS];
  load_row<T, CHUNKS, WHOLE>(row, row_bytes, chunks, map, first, last, x);
  GroupSum<1> group_sum(group, scratch);
  const float inv_dim = a.inv_dim;
  float sum[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int e = 0; e < C::kElems; ++e) sum[0] += x[c].get(e);
  }
  group_sum(sum);
  const float mean = sum[0] * inv_dim;
  float sq[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t column = map(c) * C::kElems;
#pragma unroll
    for (int e = 0; e < C::kElems; ++e) {
      const float d = x[c].get(e) - mean;
      if (column + (WHOLE ? 0 : e) < a.dim) sq[0] = fmaf(d, d, sq[0]);
    }
  }
  group_sum(sq);
  const float rstd = 1.f / sqrtf(fmaf(sq[0], inv_dim, a.eps));
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    if (map(c) >= chunks) break;
    float w[C::kElems], b[C::kElems];
    const uint32_t column = map(c) * C::kElems;
    load_params<T, WHOLE>(a.weight, a.params_f32, column, uint32_t(a.dim), 1.f, w);
    load_params<T, WHOLE>(a.bias, a.params_f32, column, uint32_t(a.dim), 0.f, b);
#pragma unroll
    for (int e = 0; e < C::kElems; ++e) x[c].set(e, fmaf((x[c].get(e) - mean) * rstd, w[e], b[e]));
  }
  uint8_t* to = row == nullptr ? nullptr : static_cast<uint8_t*>(a.y) + r * a.y_stride;
  store_row<T, CHUNKS, WHOLE>(to, row_bytes, chunks, map, x);
  if (row != nullptr && (threadIdx.x & (group - 1u)) == 0) {
    if (a.mean != nullptr) a.mean[r] = mean;
    if (a.rstd != nullptr) a.rstd[r] = rstd;
  }
}

// Rows too long for the registers of a block: three passes over the row, which
// stays in L2 between them.
template <typename T>
__global__ void __launch_bounds__(1024)
    norm_long_kernel(const NormArgs a) {
  __shared__ float scratch[32][2][1];
  GroupSum<1> group_sum(blockDim.x, scratch);
  const uint32_t dim = uint32_t(a.dim);
  for (uint64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    const T* row = a.row_ptrs != nullptr
                       ? static_cast<const T*>(a.row_ptrs[r])
                       : reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.x) + r * a.x_stride);
    if (row == nullptr) continue;
    float sum[1] = {0.f};
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) sum[0] += to_float(row[i]);
    group_sum(sum);
    const float mean = sum[0] * a.inv_dim;
    float sq[1] = {0.f};
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      const float d = to_float(row[i]) - mean;
      sq[0] = fmaf(d, d, sq[0]);
    }
    group_sum(sq);
    const float rstd = 1.f / sqrtf(fmaf(sq[0], a.inv_dim, a.eps));
    T* out = reinterpret_cast<T*>(static_cast<uint8_t*>(a.y) + r * a.y_stride);
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      float w[1], b[1];
      load_params<T, false>(a.weight, a.params_f32, i, dim, 1.f, w);
      load_params<T, false>(a.bias, a.params_f32, i, dim, 0.f, b);
      out[i] = from_float<T>(fmaf((to_float(row[i]) - mean) * rstd, w[0], b[0]));
    }
    if (threadIdx.x == 0) {
      if (a.mean != nullptr) a.mean[r] = mean;
      if (a.rstd != nullptr) a.rstd[r] = rstd;
    }
  }
}

// ---- backward -----------------------------------------------------------------
//
// The blocks stay on the device and take rows in turn: a thread sees the same
// columns of every row it touches, so the column sums d_weight and d_bias build
// up in its registers beside the row's own work, and x and dy are read once.
// The next row's chunks are on their way while the current row is reduced.
// At the end each block writes one row of column sums (its groups added in a
// fixed order), and norm_reduce_kernel adds the blocks' rows in a fixed order.

struct NormBackwardPlan {
  uint32_t group, chunks, per_thread, blocks;
  bool fits;   // a row fits the registers of a block
};

template <typename T, int CHUNKS, bool WHOLE>
__global__ void __launch_bounds__(kBackwardBlock, 1)
    norm_backward_kernel(const NormBackwardArgs a, const uint32_t group, const uint32_t chunks,
                         const RowsIn x_in, const RowsIn dy_in, float* __restrict__ sums) {
  using C = Chunk<T>;
  constexpr int kElems = C::kElems;
  extern __shared__ float columns[];   // [copies][dim]: the column sums of each warp or group
  __shared__ float scratch[kBackwardBlock / 32][2][2];
  GroupSum<2> group_sum(group, scratch);
  const ChunkMap map(group, CHUNKS);
  const uint32_t dim = uint32_t(a.dim);
  const uint64_t row_bytes = a.dim * sizeof(T);
  const uint32_t groups = kBackwardBlock / group;
  float w[CHUNKS][kElems], dw[CHUNKS][kElems], db[CHUNKS][kElems];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int e = 0; e < kElems; ++e) dw[c][e] = db[c][e] = w[c][e] = 0.f;
    if (map(c) < chunks) {
      load_params<T, WHOLE>(a.weight, a.params_f32, map(c) * kElems, dim, 1.f, w[c]);
    }
  }
  const uint64_t step = uint64_t(gridDim.x) * groups;
  uint64_t r = uint64_t(blockIdx.x) * groups + threadIdx.x / group;
  C x[CHUNKS], dy[CHUNKS];
  float mean = 0.f, rstd = 0.f;
  auto fetch = [&](uint64_t row) {
    const bool live = row < a.n;
    mean = live ? __ldg(a.mean + row) : 0.f;
    rstd = live ? __ldg(a.rstd + row) : 0.f;
    load_row<T, CHUNKS, WHOLE>(live ? x_in.first + row * x_in.stride : nullptr, row_bytes, chunks, map,
                               x_in.first, x_in.last, x);
    load_row<T, CHUNKS, WHOLE>(live ? dy_in.first + row * dy_in.stride : nullptr, row_bytes, chunks,
                               map, dy_in.first, dy_in.last, dy);
  };
  fetch(r);
  // the lanes of a warp leave together: their rows are done when the warp's first is
  for (uint64_t warp_row = r - (threadIdx.x & 31u) / group; warp_row < a.n;
       warp_row += step, r += step) {
    float xhat[CHUNKS][kElems], g[CHUNKS][kElems];
    float sum[2] = {0.f, 0.f};
    const float row_rstd = rstd;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        const float d = dy[c].get(e);
        xhat[c][e] = (x[c].get(e) - mean) * rstd;
        g[c][e] = d * w[c][e];
        sum[0] += g[c][e];
        sum[1] = fmaf(g[c][e], xhat[c][e], sum[1]);
        dw[c][e] = fmaf(d, xhat[c][e], dw[c][e]);
        db[c][e] += d;
      }
    }
    fetch(r + step);
    group_sum(sum);
    const float m0 = sum[0] * a.inv_dim, m1 = sum[1] * a.inv_dim;
    C dx[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        dx[c].set(e, row_rstd * (fmaf(-m1, xhat[c][e], g[c][e]) - m0));
      }
    }
    store_row<T, CHUNKS, WHOLE>(
        r < a.n ? static_cast<uint8_t*>(a.dx) + r * a.dx_stride : nullptr, row_bytes, chunks, map, dx);
  }
  // the sums of the block's groups: those of one warp by exchange, the others
  // one after the other
  const uint32_t copies = group < 32u ? kBackwardBlock / 32 : groups;
  const uint32_t copy = group < 32u ? threadIdx.x >> 5 : threadIdx.x / group;
  for (uint32_t d = 16; d >= group; d >>= 1) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        dw[c][e] += __shfl_xor_sync(kFull, dw[c][e], d);
        db[c][e] += __shfl_xor_sync(kFull, db[c][e], d);
      }
    }
  }
  const bool writes = group >= 32u || (threadIdx.x & 31u) < group;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which == 0 ? a.d_weight == nullptr : a.d_bias == nullptr) continue;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        const uint32_t column = map(c) * kElems + e;
        if (writes && column < dim) columns[copy * dim + column] = which == 0 ? dw[c][e] : db[c][e];
      }
    }
    __syncthreads();
    float* mine = sums + (uint64_t(which) * gridDim.x + blockIdx.x) * dim;
    for (uint32_t i = threadIdx.x; i < dim; i += kBackwardBlock) {
      float v = columns[i];
      for (uint32_t k = 1; k < copies; ++k) v += columns[k * dim + i];
      mine[i] = v;
    }
  }
}

// Rows too long for the registers of a block: the row's two sums and dx first,
// re-reading the row from L2, then the column sums on their own.
template <typename T>
__global__ void __launch_bounds__(512)
    norm_backward_long_kernel(const NormBackwardArgs a) {
  __shared__ float scratch[16][2][2];
  GroupSum<2> group_sum(blockDim.x, scratch);
  const uint32_t dim = uint32_t(a.dim);
  for (uint64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.x) + r * a.x_stride);
    const T* dy = reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.dy) + r * a.dy_stride);
    T* dx = reinterpret_cast<T*>(static_cast<uint8_t*>(a.dx) + r * a.dx_stride);
    const float mean = a.mean[r], rstd = a.rstd[r];
    float sum[2] = {0.f, 0.f};
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      float w[1];
      load_params<T, false>(a.weight, a.params_f32, i, dim, 1.f, w);
      const float g = to_float(dy[i]) * w[0];
      sum[0] += g;
      sum[1] = fmaf(g, (to_float(x[i]) - mean) * rstd, sum[1]);
    }
    group_sum(sum);
    const float m0 = sum[0] * a.inv_dim, m1 = sum[1] * a.inv_dim;
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      float w[1];
      load_params<T, false>(a.weight, a.params_f32, i, dim, 1.f, w);
      const float xhat = (to_float(x[i]) - mean) * rstd;
      dx[i] = from_float<T>(rstd * (fmaf(-m1, xhat, to_float(dy[i]) * w[0]) - m0));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kNormBlock)
    norm_columns_kernel(const NormBackwardArgs a, float* __restrict__ sums) {
  const uint64_t i = uint64_t(blockIdx.x) * kNormBlock + threadIdx.x;
  if (i >= a.dim) return;
  float dw = 0.f, db = 0.f;
#pragma unroll 4
  for (uint64_t r = blockIdx.y; r < a.n; r += gridDim.y) {
    const float d = to_float(
        reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.dy) + r * a.dy_stride)[i]);
    const float v = to_float(
        reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.x) + r * a.x_stride)[i]);
    dw = fmaf(d, (v - a.mean[r]) * a.rstd[r], dw);
    db += d;
  }
  if (a.d_weight != nullptr) sums[uint64_t(blockIdx.y) * a.dim + i] = dw;
  if (a.d_bias != nullptr) sums[(uint64_t(gridDim.y) + blockIdx.y) * a.dim + i] = db;
}

// Adds the blocks' rows of column sums: 32 columns per block, warp w takes
// rows w, w + 32, ...
template <typename T>
__global__ void __launch_bounds__(1024)
    norm_reduce_kernel(const float* __restrict__ sums, const uint32_t rows, const uint64_t dim,
                       const bool params_f32, void* __restrict__ d_weight, void* __restrict__ d_bias) {
  __shared__ float part[32][33];
  void* to = blockIdx.y == 0 ? d_weight : d_bias;
  if (to == nullptr) return;
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint64_t i = uint64_t(blockIdx.x) * 32u + lane;
  const float* from = sums + uint64_t(blockIdx.y) * rows * dim;
  float sum = 0.f;
  if (i < dim) {
#pragma unroll 8
    for (uint32_t r = warp; r < rows; r += 32u) sum += from[r * dim + i];
  }
  part[warp][lane] = sum;
  __syncthreads();
  // warp w adds column w of this block
  float v = part[lane][warp];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  const uint64_t column = uint64_t(blockIdx.x) * 32u + warp;
  if (lane == 0 && column < dim) {
    if (params_f32) static_cast<float*>(to)[column] = v;
    else static_cast<T*>(to)[column] = from_float<T>(v);
  }
}

// ---- launch -------------------------------------------------------------------

uint32_t pow2_at_least(uint64_t v) {
  uint32_t p = 1;
  while (p < v) p <<= 1;
  return p;
}

// Chunks of a row; the last one may be part of one.
uint64_t chunks_of(uint64_t row_bytes) { return (row_bytes + 15) / 16; }

// Parameters are read in chunks where the rows are: their addresses count too.
uint64_t param_bits(const void* weight, const void* bias) {
  return address_bits(weight) | address_bits(bias);
}

constexpr uint32_t kMaxGroup = 1024;

template <typename T>
void launch_norm_type(const NormArgs& a, bool whole, cudaStream_t stream) {
  const uint64_t chunks = chunks_of(a.dim * sizeof(T));
  if (chunks > 4ull * kMaxGroup) {
    const uint64_t cap = uint64_t(sm_count()) * 2;
    norm_long_kernel<T><<<unsigned(a.n < cap ? a.n : cap), kMaxGroup, 0, stream>>>(a);
    return;
  }
  // four chunks per thread where the row has them, fewer where there are too
  // few rows to fill the device with that
  const uint64_t enough = uint64_t(sm_count()) * 512;
  uint32_t per_thread = 4, group = pow2_at_least((chunks + 3) / 4);
  while (per_thread > 1 && group < kMaxGroup &&
         (a.n * group < enough || pow2_at_least(chunks) <= 2)) {
    per_thread >>= 1;
    group = pow2_at_least((chunks + per_thread - 1) / per_thread);
  }
  const uint32_t block = group > kNormBlock ? group : kNormBlock;
  const uint64_t grid = (a.n * group + block - 1) / block;
  const RowsIn in = a.row_ptrs != nullptr ? RowsIn{} : rows_in(a.x, a.n, a.x_stride, a.dim * sizeof(T));
  auto kernel = whole ? (per_thread == 1   ? norm_kernel<T, 1, true>
                         : per_thread == 2 ? norm_kernel<T, 2, true>
                                           : norm_kernel<T, 4, true>)
                      : (per_thread == 1   ? norm_kernel<T, 1, false>
                         : per_thread == 2 ? norm_kernel<T, 2, false>
                                           : norm_kernel<T, 4, false>);
  kernel<<<unsigned(grid), block, 0, stream>>>(a, group, uint32_t(chunks), in);
}

// Chunks a thread of the backward kernel holds: 16 elements' column sums, row
// values and weights fill the registers that 512 threads have.
constexpr uint32_t backward_chunks(uint32_t size) { return size == 4 ? 4 : 2; }

NormBackwardPlan plan_backward(uint64_t n, uint64_t dim, uint32_t size) {
  NormBackwardPlan p{};
  const uint64_t chunks = chunks_of(dim * size);
  p.per_thread = backward_chunks(size);
  p.fits = chunks <= uint64_t(kBackwardBlock) * p.per_thread;
  if (!p.fits) {
    p.blocks = uint32_t(n < 64 ? n : 64);   // row splits of the column sums
    return p;
  }
  p.chunks = uint32_t(chunks);
  p.group = pow2_at_least((chunks + p.per_thread - 1) / p.per_thread);
  const uint64_t groups = kBackwardBlock / p.group;
  const uint64_t want = (n + groups - 1) / groups;
  const uint64_t cap = uint64_t(sm_count());
  p.blocks = uint32_t(want < cap ? want : cap);
  return p;
}

template <typename T>
void launch_backward_type(const NormBackwardArgs& a, const NormBackwardPlan& p, bool whole, float* sums,
                          cudaStream_t stream) {
  constexpr int kChunks = backward_chunks(sizeof(T));
  const uint64_t row_bytes = a.dim * sizeof(T);
  const uint32_t copies = p.group < 32 ? kBackwardBlock / 32 : kBackwardBlock / p.group;
  auto kernel = whole ? norm_backward_kernel<T, kChunks, true> : norm_backward_kernel<T, kChunks, false>;
  kernel<<<p.blocks, kBackwardBlock, copies * a.dim * sizeof(float), stream>>>(
      a, p.group, p.chunks, rows_in(a.x, a.n, a.x_stride, row_bytes),
      rows_in(a.dy, a.n, a.dy_stride, row_bytes), sums);
}

template <typename T>
void launch_backward_long(const NormBackwardArgs& a, const NormBackwardPlan& p, float* sums,
                          cudaStream_t stream) {
  const uint64_t cap = uint64_t(sm_count()) * 4;
  norm_backward_long_kernel<T><<<unsigned(a.n < cap ? a.n : cap), 512, 0, stream>>>(a);
  if (sums != nullptr) {
    const dim3 grid(unsigned((a.dim + kNormBlock - 1) / kNormBlock), p.blocks);
    norm_columns_kernel<T><<<grid, kNormBlock, 0, stream>>>(a, sums);
  }
}

template <typename T>
void launch_reduce(const NormBackwardArgs& a, uint32_t rows, const float* sums, cudaStream_t stream) {
  const dim3 grid(unsigned((a.dim + 31) / 32), 2);
  norm_reduce_kernel<T><<<grid, 1024, 0, stream>>>(sums, rows, a.dim, a.params_f32, a.d_weight,
                                                   a.d_bias);
}

int check_norm(uint64_t n, uint64_t dim, uint32_t value_kind, uint32_t param_kind, float eps) {
  HKV_ROWS_CHECK(n < (1ull << 31), "batches of 2^31 or more rows");
  HKV_ROWS_CHECK(dim >= 1 && dim < (1ull << 24), "dim must be between 1 and 2^24 - 1");
  HKV_ROWS_CHECK(is_row_kind(value_kind), "rows are float32, float16 or bfloat16");
  HKV_ROWS_CHECK(param_kind == value_kind || param_kind == kValueF32,
                 "weight and bias have the rows' type or float32");
  HKV_ROWS_CHECK(eps >= 0.f && eps <= 3.4e38f, "eps must be finite and not negative");
  return HKV_OK;
}

}  // namespace

int launch_norm(const NormArgs& args, uint32_t value_kind, cudaStream_t stream) {
  const uint32_t size = row_kind_size(value_kind);
  const uint64_t row_bytes = args.dim * size;
  uint64_t bits = row_bytes | address_bits(args.y) | args.y_stride;
  // the pointer form's addresses are on the device: table rows start at
  // multiples of the widest access their length allows
  if (args.row_ptrs == nullptr) bits |= address_bits(args.x) | args.x_stride;
  HKV_ROWS_CHECK(bits % size == 0, "a row does not start at a multiple of its element size");
  const bool whole = whole_chunks(bits | param_bits(args.weight, args.bias));
  if (value_kind == kValueF32) launch_norm_type<float>(args, whole, stream);
  else if (value_kind == kValueF16) launch_norm_type<__half>(args, whole, stream);
  else launch_norm_type<__nv_bfloat16>(args, whole, stream);
  return rows_launched();
}

}  // namespace hkv

using namespace hkv;

extern "C" {

int hkv_layer_norm(uint64_t n, uint64_t dim, uint32_t value_kind, const void* x, uint64_t x_stride,
                   const void* weight, const void* bias, uint32_t param_kind, float eps, void* y,
                   uint64_t y_stride, float* mean, float* rstd, hkv_stream stream) {
  const int rc = check_norm(n, dim, value_kind, param_kind, eps);
  if (rc != HKV_OK) return rc;
  HKV_ROWS_CHECK(y_stride >= dim * row_kind_size(value_kind), "the output rows overlap");
  if (n == 0) return HKV_OK;
  HKV_ROWS_CHECK(x != nullptr && y != nullptr, "x and y must not be null");
  NormArgs a{};
  a.n = n;
  a.dim = dim;
  a.x = x;
  a.x_stride = x_stride;
  a.weight = weight;
  a.bias = bias;
  a.params_f32 = param_kind == kValueF32;
  a.eps = eps;
  a.inv_dim = 1.f / float(dim);
  a.y = y;
  a.y_stride = y_stride;
  a.mean = mean;
  a.rstd = rstd;
  return launch_norm(a, value_kind, static_cast<cudaStream_t>(stream));
}

int hkv_layer_norm_ptr(uint64_t n, uint64_t dim, uint32_t value_kind, const void* const* row_ptrs,
                       const void* weight, const void* bias, uint32_t param_kind, float eps, void* y,
                       uint64_t y_stride, float* mean, float* rstd, hkv_stream stream) {
  const int rc = check_norm(n, dim, value_kind, param_kind, eps);
  if (rc != HKV_OK) return rc;
  HKV_ROWS_CHECK(y_stride >= dim * row_kind_size(value_kind), "the output rows overlap");
  if (n == 0) return HKV_OK;
  HKV_ROWS_CHECK(row_ptrs != nullptr && y != nullptr, "row_ptrs and y must not be null");
  NormArgs a{};
  a.n = n;
  a.dim = dim;
  a.row_ptrs = row_ptrs;
  a.weight = weight;
  a.bias = bias;
  a.params_f32 = param_kind == kValueF32;
  a.eps = eps;
  a.inv_dim = 1.f / float(dim);
  a.y = y;
  a.y_stride = y_stride;
  a.mean = mean;
  a.rstd = rstd;
  return launch_norm(a, value_kind, static_cast<cudaStream_t>(stream));
}

uint64_t hkv_layer_norm_backward_workspace_bytes(uint64_t n, uint64_t dim, uint32_t value_kind) {
  if (check_norm(n, dim, value_kind, value_kind, 0.f) != HKV_OK || n == 0) return 0;
  return 2ull * plan_backward(n, dim, row_kind_size(value_kind)).blocks * dim * sizeof(float);
}

int hkv_layer_norm_backward(uint64_t n, uint64_t dim, uint32_t value_kind, const void* dy,
                            uint64_t dy_stride, const void* x, uint64_t x_stride,
                            const void* weight, uint32_t param_kind, const float* mean,
                            const float* rstd, void* dx, uint64_t dx_stride, void* d_weight,
                            void* d_bias, void* work, uint64_t work_bytes, hkv_stream stream) {
  const int rc = check_norm(n, dim, value_kind, param_kind, 0.f);
  if (rc != HKV_OK) return rc;
  const uint32_t size = row_kind_size(value_kind);
  HKV_ROWS_CHECK(dx_stride >= dim * size, "the rows of dx overlap");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    // the gradients of no rows are zeros
    const size_t bytes = dim * (param_kind == kValueF32 ? 4 : size);
    if (d_weight != nullptr) cudaMemsetAsync(d_weight, 0, bytes, s);
    if (d_bias != nullptr) cudaMemsetAsync(d_bias, 0, bytes, s);
    return rows_launched();
  }
  HKV_ROWS_CHECK(dy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr && dx != nullptr,
                 "dy, x, mean, rstd and dx must not be null");
  const bool sums_wanted = d_weight != nullptr || d_bias != nullptr;
  HKV_ROWS_CHECK(!sums_wanted ||
                     (work != nullptr &&
                      work_bytes >= hkv_layer_norm_backward_workspace_bytes(n, dim, value_kind)),
                 "workspace smaller than hkv_layer_norm_backward_workspace_bytes");
  NormBackwardArgs a{};
  a.n = n;
  a.dim = dim;
  a.x = x;
  a.x_stride = x_stride;
  a.dy = dy;
  a.dy_stride = dy_stride;
  a.weight = weight;
  a.params_f32 = param_kind == kValueF32;
  a.inv_dim = 1.f / float(dim);
  a.mean = mean;
  a.rstd = rstd;
  a.dx = dx;
  a.dx_stride = dx_stride;
  a.d_weight = d_weight;
  a.d_bias = d_bias;
  const uint64_t bits = dim * size | address_bits(dy) | dy_stride | address_bits(x) | x_stride |
                        address_bits(dx) | dx_stride;
  HKV_ROWS_CHECK(bits % size == 0, "a row does not start at a multiple of its element size");
  const bool whole = whole_chunks(bits | param_bits(weight, nullptr));
  const NormBackwardPlan p = plan_backward(n, dim, size);
  float* sums = sums_wanted ? static_cast<float*>(work) : nullptr;
  if (p.fits) {
    if (value_kind == kValueF32) launch_backward_type<float>(a, p, whole, sums, s);
    else if (value_kind == kValueF16) launch_backward_type<__half>(a, p, whole, sums, s);
    else launch_backward_type<__nv_bfloat16>(a, p, whole, sums, s);
  } else if (value_kind == kValueF32) {
    launch_backward_long<float>(a, p, sums, s);
  } else if (value_kind == kValueF16) {
    launch_backward_long<__half>(a, p, sums, s);
  } else {
    launch_backward_long<__nv_bfloat16>(a, p, sums, s);
  }
  if (sums_wanted) {
    if (value_kind == kValueF32) launch_reduce<float>(a, p.blocks, sums, s);
    else if (value_kind == kValueF16) launch_reduce<__half>(a, p.blocks, sums, s);
    else launch_reduce<__nv_bfloat16>(a, p.blocks, sums, s);
  }
  return rows_launched();
}

}  // extern "C"
