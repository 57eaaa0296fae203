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
constexpr int kNormBlock = 256;   // of a batch of few rows; more where a row needs more
constexpr int kPipeBlock = 512;   // of the kernels that stay on the device
constexpr int kStages = 3;        // rows of a warp's queue: one in use, two on their way

// Sum over the `group` threads of a row (a power of two: part of a warp, or
// whole warps of this block); every thread gets it.  WIDE: group >= 32.
// scratch: two floats of each value per warp, used in turn, so that one barrier
// of the group's own (named 1 + its number in the block) is enough.
template <int N, bool WIDE>
struct GroupSum {
  uint32_t group, warps, from, barrier;   // warps: of the group
  float (*scratch)[2][N];                 // [warps of the block]
  uint32_t turn = 0;

  __device__ __forceinline__ GroupSum(uint32_t group_, float (*scratch_)[2][N])
      : group(group_), warps(group_ >> 5), barrier(1u + threadIdx.x / group_), scratch(scratch_) {
    // where this lane reads when the group's warps exchange their sums
    from = WIDE ? ((threadIdx.x >> 5) & ~(warps - 1u)) + (threadIdx.x & (warps - 1u)) : 0u;
  }

  __device__ __forceinline__ void operator()(float (&v)[N]) {
    if (WIDE) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kFull, v[i], d);
      }
      if (warps == 1) return;
      if ((threadIdx.x & 31u) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) scratch[threadIdx.x >> 5][turn][i] = v[i];
      }
      asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(group) : "memory");
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = scratch[from][turn][i];
      for (uint32_t d = warps >> 1; d > 0; d >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kFull, v[i], d);
      }
      turn ^= 1u;
    } else {
      for (uint32_t d = group >> 1; d > 0; d >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kFull, v[i], d);
      }
    }
  }
};

// Where a thread's chunks lie in its row: chunk c of the thread is
// first + c * width.  A warp of a group above 32 owns consecutive chunks, so that
// neighbouring chunks are in neighbouring lanes whatever the group.
template <int CHUNKS, bool WIDE>
struct ChunkMap {
  uint32_t first, width, lane;   // lane: within the width

  __device__ __forceinline__ explicit ChunkMap(uint32_t group) {
    width = WIDE ? 32u : group;
    lane = threadIdx.x & (width - 1u);
    const uint32_t warp_in_group = WIDE ? (threadIdx.x & (group - 1u)) >> 5 : 0u;
    first = warp_in_group * 32u * CHUNKS + lane;
  }
  __device__ __forceinline__ uint32_t operator()(int c) const {
    return first + uint32_t(c) * (WIDE ? 32u : width);
  }
};

// Elements of a chunk that lie behind the row's end (only the last chunk has some).
template <typename T, int N>
__device__ __forceinline__ void clear_tail(uint32_t chunk, uint32_t chunks, uint32_t dim, float fill,
                                           float (&f)[N]) {
  if (chunk + 1 != chunks) return;
  const int have = int(dim - chunk * N);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    if (e >= have) f[e] = fill;
  }
}

// Stores the thread's chunks of a row.  At an unaligned address every aligned 16
// bytes belong to two neighbouring chunks: a lane gets its left neighbour's and
// stores the joint; only the ends of the row, and of a warp's run of it, are
// stored element by element.  The whole warp calls; row == nullptr: nothing.
template <typename T, int CHUNKS, bool WHOLE, bool WIDE>
__device__ __forceinline__ void store_row(uint8_t* row, uint32_t row_bytes, uint32_t chunks,
                                          const ChunkMap<CHUNKS, WIDE>& map,
                                          const uint4 (&y)[CHUNKS]) {
  if (WHOLE) {
    uint4* to = reinterpret_cast<uint4*>(row) + map.first;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (row != nullptr && map(c) < chunks) to[map(c) - map.first] = y[c];
    }
    return;
  }
  const int s = int(reinterpret_cast<uintptr_t>(row) & 15u), end = int(row_bytes);
  const uint32_t left = (threadIdx.x & 31u & ~(map.width - 1u)) | ((map.lane - 1u) & (map.width - 1u));
  const bool last_lane = map.lane == map.width - 1u;   // its right neighbour is in the next round
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint4 give = last_lane && c > 0 ? y[c > 0 ? c - 1 : 0] : y[c];
    uint4 prev;
    prev.x = __shfl_sync(kFull, give.x, left);
    prev.y = __shfl_sync(kFull, give.y, left);
    prev.z = __shfl_sync(kFull, give.z, left);
    prev.w = __shfl_sync(kFull, give.w, left);
    const int off = int(map(c) * 16u);
    if (row == nullptr || map(c) > chunks) continue;
    // the left neighbour's bytes are here, but for the first lane of the run
    const int from = map.lane != 0 || c > 0 ? 0 : off;
    store_chunk<sizeof(T)>(row, off - s, s == 0 ? y[c] : shifted(prev, y[c], 16u - s), from, end);
    if (c == CHUNKS - 1 && last_lane && s != 0) {
      // the end of the warp's run: nobody joins this chunk's last bytes
      store_chunk<sizeof(T)>(row, off - s + 16, shifted(y[c], make_uint4(0, 0, 0, 0), 16u - s), 0,
                             off + 16 < end ? off + 16 : end);
    }
  }
}

// A warp's queue of rows in shared memory, filled ahead with asynchronous copies
// that hold no registers.  The slots belong to the warp alone: no barrier of the
// block is needed, and of the warp only for unaligned rows.  A slot holds an
// aligned chunk; unaligned rows have one more chunk per row (of the warp's part of
// the row), and a thread cuts its chunks out of neighbouring slots.
template <typename T, int CHUNKS, bool WHOLE, bool WIDE>
struct RowQueue {
  using Map = ChunkMap<CHUNKS, WIDE>;
  uint32_t mine;         // shared address of this lane's slot 0 (WHOLE) or of its row's first
  uint32_t stage_bytes;  // distance of a warp's stages
  uint32_t row_bytes;
  uint32_t chunks;

  // `shared`: kStages * operands * warps * slots_per_warp slots; operand: which
  // of the row's matrices this queue holds
  __device__ __forceinline__ RowQueue(const uint4* shared, uint32_t operand, uint32_t operands,
                                      const Map& map, uint32_t row_bytes_, uint32_t chunks_)
      : row_bytes(row_bytes_), chunks(chunks_) {
    const uint32_t warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t slots = slots_per_warp(map.width);
    stage_bytes = operands * warps * slots * 16u;
    mine = static_cast<uint32_t>(__cvta_generic_to_shared(shared)) +
           (operand * warps + warp) * slots * 16u +
           (WHOLE ? lane : (lane / map.width) * (map.width * CHUNKS + 1u)) * 16u;
  }
  static __host__ __device__ __forceinline__ uint32_t slots_per_warp(uint32_t width) {
    return WHOLE ? 32u * CHUNKS : 32u * CHUNKS + 32u / width;
  }

  // Puts a row (null: none) into a stage.
  __device__ __forceinline__ void fill(uint32_t stage, const uint8_t* row, const Map& map,
                                       const uint8_t* first, const uint8_t* last) const {
    if (row == nullptr) return;
    const uint32_t to = mine + stage * stage_bytes;
    if (WHOLE) {
      const uint8_t* from = row + map.first * 16u;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        if (map(c) < chunks) copy_async(to + c * 512u, from + (map(c) - map.first) * 16u);
      }
    } else {
      const int s = int(reinterpret_cast<uintptr_t>(row) & 15u), end = int(row_bytes);
      const uint8_t* aligned = row - s;
      const bool inside = aligned >= first && row + row_bytes + 16 <= last;   // not at the matrix's ends
#pragma unroll
      for (int c = 0; c <= CHUNKS; ++c) {
        if (c == CHUNKS && map.lane != 0) break;
        const int off = int(map(c) * 16u);
        if (off - s >= end) break;
        const uint8_t* a = aligned + off;
        const uint32_t slot = to + (c * map.width + map.lane) * 16u;
        if (inside || (a >= first && a + 16 <= last)) {
          copy_async(slot, a);
        } else {
          const uint4 v = pieces<sizeof(T)>(a, row, row + row_bytes);
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(slot), "r"(v.x), "r"(v.y),
                       "r"(v.z), "r"(v.w)
                       : "memory");
        }
      }
    }
  }

  static __device__ __forceinline__ uint4 slot_at(uint32_t address) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(address)
                 : "memory");
    return v;
  }

  // Chunk c of the thread of the row in a stage, as floats; zeros where there is none.
  __device__ __forceinline__ void take(uint32_t stage, int c, const uint8_t* row, const Map& map,
                                       uint32_t dim, float (&f)[kChunkElems<T>]) const {
    uint4 v = make_uint4(0, 0, 0, 0);
    const uint32_t from = mine + stage * stage_bytes;
    if (row != nullptr && map(c) < chunks) {
      if (WHOLE) {
        v = slot_at(from + c * 512u);
      } else {
        const uint32_t s = uint32_t(reinterpret_cast<uintptr_t>(row)) & 15u;
        const uint32_t slot = from + (c * map.width + map.lane) * 16u;
        v = slot_at(slot);
        if (s != 0) v = shifted(v, slot_at(slot + 16u), s);
      }
    }
    unpack<T>(v, f);
    if (!WHOLE) clear_tail<T>(map(c), chunks, dim, 0.f, f);
  }
};

// Weights or biases of a chunk's columns; `none` where there is no pointer or no
// column.  vec: the address is a multiple of 16 (of the columns, only the last
// chunk's may be part of a chunk).
template <typename T, int N>
__device__ __forceinline__ void load_params(const void* p, bool f32, bool vec, uint32_t column,
                                            uint32_t dim, float none, float (&out)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) out[e] = none;
  if (p == nullptr) return;
  if constexpr (N == kChunkElems<T>) {
    if (vec && column + N <= dim) {
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
        unpack<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p) + column)), out);
      }
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    if (column + e < dim) {
      out[e] = f32 ? static_cast<const float*>(p)[column + e]
                   : to_float(static_cast<const T*>(p)[column + e]);
    }
  }
}

// Normalises the row whose elements are in x and stores it; row == nullptr: none.
// w, b: the thread's columns of weight and bias.
template <typename T, int CHUNKS, bool WHOLE, bool WIDE>
__device__ __forceinline__ void norm_row(const NormArgs& a, uint32_t r, const uint8_t* row,
                                         uint32_t chunks, const ChunkMap<CHUNKS, WIDE>& map,
                                         GroupSum<1, WIDE>& group_sum,
                                         float (&x)[CHUNKS][kChunkElems<T>],
                                         const float (&w)[CHUNKS][kChunkElems<T>],
                                         const float (&b)[CHUNKS][kChunkElems<T>]) {
  constexpr int kElems = kChunkElems<T>;
  const uint32_t dim = uint32_t(a.dim);
  float sum[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int e = 0; e < kElems; ++e) sum[0] += x[c][e];
  }
  group_sum(sum);
  const float mean = sum[0] * a.inv_dim;
  float sq[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    if (map(c) < chunks) {
      if (!WHOLE) clear_tail<T>(map(c), chunks, dim, mean, x[c]);
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        x[c][e] -= mean;
        sq[0] = fmaf(x[c][e], x[c][e], sq[0]);
      }
    }
  }
  group_sum(sq);
  const float rstd = rsqrtf(fmaf(sq[0], a.inv_dim, a.eps));
  uint4 y[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int e = 0; e < kElems; ++e) x[c][e] = fmaf(x[c][e] * rstd, w[c][e], b[c][e]);
    y[c] = pack<T>(x[c]);
  }
  uint8_t* to = row == nullptr ? nullptr : static_cast<uint8_t*>(a.y) + r * a.y_stride;
  store_row<T, CHUNKS, WHOLE, WIDE>(to, dim * uint32_t(sizeof(T)), chunks, map, y);
  if (row != nullptr && map.first == 0) {
    if (a.mean != nullptr) a.mean[r] = mean;
    if (a.rstd != nullptr) a.rstd[r] = rstd;
  }
}

template <typename T, int CHUNKS, bool WIDE>
__device__ __forceinline__ void load_norm_params(const NormArgs& a, uint32_t chunks,
                                                 const ChunkMap<CHUNKS, WIDE>& map,
                                                 float (&w)[CHUNKS][kChunkElems<T>],
                                                 float (&b)[CHUNKS][kChunkElems<T>]) {
  const uint32_t dim = uint32_t(a.dim);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t column = map(c) < chunks ? map(c) * kChunkElems<T> : dim;
    load_params<T>(a.weight, a.params_f32, a.params_vec, column, dim, 1.f, w[c]);
    load_params<T>(a.bias, a.params_f32, a.params_vec, column, dim, 0.f, b[c]);
  }
}

// Few rows: one per group of `group` threads, CHUNKS chunks per thread.  The
// weights are on their way while the row is reduced.
template <typename T, int CHUNKS, bool WHOLE, bool WIDE>
__global__ void __launch_bounds__(1024)
    norm_kernel(const NormArgs a, const uint32_t group, const uint32_t chunks, const RowsIn in) {
  __shared__ float scratch[32][2][1];
  const uint32_t r = uint32_t((uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) / group);
  const ChunkMap<CHUNKS, WIDE> map(group);
  const uint32_t dim = uint32_t(a.dim), row_bytes = dim * uint32_t(sizeof(T));
  const uint8_t *row = nullptr, *first = in.first, *last = in.last;
  if (r < a.n) {
    if (a.row_ptrs != nullptr) {
      row = first = static_cast<const uint8_t*>(a.row_ptrs[r]);
      last = row + row_bytes;
    } else {
      row = in.first + r * in.stride;
    }
  }
  float x[CHUNKS][kChunkElems<T>], w[CHUNKS][kChunkElems<T>], b[CHUNKS][kChunkElems<T>];
  Cut cut[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    cut[c].none();
    if (row != nullptr && map(c) < chunks) {
      if (WHOLE) cut[c].lo = __ldg(reinterpret_cast<const uint4*>(row) + map(c));
      else cut[c].load(row + map(c) * 16u, first, last);
    }
  }
  load_norm_params<T, CHUNKS, WIDE>(a, chunks, map, w, b);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint8_t* p = row + map(c) * 16u;
    unpack<T>(WHOLE ? cut[c].lo : cut[c].template get<sizeof(T)>(p, row, row + row_bytes), x[c]);
    if (!WHOLE) clear_tail<T>(map(c), chunks, dim, 0.f, x[c]);
  }
  GroupSum<1, WIDE> group_sum(group, scratch);
  norm_row<T, CHUNKS, WHOLE, WIDE>(a, r, row, chunks, map, group_sum, x, w, b);
}

// Many rows: the blocks stay on the device, their threads keep the weights of
// their columns, and their groups take rows in turn out of the warps' queues.
template <typename T, int CHUNKS, bool WHOLE, bool WIDE>
__global__ void __launch_bounds__(kPipeBlock, 1)
    norm_pipe_kernel(const NormArgs a, const uint32_t group, const uint32_t chunks, const RowsIn in) {
  extern __shared__ uint4 slots[];
  __shared__ float scratch[kPipeBlock / 32][2][1];
  GroupSum<1, WIDE> group_sum(group, scratch);
  const ChunkMap<CHUNKS, WIDE> map(group);
  const uint32_t n = uint32_t(a.n), dim = uint32_t(a.dim), row_bytes = dim * uint32_t(sizeof(T));
  const RowQueue<T, CHUNKS, WHOLE, WIDE> queue(slots, 0, 1, map, row_bytes, chunks);
  float w[CHUNKS][kChunkElems<T>], b[CHUNKS][kChunkElems<T>];
  load_norm_params<T, CHUNKS, WIDE>(a, chunks, map, w, b);
  const uint32_t step = gridDim.x * (kPipeBlock / group);
  uint32_t r = blockIdx.x * (kPipeBlock / group) + threadIdx.x / group;
  auto address = [&](uint32_t row) -> const uint8_t* {
    if (row >= n) return nullptr;
    return a.row_ptrs != nullptr ? static_cast<const uint8_t*>(a.row_ptrs[row])
                                 : in.first + row * in.stride;
  };
  auto fill = [&](uint32_t stage, const uint8_t* row) {
    const bool by_address = a.row_ptrs != nullptr;
    queue.fill(stage, row, map, by_address ? row : in.first, by_address ? row + row_bytes : in.last);
    copies_commit();
  };
  // rows[0]: the current row, rows[1 ...]: those in the queue, rows[kStages]: the
  // one whose address has arrived by the time its copies start
  const uint8_t* rows[kStages + 1];
#pragma unroll
  for (int i = 0; i < kStages; ++i) rows[i + 1] = address(r + i * step);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fill(i, rows[i + 1]);
  uint32_t stage = 0;
  // the lanes of a warp leave together: when the row of its first group is past the end
  for (uint32_t warp_row = r - (WIDE ? 0u : (threadIdx.x & 31u) / group); warp_row < n;
       warp_row += step, r += step) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) rows[i] = rows[i + 1];
    fill(stage == 0 ? kStages - 1 : stage - 1, rows[kStages - 1]);
    rows[kStages] = address(r + kStages * step);
    copies_wait<kStages - 1>();
    if (!WHOLE) __syncwarp();
    float x[CHUNKS][kChunkElems<T>];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) queue.take(stage, c, rows[0], map, dim, x[c]);
    if (!WHOLE) __syncwarp();   // the slots are free again
    norm_row<T, CHUNKS, WHOLE, WIDE>(a, r, rows[0], chunks, map, group_sum, x, w, b);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  copies_wait<0>();
}

// Rows too long for the registers of a block: three passes over the row, which
// stays in L2 between them.
template <typename T>
__global__ void __launch_bounds__(1024)
    norm_long_kernel(const NormArgs a) {
  __shared__ float scratch[32][2][1];
  GroupSum<1, true> group_sum(blockDim.x, scratch);
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
    const float rstd = rsqrtf(fmaf(sq[0], a.inv_dim, a.eps));
    T* out = reinterpret_cast<T*>(static_cast<uint8_t*>(a.y) + r * a.y_stride);
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      float w[1], b[1];
      load_params<T>(a.weight, a.params_f32, false, i, dim, 1.f, w);
      load_params<T>(a.bias, a.params_f32, false, i, dim, 0.f, b);
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
// The next rows are on their way into the warps' queues meanwhile.
// At the end each block writes one row of column sums (its groups added in a
// fixed order), and norm_reduce_kernel adds the blocks' rows in a fixed order.

struct NormBackwardPlan {
  uint32_t group, chunks, per_thread, blocks;
  bool fits;   // a row fits the registers of a block
};

template <typename T, int CHUNKS, bool WHOLE, bool WIDE>
__global__ void __launch_bounds__(kPipeBlock, 1)
    norm_backward_kernel(const NormBackwardArgs a, const uint32_t group, const uint32_t chunks,
                         const RowsIn x_in, const RowsIn dy_in, float* __restrict__ sums) {
  constexpr int kElems = kChunkElems<T>;
  extern __shared__ uint4 slots[];
  float* columns = reinterpret_cast<float*>(slots);   // [copies][dim], after the last row
  __shared__ float scratch[kPipeBlock / 32][2][2];
  GroupSum<2, WIDE> group_sum(group, scratch);
  const ChunkMap<CHUNKS, WIDE> map(group);
  const uint32_t n = uint32_t(a.n), dim = uint32_t(a.dim), row_bytes = dim * uint32_t(sizeof(T));
  const uint32_t groups = kPipeBlock / group;
  const RowQueue<T, CHUNKS, WHOLE, WIDE> x_queue(slots, 0, 2, map, row_bytes, chunks);
  const RowQueue<T, CHUNKS, WHOLE, WIDE> dy_queue(slots, 1, 2, map, row_bytes, chunks);
  float w[CHUNKS][kElems], dw[CHUNKS][kElems], db[CHUNKS][kElems];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int e = 0; e < kElems; ++e) dw[c][e] = db[c][e] = 0.f;
    load_params<T>(a.weight, a.params_f32, a.params_vec, map(c) < chunks ? map(c) * kElems : dim, dim,
                   1.f, w[c]);
  }
  const uint32_t step = gridDim.x * groups;
  uint32_t r = blockIdx.x * groups + threadIdx.x / group;
  auto x_row = [&](uint32_t row) { return row < n ? x_in.first + row * x_in.stride : nullptr; };
  auto dy_row = [&](uint32_t row) { return row < n ? dy_in.first + row * dy_in.stride : nullptr; };
  auto fill = [&](uint32_t stage, uint32_t row) {
    x_queue.fill(stage, x_row(row), map, x_in.first, x_in.last);
    dy_queue.fill(stage, dy_row(row), map, dy_in.first, dy_in.last);
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fill(i, r + i * step);
  // of the rows in the queue, the current one's first
  float means[kStages], rstds[kStages];
#pragma unroll
  for (int i = 0; i < kStages; ++i) {
    means[i] = i > 0 && r + (i - 1) * step < n ? __ldg(a.mean + r + (i - 1) * step) : 0.f;
    rstds[i] = i > 0 && r + (i - 1) * step < n ? __ldg(a.rstd + r + (i - 1) * step) : 0.f;
  }
  uint32_t stage = 0;
  // the lanes of a warp leave together: when the row of its first group is past the end
  for (uint32_t warp_row = r - (WIDE ? 0u : (threadIdx.x & 31u) / group); warp_row < n;
       warp_row += step, r += step) {
    fill(stage == 0 ? kStages - 1 : stage - 1, r + (kStages - 1) * step);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      means[i] = means[i + 1];
      rstds[i] = rstds[i + 1];
    }
    const uint32_t ahead = r + (kStages - 1) * step;
    means[kStages - 1] = ahead < n ? __ldg(a.mean + ahead) : 0.f;
    rstds[kStages - 1] = ahead < n ? __ldg(a.rstd + ahead) : 0.f;
    const float mean = means[0], rstd = rstds[0];
    copies_wait<kStages - 1>();
    if (!WHOLE) __syncwarp();
    float xhat[CHUNKS][kElems], g[CHUNKS][kElems];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float x[kElems], dy[kElems];
      x_queue.take(stage, c, x_row(r), map, dim, x);
      dy_queue.take(stage, c, dy_row(r), map, dim, dy);
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        xhat[c][e] = (x[e] - mean) * rstd;
        g[c][e] = dy[e] * w[c][e];
        sum[0] += g[c][e];
        sum[1] = fmaf(g[c][e], xhat[c][e], sum[1]);
        dw[c][e] = fmaf(dy[e], xhat[c][e], dw[c][e]);
        db[c][e] += dy[e];
      }
    }
    if (!WHOLE) __syncwarp();   // the slots are free again
    group_sum(sum);
    // dx = rstd * (g - m0 - xhat * m1)
    const float r0 = rstd * (sum[0] * a.inv_dim), m1 = sum[1] * a.inv_dim;
    uint4 dx[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float f[kElems];
#pragma unroll
      for (int e = 0; e < kElems; ++e) f[e] = fmaf(rstd, fmaf(-m1, xhat[c][e], g[c][e]), -r0);
      dx[c] = pack<T>(f);
    }
    store_row<T, CHUNKS, WHOLE, WIDE>(r < n ? static_cast<uint8_t*>(a.dx) + r * a.dx_stride : nullptr,
                                      row_bytes, chunks, map, dx);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  copies_wait<0>();
  // the sums of the block's groups: those of one warp by exchange, the others
  // one after the other
  const uint32_t copies = group < 32u ? kPipeBlock / 32 : groups;
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
    for (uint32_t i = threadIdx.x; i < dim; i += kPipeBlock) {
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
  GroupSum<2, true> group_sum(blockDim.x, scratch);
  const uint32_t dim = uint32_t(a.dim);
  for (uint64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.x) + r * a.x_stride);
    const T* dy = reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.dy) + r * a.dy_stride);
    T* dx = reinterpret_cast<T*>(static_cast<uint8_t*>(a.dx) + r * a.dx_stride);
    const float mean = a.mean[r], rstd = a.rstd[r];
    float sum[2] = {0.f, 0.f};
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      float w[1];
      load_params<T>(a.weight, a.params_f32, false, i, dim, 1.f, w);
      const float g = to_float(dy[i]) * w[0];
      sum[0] += g;
      sum[1] = fmaf(g, (to_float(x[i]) - mean) * rstd, sum[1]);
    }
    group_sum(sum);
    const float m0 = sum[0] * a.inv_dim, m1 = sum[1] * a.inv_dim;
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      float w[1];
      load_params<T>(a.weight, a.params_f32, false, i, dim, 1.f, w);
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

// A kernel that needs more shared memory than the default.
template <typename Kernel>
int allow_shared(Kernel kernel, size_t bytes) {
  if (bytes <= 40 * 1024) return HKV_OK;   // the kernels' static part comes on top
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  if (e == cudaSuccess) return HKV_OK;
  cudaGetLastError();
  return rows_fail(HKV_ERR_CUDA, cudaGetErrorString(e));
}

template <typename T, bool WHOLE, bool WIDE>
int launch_norm_pipe(const NormArgs& a, uint32_t group, uint32_t chunks, const RowsIn& in,
                     cudaStream_t stream) {
  auto kernel = norm_pipe_kernel<T, 4, WHOLE, WIDE>;
  const size_t shared = size_t(kStages) * (kPipeBlock / 32) *
                        RowQueue<T, 4, WHOLE, WIDE>::slots_per_warp(group < 32 ? group : 32) * 16;
  const int rc = allow_shared(kernel, shared);
  if (rc != HKV_OK) return rc;
  const uint64_t want = (a.n * group + kPipeBlock - 1) / kPipeBlock, cap = uint64_t(sm_count());
  kernel<<<unsigned(want < cap ? want : cap), kPipeBlock, shared, stream>>>(a, group, chunks, in);
  return HKV_OK;
}

template <typename T, int CHUNKS>
void launch_norm_few(const NormArgs& a, bool whole, uint32_t group, uint32_t chunks, const RowsIn& in,
                     cudaStream_t stream) {
  const uint32_t block = group > kNormBlock ? group : kNormBlock;
  const unsigned grid = unsigned((a.n * group + block - 1) / block);
  auto kernel = group >= 32 ? (whole ? norm_kernel<T, CHUNKS, true, true> : norm_kernel<T, CHUNKS, false, true>)
                            : (whole ? norm_kernel<T, CHUNKS, true, false> : norm_kernel<T, CHUNKS, false, false>);
  kernel<<<grid, block, 0, stream>>>(a, group, chunks, in);
}

// Threads on a row that hold `per_thread` chunks each.  Two at least: they share a
// sector of 32 bytes, and a queue for rows of single threads would not fit.
uint32_t group_for(uint64_t chunks, uint32_t per_thread) {
  const uint32_t group = pow2_at_least((chunks + per_thread - 1) / per_thread);
  return group < 2 ? 2 : group;
}

template <typename T>
int launch_norm_type(const NormArgs& a, bool whole, cudaStream_t stream) {
  const uint64_t chunks = chunks_of(a.dim * sizeof(T));
  if (chunks > 4ull * kPipeBlock) {
    const uint64_t cap = uint64_t(sm_count()) * 2;
    norm_long_kernel<T><<<unsigned(a.n < cap ? a.n : cap), 1024, 0, stream>>>(a);
    return HKV_OK;
  }
  const RowsIn in = a.row_ptrs != nullptr ? RowsIn{} : rows_in(a.x, a.n, a.x_stride, a.dim * sizeof(T));
  const uint32_t count = uint32_t(chunks);
  uint32_t group = group_for(chunks, 4);
  // more than two rows for every group that the device holds: they are worth a queue
  if (a.n * group > uint64_t(sm_count()) * kPipeBlock * 2) {
    if (group >= 32) {
      return whole ? launch_norm_pipe<T, true, true>(a, group, count, in, stream)
                   : launch_norm_pipe<T, false, true>(a, group, count, in, stream);
    }
    return whole ? launch_norm_pipe<T, true, false>(a, group, count, in, stream)
                 : launch_norm_pipe<T, false, false>(a, group, count, in, stream);
  }
  // few: as many threads on a row as it has chunks for
  if (chunks > 1024) launch_norm_few<T, 2>(a, whole, group_for(chunks, 2), count, in, stream);
  else launch_norm_few<T, 1>(a, whole, group_for(chunks, 1), count, in, stream);
  return HKV_OK;
}

// Chunks a thread of the backward kernel holds: 16 elements' column sums, row
// values and weights fill the registers that 512 threads have.
constexpr uint32_t backward_chunks(uint32_t size) { return size == 4 ? 4 : 2; }

NormBackwardPlan plan_backward(uint64_t n, uint64_t dim, uint32_t size) {
  NormBackwardPlan p{};
  const uint64_t chunks = chunks_of(dim * size);
  p.per_thread = backward_chunks(size);
  p.fits = chunks <= uint64_t(kPipeBlock) * p.per_thread;
  if (!p.fits) {
    p.blocks = uint32_t(n < 64 ? n : 64);   // row splits of the column sums
    return p;
  }
  p.chunks = uint32_t(chunks);
  p.group = group_for(chunks, p.per_thread);
  const uint64_t groups = kPipeBlock / p.group;
  const uint64_t want = (n + groups - 1) / groups;
  const uint64_t cap = uint64_t(sm_count());
  p.blocks = uint32_t(want < cap ? want : cap);
  return p;
}

template <typename T, bool WHOLE, bool WIDE>
int launch_backward_pipe(const NormBackwardArgs& a, const NormBackwardPlan& p, float* sums,
                         cudaStream_t stream) {
  constexpr int kChunks = backward_chunks(sizeof(T));
  const uint64_t row_bytes = a.dim * sizeof(T);
  const size_t copies = p.group < 32 ? kPipeBlock / 32 : kPipeBlock / p.group;
  const size_t queue = size_t(kStages) * 2 * (kPipeBlock / 32) * 16 *
                       RowQueue<T, kChunks, WHOLE, WIDE>::slots_per_warp(p.group < 32 ? p.group : 32);
  const size_t columns = copies * a.dim * sizeof(float);
  const size_t shared = queue > columns ? queue : columns;
  auto kernel = norm_backward_kernel<T, kChunks, WHOLE, WIDE>;
  const int rc = allow_shared(kernel, shared);
  if (rc != HKV_OK) return rc;
  kernel<<<p.blocks, kPipeBlock, shared, stream>>>(
      a, p.group, p.chunks, rows_in(a.x, a.n, a.x_stride, row_bytes),
      rows_in(a.dy, a.n, a.dy_stride, row_bytes), sums);
  return HKV_OK;
}

template <typename T>
int launch_backward_type(const NormBackwardArgs& a, const NormBackwardPlan& p, bool whole, float* sums,
                         cudaStream_t stream) {
  if (p.group >= 32) {
    return whole ? launch_backward_pipe<T, true, true>(a, p, sums, stream)
                 : launch_backward_pipe<T, false, true>(a, p, sums, stream);
  }
  return whole ? launch_backward_pipe<T, true, false>(a, p, sums, stream)
               : launch_backward_pipe<T, false, false>(a, p, sums, stream);
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
  const bool whole = whole_chunks(bits);
  const int rc = value_kind == kValueF32   ? launch_norm_type<float>(args, whole, stream)
                 : value_kind == kValueF16 ? launch_norm_type<__half>(args, whole, stream)
                                           : launch_norm_type<__nv_bfloat16>(args, whole, stream);
  return rc != HKV_OK ? rc : rows_launched();
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
  a.params_vec = whole_chunks(address_bits(weight) | address_bits(bias));
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
  a.params_vec = whole_chunks(address_bits(weight) | address_bits(bias));
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
  a.params_vec = whole_chunks(address_bits(weight));
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
  const bool whole = whole_chunks(bits);
  const NormBackwardPlan p = plan_backward(n, dim, size);
  float* sums = sums_wanted ? static_cast<float*>(work) : nullptr;
  if (p.fits) {
#define HKV_CALL(T) launch_backward_type<T>(a, p, whole, sums, s)
    const int launched = value_kind == kValueF32   ? HKV_CALL(float)
                         : value_kind == kValueF16 ? HKV_CALL(__half)
                                                   : HKV_CALL(__nv_bfloat16);
#undef HKV_CALL
    if (launched != HKV_OK) return launched;
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
