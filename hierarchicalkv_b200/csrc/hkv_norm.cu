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
constexpr int kNormBlock = 256;

// Sum over the `group` threads of a row (a power of two: part of a warp, or
// whole warps of this block); every thread gets it.  `scratch`: one float per
// warp of the block.  With groups above a warp every thread of the block calls.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], uint32_t group, float (*scratch)[N]) {
  const uint32_t width = group < 32u ? group : 32u;
  for (uint32_t d = width >> 1; d > 0; d >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kFull, v[i], d);
  }
  if (group > 32u) {
    const uint32_t warp = threadIdx.x >> 5;
    __syncthreads();   // the previous sum has been read
    if ((threadIdx.x & 31u) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) scratch[warp][i] = v[i];
    }
    __syncthreads();
    const uint32_t first = warp & ~((group >> 5) - 1u);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    for (uint32_t w = 0; w < group >> 5; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += scratch[first + w][i];
    }
  }
}

// CHUNKS accesses of VB bytes per thread; `group` threads per row.
template <typename T, int VB, int CHUNKS>
__global__ void __launch_bounds__(1024)
    norm_kernel(const NormArgs a, const uint32_t group, const uint32_t chunks) {
  using P = Pack<T, VB>;
  __shared__ float scratch[32][1];
  const uint32_t lane = threadIdx.x & (group - 1u);
  const uint64_t r = (uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) / group;
  const uint8_t* row = nullptr;
  if (r < a.n) {
    row = a.row_ptrs != nullptr ? static_cast<const uint8_t*>(a.row_ptrs[r])
                                : static_cast<const uint8_t*>(a.x) + r * a.x_stride;
  }
  P x[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t at = lane + c * group;
    if (row != nullptr && at < chunks) {
      x[c].raw = *reinterpret_cast<const typename P::Raw*>(row + uint64_t(at) * VB);
    } else {
      x[c].raw = typename P::Raw{};
    }
  }
  const float inv_dim = a.inv_dim;
  float sum[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int e = 0; e < P::kElems; ++e) sum[0] += x[c].get(e);
  }
  group_sum<1>(sum, group, scratch);
  const float mean = sum[0] * inv_dim;
  float sq[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    if (lane + c * group < chunks) {
#pragma unroll
      for (int e = 0; e < P::kElems; ++e) {
        const float d = x[c].get(e) - mean;
        sq[0] = fmaf(d, d, sq[0]);
      }
    }
  }
  group_sum<1>(sq, group, scratch);
  if (row == nullptr) return;
  const float rstd = 1.f / sqrtf(fmaf(sq[0], inv_dim, a.eps));
  uint8_t* out = static_cast<uint8_t*>(a.y) + r * a.y_stride;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const uint32_t at = lane + c * group;
    if (at >= chunks) break;
    float w[P::kElems], b[P::kElems];
#pragma unroll
    for (int e = 0; e < P::kElems; ++e) {
      w[e] = 1.f;
      b[e] = 0.f;
    }
    if (a.weight != nullptr) load_params<T>(a.weight, a.params_f32, at * P::kElems, w);
    if (a.bias != nullptr) load_params<T>(a.bias, a.params_f32, at * P::kElems, b);
    P y;
#pragma unroll
    for (int e = 0; e < P::kElems; ++e) y.set(e, fmaf((x[c].get(e) - mean) * rstd, w[e], b[e]));
    *reinterpret_cast<typename P::Raw*>(out + uint64_t(at) * VB) = y.raw;
  }
  if (lane == 0) {
    if (a.mean != nullptr) a.mean[r] = mean;
    if (a.rstd != nullptr) a.rstd[r] = rstd;
  }
}

// Rows too long for the registers of a block: three passes over the row, which
// stays in L2 between them.
template <typename T, int VB>
__global__ void __launch_bounds__(1024)
    norm_long_kernel(const NormArgs a, const uint32_t chunks) {
  using P = Pack<T, VB>;
  __shared__ float scratch[32][1];
  for (uint64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    const uint8_t* row = a.row_ptrs != nullptr ? static_cast<const uint8_t*>(a.row_ptrs[r])
                                               : static_cast<const uint8_t*>(a.x) + r * a.x_stride;
    if (row == nullptr) continue;
    float sum[1] = {0.f};
    for (uint32_t at = threadIdx.x; at < chunks; at += blockDim.x) {
      P x;
      x.raw = *reinterpret_cast<const typename P::Raw*>(row + uint64_t(at) * VB);
#pragma unroll
      for (int e = 0; e < P::kElems; ++e) sum[0] += x.get(e);
    }
    group_sum<1>(sum, blockDim.x, scratch);
    const float mean = sum[0] * a.inv_dim;
    float sq[1] = {0.f};
    for (uint32_t at = threadIdx.x; at < chunks; at += blockDim.x) {
      P x;
      x.raw = *reinterpret_cast<const typename P::Raw*>(row + uint64_t(at) * VB);
#pragma unroll
      for (int e = 0; e < P::kElems; ++e) {
        const float d = x.get(e) - mean;
        sq[0] = fmaf(d, d, sq[0]);
      }
    }
    group_sum<1>(sq, blockDim.x, scratch);
    const float rstd = 1.f / sqrtf(fmaf(sq[0], a.inv_dim, a.eps));
    uint8_t* out = static_cast<uint8_t*>(a.y) + r * a.y_stride;
    for (uint32_t at = threadIdx.x; at < chunks; at += blockDim.x) {
      P x, y;
      x.raw = *reinterpret_cast<const typename P::Raw*>(row + uint64_t(at) * VB);
      float w[P::kElems], b[P::kElems];
#pragma unroll
      for (int e = 0; e < P::kElems; ++e) {
        w[e] = 1.f;
        b[e] = 0.f;
      }
      if (a.weight != nullptr) load_params<T>(a.weight, a.params_f32, at * P::kElems, w);
      if (a.bias != nullptr) load_params<T>(a.bias, a.params_f32, at * P::kElems, b);
#pragma unroll
      for (int e = 0; e < P::kElems; ++e) y.set(e, fmaf((x.get(e) - mean) * rstd, w[e], b[e]));
      *reinterpret_cast<typename P::Raw*>(out + uint64_t(at) * VB) = y.raw;
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
// At the end each block writes one row of column sums (its groups added in a
// fixed order), and norm_reduce_kernel adds the blocks' rows in a fixed order.

struct NormBackwardPlan {
  uint32_t group, chunks, per_thread, blocks;
  bool fits;   // a row fits the registers of a block
};

template <typename T, int VB, int CHUNKS>
__global__ void __launch_bounds__(kNormBlock)
    norm_backward_kernel(const NormBackwardArgs a, const uint32_t group, const uint32_t chunks,
                         float* __restrict__ sums) {
  using P = Pack<T, VB>;
  extern __shared__ float columns[];   // [dim]
  __shared__ float scratch[kNormBlock / 32][2];
  const uint32_t lane = threadIdx.x & (group - 1u);
  const uint32_t groups = kNormBlock / group;
  const uint32_t my_group = threadIdx.x / group;
  float dw[CHUNKS][P::kElems], db[CHUNKS][P::kElems];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int e = 0; e < P::kElems; ++e) dw[c][e] = db[c][e] = 0.f;
  }
  // every group of the block runs the same number of turns (the sums of groups
  // above a warp use block barriers)
  for (uint64_t first = uint64_t(blockIdx.x) * groups; first < a.n;
       first += uint64_t(gridDim.x) * groups) {
    const uint64_t r = first + my_group;
    const bool live = r < a.n;
    P x[CHUNKS], dy[CHUNKS];
    float mean = 0.f, rstd = 0.f;
    if (live) {
      mean = a.mean[r];
      rstd = a.rstd[r];
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const uint32_t at = lane + c * group;
      x[c].raw = dy[c].raw = typename P::Raw{};
      if (live && at < chunks) {
        x[c].raw = *reinterpret_cast<const typename P::Raw*>(static_cast<const uint8_t*>(a.x) +
                                                             r * a.x_stride + uint64_t(at) * VB);
        dy[c].raw = *reinterpret_cast<const typename P::Raw*>(static_cast<const uint8_t*>(a.dy) +
                                                              r * a.dy_stride + uint64_t(at) * VB);
      }
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const uint32_t at = lane + c * group;
      if (!live || at >= chunks) continue;
      float w[P::kElems];
#pragma unroll
      for (int e = 0; e < P::kElems; ++e) w[e] = 1.f;
      if (a.weight != nullptr) load_params<T>(a.weight, a.params_f32, at * P::kElems, w);
#pragma unroll
      for (int e = 0; e < P::kElems; ++e) {
        const float xhat = (x[c].get(e) - mean) * rstd;
        const float d = dy[c].get(e);
        const float g = d * w[e];
        sum[0] += g;
        sum[1] = fmaf(g, xhat, sum[1]);
        dw[c][e] = fmaf(d, xhat, dw[c][e]);
        db[c][e] += d;
      }
    }
    group_sum<2>(sum, group, scratch);
    if (!live) continue;
    const float m0 = sum[0] * a.inv_dim, m1 = sum[1] * a.inv_dim;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const uint32_t at = lane + c * group;
      if (at >= chunks) break;
      float w[P::kElems];
#pragma unroll
      for (int e = 0; e < P::kElems; ++e) w[e] = 1.f;
      if (a.weight != nullptr) load_params<T>(a.weight, a.params_f32, at * P::kElems, w);
      P dx;
#pragma unroll
      for (int e = 0; e < P::kElems; ++e) {
        const float xhat = (x[c].get(e) - mean) * rstd;
        dx.set(e, rstd * (dy[c].get(e) * w[e] - m0 - xhat * m1));
      }
      *reinterpret_cast<typename P::Raw*>(static_cast<uint8_t*>(a.dx) + r * a.dx_stride +
                                          uint64_t(at) * VB) = dx.raw;
    }
  }
  // the block's groups, one after the other
  const uint32_t dim = a.dim;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which == 0 ? a.d_weight == nullptr : a.d_bias == nullptr) continue;
    for (uint32_t turn = 0; turn < groups; ++turn) {
      if (turn == my_group) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const uint32_t at = lane + c * group;
          if (at >= chunks) break;
#pragma unroll
          for (int e = 0; e < P::kElems; ++e) {
            const float v = which == 0 ? dw[c][e] : db[c][e];
            float* to = columns + at * P::kElems + e;
            *to = turn == 0 ? v : *to + v;
          }
        }
      }
      __syncthreads();
    }
    float* mine = sums + (uint64_t(which) * gridDim.x + blockIdx.x) * dim;
    for (uint32_t i = threadIdx.x; i < dim; i += kNormBlock) mine[i] = columns[i];
    __syncthreads();
  }
}

// Rows too long for the registers of a block: the row's two sums and dx first,
// re-reading the row from L2, then the column sums on their own.
template <typename T>
__global__ void __launch_bounds__(512)
    norm_backward_long_kernel(const NormBackwardArgs a) {
  __shared__ float scratch[16][2];
  for (uint64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.x) + r * a.x_stride);
    const T* dy = reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.dy) + r * a.dy_stride);
    T* dx = reinterpret_cast<T*>(static_cast<uint8_t*>(a.dx) + r * a.dx_stride);
    const float mean = a.mean[r], rstd = a.rstd[r];
    float sum[2] = {0.f, 0.f};
    for (uint32_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
      float w[1] = {1.f};
      if (a.weight != nullptr) load_params<T>(a.weight, a.params_f32, i, w);
      const float g = to_float(dy[i]) * w[0];
      sum[0] += g;
      sum[1] = fmaf(g, (to_float(x[i]) - mean) * rstd, sum[1]);
    }
    group_sum<2>(sum, blockDim.x, scratch);
    const float m0 = sum[0] * a.inv_dim, m1 = sum[1] * a.inv_dim;
    for (uint32_t i = threadIdx.x; i < a.dim; i += blockDim.x) {
      float w[1] = {1.f};
      if (a.weight != nullptr) load_params<T>(a.weight, a.params_f32, i, w);
      const float xhat = (to_float(x[i]) - mean) * rstd;
      dx[i] = from_float<T>(rstd * (to_float(dy[i]) * w[0] - m0 - xhat * m1));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kNormBlock)
    norm_columns_kernel(const NormBackwardArgs a, float* __restrict__ sums) {
  const uint64_t i = uint64_t(blockIdx.x) * kNormBlock + threadIdx.x;
  if (i >= a.dim) return;
  float dw = 0.f, db = 0.f;
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

#define HKV_FOR_NORM_TYPE(kind, vb, CALL)    \
  if ((kind) == kValueF32) {                 \
    switch (vb) {                            \
      case 16: CALL(float, 16); break;       \
      default: CALL(float, 4); break;        \
    }                                        \
  } else if ((kind) == kValueF16) {          \
    switch (vb) {                            \
      case 16: CALL(__half, 16); break;      \
      case 4: CALL(__half, 4); break;        \
      default: CALL(__half, 2); break;       \
    }                                        \
  } else {                                   \
    switch (vb) {                            \
      case 16: CALL(__nv_bfloat16, 16); break; \
      case 4: CALL(__nv_bfloat16, 4); break; \
      default: CALL(__nv_bfloat16, 2); break; \
    }                                        \
  }

// 16 bytes, 4, or one element; 0 when an address is no multiple of the element.
uint32_t norm_access(uint64_t bits, uint32_t size) {
  const uint32_t v = access_bytes(bits);
  if (v < size) return 0;
  return v == 16 ? 16 : v >= 4 ? 4 : size;
}

constexpr uint32_t kMaxChunks = 8;   // accesses a thread of norm_kernel holds

template <typename T, int VB>
void launch_norm_vb(const NormArgs& a, cudaStream_t stream) {
  const uint64_t chunks = a.dim * sizeof(T) / VB;
  if (chunks > 1024ull * kMaxChunks) {
    const uint64_t cap = uint64_t(sm_count()) * 2;
    norm_long_kernel<T, VB><<<unsigned(a.n < cap ? a.n : cap), 1024, 0, stream>>>(a, uint32_t(chunks));
    return;
  }
  // four accesses per thread where the row has them, with at least two threads
  // on a row
  uint32_t group = pow2_at_least((chunks + 3) / 4);
  if (group < 2 && chunks > 1) group = 2;
  uint32_t per_thread = uint32_t((chunks + group - 1) / group);
  if (group > 1024) {
    group = 1024;
    per_thread = uint32_t((chunks + 1023) / 1024);
  }
  const uint32_t block = group > kNormBlock ? group : kNormBlock;
  const uint64_t grid = (a.n * group + block - 1) / block;
  auto kernel = per_thread <= 1   ? norm_kernel<T, VB, 1>
                : per_thread <= 2 ? norm_kernel<T, VB, 2>
                : per_thread <= 4 ? norm_kernel<T, VB, 4>
                                  : norm_kernel<T, VB, 8>;
  kernel<<<unsigned(grid), block, 0, stream>>>(a, group, uint32_t(chunks));
}

// Accesses a thread of the backward kernel holds: their column sums stay in
// registers, 16 or 32 elements' worth.
template <typename T, int VB>
constexpr int backward_chunks() {
  return VB == 16 ? 4 : 16;
}

NormBackwardPlan plan_backward(uint64_t n, uint64_t dim, uint32_t size, uint32_t vb) {
  NormBackwardPlan p{};
  const uint64_t chunks = dim * size / vb;
  const uint32_t most = vb == 16 ? 4 : 16;
  p.fits = chunks <= uint64_t(kNormBlock) * most;
  const uint64_t sms = uint64_t(sm_count());
  if (!p.fits) {
    p.blocks = uint32_t(n < 64 ? n : 64);   // row splits of the column sums
    return p;
  }
  p.chunks = uint32_t(chunks);
  p.per_thread = most;
  p.group = pow2_at_least((chunks + most - 1) / most);
  if (p.group < 2 && chunks > 1) p.group = 2;
  if (vb < 16) {
    // narrow accesses: a warp reads along the row
    const uint32_t along = pow2_at_least(chunks);
    p.group = along > 32 ? (p.group > 32 ? p.group : 32) : along;
  }
  const uint64_t groups = kNormBlock / p.group;
  const uint64_t want = (n + groups - 1) / groups;
  const uint64_t cap = sms * 2;
  p.blocks = uint32_t(want < cap ? want : cap);
  return p;
}

template <typename T, int VB>
void launch_backward_vb(const NormBackwardArgs& a, const NormBackwardPlan& p, float* sums,
                        cudaStream_t stream) {
  constexpr int kChunks = backward_chunks<T, VB>();
  norm_backward_kernel<T, VB, kChunks>
      <<<p.blocks, kNormBlock, a.dim * sizeof(float), stream>>>(a, p.group, p.chunks, sums);
}

template <typename T>
void launch_backward_long(const NormBackwardArgs& a, const NormBackwardPlan& p, float* sums,
                          cudaStream_t stream) {
  const uint64_t cap = uint64_t(sm_count()) * 4;
  norm_backward_long_kernel<T><<<unsigned(a.n < cap ? a.n : cap), 512, 0, stream>>>(a);
  if (a.d_weight != nullptr || a.d_bias != nullptr) {
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
  const uint32_t vb = norm_access(bits, size);
  HKV_ROWS_CHECK(vb != 0, "a row does not start at a multiple of its element size");
#define HKV_CALL(T, VB) launch_norm_vb<T, VB>(args, stream)
  HKV_FOR_NORM_TYPE(value_kind, vb, HKV_CALL)
#undef HKV_CALL
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
  // the most blocks any access width runs
  uint64_t rows = uint64_t(sm_count()) * 2;
  rows = rows < 64 ? 64 : rows;
  return 2 * (n < rows ? n : rows) * dim * sizeof(float);
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
  const uint32_t vb = norm_access(dim * size | address_bits(dy) | dy_stride | address_bits(x) |
                                      x_stride | address_bits(dx) | dx_stride,
                                  size);
  HKV_ROWS_CHECK(vb != 0, "a row does not start at a multiple of its element size");
  const NormBackwardPlan p = plan_backward(n, dim, size, vb);
  float* sums = static_cast<float*>(work);
  if (p.fits) {
#define HKV_CALL(T, VB) launch_backward_vb<T, VB>(a, p, sums, s)
    HKV_FOR_NORM_TYPE(value_kind, vb, HKV_CALL)
#undef HKV_CALL
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
