// The gradient of layer norm (hkv_norm.cu), from the mean and rstd it kept.
//
//   xhat = (x - mean) * rstd      g = dy * weight
//   dx = rstd * (g - sum(g) / D - xhat * sum(g * xhat) / D)
//   d_weight = sum over rows of dy * xhat        d_bias = sum over rows of dy
//
// Bound by HBM: x and dy are read and dx is written once.  Sums and products are
// 32-bit floats and every result is rounded once.
//
// The blocks stay on the device and take rows in turn: a thread sees the same
// columns of every row it touches, so the column sums d_weight and d_bias build
// up in its registers beside the row's own work.  The next rows are on their way
// into the warps' queues meanwhile, and their mean and rstd into registers (asked
// for one row ahead instead of two they cost 59 us more at 16384 x 8192 bf16).  That
// size takes 151 us, 83 % of the bandwidth of a copy (norm_reduce_kernel is 6 of them),
// bound by the instructions that a row costs its 16 warps beside the arithmetic;
// 1048576 x 64 f32 134 us, 94 %; rows past the registers, 4096 x 12288 bf16, 302 us,
// 16 %: scalar loads, and x and dy read twice.  At the
// end each block writes one row of column sums (its groups added in a fixed order),
// and norm_reduce_kernel adds the blocks' rows in a fixed order: no atomics, the same
// bits every time.  A thread's column sum is one chain over the rows of its group, n /
// (blocks * groups of a block) additions, 1771 of 262144 rows of 8192: a second level
// would need the registers that the row has.
#include "hkv_norm.cuh"

namespace hkv {

namespace {

constexpr int kColumnBlock = 256;

struct NormBackwardPlan {
  uint32_t units;    // per thread; 0: the row is too long for a block
  uint32_t group, blocks;
};

template <typename T, int BYTES, int UNITS, int WIDTH>
__global__ void __launch_bounds__(kPipeBlock, 1)
    norm_backward_kernel(const NormBackwardArgs a, const uint32_t group, const RowsIn x_in,
                         const RowsIn dy_in, float* __restrict__ sums) {
  using U = Unit<T, BYTES>;
  constexpr int kElems = U::kElems;
  constexpr bool WIDE = WIDTH >= 32;
  extern __shared__ uint4 slots[];
  float* columns = reinterpret_cast<float*>(slots);   // [copies][dim], after the last row
  __shared__ float scratch[kPipeBlock / 32][2][2];
  GroupSum<2, WIDTH> group_sum(group, scratch);
  const uint32_t n = uint32_t(a.n), dim = uint32_t(a.dim);
  const UnitMap<UNITS, WIDTH> map(group, dim / kElems);
  const RowDeal deal(group);
  const RowQueue<T, BYTES, UNITS, WIDTH> x_queue(slots, 0, 2, map);
  const RowQueue<T, BYTES, UNITS, WIDTH> dy_queue(slots, 1, 2, map);
  float w[1][UNITS][kElems], dw[UNITS][kElems], db[UNITS][kElems];
  load_params<T, BYTES>({a.weight}, a.params_f32, a.params_vec, map, dim, {1.f}, w);
#pragma unroll
  for (int c = 0; c < UNITS; ++c) {
#pragma unroll
    for (int e = 0; e < kElems; ++e) dw[c][e] = db[c][e] = 0.f;
  }
  const uint32_t step = deal.step;
  uint32_t r = deal.row;
  // the rows that are fetched next, the lower halves of the current ones' addresses,
  // and the thread's place in the row that is written, moved on from row to row
  const uint8_t *x_next = x_in.first + r * x_in.stride, *dy_next = dy_in.first + r * dy_in.stride;
  uint32_t x_current = uint32_t(reinterpret_cast<uintptr_t>(x_next));
  uint32_t dy_current = uint32_t(reinterpret_cast<uintptr_t>(dy_next));
  uint8_t* out = static_cast<uint8_t*>(a.dx) + r * a.dx_stride + (map.part + map.lane) * BYTES;
  const uint64_t x_step = step * x_in.stride, dy_step = step * dy_in.stride, out_step = step * a.dx_stride;
  auto fill = [&](uint32_t stage, uint32_t row) {
    if (row < n) {
      x_queue.fill(stage, x_next, map);
      dy_queue.fill(stage, dy_next, map);
    }
    x_next += x_step;
    dy_next += dy_step;
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
  // the lanes of a warp leave together
  for (uint32_t warp_row = deal.warp_row; warp_row < n; warp_row += step) {
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
    x_queue.arrive();
    float xhat[UNITS][kElems], g[UNITS][kElems];
    Partial gs, products;
    if (r < n) {
      const uint32_t x_from = x_queue.place(stage, x_current, map);
      const uint32_t dy_from = dy_queue.place(stage, dy_current, map);
      map.template each<kRun<BYTES, UNITS>>([&](int c, bool mine) {
        float x[kElems], dy[kElems];
        x_queue.take(x_from, c, mine, map, x);
        dy_queue.take(dy_from, c, mine, map, dy);
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
          xhat[c][e] = (x[e] - mean) * rstd;
          g[c][e] = dy[e] * w[0][c][e];
          gs.part[(c * kElems + e) % 4] += g[c][e];
          float& product = products.part[(c * kElems + e) % 4];
          product = fmaf(g[c][e], xhat[c][e], product);
          dw[c][e] = fmaf(dy[e], xhat[c][e], dw[c][e]);
          db[c][e] += dy[e];
        }
      });
    }
    x_queue.arrive();
    float sum[2] = {gs.sum(), products.sum()};
    group_sum(sum);
    // dx = rstd * (g - m0 - xhat * m1)
    const float r0 = rstd * (sum[0] * a.inv_dim), m1 = sum[1] * a.inv_dim;
    if (r < n) {
      auto* to = reinterpret_cast<typename U::Raw*>(out);
      map.template each<kRun<BYTES, UNITS>>([&](int c, bool mine) {
        float f[kElems];
#pragma unroll
        for (int e = 0; e < kElems; ++e) f[e] = fmaf(rstd, fmaf(-m1, xhat[c][e], g[c][e]), -r0);
        if (mine) to[map(c) - map.lane] = U::pack(f);
      });
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
    r += step;
    x_current += uint32_t(x_step);
    dy_current += uint32_t(dy_step);
    out += out_step;
  }
  copies_wait<0>();
  // the sums of the block's groups: those of one warp by exchange, the others
  // one after the other
  const uint32_t copies = WIDE ? blockDim.x / group : blockDim.x >> 5;
  const uint32_t copy = WIDE ? threadIdx.x / group : threadIdx.x >> 5;
  if (!WIDE) {
    for (uint32_t d = 16; d >= group; d >>= 1) {
#pragma unroll
      for (int c = 0; c < UNITS; ++c) {
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
          dw[c][e] += __shfl_xor_sync(kFull, dw[c][e], d);
          db[c][e] += __shfl_xor_sync(kFull, db[c][e], d);
        }
      }
    }
  }
  const bool writes = WIDE || (threadIdx.x & 31u) < group;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which == 0 ? a.d_weight == nullptr : a.d_bias == nullptr) continue;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < UNITS; ++c) {
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        const uint32_t column = (map.part + map(c)) * kElems + e;
        if (writes && column < dim) columns[copy * dim + column] = which == 0 ? dw[c][e] : db[c][e];
      }
    }
    __syncthreads();
    float* mine = sums + (uint64_t(which) * gridDim.x + blockIdx.x) * dim;
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
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
  GroupSum<2, kWarps> group_sum(blockDim.x, scratch);
  const uint32_t dim = uint32_t(a.dim);
  for (uint64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.x) + r * a.x_stride);
    const T* dy = reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.dy) + r * a.dy_stride);
    T* dx = reinterpret_cast<T*>(static_cast<uint8_t*>(a.dx) + r * a.dx_stride);
    const float mean = a.mean[r], rstd = a.rstd[r];
    float sum[2] = {0.f, 0.f};
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      const float w = load_param<T>(a.weight, a.params_f32, i, 1.f);
      const float g = to_float(dy[i]) * w;
      sum[0] += g;
      sum[1] = fmaf(g, (to_float(x[i]) - mean) * rstd, sum[1]);
    }
    group_sum(sum);
    const float m0 = sum[0] * a.inv_dim, m1 = sum[1] * a.inv_dim;
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      const float w = load_param<T>(a.weight, a.params_f32, i, 1.f);
      const float xhat = (to_float(x[i]) - mean) * rstd;
      dx[i] = from_float<T>(rstd * (fmaf(-m1, xhat, to_float(dy[i]) * w) - m0));
    }
  }
}

// A thread adds the rows of a column in runs of kColumnRun and then the runs' sums, so
// that of n rows no term passes more than kColumnRun + n / (64 * kColumnRun) of its
// additions.  (In one chain of n / 64 a constant of 0.1 in 262,144 rows was off by 4e-5.)
constexpr uint32_t kColumnRun = 64;
template <typename T>
__global__ void __launch_bounds__(kColumnBlock)
    norm_columns_kernel(const NormBackwardArgs a, float* __restrict__ sums) {
  const uint64_t i = uint64_t(blockIdx.x) * kColumnBlock + threadIdx.x;
  if (i >= a.dim) return;
  float dw = 0.f, db = 0.f;
  const uint64_t run = uint64_t(kColumnRun) * gridDim.y;
  for (uint64_t begin = blockIdx.y; begin < a.n; begin += run) {
    const uint64_t end = min(a.n, begin + run);
    float run_dw = 0.f, run_db = 0.f;
#pragma unroll 4
    for (uint64_t r = begin; r < end; r += gridDim.y) {
      const float d = to_float(
          reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.dy) + r * a.dy_stride)[i]);
      const float v = to_float(
          reinterpret_cast<const T*>(static_cast<const uint8_t*>(a.x) + r * a.x_stride)[i]);
      run_dw = fmaf(d, (v - a.mean[r]) * a.rstd[r], run_dw);
      run_db += d;
    }
    dw += run_dw;
    db += run_db;
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

// Units per thread that the kernel is built for: row values, weights and column
// sums of 16 elements fill the registers that 512 threads have.
const uint32_t* backward_choices(uint32_t unit, uint32_t size) {
  static const uint32_t whole2[] = {1, 2, 0}, whole4[] = {2, 3, 4, 0};
  static const uint32_t pairs[] = {4, 8, 0}, ones[] = {8, 16, 0};
  return unit == 16 ? (size == 2 ? whole2 : whole4) : unit == size ? ones : pairs;
}

NormBackwardPlan plan_backward(uint64_t n, uint64_t dim, uint32_t size, uint32_t unit) {
  NormBackwardPlan p{};
  const uint64_t units = dim * size / unit;
  p.units = fitting_units(units, unit, backward_choices(unit, size));
  if (p.units == 0) {
    p.blocks = uint32_t(n < 64 ? n : 64);   // row splits of the column sums
    return p;
  }
  p.group = group_for(units, p.units, unit);
  p.blocks = pipe_blocks(n, p.group);
  return p;
}

template <typename T, int BYTES, int UNITS, int WIDTH>
int launch_backward_pipe(const NormBackwardArgs& a, const NormBackwardPlan& p, float* sums,
                         cudaStream_t stream) {
  const size_t copies = WIDTH >= 32 ? kPipeBlock / p.group : kPipeBlock / 32;   // of the column sums
  const size_t queue = RowQueue<T, BYTES, UNITS, WIDTH>::bytes(p.group, 2);
  const size_t columns = copies * a.dim * sizeof(float);
  const size_t shared = queue > columns ? queue : columns;
  constexpr auto kKernel = norm_backward_kernel<T, BYTES, UNITS, WIDTH>;
  const int rc = allow_shared<kKernel>();
  if (rc != HKV_OK) return rc;
  kKernel<<<p.blocks, pipe_threads(p.group), shared, stream>>>(
      a, p.group, rows_in(a.x, a.x_stride), rows_in(a.dy, a.dy_stride), sums);
  return HKV_OK;
}

template <typename T, int BYTES, int UNITS>
int launch_backward_units(const NormBackwardArgs& a, const NormBackwardPlan& p, float* sums,
                          cudaStream_t stream) {
  // the widths that fitting_units() gives rows of so many units per thread
  if constexpr (BYTES != 16 || UNITS != 1) {
    if constexpr (BYTES == 16 || UNITS * Unit<T, BYTES>::kElems == 16) {
      if (p.group > 32) return launch_backward_pipe<T, BYTES, UNITS, kWarps>(a, p, sums, stream);
    }
    if (p.group == 32) return launch_backward_pipe<T, BYTES, UNITS, 32>(a, p, sums, stream);
  }
  if constexpr (BYTES == 16) return launch_backward_pipe<T, BYTES, UNITS, 0>(a, p, sums, stream);
  else if (p.group == 16) return launch_backward_pipe<T, BYTES, UNITS, 16>(a, p, sums, stream);
  else return launch_backward_pipe<T, BYTES, UNITS, 8>(a, p, sums, stream);
}

template <typename T, int BYTES>
int launch_backward_type(const NormBackwardArgs& a, const NormBackwardPlan& p, float* sums,
                         cudaStream_t stream) {
#define HKV_CALL(N) return launch_backward_units<T, BYTES, N>(a, p, sums, stream)
  if constexpr (BYTES == 16 && sizeof(T) == 2) {
    switch (p.units) {
      case 1: HKV_CALL(1);
      default: HKV_CALL(2);
    }
  } else if constexpr (BYTES == 16) {
    switch (p.units) {
      case 2: HKV_CALL(2);
      case 3: HKV_CALL(3);
      default: HKV_CALL(4);
    }
  } else if constexpr (BYTES != sizeof(T)) {
    switch (p.units) {
      case 4: HKV_CALL(4);
      default: HKV_CALL(8);
    }
  } else {
    switch (p.units) {
      case 8: HKV_CALL(8);
      default: HKV_CALL(16);
    }
  }
#undef HKV_CALL
}

template <typename T>
void launch_backward_long(const NormBackwardArgs& a, const NormBackwardPlan& p, float* sums,
                          cudaStream_t stream) {
  const uint64_t cap = uint64_t(sm_count()) * 4;
  norm_backward_long_kernel<T><<<unsigned(a.n < cap ? a.n : cap), 512, 0, stream>>>(a);
  if (sums != nullptr) {
    const dim3 grid(unsigned((a.dim + kColumnBlock - 1) / kColumnBlock), p.blocks);
    norm_columns_kernel<T><<<grid, kColumnBlock, 0, stream>>>(a, sums);
  }
}

template <typename T>
void launch_reduce(const NormBackwardArgs& a, uint32_t rows, const float* sums, cudaStream_t stream) {
  const dim3 grid(unsigned((a.dim + 31) / 32), 2);
  norm_reduce_kernel<T><<<grid, 1024, 0, stream>>>(sums, rows, a.dim, a.params_f32, a.d_weight,
                                                   a.d_bias);
}

}  // namespace
}  // namespace hkv

using namespace hkv;

extern "C" {

uint64_t hkv_layer_norm_backward_workspace_bytes(uint64_t n, uint64_t dim, uint32_t value_kind) {
  if (check_norm(n, dim, value_kind, value_kind, 0.f) != HKV_OK || n == 0) return 0;
  // the most of any unit: the rows' alignment is not known here
  const uint32_t size = row_kind_size(value_kind);
  uint32_t blocks = 0;
  for (uint32_t unit : {16u, 4u, 2u}) {
    if (unit < size || dim * size % unit != 0) continue;
    const uint32_t b = plan_backward(n, dim, size, unit).blocks;
    blocks = b > blocks ? b : blocks;
  }
  return 2ull * blocks * dim * sizeof(float);
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
  HKV_ROWS_CHECK(all_aligned(row_kind_size(param_kind), weight, d_weight, d_bias) &&
                     all_aligned(4, mean, rstd, work),
                 "a buffer does not start at a multiple of its element size, or work of 4");
  NormBackwardArgs a{};
  a.n = n;
  a.dim = dim;
  a.x = x;
  a.x_stride = x_stride;
  a.dy = dy;
  a.dy_stride = dy_stride;
  a.weight = weight;
  a.params_f32 = param_kind == kValueF32;
  a.params_vec = address_bits(weight) % 16 == 0;
  a.inv_dim = 1.f / float(dim);
  a.mean = mean;
  a.rstd = rstd;
  a.dx = dx;
  a.dx_stride = dx_stride;
  a.d_weight = d_weight;
  a.d_bias = d_bias;
  const uint64_t bits = dim * size | address_bits(dy) | dy_stride | address_bits(x) | x_stride |
                        address_bits(dx) | dx_stride;
  const uint32_t unit = unit_bytes(bits, size);
  HKV_ROWS_CHECK(unit != 0, "a row does not start at a multiple of its element size");
  const NormBackwardPlan p = plan_backward(n, dim, size, unit);
  float* sums = sums_wanted ? static_cast<float*>(work) : nullptr;
  if (p.units != 0) {
    int launched = HKV_OK;
#define HKV_CALL(T, BYTES) launched = launch_backward_type<T, BYTES>(a, p, sums, s)
    HKV_FOR_UNIT(value_kind, unit, HKV_CALL)
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
