// Layer norm of rows.
//
//   mean = sum(x) / D    rstd = 1 / sqrt(sum((x - mean)^2) / D + eps)
//   y = (x - mean) * rstd * weight + bias
//
// Bound by HBM: every row is read and written once.  A row stays in registers
// between its reduction and its use.  Statistics, sums and products are 32-bit
// floats, and every result is rounded once.  The variance is the sum of squared
// distances from the mean, not of squares.  The mean itself is rounded (a sum times a
// rounded 1 / D), by up to a few 2^-24 of |x|, which counts as much as the deviations
// are smaller than the mean: 1000 elements of 30000 would come out as -0.53 instead of
// 0.  So where the mean lies more than 8 deviations from zero, the mean of the
// distances is taken off them and their squares are summed again, after which the
// distances are as exact as those of a row about zero.  Other rows do not pay for it
// (the test costs 0 - 5 %, summing the distances of every row up to 15 %: 16384 x 8192
// bf16 91 us without either, 94 and 104; 300000 x 100 half 37, 38 and 42; with far rows
// only, 135 us at 16384 x 8192 bf16).
// Measured, us, and the share of the bandwidth of a copy: 1048576 x 64 f32 98, 87 %
// (by address with a tenth missing 80, 95 %); 16384 x 8192 bf16 94, 89 %; rows in
// narrow units, which are bound by their instructions: 65536 x 1001 bf16 50, 82 %,
// 65537 x 333 half 25, 55 %; rows past the registers, in scalar loads: 4096 x 12288 f32
// 191, 33 %.  (The comparisons beside the code below were taken before the means of far
// rows were corrected, but for that of rows by address.)
//
// Rows are given by base and stride, or (the pointer form) by one address per
// row, as find* returns them: rows are then normalised straight from where the
// table keeps them, rows in pinned host memory included, and the output rows of
// misses (null addresses) are left as they are, as find leaves them.  So are those
// of addresses that the row's length does not allow: a row of whole 16-byte (else
// 4-byte) units starts at a multiple of the unit, as the table's rows do, and the
// host cannot see the addresses to refuse them.
//
// The reference has no such operator; what it hands to one are the rows of
// find (include/merlin_hashtable.cuh:2464-2577) and find* (2729-2787).
#include "hkv_norm.cuh"

namespace hkv {

namespace {

constexpr int kNormBlock = 256;   // of a batch of few rows; more where a row needs more

__device__ __forceinline__ const uint8_t* valid_row(const NormArgs& a, const void* row) {
  return (reinterpret_cast<uintptr_t>(row) & a.row_mask) != 0 ? nullptr : static_cast<const uint8_t*>(row);
}

// Rows whose mean lies more than 8 deviations from zero: the mean is corrected.
__device__ __forceinline__ bool is_far(float mean, float rstd) { return fabsf(mean) * rstd > 8.f; }

// Normalises the row whose elements are in x, and whose sum over the thread's is
// `sum`, and stores it from `out` on, the thread's first unit; has: there is such a
// row.  w, b: the thread's columns of weight and bias.
template <typename T, int BYTES, int UNITS, int WIDTH>
__device__ __forceinline__ void norm_row(const NormArgs& a, uint32_t r, bool has, uint8_t* out, float sum,
                                         const UnitMap<UNITS, WIDTH>& map,
                                         GroupSum<1, WIDTH>& group_sum,
                                         float (&x)[UNITS][Unit<T, BYTES>::kElems],
                                         const float (&w)[UNITS][Unit<T, BYTES>::kElems],
                                         const float (&b)[UNITS][Unit<T, BYTES>::kElems]) {
  using U = Unit<T, BYTES>;
  float total[1] = {sum};
  group_sum(total);
  float mean = total[0] * a.inv_dim;
  // takes `off` from the elements; the mean of their squares
  auto centre = [&](float off) {
    Partial squares;
    if (has) {
      map.template each<kRun<BYTES, UNITS>>([&](int c, bool mine) {
#pragma unroll
        for (int e = 0; e < U::kElems; ++e) {
          x[c][e] -= off;
          if (mine) {
            float& sq = squares.part[(c * U::kElems + e) % 4];
            sq = fmaf(x[c][e], x[c][e], sq);
          }
        }
      });
    }
    float sq[1] = {squares.sum()};
    group_sum(sq);
    return rsqrtf(fmaf(sq[0], a.inv_dim, a.eps));
  };
  float rstd = centre(mean);
  // uniform over the threads of a row; the rows of a warp go together, and those that
  // lie near have 0 taken off, so that no row's bits depend on its neighbours'
  const bool far = is_far(mean, rstd);
  if (WIDTH >= 32 ? far : __any_sync(kFull, far) != 0) {
    Partial rests;
    if (has) {
      map.template each<kRun<BYTES, UNITS>>([&](int c, bool mine) {
#pragma unroll
        for (int e = 0; e < U::kElems; ++e) {
          if (mine) rests.part[(c * U::kElems + e) % 4] += x[c][e];
        }
      });
    }
    float rest[1] = {rests.sum()};
    group_sum(rest);
    const float off = far ? rest[0] * a.inv_dim : 0.f;
    mean += off;
    rstd = centre(off);
  }
  if (!has) return;
  auto* to = reinterpret_cast<typename U::Raw*>(out);
  map.template each<kRun<BYTES, UNITS>>([&](int c, bool mine) {
#pragma unroll
    for (int e = 0; e < U::kElems; ++e) x[c][e] = fmaf(x[c][e] * rstd, w[c][e], b[c][e]);
    if (mine) to[map(c) - map.lane] = U::pack(x[c]);
  });
  if (map.part + map.lane == 0) {
    if (a.mean != nullptr) a.mean[r] = mean;
    if (a.rstd != nullptr) a.rstd[r] = rstd;
  }
}

// Few rows: one per group of threads.  The weights are on their way while the row
// is reduced.
template <typename T, int BYTES, int UNITS, int WIDTH>
__global__ void __launch_bounds__(1024)
    norm_kernel(const NormArgs a, const uint32_t group, const RowsIn in) {
  using U = Unit<T, BYTES>;
  __shared__ float scratch[32][2][1];
  const uint32_t r = blockIdx.x * (blockDim.x / group) + threadIdx.x / group;
  const UnitMap<UNITS, WIDTH> map(group, uint32_t(a.dim) / U::kElems);
  const uint8_t* row = nullptr;
  if (r < a.n) {
    row = a.row_ptrs != nullptr ? valid_row(a, a.row_ptrs[r]) : in.first + r * in.stride;
  }
  typename U::Raw raw[UNITS];
#pragma unroll
  for (int c = 0; c < UNITS; ++c) {
    raw[c] = no_unit<typename U::Raw>();
    if (row != nullptr && map(c) < map.count) {
      raw[c] = __ldg(reinterpret_cast<const typename U::Raw*>(row) + map.part + map(c));
    }
  }
  float x[UNITS][U::kElems], params[2][UNITS][U::kElems], sum = 0.f;
  load_params<T, BYTES>({a.weight, a.bias}, a.params_f32, a.params_vec, map, uint32_t(a.dim), {1.f, 0.f}, params);
#pragma unroll
  for (int c = 0; c < UNITS; ++c) {
    U::unpack(raw[c], x[c]);
#pragma unroll
    for (int e = 0; e < U::kElems; ++e) sum += x[c][e];
  }
  GroupSum<1, WIDTH> group_sum(group, scratch);
  norm_row<T, BYTES, UNITS, WIDTH>(a, r, row != nullptr,
                                   static_cast<uint8_t*>(a.y) + r * a.y_stride + (map.part + map.lane) * BYTES,
                                   sum, map, group_sum, x, params[0], params[1]);
}

// Many rows: the blocks stay on the device, their threads keep the weights of
// their columns, and their groups take rows in turn out of the warps' queues.
// Two blocks per multiprocessor where the registers allow (us, with two and with one:
// 65537 x 333 half 23.2 and 24.5, 300000 x 100 half 36 and 42, 1048576 x 8 f32 12.5 and 15.0).
template <typename T, int BYTES, int UNITS>
constexpr int kResident = UNITS * Unit<T, BYTES>::kElems <= 12 ? 2 : 1;   // blocks, by their registers
template <typename T, int BYTES, int UNITS, int WIDTH, bool BY_ADDRESS>
__global__ void __launch_bounds__(kPipeBlock, (kResident<T, BYTES, UNITS>))
    norm_pipe_kernel(const NormArgs a, const uint32_t group, const RowsIn in) {
  using U = Unit<T, BYTES>;
  extern __shared__ uint4 slots[];
  __shared__ float scratch[kPipeBlock / 32][2][1];
  GroupSum<1, WIDTH> group_sum(group, scratch);
  const UnitMap<UNITS, WIDTH> map(group, uint32_t(a.dim) / U::kElems);
  const RowDeal deal(group);
  const uint32_t n = uint32_t(a.n);
  const RowQueue<T, BYTES, UNITS, WIDTH> queue(slots, 0, 1, map);
  float params[2][UNITS][U::kElems];
  load_params<T, BYTES>({a.weight, a.bias}, a.params_f32, a.params_vec, map, uint32_t(a.dim), {1.f, 0.f}, params);
  uint32_t r = deal.row;
  // Rows by base and stride: the address of the row that is fetched next, and of
  // the current row the lower half, both moved on from row to row.  (With a product
  // of 64 bits for each, and the choice between the two forms in the loop,
  // 16384 x 8192 bf16 took 101 us instead of 91, 65537 x 333 half 30 instead of 23.)
  const uint8_t* next = in.first + r * in.stride;
  uint32_t current = uint32_t(reinterpret_cast<uintptr_t>(next));
  const uint64_t in_step = deal.step * in.stride, out_step = deal.step * a.y_stride;
  uint8_t* out = static_cast<uint8_t*>(a.y) + r * a.y_stride + (map.part + map.lane) * BYTES;
  // Rows by address: rows[0] is the current row, rows[1 ...] those in the queue (null:
  // none), rows[kStages] an address that will have arrived when its copies start
  const uint8_t* rows[kStages + 1];
  auto address = [&](uint32_t row) {
    return row < n ? static_cast<const uint8_t*>(a.row_ptrs[row]) : nullptr;
  };
  if constexpr (BY_ADDRESS) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) rows[i + 1] = address(r + i * deal.step);
  }
  // row i of the thread's, counted from the current one
  auto fill = [&](uint32_t stage, int i) {
    if constexpr (BY_ADDRESS) {
      rows[i + 1] = valid_row(a, rows[i + 1]);
      if (rows[i + 1] != nullptr) queue.fill(stage, rows[i + 1], map);
    } else {
      if (r + i * deal.step < n) queue.fill(stage, next, map);
      next += in_step;
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fill(i, i);
  uint32_t stage = 0;
  // the lanes of a warp leave together
  for (uint32_t warp_row = deal.warp_row; warp_row < n; warp_row += deal.step) {
    fill(stage == 0 ? kStages - 1 : stage - 1, kStages - 1);
    if constexpr (BY_ADDRESS) {
#pragma unroll
      for (int i = 0; i < kStages; ++i) rows[i] = rows[i + 1];
      rows[kStages] = address(r + kStages * deal.step);
      current = uint32_t(reinterpret_cast<uintptr_t>(rows[0]));
    }
    const bool has = BY_ADDRESS ? rows[0] != nullptr : r < n;
    copies_wait<kStages - 1>();
    queue.arrive();
    float x[UNITS][U::kElems];
    Partial sum;
    if (has) {
      const uint32_t from = queue.place(stage, current, map);
      map.template each<kRun<BYTES, UNITS>>([&](int c, bool mine) {
        queue.take(from, c, mine, map, x[c]);
#pragma unroll
        for (int e = 0; e < U::kElems; ++e) sum.part[(c * U::kElems + e) % 4] += x[c][e];
      });
    }
    queue.arrive();
    norm_row<T, BYTES, UNITS, WIDTH>(a, r, has, out, sum.sum(), map, group_sum, x, params[0], params[1]);
    stage = stage + 1 == kStages ? 0 : stage + 1;
    r += deal.step;
    out += out_step;
    current += uint32_t(in_step);
  }
  copies_wait<0>();
}

// Rows too long for the registers of a block: three passes over the row, which
// stays in L2 between them.
template <typename T>
__global__ void __launch_bounds__(1024)
    norm_long_kernel(const NormArgs a) {
  __shared__ float scratch[32][2][1];
  GroupSum<1, kWarps> group_sum(blockDim.x, scratch);
  const uint32_t dim = uint32_t(a.dim);
  for (uint64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    const T* row = reinterpret_cast<const T*>(
        a.row_ptrs != nullptr ? valid_row(a, a.row_ptrs[r]) : static_cast<const uint8_t*>(a.x) + r * a.x_stride);
    if (row == nullptr) continue;
    float sum[1] = {0.f};
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) sum[0] += to_float(row[i]);
    group_sum(sum);
    const float mean = sum[0] * a.inv_dim;
    float rest[1];    // the sum of the distances from the mean
    auto centre = [&](float off) {
      float sq[1] = {0.f};
      rest[0] = 0.f;
      for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
        const float d = (to_float(row[i]) - mean) - off;
        sq[0] = fmaf(d, d, sq[0]);
        rest[0] += d;
      }
      group_sum(sq);
      return rsqrtf(fmaf(sq[0], a.inv_dim, a.eps));
    };
    float rstd = centre(0.f), off = 0.f;
    if (is_far(mean, rstd)) {   // uniform over the block
      group_sum(rest);
      off = rest[0] * a.inv_dim;
      rstd = centre(off);
    }
    T* out = reinterpret_cast<T*>(static_cast<uint8_t*>(a.y) + r * a.y_stride);
    for (uint32_t i = threadIdx.x; i < dim; i += blockDim.x) {
      const float w = load_param<T>(a.weight, a.params_f32, i, 1.f);
      const float b = load_param<T>(a.bias, a.params_f32, i, 0.f);
      out[i] = from_float<T>(fmaf(((to_float(row[i]) - mean) - off) * rstd, w, b));
    }
    if (threadIdx.x == 0) {
      if (a.mean != nullptr) a.mean[r] = mean + off;
      if (a.rstd != nullptr) a.rstd[r] = rstd;
    }
  }
}

// Units per thread that the kernels are built for: a thread holds a row's
// elements, weights and biases, 32 of each at most.
template <typename T, int BYTES>
const uint32_t* unit_choices() {
  static const uint32_t whole[] = {1, 2, 3, 4, 0}, pairs[] = {4, 8, 16, 0}, ones[] = {8, 12, 16, 32, 0};
  return BYTES == 16 ? whole : Unit<T, BYTES>::kElems == 2 ? pairs : ones;
}

template <typename T, int BYTES, int UNITS, int WIDTH>
int launch_norm_width(const NormArgs& a, uint32_t group, const RowsIn& in, cudaStream_t stream) {
  using Queue = RowQueue<T, BYTES, UNITS, WIDTH>;
  constexpr auto kRows = norm_pipe_kernel<T, BYTES, UNITS, WIDTH, false>;
  constexpr auto kAddresses = norm_pipe_kernel<T, BYTES, UNITS, WIDTH, true>;
  const bool by_address = a.row_ptrs != nullptr;
  const int rc = by_address ? allow_shared<kAddresses>() : allow_shared<kRows>();
  if (rc != HKV_OK) return rc;
  (by_address ? kAddresses : kRows)<<<pipe_blocks(a.n, group, kResident<T, BYTES, UNITS>),
                                      pipe_threads(group), Queue::bytes(group, 1), stream>>>(a, group, in);
  return HKV_OK;
}
template <typename T, int BYTES, int UNITS>
int launch_norm_pipe(const NormArgs& a, uint32_t group, const RowsIn& in, cudaStream_t stream) {
  // the widths that fitting_units() gives rows of so many units per thread
  if constexpr (BYTES != 16 || UNITS != 1) {
    if constexpr (BYTES == 16 || UNITS * Unit<T, BYTES>::kElems == 32) {
      if (group > 32) return launch_norm_width<T, BYTES, UNITS, kWarps>(a, group, in, stream);
    }
    if (group == 32) return launch_norm_width<T, BYTES, UNITS, 32>(a, group, in, stream);
  }
  if constexpr (BYTES == 16) return launch_norm_width<T, BYTES, UNITS, 0>(a, group, in, stream);
  else if (group == 16) return launch_norm_width<T, BYTES, UNITS, 16>(a, group, in, stream);
  else return launch_norm_width<T, BYTES, UNITS, 8>(a, group, in, stream);
}

template <typename T, int BYTES, int UNITS, int WIDTH>
void launch_norm_few(const NormArgs& a, uint32_t group, const RowsIn& in, cudaStream_t stream) {
  const uint32_t groups = group > kNormBlock ? 1 : kNormBlock / group;
  const unsigned grid = unsigned((a.n + groups - 1) / groups);
  norm_kernel<T, BYTES, UNITS, WIDTH><<<grid, groups * group, 0, stream>>>(a, group, in);
}

template <typename T, int BYTES>
int launch_norm_type(const NormArgs& a, cudaStream_t stream) {
  const uint64_t units = a.dim / Unit<T, BYTES>::kElems;
  const RowsIn in = rows_in(a.x, a.x_stride);
  uint32_t per_thread = fitting_units(units, BYTES, unit_choices<T, BYTES>());
  // rows of floats by address: two units, for two blocks per multiprocessor, whose
  // warps wait for addresses and rows in turn (us, with two units and without the
  // rule, a tenth missing: 1048576 x 48 76 and 78, x 64 81 and 85, 524288 x 128 77 and 83,
  // 300000 x 200 75 and 80, 131072 x 512 76 and 81, 65536 x 1024 77 and 76; it loses at
  // 262144 x 256, 84 and 76, and 100000 x 600, 90 and 82; by base and stride 1048576 x
  // 64 takes 100 with two units and 96 with four)
  if (BYTES == 16 && sizeof(T) == 4 && a.row_ptrs != nullptr && per_thread > 2 && units <= 2 * kPipeBlock) {
    per_thread = 2;
  }
  if (per_thread == 0) {
    const uint64_t cap = uint64_t(sm_count()) * 2;
    norm_long_kernel<T><<<unsigned(a.n < cap ? a.n : cap), 1024, 0, stream>>>(a);
    return HKV_OK;
  }
  const uint32_t group = group_for(units, per_thread, BYTES);
  // Few rows are not worth a queue: a group of as many threads as the row has units
  // (two units each in long rows) takes one, as long as all of them run at once, in
  // the 1024 threads per multiprocessor that their registers allow.  us, one row per
  // group and queues: 5000 x 64 f32 2.4 and 3.7, 16 x 8192 bf16 3.5 and 3.7, 1000 x 1000
  // bf16 3.2 and 3.7, 300 x 333 half 2.8 and 3.1; beyond it 20000 x 64 by
  // address 4.6 and 4.2, 220 x 8192 6.1 and 4.2, 1700 x 1000 4.6 and 3.8, 500 x 333 3.5 and 3.1.
  if (units <= 2048) {
    const bool two = units > 1024, narrow_warp = BYTES == 16 && units <= 16;
    const uint32_t threads = two           ? group_for(units, 2, BYTES)
                             : narrow_warp ? group_for(units, 1, BYTES)
                                           : uint32_t((units + 31) / 32 * 32);
    if (a.n * threads <= uint64_t(sm_count()) * 1024) {
      if (two) launch_norm_few<T, BYTES, 2, kWarps>(a, threads, in, stream);
      else if (!narrow_warp) launch_norm_few<T, BYTES, 1, kWarps>(a, threads, in, stream);
      else if constexpr (BYTES == 16) launch_norm_few<T, BYTES, 1, 0>(a, threads, in, stream);
      return HKV_OK;
    }
  }
#define HKV_CALL(N) return launch_norm_pipe<T, BYTES, N>(a, group, in, stream)
  if constexpr (BYTES == 16) {
    switch (per_thread) {
      case 1: HKV_CALL(1);
      case 2: HKV_CALL(2);
      case 3: HKV_CALL(3);
      default: HKV_CALL(4);
    }
  } else if constexpr (Unit<T, BYTES>::kElems == 2) {
    switch (per_thread) {
      case 4: HKV_CALL(4);
      case 8: HKV_CALL(8);
      default: HKV_CALL(16);
    }
  } else {
    switch (per_thread) {
      case 8: HKV_CALL(8);
      case 12: HKV_CALL(12);
      case 16: HKV_CALL(16);
      default: HKV_CALL(32);
    }
  }
#undef HKV_CALL
}

}  // namespace

int check_norm(uint64_t n, uint64_t dim, uint32_t value_kind, uint32_t param_kind, float eps) noexcept {
  HKV_ROWS_CHECK(n < (1ull << 31), "batches of 2^31 or more rows");
  HKV_ROWS_CHECK(dim >= 1 && dim < (1ull << 24), "dim must be between 1 and 2^24 - 1");
  HKV_ROWS_CHECK(is_row_kind(value_kind), "rows are float32, float16 or bfloat16");
  HKV_ROWS_CHECK(param_kind == value_kind || param_kind == kValueF32,
                 "weight and bias have the rows' type or float32");
  HKV_ROWS_CHECK(eps >= 0.f && eps <= 3.4e38f, "eps must be finite and not negative");
  return HKV_OK;
}

int launch_norm(NormArgs args, uint32_t value_kind, cudaStream_t stream) {
  const uint32_t size = row_kind_size(value_kind);
  uint64_t bits = args.dim * size | address_bits(args.y) | args.y_stride;
  if (args.row_ptrs == nullptr) bits |= address_bits(args.x) | args.x_stride;
  const uint32_t unit = unit_bytes(bits, size);
  args.row_mask = unit_bytes(args.dim * size, size) - 1u;
  HKV_ROWS_CHECK(unit != 0, "a row does not start at a multiple of its element size");
  int rc = HKV_OK;
#define HKV_CALL(T, BYTES) rc = launch_norm_type<T, BYTES>(args, stream)
  HKV_FOR_UNIT(value_kind, unit, HKV_CALL)
#undef HKV_CALL
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
  HKV_ROWS_CHECK(all_aligned(row_kind_size(param_kind), weight, bias) && all_aligned(4, mean, rstd),
                 "weight, bias, mean and rstd must start at a multiple of their element size");
  NormArgs a{};
  a.n = n;
  a.dim = dim;
  a.x = x;
  a.x_stride = x_stride;
  a.weight = weight;
  a.bias = bias;
  a.params_f32 = param_kind == kValueF32;
  a.params_vec = (address_bits(weight) | address_bits(bias)) % 16 == 0;
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
  HKV_ROWS_CHECK(all_aligned(row_kind_size(param_kind), weight, bias) && all_aligned(4, mean, rstd) &&
                     all_aligned(8, row_ptrs),
                 "weight, bias, mean, rstd and row_ptrs must start at a multiple of their element size");
  NormArgs a{};
  a.n = n;
  a.dim = dim;
  a.row_ptrs = row_ptrs;
  a.weight = weight;
  a.bias = bias;
  a.params_f32 = param_kind == kValueF32;
  a.params_vec = (address_bits(weight) | address_bits(bias)) % 16 == 0;
  a.eps = eps;
  a.inv_dim = 1.f / float(dim);
  a.y = y;
  a.y_stride = y_stride;
  a.mean = mean;
  a.rstd = rstd;
  return launch_norm(a, value_kind, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
