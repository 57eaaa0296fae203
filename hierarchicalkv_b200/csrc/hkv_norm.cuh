// What layer norm and its gradient share: how a row is dealt to threads, the sums
// over it, and the queues rows wait in.
#pragma once

#include "hkv_norm.h"
#include "hkv_rows.cuh"

namespace hkv {

constexpr uint32_t kFull = 0xFFFFFFFFu;
constexpr int kPipeBlock = 512;   // threads of the kernels that stay on the device
constexpr int kStages = 3;        // rows of a warp's queue: one in use, two on their way

// WIDTH, of a kernel: how many lanes have a row.  8, 16 or 32; 0: a power of two
// below 32 known at run time; kWarps: several whole warps.
constexpr int kWarps = 64;

// A thread's sum in four parts: one would be a chain of additions that wait for
// one another.
struct Partial {
  float part[4] = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ float sum() const { return (part[0] + part[1]) + (part[2] + part[3]); }
};

// Sum over the `group` threads of a row; every thread gets it.  scratch: two floats
// of each value per warp, used in turn, so that one barrier of the group's own
// (named 1 + its number in the block) is enough.
template <int N, int WIDTH>
struct GroupSum {
  static constexpr bool WIDE = WIDTH == kWarps;
  uint32_t group, warps, span, from, barrier;   // warps: of the group; span: the next power of two
  float (*scratch)[2][N];                       // [warps of the block]
  uint32_t turn = 0;

  __device__ __forceinline__ GroupSum(uint32_t group_, float (*scratch_)[2][N])
      : group(group_), warps(group_ >> 5), barrier(1u + threadIdx.x / group_), scratch(scratch_) {
    span = 1;
    while (span < warps) span <<= 1;
    // where this lane reads when the group's warps exchange their sums
    from = WIDE ? threadIdx.x / group * warps + (threadIdx.x & (span - 1u)) : 0u;
  }

  __device__ __forceinline__ void operator()(float (&v)[N]) {
    if (WIDE) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kFull, v[i], d);
      }
      if (warps == 1) return;   // few rows, on one warp each
      if ((threadIdx.x & 31u) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) scratch[threadIdx.x >> 5][turn][i] = v[i];
      }
      asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(group) : "memory");
      const bool has = (threadIdx.x & (span - 1u)) < warps;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = has ? scratch[from][turn][i] : 0.f;
      for (uint32_t d = span >> 1; d > 0; d >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kFull, v[i], d);
      }
      turn ^= 1u;
    } else {
#pragma unroll
      for (uint32_t d = (WIDTH ? uint32_t(WIDTH) : group) >> 1; d > 0; d >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kFull, v[i], d);
      }
    }
  }
};

// Keeps an address as it is: the compiler would work it out again for every unit.
__device__ __forceinline__ uint32_t keep(uint32_t shared) {
  asm volatile("" : "+r"(shared));
  return shared;
}

// Where a thread's units lie in its row: unit c of the thread is first + c * width
// of the row.  A warp of a group of several owns a part of consecutive units, which
// begins at unit `part` and has `count`; the lanes of a group below a warp own all.
template <int UNITS, int WIDTH>
struct UnitMap {
  static constexpr uint32_t kWidth = WIDTH == kWarps ? 32 : WIDTH;
  uint32_t part, count, lane, width;   // lane: within the width

  __device__ __forceinline__ UnitMap(uint32_t group, uint32_t units) {
    width = WIDTH == 0 ? group : kWidth;
    lane = threadIdx.x & (width - 1u);
    part = WIDTH == kWarps ? (threadIdx.x % group >> 5) * 32u * UNITS : 0u;
    count = units > part ? min(units - part, width * UNITS) : 0u;
  }
  // The unit's number within the part.
  __device__ __forceinline__ uint32_t operator()(int c) const {
    return lane + uint32_t(c) * (WIDTH == 0 ? width : kWidth);
  }
  // f(c, mine) for the thread's units c, in runs of RUN: `mine` is a constant where
  // all lanes have the whole run, and runs that none has are left out.  One test
  // serves rows that reach into the last run (65536 x 1001 bf16: 50 us, with a test
  // per run 58).  A single run is not tested, only its units, on a row of one warp or
  // less (262144 x 128 bf16: 22.2 us, with a test 23.6); on several warps, whose
  // last may have none, it is (16384 x 8192 bf16: 91 us, without 110).
  template <int RUN, typename F>
  __device__ __forceinline__ void each(F&& f) const {
    static_assert(UNITS % RUN == 0, "whole runs");
    if ((WIDTH != kWarps || RUN < UNITS) && (UNITS - RUN) * (WIDTH == 0 ? width : kWidth) <= count) {
#pragma unroll
      for (int c = 0; c < UNITS - RUN; ++c) f(c, true);
#pragma unroll
      for (int c = UNITS - RUN; c < UNITS; ++c) f(c, (*this)(c) < count);
      return;
    }
#pragma unroll
    for (int b = 0; b < UNITS; b += RUN) {
      if ((b + RUN) * (WIDTH == 0 ? width : kWidth) <= count) {
#pragma unroll
        for (int i = 0; i < RUN; ++i) f(b + i, true);
      } else if (b * (WIDTH == 0 ? width : kWidth) < count) {
#pragma unroll
        for (int i = 0; i < RUN; ++i) f(b + i, (*this)(b + i) < count);
      }
    }
  }
};
// Units of 16 bytes: one run, the loops are straight.
template <int BYTES, int UNITS>
constexpr int kRun = BYTES == 16 || UNITS % 4 != 0 ? UNITS : 4;

// A warp's queue of rows (or of its parts of rows) in shared memory, filled ahead
// with asynchronous copies that hold no registers.  The slots of 16 bytes belong
// to the warp alone, so no barrier of the block is needed.  Rows in 16-byte units:
// a lane copies the units it will take.  Narrower units: the lanes of a row copy
// the aligned 16 bytes around it together and take their units at any alignment.
// Nothing behind a row's end is read; the up to 14 bytes before its first element
// are, which lie in the row's allocation, since no allocation starts inside aligned
// 16 bytes.
template <typename T, int BYTES, int UNITS, int WIDTH>
struct RowQueue {
  using Map = UnitMap<UNITS, WIDTH>;
  uint32_t mine;         // shared address of this lane's slot 0 (16-byte units) or of its row's first
  uint32_t stage_bytes;  // distance of a warp's stages

  static constexpr __host__ __device__ __forceinline__ uint32_t slots_per_row(uint32_t width) {
    return BYTES == 16 ? width * UNITS : (width * UNITS * BYTES + 15u) / 16u + 1u;
  }
  static __host__ __device__ __forceinline__ uint32_t slots_per_warp(uint32_t width) {
    return 32u / width * slots_per_row(width);
  }
  // Shared memory of a block with queues for `operands` matrices.
  static size_t bytes(uint32_t group, uint32_t operands) {
    return size_t(kStages) * operands * (kPipeBlock / 32) * slots_per_warp(group < 32 ? group : 32) * 16;
  }

  // operand: which of the row's matrices this queue holds
  __device__ __forceinline__ RowQueue(const uint4* shared, uint32_t operand, uint32_t operands,
                                      const Map& map) {
    const uint32_t warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t slots = slots_per_warp(map.width);
    stage_bytes = operands * warps * slots * 16u;
    mine = static_cast<uint32_t>(__cvta_generic_to_shared(shared)) +
           (operand * warps + warp) * slots * 16u +
           (BYTES == 16 ? lane : lane / map.width * slots_per_row(map.width)) * 16u;
  }

  // Puts a row into a stage.
  __device__ __forceinline__ void fill(uint32_t stage, const uint8_t* row, const Map& map) const {
    const uint32_t to = mine + stage * stage_bytes;
    if constexpr (BYTES == 16) {
      const uint8_t* from = row + (map.part + map.lane) * 16u;
#pragma unroll
      for (int c = 0; c < UNITS; ++c) {
        if (map(c) < map.count) copy_async(to + c * 512u, from + (map(c) - map.lane) * 16u);
      }
    } else {
      const uint32_t ahead = shift(uint32_t(reinterpret_cast<uintptr_t>(row)), map);
      const uint8_t* from = row + map.part * BYTES - ahead;   // aligned
      const int end = map.count != 0 ? int(ahead + map.count * BYTES) : 0;
      constexpr int kSlots = int(slots_per_row(Map::kWidth));
#pragma unroll
      for (int i = 0; i < kSlots; i += int(Map::kWidth)) {
        const int at = (i + int(map.lane)) * 16;
        if (at < end) copy_async(to + at, from + at, uint32_t(min(16, end - at)));
      }
    }
  }

  // Where the warp's part of a row begins in its first slot; `row`: the address's
  // lower half.
  __device__ __forceinline__ uint32_t shift(uint32_t row, const Map& map) const {
    return BYTES == 16 ? 0u : (row + map.part * BYTES) & 15u;
  }

  // Before the first take() from a stage and after the last.
  __device__ __forceinline__ void arrive() const {
    if (BYTES != 16) __syncwarp();   // other lanes' copies; 16-byte units are a lane's own
  }

  // Where the lane's first unit of the row in a stage is.
  __device__ __forceinline__ uint32_t place(uint32_t stage, uint32_t row, const Map& map) const {
    return keep(mine + stage * stage_bytes + (BYTES == 16 ? 0u : shift(row, map) + map.lane * BYTES));
  }
  // Unit c of the lane, `from` place(), as floats; zeros where it has none.
  static __device__ __forceinline__ void take(uint32_t from, int c, bool mine, const Map& map,
                                              float (&f)[Unit<T, BYTES>::kElems]) {
    // inside the queue's slots even where the lane has no such unit
    const auto v = load_shared<BYTES>(from + (BYTES == 16 ? c * 512u : (map(c) - map.lane) * BYTES));
    Unit<T, BYTES>::unpack(v, f);
#pragma unroll
    for (int e = 0; e < Unit<T, BYTES>::kElems; ++e) f[e] = mine ? f[e] : 0.f;
  }
};

// One weight or bias; `none` where there are none.
template <typename T>
__device__ __forceinline__ float load_param(const void* p, bool f32, uint32_t column, float none) {
  if (p == nullptr) return none;
  return f32 ? __ldg(static_cast<const float*>(p) + column) : to_float(static_cast<const T*>(p)[column]);
}

// A thread's weights, or weights and biases (the P vectors p): those of the columns of
// its units, none[i] where p[i] is null.  The choice between the types is made once
// for all of them and no load is behind a condition, so that all are in flight
// together: columns past the row's end read its last unit again.  (With the
// choice made unit by unit each load waited for the one before: 65536 x 1001 bf16
// took 86 us instead of 64.)  vec: the addresses are multiples of 16.
template <typename T, int BYTES, int UNITS, int WIDTH, int P>
__device__ __forceinline__ void load_params(const void* const (&p)[P], bool f32, bool vec,
                                            const UnitMap<UNITS, WIDTH>& map, uint32_t dim,
                                            const float (&none)[P],
                                            float (&out)[P][UNITS][Unit<T, BYTES>::kElems]) {
  constexpr int N = Unit<T, BYTES>::kElems;
  const void* any = p[0] != nullptr ? p[0] : p[P - 1];
  if (any == nullptr) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int c = 0; c < UNITS; ++c) {
#pragma unroll
        for (int e = 0; e < N; ++e) out[i][c][e] = none[i];
      }
    }
    return;
  }
  auto column = [&](int c) { return min((map.part + map(c)) * N, dim - N); };   // rows are whole units
  auto from = [&](int i, auto* type) {
    return static_cast<decltype(type)>(p[i] != nullptr ? p[i] : any);
  };
  if (f32) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float* at = from(i, static_cast<const float*>(nullptr));
#pragma unroll
      for (int c = 0; c < UNITS; ++c) {
        if (N % 4 == 0 && vec) {
#pragma unroll
          for (int e = 0; e + 3 < N; e += 4) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(at + column(c) + e));
            out[i][c][e] = v.x;
            out[i][c][e + 1] = v.y;
            out[i][c][e + 2] = v.z;
            out[i][c][e + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) out[i][c][e] = __ldg(at + column(c) + e);
        }
      }
    }
  } else if (BYTES == 16 && vec) {
    typename Unit<T, BYTES>::Raw raw[P][UNITS];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const T* at = from(i, static_cast<const T*>(nullptr));
#pragma unroll
      for (int c = 0; c < UNITS; ++c) {
        raw[i][c] = __ldg(reinterpret_cast<const typename Unit<T, BYTES>::Raw*>(at + column(c)));
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int c = 0; c < UNITS; ++c) Unit<T, BYTES>::unpack(raw[i][c], out[i][c]);
    }
  } else {
    T raw[P][UNITS][N];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const T* at = from(i, static_cast<const T*>(nullptr));
#pragma unroll
      for (int c = 0; c < UNITS; ++c) {
#pragma unroll
        for (int e = 0; e < N; ++e) raw[i][c][e] = at[column(c) + e];
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int c = 0; c < UNITS; ++c) {
#pragma unroll
        for (int e = 0; e < N; ++e) out[i][c][e] = to_float(raw[i][c][e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (p[i] != nullptr) continue;
#pragma unroll
    for (int c = 0; c < UNITS; ++c) {
#pragma unroll
      for (int e = 0; e < N; ++e) out[i][c][e] = none[i];
    }
  }
}

// The rows a group takes.
struct RowDeal {
  uint32_t row, step;   // the first row and the distance to the next
  uint32_t warp_row;    // the first row of the warp's first group: the warp is done when it is

  __device__ __forceinline__ explicit RowDeal(uint32_t group) {
    const uint32_t groups = blockDim.x / group;
    step = gridDim.x * groups;
    row = blockIdx.x * groups + threadIdx.x / group;
    warp_row = group >= 32u ? row : row - (threadIdx.x & 31u) / group;
  }
};

// ---- host ----------------------------------------------------------------------

// Threads on a row that hold `per_thread` units each.  Units of 16 bytes: whole
// warps, or a power of two, two at least (a sector of 32 bytes).  Narrow units:
// whole warps, or a quarter or half of one, widths the kernels know when they are built.
inline uint32_t group_for(uint64_t units, uint32_t per_thread, uint32_t unit) {
  const uint64_t threads = (units + per_thread - 1) / per_thread;
  if (unit != 16) return threads <= 8 ? 8 : threads <= 16 ? 16 : uint32_t((threads + 31) / 32 * 32);
  if (threads > 16) return uint32_t((threads + 31) / 32 * 32);
  uint32_t group = 2;
  while (group < threads) group <<= 1;
  return group;
}

// Of the numbers of units per thread (ascending, 0 ends them) the one that leaves
// the fewest places of the group empty; 0: the row is too long for a block.  A row
// shared by warps counts one and a half times: its sums need barriers (65536 x
// 1001 bf16: 92 us on four warps of 8 units per lane, 50 us on one of 32).  Of
// equals the most units per thread, for the fewest threads; but narrow units that fit
// a warp the fewest, for the registers (1 Mi x 33 half, gradient: 96 us with 8
// units on eight lanes, 110 us with 16).
// Not among them: one unit of 16 bytes where a warp or more has the row (60000 x 516
// f32: 78 us with one, 46 with three; gradient 20000 x 2240 bf16 99 and 61 with two; but
// 1048576 x 8 f32 12.5 with one, 14.4 with two), and narrow units on several warps unless
// they are the most per thread.
inline uint32_t fitting_units(uint64_t units, uint32_t unit, const uint32_t* choices) {
  uint32_t best = 0;
  uint64_t least = 0;
  for (; *choices != 0; ++choices) {
    const uint64_t group = group_for(units, *choices, unit);
    if (group > uint32_t(kPipeBlock)) continue;
    if (unit == 16 ? *choices == 1 && group > 16 : choices[1] != 0 && group > 32) continue;
    // narrow units: runs of four that no lane of the group has are left out
    const uint64_t run = unit == 16 ? *choices : 4;
    const uint64_t width = group < 32 ? group : 32, warps = group / width;
    uint64_t runs = 0;
    for (uint64_t w = 0; w < warps; ++w) {
      const uint64_t from = w * width * *choices;
      const uint64_t mine = from < units ? units - from : 0;
      const uint64_t most = (mine + width * run - 1) / (width * run);
      runs += most < *choices / run ? most : *choices / run;
    }
    const uint64_t cost = runs * run * width * (warps > 1 ? 3 : 2);
    if (best == 0 || cost < least || (cost == least && (unit == 16 || group > 32))) {
      best = *choices;
      least = cost;
    }
  }
  return best;
}

// Blocks of the kernels that stay on the device: as many as take part, at most
// `resident` per multiprocessor.
inline uint32_t pipe_blocks(uint64_t n, uint32_t group, int resident = 1) {
  const uint32_t groups = kPipeBlock / group;
  const uint64_t want = (n + groups - 1) / groups, most = uint64_t(sm_count()) * resident;
  return uint32_t(want < most ? want : most);
}
// Threads of such a block: whole groups.
inline uint32_t pipe_threads(uint32_t group) { return kPipeBlock / group * group; }

int check_norm(uint64_t n, uint64_t dim, uint32_t value_kind, uint32_t param_kind, float eps) noexcept;

}  // namespace hkv
