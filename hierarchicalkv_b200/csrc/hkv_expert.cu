// Token rows sorted by expert and back: the routing of a mixture-of-experts
// layer between the rows of a table and the experts' products.
//
// T tokens, each assigned to k experts (expert_ids[T][k]); N = T * k
// assignments, assignment i = t * k + j.  An id outside [0, E) is dropped.
//
//   sort              stable: offsets[E + 1], position[N] (the place of
//                     assignment i among the sorted rows, or -1), source[N]
//                     (the assignment at each place, -1 behind the last)
//   dispatch          rows[position[t, j]] = x[t]
//   combine           out[t]  = sum_j w[t, j] * rows[position[t, j]]
//                     (without weights: the gradient of dispatch)
//   combine backward  d_rows[position[t, j]] = w[t, j] * d_out[t]
//                     d_w[t, j] = <d_out[t], rows[position[t, j]]>
//
// Sums and products are in 32-bit floats and every result is rounded once.
// No floats are added with atomics: results do not depend on the order in which
// blocks run.  Measured, us, and the share of the bandwidth of a copy: 16384 tokens of
// 8 rows of 4096 bf16, sort 12 and dispatch 187, 94 % together; combine 65536 of 2 of
// 128 f32 15, 95 %; its gradient 8192 of 8 of 2048 bf16 93, 95 %; rows of 1001 half,
// moved in 2-byte units and bound by the latency of so many small loads, combine 85,
// 69 % (30011 of 6), gradient 130, 59 % (20000 of 6).
//
// The reference has no such operators; hkv_shard.cu groups keys by their
// owner rank and moves whole rows by index, unordered inside an owner.
#include <atomic>

#include "hkv_rows.cuh"

namespace hkv {

namespace {

thread_local std::string g_rows_error;

}  // namespace

int rows_fail(int code, const char* message) noexcept {
  try {
    g_rows_error = message;
  } catch (...) {
    g_rows_error.clear();
  }
  return code;
}

int rows_launched() noexcept {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HKV_OK : rows_fail(HKV_ERR_CUDA, cudaGetErrorString(e));
}

// Asked of the driver once per device: the query takes longer than a launch.
int sm_count() noexcept {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  int sms = known[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
      cudaGetLastError();
      return 148;
    }
    known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}

namespace {

constexpr uint32_t kMaxExperts = 1024;
constexpr uint32_t kMaxTopK = 64;
constexpr uint32_t kFull = 0xFFFFFFFFu;

// ---- sort -------------------------------------------------------------------
//
// A counting sort.  Warp w of a block owns a contiguous run of assignments and
// a row of counters in shared memory; the lanes that hold the same expert are
// found with one ballot per bit of the expert's number, so an assignment's rank
// among the warp's earlier ones of its expert is the counter plus the equal
// lanes below it, and no two lanes touch a counter at once.  Scanning the
// counters over the warps, the blocks and the experts turns ranks into places.
// (__match_any_sync finds the same lanes in one instruction, at a rate that made
// 131,072 assignments to 128 experts take 39 us on eight blocks.)

constexpr int kSortCounters = 16384;   // 16-bit counters: warps x experts of a block

struct SortShared {
  uint16_t count[kSortCounters];
  uint32_t total[kMaxExperts];   // this block's assignments per expert
  uint32_t base[kMaxExperts];    // where this block's first row of each expert goes
  uint32_t scan[32];
};

// ITEMS ids per lane: id i of the lane is assignment first + i * 32 + lane.
// Out: the expert of each (experts: dropped) and its rank in the warp.
template <typename ID, int ITEMS>
__device__ __forceinline__ void rank_in_warp(const ID* __restrict__ ids, uint64_t first, uint64_t n,
                                             uint32_t experts, uint16_t* count, uint32_t lane,
                                             uint32_t (&expert)[ITEMS], uint32_t (&rank)[ITEMS]) {
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const uint64_t at = first + uint32_t(i) * 32u + lane;
    ID id = -1;
    if (at < n) id = ids[at];
    expert[i] = (id >= 0 && id < ID(experts)) ? uint32_t(id) : experts;
  }
  uint32_t same[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) same[i] = kFull;
  for (uint32_t bit = 1; bit <= experts; bit <<= 1) {   // `experts` itself marks the dropped
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t set = __ballot_sync(kFull, (expert[i] & bit) != 0);
      same[i] &= (expert[i] & bit) != 0 ? set : ~set;
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const uint32_t below = __popc(same[i] & ((1u << lane) - 1u));
    rank[i] = 0;
    if (expert[i] < experts) {
      const uint32_t before = count[expert[i]];
      rank[i] = before + below;
      __syncwarp(same[i]);
      if (below == 0) count[expert[i]] = static_cast<uint16_t>(before + __popc(same[i]));
    }
    __syncwarp();
  }
}

// Exclusive scan of value(e) over e < experts by the whole block; out[e] and
// the total.  Any block of whole warps with at most 1024 threads.
template <typename Value>
__device__ __forceinline__ uint32_t block_scan(uint32_t experts, Value value, uint32_t* out,
                                               uint32_t* scratch) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  // segments of 32 experts, at most 32 of them, round robin over the warps
  for (uint32_t seg = warp; seg * 32u < experts; seg += warps) {
    const uint32_t e = seg * 32u + lane;
    const uint32_t v = e < experts ? value(e) : 0u;
    uint32_t sum = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t other = __shfl_up_sync(kFull, sum, d);
      if (lane >= uint32_t(d)) sum += other;
    }
    if (e < experts) out[e] = sum - v;
    if (lane == 31) scratch[seg] = sum;
  }
  __syncthreads();
  const uint32_t segments = (experts + 31u) / 32u;
  uint32_t total = 0;
  if (warp == 0) {
    const uint32_t v = lane < segments ? scratch[lane] : 0u;
    uint32_t sum = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t other = __shfl_up_sync(kFull, sum, d);
      if (lane >= uint32_t(d)) sum += other;
    }
    __syncwarp();
    scratch[lane] = sum;
  }
  __syncthreads();
  total = scratch[segments - 1];
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
    if (e >= 32u) out[e] += scratch[(e >> 5) - 1];
  }
  __syncthreads();
  return total;
}

// The warps' counters become their exclusive sums over the block's earlier
// warps; total[e] the block's count.
__device__ __forceinline__ void scan_warps(SortShared& s, uint32_t experts) {
  const uint32_t warps = blockDim.x >> 5;
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
    uint32_t sum = 0;
    for (uint32_t w = 0; w < warps; ++w) {
      const uint32_t c = s.count[w * experts + e];
      s.count[w * experts + e] = static_cast<uint16_t>(sum);
      sum += c;
    }
    s.total[e] = sum;
  }
}

template <int ITEMS>
__device__ __forceinline__ void write_places(const SortShared& s, uint64_t first, uint64_t n,
                                             uint32_t experts, uint32_t lane, uint32_t warp,
                                             const uint32_t (&expert)[ITEMS],
                                             const uint32_t (&rank)[ITEMS],
                                             int32_t* __restrict__ position,
                                             int32_t* __restrict__ source) {
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const uint64_t at = first + uint32_t(i) * 32u + lane;
    if (at >= n) continue;
    int32_t place = -1;
    if (expert[i] < experts) {
      place = int32_t(s.base[expert[i]] + s.count[warp * experts + expert[i]] + rank[i]);
      source[place] = int32_t(at);
    }
    position[at] = place;
  }
}

// Small batches: one cluster of 1 ... 8 blocks does everything in one launch;
// the blocks exchange their counts through distributed shared memory.
template <typename ID, int ITEMS>
__global__ void __launch_bounds__(1024)
    sort_cluster_kernel(const ID* __restrict__ ids, const uint64_t n, const uint32_t experts,
                        int32_t* __restrict__ offsets, int32_t* __restrict__ position,
                        int32_t* __restrict__ source) {
  __shared__ SortShared s;
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t blocks = gridDim.x;   // one cluster
  for (uint32_t c = threadIdx.x; c < warps * experts; c += blockDim.x) s.count[c] = 0;
  __syncthreads();
  uint32_t expert[ITEMS], rank[ITEMS];
  const uint64_t first = (uint64_t(blockIdx.x) * warps + warp) * (ITEMS * 32);
  rank_in_warp<ID, ITEMS>(ids, first, n, experts, s.count + warp * experts, lane, expert, rank);
  __syncthreads();
  scan_warps(s, experts);
  uint32_t total;
  if (blocks == 1) {
    __syncthreads();
    total = block_scan(experts, [&](uint32_t e) { return s.total[e]; }, s.base, s.scan);
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) offsets[e] = int32_t(s.base[e]);
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                     : "memory");
    const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(s.total));
    auto of_block = [&](uint32_t block, uint32_t e) {
      uint32_t address, v;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(address) : "r"(mine + e * 4u), "r"(block));
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(address));
      return v;
    };
    total = block_scan(
        experts,
        [&](uint32_t e) {
          uint32_t sum = 0;
          for (uint32_t b = 0; b < blocks; ++b) sum += of_block(b, e);
          return sum;
        },
        s.base, s.scan);
    if (blockIdx.x == 0) {
      for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) offsets[e] = int32_t(s.base[e]);
      __syncthreads();
    }
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
      uint32_t before = 0;
      for (uint32_t b = 0; b < blockIdx.x; ++b) before += of_block(b, e);
      s.base[e] += before;
    }
    // no block leaves, or reuses its counts, while another still reads them
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                     : "memory");
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offsets[experts] = int32_t(total);
  __syncthreads();
  write_places<ITEMS>(s, first, n, experts, lane, warp, expert, rank, position, source);
  for (uint64_t p = total + uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; p < n;
       p += uint64_t(blocks) * blockDim.x) {
    source[p] = -1;
  }
}

// Large batches: count per tile, scan over the tiles, place.  With up to
// kCountsSummed counts the placing blocks sum those of the tiles before theirs
// themselves and the scan's launch is saved (64 tiles x 128 experts: 8.9 us where
// scan and placement take 12; with 128 x 512 counts it is 30 us against 16).
constexpr uint32_t kCountsSummed = 16384;

template <typename ID>
__global__ void __launch_bounds__(1024)
    sort_count_kernel(const ID* __restrict__ ids, const uint64_t n, const uint32_t experts,
                      const uint32_t tile, uint32_t* __restrict__ counts) {
  __shared__ uint32_t local[kMaxExperts];
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) local[e] = 0;
  __syncthreads();
  const uint64_t first = uint64_t(blockIdx.x) * tile;
  const uint64_t last = min(n, first + tile);
#pragma unroll 4
  for (uint64_t at = first + threadIdx.x; at < last; at += blockDim.x) {
    const ID id = __ldg(ids + at);
    if (id >= 0 && id < ID(experts)) atomicAdd(&local[uint32_t(id)], 1u);
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
    counts[uint64_t(blockIdx.x) * experts + e] = local[e];
  }
}

// A block takes 32 experts, lane by expert; warp w sums a run of the tiles.
// counts becomes its exclusive sum over the tiles, totals[e] the sum.
__global__ void __launch_bounds__(1024)
    sort_scan_kernel(const uint32_t experts, const uint32_t tiles, uint32_t* __restrict__ counts,
                     uint32_t* __restrict__ totals) {
  __shared__ uint32_t sums[32][33];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint32_t e = blockIdx.x * 32u + lane;
  const uint32_t per_warp = (tiles + 31u) / 32u;
  const uint32_t first = min(tiles, warp * per_warp), last = min(tiles, first + per_warp);
  uint32_t sum = 0;
  if (e < experts) {
#pragma unroll 4
    for (uint32_t t = first; t < last; ++t) sum += counts[uint64_t(t) * experts + e];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  uint32_t run = 0, total = 0;
  for (uint32_t w = 0; w < 32u; ++w) {
    const uint32_t v = sums[w][lane];
    if (w < warp) run += v;
    total += v;
  }
  if (e < experts) {
    if (warp == 0) totals[e] = total;
#pragma unroll 4
    for (uint32_t t = first; t < last; ++t) {
      uint32_t* at = counts + uint64_t(t) * experts + e;
      const uint32_t v = *at;
      *at = run;
      run += v;
    }
  }
}

// totals == nullptr: counts are not scanned yet.
template <typename ID, int ITEMS>
__global__ void __launch_bounds__(1024)
    sort_place_kernel(const ID* __restrict__ ids, const uint64_t n, const uint32_t experts,
                      const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
                      int32_t* __restrict__ offsets, int32_t* __restrict__ position,
                      int32_t* __restrict__ source) {
  __shared__ SortShared s;
  __shared__ uint32_t before[kMaxExperts];   // the earlier tiles' assignments of each expert
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (uint32_t c = threadIdx.x; c < warps * experts; c += blockDim.x) s.count[c] = 0;
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
    before[e] = totals != nullptr ? counts[uint64_t(blockIdx.x) * experts + e] : 0u;
  }
  __syncthreads();
  uint32_t expert[ITEMS], rank[ITEMS];
  const uint64_t first = (uint64_t(blockIdx.x) * warps + warp) * (ITEMS * 32);
  rank_in_warp<ID, ITEMS>(ids, first, n, experts, s.count + warp * experts, lane, expert, rank);
  __syncthreads();
  scan_warps(s, experts);
  __syncthreads();   // total[] is the block's own now; from here it is every tile's
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
    s.total[e] = totals != nullptr ? totals[e] : 0u;
  }
  __syncthreads();
  if (totals == nullptr) {
    // whole numbers: the order of these additions does not matter
    for (uint32_t c = threadIdx.x; c < gridDim.x * experts; c += blockDim.x) {
      const uint32_t tile = c / experts, e = c - tile * experts;
      const uint32_t v = counts[c];
      if (v == 0) continue;
      atomicAdd(&s.total[e], v);
      if (tile < blockIdx.x) atomicAdd(&before[e], v);
    }
    __syncthreads();
  }
  const uint32_t total =
      block_scan(experts, [&](uint32_t e) { return s.total[e]; }, s.base, s.scan);
  if (blockIdx.x == 0) {
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) offsets[e] = int32_t(s.base[e]);
    if (threadIdx.x == 0) offsets[experts] = int32_t(total);
    __syncthreads();
  }
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) s.base[e] += before[e];
  __syncthreads();
  write_places<ITEMS>(s, first, n, experts, lane, warp, expert, rank, position, source);
  for (uint64_t p = total + uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; p < n;
       p += uint64_t(gridDim.x) * blockDim.x) {
    source[p] = -1;
  }
}

// Threads of a sorting block: as many warps as have counters for every expert.
uint32_t sort_block(uint32_t experts) {
  const uint32_t warps = kSortCounters / experts;
  return (warps < 32u ? warps : 32u) * 32u;
}

struct SortPlan {
  uint32_t block, items;
  uint32_t cluster;   // blocks of the one-launch form; 0: one block per tile, several launches
  uint32_t tiles;
};

SortPlan plan_sort(uint64_t n, uint32_t experts) {
  SortPlan p{sort_block(experts), 1, 0, 0};
  if (n <= p.block) {
    p.block = n ? uint32_t((n + 31) / 32) * 32u : 32u;
    p.cluster = 1;
    return p;
  }
  for (uint32_t items : {1u, 4u}) {
    p.items = items;
    for (uint32_t blocks : {1u, 2u, 4u, 8u}) {
      if (n <= uint64_t(p.block) * items * blocks) {
        p.cluster = blocks;
        return p;
      }
    }
  }
  // tiles that fill the device, larger ones where there are many
  p.items = n <= uint64_t(p.block) * 2 * 128 ? 2 : n <= uint64_t(p.block) * 4 * 512 ? 4 : 16;
  const uint64_t tile = uint64_t(p.block) * p.items;
  p.tiles = uint32_t((n + tile - 1) / tile);
  return p;
}

template <typename ID>
int launch_sort(uint64_t n, const ID* ids, uint32_t experts, int32_t* offsets, int32_t* position,
                int32_t* source, void* work, cudaStream_t stream) {
  const SortPlan p = plan_sort(n, experts);
  if (p.cluster != 0) {
    auto kernel = p.items == 1 ? sort_cluster_kernel<ID, 1> : sort_cluster_kernel<ID, 4>;
    if (p.cluster == 1) {
      kernel<<<1, p.block, 0, stream>>>(ids, n, experts, offsets, position, source);
      return rows_launched();
    }
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(p.cluster);
    config.blockDim = dim3(p.block);
    config.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = p.cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    const cudaError_t e =
        cudaLaunchKernelEx(&config, kernel, ids, n, experts, offsets, position, source);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return rows_fail(HKV_ERR_CUDA, cudaGetErrorString(e));
    }
    return HKV_OK;
  }
  uint32_t* counts = static_cast<uint32_t*>(work);
  uint32_t* totals = uint64_t(p.tiles) * experts > kCountsSummed ? counts + uint64_t(p.tiles) * experts : nullptr;
  sort_count_kernel<ID><<<p.tiles, 1024, 0, stream>>>(ids, n, experts, p.block * p.items, counts);
  if (totals != nullptr) {
    sort_scan_kernel<<<(experts + 31u) / 32u, 1024, 0, stream>>>(experts, p.tiles, counts, totals);
  }
  auto place = p.items == 2   ? sort_place_kernel<ID, 2>
               : p.items == 4 ? sort_place_kernel<ID, 4>
                              : sort_place_kernel<ID, 16>;
  place<<<p.tiles, p.block, 0, stream>>>(ids, n, experts, counts, totals, offsets, position, source);
  return rows_launched();
}

// ---- rows -----------------------------------------------------------------------
//
// The three operators below are bound by HBM.  A group of lanes (a power of two up
// to a warp) takes a part of a token's row, V units per lane, and goes through the
// token's assignments: their places and weights are looked up once for V units.

constexpr int kMoveBlock = 256;

// How many units a lane takes at a time, and for how many assignments: as many
// loads as keep the memory busy while the registers leave room for enough warps.
// Measured, us, units x assignments (16-byte units; dispatch and combine 16384 tokens
// of 8 rows of 4096 bf16, combine 300000 of 2 of 64 f32, gradient of combine 8192 of 8
// of 2048 bf16 and 65536 of 2 of 128 f32; units of 2: 20000 of 6 of 1001 half; units
// of 4: 30000 of 4 of 334 bf16 and 333 f32):
//   dispatch            2: 187    1: 195    4: 190    8: 190
//     units of 4        4: 17.6   8: 21.2
//   combine             2 x 2: 182, 37   1 x 4: 184    2 x 3: 177   4 x 2: -, 48
//     units of 2        8 x 1: 64   8 x 2: 66   4 x 1: 94   4 x 2: 71   8 x 4: 82   12 x 1: 116
//     units of 4        8 x 1: 30, 36   8 x 2: 29, 35   4 x 2: 28, 36   4 x 1: 29, 44   4 x 4: 26, 42
//   gradient of combine 2 x 4: 93    2 x 2: 97, 29    1 x 4: 101    4 x 2: 97, 28
//     units of 2        8 x 2: 129   4 x 3: 134   4 x 2: 142   8 x 1: 145
//     units of 4        4 x 2: 45, 73   8 x 2: 48, 73   4 x 3: 57, 77   8 x 1: 64, 84
// The gradient of combine takes 2 x 4 where a token has more than two experts.  With one or
// two half or more of the four places would stay empty, so there it takes 4 x 2 (4 x 2 and
// 2 x 4, one expert: 65536 x 128 f32 18 and 28, 16384 x 2048 bf16 34 and 50, 8192 x 4096 f32
// 69 and 91, 300000 x 64 bf16 30 and 67; two: 28 and 33, 52 and 62, 107 and 118, 41 and 72;
// only 100 x 4096 bf16 goes the other way, 3.4 and 3.2).
struct Shape {
  int units, assigned;
};
constexpr Shape dispatch_shape(int unit) {
  return unit == 16 ? Shape{2, 0} : unit == 4 ? Shape{4, 0} : Shape{8, 0};
}
constexpr Shape combine_shape(int unit) { return unit == 16 ? Shape{2, 2} : Shape{8, 1}; }
constexpr Shape backward_shape(int unit, bool few) {
  return unit == 2 ? Shape{8, 2} : unit == 4 || few ? Shape{4, 2} : Shape{2, 4};
}

// The part of a token's row that a group of LANES lanes takes: V units per lane.
struct RowParts {
  uint32_t units;    // of a row
  uint32_t parts;    // per row
  uint64_t magic;    // floor(2^64 / parts) + 1, 0 for one part: division by multiplication,
                     // exact while the dividend times the divisor stays below 2^64
};

template <int LANES, int V>
struct MyPart {
  uint64_t token;
  uint32_t first;    // unit v of the lane is first + v * LANES
  bool full;         // the part has all its units
  uint32_t units;
  __device__ __forceinline__ explicit MyPart(const RowParts& p) {
    const uint64_t task = (uint64_t(blockIdx.x) * kMoveBlock + threadIdx.x) / LANES;
    token = p.magic == 0 ? task : __umul64hi(task, p.magic);
    const uint32_t begin = uint32_t(task - token * p.parts) * (LANES * V);
    first = begin + (threadIdx.x & (LANES - 1u));
    full = begin + LANES * V <= p.units;
    units = p.units;
  }
  __device__ __forceinline__ bool has(int v) const { return first + v * LANES < units; }
};

// Zeroes the rows behind the last expert's, if the caller asked for it.
template <int BYTES>
__device__ __forceinline__ void zero_behind(const int32_t* kept, uint64_t n, uint8_t* rows,
                                            uint64_t rows_stride, uint32_t units) {
  using Raw = typename VecType<BYTES>::type;
  if (kept == nullptr) return;
  for (uint64_t r = uint64_t(max(*kept, 0)) + blockIdx.x; r < n; r += gridDim.x) {
    Raw* row = reinterpret_cast<Raw*>(rows + r * rows_stride);
    for (uint32_t u = threadIdx.x; u < units; u += blockDim.x) row[u] = Raw{};
  }
}

// ---- dispatch
//
// T rows read, N written: a lane loads its units of the token's row and stores
// them to the row's k places, so every row is read once whatever k is.
template <int BYTES, int LANES, int V, bool FULL>
__device__ __forceinline__ void dispatch_part(const MyPart<LANES, V>& my, uint64_t n, uint32_t top_k,
                                              const RowsIn& x, const int32_t* __restrict__ position,
                                              uint8_t* __restrict__ rows, uint64_t rows_stride) {
  using Raw = typename VecType<BYTES>::type;
  const Raw* from = reinterpret_cast<const Raw*>(x.first + my.token * x.stride) + my.first;
  Raw v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (FULL || my.has(i)) v[i] = __ldg(from + i * LANES);
  }
  const int32_t* at = position + my.token * top_k;
  for (uint32_t j = 0; j < top_k; ++j) {
    const uint32_t place = uint32_t(__ldg(at + j));   // -1 is above every place
    if (place >= n) continue;
    Raw* to = reinterpret_cast<Raw*>(rows + place * rows_stride) + my.first;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (FULL || my.has(i)) to[i * LANES] = v[i];
    }
  }
}

template <int BYTES, int LANES, int V>
__global__ void __launch_bounds__(kMoveBlock)
    dispatch_kernel(const uint64_t tokens, const uint32_t top_k, const RowParts parts, const RowsIn x,
                    const int32_t* __restrict__ position, uint8_t* __restrict__ rows,
                    const uint64_t rows_stride, const int32_t* __restrict__ kept) {
  const uint64_t n = tokens * top_k;
  zero_behind<BYTES>(kept, n, rows, rows_stride, parts.units);
  const MyPart<LANES, V> my(parts);
  if (my.token >= tokens) return;
  if (my.full) dispatch_part<BYTES, LANES, V, true>(my, n, top_k, x, position, rows, rows_stride);
  else dispatch_part<BYTES, LANES, V, false>(my, n, top_k, x, position, rows, rows_stride);
}

// J assignments of a token, from j0 on: their rows' places and weights.  No branch
// stands between the loads, so that all of them are in flight together (with one
// per assignment, to skip the dropped, 16384 x 4096 bf16 of 8 rows each took 272 us
// instead of 190): beyond the last assignment the last is read again, a dropped
// one reads row 0, and neither is used.
template <typename T, int J>
struct Assigned {
  uint32_t place[J];   // 0 if not ok
  bool ok[J];
  float w[J];
  __device__ __forceinline__ Assigned(uint64_t token, uint32_t top_k, uint32_t j0, uint64_t n,
                                      const int32_t* __restrict__ position,
                                      const void* __restrict__ weights, bool weights_f32) {
    const uint64_t first = token * top_k;
#pragma unroll
    for (int u = 0; u < J; ++u) {
      place[u] = uint32_t(__ldg(position + first + min(j0 + u, top_k - 1u)));
      w[u] = 1.f;
    }
    if (weights != nullptr) {
      if (weights_f32) {
        const float* from = static_cast<const float*>(weights) + first;
#pragma unroll
        for (int u = 0; u < J; ++u) w[u] = __ldg(from + min(j0 + u, top_k - 1u));
      } else {
        const T* from = static_cast<const T*>(weights) + first;
#pragma unroll
        for (int u = 0; u < J; ++u) w[u] = to_float(from[min(j0 + u, top_k - 1u)]);
      }
    }
#pragma unroll
    for (int u = 0; u < J; ++u) {
      ok[u] = j0 + u < top_k && place[u] < n;   // -1 is above every place
      place[u] = ok[u] ? place[u] : 0u;
    }
  }
};

// ---- combine
//
// N rows read, T written: a lane sums its units of the k rows in registers, in the
// order of j, with the loads of J assignments in flight.
template <typename T, int BYTES, int LANES, int V, int J, bool FULL>
__device__ __forceinline__ void combine_part(const MyPart<LANES, V>& my, uint64_t n, uint32_t top_k,
                                             const RowsIn& rows, const void* __restrict__ weights,
                                             bool weights_f32, const int32_t* __restrict__ position,
                                             uint8_t* __restrict__ out, uint64_t out_stride) {
  using U = Unit<T, BYTES>;
  using Raw = typename U::Raw;
  float sum[V][U::kElems];
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int e = 0; e < U::kElems; ++e) sum[i][e] = 0.f;
  }
#pragma unroll 1
  for (uint32_t j0 = 0; j0 < top_k; j0 += J) {
    const Assigned<T, J> a(my.token, top_k, j0, n, position, weights, weights_f32);
    Raw row[J][V];
#pragma unroll
    for (int u = 0; u < J; ++u) {
      const Raw* from = reinterpret_cast<const Raw*>(rows.first + a.place[u] * rows.stride) + my.first;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        row[u][v] = no_unit<Raw>();
        if (FULL || my.has(v)) row[u][v] = __ldg(from + v * LANES);
      }
    }
#pragma unroll
    for (int u = 0; u < J; ++u) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float f[U::kElems];
        U::unpack(row[u][v], f);
#pragma unroll
        for (int e = 0; e < U::kElems; ++e) {
          if (a.ok[u]) sum[v][e] = fmaf(a.w[u], f[e], sum[v][e]);
        }
      }
    }
  }
  Raw* to = reinterpret_cast<Raw*>(out + my.token * out_stride) + my.first;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (FULL || my.has(v)) to[v * LANES] = U::pack(sum[v]);
  }
}

template <typename T, int BYTES, int LANES, int V, int J>
__global__ void __launch_bounds__(kMoveBlock)
    combine_kernel(const uint64_t tokens, const uint32_t top_k, const RowParts parts, const RowsIn rows,
                   const void* __restrict__ weights, const bool weights_f32,
                   const int32_t* __restrict__ position, uint8_t* __restrict__ out,
                   const uint64_t out_stride) {
  const MyPart<LANES, V> my(parts);
  if (my.token >= tokens) return;
  const uint64_t n = tokens * top_k;
  if (my.full) {
    combine_part<T, BYTES, LANES, V, J, true>(my, n, top_k, rows, weights, weights_f32, position, out,
                                              out_stride);
  } else {
    combine_part<T, BYTES, LANES, V, J, false>(my, n, top_k, rows, weights, weights_f32, position, out,
                                               out_stride);
  }
}

// ---- combine, backward
//
// T + N rows read, N written.  A group of threads takes a token's whole row (the
// dot products run over it): LANES of a warp, or (LANES == 32) some warps, which go
// over it in steps of V units per lane.  For J assignments at a time a lane loads
// its units of the rows, stores w * d_out and adds to its J partial dot products,
// which the group sums at the end.
template <typename T, int BYTES, int LANES, int V, int J, bool FULL>
__device__ __forceinline__ void combine_backward_step(
    uint32_t first, uint32_t units, const Assigned<T, J>& a,
    const typename Unit<T, BYTES>::Raw* __restrict__ d_from,
    const typename Unit<T, BYTES>::Raw* const (&from)[J], typename Unit<T, BYTES>::Raw* const (&to)[J],
    float (&dot)[J]) {
  using U = Unit<T, BYTES>;
  using Raw = typename U::Raw;
  Raw d[V], row[J][V];
  // from here on constants tell the units apart, which cost no instructions
  const Raw* d_at = d_from + first;
  const Raw* at[J];
#pragma unroll
  for (int u = 0; u < J; ++u) at[u] = from[u] + first;
  float part[J];   // the step's share of the dot products, added to them at once
#pragma unroll
  for (int u = 0; u < J; ++u) part[u] = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    d[v] = no_unit<Raw>();
    if (FULL || first + v * LANES < units) d[v] = __ldg(d_at + v * LANES);
  }
#pragma unroll
  for (int u = 0; u < J; ++u) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      row[u][v] = no_unit<Raw>();
      if (FULL || first + v * LANES < units) row[u][v] = __ldg(at[u] + v * LANES);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float f[U::kElems];
    U::unpack(d[v], f);
#pragma unroll
    for (int u = 0; u < J; ++u) {
      float y[U::kElems];
      U::unpack(row[u][v], y);
#pragma unroll
      for (int e = 0; e < U::kElems; ++e) {
        part[u] = fmaf(f[e], y[e], part[u]);
        y[e] = a.w[u] * f[e];
      }
      if (a.ok[u] && (FULL || first + v * LANES < units)) (to[u] + first)[v * LANES] = U::pack(y);
    }
  }
#pragma unroll
  for (int u = 0; u < J; ++u) {
    if (a.ok[u]) dot[u] += part[u];
  }
}

template <typename T, int BYTES, int LANES, int V, int J>
__global__ void __launch_bounds__(256)
    combine_backward_kernel(const uint64_t tokens, const uint32_t top_k, const uint32_t units,
                            const uint32_t warps, const RowsIn d_out, const RowsIn rows,
                            const void* __restrict__ weights, const bool weights_f32,
                            const int32_t* __restrict__ position, uint8_t* __restrict__ d_rows,
                            const uint64_t d_rows_stride, void* __restrict__ d_weights,
                            const int32_t* __restrict__ kept) {
  using Raw = typename Unit<T, BYTES>::Raw;
  __shared__ float partial[8][J];
  const uint64_t n = tokens * top_k;
  zero_behind<BYTES>(kept, n, d_rows, d_rows_stride, units);
  // warps: of a group, a power of two; the part of the row between its warps' steps
  const uint32_t group = LANES == 32 ? warps * 32u : uint32_t(LANES);
  const uint32_t lane = threadIdx.x & (group - 1u);
  const uint64_t token = (uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) / group;
  const bool live = token < tokens;
  const Raw* d_from = reinterpret_cast<const Raw*>(d_out.first + token * d_out.stride);
#pragma unroll 1
  for (uint32_t j0 = 0; j0 < top_k; j0 += J) {
    const Assigned<T, J> a(live ? token : 0, top_k, j0, n, position, weights, weights_f32);
    const Raw* from[J];
    Raw* to[J];
    float dot[J];
#pragma unroll
    for (int u = 0; u < J; ++u) {
      from[u] = reinterpret_cast<const Raw*>(rows.first + a.place[u] * rows.stride);
      to[u] = reinterpret_cast<Raw*>(d_rows + a.place[u] * d_rows_stride);
      dot[u] = 0.f;
    }
    if (live) {
      const uint32_t own = threadIdx.x & (LANES - 1u);
#pragma unroll 1
      for (uint32_t begin = (lane - own) * V; begin < units; begin += group * V) {
        if (begin + LANES * V <= units) {
          combine_backward_step<T, BYTES, LANES, V, J, true>(begin + own, units, a, d_from, from, to, dot);
        } else {
          combine_backward_step<T, BYTES, LANES, V, J, false>(begin + own, units, a, d_from, from, to, dot);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < J; ++u) {
#pragma unroll
      for (int d = LANES >> 1; d > 0; d >>= 1) dot[u] += __shfl_xor_sync(kFull, dot[u], d);
    }
    if (group > 32u) {   // uniform over the block: all of it arrives
      __syncthreads();
      const uint32_t warp = threadIdx.x >> 5;
      if ((threadIdx.x & 31u) == 0) {
#pragma unroll
        for (int u = 0; u < J; ++u) partial[warp][u] = dot[u];
      }
      __syncthreads();
      if (lane == 0) {
        for (uint32_t v = 1; v < group >> 5; ++v) {
#pragma unroll
          for (int u = 0; u < J; ++u) dot[u] += partial[warp + v][u];
        }
      }
    }
    if (live && lane == 0) {
#pragma unroll
      for (int u = 0; u < J; ++u) {
        if (j0 + u >= top_k) continue;
        const uint64_t i = token * top_k + j0 + u;
        if (weights_f32) static_cast<float*>(d_weights)[i] = dot[u];
        else static_cast<T*>(d_weights)[i] = from_float<T>(dot[u]);
      }
    }
  }
}

uint32_t pow2_at_least(uint64_t v) {
  uint32_t p = 1;
  while (p < v) p <<= 1;
  return p;
}

// Lanes on a part of a row of `units` units with `per_lane` units each: a warp where
// the row has units for all its lanes, else eight, or two where the row has no more.
uint32_t lanes_for(uint64_t units, uint32_t per_lane) {
  return units >= 32ull * per_lane ? 32 : units > 2ull * per_lane ? 8 : 2;
}
RowParts row_parts(uint64_t units, uint32_t lanes, uint32_t per_lane) {
  RowParts p{};
  p.units = uint32_t(units);
  const uint64_t part = uint64_t(lanes) * per_lane;
  p.parts = uint32_t((units + part - 1) / part);
  p.magic = p.parts == 1 ? 0 : ~0ull / p.parts + 1;
  return p;
}
// CALL(LANES) for the number of lanes.
#define HKV_FOR_LANES(lanes, CALL) \
  switch (lanes) {                 \
    case 32: CALL(32); break;      \
    case 8: CALL(8); break;        \
    default: CALL(2); break;       \
  }

int check_order(uint64_t tokens, uint32_t top_k, uint32_t experts) {
  HKV_ROWS_CHECK(top_k >= 1 && top_k <= kMaxTopK, "top_k must be between 1 and 64");
  HKV_ROWS_CHECK(experts >= 1 && experts <= kMaxExperts, "experts must be between 1 and 1024");
  HKV_ROWS_CHECK(tokens < (1ull << 31) && tokens * top_k < (1ull << 31),
                 "batches of 2^31 or more assignments");
  return HKV_OK;
}

// Blocks of `threads` threads for `items` threads' work.
int grid_of(uint64_t items, uint32_t threads, unsigned* grid) noexcept {
  const uint64_t blocks = (items + threads - 1) / threads;
  HKV_ROWS_CHECK(blocks < (1ull << 31), "batch too large for one launch");
  *grid = unsigned(blocks);
  return HKV_OK;
}

}  // namespace
}  // namespace hkv

using namespace hkv;

extern "C" {

const char* hkv_rows_last_error(void) { return g_rows_error.c_str(); }

uint64_t hkv_expert_sort_workspace_bytes(uint64_t tokens, uint32_t top_k, uint32_t experts) {
  if (check_order(tokens, top_k, experts) != HKV_OK) return 0;
  const uint64_t n = tokens * top_k;
  const SortPlan p = plan_sort(n, experts);
  return p.cluster != 0 ? 0 : (uint64_t(p.tiles) + 1) * experts * sizeof(uint32_t);
}

int hkv_expert_sort(uint64_t tokens, uint32_t top_k, const void* expert_ids, uint32_t id_bytes,
                    uint32_t experts, int32_t* offsets, int32_t* position, int32_t* source,
                    void* work, uint64_t work_bytes, hkv_stream stream) {
  const int rc = check_order(tokens, top_k, experts);
  if (rc != HKV_OK) return rc;
  HKV_ROWS_CHECK(id_bytes == 4 || id_bytes == 8, "expert ids are int32 or int64");
  const uint64_t n = tokens * top_k;
  HKV_ROWS_CHECK(offsets != nullptr, "offsets must not be null");
  HKV_ROWS_CHECK(n == 0 || (expert_ids != nullptr && position != nullptr && source != nullptr),
                 "expert_ids, position and source must not be null");
  HKV_ROWS_CHECK(work_bytes >= hkv_expert_sort_workspace_bytes(tokens, top_k, experts) &&
                     (work_bytes == 0 || work != nullptr),
                 "workspace smaller than hkv_expert_sort_workspace_bytes");
  HKV_ROWS_CHECK(all_aligned(id_bytes, expert_ids) && all_aligned(4, offsets, position, source, work),
                 "a buffer does not start at a multiple of its element size, or work of 4");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return id_bytes == 4
             ? launch_sort(n, static_cast<const int32_t*>(expert_ids), experts, offsets, position,
                           source, work, s)
             : launch_sort(n, static_cast<const int64_t*>(expert_ids), experts, offsets, position,
                           source, work, s);
}

int hkv_expert_dispatch(uint64_t tokens, uint32_t top_k, uint64_t row_bytes, const void* x,
                        uint64_t x_stride, uint32_t experts, const int32_t* offsets,
                        const int32_t* position, void* rows, uint64_t rows_stride,
                        int zero_rows_behind, hkv_stream stream) {
  int rc = check_order(tokens, top_k, experts);
  if (rc != HKV_OK) return rc;
  HKV_ROWS_CHECK(row_bytes >= 1 && row_bytes < (1ull << 30), "row_bytes must be between 1 and 2^30 - 1");
  HKV_ROWS_CHECK(rows_stride >= row_bytes, "the sorted rows overlap");
  if (tokens == 0) return HKV_OK;
  HKV_ROWS_CHECK(x != nullptr && position != nullptr && rows != nullptr && offsets != nullptr,
                 "x, offsets, position and rows must not be null");
  HKV_ROWS_CHECK(all_aligned(4, offsets, position),
                 "offsets and position must start at a multiple of their element size");
  const uint64_t bits = row_bytes | address_bits(x) | x_stride | address_bits(rows) | rows_stride;
  uint32_t unit = 16;
  while (bits % unit != 0) unit >>= 1;
  const uint32_t per_lane = dispatch_shape(unit).units;
  const uint32_t lanes = lanes_for(row_bytes / unit, per_lane);
  const RowParts parts = row_parts(row_bytes / unit, lanes, per_lane);
  unsigned grid = 0;
  rc = grid_of(tokens * parts.parts * lanes, kMoveBlock, &grid);
  if (rc != HKV_OK) return rc;
  const RowsIn in = rows_in(x, x_stride);
  const int32_t* kept = zero_rows_behind ? offsets + experts : nullptr;
#define HKV_RUN(BYTES, LANES)                                                            \
  dispatch_kernel<BYTES, LANES, dispatch_shape(BYTES).units>                             \
      <<<grid, kMoveBlock, 0, static_cast<cudaStream_t>(stream)>>>(                      \
          tokens, top_k, parts, in, position, static_cast<uint8_t*>(rows), rows_stride, kept)
#define HKV_CALL(LANES)                     \
  switch (unit) {                           \
    case 16: HKV_RUN(16, LANES); break;     \
    case 8: HKV_RUN(8, LANES); break;       \
    case 4: HKV_RUN(4, LANES); break;       \
    case 2: HKV_RUN(2, LANES); break;       \
    default: HKV_RUN(1, LANES); break;      \
  }
  HKV_FOR_LANES(lanes, HKV_CALL)
#undef HKV_CALL
#undef HKV_RUN
  return rows_launched();
}

int hkv_expert_combine(uint64_t tokens, uint32_t top_k, uint64_t dim, uint32_t value_kind,
                       const void* rows, uint64_t rows_stride, const void* weights,
                       uint32_t weight_kind, const int32_t* position, void* out,
                       uint64_t out_stride, hkv_stream stream) {
  int rc = check_order(tokens, top_k, 1);
  if (rc != HKV_OK) return rc;
  HKV_ROWS_CHECK(is_row_kind(value_kind), "rows are float32, float16 or bfloat16");
  HKV_ROWS_CHECK(weights == nullptr || weight_kind == value_kind || weight_kind == kValueF32,
                 "weights have the rows' type or float32");
  const uint32_t size = row_kind_size(value_kind);
  HKV_ROWS_CHECK(dim >= 1 && dim < (1ull << 28), "dim must be between 1 and 2^28 - 1");
  HKV_ROWS_CHECK(out_stride >= dim * size, "the output rows overlap");
  if (tokens == 0) return HKV_OK;
  HKV_ROWS_CHECK(rows != nullptr && position != nullptr && out != nullptr,
                 "rows, position and out must not be null");
  HKV_ROWS_CHECK(all_aligned(4, position) && all_aligned(row_kind_size(weight_kind), weights),
                 "position and weights must start at a multiple of their element size");
  const uint64_t row_bytes = dim * size;
  const uint32_t unit =
      unit_bytes(row_bytes | address_bits(rows) | rows_stride | address_bits(out) | out_stride, size);
  HKV_ROWS_CHECK(unit != 0, "a row does not start at a multiple of its element size");
  const uint32_t per_lane = combine_shape(unit).units;
  const uint32_t lanes = lanes_for(row_bytes / unit, per_lane);
  const RowParts parts = row_parts(row_bytes / unit, lanes, per_lane);
  unsigned grid = 0;
  rc = grid_of(tokens * parts.parts * lanes, kMoveBlock, &grid);
  if (rc != HKV_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const RowsIn in = rows_in(rows, rows_stride);
#define HKV_LANES(LANES)                                                                  \
  combine_kernel<RowT, kUnit, LANES, combine_shape(kUnit).units,                          \
                 combine_shape(kUnit).assigned><<<grid, kMoveBlock, 0, s>>>(              \
      tokens, top_k, parts, in, weights, weight_kind == kValueF32, position,              \
      static_cast<uint8_t*>(out), out_stride)
#define HKV_CALL(T, BYTES)         \
  using RowT = T;                  \
  constexpr int kUnit = BYTES;     \
  HKV_FOR_LANES(lanes, HKV_LANES)
  HKV_FOR_UNIT(value_kind, unit, HKV_CALL)
#undef HKV_CALL
#undef HKV_LANES
  return rows_launched();
}

int hkv_expert_combine_backward(uint64_t tokens, uint32_t top_k, uint64_t dim, uint32_t value_kind,
                                const void* d_out, uint64_t d_out_stride, const void* rows,
                                uint64_t rows_stride, const void* weights, uint32_t weight_kind,
                                uint32_t experts, const int32_t* offsets, const int32_t* position,
                                void* d_rows, uint64_t d_rows_stride, int zero_rows_behind,
                                void* d_weights, hkv_stream stream) {
  int rc = check_order(tokens, top_k, experts);
  if (rc != HKV_OK) return rc;
  HKV_ROWS_CHECK(is_row_kind(value_kind), "rows are float32, float16 or bfloat16");
  HKV_ROWS_CHECK(weight_kind == value_kind || weight_kind == kValueF32,
                 "weights have the rows' type or float32");
  const uint32_t size = row_kind_size(value_kind);
  HKV_ROWS_CHECK(dim >= 1 && dim < (1ull << 28), "dim must be between 1 and 2^28 - 1");
  HKV_ROWS_CHECK(d_rows_stride >= dim * size, "the rows of the gradient overlap");
  if (tokens == 0) return HKV_OK;
  HKV_ROWS_CHECK(d_out != nullptr && rows != nullptr && weights != nullptr && offsets != nullptr &&
                     position != nullptr && d_rows != nullptr && d_weights != nullptr,
                 "no argument may be null");
  HKV_ROWS_CHECK(all_aligned(4, offsets, position) &&
                     all_aligned(row_kind_size(weight_kind), weights, d_weights),
                 "offsets, position and weights must start at a multiple of their element size");
  const uint64_t row_bytes = dim * size;
  const uint32_t unit = unit_bytes(row_bytes | address_bits(d_out) | d_out_stride | address_bits(rows) |
                                       rows_stride | address_bits(d_rows) | d_rows_stride,
                                   size);
  HKV_ROWS_CHECK(unit != 0, "a row does not start at a multiple of its element size");
  const uint64_t units = row_bytes / unit;
  const bool few = top_k <= 2;
  const uint32_t per_lane = backward_shape(unit, few).units;
  const uint32_t lanes = lanes_for(units, per_lane);
  // a warp goes over four steps of a row at least, which spreads what it does per
  // row; more warps share one where there are too few tokens to fill the device
  const uint64_t step = 32ull * per_lane;
  uint32_t warps = 1;
  while (warps < 8 && (units >= step * 8 * warps ||
                       (units > step * warps && tokens * warps < uint64_t(sm_count()) * 16))) {
    warps <<= 1;
  }
  unsigned grid = 0;
  rc = grid_of(tokens * (lanes == 32 ? warps * 32 : lanes), 256, &grid);
  if (rc != HKV_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const RowsIn d_in = rows_in(d_out, d_out_stride);
  const RowsIn in = rows_in(rows, rows_stride);
  const int32_t* kept = zero_rows_behind ? offsets + experts : nullptr;
#define HKV_RUN(T, BYTES, LANES, FEW)                                                               \
  combine_backward_kernel<T, BYTES, LANES, backward_shape(BYTES, FEW).units,                        \
                          backward_shape(BYTES, FEW).assigned><<<grid, 256, 0, s>>>(                \
      tokens, top_k, uint32_t(units), warps, d_in, in, weights, weight_kind == kValueF32, position, \
      static_cast<uint8_t*>(d_rows), d_rows_stride, d_weights, kept)
#define HKV_LANES(LANES)                                       \
  if (kUnit != 16 || few) HKV_RUN(RowT, kUnit, LANES, true);   \
  else HKV_RUN(RowT, kUnit, LANES, (kUnit != 16))
#define HKV_CALL(T, BYTES)         \
  using RowT = T;                  \
  constexpr int kUnit = BYTES;     \
  HKV_FOR_LANES(lanes, HKV_LANES)
  HKV_FOR_UNIT(value_kind, unit, HKV_CALL)
#undef HKV_CALL
#undef HKV_LANES
#undef HKV_RUN
  return rows_launched();
}

}  // extern "C"
