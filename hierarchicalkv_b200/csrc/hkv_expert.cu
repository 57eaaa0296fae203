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
// Nothing is accumulated with atomics: results do not depend on the order in
// which blocks run.
//
// The reference has no such operators; hkv_shard.cu groups keys by their
// owner rank and moves whole rows by index, unordered inside an owner.
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

int sm_count() noexcept {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
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

// Large batches: count per tile, scan over the tiles, place.  Up to
// kTilesSummed tiles the placing blocks sum the counts of the tiles before theirs
// themselves and the scan's launch is saved.
constexpr uint32_t kTilesSummed = 64;

template <typename ID>
__global__ void __launch_bounds__(512)
    sort_count_kernel(const ID* __restrict__ ids, const uint64_t n, const uint32_t experts,
                      const uint32_t tile, uint32_t* __restrict__ counts) {
  __shared__ uint32_t local[kMaxExperts];
  for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) local[e] = 0;
  __syncthreads();
  const uint64_t first = uint64_t(blockIdx.x) * tile;
  const uint64_t last = min(n, first + tile);
  for (uint64_t at = first + threadIdx.x; at < last; at += blockDim.x) {
    const ID id = ids[at];
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
  // tiles that still fill the device, large ones where there are many
  p.items = n <= uint64_t(p.block) * 4 * 512 ? 4 : 16;
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
  uint32_t* totals = p.tiles > kTilesSummed ? counts + uint64_t(p.tiles) * experts : nullptr;
  sort_count_kernel<ID><<<p.tiles, 512, 0, stream>>>(ids, n, experts, p.block * p.items, counts);
  if (totals != nullptr) {
    sort_scan_kernel<<<(experts + 31u) / 32u, 1024, 0, stream>>>(experts, p.tiles, counts, totals);
  }
  auto place = p.items == 4 ? sort_place_kernel<ID, 4> : sort_place_kernel<ID, 16>;
  place<<<p.tiles, p.block, 0, stream>>>(ids, n, experts, counts, totals, offsets, position, source);
  return rows_launched();
}

// ---- dispatch -----------------------------------------------------------------
//
// Bound by HBM: T rows read, N written.  Token by token: a thread loads one
// chunk of a token's row and stores it to the row's k places, so every row is
// read from memory once whatever k is.  Unaligned rows: the thread owns chunk i
// of each place instead (places have alignments of their own) and cuts it out of
// the token's row, which is in L1 after the first place.

constexpr int kMoveBlock = 256;

// Division by the chunks of a row, by multiplication: exact while the dividend
// times the divisor stays below 2^64.
struct PerRow {
  uint32_t chunks;
  uint64_t magic;   // floor(2^64 / chunks) + 1; 0 for one chunk
  __device__ __forceinline__ uint64_t row(uint64_t c) const {
    return magic == 0 ? c : __umul64hi(c, magic);
  }
};

// Zeroes the rows behind the last expert's, if the caller asked for it.
template <int G>
__device__ __forceinline__ void zero_behind(const int32_t* kept, uint64_t n, uint8_t* rows,
                                            uint64_t rows_stride, uint64_t row_bytes) {
  if (kept == nullptr) return;
  for (uint64_t r = uint64_t(max(*kept, 0)) + blockIdx.x; r < n; r += gridDim.x) {
    uint8_t* row = rows + r * rows_stride;
    const int ahead = int(reinterpret_cast<uintptr_t>(row) & 15u);
    for (int64_t at = threadIdx.x * 16ll - ahead; at < int64_t(row_bytes); at += blockDim.x * 16ll) {
      store_chunk<G>(row, int(at), make_uint4(0, 0, 0, 0), 0, int(row_bytes));
    }
  }
}

// G == 0: all rows are whole aligned chunks; else pieces of G bytes at their ends.
template <int G>
__global__ void __launch_bounds__(kMoveBlock)
    dispatch_kernel(const uint64_t tokens, const uint32_t top_k, const PerRow per_row,
                    const uint32_t row_bytes, const RowsIn x, const int32_t* __restrict__ position,
                    uint8_t* __restrict__ rows, const uint64_t rows_stride,
                    const int32_t* __restrict__ kept) {
  const uint64_t n = tokens * top_k;
  zero_behind<(G ? G : 8)>(kept, n, rows, rows_stride, row_bytes);
  const uint64_t c = uint64_t(blockIdx.x) * kMoveBlock + threadIdx.x;
  const uint64_t token = per_row.row(c);
  if (token >= tokens) return;
  const uint32_t off = uint32_t(c - token * per_row.chunks) * 16;
  const int32_t* at = position + token * top_k;
  const uint8_t* from = x.first + token * x.stride;
  if (G == 0) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(from + off));
    for (uint32_t j = 0; j < top_k; ++j) {
      const uint32_t place = uint32_t(at[j]);   // -1 is above every place
      if (place < n) *reinterpret_cast<uint4*>(rows + place * rows_stride + off) = v;
    }
  } else {
    for (uint32_t j = 0; j < top_k; ++j) {
      const uint32_t place = uint32_t(at[j]);
      if (place >= n) continue;
      uint8_t* row = rows + place * rows_stride;
      const int o = int(off) - int(reinterpret_cast<uintptr_t>(row) & 15u);
      if (o >= int(row_bytes)) continue;
      Cut cut;
      cut.load(from + o, x.first, x.last);
      store_chunk<(G ? G : 8)>(row, o, cut.get<(G ? G : 8)>(from + o, from, from + row_bytes), 0,
                               int(row_bytes));
    }
  }
}

// ---- combine ------------------------------------------------------------------
//
// Bound by HBM: N rows read, T written.  A thread owns one chunk of a token's
// output row and sums the k rows' chunks in registers, in the order of j.

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(kMoveBlock)
    combine_kernel(const uint64_t tokens, const uint32_t top_k, const PerRow per_row,
                   const uint32_t row_bytes, const RowsIn rows, const void* __restrict__ weights,
                   const bool weights_f32, const int32_t* __restrict__ position,
                   uint8_t* __restrict__ out, const uint64_t out_stride) {
  constexpr int kElems = kChunkElems<T>;
  const uint64_t c = uint64_t(blockIdx.x) * kMoveBlock + threadIdx.x;
  const uint64_t token = per_row.row(c);
  if (token >= tokens) return;
  const uint64_t n = tokens * top_k;
  uint8_t* to = out + token * out_stride;
  int off = int(c - token * per_row.chunks) * 16;
  if (!WHOLE) off -= int(reinterpret_cast<uintptr_t>(to) & 15u);
  if (!WHOLE && off >= int(row_bytes)) return;
  float sum[kElems];
#pragma unroll
  for (int e = 0; e < kElems; ++e) sum[e] = 0.f;
  for (uint32_t j0 = 0; j0 < top_k; j0 += 4) {
    uint4 row[4];
    Cut cut[WHOLE ? 1 : 4];
    const uint8_t* from[4];
    float w[4];
    bool ok[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint64_t i = token * top_k + j0 + u;
      uint32_t place = kFull;
      if (j0 + u < top_k) place = uint32_t(position[i]);
      ok[u] = place < n;
      from[u] = rows.first + (ok[u] ? place * rows.stride : 0);
      w[u] = 1.f;
      if (ok[u] && weights != nullptr) {
        w[u] = weights_f32 ? static_cast<const float*>(weights)[i]
                           : to_float(static_cast<const T*>(weights)[i]);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (WHOLE) {
        if (ok[u]) row[u] = __ldg(reinterpret_cast<const uint4*>(from[u] + off));
      } else if (ok[u]) {
        cut[WHOLE ? 0 : u].load(from[u] + off, rows.first, rows.last);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (!ok[u]) continue;
      if (!WHOLE) {
        row[u] = cut[WHOLE ? 0 : u].template get<sizeof(T)>(from[u] + off, from[u],
                                                            from[u] + row_bytes);
      }
      float f[kElems];
      unpack<T>(row[u], f);
#pragma unroll
      for (int e = 0; e < kElems; ++e) sum[e] = fmaf(w[u], f[e], sum[e]);
    }
  }
  if (WHOLE) *reinterpret_cast<uint4*>(to + off) = pack<T>(sum);
  else store_chunk<sizeof(T)>(to, off, pack<T>(sum), 0, int(row_bytes));
}

// ---- combine, backward ----------------------------------------------------------
//
// Bound by HBM: T + N rows read, N written.  A group of threads takes a token;
// for four assignments at a time a lane loads its chunks of the rows, stores
// w * d_out and adds to its four partial dot products, which the group sums at
// the end.  d_out's chunk is loaded once for the four; with unaligned rows each
// place has its own cut of it, out of L1.

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(256)
    combine_backward_kernel(const uint64_t tokens, const uint32_t top_k, const uint32_t chunks,
                            const uint32_t group, const uint32_t row_bytes, const RowsIn d_out,
                            const RowsIn rows, const void* __restrict__ weights,
                            const bool weights_f32, const int32_t* __restrict__ position,
                            uint8_t* __restrict__ d_rows, const uint64_t d_rows_stride,
                            void* __restrict__ d_weights, const int32_t* __restrict__ kept) {
  constexpr int kElems = kChunkElems<T>;
  __shared__ float partial[8][4];
  const uint64_t n = tokens * top_k;
  zero_behind<sizeof(T)>(kept, n, d_rows, d_rows_stride, row_bytes);
  const uint32_t lane = threadIdx.x & (group - 1u);
  const uint64_t token = (uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) / group;
  const bool live = token < tokens;
  const uint8_t* d_from = d_out.first + token * d_out.stride;
  for (uint32_t j0 = 0; j0 < top_k; j0 += 4) {
    uint32_t place[4];
    float w[4], dot[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint64_t i = token * top_k + j0 + u;
      place[u] = kFull;
      w[u] = dot[u] = 0.f;
      if (live && j0 + u < top_k) {
        place[u] = uint32_t(position[i]);
        w[u] = weights_f32 ? static_cast<const float*>(weights)[i]
                           : to_float(static_cast<const T*>(weights)[i]);
      }
    }
    if (live) {
      for (uint32_t c = lane; c < chunks; c += group) {
        uint4 d[WHOLE ? 1 : 4], row[4];
        Cut d_cut[WHOLE ? 1 : 4], row_cut[WHOLE ? 1 : 4];
        int off[4];
        if (WHOLE) d[0] = __ldg(reinterpret_cast<const uint4*>(d_from + uint64_t(c) * 16));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (place[u] >= n) continue;
          const uint8_t* from = rows.first + place[u] * rows.stride;
          if (WHOLE) {
            row[u] = __ldg(reinterpret_cast<const uint4*>(from + uint64_t(c) * 16));
          } else {
            const uint8_t* to = d_rows + place[u] * d_rows_stride;
            off[u] = int(c) * 16 - int(reinterpret_cast<uintptr_t>(to) & 15u);
            row_cut[WHOLE ? 0 : u].none();
            d_cut[WHOLE ? 0 : u].none();
            if (off[u] < int(row_bytes)) {
              row_cut[WHOLE ? 0 : u].load(from + off[u], rows.first, rows.last);
              d_cut[WHOLE ? 0 : u].load(d_from + off[u], d_out.first, d_out.last);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (place[u] >= n) continue;
          if (!WHOLE) {
            const uint8_t* from = rows.first + place[u] * rows.stride;
            row[u] = row_cut[WHOLE ? 0 : u].template get<sizeof(T)>(from + off[u], from,
                                                                        from + row_bytes);
            d[WHOLE ? 0 : u] = d_cut[WHOLE ? 0 : u].template get<sizeof(T)>(
                d_from + off[u], d_from, d_from + row_bytes);
          }
          uint8_t* to = d_rows + place[u] * d_rows_stride;
          float du[kElems], y[kElems];
          unpack<T>(d[WHOLE ? 0 : u], du);
          unpack<T>(row[u], y);
          if (!WHOLE && (off[u] < 0 || off[u] + 16 > int(row_bytes))) {   // an end of the row
#pragma unroll
            for (int e = 0; e < kElems; ++e) {
              const int b = off[u] + e * int(sizeof(T));
              if (b < 0 || b >= int(row_bytes)) du[e] = y[e] = 0.f;
            }
          }
#pragma unroll
          for (int e = 0; e < kElems; ++e) {
            dot[u] = fmaf(du[e], y[e], dot[u]);
            du[e] *= w[u];
          }
          if (WHOLE) *reinterpret_cast<uint4*>(to + uint64_t(c) * 16) = pack<T>(du);
          else store_chunk<sizeof(T)>(to, off[u], pack<T>(du), 0, int(row_bytes));
        }
      }
    }
    const uint32_t width = group < 32u ? group : 32u;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      for (uint32_t d = width >> 1; d > 0; d >>= 1) dot[u] += __shfl_xor_sync(kFull, dot[u], d);
    }
    if (group > 32u) {   // uniform over the block: all of it arrives
      __syncthreads();
      const uint32_t warp = threadIdx.x >> 5;
      if ((threadIdx.x & 31u) == 0) {
#pragma unroll
        for (int u = 0; u < 4; ++u) partial[warp][u] = dot[u];
      }
      __syncthreads();
      if (lane == 0) {
        for (uint32_t v = 1; v < group >> 5; ++v) {
#pragma unroll
          for (int u = 0; u < 4; ++u) dot[u] += partial[warp + v][u];
        }
      }
    }
    if (live && lane == 0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
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

// Chunks per row: unaligned rows touch up to one more at either end.
uint32_t chunks_of(uint64_t row_bytes, bool whole) {
  return uint32_t(whole ? row_bytes / 16 : (row_bytes + 30) / 16);
}
PerRow per_row(uint32_t chunks) {
  return PerRow{chunks, chunks == 1 ? 0 : ~0ull / chunks + 1};
}

#define HKV_FOR_TYPE(kind, whole, CALL)                         \
  if ((kind) == hkv::kValueF32) {                               \
    if (whole) { CALL(float, true); } else { CALL(float, false); } \
  } else if ((kind) == hkv::kValueF16) {                        \
    if (whole) { CALL(__half, true); } else { CALL(__half, false); } \
  } else {                                                      \
    if (whole) { CALL(__nv_bfloat16, true); } else { CALL(__nv_bfloat16, false); } \
  }

int check_order(uint64_t tokens, uint32_t top_k, uint32_t experts) {
  HKV_ROWS_CHECK(top_k >= 1 && top_k <= kMaxTopK, "top_k must be between 1 and 64");
  HKV_ROWS_CHECK(experts >= 1 && experts <= kMaxExperts, "experts must be between 1 and 1024");
  HKV_ROWS_CHECK(tokens < (1ull << 31) && tokens * top_k < (1ull << 31),
                 "batches of 2^31 or more assignments");
  return HKV_OK;
}

// Blocks of `threads` threads for `items` threads' work.
int grid_of(uint64_t items, uint32_t threads, unsigned* grid) {
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
  const uint64_t bits =
      row_bytes | address_bits(x) | x_stride | address_bits(rows) | rows_stride;
  const bool whole = whole_chunks(bits);
  const uint32_t chunks = chunks_of(row_bytes, whole);
  unsigned grid = 0;
  rc = grid_of(tokens * chunks, kMoveBlock, &grid);
  if (rc != HKV_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const RowsIn in = rows_in(x, tokens, x_stride, row_bytes);
  const int32_t* kept = zero_rows_behind ? offsets + experts : nullptr;
#define HKV_CALL(G)                                                                              \
  dispatch_kernel<G><<<grid, kMoveBlock, 0, s>>>(tokens, top_k, per_row(chunks), uint32_t(row_bytes), in, position, \
                                                 static_cast<uint8_t*>(rows), rows_stride, kept)
  switch (whole ? 0u : piece_bytes(bits)) {
    case 0: HKV_CALL(0); break;
    case 8: HKV_CALL(8); break;
    case 4: HKV_CALL(4); break;
    case 2: HKV_CALL(2); break;
    default: HKV_CALL(1); break;
  }
#undef HKV_CALL
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
  const uint64_t row_bytes = dim * size;
  const uint64_t bits =
      row_bytes | address_bits(rows) | rows_stride | address_bits(out) | out_stride;
  HKV_ROWS_CHECK(bits % size == 0, "a row does not start at a multiple of its element size");
  const bool whole = whole_chunks(bits);
  const uint32_t chunks = chunks_of(row_bytes, whole);
  unsigned grid = 0;
  rc = grid_of(tokens * chunks, kMoveBlock, &grid);
  if (rc != HKV_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const RowsIn in = rows_in(rows, tokens * top_k, rows_stride, row_bytes);
#define HKV_CALL(T, WHOLE)                                                                \
  combine_kernel<T, WHOLE><<<grid, kMoveBlock, 0, s>>>(                                   \
      tokens, top_k, per_row(chunks), uint32_t(row_bytes), in, weights, weight_kind == kValueF32, position,  \
      static_cast<uint8_t*>(out), out_stride)
  HKV_FOR_TYPE(value_kind, whole, HKV_CALL)
#undef HKV_CALL
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
  const uint64_t row_bytes = dim * size;
  const uint64_t bits = row_bytes | address_bits(d_out) | d_out_stride | address_bits(rows) |
                        rows_stride | address_bits(d_rows) | d_rows_stride;
  HKV_ROWS_CHECK(bits % size == 0, "a row does not start at a multiple of its element size");
  const bool whole = whole_chunks(bits);
  const uint32_t chunks = chunks_of(row_bytes, whole);
  uint32_t group = pow2_at_least(chunks);
  group = group > 256u ? 256u : group;
  unsigned grid = 0;
  rc = grid_of(tokens * group, 256, &grid);
  if (rc != HKV_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const RowsIn d_in = rows_in(d_out, tokens, d_out_stride, row_bytes);
  const RowsIn in = rows_in(rows, tokens * top_k, rows_stride, row_bytes);
  const int32_t* kept = zero_rows_behind ? offsets + experts : nullptr;
#define HKV_CALL(T, WHOLE)                                                                       \
  combine_backward_kernel<T, WHOLE><<<grid, 256, 0, s>>>(                                        \
      tokens, top_k, chunks, group, uint32_t(row_bytes), d_in, in, weights, weight_kind == kValueF32,      \
      position, static_cast<uint8_t*>(d_rows), d_rows_stride, d_weights, kept)
  HKV_FOR_TYPE(value_kind, whole, HKV_CALL)
#undef HKV_CALL
  return rows_launched();
}

}  // extern "C"
