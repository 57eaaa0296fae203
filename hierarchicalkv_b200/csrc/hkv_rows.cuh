// What the row operators share (hkv_expert.cu, hkv_norm.cu): element types,
// 16-byte chunks of rows at any alignment and the error text of their C entries.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/hkv_b200.h"
#include "hkv_device.cuh"

namespace hkv {

// Element types of the row operators (values of hkv_value_kind).
inline bool is_row_kind(uint32_t kind) {
  return kind == kValueF32 || kind == kValueF16 || kind == kValueBF16;
}
inline uint32_t row_kind_size(uint32_t kind) { return kind == kValueF32 ? 4u : 2u; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// The one rounding of a result, to nearest even.
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// ---- 16-byte chunks of rows ---------------------------------------------------
//
// Every kernel moves rows in accesses of 16 bytes, whatever their alignment:
// rows of odd lengths start at multiples of their element only, and accesses of
// one 2-byte element ran at an eighth of the rate of 16 bytes (layer norm of
// 65537 x 333 half: 100 us with them, 27 us with chunks).  A chunk at an
// unaligned address is cut out of the two aligned ones it touches.

template <typename T>
struct Chunk {
  static constexpr int kElems = 16 / int(sizeof(T));
  union {
    uint4 raw;
    T elem[kElems];
  };
  __device__ __forceinline__ Chunk() {}
  __device__ __forceinline__ float get(int i) const { return to_float(elem[i]); }
  __device__ __forceinline__ void set(int i, float v) { elem[i] = from_float<T>(v); }
};

// A matrix of rows: base, distance and count of the rows in bytes; every row
// that is read lies in [first, last).
struct RowsIn {
  const uint8_t* first;
  const uint8_t* last;
  uint64_t stride;
};
inline RowsIn rows_in(const void* base, uint64_t n, uint64_t stride, uint64_t row_bytes) {
  const uint8_t* p = static_cast<const uint8_t*>(base);
  return RowsIn{p, p + (n - 1) * stride + row_bytes, stride};
}

// Bytes s ... s + 15 of the 32 bytes lo, hi.
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, uint32_t s) {
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  const bool by8 = (s & 8u) != 0, by4 = (s & 4u) != 0;
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = by8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = by4 ? w[i + 1] : w[i];
  const uint32_t bits = (s & 3u) * 8u;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// An element of G bytes of a chunk, for the ends of rows.
template <int G>
__device__ __forceinline__ void put_piece(uint4& v, int at, const uint8_t* from) {
  *reinterpret_cast<typename VecType<G>::type*>(reinterpret_cast<uint8_t*>(&v) + at) =
      *reinterpret_cast<const typename VecType<G>::type*>(from);
}

// The 16 bytes at p, of which those inside [from, to) matter (the others are
// anything).  Aligned chunks are read whole where they lie inside the matrix,
// element by element (of G bytes) at its ends: nothing outside it is touched.
template <int G>
__device__ __forceinline__ uint4 load_chunk(const uint8_t* p, const uint8_t* from,
                                            const uint8_t* to, const uint8_t* first,
                                            const uint8_t* last) {
  const uint32_t s = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
  const uint8_t* a = p - s;
  const bool need_lo = from < a + 16;
  const bool need_hi = s != 0 && to > a + 16;
  if ((need_lo && (a < first || a + 16 > last)) || (need_hi && (a + 16 < first || a + 32 > last))) {
    uint4 v = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int b = 0; b < 16; b += G) {
      if (p + b >= from && p + b < to) put_piece<G>(v, b, p + b);
    }
    return v;
  }
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (need_lo) lo = __ldg(reinterpret_cast<const uint4*>(a));
  if (need_hi) hi = __ldg(reinterpret_cast<const uint4*>(a + 16));
  return s == 0 ? lo : shifted(lo, hi, s);
}

// Stores the bytes of v (for the aligned address q) that lie inside [from, to).
template <int G>
__device__ __forceinline__ void store_chunk(uint8_t* q, const uint4& v, const uint8_t* from,
                                            const uint8_t* to) {
  if (q >= from && q + 16 <= to) {
    *reinterpret_cast<uint4*>(q) = v;
    return;
  }
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(&v);
#pragma unroll
  for (int b = 0; b < 16; b += G) {
    if (q + b >= from && q + b < to) {
      *reinterpret_cast<typename VecType<G>::type*>(q + b) =
          *reinterpret_cast<const typename VecType<G>::type*>(bytes + b);
    }
  }
}

// Or of addresses, strides and lengths in bytes: 16 divides all of them?
inline bool whole_chunks(uint64_t bits) { return (bits & 15u) == 0; }
inline uint64_t address_bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }
// The largest power of two up to 8 that divides `bits`.
inline uint32_t piece_bytes(uint64_t bits) {
  uint32_t v = 8;
  while (v > 1 && (bits & (v - 1)) != 0) v >>= 1;
  return v;
}

int rows_fail(int code, const char* message) noexcept;
int rows_launched() noexcept;   // HKV_OK, or the launch's error
int sm_count() noexcept;        // of the current device

#define HKV_ROWS_CHECK(cond, message) \
  do {                                \
    if (!(cond)) return hkv::rows_fail(HKV_ERR_INVALID_ARG, (message)); \
  } while (0)

}  // namespace hkv
