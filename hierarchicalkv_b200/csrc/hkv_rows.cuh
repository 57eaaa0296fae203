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
constexpr int kChunkElems = 16 / int(sizeof(T));

// A chunk's elements as floats, and back with one rounding each.
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[4], const float*) {
  f[0] = __uint_as_float(v.x);
  f[1] = __uint_as_float(v.y);
  f[2] = __uint_as_float(v.z);
  f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8], const __half*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = two.x;
    f[2 * i + 1] = two.y;
  }
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8], const __nv_bfloat16*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {   // a bfloat16 is the upper half of its float
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[kChunkElems<T>]) {
  unpack(v, f, static_cast<const T*>(nullptr));
}
__device__ __forceinline__ uint4 pack(const float (&f)[4], const float*) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                    __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], const __half*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 two = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&two);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], const __nv_bfloat16*) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 two = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&two);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&f)[kChunkElems<T>]) {
  return pack(f, static_cast<const T*>(nullptr));
}

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

// The 16 bytes at p, those inside [from, to) element by element (of G bytes) and
// zeros for the others.
template <int G>
__device__ __forceinline__ uint4 pieces(const uint8_t* p, const uint8_t* from, const uint8_t* to) {
  uint64_t half[2] = {0, 0};
#pragma unroll 1
  for (int b = 0; b < 16; b += G) {
    if (p + b < from || p + b >= to) continue;
    uint64_t piece;
    if constexpr (G == 8) piece = *reinterpret_cast<const uint64_t*>(p + b);
    else piece = *reinterpret_cast<const typename VecType<G>::type*>(p + b);
    half[0] |= b < 8 ? piece << (8 * b) : 0;
    half[1] |= b < 8 ? 0 : piece << (8 * (b - 8));
  }
  return make_uint4(uint32_t(half[0]), uint32_t(half[0] >> 32), uint32_t(half[1]),
                    uint32_t(half[1] >> 32));
}

// The 16 bytes at an address p of any alignment, of which those inside a row
// [from, to) matter (the others are anything).  The aligned chunks that hold them
// are read whole where they lie inside the matrix [first, last), and element by
// element (of G bytes) at its ends: nothing outside it is touched.  Loading and
// cutting are two steps, without a branch in the first, so that the loads of
// several chunks are in flight together.
struct Cut {
  uint4 lo, hi;
  uint32_t s;
  bool inside;

  __device__ __forceinline__ void load(const uint8_t* p, const uint8_t* first, const uint8_t* last) {
    s = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
    const uint8_t* a = p - s;
    inside = a >= first && a + (s ? 32 : 16) <= last;
    lo = hi = make_uint4(0, 0, 0, 0);
    if (inside) lo = __ldg(reinterpret_cast<const uint4*>(a));
    if (inside && s) hi = __ldg(reinterpret_cast<const uint4*>(a + 16));
  }
  __device__ __forceinline__ void none() {
    lo = hi = make_uint4(0, 0, 0, 0);
    s = 0;
    inside = true;
  }
  template <int G>
  __device__ __forceinline__ uint4 get(const uint8_t* p, const uint8_t* from, const uint8_t* to) const {
    if (inside) return s == 0 ? lo : shifted(lo, hi, s);
    return pieces<G>(p, from, to);
  }
};

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i < 2 ? (i == 0 ? v.x : v.y) : (i == 2 ? v.z : v.w);
}

// Stores those bytes of the aligned 16 at row + off (v's) that lie in
// [from, to) of the row, all three in bytes from its start.  A row's first and
// last bytes go out in at most one piece of 8, 4, 2 and 1 bytes each, down to the
// element size G; only rows that begin and end in the same 16 bytes are stored
// element by element.
template <int G>
__device__ __forceinline__ void store_chunk(uint8_t* row, int off, const uint4& v, int from, int to) {
  const int lo = from > off ? from - off : 0, hi = to - off < 16 ? to - off : 16;
  uint8_t* q = row + off;
  if (lo == 0 && hi == 16) {
    *reinterpret_cast<uint4*>(q) = v;
  } else if (hi <= lo) {
    return;
  } else if (hi == 16) {   // the row's head: pieces that end at the boundary
    const int h = 16 - lo;
    if (h & 8) *reinterpret_cast<uint2*>(q + 8) = make_uint2(v.z, v.w);
    if (G <= 4 && (h & 4)) *reinterpret_cast<uint32_t*>(q + 12 - (h & 8)) = h & 8 ? v.y : v.w;
    if (G <= 2 && (h & 2)) {
      const int at = 14 - (h & 12);
      *reinterpret_cast<uint16_t*>(q + at) = static_cast<uint16_t>(word_of(v, at >> 2) >> 16);
    }
    if (G <= 1 && (h & 1)) {
      const int at = 15 - (h & 14);
      q[at] = static_cast<uint8_t>(word_of(v, at >> 2) >> (8 * (at & 3)));
    }
  } else if (lo == 0) {    // its tail: pieces that start at the boundary
    if (hi & 8) *reinterpret_cast<uint2*>(q) = make_uint2(v.x, v.y);
    if (G <= 4 && (hi & 4)) *reinterpret_cast<uint32_t*>(q + (hi & 8)) = hi & 8 ? v.z : v.x;
    if (G <= 2 && (hi & 2)) {
      const int at = hi & 12;
      *reinterpret_cast<uint16_t*>(q + at) = static_cast<uint16_t>(word_of(v, at >> 2));
    }
    if (G <= 1 && (hi & 1)) {
      const int at = hi & 14;
      q[at] = static_cast<uint8_t>(word_of(v, at >> 2) >> (8 * (at & 3)));
    }
  } else {
#pragma unroll 1
    for (int b = lo; b < hi; ++b) q[b] = static_cast<uint8_t>(word_of(v, b >> 2) >> (8 * (b & 3)));
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

__device__ __forceinline__ void copy_async(uint32_t shared, const uint8_t* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

int rows_fail(int code, const char* message) noexcept;
int rows_launched() noexcept;   // HKV_OK, or the launch's error
int sm_count() noexcept;        // of the current device

#define HKV_ROWS_CHECK(cond, message) \
  do {                                \
    if (!(cond)) return hkv::rows_fail(HKV_ERR_INVALID_ARG, (message)); \
  } while (0)

}  // namespace hkv
