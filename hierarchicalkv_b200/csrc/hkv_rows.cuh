// What the row operators share (hkv_expert.cu, hkv_norm.cu, hkv_norm_backward.cu):
// element types, the units rows are moved in, asynchronous copies and the error
// text of their C entries.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <string>
#include <type_traits>

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
__device__ __forceinline__ float low_to_float(uint32_t v, const __half*) {
  return __half2float(__ushort_as_half(static_cast<uint16_t>(v)));
}
__device__ __forceinline__ float low_to_float(uint32_t v, const __nv_bfloat16*) {
  return __uint_as_float(v << 16);   // a bfloat16 is the upper half of its float
}

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

// ---- units -------------------------------------------------------------------
//
// Rows are moved in units: 16 bytes where every row starts at a multiple of 16
// and is a multiple of 16 long, else 4 bytes or one element, neighbouring units
// in neighbouring lanes.  Narrow units cost instructions, not bandwidth, as long
// as a thread's work per unit is the load, the arithmetic and the store and
// nothing else.  (Cutting 16-byte chunks out of the aligned ones around them
// instead, with their masks and shifts, took 1043 instructions per row of 1001
// bfloat16 in layer norm, where the units take 617.)

// A 32-bit word's elements as floats, and back.
__device__ __forceinline__ void unpack_word(uint32_t w, float* f, const float*) {
  f[0] = __uint_as_float(w);
}
__device__ __forceinline__ void unpack_word(uint32_t w, float* f, const __half*) {
  const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&w));
  f[0] = two.x;
  f[1] = two.y;
}
__device__ __forceinline__ void unpack_word(uint32_t w, float* f, const __nv_bfloat16*) {
  f[0] = __uint_as_float(w << 16);
  f[1] = __uint_as_float(w & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t pack_word(const float* f, const float*) {
  return __float_as_uint(f[0]);
}
__device__ __forceinline__ uint32_t pack_word(const float* f, const __half*) {
  const __half2 two = __floats2half2_rn(f[0], f[1]);
  return *reinterpret_cast<const uint32_t*>(&two);
}
__device__ __forceinline__ uint32_t pack_word(const float* f, const __nv_bfloat16*) {
  const __nv_bfloat162 two = __floats2bfloat162_rn(f[0], f[1]);
  return *reinterpret_cast<const uint32_t*>(&two);
}

template <typename T, int BYTES>
struct Unit {
  static constexpr int kElems = BYTES / int(sizeof(T));
  using Raw = typename VecType<BYTES>::type;
  using Loaded = std::conditional_t<BYTES == 2, uint32_t, Raw>;   // 16 bits, in a register's lower half

  static __device__ __forceinline__ void unpack(const Loaded& v, float (&f)[kElems]) {
    if constexpr (BYTES == 16) {
      constexpr int kPer = 4 / int(sizeof(T));
      unpack_word(v.x, f, static_cast<const T*>(nullptr));
      unpack_word(v.y, f + kPer, static_cast<const T*>(nullptr));
      unpack_word(v.z, f + 2 * kPer, static_cast<const T*>(nullptr));
      unpack_word(v.w, f + 3 * kPer, static_cast<const T*>(nullptr));
    } else if constexpr (BYTES == 4) {
      unpack_word(v, f, static_cast<const T*>(nullptr));
    } else {
      f[0] = low_to_float(v, static_cast<const T*>(nullptr));
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[kElems]) {
    if constexpr (BYTES == 16) {
      constexpr int kPer = 4 / int(sizeof(T));
      return make_uint4(pack_word(f, static_cast<const T*>(nullptr)),
                        pack_word(f + kPer, static_cast<const T*>(nullptr)),
                        pack_word(f + 2 * kPer, static_cast<const T*>(nullptr)),
                        pack_word(f + 3 * kPer, static_cast<const T*>(nullptr)));
    } else if constexpr (BYTES == 4) {
      return pack_word(f, static_cast<const T*>(nullptr));
    } else {
      const T one = from_float<T>(f[0]);
      return *reinterpret_cast<const Raw*>(&one);
    }
  }
};

template <typename Raw>
__device__ __forceinline__ Raw no_unit() {
  return Raw{};
}

inline uint64_t address_bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Whether every address is a multiple of `bytes` (null is).
template <typename... P>
inline bool all_aligned(uint32_t bytes, const P*... p) {
  return ((address_bits(p) | ...) & (bytes - 1u)) == 0;
}

// Unit for rows whose addresses, strides and lengths in bytes have these bits (or
// of all of them) set: 16, 4 or one element; 0 where an element would be split.
inline uint32_t unit_bytes(uint64_t bits, uint32_t element) {
  if (bits % 16 == 0) return 16;
  if (bits % 4 == 0) return 4;
  return bits % element == 0 ? element : 0;
}

// CALL(type, unit) for the unit and kind of a launch.
#define HKV_FOR_UNIT(kind, unit, CALL)                      \
  if ((kind) == hkv::kValueF32) {                           \
    if ((unit) == 16) { CALL(float, 16); }                  \
    else { CALL(float, 4); }                                \
  } else if ((kind) == hkv::kValueF16) {                    \
    if ((unit) == 16) { CALL(__half, 16); }                 \
    else if ((unit) == 4) { CALL(__half, 4); }              \
    else { CALL(__half, 2); }                               \
  } else {                                                  \
    if ((unit) == 16) { CALL(__nv_bfloat16, 16); }          \
    else if ((unit) == 4) { CALL(__nv_bfloat16, 4); }       \
    else { CALL(__nv_bfloat16, 2); }                        \
  }

// A matrix of rows that is read.
struct RowsIn {
  const uint8_t* first;
  uint64_t stride;
};
inline RowsIn rows_in(const void* base, uint64_t stride) {
  return RowsIn{static_cast<const uint8_t*>(base), stride};
}

int rows_fail(int code, const char* message) noexcept;

__device__ __forceinline__ void copy_async(uint32_t shared, const uint8_t* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
}
// Its first `bytes` bytes (1 ... 16), and zeros: nothing behind them is read.
__device__ __forceinline__ void copy_async(uint32_t shared, const uint8_t* global, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared), "l"(global), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int BYTES>
__device__ __forceinline__ auto load_shared(uint32_t at) {
  std::conditional_t<BYTES == 16, uint4, uint32_t> v;
  if constexpr (BYTES == 16) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(at)
                 : "memory");
  } else if constexpr (BYTES == 4) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  } else {
    asm volatile("ld.shared.u16 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  }
  return v;
}

// Allows a kernel the shared memory of any of its queues, once per device: the
// call takes as long as a launch.
constexpr size_t kMostShared = 220 * 1024;
template <auto KERNEL>
int allow_shared() noexcept {
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  if (allowed.load(std::memory_order_relaxed) & bit) return HKV_OK;
  const cudaError_t e =
      cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kMostShared));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return rows_fail(HKV_ERR_CUDA, cudaGetErrorString(e));
  }
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return HKV_OK;
}

int rows_launched() noexcept;   // HKV_OK, or the launch's error
int sm_count() noexcept;        // of the current device

#define HKV_ROWS_CHECK(cond, message) \
  do {                                \
    if (!(cond)) return hkv::rows_fail(HKV_ERR_INVALID_ARG, (message)); \
  } while (0)

}  // namespace hkv
