// What the row operators share (hkv_expert.cu, hkv_norm.cu): element types,
// packs of elements moved with one access, the choice of the access width and
// the error text of their C entries.
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

// VB bytes of elements that one access moves.
template <typename T, int VB>
struct Pack {
  static constexpr int kElems = VB / int(sizeof(T));
  using Raw = typename VecType<VB>::type;
  union {
    Raw raw;
    T elem[kElems];
  };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ float get(int i) const { return to_float(elem[i]); }
  __device__ __forceinline__ void set(int i, float v) { elem[i] = from_float<T>(v); }
};

// Parameters (weights, biases) may have the rows' type or float: a pack's
// worth of them as floats.  The branch is uniform over the launch.
template <typename T, int N>
__device__ __forceinline__ void load_params(const void* p, bool f32, uint32_t at, float (&out)[N]) {
  if (f32) {
    const float* s = static_cast<const float*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = __ldg(s + i);
  } else {
    const T* s = static_cast<const T*>(p) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = to_float(s[i]);
  }
}

// Widest access of 16, 8, 4, 2 or 1 bytes that every address in `bits` (the
// or of base addresses, strides and row lengths in bytes) is a multiple of.
inline uint32_t access_bytes(uint64_t bits) {
  uint32_t v = 16;
  while (v > 1 && (bits & (v - 1)) != 0) v >>= 1;
  return v;
}
inline uint64_t address_bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

int rows_fail(int code, const char* message) noexcept;
int rows_launched() noexcept;   // HKV_OK, or the launch's error
int sm_count() noexcept;        // of the current device

#define HKV_ROWS_CHECK(cond, message) \
  do {                                \
    if (!(cond)) return hkv::rows_fail(HKV_ERR_INVALID_ARG, (message)); \
  } while (0)

}  // namespace hkv
