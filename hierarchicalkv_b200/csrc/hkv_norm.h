// Layer norm launcher shared with the C-ABI layer (find with layer norm).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace hkv {

// Strides are in bytes.
struct NormArgs {
  uint64_t n = 0;
  uint64_t dim = 0;
  const void* x = nullptr;                 // rows by base and stride ...
  uint64_t x_stride = 0;
  const void* const* row_ptrs = nullptr;   // ... or one address each; null: leave the output row
  uint32_t row_mask = 0;                   // as for null where an address has one of these bits
  const void* weight = nullptr;            // null: ones
  const void* bias = nullptr;              // null: zeros
  bool params_f32 = false;                 // weight and bias are float, else the rows' type
  bool params_vec = false;                 // both start at a multiple of 16 bytes
  float eps = 0.f;
  float inv_dim = 1.f;
  void* y = nullptr;
  uint64_t y_stride = 0;
  float* mean = nullptr;                   // null: not kept
  float* rstd = nullptr;
};

struct NormBackwardArgs {
  uint64_t n = 0;
  uint64_t dim = 0;
  const void* dy = nullptr;
  uint64_t dy_stride = 0;
  const void* x = nullptr;
  uint64_t x_stride = 0;
  const void* weight = nullptr;
  bool params_f32 = false;
  bool params_vec = false;
  float inv_dim = 1.f;
  const float* mean = nullptr;
  const float* rstd = nullptr;
  void* dx = nullptr;
  uint64_t dx_stride = 0;
  void* d_weight = nullptr;                // null: not wanted
  void* d_bias = nullptr;
};

// HKV_OK or the error; value_kind is one of the row kinds.
int launch_norm(NormArgs args, uint32_t value_kind, cudaStream_t stream);

}  // namespace hkv
