// What the attention kernels share: the 16-bit types, wave reductions, argument checks.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fsp_device.hpp"
#include "fsp_internal.hpp"

namespace fsp {

constexpr int64_t kAttnDimCap = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef __bf16 bf16;
typedef _Float16 f16;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

inline bool aligned16(const void* p, int64_t a, int64_t b) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a % 8 == 0 && b % 8 == 0;
}

inline bool attn_dtype(int64_t d) { return d == FSP_BF16 || d == FSP_F16; }

inline bool attn_dim(int64_t d) { return d >= 8 && d % 8 == 0 && d <= kAttnDimCap; }

}  // namespace fsp
