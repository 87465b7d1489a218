// What the attention kernels share: the 16-bit types, matrix products, argument checks.
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
// Tokens of a batch or of a page table: a place that lies past the last one by less than a step (up to
// 1024 tokens) is still an int.
constexpr int64_t kAttnTokensCap = 0x80000000LL - 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef __bf16 bf16;
typedef _Float16 f16;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Vec;
template <> struct Vec<bf16> { typedef bf16x8 v8; typedef bf16x4 v4; };
template <> struct Vec<f16> { typedef f16x8 v8; typedef f16x4 v4; };
template <typename T> using V8 = typename Vec<T>::v8;
template <typename T> using V4 = typename Vec<T>::v4;

// C += A B on the matrix cores, 32 x 32 x 16.  Lane l holds A[l % 32][8 * (l / 32) + 0..7],
// B[8 * (l / 32) + 0..7][l % 32] and, in register r, C[8 * (r / 4) + 4 * (l / 32) + r % 4][l % 32].
// The order of the 16 summed elements is free as long as A and B share it.
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// 16 x 16 x 32: A[l % 16][8 * (l / 16) + 0..7], B[8 * (l / 16) + 0..7][l % 16],
// C[4 * (l / 16) + r][l % 16].
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) s16x8 lds_s16x8;

// A transposed read of 16-bit elements from LDS: in each group of 16 lanes, lane j names four
// consecutive elements of row j / 4, columns 4 * (j % 4) + 0..3, and gets column j of the four rows.
__device__ __forceinline__ s16x4 lds_transposed(const lds_char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
}

// The other half's value: lanes l and l + 32 exchange.
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// Scores are scale * q . k, and weights exp(score - max) = exp2(c q . k - c max) with c = scale *
// log2(e) > 0: a negative scale turns the sign of one factor, and one that is zero, or too small to
// show in 32 bits, makes it zero.
constexpr float kNoScale = 1e-30f;

// A forward pass's weights follow a maximum of their row that is moved only when the row's grows by more
// than 2^lag of it, and are taken times 2^up before they are rounded to the inputs' type: float16 holds
// those below 2^-14 with fewer bits, so a row's weights down to 2^-25 of its largest have them all.
// With lag 8 and up 0 the output beside a key of value zero that outweighs the others by 16 e-folds was
// off by 24 times what one rounding gives.
template <typename T> struct Weights { static constexpr float lag = 8, up = 0, down = 1; };
template <> struct Weights<f16> { static constexpr float lag = 4, up = 11, down = 1.0f / 2048; };

// Eight elements, or zeros.  A mask, not a choice: a choice becomes a branch around the load, and loads
// in branches wait for each other.
template <typename T>
__device__ __forceinline__ V8<T> keep_if(V8<T> x, bool in) {
  const int m = in ? -1 : 0;
  return __builtin_bit_cast(V8<T>, __builtin_bit_cast(i32x4, x) & i32x4{m, m, m, m});
}

template <typename T>
__device__ __forceinline__ V8<T> scaled_sign(V8<T> q, float scale, bool in) {
  const int m = scale < 0 ? (int)0x80008000 : 0;
  const i32x4 x = __builtin_bit_cast(i32x4, keep_if<T>(q, in && fabsf(scale) > kNoScale));
  return __builtin_bit_cast(V8<T>, x ^ i32x4{m, m, m, m});
}

__device__ __forceinline__ float exp2_scale(float scale) {
  return fabsf(scale) > kNoScale ? fabsf(scale) * kLog2e : 1.0f;
}

inline bool aligned16(const void* p, int64_t a, int64_t b) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a % 8 == 0 && b % 8 == 0;
}

inline bool attn_dtype(int64_t d) { return d == FSP_BF16 || d == FSP_F16; }

inline bool attn_dim(int64_t d) { return d >= 8 && d % 8 == 0 && d <= kAttnDimCap; }

}  // namespace fsp
