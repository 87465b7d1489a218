// Tiles of rows in LDS and the matrix operands that are read from them, 32 x 32 x 16 products.
#pragma once

#include "attn.hpp"

namespace fsp {

// Rows of one step, and how they lie in LDS: PITCH bytes each in chunks of 16, a row's chunks permuted
// by the row so that the lanes of one read meet different banks, in reads of one chunk of 8 (or
// 16) consecutive rows and in transposed reads of four chunks of four rows.
constexpr int kRows = 64;

template <int DP>
struct Lay {
  static constexpr int PITCH = DP <= 64 ? 128 : 256;
  static constexpr int CH = PITCH / 16;
  static constexpr int BYTES = kRows * PITCH;
  __device__ static int swizzle(int r) {
    const int r0 = r & 1, r1 = (r >> 1) & 1, r2 = (r >> 2) & 1, r3 = (r >> 3) & 1;
    return CH == 8 ? (r1 << 2 | r2 << 1 | (r0 ^ r3)) : (r1 << 3 | r0 << 2 | r2 << 1 | (r1 ^ r3));
  }
  // Where lane finds 8 elements of row lane % 32, from 8 * (lane / 32) on; 16 * i elements on and
  // 32 * u rows on: (this ^ 32 * i) + 32 * u * PITCH.
  __device__ static int row_at(int lane) {
    return (lane & 31) * PITCH + (((lane >> 5) ^ swizzle(lane & 31)) << 4);
  }
  // What lane names in a transposed read of the columns 0..31 of rows 4 * (lane / 32) + 0..3: it gets
  // column lane % 32.  32 * n columns on: this ^ 64 * n; 8 rows on: (this ^ 16) + 8 * PITCH;
  // 16 * i rows on: + 16 * i * PITCH.
  __device__ static int col_at(int lane) {
    const int j = lane & 15, row = 4 * (lane >> 5) + (j >> 2);
    const int chunk = (2 * ((lane >> 4) & 1) + ((j & 3) >> 1)) ^ swizzle(row);
    return row * PITCH + chunk * 16 + (j & 1) * 8;
  }
};

// The order of the LDS reads and matrix instructions before it: AHEAD reads, then a product and a read
// in turn, then the products that are left.  Left to itself the compiler reads an operand just
// before its product and waits out the LDS's latency each time.
template <int READS, int AHEAD>
__device__ __forceinline__ void read_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < READS - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// Matrix operands from LDS: 8 consecutive elements of a row a lane, and 8 rows' elements of a column
// (rows 16 * i + {0..3, 8..11} + 4 * (lane / 32), the ones that the lane's accumulator registers
// 8 * i..8 * i + 7 stand for).
template <typename T>
__device__ __forceinline__ V8<T> row_frag(const lds_char* p) {
  return __builtin_bit_cast(V8<T>, *(const lds_s16x8*)p);
}

template <typename T, int PITCH>
__device__ __forceinline__ V8<T> col_frag(const lds_char* base, int at, int i) {
  const s16x4 low = lds_transposed(base + at + 16 * i * PITCH);
  const s16x4 high = lds_transposed(base + (at ^ 16) + (16 * i + 8) * PITCH);
  return __builtin_bit_cast(V8<T>, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <typename T>
__device__ __forceinline__ V8<T> to16(const f32x16& x, int at) {
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x[at + e];
  return __builtin_convertvector(v, V8<T>);
}

// One row of a result from the accumulators of its column, times f.
template <typename T, int NT>
__device__ __forceinline__ void store_rows(T* to, const f32x16 (&x)[NT], float f, int dim, int half) {
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * i + 2 * r + 4 * half;
      if (d < dim) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = x[i][r + e] * f;
        if constexpr (std::is_same<T, float>::value)
          *reinterpret_cast<f32x4*>(to + d) = y;
        else
          *reinterpret_cast<V4<T>*>(to + d) = __builtin_convertvector(y, V4<T>);
      }
    }
}

// Bits of 32 keys, from bit x on.
__device__ __forceinline__ uint32_t bits_from(int x) { return x <= 0 ? ~0u : x > 31 ? 0u : ~0u << x; }

// x where bit K is set, else minus infinity or, with ZERO, 0; without a condition, which would hold a pair of
// scalar registers for each element.
template <int K, bool ZERO = false>
__device__ __forceinline__ float seen_or_none(uint32_t bits, float x) {
  const uint32_t m = (uint32_t)((int)(bits << (31 - K)) >> 31);
  return __uint_as_float((__float_as_uint(x) & m) | (ZERO ? 0u : 0xff800000u & ~m));
}

// The same for the 16 keys of 32 that an accumulator holds in this half of the lanes.
template <bool ZERO = false>
__device__ __forceinline__ void seen_or_none(uint32_t bits, int half, f32x16& x) {
  bits >>= 4 * half;
#pragma unroll
  for (int r = 0; r < 16; r += 4) {
    const uint32_t b = bits >> (2 * r);
    x[r] = seen_or_none<0, ZERO>(b, x[r]);
    x[r + 1] = seen_or_none<1, ZERO>(b, x[r + 1]);
    x[r + 2] = seen_or_none<2, ZERO>(b, x[r + 2]);
    x[r + 3] = seen_or_none<3, ZERO>(b, x[r + 3]);
  }
}

}  // namespace fsp
