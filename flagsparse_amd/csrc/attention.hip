// Attention over packed sequences, forward and backward.
#include "attn.hpp"

namespace fsp {
namespace {

constexpr int kTile = 128;  // query rows of a workgroup, 32 a wave

constexpr int64_t kTokenStep = 1 << 23;  // the bytes of a load's 128 rows are a 32-bit offset

struct Tile {
  int first, rows, at, q_begin, nq, k_begin, nk, pad;
};

struct Shape {
  int heads, kv_heads, dim, causal, window;
  float scale;
};

// Workgroups go to the 8 XCDs in turn.  Where the heads divide by them, each XCD has heads of its own, so
// that the tiles it works on at a time read the same keys through its L2; within an XCD (and
// otherwise over all of them) the tiles run in the list's order, heavy ones first.
__device__ __forceinline__ void tile_and_head(int block, int n_tiles, int heads, int& tile, int& head) {
  if (heads % 8 == 0) {
    const int per = heads / 8, j = block >> 3;
    tile = j / per;
    head = (block & 7) * per + j % per;
  } else {
    tile = block / heads;
    head = block % heads;
  }
}

// Query i of a sequence sees the keys [lo, hi).
__device__ __forceinline__ void seen_by(const Shape& s, const Tile& t, int i, int& lo, int& hi) {
  lo = 0;
  hi = t.nk;
  if (s.causal) {
    hi = i + t.nk - t.nq + 1;
    if (s.window && hi > s.window) lo = hi - s.window;
    if (hi < 0) hi = 0;
  }
}

// Key j of a sequence is seen by the queries [lo, hi).
__device__ __forceinline__ void seen_of(const Shape& s, const Tile& t, int j, int& lo, int& hi) {
  lo = 0;
  hi = t.nq;
  if (s.causal) {
    lo = j - t.nk + t.nq;
    if (s.window && lo < t.nq - s.window) hi = lo + s.window;
    if (lo < 0) lo = 0;
  }
}

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

// Rows [0, n) of a 16-bit array, ``bytes`` apart, straight to LDS: ROWS of them by WAVES waves, 1024
// bytes a wave and load.  What lies past the rows or the head's dim is read as zero: the buffer's
// bounds end there.
template <int DP, int ROWS, int WAVES>
__device__ __forceinline__ void load_rows(char* lds, const void* src, int n, uint32_t bytes, int dim,
                                          int wave, int lane) {
  typedef Lay<DP> L;
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<void*>(src), 0, (int)((uint32_t)(n - 1) * bytes + 2 * dim), 0x00027000);
  constexpr int PER = ROWS * L::PITCH / 1024 / WAVES;  // loads of a wave
  constexpr int EACH = 1024 / L::PITCH;                // rows of a load
  // swizzle(a ^ b) = swizzle(a) ^ swizzle(b): the wave's, the lane's and the load's rows share no bit
  const int chunk = (lane % L::CH) ^ L::swizzle(lane / L::CH) ^ L::swizzle(wave * PER * EACH);
  const uint32_t first = (uint32_t)(wave * PER * EACH + lane / L::CH) * bytes;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = 16 * (chunk ^ L::swizzle(i * EACH));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rsrc, (__attribute__((address_space(3))) void*)(lds + (wave * PER + i) * 1024), 16,
        (int)(at < 2 * dim ? first + i * EACH * bytes + at : 0x80000000u), 0, 0, 0);
  }
}

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

// out = sum_j w_j v_j / sum_j w_j with w_j = exp2(c q . k_j - m), m a maximum of the row that follows it
// (Weights).  With S^T = K Q^T a query is a lane: its maximum and sum are its own (and
// the other half's, 32 lanes on), and its weights are the operand of O^T = V^T P^T where they lie, in
// registers.  Keys and values go straight to LDS, the next step's while this one is worked on; weights
// are rounded to the inputs' type for the second product, as its operands have to be, and all sums
// are held in 32 bits, that of the weights from the unrounded ones.
//
// A tile of BLOCKS * 32 queries.  A wave goes to 32 of them and, of every PARTS * 64 keys, to 64: with
// PARTS = 2 two waves share the queries, and their sums are joined at the end: half the chain of
// steps (share_queries, halve_tiles).
//
// 16384 tokens, 16 heads of 128 over 2, causal: 1.1e12 operations in 990 to 1030 us, 1.07 to 1.11 PFLOP/s,
// where a library's 8192^3 product reaches 1.21.  Products take 62 % of the SIMDs' cycles, vector
// instructions 46 %, both at a time 23 %: the two mostly follow each other, at the clock that their power
// leaves (1.75 GHz); neither LDS (no bank conflicts) nor memory (0.36 GB) holds it up.  Two heads a workgroup
// over the same keys, or four buffers in turn, were no faster (284 / 289, 279 / 282 us).  16 ragged prompts
// of up to 2047, 32 heads over 8: 82 us, 0.69 PFLOP/s: short loops between the first loads and the last
// stores, 38 % of the cycles with neither.
template <typename T, int DP, int BLOCKS, int PARTS>
__global__ __launch_bounds__(64 * BLOCKS * PARTS, 2) void attention_packed_kernel(
    Shape s, const Tile* __restrict__ tiles, int n_tiles, const T* __restrict__ q, int64_t q_token,
    int64_t q_head, const T* __restrict__ k, int64_t k_token, int64_t k_head,
    const T* __restrict__ v, int64_t v_token, int64_t v_head, T* __restrict__ out,
    int64_t o_token, int64_t o_head, float* __restrict__ lse) {
  typedef Lay<DP> L;
  constexpr int NS = DP / 16, NT = DP / 32;
  constexpr int BYTES = PARTS * L::BYTES, ROWS = PARTS * kRows;
  __shared__ __attribute__((aligned(1024))) char s_k0[BYTES], s_v0[BYTES], s_k1[BYTES], s_v1[BYTES];
  int tile, a;
  tile_and_head(blockIdx.x, n_tiles, s.heads, tile, a);
  const Tile t = tiles[tile];
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = a / (s.heads / s.kv_heads);
  const int part = wave / BLOCKS, block = wave % BLOCKS, q0 = block * 32;
  const int mine = q0 + col;  // this lane's row of the tile
  const bool active = q0 < t.rows;

  V8<T> qf[NS];
  {
    const T* qr = q + (t.first + (int64_t)min(mine, t.rows - 1)) * q_token + a * q_head;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int d = 16 * i + 8 * half;
      const V8<T> x = *reinterpret_cast<const V8<T>*>(qr + (d < s.dim ? d : 0));
      qf[i] = scaled_sign<T>(x, s.scale, d < s.dim);
    }
  }
  const float c = exp2_scale(s.scale);

  // the keys that this lane's row sees, and those of the wave's first and last rows
  int lo, hi, lo0, hi0, lo1, hi1, lot, hit, none;
  seen_by(s, t, t.at + min(mine, t.rows - 1), lo, hi);
  seen_by(s, t, t.at + min(q0, t.rows - 1), lo0, hi0);
  seen_by(s, t, t.at + min(q0 + 31, t.rows - 1), lo1, hi1);
  seen_by(s, t, t.at, lot, none);
  seen_by(s, t, t.at + t.rows - 1, none, hit);

  f32x16 o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = f32x16{};
  float top = -INFINITY, sum = 0;

  const T* kb = k + (int64_t)t.k_begin * k_token + g * k_head;
  const T* vb = v + (int64_t)t.k_begin * v_token + g * v_head;
  auto load = [&](int j0, char* sk, char* sv) {
    const int n = min(ROWS, t.nk - j0);
    load_rows<DP, ROWS, BLOCKS * PARTS>(sk, kb + j0 * k_token, n, (uint32_t)(2 * k_token), s.dim,
                                        wave, lane);
    load_rows<DP, ROWS, BLOCKS * PARTS>(sv, vb + j0 * v_token, n, (uint32_t)(2 * v_token), s.dim,
                                        wave, lane);
  };
  const int k_at = L::row_at(lane);
  const int v_at = L::col_at(lane);

  auto step = [&](int j0, const char* sk_, const char* sv_) {
    j0 += part * kRows;
    if (!active || j0 >= hi1 || j0 + kRows <= lo0) return;
    const lds_char* sk = (const lds_char*)sk_ + part * L::BYTES;
    const lds_char* sv = (const lds_char*)sv_ + part * L::BYTES;
    f32x16 x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      x[u] = f32x16{};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        x[u] = mfma32(row_frag<T>(sk + (k_at ^ (i * 32)) + u * 32 * L::PITCH), qf[i], x[u]);
      }
    }
    read_ahead<2 * NS, NS>();
    if (j0 + kRows > hi0 || j0 < lo1) {
      const int first = lo - j0 - 4 * half, last = hi - j0 - 4 * half;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = 32 * u + 8 * (r / 4) + r % 4;
          x[u][r] = j >= first && j < last ? x[u][r] : -INFINITY;
        }
    }
    float m = x[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, x[u][r]);
    m = fmaxf(m, other_half(m));
    if (__any((m - top) * c > Weights<T>::lag)) {
      const float now = fmaxf(top, m);
      const float fade = top == -INFINITY ? 0.0f : exp2f((top - now) * c);
      top = now;
      sum *= fade;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] *= fade;
    }
    const float base = top == -INFINITY ? 0.0f : top * c - Weights<T>::up;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[u][r] = __builtin_amdgcn_exp2f(fmaf(x[u][r], c, -base));
        sum += x[u][r];
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // 16 keys: the ones that this lane holds the weights of
      const V8<T> pf = to16<T>(x[i / 2], 8 * (i % 2));
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        o[n] = mfma32(col_frag<T, L::PITCH>(sv, v_at ^ (64 * n), i), pf, o[n]);
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4 * NT, 1);  // the first values early
  };

  int j0 = lot;
  if (j0 < hit) load(j0, s_k0, s_v0);
  __syncthreads();
  while (j0 < hit) {
    if (j0 + ROWS < hit) load(j0 + ROWS, s_k1, s_v1);
    step(j0, s_k0, s_v0);
    __syncthreads();
    j0 += ROWS;
    if (j0 >= hit) break;
    if (j0 + ROWS < hit) load(j0 + ROWS, s_k0, s_v0);
    step(j0, s_k1, s_v1);
    __syncthreads();
    j0 += ROWS;
  }

  sum += other_half(sum);
  if constexpr (PARTS > 1) {
    float* theirs = reinterpret_cast<float*>(block == 0   ? s_k0
                                             : block == 1 ? s_v0
                                             : block == 2 ? s_k1
                                                          : s_v1);
    __shared__ f32x2 s_stat[BLOCKS][64];
    static_assert(NT * 16 * 64 * 4 <= BYTES, "");
    if (part == 1) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) theirs[(16 * i + r) * 64 + lane] = o[i][r];
      s_stat[block][lane] = f32x2{top, sum};
    }
    __syncthreads();
    if (part == 1) return;
    const f32x2 other = s_stat[block][lane];
    const float now = fmaxf(top, other.x), base = now == -INFINITY ? 0.0f : now;
    const float f0 = exp2f((top - base) * c), f1 = exp2f((other.x - base) * c);
    top = now;
    sum = sum * f0 + other.y * f1;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] = o[i][r] * f0 + theirs[(16 * i + r) * 64 + lane] * f1;
  }
  if (mine >= t.rows) return;
  const int64_t row = t.first + mine;
  const float inv = sum > 0 ? 1.0f / sum : (sum == 0 ? 0.0f : sum);
  if (half == 0)
    lse[row * s.heads + a] =
        sum == 0 ? -INFINITY : (top * c + log2f(sum * Weights<T>::down)) * kLn2;
  if (sum == 0)  // nothing seen: zeros, whatever lies in the rows of V
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] = f32x16{};
  store_rows<T, NT>(out + row * o_token + a * o_head, o, inv, s.dim, half);
}

// The normalised weights of the keys' gradients are taken times 2^up: float16 holds those of long rows
// (2^-14 and less) with fewer bits.
template <typename T> struct Lift { static constexpr float up = 0, down = 1; };
template <> struct Lift<f16> { static constexpr float up = 14, down = 1.0f / 16384; };

// Gradients far from 1 in float16: dS is rounded as 2^n times itself, with an n of the lane's query (or
// key) that falls whenever 2^n dS would pass kHighest, and the sums fall with it; so that its largest
// elements lie between 2^11 and 2^15, whatever the size of grad_out and v, and what float16 holds with
// fewer bits is 2^25 times smaller.  As it is, dS of 2048 keys and a grad_out of 2^-13 lies below
// float16's normal numbers (grad_k off by 28 times the bound that one rounding gives), and that of large
// gradients past its largest.  Without and with it, us, forward and backward: two sequences of
// 4096, 32 heads of 128 over 8 1271 / 1314; 12 ragged ones, window 1024, 16 heads of 64 over 4 104 / 112;
// 7 short ones, 12 heads of 96 42.7 / 46.0.
constexpr int kRaise = 60;  // n to begin with: 2^n dS is a float32 for all float16 inputs
constexpr float kHighest = 32768.0f;

// By how much n falls (0 most of the time) for 16 of a lane's elements and those of its other half.
template <int NT>
__device__ __forceinline__ int lower(f32x16& y, f32x16 (&acc)[NT]) {
  // what is masked is zero by now: chosen later, 16 masks would be kept until then
  asm volatile("" : "+v"(y));
  float m = 0;
#pragma unroll
  for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(y[r]));
  if (!__any(m > kHighest)) return 0;
  m = fmaxf(m, other_half(m));
  // what is not finite stays so
  const int by = m > kHighest && m < INFINITY ? __builtin_amdgcn_frexp_expf(m) - 12 : 0;
  const float f = ldexpf(1.0f, -by);
  y *= f;
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] *= f;
  return by;
}

// Query tiles that see at most so many keys make delta anew.  Error of the queries' gradient against 64
// bits over that of one rounding (bfloat16, 12 packed sequences up to 2500; two of 4096): 1.59 and 1.50
// without, 1.47 and 1.45 with it, 1.45 and 1.44 with 256 keys; backward of 30 sequences of 200, 32 heads
// 127 / 135 / 147 us, of two of 4096 no different.
constexpr int kFewKeys = 128;

// Gradient of the queries: the forward pass's loop over keys with dP^T = V grad_out^T beside S^T; dS^T
// = P^T (dP^T - delta), delta = grad_out . out, is the operand of dQ^T = K^T dS^T where it lies.  P comes
// from the rows' lse, so nothing of the size of S is kept.  Bound as the forward pass: two sequences of
// 4096, 32 heads of 128 over 8, causal, 4.2e11 operations in 413 us, 1.0 PFLOP/s.
template <typename T, int DP, int BLOCKS, int PARTS>
__global__ __launch_bounds__(64 * BLOCKS * PARTS, DP <= 64 ? 3 : 2) void attention_grad_q_kernel(
    Shape s, const Tile* __restrict__ tiles, int n_tiles, const T* __restrict__ q, int64_t q_token,
    int64_t q_head, const T* __restrict__ k, int64_t k_token, int64_t k_head,
    const T* __restrict__ v, int64_t v_token, int64_t v_head, const T* __restrict__ out,
    int64_t o_token, int64_t o_head, const float* __restrict__ lse, const T* __restrict__ go,
    int64_t go_token, int64_t go_head, T* __restrict__ dq, int64_t dq_token, int64_t dq_head,
    float* __restrict__ stats, int64_t q_tokens) {
  typedef Lay<DP> L;
  constexpr int NS = DP / 16, NT = DP / 32;
  constexpr int BYTES = PARTS * L::BYTES, ROWS = PARTS * kRows;
  __shared__ __attribute__((aligned(1024))) char s_k0[BYTES], s_v0[BYTES], s_k1[BYTES], s_v1[BYTES];
  int tile, a;
  tile_and_head(blockIdx.x, n_tiles, s.heads, tile, a);
  const Tile t = tiles[tile];
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = a / (s.heads / s.kv_heads);
  const int part = wave / BLOCKS, block = wave % BLOCKS, q0 = block * 32, mine = q0 + col;
  const bool active = q0 < t.rows;
  const int64_t row = t.first + (int64_t)min(mine, t.rows - 1);

  V8<T> qf[NS], gf[NS];
  float delta = 0;
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int d = 16 * i + 8 * half, at = d < s.dim ? d : 0;
    const V8<T> x = *reinterpret_cast<const V8<T>*>(q + row * q_token + a * q_head + at);
    const V8<T> y = *reinterpret_cast<const V8<T>*>(go + row * go_token + a * go_head + at);
    const V8<T> z = *reinterpret_cast<const V8<T>*>(out + row * o_token + a * o_head + at);
    qf[i] = scaled_sign<T>(x, s.scale, d < s.dim);
    gf[i] = keep_if<T>(y, d < s.dim);
#pragma unroll
    for (int e = 0; e < 8; ++e) delta += (float)gf[i][e] * (float)keep_if<T>(z, d < s.dim)[e];
  }
  delta += other_half(delta);
  const float c = exp2_scale(s.scale);
  float base = lse[row * s.heads + a];
  base = base == -INFINITY ? INFINITY : base * kLog2e;

  int lo, hi, lo0, hi0, lo1, hi1, lot, hit, none;
  seen_by(s, t, t.at + min(mine, t.rows - 1), lo, hi);
  seen_by(s, t, t.at + min(q0, t.rows - 1), lo0, hi0);
  seen_by(s, t, t.at + min(q0 + 31, t.rows - 1), lo1, hi1);
  seen_by(s, t, t.at, lot, none);
  seen_by(s, t, t.at + t.rows - 1, none, hit);

  f32x16 acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = f32x16{};

  const T* kb = k + (int64_t)t.k_begin * k_token + g * k_head;
  const T* vb = v + (int64_t)t.k_begin * v_token + g * v_head;
  auto load = [&](int j0, char* sk, char* sv) {
    const int n = min(ROWS, t.nk - j0);
    load_rows<DP, ROWS, BLOCKS * PARTS>(sk, kb + j0 * k_token, n, (uint32_t)(2 * k_token), s.dim,
                                        wave, lane);
    load_rows<DP, ROWS, BLOCKS * PARTS>(sv, vb + j0 * v_token, n, (uint32_t)(2 * v_token), s.dim,
                                        wave, lane);
  };
  const int r_at = L::row_at(lane);
  const int c_at = L::col_at(lane);

  // the scores and dP of 32 keys
  auto products = [&](const lds_char* sk, const lds_char* sv, int u, f32x16& x, f32x16& y) {
    x = f32x16{};
    y = f32x16{};
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      x = mfma32(row_frag<T>(sk + (r_at ^ (i * 32)) + u * 32 * L::PITCH), qf[i], x);
      y = mfma32(row_frag<T>(sv + (r_at ^ (i * 32)) + u * 32 * L::PITCH), gf[i], y);
    }
  };
  auto hide = [&](int j0, int u, f32x16& x) {
    if (j0 + kRows > hi0 || j0 < lo1) {
      const int first = lo - j0 - 4 * half, last = hi - j0 - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = 32 * u + 8 * (r / 4) + r % 4;
        x[r] = j >= first && j < last ? x[r] : 0.0f;
      }
    }
  };
  auto walk = [&](auto&& step) {
    auto wave_step = [&](int j0, const char* sk, const char* sv) {
      j0 += part * kRows;
      if (!active || j0 >= hi1 || j0 + kRows <= lo0) return;
      step(j0, (const lds_char*)sk + part * L::BYTES, (const lds_char*)sv + part * L::BYTES);
    };
    int j0 = lot;
    if (j0 < hit) load(j0, s_k0, s_v0);
    __syncthreads();
    while (j0 < hit) {
      if (j0 + ROWS < hit) load(j0 + ROWS, s_k1, s_v1);
      wave_step(j0, s_k0, s_v0);
      __syncthreads();
      j0 += ROWS;
      if (j0 >= hit) break;
      if (j0 + ROWS < hit) load(j0 + ROWS, s_k0, s_v0);
      wave_step(j0, s_k1, s_v1);
      __syncthreads();
      j0 += ROWS;
    }
  };

  // An output of few keys is large, and so is what its rounding does to delta = grad_out . out: there
  // delta is made anew, as the sum of the weights times dP.
  if (hit - lot <= kFewKeys) {
    delta = 0;
    walk([&](int j0, const lds_char* sk, const lds_char* sv) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x16 x, y;
        products(sk, sv, u, x, y);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], c, -base)) * y[r];
        hide(j0, u, x);
#pragma unroll
        for (int r = 0; r < 16; ++r) delta += x[r];
      }
    });
    delta += other_half(delta);
    if constexpr (PARTS > 1) {
      __shared__ float s_delta[PARTS][128];
      if (half == 0) s_delta[part][mine] = delta;
      __syncthreads();
      delta = s_delta[0][mine] + s_delta[1][mine];
    }
  }
  // what the keys' gradients start their products from: see there
  if (part == 0 && half == 0 && mine < t.rows) {
    stats[a * q_tokens + row] = (Lift<T>::up - base) / c;
    stats[(s.heads + a) * q_tokens + row] = -delta;
  }

  constexpr bool RAISED = std::is_same<T, f16>::value;
  int n = RAISED ? kRaise : 0;
  base -= n;
  walk([&](int j0, const lds_char* sk, const lds_char* sv) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (j0 + 32 * u >= hi1 || j0 + 32 * u + 32 <= lo0) continue;
      f32x16 x, y;
      products(sk, sv, u, x, y);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], c, -base)) * (y[r] - delta);
      hide(j0, u, x);
      if constexpr (RAISED) {
        const int by = lower(x, acc);
        base += by;
        n -= by;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const V8<T> f = to16<T>(x, 8 * i);
#pragma unroll
        for (int n = 0; n < NT; ++n)
          acc[n] = mfma32(col_frag<T, L::PITCH>(sk, c_at ^ (64 * n), 2 * u + i), f, acc[n]);
      }
    }
  });
  if constexpr (RAISED) {
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] *= ldexpf(1.0f, -n);
  }
  if constexpr (PARTS > 1) {
    float* theirs = reinterpret_cast<float*>(block == 0   ? s_k0
                                             : block == 1 ? s_v0
                                             : block == 2 ? s_k1
                                                          : s_v1);
    if (part == 1)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) theirs[(16 * i + r) * 64 + lane] = acc[i][r];
    __syncthreads();
    if (part == 1) return;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] += theirs[(16 * i + r) * 64 + lane];
  }
  if (mine < t.rows)
    store_rows<T, NT>(dq + row * dq_token + a * dq_head, acc, s.scale, s.dim, half);
}

// Gradients of the keys and values, BLOCKS * 32 keys a workgroup, over the heads of the group and their
// queries.  S and dP are [queries, keys], so P and dS are the operands of dV^T = grad_out^T P and
// dK^T = Q^T dS where they lie.  The products start from a row's -lse / scale and -delta, so that they
// give S - lse and dP - delta.  PARTS waves share 32 keys, one to every PARTS-th 32 queries;
// their sums are joined through LDS at the end, in their order.  S and dP are made a second time here:
// sums of dQ over the workgroups of a row's keys would cost atomics whose order changes results, or
// 32-bit copies in memory.  Bound as the forward pass: two sequences of 4096, 32 heads of 128 over 8,
// causal, 5.5e11 operations in 577 us, 0.96 PFLOP/s.
template <typename T, int DP, int BLOCKS, int PARTS>
__global__ __launch_bounds__(64 * BLOCKS * PARTS, 2) void attention_grad_kv_kernel(
    Shape s, const Tile* __restrict__ tiles, int n_tiles, const T* __restrict__ q, int64_t q_token,
    int64_t q_head, const T* __restrict__ k, int64_t k_token, int64_t k_head,
    const T* __restrict__ v, int64_t v_token, int64_t v_head, const T* __restrict__ go,
    int64_t go_token, int64_t go_head, const float* __restrict__ stats, int64_t q_tokens,
    T* __restrict__ dk, int64_t dk_token, int64_t dk_head, T* __restrict__ dv, int64_t dv_token,
    int64_t dv_head, int split, float* __restrict__ sums, int64_t k_tokens) {
  typedef Lay<DP> L;
  constexpr int NS = DP / 16, NT = DP / 32;
  constexpr int ROWS = 32 * PARTS, BYTES = ROWS * L::PITCH;
  __shared__ __attribute__((aligned(1024))) char s_q0[BYTES], s_g0[BYTES], s_q1[BYTES], s_g1[BYTES];
  __shared__ __attribute__((aligned(256))) float s_x0[ROWS], s_y0[ROWS], s_x1[ROWS], s_y1[ROWS];
  int tile, g;
  tile_and_head(blockIdx.x, n_tiles, s.kv_heads * split, tile, g);
  const int share = g % split;  // of the group's heads
  g /= split;
  const Tile t = tiles[tile];
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave % PARTS, block = wave / PARTS, k0 = block * 32, mine = k0 + col;
  const bool active = k0 < t.rows;
  const int group = s.heads / s.kv_heads / split;
  const int64_t row = t.first + (int64_t)min(mine, t.rows - 1);

  V8<T> kf[NS], vf[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int d = 16 * i + 8 * half, at = d < s.dim ? d : 0;
    const V8<T> x = *reinterpret_cast<const V8<T>*>(k + row * k_token + g * k_head + at);
    const V8<T> y = *reinterpret_cast<const V8<T>*>(v + row * v_token + g * v_head + at);
    kf[i] = scaled_sign<T>(x, s.scale, d < s.dim);
    vf[i] = keep_if<T>(y, d < s.dim);
  }
  const float c = exp2_scale(s.scale);

  // the queries that see any of the wave's keys and of the tile's
  int lo0, hi0, lo1, hi1, lot, hit, none;
  seen_of(s, t, t.at + min(k0, t.rows - 1), lo0, hi0);
  seen_of(s, t, t.at + min(k0 + 31, t.rows - 1), lo1, hi1);
  seen_of(s, t, t.at, lot, none);
  seen_of(s, t, t.at + t.rows - 1, none, hit);

  f32x16 ak[NT], av[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) ak[i] = av[i] = f32x16{};

  constexpr bool RAISED = std::is_same<T, f16>::value;
  float raised = RAISED ? ldexpf(Lift<T>::down, kRaise) : 1.0f;  // 2^n, and P's lift taken back

  const int r_at = L::row_at(lane) + part * 32 * L::PITCH;
  const int c_at = L::col_at(lane) + part * 32 * L::PITCH;

  auto load = [&](int a, int i0, char* sq, char* sg, float* sx, float* sy) {
    const int n = min(ROWS, t.nq - i0);
    const int64_t first = (int64_t)t.q_begin + i0;
    // the rows' offsets are made anew in every step: kept, they would not fit the registers
    int l = lane;
    asm volatile("" : "+v"(l));
    load_rows<DP, ROWS, BLOCKS * PARTS>(sq, q + first * q_token + a * q_head, n,
                                        (uint32_t)(2 * q_token), s.dim, wave, l);
    load_rows<DP, ROWS, BLOCKS * PARTS>(sg, go + first * go_token + a * go_head, n,
                                        (uint32_t)(2 * go_token), s.dim, wave, l);
    if (wave < PARTS) {  // 64 rows' statistics a wave
      const int which = wave & 1, at = (wave >> 1) * 64;
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<float*>(stats + (which * s.heads + a) * q_tokens + first), 0, 4 * n, 0x00027000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)((which ? sy : sx) + at), 4, 4 * (at + l), 0,
          0, 0);
    }
  };

  auto step = [&](int i0, const char* sq_, const char* sg_, const float* sx, const float* sy) {
    const int i1 = i0 + 32 * part;  // the wave's first query
    if (!active || i1 >= hi1 || i1 + 32 <= lo0) return;
    const lds_char* sq = (const lds_char*)sq_;
    const lds_char* sg = (const lds_char*)sg_;
    int ra = r_at, ca = c_at;  // what is made of them is made anew, as in load
    asm volatile("" : "+v"(ra), "+v"(ca));
    f32x16 x, y;
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const f32x4 x0 = *reinterpret_cast<const f32x4*>(sx + 32 * part + 2 * r + 4 * half);
      const f32x4 y0 = *reinterpret_cast<const f32x4*>(sy + 32 * part + 2 * r + 4 * half);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[r + e] = x0[e], y[r + e] = y0[e];
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      x = mfma32(row_frag<T>(sq + (ra ^ (i * 32))), kf[i], x);
      y = mfma32(row_frag<T>(sg + (ra ^ (i * 32))), vf[i], y);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = __builtin_amdgcn_exp2f(x[r] * c);
      y[r] *= x[r] * raised;
    }
    if (i1 + 32 > hi0 || i1 < lo1) {
      int key = mine, lo, hi;  // what sees this lane's key: made anew, as above
      asm volatile("" : "+v"(key));
      seen_of(s, t, t.at + min(key, t.rows - 1), lo, hi);
      const int first = lo - i1 - 4 * half, last = hi - i1 - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = 8 * (r / 4) + r % 4;
        const bool in = i >= first && i < last;
        x[r] = in ? x[r] : 0.0f;
        y[r] = in ? y[r] : 0.0f;
      }
    }
    if constexpr (RAISED) raised = ldexpf(raised, -lower(y, ak));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const V8<T> p = to16<T>(x, 8 * i), ds = to16<T>(y, 8 * i);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        av[n] = mfma32(col_frag<T, L::PITCH>(sg, ca ^ (64 * n), i), p, av[n]);
        ak[n] = mfma32(col_frag<T, L::PITCH>(sq, ca ^ (64 * n), i), ds, ak[n]);
      }
    }
  };

  // From the last queries back, the heads of the group in turn: the tiles of a sequence that started
  // together read the same rows together, wherever their keys' first queries lie.  Two sequences of 4096,
  // 32 heads of 128 over 8: 1.98 GB past the L2s with a head after the other from its first query
  // on, 0.56 GB so; forward and backward 1222 and 1194 us.
  const int steps = hit > lot ? (hit - lot + ROWS - 1) / ROWS : 0;
  const int total = steps * group, a0 = (g * split + share) * group;
  int a = a0, i0 = lot + (steps - 1) * ROWS;  // of this step
  int a1 = a, i1 = i0;                        // of the one being loaded
  auto next = [&] {
    if (++a1 == a0 + group) a1 = a0, i1 -= ROWS;
  };
  if (total) load(a, i0, s_q0, s_g0, s_x0, s_y0);
  __syncthreads();
  for (int n = 0; n < total;) {
    next();
    if (n + 1 < total) load(a1, i1, s_q1, s_g1, s_x1, s_y1);
    step(i0, s_q0, s_g0, s_x0, s_y0);
    __syncthreads();
    a = a1, i0 = i1;
    if (++n >= total) break;
    next();
    if (n + 1 < total) load(a1, i1, s_q0, s_g0, s_x0, s_y0);
    step(i0, s_q1, s_g1, s_x1, s_y1);
    __syncthreads();
    a = a1, i0 = i1;
    ++n;
  }

  if constexpr (RAISED) {
#pragma unroll
    for (int i = 0; i < NT; ++i) ak[i] *= Lift<T>::down / raised;
  }
  // join the waves of the same keys
  float* joined = reinterpret_cast<float*>(block ? s_q1 : s_q0);
  static_assert((PARTS - 1) * 16 * 64 * 4 <= BYTES, "");
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    f32x16* acc = which ? ak : av;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if (part)
#pragma unroll
        for (int r = 0; r < 16; ++r) joined[(16 * (part - 1) + r) * 64 + lane] = acc[i][r];
      __syncthreads();
      if (part == 0)
#pragma unroll
        for (int p = 0; p < PARTS - 1; ++p)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] += joined[(16 * p + r) * 64 + lane];
      __syncthreads();
    }
  }
  if (part == 0 && mine < t.rows) {
    if (split > 1) {
      float* to = sums + ((int64_t)(share * s.kv_heads + g) * k_tokens + row) * s.dim;
      store_rows<float, NT>(to, av, Lift<T>::down, s.dim, half);
      store_rows<float, NT>(to + (int64_t)split * s.kv_heads * k_tokens * s.dim, ak, s.scale, s.dim, half);
      return;
    }
    store_rows<T, NT>(dv + row * dv_token + g * dv_head, av, Lift<T>::down, s.dim, half);
    store_rows<T, NT>(dk + row * dk_token + g * dk_head, ak, s.scale, s.dim, half);
  }
}

// The keys' and values' gradients as the sums of ``split`` shares of the heads, in their order: a thread
// to four elements.  Bound by memory and its launch: 12 ragged sequences up to 2500, 4 key heads of 64
// by 2 shares, 26 MB in 5.9 us.
template <typename T>
__global__ __launch_bounds__(256) void attention_grad_kv_sum_kernel(
    Shape s, int split, const float* __restrict__ sums, int64_t k_tokens, T* __restrict__ dk,
    int64_t dk_token, int64_t dk_head, T* __restrict__ dv, int64_t dv_token, int64_t dv_head) {
  const int64_t each = (int64_t)s.kv_heads * k_tokens * s.dim;  // elements of one share
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= 2 * each) return;
  const bool keys = i >= each;
  const int64_t at = keys ? i - each : i;
  const float* from = sums + (keys ? split * each : 0) + at;
  f32x4 y = *reinterpret_cast<const f32x4*>(from);
  for (int p = 1; p < split; ++p) y += *reinterpret_cast<const f32x4*>(from + p * each);
  const int64_t row = at / s.dim;
  const int64_t g = row / k_tokens, t = row - g * k_tokens;
  T* to = (keys ? dk + t * dk_token + g * dk_head : dv + t * dv_token + g * dv_head) + at % s.dim;
  *reinterpret_cast<V4<T>*>(to) = __builtin_convertvector(y, V4<T>);
}

template <typename T>
const T* in(const void* p) { return static_cast<const T*>(p); }

Shape shape_of(const fsp_attention_packed_args& a) {
  return {(int)a.heads, (int)a.kv_heads, (int)a.dim, a.causal != 0, (int)a.window,
          (float)a.scale};
}

// Twice as many waves share a tile where that fills CUs, or shortens the chains that the others end up
// waiting for: those of a long causal sequence without a window, where the tiles are uneven and all
// on the chip at once.  Measured without and with it, us, 16 heads over 4 (tiles times heads):
// forward, dim 128: one sequence of 2048 (256) 41 / 33, of 4096 (512) 91 / 82, under a window of 1024
// 45 / 49; dim 64, whose workgroups go four to a CU: 4096 (512) 53 / 46, two of 4096 (1024) 90 / 85.
// Gradient of the queries, dim 128: 2048 56 / 48, 4096 under a window 63 / 70; 8192, 8 heads 232 / 203.
// Gradients of the keys, dim 128: 3000, 4 heads over 4 (188) 48 / 35; two of 4096 (512) 378 / 286; two
// of 2048 under a window (512) 77 / 96; three short ones (40) 9 / 12; the whole backward pass of 900, 16
// heads (240) 50.3 / 48.5, of two of 700, 8 heads (176) 42.7 / 42.7.
constexpr int64_t kCus = 256;

int64_t seen_at_most(const fsp_attention_packed_args& a, int64_t longest) {
  return a.window && a.window < longest ? a.window : longest;
}

bool share_queries(const fsp_attention_packed_args& a, int64_t fill) {
  const int64_t n = a.n_q_tiles * a.heads;
  return seen_at_most(a, a.k_longest) >= 512 &&
         (n <= fill || (n <= 2 * kCus && a.causal && !a.window && a.k_longest >= 2048));
}

// Tiles of half the queries, with two waves to 32 of them, where whole tiles would leave CUs without any
// and there is more than one step of keys.  Measured without and with them, us (tiles times heads):
// forward, dim 128: one sequence of 512, 16 heads (64) 14.4 / 12.6, of 2048, 4 heads (64) 31.9 / 30.1, of
// 4000, 8 heads (256) 58 / 64; four of 64, 4 heads (16) 6.0 / 7.9; dim 64, whose workgroups go two
// to a CU: 2048, 8 heads (128) 22.4 / 18.5, 4000 (256) 39.6 / 35.4.  Gradient of the queries, dim 128:
// 512 (64) 20.4 / 15.9, 2048 (64) 44.8 / 38.6, 4000 (256) 82 / 86; dim 64: 2048 (128) 28.9 / 25.3.
bool halve_tiles(const fsp_attention_packed_args& a, int64_t most) {
  return a.n_q_tiles * a.heads <= most && seen_at_most(a, a.k_longest) > kRows;
}

bool share_keys(const fsp_attention_packed_args& a, int split) {
  const int64_t n = a.n_k_tiles * a.kv_heads * split;
  return (n <= kCus && a.heads / a.kv_heads / split * seen_at_most(a, a.q_longest) >= 768) ||
         (n <= 2 * kCus && a.causal && !a.window && a.q_longest >= 4096);
}

// Tiles of half the keys, with four waves to them, where whole ones leave CUs without any.  Measured
// without and with them, us, the whole backward pass (tiles times heads): dim 128: two of 256, 4 heads (32)
// 29.7 / 30.6, one of 500, 16 heads over 4 (128) 40.7 / 38.1, 4000, 2 heads (126) 136 / 127, 2000, 8
// heads (256) 79 / 84; dim 64: 65 tokens 15.8 / 15.4, two of 256 (32) 19.9 / 18.9, 2000, 8 heads (256)
// 49.2 / 46.8.
bool halve_keys(const fsp_attention_packed_args& a, int split) {
  const bool small = a.dim <= 64;
  return a.n_k_tiles * a.kv_heads * split <= (small ? kCus : kCus / 2) &&
         seen_at_most(a, a.q_longest) > (small ? kRows : 4 * kRows);
}

// Shares of a group's heads that go to workgroups of their own, for their sums to be added by another
// launch: as many as three workgroups to a CU take, or five and a half where the tiles are uneven
// (causal without a window) and smaller ones even them out.  Gradients of the keys with the limit at
// 2, 3, 4 and 6, us: 12 ragged sequences up to 2500, 16 heads of 64 over 4: 135 / 80 / 79 / 56, under a
// window of 1024 61 / 43 / 43 / 48; 4096 under that window, heads of 128: 85 / 83 / 95 / 95; 5000, 32 heads
// of 128 over 8: 485 / 488 / 492 / 424; 4096, 24 heads over 8: 220 / 218 / 218 / 233.
int split_heads(int64_t n_k_tiles, int64_t heads, int64_t kv_heads, bool uneven) {
  const int64_t group = heads / kv_heads, n = n_k_tiles * kv_heads;
  const int64_t most = uneven ? 11 * kCus / 2 : 3 * kCus;
  int64_t split = 1;
  for (int64_t i = 2; i <= group && i * n <= most; ++i)
    if (group % i == 0) split = i;
  return (int)split;
}

template <typename T, int DP, int BLOCKS, int PARTS>
int launch_forward(const fsp_attention_packed_args& a, hipStream_t st) {
  const int32_t* tiles = BLOCKS == 2 ? a.q_halves : a.q_tiles;
  const int64_t n = BLOCKS == 2 ? a.n_q_halves : a.n_q_tiles;
  hipLaunchKernelGGL((attention_packed_kernel<T, DP, BLOCKS, PARTS>),
                     dim3((unsigned)(n * a.heads)), dim3(64 * BLOCKS * PARTS), 0, st, shape_of(a),
                     reinterpret_cast<const Tile*>(tiles), (int)n, in<T>(a.q),
                     a.q_token, a.q_head, in<T>(a.k), a.k_token, a.k_head, in<T>(a.v), a.v_token,
                     a.v_head, static_cast<T*>(a.out), a.out_token, a.out_head, a.lse);
  return check_hip(hipGetLastError(), "attention_packed_kernel launch");
}

template <typename T, int DP>
int launch_forward_parts(const fsp_attention_packed_args& a, hipStream_t st) {
  if (halve_tiles(a, DP <= 64 ? kCus : kCus / 2)) return launch_forward<T, DP, 2, 2>(a, st);
  return share_queries(a, DP <= 64 ? 4 * kCus : kCus) ? launch_forward<T, DP, 4, 2>(a, st)
                                                      : launch_forward<T, DP, 4, 1>(a, st);
}

template <typename T>
int launch_forward_dim(const fsp_attention_packed_args& a, hipStream_t st) {
  if (a.dim <= 64) return launch_forward_parts<T, 64>(a, st);
  if (a.dim <= 96) return launch_forward_parts<T, 96>(a, st);
  return launch_forward_parts<T, 128>(a, st);
}

template <typename T, int DP, int BLOCKS, int PARTS>
int launch_grad_q(const fsp_attention_packed_args& a, hipStream_t st) {
  const int32_t* tiles = BLOCKS == 2 ? a.q_halves : a.q_tiles;
  const int64_t n = BLOCKS == 2 ? a.n_q_halves : a.n_q_tiles;
  hipLaunchKernelGGL((attention_grad_q_kernel<T, DP, BLOCKS, PARTS>),
                     dim3((unsigned)(n * a.heads)), dim3(64 * BLOCKS * PARTS), 0, st, shape_of(a),
                     reinterpret_cast<const Tile*>(tiles), (int)n, in<T>(a.q),
                     a.q_token, a.q_head, in<T>(a.k), a.k_token, a.k_head, in<T>(a.v), a.v_token,
                     a.v_head, in<T>(a.out), a.out_token, a.out_head, a.lse, in<T>(a.grad_out),
                     a.grad_out_token, a.grad_out_head, static_cast<T*>(a.grad_q), a.grad_q_token,
                     a.grad_q_head, static_cast<float*>(a.workspace), a.q_tokens);
  return check_hip(hipGetLastError(), "attention_grad_q_kernel launch");
}

template <typename T, int DP, int BLOCKS, int PARTS>
int launch_grad_kv(const fsp_attention_packed_args& a, int split, hipStream_t st) {
  const int32_t* tiles = BLOCKS == 1 ? a.k_halves : a.k_tiles;
  const int64_t n = BLOCKS == 1 ? a.n_k_halves : a.n_k_tiles;
  float* stats = static_cast<float*>(a.workspace);
  float* sums = stats + ((2 * a.heads * a.q_tokens + 3) & ~int64_t(3));
  hipLaunchKernelGGL((attention_grad_kv_kernel<T, DP, BLOCKS, PARTS>),
                     dim3((unsigned)(n * a.kv_heads * split)), dim3(64 * BLOCKS * PARTS), 0, st,
                     shape_of(a), reinterpret_cast<const Tile*>(tiles), (int)n,
                     in<T>(a.q), a.q_token, a.q_head, in<T>(a.k), a.k_token, a.k_head, in<T>(a.v),
                     a.v_token, a.v_head, in<T>(a.grad_out), a.grad_out_token, a.grad_out_head,
                     stats, a.q_tokens, static_cast<T*>(a.grad_k), a.grad_k_token, a.grad_k_head,
                     static_cast<T*>(a.grad_v), a.grad_v_token, a.grad_v_head, split, sums,
                     a.k_tokens);
  if (int rc = check_hip(hipGetLastError(), "attention_grad_kv_kernel launch")) return rc;
  if (split == 1) return FSP_OK;
  const int64_t quads = a.kv_heads * a.k_tokens * a.dim / 2;
  hipLaunchKernelGGL((attention_grad_kv_sum_kernel<T>), dim3((unsigned)((quads + 255) / 256)),
                     dim3(256), 0, st, shape_of(a), split, sums, a.k_tokens,
                     static_cast<T*>(a.grad_k), a.grad_k_token, a.grad_k_head,
                     static_cast<T*>(a.grad_v), a.grad_v_token, a.grad_v_head);
  return check_hip(hipGetLastError(), "attention_grad_kv_sum_kernel launch");
}

template <typename T, int DP>
int launch_backward(const fsp_attention_packed_args& a, hipStream_t st) {
  if (a.n_q_tiles > 0) {
    const int rc = halve_tiles(a, kCus / 2) ? launch_grad_q<T, DP, 2, 2>(a, st)
                   : share_queries(a, kCus) ? launch_grad_q<T, DP, 4, 2>(a, st)
                                            : launch_grad_q<T, DP, 4, 1>(a, st);
    if (rc) return rc;
  }
  if (a.n_k_tiles > 0) {
    const int split = split_heads(a.n_k_tiles, a.heads, a.kv_heads, a.causal && !a.window);
    if (halve_keys(a, split)) return launch_grad_kv<T, DP, 1, 4>(a, split, st);
    return share_keys(a, split) ? launch_grad_kv<T, DP, 2, 4>(a, split, st)
                                : launch_grad_kv<T, DP, 2, 2>(a, split, st);
  }
  return FSP_OK;
}

template <typename T>
int launch_backward_dim(const fsp_attention_packed_args& a, hipStream_t st) {
  if (a.dim <= 64) return launch_backward<T, 64>(a, st);
  if (a.dim <= 96) return launch_backward<T, 96>(a, st);
  return launch_backward<T, 128>(a, st);
}

int check_packed(const fsp_attention_packed_args& a, const std::string& who) {
  if (!attn_dtype(a.dtype)) return set_error(FSP_ENOTSUP, who + ": dtype");
  if (!attn_dim(a.dim)) return set_error(FSP_ENOTSUP, who + ": dim");
  if (a.kv_heads < 1 || a.heads < 1 || a.heads % a.kv_heads || a.heads > 0xffff)
    return set_error(FSP_EINVAL, who + ": heads must be a multiple of kv_heads");
  if (a.q_tokens < 0 || a.k_tokens < 0 || a.n_q_tiles < 0 || a.n_k_tiles < 0 ||
      a.n_q_halves < 0 || a.n_k_halves < 0 || a.window < 0 || a.q_longest < 0 || a.k_longest < 0 ||
      a.q_tokens > kAttnTokensCap || a.k_tokens > kAttnTokensCap || a.window > 0x7fffffffLL ||
      a.n_q_tiles > kMaxBlocks / a.heads || a.n_q_halves > kMaxBlocks / a.heads ||
      a.n_k_tiles > kMaxBlocks / a.heads || a.n_k_halves > kMaxBlocks / a.heads)
    return set_error(FSP_EINVAL, who + ": size out of range");
  auto step = [&](int64_t tokens, int64_t by) {
    return (tokens < 2 || by >= a.dim) && by >= 0 && by <= kTokenStep;
  };
  if (!step(a.q_tokens, a.q_token) || !step(a.k_tokens, a.k_token) ||
      !step(a.k_tokens, a.v_token) || (a.n_k_tiles > 0 && !step(a.q_tokens, a.grad_out_token)))
    return set_error(FSP_EINVAL, who + ": a token's step must lie between dim and 2^23");
  if (!isfinite((float)a.scale)) return set_error(FSP_EINVAL, who + ": scale must be finite in 32 bits");
  if (a.window && !a.causal) return set_error(FSP_EINVAL, who + ": window needs causal");
  if ((a.n_q_tiles > 0 && (!a.q_tiles || !a.q_halves || !a.q || !a.out || !a.lse)) ||
      (a.n_k_tiles > 0 && (!a.k_tiles || !a.k_halves)) || (a.k_tokens > 0 && (!a.k || !a.v)))
    return set_error(FSP_EINVAL, who + ": null pointer");
  if (!aligned16(a.q, a.q_token, a.q_head) || !aligned16(a.k, a.k_token, a.k_head) ||
      !aligned16(a.v, a.v_token, a.v_head) || !aligned16(a.out, a.out_token, a.out_head))
    return set_error(FSP_EINVAL, who + ": rows must be 16-byte aligned");
  return FSP_OK;
}

}  // namespace
}  // namespace fsp

using namespace fsp;

extern "C" int64_t fsp_attention_packed_workspace(int64_t n_k_tiles, int64_t heads, int64_t kv_heads,
                                                  int64_t dim, int64_t q_tokens, int64_t k_tokens,
                                                  int uneven) {
  if (n_k_tiles < 0 || heads < 1 || kv_heads < 1 || dim < 0 || q_tokens < 0 || k_tokens < 0) return 0;
  const int split = split_heads(n_k_tiles, heads, kv_heads, uneven);
  const int64_t stats = (2 * heads * q_tokens + 3) & ~int64_t(3);
  return sizeof(float) * (stats + (split > 1 ? 2 * split * kv_heads * k_tokens * dim : 0));
}

extern "C" int64_t fsp_attention_packed_tile(int which) {
  return which == 0 ? kTile : which == 1 ? kTile / 2 : which == 2 ? kRows : kRows / 2;
}

extern "C" int fsp_attention_packed(const fsp_attention_packed_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_packed: null arguments");
  const fsp_attention_packed_args& a = *args;
  if (int rc = check_packed(a, "fsp_attention_packed")) return rc;
  if (a.n_q_tiles == 0) return FSP_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FSP_BF16 ? launch_forward_dim<bf16>(a, st) : launch_forward_dim<f16>(a, st);
}

extern "C" int fsp_attention_packed_backward(const fsp_attention_packed_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_packed_backward: null arguments");
  const fsp_attention_packed_args& a = *args;
  if (int rc = check_packed(a, "fsp_attention_packed_backward")) return rc;
  // without queries, and with one share of the heads, there is nothing to keep
  const bool work = a.n_k_tiles > 0 && fsp_attention_packed_workspace(a.n_k_tiles, a.heads, a.kv_heads, a.dim,
                                                                      a.q_tokens, a.k_tokens,
                                                                      a.causal && !a.window) > 0;
  if ((a.n_q_tiles > 0 && (!a.grad_out || !a.grad_q || !a.workspace)) ||
      (a.n_k_tiles > 0 && (!a.grad_k || !a.grad_v)) || (work && !a.workspace))
    return set_error(FSP_EINVAL, "fsp_attention_packed_backward: null pointer");
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return set_error(FSP_EINVAL, "fsp_attention_packed_backward: workspace must be 16-byte aligned");
  if (!aligned16(a.grad_out, a.grad_out_token, a.grad_out_head) ||
      !aligned16(a.grad_q, a.grad_q_token, a.grad_q_head) ||
      !aligned16(a.grad_k, a.grad_k_token, a.grad_k_head) ||
      !aligned16(a.grad_v, a.grad_v_token, a.grad_v_head))
    return set_error(FSP_EINVAL, "fsp_attention_packed_backward: rows must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FSP_BF16 ? launch_backward_dim<bf16>(a, st) : launch_backward_dim<f16>(a, st);
}
