// Attention over packed sequences, forward and backward.
#include "tiles.hpp"

namespace fsp {
namespace {

constexpr int kTile = 128;  // query rows of a workgroup, 32 a wave

constexpr int64_t kTokenStep = 1 << 23;  // the bytes of a load's 128 rows are a 32-bit offset

struct Tile {
  int first, rows, at, q_begin, nq, k_begin, nk, pad;
};

// sinks: so many first keys of a sequence stay visible to queries whose window has left them.  width: so many
// heads of a group lie side by side in a tile of queries, each token's in turn (1 without sinks).
struct Shape {
  int heads, kv_heads, dim, causal, window;
  float scale;
  int sinks, width;
};

// The keys that a tile of queries reads in steps: those that its window holds, [lot, hit), and the first ones
// before them that stay visible, as if these lay right before lot: places [begin, end), of which place i is key i
// below ``sinks`` and key at(i) from there on.  Without any, places are keys: counted from lot, the gradient of the
// queries took 33.5 us for 33.0 (12 ragged sequences up to 2500, window 1024, 16 heads of 64).
template <bool SINKS>
struct Walk {
  int lot, sinks, begin, end;
  __device__ Walk(const Shape& s, int lot, int hit)
      : lot(lot), sinks(SINKS ? min(s.sinks, lot) : 0), begin(SINKS ? 0 : lot),
        end(!SINKS ? hit : hit > lot ? hit - lot + sinks : 0) {}
  __device__ int at(int i) const { return SINKS ? lot - sinks + i : i; }
  __device__ bool gap(int i) const { return SINKS && i < sinks && sinks < lot; }  // in a step from i on
};

// The rows of a tile of queries: row r is token r / width of the tile, of ``width`` heads from a on.
template <bool SINKS>
struct Rows {
  int width;
  __device__ Rows(const Shape& s) : width(SINKS ? s.width : 1) {}
  __device__ int token(int r) const { return SINKS ? r / width : r; }
  __device__ int head(int r) const { return SINKS ? r % width : 0; }
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

// The same where the first ``sinks`` - i0 of the rows lie at row i0 and the others, up to row n, from row lot on.
template <int DP, int ROWS, int WAVES>
__device__ __forceinline__ void load_rows_apart(char* lds, const void* src, int i0, int sinks, int lot, int n,
                                                uint32_t bytes, int64_t step, int dim, int wave, int lane) {
  typedef Lay<DP> L;
  const char* from = static_cast<const char*>(src);
  const int first = sinks - i0;
  const __amdgpu_buffer_rsrc_t near = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(from + i0 * step), 0, (int)((uint32_t)(min(first, ROWS) - 1) * bytes + 2 * dim), 0x00027000);
  const __amdgpu_buffer_rsrc_t far = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(from + lot * step), 0, (int)((uint32_t)(min(n - lot, ROWS) - 1) * bytes + 2 * dim),
      0x00027000);
  constexpr int PER = ROWS * L::PITCH / 1024 / WAVES, EACH = 1024 / L::PITCH;
  const int chunk = (lane % L::CH) ^ L::swizzle(lane / L::CH) ^ L::swizzle(wave * PER * EACH);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = 16 * (chunk ^ L::swizzle(i * EACH)), r = (wave * PER + i) * EACH + lane / L::CH;
    const uint32_t off = at < 2 * dim ? (uint32_t)(r < first ? r : r - first) * bytes + at : 0x80000000u;
    const auto to = (__attribute__((address_space(3))) void*)(lds + (wave * PER + i) * 1024);
    if (r < first)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(near, to, 16, (int)off, 0, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(far, to, 16, (int)off, 0, 0, 0);
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
template <typename T, int DP, int BLOCKS, int PARTS, bool SINKS>
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
  tile_and_head(blockIdx.x, n_tiles, SINKS ? s.heads / s.width : s.heads, tile, a);
  const Tile t = tiles[tile];
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Rows<SINKS> row_of(s);
  if (SINKS) a *= row_of.width;
  const int g = a / (s.heads / s.kv_heads), rows = t.rows * row_of.width;
  const int part = wave / BLOCKS, block = wave % BLOCKS, q0 = block * 32;
  const int mine = q0 + col;  // this lane's row of the tile
  const bool active = q0 < rows;

  V8<T> qf[NS];
  {
    const int r = min(mine, rows - 1);
    const T* qr = q + (t.first + (int64_t)row_of.token(r)) * q_token + (a + row_of.head(r)) * q_head;
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
  seen_by(s, t, t.at + row_of.token(min(mine, rows - 1)), lo, hi);
  seen_by(s, t, t.at + row_of.token(min(q0, rows - 1)), lo0, hi0);
  seen_by(s, t, t.at + row_of.token(min(q0 + 31, rows - 1)), lo1, hi1);
  seen_by(s, t, t.at, lot, none);
  seen_by(s, t, t.at + t.rows - 1, none, hit);

  f32x16 o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = f32x16{};
  float top = -INFINITY, sum = 0;

  const T* kb = k + (int64_t)t.k_begin * k_token + g * k_head;
  const T* vb = v + (int64_t)t.k_begin * v_token + g * v_head;
  const Walk<SINKS> keys(s, lot, hit);
  auto load = [&](int i0, char* sk, char* sv) {
    if (keys.gap(i0)) {
      load_rows_apart<DP, ROWS, BLOCKS * PARTS>(sk, kb, i0, keys.sinks, lot, t.nk, (uint32_t)(2 * k_token),
                                                2 * k_token, s.dim, wave, lane);
      load_rows_apart<DP, ROWS, BLOCKS * PARTS>(sv, vb, i0, keys.sinks, lot, t.nk, (uint32_t)(2 * v_token),
                                                2 * v_token, s.dim, wave, lane);
      return;
    }
    const int j0 = keys.at(i0), n = min(ROWS, t.nk - j0);
    load_rows<DP, ROWS, BLOCKS * PARTS>(sk, kb + j0 * k_token, n, (uint32_t)(2 * k_token), s.dim,
                                        wave, lane);
    load_rows<DP, ROWS, BLOCKS * PARTS>(sv, vb + j0 * v_token, n, (uint32_t)(2 * v_token), s.dim,
                                        wave, lane);
  };
  const int k_at = L::row_at(lane);
  const int v_at = L::col_at(lane);

  auto step = [&](int i0, const char* sk_, const char* sv_) {
    i0 += part * kRows;
    const int j0 = keys.at(i0);  // the first key, or what it would be without the ones before the window
    if (!active || j0 >= hi1 || (j0 + kRows <= lo0 && !(SINKS && i0 < s.sinks))) return;
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
      if constexpr (SINKS) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          seen_or_none((bits_from(lo - j0 - 32 * u) | ~bits_from(s.sinks - i0 - 32 * u)) &
                           ~bits_from(hi - j0 - 32 * u), half, x[u]);
      } else {
        const int first = lo - j0 - 4 * half, last = hi - j0 - 4 * half;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = 32 * u + 8 * (r / 4) + r % 4;
            x[u][r] = j >= first && j < last ? x[u][r] : -INFINITY;
          }
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

  int i0 = keys.begin;
  if (i0 < keys.end) load(i0, s_k0, s_v0);
  __syncthreads();
  while (i0 < keys.end) {
    if (i0 + ROWS < keys.end) load(i0 + ROWS, s_k1, s_v1);
    step(i0, s_k0, s_v0);
    __syncthreads();
    i0 += ROWS;
    if (i0 >= keys.end) break;
    if (i0 + ROWS < keys.end) load(i0 + ROWS, s_k0, s_v0);
    step(i0, s_k1, s_v1);
    __syncthreads();
    i0 += ROWS;
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
  if (mine >= rows) return;
  const int64_t row = t.first + row_of.token(mine);
  a += row_of.head(mine);
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
// Under a window with first tokens, where no query may come to see many, the rule is finer: by what a tile's first
// query sees, and by the dim, as what the output's rounding does to delta against what one rounding does to
// the gradient falls with its root.  The same ratio without it, of rows that see 140 / 300 / 500 / 700 / 1200 / 1600
// keys, the mean of both types: dim 48 1.53 / 1.50 / 1.51 / 1.50 / 1.50 / 1.51, 64 1.51 / 1.51 / 1.50 / 1.49 / 1.49 /
// 1.49, 72 1.51 / 1.51 / 1.48 / 1.48 / 1.48 / 1.47, 80 1.50 / 1.48 / 1.47 / 1.49 / 1.48 / 1.47, 96 1.50 / 1.48 / 1.48 /
// 1.46 / 1.47 / 1.46, 128 1.49 / 1.47 / 1.47 / 1.45 / 1.46 / 1.45, some 0.02 up or down from case to case; with it
// 1.42 to 1.47 everywhere.  There is no step in that: it is made anew up to the power of two from which on the mean is
// below 1.50 without (dims below 64 never get there).  This kernel with delta made anew by no tile / by this rule / by
// all: four sequences of 4096, 16 heads of 64, 528 keys a query 72.5 / 81.7 / 114.5 us; 6 up to 1501, 12 heads of 96,
// 270 keys, where the longest tile is all of it, 18.9 / 27.8 / 27.6.
__device__ __forceinline__ bool delta_anew(int dim, int seen) {
  return seen <= 256 || dim < 64 || (dim < 80 && seen <= 512);
}

// Gradient of the queries: the forward pass's loop over keys with dP^T = V grad_out^T beside S^T; dS^T
// = P^T (dP^T - delta), delta = grad_out . out, is the operand of dQ^T = K^T dS^T where it lies.  P comes
// from the rows' lse, so nothing of the size of S is kept.  Bound as the forward pass: two sequences of
// 4096, 32 heads of 128 over 8, causal, 4.2e11 operations in 413 us, 1.0 PFLOP/s.
template <typename T, int DP, int BLOCKS, int PARTS, bool SINKS>
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
  tile_and_head(blockIdx.x, n_tiles, SINKS ? s.heads / s.width : s.heads, tile, a);
  const Tile t = tiles[tile];
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Rows<SINKS> row_of(s);
  if (SINKS) a *= row_of.width;
  const int g = a / (s.heads / s.kv_heads), rows = t.rows * row_of.width;
  const int part = wave / BLOCKS, block = wave % BLOCKS, q0 = block * 32, mine = q0 + col;
  const bool active = q0 < rows;
  const int64_t row = t.first + (int64_t)row_of.token(min(mine, rows - 1));
  a += row_of.head(min(mine, rows - 1));

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
  seen_by(s, t, t.at + row_of.token(min(mine, rows - 1)), lo, hi);
  seen_by(s, t, t.at + row_of.token(min(q0, rows - 1)), lo0, hi0);
  seen_by(s, t, t.at + row_of.token(min(q0 + 31, rows - 1)), lo1, hi1);
  seen_by(s, t, t.at, lot, none);
  seen_by(s, t, t.at + t.rows - 1, none, hit);

  f32x16 acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = f32x16{};

  const T* kb = k + (int64_t)t.k_begin * k_token + g * k_head;
  const T* vb = v + (int64_t)t.k_begin * v_token + g * v_head;
  const Walk<SINKS> keys(s, lot, hit);
  auto load = [&](int i0, char* sk, char* sv) {
    if (keys.gap(i0)) {
      load_rows_apart<DP, ROWS, BLOCKS * PARTS>(sk, kb, i0, keys.sinks, lot, t.nk, (uint32_t)(2 * k_token),
                                                2 * k_token, s.dim, wave, lane);
      load_rows_apart<DP, ROWS, BLOCKS * PARTS>(sv, vb, i0, keys.sinks, lot, t.nk, (uint32_t)(2 * v_token),
                                                2 * v_token, s.dim, wave, lane);
      return;
    }
    const int j0 = keys.at(i0), n = min(ROWS, t.nk - j0);
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
  // whether none of the wave's rows sees any of n keys from place i0 on
  auto unseen = [&](int i0, int n) {
    const int j0 = keys.at(i0);
    return j0 >= hi1 || (j0 + n <= lo0 && !(SINKS && i0 < s.sinks));
  };
  auto hide = [&](int i0, int u, f32x16& x) {
    const int j0 = keys.at(i0);
    if (j0 + kRows > hi0 || j0 < lo1) {
      if constexpr (SINKS) {
        seen_or_none<true>((bits_from(lo - j0 - 32 * u) | ~bits_from(s.sinks - i0 - 32 * u)) &
                               ~bits_from(hi - j0 - 32 * u), half, x);
      } else {
        const int first = lo - j0 - 4 * half, last = hi - j0 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = 32 * u + 8 * (r / 4) + r % 4;
          x[r] = j >= first && j < last ? x[r] : 0.0f;
        }
      }
    }
  };
  auto walk = [&](auto&& step) {
    auto wave_step = [&](int i0, const char* sk, const char* sv) {
      i0 += part * kRows;
      if (!active || unseen(i0, kRows)) return;
      step(i0, (const lds_char*)sk + part * L::BYTES, (const lds_char*)sv + part * L::BYTES);
    };
    int i0 = keys.begin;
    if (i0 < keys.end) load(i0, s_k0, s_v0);
    __syncthreads();
    while (i0 < keys.end) {
      if (i0 + ROWS < keys.end) load(i0 + ROWS, s_k1, s_v1);
      wave_step(i0, s_k0, s_v0);
      __syncthreads();
      i0 += ROWS;
      if (i0 >= keys.end) break;
      if (i0 + ROWS < keys.end) load(i0 + ROWS, s_k0, s_v0);
      wave_step(i0, s_k1, s_v1);
      __syncthreads();
      i0 += ROWS;
    }
  };

  // An output of few keys is large, and so is what its rounding does to delta = grad_out . out: there
  // delta is made anew, as the sum of the weights times dP.
  int first_lo, first_hi;
  seen_by(s, t, t.at, first_lo, first_hi);
  const int seen = SINKS ? first_hi - first_lo + min(s.sinks, first_lo) : hit - lot;
  if (SINKS ? delta_anew(s.dim, seen) : seen <= kFewKeys) {
    delta = 0;
    walk([&](int i0, const lds_char* sk, const lds_char* sv) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x16 x, y;
        products(sk, sv, u, x, y);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], c, -base)) * y[r];
        hide(i0, u, x);
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
  if (part == 0 && half == 0 && mine < rows) {
    stats[a * q_tokens + row] = (Lift<T>::up - base) / c;
    stats[(s.heads + a) * q_tokens + row] = -delta;
  }

  constexpr bool RAISED = std::is_same<T, f16>::value;
  int n = RAISED ? kRaise : 0;
  base -= n;
  walk([&](int i0, const lds_char* sk, const lds_char* sv) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (unseen(i0 + 32 * u, 32)) continue;
      f32x16 x, y;
      products(sk, sv, u, x, y);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], c, -base)) * (y[r] - delta);
      hide(i0, u, x);
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
  if (mine < rows)
    store_rows<T, NT>(dq + row * dq_token + a * dq_head, acc, s.scale, s.dim, half);
}

// Where first keys stay visible to all later queries, their tiles would have many times the others' work
// under a window (four of 4096 under 512: eight times): with SINKS those of sequences with more than ``chunk``
// queries go to jobs of ``chunk`` queries each, whose sums another launch adds in their order.  Slot first_slot + i
// is the job of the queries [i * chunk, (i + 1) * chunk) of sequence b: no two are the same, also where the first
// slot is 2 * q_begin / chunk (``twice``), as x > 1 chunks are at most 2 * x slots, whole numbers of both; there
// are at most q_tokens / chunk + batch, and so 2 * (q_tokens / chunk + 1).  A slot holds, for each share of the
// heads, key head and first key, the values' sums and then the keys'.
struct Jobs {
  const Tile* sequences;  // of each its q_begin, nq, k_begin, nk
  float* sums;
  int batch, chunk, slots, tiles, blocks;  // tiles of first keys a sequence; workgroups of all jobs
  bool twice;
  __device__ int first_slot(int q_begin, int b) const {
    return (int)(((uint32_t)q_begin << (twice ? 1 : 0)) / (uint32_t)chunk) + (twice ? 0 : b);
  }
  // Whether a sequence's first keys go to jobs.  Those that need no sums do too where they have a slot: they are more
  // work than most tiles of the list, and so start before them (6 sequences up to 1501, 4 key heads of 96: 24.0 /
  // 23.9 us).
  __device__ bool takes(const Tile& t) const { return t.nq > chunk || (slots > 0 && !twice && t.nq > 0); }
  // The last sequence whose slots start at or before this one, the same in a wave: 64 of those it may be at a look.
  __device__ int sequence_of(int slot) const {
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int n = batch; n > 1;) {  // it is one of n from b on
      const int step = (n + kWave - 1) / kWave, of = b + min(lane * step, n - 1);
      const bool in = lane * step < n && first_slot(sequences[of].q_begin, of) <= slot;
      const int count = max(__popcll(__ballot(in)), 1);  // b itself starts no later
      b += (count - 1) * step;
      n = min(step, n - (count - 1) * step);
    }
    return __builtin_amdgcn_readfirstlane(b);
  }
};

template <int ROWS>
__device__ __forceinline__ float* job_sums(const Jobs& jobs, const Shape& s, int split, int slot, int share,
                                           int g, int row) {
  return jobs.sums + ((((int64_t)slot * split + share) * s.kv_heads + g) * (2 * jobs.tiles * ROWS) + row) * s.dim;
}

// The tile of first keys, key head, share and queries [from, to) of job n; false if there are none.
template <int ROWS>
__device__ __forceinline__ bool job_of(const Jobs& jobs, const Shape& s, int split, int n, Tile& t, int& g,
                                       int& slot, int& from, int& to) {
  const int per = s.kv_heads * split;
  g = n % per;
  n /= per;
  slot = n % jobs.slots;
  const int at = n / jobs.slots * ROWS;
  if (at / ROWS >= jobs.tiles) return false;
  const int b = jobs.sequence_of(slot);
  t = jobs.sequences[b];
  const int64_t begin = (int64_t)(slot - jobs.first_slot(t.q_begin, b)) * jobs.chunk;
  t.first = t.k_begin + at;
  t.at = at;
  t.rows = min(ROWS, t.nk - at);
  if (begin >= t.nq || at >= min(t.nk, s.sinks) || !jobs.takes(t)) return false;
  from = (int)begin;
  to = (int)min(begin + jobs.chunk, (int64_t)t.nq);
  if (t.nq <= jobs.chunk) slot = -1;  // nothing to add: as a tile of the list
  return true;
}

// Gradients of the keys and values, BLOCKS * 32 keys a workgroup, over the heads of the group and their
// queries.  S and dP are [queries, keys], so P and dS are the operands of dV^T = grad_out^T P and
// dK^T = Q^T dS where they lie.  The products start from a row's -lse / scale and -delta, so that they
// give S - lse and dP - delta.  PARTS waves share 32 keys, one to every PARTS-th 32 queries;
// their sums are joined through LDS at the end, in their order.  S and dP are made a second time here:
// sums of dQ over the workgroups of a row's keys would cost atomics whose order changes results, or
// 32-bit copies in memory.  Bound as the forward pass: two sequences of 4096, 32 heads of 128 over 8,
// causal, 5.5e11 operations in 577 us, 0.96 PFLOP/s.
template <typename T, int DP, int BLOCKS, int PARTS, bool SINKS>
__global__ __launch_bounds__(64 * BLOCKS * PARTS, 2) void attention_grad_kv_kernel(
    Shape s, const Tile* __restrict__ tiles, int n_tiles, const T* __restrict__ q, int64_t q_token,
    int64_t q_head, const T* __restrict__ k, int64_t k_token, int64_t k_head,
    const T* __restrict__ v, int64_t v_token, int64_t v_head, const T* __restrict__ go,
    int64_t go_token, int64_t go_head, const float* __restrict__ stats, int64_t q_tokens,
    T* __restrict__ dk, int64_t dk_token, int64_t dk_head, T* __restrict__ dv, int64_t dv_token,
    int64_t dv_head, int split, float* __restrict__ sums, int64_t k_tokens, Jobs jobs) {
  typedef Lay<DP> L;
  constexpr int NS = DP / 16, NT = DP / 32;
  constexpr int ROWS = 32 * PARTS, BYTES = ROWS * L::PITCH;
  __shared__ __attribute__((aligned(1024))) char s_q0[BYTES], s_g0[BYTES], s_q1[BYTES], s_g1[BYTES];
  __shared__ __attribute__((aligned(256))) float s_x0[ROWS], s_y0[ROWS], s_x1[ROWS], s_y1[ROWS];
  int tile, g, slot = -1, from = 0, to = 0x7fffffff;
  Tile t;
  if (SINKS && (int)blockIdx.x < jobs.blocks) {
    if (!job_of<32 * BLOCKS>(jobs, s, split, blockIdx.x, t, g, slot, from, to)) return;
  } else {
    tile_and_head(blockIdx.x - (SINKS ? jobs.blocks : 0), n_tiles, s.kv_heads * split, tile, g);
    t = tiles[tile];
    if (SINKS && t.at < s.sinks && jobs.takes(t)) return;
  }
  const int share = g % split;  // of the group's heads
  g /= split;
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
  auto sees = [&](int at, int& lo, int& hi) {  // which queries of the job see the sequence's key ``at``
    seen_of(s, t, at, lo, hi);
    if constexpr (SINKS) {
      if (at < s.sinks) hi = t.nq;
      lo = max(lo, from);
      hi = min(hi, to);
    }
  };
  {
    const int first = t.at + min(k0, t.rows - 1), last = t.at + min(k0 + 31, t.rows - 1);
    sees(first, lo0, hi0);
    sees(last, lo1, hi1);
    sees(t.at, lot, none);
    sees(t.at + t.rows - 1, none, hit);
    if constexpr (SINKS) {  // first keys, which all queries see, and others after them
      hit = max(hit, t.at < s.sinks ? min(t.nq, to) : 0);
      hi1 = max(hi0, hi1);
      sees(min(max(first, s.sinks), last), none, hi0);
    }
  }

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
      sees(t.at + min(key, t.rows - 1), lo, hi);
      if constexpr (SINKS) {
        const uint32_t bits = bits_from(lo - i1) & ~bits_from(hi - i1);
        seen_or_none<true>(bits, half, x);
        seen_or_none<true>(bits, half, y);
      } else {
        const int first = lo - i1 - 4 * half, last = hi - i1 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int i = 8 * (r / 4) + r % 4;
          const bool in = i >= first && i < last;
          x[r] = in ? x[r] : 0.0f;
          y[r] = in ? y[r] : 0.0f;
        }
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
  // Under a window with first keys the rows are few enough that a head after the other lets the tiles share
  // them: two of 8192, 32 heads of 128 over 8, window 1024, forward and backward 1491 us with the heads
  // in turn, 1374 so; four of 4096, 16 heads of 64 over 4, window 512 243 and 231 (416 and 149 MB past the L2s).
  auto next = [&] {
    if constexpr (SINKS) {
      if ((i1 -= ROWS) < lot) ++a1, i1 = lot + (steps - 1) * ROWS;
    } else {
      if (++a1 == a0 + group) a1 = a0, i1 -= ROWS;
    }
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
    if (SINKS && slot >= 0) {
      float* to_v = job_sums<32 * BLOCKS>(jobs, s, split, slot, share, g, t.at + mine);
      store_rows<float, NT>(to_v, av, Lift<T>::down, s.dim, half);
      store_rows<float, NT>(to_v + (int64_t)jobs.tiles * 32 * BLOCKS * s.dim, ak, s.scale, s.dim, half);
      return;
    }
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

// The same where first keys have jobs: theirs as the sums of these, chunk by chunk and in each the shares of the
// heads, by workgroups of their own, [0, of_jobs): a thread to four elements, a workgroup's of one sequence
// and key head.  The others add the shares of all other keys, whose sequence each thread looks up: one launch of
// 5.7 us for 6 sequences up to 1501, 4 key heads of 96, where two took 4.3 and 4.2 and the gap between them.
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void attention_grad_sinks_sum_kernel(
    Shape s, int split, Jobs jobs, int of_jobs, const float* __restrict__ sums, int64_t k_tokens,
    T* __restrict__ dk, int64_t dk_token, int64_t dk_head, T* __restrict__ dv, int64_t dv_token,
    int64_t dv_head) {
  if ((int)blockIdx.x >= of_jobs) {
    const int64_t each = (int64_t)s.kv_heads * k_tokens * s.dim;
    const int64_t i = ((int64_t)(blockIdx.x - of_jobs) * 256 + threadIdx.x) * 4;
    if (i >= 2 * each) return;
    const bool keys = i >= each;
    const int64_t at = keys ? i - each : i;
    const int64_t row = at / s.dim, g = row / k_tokens, t = row - g * k_tokens;
    int b = 0;  // the last sequence that starts at or before t
    for (int end = jobs.batch; end - b > 1;) {
      const int mid = (b + end) / 2;
      if (jobs.sequences[mid].k_begin <= t) b = mid;
      else end = mid;
    }
    const Tile q = jobs.sequences[b];
    if ((t - q.k_begin) / ROWS * ROWS < s.sinks && q.nq > jobs.chunk) return;
    const float* from = sums + (keys ? split * each : 0) + at;
    f32x4 y = *reinterpret_cast<const f32x4*>(from);
    for (int p = 1; p < split; ++p) y += *reinterpret_cast<const f32x4*>(from + p * each);
    T* to = (keys ? dk + t * dk_token + g * dk_head : dv + t * dv_token + g * dv_head) + at % s.dim;
    *reinterpret_cast<V4<T>*>(to) = __builtin_convertvector(y, V4<T>);
    return;
  }
  const int quads = s.dim / 4, per = 2 * jobs.tiles * ROWS * quads, blocks = (per + 255) / 256;
  const int i = (blockIdx.x % blocks) * 256 + threadIdx.x;
  const int g = blockIdx.x / blocks % s.kv_heads, of_all = blockIdx.x / blocks / s.kv_heads;
  const int b = jobs.twice ? jobs.sequence_of(of_all) : of_all;  // of few slots beside sequences, or of sequences
  const Tile t = jobs.sequences[b];
  const int first = jobs.first_slot(t.q_begin, b);
  if (i >= per || (jobs.twice && first != of_all)) return;
  const int d = i % quads * 4, of = i / quads;
  const bool keys = of >= jobs.tiles * ROWS;
  const int row = keys ? of - jobs.tiles * ROWS : of;
  // the rows of the tiles that have a first key
  if (t.nq <= jobs.chunk || row >= t.nk || row / ROWS * ROWS >= s.sinks) return;
  int lot, hit;
  seen_of(s, t, row / ROWS * ROWS, lot, hit);
  f32x4 y{};
  const int from = (uint32_t)lot / (uint32_t)jobs.chunk, last = (uint32_t)(t.nq - 1) / (uint32_t)jobs.chunk;
  if (lot < t.nq)
    for (int c = from; c <= last; ++c)
      for (int p = 0; p < split; ++p)
        y += *reinterpret_cast<const f32x4*>(job_sums<ROWS>(jobs, s, split, first + c, p, g, of) + d);
  const int64_t at = t.k_begin + row;
  T* to = keys ? dk + at * dk_token + g * dk_head : dv + at * dv_token + g * dv_head;
  *reinterpret_cast<V4<T>*>(to + d) = __builtin_convertvector(y, V4<T>);
}

template <typename T>
const T* in(const void* p) { return static_cast<const T*>(p); }

// Under a window with first keys a tile of queries is of several heads of a group, the largest divisor of its
// size up to 32: its rows see nearly the same keys, where as many queries of one head see as many more.  With
// tiles of one head (and steps of their own for the first keys) and so, us: two of 8192, window 1024, 16 heads of
// 128 over 4 170 / 166; forward and backward: four of 4096, window 512, 16 heads of 64 over 4 244 / 231; 6 ragged
// ones up to 1501, window 200, 70 first keys, 12 heads of 96 over 4 77 / 67.
int heads_beside(int64_t group) {
  int width = 1;
  for (int i = 2; i <= 32; ++i)
    if (group % i == 0) width = i;
  return width;
}

// A call's arguments, with its first keys and, for a backward pass, the sequences.
struct Call : fsp_attention_packed_args {
  int64_t sinks = 0, batch = 0;
  const int32_t* sequences = nullptr;
  int width() const { return sinks ? heads_beside(heads / kv_heads) : 1; }
  int64_t query_tiles() const { return n_q_tiles * heads / width(); }  // workgroups
};

Shape shape_of(const Call& a) {
  return {(int)a.heads, (int)a.kv_heads, (int)a.dim, a.causal != 0, (int)a.window, (float)a.scale,
          (int)a.sinks, a.width()};
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

int64_t seen_at_most(const Call& a, int64_t longest) {
  return a.window && a.window + a.sinks < longest ? a.window + a.sinks : longest;
}

bool share_queries(const Call& a, int64_t fill) {
  const int64_t n = a.query_tiles();
  return seen_at_most(a, a.k_longest) >= 512 &&
         (n <= fill || (n <= 2 * kCus && a.causal && !a.window && a.k_longest >= 2048));
}

// Tiles of half the queries, with two waves to 32 of them, where whole tiles would leave CUs without any
// and there is more than one step of keys.  Measured without and with them, us (tiles times heads):
// forward, dim 128: one sequence of 512, 16 heads (64) 14.4 / 12.6, of 2048, 4 heads (64) 31.9 / 30.1, of
// 4000, 8 heads (256) 58 / 64; four of 64, 4 heads (16) 6.0 / 7.9; dim 64, whose workgroups go two
// to a CU: 2048, 8 heads (128) 22.4 / 18.5, 4000 (256) 39.6 / 35.4.  Gradient of the queries, dim 128:
// 512 (64) 20.4 / 15.9, 2048 (64) 44.8 / 38.6, 4000 (256) 82 / 86; dim 64: 2048 (128) 28.9 / 25.3.
bool halve_tiles(const Call& a, int64_t most) {
  return a.query_tiles() <= most && seen_at_most(a, a.k_longest) > kRows;
}

bool share_keys(const Call& a, int split) {
  const int64_t n = a.n_k_tiles * a.kv_heads * split;
  return (n <= kCus && a.heads / a.kv_heads / split * seen_at_most(a, a.q_longest) >= 768) ||
         (n <= 2 * kCus && a.causal && !a.window && a.q_longest >= 4096);
}

// Tiles of half the keys, with four waves to them, where whole ones leave CUs without any.  Measured
// without and with them, us, the whole backward pass (tiles times heads): dim 128: two of 256, 4 heads (32)
// 29.7 / 30.6, one of 500, 16 heads over 4 (128) 40.7 / 38.1, 4000, 2 heads (126) 136 / 127, 2000, 8
// heads (256) 79 / 84; dim 64: 65 tokens 15.8 / 15.4, two of 256 (32) 19.9 / 18.9, 2000, 8 heads (256)
// 49.2 / 46.8.
bool halve_keys(const Call& a, int split) {
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

template <typename T, int DP, int BLOCKS, int PARTS, bool SINKS>
int launch_forward(const Call& a, hipStream_t st) {
  const int32_t* tiles = BLOCKS == 2 ? a.q_halves : a.q_tiles;
  const int64_t n = BLOCKS == 2 ? a.n_q_halves : a.n_q_tiles;
  hipLaunchKernelGGL((attention_packed_kernel<T, DP, BLOCKS, PARTS, SINKS>),
                     dim3((unsigned)(n * a.heads / a.width())), dim3(64 * BLOCKS * PARTS), 0, st, shape_of(a),
                     reinterpret_cast<const Tile*>(tiles), (int)n, in<T>(a.q),
                     a.q_token, a.q_head, in<T>(a.k), a.k_token, a.k_head, in<T>(a.v), a.v_token,
                     a.v_head, static_cast<T*>(a.out), a.out_token, a.out_head, a.lse);
  return check_hip(hipGetLastError(), "attention_packed_kernel launch");
}

template <typename T, int DP, bool SINKS>
int launch_forward_parts(const Call& a, hipStream_t st) {
  if (halve_tiles(a, DP <= 64 ? kCus : kCus / 2)) return launch_forward<T, DP, 2, 2, SINKS>(a, st);
  return share_queries(a, DP <= 64 ? 4 * kCus : kCus) ? launch_forward<T, DP, 4, 2, SINKS>(a, st)
                                                      : launch_forward<T, DP, 4, 1, SINKS>(a, st);
}

template <typename T, bool SINKS>
int launch_forward_dim(const Call& a, hipStream_t st) {
  if (a.dim <= 64) return launch_forward_parts<T, 64, SINKS>(a, st);
  if (a.dim <= 96) return launch_forward_parts<T, 96, SINKS>(a, st);
  return launch_forward_parts<T, 128, SINKS>(a, st);
}

template <typename T, int DP, int BLOCKS, int PARTS, bool SINKS>
int launch_grad_q(const Call& a, hipStream_t st) {
  const int32_t* tiles = BLOCKS == 2 ? a.q_halves : a.q_tiles;
  const int64_t n = BLOCKS == 2 ? a.n_q_halves : a.n_q_tiles;
  hipLaunchKernelGGL((attention_grad_q_kernel<T, DP, BLOCKS, PARTS, SINKS>),
                     dim3((unsigned)(n * a.heads / a.width())), dim3(64 * BLOCKS * PARTS), 0, st, shape_of(a),
                     reinterpret_cast<const Tile*>(tiles), (int)n, in<T>(a.q),
                     a.q_token, a.q_head, in<T>(a.k), a.k_token, a.k_head, in<T>(a.v), a.v_token,
                     a.v_head, in<T>(a.out), a.out_token, a.out_head, a.lse, in<T>(a.grad_out),
                     a.grad_out_token, a.grad_out_head, static_cast<T*>(a.grad_q), a.grad_q_token,
                     a.grad_q_head, static_cast<float*>(a.workspace), a.q_tokens);
  return check_hip(hipGetLastError(), "attention_grad_q_kernel launch");
}

// Queries of a job of the first keys: about what the other tiles have under their window, and no fewer than there
// are first keys, whose tiles are workgroups enough then and whose sums would take more room than the keys.
int64_t chunk_of(int64_t window, int64_t firsts) {
  const int64_t least = window > firsts ? window : firsts;
  return least <= 512 ? 512 : least < kAttnTokensCap ? (least + 127) / 128 * 128 : kAttnTokensCap;
}

// By twice the chunks where that is less than half as many, as most sequences have no job: 20000 of 64 tokens beside
// one of 1000, 8 key heads of 128, jobs of 512 queries take 2.6 GB instead of 11.8.  Otherwise those without a job of
// their own have a slot too, to start early (takes): 50 of 200 beside one of 4000, the backward pass is 1 % longer by
// twice the chunks.
bool slots_twice(int64_t q_tokens, int64_t batch, int64_t chunk) {
  return 4 * (q_tokens / chunk + 1) < q_tokens / chunk + batch;
}

int64_t job_slots(int64_t q_tokens, int64_t batch, int64_t chunk) {
  return slots_twice(q_tokens, batch, chunk) ? 2 * (q_tokens / chunk + 1) : q_tokens / chunk + batch;
}

// Elements of one share's sums over all keys, and of the jobs' of the first keys in tiles of ``rows``.
int64_t share_floats(int split, int64_t kv_heads, int64_t k_tokens, int64_t dim) {
  return split > 1 ? 2 * split * kv_heads * k_tokens * dim : 0;
}

int64_t first_keys(int64_t sinks, int64_t k_longest) { return sinks < k_longest ? sinks : k_longest; }

// Whether any sequence has more queries than one job.
bool has_jobs(const Call& a) {
  return a.sinks && a.q_longest > chunk_of(a.window, first_keys(a.sinks, a.k_longest));
}

Jobs jobs_of(const Call& a, int split, int rows, float* sums) {
  Jobs j;
  const int64_t firsts = first_keys(a.sinks, a.k_longest), chunk = chunk_of(a.window, firsts);
  j.sequences = reinterpret_cast<const Tile*>(a.sequences);
  j.sums = sums + share_floats(split, a.kv_heads, a.k_tokens, a.dim);
  j.batch = (int)a.batch;
  j.chunk = (int)chunk;
  j.slots = has_jobs(a) ? (int)job_slots(a.q_tokens, a.batch, chunk) : 0;
  j.twice = slots_twice(a.q_tokens, a.batch, chunk);
  j.tiles = (int)((firsts + rows - 1) / rows);
  j.blocks = (int)((j.tiles * (int64_t)j.slots * a.kv_heads * split + 7) / 8 * 8);
  return j;
}

template <typename T, int DP, int BLOCKS, int PARTS, bool SINKS>
int launch_grad_kv(const Call& a, int split, hipStream_t st) {
  const int32_t* tiles = BLOCKS == 1 ? a.k_halves : a.k_tiles;
  const int64_t n = BLOCKS == 1 ? a.n_k_halves : a.n_k_tiles;
  float* stats = static_cast<float*>(a.workspace);
  float* sums = stats + ((2 * a.heads * a.q_tokens + 3) & ~int64_t(3));
  const Jobs jobs = SINKS ? jobs_of(a, split, 32 * BLOCKS, sums) : Jobs{};
  hipLaunchKernelGGL((attention_grad_kv_kernel<T, DP, BLOCKS, PARTS, SINKS>),
                     dim3((unsigned)(jobs.blocks + n * a.kv_heads * split)), dim3(64 * BLOCKS * PARTS), 0, st,
                     shape_of(a), reinterpret_cast<const Tile*>(tiles), (int)n,
                     in<T>(a.q), a.q_token, a.q_head, in<T>(a.k), a.k_token, a.k_head, in<T>(a.v),
                     a.v_token, a.v_head, in<T>(a.grad_out), a.grad_out_token, a.grad_out_head,
                     stats, a.q_tokens, static_cast<T*>(a.grad_k), a.grad_k_token, a.grad_k_head,
                     static_cast<T*>(a.grad_v), a.grad_v_token, a.grad_v_head, split, sums,
                     a.k_tokens, jobs);
  if (int rc = check_hip(hipGetLastError(), "attention_grad_kv_kernel launch")) return rc;
  const int64_t quads = split > 1 ? a.kv_heads * a.k_tokens * a.dim / 2 : 0;
  if (SINKS && jobs.slots > 0) {
    const int64_t of_jobs = (2 * jobs.tiles * 32 * BLOCKS * (a.dim / 4) + 255) / 256 * a.kv_heads *
                            (jobs.twice ? jobs.slots : a.batch);
    hipLaunchKernelGGL((attention_grad_sinks_sum_kernel<T, 32 * BLOCKS>),
                       dim3((unsigned)(of_jobs + (quads + 255) / 256)), dim3(256), 0, st, shape_of(a), split,
                       jobs, (int)of_jobs, sums, a.k_tokens, static_cast<T*>(a.grad_k), a.grad_k_token,
                       a.grad_k_head, static_cast<T*>(a.grad_v), a.grad_v_token, a.grad_v_head);
    return check_hip(hipGetLastError(), "attention_grad_sinks_sum_kernel launch");
  }
  if (split == 1) return FSP_OK;
  hipLaunchKernelGGL((attention_grad_kv_sum_kernel<T>), dim3((unsigned)((quads + 255) / 256)),
                     dim3(256), 0, st, shape_of(a), split, sums, a.k_tokens,
                     static_cast<T*>(a.grad_k), a.grad_k_token, a.grad_k_head,
                     static_cast<T*>(a.grad_v), a.grad_v_token, a.grad_v_head);
  return check_hip(hipGetLastError(), "attention_grad_kv_sum_kernel launch");
}

template <typename T, int DP, bool SINKS>
int launch_backward(const Call& a, hipStream_t st) {
  if (a.n_q_tiles > 0) {
    const int rc = halve_tiles(a, kCus / 2) ? launch_grad_q<T, DP, 2, 2, SINKS>(a, st)
                   : share_queries(a, kCus) ? launch_grad_q<T, DP, 4, 2, SINKS>(a, st)
                                            : launch_grad_q<T, DP, 4, 1, SINKS>(a, st);
    if (rc) return rc;
  }
  if (a.n_k_tiles > 0) {
    const int split = split_heads(a.n_k_tiles, a.heads, a.kv_heads, a.causal && !a.window);
    if (halve_keys(a, split)) return launch_grad_kv<T, DP, 1, 4, SINKS>(a, split, st);
    return share_keys(a, split) ? launch_grad_kv<T, DP, 2, 4, SINKS>(a, split, st)
                                : launch_grad_kv<T, DP, 2, 2, SINKS>(a, split, st);
  }
  return FSP_OK;
}

template <typename T, bool SINKS>
int launch_backward_dim(const Call& a, hipStream_t st) {
  if (a.dim <= 64) return launch_backward<T, 64, SINKS>(a, st);
  if (a.dim <= 96) return launch_backward<T, 96, SINKS>(a, st);
  return launch_backward<T, 128, SINKS>(a, st);
}

int check_packed(const Call& a, const std::string& who) {
  if (!attn_dtype(a.dtype)) return set_error(FSP_ENOTSUP, who + ": dtype");
  if (!attn_dim(a.dim)) return set_error(FSP_ENOTSUP, who + ": dim");
  if (a.kv_heads < 1 || a.heads < 1 || a.heads % a.kv_heads || a.heads > 0xffff)
    return set_error(FSP_EINVAL, who + ": heads must be a multiple of kv_heads");
  if (a.q_tokens < 0 || a.k_tokens < 0 || a.n_q_tiles < 0 || a.n_k_tiles < 0 ||
      a.n_q_halves < 0 || a.n_k_halves < 0 || a.window < 0 || a.q_longest < 0 || a.k_longest < 0 ||
      a.q_tokens > kAttnTokensCap || a.k_tokens > kAttnTokensCap || a.window > 0x7fffffffLL ||
      a.n_q_tiles > kMaxBlocks / (a.heads / a.width()) || a.n_q_halves > kMaxBlocks / (a.heads / a.width()) ||
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
  if (a.sinks < 0 || a.sinks > kAttnTokensCap || (a.sinks && !a.window))
    return set_error(FSP_EINVAL, who + ": sinks need a window");
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
  return sizeof(float) * (stats + share_floats(split, kv_heads, k_tokens, dim));
}

extern "C" int64_t fsp_attention_packed_sinks_workspace(int64_t n_k_tiles, int64_t heads,
                                                        int64_t kv_heads, int64_t dim, int64_t q_tokens,
                                                        int64_t k_tokens, int64_t k_longest,
                                                        int64_t batch, int64_t window, int64_t sinks) {
  const int64_t rest = fsp_attention_packed_workspace(n_k_tiles, heads, kv_heads, dim, q_tokens, k_tokens, 0);
  if (sinks <= 0 || batch < 0 || window < 1 || k_longest < 0 || n_k_tiles < 0 || heads < 1 || kv_heads < 1 ||
      dim < 0 || q_tokens < 0 || k_tokens < 0)
    return rest;
  const int64_t firsts = first_keys(sinks, k_longest), rows = (firsts + kRows - 1) / kRows * kRows;
  return rest + sizeof(float) * 2 * job_slots(q_tokens, batch, chunk_of(window, firsts)) *
                    split_heads(n_k_tiles, heads, kv_heads, false) * kv_heads * rows * dim;
}

extern "C" int64_t fsp_attention_packed_sinks_chunk(int64_t window, int64_t sinks, int64_t k_longest) {
  return window < 1 || sinks < 1 || k_longest < 0 ? 0 : chunk_of(window, first_keys(sinks, k_longest));
}

extern "C" int64_t fsp_attention_packed_tile(int which) {
  return which == 0 ? kTile : which == 1 ? kTile / 2 : which == 2 ? kRows : kRows / 2;
}

namespace {

int run_forward(const Call& a, const std::string& who, void* stream) {
  if (int rc = check_packed(a, who)) return rc;
  if (a.n_q_tiles == 0) return FSP_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.sinks)
    return a.dtype == FSP_BF16 ? launch_forward_dim<bf16, true>(a, st) : launch_forward_dim<f16, true>(a, st);
  return a.dtype == FSP_BF16 ? launch_forward_dim<bf16, false>(a, st) : launch_forward_dim<f16, false>(a, st);
}

int run_backward(const Call& a, const std::string& who, void* stream) {
  if (int rc = check_packed(a, who)) return rc;
  if (a.sinks && a.n_k_tiles > 0) {
    if (a.batch < 1 || !a.sequences) return set_error(FSP_EINVAL, who + ": sequences");
    // tiles of 32 keys, the most jobs
    const int64_t firsts = first_keys(a.sinks, a.k_longest), tiles = (firsts + kRows / 2 - 1) / (kRows / 2);
    const int64_t all = kMaxBlocks / a.heads - a.n_k_halves - 8;
    const int64_t batch = has_jobs(a) ? a.batch : 1, chunk = chunk_of(a.window, firsts);
    const int64_t slots = job_slots(a.q_tokens, batch, chunk);
    // the vectors of a sequence's sums, which are counted in 32 bits, and the workgroups that add or look at them;
    // those that add the shares of other keys are few, as shares are made where tiles are
    const int64_t vectors = 2 * ((firsts + kRows - 1) / kRows * kRows) * (a.dim / 4);
    const int64_t sums = slots_twice(a.q_tokens, batch, chunk) ? slots : batch;
    if (a.batch > 0x7fffffffLL || (tiles > 0 && slots > all / tiles) || vectors > (1 << 30) ||
        sums > (kMaxBlocks - (1 << 16)) / a.kv_heads / (vectors / 256 + 1))
      return set_error(FSP_EINVAL, who + ": sinks of so many sequences");
  }
  // without queries, and with one share of the heads, there is nothing to keep
  const bool work = a.n_k_tiles > 0 && (has_jobs(a) || fsp_attention_packed_workspace(
      a.n_k_tiles, a.heads, a.kv_heads, a.dim, a.q_tokens, a.k_tokens, a.causal && !a.window) > 0);
  if ((a.n_q_tiles > 0 && (!a.grad_out || !a.grad_q || !a.workspace)) ||
      (a.n_k_tiles > 0 && (!a.grad_k || !a.grad_v)) || (work && !a.workspace))
    return set_error(FSP_EINVAL, who + ": null pointer");
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return set_error(FSP_EINVAL, who + ": workspace must be 16-byte aligned");
  if (!aligned16(a.grad_out, a.grad_out_token, a.grad_out_head) ||
      !aligned16(a.grad_q, a.grad_q_token, a.grad_q_head) ||
      !aligned16(a.grad_k, a.grad_k_token, a.grad_k_head) ||
      !aligned16(a.grad_v, a.grad_v_token, a.grad_v_head))
    return set_error(FSP_EINVAL, who + ": rows must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a.sinks)
    return a.dtype == FSP_BF16 ? launch_backward_dim<bf16, true>(a, st) : launch_backward_dim<f16, true>(a, st);
  return a.dtype == FSP_BF16 ? launch_backward_dim<bf16, false>(a, st) : launch_backward_dim<f16, false>(a, st);
}

}  // namespace

extern "C" int fsp_attention_packed(const fsp_attention_packed_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_packed: null arguments");
  return run_forward({*args}, "fsp_attention_packed", stream);
}

extern "C" int fsp_attention_packed_backward(const fsp_attention_packed_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_packed_backward: null arguments");
  return run_backward({*args}, "fsp_attention_packed_backward", stream);
}

extern "C" int64_t fsp_attention_packed_sinks_tile(int which, int64_t group) {
  return group < 1 ? 1 : (which == 0 ? kTile : kTile / 2) / heads_beside(group);
}

extern "C" int fsp_attention_packed_sinks(const fsp_attention_packed_args* args, int64_t sinks,
                                          void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_packed_sinks: null arguments");
  return run_forward({*args, sinks}, "fsp_attention_packed_sinks", stream);
}

extern "C" int fsp_attention_packed_sinks_backward(const fsp_attention_packed_args* args, int64_t sinks,
                                                   const int32_t* sequences, int64_t batch,
                                                   void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_packed_sinks_backward: null arguments");
  return run_backward({*args, sinks, batch, sequences}, "fsp_attention_packed_sinks_backward", stream);
}
