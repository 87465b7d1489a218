// A paged cache of keys and values: appending to it with the rotation of positions, and attention
// of one query per sequence over it.
#include "attn.hpp"

namespace fsp {
namespace {

constexpr int kAppendThreads = 256;

struct Cache {
  const int32_t *indptr, *indices;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  int batch, page_size, dim, kv_heads;
};

// How the first 2 * half elements of a head turn: not at all; by pairs half apart or of neighbours, eight
// elements of a vector against eight others or among themselves; or element by element, where
// half is no whole number of vectors.
enum { kStill, kHalves, kNeighbours, kEach };

// Eight elements from d on of a head that turns by row ``turn`` of the table.
template <typename T, int MODE>
__device__ __forceinline__ V8<T> turned(const T* row, int d, const float* cos, const float* sin,
                                        int half, int interleaved) {
  const V8<T> x = *reinterpret_cast<const V8<T>*>(row + d);
  if (MODE == kStill || d >= 2 * half) return x;
  f32x8 y = __builtin_convertvector(x, f32x8);
  if constexpr (MODE == kHalves) {
    const bool low = d < half;
    const int j = low ? d : d - half;
    const f32x8 z = __builtin_convertvector(
        *reinterpret_cast<const V8<T>*>(row + (low ? d + half : j)), f32x8);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const f32x4 c = *reinterpret_cast<const f32x4*>(cos + j + 4 * u);
      const f32x4 s = *reinterpret_cast<const f32x4*>(sin + j + 4 * u);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[4 * u + e] = y[4 * u + e] * c[e] + (low ? -z[4 * u + e] : z[4 * u + e]) * s[e];
    }
  } else if constexpr (MODE == kNeighbours) {
    const f32x4 c = *reinterpret_cast<const f32x4*>(cos + d / 2);
    const f32x4 s = *reinterpret_cast<const f32x4*>(sin + d / 2);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float u = y[e], v = y[e + 1];
      y[e] = u * c[e / 2] - v * s[e / 2];
      y[e + 1] = u * s[e / 2] + v * c[e / 2];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = d + e;
      if (at < 2 * half) {
        const bool low = interleaved ? !(at & 1) : at < half;
        const int j = interleaved ? at >> 1 : low ? at : at - half;
        const float z = (float)row[interleaved ? at ^ 1 : low ? at + half : j];
        y[e] = y[e] * cos[j] + (low ? -z : z) * sin[j];
      }
    }
  }
  return __builtin_convertvector(y, V8<T>);
}

struct AppendShape {
  int64_t n_tokens, k_token, k_head, v_token, v_head, q_token, q_head, qo_token, qo_head;
  int heads, half, table_rows, interleaved, parts;
};

// A wave to a token, or to one of ``parts`` interleaved parts of its vectors of eight elements, where
// there are few tokens.  Bound by memory for prompts (a read and a write of every element: 24 of up to 2000
// tokens, 16 query and 16 key heads of 64, 111 MB in 20.8 us, 5.3 TB/s, part of it still in the
// last-level cache) and by the chain token -> sequence -> page -> row for single tokens (16 tokens, 32
// query and 8 key heads of 128: 3.8 us).  An element a thread took 48 us for those prompts.
template <typename T, int MODE>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(
    Cache c, AppendShape s, T* __restrict__ k_pages, T* __restrict__ v_pages,
    const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ q,
    T* __restrict__ q_out, const float* __restrict__ cos, const float* __restrict__ sin,
    const int32_t* __restrict__ tokens, const int32_t* __restrict__ lengths) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (kAppendThreads / kWave) +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = unit / s.parts;
  if (t >= s.n_tokens) return;
  int b = (int)t;
  int64_t pos;
  bool mine = true;
  if (tokens) {  // the last sequence that starts at or before t, 64 at a look
    b = -1;
    for (int at = 0; at < c.batch; at += kWave) {
      const int n = __popcll(__ballot(at + lane < c.batch && tokens[min(at + lane, c.batch)] <= t));
      b += n;
      if (n < kWave) break;
    }
    b = __builtin_amdgcn_readfirstlane(max(b, 0));
    const int begin = tokens[b], end = tokens[b + 1];
    mine = begin <= t && t < end;
    pos = (int64_t)lengths[b] - end + t;
  } else {
    pos = (int64_t)lengths[b] - 1;
  }
  const int first = c.indptr[b], last = c.indptr[b + 1];
  const bool ok = mine && pos >= 0 && pos < (int64_t)(last - first) * c.page_size &&
                  (MODE == kStill || pos < s.table_rows);
  int64_t page = 0, slot = 0;
  if (ok) {
    const uint32_t at = (uint32_t)pos / (uint32_t)c.page_size;
    page = c.indices[first + at];
    slot = (uint32_t)pos - at * c.page_size;
    cos += pos * s.half;
    sin += pos * s.half;
  }
  const T nan = (T)__builtin_nanf("");
  const uint32_t per = c.dim / 8, rows = s.heads + 2 * c.kv_heads;
  const T* kr = k + t * s.k_token;
  const T* vr = v + t * s.v_token;
  const T* qr = q + t * s.q_token;
  T* kt = k_pages + page * c.k_page + slot * c.k_slot;
  T* vt = v_pages + page * c.v_page + slot * c.v_slot;
  T* qt = q_out + t * s.qo_token;
#pragma unroll 2
  for (uint32_t i = (uint32_t)(unit % s.parts) * kWave + lane; i < rows * per; i += s.parts * kWave) {
    int h = i / per;
    const int d = 8 * (i - h * per);
    if (h < s.heads) {
      V8<T> x{nan, nan, nan, nan, nan, nan, nan, nan};
      if (ok) x = turned<T, MODE>(qr + h * s.q_head, d, cos, sin, s.half, s.interleaved);
      *reinterpret_cast<V8<T>*>(qt + h * s.qo_head + d) = x;
    } else if (ok) {
      h -= s.heads;
      if (h < c.kv_heads) {
        *reinterpret_cast<V8<T>*>(kt + h * c.k_head + d) =
            turned<T, MODE>(kr + h * s.k_head, d, cos, sin, s.half, s.interleaved);
      } else {
        h -= c.kv_heads;
        *reinterpret_cast<V8<T>*>(vt + h * c.v_head + d) =
            *reinterpret_cast<const V8<T>*>(vr + h * s.v_head + d);
      }
    }
  }
}

// Results that another workgroup, perhaps of another XCD, picks up: stored past this XCD's L2 and read
// past the reader's, so that a wait for the stores (all_stored) is all that has to come between
// them and the word that they are there.  A release and an acquire of everything write back and drop
// an L2 each time instead: 96 sequences of up to 4096 tokens took 59 us with them, 41 us so.
__device__ __forceinline__ void put(float* to, float a, float b) {
  const uint64_t v = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(to), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ f32x2 get(const float* from) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(from), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  return f32x2{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

__device__ __forceinline__ void all_stored() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Attention of one query per sequence.  A workgroup takes a piece of a sequence's tokens for one key
// head and up to 16 of the query heads that share it; its four waves take every fourth 32 keys.
//
// Values go from memory to the matrix instructions' registers with no stop in LDS, keys with a short
// one: with a lane to a key a load would fetch 64 bytes of each of 16 rows, and whole rows are the
// faster to fetch (a bare loop of such loads over 3.2 GB: 64 bytes 540 us, rows 490), so that a wave
// writes the rows to LDS of its own and reads its lanes' keys there.  With S^T = K Q^T lane l has head
// l % 16 and, of 32 keys, the eight 4 * (l / 16) + {0..3, 16..19}: its weights are the operand of
// O^T = V^T P^T as they lie, since the order of the summed keys is free.  For V a lane loads DP / 16
// consecutive elements of those same eight keys, and the operand of one
// product is one element of each: pairs of 16-bit halves, a byte permutation each.  Row m of product
// i is element DP / 16 * m + i of the head, so a lane's results are consecutive.
//
// Where each key lies (its page, its place in it) is found once for the piece and kept in LDS.
constexpr int kHeadTile = 16;
constexpr int kPieceMost = 1024;
// The workgroup that finishes a sequence joins its pieces where they are at most so many and the workgroups
// no more than a few rounds of the chip's (three to a CU): each waits for its stores, which in many rounds
// holds up those that follow.  Else a second launch does.  By a second launch and so, us: 1000 tokens, 16
// heads of 64 11.9 / 8.7 a call, both bound by the host (8.4 / 9.2 in a graph, whose replays zero the
// counts); 96 ragged sequences of up to 4096, 8 heads of 128 (1344 workgroups) 49.5 / 44.6; 200 of 2048, 16
// heads of 64 (6400) 263 / 283; 400 of 1500, 8 heads of 128 (6400) 418 / 408.  Up to 27 pieces 15.7 / 20.7 (2
// of 6760, 8 heads), up to 128 542 / 560.
constexpr int kJoinMost = 8;
constexpr int kJoinBlocks = 8 * 256;

// Tokens [begin, begin + piece) of seq, of the room that its pages give; slot: of the sequence's first
// piece; page: its first place in the page table.
struct Piece {
  int seq, begin, slot, page, room, pad[3];
};

// Workgroups go to the 8 XCDs in turn: a piece's heads, which lie side by side in memory, go to one.
// With a head to an XCD each L2 would see every eighth 256 bytes, a few of its channels.
__device__ __forceinline__ void piece_and_head(int block, int n_pieces, int heads, int& piece, int& head) {
  const int set = block / (8 * heads), in = block - set * 8 * heads;
  const int width = min(8, n_pieces - 8 * set);  // pieces of this set
  piece = 8 * set + in % width;
  head = in / width;
}

struct PagedShape {
  int heads, window, piece, n_pieces;
  float scale;
};

// The next step's keys are asked for once this step's scores are made, its values once this step's
// output is; without conditions (the last step asks for one row that it has had; for all of its own,
// which NT loads may have to fetch anew, 2 sequences of 102400 tokens, 16 heads took 292 us, so 278),
// so that the wait for the values does not wait for the keys asked for after them.  EXACT: the head
// has DP elements.  NT: loads that do not claim a place in the caches.
//
// Bound by memory for long caches: 6 sequences of 131072 tokens, 8 heads of 128, 64 queries, 3.2 GB,
// 532 us, 6.1 TB/s of the 7.0 of a plain read, as for 256 of 4096, 32 queries; 96 ragged ones of up to
// 4096, 200 MB, 44 us, 4.6 TB/s: less than two rounds of workgroups, each with the chain piece -> length
// -> page -> keys before it.  For 1000 tokens that chain, the join and the launch are all of its 7.8 us.
template <typename T, int DP, bool EXACT, bool NT>
__global__ __launch_bounds__(256, 3) void attention_paged_kernel(
    Cache c, PagedShape s, const Piece* __restrict__ pieces, const T* __restrict__ k_pages,
    const T* __restrict__ v_pages, const T* __restrict__ q, int64_t q_token, int64_t q_head,
    T* __restrict__ out, int64_t out_token, int64_t out_head, float* __restrict__ lse,
    const int32_t* __restrict__ lengths, float* part_o, float* part_ml, unsigned* arrived) {
  constexpr int E = DP / 16, NS = DP / 32, W = 4;  // elements of V and steps of K a lane; waves
  typedef T VE __attribute__((ext_vector_type(E)));
  constexpr int CH = DP / 8, KL = DP / 16;  // chunks of 16 bytes in a row; loads of 32 rows of K
  __shared__ int64_t s_k[kPieceMost], s_v[kPieceMost];  // where the keys and values lie
  // each wave's keys; then, its sums
  typedef float Sums[kHeadTile][DP + 4];
  static_assert(sizeof(Sums) >= 64 * DP, "");
  __shared__ __attribute__((aligned(16))) char s_raw[W * sizeof(Sums)];
  __shared__ f32x2 s_ml[W][kHeadTile];
  Sums* s_o = reinterpret_cast<Sums*>(s_raw);
  const int group = s.heads / c.kv_heads, tiles = (group + kHeadTile - 1) / kHeadTile;
  int piece, g, ht;
  piece_and_head(blockIdx.x, s.n_pieces, c.kv_heads * tiles, piece, ht);
  g = ht / tiles;
  ht -= g * tiles;
  const Piece pc = pieces[piece];
  const int b = pc.seq, lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n_heads = min(kHeadTile, group - ht * kHeadTile), head0 = g * group + ht * kHeadTile;
  const int length = lengths[b];
  const bool ok = length >= 0 && length <= pc.room;
  // the query sees tokens [first, last); the sequence's pieces in use, and whether this is one
  const int last = ok ? length : 0, first = s.window && last > s.window ? last - s.window : 0;
  const int p0 = first / s.piece, p1 = max(p0 + 1, (last + s.piece - 1) / s.piece);
  const int mine = pc.begin / s.piece;
  if (mine < p0 || mine >= p1) return;
  const int begin = max(first, pc.begin), n = min(last, pc.begin + s.piece) - begin;

  V8<T> qf[NS];
  {
    const T* qr = q + b * q_token + (head0 + min(col, n_heads - 1)) * q_head;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int d = 32 * i + 8 * quad;
      const V8<T> x = *reinterpret_cast<const V8<T>*>(qr + (d < c.dim ? d : 0));
      qf[i] = scaled_sign<T>(x, s.scale, d < c.dim);
    }
  }
  const float cs = exp2_scale(s.scale);

  // where the keys lie; those past the end stand for the first one, and weigh nothing
  const int padded = (n + 127) & ~127;
  for (int i = threadIdx.x; i < padded; i += 256) {
    const uint32_t j = begin + (i < n ? i : 0);
    const uint32_t at = j / (uint32_t)c.page_size;
    const int64_t page = n > 0 ? c.indices[pc.page + at] : 0, slot = j - at * c.page_size;
    s_k[i] = page * c.k_page + slot * c.k_slot;
    s_v[i] = page * c.v_page + slot * c.v_slot;
  }
  __syncthreads();

  const T* kb = k_pages + g * c.k_head;
  const T* vb = v_pages + g * c.v_head;
  i32x4 kr[KL];
  VE vf[8];
  // load i: rows 64 / CH * i + lane / CH, chunk lane % CH of each; it lies in LDS at chunk ^ row
  const int k_row = lane / CH, k_chunk = lane % CH;
  auto load_k = [&](int j, int most) {
#pragma unroll
    for (int i = 0; i < KL; ++i)
      kr[i] = ld_stream<NT>(reinterpret_cast<const i32x4*>(
          kb + s_k[min(j + 64 / CH * i + k_row, most)] +
          (EXACT || 8 * k_chunk < c.dim ? 8 * k_chunk : 0)));
  };
  char* s_rows = s_raw + wave * sizeof(Sums);
  const int ve = E * col < c.dim ? E * col : 0;
  auto load_v = [&](int j, int most) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      vf[e] = ld_stream<NT>(reinterpret_cast<const VE*>(
          vb + s_v[min(j + 16 * (e / 4) + 4 * quad + e % 4, most)] + ve));
  };

  float top = -INFINITY, sum = 0;
  f32x4 o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = f32x4{};

  int j = 32 * wave;
  if (j < n) load_k(j, kPieceMost), load_v(j, kPieceMost);
  for (; j < n; j += 32 * W) {
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int row = 64 / CH * i + k_row;
      // past the head: zeros, as in q, or an infinity there would show
      *reinterpret_cast<i32x4*>(s_rows + row * 2 * DP + 16 * (k_chunk ^ (row & (CH - 1)))) =
          EXACT ? kr[i] : kr[i] & (8 * k_chunk < c.dim ? -1 : 0);
    }
    f32x4 x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      x[u] = f32x4{};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int row = 16 * u + col;
        x[u] = mfma16(*reinterpret_cast<const V8<T>*>(
                          s_rows + row * 2 * DP + 16 * ((4 * i + quad) ^ (row & (CH - 1)))),
                      qf[i], x[u]);
      }
    }
    const bool more = j + 32 * W < n;
    const int next = more ? j + 32 * W : j, most = more ? kPieceMost : j;
    load_k(next, most);
    const bool partial = j + 32 > n;
    if (partial) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = j + 16 * (e / 4) + 4 * quad + e % 4 < n;
        x[e / 4][e % 4] = in ? x[e / 4][e % 4] : -INFINITY;
        vf[e] = in ? vf[e] : VE{};
      }
    }
    float m = x[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) m = fmaxf(m, x[e / 4][e % 4]);
    if (__any((m - top) * cs > Weights<T>::lag)) {
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      const float now = fmaxf(top, m);
      const float fade = top == -INFINITY ? 0.0f : exp2f((top - now) * cs);
      top = now;
      sum *= fade;
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] *= fade;
    }
    const float base = top == -INFINITY ? 0.0f : top * cs - Weights<T>::up;
    f32x8 p;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = __builtin_amdgcn_exp2f(fmaf(x[e / 4][e % 4], cs, -base));
      sum += p[e];
    }
    const V8<T> pf = __builtin_convertvector(p, V8<T>);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      V8<T> a;
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = vf[e][i];
      o[i] = mfma16(a, pf, o[i]);
    }
    load_v(next, most);
  }

  // join the waves
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  const float ml = top == -INFINITY ? -INFINITY : top * cs;  // of all sums alike, 2^up is left in them
  if (quad == 0) s_ml[wave][col] = f32x2{ml, sum};
#pragma unroll
  for (int i = 0; i < E; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) s_o[wave][col][4 * E * quad + E * r + i] = o[i][r];
  __syncthreads();
  const bool split = p1 - p0 > 1;
  const float nan = __builtin_nanf("");
  for (int i = threadIdx.x; i < n_heads * (DP / 4); i += 256) {
    const int h = i / (DP / 4), d = i % (DP / 4) * 4;
    if (d >= c.dim) continue;
    float most = -INFINITY, total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) most = fmaxf(most, s_ml[w][h].x);
    f32x4 y{};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const f32x2 v = s_ml[w][h];
      const float f = v.x == -INFINITY ? 0.0f : exp2f(v.x - most);
      if (v.y == 0) continue;  // saw nothing: its sums are zeros
      total += f * v.y;
      y += f * *reinterpret_cast<const f32x4*>(&s_o[w][h][d]);
    }
    if (split) {
      const int64_t at = (int64_t)(pc.slot + mine) * s.heads + head0 + h;
      if (arrived) {
        put(part_o + at * c.dim + d, y.x, y.y);
        put(part_o + at * c.dim + d + 2, y.z, y.w);
        if (d == 0) put(part_ml + 2 * at, most, total);
      } else {
        *reinterpret_cast<f32x4*>(part_o + at * c.dim + d) = y;
        if (d == 0) *reinterpret_cast<f32x2*>(part_ml + 2 * at) = f32x2{most, total};
      }
    } else {
      const float f = total == 0 ? 0.0f : 1.0f / total;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = ok ? y[e] * f : nan;
      *reinterpret_cast<V4<T>*>(out + b * out_token + (head0 + h) * out_head + d) =
          __builtin_convertvector(y, V4<T>);
      if (lse && d == 0)
        lse[(int64_t)b * s.heads + head0 + h] =
            !ok ? nan : total == 0 ? -INFINITY : (most + log2f(total * Weights<T>::down)) * kLn2;
    }
  }
  if (!split || !arrived) return;  // without counts, another launch joins them

  // The last workgroup of a sequence's pieces to arrive joins them, in their order, and leaves the
  // count as it was before the call.
  __shared__ unsigned s_before;
  all_stored();
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* count = arrived + ((int64_t)b * c.kv_heads + g) * tiles + ht;
    s_before = atomicAdd(count, 1u);
    if (s_before == (unsigned)(p1 - p0 - 1)) atomicExch(count, 0u);
  }
  __syncthreads();
  if (s_before != (unsigned)(p1 - p0 - 1)) return;
  const int64_t at = (int64_t)(pc.slot + p0) * s.heads + head0;  // the first piece's first head
  const int count = p1 - p0;
  constexpr int PER = 256 / (DP / 4);  // heads side by side, each by DP / 4 threads
  for (int h0 = 0; h0 < n_heads; h0 += PER) {
    const int h = h0 + threadIdx.x / (DP / 4), d = threadIdx.x % (DP / 4) * 4;
    if (h >= n_heads) break;
    const float* ml = part_ml + 2 * (at + h);
    const float* o4 = part_o + (at + h) * c.dim + (d < c.dim ? d : 0);
    const int64_t ml_step = 2 * (int64_t)s.heads, o_step = (int64_t)s.heads * c.dim;
    float most = -INFINITY, total = 0;
    f32x4 y{};
    for (int p = 0; p < count; p += kJoinMost) {  // their loads are under way together
      f32x2 v[kJoinMost], u[kJoinMost], w[kJoinMost];
#pragma unroll
      for (int e = 0; e < kJoinMost; ++e) {
        const int64_t i = min(p + e, count - 1);
        v[e] = get(ml + i * ml_step);
        u[e] = get(o4 + i * o_step);
        w[e] = get(o4 + i * o_step + 2);
      }
#pragma unroll
      for (int e = 0; e < kJoinMost; ++e) {
        if (p + e >= count) break;
        const float now = fmaxf(most, v[e].x);
        const float base = now == -INFINITY ? 0.0f : now;
        const float fade = exp2f(most - base), f = exp2f(v[e].x - base);
        most = now;
        total = total * fade + f * v[e].y;
        y = y * fade + f * f32x4{u[e].x, u[e].y, w[e].x, w[e].y};
      }
    }
    if (d >= c.dim) continue;
    y *= total == 0 ? 0.0f : 1.0f / total;
    *reinterpret_cast<V4<T>*>(out + b * out_token + (head0 + h) * out_head + d) =
        __builtin_convertvector(y, V4<T>);
    if (lse && d == 0)
      lse[(int64_t)b * s.heads + head0 + h] =
          total == 0 ? -INFINITY : (most + log2f(total * Weights<T>::down)) * kLn2;
  }
}

// Joins the pieces of sequences that have several: a workgroup a sequence and head, half a wave to every
// eighth piece, eight of each at a time with their weights, so that up to 64 pieces wait for memory
// once.
template <typename T>
__global__ __launch_bounds__(256) void attention_paged_join_kernel(
    Cache c, PagedShape s, const int32_t* __restrict__ first_piece, T* __restrict__ out,
    int64_t out_token, int64_t out_head, float* __restrict__ lse,
    const int32_t* __restrict__ lengths, const float* __restrict__ part_o,
    const f32x2* __restrict__ part_ml) {
  constexpr int W = 8, U = 8;
  __shared__ f32x4 s_o[W][32];
  __shared__ f32x2 s_ml[W];
  const int b = blockIdx.x / s.heads, h = blockIdx.x % s.heads;
  const int d = 4 * (threadIdx.x & 31), mine = threadIdx.x >> 5;
  const int length = lengths[b], room = (c.indptr[b + 1] - c.indptr[b]) * c.page_size;
  const int slot = first_piece[b];
  const int last = length >= 0 && length <= room ? length : 0;
  const int first = s.window && last > s.window ? last - s.window : 0;
  const int p0 = first / s.piece, p1 = max(p0 + 1, (last + s.piece - 1) / s.piece), n = p1 - p0;
  if (n < 2) return;
  const int64_t at = (int64_t)(slot + p0) * s.heads + h;
  const f32x2* ml = part_ml + at;
  const float* o = part_o + at * c.dim + (d < c.dim ? d : 0);
  float most = -INFINITY, total = 0;
  f32x4 y{};
  for (int p = mine; p < n; p += W * U) {
    f32x2 v[U];
    f32x4 u[U];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int64_t i = (int64_t)min(p + W * e, n - 1) * s.heads;
      v[e] = ml[i];
      u[e] = *reinterpret_cast<const f32x4*>(o + i * c.dim);
    }
    float now = most;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      v[e] = p + W * e < n ? v[e] : f32x2{-INFINITY, 0};
      now = fmaxf(now, v[e].x);
    }
    const float base = now == -INFINITY ? 0.0f : now;
    const float fade = exp2f(most - base);
    most = now;
    total *= fade;
    y *= fade;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const float f = exp2f(v[e].x - base);
      total += f * v[e].y;
      y += f * u[e];
    }
  }
  s_o[mine][threadIdx.x & 31] = y;
  if (d == 0) s_ml[mine] = f32x2{most, total};
  __syncthreads();
  if (threadIdx.x >= 32) return;
  most = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) most = fmaxf(most, s_ml[w].x);
  const float base = most == -INFINITY ? 0.0f : most;
  total = 0;
  y = f32x4{};
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const f32x2 v = s_ml[w];
    const float f = exp2f(v.x - base);
    total += f * v.y;
    y += f * s_o[w][threadIdx.x];
  }
  y *= total == 0 ? 0.0f : 1.0f / total;
  if (d < c.dim)
    *reinterpret_cast<V4<T>*>(out + b * out_token + h * out_head + d) =
        __builtin_convertvector(y, V4<T>);
  if (lse && d == 0)
    lse[(int64_t)b * s.heads + h] =
        total == 0 ? -INFINITY : (most + log2f(total * Weights<T>::down)) * kLn2;
}

int check_cache(const fsp_paged_cache& c, const std::string& who) {
  if (!attn_dtype(c.dtype)) return set_error(FSP_ENOTSUP, who + ": dtype");
  if (!attn_dim(c.dim)) return set_error(FSP_ENOTSUP, who + ": dim");
  if (c.kv_heads < 1 || c.page_size < 1 || c.n_pages < 0 || c.batch < 0 || c.table_len < 0)
    return set_error(FSP_EINVAL, who + ": negative or zero size");
  if (c.kv_heads > 0xffff || c.batch > 0x7fffffffLL || c.page_size > 0x7fffffffLL ||
      c.n_pages > 0x7fffffffLL / c.page_size || c.table_len > kAttnTokensCap / c.page_size)
    return set_error(FSP_EINVAL, who + ": size exceeds 2^31-1024 tokens");
  if (c.batch > 0 && (!c.page_indptr || (c.table_len > 0 && (!c.page_indices || !c.k_pages || !c.v_pages))))
    return set_error(FSP_EINVAL, who + ": null pointer");
  if (!aligned16(c.k_pages, c.k_page | c.k_slot, c.k_head) ||
      !aligned16(c.v_pages, c.v_page | c.v_slot, c.v_head))
    return set_error(FSP_EINVAL, who + ": rows of the cache must be 16-byte aligned");
  return FSP_OK;
}

Cache cache_of(const fsp_paged_cache& c) {
  return {c.page_indptr, c.page_indices, c.k_page, c.k_slot, c.k_head, c.v_page, c.v_slot,
          c.v_head, (int)c.batch, (int)c.page_size, (int)c.dim, (int)c.kv_heads};
}

template <typename T, int MODE>
int launch_append(const fsp_paged_append_args& a, hipStream_t st) {
  const int64_t steps = ((a.heads + 2 * a.cache.kv_heads) * (a.cache.dim / 8) + kWave - 1) / kWave;
  int64_t parts = (4096 + a.n_tokens - 1) / a.n_tokens;  // waves enough for every SIMD
  if (parts > steps) parts = steps;
  const AppendShape s{a.n_tokens, a.k_token, a.k_head,    a.v_token,         a.v_head,           a.q_token,
                      a.q_head,   a.q_out_token, a.q_out_head, (int)a.heads, (int)a.half, (int)a.table_rows,
                      a.interleaved != 0, (int)parts};
  constexpr int kWaves = kAppendThreads / kWave;
  hipLaunchKernelGGL((paged_append_kernel<T, MODE>),
                     dim3((unsigned)((a.n_tokens * parts + kWaves - 1) / kWaves)),
                     dim3(kAppendThreads), 0, st, cache_of(a.cache), s,
                     static_cast<T*>(a.cache.k_pages), static_cast<T*>(a.cache.v_pages),
                     static_cast<const T*>(a.k), static_cast<const T*>(a.v),
                     static_cast<const T*>(a.q), static_cast<T*>(a.q_out), a.cos, a.sin,
                     a.token_indptr, a.lengths);
  return check_hip(hipGetLastError(), "paged_append_kernel launch");
}

template <typename T>
int launch_append_mode(const fsp_paged_append_args& a, hipStream_t st) {
  const bool aligned = (reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) % 16 == 0;
  if (a.half == 0) return launch_append<T, kStill>(a, st);
  if (aligned && !a.interleaved && a.half % 8 == 0) return launch_append<T, kHalves>(a, st);
  if (aligned && a.interleaved && a.half % 4 == 0) return launch_append<T, kNeighbours>(a, st);
  return launch_append<T, kEach>(a, st);
}

int64_t paged_workgroups(const fsp_attention_paged_args& a) {
  const int64_t group = a.heads / a.cache.kv_heads;
  return a.n_pieces * a.cache.kv_heads * ((group + kHeadTile - 1) / kHeadTile);
}

template <typename T, int DP, bool EXACT, bool NT>
int launch_paged(const fsp_attention_paged_args& a, hipStream_t st) {
  const PagedShape s{(int)a.heads, (int)a.window, (int)a.piece, (int)a.n_pieces, (float)a.scale};
  float* part_o = static_cast<float*>(a.workspace);
  float* part_ml = part_o + a.n_pieces * a.heads * a.cache.dim;
  hipLaunchKernelGGL((attention_paged_kernel<T, DP, EXACT, NT>), dim3((unsigned)paged_workgroups(a)),
                     dim3(256), 0, st, cache_of(a.cache), s,
                     reinterpret_cast<const Piece*>(a.pieces),
                     static_cast<const T*>(a.cache.k_pages),
                     static_cast<const T*>(a.cache.v_pages), static_cast<const T*>(a.q),
                     a.q_token, a.q_head, static_cast<T*>(a.out), a.out_token, a.out_head, a.lse,
                     a.lengths, part_o, part_ml, static_cast<unsigned*>(a.arrived));
  if (int rc = check_hip(hipGetLastError(), "attention_paged_kernel launch")) return rc;
  if (a.arrived || a.n_pieces == a.cache.batch) return FSP_OK;
  hipLaunchKernelGGL((attention_paged_join_kernel<T>), dim3((unsigned)(a.cache.batch * a.heads)),
                     dim3(256), 0, st, cache_of(a.cache), s, a.first_piece,
                     static_cast<T*>(a.out), a.out_token, a.out_head, a.lse, a.lengths, part_o,
                     reinterpret_cast<const f32x2*>(part_ml));
  return check_hip(hipGetLastError(), "attention_paged_join_kernel launch");
}

// A cache that the last-level cache (256 MB) cannot hold from step to step is read with loads that
// leave no lines behind, unless several workgroups read the same keys.  6 sequences of 131072 tokens,
// 3.2 GB: 601 us with ordinary loads, 554 so; 200 MB read again and again: 42 and 55 us.
template <typename T, int DP, bool EXACT>
int launch_paged_nt(const fsp_attention_paged_args& a, hipStream_t st) {
  const int64_t bytes = a.cache.table_len * a.cache.page_size * a.cache.kv_heads * a.cache.dim * 4;
  return bytes > (256 << 20) && a.heads / a.cache.kv_heads <= kHeadTile
             ? launch_paged<T, DP, EXACT, true>(a, st)
             : launch_paged<T, DP, EXACT, false>(a, st);
}

template <typename T>
int launch_paged_dim(const fsp_attention_paged_args& a, hipStream_t st) {
  if (a.cache.dim == 64) return launch_paged_nt<T, 64, true>(a, st);
  if (a.cache.dim < 64) return launch_paged_nt<T, 64, false>(a, st);
  if (a.cache.dim < 128) return launch_paged_nt<T, 128, false>(a, st);
  return launch_paged_nt<T, 128, true>(a, st);
}

}  // namespace
}  // namespace fsp

using namespace fsp;

extern "C" int64_t fsp_attention_dim_cap(void) { return kAttnDimCap; }

extern "C" int fsp_paged_append(const fsp_paged_append_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_paged_append: null arguments");
  const fsp_paged_append_args& a = *args;
  if (int rc = check_cache(a.cache, "fsp_paged_append")) return rc;
  if (a.n_tokens < 0 || a.heads < 0 || a.heads > 0xffff || a.half < 0 || a.table_rows < 0 ||
      2 * a.half > a.cache.dim || a.table_rows > 0x7fffffffLL || a.n_tokens > kMaxBlocks)
    return set_error(FSP_EINVAL, "fsp_paged_append: size out of range");
  if (a.n_tokens == 0) return FSP_OK;
  if (!a.token_indptr && a.n_tokens != a.cache.batch)
    return set_error(FSP_EINVAL, "fsp_paged_append: one token per sequence without token_indptr");
  if (a.cache.batch < 1)
    return set_error(FSP_EINVAL, "fsp_paged_append: tokens of no sequence");
  if (!a.k || !a.v || !a.lengths || (a.heads && (!a.q || !a.q_out)) ||
      (a.half && (!a.cos || !a.sin)))
    return set_error(FSP_EINVAL, "fsp_paged_append: null pointer");
  if (!aligned16(a.k, a.k_token, a.k_head) || !aligned16(a.v, a.v_token, a.v_head) ||
      !aligned16(a.q, a.q_token, a.q_head) || !aligned16(a.q_out, a.q_out_token, a.q_out_head))
    return set_error(FSP_EINVAL, "fsp_paged_append: rows must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.cache.dtype == FSP_BF16 ? launch_append_mode<bf16>(a, st) : launch_append_mode<f16>(a, st);
}

extern "C" int64_t fsp_attention_paged_piece(int64_t tokens, int64_t kv_heads) {
  // Two steps of the four waves, longer while that leaves a round of workgroups.  Pieces of 128 / 256 /
  // 512 / 1024 tokens, us: 96 sequences of up to 4096 tokens, 8 heads 58 / 55 / 55 / 61; 6 of 131072,
  // 8 heads 888 / 717 / 614 / 554; 18 of up to 4183, 2 heads 11 / 12 / 13 / 16
  int64_t piece = 256;
  while (piece < kPieceMost && tokens / piece * kv_heads > 1024) piece *= 2;
  return piece;
}

extern "C" int64_t fsp_attention_paged_counts(int64_t n_pieces, int64_t most, int64_t batch,
                                              int64_t heads, int64_t kv_heads) {
  if (batch < 0 || heads < 1 || kv_heads < 1 || n_pieces <= batch || most > kJoinMost) return 0;
  const int64_t per = kv_heads * ((heads / kv_heads + kHeadTile - 1) / kHeadTile);
  return n_pieces * per <= kJoinBlocks ? batch * per : 0;
}

extern "C" int64_t fsp_attention_paged_workspace(int64_t n_pieces, int64_t heads, int64_t dim) {
  if (n_pieces < 0 || heads < 0 || dim < 0) return 0;
  return n_pieces * heads * (dim + 2) * (int64_t)sizeof(float);
}

extern "C" int fsp_attention_paged(const fsp_attention_paged_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_paged: null arguments");
  const fsp_attention_paged_args& a = *args;
  if (int rc = check_cache(a.cache, "fsp_attention_paged")) return rc;
  if (a.heads < 1 || a.heads % a.cache.kv_heads || a.heads > 0xffff)
    return set_error(FSP_EINVAL, "fsp_attention_paged: heads must be a multiple of kv_heads");
  if (!isfinite((float)a.scale))
    return set_error(FSP_EINVAL, "fsp_attention_paged: scale must be finite in 32 bits");
  if (a.window < 0 || a.window > 0x7fffffffLL)
    return set_error(FSP_EINVAL, "fsp_attention_paged: window");
  if (a.piece < 128 || a.piece > kPieceMost || a.piece % 128)
    return set_error(FSP_EINVAL, "fsp_attention_paged: piece must be a multiple of 128 up to 1024");
  if (a.n_pieces < a.cache.batch || a.n_pieces > 0x7fffffffLL || a.cache.batch * a.heads > kMaxBlocks ||
      paged_workgroups(a) > kMaxBlocks)
    return set_error(FSP_EINVAL, "fsp_attention_paged: pieces out of range");
  if (a.cache.batch == 0) return FSP_OK;
  if (!a.q || !a.out || !a.lengths || !a.pieces ||
      (a.n_pieces > a.cache.batch && (!a.workspace || (!a.arrived && !a.first_piece))))
    return set_error(FSP_EINVAL, "fsp_attention_paged: null pointer");
  if (!aligned16(a.q, a.q_token, a.q_head) || !aligned16(a.out, a.out_token, a.out_head) ||
      reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return set_error(FSP_EINVAL, "fsp_attention_paged: rows must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.cache.dtype == FSP_BF16 ? launch_paged_dim<bf16>(a, st) : launch_paged_dim<f16>(a, st);
}
