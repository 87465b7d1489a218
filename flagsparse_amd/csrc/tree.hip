// Attention of trees of drafted tokens over a paged cache that holds them at its sequences' ends.
#include "paged.hpp"
#include "tiles.hpp"

namespace fsp {
namespace {

// More rows than so many beside a key go to wide tiles.  Tiles of 32 rows / wide ones, us, 8 key heads of 128: 8
// sequences of 30000, 36 rows 225 / 192, 64 rows 225 / 195; 4 of 2000, 64 rows 20.6 / 19.5; 96 ragged ones of up to
// 8000, 64 rows 126 / 97; 4 heads of 64, 8 of 30000, 36 rows 68 / 59.
constexpr int kWideFrom = 32;
// The workgroup that finishes a sequence's tile of 16 rows joins its pieces where they are at most so many and the
// workgroups few; else a second launch does.  By a launch and so, us: 1200 tokens, 16 heads of 64, 8 rows 12.5 /
// 9.9; 4 sequences of 2000, 8 heads of 128, 16 rows 15.4 / 14.8; with 16 pieces 13.8 / 14.8.  More rows a workgroup
// take it longer than a launch: 64 rows 20.9 / 23.7, 128 27 / 50.
constexpr int kJoinMost = 8;
constexpr int kJoinBlocks = 2048;
constexpr int kTableKeys = 1024;  // keys whose places LDS holds at a time

struct TreeShape {
  int heads, window, sinks, piece, n_pieces, n_tokens, longest, tiles;
  float scale;
  int by_tokens;  // how partial sums lie, and how far the rows of a piece behind those of the one before: see Sums
  int64_t step;
};

// A sequence's drafted tokens and what of its keys any of them sees: the places [first, last), where
// place e is token e from ``old`` on, and one of the first tokens, e - first, before it.
struct Drafted {
  int begin, count, past, first, old, last;
  bool ok;
  __device__ Drafted(const TreeShape& s, const int32_t* tokens, int b, int length, int room) {
    begin = tokens ? tokens[b] : b * s.longest;
    const int end = tokens ? tokens[b + 1] : begin + s.longest;
    ok = begin >= 0 && begin <= end && end <= s.n_tokens && end - begin <= s.longest &&
         length >= end - begin && length <= room;
    count = ok ? end - begin : 0;
    past = ok ? length - count : 0;
    last = ok ? length : 0;
    old = s.window ? max(past + 1 - s.window, 0) : 0;
    first = s.window ? (int)max((int64_t)past + 1 - s.window - s.sinks, (int64_t)0) : 0;
  }
  __device__ int pieces_end(int piece) const { return last / piece + (last % piece > 0); }
};

// Where the partial sums of a sequence's rows for one key head start.  By pieces, ``longest`` tokens' rows each, or by
// tokens, all rows of the call for each piece that a sequence has at most: the caller takes that where it is less than
// half as much.  It is where most sequences have fewer drafted tokens than ``longest``, or no bound is given: 64
// sequences with room for 131072 tokens and 8 drafted ones each, 32 heads of 128, 136 MB instead of 4.4 GB (pieces of
// 8192).
__device__ __forceinline__ int64_t sums_at(const TreeShape& s, const Drafted& t, int slot, int g, int group) {
  const int64_t token = s.by_tokens ? t.begin : (int64_t)slot * s.longest;
  return token * s.heads + g * ((s.by_tokens ? t.count : s.longest) * group);
}

// Rows of NaN for the tokens [from, to), those of one key head's queries.
template <typename T>
__device__ void nan_rows(T* out, int64_t out_token, int64_t out_head, float* lse, int heads, int head0, int group,
                         int dim, int from, int to) {
  const T nan = (T)__builtin_nanf("");
  const int per = group * (dim / 8);
  for (int64_t i = threadIdx.x; i < (int64_t)max(to - from, 0) * per; i += 256) {
    const int64_t t = from + i / per;
    const int h = head0 + (int)(i % per) / (dim / 8), d = (int)(i % per) % (dim / 8) * 8;
    *reinterpret_cast<V8<T>*>(out + t * out_token + h * out_head + d) =
        V8<T>{nan, nan, nan, nan, nan, nan, nan, nan};
    if (lse && d == 0) lse[t * heads + h] = __builtin_nanf("");
  }
}

// The rows that belong to no sequence, and those of one that is not as it should be.
template <typename T>
__device__ __forceinline__ void nan_outside(const TreeShape& s, const Drafted& t, const int32_t* tokens, int b,
                                            int batch, T* out, int64_t out_token, int64_t out_head, float* lse,
                                            int head0, int group, int dim) {
  const int from = tokens ? min(max(tokens[b], 0), s.n_tokens) : t.begin;
  const int to = tokens ? min(max(tokens[b + 1], 0), s.n_tokens) : t.begin + s.longest;
  if (!t.ok) nan_rows(out, out_token, out_head, lse, s.heads, head0, group, dim, from, to);
  if (b == 0) nan_rows(out, out_token, out_head, lse, s.heads, head0, group, dim, 0, from);
  if (b == batch - 1) nan_rows(out, out_token, out_head, lse, s.heads, head0, group, dim, to, s.n_tokens);
}

// Which drafted tokens a row's token sees, itself among them, by its way up the tree, as words 1 .. 8 of
// ``mask`` between one of ones and one of zeros; returns its depth, or -1 where the way does not lead up.
__device__ __forceinline__ int row_mask(const TreeShape& s, const Drafted& t, const int* up, int i,
                                        uint32_t* mask) {
  auto clear = [&] {
    mask[0] = ~0u;
#pragma unroll
    for (int w = 1; w < 11; ++w) mask[w] = 0;
  };
  clear();
  int depth = 0;
  for (int at = i;; ++depth) {
    mask[1 + at / 32] |= 1u << (at & 31);
    const int p = up ? up[at] : at - 1;
    if (p < -1 || p >= at) return -1;
    if (p < 0) break;
    at = p;
  }
  if (s.window && s.window <= depth) {  // the window leaves some of the way out
    clear();
    for (int at = i, n = 0; at >= 0; at = up ? up[at] : at - 1, ++n)
      if (n < s.window || t.past + depth - n < s.sinks) mask[1 + at / 32] |= 1u << (at & 31);
  }
  return depth;
}

// Whether the keys [begin, end) hold any that some row does not see: drafted ones, or some that a window leaves
// deep rows only, whose depth is less than the number of them.  Or whether a step that the end cuts, of 32 keys from
// one before it on, reaches drafted ones: seen_keys reads the rows' masks for it.
__device__ __forceinline__ bool some_hidden(const TreeShape& s, const Drafted& t, int begin, int end) {
  return end > t.past - 32 || (s.window && begin < t.past + t.count - s.window);
}

// Which of the 32 keys from place e0 on a row sees, whose first token by its window is ``lo``; ``count`` of them
// are keys of the piece.
__device__ __forceinline__ uint32_t seen_keys(const TreeShape& s, const Drafted& t, const uint32_t* mask, int lo,
                                              int e0, int count) {
  uint32_t bits = ~0u;
  const int off = e0 - t.past;
  if (off > -32) {
    const uint32_t* m = mask + 1 + (off >> 5);
    bits = off & 31 ? m[0] >> (off & 31) | m[1] << (32 - (off & 31)) : m[0];
  }
  const uint32_t far = ~bits_from(max(s.sinks, t.old) - e0);  // the first tokens that stay visible
  return bits & (bits_from(lo - e0) | far | bits_from(t.past - e0)) & ~bits_from(count);
}

// Whether this workgroup is the last of ``pieces`` to arrive, which joins them; it leaves the count as it was
// before the call.  What they put is stored by then.
__device__ __forceinline__ bool last_to_arrive(unsigned* count, int pieces) {
  __shared__ unsigned s_before;
  all_stored();
  __syncthreads();
  if (threadIdx.x == 0) {
    s_before = atomicAdd(count, 1u);
    if (s_before == (unsigned)(pieces - 1)) atomicExch(count, 0u);
  }
  __syncthreads();
  return s_before == (unsigned)(pieces - 1);
}

// Joins ``pieces`` of the rows [0, n) of a tile, in their order: row r's sums of a piece start at
// part_o + (at + r) * dim, those of the next one ``step`` rows on.
template <typename T, int DP, typename To>
__device__ __forceinline__ void join_tile(const float* part_o, const float* part_ml, int64_t at, int64_t step,
                                          int pieces, int n, int dim, const To& to) {
  constexpr int U = 8, ACROSS = DP / 4;
  for (int i = threadIdx.x; i < n * ACROSS; i += 256) {
    const int r = i / ACROSS, d = i % ACROSS * 4;
    const float* ml = part_ml + 2 * (at + r);
    const float* o = part_o + (at + r) * dim + (d < dim ? d : 0);
    float most = -INFINITY, total = 0;
    f32x4 y{};
    for (int p = 0; p < pieces; p += U) {  // their loads are under way together
      f32x2 v[U], a[U], b[U];
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int64_t k = min(p + e, pieces - 1) * step;
        v[e] = get(ml + 2 * k);
        a[e] = get(o + k * dim);
        b[e] = get(o + k * dim + 2);
      }
#pragma unroll
      for (int e = 0; e < U; ++e) {
        if (p + e >= pieces) break;
        const float now = fmaxf(most, v[e].x), base = now == -INFINITY ? 0.0f : now;
        const float fade = exp2f(most - base), f = exp2f(v[e].x - base);
        most = now;
        total = total * fade + f * v[e].y;
        y = y * fade + f * f32x4{a[e].x, a[e].y, b[e].x, b[e].y};
      }
    }
    if (d < dim) to(r, d, y, most, total);
  }
}

// The rows are the drafted tokens' queries of the heads that share a key head, a token's side by side: row r is
// token r / group, head r % group.  A workgroup takes a piece of a sequence's tokens for one key
// head and RT * 16 rows, so that what it reads of the cache serves all of them; its four waves take
// every fourth 32 keys.  Keys, values and products lie as in attention_paged_kernel, with RT times
// the rows beside each key: a key's fragment is read from LDS once for all, a value's put together once.
// Bound by memory: 8 sequences of 30000, 8 heads of 128, 983 MB in 166 us with 8 rows, 174 us with 32, 5.7 to
// 5.9 TB/s of the 7.0 of a plain read.  Rows for four tiles at once would not fit the registers (480 for dim 128).
// For 1200 tokens, 16 heads of 64 and 8 rows the chain piece -> length, offsets -> pages -> keys and the join are
// all of its 9 us.
template <typename T, int DP, bool EXACT, bool NT, int RT>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void attention_tree_kernel(
    Cache c, TreeShape s, const Piece* __restrict__ pieces, const T* __restrict__ k_pages,
    const T* __restrict__ v_pages, const T* __restrict__ q, int64_t q_token, int64_t q_head,
    T* __restrict__ out, int64_t out_token, int64_t out_head, float* __restrict__ lse,
    const int32_t* __restrict__ lengths, const int32_t* __restrict__ tokens,
    const int32_t* __restrict__ parents, float* part_o, float* part_ml, unsigned* arrived) {
  constexpr int E = DP / 16, NS = DP / 32, W = 4, ROWS = 16 * RT;
  typedef T VE __attribute__((ext_vector_type(E)));
  constexpr int CH = DP / 8, KL = DP / 16;
  __shared__ int64_t s_k[kTableKeys], s_v[kTableKeys];
  typedef float Rows[16][DP + 4];
  static_assert(sizeof(Rows) >= 64 * DP, "");
  __shared__ __attribute__((aligned(16))) char s_raw[W * sizeof(Rows)];
  __shared__ f32x2 s_ml[W][16];
  __shared__ uint32_t s_mask[ROWS][11];
  __shared__ int s_depth[ROWS], s_up[kDrafts];
  Rows* s_o = reinterpret_cast<Rows*>(s_raw);
  const int group = s.heads / c.kv_heads;
  int piece, g, tile;
  piece_and_head(blockIdx.x, s.n_pieces, c.kv_heads * s.tiles, piece, tile);
  g = tile / s.tiles;
  tile -= g * s.tiles;
  const Piece pc = pieces[piece];
  const int b = pc.seq, lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head0 = g * group;
  const Drafted t(s, tokens, b, lengths[b], pc.room);
  if (pc.begin == 0 && tile == 0)
    nan_outside(s, t, tokens, b, c.batch, out, out_token, out_head, lse, head0, group, c.dim);
  const int rows = t.count * group, r0 = tile * ROWS;
  if (r0 >= rows) return;
  const int p0 = t.first / s.piece, p1 = t.pieces_end(s.piece);
  const int mine = p0 + pc.begin / s.piece;
  if (mine >= p1) return;
  const int begin = max(t.first, mine * s.piece);
  const int end = (int)min((int64_t)t.last, ((int64_t)mine + 1) * s.piece);

  V8<T> qf[RT][NS];
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    const int r = min(r0 + 16 * n + col, rows - 1);
    const T* qr = q + (int64_t)(t.begin + r / group) * q_token + (head0 + r % group) * q_head;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int d = 32 * i + 8 * quad;
      const V8<T> x = *reinterpret_cast<const V8<T>*>(qr + (d < c.dim ? d : 0));
      qf[n][i] = scaled_sign<T>(x, s.scale, d < c.dim);
    }
  }
  const float cs = exp2_scale(s.scale);

  const bool masked = some_hidden(s, t, begin, end);
  if (masked) {
    if (parents)
      for (int i = threadIdx.x; i < t.count; i += 256) s_up[i] = parents[t.begin + i];
    __syncthreads();
    if (threadIdx.x < ROWS)
      s_depth[threadIdx.x] = row_mask(s, t, parents ? s_up : nullptr,
                                      min(r0 + (int)threadIdx.x, rows - 1) / group, s_mask[threadIdx.x]);
    __syncthreads();
  }
  int lo[RT];  // the first token that each row's window holds
#pragma unroll
  for (int n = 0; n < RT; ++n) lo[n] = s.window && masked ? t.past + s_depth[16 * n + col] - s.window + 1 : 0;

  const T* kb = k_pages + g * c.k_head;
  const T* vb = v_pages + g * c.v_head;
  i32x4 kr[KL];
  VE vf[8];
  const int k_row = lane / CH, k_chunk = lane % CH;
  auto load_k = [&](int j, int most) {
#pragma unroll
    for (int i = 0; i < KL; ++i)
      kr[i] = ld_stream<NT>(reinterpret_cast<const i32x4*>(
          kb + s_k[min(j + 64 / CH * i + k_row, most)] +
          (EXACT || 8 * k_chunk < c.dim ? 8 * k_chunk : 0)));
  };
  char* s_rows = s_raw + wave * sizeof(Rows);
  const int ve = E * col < c.dim ? E * col : 0;
  auto load_v = [&](int j, int most) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      vf[e] = ld_stream<NT>(reinterpret_cast<const VE*>(
          vb + s_v[min(j + 16 * (e / 4) + 4 * quad + e % 4, most)] + ve));
  };

  float top[RT], sum[RT];
  f32x4 o[RT][E];
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    top[n] = -INFINITY;
    sum[n] = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) o[n][i] = f32x4{};
  }

  for (int c0 = begin; c0 < end; c0 += kTableKeys) {
    const int n_keys = min(kTableKeys, end - c0), padded = (n_keys + 127) & ~127;
    if (c0 > begin) __syncthreads();
    for (int i = threadIdx.x; i < padded; i += 256) {
      const int e = c0 + (i < n_keys ? i : 0);
      const uint32_t j = e < t.old ? e - t.first : e;
      const uint32_t at = j / (uint32_t)c.page_size;
      const int64_t page = c.indices[pc.page + at], slot = j - at * c.page_size;
      s_k[i] = page * c.k_page + slot * c.k_slot;
      s_v[i] = page * c.v_page + slot * c.v_slot;
    }
    __syncthreads();
    int j = 32 * wave;
    if (j < n_keys) load_k(j, kTableKeys - 1), load_v(j, kTableKeys - 1);
    for (; j < n_keys; j += 32 * W) {
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const int row = 64 / CH * i + k_row;
        *reinterpret_cast<i32x4*>(s_rows + row * 2 * DP + 16 * (k_chunk ^ (row & (CH - 1)))) =
            EXACT ? kr[i] : kr[i] & (8 * k_chunk < c.dim ? -1 : 0);
      }
      f32x4 x[RT][2];
#pragma unroll
      for (int n = 0; n < RT; ++n) x[n][0] = x[n][1] = f32x4{};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        V8<T> kf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = 16 * u + col;
          kf[u] = *reinterpret_cast<const V8<T>*>(s_rows + row * 2 * DP +
                                                  16 * ((4 * i + quad) ^ (row & (CH - 1))));
        }
#pragma unroll
        for (int n = 0; n < RT; ++n)
#pragma unroll
          for (int u = 0; u < 2; ++u) x[n][u] = mfma16(kf[u], qf[n][i], x[n][u]);
      }
      const bool more = j + 32 * W < n_keys;
      const int next = more ? j + 32 * W : j, most = more ? kTableKeys - 1 : j;
      load_k(next, most);
      const int e0 = c0 + j;  // the places of these keys
      const bool tail = e0 + 32 > t.past, partial = j + 32 > n_keys;
      if (partial) {
#pragma unroll
        for (int e = 0; e < 8; ++e) vf[e] = j + 16 * (e / 4) + 4 * quad + e % 4 < n_keys ? vf[e] : VE{};
      }
      V8<T> pf[RT];
#pragma unroll
      for (int n = 0; n < RT; ++n) {
        if (partial || tail || __any(lo[n] > max(e0, t.old))) {
          const uint32_t bits = seen_keys(s, t, s_mask[16 * n + col], lo[n], e0, n_keys - j) >> (4 * quad);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t b = bits >> (16 * u);
            x[n][u][0] = seen_or_none<0>(b, x[n][u][0]);
            x[n][u][1] = seen_or_none<1>(b, x[n][u][1]);
            x[n][u][2] = seen_or_none<2>(b, x[n][u][2]);
            x[n][u][3] = seen_or_none<3>(b, x[n][u][3]);
          }
        }
        float m = x[n][0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) m = fmaxf(m, x[n][e / 4][e % 4]);
        if (__any((m - top[n]) * cs > Weights<T>::lag)) {
          m = fmaxf(m, __shfl_xor(m, 16));
          m = fmaxf(m, __shfl_xor(m, 32));
          const float now = fmaxf(top[n], m);
          const float fade = top[n] == -INFINITY ? 0.0f : exp2f((top[n] - now) * cs);
          top[n] = now;
          sum[n] *= fade;
#pragma unroll
          for (int i = 0; i < E; ++i) o[n][i] *= fade;
        }
        const float base = top[n] == -INFINITY ? 0.0f : top[n] * cs - Weights<T>::up;
        f32x8 p;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(fmaf(x[n][e / 4][e % 4], cs, -base));
          sum[n] += p[e];
        }
        pf[n] = __builtin_convertvector(p, V8<T>);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) {
        V8<T> a;
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = vf[e][i];
#pragma unroll
        for (int n = 0; n < RT; ++n) o[n][i] = mfma16(a, pf[n], o[n][i]);
      }
      load_v(next, most);
    }
  }

  // join the waves, 16 rows at a time
  const bool split = p1 - p0 > 1;
  const int64_t first = sums_at(s, t, pc.slot, g, group), slot = first + (mine - p0) * s.step;
  auto to_out = [&](int r, int d, f32x4 y, float most, float total) {
    const int64_t token = t.begin + (r0 + r) / group;
    const int head = head0 + (r0 + r) % group;
    y *= total == 0 ? 0.0f : 1.0f / total;
    *reinterpret_cast<V4<T>*>(out + token * out_token + head * out_head + d) = __builtin_convertvector(y, V4<T>);
    if (lse && d == 0)
      lse[token * s.heads + head] = total == 0 ? -INFINITY : (most + log2f(total * Weights<T>::down)) * kLn2;
  };
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    if (r0 + 16 * n >= rows) break;
    sum[n] += __shfl_xor(sum[n], 16);
    sum[n] += __shfl_xor(sum[n], 32);
    const float ml = top[n] == -INFINITY ? -INFINITY : top[n] * cs;
    __syncthreads();
    if (quad == 0) s_ml[wave][col] = f32x2{ml, sum[n]};
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) s_o[wave][col][4 * E * quad + E * r + i] = o[n][i][r];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (DP / 4); i += 256) {
      const int row = i / (DP / 4), d = i % (DP / 4) * 4, r = r0 + 16 * n + row;
      if (d >= c.dim || r >= rows) continue;
      float most = -INFINITY, total = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) most = fmaxf(most, s_ml[w][row].x);
      f32x4 y{};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const f32x2 v = s_ml[w][row];
        const float f = v.x == -INFINITY ? 0.0f : exp2f(v.x - most);
        if (v.y == 0) continue;  // saw nothing: its sums are zeros
        total += f * v.y;
        y += f * *reinterpret_cast<const f32x4*>(&s_o[w][row][d]);
      }
      if (masked && s_depth[16 * n + row] < 0) total = __builtin_nanf("");
      if (!split) {
        to_out(r - r0, d, y, most, total);
      } else if (RT == 1 && arrived) {
        put(part_o + (slot + r) * c.dim + d, y.x, y.y);
        put(part_o + (slot + r) * c.dim + d + 2, y.z, y.w);
        if (d == 0) put(part_ml + 2 * (slot + r), most, total);
      } else {
        *reinterpret_cast<f32x4*>(part_o + (slot + r) * c.dim + d) = y;
        if (d == 0) *reinterpret_cast<f32x2*>(part_ml + 2 * (slot + r)) = f32x2{most, total};
      }
    }
  }
  if constexpr (RT > 1) return;
  if (!split || !arrived) return;  // without counts, another launch joins them
  if (last_to_arrive(arrived + ((int64_t)b * c.kv_heads + g) * s.tiles + tile, p1 - p0))
    join_tile<T, DP>(part_o, part_ml, first + r0, s.step, p1 - p0, min(ROWS, rows - r0), c.dim, to_out);
}

// Rows past a head's dim are read from here.
__device__ const i32x4 kZeros = {0, 0, 0, 0};

// Many rows: 128 of them a workgroup, 32 a wave, over the same 64 keys, which go straight to LDS by the places
// that a table there holds, the next step's while this one's are worked on: as attention_packed_kernel, whose
// comments say how the products lie.  The table's two halves of 256 keys are filled in turn, the pages of
// the next one asked for four steps before.  8 sequences of 30000, 8 heads of 128, 256 rows, 2.5e11 operations and
// 983 MB: 288 us and 11 for the join, 0.84 PFLOP/s (a library's 8192^3 product: 1.21); products take 47 % of
// the SIMDs' cycles, vector instructions 44 %, both at a time 16 %, at the 1.94 GHz that power leaves; no bank
// conflicts.  128 rows: 203 us in all, 4.9 TB/s.  Choosing addresses for rows past a head's dim by a branch made
// it 373 us, conditions instead of bits for the masks 348: they kept scalar registers in memory.  A higher
// priority of waves in their products, or exponentials put between them, changed nothing (315 / 315, 312 / 320).
template <typename T, int DP, bool EXACT>
__global__ __launch_bounds__(256, 2) void attention_tree_wide_kernel(
    Cache c, TreeShape s, const Piece* __restrict__ pieces, const T* __restrict__ k_pages,
    const T* __restrict__ v_pages, const T* __restrict__ q, int64_t q_token, int64_t q_head,
    T* __restrict__ out, int64_t out_token, int64_t out_head, float* __restrict__ lse,
    const int32_t* __restrict__ lengths, const int32_t* __restrict__ tokens,
    const int32_t* __restrict__ parents, float* part_o, float* part_ml) {
  typedef Lay<DP> L;
  constexpr int NS = DP / 16, NT = DP / 32, ROWS = 128, HALF = 256;
  __shared__ __attribute__((aligned(1024))) char s_k0[L::BYTES], s_v0[L::BYTES], s_k1[L::BYTES], s_v1[L::BYTES];
  __shared__ int64_t s_k[2 * HALF], s_v[2 * HALF];
  __shared__ uint32_t s_mask[ROWS][11];
  __shared__ int s_depth[ROWS], s_up[kDrafts];
  const int group = s.heads / c.kv_heads;
  int piece, g, tile;
  piece_and_head(blockIdx.x, s.n_pieces, c.kv_heads * s.tiles, piece, tile);
  g = tile / s.tiles;
  tile -= g * s.tiles;
  const Piece pc = pieces[piece];
  const int b = pc.seq, lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head0 = g * group;
  const Drafted t(s, tokens, b, lengths[b], pc.room);
  if (pc.begin == 0 && tile == 0)
    nan_outside(s, t, tokens, b, c.batch, out, out_token, out_head, lse, head0, group, c.dim);
  const int rows = t.count * group, r0 = tile * ROWS;
  if (r0 >= rows) return;
  const int p0 = t.first / s.piece, p1 = t.pieces_end(s.piece);
  const int mine = p0 + pc.begin / s.piece;
  if (mine >= p1) return;
  const int begin = max(t.first, mine * s.piece);
  const int end = (int)min((int64_t)t.last, ((int64_t)mine + 1) * s.piece);
  const int n = end - begin, steps = (n + kRows - 1) / kRows;

  const int q0 = r0 + 32 * wave, row = q0 + col;
  const bool active = q0 < rows;
  V8<T> qf[NS];
  {
    const int r = min(row, rows - 1);
    const T* qr = q + (int64_t)(t.begin + r / group) * q_token + (head0 + r % group) * q_head;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int d = 16 * i + 8 * half;
      const V8<T> x = *reinterpret_cast<const V8<T>*>(qr + (d < c.dim ? d : 0));
      qf[i] = scaled_sign<T>(x, s.scale, d < c.dim);
    }
  }
  const float cs = exp2_scale(s.scale);

  // the page of key 256 * h + threadIdx.x of the piece, and then where that lies; those past the end stand
  // for the first one
  auto key_of = [&](int h) {
    const int i = HALF * h + threadIdx.x, e = begin + (i < n ? i : 0);
    return (uint32_t)(e < t.old ? e - t.first : e);
  };
  auto page_of = [&](int h) { return c.indices[pc.page + key_of(h) / (uint32_t)c.page_size]; };
  auto place = [&](int h, int64_t page) {
    const int64_t slot = key_of(h) % (uint32_t)c.page_size;
    const int at = h % 2 * HALF + threadIdx.x;
    s_k[at] = page * c.k_page + slot * c.k_slot;
    s_v[at] = page * c.v_page + slot * c.v_slot;
  };
#pragma unroll
  for (int h = 0; h < 2; ++h) place(h, page_of(h));
  const bool masked = some_hidden(s, t, begin, end);
  if (masked && parents)
    for (int i = threadIdx.x; i < t.count; i += 256) s_up[i] = parents[t.begin + i];
  __syncthreads();

  const T* kb = k_pages + g * c.k_head;
  const T* vb = v_pages + g * c.v_head;
  constexpr int PER = kRows * L::PITCH / 1024 / 4, EACH = 1024 / L::PITCH;
  const int l_row = wave * PER * EACH + lane / L::CH;
  const int l_chunk = (lane % L::CH) ^ L::swizzle(lane / L::CH) ^ L::swizzle(wave * PER * EACH);
  typedef __attribute__((address_space(3))) void lds_void;
  typedef __attribute__((address_space(1))) void global_void;
  auto load = [&](int step, char* sk, char* sv) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = (step * kRows & (2 * HALF - 1)) + l_row + i * EACH;
      const int d = 8 * (l_chunk ^ L::swizzle(i * EACH));
      uint64_t k = (uint64_t)(kb + s_k[at] + d), v = (uint64_t)(vb + s_v[at] + d);
      if constexpr (!EXACT) {
        asm volatile("" : "+v"(k), "+v"(v));  // a choice of addresses, not a branch around their reads
        k = d < c.dim ? k : (uint64_t)&kZeros;
        v = d < c.dim ? v : (uint64_t)&kZeros;
      }
      __builtin_amdgcn_global_load_lds((const global_void*)k, (lds_void*)(sk + (wave * PER + i) * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const global_void*)v, (lds_void*)(sv + (wave * PER + i) * 1024), 16, 0, 0);
    }
  };
  load(0, s_k0, s_v0);
  if (masked && threadIdx.x < ROWS)
    s_depth[threadIdx.x] = row_mask(s, t, parents ? s_up : nullptr,
                                    min(r0 + (int)threadIdx.x, rows - 1) / group, s_mask[threadIdx.x]);

  f32x16 o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = f32x16{};
  float top = -INFINITY, sum = 0;
  const int k_at = L::row_at(lane), v_at = L::col_at(lane);
  all_stored();
  __syncthreads();
  const int lo = s.window && masked ? t.past + s_depth[32 * wave + col] - s.window + 1 : 0;

  auto work = [&](int step, const char* sk_, const char* sv_) {
    if (!active) return;
    const lds_char* sk = (const lds_char*)sk_;
    const lds_char* sv = (const lds_char*)sv_;
    f32x16 x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      x[u] = f32x16{};
#pragma unroll
      for (int i = 0; i < NS; ++i)
        x[u] = mfma32(row_frag<T>(sk + (k_at ^ (i * 32)) + u * 32 * L::PITCH), qf[i], x[u]);
    }
    read_ahead<2 * NS, NS>();
    const int j0 = step * kRows, e0 = begin + j0;
    const bool tail = e0 + kRows > t.past;
    if (tail || j0 + kRows > n || __any(lo > max(e0, t.old))) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        seen_or_none(seen_keys(s, t, s_mask[32 * wave + col], lo, e0 + 32 * u, n - j0 - 32 * u), half, x[u]);
    }
    float m = x[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, x[u][r]);
    m = fmaxf(m, other_half(m));
    if (__any((m - top) * cs > Weights<T>::lag)) {
      const float now = fmaxf(top, m);
      const float fade = top == -INFINITY ? 0.0f : exp2f((top - now) * cs);
      top = now;
      sum *= fade;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] *= fade;
    }
    const float base = top == -INFINITY ? 0.0f : top * cs - Weights<T>::up;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[u][r] = __builtin_amdgcn_exp2f(fmaf(x[u][r], cs, -base));
        sum += x[u][r];
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const V8<T> pf = to16<T>(x[i / 2], 8 * (i % 2));
#pragma unroll
      for (int d = 0; d < NT; ++d)
        o[d] = mfma32(col_frag<T, L::PITCH>(sv, v_at ^ (64 * d), i), pf, o[d]);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4 * NT, 1);  // the first values early
  };
  // one step; the table's other half is filled when the last of its keys have been asked for
  auto pass = [&](int step, char* sk, char* sv, char* next_k, char* next_v) {
    const bool fill = step % 4 == 0 && step > 0 && (step + 4) * kRows < n;
    int page = 0;
    if (fill) page = page_of(step / 4 + 1);
    if (step + 1 < steps) load(step + 1, next_k, next_v);
    work(step, sk, sv);
    if (fill) place(step / 4 + 1, page);
    all_stored();
    __syncthreads();
  };
  for (int step = 0; step < steps;) {
    pass(step, s_k0, s_v0, s_k1, s_v1);
    if (++step >= steps) break;
    pass(step, s_k1, s_v1, s_k0, s_v0);
    ++step;
  }

  if (row >= rows) return;
  sum += other_half(sum);
  if (sum == 0)  // nothing seen: zeros, whatever lies in the rows of V
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] = f32x16{};
  if (masked && s_depth[32 * wave + col] < 0) sum = __builtin_nanf("");
  if (p1 - p0 == 1) {
    const int64_t token = t.begin + row / group;
    const int head = head0 + row % group;
    if (half == 0 && lse)
      lse[token * s.heads + head] =
          sum == 0 ? -INFINITY : (top * cs + log2f(sum * Weights<T>::down)) * kLn2;
    store_rows<T, NT>(out + token * out_token + head * out_head, o, sum == 0 ? 0.0f : 1.0f / sum, c.dim, half);
    return;
  }
  const int64_t at = sums_at(s, t, pc.slot, g, group) + (mine - p0) * s.step + row;
  store_rows<float, NT>(part_o + at * c.dim, o, 1.0f, c.dim, half);
  if (half == 0)
    *reinterpret_cast<f32x2*>(part_ml + 2 * at) = f32x2{top == -INFINITY ? -INFINITY : top * cs, sum};
}

// Joins the pieces of sequences that have several: half a wave to a row, eight pieces of it at a time (sixteen:
// 24.3 / 26.0 us for 33 ragged sequences, 23 heads of 80, where it takes 7.6 of them).  Bound by its loads one after
// the other: lengths and offsets, sums, and a second round from nine pieces on.
template <typename T>
__global__ __launch_bounds__(256) void attention_tree_join_kernel(
    Cache c, TreeShape s, const int32_t* __restrict__ first_piece, T* __restrict__ out, int64_t out_token,
    int64_t out_head, float* __restrict__ lse, const int32_t* __restrict__ lengths,
    const int32_t* __restrict__ tokens, const float* __restrict__ part_o,
    const f32x2* __restrict__ part_ml) {
  constexpr int U = 8;
  const int group = s.heads / c.kv_heads;
  const int per = (s.longest * s.heads + 7) / 8, b = blockIdx.x / per;
  const int i = blockIdx.x % per * 8 + (threadIdx.x >> 5), d = 4 * (threadIdx.x & 31);
  const int g = i / (s.longest * group), r = i % (s.longest * group);
  const Drafted t(s, tokens, b, lengths[b], (c.indptr[b + 1] - c.indptr[b]) * c.page_size);
  const int p0 = t.first / s.piece, n = t.pieces_end(s.piece) - p0;
  if (n < 2 || g >= c.kv_heads || r >= t.count * group) return;
  const int64_t step = s.step, at = sums_at(s, t, first_piece[b], g, group) + r;
  const f32x2* ml = part_ml + at;
  const float* o = part_o + at * c.dim + (d < c.dim ? d : 0);
  float most = -INFINITY, total = 0;
  f32x4 y{};
  for (int p = 0; p < n; p += U) {
    f32x2 v[U];
    f32x4 u[U];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int64_t k = min(p + e, n - 1) * step;
      v[e] = ml[k];
      u[e] = *reinterpret_cast<const f32x4*>(o + k * c.dim);
    }
    float now = most;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      v[e] = p + e < n ? v[e] : f32x2{-INFINITY, 0};
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
  if (d >= c.dim) return;
  y *= total == 0 ? 0.0f : 1.0f / total;
  const int64_t token = t.begin + r / group;
  const int head = g * group + r % group;
  *reinterpret_cast<V4<T>*>(out + token * out_token + head * out_head + d) = __builtin_convertvector(y, V4<T>);
  if (lse && d == 0)
    lse[token * s.heads + head] = total == 0 ? -INFINITY : (most + log2f(total * Weights<T>::down)) * kLn2;
}

// Rows of a workgroup's tile.
int64_t tile_rows(int64_t longest, int64_t group) {
  const int64_t rows = longest * group;
  return rows <= 16 ? 16 : rows <= kWideFrom ? 32 : 128;
}

// A call's arguments, with the most pieces of a sequence where partial sums lie by tokens (0: by pieces).
struct TreeCall : fsp_attention_tree_args {
  int64_t most = 0;
};

int64_t tiles_of(int64_t longest, int64_t group) {
  const int64_t each = tile_rows(longest, group);
  return (longest * group + each - 1) / each;
}

// Whether another launch joins the pieces.
bool joined(const TreeCall& a) {
  return a.n_pieces > a.cache.batch &&
         !(a.arrived && tile_rows(a.longest, a.heads / a.cache.kv_heads) == 16);
}

template <typename T, typename Kernel, typename... More>
int launch_tree(const TreeCall& a, Kernel kernel, hipStream_t st, More... more) {
  const int64_t tiles = tiles_of(a.longest, a.heads / a.cache.kv_heads);
  const TreeShape s{(int)a.heads,    (int)a.window,  (int)a.sinks, (int)a.piece,  (int)a.n_pieces,
                    (int)a.n_tokens, (int)a.longest, (int)tiles,   (float)a.scale,
                    a.most > 0,      (a.most ? a.n_tokens : a.longest) * a.heads};
  float* part_o = static_cast<float*>(a.workspace);
  float* part_ml = part_o + (a.most ? a.most * a.n_tokens : a.n_pieces * a.longest) * a.heads * a.cache.dim;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.n_pieces * a.cache.kv_heads * tiles)), dim3(256), 0, st,
                     cache_of(a.cache), s, reinterpret_cast<const Piece*>(a.pieces),
                     static_cast<const T*>(a.cache.k_pages), static_cast<const T*>(a.cache.v_pages),
                     static_cast<const T*>(a.q), a.q_token, a.q_head, static_cast<T*>(a.out), a.out_token,
                     a.out_head, a.lse, a.lengths, a.token_indptr, a.parents, part_o, part_ml,
                     more...);
  if (int rc = check_hip(hipGetLastError(), "attention_tree_kernel launch")) return rc;
  if (!joined(a)) return FSP_OK;
  hipLaunchKernelGGL((attention_tree_join_kernel<T>),
                     dim3((unsigned)(a.cache.batch * ((a.longest * a.heads + 7) / 8))), dim3(256), 0, st,
                     cache_of(a.cache), s, a.first_piece, static_cast<T*>(a.out), a.out_token, a.out_head,
                     a.lse, a.lengths, a.token_indptr, part_o, reinterpret_cast<const f32x2*>(part_ml));
  return check_hip(hipGetLastError(), "attention_tree_join_kernel launch");
}

template <typename T, int DP, bool EXACT, bool NT>
int launch_tree_rows(const TreeCall& a, hipStream_t st) {
  unsigned* arrived = static_cast<unsigned*>(a.arrived);
  return tile_rows(a.longest, a.heads / a.cache.kv_heads) == 16
             ? launch_tree<T>(a, attention_tree_kernel<T, DP, EXACT, NT, 1>, st, arrived)
             : launch_tree<T>(a, attention_tree_kernel<T, DP, EXACT, NT, 2>, st, arrived);
}

template <typename T, int DP, bool EXACT>
int launch_tree_nt(const TreeCall& a, hipStream_t st) {
  const int64_t bytes = a.cache.table_len * a.cache.page_size * a.cache.kv_heads * a.cache.dim * 4;
  return bytes > (256 << 20)
             ? launch_tree_rows<T, DP, EXACT, true>(a, st)
             : launch_tree_rows<T, DP, EXACT, false>(a, st);
}

template <typename T>
int launch_tree_dim(const TreeCall& a, hipStream_t st) {
  const int64_t dim = a.cache.dim;
  if (tile_rows(a.longest, a.heads / a.cache.kv_heads) == 128)
    return dim < 64     ? launch_tree<T>(a, attention_tree_wide_kernel<T, 64, false>, st)
           : dim == 64  ? launch_tree<T>(a, attention_tree_wide_kernel<T, 64, true>, st)
           : dim <= 96  ? launch_tree<T>(a, attention_tree_wide_kernel<T, 96, false>, st)
           : dim == 128 ? launch_tree<T>(a, attention_tree_wide_kernel<T, 128, true>, st)
                        : launch_tree<T>(a, attention_tree_wide_kernel<T, 128, false>, st);
  if (dim == 64) return launch_tree_nt<T, 64, true>(a, st);
  if (dim < 64) return launch_tree_nt<T, 64, false>(a, st);
  if (dim < 128) return launch_tree_nt<T, 128, false>(a, st);
  return launch_tree_nt<T, 128, true>(a, st);
}

}  // namespace
}  // namespace fsp

using namespace fsp;

extern "C" int64_t fsp_attention_tree_drafts(void) { return kDrafts; }

extern "C" int64_t fsp_attention_tree_rows(int64_t group, int64_t longest) {
  return group < 1 || longest < 1 ? 16 : tile_rows(longest, group);
}

extern "C" int64_t fsp_attention_tree_counts(int64_t n_pieces, int64_t most, int64_t batch, int64_t kv_heads,
                                             int64_t group, int64_t longest) {
  if (batch < 0 || kv_heads < 1 || group < 1 || longest < 1 || n_pieces <= batch || most > kJoinMost) return 0;
  if (tile_rows(longest, group) != 16) return 0;
  return n_pieces * kv_heads <= kJoinBlocks ? batch * kv_heads : 0;
}

extern "C" int64_t fsp_attention_tree_workspace(int64_t n_pieces, int64_t heads, int64_t dim, int64_t longest) {
  if (n_pieces < 0 || heads < 0 || dim < 0 || longest < 0) return 0;
  return n_pieces * longest * heads * (dim + 2) * (int64_t)sizeof(float);
}

extern "C" int64_t fsp_attention_tree_by_tokens_workspace(int64_t most, int64_t n_tokens, int64_t heads,
                                                          int64_t dim) {
  if (most < 0 || n_tokens < 0 || heads < 0 || dim < 0) return 0;
  return most * n_tokens * heads * (dim + 2) * (int64_t)sizeof(float);
}

namespace {

int run_tree(const TreeCall& a, const std::string& who, void* stream) {
  if (int rc = check_cache(a.cache, who)) return rc;
  if (a.heads < 1 || a.heads % a.cache.kv_heads || a.heads > 0xffff)
    return set_error(FSP_EINVAL, who + ": heads must be a multiple of kv_heads");
  if (!isfinite((float)a.scale))
    return set_error(FSP_EINVAL, who + ": scale must be finite in 32 bits");
  if (a.window < 0 || a.window > kAttnTokensCap || a.sinks < 0 || a.sinks > kAttnTokensCap ||
      (a.sinks && !a.window))
    return set_error(FSP_EINVAL, who + ": window, or sinks without one");
  if (a.piece < 128 || a.piece > (1 << 20) || a.piece % 128)
    return set_error(FSP_EINVAL, who + ": piece must be a multiple of 128 up to 2^20");
  if (a.n_tokens < 0 || a.n_tokens > kAttnTokensCap || a.longest < 0 || a.longest > kDrafts ||
      a.n_pieces < a.cache.batch || a.n_pieces > 0x7fffffffLL)
    return set_error(FSP_EINVAL, who + ": size out of range");
  if (!a.token_indptr && a.n_tokens != a.longest * a.cache.batch)
    return set_error(FSP_EINVAL, who + ": longest tokens per sequence without token_indptr");
  if (a.n_tokens == 0) return FSP_OK;
  if (a.cache.batch == 0 || a.longest == 0)
    return set_error(FSP_EINVAL, who + ": tokens of no sequence");
  const int64_t rows = a.longest * a.heads, group = a.heads / a.cache.kv_heads;
  if (a.n_pieces > kMaxBlocks / (a.cache.kv_heads * tiles_of(a.longest, group)) ||
      (joined(a) && a.cache.batch > kMaxBlocks / ((rows + 7) / 8)))
    return set_error(FSP_EINVAL, who + ": pieces out of range");
  if (!a.q || !a.out || !a.lengths || !a.pieces ||
      (a.n_pieces > a.cache.batch && (!a.workspace || !a.first_piece)))
    return set_error(FSP_EINVAL, who + ": null pointer");
  if (!aligned16(a.q, a.q_token, a.q_head) || !aligned16(a.out, a.out_token, a.out_head) ||
      reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return set_error(FSP_EINVAL, who + ": rows must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.cache.dtype == FSP_BF16 ? launch_tree_dim<bf16>(a, st) : launch_tree_dim<f16>(a, st);
}

}  // namespace

extern "C" int fsp_attention_tree(const fsp_attention_tree_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_tree: null arguments");
  return run_tree({*args}, "fsp_attention_tree", stream);
}

extern "C" int fsp_attention_tree_by_tokens(const fsp_attention_tree_args* args, int64_t most, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_tree_by_tokens: null arguments");
  if (most < 1 || most > args->n_pieces)
    return set_error(FSP_EINVAL, "fsp_attention_tree_by_tokens: the pieces of one sequence");
  return run_tree({*args, most}, "fsp_attention_tree_by_tokens", stream);
}
