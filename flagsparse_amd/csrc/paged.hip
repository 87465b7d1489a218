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
// there are few tokens.  Bound by memory for prompts (a read and a write of every element) and by
// the chain token -> sequence -> page -> row for single tokens.
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

// Attention of one query per sequence.  A workgroup takes a piece of a sequence's tokens for one key
// head and up to 16 of the query heads that share it; its four waves take every fourth 32 keys.
//
// Keys and values go from memory to the matrix instructions' registers with no stop in LDS.  With
// S^T = K Q^T lane l has head l % 16 and, of 32 keys, the eight 4 * (l / 16) + {0..3, 16..19}: its
// weights are the operand of O^T = V^T P^T as they lie, since the order of the summed keys is free.
// For V a lane loads DP / 16 consecutive elements of those same eight keys, and the operand of one
// product is one element of each: pairs of 16-bit halves, a byte permutation each.  Row m of product
// i is element DP / 16 * m + i of the head, so a lane's results are consecutive.
//
// Where each key lies (its page, its place in it) is found once for the piece and kept in LDS.
constexpr int kHeadTile = 16;
constexpr int kPieceMost = 1024;

struct Piece {
  int seq, begin, slot, pad;  // tokens [begin, begin + piece) of seq; slot: of the sequence's first piece
};

struct PagedShape {
  int heads, window, piece;
  float scale;
};

// Tokens [first, last) are seen by the query; ok: the pages hold them.
__device__ __forceinline__ bool paged_range(const Cache& c, int b, int n, int window, int& first,
                                            int& last) {
  const bool ok = n >= 0 && n <= (int64_t)(c.indptr[b + 1] - c.indptr[b]) * c.page_size;
  last = ok ? n : 0;
  first = window && last > window ? last - window : 0;
  return ok;
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void attention_paged_kernel(
    Cache c, PagedShape s, const Piece* __restrict__ pieces, const T* __restrict__ k_pages,
    const T* __restrict__ v_pages, const T* __restrict__ q, int64_t q_token, int64_t q_head,
    T* __restrict__ out, int64_t out_token, int64_t out_head, float* __restrict__ lse,
    const int32_t* __restrict__ lengths, float* __restrict__ part_o, f32x2* __restrict__ part_ml) {
  constexpr int E = DP / 16, NS = DP / 32, W = 4;  // elements of V and steps of K a lane; waves
  typedef T VE __attribute__((ext_vector_type(E)));
  __shared__ int64_t s_k[kPieceMost], s_v[kPieceMost];
  __shared__ f32x2 s_ml[W][kHeadTile];
  __shared__ __attribute__((aligned(16))) float s_o[W][kHeadTile][DP + 4];

  const int group = s.heads / c.kv_heads, tiles = (group + kHeadTile - 1) / kHeadTile;
  int id = blockIdx.x;
  const int g = id % c.kv_heads;
  id /= c.kv_heads;
  const int ht = id % tiles;
  const Piece pc = pieces[id / tiles];
  const int b = pc.seq, lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int first, last;
  const bool ok = paged_range(c, b, lengths[b], s.window, first, last);
  const int n_heads = min(kHeadTile, group - ht * kHeadTile), head0 = g * group + ht * kHeadTile;
  // the sequence's pieces in use, and whether this one is
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
      qf[i] = d < c.dim ? scaled_sign<T>(x, s.scale) : V8<T>{};
    }
  }
  const float cs = exp2_scale(s.scale);

  // where the keys lie; those past the end stand for the first one, and weigh nothing
  const int padded = (n + 127) & ~127;
  const int pages = c.indptr[b];
  for (int i = threadIdx.x; i < padded; i += 256) {
    const uint32_t j = begin + (i < n ? i : 0);
    const uint32_t at = j / (uint32_t)c.page_size;
    const int64_t page = n > 0 ? c.indices[pages + at] : 0, slot = j - at * c.page_size;
    s_k[i] = page * c.k_page + slot * c.k_slot;
    s_v[i] = page * c.v_page + slot * c.v_slot;
  }
  __syncthreads();

  const T* kb = k_pages + g * c.k_head;
  const T* vb = v_pages + g * c.v_head;
  V8<T> kf[2][NS];
  VE vf[8];
  auto load_k = [&](int j) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const T* row = kb + s_k[j + 16 * u + col];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int d = 32 * i + 8 * quad;
        kf[u][i] = *reinterpret_cast<const V8<T>*>(row + (d < c.dim ? d : 0));
      }
    }
    if (c.dim < DP) {  // past the head: zeros, as in q, or an infinity there would show
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < NS; ++i) kf[u][i] = 32 * i + 8 * quad < c.dim ? kf[u][i] : V8<T>{};
    }
  };
  const int ve = E * col < c.dim ? E * col : 0;
  auto load_v = [&](int j) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      vf[e] = *reinterpret_cast<const VE*>(vb + s_v[j + 16 * (e / 4) + 4 * quad + e % 4] + ve);
  };

  float top = -INFINITY, sum = 0;
  f32x4 o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = f32x4{};

  int j = 32 * wave;
  if (j < n) load_k(j), load_v(j);
  for (; j < n; j += 32 * W) {
    f32x4 x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      x[u] = f32x4{};
#pragma unroll
      for (int i = 0; i < NS; ++i) x[u] = mfma16(kf[u][i], qf[i], x[u]);
    }
    if (j + 32 * W < n) load_k(j + 32 * W);
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
    // the weights are taken against an older maximum until a head's grows by more than 2^8 of it
    if (__any((m - top) * cs > 8.0f)) {
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      const float now = fmaxf(top, m);
      const float fade = top == -INFINITY ? 0.0f : exp2f((top - now) * cs);
      top = now;
      sum *= fade;
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] *= fade;
    }
    const float base = top == -INFINITY ? 0.0f : top * cs;
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
    if (j + 32 * W < n) load_v(j + 32 * W);
  }

  // join the waves
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  const float ml = top == -INFINITY ? -INFINITY : top * cs;
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
      const int64_t at = ((int64_t)(pc.slot + mine)) * s.heads + head0 + h;
      *reinterpret_cast<f32x4*>(part_o + at * c.dim + d) = y;
      if (d == 0) part_ml[at] = f32x2{most, total};
    } else {
      const float f = total == 0 ? 0.0f : 1.0f / total;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = ok ? y[e] * f : nan;
      *reinterpret_cast<V4<T>*>(out + b * out_token + (head0 + h) * out_head + d) =
          __builtin_convertvector(y, V4<T>);
      if (lse && d == 0)
        lse[(int64_t)b * s.heads + head0 + h] =
            !ok ? nan : total == 0 ? -INFINITY : (most + log2f(total)) * kLn2;
    }
  }
}

// Joins the pieces of sequences that have several: a workgroup a sequence and head, a wave to every
// fourth piece.
template <typename T>
__global__ __launch_bounds__(256) void attention_paged_join_kernel(
    Cache c, PagedShape s, const int32_t* __restrict__ slots, T* __restrict__ out,
    int64_t out_token, int64_t out_head, float* __restrict__ lse,
    const int32_t* __restrict__ lengths, const float* __restrict__ part_o,
    const f32x2* __restrict__ part_ml) {
  __shared__ f32x2 s_ml[4];
  __shared__ f32x2 s_o[4][64];
  const int b = blockIdx.x / s.heads, h = blockIdx.x % s.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int first, last;
  paged_range(c, b, lengths[b], s.window, first, last);
  const int p0 = first / s.piece, p1 = max(p0 + 1, (last + s.piece - 1) / s.piece);
  if (p1 - p0 < 2) return;
  const int64_t at = (int64_t)slots[b] * s.heads + h;
  float most = -INFINITY, total = 0;
  for (int p = p0 + lane; p < p1; p += 64) most = fmaxf(most, part_ml[at + (int64_t)p * s.heads].x);
  most = wave_max(most);
  f32x2 y{};
  const int d = 2 * lane < c.dim ? 2 * lane : 0;
  for (int p = p0 + wave; p < p1; p += 4) {
    const int64_t i = at + (int64_t)p * s.heads;
    const f32x2 v = part_ml[i];
    const float f = v.x == -INFINITY ? 0.0f : exp2f(v.x - most);
    total += f * v.y;
    y += f * *reinterpret_cast<const f32x2*>(part_o + i * c.dim + d);
  }
  if (lane == 0) s_ml[wave] = f32x2{most, total};
  s_o[wave][lane] = y;
  __syncthreads();
  if (wave) return;
  total = s_ml[0].y + s_ml[1].y + s_ml[2].y + s_ml[3].y;
  y = s_o[0][lane] + s_o[1][lane] + s_o[2][lane] + s_o[3][lane];
  const float f = total == 0 ? 0.0f : 1.0f / total;
  if (2 * lane < c.dim) {
    T* to = out + b * out_token + h * out_head + 2 * lane;
    to[0] = (T)(y.x * f);
    to[1] = (T)(y.y * f);
  }
  if (lse && lane == 0) lse[(int64_t)b * s.heads + h] = total == 0 ? -INFINITY : (most + log2f(total)) * kLn2;
}

int check_cache(const fsp_paged_cache& c, const std::string& who) {
  if (!attn_dtype(c.dtype)) return set_error(FSP_ENOTSUP, who + ": dtype");
  if (!attn_dim(c.dim)) return set_error(FSP_ENOTSUP, who + ": dim");
  if (c.kv_heads < 1 || c.page_size < 1 || c.n_pages < 0 || c.batch < 0 || c.table_len < 0)
    return set_error(FSP_EINVAL, who + ": negative or zero size");
  if (c.kv_heads > 0xffff || c.batch > 0x7fffffffLL || c.page_size > 0x7fffffffLL ||
      c.n_pages > 0x7fffffffLL / c.page_size || c.table_len > 0x7fffffffLL / c.page_size)
    return set_error(FSP_EINVAL, who + ": size exceeds 2^31-1 tokens");
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
                      (int)a.interleaved, (int)parts};
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

template <typename T, int DP>
int launch_paged(const fsp_attention_paged_args& a, hipStream_t st) {
  const PagedShape s{(int)a.heads, (int)a.window, (int)a.piece, (float)a.scale};
  float* part_o = static_cast<float*>(a.workspace);
  f32x2* part_ml = reinterpret_cast<f32x2*>(part_o + a.n_pieces * a.heads * a.cache.dim);
  hipLaunchKernelGGL((attention_paged_kernel<T, DP>), dim3((unsigned)paged_workgroups(a)),
                     dim3(256), 0, st, cache_of(a.cache), s,
                     reinterpret_cast<const Piece*>(a.pieces),
                     static_cast<const T*>(a.cache.k_pages),
                     static_cast<const T*>(a.cache.v_pages), static_cast<const T*>(a.q),
                     a.q_token, a.q_head, static_cast<T*>(a.out), a.out_token, a.out_head, a.lse,
                     a.lengths, part_o, part_ml);
  if (int rc = check_hip(hipGetLastError(), "attention_paged_kernel launch")) return rc;
  if (a.n_pieces == a.cache.batch) return FSP_OK;  // a piece each
  hipLaunchKernelGGL((attention_paged_join_kernel<T>), dim3((unsigned)(a.cache.batch * a.heads)),
                     dim3(256), 0, st, cache_of(a.cache), s, a.slots, static_cast<T*>(a.out),
                     a.out_token, a.out_head, a.lse, a.lengths, part_o, part_ml);
  return check_hip(hipGetLastError(), "attention_paged_join_kernel launch");
}

template <typename T>
int launch_paged_dim(const fsp_attention_paged_args& a, hipStream_t st) {
  return a.cache.dim <= 64 ? launch_paged<T, 64>(a, st) : launch_paged<T, 128>(a, st);
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
  // a thousand workgroups, if pieces of 128 tokens (one step of the four waves) give them
  int64_t piece = 128;
  while (piece < kPieceMost && tokens / piece * kv_heads > 1024) piece *= 2;
  return piece;
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
  if (a.window < 0 || a.window > 0x7fffffffLL)
    return set_error(FSP_EINVAL, "fsp_attention_paged: window");
  if (a.piece < 128 || a.piece > kPieceMost || a.piece % 128)
    return set_error(FSP_EINVAL, "fsp_attention_paged: piece must be a multiple of 128 up to 1024");
  if (a.n_pieces < a.cache.batch || a.n_pieces > 0x7fffffffLL || a.cache.batch * a.heads > kMaxBlocks ||
      paged_workgroups(a) > kMaxBlocks)
    return set_error(FSP_EINVAL, "fsp_attention_paged: pieces out of range");
  if (a.cache.batch == 0) return FSP_OK;
  if (!a.q || !a.out || !a.lengths || !a.pieces || !a.slots ||
      (a.n_pieces > a.cache.batch && !a.workspace))
    return set_error(FSP_EINVAL, "fsp_attention_paged: null pointer");
  if (!aligned16(a.q, a.q_token, a.q_head) || !aligned16(a.out, a.out_token, a.out_head) ||
      reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return set_error(FSP_EINVAL, "fsp_attention_paged: rows must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.cache.dtype == FSP_BF16 ? launch_paged_dim<bf16>(a, st) : launch_paged_dim<f16>(a, st);
}
