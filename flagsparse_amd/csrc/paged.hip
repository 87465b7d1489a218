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

// One workgroup a token.
template <typename T>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(
    Cache c, T* __restrict__ k_pages, T* __restrict__ v_pages, const T* __restrict__ k,
    int64_t k_token, int64_t k_head, const T* __restrict__ v, int64_t v_token, int64_t v_head,
    const T* __restrict__ q, int64_t q_token, int64_t q_head, T* __restrict__ q_out,
    int64_t qo_token, int64_t qo_head, const float* __restrict__ cos,
    const float* __restrict__ sin, const int32_t* __restrict__ tokens,
    const int32_t* __restrict__ lengths, int heads, int half, int table_rows, int interleaved) {
  const int64_t t = blockIdx.x;
  int b = (int)t;
  int64_t pos;
  bool mine = true;
  if (tokens) {
    int lo = 0, hi = c.batch;  // the last sequence that starts at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tokens[mid] <= t) lo = mid; else hi = mid;
    }
    b = lo;
    mine = tokens[b] <= t && t < tokens[b + 1];
    pos = (int64_t)lengths[b] - tokens[b + 1] + t;
  } else {
    pos = (int64_t)lengths[b] - 1;
  }
  const int first = c.indptr[b], last = c.indptr[b + 1];
  const bool ok = mine && pos >= 0 && pos < (int64_t)(last - first) * c.page_size &&
                  (half == 0 || pos < table_rows);
  const float nan = __builtin_nanf("");
  int64_t page = 0, slot = 0;
  if (ok) {
    page = c.indices[first + pos / c.page_size];
    slot = pos % c.page_size;
  }
  const int per = c.dim;
  for (int i = threadIdx.x; i < (heads + 2 * c.kv_heads) * per; i += kAppendThreads) {
    int h = i / per;
    const int d = i % per;
    const T* row;
    T* to;
    bool turn = true;
    if (h < c.kv_heads) {
      row = k + t * k_token + h * k_head;
      to = k_pages + page * c.k_page + slot * c.k_slot + h * c.k_head;
    } else if (h < 2 * c.kv_heads) {
      h -= c.kv_heads;
      row = v + t * v_token + h * v_head;
      to = v_pages + page * c.v_page + slot * c.v_slot + h * c.v_head;
      turn = false;
    } else {
      h -= 2 * c.kv_heads;
      row = q + t * q_token + h * q_head;
      to = q_out + t * qo_token + h * qo_head;
      if (!ok) to[d] = (T)nan;
    }
    if (!ok) continue;
    float x = (float)row[d];
    if (turn && d < 2 * half) {
      const bool low = interleaved ? !(d & 1) : d < half;
      const int j = interleaved ? d >> 1 : (low ? d : d - half);
      const int mate = interleaved ? (d ^ 1) : (low ? d + half : d - half);
      const float y = (float)row[mate], cs = cos[pos * half + j], sn = sin[pos * half + j];
      x = low ? x * cs - y * sn : y * sn + x * cs;
    }
    to[d] = (T)x;
  }
}

// One wave a query row: 64 keys at a time, a lane to a key for the scores and to elements of the
// head for the products.
template <typename T>
__global__ __launch_bounds__(kWave) void attention_paged_kernel(
    Cache c, const T* __restrict__ k_pages, const T* __restrict__ v_pages,
    const T* __restrict__ q, int64_t q_token, int64_t q_head, T* __restrict__ out,
    int64_t out_token, int64_t out_head, float* __restrict__ lse,
    const int32_t* __restrict__ lengths, int heads, int window, float scale) {
  __shared__ float s_q[kAttnDimCap];
  const int b = blockIdx.x / heads, a = blockIdx.x % heads, lane = threadIdx.x;
  const int g = a / (heads / c.kv_heads);
  const T* qr = q + b * q_token + a * q_head;
  for (int d = lane; d < c.dim; d += kWave) s_q[d] = (float)qr[d];
  __syncthreads();
  const int first = c.indptr[b], last = c.indptr[b + 1], n = lengths[b];
  const bool ok = n >= 0 && n <= (int64_t)(last - first) * c.page_size;
  float m = -INFINITY, l = 0, acc[2] = {0, 0};
  for (int j0 = window && n > window ? n - window : 0; ok && j0 < n; j0 += kWave) {
    const int j = j0 + lane;
    float s = -INFINITY;
    int64_t voff = 0;
    if (j < n) {
      const int64_t page = c.indices[first + j / c.page_size];
      const T* kr = k_pages + page * c.k_page + (j % c.page_size) * c.k_slot + g * c.k_head;
      voff = page * c.v_page + (j % c.page_size) * c.v_slot + g * c.v_head;
      s = 0;
      for (int d = 0; d < c.dim; ++d) s += s_q[d] * (float)kr[d];
      s *= scale;
    }
    const float top = fmaxf(m, wave_max(s));
    const float base = top == -INFINITY ? 0.0f : top;
    const float p = expf(s - base), fade = expf(m - base);
    l = l * fade + wave_add(p);
    acc[0] *= fade;
    acc[1] *= fade;
    m = top;
    for (int e = 0; e < kWave && j0 + e < n; ++e) {
      const float pe = __shfl(p, e);
      const T* vr = v_pages + __shfl(voff, e);
      for (int u = 0; u < 2; ++u)
        if (lane + u * kWave < c.dim) acc[u] += pe * (float)vr[lane + u * kWave];
    }
  }
  T* o = out + b * out_token + a * out_head;
  const float nan = __builtin_nanf("");
  for (int u = 0; u < 2; ++u)
    if (lane + u * kWave < c.dim)
      o[lane + u * kWave] = (T)(!ok ? nan : l > 0 ? acc[u] / l : acc[u]);
  if (lse && lane == 0) lse[(int64_t)b * heads + a] = ok ? m + logf(l) : nan;
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

template <typename T>
int launch_append(const fsp_paged_append_args& a, hipStream_t st) {
  hipLaunchKernelGGL((paged_append_kernel<T>), dim3((unsigned)a.n_tokens), dim3(kAppendThreads), 0,
                     st, cache_of(a.cache), static_cast<T*>(a.cache.k_pages),
                     static_cast<T*>(a.cache.v_pages), static_cast<const T*>(a.k), a.k_token,
                     a.k_head, static_cast<const T*>(a.v), a.v_token, a.v_head,
                     static_cast<const T*>(a.q), a.q_token, a.q_head, static_cast<T*>(a.q_out),
                     a.q_out_token, a.q_out_head, a.cos, a.sin, a.token_indptr, a.lengths,
                     (int)a.heads, (int)a.half, (int)a.table_rows, (int)a.interleaved);
  return check_hip(hipGetLastError(), "paged_append_kernel launch");
}

template <typename T>
int launch_paged(const fsp_attention_paged_args& a, hipStream_t st) {
  hipLaunchKernelGGL((attention_paged_kernel<T>), dim3((unsigned)(a.cache.batch * a.heads)),
                     dim3(kWave), 0, st, cache_of(a.cache),
                     static_cast<const T*>(a.cache.k_pages),
                     static_cast<const T*>(a.cache.v_pages), static_cast<const T*>(a.q),
                     a.q_token, a.q_head, static_cast<T*>(a.out), a.out_token, a.out_head, a.lse,
                     a.lengths, (int)a.heads, (int)a.window, (float)a.scale);
  return check_hip(hipGetLastError(), "attention_paged_kernel launch");
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
  return a.cache.dtype == FSP_BF16 ? launch_append<bf16>(a, st) : launch_append<f16>(a, st);
}

static int check_paged(const fsp_attention_paged_args& a) {
  const char* who = "fsp_attention_paged";
  if (int rc = check_cache(a.cache, who)) return rc;
  if (a.heads < 1 || a.heads % a.cache.kv_heads || a.heads > 0xffff)
    return set_error(FSP_EINVAL, "fsp_attention_paged: heads must be a multiple of kv_heads");
  if (a.window < 0 || a.window > 0x7fffffffLL)
    return set_error(FSP_EINVAL, "fsp_attention_paged: window");
  if (a.cache.batch * a.heads > kMaxBlocks)
    return set_error(FSP_EINVAL, "fsp_attention_paged: more rows than a launch holds");
  return FSP_OK;
}

extern "C" int64_t fsp_attention_paged_workspace(const fsp_attention_paged_args* args) {
  return 0;
}

extern "C" int fsp_attention_paged(const fsp_attention_paged_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_paged: null arguments");
  const fsp_attention_paged_args& a = *args;
  if (int rc = check_paged(a)) return rc;
  if (a.cache.batch == 0) return FSP_OK;
  if (!a.q || !a.out || !a.lengths)
    return set_error(FSP_EINVAL, "fsp_attention_paged: null pointer");
  if (!aligned16(a.q, a.q_token, a.q_head) || !aligned16(a.out, a.out_token, a.out_head))
    return set_error(FSP_EINVAL, "fsp_attention_paged: rows must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.cache.dtype == FSP_BF16 ? launch_paged<bf16>(a, st) : launch_paged<f16>(a, st);
}
