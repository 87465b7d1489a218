// Moving what a paged cache holds: tokens that stay close up, pages are copied.
#include "paged.hpp"

namespace fsp {
namespace {

constexpr int kThreads = 256;
constexpr int kList = 1024;  // tokens whose places LDS holds at a time

// A sequence's marked tokens, its last ones: rows [begin, begin + count) of the marks, after ``past``
// others.
struct Marked {
  int begin, count, past;
  bool ok;
  __device__ Marked(const int32_t* tokens, int each, int n_tokens, int b, int length, int room) {
    begin = tokens ? tokens[b] : b * each;
    const int end = tokens ? tokens[b + 1] : begin + each;
    ok = begin >= 0 && begin <= end && end <= n_tokens && length >= end - begin && length <= room;
    count = ok ? end - begin : 0;
    past = ok ? length - count : 0;
  }
};

struct KeepShape {
  int n_tokens, each;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;  // of the cache that is written
  const int32_t *indptr, *indices;
  int page_size;
};

// The tokens that stay of [at, at + kList) marks, their places in turn, to LDS; how many.
__device__ __forceinline__ int list_kept(const uint8_t* keep, int at, int count, int* list) {
  __shared__ int s_count[kList / kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t votes[kList / kThreads];
#pragma unroll
  for (int i = 0; i < kList / kThreads; ++i) {
    const int t = at + i * kThreads + (int)threadIdx.x;
    votes[i] = __ballot(t < count && keep[t]);
    if (lane == 0) s_count[i * 4 + wave] = __popcll(votes[i]);
  }
  __syncthreads();
  int total = 0, before[kList / kThreads];
#pragma unroll
  for (int i = 0; i < kList / kWave; ++i) {
    if (i % 4 == wave) before[i / 4] = total;
    total += s_count[i];
  }
#pragma unroll
  for (int i = 0; i < kList / kThreads; ++i)
    if (votes[i] >> lane & 1)
      list[before[i] + __popcll(votes[i] & ((1ull << lane) - 1))] = at + i * kThreads + threadIdx.x;
  __syncthreads();
  return total;
}

// In place, for drafted tokens.  A workgroup takes one sequence, one key head and its keys or values, so that
// nobody else writes what it reads.  The n-th token that stays comes from a place n or later, each from a later
// one than the one before it: rows that are read after others were written are theirs still.  Of the rows of
// one step all are read before any is written.  16 sequences of up to 26 drafted tokens, 8 heads of 128: 3.9 us,
// a chain of dependent loads (offsets -> marks -> pages -> rows).  A long text is a chain of steps of 64 rows (dim
// 128), 1 us each: half of one of 131072 tokens in 2180 us, where other pages take it in 122.
template <typename T>
__global__ __launch_bounds__(kThreads) void paged_keep_kernel(
    Cache c, KeepShape s, T* __restrict__ k_pages, T* __restrict__ v_pages,
    const uint8_t* __restrict__ keep, const int32_t* __restrict__ tokens,
    const int32_t* __restrict__ lengths, int32_t* __restrict__ kept) {
  constexpr int U = 4;
  __shared__ int s_list[kList];
  const int per = 2 * c.kv_heads, b = blockIdx.x / per, which = blockIdx.x % per;
  const bool values = which >= c.kv_heads;
  const int g = values ? which - c.kv_heads : which;
  const int first = c.indptr[b];
  const Marked m(tokens, s.each, s.n_tokens, b, lengths[b], (c.indptr[b + 1] - first) * c.page_size);
  T* pages = values ? v_pages + g * c.v_head : k_pages + g * c.k_head;
  const int64_t page_step = values ? c.v_page : c.k_page, slot_step = values ? c.v_slot : c.k_slot;
  const int chunks = c.dim / 8, rows = kThreads / chunks;  // rows side by side
  const int row = threadIdx.x / chunks, d = threadIdx.x % chunks * 8;
  auto place = [&](int pos) {
    const uint32_t at = (uint32_t)pos / (uint32_t)c.page_size;
    return pages + c.indices[first + at] * page_step + ((uint32_t)pos - at * c.page_size) * slot_step + d;
  };
  int stay = 0;
  for (int at = 0; at < m.count; at += kList) {
    const int n = list_kept(keep + m.begin, at, m.count, s_list);
    for (int i = 0; i < n; i += rows * U) {
      i32x4 x[U];
      int from[U], to[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = min(i + u * rows + row, n - 1);  // one that is another's too is not written twice
        to[u] = m.past + stay + r;
        from[u] = m.past + s_list[r];
        x[u] = *reinterpret_cast<const i32x4*>(place(from[u]));
      }
      all_stored();  // and read
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (row < rows && i + u * rows + row < n && from[u] != to[u])
          *reinterpret_cast<i32x4*>(place(to[u])) = x[u];
    }
    stay += n;
    __syncthreads();
  }
  if (which == 0 && threadIdx.x == 0) kept[b] = m.ok ? m.past + stay : -1;
}

// How many of a sequence's places [from, to) stay, the ``past`` before the marked ones among them: the same in all
// threads.
__device__ __forceinline__ int kept_in(const uint8_t* marks, int past, int from, int to) {
  __shared__ int s_count[kThreads / kWave];
  int count = 0;
  for (int pos = from + (int)threadIdx.x; pos < to; pos += kThreads) count += pos < past || marks[pos - past] != 0;
#pragma unroll
  for (int x = 1; x < kWave; x *= 2) count += __shfl_xor(count, x);
  if ((threadIdx.x & 63) == 0) s_count[threadIdx.x >> 6] = count;
  __syncthreads();
  return s_count[0] + s_count[1] + s_count[2] + s_count[3];
}

// How many tokens of each piece stay, by the slot of its sequence's first one and its place in the sequence.
__global__ __launch_bounds__(kThreads) void paged_keep_count_kernel(
    KeepShape s, const Piece* __restrict__ pieces, int piece_size, const uint8_t* __restrict__ keep,
    const int32_t* __restrict__ tokens, const int32_t* __restrict__ lengths, int32_t* __restrict__ counts) {
  const Piece pc = pieces[blockIdx.x];
  const Marked m(tokens, s.each, s.n_tokens, pc.seq, lengths[pc.seq], pc.room);
  const int64_t end = min((int64_t)pc.begin + piece_size, (int64_t)m.past + m.count);
  const int count = kept_in(keep + m.begin, m.past, pc.begin, (int)end);
  if (threadIdx.x == 0) counts[pc.slot + pc.begin / piece_size] = count;
}

// Each piece's count becomes what stays before it; totals[b]: what stays of sequence b.  A workgroup to a sequence.
__global__ __launch_bounds__(kThreads) void paged_keep_before_kernel(
    Cache c, int piece_size, const int32_t* __restrict__ first_piece, const int32_t* __restrict__ lengths,
    int32_t* __restrict__ counts, int32_t* __restrict__ totals) {
  __shared__ int s_sum[kThreads / kWave];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int room = (c.indptr[b + 1] - c.indptr[b]) * c.page_size;
  const int length = min(max(lengths[b], 0), room);
  const int n = length / piece_size + (length % piece_size > 0);
  int32_t* of = counts + first_piece[b];
  int before = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + (int)threadIdx.x, own = i < n ? of[i] : 0;
    int sum = own;
#pragma unroll
    for (int x = 1; x < kWave; x *= 2) {
      const int other = __shfl_up(sum, x);
      if (lane >= x) sum += other;
    }
    if (lane == 63) s_sum[wave] = sum;
    __syncthreads();
    int here = before;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) {
      if (w < wave) here += s_sum[w];
      before += s_sum[w];
    }
    if (i < n) of[i] = here + sum - own;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[b] = before;
}

// Into other pages: a workgroup takes kSpan of a sequence's tokens, all heads of their keys and values.  How many
// tokens stay before them, and of all, it counts itself, four marks to a word; or, COUNTED, has two launches before
// it count by pieces, as what all workgroups count grows with the square of the marks.  Bound by memory where heads
// are large: half of 16 sequences of 8192, 8 heads of 128, 537 MB in 110 to 125 us, 4.3 to 4.9 TB/s, of 4 of 131072
// 2147 MB in 430 us, 5.0 TB/s, where a plain copy has 4.7 to 4.9; one of 2^20 tokens, one head of 64, 268 MB in 112 us:
// a workgroup moves 16 KB after its chain of loads.  A workgroup to a head of 1024 tokens, whose rows of 256 bytes
// lie apart, took 155 us for the first.
constexpr int kSpan = kWave;

template <typename T, bool COUNTED>
__global__ __launch_bounds__(kThreads) void paged_keep_into_kernel(
    Cache c, KeepShape s, int first_block, const Piece* __restrict__ pieces, int piece_size,
    const T* __restrict__ k_pages, const T* __restrict__ v_pages, T* __restrict__ to_k, T* __restrict__ to_v,
    const uint8_t* __restrict__ keep, const int32_t* __restrict__ tokens,
    const int32_t* __restrict__ lengths, int32_t* __restrict__ kept, const int32_t* __restrict__ counts,
    const int32_t* __restrict__ totals) {
  constexpr int U = 8;
  __shared__ int64_t s_from[2][kSpan], s_to[2][kSpan];  // where keys and values lie, and go
  __shared__ int s_before[4], s_all[4], s_n;
  const int parts = piece_size / kSpan, block = first_block + (int)blockIdx.x;
  const Piece pc = pieces[block / parts];
  const int b = pc.seq, at = pc.begin + block % parts * kSpan;
  const Marked m(tokens, s.each, s.n_tokens, b, lengths[b], pc.room);
  const int length = m.past + m.count;
  if (at >= length && at > 0) return;

  const uint8_t* marks = keep + m.begin;
  int before = 0, all = 0;  // marks that stay
  if constexpr (COUNTED) {
    const int here = kept_in(marks, m.past, pc.begin, min(at, length));
    before = counts[pc.slot + pc.begin / piece_size] + here - min(at, m.past);
    all = m.ok ? totals[b] - m.past : 0;
  } else {
    // whole words of the array that the marks lie in, those of others masked
    const uintptr_t from = reinterpret_cast<uintptr_t>(marks);
    const uint32_t* words = reinterpret_cast<const uint32_t*>(from & ~uintptr_t(3));
    const int skip = (int)(from & 3), stop = at - m.past;
    for (int64_t i = threadIdx.x; 4 * i < (int64_t)m.count + skip; i += kThreads) {
      const int t = (int)(4 * i) - skip;
      uint32_t w;
      if (t >= 0 && t + 4 <= m.count) {
        w = words[i];
      } else {
        w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t + e >= 0 && t + e < m.count) w |= (uint32_t)marks[t + e] << (8 * e);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int one = (w >> (8 * e) & 255) != 0;
        all += one;
        before += t + e < stop ? one : 0;
      }
    }
#pragma unroll
    for (int x = 1; x < kWave; x *= 2) {
      before += __shfl_xor(before, x);
      all += __shfl_xor(all, x);
    }
    if ((threadIdx.x & 63) == 0) {
      s_before[threadIdx.x >> 6] = before;
      s_all[threadIdx.x >> 6] = all;
    }
    __syncthreads();
    before = s_before[0] + s_before[1] + s_before[2] + s_before[3];
    all = s_all[0] + s_all[1] + s_all[2] + s_all[3];
  }
  const int first = s.indptr[b];
  const bool ok = m.ok && m.past + (int64_t)all <= (int64_t)(s.indptr[b + 1] - first) * s.page_size;
  if (at == 0 && threadIdx.x == 0) kept[b] = ok ? m.past + all : -1;
  if (!ok) return;

  if (threadIdx.x < kWave) {
    const int pos = at + threadIdx.x;
    const bool stays = pos < length && (pos < m.past || marks[pos - m.past]);
    const uint64_t votes = __ballot(stays);
    if (stays) {
      const int n = __popcll(votes & ((1ull << threadIdx.x) - 1));
      const uint32_t to = min(at, m.past) + before + n;  // the tokens before the marked ones all stay
      const uint32_t p = (uint32_t)pos / (uint32_t)c.page_size, q = to / (uint32_t)s.page_size;
      const int64_t page = c.indices[pc.page + p], slot = (uint32_t)pos - p * c.page_size;
      const int64_t to_page = s.indices[first + q], to_slot = to - q * s.page_size;
      s_from[0][n] = page * c.k_page + slot * c.k_slot;
      s_from[1][n] = page * c.v_page + slot * c.v_slot;
      s_to[0][n] = to_page * s.k_page + to_slot * s.k_slot;
      s_to[1][n] = to_page * s.v_page + to_slot * s.v_slot;
    }
    if (threadIdx.x == 0) s_n = __popcll(votes);
  }
  __syncthreads();
  const uint32_t chunks = c.dim / 8, line = chunks * c.kv_heads, items = s_n * line;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const T* from = which ? v_pages : k_pages;
    T* to = which ? to_v : to_k;
    const int64_t from_head = which ? c.v_head : c.k_head, to_head = which ? s.v_head : s.k_head;
    for (uint32_t i = threadIdx.x; i < items; i += U * kThreads) {
      i32x4 x[U];
      int64_t off[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t j = min(i + u * kThreads, items - 1), n = j / line, r = j - n * line, h = r / chunks;
        const int d = (r - h * chunks) * 8;
        x[u] = *reinterpret_cast<const i32x4*>(from + s_from[which][n] + h * from_head + d);
        off[u] = s_to[which][n] + h * to_head + d;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < items) *reinterpret_cast<i32x4*>(to + off[u]) = x[u];
    }
  }
}

// Page sources[i] to targets[i], ``parts`` workgroups to the keys or values of one, a vector of eight elements
// a thread and step.  Bound by memory: 4001 pages of 16 tokens, 8 heads of 128, 524 MB in 109 us, 4.8 TB/s, a plain
// copy's rate; 7 pages in 3.0 us, a launch and two dependent loads.
template <typename T>
__global__ __launch_bounds__(kThreads) void paged_copy_kernel(
    Cache c, int n_pages, T* __restrict__ k_pages, T* __restrict__ v_pages,
    const int32_t* __restrict__ sources, const int32_t* __restrict__ targets, int parts) {
  constexpr int U = 4;
  const int part = blockIdx.x % parts, which = blockIdx.x / parts & 1;
  const int64_t i = blockIdx.x / parts / 2;
  const int source = sources[i], target = targets[i];
  if (source < 0 || target < 0 || source >= n_pages || target >= n_pages || source == target) return;
  const int64_t page = which ? c.v_page : c.k_page, slot = which ? c.v_slot : c.k_slot,
                head = which ? c.v_head : c.k_head;
  const T* from = (which ? v_pages : k_pages) + source * page;
  T* to = (which ? v_pages : k_pages) + target * page;
  const uint32_t chunks = c.dim / 8, line = chunks * c.kv_heads, all = line * c.page_size;
  for (uint32_t at = part * kThreads + threadIdx.x; at < all; at += U * parts * kThreads) {
    i32x4 x[U];
    int64_t off[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t j = min(at + u * parts * kThreads, all - 1);
      const uint32_t s = j / line, r = j - s * line, h = r / chunks;
      off[u] = s * slot + h * head + (r - h * chunks) * 8;
      x[u] = *reinterpret_cast<const i32x4*>(from + off[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at + u * parts * kThreads < all) *reinterpret_cast<i32x4*>(to + off[u]) = x[u];
  }
}

// A call's arguments, with the places of counts by pieces, or none.
struct KeepCall : fsp_paged_keep_args {
  const int32_t* first_piece = nullptr;
  int32_t* counts = nullptr;
};

template <typename T>
int launch_keep(const KeepCall& a, hipStream_t st) {
  const fsp_paged_cache& to = a.into;
  const KeepShape s{(int)a.n_tokens, (int)a.each, to.k_page, to.k_slot,       to.k_head,       to.v_page,
                    to.v_slot,       to.v_head,   to.page_indptr, to.page_indices, (int)to.page_size};
  if (!a.other) {
    hipLaunchKernelGGL((paged_keep_kernel<T>), dim3((unsigned)(a.cache.batch * 2 * a.cache.kv_heads)),
                       dim3(kThreads), 0, st, cache_of(a.cache), s, static_cast<T*>(a.cache.k_pages),
                       static_cast<T*>(a.cache.v_pages), a.keep, a.token_indptr, a.lengths, a.kept);
    return check_hip(hipGetLastError(), "paged_keep_kernel launch");
  }
  const Piece* pieces = reinterpret_cast<const Piece*>(a.pieces);
  int32_t* totals = nullptr;
  if (a.counts) {
    totals = a.counts + a.n_pieces;
    hipLaunchKernelGGL(paged_keep_count_kernel, dim3((unsigned)a.n_pieces), dim3(kThreads), 0, st, s, pieces,
                       (int)a.piece, a.keep, a.token_indptr, a.lengths, a.counts);
    if (int rc = check_hip(hipGetLastError(), "paged_keep_count_kernel launch")) return rc;
    hipLaunchKernelGGL(paged_keep_before_kernel, dim3((unsigned)a.cache.batch), dim3(kThreads), 0, st,
                       cache_of(a.cache), (int)a.piece, a.first_piece, a.lengths, a.counts, totals);
    if (int rc = check_hip(hipGetLastError(), "paged_keep_before_kernel launch")) return rc;
  }
  const int64_t blocks = a.n_pieces * (a.piece / kSpan);
  for (int64_t first = 0; first < blocks; first += kMaxBlocks) {  // one launch, but for tables of more than 2^30 tokens
    const int64_t n = blocks - first < kMaxBlocks ? blocks - first : kMaxBlocks;
    hipLaunchKernelGGL((a.counts ? paged_keep_into_kernel<T, true> : paged_keep_into_kernel<T, false>),
                       dim3((unsigned)n), dim3(kThreads), 0, st, cache_of(a.cache), s, (int)first, pieces,
                       (int)a.piece, static_cast<const T*>(a.cache.k_pages),
                       static_cast<const T*>(a.cache.v_pages), static_cast<T*>(to.k_pages),
                       static_cast<T*>(to.v_pages), a.keep, a.token_indptr, a.lengths, a.kept, a.counts, totals);
    if (int rc = check_hip(hipGetLastError(), "paged_keep_into_kernel launch")) return rc;
  }
  return FSP_OK;
}

template <typename T>
int launch_copy(const fsp_paged_cache& c, const int32_t* sources, const int32_t* targets, int64_t n,
                hipStream_t st) {
  const int64_t steps = (c.page_size * c.kv_heads * (c.dim / 8) + kThreads - 1) / kThreads;
  constexpr int64_t kMost = kMaxBlocks / 4;  // pages of a launch
  for (; n > 0; n -= kMost, sources += kMost, targets += kMost) {
    const int64_t here = n < kMost ? n : kMost;
    int64_t parts = (4096 + 2 * here - 1) / (2 * here);
    if (parts > steps) parts = steps;
    hipLaunchKernelGGL((paged_copy_kernel<T>), dim3((unsigned)(2 * here * parts)), dim3(kThreads), 0, st,
                       cache_of(c), (int)c.n_pages, static_cast<T*>(c.k_pages), static_cast<T*>(c.v_pages),
                       sources, targets, (int)parts);
    if (int rc = check_hip(hipGetLastError(), "paged_copy_kernel launch")) return rc;
  }
  return FSP_OK;
}

}  // namespace
}  // namespace fsp

using namespace fsp;

namespace {

int run_keep(const KeepCall& a, const std::string& who, void* stream) {
  if (int rc = check_cache(a.cache, who)) return rc;
  if (a.n_tokens < 0 || a.n_tokens > kAttnTokensCap || a.each < 0 ||
      a.cache.batch > kMaxBlocks / (2 * a.cache.kv_heads))
    return set_error(FSP_EINVAL, who + ": size out of range");
  if (a.cache.batch == 0) return FSP_OK;
  if (!a.token_indptr && (a.each > a.n_tokens / a.cache.batch || a.each * a.cache.batch != a.n_tokens))
    return set_error(FSP_EINVAL, who + ": each tokens per sequence without token_indptr");
  if ((a.n_tokens > 0 && !a.keep) || !a.lengths || !a.kept)
    return set_error(FSP_EINVAL, who + ": null pointer");
  if (a.other) {
    if (int rc = check_cache(a.into, who)) return rc;
    if (a.into.dtype != a.cache.dtype || a.into.kv_heads != a.cache.kv_heads || a.into.dim != a.cache.dim ||
        a.into.batch != a.cache.batch)
      return set_error(FSP_EINVAL, who + ": the caches differ in type, heads, dim or sequences");
    if (a.piece < 128 || a.piece > kList || a.piece % 128 || a.n_pieces < a.cache.batch || !a.pieces ||
        a.n_pieces > kMaxBlocks || a.n_pieces > 0x7fffffff / (a.piece / kSpan) ||
        a.cache.kv_heads * (a.cache.dim / 8) > 0x7fffffff / kSpan)
      return set_error(FSP_EINVAL, who + ": pieces");
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  // rows are moved as they are: one kernel for both types of 16 bits
  return launch_keep<f16>(a, st);
}

}  // namespace

extern "C" int fsp_paged_keep(const fsp_paged_keep_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_paged_keep: null arguments");
  return run_keep({*args}, "fsp_paged_keep", stream);
}

extern "C" int fsp_paged_keep_counted(const fsp_paged_keep_args* args, const int32_t* first_piece, int32_t* counts,
                                      void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_paged_keep_counted: null arguments");
  if (!args->other) return set_error(FSP_EINVAL, "fsp_paged_keep_counted: in place nothing is counted");
  if (args->cache.batch > 0 && (!first_piece || !counts))
    return set_error(FSP_EINVAL, "fsp_paged_keep_counted: null pointer");
  return run_keep({*args, first_piece, counts}, "fsp_paged_keep_counted", stream);
}

extern "C" int fsp_paged_copy(const fsp_paged_cache* cache, const int32_t* sources, const int32_t* targets,
                              int64_t n, void* stream) {
  if (!cache) return set_error(FSP_EINVAL, "fsp_paged_copy: null arguments");
  if (int rc = check_cache(*cache, "fsp_paged_copy")) return rc;
  if (n < 0 || n > 0x7fffffffLL || cache->page_size * cache->kv_heads > (1 << 30) / (cache->dim / 8))
    return set_error(FSP_EINVAL, "fsp_paged_copy: size out of range");
  if (n == 0) return FSP_OK;
  if (!sources || !targets || (cache->n_pages > 0 && (!cache->k_pages || !cache->v_pages)))
    return set_error(FSP_EINVAL, "fsp_paged_copy: null pointer");
  return launch_copy<f16>(*cache, sources, targets, n, static_cast<hipStream_t>(stream));
}
