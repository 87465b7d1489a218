// What the kernels over a paged cache share: the cache, the pieces of its sequences, words between workgroups.
#pragma once

#include "attn.hpp"

namespace fsp {

constexpr int kDrafts = 256;  // drafted tokens of one sequence, at most

struct Cache {
  const int32_t *indptr, *indices;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  int batch, page_size, dim, kv_heads;
};

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

inline int check_cache(const fsp_paged_cache& c, const std::string& who) {
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

inline Cache cache_of(const fsp_paged_cache& c) {
  return {c.page_indptr, c.page_indices, c.k_page, c.k_slot, c.k_head, c.v_page, c.v_slot,
          c.v_head, (int)c.batch, (int)c.page_size, (int)c.dim, (int)c.kv_heads};
}

}  // namespace fsp
