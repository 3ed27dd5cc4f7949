// Shared by the operators of the fp16 key/value cache: [batch, KV heads, capacity, head_dim], each sequence of a length of its own.
#pragma once
#include "common.h"
#include "extent.h"
#include <type_traits>

namespace trn {

// The keys of a sequence (its new tokens among them) and its new tokens, as they stand on the device; nothing outside the cache or the
// launch is ever addressed by them.
__device__ __forceinline__ int length_of(const int32_t* lengths, int b, int capacity) { return lengths ? min(max(lengths[b], 0), capacity) : capacity; }
__device__ __forceinline__ int count_of(const int32_t* counts, int b, int tokens) { return counts ? min(max(counts[b], 0), tokens) : tokens; }

// The checks of a cache that every entry point makes.
int cache16_check(const trn_cache16* c, bool values = true);
// ... of fp16 rows [batch, heads, tokens, head_dim] on `bytes` bytes; written: no two rows may be one.
int rows16_check(const void* p, const int64_t* st, int64_t b, int64_t h, int64_t s, int bytes, bool written);
// What such rows cover.
inline Extent rows_extent(const void* p, const int64_t* st, int64_t b, int64_t h, int64_t s, int64_t d) { return Extent{p, {b, h, s}, {2 * st[0], 2 * st[1], 2 * st[2]}, 2 * d}; }
// The checks of queries and outputs that an attention makes, behind those of the cache; and of their numbers.
int attn16_check(const trn_cache16* c, const void* q, const void* o, int32_t n_q_heads, int32_t seq_q, const int64_t* q_stride, const int64_t* o_stride, float scale, const void* workspace);
int attn16_rows(int32_t batch, int32_t n_kv_heads, int32_t n_q_heads, int32_t seq_q);

}  // namespace trn
