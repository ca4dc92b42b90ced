// The block-scaled KV cache: what the kernels that write, read and attend over it share.
//
// Positions are cut into blocks of P tokens. A complete block of one KV head is P * D int8 codes
// with ONE fp32 scale for the keys and one for the values, in a page of a pool that the table
// [batch, max_blocks] names. The rows of the incomplete block, and of the block before it, are
// held as they came in a ring of 2P rows per sequence and head: position p lives at row p % 2P.
// So a block is quantized once, from the values that arrived, when its last token arrives: the
// stored state depends on the tokens alone, not on how they were cut into calls, and tokens can
// be taken back without loss as far as the ring reaches.
#pragma once

#include "common.cuh"

namespace lq {

// What a launch is about: sequence b has start tokens in the cache before it and adds count.
struct BlockSpan {
  const int64_t* start_dev;
  int64_t start_host;
  const int64_t* count_dev;
  int start_stride;
  int tokens;
};

struct SeqSpan {
  int start, n;
};

enum { LQ_BLOCK_BAD_PAGE = 1, LQ_BLOCK_BAD_POSITION = 2, LQ_BLOCK_BAD_ANGLE = 3, LQ_BLOCK_WAIT = 4 };

// (start, count) of sequence b. A span that leaves the table's positions is treated as no tokens;
// `bad` tells. count is cut to [0, tokens].
__device__ __forceinline__ SeqSpan span_of(const lq_block_kv& c, const BlockSpan& sp, int b, bool& bad) {
  const int64_t start = sp.start_dev != nullptr ? sp.start_dev[(int64_t)b * sp.start_stride] : sp.start_host;
  int64_t n = sp.tokens;
  if (sp.count_dev != nullptr) {
    const int64_t m = sp.count_dev[b];
    n = m < 0 ? 0 : (m < n ? m : n);
  }
  bad = start < 0 || start > (int64_t)c.max_blocks * c.block - n;
  return bad ? SeqSpan{0, 0} : SeqSpan{(int)start, (int)n};
}

// Page of block j of sequence b, or -1 where the table names none of the pool.
__device__ __forceinline__ int64_t page_of(const lq_block_kv& c, int b, int j) {
  const int id = c.table[(int64_t)b * c.max_blocks + j];
  return id >= 0 && id < c.num_pages ? id : -1;
}

// Two 16-bit values in a word, to and from fp32
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t v);
template <>
__device__ __forceinline__ float2 pair_of<__half>(uint32_t v) {
  return __half22float2(as_h2(v));
}
template <>
__device__ __forceinline__ float2 pair_of<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pair_to(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pair_to<__half>(float lo, float hi) {
  return as_u32(__floats2half2_rn(lo, hi));
}
template <>
__device__ __forceinline__ uint32_t pair_to<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Address of the current device's error word (NULL and a message if it cannot be resolved).
int* block_error_word();
// Host checks shared by every entry point that takes a cache.
int check_block_kv(const lq_block_kv* c, const char* what);

}  // namespace lq
