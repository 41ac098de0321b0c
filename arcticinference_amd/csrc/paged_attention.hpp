// What the attention kernels over a paged cache share: the description of a call, which keys a query sees, and the
// cache's element types.
#pragma once

#include "common.hpp"

namespace arctic {

// One call.  Strides in bytes; of the cache's three the innermost is dense.
struct AttentionParams {
  const char *query;
  char *out;
  const char *key_cache, *value_cache;
  const int32_t *table;         // [batch, max_blocks]
  const int32_t *seq_lens;      // [batch]
  const int32_t *query_start;   // [batch + 1], or null: new_tokens queries for every sequence
  const float *k_scale, *v_scale;   // null: 1
  int64_t query_token, query_head, out_token, out_head;
  int64_t key_block, key_token, key_head, value_block, value_token, value_head;
  int64_t table_row;   // elements
  int64_t num_blocks;
  int64_t total_tokens;
  int batch, new_tokens, max_blocks, block_size;
  Divisor by_block, by_new, by_group, by_heads;
  int heads, kv_heads, group, head_size;
  int window, sinks;   // window 0: no limit
  float scale;
};

// A sequence's queries and keys: `length` tokens are in the cache, its `count` queries are the last of them and start
// at row `first` of the query tensor.
struct Sequence {
  int length, count;
  int64_t first;
};

__device__ __forceinline__ int clamped_length(const AttentionParams &p, int b) {
  const int64_t most = min((int64_t)p.max_blocks * p.block_size, (int64_t)0x7fffffff);
  return (int)max((int64_t)0, min((int64_t)p.seq_lens[b], most));
}

// The first position inside the window of a query at `position`: what lies before it is seen only among the sinks.
__device__ __forceinline__ int window_start(const AttentionParams &p, int position) {
  return p.window > 0 ? max(0, position - p.window + 1) : 0;
}

// ---- elements of a query (and of a cache of the query's type), and of an fp8 cache -----------------------------
struct F32 {
  static constexpr int kBytes = 4;
  __device__ static __forceinline__ float load(const char *p) { return *(const ARCTIC_GLOBAL float *)p; }
  __device__ static __forceinline__ void store(char *p, float v) { *(ARCTIC_GLOBAL float *)p = v; }
};
template <typename T>
struct Half {
  static constexpr int kBytes = 2;
  __device__ static __forceinline__ float load(const char *p) { return T::lo(*(const ARCTIC_GLOBAL uint16_t *)p); }
  __device__ static __forceinline__ void store(char *p, float v) { *(ARCTIC_GLOBAL uint16_t *)p = (uint16_t)T::round_bits(v); }
};
struct CacheE4M3 {
  static constexpr int kBytes = 1;
  __device__ static __forceinline__ float load(const char *p) {
    return __builtin_amdgcn_cvt_f32_fp8((int)*(const ARCTIC_GLOBAL uint8_t *)p, 0);
  }
};
struct CacheE5M2 {
  static constexpr int kBytes = 1;
  __device__ static __forceinline__ float load(const char *p) {
    return __builtin_amdgcn_cvt_f32_bf8((int)*(const ARCTIC_GLOBAL uint8_t *)p, 0);
  }
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

}  // namespace arctic
