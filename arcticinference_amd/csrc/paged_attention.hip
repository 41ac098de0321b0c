// Attention of new tokens over a paged key-value cache, gfx950.
//
// The caches are the ones that reshape_and_cache_flash_bulk writes.  Sequence b has L tokens in them, its n queries are
// the last n; the query at position p sees the keys j <= p that lie in its window (j > p - window) or among the first
// `sinks` tokens:
//   s_j = scale k_scale <q, K_j>,   out = v_scale sum_j exp(s_j - m) V_j / sum_j exp(s_j - m),   m = max_j s_j
// A query that sees nothing answers zeros.  A page outside the cache holds no keys.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "paged_attention_many.hpp"

namespace arctic {

// Any head size up to 512, any type, alignment and stride: a workgroup per query and head, whose waves take 64 keys each in
// turn.  Every lane takes the product of one key with the query, the running maximum and sum are the wave's, then every lane
// adds the weighted values of its elements, key by key; the waves' parts are joined in LDS.  A key that is not seen is not
// read, so what it holds does not matter.  Bound by loads of single elements, a row a lane: fp32, 32 heads over 8 x 128, one
// sequence of 777 keys 43 us (four waves 64, one 278), 64 of 2000 736 us, 1.4 TB/s (753, 2022); four prompts of 300 tokens
// with 8 heads 574 us (four waves 511).
constexpr int kGeneralMostHead = 512, kGeneralWaves = 8;

template <typename Q, typename C>
__global__ __launch_bounds__(64 * kGeneralWaves) void attention_general_kernel(const AttentionParams p) {
  __shared__ float query[kGeneralMostHead];
  __shared__ float parts[kGeneralWaves][kGeneralMostHead], statistics[kGeneralWaves][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const uint32_t unit = blockIdx.y * gridDim.x + blockIdx.x;
  if (unit >= (uint32_t)p.total_tokens * (uint32_t)p.heads) return;
  const uint32_t token = p.by_heads.quotient(unit);
  const int head = (int)(unit - token * (uint32_t)p.heads);
  int b, count, first;
  if (p.query_start) {
    int lo = 0, hi = p.batch;   // the last sequence that starts at or before this row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.query_start[mid] <= (int)token) lo = mid;
      else hi = mid;
    }
    b = lo;
    first = p.query_start[b];
    count = p.query_start[b + 1] - first;
    if (first < 0 || (int)token < first || (int)token - first >= count) return;   // a row of no sequence
  } else {
    b = (int)p.by_new.quotient(token);
    first = b * p.new_tokens;
    count = p.new_tokens;
  }
  const int position = clamped_length(p, b) - count + ((int)token - first);
  const int kv_head = (int)p.by_group.quotient((uint32_t)head);
  const int D = p.head_size;
  const char *q = p.query + (int64_t)token * p.query_token + (int64_t)head * p.query_head;
  for (int d = threadIdx.x; d < D; d += 64 * kGeneralWaves) query[d] = Q::load(q + (int64_t)d * Q::kBytes);
  __syncthreads();
  const float scale = p.scale * (p.k_scale ? *p.k_scale : 1.f);
  const int start = window_start(p, position);
  const int sinks = min(p.sinks, start);
  const int keys = position < 0 ? 0 : sinks + (position - start + 1);
  float acc[kGeneralMostHead / 64] = {};
  float m = -__builtin_inff(), sum = 0.f;
  for (int k0 = 64 * wave; k0 < keys; k0 += 64 * kGeneralWaves) {
    const int k = k0 + lane;
    float s = -__builtin_inff();
    int64_t at = -1;
    if (k < keys) {
      const int j = k < sinks ? k : start + (k - sinks);
      const int block = (int)p.by_block.quotient((uint32_t)j);
      const int64_t page = p.table[(int64_t)b * p.table_row + block];
      if (page >= 0 && page < p.num_blocks) {
        const int off = j - block * p.block_size;
        const char *key = p.key_cache + page * p.key_block + (int64_t)off * p.key_token + (int64_t)kv_head * p.key_head;
        at = page * p.value_block + (int64_t)off * p.value_token + (int64_t)kv_head * p.value_head;
        float dot = 0.f;
#pragma unroll 8
        for (int d = 0; d < D; ++d) dot = fmaf(query[d], C::load(key + (int64_t)d * C::kBytes), dot);
        s = dot * scale;
      }
    }
    const bool nan = __any(s != s);
    const float top = nan ? __builtin_nanf("") : fmaxf(m, wave_max(s));
    const float base = top == -__builtin_inff() ? 0.f : top;
    const float w = at < 0 ? 0.f : __expf(s - base);
    const float keep = __expf(m - base);
    float chunk = w;
#pragma unroll
    for (int d = 32; d; d >>= 1) chunk += __shfl_xor(chunk, d);
    sum = sum * keep + chunk;
    m = top;
#pragma unroll
    for (int i = 0; i < kGeneralMostHead / 64; ++i) acc[i] *= keep;
    const int n = min(64, keys - k0);
    for (int k = 0; k < n; k += 4) {   // four keys' values are requested before the first is used
      float value[4][kGeneralMostHead / 64], of[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int from = min(k + a, 63);   // (beyond the last key no lane has one)
        const uint32_t high = (uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), from), low = (uint32_t)__builtin_amdgcn_readlane((int)at, from);
        const int64_t place = (int64_t)((uint64_t)high << 32 | low);
        of[a] = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(w), from));
#pragma unroll
        for (int i = 0; i < kGeneralMostHead / 64; ++i) {
          value[a][i] = 0.f;
          if (place >= 0 && k + a < n && lane + 64 * i < D)
            value[a][i] = C::load(p.value_cache + place + ((int64_t)lane + 64 * i) * C::kBytes);
        }
        if (place < 0 || k + a >= n) of[a] = 0.f;
      }
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int i = 0; i < kGeneralMostHead / 64; ++i) acc[i] = fmaf(of[a], value[a][i], acc[i]);
    }
  }
  if (lane == 0) statistics[wave][0] = m, statistics[wave][1] = sum;
#pragma unroll
  for (int i = 0; i < kGeneralMostHead / 64; ++i) parts[wave][lane + 64 * i] = acc[i];
  __syncthreads();
  bool nan = false;
  float top = -__builtin_inff(), all = 0.f;
#pragma unroll
  for (int v = 0; v < kGeneralWaves; ++v) {
    nan |= statistics[v][0] != statistics[v][0];
    top = fmaxf(top, statistics[v][0]);
  }
  const float base = nan ? __builtin_nanf("") : top == -__builtin_inff() ? 0.f : top;
  float share[kGeneralWaves];
#pragma unroll
  for (int v = 0; v < kGeneralWaves; ++v) {
    share[v] = __expf(statistics[v][0] - base);
    all = fmaf(statistics[v][1], share[v], all);
  }
  const float norm = all == 0.f ? 0.f : (p.v_scale ? *p.v_scale : 1.f) / all;
  char *out = p.out + (int64_t)token * p.out_token + (int64_t)head * p.out_head;
  for (int d = threadIdx.x; d < D; d += 64 * kGeneralWaves) {
    float o = 0.f;
#pragma unroll
    for (int v = 0; v < kGeneralWaves; ++v) o = fmaf(parts[v][d], share[v], o);
    Q::store(out + (int64_t)d * Q::kBytes, o * norm);
  }
}

}  // namespace arctic

using namespace arctic;

// The checks that both entry points share, and the call's description for the kernels.
static int describe(const char *fn, AttentionParams &p, void *out, const void *query, const arctic_paged_cache *cache,
                    const int32_t *block_table, const int32_t *seq_lens, int64_t batch, int64_t max_blocks,
                    int64_t table_stride, int64_t total_tokens, int num_heads, int64_t query_token_stride,
                    int64_t query_head_stride, int64_t out_token_stride, int64_t out_head_stride, float scale,
                    int64_t window, int64_t num_sinks, int dtype) {
  if (dtype != ARCTIC_DTYPE_F32 && dtype != ARCTIC_DTYPE_F16 && dtype != ARCTIC_DTYPE_BF16)
    return fail(ARCTIC_ERR_UNSUPPORTED, "%s: queries must be fp32, fp16 or bf16", fn);
  if (!cache) return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: null cache description", fn);
  const arctic_paged_cache &c = *cache;
  if (c.kv_cache_dtype != ARCTIC_KV_AUTO && c.kv_cache_dtype != ARCTIC_KV_FP8_E4M3 && c.kv_cache_dtype != ARCTIC_KV_FP8_E5M2)
    return fail(ARCTIC_ERR_UNSUPPORTED, "%s: Unsupported data type of kv cache: code %d", fn, c.kv_cache_dtype);
  if (batch < 0 || total_tokens < 0 || num_heads <= 0 || c.num_kv_heads <= 0 || c.head_size <= 0 || c.block_size <= 0 ||
      max_blocks < 0 || c.num_blocks < 0)
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: sizes must be positive", fn);
  if (num_heads % c.num_kv_heads)
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: num_heads (%d) must be a multiple of num_kv_heads (%d)", fn, num_heads,
                c.num_kv_heads);
  if (c.head_size > kGeneralMostHead)
    return fail(ARCTIC_ERR_UNSUPPORTED, "%s: head_size must be at most %d", fn, kGeneralMostHead);
  if (batch > 0x7ffffffeLL || total_tokens > 0x7fffffffLL || num_heads > (1 << 20) || c.block_size > (1 << 20) ||
      c.num_blocks > ((int64_t)1 << 31) || max_blocks > 0x7fffffffLL || total_tokens * num_heads > 0x7fffffffLL)
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: batch, tokens, tokens * num_heads, max_blocks or num_blocks beyond 2^31, "
                "num_heads or block_size beyond 2^20", fn);
  if (window < 0 || num_sinks < 0)
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: window and num_sinks must not be negative", fn);
  const int es = dtype == ARCTIC_DTYPE_F32 ? 4 : 2, cs = c.kv_cache_dtype == ARCTIC_KV_AUTO ? es : 1;
  if (!pitch_ok(query_token_stride, total_tokens, es) || !pitch_ok(query_head_stride, num_heads, es) ||
      !pitch_ok(out_token_stride, total_tokens, es) || !pitch_ok(out_head_stride, num_heads, es) ||
      !pitch_ok(c.key_block_stride, c.num_blocks, cs) || !pitch_ok(c.key_token_stride, c.block_size, cs) ||
      !pitch_ok(c.key_head_stride, c.num_kv_heads, cs) || !pitch_ok(c.value_block_stride, c.num_blocks, cs) ||
      !pitch_ok(c.value_token_stride, c.block_size, cs) || !pitch_ok(c.value_head_stride, c.num_kv_heads, cs) ||
      !pitch_ok(table_stride, batch, 4))
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: query, output, cache or table pitch out of range", fn);
  if (batch == 0 || total_tokens == 0) return ARCTIC_OK;
  if (!out || !query || !seq_lens || (max_blocks > 0 && !block_table) || (c.num_blocks > 0 && (!c.key_cache || !c.value_cache)))
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", fn);
  if (c.kv_cache_dtype != ARCTIC_KV_AUTO && (!c.k_scale || !c.v_scale))
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: an fp8 cache needs k_scale and v_scale", fn);
  if (((uintptr_t)out | (uintptr_t)query) % es ||
      ((uintptr_t)c.key_cache | (uintptr_t)c.value_cache) % cs || ((uintptr_t)block_table | (uintptr_t)seq_lens) % 4)
    return fail(ARCTIC_ERR_UNSUPPORTED, "%s: a tensor does not start at a multiple of its element size", fn);
  const bool quantised = c.kv_cache_dtype != ARCTIC_KV_AUTO;
  p.query = (const char *)query;
  p.out = (char *)out;
  p.key_cache = (const char *)c.key_cache;
  p.value_cache = (const char *)c.value_cache;
  p.table = block_table;
  p.seq_lens = seq_lens;
  p.query_start = nullptr;
  p.k_scale = quantised ? c.k_scale : nullptr;
  p.v_scale = quantised ? c.v_scale : nullptr;
  p.query_token = query_token_stride * es;
  p.query_head = query_head_stride * es;
  p.out_token = out_token_stride * es;
  p.out_head = out_head_stride * es;
  p.key_block = c.key_block_stride * cs;
  p.key_token = c.key_token_stride * cs;
  p.key_head = c.key_head_stride * cs;
  p.value_block = c.value_block_stride * cs;
  p.value_token = c.value_token_stride * cs;
  p.value_head = c.value_head_stride * cs;
  p.table_row = table_stride;
  p.num_blocks = c.num_blocks;
  p.total_tokens = total_tokens;
  p.batch = (int)batch;
  p.new_tokens = 0;
  p.max_blocks = (int)max_blocks;
  p.block_size = c.block_size;
  p.heads = num_heads;
  p.kv_heads = c.num_kv_heads;
  p.group = num_heads / c.num_kv_heads;
  p.head_size = c.head_size;
  p.window = (int)(window > 0x7fffffffLL ? 0 : window);   // every position is below 2^31
  p.sinks = (int)(num_sinks > 0x7fffffffLL ? 0x7fffffffLL : num_sinks);
  p.scale = scale;
  p.by_block = Divisor((uint32_t)c.block_size);
  p.by_group = Divisor((uint32_t)p.group);
  p.by_heads = Divisor((uint32_t)num_heads);
  p.by_new = Divisor(1);
  return ARCTIC_OK;
}

template <typename Q>
static void launch_general(const AttentionParams &p, int kv, hipStream_t s) {
  // a launch has fewer than 2^32 lanes along an axis
  constexpr int64_t kMost = 1 << 22;
  const int64_t units = p.total_tokens * p.heads;
  const dim3 grid((unsigned)std::min(units, kMost), (unsigned)((units + kMost - 1) / kMost));
  if (kv == ARCTIC_KV_AUTO) launch(attention_general_kernel<Q, Q>, grid, 64 * kGeneralWaves, s, p);
  else if (kv == ARCTIC_KV_FP8_E4M3) launch(attention_general_kernel<Q, CacheE4M3>, grid, 64 * kGeneralWaves, s, p);
  else launch(attention_general_kernel<Q, CacheE5M2>, grid, 64 * kGeneralWaves, s, p);
}

static int run_attention(const char *fn, const AttentionParams &p, int dtype, int kv, hipStream_t s) {
  if (dtype == ARCTIC_DTYPE_F32) launch_general<F32>(p, kv, s);
  else if (dtype == ARCTIC_DTYPE_F16) launch_general<Half<F16>>(p, kv, s);
  else launch_general<Half<BF16>>(p, kv, s);
  return check_launch(fn);
}

// ---- few new tokens of each sequence ---------------------------------------------------------------------------

// Tiles of 32 keys that a sequence has at most, as far as max_seq_len says.
static int64_t most_tiles(int64_t max_seq_len, int64_t new_tokens, int64_t window, int64_t num_sinks) {
  const int64_t length = std::min(max_seq_len, (int64_t)0x7fffffff);
  const int64_t all = (length + 31) / 32;
  if (window <= 0 || window > length) return std::max<int64_t>(all, 1);
  return std::max<int64_t>(1, std::min(all, (std::min(num_sinks, length) + 31) / 32 + (window + new_tokens + 62) / 32));
}

static bool few_shape(FewShape &f, int64_t batch, int64_t new_tokens, int num_heads, const arctic_paged_cache &c,
                      int64_t max_seq_len, int64_t window, int64_t num_sinks, int dtype) {
  if (dtype == ARCTIC_DTYPE_F32 || c.head_size > 256 || c.head_size % (c.kv_cache_dtype == ARCTIC_KV_AUTO ? 8 : 16)) return false;
  const int64_t rows = new_tokens * (num_heads / c.num_kv_heads);
  f.padded = c.head_size <= 64 ? 64 : c.head_size <= 128 ? 128 : 256;
  f.columns = rows <= 16 ? 1 : rows <= 32 || f.padded > 64 ? 2 : 4;
  const int64_t row_tiles = (rows + 16 * f.columns - 1) / (16 * f.columns);
  f.plain = c.head_size == f.padded && c.block_size % 16 == 0;
  // rows of 128 bytes and less of neighbouring heads are read together
  const int row_bytes = f.padded * (c.kv_cache_dtype == ARCTIC_KV_AUTO ? 2 : 1);
  f.heads = row_bytes <= 64 && f.plain && c.num_kv_heads % 4 == 0 ? 4 : row_bytes == 128 && f.plain && c.num_kv_heads % 2 == 0 ? 2 : 1;
  f.row_tiles = (int)row_tiles;
  const int64_t tiles = most_tiles(max_seq_len, new_tokens, window, num_sinks), units = (c.num_kv_heads / f.heads) * row_tiles;
  // Two workgroups for every CU, all alike, read at the rate that a large read reaches; four lose 5 to 10 % (64 sequences of
  // 2048 to 8192 keys, 8 heads x 128: fp8 136 us / 152, bf16 259 / 273).  A piece has four tiles at least (one sequence of 777
  // keys: 9.8 us, with eight 10.2).  Sequences of few tiles are not worth the join; how many that is depends on the CUs that
  // would idle.  Whole / dealt, 32 heads over 8, us: 16 of 1000 keys (128 workgroups) 17.2 / 20.1, of 777 15.6 / 16.8; 4 of
  // 1000 15.0 / 10.9; 32 of 1500 (256 workgroups) 33.3 / 37.7, fp8 64 of 1500 34.8 / 40.7; 4 of 1500 19.1 / 12.6.
  constexpr int64_t kWorkgroups = 512, kLeast = 4;
  const int64_t whole = batch * units >= 256 ? 64 : batch * units >= 128 ? 32 : 16;
  if (tiles <= whole) {
    f.workers = (int)batch;
    f.least = 0;
  } else {
    f.least = (int)kLeast;
    f.workers = (int)std::max<int64_t>(1, std::min((kWorkgroups + units - 1) / units, batch * ((tiles + kLeast - 1) / kLeast)));
  }
  // fewer than 2^32 lanes in either launch (a wave joins a row)
  return units * f.workers <= 0xffffffLL && batch * new_tokens * num_heads <= 0x3ffffffLL;
}

// What a lane of few_launch's kernels loads or stores at once, and the 32-bit offsets of a block's 16 tokens.
static bool few_takes(const AttentionParams &p) {
  const uint64_t wide = (uintptr_t)p.query | p.query_token | p.query_head | (uintptr_t)p.out | p.out_token | p.out_head |
                        (uintptr_t)p.key_cache | p.key_block | p.key_token | p.key_head | (uintptr_t)p.value_cache |
                        p.value_block | p.value_token | p.value_head;
  return wide % 16 == 0 && p.key_token < (1 << 26) && p.value_token < (1 << 26) && p.num_blocks > 0 && p.max_blocks > 0;
}

// ... and in the kernel for many tokens a block's stride and what lies inside one have 32 bits.
static bool many_takes(const AttentionParams &p) {
  return few_takes(p) && p.key_block <= 0xffffffffLL && p.value_block <= 0xffffffffLL &&
         p.key_token * p.block_size <= 0xffffffffLL && p.value_token * p.block_size <= 0xffffffffLL;
}

static int64_t few_bytes(const FewShape &f, int64_t batch, int64_t new_tokens, int num_heads, int head_size) {
  return f.least == 0 ? 0 : new_tokens * num_heads * 2 * f.workers * ((int64_t)head_size + 2) * 4 + batch * (int64_t)sizeof(int2);
}

// ---- many ------------------------------------------------------------------------------------------------------

// `total_tokens` query tokens of `batch` sequences, new_tokens of each or (0) ragged.
static bool many_shape(ManyShape &f, int64_t batch, int64_t new_tokens, int64_t total_tokens, int num_heads,
                       const arctic_paged_cache &c, int64_t max_seq_len, int64_t window, int64_t num_sinks, int dtype) {
  if (dtype == ARCTIC_DTYPE_F32 || c.head_size > 256 || c.head_size % (c.kv_cache_dtype == ARCTIC_KV_AUTO ? 8 : 16)) return false;
  const int64_t group = num_heads / c.num_kv_heads, rows = total_tokens * group;
  f.padded = c.head_size <= 64 ? 64 : c.head_size <= 128 ? 128 : 256;
  f.per_sequence = (int)std::min<int64_t>((new_tokens * group + kManyRows - 1) / kManyRows, 0x7fffffff);
  f.slots = new_tokens ? batch * f.per_sequence : rows / kManyRows + batch;
  // The row tiles that there are for sure: rows / kManyRows.  A CU has two workgroups at a time, and those of long and short
  // sequences, of a sequence's first and last rows differ: splits that make four for a CU even them out (two chunks of up to
  // 512 tokens behind up to 24000 keys, 64 heads over 8: 647 us; two for a CU 705, eight 632 with twice the workspace).  A
  // split of fewer than 8 tiles is not worth the join.
  const int64_t units = std::max<int64_t>(1, rows / kManyRows) * c.num_kv_heads;
  const int64_t keys = many_keys(f.padded), tiles = (most_tiles(max_seq_len, kManyRows / group + 1, window, num_sinks) * 32 + keys - 1) / keys;
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(1024 / units, (tiles + 7) / 8));
  f.tiles_per_split = (int)((tiles + splits - 1) / splits);
  f.splits = (int)((tiles + f.tiles_per_split - 1) / f.tiles_per_split);
  return f.slots * f.splits * c.num_kv_heads <= 0xffffffLL;   // fewer than 2^32 lanes
}

static int64_t many_bytes(const ManyShape &f, int num_kv_heads, int head_size) {
  return f.splits == 1 ? 0 : f.slots * num_kv_heads * f.splits * kManyRows * ((int64_t)head_size + 2) * 4;
}

static int workspace_error(const char *fn, int64_t need) {
  return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned and hold %lld bytes", fn, (long long)need);
}

static int run_many(const char *fn, const AttentionParams &p, const ManyShape &f, int dtype, int kv, void *workspace,
                    int64_t workspace_bytes, hipStream_t s) {
  const int64_t need = many_bytes(f, p.kv_heads, p.head_size);
  if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)) return workspace_error(fn, need);
  ManyParams mp;
  mp.a = p;
  mp.slots = (int)f.slots;
  mp.splits = f.splits;
  mp.tiles_per_split = f.tiles_per_split;
  mp.per_sequence = f.per_sequence;
  mp.by_kv_heads = Divisor((uint32_t)p.kv_heads);
  mp.by_splits = Divisor((uint32_t)f.splits);
  mp.by_per_sequence = Divisor((uint32_t)std::max(1, f.per_sequence));
  mp.by_group = Divisor((uint32_t)p.group);
  mp.partial = need ? (float *)workspace : nullptr;
  mp.statistics = need ? mp.partial + f.slots * p.kv_heads * f.splits * kManyRows * p.head_size : nullptr;
  if (dtype == ARCTIC_DTYPE_BF16) many_launch_bf16(mp, f, kv, s);
  else many_launch_f16(mp, f, kv, s);
  return check_launch(fn);
}

// Query rows of a key head beyond which the kernel for many tokens is the faster one.  32 heads over 8, few / many tokens, us:
//                     16 x 2000 keys, 48 rows   48 x 4000, 32 rows   48 x 4000, 48 rows   4 x 32000, 64 rows
//   128, 16 bits      87 / 34                   176 / 194            235 / 207            164 / 184
//   128, fp8          63 / 32                   105 / 137            171 / 156            122 / 134
//   256, 16 bits      165 / 100                 465 / 470            681 / 487            441 / 354
//   256, fp8          90 / 92                   204 / 417            301 / 443            193 / 324
//   64, 16 bits       33 / 26                   101 / 108            105 / 117            65 / 104
static int64_t most_few_rows(const arctic_paged_cache &c) {
  return c.head_size <= 64 || (c.head_size > 128 && c.kv_cache_dtype != ARCTIC_KV_AUTO) ? 64 : 32;
}

extern "C" int64_t arctic_paged_attention_workspace_bytes(int64_t batch, int new_tokens, int num_heads,
                                                          const arctic_paged_cache *cache, int64_t max_seq_len,
                                                          int64_t window, int64_t num_sinks, int dtype) {
  // (what the call itself would refuse needs none)
  if (!cache || batch <= 0 || new_tokens <= 0 || batch > 0x7fffffffLL / new_tokens || num_heads <= 0 || num_heads > (1 << 20) ||
      cache->num_kv_heads <= 0 || num_heads % cache->num_kv_heads || cache->head_size <= 0 || cache->block_size <= 0 || max_seq_len < 0 ||
      window < 0 || num_sinks < 0 || batch * new_tokens > 0x7fffffffLL / num_heads)
    return 0;
  FewShape f;
  ManyShape m;
  if (new_tokens * (int64_t)(num_heads / cache->num_kv_heads) > most_few_rows(*cache))
    return many_shape(m, batch, new_tokens, batch * new_tokens, num_heads, *cache, max_seq_len, window, num_sinks, dtype)
               ? many_bytes(m, cache->num_kv_heads, cache->head_size)
               : 0;
  return few_shape(f, batch, new_tokens, num_heads, *cache, max_seq_len, window, num_sinks, dtype)
             ? few_bytes(f, batch, new_tokens, num_heads, cache->head_size)
             : 0;
}

extern "C" int arctic_paged_attention(void *out, const void *query, const arctic_paged_cache *cache,
                                      const int32_t *block_table, const int32_t *seq_lens, int64_t batch, int new_tokens,
                                      int num_heads, int64_t max_blocks, int64_t table_stride,
                                      int64_t query_token_stride, int64_t query_head_stride, int64_t out_token_stride,
                                      int64_t out_head_stride, float scale, int64_t max_seq_len, int64_t window,
                                      int64_t num_sinks, int dtype, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *fn = "paged_attention";
  if (new_tokens < 0 || batch < 0 || (new_tokens > 0 && batch > 0x7fffffffLL / new_tokens))
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: batch and new_tokens must not be negative, nor their product beyond 2^31", fn);
  AttentionParams p;
  const int rc = describe(fn, p, out, query, cache, block_table, seq_lens, batch, max_blocks, table_stride, batch * new_tokens,
                          num_heads, query_token_stride, query_head_stride, out_token_stride, out_head_stride, scale, window,
                          num_sinks, dtype);
  if (rc != ARCTIC_OK || batch == 0 || new_tokens == 0) return rc;
  if (max_seq_len < 0) return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: max_seq_len must not be negative", fn);
  p.new_tokens = new_tokens;
  p.by_new = Divisor((uint32_t)new_tokens);
  FewShape f;
  ManyShape m;
  if ((int64_t)new_tokens * p.group > most_few_rows(*cache)) {
    if (many_takes(p) && many_shape(m, batch, new_tokens, p.total_tokens, num_heads, *cache, max_seq_len, window, num_sinks, dtype))
      return run_many(fn, p, m, dtype, cache->kv_cache_dtype, workspace, workspace_bytes, (hipStream_t)stream);
  } else if (few_takes(p) && few_shape(f, batch, new_tokens, num_heads, *cache, max_seq_len, window, num_sinks, dtype)) {
    const int64_t need = few_bytes(f, batch, new_tokens, num_heads, cache->head_size);
    if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)) return workspace_error(fn, need);
    FewParams fp;
    fp.a = p;
    fp.rows = new_tokens * p.group;
    fp.row_tiles = f.row_tiles;
    fp.workers = f.workers;
    fp.least = f.least;
    fp.by_row_tiles = Divisor((uint32_t)f.row_tiles);
    fp.by_head_groups = Divisor((uint32_t)(p.kv_heads / f.heads));
    fp.partial = (float *)workspace;
    const int64_t pieces = (int64_t)new_tokens * num_heads * 2 * f.workers;
    fp.statistics = need ? fp.partial + pieces * p.head_size : nullptr;
    fp.dealt = need ? (int2 *)(fp.statistics + pieces * 2) : nullptr;
    if (dtype == ARCTIC_DTYPE_BF16) few_launch_bf16(fp, f, cache->kv_cache_dtype, (hipStream_t)stream);
    else few_launch_f16(fp, f, cache->kv_cache_dtype, (hipStream_t)stream);
    return check_launch(fn);
  }
  return run_attention(fn, p, dtype, cache->kv_cache_dtype, (hipStream_t)stream);
}

extern "C" int64_t arctic_paged_attention_ragged_workspace_bytes(int64_t batch, int64_t total_tokens, int num_heads,
                                                                 const arctic_paged_cache *cache, int64_t max_seq_len,
                                                                 int64_t window, int64_t num_sinks, int dtype) {
  if (!cache || batch <= 0 || batch > 0x7ffffffeLL || total_tokens <= 0 || num_heads <= 0 || num_heads > (1 << 20) ||
      cache->num_kv_heads <= 0 || num_heads % cache->num_kv_heads || cache->head_size <= 0 || cache->block_size <= 0 || max_seq_len < 0 ||
      window < 0 || num_sinks < 0 || total_tokens > 0x7fffffffLL / num_heads)
    return 0;
  ManyShape m;
  return many_shape(m, batch, 0, total_tokens, num_heads, *cache, max_seq_len, window, num_sinks, dtype)
             ? many_bytes(m, cache->num_kv_heads, cache->head_size)
             : 0;
}

extern "C" int arctic_paged_attention_ragged(void *out, const void *query, const int32_t *query_start,
                                             const arctic_paged_cache *cache, const int32_t *block_table,
                                             const int32_t *seq_lens, int64_t batch, int64_t total_tokens, int num_heads,
                                             int64_t max_blocks, int64_t table_stride, int64_t query_token_stride,
                                             int64_t query_head_stride, int64_t out_token_stride, int64_t out_head_stride,
                                             float scale, int64_t max_seq_len, int64_t window, int64_t num_sinks, int dtype,
                                             void *workspace, int64_t workspace_bytes, void *stream) {
  const char *fn = "paged_attention_ragged";
  AttentionParams p;
  const int rc = describe(fn, p, out, query, cache, block_table, seq_lens, batch, max_blocks, table_stride, total_tokens,
                          num_heads, query_token_stride, query_head_stride, out_token_stride, out_head_stride, scale, window,
                          num_sinks, dtype);
  if (rc != ARCTIC_OK || batch == 0 || total_tokens == 0) return rc;
  if (!query_start || (uintptr_t)query_start % 4)
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: query_start is missing or not aligned", fn);
  if (max_seq_len < 0) return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: max_seq_len must not be negative", fn);
  p.query_start = query_start;
  ManyShape m;
  if (many_takes(p) && many_shape(m, batch, 0, total_tokens, num_heads, *cache, max_seq_len, window, num_sinks, dtype))
    return run_many(fn, p, m, dtype, cache->kv_cache_dtype, workspace, workspace_bytes, (hipStream_t)stream);
  return run_attention(fn, p, dtype, cache->kv_cache_dtype, (hipStream_t)stream);
}
