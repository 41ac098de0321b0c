// Attention of many new tokens of a sequence: a workgroup of four waves per key head and tile of query rows (token by token,
// head by head of the key head's group), 32 rows a wave, over the keys that any of them sees, 64 at a time.
//
// What bounds it is the matrix cores, so K and V are read from the cache once for all waves, widened to 16 bits and kept
// in LDS twice, one tile ahead.  Query rows are the columns of both products (32x32x16):
//   S^T = K Q^T,   O^T = V^T P^T.
// The scores leave the first one with 4 x 4 consecutive keys of one row in a lane; laid over the keys to suit, the second
// one's contraction takes them as they are, and V's operand, 4 consecutive keys of one element at a time, is what the
// transposing LDS read gives.  Rows of LDS are permuted in chunks of 16 bytes so that neither read meets itself on a bank.
//
// A CU has two such workgroups, and one's products run beside the other's softmax.  Tried and slower: a workgroup of eight
// waves that share K and V (10 % for windows, even elsewhere: they wait for each other); 64 rows a wave, one wave a SIMD, each
// LDS read feeding two products (272 us for 187); a wave's weights computed in the middle of its own products (212 for 203).
// Four prompts of up to 2500 tokens, 32 heads over 8 x 128: 187 us, 730 TFLOP/s; two chunks of up to 512 tokens behind up to
// 24000 fp8 keys, 64 heads over 8 x 128: 640 us, 860 TFLOP/s.
#pragma once

#include "paged_attention_few.hpp"

namespace arctic {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 mfma32(BF16, const u32x4 &a, const u32x4 &b, const f32x16 &c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(F16, const u32x4 &a, const u32x4 &b, const f32x16 &c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// the two 16-bit numbers of a word added to c
__device__ __forceinline__ float add_two(BF16, uint32_t w, float c) {
  const bf16x2v ones = {(__bf16)1.f, (__bf16)1.f};
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, w), ones, c, false);
}
__device__ __forceinline__ float add_two(F16, uint32_t w, float c) {
  const f16x2v ones = {(_Float16)1.f, (_Float16)1.f};
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2v, w), ones, c, false);
}

struct ManyParams {
  AttentionParams a;
  float *partial;      // [slots][kv_heads][splits][rows of a slot][head_size]; null: one split
  float *statistics;   // [slots][kv_heads][splits][rows of a slot][2]: maximum (base 2), sum
  int slots;           // row tiles that there are room for
  int splits, tiles_per_split;
  int per_sequence;    // row tiles of every sequence; 0: ragged
  Divisor by_kv_heads, by_splits, by_per_sequence, by_group;
};

constexpr int kManyWaves = 4, kManyRows = 32 * kManyWaves;
constexpr int many_keys(int padded) { return padded > 128 ? 32 : 64; }   // of a tile: the rows in flight stay in registers

// A row tile: `rows` query rows from `row0` on of sequence b, whose queries are `count` and start at row `first` of the
// query tensor.  Ragged sequences have room for floor(query_start[b + 1] rows) - floor(query_start[b] rows) + 1 tiles, as
// many as they can need wherever they start.  By one wave.
struct RowTile {
  int b, row0, rows, count, length;
  int64_t first;
  __device__ __forceinline__ RowTile(const ManyParams &mp, int slot) {
    const AttentionParams &p = mp.a;
    int64_t begin_row;
    if (mp.per_sequence) {
      b = (int)mp.by_per_sequence.quotient((uint32_t)slot);
      begin_row = (int64_t)(slot - b * mp.per_sequence) * kManyRows;
      count = p.new_tokens;
      first = (int64_t)b * count;
    } else {
      const int lane = threadIdx.x & 63;
      auto begin = [&](int i) { return (int64_t)p.query_start[i] * p.group / kManyRows + i; };
      int lo = 0, n = p.batch;   // the sequence is one of lo .. lo + n - 1
      while (n > 1) {
        const int step = (n + 63) / 64, at = lo + lane * step;
        const uint64_t before = __ballot(lane * step < n && begin(at) <= slot);
        const int k = 63 - __builtin_clzll(before | 1);
        n = min(step, n - k * step);
        lo += k * step;
      }
      b = lo;
      first = p.query_start[b];
      count = p.query_start[b + 1] - (int)first;
      begin_row = (slot - min(max(begin(b), (int64_t)0), (int64_t)slot)) * kManyRows;
      if (first < 0 || first + count > p.total_tokens) count = 0;
    }
    const int64_t all = count > 0 ? (int64_t)count * p.group : 0;
    rows = (int)max((int64_t)0, min((int64_t)kManyRows, all - begin_row));
    row0 = rows ? (int)begin_row : 0;
    length = clamped_length(p, b);
  }
};

// The tiles of keys that the queries at positions first .. last see: those that hold sinks, then those from the first
// one's window on.
template <int kKeys>
struct ManyTiles {
  int sink_tiles, window_tile, count;
  __device__ __forceinline__ ManyTiles(const AttentionParams &p, int first, int last) {
    const int start = window_start(p, max(0, first));
    window_tile = start / kKeys;
    sink_tiles = min(window_tile, (min(p.sinks, start) + kKeys - 1) / kKeys);
    count = last >= 0 ? sink_tiles + (last / kKeys - window_tile + 1) : 0;
  }
  __device__ __forceinline__ int start(int t) const { return (t < sink_tiles ? t : window_tile + (t - sink_tiles)) * kKeys; }
};

// Of a word of 32 keys, those before the n-th.
__device__ __forceinline__ uint32_t before(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

template <typename T, typename C, int kPadded>
__global__ __launch_bounds__(64 * kManyWaves, kPadded > 128 ? 1 : 2) void attention_many_kernel(const ManyParams mp) {
  const AttentionParams &p = mp.a;
  constexpr int kElt = C::kBytes;
  constexpr int kThreads = 64 * kManyWaves;
  constexpr int kKeys = many_keys(kPadded), kSubs = kKeys / 32;
  constexpr int kChunks = kPadded / 8;                      // 16-byte chunks of an LDS row
  constexpr int kCacheChunks = kPadded * kElt / 16;         // of a cache row
  constexpr int kPassRows = kThreads / kCacheChunks;
  constexpr int kPasses = kKeys / kPassRows;
  constexpr int kSteps = kPadded / 16;                      // of the first product
  constexpr int kTiles = kPadded / 32;                      // row tiles of the second
  constexpr int kBuffer = kKeys * kChunks;
  __shared__ u32x4 keys[2][kBuffer], values[2][kBuffer];
  __shared__ int odd[2][kManyWaves];   // whether a wave kept a value that is infinite or NaN

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t unit = mp.by_kv_heads.quotient(blockIdx.x);
  const int kv_head = (int)(blockIdx.x - unit * (uint32_t)p.kv_heads);
  const uint32_t from_end = mp.by_splits.quotient(unit);
  const int split = (int)(unit - from_end * (uint32_t)mp.splits);
  const int slot = mp.slots - 1 - (int)from_end;   // a sequence's last rows see most keys: they begin first
  const RowTile tile(mp, slot);
  const int b = __builtin_amdgcn_readfirstlane(tile.b), rows = __builtin_amdgcn_readfirstlane(tile.rows),
            row0 = __builtin_amdgcn_readfirstlane(tile.row0), count = __builtin_amdgcn_readfirstlane(tile.count),
            length = __builtin_amdgcn_readfirstlane(tile.length);
  if (rows == 0) return;
  const int behind = length - count;   // position of the sequence's first query
  auto position_of = [&](int row) { return behind + (int)mp.by_group.quotient((uint32_t)(row0 + min(row, rows - 1))); };
  const ManyTiles<kKeys> tiles(p, position_of(0), position_of(rows - 1));
  const int per_split = max(mp.tiles_per_split, (tiles.count + mp.splits - 1) / mp.splits);
  const int first = split * per_split, end = min(tiles.count, first + per_split);
  if (first >= end && split > 0) return;   // the first split answers for rows that see nothing

  // ---- the wave's query rows ------------------------------------------------------------------------------------
  const int row = wave * 32 + c;
  const bool busy = wave * 32 < rows;
  const int position = position_of(row), lowest = position_of(wave * 32), highest = position_of(wave * 32 + 31);
  u32x4 q[kSteps];
  {
    const int r = row0 + min(row, rows - 1), token = (int)mp.by_group.quotient((uint32_t)r);
    const char *at = p.query + (tile.first + token) * p.query_token + (int64_t)(kv_head * p.group + r - token * p.group) * p.query_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      q[s] = u32x4{0, 0, 0, 0};
      if (row < rows && s * 16 + g * 8 < p.head_size) q[s] = *(const ARCTIC_GLOBAL u32x4 *)(at + (s * 16 + g * 8) * 2);
    }
  }
  // The scores are scaled where their maximum is subtracted, so the scale has to be positive: the rows take the sign.
  float scale = p.scale * (p.k_scale ? *p.k_scale : 1.f) * 1.44269504088896340736f;
  if (scale < 0.f) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[s] ^= 0x80008000u;
  }
  scale = fabsf(scale);
  if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;   // (a NaN stays one; -inf times zero would be another)
  // m follows the maximum when that is more than 2^8 ahead: any m serves, and weights of up to 256 are as precise as those
  // up to 1.  (Followed at once, o is multiplied for nearly every tile: some row of 32 has a new maximum.)
  const float slack = fminf(8.f / scale, 3e38f);

  // ---- from the cache into LDS ------------------------------------------------------------------------------------
  const int32_t *table = p.table + (int64_t)b * p.table_row;
  // The table's entry for the tile's key `lane`, issued before the rows of the tile before it and asked for after them:
  // loads return in order.
  auto look_up = [&](int t) {
    const int j = min(tiles.start(min(t, end - 1)) + (lane & (kKeys - 1)), length - 1);
    return table[p.by_block.quotient((uint32_t)j)];
  };
  auto holding = [&](int t, int entry) {   // which of the tile's keys there are, and have a page
    return __ballot(lane < kKeys && tiles.start(t) + lane < length && (uint32_t)entry < (uint32_t)p.num_blocks);
  };
  const int load_row = tid / kCacheChunks, load_chunk = tid % kCacheChunks;
  const bool loads = load_chunk * (16 / kElt) < p.head_size;   // the others load the row's beginning and keep nothing
  const char *const key_from = p.key_cache + (int64_t)kv_head * p.key_head + (loads ? load_chunk * 16 : 0),
             *const value_from = p.value_cache + (int64_t)kv_head * p.value_head + (loads ? load_chunk * 16 : 0);
  u32x4 key_in[kPasses], value_in[kPasses];
  auto request = [&](int t, int entry) {   // every lane finds the tile's key `lane`, for those who load it
    const uint32_t j = (uint32_t)(tiles.start(min(t, end - 1)) + (lane & (kKeys - 1)));
    const uint32_t off = j - p.by_block.quotient(j) * (uint32_t)p.block_size;
    const uint32_t page = (uint32_t)entry < (uint32_t)p.num_blocks ? (uint32_t)entry : 0u;   // of a page that is not there: not used
    // (a block's stride and what lies inside one have 32 bits)
    const uint64_t key = (uint64_t)page * (uint32_t)p.key_block + off * (uint32_t)p.key_token,
                   value = (uint64_t)page * (uint32_t)p.value_block + off * (uint32_t)p.value_token;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int k = load_row + i * kPassRows;
      const uint64_t key_at = (uint64_t)(uint32_t)__shfl((int)(key >> 32), k) << 32 | (uint32_t)__shfl((int)key, k),
                     value_at = (uint64_t)(uint32_t)__shfl((int)(value >> 32), k) << 32 | (uint32_t)__shfl((int)value, k);
      key_in[i] = *(const ARCTIC_GLOBAL u32x4 *)(key_from + key_at);
      value_in[i] = *(const ARCTIC_GLOBAL u32x4 *)(value_from + value_at);
    }
  };
  // Chunk of row k, where it lies.  K's readers take one chunk of 32 rows, V's four chunks of four rows.  Eight lanes write
  // at once, of an fp8 cache every other chunk of a row or two: the last bit parts those that would meet within 128 bytes.
  auto key_place = [](int k, int chunk) { return k * kChunks + (chunk ^ (chunk >> 3 & 1) ^ (kChunks == 8 ? (k >> 1 & 7) ^ (k & 1) : k & 15)); };
  auto value_place = [](int k, int chunk) { return k * kChunks + (chunk ^ (chunk >> 3 & 1) ^ (kChunks == 8 ? (k >> 1 & 1) << 2 | (k & 1) : (k & 3) << 2)); };
  // Into LDS; with `look`, looking for values that are infinite or NaN.
  auto keep = [&](int buffer, bool look) {
    bool found = false;
    if (look) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t word = value_in[i][w];
          asm volatile("" : "+v"(word));   // looked at in here alone
          if constexpr (kElt == 2) found |= unusual(T{}, word);
          else found |= unusual(T{}, widen<false>(T{}, C{}, word)) || unusual(T{}, widen<true>(T{}, C{}, word));
        }
      odd[buffer][wave] = __any(found && loads);
    }
    if (!loads) return;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int k = load_row + i * kPassRows;
      if constexpr (kElt == 2) {
        keys[buffer][key_place(k, load_chunk)] = key_in[i];
        values[buffer][value_place(k, load_chunk)] = value_in[i];
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 x, y;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t kw = key_in[i][2 * h + (w >> 1)], vw = value_in[i][2 * h + (w >> 1)];
            x[w] = w & 1 ? widen<true>(T{}, C{}, kw) : widen<false>(T{}, C{}, kw);
            y[w] = w & 1 ? widen<true>(T{}, C{}, vw) : widen<false>(T{}, C{}, vw);
          }
          keys[buffer][key_place(k, 2 * load_chunk + h)] = x;
          values[buffer][value_place(k, 2 * load_chunk + h)] = y;
        }
      }
    }
  };

  // ---- the products -----------------------------------------------------------------------------------------------
  f32x16 o[kTiles];
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int d = 0; d < kTiles; ++d) o[d] = f32x16{};
  auto scores = [&](int buffer, int h, f32x16 &s) {   // of 32 of the tile's keys
    s = f32x16{};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) s = mfma32(T{}, keys[buffer][key_place(32 * h + c, 2 * i + g)], q[i], s);
  };
  // V's operand for the elements 32 d .. and the keys 16 t + 4 g + {0 .. 3}, + 8
  auto operand = [&](int buffer, int t, int d) {
    u32x4 v;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = 16 * t + 8 * h + 4 * g + (lane >> 2 & 3), chunk = 4 * d + 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)((__attribute__((address_space(3))) char *)&values[buffer][value_place(k, chunk)] + 8 * (lane & 1)));
      const u32x2 w = __builtin_bit_cast(u32x2, x);
      v[2 * h] = w.x, v[2 * h + 1] = w.y;
    }
    return v;
  };
  // scores (base 2 once multiplied by `scale`; -inf where a key is not seen) into weights, two keys to a word.  m is a score.
  auto weigh = [&](const auto &s, auto &weight) {
    constexpr int kHalves = sizeof(s) / sizeof(s[0]);
    float top = -__builtin_inff();
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[h][i]);
    const auto half = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = fmaxf(__uint_as_float(half[0]), __uint_as_float(half[1]));
    if (__any(top > m + slack)) {
      const float now = fmaxf(m, top);
      const float keep_ = __builtin_amdgcn_exp2f((m - (now == -__builtin_inff() ? 0.f : now)) * scale);
      m = now;
      l *= keep_;
#pragma unroll
      for (int d = 0; d < kTiles; ++d) o[d] *= keep_;
    }
    const float base = m == -__builtin_inff() ? 0.f : -m * scale;
#pragma unroll
    for (int t = 0; t < 2 * kHalves; ++t)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int i = 8 * (t & 1) + 2 * w;
        weight[t][w] = T::pack(__builtin_amdgcn_exp2f(fmaf(s[t >> 1][i], scale, base)), __builtin_amdgcn_exp2f(fmaf(s[t >> 1][i + 1], scale, base)));
        l = add_two(T{}, weight[t][w], l);
      }
  };

  int t = first;
  int entry = 0;
  uint64_t holds = 0, holds_next = 0;
  constexpr uint64_t kAll = kKeys == 64 ? ~(uint64_t)0 : 0xffffffffull;
  auto whole = [&](int t, uint64_t holds, int lowest, int highest) {   // rows of those positions see every key of the tile
    const int start = tiles.start(t);
    return holds == kAll && start + kKeys - 1 <= lowest && (p.window <= 0 || start > highest - p.window);
  };
  const int tile_lowest = position_of(0), tile_highest = position_of(rows - 1);
  if (p.head_size < kPadded) {
    for (int i = tid; i < 2 * kBuffer; i += kThreads) (&keys[0][0])[i] = (&values[0][0])[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  if (t < end) {
    const int first_entry = look_up(t);
    entry = look_up(t + 1);
    holds = holding(t, first_entry);
    request(t, first_entry);
    keep(0, !whole(t, holds, tile_lowest, tile_highest));
  }
  __syncthreads();
  auto begin_tile = [&]() {   // (after the last tile's: what is read is not used)
    holds_next = holding(t + 1, entry);
    const int now = entry;
    entry = look_up(t + 2);
    request(t + 1, now);
  };
  auto end_tile = [&]() {
    keep((t + 1 - first) & 1, !whole(t + 1, holds_next, tile_lowest, tile_highest));
    holds = holds_next;
    ++t;
    __syncthreads();
  };
  while (t < end) {
    while (t < end && busy && whole(t, holds, lowest, highest)) {
      begin_tile();
      const int buffer = (t - first) & 1;
      f32x16 s[kSubs];
      u32x4 weight[2 * kSubs];
#pragma unroll
      for (int h = 0; h < kSubs; ++h) scores(buffer, h, s[h]);
      weigh(s, weight);
#pragma unroll
      for (int i = 0; i < 2 * kSubs; ++i)
#pragma unroll
        for (int d = 0; d < kTiles; ++d) o[d] = mfma32(T{}, operand(buffer, i, d), weight[i], o[d]);
      end_tile();
    }
    while (t < end && !(busy && whole(t, holds, lowest, highest))) {
      begin_tile();
      const int start = tiles.start(t), buffer = (t - first) & 1;
      // (the lane's number as if it were another for every tile: what follows from it is not kept over the other loop)
      int other = lane;
      asm volatile("" : "+v"(other));
      const int g = other >> 5;
      const uint32_t one = T::pack(1.f, 1.f);
      bool careful = false;
#pragma unroll
      for (int w = 0; w < kManyWaves; ++w) careful = careful || odd[buffer][w];
#pragma unroll 1
      for (int h = 0; h < kSubs; ++h) {
        const int at = start + 32 * h;
        // keys that no row of the wave sees are passed over
        if (!busy || at > highest || (at + 32 <= window_start(p, lowest) && at >= p.sinks)) continue;
        const uint32_t there = (uint32_t)(holds >> (32 * h));
        f32x16 s[1];
        u32x4 weight[2];
        scores(buffer, h, s[0]);
        const uint32_t seen = (there & before(position - at + 1) & (~before(window_start(p, position) - at) | before(p.sinks - at))) >> (4 * g);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[0][i] = seen >> (8 * (i >> 2) + (i & 3)) & 1 ? s[0][i] : -__builtin_inff();
        weigh(s, weight);
        // a weight of zero must not meet an infinity or a NaN (as in the kernel for few tokens)
        const uint32_t any = (there & before(highest - at + 1) & (~before(window_start(p, lowest) - at) | before(p.sinks - at))) >> (4 * g);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int d = 0; d < kTiles; ++d) {
            u32x4 v = operand(buffer, 2 * h + i, d);
            if (careful) {
              u32x4 codes, has_weight;
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const uint32_t two = any >> (16 * i + 8 * (w >> 1) + 2 * (w & 1));
                v[w] &= (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
                codes[w] = unusual_codes(T{}, v[w]);
                v[w] &= (codes[w] & 0xffffu ? 0u : 0xffffu) | (codes[w] >> 16 ? 0u : 0xffff0000u);
                has_weight[w] = one & ((weight[i][w] & 0xffffu ? 0xffffu : 0u) | (weight[i][w] >> 16 ? 0xffff0000u : 0u));
              }
              const f32x16 counts = mfma32(T{}, codes, has_weight, f32x16{});
#pragma unroll
              for (int e = 0; e < 16; ++e) o[d][e] += unusual_sum((int)counts[e]);
            }
            o[d] = mfma32(T{}, v, weight[i], o[d]);
          }
      }
      end_tile();
    }
  }

  // ---- results: a lane has 4 consecutive elements of its row at a time ----------------------------------------------
  {
    const auto half = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(half[0]) + __uint_as_float(half[1]);
  }
  if (row >= rows) return;
  if (mp.partial) {
    const int64_t at = (((int64_t)slot * p.kv_heads + kv_head) * mp.splits + split) * kManyRows + row;
    if (g == 0) {
      mp.statistics[at * 2] = m * scale;
      mp.statistics[at * 2 + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < kTiles; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 32 * d + 8 * i + 4 * g;
        if (e < p.head_size)
          *(ARCTIC_GLOBAL f32x4 *)(mp.partial + at * p.head_size + e) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
      }
  } else {
    const float norm = l == 0.f ? 0.f : (p.v_scale ? *p.v_scale : 1.f) / l;
    const int r = row0 + row, token = (int)mp.by_group.quotient((uint32_t)r);
    char *at = p.out + (tile.first + token) * p.out_token + (int64_t)(kv_head * p.group + r - token * p.group) * p.out_head;
#pragma unroll
    for (int d = 0; d < kTiles; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 32 * d + 8 * i + 4 * g;
        if (e < p.head_size)
          *(ARCTIC_GLOBAL u32x2 *)(at + e * 2) = u32x2{T::pack(o[d][4 * i] * norm, o[d][4 * i + 1] * norm),
                                                       T::pack(o[d][4 * i + 2] * norm, o[d][4 * i + 3] * norm)};
      }
  }
}

// The splits of a row tile, joined; a wave per row, 4 elements a lane.  Two chunks of 512 tokens, 64 heads, in two splits: 17 us.
template <typename T, int kKeys>
__global__ __launch_bounds__(256) void attention_many_join_kernel(const ManyParams mp) {
  const AttentionParams &p = mp.a;
  const uint32_t slot = mp.by_kv_heads.quotient(blockIdx.x);
  const int kv_head = (int)(blockIdx.x - slot * (uint32_t)p.kv_heads);
  const RowTile tile(mp, (int)slot);
  if (tile.rows == 0) return;
  const int behind = tile.length - tile.count;
  const ManyTiles<kKeys> tiles(p, behind + (int)mp.by_group.quotient((uint32_t)tile.row0),
                        behind + (int)mp.by_group.quotient((uint32_t)(tile.row0 + tile.rows - 1)));
  const int per_split = max(mp.tiles_per_split, (tiles.count + mp.splits - 1) / mp.splits);
  const int used = max(1, (tiles.count + per_split - 1) / per_split);
  const int lane = threadIdx.x & 63, d = lane * 4;
  const float v_scale = p.v_scale ? *p.v_scale : 1.f;
  for (int row = blockIdx.y * 4 + (int)(threadIdx.x >> 6); row < tile.rows; row += 4 * kManyRows / 32) {
    const int64_t at = ((int64_t)slot * p.kv_heads + kv_head) * mp.splits * kManyRows + row;
    float top = -__builtin_inff(), sum = 0.f;
    f32x4 acc = {0, 0, 0, 0};
    for (int s0 = 0; s0 < used; s0 += 4) {
      float2 st[4];
      f32x4 part[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        st[k] = make_float2(-__builtin_inff(), 0.f);
        part[k] = f32x4{0, 0, 0, 0};
        if (s0 + k < used) {
          st[k] = *(const float2 *)(mp.statistics + (at + (int64_t)(s0 + k) * kManyRows) * 2);
          if (d < p.head_size) part[k] = *(const ARCTIC_GLOBAL f32x4 *)(mp.partial + (at + (int64_t)(s0 + k) * kManyRows) * p.head_size + d);
        }
      }
      float now = top;
#pragma unroll
      for (int k = 0; k < 4; ++k) now = fmaxf(now, st[k].x);
      const float base = now == -__builtin_inff() ? 0.f : now, keep = __builtin_amdgcn_exp2f(top - base);
      sum *= keep;
      acc *= keep;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float own = __builtin_amdgcn_exp2f(st[k].x - base);
        sum += st[k].y * own;
        acc += part[k] * own;
      }
      top = now;
    }
    if (d < p.head_size) {
      acc *= sum == 0.f ? 0.f : v_scale / sum;
      const int r = tile.row0 + row, token = (int)mp.by_group.quotient((uint32_t)r);
      *(ARCTIC_GLOBAL u32x2 *)(p.out + (tile.first + token) * p.out_token + (int64_t)(kv_head * p.group + r - token * p.group) * p.out_head + d * 2) =
          u32x2{T::pack(acc[0], acc[1]), T::pack(acc[2], acc[3])};
    }
  }
}

struct ManyShape {
  int padded;
  int64_t slots;
  int splits, tiles_per_split, per_sequence;
};
void many_launch_bf16(const ManyParams &p, const ManyShape &f, int kv, hipStream_t s);
void many_launch_f16(const ManyParams &p, const ManyShape &f, int kv, hipStream_t s);

template <typename T, typename C>
inline void many_launch_padded(const ManyParams &p, const ManyShape &f, dim3 grid, hipStream_t s) {
  if (f.padded == 256) launch(attention_many_kernel<T, C, 256>, grid, 64 * kManyWaves, s, p);
  else if (f.padded == 128) launch(attention_many_kernel<T, C, 128>, grid, 64 * kManyWaves, s, p);
  else launch(attention_many_kernel<T, C, 64>, grid, 64 * kManyWaves, s, p);
}
template <typename T>
inline void many_launch(const ManyParams &p, const ManyShape &f, int kv, hipStream_t s) {
  const dim3 grid((unsigned)(f.slots * f.splits * p.a.kv_heads));
  if (kv == ARCTIC_KV_AUTO) many_launch_padded<T, Half<T>>(p, f, grid, s);
  else if (kv == ARCTIC_KV_FP8_E4M3) many_launch_padded<T, CacheE4M3>(p, f, grid, s);
  else many_launch_padded<T, CacheE5M2>(p, f, grid, s);
  if (f.splits == 1) return;
  const dim3 tiles((unsigned)(f.slots * p.a.kv_heads), kManyWaves);
  if (f.padded == 256) launch(attention_many_join_kernel<T, many_keys(256)>, tiles, 256, s, p);
  else launch(attention_many_join_kernel<T, many_keys(128)>, tiles, 256, s, p);
}

}  // namespace arctic
