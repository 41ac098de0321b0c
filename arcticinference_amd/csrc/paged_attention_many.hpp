// Attention of many new tokens of a sequence: a workgroup per key head and tile of query rows (token by token, head by head
// of the key head's group), 32 rows a wave, over the keys that any of them sees, 64 at a time.
//
// What bounds it is the matrix cores, so K and V are read from the cache once for all waves, widened to 16 bits and kept
// in LDS twice, one tile ahead.  Query rows are the columns of both products (32x32x16):
//   S^T = K Q^T,   O^T = V^T P^T.
// The scores leave the first one with 4 x 4 consecutive keys of one row in a lane; laid over the keys to suit, the second
// one's contraction takes them as they are, and V's operand, 4 consecutive keys of one element at a time, is what the
// transposing LDS read gives.  Rows of LDS are permuted in chunks of 16 bytes so that neither read meets itself on a bank.
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

constexpr int kManyKeys = 64;

// A row tile: `rows` query rows from `row0` on of sequence b, whose queries are `count` and start at row `first` of the
// query tensor.  Ragged sequences have room for floor(query_start[b + 1] rows) - floor(query_start[b] rows) + 1 tiles, as
// many as they can need wherever they start.  By one wave.
template <int kRows>
struct RowTile {
  int b, row0, rows, count, length;
  int64_t first;
  __device__ __forceinline__ RowTile(const ManyParams &mp, int slot) {
    const AttentionParams &p = mp.a;
    int64_t begin_row;
    if (mp.per_sequence) {
      b = (int)mp.by_per_sequence.quotient((uint32_t)slot);
      begin_row = (int64_t)(slot - b * mp.per_sequence) * kRows;
      count = p.new_tokens;
      first = (int64_t)b * count;
    } else {
      const int lane = threadIdx.x & 63;
      auto begin = [&](int i) { return (int64_t)p.query_start[i] * p.group / kRows + i; };
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
      begin_row = (slot - min(max(begin(b), (int64_t)0), (int64_t)slot)) * kRows;
      if (first < 0 || first + count > p.total_tokens) count = 0;
    }
    const int64_t all = count > 0 ? (int64_t)count * p.group : 0;
    rows = (int)max((int64_t)0, min((int64_t)kRows, all - begin_row));
    row0 = rows ? (int)begin_row : 0;
    length = clamped_length(p, b);
  }
};

// The tiles of 64 keys that the queries at positions first .. last see: those that hold sinks, then those from the first
// one's window on.
struct ManyTiles {
  int sink_tiles, window_tile, count;
  __device__ __forceinline__ ManyTiles(const AttentionParams &p, int first, int last) {
    const int start = window_start(p, max(0, first));
    window_tile = start / kManyKeys;
    sink_tiles = min(window_tile, (min(p.sinks, start) + kManyKeys - 1) / kManyKeys);
    count = last >= 0 ? sink_tiles + (last / kManyKeys - window_tile + 1) : 0;
  }
  __device__ __forceinline__ int start(int t) const { return (t < sink_tiles ? t : window_tile + (t - sink_tiles)) * kManyKeys; }
};

template <typename T, typename C, int kPadded, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kPadded > 128 ? 1 : 2) void attention_many_kernel(const ManyParams mp) {
  const AttentionParams &p = mp.a;
  constexpr int kElt = C::kBytes;
  constexpr int kThreads = 64 * kWaves, kRows = 32 * kWaves;
  constexpr int kChunks = kPadded / 8;                      // 16-byte chunks of an LDS row
  constexpr int kCacheChunks = kPadded * kElt / 16;         // of a cache row
  constexpr int kPassRows = kThreads / kCacheChunks > kManyKeys ? kManyKeys : kThreads / kCacheChunks;
  constexpr int kPasses = kManyKeys / kPassRows;
  constexpr int kSteps = kPadded / 16;                      // of the first product
  constexpr int kTiles = kPadded / 32;                      // row tiles of the second
  constexpr int kBuffer = kManyKeys * kChunks;
  __shared__ u32x4 keys[2][kBuffer], values[2][kBuffer];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t unit = mp.by_kv_heads.quotient(blockIdx.x);
  const int kv_head = (int)(blockIdx.x - unit * (uint32_t)p.kv_heads);
  const uint32_t from_end = mp.by_splits.quotient(unit);
  const int split = (int)(unit - from_end * (uint32_t)mp.splits);
  const int slot = mp.slots - 1 - (int)from_end;   // a sequence's last rows see most keys: they begin first
  const RowTile<kRows> tile(mp, slot);
  const int b = __builtin_amdgcn_readfirstlane(tile.b), rows = __builtin_amdgcn_readfirstlane(tile.rows),
            row0 = __builtin_amdgcn_readfirstlane(tile.row0), count = __builtin_amdgcn_readfirstlane(tile.count),
            length = __builtin_amdgcn_readfirstlane(tile.length);
  if (rows == 0) return;
  const int behind = length - count;   // position of the sequence's first query
  auto position_of = [&](int row) { return behind + (int)mp.by_group.quotient((uint32_t)(row0 + min(row, rows - 1))); };
  const ManyTiles tiles(p, position_of(0), position_of(rows - 1));
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
  const float scale = p.scale * (p.k_scale ? *p.k_scale : 1.f) * 1.44269504088896340736f;

  // ---- from the cache into LDS ------------------------------------------------------------------------------------
  const int32_t *table = p.table + (int64_t)b * p.table_row;
  auto look_up = [&](int t) {   // the page of the tile's key `lane`, or -1
    const int j = t < end ? tiles.start(t) + lane : length;
    if (j >= length) return -1;
    const int page = table[p.by_block.quotient((uint32_t)j)];
    return page >= 0 && page < p.num_blocks ? page : -1;
  };
  const int load_row = tid / kCacheChunks, load_chunk = tid % kCacheChunks;
  const bool loads = load_row < kPassRows && load_chunk * (16 / kElt) < p.head_size;
  u32x4 key_in[kPasses], value_in[kPasses];
  auto request = [&](int t, int pages) {
    const int start = tiles.start(t);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int k = load_row + i * kPassRows;
      const int64_t page = max(__shfl(pages, k & 63), 0);   // of a page that is not there: what is loaded is not used
      const int j = start + k, off = j - (int)p.by_block.quotient((uint32_t)j) * p.block_size;
      key_in[i] = value_in[i] = u32x4{0, 0, 0, 0};
      if (loads) {
        key_in[i] = *(const ARCTIC_GLOBAL u32x4 *)(p.key_cache + page * p.key_block + (int64_t)off * p.key_token +
                                                   (int64_t)kv_head * p.key_head + load_chunk * 16);
        value_in[i] = *(const ARCTIC_GLOBAL u32x4 *)(p.value_cache + page * p.value_block + (int64_t)off * p.value_token +
                                                     (int64_t)kv_head * p.value_head + load_chunk * 16);
      }
    }
  };
  // chunk of row k, where it lies: K's readers take one chunk of 32 rows, V's four chunks of four rows
  auto key_place = [](int k, int chunk) { return k * kChunks + (chunk ^ (kChunks == 8 ? k >> 1 & 7 : k & 15)); };
  auto value_place = [](int k, int chunk) { return k * kChunks + (chunk ^ (kChunks == 8 ? (k >> 1 & 1) << 2 : (k & 3) << 2)); };
  auto keep = [&](int buffer) {
    if (load_row >= kPassRows) return;
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
  auto scores = [&](int buffer, f32x16 (&s)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = f32x16{};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) s[h] = mfma32(T{}, keys[buffer][key_place(32 * h + c, 2 * i + g)], q[i], s[h]);
    }
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
  // scores (base 2 once multiplied by `scale`; -inf where a key is not seen) into weights, two keys to a word
  auto weigh = [&](f32x16 (&s)[2], u32x4 (&weight)[4]) {
    float top = -__builtin_inff();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[h][i]);
    const auto half = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = fmaxf(__uint_as_float(half[0]), __uint_as_float(half[1]));
    if (__any(top > m)) {
      const float now = fmaxf(m, top);
      const float keep_ = __builtin_amdgcn_exp2f(m - (now == -__builtin_inff() ? 0.f : now));
      m = now;
      l *= keep_;
#pragma unroll
      for (int d = 0; d < kTiles; ++d) o[d] *= keep_;
    }
    const float base = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int i = 8 * (t & 1) + 2 * w;
        weight[t][w] = T::pack(__builtin_amdgcn_exp2f(s[t >> 1][i] - base), __builtin_amdgcn_exp2f(s[t >> 1][i + 1] - base));
        l = add_two(T{}, weight[t][w], l);
      }
  };

  int t = first;
  int pages = look_up(t);
  uint64_t holds = __ballot(pages >= 0), holds_next = 0;
  if (t < end) {
    request(t, pages);
    pages = look_up(t + 1);
    keep(0);
  }
  __syncthreads();
  auto begin_tile = [&]() {
    holds_next = __ballot(pages >= 0);
    if (t + 1 < end) {
      request(t + 1, pages);
      pages = look_up(t + 2);
    }
  };
  auto end_tile = [&]() {
    if (t + 1 < end) keep((t + 1 - first) & 1);
    holds = holds_next;
    ++t;
    __syncthreads();
  };
  auto whole = [&]() {   // every row of the wave sees every key
    const int start = tiles.start(t);
    return busy && holds == ~(uint64_t)0 && start + kManyKeys - 1 <= lowest && (p.window <= 0 || start > highest - p.window);
  };
  while (t < end) {
    while (t < end && whole()) {
      begin_tile();
      const int buffer = (t - first) & 1;
      f32x16 s[2];
      u32x4 weight[4];
      scores(buffer, s);
#pragma unroll
      for (int h = 0; h < 2; ++h) s[h] *= scale;
      weigh(s, weight);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < kTiles; ++d) o[d] = mfma32(T{}, operand(buffer, i, d), weight[i], o[d]);
      end_tile();
    }
    while (t < end && !whole()) {
      begin_tile();
      const int start = tiles.start(t), buffer = (t - first) & 1;
      // (the lane's number as if it were another for every tile: what follows from it is not kept over the other loop)
      int other = lane;
      asm volatile("" : "+v"(other));
      const int g = other >> 5;
      // a tile that no row of the wave sees is passed over
      if (busy && start <= highest && (start + kManyKeys > window_start(p, lowest) || start < p.sinks)) {
        f32x16 s[2];
        u32x4 weight[4];
        scores(buffer, s);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int k = 32 * h + 8 * (i >> 2) + 4 * g + (i & 3), j = start + k;
            const bool seen = (holds >> k & 1) && j <= position && (j >= window_start(p, position) || j < p.sinks);
            s[h][i] = seen ? s[h][i] * scale : -__builtin_inff();
          }
        weigh(s, weight);
        // a weight of zero must not meet an infinity or a NaN (as in the kernel for few tokens)
        const uint32_t one = T::pack(1.f, 1.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u32x4 any;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            any[w] = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int k = 16 * i + 8 * (w >> 1) + 4 * g + 2 * (w & 1) + e, j = start + k;
              if ((holds >> k & 1) && j <= highest && (j >= window_start(p, lowest) || j < p.sinks)) any[w] |= e ? 0xffff0000u : 0xffffu;
            }
          }
#pragma unroll
          for (int d = 0; d < kTiles; ++d) {
            u32x4 v = operand(buffer, i, d) & any;
            if (__any(unusual(T{}, v.x) || unusual(T{}, v.y) || unusual(T{}, v.z) || unusual(T{}, v.w))) {
              u32x4 codes, seen;
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                codes[w] = unusual_codes(T{}, v[w]);
                v[w] &= (codes[w] & 0xffffu ? 0u : 0xffffu) | (codes[w] >> 16 ? 0u : 0xffff0000u);
                seen[w] = one & ((weight[i][w] & 0xffffu ? 0xffffu : 0u) | (weight[i][w] >> 16 ? 0xffff0000u : 0u));
              }
              const f32x16 counts = mfma32(T{}, codes, seen, f32x16{});
#pragma unroll
              for (int e = 0; e < 16; ++e) o[d][e] += unusual_sum((int)counts[e]);
            }
            o[d] = mfma32(T{}, v, weight[i], o[d]);
          }
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
    const int64_t at = (((int64_t)slot * p.kv_heads + kv_head) * mp.splits + split) * kRows + row;
    if (g == 0) {
      mp.statistics[at * 2] = m;
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

// The splits of a row tile, joined; a wave per row, 4 elements a lane.
template <typename T, int kRows>
__global__ __launch_bounds__(256) void attention_many_join_kernel(const ManyParams mp) {
  const AttentionParams &p = mp.a;
  const uint32_t slot = mp.by_kv_heads.quotient(blockIdx.x);
  const int kv_head = (int)(blockIdx.x - slot * (uint32_t)p.kv_heads);
  const RowTile<kRows> tile(mp, (int)slot);
  if (tile.rows == 0) return;
  const int behind = tile.length - tile.count;
  const ManyTiles tiles(p, behind + (int)mp.by_group.quotient((uint32_t)tile.row0),
                        behind + (int)mp.by_group.quotient((uint32_t)(tile.row0 + tile.rows - 1)));
  const int per_split = max(mp.tiles_per_split, (tiles.count + mp.splits - 1) / mp.splits);
  const int used = max(1, (tiles.count + per_split - 1) / per_split);
  const int lane = threadIdx.x & 63, d = lane * 4;
  const float v_scale = p.v_scale ? *p.v_scale : 1.f;
  for (int row = blockIdx.y * 4 + (int)(threadIdx.x >> 6); row < tile.rows; row += 4 * kRows / 32) {
    const int64_t at = ((int64_t)slot * p.kv_heads + kv_head) * mp.splits * kRows + row;
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
          st[k] = *(const float2 *)(mp.statistics + (at + (int64_t)(s0 + k) * kRows) * 2);
          if (d < p.head_size) part[k] = *(const ARCTIC_GLOBAL f32x4 *)(mp.partial + (at + (int64_t)(s0 + k) * kRows) * p.head_size + d);
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
  int padded, waves;
  int64_t slots;
  int splits, tiles_per_split, per_sequence;
};
void many_launch_bf16(const ManyParams &p, const ManyShape &f, int kv, hipStream_t s);
void many_launch_f16(const ManyParams &p, const ManyShape &f, int kv, hipStream_t s);

template <typename T, typename C>
inline void many_launch_padded(const ManyParams &p, const ManyShape &f, dim3 grid, hipStream_t s) {
  if (f.padded == 256) launch(attention_many_kernel<T, C, 256, 4>, grid, 256, s, p);
  else if (f.padded == 128 && f.waves == 8) launch(attention_many_kernel<T, C, 128, 8>, grid, 512, s, p);
  else if (f.padded == 128) launch(attention_many_kernel<T, C, 128, 4>, grid, 256, s, p);
  else if (f.waves == 8) launch(attention_many_kernel<T, C, 64, 8>, grid, 512, s, p);
  else launch(attention_many_kernel<T, C, 64, 4>, grid, 256, s, p);
}
template <typename T>
inline void many_launch(const ManyParams &p, const ManyShape &f, int kv, hipStream_t s) {
  const dim3 grid((unsigned)(f.slots * f.splits * p.a.kv_heads));
  if (kv == ARCTIC_KV_AUTO) many_launch_padded<T, Half<T>>(p, f, grid, s);
  else if (kv == ARCTIC_KV_FP8_E4M3) many_launch_padded<T, CacheE4M3>(p, f, grid, s);
  else many_launch_padded<T, CacheE5M2>(p, f, grid, s);
  if (f.splits == 1) return;
  const dim3 tiles((unsigned)(f.slots * p.a.kv_heads), (unsigned)f.waves);
  if (f.waves == 8) launch(attention_many_join_kernel<T, 256>, tiles, 256, s, p);
  else launch(attention_many_join_kernel<T, 128>, tiles, 256, s, p);
}

}  // namespace arctic
