// Attention of few new tokens of each sequence.  The sequences' keys, in tiles of 32, one sequence behind the other, are
// dealt out evenly over a number of workgroups per key head; the four waves of one take its tiles in turn and join what
// they found.  A sequence that is dealt to several workgroups is joined by a second kernel.
//
// What bounds it is the reading of the cache, so nothing passes through LDS on the way to the matrix cores.  A group's
// query rows (head by head, token by token) are the columns of every product, 16 to a column tile:
//   S^T = K Q^T   (16x16x32, rows: keys).   K's operand wants 8 consecutive elements of one key from a lane: a 16-byte load.
//   O^T = V^T P^T (rows: elements of the head, contraction: keys).  The scores leave the first product with 4 consecutive
//         keys of one query row in a lane, which is where P's operand wants them once the contraction's index is laid
//         over the keys to suit: slots 0-3 of lane group g are keys 4g..4g+3 of the tile's first half, slots 4-7 of its
//         second.  V's operand then wants 8 keys' values of one element; a lane loads consecutive elements of its 8 keys
//         (the 16 lanes of a group one whole row) and pairs the keys with one v_perm a word, row tile a holding the
//         elements a, a + s, a + 2s ... (s = padded head size / 16).
// The sum of the weights is one more product, with rows of ones: it takes the weights as the values do, rounded to 16
// bits, so that the rounding of a weight that stands alone cancels, and it needs no exchange between lanes.
//
// Heads of 128, 32 over 8: 64 sequences of up to 8192 fp8 keys 130 us, 5.0 TB/s; 3 of up to 131072 16-bit keys 242 us,
// 5.5 TB/s; one of 777 keys 10.6 us, 8.1 of them here (memory latencies in a row) and 3.4 in the join.
#pragma once

#include "paged_attention.hpp"

namespace arctic {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma16(BF16, const u32x4 &a, const u32x4 &b, const f32x4 &c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(F16, const u32x4 &a, const u32x4 &b, const f32x4 &c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two fp8 numbers of a word's lower or upper half as 16-bit floats: exact (both types hold every e4m3 and e5m2 number).
template <bool kHi>
__device__ __forceinline__ uint32_t widen(BF16, CacheE4M3, uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHi));
}
template <bool kHi>
__device__ __forceinline__ uint32_t widen(BF16, CacheE5M2, uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, kHi));
}
template <bool kHi>
__device__ __forceinline__ uint32_t widen(F16, CacheE4M3, uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, kHi));
}
template <bool kHi>
__device__ __forceinline__ uint32_t widen(F16, CacheE5M2, uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, kHi));
}

// Whether either half of a word of two 16-bit floats is infinite or NaN.
__device__ __forceinline__ bool unusual(BF16, uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ bool unusual(F16, uint32_t w) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; }

// For each half that is infinite or NaN a number that says which (1, 64 or 4096), zero for others; and what the sum of up
// to 32 such numbers stands for.
template <typename T>
__device__ __forceinline__ uint32_t unusual_codes(T, uint32_t w) {
  constexpr uint32_t kInf = T::kCode == ARCTIC_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  uint32_t code[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t x = w >> (16 * h) & 0xffffu, e = x & 0x7fffu;
    code[h] = e < kInf ? 0u : T::round_bits(e > kInf ? 4096.f : x >> 15 ? 64.f : 1.f);
  }
  return code[0] | code[1] << 16;
}
__device__ __forceinline__ float unusual_sum(int count) {
  float v = 0.f;
  if (count & 63) v += __builtin_inff();
  if (count >> 6 & 63) v -= __builtin_inff();
  if (count >> 12) v = __builtin_nanf("");
  return v;
}

// The largest of a query row's values in its four lanes l, l + 16, l + 32, l + 48, in each of them.
__device__ __forceinline__ float max_over_groups(float v) {
  auto half = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(half[0]), __uint_as_float(half[1]));
  auto row = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(row[0]), __uint_as_float(row[1]));
}

template <int kBytes>
struct Raw;   // what a lane loads of one row of V
template <>
struct Raw<4> {
  uint32_t w[1];
  __device__ __forceinline__ void load(const char *p) { w[0] = *(const ARCTIC_GLOBAL uint32_t *)p; }
};
template <>
struct Raw<8> {
  uint32_t w[2];
  __device__ __forceinline__ void load(const char *p) {
    const u32x2 v = *(const ARCTIC_GLOBAL u32x2 *)p;
    w[0] = v.x, w[1] = v.y;
  }
};
template <int kBytes>
struct Raw {   // 16 and 32
  uint32_t w[kBytes / 4];
  __device__ __forceinline__ void load(const char *p) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) {
      const u32x4 v = *(const ARCTIC_GLOBAL u32x4 *)(p + 16 * i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  }
};

struct FewParams {
  AttentionParams a;
  float *partial;        // [kv_heads][2 * workers][rows][head_size]
  float *statistics;     // [kv_heads][2 * workers][rows][2]: maximum (base 2), sum
  int2 *dealt;           // [batch]: the first and the last worker that a sequence was dealt to
  int rows;              // new_tokens * group
  int row_tiles;         // workgroups that share the rows
  int workers;           // workgroups that share the keys of one head (and of one row tile)
  int least;             // tiles that a worker takes at least; 0: worker b takes sequence b
  Divisor by_row_tiles, by_head_groups;
};

// The tiles of 32 keys of a sequence's queries: those that hold sinks, then those from the first query's window on.
struct Tiles {
  int sink_tiles, window_tile, count;
  __device__ __forceinline__ Tiles(const AttentionParams &p, int length, int new_tokens) {
    const int start = window_start(p, max(0, length - new_tokens));
    window_tile = start >> 5;
    sink_tiles = min(window_tile, (min(p.sinks, start) + 31) >> 5);
    // a sequence without keys has one tile without keys, in which its queries are answered
    count = length > 0 ? sink_tiles + (((length - 1) >> 5) - window_tile + 1) : 1;
  }
  __device__ __forceinline__ int start(int t) const { return (t < sink_tiles ? t : window_tile + (t - sink_tiles)) << 5; }
};
// How the sequences' tiles, one sequence behind the other, are dealt out: found by every wave for itself.
struct Deal {
  int64_t at, stop;   // a worker's tiles
  int64_t begin;      // the first tile of sequence b, which tile `at` belongs to (a multiple of `per` where shares are of one
                      // sequence each: the last one's tiles that there are not count too)
  int64_t per;        // tiles of a worker
  int b;
  template <typename I>
  __device__ __forceinline__ static I up_to(I v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const I other = __shfl_up(v, d);
      if (lane >= d) v += other;
    }
    return v;
  }
  __device__ __forceinline__ Deal(const FewParams &fp, int worker) {
    const AttentionParams &p = fp.a;
    const int lane = threadIdx.x & 63;
    auto count = [&](int i) { return i < p.batch ? Tiles(p, clamped_length(p, i), p.new_tokens).count : 0; };
    const int n = count(lane);
    const int64_t upto = up_to((int64_t)n, lane);
    int64_t total = __shfl(upto, 63);
    if (p.batch > 64) {
      int64_t rest = 0;
      for (int i = 64 + lane; i < p.batch; i += 64) rest += count(i);
      total += __shfl(up_to(rest, lane), 63);
    }
    per = max((int64_t)fp.least, (total + fp.workers - 1) / fp.workers);
    // A worker whose tiles are of two sequences does everything but reading them twice.  Where shares are small that is much,
    // and no worker does if every sequence begins with one, for which shares an eighth or a quarter larger may do.
    if (p.batch > 1 && p.batch <= 64 && per <= 64) {
      for (int grown = 0; grown < 3; ++grown) {
        const uint32_t share = ((uint32_t)per * (8 + grown) + 7) / 8;
        const int pieces = (int)(((uint32_t)n + share - 1) / share), last = up_to(pieces, lane);
        if (__shfl(last, 63) > fp.workers) continue;
        per = share;
        at = (int64_t)worker * per;
        stop = b = 0;
        const uint64_t beyond = __ballot(last > worker);
        if (!beyond) return;
        b = __builtin_ctzll(beyond);
        begin = (int64_t)__shfl(last - pieces, b) * per;
        stop = min(at + per, begin + __shfl(n, b));
        return;
      }
    }
    at = (int64_t)worker * per;
    stop = min(total, at + per);
    b = 0;
    begin = 0;
    if (at >= stop) return;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
      const int own = b0 ? count(b0 + lane) : n;
      const int64_t now = before + (b0 ? up_to((int64_t)own, lane) : upto);
      const uint64_t beyond = __ballot(now > at);
      if (beyond) {
        const int l = __builtin_ctzll(beyond);
        begin = __shfl(now - own, l);
        b = b0 + l;
        return;
      }
      before = __shfl(now, 63);
    }
  }
};

constexpr int kFewWaves = 4;

// Waves on a SIMD, which is what a kernel's registers are allotted by: K and V of a tile, the query rows, their results
// and about 70 more have to fit without spilling.  (Two, a workgroup's waves over, already read at the full rate.)
constexpr int few_waves(int padded, int element, int columns) {
  const int registers = padded * element / 4 + columns * (padded * 3 / 8 + 8) + 70;
  return registers <= 168 ? 3 : registers <= 256 ? 2 : 1;
}

// kPadded: head size that the products are made for; kColumns: column tiles of 16 query rows; kHeads: key heads that a
// workgroup's waves share (rows of 128 bytes or less lie side by side in one stretch of memory); kPlain: the head fills
// kPadded and 16 keys that start at a multiple of 16 lie in one block.
template <typename T, typename C, int kPadded, int kColumns, int kHeads, bool kPlain>
__global__ __launch_bounds__(64 * kFewWaves, few_waves(kPadded, C::kBytes, kColumns)) void attention_few_kernel(const FewParams fp) {
  const AttentionParams &p = fp.a;
  constexpr int kElt = C::kBytes;
  constexpr int kSteps = kPadded / 32;             // of the first product
  constexpr int kLoads = kPadded * kElt / 64;      // 16-byte loads of a key by its four lanes
  constexpr int kStepsPerLoad = kSteps / kLoads;   // 1, or 2 of fp8
  constexpr int kSpan = kPadded / 16;              // row tiles of the second product, consecutive elements of V in a lane
  constexpr int kRows = 16 * kColumns;
  constexpr int kStride = kFewWaves / kHeads;      // waves that take one head's tiles in turn
  __shared__ float tops[kFewWaves][kRows], sums[kFewWaves][kRows];
  __shared__ float joined[kHeads][kRows][kPadded + 4];
  const int all_waves = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wave = all_waves % kStride, head_at = all_waves / kStride;
  // the heads of a worker's tiles one behind the other: they read neighbouring bytes
  const uint32_t unit = fp.by_head_groups.quotient(blockIdx.x);
  const int kv_head = (int)(blockIdx.x - unit * fp.by_head_groups.d) * kHeads + head_at;
  const int worker = (int)fp.by_row_tiles.quotient(unit);
  const int row0 = (int)(unit - (uint32_t)worker * (uint32_t)fp.row_tiles) * kRows;
  const float scale = p.scale * (p.k_scale ? *p.k_scale : 1.f) * 1.44269504088896340736f;
  const uint32_t one = T::pack(1.f, 1.f);
  const u32x4 ones = {one, one, one, one};

  int b = worker;
  int64_t at = 0, stop = 0, begin = 0, per = 1;   // of the row of all tiles: what is left to do, and where sequence b begins
  if (fp.least) {
    const Deal deal(fp, worker);
    at = deal.at, stop = deal.stop, begin = deal.begin, per = deal.per;
    if (at >= stop) return;
    b = __builtin_amdgcn_readfirstlane(deal.b);
  }
  for (;;) {
  // (the lane's number as if it were another for every piece: what follows from it is then computed where it is needed and
  // not kept over the loop, which would cost a fifth of the registers)
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  const int g = lane >> 4, c = lane & 15;
  const uint32_t key_lane = (uint32_t)(c * (int)p.key_token + g * 16);
  const uint32_t value_lane = (uint32_t)(4 * g * (int)p.value_token + c * kSpan * kElt);
  const int length = clamped_length(p, b);
  const Tiles tiles(p, length, p.new_tokens);
  const int first = fp.least ? (int)(at - begin) : 0, end = fp.least ? (int)min((int64_t)tiles.count, stop - begin) : tiles.count;
  const bool split = first > 0 || end < tiles.count;

  // query rows: their positions, and the first product's operand
  int position[kColumns];
  u32x4 q[kColumns][kSteps];
#pragma unroll
  for (int n = 0; n < kColumns; ++n) {
    const int row = row0 + 16 * n + c;
    const int token = (int)p.by_group.quotient((uint32_t)min(row, fp.rows - 1));
    const int head = kv_head * p.group + min(row, fp.rows - 1) - token * p.group;
    position[n] = row < fp.rows ? length - p.new_tokens + token : length - 1;
    const char *at = p.query + ((int64_t)b * p.new_tokens + token) * p.query_token + (int64_t)head * p.query_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = kStepsPerLoad == 1 ? s * 32 + g * 8 : (s >> 1) * 64 + g * 16 + (s & 1) * 8;
      q[n][s] = u32x4{0, 0, 0, 0};
      if (row < fp.rows && (kPlain || d < p.head_size)) q[n][s] = *(const ARCTIC_GLOBAL u32x4 *)(at + d * 2);
    }
  }
  const int first_position = length - p.new_tokens + (int)p.by_group.quotient((uint32_t)row0);

  f32x4 o[kColumns][kSpan], l[kColumns];
  float m[kColumns];
#pragma unroll
  for (int n = 0; n < kColumns; ++n) {
    m[n] = -__builtin_inff();
    l[n] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int a = 0; a < kSpan; ++a) o[n][a] = f32x4{0, 0, 0, 0};
  }

  u32x4 key[2][kLoads];
  Raw<kSpan * kElt> value[8];
  const int32_t *table = p.table + (int64_t)b * p.table_row;
  // The page of key j, or -1 where there is none.  What is loaded for such a key comes from page 0 and is not used.
  auto page_of = [&](int j) {
    if (j >= length) return -1;
    const int page = table[p.by_block.quotient((uint32_t)j)];
    return page >= 0 && page < p.num_blocks ? page : -1;
  };
  // Pages are looked up for tiles ahead, so that no load of keys waits for one: a wave's loads return in order, and one
  // that is waited for has all before it waited for.  kPlain: the two pages of each of the wave's next 32 tiles, tile u
  // of them in the lanes 2u and 2u + 1; else those of one tile's 32 keys.
  auto look_up = [&](int t) {
    if constexpr (kPlain) {
      const int tile = t + (lane >> 1) * kStride;
      return tile < end ? page_of(tiles.start(tile) + 16 * (lane & 1)) : -1;
    } else {
      return t < end ? page_of(tiles.start(t) + (lane & 31)) : -1;
    }
  };
  // a tile's pages: of its two halves (kPlain), of the lane's two keys of K's operand and of its 8 of V's
  struct TilePages {
    int key[2], value[8];
  };
  auto pages_of = [&](int looked_up, int u) {
    TilePages found;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      found.key[h] = kPlain ? __builtin_amdgcn_readlane(looked_up, 2 * u + h) : __shfl(looked_up, 16 * h + c);
#pragma unroll
    for (int i = 0; i < 8; ++i) found.value[i] = kPlain ? found.key[i >> 2] : __shfl(looked_up, 16 * (i >> 2) + 4 * g + (i & 3));
    return found;
  };
  auto load_keys = [&](int start, const TilePages &pages) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = start + 16 * h + (kPlain ? 0 : c);
      const int off = j - (int)p.by_block.quotient((uint32_t)j) * p.block_size;
      const char *at = p.key_cache + max(pages.key[h], 0) * p.key_block + (int64_t)off * p.key_token + (int64_t)kv_head * p.key_head;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if constexpr (kPlain) {
          key[h][i] = *(const ARCTIC_GLOBAL u32x4 *)(at + key_lane + i * 64);
        } else {
          key[h][i] = u32x4{0, 0, 0, 0};
          if (i * (64 / kElt) + g * (16 / kElt) < p.head_size) key[h][i] = *(const ARCTIC_GLOBAL u32x4 *)(at + g * 16 + i * 64);
        }
      }
    }
  };
  auto load_values = [&](int start, const TilePages &pages) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (kPlain) {
        const int j = start + 16 * h;
        const int off = j - (int)p.by_block.quotient((uint32_t)j) * p.block_size;
        const char *at = p.value_cache + max(pages.value[4 * h], 0) * p.value_block + (int64_t)off * p.value_token +
                         (int64_t)kv_head * p.value_head;
#pragma unroll
        for (int i = 0; i < 4; ++i) value[4 * h + i].load(at + (int64_t)i * p.value_token + value_lane);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = start + 16 * h + 4 * g + i;
          const int off = j - (int)p.by_block.quotient((uint32_t)j) * p.block_size;
          value[4 * h + i] = {};
          if (c * kSpan < p.head_size)
            value[4 * h + i].load(p.value_cache + max(pages.value[4 * h + i], 0) * p.value_block + (int64_t)off * p.value_token +
                                  (int64_t)kv_head * p.value_head + c * kSpan * kElt);
        }
      }
    }
  };

  // V's operand: word w of row tile a pairs the keys 2w and 2w + 1
  auto operand = [&](int a) {
    u32x4 v;
    if constexpr (kElt == 2) {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        v[w] = __builtin_amdgcn_perm(value[2 * w + 1].w[a >> 1], value[2 * w].w[a >> 1], (a & 1) ? 0x07060302u : 0x05040100u);
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // both keys' elements a and a + 1 (a even): k0[a] k1[a] k0[a + 1] k1[a + 1]
        const uint32_t four = __builtin_amdgcn_perm(value[2 * w + 1].w[a >> 2], value[2 * w].w[a >> 2], (a & 2) ? 0x07030602u : 0x05010400u);
        v[w] = (a & 1) ? widen<true>(T{}, C{}, four) : widen<false>(T{}, C{}, four);
      }
    }
    return v;
  };
  auto scores = [&](f32x4 (&s)[kColumns][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < kColumns; ++n) s[n][h] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if constexpr (kStepsPerLoad == 1) {
#pragma unroll
          for (int n = 0; n < kColumns; ++n) s[n][h] = mfma16(T{}, key[h][i], q[n][i], s[n][h]);
        } else {
          const u32x4 &w = key[h][i];
          const u32x4 lo = {widen<false>(T{}, C{}, w.x), widen<true>(T{}, C{}, w.x), widen<false>(T{}, C{}, w.y), widen<true>(T{}, C{}, w.y)};
          const u32x4 hi = {widen<false>(T{}, C{}, w.z), widen<true>(T{}, C{}, w.z), widen<false>(T{}, C{}, w.w), widen<true>(T{}, C{}, w.w)};
#pragma unroll
          for (int n = 0; n < kColumns; ++n) s[n][h] = mfma16(T{}, lo, q[n][2 * i], s[n][h]);
#pragma unroll
          for (int n = 0; n < kColumns; ++n) s[n][h] = mfma16(T{}, hi, q[n][2 * i + 1], s[n][h]);
        }
      }
    }
  };
  // column tile n's scores (base 2, -inf where a key is not seen) into its weights; m, l and o follow the maximum
  auto weigh = [&](int n, const float (&z)[8]) {
    float top = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7])));
    top = max_over_groups(top);
    if (__any(top > m[n])) {
      const float now = fmaxf(m[n], top);
      const float keep = __builtin_amdgcn_exp2f(m[n] - (now == -__builtin_inff() ? 0.f : now));
      m[n] = now;
      l[n] *= keep;
#pragma unroll
      for (int a = 0; a < kSpan; ++a) o[n][a] *= keep;
    }
    const float base = m[n] == -__builtin_inff() ? 0.f : m[n];
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __builtin_amdgcn_exp2f(z[i] - base);
    return u32x4{T::pack(w[0], w[1]), T::pack(w[2], w[3]), T::pack(w[4], w[5]), T::pack(w[6], w[7])};
  };

  // ---- tiles that every row sees whole: keys of the next one are requested before the weights of this one, its values
  // behind the last product with this one's.  Up to a tile with a page that is not there.
  const int whole_begin = max(tiles.window_tile, p.window > 0 && length > p.window ? ((length - 1 - p.window) >> 5) + 1 : 0),
            whole_end = first_position >= 31 ? ((first_position - 31) >> 5) + 1 : 0;
  const int from = max(first, whole_begin - tiles.window_tile + tiles.sink_tiles),
            to = min(end, whole_end - tiles.window_tile + tiles.sink_tiles);
  const int whole_first = first + wave + (max(0, from - first - wave) + kStride - 1) / kStride * kStride;
  auto there = [&](const TilePages &pages) {
    if constexpr (kPlain) return pages.value[0] >= 0 && pages.value[4] >= 0;
    bool all = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) all = all && pages.value[i] >= 0;
    return (bool)__all(all);
  };
  int t = whole_first, u = 0;   // the tile, and its place among the looked-up ones
  {
    int looked_up = look_up(t);
    TilePages pages = pages_of(looked_up, 0);
    bool more = t < to && there(pages);
    if (more) {
      load_keys(tiles.start(t), pages);
      if constexpr (!kPlain) looked_up = look_up(t + kStride);
      load_values(tiles.start(t), pages);
    }
    while (more) {
      f32x4 s[kColumns][2];
      scores(s);
      t += kStride;
      more = t < to;
      if (more) {
        u = kPlain ? (u + 1) & 31 : 0;
        if (kPlain && u == 0) looked_up = look_up(t);
        pages = pages_of(looked_up, u);
        more = there(pages);
      }
      if (more) load_keys(tiles.start(t), pages);
      u32x4 weight[kColumns];
#pragma unroll
      for (int n = 0; n < kColumns; ++n) {
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = s[n][i >> 2][i & 3] * scale;
        weight[n] = weigh(n, z);
        l[n] = mfma16(T{}, ones, weight[n], l[n]);
      }
#pragma unroll
      for (int a = 0; a < kSpan; ++a) {
        const u32x4 v = operand(a);
#pragma unroll
        for (int n = 0; n < kColumns; ++n) o[n][a] = mfma16(T{}, v, weight[n], o[n][a]);
      }
      if (more) {
        if constexpr (!kPlain) looked_up = look_up(t + kStride);
        load_values(tiles.start(t), pages);
      }
    }
  }

  // ---- the others, one after the other
  const int whole_stop = t;
  for (t = first + wave; t < end; t += kStride) {
    if (t == whole_first && whole_stop > t) {
      t = whole_stop - kStride;
      continue;
    }
    const int start = tiles.start(t);
    const TilePages pages = pages_of(look_up(t), 0);
    load_keys(start, pages);
    load_values(start, pages);
    f32x4 s[kColumns][2];
    scores(s);
    u32x4 weight[kColumns];
    auto sees = [&](int i, int position) {   // the lane's key i
      const int j = start + 16 * (i >> 2) + 4 * g + (i & 3);
      return pages.value[i] >= 0 && j <= position && (j >= window_start(p, position) || j < p.sinks);
    };
#pragma unroll
    for (int n = 0; n < kColumns; ++n) {
      float z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = sees(i, position[n]) ? s[n][i >> 2][i & 3] * scale : -__builtin_inff();
      weight[n] = weigh(n, z);
      l[n] = mfma16(T{}, ones, weight[n], l[n]);
    }
    // A weight of zero must not meet an infinity or a NaN: what no row sees is cleared; of what some rows see and others
    // do not, the finite elements are taken as ever, and of the rest a product with the keys' visibility counts, for
    // every row and element, what the row sees: an infinity as 1, a negative one as 64, a NaN as 4096, of 32 keys at most.
    bool careful = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = start + 16 * (i >> 2) + 4 * g + (i & 3);
      if (!(pages.value[i] >= 0 && j < length && (j >= window_start(p, first_position) || j < p.sinks))) value[i] = {};
#pragma unroll
      for (int w = 0; w < kSpan * kElt / 4; ++w) {
        if constexpr (kElt == 2) careful |= unusual(T{}, value[i].w[w]);
        else careful |= unusual(T{}, widen<false>(T{}, C{}, value[i].w[w])) || unusual(T{}, widen<true>(T{}, C{}, value[i].w[w]));
      }
    }
    careful = __any(careful);
#pragma unroll
    for (int a = 0; a < kSpan; ++a) {
      u32x4 v = operand(a);
      if (careful) {
        u32x4 codes;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          codes[w] = unusual_codes(T{}, v[w]);
          v[w] &= (codes[w] & 0xffffu ? 0u : 0xffffu) | (codes[w] >> 16 ? 0u : 0xffff0000u);
        }
#pragma unroll
        for (int n = 0; n < kColumns; ++n) {
          u32x4 seen;
#pragma unroll
          for (int w = 0; w < 4; ++w) seen[w] = one & ((weight[n][w] & 0xffffu ? 0xffffu : 0u) | (weight[n][w] >> 16 ? 0xffff0000u : 0u));
          const f32x4 count = mfma16(T{}, codes, seen, f32x4{0, 0, 0, 0});
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][a][i] += unusual_sum((int)count[i]);
        }
      }
#pragma unroll
      for (int n = 0; n < kColumns; ++n) o[n][a] = mfma16(T{}, v, weight[n], o[n][a]);
    }
  }

  // ---- the waves' parts of a head, joined in LDS in the order of the waves ---------------------------------------
#pragma unroll
  for (int n = 0; n < kColumns; ++n)
    if (g == 0) {
      tops[all_waves][16 * n + c] = m[n];
      sums[all_waves][16 * n + c] = l[n][0];
    }
  __syncthreads();
  float top[kColumns], sum[kColumns], mine[kColumns];
#pragma unroll
  for (int n = 0; n < kColumns; ++n) {
    top[n] = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kStride; ++w) top[n] = fmaxf(top[n], tops[head_at * kStride + w][16 * n + c]);
    const float base = top[n] == -__builtin_inff() ? 0.f : top[n];
    sum[n] = 0.f;
#pragma unroll
    for (int w = 0; w < kStride; ++w)
      sum[n] += sums[head_at * kStride + w][16 * n + c] * __builtin_amdgcn_exp2f(tops[head_at * kStride + w][16 * n + c] - base);
    mine[n] = __builtin_amdgcn_exp2f(m[n] - base);
  }
  for (int w = 0; w < kStride; ++w) {
    if (w == wave) {
#pragma unroll
      for (int n = 0; n < kColumns; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int a = 0; a < kSpan; ++a) {
            float &to_join = joined[head_at][16 * n + c][(4 * g + i) * kSpan + a];
            to_join = (w ? to_join : 0.f) + o[n][a][i] * mine[n];
          }
    }
    __syncthreads();
  }
  if (fp.least && first == 0 && kv_head == 0 && row0 == 0 && wave == 0 && lane == 0)
    fp.dealt[b] = make_int2((int)(begin / per), (int)((begin + tiles.count - 1) / per));
  // a head's result by its waves; a worker has at most one piece that goes on with a sequence (the first place) and one
  // that begins one and does not end it (the second)
  const int64_t place = (int64_t)kv_head * 2 * fp.workers + 2 * worker + (first == 0 ? 1 : 0);
  if (split && wave == 0 && g == 0) {
#pragma unroll
    for (int n = 0; n < kColumns; ++n)
      if (row0 + 16 * n + c < fp.rows) {
        float *st = fp.statistics + (place * fp.rows + row0 + 16 * n + c) * 2;
        st[0] = top[n];
        st[1] = sum[n];
      }
  }
  // (the barrier of the last wave's turn stands between the reads of these and the writes)
  const float v_scale = p.v_scale ? *p.v_scale : 1.f;
  if (wave == 0 && g == 0) {
#pragma unroll
    for (int n = 0; n < kColumns; ++n) tops[head_at][16 * n + c] = sum[n] == 0.f ? 0.f : v_scale / sum[n];
  }
  __syncthreads();
  const int chunks = p.head_size / 8;   // of 8 elements
  for (int k = wave * 64 + lane; k < kRows * (kPadded / 8); k += 64 * kStride) {
    const int r = k / (kPadded / 8), chunk = k % (kPadded / 8), row = row0 + r;
    if (row >= fp.rows || chunk >= chunks) continue;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = joined[head_at][r][chunk * 8 + i];
    if (split) {
      float *to = fp.partial + (place * fp.rows + row) * p.head_size + chunk * 8;
      *(ARCTIC_GLOBAL f32x4 *)to = f32x4{x[0], x[1], x[2], x[3]};
      *(ARCTIC_GLOBAL f32x4 *)(to + 4) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
      const int token = (int)p.by_group.quotient((uint32_t)row), head = kv_head * p.group + row - token * p.group;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= tops[head_at][r];
      const uint4 v = pack8<T>(x);
      *(ARCTIC_GLOBAL u32x4 *)(p.out + ((int64_t)b * p.new_tokens + token) * p.out_token + (int64_t)head * p.out_head + chunk * 16) =
          u32x4{v.x, v.y, v.z, v.w};
    }
  }
  if (!fp.least) return;
  at = begin + end;
  if (at >= stop) return;
  begin += tiles.count;   // the piece ended with its sequence: the next one
  ++b;
  __syncthreads();
  }
}

// Sequences that were dealt to several workers: out = v_scale sum_w 2^(m_w - M) o_w / sum_w 2^(m_w - M) l_w, a wave per
// row.  kPadded / 4 lanes take a piece's values, 256 / kPadded pieces at a time and four such groups requested ahead.
// 3 to 7 us, a launch and three memory latencies.  (In the kernel itself, by the worker that ends last: 16 to 28 us more,
// for the pieces then pass through the memory that all XCDs see.)
constexpr int kJoinWaves = 4;
template <typename T, int kPadded>
__global__ __launch_bounds__(64 * kJoinWaves) void attention_join_kernel(const FewParams fp) {
  const AttentionParams &p = fp.a;
  constexpr int kLanes = kPadded / 4, kSide = 64 / kLanes, kAhead = 4;
  const int lane = threadIdx.x & 63, side = lane / kLanes, d = lane % kLanes * 4;
  const uint32_t at = blockIdx.x * kJoinWaves + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const uint32_t token = p.by_heads.quotient(at);   // b * new_tokens + i
  if (token >= p.total_tokens) return;
  const int head = (int)(at - token * (uint32_t)p.heads);
  const int b = (int)p.by_new.quotient(token), i = (int)token - b * p.new_tokens;
  const int2 dealt = fp.dealt[b];
  const int first = dealt.x, last = dealt.y;
  if (first == last) return;   // written by the worker
  const int kv_head = (int)p.by_group.quotient((uint32_t)head);
  const int row = i * p.group + head - kv_head * p.group;
  const int64_t place = (int64_t)kv_head * 2 * fp.workers;
  // the first worker's piece begins the sequence, the others' go on with it
  auto piece = [&](int w) { return (place + 2 * w + (w == first ? 1 : 0)) * fp.rows + row; };
  float top = -__builtin_inff(), sum = 0.f;
  f32x4 acc = {0, 0, 0, 0};
  for (int w0 = first; w0 <= last; w0 += kSide * kAhead) {
    float2 st[kAhead];
    f32x4 part[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int w = w0 + k * kSide + side;
      st[k] = make_float2(-__builtin_inff(), 0.f);
      part[k] = f32x4{0, 0, 0, 0};
      if (w <= last) {
        st[k] = *(const float2 *)(fp.statistics + piece(w) * 2);
        if (d < p.head_size) part[k] = *(const ARCTIC_GLOBAL f32x4 *)(fp.partial + piece(w) * p.head_size + d);
      }
    }
    float now = top;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) now = fmaxf(now, st[k].x);
    const float base = now == -__builtin_inff() ? 0.f : now, keep = __builtin_amdgcn_exp2f(top - base);
    sum *= keep;
    acc *= keep;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const float own = __builtin_amdgcn_exp2f(st[k].x - base);
      sum += st[k].y * own;
      acc += part[k] * own;
    }
    top = now;
  }
  // the sides' results
#pragma unroll
  for (int s = kLanes; s < 64; s <<= 1) {
    const float other = __shfl_xor(top, s), now = fmaxf(top, other), base = now == -__builtin_inff() ? 0.f : now;
    const float keep = __builtin_amdgcn_exp2f(top - base);
    sum *= keep;
    acc *= keep;
    sum += __shfl_xor(sum, s);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] += __shfl_xor(acc[k], s);
    top = now;
  }
  if (side || d >= p.head_size) return;
  acc *= sum == 0.f ? 0.f : (p.v_scale ? *p.v_scale : 1.f) / sum;
  *(ARCTIC_GLOBAL u32x2 *)(p.out + (int64_t)token * p.out_token + (int64_t)head * p.out_head + d * 2) =
      u32x2{T::pack(acc[0], acc[1]), T::pack(acc[2], acc[3])};
}

struct FewShape {
  int padded, columns, heads, row_tiles, workers, least;
  bool plain;
};
void few_launch_bf16(const FewParams &p, const FewShape &f, int kv, hipStream_t s);
void few_launch_f16(const FewParams &p, const FewShape &f, int kv, hipStream_t s);

template <typename T, typename C, int kPadded, int kColumns>
inline void few_launch_plain(const FewParams &p, const FewShape &f, dim3 grid, hipStream_t s) {
  constexpr int kShared = kPadded * C::kBytes <= 64 ? 4 : kPadded * C::kBytes <= 128 ? 2 : 1;
  if (f.plain && f.heads > 1) launch(attention_few_kernel<T, C, kPadded, kColumns, kShared, true>, grid, 64 * kFewWaves, s, p);
  else if (f.plain) launch(attention_few_kernel<T, C, kPadded, kColumns, 1, true>, grid, 64 * kFewWaves, s, p);
  else launch(attention_few_kernel<T, C, kPadded, kColumns, 1, false>, grid, 64 * kFewWaves, s, p);
}
template <typename T, typename C, int kPadded>
inline void few_launch_columns(const FewParams &p, const FewShape &f, dim3 grid, hipStream_t s) {
  if (f.columns == 1) return few_launch_plain<T, C, kPadded, 1>(p, f, grid, s);
  if constexpr (kPadded == 64)
    if (f.columns == 4) return few_launch_plain<T, C, kPadded, 4>(p, f, grid, s);
  few_launch_plain<T, C, kPadded, 2>(p, f, grid, s);
}
template <typename T, typename C>
inline void few_launch_padded(const FewParams &p, const FewShape &f, dim3 grid, hipStream_t s) {
  if (f.padded == 64) few_launch_columns<T, C, 64>(p, f, grid, s);
  else if (f.padded == 128) few_launch_columns<T, C, 128>(p, f, grid, s);
  else few_launch_columns<T, C, 256>(p, f, grid, s);
}
template <typename T>
inline void few_launch(const FewParams &p, const FewShape &f, int kv, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)f.workers * (p.a.kv_heads / f.heads) * f.row_tiles));
  if (kv == ARCTIC_KV_AUTO) few_launch_padded<T, Half<T>>(p, f, grid, s);
  else if (kv == ARCTIC_KV_FP8_E4M3) few_launch_padded<T, CacheE4M3>(p, f, grid, s);
  else few_launch_padded<T, CacheE5M2>(p, f, grid, s);
  if (!f.least) return;
  const dim3 rows((unsigned)((p.a.total_tokens * p.a.heads + kJoinWaves - 1) / kJoinWaves));
  if (f.padded == 64) launch(attention_join_kernel<T, 64>, rows, 64 * kJoinWaves, s, p);
  else if (f.padded == 128) launch(attention_join_kernel<T, 128>, rows, 64 * kJoinWaves, s, p);
  else launch(attention_join_kernel<T, 256>, rows, 64 * kJoinWaves, s, p);
}

}  // namespace arctic
