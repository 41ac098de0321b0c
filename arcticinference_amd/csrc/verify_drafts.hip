// Verification of drafted tokens against the target model's logits, gfx950.
//
// Two launches.  The first walks every row of logits in segments, one wave each: the segment's argmax and, relative
// to its maximum, the sum of its weights exp((x - m) / T) without the drafted token's.  The second, one workgroup per
// request, joins the segments of the request's rows, runs down its drafts to the first that is not accepted, finds the
// segment in which the running sum passes the drawn number and walks that segment alone.
//
// The sums decide whole numbers: with 128256 weights there are as many borders, and an error of 2^-24 in them would move
// one past the drawn number in about one request of a hundred.  They and the weights are therefore held in fp64.  The
// drafted token is left out of the segments' sums and added where it belongs, so that what remains of a row whose draft
// holds nearly everything is no difference of nearly equal numbers.
//
// The first launch reads the logits once: 160 requests with up to 7 drafts, 128257 fp32 logits a row, 75 us, 5.0 TB/s.  With
// 16-bit logits the fp64 arithmetic takes longer than the reading: 64 requests with up to 5 drafts, 128256 bf16 logits, 24 us,
// 2.3 TB/s.  The second is a row of latencies, 6 to 9 us.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "winner.hpp"

namespace arctic {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kVerifyLanes = 256;
constexpr int kVerifySegment = 2048;
constexpr int kVerifyPerLane = kVerifySegment / kVerifyLanes;   // where a workgroup walks a segment

struct VerifySegment {
  double sum;     // of the weights relative to the segment's maximum, without the draft's
  uint64_t key;   // the segment's maximum, and its argmax where no token is drawn: of a temperature that is not positive, and
                  // of a maximum that is not finite
};

struct VerifyParams {
  int64_t *out_tokens, *out_counts;
  const char *logits;
  const int32_t *row_start;
  const int64_t *drafts;
  const float *accept, *sample, *temperatures;
  VerifySegment *segments;   // [batch][max_drafts + 1][parts]
  int64_t row_stride_bytes, draft_stride, accept_stride, num_rows;
  int vocab, max_drafts, parts;
  uint32_t places;   // batch * (max_drafts + 1)
  Divisor by_parts, by_places;   // by_places: max_drafts + 1
};

template <int kDtype>
__device__ __forceinline__ float logit(const char *row, int i) {
  if constexpr (kDtype == ARCTIC_DTYPE_F32) return ((const ARCTIC_GLOBAL float *)row)[i];
  const uint32_t bits = ((const ARCTIC_GLOBAL uint16_t *)row)[i];
  return kDtype == ARCTIC_DTYPE_BF16 ? BF16::lo(bits) : F16::lo(bits);
}

// kChunks chunks of 16 bytes of logits, `stride` logits from one to the next, from `first` on; rows may start anywhere.
// -inf for logits at `end` and beyond, where the wave's chunks reach it (`last`: the wave's last logit and one).  Returns
// their sum (two 16-bit ones to an instruction): NaN if there is a NaN among them, or infinities of both signs.
template <int kDtype, int kChunks>
__device__ __forceinline__ float some_logits(const char *row, int first, int stride, int last, int end,
                                            float (&x)[kChunks][kDtype == ARCTIC_DTYPE_F32 ? 4 : 8]) {
  constexpr int kElt = kDtype == ARCTIC_DTYPE_F32 ? 4 : 2, kPerChunk = 16 / kElt;
  float sum = 0.f;
  if (last <= end) {
    uint4 raw[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) raw[i] = load16<true>(row + (int64_t)(first + i * stride) * kElt);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      if constexpr (kDtype == ARCTIC_DTYPE_F32) {
        x[i][0] = __uint_as_float(raw[i].x), x[i][1] = __uint_as_float(raw[i].y);
        x[i][2] = __uint_as_float(raw[i].z), x[i][3] = __uint_as_float(raw[i].w);
        sum += (x[i][0] + x[i][1]) + (x[i][2] + x[i][3]);
      } else {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kDtype == ARCTIC_DTYPE_BF16) {
            const bf16x2 ones = {(__bf16)1.f, (__bf16)1.f};
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w[j]), ones, sum, false);
            x[i][2 * j] = BF16::lo(w[j]), x[i][2 * j + 1] = BF16::hi(w[j]);
          } else {
            const f16x2 ones = {(_Float16)1.f, (_Float16)1.f};
            sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w[j]), ones, sum, false);
            x[i][2 * j] = F16::lo(w[j]), x[i][2 * j + 1] = F16::hi(w[j]);
          }
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < kPerChunk; ++j) {
        const int at = first + i * stride + j;
        x[i][j] = at < end ? logit<kDtype>(row, at) : -__builtin_inff();
        sum += at < end ? x[i][j] : 0.f;
      }
  }
  return sum;
}

// The value that a key was made of (NaN for any NaN, -inf for no key).
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  if (o == 0xffffffffu) return __builtin_nanf("");
  if (o == 0) return -__builtin_inff();
  return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

// 2^((x - m) c) in fp64, relative error 2e-14, for x <= m: with (x - m) c = n + f, n whole (found by adding 1.5 2^52, whose
// last bit is worth 1) and |f| <= 1/2, 2^f by its Chebyshev interpolation of degree 9 there.  (One product and difference in
// place of the difference and the product would do for temperatures about 1; at 1e-30 it leaves x = m with a weight that is
// not 1.)
__device__ __forceinline__ double power_of_fraction(double f) {
  double v = 0x1.b6571ea79d565p-24;
  v = fma(v, f, 0x1.63ef969b0e64ep-20);
  v = fma(v, f, 0x1.ffcb7677a5f5cp-17);
  v = fma(v, f, 0x1.43088e257e65bp-13);
  v = fma(v, f, 0x1.5d87fe908fed1p-10);
  v = fma(v, f, 0x1.3b2ab72b175f8p-7);
  v = fma(v, f, 0x1.c6b08d7044115p-5);
  v = fma(v, f, 0x1.ebfbdff8149f2p-3);
  v = fma(v, f, 0x1.62e42fefa39f7p-1);
  return fma(v, f, 0x1.000000000003dp+0);
}
constexpr double kWholeBits = 6755399441055744.0;   // 1.5 2^52
// for any x, -inf among them, and any c: 0 below 2^-1074
__device__ __forceinline__ double weight_of(double x, double m, double c) {
  const double t = fmax((x - m) * c, -1100.0);
  const double shifted = t + kWholeBits;
  return __builtin_amdgcn_ldexp(power_of_fraction(t - (shifted - kWholeBits)), (int)(uint32_t)__double_as_longlong(shifted));
}
// where (x - m) c is known to be above -1020: the exponent takes n as it is.  (fp64 maxima, scalings and conversions run at a
// fraction of the products' rate.)
__device__ __forceinline__ double weight_in_range(double x, double m, double c) {
  const double d = x - m, shifted = fma(d, c, kWholeBits);
  const double v = power_of_fraction(fma(d, c, -(shifted - kWholeBits)));
  return __hiloint2double(__double2hiint(v) + ((int)(uint32_t)__double_as_longlong(shifted) << 20), __double2loint(v));
}
// What a segment's 2048 weights below 2^-1001, logits at the end of that range and beyond, may add up to counts as none.
constexpr double kLeastSum = 0x1p-980;
// c for temperature t: log2(e) / t
__device__ __forceinline__ double per_unit(float t) { return 1.4426950408889634074 / (double)t; }

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }

// The same sum in every lane: inside the rows of 16 lanes by DPP, then the four rows'.
template <int kCtrl>
__device__ __forceinline__ double dpp_add64(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), kCtrl, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), kCtrl, 0xf, 0xf, true);
  return v + __hiloint2double(hi, lo);
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v = dpp_add64<0xB1>(v);    // quad_perm [1,0,3,2]
  v = dpp_add64<0x4E>(v);    // quad_perm [2,3,0,1]
  v = dpp_add64<0x141>(v);   // row_half_mirror
  v = dpp_add64<0x140>(v);   // row_mirror
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
// the sum of a lane's value and those of the lanes before it
__device__ __forceinline__ double sum_up_to(double v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double other = __shfl_up(v, d);
    if (lane >= d) v += other;
  }
  return v;
}

// The rows of request b: the first one and the number of drafts, -1 where it has no row.
__device__ __forceinline__ int drafts_of(const VerifyParams &p, int b, int64_t *start) {
  const int64_t first = p.row_start[b], end = min((int64_t)p.row_start[b + 1], p.num_rows);
  *start = first;
  return first < 0 || end <= first ? -1 : (int)min((int64_t)p.max_drafts, end - first - 1);
}

// A segment per wave: nothing is shared and nothing waited for but the logits, 64 or 128 bytes a lane.  (Segments of 4096
// by workgroups of 256 lanes, with three barriers, took 26.6 us where this takes 24 of 64 requests' 219 rows of 128256
// bf16 logits.)
template <int kDtype>
__global__ __launch_bounds__(kVerifyLanes) void verify_segments_kernel(const VerifyParams p) {
  constexpr int kChunk = kDtype == ARCTIC_DTYPE_F32 ? 4 : 8, kLoads = kVerifySegment / 64 / kChunk;
  const uint32_t unit = blockIdx.x * (kVerifyLanes / 64) + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const uint32_t place = p.by_parts.quotient(unit);   // b * (max_drafts + 1) + k
  const int part = (int)(unit - place * (uint32_t)p.parts);
  if (place >= p.places) return;
  const int b = (int)p.by_places.quotient(place), k = (int)(place - (uint32_t)b * (uint32_t)(p.max_drafts + 1));
  int64_t start;
  const int n = drafts_of(p, b, &start);
  if (k > n) return;
  const char *row = p.logits + (start + k) * p.row_stride_bytes;
  const int lane = threadIdx.x & 63, first = part * kVerifySegment, end = min(p.vocab, first + kVerifySegment);
  // neighbouring lanes take neighbouring chunks
  float x[kLoads][kChunk];
  const float probe = some_logits<kDtype, kLoads>(row, first + lane * kChunk, 64 * kChunk, first + kVerifySegment, p.vocab, x);
  const float t = p.temperatures ? p.temperatures[b] : 1.f;
  const int64_t draft = k < n ? p.drafts[b * p.draft_stride + k] : -1;
  // the lane's maximum; a NaN is above every number, and is looked for only where a sum says that there may be one
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
#pragma unroll
    for (int j = 0; j < kChunk; j += 2) top = fmaxf(fmaxf(top, x[i][j]), x[i][j + 1]);
  // (a value by another name: what is asked of it must not be worked out beforehand and thrown away)
  auto renamed = [](float v) {
    asm volatile("" : "+v"(v));
    return v;
  };
  if (__any(probe != probe)) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        const float v = renamed(x[i][j]);
        if (v != v) top = __builtin_nanf("");
      }
  }
  const uint32_t mine = (uint32_t)(winner_key(top, 0) >> 32), all_top = wave_max<4>(mine);
  const float m = key_value((uint64_t)all_top << 32);
  const bool drawn = t > 0.f && finite(m);
  uint32_t not_lowest = 0;   // the complement of the lowest index that has the maximum, where it is asked for
  if (!drawn) {
    int at = 0x7fffffff;
    if (mine == all_top) {
#pragma unroll
      for (int i = kLoads - 1; i >= 0; --i)
#pragma unroll
        for (int j = kChunk - 1; j >= 0; --j) {
          const int index = first + (i * 64 + lane) * kChunk + j;
          const float v = renamed(x[i][j]);
          if (index < end && (v == m || (m != m && v != v))) at = index;
        }
    }
    not_lowest = wave_max<4>(~(uint32_t)at);
  }
  double sum = 0.0;
  if (drawn) {
    const double c = per_unit(t);
    if (draft >= first && draft < end) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
          if (first + (i * 64 + lane) * kChunk + j == draft) x[i][j] = -__builtin_inff();
    }
    // Below `lowest` weights are as good as none.  Where the type's steps are too wide to say so (tiny temperatures), or its
    // range too narrow (huge ones), every weight is looked at.
    const float lowest = (float)((double)m - 1010.0 / c);
    const double span = ((double)m - (double)lowest) * c;
    if (span > 1001.0 && span < 1020.0) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          float v;   // (no NaN is left here that fmaxf would first have to quieten)
          asm("v_max_f32 %0, %1, %2" : "=v"(v) : "v"(x[i][j]), "v"(lowest));
          sum += weight_in_range(v, m, c);
        }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) sum += weight_of(x[i][j], m, c);
    }
    sum = wave_sum64(sum);
    sum = sum < kLeastSum ? 0.0 : sum;
  }
  if (lane == 0) p.segments[unit] = {sum, (uint64_t)all_top << 32 | not_lowest};
}

template <int kDtype>
__global__ __launch_bounds__(kVerifyLanes) void verify_requests_kernel(const VerifyParams p) {
  constexpr int kWaves = kVerifyLanes / 64;
  __shared__ int rejected;          // the first row whose draft is not accepted, n at the end
  __shared__ uint64_t row_key_at;   // of that row
  __shared__ double target_at;
  __shared__ int segment_at;
  __shared__ double wave_sums[kWaves];
  __shared__ int passes_at[kWaves], some_at[kWaves];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t start;
  const int n = drafts_of(p, b, &start);
  int64_t *tokens = p.out_tokens + (int64_t)b * (p.max_drafts + 1);
  if (n < 0) {
    for (int k = threadIdx.x; k <= p.max_drafts; k += kVerifyLanes) tokens[k] = -1;
    if (threadIdx.x == 0) p.out_counts[b] = 0;
    return;
  }
  const float t = p.temperatures ? p.temperatures[b] : 1.f;
  const double c = t > 0.f ? per_unit(t) : 0.0;
  const VerifySegment *segments = p.segments + (int64_t)b * (p.max_drafts + 1) * p.parts;
  if (threadIdx.x == 0) rejected = n;
  __syncthreads();
  // the weights of a segment, relative to the row's maximum m
  auto segment_sum = [&](const VerifySegment &g, float m) {
    const float own = key_value(g.key);
    return own == -__builtin_inff() ? 0.0 : g.sum * weight_of(own, m, c);
  };
  for (int k = wave; k < n; k += kWaves) {
    const int64_t draft = p.drafts[b * p.draft_stride + k];
    const bool known = draft >= 0 && draft < p.vocab;
    const float x = known ? logit<kDtype>(p.logits + (start + k) * p.row_stride_bytes, (int)draft) : 0.f;
    const float u = p.accept[b * p.accept_stride + k];
    const VerifySegment one = lane < p.parts ? segments[(int64_t)k * p.parts + lane] : VerifySegment{0.0, 0};
    uint64_t key = one.key;
    for (int s = 64 + lane; s < p.parts; s += 64) key = max(key, segments[(int64_t)k * p.parts + s].key);
    key = wave_winner(key);
    const float m = key_value(key);
    bool accepted = false;
    if (finite(m) && known) {
      if (t > 0.f) {
        double sum = lane < p.parts ? segment_sum(one, m) : 0.0;
        for (int s = 64 + lane; s < p.parts; s += 64) sum += segment_sum(segments[(int64_t)k * p.parts + s], m);
        sum = wave_sum64(sum);
        const double own = weight_of(x, m, c);
        accepted = (double)u * (sum + own) < own;
      } else {
        accepted = draft == winner_index(key);
      }
    }
    if (!accepted && lane == 0) atomicMin(&rejected, k);
  }
  __syncthreads();
  const int a = rejected;
  const char *row = p.logits + (start + a) * p.row_stride_bytes;
  const int64_t draft = a < n ? p.drafts[b * p.draft_stride + a] : -1;
  for (int k = threadIdx.x; k <= p.max_drafts; k += kVerifyLanes)
    if (k != a) tokens[k] = k < a ? p.drafts[b * p.draft_stride + k] : -1;
  if (threadIdx.x == 0) p.out_counts[b] = a + 1;
  if (wave == 0) {
    const VerifySegment one = lane < p.parts ? segments[(int64_t)a * p.parts + lane] : VerifySegment{0.0, 0};
    uint64_t key = one.key;
    for (int s = 64 + lane; s < p.parts; s += 64) key = max(key, segments[(int64_t)a * p.parts + s].key);
    key = wave_winner(key);
    const float m = key_value(key);
    int at = -1;
    if (t > 0.f && finite(m)) {
      auto mine_of = [&](int s0) {
        if (s0 + lane >= p.parts) return 0.0;
        return segment_sum(s0 ? segments[(int64_t)a * p.parts + s0 + lane] : one, m);
      };
      double total = 0.0;
      for (int s0 = 0; s0 < p.parts; s0 += 64) total += mine_of(s0);
      total = wave_sum64(total);
      if (total > 0.0) {
        // the first segment whose running sum passes the drawn number, or the last that has any weight
        const double target = (double)p.sample[b] * total;
        double before = 0.0;
        for (int s0 = 0; s0 < p.parts; s0 += 64) {
          const double mine = mine_of(s0), upto = before + sum_up_to(mine, lane);
          const uint64_t passes = __ballot(mine > 0.0 && upto > target), some = __ballot(mine > 0.0);
          const int l = passes ? __builtin_ctzll(passes) : some ? 63 - __builtin_clzll(some) : -1;
          if (l >= 0) {
            at = s0 + l;
            if (lane == l) target_at = target - (upto - mine);
          }
          if (passes) break;
          before = __shfl(upto, 63);
        }
      }
    }
    if (lane == 0) {
      segment_at = at;
      row_key_at = key;
    }
  }
  __syncthreads();
  const uint64_t key = row_key_at;
  // the argmax: of a row with a distribution in which no other token has any weight the rejected draft
  const int64_t otherwise = t > 0.f && finite(key_value(key)) ? draft : (int64_t)winner_index(key);
  if (segment_at < 0) {
    if (threadIdx.x == 0) tokens[a] = otherwise;
    return;
  }
  // the segment's weights, relative to the row's maximum as the sums before; each lane takes consecutive elements
  const float m = key_value(key);
  const int first = segment_at * kVerifySegment + (int)threadIdx.x * kVerifyPerLane;
  constexpr int kChunk = kDtype == ARCTIC_DTYPE_F32 ? 4 : 8;
  float x[kVerifyPerLane / kChunk][kChunk];
  some_logits<kDtype, kVerifyPerLane / kChunk>(row, first, kChunk, segment_at * kVerifySegment + kVerifySegment, p.vocab, x);
  double w[kVerifyPerLane], mine = 0.0;
#pragma unroll
  for (int i = 0; i < kVerifyPerLane; ++i) {
    w[i] = first + i == draft ? 0.0 : weight_of(x[i / kChunk][i % kChunk], m, c);
    mine += w[i];
  }
  double upto = sum_up_to(mine, lane);
  if (lane == 63) wave_sums[wave] = upto;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kWaves; ++k) upto += k < wave ? wave_sums[k] : 0.0;
  const uint64_t passes = __ballot(mine > 0.0 && upto > target_at), some = __ballot(mine > 0.0);
  if (lane == 0) {
    passes_at[wave] = passes ? __builtin_ctzll(passes) : -1;
    some_at[wave] = some ? 63 - __builtin_clzll(some) : -1;
  }
  __syncthreads();
  int chosen = -1;   // the first lane whose running sum passes, or the last that has any weight
#pragma unroll
  for (int k = 0; k < kWaves; ++k)
    if (some_at[k] >= 0) chosen = 64 * k + some_at[k];
#pragma unroll
  for (int k = kWaves - 1; k >= 0; --k)
    if (passes_at[k] >= 0) chosen = 64 * k + passes_at[k];
  if (chosen < 0) {   // (no weight here after all)
    if (threadIdx.x == 0) tokens[a] = otherwise;
  } else if ((int)threadIdx.x == chosen) {
    double sum = upto - mine;
    int last = 0, at = -1;
#pragma unroll
    for (int i = 0; i < kVerifyPerLane; ++i) {
      sum += w[i];
      if (w[i] > 0.0) {
        last = i;
        if (at < 0 && sum > target_at) at = i;
      }
    }
    tokens[a] = first + (at < 0 ? last : at);
  }
}

}  // namespace arctic

using namespace arctic;

static int64_t verify_parts(int vocab_size) { return ((int64_t)vocab_size + kVerifySegment - 1) / kVerifySegment; }

extern "C" int64_t arctic_verify_drafts_workspace_bytes(int64_t batch, int max_drafts, int vocab_size, int dtype) {
  (void)dtype;
  if (batch <= 0 || batch > 0x7fffffffLL || max_drafts < 0 || max_drafts > 1024 || vocab_size <= 0 || vocab_size > (1 << 30)) return 0;
  const int64_t segments = batch * (max_drafts + 1) * verify_parts(vocab_size);
  return segments > 0x7fffffffLL ? 0 : segments * (int64_t)sizeof(VerifySegment);   // more than a call takes
}

extern "C" int arctic_verify_drafts(int64_t *out_tokens, int64_t *out_counts, const void *logits, const int32_t *row_start,
                                    const int64_t *drafts, const float *accept_uniforms, const float *sample_uniforms,
                                    const float *temperatures, int64_t batch, int max_drafts, int64_t num_rows,
                                    int vocab_size, int64_t row_stride, int64_t draft_stride, int64_t accept_stride, int dtype,
                                    void *workspace, int64_t workspace_bytes, void *stream) {
  const char *fn = "verify_drafts";
  if (dtype != ARCTIC_DTYPE_F32 && dtype != ARCTIC_DTYPE_F16 && dtype != ARCTIC_DTYPE_BF16)
    return fail(ARCTIC_ERR_UNSUPPORTED, "%s: logits must be fp32, fp16 or bf16", fn);
  if (batch < 0 || batch > 0x7ffffffeLL || max_drafts < 0 || max_drafts > 1024 || num_rows < 0 || num_rows > 0x7fffffffLL ||
      vocab_size <= 0 || vocab_size > (1 << 30))
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: batch and num_rows must be in [0, 2^31), max_drafts in [0, 1024] and vocab_size "
                "in [1, 2^30]", fn);
  const int es = dtype == ARCTIC_DTYPE_F32 ? 4 : 2;
  if (!pitch_ok(row_stride, num_rows, es) || !pitch_ok(draft_stride, batch, 8) || !pitch_ok(accept_stride, batch, 4))
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: a row pitch is out of range", fn);
  if (batch == 0) return ARCTIC_OK;
  if (!out_tokens || !out_counts || !row_start || !sample_uniforms || (num_rows > 0 && !logits) ||
      (max_drafts > 0 && (!drafts || !accept_uniforms)))
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", fn);
  if ((uintptr_t)logits % es)
    return fail(ARCTIC_ERR_UNSUPPORTED, "%s: logits do not start at a multiple of their element size", fn);
  const int64_t parts = verify_parts(vocab_size);
  const int64_t grid = batch * (max_drafts + 1) * parts;
  if (grid > 0x3ffffffLL || batch > 0xffffffLL) return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: too many requests for this vocabulary", fn);
  const int64_t need = arctic_verify_drafts_workspace_bytes(batch, max_drafts, vocab_size, dtype);
  if (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < need)
    return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: the workspace must be 8-byte aligned and hold %lld bytes", fn, (long long)need);
  VerifyParams p;
  p.out_tokens = out_tokens;
  p.out_counts = out_counts;
  p.logits = (const char *)logits;
  p.row_start = row_start;
  p.drafts = drafts;
  p.accept = accept_uniforms;
  p.sample = sample_uniforms;
  p.temperatures = temperatures;
  p.segments = (VerifySegment *)workspace;
  p.row_stride_bytes = row_stride * es;
  p.draft_stride = draft_stride;
  p.accept_stride = accept_stride;
  p.num_rows = num_rows;
  p.vocab = vocab_size;
  p.max_drafts = max_drafts;
  p.parts = (int)parts;
  p.places = (uint32_t)(batch * (max_drafts + 1));
  p.by_parts = Divisor((uint32_t)parts);
  p.by_places = Divisor((uint32_t)(max_drafts + 1));
  hipStream_t s = (hipStream_t)stream;
#define ARCTIC_VERIFY(DTYPE)                                                                   \
  do {                                                                                         \
    launch(verify_segments_kernel<DTYPE>, dim3((unsigned)((grid + 3) / 4)), kVerifyLanes, s, p); \
    launch(verify_requests_kernel<DTYPE>, dim3((unsigned)batch), kVerifyLanes, s, p);          \
  } while (0)
  if (dtype == ARCTIC_DTYPE_F32) ARCTIC_VERIFY(ARCTIC_DTYPE_F32);
  else if (dtype == ARCTIC_DTYPE_F16) ARCTIC_VERIFY(ARCTIC_DTYPE_F16);
  else ARCTIC_VERIFY(ARCTIC_DTYPE_BF16);
#undef ARCTIC_VERIFY
  return check_launch(fn);
}
