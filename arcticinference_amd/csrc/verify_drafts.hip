// Verification of drafted tokens against the target model's logits, gfx950.
//
// Two launches.  The first walks every row of logits in segments, one workgroup each: the segment's argmax and, relative
// to its maximum, the sum of its weights exp((x - m) / T) without the drafted token's.  The second, one workgroup per
// request, joins the segments of the request's rows, runs down its drafts to the first that is not accepted, finds the
// segment in which the running sum passes the drawn number and walks that segment alone.
//
// The sums decide whole numbers: with 128256 weights there are as many borders, and an error of 2^-24 in them would move
// one past the drawn number in about one request of a hundred.  They and the weights are therefore held in fp64.  The
// drafted token is left out of the segments' sums and added where it belongs, so that what remains of a row whose draft
// holds nearly everything is no difference of nearly equal numbers.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "winner.hpp"

namespace arctic {

constexpr int kVerifyLanes = 256;
constexpr int kVerifyPerLane = 16;
constexpr int kVerifySegment = kVerifyLanes * kVerifyPerLane;

struct VerifySegment {
  double sum;     // of the weights relative to the segment's maximum, without the draft's
  uint64_t key;   // the segment's argmax
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
  Divisor by_parts, by_places;   // by_places: max_drafts + 1
};

template <int kDtype>
__device__ __forceinline__ float logit(const char *row, int i) {
  if constexpr (kDtype == ARCTIC_DTYPE_F32) return ((const ARCTIC_GLOBAL float *)row)[i];
  const uint32_t bits = ((const ARCTIC_GLOBAL uint16_t *)row)[i];
  return kDtype == ARCTIC_DTYPE_BF16 ? BF16::lo(bits) : F16::lo(bits);
}

// The value that a key was made of (NaN for any NaN, -inf for no key).
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  if (o == 0xffffffffu) return __builtin_nanf("");
  if (o == 0) return -__builtin_inff();
  return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

// exp((x - m) / T); x = -inf has no weight whatever T says.
__device__ __forceinline__ double weight_of(float x, float m, double inv_t) {
  return x == -__builtin_inff() ? 0.0 : exp(((double)x - (double)m) * inv_t);
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// The rows of request b: the first one and the number of drafts, -1 where it has no row.
__device__ __forceinline__ int drafts_of(const VerifyParams &p, int b, int64_t *start) {
  const int64_t first = p.row_start[b], end = min((int64_t)p.row_start[b + 1], p.num_rows);
  *start = first;
  return first < 0 || end <= first ? -1 : (int)min((int64_t)p.max_drafts, end - first - 1);
}

template <int kDtype>
__global__ __launch_bounds__(kVerifyLanes) void verify_segments_kernel(const VerifyParams p) {
  __shared__ uint64_t keys[kVerifyLanes / 64];
  __shared__ double sums[kVerifyLanes / 64];
  const uint32_t place = p.by_parts.quotient(blockIdx.x);   // b * (max_drafts + 1) + k
  const int part = (int)(blockIdx.x - place * (uint32_t)p.parts);
  const int b = (int)p.by_places.quotient(place), k = (int)(place - (uint32_t)b * (uint32_t)(p.max_drafts + 1));
  int64_t start;
  const int n = drafts_of(p, b, &start);
  if (k > n) return;
  const char *row = p.logits + (start + k) * p.row_stride_bytes;
  const float t = p.temperatures ? p.temperatures[b] : 1.f;
  const int64_t draft = k < n ? p.drafts[b * p.draft_stride + k] : -1;
  const int lane = threadIdx.x, first = part * kVerifySegment, end = min(p.vocab, first + kVerifySegment);
  float x[kVerifyPerLane];
  uint64_t key = 0;
#pragma unroll
  for (int i = 0; i < kVerifyPerLane; ++i) {
    const int j = first + i * kVerifyLanes + lane;
    x[i] = -__builtin_inff();
    if (j < end) {
      x[i] = logit<kDtype>(row, j);
      key = max(key, winner_key(x[i], j));
    }
  }
  key = wave_winner(key);
  if ((lane & 63) == 0) keys[lane >> 6] = key;
  __syncthreads();
  key = max(max(keys[0], keys[1]), max(keys[2], keys[3]));
  const float m = key_value(key);
  double sum = 0.0;
  if (t > 0.f && finite(m)) {
    const double inv_t = 1.0 / (double)t;
#pragma unroll
    for (int i = 0; i < kVerifyPerLane; ++i)
      if (first + i * kVerifyLanes + lane != draft) sum += weight_of(x[i], m, inv_t);
  }
  sum = wave_sum64(sum);
  if ((lane & 63) == 0) sums[lane >> 6] = sum;
  __syncthreads();
  if (lane == 0) p.segments[blockIdx.x] = {(sums[0] + sums[1]) + (sums[2] + sums[3]), key};
}

template <int kDtype>
__global__ __launch_bounds__(kVerifyLanes) void verify_requests_kernel(const VerifyParams p) {
  __shared__ int rejected;          // the first row whose draft is not accepted, n at the end
  __shared__ uint64_t found;        // by the first row's wave: its key
  __shared__ double lane_sums[kVerifyLanes];
  __shared__ int segment_at;
  __shared__ double target_at;
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
  const double inv_t = t > 0.f ? 1.0 / (double)t : 0.0;
  const VerifySegment *segments = p.segments + (int64_t)b * (p.max_drafts + 1) * p.parts;
  if (threadIdx.x == 0) rejected = n;
  __syncthreads();
  auto row_key = [&](int k) {
    uint64_t key = 0;
    for (int s = lane; s < p.parts; s += 64) key = max(key, segments[(int64_t)k * p.parts + s].key);
    return wave_winner(key);
  };
  // the weights of a segment, relative to the row's maximum m
  auto segment_sum = [&](int k, int s, float m) {
    const VerifySegment g = segments[(int64_t)k * p.parts + s];
    const float gm = key_value(g.key);
    return gm == -__builtin_inff() ? 0.0 : g.sum * exp(((double)gm - (double)m) * inv_t);
  };
  for (int k = wave; k < n; k += kVerifyLanes / 64) {
    const uint64_t key = row_key(k);
    const float m = key_value(key);
    const int64_t draft = p.drafts[b * p.draft_stride + k];
    bool accepted = false;
    if (finite(m) && draft >= 0 && draft < p.vocab) {
      if (t > 0.f) {
        double sum = 0.0;
        for (int s = lane; s < p.parts; s += 64) sum += segment_sum(k, s, m);
        sum = wave_sum64(sum);
        const double own = weight_of(logit<kDtype>(p.logits + (start + k) * p.row_stride_bytes, (int)draft), m, inv_t);
        accepted = (double)p.accept[b * p.accept_stride + k] * (sum + own) < own;
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
  if (wave == 0) {
    const uint64_t key = row_key(a);
    const float m = key_value(key);
    double total = 0.0;
    if (t > 0.f && finite(m)) {
      for (int s = lane; s < p.parts; s += 64) total += segment_sum(a, s, m);
      total = wave_sum64(total);
    }
    int at = -1;
    double before = 0.0;
    if (total > 0.0) {
      // the first segment whose running sum passes the drawn number, or the last that has any weight
      const double target = (double)p.sample[b] * total;
      for (int s0 = 0; s0 < p.parts; s0 += 64) {
        const double mine = s0 + lane < p.parts ? segment_sum(a, s0 + lane, m) : 0.0;
        double upto = mine;
        for (int d = 1; d < 64; d <<= 1) {
          const double other = __shfl_up(upto, d);
          if (lane >= d) upto += other;
        }
        upto += before;
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
    if (lane == 0) {
      segment_at = at;
      found = key;
    }
  }
  __syncthreads();
  int token = winner_index(found);
  if (segment_at >= 0) {
    // relative to the row's maximum, as the sums before; each lane takes consecutive elements
    const float m = key_value(found);
    const int first = segment_at * kVerifySegment + (int)threadIdx.x * kVerifyPerLane;
    const int end = min(p.vocab, first + kVerifyPerLane);
    double w[kVerifyPerLane], mine = 0.0;
#pragma unroll
    for (int i = 0; i < kVerifyPerLane; ++i) {
      w[i] = first + i < end && first + i != draft ? weight_of(logit<kDtype>(row, first + i), m, inv_t) : 0.0;
      mine += w[i];
    }
    lane_sums[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
      double upto = 0.0;
      int at = 0, last = 0;
      for (; at < kVerifyLanes; ++at) {
        if (lane_sums[at] > 0.0) {
          last = at;
          if (upto + lane_sums[at] > target_at) break;
        }
        if (at + 1 < kVerifyLanes) upto += lane_sums[at];
      }
      if (at == kVerifyLanes) {
        at = last;
        target_at = __builtin_inf();
      } else {
        target_at -= upto;
      }
      segment_at = at;
    }
    __syncthreads();
    if ((int)threadIdx.x == segment_at) {
      double upto = 0.0;
      int last = 0, at = -1;
#pragma unroll
      for (int i = 0; i < kVerifyPerLane; ++i) {
        upto += w[i];
        if (w[i] > 0.0) {
          last = i;
          if (at < 0 && upto > target_at) at = i;
        }
      }
      rejected = first + (at < 0 ? last : at);
    }
    __syncthreads();
    token = rejected;
  }
  for (int k = threadIdx.x; k <= p.max_drafts; k += kVerifyLanes)
    tokens[k] = k < a ? p.drafts[b * p.draft_stride + k] : k == a ? (int64_t)token : -1;
  if (threadIdx.x == 0) p.out_counts[b] = a + 1;
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
  if (grid > 0x7fffffffLL) return fail(ARCTIC_ERR_INVALID_ARGUMENT, "%s: too many requests for this vocabulary", fn);
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
  p.by_parts = Divisor((uint32_t)parts);
  p.by_places = Divisor((uint32_t)(max_drafts + 1));
  hipStream_t s = (hipStream_t)stream;
#define ARCTIC_VERIFY(DTYPE)                                                                   \
  do {                                                                                         \
    launch(verify_segments_kernel<DTYPE>, dim3((unsigned)grid), kVerifyLanes, s, p);           \
    launch(verify_requests_kernel<DTYPE>, dim3((unsigned)batch), kVerifyLanes, s, p);          \
  } while (0)
  if (dtype == ARCTIC_DTYPE_F32) ARCTIC_VERIFY(ARCTIC_DTYPE_F32);
  else if (dtype == ARCTIC_DTYPE_F16) ARCTIC_VERIFY(ARCTIC_DTYPE_F16);
  else ARCTIC_VERIFY(ARCTIC_DTYPE_BF16);
#undef ARCTIC_VERIFY
  return check_launch(fn);
}
