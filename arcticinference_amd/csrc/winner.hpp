// The order in which the token selections rank their candidates, as 64-bit keys, and the wave's winner.
#pragma once

#include "common.hpp"

namespace arctic {

// A candidate as one 64-bit key whose unsigned order is torch's order of winners (GreaterOrNan with the index as tie
// break, aten/src/ATen/native/SharedReduceOps.h): the value's bits mapped monotonically to an unsigned number in the
// upper half (-0 counts as +0, every NaN as the largest number of all), the complement of the index in the lower half
// (among equal values the lowest index is the largest key).  0 = nothing seen: no element maps to upper half 0.
// Merging two candidates is then one 64-bit unsigned maximum instead of a cascade of floating-point cases.
__device__ __forceinline__ uint64_t winner_key(float value, int index) {
  if (index < 0) return 0;
  uint32_t b = __float_as_uint(value);
  if (b == 0x80000000u) b = 0;   // -0 -> +0 (on the bits: no arithmetic that a denormal mode could touch)
  uint32_t o = b ^ ((b & 0x80000000u) ? 0xffffffffu : 0x80000000u);
  if (value != value) o = 0xffffffffu;
  return ((uint64_t)o << 32) | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ int winner_index(uint64_t key) { return key ? (int)~(uint32_t)key : -1; }

// The wave's winner in every lane, in two 32-bit passes: the largest upper half, then the largest lower half among the
// candidates that have it.  A step of a pass is one v_max_u32 with a DPP operand (the 64-bit maximum it stands for
// takes two moves, a compare and two selects): partners at distance 1 and 2 inside a quad, then the mirrored half and
// the mirrored row of 16 lanes, then the row in front and the two rows in front broadcast into the next ones, which
// leaves the wave's maximum in lane 63.  kRows = 1: only lanes 0 ... 15 hold candidates.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRowMask, 0xf, kRowMask == 0xf));
}
template <int kRows>
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max_dpp<0xB1, 0xf>(v);    // quad_perm [1,0,3,2]
  v = max_dpp<0x4E, 0xf>(v);    // quad_perm [2,3,0,1]
  v = max_dpp<0x141, 0xf>(v);   // row_half_mirror
  v = max_dpp<0x140, 0xf>(v);   // row_mirror
  if constexpr (kRows == 1) return (uint32_t)__builtin_amdgcn_readlane((int)v, 0);
  v = max_dpp<0x142, 0xa>(v);   // row_bcast15 into rows 1 and 3
  v = max_dpp<0x143, 0xc>(v);   // row_bcast31 into rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
template <int kRows = 4>
__device__ __forceinline__ uint64_t wave_winner(uint64_t k) {
  const uint32_t value = (uint32_t)(k >> 32);
  const uint32_t top = wave_max<kRows>(value);
  const uint32_t index = wave_max<kRows>(value == top ? (uint32_t)k : 0u);
  return ((uint64_t)top << 32) | index;
}

}  // namespace arctic
