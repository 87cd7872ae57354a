// Helpers shared by the 8-bit translation units (int8_conv.hip, int8_tape.hip).
#pragma once
#include "tde_common.h"

// maximum over the aligned group of L lanes (a power of two <= 64), in every lane: quad swaps and the mirrors of half a
// DPP row and of the row (no LDS), then exchanges across rows.  All L lanes must be active.
template <int L>
__device__ __forceinline__ unsigned group_umax(unsigned v) {
  if (L >= 2) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));   // lane ^ 1
  if (L >= 4) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));   // lane ^ 2
  if (L >= 8) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));  // 7 - lane
  if (L >= 16) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true)); // 15 - lane
  if (L >= 32) v = max(v, (unsigned)__shfl_xor((int)v, 16, 64));
  if (L >= 64) v = max(v, (unsigned)__shfl_xor((int)v, 32, 64));
  return v;
}

__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// byte j of p := the whole number v in [0, 255]
template <int J>
__device__ __forceinline__ unsigned put_byte(float v, unsigned p) { return __builtin_amdgcn_cvt_pk_u8_f32(v, J, p); }
