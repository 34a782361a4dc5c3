// The 4-bit KV cache: what a row holds, and how bf16 values become codes.
//
// A row (sequence, kv head, slot) is D values in groups of 32 neighbouring dims.  A group has one bf16 scale
// s = bf16(a / 7), a its largest magnitude, and a value is s * c with c in [-7, 7] held as the nibble c + 8: 4.5 bits a
// value.  c is the nearest code, halves go to the smaller magnitude.  A group below 2^-100 is held as zeros; one with an
// infinity or a NaN gets a NaN scale, so that it reads back as NaN instead of as something plausible.
//
// Codes are exact whichever way the quotient is taken: x and s have 8-bit significands, so for |x| / s >= 1/2 the distance
// of |x| / s from a half is 0 or at least 1 / 510 (2 |x| - (2 k + 1) s is a multiple of s's last bit).  |x| * (1 / s) is off
// by 2^-22 of itself; times (1 - 2^-14) it is below the half for every exact half and on the right side for all else.
//
// Order of the codes in a row.  Keys are an MMA operand whose lane c (of four) holds, group by group, eight neighbouring
// dims of a key; values one whose lane r (of eight) holds four dims a group.  So
//   key   dim d: byte (d % 32 / 8) * (D / 8)  + (d / 32) * 4 + d % 8 / 2
//   value dim d: byte (d % 32 / 4) * (D / 16) + (d / 32) * 2 + d % 4 / 2      low nibble for even d
// and a lane's part is contiguous in both.  Slots of a head are contiguous: a head's stream is one run of memory.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "../device/vec.cuh"
#include "launch.h"

namespace smr {
namespace kv4 {

constexpr int kGroup = 32;
constexpr int kTile = 64;        // a cache has a whole number of tiles of this many slots

// Scale of a group whose largest magnitude is `a`, with the factor that x is multiplied by before it is rounded.
struct Scale {
  __nv_bfloat16 s;
  float inv;
};
__device__ __forceinline__ Scale scale_of(float a, bool finite) {
  Scale r;
  if (!finite) {
    r.s = __ushort_as_bfloat16((unsigned short)0x7FFF);
    r.inv = 0.0f;
  } else if (a < 7.888609052210118e-31f) {      // 2^-100
    r.s = __ushort_as_bfloat16((unsigned short)0);
    r.inv = 0.0f;
  } else {
    r.s = __float2bfloat16_rn(__fdiv_rn(a, 7.0f));
    r.inv = __fmul_rn(__frcp_rn(__bfloat162float(r.s)), 0.99993896484375f);      // 1 - 2^-14
  }
  return r;
}
// Nibble of x under a scale; 8 (the value zero) under a scale of zero or NaN.
__device__ __forceinline__ uint32_t nibble_of(float x, const Scale& s) {
  if (s.inv == 0.0f) return 8;
  const float steps = fminf(rintf(__fmul_rn(fabsf(x), s.inv)), 7.0f);
  return (uint32_t)((int)(x < 0.0f ? -steps : steps) + 8);
}
__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

}  // namespace kv4
}  // namespace smr
