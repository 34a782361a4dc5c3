// The 4-bit KV cache: what a row holds, and how bf16 values become codes.
//
// A row (sequence, kv head, slot) is D values in groups of 32 neighbouring dims.  A group has one bf16 scale
// s = bf16(a / 7), a its largest magnitude, and a value is s * c with c in [-7, 7] held as the nibble c + 8: 4.5 bits a
// value.  c is the nearest code, halves go to the smaller magnitude.  A group below 2^-100 is held as zeros; one with an
// infinity or a NaN gets a NaN scale, so that it reads back as NaN instead of as something plausible.
//
// Codes are exact whichever way the quotient is taken: x and s have 8-bit significands, so for |x| / s >= 1/2 the distance
// of |x| / s from a half is 0 or at least 1 / 510 (2 |x| - (2 k + 1) s is a multiple of s's last bit).  x * (1 / s) * (1 - 2^-14)
// is off by 2^-22 of itself besides the factor: below the half for every exact half, on the right side for all else, and
// never a half itself, so one fused multiply-add onto 1.5 * 2^23 + 8 rounds it and leaves the nibble in the low bits.  In the
// same way a / 7 may be a * (1 / 7): 7 times a midpoint of two bf16 numbers is at least 2^-12 of itself away from any a.
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

// Scale of a group and the factor that x is multiplied by before it is rounded; `largest` is the largest magnitude's bits (an
// infinity or a NaN counts as larger than any number).
struct Scale {
  uint16_t bits;
  bool finite;
  float inv;
};
__device__ __forceinline__ Scale scale_of(uint32_t largest) {
  Scale r;
  r.finite = largest < 0x7F80u;
  const float a = __uint_as_float(largest << 16);
  r.bits = __bfloat16_as_ushort(__float2bfloat16_rn(a * 0.14285714285714285f));
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(__uint_as_float((uint32_t)r.bits << 16)));
  r.inv = inv * 0.99993896484375f;                      // 1 - 2^-14
  if (largest < 0x0D80u) r.bits = 0, r.inv = 0.0f;      // 2^-100: held as zeros
  if (!r.finite) r.bits = 0x7FFF;
  return r;
}
// 0x4B400000 + nibble of x under a finite scale.
__device__ __forceinline__ uint32_t rounded(float x, const Scale& s) {
  return __float_as_uint(fmaf(x, s.inv, 12582920.0f));
}
// Largest magnitude, as bits, of a pair of bf16 numbers and another two.
__device__ __forceinline__ uint32_t max_magnitude(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(x & 0x7FFF7FFFu), "r"(y & 0x7FFF7FFFu));
  return r;
}

}  // namespace kv4
}  // namespace smr
