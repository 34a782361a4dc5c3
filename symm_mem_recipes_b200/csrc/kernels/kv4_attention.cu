// One decode step of attention over a 4-bit KV cache (kv4.cuh): append the new token, softmax(q K^T / sqrt(D)) V over
// sequences of their own lengths, attention weights accumulated.
//
// The work is the caches' bytes.  Tiles of 64 slots of all heads and sequences form one list, cut evenly among the grid's
// warps whatever the lengths are; a warp streams its tiles through a ring in shared memory by asynchronous copies and
// nothing synchronises warps until the end.  A head whose tiles are all one CTA's is finished there, the others leave a piece
// (maximum, sum, weighted values) a CTA, which a second kernel joins in the CTAs' order: results do not depend on timing.
//
// Codes are multiplied as they are.  A nibble in the low bits of a 16-bit float is the subnormal n * 2^-133 (bf16), one in
// the next four bits sixteen times that, and the tensor cores take subnormals exactly and at full rate (as many cycles an
// MMA as for normal numbers): one AND makes two operands, where a conversion would take three instructions.  Of
// n = c + 8 the eight is taken out of the sums: in S by an accumulator that starts at -8 sum(q), in the values by one
// more MMA a group whose operand is eight everywhere.  The cores align addends by their nominal exponents, a subnormal's being 2^-14 (fp16)
// however small it is: in the lowest bits a nibble would lose ten bits of the sum's 24.  fp16 nibbles therefore stand two bits
// higher, where the lower one loses six at most, the upper two, and what is cut off the sums of eights in the same places
// takes the bias out.
//
//   S^T [16 keys x 8 heads] = K q^T, bf16: q is exact, scaled by a power of two per head so that its largest element is
//   near 2^120; a group's 32 dims are two MMAs, whose sum the key's scale multiplies in fp32.  No operand is rounded.
//   O^T [16 dims x 8 heads] += V^T P'^T, fp16: P' = 2^(S - M) * scale, where the values' scale of the key and group goes
//   into the probability.  M is at least (largest S of a tile) + (exponent of its largest scale) - 15, so P' stays below
//   2^15 and is rounded to 11 bits (2^-11 of itself) down to 2^-29 of the largest; the output is rounded to 8 bits.
// S^T's accumulators hold heads in rows of four lanes, the second MMA wants keys there: movmatrix transposes in registers.
//
// Measured: 1.67 us per 1000 tiles at D = 128 (5.5 TB/s, 84 % of the copy rate) and 18 us besides; 32 x 8 heads of 6600 to 16384 slots
// (46592 tiles) 96 us in bursts and 103 in a long loop, where the 1000 W cap lowers the clock; 8 heads of 131072 with weights 53.
// Reading alone takes 72, computing alone 80: neither memory nor one pipe is full (issue 52 %, ALU 51 %, tensor 32 %).  Three CTAs
// an SM, bulk copies and one stage less are no faster.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "../device/pdl.cuh"
#include "kv4.cuh"
#include "kv4_shares.h"
#include "launch.h"
#include "pdl_launch.h"

namespace smr {

namespace {

using namespace kv4;

constexpr int kHeads = 8;                 // query heads a kv head at most, the MMA's N
constexpr int kRing = 27648;              // bytes of a warp's ring: two CTAs an SM
constexpr int kJoinThreads = 256;
constexpr int kJoinTiles = 4;             // tiles whose weights a CTA of the second kernel accumulates at a time: a slot a thread
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct Layout {
  static constexpr int kGroups = D / kGroup;
  static constexpr int kCodes = kTile * D / 2;              // bytes of a tile's codes of keys
  static constexpr int kScales = kTile * kGroups * 2;       // and of their scales
  static constexpr int kBytes = 2 * (kCodes + kScales);
  static constexpr int kStages = kRing / kBytes;
  static constexpr int kPiece = kHeads * (D + 2);           // floats: maxima, sums, weighted values [head][D]
};

// The calls' scratch: pieces of the warps, (M, l) of the heads that one warp finished, scores of all tiles.
struct Workspace {
  float* pieces;      // [warps][2][kPiece]: a warp's first head and its last one, where they are shared with others
  float2* stats;      // [batch * hkv][kHeads]
  int* start;         // [batch + 1]: first tile of a sequence
  float* scores;      // [tiles][kTile][padded group], units of log2
};
__host__ __device__ inline int padded_group(int group) { return (group + 1) & ~1; }
__host__ __device__ inline int padded_starts(int batch) { return (batch + 2) & ~1; }
__host__ __device__ inline Workspace carve(void* base, int head_dim, int batch, int hkv, int warps) {
  Workspace w;
  w.pieces = static_cast<float*>(base);
  w.stats = reinterpret_cast<float2*>(w.pieces + (size_t)warps * 2 * kHeads * (head_dim + 2));
  w.start = reinterpret_cast<int*>(w.stats + (size_t)batch * hkv * kHeads);
  w.scores = reinterpret_cast<float*>(w.start + padded_starts(batch));
  return w;
}

__device__ __forceinline__ int length_of(const Kv4AttentionArgs& a, int b) { return a.lengths ? a.lengths[b] : a.length; }
// Tiles of a head of sequence b, the new token's included; none for an idle sequence.
__device__ __forceinline__ int tiles_of(const Kv4AttentionArgs& a, int b) {
  const int n = length_of(a, b);
  return n >= 0 && n < a.cache.max_seq ? n / kTile + 1 : 0;
}
// kOnce: the lines are the first to leave L2, where others are wanted again.
template <bool kOnce>
__device__ __forceinline__ void copy_async_16(uint32_t dst, const void* src, uint64_t policy) {
  if constexpr (kOnce)
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
  else
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with an accumulator that starts at (c0, c1) in both rows and is left as it is.
__device__ __forceinline__ void mma_bf16_from(float (&d)[4], float c0, float c1, uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mma_fp16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lo_of(uint32_t bf16x2) { return __uint_as_float(bf16x2 << 16); }
__device__ __forceinline__ float hi_of(uint32_t bf16x2) { return __uint_as_float(bf16x2 & 0xFFFF0000u); }

// Where a warp is in the list of tiles.
struct Cursor {
  int b, h, t, n;      // sequence, kv head, tile of it, tiles of the head
};

// Row of a tile that stands in row `rho` of the MMAs' 16 keys: neighbours keep opposite parity, and so do rows 0, 2, 4, 6, for
// shared memory's banks (64 bytes a row at D = 128).
__device__ __forceinline__ int row_of(int rho) { return rho ^ ((rho >> 1) & 1); }

template <int D, bool kScores>
struct Attend {
  using L = Layout<D>;
  static constexpr int kG = L::kGroups;

  // Lane (r = lane / 4, c = lane % 4).  q: operand B, head r, dims 32 g + 8 c + .. in the codes' order: of a word's nibbles
  // j and j + 4 make a pair; [g][half][b0 / b1].
  uint32_t q[kG][2][2];
  float minus8[kG][2];      // accumulators' start for heads 2c, 2c + 1
  float to_log2[2];         // S in the accumulators' units -> units of log2
  float m[2], l[2];         // M, and this lane's rows' share of the sum, of heads 2c and 2c + 1
  float acc[kG][2][4];      // [g][t]: dims 32 g + 4 r + 2 t (first two, 2^-22 n P') and the next one (last two, 2^-18 n P')
  float sum[kG][4];         // sum of 8 P', in the units of the two halves of acc

  __device__ __forceinline__ void start(const Kv4AttentionArgs& a, int b, int h) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(a.qkv) + (size_t)b * a.qkv_stride +
                               ((size_t)h * a.group + r) * D + 8 * c;
    Vec16 raw[kG];
#pragma unroll
    for (int g = 0; g < kG; ++g) raw[g] = r < a.group ? ld_16_stream(row + kGroup * g) : Vec16{0, 0, 0, 0};
    float largest = 0.0f;
#pragma unroll
    for (int g = 0; g < kG; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = i == 0 ? raw[g].x : i == 1 ? raw[g].y : i == 2 ? raw[g].z : raw[g].w;
        largest = fmaxf(largest, fmaxf(fabsf(lo_of(w)), fabsf(hi_of(w))));
      }
    }
    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    // 2^(120 - e): the largest element comes to [2^120, 2^121); e is held in [-6, 127], where the factor is a normal number
    const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127, -6), 127);
    const float up = __uint_as_float((uint32_t)(120 - e + 127) << 23);
    // S = 2^-133 n 2^(120 - e) q: back by 2^(13 + e), then log2(e) / sqrt(D); an infinity from e = 118 on, the head's outputs NaN
    const float back = ldexpf(kLog2e * rsqrtf((float)D), 13 + e);
#pragma unroll
    for (int j = 0; j < 2; ++j) to_log2[j] = __shfl_sync(0xffffffffu, back, 4 * (2 * c + j));
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      const uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
      float f[8], sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = lo_of(w[i]) * up;
        f[2 * i + 1] = hi_of(w[i]) * up;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += f[i];
      // nibbles 0, 4 | 1, 5 (times 16) of the word, then 2, 6 | 3, 7; a multiplication by a power of two rounds nothing
      q[g][0][0] = pack_bf16x2(f[0], f[4]);
      q[g][0][1] = pack_bf16x2(f[1] * 0.0625f, f[5] * 0.0625f);
      q[g][1][0] = pack_bf16x2(f[2], f[6]);
      q[g][1][1] = pack_bf16x2(f[3] * 0.0625f, f[7] * 0.0625f);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= -0.0625f;                               // -8 * 2^-133 as -2^-4 and 2^-126
      sum *= 1.1754943508222875e-38f;
#pragma unroll
      for (int j = 0; j < 2; ++j) minus8[g][j] = __shfl_sync(0xffffffffu, sum, 4 * (2 * c + j));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[j] = -INFINITY;
      l[j] = 0.0f;
    }
#pragma unroll
    for (int g = 0; g < kG; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[g][0][i] = acc[g][1][i] = sum[g][i] = 0.0f;
    }
  }

  // One tile in shared memory; the first `valid` slots are seen.  `scores`: where the tile's scores go.
  __device__ __forceinline__ void tile(const uint8_t* stage, int valid, float* scores, int group, int pitch) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const uint8_t* kc = stage;
    const uint8_t* vc = stage + L::kCodes;
    const uint8_t* ks = stage + 2 * L::kCodes;
    const uint8_t* vs = ks + L::kScales;
    float s[4][4];
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
      uint32_t w[2][kG], sc[2][kG / 2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = sub * 16 + row_of(r) + 8 * j;
        const uint8_t* p = kc + row * (D / 2) + c * (D / 8);
        const uint8_t* ps = ks + row * (2 * kG);
        if constexpr (D == 128) {
          const uint4 x = *reinterpret_cast<const uint4*>(p);
          w[j][0] = x.x; w[j][1] = x.y; w[j][2] = x.z; w[j][3] = x.w;
          const uint2 y = *reinterpret_cast<const uint2*>(ps);
          sc[j][0] = y.x; sc[j][1] = y.y;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(p);
          w[j][0] = x.x; w[j][1] = x.y;
          sc[j][0] = *reinterpret_cast<const uint32_t*>(ps);
        }
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        float d[4];
        const uint32_t x = w[0][g], y = w[1][g];
        mma_bf16_from(d, minus8[g][0], minus8[g][1], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u,
                      q[g][0][0], q[g][0][1]);
        mma_bf16(d, x >> 8 & 0x000F000Fu, y >> 8 & 0x000F000Fu, x >> 8 & 0x00F000F0u, y >> 8 & 0x00F000F0u, q[g][1][0],
                 q[g][1][1]);
        const float sx = g & 1 ? hi_of(sc[0][g / 2]) : lo_of(sc[0][g / 2]);
        const float sy = g & 1 ? hi_of(sc[1][g / 2]) : lo_of(sc[1][g / 2]);
        s[sub][0] = g == 0 ? d[0] * sx : fmaf(d[0], sx, s[sub][0]);
        s[sub][1] = g == 0 ? d[1] * sx : fmaf(d[1], sx, s[sub][1]);
        s[sub][2] = g == 0 ? d[2] * sy : fmaf(d[2], sy, s[sub][2]);
        s[sub][3] = g == 0 ? d[3] * sy : fmaf(d[3], sy, s[sub][3]);
      }
      if constexpr (kScores) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = sub * 16 + row_of(r) + 8 * j;
          if (2 * c < group && row < valid)
            *reinterpret_cast<float2*>(scores + row * pitch + 2 * c) =
                make_float2(s[sub][2 * j] * to_log2[0], s[sub][2 * j + 1] * to_log2[1]);
        }
      }
    }
    // scales of the values of this lane's rows; a row that is not seen has a score of minus infinity and scales of zero
    uint32_t sv[4][2][kG / 2];
    __nv_bfloat162 top2 = __float2bfloat162_rn(0.0f);
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = sub * 16 + row_of(r) + 8 * j;
        const uint8_t* ps = vs + row * (2 * kG);
        if constexpr (D == 128) {
          const uint2 y = *reinterpret_cast<const uint2*>(ps);
          sv[sub][j][0] = y.x; sv[sub][j][1] = y.y;
        } else {
          sv[sub][j][0] = *reinterpret_cast<const uint32_t*>(ps);
        }
      }
    }
    if (valid < kTile) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i / 2 * 16 + row_of(r) + 8 * (i & 1) >= valid) {
#pragma unroll
          for (int k = 0; k < kG / 2; ++k) sv[i / 2][i & 1][k] = 0;
          s[i / 2][2 * (i & 1)] = s[i / 2][2 * (i & 1) + 1] = -INFINITY;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int k = 0; k < kG / 2; ++k)      // of a NaN and a number this is the number
        top2 = __hmax2(top2, *reinterpret_cast<const __nv_bfloat162*>(&sv[i / 2][i & 1][k]));
    }
    float top = fmaxf(__low2float(top2), __high2float(top2));
    float high[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      high[j] = fmaxf(fmaxf(fmaxf(s[0][j], s[0][j + 2]), fmaxf(s[1][j], s[1][j + 2])),
                      fmaxf(fmaxf(s[2][j], s[2][j + 2]), fmaxf(s[3][j], s[3][j + 2])));
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      high[0] = fmaxf(high[0], __shfl_xor_sync(0xffffffffu, high[0], o));
      high[1] = fmaxf(high[1], __shfl_xor_sync(0xffffffffu, high[1], o));
    }
    // 2^(e - 126) is above the largest scale; below 2^-60 it does not matter
    const float exponent = (float)(max((int)(__float_as_uint(top) >> 23), 66) - 126 - 15);
    const float m0 = fmaxf(m[0], fmaf(high[0], to_log2[0], exponent)), m1 = fmaxf(m[1], fmaf(high[1], to_log2[1], exponent));
    if (__any_sync(0xffffffffu, m0 != m[0] || m1 != m[1])) {
      const float f0 = exp2_of(m[0] - m0), f1 = exp2_of(m[1] - m1);
      m[0] = m0;
      m[1] = m1;
      l[0] *= f0;
      l[1] *= f1;
#pragma unroll
      for (int g = 0; g < kG; ++g) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[g][0][i] *= i & 1 ? f1 : f0;
          acc[g][1][i] *= i & 1 ? f1 : f0;
          sum[g][i] *= i & 1 ? f1 : f0;
        }
      }
    }
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[sub][i] = exp2_of(fmaf(s[sub][i], to_log2[i & 1], -m[i & 1]));
        l[i & 1] += s[sub][i];
      }
    }
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
      uint32_t x[4][kG / 2];      // this lane's part of the values of MMA rows 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint8_t* p = vc + (sub * 16 + row_of(2 * c + (k & 1)) + 8 * (k >> 1)) * (D / 2) + r * (D / 16);
        if constexpr (D == 128) {
          const uint2 y = *reinterpret_cast<const uint2*>(p);
          x[k][0] = y.x; x[k][1] = y.y;
        } else {
          x[k][0] = *reinterpret_cast<const uint32_t*>(p);
        }
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        const float sx = g & 1 ? hi_of(sv[sub][0][g / 2]) : lo_of(sv[sub][0][g / 2]);
        const float sy = g & 1 ? hi_of(sv[sub][1][g / 2]) : lo_of(sv[sub][1][g / 2]);
        const uint32_t b0 = transpose_8x8(half2_of(s[sub][0] * sx, s[sub][1] * sx));
        const uint32_t b1 = transpose_8x8(half2_of(s[sub][2] * sy, s[sub][3] * sy));
        const uint32_t y0 = __byte_perm(x[0][g / 2], x[1][g / 2], g & 1 ? 0x7632 : 0x5410);
        const uint32_t y1 = __byte_perm(x[2][g / 2], x[3][g / 2], g & 1 ? 0x7632 : 0x5410);
        mma_fp16(acc[g][0], y0 << 2 & 0x003C003Cu, y0 << 2 & 0x03C003C0u, y1 << 2 & 0x003C003Cu, y1 << 2 & 0x03C003C0u, b0, b1);
        mma_fp16(acc[g][1], y0 >> 6 & 0x003C003Cu, y0 >> 6 & 0x03C003C0u, y1 >> 6 & 0x003C003Cu, y1 >> 6 & 0x03C003C0u, b0, b1);
        mma_fp16(sum[g], 0x00200020u, 0x02000200u, 0x00200020u, 0x02000200u, b0, b1);
      }
    }
  }

  // Weighted values of head 2c + j: dims 32 g + 4 r .. + 3.
  __device__ __forceinline__ float4 values(int g, int j) const {
    constexpr float kEven = 4194304.0f, kOdd = 262144.0f;      // 2^22, 2^18
    const float even = sum[g][j], odd = sum[g][2 + j];
    return make_float4((acc[g][0][j] - even) * kEven, (acc[g][0][2 + j] - odd) * kOdd, (acc[g][1][j] - even) * kEven,
                       (acc[g][1][2 + j] - odd) * kOdd);
  }
  // The piece: maxima, sums (after join_lanes), weighted values.
  __device__ __forceinline__ void leave(float* piece, int group) const {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int head = 2 * c + j;
      if (head >= group) continue;
      if (r == 0) {
        piece[head] = m[j];
        piece[kHeads + head] = l[j];
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) *reinterpret_cast<float4*>(piece + 2 * kHeads + head * D + kGroup * g + 4 * r) = values(g, j);
    }
  }
  __device__ __forceinline__ void join_lanes() {
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
    }
  }
};

// The new token's row, four dims a lane: into the tile in shared memory and into the cache.
template <int D>
__device__ __forceinline__ void append_row(const Kv4AttentionArgs& a, int b, int h, int slot, uint8_t* stage) {
  using L = Layout<D>;
  const int lane = threadIdx.x & 31, g = lane >> 3, hkv = a.cache.hkv;
  const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(a.qkv) + (size_t)b * a.qkv_stride + (size_t)a.group * hkv * D;
  const size_t at = ((size_t)b * hkv + h) * a.cache.slots + slot;
  const int in_tile = slot % kTile;
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    uint2 raw = make_uint2(0, 0);
    if (lane < D / 4) raw = *reinterpret_cast<const uint2*>(row + ((size_t)kind * hkv + h) * D + 4 * lane);
    uint32_t largest = max_magnitude(raw.x, raw.y);
    largest = max(largest & 0xFFFFu, largest >> 16);
#pragma unroll
    for (int o = 1; o <= 4; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    const Scale s = scale_of(largest);
    uint32_t half = 0x4B400000u * 0xFFFFEEEFu;      // less 0x4B400000 in four nibbles' places
    half += rounded(lo_of(raw.x), s) + (rounded(hi_of(raw.x), s) << 4) + (rounded(lo_of(raw.y), s) << 8) + (rounded(hi_of(raw.y), s) << 12);
    if (!s.finite) half = 0x8888u;
    if (lane < D / 4) {
      const int byte = kind == 0 ? (lane & 7) / 2 * (D / 8) + g * 4 + (lane & 1) * 2 : (lane & 7) * (D / 16) + g * 2;
      uint8_t* codes = kind == 0 ? a.cache.k_codes : a.cache.v_codes;
      *reinterpret_cast<uint16_t*>(codes + at * (D / 2) + byte) = (uint16_t)half;
      *reinterpret_cast<uint16_t*>(stage + kind * L::kCodes + in_tile * (D / 2) + byte) = (uint16_t)half;
      if ((lane & 7) == 0) {
        static_cast<uint16_t*>(kind == 0 ? a.cache.k_scales : a.cache.v_scales)[at * L::kGroups + g] = s.bits;
        reinterpret_cast<uint16_t*>(stage + 2 * L::kCodes + kind * L::kScales)[in_tile * L::kGroups + g] = s.bits;
      }
    }
  }
}

// Joins `n` pieces of one head into (m, l, four dims); `get(i, what)`: what = 0 the maximum, 1 the sum, and get4(i) the dims.  A
// piece that saw no tile has a maximum of minus infinity and zeros; one whose scores were all NaN has the same maximum and
// a sum of NaN, which stays one.
template <int N, class Get, class Get4>
__device__ __forceinline__ void join_pieces(int n, Get get, Get4 get4, float& m, float& l, float4& o) {
  float mi[N], li[N];
  float4 oi[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mi[i] = i < n ? get(i, 0) : -INFINITY;
    li[i] = i < n ? get(i, 1) : 0.0f;
    oi[i] = i < n ? get4(i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  m = mi[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, mi[i]);
  l = 0.0f;
  o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float f = mi[i] == -INFINITY ? 0.0f : exp2_of(mi[i] - m);
    l += f * li[i];
    o.x += f * oi[i].x; o.y += f * oi[i].y; o.z += f * oi[i].z; o.w += f * oi[i].w;
  }
}

// A warp's copy of the tile that starts at row `slot` (of all heads) into a stage of its ring.  Where scores are kept for the second
// kernel the cache's lines make room for them in L2 (kOnce).
template <int D, bool kOnce>
__device__ __forceinline__ void fetch_tile(const Kv4Cache& cache, size_t slot, uint32_t stage) {
  using L = Layout<D>;
  const int lane = threadIdx.x & 31;
  uint64_t policy = 0;
  if constexpr (kOnce) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  const uint32_t dst = stage + lane * 16;
  const uint8_t* kc = cache.k_codes + slot * (D / 2) + lane * 16;
  const uint8_t* vc = cache.v_codes + slot * (D / 2) + lane * 16;
#pragma unroll
  for (int i = 0; i < L::kCodes / 512; ++i) {
    copy_async_16<kOnce>(dst + i * 512, kc + i * 512, policy);
    copy_async_16<kOnce>(dst + L::kCodes + i * 512, vc + i * 512, policy);
  }
  const uint8_t* ks = static_cast<const uint8_t*>(cache.k_scales) + slot * (2 * L::kGroups);
  const uint8_t* vs = static_cast<const uint8_t*>(cache.v_scales) + slot * (2 * L::kGroups);
  if constexpr (D == 128) {
    copy_async_16<kOnce>(dst + 2 * L::kCodes, ks + lane * 16, policy);
    copy_async_16<kOnce>(dst + 2 * L::kCodes + L::kScales, vs + lane * 16, policy);
  } else {      // 256 bytes of either, half a warp each
    copy_async_16<kOnce>(dst + 2 * L::kCodes, lane < 16 ? ks + lane * 16 : vs + (lane - 16) * 16, policy);
  }
}

template <int D, bool kScores>
__global__ void __launch_bounds__(32 * kWarps, 2) attend_kernel(const __grid_constant__ Kv4AttentionArgs a) {
  using L = Layout<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ FinalPiece final_of[kWarps];
  int* start = reinterpret_cast<int*>(smem + kWarps * kRing);      // [batch + 1]: first tile of a sequence
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hkv = a.cache.hkv;
  if (lane == 0) final_of[warp] = FinalPiece{kNoTiles, false, false, 0};
  pdl_wait();
  pdl_launch_dependents();
  // Every warp finds its first tile by itself, so that the copies start without a barrier; the first one leaves the sequences' first
  // tiles for later.
  const int per = (a.batch + 31) / 32, b0 = lane * per;
  int mine = 0;
  for (int i = 0; i < per; ++i) mine += b0 + i < a.batch ? tiles_of(a, b0 + i) * hkv : 0;
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += y;
  }
  const int tiles = __shfl_sync(0xffffffffu, before, 31);
  before -= mine;
  const int warps = gridDim.x * kWarps, w = blockIdx.x * kWarps + warp;
  const Workspace ws = carve(a.workspace, D, a.batch, hkv, warps);
  if (tiles == 0) {      // every CTA
    for (int i = threadIdx.x; blockIdx.x == 0 && i <= a.batch; i += 32 * kWarps) ws.start[i] = 0;
    return;
  }
  const Shares shares(tiles, warps);
  const int first = shares.first(w), end = shares.first(w + 1);
  Cursor now{0, 0, 0, 1};
  if (first < end) {
    int left = first - before;      // of the sequence that `first` is in, in the lane that has it
    const bool has = left >= 0 && left < mine;
    if (has) {
      now.b = b0;
      while (left >= (now.n = tiles_of(a, now.b)) * hkv) {
        left -= now.n * hkv;
        ++now.b;
      }
      now.h = left / now.n;
      now.t = left - now.h * now.n;
    }
    const int from = __ffs(__ballot_sync(0xffffffffu, has)) - 1;
    now.b = __shfl_sync(0xffffffffu, now.b, from);
    now.h = __shfl_sync(0xffffffffu, now.h, from);
    now.t = __shfl_sync(0xffffffffu, now.t, from);
    now.n = __shfl_sync(0xffffffffu, now.n, from);
  }
  uint8_t* ring = smem + warp * kRing;
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
  auto fetch = [&](const Cursor& at, int stage) {
    fetch_tile<D, kScores>(a.cache, ((size_t)at.b * hkv + at.h) * a.cache.slots + (size_t)at.t * kTile, ring_addr + stage * L::kBytes);
  };
  int to_fetch = first;
  if (to_fetch < end) {
    fetch(now, 0);
    ++to_fetch;
    if (lane == 0) final_of[warp].head = kNoPiece;
  }
  copy_commit();
  if (warp == 0) {
    for (int i = 0; i < per && b0 + i < a.batch; ++i) {
      start[b0 + i] = before;
      if (blockIdx.x == 0) ws.start[b0 + i] = before;      // for the second kernel
      before += tiles_of(a, b0 + i) * hkv;
    }
    if (lane == 31) {
      start[a.batch] = tiles;
      if (blockIdx.x == 0) ws.start[a.batch] = tiles;
    }
  }
  __syncthreads();
  auto advance = [&](Cursor& at) {
    if (++at.t < at.n) return;
    at.t = 0;
    if (++at.h < hkv) return;
    at.h = 0;
    do {
      ++at.b;
    } while (at.b < a.batch && start[at.b + 1] == start[at.b]);
    if (at.b < a.batch) at.n = (start[at.b + 1] - start[at.b]) / hkv;
  };
  Cursor ahead = now;
#pragma unroll
  for (int i = 1; i < L::kStages - 1; ++i) {
    if (to_fetch < end) {
      advance(ahead);
      fetch(ahead, i);
      ++to_fetch;
    }
    copy_commit();
  }

  Attend<D, kScores> at;
  const int pitch = padded_group(a.group);
  bool first_head = true, whole = now.t == 0;      // `whole`: this warp has the head's tiles from the first on
  int stage = 0;
  for (int i = first; i < end; ++i) {
    if (now.t == 0 || i == first) at.start(a, now.b, now.h);
    copy_wait<L::kStages - 2>();
    __syncwarp();      // the tile is there for every lane, and every lane is done with the stage that is filled next
    if (to_fetch < end) {
      advance(ahead);
      fetch(ahead, stage == 0 ? L::kStages - 1 : stage - 1);
      ++to_fetch;
    }
    copy_commit();
    uint8_t* buf = ring + stage * L::kBytes;
    const bool last = now.t == now.n - 1;
    int valid = kTile;
    if (last) {
      const int slot = length_of(a, now.b);
      valid = slot % kTile + 1;
      append_row<D>(a, now.b, now.h, slot, buf);
      __syncwarp();
    }
    at.tile(buf, valid, ws.scores + (size_t)i * kTile * pitch, a.group, pitch);
    stage = stage == L::kStages - 1 ? 0 : stage + 1;
    if (last || i + 1 == end) {
      at.join_lanes();
      const int r = lane >> 2, c = lane & 3, bh = now.b * hkv + now.h;
      if (last && whole) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int head = 2 * c + j;
          if (head >= a.group) continue;
          const float inv = 1.0f / at.l[j];
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + ((size_t)bh * a.group + head) * D + 4 * r;
#pragma unroll
          for (int g = 0; g < L::kGroups; ++g) {
            const float4 v = at.values(g, j);
            *reinterpret_cast<uint2*>(out + kGroup * g) =
                make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
          }
          if (kScores && r == 0) ws.stats[(size_t)bh * kHeads + head] = make_float2(at.m[j], at.l[j]);
        }
      } else if (i + 1 < end) {      // the end of a head that other warps began
        at.leave(ws.pieces + (size_t)w * 2 * L::kPiece, a.group);
      } else {                       // stays in shared memory for the CTA's other warps
        copy_wait<0>();
        __syncwarp();
        at.leave(reinterpret_cast<float*>(ring), a.group);
        if (lane == 0) final_of[warp] = FinalPiece{bh, whole, last, first_head ? 0 : 1};
      }
      first_head = false;
      whole = true;
    }
    advance(now);
  }
  __syncthreads();
  // Neighbouring warps that ended in the same head join their pieces: into the output where that is all of the head, else into
  // the place of the first of them.
  for (int w0 = 0; w0 < kWarps; ++w0) {
    const FinalPiece lead = final_of[w0];
    if (lead.head < 0) continue;
    bool last;
    const int w1 = run_of(final_of, w0, last);
    constexpr int kSide = D / 4, kSides = 32 * kWarps / kSide;      // threads a query head, four dims each
    const int d = threadIdx.x % kSide;
    for (int q = threadIdx.x / kSide; q < a.group; q += kSides) {
      float m, l;
      float4 o;
      auto piece = [&](int k) { return reinterpret_cast<const float*>(smem + (w0 + k) * kRing); };
      auto has = [&](int k) { return w0 + k < w1 && final_of[w0 + k].head == lead.head; };
      join_pieces<kWarps>(
          kWarps, [&](int k, int what) { return has(k) ? piece(k)[what * kHeads + q] : (what == 0 ? -INFINITY : 0.0f); },
          [&](int k) {
            return has(k) ? reinterpret_cast<const float4*>(piece(k))[(2 * kHeads + q * D) / 4 + d] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          },
          m, l, o);
      if (lead.whole && last) {
        const float inv = 1.0f / l;
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + ((size_t)lead.head * a.group + q) * D + 4 * d) =
            make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
        if (kScores && d == 0) ws.stats[(size_t)lead.head * kHeads + q] = make_float2(m, l);
      } else {
        float* to = ws.pieces + ((size_t)(blockIdx.x * kWarps + w0) * 2 + lead.slot) * L::kPiece;
        if (d == 0) {
          to[q] = m;
          to[kHeads + q] = l;
        }
        reinterpret_cast<float4*>(to)[(2 * kHeads + q * D) / 4 + d] = o;
      }
    }
    w0 = w1 - 1;
  }
}

__device__ __forceinline__ void add_piece(float& m, float& l, float mi, float li) {
  const float top = fmaxf(m, mi);
  l = (m == -INFINITY ? 0.0f : exp2_of(m - top)) * l + (mi == -INFINITY ? 0.0f : exp2_of(mi - top)) * li;
  m = top;
}

// blockIdx.x: (sequence, kv head).  blockIdx.y < outputs: joins the pieces of group / outputs query heads, where the head was
// cut.  blockIdx.y >= outputs: accumulates the weights of every `chunks`-th kJoinTiles tiles.
template <int D, bool kScores>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ Kv4AttentionArgs a, int warps, int outputs,
                                                            int chunks) {
  using L = Layout<D>;
  constexpr int kJoinWarps = kJoinThreads / 32, kSide = D / 4, kLanes = 32 / kSide;      // kLanes pieces side by side in a warp
  __shared__ float norms[2][kHeads];
  __shared__ float part[kJoinWarps][2];
  __shared__ float4 parts[kJoinWarps][kSide];
  const int bh = blockIdx.x, hkv = a.cache.hkv, b = bh / hkv, h = bh % hkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const Workspace ws = carve(a.workspace, D, a.batch, hkv, warps);
  // three loads side by side; the lengths too belong to the kernels in front, and are nobody's to read before the wait
  const int n = tiles_of(a, b), first = ws.start[b], all = ws.start[a.batch];
  const int chunk0 = (int)blockIdx.y - outputs;
  if (n == 0) {      // idle: the output row is zero
    if (blockIdx.y == 0)
      for (int i = tid; i < a.group * D / 8; i += kJoinThreads)
        st_16(static_cast<__nv_bfloat16*>(a.out) + (size_t)bh * a.group * D + i * 8, Vec16{0, 0, 0, 0});
    return;
  }
  if (kScores && chunk0 >= 0 && chunk0 * kJoinTiles >= n) return;
  const int s0 = first + h * n;
  const HeadCut cut(Shares(all, warps), s0, s0 + n);
  auto piece = [&](int k) -> const float* { return ws.pieces + (size_t)cut.place(k) * L::kPiece; };

  if (chunk0 < 0) {
    if (cut.finished) return;
    // kJoinWarps / per warps a query head, each every `sides`-th group of pieces; four dims a thread
    const int per = a.group / outputs, sides = kJoinWarps / per, q = blockIdx.y * per + warp / sides, side = warp % sides;
    const int d = lane % kSide;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (warp < per * sides) {
      for (int k = lane; k < cut.count; k += 32) m = fmaxf(m, piece(k)[q]);      // first, so that every piece is scaled once
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
#pragma unroll 4
      for (int k = side * kLanes + lane / kSide; k < cut.count; k += sides * kLanes) {
        const float* p = piece(k);
        const float f = p[q] == -INFINITY ? 0.0f : exp2_of(p[q] - m);
        const float4 v = *reinterpret_cast<const float4*>(p + 2 * kHeads + q * D + 4 * d);
        l += f * p[kHeads + q];
        o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
      }
      if (kLanes == 2) {
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        o.x += __shfl_xor_sync(0xffffffffu, o.x, 16); o.y += __shfl_xor_sync(0xffffffffu, o.y, 16);
        o.z += __shfl_xor_sync(0xffffffffu, o.z, 16); o.w += __shfl_xor_sync(0xffffffffu, o.w, 16);
      }
      if (lane < kSide) parts[warp][d] = o;
      if (lane == 0) part[warp][0] = l;
    }
    __syncthreads();
    if (warp < per * sides && side == 0 && lane < kSide) {
      for (int i = 1; i < sides; ++i) {
        const float4 v = parts[warp + i][d];
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
        l += part[warp + i][0];
      }
      const float inv = 1.0f / l;
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + ((size_t)bh * a.group + q) * D + 4 * d) =
          make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
    }
    return;
  }
  if constexpr (kScores) {
    // the first slots' scores come in while the heads' maxima and sums are found, the next ones while these are worked on
    constexpr int kMine = kJoinTiles * kTile / kJoinThreads;
    const int pitch = padded_group(a.group), len = length_of(a, b);
    const float* scores = ws.scores + (size_t)s0 * kTile * pitch;
    float* weights = a.cache.weights + (size_t)bh * a.cache.slots;
    struct Mine {
      float2 s[kMine][kHeads / 2];
      float weight[kMine];
    };
    auto fetch = [&](int chunk, Mine& x) {
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int i = chunk * kJoinTiles * kTile + k * kJoinThreads + tid;
        if (i > len) continue;
        x.weight[k] = weights[i];
#pragma unroll
        for (int j = 0; j < kHeads / 2; ++j)
          if (2 * j < a.group) x.s[k][j] = *reinterpret_cast<const float2*>(scores + (size_t)i * pitch + 2 * j);
      }
    };
    Mine x;
    fetch(chunk0, x);
    if (warp < a.group) {      // a warp a query head
      float m = -INFINITY, l = 0.0f;
      if (cut.finished) {
        const float2 s = ws.stats[(size_t)bh * kHeads + warp];
        m = s.x;
        l = s.y;
      } else {
        for (int k = lane; k < cut.count; k += 32) add_piece(m, l, piece(k)[warp], piece(k)[kHeads + warp]);
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) {
          const float mi = __shfl_xor_sync(0xffffffffu, m, k), li = __shfl_xor_sync(0xffffffffu, l, k);
          add_piece(m, l, mi, li);
        }
      }
      if (lane == 0) {
        norms[0][warp] = m;
        norms[1][warp] = 1.0f / l;
      }
    }
    __syncthreads();
    float top[kHeads], inv[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {      // a head that is not there adds nothing
      top[j] = j < a.group ? norms[0][j] : 0.0f;
      inv[j] = j < a.group ? norms[1][j] : 0.0f;
    }
    for (int chunk = chunk0; chunk * kJoinTiles < n; chunk += chunks) {
      Mine ahead;
      fetch(chunk + chunks, ahead);
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int i = chunk * kJoinTiles * kTile + k * kJoinThreads + tid;
        if (i > len) continue;
        float p = 0.0f;
#pragma unroll
        for (int j = 0; j < kHeads / 2; ++j) {
          if (2 * j < a.group) p = fmaf(exp2_of(x.s[k][j].x - top[2 * j]), inv[2 * j], p);
          if (2 * j + 1 < a.group) p = fmaf(exp2_of(x.s[k][j].y - top[2 * j + 1]), inv[2 * j + 1], p);
        }
        weights[i] = i == len ? p : x.weight[k] + p;
      }
      x = ahead;
    }
  }
}

// ---- one launch for caches of up to 2048 slots a head and CTA ----
// A cluster of C CTAs takes a head, tile i the warp i % (8 C).  The warps' pieces meet in shared memory, the CTAs' over
// distributed shared memory, and the scores wait in shared memory for their maxima and sums: no scratch, no second kernel.
// 16 heads of 5300 to 8192 slots with weights: 14.3 us, 16.7 as two launches.  A tile takes a warp 1.85 us with another on its
// scheduler.
constexpr int kHeadWarps = 8;
constexpr int kHeadTiles = 4;        // of a warp at most
constexpr int kHeadStages = 2;
constexpr int kHeadCtas = 8;

__device__ __forceinline__ uint32_t remote_of(const void* local, int cta) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(cta));
  return r;
}
__device__ __forceinline__ float load_remote(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 load_remote_4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <int D, bool kScores>
__global__ void __launch_bounds__(32 * kHeadWarps, 1) attend_head_kernel(const __grid_constant__ Kv4AttentionArgs a, int ctas,
                                                                         int tiles_a_warp) {
  using L = Layout<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(16) float cta_piece[L::kPiece];
  __shared__ float norms[2][kHeads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x, hkv = a.cache.hkv;
  const int bh = blockIdx.x / ctas, rank = blockIdx.x % ctas, b = bh / hkv, h = bh % hkv;
  pdl_wait();
  pdl_launch_dependents();
  const int len = length_of(a, b);
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + (size_t)bh * a.group * D;
  if (len < 0 || len >= a.cache.max_seq) {      // idle, for the whole cluster
    for (int i = tid; rank == 0 && i < a.group * D / 8; i += 32 * kHeadWarps) st_16(out + 8 * i, Vec16{0, 0, 0, 0});
    return;
  }
  const int n = len / kTile + 1, step = kHeadWarps * ctas, first = rank * kHeadWarps + warp, pitch = padded_group(a.group);
  const int score_bytes = kScores ? tiles_a_warp * kTile * pitch * (int)sizeof(float) : 0;
  uint8_t* ring = smem + warp * (kHeadStages * L::kBytes + score_bytes);
  float* scores = reinterpret_cast<float*>(ring + kHeadStages * L::kBytes);      // [tile][kTile][pitch]
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
  const size_t base = (size_t)bh * a.cache.slots;
#pragma unroll
  for (int i = 0; i < kHeadStages; ++i) {
    const int t = first + i * step;
    if (t < n) fetch_tile<D, false>(a.cache, base + (size_t)t * kTile, ring_addr + i * L::kBytes);
    copy_commit();
  }
  // the weights so far, of this lane's two slots a tile, come in meanwhile
  float* weights = kScores ? a.cache.weights + base : nullptr;
  float so_far[kScores ? kHeadTiles : 1][kTile / 32];
  if constexpr (kScores) {
#pragma unroll
    for (int i = 0; i < kHeadTiles; ++i) {
#pragma unroll
      for (int k = 0; k < kTile / 32; ++k) {
        const int slot = (first + i * step) * kTile + k * 32 + lane;
        so_far[i][k] = slot < len ? weights[slot] : 0.0f;      // the new token's starts from zero
      }
    }
  }
  Attend<D, kScores> at;
  at.start(a, b, h);
  for (int t = first, i = 0; t < n; t += step, ++i) {
    copy_wait<kHeadStages - 1>();
    __syncwarp();
    uint8_t* stage = ring + (i % kHeadStages) * L::kBytes;
    int valid = kTile;
    if (t == n - 1) {
      valid = len % kTile + 1;
      append_row<D>(a, b, h, len, stage);
      __syncwarp();
    }
    at.tile(stage, valid, scores + i * kTile * pitch, a.group, pitch);
    __syncwarp();
    const int next = t + kHeadStages * step;
    if (next < n) fetch_tile<D, false>(a.cache, base + (size_t)next * kTile, ring_addr + (i % kHeadStages) * L::kBytes);
    copy_commit();
  }
  copy_wait<0>();
  __syncwarp();
  at.join_lanes();
  at.leave(reinterpret_cast<float*>(ring), a.group);      // where the tiles were
  __syncthreads();
  constexpr int kSide = D / 4;                            // threads a query head, four dims each
  const int side = tid / kSide, d = tid % kSide;
  float m, l;
  float4 o;
  if (side < a.group) {
    join_pieces<kHeadWarps>(
        kHeadWarps,
        [&](int i, int what) {
          return reinterpret_cast<const float*>(smem + i * (kHeadStages * L::kBytes + score_bytes))[what * kHeads + side];
        },
        [&](int i) {
          return reinterpret_cast<const float4*>(smem + i * (kHeadStages * L::kBytes + score_bytes))[(2 * kHeads + side * D) / 4 + d];
        },
        m, l, o);
    if (d == 0) {
      cta_piece[side] = m;
      cta_piece[kHeads + side] = l;
    }
    reinterpret_cast<float4*>(cta_piece)[(2 * kHeads + side * D) / 4 + d] = o;
  }
  int q = side;
  bool mine = side < a.group;
  __syncwarp();
  if (ctas > 1) {
    cluster_arrive();
    cluster_wait();
    q = rank + side * ctas;      // query heads are dealt to the CTAs
    mine = q < a.group;
    if (mine)
      join_pieces<kHeadCtas>(
          ctas, [&](int i, int what) { return load_remote(remote_of(cta_piece + what * kHeads + q, i)); },
          [&](int i) { return load_remote_4(remote_of(cta_piece + 2 * kHeads + q * D + 4 * d, i)); }, m, l, o);
  } else {
    __syncthreads();      // cta_piece is read by other threads than it was written by
  }
  if (mine) {
    const float inv = 1.0f / l;
    *reinterpret_cast<uint2*>(out + q * D + 4 * d) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  }
  if constexpr (kScores) {
    if (warp == kHeadWarps - 1 && lane < a.group) {      // a warp that has joined few heads or none
      float4 none;
      if (ctas > 1)
        join_pieces<kHeadCtas>(
            ctas, [&](int i, int what) { return load_remote(remote_of(cta_piece + what * kHeads + lane, i)); },
            [&](int) { return make_float4(0.0f, 0.0f, 0.0f, 0.0f); }, m, l, none);
      else
        m = cta_piece[lane], l = cta_piece[kHeads + lane];
      norms[0][lane] = m;
      norms[1][lane] = 1.0f / l;
    }
  }
  __syncwarp();
  if (ctas > 1) cluster_arrive();      // nothing of another CTA's is read from here on
  if constexpr (kScores) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kHeadTiles; ++i) {
#pragma unroll
      for (int k = 0; k < kTile / 32; ++k) {
        const int slot = (first + i * step) * kTile + k * 32 + lane;
        if (slot > len) continue;
        const float* s = scores + (i * kTile + k * 32 + lane) * pitch;
        float p = 0.0f;
#pragma unroll
        for (int j = 0; j < kHeads; ++j)
          if (j < a.group) p += exp2_of(s[j] - norms[0][j]) * norms[1][j];
        weights[slot] = so_far[i][k] + p;
      }
    }
  }
  __syncwarp();
  if (ctas > 1) cluster_wait();
}

template <int D>
constexpr size_t head_smem(int tiles_a_warp, int score_pitch) {      // pitch 0: no scores
  return kHeadWarps * ((size_t)kHeadStages * Layout<D>::kBytes + (size_t)tiles_a_warp * kTile * score_pitch * sizeof(float));
}

// Clusters of `ctas` of the kernel's largest CTAs that the current device holds at once, asked once per device: SMs are grouped,
// and a group holds whole clusters (148 SMs: 15 of eight, 22 of six, 33 of four).
int resident_clusters(int ctas) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][kHeadCtas + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return 0;
  int n = known[dev][ctas].load(std::memory_order_relaxed);
  if (n > 0) return n - 1;
  const auto kernel = attend_head_kernel<128, true>;
  const size_t smem = head_smem<128>(kHeadTiles, kHeads);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(32 * kHeadWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    clusters = 0;
  }
  known[dev][ctas].store(clusters + 1, std::memory_order_relaxed);
  return clusters;
}

// CTAs a head of the kernel above, or 0 where it does not take the call: as many as there is work and room for at once, and
// slots that they hold; without clusters up to two CTAs an SM one after the other.  Microseconds of one launch and of two, heads x slots
// (0.3 to all of them in use, with weights):
//     1 x 4096     8.1   9.8  |  64 x 2048  11.4  18.3  |  128 x 2048  15.9  25.7  |  256 x 1024  19.3  23.0
//     256 x 2048  31.4  31.0  |  512 x 512  25.1  23.9  |  16 x 8192 with sixteen clusters of eight, which do not fit, 21.0  16.7
int head_ctas(const Kv4Cache& cache, int batch, int num_sms) {
  const long long heads = (long long)batch * cache.hkv;
  const int tiles = cache.slots / kTile;
  int ctas = std::max(1, std::min(kHeadCtas, (tiles + kHeadWarps - 1) / kHeadWarps));
  while (ctas > 1 && heads > resident_clusters(ctas)) --ctas;
  return heads <= (ctas == 1 ? 2 * num_sms : num_sms) && tiles <= ctas * kHeadWarps * kHeadTiles ? ctas : 0;
}

int attention_ctas(const Kv4Cache& cache, int batch, int num_sms) {
  const long long tiles = (long long)batch * cache.hkv * (cache.slots / kTile);
  return (int)std::max<long long>(1, std::min<long long>(2ll * num_sms, (tiles + kWarps - 1) / kWarps));
}

template <int D, bool kScores>
int launch(const Kv4AttentionArgs& a, cudaStream_t stream) {
  const int tiles = a.cache.slots / kTile;
  if (const int ctas = head_ctas(a.cache, a.batch, a.num_sms)) {
    const int a_warp = std::max(1, (tiles + ctas * kHeadWarps - 1) / (ctas * kHeadWarps));
    const size_t smem = head_smem<D>(a_warp, kScores ? padded_group(a.group) : 0);
    return launch_pdl(attend_head_kernel<D, kScores>, dim3((unsigned)(a.batch * a.cache.hkv * ctas)), 32 * kHeadWarps, smem, ctas,
                         stream, a, ctas, a_warp);
  }
  const int ctas = attention_ctas(a.cache, a.batch, a.num_sms);
  const size_t smem = kWarps * kRing + (size_t)(a.batch + 1) * sizeof(int);
  if (int e = launch_pdl(attend_kernel<D, kScores>, dim3(ctas), 32 * kWarps, smem, 1, stream, a)) return e;
  // A CTA a query head where there are few heads, whose pieces are many, else one a kv head; for the weights four CTAs an SM in all.
  // In us, heads x slots, with a slot a thread, two and four (and two CTAs an SM): 8 x 131072 53.0, 54.0, 53.2; 320 x 8192 84.1, 86.7, 87.5;
  // 1024 x 512 36.1, 37.7, 42.8.
  const int heads = a.batch * a.cache.hkv, outputs = heads * a.group <= 8 * a.num_sms ? a.group : 1;
  const int chunks =
      kScores ? std::max(1, std::min((tiles + kJoinTiles - 1) / kJoinTiles, (4 * a.num_sms + heads - 1) / heads)) : 0;
  return launch_pdl(join_kernel<D, kScores>, dim3(heads, outputs + chunks), kJoinThreads, 0, 1, stream, a, ctas * kWarps, outputs,
                    chunks);
}

}  // namespace

size_t kv4_attention_workspace_bytes(const Kv4Cache& cache, int batch, int group, int num_sms) {
  if (head_ctas(cache, batch, num_sms) > 0) return 0;
  const size_t warps = (size_t)attention_ctas(cache, batch, num_sms) * kWarps;
  size_t bytes = warps * 2 * kHeads * (cache.head_dim + 2) * sizeof(float) + (size_t)batch * cache.hkv * kHeads * sizeof(float2) +
                 padded_starts(batch) * sizeof(int);
  if (cache.weights != nullptr) bytes += (size_t)batch * cache.hkv * cache.slots * padded_group(group) * sizeof(float);
  return bytes;
}

int launch_kv4_attention(const Kv4AttentionArgs& a, cudaStream_t stream) {
  if (a.batch == 0) return 0;
  const bool scores = a.cache.weights != nullptr;
  if (a.cache.head_dim == 128) return scores ? launch<128, true>(a, stream) : launch<128, false>(a, stream);
  return scores ? launch<64, true>(a, stream) : launch<64, false>(a, stream);
}

}  // namespace smr
