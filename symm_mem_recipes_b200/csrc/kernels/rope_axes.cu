// Rotary embedding in place, with a position of its own for every token and axis (time, row, column of images and video).
//
// Pair i of a head, (x_i, x_{i + D/2}), turns by pos[axis(i)] * theta^(-2i / D); the frequencies run over the whole head
// and the axis only chooses whose position a pair sees.  Angles are reduced as turns in 64-bit fixed point: frequency
// theta^(-2i / D) / (2 pi) times 2^64, rounded, times the integer position, modulo 2^64, is the angle's fraction of a turn
// to 2^-34 for every 32-bit position, where an fp32 product has lost 0.01 rad at position 200000.  Of it the upper 32 bits are
// used (2^-32 of a turn), turned into an fp32 angle, at most 2^-21.3 off; the sine and cosine intrinsics add 2^-21.1: 2^-20 of
// |x| + |y|, where the result is rounded to 2^-8 of itself.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../device/pdl.cuh"
#include "../device/vec.cuh"
#include "launch.h"
#include "pdl_launch.h"

namespace smr {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;      // of a CTA

__device__ __forceinline__ void unpack8(const Vec16& v, float (&f)[8]) {
  f[0] = bf16lo_to_f32(v.x); f[1] = bf16hi_to_f32(v.x);
  f[2] = bf16lo_to_f32(v.y); f[3] = bf16hi_to_f32(v.y);
  f[4] = bf16lo_to_f32(v.z); f[5] = bf16hi_to_f32(v.z);
  f[6] = bf16lo_to_f32(v.w); f[7] = bf16hi_to_f32(v.w);
}
__device__ __forceinline__ Vec16 pack8(const float (&f)[8]) {
  Vec16 o;
  o.x = pack_bf16x2(f[0], f[1]); o.y = pack_bf16x2(f[2], f[3]);
  o.z = pack_bf16x2(f[4], f[5]); o.w = pack_bf16x2(f[6], f[7]);
  return o;
}

// A CTA takes `per` tokens: first the (cos, sin) of their D / 2 pairs, then the heads, eight pairs a thread and step.  Bound by
// HBM: 8192 tokens of 72 heads of 128 (302 MB read and written) 58.5 us, 79 % of the copy rate; several steps' loads in
// flight at a time were slower (two by 2 %, four by 29 %).  kOnce: the result is more than L2 keeps, its lines are the first to
// leave (61.0 us without).
template <int D, bool kOnce>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ RopeAxesArgs a, int per) {
  constexpr int kPairs = D / 2, kVecs = D / 16;
  __shared__ __align__(16) float cosine[kMaxTokens * kPairs], sine[kMaxTokens * kPairs];
  const long long first = (long long)blockIdx.x * per;
  const int tokens = (int)min((long long)per, a.tokens - first);
  const int pair = threadIdx.x % kPairs;
  const uint64_t frequency = a.frequency[pair];
  const int* pos = a.positions + (size_t)a.axis[pair] * a.position_stride + first;
  pdl_wait();
  pdl_launch_dependents();
  for (int t = threadIdx.x / kPairs; t < tokens; t += kThreads / kPairs) {
    const uint64_t turns = frequency * (uint64_t)(int64_t)pos[t];
    float s, c;
    __sincosf((float)(int32_t)(turns >> 32) * 1.4629180792671596e-09f, &s, &c);      // 2 pi / 2^32
    cosine[t * kPairs + pair] = c;
    sine[t * kPairs + pair] = a.inverse ? -s : s;
  }
  __syncthreads();
  const int vec = threadIdx.x % kVecs, items = tokens * a.n_heads;
  __nv_bfloat16* base = static_cast<__nv_bfloat16*>(a.qkv) + (size_t)first * a.row_stride + vec * 8;
  for (int i = threadIdx.x / kVecs; i < items; i += kThreads / kVecs) {
    const int t = i / a.n_heads, h = i - t * a.n_heads;
    __nv_bfloat16* p = base + (size_t)t * a.row_stride + h * D;
    float x[8], y[8], u[8], v[8];
    unpack8(ld_16_stream(p), x);
    unpack8(ld_16_stream(p + kPairs), y);
    const float* c = cosine + t * kPairs + vec * 8;
    const float* s = sine + t * kPairs + vec * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      u[k] = x[k] * c[k] - y[k] * s[k];
      v[k] = y[k] * c[k] + x[k] * s[k];
    }
    if constexpr (kOnce) {
      st_16_stream(p, pack8(u));
      st_16_stream(p + kPairs, pack8(v));
    } else {
      st_16(p, pack8(u));
      st_16(p + kPairs, pack8(v));
    }
  }
}

}  // namespace

int launch_rope_axes(const RopeAxesArgs& a, cudaStream_t stream) {
  if (a.tokens == 0 || a.n_heads == 0) return 0;
  const int items = a.n_heads * (a.head_dim / 16);      // vectors of a token
  const int per = min(kMaxTokens, max(1, 1024 / items));
  const long long blocks = (a.tokens + per - 1) / per;
  if (blocks > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  const bool once = a.tokens * a.n_heads * a.head_dim * 2 >= (64ll << 20);
  const auto kernel = a.head_dim == 128 ? (once ? rope_axes_kernel<128, true> : rope_axes_kernel<128, false>)
                                        : (once ? rope_axes_kernel<64, true> : rope_axes_kernel<64, false>);
  return launch_pdl(kernel, dim3((unsigned)blocks), kThreads, 0, 1, stream, a, per);
}

}  // namespace smr
