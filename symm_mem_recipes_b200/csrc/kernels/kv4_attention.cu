// One decode step of attention over a 4-bit KV cache (kv4.cuh).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../device/pdl.cuh"
#include "kv4.cuh"
#include "launch.h"

namespace smr {

namespace {

using namespace kv4;

constexpr int kThreads = 256;

template <int D>
__device__ __forceinline__ float key_value(const uint8_t* row, const __nv_bfloat16* scales, int d) {
  const uint8_t byte = row[(d % 32 / 8) * (D / 8) + (d / 32) * 4 + d % 8 / 2];
  return __bfloat162float(scales[d / 32]) * (float)((int)(d & 1 ? byte >> 4 : byte & 15) - 8);
}
template <int D>
__device__ __forceinline__ float value_value(const uint8_t* row, const __nv_bfloat16* scales, int d) {
  const uint8_t byte = row[(d % 32 / 4) * (D / 16) + (d / 32) * 2 + d % 4 / 2];
  return __bfloat162float(scales[d / 32]) * (float)((int)(d & 1 ? byte >> 4 : byte & 15) - 8);
}

__device__ float block_reduce(float v, bool is_max, float* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float y = __shfl_xor_sync(0xffffffffu, v, o);
    v = is_max ? fmaxf(v, y) : v + y;
  }
  __syncthreads();
  if (lane == 0) buf[warp] = v;
  __syncthreads();
  float r = buf[0];
  for (int i = 1; i < kThreads / 32; ++i) r = is_max ? fmaxf(r, buf[i]) : r + buf[i];
  return r;
}

// One CTA a (sequence, kv head): append, scores into the workspace, softmax, weights, output.
template <int D>
__global__ void __launch_bounds__(kThreads) attend_kernel(Kv4AttentionArgs a) {
  pdl_wait();
  __shared__ float q[8][D];
  __shared__ float buf[kThreads / 32];
  __shared__ float norm[8];
  const int head = blockIdx.x, hkv = a.cache.hkv, b = head / hkv, h = head % hkv, g = a.group, tid = threadIdx.x;
  const int len = a.lengths ? a.lengths[b] : a.length;
  const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(a.qkv) + (size_t)b * a.qkv_stride;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + ((size_t)b * hkv + h) * g * D;
  if (len < 0 || len >= a.cache.max_seq) {
    for (int i = tid; i < g * D; i += kThreads) out[i] = __float2bfloat16_rn(0.0f);
    return;
  }
  for (int i = tid; i < g * D; i += kThreads) q[i / D][i % D] = __bfloat162float(row[h * g * D + i]);
  const size_t base = (size_t)head * a.cache.slots;
  __nv_bfloat16* ks = static_cast<__nv_bfloat16*>(a.cache.k_scales) + base * (D / kGroup);
  __nv_bfloat16* vs = static_cast<__nv_bfloat16*>(a.cache.v_scales) + base * (D / kGroup);
  uint8_t* kc = a.cache.k_codes + base * (D / 2);
  uint8_t* vc = a.cache.v_codes + base * (D / 2);
  if (tid < 2 * (D / kGroup)) {
    const bool is_value = tid >= D / kGroup;
    const int grp = tid % (D / kGroup);
    const __nv_bfloat16* src = row + (a.group * hkv + (is_value ? hkv : 0) + h) * D + grp * kGroup;
    float largest = 0.0f;
    bool finite = true;
    for (int i = 0; i < kGroup; ++i) {
      const float x = __bfloat162float(src[i]);
      finite = finite && is_finite(x);
      largest = fmaxf(largest, fabsf(x));
    }
    const Scale s = scale_of(largest, finite);
    (is_value ? vs : ks)[(size_t)len * (D / kGroup) + grp] = s.s;
    for (int i = 0; i < kGroup; i += 2) {
      const uint32_t byte = nibble_of(__bfloat162float(src[i]), s) | nibble_of(__bfloat162float(src[i + 1]), s) << 4;
      if (is_value) vc[(size_t)len * (D / 2) + (i / 4) * (D / 16) + grp * 2 + i % 4 / 2] = (uint8_t)byte;
      else kc[(size_t)len * (D / 2) + (i / 8) * (D / 8) + grp * 4 + i % 8 / 2] = (uint8_t)byte;
    }
  }
  __syncthreads();
  const int n = len + 1;
  float* score = static_cast<float*>(a.workspace) + base * g;
  float top[8];
  for (int j = 0; j < g; ++j) top[j] = -INFINITY;
  for (int i = tid; i < n; i += kThreads) {
    float s[8] = {};
    for (int d = 0; d < D; ++d) {
      const float k = key_value<D>(kc + (size_t)i * (D / 2), ks + (size_t)i * (D / kGroup), d);
      for (int j = 0; j < g; ++j) s[j] += q[j][d] * k;
    }
    for (int j = 0; j < g; ++j) {
      s[j] *= rsqrtf((float)D);
      score[(size_t)i * g + j] = s[j];
      top[j] = fmaxf(top[j], s[j]);
    }
  }
  for (int j = 0; j < g; ++j) {
    const float m = block_reduce(top[j], true, buf);
    float sum = 0.0f;
    for (int i = tid; i < n; i += kThreads) {
      const float p = __expf(score[(size_t)i * g + j] - m);
      score[(size_t)i * g + j] = p;
      sum += p;
    }
    sum = block_reduce(sum, false, buf);
    if (tid == 0) norm[j] = 1.0f / sum;
  }
  __syncthreads();
  if (a.cache.weights != nullptr) {
    float* w = a.cache.weights + base;
    for (int i = tid; i < n; i += kThreads) {
      float sum = 0.0f;
      for (int j = 0; j < g; ++j) sum += score[(size_t)i * g + j] * norm[j];
      w[i] = i == len ? sum : w[i] + sum;
    }
  }
  for (int e = tid; e < g * D; e += kThreads) {
    const int j = e / D, d = e % D;
    float o = 0.0f;
    for (int i = 0; i < n; ++i)
      o += score[(size_t)i * g + j] * value_value<D>(vc + (size_t)i * (D / 2), vs + (size_t)i * (D / kGroup), d);
    out[e] = __float2bfloat16_rn(o * norm[j]);
  }
}

}  // namespace

size_t kv4_attention_workspace_bytes(const Kv4Cache& cache, int batch, int group, int) {
  return (size_t)batch * cache.hkv * cache.slots * group * sizeof(float);
}

int launch_kv4_attention(const Kv4AttentionArgs& a, cudaStream_t stream) {
  if (a.batch == 0) return 0;
  if (a.cache.head_dim == 128) attend_kernel<128><<<a.batch * a.cache.hkv, kThreads, 0, stream>>>(a);
  else attend_kernel<64><<<a.batch * a.cache.hkv, kThreads, 0, stream>>>(a);
  return (int)cudaGetLastError();
}

}  // namespace smr
