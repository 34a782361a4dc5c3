// Rows into and out of a 4-bit KV cache (kv4.cuh), and the eviction that compacts it.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../device/pdl.cuh"
#include "kv4.cuh"
#include "launch.h"

namespace smr {

namespace {

using namespace kv4;

__device__ __forceinline__ void unpack8(const Vec16& v, float (&f)[8]) {
  f[0] = bf16lo_to_f32(v.x); f[1] = bf16hi_to_f32(v.x);
  f[2] = bf16lo_to_f32(v.y); f[3] = bf16hi_to_f32(v.y);
  f[4] = bf16lo_to_f32(v.z); f[5] = bf16hi_to_f32(v.z);
  f[6] = bf16lo_to_f32(v.w); f[7] = bf16hi_to_f32(v.w);
}

// D / 8 lanes take a row of keys or of values, eight dims a lane; units 2 i and 2 i + 1 are key and value of row i, where
// row i is (sequence, token, head).  Memory-bound: 2 bytes a value in, 0.56 out.
template <int D>
__global__ void __launch_bounds__(256) append_kernel(Kv4AppendArgs a) {
  pdl_wait();
  constexpr int kLanes = D / 8;
  const long long units = 2ll * a.batch * a.tokens * a.cache.hkv;
  const long long unit = ((long long)blockIdx.x * 256 + threadIdx.x) / kLanes;
  const int l = threadIdx.x % kLanes, g = l >> 2, c = l & 3;
  const bool is_value = unit & 1;
  const long long row = unit >> 1;
  const int h = (int)(row % a.cache.hkv);
  const long long bt = row / a.cache.hkv;
  const int t = (int)(bt % a.tokens), b = (int)(bt / a.tokens);
  bool live = unit < units;
  int slot = 0;
  Vec16 raw{0, 0, 0, 0};
  if (live) {
    // `first` may be any number: nothing is added to it before it is known to be a slot
    const int first = a.start_dev ? a.start_dev[b] : a.start;
    live = first >= 0 && first < a.cache.max_seq && t < a.cache.max_seq - first && (a.counts == nullptr || t < a.counts[b]);
    if (live) slot = first + t;
  }
  if (live) {
    const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(is_value ? a.v : a.k) +
                               (is_value ? b * a.v_stride[0] + t * a.v_stride[1] + h * a.v_stride[2]
                                         : b * a.k_stride[0] + t * a.k_stride[1] + h * a.k_stride[2]);
    raw = ld_16_nc(src + l * 8);
  }
  float f[8];
  unpack8(raw, f);
  float largest = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    finite = finite && is_finite(f[i]);
    largest = fmaxf(largest, fabsf(f[i]));
  }
  if (!finite) largest = __uint_as_float(0x7F800000u);
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  const Scale s = scale_of(largest, is_finite(largest));
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) word |= nibble_of(f[i], s) << (4 * i);
  // a value row's part has two bytes a group: two lanes of neighbouring groups trade halves and write four bytes each
  const uint32_t other = __shfl_xor_sync(0xffffffffu, (g & 1) ? word & 0xFFFFu : word >> 16, 4);
  if (!live) return;
  const size_t at = ((size_t)b * a.cache.hkv + h) * a.cache.slots + slot;
  uint8_t* codes = (is_value ? a.cache.v_codes : a.cache.k_codes) + at * (D / 2);
  if (!is_value) {
    *reinterpret_cast<uint32_t*>(codes + c * (D / 8) + g * 4) = word;
  } else {
    const uint32_t pair = (g & 1) ? other | (word & 0xFFFF0000u) : (word & 0xFFFFu) | (other << 16);
    *reinterpret_cast<uint32_t*>(codes + (2 * c + (g & 1)) * (D / 16) + (g >> 1) * 4) = pair;
  }
  if (c == 0)
    static_cast<__nv_bfloat16*>(is_value ? a.cache.v_scales : a.cache.k_scales)[at * (D / kGroup) + g] = s.s;
  if (l == 0 && !is_value && a.cache.weights != nullptr) a.cache.weights[at] = 0.0f;      // of the slot's last tenant
}

template <int D>
__global__ void __launch_bounds__(256) read_kernel(Kv4Cache cache, int batch, int n, void* k_out, void* v_out) {
  pdl_wait();
  constexpr int kLanes = D / 8;
  const long long unit = ((long long)blockIdx.x * 256 + threadIdx.x) / kLanes;
  if (unit >= 2ll * batch * n * cache.hkv) return;
  const int l = threadIdx.x % kLanes, g = l >> 2, c = l & 3;
  const bool is_value = unit & 1;
  const long long row = unit >> 1;
  const int h = (int)(row % cache.hkv);
  const long long bt = row / cache.hkv;
  const int t = (int)(bt % n), b = (int)(bt / n);
  const size_t at = ((size_t)b * cache.hkv + h) * cache.slots + t;
  const uint8_t* codes = (is_value ? cache.v_codes : cache.k_codes) + at * (D / 2);
  uint32_t word;
  if (!is_value) {
    word = *reinterpret_cast<const uint32_t*>(codes + c * (D / 8) + g * 4);
  } else {
    word = *reinterpret_cast<const uint16_t*>(codes + 2 * c * (D / 16) + g * 2) |
           (uint32_t)*reinterpret_cast<const uint16_t*>(codes + (2 * c + 1) * (D / 16) + g * 2) << 16;
  }
  const float s = __bfloat162float(
      static_cast<const __nv_bfloat16*>(is_value ? cache.v_scales : cache.k_scales)[at * (D / kGroup) + g]);
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = s * (float)((int)(word >> (4 * i) & 15u) - 8);
  Vec16 o;
  o.x = pack_bf16x2(f[0], f[1]); o.y = pack_bf16x2(f[2], f[3]);
  o.z = pack_bf16x2(f[4], f[5]); o.w = pack_bf16x2(f[6], f[7]);
  st_16(static_cast<__nv_bfloat16*>(is_value ? v_out : k_out) + row * D + l * 8, o);
}

// ---- eviction ----
// Of a head's n slots the last `recent` stay, and of the others the heaviest, so that `keep` stay in all; equal weights go
// to the lower slot.  The kept rows move down in slot order.  One CTA a head:
//   1. a radix selection over the weights as ordered integers finds the weight of the last one kept, eight bits a pass, and
//      how many slots of exactly that weight stay;
//   2. every thread counts the kept slots of its own run, a scan makes their places, and the places' sources are listed;
//   3. the rows move in chunks of places.  A chunk is read whole before any of it is written; a place is never above its
//      source and sources increase, so a chunk's writes cannot reach the sources of a later one.
constexpr int kEvictThreads = 512;

// Order of a weight as an integer; NaN counts as an infinity; above all weights: the slots that stay anyway.
__device__ __forceinline__ uint32_t worth_of(float w, bool stays) {
  if (stays) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFF800000u;
  if (u == 0x80000000u) return u;                    // -0 and 0 are equal
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ int block_scan_exclusive(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < kEvictThreads / 32; ++i) {
    if (i < warp) before += warp_sums[i];
    all += warp_sums[i];
  }
  *total = all;
  return before + x - v;
}

template <int D>
__global__ void __launch_bounds__(kEvictThreads) evict_kernel(Kv4EvictArgs a) {
  pdl_wait();
  __shared__ int hist[256];
  __shared__ int warp_sums[kEvictThreads / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  const int head = blockIdx.x, tid = threadIdx.x;
  const int b = head / a.cache.hkv;
  const int n = a.lengths[b], keep = a.keep;
  if (n <= keep || n > a.cache.max_seq) return;
  const size_t base = (size_t)head * a.cache.slots;
  float* w = a.cache.weights + base;
  const int protect = n - a.recent;
  uint32_t prefix = 0, mask = 0;
  int left = keep;                                  // slots still to be found among those that match the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kEvictThreads) {
      const uint32_t u = worth_of(w[i], i >= protect);
      if ((u & mask) == prefix) atomicAdd(&hist[u >> shift & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int digit = 255, seen = 0;
      while (seen + hist[digit] < left) seen += hist[digit--];
      s_prefix = prefix | (uint32_t)digit << shift;
      s_left = left - seen;
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    mask |= 255u << shift;
  }
  // `prefix` is the least worth that stays, of which the first `left` slots do
  int* list = a.list + (size_t)head * keep;
  int placed = 0, equal = 0;
  for (int first = 0; first < n; first += kEvictThreads) {
    const int i = first + tid;
    const uint32_t u = i < n ? worth_of(w[i], i >= protect) : 0;
    const bool same = i < n && u == prefix;
    int all_same, all;
    const int rank = equal + block_scan_exclusive(same, warp_sums, &all_same);
    const bool stays = i < n && (u > prefix || (same && rank < left));
    const int place = placed + block_scan_exclusive(stays, warp_sums, &all);
    if (stays) list[place] = i;
    equal += all_same;
    placed += all;
  }
  __syncthreads();
  // a row in parts of 16 bytes (keys, values), then its scales and its weight
  constexpr int kVecs = D / 32, kParts = 2 * kVecs + 1;
  const Vec16* kc = reinterpret_cast<const Vec16*>(a.cache.k_codes + base * (D / 2));
  const Vec16* vc = reinterpret_cast<const Vec16*>(a.cache.v_codes + base * (D / 2));
  Vec16* kc_w = const_cast<Vec16*>(kc);
  Vec16* vc_w = const_cast<Vec16*>(vc);
  uint32_t* ks = static_cast<uint32_t*>(a.cache.k_scales) + base * (D / 64);
  uint32_t* vs = static_cast<uint32_t*>(a.cache.v_scales) + base * (D / 64);
  for (int first = 0; first < keep; first += kEvictThreads / kParts) {
    const int j = first + tid / kParts, part = tid % kParts;
    const bool live = j < keep && tid / kParts < kEvictThreads / kParts;
    Vec16 x{};
    float weight = 0.0f;
    if (live) {
      const size_t src = list[j];
      if (part < kVecs) x = kc[src * kVecs + part];
      else if (part < 2 * kVecs) x = vc[src * kVecs + part - kVecs];
      else {
        x.x = ks[src * (D / 64)];
        x.z = vs[src * (D / 64)];
        if (D == 128) { x.y = ks[src * (D / 64) + D / 128]; x.w = vs[src * (D / 64) + D / 128]; }
        weight = w[src];
      }
    }
    __syncthreads();
    if (live) {
      const size_t dst = j;
      if (part < kVecs) kc_w[dst * kVecs + part] = x;
      else if (part < 2 * kVecs) vc_w[dst * kVecs + part - kVecs] = x;
      else {
        ks[dst * (D / 64)] = x.x;
        vs[dst * (D / 64)] = x.z;
        if (D == 128) { ks[dst * (D / 64) + D / 128] = x.y; vs[dst * (D / 64) + D / 128] = x.w; }
        w[dst] = weight;
      }
    }
    __syncthreads();
  }
}

__global__ void clamp_lengths_kernel(const int* lengths, int* out, int batch, int keep, int max_seq) {
  pdl_wait();
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < batch) out[b] = lengths[b] <= max_seq ? min(lengths[b], keep) : lengths[b];
}

}  // namespace

int launch_kv4_append(const Kv4AppendArgs& a, cudaStream_t stream) {
  const long long units = 2ll * a.batch * a.tokens * a.cache.hkv, threads = units * (a.cache.head_dim / 8);
  if (units == 0) return 0;
  const long long blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  if (a.cache.head_dim == 128) append_kernel<128><<<(unsigned)blocks, 256, 0, stream>>>(a);
  else append_kernel<64><<<(unsigned)blocks, 256, 0, stream>>>(a);
  return (int)cudaGetLastError();
}

int launch_kv4_read(const Kv4Cache& cache, int batch, int n, void* k_out, void* v_out, cudaStream_t stream) {
  const long long units = 2ll * batch * n * cache.hkv, threads = units * (cache.head_dim / 8);
  if (units == 0) return 0;
  const long long blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  if (cache.head_dim == 128) read_kernel<128><<<(unsigned)blocks, 256, 0, stream>>>(cache, batch, n, k_out, v_out);
  else read_kernel<64><<<(unsigned)blocks, 256, 0, stream>>>(cache, batch, n, k_out, v_out);
  return (int)cudaGetLastError();
}

int launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t stream) {
  if (a.batch == 0) return 0;
  if (a.cache.head_dim == 128) evict_kernel<128><<<a.batch * a.cache.hkv, kEvictThreads, 0, stream>>>(a);
  else evict_kernel<64><<<a.batch * a.cache.hkv, kEvictThreads, 0, stream>>>(a);
  clamp_lengths_kernel<<<(a.batch + 255) / 256, 256, 0, stream>>>(a.lengths, a.new_lengths, a.batch, a.keep,
                                                                    a.cache.max_seq);
  return (int)cudaGetLastError();
}

}  // namespace smr
