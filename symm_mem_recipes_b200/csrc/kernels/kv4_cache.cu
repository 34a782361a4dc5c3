// Rows into and out of a 4-bit KV cache (kv4.cuh), and the eviction that compacts it.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../device/mbarrier.cuh"
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

// D / 8 lanes take a row of keys or of values, eight dims a lane, kRows rows a thread one after the other: their loads are in
// flight together.  blockIdx.y is the sequence, blockIdx.z keys or values; row i of a sequence is head i % hkv of token i / hkv.
// Memory-bound: 2 bytes a value on one side, 0.56 on the other.
template <int D, int kRows>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ Kv4AppendArgs a) {
  pdl_wait();
  constexpr int kLanes = D / 8, kStep = 256 / kLanes;
  const int l = threadIdx.x % kLanes, g = l >> 2, c = l & 3, b = blockIdx.y, hkv = a.cache.hkv;
  const bool is_value = blockIdx.z != 0;
  const long long* stride = is_value ? a.v_stride : a.k_stride;
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(is_value ? a.v : a.k) + b * stride[0] + l * 8;
  // `start` and `counts` may be any numbers: nothing is added to them before they are known to be slots
  const int start = a.start_dev ? a.start_dev[b] : a.start;
  int tokens = start >= 0 && start < a.cache.max_seq ? min(a.tokens, a.cache.max_seq - start) : 0;
  if (a.counts != nullptr) tokens = min(tokens, a.counts[b]);
  const int rows = tokens > 0 ? tokens * hkv : 0;      // at most the sequence's slots in all heads
  const int first = blockIdx.x * (kStep * kRows) + threadIdx.x / kLanes;
  Vec16 raw[kRows];
  int t[kRows], h[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int i = first + u * kStep;
    raw[u] = Vec16{0, 0, 0, 0};
    t[u] = i / hkv;
    h[u] = i - t[u] * hkv;
    if (i < rows) raw[u] = ld_16_nc(src + t[u] * stride[1] + h[u] * stride[2]);
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    float f[8];
    unpack8(raw[u], f);
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
    if (first + u * kStep >= rows) continue;
    const size_t at = ((size_t)b * hkv + h[u]) * a.cache.slots + start + t[u];
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
}

template <int D, int kRows>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ Kv4Cache cache, int n, void* k_out, void* v_out) {
  pdl_wait();
  constexpr int kLanes = D / 8, kStep = 256 / kLanes;
  const int l = threadIdx.x % kLanes, g = l >> 2, c = l & 3, b = blockIdx.y, hkv = cache.hkv, rows = n * hkv;
  const bool is_value = blockIdx.z != 0;
  const uint8_t* codes = (is_value ? cache.v_codes : cache.k_codes) + (is_value ? 2 * c * (D / 16) + g * 2 : c * (D / 8) + g * 4);
  const __nv_bfloat16* scales = static_cast<const __nv_bfloat16*>(is_value ? cache.v_scales : cache.k_scales) + g;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(is_value ? v_out : k_out) + (size_t)b * rows * D + l * 8;
  const int first = blockIdx.x * (kStep * kRows) + threadIdx.x / kLanes;
  uint32_t word[kRows];
  float s[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int i = first + u * kStep;
    if (i >= rows) continue;
    const int t = i / hkv, h = i - t * hkv;
    const size_t at = ((size_t)b * hkv + h) * cache.slots + t;
    const uint8_t* p = codes + at * (D / 2);
    word[u] = is_value ? *reinterpret_cast<const uint16_t*>(p) | (uint32_t)*reinterpret_cast<const uint16_t*>(p + D / 16) << 16
                       : *reinterpret_cast<const uint32_t*>(p);
    s[u] = __bfloat162float(scales[at * (D / kGroup)]);
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int i = first + u * kStep;
    if (i >= rows) continue;
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = s[u] * (float)((int)(word[u] >> (4 * k) & 15u) - 8);
    Vec16 o;
    o.x = pack_bf16x2(f[0], f[1]); o.y = pack_bf16x2(f[2], f[3]);
    o.z = pack_bf16x2(f[4], f[5]); o.w = pack_bf16x2(f[6], f[7]);
    st_16(out + (size_t)i * D, o);
  }
}

// ---- eviction ----
// Of a head's n slots the last `recent` stay, and of the others the heaviest, so that `keep` stay in all; equal weights go
// to the lower slot.  The kept rows move down in slot order.  A cluster of C CTAs takes a head, each a run of its slots:
//   1. a radix selection over the weights as ordered integers (kept in shared memory, so weights are read once) finds the
//      weight of the last one kept, eight bits a pass; the CTAs' counts meet over distributed shared memory;
//   2. warps count what stays of their own runs, the counts give every kept slot its place, and the places' sources are listed;
//   3. rows move in chunks of places, 128 bytes and more a thread in registers.  A chunk is read whole before any of it
//      is written; a place is never above its source and sources increase, so a chunk's writes cannot reach the sources of
//      a later one.
constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictKeys = 40960;      // weights of a CTA that stay in shared memory; beyond them they are read again

// Order of a weight as an integer; NaN counts as an infinity; above all weights: the slots that stay anyway.
__device__ __forceinline__ uint32_t worth_of(float w, bool stays) {
  if (stays) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFF800000u;
  if (u == 0x80000000u) return u;                    // -0 and 0 are equal
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ int load_remote(const int* local, int cta) {
  uint32_t remote;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(cta));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int D>
__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const __grid_constant__ Kv4EvictArgs a, int ctas, int cached) {
  pdl_wait();
  extern __shared__ uint32_t keys[];                 // [cached]
  __shared__ int hist[2][256];                       // two passes in turn: one barrier a pass
  __shared__ int total[256];
  __shared__ int counts[2];                          // of this CTA: slots above the last worth kept, slots equal to it
  __shared__ int warp_counts[2][kEvictWarps];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.x / ctas, cta = blockIdx.x % ctas, b = head / a.cache.hkv;
  const int n = a.lengths[b], keep = a.keep;
  const bool cut = n > keep && n <= a.cache.max_seq;
  if (tid == 0 && cta == 0 && head % a.cache.hkv == 0) a.new_lengths[b] = cut ? keep : n;
  if (!cut) return;                                  // the whole cluster
  const size_t base = (size_t)head * a.cache.slots;
  float* w = a.cache.weights + base;
  const int protect = n - a.recent;
  // a whole number of warps' turns a CTA and a warp
  const int run = ((n + ctas - 1) / ctas + kEvictThreads - 1) / kEvictThreads * kEvictThreads;
  const int lo = min(cta * run, n), mine = min(lo + run, n) - lo;
  for (int i = tid; i < min(mine, cached); i += kEvictThreads) keys[i] = worth_of(w[lo + i], lo + i >= protect);
  auto key = [&](int i) { return i < cached ? keys[i] : worth_of(w[lo + i], lo + i >= protect); };
  if (tid < 256) hist[0][tid] = hist[1][tid] = 0;
  __syncthreads();

  uint32_t prefix = 0, mask = 0;
  int left = keep;                                   // slots still to be found among those that match the prefix
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    int* bins = hist[pass & 1];
    for (int i = tid; i < mine; i += kEvictThreads) {
      const uint32_t u = key(i);
      if ((u & mask) == prefix) atomicAdd(&bins[u >> shift & 255], 1);
    }
    if (ctas > 1) cluster_barrier();
    else __syncthreads();
    if (tid < 256) {
      int sum = 0;
      if (ctas == 1) sum = bins[tid];
      else
        for (int r = 0; r < ctas; ++r) sum += load_remote(&bins[tid], r);
      total[tid] = sum;
      if (pass > 0) hist[(pass + 1) & 1][tid] = 0;   // the last pass's, which nobody reads any more
    }
    __syncthreads();
    if (warp == 0) {      // a lane has eight bins, from the top down
      int v[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += v[i] = total[255 - 8 * lane - i];
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
      }
      before -= sum;
      if (before < left && before + sum >= left) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (before < left && before + v[i] >= left) {
            found[0] = 255 - 8 * lane - i;
            found[1] = left - before;
          }
          before += v[i];
        }
      }
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    left = found[1];
    mask |= 255u << shift;
  }
  // `prefix` is the least worth that stays, of which the first `left` slots do
  const int per_warp = run / kEvictWarps, w0 = min(warp * per_warp, mine), w1 = min(w0 + per_warp, mine);
  int above = 0, equal = 0;
  for (int i = w0 + lane; i - lane < w1; i += 32) {
    const uint32_t u = i < w1 ? key(i) : 0;
    above += __popc(__ballot_sync(0xffffffffu, i < w1 && u > prefix));
    equal += __popc(__ballot_sync(0xffffffffu, i < w1 && u == prefix));
  }
  if (lane == 0) {
    warp_counts[0][warp] = above;
    warp_counts[1][warp] = equal;
  }
  __syncthreads();
  if (tid < 2) {
    int sum = 0;
    for (int i = 0; i < kEvictWarps; ++i) sum += warp_counts[tid][i];
    counts[tid] = sum;
  }
  if (ctas > 1) cluster_barrier();
  else __syncthreads();
  // slots above and equal in front of this warp's run
  int above_before = 0, equal_before = 0;
  for (int r = 0; r < cta; ++r) {
    above_before += load_remote(&counts[0], r);
    equal_before += load_remote(&counts[1], r);
  }
  for (int i = 0; i < warp; ++i) {
    above_before += warp_counts[0][i];
    equal_before += warp_counts[1][i];
  }
  int* list = a.list + (size_t)head * keep;
  const uint32_t below = (1u << lane) - 1;
  for (int i = w0 + lane; i - lane < w1; i += 32) {
    const uint32_t u = i < w1 ? key(i) : 0;
    const uint32_t is_above = __ballot_sync(0xffffffffu, i < w1 && u > prefix);
    const uint32_t is_equal = __ballot_sync(0xffffffffu, i < w1 && u == prefix);
    const int equal_rank = equal_before + __popc(is_equal & below);
    const int place = above_before + __popc(is_above & below) + min(equal_rank, left);
    if ((is_above >> lane & 1) || ((is_equal >> lane & 1) && equal_rank < left)) list[place] = lo + i;
    above_before += __popc(is_above);
    equal_before += __popc(is_equal);
  }
  if (ctas > 1) cluster_barrier();      // the list is written, and nothing of another CTA's shared memory is read any more
  else __syncthreads();

  constexpr int kVecs = D / 32, kParts = 2 * kVecs, kWords = D / 64;      // 16-byte parts of codes, words of scales a row
  Vec16* kc = reinterpret_cast<Vec16*>(a.cache.k_codes + base * (D / 2));
  Vec16* vc = reinterpret_cast<Vec16*>(a.cache.v_codes + base * (D / 2));
  uint32_t* ks = static_cast<uint32_t*>(a.cache.k_scales) + base * kWords;
  uint32_t* vs = static_cast<uint32_t*>(a.cache.v_scales) + base * kWords;
  const int threads = ctas * kEvictThreads, me = cta * kEvictThreads + tid;
  for (int first = 0; first < keep; first += threads) {      // a chunk: a row a thread, its codes spread over kParts threads
    Vec16 x[kParts];
    uint32_t scale[2 * kWords];
    float weight = 0.0f;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int item = i * threads + me, row = first + item / kParts, part = item % kParts;
      if (row < keep) {
        const size_t src = list[row];
        x[i] = part < kVecs ? kc[src * kVecs + part] : vc[src * kVecs + part - kVecs];
      }
    }
    const int row = first + me;
    if (row < keep) {
      const size_t src = list[row];
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        scale[i] = ks[src * kWords + i];
        scale[kWords + i] = vs[src * kWords + i];
      }
      weight = w[src];
    }
    if (ctas > 1) cluster_barrier();
    else __syncthreads();
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int item = i * threads + me, to = first + item / kParts, part = item % kParts;
      if (to < keep) (part < kVecs ? kc[(size_t)to * kVecs + part] : vc[(size_t)to * kVecs + part - kVecs]) = x[i];
    }
    if (row < keep) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        ks[(size_t)row * kWords + i] = scale[i];
        vs[(size_t)row * kWords + i] = scale[kWords + i];
      }
      w[row] = weight;
    }
  }
}

template <class... Params, class... Args>
int launch_kernel(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attrs[2] = {};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Four rows a thread once that still gives every SM several CTAs.
constexpr int kManyRows = 4;
bool many_rows(long long rows, int batch, int head_dim) {
  const int step = 256 / (head_dim / 8);
  return 2 * batch * rows / (step * kManyRows) >= 148 * 4;
}

template <int D, int kRows>
int append(const Kv4AppendArgs& a, long long rows, cudaStream_t stream) {
  constexpr int kBlock = 256 / (D / 8) * kRows;
  return launch_kernel(append_kernel<D, kRows>, dim3((unsigned)((rows + kBlock - 1) / kBlock), a.batch, 2), 256, 0, 1, stream, a);
}
template <int D, int kRows>
int read(const Kv4Cache& cache, int batch, int n, void* k_out, void* v_out, cudaStream_t stream) {
  constexpr int kBlock = 256 / (D / 8) * kRows;
  const long long rows = (long long)n * cache.hkv;
  return launch_kernel(read_kernel<D, kRows>, dim3((unsigned)((rows + kBlock - 1) / kBlock), batch, 2), 256, 0, 1, stream, cache, n,
                       k_out, v_out);
}

}  // namespace

int launch_kv4_append(const Kv4AppendArgs& a, cudaStream_t stream) {
  const long long rows = (long long)std::min(a.tokens, a.cache.max_seq) * a.cache.hkv;      // no more fit
  if (rows == 0 || a.batch == 0) return 0;
  const bool many = many_rows(rows, a.batch, a.cache.head_dim);
  if (a.cache.head_dim == 128) return many ? append<128, kManyRows>(a, rows, stream) : append<128, 1>(a, rows, stream);
  return many ? append<64, kManyRows>(a, rows, stream) : append<64, 1>(a, rows, stream);
}

int launch_kv4_read(const Kv4Cache& cache, int batch, int n, void* k_out, void* v_out, cudaStream_t stream) {
  const long long rows = (long long)n * cache.hkv;
  if (rows == 0 || batch == 0) return 0;
  const bool many = many_rows(rows, batch, cache.head_dim);
  if (cache.head_dim == 128)
    return many ? read<128, kManyRows>(cache, batch, n, k_out, v_out, stream) : read<128, 1>(cache, batch, n, k_out, v_out, stream);
  return many ? read<64, kManyRows>(cache, batch, n, k_out, v_out, stream) : read<64, 1>(cache, batch, n, k_out, v_out, stream);
}

int launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t stream) {
  if (a.batch == 0) return 0;
  // CTAs a head: 1024 slots each and more, eight at most (what a cluster may have everywhere)
  const int ctas = a.cache.slots <= 1024 ? 1 : a.cache.slots <= 2048 ? 2 : a.cache.slots <= 4096 ? 4 : 8;
  const int run = ((a.cache.max_seq + ctas - 1) / ctas + kEvictThreads - 1) / kEvictThreads * kEvictThreads;
  const int cached = std::min(run, kEvictKeys);
  const size_t smem = (size_t)cached * sizeof(uint32_t);
  auto kernel = a.cache.head_dim == 128 ? evict_kernel<128> : evict_kernel<64>;
  if (int e = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) return e;
  return launch_kernel(kernel, dim3((unsigned)(a.batch * a.cache.hkv * ctas)), kEvictThreads, smem, ctas, stream, a, ctas, cached);
}

}  // namespace smr
