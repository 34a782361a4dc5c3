// Rows into and out of a 4-bit KV cache (kv4.cuh), and the eviction that compacts it.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../device/mbarrier.cuh"
#include "../device/pdl.cuh"
#include "kv4.cuh"
#include "launch.h"
#include "pdl_launch.h"
#include "residency.h"

namespace smr {

namespace {

using namespace kv4;

__device__ __forceinline__ void unpack8(const Vec16& v, float (&f)[8]) {
  f[0] = bf16lo_to_f32(v.x); f[1] = bf16hi_to_f32(v.x);
  f[2] = bf16lo_to_f32(v.y); f[3] = bf16hi_to_f32(v.y);
  f[4] = bf16lo_to_f32(v.z); f[5] = bf16hi_to_f32(v.z);
  f[6] = bf16lo_to_f32(v.w); f[7] = bf16hi_to_f32(v.w);
}

// i / d for i < 2^30 by a multiplication: with s = 30 + ceil(log2 d) and m = 2^s / d rounded up, m * i / 2^s is above i / d by
// less than i * d / (d * 2^s) <= 1 / d, which reaches no whole number; m <= 2^31 + 1, so m * i stays below 2^62.
struct Divisor {
  uint32_t d, step_div, step_mod;      // and of one number, the step from a thread's row to its next
  uint32_t shift;
  uint64_t m;
  Divisor(uint32_t by, uint32_t step) : d(by), step_div(step / by), step_mod(step % by), shift(30) {
    while (1ull << (shift - 30) < by) ++shift;
    m = ((1ull << shift) + by - 1) / by;
  }
};
// The row of a thread: token t, head h; kRows of them, a step apart.
struct Row {
  int t, h;
  __device__ __forceinline__ Row(int i, const Divisor& by) : t((int)(by.m * (uint64_t)i >> by.shift)), h(i - t * (int)by.d) {}
  __device__ __forceinline__ void next(const Divisor& by) {
    t += by.step_div;
    h += by.step_mod;
    if (h >= (int)by.d) {
      h -= by.d;
      ++t;
    }
  }
};

// D / 8 lanes take a row of keys or of values, eight dims a lane, kRows rows a thread one after the other: their loads are in
// flight together.  blockIdx.y is the sequence, blockIdx.z keys or values; row i of a sequence is head i % hkv of token i / hkv.
// 2 bytes a value on one side, 0.56 on the other: 16384 tokens of 8 heads of 128 go in in 19 us and come back in 15, 34 together
// where the bytes take 26 at the copy rate; the rest is two launches that fill and drain.  (57 us with a 64-bit division for
// the row and an IEEE division and a comparison a value.)  Two rows a thread at a time 35, eight 38; half a group a lane, which
// halves the instructions, and tokens before heads, which makes a CTA's side of the cache one run of memory, 33 to 36.
template <int D, int kRows, bool kValue>
__device__ __forceinline__ void append_rows(const Kv4AppendArgs& a, const Divisor& hkv) {
  constexpr int kLanes = D / 8, kStep = 256 / kLanes;
  const int l = threadIdx.x % kLanes, g = l >> 2, c = l & 3, b = blockIdx.y;
  const long long* stride = kValue ? a.v_stride : a.k_stride;
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(kValue ? a.v : a.k) + b * stride[0] + l * 8;
  // `start` and `counts` may be any numbers: nothing is added to them before they are known to be slots
  const int start = a.start_dev ? a.start_dev[b] : a.start;
  int tokens = start >= 0 && start < a.cache.max_seq ? min(a.tokens, a.cache.max_seq - start) : 0;
  if (a.counts != nullptr) tokens = min(tokens, a.counts[b]);
  const int first = blockIdx.x * (kStep * kRows) + threadIdx.x / kLanes;
  Vec16 raw[kRows];
  Row row(first, hkv);
#pragma unroll
  for (int u = 0; u < kRows; ++u, row.next(hkv)) {
    raw[u] = Vec16{0, 0, 0, 0};
    if (row.t < tokens) raw[u] = ld_16_stream(src + row.t * stride[1] + row.h * stride[2]);
  }
  row = Row(first, hkv);
  const size_t base = (size_t)b * hkv.d * a.cache.slots + max(start, 0);
  // a value row's part has two bytes a group: two lanes of neighbouring groups trade halves and write four bytes each
  uint8_t* codes = kValue ? a.cache.v_codes + (2 * c + (g & 1)) * (D / 16) + (g >> 1) * 4 : a.cache.k_codes + c * (D / 8) + g * 4;
  uint16_t* scales = static_cast<uint16_t*>(kValue ? a.cache.v_scales : a.cache.k_scales) + g;
#pragma unroll
  for (int u = 0; u < kRows; ++u, row.next(hkv)) {
    uint32_t largest = max_magnitude(max_magnitude(raw[u].x, raw[u].y), max_magnitude(raw[u].z, raw[u].w));
    largest = max(largest & 0xFFFFu, largest >> 16);
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    const Scale s = scale_of(largest);
    float f[8];
    unpack8(raw[u], f);
    uint32_t word = 0x4B400000u * 0xEEEEEEEFu;      // less 0x4B400000 in every nibble's place: 0x11111111 of them
#pragma unroll
    for (int i = 0; i < 8; ++i) word += rounded(f[i], s) << (4 * i);
    if (!s.finite) word = 0x88888888u;
    if (kValue) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, __byte_perm(word, 0, (g & 1) ? 0x5410 : 0x7632), 4);
      word = __byte_perm(word, other, (g & 1) ? 0x3254 : 0x5410);
    }
    if (row.t < tokens) {
      const size_t at = base + (size_t)row.h * a.cache.slots + row.t;
      *reinterpret_cast<uint32_t*>(codes + at * (D / 2)) = word;
      if (c == 0) scales[at * (D / kGroup)] = s.bits;
      if (!kValue && l == 0 && a.cache.weights != nullptr) a.cache.weights[at] = 0.0f;      // of the slot's last tenant
    }
  }
}
template <int D, int kRows>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ Kv4AppendArgs a, const __grid_constant__ Divisor hkv) {
  pdl_wait();
  if (blockIdx.z == 0) append_rows<D, kRows, false>(a, hkv);
  else append_rows<D, kRows, true>(a, hkv);
}

template <int D, int kRows, bool kValue>
__device__ __forceinline__ void read_rows(const Kv4Cache& cache, const Divisor& hkv, int n, void* to) {
  constexpr int kLanes = D / 8, kStep = 256 / kLanes;
  const int l = threadIdx.x % kLanes, g = l >> 2, c = l & 3, b = blockIdx.y;
  const uint8_t* codes = kValue ? cache.v_codes + 2 * c * (D / 16) + g * 2 : cache.k_codes + c * (D / 8) + g * 4;
  const uint16_t* scales = static_cast<const uint16_t*>(kValue ? cache.v_scales : cache.k_scales) + g;
  const int first = blockIdx.x * (kStep * kRows) + threadIdx.x / kLanes;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(to) + ((size_t)b * n * hkv.d + first) * D + l * 8;
  const size_t base = (size_t)b * hkv.d * cache.slots;
  uint32_t word[kRows];
  uint16_t s[kRows];
  Row row(first, hkv);
  int rows = 0;
#pragma unroll
  for (int u = 0; u < kRows; ++u, row.next(hkv)) {
    word[u] = s[u] = 0;
    if (row.t < n) {
      rows = u + 1;
      const size_t at = base + (size_t)row.h * cache.slots + row.t;
      const uint8_t* p = codes + at * (D / 2);
      word[u] = kValue ? *reinterpret_cast<const uint16_t*>(p) | (uint32_t)*reinterpret_cast<const uint16_t*>(p + D / 16) << 16
                       : *reinterpret_cast<const uint32_t*>(p);
      s[u] = scales[at * (D / kGroup)];
    }
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (u >= rows) break;
    // 128 + n as bf16, less 136, is exact; the product with the scale is rounded once
    const __nv_bfloat162 scale = __bfloat162bfloat162(__ushort_as_bfloat16(s[u]));
    uint32_t v[4];      // dims j and j + 4
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t n4 = (word[u] >> (4 * j) & 0x000F000Fu) | 0x43004300u;
      const __nv_bfloat162 x = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&n4), __float2bfloat162_rn(136.0f)), scale);
      v[j] = *reinterpret_cast<const uint32_t*>(&x);
    }
    st_16(out + (size_t)u * kStep * D, Vec16{__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                                             __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632)});
  }
}
template <int D, int kRows>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ Kv4Cache cache, const __grid_constant__ Divisor hkv, int n,
                                                   void* k_out, void* v_out) {
  pdl_wait();
  if (blockIdx.z == 0) read_rows<D, kRows, false>(cache, hkv, n, k_out);
  else read_rows<D, kRows, true>(cache, hkv, n, v_out);
}

// ---- eviction ----
// Of a head's n slots the last `recent` stay, and of the others the heaviest, so that `keep` stay in all; equal weights go
// to the lower slot.  The kept rows move down in slot order.  A cluster of C CTAs takes a head, each a run of its slots:
//   1. a radix selection over the weights as ordered integers (kept in shared memory, so weights are read once) finds the
//      weight of the last one kept, eight bits a pass; the CTAs' counts meet over distributed shared memory;
//   2. the CTAs' counts of the passes and the warps' of their own runs give every kept slot its place, and the places' sources
//      are listed;
//   3. rows move in chunks of places, through shared memory by asynchronous copies (in registers 2048 rows of a cluster spilled
//      and took 28 us of a prompt's 50).  A chunk is read whole before any of it is written; a place is never above its source
//      and sources increase, so a chunk's writes cannot reach the sources of a later one.
// 64 heads of up to 32768 to 4096 slots take 43 us: 3 for the weights, 2.3 a pass (a cluster barrier and remote loads), 4 for counts and
// list, 16 for the rows.
constexpr int kEvictThreads = 256;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictCtas = 8;          // of a cluster at most
constexpr int kEvictKeys = 40960;      // weights of a CTA that stay in shared memory; beyond them they are read again

// Order of a weight as an integer; NaN counts as an infinity; above all weights: the slots that stay anyway.
__device__ __forceinline__ uint32_t worth_of(float w, bool stays) {
  if (stays) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFF800000u;
  if (u == 0x80000000u) return u;                    // -0 and 0 are equal
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
template <int D>
struct EvictRows {
  static constexpr int kVecs = D / 32, kWords = D / 64;      // 16-byte parts of a row's codes, words of its scales
  Vec16 codes[kEvictThreads * 2 * kVecs];
  uint32_t scales[2][kEvictThreads][kWords];
  float weights[kEvictThreads];
};
template <int N>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(N) : "memory");
}
// Sums of an integer in shared memory over the cluster's first `mine` and `ctas` CTAs; the loads are in flight together.
__device__ __forceinline__ int2 sum_over_ctas(const int* local, int mine, int ctas) {
  int v[kEvictCtas];
#pragma unroll
  for (int r = 0; r < kEvictCtas; ++r) {
    v[r] = 0;
    if (r < ctas) {
      uint32_t remote;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(r));
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v[r]) : "r"(remote) : "memory");
    }
  }
  int2 sum = make_int2(0, 0);
#pragma unroll
  for (int r = 0; r < kEvictCtas; ++r) {
    sum.x += r < mine ? v[r] : 0;
    sum.y += v[r];
  }
  return sum;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int D>
__global__ void __launch_bounds__(kEvictThreads, 4) evict_kernel(const __grid_constant__ Kv4EvictArgs a, int ctas, int cached) {
  pdl_wait();
  extern __shared__ __align__(16) uint32_t keys[];   // [cached], then EvictRows
  __shared__ int hist[2][256];                       // two passes in turn: one barrier a pass
  __shared__ int2 total[256];                        // counts of the CTAs in front of this one, and of all
  __shared__ int warp_counts[2][kEvictWarps];
  __shared__ int found[4];                           // the digit, how many are left, and in front of this CTA: above it, with it
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
  int above_before = 0, equal_before = 0;            // in front of this CTA's run: slots of more worth, slots that match
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
      total[tid] = ctas == 1 ? make_int2(0, bins[tid]) : sum_over_ctas(&bins[tid], cta, ctas);
      if (pass > 0) hist[(pass + 1) & 1][tid] = 0;   // the last pass's, which nobody reads any more
    }
    __syncthreads();
    if (warp == 0) {      // a lane has eight bins, from the top down
      int2 v[8], sum = make_int2(0, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = total[255 - 8 * lane - i];
        sum.x += v[i].x;
        sum.y += v[i].y;
      }
      int2 before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, before.x, o), y = __shfl_up_sync(0xffffffffu, before.y, o);
        if (lane >= o) {
          before.x += x;
          before.y += y;
        }
      }
      before.x -= sum.x;
      before.y -= sum.y;
      if (before.y < left && before.y + sum.y >= left) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (before.y < left && before.y + v[i].y >= left) {
            found[0] = 255 - 8 * lane - i;
            found[1] = left - before.y;
            found[2] = before.x;
            found[3] = v[i].x;
          }
          before.x += v[i].x;
          before.y += v[i].y;
        }
      }
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    left = found[1];
    above_before += found[2];
    equal_before = found[3];
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
  for (int i = 0; i < warp; ++i) {                   // and in front of this warp's
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

  using Staged = EvictRows<D>;
  constexpr int kVecs = Staged::kVecs, kParts = 2 * kVecs, kWords = Staged::kWords;
  Vec16* kc = reinterpret_cast<Vec16*>(a.cache.k_codes + base * (D / 2));
  Vec16* vc = reinterpret_cast<Vec16*>(a.cache.v_codes + base * (D / 2));
  uint32_t* ks = static_cast<uint32_t*>(a.cache.k_scales) + base * kWords;
  uint32_t* vs = static_cast<uint32_t*>(a.cache.v_scales) + base * kWords;
  Staged& rows = *reinterpret_cast<Staged*>(keys);   // the keys are done with
  for (int chunk = 0; chunk < keep; chunk += ctas * kEvictThreads) {
    const int first = chunk + cta * kEvictThreads;   // this CTA's places: a row a thread, its codes spread over kParts threads
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int item = i * kEvictThreads + tid, row = first + item / kParts, part = item % kParts;
      if (row < keep) {
        const size_t src = list[row];
        copy_async<16>(&rows.codes[item], part < kVecs ? kc + src * kVecs + part : vc + src * kVecs + part - kVecs);
      }
    }
    if (first + tid < keep) {
      const size_t src = list[first + tid];
      copy_async<4 * kWords>(rows.scales[0][tid], ks + src * kWords);
      copy_async<4 * kWords>(rows.scales[1][tid], vs + src * kWords);
      copy_async<4>(&rows.weights[tid], w + src);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (ctas > 1) cluster_barrier();
    else __syncthreads();
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int item = i * kEvictThreads + tid, part = item % kParts;
      const size_t to = first + item / kParts;
      if (to < keep) *(part < kVecs ? kc + to * kVecs + part : vc + to * kVecs + part - kVecs) = rows.codes[item];
    }
    if (first + tid < keep) {
      const size_t to = first + tid;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        ks[to * kWords + i] = rows.scales[0][tid][i];
        vs[to * kWords + i] = rows.scales[1][tid][i];
      }
      w[to] = rows.weights[tid];
    }
    __syncthreads();      // the staged rows are written before the next ones come in
  }
}

// Four rows a thread once that still gives every SM several CTAs.
constexpr int kManyRows = 4;
bool many_rows(long long rows, int batch, int head_dim) {
  const int step = 256 / (head_dim / 8);
  return 2 * batch * rows / (step * kManyRows) >= 4 * device_sms();
}

template <int D, int kRows>
int append(const Kv4AppendArgs& a, long long rows, cudaStream_t stream) {
  constexpr int kBlock = 256 / (D / 8) * kRows;
  return launch_pdl(append_kernel<D, kRows>, dim3((unsigned)((rows + kBlock - 1) / kBlock), a.batch, 2), 256, 0, 1, stream, a,
                       Divisor(a.cache.hkv, 256 / (D / 8)));
}
template <int D, int kRows>
int read(const Kv4Cache& cache, int batch, int n, void* k_out, void* v_out, cudaStream_t stream) {
  constexpr int kBlock = 256 / (D / 8) * kRows;
  const long long rows = (long long)n * cache.hkv;
  return launch_pdl(read_kernel<D, kRows>, dim3((unsigned)((rows + kBlock - 1) / kBlock), batch, 2), 256, 0, 1, stream, cache,
                       Divisor(cache.hkv, 256 / (D / 8)), n, k_out, v_out);
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
  const size_t smem = std::max(cached * sizeof(uint32_t), a.cache.head_dim == 128 ? sizeof(EvictRows<128>) : sizeof(EvictRows<64>));
  auto kernel = a.cache.head_dim == 128 ? evict_kernel<128> : evict_kernel<64>;
  return launch_pdl(kernel, dim3((unsigned)(a.batch * a.cache.hkv * ctas)), kEvictThreads, smem, ctas, stream, a, ctas, cached);
}

}  // namespace smr
