// The paged cache in 4 bits: quantising keys and values as they are written, and
// reading them back.
//
// Sixteen numbers x of one head of one token share a scale s = e4m3(max |x| / 6)
// and are held as c = e2m1(x / s), 4.5 bits a number (x in units of the cache, a
// power of two).  Both roundings are to nearest even and saturate.  The
// quotients are fp32; rounding them first changes no code, for any fp32 x: an
// edge m between two codes times s is an fp32 number T (at most 6 bits).  At
// x = T the quotient is m exactly, and for x != T it is off m by more than half a
// step at m: x differs from T by a step of T, more than 2^-24 of it, and half a
// step at m is 2^-24 of m by m's leading digits (1, 1.25, 1.5 or 1.75), so that
// 2 m' / T' > 1.06 remains between them (T' < 2 the leading digits of T, at most
// 15/8 where m' is 1).  The same holds for the scale, with 6 in the place of s.
//
// Both kernels only move memory: a scale's sixteen numbers to a thread, 32 bytes
// of bf16 on one side and 9 on the other.  65536 tokens of 8 heads of 128 are read
// in 61 us (5.6 TB/s, bound by memory), 16384 written in 27 to 29 (3 TB/s): half of that
// is instructions (two thirds of cycles issue: 270 for sixteen numbers, 126 of them
// the quantising), the rest the chain from the slots to the first store.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "attention.h"
#include "serving.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

constexpr int kWriteThreads = 256;
constexpr int kWriteTokens = 2048;         // of a CTA at most
constexpr int kWriteAtOnce = 1 << 20;      // of a launch at most

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The slot of token i, -1 for none; one outside of the cache is recorded and counts as none.
__device__ __forceinline__ int cache_slot(const void* slots, int wide, long long i, const CacheView& c, DeviceStatus* st, int kernel_id) {
  const long long s = wide ? ((const long long*)slots)[i] : (long long)((const int*)slots)[i];
  if (s < 0) return -1;
  const long long bound = (long long)c.pages << c.page_shift;
  if (s >= bound) {
    record_status(st, kBoundsViolation, kernel_id, s, bound);
    return -1;
  }
  return (int)s;
}

// Byte offset of a head's token in the codes; its scales lie at an eighth of it.  A page has less than 2^31 bytes.
template <int D>
__device__ __forceinline__ long long cache_offset(const CacheView& c, int slot, int head) {
  const uint32_t page = slot >> c.page_shift, at = slot & ((1 << c.page_shift) - 1);
  return (long long)((unsigned long long)page * (((uint32_t)c.heads << c.page_shift) * (uint32_t)(D / 2))) +
         (((uint32_t)head << c.page_shift) + at) * (uint32_t)(D / 2);
}

// Sixteen numbers of one row, as they lie.
template <typename T>
struct Sixteen {
  uint4 w[16 * sizeof(T) / 16];
};

template <typename T>
__device__ __forceinline__ void load16(const T* p, int vec, Sixteen<T>& x) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) x.w[i] = __ldg((const uint4*)p + i);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) ((T*)x.w)[i] = p[i];
  }
}

template <typename T>
__device__ __forceinline__ void as_floats(const Sixteen<T>& x, float (&f)[16]) {
  constexpr int W = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) {
    float part[W];
    unpack16<T>(x.w[i], part);
#pragma unroll
    for (int j = 0; j < W; ++j) f[W * i + j] = part[j];
  }
}

// x / s from the rounded reciprocal r of s: the product, and one correction by its remainder, which is exact in an fma
// (P. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990).  At x = m s it is m: the
// remainder is (m - q) s, and what it adds is off by 2^-24 of a step.  Where it underflows the code is 0 anyway.
__device__ __forceinline__ float divide(float x, float s, float r) {
  const float q = x * r;
  return fmaf(fmaf(-s, q, x), r, q);
}

// Four bytes of two codes each as f16 pairs, and eight fp32 numbers as codes; lower code first.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

__device__ __forceinline__ uint32_t codes_from_f32(const float* q) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return w;
}

// The scale (returned, a byte) and the codes of sixteen numbers.
__device__ __forceinline__ uint32_t quantise16(float (&x)[16], float unit, float per_unit, uint32_t (&codes)[2]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max_nan(top, fabsf(x[i]));
  top *= per_unit;
  if (top > 8192.f) {                 // behind 448 * 6 everything saturates; cut here, infinities do not meet below
    const float most = 8192.f * unit;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = fminf(fmaxf(x[i], -most), most);
    top = 8192.f;
  }
  const uint32_t scale = __nv_cvt_float_to_fp8(divide(top, 6.f, 1.f / 6.f), __NV_SATFINITE, __NV_E4M3);
  const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)scale, __NV_E4M3)));
  const float r = s > 0.f ? __frcp_rn(s) * per_unit : 0.f, back = s * unit;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = divide(x[i], back, r);
  codes[0] = codes_from_f32(x);
  codes[1] = codes_from_f32(x + 8);
  return scale;
}

// A CTA has `per` consecutive tokens (a power of two).  Where several tokens of
// a call name one slot, the last of them is kept: the CTA enters its tokens'
// slots into a hash table, the highest token of each, and looks up all later
// tokens' slots in it.
//
// Sixteen numbers to a thread, D / 16 lanes to a row of a head; rows go by value
// or key, head and token, the token fastest, so that no index needs a division.
// Two rows to a thread are loaded ahead, the first ones before the slots are
// looked through.
template <typename T, int D>
__global__ void __launch_bounds__(kWriteThreads) kv_cache_write_kernel(CacheWriteParams p) {
  extern __shared__ int table[];      // [per] slots, [size] keys, [size] last tokens
  const CacheView& c = p.c;
  griddep_wait();
  griddep_launch_dependents();
  const int per = 1 << p.per_shift, size = 2 * per;
  int *slot_of = table, *key = table + per, *last = key + size;
  const long long first = (long long)blockIdx.x << p.per_shift;
  const int n = (int)(p.N - first < per ? p.N - first : per);
  __shared__ int range[2];            // the least and the largest slot of the CTA's tokens
  if (threadIdx.x == 0) { range[0] = INT_MAX; range[1] = -1; }
  for (int i = threadIdx.x; i < size; i += kWriteThreads) { key[i] = -1; last[i] = -1; }
  constexpr int lane_shift = D == 128 ? 3 : 2, step = kWriteThreads >> lane_shift, U = 2;
  const int l = threadIdx.x & ((1 << lane_shift) - 1), rows = 2 * c.heads << p.per_shift;
  Sixteen<T> ahead[U];
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * step + (int)(threadIdx.x >> lane_shift), t = r & (per - 1), hv = r >> p.per_shift;
      if (r >= rows || t >= n) continue;
      const T* src = hv < c.heads ? (const T*)p.k + (first + t) * p.k_token + hv * p.k_head
                                  : (const T*)p.v + (first + t) * p.v_token + (hv - c.heads) * p.v_head;
      load16(src + 16 * l, p.vec, ahead[u]);
    }
  };
  load(0);
  __syncthreads();
  auto at = [&](int slot) { return (int)(((uint32_t)slot * 2654435761u) >> 16) & (size - 1); };
  for (int i = threadIdx.x; i < per; i += kWriteThreads) {
    const int s = i < n ? cache_slot(p.slots, p.slots64, first + i, c, p.status, kCacheWriteKernelId) : -1;
    slot_of[i] = s;
    if (s < 0) continue;
    int e = at(s);
    while (true) {                    // ends: the table is at most half full
      const int old = atomicCAS(&key[e], -1, s);
      if (old == -1 || old == s) break;
      e = (e + 1) & (size - 1);
    }
    atomicMax(&last[e], i);
    atomicMin(&range[0], s);
    atomicMax(&range[1], s);
  }
  __syncthreads();
  const long long low = range[0], high = range[1];
  auto look = [&](long long wide) {
    if (wide < low || wide > high) return;     // most of them: a CTA's tokens are neighbours in few pages
    const int s = (int)wide;
    int e = at(s), k;
    while ((k = key[e]) != -1 && k != s) e = (e + 1) & (size - 1);
    if (k == s) last[e] = 1 << 30;             // a later CTA has it
  };
  auto scan = [&](auto* slots) {
    // four at a time, eight such loads in flight; the tensor starts on the type's alignment only, and ends anywhere
    using S = std::remove_cv_t<std::remove_pointer_t<decltype(slots)>>;
    long long from = first + n;
    while (from < p.N && ((uintptr_t)(slots + from) & 15)) ++from;
    for (long long i = first + n + threadIdx.x; i < from; i += kWriteThreads) look(slots[i]);
    constexpr int V = 16 / sizeof(S), L = 8;
    const long long words = from < p.N ? (p.N - from) / V : 0;
    const uint4* const w = (const uint4*)(slots + from);
    for (long long i = threadIdx.x; i < words; i += L * kWriteThreads) {
      uint4 v[L];
#pragma unroll
      for (int u = 0; u < L; ++u)
        v[u] = i + u * kWriteThreads < words ? __ldg(w + i + u * kWriteThreads) : make_uint4(~0u, ~0u, ~0u, ~0u);   // -1: none
#pragma unroll
      for (int u = 0; u < L; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) look(((const S*)&v[u])[e]);
    }
    for (long long i = from + words * V + threadIdx.x; i < p.N; i += kWriteThreads) look(slots[i]);
  };
  if (high >= 0) {
    if (p.slots64) scan((const long long*)p.slots);
    else scan((const int*)p.slots);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kWriteThreads) {
    const int s = slot_of[i];
    if (s < 0) continue;
    int e = at(s);
    while (key[e] != s) e = (e + 1) & (size - 1);
    if (last[e] != i) slot_of[i] = -1;
  }
  __syncthreads();
  for (int r0 = 0; r0 < rows; r0 += U * step) {
    Sixteen<T> now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = ahead[u];
    load(r0 + U * step);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * step + (int)(threadIdx.x >> lane_shift), hv = r >> p.per_shift;
      const int slot = r < rows ? slot_of[r & (per - 1)] : -1;
      const bool value = hv >= c.heads;
      uint32_t codes[2], word = 0;
      if (slot >= 0) {
        float x[16];
        as_floats(now[u], x);
        word = quantise16(x, value ? c.v_unit : c.k_unit, value ? p.per_v_unit : p.per_k_unit, codes);
      }
      word <<= 8 * (l & 3);             // four lanes' scales to a word; a row's lanes have one slot
      word |= __shfl_xor_sync(0xffffffffu, word, 1);
      word |= __shfl_xor_sync(0xffffffffu, word, 2);
      if (slot >= 0) {
        const long long off = cache_offset<D>(c, slot, value ? hv - c.heads : hv);
        *(uint2*)((value ? c.v_codes : c.k_codes) + off + 8 * l) = make_uint2(codes[0], codes[1]);
        if ((l & 3) == 0) *(uint32_t*)((value ? c.v_scales : c.k_scales) + (off >> 3) + l) = word;
      }
    }
  }
}

// Sixteen numbers to a thread, of one head of four tokens in turn (all loads
// before the first store).  A code times its scale has at most 6 bits: nothing is
// rounded in bf16 either.
constexpr int kReadTokens = 4;

template <typename T, int D>
__global__ void __launch_bounds__(256) kv_cache_read_kernel(CacheReadParams p) {
  const CacheView& c = p.c;
  griddep_wait();
  griddep_launch_dependents();
  constexpr int lane_shift = D == 128 ? 3 : 2, step = 256 >> lane_shift;
  const int l = threadIdx.x & ((1 << lane_shift) - 1);
  const bool value = blockIdx.y >= c.heads;
  const int h = value ? blockIdx.y - c.heads : blockIdx.y;
  const uint8_t* const codes_of = (value ? c.v_codes : c.k_codes) + 8 * l;
  const uint8_t* const scales_of = (value ? c.v_scales : c.k_scales) + l;
  const float unit = value ? c.v_unit : c.k_unit;
  const long long first = (long long)blockIdx.x * (kReadTokens * step) + (threadIdx.x >> lane_shift);
  uint2 codes[kReadTokens];
  uint32_t scale[kReadTokens];
#pragma unroll
  for (int u = 0; u < kReadTokens; ++u) {
    const long long t = first + u * step;
    const int slot = t < p.N ? cache_slot(p.slots, p.slots64, t, c, p.status, kCacheReadKernelId) : -1;
    codes[u] = make_uint2(0, 0);
    scale[u] = 0;
    if (slot >= 0) {
      const long long off = cache_offset<D>(c, slot, h);
      codes[u] = __ldg((const uint2*)(codes_of + off));
      scale[u] = __ldg(scales_of + (off >> 3));
    }
  }
  const long long token = value ? p.v_token : p.k_token;
  T* dst = (value ? (T*)p.v + h * p.v_head : (T*)p.k + h * p.k_head) + first * token + 16 * l;
#pragma unroll
  for (int u = 0; u < kReadTokens; ++u, dst += step * token) {
    if (first + u * step >= p.N) return;
    uint32_t s = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)scale[u], __NV_E4M3).x;
    s |= s << 16;
    uint32_t half[2][4];
    codes_to_f16(codes[u].x, half[0]);
    codes_to_f16(codes[u].y, half[1]);
    float x[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = __half22float2(__hmul2(*(const __half2*)&half[j / 4][j % 4], *(const __half2*)&s));   // exact
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
    if (unit != 1.f) {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] *= unit;
    }
    if (p.vec) {
      if constexpr (sizeof(T) == 2) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
          w[j] = *(const uint32_t*)&b;
        }
        // all 32 bytes in one instruction where they are a sector: in two, each of which has a half of every sector of its
        // warp, the load-store unit was the limit (65536 tokens: 80 us)
        if (p.vec == 2) {
          asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                       "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                       : "memory");
        } else {
          ((uint4*)dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
          ((uint4*)dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) ((float4*)dst)[j] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) store_elem(dst, j, x[j], sizeof(T) == 2);
    }
  }
}

// Tokens of a CTA: up to four CTAs to an SM, which all fit.  A CTA looks through all later slots of its launch, so that grows with the
// square of the tokens: launches have up to kWriteAtOnce, in the tokens' order, the later one's tokens over the earlier one's (2^23
// tokens of one head of 64: 7.9 -> 2.5 ms, in slots all over the cache 68 -> 21).
void launch_cache_write(const CacheWriteParams& params, cudaStream_t s) {
  const long long wave = 4ll * serving_sm_count();
  for (long long done = 0; done < params.N; done += kWriteAtOnce) {
    CacheWriteParams p = params;
    p.N = std::min<long long>(params.N - done, kWriteAtOnce);
    const long long eb = p.bf16 ? 2 : 4;
    p.k = (const char*)p.k + done * p.k_token * eb;
    p.v = (const char*)p.v + done * p.v_token * eb;
    p.slots = (const char*)p.slots + done * (p.slots64 ? 8 : 4);
    while ((p.N >> p.per_shift) > wave && (1 << p.per_shift) < kWriteTokens) ++p.per_shift;
    const int per = 1 << p.per_shift;
    const dim3 grid((unsigned)((p.N + per - 1) / per));
    const size_t smem = 5 * per * sizeof(int);
    p.per_k_unit = 1.f / p.c.k_unit;
    p.per_v_unit = 1.f / p.c.v_unit;
    auto run = [&](auto kern) { launch_with_pdl(kern, grid, dim3(kWriteThreads), smem, s, true, p); };
    if (p.c.D == 128) p.bf16 ? run(kv_cache_write_kernel<__nv_bfloat16, 128>) : run(kv_cache_write_kernel<float, 128>);
    else p.bf16 ? run(kv_cache_write_kernel<__nv_bfloat16, 64>) : run(kv_cache_write_kernel<float, 64>);
  }
}

void launch_cache_read(const CacheReadParams& p, cudaStream_t s) {
  const int tokens = kReadTokens * 256 / (p.c.D / 16);
  const dim3 grid((unsigned)((p.N + tokens - 1) / tokens), 2 * p.c.heads);
  auto run = [&](auto kern) { launch_with_pdl(kern, grid, dim3(256), 0, s, true, p); };
  if (p.c.D == 128) p.bf16 ? run(kv_cache_read_kernel<__nv_bfloat16, 128>) : run(kv_cache_read_kernel<float, 128>);
  else p.bf16 ? run(kv_cache_read_kernel<__nv_bfloat16, 64>) : run(kv_cache_read_kernel<float, 64>);
}

}  // namespace raiccl
