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
// Both kernels only move memory: eight numbers to a thread, 16 bytes in and 4
// out for bf16.
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "attention.h"
#include "serving.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

constexpr int kWriteThreads = 512;
constexpr int kWriteTokens = 2048;         // of a CTA at most

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

// Row (of D numbers) of a head's token in the cache.
__device__ __forceinline__ long long cache_row(const CacheView& c, int slot, int head) {
  const int page = slot >> c.page_shift, at = slot & ((1 << c.page_shift) - 1);
  return ((((long long)page * c.heads + head) << c.page_shift) + at);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int vec, float (&x)[8]) {
  if (vec) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += W) {
      float f[W];
      unpack16<T>(*(const uint4*)(p + i), f);
#pragma unroll
      for (int j = 0; j < W; ++j) x[i + j] = f[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = as_float(p[i]);
  }
}

// Two lanes have a group of sixteen: its scale (both get it) and this lane's eight codes.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], float unit, float per_unit, uint32_t& scale) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(x[i]));
  top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1)) * per_unit;
  scale = __nv_cvt_float_to_fp8(__fdiv_rn(top, 6.f), __NV_SATFINITE, __NV_E4M3);
  const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)scale, __NV_E4M3)));
  const float r = s > 0.f ? __frcp_rn(s) * per_unit : 0.f, back = s * unit;
  // Behind 448 * 6 everything saturates; there numbers are cut, so that no infinities meet below.
  const float most = 8192.f * unit;
  const bool cut = top > 8192.f;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float q[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float v = cut ? fminf(fmaxf(x[i + j], -most), most) : x[i + j];
      // x / s: the product by the rounded reciprocal, and one correction by its remainder, which is exact in an fma
      // (P. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990).
      q[j] = v * r;
      q[j] = fmaf(fmaf(-back, q[j], v), r, q[j]);
    }
    codes |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(q[0], q[1]), __NV_E2M1, cudaRoundNearest) << (4 * i);
  }
  return codes;
}

// A CTA has `per` consecutive tokens (a power of two).  Where several tokens of
// a call name one slot, the last of them is kept: the CTA enters its tokens'
// slots into a hash table, the highest token of each, and looks up all later
// tokens' slots in it.
//
// A row of a head is D / 8 lanes; rows go by value or key, head and token, the
// token fastest, so that no index needs a division.  Four rows to a thread are
// loaded before the first is worked on.
template <typename T>
__global__ void __launch_bounds__(kWriteThreads) kv_cache_write_kernel(CacheWriteParams p) {
  extern __shared__ int table[];      // [per] slots, [size] keys, [size] last tokens
  const CacheView& c = p.c;
  griddep_wait();
  griddep_launch_dependents();
  const int per = 1 << p.per_shift, size = 2 * per;
  int *slot_of = table, *key = table + per, *last = key + size;
  const long long first = (long long)blockIdx.x << p.per_shift;
  const int n = (int)(p.N - first < per ? p.N - first : per);
  for (int i = threadIdx.x; i < size; i += kWriteThreads) { key[i] = -1; last[i] = -1; }
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
  }
  __syncthreads();
  const long long bound = (long long)c.pages << c.page_shift;
#pragma unroll 4
  for (long long i = first + n + threadIdx.x; i < p.N; i += kWriteThreads) {
    const long long wide = p.slots64 ? ((const long long*)p.slots)[i] : (long long)((const int*)p.slots)[i];
    if (wide < 0 || wide >= bound) continue;
    const int s = (int)wide;
    int e = at(s), k;
    while ((k = key[e]) != -1 && k != s) e = (e + 1) & (size - 1);
    if (k == s) last[e] = 1 << 30;    // a later CTA has it
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
  const int lane_shift = c.D == 128 ? 4 : 3, l = threadIdx.x & ((1 << lane_shift) - 1);
  const int step = kWriteThreads >> lane_shift, rows = 2 * c.heads << p.per_shift;
  constexpr int U = 4;
  for (int r0 = 0; r0 < rows; r0 += U * step) {
    float x[U][8];
    int slot[U], hv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * step + (int)(threadIdx.x >> lane_shift), t = r & (per - 1);
      hv[u] = r >> p.per_shift;
      slot[u] = r < rows ? slot_of[t] : -1;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
      if (slot[u] >= 0) {
        const T* src = hv[u] < c.heads ? (const T*)p.k + (first + t) * p.k_token + hv[u] * p.k_head
                                       : (const T*)p.v + (first + t) * p.v_token + (hv[u] - c.heads) * p.v_head;
        load8(src + 8 * l, p.vec, x[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u * step >= rows) break;              // the same for all threads
      const bool value = hv[u] >= c.heads;
      const float unit = value ? c.v_unit : c.k_unit;
      uint32_t scale;
      const uint32_t codes = quantise8(x[u], unit, 1.f / unit, scale);
      uint32_t word = scale << (8 * ((l >> 1) & 3));   // four groups' scales, eight lanes
      word |= __shfl_xor_sync(0xffffffffu, word, 2);
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      if (slot[u] >= 0) {
        const long long at_row = cache_row(c, slot[u], value ? hv[u] - c.heads : hv[u]);
        *(uint32_t*)((value ? c.v_codes : c.k_codes) + at_row * (c.D / 2) + 4 * l) = codes;
        if ((l & 7) == 0) *(uint32_t*)((value ? c.v_scales : c.k_scales) + at_row * (c.D / 16) + l / 2) = word;
      }
    }
  }
}

// Eight numbers to a thread, of one head of four tokens in turn (all loads before
// the first store).  A code times its scale has at most 6 bits: nothing is
// rounded in bf16 either.
constexpr int kReadTokens = 4;

template <typename T>
__global__ void __launch_bounds__(256) kv_cache_read_kernel(CacheReadParams p) {
  const CacheView& c = p.c;
  griddep_wait();
  griddep_launch_dependents();
  const int lane_shift = c.D == 128 ? 4 : 3, l = threadIdx.x & ((1 << lane_shift) - 1), step = 256 >> lane_shift;
  const bool value = blockIdx.y >= c.heads;
  const int h = value ? blockIdx.y - c.heads : blockIdx.y;
  const uint8_t* const codes_of = (value ? c.v_codes : c.k_codes) + 4 * l;
  const uint8_t* const scales_of = (value ? c.v_scales : c.k_scales) + (l >> 1);
  const float unit = value ? c.v_unit : c.k_unit;
  const long long first = (long long)blockIdx.x * (kReadTokens * step) + (threadIdx.x >> lane_shift);
  uint32_t codes[kReadTokens], scale[kReadTokens];
#pragma unroll
  for (int u = 0; u < kReadTokens; ++u) {
    const long long t = first + u * step;
    const int slot = t < p.N ? cache_slot(p.slots, p.slots64, t, c, p.status, kCacheReadKernelId) : -1;
    codes[u] = scale[u] = 0;
    if (slot >= 0) {
      const long long row = cache_row(c, slot, h);
      codes[u] = __ldg((const uint32_t*)(codes_of + row * (c.D / 2)));
      scale[u] = __ldg(scales_of + row * (c.D / 16));
    }
  }
#pragma unroll
  for (int u = 0; u < kReadTokens; ++u) {
    const long long t = first + u * step;
    if (t >= p.N) return;
    float x[8];
    const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)scale[u], __NV_E4M3))) * unit;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(codes[u] >> (8 * j)), __NV_E2M1)));
      x[2 * j] = f.x * s;
      x[2 * j + 1] = f.y * s;
    }
    T* dst = value ? (T*)p.v + t * p.v_token + h * p.v_head + 8 * l : (T*)p.k + t * p.k_token + h * p.k_head + 8 * l;
    if (p.vec) {
      if constexpr (sizeof(T) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
          w[j] = *(const uint32_t*)&b;
        }
        *(uint4*)dst = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        ((float4*)dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
        ((float4*)dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) store_elem(dst, j, x[j], sizeof(T) == 2);
    }
  }
}

// Tokens of a CTA: about three CTAs to an SM.
void launch_cache_write(const CacheWriteParams& params, cudaStream_t s) {
  CacheWriteParams p = params;
  const long long wave = 3ll * serving_sm_count();
  while ((p.N >> p.per_shift) > wave && (1 << p.per_shift) < kWriteTokens) ++p.per_shift;
  const int per = 1 << p.per_shift;
  const dim3 grid((unsigned)((p.N + per - 1) / per));
  const size_t smem = 5 * per * sizeof(int);
  if (p.bf16) launch_with_pdl(kv_cache_write_kernel<__nv_bfloat16>, grid, dim3(kWriteThreads), smem, s, true, p);
  else launch_with_pdl(kv_cache_write_kernel<float>, grid, dim3(kWriteThreads), smem, s, true, p);
}

void launch_cache_read(const CacheReadParams& p, cudaStream_t s) {
  const int tokens = kReadTokens * 256 / (p.c.D / 8);
  const dim3 grid((unsigned)((p.N + tokens - 1) / tokens), 2 * p.c.heads);
  if (p.bf16) launch_with_pdl(kv_cache_read_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, true, p);
  else launch_with_pdl(kv_cache_read_kernel<float>, grid, dim3(256), 0, s, true, p);
}

}  // namespace raiccl
