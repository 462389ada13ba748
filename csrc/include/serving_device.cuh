// Device helpers shared by the serving operators.
#pragma once

#include <cuda_bf16.h>

#include <cstdint>

#include "sm100_ptx.cuh"
#include "serving.h"
#include "types.h"

namespace raiccl {

// One try with a time hint: the thread may be put aside for so long instead of
// polling, which takes issue and shared-memory slots from the warps at work.
__device__ __forceinline__ bool mbar_try_wait_hint(uint64_t* bar, uint32_t parity, uint32_t ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P1;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, P1;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(ns)
      : "memory");
  return ok != 0;
}

// A wait of one thread.  When `limit_ns` have passed it records that and gives
// up.  Unlike mbar_wait_bounded it does not look at what others have recorded:
// the record of a device stays until it is read, and the calls behind a failed
// one must not end early for it.
__device__ __forceinline__ bool serving_wait(uint64_t* bar, uint32_t parity, DeviceStatus* st, int kernel_id, uint64_t limit_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t start = globaltimer_ns();
  uint32_t polls = 0;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++polls & 63u) == 0 && globaltimer_ns() - start > limit_ns) {
      record_status(st, kTimeoutPipeline, kernel_id, (long long)parity, (long long)limit_ns);
      return false;
    }
  }
}

// The same wait of a whole warp.  The lanes may leave the loop apart, and the aligned instructions that follow (tcgen05.ld, cluster
// barriers) need the warp in one piece; all lanes return the same.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, DeviceStatus* st, int kernel_id, uint64_t limit_ns) {
  bool ok = mbar_try_wait_hint(bar, parity, 20000u);
  if (!ok) {
    const uint64_t start = globaltimer_ns();
    uint32_t polls = 0;
#pragma unroll 1
    while (!(ok = mbar_try_wait_hint(bar, parity, 20000u))) {
      if ((++polls & 63u) == 0 && globaltimer_ns() - start > limit_ns) {
        record_status(st, kTimeoutPipeline, kernel_id, (long long)parity, (long long)limit_ns);
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Lets so much time pass.
__device__ __forceinline__ void serving_hold(uint64_t ns) {
  const uint64_t start = globaltimer_ns();
#pragma unroll 1
  for (uint32_t i = 0; i < (1u << 20) && globaltimer_ns() - start < ns; ++i) __nanosleep(1000u);
}

// A loading thread's last step, whether its loop ended or gave up: the copies
// that it has issued land before its CTA leaves and another one gets the shared
// memory.  `filled` stages so far, the next one would be (stage, phase).  In a
// call that went well all of them have landed or are about to.
__device__ __forceinline__ void await_loads(uint64_t* full, int S, int stage, uint32_t phase, int filled, DeviceStatus* st, int kernel_id,
                                            uint64_t limit_ns) {
  for (int i = filled < S ? filled : S; i > 0; --i) {
    fill_before(S, stage, phase);
    if (!serving_wait(&full[stage], phase, st, kernel_id, limit_ns)) return;
  }
}

// Shared-memory descriptors by addition: the fields of umma_desc_k_sw128 (or
// umma_desc_k_narrow) without an address, plus the address in 16-byte units.
// A product issues four to twelve of them for each 128 bytes of K.
__device__ __forceinline__ uint64_t desc_at(uint64_t fields, uint32_t smem_addr) { return fields + (smem_addr >> 4); }

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// The elements of sixteen bytes as fp32.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& v, float (&f)[16 / sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) f[i] = as_float(((const T*)&v)[i]);
}

// One element of a tensor of either type, by element offset.
__device__ __forceinline__ float load_elem(const void* p, long long i, int bf16) {
  return bf16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : ((const float*)p)[i];
}

// The result's one rounding: every sum before it is kept in 32 bits.
__device__ __forceinline__ void store_elem(void* p, long long i, float v, int bf16) {
  if (bf16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  else ((float*)p)[i] = v;
}

// Activations in 32 bits, by the approximate exponential and quotient.  Their
// errors are small against the argument, not against a result near zero: the
// exponential is off by 2 + 1.2 |z| units in the last place, and GELU's tail by
// an absolute 0.75e-7 |z| (at -4 that is 5e-4 of the value, about what a sum 1 +
// erf in 32 bits loses there too).  An epilogue has 64 to 128 of them per
// thread, and with expf, erfcf and exact quotients they took as long as the
// products: 4096 x 1024 x 4096 fp32 with GELU 212 us, without 159.  ReLU keeps a
// NaN.
__device__ __forceinline__ float serving_sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

// z Phi(z), with the normal distribution's tail from the rational-exponential
// form 7.1.26 of Abramowitz and Stegun, Handbook of Mathematical Functions
// (absolute error of erf at most 1.5e-7, so 0.75e-7 |z| here).
__device__ __forceinline__ float serving_gelu(float z) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __fdividef(1.f, fmaf(0.3275911f, x, 1.f));
  float q = fmaf(1.061405429f, t, -1.453152027f);
  q = fmaf(q, t, 1.421413741f);
  q = fmaf(q, t, -0.284496736f);
  q = fmaf(q, t, 0.254829592f);
  const float tail = 0.5f * q * t * __expf(-x * x);   // Phi(-|z|)
  return z * (z < 0.f ? tail : 1.f - tail);
}

__device__ __forceinline__ float serving_act(float z, int act) {
  switch ((Act)act) {
    case Act::kRelu: return z < 0.f ? 0.f : z;
    case Act::kGelu: return serving_gelu(z);
    case Act::kSilu: return z * serving_sigmoid(z);
    default: return z;
  }
}

// Several at a time, one loop to an activation: a launch fetches only the code of its own.
template <int N>
__device__ __forceinline__ void serving_act_each(float (&v)[N], int act) {
  if (act == (int)Act::kRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = serving_act(v[i], (int)Act::kRelu);
  } else if (act == (int)Act::kGelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = serving_act(v[i], (int)Act::kGelu);
  } else if (act == (int)Act::kSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = serving_act(v[i], (int)Act::kSilu);
  }
}

__device__ __forceinline__ float serving_swiglu(float gate, float up) { return gate * serving_sigmoid(gate) * up; }

// fp32 as two tf32 numbers: hi is v rounded to 11 significant bits, lo what is
// left (at most 12 bits, of which the tensor core reads 11: 2^-23 of v is lost).
// Rounding up from the last 2^-12 of the range would give an infinity, so v is
// cut there (lo then has 13 bits: 2^-21 of v is lost).  An infinity has no low
// part.  No branches: with one this took twice as long.
__device__ __forceinline__ void split_tf32(float v, float& hi, float& lo) {
  uint32_t h;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(h) : "f"(v));
  hi = fabsf(__uint_as_float(h)) == INFINITY ? __uint_as_float(__float_as_uint(v) & 0xffffe000u) : __uint_as_float(h);
  lo = fabsf(v) == INFINITY ? 0.f : v - hi;
}

// fp32 as two bf16 numbers: hi is v rounded to 8 significant bits, or cut where
// rounding would give an infinity, lo what is left, rounded (2^-16 of v is lost
// at most).
__device__ __forceinline__ void split_bf16(float v, __nv_bfloat16& hi, __nv_bfloat16& lo) {
  const float r = __bfloat162float(__float2bfloat16_rn(v));
  const float h = fabsf(r) == INFINITY ? __uint_as_float(__float_as_uint(v) & 0xffff0000u) : r;
  hi = __float2bfloat16_rn(h);
  lo = __float2bfloat16_rn(fabsf(v) == INFINITY ? 0.f : v - h);
}

// What the tensor core does not read of an fp32 number, which it takes by its
// upper 19 bits: v less those, 13 bits rounded to 11 (2^-22 of v is lost at most).
// Numbers behind the last one of 22 bits, infinities too, count as that one, so
// that rounding never carries the two parts into an infinity.
__device__ __forceinline__ float rest_tf32(float v) {
  float c;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(c) : "f"(v), "f"(__uint_as_float(0x7f7ffffcu)));
  uint32_t l;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(l) : "f"(c - __uint_as_float(__float_as_uint(c) & 0xffffe000u)));
  return __uint_as_float(l);
}

// Sixteen bytes of a tile: BOTH, in place into high parts, the low parts to
// `low`; else only the rests to `low`, and the tile serves as the high parts.
template <bool BOTH>
__device__ __forceinline__ void split_store(uint8_t* at, uint8_t* low, const float4& v) {
  float4 h, l;
  if constexpr (BOTH) {
    split_tf32(v.x, h.x, l.x);
    split_tf32(v.y, h.y, l.y);
    split_tf32(v.z, h.z, l.z);
    split_tf32(v.w, h.w, l.w);
    *(float4*)at = h;
  } else {
    l = make_float4(rest_tf32(v.x), rest_tf32(v.y), rest_tf32(v.z), rest_tf32(v.w));
  }
  *(float4*)low = l;
}

// `bytes` of a tile (a multiple of 16) by the 128 threads of a group: eight
// loads in flight, without a test while whole rounds of 16 KB are left.
template <bool BOTH>
__device__ __forceinline__ void split_tile(uint8_t* at, uint8_t* low, int tid, int bytes) {
  constexpr int STEP = 128 * 16;
  at += tid * 16;
  low += tid * 16;
  for (; bytes >= 8 * STEP; bytes -= 8 * STEP, at += 8 * STEP, low += 8 * STEP) {
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *(const float4*)(at + i * STEP);
#pragma unroll
    for (int i = 0; i < 8; ++i) split_store<BOTH>(at + i * STEP, low + i * STEP, v[i]);
  }
  for (bytes -= tid * 16; bytes > 0; bytes -= STEP, at += STEP, low += STEP) split_store<BOTH>(at, low, *(const float4*)at);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace raiccl
