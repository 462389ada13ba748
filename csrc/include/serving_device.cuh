// Device helpers shared by the serving operators.
#pragma once

#include <cuda_bf16.h>

#include <cstdint>

#include "types.h"

namespace raiccl {

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// One element of a tensor of either type, by element offset.
__device__ __forceinline__ float load_elem(const void* p, long long i, int bf16) {
  return bf16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : ((const float*)p)[i];
}

// The result's one rounding: every sum before it is kept in 32 bits.
__device__ __forceinline__ void store_elem(void* p, long long i, float v, int bf16) {
  if (bf16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  else ((float*)p)[i] = v;
}

// Activations in 32 bits.  ReLU keeps a NaN; GELU by the complementary error
// function, which loses nothing where 1 + erf would cancel.
__device__ __forceinline__ float serving_act(float z, int act) {
  switch ((Act)act) {
    case Act::kRelu: return z < 0.f ? 0.f : z;
    case Act::kGelu: return 0.5f * z * erfcf(z * -0.70710678118654752f);
    case Act::kSilu: return z / (1.f + expf(-z));
    default: return z;
  }
}

__device__ __forceinline__ float serving_swiglu(float gate, float up) { return gate / (1.f + expf(-gate)) * up; }

// fp32 as two tf32 numbers of 11 significant bits, rounded to nearest; what
// would round to infinity is cut instead, and an infinity has no low part.
__device__ __forceinline__ void split_tf32(float v, float& hi, float& lo) {
  const uint32_t b = __float_as_uint(v);
  uint32_t h = (b + 0x1000u) & ~0x1fffu;
  if ((h & 0x7f800000u) == 0x7f800000u) h = b & ~0x1fffu;
  hi = __uint_as_float(h);
  const float l = v == hi ? 0.f : v - hi;
  lo = l != l ? l : __uint_as_float((__float_as_uint(l) + 0x1000u) & ~0x1fffu);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace raiccl
