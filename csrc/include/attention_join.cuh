// Joining parts of a softmax: sums of exponentials over parts of the keys, each
// with a maximum of its own.
#pragma once

#include <cuda_runtime.h>

namespace raiccl {

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row of D numbers over a warp: lane i has numbers D / 32 * i and on.
template <int D>
__device__ __forceinline__ void load_lanes(const float* p, float (&v)[D / 32]) {
  const int lane = threadIdx.x & 31;
  if constexpr (D == 128) {
    const float4 x = *(const float4*)(p + 4 * lane);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else {
    const float2 x = *(const float2*)(p + 2 * lane);
    v[0] = x.x; v[1] = x.y;
  }
}

template <int D>
__device__ __forceinline__ void store_lanes(float* p, const float (&v)[D / 32]) {
  const int lane = threadIdx.x & 31;
  if constexpr (D == 128) *(float4*)(p + 4 * lane) = make_float4(v[0], v[1], v[2], v[3]);
  else *(float2*)(p + 2 * lane) = make_float2(v[0], v[1]);
}

// n parts of a row, each with its own maximum and sum of exponentials, joined by a warp in their order.
template <int D, typename Stat, typename Row>
__device__ __forceinline__ void warp_join(int n, Stat stat, Row row, float& top, float& l, float (&v)[D / 32]) {
  const int lane = threadIdx.x & 31;
  top = -INFINITY;
  for (int j = lane; j < n; j += 32) top = fmaxf(top, stat(j).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  l = 0.f;
#pragma unroll
  for (int d = 0; d < D / 32; ++d) v[d] = 0.f;
  for (int j0 = 0; j0 < n; j0 += 32) {
    float f = 0.f, y = 0.f;
    bool some = false;
    if (j0 + lane < n) {
      const float2 st = stat(j0 + lane);
      some = st.x != -INFINITY || st.y != 0.f;
      // no maximum: nothing there, or logits that are all NaN or -inf, whose sum is NaN
      f = st.x == -INFINITY ? (st.y == 0.f ? 0.f : NAN) : exp2_fast(st.x - top);
      y = st.y;
    }
    const uint32_t with = __ballot_sync(0xffffffffu, some);
    const int here = n - j0 < 32 ? n - j0 : 32;
#pragma unroll 4
    for (int j = 0; j < here; ++j) {
      float a[D / 32];
      load_lanes<D>(row(j0 + j), a);
      const float fj = __shfl_sync(0xffffffffu, f, j);
      l = fmaf(__shfl_sync(0xffffffffu, y, j), fj, l);
      if (!(with >> j & 1)) continue;      // a part that is nothing holds anything; one whose factor vanishes may hold a NaN
#pragma unroll
      for (int d = 0; d < D / 32; ++d) v[d] = fmaf(a[d], fj, v[d]);
    }
  }
}

}  // namespace raiccl
