// Dense product for very few rows of x, on CUDA cores: weights go from memory
// straight to registers, so a call costs its loads and one launch.  fp32 needs
// no splitting here, and rows that do not start on 16 bytes no copy.
//
// A CTA has four outputs (SwiGLU: their gate and up rows) and up to eight rows
// of x; its eight warps share K.  Each lane adds products of 16 bytes at a time
// in 32 bits, a butterfly adds the lanes, shared memory the warps in order.
// Four outputs for a CTA: fewer read x more often, more leave SMs empty at the
// smallest widths.  Loads bound it: one row of 4096 x 4096 bf16 takes 9.1 us
// (33.6 MB from L2, 3.7 TB/s), of 16384 x 4096 fp32 43 us (268 MB, 6.2 TB/s),
// 7 rows of 2048 x 33 fp32 5.3 us, nearly all of it the launch.
#pragma once

#include "serving.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

constexpr int kVectorThreads = 256;
constexpr int kVectorWarps = kVectorThreads / 32;
constexpr int kVectorOut = 4;

// NT rows of x; VEC: x and w rows start on 16 bytes and hold whole 16-byte words.
template <typename T, bool VEC, bool GLU, int NT>
__global__ void __launch_bounds__(kVectorThreads) linear_vector_kernel(LinearParams p) {
  constexpr int R = GLU ? 2 * kVectorOut : kVectorOut;
  constexpr int V = VEC ? 16 / sizeof(T) : 1;
  __shared__ float part[kVectorWarps][R][NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * kVectorOut;
  const long long m0 = (long long)blockIdx.y * NT;
  const int words = (p.K + V - 1) / V;
  const int i1 = (int)((long long)words * (warp + 1) / kVectorWarps);
  griddep_wait();
  griddep_launch_dependents();
  const T* w[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int n = n0 + r % kVectorOut;
    w[r] = (const T*)p.w + ((long long)(r / kVectorOut) * p.N + (n < p.N ? n : p.N - 1)) * p.w_stride;
  }
  const T* x[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = (const T*)p.x + (m0 + t < p.M ? m0 + t : p.M - 1) * p.x_stride;
  float acc[R][NT] = {};
#pragma unroll(R * NT <= 16 ? 4 : 2)
  for (int i = (int)((long long)words * warp / kVectorWarps) + lane; i < i1; i += 32) {
    if constexpr (VEC) {
      uint4 wv[R];
#pragma unroll
      for (int r = 0; r < R; ++r) wv[r] = __ldg((const uint4*)w[r] + i);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float fx[V];
        unpack16<T>(__ldg((const uint4*)x[t] + i), fx);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float fw[V], s = 0.f;
          unpack16<T>(wv[r], fw);
#pragma unroll
          for (int v = 0; v < V; ++v) s = fmaf(fw[v], fx[v], s);
          acc[r][t] += s;
        }
      }
    } else {
      float fw[R];
#pragma unroll
      for (int r = 0; r < R; ++r) fw[r] = as_float(w[r][i]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float fx = as_float(x[t][i]);
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][t] = fmaf(fw[r], fx, acc[r][t]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float v = warp_sum(acc[r][t]);
      if (lane == 0) part[warp][r][t] = v;
    }
  __syncthreads();
  const int c = threadIdx.x % kVectorOut, t = threadIdx.x / kVectorOut, n = n0 + c;
  const long long m = m0 + t;
  if (t >= NT || m >= p.M || n >= p.N) return;
  float v = 0.f, up = 0.f;
#pragma unroll
  for (int i = 0; i < kVectorWarps; ++i) {
    v += part[i][c][t];
    if constexpr (GLU) up += part[i][kVectorOut + c][t];
  }
  if (p.bias) v += __ldg(p.bias + n);
  if constexpr (GLU) {
    if (p.bias) up += __ldg(p.bias + p.N + n);
    v = serving_swiglu(v, up);
  } else {
    v = serving_act(v, p.act);
  }
  if (p.residual) v += load_elem(p.residual, m * p.res_stride + n, p.res_bf16);
  store_elem(p.out, m * p.out_stride + n, v, p.out_bf16);
}

}  // namespace raiccl
