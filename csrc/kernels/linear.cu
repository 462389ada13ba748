// out = act(x w^T + bias) + residual: a dense product with its epilogue, from
// one row to a whole batch, any sizes.
#include <stdexcept>

#include "serving.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

// 64 x 64 output tile per CTA, 16 K at a time through shared memory, 4 x 4
// outputs per thread, 32-bit sums (SwiGLU: a gate and an up sum of each).
constexpr int kTile = 64, kTileK = 16;

template <typename T, bool GLU>
__global__ void __launch_bounds__(256) linear_tile_kernel(LinearParams p) {
  __shared__ float xs[kTileK][kTile + 4], ws[GLU ? 2 : 1][kTileK][kTile + 4];
  const long long m0 = (long long)blockIdx.x * kTile;
  const int n0 = blockIdx.y * kTile;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[GLU ? 2 : 1][4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += kTileK) {
    for (int i = threadIdx.x; i < kTile * kTileK; i += 256) {
      const int r = i / kTileK, c = i % kTileK;
      const bool in = k0 + c < p.K;
      xs[c][r] = in && m0 + r < p.M ? as_float(((const T*)p.x)[(m0 + r) * p.x_stride + k0 + c]) : 0.f;
#pragma unroll
      for (int g = 0; g < (GLU ? 2 : 1); ++g)
        ws[g][c][r] = in && n0 + r < p.N ? as_float(((const T*)p.w)[(long long)(g * p.N + n0 + r) * p.w_stride + k0 + c]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kTileK; ++c)
#pragma unroll
      for (int g = 0; g < (GLU ? 2 : 1); ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[g][i][j] = fmaf(xs[c][ty * 4 + i], ws[g][c][tx * 4 + j], acc[g][i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long m = m0 + ty * 4 + i;
      const int n = n0 + tx * 4 + j;
      if (m >= p.M || n >= p.N) continue;
      float v = acc[0][i][j] + (p.bias ? p.bias[n] : 0.f);
      if constexpr (GLU) v = serving_swiglu(v, acc[1][i][j] + (p.bias ? p.bias[p.N + n] : 0.f));
      else v = serving_act(v, p.act);
      if (p.residual) v += load_elem(p.residual, m * p.res_stride + n, p.res_bf16);
      store_elem(p.out, m * p.out_stride + n, v, p.out_bf16);
    }
}

void launch_linear(const LinearParams& p, cudaStream_t s) {
  const dim3 grid((unsigned)((p.M + kTile - 1) / kTile), (unsigned)((p.N + kTile - 1) / kTile));
  const bool glu = p.act == (int)Act::kSwiGLU;
  if (p.bf16) {
    if (glu) linear_tile_kernel<__nv_bfloat16, true><<<grid, 256, 0, s>>>(p);
    else linear_tile_kernel<__nv_bfloat16, false><<<grid, 256, 0, s>>>(p);
  } else {
    if (glu) linear_tile_kernel<float, true><<<grid, 256, 0, s>>>(p);
    else linear_tile_kernel<float, false><<<grid, 256, 0, s>>>(p);
  }
}

}  // namespace raiccl
