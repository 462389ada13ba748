// Dense product for few rows, and for problems with few tiles: every weight is
// read once for up to 256 rows of x, and the K axis is split over a cluster
// when the tiles alone would leave SMs idle.
//
// The weights are the 128-row operand of tcgen05.mma (SwiGLU: 64 gate and 64 up
// rows), the rows of x its N side, so that one row costs 16 columns and not a
// 128-row tile.  One TMA thread, one MMA thread; the accumulator (fp32, TMEM)
// goes to shared memory as [row of x][weight row], the CTAs of a cluster, each
// with its share of K, meet at the cluster barrier, and each CTA finishes a
// part of the tile: it adds the cluster's sums in rank order (distributed
// shared memory, no global scratch and no counters, the same result every
// time), then bias, activation and residual, and rounds once.
//
// fp32: eight warps split the staged tiles into two tf32 parts of 11 bits (see
// split_tf32), in place and into a short ring for the weights' low parts;
// h h' + h l' + l h' is the product to 2^-21.
#pragma once

#include "serving.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

constexpr int kRowsTile = 128 * 128;       // bytes of a weight tile: 128 rows of 128 bytes
constexpr int kRowsMaxStages = 12;
constexpr int kRowsLow = 3;                // weight tiles of low parts in flight
constexpr int kRowsKernelId = 610;
constexpr unsigned long long kServingWaitNs = 2000000000ull;

struct LinearRowsParams {
  LinearParams l;
  int Mp;        // rows of x of a tile: a multiple of 16, at most 256 (fp32: 128)
  int stages;
};

template <bool FP32>
struct LinearRows {
  static constexpr int PARTS = FP32 ? 2 : 1;
  static constexpr int BK = FP32 ? 32 : 64;          // elements of 128 bytes
  static constexpr int THREADS = FP32 ? 448 : 192;
  static __host__ __device__ int stage_bytes(int Mp) { return kRowsTile + PARTS * Mp * 128; }
  static __host__ __device__ int low_bytes() { return FP32 ? kRowsLow * kRowsTile : 0; }
};

template <bool FP32, bool GLU>
__global__ void __launch_bounds__(LinearRows<FP32>::THREADS)
linear_rows_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, LinearRowsParams p,
                   DeviceStatus* status) {
  using C = LinearRows<FP32>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[kRowsMaxStages], empty[kRowsMaxStages], parted[kRowsMaxStages], done;
  __shared__ uint32_t tmem_slot;
  const LinearParams& l = p.l;
  const int SB = C::stage_bytes(p.Mp), S = p.stages;
  uint8_t* const low = smem + S * SB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  constexpr int W = GLU ? 64 : 128;                     // output columns of a tile
  const int n0 = (int)(blockIdx.x / ranks) * W;
  const long long m0 = (long long)blockIdx.y * p.Mp;
  const int cols0 = C::PARTS * p.Mp;
  const int cols = cols0 <= 32 ? 32 : cols0 <= 64 ? 64 : cols0 <= 128 ? 128 : 256;
  const int KB = (l.K + C::BK - 1) / C::BK;
  const int kb0 = (int)((long long)KB * rank / ranks), kb1 = (int)((long long)KB * (rank + 1) / ranks);

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); mbar_init(&parted[i], 4); }
    mbar_init(&done, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tx); tma_prefetch_desc(&tw);
  }
  if (warp == 1) { tmem_alloc(&tmem_slot, cols); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (elect_one_sync()) {
      for (int i = 0; kb0 + i < kb1; ++i) {
        const int s = i % S;
        if (!mbar_wait_bounded(&empty[s], ((i / S) & 1) ^ 1u, status, kRowsKernelId, kServingWaitNs)) break;
        uint8_t* w = smem + s * SB;
        const int k = (kb0 + i) * C::BK;
        mbar_arrive_expect_tx(&full[s], kRowsTile + p.Mp * 128);
        if constexpr (GLU) {
          tma_load_2d(w, &tw, &full[s], k, n0);
          tma_load_2d(w + kRowsTile / 2, &tw, &full[s], k, l.N + n0);
        } else {
          tma_load_2d(w, &tw, &full[s], k, n0);
        }
        tma_load_2d(w + kRowsTile, &tx, &full[s], k, (int)m0);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    if (elect_one_sync()) {
      uint64_t* ready = FP32 ? parted : full;
      for (int i = 0; kb0 + i < kb1; ++i) {
        const int s = i % S;
        if (!mbar_wait_bounded(&ready[s], (i / S) & 1, status, kRowsKernelId, kServingWaitNs)) break;
        tc_fence_after_sync();
        const uint32_t w = smem_u32(smem + s * SB), x = w + kRowsTile, wl = smem_u32(low) + i % kRowsLow * kRowsTile;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint64_t a = umma_desc_k_sw128(w + k * 32), b = umma_desc_k_sw128(x + k * 32);
          const uint32_t more = (i | k) ? 1u : 0u;
          if constexpr (FP32) {
            umma_tf32(tmem, a, b, umma_idesc(2u, 128, 2 * p.Mp), more);
            umma_tf32(tmem, umma_desc_k_sw128(wl + k * 32), b, umma_idesc(2u, 128, p.Mp), 1u);
          } else {
            umma_f16(tmem, a, b, umma_idesc(1u, 128, p.Mp), more);
          }
        }
        umma_commit(&empty[s]);
      }
      umma_commit(&done);
    }
  } else if (FP32 && warp >= 6) {
    // ---------------------------------------------------------------- tf32 parts: two groups take stages in turn
    const int tid = (threadIdx.x - 192) & 127, g = (threadIdx.x - 192) >> 7;
    for (int i = g; kb0 + i < kb1; i += 2) {
      const int s = i % S;
      if (!mbar_wait_bounded(&full[s], (i / S) & 1, status, kRowsKernelId, kServingWaitNs)) break;
      if (i >= kRowsLow) {  // the products that read this tile of low parts
        const int j = i - kRowsLow;
        if (!mbar_wait_bounded(&empty[j % S], (j / S) & 1, status, kRowsKernelId, kServingWaitNs)) break;
      }
      uint8_t* w = smem + s * SB;
      uint8_t* wl = low + i % kRowsLow * kRowsTile;
      auto part = [&](float4* at, float4* lo_at) {
        const float4 v = *at;
        float4 h, lo;
        split_tf32(v.x, h.x, lo.x);
        split_tf32(v.y, h.y, lo.y);
        split_tf32(v.z, h.z, lo.z);
        split_tf32(v.w, h.w, lo.w);
        *at = h;
        *lo_at = lo;
      };
#pragma unroll 4
      for (int o = tid * 16; o < kRowsTile; o += 128 * 16) part((float4*)(w + o), (float4*)(wl + o));
      uint8_t* x = w + kRowsTile;
      for (int o = tid * 16; o < p.Mp * 128; o += 128 * 16) part((float4*)(x + o), (float4*)(x + p.Mp * 128 + o));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&parted[s]);
    }
  }
  __syncwarp();
  // -------------------------------------------------------------------- the CTA's sums to shared memory
  float* const sums = (float*)smem;   // [Mp][128], over the stages
  const bool ok = mbar_wait_bounded(&done, 0, status, kRowsKernelId, kServingWaitNs);
  const int rows = (int)(l.M - m0 < p.Mp ? l.M - m0 : p.Mp);
  __syncthreads();                    // every role has left the stages
  if (warp >= 2 && warp < 6) {
    const int q = warp & 3;
    tc_fence_after_sync();
    const uint32_t base = tmem + ((uint32_t)(q * 32) << 16);
    for (int c = 0; c < rows; c += 16) {
      uint32_t v[16];
      tmem_ld16(base + c, v);
      if constexpr (FP32) {
        uint32_t u[16];
        tmem_ld16(base + p.Mp + c, u);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(u[j]));
      } else {
        tmem_ld_wait();
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[(c + j) * 128 + q * 32 + lane] = kb0 < kb1 ? __uint_as_float(v[j]) : 0.f;
    }
    tc_fence_before_sync();
  }
  if (ranks > 1) cluster_sync_all();
  else __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, cols);
  // -------------------------------------------------------------------- add the cluster's sums, finish
  if (ok) {
    const uint32_t own = smem_u32(sums);
    auto total = [&](int at) {
      if (ranks == 1) return sums[at];
      float v = 0.f;
#pragma unroll 4
      for (uint32_t r = 0; r < ranks; ++r) {
        float a;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(a) : "r"(mapa_shared(own + at * 4, r)));
        v += a;
      }
      return v;
    };
    for (int i = (int)rank * C::THREADS + threadIdx.x; i < rows * W; i += (int)ranks * C::THREADS) {
      const int m = i / W, c = i % W, n = n0 + c;
      if (n >= l.N) continue;
      float v = total(m * 128 + c);
      if (l.bias) v += __ldg(l.bias + n);
      if constexpr (GLU) {
        float up = total(m * 128 + 64 + c);
        if (l.bias) up += __ldg(l.bias + l.N + n);
        v = serving_swiglu(v, up);
      } else {
        v = serving_act(v, l.act);
      }
      if (l.residual) v += load_elem(l.residual, (m0 + m) * l.res_stride + n, l.res_bf16);
      store_elem(l.out, (m0 + m) * l.out_stride + n, v, l.out_bf16);
    }
  }
  if (ranks > 1) cluster_sync_all();   // nobody leaves while its sums may be read
}

}  // namespace raiccl
