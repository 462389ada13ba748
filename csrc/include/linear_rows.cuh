// Dense product for few rows, and for problems with few tiles: every weight is
// read once for up to 64 rows of x, and the K axis is split over a cluster
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
// The tensor core cuts what does not fit its accumulator instead of rounding,
// which drifts toward zero with the length of the chain (2e-6 of the result for
// each 1024 of K).  For fp32 results the sums therefore go to registers after
// every 128 of K (bf16 operands: 512) and are added there, rounded to nearest,
// while the next piece runs into the other of two accumulators.  bf16 results
// are rounded to 2^-8, where the drift of a whole K does not show.
//
// fp32: two tf32 parts of 11 bits each, made by eight warps from the staged
// tiles: x in place and beside it (split_tf32), of the weights, whose upper 19
// bits the tensor core reads, only the rests (rest_tf32), into a short ring;
// h h' + h l' + l h' is the product to 2^-20.
#pragma once

#include "serving.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

constexpr int kRowsTile = 128 * 128;       // bytes of a weight tile: 128 rows of 128 bytes
constexpr int kRowsPack = 2;               // 128-byte steps of K in a stage: a stage costs its waits and its commit, 0.15 us
constexpr int kRowsMaxStages = 12;
constexpr int kRowsKernelId = 610;
constexpr unsigned long long kServingWaitNs = 2000000000ull;

struct LinearRowsParams {
  LinearParams l;
  int Mp;        // rows of x of a tile: a multiple of 16, at most 64 (fp32: 16, 32 or 64)
  int stages;
  int vec_out;   // four outputs of a row may be written at once
  int low;       // fp32: stages whose low parts of the weights are kept, at most as many as stages
};

template <bool FP32>
struct LinearRows {
  static constexpr int PARTS = FP32 ? 2 : 1;
  static constexpr int BK = FP32 ? 32 : 64;          // elements of 128 bytes
  static constexpr int THREADS = FP32 ? 448 : 192;
  static constexpr int CHAIN = FP32 ? 2 : 4;         // stages into one accumulator, where sums are kept in registers
  static __host__ __device__ int stage_bytes(int Mp) { return kRowsPack * (kRowsTile + PARTS * Mp * 128); }   // weight tiles, then x tiles (h rows, l rows)
};

// MP: rows of x of a tile where the sums are kept in registers (fp32 operands, fp32 results), else 0.
template <bool FP32, bool GLU, int MP>
__global__ void __launch_bounds__(LinearRows<FP32>::THREADS)
linear_rows_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, LinearRowsParams p,
                   DeviceStatus* status) {
  using C = LinearRows<FP32>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[kRowsMaxStages], empty[kRowsMaxStages], parted[kRowsMaxStages], done, acc_full[2], acc_empty[2];
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
  const int cols0 = MP > 0 ? 2 * C::PARTS * MP : p.Mp;  // two accumulators where chains are cut; fp32: of [h | l] columns
  const int cols = cols0 <= 32 ? 32 : cols0 <= 64 ? 64 : cols0 <= 128 ? 128 : cols0 <= 256 ? 256 : 512;
  const int KB = (l.K + C::BK - 1) / C::BK;
  const int kb0 = (int)((long long)KB * rank / ranks), kb1 = (int)((long long)KB * (rank + 1) / ranks);

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); mbar_init(&parted[i], 4); }
    mbar_init(&done, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 4); }
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
  [[maybe_unused]] float acc[MP > 0 ? MP : 1];
  [[maybe_unused]] bool added = true;
#pragma unroll
  for (int i = 0; i < MP; ++i) acc[i] = 0.f;

  const int steps = kb1 - kb0;
  const int count = (steps + kRowsPack - 1) / kRowsPack;   // stages' worth
  int stage = 0;
  uint32_t phase = 0;
  auto advance = [&]() { if (++stage == S) { stage = 0; phase ^= 1u; } };

  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (elect_one_sync()) {
      int i = 0;
      for (; i < count; ++i, advance()) {
        if (!serving_wait(&empty[stage], phase ^ 1u, status, kRowsKernelId, kServingWaitNs)) break;
        uint8_t* w = smem + stage * SB;
        uint8_t* x = w + kRowsPack * kRowsTile;
        const int n = steps - i * kRowsPack < kRowsPack ? steps - i * kRowsPack : kRowsPack;
        int k = (kb0 + i * kRowsPack) * C::BK;
        mbar_arrive_expect_tx(&full[stage], n * (kRowsTile + p.Mp * 128));
        for (int j = 0; j < n; ++j, k += C::BK, w += kRowsTile, x += C::PARTS * p.Mp * 128) {
          tma_load_2d(w, &tw, &full[stage], k, n0);
          if constexpr (GLU) tma_load_2d(w + kRowsTile / 2, &tw, &full[stage], k, l.N + n0);
          tma_load_2d(x, &tx, &full[stage], k, (int)m0);
        }
      }
      await_loads(full, S, stage, phase, i, status, kRowsKernelId, kServingWaitNs);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    if (elect_one_sync()) {
      uint64_t* ready = FP32 ? parted : full;
      const uint64_t row = umma_desc_k_sw128(0);
      const uint32_t id = umma_idesc(FP32 ? 2u : 1u, 128, (uint32_t)(C::PARTS * p.Mp)), idl = umma_idesc(2u, 128, (uint32_t)p.Mp);
      int lo = 0;
      for (int i = 0; i < count; ++i, advance()) {
        if (MP > 0 && i % C::CHAIN == 0) {
          const int c = i / C::CHAIN;
          if (!serving_wait(&acc_empty[c & 1], ((c >> 1) & 1) ^ 1u, status, kRowsKernelId, kServingWaitNs)) break;
        }
        if (!serving_wait(&ready[stage], phase, status, kRowsKernelId, kServingWaitNs)) break;
        tc_fence_after_sync();
        const uint32_t d = tmem + (MP > 0 ? (i / C::CHAIN & 1) * C::PARTS * MP : 0);
        const uint32_t w = smem_u32(smem + stage * SB);
        uint64_t da = desc_at(row, w), dx = desc_at(row, w + kRowsPack * kRowsTile), dl = desc_at(row, smem_u32(low) + lo * kRowsPack * kRowsTile);
        const int n = steps - i * kRowsPack < kRowsPack ? steps - i * kRowsPack : kRowsPack;
        for (int j = 0; j < n; ++j, da += kRowsTile / 16, dx += C::PARTS * p.Mp * 8, dl += kRowsTile / 16) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t more = ((MP > 0 ? i % C::CHAIN : i) | j | k) ? 1u : 0u;
            if constexpr (FP32) {
              umma_tf32(d, da + 2 * k, dx + 2 * k, id, more);
              umma_tf32(d + p.Mp, dl + 2 * k, dx + 2 * k, idl, 1u);   // with the other small products
            } else {
              umma_f16(d, da + 2 * k, dx + 2 * k, id, more);
            }
          }
        }
        umma_commit(&empty[stage]);
        if (MP > 0 && (i % C::CHAIN == C::CHAIN - 1 || i + 1 == count)) umma_commit(&acc_full[i / C::CHAIN & 1]);
        if (++lo == p.low) lo = 0;
      }
      umma_commit(&done);
    }
  } else if (MP > 0 && warp < 6) {
    // ---------------------------------------------------------------- a chain's sums into registers
    const uint32_t base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    for (int c = 0; c * C::CHAIN < count; ++c) {
      added = mbar_wait_warp(&acc_full[c & 1], (c >> 1) & 1, status, kRowsKernelId, kServingWaitNs);
      if (!added) break;
      tc_fence_after_sync();
#pragma unroll
      for (int i = 0; i < MP; i += 16) {
        uint32_t v[16], u[16];
        tmem_ld16(base + (c & 1) * C::PARTS * MP + i, v);
        if constexpr (FP32) tmem_ld16(base + (c & 1) * 2 * MP + MP + i, u);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i + j] += FP32 ? __uint_as_float(v[j]) + __uint_as_float(u[j]) : __uint_as_float(v[j]);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[c & 1]);
    }
  } else if (FP32 && warp >= 6) {
    // ---------------------------------------------------------------- tf32 parts: two groups take stages in turn
    const int tid = (threadIdx.x - 192) & 127, g = (threadIdx.x - 192) >> 7;
    int lo = 0, old = 0;          // slot of low parts; stage of the products that read it last, and their phase
    uint32_t old_phase = 0;
    for (int i = 0; i < count; ++i, advance()) {
      const int slot = lo;
      if (++lo == p.low) lo = 0;
      const int was = old;
      const uint32_t was_phase = old_phase;
      if (i >= p.low && ++old == S) { old = 0; old_phase ^= 1u; }
      if ((i & 1) != g) continue;
      if (!mbar_wait_warp(&full[stage], phase, status, kRowsKernelId, kServingWaitNs)) break;
      if (i >= p.low && !mbar_wait_warp(&empty[was], was_phase, status, kRowsKernelId, kServingWaitNs)) break;
      uint8_t* w = smem + stage * SB;
      uint8_t* x = w + kRowsPack * kRowsTile;
      const int n = steps - i * kRowsPack < kRowsPack ? steps - i * kRowsPack : kRowsPack;
      split_tile<false>(w, low + slot * kRowsPack * kRowsTile, tid, n * kRowsTile);
      for (int j = 0; j < n; ++j, x += C::PARTS * p.Mp * 128) split_tile<true>(x, x + p.Mp * 128, tid, p.Mp * 128);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&parted[stage]);
    }
  }
  __syncwarp();
  // -------------------------------------------------------------------- the CTA's sums to shared memory
  float* const sums = (float*)smem;   // [Mp][128], over the stages
  const bool ok = mbar_wait_warp(&done, 0, status, kRowsKernelId, kServingWaitNs) && added;
  const int rows = (int)(l.M - m0 < p.Mp ? l.M - m0 : p.Mp);
  __syncthreads();                    // every role has left the stages
  __syncwarp();
  if (warp >= 2 && warp < 6) {
    const int q = warp & 3;
    if constexpr (MP > 0) {
#pragma unroll
      for (int i = 0; i < MP; ++i)
        if (i < rows) sums[i * 128 + q * 32 + lane] = acc[i];
    } else {
      tc_fence_after_sync();
      const uint32_t base = tmem + ((uint32_t)(q * 32) << 16);
      for (int c = 0; c < rows; c += 16) {
        uint32_t v[16];
        tmem_ld16(base + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) sums[(c + j) * 128 + q * 32 + lane] = kb0 < kb1 ? __uint_as_float(v[j]) : 0.f;
      }
      tc_fence_before_sync();
    }
  }
  __syncwarp();
  if (ranks > 1) cluster_sync_all();
  else __syncthreads();
  __syncwarp();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, cols);
  // -------------------------------------------------------------------- add the cluster's sums, finish
  if (ok) {
    const uint32_t own = smem_u32(sums);
    // four columns at a time, added over the cluster in rank order
    auto total = [&](int at, float (&v)[4]) {
      if (ranks == 1) {
        const float4 a = *(const float4*)(sums + at);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        return;
      }
      v[0] = v[1] = v[2] = v[3] = 0.f;
#pragma unroll 4
      for (uint32_t r = 0; r < ranks; ++r) {
        float a, b, c, d;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(a), "=f"(b), "=f"(c), "=f"(d) : "r"(mapa_shared(own + at * 4, r)));
        v[0] += a; v[1] += b; v[2] += c; v[3] += d;
      }
    };
#pragma unroll 1
    for (int i = ((int)rank * C::THREADS + threadIdx.x) * 4; i < rows * W; i += (int)ranks * C::THREADS * 4) {
      const int m = i / W, c = i % W, n = n0 + c;
      if (n >= l.N) continue;
      float v[4], up[4];
      total(m * 128 + c, v);
      if constexpr (GLU) total(m * 128 + 64 + c, up);
      const bool whole = n + 4 <= l.N;
      if (l.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (whole || n + j < l.N) {
            v[j] += __ldg(l.bias + n + j);
            if constexpr (GLU) up[j] += __ldg(l.bias + l.N + n + j);
          }
      }
      if constexpr (GLU) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = serving_swiglu(v[j], up[j]);
      } else {
        serving_act_each(v, l.act);
      }
      if (l.residual) {
        const long long at = (m0 + m) * l.res_stride + n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (whole || n + j < l.N) v[j] += load_elem(l.residual, at + j, l.res_bf16);
      }
      const long long at = (m0 + m) * l.out_stride + n;
      if (whole && p.vec_out) {
        if (l.out_bf16) {
          const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
          *(uint2*)((__nv_bfloat16*)l.out + at) = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
        } else {
          *(float4*)((float*)l.out + at) = make_float4(v[0], v[1], v[2], v[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (whole || n + j < l.N) store_elem(l.out, at + j, v[j], l.out_bf16);
      }
    }
  }
  __syncwarp();
  if (ranks > 1) cluster_sync_all();   // nobody leaves while its sums may be read
}

}  // namespace raiccl
