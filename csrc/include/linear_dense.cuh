// Dense product for many rows: persistent CTA pairs (tcgen05 cta_group::2), a
// 256 x BN tile of sums per pair, two accumulators in TMEM so that one tile's
// epilogue runs under the next tile's products.
//
// Each CTA of a pair stages its 128 rows of x and half of the tile's BN weight
// rows; the pair's first CTA issues M = 256 products that read both.  SwiGLU:
// the first CTA's half are gate rows and the second's the up rows of the same
// outputs, so a thread finds both in its accumulator row and the weights need
// no other order than gate rows, then up rows.
//
// The tensor core cuts what does not fit its accumulator, which drifts with the
// length of the chain (2e-6 of the result for each 1024 of K), so for fp32
// results K is taken in chains, each into an accumulator of its own; the
// epilogue warps add the chains in registers, rounded to nearest, while the
// next one runs.  Chains of 1024 of K for bf16 operands (4096 x 8192 x 4096 to
// fp32: 269 us, all of K in one 244 and 1.6e-5 off), of 128 for fp32 ones (4096
// x 1024 x 4096: 199 us and 0.35e-6 off; 256 at a time 188 and 0.64e-6, twice
// that behind SwiGLU).
//
// fp32: x and w come as two tf32 parts each (linear_split_kernel), h + l.  The
// small products l h' and h l' have an accumulator for the whole tile.  A stage
// holds both parts of both operands for the three products: two thirds of the
// bytes that three walks over K would fetch.
//
// Tiles go by groups of eight row tiles, so that the pairs at work share rows
// of x and of w in L2.  Every wait is bounded.
#pragma once

#include "serving.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

constexpr int kDenseThreads = 320;         // TMA, MMA, eight epilogue warps
constexpr int kDenseKernelId = 620;
constexpr int kDenseGroup = 8;
constexpr unsigned long long kDenseWaitNs = 2000000000ull;

struct LinearDenseParams {
  LinearParams l;
  int mt, nt;      // tiles
  int vec_out, vec_res;   // rows may be read and written 16 bytes at a time
};

template <int BN, bool FP32>
struct LinearDense {
  static constexpr int BK = FP32 ? 32 : 64;
  static constexpr int HALF = BN / 2;
  static constexpr int PARTS = FP32 ? 2 : 1;
  static constexpr int X_BYTES = 128 * 128, W_BYTES = HALF * 128;
  static constexpr int STAGE = PARTS * (X_BYTES + W_BYTES);   // x parts, then w parts
  static constexpr int STAGES_FIT = 216 * 1024 / STAGE;
  static constexpr int STAGES = STAGES_FIT > 8 ? 8 : STAGES_FIT;
  static constexpr int SMEM = 1024 + STAGES * STAGE;
  static constexpr int CHAIN = FP32 ? 4 : 16;   // 128-byte steps of K of a chain
  static constexpr int COLS = FP32 ? 4 * BN : 2 * BN;   // fp32: two for chains, two for small products
};

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const void* desc, uint32_t bar_cluster_addr, int32_t x, int32_t y,
                                                 int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(desc), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ void dense_tile(const LinearDenseParams& p, int t, int& mb, int& nb) {
  const int per = kDenseGroup * p.nt, g = t / per, first = g * kDenseGroup;
  const int rows = p.mt - first < kDenseGroup ? p.mt - first : kDenseGroup;
  const int local = t - g * per;
  mb = first + local % rows;
  nb = local / rows;
}

// residual[m, n .. n + 16) as it lies, where it may be read 16 bytes at a time
__device__ __forceinline__ void dense_residual16(const LinearDenseParams& p, long long m, int n, uint4 (&r)[4]) {
  const LinearParams& l = p.l;
  if (l.residual == nullptr || !p.vec_res || m >= l.M || n + 16 > l.N) return;
  const long long at = m * l.res_stride + n;
  if (l.res_bf16) {
    const uint4* s = (const uint4*)((const __nv_bfloat16*)l.residual + at);
    r[0] = s[0]; r[1] = s[1];
  } else {
    const uint4* s = (const uint4*)((const float*)l.residual + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = s[i];
  }
}

// Sixteen consecutive outputs of one row: residual (`ahead` is what
// dense_residual16 read), rounding, store.
__device__ __forceinline__ void dense_store16(const LinearDenseParams& p, long long m, int n, const uint4 (&ahead)[4], float (&v)[16]) {
  const LinearParams& l = p.l;
  const bool whole = n + 16 <= l.N;
  if (l.residual) {
    const long long at = m * l.res_stride + n;
    if (whole && p.vec_res) {
      if (l.res_bf16) {
        const uint4 a = ahead[0], b = ahead[1];
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[2 * i] += __uint_as_float(w[i] << 16);
          v[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 a = ahead[i];
          v[4 * i] += __uint_as_float(a.x); v[4 * i + 1] += __uint_as_float(a.y);
          v[4 * i + 2] += __uint_as_float(a.z); v[4 * i + 3] += __uint_as_float(a.w);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (n + i < l.N) v[i] += load_elem(l.residual, at + i, l.res_bf16);
    }
  }
  const long long at = m * l.out_stride + n;
  if (whole && p.vec_out) {
    if (l.out_bf16) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *(const uint32_t*)&h;
      }
      uint4* o = (uint4*)((__nv_bfloat16*)l.out + at);
      o[0] = make_uint4(w[0], w[1], w[2], w[3]);
      o[1] = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
      float4* o = (float4*)((float*)l.out + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (n + i < l.N) store_elem(l.out, at + i, v[i], l.out_bf16);
  }
}

// bias[n .. n + 32 NB), a lane has every 32nd of them; zeros behind the last.
template <int NB>
__device__ __forceinline__ void dense_bias(const float* bias, int n, int N, float (&b)[NB]) {
  const int at = n + (int)(threadIdx.x & 31);
#pragma unroll
  for (int i = 0; i < NB; ++i) b[i] = bias != nullptr && at + 32 * i < N ? __ldg(bias + at + 32 * i) : 0.f;
}

// b[c .. c + 16) of them in every lane, added to v; c a multiple of 16.
template <int NB>
__device__ __forceinline__ void dense_add_bias16(const float (&b)[NB], int c, float (&v)[16]) {
  float mine = b[0];
#pragma unroll
  for (int i = 1; i < NB; ++i) mine = (c >> 5) == i ? b[i] : mine;
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] += __shfl_sync(0xffffffffu, mine, (c & 16) + i);
}

// CHAINED: the sums leave the tensor core after every chain, else after the whole of K.
template <int BN, bool FP32, bool GLU, bool CHAINED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kDenseThreads, 1)
linear_dense_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, LinearDenseParams p,
                    DeviceStatus* status) {
  using C = LinearDense<BN, FP32>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[C::STAGES], empty[C::STAGES], acc_full[2], acc_empty[2], low_full[2], low_empty[2], drained;
  __shared__ uint32_t tmem_slot;
  const LinearParams& l = p.l;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 16);
      mbar_init(&low_full[i], 1); mbar_init(&low_empty[i], 16);
    }
    mbar_init(&drained, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tx); tma_prefetch_desc(&tw);
  }
  if (warp == 1) { tmem_alloc_pair(&tmem_slot, C::COLS); tmem_relinquish_pair(); }
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  constexpr int W = GLU ? BN / 2 : BN;      // outputs of a tile
  const int KB = (l.K + C::BK - 1) / C::BK;
  const int chain = CHAINED ? C::CHAIN : KB;             // 128-byte steps of K of an accumulator
  const int tiles = p.mt * p.nt;

  if (warp == 0) {
    // ---------------------------------------------------------------- loads, both CTAs
    if (elect_one_sync()) {
      int stage = 0, filled = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += npairs) {
        int mb, nb;
        dense_tile(p, t, mb, nb);
        const int xrow = mb * 256 + (int)rank * 128;
        const int wrow = GLU ? nb * W + (int)rank * l.N : nb * W + (int)rank * C::HALF;
        for (int kb = 0; kb < KB; ++kb) {
          if (!(ok = serving_wait(&empty[stage], phase ^ 1u, status, kDenseKernelId, kDenseWaitNs))) break;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * C::STAGE);
          const uint32_t lead = mapa_shared(smem_u32(&full[stage]), 0);
          uint8_t* s = smem + stage * C::STAGE;
#pragma unroll
          for (int part = 0; part < C::PARTS; ++part) {
            tma_load_3d_pair(s + part * C::X_BYTES, &tx, lead, kb * C::BK, xrow, part);
            tma_load_3d_pair(s + C::PARTS * C::X_BYTES + part * C::W_BYTES, &tw, lead, kb * C::BK, wrow, part);
          }
          ++filled;
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      // Both CTAs' copies count on the first one's barriers, and the pair leaves together.  Where one thread gave up before
      // the other, the second CTA may have filled a stage more than the first knows of: that one gets a millisecond.
      if (rank == 0) await_loads(full, C::STAGES, stage, phase, filled, status, kDenseKernelId, kDenseWaitNs);
      if (!ok) serving_hold(1000000ull);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products, first CTA
    if (rank == 0 && elect_one_sync()) {
      int stage = 0, iter = 0;
      uint32_t phase = 0;
      bool ok = true;
      constexpr uint32_t idesc = umma_idesc(FP32 ? 2u : 1u, 256, BN);
      const uint64_t row = umma_desc_k_sw128(0);
      int nth = 0;
      for (int t = pair; ok && t < tiles; t += npairs, ++nth) {
        const int lb = nth & 1;
        const uint32_t dl = tmem + (2 + lb) * BN;
        if (FP32 && !(ok = serving_wait(&low_empty[lb], ((nth >> 1) & 1) ^ 1u, status, kDenseKernelId, kDenseWaitNs))) break;
        for (int k0 = 0; ok && k0 < KB; k0 += chain, ++iter) {
          const int steps = k0 + chain < KB ? chain : KB - k0;
          const int b = iter & 1;
          if (!(ok = serving_wait(&acc_empty[b], ((iter >> 1) & 1) ^ 1u, status, kDenseKernelId, kDenseWaitNs))) break;
          tc_fence_after_sync();
          const uint32_t d = tmem + b * BN;
          for (int kb = 0; kb < steps; ++kb) {
            if (!(ok = serving_wait(&full[stage], phase, status, kDenseKernelId, kDenseWaitNs))) break;
            tc_fence_after_sync();
            const uint64_t dx = desc_at(row, smem_u32(smem + stage * C::STAGE)), dw = dx + C::PARTS * C::X_BYTES / 16;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (FP32) {
                umma_tf32_pair(dl, dx + C::X_BYTES / 16 + 2 * k, dw + 2 * k, idesc, (k0 | kb | k) ? 1u : 0u);
                umma_tf32_pair(dl, dx + 2 * k, dw + C::W_BYTES / 16 + 2 * k, idesc, 1u);
                umma_tf32_pair(d, dx + 2 * k, dw + 2 * k, idesc, (kb | k) ? 1u : 0u);
              } else {
                umma_f16_pair(d, dx + 2 * k, dw + 2 * k, idesc, (kb | k) ? 1u : 0u);
              }
            }
            const uint32_t e = smem_u32(&empty[stage]);
            umma_commit_pair(mapa_shared(e, 0));
            umma_commit_pair(mapa_shared(e, 1));
            if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
          }
          if (!ok) break;
          const uint32_t f = smem_u32(&acc_full[b]);
          umma_commit_pair(mapa_shared(f, 0));
          umma_commit_pair(mapa_shared(f, 1));
        }
        if (FP32 && ok) {
          const uint32_t f = smem_u32(&low_full[lb]);
          umma_commit_pair(mapa_shared(f, 0));
          umma_commit_pair(mapa_shared(f, 1));
        }
      }
      umma_commit_pair(mapa_shared(smem_u32(&drained), 0));
      serving_wait(&drained, 0, status, kDenseKernelId, kDenseWaitNs);
    }
  } else {
    // ---------------------------------------------------------------- epilogue, both CTAs
    const int q = warp & 3, side = (warp - 2) >> 2;   // TMEM lanes 32 q ..; half of the tile's columns
    constexpr int OUT = W / 2;                        // outputs of a thread
    int iter = 0;
    [[maybe_unused]] int nth = 0;
    bool ok = true;
    // Biases and the first pieces (16 columns) of the residual are read before the sums are waited for, the others as many
    // pieces ahead.
    constexpr int AHEAD = CHAINED ? (BN == 256 ? 1 : 2) : 4;   // by the registers that the sums leave
    constexpr int NB = (OUT + 31) / 32;
    float bias[NB], up[NB];
    uint4 ahead[AHEAD][4];
    auto begin = [&](long long m, int n) {
      dense_bias(l.bias, n, l.N, bias);
      if constexpr (GLU) dense_bias(l.bias ? l.bias + l.N : nullptr, n, l.N, up);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (16 * j < OUT) dense_residual16(p, m, n + 16 * j, ahead[j]);
    };
    // columns c .. c + 16 of the thread's OUT, which begin at n0
    auto finish = [&](long long m, int n0, int c, float (&v)[16], float (&vu)[16]) {
      if (l.bias) {
        dense_add_bias16(bias, c, v);
        if constexpr (GLU) dense_add_bias16(up, c, vu);
      }
      if constexpr (GLU) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = serving_swiglu(v[i], vu[i]);
      } else {
        serving_act_each(v, l.act);
      }
      if (m < l.M && n0 + c < l.N) dense_store16(p, m, n0 + c, ahead[0], v);
#pragma unroll
      for (int j = 1; j < AHEAD; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) ahead[j - 1][i] = ahead[j][i];
      if (c + 16 * AHEAD < OUT) dense_residual16(p, m, n0 + c + 16 * AHEAD, ahead[AHEAD - 1]);
      __syncwarp();
    };
    for (int t = pair; ok && t < tiles; t += npairs) {
      int mb, nb;
      dense_tile(p, t, mb, nb);
      const long long m = (long long)mb * 256 + rank * 128 + q * 32 + lane;
      const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
      const int c0 = side * OUT, n0 = nb * W + c0;
      if constexpr (CHAINED) {
        float sum[OUT], sum_up[GLU ? OUT : 16];
#pragma unroll
        for (int i = 0; i < OUT; ++i) sum[i] = 0.f;
#pragma unroll
        for (int i = 0; i < (GLU ? OUT : 16); ++i) sum_up[i] = 0.f;
        auto add = [&](uint32_t base) {
#pragma unroll
          for (int c = 0; c < OUT; c += 16) {
            uint32_t r[16];
            tmem_ld16(base + c, r);
            if constexpr (GLU) {
              uint32_t u[16];
              tmem_ld16(base + C::HALF + c, u);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) sum_up[c + i] += __uint_as_float(u[i]);
            } else {
              tmem_ld_wait();
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[c + i] += __uint_as_float(r[i]);
          }
          tc_fence_before_sync();
          __syncwarp();
        };
        for (int k0 = 0; k0 < KB; k0 += chain, ++iter) {
          const int b = iter & 1;
          if (!(ok = mbar_wait_warp(&acc_full[b], (iter >> 1) & 1, status, kDenseKernelId, kDenseWaitNs))) break;
          tc_fence_after_sync();
          add(lanes + b * BN + c0);
          if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[b]), 0));
        }
        if (!ok) break;
        begin(m, n0);
        if constexpr (FP32) {
          if (!(ok = mbar_wait_warp(&low_full[nth & 1], (nth >> 1) & 1, status, kDenseKernelId, kDenseWaitNs))) break;
          tc_fence_after_sync();
          add(lanes + (2 + (nth & 1)) * BN + c0);
          if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&low_empty[nth & 1]), 0));
          ++nth;
        }
#pragma unroll
        for (int c = 0; c < OUT; c += 16) {
          float z[16], zu[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) { z[i] = sum[c + i]; zu[i] = sum_up[GLU ? c + i : i]; }
          finish(m, n0, c, z, zu);
        }
      } else {
        const int b = iter & 1;
        begin(m, n0);
        if (!(ok = mbar_wait_warp(&acc_full[b], (iter >> 1) & 1, status, kDenseKernelId, kDenseWaitNs))) break;
        ++iter;
        tc_fence_after_sync();
        const uint32_t base = lanes + b * BN + c0;
#pragma unroll 1   // code that a launch's only tile runs once is fetched while it waits: unrolled four times, 2.4 us more
        for (int c = 0; c < OUT; c += 16) {
          if (n0 + c >= l.N) break;
          uint32_t r[16], u[16];
          tmem_ld16(base + c, r);
          if constexpr (GLU) tmem_ld16(base + C::HALF + c, u);
          tmem_ld_wait();
          float z[16], zu[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) { z[i] = __uint_as_float(r[i]); zu[i] = GLU ? __uint_as_float(u[i]) : 0.f; }
          finish(m, n0, c, z, zu);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[b]), 0));
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync_all();   // both CTAs have finished before the pair frees its memory
  __syncwarp();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc_pair(tmem, C::COLS);
}

// fp32 rows as two tf32 parts, [2][rows, packed]: what linear_dense_kernel
// reads.  Both operands in one launch: one read and two writes of each, at the
// rate of memory (64 + 64 MB: 53 us; 5.4 TB/s).
struct SplitOperand {
  const float* src;
  long long stride;
  float* dst;
  long long rows;
  int vec;   // rows may be read 16 bytes at a time
};

__device__ __forceinline__ void split_operand(const SplitOperand& o, int packed, int K) {
  float* low = o.dst + o.rows * packed;
  if (o.vec) {   // four at a time over all rows
    const long long per = K / 4, n = o.rows * per;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
      const long long r = i / per, k = (i - r * per) * 4;
      const float4 v = *(const float4*)(o.src + r * o.stride + k);
      float4 h, l;
      split_tf32(v.x, h.x, l.x);
      split_tf32(v.y, h.y, l.y);
      split_tf32(v.z, h.z, l.z);
      split_tf32(v.w, h.w, l.w);
      *(float4*)(o.dst + r * packed + k) = h;
      *(float4*)(low + r * packed + k) = l;
    }
  } else {
    for (long long r = blockIdx.x; r < o.rows; r += gridDim.x)
      for (int k = threadIdx.x; k < K; k += 256) split_tf32(o.src[r * o.stride + k], o.dst[r * packed + k], low[r * packed + k]);
  }
}

__global__ void __launch_bounds__(256) linear_split_kernel(SplitOperand x, SplitOperand w, int packed, int K) {
  griddep_wait();
  griddep_launch_dependents();
  split_operand(x, packed, K);
  split_operand(w, packed, K);
}

}  // namespace raiccl
