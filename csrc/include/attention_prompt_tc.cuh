// Attention over whole prompts on the tensor cores, bf16.
//
// A CTA has two tiles, A and B, of 128 rows each; a row is a token and a query
// head of one key head's group, so that a group shares every key that is read.
// It walks over the keys in tiles of 128 and keeps the running maximum m and sum
// l of a softmax:
//
//   S = Q K^T,  P = exp2(c S - m),  O = O + P V,  l = l + sum P
//
// with O and l multiplied by exp2 of the change where m has to follow the maximum.
//
// One warp loads (TMA), one issues the products (tcgen05.mma, 128 x 128 sums in
// TMEM), and a warpgroup to each tile does the softmax, one row to a thread: no
// shuffles.  P goes back into TMEM as bf16 over S, as the operand of the second
// product.  While tile A's softmax runs, the tensor core has B's products, and
// the other way round; S of the next step is issued behind P V of this one, so
// its arrival tells the softmax that O may be touched too.
//
// TMEM: S (and P) of A and B, O of A and B, 128 columns each.
//
// What bounds it.  16384 tokens, causal, 32 heads of 128 over 8 key heads: 1.82 to
// 2.07 ms, 1.06 to 1.21 PFLOP/s, where cuBLAS sustains 1.36 under the same power
// limit (clocks near 1.45 GHz); heads of 64, where exponentials are as many and
// products half: 1.56 ms.  A step of both tiles takes 3000 clocks, 2048 of
// them products: softmax 1750 (loads 90, the first half of the weights with the
// maxima 1100, the other 600), then the rest of P V and Q K^T behind it.
//
// A CTA that has loaded all of its pair of tiles takes over one that has not
// begun yet (cluster launch control), and loads that while the last two steps and
// the results of the first are worked on: beginnings and ends, about 4 us of every
// pair, are hidden, and the last ones spread over the SMs as they become free.
// Eight chunks of 512 tokens on average, 3.7 pairs to an SM: 161 -> 150 us on one
// box (142 to 164 over all of them; the tensor cores are busy 55 % of it).
//
// Two more warps look through the tiles of values that some row does not see
// whole (attention_prompt.cuh), and clear what lies behind the sequence's end.
#pragma once

#include "attention_prompt.cuh"

namespace raiccl {

constexpr int kPromptThreads = 384;   // two warpgroups of softmax; loads, products, two warps for masked tiles' values
constexpr int kPromptKeys = 128;
constexpr unsigned long long kPromptWaitNs = 2000000000ull;
// Warps that have nothing to do for a pair of tiles wait for all its steps: 1.5 to 2 us for 128 keys, and 20 at most.
constexpr unsigned long long kPromptKeyNs = 160ull;

template <int D>
struct PromptTc {
  static constexpr int HALVES = D / 64;                       // 128-byte swizzled columns of 64 dimensions
  static constexpr int TILE = 128 * D * 2;                    // bytes of 128 rows
  static constexpr int STAGES = 2;                            // of keys, and as many of values
  static constexpr int SMEM = 1024 + (2 + 2 * STAGES) * TILE;
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem], kind::f16: A's rows are lanes, two 16-bit elements to a column.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const void* desc, uint64_t* bar, int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(desc), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Shared-memory descriptor of an operand whose rows (of 128 bytes, swizzled) run
// along the product's sum: 64 columns to a row, the next 64 `apart` bytes on,
// eight rows 1024 bytes on.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr, uint32_t apart) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((apart >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}

__device__ __forceinline__ float prompt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 numbers to an instruction.
__device__ __forceinline__ uint64_t pair_f32(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair_f32(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Asks for a CTA of the grid that has not begun: this one will do its work.  The answer arrives at `at` (16 bytes), and on `bar`.
__device__ __forceinline__ void ask_next_cta(void* at, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(at)),
               "r"(smem_u32(bar))
               : "memory");
}

// The answer: false where no CTA is left.
__device__ __forceinline__ bool next_cta(const void* at, int& x, int& y) {
  uint32_t some, cx, cy;
  asm volatile(
      "{\n\t.reg .b128 answer;\n\t.reg .pred some;\n\t.reg .b32 z, none;\n\t"
      "ld.shared.b128 answer, [%3];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 some, answer;\n\t"
      "selp.u32 %0, 1, 0, some;\n\t"
      "mov.u32 %1, 0;\n\t"
      "mov.u32 %2, 0;\n\t"
      "@some clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, z, none}, answer;\n\t}"
      : "=r"(some), "=r"(cx), "=r"(cy)
      : "r"(smem_u32(at))
      : "memory");
  x = (int)cx;
  y = (int)cy;
  return some != 0;
}

// A pair of tiles: which rows, and how far over the keys.
struct PromptItem {
  PromptSeq s;
  int token0, head, split;       // A's first token, of the sequence; the key head; which share of the keys
  int tiles, steps;              // steps -1: there are no more
  int first_fixed;               // tiles of values from here on, which some row does not see whole, go through two warps first
};

template <int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
prompt_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                 PromptParams p) {
  using C = PromptTc<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* const sq = smem;                                   // tiles A and B
  uint8_t* const sk = smem + 2 * C::TILE;
  uint8_t* const sv = sk + C::STAGES * C::TILE;
  __shared__ uint64_t q_full[2], q_empty[2], k_full[C::STAGES], k_empty[C::STAGES], v_full[C::STAGES], v_empty[C::STAGES],
      v_raw[C::STAGES], v_ready[C::STAGES], s_full[2], p_half[2], p_full[2], o_full[2], item_full[2], item_empty[2], answered, drained;
  __shared__ __align__(16) uint4 answer;
  __shared__ PromptItem items[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int odd[2][3][D], any_odd[2];                    // of both items
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Nothing of this needs what the kernels before wrote.  TMEM has to be taken before the next kernel may start: one that took
  // it first would keep it until this CTA is done.
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); mbar_init(&s_full[i], 1);
      mbar_init(&p_half[i], 4); mbar_init(&p_full[i], 4); mbar_init(&o_full[i], 1);
      mbar_init(&item_full[i], 1); mbar_init(&item_empty[i], 11);     // 8 warps of softmax, the products, two for values
      any_odd[i] = 0;
    }
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); mbar_init(&v_raw[i], 1); mbar_init(&v_ready[i], 2);
    }
    mbar_init(&answered, 1);
    mbar_init(&drained, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tq); tma_prefetch_desc(&tk); tma_prefetch_desc(&tv);
  }
  for (int i = threadIdx.x; i < 2 * 3 * D; i += kPromptThreads) ((int*)odd)[i] = INT_MAX;
  if (warp == 9) { tmem_alloc(&tmem_slot, 512); tmem_relinquish(); }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  griddep_wait();
  griddep_launch_dependents();
  if (blockIdx.x + blockIdx.y == 0 && warp == 11) prompt_record(p);
  const int tokens = 128 / p.group;                           // of a tile

  // Barriers are waited for by what went through them before: items n by turns through two places, all steps of all items by
  // turns through the stages.  168 registers to a thread at launch: the warpgroups of the softmax, which hold a row of S, get
  // 224, the other 56.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 8) {
      // -------------------------------------------------------------- items, and their loads
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return serving_wait(bar, parity, p.status, kPromptKernelId, kPromptWaitNs); };
      int n = 0, asked = 0, x = blockIdx.x, y = blockIdx.y, base = 0;
      uint32_t q_phase = 0, k_phase = 0, raw_phase = 0, full_phase = 0;   // bits: of what comes next
      auto load_q = [&](const PromptItem& it, int t) {
        if (!(ok = wait(&q_empty[t], (q_phase >> t & 1) ^ 1u))) return;
        q_phase ^= 1u << t;
        mbar_arrive_expect_tx(&q_full[t], C::HALVES * tokens * p.group * 128);
        for (int h = 0; h < C::HALVES; ++h)
          tma_load_3d(sq + t * C::TILE + h * 128 * 128, &tq, &q_full[t], 64 * h, it.head * p.group, it.s.q0 + it.token0 + t * tokens);
      };
      auto load = [&](const PromptItem& it, uint8_t* at, const CUtensorMap* map, uint64_t* full, int i) {
        mbar_arrive_expect_tx(full, C::TILE);
        for (int h = 0; h < C::HALVES; ++h)
          tma_load_3d(at + ((base + i) % C::STAGES) * C::TILE + h * 128 * 128, map, full, 64 * h, it.head, it.s.k0 + i * kPromptKeys);
      };
      auto load_k = [&](const PromptItem& it, int i) {
        const int stage = (base + i) % C::STAGES;
        if (!(ok = wait(&k_empty[stage], (((base + i) / C::STAGES) & 1) ^ 1u))) return;
        k_phase ^= 1u << stage;
        load(it, sk, &tk, &k_full[stage], i);
      };
      auto publish = [&](const PromptItem& it) {
        const int at = n & 1;
        if (lane == 0) ok = wait(&item_empty[at], ((n >> 1) & 1) ^ 1u);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        __syncwarp();
        if (!ok) return;
        if (any_odd[at] != 0) {
          for (int i = lane; i < 3 * D; i += 32) ((int*)odd[at])[i] = INT_MAX;
          __syncwarp();
          if (lane == 0) any_odd[at] = 0;
        }
        if (lane == 0) items[at] = it;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_full[at]);
        ++n;
      };
      bool more = true;
      int end = INT_MAX;                                      // no tile is there or behind it
      while (ok && more) {
        PromptItem it;
        int pair;
        const int index = x / p.Hk;
        if (index < end && !prompt_tile(p, index, 2 * tokens, it.s, pair)) end = index;
        if (index < end) {
          it.head = x % p.Hk;
          it.split = y;
          it.token0 = pair * 2 * tokens;
          it.tiles = it.token0 + tokens < it.s.nq ? 2 : 1;
          const int keys = prompt_visible(p, it.s, min(it.token0 + 2 * tokens, it.s.nq) - 1);
          it.steps = prompt_share(p, y, (keys + kPromptKeys - 1) / kPromptKeys, kPromptKeys, it.s);
          it.first_fixed = min(prompt_visible(p, it.s, it.token0), it.s.nk) / kPromptKeys;
          publish(it);
          if (ok && it.steps > 0 && lane == 0) {
            load_q(it, 0);
            if (ok) load_k(it, 0);
            if (ok && it.tiles == 2) load_q(it, 1);
            for (int i = 0; ok && i < it.steps; ++i) {
              const int stage = (base + i) % C::STAGES;
              if (!(ok = wait(&v_empty[stage], (((base + i) / C::STAGES) & 1) ^ 1u))) break;
              (i < it.first_fixed ? full_phase : raw_phase) ^= 1u << stage;
              load(it, sv, &tv, i < it.first_fixed ? &v_full[stage] : &v_raw[stage], i);
              if (i + 1 < it.steps) load_k(it, i + 1);
            }
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          base += max(it.steps, 0);
        }
        // Asked for when the last two steps are to be done yet, not before: a CTA that is done earlier may take it.
        if (ok) {
          if (lane == 0) {
            mbar_arrive_expect_tx(&answered, 16);
            ask_next_cta(&answer, &answered);
            ok = wait(&answered, asked & 1);
            if (ok) more = next_cta(&answer, x, y);
            fence_proxy_async_smem();
          }
          ++asked;
          ok = __shfl_sync(0xffffffffu, ok, 0);
          more = __shfl_sync(0xffffffffu, more, 0);
          x = __shfl_sync(0xffffffffu, x, 0);
          y = __shfl_sync(0xffffffffu, y, 0);
        }
      }
      if (ok) {
        PromptItem none{};
        none.steps = -1;
        publish(none);
      }
      // the copies land before the CTA leaves
      if (lane == 0) {
        for (int i = 0; i < 2; ++i) wait(&q_full[i], (q_phase >> i & 1) ^ 1u);
        for (int i = 0; i < C::STAGES; ++i) {
          wait(&k_full[i], (k_phase >> i & 1) ^ 1u);
          wait(&v_full[i], (full_phase >> i & 1) ^ 1u);
          wait(&v_raw[i], (raw_phase >> i & 1) ^ 1u);
        }
      }
    } else if (warp == 9) {
      // -------------------------------------------------------------- products
      if (elect_one_sync()) {
        constexpr uint32_t iqk = umma_idesc(1u, 128, 128), ipv = umma_idesc(1u, 128, D) | (1u << 16);
        const uint64_t krow = umma_desc_k_sw128(0), vrow = umma_desc_mn_sw128(0, 128 * 128);
        auto wait = [&](uint64_t* bar, uint32_t parity) { return serving_wait(bar, parity, p.status, kPromptKernelId, kPromptWaitNs); };
        int base = 0, base_b = 0;                              // steps before, of A and of B
        uint32_t q_phase = 0, ready_phase = 0, full_phase = 0;
        auto qk = [&](int x, int i) {
          const uint64_t a = desc_at(krow, smem_u32(sq + x * C::TILE)),
                         b = desc_at(krow, smem_u32(sk + ((base + i) % C::STAGES) * C::TILE));
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = (k / 4) * (128 * 128 / 16) + (k % 4) * 2;
            umma_f16(tmem + 128 * x, a + at, b + at, iqk, k > 0);
          }
          umma_commit(&s_full[x]);
        };
        bool ok = true;
        for (int n = 0; ok; ++n) {
          if (!(ok = wait(&item_full[n & 1], (n >> 1) & 1))) break;
          const int tiles = items[n & 1].tiles, steps = items[n & 1].steps, first_fixed = items[n & 1].first_fixed;
          if (steps < 0) break;
          for (int i = -1; ok && i < steps && steps > 0; ++i) {  // P V of step i, then Q K^T of the next
            const int stage = (base + i) % C::STAGES, next = (base + i + 1) % C::STAGES;
            for (int x = 0; ok && x < tiles; ++x) {
              if (i >= 0) {
                if (x == 0) {
                  uint32_t& phase = i < first_fixed ? full_phase : ready_phase;
                  if (!(ok = wait(i < first_fixed ? &v_full[stage] : &v_ready[stage], phase >> stage & 1))) break;
                  phase ^= 1u << stage;
                }
                const uint64_t b = desc_at(vrow, smem_u32(sv + stage * C::TILE));
                for (int h = 0; ok && h < 2; ++h) {            // the first half of P's columns, then the other
                  if (!(ok = wait(h ? &p_full[x] : &p_half[x], ((x ? base_b : base) + i) & 1))) break;
                  tc_fence_after_sync();
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    umma_f16_ts(tmem + 256 + 128 * x, tmem + 128 * x + 32 * h + 8 * k, b + (4 * h + k) * (16 * 128 / 16), ipv,
                                i > 0 || h > 0 || k > 0);
                }
                if (!ok) break;
                if (x + 1 == tiles) umma_commit(&v_empty[stage]);
                if (i + 1 == steps) {
                  umma_commit(&o_full[x]);
                  continue;
                }
              } else {
                if (!(ok = wait(&q_full[x], q_phase >> x & 1))) break;
                q_phase ^= 1u << x;
              }
              if (x == 0 && !(ok = wait(&k_full[next], ((base + i + 1) / C::STAGES) & 1))) break;
              tc_fence_after_sync();
              qk(x, i + 1);
              if (i + 2 == steps) umma_commit(&q_empty[x]);
              if (x + 1 == tiles) umma_commit(&k_empty[next]);
            }
          }
          base += steps;
          if (tiles == 2) base_b += steps;
          mbar_arrive(&item_empty[n & 1]);
        }
        umma_commit(&drained);
        wait(&drained, 0);
      }
    } else {
      // -------------------------------------------------------------- values of tiles that some row does not see whole
      int base = 0;
      uint32_t raw_phase = 0;
      const unsigned long long limit = kPromptWaitNs + p.Nk * kPromptKeyNs;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        if (!(ok = mbar_wait_warp(&item_full[n & 1], (n >> 1) & 1, p.status, kPromptKernelId, limit))) break;
        const int k_end = items[n & 1].s.nk, steps = items[n & 1].steps;
        if (steps < 0) break;
        for (int i = items[n & 1].first_fixed; i < steps; ++i) {
          const int stage = (base + i) % C::STAGES;
          if (!(ok = mbar_wait_warp(&v_raw[stage], raw_phase >> stage & 1, p.status, kPromptKernelId, limit))) break;
          raw_phase ^= 1u << stage;
          uint8_t* const at[1] = {sv + stage * C::TILE};
          const int key0 = i * kPromptKeys;
          prompt_fix_values<D, kPromptKeys, 4>(at, threadIdx.x - 320, key0, k_end - key0, odd[n & 1], &any_odd[n & 1]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_ready[stage]);
        }
        base += steps;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[n & 1]);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax, one row to a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int x = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + 128 * x, to = tmem + lanes + 256 + 128 * x;
    // logits are turned positive multiples of S: a scale that is not positive goes into S itself
    float mult = p.scale * 1.44269504088896341f;
    mult = mult == 0.f ? 1.f : fabsf(mult);
    bool ok = true;
    uint32_t s_phase = 0, o_phase = 0;
    for (int n = 0; ok; ++n) {
      if (!(ok = mbar_wait_warp(&item_full[n & 1], (n >> 1) & 1, p.status, kPromptKernelId, kPromptWaitNs + p.Nk * kPromptKeyNs))) break;
      const int steps = items[n & 1].steps;
      if (steps < 0) break;
      if (x < items[n & 1].tiles) {
        int visible = 0;
        bool mine;
        {
          const PromptSeq s = items[n & 1].s;
          const int token = items[n & 1].token0 + x * tokens + row / p.group;
          mine = row < tokens * p.group && token < s.nq;
          if (mine) visible = min(prompt_visible(p, s, token), s.nk);
        }
        const int all = __reduce_min_sync(0xffffffffu, mine ? visible : INT_MAX);   // keys that the warp's rows all see
        float m = -INFINITY, l = 0.f;
        auto follow = [&](float now, bool sums) {
          const float shrink = m == -INFINITY ? 0.f : prompt_exp2(m - now);
          m = now;
          l *= shrink;
          if (!sums) return;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(to + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
            tmem_st32(to + c, o);
          }
        };
        for (int i = 0; ok && i < steps; ++i) {
          if (!(ok = mbar_wait_warp(&s_full[x], s_phase, p.status, kPromptKernelId, kPromptWaitNs))) break;
          s_phase ^= 1u;
          tc_fence_after_sync();
          if (__any_sync(0xffffffffu, l > kPromptSum)) {
            follow(l > kPromptSum ? m + kPromptLeast : m, true);
            tmem_st_wait();
          }
          uint32_t r[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, r + 32 * c);
          tmem_ld_wait();
          if (!(p.scale > 0.f)) {
            const float turn = p.scale < 0.f ? -1.f : 0.f;

#pragma unroll
            for (int c = 0; c < 128; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * turn);
          }
          const int k0 = i * kPromptKeys;
          if (k0 + kPromptKeys > all) {
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if (k0 + c >= visible) r[c] = __float_as_uint(-INFINITY);
          }
          // The first half of the weights is worked out before it is known whether m has to follow the maximum (attention_prompt.cuh),
          // which is rare, and the product begins with that half.  (A quarter of the exponentials by a polynomial, to spare the
          // special-function unit: no difference, 16384 tokens run into the power limit.)
          uint64_t sum[2];
          uint32_t w[32];
          auto half = [&](int h, float base) {
            const uint64_t mult2 = pair_f32(mult, mult), base2 = pair_f32(base, base);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              float a, b;
              unpair_f32(fma2(pair_f32(__uint_as_float(r[64 * h + 2 * c]), __uint_as_float(r[64 * h + 2 * c + 1])), mult2, base2), a, b);
              a = prompt_exp2(a);
              b = prompt_exp2(b);
              sum[c & 1] = add2(sum[c & 1], pair_f32(a, b));
              w[c] = pack_bf16(a, b);
            }
          };
          auto store = [&](int h) {
            tmem_st32(ts + 32 * h, w);
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(h ? &p_full[x] : &p_half[x]);
          };
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          bool again;
#pragma unroll 1
          do {
            sum[0] = sum[1] = 0;
            half(0, m == -INFINITY ? 0.f : -m);
#pragma unroll
            for (int c = 0; c < 128; c += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(r[c + 2 * e]), __uint_as_float(r[c + 2 * e + 1]));
            const float peak = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * mult;
            const bool grow = peak > m - kPromptNear;
            again = __any_sync(0xffffffffu, grow);   // once: it does not hold for peak + 31, however that is rounded
            if (again) follow(fmaxf(m, peak + (i > 0 ? kPromptHeadAgain : kPromptHeadTc)), i > 0);
          } while (again);
          store(0);
          half(1, m == -INFINITY ? 0.f : -m);
          store(1);
          float s0, s1;
          unpair_f32(add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
        }
        if (ok && steps > 0) {
          ok = mbar_wait_warp(&o_full[x], o_phase, p.status, kPromptKernelId, kPromptWaitNs);
          o_phase ^= 1u;
          tc_fence_after_sync();
        }
        const volatile PromptItem& it = items[n & 1];             // not kept over the steps: S takes the registers
        const int token = it.token0 + x * tokens + row / p.group, hq = it.head * p.group + row % p.group;
        if (l == 0.f && visible > 0 && steps > 0) l = -0.f;
        const float inv = prompt_per_sum(p, l);
        const bool put_back = any_odd[n & 1] != 0;
        const long long at = (long long)(it.s.q0 + token) * p.o_token + (long long)hq * p.o_head;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          if (steps > 0) {
            tmem_ld32(to + c, o);
            tmem_ld_wait();
          }
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = steps > 0 && visible > 0 ? __uint_as_float(o[e]) * inv : 0.f;
          // weights that were rounded up may lift a mean of the largest numbers past them
          constexpr float most = 3.3895313892515355e38f;
          float size = 0.f;
#pragma unroll
          for (int e = 0; e < 32; e += 2) size = max3(size, fabsf(v[e]), fabsf(v[e + 1]));
          if (size > most) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (fabsf(__uint_as_float(o[e])) < INFINITY) v[e] = fminf(fmaxf(v[e], -most), most);
          }
          if (put_back) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = put_back_odd<D>(odd[n & 1], c + e, visible, v[e]);
          }
          if (mine && p.splits > 1) {
            float4* const dst = (float4*)(p.parts + (((long long)it.split * p.Nq + it.s.q0 + token) * p.Hq + hq) * D + c);
#pragma unroll
            for (int e = 0; e < 32; e += 4) dst[e / 4] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          } else if (mine) {
            __nv_bfloat16* const dst = (__nv_bfloat16*)p.out + at + c;
            if (p.o_vec) {
#pragma unroll
              for (int e = 0; e < 32; e += 8)
                *(uint4*)(dst + e) = make_uint4(pack_bf16(v[e], v[e + 1]), pack_bf16(v[e + 2], v[e + 3]), pack_bf16(v[e + 4], v[e + 5]),
                                                pack_bf16(v[e + 6], v[e + 7]));
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) dst[e] = __float2bfloat16_rn(v[e]);
            }
          }
          __syncwarp();
        }
        if (mine && p.splits > 1) p.stats[((long long)it.split * p.Nq + it.s.q0 + token) * p.Hq + hq] = make_float2(m, l);
        else if (mine && p.lse != nullptr) p.lse[(long long)(it.s.q0 + token) * p.Hq + hq] = prompt_lse(m, l, kPromptHeadTc);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[n & 1]);
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace raiccl
