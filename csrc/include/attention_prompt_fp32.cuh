// Attention over whole prompts on the tensor cores, fp32.
//
// Every number is three bf16 parts, x = x0 + x1 + x2 (24 bits, fp32's range), and
// a product the six of their products that fp32 can show: twelve bits below the
// largest the others are lost in its rounding.  (Two f16 parts would take three
// products, but their range is not fp32's; tf32 ones have half the rate and no
// transposed values.)  The parts of q, k and v are written first, by
// prompt_split_kernel, as TMA reads them; those of the weights P by the threads
// that work them out, into TMEM.
//
// One tile of 128 rows to a CTA; KT keys a step, half a row of them to a thread
// of the softmax.  S has two buffers, so that Q K^T of the next step runs while
// the softmax has this one; the softmax waits for P V of the last step before it
// writes P.  Keys and values go through one ring, by their parts.  The tensor core
// cuts what does not fit its sums: the largest product comes last, and P V leaves
// it after every step and is added up in registers (with one sum for all steps
// 2048 keys were 4e-6 off).
//
// What bounds it.  Three sequences of 2049 tokens in all, 16 heads of 64, every key
// seen: 53 to 59 us, 11 of them the splitting, 0.45e-6 off (the formula in 32 bits: 0.68e-6).
// The six products would take 24.  A step takes about 3900 clocks, 3400 of them
// products (P V, with heads of 64, 1850): weights from S to P are 1800 of 8 warps,
// half of them behind the sums of the last step.  A row to a thread: 76 us; values
// in one stage, loaded when the last ones were done: 72 us.  As two tf32 parts on
// mma.sync: 200 us.
//
// Values go through two warps that look for numbers that are not finite
// (attention_prompt.cuh): an infinity times a part of a weight that is negative
// would be NaN.
#pragma once

#include "attention_prompt_tc.cuh"

namespace raiccl {

constexpr int kFp32Threads = 384;   // two warpgroups of softmax; loads, products, two warps for the values

template <int D>
struct PromptFp32 {
  static constexpr int KT = D == 64 ? 128 : 64;               // keys of a step
  static constexpr int HALVES = D / 64;
  static constexpr int Q_PART = 128 * D * 2, KV_PART = KT * D * 2;
  static constexpr int SLOTS = D == 64 ? 10 : 7;              // of one part of a step's keys or values each
  static constexpr int SMEM = 1024 + 3 * Q_PART + SLOTS * KV_PART;
  static constexpr uint32_t P_AT = 2 * KT, O_AT = D == 64 ? 448 : 256;   // columns of TMEM behind the two of S
};

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const void* desc, uint64_t* bar, int32_t x, int32_t y, int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(desc), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Three bf16 parts, each rounded to nearest, but cut where that would give an infinity; an infinity or NaN is its first part.
__device__ __forceinline__ void split3(float v, float (&part)[3]) {
  const float r = __bfloat162float(__float2bfloat16_rn(v));
  part[0] = fabsf(r) == INFINITY ? __uint_as_float(__float_as_uint(v) & 0xffff0000u) : r;
  if (!(fabsf(v) < INFINITY)) {
    part[0] = v;
    part[1] = part[2] = 0.f;
    return;
  }
  part[1] = __bfloat162float(__float2bfloat16_rn(v - part[0]));
  part[2] = v - part[0] - part[1];
}

struct SplitTensor {
  const float* src;            // [n, heads, D]
  long long token, head, n;
  __nv_bfloat16* dst;          // [3][n][heads][D]
  int heads, vec;
};

// One read, and three writes of half the size; eight numbers to a thread.
template <int D>
__global__ void __launch_bounds__(256) prompt_split_kernel(SplitTensor q, SplitTensor k, SplitTensor v) {
  griddep_wait();
  griddep_launch_dependents();
  const SplitTensor& s = blockIdx.y == 0 ? q : blockIdx.y == 1 ? k : v;
  const long long numbers = s.n * s.heads * D;
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8; i < numbers; i += (long long)gridDim.x * 2048) {
    const long long row = i / D, token = row / s.heads;
    const float* const src = s.src + token * s.token + (row - token * s.heads) * s.head + i % D;
    float x[8];
    if (s.vec) {
      *(float4*)x = __ldg((const float4*)src);
      *(float4*)(x + 4) = __ldg((const float4*)src + 1);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = src[e];
    }
    float part[8][3];
#pragma unroll
    for (int e = 0; e < 8; ++e) split3(x[e], part[e]);
#pragma unroll
    for (int j = 0; j < 3; ++j)
      *(uint4*)(s.dst + j * numbers + i) = make_uint4(pack_bf16(part[0][j], part[1][j]), pack_bf16(part[2][j], part[3][j]),
                                                      pack_bf16(part[4][j], part[5][j]), pack_bf16(part[6][j], part[7][j]));
  }
}

template <int D>
__global__ void __launch_bounds__(kFp32Threads, 1)
prompt_fp32_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                   PromptParams p) {
  using C = PromptFp32<D>;
  constexpr int KT = C::KT;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* const sq = smem;
  uint8_t* const ring = smem + 3 * C::Q_PART;
  __shared__ uint64_t q_full, full[C::SLOTS], empty[C::SLOTS], v_ready[2], s_full[2], p_full, o_full, met[4], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int odd[3][D], any_odd;
  __shared__ float2 told[2][2][128];                          // by turns, from each half of a row to the other
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Nothing of this needs what the kernels before wrote.  TMEM has to be taken before the next kernel may start: one that took
  // it first would keep it until this CTA is done.
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int i = 0; i < C::SLOTS; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(&v_ready[0], 2); mbar_init(&v_ready[1], 2);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1);
    for (int i = 0; i < 4; ++i) mbar_init(&met[i], 2);
    mbar_init(&p_full, 8); mbar_init(&o_full, 1); mbar_init(&drained, 1);
    fence_mbarrier_init();
    any_odd = 0;
    tma_prefetch_desc(&tq); tma_prefetch_desc(&tk); tma_prefetch_desc(&tv);
  }
  for (int i = threadIdx.x; i < 3 * D; i += kFp32Threads) ((int*)odd)[i] = INT_MAX;
  if (warp == 9) { tmem_alloc(&tmem_slot, 512); tmem_relinquish(); }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  griddep_wait();
  griddep_launch_dependents();
  if (blockIdx.x + blockIdx.y == 0 && warp == 11) prompt_record(p);

  const int tokens = 128 / p.group;
  const int head = blockIdx.x % p.Hk;
  PromptSeq s;
  int tile;
  const bool some = prompt_tile(p, blockIdx.x / p.Hk, tokens, s, tile);
  if (!some) {
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, 512);
    return;
  }
  const int token0 = tile * tokens;
  const int keys = prompt_visible(p, s, min(token0 + tokens, s.nq) - 1);
  const int steps = prompt_share(p, blockIdx.y, (keys + KT - 1) / KT, KT, s);

  auto wait = [&](uint64_t* bar, uint32_t parity) { return serving_wait(bar, parity, p.status, kPromptKernelId, kPromptWaitNs); };

  // Parts go through the ring in the order of their products: K(0), K(1), V(0), K(2), V(1), ..., of each the last part first.
  auto k_at = [&](int i) { return i == 0 ? 0 : 6 * i - 3; };
  auto v_at = [&](int i) { return 6 * i + (i + 1 < steps ? 6 : 3); };

  if (warp == 8) {
    // ---------------------------------------------------------------- loads
    if (steps > 0 && elect_one_sync()) {
      mbar_arrive_expect_tx(&q_full, 3 * C::HALVES * tokens * p.group * 128);
      for (int part = 0; part < 3; ++part)
        for (int h = 0; h < C::HALVES; ++h)
          tma_load_4d(sq + part * C::Q_PART + h * 128 * 128, &tq, &q_full, 64 * h, head * p.group, s.q0 + token0, part);
      int n = 0;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, int i) {
        for (int part = 2; ok && part >= 0; --part) {
          const int slot = n % C::SLOTS;
          if (!(ok = wait(&empty[slot], ((n / C::SLOTS) & 1) ^ 1u))) return;
          mbar_arrive_expect_tx(&full[slot], C::KV_PART);
          for (int h = 0; h < C::HALVES; ++h)
            tma_load_4d(ring + slot * C::KV_PART + h * KT * 128, map, &full[slot], 64 * h, head, s.k0 + i * KT, part);
          ++n;
        }
      };
      load(&tk, 0);
      for (int i = 0; ok && i < steps; ++i) {
        if (i + 1 < steps) load(&tk, i + 1);
        if (ok) load(&tv, i);
      }
      // the copies land before the CTA leaves
      wait(&q_full, 0);
      for (int i = max(0, n - C::SLOTS); i < n; ++i) wait(&full[i % C::SLOTS], (i / C::SLOTS) & 1);
    }
  } else if (warp == 9) {
    // ---------------------------------------------------------------- products
    if (steps > 0 && elect_one_sync()) {
      constexpr uint32_t iqk = umma_idesc(1u, 128, KT), ipv = umma_idesc(1u, 128, D) | (1u << 16);
      const uint64_t krow = umma_desc_k_sw128(0), vrow = umma_desc_mn_sw128(0, KT * 128);
      bool ok = wait(&q_full, 0);
      // The parts b of keys or values come in the order 2, 1, 0, and with them the parts a + b <= 2 of q or P: the largest
      // product is the last, and a part's place is free after its own products.
      auto qk = [&](int i) {
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          const int n = k_at(i) + j, slot = n % C::SLOTS;
          if (!(ok = ok && wait(&full[slot], (n / C::SLOTS) & 1))) return;
          tc_fence_after_sync();
          const uint64_t a = desc_at(krow, smem_u32(sq)), b = desc_at(krow, smem_u32(ring + slot * C::KV_PART));
#pragma unroll
          for (int part = j; part >= 0; --part)
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              umma_f16(tmem + KT * (i & 1), a + (part * C::Q_PART + (k / 4) * 128 * 128) / 16 + (k % 4) * 2,
                       b + ((k / 4) * KT * 128) / 16 + (k % 4) * 2, iqk, j > 0 || k > 0);
          umma_commit(&empty[slot]);
        }
        umma_commit(&s_full[i & 1]);
      };
      qk(0);
      for (int i = 0; ok && i < steps; ++i) {
        // S of the step after this one goes where the one before was, which was read before its P came
        if (i + 1 < steps) qk(i + 1);
        if (!(ok = ok && wait(&v_ready[i & 1], (i >> 1) & 1) && wait(&p_full, i & 1))) break;
        tc_fence_after_sync();
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          const int slot = (v_at(i) + j) % C::SLOTS;
          const uint64_t b = desc_at(vrow, smem_u32(ring + slot * C::KV_PART));
#pragma unroll
          for (int part = j; part >= 0; --part)
#pragma unroll
            for (int k = 0; k < KT / 16; ++k)
              umma_f16_ts(tmem + C::O_AT, tmem + C::P_AT + part * (KT / 2) + 8 * k, b + (k * 16 * 128) / 16, ipv, j > 0 || k > 0);
          umma_commit(&empty[slot]);
        }
        umma_commit(&o_full);
      }
      umma_commit(&drained);
      wait(&drained, 0);
    }
  } else if (warp >= 10) {
    // ---------------------------------------------------------------- values
    for (int i = 0; i < steps; ++i) {
      uint8_t* at[3];              // the parts
      bool ok = true;
      for (int part = 2; ok && part >= 0; --part) {
        const int n = v_at(i) + 2 - part, slot = n % C::SLOTS;
        ok = mbar_wait_warp(&full[slot], (n / C::SLOTS) & 1, p.status, kPromptKernelId, kPromptWaitNs);
        at[part] = ring + slot * C::KV_PART;
      }
      if (!ok) break;
      prompt_fix_values<D, KT, 8>(at, threadIdx.x - 320, i * KT, s.nk - i * KT, odd, &any_odd);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_ready[i & 1]);
    }
  } else {
    // ---------------------------------------------------------------- softmax, half a row to a thread
    constexpr int KH = KT / 2, DH = D / 2;                      // keys and dimensions of one half
    const int half = warp >> 2, row = threadIdx.x & 127, token = token0 + row / p.group, hq = head * p.group + row % p.group;
    const bool mine = row < tokens * p.group && token < s.nq;
    const int visible = mine ? min(prompt_visible(p, s, token), s.nk) : 0;
    const int all = __reduce_min_sync(0xffffffffu, mine ? visible : INT_MAX);
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float mult = p.scale * 1.44269504088896341f;
    const float turn = mult > 0.f ? 1.f : mult < 0.f ? -1.f : 0.f;
    mult = turn == 0.f ? 1.f : fabsf(mult);
    float m = -INFINITY, l = 0.f, o[DH];
#pragma unroll
    for (int d = 0; d < DH; ++d) o[d] = 0.f;
    // The other half's numbers of the same row; the place is written again two turns on, when both have met once more.
    auto exchange = [&](int turn_of, float2 v, float2& other) {
      told[turn_of & 1][half][row] = v;
      __syncwarp();
      if (lane == 0) mbar_arrive(&met[warp & 3]);
      if (!mbar_wait_warp(&met[warp & 3], turn_of & 1, p.status, kPromptKernelId, kPromptWaitNs)) return false;
      other = told[turn_of & 1][half ^ 1][row];
      return true;
    };
    // the sums of step i, once its products are done
    auto add = [&](int i) {
      if (!mbar_wait_warp(&o_full, i & 1, p.status, kPromptKernelId, kPromptWaitNs)) return false;
      tc_fence_after_sync();
#pragma unroll
      for (int c = 0; c < DH; c += 32) {
        uint32_t r[32];
        tmem_ld32(lanes + C::O_AT + half * DH + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) o[c + e] += __uint_as_float(r[e]);
      }
      return true;
    };
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      if (!(ok = mbar_wait_warp(&s_full[i & 1], (i >> 1) & 1, p.status, kPromptKernelId, kPromptWaitNs))) break;
      tc_fence_after_sync();
      uint32_t r[KH];
#pragma unroll
      for (int c = 0; c < KH; c += 32) tmem_ld32(lanes + KT * (i & 1) + half * KH + c, r + c);
      tmem_ld_wait();
      if (turn != 1.f) {
#pragma unroll
        for (int c = 0; c < KH; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * turn);
      }
      const int k0 = i * KT + half * KH;
      if (k0 + KH > all) {
#pragma unroll
        for (int c = 0; c < KH; ++c)
          if (k0 + c >= visible) r[c] = __float_as_uint(-INFINITY);
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < KH; c += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(r[c + 2 * e]), __uint_as_float(r[c + 2 * e + 1]));
      float peak = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      float2 other;
      if (!(ok = exchange(i, make_float2(peak, l), other))) break;
      peak = fmaxf(peak, other.x) * mult;
      const bool grow = peak > m - kPromptNear || l + other.y > kPromptSum, follow = __any_sync(0xffffffffu, grow);
      float shrink = 1.f;
      if (follow) {
        const float now = grow ? fmaxf(peak + kPromptHeadFp32, m + kPromptLeast) : m;
        shrink = m == -INFINITY ? 0.f : prompt_exp2(m - now);
        m = now;
        l *= shrink;
      }
      // P is written where the last step's was, so that one's products come first: ahead of them the first 32 weights, where
      // a thread has 64 (three sequences of 2049 tokens in all, heads of 64: 56 -> 53 us); where it has 32, that is slower
      // (2000 tokens, 32 heads of 128: 381 -> 386 us; causal, over 8 key heads, 184 -> 187).
      constexpr bool AHEAD = KH > 32;
      auto sums = [&] {
        if (i > 0 && !add(i - 1)) return false;
        if (follow) {
#pragma unroll
          for (int d = 0; d < DH; ++d) o[d] *= shrink;
        }
        return true;
      };
      if (!AHEAD && !(ok = sums())) break;
      const float base = m == -INFINITY ? 0.f : -m;
      const uint64_t mult2 = pair_f32(mult, mult), base2 = pair_f32(base, base);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int h = 0; h < KH; h += 32) {
        uint32_t w[3][16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          float u, v;
          unpair_f32(fma2(pair_f32(__uint_as_float(r[h + 2 * c]), __uint_as_float(r[h + 2 * c + 1])), mult2, base2), u, v);
          uint64_t x = pair_f32(prompt_exp2(u), prompt_exp2(v));
          sum[c & 1] = add2(sum[c & 1], x);
#pragma unroll
          for (int part = 0; part < 3; ++part) {
            unpair_f32(x, u, v);
            const uint32_t rounded = pack_bf16(u, v);
            w[part][c] = rounded;
            if (part < 2) x = add2(x, pair_f32(__uint_as_float((rounded << 16) ^ 0x80000000u), __uint_as_float((rounded & 0xffff0000u) ^ 0x80000000u)));
          }
        }
        if (AHEAD && h == 0 && !(ok = sums())) break;
#pragma unroll
        for (int part = 0; part < 3; ++part) tmem_st16(lanes + C::P_AT + part * (KT / 2) + (half * KH + h) / 2, w[part]);
      }
      if (!ok) break;
      float s0, s1;
      unpair_f32(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full);
    }
    if (ok && steps > 0) ok = add(steps - 1);
    float2 other;
    if (ok && exchange(max(steps, 0), make_float2(0.f, l), other)) l += other.y;
    if (l == 0.f && visible > 0 && steps > 0) l = -0.f;
    const float inv = prompt_per_sum(p, l);
    const long long at = ((long long)blockIdx.y * p.Nq + s.q0 + token) * p.Hq + hq;   // of the parts
    float* const dst = half * DH + (p.splits > 1 ? p.parts + at * D
                                                 : (float*)p.out + (long long)(s.q0 + token) * p.o_token + (long long)hq * p.o_head);
    if (any_odd) {
#pragma unroll
      for (int d = 0; d < DH; ++d) o[d] = put_back_odd<D>(odd, half * DH + d, visible, o[d] * inv);
    } else {
#pragma unroll
      for (int d = 0; d < DH; ++d) o[d] *= inv;
    }
    if (mine) {
      if (p.o_vec || p.splits > 1) {
#pragma unroll
        for (int d = 0; d < DH; d += 4) *(float4*)(dst + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
      } else {
#pragma unroll
        for (int d = 0; d < DH; ++d) dst[d] = o[d];
      }
      if (half == 0) {
        if (p.splits > 1) p.stats[at] = make_float2(m, l);
        else if (p.lse != nullptr) p.lse[(long long)(s.q0 + token) * p.Hq + hq] = prompt_lse(m, l, kPromptHeadFp32);
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace raiccl
