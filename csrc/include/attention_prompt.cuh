// What the kernels of attention over whole prompts share: which rows of which
// sequence a CTA has, and numbers of values that are not finite.
#pragma once

#include "attention.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

// A sequence's tokens in q and in k, v.
struct PromptSeq {
  int q0, nq, k0, nk;
};

// Ends outside of the tensors, or before their beginnings, are cut, and recorded by one warp of the launch.
template <bool RECORD = false>
__device__ __forceinline__ PromptSeq prompt_seq(const PromptParams& p, int b) {
  const int q0 = __ldg(p.cu_q + b), q1 = __ldg(p.cu_q + b + 1), k0 = __ldg(p.cu_k + b), k1 = __ldg(p.cu_k + b + 1);
  PromptSeq s;
  s.q0 = q0 < 0 ? 0 : q0 > p.Nq ? (int)p.Nq : q0;
  s.k0 = k0 < 0 ? 0 : k0 > p.Nk ? (int)p.Nk : k0;
  const int qe = q1 < s.q0 ? s.q0 : q1 > p.Nq ? (int)p.Nq : q1, ke = k1 < s.k0 ? s.k0 : k1 > p.Nk ? (int)p.Nk : k1;
  s.nq = qe - s.q0;
  s.nk = ke - s.k0;
  if (RECORD && (s.q0 != q0 || qe != q1)) record_status(p.status, kBoundsViolation, kPromptKernelId, q1, p.Nq);
  if (RECORD && (s.k0 != k0 || ke != k1)) record_status(p.status, kBoundsViolation, kPromptKernelId, k1, p.Nk);
  return s;
}

__device__ __forceinline__ void prompt_record(const PromptParams& p) {
  for (int b = threadIdx.x & 31; b < p.B; b += 32) prompt_seq<true>(p, b);
}

// Tiles of `tokens` tokens of q that sequence b has, by its cut ends.
__device__ __forceinline__ int prompt_tiles(const PromptParams& p, int b, int tokens) {
  const int n = (int)p.Nq, q0 = min(max(__ldg(p.cu_q + b), 0), n), q1 = min(max(__ldg(p.cu_q + b + 1), q0), n);
  return (q1 - q0 + tokens - 1) / tokens;
}

// The tile `index` of all sequences' tiles of `tokens` tokens of q; false behind the last.  A whole warp calls it.  Within a
// sequence the last tile, which sees the most keys, comes first.
//
// Up to 32 sequences, one to a lane, go by their number of keys, the longest first, so that no long tile begins when the
// others are done (eight chunks of 512 tokens on average: 168 -> 161 us).  More of them even that out by themselves and go in their
// order: every lane counts an equal number of
// sequences, then the warp goes through those of the lane that has the tile.
__device__ __forceinline__ bool prompt_tile(const PromptParams& p, int index, int tokens, PromptSeq& s, int& tile) {
  const int lane = threadIdx.x & 31;
  if (p.B <= 32) {
    PromptSeq mine{0, 0, 0, 0};
    if (lane < p.B) mine = prompt_seq(p, lane);
    const int tiles = (mine.nq + tokens - 1) / tokens;
    int ahead = 0;
    for (int b = 0; b < p.B; ++b) {
      const int nk = __shfl_sync(0xffffffffu, mine.nk, b), n = __shfl_sync(0xffffffffu, tiles, b);
      if (nk > mine.nk || (nk == mine.nk && b < lane)) ahead += n;
    }
    const uint32_t in = __ballot_sync(0xffffffffu, index >= ahead && index - ahead < tiles);
    if (in == 0) return false;
    const int at = __ffs(in) - 1;
    s.q0 = __shfl_sync(0xffffffffu, mine.q0, at);
    s.nq = __shfl_sync(0xffffffffu, mine.nq, at);
    s.k0 = __shfl_sync(0xffffffffu, mine.k0, at);
    s.nk = __shfl_sync(0xffffffffu, mine.nk, at);
    tile = __shfl_sync(0xffffffffu, ahead + tiles - 1, at) - index;
    return true;
  }
  int first = 0, each = p.B, before = 0;
  while (true) {
    const int per = (each + 31) / 32, b0 = first + lane * per, b1 = min(b0 + per, first + each);
    int sum = 0;
#pragma unroll 8
    for (int b = b0; b < b1; ++b) sum += prompt_tiles(p, b, tokens);
    const int mine = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t in = __ballot_sync(0xffffffffu, index < before + sum);
    if (in == 0) return false;
    const int at = __ffs(in) - 1;
    before += __shfl_sync(0xffffffffu, sum - mine, at);
    first += at * per;
    if (per == 1) {
      s = prompt_seq(p, first);
      tile = before + __shfl_sync(0xffffffffu, mine, at) - 1 - index;
      return true;
    }
    each = min(per, p.B - first);
  }
}

// This CTA's share of a tile's `steps` steps of `width` keys, where several CTAs share them: the sequence is cut to it, so
// that everything behind goes by the share alone.
__device__ __forceinline__ int prompt_share(const PromptParams& p, int split, int steps, int width, PromptSeq& s) {
  const int each = (steps + p.splits - 1) / p.splits, first = min(steps, split * each);
  s.k0 += first * width;
  s.nk -= first * width;
  return min(each, steps - first);
}

// Keys that row `token` of q sees.
__device__ __forceinline__ int prompt_visible(const PromptParams& p, const PromptSeq& s, int token) {
  if (!p.causal) return s.nk;
  const int n = s.nk - s.nq + token + 1;
  return n < 0 ? 0 : n;
}

// Weights are exp2(z - m).  Where m is set it is HEAD above the row's maximum, and it is set again once a logit comes nearer to
// it than 9 or the sum l of the weights passes 1/4 (by 8 at least).  So no weight is above 2^-9, a step's 128 add 1/4 at
// most, l stays below 1/2, and sums of weights times finite values below the largest of those: they never overflow,
// however large the values.  (At logits of 2^27 the distance is lost in rounding, and values above 2^128 / keys may overflow.)
// With m at the maximum, and followed at 2^64 times (bf16) or 2^8 times (fp32) that, values above 2^64 or 2^120 by the number of
// keys became infinities.
//
// What HEAD costs: weights near the largest are 2^-HEAD and up, whose products with values below 2^(HEAD - 130) or so lose
// bits; and z - m is off by half a last place of HEAD.  What it gives: m is set again only where logits rise by HEAD - 9 after a
// row's first step.  In fp32, where sums are in registers, that costs little: 15.  In bf16 it takes a third of a step from all
// 128 rows of a tile, and for logits that spread by 3 nats or more a HEAD of 15 made prompts 25 % slower: 31 (22 powers of two, 15
// nats); and 47 from then on, for rows that rise like that will again, and all rows of the warp at once.
constexpr int kPromptHeadFp32 = 15, kPromptHeadTc = 31, kPromptHeadAgain = 47;
constexpr float kPromptNear = 9.f, kPromptSum = 0.25f, kPromptLeast = 8.f;

// log sum exp(z); l is mostly near 2^-head of exponents at the maximum.
__device__ __forceinline__ float prompt_lse(float m, float l, int head) {
  return ((m - head) + log2f(scalbnf(l, head))) * 0.69314718055994531f;
}

// 1 / l.  A row without keys has l = 0, and zeros for a result.  One that sees keys whose logits are all -inf has l = -0: NaN,
// but not yet where other CTAs have some of its keys, whose logits may be finite; -0 tells the join that there were keys.
__device__ __forceinline__ float prompt_per_sum(const PromptParams& p, float l) {
  return l != 0.f ? 1.f / l : __float_as_uint(l) != 0u && p.splits == 1 ? NAN : 0.f;
}

// Values that are not finite must not reach rows that do not see them, but a
// product adds 0 * NaN there.  They go into the products as zeros, and for each
// kind and dimension the first key that has one is kept; a row sees a prefix of
// the keys, so that is enough to put them back.  first[0]: NaN, [1]: +inf, [2]: -inf.
__device__ __forceinline__ int odd_kind(float v) { return v != v ? 0 : v > 0.f ? 1 : 2; }

// So 64 threads look through a tile of KT values (rows of 128 bytes in the 128-byte swizzle, 64 dimensions; the next 64
// behind them), of which rows from `behind` on are of no key of this sequence's: those become zeros, in every part.  What is not
// finite is in the first part.  16-byte pieces are loaded BATCH at a time, and put back one by one only where one of them has such
// a number: with each stored before the next was loaded a tile of 16 KB took 4000 clocks, more than its products.
template <int D, int KT, int BATCH, int PARTS>
__device__ __forceinline__ void prompt_fix_values(uint8_t* const (&part)[PARTS], int thread, int key0, int behind, int (*first)[D], int* any_odd) {
  constexpr int PIECES = KT * D / 8;
  static_assert(PIECES % (64 * BATCH) == 0, "whole batches");
  if (behind < KT) {
    for (int c = thread; c < PIECES; c += 64)
      if ((c / 8) % KT >= behind)
#pragma unroll
        for (int j = 0; j < PARTS; ++j) ((uint4*)part[j])[c] = make_uint4(0, 0, 0, 0);
  }
  auto bad = [](uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };   // an exponent of ones
  uint4* const at = (uint4*)part[0];
#pragma unroll 1
  for (int c0 = thread; c0 < PIECES; c0 += 64 * BATCH) {
    uint32_t some = 0;
    uint4 v[BATCH];
#pragma unroll
    for (int e = 0; e < BATCH; ++e) v[e] = at[c0 + 64 * e];
#pragma unroll
    for (int e = 0; e < BATCH; ++e) some |= bad(v[e].x) | bad(v[e].y) | bad(v[e].z) | bad(v[e].w);
    if (some == 0) continue;
#pragma unroll 1
    for (int c = c0; c < c0 + 64 * BATCH; c += 64) {
      const int row = (c / 8) % KT, d = 64 * (c / (8 * KT)) + 8 * ((c & 7) ^ (row & 7));
      __nv_bfloat16* const x = (__nv_bfloat16*)(at + c);
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        const float f = __bfloat162float(x[e]);
        if (fabsf(f) < INFINITY) continue;
        atomicMin(&first[odd_kind(f)][d + e], key0 + row);
        x[e] = __float2bfloat16_rn(0.f);
      }
    }
    *any_odd = 1;
  }
}

template <int D>
__device__ __forceinline__ float put_back_odd(const int (*first)[D], int d, int visible, float v) {
  // v may hold some already, of tiles that all rows saw whole
  const bool nan = v != v || first[0][d] < visible, up = v == INFINITY || first[1][d] < visible, down = v == -INFINITY || first[2][d] < visible;
  if (nan || (up && down)) return NAN;
  return up ? INFINITY : down ? -INFINITY : v;
}

}  // namespace raiccl
