// Attention over whole prompts: packed sequences, causal or not, grouped heads.
// bf16 on tcgen05 (attention_prompt_tc.cuh); fp32 here, as two tf32 parts of each
// number.
#include <algorithm>
#include <atomic>
#include <climits>
#include <stdexcept>

#include "attention.h"
#include "attention_join.cuh"
#include "attention_prompt.cuh"
#include "attention_prompt_tc.cuh"
#include "serving.h"
#include "serving_device.cuh"
#include "serving_tma.h"
#include "sm100_ptx.cuh"

namespace raiccl {

constexpr int kRowsTile = 128, kRowsKeys = 32;

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D>
struct PromptRows {
  static constexpr int KS = D + 8, VS = D + 4;   // strides of a key's and a value's row, without conflicts of the fragments' loads
  static constexpr int TILE = kRowsKeys * (KS + VS);        // numbers: keys, then values
  static constexpr int SMEM = 4 * 3 * TILE;                 // two tiles as they lie, the rests of one
  static constexpr int CTAS = D == 64 ? 2 : 1;              // to an SM, by registers
};

__device__ __forceinline__ void rows_copy(uint32_t to, const float* from, bool there, bool vec) {
  const int n = there ? 16 : 0;      // what is not read is zeros
  if (vec) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 4 * i), "l"(there ? from + i : from), "r"(n / 4) : "memory");
  }
}

// fp32: every number is two tf32 parts, its upper 19 bits, which is what the
// tensor core reads of it, and the rest; three products.  One CTA: 128 rows (a
// token and a query head of the group), eight warps of sixteen; 32 keys at a time
// by cp.async, a tile ahead; the rests are worked out in shared memory, once for
// all warps.
//
// The tensor core cuts what does not fit its sums, so the products with a rest
// have sums of their own, and those of the values leave it every 32 keys.
template <int D>
__global__ void __launch_bounds__(256, PromptRows<D>::CTAS) prompt_rows_kernel(PromptParams p, bool vec) {
  using C = PromptRows<D>;
  extern __shared__ __align__(16) float sm[];
  float* const rest = sm + 2 * C::TILE;
  __shared__ int odd[3][D], any_odd;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  for (int i = threadIdx.x; i < 3 * D; i += 256) ((int*)odd)[i] = INT_MAX;
  if (threadIdx.x == 0) any_odd = 0;
  griddep_wait();
  griddep_launch_dependents();
  const int tokens = kRowsTile / p.group, head = blockIdx.y;
  PromptSeq s;
  int tile;
  if (!prompt_tile(p, blockIdx.x, tokens, s, tile)) return;
  const int rows = min(tokens, s.nq - tile * tokens) * p.group;

  const int all = prompt_visible(p, s, min(tile * tokens + tokens, s.nq) - 1);
  const int keys = kRowsKeys * prompt_share(p, blockIdx.z, (all + kRowsKeys - 1) / kRowsKeys, kRowsKeys, s);
  int visible[2], token[2], hq[2];
  bool row_in[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = 16 * warp + 8 * r + g;
    row_in[r] = row < rows;
    token[r] = tile * tokens + row / p.group;
    hq[r] = head * p.group + row % p.group;
    visible[r] = row_in[r] ? min(prompt_visible(p, s, token[r]), s.nk) : 0;
  }

  auto copy = [&](int k0, int stage) {
    const uint32_t to = smem_u32(sm + stage * C::TILE);
    for (int i = threadIdx.x; i < kRowsKeys * D / 4; i += 256) {
      const int row = i / (D / 4), d = 4 * (i - row * (D / 4));
      const bool there = k0 + row < s.nk;
      const long long at = s.k0 + (there ? k0 + row : 0);
      rows_copy(to + 4 * (row * C::KS + d), (const float*)p.k + at * p.k_token + head * p.k_head + d, there, vec);
      rows_copy(to + 4 * (kRowsKeys * C::KS + row * C::VS + d), (const float*)p.v + at * p.v_token + head * p.v_head + d, there, vec);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (keys > 0) copy(0, 0);

  float q[2][D / 4];   // dimensions 8 j + 2 t and + 1
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      const long long at = (long long)(s.q0 + token[r]) * p.q_token + (long long)hq[r] * p.q_head + 8 * j + 2 * t;
      q[r][2 * j] = row_in[r] ? ((const float*)p.q)[at] : 0.f;
      q[r][2 * j + 1] = row_in[r] ? ((const float*)p.q)[at + 1] : 0.f;
    }
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[n][j] = 0.f;
  const float mult = p.scale * 1.44269504088896341f;

  for (int k0 = 0, stage = 0; k0 < keys; k0 += kRowsKeys, stage ^= 1) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (k0 + kRowsKeys < keys) copy(k0 + kRowsKeys, stage ^ 1);
    float *const kh = sm + stage * C::TILE, *const vh = kh + kRowsKeys * C::KS;
    float *const kl = rest, *const vl = rest + kRowsKeys * C::KS;
    for (int i = threadIdx.x; i < kRowsKeys * D / 4; i += 256) {
      const int row = i / (D / 4), d = 4 * (i - row * (D / 4));
      const float4 x = *(const float4*)(kh + row * C::KS + d);
      *(float4*)(kl + row * C::KS + d) = make_float4(rest_tf32(x.x), rest_tf32(x.y), rest_tf32(x.z), rest_tf32(x.w));
      const float4 v = *(const float4*)(vh + row * C::VS + d);
      float y[4] = {v.x, v.y, v.z, v.w};
      bool finite = true;
#pragma unroll
      for (int j = 0; j < 4; ++j) finite &= fabsf(y[j]) < INFINITY;
      if (!finite) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!(fabsf(y[j]) < INFINITY)) {
            atomicMin(&odd[odd_kind(y[j])][d + j], k0 + row);
            any_odd = 1;
            y[j] = 0.f;
            vh[row * C::VS + d + j] = 0.f;
          }
      }
      *(float4*)(vl + row * C::VS + d) = make_float4(rest_tf32(y[0]), rest_tf32(y[1]), rest_tf32(y[2]), rest_tf32(y[3]));
    }
    __syncthreads();
    float z[kRowsKeys / 8][4];
    {
      float zl[kRowsKeys / 8][4];
#pragma unroll
      for (int n = 0; n < kRowsKeys / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) z[n][j] = zl[n][j] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = q[i & 1][2 * j + (i >> 1)];
          ah[i] = __float_as_uint(v);
          al[i] = __float_as_uint(rest_tf32(v));
        }
        // four products in a row that do not wait for one another
        float2 h[kRowsKeys / 8], low[kRowsKeys / 8];
#pragma unroll
        for (int n = 0; n < kRowsKeys / 8; ++n) {
          h[n] = *(const float2*)(kh + (8 * n + g) * C::KS + 8 * j + 2 * t);
          low[n] = *(const float2*)(kl + (8 * n + g) * C::KS + 8 * j + 2 * t);
        }
#pragma unroll
        for (int n = 0; n < kRowsKeys / 8; ++n) mma_tf32(z[n], ah, __float_as_uint(h[n].x), __float_as_uint(h[n].y));
#pragma unroll
        for (int n = 0; n < kRowsKeys / 8; ++n) mma_tf32(zl[n], al, __float_as_uint(h[n].x), __float_as_uint(h[n].y));
#pragma unroll
        for (int n = 0; n < kRowsKeys / 8; ++n) mma_tf32(zl[n], ah, __float_as_uint(low[n].x), __float_as_uint(low[n].y));
      }
#pragma unroll
      for (int n = 0; n < kRowsKeys / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) z[n][j] += zl[n][j];
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kRowsKeys / 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + 8 * n + 2 * t + (j & 1);
        if (key < visible[j >> 1]) top[j >> 1] = fmaxf(top[j >> 1], z[n][j] * mult);
      }
    float now[2], shrink[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      now[r] = fmaxf(m[r], top[r]);
      shrink[r] = now[r] == -INFINITY ? 1.f : exp2f(m[r] - now[r]);
      m[r] = now[r];
      l[r] *= shrink[r];
    }
    uint32_t ph[kRowsKeys / 8][4], pl[kRowsKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kRowsKeys / 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // a masked key adds nothing, whatever m is; a row of -inf alone is NaN, as its formula is.  One fma: off by a
        // rounding of the difference, not of the logit.
        const int key = k0 + 8 * n + 2 * t + (j & 1);
        const float e = key < visible[j >> 1] ? exp2f(fmaf(z[n][j], mult, -m[j >> 1])) : 0.f;
        l[j >> 1] += e;
        const int at = (j & 1) * 2 + (j >> 1);         // the other operand's order
        ph[n][at] = __float_as_uint(e);
        pl[n][at] = __float_as_uint(rest_tf32(e));
      }
#pragma unroll
    for (int n = 0; n < D / 8; n += 2) {
      float fresh[2][4] = {}, low[2][4] = {};
#pragma unroll
      for (int k = 0; k < kRowsKeys / 8; ++k) {
        uint32_t h[2][2], v[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = (8 * k + 2 * t) * C::VS + 8 * (n + e) + g;
          h[e][0] = __float_as_uint(vh[at]);
          h[e][1] = __float_as_uint(vh[at + C::VS]);
          v[e][0] = __float_as_uint(vl[at]);
          v[e][1] = __float_as_uint(vl[at + C::VS]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) mma_tf32(fresh[e], ph[k], h[e][0], h[e][1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) mma_tf32(low[e], pl[k], h[e][0], h[e][1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) mma_tf32(low[e], ph[k], v[e][0], v[e][1]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n + e][j] = fmaf(o[n + e][j], shrink[j >> 1], fresh[e][j] + low[e][j]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (!row_in[r]) continue;
    const long long row = ((long long)blockIdx.z * p.Nq + s.q0 + token[r]) * p.Hq + hq[r];   // of the parts
    const float inv = p.splits > 1 ? 1.f : l[r] == 0.f ? 0.f : 1.f / l[r];
    const long long at = (long long)(s.q0 + token[r]) * p.o_token + (long long)hq[r] * p.o_head;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      float v[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        v[e] = o[n][2 * r + e] * inv;
        if (any_odd) v[e] = put_back_odd<D>(odd, 8 * n + 2 * t + e, visible[r], v[e]);
      }
      float* const out = (p.splits > 1 ? p.parts + row * D : (float*)p.out + at) + 8 * n + 2 * t;
      if (p.o_vec || p.splits > 1) *(float2*)out = make_float2(v[0], v[1]);
      else { out[0] = v[0]; out[1] = v[1]; }
    }
    if (p.splits > 1) {
      if (t == 0) p.stats[row] = make_float2(m[r], l[r]);
    } else if (p.lse != nullptr && t == 0)
      p.lse[(long long)(s.q0 + token[r]) * p.Hq + hq[r]] = (m[r] + log2f(l[r])) * 0.69314718055994531f;
  }
}

// The results of tiles whose keys several CTAs shared, a warp to a row.  Rows before the first sequence and behind the last
// stay as they are.
template <int D>
__global__ void __launch_bounds__(256) prompt_join_kernel(PromptParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= p.Nq * p.Hq) return;
  const long long token = row / p.Hq, hq = row - token * p.Hq;
  if (token < __ldg(p.cu_q) || token >= __ldg(p.cu_q + p.B)) return;
  float top, l, v[D / 32];
  auto at = [&](int j) { return j * p.Nq * p.Hq + row; };
  warp_join<D>(p.splits, [&](int j) { return p.stats[at(j)]; }, [&](int j) { return p.parts + at(j) * D; }, top, l, v);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) store_elem(p.out, token * p.o_token + hq * p.o_head + D / 32 * lane + i, v[i] * inv, p.bf16);
  if (p.lse != nullptr && lane == 0) p.lse[row] = (top + log2f(l)) * 0.69314718055994531f;
}

// Rows of a tensor [n, heads, D] that TMA can read: on 16 bytes, and apart.
static bool tma_rows(const void* t, long long token, long long head, long long n, int heads) {
  return ((uintptr_t)t & 15) == 0 && (n <= 1 || (token > 0 && token % 8 == 0)) && (heads <= 1 || (head > 0 && head % 8 == 0));
}

// CTAs share a tile's keys where there are fewer tiles than SMs, at least 512 keys to one.
PromptPlan plan_prompt(const PromptParams& p, int sms) {
  PromptPlan plan{};
  const int tokens = (p.bf16 ? 2 * (128 / p.group) : kRowsTile / p.group);
  const long long tiles = ((p.Nq + tokens - 1) / tokens + p.B - 1) * p.Hk;   // at most
  plan.splits = (int)std::max<long long>(1, std::min<long long>({sms / tiles, p.Nk / 512, 32}));
  if (plan.splits > 1) {
    plan.parts_bytes = (long long)plan.splits * p.Nq * p.Hq * p.D * 4;
    plan.stats_bytes = ((long long)plan.splits * p.Nq * p.Hq * 8 + 255) / 256 * 256;
  }
  if (!p.bf16) return plan;
  auto bytes = [&](long long n, int heads) { return (n * heads * p.D * 2 + 255) / 256 * 256; };
  plan.pack_q = !tma_rows(p.q, p.q_token, p.q_head, p.Nq, p.Hq);
  plan.pack_k = p.Nk > 0 && !tma_rows(p.k, p.k_token, p.k_head, p.Nk, p.Hk);
  plan.pack_v = p.Nk > 0 && !tma_rows(p.v, p.v_token, p.v_head, p.Nk, p.Hk);
  if (plan.pack_q) plan.q_bytes = bytes(p.Nq, p.Hq);
  if (plan.pack_k) plan.k_bytes = bytes(p.Nk, p.Hk);
  if (plan.pack_v) plan.v_bytes = bytes(p.Nk, p.Hk);
  return plan;
}

template <typename K>
static void configure(K kern, int smem, std::atomic<unsigned long long>& configured) {
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (configured.load() & bit) return;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    throw std::runtime_error("attention_prompt: shared memory");
  configured.fetch_or(bit);
}

template <int D>
static void launch_prompt_rows(const PromptParams& p, cudaStream_t s) {
  using C = PromptRows<D>;
  auto kern = prompt_rows_kernel<D>;
  static std::atomic<unsigned long long> configured;   // by device
  configure(kern, C::SMEM, configured);
  const int tokens = kRowsTile / p.group;
  auto aligned = [&](const void* t, long long a, long long b) { return (((uintptr_t)t | (a * 4) | (b * 4)) & 15) == 0; };
  const bool vec = aligned(p.k, p.k_token, p.k_head) && aligned(p.v, p.v_token, p.v_head);
  const dim3 grid((unsigned)((p.Nq + tokens - 1) / tokens + p.B - 1), (unsigned)p.Hk, (unsigned)p.splits);
  launch_with_pdl(kern, grid, dim3(256), C::SMEM, s, true, p, vec);
}

// [tokens, heads, D] as TMA reads it: boxes of 64 dimensions, `heads_box` heads and `tokens_box` tokens.
static CUtensorMap prompt_map(const void* base, long long token, long long head, long long n, int heads, int D, int heads_box, int tokens_box) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)n};
  const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? head * 2 : D * 2), (cuuint64_t)(n > 1 ? token * 2 : D * 2)};
  const cuuint32_t box[3] = {64, (cuuint32_t)heads_box, (cuuint32_t)tokens_box};
  return make_tmap(base, true, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D>
static void launch_prompt_tc(const PromptParams& p, cudaStream_t s) {
  using C = PromptTc<D>;
  auto kern = prompt_tc_kernel<D>;
  static std::atomic<unsigned long long> configured;   // by device
  configure(kern, C::SMEM, configured);
  const int tokens = 128 / p.group;
  const CUtensorMap tq = prompt_map(p.q, p.q_token, p.q_head, p.Nq, p.Hq, D, p.group, tokens);
  // without keys nothing is loaded; a map has to name something
  const CUtensorMap tk = p.Nk > 0 ? prompt_map(p.k, p.k_token, p.k_head, p.Nk, p.Hk, D, 1, kPromptKeys) : tq;
  const CUtensorMap tv = p.Nk > 0 ? prompt_map(p.v, p.v_token, p.v_head, p.Nk, p.Hk, D, 1, kPromptKeys) : tq;
  const long long tiles = (p.Nq + 2 * tokens - 1) / (2 * tokens) + p.B - 1;   // at most
  launch_with_pdl(kern, dim3((unsigned)(tiles * p.Hk), (unsigned)p.splits), dim3(kPromptThreads), C::SMEM, s, true, tq, tk, tv, p);
}

void launch_prompt(const PromptParams& params, const PromptPlan& plan, void* workspace, cudaStream_t s) {
  PromptParams p = params;
  char* ws = (char*)workspace;
  p.splits = plan.splits;
  p.parts = (float*)ws;
  p.stats = (float2*)(ws + plan.parts_bytes);
  ws += plan.parts_bytes + plan.stats_bytes;
  auto join = [&] {
    if (p.splits == 1) return;
    const dim3 grid((unsigned)((p.Nq * p.Hq + 7) / 8));
    if (p.D == 128) launch_with_pdl(prompt_join_kernel<128>, grid, dim3(256), 0, s, true, p);
    else launch_with_pdl(prompt_join_kernel<64>, grid, dim3(256), 0, s, true, p);
  };
  if (!p.bf16) {
    if (p.D == 128) launch_prompt_rows<128>(p, s);
    else launch_prompt_rows<64>(p, s);
    return join();
  }
  auto pack = [&](const void*& t, long long& token, long long& head, long long n, int heads, long long bytes) {
    launch_pack_rows(t, token, head, heads, ws, p.D, n, p.D, 1, s);   // [heads, tokens, D]
    t = ws;
    token = p.D;
    head = n * p.D;
    ws += bytes;
  };
  if (plan.pack_q) pack(p.q, p.q_token, p.q_head, p.Nq, p.Hq, plan.q_bytes);
  if (plan.pack_k) pack(p.k, p.k_token, p.k_head, p.Nk, p.Hk, plan.k_bytes);
  if (plan.pack_v) pack(p.v, p.v_token, p.v_head, p.Nk, p.Hk, plan.v_bytes);
  if (p.D == 128) launch_prompt_tc<128>(p, s);
  else launch_prompt_tc<64>(p, s);
  join();
}

}  // namespace raiccl
