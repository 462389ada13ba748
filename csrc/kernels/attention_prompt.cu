// Attention over whole prompts: packed sequences, causal or not, grouped heads.
// bf16 in attention_prompt_tc.cuh, fp32 in attention_prompt_fp32.cuh.
#include <algorithm>
#include <atomic>
#include <climits>
#include <stdexcept>

#include "attention.h"
#include "attention_join.cuh"
#include "attention_prompt.cuh"
#include "attention_prompt_fp32.cuh"
#include "attention_prompt_tc.cuh"
#include "serving.h"
#include "serving_device.cuh"
#include "serving_tma.h"
#include "sm100_ptx.cuh"

namespace raiccl {

// The results of tiles whose keys up to 32 CTAs shared, a warp to a row.  Parts are means of their own keys' values, so that what
// is added up here stays below the largest of these too.  Rows before the first sequence and behind the last stay as they are.
template <int D>
__global__ void __launch_bounds__(256) prompt_join_kernel(PromptParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= p.Nq * p.Hq) return;
  const long long token = row / p.Hq, hq = row - token * p.Hq;
  if (token < __ldg(p.cu_q) || token >= __ldg(p.cu_q + p.B)) return;
  auto at = [&](int j) { return j * p.Nq * p.Hq + row; };
  const float2 st = lane < p.splits ? p.stats[at(lane)] : make_float2(-INFINITY, 0.f);
  float top = st.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // no maximum: no keys (0), logits that are all -inf (-0), or NaN
  const float share = st.x == -INFINITY ? (st.y == 0.f ? 0.f : NAN) : st.y * exp2_fast(st.x - top);
  const uint32_t with = __ballot_sync(0xffffffffu, st.x != -INFINITY || __float_as_uint(st.y) != 0u);
  float l = share;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  const float weight = l != 0.f ? share / l : with != 0 ? NAN : 0.f;
  float v[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) v[d] = 0.f;
#pragma unroll 4
  for (int j = 0; j < p.splits; ++j) {
    float a[D / 32];
    load_lanes<D>(p.parts + at(j) * D, a);
    const float w = __shfl_sync(0xffffffffu, weight, j);
    if (!(with >> j & 1)) continue;
    // an infinity or NaN of a part whose weight vanishes is seen all the same
#pragma unroll
    for (int d = 0; d < D / 32; ++d) v[d] = fabsf(a[d]) < INFINITY ? fmaf(a[d], w, v[d]) : v[d] + a[d];
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i) store_elem(p.out, token * p.o_token + hq * p.o_head + D / 32 * lane + i, v[i], p.bf16);
  if (p.lse != nullptr && lane == 0) p.lse[row] = prompt_lse(top, l, p.bf16 ? kPromptHeadTc : kPromptHeadFp32);
}

// Rows of a tensor [n, heads, D] that TMA can read: on 16 bytes, and apart.
static bool tma_rows(const void* t, long long token, long long head, long long n, int heads) {
  return ((uintptr_t)t & 15) == 0 && (n <= 1 || (token > 0 && token % 8 == 0)) && (heads <= 1 || (head > 0 && head % 8 == 0));
}

// CTAs share a tile's keys where there are at least two SMs to a tile, at least 512 keys (of all sequences) to one.  32 heads of 128
// over 8 key heads, bf16, us with one CTA to a tile and with two (or more, by the rule):
//   tiles   1024 keys   2048 keys   8192 keys   32768 keys
//     8     23.0 21.8   36.6 22.4   119  28.7   448  51.8
//    40     23.5 26.3   37.5 30.4   121  58.8   455  172
//    72     24.7 30.8   39.0 37.6   122  79.4   461  257
//    80     26.4 43.1   41.6 57.2   128  140    490  480    (not shared)
//   104     25.2 43.3   39.6 56.5   127  141    477  477    (not shared)
//   144                 41.7 62.7   123  145    483  581    (not shared)
// So the limit of two SMs is where it should be for two CTAs; 1024 keys are better not shared by 40 tiles and more.  Not taken: three
// or four CTAs to each of 80 to 110 tiles of 8192 keys and more, in two rounds, 108 and 334 us for 80 of them.
PromptPlan plan_prompt(const PromptParams& p, int sms) {
  PromptPlan plan{};
  const int tokens = (p.bf16 ? 2 : 1) * (128 / p.group);
  const long long tiles = std::max<long long>(1, ((p.Nq + tokens - 1) / tokens + p.B - 1) * p.Hk);   // at most
  plan.splits = (int)std::max<long long>(1, std::min<long long>({sms / tiles, p.Nk / 512, 32}));
  if (plan.splits > 1) {
    plan.parts_bytes = (long long)plan.splits * p.Nq * p.Hq * p.D * 4;
    plan.stats_bytes = ((long long)plan.splits * p.Nq * p.Hq * 8 + 255) / 256 * 256;
  }
  if (!p.bf16) {                       // three bf16 parts of each
    auto parts = [&](long long n, int heads) { return (3 * 2 * n * heads * p.D + 255) / 256 * 256; };
    plan.q_bytes = parts(p.Nq, p.Hq);
    plan.k_bytes = plan.v_bytes = parts(p.Nk, p.Hk);
    return plan;
  }
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

// [parts, tokens, heads, D] as TMA reads it: boxes of 64 dimensions, `heads_box` heads and `tokens_box` tokens of one part.
static CUtensorMap prompt_map(const void* base, int parts, long long token, long long head, long long n, int heads, int D, int heads_box,
                              int tokens_box) {
  const cuuint64_t row = D * 2, dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)n, (cuuint64_t)parts};
  const cuuint64_t strides[3] = {heads > 1 ? (cuuint64_t)head * 2 : row, n > 1 ? (cuuint64_t)token * 2 : row, (cuuint64_t)n * heads * row};
  const cuuint32_t box[4] = {64, (cuuint32_t)heads_box, (cuuint32_t)tokens_box, 1};
  return make_tmap(base, true, parts > 1 ? 4 : 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D>
static void launch_prompt_tc(const PromptParams& p, cudaStream_t s) {
  using C = PromptTc<D>;
  auto kern = prompt_tc_kernel<D>;
  static std::atomic<unsigned long long> configured;   // by device
  configure(kern, C::SMEM, configured);
  const int tokens = 128 / p.group;
  const CUtensorMap tq = prompt_map(p.q, 1, p.q_token, p.q_head, p.Nq, p.Hq, D, p.group, tokens);
  // without keys nothing is loaded; a map has to name something
  const CUtensorMap tk = p.Nk > 0 ? prompt_map(p.k, 1, p.k_token, p.k_head, p.Nk, p.Hk, D, 1, kPromptKeys) : tq;
  const CUtensorMap tv = p.Nk > 0 ? prompt_map(p.v, 1, p.v_token, p.v_head, p.Nk, p.Hk, D, 1, kPromptKeys) : tq;
  const long long tiles = (p.Nq + 2 * tokens - 1) / (2 * tokens) + p.B - 1;   // at most
  launch_with_pdl(kern, dim3((unsigned)(tiles * p.Hk), (unsigned)p.splits), dim3(kPromptThreads), C::SMEM, s, true, tq, tk, tv, p);
}

template <int D>
static void launch_prompt_fp32(const PromptParams& p, const PromptPlan& plan, char* ws, cudaStream_t s) {
  using C = PromptFp32<D>;
  auto kern = prompt_fp32_kernel<D>;
  static std::atomic<unsigned long long> configured;   // by device
  configure(kern, C::SMEM, configured);
  auto tensor = [&](const void* t, long long token, long long head, long long n, int heads) {
    const bool vec = (((uintptr_t)t | (token * 4) | (head * 4)) & 15) == 0;
    SplitTensor x{(const float*)t, token, head, n, (__nv_bfloat16*)ws, heads, vec};
    ws += (3 * 2 * n * heads * D + 255) / 256 * 256;
    return x;
  };
  const SplitTensor q = tensor(p.q, p.q_token, p.q_head, p.Nq, p.Hq), k = tensor(p.k, p.k_token, p.k_head, p.Nk, p.Hk),
                    v = tensor(p.v, p.v_token, p.v_head, p.Nk, p.Hk);
  const long long most = std::max(p.Nq * p.Hq, p.Nk * p.Hk) * D / 2048 + 1;
  launch_with_pdl(prompt_split_kernel<D>, dim3((unsigned)std::min<long long>(most, 8ll * serving_sm_count()), 3), dim3(256), 0, s, true, q, k, v);
  const int tokens = 128 / p.group;
  auto map = [&](const SplitTensor& x, int heads_box, int tokens_box) {
    return prompt_map(x.dst, 3, (long long)x.heads * D, D, x.n, x.heads, D, heads_box, tokens_box);
  };
  const CUtensorMap tq = map(q, p.group, tokens), tk = p.Nk > 0 ? map(k, 1, C::KT) : tq, tv = p.Nk > 0 ? map(v, 1, C::KT) : tq;
  const long long tiles = (p.Nq + tokens - 1) / tokens + p.B - 1;   // at most
  launch_with_pdl(kern, dim3((unsigned)(tiles * p.Hk), (unsigned)p.splits), dim3(kFp32Threads), C::SMEM, s, true, tq, tk, tv, p);
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
    if (p.D == 128) launch_prompt_fp32<128>(p, plan, ws, s);
    else launch_prompt_fp32<64>(p, plan, ws, s);
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
