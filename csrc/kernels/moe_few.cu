// A whole mixture-of-experts layer for a few tokens (1 to 64): one decode step
// of a served model.  The progressive layer handles thousands of tokens per
// call, chunk by chunk; here every cost but reading the chosen experts'
// weights once is overhead.
//
//   l[t, e] = x[t] . Wr[e] + br[e]           blocked experts: -inf
//   ids[t]  = the k largest (larger value, then smaller expert; NaN last)
//   g[t]    = 1, softmax over the chosen, or softmax over all
//   out[t]  = sum_j g[t, j] (W2[e] act(W1[e] x[t] + b1[e]) + b2[e]) + residual[t],  e = ids[t, j]
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <stdexcept>

#include "moe_few_tc.cuh"
#include "serving.h"
#include "serving_device.cuh"
#include "serving_tma.h"
#include "sm100_ptx.cuh"

namespace cg = cooperative_groups;

namespace raiccl {

__device__ DeviceStatus g_serving_status;

static int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev & 63;
}

DeviceStatus* serving_status() {
  static std::atomic<void*> at[64];
  const int dev = current_device();
  void* p = at[dev].load();
  if (p == nullptr) {
    if (cudaGetSymbolAddress(&p, g_serving_status) != cudaSuccess) throw std::runtime_error("serving operators: no device status");
    at[dev].store(p);
  }
  return (DeviceStatus*)p;
}

// ---------------------------------------------------------------------------
// Routing: one cluster per token, its CTAs and their warps share the experts.
// ---------------------------------------------------------------------------
constexpr int kRouteThreads = 256;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteCuts = 8;
static_assert(kRouteThreads > kFewExperts, "a thread per expert");

// Sort key, larger = preferred: 0 for no candidate (blocked, or a logit of
// -inf), then NaN, then numbers by value (an order-preserving map of the float
// bits, -0 taken as +0); among equals the smaller expert.
__device__ __forceinline__ unsigned long long few_key(float v, int e) {
  if (v == -INFINITY) return 0ull;
  if (v != v) return (1ull << 40) | (unsigned long long)(255 - e);
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
  const uint32_t u = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (2ull << 40) | ((unsigned long long)u << 8) | (unsigned long long)(255 - e);
}

// x . w over vectors (elements where rows are not aligned) [i0, i1) by one
// warp, in 32 bits: each lane adds its vectors' partial sums, a butterfly adds
// the lanes.
template <typename T>
__device__ __forceinline__ float route_dot(const T* x, const T* w, int i0, int i1, int vec) {
  const int lane = threadIdx.x & 31;
  float acc = 0.f;
  if (vec) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll 8
    for (int i = i0 + lane; i < i1; i += 32) {
      const uint4 xr = __ldg((const uint4*)x + i);
      const uint4 wr = __ldg((const uint4*)w + i);
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) s = fmaf(as_float(((const T*)&xr)[v]), as_float(((const T*)&wr)[v]), s);
      acc += s;
    }
  } else {
#pragma unroll 8
    for (int i = i0 + lane; i < i1; i += 32) acc = fmaf(as_float(x[i]), as_float(w[i]), acc);
  }
  return warp_sum(acc);
}

// One cluster per token.  The experts' rows, cut into `cuts` pieces each, are
// dealt to the warps of its CTAs; the first CTA adds the pieces in order and
// finds each expert's rank among all (the number of experts with a larger key),
// so the choices need no rounds.
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) few_route_kernel(FewRouteParams p) {
  __shared__ float piece[kRouteCuts][kFewExperts + 1];
  __shared__ float logits[kFewExperts + 1];
  __shared__ unsigned long long keys[kFewExperts + 1];
  __shared__ int chosen[kFewTopK];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int t = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = (const T*)p.x + (long long)t * p.x_stride;
  float* lead = cluster.map_shared_rank(&piece[0][0], 0);
  griddep_wait();
  griddep_launch_dependents();
  if (p.packed) {
    const int share = rank * kRouteThreads + threadIdx.x, shares = ranks * kRouteThreads;
    for (int d = share; d < p.D; d += shares) {
      if constexpr (sizeof(T) == 4) {
        float* at = (float*)p.packed + (long long)t * p.packed_stride + d;
        split_tf32(x[d], at[0], at[(long long)p.packed_rows * p.packed_stride]);
      } else {
        ((T*)p.packed)[(long long)t * p.packed_stride + d] = x[d];
      }
    }
  }
  const int n = p.vec ? p.D * (int)sizeof(T) / 16 : p.D;   // vectors (elements) of a row
  const int per = (n + p.cuts - 1) / p.cuts;
  for (int i = warp * ranks + rank; i < p.E * p.cuts; i += kRouteWarps * ranks) {
    const int e = i / p.cuts, c = i - e * p.cuts;
    const int i0 = c * per, i1 = i0 + per < n ? i0 + per : n;
    const float v = route_dot(x, (const T*)p.w + (long long)e * p.w_stride, i0, i1, p.vec);
    if (lane == 0) lead[c * (kFewExperts + 1) + e] = v;
  }
  cluster.sync();
  if (rank != 0) return;
  const int e = threadIdx.x;   // kRouteThreads > kFewExperts
  unsigned long long key = 0ull;
  if (e < p.E) {
    float v = piece[0][e];
    for (int c = 1; c < p.cuts; ++c) v += piece[c][e];
    if (p.bias) v += p.bias[e];
    if (p.mask && p.mask[(long long)t * p.mask_stride + e]) v = -INFINITY;
    logits[e] = v;
    keys[e] = key = few_key(v, e);
  }
  if (e < kFewTopK) chosen[e] = -1;
  __syncthreads();
  if (key != 0ull) {
    int above = 0;
#pragma unroll 8
    for (int o = 0; o < p.E; ++o) above += keys[o] > key ? 1 : 0;
    if (above < p.k) chosen[above] = e;
  }
  __syncthreads();
  if (warp != 0) return;
  const int mine = lane < p.k ? chosen[lane] : -1;   // lane j: choice j
  const float top = mine < 0 ? 0.f : logits[mine];
  float gate = mine < 0 ? 0.f : 1.f;
  if (p.gate_mode != 0) {
    const float peak = __shfl_sync(0xffffffffu, top, 0);  // the largest number, or NaN if there is none
    float part = 0.f;
    if (p.gate_mode == 1) {
      part = mine < 0 ? 0.f : expf(top - peak);
    } else {
      for (int o = lane; o < p.E; o += 32) part += logits[o] == -INFINITY ? 0.f : expf(logits[o] - peak);
    }
    const float total = warp_sum(part);
    if (mine >= 0) gate = expf(top - peak) / total;
  }
  if (lane < p.k) {
    p.ids[(long long)t * p.k + lane] = mine;
    p.gates[(long long)t * p.k + lane] = gate;
  }
}

void launch_few_route(const FewRouteParams& params, cudaStream_t s) {
  // Pieces of a row so that the cluster's warps have one each, down to one
  // vector per lane; clusters of eight CTAs at most.
  FewRouteParams p = params;
  const int n = p.vec ? p.D * (p.bf16 ? 2 : 4) / 16 : p.D;
  p.cuts = std::max(1, std::min({kRouteCuts, 8 * kRouteWarps / p.E, n / 32}));
  const int want = (p.E * p.cuts + kRouteWarps - 1) / kRouteWarps;
  const int ranks = want > 4 ? 8 : want > 2 ? 4 : want;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, p.T);
  cfg.blockDim = dim3(kRouteThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (p.bf16) cudaLaunchKernelEx(&cfg, few_route_kernel<__nv_bfloat16>, p);
  else cudaLaunchKernelEx(&cfg, few_route_kernel<float>, p);
}

// ---------------------------------------------------------------------------
// Experts: one warp per weight row and expert; a row is read once for up to
// eight of the expert's tokens at a time.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;
constexpr int kRowTokens = 8;

// The expert's (token, choice) pairs t k + j in token order -> list; returns their number.
__device__ __forceinline__ int few_pairs(const int* ids, int T, int k, int e, int* list) {
  __shared__ unsigned long long mask;
  if (threadIdx.x == 0) mask = 0ull;
  __syncthreads();
  for (int i = threadIdx.x; i < T * k; i += blockDim.x)
    if (ids[i] == e) atomicOr(&mask, 1ull << (i / k));
  __syncthreads();
  const unsigned long long m = mask;
  for (int i = threadIdx.x; i < T * k; i += blockDim.x)
    if (ids[i] == e) list[__popcll(m & ((1ull << (i / k)) - 1ull))] = i;
  __syncthreads();
  return __popcll(m);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) few_hidden_kernel(FewExpertParams p, float* h) {
  __shared__ int list[kFewTokens];
  const int e = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = few_pairs(p.ids, p.T, p.k, e, list);
  const int f = blockIdx.x * (kRowThreads / 32) + warp;
  if (n == 0 || f >= p.F) return;
  const bool glu = p.act == (int)Act::kSwiGLU;
  const T* wg = (const T*)p.w1 + (long long)e * p.w1_estride + (long long)f * p.w1_stride;
  const T* wu = wg + (long long)p.F * p.w1_stride;
  for (int i0 = 0; i0 < n; i0 += kRowTokens) {
    float g[kRowTokens] = {}, u[kRowTokens] = {};
    const T* x[kRowTokens];
    for (int i = 0; i < kRowTokens; ++i)
      x[i] = (const T*)p.x + (long long)(list[min(i0 + i, n - 1)] / p.k) * p.x_stride;
    for (int d = lane; d < p.D; d += 32) {
      const float a = as_float(wg[d]), b = glu ? as_float(wu[d]) : 0.f;
#pragma unroll
      for (int i = 0; i < kRowTokens; ++i) {
        const float v = as_float(x[i][d]);
        g[i] = fmaf(a, v, g[i]);
        if (glu) u[i] = fmaf(b, v, u[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < kRowTokens; ++i) {
      g[i] = warp_sum(g[i]);
      u[i] = warp_sum(u[i]);
      if (lane == 0 && i0 + i < n) {
        const float* b1 = p.b1 ? p.b1 + (long long)e * (glu ? 2 : 1) * p.F : nullptr;
        const float z = g[i] + (b1 ? b1[f] : 0.f);
        h[(long long)list[i0 + i] * p.F + f] =
            glu ? serving_swiglu(z, u[i] + (b1 ? b1[p.F + f] : 0.f)) : serving_act(z, p.act);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) few_output_kernel(FewExpertParams p, const float* hidden, float* y) {
  __shared__ int list[kFewTokens];
  const int e = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = few_pairs(p.ids, p.T, p.k, e, list);
  const int o = blockIdx.x * (kRowThreads / 32) + warp;
  if (n == 0 || o >= p.O) return;
  const T* w = (const T*)p.w2 + (long long)e * p.w2_estride + (long long)o * p.w2_stride;
  for (int i0 = 0; i0 < n; i0 += kRowTokens) {
    float acc[kRowTokens] = {};
    const float* h[kRowTokens];
    for (int i = 0; i < kRowTokens; ++i) h[i] = hidden + (long long)list[min(i0 + i, n - 1)] * p.F;
    for (int f = lane; f < p.F; f += 32) {
      const float a = as_float(w[f]);
#pragma unroll
      for (int i = 0; i < kRowTokens; ++i) acc[i] = fmaf(a, h[i][f], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < kRowTokens; ++i) {
      acc[i] = warp_sum(acc[i]);
      if (lane == 0 && i0 + i < n)
        y[(long long)list[i0 + i] * p.O + o] = acc[i] + (p.b2 ? p.b2[(long long)e * p.O + o] : 0.f);
    }
  }
}

__global__ void __launch_bounds__(kRowThreads) few_join_kernel(FewExpertParams p, const float* y) {
  const long long i = (long long)blockIdx.x * kRowThreads + threadIdx.x;
  if (i >= (long long)p.T * p.O) return;
  const int t = (int)(i / p.O), o = (int)(i % p.O);
  float acc = 0.f;
  for (int j = 0; j < p.k; ++j)
    if (p.ids[t * p.k + j] >= 0) acc = fmaf(p.gates[t * p.k + j], y[(long long)(t * p.k + j) * p.O + o], acc);
  if (p.residual) acc += load_elem(p.residual, (long long)t * p.res_stride + o, p.res_bf16);
  store_elem(p.out, (long long)t * p.out_stride + o, acc, p.out_bf16);
}

template <typename T>
static void launch_rows(const FewExpertParams& p, float* h, float* y, cudaStream_t s) {
  constexpr int W = kRowThreads / 32;
  few_hidden_kernel<T><<<dim3((p.F + W - 1) / W, p.E), kRowThreads, 0, s>>>(p, h);
  few_output_kernel<T><<<dim3((p.O + W - 1) / W, p.E), kRowThreads, 0, s>>>(p, h, y);
  few_join_kernel<<<(unsigned)(((long long)p.T * p.O + kRowThreads - 1) / kRowThreads), kRowThreads, 0, s>>>(p, y);
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------
int serving_sm_count() {
  static std::atomic<int> n[64];
  const int dev = current_device();
  int v = n[dev].load();
  if (v == 0) {
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1)
      throw std::runtime_error("serving operators: no SM count");
    n[dev].store(v);
  }
  return v;
}

static long long up256(long long v) { return (v + 255) / 256 * 256; }

constexpr int kFewShared = 232448 - 10 * 1024 - 1024;  // dynamic shared memory besides the kernel's own and the alignment
constexpr int kFewJoinRoom = 24 * 1024;                // of the join's CTA beside it

FewExpertPlan plan_few_experts(const FewExpertParams& p) {
  FewExpertPlan r{};
  const int eb = p.bf16 ? 2 : 4, parts = p.bf16 ? 1 : 2;
  auto aligned = [&](const void* base, long long row, long long expert) {
    return ((uintptr_t)base & 15) == 0 && (row * eb) % 16 == 0 && (p.E == 1 || (expert * eb) % 16 == 0);
  };
  // TMA reads rows that start on 16 bytes
  r.tensor = aligned(p.w1, p.w1_stride, p.w1_estride) && aligned(p.w2, p.w2_stride, p.w2_estride);
  const int pairs = p.T * p.k;
  if (!r.tensor) {
    r.a_bytes = up256((long long)pairs * p.F * 4);
    r.b_bytes = up256((long long)pairs * p.O * 4);
    return r;
  }
  r.grid = serving_sm_count();
  r.Op = (p.O + 127) / 128 * 128;
  r.Tp = (p.T + 15) / 16 * 16;
  const int UE = (p.F + 15) / 16, ups = 128 / eb / 16;
  r.pack = !p.bf16 || !aligned(p.x, p.T > 1 ? p.x_stride : 0, 0);
  r.packed_stride = (p.D + 7) / 8 * 8;
  if (r.pack) r.packed_bytes = up256((long long)parts * r.Tp * r.packed_stride * eb);
  // An expert's tokens times the CTAs that share it, over all experts: n experts have at most min(T k, n T) tokens
  // and (grid / n + 2) CTAs each, so T (grid + 2 k) rows at most, whatever n is.
  r.a_bytes = up256((long long)p.T * (r.grid + 2 * p.k) * r.Op * 4);
  // Activations of the longest range of a CTA, if that leaves four stages; else the range is worked off in pieces, which
  // costs a sum in memory each.  The rest holds stages.
  const int sb = p.bf16 ? FewTc<false>::stage_bytes(r.Tp) : FewTc<true>::stage_bytes(r.Tp);
  // Up to 16 tokens the join's CTAs find room beside the experts' (64 experts, 1 token: 49.7 -> 43.5 us); with more, the
  // stages are worth more (37 tokens: 193 against 196 us).
  const int room = kFewShared - (p.T <= 16 ? kFewJoinRoom : 0) - (p.bf16 ? 0 : FewTc<true>::low_bytes());
  const long long most = ((long long)std::min(p.E, pairs) * UE + r.grid - 1) / r.grid;
  const long long rows = (std::min<long long>(most, UE) + ups - 1) / ups + 1;
  r.hbytes = (int)std::min<long long>(rows * parts * r.Tp * 128, room - 4 * sb);
  r.hbytes = std::max({r.hbytes, parts * r.Tp * 128, kFewSlack});
  r.stages = std::min(kFewMaxStages, (room - r.hbytes) / sb);
  return r;
}

template <bool FP32, bool GLU>
static void launch_tensor(const CUtensorMap& tx, const CUtensorMap& t1, const CUtensorMap& t1w, const CUtensorMap& t2,
                          const CUtensorMap& t2u, const FewTcParams& tp, int grid, cudaStream_t s) {
  auto kern = few_experts_kernel<FP32, GLU>;
  static std::atomic<unsigned long long> configured;  // by device
  const unsigned long long bit = 1ull << current_device();
  if (!(configured.load() & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewShared + 1024) != cudaSuccess)
      throw std::runtime_error("moe_few_tokens: shared memory");
    configured.fetch_or(bit);
  }
  const size_t smem = 1024 + (size_t)tp.stages * FewTc<FP32>::stage_bytes(tp.Tp) + FewTc<FP32>::low_bytes() + tp.hbytes;
  launch_with_pdl(kern, dim3(grid), dim3(FewTc<FP32>::THREADS), smem, s, true, tx, t1, t1w, t2, t2u, tp, serving_status());
}

void launch_few_experts(const FewExpertParams& p, const FewExpertPlan& plan, void* workspace, cudaStream_t s) {
  char* ws = (char*)workspace;
  float* a = (float*)(ws + plan.packed_bytes);
  float* b = (float*)(ws + plan.packed_bytes + plan.a_bytes);
  if (!plan.tensor) {
    if (p.bf16) launch_rows<__nv_bfloat16>(p, a, b, s);
    else launch_rows<float>(p, a, b, s);
    return;
  }
  const cuuint64_t eb = p.bf16 ? 2 : 4;
  const cuuint32_t bk = 128 / eb;
  const int parts = p.bf16 ? 1 : 2;
  const bool glu = p.act == (int)Act::kSwiGLU, wide = !glu || p.F % 16 == 0;
  const cuuint64_t D = p.D, F = p.F, O = p.O, E = p.E;
  // a stride along a single expert or token is never used
  const cuuint64_t e1 = p.E > 1 ? p.w1_estride * eb : 16, e2 = p.E > 1 ? p.w2_estride * eb : 16;
  CUtensorMap tx, t1, t1w, t2, t2u;
  {
    const cuuint64_t dims[2] = {D, plan.pack ? (cuuint64_t)parts * plan.Tp : (cuuint64_t)p.T};
    const cuuint64_t strides[1] = {plan.pack ? plan.packed_stride * eb : p.T > 1 ? p.x_stride * eb : (D * eb + 15) / 16 * 16};
    const cuuint32_t box[2] = {bk, (cuuint32_t)(parts * plan.Tp)};
    tx = make_tmap(plan.pack ? ws : p.x, p.bf16, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (glu) {
    const cuuint64_t dims[4] = {D, F, 2, E};
    const cuuint64_t strides[3] = {p.w1_stride * eb, F * p.w1_stride * eb, e1};
    const cuuint32_t box[4] = {bk, 16, 2, 1};
    t1 = t1w = make_tmap(p.w1, p.bf16, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (wide) {  // 16 rows of F by gate and up by four of these groups: the order of a tile's rows
      const cuuint64_t dims[5] = {D, 16, 2, F / 16, E};
      const cuuint64_t strides[4] = {p.w1_stride * eb, F * p.w1_stride * eb, 16 * p.w1_stride * eb, e1};
      const cuuint32_t box[5] = {bk, 16, 2, 4, 1};
      t1w = make_tmap(p.w1, p.bf16, 5, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    }
  } else {
    const cuuint64_t dims[3] = {D, F, E};
    const cuuint64_t strides[2] = {p.w1_stride * eb, e1};
    const cuuint32_t box[3] = {bk, 16, 1}, tile[3] = {bk, 128, 1};
    t1 = make_tmap(p.w1, p.bf16, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    t1w = make_tmap(p.w1, p.bf16, 3, dims, strides, tile, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  {
    const cuuint64_t dims[3] = {F, O, E};
    const cuuint64_t strides[2] = {p.w2_stride * eb, e2};
    const cuuint32_t box[3] = {bk, 128, 1}, unit[3] = {16, 128, 1};
    t2 = make_tmap(p.w2, p.bf16, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    t2u = make_tmap(p.w2, p.bf16, 3, dims, strides, unit, p.bf16 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_64B);
  }
  FewTcParams tp{};
  tp.e = p;
  tp.part = a;
  tp.grid = plan.grid;
  tp.Op = plan.Op;
  tp.Tp = plan.Tp;
  tp.stages = plan.stages;
  tp.hbytes = plan.hbytes;
  tp.wide = wide;
  if (p.bf16) {
    if (glu) launch_tensor<false, true>(tx, t1, t1w, t2, t2u, tp, plan.grid, s);
    else launch_tensor<false, false>(tx, t1, t1w, t2, t2u, tp, plan.grid, s);
  } else {
    if (glu) launch_tensor<true, true>(tx, t1, t1w, t2, t2u, tp, plan.grid, s);
    else launch_tensor<true, false>(tx, t1, t1w, t2, t2u, tp, plan.grid, s);
  }
  launch_with_pdl(few_join_parts_kernel, dim3(plan.Op / 128, p.T), dim3(kFewJoinThreads), 0, s, true, tp);
}

}  // namespace raiccl
