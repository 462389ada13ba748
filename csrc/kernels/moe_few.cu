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

// What a CTA holds of a token's routing.
struct FewRoute {
  float piece[kRouteCuts][kFewExperts + 1];
  float logits[kFewExperts + 1];
  unsigned long long keys[kFewExperts + 1];
  int chosen[kFewTopK];
};

// The experts' rows, cut into `cuts` pieces each, are dealt to warps: warp `at` of `of`.
template <typename T>
__device__ __forceinline__ void route_pieces(const FewRouteParams& p, const T* x, float* piece, int at, int of) {
  const int n = p.vec ? p.D * (int)sizeof(T) / 16 : p.D;   // vectors (elements) of a row
  const int per = (n + p.cuts - 1) / p.cuts;
  for (int i = at; i < p.E * p.cuts; i += of) {
    const int e = i / p.cuts, c = i - e * p.cuts;
    const int i0 = c * per, i1 = i0 + per < n ? i0 + per : n;
    const float v = route_dot(x, (const T*)p.w + (long long)e * p.w_stride, i0, i1, p.vec);
    if ((threadIdx.x & 31) == 0) piece[c * (kFewExperts + 1) + e] = v;
  }
}

// Adds the pieces in order and finds each expert's rank among all (the number
// of experts with a larger key), so the choices need no rounds.
__device__ __forceinline__ void route_choose(const FewRouteParams& p, FewRoute& s, int t) {
  const int e = threadIdx.x;   // kRouteThreads > kFewExperts
  unsigned long long key = 0ull;
  if (e < p.E) {
    float v = s.piece[0][e];
    for (int c = 1; c < p.cuts; ++c) v += s.piece[c][e];
    if (p.bias) v += p.bias[e];
    if (p.mask && p.mask[(long long)t * p.mask_stride + e]) v = -INFINITY;
    s.logits[e] = v;
    s.keys[e] = key = few_key(v, e);
  }
  if (e < kFewTopK) s.chosen[e] = -1;
  __syncthreads();
  if (key != 0ull) {
    int above = 0;
#pragma unroll 8
    for (int o = 0; o < p.E; ++o) above += s.keys[o] > key ? 1 : 0;
    if (above < p.k) s.chosen[above] = e;
  }
  __syncthreads();
}

// By one warp: the choices and gates of the token.
__device__ __forceinline__ void route_write(const FewRouteParams& p, const FewRoute& s, int t) {
  const int lane = threadIdx.x & 31;
  const int mine = lane < p.k ? s.chosen[lane] : -1;   // lane j: choice j
  const float top = mine < 0 ? 0.f : s.logits[mine];
  float gate = mine < 0 ? 0.f : 1.f;
  if (p.gate_mode != 0) {
    const float peak = __shfl_sync(0xffffffffu, top, 0);  // the largest number, or NaN if there is none
    float part = 0.f;
    if (p.gate_mode == 1) {
      part = mine < 0 ? 0.f : expf(top - peak);
    } else {
      for (int o = lane; o < p.E; o += 32) part += s.logits[o] == -INFINITY ? 0.f : expf(s.logits[o] - peak);
    }
    const float total = warp_sum(part);
    if (mine >= 0) gate = expf(top - peak) / total;
  }
  if (lane < p.k) {
    p.ids[(long long)t * p.k + lane] = mine;
    p.gates[(long long)t * p.k + lane] = gate;
  }
}

// One cluster per token: its CTAs share the pieces, the first one chooses.
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) few_route_kernel(FewRouteParams p) {
  __shared__ FewRoute s;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int t = blockIdx.y;
  const T* x = (const T*)p.x + (long long)t * p.x_stride;
  float* lead = cluster.map_shared_rank(&s.piece[0][0], 0);
  cluster.barrier_arrive();   // of the CTAs that write to the first one's shared memory: it has begun
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
  cluster.barrier_wait();
  route_pieces(p, x, lead, (threadIdx.x >> 5) * ranks + rank, kRouteWarps * ranks);
  cluster.sync();
  if (rank != 0) return;
  route_choose(p, s, t);
  if (threadIdx.x < 32) route_write(p, s, t);
}

// Pieces of a row so that `warps` warps have one each, down to one vector per lane.
static int route_cuts(const FewRouteParams& p, int warps) {
  const int n = p.vec ? p.D * (p.bf16 ? 2 : 4) / 16 : p.D;
  return std::max(1, std::min({kRouteCuts, warps / p.E, n / 32}));
}

static void launch_route(const FewRouteParams& params, cudaStream_t s) {
  FewRouteParams p = params;
  p.cuts = route_cuts(p, 8 * kRouteWarps);   // clusters of eight CTAs at most
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
// Experts by rows, on CUDA cores: for the smallest calls, where a pipeline's
// start costs more than it brings, and for weights that TMA cannot read.  One
// warp per pair of W1 rows and per row of W2; fp32 sums, activations in fp32.
// What bounds the large ones is memory (24 loads of 16 bytes in flight per
// lane): 64 experts, 1 token (104 MB) 42 us, against 34 by tensor cores; the
// small ones are two or three launches and their first loads: 4 experts, 2048 to
// 32 to 16 fp32, 1 token 8.3 us in a graph, against 32.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;

// An expert's (token, choice) pairs in token order go four to a CTA: that of the
// pair `y` takes list[0 .. n) if it is the first of its four, else none.
constexpr int kRowTokens = 4;

__device__ __forceinline__ int few_pairs(const int* ids, int T, int k, int y, int* list, int& e) {
  __shared__ unsigned long long mask;
  if (threadIdx.x == 0) mask = 0ull;
  e = __ldcg(ids + y);
  if (e < 0) return 0;
  __syncthreads();
  for (int i = threadIdx.x; i < T * k; i += blockDim.x)
    if (__ldcg(ids + i) == e) atomicOr(&mask, 1ull << (i / k));
  __syncthreads();
  const unsigned long long m = mask;
  const int first = __popcll(m & ((1ull << (y / k)) - 1ull)), n = __popcll(m) - first;
  if (first % kRowTokens != 0) return 0;
  for (int i = threadIdx.x; i < T * k; i += blockDim.x)
    if (__ldcg(ids + i) == e) {
      const int at = __popcll(m & ((1ull << (i / k)) - 1ull)) - first;
      if (at >= 0 && at < kRowTokens) list[at] = i;
    }
  __syncthreads();
  return n < kRowTokens ? n : kRowTokens;
}

// Two rows of W1 against NT of the expert's tokens, pairs list[0 .. n): h[pair, f] = act(W1[e] x + b1).
template <typename T, bool VEC, int NT>
__device__ __forceinline__ void few_hidden_rows(const FewExpertParams& p, float* h, const int* list, int n, int e, int f, bool glu) {
  const int lane = threadIdx.x & 31;
  const bool two = glu || f + 1 < p.F;
  const T* wa = (const T*)p.w1 + (long long)e * p.w1_estride + (long long)f * p.w1_stride;
  const T* wb = !two ? wa : wa + (glu ? p.F : 1) * p.w1_stride;
  float a[NT] = {}, b[NT] = {};
  const T* x[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) x[i] = (const T*)p.x + (long long)(list[i < n ? i : n - 1] / p.k) * p.x_stride;
  if constexpr (VEC) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll(NT == 1 ? 8 : 4)
    for (int d = lane * V; d < p.D; d += 32 * V) {
      float fa[V], fb[V], fx[V];
      unpack16<T>(__ldg((const uint4*)(wa + d)), fa);
      unpack16<T>(__ldg((const uint4*)(wb + d)), fb);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        unpack16<T>(__ldg((const uint4*)(x[i] + d)), fx);
        float sa = 0.f, sb = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          sa = fmaf(fa[v], fx[v], sa);
          sb = fmaf(fb[v], fx[v], sb);
        }
        a[i] += sa;
        b[i] += sb;
      }
    }
  } else {
#pragma unroll(NT == 1 ? 8 : 4)
    for (int d = lane; d < p.D; d += 32) {
      const float fa = as_float(wa[d]), fb = as_float(wb[d]);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float fx = as_float(x[i][d]);
        a[i] = fmaf(fa, fx, a[i]);
        b[i] = fmaf(fb, fx, b[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    a[i] = warp_sum(a[i]);
    b[i] = warp_sum(b[i]);
    if (lane == 0 && i < n) {
      const float* b1 = p.b1 ? p.b1 + (long long)e * (glu ? 2 : 1) * p.F : nullptr;
      float* at = h + (long long)list[i] * p.F + f;
      const float za = a[i] + (b1 ? b1[f] : 0.f);
      const float zb = b[i] + (b1 && two ? b1[glu ? p.F + f : f + 1] : 0.f);
      at[0] = glu ? serving_swiglu(za, zb) : serving_act(za, p.act);
      if (!glu && two) at[1] = serving_act(zb, p.act);
    }
  }
}

// ROUTE: every CTA routes the call's one token for itself, and the first one writes its choices and gates.
template <typename T, bool VEC, bool ROUTE>
__global__ void __launch_bounds__(kRowThreads) few_hidden_kernel(FewExpertParams p, float* h, FewRouteParams r) {
  __shared__ int list[kRowTokens];
  const bool glu = p.act == (int)Act::kSwiGLU;
  griddep_wait();
  griddep_launch_dependents();
  int e, n;
  if constexpr (ROUTE) {
    __shared__ FewRoute s;
    route_pieces(r, (const T*)r.x, &s.piece[0][0], threadIdx.x >> 5, kRowWarps);
    __syncthreads();
    if (threadIdx.x == 0) list[0] = blockIdx.y;
    route_choose(r, s, 0);
    if ((blockIdx.x | blockIdx.y) == 0 && threadIdx.x < 32) route_write(r, s, 0);
    e = s.chosen[blockIdx.y];
    n = e < 0 ? 0 : 1;
  } else {
    n = few_pairs(p.ids, p.T, p.k, blockIdx.y, list, e);
  }
  const int f = (blockIdx.x * kRowWarps + (threadIdx.x >> 5)) * (glu ? 1 : 2);   // rows f and F + f, or f and f + 1
  if (n == 0 || f >= p.F) return;
  if (ROUTE || n == 1) few_hidden_rows<T, VEC, 1>(p, h, list, 1, e, f, glu);
  else few_hidden_rows<T, VEC, kRowTokens>(p, h, list, n, e, f, glu);
}

// out[t, o] = sum_j gate (W2[e] h[t, j] + b2[e]) + residual, four o to a CTA: its
// warps share the choices and, where these are fewer than the warps, their F.
constexpr int kOutRows = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kRowThreads) few_output_kernel(FewExpertParams p, const float* h) {
  __shared__ float part[kRowWarps][kOutRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = blockIdx.y;
  const int o0 = blockIdx.x * kOutRows;
  const int pieces = kRowWarps / p.k, j = warp % p.k, piece = warp / p.k;
  griddep_wait();
  griddep_launch_dependents();
  float acc[kOutRows] = {};
  const int e = piece < pieces ? __ldcg(p.ids + t * p.k + j) : -1;
  if (e >= 0) {
    const T* w = (const T*)p.w2 + (long long)e * p.w2_estride;
    const T* row[kOutRows];
#pragma unroll
    for (int r = 0; r < kOutRows; ++r) row[r] = w + (long long)(o0 + r < p.O ? o0 + r : p.O - 1) * p.w2_stride;
    const float* hj = h + (long long)(t * p.k + j) * p.F;
    constexpr int V = VEC ? 16 / sizeof(T) : 1;
    const int n = p.F / V, i1 = (int)((long long)n * (piece + 1) / pieces);
    if constexpr (VEC) {
#pragma unroll 4
      for (int i = (int)((long long)n * piece / pieces) + lane; i < i1; i += 32) {
        float fh[V];
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
          const float4 v = __ldcg((const float4*)(hj + i * V) + q);
          fh[4 * q] = v.x; fh[4 * q + 1] = v.y; fh[4 * q + 2] = v.z; fh[4 * q + 3] = v.w;
        }
#pragma unroll
        for (int r = 0; r < kOutRows; ++r) {
          float fw[V], s = 0.f;
          unpack16<T>(__ldg((const uint4*)row[r] + i), fw);
#pragma unroll
          for (int v = 0; v < V; ++v) s = fmaf(fw[v], fh[v], s);
          acc[r] += s;
        }
      }
    } else {
#pragma unroll 4
      for (int i = (int)((long long)n * piece / pieces) + lane; i < i1; i += 32) {
        const float fh = __ldcg(hj + i);
#pragma unroll
        for (int r = 0; r < kOutRows; ++r) acc[r] = fmaf(as_float(row[r][i]), fh, acc[r]);
      }
    }
  }
  const float g = e >= 0 ? __ldcg(p.gates + t * p.k + j) : 0.f;
#pragma unroll
  for (int r = 0; r < kOutRows; ++r) {
    acc[r] = warp_sum(acc[r]);
    if (lane == r) {
      float v = acc[r];
      if (e >= 0 && piece == 0 && p.b2 && o0 + r < p.O) v += __ldg(p.b2 + (long long)e * p.O + o0 + r);
      part[warp][r] = e >= 0 ? g * v : 0.f;
    }
  }
  __syncthreads();
  const int o = o0 + threadIdx.x;
  if (threadIdx.x >= kOutRows || o >= p.O) return;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < kRowWarps; ++i) v += part[i][threadIdx.x];
  if (p.residual) v += load_elem(p.residual, (long long)t * p.res_stride + o, p.res_bf16);
  store_elem(p.out, (long long)t * p.out_stride + o, v, p.out_bf16);
}

template <typename T, bool VEC>
static void launch_rows_vec(const FewExpertParams& p, const FewRouteParams& route, bool own, float* h, cudaStream_t s) {
  const int per = kRowWarps * (p.act == (int)Act::kSwiGLU ? 1 : 2);
  const dim3 grid((p.F + per - 1) / per, p.T * p.k);
  FewRouteParams r = route;
  r.cuts = route_cuts(r, kRowWarps);
  if (own) launch_with_pdl(few_hidden_kernel<T, VEC, true>, grid, dim3(kRowThreads), 0, s, true, p, h, r);
  else launch_with_pdl(few_hidden_kernel<T, VEC, false>, grid, dim3(kRowThreads), 0, s, true, p, h, r);
  launch_with_pdl(few_output_kernel<T, VEC>, dim3((p.O + kOutRows - 1) / kOutRows, p.T), dim3(kRowThreads), 0, s, true, p,
                  (const float*)h);
}

template <typename T>
static void launch_rows(const FewExpertParams& p, const FewRouteParams& r, const FewExpertPlan& plan, float* h, cudaStream_t s) {
  if (plan.vec) launch_rows_vec<T, true>(p, r, plan.route != 0, h, s);
  else launch_rows_vec<T, false>(p, r, plan.route != 0, h, s);
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
static long long up8(long long v) { return (v + 7) / 8 * 8; }

constexpr int kFewShared = 232448 - 10 * 1024 - 1024;  // dynamic shared memory besides the kernel's own and the alignment
// By rows up to so many bytes of weights, counted once for each (token, choice).  Measured, rows against tensor cores (us):
// bf16 64 experts 512 x 352, 1 token (6.5 MB) 11 / 17, 4 tokens (26 MB) 21 / 21, 32 experts 1024 x 1024, 2 tokens (50 MB)
// 29 / 26; fp32 8 experts 1024 x 4096, 1 token (67 MB) 20 / 42, 4 (268 MB) 46 / 72, 8 (537 MB) 77 / 80, 12 105 / 81.
constexpr double kFewRowBytes = 30e6, kFewRowBytesFp32 = 540e6;
// One token: with few experts every CTA routes for itself and a launch is saved (us, apart against together): 4 experts, rows
// of 2048 fp32 9.4 / 8.3 in a graph, 11.7 / 9.3 outside one; 16 experts, 2048 bf16 9.3 / 9.4 and 11.8 / 9.8; 64 experts, 512
// bf16 10.1 / 13.1, since a warp takes its experts one after the other; 32 experts, 2048 bf16 9.6 / 11.3.
constexpr int kFewOwnExperts = 16, kFewOwnBytes = 65536;
// Weights that TMA cannot read go by rows, element by element (bytes of (token, choice) pairs each us), or all experts are copied
// first (bytes read and written each us) where that is less: few experts and many tokens (27 tokens top-3, 4 experts 1803 x
// 1809 bf16, us: 298 by rows, 77 with the copy).
constexpr double kFewOddRate = 4.5e6, kFewPackRate = 5e6;
constexpr int kFewJoinRoom = 24 * 1024;                // of the join's CTA beside it

FewExpertPlan plan_few_experts(const FewExpertParams& p, int sms) {
  FewExpertPlan r{};
  const int eb = p.bf16 ? 2 : 4, parts = p.bf16 ? 1 : 2;
  auto aligned = [&](const void* base, long long row, long long expert) {
    return ((uintptr_t)base & 15) == 0 && (row * eb) % 16 == 0 && (p.E == 1 || (expert * eb) % 16 == 0);
  };
  const int n1 = (p.act == (int)Act::kSwiGLU ? 2 : 1) * p.F;
  // TMA reads rows that start on 16 bytes and do not overlap, of experts that lie apart
  const bool rows16 = aligned(p.w1, p.w1_stride, p.w1_estride) && aligned(p.w2, p.w2_stride, p.w2_estride) &&
                      p.w1_stride >= p.D && p.w2_stride >= p.F && (p.E == 1 || (p.w1_estride > 0 && p.w2_estride > 0));
  const int pairs = p.T * p.k;
  const double expert = (double)eb * ((double)n1 * p.D + (double)p.O * p.F), bytes = pairs * expert;
  if (rows16) {
    r.tensor = bytes > (p.bf16 ? kFewRowBytes : kFewRowBytesFp32);
  } else if (bytes / kFewOddRate > p.E * expert * 2 / kFewPackRate + std::min(p.E, pairs) * expert / (p.bf16 ? 5e6 : 3e6) + 20) {
    r.tensor = r.pack_w = 1;
    r.w1_bytes = up256((long long)p.E * n1 * up8(p.D) * eb);
    r.w2_bytes = up256((long long)p.E * p.O * up8(p.F) * eb);
  }
  if (!r.tensor) {
    r.vec = rows16 && (p.D * eb) % 16 == 0 && (p.F * eb) % 16 == 0 && aligned(p.x, p.T > 1 ? p.x_stride : 0, 0);
    r.a_bytes = up256((long long)pairs * p.F * 4);
    r.route = p.T == 1 && p.E <= kFewOwnExperts && (long long)p.E * p.D * eb <= kFewOwnBytes;
    return r;
  }
  // fp32: so many tokens at a time that no accumulator takes more than 160 of K, if 16 can (D 4960), since it is cut at each
  // step: 64 tokens to a D of 1120, 48 to 1440, 32 to 2400.  The weights are then read again for each (64 tokens, 4 experts
  // 4096 x 1024 SwiGLU: error 0.9e-6 and 484 us by 16; all at once, with chains of 1024, it was 6.6e-6 and 130 us).
  r.slice = p.T;
  if (!p.bf16) {
    const int steps = (p.D + 31) / 32;
    auto fits = [&](int T) {
      return steps <= FewAcc((T + 15) / 16 * 16, true, steps).chains * kFewChain;
    };
    if (!fits(p.T)) r.slice = std::min(p.T, fits(32) ? 32 : 16);
  }
  const int T = r.slice;
  r.grid = std::min(sms, kFewJoinItems - 2 * kFewTopK);
  r.Op = (p.O + 127) / 128 * 128;
  r.Tp = (T + 15) / 16 * 16;
  const int UE = (p.F + 15) / 16, ups = 128 / eb / 16;
  r.pack = !p.bf16 || !aligned(p.x, p.T > 1 ? p.x_stride : 0, 0) || (p.T > 1 && p.x_stride < p.D);   // tokens that are one, expanded
  r.packed_stride = (p.D + 7) / 8 * 8;
  if (r.pack) r.packed_bytes = up256((long long)parts * r.Tp * r.packed_stride * eb);
  // An expert's tokens times the CTAs that share it, over all experts: n experts have at most min(T k, n T) tokens
  // and (grid / n + 2) CTAs each, so T (grid + 2 k) rows at most, whatever n is.
  r.a_bytes = up256((long long)T * (r.grid + 2 * p.k) * r.Op * 4);
  // Activations of the longest range of a CTA (bf16: for an expert of four times the average tokens), if that leaves four
  // stages; where there are more the range is worked off in pieces, which costs a sum in memory each.  The rest holds stages (64
  // experts top-6, 37 tokens: 188 us with seven, 205 with the four that room for all tokens on one expert leaves).
  const int sb = p.bf16 ? FewTc<false>::stage_bytes(r.Tp) : FewTc<true>::stage_bytes(r.Tp);
  // Up to 16 tokens the join's CTAs find room beside the experts' (64 experts, 1 token: 49.7 -> 43.5 us); with more, the
  // stages are worth more (37 tokens: 193 against 196 us).
  const int room = kFewShared - (T <= 16 ? kFewJoinRoom : 0) - (p.bf16 ? 0 : FewTc<true>::low_bytes());
  const long long most = ((long long)std::min(p.E, T * p.k) * UE + r.grid - 1) / r.grid;
  const long long rows = (std::min<long long>(most, UE) + ups - 1) / ups + 1;
  constexpr int hparts = FewTc<false>::HPARTS;
  const int crowd = p.bf16 ? std::min(r.Tp, (4 * T * p.k / p.E + 16) / 16 * 16) : r.Tp;
  r.hbytes = (int)std::min<long long>(rows * hparts * crowd * 128, room - 4 * sb);
  r.hbytes = std::max({r.hbytes, hparts * r.Tp * 128, kFewSlack});
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

static void launch_few_tensor(const FewExpertParams& p, const FewExpertPlan& plan, char* ws, cudaStream_t s);

void launch_few(const FewRouteParams& route, const FewExpertParams& params, const FewExpertPlan& plan, void* workspace, cudaStream_t s) {
  FewRouteParams r = route;
  FewExpertParams p = params;
  char* ws = (char*)workspace;
  float* a = (float*)(ws + plan.packed_bytes);
  if (!plan.tensor) {
    if (!plan.route) launch_route(r, s);
    if (p.bf16) launch_rows<__nv_bfloat16>(p, r, plan, a, s);
    else launch_rows<float>(p, r, plan, a, s);
    return;
  }
  if (plan.pack_w) {
    char* const w1 = ws + plan.packed_bytes + plan.a_bytes;
    char* const w2 = w1 + plan.w1_bytes;
    const int n1 = (p.act == (int)Act::kSwiGLU ? 2 : 1) * p.F, s1 = (int)up8(p.D), s2 = (int)up8(p.F);
    launch_pack_rows(p.w1, p.w1_stride, p.w1_estride, p.E, w1, s1, n1, p.D, p.bf16, s);
    launch_pack_rows(p.w2, p.w2_stride, p.w2_estride, p.E, w2, s2, p.O, p.F, p.bf16, s);
    p.w1 = w1;
    p.w2 = w2;
    p.w1_stride = s1;
    p.w2_stride = s2;
    p.w1_estride = (long long)n1 * s1;
    p.w2_estride = (long long)p.O * s2;
  }
  const int eb = p.bf16 ? 2 : 4, ob = p.out_bf16 ? 2 : 4, rb = p.res_bf16 ? 2 : 4;
  for (int t = 0; t < params.T; t += plan.slice) {   // each uses the workspace when the one before has ended
    r.T = p.T = std::min(plan.slice, params.T - t);
    r.x = p.x = (const char*)params.x + t * params.x_stride * eb;
    r.ids = route.ids + t * p.k;
    r.gates = route.gates + t * p.k;
    if (route.mask) r.mask = route.mask + t * route.mask_stride;
    p.ids = r.ids;
    p.gates = r.gates;
    p.out = (char*)params.out + t * params.out_stride * ob;
    if (params.residual) p.residual = (const char*)params.residual + t * params.res_stride * rb;
    launch_route(r, s);
    launch_few_tensor(p, plan, ws, s);
  }
}

static void launch_few_tensor(const FewExpertParams& p, const FewExpertPlan& plan, char* ws, cudaStream_t s) {
  float* const a = (float*)(ws + plan.packed_bytes);
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
  if (p.T >= 5) launch_with_pdl(few_join_parts_kernel<4>, dim3(plan.Op / 128, (p.T + 3) / 4), dim3(kFewJoinThreads), 0, s, true, tp);
  else launch_with_pdl(few_join_parts_kernel<1>, dim3(plan.Op / 128, p.T), dim3(kFewJoinThreads), 0, s, true, tp);
}

}  // namespace raiccl
