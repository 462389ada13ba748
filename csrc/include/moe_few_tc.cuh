// Experts of a few-token mixture-of-experts layer on the tensor cores: the
// chosen experts' weights are read once, at the rate that memory gives them.
//
// Both products run with the weights as the 128-row operand of tcgen05.mma and
// the tokens as its narrow N side, so a weight goes from memory to shared
// memory (TMA) to the tensor core without passing through registers.
//
// Split.  The hidden rows of all chosen experts, in units of 16, are dealt to
// the CTAs (one per SM) as contiguous ranges of equal size; a range may span
// experts.  Hidden row f needs row f of W1 (rows f and F + f for SwiGLU) and
// column f of W2, so a CTA makes its rows' activations for the expert's tokens,
// keeps them in shared memory, and multiplies them by its columns of W2: no
// CTA waits for another between the two products, and every CTA has the same
// number of weights to read.  What remains is a sum over the CTAs of an expert
// and over the experts of a token: each CTA writes its part of the expert's
// result, and a third, small kernel adds a token's parts in a fixed order (by
// choice, then CTA), applies the gates and adds the residual.  Adding them in
// this kernel by the last CTA to arrive was tried first: a fence and an atomic
// round trip for each 128 columns made the epilogue, not memory, set the pace
// (64 experts, 1 token: 149 us).
//
// Steps of a CTA's range (roles: one TMA thread, one MMA thread, two groups of
// four epilogue warps that take tiles in turn; fp32 also eight splitting
// warps).  The range is worked off in batches of runs, each of one expert,
// whose activations fit in shared memory together: first product 1 of all its
// runs, then product 2 of all, so that the wait for the activations comes once:
//   product 1   tiles of 128 rows of W1 (64 gate + 64 up rows, 16 by 16), K = D
//               in 128-byte steps, against all T tokens; the epilogue applies
//               bias and activation and keeps the expert's own tokens, as two
//               parts each (bf16, or tf32 for fp32), in the swizzled layout that
//               product 2 reads
//   product 2   tiles of 128 rows of W2, K = the range's hidden rows
//
// The activations of a bf16 layer go into product 2 as two bf16 parts, 2^-16
// together, so that the result is the formula's, rounded once.  The weights of
// product 2 pass the tensor core once for both: the second product takes them
// from the collector buffer, which holds because no other CTA that multiplies
// finds shared memory on the same SM (64 experts, 1 token 33.3 us, 37
// tokens 189; with bf16 activations 32.9 and 188, 0.0022 instead of 0.0016 off).
//
// fp32 numbers are taken as two tf32 parts of 11 bits each, h + l: x and the
// activations as two copies, the weights as they lie (the tensor core reads
// their upper 19 bits) with the rests written beside them in shared memory.
// h h' + h l' + l h' is the product to 2^-20.  The tensor core cuts what does not
// fit its accumulator, which drifts with the length of the chain (2e-6 of the
// result for each 1024 of K, twice that behind SwiGLU), so fp32 sums h h' in
// chains, 128 to 160 of K in product 1 and about 128 hidden rows in product 2,
// each into an accumulator of its own; they are added in registers.  The small
// products, whose cuts do not show, have one accumulator for all of K.  Two
// groups of splitting
// warps set the pace of fp32 (8 experts 1024 x 4096, 16 tokens: 82 us; writing
// the high parts too 90, writing nothing 68).
#pragma once

#include <type_traits>

#include "serving.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

constexpr int kFewTile = 128 * 128;           // bytes of a weight tile: 128 rows of 128 bytes
constexpr int kFewSlack = 12 * 1024;          // behind the last tile: rows that an instruction reads past a short one
constexpr int kFewMaxStages = 12;
constexpr int kFewChain = 5;                  // fp32: 128-byte steps of K of an accumulator at most (160) ...
constexpr int kFewShort = 4;                  // ... and at least (128): each one more is another read in the epilogue
constexpr int kFewLow = 2;                    // fp32: stages whose low parts of the weights are kept (3: a stage less, 2 us more of 82)
constexpr unsigned long long kFewWaitNs = 2000000000ull;
constexpr int kFewKernelId = 600;

// What the launch fixes.
struct FewTcParams {
  FewExpertParams e;
  float* part;        // [rows, Op] the CTAs' parts of the experts' results
  int grid;           // CTAs of the experts' kernel
  int Op;             // O rounded up to 128
  int Tp;             // T rounded up to 16
  int stages;
  int wide;           // whole tiles of W1 in one copy
  int hbytes;         // shared memory of the activations
};

template <bool FP32>
struct FewTc {
  static constexpr int EB = FP32 ? 4 : 2;
  static constexpr int BK = 128 / EB;              // elements of a 128-byte row
  static constexpr int PARTS = FP32 ? 2 : 1;       // of the tokens and the weights
  static constexpr int HPARTS = 2;                 // of the activations
  static constexpr int UPS = BK / 16;              // units of 16 hidden rows in a 128-byte row of activations
  static constexpr int TAIL = 16 * EB;             // bytes of one unit in a row
  static constexpr int THREADS = FP32 ? 576 : 320;
  static constexpr uint32_t FORMAT = FP32 ? 2u : 1u;
  // A stage holds a weight tile and its tile of tokens, or, where the weight tile has few rows, several K steps of
  // both (weights first, tokens at the end): a stage costs its waits and its commit, 0.2 us, whatever it holds.
  static __host__ __device__ int stage_bytes(int Tp) { return kFewTile + (PARTS * Tp * 128 < 4096 ? 4096 : PARTS * Tp * 128); }
  static __host__ __device__ int low_bytes() { return FP32 ? kFewLow * kFewTile : 0; }
};

// The plan that every CTA makes of the routed tokens.
struct FewPlan {
  unsigned long long mask[kFewExperts + 1];  // by expert: its tokens
  int used[kFewExperts + 1];                 // the chosen experts, by number
  int index[kFewExperts + 1];                // their place in used, by expert
  int part0[kFewExperts + 1];                // by place: first row in part
  int parts[kFewExperts + 1];                // by place: CTAs with a part
  int ne;
  int q, groups;                             // units that stay together; of these to an expert
};

// CTA of group u where U groups are dealt to G <= U CTAs: CTA c has groups [U c / G, U (c + 1) / G).
__device__ __forceinline__ int few_cta(long long u, long long U, int G) { return (int)(((u + 1) * G - 1) / U); }

__device__ __forceinline__ void few_plan(const FewExpertParams& p, FewPlan& s, int UE, int grid) {
  const int pairs = p.T * p.k;   // mask is zero on entry
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
    const int e = __ldcg(p.ids + i);
    if (e >= 0) atomicOr(&s.mask[e], 1ull << (i / p.k));
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int ne = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const bool has = e0 + lane < p.E && s.mask[e0 + lane] != 0ull;
      const unsigned b = __ballot_sync(0xffffffffu, has);
      if (has) {
        const int at = ne + __popc(b & ((1u << lane) - 1u));
        s.used[at] = e0 + lane;
        s.index[e0 + lane] = at;
      }
      ne += __popc(b);
    }
    __syncwarp();
    // Where a CTA has few units, they go by fours (64 hidden rows, whole 128-byte rows of W2) or pairs if no CTA gets more
    // of them for that than a thirty-second: fewer CTAs then share two experts, and fewer loads are short (64 experts, 1
    // token: 43.5 -> 31.7 us).
    long long U = 0, least = ((long long)ne * UE + grid - 1) / grid;
    int q = least <= 32 ? 4 : 1, groups = 0;
    for (;; q >>= 1) {
      groups = (UE + q - 1) / q;
      U = (long long)ne * groups;
      if (q == 1 || (U + grid - 1) / grid * q * 32 <= least * 33) break;
    }
    const int G = U < grid ? (int)U : grid;
    int part = 0;
    for (int i0 = 0; i0 < ne; i0 += 32) {
      const int i = i0 + lane;
      int n = 0, rows = 0;
      if (i < ne) {
        n = few_cta((long long)(i + 1) * groups - 1, U, G) - few_cta((long long)i * groups, U, G) + 1;
        rows = n * __popcll(s.mask[s.used[i]]);
      }
      int rs = rows;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, rs, o);
        if (lane >= o) rs += a;
      }
      if (i < ne) { s.part0[i] = part + rs - rows; s.parts[i] = n; }
      part += __shfl_sync(0xffffffffu, rs, 31);
    }
    if (lane == 0) { s.ne = ne; s.q = q; s.groups = groups; }
  }
  __syncthreads();
}

// A run of units of one expert; the roles walk the same runs.
struct FewRun {
  int place, expert, tokens, np;   // place in used, expert, its tokens, their number rounded up to 16
  int f0, units;                   // first hidden row, units of 16
  int h;                           // its activations' first 128-byte row in shared memory
  bool first;                      // of the CTA's runs of this expert
};

struct FewWalk {
  long long u, u1, U;   // groups
  int UE, G, s, n, a, place;
  __device__ void start(const FewPlan& plan, int UE_, int grid) {
    UE = UE_;
    U = (long long)plan.ne * plan.groups;
    G = U < grid ? (int)U : grid;
    const int c = blockIdx.x;
    u = c < G ? U * c / G : 0;
    u1 = c < G ? U * (c + 1) / G : 0;
    s = n = a = place = 0;
  }
  // The next run of a batch that has used `off` of the hrows rows of activations so far; false at its end.
  // Only a batch's first run may be cut to fit, and it is then the only one.
  __device__ bool next(const FewPlan& plan, int hrows, int parts, int ups, int& off, FewRun& r) {
    if (s >= n) {
      if (u >= u1) return false;
      const int pl = (int)(u / plan.groups), first = (int)(u - (long long)pl * plan.groups);
      const int take = (int)(u1 - u < plan.groups - first ? u1 - u : plan.groups - first);
      const int count = take * plan.q < UE - first * plan.q ? take * plan.q : UE - first * plan.q;   // units
      const int np = (__popcll(plan.mask[plan.used[pl]]) + 15) & ~15;
      if (off > 0 && off + (count + ups - 1) / ups * np * parts > hrows) return false;
      place = pl;
      a = first * plan.q;
      n = count;
      s = 0;
      u += take;
    } else if (off > 0) {
      return false;
    }
    r.place = place;
    r.expert = plan.used[place];
    r.tokens = __popcll(plan.mask[r.expert]);
    r.np = (r.tokens + 15) & ~15;
    const int cap = (hrows - off) / (r.np * parts) * ups;
    r.units = n - s < cap ? n - s : cap;
    r.f0 = (a + s) * 16;
    r.h = off;
    r.first = s == 0;
    off += (r.units + ups - 1) / ups * r.np * parts;
    s += r.units;
    return true;
  }
};

// Accumulators in TMEM, for one or two epilogue groups with one or two sets of
// buffers: `chains` of product 1 for one tile, and of product 2 `tiles` tiles of
// 128 outputs, `chains2` each, so that a few tokens' tiles share a hand-over.
// fp32 cuts K into so many chains; the small products, whose own cuts do not
// show, have one more for all of K (`small`), and product 2 has its accumulators
// in product 1's place: neither begins in a batch before the other's have been
// read.  At most 512 columns in all.
struct FewAcc {
  int Tp, groups, nbuf, chains, chains2, tiles, small;
  // fp32: one epilogue group has more accumulators; two where the chains stay within kFewChain steps (16 tokens, 8 experts
  // 1536 x 4096: 113 us against 130 with one)
  __host__ __device__ FewAcc(int Tp_, bool fp32, int steps) : Tp(Tp_) {
    if (fp32) {
      nbuf = 1;
      small = 1;
      chains2 = 5;
      tiles = Tp <= 16 ? 2 : 1;
      const int two = 256 / Tp - small;
      groups = Tp <= 32 && steps <= two * kFewChain ? 2 : 1;
      chains = groups == 2 ? two : 512 / Tp - small;
    } else {
      groups = 2;
      nbuf = 2;
      small = 0;
      chains = chains2 = 1;
      tiles = Tp <= 16 ? 4 : Tp <= 32 ? 2 : 1;
    }
  }
  __device__ uint32_t first(int g, int b) const { return (g * nbuf + b) * (chains + small) * Tp; }
  __device__ uint32_t second(int g, int b) const {   // fp32: tiles * (chains2 + small) of at least 8
    return small ? first(g, b) : (groups * nbuf * chains + (g * nbuf + b) * tiles * chains2) * Tp;
  }
  __device__ int columns() const {
    const int c = groups * nbuf * (chains + small + (small ? 0 : tiles * chains2)) * Tp;
    return c <= 32 ? 32 : c <= 64 ? 64 : c <= 128 ? 128 : c <= 256 ? 256 : 512;
  }
  // Steps to a chain where `all` are dealt to n chains.
  static __device__ int each(int all, int n) {
    const int k = (all + n - 1) / n;
    return k > kFewShort ? k : kFewShort;
  }
};

// out[t, o0 .. o0 + 128) of a token: the parts of all its choices, by choice,
// then CTA, are dealt to its warps in turn, each times its choice's gate; the
// warps' sums are added in order.  A CTA has one token, or from five on four of
// them.  At most grid + 2 k loads of a column for each, so what counts is how
// many are in flight, and, up to 16 tokens, that all but these loads is done
// before the experts' kernel ends: its CTAs then leave room for these beside
// them, and which rows to add follows from the routing alone, whose kernel had
// ended before the experts' kernel allowed this launch.
constexpr int kFewJoinThreads = 512;
constexpr int kFewJoinItems = 192;       // of a token at most; the launch checks grid + 2 k

template <int TOKENS>
__global__ void __launch_bounds__(kFewJoinThreads) few_join_parts_kernel(FewTcParams p) {
  constexpr int W = kFewJoinThreads / 32, tokens = TOKENS;
  __shared__ FewPlan plan;
  __shared__ __align__(16) float red[W][128];
  __shared__ int row[TOKENS * kFewJoinItems];
  __shared__ float weight[TOKENS * kFewJoinItems];
  __shared__ int4 term[TOKENS][kFewTopK];     // a choice's first row in part, rows to the next part, parts, expert
  __shared__ float gate[TOKENS][kFewTopK];
  __shared__ int items[TOKENS];
  const FewExpertParams& e = p.e;
  const int t0 = blockIdx.y * tokens, o0 = blockIdx.x * 128;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // this thread's output
  const int sub = threadIdx.x >> 7, t = t0 + sub, o = o0 + (threadIdx.x & 127);
  const bool writes = sub < tokens && t < e.T && o < e.O;
  float res = 0.f, bias = 0.f;
  if (writes && e.residual) res = load_elem(e.residual, (long long)t * e.res_stride + o, e.res_bf16);
  for (int i = threadIdx.x; i < e.E; i += kFewJoinThreads) plan.mask[i] = 0ull;
  __syncthreads();
  few_plan(e, plan, (e.F + 15) / 16, p.grid);
  if (threadIdx.x < TOKENS * kFewTopK) {
    const int s = threadIdx.x / kFewTopK, j = threadIdx.x % kFewTopK, tt = t0 + s;
    const bool in = tt < e.T && j < e.k;
    const int x = in ? __ldcg(e.ids + tt * e.k + j) : -1;
    int4 v = make_int4(0, 0, 0, 0);
    if (x >= 0) {
      const unsigned long long m = plan.mask[x];
      const int place = plan.index[x];
      v = make_int4(plan.part0[place] + __popcll(m & ((1ull << tt) - 1ull)), __popcll(m), plan.parts[place], x);
    }
    term[s][j] = v;
    gate[s][j] = in ? __ldcg(e.gates + tt * e.k + j) : 0.f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tokens * kFewJoinItems; i += kFewJoinThreads) {
    const int s = i / kFewJoinItems;
    int c = i - s * kFewJoinItems, j = 0;
    while (j < e.k && c >= term[s][j].z) c -= term[s][j++].z;
    if (j < e.k) {
      row[i] = term[s][j].x + c * term[s][j].y;
      weight[i] = gate[s][j];
    }
  }
  if (threadIdx.x < tokens) {
    int n = 0;
    for (int j = 0; j < e.k; ++j) n += term[threadIdx.x][j].z;
    items[threadIdx.x] = n;
  }
  if (e.b2 && writes)
    for (int j = 0; j < e.k; ++j)
      if (term[sub][j].z > 0) bias = fmaf(gate[sub][j], __ldg(e.b2 + (long long)term[sub][j].w * e.O + o), bias);
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  constexpr int per = W / tokens;
  const int mine = w / per;
  const float* col = p.part + o0 + lane * 4;
  const int* rows = row + mine * kFewJoinItems;
  const float* weights = weight + mine * kFewJoinItems;
  const int n = items[mine];
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = w % per; i < n; i += per) {
    const float4 a = __ldcg((const float4*)(col + (long long)rows[i] * p.Op));
    const float g = weights[i];
    v.x = fmaf(g, a.x, v.x);
    v.y = fmaf(g, a.y, v.y);
    v.z = fmaf(g, a.z, v.z);
    v.w = fmaf(g, a.w, v.w);
  }
  *(float4*)&red[w][lane * 4] = v;
  __syncthreads();
  if (!writes) return;
  float out = 0.f;
#pragma unroll
  for (int i = 0; i < per; ++i) out += red[sub * per + i][threadIdx.x & 127];
  store_elem(e.out, (long long)t * e.out_stride + o, out + bias + res, e.out_bf16);
}

// Maps: x [T, D] in boxes of 128 bytes x Tp rows (fp32: [2 Tp, D] parts, 2 Tp
// rows); W1 in boxes of 128 bytes x 16 rows (SwiGLU: x 2, gate and up) and of a
// whole tile; W2 in boxes of 128 bytes x 128 rows and of one unit x 128 rows.
template <bool FP32, bool GLU>
__global__ void __launch_bounds__(FewTc<FP32>::THREADS, 1)
few_experts_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap t1,
                   const __grid_constant__ CUtensorMap t1w, const __grid_constant__ CUtensorMap t2,
                   const __grid_constant__ CUtensorMap t2u, FewTcParams p, DeviceStatus* status) {
  using C = FewTc<FP32>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* const smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ FewPlan plan;
  __shared__ uint64_t full[kFewMaxStages], empty[kFewMaxStages], parted[kFewMaxStages];
  __shared__ uint64_t acc1_full[4], acc1_empty[4], acc2_full[4], acc2_empty[4], drained;
  __shared__ uint32_t tmem_slot;
  const int SB = C::stage_bytes(p.Tp), S = p.stages;
  uint8_t* const low = smem + S * SB;
  uint8_t* const hbuf = low + C::low_bytes();
  const FewExpertParams& e = p.e;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n1 = C::PARTS * p.Tp;                       // rows of tokens in a step
  const FewAcc acc(p.Tp, FP32, (e.D + C::BK - 1) / C::BK);

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); mbar_init(&parted[i], 4); }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&acc1_full[i], 1); mbar_init(&acc1_empty[i], 4);
      mbar_init(&acc2_full[i], 1); mbar_init(&acc2_empty[i], 4);
    }
    mbar_init(&drained, 1);
    fence_mbarrier_init();
    tma_prefetch_desc(&tx); tma_prefetch_desc(&t1); tma_prefetch_desc(&t1w); tma_prefetch_desc(&t2); tma_prefetch_desc(&t2u);
  }
  for (int i = threadIdx.x; i < e.E; i += blockDim.x) plan.mask[i] = 0ull;
  if (warp == 1) { tmem_alloc(&tmem_slot, acc.columns()); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  griddep_wait();
  const int UE = (e.F + 15) / 16;
  few_plan(e, plan, UE, gridDim.x);   // holds __syncthreads
  griddep_launch_dependents();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const int KB = (e.D + C::BK - 1) / C::BK;             // 128-byte steps of product 1
  const int per = FP32 ? FewAcc::each(KB, acc.chains) : KB;   // of them to an accumulator
  const int nO = p.Op / 128;
  constexpr int TU = GLU ? 4 : 8;                       // units of a product-1 tile
  constexpr int UB = GLU ? 4096 : 2048;                 // bytes of one in a step
  constexpr int UPT = kFewTile / (128 * C::TAIL);       // units of 128 rows of W2 in a tile's bytes
  const int hrows = p.hbytes / 128;
  FewWalk walk;
  walk.start(plan, UE, gridDim.x);
  FewRun r;
  int stage = 0;
  uint32_t phase = 0;
  auto advance = [&]() { if (++stage == S) { stage = 0; phase ^= 1u; } };
  // K steps that share a stage for a tile of nu units
  auto pack_of = [&](int nu) { const int n = SB / (nu * UB + n1 * 128); return n < 4 ? n : 4; };

  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (elect_one_sync()) {
      // weights are read once: they leave the rest of L2 (code, router, tokens, parts) alone
      const uint64_t once = l2_evict_first();
      bool ok = true;
      int filled = 0;
      while (ok) {
        FewWalk again = walk;
        int off = 0, runs = 0;
        for (; ok && walk.next(plan, hrows, C::HPARTS, C::UPS, off, r); ++runs) {
          for (int u0 = 0; ok && u0 < r.units; u0 += TU) {
            const int nu = r.units - u0 < TU ? r.units - u0 : TU, pack = pack_of(nu), f0 = r.f0 + u0 * 16;
            for (int kb = 0; kb < KB; kb += pack) {
              if (!(ok = serving_wait(&empty[stage], phase ^ 1u, status, kFewKernelId, kFewWaitNs))) break;
              uint8_t* w = smem + stage * SB;
              uint8_t* x = w + SB - pack * n1 * 128;
              const int n = KB - kb < pack ? KB - kb : pack;
              mbar_arrive_expect_tx(&full[stage], n * (nu * UB + n1 * 128));
              for (int k = 0; k < n; ++k, w += nu * UB, x += n1 * 128) {
                const int d = (kb + k) * C::BK;
                if (nu == TU && p.wide) {
                  if constexpr (GLU) tma_load_5d_hint(w, &t1w, &full[stage], d, 0, 0, f0 / 16, r.expert, once);
                  else tma_load_3d_hint(w, &t1w, &full[stage], d, f0, r.expert, once);
                } else {
                  for (int u = 0; u < nu; ++u) {
                    if constexpr (GLU) tma_load_4d_hint(w + u * UB, &t1, &full[stage], d, f0 + u * 16, 0, r.expert, once);
                    else tma_load_3d_hint(w + u * UB, &t1, &full[stage], d, f0 + u * 16, r.expert, once);
                  }
                }
                tma_load_2d(x, &tx, &full[stage], d, 0);
              }
              advance();
              ++filled;
            }
          }
        }
        if (runs == 0) break;
        off = 0;
        for (; ok && runs > 0; --runs) {
          again.next(plan, hrows, C::HPARTS, C::UPS, off, r);
          const int slices = r.units / C::UPS, tail = r.units % C::UPS;
          const int share = tail ? UPT / tail : 1;   // tiles whose last units share a stage
          for (int i0 = 0; ok && i0 < nO; i0 += acc.tiles) {
            const int nt = nO - i0 < acc.tiles ? nO - i0 : acc.tiles;
            for (int s = 0; ok && s < slices; ++s)
              for (int i = 0; i < nt; ++i) {
                if (!(ok = serving_wait(&empty[stage], phase ^ 1u, status, kFewKernelId, kFewWaitNs))) break;
                mbar_arrive_expect_tx(&full[stage], kFewTile);
                tma_load_3d_hint(smem + stage * SB, &t2, &full[stage], r.f0 + s * C::BK, (i0 + i) * 128, r.expert, once);
                advance();
                ++filled;
              }
            for (int i = 0; ok && tail && i < nt; i += share) {
              const int n = nt - i < share ? nt - i : share;
              if (!(ok = serving_wait(&empty[stage], phase ^ 1u, status, kFewKernelId, kFewWaitNs))) break;
              mbar_arrive_expect_tx(&full[stage], n * tail * 128 * C::TAIL);
              uint8_t* w = smem + stage * SB;
              for (int m = 0; m < n; ++m)
                for (int u = 0; u < tail; ++u, w += 128 * C::TAIL)
                  tma_load_3d_hint(w, &t2u, &full[stage], r.f0 + slices * C::BK + u * 16, (i0 + i + m) * 128, r.expert, once);
              advance();
              ++filled;
            }
          }
        }
      }
      await_loads(full, S, stage, phase, filled, status, kFewKernelId, kFewWaitNs);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    if (elect_one_sync()) {
      uint64_t* ready = FP32 ? parted : full;
      int i1 = 0, j2[2] = {0, 0};   // tiles of product 1; tiles of product 2 by group
      int lo = 0;                   // slot of low parts
      auto next = [&]() {
        advance();
        if (++lo == kFewLow) lo = 0;
      };
      bool ok = true;
      const uint64_t wide_row = umma_desc_k_sw128(0), unit_row = umma_desc_k_narrow(0, C::TAIL);
      const uint32_t id1 = umma_idesc(C::FORMAT, 128, (uint32_t)p.Tp);
      // 32 bytes of K, fp32: weights a and their rests al against the high parts of tokens or activations, b, and the low
      // parts, `lows` 16-byte units behind: into a chain's sum d, and the small products into ds
      auto step = [&](uint32_t d, uint32_t ds, uint64_t a, uint64_t al, uint64_t b, uint32_t lows, uint32_t id, uint32_t more,
                      uint32_t more_small) {
        umma_tf32_twice(d, ds, a, b, b + lows, id, more, more_small);
        umma_tf32(ds, al, b, id, 1u);
      };
      // The same for product 2: step `at` of slice s of the run's hidden rows, whose activations are np rows of high parts,
      // then np of low parts.  bf16: both parts into one sum (no further columns), by two products that read the weights once.
      // fp32: the slice is number `nth` of a chain, whose sum lies `chain` columns behind d.
      auto step2 = [&](uint32_t d, int s, uint32_t chain, int nth, int np, uint64_t a, uint64_t al, uint64_t b, uint32_t id, int at) {
        if constexpr (FP32)
          step(d + chain, d + acc.chains2 * np, a, al, b, np * 8, id, (nth | at) ? 1u : 0u, (s | at) ? 1u : 0u);
        else
          umma_f16_twice(d, a, b, b + np * 8, id, (s | at) ? 1u : 0u);
      };
      while (ok) {
        FewWalk again = walk;
        int off = 0, runs = 0;
        if constexpr (FP32) {   // the batch before has been read: its product 2 in this product 1's place
          for (int g = 0; ok && g < acc.groups; ++g)
            if (j2[g] > 0) ok = serving_wait(&acc2_empty[g * 2], (j2[g] - 1) & 1, status, kFewKernelId, kFewWaitNs);
          tc_fence_after_sync();
        }
        for (; ok && walk.next(plan, hrows, C::HPARTS, C::UPS, off, r); ++runs) {
          for (int u0 = 0; ok && u0 < r.units; u0 += TU, ++i1) {
            const int nu = r.units - u0 < TU ? r.units - u0 : TU, pack = pack_of(nu);
            const int g = i1 % acc.groups, j = i1 / acc.groups, b = j & (acc.nbuf - 1);
            if (!(ok = serving_wait(&acc1_empty[g * 2 + b], ((j / acc.nbuf) & 1) ^ 1u, status, kFewKernelId, kFewWaitNs))) break;
            tc_fence_after_sync();
            uint32_t dc = tmem + acc.first(g, b);
            [[maybe_unused]] const uint32_t ds = dc + acc.chains * p.Tp;
            int at = 0;   // steps of the chain
            for (int kb = 0; kb < KB; kb += pack) {
              if (!(ok = serving_wait(&ready[stage], phase, status, kFewKernelId, kFewWaitNs))) break;
              tc_fence_after_sync();
              const uint32_t w = smem_u32(smem + stage * SB), x = w + SB - pack * n1 * 128, wl = smem_u32(low) + lo * kFewTile;
              const int n = KB - kb < pack ? KB - kb : pack;
              uint64_t da = desc_at(wide_row, w), dl = desc_at(wide_row, wl), dx = desc_at(wide_row, x);
              for (int kk = 0; kk < n; ++kk, da += nu * UB / 16, dl += nu * UB / 16, dx += n1 * 8) {
                if (FP32 && at == per) { at = 0; dc += p.Tp; }   // the next chain
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  if constexpr (FP32) step(dc, ds, da + 2 * k, dl + 2 * k, dx + 2 * k, p.Tp * 8, id1, (at | k) ? 1u : 0u, (kb | kk | k) ? 1u : 0u);
                  else umma_f16(dc, da + 2 * k, dx + 2 * k, id1, (at | k) ? 1u : 0u);
                }
                ++at;
              }
              umma_commit(&empty[stage]);
              next();
            }
            umma_commit(&acc1_full[g * 2 + b]);
          }
        }
        if (runs == 0) break;
        // a tile's activations are in shared memory once its accumulator was released
        for (int g = 0; g < acc.groups; ++g)
          for (int b = 0; ok && b < acc.nbuf; ++b) {
            const int tiles = (i1 + acc.groups - 1 - g) / acc.groups, uses = (tiles + acc.nbuf - 1 - b) / acc.nbuf;
            if (uses > 0) ok = serving_wait(&acc1_empty[g * 2 + b], (uses - 1) & 1, status, kFewKernelId, kFewWaitNs);
          }
        tc_fence_after_sync();
        off = 0;
        for (; ok && runs > 0; --runs) {
          again.next(plan, hrows, C::HPARTS, C::UPS, off, r);
          const int slices = r.units / C::UPS, tail = r.units % C::UPS;
          const uint32_t hrow = C::HPARTS * r.np * 128;   // bytes of a slice of activations
          const uint32_t id2 = umma_idesc(C::FORMAT, 128, (uint32_t)r.np);
          [[maybe_unused]] const int each = FewAcc::each(slices + (tail ? 1 : 0), acc.chains2);
          const int share = tail ? UPT / tail : 1;
          for (int i0 = 0, g = 0; ok && i0 < nO; i0 += acc.tiles, g = acc.groups - 1 - g) {
            const int nt = nO - i0 < acc.tiles ? nO - i0 : acc.tiles;
            const int j = j2[g]++, b = j & (acc.nbuf - 1);
            if (!(ok = serving_wait(&acc2_empty[g * 2 + b], ((j / acc.nbuf) & 1) ^ 1u, status, kFewKernelId, kFewWaitNs))) break;
            tc_fence_after_sync();
            const uint32_t d = tmem + acc.second(g, b), dn = (acc.chains2 + acc.small) * r.np;
            const uint32_t h0 = smem_u32(hbuf) + r.h * 128;
            uint32_t chain = 0;
            int nth = 0;
            for (int s = 0; ok && s < slices; ++s) {
              for (int i = 0; i < nt; ++i) {
                if (!(ok = serving_wait(&ready[stage], phase, status, kFewKernelId, kFewWaitNs))) break;
                tc_fence_after_sync();
                const uint64_t da = desc_at(wide_row, smem_u32(smem + stage * SB)), dl = desc_at(wide_row, smem_u32(low) + lo * kFewTile);
                const uint64_t dh = desc_at(wide_row, h0 + s * hrow);
#pragma unroll
                for (int k = 0; k < 4; ++k) step2(d + i * dn, s, chain, nth, r.np, da + 2 * k, dl + 2 * k, dh + 2 * k, id2, k);
                umma_commit(&empty[stage]);
                next();
              }
              if (FP32 && ++nth == each) { nth = 0; chain += r.np; }
            }
            for (int i = 0; ok && tail && i < nt; i += share) {
              const int n = nt - i < share ? nt - i : share;
              if (!(ok = serving_wait(&ready[stage], phase, status, kFewKernelId, kFewWaitNs))) break;
              tc_fence_after_sync();
              constexpr int KS = C::TAIL / 32;   // 32-byte steps of a unit
              uint64_t da = desc_at(unit_row, smem_u32(smem + stage * SB)), dl = desc_at(unit_row, smem_u32(low) + lo * kFewTile);
              const uint64_t dh = desc_at(wide_row, h0 + slices * hrow);
              for (int m = 0; m < n; ++m)
                for (int u = 0; u < tail; ++u, da += 8 * C::TAIL, dl += 8 * C::TAIL)
#pragma unroll
                  for (int k = 0; k < KS; ++k)
                    step2(d + (i + m) * dn, slices, chain, nth, r.np, da + 2 * k, dl + 2 * k, dh + 2 * (u * KS + k), id2, u | k);
              umma_commit(&empty[stage]);
              next();
            }
            umma_commit(&acc2_full[g * 2 + b]);
          }
        }
      }
      // every product has finished before the accumulators are freed
      umma_commit(&drained);
      serving_wait(&drained, 0, status, kFewKernelId, kFewWaitNs);
    }
  } else if (warp < 10) {
    // ---------------------------------------------------------------- epilogues
    const int q = warp & 3, g = (warp - 2) >> 2;          // TMEM lanes 32 q .. 32 q + 31; group
    const uint32_t lane_addr = tmem + ((uint32_t)(q * 32) << 16);
    int i1 = 0, j2 = 0;
    bool ok = true;
    while (ok && g < acc.groups) {
      FewWalk again = walk;
      int off = 0, runs = 0;
      for (; ok && walk.next(plan, hrows, C::HPARTS, C::UPS, off, r); ++runs) {
        const unsigned long long mask = plan.mask[r.expert];
        const float* b1 = e.b1 ? e.b1 + (long long)r.expert * (GLU ? 2 : 1) * e.F : nullptr;
        const uint32_t hrow = C::HPARTS * r.np * 128;
        for (int u0 = 0; ok && u0 < r.units; u0 += TU, ++i1) {
          if (i1 % acc.groups != g) continue;
          const int j = i1 / acc.groups, b = j & (acc.nbuf - 1);
          const int unit = u0 + (GLU ? q : 2 * q + (lane >> 4));  // of the run
          const int fl = unit * 16 + (lane & 15);           // hidden row of the run
          const int f = r.f0 + fl;
          const bool real = f < e.F;
          float bias = 0.f, bias_up = 0.f;
          if (b1 && real && unit < r.units) {
            bias = __ldg(b1 + f);
            if constexpr (GLU) bias_up = __ldg(b1 + e.F + f);
          }
          ok = mbar_wait_warp(&acc1_full[g * 2 + b], (j / acc.nbuf) & 1, status, kFewKernelId, kFewWaitNs);
          tc_fence_after_sync();
          const uint32_t base = lane_addr + acc.first(g, b);
          uint8_t* hcol = hbuf + r.h * 128 + (fl / C::BK) * hrow;
          const int byte = (fl % C::BK) * C::EB;
          const bool any = u0 + (GLU ? q : 2 * q) < r.units;  // this warp has a unit of the tile
          for (int c = 0; any && c < p.Tp; c += 16) {
            __syncwarp();
            const unsigned take = (unsigned)(mask >> c) & 0xffffu;   // the expert's tokens among these 16
            if (take == 0u) continue;
            uint32_t v[16];
            tmem_ld16(base + c, v);
            if constexpr (FP32) {
              uint32_t h[16];
              tmem_ld16(base + acc.chains * p.Tp + c, h);   // the small products
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(h[i]));
              for (int q1 = 1; q1 * per < KB; ++q1) {
                tmem_ld16(base + q1 * p.Tp + c, h);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(h[i]));
              }
            } else {
              tmem_ld_wait();
            }
            const int below = __popcll(mask & ((1ull << c) - 1ull));
            auto put = [&](int i, float val) {   // activation of token c + i
              const int n = below + __popc(take & ((1u << i) - 1u));
              const float h = real ? val : 0.f;
              uint8_t* at = hcol + (n >> 3) * 1024 + (n & 7) * 128 + (byte ^ ((n & 7) << 4));
              if constexpr (FP32) {
                float hi, lo;
                split_tf32(h, hi, lo);
                *(float*)at = hi;
                *(float*)(at + r.np * 128) = lo;
              } else {
                split_bf16(h, *(__nv_bfloat16*)at, *(__nv_bfloat16*)(at + r.np * 128));
              }
            };
            if constexpr (GLU) {
              // lanes 0-15 hold gate rows, 16-31 the up rows of the same f: each half takes eight of the columns
              const bool up = lane >= 16;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float mine = __uint_as_float(up ? v[8 + i] : v[i]);
                const float other = __shfl_xor_sync(0xffffffffu, __uint_as_float(up ? v[i] : v[8 + i]), 16);
                const int col = up ? 8 + i : i;
                const float gate = (up ? other : mine) + bias, lin = (up ? mine : other) + bias_up;
                if (take >> col & 1u) put(col, serving_swiglu(gate, lin));
              }
            } else {
              auto all = [&](auto act) {   // one loop to an activation: a launch fetches only the code of its own
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  if ((take >> i & 1u) && unit < r.units) put(i, serving_act(__uint_as_float(v[i]) + bias, (int)decltype(act)::value));
              };
              if (e.act == (int)Act::kRelu) all(std::integral_constant<Act, Act::kRelu>{});
              else if (e.act == (int)Act::kGelu) all(std::integral_constant<Act, Act::kGelu>{});
              else if (e.act == (int)Act::kSilu) all(std::integral_constant<Act, Act::kSilu>{});
              else all(std::integral_constant<Act, Act::kNone>{});
            }
          }
          fence_proxy_async_smem();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc1_empty[g * 2 + b]);
        }
      }
      if (runs == 0) break;
      off = 0;
      for (; ok && runs > 0; --runs) {
        again.next(plan, hrows, C::HPARTS, C::UPS, off, r);
        // product 2: this CTA's part of the expert's result.  A group of tiles always belongs to the same epilogue
        // group, so a cut run's later pieces are added by the thread that wrote the first.
        const int mine = (int)blockIdx.x - few_cta((long long)r.place * plan.groups, walk.U, walk.G);
        const int all = (r.units + C::UPS - 1) / C::UPS, each = FewAcc::each(all, acc.chains2);
        float* dst = p.part + (long long)(plan.part0[r.place] + mine * r.tokens) * p.Op + q * 32 + lane;
        for (int i0 = g * acc.tiles; ok && i0 < nO; i0 += acc.groups * acc.tiles, ++j2) {
          const int b = j2 & (acc.nbuf - 1), nt = nO - i0 < acc.tiles ? nO - i0 : acc.tiles;
          ok = mbar_wait_warp(&acc2_full[g * 2 + b], (j2 / acc.nbuf) & 1, status, kFewKernelId, kFewWaitNs);
          tc_fence_after_sync();
          for (int i = 0; i < nt; ++i) {
            const uint32_t base = lane_addr + acc.second(g, b) + i * (acc.chains2 + acc.small) * r.np;
            for (int c = 0; c < r.tokens; c += 16) {
              __syncwarp();
              uint32_t v[16];
              float was[16];   // of the run's earlier pieces: all loads before the first store
              float* at = dst + (long long)c * p.Op + (i0 + i) * 128;
#pragma unroll
              for (int j = 0; j < 16; ++j) was[j] = !r.first && c + j < r.tokens ? __ldcg(at + (long long)j * p.Op) : 0.f;
              tmem_ld16(base + c, v);
              if constexpr (FP32) {
                uint32_t l[16];
                tmem_ld16(base + acc.chains2 * r.np + c, l);   // the small products
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(l[j]));
                for (int q2 = 1; q2 * each < all; ++q2) {
                  tmem_ld16(base + q2 * r.np + c, l);
                  tmem_ld_wait();
#pragma unroll
                  for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(l[j]));
                }
              } else {
                tmem_ld_wait();
              }
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (c + j < r.tokens) __stcg(at + (long long)j * p.Op, __uint_as_float(v[j]) + was[j]);
            }
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc2_empty[g * 2 + b]);
        }
      }
    }
  } else if constexpr (FP32) {
    // ---------------------------------------------------------------- weights into tf32 parts
    const int tid = (threadIdx.x - 320) & 127, g = (threadIdx.x - 320) >> 7;   // two groups take stages in turn
    int turn = 0, lo = 0, old = 0;   // slot of low parts; stage of the products that read it last, and their phase
    uint32_t old_phase = 0;
    bool ok = true;
    auto part = [&](int bytes) {
      const int slot = lo, was = old;
      const uint32_t was_phase = old_phase;
      if (++lo == kFewLow) lo = 0;
      if (turn >= kFewLow && ++old == S) { old = 0; old_phase ^= 1u; }
      if (turn % 2 == g) {
        ok = mbar_wait_warp(&full[stage], phase, status, kFewKernelId, kFewWaitNs) &&
             (turn < kFewLow || mbar_wait_warp(&empty[was], was_phase, status, kFewKernelId, kFewWaitNs));
        split_tile<false>(smem + stage * SB, low + slot * kFewTile, tid, bytes);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&parted[stage]);
      }
      ++turn;
      advance();
    };
    while (ok) {
      FewWalk again = walk;
      int off = 0, runs = 0;
      for (; ok && walk.next(plan, hrows, C::HPARTS, C::UPS, off, r); ++runs) {
        for (int u0 = 0; ok && u0 < r.units; u0 += TU) {
          const int nu = r.units - u0 < TU ? r.units - u0 : TU, pack = pack_of(nu);
          for (int kb = 0; ok && kb < KB; kb += pack) part((KB - kb < pack ? KB - kb : pack) * nu * UB);
        }
      }
      if (runs == 0) break;
      off = 0;
      for (; ok && runs > 0; --runs) {
        again.next(plan, hrows, C::HPARTS, C::UPS, off, r);
        const int slices = r.units / C::UPS, tail = r.units % C::UPS;
        const int share = tail ? UPT / tail : 1;
        for (int i0 = 0; ok && i0 < nO; i0 += acc.tiles) {
          const int nt = nO - i0 < acc.tiles ? nO - i0 : acc.tiles;
          for (int s = 0; ok && s < slices * nt; ++s) part(kFewTile);
          for (int i = 0; ok && tail && i < nt; i += share) part((nt - i < share ? nt - i : share) * tail * 128 * C::TAIL);
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  __syncwarp();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, acc.columns());
}

}  // namespace raiccl
