// Parameters and launch entry points of the serving operators: the mixture-of-
// experts layer for a few tokens (csrc/kernels/moe_few.cu) and the dense
// product with an epilogue (csrc/kernels/linear.cu).  The torch bindings in
// csrc/kernels/serving_bindings.cpp check the tensors and fill these.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "types.h"

namespace raiccl {

constexpr int kFewTokens = 64;     // tokens of one call at most: an expert's tokens are the bits of one 64-bit word
constexpr int kFewExperts = 255;   // experts at most (the routing key's byte for the expert)
constexpr int kFewTopK = 8;

// A ring of S stages is filled in turn, the phase of its barriers changes with
// every round.  From the stage and phase of the next fill back to those of the
// fill before it.
__host__ __device__ inline void fill_before(int S, int& stage, uint32_t& phase) {
  if (stage == 0) {
    stage = S;
    phase ^= 1u;
  }
  --stage;
}

// Routing of T tokens.  Element strides; mask_stride 0 for one mask of all tokens.
struct FewRouteParams {
  const void* x;          // [T, D]
  long long x_stride;
  const void* w;          // [E, D]
  long long w_stride;
  const float* bias;      // [E] or nullptr
  const uint8_t* mask;    // [T, E] or [E], nonzero: never chosen; or nullptr
  long long mask_stride;
  int T, D, E, k;
  int gate_mode;          // 0 ones, 1 softmax over the chosen, 2 softmax over all that are not blocked
  int bf16;               // element type of x and w
  int vec;                // rows of x and w are 16-byte aligned multiples of 16 bytes
  int* ids;               // [T, k], -1 where no expert was left
  float* gates;           // [T, k], 0 there
  void* packed;           // x for the experts' kernel, or nullptr: bf16 rows [T, packed_stride] as they are;
  long long packed_stride;  // fp32 [2][packed_rows, packed_stride] as two tf32 parts
  int packed_rows;
  int cuts;               // pieces of a row, by the launch
};

// The experts' MLPs and the weighted sum of the routed tokens.
struct FewExpertParams {
  const void* x;          // [T, D]
  long long x_stride;
  const void* w1;         // [E, N1, D], N1 = F, or 2F (gate rows, then up rows) for SwiGLU
  long long w1_estride, w1_stride;
  const void* w2;         // [E, O, F]
  long long w2_estride, w2_stride;
  const float* b1;        // [E, N1] or nullptr
  const float* b2;        // [E, O] or nullptr
  const void* residual;   // [T, O] or nullptr
  long long res_stride;
  void* out;              // [T, O]
  long long out_stride;
  const int* ids;         // [T, k]
  const float* gates;     // [T, k]
  int T, D, E, k, F, O;
  int act;
  int bf16, out_bf16, res_bf16;
};

// How the experts of a call run, and the device memory that they need besides.
struct FewExpertPlan {
  int tensor;             // on the tensor cores (else by rows, on CUDA cores)
  int vec;                // by rows: 16 bytes at a time
  int route;              // by rows: the experts' kernel routes too
  int grid, stages, hbytes, Op, Tp;
  int pack;               // x is packed by the routing kernel
  int packed_stride;
  int slice;              // fp32 on the tensor cores: tokens that go together
  int pack_w;             // the experts are copied to rows that TMA can read
  long long packed_bytes, a_bytes, w1_bytes, w2_bytes;  // multiples of 256; in this order in the workspace
  long long bytes() const { return packed_bytes + a_bytes + w1_bytes + w2_bytes; }
};

FewExpertPlan plan_few_experts(const FewExpertParams& p, int sms);
void launch_few(const FewRouteParams& r, const FewExpertParams& p, const FewExpertPlan& plan, void* workspace, cudaStream_t s);

// `groups` blocks of rows of K elements, `group` apart, to one block of rows that start on 16 bytes, `packed` apart.
void launch_pack_rows(const void* src, long long stride, long long group, int groups, void* dst, int packed, long long rows, int K,
                      int bf16, cudaStream_t s);

// The current device's record of a wait that ran out in a serving operator (device memory).
DeviceStatus* serving_status();

// out = act(x w^T + bias) + residual; SwiGLU: w holds F gate rows, then F up
// rows, and N = F is the width of out.
struct LinearParams {
  const void* x;          // [M, K]
  long long x_stride;
  const void* w;          // [N, K] (SwiGLU: [2N, K])
  long long w_stride;
  const float* bias;      // [N] (SwiGLU: [2N]) or nullptr
  const void* residual;   // [M, N] or nullptr
  long long res_stride;
  void* out;              // [M, N]
  long long out_stride;
  long long M;
  int N, K;
  int act;
  int bf16, out_bf16, res_bf16;
};

// How a product runs, and the device memory that it needs besides.
struct LinearPlan {
  int vector, vec;         // very few rows, on CUDA cores; 16 bytes at a time
  int dense;               // CTA pairs with tiles of 256 x dense sums; 0: few rows
  int Mp, ranks, stages, low;   // few rows: rows of x of a tile, CTAs that share K, stages, tiles of low parts
  int chained;             // bf16 operands, fp32 result: sums leave the tensor core in pieces of K
  int pack_x, pack_w;      // rows that TMA cannot read are copied to aligned ones first
  int packed_stride;
  long long x_bytes, w_bytes;
  long long bytes() const { return x_bytes + w_bytes; }
};

LinearPlan plan_linear(const LinearParams& p, int sms);
void launch_linear(const LinearParams& p, const LinearPlan& plan, void* workspace, cudaStream_t s);

int serving_sm_count();   // of the current device

}  // namespace raiccl
