// Parameters and launch entry points of the attention operators: the paged
// cache in 4 bits (csrc/kernels/kv_cache.cu), attention of single tokens over it
// (csrc/kernels/attention_cached.cu) and attention over whole prompts
// (csrc/kernels/attention_prompt.cu).  The torch bindings in
// csrc/kernels/attention_bindings.cpp check the tensors and fill these.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "types.h"

namespace raiccl {

constexpr int kCacheGroup = 16;      // numbers that share a scale
constexpr int kCachePage = 16;       // smallest page
constexpr int kCachedTile = 64;      // tokens of a sequence that attention_cached works on at once
constexpr int kCachedKernelId = 640, kCacheWriteKernelId = 641, kCacheReadKernelId = 642, kPromptKernelId = 643;

// The cache: pages of page_size tokens, [pages, heads, page_size, D / 2] codes
// (even dimension in the low four bits) and [pages, heads, page_size, D / 16]
// e4m3 scales, for keys and for values.  A number is code * scale * unit.
struct CacheView {
  uint8_t* k_codes;
  uint8_t* k_scales;
  uint8_t* v_codes;
  uint8_t* v_scales;
  int pages, heads, D;
  int page_shift;                    // page_size = 1 << page_shift
  float k_unit, v_unit;              // powers of two
};

// New keys and values [N, heads, D] to their slots (page * page_size + place; below zero: nowhere).
struct CacheWriteParams {
  CacheView c;
  const void* k;
  const void* v;
  long long k_token, k_head, v_token, v_head;   // element strides
  const void* slots;                 // [N] int32 or int64
  int slots64, bf16, vec;            // vec: rows may be read 16 bytes at a time
  long long N;
  int per_shift;                     // a CTA has 1 << per_shift tokens, by the launch
  float per_k_unit, per_v_unit;      // the units' reciprocals, by the launch
  DeviceStatus* status;
};

// The other way round; tokens without a slot are zeros.
struct CacheReadParams {
  CacheView c;
  void* k;
  void* v;
  long long k_token, k_head, v_token, v_head;
  const void* slots;
  int slots64, bf16, vec;            // vec: rows may be written 16 (1) or 32 (2) bytes at a time
  long long N;
  DeviceStatus* status;
};

void launch_cache_write(const CacheWriteParams& p, cudaStream_t s);
void launch_cache_read(const CacheReadParams& p, cudaStream_t s);

// What a CTA of attention_cached and those behind it have parts of: query heads of a sequence, up to tile `last` of all `tiles`.
struct CachedJoin {
  int b, head0, heads;
  long long last, tiles;
};

// out[b, h] = softmax(scale q[b, h] K^T) V over the first lengths[b] tokens of sequence b.
struct CachedParams {
  CacheView c;
  const void* q;                     // [B, Hq, D]
  long long q_seq, q_head;
  void* out;                         // [B, Hq, D]
  long long o_seq, o_head;
  float* lse;                        // [B, Hq] or nullptr
  const int* table;                  // [B, table_stride] pages of each sequence
  long long table_stride;
  int table_pages;                   // entries of a row
  const int* lengths;                // [B]
  int B, Hq, group;                  // group = Hq / heads
  int bf16, out_bf16;
  int q_vec, o_vec;                  // rows may be read and written 16 bytes at a time
  float mult;                        // logits to base 2 are q . codes * scales by mult 2^mult_exp: scale, log2(e) and the keys' unit
  int mult_exp;
  // by the plan
  int chunk, chunks;                 // query heads that are worked on together, such chunks of a group
  int ctas;                          // that share the work
  int notes;                         // joins are told by p.joins, not found from the lengths
  float* parts;                      // [ctas][2][chunk][D] sums of sequences that several CTAs share
  float2* stats;                     // [ctas][2][chunk] their maxima and sums of exponentials
  float* spill;                      // [ctas][warps][8 or 16][D] sums that a warp puts aside
  CachedJoin* joins;                 // [ctas] pieces that begin within a CTA's share and end behind it; no heads: none
  DeviceStatus* status;
};

struct CachedPlan {
  int chunk, chunks, ctas;
  long long parts_bytes, stats_bytes, spill_bytes, joins_bytes;
  long long bytes() const { return parts_bytes + stats_bytes + spill_bytes + joins_bytes; }
};

CachedPlan plan_cached(const CachedParams& p, int sms);
void launch_cached(const CachedParams& p, const CachedPlan& plan, void* workspace, cudaStream_t s);

// Packed sequences: tokens cu_q[b] .. cu_q[b + 1] of q attend to cu_k[b] .. cu_k[b + 1] of k and v.
struct PromptParams {
  const void* q;                     // [Nq, Hq, D]
  const void* k;                     // [Nk, Hk, D]
  const void* v;
  long long q_token, q_head, k_token, k_head, v_token, v_head;
  void* out;                         // [Nq, Hq, D]
  long long o_token, o_head;
  float* lse;                        // [Nq, Hq] or nullptr
  const int* cu_q;                   // [B + 1]
  const int* cu_k;
  long long Nq, Nk;
  int B, Hq, Hk, group, D;
  int bf16, causal, o_vec;
  float scale;
  // by the plan: CTAs that share a tile's keys, [splits][Nq][Hq][D] means over their keys, [splits][Nq][Hq] their maxima and sums of weights
  int splits;
  float* parts;
  float2* stats;
  DeviceStatus* status;
};

struct PromptPlan {
  int pack_q, pack_k, pack_v;        // rows that are copied to aligned ones first
  int splits;                        // CTAs that share a tile's keys
  long long q_bytes, k_bytes, v_bytes, parts_bytes, stats_bytes;
  long long bytes() const { return q_bytes + k_bytes + v_bytes + parts_bytes + stats_bytes; }
};

PromptPlan plan_prompt(const PromptParams& p, int sms);
void launch_prompt(const PromptParams& p, const PromptPlan& plan, void* workspace, cudaStream_t s);

}  // namespace raiccl
