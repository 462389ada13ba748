// Attention of one new token of each sequence over the paged cache in 4 bits.
//
//   z_j = scale q . k_j,   out = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m)
//
// in one pass over the cache, with the running maximum m and sum l of a softmax.
// The floor is the cache's own bytes, 9/16 of a byte a number.
//
// Work.  Tiles of 64 tokens of one sequence and one key head, in the order of
// sequences and heads, are dealt to the CTAs in equal contiguous shares, and a
// CTA's share to its warps.  A warp is on its own from the first tile to the
// last: it copies its tiles to its own ring in shared memory (cp.async), and meets
// no other before its share is done.  What it has of a sequence
// whose tiles others have too is joined then, in a fixed order: within the CTA
// through shared memory, between CTAs by a second, small kernel.
//
// Products.  Tokens are the 16-row operand of mma.sync (m16n8k16, f16, fp32
// sums), the group's query heads its eight columns: the operand that comes from
// the cache goes straight from its 4 bits into registers.  A lane takes D / 4
// consecutive numbers of a key (the dimensions' order within the product is
// free) and D / 8 of each of four values, so that both are read as they lie.  A
// code times its scale has at most 6 bits and is exact in f16.  tcgen05 has no
// mixed product of f16 by 4 bits with scales along the rows; the operand would
// have to be written back to shared memory, twice the bytes that a tile reads.
//
// The sums S^T = K Q^T come out with tokens as rows; movmatrix turns two 8 x 8
// blocks of exp(S) into the other operand of out^T = V^T P^T.
//
// What bounds it.  64 sequences of 16384 tokens, 8 key heads of 128: 219 to 253 us
// by the box, 4.8 to 5.5 TB/s of the cache, where a copy reaches 6.4.  A tile of 32 tokens takes 520
// instructions of a warp, 128 of them conversions and as many products by scales,
// at half rate each: schedulers issue in 60 % of cycles, the ALUs are busy in 52 %.
// More, smaller warps (128 registers) moved and spilled (790 instructions); one
// warp that loads for all (bulk copies) could not keep up (408 us).  Few tokens
// are a chain of latencies: lengths, table, tiles, join (1000 tokens: 11 us).  More
// than 16 query heads to a key head (8 with two parts) go through the cache again
// for each such chunk: 16 sequences of 16384 tokens, 128 heads over one, 106 us,
// where one pass over the cache would be 6 at copy speed.
//
// Roundings.  Queries are scaled by a power of two and held in f16 (bf16 queries
// exactly but for numbers 2^-14 below the row's largest, which lose bits below
// 2^-25 of it), fp32 queries as two f16 parts (2^-22 of a number's size).  Probabilities go into
// the second product in f16 (2^-12 of each, unbiased, small against a bf16
// result's own 2^-9), for fp32 results in two parts.  Maxima, sums and outputs
// are fp32.  Tensor-core sums are cut rather than rounded, so for fp32 results
// they leave it every 32 tokens.
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <stdexcept>
#include <type_traits>

#include "attention.h"
#include "attention_join.cuh"
#include "serving.h"
#include "serving_device.cuh"
#include "sm100_ptx.cuh"

namespace raiccl {

// Probabilities are exp2(z - m + 7) and m follows the maximum once that passes 15: f16 holds them (below 2^15), and small
// ones keep their bits down to 2^-21 of the largest.
constexpr float kCachedHead = 7.f, kCachedRoom = 15.f;

// Warps of a CTA, by the registers that queries, sums and the operands in flight take.
template <int NT, int PARTS>
constexpr int kCachedWarps = NT == 1 && PARTS == 1 ? 12 : 8;

template <int D, int NT, int PARTS>
struct Cached {
  static constexpr int WARPS = kCachedWarps<NT, PARTS>, THREADS = 32 * WARPS;
  static constexpr int HEADS = 8 * NT;                       // query heads of a chunk at most
  static constexpr int CODES = kCachedTile * D / 2, SCALES = kCachedTile * D / 16;
  static constexpr int STAGE = 2 * (CODES + SCALES);         // K codes, V codes, K scales, V scales
  static constexpr int PART = HEADS * D * 4;                 // a warp's sums of a sequence that it shares
  static constexpr int STAGES = 216 * 1024 / (WARPS * STAGE) < 4 ? 216 * 1024 / (WARPS * STAGE) : 4;
  static constexpr int SMEM = WARPS * STAGES * STAGE;
  static_assert(STAGES >= 2 && STAGES * STAGE >= PART, "the ring holds the warp's last part too");
};

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Four bytes of two codes each as f16 pairs, lower code first.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

// Two e4m3 numbers (the lower sixteen bits) as an f16 pair.
__device__ __forceinline__ uint32_t scales_f16(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  return h;
}

__device__ __forceinline__ uint32_t mul_f16(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *(const uint32_t*)&h;
}

// What f16 rounding leaves of two numbers, in f16.
__device__ __forceinline__ uint32_t rest_f16(float lo, float hi, uint32_t rounded) {
  const float2 f = __half22float2(*(const __half2*)&rounded);
  return pack_f16(lo - f.x, hi - f.y);
}

// Tokens of a sequence, within its row of the table, from the length read.
__device__ __forceinline__ int cached_tokens(const CachedParams& p, int n) {
  const long long most = (long long)p.table_pages << p.c.page_shift;
  return n < 0 ? 0 : (long long)n > most ? (int)most : n;
}
__device__ __forceinline__ int cached_length(const CachedParams& p, int b) { return cached_tokens(p, __ldg(p.lengths + b)); }

// Tiles of n tokens, which may be 2^31 - 16.
__device__ __forceinline__ int tiles_of(int n) { return n / kCachedTile + (n % kCachedTile != 0); }
__device__ __forceinline__ int cached_tiles(const CachedParams& p, int b) { return tiles_of(cached_length(p, b)); }

// CTAs that take part (two tiles to one at least), the first tile of one, and the CTA of a tile.
__device__ __forceinline__ int cached_ctas(long long tiles, int ctas) {
  const long long most = (tiles + 1) / 2;
  return most < ctas ? (int)most : ctas;
}
// The first tiles % ctas CTAs have one tile more than the others.
__device__ __forceinline__ long long divide_tiles(long long a, long long b) {
  return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}
__device__ __forceinline__ long long cached_first(long long tiles, int ctas, int c) {
  const long long each = divide_tiles(tiles, ctas), more = tiles - each * ctas;
  return each * c + (c < more ? c : more);
}
__device__ __forceinline__ int cached_cta(long long tiles, int ctas, long long tile) {
  const long long each = divide_tiles(tiles, ctas), more = tiles - each * ctas, behind = tile - more * (each + 1);
  return (int)(behind < 0 ? divide_tiles(tile, each + 1) : more + divide_tiles(behind, each));
}

// A sequence and chunk of heads, as a piece of the order of all tiles.
struct CachedPiece {
  int b, hc, n;        // tiles
  long long first;     // its first tile
};

__device__ __forceinline__ void next_piece(const CachedParams& p, CachedPiece& s) {
  s.first += s.n;
  if (++s.hc < p.c.heads * p.chunks) return;
  s.hc = 0;
  do {
    ++s.b;
    s.n = s.b < p.B ? cached_tiles(p, s.b) : 1;
  } while (s.n == 0);
}

__device__ __forceinline__ int piece_heads(const CachedParams& p, int hc, int& head) {
  const int kv = hc / p.chunks, chunk = hc - kv * p.chunks;
  head = kv * p.group + chunk * p.chunk;
  const int left = p.group - chunk * p.chunk;
  return left < p.chunk ? left : p.chunk;
}

__device__ __forceinline__ float cached_lse(float m, float l) { return (m + log2f(l)) * 0.69314718055994531f; }

// Four outputs of a row from sums and the reciprocal of l.
__device__ __forceinline__ void cached_store4(const CachedParams& p, int b, int head, int d, float4 v) {
  const long long at = b * p.o_seq + head * p.o_head + d;
  if (p.out_bf16) {
    __nv_bfloat16* o = (__nv_bfloat16*)p.out + at;
    const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
    if (p.o_vec) *(uint2*)o = make_uint2(*(const uint32_t*)&x, *(const uint32_t*)&y);
    else { o[0] = x.x; o[1] = x.y; o[2] = y.x; o[3] = y.y; }
  } else {
    float* o = (float*)p.out + at;
    if (p.o_vec) *(float4*)o = v;
    else { o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w; }
  }
}

// The result's row from sums over a warp.
template <int N>
__device__ __forceinline__ void cached_row(const CachedParams& p, int b, int head, float top, float l, const float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  const float r = l == 0.f ? 0.f : p.c.v_unit / l;
  const long long at = b * p.o_seq + head * p.o_head + N * lane;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    if (p.out_bf16) {
      const __nv_bfloat162 x = __floats2bfloat162_rn(v[i] * r, v[i + 1] * r);
      __nv_bfloat16* const o = (__nv_bfloat16*)p.out + at + i;
      if (p.o_vec) *(__nv_bfloat162*)o = x;
      else { o[0] = x.x; o[1] = x.y; }
    } else {
      float* const o = (float*)p.out + at + i;
      if (p.o_vec) *(float2*)o = make_float2(v[i] * r, v[i + 1] * r);
      else { o[0] = v[i] * r; o[1] = v[i + 1] * r; }
    }
  }
  if (p.lse != nullptr && lane == 0) p.lse[(long long)b * p.Hq + head] = cached_lse(top, l);
}

// A warp's part of a piece that it shares; used: 1 the sums are in its ring, 2 in device memory.
struct CachedPart {
  CachedPiece s;
  int used;
};

// A piece that warps of a CTA share: the first of them and the side of its part, the warp behind the last; where the sum goes:
// the CTA's parts 0 (it began before the CTA's share) and 1 (it ends after it), 2 the output.
struct CachedChain {
  int warp, side, end, b, head0, heads, where;
  long long last;      // its last tile
};

template <int D, int NT, int PARTS>
__global__ void __launch_bounds__(Cached<D, NT, PARTS>::THREADS, 1) cached_kernel(CachedParams p) {
  using C = Cached<D, NT, PARTS>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long before[C::THREADS + 1], sum_of[C::WARPS], base_of[C::WARPS];
  __shared__ CachedChain chain[C::WARPS + 1];
  __shared__ int chains;
  __shared__ uint32_t all_with;
  __shared__ CachedPart part[C::WARPS][2];
  __shared__ float2 stat[C::WARPS][2][C::HEADS];
  __shared__ int nonempty[C::WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  griddep_wait();
  griddep_launch_dependents();
  if (p.notes && tid == 0) p.joins[blockIdx.x].heads = 0;   // none, unless a piece is found to go on behind this CTA's share

  // ------------------------------------------------------------ all tiles, and this CTA's and this warp's
  const int HC = p.c.heads * p.chunks, per = (p.B + C::THREADS - 1) / C::THREADS;
  {
    long long n = 0;
    for (int b = tid * per; b < p.B && b < (tid + 1) * per; ++b) {
      const int len = __ldg(p.lengths + b);
      const long long most = (long long)p.table_pages << p.c.page_shift;
      if (blockIdx.x == 0 && (len < 0 || (long long)len > most)) record_status(p.status, kBoundsViolation, kCachedKernelId, len, most);
      n += cached_tiles(p, b);
    }
    long long sum = n;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const long long up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) sum_of[warp] = sum;
    __syncthreads();
    long long base = 0;
    for (int w = 0; w < warp; ++w) base += sum_of[w];
    before[tid + 1] = (base + sum) * HC;
    if (tid == 0) before[0] = 0;
    if (lane == 0) base_of[warp] = base * HC;
    __syncthreads();
  }
  const long long tiles = before[C::THREADS];
  if (tiles == 0) return;
  const int ctas = cached_ctas(tiles, p.ctas);
  if ((int)blockIdx.x >= ctas) return;
  const long long c0 = cached_first(tiles, ctas, blockIdx.x), c1 = cached_first(tiles, ctas, blockIdx.x + 1);
  const int share = (int)(c1 - c0);
  // A warp's part of a sequence: the one that began before its share (0), the one that ends after it (1).  The last that it
  // works on goes into its ring, which is done then; a first one with others behind it to device memory.
  auto spilled = [&](int w) { return p.spill + ((long long)blockIdx.x * C::WARPS + w) * (C::HEADS * D); };
  auto ringed = [&](int w) { return (float*)(smem + w * C::STAGES * C::STAGE); };
  auto piece_at = [&](long long u) {
    // the last thread whose sequences begin at or before u: its warp, then itself
    const uint32_t w = __ballot_sync(0xffffffffu, lane < C::WARPS && base_of[lane < C::WARPS ? lane : 0] <= u);
    const int in = 31 - __clz(w);
    const uint32_t m = __ballot_sync(0xffffffffu, before[32 * in + lane] <= u);
    const int lo = 32 * in + 31 - __clz(m);
    long long first = before[lo];
    int b = lo * per, n = cached_tiles(p, b);
    while (first + (long long)n * HC <= u) {
      first += (long long)n * HC;
      n = cached_tiles(p, ++b);
    }
    const int hc = (int)((uint32_t)(u - first) / (uint32_t)n);
    return CachedPiece{b, hc, n, first + (long long)hc * n};
  };

  const long long u0 = c0 + share / C::WARPS * warp + min(warp, share % C::WARPS);
  const int count = share / C::WARPS + (warp < share % C::WARPS);
  const long long u1 = u0 + count;
  uint8_t* const ring = smem + warp * C::STAGES * C::STAGE;
  if (lane == 0) {
    part[warp][0].used = part[warp][1].used = 0;
    nonempty[warp] = count > 0;
  }
  __syncwarp();

  if (count > 0) {
    CachedPiece piece = piece_at(u0);

    // ---------------------------------------------------------- copies, STAGES tiles ahead
    // Sixteen bytes to a lane and copy.  Of a tile, or of the page that is a part of it: K codes, V codes, the scales of both.
    const uint32_t page_mask = (1u << p.c.page_shift) - 1, page_bytes = ((uint32_t)p.c.heads << p.c.page_shift) * (D / 2);
    const uint32_t ring_at = smem_u32(ring);
    auto copy = [&](uint32_t stage_at, int row_to, int page, uint32_t row, auto rows_of) {
      constexpr int ROWS = decltype(rows_of)::value, SCALES = ROWS * (D / 16), N = SCALES / 16;
      const unsigned long long off = (unsigned long long)(uint32_t)page * page_bytes + row * (D / 2);
      const uint8_t *k = p.c.k_codes + off + lane * 16, *v = p.c.v_codes + off + lane * 16;
      const uint32_t to = stage_at + row_to * (D / 2) + lane * 16;
#pragma unroll
      for (int i = 0; i < ROWS * (D / 2); i += 512) {
        cp_async16(to + i, k + i);
        cp_async16(to + C::CODES + i, v + i);
      }
      const uint32_t mine = (lane & (N - 1)) * 16, st = stage_at + 2 * C::CODES + row_to * (D / 16) + mine;
      if constexpr (N == 32) {
        cp_async16(st, p.c.k_scales + (off >> 3) + mine);
        cp_async16(st + C::SCALES, p.c.v_scales + (off >> 3) + mine);
      } else if (lane < 2 * N) {                   // both in one copy
        cp_async16(st + (lane < N ? 0 : C::SCALES), (lane < N ? p.c.k_scales : p.c.v_scales) + (off >> 3) + mine);
      }
    };
    CachedPiece ahead = piece;
    int ahead_len = cached_length(p, piece.b), ahead_at = (int)(u0 - piece.first) * kCachedTile;   // the next copy's tokens
    int ahead_end = (int)min((long long)count, piece.first + piece.n - u0);                         // tiles of the share up to the piece's end
    const int* ahead_pages = p.table + (long long)piece.b * p.table_stride;
    uint32_t ahead_row = (uint32_t)(piece.hc / p.chunks) << p.c.page_shift;
    int issued = 0, fill = 0;
    uint32_t missing = 0;                          // sixteens of tokens without a page of the cache: four bits to a stage
    auto issue = [&]() {
      if (issued == ahead_end) {
        next_piece(p, ahead);
        ahead_len = cached_length(p, ahead.b);
        ahead_at = 0;
        ahead_end = (int)min((long long)count, (long long)ahead_end + ahead.n);
        ahead_pages = p.table + (long long)ahead.b * p.table_stride;
        ahead_row = (uint32_t)(ahead.hc / p.chunks) << p.c.page_shift;
      }
      const uint32_t stage_at = ring_at + fill * C::STAGE;
      uint32_t lost = 0;
      if (p.c.page_shift >= 6) {
        const int page = __ldg(ahead_pages + (ahead_at >> p.c.page_shift));
        if ((uint32_t)page < (uint32_t)p.c.pages) {
          copy(stage_at, 0, page, ahead_row + (ahead_at & page_mask), std::integral_constant<int, 64>{});
        } else {
          lost = 15;
          if (lane == 0) record_status(p.status, kBoundsViolation, kCachedKernelId, page, p.c.pages);
        }
      } else {                                     // several pages: their numbers first, by a lane each
        const int at = ahead_at + ((lane & 3) << p.c.page_shift);
        const bool is = lane < (kCachedTile >> p.c.page_shift) && at < ahead_len;
        int page = is ? __ldg(ahead_pages + (at >> p.c.page_shift)) : -1;
        if (is && (uint32_t)page >= (uint32_t)p.c.pages) {
          record_status(p.status, kBoundsViolation, kCachedKernelId, page, p.c.pages);
          page = -1;
        }
        if (p.c.page_shift == 5) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int one = __shfl_sync(0xffffffffu, page, r);
            if (one >= 0) copy(stage_at, 32 * r, one, ahead_row, std::integral_constant<int, 32>{});
            else lost |= 3u << (2 * r);
          }
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int one = __shfl_sync(0xffffffffu, page, r);
            if (one >= 0) copy(stage_at, 16 * r, one, ahead_row, std::integral_constant<int, 16>{});
            else lost |= 1u << r;
          }
        }
      }
      missing = (missing & ~(15u << (4 * fill))) | lost << (4 * fill);
      ++issued;
      ahead_at += kCachedTile;
      fill = fill + 1 == C::STAGES ? 0 : fill + 1;
    };

    // ---------------------------------------------------------- tiles
    constexpr int KS = D / 16;         // products of a row of sixteen tokens over D
    constexpr int DM = D / 16;         // blocks of sixteen dimensions of the output
    uint32_t bq[PARTS][NT][KS][2];
    float mult[NT][2];                 // from sums to logits in powers of two, heads 8 nt + 2t and 2t + 1
    float m[NT][2], l[NT][2];
    float o[DM][NT][4];
    int head0 = 0, heads = 0;

    auto begin = [&]() {
      heads = piece_heads(p, piece.hc, head0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = 8 * nt + g;
        float x[D / 4];
#pragma unroll
        for (int i = 0; i < D / 4; ++i) x[i] = 0.f;
        if (h < heads) {
          const long long at = piece.b * p.q_seq + (head0 + h) * p.q_head + t * (D / 4);
          if (p.bf16) {
            const __nv_bfloat16* q = (const __nv_bfloat16*)p.q + at;
            if (p.q_vec) {
#pragma unroll
              for (int i = 0; i < D / 4; i += 8) {
                float f[8];
                unpack16<__nv_bfloat16>(*(const uint4*)(q + i), f);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[i + j] = f[j];
              }
            } else {
#pragma unroll
              for (int i = 0; i < D / 4; ++i) x[i] = __bfloat162float(q[i]);
            }
          } else {
            const float* q = (const float*)p.q + at;
            if (p.q_vec) {
#pragma unroll
              for (int i = 0; i < D / 4; i += 4) *(float4*)(x + i) = *(const float4*)(q + i);
            } else {
#pragma unroll
              for (int i = 0; i < D / 4; ++i) x[i] = q[i];
            }
          }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the power of two at or below the largest (1 for infinities, the least normal number for what lies below it), and its reciprocal
        uint32_t e = __float_as_uint(top) >> 23;
        if (e == 0) e = 1;
        if (e == 255) e = 127;
        if (e > 253) e = 253;
        const float down = __uint_as_float((254u - e) << 23);
        const float up = scalbnf(p.mult, (int)e - 127 + p.mult_exp);   // one after the other, the factors may overflow
        mult[nt][0] = __shfl_sync(0xffffffffu, up, 8 * t);
        mult[nt][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
#pragma unroll
        for (int i = 0; i < D / 4; i += 2) {
          const float a = x[i] * down, b = x[i + 1] * down;
          const uint32_t w = pack_f16(a, b);
          bq[0][nt][i / 4][(i / 2) & 1] = w;
          if constexpr (PARTS == 2) bq[1][nt][i / 4][(i / 2) & 1] = rest_f16(a, b, w);
        }
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < DM; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][nt][j] = 0.f;
    };

    // The piece's end, for this warp: written where all its tiles were this warp's, else left for the join.
    auto finish = [&](bool last) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float s = l[nt][j];
          s += __shfl_xor_sync(0xffffffffu, s, 4);
          s += __shfl_xor_sync(0xffffffffu, s, 8);
          s += __shfl_xor_sync(0xffffffffu, s, 16);
          l[nt][j] = s;
        }
      const bool early = piece.first < u0, late = piece.first + piece.n > u1;
      if (!early && !late) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int h = 8 * nt + 2 * t + j;
            if (h >= heads) continue;
            const float s = l[nt][j], r = s == 0.f ? 0.f : p.c.v_unit / s;
#pragma unroll
            for (int i = 0; i < DM; i += 2)
              cached_store4(p, piece.b, head0 + h, g * (D / 8) + 2 * i,
                            make_float4(o[i][nt][j] * r, o[i][nt][j + 2] * r, o[i + 1][nt][j] * r, o[i + 1][nt][j + 2] * r));
            if (p.lse != nullptr && g == 0) p.lse[(long long)piece.b * p.Hq + head0 + h] = cached_lse(m[nt][j], s);
          }
        return;
      }
      const int side = early ? 0 : 1;
      if (lane == 0) part[warp][side] = {piece, last ? 1 : 2};
      float* const at = last ? ringed(warp) : spilled(warp);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int h = 8 * nt + 2 * t + j;
          if (g == 0) stat[warp][side][h] = make_float2(m[nt][j], l[nt][j]);
#pragma unroll
          for (int i = 0; i < DM; i += 2)
            *(float4*)(at + h * D + g * (D / 8) + 2 * i) =
                make_float4(o[i][nt][j], o[i][nt][j + 2], o[i + 1][nt][j], o[i + 1][nt][j + 2]);
        }
    };

    // One loop, in which copies, beginnings and ends have one place each: with two places the code was a fifth longer (64 x
    // 16384 tokens 229 us, so 221).
    int stage = 0, end = 0, left = 0;   // tiles up to the piece's end; tokens of the piece from this tile on
#pragma unroll 1
    for (int done = -C::STAGES; done < count; ++done) {
     if (done >= 0) {
      if (done == end) {
        if (done > 0) next_piece(p, piece);
        begin();
        end = (int)min((long long)count, piece.first + piece.n - u0);
        left = cached_length(p, piece.b) - (done == 0 ? (int)(u0 - piece.first) * kCachedTile : 0);
      }
      cp_async_wait<C::STAGES - 1>();
      __syncwarp();
      uint8_t* const s = ring + stage * C::STAGE;
      const uint32_t lost = missing >> (4 * stage) & 15;
      const bool all = left >= kCachedTile && lost == 0;
      auto seen_at = [&](int row) -> uint32_t {      // tokens row .. row + 31 of the tile that the sequence has
        const int n = left - row;
        uint32_t has = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1;
        if (lost >> (row / 16) & 1) has &= 0xffff0000u;
        if (lost >> (row / 16) & 2) has &= 0x0000ffffu;
        return has;
      };
      if (!all) {
        // a page's rest may hold anything: its values count as zeros
#pragma unroll
        for (int row = 0; row < kCachedTile; row += 32) {
          if (seen_at(row) >> lane & 1) continue;
          uint8_t* const scales = s + 2 * C::CODES + C::SCALES + (row + lane) * (D / 16);
          if constexpr (D == 128) *(uint2*)scales = make_uint2(0, 0);
          else *(uint32_t*)scales = 0;
        }
        __syncwarp();
      }
#pragma unroll 1
      for (int half = 0; half < kCachedTile; half += 32) {   // 32 tokens at a time, by the registers that more would take
        const uint32_t seen = all ? 0xffffffffu : seen_at(half);
        if (seen == 0) continue;
        const uint8_t *const sk = s + half * (D / 2), *const ss = s + 2 * C::CODES + half * (D / 16);
        float z[2][NT][4];
        // -------------------------------------------------- S^T = K Q^T
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) z[mt][nt][j] = 0.f;
          uint32_t w[2][D / 32], sc[2][D / 64];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int row = 16 * mt + 8 * r + g;
            if constexpr (D == 128) {
              const uint4 v = *(const uint4*)(sk + row * 64 + 16 * t);
              w[r][0] = v.x; w[r][1] = v.y; w[r][2] = v.z; w[r][3] = v.w;
              const uint32_t two = scales_f16(*(const uint16_t*)(ss + row * 8 + 2 * t));
              sc[r][0] = __byte_perm(two, two, 0x1010);
              sc[r][1] = __byte_perm(two, two, 0x3232);
            } else {
              const uint2 v = *(const uint2*)(sk + row * 32 + 8 * t);
              w[r][0] = v.x; w[r][1] = v.y;
              const uint32_t two = scales_f16(ss[row * 4 + t]);
              sc[r][0] = __byte_perm(two, two, 0x1010);
            }
          }
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            uint32_t lo[4], hi[4];
            codes_f16(w[0][j], lo);
            codes_f16(w[1][j], hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              lo[i] = mul_f16(lo[i], sc[0][j / 2]);
              hi[i] = mul_f16(hi[i], sc[1][j / 2]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t a[4] = {lo[2 * k], hi[2 * k], lo[2 * k + 1], hi[2 * k + 1]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = PARTS - 1; q >= 0; --q) mma_f16(z[mt][nt], a, bq[q][nt][2 * j + k][0], bq[q][nt][2 * j + k][1]);
            }
          }
        }
        // -------------------------------------------------- softmax
        // x = z - m by one fma: off by a rounding of the difference, not of the logit
        float x[2][NT][4];
        auto below = [&]() {
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 4; ++j) x[mt][nt][j] = fmaf(z[mt][nt][j], mult[nt][j & 1], -m[nt][j & 1]);
          if (!all) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (!(seen >> (16 * mt + 8 * (j >> 1) + g) & 1)) x[mt][nt][j] = -INFINITY;
          }
        };
        below();
        float most = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) most = fmaxf(most, x[mt][nt][j]);
        if (__any_sync(0xffffffffu, most > kCachedRoom)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float top = -INFINITY;
#pragma unroll
              for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                  if (seen >> (16 * mt + 8 * r + g) & 1) top = fmaxf(top, z[mt][nt][j + 2 * r] * mult[nt][j]);
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
              const float now = fmaxf(m[nt][j], top - kCachedHead);
              const float shrink = now == -INFINITY ? 1.f : exp2_fast(m[nt][j] - now);
              m[nt][j] = now;
              l[nt][j] *= shrink;
#pragma unroll
              for (int i = 0; i < DM; ++i) {
                o[i][nt][j] *= shrink;
                o[i][nt][j + 2] *= shrink;
              }
            }
          below();
        }
        uint32_t bp[PARTS][2][NT][2];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              e[j] = exp2_fast(x[mt][nt][j]);
              l[nt][j & 1] += e[j];
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint32_t h = pack_f16(e[2 * r], e[2 * r + 1]);
              bp[0][mt][nt][r] = transpose8(h);
              if constexpr (PARTS == 2) bp[1][mt][nt][r] = transpose8(rest_f16(e[2 * r], e[2 * r + 1], h));
            }
          }
        // -------------------------------------------------- out^T += V^T P^T
        // words of four tokens; pairs of tokens to one register by their nibbles
        constexpr int WV = D / 64;     // words of a lane's D / 8 numbers
        float fresh[PARTS == 2 ? DM : 1][NT][4];
        if constexpr (PARTS == 2) {
#pragma unroll
          for (int i = 0; i < DM; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 4; ++j) fresh[i][nt][j] = 0.f;
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t pair[2][2][WV], sv[2];   // [tokens 2t, 2t + 1 / + 8][even, odd dimensions]
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t y[2][WV], byte[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = 16 * mt + 8 * r + 2 * t + e;
              if constexpr (D == 128) {
                const uint2 v = *(const uint2*)(sk + C::CODES + row * 64 + 8 * g);
                y[e][0] = v.x; y[e][1] = v.y;
                byte[e] = ss[C::SCALES + row * 8 + g];
              } else {
                y[e][0] = *(const uint32_t*)(sk + C::CODES + row * 32 + 4 * g);
                byte[e] = ss[C::SCALES + row * 4 + (g >> 1)];
              }
            }
            sv[r] = scales_f16(byte[0] | byte[1] << 8);
#pragma unroll
            for (int i = 0; i < WV; ++i) {
              pair[r][0][i] = (y[0][i] & 0x0f0f0f0fu) | ((y[1][i] << 4) & 0xf0f0f0f0u);
              pair[r][1][i] = ((y[0][i] >> 4) & 0x0f0f0f0fu) | (y[1][i] & 0xf0f0f0f0u);
            }
          }
#pragma unroll
          for (int i = 0; i < WV; ++i) {
            uint32_t h[2][2][4];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                codes_f16(pair[r][e][i], h[r][e]);
#pragma unroll
                for (int y = 0; y < 4; ++y) h[r][e][y] = mul_f16(h[r][e][y], sv[r]);
              }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t a[4] = {h[0][0][y], h[0][1][y], h[1][0][y], h[1][1][y]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = PARTS - 1; q >= 0; --q)
                  mma_f16(PARTS == 2 ? fresh[PARTS == 2 ? 4 * i + y : 0][nt] : o[4 * i + y][nt], a, bp[q][mt][nt][0], bp[q][mt][nt][1]);
            }
          }
        }
        if constexpr (PARTS == 2) {
#pragma unroll
          for (int i = 0; i < DM; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[i][nt][j] += fresh[i][nt][j];
        }
      }
      left -= kCachedTile;
      if (++stage == C::STAGES) stage = 0;
      __syncwarp();   // every lane has read the tile
      if (done + 1 == end) finish(done + 1 == count);
     }
     if (issued < count) issue();
     cp_async_commit();
    }
  }

  // ------------------------------------------------------------ the CTA's shared pieces
  __syncthreads();
  // A piece's parts: its first one (a tail, or the head of the CTA's first warp), then the heads of the warps behind it, up
  // to the one that it ends in.  The warps between have shares, if the CTA has tiles for all of them.
  if (warp == 0) {
    const bool mine = lane < C::WARPS && nonempty[lane < C::WARPS ? lane : 0];
    const uint32_t with = __ballot_sync(0xffffffffu, mine);
    const bool tail = mine && part[lane][1].used, head = mine && part[lane][0].used && lane == __ffs(with) - 1;
    const uint32_t tails = __ballot_sync(0xffffffffu, tail), heads = __ballot_sync(0xffffffffu, head);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      if (!(side ? tail : head)) continue;
      const CachedPiece s = part[lane][side].s;
      int end = lane + 1, parts = 1;
      for (; end < C::WARPS; ++end) {
        if (!(with >> end & 1)) continue;
        if (!part[end][0].used || part[end][0].s.first != s.first) break;
        ++parts;
      }
      int head0;
      const int nheads = piece_heads(p, s.hc, head0);
      const bool early = s.first < c0, late = s.first + s.n > c1;
      chain[(heads != 0) * side + (side ? __popc(tails & ((1u << lane) - 1)) : 0)] = {lane,  side,   end,
                                                                                      s.b,   head0,  nheads,
                                                                                      early ? 0 : late ? 1 : 2, s.first + s.n - 1};
    }
    if (lane == 0) { chains = __popc(tails) + (heads != 0); all_with = with; }
  }
  __syncthreads();
  for (int i = warp; i < chains * C::HEADS; i += C::WARPS) {   // a warp to a head of a piece
    const CachedChain x = chain[i / C::HEADS];
    const int h = i % C::HEADS;
    if (h >= x.heads) continue;
    auto side_of = [&](int w) { return w == x.warp ? x.side : 0; };
    float top, l, v[D / 32];
    warp_join<D>(
        x.end - x.warp, [&](int j) { return all_with >> (x.warp + j) & 1 ? stat[x.warp + j][side_of(x.warp + j)][h] : make_float2(-INFINITY, 0.f); },
        [&](int j) {
          const int w = x.warp + j;
          return (!(all_with >> w & 1) || part[w][side_of(w)].used == 1 ? ringed(w) : spilled(w)) + h * D;
        },
        top, l, v);
    if (x.where == 2) {
      cached_row(p, x.b, x.head0 + h, top, l, v);
    } else {
      const long long at = ((long long)blockIdx.x * 2 + x.where) * p.chunk + h;
      store_lanes<D>(p.parts + at * D, v);
      if (lane == 0) {
        p.stats[at] = make_float2(top, l);
        if (p.notes && x.where == 1 && h == 0) p.joins[blockIdx.x] = {x.b, x.head0, x.heads, x.last, tiles};
      }
    }
  }
}

// Pieces that several CTAs share, one head to a CTA; a warp takes every eighth part.  Empty sequences too, which no tile stands for.
//
// With no more pieces than CTAs in the kernel before, a CTA to each piece finds out whose parts it has from the lengths.  They are
// final once this kernel runs at all, since every CTA of the kernel before lets it start only after its own wait, so that is done
// ahead of the wait for the parts (one sequence of 1000 tokens 13.5 -> 11.0 us, 37 ragged ones 25.0 -> 22.8).  Read from L2, which
// the lengths' writer has reached: no wait of this kernel's has dropped what this SM's L1 may hold of them.
//
// With more pieces that would read the lengths by the square of the batch (65536 sequences of one token: 129 ms, now 1.3; 4096: 940
// us, now 83).  A CTA of the kernel before has at most one piece that begins in its share and ends behind it, and leaves a note of
// it (p.joins) for the CTA here; empty sequences are found by a lane each.  (32 sequences of 100 tokens, 256 pieces: 14.0 -> 11.5
// us.  With notes, one sequence of 1000 tokens took 11.2 us instead of 10.8, by one more load behind the wait.)
template <int D>
__global__ void __launch_bounds__(256) cached_join_kernel(CachedParams p) {
  __shared__ long long sum_of[2][8];
  __shared__ float4 acc[8][D / 4];
  __shared__ float2 ml[8];
  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const auto tiles_at = [&](int i) { return tiles_of(cached_tokens(p, __ldcg(p.lengths + i))); };
  int b = 0, head0 = 0, heads = 0, c0 = blockIdx.x, c1 = c0;
  if (!p.notes) {
    const int HC = p.c.heads * p.chunks;
    b = blockIdx.x / HC;
    const int hc = blockIdx.x - b * HC;
    heads = piece_heads(p, hc, head0);
    long long all = 0, ahead = 0;
    for (int i = threadIdx.x; i < p.B; i += 256) {
      const int n = tiles_at(i);
      all += n;
      if (i < b) ahead += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, o);
      ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    }
    if (lane == 0) { sum_of[0][warp] = all; sum_of[1][warp] = ahead; }
    __syncthreads();
    all = ahead = 0;
    for (int w = 0; w < 8; ++w) { all += sum_of[0][w]; ahead += sum_of[1][w]; }
    const int n = tiles_at(b);
    c0 = c1 = 0;
    if (n > 0) {
      const long long tiles = all * HC, first = ahead * HC + (long long)hc * n;
      const int ctas = cached_ctas(tiles, p.ctas);
      c0 = cached_cta(tiles, ctas, first);
      c1 = cached_cta(tiles, ctas, first + n - 1);
    } else if (warp == 0 && h < heads) {   // (nothing before this kernel's predecessor is still at work on the result)
      const float zeros[D / 32] = {};
      cached_row(p, b, head0 + h, -INFINITY, 0.f, zeros);
    }
  } else {
    for (int b0 = 32 * (warp * gridDim.x + blockIdx.x); b0 < p.B; b0 += 256 * gridDim.x) {
      const bool none = b0 + lane < p.B && tiles_at(b0 + lane) == 0;
      for (uint32_t empty = __ballot_sync(0xffffffffu, none); empty != 0; empty &= empty - 1)
        for (int head = h; head < p.Hq; head += gridDim.y) {
          const float zeros[D / 32] = {};
          cached_row(p, b0 + __ffs(empty) - 1, head, -INFINITY, 0.f, zeros);
        }
    }
  }
  griddep_wait();
  griddep_launch_dependents();
  if (p.notes) {
    const CachedJoin join = p.joins[c0];
    b = join.b;
    head0 = join.head0;
    heads = join.heads;
    if (heads > 0) c1 = cached_cta(join.tiles, cached_ctas(join.tiles, p.ctas), join.last);
  }
  if (h >= heads || c0 == c1) return;
  float m = -INFINITY, l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool mine = lane < D / 4;
#pragma unroll 4
  for (int c = c0 + warp; c <= c1; c += 8) {
    const long long at = ((long long)c * 2 + (c == c0 ? 1 : 0)) * p.chunk + h;
    const float2 st = p.stats[at];
    const float4 a = mine ? *(const float4*)(p.parts + at * D + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float top = fmaxf(m, st.x);
    const float f0 = m == -INFINITY ? (l == 0.f ? 0.f : NAN) : exp2_fast(m - top);
    const float f1 = st.x == -INFINITY ? (st.y == 0.f ? 0.f : NAN) : exp2_fast(st.x - top);
    m = top;
    l = l * f0 + st.y * f1;
    v.x = v.x * f0 + a.x * f1; v.y = v.y * f0 + a.y * f1; v.z = v.z * f0 + a.z * f1; v.w = v.w * f0 + a.w * f1;
  }
  if (mine) acc[warp][lane] = v;
  if (lane == 0) ml[warp] = make_float2(m, l);
  __syncthreads();
  if (warp != 0 || !mine) return;
  m = -INFINITY;
  for (int w = 0; w < 8; ++w) m = fmaxf(m, ml[w].x);
  l = 0.f;
  v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = 0; w < 8; ++w) {
    const float f = ml[w].x == -INFINITY ? (ml[w].y == 0.f ? 0.f : NAN) : exp2_fast(ml[w].x - m);
    const float4 a = acc[w][lane];
    l = fmaf(ml[w].y, f, l);
    v.x = fmaf(a.x, f, v.x); v.y = fmaf(a.y, f, v.y); v.z = fmaf(a.z, f, v.z); v.w = fmaf(a.w, f, v.w);
  }
  const float r = l == 0.f ? 0.f : p.c.v_unit / l;
  cached_store4(p, b, head0 + h, 4 * lane, make_float4(v.x * r, v.y * r, v.z * r, v.w * r));
  if (p.lse != nullptr && lane == 0) p.lse[(long long)b * p.Hq + head0 + h] = cached_lse(m, l);
}

// Query heads that are worked on together: up to 16 of a group, 8 where queries and probabilities have two parts.
CachedPlan plan_cached(const CachedParams& p, int sms) {
  CachedPlan plan{};
  const int most = p.bf16 && p.out_bf16 ? 16 : 8;
  plan.chunks = (p.group + most - 1) / most;
  plan.chunk = (p.group + plan.chunks - 1) / plan.chunks;
  plan.ctas = sms;
  plan.parts_bytes = (long long)plan.ctas * 2 * plan.chunk * p.c.D * 4;
  plan.stats_bytes = ((long long)plan.ctas * 2 * plan.chunk * 8 + 255) / 256 * 256;
  const int warps = most == 8 ? kCachedWarps<1, 2> : plan.chunk <= 8 ? kCachedWarps<1, 1> : kCachedWarps<2, 1>;
  plan.spill_bytes = (long long)plan.ctas * warps * (plan.chunk > 8 ? 16 : 8) * p.c.D * 4;
  plan.joins_bytes = plan.ctas * (long long)sizeof(CachedJoin);
  return plan;
}

template <int D, int NT, int PARTS>
static void launch_cached_as(const CachedParams& p, cudaStream_t s) {
  using C = Cached<D, NT, PARTS>;
  auto kern = cached_kernel<D, NT, PARTS>;
  static std::atomic<unsigned long long> configured;   // by device
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
      throw std::runtime_error("attention_cached: shared memory");
    configured.fetch_or(bit);
  }
  launch_with_pdl(kern, dim3(p.ctas), dim3(C::THREADS), C::SMEM, s, true, p);
  launch_with_pdl(cached_join_kernel<D>, dim3(p.notes ? p.ctas : p.B * p.c.heads * p.chunks, p.chunk), dim3(256), 0, s, true, p);
}

void launch_cached(const CachedParams& params, const CachedPlan& plan, void* workspace, cudaStream_t s) {
  CachedParams p = params;
  p.chunk = plan.chunk;
  p.chunks = plan.chunks;
  p.ctas = plan.ctas;
  p.notes = (long long)p.B * p.c.heads * p.chunks > p.ctas;
  p.parts = (float*)workspace;
  p.stats = (float2*)((char*)workspace + plan.parts_bytes);
  p.spill = (float*)((char*)workspace + plan.parts_bytes + plan.stats_bytes);
  p.joins = (CachedJoin*)((char*)workspace + plan.parts_bytes + plan.stats_bytes + plan.spill_bytes);
  const bool two = !(p.bf16 && p.out_bf16);
  if (p.c.D == 128) {
    if (two) launch_cached_as<128, 1, 2>(p, s);
    else if (p.chunk > 8) launch_cached_as<128, 2, 1>(p, s);
    else launch_cached_as<128, 1, 1>(p, s);
  } else {
    if (two) launch_cached_as<64, 1, 2>(p, s);
    else if (p.chunk > 8) launch_cached_as<64, 2, 1>(p, s);
    else launch_cached_as<64, 1, 1>(p, s);
  }
}

}  // namespace raiccl
