// out = act(x w^T + bias) + residual: a dense product with its epilogue, from
// one row to a whole batch, any sizes.
#include <algorithm>
#include <atomic>
#include <stdexcept>
#include <type_traits>

#include "linear_dense.cuh"
#include "linear_rows.cuh"
#include "linear_vector.cuh"
#include "serving.h"
#include "serving_device.cuh"
#include "serving_tma.h"
#include "sm100_ptx.cuh"

namespace raiccl {

// Rows that TMA cannot read (a start or a stride off 16 bytes) are copied to
// aligned ones: one read and one write of what the product then reads.  Sixteen
// bytes at a time from the two aligned words around them, shifted together; the
// last word of a row, whose second neighbour may lie behind the tensor, by
// elements.  (One element at a time took 35 us for 1728 x 9097 bf16.)
// Groups of rows (experts) are a grid row each.
template <typename T>
__global__ void __launch_bounds__(256) linear_pack_kernel(const T* src, long long stride, long long group, T* dst, int packed,
                                                          long long rows, int K) {
  constexpr int V = 16 / sizeof(T);
  src += blockIdx.y * group;
  dst += blockIdx.y * rows * packed;
  griddep_wait();
  griddep_launch_dependents();
  const int per = (K + V - 1) / V;   // 16-byte words of a row
  const long long n = rows * per;
#pragma unroll 2
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long r = i / per;
    const int at = (int)(i - r * per) * V;
    const T* s = src + r * stride + at;
    T* d = dst + r * packed + at;
    if (at + 2 * V <= K) {
      const uint32_t off = (uint32_t)((uintptr_t)s & 15);
      const uint4* w = (const uint4*)((uintptr_t)s - off);
      const uint4 a = __ldg(w), b = off ? __ldg(w + 1) : a;
      uint32_t x0 = a.x, x1 = a.y, x2 = a.z, x3 = a.w, x4 = b.x;
      switch (off >> 2) {
        case 1: x0 = a.y; x1 = a.z; x2 = a.w; x3 = b.x; x4 = b.y; break;
        case 2: x0 = a.z; x1 = a.w; x2 = b.x; x3 = b.y; x4 = b.z; break;
        case 3: x0 = a.w; x1 = b.x; x2 = b.y; x3 = b.z; x4 = b.w; break;
        default: break;
      }
      const uint32_t bits = (off & 3) * 8;
      *(uint4*)d = make_uint4(__funnelshift_r(x0, x1, bits), __funnelshift_r(x1, x2, bits), __funnelshift_r(x2, x3, bits),
                              __funnelshift_r(x3, x4, bits));
    } else {
      for (int k = 0; k < V && at + k < K; ++k) d[k] = s[k];
    }
  }
}

constexpr int kRowsShared = 232448 - 2048;   // dynamic shared memory of a CTA, besides the kernel's own

static long long up256(long long v) { return (v + 255) / 256 * 256; }

// bf16 operands with an fp32 result: so much of K goes into one accumulator at least, in dense tiles up to twice as much.
constexpr int kLinearChain = 512;
static_assert(kLinearChain == LinearRows<false>::CHAIN * kRowsPack * LinearRows<false>::BK &&
              2 * kLinearChain == LinearDense<256, false>::CHAIN * LinearDense<256, false>::BK);

// Which kernel, by what each was measured to take on one B200 (us; sizes 32 to 2048 rows, 1024 to 5632 outputs, K 1024 to
// 4096; the sums below are within a seventh of most):
//   rows       3 + 4 Mp / (64 ranks) for each round of CTAs, and for each 128 bytes of its K 0.14 to 0.24 (fp32: 0.55 to
//              0.9); a quarter more where clusters share SMs
//   dense 128  3.2 + 0.9 for each round of pairs and 0.19 for each 128 bytes of K; fp32 7 + 0.5 and 0.44, and 1.6 for each
//              million numbers that are split
//   dense 256  4.2 + 1.8 and 0.29: fewer rounds, each longer
//   vector     very few rows, see below
// So 4096 x 4096 takes (rows, 128, 256) for 64 rows 11.9, 16.2, 24.1, for 384 rows 26.1, 17.5, 24.8, for 2048 rows 117, 60,
// 50; 1024 x 4096 fp32 for 64 rows 13.4, 27.2, for 384 rows 60, 31.
LinearPlan plan_linear(const LinearParams& p, int sms) {
  LinearPlan r{};
  const int eb = p.bf16 ? 2 : 4;
  const bool glu = p.act == (int)Act::kSwiGLU;
  const long long wrows = glu ? 2ll * p.N : p.N;
  auto aligned = [&](const void* base, long long rows, long long stride) {
    return ((uintptr_t)base & 15) == 0 && (rows <= 1 || ((stride * eb) % 16 == 0 && stride >= p.K));
  };
  r.packed_stride = (std::max(p.K, 1) + 7) / 8 * 8;
  r.pack_x = p.K > 0 && !aligned(p.x, p.M, p.x_stride);
  r.pack_w = p.K > 0 && !aligned(p.w, wrows, p.w_stride);
  const int KB = (p.K + 128 / eb - 1) / (128 / eb);   // 128-byte steps of K

  // rows: CTAs that share K
  r.Mp = (int)std::min<long long>(64, (p.M + 15) / 16 * 16);
  r.chained = p.bf16 && !p.out_bf16 && p.K > kLinearChain;
  if ((!p.bf16 || r.chained) && r.Mp == 48) r.Mp = 64;
  const long long mt = (p.M + r.Mp - 1) / r.Mp, tiles = (p.N + (glu ? 63 : 127)) / (glu ? 64 : 128) * mt;
  const int per = p.bf16 ? 2 : 1;   // CTAs per SM; fp32 holds a stage through splitting and product, so one with as many as fit
  double best = 0;
  for (int ranks = 1; ranks <= 8; ranks *= 2) {
    if (ranks > 1 && KB < 2 * ranks) break;
    const long long slots = (long long)per * sms * (ranks == 8 ? 81 : ranks == 4 ? 89 : 100) / 100;   // clusters leave SMs empty
    const long long rounds = (tiles * ranks + slots - 1) / slots;
    const double step = p.bf16 ? 0.14 + 0.1 * r.Mp / 64 : 0.55 + 0.35 * r.Mp / 64;
    const double shared = p.bf16 && ranks > 1 && tiles * ranks > sms ? 1.25 : 1.0;
    const double cost = rounds * (3.0 + 4.0 * r.Mp / 64 / ranks + (KB + ranks - 1) / ranks * step) * shared + 0.1 * ranks;
    if (r.ranks == 0 || cost < best) {
      best = cost;
      r.ranks = ranks;
    }
  }
  if (mt > 65535) best = 1e30;   // more tiles than a grid has rows
  // Rows of out or residual off 16 bytes: a thread of a dense tile has a row of its own and goes through it element by
  // element, 20 us for a tile of 128 columns (bf16, dense / rows, us: 269 x 64 x 10735 71 / 16, 4096 x 1024 x 4097 281 / 106).
  const int ob = p.out_bf16 ? 2 : 4, rb = p.res_bf16 ? 2 : 4;
  const bool odd = (((uintptr_t)p.out | (uintptr_t)(p.out_stride * ob)) & 15) != 0 ||
                   (p.residual != nullptr && (((uintptr_t)p.residual | (uintptr_t)(p.res_stride * rb)) & 15) != 0);
  // dense tiles
  if (p.K > 0 && p.M < (1ll << 30)) {
    for (int bn = 128; bn <= (p.bf16 ? 256 : 128); bn *= 2) {
      const int w = glu ? bn / 2 : bn;
      const long long t = (p.M + 255) / 256 * ((p.N + w - 1) / w), rounds = (t + sms / 2 - 1) / (sms / 2);
      const double cost = p.bf16 ? (bn == 256 ? 4.2 + rounds * std::max(1.8 + 0.29 * KB, odd ? 40.0 : 0.0)
                                               : 3.2 + rounds * std::max(0.9 + 0.19 * KB, odd ? 20.0 : 0.0))
                                 : 7 + rounds * std::max(0.5 + 0.44 * KB, odd ? 20.0 : 0.0) + (double)(p.M + wrows) * p.K * 1.6e-6;
      if (cost < best) {
        best = cost;
        r.dense = bn;
      }
    }
  }
  if (r.dense && p.K <= 2 * kLinearChain) r.chained = 0;
  // Very few rows: without pipelines, splits and copies.  Up to so many weights (millions), by where the two cross; us, here
  // against there: bf16 1 row 1024 x 1024 2.4 / 4.0, 4096 x 4096 9.1 / 9.7, 16384 x 4096 26.5 / 23.5, 4 rows 1024 x 1024
  // 3.1 / 4.1, 4096 x 1024 9.0 / 4.6; fp32 1 row 16384 x 4096 43 / 74, 4 rows 68 / 75, 8 rows 1024 x 1024 4.9 / 7.7; SwiGLU
  // holds twice the sums: 2 rows 2 x 4096 x 4096 fp32 45 / 42.  Off 16 bytes: bf16 4 rows 1728 x 9097 18 / 20, fp32 8 rows
  // 23 / 49.
  const bool packs = r.pack_x || r.pack_w;
  const double weights = 1e-6 * wrows * p.K, all = 1e30;
  double most = 0;
  if (packs && p.K > 0) most = p.M <= (p.bf16 ? 4 : 8) ? all : 0;
  else if (p.bf16) most = p.M == 1 ? (glu ? 2.5 : 17) : p.M == 2 ? 2.5 : p.M <= 4 ? 1.2 : p.M <= 8 ? 0.2 : 0;
  else most = p.M == 1 ? all : p.M == 2 ? (glu ? 9 : all) : p.M <= 4 ? (glu ? 2.5 : all) : p.M <= 8 ? 2.5 : 0;
  if (p.M <= 8 && weights <= most) {
    r.vector = 1;
    r.vec = !packs && (p.K * eb) % 16 == 0;
    r.dense = r.pack_x = r.pack_w = 0;
    return r;
  }
  if (p.K == 0) r.x_bytes = 256;   // an address for the maps; nothing is read
  if (r.dense && !p.bf16) {        // both operands as two tf32 parts
    r.x_bytes = up256(2ll * p.M * r.packed_stride * eb);
    r.w_bytes = up256(2ll * wrows * r.packed_stride * eb);
    return r;
  }
  if (r.pack_x) r.x_bytes = up256(p.M * r.packed_stride * eb);
  if (r.pack_w) r.w_bytes = up256(wrows * r.packed_stride * eb);
  const int sb = p.bf16 ? LinearRows<false>::stage_bytes(r.Mp) : LinearRows<true>::stage_bytes(r.Mp);
  r.low = p.bf16 ? 0 : 2;
  const int fit = std::min(kRowsMaxStages, (kRowsShared / per - (per - 1) * 2048 - 1024 - r.low * kRowsPack * kRowsTile) / sb);
  r.stages = std::max(2, std::min(fit, ((KB + r.ranks - 1) / r.ranks + kRowsPack - 1) / kRowsPack));
  return r;
}

template <bool FP32, bool GLU, int MP>
static void launch_rows(const LinearParams& p, const LinearPlan& plan, cudaStream_t s) {
  using C = LinearRows<FP32>;
  auto kern = linear_rows_kernel<FP32, GLU, MP>;
  static std::atomic<unsigned long long> configured;  // by device
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsShared) != cudaSuccess)
      throw std::runtime_error("linear: shared memory");
    configured.fetch_or(bit);
  }
  const cuuint64_t eb = FP32 ? 4 : 2, K = std::max(p.K, 1);
  const cuuint64_t wrows = GLU ? 2ull * p.N : p.N;
  CUtensorMap tx, tw;
  {
    const cuuint64_t dims[2] = {K, (cuuint64_t)p.M}, strides[1] = {p.M > 1 ? p.x_stride * eb : (K * eb + 15) / 16 * 16};
    const cuuint32_t box[2] = {C::BK, (cuuint32_t)plan.Mp};
    tx = make_tmap(p.x, !FP32, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  {
    const cuuint64_t dims[2] = {K, wrows}, strides[1] = {wrows > 1 ? p.w_stride * eb : (K * eb + 15) / 16 * 16};
    const cuuint32_t box[2] = {C::BK, GLU ? 64 : 128};
    tw = make_tmap(p.w, !FP32, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  LinearRowsParams rp{};
  rp.l = p;
  rp.Mp = plan.Mp;
  rp.stages = plan.stages;
  rp.low = plan.low;
  const int ob = p.out_bf16 ? 2 : 4;
  rp.vec_out = ((uintptr_t)p.out & (4 * ob - 1)) == 0 && p.out_stride % 4 == 0;
  cudaLaunchConfig_t cfg = {};
  const int W = GLU ? 64 : 128;
  cfg.gridDim = dim3((unsigned)((p.N + W - 1) / W * plan.ranks), (unsigned)((p.M + plan.Mp - 1) / plan.Mp));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = 1024 + (size_t)std::max(plan.stages * C::stage_bytes(plan.Mp) + plan.low * kRowsPack * kRowsTile, plan.Mp * 512);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = plan.ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kern, tx, tw, rp, serving_status());
}

template <int BN, bool FP32, bool GLU, bool CHAINED>
static void launch_dense(const LinearParams& p, cudaStream_t s) {
  using C = LinearDense<BN, FP32>;
  auto kern = linear_dense_kernel<BN, FP32, GLU, CHAINED>;
  static std::atomic<unsigned long long> configured;  // by device
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
      throw std::runtime_error("linear: shared memory");
    configured.fetch_or(bit);
  }
  const cuuint64_t eb = FP32 ? 4 : 2, K = p.K, parts = FP32 ? 2 : 1, wrows = GLU ? 2ull * p.N : p.N;
  auto map = [&](const void* base, cuuint64_t rows, cuuint64_t stride, cuuint32_t box_rows) {
    const cuuint64_t row = rows > 1 ? stride * eb : (K * eb + 15) / 16 * 16;
    const cuuint64_t dims[3] = {K, rows, parts}, strides[2] = {row, FP32 ? rows * stride * eb : row};
    const cuuint32_t box[3] = {C::BK, box_rows, 1};
    return make_tmap(base, !FP32, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  const CUtensorMap tx = map(p.x, p.M, p.x_stride, 128), tw = map(p.w, wrows, p.w_stride, C::HALF);
  LinearDenseParams dp{};
  dp.l = p;
  dp.mt = (int)((p.M + 255) / 256);
  const int W = GLU ? BN / 2 : BN;
  dp.nt = (p.N + W - 1) / W;
  const int ob = p.out_bf16 ? 2 : 4, rb = p.res_bf16 ? 2 : 4;
  dp.vec_out = ((uintptr_t)p.out & 15) == 0 && (p.out_stride * ob) % 16 == 0;
  dp.vec_res = ((uintptr_t)p.residual & 15) == 0 && (p.res_stride * rb) % 16 == 0;
  const long long tiles = (long long)dp.mt * dp.nt;
  const int pairs = (int)std::min<long long>(tiles, serving_sm_count() / 2);
  launch_with_pdl(kern, dim3(2 * pairs), dim3(kDenseThreads), C::SMEM, s, true, tx, tw, dp, serving_status());
}

// fp32 stages hold four tiles: at 256 columns three stages of 64 KB, at 128 four of 48 KB, which is what it takes
// (2048 x 4096 x 4096: 340 against 275 us).
static void launch_dense_any(const LinearParams& p, const LinearPlan& plan, cudaStream_t s) {
  auto run = [&](auto bn, auto fp32, auto chained) {
    constexpr int BN = decltype(bn)::value;
    constexpr bool FP32 = decltype(fp32)::value, CHAINED = decltype(chained)::value;
    if (p.act == (int)Act::kSwiGLU) launch_dense<BN, FP32, true, CHAINED>(p, s);
    else launch_dense<BN, FP32, false, CHAINED>(p, s);
  };
  auto bf16 = [&](auto bn) {
    if (plan.chained) run(bn, std::false_type{}, std::true_type{});
    else run(bn, std::false_type{}, std::false_type{});
  };
  if (!p.bf16) run(std::integral_constant<int, 128>{}, std::true_type{}, std::true_type{});
  else if (plan.dense == 256) bf16(std::integral_constant<int, 256>{});
  else bf16(std::integral_constant<int, 128>{});
}

template <typename T, bool VEC, bool GLU>
static void launch_vector(const LinearParams& p, cudaStream_t s) {
  auto run = [&](auto kern, int nt) {
    launch_with_pdl(kern, dim3((p.N + kVectorOut - 1) / kVectorOut, (unsigned)((p.M + nt - 1) / nt)), dim3(kVectorThreads), 0, s, true, p);
  };
  if (p.M == 1) run(linear_vector_kernel<T, VEC, GLU, 1>, 1);
  else if (p.M == 2) run(linear_vector_kernel<T, VEC, GLU, 2>, 2);
  else if (p.M <= 4) run(linear_vector_kernel<T, VEC, GLU, 4>, 4);
  else run(linear_vector_kernel<T, VEC, GLU, 8>, 8);
}

static void launch_vector_any(const LinearParams& p, bool vec, cudaStream_t s) {
  const bool glu = p.act == (int)Act::kSwiGLU;
  auto run = [&](auto type, auto v) {
    using T = decltype(type);
    if (glu) launch_vector<T, decltype(v)::value, true>(p, s);
    else launch_vector<T, decltype(v)::value, false>(p, s);
  };
  if (p.bf16) {
    if (vec) run(__nv_bfloat16{}, std::true_type{});
    else run(__nv_bfloat16{}, std::false_type{});
  } else {
    if (vec) run(float{}, std::true_type{});
    else run(float{}, std::false_type{});
  }
}

void launch_pack_rows(const void* src, long long stride, long long group, int groups, void* dst, int packed, long long rows, int K,
                      int bf16, cudaStream_t s) {
  const dim3 grid((unsigned)((8 * serving_sm_count() + groups - 1) / groups), groups);
  if (bf16)
    launch_with_pdl(linear_pack_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, true, (const __nv_bfloat16*)src, stride, group,
                    (__nv_bfloat16*)dst, packed, rows, K);
  else
    launch_with_pdl(linear_pack_kernel<float>, grid, dim3(256), 0, s, true, (const float*)src, stride, group, (float*)dst, packed,
                    rows, K);
}

void launch_linear(const LinearParams& params, const LinearPlan& plan, void* workspace, cudaStream_t s) {
  LinearParams p = params;
  const bool glu = p.act == (int)Act::kSwiGLU;
  char* ws = (char*)workspace;
  if (plan.vector) return launch_vector_any(p, plan.vec != 0, s);
  if (p.K == 0) {
    p.x = p.w = ws;
    p.x_stride = p.w_stride = 8;
  }
  if (plan.dense && !p.bf16) {
    const long long wrows = glu ? 2ll * p.N : p.N;
    auto operand = [&](const void* src, long long stride, void* dst, long long rows) {
      return SplitOperand{(const float*)src, stride, (float*)dst, rows,
                          p.K % 4 == 0 && ((uintptr_t)src & 15) == 0 && (rows <= 1 || stride % 4 == 0)};
    };
    launch_with_pdl(linear_split_kernel, dim3((unsigned)(8 * serving_sm_count())), dim3(256), 0, s, true,
                    operand(p.x, p.x_stride, ws, p.M), operand(p.w, p.w_stride, ws + plan.x_bytes, wrows), plan.packed_stride, p.K);
    p.x = ws;
    p.w = ws + plan.x_bytes;
    p.x_stride = p.w_stride = plan.packed_stride;
  }
  if (plan.pack_x && !(plan.dense && !p.bf16)) {
    launch_pack_rows(p.x, p.x_stride, 0, 1, ws, plan.packed_stride, p.M, p.K, p.bf16, s);
    p.x = ws;
    p.x_stride = plan.packed_stride;
  }
  if (plan.pack_w && !(plan.dense && !p.bf16)) {
    launch_pack_rows(p.w, p.w_stride, 0, 1, ws + plan.x_bytes, plan.packed_stride, glu ? 2ll * p.N : p.N, p.K, p.bf16, s);
    p.w = ws + plan.x_bytes;
    p.w_stride = plan.packed_stride;
  }
  if (plan.dense) return launch_dense_any(p, plan, s);
  auto rows = [&](auto fp32, auto mp) {
    if (glu) launch_rows<decltype(fp32)::value, true, decltype(mp)::value>(p, plan, s);
    else launch_rows<decltype(fp32)::value, false, decltype(mp)::value>(p, plan, s);
  };
  auto chained = [&](auto fp32) {
    if (plan.Mp == 16) rows(fp32, std::integral_constant<int, 16>{});
    else if (plan.Mp == 32) rows(fp32, std::integral_constant<int, 32>{});
    else rows(fp32, std::integral_constant<int, 64>{});
  };
  if (!p.bf16) chained(std::true_type{});
  else if (plan.chained) chained(std::false_type{});
  else rows(std::false_type{}, std::integral_constant<int, 0>{});
}

}  // namespace raiccl
