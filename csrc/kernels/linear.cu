// out = act(x w^T + bias) + residual: a dense product with its epilogue, from
// one row to a whole batch, any sizes.
#include <algorithm>
#include <atomic>
#include <stdexcept>

#include "linear_rows.cuh"
#include "serving.h"
#include "serving_device.cuh"
#include "serving_tma.h"
#include "sm100_ptx.cuh"

namespace raiccl {

// Rows that TMA cannot read (a start or a stride off 16 bytes) are copied to
// aligned ones: one read and one write of what the product then reads.
template <typename T>
__global__ void __launch_bounds__(256) linear_pack_kernel(const T* src, long long stride, T* dst, int packed, long long rows, int K) {
  griddep_wait();
  griddep_launch_dependents();
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* s = src + r * stride;
    T* d = dst + r * packed;
#pragma unroll 4
    for (int k = threadIdx.x; k < K; k += 256) d[k] = s[k];
  }
}

constexpr int kRowsShared = 232448 - 2048;   // dynamic shared memory of a CTA, besides the kernel's own

static long long up256(long long v) { return (v + 255) / 256 * 256; }

LinearPlan plan_linear(const LinearParams& p) {
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
  if (r.pack_x) r.x_bytes = up256(p.M * r.packed_stride * eb);
  if (r.pack_w) r.w_bytes = up256(wrows * r.packed_stride * eb);
  if (p.K == 0) r.x_bytes = 256;   // an address for the maps; nothing is read
  const int most = p.bf16 ? 256 : 128;
  r.Mp = (int)std::min<long long>(most, (p.M + 15) / 16 * 16);
  const long long mt = (p.M + r.Mp - 1) / r.Mp, tiles = (p.N + (glu ? 63 : 127)) / (glu ? 64 : 128) * mt;
  const int KB = (p.K + 128 / eb - 1) / (128 / eb), slots = 2 * serving_sm_count();
  r.ranks = 1;
  while (r.ranks < 8 && tiles * r.ranks * 2 <= slots && KB >= r.ranks * 2 * 4) r.ranks *= 2;
  const int sb = p.bf16 ? LinearRows<false>::stage_bytes(r.Mp) : LinearRows<true>::stage_bytes(r.Mp);
  const int low = p.bf16 ? 0 : LinearRows<true>::low_bytes();
  // two CTAs per SM where four stages fit in half of its shared memory
  const int half = kRowsShared / 2 - 2048;
  const int room = (half - 1024 - low) / sb >= 4 ? half : kRowsShared;
  r.stages = std::max(2, std::min({kRowsMaxStages, (room - 1024 - low) / sb, std::max(4, (KB + r.ranks - 1) / r.ranks)}));
  return r;
}

template <bool FP32, bool GLU>
static void launch_rows(const LinearParams& p, const LinearPlan& plan, cudaStream_t s) {
  using C = LinearRows<FP32>;
  auto kern = linear_rows_kernel<FP32, GLU>;
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
  cudaLaunchConfig_t cfg = {};
  const int W = GLU ? 64 : 128;
  cfg.gridDim = dim3((unsigned)((p.N + W - 1) / W * plan.ranks), (unsigned)((p.M + plan.Mp - 1) / plan.Mp));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = 1024 + (size_t)std::max(plan.stages * C::stage_bytes(plan.Mp) + C::low_bytes(), plan.Mp * 512);
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

static void pack(const void* src, long long stride, void* dst, int packed, long long rows, int K, int bf16, cudaStream_t s) {
  const dim3 grid((unsigned)std::min<long long>(rows, 8ll * serving_sm_count()));
  if (bf16)
    launch_with_pdl(linear_pack_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, true, (const __nv_bfloat16*)src, stride,
                    (__nv_bfloat16*)dst, packed, rows, K);
  else
    launch_with_pdl(linear_pack_kernel<float>, grid, dim3(256), 0, s, true, (const float*)src, stride, (float*)dst, packed, rows, K);
}

void launch_linear(const LinearParams& params, const LinearPlan& plan, void* workspace, cudaStream_t s) {
  LinearParams p = params;
  const bool glu = p.act == (int)Act::kSwiGLU;
  char* ws = (char*)workspace;
  if (p.K == 0) {
    p.x = p.w = ws;
    p.x_stride = p.w_stride = 8;
  }
  if (plan.pack_x) {
    pack(p.x, p.x_stride, ws, plan.packed_stride, p.M, p.K, p.bf16, s);
    p.x = ws;
    p.x_stride = plan.packed_stride;
  }
  if (plan.pack_w) {
    pack(p.w, p.w_stride, ws + plan.x_bytes, plan.packed_stride, glu ? 2ll * p.N : p.N, p.K, p.bf16, s);
    p.w = ws + plan.x_bytes;
    p.w_stride = plan.packed_stride;
  }
  if (p.bf16) {
    if (glu) launch_rows<false, true>(p, plan, s);
    else launch_rows<false, false>(p, plan, s);
  } else {
    if (glu) launch_rows<true, true>(p, plan, s);
    else launch_rows<true, false>(p, plan, s);
  }
}

}  // namespace raiccl
