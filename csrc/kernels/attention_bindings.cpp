// Torch bindings of the attention operators: argument checks, outputs,
// workspaces and launches.  A call only enqueues work on the current stream of
// its tensors' device; outputs and workspaces come from torch's allocator on
// that stream, so nothing is shared between calls or captured graphs.
#include <algorithm>
#include <cmath>
#include <tuple>
#include <utility>
#include <vector>

#include "attention.h"
#include "serving.h"
#include "serving_checks.h"

namespace {

using namespace raiccl;

bool aligned16(const torch::Tensor& t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }

// Rows of a tensor [n, heads, D] that start on 16 (or 32) bytes.
bool rows16(const torch::Tensor& t, int64_t bytes = 16) {
  const int64_t eb = t.element_size();
  return (uintptr_t)t.data_ptr() % bytes == 0 && (t.size(0) <= 1 || (t.stride(0) * eb) % bytes == 0) &&
         (t.size(1) <= 1 || (t.stride(1) * eb) % bytes == 0);
}

// A tensor to be written whose elements share no memory with each other: some order of its dimensions nests.
bool apart(const torch::Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> d;
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) == 0) return true;
    if (t.size(i) > 1) d.emplace_back(t.stride(i), t.size(i));
  }
  std::sort(d.begin(), d.end());
  int64_t reach = 1;
  for (auto& x : d) {
    if (x.first < reach) return false;
    reach += (x.second - 1) * x.first;
  }
  return true;
}

void check_head_dim(const char* op, int64_t D) {
  TORCH_CHECK_VALUE(D == 64 || D == 128, op, ": heads must have 64 or 128 dimensions, got ", text(D));
}

void check_one(const char* op, const char* name, const torch::Tensor& t, const torch::Device& dev) {
  check_input(op, name, t, dev);
  TORCH_CHECK_VALUE(t.dim() == 3 && inner_contiguous(t), op, ": ", name, " must be [tokens, heads, head_dim] with contiguous rows");
}

void check_index(const char* op, const char* name, const torch::Tensor& t, const torch::Device& dev, int64_t n) {
  check_input(op, name, t, dev);
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kInt32 && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), op, ": ", name,
                    " must be a contiguous int32 tensor of shape ", text({n}));
}

constexpr double kLog2e = 1.44269504088896340736;

double check_scale(const char* op, c10::optional<double> scale, int64_t D) {
  const double s = scale ? *scale : 1.0 / std::sqrt((double)D);
  TORCH_CHECK_VALUE(std::isfinite((float)(s * kLog2e)), op, ": scale must be a finite number, and by log2(e) in fp32 too");
  return s;
}

float check_unit(const char* op, const char* name, double unit) {
  int e;
  TORCH_CHECK_VALUE(std::isfinite(unit) && unit > 0 && std::frexp(unit, &e) == 0.5 && e > -64 && e <= 64, op, ": ", name,
                    " must be a power of two between 2^-64 and 2^63");
  return (float)unit;
}

struct Cache {
  const torch::Tensor &k_codes, &k_scales, &v_codes, &v_scales;
  double k_unit, v_unit;
};

CacheView check_cache(const char* op, const Cache& c, const torch::Device& dev) {
  TORCH_CHECK_VALUE(c.k_codes.dim() == 4, op, ": the cache's codes must be [pages, kv_heads, page_size, head_dim / 2]");
  const int64_t pages = c.k_codes.size(0), heads = c.k_codes.size(1), page = c.k_codes.size(2), D = 2 * c.k_codes.size(3);
  auto codes = [&](const char* name, const torch::Tensor& t) {
    check_input(op, name, t, dev);
    TORCH_CHECK_VALUE(t.scalar_type() == torch::kUInt8 && t.sizes() == c.k_codes.sizes() && t.is_contiguous() && aligned16(t), op, ": ",
                      name, " must be a contiguous uint8 tensor [pages, kv_heads, page_size, head_dim / 2] on 16 bytes");
  };
  auto scales = [&](const char* name, const torch::Tensor& t) {
    check_input(op, name, t, dev);
    TORCH_CHECK_VALUE(t.scalar_type() == torch::kFloat8_e4m3fn && t.sizes() == at::IntArrayRef({pages, heads, page, D / kCacheGroup}) &&
                          t.is_contiguous() && aligned16(t),
                      op, ": ", name, " must be a contiguous float8_e4m3fn tensor [pages, kv_heads, page_size, head_dim / 16] on 16 bytes");
  };
  check_head_dim(op, D);
  TORCH_CHECK_VALUE(page >= kCachePage && page <= 65536 && (page & (page - 1)) == 0, op, ": page_size must be a power of two from 16 to 65536, got ",
                    text(page));
  TORCH_CHECK_VALUE(heads >= 1 && heads <= 1024, op, ": 1 to 1024 kv_heads, got ", text(heads));
  TORCH_CHECK_VALUE(heads * page <= (1 << 24), op, ": kv_heads times page_size must be at most 2^24");
  TORCH_CHECK_VALUE(pages < (1ll << 31) / page, op, ": the cache must have less than 2^31 places");
  codes("k_codes", c.k_codes);
  codes("v_codes", c.v_codes);
  scales("k_scales", c.k_scales);
  scales("v_scales", c.v_scales);
  CacheView v{};
  v.k_codes = (uint8_t*)c.k_codes.data_ptr();
  v.k_scales = (uint8_t*)c.k_scales.data_ptr();
  v.v_codes = (uint8_t*)c.v_codes.data_ptr();
  v.v_scales = (uint8_t*)c.v_scales.data_ptr();
  v.pages = (int)pages;
  v.heads = (int)heads;
  v.D = (int)D;
  while ((1 << v.page_shift) < page) ++v.page_shift;
  v.k_unit = check_unit(op, "k_unit", c.k_unit);
  v.v_unit = check_unit(op, "v_unit", c.v_unit);
  return v;
}

void check_slots(const char* op, const torch::Tensor& slots, const torch::Device& dev) {
  check_input(op, "slots", slots, dev);
  TORCH_CHECK_VALUE((slots.scalar_type() == torch::kInt32 || slots.scalar_type() == torch::kInt64) && slots.dim() == 1 && slots.is_contiguous(),
                    op, ": slots must be a contiguous int32 or int64 tensor [tokens]");
  TORCH_CHECK_VALUE(slots.size(0) < (1ll << 31), op, ": less than 2^31 tokens in one call");
}

void check_apart(const char* op, const char* name, const torch::Tensor& out, std::initializer_list<const torch::Tensor*> inputs) {
  TORCH_CHECK_VALUE(apart(out), op, ": the elements of ", name, " share memory");
  for (const torch::Tensor* t : inputs)
    TORCH_CHECK_VALUE(!may_share_memory(out, *t), op, ": ", name, " shares memory with another tensor of the call, or lies between its elements by "
                      "other strides");
}

void kv_cache_write(torch::Tensor k_codes, torch::Tensor k_scales, torch::Tensor v_codes, torch::Tensor v_scales, double k_unit,
                    double v_unit, torch::Tensor k, torch::Tensor v, torch::Tensor slots) {
  const char* op = "kv_cache_write";
  const torch::Device dev = k.device();
  const CacheView c = check_cache(op, {k_codes, k_scales, v_codes, v_scales, k_unit, v_unit}, dev);
  check_one(op, "k", k, dev);
  check_one(op, "v", v, dev);
  check_slots(op, slots, dev);
  const int64_t N = slots.size(0);
  TORCH_CHECK_VALUE(k.sizes() == at::IntArrayRef({N, c.heads, c.D}) && v.sizes() == k.sizes(), op, ": k and v must be [",
                    "tokens, kv_heads, head_dim] = ", text({N, c.heads, c.D}), " by the slots and the cache");
  TORCH_CHECK_VALUE(is_float_type(k) && v.scalar_type() == k.scalar_type(), op, ": k and v must both be bf16 or both be fp32");
  const torch::Tensor* parts[4] = {&k_codes, &k_scales, &v_codes, &v_scales};
  for (int i = 0; i < 4; ++i) {
    check_apart(op, "the cache", *parts[i], {&k, &v, &slots});
    for (int j = 0; j < i; ++j) check_apart(op, "the cache", *parts[i], {parts[j]});
  }
  check_cuda(op, dev);
  if (N == 0) return;
  const c10::cuda::CUDAGuard guard(dev);
  CacheWriteParams p{};
  p.c = c;
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.k_token = k.stride(0);
  p.k_head = k.stride(1);
  p.v_token = v.stride(0);
  p.v_head = v.stride(1);
  p.slots = slots.data_ptr();
  p.slots64 = slots.scalar_type() == torch::kInt64;
  p.bf16 = k.scalar_type() == torch::kBFloat16;
  p.vec = rows16(k) && rows16(v);
  p.N = N;
  p.status = serving_status();
  launch_cache_write(p, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  for (const torch::Tensor* t : parts) written(*t);
}

std::tuple<torch::Tensor, torch::Tensor> kv_cache_read(torch::Tensor k_codes, torch::Tensor k_scales, torch::Tensor v_codes,
                                                       torch::Tensor v_scales, double k_unit, double v_unit, torch::Tensor slots,
                                                       c10::optional<torch::ScalarType> dtype, OptTensor k_out, OptTensor v_out) {
  const char* op = "kv_cache_read";
  const torch::Device dev = slots.device();
  const CacheView c = check_cache(op, {k_codes, k_scales, v_codes, v_scales, k_unit, v_unit}, dev);
  check_slots(op, slots, dev);
  const int64_t N = slots.size(0);
  TORCH_CHECK_VALUE(k_out.has_value() == v_out.has_value(), op, ": k_out and v_out are given together or not at all");
  const torch::ScalarType dt = dtype ? *dtype : k_out ? k_out->scalar_type() : torch::kBFloat16;
  TORCH_CHECK_VALUE(dt == torch::kBFloat16 || dt == torch::kFloat32, op, ": the result is bf16 or fp32");
  if (k_out) {
    for (const OptTensor* o : {&k_out, &v_out}) {
      const char* name = o == &k_out ? "k_out" : "v_out";
      check_one(op, name, **o, dev);
      TORCH_CHECK_VALUE((*o)->sizes() == at::IntArrayRef({N, c.heads, c.D}) && (*o)->scalar_type() == dt, op, ": ", name, " must have shape ",
                        text({N, c.heads, c.D}), " and the result's type");
      check_apart(op, name, **o, {&k_codes, &k_scales, &v_codes, &v_scales, &slots});
    }
    check_apart(op, "v_out", *v_out, {&*k_out});
  }
  check_cuda(op, dev);
  const c10::cuda::CUDAGuard guard(dev);
  torch::Tensor k = k_out ? *k_out : fresh({N, c.heads, c.D}, dt, dev), v = v_out ? *v_out : fresh({N, c.heads, c.D}, dt, dev);
  if (N == 0) return {k, v};
  CacheReadParams p{};
  p.c = c;
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.k_token = k.stride(0);
  p.k_head = k.stride(1);
  p.v_token = v.stride(0);
  p.v_head = v.stride(1);
  p.slots = slots.data_ptr();
  p.slots64 = slots.scalar_type() == torch::kInt64;
  p.bf16 = dt == torch::kBFloat16;
  p.vec = rows16(k, 32) && rows16(v, 32) ? 2 : rows16(k) && rows16(v) ? 1 : 0;
  p.N = N;
  p.status = serving_status();
  launch_cache_read(p, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  written(k_out);
  written(v_out);
  return {k, v};
}

// out [n, heads, D]: given, or allocated once the device is known to be one.
torch::Tensor attention_out(const char* op, const OptTensor& out, torch::ScalarType dt, const torch::Tensor& q,
                            std::initializer_list<const torch::Tensor*> inputs) {
  if (out) {
    check_one(op, "out", *out, q.device());
    TORCH_CHECK_VALUE(out->sizes() == q.sizes() && out->scalar_type() == dt, op, ": out must have q's shape, ", text(q.sizes()),
                      ", and the result's type");
    check_apart(op, "out", *out, inputs);
  }
  check_cuda(op, q.device());
  return out ? *out : fresh(q.sizes(), dt, q.device());
}

std::tuple<torch::Tensor, OptTensor> attention_cached(torch::Tensor q, torch::Tensor k_codes, torch::Tensor k_scales, torch::Tensor v_codes,
                                                      torch::Tensor v_scales, double k_unit, double v_unit, torch::Tensor block_table,
                                                      torch::Tensor lengths, c10::optional<double> scale, OptTensor out,
                                                      c10::optional<torch::ScalarType> out_dtype, bool return_lse) {
  const char* op = "attention_cached";
  const torch::Device dev = q.device();
  check_one(op, "q", q, dev);
  const CacheView c = check_cache(op, {k_codes, k_scales, v_codes, v_scales, k_unit, v_unit}, dev);
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2);
  TORCH_CHECK_VALUE(D == c.D, op, ": q has ", text(D), " dimensions to a head, the cache ", text(c.D));
  TORCH_CHECK_VALUE(Hq >= 1 && Hq % c.heads == 0 && Hq / c.heads <= 128, op, ": q must have 1 to 128 heads for each of the cache's ", text(c.heads),
                    ", got ", text(Hq));
  TORCH_CHECK_VALUE(B < (1 << 20), op, ": less than 2^20 sequences in one call");
  TORCH_CHECK_VALUE(is_float_type(q), op, ": q must be bf16 or fp32");
  check_index(op, "lengths", lengths, dev, B);
  check_input(op, "block_table", block_table, dev);
  TORCH_CHECK_VALUE(block_table.scalar_type() == torch::kInt32 && block_table.dim() == 2 && block_table.size(0) == B &&
                        inner_contiguous(block_table),
                    op, ": block_table must be an int32 tensor [sequences, pages] with contiguous rows");
  TORCH_CHECK_VALUE(block_table.size(1) < (1ll << 31 >> c.page_shift), op, ": block_table has room for 2^31 tokens of a sequence or more");
  const torch::ScalarType dt = out_dtype ? *out_dtype : out ? out->scalar_type() : q.scalar_type();
  TORCH_CHECK_VALUE(dt == torch::kFloat32 || (dt == torch::kBFloat16 && q.scalar_type() == torch::kBFloat16), op,
                    ": the output is fp32, or bf16 where q is bf16");
  CachedParams p{};
  p.mult = (float)std::frexp(check_scale(op, scale, D) * kLog2e * c.k_unit, &p.mult_exp);
  p.c = c;
  p.group = (int)(Hq / c.heads);
  p.bf16 = q.scalar_type() == torch::kBFloat16;
  p.out_bf16 = dt == torch::kBFloat16;
  // tiles that the table has room for, as the kernels count them: in 32 bits within a sequence, and a CTA's share
  const int64_t tiles = ((block_table.size(1) << c.page_shift) + kCachedTile - 1) / kCachedTile * c.heads * plan_cached(p, 1).chunks;
  TORCH_CHECK_VALUE(tiles < (1ll << 32), op, ": block_table has room for ", text(tiles), " tiles of 64 tokens of a sequence and a chunk of heads, "
                    "2^32 or more");
  TORCH_CHECK_VALUE(B * tiles < (1ll << 37), op, ": block_table has room for ", text(B * tiles), " tiles of 64 tokens of a sequence and a chunk of "
                    "heads in all, 2^37 or more");
  torch::Tensor res = attention_out(op, out, dt, q, {&q, &k_codes, &k_scales, &v_codes, &v_scales, &block_table, &lengths});
  const c10::cuda::CUDAGuard guard(dev);
  OptTensor lse;
  if (return_lse) lse = fresh({B, Hq}, torch::kFloat32, dev);
  if (B == 0) return {res, lse};
  p.q = q.data_ptr();
  p.q_seq = q.stride(0);
  p.q_head = q.stride(1);
  p.out = res.data_ptr();
  p.o_seq = res.stride(0);
  p.o_head = res.stride(1);
  p.lse = lse ? lse->data_ptr<float>() : nullptr;
  p.table = block_table.numel() ? block_table.data_ptr<int>() : nullptr;
  p.table_stride = block_table.stride(0);
  p.table_pages = (int)block_table.size(1);
  p.lengths = lengths.data_ptr<int>();
  p.B = (int)B;
  p.Hq = (int)Hq;
  p.q_vec = rows16(q);
  p.o_vec = rows16(res);
  p.status = serving_status();
  const CachedPlan plan = plan_cached(p, serving_sm_count());
  const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)plan.bytes());   // of the current stream
  launch_cached(p, plan, ws.get(), at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  written(out);
  return {res, lse};
}

// What the plan of a call goes by: shapes, types, addresses and strides.
void prompt_tensors(PromptParams& p, const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v) {
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.q_token = q.stride(0);
  p.q_head = q.stride(1);
  p.k_token = k.stride(0);
  p.k_head = k.stride(1);
  p.v_token = v.stride(0);
  p.v_head = v.stride(1);
  p.Nq = q.size(0);
  p.Nk = k.size(0);
  p.Hq = (int)q.size(1);
  p.Hk = (int)k.size(1);
  p.group = p.Hq / p.Hk;
  p.D = (int)q.size(2);
  p.bf16 = q.scalar_type() == torch::kBFloat16;
}

// How a call runs on a device of `sms` SMs: for tests.  Launches nothing; the tensors may lie on any device.
py::dict attention_prompt_plan(torch::Tensor q, torch::Tensor k, torch::Tensor v, int64_t seqs, int64_t sms) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.dim() == 3 && k.size(1) >= 1 && q.size(1) >= k.size(1) && q.size(1) / k.size(1) <= 128,
                    "attention_prompt_plan: tensors [tokens, heads, head_dim], 1 to 128 heads of q for each of k's");
  PromptParams p{};
  prompt_tensors(p, q, k, v);
  p.B = (int)seqs;
  const PromptPlan plan = plan_prompt(p, (int)sms);
  py::dict d;
  d["splits"] = plan.splits;
  d["pack_q"] = plan.pack_q != 0;
  d["pack_k"] = plan.pack_k != 0;
  d["pack_v"] = plan.pack_v != 0;
  d["bytes"] = plan.bytes();
  return d;
}

std::tuple<torch::Tensor, OptTensor> attention_prompt(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor cu_seqlens_q,
                                                      torch::Tensor cu_seqlens_k, bool causal, c10::optional<double> scale, OptTensor out,
                                                      bool return_lse) {
  const char* op = "attention_prompt";
  const torch::Device dev = q.device();
  check_one(op, "q", q, dev);
  check_one(op, "k", k, dev);
  check_one(op, "v", v, dev);
  const int64_t Nq = q.size(0), Hq = q.size(1), D = q.size(2), Nk = k.size(0), Hk = k.size(1);
  check_head_dim(op, D);
  TORCH_CHECK_VALUE(k.size(2) == D && v.sizes() == k.sizes(), op, ": k and v must be [tokens, kv_heads, ", text(D), "], alike");
  TORCH_CHECK_VALUE(Hk >= 1 && Hk <= 1024 && Hq >= 1 && Hq % Hk == 0 && Hq / Hk <= 128 && Hq < 65536, op,
                    ": q must have 1 to 128 heads for each of k's (1 to 1024; less than 65536 in all), got ", text(Hq), " and ", text(Hk));
  TORCH_CHECK_VALUE(is_float_type(q) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), op,
                    ": q, k and v must all be bf16 or all be fp32");
  TORCH_CHECK_VALUE(Nq < (1ll << 30) && Nk < (1ll << 30), op, ": less than 2^30 tokens");
  TORCH_CHECK_VALUE(cu_seqlens_q.dim() == 1 && cu_seqlens_q.size(0) >= 1, op, ": cu_seqlens_q must have one entry more than there are sequences");
  const int64_t B = cu_seqlens_q.size(0) - 1;
  TORCH_CHECK_VALUE(B <= (1 << 16), op, ": at most 2^16 sequences in one call");
  check_index(op, "cu_seqlens_q", cu_seqlens_q, dev, B + 1);
  check_index(op, "cu_seqlens_k", cu_seqlens_k, dev, B + 1);
  PromptParams p{};
  p.scale = (float)check_scale(op, scale, D);
  torch::Tensor res = attention_out(op, out, q.scalar_type(), q, {&q, &k, &v, &cu_seqlens_q, &cu_seqlens_k});
  const c10::cuda::CUDAGuard guard(dev);
  OptTensor lse;
  if (return_lse) lse = fresh({Nq, Hq}, torch::kFloat32, dev);
  if (Nq == 0 || B == 0) return {res, lse};
  prompt_tensors(p, q, k, v);
  p.out = res.data_ptr();
  p.o_token = res.stride(0);
  p.o_head = res.stride(1);
  p.lse = lse ? lse->data_ptr<float>() : nullptr;
  p.cu_q = cu_seqlens_q.data_ptr<int>();
  p.cu_k = cu_seqlens_k.data_ptr<int>();
  p.B = (int)B;
  p.causal = causal;
  p.o_vec = rows16(res);
  p.status = serving_status();
  const PromptPlan plan = plan_prompt(p, serving_sm_count());
  c10::DataPtr ws;   // of the current stream
  if (plan.bytes() > 0) ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)plan.bytes());
  launch_prompt(p, plan, ws.get(), at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  written(out);
  return {res, lse};
}

}  // namespace

void register_attention(py::module_& m) {
  m.def("kv_cache_write", &kv_cache_write);
  m.def("kv_cache_read", &kv_cache_read);
  m.def("attention_cached", &attention_cached);
  m.def("attention_prompt", &attention_prompt);
  m.def("attention_prompt_plan", &attention_prompt_plan);
}
