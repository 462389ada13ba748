// Torch bindings of the serving operators: argument checks, outputs,
// workspaces and launches.  A call only enqueues work on the current stream of
// its tensors' device; outputs and workspaces come from torch's allocator on
// that stream, so nothing is shared between calls or captured graphs.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "serving.h"

namespace {

using OptTensor = c10::optional<torch::Tensor>;

// Numbers and shapes as text.  Messages are put together from texts alone:
// streaming a number through the C++ library that this process has loaded ends it.
std::string text(int64_t v) { return std::to_string(v); }

std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}

bool inner_contiguous(const torch::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

bool is_float_type(const torch::Tensor& t) {
  return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16;
}

// A new tensor without the dispatcher's rounds, which cost the smallest calls as
// much as a launch.
torch::Tensor fresh(at::IntArrayRef shape, torch::ScalarType dt, const torch::Device& dev) {
  return at::detail::empty_cuda(shape, dt, dev, c10::nullopt);
}

// [first, last) bytes that the tensor's elements lie in.
std::pair<const char*, const char*> extent(const torch::Tensor& t) {
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) == 0) return {nullptr, nullptr};
    last += (t.size(d) - 1) * t.stride(d);
  }
  const char* p = (const char*)t.data_ptr();
  return {p, p + (last + 1) * t.element_size()};
}

bool overlap(const torch::Tensor& a, const torch::Tensor& b) {
  const auto x = extent(a), y = extent(b);
  return x.first < y.second && y.first < x.second;
}

// Behind a shape there may be no numbers to read: a sparse layout, a lazy zero or
// negation, a storage that was freed (sharded parameters between their uses), or
// a wrapper of other tensors (distributed, quantised or fake ones).
void check_memory(const char* op, const char* name, const torch::Tensor& t) {
  TORCH_CHECK_VALUE(t.layout() == c10::kStrided && !t.is_neg() && !t._is_zerotensor(), op, ": ", name,
                    " must be a dense tensor, without a pending negation or zero");
  if (t.numel() == 0 || !t.has_storage()) return;   // without one, data_ptr raises
  int64_t last = t.storage_offset();
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  TORCH_CHECK_VALUE((int64_t)t.storage().nbytes() >= (last + 1) * (int64_t)t.element_size(), op, ": ", name,
                    " reaches behind its storage, which holds ", text((int64_t)t.storage().nbytes()), " bytes");
  TORCH_CHECK_VALUE(t.is_meta() || t.data_ptr() != nullptr, op, ": ", name, " has no memory of its own (a wrapper of other tensors?)");
}

// Every tensor of a call lies on the CUDA device of x; checked behind the
// shapes, types and strides, whose refusals need no device.
void check_input(const char* op, const char* name, const torch::Tensor& t, const torch::Device& dev) {
  TORCH_CHECK_VALUE(t.device() == dev, op, ": ", name, " must be on ", dev.str(), ", not on ", t.device().str());
  TORCH_CHECK(!(t.requires_grad() && c10::GradMode::is_enabled()), op, ": ", name,
              " requires a gradient, but the operator has no backward; call it under torch.no_grad()");
  TORCH_CHECK(!(t._fw_grad(/*level=*/0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode()), op, ": ", name,
              " carries a forward-mode tangent, but the operator has no derivative; take the primal of it");
  check_memory(op, name, t);
}

void check_cuda(const char* op, const torch::Device& dev) {
  TORCH_CHECK_VALUE(dev.is_cuda(), op, ": the tensors must be on a CUDA device, not on ", dev.str());
}

void check_vector(const char* op, const char* name, const torch::Tensor& t, const torch::Device& dev, at::IntArrayRef shape) {
  check_input(op, name, t, dev);
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kFloat32 && t.sizes() == shape && t.is_contiguous(), op, ": ", name,
                    " must be a contiguous fp32 tensor of shape ", text(shape));
}

// out and residual of [rows, width]; out is allocated where none is given.
torch::Tensor check_out(const char* op, const OptTensor& out, const OptTensor& residual, const torch::Tensor& like,
                        c10::optional<torch::ScalarType> out_dtype, int64_t rows, int64_t width,
                        std::initializer_list<const torch::Tensor*> inputs, std::initializer_list<const OptTensor*> more) {
  const torch::Device dev = like.device();
  torch::ScalarType dt = out_dtype ? *out_dtype : out ? out->scalar_type() : like.scalar_type();
  TORCH_CHECK_VALUE(dt == torch::kFloat32 || (dt == torch::kBFloat16 && like.scalar_type() == torch::kBFloat16), op,
                    ": the output is fp32, or bf16 where the inputs are bf16");
  if (residual) {
    check_input(op, "residual", *residual, dev);
    TORCH_CHECK_VALUE(residual->dim() == 2 && residual->size(0) == rows && residual->size(1) == width, op,
                      ": residual must have the shape of the output, ", text({rows, width}));
    TORCH_CHECK_VALUE(is_float_type(*residual) && inner_contiguous(*residual), op,
                      ": residual must be fp32 or bf16 with contiguous rows");
  }
  if (!out) {
    check_cuda(op, dev);
    return fresh({rows, width}, dt, dev);
  }
  check_input(op, "out", *out, dev);
  TORCH_CHECK_VALUE(out->dim() == 2 && out->size(0) == rows && out->size(1) == width, op, ": out must have shape ",
                    text({rows, width}));
  TORCH_CHECK_VALUE(out->scalar_type() == dt, op, ": out has another type than out_dtype");
  TORCH_CHECK_VALUE(inner_contiguous(*out) && (rows <= 1 || out->stride(0) >= width), op,
                    ": out must have contiguous rows that do not overlap");
  for (const torch::Tensor* t : inputs)
    TORCH_CHECK_VALUE(!overlap(*out, *t), op, ": out shares memory with an input");
  for (const OptTensor* t : more)
    TORCH_CHECK_VALUE(!*t || !overlap(*out, **t), op, ": out shares memory with an input");
  if (residual && overlap(*out, *residual))  // in place: each element is read and written by one thread
    TORCH_CHECK_VALUE(out->data_ptr() == residual->data_ptr() && out->scalar_type() == residual->scalar_type() &&
                          (rows <= 1 || out->stride(0) == residual->stride(0)),
                      op, ": out shares memory with residual without being the same tensor");
  check_cuda(op, dev);
  return *out;
}

// What the plan of a call goes by: shapes, types, addresses and strides.
raiccl::FewExpertParams few_expert_params(const torch::Tensor& x, const torch::Tensor& w1, const torch::Tensor& w2, int64_t top_k,
                                          int64_t act) {
  raiccl::FewExpertParams e{};
  e.x = x.data_ptr();
  e.x_stride = x.stride(0);
  e.w1 = w1.data_ptr();
  e.w1_estride = w1.stride(0);
  e.w1_stride = w1.stride(1);
  e.w2 = w2.data_ptr();
  e.w2_estride = w2.stride(0);
  e.w2_stride = w2.stride(1);
  e.T = (int)x.size(0);
  e.D = (int)x.size(1);
  e.E = (int)w1.size(0);
  e.k = (int)top_k;
  e.F = (int)w2.size(2);
  e.O = (int)w2.size(1);
  e.act = (int)act;
  e.bf16 = x.scalar_type() == torch::kBFloat16;
  return e;
}

raiccl::LinearParams linear_params(const torch::Tensor& x, const torch::Tensor& weight, int64_t act, const OptTensor& residual,
                                   void* out, int64_t out_stride, torch::ScalarType out_type) {
  raiccl::LinearParams p{};
  p.x = x.data_ptr();
  p.x_stride = x.stride(0);
  p.w = weight.data_ptr();
  p.w_stride = weight.stride(0);
  p.residual = residual ? residual->data_ptr() : nullptr;
  p.res_stride = residual ? residual->stride(0) : 0;
  p.out = out;
  p.out_stride = out_stride;
  p.M = x.size(0);
  p.N = (int)(act == (int64_t)raiccl::Act::kSwiGLU ? weight.size(0) / 2 : weight.size(0));
  p.K = (int)x.size(1);
  p.act = (int)act;
  p.bf16 = x.scalar_type() == torch::kBFloat16;
  p.out_bf16 = out_type == torch::kBFloat16;
  p.res_bf16 = residual && residual->scalar_type() == torch::kBFloat16;
  return p;
}

// A given out was written: an operation that saved it for its backward pass has to notice.
void written(const OptTensor& out) {
  if (out && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> moe_few_tokens(
    torch::Tensor x, torch::Tensor router_w, torch::Tensor w1, torch::Tensor w2, int64_t top_k, int64_t act,
    int64_t gate_mode, OptTensor router_b, OptTensor b1, OptTensor b2, OptTensor block_mask, OptTensor residual,
    OptTensor out, c10::optional<torch::ScalarType> out_dtype) {
  const char* op = "moe_few_tokens";
  const torch::Device dev = x.device();
  TORCH_CHECK_VALUE(x.dim() == 2 && router_w.dim() == 2 && w1.dim() == 3 && w2.dim() == 3, op,
                    ": x is [T, D], router_w [E, D], w1 [E, N1, D], w2 [E, O, F]");
  check_input(op, "x", x, dev);
  check_input(op, "router_w", router_w, dev);
  check_input(op, "w1", w1, dev);
  check_input(op, "w2", w2, dev);
  const int64_t T = x.size(0), D = x.size(1), E = router_w.size(0), O = w2.size(1), F = w2.size(2);
  const bool glu = act == (int64_t)raiccl::Act::kSwiGLU;
  TORCH_CHECK_VALUE(T <= raiccl::kFewTokens, op, ": at most ", text(raiccl::kFewTokens), " tokens in one call, got ", text(T));
  TORCH_CHECK_VALUE(E >= 1 && E <= raiccl::kFewExperts, op, ": 1 to ", text(raiccl::kFewExperts), " experts, got ", text(E));
  TORCH_CHECK_VALUE(top_k >= 1 && top_k <= std::min<int64_t>(raiccl::kFewTopK, E), op, ": top_k must be in 1..min(8, experts)");
  TORCH_CHECK_VALUE(D >= 1 && F >= 1 && O >= 1 && D < (1 << 24) && F < (1 << 24) && O < (1 << 24), op,
                    ": widths must be in 1..2^24");
  TORCH_CHECK_VALUE(router_w.size(1) == D && w1.size(0) == E && w1.size(1) == (glu ? 2 * F : F) && w1.size(2) == D &&
                        w2.size(0) == E,
                    op, ": shapes differ: x [T, D], router_w [E, D], w1 [E, ", glu ? "2F" : "F", ", D], w2 [E, O, F]");
  const bool bf16 = x.scalar_type() == torch::kBFloat16;
  TORCH_CHECK_VALUE(is_float_type(x) && router_w.scalar_type() == x.scalar_type() && w1.scalar_type() == x.scalar_type() &&
                        w2.scalar_type() == x.scalar_type(),
                    op, ": x, router_w, w1 and w2 must all be bf16 or all be fp32");
  TORCH_CHECK_VALUE(inner_contiguous(x) && inner_contiguous(router_w) && inner_contiguous(w1) && inner_contiguous(w2), op,
                    ": x, router_w, w1 and w2 must have contiguous rows");
  TORCH_CHECK_VALUE(gate_mode >= 0 && gate_mode <= 2, op, ": unknown gate mode");
  if (router_b) check_vector(op, "router_b", *router_b, dev, {E});
  if (b1) check_vector(op, "b1", *b1, dev, {E, w1.size(1)});
  if (b2) check_vector(op, "b2", *b2, dev, {E, O});
  if (block_mask) {
    check_input(op, "block_mask", *block_mask, dev);
    TORCH_CHECK_VALUE((block_mask->scalar_type() == torch::kBool || block_mask->scalar_type() == torch::kUInt8) &&
                          ((block_mask->dim() == 1 && block_mask->size(0) == E) ||
                           (block_mask->dim() == 2 && block_mask->size(0) == T && block_mask->size(1) == E)) &&
                          inner_contiguous(*block_mask),
                      op, ": block_mask must be bool or uint8 of shape [E] or [T, E] with contiguous rows");
  }
  torch::Tensor res = check_out(op, out, residual, x, out_dtype, T, O, {&x, &router_w, &w1, &w2}, {&router_b, &b1, &b2, &block_mask});
  const c10::cuda::CUDAGuard guard(dev);
  torch::Tensor ids = fresh({T, top_k}, torch::kInt32, dev);
  torch::Tensor gates = fresh({T, top_k}, torch::kFloat32, dev);
  if (T == 0) return {res, ids, gates};
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();

  raiccl::FewRouteParams r{};
  const int64_t eb = x.element_size();
  auto rows16 = [&](const torch::Tensor& t) {
    return ((uintptr_t)t.data_ptr() & 15) == 0 && (t.size(0) <= 1 || (t.stride(0) * eb) % 16 == 0);
  };
  r.x = x.data_ptr();
  r.x_stride = x.stride(0);
  r.w = router_w.data_ptr();
  r.w_stride = router_w.stride(0);
  r.bias = router_b ? router_b->data_ptr<float>() : nullptr;
  r.mask = block_mask ? (const uint8_t*)block_mask->data_ptr() : nullptr;
  r.mask_stride = block_mask && block_mask->dim() == 2 ? block_mask->stride(0) : 0;
  r.T = (int)T;
  r.D = (int)D;
  r.E = (int)E;
  r.k = (int)top_k;
  r.gate_mode = (int)gate_mode;
  r.bf16 = bf16;
  r.vec = (D * eb) % 16 == 0 && rows16(x) && rows16(router_w);
  r.ids = ids.data_ptr<int>();
  r.gates = gates.data_ptr<float>();
  raiccl::FewExpertParams e = few_expert_params(x, w1, w2, top_k, act);
  e.b1 = b1 ? b1->data_ptr<float>() : nullptr;
  e.b2 = b2 ? b2->data_ptr<float>() : nullptr;
  e.residual = residual ? residual->data_ptr() : nullptr;
  e.res_stride = residual ? residual->stride(0) : 0;
  e.out = res.data_ptr();
  e.out_stride = res.stride(0);
  e.ids = r.ids;
  e.gates = r.gates;
  e.out_bf16 = res.scalar_type() == torch::kBFloat16;
  e.res_bf16 = residual && residual->scalar_type() == torch::kBFloat16;
  const raiccl::FewExpertPlan plan = raiccl::plan_few_experts(e, raiccl::serving_sm_count());
  const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)plan.bytes());   // of the current stream
  char* base = (char*)ws.get();
  r.packed = plan.pack ? base : nullptr;
  r.packed_stride = plan.packed_stride;
  r.packed_rows = plan.Tp;
  raiccl::launch_few(r, e, plan, base, stream);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  written(out);
  return {res, ids, gates};
}

torch::Tensor linear(torch::Tensor x, torch::Tensor weight, OptTensor bias, int64_t act, OptTensor residual, OptTensor out,
                     c10::optional<torch::ScalarType> out_dtype) {
  const char* op = "linear";
  const torch::Device dev = x.device();
  TORCH_CHECK_VALUE(x.dim() == 2 && weight.dim() == 2, op, ": x is [M, K], weight [N, K]");
  check_input(op, "x", x, dev);
  check_input(op, "weight", weight, dev);
  const int64_t M = x.size(0), K = x.size(1), rows = weight.size(0);
  const bool glu = act == (int64_t)raiccl::Act::kSwiGLU;
  TORCH_CHECK_VALUE(weight.size(1) == K, op, ": weight has ", text(weight.size(1)), " columns, x has ", text(K));
  TORCH_CHECK_VALUE(!glu || rows % 2 == 0, op, ": SwiGLU needs as many up rows as gate rows in weight");
  TORCH_CHECK_VALUE(M < (1ll << 30) && rows < (1 << 24) && K < (1 << 24), op, ": at most 2^30 rows and 2^24 columns");
  TORCH_CHECK_VALUE(K > 0 || M <= (1 << 21), op, ": at most 2^21 rows without columns");
  TORCH_CHECK_VALUE(is_float_type(x) && weight.scalar_type() == x.scalar_type(), op, ": x and weight must both be bf16 or both be fp32");
  TORCH_CHECK_VALUE(inner_contiguous(x) && inner_contiguous(weight), op, ": x and weight must have contiguous rows");
  const int64_t N = glu ? rows / 2 : rows;
  if (bias) check_vector(op, "bias", *bias, dev, {rows});
  torch::Tensor res = check_out(op, out, residual, x, out_dtype, M, N, {&x, &weight}, {&bias});
  c10::cuda::CUDAGuard guard(dev);
  if (M == 0 || N == 0) return res;
  raiccl::LinearParams p = linear_params(x, weight, act, residual, res.data_ptr(), res.stride(0), res.scalar_type());
  p.bias = bias ? bias->data_ptr<float>() : nullptr;
  const raiccl::LinearPlan plan = raiccl::plan_linear(p, raiccl::serving_sm_count());
  c10::DataPtr ws;   // of the current stream
  if (plan.bytes() > 0) ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)plan.bytes());
  raiccl::launch_linear(p, plan, ws.get(), at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  written(out);
  return res;
}

// Which kernels a call takes on a device of `sms` SMs: for tests, which name the path that they are about.  Launches
// nothing; the tensors may lie on any device.
py::dict moe_few_plan(torch::Tensor x, torch::Tensor w1, torch::Tensor w2, int64_t top_k, int64_t act, int64_t sms) {
  const raiccl::FewExpertPlan plan = raiccl::plan_few_experts(few_expert_params(x, w1, w2, top_k, act), (int)sms);
  py::dict d;
  d["path"] = plan.tensor ? "tensor" : "rows";
  d["vec"] = plan.vec != 0;
  d["routes"] = plan.route != 0;
  d["pack_x"] = plan.pack != 0;
  d["pack_w"] = plan.pack_w != 0;
  d["slice"] = plan.slice;
  d["bytes"] = plan.bytes();
  return d;
}

py::dict linear_plan(torch::Tensor x, torch::Tensor weight, int64_t act, OptTensor residual, OptTensor out, bool out_bf16,
                     int64_t sms) {
  raiccl::LinearParams p = linear_params(x, weight, act, residual, out ? out->data_ptr() : nullptr, out ? out->stride(0) : 0,
                                         out_bf16 ? torch::kBFloat16 : torch::kFloat32);
  if (!out) p.out_stride = p.N;
  const raiccl::LinearPlan plan = raiccl::plan_linear(p, (int)sms);
  py::dict d;
  d["kernel"] = plan.vector ? "vector" : plan.dense ? "dense" : "rows";
  d["tile"] = plan.dense;
  d["chained"] = !plan.vector && plan.chained;
  d["ranks"] = plan.vector || plan.dense ? 0 : plan.ranks;
  d["pack_x"] = plan.pack_x != 0;
  d["pack_w"] = plan.pack_w != 0;
  d["bytes"] = plan.bytes();
  return d;
}

// Where the device's record lies.
int64_t serving_status_address(int64_t device) {
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  return (int64_t)raiccl::serving_status();
}

// Stages and phases of the last fills of a ring of `stages`, newest first, after `filled` fills: what a loading thread waits for.
std::vector<std::pair<int, int>> serving_last_fills(int64_t stages, int64_t filled) {
  int stage = (int)(filled % stages);
  uint32_t phase = (uint32_t)(filled / stages & 1);
  std::vector<std::pair<int, int>> v;
  for (int64_t i = std::min(stages, filled); i > 0; --i) {
    raiccl::fill_before((int)stages, stage, phase);
    v.emplace_back(stage, (int)phase);
  }
  return v;
}

// The device's record of the first wait that ran out in a serving operator
// since the last call (eight words, DeviceStatus); waits for the device and
// clears the record.
torch::Tensor serving_status(int64_t device) {
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  torch::Tensor words = torch::zeros({(int64_t)(sizeof(raiccl::DeviceStatus) / 4)}, torch::kInt32);
  raiccl::DeviceStatus* at = raiccl::serving_status();
  C10_CUDA_CHECK(cudaDeviceSynchronize());
  C10_CUDA_CHECK(cudaMemcpy(words.data_ptr(), at, sizeof(raiccl::DeviceStatus), cudaMemcpyDeviceToHost));
  C10_CUDA_CHECK(cudaMemset(at, 0, sizeof(raiccl::DeviceStatus)));
  C10_CUDA_CHECK(cudaDeviceSynchronize());
  return words;
}

}  // namespace

void register_serving(py::module_& m) {
  m.def("moe_few_tokens", &moe_few_tokens, py::arg("x"), py::arg("router_w"), py::arg("w1"), py::arg("w2"), py::arg("top_k"),
        py::arg("act"), py::arg("gate_mode"), py::arg("router_b"), py::arg("b1"), py::arg("b2"), py::arg("block_mask"),
        py::arg("residual"), py::arg("out"), py::arg("out_dtype"));
  m.def("moe_few_plan", &moe_few_plan, py::arg("x"), py::arg("w1"), py::arg("w2"), py::arg("top_k"), py::arg("act"), py::arg("sms"));
  m.def("linear_plan", &linear_plan, py::arg("x"), py::arg("weight"), py::arg("act"), py::arg("residual"), py::arg("out"),
        py::arg("out_bf16"), py::arg("sms"));
  m.def("serving_status_address", &serving_status_address, py::arg("device"));
  m.def("serving_last_fills", &serving_last_fills, py::arg("stages"), py::arg("filled"));
  m.def("serving_status", &serving_status, py::arg("device"));
  m.def("linear", &linear, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("act"), py::arg("residual"),
        py::arg("out"), py::arg("out_dtype"));
}
