// Checks of tensors that the torch bindings of the serving operators share.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

namespace raiccl {

using OptTensor = c10::optional<torch::Tensor>;

// Numbers and shapes as text.  Messages are put together from texts alone:
// streaming a number through the C++ library that this process has loaded ends it.
inline std::string text(int64_t v) { return std::to_string(v); }

inline std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}

inline bool inner_contiguous(const torch::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

inline bool is_float_type(const torch::Tensor& t) {
  return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16;
}

// A new tensor without the dispatcher's rounds, which cost the smallest calls as
// much as a launch.
inline torch::Tensor fresh(at::IntArrayRef shape, torch::ScalarType dt, const torch::Device& dev) {
  return at::detail::empty_cuda(shape, dt, dev, c10::nullopt);
}

// [first, last) bytes that the tensor's elements lie in.
inline std::pair<const char*, const char*> extent(const torch::Tensor& t) {
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) == 0) return {nullptr, nullptr};
    last += (t.size(d) - 1) * t.stride(d);
  }
  const char* p = (const char*)t.data_ptr();
  return {p, p + (last + 1) * t.element_size()};
}

inline bool overlap(const torch::Tensor& a, const torch::Tensor& b) {
  const auto x = extent(a), y = extent(b);
  return x.first < y.second && y.first < x.second;
}

// A tensor's elements as bytes: dimensions by falling stride, the element itself last.
struct Spread {
  const char* at;
  std::vector<std::pair<int64_t, int64_t>> dims;   // stride, size
  int64_t element;
  explicit Spread(const torch::Tensor& t) : at((const char*)t.data_ptr()), element(t.element_size()) {
    for (int64_t d = 0; d < t.dim(); ++d)
      if (t.size(d) > 1 && t.stride(d) != 0) dims.emplace_back(t.stride(d) * element, t.size(d));
    std::sort(dims.rbegin(), dims.rend());
  }
  int64_t span(size_t from) const {                // bytes from the first to the last, of the dimensions from this one on
    int64_t n = element;
    for (size_t i = from; i < dims.size(); ++i) n += (dims[i].second - 1) * dims[i].first;
    return n;
  }
};

// Whether b, which begins d bytes behind a, may have a byte of a's; `i` dimensions of both are done with.  Where both go on
// by the same stride and fit into it, a block of a's meets at most two of b's: those that begin less than a stride before or
// behind it.  Otherwise what lies within the other's reach counts as shared.
inline bool may_meet(const Spread& a, const Spread& b, size_t i, int64_t d) {
  if (d >= a.span(i) || d + b.span(i) <= 0) return false;
  if (i >= a.dims.size() || i >= b.dims.size() || a.dims[i].first != b.dims[i].first) return true;
  const int64_t s = a.dims[i].first;
  if (a.span(i + 1) > s || b.span(i + 1) > s) return true;
  const int64_t r = (d % s + s) % s;
  return may_meet(a, b, i + 1, r) || may_meet(a, b, i + 1, r - s);
}

inline bool may_share_memory(const torch::Tensor& a, const torch::Tensor& b) {
  if (!overlap(a, b)) return false;
  const Spread x(a), y(b);
  return may_meet(x, y, 0, y.at - x.at);
}

// Behind a shape there may be no numbers to read: a sparse layout, a lazy zero or
// negation, a storage that was freed (sharded parameters between their uses), or
// a wrapper of other tensors (distributed, quantised or fake ones).
inline void check_memory(const char* op, const char* name, const torch::Tensor& t) {
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
inline void check_input(const char* op, const char* name, const torch::Tensor& t, const torch::Device& dev) {
  TORCH_CHECK_VALUE(t.device() == dev, op, ": ", name, " must be on ", dev.str(), ", not on ", t.device().str());
  TORCH_CHECK(!(t.requires_grad() && c10::GradMode::is_enabled()), op, ": ", name,
              " requires a gradient, but the operator has no backward; call it under torch.no_grad()");
  TORCH_CHECK(!(t._fw_grad(/*level=*/0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode()), op, ": ", name,
              " carries a forward-mode tangent, but the operator has no derivative; take the primal of it");
  check_memory(op, name, t);
}

inline void check_cuda(const char* op, const torch::Device& dev) {
  TORCH_CHECK_VALUE(dev.is_cuda(), op, ": the tensors must be on a CUDA device, not on ", dev.str());
}

inline void check_vector(const char* op, const char* name, const torch::Tensor& t, const torch::Device& dev, at::IntArrayRef shape) {
  check_input(op, name, t, dev);
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kFloat32 && t.sizes() == shape && t.is_contiguous(), op, ": ", name,
                    " must be a contiguous fp32 tensor of shape ", text(shape));
}

// A given out was written: an operation that saved it for its backward pass has to notice.
inline void written(const OptTensor& out) {
  if (out && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
}

}  // namespace raiccl
