// What the host side of the operators around a language model shares: checks, leading dimensions as two strides, autograd nodes.
#pragma once

#include <ATen/cuda/EmptyTensor.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <cmath>

#include "host.h"

namespace blstm_host {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

inline py::value_error wrong(const std::string& what) { return py::value_error(what); }

inline void on_gpu(const Tensor& t, const char* name) {
  if (!t.is_cuda()) throw wrong(std::string(name) + " must be a CUDA tensor (there is no CPU path)");
}
inline void beside(const Tensor& t, const char* name, const Tensor& other) {
  on_gpu(t, name);
  if (t.device() != other.device()) throw wrong(std::string(name) + " is on " + t.device().str() + ", expected " + other.device().str());
}
inline void same(const Tensor& t, const char* name, at::ScalarType dt, at::IntArrayRef shape) {
  if (t.scalar_type() != dt) throw wrong(std::string(name) + " has dtype " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(dt));
  if (t.sizes() != shape) throw wrong(std::string(name) + " has shape " + shape_str(t.sizes()) + ", expected " + shape_str(shape));
}
inline int token_bits(const Tensor& tokens) {
  if (tokens.scalar_type() == at::kLong) return 64;
  if (tokens.scalar_type() == at::kInt) return 32;
  throw wrong(std::string("tokens have dtype ") + c10::toString(tokens.scalar_type()) + ", expected int64 or int32");
}

// The numbers themselves where their signs are still to be turned (z.conj().imag).
inline Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// The leading dimensions of an operator's tensors as [n0, n1].
struct Lead {
  int64_t dims, n0, n1;
  explicit Lead(at::IntArrayRef s) : dims((int64_t)s.size()), n0(1), n1(1) {
    if (dims == 2) { n0 = s[0]; n1 = s[1]; }
    else n1 = c10::multiply_integers(s);
    if (n0 > 0 && n1 > INT32_MAX / n0) throw wrong("more than 2^31 - 1 rows");
  }
  // t with `dims` leading dimensions as one whose rows stride[0..1] reach
  Tensor rows(const Tensor& t, int64_t stride[2]) const {
    Tensor v = plain(dims > 2 ? t.flatten(0, dims - 1) : t);
    const int64_t lead = dims > 2 ? 1 : dims;
    if (v.dim() > lead && v.size(-1) > 1 && v.stride(-1) != 1) v = v.contiguous();
    stride[0] = lead == 2 ? v.stride(0) : 0;
    stride[1] = lead == 0 ? 0 : v.stride(lead - 1);
    return v;
  }
};

inline Tensor fresh(at::IntArrayRef sizes, at::ScalarType dt, const Tensor& like) { return at::detail::empty_cuda(sizes, dt, like.device(), std::nullopt); }

// A leaf whose gradients are added up on the default stream, because a graph from before the capture lives: that stream cannot wait for a captured
// one, so the backward pass cannot be captured, and trying ends the process.  (Other streams are joined into the capture.)
inline void check_capture(const Tensor& t) {
  if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
  const auto adds = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!adds || adds->num_inputs() == 0) return;
  const auto device = t.device().index();
  if (adds->input_metadata(0).stream() != at::cuda::getDefaultCUDAStream(device).unwrap()) return;
  cudaStreamCaptureStatus status;
  cuda_ok(cudaStreamIsCapturing(at::cuda::getCurrentCUDAStream(device).stream(), &status), "cudaStreamIsCapturing");
  TORCH_CHECK(status == cudaStreamCaptureStatusNone,
              "fastlstm_b200: a graph of this leaf from before the capture lives, on the default stream; free it (or warm up on another stream) first");
}

// A node of the graph that an operator's gradient is, with what it needs as members (a torch::autograd::Function keeps that in a
// dictionary: 4 us a call).  Backward goes through it once.
template <typename N, typename... I>
std::shared_ptr<N> make_node(const I&... inputs) {
  (check_capture(inputs), ...);
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}

inline bool wants_grad(const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), "fastlstm_b200: forward-mode gradients are not there for this operator");
  return at::GradMode::is_enabled() && t.requires_grad();
}
inline void only_once() { TORCH_CHECK(!at::GradMode::is_enabled(), "fastlstm_b200: gradients of gradients (create_graph) are not there for this operator"); }

inline std::vector<int64_t> plus(at::IntArrayRef s, int64_t last) {
  std::vector<int64_t> v = s.vec();
  v.push_back(last);
  return v;
}

}  // namespace blstm_host
