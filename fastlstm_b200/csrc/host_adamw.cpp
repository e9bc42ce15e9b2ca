// Host side of the AdamW step: lists of tensors checked and handed to the C ABI, tensors of one type to a call.
#include "host_language.h"

#include <torch/csrc/autograd/variable.h>

namespace {

using namespace blstm_host;

const Tensor& flat(const Tensor& t, const char* name, const Tensor& param, at::ScalarType dt) {
  beside(t, name, param);
  if (t.scalar_type() != dt) throw wrong(std::string(name) + " has dtype " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(dt));
  if (t.sizes() != param.sizes()) throw wrong(std::string(name) + " has shape " + shape_str(t.sizes()) + ", expected " + shape_str(param.sizes()));
  if (!t.is_contiguous()) throw wrong(std::string(name) + " must be contiguous");
  return t;
}

// A gradient as the kernels read it: dense and in the parameter's order (a copy where it is not).
Tensor dense_grad(const Tensor& g, const Tensor& param) {
  if (g.layout() != at::kStrided) throw wrong("sparse gradients are not there for AdamW");
  beside(g, "a gradient", param);
  same(g, "a gradient", param.scalar_type(), param.sizes());
  return g.contiguous();
}

float* f32(const Tensor& t, const char* name, const Tensor& param, int64_t n) {
  beside(t, name, param);
  if (t.scalar_type() != at::kFloat || t.numel() != n || !t.is_contiguous())
    throw wrong(std::string(name) + " must be " + std::to_string(n) + " contiguous float32 elements");
  return static_cast<float*>(t.data_ptr());
}

// params [k], and of each {exp_avg, exp_avg_sq (8 bits: its root), step [, scale, scale] [, master]}; norm: {norm, factor}, written first
// where max_norm is positive.
void adamw(const std::vector<Tensor>& params, const std::vector<Tensor>& grads_in, const std::vector<std::vector<Tensor>>& states,
           const std::vector<uint32_t>& numbers, int bits, bool masters, double lr, const OptTensor& lr_at, double beta1, double beta2, double eps,
           double weight_decay, uint64_t seed, const OptTensor& norm, const Tensor& ticket) {
  py::gil_scoped_release nogil;
  if (params.empty()) return;
  const Tensor& first = params[0];
  on_gpu(first, "a parameter");
  std::vector<Tensor> grads;
  std::vector<blstm_adamw_item> items;
  grads.reserve(params.size());
  items.reserve(params.size());
  blstm_adamw_desc d{};
  d.dtype = dtype_code(first.scalar_type());
  const size_t expected = 3 + (bits == 8 ? 2 : 0) + (masters ? 1 : 0);
  const at::ScalarType state_type = bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
  for (size_t k = 0; k < params.size(); ++k) {
    const Tensor& p = params[k];
    beside(p, "a parameter", first);
    if (p.scalar_type() != first.scalar_type()) throw wrong("parameters of one call have one dtype");
    if (!p.is_contiguous()) throw wrong("a parameter of shape " + shape_str(p.sizes()) + " must be contiguous");
    const std::vector<Tensor>& s = states[k];
    if (s.size() != expected) throw wrong("an optimizer state has other tensors than expected");
    if (p.numel() == 0) continue;
    grads.push_back(dense_grad(grads_in[k], p));
    blstm_adamw_item a{};
    a.param = p.data_ptr();
    a.grad = ptr(grads.back());
    a.exp_avg = flat(s[0], "exp_avg", p, state_type).data_ptr();
    a.exp_avg_sq = flat(s[1], "exp_avg_sq", p, state_type).data_ptr();
    beside(s[2], "step", p);
    if (s[2].scalar_type() != at::kLong || s[2].numel() != 1) throw wrong("step must be one int64 element");
    a.step = static_cast<int64_t*>(s[2].data_ptr());
    a.n = p.numel();
    a.number = numbers[k];
    if (bits == 8) {
      a.exp_avg_scale = f32(s[3], "exp_avg_scale", p, (a.n + 255) / 256);
      a.exp_avg_sq_scale = f32(s[4], "exp_avg_sq_root_scale", p, (a.n + 255) / 256);
    }
    if (masters) a.master = f32(flat(s.back(), "master", p, at::kFloat), "master", p, a.n);
    items.push_back(a);
  }
  if (items.empty()) return;
  if (lr_at) {
    beside(*lr_at, "lr", first);
    if (lr_at->scalar_type() != at::kFloat || lr_at->numel() != 1) throw wrong("lr on the GPU must be one float32 element");
    d.lr_at = static_cast<const float*>(ptr(*lr_at));
  }
  d.bits = bits;
  d.items = (int32_t)items.size();
  d.item = items.data();
  d.lr = lr; d.beta1 = beta1; d.beta2 = beta2; d.eps = eps; d.weight_decay = weight_decay;
  d.seed = seed;
  if (norm) d.factor = static_cast<const float*>(ptr(*norm)) + 1;
  d.ticket = static_cast<uint32_t*>(ticket.data_ptr());
  Call call(first.device());
  check(blstm_adamw(&d, call.stream), "adamw");
  for (const Tensor& p : params) torch::autograd::impl::bump_version(p);
}

void grad_norm(const std::vector<Tensor>& grads_in, double max_norm, const Tensor& out, const Tensor& ticket) {
  py::gil_scoped_release nogil;
  std::vector<Tensor> grads;
  std::vector<blstm_grad_item> items;
  for (const Tensor& g_in : grads_in) {
    if (g_in.layout() != at::kStrided) throw wrong("sparse gradients are not there for AdamW");
    beside(g_in, "a gradient", out);
    if (g_in.numel() == 0) continue;
    grads.push_back(g_in.contiguous());
    blstm_grad_item a{};
    a.grad = ptr(grads.back());
    a.n = grads.back().numel();
    a.dtype = dtype_code(g_in.scalar_type());
    items.push_back(a);
  }
  if (items.empty()) return;
  Call call(out.device());
  blstm_grad_norm_desc d{};
  d.item = items.data();
  d.items = (int32_t)items.size();
  d.max_norm = (float)max_norm;
  d.out = static_cast<float*>(out.data_ptr());
  d.ticket = static_cast<uint32_t*>(ticket.data_ptr());
  d.workspace_bytes = blstm_grad_norm_workspace(d.items);
  const Tensor ws = fresh({(int64_t)d.workspace_bytes}, at::kByte, out);
  d.workspace = ws.data_ptr();
  check(blstm_grad_norm(&d, call.stream), "gradient norm");
}

}  // namespace

namespace blstm_host {

void bind_adamw(py::module_& m) {
  m.def("adamw", &adamw);
  m.def("grad_norm", &grad_norm);
}

}  // namespace blstm_host
