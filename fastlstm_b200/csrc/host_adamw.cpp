// Host side of the AdamW step: parameters, gradients and states collected and checked, tensors of one type handed to a call of the C ABI.  (A
// step over a layer's four tensors took 31 us where Python collected them.)
#include "host_language.h"

#include <algorithm>
#include <cfloat>

#include <torch/csrc/autograd/python_variable.h>
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
  return plain(g).contiguous();
}

float* f32(const Tensor& t, const char* name, const Tensor& param, int64_t n) {
  beside(t, name, param);
  if (t.scalar_type() != at::kFloat || t.numel() != n || !t.is_contiguous())
    throw wrong(std::string(name) + " must be " + std::to_string(n) + " contiguous float32 elements");
  return static_cast<float*>(t.data_ptr());
}

// The tensors of one call: of a group, a device and a type.
struct Bucket {
  std::vector<Tensor> params, grads;           // (grads dense, held until the launch)
  std::vector<blstm_adamw_item> items;
  blstm_adamw_desc d{};
  Tensor ticket;
};

PyObject* interned(const char* name) { return PyUnicode_InternFromString(name); }

const Tensor& state_tensor(PyObject* state, PyObject* name) {
  PyObject* t = PyDict_GetItemWithError(state, name);
  if (!t || !THPVariable_Check(t)) throw wrong("an optimizer state has no tensor " + std::string(PyUnicode_AsUTF8(name)));
  return THPVariable_Unpack(t);
}

py::handle entry(PyObject* group, PyObject* name) {
  PyObject* v = PyDict_GetItemWithError(group, name);
  if (!v) throw wrong("a parameter group has no " + std::string(PyUnicode_AsUTF8(name)));
  return v;
}

// A finite number of 32 bits, `low` or more.
double number_of(PyObject* group, PyObject* name, double low) {
  PyObject* v = entry(group, name).ptr();
  const double d = THPVariable_Check(v) ? THPVariable_Unpack(v).item<double>() : PyFloat_AsDouble(v);
  if (d == -1.0 && PyErr_Occurred()) throw py::error_already_set();
  if (!(d >= low && std::isfinite((float)d)))
    throw wrong(std::string(PyUnicode_AsUTF8(name)) + " must be " + (low == 0 ? "at least 0 and " : "") + "finite in 32 bits, got " + std::to_string(d));
  return d;
}

template <typename T>
T cast(PyObject* group, PyObject* name, const char* what) {
  try {
    return entry(group, name).cast<T>();
  } catch (const py::cast_error&) {
    throw wrong(std::string(PyUnicode_AsUTF8(name)) + " must be " + what);
  }
}

// A step over the parameter groups of an optimizer (optim.py).  start(p): makes the state of a parameter that has none; scratch(p): the
// counter of p's device and its {norm, factor}.  Returns {norm, factor} where max_norm is given and there was anything to do.
std::optional<Tensor> adamw_step(const py::list& groups, const py::dict& state, int bits, bool masters, std::optional<double> max_norm,
                                 const py::object& start, const py::object& scratch) {
  static PyObject *const k_params = interned("params"), *const k_m = interned("exp_avg"), *const k_v = interned("exp_avg_sq"),
                  *const k_u = interned("exp_avg_sq_root"), *const k_ms = interned("exp_avg_scale"), *const k_us = interned("exp_avg_sq_root_scale"),
                  *const k_step = interned("step"), *const k_master = interned("master"), *const k_lr = interned("lr"), *const k_betas = interned("betas"),
                  *const k_eps = interned("eps"), *const k_decay = interned("weight_decay"), *const k_seed = interned("seed");
  const at::ScalarType state_type = bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
  std::vector<std::pair<PyObject*, Bucket>> calls;       // with the group of each
  uint32_t number = 0;
  for (const py::handle group_in : groups) {
    PyObject* group = group_in.ptr();
    const size_t begin = calls.size();
    const py::list params = py::reinterpret_borrow<py::list>(PyDict_GetItemWithError(group, k_params));
    for (const py::handle at : params) {
      const uint32_t mine = number++;
      if (!THPVariable_Check(at.ptr())) throw wrong("a parameter must be a tensor");
      const Tensor& p = THPVariable_Unpack(at.ptr());
      if (!p.grad().defined()) continue;
      on_gpu(p, "a parameter");
      dtype_code(p.scalar_type());
      if (p.is_neg()) throw wrong("a parameter must not be a lazily negated tensor");
      if (!p.is_contiguous()) throw wrong("a parameter of shape " + shape_str(p.sizes()) + " must be contiguous");
      PyObject* s = PyDict_GetItemWithError(state.ptr(), at.ptr());
      py::object made;
      if (!s || PyDict_GET_SIZE(s) == 0) {
        made = start(at);
        s = made.ptr();
      }
      Bucket* b = nullptr;
      for (size_t k = begin; k < calls.size(); ++k)
        if (calls[k].second.params[0].device() == p.device() && calls[k].second.params[0].scalar_type() == p.scalar_type()) b = &calls[k].second;
      if (!b) {
        calls.emplace_back(group, Bucket());
        b = &calls.back().second;
      }
      blstm_adamw_item a{};
      a.n = p.numel();
      a.number = mine;
      a.exp_avg = flat(state_tensor(s, k_m), "exp_avg", p, state_type).data_ptr();
      a.exp_avg_sq = flat(state_tensor(s, bits == 8 ? k_u : k_v), bits == 8 ? "exp_avg_sq_root" : "exp_avg_sq", p, state_type).data_ptr();
      const Tensor& step = state_tensor(s, k_step);
      beside(step, "step", p);
      if (step.scalar_type() != at::kLong || step.numel() != 1) throw wrong("step must be one int64 element");
      a.step = static_cast<int64_t*>(step.data_ptr());
      if (bits == 8) {
        a.exp_avg_scale = f32(state_tensor(s, k_ms), "exp_avg_scale", p, (a.n + 255) / 256);
        a.exp_avg_sq_scale = f32(state_tensor(s, k_us), "exp_avg_sq_root_scale", p, (a.n + 255) / 256);
      }
      if (masters && p.scalar_type() != at::kFloat) a.master = f32(flat(state_tensor(s, k_master), "master", p, at::kFloat), "master", p, a.n);
      b->params.push_back(p);
      b->grads.push_back(dense_grad(p.grad(), p));
      a.param = p.data_ptr();
      a.grad = ptr(b->grads.back());
      if (a.n) b->items.push_back(a);
    }
  }
  if (calls.empty()) return std::nullopt;
  // (a launch works on all of its tensors at a time)
  std::vector<std::pair<uintptr_t, uintptr_t>> ranges;
  for (const auto& [group, b] : calls)
    for (const Tensor& p : b.params)
      if (p.numel()) ranges.emplace_back(reinterpret_cast<uintptr_t>(ptr(p)), reinterpret_cast<uintptr_t>(ptr(p)) + p.nbytes());
  std::sort(ranges.begin(), ranges.end());
  for (size_t k = 1; k < ranges.size(); ++k)
    if (ranges[k].first < ranges[k - 1].second) throw wrong("parameters share memory");
  // Everything that can be refused is, before the first launch: groups and types are launched one by one, and a step is taken by all of
  // them or by none.
  auto scratch_of = [&](const Bucket& b) { return scratch(b.params[0].device().index()).cast<std::pair<Tensor, Tensor>>(); };
  std::optional<Tensor> norm;
  blstm_grad_norm_desc n{};
  std::vector<blstm_grad_item> grads;
  Tensor ws;
  if (max_norm) {
    const Bucket& first = calls[0].second;
    for (const auto& [group, b] : calls) {
      if (b.params[0].device() != first.params[0].device()) throw wrong("max_norm takes parameters on one device");
      for (const blstm_adamw_item& a : b.items) grads.push_back({a.grad, a.n, dtype_code(b.params[0].scalar_type()), 0});
    }
    const auto [ticket, out] = scratch_of(first);
    norm = out;
    n.item = grads.data();
    n.items = (int32_t)grads.size();
    n.max_norm = (float)*max_norm;
    n.out = static_cast<float*>(out.data_ptr());
    n.ticket = static_cast<uint32_t*>(ticket.data_ptr());
    n.workspace_bytes = blstm_grad_norm_workspace(n.items);
    ws = fresh({(int64_t)n.workspace_bytes}, at::kByte, out);
    n.workspace = ws.data_ptr();
  }
  for (auto& [group, b] : calls) {
    if (b.items.empty()) continue;
    blstm_adamw_desc& d = b.d;
    d.dtype = dtype_code(b.params[0].scalar_type());
    d.bits = bits;
    d.items = (int32_t)b.items.size();
    d.item = b.items.data();
    PyObject* lr = entry(group, k_lr).ptr();
    if (THPVariable_Check(lr) && THPVariable_Unpack(lr).is_cuda()) {
      const Tensor& t = THPVariable_Unpack(lr);
      beside(t, "lr", b.params[0]);
      if (t.scalar_type() != at::kFloat || t.numel() != 1) throw wrong("lr on the GPU must be one float32 element");
      d.lr_at = static_cast<const float*>(ptr(t));
    } else {
      d.lr = number_of(group, k_lr, -HUGE_VAL);
    }
    const auto betas = cast<std::pair<double, double>>(group, k_betas, "two numbers");
    for (const double beta : {betas.first, betas.second})
      if (!(beta >= 0 && beta < 1)) throw wrong("betas must be in [0, 1), got " + std::to_string(beta));
    d.beta1 = betas.first; d.beta2 = betas.second;
    d.eps = number_of(group, k_eps, 0);
    if (d.eps > 0 && d.eps < FLT_MIN) throw wrong("eps must be 0 or at least 2^-126");
    d.weight_decay = number_of(group, k_decay, -HUGE_VAL);
    d.seed = cast<uint64_t>(group, k_seed, "a whole number in [0, 2^64)");
    if (norm) d.factor = static_cast<const float*>(ptr(*norm)) + 1;
    b.ticket = scratch_of(b).first;
    d.ticket = static_cast<uint32_t*>(b.ticket.data_ptr());
  }
  for (const auto& [group, b] : calls) {
    const Call heard(b.params[0].device());     // (throws what an earlier launch has left)
    if (!b.items.empty())
      for (const Tensor& p : b.params) torch::autograd::impl::bump_version(p);
  }
  if (!grads.empty()) {
    const Call call(norm->device(), false);
    check(blstm_grad_norm(&n, call.stream), "gradient norm");
  }
  for (const auto& [group, b] : calls) {
    if (b.items.empty()) continue;
    const Call call(b.params[0].device(), false);
    check(blstm_adamw(&b.d, call.stream), "adamw");
  }
  return norm;
}

}  // namespace

namespace blstm_host {

void bind_adamw(py::module_& m) {
  m.def("adamw_step", &adamw_step);
}

}  // namespace blstm_host
