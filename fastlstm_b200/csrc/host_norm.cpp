// Host side of the root-mean-square norm: argument checks, buffers, the calls of the C ABI and the autograd node.
#include "host_language.h"

namespace {

using namespace blstm_host;

blstm_norm_desc norm_desc(const Tensor& x, const Lead& lead, double eps) {
  blstm_norm_desc d{};
  d.dtype = dtype_code(x.scalar_type());
  d.eps = (float)eps;
  d.n0 = lead.n0; d.n1 = lead.n1;
  d.width = x.size(-1);
  return d;
}

void check_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
  on_gpu(x, "x");
  dtype_code(x.scalar_type());
  if (x.dim() < 1 || x.size(-1) == 0) throw wrong("expected x as [..., width], got " + shape_str(x.sizes()));
  beside(weight, "weight", x);
  same(weight, "weight", x.scalar_type(), {x.size(-1)});
  if (residual) {
    beside(*residual, "residual", x);
    same(*residual, "residual", x.scalar_type(), x.sizes());
  }
  if (!(eps >= 0 && std::isfinite((float)eps))) throw wrong("eps must be at least 0 and finite in 32 bits");
}

// {y, h}, or {values, scales, h} in 8 bits; h is undefined without a residual.  rstd, where it is asked for.
std::array<Tensor, 3> norm_impl(const Tensor& x_in, const Tensor& weight_in, const OptTensor& residual, double eps, bool eight_bits, Tensor* rstd) {
  const auto lead_sizes = x_in.sizes().slice(0, x_in.dim() - 1);
  const Lead lead(lead_sizes);
  blstm_norm_desc d = norm_desc(x_in, lead, eps);
  const Tensor x = lead.rows(x_in, d.x_stride), weight = plain(weight_in).contiguous();
  const Tensor r = residual ? lead.rows(*residual, d.residual_stride) : Tensor();
  Call call(x.device());
  const Tensor h = residual ? fresh(x_in.sizes(), x.scalar_type(), x) : Tensor();
  const void* rp = residual ? ptr(r) : nullptr;
  void* hp = residual ? h.data_ptr() : nullptr;
  if (eight_bits) {
    const Tensor q = fresh(x_in.sizes(), at::kFloat8_e4m3fn, x), scales = fresh(lead_sizes, at::kFloat, x);
    check(blstm_rms_norm_e4m3(&d, ptr(x), rp, ptr(weight), q.data_ptr(), (float*)scales.data_ptr(), hp, call.stream), "rms_norm_e4m3");
    return {q, scales, h};
  }
  const Tensor y = fresh(x_in.sizes(), x.scalar_type(), x);
  if (rstd) *rstd = fresh({lead.n0 * lead.n1}, at::kFloat, x);
  check(blstm_rms_norm(&d, ptr(x), rp, ptr(weight), y.data_ptr(), hp, rstd ? (float*)rstd->data_ptr() : nullptr, call.stream), "rms_norm");
  return {y, h, Tensor()};
}

struct NormGrad : public Node {
  SavedVariable h, weight, rstd;
  bool sum = false, h_is_output = false;      // whether h is a sum, and one that the graph knows
  double eps = 0;
  void release_variables() override {
    for (SavedVariable* v : {&h, &weight, &rstd}) v->reset_data();
  }
  variable_list apply(variable_list&& g) override {
    only_once();
    const size_t last = sum ? 2 : 1;            // the weight among the inputs
    variable_list r(last + 1);
    const Tensor dy = g[0], dsum = h_is_output ? g[1] : Tensor();
    if (!dy.defined()) {                        // only the sum was used
      for (size_t k = 0; k < last; ++k) r[k] = dsum;
      return r;
    }
    const Tensor at_h = h_is_output ? h.unpack(getptr()) : h.unpack(), w_in = weight.unpack(), i = rstd.unpack();
    const Lead lead(at_h.sizes().slice(0, at_h.dim() - 1));
    blstm_norm_desc d = norm_desc(at_h, lead, eps);
    const Tensor rows = lead.rows(at_h, d.x_stride), w = plain(w_in).contiguous(), up = lead.rows(dy, d.dy_stride);
    const Tensor ds = dsum.defined() ? lead.rows(dsum, d.residual_stride) : Tensor();
    Call call(rows.device());
    const Tensor dx = fresh(at_h.sizes(), at_h.scalar_type(), at_h);
    Tensor dw, ws;
    const size_t bytes = task_should_compute_output(last) ? blstm_rms_norm_grad_workspace(&d) : 0;
    if (task_should_compute_output(last)) {
      dw = fresh(w.sizes(), w.scalar_type(), w);
      ws = fresh({(int64_t)bytes}, at::kByte, w);
    }
    check(blstm_rms_norm_grad(&d, ptr(up), dsum.defined() ? ptr(ds) : nullptr, ptr(rows), ptr(w), static_cast<const float*>(ptr(i)), dx.data_ptr(),
                              dw.defined() ? dw.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, call.stream),
          "rms_norm gradient");
    for (size_t k = 0; k < last; ++k) r[k] = dx;
    r[last] = dw;
    return r;
  }
};

py::object rms_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
  std::array<Tensor, 3> r;
  {
    py::gil_scoped_release nogil;
    check_norm(x, weight, residual, eps);
    const bool of_x = wants_grad(x), of_r = residual && wants_grad(*residual), of_w = wants_grad(weight);
    if (!(of_x || of_r || of_w)) {
      r = norm_impl(x, weight, residual, eps, false, nullptr);
    } else {
      const auto node = residual ? make_node<NormGrad>(x, *residual, weight) : make_node<NormGrad>(x, weight);
      Tensor rstd;
      {
        at::AutoDispatchBelowADInplaceOrView guard;
        r = norm_impl(x, weight, residual, eps, false, &rstd);
      }
      node->sum = residual.has_value();
      node->h_is_output = node->sum && (of_x || of_r);
      node->eps = eps;
      torch::autograd::set_history(r[0], node);
      if (node->h_is_output) torch::autograd::set_history(r[1], node);
      node->h = SavedVariable(residual ? r[1] : x, node->h_is_output);
      node->weight = SavedVariable(weight, false);
      node->rstd = SavedVariable(rstd, false);
    }
  }
  if (!residual) return py::cast(r[0]);
  return py::make_tuple(r[0], r[1]);
}

py::tuple rms_norm_e4m3(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
  std::array<Tensor, 3> r;
  {
    py::gil_scoped_release nogil;
    check_norm(x, weight, residual, eps);
    if (wants_grad(x) || wants_grad(weight) || (residual && wants_grad(*residual)))
      throw wrong("an output in 8 bits has no gradient: call rms_norm_e4m3 under torch.no_grad() or on detached tensors");
    r = norm_impl(x, weight, residual, eps, true, nullptr);
  }
  return py::make_tuple(r[0], r[1], residual ? py::cast(r[2]) : py::none());
}

}  // namespace

namespace blstm_host {

void bind_norm(py::module_& m) {
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_e4m3", &rms_norm_e4m3);
}

}  // namespace blstm_host
