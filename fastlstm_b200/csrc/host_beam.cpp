// Host side of beam search: argument checks, buffers, the calls of the C ABI.
#include "host_language.h"

#include <torch/csrc/autograd/python_variable.h>

namespace {

using namespace blstm_host;

void without_grad(const Tensor& t, const char* what) {
  if (wants_grad(t)) throw wrong(std::string(what) + " has no gradient: call it under torch.no_grad() or on detached tensors");
}

py::tuple beam_step(const Tensor& logits_in, const Tensor& scores_in, std::optional<int64_t> width_in, std::optional<int64_t> end_token,
                    const OptTensor& finished_in, const OptTensor& lengths_in, double length_penalty) {
  Tensor scores, parents, tokens, finished, lengths;
  {
    py::gil_scoped_release nogil;
    on_gpu(logits_in, "logits");
    blstm_beam_desc d{};
    d.dtype = dtype_code(logits_in.scalar_type());
    if (logits_in.dim() != 3 || logits_in.size(2) == 0 || logits_in.size(1) == 0)
      throw wrong("expected logits as [batch, hypotheses, vocabulary], got " + shape_str(logits_in.sizes()));
    d.batch = logits_in.size(0); d.beams = logits_in.size(1); d.vocab = logits_in.size(2);
    if (d.beams > BLSTM_MAX_BEAMS) throw wrong("at most " + std::to_string(BLSTM_MAX_BEAMS) + " hypotheses of a sentence");
    if (d.beams * d.vocab > UINT32_MAX) throw wrong("at most 2^32 - 1 continuations of a sentence");
    const auto shape = logits_in.sizes().slice(0, 2);
    const int64_t width = width_in.value_or(d.beams);
    const int64_t most = std::min<int64_t>(BLSTM_MAX_TOP, d.beams * d.vocab);
    if (width < 1 || width > most) throw wrong("width must be between 1 and " + std::to_string(most));
    d.width = (int32_t)width;
    beside(scores_in, "scores", logits_in);
    same(scores_in, "scores", at::kFloat, shape);
    if (end_token && (*end_token < 0 || *end_token >= d.vocab)) throw wrong("end_token is outside of the vocabulary of " + std::to_string(d.vocab));
    d.end_token = end_token.value_or(-1);
    if (finished_in) {
      if (!end_token) throw wrong("finished needs an end_token");
      beside(*finished_in, "finished", logits_in);
      same(*finished_in, "finished", at::kBool, shape);
    }
    if (lengths_in) {
      beside(*lengths_in, "lengths", logits_in);
      same(*lengths_in, "lengths", at::kLong, shape);
    }
    if (!(length_penalty >= 0 && length_penalty <= BLSTM_MAX_LENGTH_PENALTY))
      throw wrong("length_penalty must be between 0 and " + std::to_string(BLSTM_MAX_LENGTH_PENALTY));
    if (length_penalty != 0 && !lengths_in) throw wrong("length_penalty needs lengths");
    d.length_penalty = length_penalty;
    without_grad(logits_in, "beam_step");
    without_grad(scores_in, "beam_step");
    const Lead lead(shape);
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor logits = lead.rows(logits_in, d.logits_stride), given = plain(scores_in).contiguous();
    const Tensor ended = finished_in ? finished_in->contiguous() : Tensor(), written = lengths_in ? lengths_in->contiguous() : Tensor();
    Call call(logits.device());
    const int64_t out[2] = {d.batch, width};
    scores = fresh(out, at::kFloat, logits);
    parents = fresh(out, at::kLong, logits);
    tokens = fresh(out, at::kLong, logits);
    if (end_token) finished = fresh(out, at::kBool, logits);
    if (lengths_in) lengths = fresh(out, at::kLong, logits);
    const size_t bytes = blstm_beam_workspace(&d);
    const Tensor ws = fresh({(int64_t)bytes}, at::kByte, logits);
    auto i64 = [](const Tensor& t) { return t.defined() ? static_cast<int64_t*>(t.data_ptr()) : nullptr; };
    check(blstm_beam_step(&d, ptr(logits), static_cast<const float*>(ptr(given)), finished_in ? static_cast<const uint8_t*>(ptr(ended)) : nullptr,
                          lengths_in ? static_cast<const int64_t*>(ptr(written)) : nullptr, static_cast<float*>(scores.data_ptr()), i64(parents),
                          i64(tokens), end_token ? static_cast<uint8_t*>(finished.data_ptr()) : nullptr, i64(lengths), ws.data_ptr(), bytes, call.stream),
          "beam_step");
  }
  return py::make_tuple(scores, parents, tokens, end_token ? py::cast(finished) : py::none(), lengths_in ? py::cast(lengths) : py::none());
}

// Whether what a tensor has behind `dim` is one piece of memory, and the dimensions in front of it are one stride.
bool in_pieces(const Tensor& t, int64_t dim, int64_t& outer_stride) {
  int64_t next = 1;
  for (int64_t i = t.dim() - 1; i > dim; --i) {
    if (t.size(i) != 1 && t.stride(i) != next) return false;
    next *= t.size(i);
  }
  outer_stride = 0;
  next = -1;
  for (int64_t i = dim - 1; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (next < 0) outer_stride = t.stride(i);
    else if (t.stride(i) != next) return false;
    next = t.stride(i) * t.size(i);
  }
  return true;
}

// [.., batch * hypotheses along dim, ..] of each tensor -> [.., batch * width, ..]
std::vector<Tensor> reorder_flat(const std::vector<Tensor>& states, const Tensor& parents_in, int64_t dim_in) {
  py::gil_scoped_release nogil;
  on_gpu(parents_in, "parents");
  token_bits(parents_in);
  if (parents_in.dim() != 2) throw wrong("expected parents as [batch, width], got " + shape_str(parents_in.sizes()));
  const int64_t batch = parents_in.size(0), width = parents_in.size(1);
  if (width == 0) throw wrong("expected parents as [batch, width], got " + shape_str(parents_in.sizes()));
  at::AutoDispatchBelowADInplaceOrView guard;
  const Tensor parents = parents_in.contiguous();
  std::vector<Tensor> held, out;
  std::vector<blstm_reorder_item> items;
  int64_t beams = -1;
  for (const Tensor& t : states) {
    beside(t, "a state", parents_in);
    without_grad(t, "reorder_states");
    if (t.layout() != at::kStrided) throw wrong("a state must be a dense tensor");
    const int64_t dim = dim_in < 0 ? dim_in + t.dim() : dim_in;
    if (dim < 0 || dim >= t.dim()) throw wrong("a state of shape " + shape_str(t.sizes()) + " has no dimension " + std::to_string(dim_in));
    const int64_t rows = t.size(dim);
    if (batch == 0 ? rows != 0 : rows == 0 || rows % batch != 0)
      throw wrong("a state of shape " + shape_str(t.sizes()) + " has no whole number of hypotheses for each of " + std::to_string(batch) + " sentences");
    if (batch && beams >= 0 && rows != batch * beams) throw wrong("states have different numbers of hypotheses");
    if (batch) beams = rows / batch;
  }
  Call call(parents.device());
  for (const Tensor& t : states) {
    const int64_t dim = dim_in < 0 ? dim_in + t.dim() : dim_in, e = t.element_size();
    std::vector<int64_t> sizes = t.sizes().vec();
    sizes[dim] = batch * width;
    out.push_back(fresh(sizes, t.scalar_type(), t));
    if (out.back().numel() == 0) continue;
    const int64_t outer = c10::multiply_integers(t.sizes().slice(0, dim)), inner = c10::multiply_integers(t.sizes().slice(dim + 1));
    Tensor v = t.resolve_conj().resolve_neg();
    int64_t outer_stride;
    if (!in_pieces(v, dim, outer_stride)) {
      v = v.contiguous();
      in_pieces(v, dim, outer_stride);
    }
    held.push_back(v);
    blstm_reorder_item a{};
    a.src = ptr(v);
    a.dst = out.back().data_ptr();
    a.outer = outer;
    a.inner_bytes = inner * e;
    a.row_stride = v.stride(dim) * e;
    a.outer_stride = outer_stride * e;
    items.push_back(a);
  }
  check(blstm_reorder(items.data(), (int)items.size(), ptr(parents), parents.scalar_type() == at::kLong ? 64 : 32, batch, beams < 1 ? 1 : beams, width,
                      call.stream),
        "reorder_states");
  return out;
}

// Tensors in (nested) lists and tuples, None among them, as one list; and one list in their place again.
void collect(PyObject* s, std::vector<Tensor>& flat) {
  if (THPVariable_Check(s)) flat.push_back(THPVariable_Unpack(s));
  else if (PyList_Check(s) || PyTuple_Check(s)) {
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(s);
    for (Py_ssize_t i = 0; i < n; ++i) collect(PySequence_Fast_GET_ITEM(s, i), flat);
  } else if (s != Py_None) {
    throw wrong(std::string("states must be tensors in lists or tuples, got ") + Py_TYPE(s)->tp_name);
  }
}
py::object rebuild(PyObject* s, const std::vector<Tensor>& flat, size_t& at) {
  if (THPVariable_Check(s)) return py::cast(flat[at++]);
  if (s == Py_None) return py::none();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(s);
  if (PyList_Check(s)) {
    py::list r(n);
    for (Py_ssize_t i = 0; i < n; ++i) r[i] = rebuild(PySequence_Fast_GET_ITEM(s, i), flat, at);
    return r;
  }
  py::tuple r(n);
  for (Py_ssize_t i = 0; i < n; ++i) r[i] = rebuild(PySequence_Fast_GET_ITEM(s, i), flat, at);
  return PyTuple_CheckExact(s) ? py::object(r) : py::reinterpret_borrow<py::object>((PyObject*)Py_TYPE(s))(*r);     // (a named tuple)
}

py::object reorder(const py::object& states, const Tensor& parents, int64_t dim) {
  std::vector<Tensor> flat;
  collect(states.ptr(), flat);
  const std::vector<Tensor> moved = reorder_flat(flat, parents, dim);
  size_t at = 0;
  return rebuild(states.ptr(), moved, at);
}

}  // namespace

namespace blstm_host {

void bind_beam(py::module_& m) {
  m.def("beam_step", &beam_step);
  m.def("reorder", &reorder);
}

}  // namespace blstm_host
