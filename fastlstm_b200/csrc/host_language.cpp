// Host side of the operators around a language model: argument checks, buffers, the calls of the C ABI and the autograd
// nodes.  Tensors keep their strides as long as two strides describe their rows and the last dimension is dense; others
// are copied first.
#include <ATen/cuda/EmptyTensor.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <cmath>

#include "host.h"

namespace {

using namespace blstm_host;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

py::value_error wrong(const std::string& what) { return py::value_error(what); }

void on_gpu(const Tensor& t, const char* name) {
  if (!t.is_cuda()) throw wrong(std::string(name) + " must be a CUDA tensor (there is no CPU path)");
}
void beside(const Tensor& t, const char* name, const Tensor& other) {
  on_gpu(t, name);
  if (t.device() != other.device()) throw wrong(std::string(name) + " is on " + t.device().str() + ", expected " + other.device().str());
}
int token_bits(const Tensor& tokens) {
  if (tokens.scalar_type() == at::kLong) return 64;
  if (tokens.scalar_type() == at::kInt) return 32;
  throw wrong(std::string("tokens have dtype ") + c10::toString(tokens.scalar_type()) + ", expected int64 or int32");
}

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
    Tensor v = dims > 2 ? t.flatten(0, dims - 1) : t;
    const int64_t lead = dims > 2 ? 1 : dims;
    if (v.dim() > lead && v.size(-1) > 1 && v.stride(-1) != 1) v = v.contiguous();
    stride[0] = lead == 2 ? v.stride(0) : 0;
    stride[1] = lead == 0 ? 0 : v.stride(lead - 1);
    return v;
  }
};

Tensor fresh(at::IntArrayRef sizes, at::ScalarType dt, const Tensor& like) { return at::detail::empty_cuda(sizes, dt, like.device(), std::nullopt); }

// A node of the graph that an operator's gradient is, with what it needs as members (a torch::autograd::Function keeps that in a
// dictionary: 4 us a call).  Backward goes through it once.
template <typename N>
std::shared_ptr<N> make_node(const Tensor& input) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(input));
  return node;
}

bool wants_grad(const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), "fastlstm_b200: forward-mode gradients are not there for this operator");
  return at::GradMode::is_enabled() && t.requires_grad();
}
void only_once() { TORCH_CHECK(!at::GradMode::is_enabled(), "fastlstm_b200: gradients of gradients (create_graph) are not there for this operator"); }

std::vector<int64_t> plus(at::IntArrayRef s, int64_t last) {
  std::vector<int64_t> v = s.vec();
  v.push_back(last);
  return v;
}

// ---------------------------------------------------------------- embedding
blstm_embed_desc embed_desc(at::ScalarType dt, const Tensor& tokens, const Lead& lead, int64_t V, int64_t D, double scale, int64_t padding) {
  blstm_embed_desc d{};
  d.dtype = dtype_code(dt);
  d.token_bits = token_bits(tokens);
  d.n0 = lead.n0; d.n1 = lead.n1;
  d.vocab = V; d.width = D;
  d.padding = padding;
  d.scale = (float)scale;
  return d;
}

Tensor embedding_impl(const Tensor& tokens_in, const Tensor& weight_in, double scale) {
  const Lead lead(tokens_in.sizes());
  const Tensor weight = weight_in.size(1) > 1 && weight_in.stride(1) != 1 ? weight_in.contiguous() : weight_in;
  blstm_embed_desc d = embed_desc(weight.scalar_type(), tokens_in, lead, weight.size(0), weight.size(1), scale, -1);
  const Tensor tokens = lead.rows(tokens_in, d.token_stride);
  d.row_stride[0] = weight.stride(0);
  Call call(weight.device());
  const Tensor out = fresh(plus(tokens_in.sizes(), weight.size(1)), weight.scalar_type(), weight);
  check(blstm_embedding(&d, ptr(tokens), ptr(weight), out.data_ptr(), call.stream), "embedding");
  return out;
}

struct EmbeddingGrad : public Node {
  SavedVariable tokens;
  at::ScalarType dtype;
  int64_t vocab, width, padding;
  double scale;
  void release_variables() override { tokens.reset_data(); }
  variable_list apply(variable_list&& g) override {
    only_once();
    if (!g[0].defined()) return {Tensor()};
    const Tensor saved = tokens.unpack();
    const Lead lead(saved.sizes());
    blstm_embed_desc d = embed_desc(dtype, saved, lead, vocab, width, scale, padding);
    const Tensor tokens = lead.rows(saved, d.token_stride), dout = lead.rows(g[0], d.row_stride);
    Call call(dout.device());
    const Tensor dW = fresh({vocab, width}, dtype, dout);
    const size_t bytes = blstm_embedding_grad_workspace(&d);
    Tensor ws;
    if (bytes) ws = fresh({(int64_t)bytes}, at::kByte, dout);
    check(blstm_embedding_grad(&d, ptr(tokens), ptr(dout), dW.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes, call.stream), "embedding gradient");
    return {dW};
  }
};

Tensor embedding(const Tensor& tokens, const Tensor& weight, double scale, std::optional<int64_t> padding_idx) {
  py::gil_scoped_release nogil;
  on_gpu(weight, "weight");
  dtype_code(weight.scalar_type());
  if (weight.dim() != 2 || weight.size(0) == 0 || weight.size(1) == 0) throw wrong("expected weight as [vocabulary, width], got " + shape_str(weight.sizes()));
  beside(tokens, "tokens", weight);
  token_bits(tokens);
  if (!std::isfinite((float)scale)) throw wrong("scale must be finite in 32 bits");
  const int64_t V = weight.size(0);
  int64_t padding = -1;
  if (padding_idx) {
    if (*padding_idx < -V || *padding_idx >= V) throw wrong("padding_idx " + std::to_string(*padding_idx) + " is outside of the vocabulary of " + std::to_string(V));
    padding = *padding_idx < 0 ? *padding_idx + V : *padding_idx;
  }
  if (!wants_grad(weight)) return embedding_impl(tokens, weight, scale);
  const auto node = make_node<EmbeddingGrad>(weight);
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    out = embedding_impl(tokens, weight, scale);
  }
  node->tokens = SavedVariable(tokens, false);
  node->dtype = weight.scalar_type();
  node->vocab = V; node->width = weight.size(1); node->padding = padding;
  node->scale = scale;
  torch::autograd::set_history(out, node);
  return out;
}

// ---------------------------------------------------------------- dropout
struct Mask {
  double p = 0;
  uint64_t seed = 0, offset = 0;
  int64_t shared = -1;        // dimension, or -1
  bool on_gpu = false;        // the seed
  Tensor seed_at;
};

Tensor dropout_impl(const Tensor& x_in, const Mask& k) {
  const auto sizes = x_in.sizes();
  const int64_t dims = x_in.dim();
  blstm_dropout_desc d{};
  d.dtype = dtype_code(x_in.scalar_type());
  d.shared = -1;
  d.p = k.p; d.seed = k.seed; d.offset = k.offset;
  d.n0 = d.n1 = 1;
  Tensor x = x_in;
  if (k.shared < 0 && dims > 3 && !x.is_contiguous()) x = x.flatten(0, dims - 2);     // (a copy where one stride does not do)
  const bool two = (x.dim() == 2 || x.dim() == 3) && !x.is_contiguous() && x.stride(-1) == 1 && x.numel() / x.size(-1) <= INT32_MAX;
  if (!two) x = x.contiguous();
  if (two) {                              // rows with strides of their own
    const bool three = x.dim() == 3;
    if (three) { d.n0 = x.size(0); d.stride[0] = x.stride(0); }
    d.n1 = x.size(-2); d.stride[1] = x.stride(-2);
    d.cols = x.size(-1);
    d.shared = k.shared < 0 ? -1 : three ? (int32_t)k.shared : 1;
  } else if (k.shared < 0) {              // one row
    d.cols = x.numel();
  } else {
    for (int64_t i = 0; i < k.shared; ++i) d.n0 *= sizes[i];
    d.n1 = sizes[k.shared];
    d.cols = 1;
    for (int64_t i = k.shared + 1; i < dims; ++i) d.cols *= sizes[i];
    d.stride[0] = d.n1 * d.cols; d.stride[1] = d.cols;
    d.shared = 1;
    if (d.n0 > 0 && d.n1 > INT32_MAX / d.n0) throw wrong("more than 2^31 - 1 rows that share masks");
  }
  Call call(x.device());
  const Tensor y = fresh(sizes, x.scalar_type(), x);
  check(blstm_dropout(&d, ptr(x), k.on_gpu ? static_cast<const int64_t*>(ptr(k.seed_at)) : nullptr, y.data_ptr(), call.stream), "dropout");
  return y;
}

struct DropoutGrad : public Node {
  Mask mask;
  SavedVariable seed_at;
  void release_variables() override { seed_at.reset_data(); }
  variable_list apply(variable_list&& g) override {
    only_once();
    if (!g[0].defined()) return {Tensor()};
    Mask k = mask;
    if (k.on_gpu) k.seed_at = seed_at.unpack();
    return {dropout_impl(g[0], k)};
  }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, const OptTensor& seed_at, uint64_t offset, std::optional<int64_t> shared_dim) {
  py::gil_scoped_release nogil;
  on_gpu(x, "x");
  dtype_code(x.scalar_type());
  if (!(p >= 0.0 && p <= 1.0)) throw wrong("p must be in the range [0, 1]");
  Mask k;
  k.p = p; k.seed = seed; k.offset = offset;
  if (shared_dim) {
    const int64_t d = *shared_dim < 0 ? *shared_dim + x.dim() : *shared_dim;
    if (d < 0 || d >= x.dim() - 1) throw wrong("shared_dim must be a dimension of x and not its last one");
    k.shared = d;
  }
  if (seed_at) {
    beside(*seed_at, "seed", x);
    if (seed_at->scalar_type() != at::kLong || seed_at->numel() != 1) throw wrong("a seed on the GPU is one int64 element");
    k.on_gpu = true;
    k.seed_at = *seed_at;
  }
  if (!wants_grad(x)) return dropout_impl(x, k);
  const auto node = make_node<DropoutGrad>(x);
  Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    y = dropout_impl(x, k);
  }
  if (k.on_gpu) node->seed_at = SavedVariable(k.seed_at, false);
  k.seed_at.reset();
  node->mask = std::move(k);
  torch::autograd::set_history(y, node);
  return y;
}

// ---------------------------------------------------------------- log probabilities
struct Score {
  int64_t top = 0;
  double temperature = 1;
  int64_t ignore = -100;
};

blstm_score_desc score_desc(const Tensor& logits, const Tensor& tokens, const Lead& lead, const Score& c) {
  blstm_score_desc d{};
  d.dtype = dtype_code(logits.scalar_type());
  d.token_bits = token_bits(tokens);
  d.n0 = lead.n0; d.n1 = lead.n1;
  d.vocab = logits.size(-1);
  d.ignore = c.ignore;
  d.top = (int32_t)c.top;
  d.temperature = (float)c.temperature;
  return d;
}

// {log_probs, entropy, top_log_probs, top_tokens, stats}; the last one for a gradient alone
std::array<Tensor, 5> score_impl(const Tensor& logits_in, const Tensor& tokens_in, const Score& c, bool grad) {
  const Lead lead(tokens_in.sizes());
  blstm_score_desc d = score_desc(logits_in, tokens_in, lead, c);
  const Tensor logits = lead.rows(logits_in, d.logits_stride), tokens = lead.rows(tokens_in, d.token_stride);
  Call call(logits.device());
  std::array<Tensor, 5> r{fresh(tokens_in.sizes(), at::kFloat, logits), fresh(tokens_in.sizes(), at::kFloat, logits)};
  if (c.top) {
    r[2] = fresh(plus(tokens_in.sizes(), c.top), at::kFloat, logits);
    r[3] = fresh(plus(tokens_in.sizes(), c.top), at::kLong, logits);
  }
  if (grad) r[4] = fresh({3, lead.n0 * lead.n1}, at::kFloat, logits);
  check(blstm_token_log_probs(&d, ptr(logits), ptr(tokens), (float*)r[0].data_ptr(), (float*)r[1].data_ptr(), c.top ? (float*)r[2].data_ptr() : nullptr,
                              c.top ? (int64_t*)r[3].data_ptr() : nullptr, grad ? (float*)r[4].data_ptr() : nullptr, call.stream),
        "token_log_probs");
  return r;
}

// Memory for the gradient of logits [n0, n1, V] with rows on the same address modulo 16: laid out as the logits are where
// that wastes little, else with the shortest strides that are the same modulo 16 bytes.
Tensor grad_like(const Tensor& logits, const Lead& lead, const int64_t stride[2], int64_t dstride[2]) {
  const int64_t e = logits.element_size(), V = logits.size(-1), per = 16 / e;
  const int64_t own = V + (lead.n0 - 1) * stride[0] + (lead.n1 - 1) * stride[1];
  const bool inner0 = stride[0] < stride[1];          // the first dimension is the inner one in memory
  const int64_t n_in = inner0 ? lead.n0 : lead.n1, s_in = stride[inner0 ? 0 : 1], n_out = inner0 ? lead.n1 : lead.n0, s_out = stride[inner0 ? 1 : 0];
  const bool apart = (n_in == 1 || s_in >= V) && (n_out == 1 || s_out >= V + (n_in - 1) * s_in);   // no two rows share an element (windows do)
  const int64_t numel = lead.n0 * lead.n1 * V;
  if (apart && own <= numel + numel / 8) {
    dstride[0] = stride[0]; dstride[1] = stride[1];
  } else {
    auto at_least = [&](int64_t least, int64_t like) { return least + (((like - least) % per) + per) % per; };
    dstride[1] = at_least(V, stride[1]);
    dstride[0] = at_least(lead.n1 * dstride[1], stride[0]);
  }
  const int64_t shift = (reinterpret_cast<uintptr_t>(logits.const_data_ptr()) & 15) / e;
  const int64_t extent = V + (lead.n0 - 1) * dstride[0] + (lead.n1 - 1) * dstride[1];
  return fresh({extent + shift}, logits.scalar_type(), logits).as_strided({lead.n0, lead.n1, V}, {dstride[0], dstride[1], 1}, shift);
}

struct ScoreGrad : public Node {
  SavedVariable logits, tokens, stats, tops;
  Score c;
  void release_variables() override {
    for (SavedVariable* v : {&logits, &tokens, &stats, &tops}) v->reset_data();
  }
  variable_list apply(variable_list&& g) override {
    only_once();
    const Tensor z = logits.unpack(), at_tokens = tokens.unpack(), saved = stats.unpack();
    const Lead lead(at_tokens.sizes());
    blstm_score_desc d = score_desc(z, at_tokens, lead, c);
    const Tensor rows = lead.rows(z, d.logits_stride), given = lead.rows(at_tokens, d.token_stride);
    if (lead.n0 * lead.n1 == 0) return {at::zeros_like(z)};
    Call call(z.device());
    int64_t ds[2], s0[2], s1[2];
    const Tensor dl = grad_like(rows, lead, d.logits_stride, ds);
    const Tensor g0 = g[0].defined() ? lead.rows(g[0], s0) : Tensor(), g1 = g[1].defined() ? lead.rows(g[1], s1) : Tensor();
    Tensor g2, best;
    if (c.top) {
      best = tops.unpack();
      if (g[2].defined()) g2 = g[2].contiguous();
    }
    auto f32 = [](const Tensor& t) { return t.defined() ? static_cast<const float*>(t.const_data_ptr()) : nullptr; };
    check(blstm_token_log_probs_grad(&d, ptr(rows), ptr(given), f32(saved), c.top ? static_cast<const int64_t*>(ptr(best)) : nullptr, f32(g0), s0,
                                     f32(g1), s1, f32(g2), dl.data_ptr(), ds, call.stream),
          "token_log_probs gradient");
    return {lead.dims == 2 ? dl : dl.reshape(z.sizes())};
  }
};

py::tuple token_log_probs(const Tensor& logits, const Tensor& tokens, int64_t top, double temperature, int64_t ignore_index) {
  variable_list r(4);
  {
    py::gil_scoped_release nogil;
    on_gpu(logits, "logits");
    dtype_code(logits.scalar_type());
    if (logits.dim() < 1 || logits.size(-1) == 0) throw wrong("expected logits as [..., vocabulary], got " + shape_str(logits.sizes()));
    beside(tokens, "tokens", logits);
    token_bits(tokens);
    if (tokens.sizes() != logits.sizes().slice(0, logits.dim() - 1))
      throw wrong("tokens have shape " + shape_str(tokens.sizes()) + ", expected " + shape_str(logits.sizes().slice(0, logits.dim() - 1)));
    if (top < 0 || top > BLSTM_MAX_TOP || top > logits.size(-1))
      throw wrong("top must be between 0 and " + std::to_string(std::min<int64_t>(BLSTM_MAX_TOP, logits.size(-1))));
    if (!(temperature >= 1e-30 && std::isfinite((float)temperature))) throw wrong("temperature must be positive (at least 1e-30) and finite");
    const Score c{top, temperature, ignore_index};
    const bool grad = wants_grad(logits);
    const auto node = grad ? make_node<ScoreGrad>(logits) : nullptr;
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto v = score_impl(logits, tokens, c, grad);
    std::copy(v.begin(), v.begin() + 4, r.begin());
    if (grad) {
      node->logits = SavedVariable(logits, false);
      node->tokens = SavedVariable(tokens, false);
      node->stats = SavedVariable(v[4], false);
      node->c = c;
      torch::autograd::set_history(r[0], node);
      torch::autograd::set_history(r[1], node);
      if (top) {
        torch::autograd::set_history(r[2], node);
        node->tops = SavedVariable(r[3], false);
      }
    }
  }
  return py::make_tuple(r[0], r[1], top ? py::cast(r[2]) : py::none(), top ? py::cast(r[3]) : py::none());
}

}  // namespace

namespace blstm_host {

void bind_language(py::module_& m) {
  m.def("embedding", &embedding);
  m.def("dropout", &dropout);
  m.def("token_log_probs", &token_log_probs);
}

}  // namespace blstm_host
