// The ordinary calls of the block norms and of what is kept in 8 bits, from torch's C++ side: contiguous tensors of the current device,
// and types and sizes that the kernels take.  A function returns None for anything else, and its caller in Python, which makes the same calls of
// tf24.h, copies and converts what can be and says what is wrong with the rest.
//
// In Python a call of residual_norm is 14 us and its backward pass 25 to 45 us of a thread that also has to wait for Python's lock, three to ten
// times what its kernels take for a few tokens.  Here it is a few allocations and the launches; the graph's node holds what the backward pass needs.
// The module belongs to the torch that it was built for (sparse/_native.py compares the versions); without it Python makes all calls.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include "tf24.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

void check(int rc) {
  if (rc) throw std::runtime_error(tf24_last_error());
}
int code_of(at::ScalarType t) { return t == at::kFloat ? TF24_F32 : t == at::kHalf ? TF24_F16 : t == at::kBFloat16 ? TF24_BF16 : -1; }
at::ScalarType type_of(int code) { return code == TF24_F32 ? at::kFloat : code == TF24_F16 ? at::kHalf : at::kBFloat16; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
Tensor make(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) { return at::empty(shape, like.options().dtype(type).requires_grad(false)); }
void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor or_none(const Maybe& t) { return t ? *t : Tensor(); }

// a strided tensor on a GPU, with nothing between a call and its storage
bool stored(const Tensor& t) {
  static const auto allowed = c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutocastCUDA});
  return t.is_cuda() && (t.key_set() | allowed) == allowed;
}
// one of floating-point numbers, contiguous and on the current device
bool plain(const Tensor& t) { return stored(t) && t.is_contiguous() && code_of(t.scalar_type()) >= 0 && t.get_device() == c10::hip::current_device(); }
bool wants_graph(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
[[noreturn]] void no_second_derivative(const char* what) { throw std::runtime_error(std::string("a graph of the gradients of ") + what + " is not supported"); }
// A gradient, or a saved tensor, as the kernels take it (undefined: zero, or none).  The engine looks at gradients, but not where a node is called by itself; a
// saved tensor is whatever its hook hands back.
Tensor as_it_was(const char* what, const Tensor& t, at::IntArrayRef shape, at::ScalarType type, c10::DeviceIndex device) {
  if (!t.defined()) return t;
  const Tensor plain = t.resolve_neg();
  if (!stored(plain) || plain.get_device() != device || plain.scalar_type() != type || plain.sizes() != shape)
    throw std::runtime_error(std::string(what) + " is not the one that was saved, or of its output: another shape, type or device");
  return plain.contiguous();
}
Tensor settled(const char* fn, const Tensor& g, at::IntArrayRef shape, at::ScalarType type, c10::DeviceIndex device) {
  if (!g.defined()) return g;
  return as_it_was(fn, g.scalar_type() == type ? g : g.to(type), shape, type, device);
}
int64_t blocks_of(int64_t cols) { return tf24_checkpoint_blocks(cols); }
std::pair<Tensor, Tensor> empty_checkpoint(int64_t rows, int64_t cols, const Tensor& like) {
  return {make({rows, 32 * blocks_of(cols)}, at::kFloat8_e4m3fn, like), make({rows, blocks_of(cols)}, at::kByte, like)};
}

// ---------------------------------------------------------------- block norms
struct NormCall {
  std::vector<int64_t> shape, gate_shape;
  int64_t rows, cols, rows_per_gate;
  at::ScalarType stream, block, param, gate;
  c10::DeviceIndex device;
  double scale;
  int post_kind, pre_kind;
  bool residual, has_n;
};

struct BlockNormBackward : public torch::autograd::Node {
  NormCall call;
  SavedVariable h, y, gate, post_weight, post_bias, pre_weight, stats;

  variable_list apply(variable_list&& grads) override {
    if (at::GradMode::is_enabled()) no_second_derivative("block_norm and residual_norm");
    std::lock_guard<std::mutex> lock(mutex_);
    const char* fn = "block_norm and residual_norm: a gradient or saved tensor";
    // of out (a call with y has one) and of n
    Tensor dout = call.residual ? grads[0] : Tensor(), dn = call.has_n ? grads[call.residual ? 1 : 0] : Tensor();
    variable_list result(7);
    if (!dout.defined() && !dn.defined()) return result;
    dout = settled(fn, dout, call.shape, call.stream, call.device);
    dn = settled(fn, dn, call.shape, call.block, call.device);
    const Tensor like = dn.defined() ? dn : dout;
    const int pre_kind = dn.defined() ? call.pre_kind : 0, post_kind = call.post_kind;
    auto saved = [&](const Tensor& t, at::IntArrayRef shape, at::ScalarType type) { return as_it_was(fn, t, shape, type, call.device); };
    const Tensor h_ = saved(h.unpack(call.residual ? shared_from_this() : nullptr), call.shape, call.stream), y_ = saved(y.unpack(), call.shape, call.block),
                 gate_ = saved(gate.unpack(), call.gate_shape, call.gate), post_weight_ = saved(post_weight.unpack(), {call.cols}, call.param),
                 post_bias_ = saved(post_bias.unpack(), {call.cols}, call.param), pre_weight_ = saved(pre_weight.unpack(), {call.cols}, call.param),
                 stats_ = saved(stats.unpack(), {4, call.rows}, at::kFloat);
    auto wanted = [&](int i) { return task_should_compute_output(i); };
    auto zeros_of = [&](at::IntArrayRef shape, at::ScalarType type) { return call.rows ? make(shape, type, like) : at::zeros(shape, like.options().dtype(type)); };
    if (wanted(0)) result[0] = make(call.shape, call.stream, like);
    if (wanted(1)) result[1] = make(call.shape, call.block, like);
    if (wanted(2)) result[2] = zeros_of(gate_.sizes(), gate_.scalar_type());
    for (int i = 3; i < 7; i++)
      if (wanted(i) && (i < 5 ? post_kind : pre_kind)) result[i] = zeros_of({call.cols}, call.param);
    if (!call.rows) return result;
    Tensor workspace;
    int64_t bytes = 0;
    if (result[2].defined() || result[3].defined() || result[4].defined() || result[5].defined() || result[6].defined()) {
      bytes = tf24_block_norm_backward_workspace_bytes(call.rows, call.cols, gate_.defined() ? call.rows_per_gate : call.rows);
      workspace = make({bytes}, at::kByte, like);
    }
    check(tf24_block_norm_backward(pointer(dout), call.cols, pointer(dn), call.cols, pre_kind ? pointer(h_) : nullptr, call.cols, pointer(y_), call.cols, code_of(call.stream),
                                   code_of(call.block), call.rows, call.cols, pointer(gate_), gate_.defined() ? code_of(gate_.scalar_type()) : TF24_F32, call.cols,
                                   call.rows_per_gate, pointer(post_weight_), pointer(post_bias_), pointer(pre_weight_), code_of(call.param), post_kind, pre_kind, call.residual,
                                   (float)call.scale, (const float*)pointer(stats_), pointer(result[0]), pointer(result[1]), pointer(result[2]), pointer(result[3]),
                                   pointer(result[4]), pointer(result[5]), pointer(result[6]), pointer(workspace), bytes, stream_of(like)));
    return result;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&h, &y, &gate, &post_weight, &post_bias, &pre_weight, &stats}) v->reset_data();
  }
  std::string name() const override { return "BlockNormBackward"; }
};

// (out, n, values, scales), None for what is not formed; None for a call that is Python's
py::object block_norm(const Tensor& x, const Maybe& y_in, const Maybe& gate_in, const Maybe& post_weight_in, const Maybe& post_bias_in, const Maybe& pre_weight_in,
                      const Maybe& pre_bias_in, double scale, int post_kind, int pre_kind, double eps, int block_code, bool keep) {
  const Tensor y = or_none(y_in), gate = or_none(gate_in), post_weight = or_none(post_weight_in), post_bias = or_none(post_bias_in), pre_weight = or_none(pre_weight_in),
               pre_bias = or_none(pre_bias_in);
  NormCall call;
  if (!plain(x) || x.dim() == 0) return py::none();
  call.shape = x.sizes().vec();
  call.cols = x.size(-1);
  if (call.cols < 1 || call.cols > 16384) return py::none();
  call.rows = x.numel() / call.cols;
  call.stream = x.scalar_type();
  call.residual = y.defined();
  if (call.residual && (!plain(y) || y.sizes() != x.sizes())) return py::none();
  if (!call.residual && (block_code < TF24_F32 || block_code > TF24_BF16)) return py::none();
  call.block = call.residual ? y.scalar_type() : type_of(block_code);
  if (call.stream != at::kFloat && call.block != call.stream) return py::none();
  call.param = at::kFloat;
  bool first = true;
  for (const Tensor* p : {&post_weight, &post_bias, &pre_weight, &pre_bias}) {
    if (!p->defined()) continue;
    if (!plain(*p) || p->dim() != 1 || p->size(0) != call.cols || (!first && p->scalar_type() != call.param)) return py::none();
    call.param = p->scalar_type();
    first = false;
  }
  call.rows_per_gate = 1;
  if (gate.defined()) {                                          // one for all rows, or for leading dimensions of y (then ones)
    if (!plain(gate) || gate.dim() == 0 || gate.size(-1) != call.cols) return py::none();
    if (gate.dim() == 1) call.rows_per_gate = call.rows;
    else {
      if (gate.dim() != y.dim()) return py::none();
      int64_t shared = gate.dim() - 1;
      while (shared && gate.size(shared - 1) == 1) call.rows_per_gate *= y.size(--shared);
      for (int64_t i = 0; i < shared; i++)
        if (gate.size(i) != y.size(i)) return py::none();
    }
  }
  if (gate.defined()) {
    call.gate_shape = gate.sizes().vec();
    call.gate = gate.scalar_type();
  }
  call.device = x.get_device();
  call.scale = scale;
  call.post_kind = post_kind;
  call.pre_kind = pre_kind;
  call.has_n = pre_kind != 0;

  const bool graph = wants_graph({&x, &y, &gate, &post_weight, &post_bias, &pre_weight, &pre_bias});
  Tensor out, n, values, scales, stats;
  if (call.residual) out = make(call.shape, call.stream, x);
  if (call.has_n) {
    n = make(call.shape, call.block, x);
    if (keep) std::tie(values, scales) = empty_checkpoint(call.rows, call.cols, x);
  }
  if (graph && (post_kind || pre_kind)) stats = make({4, call.rows}, at::kFloat, x);
  check(tf24_block_norm_forward(pointer(x), call.cols, pointer(y), call.cols, code_of(call.stream), code_of(call.block), call.rows, call.cols, pointer(gate),
                                gate.defined() ? code_of(gate.scalar_type()) : TF24_F32, call.cols, call.rows_per_gate, pointer(post_weight), pointer(post_bias),
                                pointer(pre_weight), pointer(pre_bias), code_of(call.param), post_kind, pre_kind, (float)scale, (float)eps, pointer(out), pointer(n),
                                (float*)pointer(stats), pointer(values), pointer(scales), stream_of(x)));
  if (graph) {
    auto node = std::shared_ptr<BlockNormBackward>(new BlockNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, y, gate, post_weight, post_bias, pre_weight, pre_bias));
    if (out.defined()) torch::autograd::set_history(out, node);
    if (n.defined()) torch::autograd::set_history(n, node);
    if (pre_kind) node->h = call.residual ? SavedVariable(out, true) : SavedVariable(x, false);
    if (y.defined() && (post_kind || (gate.defined() && gate.requires_grad()))) node->y = SavedVariable(y, false);
    if (gate.defined()) node->gate = SavedVariable(gate, false);
    if (post_weight.defined()) node->post_weight = SavedVariable(post_weight, false);
    if (post_bias.defined()) node->post_bias = SavedVariable(post_bias, false);
    if (pre_weight.defined()) node->pre_weight = SavedVariable(pre_weight, false);
    if (stats.defined()) node->stats = SavedVariable(stats, false);
    node->call = std::move(call);
  }
  auto or_python_none = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
  return py::make_tuple(or_python_none(out), or_python_none(n), or_python_none(values), or_python_none(scales));
}

// ---------------------------------------------------------------- the gated activation
struct GeluGluBackward : public torch::autograd::Node {
  std::vector<int64_t> shape;
  at::ScalarType type;
  c10::DeviceIndex device;
  SavedVariable values, scales;

  variable_list apply(variable_list&& grads) override {
    if (at::GradMode::is_enabled()) no_second_derivative("gelu_glu_checkpoint");
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor()};
    const char* fn = "gelu_glu_checkpoint: a gradient or saved tensor";
    const int64_t cols = shape.back(), rows = c10::multiply_integers(shape) / cols, blocks = blocks_of(cols / 2);
    auto out_shape = shape;
    out_shape.back() = cols / 2;
    const Tensor go = settled(fn, grads[0], out_shape, type, device), v = as_it_was(fn, values.unpack(), {2 * rows, 32 * blocks}, at::kFloat8_e4m3fn, device),
                 s = as_it_was(fn, scales.unpack(), {2 * rows, blocks}, at::kByte, device);
    const Tensor result = make(shape, type, go);
    check(tf24_gelu_glu_backward_checkpoint(pointer(go), cols / 2, pointer(v), pointer(s), code_of(type), rows, cols, pointer(result), cols, stream_of(go)));
    return {result};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    values.reset_data();
    scales.reset_data();
  }
  std::string name() const override { return "GeluGluBackward"; }
};

// out, or with keep_output (out, values, scales); None for a call that is Python's
py::object gelu_glu_checkpoint(const Tensor& x, bool keep_output) {
  if (!plain(x) || x.dim() == 0 || x.size(-1) == 0 || x.size(-1) % 2) return py::none();
  const int64_t cols = x.size(-1), half = cols / 2, rows = x.numel() / cols;
  auto shape = x.sizes().vec();
  shape.back() = half;
  Tensor out = make(shape, x.scalar_type(), x), values, scales, out_values, out_scales;
  const bool graph = wants_graph({&x});
  if (graph) std::tie(values, scales) = empty_checkpoint(2 * rows, half, x);
  if (keep_output) std::tie(out_values, out_scales) = empty_checkpoint(rows, half, x);
  check(tf24_gelu_glu_forward_checkpoint(pointer(x), code_of(x.scalar_type()), cols, rows, cols, pointer(out), half, pointer(values), pointer(scales), pointer(out_values),
                                         pointer(out_scales), stream_of(x)));
  if (graph) {
    auto node = std::shared_ptr<GeluGluBackward>(new GeluGluBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    torch::autograd::set_history(out, node);
    node->values = SavedVariable(values, false);
    node->scales = SavedVariable(scales, false);
    node->shape = x.sizes().vec();
    node->type = x.scalar_type();
    node->device = x.get_device();
  }
  if (!keep_output) return py::cast(out);
  return py::make_tuple(out, out_values, out_scales);
}

// ---------------------------------------------------------------- activations in 8 bits
py::object checkpoint_encode(const Tensor& x) {
  if (!plain(x) || x.dim() == 0 || x.size(-1) == 0) return py::none();
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  const auto [values, scales] = empty_checkpoint(rows, cols, x);
  check(tf24_checkpoint_encode(pointer(x), code_of(x.scalar_type()), cols, rows, cols, pointer(values), pointer(scales), stream_of(x)));
  return py::make_tuple(values, scales);
}

// what is kept of `rows` rows of `cols` columns, as it was made
bool holds(const Tensor& values, const Tensor& scales, int64_t rows, int64_t cols) {
  return values.dim() == 2 && scales.dim() == 2 && values.size(0) == rows && scales.size(0) == rows && values.size(1) == 32 * blocks_of(cols) &&
         scales.size(1) == blocks_of(cols) && values.is_contiguous() && scales.is_contiguous() && values.scalar_type() == at::kFloat8_e4m3fn &&
         scales.scalar_type() == at::kByte && values.is_cuda() && scales.is_cuda() && values.get_device() == scales.get_device() &&
         values.get_device() == c10::hip::current_device();
}

py::object checkpoint_decode(const Tensor& values, const Tensor& scales, const std::vector<int64_t>& shape, int code) {
  if (shape.empty() || shape.back() < 1) return py::none();
  int64_t rows = 1;
  for (size_t i = 0; i + 1 < shape.size(); i++) rows *= shape[i];
  if (!holds(values, scales, rows, shape.back())) return py::none();
  const Tensor out = make(shape, type_of(code), values);
  check(tf24_checkpoint_decode(pointer(values), pointer(scales), values.size(0), shape.back(), pointer(out), code, shape.back(), stream_of(values)));
  return py::cast(out);
}

// (dW, db or None), of arguments that checkpoint_weight_gradient has looked at; None for a call that is Python's
py::object checkpoint_weight_grad(const Tensor& g, const Tensor& values, const Tensor& scales, int64_t n, bool bias, int out_code) {
  if (!plain(g) || g.size(-1) == 0 || g.size(-1) % 8 || (uintptr_t)g.data_ptr() % 16) return py::none();
  const int64_t m = g.size(-1), tokens = g.numel() / m;
  if (tokens == 0 || !holds(values, scales, tokens, n)) return py::none();
  Tensor dw = make({m, n}, type_of(out_code), g), db, workspace;
  if (bias) db = make({m}, type_of(out_code), g);
  const int64_t bytes = tf24_checkpoint_weight_grad_workspace_bytes(tokens, m, n);
  if (bytes) workspace = make({bytes}, at::kByte, g);
  check(tf24_checkpoint_weight_grad(pointer(g), m, code_of(g.scalar_type()), pointer(values), pointer(scales), tokens, m, n, pointer(dw), pointer(db), out_code, pointer(workspace),
                                    bytes, stream_of(g)));
  return py::make_tuple(dw, db.defined() ? py::cast(db) : py::none());
}

}  // namespace

PYBIND11_MODULE(_torchcall, m) {
  m.attr("built_for") = TF24_TORCH_VERSION;
  m.def("block_norm", &block_norm);
  m.def("gelu_glu_checkpoint", &gelu_glu_checkpoint);
  m.def("checkpoint_encode", &checkpoint_encode);
  m.def("checkpoint_decode", &checkpoint_decode);
  m.def("checkpoint_weight_grad", &checkpoint_weight_grad);
}
