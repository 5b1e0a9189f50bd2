// The torch side of the policy-network operators (include/goenv.h): argument checks, outputs and workspaces from torch's allocator,
// torch's current stream, and the gradients as nodes of torch's autograd.  elf_amd/policy_ops.py holds the documentation.
// In C++ because the backward pass of a small tensor costs more in Python (the engine's thread has to take the interpreter's
// lock) than its kernels take: a dropout of 255 x 722, forward and backward, took 97 us there and 46 here.  Every kernel is reached through the C-ABI.
#include <ATen/ATen.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cstring>
#include <optional>
#include <sstream>
#include <string>
#include <vector>

#include "../../include/goenv.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;   // (autograd's apply takes no undefined tensors)
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct OpError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw OpError(s.str());
}

void check_rc(int rc) {
  if (rc != 0) throw OpError(goenv_last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

bool is_float_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
int dtype_of(at::ScalarType t) { return t == at::kFloat ? GOENV_DT_F32 : t == at::kBFloat16 ? GOENV_DT_BF16 : GOENV_DT_F16; }

// ---- arguments ------------------------------------------------------------------------------------

// What a kernel, which sees memory and no more, would lose
void check_plain(const Tensor& t, const char* name) {
  if (t._fw_grad(/*level=*/0).defined()) refuse(name, " carries a forward-mode derivative: the policy-network operators have none");
  // (to a kernel an optional argument without memory is one that was left out)
  if (t.layout() == at::kStrided && (!t.has_storage() || (t.numel() > 0 && t.const_data_ptr() == nullptr)))
    refuse(name, " must have memory of its own (a plain tensor, not a wrapper or a placeholder of one)");
}

// A trace would record the outputs' allocation and not what fills them
void check_not_traced() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  if (torch::jit::tracer::isTracing() || Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE))
    refuse("the policy-network operators cannot be recorded in a trace");
}

Tensor main_tensor(py::handle h, const char* name) {
  if (!THPVariable_Check(h.ptr())) refuse(name, " must be a tensor on the GPU");
  const Tensor& t = THPVariable_Unpack(h.ptr());
  check_plain(t, name);
  if (!t.is_cuda() || t.layout() != at::kStrided) refuse(name, " must be a tensor on the GPU");
  if (!is_float_type(t.scalar_type())) refuse(name, " must be float32, bfloat16 or float16 (got ", t.scalar_type(), ")");
  return t.resolve_neg();   // (the imaginary part of a conjugate: its memory holds the values with the other sign)
}

Tensor optional_tensor(py::handle h, const char* name) {
  if (h.is_none()) return Tensor();
  if (!THPVariable_Check(h.ptr())) refuse(name, " must be a tensor (got ", py::str(py::type::handle_of(h)).cast<std::string>(), ")");
  const Tensor& t = THPVariable_Unpack(h.ptr());
  check_plain(t, name);
  return t.resolve_neg();
}

void check_like(const Tensor& t, const char* name, const Tensor& like, std::initializer_list<at::ScalarType> types, at::IntArrayRef shape) {
  const bool typed = std::find(types.begin(), types.end(), t.scalar_type()) != types.end();
  if (typed && t.layout() == at::kStrided && t.device() == like.device() && t.sizes() == shape) return;
  std::ostringstream s;
  const char* between = "";
  for (auto d : types) s << between << d, between = " or ";
  refuse(name, " must be a tensor of ", s.str(), " of shape ", shape, " on ", like.device(), " (got ", t.scalar_type(), " ", t.sizes(), " on ",
         t.device(), ")");
}

double number(py::handle h, const char* name) {
  if (PyBool_Check(h.ptr()) || (!PyFloat_Check(h.ptr()) && !PyLong_Check(h.ptr()))) refuse(name, " must be a number");
  return h.cast<double>();
}

// -1 for what is no whole number of 64 bits
int64_t whole(py::handle h) {
  if (PyBool_Check(h.ptr()) || !PyLong_Check(h.ptr())) return -1;
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(h.ptr(), &over);
  return over ? -1 : v;
}

// What torch's once_differentiable does: the gradients have no gradients
void once(variable_list& grads, const variable_list& given) {
  if (!at::GradMode::is_enabled()) return;
  variable_list from;
  for (const Tensor& t : given)
    if (t.defined() && t.requires_grad()) from.push_back(t);
  if (from.empty()) return;
  for (Tensor& t : grads) {
    if (!t.defined()) continue;
    auto fn = std::make_shared<torch::autograd::Error>("the policy-network operators are differentiable once",
                                                       torch::autograd::collect_next_edges(from));
    t = t.detach();
    torch::autograd::set_history(t, fn);
  }
}

Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor tensor_of(const Maybe& t) { return t ? *t : Tensor(); }

// Whether the node's tensor arguments want gradients; autograd counts the arguments that are there
struct Needs {
  AutogradContext* ctx;
  size_t edge = 0;
  bool operator()(const Tensor& t) { return t.defined() && ctx->needs_input_grad(edge++); }
};

// A leaf's gradients are accumulated on the stream where its first graph that still lives was made.  If that is the default
// stream, which no capture can take in, the backward pass of a graph under capture makes it wait for the capture: torch
// ends the process.  So such a call is refused.
void check_capture(const Tensor& t) {
  if (!t.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return;
  const auto made = node->stream();
  const auto now = c10::hip::getCurrentHIPStream(t.device().index()), eager = c10::hip::getDefaultHIPStream(t.device().index());
  if (made && made->id() == eager.id() && now != eager && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
    refuse("a graph made outside the capture still lives and shares a leaf with this call: delete what it returned, or capture with leaves of its own");
}

bool wants_grad(std::initializer_list<Tensor> all) {
  if (!at::GradMode::is_enabled()) return false;
  bool wants = false;
  for (const Tensor& t : all)
    if (t.defined() && t.requires_grad()) {
      check_capture(t);
      wants = true;
    }
  return wants;
}

// ---- group norm -----------------------------------------------------------------------------------

struct Layout {
  bool ok;
  int64_t sample, position;
};
// Of a channels-last [n, c, *positions] tensor
Layout layout_of(const Tensor& t) {
  const auto shape = t.sizes(), stride = t.strides();
  Layout l{false, 0, 0};
  if (shape[1] != 1 && stride[1] != 1) return l;
  int64_t want = 0;
  bool any = false;
  for (int64_t d = (int64_t)shape.size() - 1; d >= 2; --d) {
    if (shape[d] == 1) continue;
    if (!any) l.position = stride[d];
    else if (stride[d] != want) return l;
    any = true;
    want = stride[d] * shape[d];
  }
  if (shape[0] != 1) l.sample = stride[0];
  l.ok = true;
  return l;
}

Tensor dense_like(const Tensor& t) {
  const auto shape = t.sizes();
  c10::SmallVector<int64_t, 6> stride(shape.size());
  int64_t step = shape[1];
  stride[1] = 1;
  for (int64_t d = (int64_t)shape.size() - 1; d >= 2; --d) {
    stride[d] = step;
    step *= std::max<int64_t>(shape[d], 1);
  }
  stride[0] = step;
  return at::empty_strided(shape, stride, t.options());
}

struct NormHow {
  int64_t groups;
  float eps, slope;
  int act;
};

goenv_norm norm_args(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias, const NormHow& how, const Tensor& stats) {
  goenv_norm p = {};
  p.device = x.device().index();
  p.dtype = dtype_of(x.scalar_type());
  p.act = how.act;
  p.n = x.size(0);
  p.positions = 1;
  for (int64_t d = 2; d < x.dim(); ++d) p.positions *= x.size(d);
  p.channels = (int32_t)x.size(1);
  p.groups = (int32_t)how.groups;
  p.eps = how.eps;
  p.slope = how.slope;
  p.x = x.data_ptr();
  Layout l = layout_of(x);
  p.x_sample = l.sample;
  p.x_position = l.position;
  if (residual.defined()) {
    l = layout_of(residual);
    p.residual = residual.data_ptr();
    p.r_sample = l.sample;
    p.r_position = l.position;
  }
  if (weight.defined()) {
    p.weight = weight.data_ptr();
    p.param_dtype = dtype_of(weight.scalar_type());
  }
  if (bias.defined()) {
    p.bias = bias.data_ptr();
    p.param_dtype = dtype_of(bias.scalar_type());
  }
  if (stats.defined()) p.stats = stats.data_ptr<float>();
  return p;
}

Tensor workspace_of(int64_t need, const Tensor& like) {
  return need > 0 ? at::empty({need}, like.options().dtype(at::kByte)) : Tensor();
}

Tensor norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias, const NormHow& how, const Tensor& stats) {
  Tensor y = dense_like(x);
  goenv_norm p = norm_args(x, residual, weight, bias, how, stats);
  const int64_t need = goenv_group_norm_workspace(p.n, p.positions, p.channels, p.groups, p.dtype, 0);
  const Tensor ws = workspace_of(need, x);
  if (need > 0) p.workspace = ws.data_ptr(), p.workspace_bytes = need;
  check_rc(goenv_group_norm_act(&p, y.data_ptr(), stream_of(x)));
  return y;
}

struct NormNode : torch::autograd::Function<NormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& r, const Maybe& w, const Maybe& b, const NormHow& how) {
    const Tensor residual = tensor_of(r), weight = tensor_of(w), bias = tensor_of(b);
    const Tensor stats = at::empty({x.size(0), how.groups, 2}, x.options().dtype(at::kFloat));
    Tensor y = norm_forward(x, residual, weight, bias, how, stats);
    ctx->save_for_backward({x, residual, weight, bias, stats});
    ctx->saved_data["groups"] = how.groups;
    ctx->saved_data["act"] = (int64_t)how.act;
    ctx->saved_data["eps"] = (double)how.eps;
    ctx->saved_data["slope"] = (double)how.slope;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_plain(grads[0], "the gradient");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &residual = saved[1], &weight = saved[2], &bias = saved[3];
    const NormHow how{ctx->saved_data["groups"].toInt(), (float)ctx->saved_data["eps"].toDouble(), (float)ctx->saved_data["slope"].toDouble(),
                      (int)ctx->saved_data["act"].toInt()};
    variable_list out(5);
    {
      at::NoGradGuard no_grad;
      Tensor dy = grads[0].resolve_neg();
      Layout l = layout_of(dy);
      if (!l.ok) {
        dy = dense_like(dy).copy_(dy);
        l = layout_of(dy);
      }
      Needs needs{ctx};
      if (needs(x)) out[0] = dense_like(x);
      if (needs(residual)) out[1] = dense_like(x);
      if (needs(weight)) out[2] = at::empty_like(weight);
      if (needs(bias)) out[3] = at::empty_like(bias);
      goenv_norm p = norm_args(x, residual, weight, bias, how, saved[4]);
      const int64_t need = goenv_group_norm_workspace(p.n, p.positions, p.channels, p.groups, p.dtype, 1);
      const Tensor ws = workspace_of(need, x);
      if (need > 0) p.workspace = ws.data_ptr(), p.workspace_bytes = need;
      auto at = [&](int i) { return out[i].defined() ? out[i].data_ptr() : nullptr; };
      check_rc(goenv_group_norm_act_grad(&p, dy.data_ptr(), l.sample, l.position, at(0), at(1), at(2), at(3), stream_of(x)));
    }
    once(out, {x, residual, weight, bias, grads[0]});
    return out;
  }
};

Tensor group_norm_act(py::handle px, py::handle pgroups, py::handle pweight, py::handle pbias, py::handle peps, const std::string& act, py::handle pslope,
                      py::handle presidual) {
  check_not_traced();
  const Tensor x = main_tensor(px, "x");
  if (x.dim() < 2) refuse("x must be [n, c, *positions] (got ", x.sizes(), ")");
  if (!layout_of(x).ok)
    refuse("x must be channels last (x.to(memory_format=torch.channels_last)); got shape ", x.sizes(), ", strides ", x.strides());
  const int64_t c = x.size(1);
  NormHow how;
  how.groups = whole(pgroups);
  if (how.groups <= 0 || how.groups > INT32_MAX || c > INT32_MAX || c % how.groups)
    refuse("num_groups must be a positive integer that divides the ", c, " channels");
  static const char* const names[] = {"none", "relu", "leaky_relu", "silu"};
  how.act = 0;
  while (how.act < 4 && act != names[how.act]) ++how.act;
  if (how.act == 4) refuse("act must be one of none, relu, leaky_relu, silu (got ", act, ")");
  how.eps = (float)number(peps, "eps");
  how.slope = (float)number(pslope, "slope");
  const Tensor residual = optional_tensor(presidual, "residual"), weight = optional_tensor(pweight, "weight"), bias = optional_tensor(pbias, "bias");
  if (residual.defined()) {
    check_like(residual, "residual", x, {x.scalar_type()}, x.sizes());
    if (!layout_of(residual).ok) refuse("residual must be channels last, as x");
  }
  for (const auto& [t, name] : {std::make_pair(&weight, "weight"), std::make_pair(&bias, "bias")}) {
    if (!t->defined()) continue;
    check_like(*t, name, x, {at::kFloat, x.scalar_type()}, {c});
    if (!t->is_contiguous()) refuse(name, " must be contiguous");
  }
  if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type())
    refuse("weight and bias must be of one type (got ", weight.scalar_type(), " and ", bias.scalar_type(), ")");
  if (wants_grad({x, residual, weight, bias})) return NormNode::apply(x, maybe(residual), maybe(weight), maybe(bias), how);
  return norm_forward(x, residual, weight, bias, how, Tensor());
}

// ---- dropout --------------------------------------------------------------------------------------

// Whether t's elements fill its memory without gaps, in some order of the dimensions
bool is_dense(const Tensor& t) {
  if (t.is_contiguous()) return true;
  c10::SmallVector<std::pair<int64_t, int64_t>, 6> d;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) != 1) d.push_back({t.stride(i), t.size(i)});
  std::sort(d.begin(), d.end());
  int64_t want = 1;
  for (const auto& [stride, size] : d) {
    if (stride != want) return false;
    want *= size;
  }
  return true;
}

bool same_order(const Tensor& a, at::IntArrayRef stride) {
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) != 1 && a.stride(i) != stride[i]) return false;
  return true;
}

Tensor dropout_run(const Tensor& x, const Tensor& residual, double p, const Tensor& rng, int64_t site) {
  Tensor y = at::empty_strided(x.sizes(), x.strides(), x.options());
  check_rc(goenv_dropout(x.device().index(), dtype_of(x.scalar_type()), x.numel(), x.data_ptr(), residual.defined() ? residual.data_ptr() : nullptr,
                         y.data_ptr(), p, rng.data_ptr<int64_t>(), (uint32_t)site, stream_of(x)));
  return y;
}

struct DropoutHow {
  Tensor rng;
  double p;
  int64_t site;
};

struct DropoutNode : torch::autograd::Function<DropoutNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& r, const DropoutHow& how) {
    const Tensor residual = tensor_of(r);
    ctx->save_for_backward({how.rng});
    ctx->saved_data["p"] = how.p;
    ctx->saved_data["site"] = how.site;
    ctx->saved_data["stride"] = x.strides().vec();
    ctx->saved_data["residual"] = residual.defined();
    return dropout_run(x, residual, how.p, how.rng, how.site);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_plain(grads[0], "the gradient");
    const Tensor rng = ctx->get_saved_variables()[0];
    variable_list out(3);
    if (ctx->needs_input_grad(0)) {
      at::NoGradGuard no_grad;
      Tensor dy = grads[0].resolve_neg();
      const auto stride = ctx->saved_data["stride"].toIntVector();
      if (!same_order(dy, stride)) dy = at::empty_strided(dy.sizes(), stride, dy.options()).copy_(dy);
      out[0] = dropout_run(dy, Tensor(), ctx->saved_data["p"].toDouble(), rng, ctx->saved_data["site"].toInt());
    }
    once(out, {grads[0]});
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) out[1] = grads[0];
    return out;
  }
};

Tensor dropout(py::handle px, py::handle pp, py::handle prng, py::handle psite, py::handle presidual) {
  check_not_traced();
  const Tensor x = main_tensor(px, "x");
  if (!is_dense(x)) refuse("x must be dense (contiguous or channels last); got shape ", x.sizes(), ", strides ", x.strides());
  const double p = number(pp, "p must be a number from 0 to 1: it");
  if (!(p >= 0. && p <= 1.)) refuse("p must be a number from 0 to 1 (got ", p, ")");
  const int64_t site = whole(psite);
  if (site < 0 || site > (int64_t)UINT32_MAX) refuse("site must be an integer from 0 to 2^32 - 1");
  const Tensor rng = optional_tensor(prng, "rng"), residual = optional_tensor(presidual, "residual");
  if (!rng.defined()) refuse("rng must be a tensor of Long of shape [2] on ", x.device());
  check_like(rng, "rng", x, {at::kLong}, {2});
  if (!rng.is_contiguous()) refuse("rng must be contiguous");
  if (residual.defined()) {
    check_like(residual, "residual", x, {x.scalar_type()}, x.sizes());
    if (!same_order(residual, x.strides())) refuse("residual must have x's strides (got ", residual.strides(), " and ", x.strides(), ")");
  }
  if (wants_grad({x, residual})) return DropoutNode::apply(x, maybe(residual), DropoutHow{rng, p, site});
  return dropout_run(x, residual, p, rng, site);
}

// ---- policy logits --------------------------------------------------------------------------------

struct LogitHow {
  Tensor legal, legal_bits, history, history_len, row[4];   // rows' repetition, presence, frequency, temperature
  float scalar[4];
  int out_kind;
  at::ScalarType out_type;
};

goenv_logit_rules logit_args(const Tensor& logits, const Tensor& bias, const LogitHow& how) {
  goenv_logit_rules p = {};
  p.device = logits.device().index();
  p.dtype = dtype_of(logits.scalar_type());
  p.out_dtype = dtype_of(how.out_type);
  p.out_kind = how.out_kind;
  p.rows = logits.size(0);
  p.cols = logits.size(1);
  p.logits = logits.data_ptr();
  p.logits_row = logits.stride(0);
  if (how.legal.defined()) {
    p.legal = static_cast<const uint8_t*>(how.legal.data_ptr());
    p.legal_row = how.legal.stride(0);
  }
  if (how.legal_bits.defined()) {
    p.legal_bits = static_cast<const uint32_t*>(how.legal_bits.data_ptr());
    p.bits_row = how.legal_bits.stride(0);
  }
  if (bias.defined()) {
    p.bias = bias.data_ptr();
    p.bias_dtype = dtype_of(bias.scalar_type());
    p.bias_row = bias.dim() == 1 ? 0 : bias.size(1);
  }
  if (how.history.defined()) {
    p.history = how.history.data_ptr();
    p.history_row = how.history.stride(0);
    p.history_max = (int32_t)how.history.size(1);
    p.history_i64 = how.history.scalar_type() == at::kLong;
    if (how.history_len.defined()) p.history_len = how.history_len.data_ptr<int32_t>();
  }
  p.repetition = how.scalar[0];
  p.presence = how.scalar[1];
  p.frequency = how.scalar[2];
  p.temperature = how.scalar[3];
  const float** rows[4] = {&p.row_repetition, &p.row_presence, &p.row_frequency, &p.row_temperature};
  for (int i = 0; i < 4; ++i)
    if (how.row[i].defined()) *rows[i] = how.row[i].data_ptr<float>();
  return p;
}

Tensor logits_forward(const Tensor& logits, const LogitHow& how, goenv_logit_rules p) {
  Tensor out = at::empty(logits.sizes(), logits.options().dtype(how.out_type));
  const int64_t need = goenv_policy_logits_workspace(p.rows, p.cols, p.out_kind, 0, 0);
  const Tensor ws = workspace_of(need, logits);
  if (need > 0) p.workspace = ws.data_ptr(), p.workspace_bytes = need;
  check_rc(goenv_policy_logits(&p, out.data_ptr(), stream_of(logits)));
  return out;
}

// What a node keeps in a tensor of bytes, one after the other: the rows' statistics, and copies of the histories, the mask (as bits) and the
// histories' lengths -- the environment writes the next position's into such buffers through plain pointers, of which a saved
// tensor's version count knows nothing.
struct Kept {
  int64_t stats = 0, mask_rows = 0, past_rows = 0, moves = 0, move_bytes = 0, lens = 0;
  int64_t past_bytes() const { return past_rows * moves * move_bytes; }
  int64_t stats_bytes() const { return stats * 2 * (int64_t)sizeof(float); }
  int64_t copy_bytes(int64_t words) const { return past_bytes() + (mask_rows * words + lens) * (int64_t)sizeof(int32_t); }
  static Kept of(const goenv_logit_rules& p) {   // (rows that are all the same one are kept once)
    Kept k;
    if (p.rows == 0 || p.cols == 0) return k;
    if (p.out_kind != GOENV_OUT_LOGITS) k.stats = p.rows;
    if (p.legal || p.legal_bits) k.mask_rows = (p.legal ? p.legal_row : p.bits_row) == 0 ? 1 : p.rows;
    if (!p.history) return k;
    k.past_rows = p.history_row == 0 ? 1 : p.rows;
    k.moves = p.history_max;
    k.move_bytes = p.history_i64 ? sizeof(int64_t) : sizeof(int32_t);
    if (p.history_len) k.lens = p.rows;
    return k;
  }
  // p with the statistics and copies that lie at `base`
  void to(goenv_logit_rules& p, char* base) const {
    const int64_t words = (p.cols + 31) / 32;
    p.stats = stats ? reinterpret_cast<float*>(base) : nullptr;
    base += stats_bytes();
    p.history = past_rows ? base : nullptr;
    p.history_row = past_rows == 1 ? 0 : moves;
    p.history_max = (int32_t)moves;
    p.history_i64 = move_bytes == sizeof(int64_t);
    base += past_bytes();
    p.legal = nullptr;
    p.legal_bits = mask_rows ? reinterpret_cast<uint32_t*>(base) : nullptr;
    p.bits_row = mask_rows == 1 ? 0 : words;
    base += mask_rows * words * sizeof(uint32_t);
    p.history_len = lens ? reinterpret_cast<int32_t*>(base) : nullptr;
  }
};

struct LogitNode : torch::autograd::Function<LogitNode> {
  struct Call {   // (a string in the node: one entry)
    float scalar[4];
    int out_kind;
    at::ScalarType out_type;
    Kept kept;
  };
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Maybe& b, const LogitHow& how) {
    const Tensor bias = tensor_of(b);
    goenv_logit_rules p = logit_args(logits, bias, how), own = p;
    Call call{{}, how.out_kind, how.out_type, Kept::of(p)};
    std::copy(how.scalar, how.scalar + 4, call.scalar);
    const int64_t copies = call.kept.copy_bytes((p.cols + 31) / 32);
    const Tensor memory = workspace_of(call.kept.stats_bytes() + copies, logits);
    if (memory.defined()) {
      call.kept.to(own, static_cast<char*>(memory.data_ptr()));
      p.stats = own.stats;
    }
    Tensor out = logits_forward(logits, how, p);
    if (copies > 0)
      check_rc(goenv_policy_logits_keep(&p, const_cast<uint32_t*>(own.legal_bits), const_cast<void*>(own.history), const_cast<int32_t*>(own.history_len),
                                        stream_of(logits)));
    ctx->save_for_backward({logits, bias, memory, how.row[0], how.row[1], how.row[2], how.row[3]});
    ctx->saved_data["call"] = std::string(reinterpret_cast<const char*>(&call), sizeof(call));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_plain(grads[0], "the gradient");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &bias = saved[1], &memory = saved[2];
    Call call;
    std::memcpy(&call, ctx->saved_data["call"].toStringRef().data(), sizeof(call));
    LogitHow how{{}, {}, {}, {}, {saved[3], saved[4], saved[5], saved[6]}, {}, call.out_kind, call.out_type};
    std::copy(call.scalar, call.scalar + 4, how.scalar);
    variable_list out(3);
    {
      at::NoGradGuard no_grad;
      Tensor dy = grads[0].resolve_neg();
      if (dy.size(1) != 1 && dy.stride(1) != 1) dy = dy.contiguous();
      Needs needs{ctx};
      if (needs(logits)) out[0] = at::empty(logits.sizes(), logits.options());
      if (needs(bias)) out[1] = at::empty(bias.sizes(), bias.options());
      goenv_logit_rules p = logit_args(logits, bias, how);
      if (memory.defined()) call.kept.to(p, static_cast<char*>(memory.data_ptr()));
      const int64_t need = goenv_policy_logits_workspace(p.rows, p.cols, p.out_kind, bias.defined() && p.bias_row == 0, 1);
      const Tensor ws = workspace_of(need, logits);
      if (need > 0) p.workspace = ws.data_ptr(), p.workspace_bytes = need;
      check_rc(goenv_policy_logits_grad(&p, dy.data_ptr(), dy.stride(0), out[0].defined() ? out[0].data_ptr() : nullptr,
                                        out[1].defined() ? out[1].data_ptr() : nullptr, stream_of(logits)));
    }
    once(out, {logits, bias, grads[0]});
    return out;
  }
};

Tensor policy_logits(py::handle plogits, py::handle plegal, py::handle pbits, py::handle pbias, py::handle phistory, py::handle plen, py::handle prepetition,
                     py::handle ppresence, py::handle pfrequency, py::handle ptemperature, const std::string& out, py::handle pdtype) {
  check_not_traced();
  const Tensor logits = main_tensor(plogits, "logits");
  if (logits.dim() != 2) refuse("logits must be [rows, cols] (got ", logits.sizes(), ")");
  const int64_t rows = logits.size(0), cols = logits.size(1);
  auto adjacent = [](const Tensor& t) { return t.size(1) == 1 || t.stride(1) == 1; };
  if (!adjacent(logits)) refuse("the columns of logits must lie next to each other (got strides ", logits.strides(), ")");
  LogitHow how;
  how.legal = optional_tensor(plegal, "legal");
  how.legal_bits = optional_tensor(pbits, "legal_bits");
  how.history = optional_tensor(phistory, "history");
  how.history_len = optional_tensor(plen, "history_len");
  const Tensor bias = optional_tensor(pbias, "bias");
  if (how.legal.defined()) {
    if (how.legal_bits.defined()) refuse("legal or legal_bits, not both");
    check_like(how.legal, "legal", logits, {at::kByte, at::kBool}, {rows, cols});
    if (!adjacent(how.legal)) refuse("the columns of legal must lie next to each other");
  }
  if (how.legal_bits.defined()) {
    check_like(how.legal_bits, "legal_bits", logits, {at::kInt}, {rows, (cols + 31) / 32});
    if (!adjacent(how.legal_bits)) refuse("the words of a row of legal_bits must lie next to each other");
  }
  if (bias.defined()) {
    if (bias.dim() == 1) check_like(bias, "bias", logits, {at::kFloat, logits.scalar_type()}, {cols});
    else check_like(bias, "bias", logits, {at::kFloat, logits.scalar_type()}, {rows, cols});
    if (!bias.is_contiguous()) refuse("bias must be contiguous");
  }
  if (how.history.defined()) {
    if (how.history.dim() != 2) refuse("history must be a tensor [rows, moves]");
    check_like(how.history, "history", logits, {at::kInt, at::kLong}, {rows, how.history.size(1)});
    if (how.history.size(1) > (1 << 28)) refuse("history must have at most 2^28 moves a row");
    if (!adjacent(how.history)) refuse("the entries of a row of history must lie next to each other");
  }
  if (how.history_len.defined()) {
    if (!how.history.defined()) refuse("history_len without history");
    check_like(how.history_len, "history_len", logits, {at::kInt}, {rows});
    if (!how.history_len.is_contiguous()) refuse("history_len must be contiguous");
  }
  if (out == "logits") how.out_kind = GOENV_OUT_LOGITS;
  else if (out == "log_probs") how.out_kind = GOENV_OUT_LOG_PROBS;
  else if (out == "probs") how.out_kind = GOENV_OUT_PROBS;
  else refuse("out must be one of logits, log_probs, probs (got ", out, ")");
  how.out_type = logits.scalar_type();
  if (!pdtype.is_none()) {
    if (!THPDtype_Check(pdtype.ptr())) refuse("dtype must be float32 or the logits' type");
    how.out_type = reinterpret_cast<THPDtype*>(pdtype.ptr())->scalar_type;
    if (how.out_type != at::kFloat && how.out_type != logits.scalar_type())
      refuse("dtype must be float32 or the logits' type (got ", how.out_type, ")");
  }
  const py::handle given[4] = {prepetition, ppresence, pfrequency, ptemperature};
  static const char* const names[4] = {"repetition", "presence", "frequency", "temperature"};
  for (int i = 0; i < 4; ++i) {
    how.scalar[i] = i % 3 == 0 ? 1.f : 0.f;
    if (!THPVariable_Check(given[i].ptr())) {
      how.scalar[i] = (float)number(given[i], (std::string(names[i]) + " must be a tensor [rows] or it").c_str());
      continue;
    }
    const Tensor t = optional_tensor(given[i], names[i]);
    check_like(t, names[i], logits, {at::kFloat}, {rows});
    if (!t.is_contiguous()) refuse(names[i], " must be contiguous");
    if (t.requires_grad() && at::GradMode::is_enabled()) refuse(names[i], " has no gradient (detach it)");
    how.row[i] = t;
  }
  if (wants_grad({logits, bias})) return LogitNode::apply(logits, maybe(bias), how);
  return logits_forward(logits, how, logit_args(logits, bias, how));
}

}  // namespace

PYBIND11_MODULE(_policy_ops, m) {
  static PyObject* error = py::object(py::module_::import("elf_amd.goenv").attr("GoEnvError")).release().ptr();   // (kept until the process ends)
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const OpError& e) {
      PyErr_SetString(error, e.what());
    }
  });
  m.def("group_norm_act", &group_norm_act);
  m.def("dropout", &dropout);
  m.def("policy_logits", &policy_logits);
}
