// operators.cpp -- the host side of the operators on tensors (metta_amd/recurrence.py, metta_amd/action_head.py): checks of the
// arguments, results and workspaces from torch's allocator, launches on torch's current stream, and the backward passes as
// nodes of autograd's graph.  In C++ because small calls are bound by the host: the same in Python took 14 us for a sampling
// call and 55 us for a backward pass, which autograd runs in a thread of its own that had to wait for the interpreter.
//
// The kernels are reached through the C interface of the library that native.py has loaded (`bind`).
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <cstring>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>

#include "../../include/mettagrid_hip.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

namespace {

#define LIBRARY(f) f(mg_last_error) f(mg_gated_recurrence_workspace) f(mg_gated_recurrence) f(mg_gated_recurrence_backward) \
    f(mg_logits_workspace) f(mg_adjust_logits) f(mg_adjust_logits_backward) f(mg_sample_actions) f(mg_evaluate_actions) \
    f(mg_evaluate_actions_backward)
#define POINTER(name) decltype(&::name) name = nullptr;
struct Library { LIBRARY(POINTER) } lib;

void bind(const py::dict& addresses) {
#define TAKE(name) lib.name = reinterpret_cast<decltype(lib.name)>(addresses[#name].cast<uintptr_t>());
  LIBRARY(TAKE)
}

[[noreturn]] void fail(const std::string& message) { throw std::runtime_error(message); }
void require(bool ok, const char* message) {
  if (!ok) fail(message);
}

// what a launch wants around it: the tensors' device as the current one, and its current stream
struct Place {
  c10::DeviceGuard guard;
  void* stream;
  explicit Place(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};
void launched(int rc) {
  if (rc) fail(lib.mg_last_error());
}

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MG_F32;
    case at::kBFloat16: return MG_BF16;
    case at::kHalf: return MG_F16;
    default: return -1;
  }
}
bool has(const Maybe& t) { return t && t->defined(); }
Tensor or_none(const Maybe& t) { return has(t) ? *t : Tensor(); }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// (a view that holds its values negated, like the imaginary part of a conjugate, is written out: kernels read memory as it is)
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor contiguous(const Tensor& t) { return t.defined() ? plain(t).contiguous() : t; }
// columns next to each other
bool adjacent_columns(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1; }
Tensor adjacent(const Tensor& t) { return !t.defined() ? t : adjacent_columns(t) ? plain(t) : t.contiguous(); }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
// whether t is a dual tensor whose tangent a forward-mode derivative would go on with
bool dual(const Tensor& t) { return t.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined(); }
Tensor empty(at::IntArrayRef shape, const Tensor& like, at::ScalarType type) { return at::empty(shape, like.options().dtype(type).requires_grad(false)); }

// A launch is no operation of torch's: a trace would hold the results' memory without what fills it.
void untraced(const char* who) {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
    fail(std::string(who) + " cannot be traced");
}

// A call without requires_grad goes past autograd, which would refuse the tangent of a dual tensor: it is refused, not dropped.
void reverse_only(const char* who, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (dual(*t)) fail(std::string(who) + " has no forward-mode derivative");
}

// A backward pass of kernels has no graph of its own: a second derivative through its results is an error, not a wrong number.
void once(variable_list& grads, const char* who) {
  if (!at::GradMode::is_enabled()) return;
  const auto node = std::make_shared<torch::autograd::Error>(std::string(who) + " is differentiable once");
  for (Tensor& g : grads)
    if (g.defined()) torch::autograd::create_gradient_edge(g, node);
}

// ---- gated linear recurrence --------------------------------------------------------------------------------------------

// [rows][steps][width] (or [rows][width]: one step) of candidates and gates, apart or side by side
struct Core {
  Tensor x, gate;
  int64_t width;

  Core(const Tensor& x_, const Tensor& gate_) : x(x_), gate(gate_), width(gate_.defined() ? x_.size(-1) : x_.size(-1) / 2) {}
  bool one() const { return x.dim() == 2; }
  int64_t rows() const { return x.size(0); }
  int64_t steps() const { return one() ? 1 : x.size(1); }

  mg_recurrence args(const Tensor& state, const Tensor& resets) const {
    const Tensor& g = gate.defined() ? gate : x;
    mg_recurrence r{};
    r.x = x.data_ptr();
    r.gate = gate.defined() ? g.data_ptr() : static_cast<char*>(x.data_ptr()) + width * x.element_size();
    r.state = static_cast<const float*>(data(state));
    r.resets = static_cast<const uint8_t*>(data(resets));
    r.rows = rows(), r.steps = steps(), r.width = width;
    r.x_row = x.stride(0), r.x_step = one() ? 0 : x.stride(1);
    r.gate_row = g.stride(0), r.gate_step = one() ? 0 : g.stride(1);
    r.type = type_of(x);
    return r;
  }
};

// the checks that both entry points share
void check_core(const Tensor& x, const Tensor& gate, const Tensor& state, const Tensor& resets, int dims) {
  if (x.dim() != dims) fail("x must be " + std::to_string(dims) + "D");
  if (!gate.defined()) require(x.size(-1) % 2 == 0, "without a gate, x holds candidates and gates side by side: its last dimension must be even");
  else require(gate.sizes() == x.sizes(), "x and gate must have the same shape");
  require(type_of(x) >= 0 && (!gate.defined() || gate.scalar_type() == x.scalar_type()), "x and gate must both be float32, bfloat16 or float16");
  const int64_t rows = x.size(0), width = gate.defined() ? x.size(-1) : x.size(-1) / 2;
  if (state.defined()) {
    require(state.scalar_type() == at::kFloat, "state must be float32");
    require(state.dim() == 2 && state.size(0) == rows && state.size(1) == width, "state must be [rows, width]");
  }
  if (resets.defined()) {
    require(resets.scalar_type() == at::kBool || resets.scalar_type() == at::kByte, "resets must be bool or uint8");
    require(resets.sizes() == x.sizes().slice(0, dims - 1), "resets must have x's shape without its last dimension");
  }
  require(width == 0 || rows <= (int64_t(1) << 31) / width, "rows * width must not exceed 2^31");
  for (const Tensor* t : {&gate, &state, &resets}) require(!t->defined() || t->device() == x.device(), "All tensors must be on same device");
}
void check_device(const Tensor& x) { require(x.is_cuda(), "All tensors must be on GPU"); }

// Whether a contiguous `out` of [rows, width] lies over what a step reads of `t` ([rows, width] from column `from` on), otherwise than
// element on element: a thread would write what another has yet to read.  (A t that is copied before the launch is no matter.)
bool written_over(const Tensor& out, const Tensor& t, int64_t from, int64_t width) {
  if (!out.numel() || !t.numel() || !adjacent_columns(t) || t.is_neg()) return false;
  const int64_t size = t.element_size(), rows = out.size(0), row = t.stride(0) * size, wide = width * size, bytes = out.numel() * out.element_size();
  // bytes from out's first to t's
  const int64_t at = reinterpret_cast<intptr_t>(t.data_ptr()) + from * size - reinterpret_cast<intptr_t>(out.data_ptr());
  if (at == 0 && size == out.element_size() && (rows == 1 || row == wide)) return false;
  // the first of t's rows that ends behind out's beginning: does it begin before out's end?
  const int64_t first = at + wide > 0 ? 0 : row ? -(at + wide) / row + 1 : rows;
  return first < rows && at + first * row < bytes;
}

// memory of this call's own (torch's allocator keeps it for the stream, and for a captured graph)
Tensor workspace(mg_recurrence& r, const Tensor& like) {
  const int64_t size = lib.mg_gated_recurrence_workspace(&r);
  if (!size) return {};
  Tensor w = empty({size}, like, at::kByte);
  r.workspace = w.data_ptr(), r.workspace_bytes = size;
  return w;
}

struct Scanned { Tensor h, last, marks; };

Scanned scan(const Core& c, const Tensor& state, const Tensor& resets, bool train) {
  Scanned s;
  const int64_t rows = c.rows(), steps = c.steps();
  s.h = empty({rows, steps, c.width}, c.x, c.x.scalar_type());
  s.last = empty({rows, c.width}, c.x, at::kFloat);
  if (train && c.x.scalar_type() != at::kFloat) s.marks = empty({rows, (steps - 1) / MG_RECURRENCE_MARK_STEPS, c.width}, c.x, at::kFloat);
  const Place place(c.x);
  mg_recurrence r = c.args(state, resets);
  const Tensor w = workspace(r, c.x);
  launched(lib.mg_gated_recurrence(&r, s.h.data_ptr(), s.last.data_ptr<float>(), static_cast<float*>(data(s.marks)), place.stream));
  return s;
}

struct Recurrence : torch::autograd::Function<Recurrence> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& gate_, const Maybe& state_, const Maybe& resets_) {
    const Tensor gate = or_none(gate_), state = or_none(state_), resets = or_none(resets_);
    ctx->set_materialize_grads(false);
    const Scanned s = scan(Core(x, gate), state, resets, true);
    // an f32 output holds the states itself, in shorter types they are kept apart
    ctx->save_for_backward({x, gate, state, resets, s.marks.defined() ? s.marks : s.h});
    ctx->saved_data["state"] = wants(state);
    return {s.h, s.last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const at::AutoDispatchBelowADInplaceOrView below;
    // (what comes back may lie elsewhere and otherwise than what was saved: a hook may have moved it)
    const variable_list saved = ctx->get_saved_variables();
    const Core c(adjacent(saved[0]), adjacent(saved[1]));
    const Tensor state = contiguous(saved[2]), resets = contiguous(saved[3]), marks = contiguous(saved[4]);
    const Tensor dh = adjacent(grads[0]), dlast = contiguous(grads[1]);
    const bool f32 = c.x.scalar_type() == at::kFloat, apart = c.gate.defined();
    const int64_t steps = c.steps(), mark = MG_RECURRENCE_MARK_STEPS;
    Tensor dx = empty(c.x.sizes(), c.x, c.x.scalar_type()), dgate, dstate;
    if (apart) dgate = empty(c.x.sizes(), c.x, c.x.scalar_type());
    if (ctx->saved_data["state"].toBool()) dstate = empty(state.sizes(), state, at::kFloat);
    const Place place(c.x);
    mg_recurrence_gradients d{};
    d.dh = data(dh);
    d.dlast = static_cast<const float*>(data(dlast));
    d.dx = dx.data_ptr();
    d.dgate = apart ? dgate.data_ptr() : static_cast<char*>(dx.data_ptr()) + c.width * dx.element_size();
    d.dstate = static_cast<float*>(data(dstate));
    if (dh.defined()) d.dh_row = dh.stride(0), d.dh_step = dh.stride(1);
    d.dx_row = d.dgate_row = dx.stride(0), d.dx_step = d.dgate_step = dx.stride(1);
    mg_recurrence r = c.args(state, resets);
    const Tensor w = workspace(r, c.x);
    const float* at = static_cast<const float*>(data(marks)) + (f32 ? (mark - 1) * c.width : 0);
    const int64_t row = f32 ? steps * c.width : (steps - 1) / mark * c.width, stride = f32 ? mark * c.width : c.width;
    launched(lib.mg_gated_recurrence_backward(&r, at, row, stride, &d, place.stream));
    variable_list out{dx, dgate, dstate, Tensor()};
    once(out, "gated_recurrence");
    return out;
  }
};

std::tuple<Tensor, Tensor> gated_recurrence(const Tensor& x_, const Maybe& gate_, const Maybe& state_, const Maybe& resets_) {
  untraced("gated_recurrence");
  Tensor gate = or_none(gate_), state = or_none(state_);
  check_core(x_, gate, state, or_none(resets_), 3);
  reverse_only("gated_recurrence", {&x_, &gate, &state});
  check_device(x_);
  const Core given(x_, gate);
  state = contiguous(state);
  if (x_.numel() == 0) {  // nothing to compute; part of the graph all the same
    const Tensor xs = gate.defined() ? x_ : x_.narrow(2, 0, given.width), gs = gate.defined() ? gate : x_.narrow(2, given.width, given.width);
    return {xs + gs, state.defined() ? state.clone() : at::zeros({x_.size(0), given.width}, x_.options().dtype(at::kFloat).requires_grad(false))};
  }
  const Tensor x = adjacent(x_), resets = contiguous(or_none(resets_));
  gate = adjacent(gate);
  if (at::GradMode::is_enabled() && (wants(x) || wants(gate) || wants(state))) {
    const auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
    const variable_list out = Recurrence::apply(x, maybe(gate), maybe(state), maybe(resets));
    return {out[0], out[1]};
  }
  const at::AutoDispatchBelowADInplaceOrView below;
  const Scanned s = scan(Core(x, gate), state, resets, false);
  return {s.h, s.last};
}

std::tuple<Tensor, Tensor> gated_recurrence_step(const Tensor& x, const Maybe& gate_, const Tensor& state, const Maybe& resets_, const Maybe& out_) {
  untraced("gated_recurrence_step");
  const Tensor gate = or_none(gate_), resets = or_none(resets_);
  check_core(x, gate, state, resets, 2);
  reverse_only("gated_recurrence_step", {&x, &gate, &state});
  const bool grad = at::GradMode::is_enabled();
  require(!grad || !(wants(x) || wants(gate) || wants(state)),
          "gated_recurrence_step has no gradient: call it under torch.no_grad(), or use gated_recurrence");
  Tensor out = or_none(out_);
  if (out.defined()) {
    require(out.sizes() == state.sizes() && out.scalar_type() == at::kFloat && out.device() == x.device() && out.is_contiguous() && !out.is_neg(),
            "out_state must be contiguous float32 [rows, width] on x's device");
    require(!grad || !out.requires_grad(), "out_state is written in place and must not require a gradient");
    require(!dual(out), "out_state is written in place and must not carry a tangent");
    const int64_t apart = std::abs(static_cast<const char*>(out.data_ptr()) - static_cast<const char*>(state.data_ptr()));
    require(apart == 0 || apart >= 4 * state.numel(), "out_state may be state itself, but not overlap it otherwise");
    const int64_t width = out.size(1);
    require(!written_over(out, x, 0, width) && !written_over(out, gate.defined() ? gate : x, gate.defined() ? 0 : width, width) &&
                !(resets.defined() && resets.is_contiguous() && written_over(out, resets.unsqueeze(-1), 0, 1)),
            "out_state may not overlap x, gate or resets other than element on element");
  }
  check_device(x);
  const at::AutoDispatchBelowADInplaceOrView below;
  if (!out.defined()) out = empty(state.sizes(), x, at::kFloat);
  const Tensor h = x.scalar_type() == at::kFloat ? out : empty(state.sizes(), x, x.scalar_type());
  if (out.numel()) {
    const Core c(adjacent(x), adjacent(gate));
    const Tensor from = contiguous(state), marked = contiguous(resets);
    const Place place(x);
    const mg_recurrence r = c.args(from, marked);
    launched(lib.mg_gated_recurrence(&r, h.is_same(out) ? nullptr : h.data_ptr(), out.data_ptr<float>(), nullptr, place.stream));
    if (has(out_) && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  }
  return {h, out};
}

// ---- action head ----------------------------------------------------------------------------------------------------------

// [..., V] as [rows, V] with adjacent columns, a view where the strides allow it
Tensor as_rows(const Tensor& t) {
  if (t.dim() == 2) return adjacent(t);
  return adjacent(t.dim() > 1 ? t.reshape({-1, t.size(-1)}) : t.unsqueeze(0));
}

// checked arguments of one call
struct Head {
  Tensor logits, allowed, bias, history;
  mg_logits a{};
  at::DimVector lead;

  Head() = default;
  Head(const Tensor& l, const Maybe& allowed_, const Maybe& bias_, const Maybe& history_, double temperature, double repetition, double presence,
       double frequency, bool gradient) {
    const Tensor given_allowed = or_none(allowed_), given_bias = or_none(bias_);
    Tensor given_history = or_none(history_);
    require(l.dim() >= 1 && l.size(-1) >= 1, "logits must be [..., V] with at least one token");
    require(type_of(l) >= 0, "logits must be float32, bfloat16 or float16");
    const int64_t v = l.size(-1);
    lead.assign(l.sizes().begin(), l.sizes().end() - 1);
    require(v < int64_t(1) << 31, "logits must have fewer than 2^31 tokens");
    require(temperature >= 1e-30 && temperature <= 1e30, "temperature must be from 1e-30 to 1e30");
    require(repetition >= 1e-30 && repetition <= 1e30, "repetition must be from 1e-30 to 1e30");
    require(std::isfinite(presence) && std::isfinite(frequency), "presence and frequency must be finite");
    for (const Tensor* t : std::initializer_list<const Tensor*>{&given_allowed, &given_bias, &given_history})
      require(!t->defined() || t->device() == l.device(), "All tensors must be on same device");
    int64_t mask_width = 0;
    if (given_allowed.defined()) {
      if (given_allowed.scalar_type() == at::kBool) a.allowed_kind = MG_ALLOWED_BOOL, mask_width = v;
      else if (given_allowed.scalar_type() == at::kInt) a.allowed_kind = MG_ALLOWED_BITS, mask_width = (v + 31) / 32;
      else fail("allowed must be bool, or int32 bits (pack_allowed)");
    }
    if (given_bias.defined()) {
      require(given_bias.scalar_type() == at::kFloat, "bias must be float32");
      require(!gradient || !given_bias.requires_grad() || !at::GradMode::is_enabled(), "bias is a constant: it must not require a gradient");
      require(!gradient || !dual(given_bias), "bias is a constant: it must not carry a tangent");
    }
    const bool penalties = repetition != 1.0 || presence != 0.0 || frequency != 0.0;
    if (given_history.defined()) {
      require(given_history.scalar_type() == at::kInt, "history must be int32");
      require(given_history.dim() >= 1 && given_history.sizes().slice(0, given_history.dim() - 1) == at::IntArrayRef(lead),
              "history must be [..., L] with the logits' leading dimensions");
      require(given_history.size(-1) <= int64_t(1) << 30, "history must have at most 2^30 entries");
      if (given_history.size(-1) == 0 || !penalties) given_history = Tensor();
    } else {
      require(!penalties, "penalties need a history");
    }
    const at::NoGradGuard no_grad;
    allowed = control("allowed", given_allowed, mask_width, a.allowed_row);
    bias = control("bias", given_bias, v, a.bias_row);
    require(l.is_cuda(), "All tensors must be on GPU");
    logits = as_rows(l);
    if (given_history.defined()) history = as_rows(given_history);
    a.temperature = temperature, a.repetition = repetition, a.presence = presence, a.frequency = frequency;
    a.width = static_cast<int32_t>(v);
    point();
  }
  // from what a backward pass gets back (which may lie elsewhere and otherwise than what was saved: a hook may have moved it)
  Head(const variable_list& saved, const mg_logits& args) : logits(adjacent(saved[0])), allowed(adjacent(saved[1])), bias(adjacent(saved[2])), history(adjacent(saved[3])), a(args) {
    a.allowed_row = allowed.defined() && allowed.dim() == 2 ? allowed.stride(0) : 0;
    a.bias_row = bias.defined() && bias.dim() == 2 ? bias.stride(0) : 0;
    point();
  }
  void point() {
    a.logits = logits.data_ptr();
    a.bias = static_cast<const float*>(data(bias));
    a.allowed = data(allowed);
    a.history = static_cast<const int32_t*>(data(history));
    a.rows = logits.size(0), a.logits_row = logits.stride(0);
    a.history_row = history.defined() ? history.stride(0) : 0;
    a.history_len = history.defined() ? static_cast<int32_t>(history.size(1)) : 0;
    a.type = type_of(logits);
    a.workspace = nullptr, a.workspace_bytes = 0;
  }
  // a control, and its row stride: 0 where one row serves all
  Tensor control(const char* name, const Tensor& t, int64_t width, int64_t& row) const {
    row = 0;
    if (!t.defined()) return t;
    const bool fits = t.dim() >= 1 && t.size(-1) == width && (t.dim() == 1 || t.sizes().slice(0, t.dim() - 1) == at::IntArrayRef(lead));
    if (!fits) {
      const std::string w = std::to_string(width);
      fail(std::string(name) + " must be [" + w + "] or [..., " + w + "] with the logits' leading dimensions");
    }
    if (t.dim() == 1) return contiguous(t);
    const Tensor rows = as_rows(t);
    row = rows.stride(0);
    return rows;
  }
  // one value per row
  Tensor per_row(const char* name, const Tensor& t, const char* types, bool typed) const {
    if (!typed) fail(std::string(name) + " must be " + types);
    if (t.sizes() != at::IntArrayRef(lead)) fail(std::string(name) + " must have the logits' shape without its last dimension");
    require(t.device() == logits.device(), "All tensors must be on same device");
    return contiguous(t);
  }
  Tensor work() {
    const int64_t size = lib.mg_logits_workspace(&a);
    if (!size) return {};
    Tensor w = empty({size}, logits, at::kByte);
    a.workspace = w.data_ptr(), a.workspace_bytes = size;
    return w;
  }
};

// a head's scalars for its backward pass, among the saved tensors' data
void keep(AutogradContext* ctx, const Head& h, at::IntArrayRef shape) {
  ctx->saved_data["args"] = c10::IValue(std::string(reinterpret_cast<const char*>(&h.a), sizeof(h.a)));
  ctx->saved_data["shape"] = shape.vec();
}
mg_logits kept(AutogradContext* ctx) {
  mg_logits a;
  std::memcpy(&a, ctx->saved_data["args"].toStringRef().data(), sizeof(a));
  return a;
}

Tensor adjust(const Head& h, at::IntArrayRef shape) {
  const Tensor out = empty(shape, h.logits, h.logits.scalar_type());
  if (out.numel()) {
    const Place place(out);
    launched(lib.mg_adjust_logits(&h.a, out.data_ptr(), place.stream));
  }
  return out;
}

struct Adjust : torch::autograd::Function<Adjust> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Head* h) {
    // (through save_for_backward, so that a tensor changed in between is noticed)
    ctx->save_for_backward({h->logits, h->allowed, h->bias, h->history});
    keep(ctx, *h, logits.sizes());
    return adjust(*h, logits.sizes());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Tensor dout = contiguous(grads[0]);
    const Tensor d = empty(ctx->saved_data["shape"].toIntVector(), dout, dout.scalar_type());
    if (d.numel()) {
      const Head h(ctx->get_saved_variables(), kept(ctx));
      const Place place(d);
      launched(lib.mg_adjust_logits_backward(&h.a, dout.data_ptr(), d.data_ptr(), place.stream));
    }
    variable_list out{d, Tensor()};
    once(out, "adjust_logits");
    return out;
  }
};

Tensor adjust_logits(const Tensor& logits, const Maybe& allowed, const Maybe& bias, const Maybe& history, double temperature, double repetition,
                     double presence, double frequency) {
  untraced("adjust_logits");
  reverse_only("adjust_logits", {&logits});
  const Head h(logits, allowed, bias, history, temperature, repetition, presence, frequency, true);
  if (at::GradMode::is_enabled() && logits.requires_grad()) return Adjust::apply(logits, &h);
  const at::AutoDispatchBelowADInplaceOrView below;
  return adjust(h, logits.sizes());
}

std::tuple<Tensor, Tensor, Tensor> sample_actions(const Tensor& logits, const Maybe& uniforms_, const Maybe& allowed, const Maybe& bias,
                                                  const Maybe& history, double temperature, double repetition, double presence, double frequency) {
  untraced("sample_actions");
  Head h(logits, allowed, bias, history, temperature, repetition, presence, frequency, false);
  const at::AutoDispatchBelowADInplaceOrView below;
  const Tensor given = or_none(uniforms_);
  const Tensor uniforms = given.defined() ? h.per_row("uniforms", given, "float32", given.scalar_type() == at::kFloat) : given;
  const Tensor actions = empty(h.lead, logits, at::kInt), log_prob = empty(h.lead, logits, at::kFloat), entropy = empty(h.lead, logits, at::kFloat);
  if (actions.numel()) {
    const Place place(logits);
    const Tensor w = h.work();
    launched(lib.mg_sample_actions(&h.a, static_cast<const float*>(data(uniforms)), actions.data_ptr<int32_t>(), log_prob.data_ptr<float>(),
                                   entropy.data_ptr<float>(), place.stream));
  }
  return {actions, log_prob, entropy};
}

struct Evaluated { Tensor log_prob, entropy, stats; };

Evaluated evaluate(Head& h, const Tensor& actions, bool train) {
  Evaluated e{empty(h.lead, h.logits, at::kFloat), empty(h.lead, h.logits, at::kFloat), {}};
  if (train && h.a.width > MG_EVALUATE_STATS_WIDTH) e.stats = empty({h.a.rows, 2}, h.logits, at::kDouble);
  if (e.log_prob.numel()) {
    const Place place(h.logits);
    const Tensor w = h.work();
    launched(lib.mg_evaluate_actions(&h.a, actions.data_ptr<int32_t>(), e.log_prob.data_ptr<float>(), e.entropy.data_ptr<float>(),
                                     static_cast<double*>(data(e.stats)), place.stream));
  }
  return e;
}

struct Evaluate : torch::autograd::Function<Evaluate> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, Head* h, const Tensor& actions) {
    ctx->set_materialize_grads(false);
    const Evaluated e = evaluate(*h, actions, true);
    ctx->save_for_backward({h->logits, h->allowed, h->bias, h->history, actions, e.entropy, e.stats});
    keep(ctx, *h, logits.sizes());
    return {e.log_prob, e.entropy};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
    const at::AutoDispatchBelowADInplaceOrView below;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor d = empty(ctx->saved_data["shape"].toIntVector(), saved[0], saved[0].scalar_type());
    if (d.numel()) {
      const Head h(saved, kept(ctx));
      const Tensor dlogp = contiguous(grads[0]), dentropy = contiguous(grads[1]);
      const Tensor actions = contiguous(saved[4]), entropy = contiguous(saved[5]), stats = contiguous(saved[6]);
      const Place place(d);
      launched(lib.mg_evaluate_actions_backward(&h.a, actions.data_ptr<int32_t>(), entropy.data_ptr<float>(), static_cast<const double*>(data(stats)),
                                                static_cast<const float*>(data(dlogp)), static_cast<const float*>(data(dentropy)), d.data_ptr(),
                                                place.stream));
    }
    variable_list out{d, Tensor(), Tensor()};
    once(out, "evaluate_actions");
    return out;
  }
};

std::tuple<Tensor, Tensor> evaluate_actions(const Tensor& logits, const Tensor& given, const Maybe& allowed, const Maybe& bias, const Maybe& history,
                                            double temperature, double repetition, double presence, double frequency) {
  untraced("evaluate_actions");
  reverse_only("evaluate_actions", {&logits});
  Head h(logits, allowed, bias, history, temperature, repetition, presence, frequency, true);
  Tensor actions = h.per_row("actions", given, "int32 or int64", given.scalar_type() == at::kInt || given.scalar_type() == at::kLong);
  if (actions.scalar_type() == at::kLong) actions = actions.clamp(-1, 0x7FFFFFFF).to(at::kInt);  // (kept outside [0, V) where it is outside)
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    const variable_list out = Evaluate::apply(logits, &h, actions);
    return {out[0], out[1]};
  }
  const at::AutoDispatchBelowADInplaceOrView below;
  const Evaluated e = evaluate(h, actions, false);
  return {e.log_prob, e.entropy};
}

}  // namespace

PYBIND11_MODULE(_operators, m) {
  const py::call_guard<py::gil_scoped_release> free;
  m.def("bind", &bind);
  m.def("gated_recurrence", &gated_recurrence, free);
  m.def("gated_recurrence_step", &gated_recurrence_step, free);
  m.def("adjust_logits", &adjust_logits, free);
  m.def("sample_actions", &sample_actions, free);
  m.def("evaluate_actions", &evaluate_actions, free);
}
