// sequence_bindings.cpp -- the compiled half of astra_cuda.sequence: argument checks, output
// and workspace tensors, the calls of include/sequence/astra_sequence.h on PyTorch's current stream,
// and the autograd nodes around them. In C++ because a call of one position, or a backward
// pass on autograd's own thread, takes less time on the GPU than a Python body would.
#include "bindings.h"

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <limits>
#include <optional>

#include "sequence/astra_sequence.h"

namespace py = pybind11;

namespace astra_bind {
namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Optional = std::optional<Tensor>;

std::string shape_text(c10::IntArrayRef s) {
  std::string t = "[";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + "]";
}

void need(bool cond, const char *name, const std::string &what) {
  if (!cond) fatal(std::string("sequence: ") + name + " " + what);
}

int32_t type_of(const Tensor &t) { return t.scalar_type() == torch::kBFloat16 ? ASTRA_SEQ_BF16 : ASTRA_SEQ_F32; }

// A float32 or bfloat16 tensor on a HIP device.
void check_data(const char *name, const Tensor &t) {
  need(t.is_cuda(), name, "must be on a HIP device");
  need(t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16, name,
       std::string("must be float32 or bfloat16, got ") + c10::toString(t.scalar_type()));
}
// likewise, of x's type and device, and of a shape
void check_like(const char *name, const Tensor &t, const Tensor &x, c10::IntArrayRef shape) {
  need(t.device() == x.device(), name, "must be on " + x.device().str() + ", got " + t.device().str());
  need(t.scalar_type() == x.scalar_type(), name,
       std::string("must be ") + c10::toString(x.scalar_type()) + ", got " + c10::toString(t.scalar_type()));
  need(t.sizes() == shape, name, "must have shape " + shape_text(shape) + ", got " + shape_text(t.sizes()));
}

// A parameter or state as a contiguous float32 tensor (differentiably), undefined for None.
Tensor param(const char *name, const Optional &t, const Tensor &x, c10::IntArrayRef shape) {
  if (!t || !t->defined()) return {};
  need(t->device() == x.device(), name, "must be on " + x.device().str() + ", got " + t->device().str());
  need(at::isFloatingType(t->scalar_type()), name, std::string("must be a floating point tensor, got ") + c10::toString(t->scalar_type()));
  need(t->sizes() == shape, name, "must have shape " + shape_text(shape) + ", got " + shape_text(t->sizes()));
  return (t->scalar_type() == torch::kFloat32 ? *t : t->to(torch::kFloat32)).contiguous();
}

Tensor lengths_of(const Optional &t, const Tensor &x, int64_t batch) {
  if (!t || !t->defined()) return {};
  need(t->device() == x.device(), "lengths", "must be on " + x.device().str() + ", got " + t->device().str());
  need(t->scalar_type() == torch::kInt32 || t->scalar_type() == torch::kInt64, "lengths",
       std::string("must be int32 or int64, got ") + c10::toString(t->scalar_type()));
  need(t->dim() == 1 && t->size(0) == batch, "lengths",
       "must have shape [" + std::to_string(batch) + "], got " + shape_text(t->sizes()));
  // (64-bit lengths beyond what 32 bits hold are clamped like all others, not cut off)
  const Tensor wide = t->scalar_type() == torch::kInt64 ? t->clamp(0, std::numeric_limits<int32_t>::max()) : *t;
  return wide.to(torch::kInt32).contiguous();
}

// t with a contiguous last dimension (a dimension of size 1 has no stride to speak of).
Tensor rows(const Tensor &t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
// [..., D] as [rows, D] (a view where the strides allow it) with contiguous rows
Tensor flat(const Tensor &t) { return rows(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})); }

template <class T = void>
T *ptr(const Tensor &t) {
  return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}

bool with_grad(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Forward-mode derivatives and traces stop here: a result would come back without its tangent,
// and a trace would hold its allocation without what fills it, since the kernels write plain
// memory.
bool has_tangent(const Tensor &t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const Optional &t) { return t && has_tangent(*t); }
template <class... Ts>
void calls_only(const char *name, const Ts &...ts) {
  if (torch::jit::tracer::isTracing()) fatal(std::string("sequence: ") + name + " cannot be part of a trace");
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && (has_tangent(ts) || ...))
    fatal(std::string("sequence: ") + name + " has no forward-mode derivative");
}

Tensor empty(const Tensor &like, c10::IntArrayRef shape, c10::ScalarType type) {
  return at::empty(shape, like.options().dtype(type));
}
Tensor empty(const Tensor &t) { return empty(t, t.sizes(), t.scalar_type()); }

Tensor workspace(const Tensor &like, size_t bytes) {
  return bytes ? empty(like, {(int64_t)bytes}, torch::kUInt8) : Tensor();
}

// Autograd nodes take absent tensors as absent optionals.
Optional maybe(const Tensor &t) { return t.defined() ? Optional(t) : Optional(); }
Tensor value(const Optional &t) { return t ? *t : Tensor(); }

// The gradients are not differentiable themselves.
void check_once() {
  if (at::GradMode::is_enabled()) fatal("sequence: the operators can be differentiated once only (create_graph)");
}

Tensor undefined_or_contiguous(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

// ------------------------------------------------------------------------ short_conv

astra_short_conv conv_struct(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &window,
                             const Tensor &lengths, int64_t activation) {
  astra_short_conv f{};
  f.x = ptr(x);
  f.weight = ptr<float>(weight);
  f.bias = ptr<float>(bias);
  f.window = ptr(window);
  f.lengths = ptr<int32_t>(lengths);
  f.batch = x.size(0);
  f.length = x.size(1);
  f.x_stride_b = x.stride(0);
  f.x_stride_t = x.stride(1);
  f.width = (int32_t)x.size(2);
  f.taps = (int32_t)weight.size(1);
  f.type = type_of(x);
  f.activation = (int32_t)activation;
  return f;
}

variable_list conv_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &window,
                           const Tensor &lengths, int64_t activation, bool want_last) {
  const c10::DeviceGuard guard(x.device());
  Tensor y = empty(x, x.sizes(), x.scalar_type()), last;
  if (want_last) last = empty(x, {x.size(0), weight.size(1) - 1, x.size(2)}, x.scalar_type());
  astra_short_conv f = conv_struct(x, weight, bias, window, lengths, activation);
  f.y = ptr(y);
  f.last = ptr(last);
  check(astra_short_conv_forward(&f, stream_of(x.get_device())));
  return want_last ? variable_list{y, last} : variable_list{y};
}

struct ShortConv : torch::autograd::Function<ShortConv> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Optional &bias,
                               const Optional &window, const Optional &lengths, int64_t activation, bool want_last) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, value(bias), value(window), value(lengths)});
    ctx->saved_data["activation"] = activation;
    return conv_forward(x, weight, value(bias), value(window), value(lengths), activation, want_last);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    check_once();
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &window = saved[3], &lengths = saved[4];
    variable_list out(7);
    Tensor dy = undefined_or_contiguous(grads[0]);
    const Tensor dlast = grads.size() > 1 ? undefined_or_contiguous(grads[1]) : Tensor();
    if (!dy.defined() && !dlast.defined()) return out;
    const c10::DeviceGuard guard(x.device());
    if (!dy.defined()) dy = at::zeros(x.sizes(), x.options());
    for (int i = 0; i < 4; ++i)
      if (saved[i].defined() && saved[i].requires_grad()) out[i] = empty(saved[i], saved[i].sizes(), saved[i].scalar_type());
    astra_short_conv_grad g{};
    g.f = conv_struct(x, weight, bias, window, lengths, ctx->saved_data["activation"].toInt());
    g.dy = ptr(dy);
    g.dlast = ptr(dlast);
    g.dx = ptr(out[0]);
    g.dweight = ptr<float>(out[1]);
    g.dbias = ptr<float>(out[2]);
    g.dwindow = ptr(out[3]);
    Tensor ws;
    if (g.dweight || g.dbias) {
      check(astra_short_conv_workspace_size(&g.f, &g.workspace_bytes));
      ws = workspace(x, g.workspace_bytes);
      g.workspace = ptr(ws);
    }
    check(astra_short_conv_backward(&g, stream_of(x.get_device())));
    return out;
  }
};

int64_t activation_of(const std::optional<std::string> &a) {
  if (!a) return ASTRA_SEQ_LINEAR;
  need(*a == "silu", "activation", "must be 'silu' or None, got '" + *a + "'");
  return ASTRA_SEQ_SILU;
}

void check_weight(const Tensor &weight) {
  need(weight.dim() == 2, "weight", "must have shape [width, taps], got " + shape_text(weight.sizes()));
  need(weight.size(1) >= 2 && weight.size(1) <= ASTRA_SEQ_MAX_TAPS, "weight",
       "must have 2 to " + std::to_string(ASTRA_SEQ_MAX_TAPS) + " taps, got " + std::to_string(weight.size(1)));
}

py::object short_conv(const Tensor &x_, const Tensor &weight_, const Optional &bias_,
                      const std::optional<std::string> &activation, const Optional &initial, const Optional &lengths_,
                      bool return_state) {
  calls_only("short_conv", x_, weight_, bias_, initial);
  check_data("x", x_);
  need(x_.dim() == 3 && x_.size(2) >= 1, "x", "must have shape [batch, length, width], got " + shape_text(x_.sizes()));
  check_weight(weight_);
  const int64_t B = x_.size(0), D = x_.size(2), K = weight_.size(1);
  const Tensor weight = param("weight", weight_, x_, {D, K}), bias = param("bias", bias_, x_, {D});
  Tensor window;
  if (initial) {
    check_like("initial_state", *initial, x_, {B, K - 1, D});
    window = initial->contiguous();
  }
  const Tensor lengths = lengths_of(lengths_, x_, B), x = rows(x_);
  const int64_t act = activation_of(activation);
  const variable_list out = with_grad({&x, &weight, &bias, &window})
                                ? ShortConv::apply(x, weight, maybe(bias), maybe(window), maybe(lengths), act, return_state)
                                : conv_forward(x, weight, bias, window, lengths, act, return_state);
  if (return_state) return py::make_tuple(out[0], out[1]);
  return py::cast(out[0]);
}

[[noreturn]] void no_gradient(const char *name) {
  fatal(std::string("sequence: ") + name +
        " moves its state on in place and has no gradient; call it under torch.no_grad(), or use the "
        "whole-sequence operator");
}

// A state was written through its pointer: what saved it for a backward pass has to notice, as
// after torch's own operations in place. (Inference tensors have no version.)
void moved_on(const Tensor &state) {
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
}

Tensor short_conv_step(const Tensor &x_, const Tensor &state, const Tensor &weight_, const Optional &bias_,
                       const std::optional<std::string> &activation) {
  calls_only("short_conv_step", x_, state, weight_, bias_);
  check_data("x", x_);
  need(x_.dim() == 2 && x_.size(1) >= 1, "x", "must have shape [batch, width], got " + shape_text(x_.sizes()));
  check_weight(weight_);
  const int64_t B = x_.size(0), D = x_.size(1), K = weight_.size(1);
  const Tensor weight = param("weight", weight_, x_, {D, K}), bias = param("bias", bias_, x_, {D});
  if (with_grad({&x_, &state, &weight, &bias})) no_gradient("short_conv_step");
  check_like("state", state, x_, {B, K - 1, D});
  need(state.is_contiguous(), "state", "must be contiguous");
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows(x_);
  Tensor y = empty(x, {B, D}, x.scalar_type());
  astra_short_conv_one o{};
  o.x = ptr(x);
  o.weight = ptr<float>(weight);
  o.bias = ptr<float>(bias);
  o.window = ptr(state);
  o.y = ptr(y);
  o.batch = B;
  o.x_stride_b = x.stride(0);
  o.width = (int32_t)D;
  o.taps = (int32_t)K;
  o.type = type_of(x);
  o.activation = (int32_t)activation_of(activation);
  check(astra_short_conv_step(&o, stream_of(x.get_device())));
  moved_on(state);
  return y;
}

// ------------------------------------------------------------------------ state_scan

astra_state_scan scan_struct(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &b, const Tensor &c,
                             const Tensor &D, const Tensor &dt_bias, const Tensor &initial, const Tensor &lengths) {
  astra_state_scan f{};
  f.x = ptr(x);
  f.dt = ptr(dt);
  f.b = ptr(b);
  f.c = ptr(c);
  f.A = ptr<float>(A);
  f.D = ptr<float>(D);
  f.dt_bias = ptr<float>(dt_bias);
  f.initial = ptr<float>(initial);
  f.lengths = ptr<int32_t>(lengths);
  f.batch = x.size(0);
  f.length = x.size(1);
  f.x_stride_b = x.stride(0);
  f.x_stride_t = x.stride(1);
  f.x_stride_h = x.stride(2);
  f.dt_stride_b = dt.stride(0);
  f.dt_stride_t = dt.stride(1);
  f.dt_stride_h = dt.stride(2);
  f.b_stride_b = b.stride(0);
  f.b_stride_t = b.stride(1);
  f.b_stride_g = b.stride(2);
  f.c_stride_b = c.stride(0);
  f.c_stride_t = c.stride(1);
  f.c_stride_g = c.stride(2);
  f.heads = (int32_t)x.size(2);
  f.dim = (int32_t)x.size(3);
  f.groups = (int32_t)b.size(2);
  f.state = (int32_t)b.size(3);
  f.type = type_of(x);
  return f;
}

// y, the last state if wanted, and with `states` the states between chunks for the backward call
variable_list scan_forward(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &b, const Tensor &c,
                           const Tensor &D, const Tensor &dt_bias, const Tensor &initial, const Tensor &lengths,
                           bool want_state, Tensor *states) {
  const c10::DeviceGuard guard(x.device());
  Tensor y = empty(x, x.sizes(), x.scalar_type()), last;
  if (want_state) last = empty(x, {x.size(0), x.size(2), x.size(3), b.size(3)}, torch::kFloat32);
  astra_state_scan f = scan_struct(x, dt, A, b, c, D, dt_bias, initial, lengths);
  f.y = ptr(y);
  f.final_state = ptr<float>(last);
  check(astra_state_scan_workspace_size(&f, &f.workspace_bytes));
  const Tensor ws = workspace(x, f.workspace_bytes);
  f.workspace = ptr(ws);
  if (states) {
    size_t n = 0;
    check(astra_state_scan_chunk_states(&f, &n));
    if (n) *states = empty(x, {(int64_t)n}, torch::kFloat32);
    f.chunk_states = ptr<float>(*states);
  }
  check(astra_state_scan_forward(&f, stream_of(x.get_device())));
  return want_state ? variable_list{y, last} : variable_list{y};
}

struct StateScan : torch::autograd::Function<StateScan> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &dt, const Tensor &A,
                               const Tensor &b, const Tensor &c, const Optional &D, const Optional &dt_bias,
                               const Optional &initial, const Optional &lengths, bool want_state) {
    Tensor states;
    variable_list out =
        scan_forward(x, dt, A, b, c, value(D), value(dt_bias), value(initial), value(lengths), want_state, &states);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, dt, A, b, c, value(D), value(dt_bias), value(initial), value(lengths), states});
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    check_once();
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &dt = s[1], &A = s[2], &b = s[3], &c = s[4], &D = s[5], &dt_bias = s[6], &initial = s[7],
                 &lengths = s[8], &states = s[9];
    variable_list out(10);
    Tensor dy = undefined_or_contiguous(grads[0]);
    const Tensor dfinal = grads.size() > 1 ? undefined_or_contiguous(grads[1]) : Tensor();
    if (!dy.defined() && !dfinal.defined()) return out;
    const c10::DeviceGuard guard(x.device());
    if (!dy.defined()) dy = at::zeros(x.sizes(), x.options());
    for (int i : {0, 1, 3, 4}) out[i] = empty(s[i], s[i].sizes(), s[i].scalar_type());
    for (int i : {2, 5, 6, 7})
      if (s[i].defined() && s[i].requires_grad()) out[i] = empty(s[i]);
    astra_state_scan_grad g{};
    g.f = scan_struct(x, dt, A, b, c, D, dt_bias, initial, lengths);
    g.f.chunk_states = ptr<float>(states);
    g.dy = ptr(dy);
    g.dfinal = ptr<float>(dfinal);
    g.dx = ptr(out[0]);
    g.ddt = ptr(out[1]);
    g.dA = ptr<float>(out[2]);
    g.db = ptr(out[3]);
    g.dc = ptr(out[4]);
    g.dD = ptr<float>(out[5]);
    g.ddt_bias = ptr<float>(out[6]);
    g.dinitial = ptr<float>(out[7]);
    check(astra_state_scan_grad_workspace_size(&g.f, &g.workspace_bytes));
    const Tensor ws = workspace(x, g.workspace_bytes);
    g.workspace = ptr(ws);
    check(astra_state_scan_backward(&g, stream_of(x.get_device())));
    return out;
  }
};

// Shapes with `lead` leading dimensions (batch, or batch and length).
void check_scan(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &b, const Tensor &c, int lead) {
  check_data("x", x);
  need(x.dim() == lead + 2, "x",
       std::string("must have shape ") + (lead == 1 ? "[batch, heads, dim]" : "[batch, length, heads, dim]") + ", got " +
           shape_text(x.sizes()));
  const int64_t H = x.size(lead), P = x.size(lead + 1);
  need(H >= 1 && P >= 1, "x", "must have at least one head and feature, got " + shape_text(x.sizes()));
  const c10::IntArrayRef head = x.sizes().slice(0, lead + 1);
  check_like("dt", dt, x, head);
  need(b.dim() == lead + 2, "B", "must have x's leading dimensions + [groups, state], got " + shape_text(b.sizes()));
  std::vector<int64_t> want(x.sizes().begin(), x.sizes().begin() + lead);
  want.push_back(b.size(lead));
  want.push_back(b.size(lead + 1));
  check_like("B", b, x, want);
  check_like("C", c, x, want);
  const int64_t G = b.size(lead), N = b.size(lead + 1);
  need(G >= 1 && H % G == 0, "B", "must have groups that divide the " + std::to_string(H) + " heads, got " + std::to_string(G));
  need(N >= 1 && N <= ASTRA_SEQ_MAX_STATE, "B",
       "must have a state of 1 to " + std::to_string(ASTRA_SEQ_MAX_STATE) + " values, got " + std::to_string(N));
}

py::object state_scan(const Tensor &x_, const Tensor &dt, const Tensor &A_, const Tensor &b_, const Tensor &c_,
                      const Optional &D_, const Optional &dt_bias_, const Optional &initial_, const Optional &lengths_,
                      bool return_state) {
  calls_only("state_scan", x_, dt, A_, b_, c_, D_, dt_bias_, initial_);
  check_scan(x_, dt, A_, b_, c_, 2);
  const int64_t B = x_.size(0), H = x_.size(2);
  const Tensor A = param("A", A_, x_, {H}), D = param("D", D_, x_, {H}), dt_bias = param("dt_bias", dt_bias_, x_, {H});
  const Tensor initial = param("initial_state", initial_, x_, {B, H, x_.size(3), b_.size(3)});
  const Tensor lengths = lengths_of(lengths_, x_, B), x = rows(x_), b = rows(b_), c = rows(c_);
  const variable_list out =
      with_grad({&x, &dt, &A, &b, &c, &D, &dt_bias, &initial})
          ? StateScan::apply(x, dt, A, b, c, maybe(D), maybe(dt_bias), maybe(initial), maybe(lengths), return_state)
          : scan_forward(x, dt, A, b, c, D, dt_bias, initial, lengths, return_state, nullptr);
  if (return_state) return py::make_tuple(out[0], out[1]);
  return py::cast(out[0]);
}

Tensor state_scan_step(const Tensor &x_, const Tensor &dt, const Tensor &A_, const Tensor &b_, const Tensor &c_,
                       const Tensor &state, const Optional &D_, const Optional &dt_bias_) {
  calls_only("state_scan_step", x_, dt, A_, b_, c_, state, D_, dt_bias_);
  check_scan(x_, dt, A_, b_, c_, 1);
  const int64_t B = x_.size(0), H = x_.size(1), P = x_.size(2), N = b_.size(2);
  const Tensor A = param("A", A_, x_, {H}), D = param("D", D_, x_, {H}), dt_bias = param("dt_bias", dt_bias_, x_, {H});
  if (with_grad({&x_, &dt, &A, &b_, &c_, &state, &D, &dt_bias})) no_gradient("state_scan_step");
  need(state.device() == x_.device() && state.scalar_type() == torch::kFloat32, "state",
       "must be a float32 tensor on " + x_.device().str());
  const int64_t want[] = {B, H, P, N};
  need(state.sizes() == c10::IntArrayRef(want, 4) && state.is_contiguous(), "state",
       "must be contiguous with shape " + shape_text({want, 4}) + ", got " + shape_text(state.sizes()));
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows(x_), b = rows(b_), c = rows(c_);
  Tensor y = empty(x, {B, H, P}, x.scalar_type());
  astra_state_scan_one o{};
  o.x = ptr(x);
  o.dt = ptr(dt);
  o.b = ptr(b);
  o.c = ptr(c);
  o.A = ptr<float>(A);
  o.D = ptr<float>(D);
  o.dt_bias = ptr<float>(dt_bias);
  o.h = ptr<float>(state);
  o.y = ptr(y);
  o.batch = B;
  o.x_stride_b = x.stride(0);
  o.x_stride_h = x.stride(1);
  o.dt_stride_b = dt.stride(0);
  o.dt_stride_h = dt.stride(1);
  o.b_stride_b = b.stride(0);
  o.b_stride_g = b.stride(1);
  o.c_stride_b = c.stride(0);
  o.c_stride_g = c.stride(1);
  o.heads = (int32_t)H;
  o.dim = (int32_t)P;
  o.groups = (int32_t)b.size(1);
  o.state = (int32_t)N;
  o.type = type_of(x);
  check(astra_state_scan_step(&o, stream_of(x.get_device())));
  moved_on(state);
  return y;
}

// ------------------------------------------------------------------------- join_norm

// Every tensor is 2-D here, [rows, width].
astra_join_norm join_struct(const Tensor &residual, const Tensor &block, const Tensor &post, const Tensor &next,
                            const Tensor &gate, const Tensor &scale, const Tensor &rstd, double eps) {
  const Tensor &like = block.defined() ? block : residual;
  astra_join_norm f{};
  f.residual = ptr(residual);
  f.block = ptr(block);
  f.gate = ptr(gate);
  f.post = ptr<float>(post);
  f.next = ptr<float>(next);
  f.scale = ptr<float>(scale);
  f.rstd = ptr<float>(rstd);
  f.rows = residual.size(0);
  f.residual_stride = residual.stride(0);
  f.block_stride = like.stride(0);
  f.gate_stride = gate.defined() ? gate.stride(0) : 0;
  f.width = (int32_t)residual.size(1);
  f.gate_width = gate.defined() ? (int32_t)gate.size(1) : 0;
  f.scale_width = scale.defined() ? (int32_t)scale.size(0) : 0;
  f.type = type_of(like);
  f.residual_type = type_of(residual);
  f.eps = (float)eps;
  return f;
}

// joined where there is a block, normed where there is a next weight
variable_list join_forward(const Tensor &residual, const Tensor &block, const Tensor &post, const Tensor &next,
                           const Tensor &gate, const Tensor &scale, const Tensor &rstd, double eps) {
  const c10::DeviceGuard guard(residual.device());
  variable_list out;
  Tensor joined, normed;
  if (block.defined()) out.push_back(joined = empty(residual, residual.sizes(), residual.scalar_type()));
  if (next.defined())
    out.push_back(normed = empty(residual, residual.sizes(), (block.defined() ? block : residual).scalar_type()));
  if (residual.size(0)) {
    astra_join_norm f = join_struct(residual, block, post, next, gate, scale, rstd, eps);
    f.joined = ptr(joined);
    f.normed = ptr(normed);
    check(astra_join_norm_forward(&f, stream_of(residual.get_device())));
  }
  return out;
}

struct JoinNorm : torch::autograd::Function<JoinNorm> {
  static variable_list forward(AutogradContext *ctx, const Tensor &residual, const Optional &block,
                               const Optional &post, const Optional &next, const Optional &gate, const Optional &scale,
                               double eps) {
    const Tensor rstd = empty(residual, {residual.size(0), 2}, torch::kFloat32);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({residual, value(block), value(post), value(next), value(gate), value(scale), rstd});
    ctx->saved_data["eps"] = eps;
    return join_forward(residual, value(block), value(post), value(next), value(gate), value(scale), rstd, eps);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    check_once();
    const auto s = ctx->get_saved_variables();
    variable_list out(7);
    Tensor djoined, dnormed;
    size_t at = 0;
    if (s[1].defined()) djoined = undefined_or_contiguous(grads[at++]);
    if (s[3].defined()) dnormed = undefined_or_contiguous(grads[at++]);
    if (!djoined.defined() && !dnormed.defined()) return out;
    const Tensor &residual = s[0];
    const c10::DeviceGuard guard(residual.device());
    const bool any = residual.size(0) > 0;
    for (int i = 0; i < 6; ++i)
      if (s[i].defined() && s[i].requires_grad()) {
        out[i] = empty(s[i], s[i].sizes(), s[i].scalar_type());
        if (!any) out[i].zero_();
      }
    if (!any) return out;
    astra_join_norm_grad g{};
    g.f = join_struct(residual, s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["eps"].toDouble());
    g.djoined = ptr(djoined);
    g.dnormed = ptr(dnormed);
    g.dresidual = ptr(out[0]);
    g.dblock = ptr(out[1]);
    g.dpost = ptr<float>(out[2]);
    g.dnext = ptr<float>(out[3]);
    g.dgate = ptr(out[4]);
    g.dscale = ptr<float>(out[5]);
    Tensor ws;
    if (g.dpost || g.dnext || g.dscale) {
      check(astra_join_norm_workspace_size(&g.f, &g.workspace_bytes));
      ws = workspace(residual, g.workspace_bytes);
      g.workspace = ptr(ws);
    }
    check(astra_join_norm_backward(&g, stream_of(residual.get_device())));
    return out;
  }
};

variable_list join(const Tensor &residual, const Tensor &block, const Tensor &post, const Tensor &next,
                   const Tensor &gate, const Tensor &scale, double eps) {
  return with_grad({&residual, &block, &post, &next, &gate, &scale})
             ? JoinNorm::apply(residual, maybe(block), maybe(post), maybe(next), maybe(gate), maybe(scale), eps)
             : join_forward(residual, block, post, next, gate, scale, Tensor(), eps);
}

void check_width(int64_t D) {
  need(D >= 1 && D <= ASTRA_SEQ_MAX_NORM_WIDTH, "width",
       "must be 1 to " + std::to_string(ASTRA_SEQ_MAX_NORM_WIDTH) + ", got " + std::to_string(D));
}

py::object join_norm(const Tensor &residual, const Tensor &block, const Tensor &post_, const Optional &next_,
                     const Optional &gate_, const Optional &scale_, double eps) {
  calls_only("join_norm", residual, block, post_, next_, gate_, scale_);
  check_data("block", block);
  check_data("residual", residual);
  need(residual.scalar_type() == block.scalar_type() || residual.scalar_type() == torch::kFloat32, "residual",
       std::string("must be ") + c10::toString(block.scalar_type()) + " or Float, got " + c10::toString(residual.scalar_type()));
  need(residual.device() == block.device(), "residual", "must be on " + block.device().str());
  need(block.dim() >= 1 && block.sizes() == residual.sizes(), "residual",
       "must have block's shape " + shape_text(block.sizes()) + ", got " + shape_text(residual.sizes()));
  const int64_t D = block.size(-1);
  check_width(D);
  Tensor gate;
  if (gate_) {
    std::vector<int64_t> one(block.sizes().begin(), block.sizes().end());
    one.back() = 1;
    check_like("gate", *gate_, block, gate_->dim() == block.dim() && gate_->size(-1) == 1 ? c10::IntArrayRef(one) : block.sizes());
    gate = flat(*gate_);
  }
  Tensor scale;
  if (scale_) {
    need(scale_->dim() == 1 && (scale_->size(0) == D || scale_->size(0) == 1), "scale",
         "must have shape [" + std::to_string(D) + "] or [1], got " + shape_text(scale_->sizes()));
    scale = param("scale", scale_, block, scale_->sizes());
  }
  const Tensor post = param("post_weight", post_, block, {D}), next = param("next_weight", next_, block, {D});
  const variable_list out = join(flat(residual), flat(block), post, next, gate, scale, eps);
  const Tensor joined = out[0].view(block.sizes());
  return next.defined() ? py::make_tuple(joined, out[1].view(block.sizes())) : py::make_tuple(joined, py::none());
}

Tensor rms_norm(const Tensor &x, const Tensor &weight_, double eps) {
  calls_only("rms_norm", x, weight_);
  check_data("x", x);
  need(x.dim() >= 1, "x", "must have at least one dimension");
  const int64_t D = x.size(-1);
  check_width(D);
  return join(flat(x), {}, {}, param("weight", weight_, x, {D}), {}, {}, eps)[0].view(x.sizes());
}

}  // namespace

void bind_sequence(py::module_ &m) {
  py::module_ s = m.def_submodule("sequence", "Sequence operators (astra_cuda.sequence documents them)");
  s.def("short_conv", &short_conv, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("activation"),
        py::arg("initial_state"), py::arg("lengths"), py::arg("return_state"));
  s.def("short_conv_step", &short_conv_step, py::arg("x"), py::arg("state"), py::arg("weight"), py::arg("bias"),
        py::arg("activation"));
  s.def("state_scan", &state_scan, py::arg("x"), py::arg("dt"), py::arg("A"), py::arg("B"), py::arg("C"), py::arg("D"),
        py::arg("dt_bias"), py::arg("initial_state"), py::arg("lengths"), py::arg("return_state"));
  s.def("state_scan_step", &state_scan_step, py::arg("x"), py::arg("dt"), py::arg("A"), py::arg("B"), py::arg("C"),
        py::arg("state"), py::arg("D"), py::arg("dt_bias"));
  s.def("join_norm", &join_norm, py::arg("residual"), py::arg("block"), py::arg("post_weight"), py::arg("next_weight"),
        py::arg("gate"), py::arg("scale"), py::arg("eps"));
  s.def("rms_norm", &rms_norm, py::arg("x"), py::arg("weight"), py::arg("eps"));
  s.attr("MAX_TAPS") = ASTRA_SEQ_MAX_TAPS;
  s.attr("MAX_STATE") = ASTRA_SEQ_MAX_STATE;
  s.attr("MAX_NORM_WIDTH") = ASTRA_SEQ_MAX_NORM_WIDTH;
}

}  // namespace astra_bind
