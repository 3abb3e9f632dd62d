// Host side of the state space mixer's operators (mixer_ops.py): argument checks, output allocation, the descriptor and the launch of one call, and the
// autograd node, without the interpreter.  A call through Python and ctypes costs the host 10 - 15 us and its backward, which autograd runs on a thread of
// its own, 100 us more; that is longer than the kernels of a night need.  Every function returns None where an argument is not as it should be: the
// caller then finds out which one and raises.  The kernels' entry points are handed over as addresses (bind), so that the library is loaded once, by lib.py.
#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../../include/w2s.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Opt;

struct {
  int (*conv_fwd)(const w2s_short_conv_args*, void*);
  int64_t (*conv_part)(const w2s_short_conv_args*);
  int (*conv_bwd)(const w2s_short_conv_args*, void*);
  int (*conv_step)(const w2s_short_conv_args*, void*);
  int64_t (*ssm_ckpt)(const w2s_ssm_args*);
  int64_t (*ssm_ws)(const w2s_ssm_args*, int);
  int (*ssm_fwd)(const w2s_ssm_args*, void*);
  int (*ssm_bwd)(const w2s_ssm_args*, void*);
  int (*ssm_step)(const w2s_ssm_args*, void*);
  int (*norm_fwd)(const w2s_add_norm_args*, void*);
  int64_t (*norm_part)(const w2s_add_norm_args*);
  int (*norm_bwd)(const w2s_add_norm_args*, void*);
} entry;

struct Failure : std::runtime_error {   // lib.W2SError in Python
  using std::runtime_error::runtime_error;
};
PyObject* failure_type = nullptr;

void bind(const std::vector<uint64_t>& at, const py::object& error) {
  TORCH_CHECK(at.size() * sizeof(void*) == sizeof entry, "w2s: ", at.size(), " entry points");
  memcpy(&entry, at.data(), sizeof entry);
  Py_XDECREF(failure_type);
  failure_type = error.inc_ref().ptr();
}

void* stream(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void done(int rc, const char* what) {
  if (rc != 0) throw Failure(std::string(what) + " failed with code " + std::to_string(rc) + (rc == W2S_EINVAL ? " (EINVAL)" : rc == W2S_ELAUNCH ? " (ELAUNCH)" : ""));
}
int64_t size(int64_t n, const char* what) {
  if (n < 0) throw Failure(std::string(what) + " failed with code " + std::to_string(n));
  return n;
}

int code(const Tensor& t) {   // W2S_F32 / W2S_BF16 / W2S_F16, or -1
  switch (t.scalar_type()) {
    case at::kFloat: return W2S_F32;
    case at::kBFloat16: return W2S_BF16;
    case at::kHalf: return W2S_F16;
    default: return -1;
  }
}
bool is(const Tensor& t, const Tensor& ref, at::ScalarType type, at::IntArrayRef shape) {
  return t.defined() && t.scalar_type() == type && t.device() == ref.device() && t.sizes() == shape && t.layout() == at::kStrided;
}
bool is(const Opt& t, const Tensor& ref, at::ScalarType type, at::IntArrayRef shape) { return !t || is(*t, ref, type, shape); }
bool sized(const Tensor& t) {   // every size within 2^30: the descriptors hold 32-bit sizes, the kernels' positions run a tile past them
  for (const int64_t n : t.sizes())
    if (n > (1 << 30)) return false;
  return true;
}
// jit.trace, make_fx and export record dispatched operators: they would keep a result's allocation and not the launch that fills it
bool traced() {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer)) return true;
  return TorchDispatchModeTLS::any_modes_set() && (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE));
}
bool io(const Tensor& t, int64_t dim) { return t.defined() && t.is_cuda() && t.layout() == at::kStrided && code(t) >= 0 && t.dim() == dim && sized(t); }

// A tensor's values may not be what lies at its address: a view that stands for the negative (part of a conjugate), a zero without memory
bool lies(const Tensor& t) { return !t.is_neg() && !t._is_zerotensor(); }
Tensor lying(const Tensor& t) { return lies(t) ? t : t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.resolve_neg(); }
Tensor rows_of(const Tensor& t) {   // contiguous last dimension
  const Tensor r = lying(t);
  return r.size(-1) <= 1 || r.stride(-1) == 1 ? r : r.contiguous();
}
// ... and positions less than 2^22 elements apart, as a scan's kernels want them (32-bit offsets inside a tile); a gradient's layout is not the caller's choice
Tensor near_rows(const Tensor& t) {
  const Tensor r = rows_of(t);
  return r.size(1) <= 1 || r.stride(1) < (1 << 22) ? r : r.clone(at::MemoryFormat::Contiguous);
}
int64_t position_stride(const Tensor& t) { return t.defined() && t.size(1) > 1 ? t.stride(1) : 0; }
Tensor plain(const Tensor& t) { return lying(t).contiguous(); }
Tensor plain(const Opt& t) { return t ? plain(*t) : Tensor(); }
Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor like_if(const Tensor& t) { return t.defined() ? like(t) : Tensor(); }
template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
bool wants(const Opt& t) { return t && t->requires_grad(); }
template <typename... Ts> bool graph(const Ts&... t) { return at::GradMode::is_enabled() && (wants(t) || ...); }
// a tangent of forward-mode differentiation: no kernel here carries one on, and a result without it would be a derivative of 0
bool tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool tangent(const Opt& t) { return t && tangent(*t); }
template <typename... Ts> bool forward_mode(const Ts&... t) { return c10::AutogradState::get_tls_state().get_fw_grad_mode() && (tangent(t) || ...); }
void no_forward_mode(const variable_list& g) {   // of gradients that arrive at a node
  for (const Tensor& t : g)
    if (forward_mode(t)) throw Failure("this operator's gradient has no forward-mode derivative: a gradient that arrived carries a tangent");
}

// A capture cannot take in the default stream, and torch hands a leaf's gradient over on the stream where the leaf first came into a graph that still lives: a
// backward that is captured while an eager graph of the same leaves lives ends the process inside the engine.  It is refused here, in front of that.
void no_captured_eager_leaf() {
  const auto node = torch::autograd::get_current_node();
  for (size_t i = 0; node && i < node->num_outputs(); ++i) {
    const auto& to = node->next_edge(i).function;
    if (!to || !node->task_should_compute_output(i) || !dynamic_cast<torch::autograd::AccumulateGrad*>(to.get())) continue;
    const auto on = to->stream();
    if (on && on->id() == 0 && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
      throw Failure("a backward cannot be captured while an eager graph of the same leaves lives: drop that graph, or use detached leaves");
  }
}

// The gradients are kernels' results: a graph through them (create_graph) has to end in an error, not in a constant
variable_list first_order(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in, out(grads.size());
  for (auto& g : grads)
    if (g.defined()) in.push_back(g.detach().requires_grad_(true));
  auto node = std::make_shared<torch::autograd::DelayedError>("this operator's gradient is not differentiable", (int64_t)in.size());
  auto marked = (*node)(std::move(in));
  size_t k = 0;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) out[i] = marked[k++];
  return out;
}

// ------------------------------------------------------------------------------------------------------------------ short convolution
w2s_short_conv_args conv_args(const Tensor& x, const Tensor& w, const Tensor& bias, int64_t act, const Tensor& state, const Tensor& lengths) {
  w2s_short_conv_args a{};
  a.x = ptr(x);
  a.w = ptr<float>(w);
  a.bias = ptr<float>(bias);
  a.state = ptr(state);
  a.lengths = ptr<int32_t>(lengths);
  const bool step = x.dim() == 2;
  a.B = (int32_t)x.size(0);
  a.L = step ? 1 : (int32_t)x.size(1);
  a.D = (int32_t)x.size(-1);
  a.K = (int32_t)w.size(1);
  a.sx_b = x.stride(0);
  a.sx_l = step ? 0 : x.stride(1);
  a.dtype = code(x);
  a.act = (int32_t)act;
  return a;
}

void conv_forward(w2s_short_conv_args& a, const Tensor& x, bool want_state, Tensor& y, Tensor& last) {
  const c10::DeviceGuard guard(x.device());
  y = like(x);
  a.y = ptr(y);
  if (want_state) {
    last = at::empty({x.size(0), a.K - 1, x.size(2)}, x.options());
    a.state_out = ptr(last);
  }
  done(entry.conv_fwd(&a, stream(x)), "w2s_short_conv_fwd");
}

struct ShortConv : torch::autograd::Function<ShortConv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const Opt& bias_, const Opt& state_, const Opt& lengths_, int64_t act, bool want_state) {
    const Tensor x = rows_of(x_), w = plain(w_), bias = plain(bias_), state = plain(state_), lengths = plain(lengths_);
    auto a = conv_args(x, w, bias, act, state, lengths);
    Tensor y, last;
    conv_forward(a, x, want_state, y, last);
    ctx->save_for_backward({x, w, bias, state, lengths});
    ctx->saved_data["k"] = act << 4 | (int64_t)x_.requires_grad() | (int64_t)(w_.requires_grad() || wants(bias_)) << 1 | (int64_t)wants(state_) << 2;
    ctx->set_materialize_grads(false);
    return want_state ? variable_list{y, last} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_forward_mode(g);
    no_captured_eager_leaf();
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &bias = s[2], &state = s[3], &lengths = s[4];
    const int64_t k = ctx->saved_data["k"].toInt();
    const bool need_x = k & 1, need_w = k & 2, need_s = k & 4;
    Tensor gx, gw, gb, gs;
    {
      const at::AutoGradMode off(false);
      const c10::DeviceGuard guard(x.device());
      Tensor gy = g[0].defined() ? rows_of(g[0]) : Tensor(), gl = g.size() > 1 && g[1].defined() ? plain(g[1]) : Tensor();
      if (need_s) gs = like(state);
      if (x.size(0) == 0 || x.size(1) == 0) {   // no positions: nothing but the state's rows, which pass through
        gx = like(x);
        gw = at::zeros_like(w);
        if (bias.defined()) gb = at::zeros_like(bias);
        if (need_s) gl.defined() ? gs.copy_(gl) : gs.zero_();
      } else {
        auto a = conv_args(x, w, bias, k >> 4, state, lengths);
        gx = like(x);
        a.gy = ptr(gy);
        if (gy.defined()) {
          a.sg_b = gy.stride(0);
          a.sg_l = gy.stride(1);
        }
        a.gstate = ptr(gl);
        a.gx = ptr(gx);
        a.gstate_in = ptr(gs);
        Tensor part;
        if (need_w) {
          gw = like(w);
          gb = like_if(bias);
          part = at::empty({size(entry.conv_part(&a), "w2s_short_conv_part")}, w.options());
          a.gw = ptr<float>(gw);
          a.gbias = ptr<float>(gb);
          a.part = ptr<float>(part);
        }
        done(entry.conv_bwd(&a, stream(x)), "w2s_short_conv_bwd");
      }
    }
    return first_order({need_x ? gx : Tensor(), need_w ? gw : Tensor(), need_w ? gb : Tensor(), gs, Tensor(), Tensor(), Tensor()});
  }
};

bool conv_ok(const Tensor& x, const Tensor& w, const Opt& bias, const Opt& state, int64_t dim) {
  if (!io(x, dim) || !w.defined() || w.dim() != 2 || traced()) return false;
  const int64_t D = x.size(-1), K = w.size(1);
  return D >= 1 && K >= 1 && K <= 8 && is(w, x, at::kFloat, {D, K}) && is(bias, x, at::kFloat, {D}) && is(state, x, x.scalar_type(), {x.size(0), K - 1, D});
}

py::object pair_or_one(const Tensor& y, const Tensor& last, bool both) { return both ? py::object(py::make_tuple(y, last)) : py::cast(y); }

py::object short_conv(const Tensor& x, const Tensor& w, const Opt& bias, int64_t act, const Opt& state, const Opt& lengths, bool want_state) {
  if (!conv_ok(x, w, bias, state, 3) || !is(lengths, x, at::kInt, {x.size(0)}) || forward_mode(x, w, bias, state)) return py::none();
  Tensor y, last;
  {
    const py::gil_scoped_release free;
    if (graph(Opt(x), Opt(w), bias, state)) {
      auto out = ShortConv::apply(x, w, bias, state, lengths, act, want_state);
      y = out[0];
      if (want_state) last = out[1];
    } else {
      const Tensor xr = rows_of(x), wc = plain(w), bc = plain(bias), sc = plain(state), lc = plain(lengths);
      auto a = conv_args(xr, wc, bc, act, sc, lc);
      conv_forward(a, xr, want_state, y, last);
    }
  }
  return pair_or_one(y, last, want_state);
}

// where a step may leave its state: another tensor than the one it reads only where the two do not overlap
bool step_state_ok(const Tensor& state, const Tensor& out) {
  if (!state.is_contiguous() || !out.is_contiguous() || !lies(state) || !lies(out) || out.requires_grad()) return false;
  const char *a = (const char*)state.data_ptr(), *b = (const char*)out.data_ptr();
  const int64_t n = state.numel() * state.element_size();
  return a == b || a + n <= b || b + n <= a;
}

py::object short_conv_step(const Tensor& x, const Tensor& state, const Tensor& w, const Opt& bias, int64_t act, const Opt& state_out) {
  if (!conv_ok(x, w, bias, state, 2) || graph(Opt(x), Opt(state), Opt(w), bias) || forward_mode(x, state, w, bias, state_out)) return py::none();
  const Tensor& out = state_out ? *state_out : state;
  if (!is(out, x, x.scalar_type(), state.sizes()) || !step_state_ok(state, out)) return py::none();
  const c10::DeviceGuard guard(x.device());
  const Tensor xr = rows_of(x), wc = plain(w), bc = plain(bias), y = like(xr);
  auto a = conv_args(xr, wc, bc, act, state, Tensor());
  a.y = ptr(y);
  a.state_out = ptr(out);
  out.unsafeGetTensorImpl()->bump_version();
  done(entry.conv_step(&a, stream(x)), "w2s_short_conv_step");
  return py::cast(y);
}

// ------------------------------------------------------------------------------------------------------------------ selective scan
struct Ssm {
  Tensor u, dt, A, B, C, D, z, bias, state, lengths;
};

w2s_ssm_args ssm_args(const Ssm& s, int64_t softplus) {
  w2s_ssm_args a{};
  const bool step = s.u.dim() == 2;
  a.u = ptr(s.u);
  a.dt = ptr(s.dt);
  a.z = ptr(s.z);
  a.Bm = ptr(s.B);
  a.Cm = ptr(s.C);
  a.A = ptr<float>(s.A);
  a.Dp = ptr<float>(s.D);
  a.dt_bias = ptr<float>(s.bias);
  a.h0 = ptr<float>(s.state);
  a.lengths = ptr<int32_t>(s.lengths);
  a.su_b = s.u.stride(0);
  a.sdt_b = s.dt.stride(0);
  a.sz_b = s.z.defined() ? s.z.stride(0) : 0;
  a.sB_b = s.B.stride(0);
  a.sC_b = s.C.stride(0);
  if (!step) {
    a.su_l = position_stride(s.u);
    a.sdt_l = position_stride(s.dt);
    a.sz_l = position_stride(s.z);
    a.sB_l = position_stride(s.B);
    a.sC_l = position_stride(s.C);
  }
  a.sB_g = s.B.stride(-2);
  a.sC_g = s.C.stride(-2);
  a.B = (int32_t)s.u.size(0);
  a.L = step ? 1 : (int32_t)s.u.size(1);
  a.D = (int32_t)s.u.size(-1);
  a.N = (int32_t)s.A.size(1);
  a.G = (int32_t)s.B.size(-2);
  a.dtype = code(s.u);
  a.softplus = (int32_t)softplus;
  return a;
}

void scan_forward(const Ssm& s, int64_t softplus, bool want_state, bool train, Tensor& y, Tensor& last, Tensor& ckpt) {
  const c10::DeviceGuard guard(s.u.device());
  auto a = ssm_args(s, softplus);
  y = like(s.u);
  a.y = ptr(y);
  if (want_state) {
    last = at::empty({s.u.size(0), s.u.size(2), s.A.size(1)}, s.A.options());
    a.h_out = ptr<float>(last);
  }
  if (train) {
    ckpt = at::empty({size(entry.ssm_ckpt(&a), "w2s_ssm_ckpt")}, s.A.options());
    a.ckpt = ptr<float>(ckpt);
  }
  Tensor ws;
  if (const int64_t n = size(entry.ssm_ws(&a, 0), "w2s_ssm_ws")) {
    ws = at::empty({n / 4}, s.A.options());
    a.ws = ptr(ws);
  }
  done(entry.ssm_fwd(&a, stream(s.u)), "w2s_ssm_scan_fwd");
}

struct SsmScan : torch::autograd::Function<SsmScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D, const Opt& z,
                               const Opt& bias, const Opt& state, const Opt& lengths, int64_t softplus, bool want_state) {
    const Ssm s{rows_of(u), rows_of(dt), plain(A), rows_of(B), rows_of(C), plain(D), z ? rows_of(*z) : Tensor(), plain(bias), plain(state), plain(lengths)};
    Tensor y, last, ckpt;
    scan_forward(s, softplus, want_state, true, y, last, ckpt);
    ctx->save_for_backward({s.u, s.dt, s.A, s.B, s.C, s.D, s.z, s.bias, s.state, s.lengths, ckpt});
    int64_t k = softplus << 16, bit = 1;
    for (const Opt& t : {Opt(u), Opt(dt), Opt(A), Opt(B), Opt(C), D, z, bias, state}) {
      if (wants(t)) k |= bit;
      bit <<= 1;
    }
    ctx->saved_data["k"] = k;
    ctx->set_materialize_grads(false);
    return want_state ? variable_list{y, last} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_forward_mode(g);
    no_captured_eager_leaf();
    const auto v = ctx->get_saved_variables();
    const Ssm s{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9]};
    const int64_t k = ctx->saved_data["k"].toInt();
    variable_list out(12);
    {
      const at::AutoGradMode off(false);
      const c10::DeviceGuard guard(s.u.device());
      auto a = ssm_args(s, k >> 16);
      Tensor gy = g[0].defined() ? near_rows(g[0]) : Tensor(), gl = g.size() > 1 && g[1].defined() ? plain(g[1]) : Tensor();
      a.gy = ptr(gy);
      if (gy.defined()) {
        a.sg_b = gy.stride(0);
        a.sg_l = position_stride(gy);
      }
      a.gh = ptr<float>(gl);
      a.ckpt = ptr<float>(v[10]);
      const Tensor gu = like(s.u), gdt = like(s.dt), gA = like(s.A), gB = like(s.B), gC = like(s.C), gD = like_if(s.D), gz = like_if(s.z), gb = like_if(s.bias),
                   gs = like_if(s.state);
      a.gu = ptr(gu);
      a.gdt = ptr(gdt);
      a.gz = ptr(gz);
      a.gB = ptr(gB);
      a.gC = ptr(gC);
      a.gA = ptr<float>(gA);
      a.gD = ptr<float>(gD);
      a.gbias = ptr<float>(gb);
      a.gh0 = ptr<float>(gs);
      const Tensor ws = at::empty({std::max<int64_t>(1, size(entry.ssm_ws(&a, 1), "w2s_ssm_ws") / 4)}, s.A.options());
      a.ws = ptr(ws);
      done(entry.ssm_bwd(&a, stream(s.u)), "w2s_ssm_scan_bwd");
      const Tensor all[9] = {gu, gdt, gA, gB, gC, gD, gz, gb, gs};
      for (int i = 0; i < 9; ++i)
        if (k >> i & 1) out[i] = all[i];
    }
    return first_order(std::move(out));
  }
};

bool ssm_ok(const Tensor& u, const Tensor& dt, const Tensor& A, Tensor& B, Tensor& C, const Opt& D, const Opt& z, const Opt& bias, const Opt& state, int64_t dim) {
  if (!io(u, dim) || !A.defined() || A.dim() != 2 || !B.defined() || !C.defined() || traced()) return false;
  if (B.dim() == dim) B = B.unsqueeze(-2);
  if (C.dim() == dim) C = C.unsqueeze(-2);
  if (B.dim() != dim + 1) return false;
  const int64_t nb = u.size(0), Dc = u.size(-1), N = A.size(1), G = B.size(-2);
  if (N < 1 || N > 64 || Dc < 1 || G < 1 || Dc % G) return false;
  const auto t = u.scalar_type();
  const int64_t one[3] = {nb, G, N}, seq[4] = {nb, dim == 3 ? u.size(1) : 0, G, N};
  const at::IntArrayRef bc = dim == 3 ? at::IntArrayRef(seq, 4) : at::IntArrayRef(one, 3);
  return is(dt, u, t, u.sizes()) && is(z, u, t, u.sizes()) && is(A, u, at::kFloat, {Dc, N}) && is(B, u, t, bc) && is(C, u, t, bc) && is(D, u, at::kFloat, {Dc}) &&
         is(bias, u, at::kFloat, {Dc}) && is(state, u, at::kFloat, {nb, Dc, N});
}

py::object ssm_scan(const Tensor& u, const Tensor& dt, const Tensor& A, Tensor B, Tensor C, const Opt& D, const Opt& z, const Opt& bias, bool softplus, const Opt& state,
                    const Opt& lengths, bool want_state) {
  if (!ssm_ok(u, dt, A, B, C, D, z, bias, state, 3) || !is(lengths, u, at::kInt, {u.size(0)}) || forward_mode(u, dt, A, B, C, D, z, bias, state)) return py::none();
  for (const Opt& t : {Opt(u), Opt(dt), Opt(B), Opt(C), z})
    if (t && position_stride(*t) >= (1 << 22)) return py::none();
  Tensor y, last;
  {
    const py::gil_scoped_release free;
    if (graph(Opt(u), Opt(dt), Opt(A), Opt(B), Opt(C), D, z, bias, state)) {
      auto out = SsmScan::apply(u, dt, A, B, C, D, z, bias, state, lengths, (int64_t)softplus, want_state);
      y = out[0];
      if (want_state) last = out[1];
    } else {
      Tensor ckpt;
      const Ssm s{rows_of(u), rows_of(dt), plain(A), rows_of(B), rows_of(C), plain(D), z ? rows_of(*z) : Tensor(), plain(bias), plain(state), plain(lengths)};
      scan_forward(s, softplus, want_state, false, y, last, ckpt);
    }
  }
  return pair_or_one(y, last, want_state);
}

py::object ssm_step(const Tensor& u, const Tensor& dt, const Tensor& A, Tensor B, Tensor C, const Tensor& state, const Opt& D, const Opt& z, const Opt& bias, bool softplus,
                    const Opt& state_out) {
  if (!ssm_ok(u, dt, A, B, C, D, z, bias, state, 2) || graph(Opt(u), Opt(dt), Opt(A), Opt(B), Opt(C), Opt(state), D, z, bias) ||
      forward_mode(u, dt, A, B, C, state, D, z, bias, state_out))
    return py::none();
  const Tensor& out = state_out ? *state_out : state;
  if (!is(out, u, at::kFloat, state.sizes()) || !step_state_ok(state, out)) return py::none();
  const c10::DeviceGuard guard(u.device());
  const Ssm s{rows_of(u), rows_of(dt), plain(A), rows_of(B), rows_of(C), plain(D), z ? rows_of(*z) : Tensor(), plain(bias), state, Tensor()};
  const Tensor y = like(s.u);
  auto a = ssm_args(s, softplus);
  a.y = ptr(y);
  a.h_out = ptr<float>(out);
  out.unsafeGetTensorImpl()->bump_version();
  done(entry.ssm_step(&a, stream(u)), "w2s_ssm_step");
  return py::cast(y);
}

// ------------------------------------------------------------------------------------------------------------------ norm with the residual's addition
Tensor flat(const Tensor& t, int64_t C) {   // [rows, C] with contiguous rows, a view where the strides allow one
  if (!t.defined()) return t;
  const Tensor r = rows_of(t);
  return r.dim() == 2 ? r : r.reshape({-1, C});
}

void norm_forward(const Tensor& x, const Tensor& w, const Tensor& res, double eps, bool fp8, bool want_rstd, Tensor& y, Tensor& r, Tensor& scale, Tensor& rstd) {
  const c10::DeviceGuard guard(x.device());
  const int64_t C = x.size(-1), rows = x.numel() / C;
  const Tensor x2 = flat(x, C), r2 = flat(res, C);
  w2s_add_norm_args a{};
  a.x = ptr(x2);
  a.w = ptr<float>(w);
  a.rows = rows;
  a.C = (int32_t)C;
  a.dtype = a.rdtype = code(x);
  a.eps = (float)eps;
  a.fp8 = fp8;
  a.ldx = x2.stride(0);
  y = at::empty(x.sizes(), fp8 ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
  a.y = ptr(y);
  if (res.defined()) {
    r = like(res);
    a.res = ptr(r2);
    a.r = ptr(r);
    a.ldres = r2.stride(0);
    a.rdtype = code(res);
  }
  if (fp8) {
    scale = at::empty(x.sizes().slice(0, x.dim() - 1), w.options());
    a.scale = ptr<float>(scale);
  }
  if (want_rstd) {
    rstd = at::empty({rows}, w.options());
    a.rstd = ptr<float>(rstd);
  }
  done(entry.norm_fwd(&a, stream(x)), "w2s_add_norm_fwd");
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_, const Opt& res_, double eps) {
    const Tensor w = plain(w_), res = res_ ? *res_ : Tensor();
    Tensor y, r, scale, rstd;
    norm_forward(x, w, res, eps, false, true, y, r, scale, rstd);
    // the backward needs the sum as it was normalised: r where that is exact (fp32), else the two addends again
    const bool exact = res.defined() && r.scalar_type() == at::kFloat;
    ctx->save_for_backward({exact ? Tensor() : x, exact ? r : res, w, rstd});
    ctx->saved_data["k"] = (int64_t)x.scalar_type() << 4 | (int64_t)x.requires_grad() | (int64_t)w_.requires_grad() << 1 | (int64_t)wants(res_) << 2;
    ctx->set_materialize_grads(false);
    return res.defined() ? variable_list{y, r} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_forward_mode(g);
    no_captured_eager_leaf();
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &res = s[1], &w = s[2], &rstd = s[3], &first = x.defined() ? x : res;
    const int64_t k = ctx->saved_data["k"].toInt(), C = w.size(0);
    const auto xt = (at::ScalarType)(k >> 4);
    const bool need_x = k & 1, need_w = k & 2, need_r = k & 4, one_type = !res.defined() || res.scalar_type() == xt;
    Tensor gx, gres, gw;
    {
      const at::AutoGradMode off(false);
      const c10::DeviceGuard guard(first.device());
      const Tensor x2 = flat(x, C), r2 = flat(res, C), gy = flat(g[0], C), gr = g.size() > 1 ? flat(g[1], C) : Tensor();
      auto ld = [](const Tensor& t) { return t.defined() ? t.stride(0) : 0; };
      if (need_x || (need_r && one_type)) gx = at::empty(first.sizes(), first.options().dtype(xt));
      if (need_r && !one_type) gres = like(res);
      w2s_add_norm_args a{};
      a.x = ptr(x2);
      a.res = ptr(r2);
      a.w = ptr<float>(w);
      a.rstd = ptr<float>(rstd);
      a.gy = ptr(gy);
      a.gr = ptr(gr);
      a.gx = ptr(gx);
      a.gres = ptr(gres);
      a.rows = rstd.size(0);
      a.C = (int32_t)C;
      a.ldx = ld(x2);
      a.ldres = ld(r2);
      a.ldgy = ld(gy);
      a.ldgr = ld(gr);
      a.dtype = xt == at::kFloat ? W2S_F32 : xt == at::kBFloat16 ? W2S_BF16 : W2S_F16;
      a.rdtype = one_type ? a.dtype : W2S_F32;
      Tensor part;
      if (need_w) {
        gw = like(w);
        part = at::empty({size(entry.norm_part(&a), "w2s_add_norm_part")}, w.options());
        a.gw = ptr<float>(gw);
        a.part = ptr<float>(part);
      }
      done(entry.norm_bwd(&a, stream(first)), "w2s_add_norm_bwd");
    }
    const Tensor& both = one_type ? gx : gres;   // of one type, both addends have the same gradient
    return first_order({need_x ? gx : Tensor(), gw, need_r ? both : Tensor(), Tensor()});
  }
};

bool norm_ok(const Tensor& x, const Tensor& w, const Opt& res, double eps) {
  if (!x.defined() || !x.is_cuda() || code(x) < 0 || x.layout() != at::kStrided || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > (1 << 30) || x.numel() / x.size(-1) > 0x7fffffff || !(eps >= 0.0))
    return false;
  return !traced() && is(w, x, at::kFloat, {x.size(-1)}) && (!res || is(*res, x, x.scalar_type(), x.sizes()) || is(*res, x, at::kFloat, x.sizes()));
}

py::object add_rms_norm(const Tensor& x, const Tensor& w, const Opt& res, double eps) {
  if (!norm_ok(x, w, res, eps) || forward_mode(x, w, res)) return py::none();
  Tensor y, r, scale, rstd;
  {
    const py::gil_scoped_release free;
    if (graph(Opt(x), Opt(w), res)) {
      auto out = AddRmsNorm::apply(x, w, res, eps);
      y = out[0];
      if (res) r = out[1];
    } else {
      norm_forward(x, plain(w), res ? *res : Tensor(), eps, false, false, y, r, scale, rstd);
    }
  }
  return py::make_tuple(y, res ? r : x);
}

py::object add_rms_norm_8bit(const Tensor& x, const Tensor& w, const Opt& res, double eps) {
  if (!norm_ok(x, w, res, eps) || graph(Opt(x), Opt(w), res) || forward_mode(x, w, res)) return py::none();
  Tensor y, r, scale, rstd;
  norm_forward(x, plain(w), res ? *res : Tensor(), eps, true, false, y, r, scale, rstd);
  return py::make_tuple(y, scale, res ? r : x);
}

}  // namespace

PYBIND11_MODULE(_w2s_torch, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure& e) {
      PyErr_SetString(failure_type ? failure_type : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("traced", &traced);
  m.def("short_conv", &short_conv);
  m.def("short_conv_step", &short_conv_step);
  m.def("ssm_scan", &ssm_scan);
  m.def("ssm_step", &ssm_step);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("add_rms_norm_8bit", &add_rms_norm_8bit);
}
