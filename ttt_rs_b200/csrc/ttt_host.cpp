// Native host path between the Python operator and the C ABI (include/ttt_b200.h): argument checks, output and workspace
// allocation, stream lookup and the launch of one call without returning to the interpreter, and the autograd nodes of
// the two inner loops.
//
// Why it exists: through ctypes a call costs 20 us (one-token step of the TTT-Linear inner model, whose kernel takes 4 us)
// to 300 us (forward + backward through a Python autograd function) of interpreter time; here it costs 4 to 40 us.
//
// Every function takes what the call needs and returns its results, or None where the arguments are not the plain case
// (not contiguous, another dtype or shape, not on a GPU, an error code from the library): the Python code then walks
// through its own checks, which convert or raise.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/autocast_mode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/torch.h>

#include "../../include/ttt_b200.h"
#include "ttt_internal.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int kMaxDevices = 64;
Tensor g_status[kMaxDevices];   // the status words of each device, handed over by the Python side when it creates them
PyObject* g_error_type = nullptr;  // TttError(code, message)

[[noreturn]] void throw_error(int rc, const char* message = nullptr) {
  pybind11::gil_scoped_acquire gil;
  PyObject* args = Py_BuildValue("(is)", rc, message != nullptr ? message : ttt_b200_last_error());
  PyObject* exc = args ? PyObject_CallObject(g_error_type, args) : nullptr;
  Py_XDECREF(args);
  if (exc) {
    PyErr_SetObject(g_error_type, exc);
    Py_DECREF(exc);
  }
  throw python_error();
}

bool on_16_bytes(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }
bool is(const Tensor& t, at::ScalarType dt, const c10::Device& dev, c10::IntArrayRef sizes) {
  return t.defined() && t.is_cuda() && t.device() == dev && t.scalar_type() == dt && t.sizes() == sizes &&
         t.is_contiguous() && t.layout() == c10::kStrided;
}

struct Dims {
  ttt_dims d;
  int64_t B, H, T, F;
  at::ScalarType dt = at::kBFloat16;
  c10::Device dev = c10::Device(c10::kCPU);
  Tensor status;
  // false: not the plain case
  bool set(const Tensor& xq, int64_t head_dim, int64_t mb, int64_t K, int64_t eps_scaled) {
    if (!xq.defined() || !xq.is_cuda() || xq.dim() != 4 || mb <= 0) return false;
    dt = xq.scalar_type();
    if (dt != at::kBFloat16 && dt != at::kFloat) return false;
    dev = xq.device();
    B = xq.size(0), H = xq.size(1), T = xq.size(2), F = xq.size(3);
    if (F != head_dim || dev.index() >= kMaxDevices || B > INT32_MAX || H > INT32_MAX || T > INT32_MAX) return false;
    status = g_status[dev.index()];
    d.batch = (int32_t)B;
    d.heads = (int32_t)H;
    d.seq_len = (int32_t)T;
    d.head_dim = (int32_t)F;
    d.mini_batch = (int32_t)mb;
    d.checkpoint_interval = (int32_t)K;
    d.epsilon = (float)eps_scaled * 1e-9f;  // float32 arithmetic, as FusedTttConfig.epsilon
    d.dtype = dt == at::kBFloat16 ? TTT_BF16 : TTT_F32;
    return true;
  }
  at::TensorOptions opt() const { return at::TensorOptions().dtype(dt).device(dev); }
  at::TensorOptions opt(at::ScalarType t) const { return at::TensorOptions().dtype(t).device(dev); }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
};

struct LinIn {  // xq, xk, xv, weight, bias, token_eta, ttt_lr_eta, ln_weight, ln_bias
  Tensor t[9];
  bool plain(const Dims& m) const {
    const int64_t B = m.B, H = m.H, T = m.T, F = m.F;
    return is(t[0], m.dt, m.dev, {B, H, T, F}) && is(t[1], m.dt, m.dev, {B, H, T, F}) &&
           is(t[2], m.dt, m.dev, {B, H, T, F}) && is(t[3], m.dt, m.dev, {B, H, F, F}) && is(t[4], m.dt, m.dev, {B, H, F}) &&
           is(t[5], m.dt, m.dev, {T}) && is(t[6], m.dt, m.dev, {B, H, T}) && is(t[7], m.dt, m.dev, {H, F}) &&
           is(t[8], m.dt, m.dev, {H, F});
  }
  const void* p(int i) const { return t[i].const_data_ptr(); }
};

// ---- TTT-Linear --------------------------------------------------------------------------------------------------
struct LinOut {
  Tensor out, w, b, wck, bck;
};
int linear_forward(const Dims& m, const LinIn& in, bool save, LinOut& o) {
  c10::cuda::CUDAGuard guard(m.dev);
  if (save) {
    const size_t wb = ttt_linear_weight_ckpt_bytes(&m.d), bb = ttt_linear_bias_ckpt_bytes(&m.d);
    if (wb == 0 || bb == 0) return TTT_ERR_SHAPE;
    o.wck = at::empty({(int64_t)(wb / (64 * 64 * 4)), 64, 64}, m.opt(at::kFloat));
    o.bck = at::empty({(int64_t)bb}, m.opt(at::kByte));
  }
  o.out = at::empty({m.B, m.H, m.T, m.F}, m.opt());
  o.w = at::empty({m.B, m.H, m.F, m.F}, m.opt());
  o.b = at::empty({m.B, m.H, m.F}, m.opt());
  return ttt_linear_forward(&m.d, in.p(0), in.p(1), in.p(2), in.p(3), in.p(4), in.p(5), in.p(6), in.p(7), in.p(8),
                            o.out.data_ptr(), o.w.data_ptr(), o.b.data_ptr(), save ? o.wck.data_ptr() : nullptr,
                            save ? o.bck.data_ptr() : nullptr, m.status.data_ptr(), m.stream());
}

// gradients in the order of the inputs
int linear_backward(const Dims& m, const LinIn& in, const Tensor& wck, const Tensor& bck, const Tensor& go,
                    const Tensor& gw_out, const Tensor& gb_out, const Tensor& packed, Tensor (&g)[9]) {
  c10::cuda::CUDAGuard guard(m.dev);
  const size_t wsb = ttt_linear_backward_workspace_bytes(&m.d);
  if (wsb == 0) return TTT_ERR_SHAPE;
  for (int i = 0; i < 3; ++i) g[i] = at::empty({m.B, m.H, m.T, m.F}, m.opt());
  g[3] = at::empty({m.B, m.H, m.F, m.F}, m.opt());
  g[4] = at::empty({m.B, m.H, m.F}, m.opt());
  g[5] = at::empty({m.T}, m.opt());
  g[6] = at::empty({m.B, m.H, m.T}, m.opt());
  g[7] = at::empty({m.H, m.F}, m.opt());
  g[8] = at::empty({m.H, m.F}, m.opt());
  Tensor ws = at::empty({(int64_t)wsb}, m.opt(at::kByte));
  return ttt_internal_linear_backward(
      &m.d, in.p(0), in.p(1), in.p(2), in.p(3), in.p(4), in.p(5), in.p(6), in.p(7), in.p(8), wck.const_data_ptr(),
      bck.const_data_ptr(), go.const_data_ptr(), gw_out.defined() ? gw_out.const_data_ptr() : nullptr,
      gb_out.defined() ? gb_out.const_data_ptr() : nullptr, g[0].data_ptr(), g[1].data_ptr(), g[2].data_ptr(),
      g[3].data_ptr(), g[4].data_ptr(), g[6].data_ptr(), g[5].data_ptr(), g[7].data_ptr(), g[8].data_ptr(), m.d.dtype,
      packed.defined() ? static_cast<float*>(packed.data_ptr()) : nullptr, ws.data_ptr(), wsb, m.status.data_ptr(),
      m.stream());
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& xq, const Tensor& xk, const Tensor& xv, const Tensor& w,
                               const Tensor& b, const Tensor& te, const Tensor& lr, const Tensor& g, const Tensor& be,
                               int64_t mb, int64_t K, int64_t eps_scaled) {
    LinIn in{{xq, xk, xv, w, b, te, lr, g, be}};
    Dims m;
    LinOut o;
    m.set(xq, xq.size(3), mb, K, eps_scaled);
    const int rc = linear_forward(m, in, true, o);
    if (rc != TTT_OK) throw_error(rc);
    // kept as plain references, without version checks, like the Python node keeps its TttSavedStateMulti
    ctx->saved_data["t"] = std::vector<Tensor>{xq, xk, xv, w, b, te, lr, g, be, o.wck, o.bck};
    ctx->saved_data["c"] = std::vector<int64_t>{mb, K, eps_scaled};
    ctx->mark_non_differentiable({o.w, o.b});
    ctx->set_materialize_grads(false);
    return {o.out, o.w, o.b};
  }
  static variable_list backward(AutogradContext* ctx, variable_list go_) {
    const std::vector<Tensor> t = ctx->saved_data["t"].toTensorVector();
    const std::vector<int64_t> c = ctx->saved_data["c"].toIntVector();
    LinIn in;
    for (int i = 0; i < 9; ++i) in.t[i] = t[i];
    Dims m;
    m.set(t[0], t[0].size(3), c[0], c[1], c[2]);
    const Tensor go = go_[0].defined() ? go_[0].contiguous() : at::zeros_like(t[0]);
    Tensor g[9];
    const int rc = linear_backward(m, in, t[9], t[10], go, Tensor(), Tensor(), Tensor(), g);
    if (rc != TTT_OK) throw_error(rc);
    variable_list r(g, g + 9);
    for (int i = 0; i < 3; ++i) r.emplace_back();
    return r;
  }
};

// ---- TTT-MLP -----------------------------------------------------------------------------------------------------
struct MlpIn {  // xq, xk, xv, w1, b1, w2, b2, token_eta, ttt_lr_eta, ln_weight, ln_bias
  Tensor t[11];
  bool plain(const Dims& m) const {
    const int64_t B = m.B, H = m.H, T = m.T, F = m.F, E = 4 * F;
    if (t[7].dim() != 1 || m.dt != at::kBFloat16) return false;
    return is(t[0], m.dt, m.dev, {B, H, T, F}) && is(t[1], m.dt, m.dev, {B, H, T, F}) &&
           is(t[2], m.dt, m.dev, {B, H, T, F}) && is(t[3], m.dt, m.dev, {B, H, F, E}) && is(t[4], m.dt, m.dev, {B, H, E}) &&
           is(t[5], m.dt, m.dev, {B, H, E, F}) && is(t[6], m.dt, m.dev, {B, H, F}) &&
           is(t[7], m.dt, m.dev, {t[7].size(0)}) && is(t[8], m.dt, m.dev, {B, H, T}) && is(t[9], m.dt, m.dev, {H, F}) &&
           is(t[10], m.dt, m.dev, {H, F});
  }
  const void* p(int i) const { return t[i].const_data_ptr(); }
};
int mlp_forward(const Dims& m, const MlpIn& in, const Tensor& ws, Tensor (&o)[5]) {
  c10::cuda::CUDAGuard guard(m.dev);
  o[0] = at::empty({m.B, m.H, m.T, m.F}, m.opt());
  for (int i = 0; i < 4; ++i) o[1 + i] = at::empty(in.t[3 + i].sizes(), m.opt());
  if (!ws.defined()) {
    size_t bytes = ttt_internal_mlp_infer_scratch_bytes(&m.d);
    Tensor scratch;
    if (bytes != 0) {
      try {
        scratch = at::empty({(int64_t)bytes}, m.opt(at::kByte));
      } catch (const c10::OutOfMemoryError&) {  // whole waves need none
        bytes = 0;
      }
    }
    return ttt_internal_mlp_infer(&m.d, in.p(0), in.p(1), in.p(2), in.p(3), in.p(4), in.p(5), in.p(6), in.p(7), in.p(8),
                                  in.p(9), in.p(10), o[0].data_ptr(), o[1].data_ptr(), o[2].data_ptr(), o[3].data_ptr(),
                                  o[4].data_ptr(), bytes != 0 ? scratch.data_ptr() : nullptr, bytes, m.status.data_ptr(),
                                  m.stream());
  }
  return ttt_mlp_forward(&m.d, in.p(0), in.p(1), in.p(2), in.p(3), in.p(4), in.p(5), in.p(6), in.p(7), in.p(8), in.p(9),
                         in.p(10), o[0].data_ptr(), o[1].data_ptr(), o[2].data_ptr(), o[3].data_ptr(), o[4].data_ptr(),
                         ws.data_ptr(), (size_t)ws.numel(), m.status.data_ptr(), m.stream());
}
// gradients in the order of the inputs; `from_forward`: ws was filled by the forward on the same inputs
int mlp_backward(const Dims& m, const MlpIn& in, const Tensor& go, const Tensor& ws, bool from_forward, Tensor (&g)[11]) {
  c10::cuda::CUDAGuard guard(m.dev);
  for (int i = 0; i < 11; ++i) g[i] = at::empty(i == 7 ? c10::IntArrayRef({m.T}) : in.t[i].sizes(), m.opt());
  return ttt_internal_mlp_backward(
      &m.d, in.p(0), in.p(1), in.p(2), in.p(3), in.p(4), in.p(5), in.p(6), in.p(7), in.p(8), in.p(9), in.p(10),
      go.const_data_ptr(), g[0].data_ptr(), g[1].data_ptr(), g[2].data_ptr(), g[3].data_ptr(), g[4].data_ptr(),
      g[5].data_ptr(), g[6].data_ptr(), g[8].data_ptr(), g[7].data_ptr(), g[9].data_ptr(), g[10].data_ptr(), m.d.dtype,
      ws.data_ptr(), (size_t)ws.numel(), from_forward ? 1 : 0, m.status.data_ptr(), m.stream());
}

struct MlpFn : torch::autograd::Function<MlpFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& xq, const Tensor& xk, const Tensor& xv,
                               const Tensor& w1, const Tensor& b1, const Tensor& w2, const Tensor& b2, const Tensor& te,
                               const Tensor& lr, const Tensor& g, const Tensor& be, int64_t mb, int64_t K,
                               int64_t eps_scaled) {
    MlpIn in{{xq, xk, xv, w1, b1, w2, b2, te, lr, g, be}};
    Dims m;
    m.set(xq, xq.size(3), mb, K, eps_scaled);
    const size_t wsb = ttt_mlp_backward_workspace_bytes(&m.d);
    if (wsb == 0) throw_error(TTT_ERR_SHAPE);
    // the forward fills the backward's workspace on the way (final state + the operands of every state update)
    Tensor ws = at::empty({(int64_t)wsb}, m.opt(at::kByte)), o[5];
    const int rc = mlp_forward(m, in, ws, o);
    if (rc != TTT_OK) throw_error(rc);
    ctx->save_for_backward({xq, xk, xv, w1, b1, w2, b2, te, lr, g, be});
    ctx->saved_data["c"] = std::vector<int64_t>{mb, K, eps_scaled};
    ctx->saved_data["ws"] = ws;
    ctx->set_materialize_grads(false);
    return {o[0], o[1], o[2], o[3], o[4]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list go_) {
    const variable_list t = ctx->get_saved_variables();
    const std::vector<int64_t> c = ctx->saved_data["c"].toIntVector();
    MlpIn in;
    for (int i = 0; i < 11; ++i) in.t[i] = t[i];
    Dims m;
    m.set(t[0], t[0].size(3), c[0], c[1], c[2]);
    const Tensor go = go_[0].defined() ? go_[0].contiguous() : at::zeros_like(t[0]);
    // the buffer is consumed by the backward: a second backward walks the sequence forward again
    auto it = ctx->saved_data.find("ws");
    const bool filled = it != ctx->saved_data.end();
    Tensor ws = filled ? it->second.toTensor()
                       : at::empty({(int64_t)ttt_mlp_backward_workspace_bytes(&m.d)}, m.opt(at::kByte));
    if (filled) ctx->saved_data.erase(it);
    Tensor g[11];
    const int rc = mlp_backward(m, in, go, ws, filled, g);
    if (rc != TTT_OK) throw_error(rc);
    variable_list r(g, g + 11);
    for (int i = 0; i < 3; ++i) r.emplace_back();
    return r;
  }
};

// ---- gated linear recurrence ---------------------------------------------------------------------------------------------
// [B,H,T,F] with any strides that the kernels take (rows contiguous, the other strides positive multiples of 16 bytes)
bool rows_of_16_bytes(const Tensor& t) {
  if (t.layout() != c10::kStrided || t.stride(3) != 1 || !on_16_bytes(t)) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) * (int64_t)t.element_size() % 16 != 0)) return false;
  return true;
}
struct Gated {
  Dims m;
  bool plain(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const Tensor& w) {
    if (!m.set(q, q.dim() == 4 ? q.size(3) : -1, 1, 1, 0) || !m.status.defined()) return false;
    const c10::IntArrayRef four = q.sizes();
    for (const Tensor* t : {&q, &k, &v})
      if (t->scalar_type() != m.dt || t->device() != m.dev || t->sizes() != four || !rows_of_16_bytes(*t)) return false;
    if (!is(g, at::kFloat, m.dev, {m.B, m.H, m.T})) return false;
    if (beta.defined() && !is(beta, at::kFloat, m.dev, {m.B, m.H, m.T})) return false;
    if (w.defined() && (!is(w, at::kFloat, m.dev, {m.B, m.H, m.F, m.F}) || !on_16_bytes(w))) return false;
    return ttt_linear_gated_saved_bytes(&m.d) != 0;
  }
  static const float* f32(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.const_data_ptr()) : nullptr; }
  template <size_t N>
  static std::array<int64_t, 3 * N> strides(const std::array<const Tensor*, N>& ts) {
    std::array<int64_t, 3 * N> s;
    for (size_t i = 0; i < N; ++i)
      for (int k = 0; k < 3; ++k) s[3 * i + k] = ts[i]->stride(k);
    return s;
  }
  int forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const Tensor& w, bool save,
              Tensor& out, Tensor& w_out, Tensor& saved) {
    c10::cuda::CUDAGuard guard(m.dev);
    out = at::empty({m.B, m.H, m.T, m.F}, m.opt());
    w_out = at::empty({m.B, m.H, m.F, m.F}, m.opt(at::kFloat));
    const auto s = strides<3>({&q, &k, &v});
    if (!save && m.T <= 16)
      return ttt_linear_gated_step(&m.d, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), s.data(), f32(g), f32(beta),
                                   f32(w), out.data_ptr(), static_cast<float*>(w_out.data_ptr()), m.stream());
    const size_t wsb = ttt_linear_gated_forward_workspace_bytes(&m.d), sb = save ? ttt_linear_gated_saved_bytes(&m.d) : 0;
    Tensor ws;
    if (wsb != 0) ws = at::empty({(int64_t)wsb}, m.opt(at::kByte));
    if (save) saved = at::empty({(int64_t)sb}, m.opt(at::kByte));
    return ttt_linear_gated_forward(&m.d, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), s.data(), f32(g), f32(beta),
                                    f32(w), out.data_ptr(), static_cast<float*>(w_out.data_ptr()), save ? saved.data_ptr() : nullptr,
                                    sb, wsb != 0 ? ws.data_ptr() : nullptr, wsb, m.status.data_ptr(), m.stream());
  }
};

// What a node's backward returns where it is itself recorded (create_graph): gradients that say so when they are differentiated, since
// the kernels' gradients are not functions that autograd knows.
variable_list only_once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  return torch::autograd::DelayedError("the gradients of this operator are not differentiable", (int64_t)grads.size())(std::move(grads));
}

struct GatedFn : torch::autograd::Function<GatedFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                               const Tensor& beta, const Tensor& w, bool has_beta, bool has_w) {
    Gated call;
    Tensor out, w_out, saved;
    call.m.set(q, q.size(3), 1, 1, 0);
    const int rc = call.forward(q, k, v, g, has_beta ? beta : Tensor(), has_w ? w : Tensor(), true, out, w_out, saved);
    if (rc != TTT_OK) throw_error(rc);
    ctx->save_for_backward({q, k, v, g, beta, saved});
    ctx->saved_data["has"] = std::vector<int64_t>{has_beta, has_w};
    ctx->set_materialize_grads(false);
    return {out, w_out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    const variable_list t = ctx->get_saved_variables();
    const std::vector<int64_t> has = ctx->saved_data["has"].toIntVector();
    const Tensor &q = t[0], &k = t[1], &v = t[2], &g = t[3], beta = has[0] ? t[4] : Tensor();
    const Tensor& saved = t[5];
    if (!go[0].defined() && !go[1].defined()) return variable_list(8);
    Gated call;
    call.m.set(q, q.size(3), 1, 1, 0);
    const Dims& m = call.m;
    c10::cuda::CUDAGuard guard(m.dev);
    Tensor u = go[0].defined() ? go[0] : at::zeros({m.B, m.H, m.T, m.F}, m.opt()), dw_out = go[1];
    if (!rows_of_16_bytes(u)) u = u.clone(at::MemoryFormat::Contiguous);
    if (dw_out.defined() && (!dw_out.is_contiguous() || !on_16_bytes(dw_out))) dw_out = dw_out.clone(at::MemoryFormat::Contiguous);
    Tensor dq = at::empty({m.B, m.H, m.T, m.F}, m.opt()), dk = at::empty_like(dq), dv = at::empty_like(dq);
    Tensor dg = at::empty({m.B, m.H, m.T}, m.opt(at::kFloat)), db, dw = at::empty({m.B, m.H, m.F, m.F}, m.opt(at::kFloat)), ws;
    if (beta.defined()) db = at::empty_like(dg);
    const size_t wsb = ttt_linear_gated_backward_workspace_bytes(&m.d);
    if (wsb != 0) ws = at::empty({(int64_t)wsb}, m.opt(at::kByte));
    const auto s = Gated::strides<4>({&q, &k, &v, &u});
    const int rc = ttt_linear_gated_backward(
        &m.d, q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), u.const_data_ptr(), s.data(), Gated::f32(g), Gated::f32(beta),
        saved.const_data_ptr(), (size_t)saved.numel(), Gated::f32(dw_out), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
        static_cast<float*>(dg.data_ptr()), beta.defined() ? static_cast<float*>(db.data_ptr()) : nullptr,
        static_cast<float*>(dw.data_ptr()), wsb != 0 ? ws.data_ptr() : nullptr, wsb, m.status.data_ptr(), m.stream());
    if (rc != TTT_OK) throw_error(rc);
    return only_once({dq, dk, dv, dg, db, has[1] ? dw : Tensor(), Tensor(), Tensor()});
  }
};

// ---- rotary positions, norm and rotation of queries and keys -----------------------------------------------------------------
// [B,H,T,F] on a GPU with contiguous rows
bool head_rows(const Tensor& t, const c10::Device& dev, at::ScalarType dt) {
  return t.defined() && t.is_cuda() && t.device() == dev && t.scalar_type() == dt && t.layout() == c10::kStrided && t.dim() == 4 &&
         (t.stride(3) == 1 || t.size(3) == 1);
}
struct Rotation {
  Tensor turns, positions;
  int64_t rdim = 0, half = 0, wrap = 0, start = 0;
  double size = 1.0;
  ttt_rotation r;
  bool set(const Dims& m) {
    r = ttt_rotation{};
    if (!turns.defined()) return true;
    if (rdim < 2 || rdim > m.F || !is(turns, at::kLong, m.dev, {rdim / 2}) || wrap < 0 || wrap > INT32_MAX) return false;
    if (positions.defined()) {
      const bool rows = positions.dim() == 2;
      if (!positions.is_cuda() || positions.device() != m.dev || positions.scalar_type() != at::kLong || !positions.is_contiguous() ||
          (!rows && positions.dim() != 1) || positions.size(-1) != m.T || (rows && positions.size(0) != m.B && positions.size(0) != 1))
        return false;
      r.positions_stride = rows && positions.size(0) > 1 ? m.T : 0;
      r.positions = static_cast<const int64_t*>(positions.const_data_ptr());
    }
    r.turns = static_cast<const uint64_t*>(turns.const_data_ptr());
    r.start_idx = start;
    r.rotary_dim = (int32_t)rdim;
    r.half = (int32_t)half;
    r.wrap = (int32_t)wrap;
    r.size = (float)size;
    return true;
  }
  const ttt_rotation* get() const { return turns.defined() ? &r : nullptr; }
  std::vector<int64_t> ints() const { return {rdim, half, wrap, start, turns.defined(), positions.defined()}; }
  void from(const std::vector<int64_t>& v, double sz, const Tensor& t, const Tensor& p) {
    rdim = v[0], half = v[1], wrap = v[2], start = v[3], size = sz;
    if (v[4]) turns = t;
    if (v[5]) positions = p;
  }
};
Tensor given(const Tensor& t) { return t.defined() ? t : at::empty({0}); }  // (a node's arguments are defined tensors)

bool head_dims(Dims& m, const Tensor& x, double eps) {
  if (!x.defined() || x.dim() != 4 || !m.set(x, x.size(3), 1, 1, 0) || !head_rows(x, m.dev, m.dt)) return false;
  m.d.epsilon = (float)eps;
  return m.B > 0 && m.H > 0 && m.T > 0 && m.F >= 2;
}
int rotary(const Dims& m, const Tensor& x, const Rotation& rot, bool inverse, Tensor& y) {
  c10::cuda::CUDAGuard guard(m.dev);
  if (!y.defined()) y = at::empty({m.B, m.H, m.T, m.F}, m.opt());
  return ttt_layer_rotary(&m.d, x.const_data_ptr(), Gated::strides<1>({&x}).data(), rot.get(), inverse, y.data_ptr(),
                          Gated::strides<1>({&y}).data(), m.stream());
}
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& turns, const Tensor& positions, std::vector<int64_t> ints,
                        double size) {
    Dims m;
    Rotation rot;
    Tensor y;
    head_dims(m, x, 0.0);
    rot.from(ints, size, turns, positions);
    rot.set(m);
    const int rc = rotary(m, x, rot, false, y);
    if (rc != TTT_OK) throw_error(rc);
    ctx->save_for_backward({turns, positions});
    ctx->saved_data["i"] = ints;
    ctx->saved_data["s"] = size;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    const variable_list t = ctx->get_saved_variables();
    Tensor g = go[0], y;
    if (g.stride(3) != 1 && g.size(3) != 1) g = g.clone(at::MemoryFormat::Contiguous);
    Dims m;
    Rotation rot;
    head_dims(m, g, 0.0);
    rot.from(ctx->saved_data["i"].toIntVector(), ctx->saved_data["s"].toDouble(), t[0], t[1]);
    rot.set(m);
    const int rc = rotary(m, g, rot, true, y);
    if (rc != TTT_OK) throw_error(rc);
    return only_once({y, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};
struct QkNorm {
  Dims m;
  int64_t Hk = 0;
  bool set(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, double eps) {
    if (!head_dims(m, q, eps) || !head_rows(k, m.dev, m.dt)) return false;
    Hk = k.size(1);
    if (k.size(0) != m.B || k.size(2) != m.T || k.size(3) != m.F || Hk < 1 || Hk > INT32_MAX) return false;
    for (const Tensor* w : {&wq, &wk})
      if (w->defined() && !is(*w, m.dt, m.dev, {m.F})) return false;
    return true;
  }
  int forward(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Rotation& rot, Tensor& yq, Tensor& yk) const {
    c10::cuda::CUDAGuard guard(m.dev);
    if (!yq.defined()) yq = at::empty({m.B, m.H, m.T, m.F}, m.opt());
    if (!yk.defined()) yk = at::empty({m.B, Hk, m.T, m.F}, m.opt());
    return ttt_layer_qk_norm_rotary(&m.d, (int)Hk, q.const_data_ptr(), k.const_data_ptr(), Gated::strides<2>({&q, &k}).data(), ptr(wq),
                                    ptr(wk), rot.get(), yq.data_ptr(), yk.data_ptr(), Gated::strides<2>({&yq, &yk}).data(), m.stream());
  }
  int backward(const Tensor& q, const Tensor& k, const Tensor& gq, const Tensor& gk, const Tensor& wq, const Tensor& wk,
               const Rotation& rot, Tensor& dq, Tensor& dk, Tensor& dwq, Tensor& dwk) const {
    c10::cuda::CUDAGuard guard(m.dev);
    if (!dq.defined()) dq = at::empty({m.B, m.H, m.T, m.F}, m.opt());
    if (!dk.defined()) dk = at::empty({m.B, Hk, m.T, m.F}, m.opt());
    if (wq.defined()) dwq = at::empty({m.F}, m.opt());
    if (wk.defined()) dwk = at::empty({m.F}, m.opt());
    const bool w = wq.defined() || wk.defined();
    const size_t wsb = w ? ttt_layer_qk_norm_rotary_backward_workspace_bytes(&m.d, (int)Hk) : 0;
    Tensor ws;
    if (wsb != 0) ws = at::empty({(int64_t)wsb}, m.opt(at::kByte));
    return ttt_layer_qk_norm_rotary_backward(
        &m.d, (int)Hk, q.const_data_ptr(), k.const_data_ptr(), gq.const_data_ptr(), gk.const_data_ptr(),
        Gated::strides<4>({&q, &k, &gq, &gk}).data(), ptr(wq), ptr(wk), rot.get(), dq.data_ptr(), dk.data_ptr(),
        Gated::strides<2>({&dq, &dk}).data(), wq.defined() ? dwq.data_ptr() : nullptr, wk.defined() ? dwk.data_ptr() : nullptr,
        wsb != 0 ? ws.data_ptr() : nullptr, wsb, m.stream());
  }
};
struct QkNormFn : torch::autograd::Function<QkNormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk,
                               const Tensor& turns, const Tensor& positions, std::vector<int64_t> ints, double size, double eps) {
    QkNorm call;
    Rotation rot;
    Tensor yq, yk;
    const Tensor w0 = ints[6] ? wq : Tensor(), w1 = ints[7] ? wk : Tensor();
    call.set(q, k, w0, w1, eps);
    rot.from(ints, size, turns, positions);
    rot.set(call.m);
    const int rc = call.forward(q, k, w0, w1, rot, yq, yk);
    if (rc != TTT_OK) throw_error(rc);
    ctx->save_for_backward({q, k, wq, wk, turns, positions});
    ctx->saved_data["i"] = ints;
    ctx->saved_data["s"] = size;
    ctx->saved_data["e"] = eps;
    return {yq, yk};
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    const variable_list t = ctx->get_saved_variables();
    const std::vector<int64_t> ints = ctx->saved_data["i"].toIntVector();
    for (Tensor& g : go)  // (undefined ones are zeros here)
      if (g.stride(3) != 1 && g.size(3) != 1) g = g.clone(at::MemoryFormat::Contiguous);
    QkNorm call;
    Rotation rot;
    const Tensor w0 = ints[6] ? t[2] : Tensor(), w1 = ints[7] ? t[3] : Tensor();
    call.set(t[0], t[1], w0, w1, ctx->saved_data["e"].toDouble());
    rot.from(ints, ctx->saved_data["s"].toDouble(), t[4], t[5]);
    rot.set(call.m);
    Tensor dq, dk, dwq, dwk;
    const int rc = call.backward(t[0], t[1], go[0], go[1], w0, w1, rot, dq, dk, dwq, dwk);
    if (rc != TTT_OK) throw_error(rc);
    return only_once({dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// ---- causal convolution, group norm: tensors [B,T,C] with contiguous channels -------------------------------------------------
bool channel_rows(const Tensor& t, const c10::Device& dev, at::ScalarType dt) {
  if (!t.defined() || !t.is_cuda() || t.device() != dev || t.scalar_type() != dt || t.layout() != c10::kStrided || t.dim() != 3) return false;
  return (t.stride(2) == 1 || t.size(2) == 1) && (t.stride(0) >= 0 || t.size(0) == 1) && (t.stride(1) >= 0 || t.size(1) == 1);
}
struct Rows {  // what [B,T,C] of a GPU operator is
  int64_t B = 0, T = 0, C = 0;
  int dtype = 0;
  at::ScalarType dt = at::kFloat;
  c10::Device dev = c10::Device(c10::kCPU);
  bool set(const Tensor& x) {
    if (!x.defined() || !x.is_cuda() || x.dim() != 3) return false;
    dt = x.scalar_type(), dev = x.device();
    if ((dt != at::kBFloat16 && dt != at::kFloat) || !channel_rows(x, dev, dt)) return false;
    B = x.size(0), T = x.size(1), C = x.size(2);
    dtype = dt == at::kBFloat16 ? TTT_BF16 : TTT_F32;
    return B > 0 && T > 0 && C > 0;
  }
  at::TensorOptions opt() const { return at::TensorOptions().dtype(dt).device(dev); }
  at::TensorOptions opt(at::ScalarType t) const { return at::TensorOptions().dtype(t).device(dev); }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
  Tensor empty() const { return at::empty({B, T, C}, opt()); }
  bool vector(const Tensor& t, at::ScalarType of) const { return !t.defined() || is(t, of, dev, {C}); }
  bool marks(const Tensor& t) const {
    return !t.defined() || ((t.scalar_type() == at::kBool || t.scalar_type() == at::kByte) && is(t, t.scalar_type(), dev, {B, T}));
  }
};
template <size_t N>
std::array<int64_t, 2 * N> row_strides(const std::array<const Tensor*, N>& ts) {
  std::array<int64_t, 2 * N> s{};
  for (size_t i = 0; i < N; ++i)
    if (ts[i]->defined()) s[2 * i] = ts[i]->stride(0), s[2 * i + 1] = ts[i]->stride(1);
  return s;
}
Tensor workspace(const Rows& m, size_t bytes) { return bytes != 0 ? at::empty({(int64_t)bytes}, m.opt(at::kByte)) : Tensor(); }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// a gradient as the kernels read it
Tensor rows_of(const Tensor& g, const Rows& m) { return channel_rows(g, m.dev, m.dt) ? g : g.clone(at::MemoryFormat::Contiguous); }

struct Conv {
  Rows m;
  int64_t K = 0;
  int act = 0;
  bool set(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state, const Tensor& starts, int64_t a) {
    if (!m.set(x) || w.dim() != 2) return false;
    K = w.size(1), act = (int)a;
    return K >= 2 && K <= 4 && is(w, m.dt, m.dev, {m.C, K}) && m.vector(bias, m.dt) && held(state) && m.marks(starts);
  }
  bool held(const Tensor& s) const { return !s.defined() || is(s, m.dt, m.dev, {m.B, K - 1, m.C}); }
  int forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state, const Tensor& starts, Tensor& y, Tensor& out) const {
    c10::cuda::CUDAGuard guard(m.dev);
    y = m.empty();
    if (!out.defined()) out = at::empty({m.B, K - 1, m.C}, m.opt());
    return ttt_layer_causal_conv(m.B, m.T, m.C, (int)K, m.dtype, act, x.const_data_ptr(), row_strides<1>({&x}).data(), w.const_data_ptr(),
                                 ptr(bias), ptr(state), ptr(starts), y.data_ptr(), out.data_ptr(), m.stream());
  }
};
struct ConvFn : torch::autograd::Function<ConvFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state,
                               const Tensor& starts, std::vector<int64_t> has) {
    Conv call;
    Tensor y, out;
    const Tensor b = has[0] ? bias : Tensor(), st = has[1] ? state : Tensor(), mk = has[2] ? starts : Tensor();
    call.set(x, w, b, st, mk, has[3]);
    const int rc = call.forward(x, w, b, st, mk, y, out);
    if (rc != TTT_OK) throw_error(rc);
    ctx->save_for_backward({x, w, bias, state, starts});
    ctx->saved_data["has"] = has;
    ctx->set_materialize_grads(false);
    return {y, out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    const variable_list t = ctx->get_saved_variables();
    const std::vector<int64_t> has = ctx->saved_data["has"].toIntVector();
    if (!go[0].defined() && !go[1].defined()) return variable_list(6);
    Conv call;
    const Tensor &x = t[0], &w = t[1], b = has[0] ? t[2] : Tensor(), st = has[1] ? t[3] : Tensor(), mk = has[2] ? t[4] : Tensor();
    call.set(x, w, b, st, mk, has[3]);
    const Rows& m = call.m;
    c10::cuda::CUDAGuard guard(m.dev);
    const Tensor gy = go[0].defined() ? rows_of(go[0], m) : at::zeros({m.B, m.T, m.C}, m.opt());
    const Tensor gs = go[1].defined() ? go[1].contiguous() : Tensor();
    Tensor gx = m.empty(), gw, gb, gst;
    if (ctx->needs_input_grad(1)) gw = at::empty_like(w);
    if (has[0] && ctx->needs_input_grad(2)) gb = at::empty_like(b);
    if (has[1]) gst = at::empty_like(st);
    const size_t wsb = gw.defined() || gb.defined() ? ttt_layer_causal_conv_backward_workspace_bytes(m.B, m.T, m.C, (int)call.K, m.dtype) : 0;
    const Tensor ws = workspace(m, wsb);
    const int rc = ttt_layer_causal_conv_backward(
        m.B, m.T, m.C, (int)call.K, m.dtype, call.act, x.const_data_ptr(), gy.const_data_ptr(), row_strides<2>({&x, &gy}).data(),
        w.const_data_ptr(), ptr(b), ptr(st), ptr(mk), ptr(gs), gx.data_ptr(), data(gw), data(gb), data(gst), data(ws), wsb, m.stream());
    if (rc != TTT_OK) throw_error(rc);
    return only_once({gx, gw, gb, gst, Tensor(), Tensor()});
  }
};

struct Norm {
  Rows m;
  int64_t G = 0;
  int act = 0, over = 0;
  float eps = 0.f;
  bool set(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& gate, int64_t groups, int64_t a, int64_t ov, double e) {
    G = groups, act = (int)a, over = (int)ov, eps = (float)e;
    return m.set(x) && G > 0 && G <= m.C && m.C % G == 0 && m.vector(w, m.dt) && m.vector(b, m.dt) &&
           (!gate.defined() || (channel_rows(gate, m.dev, m.dt) && gate.sizes() == x.sizes()));
  }
  int forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& gate, bool save, Tensor& y, Tensor& stats) const {
    c10::cuda::CUDAGuard guard(m.dev);
    y = m.empty();
    const size_t wsb = over == TTT_OVER_SEQUENCE ? ttt_layer_group_norm_workspace_bytes(m.B, m.T, m.C, (int)G, over, m.dtype) : 0;
    const Tensor ws = workspace(m, wsb);
    if (save && over == TTT_OVER_SEQUENCE) stats = at::empty({m.B, G, 2}, m.opt(at::kFloat));
    return ttt_layer_group_norm(m.B, m.T, m.C, (int)G, over, m.dtype, act, eps, x.const_data_ptr(), ptr(gate),
                                row_strides<2>({&x, &gate}).data(), ptr(w), ptr(b), y.data_ptr(), static_cast<float*>(data(stats)),
                                data(ws), wsb, m.stream());
  }
};
struct NormFn : torch::autograd::Function<NormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& gate,
                        std::vector<int64_t> has, double eps) {  // has: weight, bias, gate; groups, activation, over
    Norm call;
    Tensor y, stats;
    const Tensor w0 = has[0] ? w : Tensor(), b0 = has[1] ? b : Tensor(), g0 = has[2] ? gate : Tensor();
    call.set(x, w0, b0, g0, has[3], has[4], has[5], eps);
    const int rc = call.forward(x, w0, b0, g0, true, y, stats);
    if (rc != TTT_OK) throw_error(rc);
    ctx->save_for_backward({x, w, b, gate, given(stats)});
    ctx->saved_data["has"] = has;
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    const variable_list t = ctx->get_saved_variables();
    const std::vector<int64_t> has = ctx->saved_data["has"].toIntVector();
    const Tensor &x = t[0], w = has[0] ? t[1] : Tensor(), b = has[1] ? t[2] : Tensor(), gate = has[2] ? t[3] : Tensor();
    Norm call;
    call.set(x, w, b, gate, has[3], has[4], has[5], ctx->saved_data["eps"].toDouble());
    const Rows& m = call.m;
    c10::cuda::CUDAGuard guard(m.dev);
    const Tensor gy = rows_of(go[0], m);
    Tensor gx = m.empty(), gw, gb, gg;
    if (has[0] && ctx->needs_input_grad(1)) gw = at::empty_like(w);
    if (has[1] && ctx->needs_input_grad(2)) gb = at::empty_like(b);
    if (has[2]) gg = m.empty();
    const bool sums = call.over == TTT_OVER_SEQUENCE || gw.defined() || gb.defined();
    const size_t wsb = sums ? ttt_layer_group_norm_backward_workspace_bytes(m.B, m.T, m.C, (int)call.G, call.over, m.dtype) : 0;
    const Tensor ws = workspace(m, wsb);
    const int rc = ttt_layer_group_norm_backward(
        m.B, m.T, m.C, (int)call.G, call.over, m.dtype, call.act, call.eps, x.const_data_ptr(), ptr(gate), gy.const_data_ptr(),
        row_strides<3>({&x, &gate, &gy}).data(), ptr(w), ptr(b), call.over == TTT_OVER_SEQUENCE ? t[4].const_data_ptr<float>() : nullptr,
        gx.data_ptr(), data(gg), data(gw), data(gb), data(ws), wsb, m.stream());
    if (rc != TTT_OK) throw_error(rc);
    return only_once({gx, gw, gb, gg, Tensor(), Tensor()});
  }
};

// x, dt, A, B, C, then D, z, dt_bias, state, starts (each or undefined)
struct Selective {
  Rows m;
  int64_t G = 0, N = 0;
  int softplus = 1;
  static bool states(const Tensor& t, const Rows& m, int64_t G, int64_t N) {  // [B,T,G,N] with contiguous states
    if (!t.defined() || !t.is_cuda() || t.device() != m.dev || t.scalar_type() != m.dt || t.layout() != c10::kStrided || t.dim() != 4) return false;
    return t.size(0) == m.B && t.size(1) == m.T && t.size(2) == G && t.size(3) == N && (t.stride(3) == 1 || N == 1);
  }
  bool held(const Tensor& t) const { return !t.defined() || (is(t, at::kFloat, m.dev, {m.B, m.C, N}) && on_16_bytes(t)); }
  bool set(const Tensor (&t)[5], const Tensor (&o)[5], int64_t sp) {
    if (!m.set(t[0]) || !channel_rows(t[1], m.dev, m.dt) || t[1].sizes() != t[0].sizes() || t[3].dim() != 4) return false;
    G = t[3].size(2), N = t[3].size(3), softplus = (int)sp;
    if (G < 1 || N < 1 || m.C % G != 0 || N > INT32_MAX) return false;
    return is(t[2], at::kFloat, m.dev, {m.C, N}) && on_16_bytes(t[2]) && states(t[3], m, G, N) && states(t[4], m, G, N) &&
           m.vector(o[0], at::kFloat) && (!o[1].defined() || (channel_rows(o[1], m.dev, m.dt) && o[1].sizes() == t[0].sizes())) &&
           m.vector(o[2], at::kFloat) && held(o[3]) && m.marks(o[4]);
  }
  static std::array<int64_t, 14> strides(std::initializer_list<const Tensor*> rows, const Tensor& b, const Tensor& c) {
    std::array<int64_t, 14> s{};
    size_t i = 0;
    for (const Tensor* t : rows)
      for (int k = 0; k < 2; ++k) s[i++] = t->defined() ? t->stride(k) : 0;
    for (const Tensor* t : {&b, &c})
      for (int k = 0; k < 3; ++k) s[i++] = t->stride(k);
    return s;
  }
  static const float* f32(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
  int forward(const Tensor (&t)[5], const Tensor (&o)[5], bool save, Tensor& y, Tensor& out, Tensor& saved) const {
    c10::cuda::CUDAGuard guard(m.dev);
    y = m.empty();
    if (!out.defined()) out = at::empty({m.B, m.C, N}, m.opt(at::kFloat));
    size_t wsb = 0, sb = 0;
    if (save || m.T > 16) wsb = ttt_linear_selective_forward_workspace_bytes(m.B, m.T, m.C, (int)G, (int)N, m.dtype);
    if (save) {
      sb = ttt_linear_selective_saved_bytes(m.B, m.T, m.C, (int)G, (int)N, m.dtype);
      if (sb == 0) return TTT_ERR_UNSUPPORTED;
      saved = at::empty({(int64_t)sb}, m.opt(at::kByte));
    }
    const Tensor ws = workspace(m, wsb);
    return ttt_linear_selective_forward(m.B, m.T, m.C, (int)G, (int)N, m.dtype, softplus, ptr(t[0]), ptr(t[1]), f32(t[2]), ptr(t[3]), ptr(t[4]),
                                        f32(o[0]), ptr(o[1]), f32(o[2]), f32(o[3]), ptr(o[4]), strides({&t[0], &t[1], &o[1]}, t[3], t[4]).data(),
                                        y.data_ptr(), static_cast<float*>(out.data_ptr()), data(saved), sb, data(ws), wsb, m.stream());
  }
};
struct SelectiveFn : torch::autograd::Function<SelectiveFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                               const Tensor& D, const Tensor& z, const Tensor& bias, const Tensor& state, const Tensor& starts,
                               std::vector<int64_t> has) {  // has: D, z, bias, state, starts; softplus
    Selective call;
    const Tensor t[5] = {x, dt, A, B, C}, o[5] = {has[0] ? D : Tensor(), has[1] ? z : Tensor(), has[2] ? bias : Tensor(), has[3] ? state : Tensor(),
                                                  has[4] ? starts : Tensor()};
    Tensor y, out, saved;
    call.set(t, o, has[5]);
    const int rc = call.forward(t, o, true, y, out, saved);
    if (rc != TTT_OK) throw_error(rc);
    ctx->save_for_backward({x, dt, A, B, C, D, z, bias, starts, saved});  // (of the state, what the tiles' states say)
    ctx->saved_data["has"] = has;
    ctx->set_materialize_grads(false);
    return {y, out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    const variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> has = ctx->saved_data["has"].toIntVector();
    if (!go[0].defined() && !go[1].defined()) return variable_list(11);
    Selective call;
    const Tensor t[5] = {s[0], s[1], s[2], s[3], s[4]}, o[5] = {has[0] ? s[5] : Tensor(), has[1] ? s[6] : Tensor(), has[2] ? s[7] : Tensor(), Tensor(),
                                                               has[4] ? s[8] : Tensor()};
    call.set(t, o, has[5]);
    const Rows& m = call.m;
    c10::cuda::CUDAGuard guard(m.dev);
    const Tensor gy = go[0].defined() ? rows_of(go[0], m) : at::zeros({m.B, m.T, m.C}, m.opt());
    Tensor gs = go[1].defined() ? go[1].contiguous() : Tensor();
    if (gs.defined() && !on_16_bytes(gs)) gs = gs.clone();
    Tensor gx = m.empty(), gdt = m.empty(), gA = at::empty({m.C, call.N}, m.opt(at::kFloat)), gB = at::empty({m.B, m.T, call.G, call.N}, m.opt()),
           gC = at::empty_like(gB), gD, gz, gbias, gstate;
    if (has[0]) gD = at::empty({m.C}, m.opt(at::kFloat));
    if (has[1]) gz = m.empty();
    if (has[2]) gbias = at::empty({m.C}, m.opt(at::kFloat));
    if (has[3]) gstate = at::empty({m.B, m.C, call.N}, m.opt(at::kFloat));
    const size_t wsb = ttt_linear_selective_backward_workspace_bytes(m.B, m.T, m.C, (int)call.G, (int)call.N, m.dtype);
    const Tensor ws = workspace(m, wsb);
    auto f = [](const Tensor& v) { return static_cast<float*>(data(v)); };
    const int rc = ttt_linear_selective_backward(
        m.B, m.T, m.C, (int)call.G, (int)call.N, m.dtype, call.softplus, ptr(t[0]), ptr(t[1]), call.f32(t[2]), ptr(t[3]), ptr(t[4]), call.f32(o[0]),
        ptr(o[1]), call.f32(o[2]), ptr(o[4]), gy.const_data_ptr(), call.strides({&t[0], &t[1], &o[1], &gy}, t[3], t[4]).data(),
        s[9].const_data_ptr(), (size_t)s[9].numel(), call.f32(gs), gx.data_ptr(), gdt.data_ptr(), f(gA), gB.data_ptr(), gC.data_ptr(), f(gD), data(gz),
        f(gbias), f(gstate), data(ws), wsb, m.stream());
    if (rc != TTT_OK) throw_error(rc);
    return only_once({gx, gdt, gA, gB, gC, gD, gz, gbias, gstate, Tensor(), Tensor()});
  }
};

// ---- Python functions ----------------------------------------------------------------------------------------------
// tensors args[0..n), false when one is not a tensor
template <int N>
bool tensors(PyObject* const* args, Tensor (&t)[N]) {
  for (int i = 0; i < N; ++i) {
    if (!THPVariable_Check(args[i])) return false;
    t[i] = THPVariable_Unpack(args[i]);
  }
  return true;
}
int64_t as_int(PyObject* o) { return PyLong_AsLongLong(o); }
PyObject* wrap(std::initializer_list<Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
  return r;
}
PyObject* wrap(const variable_list& ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  for (size_t i = 0; i < ts.size(); ++i) PyTuple_SET_ITEM(r, (Py_ssize_t)i, THPVariable_Wrap(ts[i]));
  return r;
}
#define NONE_IF(cond) \
  if (cond) Py_RETURN_NONE
bool arity(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

// init(TttError)
PyObject* py_init(PyObject*, PyObject* err) {
  Py_XINCREF(err);
  Py_XSETREF(g_error_type, err);
  Py_RETURN_NONE;
}
// set_status(device index, tensor)
PyObject* py_set_status(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 2)) return nullptr;
  const int64_t i = as_int(args[0]);
  if (i >= 0 && i < kMaxDevices && THPVariable_Check(args[1])) g_status[i] = THPVariable_Unpack(args[1]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// linear_forward(9 tensors, mini_batch, head_dim, K, eps_scaled, save) -> (out, w, b, w_ckpt | None, b_ckpt | None) | None
PyObject* py_linear_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 14)) return nullptr;
  LinIn in;
  Dims m;
  NONE_IF(!tensors(args, in.t));
  NONE_IF(!m.set(in.t[0], as_int(args[10]), as_int(args[9]), as_int(args[11]), as_int(args[12])));
  NONE_IF(!m.status.defined() || !in.plain(m));
  LinOut o;
  NONE_IF(linear_forward(m, in, args[13] == Py_True, o) != TTT_OK);
  return wrap({o.out, o.w, o.b, o.wck, o.bck});
  END_HANDLE_TH_ERRORS
}
// linear_partial(9 tensors, mini_batch, head_dim, K, eps_scaled, in_place) -> (out, w, b) | None
PyObject* py_linear_partial(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 14)) return nullptr;
  LinIn in;
  Dims m;
  NONE_IF(!tensors(args, in.t));
  NONE_IF(!m.set(in.t[0], as_int(args[10]), as_int(args[9]), as_int(args[11]), as_int(args[12])) || !in.plain(m));
  c10::cuda::CUDAGuard guard(m.dev);
  const bool in_place = args[13] == Py_True;
  Tensor out = at::empty({m.B, m.H, m.T, m.F}, m.opt());
  Tensor w = in_place ? in.t[3] : at::empty({m.B, m.H, m.F, m.F}, m.opt());
  Tensor b = in_place ? in.t[4] : at::empty({m.B, m.H, m.F}, m.opt());
  NONE_IF(ttt_linear_forward_partial(&m.d, in.p(0), in.p(1), in.p(2), in.p(3), in.p(4), in.p(5), in.p(6), in.p(7),
                                     in.p(8), out.data_ptr(), const_cast<void*>(w.const_data_ptr()),
                                     const_cast<void*>(b.const_data_ptr()), m.stream()) != TTT_OK);
  return wrap({out, w, b});
  END_HANDLE_TH_ERRORS
}
// linear_backward(9 tensors, w_ckpt, b_ckpt, grad_out, mini_batch, head_dim, K, eps_scaled, packed | None,
//                 grad_weight_out | None, grad_bias_out | None) -> 9 gradients | None
PyObject* py_linear_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 19)) return nullptr;
  LinIn in;
  Dims m;
  Tensor c[3], opt[3];
  NONE_IF(!tensors(args, in.t) || !tensors(args + 9, c));
  for (int i = 0; i < 3; ++i)
    if (args[16 + i] != Py_None) {
      NONE_IF(!THPVariable_Check(args[16 + i]));
      opt[i] = THPVariable_Unpack(args[16 + i]);
      NONE_IF(!opt[i].is_contiguous());
    }
  NONE_IF(!m.set(in.t[0], as_int(args[13]), as_int(args[12]), as_int(args[14]), as_int(args[15])));
  NONE_IF(!m.status.defined() || !in.plain(m) || !is(c[2], m.dt, m.dev, {m.B, m.H, m.T, m.F}));
  NONE_IF(!c[0].is_contiguous() || !c[1].is_contiguous() || c[0].device() != m.dev || c[1].device() != m.dev);
  NONE_IF((opt[0].defined() && (opt[0].scalar_type() != at::kFloat || opt[0].device() != m.dev)));
  NONE_IF(opt[1].defined() && !is(opt[1], m.dt, m.dev, {m.B, m.H, m.F, m.F}));
  NONE_IF(opt[2].defined() && !is(opt[2], m.dt, m.dev, {m.B, m.H, m.F}));
  Tensor g[9];
  NONE_IF(linear_backward(m, in, c[0], c[1], c[2], opt[1], opt[2], opt[0], g) != TTT_OK);
  return wrap(variable_list(g, g + 9));
  END_HANDLE_TH_ERRORS
}
// linear_apply(9 tensors, mini_batch, head_dim, K, eps_scaled) -> (out, w, b), recorded for autograd | None
PyObject* py_linear_apply(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 13)) return nullptr;
  LinIn in;
  Dims m;
  NONE_IF(!tensors(args, in.t));
  const int64_t mb = as_int(args[9]), K = as_int(args[11]), eps = as_int(args[12]);
  NONE_IF(!m.set(in.t[0], as_int(args[10]), mb, K, eps));
  NONE_IF(!m.status.defined() || !in.plain(m) || ttt_linear_num_checkpoints(&m.d) < 0);
  Tensor* t = in.t;
  return wrap(LinearFn::apply(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], mb, K, eps));
  END_HANDLE_TH_ERRORS
}
// mlp_forward(11 tensors, mini_batch, head_dim, K, eps_scaled, workspace | None) -> (out, w1, b1, w2, b2) | None
PyObject* py_mlp_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 16)) return nullptr;
  MlpIn in;
  Dims m;
  Tensor ws, o[5];
  NONE_IF(!tensors(args, in.t));
  if (args[15] != Py_None) {
    NONE_IF(!THPVariable_Check(args[15]));
    ws = THPVariable_Unpack(args[15]);
    NONE_IF(ws.scalar_type() != at::kByte || !ws.is_contiguous());
  }
  NONE_IF(!m.set(in.t[0], as_int(args[12]), as_int(args[11]), as_int(args[13]), as_int(args[14])));
  NONE_IF(!m.status.defined() || !in.plain(m) || (ws.defined() && ws.device() != m.dev));
  NONE_IF(mlp_forward(m, in, ws, o) != TTT_OK);
  return wrap({o[0], o[1], o[2], o[3], o[4]});
  END_HANDLE_TH_ERRORS
}
// mlp_apply(11 tensors, mini_batch, head_dim, K, eps_scaled) -> (out, w1, b1, w2, b2), recorded for autograd | None
PyObject* py_mlp_apply(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 15)) return nullptr;
  MlpIn in;
  Dims m;
  NONE_IF(!tensors(args, in.t));
  const int64_t mb = as_int(args[11]), K = as_int(args[13]), eps = as_int(args[14]);
  NONE_IF(!m.set(in.t[0], as_int(args[12]), mb, K, eps));
  NONE_IF(!m.status.defined() || !in.plain(m) || ttt_mlp_backward_workspace_bytes(&m.d) == 0);
  Tensor* t = in.t;
  return wrap(MlpFn::apply(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], t[9], t[10], mb, K, eps));
  END_HANDLE_TH_ERRORS
}

// ---- the outer layer, inference ------------------------------------------------------------------------------------
// tensors (None entries allowed) -> 16 bytes each that change with its storage, version, dtype or device
void fill_key(PyObject* const* args, Py_ssize_t n, uint64_t* k) {
  for (Py_ssize_t i = 0; i < n; ++i) {
    k[2 * i] = k[2 * i + 1] = 0;
    if (!THPVariable_Check(args[i])) continue;
    const Tensor& t = THPVariable_Unpack(args[i]);
    k[2 * i] = reinterpret_cast<uint64_t>(t.const_data_ptr());
    k[2 * i + 1] = ((uint64_t)t._version() << 16) | ((uint64_t)t.scalar_type() << 8) | (uint64_t)(uint8_t)t.device().index();
  }
}
// param_key(tensors...) -> their key
PyObject* py_param_key(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  PyObject* r = PyBytes_FromStringAndSize(nullptr, n * 16);
  if (r) fill_key(args, n, reinterpret_cast<uint64_t*>(PyBytes_AS_STRING(r)));
  return r;
  END_HANDLE_TH_ERRORS
}
// stream_key(device index, tensors...) -> the current stream of that device, then their key
PyObject* py_stream_key(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n < 1) return arity(n, 1), nullptr;
  const int64_t dev = as_int(args[0]);
  if (PyErr_Occurred()) return nullptr;
  const uint64_t st = reinterpret_cast<uint64_t>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
  PyObject* r = PyBytes_FromStringAndSize(nullptr, 8 + (n - 1) * 16);
  if (!r) return nullptr;
  uint64_t* const k = reinterpret_cast<uint64_t*>(PyBytes_AS_STRING(r));
  k[0] = st;
  fill_key(args + 1, n - 1, k + 1);
  return r;
  END_HANDLE_TH_ERRORS
}

// layer_infer(x, stacked weights, token_idx of one mini-batch, lr_bias, conv q weight / bias, conv k weight / bias (or four
//             None), state weight, state bias, ln weight, ln bias, post norm weight, bias, o_proj, gate 0/1, heads,
//             mini_batch, rope_mode, rope_theta, base_lr, lr_col, eps_scaled, allow_partial, in_place, start_idx,
//             learnable_token_idx)
//   -> (y, state weight, state bias) | None
// One call of TTT.forward without gradients, bf16: projections + prologue, inner loop (whole mini-batches, then the
// remainder as a mini-batch of its own), post norm (+ gate), output projection.
// None comes before the first launch only (what a later launch would refuse is looked at up front): the caller then takes
// another way from the same state.  An error after that is raised.
PyObject* py_layer_infer(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 27)) return nullptr;
  Tensor t[15], te_add;
  for (int i = 0; i < 15; ++i) {
    if (args[i] == Py_None && i >= 4 && i < 8) continue;
    NONE_IF(!THPVariable_Check(args[i]));
    t[i] = THPVariable_Unpack(args[i]);
  }
  NONE_IF(!THPVariable_Check(args[26]));
  te_add = THPVariable_Unpack(args[26]);
  const Tensor &x = t[0], &wcat = t[1], &te_idx = t[2], &lr_bias = t[3], &sw = t[8], &sb = t[9];
  const bool use_gate = as_int(args[15]) != 0, conv = t[4].defined();
  const int64_t H = as_int(args[16]), mb = as_int(args[17]), rope = as_int(args[18]), lr_col = as_int(args[21]);
  const float theta = (float)PyFloat_AsDouble(args[19]), base_lr = (float)PyFloat_AsDouble(args[20]);
  const int64_t eps_scaled = as_int(args[22]), start = as_int(args[25]);
  const bool allow_partial = args[23] == Py_True, in_place = args[24] == Py_True;
  if (PyErr_Occurred()) return nullptr;

  NONE_IF(!x.is_cuda() || x.dim() != 3 || x.scalar_type() != at::kBFloat16 || H <= 0 || mb <= 0);
  const c10::Device dev = x.device();
  const at::ScalarType bf = at::kBFloat16;
  const int64_t B = x.size(0), T = x.size(1), C = x.size(2), F = C / H, M = B * T;
  // rows of x: one pitch for all tokens
  NONE_IF(M <= 0 || F * H != C || (F != 64 && F != 32) || C > 2048 || C % 8 != 0 || x.stride(2) != 1);
  const int64_t x_ld = T > 1 ? x.stride(1) : x.stride(0);
  NONE_IF((T > 1 && B > 1 && x.stride(0) != T * x_ld) || x_ld < C || x_ld % 8 != 0);
  const int64_t N = wcat.size(0);
  NONE_IF(!is(wcat, bf, dev, {N, C}) || te_idx.dim() != 1 || te_idx.size(0) < mb ||
          !is(te_idx, bf, dev, {te_idx.size(0)}) || !is(te_add, bf, dev, {te_idx.size(0)}));
  NONE_IF(lr_bias.numel() != H || lr_bias.scalar_type() != bf || !lr_bias.is_contiguous() || lr_bias.device() != dev);
  NONE_IF(!is(sw, bf, dev, {B, H, F, F}) || !is(sb, bf, dev, {B, H, F}) || !is(t[10], bf, dev, {H, F}) ||
          !is(t[11], bf, dev, {H, F}) || !is(t[12], bf, dev, {C}) || !is(t[13], bf, dev, {C}) || !is(t[14], bf, dev, {C, C}));
  int conv_k = 0;
  if (conv) {
    for (int i = 4; i < 8; ++i)
      NONE_IF(!t[i].defined() || t[i].scalar_type() != bf || !t[i].is_contiguous() || t[i].device() != dev || t[i].size(0) != C);
    conv_k = (int)(t[4].numel() / C);
    NONE_IF(t[5].numel() != C || t[7].numel() != C || t[6].numel() != t[4].numel());
  }
  const int64_t L = T / mb * mb, R = T - L;
  NONE_IF(R > 16 || (R != 0 && !allow_partial));
  NONE_IF(L > 0 && ((mb != 16 && mb != 8) || (F == 32 && H % 2 != 0)));
  for (int i : {0, 1, 14}) NONE_IF(!on_16_bytes(t[i]));
  for (int i : {8, 9, 10, 11}) NONE_IF(L > 0 && !on_16_bytes(t[i]));  // (the remainder's kernel takes any alignment)
  Dims m;
  m.dt = bf;
  m.dev = dev;
  m.status = g_status[dev.index()];
  NONE_IF(!m.status.defined() || M > INT32_MAX || H > 64);
  ttt_dims d{(int32_t)B, (int32_t)H, (int32_t)T, (int32_t)F, (int32_t)mb, 1, (float)eps_scaled * 1e-9f, TTT_BF16};

  c10::cuda::CUDAGuard guard(dev);
  void* const st = m.stream();
  void* const status = m.status.data_ptr();
  const bool small = !conv && ttt_internal_layer_small_fits(&d);  // few-token form of the projections,
  const bool small_out = small && ttt_internal_layer_small_out_fits(&d, use_gate);  // of the output side
  NONE_IF(small_out && (!on_16_bytes(t[12]) || !on_16_bytes(t[13])));
  NONE_IF(!small && N % 8 != 0);
  auto must = [](int rc) {
    if (rc != TTT_OK) throw_error(rc);
  };
  const bool fused = !small && !conv && T % 128 == 0 && F == 64 && rope != 2 && mb <= 16 && lr_col % 64 == 0;
  // temporaries from one allocation, each on a 256-byte boundary
  int64_t at_ = 0;
  auto room = [&](int64_t elements) {
    const int64_t o = at_;
    at_ += (elements * 2 + 255) & ~(int64_t)255;
    return o;
  };
  const int64_t lr_pitch = (T + 7) & ~(int64_t)7;
  const int64_t o_q = room(M * C), o_k = room(M * C), o_v = room(M * C), o_lr = room(B * H * lr_pitch), o_in = room(M * C),
                o_te = room(16);
  const int64_t o_proj = small || fused ? 0 : room(M * N);
  const int64_t o_gate = use_gate && (small || fused) ? room(M * C) : 0;
  const int64_t o_y = small_out ? 0 : room(M * C);
  Tensor tmp = at::empty({at_}, m.opt(at::kByte));
  uint8_t* const base = static_cast<uint8_t*>(tmp.data_ptr());
  Tensor y = at::empty({B, T, C}, m.opt());
  const void* const idx = te_idx.const_data_ptr();
  const void* const learnable = te_add.const_data_ptr();
  void* const te = base + o_te;
  const uint8_t* gate = nullptr;
  int64_t gate_ld = C;
  const int64_t g_col = lr_col - C;
  // ---- projections, head split, rotary embedding, learning rates, token_eta
  if (small) {
    NONE_IF(ttt_internal_layer_small_proj(&d, x.const_data_ptr(), x_ld, wcat.const_data_ptr(), C, (int)N, (int)lr_col,
                                          lr_bias.const_data_ptr(), (int)start, (int)rope, theta, base_lr, idx, learnable, te,
                                          base + o_q, base + o_k, base + o_v, use_gate ? base + o_gate : nullptr, base + o_lr,
                                          (int)lr_pitch, st) != TTT_OK);
    if (use_gate) gate = base + o_gate;
  } else if (fused) {
    NONE_IF(ttt_internal_layer_projections(&d, x.const_data_ptr(), x_ld, C, wcat.const_data_ptr(), C, N, 0, C, 2 * C,
                                           use_gate ? g_col : -1, lr_col, lr_bias.const_data_ptr(), (int)start,
                                           (int)rope, theta, base_lr, 0, idx, learnable, te, base + o_q, base + o_k,
                                           base + o_v, use_gate ? base + o_gate : nullptr, base + o_lr, status,
                                           st) != TTT_OK);
    if (use_gate) gate = base + o_gate;
  } else {
    uint8_t* const proj = base + o_proj;
    NONE_IF(ttt_gemm_bf16_tn(M, N, C, x.const_data_ptr(), x_ld, wcat.const_data_ptr(), C, proj, N, status, st) != TTT_OK);
    const int64_t k_col = conv ? 0 : C, v_col = conv ? C : 2 * C;
    must(ttt_internal_layer_prologue(&d, proj, proj + 2 * k_col, proj + 2 * v_col, N, proj + 2 * lr_col, N,
                                     lr_bias.const_data_ptr(), conv ? t[4].const_data_ptr() : nullptr,
                                     conv ? t[5].const_data_ptr() : nullptr, conv ? t[6].const_data_ptr() : nullptr,
                                     conv ? t[7].const_data_ptr() : nullptr, conv_k, (int)start, (int)rope, theta,
                                     base_lr, idx, learnable, te, base + o_q, base + o_k, base + o_v, base + o_lr,
                                     (int)lr_pitch, st));
    if (use_gate) gate = proj + 2 * g_col, gate_ld = N;
  }
  // ---- inner loop
  Tensor w = sw, b = sb;
  if (L > 0) {
    w = at::empty({B, H, F, F}, m.opt());
    b = at::empty({B, H, F}, m.opt());
    ttt_dims di = d;
    di.seq_len = (int32_t)L;
    must(ttt_internal_linear_infer(&di, (int)T, (int)lr_pitch, base + o_q, base + o_k, base + o_v,
                                   sw.const_data_ptr(), sb.const_data_ptr(), te, base + o_lr,
                                   t[10].const_data_ptr(), t[11].const_data_ptr(), base + o_in, w.data_ptr(),
                                   b.data_ptr(), status, st));
  }
  if (R > 0) {
    const Tensor w_in = w, b_in = b;
    if (L == 0 && !in_place) {
      w = at::empty({B, H, F, F}, m.opt());
      b = at::empty({B, H, F}, m.opt());
    }
    ttt_dims dt = d;
    dt.seq_len = (int32_t)R;
    must(ttt_internal_linear_tail(&dt, (int)T, (int)L, (int)lr_pitch, small && L == 0, base + o_q, base + o_k, base + o_v,
                                  w_in.const_data_ptr(), b_in.const_data_ptr(), te, base + o_lr,
                                  t[10].const_data_ptr(), t[11].const_data_ptr(), base + o_in,
                                  const_cast<void*>(w.const_data_ptr()), const_cast<void*>(b.const_data_ptr()),
                                  st));
  }
  // ---- post norm, gate, output projection
  if (small_out) {
    must(ttt_internal_layer_small_out(&d, base + o_in, gate, (int)gate_ld, t[12].const_data_ptr(),
                                      t[13].const_data_ptr(), 1e-6f, t[14].const_data_ptr(), C, y.data_ptr(), st));
  } else {
    must(ttt_layer_epilogue(&d, base + o_in, gate, gate != nullptr ? gate_ld : 0, t[12].const_data_ptr(),
                            t[13].const_data_ptr(), 1e-6f, base + o_y, st));
    must(ttt_gemm_bf16_tn(M, C, C, base + o_y, C, t[14].const_data_ptr(), C, y.data_ptr(), C, status, st));
  }
  return wrap({y, w, b});
  END_HANDLE_TH_ERRORS
}

// ---- the outer layer, training -----------------------------------------------------------------------------------------
// The whole layer as one node of the graph, for the lengths whose projections are a product of their own: the steps of the
// Python composition (a node per step: its interpreter time is most of a training step of a few thousand tokens) with the
// same kernels and roundings, forward and backward.  The projections' gradients, the gate's among them, are the columns of one
// buffer, so the weights' and the input's are one product each.  5 x 192 tokens of 768 features, forward + backward: 1148 us
// through the composition, 528 here.
struct LayerDims {
  ttt_dims d;
  int64_t B, T, C, H, F, mb, M;
  int64_t v, lr, N0, g, N;  // columns q | k | v | lr (and padding) up to N0 | gate from g (-1: none) up to N
  int64_t taps;             // shared q / k projection (v = C then): taps of its two convolutions; 0: projections of their own
  int64_t K, rope, start, eps_scaled;
  float theta, base_lr;
};
struct LayerFn : torch::autograd::Function<LayerFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& g, const Tensor& lrw, const Tensor& lrb, const Tensor& learnable,
                               const Tensor& post_w, const Tensor& post_b, const Tensor& o, const Tensor& w0,
                               const Tensor& b0, const Tensor& ln_w, const Tensor& ln_b, const Tensor& cqw, const Tensor& cqb,
                               const Tensor& ckw, const Tensor& ckb, const Tensor& idx, const LayerDims& l) {
    Dims m;
    m.d = l.d;
    m.B = l.B, m.H = l.H, m.T = l.T, m.F = l.F;
    m.dt = x.scalar_type();
    m.dev = x.device();
    m.status = g_status[m.dev.index()];
    c10::cuda::CUDAGuard guard(m.dev);
    void* const st = m.stream();
    auto must = [](int rc) {
      if (rc != TTT_OK) throw_error(rc);
    };
    const bool gated = l.g >= 0, bf = m.dt == at::kBFloat16;
    const Tensor x2 = x.reshape({l.M, l.C}).contiguous();
    const Tensor lr2 = lrw.reshape({l.H, l.C});  // weights stacked in the order of the columns
    std::vector<Tensor> rows{q};
    if (!l.taps) rows.push_back(k);
    rows.push_back(v);
    rows.push_back(lr2);
    if (l.N0 > l.lr + l.H) rows.push_back(at::zeros({l.N0 - l.lr - l.H, l.C}, m.opt()));
    if (gated) rows.push_back(g);
    const Tensor wcat = at::cat(rows, 0);
    const Tensor te = at::add(idx, learnable);
    // token_eta of one mini-batch, which is all that is read of it: by the projections' kernel, or here in float32
    Tensor te16 = bf ? at::empty({16}, m.opt()) : at::clamp_min(te, 0.0);
    Tensor s[4];
    for (int i = 0; i < 3; ++i) s[i] = at::empty({l.B, l.H, l.T, l.F}, m.opt());
    s[3] = at::empty({l.B, l.H, l.T}, m.opt());
    const void* const ip = bf ? idx.const_data_ptr() : nullptr;
    const void* const lp = bf ? learnable.const_data_ptr() : nullptr;
    Tensor gate, proj = at::mm(x2, wcat.narrow(0, 0, l.N0).t());
    {
      const uint8_t* const p = static_cast<const uint8_t*>(proj.const_data_ptr());
      const int64_t e = proj.element_size();
      const bool cv = l.taps != 0;
      must(ttt_internal_layer_prologue(&l.d, p, p + (cv ? 0 : e * l.C), p + e * l.v, l.N0, p + e * l.lr, l.N0, lrb.const_data_ptr(),
                                       cv ? cqw.const_data_ptr() : nullptr, cv ? cqb.const_data_ptr() : nullptr,
                                       cv ? ckw.const_data_ptr() : nullptr, cv ? ckb.const_data_ptr() : nullptr, (int)l.taps,
                                       (int)l.start, (int)l.rope, l.theta, l.base_lr, ip, lp, bf ? te16.data_ptr() : nullptr,
                                       s[0].data_ptr(), s[1].data_ptr(), s[2].data_ptr(), s[3].data_ptr(), (int)l.T, st));
    }
    if (!l.taps) proj = Tensor();  // (the convolutions' gradient reads it)
    if (gated) gate = at::mm(x2, wcat.narrow(0, l.g, l.C).t());
    LinIn in{{s[0], s[1], s[2], w0, b0, te16, s[3], ln_w, ln_b}};
    LinOut lo;
    must(linear_forward(m, in, true, lo));
    const Tensor y = at::empty({l.M, l.C}, m.opt());
    must(ttt_layer_epilogue(&l.d, lo.out.const_data_ptr(), gated ? gate.const_data_ptr() : nullptr, gated ? l.C : 0,
                            post_w.const_data_ptr(), post_b.const_data_ptr(), 1e-6f, y.data_ptr(), st));
    const Tensor out = at::mm(y, o.t()).view({l.B, l.T, l.C});
    ctx->save_for_backward({x, wcat, te, lo.out, gate, post_w, post_b, y, o, proj, cqw, ckw});
    // kept as plain references, as the inner loop's own node keeps what it saves
    ctx->saved_data["t"] = std::vector<Tensor>{s[0], s[1], s[2], w0, b0, te16, s[3], ln_w, ln_b, lo.wck, lo.bck};
    ctx->saved_data["l"] = c10::IValue(std::string(reinterpret_cast<const char*>(&l), sizeof(l)));
    ctx->saved_data["s"] = std::vector<std::vector<int64_t>>{lrw.sizes().vec(), lrb.sizes().vec()};
    ctx->mark_non_differentiable({lo.w, lo.b});
    ctx->set_materialize_grads(false);
    return {out, lo.w, lo.b};
  }
  static variable_list backward(AutogradContext* ctx, variable_list go_) {
    const variable_list sv = ctx->get_saved_variables();
    const Tensor &x = sv[0], &wcat = sv[1], &te = sv[2], &inner_out = sv[3], &gate = sv[4], &post_w = sv[5], &post_b = sv[6],
                 &y = sv[7], &o = sv[8];
    const std::vector<Tensor> t = ctx->saved_data["t"].toTensorVector();
    LayerDims l;
    memcpy(&l, ctx->saved_data["l"].toStringRef().data(), sizeof(l));
    const auto shapes = ctx->saved_data["s"].toList();
    Dims m;
    m.d = l.d;
    m.B = l.B, m.H = l.H, m.T = l.T, m.F = l.F;
    m.dt = x.scalar_type();
    m.dev = x.device();
    m.status = g_status[m.dev.index()];
    c10::cuda::CUDAGuard guard(m.dev);
    void* const st = m.stream();
    auto must = [](int rc) {
      if (rc != TTT_OK) throw_error(rc);
    };
    const Tensor go = (go_[0].defined() ? go_[0] : at::zeros_like(x)).reshape({l.M, l.C}).contiguous();
    variable_list r(21);  // x q k v g lrw lrb learnable post_w post_b o w0 b0 ln_w ln_b, four of the convolutions, idx dims
    if (ctx->needs_input_grad(10)) r[10] = at::mm(go.t(), y);
    const Tensor dy = at::mm(go, o);
    // post norm and gate: the gate's gradient goes to its columns of the projections' gradient
    const Tensor dproj = at::empty({l.M, l.N}, m.opt());
    uint8_t* const dp = static_cast<uint8_t*>(dproj.data_ptr());
    const int64_t e = dproj.element_size();
    const bool gated = gate.defined();
    const Tensor d_inner = at::empty({l.B, l.H, l.T, l.F}, m.opt()), dn = at::empty({2, l.C}, m.opt(at::kFloat));
    {
      const size_t wsb = ttt_layer_epilogue_backward_workspace_bytes(&l.d);
      const Tensor ws = at::empty({(int64_t)wsb}, m.opt(at::kByte));
      must(ttt_layer_epilogue_backward(&l.d, dy.const_data_ptr(), inner_out.const_data_ptr(), gated ? gate.const_data_ptr() : nullptr,
                                       gated ? l.C : 0, post_w.const_data_ptr(), post_b.const_data_ptr(), 1e-6f, d_inner.data_ptr(),
                                       gated ? dp + e * l.g : nullptr, gated ? l.N : 0, static_cast<float*>(dn.data_ptr()),
                                       static_cast<float*>(dn.data_ptr()) + l.C, ws.data_ptr(), wsb, st));
    }
    const Tensor dnt = m.dt == at::kFloat ? dn : dn.to(m.dt);
    r[8] = dnt.select(0, 0);
    r[9] = dnt.select(0, 1);
    LinIn in;
    for (int i = 0; i < 9; ++i) in.t[i] = t[i];
    Tensor gr[9];
    must(linear_backward(m, in, t[9], t[10], d_inner, Tensor(), Tensor(), Tensor(), gr));
    r[11] = gr[3];
    r[12] = gr[4];
    r[13] = gr[7];
    r[14] = gr[8];
    auto prologue_backward = [&](void* dq, void* dk, void* dv, int64_t ld) {
      must(ttt_layer_prologue_backward(&l.d, gr[0].const_data_ptr(), gr[1].const_data_ptr(), gr[2].const_data_ptr(),
                                       gr[6].const_data_ptr(), t[6].const_data_ptr(), (int)l.start, (int)l.rope, l.theta, l.base_lr,
                                       dq, dk, dv, ld, dp + e * l.lr, l.N, (int)(l.N0 - l.lr), st));
    };
    if (!l.taps) {
      prologue_backward(dp, dp + e * l.C, dp + e * l.v, l.N);
    } else {
      // through the two convolutions to their shared projection
      const Tensor &proj = sv[9], d4 = at::empty({4, l.M, l.C}, m.opt());  // of q, k, v, and of the shared projection
      uint8_t* const d0 = static_cast<uint8_t*>(d4.data_ptr());
      const int64_t one = e * l.M * l.C;
      prologue_backward(d0, d0 + one, d0 + 2 * one, l.C);
      const Tensor gp = at::empty({2, 5, l.C}, m.opt(at::kFloat));  // four taps and the bias, of each
      auto taps4 = [&](const Tensor& w) {  // [C][4], aligned to the end
        const Tensor w2 = w.reshape({l.C, l.taps});
        if (l.taps == 4) return w2;
        Tensor w4 = at::zeros({l.C, 4}, w2.options());
        w4.narrow(1, 4 - l.taps, l.taps).copy_(w2);
        return w4;
      };
      const Tensor wq4 = taps4(sv[10]), wk4 = taps4(sv[11]);
      const size_t wsb = ttt_layer_qk_conv_backward_workspace_bytes(&l.d);
      const Tensor ws = at::empty({(int64_t)wsb}, m.opt(at::kByte));
      must(ttt_layer_qk_conv_backward(&l.d, d0, d0 + one, proj.const_data_ptr(), l.N0, wq4.const_data_ptr(), wk4.const_data_ptr(),
                                      d0 + 3 * one, static_cast<float*>(gp.data_ptr()), static_cast<float*>(gp.data_ptr()) + 5 * l.C,
                                      ws.data_ptr(), wsb, st));
      dproj.narrow(1, 0, l.C).copy_(d4.select(0, 3));
      dproj.narrow(1, l.v, l.C).copy_(d4.select(0, 2));
      const Tensor gpt = gp.to(m.dt);
      for (int i = 0; i < 2; ++i) {
        r[15 + 2 * i] = gpt.select(0, i).narrow(0, 4 - l.taps, l.taps).t().reshape(sv[10 + i].sizes());
        r[16 + 2 * i] = gpt.select(0, i).select(0, 4);
      }
    }
    if (ctx->needs_input_grad(0)) r[0] = at::mm(dproj, wcat).view(x.sizes());
    bool weights = false;
    for (int i = 1; i <= 5; ++i) weights = weights || ctx->needs_input_grad(i);
    if (weights) {
      const Tensor dw = at::mm(dproj.t(), x.reshape({l.M, l.C}));
      r[1] = dw.narrow(0, 0, l.C);
      if (!l.taps) r[2] = dw.narrow(0, l.C, l.C);
      r[3] = dw.narrow(0, l.v, l.C);
      if (gated) r[4] = dw.narrow(0, l.g, l.C);
      r[5] = dw.narrow(0, l.lr, l.H).view(shapes.get(0).toIntVector());
    }
    if (ctx->needs_input_grad(6))
      r[6] = at::sum(dproj.narrow(1, l.lr, l.H), {0}, false, at::kFloat).to(m.dt).view(shapes.get(1).toIntVector());
    if (ctx->needs_input_grad(7)) {
      const Tensor sum = at::sum(gr[5].view({l.T / l.mb, l.mb}), {0}, false, m.dt);
      r[7] = at::where(at::ge(te, 0), sum, at::zeros({}, sum.options()));
    }
    return r;
  }
};
// layer_train(x, q_proj, k_proj | None, v_proj, g_proj | None, lr weight, lr bias, learnable_token_idx, post norm weight, bias,
//             o_proj, state weight, state bias, ln weight, ln bias, conv q weight, bias, conv k weight, bias (with k_proj: four
//             None), token_idx, heads, mini_batch, rope_mode, rope_theta, base_lr,
//             checkpoint interval, eps_scaled, start_idx) -> (y, state weight, state bias), recorded for autograd | None
PyObject* py_layer_train(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 28)) return nullptr;
  Tensor t[20];
  const bool shared = args[2] == Py_None;
  for (int i = 0; i < 20; ++i) {
    if (args[i] == Py_None && (i == 4 || (shared ? i == 2 : i >= 15 && i < 19))) continue;
    NONE_IF(!THPVariable_Check(args[i]));
    t[i] = THPVariable_Unpack(args[i]);
    NONE_IF(t[i].unsafeGetTensorImpl()->is_python_dispatch());
  }
  LayerDims l;
  l.H = as_int(args[20]), l.mb = as_int(args[21]), l.rope = as_int(args[22]);
  l.theta = (float)PyFloat_AsDouble(args[23]), l.base_lr = (float)PyFloat_AsDouble(args[24]);
  l.K = as_int(args[25]), l.eps_scaled = as_int(args[26]), l.start = as_int(args[27]);
  if (PyErr_Occurred()) return nullptr;
  const Tensor& x = t[0];
  NONE_IF(at::autocast::is_autocast_enabled(at::kCUDA));
  NONE_IF(!x.is_cuda() || x.layout() != c10::kStrided || x.dim() != 3 || l.H <= 0 || l.mb <= 0);
  const c10::Device dev = x.device();
  const at::ScalarType dt = x.scalar_type();
  NONE_IF((dt != at::kBFloat16 && dt != at::kFloat) || dev.index() >= kMaxDevices || !g_status[dev.index()].defined());
  l.B = x.size(0), l.T = x.size(1), l.C = x.size(2), l.F = l.C / l.H, l.M = l.B * l.T;
  NONE_IF(l.M <= 0 || l.M > INT32_MAX || l.F * l.H != l.C || (l.F != 64 && l.F != 32) || l.C > 2048 || l.H > 64 || l.C % 8 != 0);
  NONE_IF((l.mb != 16 && l.mb != 8) || l.T % l.mb != 0 || (l.F == 32 && l.H % 2 != 0));
  for (int i : {1, 2, 3, 10}) NONE_IF(t[i].defined() && !is(t[i], dt, dev, {l.C, l.C}));
  const bool gated = t[4].defined();
  NONE_IF(gated && !is(t[4], dt, dev, {l.C, l.C}));
  NONE_IF(t[5].numel() != l.H * l.C || t[5].size(0) != l.H || t[5].scalar_type() != dt || t[5].device() != dev || !t[5].is_contiguous());
  NONE_IF(t[6].numel() != l.H || t[6].scalar_type() != dt || t[6].device() != dev || !t[6].is_contiguous());
  for (int i : {7, 19}) NONE_IF(!is(t[i], dt, dev, {l.mb}));
  for (int i : {8, 9}) NONE_IF(!is(t[i], dt, dev, {l.C}));
  NONE_IF(!is(t[11], dt, dev, {l.B, l.H, l.F, l.F}) || !is(t[12], dt, dev, {l.B, l.H, l.F}));
  for (int i : {13, 14}) NONE_IF(!is(t[i], dt, dev, {l.H, l.F}));
  l.taps = 0;
  if (shared) {
    for (int i = 15; i < 19; ++i)
      NONE_IF(t[i].dim() < 1 || t[i].size(0) != l.C || t[i].scalar_type() != dt || t[i].device() != dev || !t[i].is_contiguous());
    l.taps = t[15].numel() / l.C;
    NONE_IF(l.taps < 1 || l.taps > 4 || t[17].numel() != t[15].numel() || t[16].numel() != l.C || t[18].numel() != l.C);
  }
  for (int i = 0; i < 20; ++i) NONE_IF(t[i].defined() && !on_16_bytes(t[i]));
  // (those run projections and prologue in one launch: the composition)
  NONE_IF(!shared && dt == at::kBFloat16 && l.T % 128 == 0 && l.F == 64 && l.rope != 2);
  l.v = shared ? l.C : 2 * l.C;
  l.lr = l.v + l.C;
  l.N0 = (l.lr + l.H + 7) & ~(int64_t)7;
  l.g = gated ? l.N0 : -1;
  l.N = l.N0 + (gated ? l.C : 0);
  l.d = ttt_dims{(int32_t)l.B, (int32_t)l.H, (int32_t)l.T, (int32_t)l.F, (int32_t)l.mb, (int32_t)l.K, (float)l.eps_scaled * 1e-9f,
                 dt == at::kBFloat16 ? TTT_BF16 : TTT_F32};
  NONE_IF(ttt_linear_num_checkpoints(&l.d) < 0);
  for (Tensor& u : t)
    if (!u.defined()) u = at::empty({0});  // (a node's arguments are defined tensors)
  return wrap(LayerFn::apply(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], t[9], t[10], t[11], t[12], t[13], t[14], t[15],
                             t[16], t[17], t[18], t[19], l));
  END_HANDLE_TH_ERRORS
}

// optional tensor: None, or a tensor (false: neither)
bool optional_tensor(PyObject* o, Tensor& t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}
// Tensors that carry a tangent (forward-mode differentiation, with or without gradients): no operator here continues one, and its
// result would silently have none
void refuse_tangents(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined())
      throw_error(TTT_ERR_UNSUPPORTED, "derivatives in forward mode are not computed by this operator");
}
// gated(q, k, v, log_decay, beta | None, weight | None) -> (out, weight), recorded for autograd where that is on and asked for | None
PyObject* py_gated(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 6)) return nullptr;
  Tensor t[4], beta, w;
  NONE_IF(!tensors(args, t) || !optional_tensor(args[4], beta) || !optional_tensor(args[5], w));
  Gated call;
  refuse_tangents({&t[0], &t[1], &t[2], &t[3], &beta, &w});
  NONE_IF(!call.plain(t[0], t[1], t[2], t[3], beta, w));
  bool grad = false;
  if (at::GradMode::is_enabled())
    for (const Tensor* x : {&t[0], &t[1], &t[2], &t[3], &beta, &w}) grad = grad || (x->defined() && x->requires_grad());
  if (grad) {  // (a node's arguments are defined tensors)
    const bool has_beta = beta.defined(), has_w = w.defined();
    return wrap(GatedFn::apply(t[0], t[1], t[2], t[3], has_beta ? beta : at::empty({0}), has_w ? w : at::empty({0}), has_beta, has_w));
  }
  Tensor out, w_out, saved;
  const int rc = call.forward(t[0], t[1], t[2], t[3], beta, w, false, out, w_out, saved);
  if (rc != TTT_OK) throw_error(rc);
  return wrap({out, w_out});
  END_HANDLE_TH_ERRORS
}

// A rotation's arguments: turns | None, rotary_dim, half, wrap, size, positions | None, start_idx
bool rotation_args(PyObject* const* a, Rotation& rot) {
  if (!optional_tensor(a[0], rot.turns) || !optional_tensor(a[5], rot.positions)) return false;
  rot.rdim = as_int(a[1]), rot.half = as_int(a[2]), rot.wrap = as_int(a[3]), rot.size = PyFloat_AsDouble(a[4]), rot.start = as_int(a[6]);
  return true;
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
bool same_shape_result(const Tensor& y, const Tensor& x, const Dims& m) {
  return !y.defined() || (head_rows(y, m.dev, m.dt) && y.sizes() == x.sizes());
}
// A tensor that a kernel has overwritten: autograd refuses what was computed from its former values, as after torch's own operations
// (inference tensors count no versions, and nothing saves them)
void overwritten(const Tensor& y) {
  if (!y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
}
// rotary(x, rotation (7), inverse, out | None) -> y, recorded for autograd where that is on and asked for | None
PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 10)) return nullptr;
  Tensor x[1], y;
  Dims m;
  Rotation rot;
  NONE_IF(!tensors(args, x) || !rotation_args(args + 1, rot) || !optional_tensor(args[9], y));
  const bool inverse = as_int(args[8]) != 0;
  if (PyErr_Occurred()) return nullptr;
  refuse_tangents({&x[0], &y});
  NONE_IF(!rot.turns.defined() || !head_dims(m, x[0], 0.0) || !rot.set(m) || !same_shape_result(y, x[0], m));
  if (wants_grad({&x[0], &y})) {  // (a given result is not recorded: the caller's check refuses it)
    NONE_IF(y.defined() || inverse);
    return THPVariable_Wrap(RotaryFn::apply(x[0], rot.turns, given(rot.positions), rot.ints(), rot.size));
  }
  const bool given_y = y.defined();
  const int rc = rotary(m, x[0], rot, inverse, y);
  if (rc != TTT_OK) throw_error(rc);
  if (given_y) overwritten(y);
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}
// qk_norm(q, k, q_weight | None, k_weight | None, rotation (7), eps, q_out | None, k_out | None) -> (q, k), recorded for autograd
// where that is on and asked for | None
PyObject* py_qk_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 14)) return nullptr;
  Tensor x[2], wq, wk, yq, yk;
  QkNorm call;
  Rotation rot;
  NONE_IF(!tensors(args, x) || !optional_tensor(args[2], wq) || !optional_tensor(args[3], wk) || !rotation_args(args + 4, rot) ||
          !optional_tensor(args[12], yq) || !optional_tensor(args[13], yk));
  const double eps = PyFloat_AsDouble(args[11]);
  if (PyErr_Occurred()) return nullptr;
  refuse_tangents({&x[0], &x[1], &wq, &wk, &yq, &yk});
  NONE_IF(!call.set(x[0], x[1], wq, wk, eps) || !rot.set(call.m) || !same_shape_result(yq, x[0], call.m) || !same_shape_result(yk, x[1], call.m));
  if (wants_grad({&x[0], &x[1], &wq, &wk, &yq, &yk})) {
    NONE_IF(yq.defined() || yk.defined());
    std::vector<int64_t> ints = rot.ints();
    ints.push_back(wq.defined());
    ints.push_back(wk.defined());
    return wrap(QkNormFn::apply(x[0], x[1], given(wq), given(wk), given(rot.turns), given(rot.positions), ints, rot.size, eps));
  }
  const bool given_q = yq.defined(), given_k = yk.defined();
  const int rc = call.forward(x[0], x[1], wq, wk, rot, yq, yk);
  if (rc != TTT_OK) throw_error(rc);
  if (given_q) overwritten(yq);
  if (given_k) overwritten(yk);
  return wrap({yq, yk});
  END_HANDLE_TH_ERRORS
}
// qk_norm_backward(q, k, grad_q_out, grad_k_out, q_weight | None, k_weight | None, rotation (7), eps, grad_q, grad_k) ->
// (grad_q, grad_k, grad_q_weight | None, grad_k_weight | None): into the given tensors, for the layer's own node
PyObject* py_qk_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 16)) return nullptr;
  Tensor x[4], wq, wk, d[2], dwq, dwk;
  QkNorm call;
  Rotation rot;
  NONE_IF(!tensors(args, x) || !optional_tensor(args[4], wq) || !optional_tensor(args[5], wk) || !rotation_args(args + 6, rot) ||
          !tensors(args + 14, d));
  const double eps = PyFloat_AsDouble(args[13]);
  if (PyErr_Occurred()) return nullptr;
  NONE_IF(!call.set(x[0], x[1], wq, wk, eps) || !rot.set(call.m));
  for (int i = 0; i < 2; ++i)
    NONE_IF(!head_rows(x[2 + i], call.m.dev, call.m.dt) || x[2 + i].sizes() != x[i].sizes() || !same_shape_result(d[i], x[i], call.m));
  const int rc = call.backward(x[0], x[1], x[2], x[3], wq, wk, rot, d[0], d[1], dwq, dwk);
  if (rc != TTT_OK) throw_error(rc);
  for (const Tensor& t : d) overwritten(t);
  return wrap({d[0], d[1], dwq, dwk});
  END_HANDLE_TH_ERRORS
}

// causal_conv(x, weight, bias | None, state | None, activation, starts | None, state_out | None) -> (y, state), recorded for autograd
// where that is on and asked for | None
PyObject* py_causal_conv(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 7)) return nullptr;
  Tensor x[2], bias, state, starts, out, y;
  NONE_IF(!tensors(args, x) || !optional_tensor(args[2], bias) || !optional_tensor(args[3], state) || !optional_tensor(args[5], starts) ||
          !optional_tensor(args[6], out));
  const int64_t act = as_int(args[4]);
  if (PyErr_Occurred()) return nullptr;
  refuse_tangents({&x[0], &x[1], &bias, &state, &out});
  Conv call;
  NONE_IF(!call.set(x[0], x[1], bias, state, starts, act) || !call.held(out));
  if (wants_grad({&x[0], &x[1], &bias, &state, &out})) {  // (a given state is not recorded: the caller's check refuses it)
    NONE_IF(out.defined());
    return wrap(ConvFn::apply(x[0], x[1], given(bias), given(state), given(starts),
                              std::vector<int64_t>{bias.defined(), state.defined(), starts.defined(), act}));
  }
  const bool given_out = out.defined();
  const int rc = call.forward(x[0], x[1], bias, state, starts, y, out);
  if (rc != TTT_OK) throw_error(rc);
  if (given_out) overwritten(out);
  return wrap({y, out});
  END_HANDLE_TH_ERRORS
}
// group_norm(x, groups, weight | None, bias | None, gate | None, activation, eps, over) -> y, recorded for autograd where that is on
// and asked for | None
PyObject* py_group_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 8)) return nullptr;
  Tensor x[1], w, b, gate, y, stats;
  NONE_IF(!tensors(args, x) || !optional_tensor(args[2], w) || !optional_tensor(args[3], b) || !optional_tensor(args[4], gate));
  const int64_t groups = as_int(args[1]), act = as_int(args[5]), over = as_int(args[7]);
  const double eps = PyFloat_AsDouble(args[6]);
  if (PyErr_Occurred()) return nullptr;
  refuse_tangents({&x[0], &w, &b, &gate});
  Norm call;
  NONE_IF(groups > INT32_MAX || !call.set(x[0], w, b, gate, groups, act, over, eps));
  if (wants_grad({&x[0], &w, &b, &gate}))
    return THPVariable_Wrap(NormFn::apply(x[0], given(w), given(b), given(gate),
                                          std::vector<int64_t>{w.defined(), b.defined(), gate.defined(), groups, act, over}, eps));
  const int rc = call.forward(x[0], w, b, gate, false, y, stats);
  if (rc != TTT_OK) throw_error(rc);
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// selective(x, dt, A, B, C, D | None, z | None, dt_bias | None, state | None, starts | None, softplus, state_out | None) -> (y, state),
// recorded for autograd where that is on and asked for | None
PyObject* py_selective(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 12)) return nullptr;
  Tensor t[5], o[5], out, y, saved;
  NONE_IF(!tensors(args, t));
  for (int i = 0; i < 5; ++i) NONE_IF(!optional_tensor(args[5 + i], o[i]));
  NONE_IF(!optional_tensor(args[11], out));
  const int64_t softplus = as_int(args[10]);
  if (PyErr_Occurred()) return nullptr;
  for (int i = 3; i < 5; ++i)
    if (t[i].dim() == 3) t[i] = t[i].unsqueeze(2);  // one group
  refuse_tangents({&t[0], &t[1], &t[2], &t[3], &t[4], &o[0], &o[1], &o[2], &o[3], &out});
  Selective call;
  NONE_IF(!call.set(t, o, softplus) || !call.held(out));
  if (wants_grad({&t[0], &t[1], &t[2], &t[3], &t[4], &o[0], &o[1], &o[2], &o[3], &out})) {
    NONE_IF(out.defined());
    return wrap(SelectiveFn::apply(t[0], t[1], t[2], t[3], t[4], given(o[0]), given(o[1]), given(o[2]), given(o[3]), given(o[4]),
                                   std::vector<int64_t>{o[0].defined(), o[1].defined(), o[2].defined(), o[3].defined(), o[4].defined(), softplus}));
  }
  const bool given_out = out.defined();
  const int rc = call.forward(t, o, false, y, out, saved);
  if (rc != TTT_OK) throw_error(rc);
  if (given_out) overwritten(out);
  return wrap({y, out});
  END_HANDLE_TH_ERRORS
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"init", py_init, METH_O, nullptr},
                         FAST(set_status),
                         FAST(linear_forward),
                         FAST(linear_partial),
                         FAST(linear_backward),
                         FAST(linear_apply),
                         FAST(mlp_forward),
                         FAST(mlp_apply),
                         FAST(param_key),
                         FAST(stream_key),
                         FAST(layer_infer),
                         FAST(layer_train),
                         FAST(gated),
                         FAST(rotary),
                         FAST(qk_norm),
                         FAST(qk_norm_backward),
                         FAST(causal_conv),
                         FAST(group_norm),
                         FAST(selective),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
