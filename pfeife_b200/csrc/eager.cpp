// Eager calls of the differentiable ops, from Python's arguments to the launches and the autograd node,
// as a Python module (`pfeife_b200_eager`).
//
// What bounds a small call is the host: through Python an op took the caller 20 to 30 us forward and as
// much again backward, where autograd's thread also has to wait for the interpreter lock.  Here it takes
// a few: linear 6.1 us, MLP 9.8, LayerNorm with residual 6.1, attention 5.4.  (As a caller sees them, forward
// and backward of a LayerNorm with residual 160 -> 81 us, what is left being autograd's hop to its thread
// and back; logits of 4 images by ViT-Tiny 2540 -> 753 us.)
//
// Only the usual call is taken: plain CUDA tensors of one device and one 16-bit type, no autocast, nothing
// that observes ops (dispatch or function modes, transforms, traces, forward-mode gradients).  For every
// other call the functions return None, and the caller goes on in Python (ops/functional.py), which
// defines what each op means.  A backward whose tensors are not plain any more, or that is itself
// recorded, calls the registered backward op through the dispatcher, as the Python formulas do.  So does
// one that unpacks something in another order or type than the forward saved: hooks on saved tensors may
// return any tensor, and what the kernels assume of their operands is tested again in each backward.
//
// The kernel library is loaded by the caller beforehand with its symbols global.
#include <ATen/autocast_mode.h>
#include <ATen/core/PythonFallbackKernel.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <atomic>
#include <cmath>

#include "api.h"

namespace pfeife {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------------------------ launching
struct Failed { int code; const char* what; };      // an entry point refused the call
std::atomic<long long> g_launches{0};
PyObject* g_status_word = nullptr;                  // kernels.status_word
PyObject* g_check = nullptr;                        // _lib.check: raises for a code
constexpr int MAX_DEVICES = 64;
Tensor g_status[MAX_DEVICES];                       // kept: the buffer lives as long as the process

void ok(int code, const char* what) {
  if (code) throw Failed{code, what};
  g_launches.fetch_add(1, std::memory_order_relaxed);
}

// Called with the interpreter lock in forwards, which come before any backward on a device.
bool learn_status(int dev) {
  if (g_status[dev].defined()) return true;
  PyObject* d = THPDevice_New(at::Device(at::kCUDA, dev));
  PyObject* t = d ? PyObject_CallOneArg(g_status_word, d) : nullptr;
  Py_XDECREF(d);
  if (!t) return false;
  g_status[dev] = THPVariable_Unpack(t);
  Py_DECREF(t);
  return true;
}

struct Env {
  int dev, sms;
  int* status;
  void* stream;
  explicit Env(const Tensor& t) : dev(t.get_device()) {
    if (const int code = pf_bind_device(dev)) throw Failed{code, "pf_bind_device"};
    sms = at::cuda::getDeviceProperties(dev)->multiProcessorCount;
    status = static_cast<int*>(g_status[dev].data_ptr());
    stream = at::cuda::getCurrentCUDAStream(dev).stream();
  }
};

int code_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kHalf ? 1 : 2; }
int code_of(const Tensor& t) { return code_of(t.scalar_type()); }
const void* at_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
// packed values are read 16 bytes at a time; others are packed into memory of their own first
template <typename... T>
bool on_vectors(const T&... t) {
  return ((!t.defined() || !t.is_contiguous() || aligned(t)) && ...);
}
bool half(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}
Tensor empty(at::IntArrayRef sizes, const Tensor& like) { return empty(sizes, like.scalar_type(), like); }
Tensor floats(long long n, const Tensor& like) { return empty({n}, at::kFloat, like); }

// ------------------------------------------------------------------------------ which calls are taken
bool unobserved() {
  return !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::impl::torch_function_mode_enabled() &&
         !c10::impl::tls_is_dispatch_key_included(at::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !torch::jit::tracer::isTracing();
}

// A tensor whose memory holds its values: no wrapper, negative view or the like (each is a dispatch key),
// no forward-mode gradient, and not empty.  The usual keys are those of a tensor made outside inference mode,
// in which tensors lack some of them, whatever the mode of the first call.
bool plain(const Tensor& t, int dev) {
  static const uint64_t usual = [] {
    const c10::InferenceMode off(false);
    return at::empty({0}, at::device(at::kCUDA).dtype(at::kHalf)).key_set().raw_repr();
  }();
  return (t.key_set().raw_repr() & ~usual) == 0 && t.get_device() == dev && t.data_ptr() != nullptr &&
         !t._fw_grad(0).defined();
}
template <typename... T>
bool all_plain(const Tensor& first, const T&... more) {
  const int dev = first.get_device();
  return plain(first, dev) && ((!more.defined() || plain(more, dev)) && ...);
}

template <typename... T>
bool recorded(const T&... t) {
  return at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...) &&
         !c10::impl::tls_is_dispatch_key_excluded(at::DispatchKey::AutogradOther);
}

// Whether a backward may launch kernels itself.
template <typename... T>
bool direct(const Tensor& first, const T&... more) {
  return !at::GradMode::is_enabled() && unobserved() && all_plain(first, more...);
}

// fp32 values one after the other, as a forward kernel wrote them or as a caller's parameters are taken
bool packed_floats(const Tensor& t, int64_t n) {
  return t.scalar_type() == at::kFloat && t.numel() == n && t.is_contiguous();
}
// values of the type and sizes of `like`
bool matches(const Tensor& t, const Tensor& like) {
  return t.scalar_type() == like.scalar_type() && t.sizes() == like.sizes();
}

c10::IValue opt(const Tensor& t) { return t.defined() ? c10::IValue(t) : c10::IValue(); }

// A registered op through the dispatcher.
torch::jit::Stack dispatched(const char* name, torch::jit::Stack stack) {
  c10::Dispatcher::singleton().findSchemaOrThrow(name, "").callBoxed(stack);
  return stack;
}
Tensor given(const c10::IValue& v) {                // an empty tensor stands for "not needed"
  const Tensor& t = v.toTensor();
  return t.numel() ? t : Tensor();
}
Tensor as(const Tensor& t, const c10::IValue& saved) {       // in the type that a forward took down
  const auto type = static_cast<at::ScalarType>(saved.toInt());
  return !t.defined() || t.scalar_type() == type ? t : t.to(type);
}

// Tensors that a call may leave out reach a node as optionals, which count as inputs only when given.
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor value(const Maybe& t) { return t ? *t : Tensor(); }

// Runs the launches of a backward below autograd; a refused call raises what it raises in Python.
template <typename F>
auto below(F&& f) {
  try {
    at::AutoDispatchBelowADInplaceOrView guard;
    return f();
  } catch (const Failed& e) {
    pybind11::gil_scoped_acquire lock;
    PyObject* r = PyObject_CallFunction(g_check, "is", e.code, e.what);
    Py_XDECREF(r);
    python_error raised;
    raised.persist();
    throw raised;
  }
}

// ------------------------------------------------------------------------------ GEMM
enum Epi { NONE, GELU, DGELU, GELU_TANH, DGELU_TANH, SILU };          // gemm_sm100.cu
constexpr int EPI_OF_ACT[4] = {NONE, GELU, GELU_TANH, SILU};

// x as rows the TMA can read
Tensor rows(const Tensor& x) {
  Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if (r.stride(1) != 1 || r.stride(0) % 8 || !aligned(r)) r = r.contiguous();
  return r;
}
bool readable(const Tensor& m) {
  return m.dim() == 2 && m.stride(1) == 1 && m.stride(0) % 8 == 0 && aligned(m);
}
// all operands of 16 bits, as is the result
Tensor gemm(const Env& e, const Tensor& a, const Tensor& b, bool a_mn, bool b_mn, const Tensor& bias = {},
            const Tensor& residual = {}, const Tensor& aux = {}, int epi = NONE) {
  const long long M = a.size(a_mn), K = a.size(!a_mn), N = b.size(b_mn);
  Tensor out = empty({M, N}, a);
  ok(pf_gemm(a.data_ptr(), b.data_ptr(), out.data_ptr(), (int)M, (int)N, (int)K, a.stride(0), b.stride(0), N,
             a_mn, b_mn, code_of(a), code_of(a), at_or_null(bias), bias.defined() ? code_of(bias) : 0,
             at_or_null(residual), residual.defined() ? residual.stride(0) : 0,
             const_cast<void*>(at_or_null(aux)), aux.defined() ? aux.stride(0) : 0, epi, 0, 1.0f, e.status,
             e.sms, 0, nullptr, 0, e.stream),
     "pf_gemm");
  return out;
}
Tensor colsum(const Env& e, const Tensor& x) {
  Tensor out = at::zeros({x.size(1)}, x.options().dtype(at::kFloat));
  ok(pf_colsum(x.data_ptr(), out.data_ptr(), x.size(0), (int)x.size(1), x.stride(0), code_of(x), e.sms,
               e.stream),
     "pf_colsum");
  return out;
}

std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  auto s = x.sizes().vec();
  s.back() = n;
  return s;
}

// ------------------------------------------------------------------------------ linear
bool bias_fits(const Tensor& b, int64_t n) { return !b.defined() || (b.dim() == 1 && b.size(0) == n && b.is_contiguous() && (half(b) || b.scalar_type() == at::kFloat)); }
bool layer_fits(const Tensor& x, const Tensor& w, const Tensor& b) {
  return x.dim() >= 2 && half(x) && w.scalar_type() == x.scalar_type() && readable(w) &&
         w.size(1) == x.size(-1) && w.size(1) % 8 == 0 && bias_fits(b, w.size(0)) &&
         x.numel() / x.size(-1) < (1ll << 31) && w.size(0) < (1ll << 31);
}
bool residual_fits(const Tensor& r, const Tensor& x, int64_t n) {
  return !r.defined() || (r.scalar_type() == x.scalar_type() && r.dim() == x.dim() && r.size(-1) == n &&
                          r.numel() / n == x.numel() / x.size(-1));
}

std::pair<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& res,
                                         int act) {
  const Env e(x);
  const Tensor x2 = rows(x), r2 = res.defined() ? rows(res) : Tensor();
  const Tensor aux = act ? empty({x2.size(0), w.size(0)}, x) : Tensor();
  const Tensor y = gemm(e, x2, w, false, false, b, r2, aux, EPI_OF_ACT[act]);
  const auto shape = with_last(x, w.size(0));
  return {y.view(shape), act ? aux.view(shape) : aux};
}
// whether linear_gradients can read what a backward unpacked, beside a gradient of the output
bool gradients_fit(const Tensor& dz, const Tensor& x, const Tensor& w) {
  return layer_fits(x, w, {}) && x.scalar_type() == dz.scalar_type() && dz.size(-1) == w.size(0) &&
         x.numel() / x.size(-1) == dz.numel() / dz.size(-1);
}
// gradients of x, w, b from that of the pre-activation
void linear_gradients(const Env& e, const Tensor& dz2, const Tensor& x, const Tensor& w, bool need_dx,
                      bool need_dw, bool need_db, Tensor& dx, Tensor& dw, Tensor& db) {
  if (need_dx) dx = gemm(e, dz2, w, false, true).view(x.sizes());
  if (need_dw) dw = gemm(e, dz2, rows(x), true, true);
  if (need_db) db = colsum(e, dz2);
}

struct DirectLinear : torch::autograd::Function<DirectLinear> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w, Maybe bias, Maybe residual, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor b = value(bias), res = value(residual);
    auto [y, aux] = linear_forward(x, w, b, res, (int)act);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, b, aux});
    ctx->saved_data["act"] = act;
    if (bias) ctx->saved_data["type"] = (int64_t)b.scalar_type();
    ctx->saved_data["res"] = res.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &b = s[2], &aux = s[3];
    if (!grads[0].defined()) return variable_list(5);
    const Tensor dy = grads[0].contiguous();
    const int act = (int)ctx->saved_data["act"].toInt();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1),
               nb = b.defined() && ctx->needs_input_grad(2),
               nr = ctx->saved_data["res"].toBool() && ctx->needs_input_grad(2 + b.defined());
    Tensor dx, dw, db;
    if (direct(dy, x, w, b, aux) && gradients_fit(dy, x, w) && (!act || matches(aux, dy))) {
      below([&] {
        const Env e(dy);
        Tensor dz = rows(dy);
        if (act) {
          constexpr int DACT[4] = {0, 10, 11, 12};                    // elementwise.cu
          const Tensor z = rows(aux).contiguous();
          Tensor out = empty(dz.sizes(), dz);
          dz = dz.contiguous();
          ok(pf_elementwise(dz.data_ptr(), z.data_ptr(), out.data_ptr(), dz.numel(), DACT[act], code_of(dz),
                            e.sms, e.stream),
             "pf_elementwise");
          dz = out;
        }
        linear_gradients(e, dz, x, w, nx, nw, nb, dx, dw, db);
        return 0;
      });
    } else {
      auto out = dispatched("pfeife::linear_bwd", {dy, x, w, aux.defined() ? aux : dy.new_empty({0}),
                                                   (int64_t)act, nx, nw, nb, opt(b)});
      dx = given(out[0]); dw = given(out[1]); db = given(out[2]);
    }
    return {nx ? dx : Tensor(), nw ? dw : Tensor(), nb ? as(db, ctx->saved_data["type"]) : Tensor(),
            nr ? dy : Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ feed-forward block
struct DirectMlp : torch::autograd::Function<DirectMlp> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w1, Maybe bias1, Tensor w2, Maybe bias2,
                        Maybe residual, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor b1 = value(bias1), b2 = value(bias2), res = value(residual);
    auto [a1, z1] = linear_forward(x, w1, b1, {}, (int)act);
    const Tensor y = linear_forward(a1, w2, b2, res, 0).first;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w1, w2, z1, a1, b1, b2});
    ctx->saved_data["act"] = act;
    if (bias1) ctx->saved_data["type1"] = (int64_t)b1.scalar_type();
    if (bias2) ctx->saved_data["type2"] = (int64_t)b2.scalar_type();
    ctx->saved_data["res"] = res.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w1 = s[1], &w2 = s[2], &z1 = s[3], &a1 = s[4], &b1 = s[5], &b2 = s[6];
    if (!grads[0].defined()) return variable_list(7);
    const Tensor dy = grads[0].contiguous();
    const int act = (int)ctx->saved_data["act"].toInt();
    const bool nx = ctx->needs_input_grad(0),
               nr = ctx->saved_data["res"].toBool() &&
                    ctx->needs_input_grad(3 + b1.defined() + b2.defined());
    Tensor dx, dw1, db1, dw2, db2, none;
    if (direct(dy, x, w1, w2, z1, a1, b1, b2) && gradients_fit(dy, a1, w2) && gradients_fit(a1, x, w1) &&
        matches(z1, a1)) {
      below([&] {
        const Env e(dy);
        const Tensor dy2 = rows(dy);
        const Tensor dz1 = gemm(e, dy2, w2, false, true, {}, {}, rows(z1), act == 1 ? DGELU : DGELU_TANH);
        linear_gradients(e, dy2, a1, w2, false, true, b2.defined(), none, dw2, db2);
        linear_gradients(e, dz1, x, w1, nx, true, b1.defined(), dx, dw1, db1);
        return 0;
      });
    } else {
      auto out = dispatched("pfeife::mlp_bwd", {dy, x, w1, w2, z1, a1, (int64_t)act, nx, b1.defined(),
                                                b2.defined(), opt(b1), opt(b2)});
      dx = given(out[0]); dw1 = given(out[1]); db1 = given(out[2]); dw2 = given(out[3]); db2 = given(out[4]);
    }
    return {nx ? dx : Tensor(), dw1, b1.defined() ? as(db1, ctx->saved_data["type1"]) : Tensor(), dw2,
            b2.defined() ? as(db2, ctx->saved_data["type2"]) : Tensor(), nr ? dy : Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ norms
struct NormOut { Tensor y, h, mean, rstd; };
NormOut norm_forward(const Tensor& x, const Tensor& gamma, const Tensor& beta, const Tensor& res, double eps,
                     bool rms) {
  const Env e(x);
  const Tensor xc = x.contiguous(), rc = res.defined() ? res.contiguous() : res;
  const int64_t N = x.size(-1), n = x.numel() / N;
  NormOut o;
  o.y = empty(x.sizes(), x);
  if (res.defined()) o.h = empty(x.sizes(), x);
  o.mean = floats(n, x);
  o.rstd = floats(n, x);
  ok(pf_norm_fwd(xc.data_ptr(), at_or_null(rc), gamma.data_ptr(), at_or_null(beta), o.y.data_ptr(),
                 const_cast<void*>(at_or_null(o.h)), o.mean.data_ptr(), o.rstd.data_ptr(), n, (int)N, (float)eps,
                 rms, code_of(x), e.stream),
     "pf_norm_fwd");
  return o;
}

struct DirectNorm : torch::autograd::Function<DirectNorm> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor gamma, Maybe bias, Maybe residual,
                               double eps, bool rms) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor beta = value(bias), res = value(residual);
    const NormOut o = norm_forward(x, gamma, beta, res, eps, rms);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({res.defined() ? o.h : x, gamma, beta, o.mean, o.rstd});
    ctx->saved_data["rms"] = rms;
    ctx->saved_data["res"] = res.defined();
    if (res.defined()) return {o.y, o.h};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &h = s[0], &gamma = s[1], &beta = s[2], &mean = s[3], &rstd = s[4];
    const bool rms = ctx->saved_data["rms"].toBool(), has_res = ctx->saved_data["res"].toBool();
    Tensor dh, dy = grads[0];
    if (has_res && grads[1].defined()) dh = grads[1].contiguous();
    if (!dy.defined()) {
      if (!dh.defined()) return variable_list(6);
      dy = at::zeros_like(h);
    }
    dy = dy.contiguous();
    const int64_t n = h.numel() / h.size(-1);
    Tensor dx, dg, db;
    if (direct(dy, dh, h, gamma, beta, mean, rstd) && half(h) && matches(h, dy) &&
        (!dh.defined() || matches(dh, dy)) && on_vectors(dy, dh, h, gamma) && packed_floats(gamma, h.size(-1)) && packed_floats(mean, n) &&
        packed_floats(rstd, n)) {
      below([&] {
        const Env e(dy);
        const Tensor hc = h.contiguous();
        const int64_t N = h.size(-1);
        dx = empty(h.sizes(), h);
        dg = floats(N, h);
        if (beta.defined() && !rms) db = floats(N, h);
        const Tensor scratch = floats((int64_t)pf_norm_bwd_ctas(n, e.sms) * 2 * N, h);
        ok(pf_norm_bwd(dy.data_ptr(), hc.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                       at_or_null(dh), dx.data_ptr(), dg.data_ptr(), const_cast<void*>(at_or_null(db)),
                       scratch.data_ptr(), n, (int)N, rms, 0, code_of(h), e.sms, e.stream),
           "pf_norm_bwd");
        return 0;
      });
    } else {
      auto out = dispatched("pfeife::norm_bwd",
                            {dy, opt(dh), h, gamma, mean, rstd, rms, beta.defined(), opt(beta)});
      dx = out[0].toTensor(); dg = given(out[1]); db = given(out[2]);
    }
    return {dx, dg, beta.defined() ? db : Tensor(), has_res ? dx : Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ attention
struct View { const char* at; long long strides[3]; };                // of q, k or v: batch, seq, head
View view_of(const Tensor& t) {
  return {static_cast<const char*>(t.data_ptr()), {t.stride(0), t.stride(1), t.stride(2)}};
}
View slice_of(const Tensor& qkv, int i) {
  return {static_cast<const char*>(qkv.data_ptr()) + i * qkv.stride(2) * 2,
          {qkv.stride(0), qkv.stride(1), qkv.stride(3)}};
}
Tensor readable_heads(const Tensor& t) {
  const bool fits = t.stride(3) == 1 && aligned(t) && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
                    t.stride(2) % 8 == 0;
  return fits ? t : t.contiguous();
}

std::pair<Tensor, Tensor> attention_forward(const Tensor& like, const View& q, const View& k, const View& v,
                                            int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t D,
                                            bool causal, double scale) {
  const Env e(like);
  const Tensor o = empty({B, Sq, H, D}, like), lse = empty({B, H, Sq}, at::kFloat, like);
  ok(pf_attn_fwd(q.at, k.at, v.at, o.data_ptr(), lse.data_ptr(), (int)B, (int)H, (int)Sq, (int)Sk, (int)D,
                 q.strides, k.strides, v.strides, causal, (float)scale, code_of(like), e.status, e.stream),
     "pf_attn_fwd");
  return {o, lse};
}
// gradients to views of equal strides for k and v
void attention_backward(const Tensor& dout, const View& q, const View& k, const View& v, const Tensor& o,
                        const Tensor& lse, const View& dq, const View& dk, const View& dv, int64_t Sk,
                        bool causal, double scale) {
  const Env e(dout);
  const int B = (int)o.size(0), Sq = (int)o.size(1), H = (int)o.size(2), D = (int)o.size(3);
  const Tensor stats = floats((int64_t)B * H * ((Sq + 127) / 128) * 256, dout);
  const int kib = pf_attn_bwd_scratch(B, H, Sq, (int)Sk, D, causal);
  const Tensor scratch = kib ? floats(kib * 256ll, dout) : Tensor();
  ok(pf_attn_bwd(dout.data_ptr(), q.at, k.at, v.at, o.data_ptr(), lse.data_ptr(), stats.data_ptr(),
                 const_cast<void*>(at_or_null(scratch)), const_cast<char*>(dq.at), const_cast<char*>(dk.at),
                 const_cast<char*>(dv.at), B, H, Sq, (int)Sk, D, q.strides, k.strides, v.strides, dq.strides,
                 dk.strides, causal, (float)scale, code_of(dout), e.status, e.sms, e.stream),
     "pf_attn_bwd");
}

std::pair<Tensor, Tensor> heads_forward(const Tensor& q, const Tensor& k, const Tensor& v, bool causal,
                                        double scale) {
  const Tensor qr = readable_heads(q), kr = readable_heads(k), vr = readable_heads(v);
  return attention_forward(q, view_of(qr), view_of(kr), view_of(vr), q.size(0), q.size(1), k.size(1),
                           q.size(2), q.size(3), causal, scale);
}

// whether a backward can read what it unpacked, beside a gradient of the output
bool heads_fit(const Tensor& dout, const Tensor& o, const Tensor& lse) {
  return half(dout) && matches(o, dout) && on_vectors(o) &&
         packed_floats(lse, dout.size(0) * dout.size(1) * dout.size(2));
}

struct DirectAttention : torch::autograd::Function<DirectAttention> {
  static Tensor forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v, bool causal, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [o, lse] = heads_forward(q, k, v, causal, scale);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, o, lse});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &o = s[3], &lse = s[4];
    if (!grads[0].defined()) return variable_list(5);
    const Tensor dout = grads[0].contiguous();
    const bool causal = ctx->saved_data["causal"].toBool();
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor dq, dk, dv;
    if (direct(dout, q, k, v, o, lse) && heads_fit(dout, o, lse) && matches(q, dout) &&
        matches(k, v) && k.scalar_type() == q.scalar_type()) {
      below([&] {
        const Tensor qr = readable_heads(q), kr = readable_heads(k), vr = readable_heads(v);
        dq = empty(q.sizes(), q);
        dk = empty(k.sizes(), k);
        dv = empty(v.sizes(), v);
        attention_backward(aligned(dout) ? dout : dout.clone(), view_of(qr), view_of(kr), view_of(vr),
                           o.contiguous(), lse, view_of(dq), view_of(dk), view_of(dv), k.size(1), causal,
                           scale);
        return 0;
      });
    } else {
      auto out = dispatched("pfeife::attn_bwd", {dout, q, k, v, o, lse, causal, scale});
      dq = out[0].toTensor(); dk = out[1].toTensor(); dv = out[2].toTensor();
    }
    return {dq, dk, dv, Tensor(), Tensor()};
  }
};

bool packed_fits(const Tensor& t) {                  // [B, S, 3, H, D], read in place
  return t.stride(4) == 1 && aligned(t) && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
         t.stride(2) % 8 == 0 && t.stride(3) % 8 == 0;
}
std::pair<Tensor, Tensor> packed_forward(const Tensor& t, bool causal, double scale) {
  return attention_forward(t, slice_of(t, 0), slice_of(t, 1), slice_of(t, 2), t.size(0), t.size(1), t.size(1),
                           t.size(3), t.size(4), causal, scale);
}

struct DirectAttentionQkv : torch::autograd::Function<DirectAttentionQkv> {
  static Tensor forward(AutogradContext* ctx, Tensor qkv, bool causal, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [o, lse] = packed_forward(qkv, causal, scale);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({qkv, o, lse});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &qkv = s[0], &o = s[1], &lse = s[2];
    if (!grads[0].defined()) return variable_list(3);
    const Tensor dout = grads[0].contiguous();
    const bool causal = ctx->saved_data["causal"].toBool();
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor d;
    if (direct(dout, qkv, o, lse) && heads_fit(dout, o, lse) && qkv.scalar_type() == dout.scalar_type() &&
        qkv.dim() == 5 && qkv.numel() == 3 * dout.numel() && packed_fits(qkv)) {
      below([&] {
        d = empty(qkv.sizes(), qkv);
        attention_backward(aligned(dout) ? dout : dout.clone(), slice_of(qkv, 0), slice_of(qkv, 1),
                           slice_of(qkv, 2), o.contiguous(), lse, slice_of(d, 0), slice_of(d, 1),
                           slice_of(d, 2), qkv.size(1), causal, scale);
        return 0;
      });
    } else {
      d = dispatched("pfeife::attn_qkv_bwd", {dout, qkv, o, lse, causal, scale})[0].toTensor();
    }
    return {d, Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ rotary embedding, GLU
Tensor rope_forward(const Tensor& x, const Tensor& cos, const Tensor& sin, bool inverse) {
  const Env e(x);
  const Tensor out = empty(x.sizes(), x);
  ok(pf_rope_qkv(x.data_ptr(), out.data_ptr(), cos.data_ptr(), sin.data_ptr(), x.size(0) * x.size(1),
                 (int)x.size(1), (int)x.size(3), (int)x.size(4), inverse, code_of(x), e.stream),
     "pf_rope_qkv");
  return out;
}
bool table_fits(const Tensor& t, const Tensor& x) {  // of cosines or sines, for x [B, S, 3, H, D]
  return t.scalar_type() == at::kFloat && t.dim() == 2 && t.is_contiguous() && aligned(t) &&
         t.size(0) >= x.size(1) && t.size(1) == x.size(4) / 2;
}
struct DirectRopeQkv : torch::autograd::Function<DirectRopeQkv> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor cos, Tensor sin) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({cos, sin});
    return rope_forward(x, cos, sin, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &cos = s[0], &sin = s[1];
    const Tensor dy = grads[0].contiguous();
    Tensor dx;
    if (direct(dy, cos, sin) && half(dy) && aligned(dy) && table_fits(cos, dy) && table_fits(sin, dy))
      below([&] { dx = rope_forward(dy, cos, sin, true); return 0; });
    else dx = dispatched("pfeife::rope_qkv_apply", {dy, cos, sin, true})[0].toTensor();
    return {dx, Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ rotations of any layout, head norms
// Heads [B, S, H, D], or one of the slices of a projection [B, S, 3, H, D], as qk_rope.cu takes them.
struct HeadView {
  char* at;
  long long steps[3];
  explicit HeadView(const Tensor& t, int slice = -1) : at(static_cast<char*>(t.data_ptr())) {
    const bool packed = slice >= 0;
    const int d[3] = {0, 1, packed ? 3 : 2};
    for (int i = 0; i < 3; ++i) steps[i] = t.size(d[i]) > 1 ? t.stride(d[i]) : 0;
    if (packed) at += slice * t.stride(2) * (long long)t.element_size();
  }
};
bool number(const Tensor& t) { return half(t) || t.scalar_type() == at::kFloat; }
bool head_view_fits(const Tensor& t, int dim) {
  return t.dim() == dim && number(t) && t.numel() > 0 && t.stride(dim - 1) == 1 && t.size(dim - 1) >= 2 &&
         t.size(dim - 1) <= 256 && (dim == 4 || t.size(2) == 3);
}
// tables and positions for x [B, S, .., D]
bool angles_fit(const Tensor& x, const Tensor& cos, const Tensor& sin, const Tensor& pos) {
  const int64_t B = x.size(0), S = x.size(1);
  for (const Tensor* t : {&cos, &sin})
    if (t->scalar_type() != at::kFloat || t->dim() != 2 || !t->is_contiguous()) return false;
  if (cos.sizes() != sin.sizes() || cos.size(1) < 1 || 2 * cos.size(1) > x.size(-1)) return false;
  if (!pos.defined()) return cos.size(0) >= S;
  return pos.scalar_type() == at::kLong &&
         ((pos.dim() == 1 && pos.size(0) == S) || (pos.dim() == 2 && pos.size(0) == B && pos.size(1) == S));
}
struct Angles {
  const Tensor &cos, &sin, &pos;
  long long steps[2];
  Angles(const Tensor& c, const Tensor& s, const Tensor& p) : cos(c), sin(s), pos(p), steps{0, 0} {
    if (!p.defined()) return;
    steps[0] = p.dim() == 2 ? p.stride(0) : 0;
    steps[1] = p.stride(-1);
  }
};
Tensor inner_packed(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

// q -> yq, and where given k -> yk and (slices of a projection) v -> yv
void heads_run(const Env& e, const Tensor& like, const HeadView& q, const HeadView* k, const HeadView* v, const HeadView& yq,
               const HeadView* yk, const HeadView* yv, const Tensor& wq, const Tensor& wk, const Angles& a,
               int64_t hq, int64_t hk, bool interleaved, bool inverse, double eps) {
  ok(pf_heads_fwd(q.at, k ? k->at : nullptr, v ? v->at : nullptr, yq.at, yk ? yk->at : nullptr, yv ? yv->at : nullptr,
                  at_or_null(wq), at_or_null(wk), a.cos.data_ptr(), a.sin.data_ptr(), at_or_null(a.pos), like.size(0),
                  (int)like.size(1), (int)hq, (int)hk, (int)like.size(-1), (int)(2 * a.cos.size(1)), q.steps,
                  k ? k->steps : nullptr, yq.steps, yk ? yk->steps : nullptr, a.steps, a.cos.size(0), interleaved,
                  inverse, (float)eps, code_of(like), e.sms, e.stream),
     "pf_heads_fwd");
}
Tensor rotate(const Tensor& x, const Tensor& cos, const Tensor& sin, const Tensor& pos, bool interleaved, bool inverse) {
  const Env e(x);
  const Tensor y = empty(x.sizes(), x);
  const Angles a(cos, sin, pos);
  if (x.dim() == 4) {
    heads_run(e, x, HeadView(x), nullptr, nullptr, HeadView(y), nullptr, nullptr, {}, {}, a, x.size(2), 0, interleaved,
              inverse, 0.0);
  } else {
    const HeadView k(x, 1), v(x, 2), yk(y, 1), yv(y, 2);
    heads_run(e, x, HeadView(x, 0), &k, &v, HeadView(y, 0), &yk, &yv, {}, {}, a, x.size(3), x.size(3), interleaved,
              inverse, 0.0);
  }
  return y;
}
struct DirectRotate : torch::autograd::Function<DirectRotate> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor cos, Tensor sin, Maybe positions, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({cos, sin, value(positions)});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["dim"] = x.dim();
    return rotate(x, cos, sin, value(positions), interleaved, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &cos = s[0], &sin = s[1], &pos = s[2];
    const Tensor dy = inner_packed(grads[0]);
    const bool interleaved = ctx->saved_data["interleaved"].toBool();
    const int dim = (int)ctx->saved_data["dim"].toInt();
    Tensor dx;
    if (direct(dy, cos, sin, pos) && head_view_fits(dy, dim) && angles_fit(dy, cos, sin, pos))
      below([&] { dx = rotate(dy, cos, sin, pos, interleaved, true); return 0; });
    else
      dx = dispatched(dim == 4 ? "pfeife::rope_at" : "pfeife::rope_qkv_at",
                      {dy, cos, sin, opt(pos), interleaved, true})[0].toTensor();
    return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

bool gain_fits(const Tensor& w, const Tensor& x) { return packed_floats(w, x.size(-1)) && w.dim() == 1; }
bool same_heads(const Tensor& q, const Tensor& k) {
  return head_view_fits(q, 4) && head_view_fits(k, 4) && q.scalar_type() == k.scalar_type() && q.size(0) == k.size(0) &&
         q.size(1) == k.size(1) && q.size(3) == k.size(3);
}
// q and k, or the projection qkv in the place of q (k not defined)
variable_list norm_rotate(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& cos,
                          const Tensor& sin, const Tensor& pos, double eps, bool interleaved) {
  const Env e(q);
  const Angles a(cos, sin, pos);
  const Tensor y = empty(q.sizes(), q);
  if (k.defined()) {
    const Tensor z = empty(k.sizes(), k);
    const HeadView kv(k), zv(z);
    heads_run(e, q, HeadView(q), &kv, nullptr, HeadView(y), &zv, nullptr, wq, wk, a, q.size(2), k.size(2), interleaved,
              false, eps);
    return {y, z};
  }
  const HeadView kv(q, 1), vv(q, 2), zk(y, 1), zv(y, 2);
  heads_run(e, q, HeadView(q, 0), &kv, &vv, HeadView(y, 0), &zk, &zv, wq, wk, a, q.size(3), q.size(3), interleaved,
            false, eps);
  return {y};
}
struct DirectNormRotate : torch::autograd::Function<DirectNormRotate> {
  static variable_list forward(AutogradContext* ctx, Tensor q, Maybe keys, Tensor wq, Tensor wk, Tensor cos,
                               Tensor sin, Maybe positions, double eps, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({q, value(keys), wq, wk, cos, sin, value(positions)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return norm_rotate(q, value(keys), wq, wk, cos, sin, value(positions), eps, interleaved);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &wq = s[2], &wk = s[3], &cos = s[4], &sin = s[5], &pos = s[6];
    const double eps = ctx->saved_data["eps"].toDouble();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), two = k.defined();
    const Tensor gq = inner_packed(grads[0]), gk = two ? inner_packed(grads[1]) : Tensor();
    Tensor dq, dk, dwq, dwk;
    const bool fits = two ? same_heads(q, k) && matches(gq, q) && matches(gk, k)
                          : head_view_fits(q, 5) && matches(gq, q);
    if (direct(gq, gk, q, k, wq, wk, cos, sin, pos) && fits && gain_fits(wq, q) && gain_fits(wk, q) &&
        angles_fit(q, cos, sin, pos)) {
      below([&] {
        const Env e(gq);
        const Angles a(cos, sin, pos);
        const int D = (int)q.size(-1), hq = (int)q.size(two ? 2 : 3), hk = (int)(two ? k.size(2) : hq);
        dq = empty(q.sizes(), q);
        if (two) dk = empty(k.sizes(), k);
        dwq = floats(D, q);
        dwk = floats(D, q);
        const Tensor scratch = floats((int64_t)pf_heads_bwd_rows(hq, hk, e.sms) * D, q);
        const int at = two ? -1 : 0;
        const HeadView vgq(gq, at), vq(q, at), vdq(dq, at);
        const HeadView vgk = two ? HeadView(gk) : HeadView(gq, 1), vk = two ? HeadView(k) : HeadView(q, 1),
                       vdk = two ? HeadView(dk) : HeadView(dq, 1);
        char* gv = two ? nullptr : HeadView(gq, 2).at;
        char* dv = two ? nullptr : HeadView(dq, 2).at;
        ok(pf_heads_bwd(vgq.at, vgk.at, gv, vq.at, vk.at, vdq.at, vdk.at, dv, wq.data_ptr(), wk.data_ptr(),
                        dwq.data_ptr(), dwk.data_ptr(), scratch.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                        at_or_null(pos), q.size(0), (int)q.size(1), hq, hk, D, (int)(2 * cos.size(1)), vgq.steps,
                        vgk.steps, vq.steps, vk.steps, vdq.steps, vdk.steps, a.steps, cos.size(0), interleaved,
                        (float)eps, 0, code_of(q), e.sms, e.stream),
           "pf_heads_bwd");
        return 0;
      });
    } else if (two) {
      auto out = dispatched("pfeife::qk_norm_rope_bwd",
                            {gq, gk, q, k, wq, wk, cos, sin, opt(pos), eps, interleaved});
      dq = out[0].toTensor(); dk = out[1].toTensor(); dwq = given(out[2]); dwk = given(out[3]);
    } else {
      auto out = dispatched("pfeife::qk_norm_rope_qkv_bwd", {gq, q, wq, wk, cos, sin, opt(pos), eps, interleaved});
      dq = out[0].toTensor(); dwq = given(out[1]); dwk = given(out[2]);
    }
    return {dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor glu_forward(const Tensor& gu, bool gelu) {
  const Env e(gu);
  const int64_t H = gu.size(-1) / 2;
  const Tensor out = empty(with_last(gu, H), gu);
  ok(pf_glu_fwd(gu.data_ptr(), out.data_ptr(), gu.numel() / (2 * H), (int)H, gelu, code_of(gu), e.sms,
                e.stream),
     "pf_glu_fwd");
  return out;
}
struct DirectGlu : torch::autograd::Function<DirectGlu> {
  static Tensor forward(AutogradContext* ctx, Tensor gu, bool gelu) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({gu});
    ctx->saved_data["gelu"] = gelu;
    return glu_forward(gu, gelu);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor gu = ctx->get_saved_variables()[0];
    const Tensor dy = grads[0].contiguous();
    const bool gelu = ctx->saved_data["gelu"].toBool();
    Tensor d;
    if (direct(dy, gu) && gu.is_contiguous() && half(gu) && gu.scalar_type() == dy.scalar_type() &&
        gu.numel() == 2 * dy.numel() && on_vectors(gu, dy)) {
      below([&] {
        const Env e(dy);
        const int64_t H = gu.size(-1) / 2;
        d = empty(gu.sizes(), gu);
        ok(pf_glu_bwd(gu.data_ptr(), dy.data_ptr(), d.data_ptr(), gu.numel() / (2 * H), (int)H, gelu,
                      code_of(gu), e.sms, e.stream),
           "pf_glu_bwd");
        return 0;
      });
    } else {
      d = dispatched("pfeife::glu_bwd", {dy, gu, gelu})[0].toTensor();
    }
    return {d, Tensor()};
  }
};

// ------------------------------------------------------------------------------ mean cross entropy
struct LossOut { Tensor mean, lse, inv; };
LossOut loss_forward(const Tensor& logits, const Tensor& target, int64_t ignore) {
  const Env e(logits);
  const Tensor lc = logits.contiguous(), tc = target.contiguous();
  const int64_t n = lc.size(0), V = lc.size(1);
  const Tensor loss = floats(n, lc);
  LossOut o{empty({}, at::kFloat, lc), floats(n, lc), empty({}, at::kFloat, lc)};
  ok(pf_ce_fwd(lc.data_ptr(), tc.data_ptr(), loss.data_ptr(), o.lse.data_ptr(), n, (int)V, V, ignore,
               code_of(lc), e.sms, e.stream),
     "pf_ce_fwd");
  const int parts = pf_ce_mean_parts(n, e.sms);
  const Tensor scratch = parts > 1 ? floats(2 * parts, lc) : Tensor();
  ok(pf_ce_mean(loss.data_ptr(), tc.data_ptr(), const_cast<void*>(at_or_null(scratch)), o.mean.data_ptr(),
                o.inv.data_ptr(), n, ignore, e.sms, e.stream),
     "pf_ce_mean");
  return o;
}
struct DirectCrossEntropy : torch::autograd::Function<DirectCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, Tensor logits, Tensor target, int64_t ignore) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const LossOut o = loss_forward(logits, target, ignore);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, target, o.lse, o.inv});
    ctx->saved_data["ignore"] = ignore;
    return o.mean;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &logits = s[0], &target = s[1], &lse = s[2], &inv = s[3];
    const Tensor& g = grads[0];
    if (!g.defined()) return variable_list(3);
    const int64_t ignore = ctx->saved_data["ignore"].toInt();
    const Tensor scale = g * inv;
    Tensor d;
    if (direct(scale, logits, target, lse) && logits.dim() == 2 &&
        (half(logits) || logits.scalar_type() == at::kFloat) && target.scalar_type() == at::kLong &&
        target.numel() == logits.size(0) && packed_floats(lse, logits.size(0)) && packed_floats(scale, 1)) {
      below([&] {
        const Env e(scale);
        const Tensor lc = logits.contiguous(), tc = target.contiguous();
        d = empty(lc.sizes(), lc);
        ok(pf_ce_bwd(lc.data_ptr(), tc.data_ptr(), lse.data_ptr(), scale.data_ptr(), d.data_ptr(), lc.size(0),
                     (int)lc.size(1), lc.size(1), ignore, 0, code_of(lc), e.sms, e.stream),
           "pf_ce_bwd");
        return 0;
      });
    } else {
      d = dispatched("pfeife::ce_bwd", {scale.expand({logits.size(0)}), logits, target, lse, ignore})[0]
              .toTensor();
    }
    return {d, Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ preference and policy losses
// Logits [N, T, V] and a label for each row.
bool tokens_fit(const Tensor& z, const Tensor& labels) {
  return z.dim() == 3 && number(z) && z.numel() > 0 && z.stride(2) == 1 && z.size(2) < (1ll << 31) &&
         z.size(1) < (1ll << 31) && labels.scalar_type() == at::kLong && labels.dim() == 2 && labels.is_contiguous() &&
         labels.size(0) == z.size(0) && labels.size(1) == z.size(1);
}
Tensor loss_scratch(const Env& e, const Tensor& like, int64_t N, int64_t T) {
  const int n = pf_token_loss_scratch(N, (int)T, (int)like.size(2), code_of(like), e.sms);
  if (n < 0) throw Failed{n, "pf_token_loss_scratch"};
  return empty({n}, at::kDouble, like);
}
float* float_at(const Tensor& t, int64_t i) { return static_cast<float*>(t.data_ptr()) + i; }

// What the backward of both needs lies in one buffer: two statistics a row, then `n` factors (one for each sequence or
// each row) and, for a policy, one over the number of tokens that count.
struct Kept {
  Tensor all;
  int64_t rows, n;
  bool inv;
  int64_t size() const { return 2 * rows + n + inv; }
  float* stats() const { return float_at(all, 0); }
  float* coef() const { return float_at(all, 2 * rows); }
  float* one_over() const { return inv ? float_at(all, 2 * rows + n) : nullptr; }
};
// An empty [N, T, V] whose rows lie to 16 bytes as those of the logits do, so that the backward goes through both by
// vectors: packed, or (some words of a padded vocabulary) with as much space between rows.
Tensor rows_like(const Tensor& z) {
  const int64_t N = z.size(0), T = z.size(1), V = z.size(2), size = z.element_size(), per = 16 / size;
  const int64_t row = T > 1 ? z.stride(1) : V;
  const int64_t off = (int64_t)(reinterpret_cast<uintptr_t>(z.data_ptr()) % 16) / size;
  if ((off == 0 && row % per == V % per) || row < V || row > V + 1024 ||
      (N > 1 && (z.stride(0) - T * row) % per))
    return empty(z.sizes(), z);
  return empty({off + N * T * row}, z).as_strided({N, T, V}, {T * row, row, 1}, off);
}
variable_list token_loss_backward(AutogradContext* ctx, const Tensor& g, int inputs) {
  variable_list out(inputs);
  if (!g.defined()) return out;
  const auto s = ctx->get_saved_variables();
  const Tensor &z = s[0], &labels = s[1];
  const int64_t ignore = ctx->saved_data["ignore"].toInt();
  const double temperature = ctx->saved_data["temperature"].toDouble();
  const bool inv = ctx->saved_data["inv"].toBool();
  const int64_t N = z.size(0), T = z.dim() > 1 ? z.size(1) : 0;
  const Kept kept{s[2], N * T, inv ? N * T : N, inv};
  if (direct(g, z, labels, kept.all) && tokens_fit(z, labels) && packed_floats(kept.all, kept.size()) &&
      aligned(kept.all) && packed_floats(g, 1)) {
    below([&] {
      const Env e(z);
      out[0] = rows_like(z);
      ok(pf_token_loss_bwd(z.data_ptr(), labels.data_ptr(), kept.stats(), kept.coef(), g.data_ptr(), kept.one_over(),
                           out[0].data_ptr(), T > 1 ? out[0].stride(1) : z.size(2), N, (int)T, (int)z.size(2),
                           z.stride(0), z.stride(1), ignore, inv ? 1 : (int)T, 1.0 / temperature, code_of(z),
                           e.sms, e.stream),
         "pf_token_loss_bwd");
      return 0;
    });
    return out;
  }
  const Tensor a = kept.all;
  Tensor coef = a.narrow(0, 2 * kept.rows, kept.n), one;
  if (inv) {
    coef = coef.view({N, T});
    one = a.select(0, 2 * kept.rows + kept.n);
  }
  out[0] = dispatched("pfeife::token_loss_bwd", {g, z, labels, a.narrow(0, 0, 2 * kept.rows).view({N, T, 2}), coef,
                                                 opt(one), ignore, temperature})[0].toTensor();
  return out;
}

variable_list preference_forward(const Tensor& z, const Tensor& labels, const Tensor& ref, double beta, double smoothing,
                                 int64_t ignore, Tensor& all) {
  const Env e(z);
  const int64_t N = z.size(0), T = z.size(1);
  const Kept kept{floats(2 * N * T + N, z), N * T, N, false};
  all = kept.all;
  const Tensor loss = empty({}, at::kFloat, z), rewards = floats(N, z), scratch = loss_scratch(e, z, N, T);
  ok(pf_preference_fwd(z.data_ptr(), labels.data_ptr(), ref.data_ptr(), loss.data_ptr(), rewards.data_ptr(),
                       kept.stats(), kept.coef(), scratch.data_ptr(), N, (int)T, (int)z.size(2), z.stride(0),
                       z.stride(1), ignore, beta, smoothing, code_of(z), e.sms, e.stream),
     "pf_preference_fwd");
  return {loss, rewards};
}
struct DirectPreference : torch::autograd::Function<DirectPreference> {
  static variable_list forward(AutogradContext* ctx, Tensor z, Tensor labels, Tensor ref, double beta, double smoothing,
                               int64_t ignore) {
    at::AutoDispatchBelowADInplaceOrView guard;
    Tensor all;
    const variable_list out = preference_forward(z, labels, ref, beta, smoothing, ignore, all);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({out[1]});
    ctx->save_for_backward({z, labels, all});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["temperature"] = 1.0;
    ctx->saved_data["inv"] = false;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return token_loss_backward(ctx, grads[0], 6);
  }
};

// the advantages' strides for [N, T]; one of a single place is expanded
bool advantages_fit(const Tensor& a, int64_t N, int64_t T) {
  return a.scalar_type() == at::kFloat && a.dim() == 2 && (a.size(0) == N || a.size(0) == 1) &&
         (a.size(1) == T || a.size(1) == 1);
}
struct Clipping { double low, high, kl, temperature; };
variable_list policy_forward(const Tensor& z, const Tensor& actions, const Tensor& old, const Tensor& adv,
                             const Tensor& ref, const Clipping& c, int64_t ignore, Tensor& all) {
  const Env e(z);
  const int64_t N = z.size(0), T = z.size(1), rows = N * T;
  const Kept kept{floats(3 * rows + 1, z), rows, rows, true};
  all = kept.all;
  const Tensor loss = empty({}, at::kFloat, z), logps = empty({N, T}, at::kFloat, z), kl = empty({}, at::kFloat, z),
               clipped = empty({}, at::kFloat, z), scratch = loss_scratch(e, z, N, T);
  ok(pf_policy_fwd(z.data_ptr(), actions.data_ptr(), old.data_ptr(), at_or_null(ref), adv.data_ptr(), loss.data_ptr(),
                   kl.data_ptr(), clipped.data_ptr(), kept.one_over(), logps.data_ptr(), kept.coef(), kept.stats(),
                   scratch.data_ptr(), N, (int)T, (int)z.size(2), z.stride(0), z.stride(1),
                   adv.size(0) > 1 ? adv.stride(0) : 0, adv.size(1) > 1 ? adv.stride(1) : 0, ignore, c.low, c.high,
                   c.kl, 1.0 / c.temperature, code_of(z), e.sms, e.stream),
     "pf_policy_fwd");
  return {loss, logps, kl, clipped};
}
struct DirectPolicy : torch::autograd::Function<DirectPolicy> {
  static variable_list forward(AutogradContext* ctx, Tensor z, Tensor actions, Tensor old, Tensor adv, Maybe ref,
                               double low, double high, double kl, double temperature, int64_t ignore) {
    at::AutoDispatchBelowADInplaceOrView guard;
    Tensor all;
    const variable_list out = policy_forward(z, actions, old, adv, value(ref), {low, high, kl, temperature}, ignore, all);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({out[1], out[2], out[3]});
    ctx->save_for_backward({z, actions, all});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["inv"] = true;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return token_loss_backward(ctx, grads[0], 10);
  }
};

// ------------------------------------------------------------------------------ GroupNorm
Tensor group_scratch(const Env& e, const Tensor& x, int64_t width) {
  const int64_t B = x.size(0), C = x.size(3), HW = x.size(1) * x.size(2);
  return floats(B * pf_groupnorm_slabs((int)B, (int)HW, (int)C, e.sms) * 2 * width, x);
}
NormOut group_norm_forward(const Tensor& x, const Tensor& gamma, const Tensor& beta, int64_t groups, double eps,
                           bool silu) {
  const Env e(x);
  const Tensor xc = x.contiguous();
  const int64_t B = x.size(0), C = x.size(3), HW = x.size(1) * x.size(2);
  NormOut o{empty(x.sizes(), x), {}, floats(B * groups, x), floats(B * groups, x)};
  const Tensor scratch = group_scratch(e, x, groups);
  ok(pf_groupnorm_fwd(xc.data_ptr(), gamma.data_ptr(), beta.data_ptr(), o.y.data_ptr(), o.mean.data_ptr(),
                      o.rstd.data_ptr(), scratch.data_ptr(), (int)B, (int)HW, (int)C, (int)groups, (float)eps,
                      silu, code_of(x), e.sms, e.stream),
     "pf_groupnorm_fwd");
  return o;
}
struct DirectGroupNorm : torch::autograd::Function<DirectGroupNorm> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor gamma, Tensor beta, int64_t groups, double eps,
                        bool silu) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const NormOut o = group_norm_forward(x, gamma, beta, groups, eps, silu);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, o.mean, o.rstd, gamma, beta});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["silu"] = silu;
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &mean = s[1], &rstd = s[2], &gamma = s[3], &beta = s[4];
    if (!grads[0].defined()) return variable_list(6);
    const Tensor dy = grads[0].contiguous();
    const int64_t groups = ctx->saved_data["groups"].toInt();
    const bool silu = ctx->saved_data["silu"].toBool();
    const int64_t stats = dy.size(0) * groups, C = dy.size(3);
    Tensor dx, dg, db;
    if (direct(dy, x, mean, rstd, gamma, beta) && half(x) && matches(x, dy) && packed_floats(mean, stats) &&
        packed_floats(rstd, stats) && packed_floats(gamma, C) && packed_floats(beta, C) && on_vectors(dy, x)) {
      below([&] {
        const Env e(dy);
        const Tensor xc = x.contiguous();
        const int64_t B = x.size(0), HW = x.size(1) * x.size(2);
        dx = empty(x.sizes(), x);
        dg = floats(C, x);
        db = floats(C, x);
        const Tensor sums = floats(2 * B * groups, x), scratch = group_scratch(e, x, C + groups);
        ok(pf_groupnorm_bwd(dy.data_ptr(), xc.data_ptr(), mean.data_ptr(), rstd.data_ptr(), gamma.data_ptr(),
                            beta.data_ptr(), dx.data_ptr(), dg.data_ptr(), db.data_ptr(), sums.data_ptr(),
                            scratch.data_ptr(), (int)B, (int)HW, (int)C, (int)groups, silu, code_of(x), e.sms,
                            e.stream),
           "pf_groupnorm_bwd");
        return 0;
      });
    } else {
      auto out = dispatched("pfeife::group_norm_bwd", {dy, x, mean, rstd, gamma, beta, groups, silu});
      dx = out[0].toTensor(); dg = out[1].toTensor(); db = out[2].toTensor();
    }
    return {dx, dg, db, Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ convolution
// The implicit-GEMM route (kernels.conv_gemm_supported, kernels.conv_wgrad_supported).
struct ConvShape {
  int64_t B, H, W, C, N, KH, KW, stride, pad, Ho, Wo;
  ConvShape(const Tensor& x, const Tensor& w, int64_t s, int64_t p)
      : B(x.size(0)), H(x.size(1)), W(x.size(2)), C(x.size(3)), N(w.size(0)), KH(w.size(2)), KW(w.size(3)),
        stride(s), pad(p), Ho((H + 2 * p - KH) / s + 1), Wo((W + 2 * p - KW) / s + 1) {}
  bool output_fits(const Tensor& y) const {
    return y.dim() == 4 && y.size(0) == B && y.size(1) == Ho && y.size(2) == Wo && y.size(3) == N;
  }
  bool one() const { return KH == 1 && KW == 1 && stride == 1 && pad == 0; }
  bool forward_fits() const {
    return !one() && C % 64 == 0 && N % 8 == 0 && KH * KW <= 64 && Wo > 0 && Ho > 0 && Wo <= 128 &&
           128 % Wo == 0 && Ho * Wo % 128 == 0 && (stride == 1 || stride == 2);
  }
  // Tiles of the input gradient are whole rows of the input.  Python keeps the gradients that take several
  // routes: strides, kernels that are not square, and up to 64 filters, which it pads.
  bool backward_fits() const {
    return stride == 1 && KH == KW && pad < KH && N % 64 == 0 && N > 64 && (64 % Wo == 0 || Wo % 64 == 0) && W <= 128 &&
           128 % W == 0 && H * W % 128 == 0;
  }
};
Tensor conv_pack(const Env& e, const Tensor& w, const ConvShape& s, bool flip) {
  const int64_t taps = s.KH * s.KW;
  const Tensor wc = w.contiguous();
  const Tensor out = flip ? empty({s.C, taps * s.N}, w) : empty({s.N, taps * s.C}, w);
  ok(pf_conv_pack(wc.data_ptr(), out.data_ptr(), (int)s.N, (int)s.C, (int)taps, (int)s.N, (int)s.C, flip,
                  e.stream),
     "pf_conv_pack");
  return out;
}
// images that the implicit GEMM reads in place
bool operands_fit(const Tensor& x, const Tensor& w) {
  return x.dim() == 4 && w.dim() == 4 && half(x) && w.scalar_type() == x.scalar_type() &&
         w.size(1) == x.size(3) && x.is_contiguous() && aligned(x);
}
Tensor conv_forward(const Tensor& x, const Tensor& w, const Tensor& b, int64_t stride, int64_t pad) {
  const Env e(x);
  const ConvShape s(x, w, stride, pad);
  const Tensor w2 = conv_pack(e, w, s, false), y = empty({s.B, s.Ho, s.Wo, s.N}, x);
  ok(pf_conv_gemm(x.data_ptr(), w2.data_ptr(), y.data_ptr(), (int)s.B, (int)s.H, (int)s.W, (int)s.C, (int)s.N,
                  (int)s.KH, (int)s.KW, (int)stride, (int)pad, w2.size(1), s.N, code_of(x), code_of(x),
                  at_or_null(b), 0, nullptr, 0, NONE, e.status, e.sms, e.stream),
     "pf_conv_gemm");
  return y;
}
struct DirectConv2d : torch::autograd::Function<DirectConv2d> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w, Maybe bias, int64_t stride, int64_t pad) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor b = value(bias);
    ctx->save_for_backward({x, w});
    ctx->saved_data["pad"] = pad;
    ctx->saved_data["bias"] = b.defined();
    return conv_forward(x, w, b, stride, pad);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    const Tensor &x = v[0], &w = v[1];
    const Tensor dy = grads[0].contiguous();
    const int64_t pad = ctx->saved_data["pad"].toInt();
    const bool bias = ctx->saved_data["bias"].toBool();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    Tensor dx, dw, db;
    if (direct(dy, x, w) && operands_fit(x, w) && x.scalar_type() == dy.scalar_type() &&
        ConvShape(x, w, 1, pad).output_fits(dy)) {
      below([&] {
        const Env e(dy);
        const ConvShape s(x, w, 1, pad);
        const Tensor dyc = aligned(dy) ? dy : dy.clone();
        const int64_t K = s.KH * s.KW * s.C, pixels = s.B * s.Ho * s.Wo;
        const Tensor dw2 = empty({s.N, K}, at::kFloat, x);
        const int kib = pf_gemm_workspace((int)s.N, (int)K, (int)pixels, 0, 2, e.sms, 0);
        const Tensor ws = kib ? floats(kib * 256ll, x) : Tensor();
        ok(pf_conv_wgrad(dyc.data_ptr(), x.data_ptr(), dw2.data_ptr(), (int)s.B, (int)s.H, (int)s.W, (int)s.C,
                         (int)s.N, (int)s.KH, (int)s.KW, 1, (int)pad, code_of(x), 0, e.status, e.sms,
                         const_cast<void*>(at_or_null(ws)), kib, e.stream),
           "pf_conv_wgrad");
        dw = empty(w.sizes(), w);
        ok(pf_conv_unpack(dw2.data_ptr(), dw.data_ptr(), (int)s.N, (int)s.C, (int)(s.KH * s.KW), (int)s.C,
                          code_of(w), e.stream),
           "pf_conv_unpack");
        if (nx) {
          const Tensor wt = conv_pack(e, w, s, true);
          dx = empty(x.sizes(), x);
          ok(pf_conv_gemm(dyc.data_ptr(), wt.data_ptr(), dx.data_ptr(), (int)s.B, (int)s.Ho, (int)s.Wo,
                          (int)s.N, (int)s.C, (int)s.KH, (int)s.KW, 1, (int)(s.KH - 1 - pad), wt.size(1), s.C,
                          code_of(x), code_of(x), nullptr, 0, nullptr, 0, NONE, e.status, e.sms, e.stream),
             "pf_conv_gemm");
        }
        if (bias) db = colsum(e, dyc.view({pixels, s.N}));
        return 0;
      });
    } else {
      auto out = dispatched("pfeife::conv2d_bwd", {dy, x, w, (int64_t)1, pad, nx, bias});
      dx = given(out[0]); dw = out[1].toTensor(); db = given(out[2]);
    }
    return {nx ? dx : Tensor(), nw ? dw : Tensor(), bias ? db : Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ gated feed-forward block
// rows that TMA reads and that are apart: tensor maps are not made for a row that stands for several
bool whole(const Tensor& m) { return readable(m) && m.stride(0) >= m.size(1); }
// 3 activations of gated_mlp.cu; weights [2H, D] and [N, H] of whole vectors
bool gated_fits(const Tensor& x, const Tensor& w1, const Tensor& w2) {
  return layer_fits(x, w1, {}) && w2.scalar_type() == x.scalar_type() && whole(w1) && whole(w2) && w1.size(0) == 2 * w2.size(1) &&
         w2.size(1) > 0 && w2.size(1) % 8 == 0 && w2.size(0) > 0 && w2.size(0) % 8 == 0 && w2.size(0) < (1ll << 31);
}
struct GatedSizes {
  int M, D, H, N;
  GatedSizes(const Tensor& x2, const Tensor& w2)
      : M((int)x2.size(0)), D((int)x2.size(1)), H((int)w2.size(1)), N((int)w2.size(0)) {}
};
Tensor gated_workspace(const GatedSizes& g, const Env& e, const Tensor& like, int& kib) {
  kib = pf_gated_mlp_scratch(g.M, g.D, g.H, g.N, e.sms);
  return kib ? floats(kib * 256ll, like) : Tensor();
}
// contiguous() leaves one row of a wider matrix and values that start anywhere as they are
Tensor whole_rows(const Tensor& x) {
  const Tensor r = rows(x);
  return whole(r) ? r : r.clone(at::MemoryFormat::Contiguous);
}
std::pair<Tensor, Tensor> gated_forward(const Tensor& x, const Tensor& w1, const Tensor& b1, const Tensor& w2,
                                        const Tensor& b2, const Tensor& res, int act, bool keep) {
  const Env e(x);
  const Tensor x2 = whole_rows(x), r2 = res.defined() ? whole_rows(res) : Tensor();
  const GatedSizes g(x2, w2);
  const Tensor h = empty({g.M, g.H}, x), gu = keep ? empty({g.M, 2 * g.H}, x) : Tensor(), y = empty({g.M, g.N}, x);
  int kib;
  const Tensor ws = gated_workspace(g, e, x, kib);
  ok(pf_gated_mlp_fwd(x2.data_ptr(), w1.data_ptr(), at_or_null(b1), b1.defined() ? code_of(b1) : 0, w2.data_ptr(),
                      at_or_null(b2), b2.defined() ? code_of(b2) : 0, at_or_null(r2), h.data_ptr(),
                      const_cast<void*>(at_or_null(gu)), y.data_ptr(), const_cast<void*>(at_or_null(ws)), kib, g.M, g.D,
                      g.H, g.N, x2.stride(0), w1.stride(0), w2.stride(0), r2.defined() ? r2.stride(0) : 0, act,
                      code_of(x), e.status, e.sms, e.stream),
     "pf_gated_mlp_fwd");
  return {y.view(with_last(x, g.N)), keep ? gu.view(with_last(x, 2 * g.H)) : gu};
}

struct DirectGatedMlp : torch::autograd::Function<DirectGatedMlp> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w1, Maybe bias1, Tensor w2, Maybe bias2,
                        Maybe residual, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor b1 = value(bias1), b2 = value(bias2), res = value(residual);
    // gate and up are for any gradient but the residual's
    bool keep = x.requires_grad() || w1.requires_grad() || w2.requires_grad();
    for (const Tensor* t : {&b1, &b2}) keep = keep || (t->defined() && t->requires_grad());
    auto [y, gu] = gated_forward(x, w1, b1, w2, b2, res, (int)act, keep);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w1, w2, gu, b1, b2});
    ctx->saved_data["act"] = act;
    if (bias1) ctx->saved_data["type1"] = (int64_t)b1.scalar_type();
    if (bias2) ctx->saved_data["type2"] = (int64_t)b2.scalar_type();
    ctx->saved_data["res"] = res.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w1 = s[1], &w2 = s[2], &gu = s[3], &b1 = s[4], &b2 = s[5];
    if (!grads[0].defined()) return variable_list(7);
    const Tensor dy = grads[0].contiguous();
    const int act = (int)ctx->saved_data["act"].toInt();
    const int i1 = 2, i2 = i1 + b1.defined(), i3 = i2 + 1, ir = i3 + b2.defined();     // inputs that were given
    const bool nx = ctx->needs_input_grad(0), nw1 = ctx->needs_input_grad(1),
               nb1 = b1.defined() && ctx->needs_input_grad(i1), nw2 = ctx->needs_input_grad(i2),
               nb2 = b2.defined() && ctx->needs_input_grad(i3),
               nr = ctx->saved_data["res"].toBool() && ctx->needs_input_grad(ir);
    Tensor dx, dw1, db1, dw2, db2;
    if (!(nx || nw1 || nb1 || nw2 || nb2)) {
      // the residual's alone
    } else if (gu.defined() && direct(dy, x, w1, w2, gu, b1, b2) && gated_fits(x, w1, w2) &&
               dy.scalar_type() == x.scalar_type() && dy.size(-1) == w2.size(0) &&
               dy.numel() / dy.size(-1) == x.numel() / x.size(-1) && gu.scalar_type() == x.scalar_type() &&
               gu.size(-1) == w1.size(0) && gu.numel() / gu.size(-1) == x.numel() / x.size(-1) &&
               (!b1.defined() || number(b1)) && (!b2.defined() || number(b2))) {
      below([&] {
        const Env e(dy);
        const Tensor x2 = whole_rows(x), dy2 = whole_rows(dy);
        Tensor kept = gu.contiguous();
        if (!aligned(kept)) kept = kept.clone();
        const GatedSizes g(x2, w2);
        const Tensor dgu = empty({g.M, 2 * g.H}, dy), h = empty({g.M, g.H}, dy);
        int kib;
        const Tensor ws = gated_workspace(g, e, dy, kib);
        if (nx) dx = empty(x.sizes(), dy);
        if (nw1) dw1 = empty(w1.sizes(), dy);
        if (nw2) dw2 = empty(w2.sizes(), dy);
        if (nb1) db1 = empty({2 * g.H}, b1);
        if (nb2) db2 = empty({g.N}, b2);
        auto out = [](const Tensor& t) { return const_cast<void*>(at_or_null(t)); };
        ok(pf_gated_mlp_bwd(dy2.data_ptr(), x2.data_ptr(), w1.data_ptr(), w2.data_ptr(), kept.data_ptr(),
                            dgu.data_ptr(), h.data_ptr(), out(dx), out(dw1), out(dw2), out(db1), out(db2), out(ws), kib,
                            g.M, g.D, g.H, g.N, dy2.stride(0), x2.stride(0), w1.stride(0), w2.stride(0), act,
                            code_of(dy), code_of(dy), code_of(dy), nb1 ? code_of(b1) : 0, nb2 ? code_of(b2) : 0, 0,
                            e.status, e.sms, e.stream),
           "pf_gated_mlp_bwd");
        return 0;
      });
    } else {
      auto out = dispatched("pfeife::gated_mlp_bwd", {dy, x, w1, w2, gu, (int64_t)act, nx, nw1, nb1, nw2, nb2, opt(b1),
                                                      opt(b2)});
      dx = given(out[0]); dw1 = given(out[1]); db1 = given(out[2]); dw2 = given(out[3]); db2 = given(out[4]);
    }
    return {dx, dw1, nb1 ? as(db1, ctx->saved_data["type1"]) : Tensor(), dw2,
            nb2 ? as(db2, ctx->saved_data["type2"]) : Tensor(), nr ? dy : Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ output head with its cross entropy
bool head_fits(const Tensor& x, const Tensor& w, const Tensor& target) {
  return x.dim() >= 2 && half(x) && x.numel() > 0 && w.scalar_type() == x.scalar_type() && whole(w) &&
         w.size(1) == x.size(-1) && w.size(1) % 8 == 0 && w.size(0) > 0 && w.size(0) <= (1ll << 28) &&
         target.scalar_type() == at::kLong && target.sizes() == x.sizes().slice(0, x.dim() - 1) &&
         target.numel() <= (1ll << 28) && w.size(1) <= (1ll << 20);
}
int64_t padded_rows(int64_t n) { return (n + 255) / 256 * 256; }
Tensor counted(int n, const char* what, at::ScalarType type, const Tensor& like) {
  if (n < 0) throw Failed{n, what};
  return empty({n}, type, like);
}
// loss, and for the backward: rows that count, index, statistics, what a sum is multiplied by
struct HeadOut { Tensor loss, xc, index, stats, inv; };
HeadOut head_forward(const Tensor& x, const Tensor& w, const Tensor& target, int64_t ignore, int reduction) {
  const Env e(x);
  Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if (x2.stride(1) != 1 || x2.stride(0) % 8) x2 = x2.contiguous();
  const Tensor t = target.contiguous();
  const int64_t N = x2.size(0), V = w.size(0), D = x2.size(1), Mp = padded_rows(N);
  HeadOut o;
  o.loss = reduction ? empty({}, at::kFloat, x) : empty(target.sizes(), at::kFloat, x);
  o.xc = empty({Mp, D}, x);
  o.index = counted(pf_head_index(N), "pf_head_index", at::kInt, x);
  o.stats = empty({Mp, 2}, at::kFloat, x);
  o.inv = empty({}, at::kFloat, x);
  const int kib = pf_head_scratch(N, V);
  if (kib < 0) throw Failed{kib, "pf_head_scratch"};
  const Tensor scratch = floats(kib * 256ll, x);
  ok(pf_head_fwd(x2.data_ptr(), w.data_ptr(), t.data_ptr(), o.xc.data_ptr(), o.index.data_ptr(), o.stats.data_ptr(),
                 o.loss.data_ptr(), o.inv.data_ptr(), scratch.data_ptr(), N, V, (int)D, (int)D,
                 N > 1 ? x2.stride(0) : D, w.stride(0), ignore, reduction, code_of(x), e.status, e.sms, e.stream),
     "pf_head_fwd");
  return o;
}

struct DirectHeadLoss : torch::autograd::Function<DirectHeadLoss> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w, Tensor target, int64_t ignore, int64_t reduction) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const HeadOut o = head_forward(x, w, target, ignore, (int)reduction);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({w, o.xc, o.index, o.stats, o.inv});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["by_row"] = reduction == 0;
    return o.loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &w = s[0], &xc = s[1], &index = s[2], &stats = s[3], &inv = s[4];
    if (!grads[0].defined()) return variable_list(5);
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const bool by_row = ctx->saved_data["by_row"].toBool();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    int64_t N = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) N *= shape[i];
    const Tensor g = by_row ? grads[0].reshape({-1}) : grads[0];
    const int64_t D = shape.back(), Mp = padded_rows(N);
    Tensor dx, dw;
    if (direct(g, w, xc, index, stats, inv) && half(xc) && w.scalar_type() == xc.scalar_type() && whole(w) &&
        w.size(1) == D && xc.dim() == 2 && xc.size(0) == Mp && xc.size(1) == D && xc.is_contiguous() && aligned(xc) &&
        packed_floats(stats, 2 * Mp) && packed_floats(inv, 1) && index.scalar_type() == at::kInt &&
        index.is_contiguous() && index.numel() == pf_head_index(N) && g.scalar_type() == at::kFloat &&
        g.numel() == (by_row ? N : 1)) {
      below([&] {
        const Env e(g);
        const int64_t V = w.size(0);
        if (nx) dx = empty(shape, xc);
        if (nw) dw = empty(w.sizes(), xc);
        const int words = pf_head_words(N, V), parts = pf_head_parts(N, V, (int)D, e.sms);
        if (words < 0 || parts < 0) throw Failed{words < 0 ? words : parts, "pf_head_words"};
        const Tensor dz = empty({Mp, words}, xc), acc = nx ? floats(parts * Mp * D + 1, xc) : Tensor();
        const Tensor factor = by_row ? floats(Mp + 1, xc) : Tensor();
        auto out = [](const Tensor& t) { return const_cast<void*>(at_or_null(t)); };
        ok(pf_head_bwd(g.data_ptr(), inv.data_ptr(), xc.data_ptr(), w.data_ptr(), index.data_ptr(), stats.data_ptr(),
                       out(dx), out(dw), dz.data_ptr(), out(acc), out(factor), N, V, (int)D, (int)D,
                       by_row ? g.stride(0) : 0, w.stride(0), D, by_row, 0, code_of(xc), code_of(xc), e.status, e.sms,
                       e.stream),
           "pf_head_bwd");
        return 0;
      });
    } else {
      auto out = dispatched("pfeife::head_loss_bwd", {g, xc, index, stats, inv, w, N, by_row, nx, nw});
      if (nx) dx = out[0].toTensor().view(shape);
      dw = given(out[1]);
    }
    return {dx, nw ? dw : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ scaled embedding
bool table_type_fits(const Tensor& table, at::ScalarType out) {
  return table.scalar_type() == at::kFloat || (half(table) && table.scalar_type() == out);
}
Tensor embed_forward(const Tensor& ids, const Tensor& table, double scale, at::ScalarType type) {
  const Env e(table);
  const Tensor ic = ids.contiguous();
  auto shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  const Tensor out = empty(shape, type, table);
  ok(pf_scaled_embed_fwd(table.data_ptr(), ic.data_ptr(), out.data_ptr(), ids.numel(), (int)table.size(1),
                         table.size(0), (float)scale, code_of(table), code_of(type), e.stream),
     "pf_scaled_embed_fwd");
  return out;
}
struct DirectScaledEmbed : torch::autograd::Function<DirectScaledEmbed> {
  static Tensor forward(AutogradContext* ctx, Tensor ids, Tensor table, double scale, int64_t type) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor y = embed_forward(ids, table, scale, static_cast<at::ScalarType>(type));
    ctx->save_for_backward({ids, table});
    ctx->saved_data["scale"] = scale;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &ids = s[0], &table = s[1];
    const double scale = ctx->saved_data["scale"].toDouble();
    const Tensor dout = grads[0].contiguous();
    Tensor d;
    if (direct(dout, ids, table) && ids.scalar_type() == at::kLong && table.dim() == 2 &&
        (half(dout) || dout.scalar_type() == at::kFloat) && table_type_fits(table, dout.scalar_type()) &&
        dout.numel() == ids.numel() * table.size(1)) {
      below([&] {
        const Env e(dout);
        const Tensor ic = ids.contiguous();
        const int64_t V = table.size(0), D = table.size(1);
        d = empty(table.sizes(), table);
        const int kib = pf_scaled_embed_scratch(ids.numel(), (int)D, V);
        if (kib < 0) throw Failed{kib, "pf_scaled_embed_scratch"};
        const Tensor scratch = floats(kib * 256ll, table);
        ok(pf_scaled_embed_bwd(dout.data_ptr(), ic.data_ptr(), d.data_ptr(), scratch.data_ptr(), ids.numel(), (int)D, V,
                               (float)scale, 0, code_of(dout), code_of(table), e.stream),
           "pf_scaled_embed_bwd");
        return 0;
      });
    } else {
      d = dispatched("pfeife::scaled_embed_bwd", {dout, ids, table, scale})[0].toTensor();
    }
    return {Tensor(), d, Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------ Python
// Arguments of one call.  `fits` turns false at the first that is not what the usual call has.
struct Args {
  PyObject* const* a;
  bool fits;
  Args(PyObject* const* args, Py_ssize_t n, Py_ssize_t expected) : a(args), fits(n == expected) {
    if (!fits) PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", expected, n);
    else fits = unobserved() && !at::autocast::is_autocast_enabled(at::kCUDA);
  }
  Tensor tensor(int i, bool optional = false) {
    if (!fits) return {};
    if (optional && a[i] == Py_None) return {};
    if (!THPVariable_CheckTypeExact(Py_TYPE(a[i]))) { fits = false; return {}; }
    const Tensor& t = THPVariable_Unpack(a[i]);
    if (!t.is_cuda()) fits = false;
    return t;
  }
  int64_t integer(int i) {
    if (!fits) return 0;
    if (!PyLong_CheckExact(a[i])) { fits = false; return 0; }
    const long long v = PyLong_AsLongLong(a[i]);
    if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); fits = false; }
    return v;
  }
  bool boolean(int i) {
    if (a[i] != Py_True && a[i] != Py_False) fits = false;
    return a[i] == Py_True;
  }
  double real(int i) {
    if (!fits) return 0;
    if (!PyFloat_CheckExact(a[i])) { fits = false; return 0; }
    return PyFloat_AS_DOUBLE(a[i]);
  }
};

// Runs `f`, which returns the outputs, without the interpreter lock; None where the kernels refuse the
// call (Python repeats it and reports why).
template <typename F>
PyObject* run(const Tensor& first, F&& f) {
  if (first.get_device() >= MAX_DEVICES) Py_RETURN_NONE;
  if (!learn_status(first.get_device())) return nullptr;
  try {
    decltype(f()) out;
    {
      pybind11::gil_scoped_release free;
      out = f();
    }
    if constexpr (std::is_same_v<decltype(out), Tensor>) {
      return THPVariable_Wrap(std::move(out));
    } else {
      if (out.size() == 1) return THPVariable_Wrap(std::move(out[0]));
      PyObject* t = PyTuple_New((Py_ssize_t)out.size());
      for (size_t i = 0; t && i < out.size(); ++i) PyTuple_SET_ITEM(t, (Py_ssize_t)i, THPVariable_Wrap(out[i]));
      return t;
    }
  } catch (const Failed&) {
    Py_RETURN_NONE;
  }
}
// HANDLE_TH_ERRORS turns C++ exceptions into Python's.
#define PF_OP(name) PyObject* name(PyObject*, PyObject* const* args, Py_ssize_t n)
template <typename F>
Tensor unrecorded(F&& f) {
  at::AutoDispatchBelowADInplaceOrView guard;
  return f();
}

PF_OP(linear) {
  HANDLE_TH_ERRORS
  Args a(args, n, 5);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), w = a.tensor(1), b = a.tensor(2, true), r = a.tensor(3, true);
  const int64_t act = a.integer(4);
  if (!a.fits || act < 0 || act > 3 || !all_plain(x, w, b, r) || !layer_fits(x, w, b) ||
      !residual_fits(r, x, w.size(0)))
    Py_RETURN_NONE;
  if (!recorded(x, w, b, r))
    return run(x, [&] { return unrecorded([&] { return linear_forward(x, w, b, r, (int)act).first; }); });
  if (w.size(0) % 8) Py_RETURN_NONE;                  // the backward's products need whole vectors
  return run(x, [&] { return DirectLinear::apply(x, w, maybe(b), maybe(r), act); });
  END_HANDLE_TH_ERRORS
}

PF_OP(mlp) {
  HANDLE_TH_ERRORS
  Args a(args, n, 7);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), w1 = a.tensor(1), b1 = a.tensor(2, true), w2 = a.tensor(3),
               b2 = a.tensor(4, true), r = a.tensor(5, true);
  const int64_t act = a.integer(6);
  if (!a.fits || act < 1 || act > 2 || !all_plain(x, w1, b1, w2, b2, r) || !layer_fits(x, w1, b1) ||
      w2.scalar_type() != x.scalar_type() || !readable(w2) || w2.size(1) != w1.size(0) || w2.size(1) % 8 ||
      !bias_fits(b2, w2.size(0)) || !residual_fits(r, x, w2.size(0)))
    Py_RETURN_NONE;
  if (!recorded(x, w1, b1, w2, b2, r))
    return run(x, [&] {
      return unrecorded([&] {
        const Tensor a1 = linear_forward(x, w1, b1, {}, (int)act).first;
        return linear_forward(a1, w2, b2, r, 0).first;
      });
    });
  if (w2.size(0) % 8) Py_RETURN_NONE;
  return run(x, [&] { return DirectMlp::apply(x, w1, maybe(b1), w2, maybe(b2), maybe(r), act); });
  END_HANDLE_TH_ERRORS
}

PF_OP(norm) {
  HANDLE_TH_ERRORS
  Args a(args, n, 6);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), g = a.tensor(1), b = a.tensor(2, true), r = a.tensor(3, true);
  const double eps = a.real(4);
  const bool rms = a.boolean(5);
  auto vector = [&](const Tensor& t) {
    return !t.defined() || (t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == x.size(-1) &&
                            t.is_contiguous());
  };
  if (!a.fits || !all_plain(x, g, b, r) || x.dim() < 1 || !half(x) || !vector(g) || !vector(b) ||
      !on_vectors(x, g, b, r) || (r.defined() && (r.scalar_type() != x.scalar_type() || r.sizes() != x.sizes())))
    Py_RETURN_NONE;
  if (!recorded(x, g, b, r))
    return run(x, [&]() -> variable_list {
      at::AutoDispatchBelowADInplaceOrView guard;
      const NormOut o = norm_forward(x, g, b, r, eps, rms);
      if (r.defined()) return {o.y, o.h};
      return {o.y};
    });
  return run(x, [&] { return DirectNorm::apply(x, g, maybe(b), maybe(r), eps, rms); });
  END_HANDLE_TH_ERRORS
}

PF_OP(attention) {
  HANDLE_TH_ERRORS
  Args a(args, n, 5);
  if (PyErr_Occurred()) return nullptr;
  const Tensor q = a.tensor(0), k = a.tensor(1), v = a.tensor(2);
  const bool causal = a.boolean(3);
  const double scale = a.real(4);
  if (!a.fits || !all_plain(q, k, v) || q.dim() != 4 || k.dim() != 4 || !half(q) ||
      k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || k.sizes() != v.sizes() ||
      k.size(0) != q.size(0) || k.size(2) != q.size(2) || k.size(3) != q.size(3) || q.size(3) % 8 ||
      q.size(3) > 128 || q.stride(3) != 1 || k.stride(3) != 1 || v.stride(3) != 1)
    Py_RETURN_NONE;
  if (!recorded(q, k, v))
    return run(q, [&] { return unrecorded([&] { return heads_forward(q, k, v, causal, scale).first; }); });
  return run(q, [&] { return DirectAttention::apply(q, k, v, causal, scale); });
  END_HANDLE_TH_ERRORS
}

PF_OP(attention_qkv) {
  HANDLE_TH_ERRORS
  Args a(args, n, 3);
  if (PyErr_Occurred()) return nullptr;
  const Tensor t = a.tensor(0);
  const bool causal = a.boolean(1);
  const double scale = a.real(2);
  if (!a.fits || !all_plain(t) || t.dim() != 5 || !half(t) || t.size(2) != 3 || t.size(4) % 8 ||
      t.size(4) > 128 || !packed_fits(t))
    Py_RETURN_NONE;
  if (!recorded(t))
    return run(t, [&] { return unrecorded([&] { return packed_forward(t, causal, scale).first; }); });
  return run(t, [&] { return DirectAttentionQkv::apply(t, causal, scale); });
  END_HANDLE_TH_ERRORS
}

PF_OP(rope_qkv) {
  HANDLE_TH_ERRORS
  Args a(args, n, 3);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), cos = a.tensor(1), sin = a.tensor(2);
  if (!a.fits || !all_plain(x, cos, sin) || x.dim() != 5 || !half(x) || x.size(2) != 3 || x.size(4) % 16 ||
      !x.is_contiguous() || !aligned(x) || !table_fits(cos, x) || !table_fits(sin, x))
    Py_RETURN_NONE;
  if (!recorded(x, cos, sin))
    return run(x, [&] { return unrecorded([&] { return rope_forward(x, cos, sin, false); }); });
  return run(x, [&] { return DirectRopeQkv::apply(x, cos, sin); });
  END_HANDLE_TH_ERRORS
}

PF_OP(glu) {
  HANDLE_TH_ERRORS
  Args a(args, n, 2);
  if (PyErr_Occurred()) return nullptr;
  const Tensor gu = a.tensor(0);
  const bool gelu = a.boolean(1);
  if (!a.fits || !all_plain(gu) || gu.dim() < 1 || !half(gu) || gu.size(-1) % 16 || !gu.is_contiguous() ||
      !on_vectors(gu))
    Py_RETURN_NONE;
  if (!recorded(gu)) return run(gu, [&] { return unrecorded([&] { return glu_forward(gu, gelu); }); });
  return run(gu, [&] { return DirectGlu::apply(gu, gelu); });
  END_HANDLE_TH_ERRORS
}

PF_OP(cross_entropy) {
  HANDLE_TH_ERRORS
  Args a(args, n, 3);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), t = a.tensor(1);
  const int64_t ignore = a.integer(2);
  if (!a.fits || !all_plain(x, t) || x.dim() != 2 || !(half(x) || x.scalar_type() == at::kFloat) ||
      t.scalar_type() != at::kLong || t.dim() != 1 || t.size(0) != x.size(0))
    Py_RETURN_NONE;
  if (!recorded(x))
    return run(x, [&] { return unrecorded([&] { return loss_forward(x, t, ignore).mean; }); });
  return run(x, [&] { return DirectCrossEntropy::apply(x, t, ignore); });
  END_HANDLE_TH_ERRORS
}

PF_OP(rotate_heads) {
  HANDLE_TH_ERRORS
  Args a(args, n, 5);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), cos = a.tensor(1), sin = a.tensor(2), pos = a.tensor(3, true);
  const bool interleaved = a.boolean(4);
  if (!a.fits || !all_plain(x, cos, sin, pos) || !head_view_fits(x, x.dim() == 5 ? 5 : 4) ||
      !angles_fit(x, cos, sin, pos) || recorded(cos, sin))            // tables get no gradient: refused in Python
    Py_RETURN_NONE;
  if (!recorded(x))
    return run(x, [&] { return unrecorded([&] { return rotate(x, cos, sin, pos, interleaved, false); }); });
  return run(x, [&] { return DirectRotate::apply(x, cos, sin, maybe(pos), interleaved); });
  END_HANDLE_TH_ERRORS
}

// queries and keys, or a projection and None
PF_OP(norm_rotate_heads) {
  HANDLE_TH_ERRORS
  Args a(args, n, 9);
  if (PyErr_Occurred()) return nullptr;
  const Tensor q = a.tensor(0), k = a.tensor(1, true), wq = a.tensor(2), wk = a.tensor(3), cos = a.tensor(4),
               sin = a.tensor(5), pos = a.tensor(6, true);
  const double eps = a.real(7);
  const bool interleaved = a.boolean(8);
  if (!a.fits || !all_plain(q, k, wq, wk, cos, sin, pos) || !(k.defined() ? same_heads(q, k) : head_view_fits(q, 5)) ||
      !gain_fits(wq, q) || !gain_fits(wk, q) || !angles_fit(q, cos, sin, pos) || recorded(cos, sin))
    Py_RETURN_NONE;
  if (!recorded(q, k, wq, wk))
    return run(q, [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      return norm_rotate(q, k, wq, wk, cos, sin, pos, eps, interleaved);
    });
  return run(q, [&] { return DirectNormRotate::apply(q, maybe(k), wq, wk, cos, sin, maybe(pos), eps, interleaved); });
  END_HANDLE_TH_ERRORS
}

PF_OP(preference_loss) {
  HANDLE_TH_ERRORS
  Args a(args, n, 6);
  if (PyErr_Occurred()) return nullptr;
  const Tensor z = a.tensor(0), labels = a.tensor(1), ref = a.tensor(2);
  const double beta = a.real(3), smoothing = a.real(4);
  const int64_t ignore = a.integer(5);
  if (!a.fits || !all_plain(z, labels, ref) || !tokens_fit(z, labels) || z.size(0) % 2 || ref.dim() != 1 ||
      !packed_floats(ref, z.size(0)) || ref.requires_grad() || !(smoothing >= 0.0 && smoothing <= 1.0))
    Py_RETURN_NONE;
  if (!recorded(z))
    return run(z, [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      Tensor all;
      return preference_forward(z, labels, ref, beta, smoothing, ignore, all);
    });
  return run(z, [&] { return DirectPreference::apply(z, labels, ref, beta, smoothing, ignore); });
  END_HANDLE_TH_ERRORS
}

PF_OP(policy_loss) {
  HANDLE_TH_ERRORS
  Args a(args, n, 10);
  if (PyErr_Occurred()) return nullptr;
  const Tensor z = a.tensor(0), actions = a.tensor(1), old = a.tensor(2), adv = a.tensor(3), ref = a.tensor(4, true);
  const Clipping c{a.real(5), a.real(6), a.real(7), a.real(8)};
  const int64_t ignore = a.integer(9);
  if (!a.fits || !all_plain(z, actions, old, adv, ref) || !tokens_fit(z, actions)) Py_RETURN_NONE;
  const int64_t N = z.size(0), T = z.size(1);
  for (const Tensor* t : {&old, &ref})
    if (t->defined() && (!packed_floats(*t, N * T) || t->dim() != 2 || t->size(0) != N || t->requires_grad()))
      Py_RETURN_NONE;
  if (!advantages_fit(adv, N, T) || adv.requires_grad() || !(c.temperature >= 1e-30 && c.temperature <= 1e30) ||
      !(c.low >= 0.0 && c.low <= 1.0) || !(c.high >= 0.0))
    Py_RETURN_NONE;
  if (!recorded(z))
    return run(z, [&] {
      at::AutoDispatchBelowADInplaceOrView guard;
      Tensor all;
      return policy_forward(z, actions, old, adv, ref, c, ignore, all);
    });
  return run(z, [&] {
    return DirectPolicy::apply(z, actions, old, adv, maybe(ref), c.low, c.high, c.kl, c.temperature, ignore);
  });
  END_HANDLE_TH_ERRORS
}

PF_OP(group_norm) {
  HANDLE_TH_ERRORS
  Args a(args, n, 6);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), g = a.tensor(1), b = a.tensor(2);
  const int64_t groups = a.integer(3);
  const double eps = a.real(4);
  const bool silu = a.boolean(5);
  auto vector = [&](const Tensor& t) {
    return t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == x.size(3) && t.is_contiguous();
  };
  if (!a.fits || !all_plain(x, g, b) || x.dim() != 4 || !half(x) || x.size(3) % 8 || x.size(3) > 8192 ||
      groups <= 0 || x.size(3) % groups || !vector(g) || !vector(b) || !on_vectors(x))
    Py_RETURN_NONE;
  if (!recorded(x, g, b))
    return run(x, [&] { return unrecorded([&] { return group_norm_forward(x, g, b, groups, eps, silu).y; }); });
  return run(x, [&] { return DirectGroupNorm::apply(x, g, b, groups, eps, silu); });
  END_HANDLE_TH_ERRORS
}

PF_OP(conv2d) {
  HANDLE_TH_ERRORS
  Args a(args, n, 5);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), w = a.tensor(1), b = a.tensor(2, true);
  const int64_t stride = a.integer(3), pad = a.integer(4);
  if (!a.fits || !all_plain(x, w, b) || !operands_fit(x, w) || stride < 1 || pad < 0 ||
      !ConvShape(x, w, stride, pad).forward_fits() ||
      (b.defined() && (b.scalar_type() != at::kFloat || !bias_fits(b, w.size(0)))))
    Py_RETURN_NONE;
  if (!recorded(x, w, b))
    return run(x, [&] { return unrecorded([&] { return conv_forward(x, w, b, stride, pad); }); });
  if (!ConvShape(x, w, stride, pad).backward_fits()) Py_RETURN_NONE;
  return run(x, [&] { return DirectConv2d::apply(x, w, maybe(b), stride, pad); });
  END_HANDLE_TH_ERRORS
}

PF_OP(gated_mlp) {
  HANDLE_TH_ERRORS
  Args a(args, n, 7);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), w1 = a.tensor(1), b1 = a.tensor(2, true), w2 = a.tensor(3), b2 = a.tensor(4, true),
               r = a.tensor(5, true);
  const int64_t act = a.integer(6);
  if (!a.fits || act < 1 || act > 3 || !all_plain(x, w1, b1, w2, b2, r) || !gated_fits(x, w1, w2) ||
      !bias_fits(b1, w1.size(0)) || !bias_fits(b2, w2.size(0)) ||
      (r.defined() && (r.scalar_type() != x.scalar_type() || r.sizes() != at::IntArrayRef(with_last(x, w2.size(0))))))
    Py_RETURN_NONE;
  if (!recorded(x, w1, b1, w2, b2, r))
    return run(x, [&] { return unrecorded([&] { return gated_forward(x, w1, b1, w2, b2, r, (int)act, false).first; }); });
  return run(x, [&] { return DirectGatedMlp::apply(x, w1, maybe(b1), w2, maybe(b2), maybe(r), act); });
  END_HANDLE_TH_ERRORS
}

PF_OP(linear_cross_entropy) {
  HANDLE_TH_ERRORS
  Args a(args, n, 5);
  if (PyErr_Occurred()) return nullptr;
  const Tensor x = a.tensor(0), w = a.tensor(1), t = a.tensor(2);
  const int64_t ignore = a.integer(3), reduction = a.integer(4);
  if (!a.fits || !all_plain(x, w, t) || !head_fits(x, w, t)) Py_RETURN_NONE;
  if (!recorded(x, w))
    return run(x, [&] { return unrecorded([&] { return head_forward(x, w, t, ignore, (int)reduction).loss; }); });
  return run(x, [&] { return DirectHeadLoss::apply(x, w, t, ignore, reduction); });
  END_HANDLE_TH_ERRORS
}

// the type of the result as the kernels' code for it
PF_OP(scaled_embedding) {
  HANDLE_TH_ERRORS
  Args a(args, n, 4);
  if (PyErr_Occurred()) return nullptr;
  const Tensor ids = a.tensor(0), table = a.tensor(1);
  const double scale = a.real(2);
  const int64_t code = a.integer(3);
  if (!a.fits || code < 0 || code > 2) Py_RETURN_NONE;
  const at::ScalarType type = code == 0 ? at::kFloat : code == 1 ? at::kHalf : at::kBFloat16;
  if (!all_plain(ids, table) || ids.scalar_type() != at::kLong || table.dim() != 2 || !table.is_contiguous() ||
      !table_type_fits(table, type) || table.size(0) >= (1ll << 30) || ids.numel() > (1ll << 30) || !std::isfinite(scale))
    Py_RETURN_NONE;
  if (!recorded(table))
    return run(table, [&] { return unrecorded([&] { return embed_forward(ids, table, scale, type); }); });
  return run(table, [&] { return DirectScaledEmbed::apply(ids, table, scale, (int64_t)type); });
  END_HANDLE_TH_ERRORS
}

PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) return PyErr_Format(PyExc_TypeError, "setup(status_word, check)");
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  g_status_word = args[0];
  g_check = args[1];
  Py_RETURN_NONE;
}
PyObject* launches(PyObject*, PyObject*) { return PyLong_FromLongLong(g_launches.load()); }

#define PF_ENTRY(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    PF_ENTRY(linear), PF_ENTRY(mlp), PF_ENTRY(norm), PF_ENTRY(attention), PF_ENTRY(attention_qkv),
    PF_ENTRY(rope_qkv), PF_ENTRY(glu), PF_ENTRY(cross_entropy), PF_ENTRY(group_norm), PF_ENTRY(conv2d),
    PF_ENTRY(rotate_heads), PF_ENTRY(norm_rotate_heads), PF_ENTRY(preference_loss), PF_ENTRY(policy_loss),
    PF_ENTRY(gated_mlp), PF_ENTRY(linear_cross_entropy), PF_ENTRY(scaled_embedding), PF_ENTRY(setup), {"launches", launches, METH_NOARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "pfeife_b200_eager", "eager calls of the ops", -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace pfeife

PyMODINIT_FUNC PyInit_pfeife_b200_eager() {
  PyObject* m = PyModule_Create(&pfeife::module_def);
  // the sources it was built from: the loader takes no module of others
  if (m && PyModule_AddStringConstant(m, "SOURCES", PF_SOURCES) < 0) Py_CLEAR(m);
  return m;
}
