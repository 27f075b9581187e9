// Torch form of the decoder's operators: argument checks, outputs and autograd nodes around the C entry points of
// include/sparsesam.h, as a Python extension module (_torch_ops, imported by ops.py).
//
// Why not ctypes and torch.autograd.Function, as the encoder's calls: these are training operators of microseconds,
// and a node in Python costs the host more than the kernels (a pass with gradients of a 4096 x 256 LayerNorm: 100 us
// of which 9 us of kernels; the forward call of one box prompt's attention 15 us, 5 us of kernel).
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <cstdint>

#include "../../include/sparsesam.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// A non-zero status; becomes sparsesam_b200._lib.SparseSAMError in Python.
struct StatusError : std::runtime_error {
  const char* fn;
  int status;
  StatusError(const char* f, int s)
      : std::runtime_error(std::string(f) + " failed with status " + std::to_string(s) + " (" + ssam_status_string(s) + ")"),
        fn(f),
        status(s) {}
};

void done(const char* fn, int status) {
  if (status != SSAM_OK) throw StatusError(fn, status);
}
#define SSAM_CALL(fn, ...) done(#fn, fn(__VA_ARGS__))

void refuse(const std::string& why) { throw py::value_error(why); }

// the calls' device and its current stream
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

int dtype_code(at::ScalarType t) {
  return t == at::kHalf ? 0 : t == at::kBFloat16 ? 1 : t == at::kFloat ? 2 : -1;
}
void check_devices(const Tensor& first, std::initializer_list<const Tensor*> others) {
  bool cuda = first.is_cuda(), same = true;
  for (const Tensor* t : others)
    if (t->defined()) cuda = cuda && t->is_cuda(), same = same && t->device() == first.device();
  if (!cuda) refuse("sparsesam_b200 ops run on CUDA tensors only (no CPU fallback)");
  if (!same) refuse("all tensors of a call must be on one device");
}
// the C entry points count tokens, heads and channels in 32 bits
void check_sizes(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    for (const int64_t n : t->sizes())
      if (n > INT32_MAX) refuse("a dimension of " + std::to_string(n) + " entries is not supported (at most 2^31 - 1)");
}
// These calls are no operators of torch's dispatcher: what follows a program operator by operator does not see them.
// A trace would hold uninitialised memory in their place and a tangent would be dropped, both without a word; tensors
// that wrap others (vmap, grad and functionalize of torch.func, fake tensors, subclasses) have no memory of their own.
bool plain(const Tensor& t) {
  constexpr c10::DispatchKeySet wrapped(
      {c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
       c10::DispatchKey::Batched, c10::DispatchKey::Functionalize, c10::DispatchKey::Conjugate,
       c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
  return t.layout() == at::kStrided && !t.is_nested() && !t.key_set().has_any(wrapped) && !t._fw_grad(0).defined();
}
bool followed() {
  return torch::jit::tracer::isTracing() ||
         c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
}
bool takes(const std::vector<Tensor>& ts) {
  for (const Tensor& t : ts)
    if (!plain(t)) return false;
  return !followed();
}
void check_plain(const char* op, std::initializer_list<const Tensor*> ts) {
  bool ok = !followed();
  for (const Tensor* t : ts) ok = ok && (!t->defined() || plain(*t));
  if (!ok)
    throw std::runtime_error(std::string(op) + " takes plain tensors outside of traces: torch.jit.trace, make_fx, torch.func "
                             "transforms, forward-mode differentiation and tensor subclasses do not see it");
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// t in row-major memory that vector loads can read (an incoming gradient may have any layout)
Tensor dense(const Tensor& t) {
  const Tensor c = t.contiguous();
  return aligned(c) ? c : c.clone();
}

// Gradients may not be differentiated again: where a graph of the backward pass is recorded (and something of it
// could require that), the results get a node that says so.
variable_list once(const char* op, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list real;
  for (const Tensor& g : grads)
    if (g.defined()) real.push_back(g.detach().requires_grad_(true));   // so that the node enters the graph
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string("the backward pass of ") + op + " cannot be differentiated", static_cast<int64_t>(real.size()));
  real = (*node)(std::move(real));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = real[i++];
  return grads;
}

// ---------------------------------------------------------------------------
// Channel LayerNorm (+ GELU) of half rows
// ---------------------------------------------------------------------------
Tensor layernorm_run(const Tensor& x, const Tensor& w, const Tensor& b, double eps, int64_t gelu) {
  Tensor out = at::empty_like(x);
  const int64_t C = x.size(-1);
  if (x.numel() == 0) return out;
  const On on(x);
  SSAM_CALL(ssam_layernorm_gelu_half, x.data_ptr(), x.numel() / C, static_cast<int>(C), w.data_ptr(), b.data_ptr(),
            static_cast<float>(eps), static_cast<int>(gelu), dtype_code(x.scalar_type()), out.data_ptr(), on.stream);
  return out;
}

struct LayerNormGelu : torch::autograd::Function<LayerNormGelu> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& b, double eps, int64_t gelu) {
    ctx->save_for_backward({x, w, b});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["gelu"] = gelu;
    return layernorm_run(x, w, b, eps, gelu);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
    const int C = static_cast<int>(x.size(-1));
    const int64_t rows = C == 0 ? 0 : x.numel() / C;
    variable_list out(5);
    {
      at::AutoGradMode off(false);
      if (rows == 0) {
        out[0] = at::zeros_like(x), out[1] = at::zeros_like(w), out[2] = at::zeros_like(b);
      } else {
        const Tensor dout = dense(grads[0]);
        out[0] = at::empty_like(x), out[1] = at::empty_like(w), out[2] = at::empty_like(b);
        const size_t n = ssam_layernorm_gelu_half_bwd_workspace_size(rows, C);
        const Tensor ws = at::empty({static_cast<int64_t>(n)}, x.options().dtype(at::kByte));
        const On on(x);
        SSAM_CALL(ssam_layernorm_gelu_half_bwd, x.data_ptr(), dout.data_ptr(), rows, C, w.data_ptr(), b.data_ptr(),
                  static_cast<float>(ctx->saved_data["eps"].toDouble()), static_cast<int>(ctx->saved_data["gelu"].toInt()),
                  dtype_code(x.scalar_type()), out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), ws.data_ptr(), n,
                  on.stream);
      }
    }
    return once("layernorm_gelu_half", std::move(out));
  }
};

Tensor layernorm_gelu_half(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool gelu) {
  check_plain("layernorm_gelu_half", {&x, &w, &b});
  const auto dt = x.scalar_type();
  if ((dt != at::kHalf && dt != at::kBFloat16) || w.scalar_type() != dt || b.scalar_type() != dt) {
    check_devices(x, {&w, &b});
    refuse("x, w and b must share one half-precision dtype");
  }
  if (!x.is_contiguous() || !w.is_contiguous() || !b.is_contiguous()) refuse("x, w and b must be contiguous");
  check_sizes({&w});
  if (x.dim() < 1 || w.numel() != x.size(-1) || b.numel() != x.size(-1)) refuse("w and b must have one entry per channel");
  check_devices(x, {&w, &b});
  if (wants_grad({&x, &w, &b})) return LayerNormGelu::apply(x, w, b, eps, static_cast<int64_t>(gelu));
  return layernorm_run(x, w, b, eps, gelu);
}

// ---------------------------------------------------------------------------
// GroupNorm + activation
// ---------------------------------------------------------------------------
struct GnSize {
  int N, C;
  int64_t HW;
  explicit GnSize(const Tensor& x)
      : N(static_cast<int>(x.size(0))), C(static_cast<int>(x.size(-1))), HW(x.numel() / (x.size(0) * x.size(-1))) {}
};
// stats: undefined, or [2, N, groups] (mean, rstd)
Tensor groupnorm_run(const Tensor& x, int groups, const Tensor& w, const Tensor& b, double eps, int act, Tensor* stats) {
  Tensor out = at::empty_like(x);
  if (x.numel() == 0) return out;
  const GnSize s(x);
  const int dt = dtype_code(x.scalar_type());
  float* mean = nullptr;
  if (stats != nullptr) {
    *stats = at::empty({2, s.N, groups}, x.options().dtype(at::kFloat));
    mean = stats->data_ptr<float>();
  }
  const size_t n = ssam_groupnorm_act_workspace_size(s.N, s.HW, s.C, groups, dt, 0);
  Tensor ws;
  if (n) ws = at::empty({static_cast<int64_t>(n)}, x.options().dtype(at::kByte));
  const On on(x);
  SSAM_CALL(ssam_groupnorm_act_fwd, x.data_ptr(), s.N, s.HW, s.C, groups, w.data_ptr(), b.data_ptr(),
            static_cast<float>(eps), act, dt, out.data_ptr(), mean,
            mean == nullptr ? nullptr : mean + static_cast<int64_t>(s.N) * groups, ptr(ws), n, on.stream);
  return out;
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& b, int64_t groups, double eps,
                        int64_t act) {
    Tensor stats;
    Tensor out = groupnorm_run(x, static_cast<int>(groups), w, b, eps, static_cast<int>(act), &stats);
    ctx->save_for_backward({x, w, b, stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
    variable_list out(6);
    {
      at::AutoGradMode off(false);
      if (x.numel() == 0) {
        out[0] = at::zeros_like(x), out[1] = at::zeros_like(w), out[2] = at::zeros_like(b);
      } else {
        const GnSize s(x);
        const int groups = static_cast<int>(ctx->saved_data["groups"].toInt()), dt = dtype_code(x.scalar_type());
        const Tensor dout = dense(grads[0]);
        out[0] = at::empty_like(x), out[1] = at::empty_like(w), out[2] = at::empty_like(b);
        const size_t n = ssam_groupnorm_act_workspace_size(s.N, s.HW, s.C, groups, dt, 1);
        const Tensor ws = at::empty({static_cast<int64_t>(n)}, x.options().dtype(at::kByte));
        const float* mean = saved[3].data_ptr<float>();
        const On on(x);
        SSAM_CALL(ssam_groupnorm_act_bwd, x.data_ptr(), dout.data_ptr(), s.N, s.HW, s.C, groups, w.data_ptr(),
                  b.data_ptr(), mean, mean + static_cast<int64_t>(s.N) * groups, static_cast<int>(ctx->saved_data["act"].toInt()),
                  dt, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), ws.data_ptr(), n, on.stream);
      }
    }
    return once("groupnorm_act", std::move(out));
  }
};

Tensor groupnorm_act(const Tensor& x, int64_t groups, const Tensor& w, const Tensor& b, double eps, int64_t act) {
  check_plain("groupnorm_act", {&x, &w, &b});
  const auto dt = x.scalar_type();
  if (dtype_code(dt) < 0 || w.scalar_type() != dt || b.scalar_type() != dt)
    throw py::type_error("x, w and b must share one dtype of fp16, bf16, fp32");
  check_sizes({&x});
  if (x.dim() < 2 || w.dim() != 1 || b.dim() != 1 || w.size(0) != x.size(-1) || b.size(0) != x.size(-1))
    refuse("x must be (N, ..., C), w and b (C,)");
  if (!x.is_contiguous() || !w.is_contiguous() || !b.is_contiguous())
    refuse("x, w and b must be contiguous (x channels-last)");
  const int64_t C = x.size(-1), unit = dt == at::kFloat ? 4 : 8;
  if (groups <= 0 || C % groups || C % unit || C > 256 * unit)
    refuse(std::to_string(groups) + " groups of " + std::to_string(C) +
           " channels are not supported: groups divide the channels, a multiple of 8 up to 2048 (fp32: of 4 up to 1024)");
  check_devices(x, {&w, &b});
  if (wants_grad({&x, &w, &b})) return GroupNormAct::apply(x, w, b, groups, eps, act);
  return groupnorm_run(x, static_cast<int>(groups), w, b, eps, static_cast<int>(act), nullptr);
}

// ---------------------------------------------------------------------------
// Cross attention
// ---------------------------------------------------------------------------
struct XSize {
  int B, Tq, Tk, H, Hk, D, dt;
  XSize(const Tensor& q, const Tensor& k)
      : B(static_cast<int>(q.size(0))), Tq(static_cast<int>(q.size(1))), Tk(static_cast<int>(k.size(1))),
        H(static_cast<int>(q.size(2))), Hk(static_cast<int>(k.size(2))), D(static_cast<int>(q.size(3))),
        dt(dtype_code(q.scalar_type())) {}
  bool empty() const { return B == 0 || Tq == 0 || Tk == 0; }
};
struct Strides {
  int64_t s[12];
  Strides(const Tensor& a, const Tensor& b, const Tensor& c, const Tensor& d) {
    int i = 0;
    for (const Tensor* t : {&a, &b, &c, &d})
      for (int k = 0; k < 3; ++k) s[i++] = t->size(k) == 1 ? 0 : t->stride(k);   // the stride of one entry means nothing
  }
};
// every (batch, token, head) row contiguous and on a 16-byte boundary
bool vector_rows(const Tensor& t) {
  const int64_t unit = 16 / static_cast<int64_t>(t.element_size());
  if (!aligned(t) || (t.stride(3) != 1 && t.size(3) > 1)) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && t.stride(i) % unit) return false;
  return true;
}

Tensor attn_run(const Tensor& q, const Tensor& k, const Tensor& v, double scale, const Tensor& lens, const Tensor& mask,
                bool train, Tensor* out32, Tensor* stats) {
  const XSize s(q, k);
  Tensor out = at::empty({s.B, s.Tq, s.H, s.D}, q.options());
  if (s.empty()) return out.zero_();
  if (train && ssam_cross_attn_bwd_uses_stats(s.Tk, s.D, s.dt)) {
    *stats = at::empty({2, s.B, s.H, s.Tq}, q.options().dtype(at::kFloat));      // lse, D
    *out32 = s.dt == 2 ? out : at::empty({s.B, s.Tq, s.H, s.D}, q.options().dtype(at::kFloat));
  }
  const Strides st(q, k, v, out);
  const On on(q);
  SSAM_CALL(ssam_cross_attn_fwd, q.data_ptr(), k.data_ptr(), v.data_ptr(), st.s, s.B, s.Tq, s.Tk, s.H, s.Hk, s.D, s.dt,
            static_cast<float>(scale), static_cast<const int32_t*>(ptr(lens)), static_cast<const uint8_t*>(ptr(mask)),
            out.data_ptr(), s.dt == 2 ? nullptr : static_cast<float*>(ptr(*out32)), static_cast<float*>(ptr(*stats)),
            on.stream);
  return out;
}

struct CrossAttn : torch::autograd::Function<CrossAttn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, double scale,
                        const std::optional<Tensor>& lens_, const std::optional<Tensor>& mask_) {
    const Tensor lens = lens_.value_or(Tensor()), mask = mask_.value_or(Tensor());
    Tensor out32, stats;
    Tensor out = attn_run(q, k, v, scale, lens, mask, true, &out32, &stats);
    ctx->save_for_backward({q, k, v, out32, stats, lens, mask});
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out32 = saved[3], &stats = saved[4];
    const XSize s(q, k);
    const bool need_q = ctx->needs_input_grad(0), need_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    variable_list out(6);
    {
      at::AutoGradMode off(false);
      if (need_q) out[0] = at::empty({s.B, s.Tq, s.H, s.D}, q.options());
      if (need_kv) {
        out[1] = at::empty({s.B, s.Tk, s.Hk, s.D}, q.options());
        out[2] = at::empty({s.B, s.Tk, s.Hk, s.D}, q.options());
      }
      if (s.empty()) {     // no keys or no queries: nothing depends on anything
        for (Tensor& g : out)
          if (g.defined()) g.zero_();
      } else {
        const Tensor dout = vector_rows(grads[0]) ? grads[0] : grads[0].clone(at::MemoryFormat::Contiguous);
        const Strides st(q, k, v, dout);
        float* lse = static_cast<float*>(ptr(stats));
        const On on(q);
        SSAM_CALL(ssam_cross_attn_bwd, q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(),
                  st.s, s.B, s.Tq, s.Tk, s.H, s.Hk, s.D, s.dt, static_cast<float>(ctx->saved_data["scale"].toDouble()),
                  static_cast<const int32_t*>(ptr(saved[5])), static_cast<const uint8_t*>(ptr(saved[6])),
                  static_cast<const float*>(ptr(out32)), lse,
                  lse == nullptr ? nullptr : lse + static_cast<int64_t>(s.B) * s.H * s.Tq, ptr(out[0]), ptr(out[1]),
                  ptr(out[2]), on.stream);
      }
      if (!ctx->needs_input_grad(1)) out[1] = Tensor();
      if (!ctx->needs_input_grad(2)) out[2] = Tensor();
    }
    return once("cross_attn", std::move(out));
  }
};

std::string shape(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

Tensor cross_attn(const Tensor& q, const Tensor& k, const Tensor& v, std::optional<double> scale_, const std::optional<Tensor>& lens_,
                  const std::optional<Tensor>& mask_) {
  const Tensor lens = lens_.value_or(Tensor()), mask = mask_.value_or(Tensor());
  check_plain("cross_attn", {&q, &k, &v, &lens, &mask});
  if (q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
    refuse("q (B, Tq, H, D), k and v (B, Tk, Hk, D) expected, got " + shape(q) + ", " + shape(k) + ", " + shape(v));
  check_sizes({&q, &k});
  const auto dt = q.scalar_type();
  if (dtype_code(dt) < 0 || k.scalar_type() != dt || v.scalar_type() != dt)
    throw py::type_error("q, k and v must share one dtype of fp16, bf16, fp32");
  const int64_t H = q.size(2), Hk = k.size(2), D = q.size(3);
  if (Hk <= 0 || H <= 0 || H % Hk || D <= 0 || D > 128 || D % 8)
    refuse("heads " + std::to_string(H) + " / " + std::to_string(Hk) + " of " + std::to_string(D) +
           " are not supported: key heads divide query heads, head size a multiple of 8 up to 128");
  if (!vector_rows(q) || !vector_rows(k) || !vector_rows(v)) refuse("q, k and v need contiguous, 16-byte aligned head rows");
  if (lens.defined() && (lens.scalar_type() != at::kInt || lens.dim() != 1 || lens.size(0) != k.size(0) || !lens.is_contiguous()))
    refuse("key_lens must be contiguous int32 (B,)");
  if (mask.defined() && (mask.scalar_type() != at::kBool || mask.dim() != 2 || mask.size(0) != k.size(0) ||
                         mask.size(1) != k.size(1) || !mask.is_contiguous()))
    refuse("key_mask must be contiguous bool (B, Tk)");
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt(static_cast<double>(D));
  if (!(scale > 0.0 && scale < 2e38)) refuse("scale must be positive and below 2e38, got " + std::to_string(scale));
  check_devices(q, {&k, &v, &lens, &mask});
  if (wants_grad({&q, &k, &v})) return CrossAttn::apply(q, k, v, scale, lens_, mask_);
  Tensor out32, stats;
  return attn_run(q, k, v, scale, lens, mask, false, &out32, &stats);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const StatusError& e) {
      const py::object type = py::module_::import("sparsesam_b200._lib").attr("SparseSAMError");
      const py::object err = type(e.fn, e.status, ssam_status_string(e.status));
      PyErr_SetObject(type.ptr(), err.ptr());
    }
  });
  m.def("layernorm_gelu_half", &layernorm_gelu_half);
  m.def("groupnorm_act", &groupnorm_act);
  m.def("cross_attn", &cross_attn);
  m.def("takes", &takes);
}
