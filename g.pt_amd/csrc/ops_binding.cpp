// Python binding of the operators of gpt_amd.ops: argument checks, result allocation and autograd nodes around the C entries of
// include/gpt_hip.h.  In C++ because a call's host time is what small batches pay: through ctypes and a Python autograd function the
// forward cost 15 - 24 us and a forward + backward 165 us of host time, several times the kernels'.
// The C entries are looked up in the library that gpt_amd._lib has loaded; this module links nothing of it.
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>

#include <cmath>
#include <optional>

#include "../../include/gpt_hip.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct GptError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <typename... A>
[[noreturn]] void fail(const char* who, A&&... a) {
  throw GptError(c10::str(who, ": ", std::forward<A>(a)...));
}
#define OPS_CHECK(cond, who, ...) \
  do {                            \
    if (!(cond)) fail(who, __VA_ARGS__); \
  } while (0)

// ------------------------------------------------------------------------------------------------------- the C entries
struct Entries {
  decltype(&gpt_last_error) last_error = nullptr;
  decltype(&gpt_dropout_add) dropout_add = nullptr;
  decltype(&gpt_add_rmsnorm) add_rmsnorm = nullptr;
  decltype(&gpt_add_rmsnorm_bwd) add_rmsnorm_bwd = nullptr;
  decltype(&gpt_add_rmsnorm_bwd_workspace) add_rmsnorm_bwd_workspace = nullptr;
  decltype(&gpt_diff_attention_keep) diff_attention = nullptr;
  decltype(&gpt_diff_attention_workspace) diff_attention_workspace = nullptr;
  decltype(&gpt_diff_attention_bwd_kept) diff_attention_bwd = nullptr;
  decltype(&gpt_diff_attention_bwd_workspace) diff_attention_bwd_workspace = nullptr;
} lib;

void bind_library(uintptr_t handle) {
  auto get = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(reinterpret_cast<void*>(handle), name));
    OPS_CHECK(f, "gpt_ops", "the library does not export ", name);
  };
  get(lib.last_error, "gpt_last_error");
  get(lib.dropout_add, "gpt_dropout_add");
  get(lib.add_rmsnorm, "gpt_add_rmsnorm");
  get(lib.add_rmsnorm_bwd, "gpt_add_rmsnorm_bwd");
  get(lib.add_rmsnorm_bwd_workspace, "gpt_add_rmsnorm_bwd_workspace");
  get(lib.diff_attention, "gpt_diff_attention_keep");
  get(lib.diff_attention_workspace, "gpt_diff_attention_workspace");
  get(lib.diff_attention_bwd, "gpt_diff_attention_bwd_kept");
  get(lib.diff_attention_bwd_workspace, "gpt_diff_attention_bwd_workspace");
}

void check(int status, const char* what) {
  if (status != 0) throw GptError(c10::str(what, " failed (status ", status, "): ", lib.last_error()));
}

// ------------------------------------------------------------------------------------------------------- small helpers
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int code(const Tensor& t, const char* who, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return GPT_BF16;
  if (t.scalar_type() == at::kFloat) return GPT_F32;
  fail(who, name, " must be float32 or bfloat16 (got ", t.scalar_type(), ")");
}

// A tracer would record the allocation of the result and none of the launches that fill it: a graph of uninitialised memory.  Refused are
// torch.jit.trace, the modes of torch that trace (fake tensors, make_fx with and without pre_dispatch, functionalization) and the
// transforms' wrapped tensors.  A caller's own dispatch mode (a FLOP counter, selective checkpointing) sees the allocation alone as well, but
// the call's result is right under it.
void not_traced(const char* who, std::initializer_list<const Tensor*> tensors) {
  using c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::BatchedNestedTensor, c10::DispatchKey::Functionalize,
                                         c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchDynamicLayerFrontMode});
  bool traced = torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
  if (TorchDispatchModeTLS::any_modes_set())
    for (Key k : {Key::FAKE, Key::PROXY, Key::FUNCTIONAL}) traced |= TorchDispatchModeTLS::get_mode(k).has_value();
  for (const Tensor* t : tensors) traced |= t && t->defined() && t->key_set().has_any(wrapped);
  OPS_CHECK(!traced, who, "tracing and function transforms (jit.trace, make_fx, fake tensors, torch.func) are not implemented");
}

// What the nodes below do not carry on is refused, not dropped: the tangents of forward-mode differentiation
void plain_call(const char* who, std::initializer_list<const Tensor*> tensors) {
  not_traced(who, tensors);
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : tensors)
    OPS_CHECK(!t || !t->defined() || !t->_fw_grad(/*level=*/0).defined(), who, "forward-mode differentiation is not implemented");
}

void same_device(const char* who, std::initializer_list<const Tensor*> tensors) {
  plain_call(who, tensors);
  const Tensor* first = nullptr;
  for (const Tensor* t : tensors) {
    if (!t || !t->defined()) continue;
    OPS_CHECK(t->is_cuda(), who, "the HIP path needs GPU tensors; there is no CPU fallback");
    if (!first) first = t;
    OPS_CHECK(t->device() == first->device(), who, "tensors on different devices (", first->device(), " and ", t->device(), ")");
  }
}
const Tensor* ptr(const OptTensor& t) { return t && t->defined() ? &*t : nullptr; }

bool needs_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}

// `t` [..., d] as rows of d consecutive elements: the tensor that holds them (a copy only where the strides do not allow it) and the
// row stride
struct Rows {
  Tensor t;
  int64_t ld;
  explicit Rows(const Tensor& x) : t(x) {
    const int64_t d = x.size(-1);
    ld = d;
    if (x.is_contiguous()) return;
    if (x.stride(-1) == 1 || d == 1) {
      int64_t below = -1;                                 // stride of the row index that the dimensions passed so far make up
      int64_t count = 1, row = d;
      bool ok = true;
      for (int64_t i = x.dim() - 2; i >= 0 && ok; --i) {
        if (x.size(i) == 1) continue;
        if (below < 0) { row = below = x.stride(i); count = x.size(i); }
        else { ok = x.stride(i) == below * count; count *= x.size(i); }
      }
      if (ok) { ld = row; return; }
    }
    t = x.contiguous();
  }
  void* p() const { return t.data_ptr(); }
};

// the mask of a call; `active` false: nothing is dropped
struct Drop {
  gpt_dropout_t c{};
  bool active = false;
  const gpt_dropout_t* get() const { return active ? &c : nullptr; }
};
Drop make_drop(const char* who, double p, uint64_t seed, uint64_t offset, const Tensor* counter) {
  OPS_CHECK(p >= 0.0 && p <= 1.0, who, "dropout probability ", p, " not in [0, 1]");
  OPS_CHECK(!counter || (counter->scalar_type() == at::kLong && counter->numel() == 1), who, "counter must be an int64 tensor of one element");
  Drop d;
  d.active = std::nearbyint(65536.0 * p) != 0.0;
  d.c.p = p;
  d.c.seed = seed;
  d.c.offset = offset;
  d.c.offset_dev = counter ? reinterpret_cast<const uint64_t*>(counter->data_ptr()) : nullptr;
  return d;
}

bool wants_grad(const Tensor* t) { return t && t->defined() && t->requires_grad(); }

// a node whose backward is not itself differentiable: with create_graph, gradients that would have a graph - because the incoming one has,
// or because they depend on inputs that require one themselves (`curved`) - are an error, not constants
struct OnceNode : torch::autograd::Node {
  // (the node's members are read under its lock: a graph may be run by one thread and released by another)
  std::lock_guard<std::mutex> hold() { return std::lock_guard<std::mutex>(mutex_); }
  void once(const char* who, const variable_list& grads) {
    for (const Tensor& g : grads) plain_call(who, {&g});
    if (!at::GradMode::is_enabled()) return;
    bool graph = curved;
    for (const Tensor& g : grads) graph |= g.defined() && g.requires_grad();
    if (graph) throw std::runtime_error(c10::str(who, ": the gradient cannot be differentiated again (create_graph)"));
  }
  bool curved = false;
};

template <typename N>
std::shared_ptr<N> make_node(std::initializer_list<const Tensor*> inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  torch::autograd::edge_list edges;
  edges.reserve(inputs.size());
  for (const Tensor* t : inputs) edges.push_back(t && t->defined() ? torch::autograd::impl::gradient_edge(*t) : torch::autograd::Edge());
  node->set_next_edges(std::move(edges));
  return node;
}

// ------------------------------------------------------------------------------------------------------------- dropout
// (resid or 0) + drop(h)
Tensor dropout_forward(const char* who, const Tensor& h, const Tensor* resid, at::ScalarType type, const gpt_dropout_t& drop) {
  c10::DeviceGuard guard(h.device());
  Tensor out = at::empty(h.sizes(), h.options().dtype(type).requires_grad(false));
  if (h.numel() == 0) return out;
  const int64_t d = h.size(-1);
  const Rows hr(h);
  std::optional<Rows> rr;
  if (resid) rr.emplace(*resid);
  check(lib.dropout_add(code(h, who, "h"), hr.p(), hr.ld, type == at::kBFloat16 ? GPT_BF16 : GPT_F32, rr ? rr->p() : nullptr, rr ? rr->ld : 0,
                        out.data_ptr(), d, h.numel() / d, d, &drop, stream_of(h)),
        "gpt_dropout_add");
  return out;
}

struct DropoutAddBackward : OnceNode {
  std::string name() const override { return "GptDropoutAddBackward"; }
  at::ScalarType h_type;
  double p;
  uint64_t seed, offset;
  bool has_resid;
  SavedVariable counter;    // saved, so that a counter advanced between forward and backward is an error and not another mask
  bool has_counter;
  variable_list apply(variable_list&& grads) override {
    const char* who = "dropout_add (backward)";
    const auto lock = hold();
    once(who, grads);
    variable_list out(has_resid ? 2 : 1);
    const Tensor& g = grads[0];
    if (!g.defined()) return out;
    at::NoGradGuard no_grad;
    if (task_should_compute_output(0)) {
      const Tensor c = has_counter ? counter.unpack() : Tensor();
      const Drop drop = make_drop(who, p, seed, offset, has_counter ? &c : nullptr);
      out[0] = dropout_forward(who, g, nullptr, h_type, drop.c);
    }
    if (has_resid && task_should_compute_output(1)) out[1] = g;
    return out;
  }
  void release_variables() override {
    const auto lock = hold();
    counter.reset_data();
  }
};

Tensor dropout_add(const Tensor& h, const OptTensor& resid_, double p, uint64_t seed, uint64_t offset, const OptTensor& counter_) {
  const Tensor *resid = ptr(resid_), *counter = ptr(counter_);
  const char* who = resid ? "dropout_add" : "dropout";
  same_device(who, {&h, resid, counter});
  code(h, who, "h");
  if (resid) code(*resid, who, "resid");
  OPS_CHECK(h.dim() > 0, who, "h must have one dimension at least");
  OPS_CHECK(!resid || h.sizes() == resid->sizes(), who, "h and resid must have the same shape (got ", h.sizes(), " and ", resid->sizes(), ")");
  const Drop drop = make_drop(who, p, seed, offset, counter);
  const bool grad = needs_grad({&h, resid});
  Tensor out;
  {
    at::NoGradGuard no_grad;
    out = dropout_forward(who, h, resid, resid ? resid->scalar_type() : h.scalar_type(), drop.c);
  }
  if (grad) {
    auto node = resid ? make_node<DropoutAddBackward>({&h, resid}) : make_node<DropoutAddBackward>({&h});
    node->h_type = h.scalar_type();
    node->p = p; node->seed = seed; node->offset = offset;
    node->has_resid = resid != nullptr;
    node->has_counter = counter != nullptr;
    if (counter) node->counter = SavedVariable(*counter, false);
    torch::autograd::create_gradient_edge(out, node);
  }
  return out;
}

// ------------------------------------------------------------------------------------------------------------ RMS norm
struct NormOut {
  Tensor y, scales, x, rho;
};

// h undefined: x is resid itself.  y_type Float8_e4m3fn: the 8-bit output with its scales.
NormOut norm_forward(const char* who, const Tensor* h, const Tensor& resid, const Tensor& weight, double eps, const Drop& drop,
                     at::ScalarType y_type, bool keep) {
  c10::DeviceGuard guard(resid.device());
  at::NoGradGuard no_grad;
  const bool mx = y_type == at::kFloat8_e4m3fn;
  const int64_t d = resid.size(-1), rows = d ? resid.numel() / d : 0;
  const auto opt = resid.options().requires_grad(false);
  NormOut o;
  o.y = at::empty(resid.sizes(), opt.dtype(y_type));
  if (mx) {
    std::vector<int64_t> shape(resid.sizes().begin(), resid.sizes().end());
    shape.back() = d / 32;
    o.scales = at::empty(shape, opt.dtype(at::kFloat8_e8m0fnu));
  }
  o.x = h ? at::empty(resid.sizes(), opt) : resid;
  if (keep) o.rho = at::empty({rows}, opt.dtype(at::kFloat));
  if (rows == 0 || d == 0) return o;
  const Rows rr(resid);
  std::optional<Rows> hr;
  if (h) hr.emplace(*h);
  const Tensor w = weight.contiguous();
  gpt_add_rmsnorm_t a{};
  const int yc = y_type == at::kBFloat16 ? GPT_BF16 : GPT_F32;
  a.h_dtype = h ? code(*h, who, "h") : yc;
  a.x_dtype = code(resid, who, "resid");
  a.y_dtype = mx ? GPT_MXFP8 : yc;
  if (h) { a.h = hr->p(); a.ldh = hr->ld; a.x_out = o.x.data_ptr(); a.ldx = d; }
  a.resid = rr.p(); a.ldr = rr.ld;
  a.weight = w.data_ptr<float>();
  a.y = o.y.data_ptr(); a.ldy = d;
  a.scales = mx ? static_cast<uint8_t*>(o.scales.data_ptr()) : nullptr;
  a.rho = keep ? o.rho.data_ptr<float>() : nullptr;
  a.rows = rows; a.d = d; a.eps = (float)eps;
  a.drop = drop.get();
  check(lib.add_rmsnorm(&a, stream_of(resid)), "gpt_add_rmsnorm");
  return o;
}

struct AddRmsNormBackward : OnceNode {
  std::string name() const override { return "GptAddRmsNormBackward"; }
  SavedVariable x, weight, rho, counter;
  at::ScalarType y_type;
  bool has_h, has_counter;
  double p;
  uint64_t seed, offset;
  variable_list apply(variable_list&& grads) override {
    const char* who = "add_rms_norm (backward)";
    const auto lock = hold();
    once(who, grads);
    variable_list out(3);                                              // h, resid, weight
    Tensor gy = grads[0];
    const Tensor gx = has_h ? grads[1] : Tensor();
    if (!gy.defined() && !gx.defined()) return out;
    at::NoGradGuard no_grad;
    const Tensor xv = x.unpack(has_h ? shared_from_this() : nullptr), wv = weight.unpack(), rv = rho.unpack();
    const Tensor cv = has_counter ? counter.unpack() : Tensor();
    c10::DeviceGuard guard(xv.device());
    const Drop drop = make_drop(who, p, seed, offset, has_counter ? &cv : nullptr);
    const int64_t d = xv.size(-1);
    const auto opt = xv.options().requires_grad(false);
    if (!gy.defined()) gy = at::zeros(xv.sizes(), opt.dtype(y_type));
    const Tensor dr = at::empty(xv.sizes(), opt);
    const Tensor dh = has_h && task_should_compute_output(0) ? at::empty(xv.sizes(), opt.dtype(y_type)) : Tensor();
    const Tensor dw = task_should_compute_output(2) ? at::empty({d}, opt.dtype(at::kFloat)) : Tensor();
    if (xv.numel() == 0) {
      if (dw.defined()) dw.zero_();
    } else {
      const Rows g(gy), xr(xv);
      std::optional<Rows> gxr;
      if (gx.defined()) gxr.emplace(gx);
      const Tensor w = wv.contiguous();
      gpt_add_rmsnorm_bwd_t a{};
      a.y_dtype = a.h_dtype = code(gy, who, "gy");
      a.x_dtype = code(xv, who, "x");
      a.gy = g.p(); a.ldgy = g.ld;
      if (gxr) { a.gx = gxr->p(); a.ldgx = gxr->ld; }
      a.x = xr.p(); a.ldx = xr.ld;
      a.weight = w.data_ptr<float>(); a.rho = rv.data_ptr<float>();
      a.dresid = dr.data_ptr(); a.lddr = d;
      if (dh.defined()) { a.dh = dh.data_ptr(); a.lddh = d; }
      a.rows = xv.numel() / d; a.d = d;
      a.drop = drop.get();
      Tensor ws;
      if (dw.defined()) {
        int64_t bytes = 0;
        check(lib.add_rmsnorm_bwd_workspace(a.rows, d, &bytes), "gpt_add_rmsnorm_bwd_workspace");
        ws = at::empty({bytes}, opt.dtype(at::kByte));
        a.dweight = dw.data_ptr<float>(); a.ws = ws.data_ptr(); a.ws_bytes = bytes;
      }
      check(lib.add_rmsnorm_bwd(&a, stream_of(xv)), "gpt_add_rmsnorm_bwd");
    }
    out[0] = dh;
    if (task_should_compute_output(1)) out[1] = dr;
    out[2] = dw;
    return out;
  }
  void release_variables() override {
    const auto lock = hold();
    x.reset_data(); weight.reset_data(); rho.reset_data(); counter.reset_data();
  }
};

void check_norm(const char* who, const Tensor* h, const Tensor& resid, const Tensor& weight, double eps, const Tensor* counter) {
  same_device(who, {h, &resid, &weight, counter});
  code(resid, who, "the stream");
  if (h) {
    code(*h, who, "h");
    OPS_CHECK(h->sizes() == resid.sizes(), who, "h and resid must have the same shape (got ", h->sizes(), " and ", resid.sizes(), ")");
  }
  OPS_CHECK(resid.dim() > 0 && weight.scalar_type() == at::kFloat && weight.dim() == 1 && weight.size(0) == resid.size(-1), who,
            "weight must be float32 of the last dimension's size (got ", weight.scalar_type(), " ", weight.sizes(), " for ", resid.sizes(), ")");
  OPS_CHECK(eps >= 0.0 && std::isfinite(eps), who, "eps must be finite and not negative (got ", eps, ")");
}

NormOut norm_autograd(const char* who, const Tensor* h, const Tensor& resid, const Tensor& weight, double eps, double p, uint64_t seed,
                      uint64_t offset, const Tensor* counter, at::ScalarType y_type) {
  check_norm(who, h, resid, weight, eps, counter);
  const Drop drop = make_drop(who, p, seed, offset, counter);
  const bool grad = needs_grad({h, &resid, &weight});
  NormOut o = norm_forward(who, h, resid, weight, eps, drop, y_type, grad);
  if (grad) {
    auto node = make_node<AddRmsNormBackward>({h, &resid, &weight});
    node->curved = wants_grad(h) || wants_grad(&resid);                  // (the weight alone: its gradient does not depend on it)
    node->y_type = y_type;
    node->has_h = h != nullptr;
    node->has_counter = counter != nullptr;
    node->p = p; node->seed = seed; node->offset = offset;
    torch::autograd::create_gradient_edge(o.y, node);
    if (h) torch::autograd::create_gradient_edge(o.x, node);
    node->x = SavedVariable(o.x, h != nullptr);
    node->weight = SavedVariable(weight, false);
    node->rho = SavedVariable(o.rho, false);
    if (counter) node->counter = SavedVariable(*counter, false);
  }
  return o;
}

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& h, const Tensor& resid, const Tensor& weight, double eps, double p, uint64_t seed,
                                        uint64_t offset, const OptTensor& counter) {
  NormOut o = norm_autograd("add_rms_norm", &h, resid, weight, eps, p, seed, offset, ptr(counter), h.scalar_type());
  return {o.y, o.x};
}

Tensor rms_norm(const Tensor& x, const Tensor& weight, double eps, const std::optional<at::ScalarType>& out_type) {
  const at::ScalarType t = out_type ? *out_type : x.scalar_type();
  OPS_CHECK(!out_type || t == at::kFloat || t == at::kBFloat16, "rms_norm", "out_dtype must be float32 or bfloat16 (got ", t, ")");
  return norm_autograd("rms_norm", nullptr, x, weight, eps, 0.0, 0, 0, nullptr, t).y;
}

std::tuple<Tensor, Tensor, Tensor> norm_mx8(const OptTensor& h_, const Tensor& resid, const Tensor& weight, double eps, double p, uint64_t seed,
                                            uint64_t offset, const OptTensor& counter_) {
  const Tensor *h = ptr(h_), *counter = ptr(counter_);
  const char* who = h ? "add_rms_norm_mx8" : "rms_norm_mx8";
  check_norm(who, h, resid, weight, eps, counter);
  OPS_CHECK(resid.size(-1) % 32 == 0 && resid.size(-1) > 0, who, "the last dimension must be a multiple of 32 (got ", resid.size(-1), ")");
  OPS_CHECK(!needs_grad({h, &resid, &weight}), who, "the 8-bit output has no gradient: call it under torch.no_grad()");
  NormOut o = norm_forward(who, h, resid, weight, eps, make_drop(who, p, seed, offset, counter), at::kFloat8_e4m3fn, false);
  return {o.y, o.scales, o.x};
}

// ---------------------------------------------------------------------------------------------- differential attention
constexpr int64_t SHORT = 32;   // up to this many queries and keys the backward recomputes the maps and keeps nothing of the forward

// `t` [B, T, w] with rows the kernels take (a copy where the strides or the alignment do not allow it): token and sample stride
struct Tokens {
  Tensor t;
  int64_t ld, bs;
  explicit Tokens(const Tensor& x) : t(x) {
    const int64_t B = x.size(0), T = x.size(1), w = x.size(2), es = x.element_size();
    ld = T > 1 ? x.stride(1) : w;
    bs = B > 1 ? x.stride(0) : 0;
    if ((x.stride(2) != 1 && w > 1) || (T > 1 && ld < w) || ld >= (int64_t)1 << 25 || ld * es % 16 || bs * es % 16 ||
        reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) {
      t = x.contiguous();
      if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) t = t.clone();
      ld = w;
      bs = T * w;
    }
  }
};

// what a call is made of, checked
struct Attention {
  Tensor q, k, v, lam, lengths;
  int n_head = 0;
  float scale = 0;
  int64_t B() const { return q.size(0); }
  int64_t Tq() const { return q.size(1); }
  int64_t Tk() const { return k.size(1); }
  bool empty() const { return B() == 0 || Tq() == 0 || Tk() == 0; }
  bool is_short() const { return Tq() <= SHORT && Tk() <= SHORT; }
};

struct AttentionCall {
  gpt_diff_attention_t c{};
  Tokens q, k, v;
  explicit AttentionCall(const Attention& a) : q(a.q), k(a.k), v(a.v) {
    c.dtype = a.q.scalar_type() == at::kBFloat16 ? GPT_BF16 : GPT_F32;
    c.B = (int)a.B(); c.Tq = (int)a.Tq(); c.Tk = (int)a.Tk();
    c.n_head = a.n_head; c.hd = (int)(a.q.size(2) / (2 * a.n_head));
    c.scale = a.scale;
    c.q = q.t.data_ptr(); c.ldq = q.ld; c.bsq = q.bs;
    c.k = k.t.data_ptr(); c.ldk = k.ld; c.bsk = k.bs;
    c.v = v.t.data_ptr(); c.ldv = v.ld; c.bsv = v.bs;
    c.lam = a.lam.data_ptr<float>();
    c.lengths = a.lengths.defined() ? a.lengths.data_ptr<int>() : nullptr;
  }
};

struct AttentionOut {
  Tensor out, lse, out2, rest;
};

AttentionOut attention_forward(const Attention& a, bool keep) {
  c10::DeviceGuard guard(a.q.device());
  at::NoGradGuard no_grad;
  const auto opt = a.q.options().requires_grad(false);
  AttentionOut o;
  o.out = at::empty({a.B(), a.Tq(), a.q.size(2)}, opt);
  if (a.empty()) {
    if (o.out.numel()) o.out.zero_();
    return o;
  }
  AttentionCall call(a);
  auto& c = call.c;
  c.out = o.out.data_ptr(); c.ldo = a.q.size(2); c.bso = a.Tq() * a.q.size(2);
  if (keep && !a.is_short()) {
    o.lse = at::empty({2, a.B(), a.n_head, a.Tq()}, opt.dtype(at::kFloat));
    o.out2 = at::empty(o.out.sizes(), opt);
    c.lse = o.lse.data_ptr<float>(); c.out2 = o.out2.data_ptr();
    if (c.dtype == GPT_BF16) o.rest = at::empty({2, a.B(), a.Tq(), a.q.size(2)}, opt);
  }
  int64_t bytes = 0;
  check(lib.diff_attention_workspace(c.dtype, c.B, c.Tq, c.Tk, c.n_head, c.hd, &bytes), "gpt_diff_attention_workspace");
  Tensor ws;
  if (bytes) {
    ws = at::empty({bytes}, opt.dtype(at::kByte));
    c.ws = ws.data_ptr(); c.ws_bytes = bytes;
  }
  check(lib.diff_attention(&c, o.rest.defined() ? o.rest.data_ptr() : nullptr, stream_of(a.q)), "gpt_diff_attention");
  return o;
}

struct DiffAttentionBackward : OnceNode {
  std::string name() const override { return "GptDiffAttentionBackward"; }
  bool fused, has_lengths, kept, has_rest;
  SavedVariable q, k, v, lam, lengths, out, lse, out2, rest;           // fused: q holds the whole projection
  int n_head;
  float scale;
  variable_list apply(variable_list&& grads) override {
    const auto lock = hold();
    once("diff_attention (backward)", grads);
    const int n = fused ? 1 : 3;
    variable_list res(n + 1);
    const Tensor& g = grads[0];
    if (!g.defined()) return res;
    at::NoGradGuard no_grad;
    Attention a;
    Tensor dq, dk, dv;
    const Tensor first = q.unpack();
    c10::DeviceGuard guard(first.device());
    if (fused) {
      const int64_t w = first.size(2) / 3;
      a.q = first.narrow(2, 0, w); a.k = first.narrow(2, w, w); a.v = first.narrow(2, 2 * w, w);
      res[0] = at::empty(first.sizes(), first.options().requires_grad(false));
      dq = res[0].narrow(2, 0, w); dk = res[0].narrow(2, w, w); dv = res[0].narrow(2, 2 * w, w);
    } else {
      a.q = first; a.k = k.unpack(); a.v = v.unpack();
      res[0] = dq = at::empty(a.q.sizes(), first.options().requires_grad(false));
      res[1] = dk = at::empty(a.k.sizes(), first.options().requires_grad(false));
      res[2] = dv = at::empty(a.v.sizes(), first.options().requires_grad(false));
    }
    a.lam = lam.unpack();
    if (has_lengths) a.lengths = lengths.unpack();
    a.n_head = n_head; a.scale = scale;
    Tensor dlam = at::empty({n_head}, a.lam.options().requires_grad(false));
    res[n] = dlam;
    if (a.empty()) {
      for (Tensor& t : res) t.zero_();
      return res;
    }
    AttentionCall call(a);
    const Tensor o = kept ? out.unpack(shared_from_this()) : dq;         // not read where nothing was kept
    call.c.out = o.data_ptr(); call.c.ldo = o.stride(1); call.c.bso = o.stride(0);
    const Tensor lse_v = kept ? lse.unpack() : Tensor(), out2_v = kept ? out2.unpack() : Tensor(), rest_v = has_rest ? rest.unpack() : Tensor();
    if (kept) { call.c.lse = lse_v.data_ptr<float>(); call.c.out2 = out2_v.data_ptr(); }
    const Tokens gt(g);
    gpt_diff_attention_bwd_t b{};
    b.dout = gt.t.data_ptr(); b.lddo = gt.ld; b.bsdo = gt.bs;
    b.dq = dq.data_ptr(); b.lddq = dq.stride(1); b.bsdq = dq.stride(0);
    b.dk = dk.data_ptr(); b.lddk = dk.stride(1); b.bsdk = dk.stride(0);
    b.dv = dv.data_ptr(); b.lddv = dv.stride(1); b.bsdv = dv.stride(0);
    b.dlam = dlam.data_ptr<float>();
    int64_t bytes = 0;
    check(lib.diff_attention_bwd_workspace(call.c.dtype, call.c.B, call.c.Tq, call.c.Tk, n_head, call.c.hd, &bytes),
          "gpt_diff_attention_bwd_workspace");
    const Tensor ws = at::empty({bytes}, a.lam.options().dtype(at::kByte).requires_grad(false));
    b.ws = ws.data_ptr(); b.ws_bytes = bytes;
    check(lib.diff_attention_bwd(&call.c, has_rest ? rest_v.data_ptr() : nullptr, &b, stream_of(first)), "gpt_diff_attention_bwd");
    return res;
  }
  void release_variables() override {
    const auto lock = hold();
    for (SavedVariable* s : {&q, &k, &v, &lam, &lengths, &out, &lse, &out2, &rest}) s->reset_data();
  }
};

Tensor diff_attention_any(const char* who, const Tensor* qkv, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam,
                          int64_t n_head, const OptTensor& lengths_, const std::optional<double>& scale_) {
  const Tensor* lengths = ptr(lengths_);
  same_device(who, {&q, &k, &v, &lam, lengths});
  code(q, who, "q");
  OPS_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), who, "q, k and v must have one type (got ",
            q.scalar_type(), ", ", k.scalar_type(), ", ", v.scalar_type(), ")");
  OPS_CHECK(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && q.size(0) == k.size(0) && q.size(2) == k.size(2), who,
            "need q [B, Tq, w], k and v [B, Tk, w] (got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes(), ")");
  const int64_t w = q.size(2), hd = n_head > 0 && w % (2 * n_head) == 0 ? w / (2 * n_head) : 0;
  OPS_CHECK(hd == 32 || hd == 64 || hd == 96 || hd == 128, who, "width ", w, " with ", n_head,
            " heads: the head dim w / (2 n_head) must be 32, 64, 96 or 128");
  OPS_CHECK(lam.scalar_type() == at::kFloat && lam.dim() == 1 && (lam.size(0) == 1 || lam.size(0) == n_head), who,
            "lam must be float32 of 1 or ", n_head, " elements (got ", lam.scalar_type(), " ", lam.sizes(), ")");
  Attention a;
  a.q = q; a.k = k; a.v = v;
  // one weight for all heads: autograd sums the heads' gradients through the expansion
  a.lam = lam.size(0) == n_head && lam.is_contiguous() ? lam : lam.expand({n_head}).contiguous();
  if (lengths) {
    OPS_CHECK((lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong) && lengths->dim() == 1 && lengths->size(0) == q.size(0),
              who, "lengths must be int32 or int64 [", q.size(0), "] (got ", lengths->scalar_type(), " ", lengths->sizes(), ")");
    a.lengths = (lengths->scalar_type() == at::kLong ? lengths->clamp(0, k.size(1)).to(at::kInt) : *lengths).contiguous();
  }
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)hd);
  OPS_CHECK(scale > 0.0 && std::isfinite(scale), who, "scale must be positive and finite (got ", scale, ")");
  a.n_head = (int)n_head;
  a.scale = (float)scale;
  const bool grad = qkv ? needs_grad({qkv, &a.lam}) : needs_grad({&q, &k, &v, &a.lam});
  AttentionOut o = attention_forward(a, grad);
  if (grad) {
    auto node = qkv ? make_node<DiffAttentionBackward>({qkv, &a.lam}) : make_node<DiffAttentionBackward>({&q, &k, &v, &a.lam});
    // (v alone, or lam alone: linear in it)
    node->curved = wants_grad(qkv) || wants_grad(&q) || wants_grad(&k) || (wants_grad(&v) && wants_grad(&a.lam));
    node->fused = qkv != nullptr;
    node->has_lengths = a.lengths.defined();
    node->kept = o.lse.defined();
    node->has_rest = o.rest.defined();
    node->n_head = a.n_head;
    node->scale = a.scale;
    torch::autograd::create_gradient_edge(o.out, node);
    node->q = SavedVariable(qkv ? *qkv : q, false);
    if (!qkv) { node->k = SavedVariable(k, false); node->v = SavedVariable(v, false); }
    node->lam = SavedVariable(a.lam, false);
    if (a.lengths.defined()) node->lengths = SavedVariable(a.lengths, false);
    if (node->kept) { node->out = SavedVariable(o.out, true); node->lse = SavedVariable(o.lse, false); node->out2 = SavedVariable(o.out2, false); }
    if (node->has_rest) node->rest = SavedVariable(o.rest, false);
  }
  return o.out;
}

Tensor diff_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, int64_t n_head, const OptTensor& lengths,
                      const std::optional<double>& scale) {
  return diff_attention_any("diff_attention", nullptr, q, k, v, lam, n_head, lengths, scale);
}

Tensor diff_attention_qkv(const Tensor& qkv, const Tensor& lam, int64_t n_head, const OptTensor& lengths, const std::optional<double>& scale) {
  const char* who = "diff_attention_qkv";
  plain_call(who, {&qkv});                                                // (the detached ranges below have no tangent)
  OPS_CHECK(qkv.dim() == 3 && qkv.size(2) % 3 == 0, who, "qkv must be a [B, T, 3 w] tensor (got ", qkv.sizes(), ")");
  const int64_t w = qkv.size(2) / 3;
  const Tensor flat = qkv.detach();
  return diff_attention_any(who, &qkv, flat.narrow(2, 0, w), flat.narrow(2, w, w), flat.narrow(2, 2 * w, w), lam, n_head, lengths, scale);
}

PyObject* error_class = nullptr;

}  // namespace

PYBIND11_MODULE(gpt_ops, m) {
  m.doc() = "host side of gpt_amd.ops";
  m.def("init", [](uintptr_t handle, py::object error) {
    bind_library(handle);
    error_class = error.release().ptr();
  });
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const GptError& e) {
      PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
    }
  });
  m.def("dropout_add", &dropout_add);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("rms_norm", &rms_norm);
  m.def("norm_mx8", &norm_mx8);
  m.def("diff_attention", &diff_attention);
  m.def("diff_attention_qkv", &diff_attention_qkv);
}
