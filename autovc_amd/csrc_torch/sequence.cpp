// The sequence-model operators (autovc_amd/sequence.py) as torch functions over the C ABI of
// include/autovc_hip.h: argument checks, outputs and scratch from torch's allocator, the current
// stream, autograd.  It is C++ because on small tensors such a call costs what the host spends on
// it: the backward runs on a thread of autograd's own, whose core has none of the interpreter's
// objects in its caches.  A dropout of [64][512] with its gradient took 76 us through Python and
// ctypes and takes 47 here, as a multiplication of torch's own with its gradient does; a frame of the
// recurrence 10 and 4.5 us, a row's log-probabilities with five alternatives 13 and 5.6 us.
//
// The library is the one that autovc_amd._lib has loaded: bind() is given its path.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>

#include "../../include/autovc_hip.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
#define AVC_ENTRY(name) decltype(&::name) name = nullptr
  AVC_ENTRY(avc_last_error);
  AVC_ENTRY(avc_gated_recurrence_states);
  AVC_ENTRY(avc_gated_recurrence_workspace);
  AVC_ENTRY(avc_gated_recurrence_forward);
  AVC_ENTRY(avc_gated_recurrence_backward);
  AVC_ENTRY(avc_gated_recurrence_step);
  AVC_ENTRY(avc_token_log_probs_workspace);
  AVC_ENTRY(avc_token_log_probs_forward);
  AVC_ENTRY(avc_token_log_probs_backward);
  AVC_ENTRY(avc_dropout);
#undef AVC_ENTRY
} lib;

struct HipLibraryError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
PyObject* hip_library_error = nullptr;

void bind(const std::string& path, py::object error) {
  void* so = dlopen(path.c_str(), RTLD_NOW);
  TORCH_CHECK(so, "HIP library ", path, ": ", dlerror());
  auto entry = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(so, name));
    TORCH_CHECK(f, "HIP library ", path, " has no ", name);
  };
#define AVC_ENTRY(name) entry(lib.name, #name)
  AVC_ENTRY(avc_last_error);
  AVC_ENTRY(avc_gated_recurrence_states);
  AVC_ENTRY(avc_gated_recurrence_workspace);
  AVC_ENTRY(avc_gated_recurrence_forward);
  AVC_ENTRY(avc_gated_recurrence_backward);
  AVC_ENTRY(avc_gated_recurrence_step);
  AVC_ENTRY(avc_token_log_probs_workspace);
  AVC_ENTRY(avc_token_log_probs_forward);
  AVC_ENTRY(avc_token_log_probs_backward);
  AVC_ENTRY(avc_dropout);
#undef AVC_ENTRY
  hip_library_error = error.release().ptr();
}

// a call's status: ValueError for refused arguments, else HipLibraryError, as autovc_amd._lib.check
void done(int status, const char* what) {
  if (status == AVC_OK) return;
  TORCH_CHECK_VALUE(status != AVC_ERR_INVALID, what, ": ", lib.avc_last_error());
  throw HipLibraryError(c10::str(what, " failed (", status, "): ", lib.avc_last_error()));
}

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return AVC_DTYPE_F32;
    case at::kBFloat16: return AVC_DTYPE_BF16;
    case at::kHalf: return AVC_DTYPE_F16;
    default: return -1;
  }
}

void check_gpu(const Tensor& t, const char* name, const Tensor* like = nullptr) {
  TORCH_CHECK(t.is_cuda(), "autovc_amd runs on the GPU only (HIP kernels); ", name, " is a CPU tensor");
  TORCH_CHECK_VALUE(!like || t.device() == like->device(), name, " is on ", t.device(), ", expected ", like->device());
}
void check_data(const Tensor& t, const char* name) {
  check_gpu(t, name);
  TORCH_CHECK_TYPE(dtype_of(t) >= 0, name, " has dtype ", t.scalar_type());
}
void check_type(const Tensor& t, const char* name, const Tensor& like, at::ScalarType a, at::ScalarType b) {
  check_gpu(t, name, &like);
  TORCH_CHECK_TYPE(t.scalar_type() == a || t.scalar_type() == b, name, " has dtype ", t.scalar_type());
}

// The outputs are filled behind torch's back: a tangent of forward-mode differentiation would be lost, and a
// trace would hold nothing but the allocation of its outputs.
template <typename... T>
void check_seen(const char* what, const T&... inputs) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Mode = c10::impl::TorchDispatchModeKey;
  TORCH_CHECK((... && !torch::autograd::isFwGradDefined(inputs)), what, " has no forward-mode derivative");
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !Modes::get_mode(Mode::FAKE) && !Modes::get_mode(Mode::PROXY) &&
                  !Modes::get_mode(Mode::FUNCTIONAL),
              what, " cannot be traced: it is no operator of torch's dispatcher");
}

// t with its values as they stand in memory (a view may be the negative of what it shows: the imaginary part
// of a conjugate)
Tensor as_stored(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor dense(const Tensor& t) { return as_stored(t).contiguous(); }

// A matrix whose rows the kernels can walk: t itself unless its rows are not dense, overlap or lie `most`
// elements apart or more.
struct Rows {
  Tensor t;
  long ld;
  explicit Rows(const Tensor& given, long most = LONG_MAX) : t(as_stored(given)), ld(t.size(1)) {
    const Tensor m = t;
    if (m.is_contiguous()) return;
    const bool dense = m.size(1) <= 1 || m.stride(1) == 1, apart = m.size(0) <= 1 || m.stride(0) >= m.size(1);
    if (!dense || !apart || (m.size(0) > 1 && m.stride(0) >= most)) t = m.contiguous();
    else if (m.size(0) > 1) ld = m.stride(0);
  }
  void* p() const { return t.data_ptr(); }
};

// The tensors' device made current, and its current stream.
struct On {
  c10::DeviceGuard guard;
  void* stream;
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

Tensor scratch(const Tensor& like, size_t bytes) {
  return bytes ? at::empty({(long)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
template <typename T = void>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

bool wants_grad(const Tensor& a) { return a.requires_grad() && at::GradMode::is_enabled(); }
bool wants_grad(const Tensor& a, const optional<Tensor>& b) {
  return (a.requires_grad() || (b && b->requires_grad())) && at::GradMode::is_enabled();
}

// Gradients (formed without a graph) that are not differentiable themselves: where a graph of them is asked for
// (create_graph), using that graph is an error.  It leads to the incoming gradients and, unless the gradients
// are linear in them alone, to the inputs of the running node.
variable_list once(const variable_list& incoming, variable_list grads, bool linear = false) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::edge_list edges = torch::autograd::collect_next_edges(incoming);
  // (a compiled backward runs without a node)
  if (const auto node = linear ? nullptr : torch::autograd::get_current_node())
    edges.insert(edges.end(), node->next_edges().begin(), node->next_edges().end());
  if (std::none_of(edges.begin(), edges.end(), [](const auto& e) { return e.is_valid(); })) return grads;
  auto error = std::make_shared<torch::autograd::Error>(
      "trying to differentiate twice a function whose gradient is not differentiable", std::move(edges));
  for (Tensor& g : grads)
    if (g.defined()) torch::autograd::set_history(g, error);
  return grads;
}

// ---- gated linear recurrence ----------------------------------------------------------------------
struct RecShape {
  long T, B, H, dirs;
  long D() const { return dirs == 3 ? 2 : 1; }
  // row strides that the kernels' 32-bit offsets do not reach, where up to 64 rows share a wave
  long too_far() const { return H >= 128 ? 1L << 29 : 1L << 23; }
};

std::tuple<Tensor, Tensor, Tensor> recurrence_forward(const Tensor& gates, const Tensor& h0, const Tensor& lengths,
                                                      const RecShape& s, bool keep) {
  const int dt = dtype_of(gates);
  const Rows g(gates, s.too_far());
  const auto f32 = gates.options().dtype(at::kFloat);
  Tensor y = at::empty({s.T * s.B, s.D() * s.H}, gates.options()), hT = at::empty({s.D(), s.B, s.H}, f32), states;
  if (keep) states = at::empty({(long)lib.avc_gated_recurrence_states(s.T, s.B, s.H, s.dirs)}, f32);
  const size_t bytes = lib.avc_gated_recurrence_workspace(dt, s.T, s.B, s.H, s.dirs);
  const Tensor ws = scratch(gates, bytes);
  const On on(gates);
  done(lib.avc_gated_recurrence_forward(dt, s.T, s.B, s.H, s.dirs, g.p(), g.ld, ptr<float>(h0), ptr<int>(lengths), y.data_ptr(),
                                        s.D() * s.H, ptr<float>(hT), ptr<float>(states), ptr(ws), bytes, on.stream),
       "avc_gated_recurrence_forward");
  return {y, hT, states};
}

struct GatedRecurrence : torch::autograd::Function<GatedRecurrence> {
  static variable_list forward(AutogradContext* ctx, const Tensor& gates, const optional<Tensor>& h0,
                               const optional<Tensor>& lengths, long T, long B, long H, long dirs) {
    const Tensor len = lengths.value_or(Tensor());
    auto [y, hT, states] = recurrence_forward(gates, h0.value_or(Tensor()), len, {T, B, H, dirs}, true);
    ctx->save_for_backward({gates, len, states});
    ctx->saved_data["shape"] = std::vector<int64_t>{T, B, H, dirs, h0 && h0->requires_grad()};
    ctx->set_materialize_grads(false);
    return {y, hT};
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) { return once(d, grads(ctx, d)); }
  static variable_list grads(AutogradContext* ctx, const variable_list& d) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &gates = saved[0], &lengths = saved[1], &states = saved[2];
    const auto v = ctx->saved_data["shape"].toIntVector();
    const RecShape s{v[0], v[1], v[2], v[3]};
    const at::NoGradGuard plain;
    const int dt = dtype_of(gates);
    const Rows g(gates, s.too_far());
    const Rows dy(d[0].defined() ? d[0] : at::zeros({s.T * s.B, s.D() * s.H}, gates.options()), s.too_far());
    const Tensor dhT = d[1].defined() ? dense(d[1]) : Tensor();
    Tensor dg = at::empty({s.T * s.B, s.D() * 3 * s.H}, gates.options()), dh0;
    if (v[4]) dh0 = at::empty({s.D(), s.B, s.H}, states.options());
    const size_t bytes = lib.avc_gated_recurrence_workspace(dt, s.T, s.B, s.H, s.dirs);
    const Tensor ws = scratch(gates, bytes);
    {
      const On on(gates);
      done(lib.avc_gated_recurrence_backward(dt, s.T, s.B, s.H, s.dirs, g.p(), g.ld, ptr<int>(lengths), ptr<float>(states),
                                             dy.p(), dy.ld, ptr<float>(dhT), dg.data_ptr(), s.D() * 3 * s.H, ptr<float>(dh0),
                                             ptr(ws), bytes, on.stream),
           "avc_gated_recurrence_backward");
    }
    return {dg, dh0, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> gated_recurrence(const Tensor& gates, long T, long B, optional<Tensor> h0, optional<Tensor> lengths,
                                            long dirs) {
  check_seen("gated_recurrence", gates, h0);
  check_data(gates, "gates");
  TORCH_CHECK_VALUE(dirs >= 1 && dirs <= 3, "dirs is 1 (forward), 2 (reverse) or 3 (both)");
  const long D = dirs == 3 ? 2 : 1, most = 1L << 30;
  TORCH_CHECK_VALUE(T >= 0 && B >= 0 && T <= most && B <= most && gates.dim() == 2 && gates.size(0) == T * B &&
                        gates.size(1) > 0 && gates.size(1) % (3 * D) == 0,
                    "gates must be [T*B = ", T, " * ", B, "][", 3 * D, " * H], got ", gates.sizes());
  const long H = gates.size(1) / (3 * D);
  TORCH_CHECK_VALUE(H <= 1L << 28, "H = ", H, " is too large");
  if (h0) {
    check_type(*h0, "h0", gates, at::kFloat, at::kFloat);
    TORCH_CHECK_VALUE(h0->dim() == 3 && h0->size(0) == D && h0->size(1) == B && h0->size(2) == H, "h0 must be [", D, ", ", B,
                      ", ", H, "], got ", h0->sizes());
    h0 = dense(*h0);
  }
  Tensor len;
  if (lengths) {
    check_type(*lengths, "lengths", gates, at::kInt, at::kLong);
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == B, "lengths must be [", B, "], got ", lengths->sizes());
    len = lengths->scalar_type() == at::kLong ? lengths->clamp(0, T).to(at::kInt) : lengths->contiguous();
  }
  if (T * B == 0) {  // no frame: the state passes through
    Tensor hT = h0 ? h0->clone() : at::zeros({D, B, H}, gates.options().dtype(at::kFloat));
    return {gates.slice(1, 0, D * H).contiguous(), hT};
  }
  if (wants_grad(gates, h0)) {
    auto out = GatedRecurrence::apply(gates, h0, len.defined() ? optional<Tensor>(len) : std::nullopt, T, B, H, dirs);
    return {out[0], out[1]};
  }
  auto [y, hT, states] = recurrence_forward(gates, h0.value_or(Tensor()), len, {T, B, H, dirs}, false);
  return {y, hT};
}

// Whether a's (contiguous) bytes and the span of b's meet.
bool overlap(const Tensor& a, const Tensor& b) {
  if (!a.numel() || !b.numel()) return false;
  long span = 1;
  for (int i = 0; i < b.dim(); ++i) span += (b.size(i) - 1) * b.stride(i);
  const char *pa = static_cast<const char*>(a.data_ptr()), *pb = static_cast<const char*>(b.data_ptr());
  return pa < pb + span * b.element_size() && pb < pa + a.numel() * a.element_size();
}

std::tuple<Tensor, Tensor> gated_recurrence_step(const Tensor& gates, const Tensor& state, optional<Tensor> out_state) {
  check_seen("gated_recurrence_step", gates, state, out_state);
  check_data(gates, "gates");
  check_type(state, "state", gates, at::kFloat, at::kFloat);
  TORCH_CHECK_VALUE(gates.dim() == 2 && gates.size(1) > 0 && gates.size(1) % 3 == 0, "gates must be [B][3 * H], got ",
                    gates.sizes());
  TORCH_CHECK(!wants_grad(gates, state), "gated_recurrence_step builds no autograd graph; use gated_recurrence");
  const long B = gates.size(0), H = gates.size(1) / 3;
  TORCH_CHECK_VALUE(B <= 1L << 30 && H <= 1L << 28, "gates of ", gates.sizes(), " are too large");
  auto fits = [&](const Tensor& t) { return t.dim() == 2 && t.size(0) == B && t.size(1) == H; };
  TORCH_CHECK_VALUE(fits(state), "state must be [", B, ", ", H, "], got ", state.sizes());
  Tensor out;
  if (out_state) {
    out = *out_state;
    check_type(out, "out_state", gates, at::kFloat, at::kFloat);
    TORCH_CHECK(!wants_grad(out), "out_state is written in place, so it cannot require a gradient");
    TORCH_CHECK_VALUE(fits(out) && out.is_contiguous() && !out.is_neg(), "out_state must be a contiguous [", B, ", ", H, "]");
    TORCH_CHECK_VALUE(!overlap(out, state) || (out.data_ptr() == state.data_ptr() && state.is_contiguous()),
                      "out_state overlaps state without being it");
    TORCH_CHECK_VALUE(!overlap(out, gates), "out_state overlaps gates");
    out.unsafeGetTensorImpl()->bump_version();
  } else {
    out = at::empty({B, H}, state.options());
  }
  Tensor y = at::empty({B, H}, gates.options());
  if (B) {
    const Rows g(gates);
    const Tensor h = dense(state);
    const On on(gates);
    done(lib.avc_gated_recurrence_step(dtype_of(gates), B, H, g.p(), g.ld, ptr<float>(h), ptr<float>(out), y.data_ptr(), H,
                                       on.stream),
         "avc_gated_recurrence_step");
  }
  return {y, out};
}

// ---- log-probabilities of given classes -------------------------------------------------------------
struct LogProbs {
  Tensor logp, entropy, top_logp, top_ids, stats;
};

LogProbs log_probs_forward(const Tensor& logits, const Tensor& tokens, long top, long ignore, bool keep) {
  const int dt = dtype_of(logits);
  const long N = logits.size(0), V = logits.size(1);
  const Rows z(logits);
  const auto f32 = logits.options().dtype(at::kFloat);
  LogProbs o{at::empty({N}, f32), at::empty({N}, f32), Tensor(), Tensor(), Tensor()};
  if (top || !keep) o.top_logp = at::empty({N, top}, f32), o.top_ids = at::empty({N, top}, f32.dtype(at::kLong));
  if (keep) o.stats = at::empty({N, 3}, f32);
  if (N) {
    const size_t bytes = lib.avc_token_log_probs_workspace(dt, N, V, top);
    const Tensor ws = scratch(logits, bytes);
    const On on(logits);
    done(lib.avc_token_log_probs_forward(dt, N, V, z.p(), z.ld, ptr<long long>(tokens), ignore, top, ptr<float>(o.logp),
                                         ptr<float>(o.entropy), ptr<float>(o.stats), ptr<float>(o.top_logp),
                                         ptr<long long>(o.top_ids), ptr(ws), bytes, on.stream),
         "avc_token_log_probs_forward");
  }
  return o;
}

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, long top, long ignore) {
    LogProbs o = log_probs_forward(logits, tokens, top, ignore, true);
    ctx->save_for_backward({logits, tokens, o.stats});
    ctx->saved_data["ignore"] = ignore;
    ctx->set_materialize_grads(false);
    if (!top) return {o.logp, o.entropy};
    ctx->mark_non_differentiable({o.top_logp, o.top_ids});
    return {o.logp, o.entropy, o.top_logp, o.top_ids};
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) { return once(d, grads(ctx, d)); }
  static variable_list grads(AutogradContext* ctx, const variable_list& d) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &tokens = saved[1], &stats = saved[2];
    const at::NoGradGuard plain;
    const long N = logits.size(0), V = logits.size(1);
    const Rows z(logits);
    Tensor dz = at::empty({N, V}, logits.options());
    const Tensor dl = d[0].defined() ? dense(d[0]) : Tensor(), de = d[1].defined() ? dense(d[1]) : Tensor();
    if (N) {
      const On on(logits);
      done(lib.avc_token_log_probs_backward(dtype_of(logits), N, V, z.p(), z.ld, ptr<long long>(tokens),
                                            ctx->saved_data["ignore"].toInt(), ptr<float>(stats), ptr<float>(dl),
                                            ptr<float>(de), dz.data_ptr(), V, on.stream),
           "avc_token_log_probs_backward");
    }
    return {dz, Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_log_probs(Tensor logits, Tensor tokens, long top, long ignore) {
  check_seen("token_log_probs", logits);
  check_data(logits, "logits");
  check_type(tokens, "tokens", logits, at::kLong, at::kInt);
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.sizes().slice(0, logits.dim() - 1) == tokens.sizes(),
                    "logits [..., V >= 1] and tokens [...] must agree, got ", logits.sizes(), " and ", tokens.sizes());
  const long V = logits.size(-1), most = std::min<long>(32, V);
  TORCH_CHECK_VALUE(top >= 0 && top <= most, "top must be 0 .. ", most, ", got ", top);
  if (tokens.scalar_type() != at::kLong) tokens = tokens.to(at::kLong);
  if (!tokens.is_contiguous()) tokens = tokens.contiguous();
  const auto lead = tokens.sizes().vec();
  const bool flat = logits.dim() == 2;
  if (!flat) logits = logits.reshape({tokens.numel(), V}), tokens = tokens.reshape({-1});
  Tensor logp, entropy, tl, ti;
  if (wants_grad(logits)) {
    auto o = TokenLogProbs::apply(logits, tokens, top, ignore);
    logp = o[0], entropy = o[1];
    if (top) {
      tl = o[2], ti = o[3];
    } else {
      tl = at::empty({tokens.numel(), 0}, logp.options()), ti = at::empty({tokens.numel(), 0}, tokens.options());
    }
  } else {
    LogProbs o = log_probs_forward(logits, tokens, top, ignore, false);
    logp = o.logp, entropy = o.entropy, tl = o.top_logp, ti = o.top_ids;
  }
  if (!flat) {
    auto with_top = lead;
    with_top.push_back(top);
    logp = logp.view(lead), entropy = entropy.view(lead), tl = tl.view(with_top), ti = ti.view(with_top);
  }
  return {logp, entropy, tl, ti};
}

// ---- counter-based dropout ----------------------------------------------------------------------------
Tensor drop(const Tensor& given, const Tensor& added, double p, const Tensor& rng, long layer) {
  const Tensor x = as_stored(given), residual = added.defined() ? as_stored(added) : added;
  Tensor y = at::empty(x.sizes(), x.options());
  if (!x.numel()) return y;
  long n = 1, c = x.numel(), ldx = c, ldr = c;
  Tensor xs = x, rs = residual;
  if (!x.is_contiguous() || (residual.defined() && !residual.is_contiguous())) {
    c = x.size(-1), n = x.numel() / c;
    const Rows rx(x.dim() == 2 ? x : x.reshape({n, c}));
    xs = rx.t, ldx = rx.ld;
    if (residual.defined()) {
      const Rows rr(residual.dim() == 2 ? residual : residual.reshape({n, c}));
      rs = rr.t, ldr = rr.ld;
    }
  }
  const On on(x);
  done(lib.avc_dropout(dtype_of(x), n, c, xs.data_ptr(), ldx, ptr(rs), ldr, p, ptr<long long>(rng), (unsigned)layer, y.data_ptr(),
                       c, on.stream),
       "avc_dropout");
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& residual, const Tensor& rng, double p,
                        long layer) {
    ctx->save_for_backward({rng});
    ctx->saved_data["p"] = p;
    ctx->saved_data["layer"] = layer;
    ctx->saved_data["needs"] = (x.requires_grad() ? 1 : 0) | (residual && residual->requires_grad() ? 2 : 0);
    return drop(x, residual.value_or(Tensor()), p, rng, layer);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const long needs = ctx->saved_data["needs"].toInt();
    // (the residual's gradient is the incoming one itself, which keeps its own history)
    return {needs & 1 ? once(d, {grad_x(ctx, d[0])}, true)[0] : Tensor(), needs & 2 ? d[0] : Tensor(), Tensor(), Tensor(), Tensor()};
  }
  static Tensor grad_x(AutogradContext* ctx, const Tensor& dy) {
    // (rng is saved, so that changing it in place before the backward is an error and not another mask)
    const Tensor rng = ctx->get_saved_variables()[0];
    const at::NoGradGuard plain;
    return drop(dy, Tensor(), ctx->saved_data["p"].toDouble(), rng, ctx->saved_data["layer"].toInt());
  }
};

Tensor dropout(const Tensor& x, double p, const Tensor& rng, optional<Tensor> residual, long layer) {
  check_seen("dropout", x, residual);
  check_data(x, "x");
  check_type(rng, "rng", x, at::kLong, at::kLong);
  TORCH_CHECK_VALUE(p >= 0.0 && p < 1.0, "p must be 0 <= p < 1, got ", p);
  TORCH_CHECK_VALUE(layer >= 0 && layer < 1L << 32, "layer must be 0 .. 2^32 - 1, got ", layer);
  TORCH_CHECK_VALUE(rng.dim() == 1 && rng.size(0) == 2 && rng.is_contiguous(), "rng must be a contiguous [2], got ", rng.sizes());
  if (residual) {
    check_type(*residual, "residual", x, x.scalar_type(), x.scalar_type());
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "residual must have x's shape ", x.sizes(), ", got ", residual->sizes());
  }
  if (wants_grad(x, residual)) return Dropout::apply(x, residual, rng, p, layer);
  return drop(x, residual.value_or(Tensor()), p, rng, layer);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const HipLibraryError& e) {
      PyErr_SetString(hip_library_error ? hip_library_error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("gated_recurrence", &gated_recurrence);
  m.def("gated_recurrence_step", &gated_recurrence_step);
  m.def("token_log_probs", &token_log_probs);
  m.def("dropout", &dropout);
}
