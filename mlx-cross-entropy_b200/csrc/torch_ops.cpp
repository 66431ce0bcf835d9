// torch operators of the losses on log-probabilities: the C ABI's forward and
// backward calls as autograd functions.
//
// The small calls of these losses take 15 us on the GPU; the same functions
// written in Python (an autograd.Function and ctypes) took 110 to 150 us of the
// host, half of it Python on the backward thread.  Arguments are checked in
// Python (losses.py), where tensors are made contiguous; these operators
// allocate, call the library and keep what the backward pass reads.  The
// library's functions come as addresses (bind), so that whichever build of it is
// loaded is the one that is called.
#include <ATen/ATen.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <unordered_set>

#include "cce_b200.h"

// Read from the file before it is loaded: another torch would fail on a symbol.
__attribute__((used)) static const char built_for[] = CCE_BUILT_FOR;

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ---- the library ----

#define CCE_FUNCTIONS(X)                                                                                        \
  X(cce_last_error)                                                                                             \
  X(cce_token_loss_workspace_bytes)                                                                             \
  X(cce_policy_loss_forward)                                                                                    \
  X(cce_policy_loss_backward)                                                                                   \
  X(cce_preference_loss_forward)                                                                                \
  X(cce_preference_loss_backward)                                                                               \
  X(cce_logp_saved_bytes)                                                                                       \
  X(cce_logp_forward_workspace_bytes)                                                                           \
  X(cce_logp_backward_workspace_bytes)                                                                          \
  X(cce_logp_forward)                                                                                           \
  X(cce_logp_backward)                                                                                          \
  X(cce_distill_saved_bytes)                                                                                    \
  X(cce_distill_forward_workspace_bytes)                                                                        \
  X(cce_distill_backward_workspace_bytes)                                                                       \
  X(cce_distill_forward)                                                                                        \
  X(cce_distill_backward)

struct Library {
#define X(name) decltype(&::name) name = nullptr;
  CCE_FUNCTIONS(X)
#undef X
} lib;

// The functions' addresses, in the order of `functions()`.
void bind_library(const std::vector<int64_t>& addresses) {
  Library l;
  size_t i = 0;
#define X(name)                                                                           \
  TORCH_CHECK(i < addresses.size() && addresses[i] != 0, "bind: no address for " #name); \
  l.name = reinterpret_cast<decltype(l.name)>(addresses[i++]);
  CCE_FUNCTIONS(X)
#undef X
  lib = l;
}

std::vector<std::string> functions() {
#define X(name) #name,
  return {CCE_FUNCTIONS(X)};
#undef X
}

// A library status as the Python package raises it.
void check(int rc, const char* what) {
  if (rc == CCE_OK) return;
  const char* msg = lib.cce_last_error();
  const bool value = rc == CCE_ERR_SHAPE || rc == CCE_ERR_DTYPE || rc == CCE_ERR_ARG || rc == CCE_ERR_ALIGN;
  TORCH_CHECK_VALUE(!value, "[", what, "] ", msg);
  TORCH_CHECK(false, "[", what, "] ", msg, " (status ", rc, ")");
}

int code(at::ScalarType t) { return t == at::kFloat ? CCE_F32 : t == at::kHalf ? CCE_F16 : CCE_BF16; }

template <typename T = void>
T* ptr(const OptTensor& t) {
  return t && t->defined() ? static_cast<T*>(t->data_ptr()) : nullptr;
}
template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
Tensor keep(const OptTensor& t) { return t ? *t : Tensor(); }

size_t pad(size_t n) { return (n + 255) & ~size_t(255); }

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({static_cast<int64_t>(n + 256)}, like.options().dtype(at::kByte));
}
Tensor f32(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }

// The operators read and write memory that torch's tracers do not see: a trace of one
// would hold its buffers and none of its kernels.
void plain(const Tensor& t) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  TORCH_CHECK(!t.key_set().has(c10::DispatchKey::Python) && !Modes::get_mode(Key::PROXY) && !Modes::get_mode(Key::FAKE),
              "the losses on log-probabilities run on plain CUDA tensors and cannot be traced or given tensor "
              "subclasses: call them outside of the traced function (torch.compiler.disable)");
}

Tensor upstream(const Tensor& g) {
  TORCH_CHECK(g.has_storage(), "the losses on log-probabilities take one gradient at a time (not is_grads_batched)");
  return g.to(at::kFloat).contiguous();
}

// Gradients for a backward pass that is itself recorded: a second derivative is
// an error, not a wrong zero.
variable_list first_order(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "the losses on log-probabilities are differentiable once", static_cast<int64_t>(grads.size()));
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  return (*error)(std::move(grads));
}

// A backward pass that is being captured must not add into a leaf whose gradient
// node an eager graph made on the default stream and still holds (a loss that was
// not deleted): the engine would wait on that stream, which no capture may, and
// the process would end.  Every such node below is looked for, once per capture.
void check_capture() {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const c10::Stream eager = c10::cuda::getDefaultCUDAStream().unwrap();
  std::vector<torch::autograd::Node*> todo{torch::autograd::get_current_node().get()};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!todo.empty()) {
    torch::autograd::Node* n = todo.back();
    todo.pop_back();
    if (n == nullptr || !seen.insert(n).second) continue;
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(n)) {
      const auto at = n->stream();
      TORCH_CHECK(!at || *at != eager,
                  "a backward pass is captured into a CUDA graph while an eager graph of the same leaves, made on the "
                  "default stream, is alive: delete its loss first (or run it on another stream)");
    }
    for (const auto& edge : n->next_edges()) todo.push_back(edge.function.get());
  }
}

// ---- losses on given log-probabilities ----

struct PolicyArgs {
  OptTensor old, ref;
  Tensor adv;
  OptTensor mask, cu;
  int64_t S;
  CcePolicyParams params;
};

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logp, const PolicyArgs& a) {
    c10::cuda::CUDAGuard guard(logp.device());
    const int64_t N = logp.numel();
    Tensor loss = a.params.reduction == CCE_REDUCE_NONE ? f32(logp.sizes(), logp) : f32({}, logp);
    Tensor stats = f32({2}, logp);
    const size_t at_weight = pad(4 * N), at_ws = at_weight + pad(4 * (1 + a.S));
    const size_t ws = lib.cce_token_loss_workspace_bytes(N, a.S);
    Tensor state = bytes(at_ws + ws, logp);  // coefficients, weights; the call's workspace behind them
    char* p = ptr<char>(state);
    check(lib.cce_policy_loss_forward(ptr(logp), ptr(a.old), ptr(a.ref), code(logp.scalar_type()), ptr<float>(a.adv),
                                      ptr<uint8_t>(a.mask), ptr<int32_t>(a.cu), N, a.S, &a.params, ptr<float>(loss),
                                      ptr<float>(stats), (float*)p, (float*)(p + at_weight), p + at_ws, ws, stream()),
          "cce_policy_loss_forward");
    ctx->save_for_backward({state, keep(a.cu)});
    ctx->saved_data["m"] = std::vector<int64_t>{a.params.reduction, a.S, static_cast<int64_t>(logp.scalar_type())};
    ctx->saved_data["shape"] = logp.sizes().vec();
    ctx->mark_non_differentiable({stats});
    ctx->set_materialize_grads(false);
    return {loss, stats};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const Tensor& state = saved[0];
    c10::cuda::CUDAGuard guard(state.device());
    check_capture();
    const auto type = static_cast<at::ScalarType>(m[2]);
    Tensor grad = at::empty(shape, state.options().dtype(type));
    const int64_t N = grad.numel();
    const Tensor g = upstream(grads[0]);
    char* p = ptr<char>(state);
    check(lib.cce_policy_loss_backward((float*)p, (float*)(p + pad(4 * N)), ptr<float>(g), (int)m[0],
                                       ptr<int32_t>(saved[1]), N, m[1], code(type), ptr(grad), stream()),
          "cce_policy_loss_backward");
    return first_order({grad, Tensor()});
  }
};

struct PreferenceArgs {
  OptTensor ref, ref_sums, mask, cu;
  int64_t pairs;
  CcePreferenceParams params;
};

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logp, const PreferenceArgs& a) {
    c10::cuda::CUDAGuard guard(logp.device());
    const int64_t N = logp.numel(), pairs = a.pairs;
    Tensor loss = a.params.reduction == CCE_REDUCE_NONE ? f32({pairs}, logp) : f32({}, logp);
    Tensor rewards = f32({2 * pairs}, logp);
    const size_t at_ws = pad(8 * pairs);
    const size_t ws = lib.cce_token_loss_workspace_bytes(N, 2 * pairs);
    Tensor state = bytes(at_ws + ws, logp);
    char* p = ptr<char>(state);
    check(lib.cce_preference_loss_forward(ptr(logp), ptr(a.ref), code(logp.scalar_type()), ptr<float>(a.ref_sums),
                                          ptr<uint8_t>(a.mask), ptr<int32_t>(a.cu), N, pairs, &a.params,
                                          ptr<float>(loss), ptr<float>(rewards), (float*)p, p + at_ws, ws, stream()),
          "cce_preference_loss_forward");
    ctx->save_for_backward({state, keep(a.mask), keep(a.cu)});
    ctx->saved_data["m"] = std::vector<int64_t>{a.params.reduction, pairs, static_cast<int64_t>(logp.scalar_type())};
    ctx->saved_data["shape"] = logp.sizes().vec();
    ctx->mark_non_differentiable({rewards});
    ctx->set_materialize_grads(false);
    return {loss, rewards};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    c10::cuda::CUDAGuard guard(saved[0].device());
    check_capture();
    const auto type = static_cast<at::ScalarType>(m[2]);
    Tensor grad = at::empty(shape, saved[0].options().dtype(type));
    const Tensor g = upstream(grads[0]);
    check(lib.cce_preference_loss_backward(ptr<float>(saved[0]), ptr<float>(g), (int)m[0], ptr<uint8_t>(saved[1]),
                                           ptr<int32_t>(saved[2]), grad.numel(), m[1], code(type), ptr(grad), stream()),
          "cce_preference_loss_backward");
    return first_order({grad, Tensor()});
  }
};

// ---- losses of a head ----

struct HeadArgs {
  Tensor targets;  // [N] int32 or int64, contiguous
  int64_t ignore_index;
  bool has_ignore;
};

int bias_code(const OptTensor& bias) { return bias && bias->defined() ? code(bias->scalar_type()) : 0; }

struct LogpSizes {
  size_t saved, ws;
  LogpSizes(const Tensor& e, const Tensor& c)
      : saved(pad(lib.cce_logp_saved_bytes(e.size(0), e.size(1), c.size(0), code(e.scalar_type())))),
        ws(pad(lib.cce_logp_forward_workspace_bytes(e.size(0), e.size(1), c.size(0), code(e.scalar_type())))) {}
};

void logp_forward(const Tensor& e, const Tensor& c, const OptTensor& bias, const HeadArgs& h, float* logp, uint8_t* mask,
                  void* saved, void* ws, const LogpSizes& z) {
  check(lib.cce_logp_forward(ptr(e), ptr(c), ptr(bias), bias_code(bias), ptr(h.targets), (int)h.targets.element_size(),
                             h.ignore_index, h.has_ignore, e.size(0), e.size(1), c.size(0), code(e.scalar_type()), logp,
                             mask, saved, z.saved, ws, z.ws, stream()),
        "cce_logp_forward");
}

// Outputs of a backward call of the head, and which of them are asked for.
struct HeadGrads {
  Tensor e, c, bias;
  int flags = 0;
  HeadGrads(AutogradContext* ctx, int64_t N, at::ScalarType type, const Tensor& w, const Tensor& b) {
    if (ctx->needs_input_grad(0)) {
      e = at::empty({N, w.size(1)}, w.options().dtype(type));
      flags |= CCE_NEED_DE;
    }
    if (ctx->needs_input_grad(1)) {
      c = at::empty_like(w);
      flags |= CCE_NEED_DC;
    }
    if (b.defined() && ctx->needs_input_grad(2)) {
      bias = f32({w.size(0)}, w);
      flags |= CCE_NEED_DBIAS;
    }
  }
  variable_list list(const Tensor& b) {
    if (bias.defined()) bias = bias.to(b.scalar_type());
    return first_order({e, c, bias, Tensor()});
  }
};

// Gradients of the head for d logp, which `d(address)` puts in front of the workspace.
template <typename F>
variable_list logp_backward(AutogradContext* ctx, const Tensor& c, const Tensor& bias, void* saved, size_t saved_bytes,
                            int64_t N, at::ScalarType type, F d) {
  HeadGrads g(ctx, N, type, c, bias);
  const int64_t V = c.size(0), D = c.size(1);
  const size_t at_ws = pad(4 * N), ws_bytes = lib.cce_logp_backward_workspace_bytes(N, D, V, code(type), g.flags);
  Tensor ws = bytes(at_ws + ws_bytes, c);
  char* w = ptr<char>(ws);
  const float* up = d((float*)w);
  check(lib.cce_logp_backward(ptr(c), ptr(bias), bias_code(bias), up, N, D, V, code(type), g.flags, saved, saved_bytes,
                              ptr(g.e), ptr(g.c), ptr<float>(g.bias), w + at_ws, ws_bytes, stream()),
        "cce_logp_backward");
  return g.list(bias);
}

struct LogProbs : torch::autograd::Function<LogProbs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& e, const Tensor& c, const OptTensor& bias,
                        const HeadArgs& h) {
    c10::cuda::CUDAGuard guard(e.device());
    const int64_t N = e.size(0);
    const LogpSizes z(e, c);
    Tensor logp = f32({N}, e), saved = bytes(z.saved, e), ws = bytes(pad(N) + z.ws, e);
    uint8_t* w = ptr<uint8_t>(ws);
    logp_forward(e, c, bias, h, ptr<float>(logp), w, ptr(saved), w + pad(N), z);
    ctx->save_for_backward({c, keep(bias), saved});
    ctx->saved_data["m"] = std::vector<int64_t>{N, static_cast<int64_t>(e.scalar_type())};
    return logp;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    c10::cuda::CUDAGuard guard(saved[0].device());
    check_capture();
    const Tensor g = upstream(grads[0]);
    return logp_backward(ctx, saved[0], saved[1], ptr(saved[2]), saved[2].numel(), m[0],
                         static_cast<at::ScalarType>(m[1]), [&](float*) { return ptr<const float>(g); });
  }
};

struct LinearPolicyLoss : torch::autograd::Function<LinearPolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& e, const Tensor& c, const OptTensor& bias,
                               const std::pair<HeadArgs, PolicyArgs>& args) {
    const PolicyArgs& a = args.second;
    c10::cuda::CUDAGuard guard(e.device());
    const int64_t N = e.size(0);
    const LogpSizes z(e, c);
    Tensor loss = a.params.reduction == CCE_REDUCE_NONE ? f32({N}, e) : f32({}, e);
    Tensor stats = f32({2}, e);
    const size_t at_weight = pad(4 * N), at_saved = at_weight + pad(4 * (1 + a.S));
    Tensor state = bytes(at_saved + z.saved, e);
    const size_t loss_ws = lib.cce_token_loss_workspace_bytes(N, a.S);
    const size_t at_mask = pad(4 * N), at_ws = at_mask + pad(N);
    Tensor ws = bytes(at_ws + std::max(z.ws, loss_ws), e);
    char *p = ptr<char>(state), *w = ptr<char>(ws);
    logp_forward(e, c, bias, args.first, (float*)w, (uint8_t*)w + at_mask, p + at_saved, w + at_ws, z);
    // (in stream order behind the log-probabilities, so their workspace is free again)
    check(lib.cce_policy_loss_forward(w, ptr(a.old), ptr(a.ref), CCE_F32, ptr<float>(a.adv), (uint8_t*)w + at_mask,
                                      ptr<int32_t>(a.cu), N, a.S, &a.params, ptr<float>(loss), ptr<float>(stats),
                                      (float*)p, (float*)(p + at_weight), w + at_ws, loss_ws, stream()),
          "cce_policy_loss_forward");
    ctx->save_for_backward({c, keep(bias), state, keep(a.cu)});
    ctx->saved_data["m"] =
        std::vector<int64_t>{N, static_cast<int64_t>(e.scalar_type()), a.params.reduction, a.S, static_cast<int64_t>(z.saved)};
    ctx->mark_non_differentiable({stats});
    ctx->set_materialize_grads(false);
    return {loss, stats};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    c10::cuda::CUDAGuard guard(saved[0].device());
    check_capture();
    const Tensor g = upstream(grads[0]);
    const int64_t N = m[0];
    char* p = ptr<char>(saved[2]);
    const size_t at_weight = pad(4 * N), at_saved = at_weight + pad(4 * (1 + m[3]));
    return logp_backward(ctx, saved[0], saved[1], p + at_saved, m[4], N, static_cast<at::ScalarType>(m[1]), [&](float* d) {
      check(lib.cce_policy_loss_backward((float*)p, (float*)(p + at_weight), ptr<float>(g), (int)m[2],
                                         ptr<int32_t>(saved[3]), N, m[3], CCE_F32, d, stream()),
            "cce_policy_loss_backward");
      return (const float*)d;
    });
  }
};

struct LinearPreferenceLoss : torch::autograd::Function<LinearPreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& e, const Tensor& c, const OptTensor& bias,
                               const std::pair<HeadArgs, PreferenceArgs>& args) {
    const PreferenceArgs& a = args.second;
    c10::cuda::CUDAGuard guard(e.device());
    const int64_t N = e.size(0), pairs = a.pairs;
    const LogpSizes z(e, c);
    Tensor loss = a.params.reduction == CCE_REDUCE_NONE ? f32({pairs}, e) : f32({}, e);
    Tensor rewards = f32({2 * pairs}, e);
    const size_t at_mask = pad(8 * pairs), at_saved = at_mask + pad(N);
    Tensor state = bytes(at_saved + z.saved, e);
    const size_t loss_ws = lib.cce_token_loss_workspace_bytes(N, 2 * pairs);
    const size_t at_ws = pad(4 * N);
    Tensor ws = bytes(at_ws + std::max(z.ws, loss_ws), e);
    char *p = ptr<char>(state), *w = ptr<char>(ws);
    logp_forward(e, c, bias, args.first, (float*)w, (uint8_t*)p + at_mask, p + at_saved, w + at_ws, z);
    check(lib.cce_preference_loss_forward(w, ptr(a.ref), CCE_F32, ptr<float>(a.ref_sums), (uint8_t*)p + at_mask,
                                          ptr<int32_t>(a.cu), N, pairs, &a.params, ptr<float>(loss),
                                          ptr<float>(rewards), (float*)p, w + at_ws, loss_ws, stream()),
          "cce_preference_loss_forward");
    ctx->save_for_backward({c, keep(bias), state, keep(a.cu)});
    ctx->saved_data["m"] =
        std::vector<int64_t>{N, static_cast<int64_t>(e.scalar_type()), a.params.reduction, pairs, static_cast<int64_t>(z.saved)};
    ctx->mark_non_differentiable({rewards});
    ctx->set_materialize_grads(false);
    return {loss, rewards};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    c10::cuda::CUDAGuard guard(saved[0].device());
    check_capture();
    const Tensor g = upstream(grads[0]);
    const int64_t N = m[0];
    char* p = ptr<char>(saved[2]);
    const size_t at_mask = pad(8 * m[3]), at_saved = at_mask + pad(N);
    return logp_backward(ctx, saved[0], saved[1], p + at_saved, m[4], N, static_cast<at::ScalarType>(m[1]), [&](float* d) {
      check(lib.cce_preference_loss_backward((float*)p, ptr<float>(g), (int)m[2], (uint8_t*)p + at_mask,
                                             ptr<int32_t>(saved[3]), N, m[3], CCE_F32, d, stream()),
            "cce_preference_loss_backward");
      return (const float*)d;
    });
  }
};

struct DistillArgs {
  Tensor ids, teacher;  // [N, K]
  OptTensor mask;
  CceDistillParams params;
};

struct Distillation : torch::autograd::Function<Distillation> {
  static Tensor forward(AutogradContext* ctx, const Tensor& e, const Tensor& c, const OptTensor& bias,
                        const DistillArgs& a) {
    c10::cuda::CUDAGuard guard(e.device());
    const int64_t N = e.size(0), D = e.size(1), V = c.size(0), K = a.ids.size(1);
    const int dt = code(e.scalar_type());
    Tensor loss = a.params.reduction == CCE_REDUCE_NONE ? f32({N}, e) : f32({}, e);
    const size_t saved_bytes = lib.cce_distill_saved_bytes(N, D, V, K, dt);
    const size_t ws_bytes = lib.cce_distill_forward_workspace_bytes(N, D, V, K, dt);
    Tensor saved = bytes(saved_bytes, e), ws = bytes(ws_bytes, e);
    check(lib.cce_distill_forward(ptr(e), ptr(c), ptr(bias), bias_code(bias), ptr(a.ids), (int)a.ids.element_size(),
                                  ptr<float>(a.teacher), ptr<uint8_t>(a.mask), N, D, V, K, dt, &a.params,
                                  ptr<float>(loss), ptr(saved), saved_bytes, ptr(ws), ws_bytes, stream()),
          "cce_distill_forward");
    ctx->save_for_backward({c, keep(bias), saved});
    ctx->saved_data["m"] = std::vector<int64_t>{N, static_cast<int64_t>(e.scalar_type()), K, a.params.tail,
                                                a.params.reduction, static_cast<int64_t>(saved_bytes)};
    ctx->saved_data["T"] = a.params.temperature;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    const Tensor &c = saved[0], &bias = saved[1];
    c10::cuda::CUDAGuard guard(c.device());
    check_capture();
    const auto type = static_cast<at::ScalarType>(m[1]);
    const CceDistillParams params{ctx->saved_data["T"].toDouble(), (int32_t)m[3], (int32_t)m[4]};
    const Tensor up = upstream(grads[0]);
    HeadGrads g(ctx, m[0], type, c, bias);
    const int64_t V = c.size(0), D = c.size(1);
    const size_t ws_bytes = lib.cce_distill_backward_workspace_bytes(m[0], D, V, code(type), g.flags);
    Tensor ws = bytes(ws_bytes, c);
    check(lib.cce_distill_backward(ptr(c), ptr(bias), bias_code(bias), ptr<float>(up), m[0], D, V, m[2], code(type),
                                   &params, g.flags, ptr(saved[2]), m[5], ptr(g.e), ptr(g.c), ptr<float>(g.bias),
                                   ptr(ws), ws_bytes, stream()),
          "cce_distill_backward");
    return g.list(bias);
  }
};

// ---- operators ----

CcePolicyParams policy_params(at::ArrayRef<double> x, int64_t reduction, bool per_token) {
  TORCH_CHECK_VALUE(x.size() == 4, "policy parameters: clip_low, clip_high, dual_clip, kl_coef");
  return CcePolicyParams{x[0], x[1], x[2], x[3], (int32_t)reduction, per_token};
}

CcePreferenceParams preference_params(at::ArrayRef<double> x, int64_t kind, int64_t reduction, bool by_length) {
  TORCH_CHECK_VALUE(x.size() == 3, "preference parameters: beta, margin, label_smoothing");
  return CcePreferenceParams{x[0], x[1], x[2], (int32_t)kind, (int32_t)reduction, by_length};
}

std::tuple<Tensor, Tensor> policy_loss(const Tensor& logp, const OptTensor& old, const OptTensor& ref, const Tensor& adv,
                                       const OptTensor& mask, const OptTensor& cu, int64_t S, at::ArrayRef<double> params,
                                       int64_t reduction, bool per_token) {
  plain(logp);
  auto out = PolicyLoss::apply(logp, PolicyArgs{old, ref, adv, mask, cu, S, policy_params(params, reduction, per_token)});
  return {out[0], out[1]};
}

std::tuple<Tensor, Tensor> preference_loss(const Tensor& logp, const OptTensor& ref, const OptTensor& ref_sums,
                                           const OptTensor& mask, const OptTensor& cu, int64_t pairs,
                                           at::ArrayRef<double> params, int64_t kind, int64_t reduction, bool by_length) {
  plain(logp);
  auto out = PreferenceLoss::apply(
      logp, PreferenceArgs{ref, ref_sums, mask, cu, pairs, preference_params(params, kind, reduction, by_length)});
  return {out[0], out[1]};
}

HeadArgs head_args(const Tensor& targets, std::optional<int64_t> ignore_index) {
  return HeadArgs{targets, ignore_index.value_or(0), ignore_index.has_value()};
}

Tensor log_probs(const Tensor& e, const Tensor& c, const OptTensor& bias, const Tensor& targets,
                 std::optional<int64_t> ignore_index) {
  plain(e);
  return LogProbs::apply(e, c, bias, head_args(targets, ignore_index));
}

std::tuple<Tensor, Tensor> linear_policy_loss(const Tensor& e, const Tensor& c, const OptTensor& bias,
                                              const Tensor& targets, std::optional<int64_t> ignore_index,
                                              const OptTensor& old, const OptTensor& ref, const Tensor& adv,
                                              const OptTensor& cu, int64_t S, at::ArrayRef<double> params,
                                              int64_t reduction, bool per_token) {
  plain(e);
  auto out = LinearPolicyLoss::apply(
      e, c, bias, std::make_pair(head_args(targets, ignore_index),
                                 PolicyArgs{old, ref, adv, std::nullopt, cu, S, policy_params(params, reduction, per_token)}));
  return {out[0], out[1]};
}

std::tuple<Tensor, Tensor> linear_preference_loss(const Tensor& e, const Tensor& c, const OptTensor& bias,
                                                  const Tensor& targets, std::optional<int64_t> ignore_index,
                                                  const OptTensor& ref, const OptTensor& ref_sums, const OptTensor& cu,
                                                  int64_t pairs, at::ArrayRef<double> params, int64_t kind,
                                                  int64_t reduction, bool by_length) {
  plain(e);
  auto out = LinearPreferenceLoss::apply(
      e, c, bias,
      std::make_pair(head_args(targets, ignore_index),
                     PreferenceArgs{ref, ref_sums, std::nullopt, cu, pairs,
                                    preference_params(params, kind, reduction, by_length)}));
  return {out[0], out[1]};
}

Tensor distillation(const Tensor& e, const Tensor& c, const OptTensor& bias, const Tensor& ids, const Tensor& teacher,
                    const OptTensor& mask, double temperature, bool tail, int64_t reduction) {
  plain(e);
  return Distillation::apply(e, c, bias,
                             DistillArgs{ids, teacher, mask, CceDistillParams{temperature, tail, (int32_t)reduction}});
}

}  // namespace

TORCH_LIBRARY(cce_b200, m) {
  m.def("bind(int[] addresses) -> ()", [](at::IntArrayRef a) { bind_library(a.vec()); });
  m.def("functions() -> str[]", [] { return functions(); });
  m.def("policy_loss(Tensor logp, Tensor? old, Tensor? ref, Tensor adv, Tensor? mask, Tensor? cu, int S, "
        "float[] params, int reduction, bool per_token) -> (Tensor, Tensor)", policy_loss);
  m.def("preference_loss(Tensor logp, Tensor? ref, Tensor? ref_sums, Tensor? mask, Tensor? cu, int pairs, "
        "float[] params, int kind, int reduction, bool by_length) -> (Tensor, Tensor)", preference_loss);
  m.def("log_probs(Tensor e, Tensor c, Tensor? bias, Tensor targets, int? ignore_index) -> Tensor", log_probs);
  m.def("linear_policy_loss(Tensor e, Tensor c, Tensor? bias, Tensor targets, int? ignore_index, Tensor? old, "
        "Tensor? ref, Tensor adv, Tensor? cu, int S, float[] params, int reduction, bool per_token) -> "
        "(Tensor, Tensor)", linear_policy_loss);
  m.def("linear_preference_loss(Tensor e, Tensor c, Tensor? bias, Tensor targets, int? ignore_index, Tensor? ref, "
        "Tensor? ref_sums, Tensor? cu, int pairs, float[] params, int kind, int reduction, bool by_length) -> "
        "(Tensor, Tensor)", linear_preference_loss);
  m.def("distillation(Tensor e, Tensor c, Tensor? bias, Tensor ids, Tensor teacher, Tensor? mask, "
        "float temperature, bool tail, int reduction) -> Tensor", distillation);
}
