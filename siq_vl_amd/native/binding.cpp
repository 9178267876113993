// Native host side of the operators of preference and policy training and of
// 8-bit activations: argument checks, allocation, launches through the C ABI and
// the autograd nodes, as cross_entropy.py and attention.py have them in Python.
//
// These calls are short: a loss of one pair takes 8 us of kernels, and with the
// same steps in Python it took 95 us with its backward.  Here it takes 57: an
// argument check costs a comparison, and a backward, which autograd runs on its
// device's thread, does not wait there for the interpreter.
//
// The library is not linked: bind() takes the addresses of its entry points from
// the ctypes handle, so there is one library, found in one way.  Errors are
// ValueError and RuntimeError with the same texts as there.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/extension.h>

#include <map>
#include <string>

#include "../../include/siq_kernels.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---------------------------------------------------------------- the library
#define SIQ_ENTRIES(X)                                                                                              \
  X(siq_last_error) X(siq_pack8) X(siq_unpack8) X(siq_swiglu8_fwd) X(siq_swiglu8_bwd) X(siq_pref_workspace_bytes)   \
  X(siq_pref_fwd) X(siq_pref_bwd) X(siq_policy_workspace_bytes) X(siq_policy_fwd) X(siq_policy_bwd)                 \
  X(siq_flp_saved_bytes) X(siq_flp_fwd_workspace_bytes) X(siq_flp_fwd) X(siq_flp_bwd_workspace_bytes) X(siq_flp_bwd)

struct Api {
#define SIQ_MEMBER(name) decltype(&::name) name = nullptr;
  SIQ_ENTRIES(SIQ_MEMBER)
#undef SIQ_MEMBER
} api;

std::vector<std::string> entries() {
  std::vector<std::string> names;
#define SIQ_NAME(name) names.push_back(#name);
  SIQ_ENTRIES(SIQ_NAME)
#undef SIQ_NAME
  return names;
}

void bind(const std::map<std::string, uintptr_t>& at) {
#define SIQ_BIND(name) api.name = reinterpret_cast<decltype(&::name)>(at.at(#name));
  SIQ_ENTRIES(SIQ_BIND)
#undef SIQ_BIND
}

void check(int rc, const char* what) {
  if (rc == SIQ_OK) return;
  const std::string text = c10::str(what, ": ", api.siq_last_error(), " (status ", rc, ")");
  TORCH_CHECK_VALUE(rc == SIQ_ERR_LAUNCH, text);
  TORCH_CHECK(false, text);
}

// ---------------------------------------------------------------- arguments
// What an error says of a type, and of a shape, as Python writes them.
std::string type_name(const Tensor& t) {
  const py::gil_scoped_acquire gil;
  return py::str(py::handle(reinterpret_cast<PyObject*>(torch::getTHPDtype(t.scalar_type()))));
}

std::string shape_name(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// No tensor, held or not: a null pointer.  A node's inputs that may be missing
// are optionals; an undefined tensor is no input that it takes.
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const optional<Tensor>& t) { return t.has_value() ? ptr(*t) : nullptr; }
template <class T>
float* fptr(const T& t) {
  return static_cast<float*>(ptr(t));
}

Tensor defined(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }

void on_gpu(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must live on the GPU, got ", t.device());
}

void on_device(const Tensor& t, const char* name, const Tensor& like) {
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " must live on ", like.device(), ", got ", t.device());
}

void no_second_derivative(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative (create_graph=True)");
}

// Where no gradient is recorded the kernels are called without their node, which would refuse a forward-mode tangent:
// a result without one would say that the derivative is zero.
void no_tangent(const char* what, std::initializer_list<Tensor> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor& t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}

// Contiguous and 16-byte aligned.
Tensor flat(const Tensor& t) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

// ---------------------------------------------------------------- 8-bit storage
int dtype_of(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, name,
                    " must be bfloat16 or float32, got ", type_name(t));
  on_gpu(t, name);
  return t.scalar_type() == at::kFloat ? SIQ_DTYPE_FP32 : SIQ_DTYPE_BF16;
}

constexpr int64_t kGroup = 32;
int64_t groups_of(int64_t numel) { return (numel + kGroup - 1) / kGroup; }

// `count` pairs of code and scale bytes for numel elements each, in one allocation.
variable_list stores(int64_t numel, int count, const Tensor& like) {
  auto up = [](int64_t n) { return (n + 255) & ~int64_t(255); };
  const int64_t step = up(numel) + up(groups_of(numel));
  const Tensor buf = bytes(step * count, like);
  variable_list out;
  for (int i = 0; i < count; ++i) {
    out.push_back(buf.narrow(0, i * step, numel));
    out.push_back(buf.narrow(0, i * step + up(numel), groups_of(numel)));
  }
  return out;
}

std::pair<Tensor, Tensor> pack8(const Tensor& x, int format) {
  const int dtype = dtype_of(x, "x");
  const c10::DeviceGuard guard(x.device());
  const at::NoGradGuard no_grad;
  const Tensor f = flat(x);
  const variable_list s = stores(f.numel(), 1, f);
  check(api.siq_pack8(f.data_ptr(), f.numel(), dtype, format, s[0].data_ptr(), s[1].data_ptr(), stream_of(f)),
        "siq_pack8");
  return {s[0], s[1]};
}

void check_stores(const Tensor& t, const char* name, int64_t n) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kByte && t.dim() == 1 && t.numel() == n && t.is_contiguous(), name, " must be ", n,
                    " contiguous uint8, got ", shape_name(t), " ", type_name(t));
}

Tensor unpack8(const Tensor& codes, const Tensor& scales, std::vector<int64_t> shape, bool fp32, int format) {
  const int64_t numel = c10::multiply_integers(shape);
  check_stores(codes, "codes", numel);
  check_stores(scales, "scales", groups_of(numel));
  TORCH_CHECK_VALUE(codes.is_cuda() && scales.device() == codes.device(), "codes and scales must live on one GPU, got ",
                    codes.device(), " and ", scales.device());
  const c10::DeviceGuard guard(codes.device());
  const Tensor x = at::empty(shape, codes.options().dtype(fp32 ? at::kFloat : at::kBFloat16));
  check(api.siq_unpack8(codes.data_ptr(), scales.data_ptr(), numel, fp32 ? SIQ_DTYPE_FP32 : SIQ_DTYPE_BF16, format,
                        x.data_ptr(), stream_of(x)),
        "siq_unpack8");
  return x;
}

// A [rows, cols] view that the kernels read in place, or a contiguous copy.
Tensor rows_of(const Tensor& t) {
  const Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  const int64_t step = r.scalar_type() == at::kFloat ? 4 : 8;
  const bool in_place = r.is_contiguous() || (r.stride(1) == 1 && r.stride(0) >= r.size(1) && r.stride(0) % step == 0 &&
                                              r.size(1) % 8 == 0);
  const bool aligned = reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0;
  if (in_place && aligned) return r;
  return r.is_contiguous() ? r.clone() : r.contiguous();
}
int64_t ld_of(const Tensor& r) { return r.size(0) > 1 && !r.is_contiguous() ? r.stride(0) : r.size(1); }

std::pair<Tensor, variable_list> swiglu8_fwd(const Tensor& gate, const Tensor& up, int format, bool keep) {
  const int dtype = dtype_of(gate, "gate");
  dtype_of(up, "up");
  TORCH_CHECK_VALUE(gate.dim() > 0 && up.dim() > 0, gate.dim() ? "up" : "gate", " must have at least one dimension");
  TORCH_CHECK_VALUE(gate.sizes() == up.sizes() && gate.scalar_type() == up.scalar_type() && gate.device() == up.device(),
                    "gate and up must be alike, got ", shape_name(gate), " ", type_name(gate), " on ", gate.device(), " and ",
                    shape_name(up), " ", type_name(up), " on ", up.device());
  const c10::DeviceGuard guard(gate.device());
  const Tensor h = at::empty(gate.sizes(), gate.options());
  variable_list s;
  if (keep) s = stores(h.numel(), 2, h);
  if (h.numel() > 0) {
    const Tensor g = rows_of(gate), u = rows_of(up);
    auto at = [&](int i) { return keep ? s[i].data_ptr() : nullptr; };
    check(api.siq_swiglu8_fwd(g.data_ptr(), u.data_ptr(), g.size(0), g.size(1), ld_of(g), ld_of(u), dtype, format,
                              h.data_ptr(), at(0), at(1), at(2), at(3), stream_of(h)),
          "siq_swiglu8_fwd");
  }
  return {h, s};
}

// (dgate, dup, h), or with `fused` (both gradients side by side, undefined, h); h undefined unless need_h.
std::tuple<Tensor, Tensor, Tensor> swiglu8_bwd(const Tensor& grad, const variable_list& s, int format, bool need_h,
                                               bool fused) {
  const int dtype = dtype_of(grad, "dh");
  TORCH_CHECK_VALUE(grad.dim() > 0, "dh must have at least one dimension");
  const int64_t numel = grad.numel(), cols = grad.size(-1);
  TORCH_CHECK_VALUE(s.size() == 4, "the packed gate and up are four tensors");
  for (int i = 0; i < 4; ++i)
    TORCH_CHECK_VALUE(s[i].scalar_type() == at::kByte && s[i].numel() == (i % 2 ? groups_of(numel) : numel) &&
                          s[i].is_contiguous() && s[i].device() == grad.device(),
                      "the packed gate and up do not belong to a gradient of shape ", shape_name(grad));
  const c10::DeviceGuard guard(grad.device());
  // the halves of one tensor are written in place where their rows start at 16-byte boundaries
  const bool halves = fused && cols % 8 == 0;
  Tensor both, dgate, dup, h;
  if (fused) {
    std::vector<int64_t> shape = grad.sizes().vec();
    shape.back() = 2 * cols;
    both = at::empty(shape, grad.options());
  }
  if (halves) {
    dgate = both.narrow(-1, 0, cols);
    dup = both.narrow(-1, cols, cols);
  } else {
    dgate = at::empty(grad.sizes(), grad.options());
    dup = at::empty(grad.sizes(), grad.options());
  }
  if (need_h) h = at::empty(grad.sizes(), grad.options());
  if (numel > 0) {
    const Tensor dh = flat(grad);
    const int64_t rows = numel / cols, ld = halves ? 2 * cols : cols;
    check(api.siq_swiglu8_bwd(dh.data_ptr(), s[0].data_ptr(), s[1].data_ptr(), s[2].data_ptr(), s[3].data_ptr(), rows, cols,
                              ld, ld, dtype, format, dgate.data_ptr(), dup.data_ptr(), ptr(h), stream_of(dh)),
          "siq_swiglu8_bwd");
    if (fused && !halves) {
      both.narrow(-1, 0, cols).copy_(dgate);
      both.narrow(-1, cols, cols).copy_(dup);
    }
  }
  if (fused) return {both, Tensor(), h};
  return {dgate, dup, h};
}

struct Swiglu8 : torch::autograd::Function<Swiglu8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up, int64_t format) {
    auto [h, s] = swiglu8_fwd(gate, up, (int)format, true);
    ctx->save_for_backward(s);
    ctx->saved_data["format"] = format;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    no_second_derivative("swiglu8");
    auto [dgate, dup, h] =
        swiglu8_bwd(grads[0], ctx->get_saved_variables(), (int)ctx->saved_data["format"].toInt(), false, false);
    return {dgate, dup, Tensor()};
  }
};

struct Swiglu8Fused : torch::autograd::Function<Swiglu8Fused> {
  static Tensor forward(AutogradContext* ctx, const Tensor& gate_up, int64_t format) {
    const int64_t cols = gate_up.size(-1) / 2;
    auto [h, s] = swiglu8_fwd(gate_up.narrow(-1, 0, cols), gate_up.narrow(-1, cols, cols), (int)format, true);
    ctx->save_for_backward(s);
    ctx->saved_data["format"] = format;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    no_second_derivative("swiglu8");
    return {std::get<0>(swiglu8_bwd(grads[0], ctx->get_saved_variables(), (int)ctx->saved_data["format"].toInt(), false,
                                    true)),
            Tensor()};
  }
};

Tensor swiglu8(const Tensor& gate, const optional<Tensor>& up, int format) {
  no_tangent("swiglu8", {gate, defined(up)});
  const bool grad = at::GradMode::is_enabled();
  if (!up.has_value()) {
    TORCH_CHECK_VALUE(gate.dim() > 0 && gate.size(-1) % 2 == 0,
                      "gate and up side by side need an even last dimension, got ", shape_name(gate));
    if (grad && gate.requires_grad()) return Swiglu8Fused::apply(gate, format);
    const int64_t cols = gate.size(-1) / 2;
    return swiglu8_fwd(gate.narrow(-1, 0, cols), gate.narrow(-1, cols, cols), format, false).first;
  }
  if (grad && (gate.requires_grad() || up->requires_grad())) return Swiglu8::apply(gate, *up, format);
  return swiglu8_fwd(gate, *up, format, false).first;
}

// ---------------------------------------------------------------- losses
// fp32 values, one a token; `like`: of that shape, on that device; `frozen`: no gradient goes there.
Tensor logps_of(const char* name, const Tensor& t, const Tensor& like, bool frozen) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, name, " must be float32, got ", type_name(t));
  on_gpu(t, name);
  TORCH_CHECK_VALUE(!like.defined() || (t.sizes() == like.sizes() && t.device() == like.device()), name, " must be ",
                    shape_name(like.defined() ? like : t), " on ",
                    (like.defined() ? like : t).device(), ", got ", shape_name(t), " on ", t.device());
  TORCH_CHECK_VALUE(!frozen || !t.requires_grad(), "gradients with respect to ", name, " are not supported (detach it)");
  return t.contiguous();
}

optional<Tensor> reference_of(const optional<Tensor>& t, const Tensor& like) {
  return t.has_value() ? optional<Tensor>(logps_of("reference_logps", *t, like, true)) : t;
}

optional<Tensor> mask_of(const optional<Tensor>& mask, const Tensor& like) {
  if (!mask.has_value()) return mask;
  TORCH_CHECK_VALUE(mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte, "mask must be bool or uint8, got ",
                    type_name(*mask));
  TORCH_CHECK_VALUE(mask->sizes() == like.sizes() && mask->device() == like.device(), "mask must be ", shape_name(like), " on ",
                    like.device(), ", got ", shape_name(*mask), " on ", mask->device());
  return mask->contiguous();
}

Tensor offsets_of(const Tensor& cu, const Tensor& like) {
  TORCH_CHECK_VALUE(cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.numel() >= 2 && cu.device() == like.device(),
                    "cu_seqlens must be int32 [sequences + 1] on ", like.device(), ", got ", shape_name(cu), " ",
                    type_name(cu), " on ", cu.device());
  return cu.contiguous();
}

// The upstream gradient of a scalar loss, fp32.
Tensor upstream(const Tensor& grad) { return grad.scalar_type() == at::kFloat ? grad : grad.to(at::kFloat); }

template <class T>
const int32_t* cu_ptr(const T& cu) {
  return static_cast<const int32_t*>(ptr(cu));
}
int64_t sequences(const optional<Tensor>& cu) { return cu.has_value() ? cu->numel() - 1 : 1; }

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& policy, const optional<Tensor>& reference,
                               const Tensor& cu, const optional<Tensor>& mask, int64_t type, int64_t order, double beta,
                               double smoothing, bool normalized, const optional<Tensor>& divisor) {
    const int64_t tokens = policy.numel(), pairs = (cu.numel() - 1) / 2;
    const Tensor loss = floats({}, policy), chosen = floats({pairs}, policy), rejected = floats({pairs}, policy);
    const Tensor coef = floats({2 * pairs}, policy), ws = bytes(api.siq_pref_workspace_bytes(pairs, tokens), policy);
    check(api.siq_pref_fwd(fptr(policy), fptr(reference), ptr(mask), cu_ptr(cu), pairs, tokens, (int)type, (int)order, beta,
                           smoothing, normalized, fptr(divisor), fptr(loss), fptr(chosen), fptr(rejected), fptr(coef),
                           ptr(ws), ws.numel(), stream_of(policy)),
          "siq_pref_fwd");
    ctx->save_for_backward({coef, cu, defined(mask)});
    ctx->saved_data["shape"] = policy.sizes().vec();
    ctx->mark_non_differentiable({chosen, rejected});
    ctx->set_materialize_grads(false);
    return {loss, chosen, rejected};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    no_second_derivative("preference_loss");
    variable_list out(10);
    if (!grads[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &coef = saved[0], &cu = saved[1], &mask = saved[2], grad = upstream(grads[0]);
    const c10::DeviceGuard guard(coef.device());
    out[0] = floats(ctx->saved_data["shape"].toIntVector(), coef);
    check(api.siq_pref_bwd(fptr(grad), fptr(coef), ptr(mask), cu_ptr(cu), (cu.numel() - 1) / 2, out[0].numel(),
                           fptr(out[0]), stream_of(coef)),
          "siq_pref_bwd");
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor> preference_loss(const Tensor& policy, const optional<Tensor>& reference, const Tensor& cu,
                                                   const optional<Tensor>& mask, int64_t type, int64_t order, double beta,
                                                   double smoothing, bool normalized, const optional<Tensor>& divisor) {
  const Tensor p = logps_of("policy_logps", policy, Tensor(), false);
  const optional<Tensor> r = reference_of(reference, p), m = mask_of(mask, p);
  const Tensor c = offsets_of(cu, p);
  TORCH_CHECK_VALUE(c.numel() % 2 == 1, "preference pairs need an even number of sequences, got ", c.numel() - 1);
  const c10::DeviceGuard guard(p.device());
  const variable_list o = PreferenceLoss::apply(p, r, c, m, type, order, beta, smoothing, normalized, divisor);
  return {o[0], o[1], o[2]};
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logps, const Tensor& old, const Tensor& advantages,
                               const optional<Tensor>& cu, const optional<Tensor>& mask, const optional<Tensor>& reference,
                               bool per_token, int64_t aggregation, int64_t kl_type, double low, double high, double dual,
                               double kl_coef, const optional<Tensor>& divisor) {
    const int64_t tokens = logps.numel(), seqs = sequences(cu);
    const Tensor loss = floats({}, logps), kl = floats({}, logps), cut = floats({}, logps);
    const Tensor dtoken = floats({tokens}, logps), weight = floats({aggregation == SIQ_AGG_SEQUENCE ? seqs : 1}, logps);
    const Tensor ws = bytes(api.siq_policy_workspace_bytes(seqs, tokens), logps);
    check(api.siq_policy_fwd(fptr(logps), fptr(old), fptr(advantages), ptr(mask), fptr(reference), cu_ptr(cu), seqs, tokens,
                             per_token, (int)aggregation, (int)kl_type, low, high, dual, kl_coef, fptr(divisor), fptr(loss),
                             fptr(kl), fptr(cut), fptr(dtoken), fptr(weight), ptr(ws), ws.numel(), stream_of(logps)),
          "siq_policy_fwd");
    ctx->save_for_backward({dtoken, weight, defined(cu)});
    ctx->saved_data["shape"] = logps.sizes().vec();
    ctx->saved_data["aggregation"] = aggregation;
    ctx->mark_non_differentiable({kl, cut});
    ctx->set_materialize_grads(false);
    return {loss, kl, cut};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    no_second_derivative("policy_loss");
    variable_list out(14);
    if (!grads[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &dtoken = saved[0], &weight = saved[1], &cu = saved[2], grad = upstream(grads[0]);
    const c10::DeviceGuard guard(dtoken.device());
    out[0] = floats(ctx->saved_data["shape"].toIntVector(), dtoken);
    check(api.siq_policy_bwd(fptr(grad), fptr(dtoken), fptr(weight), cu_ptr(cu), cu.defined() ? cu.numel() - 1 : 1,
                             dtoken.numel(), (int)ctx->saved_data["aggregation"].toInt(), fptr(out[0]), stream_of(dtoken)),
          "siq_policy_bwd");
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor> policy_loss(const Tensor& logps, const Tensor& old, const Tensor& advantages,
                                               const optional<Tensor>& cu, const optional<Tensor>& mask,
                                               const optional<Tensor>& reference, int64_t aggregation, int64_t kl_type,
                                               double low, double high, double dual, double kl_coef,
                                               const optional<Tensor>& divisor) {
  const Tensor lp = logps_of("logps", logps, Tensor(), false), o = logps_of("old_logps", old, lp, true);
  const optional<Tensor> ref = reference_of(reference, lp), m = mask_of(mask, lp);
  const optional<Tensor> c = cu.has_value() ? optional<Tensor>(offsets_of(*cu, lp)) : cu;
  const int64_t seqs = sequences(c);
  const bool per_token = advantages.sizes() == lp.sizes();
  const Tensor adv = logps_of("advantages", advantages, per_token ? lp : Tensor(), true);
  TORCH_CHECK_VALUE(per_token || (adv.dim() == 1 && adv.numel() == seqs && adv.device() == lp.device()), "advantages must be ",
                    shape_name(lp), " (one a token) or [", seqs, "] (one a sequence) on ", lp.device(), ", got ", shape_name(adv),
                    " on ", adv.device());
  const c10::DeviceGuard guard(lp.device());
  const variable_list out =
      PolicyLoss::apply(lp, o, adv, c, m, ref, per_token, aggregation, kl_type, low, high, dual, kl_coef, divisor);
  return {out[0], out[1], out[2]};
}

// ---------------------------------------------------------------- log-probabilities of the labels
void check_head(const Tensor& hidden, const Tensor& weight, const Tensor& labels) {
  TORCH_CHECK_VALUE(hidden.dim() == 2 && weight.dim() == 2, "hidden must be [n, hdim] and weight [vocab, hdim]");
  TORCH_CHECK_VALUE(weight.size(1) == hidden.size(1), "weight hdim ", weight.size(1), " != hidden hdim ", hidden.size(1));
  TORCH_CHECK_VALUE(hidden.scalar_type() == at::kBFloat16, "hidden must be bfloat16, got ", type_name(hidden));
  on_gpu(hidden, "hidden");
  TORCH_CHECK_VALUE(weight.scalar_type() == at::kBFloat16, "weight must be bfloat16, got ", type_name(weight));
  TORCH_CHECK_VALUE(labels.dim() == 1 && labels.size(0) == hidden.size(0), "labels must be [n] = [", hidden.size(0), "], got ",
                    shape_name(labels));
  TORCH_CHECK_VALUE(labels.scalar_type() == at::kLong, "labels must be int64, got ", type_name(labels));
  on_device(weight, "weight", hidden);
  on_device(labels, "labels", hidden);
}

// (logp of that shape, what is kept or undefined); counts: the valid and the bad labels
std::pair<Tensor, Tensor> flp_fwd(const Tensor& hidden, const Tensor& weight, const Tensor& labels, int64_t ignore_index,
                                  double temperature, bool keep, at::IntArrayRef shape, int64_t* counts) {
  check_head(hidden, weight, labels);
  const c10::DeviceGuard guard(hidden.device());
  const Tensor h = hidden.contiguous(), w = weight.contiguous(), y = labels.contiguous();
  const int64_t n = h.size(0), hdim = h.size(1), vocab = w.size(0);
  const Tensor logp = floats(shape, h);
  const Tensor saved = keep ? bytes(api.siq_flp_saved_bytes(n, vocab), h) : Tensor();
  const Tensor ws = bytes(api.siq_flp_fwd_workspace_bytes(n, hdim, vocab, keep), h);
  check(api.siq_flp_fwd(h.data_ptr(), w.data_ptr(), static_cast<const int64_t*>(ptr(y)), n, hdim, vocab, ignore_index,
                        temperature, fptr(logp), counts, counts + 1, ptr(saved), keep ? saved.numel() : 0, ptr(ws), ws.numel(),
                        stream_of(h)),
        "siq_flp_fwd");
  return {logp, saved};
}

std::pair<Tensor, Tensor> flp_bwd(const Tensor& hidden, const Tensor& weight, const Tensor& labels, const Tensor& dlogp,
                                  int64_t ignore_index, double temperature, const Tensor& saved, bool need_dhidden,
                                  bool need_dweight, int64_t chunk) {
  check_head(hidden, weight, labels);
  const int64_t n = hidden.size(0), hdim = hidden.size(1), vocab = weight.size(0);
  TORCH_CHECK_VALUE(dlogp.dim() == 1 && dlogp.size(0) == n && dlogp.scalar_type() == at::kFloat, "dlogp must be float32 [", n,
                    "], got ", type_name(dlogp), " ", shape_name(dlogp));
  on_device(dlogp, "dlogp", hidden);
  if (saved.defined()) {
    on_device(saved, "saved", hidden);
    const int64_t size = api.siq_flp_saved_bytes(n, vocab);
    TORCH_CHECK_VALUE(saved.scalar_type() == at::kByte && saved.dim() == 1 && saved.numel() == size && saved.is_contiguous(),
                      "saved must be what the forward kept (", size, " bytes), got ", shape_name(saved), " ", type_name(saved));
  }
  TORCH_CHECK_VALUE(chunk > 0, "chunk_tokens must be positive");
  const c10::DeviceGuard guard(hidden.device());
  const Tensor h = hidden.contiguous(), w = weight.contiguous(), y = labels.contiguous(), g = dlogp.contiguous();
  const Tensor dh = need_dhidden ? at::empty(h.sizes(), h.options()) : Tensor();
  const Tensor dw = need_dweight ? at::empty(w.sizes(), w.options()) : Tensor();
  const bool have = saved.defined();
  const Tensor ws = bytes(api.siq_flp_bwd_workspace_bytes(n, hdim, vocab, chunk, need_dweight, have), h);
  check(api.siq_flp_bwd(h.data_ptr(), w.data_ptr(), static_cast<const int64_t*>(ptr(y)), fptr(g), n, hdim, vocab,
                        ignore_index, temperature, ptr(saved), have ? saved.numel() : 0, ptr(dh), ptr(dw), chunk, ptr(ws),
                        ws.numel(), stream_of(h)),
        "siq_flp_bwd");
  return {dh, dw};
}

Tensor rows_2d(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }
Tensor rows_1d(const Tensor& t) { return t.dim() == 1 ? t : t.reshape({-1}); }

struct LinearLogProbs : torch::autograd::Function<LinearLogProbs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& labels,
                        int64_t ignore_index, double temperature, int64_t chunk, int64_t keep_bytes, int64_t* counts) {
    const Tensor h = rows_2d(hidden), y = rows_1d(labels);
    const bool keep = weight.dim() == 2 && (int64_t)api.siq_flp_saved_bytes(h.size(0), weight.size(0)) <= keep_bytes;
    auto [logp, saved] = flp_fwd(h, weight, y, ignore_index, temperature, keep, labels.sizes(), counts);
    ctx->save_for_backward({hidden, weight, labels, saved});
    ctx->saved_data["ignore"] = ignore_index;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["chunk"] = chunk;
    ctx->set_materialize_grads(false);
    return logp;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    no_second_derivative("fused_linear_log_probs");
    variable_list out(8);
    if (!grads[0].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    auto [dh, dw] = flp_bwd(rows_2d(s[0]), s[1], rows_1d(s[2]), rows_1d(grads[0]), ctx->saved_data["ignore"].toInt(),
                            ctx->saved_data["temperature"].toDouble(), s[3], ctx->needs_input_grad(0),
                            ctx->needs_input_grad(1), ctx->saved_data["chunk"].toInt());
    if (dh.defined()) out[0] = dh.view(s[0].sizes());
    out[1] = dw;
    return out;
  }
};

// (logp, [count, bad labels]); nothing is kept where no gradient can flow.  `host`: pinned memory that the kernel
// writes the counts to, so that no copy follows it; the caller keeps it until the call has run.
std::pair<Tensor, Tensor> linear_log_probs(const Tensor& hidden, const Tensor& weight, const Tensor& labels,
                                           int64_t ignore_index, double temperature, int64_t chunk, int64_t keep_bytes,
                                           const optional<Tensor>& host) {
  TORCH_CHECK_VALUE(chunk > 0, "chunk_tokens must be positive");
  no_tangent("fused_linear_log_probs", {hidden, weight});
  const Tensor counts = host.has_value() ? *host : at::empty({2}, hidden.options().dtype(at::kLong));
  int64_t* const c = counts.data_ptr<int64_t>();
  if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad()))
    return {LinearLogProbs::apply(hidden, weight, labels, ignore_index, temperature, chunk, keep_bytes, c), counts};
  return {flp_fwd(rows_2d(hidden), weight, rows_1d(labels), ignore_index, temperature, false, labels.sizes(), c).first,
          counts};
}

// The raw forms.
std::tuple<Tensor, Tensor, Tensor> raw_flp_fwd(const Tensor& hidden, const Tensor& weight, const Tensor& labels,
                                               int64_t ignore_index, double temperature, bool keep) {
  check_head(hidden, weight, labels);
  const Tensor counts = at::empty({2}, labels.options());
  auto [logp, saved] =
      flp_fwd(hidden, weight, labels, ignore_index, temperature, keep, labels.sizes(), counts.data_ptr<int64_t>());
  return {logp, counts, saved};
}

std::pair<Tensor, Tensor> raw_flp_bwd(const Tensor& hidden, const Tensor& weight, const Tensor& labels, const Tensor& dlogp,
                                      int64_t ignore_index, double temperature, const optional<Tensor>& saved,
                                      bool need_dhidden, bool need_dweight, int64_t chunk) {
  return flp_bwd(hidden, weight, labels, dlogp, ignore_index, temperature, defined(saved), need_dhidden, need_dweight,
                 chunk);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("entries", &entries);
  m.def("bind", &bind);
  // as torch's own operators, these run without the interpreter's lock: an allocation may wait for the GPU
#define SIQ_DEF(name, fn) m.def(name, torch::wrap_pybind_function_no_gil(fn))
  SIQ_DEF("pack8", pack8);
  SIQ_DEF("unpack8", unpack8);
  SIQ_DEF("swiglu8_fwd", swiglu8_fwd);
  SIQ_DEF("swiglu8_bwd", swiglu8_bwd);
  SIQ_DEF("swiglu8", swiglu8);
  SIQ_DEF("preference_loss", preference_loss);
  SIQ_DEF("policy_loss", policy_loss);
  SIQ_DEF("flp_fwd", raw_flp_fwd);
  SIQ_DEF("flp_bwd", raw_flp_bwd);
  SIQ_DEF("linear_log_probs", linear_log_probs);
  m.def("no_tangent", [](const char* what, const std::vector<Tensor>& inputs) {
    for (const Tensor& t : inputs) no_tangent(what, {t});
  });
#undef SIQ_DEF
}
