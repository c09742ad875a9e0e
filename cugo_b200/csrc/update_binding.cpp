// The policy update's operators as Python calls: argument checks, outputs, autograd
// functions and the calls of the C ABI (include/cugo_b200.h).  These operators run for a
// few microseconds on a minibatch, less than Python takes to check fifteen tensors, enter
// an autograd function and fill a C call's arguments; the rest of the package's calls
// stay on ctypes (ext.py).
//
// Every call checks its tensors on the host, allocates its outputs and scratch with torch
// (in a captured graph, from the graph's own pool) and enqueues on the current stream of
// the tensors' device.  Errors are std::runtime_error: RuntimeError in Python.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/cugo_b200.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

[[noreturn]] void fail(const std::string& op, const std::string& what) { throw std::runtime_error(op + ": " + what); }

void check(int rc, const char* op) {
  if (rc == CUGO_B200_OK) return;
  const char* what = rc == CUGO_B200_ERR_ARG      ? "invalid argument"
                     : rc == CUGO_B200_ERR_ALIGN  ? "misaligned pointer"
                     : rc == CUGO_B200_ERR_LAUNCH ? "kernel launch failed"
                                                  : "over a fixed capacity";
  throw std::runtime_error(std::string("cugo_b200 ") + op + ": " + what);
}

bool there(const Maybe& t) { return t && t->defined(); }
int cuda_index(const Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }

int type_code(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

// t [rows, >= cols] with unit column stride and rows that do not overlap; its row stride.
int64_t matrix(const char* op, const char* name, const Tensor& t, int64_t rows, int64_t cols, int device) {
  if (cuda_index(t) != device) fail(op, std::string(name) + " must be on the logits' device");
  if (t.dim() != 2 || t.size(0) != rows || t.size(1) < cols) fail(op, std::string(name) + " has the wrong shape");
  if ((t.stride(1) != 1 && t.size(1) > 1) || (t.stride(0) < t.size(1) && rows > 1))
    fail(op, std::string(name) + " must be row-major (unit column stride)");
  return t.stride(0);
}

void vector(const char* op, const char* name, const Tensor& t, int64_t n, at::ScalarType type, int device) {
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    fail(op, std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor of " + std::to_string(n) +
                 " entries");
  if (cuda_index(t) != device) fail(op, std::string(name) + " must be on cuda:" + std::to_string(device));
}

const float* scalar(const char* op, const char* name, const Maybe& t, int device) {
  if (!there(t)) return nullptr;
  if (t->scalar_type() != at::kFloat || t->numel() != 1 || cuda_index(*t) != device)
    fail(op, std::string(name) + " must be one fp32 value on cuda:" + std::to_string(device));
  return t->const_data_ptr<float>();
}

const float* floats(const Maybe& t) { return there(t) ? t->const_data_ptr<float>() : nullptr; }
float* out_floats(Tensor& t) { return t.defined() ? t.mutable_data_ptr<float>() : nullptr; }

// The rows of a loss, checked.
struct Rows {
  const void* logits;
  const bool* legal = nullptr;
  const int64_t* actions;
  const float* weight = nullptr;
  int64_t ld, ldm = 0, rows, vocab;
  int type, device;
  at::TensorOptions fp32;

  Rows(const char* op, const Tensor& x, const Tensor& act, const Maybe& mask, const Maybe& w) {
    device = cuda_index(x);
    if (device < 0) fail(op, "logits must be a CUDA tensor");
    type = type_code(x.scalar_type());
    if (type < 0) fail(op, "logits must be fp32, bf16 or fp16");
    if (x.dim() != 2 || x.size(1) < 1) fail(op, "logits must be [rows, entries >= 1]");
    rows = x.size(0);
    vocab = x.size(1);
    ld = matrix(op, "logits", x, rows, vocab, device);
    vector(op, "actions", act, rows, at::kLong, device);
    logits = x.const_data_ptr();
    actions = act.const_data_ptr<int64_t>();
    if (there(mask)) {
      if (mask->scalar_type() != at::kBool || mask->sizes() != x.sizes())
        fail(op, "legal must be bool of the logits' shape");
      ldm = mask->stride(0);
      if (ldm != 0 || rows < 2)  // one mask expanded over the rows is fine
        ldm = matrix(op, "legal", *mask, rows, vocab, device);
      else if (cuda_index(*mask) != device || (mask->stride(1) != 1 && vocab > 1))
        fail(op, "legal must be row-major on the logits' device");
      legal = mask->const_data_ptr<bool>();
    }
    if (there(w)) {
      vector(op, "weight", *w, rows, at::kFloat, device);
      weight = w->const_data_ptr<float>();
    }
    fp32 = x.options().dtype(at::kFloat);
  }
};

// Whether the memory from the first to the last entry of two matrices overlaps.
bool overlap(const Tensor& a, const Tensor& b) {
  const auto end = [](const Tensor& t) {
    int64_t n = 1;
    for (int64_t d = 0; d < t.dim(); ++d) {
      if (t.size(d) == 0) return static_cast<const char*>(nullptr);
      n += (t.size(d) - 1) * t.stride(d);
    }
    return static_cast<const char*>(t.const_data_ptr()) + n * t.element_size();
  };
  return static_cast<const char*>(a.const_data_ptr()) < end(b) && static_cast<const char*>(b.const_data_ptr()) < end(a);
}

cudaStream_t stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

Tensor bytes(int64_t n, const at::TensorOptions& options) { return at::empty({n}, options.dtype(at::kByte)); }

// The kernels see the primal of a dual tensor only, and a trace sees their outputs'
// allocation only: a tangent, or the call itself, would be lost without a word.
void primal_only(const char* op, std::initializer_list<const Tensor*> tensors) {
  if (torch::jit::tracer::isTracing()) fail(op, "the call cannot be traced");
  for (const Tensor* t : tensors)
    if (t && t->defined() && t->_fw_grad(0).defined()) fail(op, "forward-mode derivatives are not built");
}
const Tensor* given(const Maybe& t) { return t ? &*t : nullptr; }

// A backward that autograd would differentiate again.
void once(const char* op) {
  if (at::GradMode::is_enabled()) fail(op, "the gradient's own gradient is not built");
}

// ---- action_logp --------------------------------------------------------------------------

struct Scored {
  Tensor logp, entropy, lse, zeros;
};

Scored score(const char* op, const Tensor& logits, const Tensor& actions, const Maybe& legal, const Maybe& weight,
             bool entropy, bool lse, bool zeros) {
  const Rows r(op, logits, actions, legal, weight);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(r.device));
  Scored s;
  s.logp = at::empty({r.rows}, r.fp32);
  if (entropy) s.entropy = at::empty({r.rows}, r.fp32);
  if (lse) s.lse = at::empty({r.rows, 2}, r.fp32);
  if (zeros) s.zeros = at::empty({r.rows}, r.fp32);
  check(cugo_b200_action_logp(r.logits, r.ld, r.type, r.legal, r.ldm, r.actions, r.weight, r.rows, r.vocab,
                              out_floats(s.logp), out_floats(s.entropy), out_floats(s.lse), out_floats(s.zeros),
                              stream_of(r.device)),
        op);
  return s;
}

Tensor score_backward(const char* op, const Tensor& logits, const Tensor& actions, const Maybe& legal,
                      const Tensor& lse, const Maybe& entropy, const Maybe& d_logp, const Maybe& d_entropy,
                      const Maybe& scale) {
  const Rows r(op, logits, actions, legal, std::nullopt);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(r.device));
  if (there(d_logp)) vector(op, "d_logp", *d_logp, r.rows, at::kFloat, r.device);
  if (there(d_entropy)) vector(op, "d_entropy", *d_entropy, r.rows, at::kFloat, r.device);
  Tensor d = at::empty({r.rows, r.vocab}, logits.options());
  check(cugo_b200_action_logp_backward(r.logits, r.ld, r.type, r.legal, r.ldm, r.actions, lse.const_data_ptr<float>(),
                                       floats(entropy), floats(d_logp), floats(d_entropy),
                                       scalar(op, "scale", scale, r.device), r.rows, r.vocab, d.mutable_data_ptr(),
                                       r.vocab, r.type, stream_of(r.device)),
        op);
  return d;
}

Maybe contiguous(const Tensor& t) { return t.defined() ? Maybe(t.contiguous()) : Maybe(); }

struct ActionLogp : torch::autograd::Function<ActionLogp> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& actions, const Maybe& legal) {
    Scored s = score("action_logp", logits, actions, legal, std::nullopt, true, true, false);
    ctx->save_for_backward({logits, actions, legal.value_or(Tensor()), s.lse, s.entropy});
    ctx->set_materialize_grads(false);
    return {s.logp, s.entropy};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("action_logp");
    primal_only("action_logp", {&grads[0], &grads[1]});
    Tensor d;
    if (grads[0].defined() || grads[1].defined()) {
      const auto s = ctx->get_saved_variables();
      d = score_backward("action_logp", s[0], s[1], s[2], s[3], s[4], contiguous(grads[0]), contiguous(grads[1]),
                         std::nullopt);
    }
    return {d, Tensor(), Tensor()};
  }
};

bool differentiable(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

std::tuple<Tensor, Tensor> action_logp(const Tensor& logits, const Tensor& actions, const Maybe& legal) {
  primal_only("action_logp", {&logits});
  if (differentiable(logits)) {
    const auto out = ActionLogp::apply(logits, actions, legal);
    return {out[0], out[1]};
  }
  Scored s = score("action_logp", logits, actions, legal, std::nullopt, true, false, false);
  return {s.logp, s.entropy};
}

// ---- policy_loss -----------------------------------------------------------------------------

// What policy_loss takes beside the logits.
struct PolicyArgs {
  Tensor actions, logp_old, adv;
  Maybe legal, weight, ref_logits, ref_logp;
  double clip_low, clip_high, kl_coef, entropy_coef, denominator;
  Maybe kl_coef_dev, entropy_coef_dev;
};

struct PolicyOut {
  Tensor loss, stats, logp, grad;
};

// stats: the loss and its statistics too, else the gradient only, with the denominator that
// an earlier call found.
PolicyOut policy(const Tensor& logits, const PolicyArgs& p, bool stats, const Maybe& denominator, double grad_scale,
                 const Maybe& grad_scale_dev, const Maybe& dlogits, std::optional<at::ScalarType> grad_type) {
  const char* op = "policy_loss";
  primal_only(op, {&logits, &p.logp_old, &p.adv, given(p.weight), given(p.ref_logits), given(p.ref_logp),
                   given(p.kl_coef_dev), given(p.entropy_coef_dev), given(grad_scale_dev), given(dlogits)});
  const Rows r(op, logits, p.actions, p.legal, p.weight);
  vector(op, "logp_old", p.logp_old, r.rows, at::kFloat, r.device);
  vector(op, "adv", p.adv, r.rows, at::kFloat, r.device);
  int64_t ldr = 0;
  const void* ref = nullptr;
  if (there(p.ref_logits)) {
    if (p.ref_logits->scalar_type() != logits.scalar_type() || p.ref_logits->sizes() != logits.sizes())
      fail(op, "ref_logits must have the logits' type and shape");
    ldr = matrix(op, "ref_logits", *p.ref_logits, r.rows, r.vocab, r.device);
    ref = p.ref_logits->const_data_ptr();
  }
  if (there(p.ref_logp)) {
    if (ref) fail(op, "give ref_logits or ref_logp, not both");
    vector(op, "ref_logp", *p.ref_logp, r.rows, at::kFloat, r.device);
  }
  if (p.denominator != 0.0 && static_cast<float>(p.denominator) == 0.0f) fail(op, "the denominator must be positive");
  // The same in double and in the kernel's float: a bound that rounds to less than 0 is not one.
  if (!(p.clip_low >= 0.0) || !(p.clip_high >= 0.0)) fail(op, "the clip's bounds must not be negative");
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(r.device));
  PolicyOut o;
  if (stats) {
    o.loss = at::empty({}, r.fp32);
    o.stats = at::empty({8}, r.fp32);
    o.logp = at::empty({r.rows}, r.fp32);
  }
  int64_t ldd = 0, width = r.vocab;
  int code = 0;
  if (there(dlogits)) o.grad = *dlogits;
  else if (grad_type) o.grad = at::empty({r.rows, r.vocab}, logits.options().dtype(*grad_type));
  if (o.grad.defined()) {
    code = type_code(o.grad.scalar_type());
    if (code < 0) fail(op, "dlogits must be fp32, bf16 or fp16");
    ldd = matrix(op, "dlogits", o.grad, r.rows, r.vocab, r.device);
    width = o.grad.size(1);
    // A long row's action is looked at once more after its gradient has been written.
    if (there(dlogits) && (overlap(o.grad, logits) || (ref && overlap(o.grad, *p.ref_logits))))
      fail(op, "dlogits must not share memory with the logits");
  }
  const int64_t need = cugo_b200_policy_loss_scratch_bytes(r.rows);
  Tensor scratch = bytes(need, r.fp32);
  check(cugo_b200_policy_loss(
            r.logits, r.ld, r.type, ref, ldr, r.legal, r.ldm, r.actions, p.logp_old.const_data_ptr<float>(),
            p.adv.const_data_ptr<float>(), r.weight, floats(p.ref_logp), r.rows, r.vocab,
            static_cast<float>(p.clip_low), static_cast<float>(p.clip_high), static_cast<float>(p.kl_coef),
            static_cast<float>(p.entropy_coef), scalar(op, "kl_coef", p.kl_coef_dev, r.device),
            scalar(op, "entropy_coef", p.entropy_coef_dev, r.device), static_cast<float>(p.denominator),
            scalar(op, "denominator", denominator, r.device), static_cast<float>(grad_scale),
            scalar(op, "grad_scale", grad_scale_dev, r.device), o.grad.defined() ? o.grad.mutable_data_ptr() : nullptr,
            ldd, code, width, out_floats(o.logp), out_floats(o.stats), out_floats(o.loss), scratch.mutable_data_ptr(),
            need, stream_of(r.device)),
        op);
  if (there(dlogits) && !dlogits->is_inference()) dlogits->unsafeGetTensorImpl()->bump_version();
  return o;
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const PolicyArgs& p) {
    PolicyOut o = policy(logits, p, true, std::nullopt, 1.0, std::nullopt, std::nullopt, std::nullopt);
    const auto or_none = [](const Maybe& t) { return t.value_or(Tensor()); };
    Tensor stats = o.stats.narrow(0, 0, 7);
    // Beside the statistics in memory, but with a version of its own: a caller may change
    // those in place before the backward.
    const Tensor denominator = o.stats.narrow(0, 7, 1).variable_data();
    ctx->save_for_backward({logits, p.actions, p.logp_old, p.adv, or_none(p.legal), or_none(p.weight),
                            or_none(p.ref_logits), or_none(p.ref_logp), or_none(p.kl_coef_dev),
                            or_none(p.entropy_coef_dev), denominator});
    ctx->saved_data["coefs"] = std::vector<double>{p.clip_low, p.clip_high, p.kl_coef, p.entropy_coef};
    ctx->mark_non_differentiable({stats, o.logp});
    ctx->set_materialize_grads(false);
    return {o.loss, stats, o.logp};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("policy_loss");
    Tensor d;
    if (grads[0].defined()) {
      const auto s = ctx->get_saved_variables();
      const auto c = ctx->saved_data["coefs"].toDoubleVector();
      // With the denominator that the forward found; the logits are read once more.
      const PolicyArgs p{s[1], s[2], s[3], s[4], s[5], s[6], s[7], c[0], c[1], c[2], c[3], 0.0, s[8], s[9]};
      d = policy(s[0], p, false, s[10], 1.0, grads[0], std::nullopt, s[0].scalar_type()).grad;
    }
    return {d, Tensor()};
  }
};

PolicyArgs policy_args(const Tensor& actions, const Tensor& logp_old, const Tensor& adv, const Maybe& legal,
                       const Maybe& weight, const Maybe& ref_logits, const Maybe& ref_logp, double clip_low,
                       double clip_high, double kl_coef, const Maybe& kl_coef_dev, double entropy_coef,
                       const Maybe& entropy_coef_dev, double denominator) {
  return {actions,  logp_old, adv,          legal,       weight,      ref_logits,      ref_logp, clip_low,
          clip_high, kl_coef, entropy_coef, denominator, kl_coef_dev, entropy_coef_dev};
}

std::tuple<Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& actions, const Tensor& logp_old,
                                               const Tensor& adv, const Maybe& legal, const Maybe& weight,
                                               const Maybe& ref_logits, const Maybe& ref_logp, double clip_low,
                                               double clip_high, double kl_coef, const Maybe& kl_coef_dev,
                                               double entropy_coef, const Maybe& entropy_coef_dev,
                                               double denominator) {
  const PolicyArgs p = policy_args(actions, logp_old, adv, legal, weight, ref_logits, ref_logp, clip_low, clip_high,
                                   kl_coef, kl_coef_dev, entropy_coef, entropy_coef_dev, denominator);
  if (differentiable(logits)) {
    const auto out = PolicyLoss::apply(logits, p);
    return {out[0], out[1], out[2]};
  }
  PolicyOut o = policy(logits, p, true, std::nullopt, 1.0, std::nullopt, std::nullopt, std::nullopt);
  return {o.loss, o.stats.narrow(0, 0, 7), o.logp};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss_grad(
    const Tensor& logits, const Tensor& actions, const Tensor& logp_old, const Tensor& adv, const Maybe& legal,
    const Maybe& weight, const Maybe& ref_logits, const Maybe& ref_logp, double clip_low, double clip_high,
    double kl_coef, const Maybe& kl_coef_dev, double entropy_coef, const Maybe& entropy_coef_dev, double denominator,
    double grad_scale, const Maybe& grad_scale_dev, std::optional<at::ScalarType> grad_type, const Maybe& dlogits) {
  const at::NoGradGuard no_grad;
  const PolicyArgs p = policy_args(actions, logp_old, adv, legal, weight, ref_logits, ref_logp, clip_low, clip_high,
                                   kl_coef, kl_coef_dev, entropy_coef, entropy_coef_dev, denominator);
  if (there(dlogits) && grad_type && dlogits->scalar_type() != *grad_type)
    fail("policy_loss", "dlogits is not of grad_dtype");
  PolicyOut o = policy(logits, p, true, std::nullopt, grad_scale, grad_scale_dev, dlogits,
                       grad_type ? *grad_type : logits.scalar_type());
  return {o.loss, o.stats.narrow(0, 0, 7), o.logp, o.grad};
}

// ---- preference_loss ----------------------------------------------------------------------------

struct PreferenceOut {
  Tensor loss, margin, logp, accuracy, lse, d_logp;
};

PreferenceOut preference(const Tensor& logits, const Tensor& actions, const Tensor& offsets, const Tensor& ref_logp,
                         const Maybe& legal, const Maybe& weight, double beta, double smoothing, bool average,
                         bool grad) {
  const char* op = "preference_loss";
  primal_only(op, {&logits, &ref_logp, given(weight)});
  Scored s = score(op, logits, actions, legal, weight, false, true, grad);
  const int device = cuda_index(logits);
  const int64_t rows = logits.size(0);
  if (offsets.scalar_type() != at::kLong || offsets.dim() != 1 || offsets.size(0) % 2 != 1 ||
      !offsets.is_contiguous() || cuda_index(offsets) != device)
    fail(op, "offsets must be contiguous int64 [2 pairs + 1] on the logits' device");
  vector(op, "ref_logp", ref_logp, rows, at::kFloat, device);
  if (!(smoothing >= 0.0 && smoothing <= 1.0)) fail(op, "label_smoothing must lie in [0, 1]");
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  const auto fp32 = s.logp.options();
  const int64_t pairs = offsets.size(0) / 2, need = cugo_b200_preference_pairs_scratch_bytes(pairs);
  PreferenceOut o{at::empty({}, fp32),   at::empty({pairs}, fp32), at::empty({2 * pairs}, fp32),
                  at::empty({}, fp32), s.lse,                    s.zeros};
  Tensor scratch = bytes(need, fp32);
  check(cugo_b200_preference_pairs(s.logp.const_data_ptr<float>(), ref_logp.const_data_ptr<float>(), floats(weight),
                                   s.lse.const_data_ptr<float>(), offsets.const_data_ptr<int64_t>(), pairs, rows,
                                   static_cast<float>(beta), static_cast<float>(smoothing), average,
                                   out_floats(o.margin), out_floats(o.logp), out_floats(o.d_logp), out_floats(o.loss),
                                   out_floats(o.accuracy), scratch.mutable_data_ptr(), need, stream_of(device)),
        op);
  return o;
}

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& actions,
                               const Tensor& offsets, const Tensor& ref_logp, const Maybe& legal, const Maybe& weight,
                               double beta, double smoothing, bool average) {
    PreferenceOut o = preference(logits, actions, offsets, ref_logp, legal, weight, beta, smoothing, average, true);
    ctx->save_for_backward({logits, actions, legal.value_or(Tensor()), o.lse, o.d_logp});
    ctx->mark_non_differentiable({o.margin, o.logp, o.accuracy});
    ctx->set_materialize_grads(false);
    return {o.loss, o.margin, o.logp, o.accuracy};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("preference_loss");
    primal_only("preference_loss", {&grads[0]});
    variable_list d(9);
    if (grads[0].defined()) {
      const auto s = ctx->get_saved_variables();
      d[0] = score_backward("preference_loss", s[0], s[1], s[2], s[3], std::nullopt, s[4], std::nullopt, grads[0]);
    }
    return d;
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> preference_loss(const Tensor& logits, const Tensor& actions,
                                                           const Tensor& offsets, const Tensor& ref_logp,
                                                           const Maybe& legal, const Maybe& weight, double beta,
                                                           double smoothing, bool average) {
  if (differentiable(logits)) {
    const auto out =
        PreferenceLoss::apply(logits, actions, offsets, ref_logp, legal, weight, beta, smoothing, average);
    return {out[0], out[1], out[2], out[3]};
  }
  PreferenceOut o = preference(logits, actions, offsets, ref_logp, legal, weight, beta, smoothing, average, false);
  return {o.loss, o.margin, o.logp, o.accuracy};
}

// ---- adamw -------------------------------------------------------------------------------------------

using Tensors = std::vector<Tensor>;

// The memory of a call's tensor.
struct Span {
  const char *begin, *end;
  const char* name;
  bool written;
};

void check_list(const char* name, const Tensors& list, const std::vector<int64_t>& sizes,
                std::initializer_list<at::ScalarType> types, int device, bool written, std::vector<Span>& spans) {
  const char* op = "adamw";
  if (list.size() != sizes.size()) fail(op, "the lists must have one tensor each per parameter");
  for (size_t k = 0; k < list.size(); ++k) {
    const Tensor& t = list[k];
    if (t.numel() != sizes[k]) fail(op, std::string(name) + " have the wrong sizes");
    bool of_type = false;
    for (const at::ScalarType type : types) of_type = of_type || t.scalar_type() == type;
    if (!of_type || cuda_index(t) != device || !t.is_contiguous())
      fail(op, std::string(name) + " must be contiguous, of one type (" + c10::toString(*types.begin()) +
                   ") and on cuda:" + std::to_string(device));
    if (sizes[k]) {
      const char* const begin = static_cast<const char*>(t.const_data_ptr());
      spans.push_back({begin, begin + t.nbytes(), name, written});
    }
  }
}

// What is written is no other tensor of the call, in whole or in part.
void check_apart(std::vector<Span>& spans) {
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  const Span *last = nullptr, *last_written = nullptr;  // those so far that end last
  for (const Span& s : spans) {
    const Span* const other = s.written ? last : last_written;
    if (other && s.begin < other->end)
      fail("adamw", std::string("a tensor is in the call twice, or shares memory with another (in ") + other->name +
                        " and " + s.name + ")");
    if (!last || s.end > last->end) last = &s;
    if (s.written && (!last_written || s.end > last_written->end)) last_written = &s;
  }
}

Maybe adamw(const Tensors& params, const Tensors& grads, const Tensors& exp_avgs, const Tensors& exp_avg_sqs,
            Tensor step, double lr, const Maybe& lr_dev, double beta1, double beta2, double eps, double weight_decay,
            std::optional<double> max_grad_norm, int64_t seed, const std::optional<Tensors>& exp_avg_scales,
            const std::optional<Tensors>& exp_avg_sq_scales) {
  const char* op = "adamw";
  for (const Tensors* list : {&params, &grads, &exp_avgs, &exp_avg_sqs})
    for (const Tensor& t : *list) primal_only(op, {&t});
  primal_only(op, {given(lr_dev)});
  const auto range = [&](const char* name, double value, bool ok) {
    if (!ok) fail(op, std::string(name) + " = " + std::to_string(value) + " is out of range");
  };
  range("betas", beta1, beta1 >= 0.0 && beta1 < 1.0);
  range("betas", beta2, beta2 >= 0.0 && beta2 < 1.0);
  range("lr", lr, there(lr_dev) || lr >= 0.0);
  range("eps", eps, eps >= 0.0);
  range("weight_decay", weight_decay, weight_decay >= 0.0);
  if (max_grad_norm) range("max_grad_norm", *max_grad_norm, *max_grad_norm >= 0.0);
  const bool eight = exp_avg_scales.has_value();
  if (eight != exp_avg_sq_scales.has_value()) fail(op, "8-bit states need both lists of scales");
  const int device = cuda_index(step);
  if (device < 0 || step.scalar_type() != at::kLong || step.numel() != 1)
    fail(op, "step must be one int64 value on a CUDA device");
  const size_t n = params.size();
  at::ScalarType p_type = at::kFloat, g_type = at::kFloat;
  if (n) {
    p_type = params[0].scalar_type();
    if (!grads.empty()) g_type = grads[0].scalar_type();
    for (const at::ScalarType t : {p_type, g_type})
      if (t != at::kFloat && t != at::kBFloat16) fail(op, "parameters and gradients must be fp32 or bf16");
  }
  std::vector<int64_t> sizes(n), blocks(n);
  for (size_t k = 0; k < n; ++k) {
    sizes[k] = params[k].numel();
    blocks[k] = (sizes[k] + 255) / 256;
  }
  std::vector<Span> spans;
  spans.reserve(6 * n + 2);
  check_list("params", params, sizes, {p_type}, device, true, spans);
  check_list("grads", grads, sizes, {g_type}, device, false, spans);
  for (const auto& [name, list] : {std::pair<const char*, const Tensors&>{"exp_avgs", exp_avgs},
                                   std::pair<const char*, const Tensors&>{"exp_avg_sqs", exp_avg_sqs}}) {
    if (eight) check_list(name, list, sizes, {at::kByte, at::kFloat8_e4m3fn}, device, true, spans);
    else check_list(name, list, sizes, {at::kFloat}, device, true, spans);
  }
  if (eight) {
    check_list("exp_avg_scales", *exp_avg_scales, blocks, {at::kByte, at::kFloat8_e8m0fnu}, device, true, spans);
    check_list("exp_avg_sq_scales", *exp_avg_sq_scales, blocks, {at::kByte, at::kFloat8_e8m0fnu}, device, true, spans);
  }
  const float* lr_ptr = scalar(op, "lr", lr_dev, device);
  const auto one = [&](const char* name, const void* at, size_t size, bool written) {
    if (at) spans.push_back({static_cast<const char*>(at), static_cast<const char*>(at) + size, name, written});
  };
  one("step", step.const_data_ptr(), sizeof(int64_t), true);
  one("lr", lr_ptr, sizeof(float), false);
  check_apart(spans);
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  std::vector<void*> at[6];
  for (auto& a : at) a.resize(n);
  for (size_t k = 0; k < n; ++k) {
    at[0][k] = params[k].data_ptr();
    at[1][k] = grads[k].data_ptr();
    at[2][k] = exp_avgs[k].data_ptr();
    at[3][k] = exp_avg_sqs[k].data_ptr();
    if (eight) {
      at[4][k] = (*exp_avg_scales)[k].data_ptr();
      at[5][k] = (*exp_avg_sq_scales)[k].data_ptr();
    }
  }
  const auto fp32 = step.options().dtype(at::kFloat);
  Maybe norm;
  if (max_grad_norm) norm = at::empty({}, fp32);
  const int64_t need = cugo_b200_adamw_scratch_bytes(static_cast<int64_t>(n));
  Tensor scratch = bytes(need, fp32);
  check(cugo_b200_adamw(static_cast<int64_t>(n), at[0].data(), at[1].data(), at[2].data(), at[3].data(),
                        eight ? at[4].data() : nullptr, eight ? at[5].data() : nullptr, sizes.data(),
                        p_type == at::kFloat ? 0 : 1, g_type == at::kFloat ? 0 : 1, eight ? 8 : 32, lr, lr_ptr, beta1,
                        beta2, eps, weight_decay, max_grad_norm.value_or(0.0), static_cast<uint32_t>(seed),
                        step.data_ptr<int64_t>(), norm ? norm->mutable_data_ptr<float>() : nullptr,
                        scratch.mutable_data_ptr(), need, stream_of(device)),
        op);
  // The kernel writes behind torch's back: what goes by the tensors' versions (the networks'
  // bf16 weights, autograd's checks of saved tensors) has to see it.
  for (const Tensor& p : params)
    if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

PYBIND11_MODULE(_cugo_b200_update, m) {
  m.attr("built_for") = CUGO_BUILT_FOR;  // the build reads it in the file, before it is loaded
  m.def("action_logp", &action_logp);
  m.def("policy_loss", &policy_loss);
  m.def("policy_loss_grad", &policy_loss_grad);
  m.def("preference_loss", &preference_loss);
  m.def("adamw", &adamw);
}
