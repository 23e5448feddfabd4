// The learner's operations of the PyTorch-ROCm extension (policy_loss,
// advantages, adamw_step) over the C ABI of libcugo_hip.so.  Like the engine's operations they
// check their tensors, allocate outputs and scratch with torch, launch on the current stream
// under the tensors' device and never synchronise.
#include "ext_common.h"

#include <algorithm>
#include <cmath>
#include <string>

namespace cugo_ext {
namespace {

using Optional = c10::optional<torch::Tensor>;

int float_code(const torch::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return CUGO_DTYPE_F32;
    case at::kHalf:
      return CUGO_DTYPE_F16;
    case at::kBFloat16:
      return CUGO_DTYPE_BF16;
    default:
      TORCH_CHECK(false, name, " must be float32, float16 or bfloat16");
  }
}

// [n, A] whose rows are runs of memory, like logits' (their distance apart is free).
void check_rows(const torch::Tensor& t, const torch::Tensor& like, at::ScalarType dtype,
                const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 2 && t.sizes() == like.sizes() && t.scalar_type() == dtype, name,
              " must be a ", c10::toString(dtype), " tensor shaped like logits");
  TORCH_CHECK(t.size(1) == 1 || t.stride(1) == 1, name,
              " must have its last dimension contiguous");
  check_same_device(like, t, "logits", name);
}

void check_entry(const torch::Tensor& t, const torch::Tensor& like, at::ScalarType dtype,
                 const char* name) {
  check_1d(t, dtype, name);
  TORCH_CHECK(t.numel() == like.size(0), name, " must have one entry per row of logits");
  check_same_device(like, t, "logits", name);
}

const float* scalar_ptr(const Optional& t, const torch::Tensor& like, const char* name) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->is_cuda() && t->numel() == 1 && t->scalar_type() == at::kFloat, name,
              " must be a one-element float32 CUDA tensor");
  check_same_device(like, *t, "input", name);
  return t->data_ptr<float>();
}

// The tensors of a loss that are not differentiated, and its numbers.
struct LossInputs {
  torch::Tensor action, old_logp, advantage;
  Optional legal, ref_logits, returns, weight, scale;
  double clip_low, clip_high, kl_coef, entropy_coef, value_coef;
  bool want_logits, want_value;
};

// The loss as an operation of autograd: the forward pass has the gradients already
// (cugo_policy_loss), the backward pass hands them on, times the loss's own gradient.  They are
// given away, not kept: a second backward pass would find them scaled or accumulated into.
struct PolicyLossFn : public torch::autograd::Function<PolicyLossFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                torch::Tensor logits, Optional value,
                                                const LossInputs* in) {
    CugoPolicyLoss p{};
    p.n = logits.size(0);
    p.actions = logits.size(1);
    p.logits_dtype = float_code(logits, "logits");
    // tensors of their own, not parts of one, so that a loss may be divided in place
    const auto loss = torch::empty({}, on(logits, at::kFloat));
    const auto stats = torch::empty({6}, on(logits, at::kFloat));
    const auto logp = torch::empty({p.n}, on(logits, at::kFloat));
    const auto partials = torch::empty({CUGO_POLICY_LOSS_PARTIALS}, on(logits, at::kDouble));
    p.logits = logits.data_ptr();
    p.logits_stride = logits.stride(0);
    p.action = in->action.data_ptr<int64_t>();
    p.old_logp = in->old_logp.data_ptr<float>();
    p.advantage = in->advantage.data_ptr<float>();
    if (in->legal.has_value()) p.legal = u8p(*in->legal), p.legal_stride = in->legal->stride(0);
    if (in->ref_logits.has_value())
      p.ref_logits = in->ref_logits->data_ptr(), p.ref_stride = in->ref_logits->stride(0);
    if (value.has_value()) {
      p.value_dtype = float_code(*value, "value");
      p.value = value->data_ptr(), p.returns = in->returns->data_ptr<float>();
    }
    if (in->weight.has_value()) p.weight = in->weight->data_ptr<float>();
    p.scale = scalar_ptr(in->scale, logits, "scale");
    p.clip_low = in->clip_low, p.clip_high = in->clip_high, p.kl_coef = in->kl_coef;
    p.entropy_coef = in->entropy_coef, p.value_coef = in->value_coef;
    if (in->want_logits) {
      const auto d = torch::empty({p.n, p.actions}, on(logits, logits.scalar_type()));
      p.d_logits = d.data_ptr(), p.d_logits_stride = p.actions;
      ctx->saved_data["d_logits"] = d;
    }
    if (in->want_value) {
      const auto d = torch::empty({p.n}, on(logits, value->scalar_type()));
      p.d_value = d.data_ptr();
      ctx->saved_data["d_value"] = d;
    }
    p.logp = logp.data_ptr<float>();
    p.loss = loss.data_ptr<float>();
    p.stats = stats.data_ptr<float>();
    p.partials = partials.data_ptr<double>();
    check_call(cugo_policy_loss(&p, stream()), "policy_loss");
    ctx->mark_non_differentiable({stats, logp});
    ctx->set_materialize_grads(false);
    return {loss, stats, logp};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "policy_loss can be differentiated once");
    TORCH_CHECK(!ctx->saved_data.empty(),
                "policy_loss hands its gradients out once; compute the loss again for a second "
                "backward pass");
    const auto take = [&](const char* name) {
      const auto at = ctx->saved_data.find(name);
      return at == ctx->saved_data.end() ? torch::Tensor() : at->second.toTensor();
    };
    const torch::Tensor d_logits = take("d_logits"), d_value = take("d_value");
    ctx->saved_data.clear();
    if (!grads[0].defined()) return {torch::Tensor(), torch::Tensor(), torch::Tensor()};
    const DeviceGuard guard(grads[0].device());
    const auto code = [](const torch::Tensor& t) {
      return t.defined() ? float_code(t, "gradients") : CUGO_DTYPE_F32;
    };
    const auto pointer = [](const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    const auto size = [](const torch::Tensor& t) { return t.defined() ? t.numel() : 0; };
    check_call(cugo_scale_gradients(code(d_logits), pointer(d_logits), size(d_logits),
                                    code(d_value), pointer(d_value), size(d_value),
                                    grads[0].data_ptr<float>(), stream()),
               "scale_gradients");
    return {d_logits, d_value, torch::Tensor()};
  }
};

// -> (loss f32 scalar, differentiable in logits and value; stats f32 [6]: policy, value, kl,
// entropy, cut, drift; logp f32 [n]), cugo_policy_loss.
std::vector<torch::Tensor> policy_loss(torch::Tensor logits, torch::Tensor action,
                                       torch::Tensor old_logp, torch::Tensor advantage,
                                       Optional legal, Optional ref_logits, Optional value,
                                       Optional returns, Optional weight, double clip_low,
                                       double clip_high, double kl_coef, double entropy_coef,
                                       double value_coef, Optional scale) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) >= 1, "logits must have shape [n, A], A >= 1");
  TORCH_CHECK(logits.size(1) <= (1 << 30), "at most 2^30 actions");
  float_code(logits, "logits");
  check_rows(logits, logits, logits.scalar_type(), "logits");
  check_entry(action, logits, at::kLong, "action");
  check_entry(old_logp, logits, at::kFloat, "old_logp");
  check_entry(advantage, logits, at::kFloat, "advantage");
  if (legal.has_value()) check_rows(*legal, logits, at::kBool, "legal");
  if (ref_logits.has_value()) check_rows(*ref_logits, logits, logits.scalar_type(), "ref_logits");
  TORCH_CHECK(value.has_value() == returns.has_value(), "value and returns go together");
  if (value.has_value()) {
    float_code(*value, "value");
    check_entry(*value, logits, value->scalar_type(), "value");
    check_entry(*returns, logits, at::kFloat, "returns");
  }
  if (weight.has_value()) check_entry(*weight, logits, at::kFloat, "weight");
  TORCH_CHECK(clip_low >= 0 && clip_high >= 0, "the clip's sides must not be negative");
  TORCH_CHECK(std::isfinite(kl_coef) && std::isfinite(entropy_coef) && std::isfinite(value_coef),
              "the coefficients must be finite");
  scalar_ptr(scale, logits, "scale");
  const DeviceGuard guard(logits.device());
  // rows too far apart for 32-bit offsets are copied together
  const auto near = [](const torch::Tensor& t) {
    return t.size(1) > 1024 || t.stride(0) < (1 << 24) ? t : t.contiguous();
  };
  logits = near(logits);
  if (legal.has_value()) legal = near(*legal);
  if (ref_logits.has_value()) ref_logits = near(*ref_logits);
  const bool grad = at::GradMode::is_enabled();
  const LossInputs in{action,   old_logp,  advantage, legal,   ref_logits,   returns,    weight,
                      scale,    clip_low,  clip_high, kl_coef, entropy_coef, value_coef,
                      grad && logits.requires_grad(),
                      grad && value.has_value() && value->requires_grad()};
  return PolicyLossFn::apply(logits, value, &in);
}

// The memory that calls write and read, and whether what one writes overlaps any other part.
class Spans {
 public:
  explicit Spans(size_t expected = 8) { spans_.reserve(expected); }
  void add(const torch::Tensor& t, bool written) {
    const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
    if (t.numel() > 0) spans_.push_back({at, at + t.nbytes(), written});
  }
  bool overlap() {
    std::sort(spans_.begin(), spans_.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
    uintptr_t any = 0, written = 0;  // the furthest ends so far
    for (const Span& s : spans_) {
      if (s.from < (s.written ? any : written)) return true;
      any = std::max(any, s.to);
      if (s.written) written = std::max(written, s.to);
    }
    return false;
  }

 private:
  struct Span {
    uintptr_t from, to;
    bool written;
  };
  std::vector<Span> spans_;
};

// -> (advantage f32 [T, B], returns f32 [T, B]), cugo_advantages.
std::vector<torch::Tensor> advantages(torch::Tensor reward, torch::Tensor value,
                                      torch::Tensor done, torch::Tensor bootstrap, double gamma,
                                      double lam, Optional player, Optional last_player,
                                      Optional advantage, Optional returns) {
  TORCH_CHECK(reward.is_cuda() && reward.is_contiguous() && reward.dim() == 2 &&
                  reward.scalar_type() == at::kFloat,
              "reward must be a contiguous CUDA float32 [steps, batch] tensor");
  const int64_t steps = reward.size(0), batch = reward.size(1);
  const auto check = [&](const torch::Tensor& t, at::IntArrayRef shape, at::ScalarType dtype,
                         const char* name) {
    TORCH_CHECK(t.is_contiguous() && t.sizes() == shape && t.scalar_type() == dtype, name,
                " must be a contiguous ", c10::toString(dtype), " tensor of shape ", shape);
    check_same_device(reward, t, "reward", name);
  };
  const int code = float_code(value, "value");
  check(value, {steps, batch}, value.scalar_type(), "value");
  check(done, {steps, batch}, at::kBool, "done");
  check(bootstrap, {batch}, value.scalar_type(), "bootstrap");
  TORCH_CHECK(player.has_value() == last_player.has_value(), "player and last_player go together");
  if (player.has_value()) {
    check(*player, {steps, batch}, at::kByte, "player");
    check(*last_player, {batch}, at::kByte, "last_player");
  }
  TORCH_CHECK(gamma >= 0 && gamma <= 1 && lam >= 0 && lam <= 1, "gamma and lam must lie in [0, 1]");
  const DeviceGuard guard(reward.device());
  auto adv = out_or_new(advantage, {steps, batch}, at::kFloat, reward, "advantage");
  auto ret = out_or_new(returns, {steps, batch}, at::kFloat, reward, "returns");
  Spans spans;
  for (const auto* t : {&reward, &value, &done, &bootstrap}) spans.add(*t, false);
  if (player.has_value()) spans.add(*player, false), spans.add(*last_player, false);
  spans.add(adv, true), spans.add(ret, true);
  TORCH_CHECK(!spans.overlap(), "advantage and returns must not overlap the inputs or each other");
  const int64_t bytes = cugo_advantages_workspace(steps, batch);
  const auto scratch = torch::empty({bytes}, on(reward, at::kByte));
  check_call(cugo_advantages(code, reward.data_ptr<float>(), value.data_ptr(), u8p(done),
                             player.has_value() ? u8p(*player) : nullptr, bootstrap.data_ptr(),
                             player.has_value() ? u8p(*last_player) : nullptr, steps, batch,
                             gamma, lam, adv.data_ptr<float>(), ret.data_ptr<float>(),
                             bytes ? scratch.data_ptr() : nullptr, bytes, stream()),
             "advantages");
  return {adv, ret};
}

// A Python list of tensors (None where `optional`), read in place: converting one into a vector of
// tensors takes as long as launching a kernel for a model's parameters and their states.
class TensorList {
 public:
  TensorList(const pybind11::handle& list, const char* name, bool optional) {
    TORCH_CHECK(PyList_Check(list.ptr()), name, " must be a list of tensors");
    const Py_ssize_t n = PyList_GET_SIZE(list.ptr());
    items_.reserve((size_t)n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* item = PyList_GET_ITEM(list.ptr(), i);
      if (optional && item == Py_None) {
        items_.push_back(nullptr);
        continue;
      }
      TORCH_CHECK(THPVariable_Check(item), name, " must be a list of tensors");
      items_.push_back(&THPVariable_Unpack(item));
    }
  }
  size_t size() const { return items_.size(); }
  bool has(size_t i) const { return items_[i] != nullptr; }
  const torch::Tensor& operator[](size_t i) const { return *items_[i]; }

 private:
  std::vector<const torch::Tensor*> items_;
};

// One step of every tensor with a gradient, in place (cugo_adamw); the gradients' norm with
// max_norm, else None.
Optional adamw_step(const pybind11::list& params_list, const pybind11::list& grads_list,
                    const pybind11::list& exp_avg_list, const pybind11::list& exp_avg_sq_list,
                    torch::Tensor steps, const std::vector<double>& lr,
                    const std::vector<double>& weight_decay, double beta1, double beta2, double eps,
                    c10::optional<double> max_norm, const pybind11::object& master_list,
                    const pybind11::object& exp_avg_scale_list,
                    const pybind11::object& exp_avg_sq_scale_list, Optional lr_scale,
                    int64_t seed) {
  const TensorList params(params_list, "params", false), grads(grads_list, "grads", true);
  const TensorList exp_avg(exp_avg_list, "exp_avg", false);
  const TensorList exp_avg_sq(exp_avg_sq_list, "exp_avg_sq", false);
  const pybind11::list none;
  const bool masters = !master_list.is_none(), eight = !exp_avg_scale_list.is_none();
  TORCH_CHECK(exp_avg_sq_scale_list.is_none() != eight, "both moments have scales, or neither");
  const TensorList master(masters ? master_list : none, "master", true);
  const TensorList exp_avg_scale(eight ? exp_avg_scale_list : none, "exp_avg_scale", false);
  const TensorList exp_avg_sq_scale(eight ? exp_avg_sq_scale_list : none, "exp_avg_sq_scale", false);
  const size_t count = params.size();
  TORCH_CHECK(count > 0, "no parameters");
  TORCH_CHECK(grads.size() == count && exp_avg.size() == count && exp_avg_sq.size() == count &&
                  lr.size() == count && weight_decay.size() == count,
              "grads, exp_avg, exp_avg_sq, lr and weight_decay must have one entry per parameter");
  TORCH_CHECK(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "betas must lie in [0, 1)");
  TORCH_CHECK(eps >= 0, "eps must not be negative");
  TORCH_CHECK(!max_norm.has_value() || *max_norm > 0, "max_norm must be positive");
  TORCH_CHECK(!eight || (exp_avg_scale.size() == count && exp_avg_sq_scale.size() == count),
              "the scales must have one entry per parameter");
  TORCH_CHECK(!masters || master.size() == count, "master must have one entry per parameter");
  const torch::Tensor& first = params[0];
  TORCH_CHECK(first.is_cuda(), "parameters must be CUDA tensors");
  check_1d(steps, at::kLong, "steps");
  TORCH_CHECK((size_t)steps.numel() == count, "steps must have one entry per parameter");
  check_same_device(first, steps, "parameters", "steps");
  const auto dense = [&](const torch::Tensor& t, const torch::Tensor& like, at::ScalarType dtype,
                         const char* name) {
    TORCH_CHECK(t.is_contiguous() && t.numel() == like.numel() && t.scalar_type() == dtype, name,
                " must be contiguous ", c10::toString(dtype), " of the parameter's size");
    check_same_device(first, t, "parameters", name);
  };
  std::vector<CugoAdamwTensor> list;
  Spans spans(7 * count);
  list.reserve(count);
  const auto written = [&](const torch::Tensor& t) { spans.add(t, true); };
  for (size_t i = 0; i < count; ++i) {
    const torch::Tensor& w = params[i];
    CugoAdamwTensor t{};
    t.param_dtype = (int16_t)float_code(w, "parameters");
    dense(w, w, w.scalar_type(), "parameters");
    const torch::Tensor* m32 = masters && master.has(i) ? &master[i] : nullptr;
    const bool wide = w.scalar_type() == at::kFloat;
    TORCH_CHECK(wide || m32, "a 16-bit parameter needs its float32 master");
    TORCH_CHECK(!wide || !m32, "a float32 parameter has no master");
    if (m32) dense(*m32, w, at::kFloat, "master");
    dense(exp_avg[i], w, eight ? at::kFloat8_e4m3fn : at::kFloat, "exp_avg");
    dense(exp_avg_sq[i], w, eight ? at::kFloat8_e5m2 : at::kFloat, "exp_avg_sq");
    if (eight) {
      const int64_t blocks = (w.numel() + CUGO_ADAMW_BLOCK - 1) / CUGO_ADAMW_BLOCK;
      for (const auto* s : {&exp_avg_scale[i], &exp_avg_sq_scale[i]}) {
        check_1d(*s, at::kFloat, "scales");
        TORCH_CHECK(s->numel() == blocks, "scales must have one entry per block of ",
                    CUGO_ADAMW_BLOCK, " values");
        check_same_device(first, *s, "parameters", "scales");
      }
    }
    if (!grads.has(i)) continue;  // left as it is
    const torch::Tensor& g = grads[i];
    t.grad_dtype = (int16_t)float_code(g, "gradients");
    dense(g, w, g.scalar_type(), "gradients");
    TORCH_CHECK(w.numel() <= (int64_t)1 << 36, "at most 2^36 values a parameter");
    spans.add(g, false);
    written(w), written(exp_avg[i]), written(exp_avg_sq[i]);
    if (m32) written(*m32);
    if (eight) written(exp_avg_scale[i]), written(exp_avg_sq_scale[i]);
    t.param = w.data_ptr();
    t.grad = g.data_ptr();
    t.master = m32 ? m32->data_ptr<float>() : nullptr;
    t.exp_avg = exp_avg[i].data_ptr();
    t.exp_avg_sq = exp_avg_sq[i].data_ptr();
    if (eight) {
      t.exp_avg_scale = exp_avg_scale[i].data_ptr<float>();
      t.exp_avg_sq_scale = exp_avg_sq_scale[i].data_ptr<float>();
    }
    t.step = steps.data_ptr<int64_t>() + i;
    t.numel = w.numel();
    t.lr = lr[i], t.weight_decay = weight_decay[i];
    t.place = (int32_t)i;
    list.push_back(t);
  }
  spans.add(steps, true);
  TORCH_CHECK(!spans.overlap(), "parameters, gradients and states must not overlap in memory");
  const DeviceGuard guard(first.device());
  Optional norm;
  if (max_norm.has_value())
    norm = list.empty() ? torch::zeros({}, on(first, at::kFloat))
                        : torch::empty({}, on(first, at::kFloat));
  const int64_t bytes = cugo_adamw_workspace((int64_t)list.size());
  const auto scratch = torch::empty({bytes}, on(first, at::kByte));
  check_call(cugo_adamw(list.data(), (int64_t)list.size(), eight ? 8 : 32, beta1, beta2, eps,
                        scalar_ptr(lr_scale, first, "lr_scale"), max_norm.value_or(0.0),
                        (uint64_t)seed, norm.has_value() ? norm->data_ptr<float>() : nullptr,
                        bytes ? scratch.data_ptr() : nullptr, bytes, stream()),
             "adamw_step");
  // what keeps a copy of a parameter by its version (seq_decode's packed weights) sees the change
  for (size_t i = 0; i < count; ++i)
    if (grads.has(i)) params[i].unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

void bind_learner(pybind11::module_& m) {
  namespace py = pybind11;
  m.attr("ADAMW_BLOCK") = py::int_(CUGO_ADAMW_BLOCK);
  m.def("policy_loss", &policy_loss,
        "The clipped policy loss with KL, entropy and value terms: (loss, stats, logp)",
        py::arg("logits"), py::arg("action"), py::arg("old_logp"), py::arg("advantage"),
        py::arg("legal") = py::none(), py::arg("ref_logits") = py::none(),
        py::arg("value") = py::none(), py::arg("returns") = py::none(),
        py::arg("weight") = py::none(), py::arg("clip_low") = 0.2, py::arg("clip_high") = 0.2,
        py::arg("kl_coef") = 0.0, py::arg("entropy_coef") = 0.0, py::arg("value_coef") = 0.5,
        py::arg("scale") = py::none());
  m.def("advantages", &advantages,
        "Generalised advantage estimation over [steps, batch] of two-player games",
        py::arg("reward"), py::arg("value"), py::arg("done"), py::arg("bootstrap"),
        py::arg("gamma"), py::arg("lam"), py::arg("player") = py::none(),
        py::arg("last_player") = py::none(), py::arg("advantage") = py::none(),
        py::arg("returns") = py::none());
  m.def("adamw_step", &adamw_step, "One AdamW step over many tensors, in place",
        py::arg("params"), py::arg("grads"), py::arg("exp_avg"), py::arg("exp_avg_sq"),
        py::arg("steps"), py::arg("lr"), py::arg("weight_decay"), py::arg("beta1"),
        py::arg("beta2"), py::arg("eps"), py::arg("max_norm") = py::none(),
        py::arg("master") = py::none(), py::arg("exp_avg_scale") = py::none(),
        py::arg("exp_avg_sq_scale") = py::none(), py::arg("lr_scale") = py::none(),
        py::arg("seed") = 0);
}

}  // namespace cugo_ext
