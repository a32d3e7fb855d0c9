// mev_torch.cpp -- binding of the policy operators (mev.h) to torch: argument checks, buffers from
// torch's allocator, the current stream, and the loss as an autograd node. It calls libmev.so
// through the entry points that Python hands it (bind), so both see one library. Compiled, because
// a small policy's update is launch-bound: one loss with its gradient takes 50 us, most
// of them torch.autograd.grad's own (56 us as an autograd Function, 153 us from Python code); an
// action's log-probability 7 us (19 us).
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <ATen/SavedTensorHooks.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <limits>
#include <memory>
#include <mutex>
#include <optional>
#include <tuple>
#include <vector>

#include "mev.h"

namespace {

using at::Tensor;
using std::optional;

#ifndef MEV_SRC_HASH
#define MEV_SRC_HASH "unknown"
#endif

struct Entries {
  decltype(&mev_policy_workspace) policy_workspace = nullptr;
  decltype(&mev_policy_rows) policy_rows = nullptr;
  decltype(&mev_advantages_workspace) advantages_workspace = nullptr;
  decltype(&mev_advantages_run) advantages_run = nullptr;
  decltype(&mev_clip_norm_workspace) clip_norm_workspace = nullptr;
  decltype(&mev_clip_norm) clip_norm = nullptr;
  decltype(&mev_strerror) strerror = nullptr;
} mev;

void bind(const std::vector<uintptr_t>& p) {
  TORCH_CHECK_VALUE(p.size() == 7, "seven entry points");
  mev.policy_workspace = reinterpret_cast<decltype(mev.policy_workspace)>(p[0]);
  mev.policy_rows = reinterpret_cast<decltype(mev.policy_rows)>(p[1]);
  mev.advantages_workspace = reinterpret_cast<decltype(mev.advantages_workspace)>(p[2]);
  mev.advantages_run = reinterpret_cast<decltype(mev.advantages_run)>(p[3]);
  mev.clip_norm_workspace = reinterpret_cast<decltype(mev.clip_norm_workspace)>(p[4]);
  mev.clip_norm = reinterpret_cast<decltype(mev.clip_norm)>(p[5]);
  mev.strerror = reinterpret_cast<decltype(mev.strerror)>(p[6]);
}

void check(int64_t code, const char* where) {
  TORCH_CHECK(code >= 0, where, " failed (", code, "): ", mev.strerror((int)code));
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// The capture that the current stream of t's device is in (0: none; the default stream never is).
int64_t capture_of(const Tensor& t) {
  const hipStream_t stream = (hipStream_t)stream_of(t);
  if (!stream) return 0;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  const hipError_t e = hipStreamGetCaptureInfo(stream, &status, &id);
  TORCH_CHECK(e == hipSuccess, "hipStreamGetCaptureInfo failed: ", hipGetErrorString(e));
  return status == hipStreamCaptureStatusNone ? 0 : (int64_t)id + 1;
}

int32_t dtype_code(at::ScalarType t) {
  return t == at::kFloat ? MEV_F32 : t == at::kBFloat16 ? MEV_BF16 : t == at::kHalf ? MEV_F16 : -1;
}

void dense(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && !t.is_neg(), name, " must be a dense tensor");
}

void on_gpu(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must live on a ROCm GPU (no CPU fallback)");
}

void data_only(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(!(t.requires_grad() && at::GradMode::is_enabled()), name,
                    " is data: no gradient reaches it (detach it)");
}

// A tangent on any input: the result would carry none, which autograd reads as a derivative of zero.
template <class... T>
void no_tangent(const char* op, const T&... inputs) {
  const auto has = [](const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); };
  TORCH_CHECK(!(has(inputs) || ...), op, " has no forward-mode derivative");
}

// The launches are no operations of torch's: a tracer would record the buffers without what fills
// them. Refused under one, and for tensors without memory of their own (functorch's wrappers, fake
// tensors and other __torch_dispatch__ subclasses).
template <class... T>
void not_traced(const char* op, const T&... inputs) {
  using Mode = c10::impl::TorchDispatchModeKey;
  const auto active = [](Mode m) {
    return c10::impl::TorchDispatchModeTLS::get_mode(m).has_value();
  };
  const bool traced = torch::jit::tracer::isTracing() ||
                      (c10::impl::TorchDispatchModeTLS::any_modes_set() &&
                       (active(Mode::PROXY) || active(Mode::FAKE) || active(Mode::FUNCTIONAL))) ||
                      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
  const auto bare = [](const Tensor& t) {
    return t.defined() && t.layout() == at::kStrided &&
           (!t.has_storage() || t.key_set().has(c10::DispatchKey::Python) ||
            t.key_set().has(c10::DispatchKey::Functionalize));
  };
  TORCH_CHECK(!traced && !(bare(inputs) || ...), op,
              " cannot be traced or transformed: call it outside (torch.compiler.disable)");
}

constexpr double kFloatMax = std::numeric_limits<float>::max();  // (float32 in the kernels)

double number(double v, const char* name, double lo, double hi) {
  TORCH_CHECK_VALUE(std::isfinite(v) && v >= lo && v <= hi, name, " must be finite and lie in [",
                    lo, ", ", hi, "], got ", v);
  return v;
}

// -- policy rows ---------------------------------------------------------------------------------
void check_logits(const Tensor& x) {
  dense(x, "logits");
  TORCH_CHECK_TYPE(dtype_code(x.scalar_type()) >= 0,
                   "logits must be float32, bfloat16 or float16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < (int64_t(1) << 31),
                    "logits must be [..., actions] with 1 to 2^31 - 1 actions, got ", x.sizes());
}

void like(const Tensor& t, const char* name, const Tensor& x) {
  dense(t, name);
  TORCH_CHECK_VALUE(t.sizes() == x.sizes().slice(0, x.dim() - 1), name,
                    " must have the logits' leading shape ", x.sizes().slice(0, x.dim() - 1),
                    ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", the logits are on ",
                    x.device());
}

Tensor check_action(const Tensor& a, const Tensor& x) {
  TORCH_CHECK_TYPE(a.scalar_type() == at::kInt || a.scalar_type() == at::kLong,
                   "action must be int32 or int64, got ", a.scalar_type());
  like(a, "action", x);
  return a.contiguous();
}

// One float32 number a row: data of the loss, never differentiated.
Tensor check_row(const optional<Tensor>& t, const char* name, const Tensor& x) {
  if (!t || !t->defined()) return Tensor();
  TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, name, " must be float32, got ",
                   t->scalar_type());
  like(*t, name, x);
  data_only(*t, name);
  return t->requires_grad() ? t->detach().contiguous() : t->contiguous();
}

// The leading axes of logits as rows in at most two strides (mev_policy): adjacent axes merged.
// False where they need more, or where a row's elements are not adjacent.
bool rows_of(const Tensor& x, mev_policy* p) {
  const int64_t V = x.size(-1);
  if (x.stride(-1) != 1 && V > 1) return false;
  int64_t size[2] = {1, 1}, stride[2] = {0, 0}, rows = 1;
  int n = 0;
  for (int64_t i = x.dim() - 2; i >= 0; --i) {
    const int64_t k = x.size(i), s = x.stride(i);
    rows *= k;
    if (k == 1) continue;
    if (n > 0 && s == size[n - 1] * stride[n - 1]) {
      size[n - 1] *= k;
    } else {
      if (n == 2) return false;
      size[n] = k;
      stride[n++] = s;
    }
  }
  p->rows = rows;
  p->inner = size[0] > 0 ? size[0] : 1;
  p->inner_stride = stride[0];
  p->outer_stride = stride[1];
  return true;
}

struct Coefs {
  double clip_low = 0.0, clip_high = 0.0, kl = 0.0, entropy = 0.0;
};

template <class T>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

struct Rows {  // what a launch forms; undefined: not asked
  Tensor loss, logp, entropy, grad;
};

// What is not differentiated; undefined tensors: not given.
struct Side {
  Tensor action, old_logp, advantage, weight, ref_logp;
  Coefs c;
};

// The logits as rows_of has them, copied where they are not.
Tensor as_rows(const Tensor& logits) {
  mev_policy a{};
  return rows_of(logits, &a) ? logits : logits.detach().contiguous();
}

// x: of as_rows
void launch_rows(const Tensor& x, const Side& in, const Rows& out, const Tensor& grad_scale,
                 bool skip_unit) {
  mev_policy a{};
  Tensor work;
  TORCH_INTERNAL_ASSERT(rows_of(x, &a));
  a.logits = x.const_data_ptr();
  a.action = in.action.const_data_ptr();
  a.old_logp = ptr<float>(in.old_logp);
  a.advantage = ptr<float>(in.advantage);
  a.weight = ptr<float>(in.weight);
  a.ref_logp = ptr<float>(in.ref_logp);
  a.logp = ptr<float>(out.logp);
  a.entropy = ptr<float>(out.entropy);
  a.loss = ptr<float>(out.loss);
  a.grad = ptr<void>(out.grad);
  a.grad_scale = ptr<float>(grad_scale);
  a.actions = (int32_t)x.size(-1);
  a.dtype = dtype_code(x.scalar_type());
  a.action_bytes = (int32_t)in.action.element_size();
  a.skip_unit_scale = skip_unit;
  a.clip_low = in.c.clip_low;
  a.clip_high = in.c.clip_high;
  a.kl_coef = in.c.kl;
  a.entropy_coef = in.c.entropy;
  const int64_t need = mev.policy_workspace(&a);
  check(need, "mev_policy_workspace");
  if (need > 0) {
    work = at::empty({need}, x.options().dtype(at::kByte));
    a.workspace = work.data_ptr();
    a.workspace_bytes = need;
  }
  check(mev.policy_rows(&a, stream_of(x)), "mev_policy_rows");
}

Tensor row_output(const Tensor& x) {
  return at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
}

Rows row_outputs(const Tensor& x, bool loss) {
  Rows r;
  r.logp = row_output(x);
  r.entropy = row_output(x);
  if (loss) r.loss = at::empty({}, x.options().dtype(at::kFloat));
  return r;
}

std::tuple<Tensor, Tensor> action_logp(const Tensor& logits, const Tensor& action) {
  not_traced("action_logp", logits, action);
  check_logits(logits);
  const Tensor act = check_action(action, logits);
  no_tangent("action_logp", logits);
  on_gpu(logits, "logits");
  const c10::DeviceGuard guard(logits.device());
  const at::NoGradGuard no_grad;
  const Rows r = row_outputs(logits, false);
  Side in;
  in.action = act;
  launch_rows(as_rows(logits), in, r, Tensor(), false);
  return {r.logp, r.entropy};
}

// The forward launch forms the gradient for an incoming gradient of one from the row it has at
// hand (one pass over the logits for both); the backward launch finds that on the device and
// leaves it, or forms it anew with the incoming gradient. Under saved-tensor hooks, which are
// there to hold less until the backward pass (offloading, recomputation), only that one forms it.
struct PolicyLossBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable logits, action, old_logp, advantage, weight, ref_logp;
  Coefs c;
  Tensor formed;        // by the forward pass; handed out once
  int64_t capture = 0;  // that the forward pass was in

  torch::autograd::variable_list apply(torch::autograd::variable_list&& g) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list out(1);
    if (!g[0].defined()) return out;
    TORCH_CHECK(!at::GradMode::is_enabled(), "policy_loss is differentiable once");
    // looked at again: saved-tensor hooks give back what they like
    const Tensor x = as_rows(logits.unpack());
    check_logits(x);
    on_gpu(x, "logits");
    const Side in{check_action(action.unpack(), x),
                  check_row(old_logp.unpack(), "old_logp", x),
                  check_row(advantage.unpack(), "advantage", x),
                  check_row(weight.unpack(), "weight", x),
                  check_row(ref_logp.unpack(), "ref_logp", x),
                  c};
    TORCH_CHECK(in.old_logp.defined() && in.advantage.defined() &&
                    (!formed.defined() || (formed.sizes() == x.sizes() &&
                                           formed.scalar_type() == x.scalar_type())),
                "a saved tensor came back as another");
    const c10::DeviceGuard guard(x.device());
    // A second backward over a retained graph forms its own gradient, and so does one that is not
    // captured (or eager) together with its forward pass: either may be replayed alone, the forward
    // pass over a gradient that was handed out, the backward pass over one that was scaled.
    const bool mine = formed.defined() && capture == capture_of(x);
    Rows r;
    r.grad = mine ? std::move(formed) : at::empty(x.sizes(), x.options());
    launch_rows(x, in, r, g[0], mine);
    out[0] = std::move(r.grad);
    return out;
  }

  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (auto* v : {&logits, &action, &old_logp, &advantage, &weight, &ref_logp}) v->reset_data();
    formed.reset();
  }

  std::string name() const override { return "PolicyLossBackward"; }
};

std::tuple<Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& action,
                                               const Tensor& old_logp, const Tensor& advantage,
                                               const optional<Tensor>& weight,
                                               const optional<Tensor>& ref_logp, double clip_low,
                                               double clip_high, double kl_coef,
                                               double entropy_coef) {
  not_traced("policy_loss", logits, action, old_logp, advantage, weight ? *weight : logits,
             ref_logp ? *ref_logp : logits);
  check_logits(logits);
  const Side in{check_action(action, logits),
                check_row(old_logp, "old_logp", logits),
                check_row(advantage, "advantage", logits),
                check_row(weight, "weight", logits),
                check_row(ref_logp, "ref_logp", logits),
                Coefs{number(clip_low, "clip_low", 0.0, 1.0),
                      number(clip_high, "clip_high", 0.0, INFINITY),
                      number(kl_coef, "kl_coef", -kFloatMax, kFloatMax),
                      number(entropy_coef, "entropy_coef", -kFloatMax, kFloatMax)}};
  no_tangent("policy_loss", logits, old_logp, advantage, weight ? *weight : logits,
             ref_logp ? *ref_logp : logits);
  on_gpu(logits, "logits");
  const c10::DeviceGuard guard(logits.device());
  if (logits.requires_grad() && at::GradMode::is_enabled()) {
    const std::shared_ptr<PolicyLossBackward> node(new PolicyLossBackward(),
                                                   torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    const Tensor x = as_rows(logits);
    Rows r;
    {
      const at::NoGradGuard no_grad;
      r = row_outputs(logits, true);
      if (at::SavedTensorDefaultHooks::get_tls_state().stack.empty())
        r.grad = at::empty(logits.sizes(), logits.options());
      launch_rows(x, in, r, Tensor(), false);
    }
    const auto save = [](const Tensor& t) { return torch::autograd::SavedVariable(t, false); };
    node->logits = save(x);  // (a copy that was made serves the backward pass too)
    node->action = save(in.action);
    node->old_logp = save(in.old_logp);
    node->advantage = save(in.advantage);
    node->weight = save(in.weight);
    node->ref_logp = save(in.ref_logp);
    node->c = in.c;
    node->formed = std::move(r.grad);
    node->capture = capture_of(logits);
    torch::autograd::set_history(r.loss, node);
    return {r.loss, r.logp, r.entropy};
  }
  const Rows r = row_outputs(logits, true);
  launch_rows(as_rows(logits), in, r, Tensor(), false);
  return {r.loss, r.logp, r.entropy};
}

// -- advantages ----------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> advantages(const Tensor& reward, const Tensor& done, const Tensor& value,
                                      const Tensor& last_value, double gamma, double lam,
                                      bool bootstrap_done) {
  not_traced("advantages", reward, done, value, last_value);
  TORCH_CHECK_TYPE(reward.scalar_type() == at::kFloat, "reward must be float32, got ",
                   reward.scalar_type());
  TORCH_CHECK_TYPE(done.scalar_type() == at::kByte || done.scalar_type() == at::kBool,
                   "done must be uint8 or bool, got ", done.scalar_type());
  TORCH_CHECK_TYPE(dtype_code(value.scalar_type()) >= 0 &&
                       last_value.scalar_type() == value.scalar_type(),
                   "value and last_value must both be float32, bfloat16 or float16, got ",
                   value.scalar_type(), " and ", last_value.scalar_type());
  TORCH_CHECK_VALUE(reward.dim() == 2 || reward.dim() == 3,
                    "reward must be [T, E] or [T, E, U], got ", reward.sizes());
  const auto shape = reward.sizes();
  const auto same = [&](const Tensor& t, const char* name, at::IntArrayRef want) {
    dense(t, name);
    TORCH_CHECK_VALUE(t.sizes() == want, name, " must be ", want, ", got ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == reward.device(), name, " is on ", t.device(), ", reward on ",
                      reward.device());
    data_only(t, name);
  };
  same(reward, "reward", shape);
  same(value, "value", shape);
  same(done, "done", shape.slice(0, 2));
  same(last_value, "last_value", shape.slice(1));
  number(gamma, "gamma", 0.0, 1.0);
  number(lam, "lam", 0.0, 1.0);
  no_tangent("advantages", reward, value, last_value);
  on_gpu(reward, "reward");
  const c10::DeviceGuard guard(reward.device());
  const bool per_ue = reward.dim() == 3;
  const Tensor adv = at::empty(shape, reward.options()), ret = at::empty(shape, reward.options());
  mev_advantages a{};
  a.reward = static_cast<const float*>(reward.const_data_ptr());
  a.value = value.const_data_ptr();
  a.last_value = last_value.const_data_ptr();
  a.done = static_cast<const uint8_t*>(done.const_data_ptr());
  a.advantage = ptr<float>(adv);
  a.returns = ptr<float>(ret);
  a.T = shape[0];
  a.E = shape[1];
  a.U = per_ue ? shape[2] : 1;
  for (int i = 0; i < (per_ue ? 3 : 2); ++i) {
    a.reward_stride[i] = reward.stride(i);
    a.value_stride[i] = value.stride(i);
    if (i < 2) a.done_stride[i] = done.stride(i);
    if (i > 0) a.last_stride[i - 1] = last_value.stride(i - 1);
  }
  a.value_dtype = dtype_code(value.scalar_type());
  a.bootstrap_done = bootstrap_done;
  a.gamma = (float)gamma;
  a.lam = (float)lam;
  Tensor work;
  const int64_t need = mev.advantages_workspace(&a);
  check(need, "mev_advantages_workspace");
  if (need > 0) {
    work = at::empty({need}, reward.options().dtype(at::kByte));
    a.workspace = work.data_ptr();
    a.workspace_bytes = need;
  }
  check(mev.advantages_run(&a, stream_of(reward)), "mev_advantages_run");
  return {adv, ret};
}

// -- clipping to the global norm -----------------------------------------------------------------
Tensor clip_grad_norm(const std::vector<Tensor>& grads, double max_norm,
                      const optional<std::vector<Tensor>>& out) {
  TORCH_CHECK_VALUE(!grads.empty(), "no gradients");
  number(max_norm, "max_norm", 0.0, kFloatMax);
  const std::vector<Tensor>& dst = out ? *out : grads;
  TORCH_CHECK_VALUE(dst.size() == grads.size(), "out has ", dst.size(), " tensors for ",
                    grads.size(), " gradients");
  const size_t n = grads.size();
  std::vector<const void*> src(n);
  std::vector<void*> to(n);
  std::vector<int64_t> numel(n);
  std::vector<int32_t> dtype(n);
  const auto device = grads[0].device();
  for (size_t i = 0; i < n; ++i) {
    const Tensor &g = grads[i], &o = dst[i];
    not_traced("clip_grad_norm", g, o);
    dense(g, "every gradient");
    dtype[i] = dtype_code(g.scalar_type());
    TORCH_CHECK_TYPE(dtype[i] >= 0, "gradients must be float32, bfloat16 or float16, got ",
                     g.scalar_type());
    TORCH_CHECK_VALUE(g.device() == device, "gradients on ", g.device(), " and ", device);
    TORCH_CHECK_VALUE(g.is_non_overlapping_and_dense(), "a gradient must fill one stretch of memory "
                      "(contiguous, or its axes in another order)");
    if (!o.is_same(g)) {
      dense(o, "out");
      TORCH_CHECK_VALUE(o.sizes() == g.sizes() && o.strides() == g.strides() &&
                            o.scalar_type() == g.scalar_type() && o.device() == device,
                        "out must match its gradient's shape, strides, dtype and device");
    }
    TORCH_CHECK_VALUE(!(o.requires_grad() && at::GradMode::is_enabled()),
                      "a tensor that requires a gradient cannot be written");
    no_tangent("clip_grad_norm", g, o);
    numel[i] = g.numel();
  }
  on_gpu(grads[0], "every gradient");
  for (size_t i = 0; i < n; ++i) {
    src[i] = grads[i].const_data_ptr();
    to[i] = dst[i].mutable_data_ptr();
  }
  const c10::DeviceGuard guard(device);
  const at::NoGradGuard no_grad;
  const int64_t need = mev.clip_norm_workspace(numel.data(), (int32_t)n);
  check(need, "mev_clip_norm_workspace");
  const auto opt = at::TensorOptions().device(device);
  const Tensor work = at::empty({need}, opt.dtype(at::kByte));
  const Tensor norm = at::empty({}, opt.dtype(at::kFloat));
  const int code = mev.clip_norm(src.data(), to.data(), numel.data(), dtype.data(), (int32_t)n,
                                 (float)max_norm, ptr<float>(norm), work.data_ptr(), need,
                                 stream_of(norm));
  TORCH_CHECK_VALUE(code != MEV_EINVAL, "gradients (or out) share memory");
  check(code, "mev_clip_norm");
  for (const Tensor& t : dst)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

PYBIND11_MODULE(mev_torch, m) {
  m.attr("abi_version") = MEV_ABI_VERSION;
  m.attr("source_hash") = MEV_SRC_HASH;
  m.def("bind", &bind);
  // launches only: the interpreter is free meanwhile
  const auto free_gil = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("action_logp", &action_logp, free_gil);
  m.def("policy_loss", &policy_loss, free_gil);
  m.def("advantages", &advantages, free_gil);
  m.def("clip_grad_norm", &clip_grad_norm, free_gil);
}
