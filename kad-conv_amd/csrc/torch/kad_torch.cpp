// kadconv._native: the training operators called from C++, where Python would cost more than their kernels.
//
// A group norm's forward and backward are a few microseconds on the GPU.  As a Python autograd function the
// pair took 170 us of host time (its backward runs on the engine's thread, and each switch between the two
// threads moves the interpreter's state from core to core); as an autograd node of C++ it takes 61 to 64, half of
// them the engine's own (and 36 in two of eight runs).
#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/FunctionsManual.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <string_view>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "kadconv_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", kad_last_error()); }

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KAD_F32;
    case at::kHalf: return KAD_F16;
    case at::kBFloat16: return KAD_BF16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type(), "; expected float32, float16 or bfloat16");
  }
}

Tensor defined(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
const void* pointer(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mutable_pointer(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// A dense channels-last map of x's shape, dtype and device.
Tensor map_like(const Tensor& x) {
  const int64_t n = x.size(0), c = x.size(1), h = x.size(2), w = x.size(3);
  return at::detail::empty_strided_cuda({n, c, h, w}, {h * w * c, 1, w * c, c}, x.scalar_type(), x.device());
}

// x [N, C, H, W] where it is channels-last, dense or a slice of the channels of a dense map; otherwise a dense
// channels-last copy.  cs: elements from pixel to pixel.  A slice whose channels are not a multiple of 16 bytes
// is copied too: its pieces would not tile the kernels' 16-byte vectors.
Tensor channels_last_pixels(const Tensor& x, int64_t& cs) {
  const int64_t n = x.size(0), c = x.size(1), h = x.size(2), w = x.size(3);
  cs = w > 1 ? x.stride(3) : h > 1 ? x.stride(2) : n > 1 ? x.stride(0) : c;
  if ((c == 1 || x.stride(1) == 1) && cs >= c && (h == 1 || x.stride(2) == w * cs) && (n == 1 || x.stride(0) == h * w * cs) &&
      (cs == c || (c % (16 / (int64_t)x.element_size()) == 0 && cs <= 1 << 20)))
    return x;
  cs = c;
  Tensor out = map_like(x);
  out.copy_(x);
  return out;
}

// The kernels take each size as an int.
void check_sizes(const Tensor& x) {
  for (const int64_t d : x.sizes()) TORCH_CHECK_VALUE(d <= INT32_MAX, "sizes up to 2^31 - 1 expected, got ", x.sizes());
}

// What the kernels take as given of a map and its parameters: the checks of kadconv.ops._group_norm_check, and that
// the map is on a GPU.
void check_norm(const Tensor& x, int64_t groups, const Tensor& weight, const Tensor& bias, double eps) {
  TORCH_CHECK_VALUE(x.dim() == 4, "input [N, C, H, W] expected");
  check_sizes(x);
  const int64_t c = x.size(1);
  TORCH_CHECK_VALUE(groups >= 1 && c >= 1 && c % groups == 0, groups, " groups do not divide ", c, " channels");
  TORCH_CHECK_VALUE(eps >= 0, "eps must be >= 0");
  for (const Tensor* p : {&weight, &bias}) {
    if (!p->defined()) continue;
    TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == c, "weight and bias must have shape (", c, ",), got ", p->sizes());
    TORCH_CHECK_VALUE(p->device() == x.device(), "input, weight and bias must be on one device");
    TORCH_CHECK_TYPE(p->scalar_type() == at::kFloat || p->scalar_type() == x.scalar_type(), "weight and bias must be float32 or ",
                     x.scalar_type(), ", got ", p->scalar_type());
  }
  TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
                   "weight and bias must share a dtype");
  TORCH_CHECK_VALUE(x.is_cuda(), "a GPU map expected, got one on ", x.device());
}

void check_gradient(const Tensor& dy, const Tensor& x) {
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.device() == x.device(), "dy must have the map's shape and device");
  TORCH_CHECK_TYPE(dy.scalar_type() == x.scalar_type(), "dy must have the map's dtype");
}

struct Norm {
  int64_t groups;
  double eps;
  int act;
};

kad_group_norm_args norm_args(const Tensor& x, int64_t cs, const Tensor& weight, const Tensor& bias, const Norm& o) {
  kad_group_norm_args a{};
  a.x = x.const_data_ptr();
  a.x_cs = cs;
  a.weight = pointer(weight);
  a.bias = pointer(bias);
  a.n = (int)x.size(0);
  a.c = (int)x.size(1);
  a.h = (int)x.size(2);
  a.w = (int)x.size(3);
  a.groups = (int)o.groups;
  a.eps = (float)o.eps;
  a.act = o.act;
  a.dtype = dtype_of(x);
  a.param_dtype = weight.defined() ? dtype_of(weight) : bias.defined() ? dtype_of(bias) : KAD_F32;
  return a;
}

Tensor floats(const Tensor& x, at::IntArrayRef sizes) {
  return at::detail::empty_cuda(sizes, at::kFloat, x.device(), std::nullopt);
}

Tensor scratch(const kad_group_norm_args& a, int backward, const Tensor& x) {
  const int64_t n = kad_group_norm_work_elems(&a, backward);
  if (n < 0) check((int)n, "kad_group_norm_work_elems");
  return n ? floats(x, {n}) : Tensor();
}

// y, with the means and reciprocal deviations [N, groups] written.
Tensor norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Norm& o, float* mean, float* rstd) {
  Tensor y = map_like(x);
  dtype_of(x);
  if (x.numel()) {
    int64_t cs;
    const Tensor v = channels_last_pixels(x, cs), w = dense(weight), b = dense(bias);
    kad_group_norm_args a = norm_args(v, cs, w, b, o);
    a.out = y.mutable_data_ptr();
    a.mean = mean;
    a.rstd = rstd;
    const Tensor work = scratch(a, 0, x);
    a.work = (float*)mutable_pointer(work);
    check(kad_group_norm_fwd(&a, stream_of(x)), "kad_group_norm_fwd");
  }
  return y;
}

struct Needs {
  bool x, weight, bias;
};

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& bias,
                                                 const float* mean, const float* rstd, const Norm& o, Needs need) {
  need.weight = need.weight && weight.defined();
  need.bias = need.bias && bias.defined();
  Tensor dx = need.x ? map_like(x) : Tensor();
  if (!x.numel())  // sums over nothing
    return {dx, need.weight ? at::zeros_like(weight) : Tensor(), need.bias ? at::zeros_like(bias) : Tensor()};
  if (!(need.x || need.weight || need.bias)) return {};
  const Tensor w = dense(weight), b = dense(bias);
  Tensor dw = need.weight ? at::detail::empty_cuda({x.size(1)}, w.scalar_type(), w.device(), std::nullopt) : Tensor();
  Tensor db = need.bias ? at::detail::empty_cuda({x.size(1)}, b.scalar_type(), b.device(), std::nullopt) : Tensor();
  int64_t cs, dcs;
  const Tensor v = channels_last_pixels(x, cs), d = channels_last_pixels(dy, dcs);
  kad_group_norm_args a = norm_args(v, cs, w, b, o);
  a.dy = d.const_data_ptr();
  a.dy_cs = dcs;
  a.out = mutable_pointer(dx);
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.dweight = mutable_pointer(dw);
  a.dbias = mutable_pointer(db);
  const Tensor work = scratch(a, 1, x);
  a.work = (float*)mutable_pointer(work);
  check(kad_group_norm_bwd(&a, stream_of(x)), "kad_group_norm_bwd");
  return {dx, dw, db};
}

struct GroupNormActBackward : torch::autograd::Node {
  torch::autograd::SavedVariable x, weight, bias, stats;  // stats: means and reciprocal deviations [2, N, groups]
  Norm norm;

  std::string name() const override { return "GroupNormActBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    bias.reset_data();
    stats.reset_data();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list out(3);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    const Tensor xs = x.unpack(), ws = weight.unpack(), bs = bias.unpack(), st = stats.unpack();
    // a hook on saved tensors may have put others in their place
    check_norm(xs, norm.groups, ws, bs, norm.eps);
    check_gradient(dy, xs);
    TORCH_CHECK_VALUE(st.is_contiguous() && st.scalar_type() == at::kFloat && st.device() == xs.device() &&
                          st.sizes() == at::IntArrayRef({2, xs.size(0), norm.groups}),
                      "the statistics must be the forward's");
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(xs.device());
      const float* mean = st.const_data_ptr<float>();
      std::tie(out[0], out[1], out[2]) =
          norm_backward(dy, xs, ws, bs, mean, mean + st.numel() / 2, norm,
                        {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)});
    }
    if (c10::GradMode::is_enabled() && torch::autograd::compute_requires_grad(dy, xs, ws, bs)) {
      // create_graph: the gradients' own gradient is not there, and says so when it is asked for
      for (Tensor& t : out)
        if (t.defined()) t.requires_grad_(true);
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "trying to differentiate twice a function that is once_differentiable: kadconv.group_norm_act", 3);
      out = (*error)(std::move(out));
    }
    return out;
  }
};

// The activation's number, after its check.
int checked_act(const std::optional<std::string_view>& act) {
  TORCH_CHECK_VALUE(!act || *act == "relu" || *act == "silu", "act '", act.value_or(""), "' is none of None, 'relu', 'silu'");
  return !act ? KAD_ACT_NONE : *act == "relu" ? KAD_ACT_RELU : KAD_ACT_SILU;
}

// Whether calls are watched (a trace, a dispatch mode) or a tensor stands for another (fake, wrapped): the caller then
// takes the registered operator, which such a program sees.  What is allocated and launched here, it would not.
bool observed(std::initializer_list<const Tensor*> tensors) {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set()) return true;
  for (const Tensor* t : tensors)
    if (t->defined() && (!t->has_storage() || t->key_set().has(c10::DispatchKey::Python))) return true;
  return false;
}

// None where the call is observed.
OptTensor group_norm_act(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, double eps,
                         const std::optional<std::string_view>& act) {
  const Tensor w = defined(weight), b = defined(bias);
  if (observed({&x, &w, &b})) return std::nullopt;
  check_norm(x, groups, w, b, eps);
  const Norm norm{groups, eps, checked_act(act)};
  std::shared_ptr<GroupNormActBackward> node;
  TORCH_CHECK_NOT_IMPLEMENTED(!(torch::autograd::isFwGradDefined(x) || torch::autograd::isFwGradDefined(w) ||
                                torch::autograd::isFwGradDefined(b)),
                              "kadconv.group_norm_act has no forward-mode gradient");
  if (torch::autograd::compute_requires_grad(x, w, b)) {
    node = std::shared_ptr<GroupNormActBackward>(new GroupNormActBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    node->x = torch::autograd::SavedVariable(x, false);
    node->weight = torch::autograd::SavedVariable(w, false);
    node->bias = torch::autograd::SavedVariable(b, false);
    node->norm = norm;
  }
  Tensor y, stats;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    stats = floats(x, {2, x.size(0), groups});
    float* mean = stats.mutable_data_ptr<float>();
    y = norm_forward(x, w, b, norm, mean, mean + x.size(0) * groups);
  }
  if (node) {
    node->stats = torch::autograd::SavedVariable(stats, false);
    torch::autograd::set_history(y, node);
  }
  return y;
}

std::tuple<Tensor, Tensor, Tensor> group_norm_act_forward(const Tensor& x, int64_t groups, const OptTensor& weight,
                                                          const OptTensor& bias, double eps, int act) {
  const Tensor w = defined(weight), b = defined(bias);
  check_norm(x, groups, w, b, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  const Tensor mean = floats(x, {x.size(0), groups}), rstd = floats(x, {x.size(0), groups});
  return {norm_forward(x, w, b, {groups, eps, act}, mean.mutable_data_ptr<float>(),
                       rstd.mutable_data_ptr<float>()),
          mean, rstd};
}

std::tuple<OptTensor, OptTensor, OptTensor> group_norm_act_backward(const Tensor& dy, const Tensor& x, int64_t groups,
                                                                    const OptTensor& weight, const OptTensor& bias,
                                                                    const Tensor& mean, const Tensor& rstd, double eps, int act,
                                                                    bool need_x, bool need_weight, bool need_bias) {
  const Tensor w = defined(weight), b = defined(bias);
  check_norm(x, groups, w, b, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  for (const Tensor& t : {mean, rstd})
    TORCH_CHECK_VALUE(t.is_contiguous() && t.scalar_type() == at::kFloat && t.device() == x.device() && t.dim() == 2 &&
                          t.size(0) == x.size(0) && t.size(1) == groups,
                      "mean and rstd must be the forward's");
  check_gradient(dy, x);
  auto [dx, dw, db] = norm_backward(dy, x, w, b, mean.const_data_ptr<float>(),
                                    rstd.const_data_ptr<float>(), {groups, eps, act}, {need_x, need_weight, need_bias});
  const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
  return {opt(dx), opt(dw), opt(db)};
}

// ---------------------------------------------------------------------------- AdamW
bool same_layout(const Tensor& a, const Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// The tensors of a plan, their gradients and the table of chunks on the GPU.
class AdamWTable {
 public:
  explicit AdamWTable(const std::vector<Tensor>& params) {
    TORCH_CHECK_VALUE(!params.empty(), "at least one parameter expected");
    const Tensor& p0 = params[0];
    std::vector<std::pair<int64_t, int64_t>> spans;
    for (const Tensor& p : params) {
      TORCH_CHECK_VALUE(p.is_cuda(), "kadconv.AdamWPlan needs GPU tensors");
      TORCH_CHECK_TYPE(p.scalar_type() == p0.scalar_type() && p.device() == p0.device(),
                       "parameters must share a dtype and a device");
      TORCH_CHECK_VALUE(p.layout() == at::kStrided && p.is_non_overlapping_and_dense(),
                        "parameters must be dense: no gaps or overlaps in their memory");
      given_.push_back(p);
      params_.push_back(p.detach());
      // views of one tensor share its version: it stands for all of them
      versioned_.push_back(p.is_view() ? Tensor(p._base()) : p);
      const int64_t at = (int64_t)p.const_data_ptr(), n = p.numel();
      at_.push_back(at);
      numels_.push_back(n);
      offsets_.push_back(elems_);
      elems_ += (n + KAD_ADAMW_SEG - 1) / KAD_ADAMW_SEG * KAD_ADAMW_SEG;
      if (n) spans.emplace_back(at, at + n * p.element_size());
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
      TORCH_CHECK_VALUE(spans[i].first >= spans[i - 1].second, "two parameters share memory");
    args_.dtype = dtype_of(p0);
  }

  void set_state(const Tensor& exp_avg, const Tensor& exp_avg_sq, const OptTensor& exp_avg_scale,
                 const OptTensor& exp_avg_sq_scale, const OptTensor& master, int state_bits, uint32_t seed) {
    state_ = {exp_avg, exp_avg_sq, defined(exp_avg_scale), defined(exp_avg_sq_scale), defined(master)};
    if (!state_stream_) state_stream_ = stream();
    args_.exp_avg = exp_avg.mutable_data_ptr();
    args_.exp_avg_sq = exp_avg_sq.mutable_data_ptr();
    args_.exp_avg_scale = (float*)mutable_pointer(state_[2]);
    args_.exp_avg_sq_scale = (float*)mutable_pointer(state_[3]);
    args_.master = (float*)mutable_pointer(state_[4]);
    args_.state_bits = state_bits;
    args_.seed = seed;
    masters_match();
  }

  // The masters are what to go on from, whatever was done to the parameters before.
  void masters_match() {
    seen_.clear();
    if (state_[4].defined())
      for (const Tensor& t : versioned_) seen_.push_back(version(t));
  }

  // Steps by these gradients from now on, and keeps them.
  void set_grads(const std::vector<OptTensor>& grads) {
    TORCH_CHECK_VALUE(grads.size() == params_.size(), grads.size(), " gradients for ", params_.size(), " parameters");
    std::vector<Tensor> held;
    std::vector<int64_t> at;
    for (size_t i = 0; i < grads.size(); ++i) {
      const Tensor g = defined(grads[i]);
      if (g.defined()) check_grad(params_[i], g);
      at.push_back(address(g));
      held.push_back(g.defined() ? g.detach() : g);
    }
    lay_out(std::move(at));
    held_ = std::move(held);
  }

  // Steps by the gradients that the parameters have now.  The caller keeps them until its step is launched.
  void follow(const std::vector<Tensor>& params) {
    TORCH_CHECK(params.size() == params_.size(), "the parameters are not those of the first step");
    std::vector<Tensor> held;
    std::vector<int64_t> at;
    at.reserve(params.size());
    for (size_t i = 0; i < params.size(); ++i) {
      const Tensor& p = params[i];
      TORCH_CHECK(p.is_same(given_[i]), "a group's parameters are not those of the first step: make a new optimizer");
      // a parameter that moved (module.to) would be written at its old address
      TORCH_CHECK((int64_t)p.const_data_ptr() == at_[i] && p.strides() == params_[i].strides() && p.sizes() == params_[i].sizes(),
                  "a parameter has moved since the first step: make a new optimizer");
      Tensor g = p.grad();
      if (g.defined()) {
        if (g.layout() == at::kStrided && g.sizes() == p.sizes() && !same_layout(p, g)) {
          const c10::DeviceGuard guard(p.device());
          Tensor same = at::empty_like(params_[i]);
          g = same.copy_(g.detach());
          held.push_back(g);
        }
        check_grad(p, g);
      }
      at.push_back(address(g));
    }
    if (at != grad_at_ || !chunks_.defined()) lay_out(std::move(at));
    held_ = std::move(held);
  }

  void step(int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay, const OptTensor& grad_scale) {
    TORCH_CHECK_VALUE(step >= 1, "step must be at least 1, got ", step);
    args_.step = step;
    args_.lr = lr;
    args_.scalars = nullptr;
    launch(beta1, beta2, eps, weight_decay, grad_scale);
  }

  // step, and lr where it is a tensor, are read when the kernels run.
  void step_later(const Tensor& step, const OptTensor& lr_at, double lr, double beta1, double beta2, double eps,
                  double weight_decay, const OptTensor& grad_scale) {
    check_scalar("step", step, at::kLong, "torch.int64");
    const Tensor rate = defined(lr_at);
    if (rate.defined()) check_scalar("lr", rate, at::kFloat, "torch.float32");
    const c10::DeviceGuard guard(params_[0].device());
    if (!scalars_.defined()) {
      scalars_ = at::empty({(int64_t)sizeof(kad_adamw_scalars)}, params_[0].options().dtype(at::kByte));
      scalars_stream_ = stream();
    }
    args_.step = 0;
    args_.lr = lr;
    args_.beta1 = beta1;
    args_.beta2 = beta2;
    args_.eps = eps;
    args_.weight_decay = weight_decay;
    args_.scalars = (const kad_adamw_scalars*)scalars_.const_data_ptr();
    check(kad_adamw_hyper(&args_, step.const_data_ptr<int64_t>(), (const float*)pointer(rate),
                          (kad_adamw_scalars*)scalars_.mutable_data_ptr(), stream_of(params_[0])),
          "kad_adamw_hyper");
    launch(beta1, beta2, eps, weight_decay, grad_scale);
  }

  std::vector<Tensor> params() const { return params_; }
  std::vector<int64_t> offsets() const { return offsets_; }
  std::vector<int64_t> numels() const { return numels_; }
  int64_t elems() const { return elems_; }
  // Whether a graph holds a step's addresses.
  bool captured() const { return !captured_.empty(); }

 private:
  static int64_t address(const Tensor& g) { return g.defined() && g.numel() ? (int64_t)g.const_data_ptr() : 0; }

  c10::hip::HIPStream stream() const { return c10::hip::getCurrentHIPStream(params_[0].device().index()); }

  static int64_t version(const Tensor& t) { return t.is_inference() ? 0 : (int64_t)t._version(); }

  static void check_grad(const Tensor& p, const Tensor& g) {
    TORCH_CHECK_VALUE(g.layout() == at::kStrided, "gradients must be dense tensors");
    TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type() && g.device() == p.device(), "a gradient is ", g.scalar_type(),
                     " on ", g.device(), ", its parameter ", p.scalar_type(), " on ", p.device());
    TORCH_CHECK_VALUE(same_layout(p, g), "a gradient must have the shape and strides of its parameter");
  }

  void check_scalar(const char* name, const Tensor& t, at::ScalarType dtype, const char* dtype_name) const {
    TORCH_CHECK_VALUE(t.scalar_type() == dtype && t.numel() == 1 && t.device() == params_[0].device(), name,
                      " must be one ", dtype_name, " value on ", params_[0].device());
  }

  void lay_out(std::vector<int64_t> grad_at) {
    const int n = (int)params_.size(), bytes = (int)params_[0].element_size();
    int64_t elems = 0;
    const int64_t count = kad_adamw_chunks(at_.data(), grad_at.data(), numels_.data(), n, bytes, nullptr, &elems);
    if (count < 0) check((int)count, "kad_adamw_chunks");
    TORCH_INTERNAL_ASSERT(elems == elems_);
    Tensor host = at::empty({count * (int64_t)sizeof(kad_adamw_chunk)}, at::TensorOptions(at::kByte));
    if (count)
      kad_adamw_chunks(at_.data(), grad_at.data(), numels_.data(), n, bytes, (kad_adamw_chunk*)host.mutable_data_ptr(), &elems);
    chunks_ = host.to(params_[0].device());
    chunks_stream_ = stream();
    args_.chunks = (const kad_adamw_chunk*)chunks_.const_data_ptr();
    args_.nchunks = count;
    args_.values = 0;
    stepped_.clear();
    std::unordered_set<const void*> seen;
    for (int i = 0; i < n; ++i) {
      if (!grad_at[i]) continue;
      args_.values += numels_[i];
      if (seen.insert(versioned_[i].unsafeGetTensorImpl()).second) stepped_.push_back(versioned_[i]);
    }
    grad_at_ = std::move(grad_at);
  }

  void launch(double beta1, double beta2, double eps, double weight_decay, const OptTensor& grad_scale) {
    if (grad_scale.has_value()) check_scalar("grad_scale", *grad_scale, at::kFloat, "torch.float32");
    args_.grad_scale = grad_scale.has_value() ? grad_scale->const_data_ptr<float>() : nullptr;
    args_.beta1 = beta1;
    args_.beta2 = beta2;
    args_.eps = eps;
    args_.weight_decay = weight_decay;
    const c10::DeviceGuard guard(params_[0].device());
    const c10::hip::HIPStream st = stream();
    const bool captured = c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
    if (captured) {
      // a graph reads the table whenever it is replayed, also after another one has been laid out; when it dies is not
      // known here, so a table (32 bytes a chunk) that was captured stays as long as this object
      if (captured_.empty() || !captured_.back().is_same(chunks_)) captured_.push_back(chunks_);
    } else {  // what the table holds is not given to others, when it dies, before this stream is through with it
      const auto used = [&](const Tensor& t, const std::optional<c10::hip::HIPStream>& own) {
        if (t.defined() && own != st) c10::hip::HIPCachingAllocator::recordStream(t.storage().data_ptr(), st);
      };
      used(chunks_, chunks_stream_);
      if (args_.scalars) used(scalars_, scalars_stream_);
      for (const Tensor& t : state_) used(t, state_stream_);
    }
    // A parameter written since its last step (its version tells) takes over from its master.  What will be written
    // between replays of a graph is not known: its steps always look.
    args_.follow = captured;
    for (size_t i = 0; i < seen_.size() && !args_.follow; ++i) args_.follow = grad_at_[i] && version(versioned_[i]) != seen_[i];
    check(kad_adamw_step(&args_, (void*)st.stream()), "kad_adamw_step");
    // the kernel wrote them: what is kept by a parameter's version (packed weights, saved tensors) is stale
    for (const Tensor& t : stepped_)
      if (!t.is_inference()) torch::autograd::impl::bump_version(t);
    if (!captured)
      for (size_t i = 0; i < seen_.size(); ++i)
        if (grad_at_[i]) seen_[i] = version(versioned_[i]);
  }

  std::vector<Tensor> given_, params_, versioned_, held_, stepped_, state_;
  std::vector<int64_t> at_, numels_, offsets_, grad_at_;
  std::vector<int64_t> seen_;  // with masters: the parameters' versions after their last steps
  int64_t elems_ = 0;
  Tensor chunks_, scalars_;
  std::vector<Tensor> captured_;
  std::optional<c10::hip::HIPStream> chunks_stream_, scalars_stream_, state_stream_;  // that they were made on
  kad_adamw_args args_{};
};

}  // namespace

PYBIND11_MODULE(_native, m) {
  py::class_<AdamWTable>(m, "AdamWTable")
      .def(py::init<const std::vector<Tensor>&>())
      .def("set_state", &AdamWTable::set_state)
      .def("masters_match", &AdamWTable::masters_match)
      .def("set_grads", &AdamWTable::set_grads)
      .def("follow", &AdamWTable::follow)
      .def("step", &AdamWTable::step)
      .def("step_later", &AdamWTable::step_later)
      .def_property_readonly("params", &AdamWTable::params)
      .def_property_readonly("offsets", &AdamWTable::offsets)
      .def_property_readonly("numels", &AdamWTable::numels)
      .def_property_readonly("elems", &AdamWTable::elems)
      .def_property_readonly("captured", &AdamWTable::captured);
  m.def("group_norm_act", &group_norm_act);
  m.def("group_norm_act_forward", &group_norm_act_forward);
  m.def("group_norm_act_backward", &group_norm_act_backward);
}
