// kadconv._native: operators on rows, which are the last axis of a tensor or the channels of a map's pixels.
#include "kad_torch.h"

#include <cmath>

namespace {

// The number of the axis along which rows run, as dim says: the last one, or the channels of [N, C, H, W].
bool is_map(const Tensor& x, int64_t dim) {
  const int64_t nd = x.dim();
  TORCH_CHECK_VALUE(nd >= 1, "an input with at least one axis expected");
  if (dim == -1 || dim == nd - 1) return false;
  TORCH_CHECK_VALUE(nd == 4 && (dim == 1 || dim == -3), "dim must be the last axis, or 1 for [N, C, H, W]; got ", dim, " for ", nd,
                    " axes");
  return true;
}

int64_t row_length(const Tensor& x, bool map) { return map ? x.size(1) : x.size(-1); }

// A tensor's rows: `count` of c values each, rs elements apart.
struct Rows {
  Tensor held;
  int64_t count, c, rs;
};

Tensor dense_like(const Tensor& x, bool map, std::optional<at::ScalarType> dtype = std::nullopt) {
  const at::ScalarType t = dtype.value_or(x.scalar_type());
  if (!map) return at::detail::empty_cuda(x.sizes(), t, x.device(), std::nullopt);
  const int64_t n = x.size(0), c = x.size(1), h = x.size(2), w = x.size(3);
  return at::detail::empty_strided_cuda({n, c, h, w}, {h * w * c, 1, w * c, c}, t, x.device());
}

// As they are where they lie a fixed distance apart, as those of dense tensors and of slices along their axis do;
// otherwise a dense copy.
Rows rows_of(const Tensor& x, bool map) {
  const int64_t nd = x.dim(), c = row_length(x, map);
  Rows r{x, 1, c, c};
  int64_t axes[4], rest = 0;  // the other axes, outermost first, of a map; of others all but the last
  if (map) axes[rest++] = 0, axes[rest++] = 2, axes[rest++] = 3;
  const int64_t others = map ? 3 : nd - 1, along = map ? 1 : nd - 1;
  const auto axis = [&](int64_t i) { return map ? axes[i] : i; };
  bool fits = c == 1 || x.stride(along) == 1, first = true;
  int64_t expected = 0;
  for (int64_t i = others - 1; i >= 0; --i) {
    const int64_t n = x.size(axis(i)), s = x.stride(axis(i));
    r.count *= n;
    if (n == 1) continue;
    if (first) r.rs = s, expected = s, first = false;
    fits = fits && s == expected;
    expected *= n;
  }
  if (fits && r.rs >= c && r.rs <= INT32_MAX) return r;
  r.held = dense_like(x, map);
  r.held.copy_(x);
  r.rs = c;
  return r;
}

void check_param(const Tensor& p, const Tensor& x, int64_t c, const char* name) {
  if (!p.defined()) return;
  TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == c, name, " must have shape (", c, ",), got ", p.sizes());
  TORCH_CHECK_VALUE(p.device() == x.device(), "input and ", name, " must be on one device");
  TORCH_CHECK_TYPE(p.scalar_type() == at::kFloat || p.scalar_type() == x.scalar_type(), name, " must be float32 or ",
                   x.scalar_type(), ", got ", p.scalar_type());
}

void check_like(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.sizes() == x.sizes() && t.device() == x.device(), name, " must have the input's shape and device");
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " must have the input's dtype");
}

// Gradients that were asked for with create_graph: their own gradient is not there, and says so when it is asked for.
torch::autograd::variable_list once_differentiable(torch::autograd::variable_list&& out, const char* name) {
  for (Tensor& t : out)
    if (t.defined()) t.requires_grad_(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice a function that is once_differentiable: ") + name, (int)out.size());
  return (*error)(std::move(out));
}

void check_no_forward_grad(std::initializer_list<const Tensor*> tensors, const char* name) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(*t), name, " has no forward-mode gradient");
}

template <typename Node>
std::shared_ptr<Node> new_node(const torch::autograd::edge_list& edges) {
  auto node = std::shared_ptr<Node>(new Node(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::edge_list(edges));
  return node;
}

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// ---------------------------------------------------------------------------- layer norm
// What the kernels take as given: the checks of kadconv.ops._layer_norm_check, and that the input is on a GPU.
bool check_layer_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, int64_t dim) {
  const bool map = is_map(x, dim);
  const int64_t c = row_length(x, map);
  TORCH_CHECK_VALUE(c >= 1, "rows of at least one value expected");
  TORCH_CHECK_VALUE(eps >= 0, "eps must be >= 0");
  check_param(weight, x, c, "weight");
  check_param(bias, x, c, "bias");
  TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
                   "weight and bias must share a dtype");
  TORCH_CHECK_VALUE(x.is_cuda(), "a GPU tensor expected, got one on ", x.device());
  dtype_of(x);
  TORCH_CHECK_VALUE(c <= KAD_LAYER_NORM_MOST, "rows of up to ", KAD_LAYER_NORM_MOST, " values expected on the GPU, got ", c);
  return map;
}

kad_layer_norm_args layer_norm_args(const Rows& x, const Tensor& weight, const Tensor& bias, double eps) {
  kad_layer_norm_args a{};
  a.x = x.held.const_data_ptr();
  a.x_rs = x.rs;
  a.rows = x.count;
  a.c = (int)x.c;
  a.weight = pointer(weight);
  a.bias = pointer(bias);
  a.eps = (float)eps;
  a.dtype = dtype_of(x.held);
  a.param_dtype = weight.defined() ? dtype_of(weight) : bias.defined() ? dtype_of(bias) : KAD_F32;
  return a;
}

// y, with the rows' means and reciprocal deviations written where they are wanted.
Tensor layer_norm_run(const Tensor& x, bool map, const Tensor& weight, const Tensor& bias, double eps, float* mean, float* rstd) {
  Tensor y = dense_like(x, map);
  if (x.numel()) {
    const Rows r = rows_of(x, map);
    const Tensor w = dense(weight), b = dense(bias);
    kad_layer_norm_args a = layer_norm_args(r, w, b, eps);
    a.out = y.mutable_data_ptr();
    a.mean = mean;
    a.rstd = rstd;
    check(kad_layer_norm_fwd(&a, stream_of(x)), "kad_layer_norm_fwd");
  }
  return y;
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_gradients(const Tensor& dy, const Tensor& x, bool map, const Tensor& weight,
                                                        const Tensor& bias, const float* mean, const float* rstd, double eps,
                                                        bool need_x, bool need_weight, bool need_bias) {
  need_weight = need_weight && weight.defined();
  need_bias = need_bias && bias.defined();
  Tensor dx = need_x ? dense_like(x, map) : Tensor();
  const auto like = [&](bool need, const Tensor& p) {
    return need ? at::detail::empty_cuda({p.size(0)}, p.scalar_type(), p.device(), std::nullopt) : Tensor();
  };
  Tensor dw = like(need_weight, weight), db = like(need_bias, bias);
  if (!x.numel()) {  // sums over nothing
    if (need_weight) dw.zero_();
    if (need_bias) db.zero_();
  } else if (need_x || need_weight || need_bias) {
    const Rows r = rows_of(x, map), d = rows_of(dy, map);
    const Tensor w = dense(weight);
    kad_layer_norm_args a = layer_norm_args(r, w, bias, eps);
    a.bias = nullptr;
    a.dy = d.held.const_data_ptr();
    a.dy_rs = d.rs;
    a.out = mutable_pointer(dx);
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.dweight = mutable_pointer(dw);
    a.dbias = mutable_pointer(db);
    Tensor work;
    if (need_weight || need_bias) {
      const int64_t n = kad_layer_norm_work_elems(&a);
      if (n < 0) check((int)n, "kad_layer_norm_work_elems");
      work = floats(x, {n});
      a.work = work.mutable_data_ptr<float>();
    }
    check(kad_layer_norm_bwd(&a, stream_of(x)), "kad_layer_norm_bwd");
  }
  return {dx, dw, db};
}

int64_t row_count(const Tensor& x, bool map) {
  return map ? x.size(0) * x.size(2) * x.size(3) : x.numel() / x.size(-1);
}

struct LayerNormBackward : torch::autograd::Node {
  torch::autograd::SavedVariable x, weight, bias, stats;  // stats: means and reciprocal deviations [2, rows]
  double eps;
  int64_t dim;

  std::string name() const override { return "LayerNormBackward"; }

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
    const bool map = check_layer_norm(xs, ws, bs, eps, dim);
    check_like(dy, xs, "dy");
    TORCH_CHECK_VALUE(st.is_contiguous() && st.scalar_type() == at::kFloat && st.device() == xs.device() &&
                          st.sizes() == at::IntArrayRef({2, row_count(xs, map)}),
                      "the statistics must be the forward's");
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(xs.device());
      const float* mean = st.const_data_ptr<float>();
      std::tie(out[0], out[1], out[2]) =
          layer_norm_gradients(dy, xs, map, ws, bs, mean, mean + st.size(1), eps, task_should_compute_output(0),
                               task_should_compute_output(1), task_should_compute_output(2));
    }
    if (c10::GradMode::is_enabled() && torch::autograd::compute_requires_grad(dy, xs, ws, bs))
      out = once_differentiable(std::move(out), "kadconv.layer_norm");
    return out;
  }
};

// None where the call is observed.
OptTensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, int64_t dim) {
  const Tensor w = defined(weight), b = defined(bias);
  if (observed({&x, &w, &b})) return std::nullopt;
  const bool map = check_layer_norm(x, w, b, eps, dim);
  check_no_forward_grad({&x, &w, &b}, "kadconv.layer_norm");
  std::shared_ptr<LayerNormBackward> node;
  if (torch::autograd::compute_requires_grad(x, w, b)) {
    node = new_node<LayerNormBackward>(torch::autograd::collect_next_edges(x, w, b));
    node->x = torch::autograd::SavedVariable(x, false);
    node->weight = torch::autograd::SavedVariable(w, false);
    node->bias = torch::autograd::SavedVariable(b, false);
    node->eps = eps;
    node->dim = dim;
  }
  Tensor y, stats;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    float *mean = nullptr, *rstd = nullptr;
    if (node) {
      const int64_t rows = row_count(x, map);
      stats = floats(x, {2, rows});
      mean = stats.mutable_data_ptr<float>();
      rstd = mean + rows;
    }
    y = layer_norm_run(x, map, w, b, eps, mean, rstd);
  }
  if (node) {
    node->stats = torch::autograd::SavedVariable(stats, false);
    torch::autograd::set_history(y, node);
  }
  return y;
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps,
                                                      int64_t dim) {
  const Tensor w = defined(weight), b = defined(bias);
  const bool map = check_layer_norm(x, w, b, eps, dim);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  const Tensor mean = floats(x, {row_count(x, map)}), rstd = floats(x, {row_count(x, map)});
  return {layer_norm_run(x, map, w, b, eps, mean.mutable_data_ptr<float>(), rstd.mutable_data_ptr<float>()), mean, rstd};
}

std::tuple<OptTensor, OptTensor, OptTensor> layer_norm_backward(const Tensor& dy, const Tensor& x, const OptTensor& weight,
                                                                const OptTensor& bias, const Tensor& mean, const Tensor& rstd,
                                                                double eps, int64_t dim, bool need_x, bool need_weight,
                                                                bool need_bias) {
  const Tensor w = defined(weight), b = defined(bias);
  const bool map = check_layer_norm(x, w, b, eps, dim);
  check_like(dy, x, "dy");
  for (const Tensor& t : {mean, rstd})
    TORCH_CHECK_VALUE(t.is_contiguous() && t.scalar_type() == at::kFloat && t.device() == x.device() && t.dim() == 1 &&
                          t.size(0) == row_count(x, map),
                      "mean and rstd must be the forward's");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  auto [dx, dw, db] = layer_norm_gradients(dy, x, map, w, b, mean.const_data_ptr<float>(), rstd.const_data_ptr<float>(), eps,
                                           need_x, need_weight, need_bias);
  return {opt(dx), opt(dw), opt(db)};
}

// ---------------------------------------------------------------------------- distillation
struct Distill {
  double temperature;
  int reduction;
  int64_t dim;
};

int checked_reduction(std::string_view r) {
  TORCH_CHECK_VALUE(r == "none" || r == "sum" || r == "mean", "reduction '", r, "' is none of 'none', 'sum', 'mean'");
  return r == "none" ? KAD_REDUCE_NONE : r == "sum" ? KAD_REDUCE_SUM : KAD_REDUCE_MEAN;
}

// What the kernels take as given: the checks of kadconv.ops._distill_check, and that the tensors are on a GPU.
bool check_distill(const Tensor& x, const Tensor& t, const Tensor& index, double temperature, int64_t dim) {
  const bool map = is_map(x, dim);
  const int64_t nd = x.dim(), axis = map ? 1 : nd - 1;
  TORCH_CHECK_VALUE(x.size(axis) >= 1, "at least one class expected");
  TORCH_CHECK_VALUE(t.dim() == nd && t.sizes() == index.sizes(), "teacher_logits and teacher_index must have one shape and the axes of logits");
  for (int64_t d = 0; d < nd; ++d)
    TORCH_CHECK_VALUE(d == axis || t.size(d) == x.size(d), "teacher_logits must have the shape of logits but for the classes, got ",
                      t.sizes(), " for ", x.sizes());
  TORCH_CHECK_VALUE(t.size(axis) >= 1 && t.size(axis) <= KAD_DISTILL_MOST, "1 to ", KAD_DISTILL_MOST, " entries expected, got ",
                    t.size(axis));
  TORCH_CHECK_VALUE(x.device() == t.device() && x.device() == index.device(), "logits and the teacher's tensors must be on one device");
  TORCH_CHECK_TYPE(index.scalar_type() == at::kInt || index.scalar_type() == at::kLong,
                   "teacher_index must be torch.int32 or torch.int64, got ", index.scalar_type());
  TORCH_CHECK_VALUE(temperature > 0 && std::isfinite((float)temperature) && (float)temperature > 0, "temperature must be positive");
  TORCH_CHECK_VALUE(x.is_cuda(), "a GPU tensor expected, got one on ", x.device());
  dtype_of(x);
  dtype_of(t);
  return map;
}

// Where the entries lie: of row (n, p), n sn + p sp + e sk.
struct Strided {
  Tensor held;
  int64_t sn, sp, sk;
};

Strided entries_of(const Tensor& t, bool map) {
  if (map) {
    const int64_t h = t.size(2), w = t.size(3);
    Strided r{t, t.stride(0), w > 1 ? t.stride(3) : t.stride(2), t.stride(1)};
    if (h > 1 && w > 1 && t.stride(2) != w * t.stride(3)) {
      r.held = t.contiguous();
      r.sn = t.size(1) * h * w, r.sp = 1, r.sk = h * w;
    }
    return r;
  }
  Strided r{t, 0, t.size(-1), t.stride(-1)};
  bool first = true;
  int64_t expected = 0;
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (first) r.sp = expected = t.stride(i), first = false;
    if (t.stride(i) != expected) {
      r.held = t.contiguous();
      r.sp = t.size(-1), r.sk = 1;
      return r;
    }
    expected *= t.size(i);
  }
  return r;
}

kad_distill_args distill_args(const Rows& x, const Strided& t, const Strided& i, bool map, const Distill& o) {
  kad_distill_args a{};
  a.logits = x.held.const_data_ptr();
  a.teacher = t.held.const_data_ptr();
  a.index = i.held.const_data_ptr();
  a.rows = x.count;
  a.z_rs = x.rs;
  a.inner = map ? x.held.size(2) * x.held.size(3) : x.count;
  a.t_sn = t.sn, a.t_sp = t.sp, a.t_sk = t.sk;
  a.i_sn = i.sn, a.i_sp = i.sp, a.i_sk = i.sk;
  a.v = (int)x.c;
  a.k = (int)t.held.size(map ? 1 : -1);
  a.temperature = (float)o.temperature;
  a.reduction = o.reduction;
  a.dtype = dtype_of(x.held);
  a.teacher_dtype = dtype_of(t.held);
  a.index_bits = i.held.scalar_type() == at::kInt ? 32 : 64;
  return a;
}

c10::DimVector row_sizes(const Tensor& x, bool map) {
  c10::DimVector s(x.sizes());
  s.erase(s.begin() + (map ? 1 : x.dim() - 1));
  return s;
}

void check_classes(const Tensor& x, bool map) {
  TORCH_CHECK_VALUE(row_length(x, map) <= 1 << 30 && row_count(x, map) <= INT32_MAX, "up to 2^30 classes and 2^31 - 1 rows expected, got ",
                    x.sizes());
}

// The loss, with stats [rows, 2] (where wanted) and share [1] written.
Tensor distill_run(const Tensor& x, bool map, const Tensor& t, const Tensor& index, const Distill& o, const Tensor& stats,
                   const Tensor& share) {
  check_classes(x, map);
  Tensor loss = o.reduction == KAD_REDUCE_NONE ? floats(x, row_sizes(x, map)) : floats(x, {});
  if (!x.numel()) {
    loss.zero_();
    if (share.defined()) share.zero_();
    return loss;
  }
  const Rows r = rows_of(x, map);
  const Strided te = entries_of(t, map), ie = entries_of(index, map);
  kad_distill_args a = distill_args(r, te, ie, map, o);
  a.loss = loss.mutable_data_ptr<float>();
  a.stats = (float*)mutable_pointer(stats);
  a.share = (float*)mutable_pointer(share);
  const int64_t n = kad_distill_work_elems(&a);
  if (n < 0) check((int)n, "kad_distill_work_elems");
  const Tensor work = n ? floats(x, {n}) : Tensor();
  a.work = (float*)mutable_pointer(work);
  check(kad_distill_fwd(&a, stream_of(x)), "kad_distill_fwd");
  return loss;
}

void check_saved(const Tensor& x, bool map, const Tensor& stats, const Tensor& share) {
  const auto floats_like = [&](const Tensor& t, at::IntArrayRef sizes) {
    return t.is_contiguous() && t.scalar_type() == at::kFloat && t.device() == x.device() && t.sizes() == sizes;
  };
  TORCH_CHECK_VALUE(floats_like(stats, {row_count(x, map), 2}) && floats_like(share, {1}), "stats and share must be the forward's");
}

Tensor distill_gradient(const Tensor& dloss, const Tensor& x, bool map, const Tensor& t, const Tensor& index, const Tensor& stats,
                        const Tensor& share, const Distill& o) {
  check_classes(x, map);
  TORCH_CHECK_VALUE(dloss.device() == x.device() && dloss.scalar_type() == at::kFloat &&
                        (o.reduction == KAD_REDUCE_NONE ? dloss.sizes() == at::IntArrayRef(row_sizes(x, map)) : dloss.numel() == 1),
                    "dloss must be float32 with the shape and device of the loss");
  Tensor dx = dense_like(x, map);
  if (!x.numel()) return dx;
  const Rows r = rows_of(x, map);
  const Strided te = entries_of(t, map), ie = entries_of(index, map);
  const Tensor g = dloss.contiguous();
  kad_distill_args a = distill_args(r, te, ie, map, o);
  a.dloss = g.const_data_ptr<float>();
  a.dlogits = dx.mutable_data_ptr();
  a.stats = const_cast<float*>(stats.const_data_ptr<float>());
  a.share = const_cast<float*>(share.const_data_ptr<float>());
  check(kad_distill_bwd(&a, stream_of(x)), "kad_distill_bwd");
  return dx;
}

struct DistillBackward : torch::autograd::Node {
  torch::autograd::SavedVariable x, t, index, stats, share;
  Distill o;

  std::string name() const override { return "DistillBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* v : {&x, &t, &index, &stats, &share}) v->reset_data();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list out(1);
    const Tensor& dloss = grads[0];
    if (!dloss.defined() || !task_should_compute_output(0)) return out;
    const Tensor xs = x.unpack(), ts = t.unpack(), is = index.unpack(), st = stats.unpack(), sh = share.unpack();
    // a hook on saved tensors may have put others in their place
    const bool map = check_distill(xs, ts, is, o.temperature, o.dim);
    check_saved(xs, map, st, sh);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(xs.device());
      out[0] = distill_gradient(dloss, xs, map, ts, is, st, sh, o);
    }
    if (c10::GradMode::is_enabled() && torch::autograd::compute_requires_grad(dloss, xs))
      out = once_differentiable(std::move(out), "kadconv.distill_loss");
    return out;
  }
};

// None where the call is observed.
OptTensor distill_loss(const Tensor& x, const Tensor& t, const Tensor& index, double temperature, std::string_view reduction,
                       int64_t dim) {
  if (observed({&x, &t, &index})) return std::nullopt;
  const bool map = check_distill(x, t, index, temperature, dim);
  const Distill o{temperature, checked_reduction(reduction), dim};
  check_no_forward_grad({&x, &t}, "kadconv.distill_loss");
  std::shared_ptr<DistillBackward> node;
  if (torch::autograd::compute_requires_grad(x)) {
    node = new_node<DistillBackward>(torch::autograd::collect_next_edges(x));
    node->x = torch::autograd::SavedVariable(x, false);
    node->t = torch::autograd::SavedVariable(t.detach(), false);
    node->index = torch::autograd::SavedVariable(index, false);
    node->o = o;
  }
  Tensor loss, stats, share;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    if (node) {
      stats = floats(x, {row_count(x, map), 2});
      share = floats(x, {1});
    }
    loss = distill_run(x, map, t, index, o, stats, share);
  }
  if (node) {
    node->stats = torch::autograd::SavedVariable(stats, false);
    node->share = torch::autograd::SavedVariable(share, false);
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

std::tuple<Tensor, Tensor, Tensor> distill_loss_forward(const Tensor& x, const Tensor& t, const Tensor& index, double temperature,
                                                        std::string_view reduction, int64_t dim) {
  const bool map = check_distill(x, t, index, temperature, dim);
  const Distill o{temperature, checked_reduction(reduction), dim};
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  const Tensor stats = floats(x, {row_count(x, map), 2}), share = floats(x, {1});
  return {distill_run(x, map, t, index, o, stats, share), stats, share};
}

Tensor distill_loss_backward(const Tensor& dloss, const Tensor& x, const Tensor& t, const Tensor& index, const Tensor& stats,
                             const Tensor& share, double temperature, std::string_view reduction, int64_t dim) {
  const bool map = check_distill(x, t, index, temperature, dim);
  const Distill o{temperature, checked_reduction(reduction), dim};
  check_saved(x, map, stats, share);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  return distill_gradient(dloss, x, map, t, index, stats, share, o);
}

}  // namespace

void kad_torch::bind_rows(py::module_& m) {
  m.def("layer_norm", &layer_norm);
  m.def("layer_norm_forward", &layer_norm_forward);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("distill_loss", &distill_loss);
  m.def("distill_loss_forward", &distill_loss_forward);
  m.def("distill_loss_backward", &distill_loss_backward);
}
