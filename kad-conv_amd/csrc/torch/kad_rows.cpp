// kadconv._native: operators on rows, which are the last axis of a tensor or the channels of a map's pixels.
#include "kad_torch.h"

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
  if (fits && r.rs >= c && r.rs <= INT32_MAX && !x.is_neg()) return r;
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
  TORCH_CHECK_VALUE(temperature >= 1e-6 && temperature <= 1e6, "temperature must lie in 1e-6 to 1e6, got ", temperature);
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
    if ((h > 1 && w > 1 && t.stride(2) != w * t.stride(3)) || r.sp > UINT32_MAX || r.sk > UINT32_MAX) {
      r.held = t.contiguous();
      r.sn = t.size(1) * h * w, r.sp = 1, r.sk = h * w;
    }
    return r;
  }
  Strided r{t, 0, t.size(-1), t.stride(-1)};
  if (r.sk > UINT32_MAX) return {t.contiguous(), 0, t.size(-1), 1};
  bool first = true;
  int64_t expected = 0;
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (first) r.sp = expected = t.stride(i), first = false;
    if (t.stride(i) != expected || r.sp > UINT32_MAX) {
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
  const Tensor g = dloss.contiguous().resolve_neg();
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
  const Tensor stats = floats(x, {row_count(x, map), 2});
  const Tensor share = o.reduction == KAD_REDUCE_MEAN ? floats(x, {1}) : floats(x, {1}).zero_();
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

// ---------------------------------------------------------------------------- products in 8 bits
int64_t blocks8(int64_t k) { return (k + 127) / 128; }
int64_t codes8(int64_t k) { return blocks8(k) * 128; }
int64_t scales8(int64_t k) { return (blocks8(k) + 3) / 4 * 4; }

// Rows of k numbers in 8 bits (kadconv_hip.h), of a caller or, codes and then scales, in a buffer of their own.
struct Held8 {
  Tensor buffer;
  void *codes = nullptr, *scales = nullptr;
  bool defined() const { return codes != nullptr; }
};

int64_t held_bytes(int64_t rows, int64_t k) { return rows * (codes8(k) + scales8(k)); }

Held8 held_in(const Tensor& buffer, int64_t rows, int64_t k) {
  char* p = (char*)buffer.mutable_data_ptr();
  return {buffer, p, p + rows * codes8(k)};
}

Held8 new_held(const Tensor& x, int64_t rows, int64_t k) {
  return held_in(at::detail::empty_cuda({held_bytes(rows, k)}, at::kByte, x.device(), std::nullopt), rows, k);
}

Held8 held_of(const Tensor& codes, const Tensor& scales) {
  return {Tensor(), const_cast<void*>(codes.const_data_ptr()), const_cast<void*>(scales.const_data_ptr())};
}

Held8 saved_held(const Tensor& buffer, int64_t rows, int64_t k, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(buffer.is_contiguous() && buffer.scalar_type() == at::kByte && buffer.device() == like.device() &&
                        buffer.numel() == held_bytes(rows, k), name, " must be the forward's");
  return held_in(buffer, rows, k);
}

void check_held(const Tensor& codes, const Tensor& scales, int64_t rows, int64_t k, const Tensor& x, const char* name) {
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kFloat8_e4m3fn && scales.scalar_type() == at::kFloat8_e8m0fnu, name,
                   ": codes must be torch.float8_e4m3fn and scales torch.float8_e8m0fnu");
  TORCH_CHECK_VALUE(codes.is_contiguous() && scales.is_contiguous() && codes.device() == x.device() && scales.device() == x.device() &&
                        codes.dim() >= 1 && scales.dim() == codes.dim() && codes.size(-1) == codes8(k) &&
                        scales.size(-1) == scales8(k) && codes.numel() == rows * codes8(k) && scales.numel() == rows * scales8(k),
                    name, ": ", rows, " dense rows of ", codes8(k), " codes and ", scales8(k), " scales on ", x.device(), " expected, got ",
                    codes.sizes(), " and ", scales.sizes());
}

// What is wanted of a matrix: along its rows, along its columns, and their sums.
void quantize(const Rows& r, const Held8& along, const Held8& across, const Tensor& sums, const Tensor& x) {
  kad_quant8_args a{};
  a.x = r.held.const_data_ptr();
  a.x_rs = r.rs;
  a.rows = r.count;
  a.c = (int)r.c;
  a.codes = along.codes;
  a.scales = along.scales;
  a.t_codes = across.codes;
  a.t_scales = across.scales;
  a.sums = mutable_pointer(sums);
  a.dtype = dtype_of(r.held);
  a.sums_dtype = sums.defined() ? dtype_of(sums) : KAD_F32;
  const int64_t n = kad_quant8_work_elems(&a);
  if (n < 0) check((int)n, "kad_quant8_work_elems");
  const Tensor work = n ? floats(x, {n}) : Tensor();
  a.work = (float*)mutable_pointer(work);
  check(kad_quant8(&a, stream_of(x)), "kad_quant8");
}

// out = act(a b^T + bias), but for a.
kad_gemm8_args product_args(const Held8& b, int64_t m, int64_t n, int64_t k, const Tensor& bias, int act, const Tensor& out) {
  TORCH_CHECK_VALUE(m <= INT32_MAX - 255 && n <= INT32_MAX - 255, "too many rows: ", m, " and ", n);
  kad_gemm8_args g{};
  g.b = b.codes;
  g.b_scales = b.scales;
  g.bias = pointer(bias);
  g.out = out.mutable_data_ptr();
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  g.act = act;
  g.dtype = dtype_of(out);
  g.bias_dtype = bias.defined() ? dtype_of(bias) : KAD_F32;
  return g;
}

void launch_product(kad_gemm8_args& g, const Tensor& out) {
  const int64_t elems = kad_gemm8_work_elems(&g);
  if (elems < 0) check((int)elems, "kad_gemm8_work_elems");
  const Tensor work = elems ? floats(out, {elems}) : Tensor();
  g.work = (float*)mutable_pointer(work);
  check(kad_gemm8(&g, stream_of(out)), "kad_gemm8");
}

void product(const Held8& a, const Held8& b, int64_t m, int64_t n, int64_t k, const Tensor& bias, int act, const Tensor& out) {
  kad_gemm8_args g = product_args(b, m, n, k, bias, act, out);
  g.a = a.codes;
  g.a_scales = a.scales;
  launch_product(g, out);
}

// Of values: by way of 8 bits along k, in memory where the product does not bring them there itself.
void product_of_values(const Rows& r, const Held8& b, int64_t n, const Tensor& bias, int act, const Tensor& out) {
  kad_gemm8_args g = product_args(b, r.count, n, r.c, bias, act, out);
  g.a = r.held.const_data_ptr();
  g.a_rs = r.rs;
  g.a_dtype = dtype_of(r.held);
  Held8 h;
  if (!kad_gemm8_takes_values(&g)) {
    h = new_held(r.held, r.count, r.c);
    quantize(r, h, {}, Tensor(), r.held);
    g.a = h.codes;
    g.a_scales = h.scales;
  }
  launch_product(g, out);
}

void check_quantized(const Tensor& x, int64_t k) {
  TORCH_CHECK_VALUE(k >= 1 && k <= KAD_QUANT8_MOST, "rows of 1 to ", KAD_QUANT8_MOST, " values expected, got ", k);
  TORCH_CHECK_VALUE(x.is_cuda(), "a GPU tensor expected, got one on ", x.device());
  dtype_of(x);
}

// x [..., K] (or a map's pixels) as codes and scales [..., ...].
std::tuple<Tensor, Tensor> quantize8_forward(const Tensor& x, int64_t dim) {
  const bool map = is_map(x, dim);
  check_quantized(x, row_length(x, map));
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  const int64_t k = row_length(x, map);
  c10::DimVector sizes = row_sizes(x, map);
  sizes.push_back(codes8(k));
  const Tensor codes = at::detail::empty_cuda(sizes, at::kFloat8_e4m3fn, x.device(), std::nullopt);
  sizes.back() = scales8(k);
  const Tensor scales = at::detail::empty_cuda(sizes, at::kFloat8_e8m0fnu, x.device(), std::nullopt);
  if (x.numel()) quantize(rows_of(x, map), held_of(codes, scales), {}, Tensor(), x);
  return {codes, scales};
}

// None where the call is observed.
std::optional<std::tuple<Tensor, Tensor>> quantize8(const Tensor& x, int64_t dim) {
  if (observed({&x})) return std::nullopt;
  return quantize8_forward(x, dim);
}

at::ScalarType checked_result(at::ScalarType t) {
  TORCH_CHECK_TYPE(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, "unsupported dtype ", t, "; expected float32, float16 or bfloat16");
  return t;
}

// a [..., K] b [N, K]^T, both in 8 bits.
Tensor matmul8_forward(const Tensor& a, const Tensor& a_scales, const Tensor& b, const Tensor& b_scales, int64_t k, const OptTensor& bias,
                       const std::optional<std::string_view>& act, at::ScalarType dtype) {
  TORCH_CHECK_VALUE(a.is_cuda(), "a GPU tensor expected, got one on ", a.device());
  TORCH_CHECK_VALUE(k >= 1 && k <= KAD_QUANT8_MOST, "rows of 1 to ", KAD_QUANT8_MOST, " values expected, got ", k);
  TORCH_CHECK_VALUE(a.dim() >= 1 && b.dim() == 2, "a of at least one axis and b of two expected");
  const int64_t m = a.numel() / std::max<int64_t>(a.size(-1), 1), n = b.size(0);
  check_held(a, a_scales, m, k, a, "a");
  check_held(b, b_scales, n, k, a, "b");
  const Tensor bi = dense(defined(bias));
  if (bi.defined()) {
    TORCH_CHECK_VALUE(bi.dim() == 1 && bi.size(0) == n && bi.device() == a.device(), "bias must have shape (", n, ",) on ", a.device());
    dtype_of(bi);
  }
  const int ac = checked_act(act);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(a.device());
  c10::DimVector sizes(a.sizes());
  sizes.back() = n;
  Tensor out = at::detail::empty_cuda(sizes, checked_result(dtype), a.device(), std::nullopt);
  if (out.numel()) product(held_of(a, a_scales), held_of(b, b_scales), m, n, k, bi, ac, out);
  return out;
}

// None where the call is observed.
OptTensor matmul8(const Tensor& a, const Tensor& a_scales, const Tensor& b, const Tensor& b_scales, int64_t k, const OptTensor& bias,
                  const std::optional<std::string_view>& act, at::ScalarType dtype) {
  const Tensor bi = defined(bias);
  if (observed({&a, &a_scales, &b, &b_scales, &bi})) return std::nullopt;
  check_no_forward_grad({&bi}, "kadconv.matmul8");
  return matmul8_forward(a, a_scales, b, b_scales, k, bias, act, dtype);
}

// What the kernels take as given: the checks of kadconv.block8._linear8_check, and that the input is on a GPU.
bool check_linear8(const Tensor& x, int64_t n, int64_t k, const Tensor& bias, int64_t dim) {
  const bool map = is_map(x, dim);
  check_quantized(x, row_length(x, map));
  TORCH_CHECK_VALUE(row_length(x, map) == k, "rows of ", k, " values expected, got ", row_length(x, map));
  TORCH_CHECK_VALUE(n >= 1, "a weight of at least one row expected");
  check_param(bias, x, n, "bias");
  return map;
}

bool check_weight8(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t dim) {
  TORCH_CHECK_VALUE(weight.dim() == 2, "weight [N, K] expected");
  TORCH_CHECK_VALUE(weight.device() == x.device(), "input and weight must be on one device");
  TORCH_CHECK_TYPE(weight.scalar_type() == at::kFloat || weight.scalar_type() == x.scalar_type(), "weight must be float32 or ",
                   x.scalar_type(), ", got ", weight.scalar_type());
  return check_linear8(x, weight.size(0), weight.size(1), bias, dim);
}

Tensor result_like(const Tensor& x, bool map, int64_t n) {
  if (map) {
    const int64_t b = x.size(0), h = x.size(2), w = x.size(3);
    return at::detail::empty_strided_cuda({b, n, h, w}, {h * w * n, 1, w * n, n}, x.scalar_type(), x.device());
  }
  c10::DimVector sizes(x.sizes());
  sizes.back() = n;
  return at::detail::empty_cuda(sizes, x.scalar_type(), x.device(), std::nullopt);
}

// What the gradients need of a forward pass: x and w along their columns.
struct Across {
  Held8 x, w;
};

// The gradient of a weight is a product over the rows, that of the input one over the outputs; for all but the input's of few
// rows the gradient of y is brought to 8 bits in memory.  The checks of kadconv.block8._gradient_check.
void check_gradients8(int64_t rows, int64_t outputs, bool need_x, bool need_weight, bool need_bias) {
  TORCH_CHECK_VALUE(!need_weight || rows <= KAD_GEMM8_MOST, "a weight has a gradient of up to ", KAD_GEMM8_MOST, " rows, got ", rows);
  const bool in_memory = need_weight || need_bias || (need_x && rows > KAD_GEMM8_FEW);
  const int64_t most = in_memory ? KAD_QUANT8_MOST : need_x ? KAD_GEMM8_MOST : outputs;
  TORCH_CHECK_VALUE(!rows || outputs <= most, "gradients of up to ", most, " outputs expected, got ", outputs);
}

// y of values and a weight, which are brought to 8 bits; `across`: where wanted, along the columns in the same reads.
Tensor linear8_run(const Tensor& x, bool map, const Tensor& weight, const Tensor& bias, int act, bool across_x, bool across_w,
                   Across& across) {
  const int64_t n = weight.size(0), k = weight.size(1);
  Tensor y = result_like(x, map, n);
  const int64_t m = row_count(x, map);
  const Rows w = rows_of(weight, false);
  const Held8 wh = new_held(x, n, k);
  if (across_w) across.w = new_held(x, k, n);
  quantize(w, wh, across.w, Tensor(), x);
  if (across_x) across.x = new_held(x, k, std::max<int64_t>(m, 1));
  if (!m) return y;
  const Rows r = rows_of(x, map);
  const Tensor b = dense(bias);
  if (!across_x) {
    product_of_values(r, wh, n, b, act, y);
  } else if (m <= KAD_GEMM8_FEW) {
    quantize(r, {}, across.x, Tensor(), x);
    product_of_values(r, wh, n, b, act, y);
  } else {
    const Held8 h = new_held(x, m, k);
    quantize(r, h, across.x, Tensor(), x);
    product(h, wh, m, n, k, b, act, y);
  }
  return y;
}

struct Linear8Sizes {
  int64_t m, n, k, dim;
  at::ScalarType x, weight, bias;
};

// x: for its sizes and device.  dx, dw and db of dy, those that are needed.
std::tuple<Tensor, Tensor, Tensor> linear8_gradients(const Tensor& dy, bool map, const Linear8Sizes& o, const Across& across,
                                                     bool need_x, bool need_weight, bool need_bias) {
  Tensor dx = need_x ? result_like(dy, map, o.k) : Tensor();
  Tensor dw = need_weight ? at::detail::empty_cuda({o.n, o.k}, o.weight, dy.device(), std::nullopt) : Tensor();
  Tensor db = need_bias ? at::detail::empty_cuda({o.n}, o.bias, dy.device(), std::nullopt) : Tensor();
  if (!o.m) {  // sums over nothing
    if (need_weight) dw.zero_();
    if (need_bias) db.zero_();
    return {dx, dw, db};
  }
  if (!(need_x || need_weight || need_bias)) return {};
  const Rows r = rows_of(dy, map);
  const bool in_memory = need_x && o.m > KAD_GEMM8_FEW;
  Held8 along, down;
  if (in_memory) along = new_held(dy, o.m, o.n);
  if (need_weight) down = new_held(dy, o.n, o.m);
  if (in_memory || need_weight || need_bias) quantize(r, along, down, db, dy);
  if (in_memory) product(along, across.w, o.m, o.k, o.n, Tensor(), KAD_ACT_NONE, dx);
  else if (need_x) product_of_values(r, across.w, o.k, Tensor(), KAD_ACT_NONE, dx);
  if (need_weight) product(down, across.x, o.n, o.k, o.m, Tensor(), KAD_ACT_NONE, dw);
  return {dx, dw, db};
}

struct Linear8Backward : torch::autograd::Node {
  torch::autograd::SavedVariable x, w;  // in 8 bits along their columns
  Linear8Sizes o;
  bool map, has_x, has_w;
  c10::DimVector sizes;  // of y

  std::string name() const override { return "Linear8Backward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    w.reset_data();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list out(3);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    TORCH_CHECK_VALUE(dy.is_cuda() && dy.sizes() == at::IntArrayRef(sizes), "dy must have the result's shape and device");
    TORCH_CHECK_TYPE(dy.scalar_type() == o.x, "dy must have the result's dtype");
    const bool need_x = has_w && task_should_compute_output(0), need_w = has_x && task_should_compute_output(1),
               need_b = task_should_compute_output(2);
    Across across;
    // a hook on saved tensors may have put others in their place
    if (need_w) across.x = saved_held(x.unpack(), o.k, std::max<int64_t>(o.m, 1), dy, "the saved input");
    if (need_x) across.w = saved_held(w.unpack(), o.k, o.n, dy, "the saved weight");
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(dy.device());
      std::tie(out[0], out[1], out[2]) = linear8_gradients(dy, map, o, across, need_x, need_w, need_b);
    }
    // rounding to 8 bits has no second derivative
    if (c10::GradMode::is_enabled()) out = once_differentiable(std::move(out), "kadconv.linear8");
    return out;
  }
};

// None where the call is observed.
OptTensor linear8(const Tensor& x, const Tensor& weight, const OptTensor& bias, const std::optional<std::string_view>& act, int64_t dim) {
  const Tensor b = defined(bias);
  if (observed({&x, &weight, &b})) return std::nullopt;
  const bool map = check_weight8(x, weight, b, dim);
  const int ac = checked_act(act);
  check_no_forward_grad({&x, &weight, &b}, "kadconv.linear8");
  const bool grad = torch::autograd::compute_requires_grad(x, weight, b);
  TORCH_CHECK_NOT_IMPLEMENTED(!grad || ac == KAD_ACT_NONE, "kadconv.linear8 with an activation has no gradient");
  std::shared_ptr<Linear8Backward> node;
  Tensor y;
  Across across;
  if (grad) {
    check_gradients8(row_count(x, map), weight.size(0), x.requires_grad(), weight.requires_grad(), b.defined() && b.requires_grad());
    node = new_node<Linear8Backward>(torch::autograd::collect_next_edges(x, weight, b));
  }
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    y = linear8_run(x, map, weight, b, ac, node && weight.requires_grad(), node && x.requires_grad(), across);
  }
  if (node) {
    node->o = {row_count(x, map), weight.size(0), weight.size(1), dim, x.scalar_type(), weight.scalar_type(),
               b.defined() ? b.scalar_type() : at::kFloat};
    node->map = map;
    node->sizes = c10::DimVector(y.sizes());
    node->has_x = across.x.defined();
    node->has_w = across.w.defined();
    if (node->has_x) node->x = torch::autograd::SavedVariable(across.x.buffer, false);
    if (node->has_w) node->w = torch::autograd::SavedVariable(across.w.buffer, false);
    torch::autograd::set_history(y, node);
  }
  return y;
}

Tensor linear8_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias, const std::optional<std::string_view>& act, int64_t dim) {
  const Tensor b = defined(bias);
  const bool map = check_weight8(x, weight, b, dim);
  const int ac = checked_act(act);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  Across across;
  return linear8_run(x, map, weight, b, ac, false, false, across);
}

std::tuple<OptTensor, OptTensor, OptTensor> linear8_backward(const Tensor& dy, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                                             int64_t dim, bool need_x, bool need_weight, bool need_bias) {
  const Tensor b = defined(bias);
  const bool map = check_weight8(x, weight, b, dim);
  const Linear8Sizes o{row_count(x, map), weight.size(0), weight.size(1), dim, x.scalar_type(), weight.scalar_type(),
                       b.defined() ? b.scalar_type() : at::kFloat};
  c10::DimVector sizes(x.sizes());
  sizes[map ? 1 : x.dim() - 1] = o.n;
  TORCH_CHECK_VALUE(dy.device() == x.device() && dy.sizes() == at::IntArrayRef(sizes), "dy must have the result's shape and device");
  TORCH_CHECK_TYPE(dy.scalar_type() == o.x, "dy must have the result's dtype");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  Across across;
  check_gradients8(o.m, o.n, need_x, need_weight, need_bias && b.defined());
  if (need_weight && o.m) {
    across.x = new_held(x, o.k, o.m);
    quantize(rows_of(x, map), {}, across.x, Tensor(), x);
  }
  if (need_x && o.m) {
    across.w = new_held(x, o.k, o.n);
    quantize(rows_of(weight, false), {}, across.w, Tensor(), x);
  }
  auto [dx, dw, db] = linear8_gradients(dy, map, o, across, need_x, need_weight, need_bias && b.defined());
  return {opt(dx), opt(dw), opt(db)};
}

// With a weight that is kept in 8 bits.  None where the call is observed.
Tensor linear8_kept_run(const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t k, const Tensor& b,
                        const std::optional<std::string_view>& act, int64_t dim) {
  TORCH_CHECK_VALUE(codes.dim() == 2, "a weight [N, K] expected");
  const int64_t n = codes.size(0);
  const bool map = check_linear8(x, n, k, b, dim);
  check_held(codes, scales, n, k, x, "weight");
  const int ac = checked_act(act);
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  Tensor y = result_like(x, map, n);
  if (y.numel()) product_of_values(rows_of(x, map), held_of(codes, scales), n, dense(b), ac, y);
  return y;
}

OptTensor linear8_kept(const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t k, const OptTensor& bias,
                       const std::optional<std::string_view>& act, int64_t dim) {
  const Tensor b = defined(bias);
  if (observed({&x, &codes, &scales, &b})) return std::nullopt;
  check_no_forward_grad({&x, &b}, "kadconv.linear8");
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::compute_requires_grad(x, b), "kadconv.linear8 with a weight in 8 bits has no gradient");
  return linear8_kept_run(x, codes, scales, k, b, act, dim);
}

Tensor linear8_kept_forward(const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t k, const OptTensor& bias,
                            const std::optional<std::string_view>& act, int64_t dim) {
  return linear8_kept_run(x, codes, scales, k, defined(bias), act, dim);
}

}  // namespace

void kad_torch::bind_rows(py::module_& m) {
  // whether a call with these two is, for the modules
  m.def("observed", [](const Tensor& a, const Tensor& b) { return observed({&a, &b}); });
  m.def("layer_norm", &layer_norm);
  m.def("layer_norm_forward", &layer_norm_forward);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("quantize8", &quantize8);
  m.def("quantize8_forward", &quantize8_forward);
  m.def("matmul8", &matmul8);
  m.def("matmul8_forward", &matmul8_forward);
  m.def("linear8", &linear8);
  m.def("linear8_forward", &linear8_forward);
  m.def("linear8_backward", &linear8_backward);
  m.def("linear8_kept", &linear8_kept);
  m.def("linear8_kept_forward", &linear8_kept_forward);
  m.def("distill_loss", &distill_loss);
  m.def("distill_loss_forward", &distill_loss_forward);
  m.def("distill_loss_backward", &distill_loss_backward);
}
