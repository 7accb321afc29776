// The operators over grouped rows as torch operators with gradients: argument checks, allocation and the autograd nodes, in
// C++ because at the sizes of one resolution level a call through ctypes and Python autograd costs several times what
// its kernels take (embedding with its gradient, smallest sizes: 97 us a pass there, 58 us here).
//
// Every call goes to the C entries of include/tsb200.h, on the current stream of the tensors' device.  All operators are
// registered with torch's dispatcher, gradients included: what traces or records a program sees them, and not merely
// the empty tensors that their kernels fill.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/tsb200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

void check_status(int status, const char* what) {
  if (status == TSB_OK) return;
  std::string text = std::string(what) + ": " + tsb_status_string(status);
  if (status == TSB_ERR_CUDA) text += std::string(": ") + tsb_last_cuda_error();
  TORCH_CHECK_VALUE(status != TSB_ERR_BAD_ARG && status != TSB_ERR_LIMIT, text);
  TORCH_CHECK(false, text);
}

void need_cuda(const Tensor& t) {
  TORCH_CHECK(!t.defined() || t.is_cuda(), "torchsparse_b200: CUDA tensors required (there is no CPU fallback)");
}

void same_device(const Tensor& first, std::initializer_list<Tensor> others) {
  need_cuda(first);
  for (const Tensor& t : others) {
    if (!t.defined()) continue;
    need_cuda(t);
    TORCH_CHECK_VALUE(t.device() == first.device(), "tensors live on ", first.device(), " and ", t.device());
  }
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TSB_F32;
    case at::kHalf: return TSB_F16;
    case at::kBFloat16: return TSB_BF16;
    default: TORCH_CHECK(false, "unsupported feature dtype ", t.scalar_type());
  }
}

void check_index(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, what, " must be int32 or int64, not ",
                    t.scalar_type());
}

void check_int32(const Tensor& t, int64_t length, const char* what) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && (length < 0 || t.size(0) == length), what,
                    " must be a contiguous int32 vector", length < 0 ? std::string() : " of length " + std::to_string(length));
}

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const int32_t* ints(const Tensor& t) { return t.defined() ? t.const_data_ptr<int32_t>() : nullptr; }
Tensor packed(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// device guard, stream and an optional workspace of one call
struct Call {
  c10::cuda::CUDAGuard guard;
  Tensor scratch;
  size_t bytes = 0;
  explicit Call(const Tensor& t) : guard(t.device()) {}
  void* workspace(size_t n, const Tensor& like) {
    bytes = n;
    if (n) scratch = at::empty({(int64_t)n}, like.options().dtype(at::kByte));
    return n ? scratch.mutable_data_ptr() : nullptr;
  }
  tsb_stream_t stream() const { return c10::cuda::getCurrentCUDAStream().stream(); }
};

// the dispatcher's handle of an operator that is registered below
template <typename Signature>
c10::TypedOperatorHandle<Signature> registered(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// Inside torch.func.grad and its like, which take torch's own operations and no C++ Function.
bool in_transform() { return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerBackMode); }

// Forward-mode differentiation: the tangent that goes with a tensor, and values put together with theirs.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
Tensor tangent(const Tensor& t) { return t._fw_grad(/*level=*/0); }
Tensor primal(const Tensor& t) { return has_tangent(t) ? t._fw_primal(/*level=*/0) : t; }
Tensor dual(const Tensor& value, const Tensor& tangent) { return at::_make_dual(value, tangent, /*level=*/0); }

void refuse_tangent(const Tensor& grad) {
  TORCH_CHECK(!has_tangent(grad), "the gradient of this operator of torchsparse_b200 has no forward-mode derivative");
}

// What a backward call returns: its kernels have no gradient of their own, and asking for one is an error, not a zero.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  int n = 0;
  for (const Tensor& t : grads) n += t.defined();
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "this operator of torchsparse_b200 can be differentiated once only", n);
  variable_list in;
  for (const Tensor& t : grads)
    if (t.defined()) in.push_back(t.detach().requires_grad_());
  variable_list made = (*refuse)(std::move(in));
  size_t k = 0;
  for (Tensor& t : grads)
    if (t.defined()) t = made[k++];
  return grads;
}

// ------------------------------------------------------------------------------------------------ grouping
// order, offsets and, where its shape is given, the position of every key
std::tuple<Tensor, Tensor, Tensor> group(const Tensor& keys, int64_t num_groups, at::OptionalIntArrayRef inverse_shape) {
  TORCH_CHECK_VALUE(num_groups >= 1 && num_groups < (1ll << 31), "the number of groups must be in [1, 2^31), not ", num_groups);
  Call call(keys);
  const int64_t n = keys.size(0);
  const auto opts = keys.options().dtype(at::kInt);
  Tensor order = at::empty({n}, opts), offsets = at::empty({num_groups + 1}, opts), inverse;
  if (inverse_shape.has_value()) inverse = at::empty(*inverse_shape, opts);
  void* ws = call.workspace(tsb_group_rows_workspace_bytes(n, num_groups), keys);
  check_status(tsb_group_rows(keys.const_data_ptr(), keys.scalar_type() == at::kLong, keys.stride(0), n, num_groups,
                              order.mutable_data_ptr<int32_t>(), (int32_t*)out_ptr(inverse), offsets.mutable_data_ptr<int32_t>(), ws,
                              call.bytes, call.stream()),
               "group_rows");
  return {order, offsets, inverse};
}

std::tuple<Tensor, Tensor> group_rows(const Tensor& keys, int64_t num_groups) {
  need_cuda(keys);
  check_index(keys, "keys");
  TORCH_CHECK_VALUE(keys.dim() == 1, "keys must be a vector, not ", keys.sizes());
  auto [order, offsets, inverse] = group(keys, num_groups, std::nullopt);
  return {order, offsets};
}

std::tuple<Tensor, Tensor> call_group_rows(const Tensor& keys, int64_t num_groups) {
  static const auto op = registered<decltype(group_rows)>("torchsparse_b200::group_rows");
  return op.call(keys, num_groups);
}

std::tuple<Tensor, Tensor, Tensor> expert_sort(const Tensor& experts, int64_t num_experts) {
  need_cuda(experts);
  check_index(experts, "experts");
  TORCH_CHECK_VALUE(experts.dim() == 1 || experts.dim() == 2, "experts must be [N, k] or [N], not ", experts.sizes());
  const int64_t shape[2] = {experts.size(0), experts.dim() == 2 ? experts.size(1) : 1};
  TORCH_CHECK_VALUE(shape[1] >= 1, "every row needs at least one choice");
  auto [order, offsets, inverse] = group(experts.reshape(-1), num_experts, at::IntArrayRef(shape, 2));
  return {order, inverse, offsets};
}

std::tuple<Tensor, Tensor, Tensor> call_expert_sort(const Tensor& experts, int64_t num_experts) {
  static const auto op = registered<decltype(expert_sort)>("torchsparse_b200::expert_sort");
  return op.call(experts, num_experts);
}

// ------------------------------------------------------------------------------------------------ group norm
struct NormArgs {
  int64_t groups;
  double eps, slope;
  int64_t act;
};

int check_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& offsets, const Tensor& order, int64_t groups) {
  same_device(x, {weight, bias, offsets, order});
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) >= 1, "group_norm expects features [N, C], not ", x.sizes());
  const int64_t c = x.size(1);
  TORCH_CHECK_VALUE(groups >= 1 && c % groups == 0, c, " channels do not divide into ", groups, " groups");
  check_int32(offsets, -1, "offsets");
  TORCH_CHECK_VALUE(offsets.size(0) >= 1, "offsets must hold the first row of every sample and the end of the last");
  if (order.defined()) check_int32(order, x.size(0), "order");
  dtype_code(x);
  int code = -1;
  for (const Tensor* p : {&weight, &bias}) {
    if (!p->defined()) continue;
    TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == c, "weight and bias must be vectors of ", c, " values, not ", p->sizes());
    TORCH_CHECK_VALUE(code < 0 || code == dtype_code(*p), "weight and bias must have one dtype");
    code = dtype_code(*p);
  }
  return code < 0 ? (int)TSB_F32 : code;
}

// (y, [2, samples, groups] of means and reciprocal deviations, or an undefined tensor)
std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& offsets, const Tensor& order,
                                       const NormArgs& a, int p_code, bool want_stats) {
  Call call(x);
  const int64_t n = x.size(0), c = x.size(1), samples = offsets.size(0) - 1;
  Tensor y = at::empty_like(x), stats;
  float *mean = nullptr, *rstd = nullptr;
  if (want_stats) {
    stats = at::empty({2, samples, a.groups}, x.options().dtype(at::kFloat));
    mean = stats.mutable_data_ptr<float>();
    rstd = mean + samples * a.groups;
  }
  const int dtype = dtype_code(x);
  void* ws = call.workspace(tsb_group_norm_fwd_workspace_bytes(n, c, a.groups, samples, dtype), x);
  check_status(tsb_group_norm_fwd(ptr(x), ints(order), ints(offsets), ptr(w), ptr(b), n, c, a.groups, samples, (float)a.eps,
                                  (int)a.act, (float)a.slope, dtype, p_code, out_ptr(y), mean, rstd, ws, call.bytes, call.stream()),
               "group_norm");
  return {y, stats};
}

// The sample of each row, `samples` for a row of none.  Entries of an order that are no rows go nowhere.
Tensor row_samples(const Tensor& offsets, const Tensor& order, int64_t n) {
  const int64_t samples = offsets.size(0) - 1;
  const Tensor off = offsets.to(at::kLong).clamp(0, n), pos = at::arange(n, off.options());
  if (samples == 0) return at::zeros_like(pos);
  const Tensor sample = at::searchsorted(off.slice(0, 1), pos, /*out_int32=*/false, /*right=*/true).masked_fill(pos.lt(off[0]), samples);
  if (!order.defined()) return sample;
  const Tensor rows = order.to(at::kLong), to = rows.masked_fill(rows.lt(0).logical_or(rows.ge(n)), n);
  return at::full({n + 1}, samples, pos.options()).scatter(0, to, sample).slice(0, 0, n);
}

// The mean over the sample and group of each value of t [n, c] (fp32), at that value; zeros in rows of no sample.  The means
// are those of the norm's own statistics: joined piece by piece in a fixed order, however long the sample.  (One sum per
// sample and group by index_add would lose 3.5e-3 of a mean square over 4M rows, and count 2^24 rows at most.)
Tensor group_mean(const Tensor& t, const Tensor& offsets, const std::optional<Tensor>& order, int64_t groups) {
  const Tensor x = t.contiguous(), o = order.value_or(Tensor());
  const int code = check_norm(x, Tensor(), Tensor(), offsets, o, groups);
  TORCH_CHECK(x.scalar_type() == at::kFloat, "group_mean expects fp32, not ", x.scalar_type());
  const Tensor stats = norm_forward(x, Tensor(), Tensor(), offsets, o, NormArgs{groups, 1.0, 0.0, 0}, code, true).second;
  const Tensor means = at::constant_pad_nd(stats[0], {0, 0, 0, 1}).repeat_interleave(x.size(1) / groups, 1);
  return means.index_select(0, row_samples(offsets, o, x.size(0)));
}

Tensor call_group_mean(const Tensor& t, const Tensor& offsets, const std::optional<Tensor>& order, int64_t groups) {
  static const auto op = registered<decltype(group_mean)>("torchsparse_b200::group_mean");
  return op.call(t, offsets, order, groups);
}

// Every value of a sample and group has an equal share in the mean at every other: the gradient is the same operator.
struct GroupMeanBackward : torch::autograd::Node {
  torch::autograd::SavedVariable offsets, order;
  int64_t groups = 1;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(1);
    return {call_group_mean(grads[0], offsets.unpack(), given(order.unpack()), groups)};
  }
  void release_variables() override {
    offsets.reset_data();
    order.reset_data();
  }
  std::string name() const override { return "GroupMeanBackward"; }
};

Tensor group_mean_autograd(const Tensor& t, const Tensor& offsets, const std::optional<Tensor>& order, int64_t groups) {
  std::shared_ptr<GroupMeanBackward> node;
  if (torch::autograd::compute_requires_grad(t)) {
    node = std::make_shared<GroupMeanBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(t));
    node->offsets = torch::autograd::SavedVariable(offsets, false);
    node->order = torch::autograd::SavedVariable(order.value_or(Tensor()), false);
    node->groups = groups;
  }
  Tensor mean;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    mean = call_group_mean(t, offsets, order, groups);
  }
  if (node) torch::autograd::set_history(mean, node);
  if (has_tangent(t)) mean._set_fw_grad(call_group_mean(tangent(t), offsets, order, groups), /*level=*/0, /*is_inplace_op=*/false);
  return mean;
}

// The same in torch's own operations and group_mean, for a gradient that is to be differentiated again (a gradient penalty) and
// for forward-mode tangents and functional transforms: slower, and differentiable as often as wanted.
Tensor norm_by_torch(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& offsets, const Tensor& order, const NormArgs& a) {
  const Tensor inside = row_samples(offsets, order, x.size(0)).lt(offsets.size(0) - 1).unsqueeze(1);
  const auto mean = [&](const Tensor& t) { return call_group_mean(t, offsets, given(order), a.groups); };
  const Tensor v = x.to(at::kFloat), zero = at::zeros({}, v.options());
  const Tensor rows = at::where(inside, v, zero), d = rows - mean(rows);
  Tensor z = d * (mean(d * d) + a.eps).rsqrt();
  if (w.defined()) z = z * w.to(at::kFloat);
  if (b.defined()) z = z + b.to(at::kFloat);
  z = a.act == 1 ? at::relu(z) : a.act == 2 ? at::leaky_relu(z, a.slope) : a.act == 3 ? z * at::sigmoid(z) : z;      // silu's gradient has no tangent
  return at::where(inside, z, zero).to(x.scalar_type());
}

Tensor group_norm(const Tensor& feats, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, const Tensor& offsets,
                  const std::optional<Tensor>& order, int64_t groups, double eps, int64_t act, double slope) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor()), o = order.value_or(Tensor());
  const int code = check_norm(feats, w, b, offsets, o, groups);
  return norm_forward(packed(feats), packed(w), packed(b), offsets, o, NormArgs{groups, eps, slope, act}, code, false).first;
}

// with the means and reciprocal deviations that the gradient needs
std::tuple<Tensor, Tensor> group_norm_stats(const Tensor& feats, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                                            const Tensor& offsets, const std::optional<Tensor>& order, int64_t groups, double eps,
                                            int64_t act, double slope) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor()), o = order.value_or(Tensor());
  const int code = check_norm(feats, w, b, offsets, o, groups);
  return norm_forward(packed(feats), packed(w), packed(b), offsets, o, NormArgs{groups, eps, slope, act}, code, true);
}

std::tuple<Tensor, Tensor, Tensor> group_norm_backward(const Tensor& grad, const Tensor& feats, const std::optional<Tensor>& weight,
                                                       const std::optional<Tensor>& bias, const Tensor& offsets,
                                                       const std::optional<Tensor>& order_, const Tensor& stats_, int64_t groups,
                                                       int64_t act, double slope) {
  const Tensor x = packed(feats), dy = packed(grad), w = packed(weight.value_or(Tensor())), b = packed(bias.value_or(Tensor()));
  const Tensor order = order_.value_or(Tensor()), stats = packed(stats_);
  const int code = check_norm(x, w, b, offsets, order, groups);
  same_device(x, {dy, stats});
  const int64_t n = x.size(0), c = x.size(1), samples = offsets.size(0) - 1;
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(), "the gradient is not like the features");
  TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.numel() == 2 * samples * groups, "stats must be fp32 [2, ", samples, ", ",
                    groups, "]");
  Call call(x);
  Tensor dx = at::empty_like(x), dw, db;
  if (w.defined()) dw = at::empty_like(w);
  if (b.defined()) db = at::empty_like(b);
  const float* mean = stats.const_data_ptr<float>();
  const int dtype = dtype_code(x);
  void* ws = call.workspace(tsb_group_norm_bwd_workspace_bytes(n, c, groups, samples, dtype), x);
  check_status(tsb_group_norm_bwd(ptr(x), ptr(dy), ints(order), ints(offsets), ptr(w), ptr(b), mean, mean + samples * groups, n, c,
                                  groups, samples, (int)act, (float)slope, dtype, code, out_ptr(dx), out_ptr(dw), out_ptr(db), ws,
                                  call.bytes, call.stream()),
               "group_norm_backward");
  return {dx, dw, db};
}

Tensor call_group_norm(const Tensor& feats, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                       const Tensor& offsets, const std::optional<Tensor>& order, int64_t groups, double eps, int64_t act,
                       double slope) {
  static const auto op = registered<decltype(group_norm)>("torchsparse_b200::group_norm");
  return op.call(feats, weight, bias, offsets, order, groups, eps, act, slope);
}

struct GroupNorm : Function<GroupNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                        const Tensor& offsets, const std::optional<Tensor>& order, int64_t groups, double eps, int64_t act,
                        double slope) {
    static const auto op = registered<decltype(group_norm_stats)>("torchsparse_b200::group_norm_stats");
    at::AutoDispatchBelowAutograd below;
    auto [y, stats] = op.call(x, weight, bias, offsets, order, groups, eps, act, slope);
    ctx->save_for_backward({x, weight.value_or(Tensor()), bias.value_or(Tensor()), offsets, order.value_or(Tensor()), stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["act"] = act;
    ctx->saved_data["slope"] = slope;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &offsets = saved[3], &order = saved[4], &stats = saved[5];
    const NormArgs a{ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["slope"].toDouble(),
                     ctx->saved_data["act"].toInt()};
    variable_list made(9);
    const bool again = at::GradMode::is_enabled();
    if (again || has_tangent(grads[0])) {
      at::AutoGradMode record(true);
      variable_list wanted;
      for (const Tensor* t : {&x, &w, &b})
        if (t->defined() && t->requires_grad()) wanted.push_back(*t);
      const auto got = torch::autograd::grad({norm_by_torch(x, w, b, offsets, order, a)}, wanted, {grads[0]}, /*retain_graph=*/again,
                                             /*create_graph=*/again, /*allow_unused=*/true);
      size_t k = 0, i = 0;
      for (const Tensor* t : {&x, &w, &b}) {
        if (t->defined() && t->requires_grad()) made[i] = got[k++];
        ++i;
      }
      return made;
    }
    static const auto op = registered<decltype(group_norm_backward)>("torchsparse_b200::group_norm_backward");
    std::tie(made[0], made[1], made[2]) =
        op.call(grads[0], x, given(w), given(b), offsets, given(order), stats, a.groups, a.act, a.slope);
    return made;
  }
};

Tensor group_norm_autograd(const Tensor& feats, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                           const Tensor& offsets, const std::optional<Tensor>& order, int64_t groups, double eps, int64_t act,
                           double slope) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  const bool wanted = wants_grad({feats, w, b});
  if (has_tangent(feats) || has_tangent(w) || has_tangent(b) || (wanted && in_transform())) {
    check_norm(feats, w, b, offsets, order.value_or(Tensor()), groups);
    return norm_by_torch(feats, w, b, offsets, order.value_or(Tensor()), NormArgs{groups, eps, slope, act});
  }
  if (!wanted) {
    at::AutoDispatchBelowAutograd below;
    return call_group_norm(feats, weight, bias, offsets, order, groups, eps, act, slope);
  }
  check_norm(feats, w, b, offsets, order.value_or(Tensor()), groups);
  return GroupNorm::apply(packed(feats), given(packed(w)), given(packed(b)), offsets, order, groups, eps, act, slope);
}

// ------------------------------------------------------------------------------------------------ embedding
void check_embedding(const Tensor& table, const Tensor& indices) {
  same_device(table, {indices});
  check_index(indices, "indices");
  dtype_code(table);
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(1) >= 1, "embedding expects a table [rows, channels], not ", table.sizes());
}

// padding: the row that gets no gradient, -1 for none
Tensor embedding(const Tensor& table_, const Tensor& indices, double scale, int64_t /*padding*/) {
  check_embedding(table_, indices);
  const Tensor table = packed(table_), flat = (indices.dim() == 1 ? indices : indices.reshape(-1)).contiguous();
  Call call(table);
  const int64_t n = flat.size(0), c = table.size(1);
  Tensor out = at::empty({n, c}, table.options());
  check_status(tsb_embedding_fwd(ptr(table), ptr(flat), flat.scalar_type() == at::kLong, n, table.size(0), c, (float)scale,
                                 dtype_code(table), out_ptr(out), call.stream()),
               "embedding");
  if (indices.dim() == 1) return out;
  auto shape = indices.sizes().vec();
  shape.push_back(c);
  return out.view(shape);
}

Tensor embedding_backward(const Tensor& grad, const Tensor& indices, int64_t rows, double scale, int64_t padding) {
  same_device(grad, {indices});
  check_index(indices, "indices");
  TORCH_CHECK_VALUE(grad.dim() == indices.dim() + 1 && grad.sizes().slice(0, indices.dim()) == indices.sizes() && grad.size(-1) >= 1 &&
                        rows >= 0,
                    "the gradient is not like the vectors of the indices");
  const int64_t n = indices.numel(), c = grad.size(-1);
  const Tensor dy = grad.contiguous(), flat = indices.contiguous();
  Call call(dy);
  Tensor dtable = at::empty({rows, c}, dy.options());
  const int dtype = dtype_code(dy);
  void* ws = call.workspace(tsb_embedding_bwd_workspace_bytes(n, rows, c, dtype), dy);
  check_status(tsb_embedding_bwd(ptr(dy), ptr(flat), flat.scalar_type() == at::kLong, n, rows, c, (float)scale, padding, dtype,
                                 out_ptr(dtable), ws, call.bytes, call.stream()),
               "embedding_backward");
  return dtable;
}

Tensor call_embedding(const Tensor& table, const Tensor& indices, double scale, int64_t padding) {
  static const auto op = registered<decltype(embedding)>("torchsparse_b200::embedding");
  return op.call(table, indices, scale, padding);
}

struct Embedding : Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& indices, double scale, int64_t padding) {
    at::AutoDispatchBelowAutograd below;
    ctx->save_for_backward({indices});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return call_embedding(table, indices, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = registered<decltype(embedding_backward)>("torchsparse_b200::embedding_backward");
    refuse_tangent(grads[0]);
    auto made = once({op.call(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
                              ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt())});
    made.resize(4);
    return made;
  }
};

Tensor embedding_autograd(const Tensor& table, const Tensor& indices, double scale, int64_t padding) {
  if (has_tangent(table))      // linear
    return dual(call_embedding(primal(table), indices, scale, padding), call_embedding(tangent(table), indices, scale, padding));
  if (!wants_grad({table})) {
    at::AutoDispatchBelowAutograd below;
    return call_embedding(table, indices, scale, padding);
  }
  check_embedding(table, indices);
  const Tensor flat = (indices.dim() == 1 ? indices : indices.reshape(-1)).contiguous();
  const Tensor out = Embedding::apply(packed(table), flat, scale, padding);
  if (indices.dim() == 1) return out;
  auto shape = indices.sizes().vec();
  shape.push_back(table.size(1));
  return out.view(shape);
}

// ------------------------------------------------------------------------------------------------ experts
// the plan of [N, k] choices: (N, k, address of the number of kept choices)
std::tuple<int64_t, int32_t, const int32_t*> plan(const Tensor& inverse, const Tensor& offsets) {
  TORCH_CHECK_VALUE(inverse.dim() == 2 && inverse.scalar_type() == at::kInt && inverse.is_contiguous() && inverse.size(1) >= 1 &&
                        inverse.size(1) < (1ll << 31),
                    "inverse must be contiguous int32 [N, k]");
  check_int32(offsets, -1, "offsets");
  TORCH_CHECK_VALUE(offsets.size(0) >= 2, "offsets must hold the first position of every expert and the end of the last");
  return {inverse.size(0), (int32_t)inverse.size(1), ints(offsets) + offsets.size(0) - 1};
}

Tensor expert_dispatch(const Tensor& feats, const Tensor& inverse, const Tensor& offsets) {
  same_device(feats, {inverse, offsets});
  const auto [n, k, kept] = plan(inverse, offsets);
  TORCH_CHECK_VALUE(feats.dim() == 2 && feats.size(0) == n && feats.size(1) >= 1, "expert_dispatch expects features [", n, ", C], not ",
                    feats.sizes());
  const int dtype = dtype_code(feats);
  const Tensor x = packed(feats);
  Call call(x);
  Tensor out = at::empty({n * k, x.size(1)}, x.options());
  check_status(tsb_expert_dispatch(ptr(x), ints(inverse), kept, n, k, x.size(1), dtype, out_ptr(out), call.stream()),
               "expert_dispatch");
  return out;
}

void check_combine(const Tensor& rows, const Tensor& weights, int64_t n, int64_t k) {
  TORCH_CHECK_VALUE(rows.dim() == 2 && rows.size(0) == n * k && rows.size(1) >= 1, "expert_combine expects sorted rows [", n * k,
                    ", C], not ", rows.sizes());
  dtype_code(rows);
  if (!weights.defined()) return;
  TORCH_CHECK_VALUE(weights.dim() == 2 && weights.size(0) == n && weights.size(1) == k, "expert_combine expects weights [", n, ", ", k,
                    "], not ", weights.sizes());
  dtype_code(weights);
}

// no weights: 1
Tensor expert_combine(const Tensor& feats, const std::optional<Tensor>& weights_, const Tensor& inverse, const Tensor& offsets) {
  const Tensor rows = packed(feats), weights = packed(weights_.value_or(Tensor()));
  same_device(rows, {weights, inverse, offsets});
  const auto [n, k, kept] = plan(inverse, offsets);
  check_combine(rows, weights, n, k);
  Call call(rows);
  Tensor out = at::empty({n, rows.size(1)}, rows.options());
  check_status(tsb_expert_combine(ptr(rows), ptr(weights), weights.defined() ? dtype_code(weights) : (int)TSB_F32, ints(inverse), kept,
                                  n, k, rows.size(1), dtype_code(rows), out_ptr(out), call.stream()),
               "expert_combine");
  return out;
}

std::tuple<Tensor, Tensor> expert_combine_backward(const Tensor& grad, const Tensor& feats, const Tensor& weights_,
                                                   const Tensor& inverse, const Tensor& offsets) {
  const Tensor dout = packed(grad), rows = packed(feats), weights = packed(weights_);
  same_device(rows, {dout, weights, inverse, offsets});
  const auto [n, k, kept] = plan(inverse, offsets);
  check_combine(rows, weights, n, k);
  TORCH_CHECK_VALUE(dout.dim() == 2 && dout.size(0) == n && dout.size(1) == rows.size(1) && dout.scalar_type() == rows.scalar_type(),
                    "the gradient is not like the sums of the rows");
  Call call(rows);
  Tensor drows = at::empty_like(rows), dweights = at::empty_like(weights);
  check_status(tsb_expert_combine_bwd(ptr(dout), ptr(rows), ptr(weights), dtype_code(weights), ints(inverse), kept, n, k, rows.size(1),
                                      dtype_code(rows), out_ptr(drows), out_ptr(dweights), call.stream()),
               "expert_combine_backward");
  return {drows, dweights};
}

Tensor call_expert_dispatch(const Tensor& feats, const Tensor& inverse, const Tensor& offsets) {
  static const auto op = registered<decltype(expert_dispatch)>("torchsparse_b200::expert_dispatch");
  return op.call(feats, inverse, offsets);
}

Tensor call_expert_combine(const Tensor& feats, const std::optional<Tensor>& weights, const Tensor& inverse, const Tensor& offsets) {
  static const auto op = registered<decltype(expert_combine)>("torchsparse_b200::expert_combine");
  return op.call(feats, weights, inverse, offsets);
}

struct Dispatch : Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& inverse, const Tensor& offsets) {
    at::AutoDispatchBelowAutograd below;
    ctx->save_for_backward({inverse, offsets});
    return call_expert_dispatch(x, inverse, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    refuse_tangent(grads[0]);
    Tensor dx;
    {
      at::AutoDispatchBelowAutograd below;
      dx = call_expert_combine(grads[0], std::nullopt, saved[0], saved[1]);
    }
    auto made = once({dx});
    made.resize(3);
    return made;
  }
};

struct Combine : Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights, const Tensor& inverse, const Tensor& offsets) {
    at::AutoDispatchBelowAutograd below;
    ctx->save_for_backward({rows, weights, inverse, offsets});
    return call_expert_combine(rows, weights, inverse, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = registered<decltype(expert_combine_backward)>("torchsparse_b200::expert_combine_backward");
    const auto saved = ctx->get_saved_variables();
    refuse_tangent(grads[0]);
    auto [drows, dweights] = op.call(grads[0], saved[0], saved[1], saved[2], saved[3]);
    auto made = once({drows, dweights});
    made.resize(4);
    return made;
  }
};

Tensor expert_dispatch_autograd(const Tensor& feats, const Tensor& inverse, const Tensor& offsets) {
  if (has_tangent(feats))      // linear
    return dual(call_expert_dispatch(primal(feats), inverse, offsets), call_expert_dispatch(tangent(feats), inverse, offsets));
  if (wants_grad({feats})) return Dispatch::apply(packed(feats), inverse, offsets);
  at::AutoDispatchBelowAutograd below;
  return call_expert_dispatch(feats, inverse, offsets);
}

Tensor expert_combine_autograd(const Tensor& feats, const std::optional<Tensor>& weights, const Tensor& inverse,
                               const Tensor& offsets) {
  const bool moves = has_tangent(feats), weighs = weights.has_value() && has_tangent(*weights);
  if (moves || weighs) {      // linear in both
    const std::optional<Tensor> w = weights.has_value() ? std::optional<Tensor>(primal(*weights)) : std::nullopt;
    const Tensor rows = primal(feats);
    Tensor t;
    if (moves) t = call_expert_combine(tangent(feats), w, inverse, offsets);
    if (weighs) {
      const Tensor by_weights = call_expert_combine(rows, tangent(*weights), inverse, offsets);
      t = t.defined() ? t + by_weights : by_weights;
    }
    return dual(call_expert_combine(rows, w, inverse, offsets), t);
  }
  if (wants_grad({feats, weights.value_or(Tensor())})) {
    TORCH_CHECK(weights.has_value(), "expert_combine without weights has no gradient");
    return Combine::apply(packed(feats), packed(*weights), inverse, offsets);
  }
  at::AutoDispatchBelowAutograd below;
  return call_expert_combine(feats, weights, inverse, offsets);
}

}  // namespace

TORCH_LIBRARY(torchsparse_b200, m) {
  m.def("group_rows(Tensor keys, int num_groups) -> (Tensor, Tensor)");
  m.def("expert_sort(Tensor experts, int num_experts) -> (Tensor, Tensor, Tensor)");
  m.def("group_mean(Tensor t, Tensor offsets, Tensor? order, int groups) -> Tensor");
  m.def("group_norm(Tensor feats, Tensor? weight, Tensor? bias, Tensor offsets, Tensor? order, int groups, float eps, int act, "
        "float slope) -> Tensor");
  m.def("group_norm_stats(Tensor feats, Tensor? weight, Tensor? bias, Tensor offsets, Tensor? order, int groups, float eps, int act, "
        "float slope) -> (Tensor, Tensor)");
  m.def("group_norm_backward(Tensor grad, Tensor feats, Tensor? weight, Tensor? bias, Tensor offsets, Tensor? order, Tensor stats, "
        "int groups, int act, float slope) -> (Tensor, Tensor, Tensor)");
  m.def("embedding(Tensor table, Tensor indices, float scale, int padding) -> Tensor");
  m.def("embedding_backward(Tensor grad, Tensor indices, int rows, float scale, int padding) -> Tensor");
  m.def("expert_dispatch(Tensor feats, Tensor inverse, Tensor offsets) -> Tensor");
  m.def("expert_combine(Tensor feats, Tensor? weights, Tensor inverse, Tensor offsets) -> Tensor");
  m.def("expert_combine_backward(Tensor grad, Tensor feats, Tensor weights, Tensor inverse, Tensor offsets) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(torchsparse_b200, CompositeExplicitAutograd, m) {
  m.impl("group_rows", &group_rows);
  m.impl("expert_sort", &expert_sort);
  m.impl("group_mean", &group_mean);
  m.impl("group_norm", &group_norm);
  m.impl("group_norm_stats", &group_norm_stats);
  m.impl("group_norm_backward", &group_norm_backward);
  m.impl("embedding", &embedding);
  m.impl("embedding_backward", &embedding_backward);
  m.impl("expert_dispatch", &expert_dispatch);
  m.impl("expert_combine", &expert_combine);
  m.impl("expert_combine_backward", &expert_combine_backward);
}

TORCH_LIBRARY_IMPL(torchsparse_b200, Autograd, m) {
  m.impl("group_mean", &group_mean_autograd);
  m.impl("group_norm", &group_norm_autograd);
  m.impl("embedding", &embedding_autograd);
  m.impl("expert_dispatch", &expert_dispatch_autograd);
  m.impl("expert_combine", &expert_combine_autograd);
  for (const char* name : {"group_rows", "expert_sort"}) m.impl(name, torch::CppFunction::makeFallthrough());      // integers only
  for (const char* name : {"group_norm_stats", "group_norm_backward", "embedding_backward", "expert_combine_backward"})
    m.impl(name, torch::CppFunction::makeFallthrough());      // parts of the nodes above, which are what autograd sees
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("group_rows", &call_group_rows);
  m.def("expert_sort", &call_expert_sort);
  m.def("group_norm", &call_group_norm);
  m.def("embedding", &call_embedding);
  m.def("expert_dispatch", &call_expert_dispatch);
  m.def("expert_combine", [](const Tensor& feats, const Tensor& weights, const Tensor& inverse, const Tensor& offsets) {
    return call_expert_combine(feats, weights, inverse, offsets);
  });
}
