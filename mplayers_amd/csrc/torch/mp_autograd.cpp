// The operators around the layers as torch sees them: checks, results and autograd nodes over the C ABI.  Host code,
// compiled against torch's headers.
//
// Their kernels take a few microseconds, and autograd runs a gradient in a thread of its own.  A node in Python has to
// get the interpreter there and give it back; these do not touch it.  Host time, us, in Python -> here: a forward call of a
// bucketed table 11 -> 5.5, with its gradient 40 -> 28 (82 -> 50 where the machine takes longer to wake the thread), dropout
// of 16 labels 64x96 with its gradient 40 -> 37 (88 -> 52), a draw of as many 9.9 -> 5.0.
//
// The entry points are those of the library that the ctypes binding has loaded (bind), not of one found by the linker.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <limits>

#include "mplayers_amd.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

struct EntryPoints {
  decltype(&mpl_bucket_context) bucket_context;
  decltype(&mpl_bucket_sums) bucket_sums;
  decltype(&mpl_dropout_labels_last) dropout_labels_last;
  decltype(&mpl_dropout_labels_first) dropout_labels_first;
  decltype(&mpl_sample_labels) sample_labels;
  decltype(&mpl_norm_labels_last) norm_labels_last;
  decltype(&mpl_norm_labels_last_grad) norm_labels_last_grad;
  decltype(&mpl_norm_workspace) norm_workspace;
  decltype(&mpl_norm_stats) norm_stats;
  decltype(&mpl_best_labels) best_labels;
  decltype(&mpl_distill_costs) distill_costs;
  decltype(&mpl_distill_costs_grad) distill_costs_grad;
  decltype(&mpl_verify_labels) verify_labels;
  decltype(&mpl_last_error) last_error;
} lib;

void bind(const std::vector<uintptr_t>& at) {
  size_t next = 0;
  const auto take = [&](auto& entry) {
    TORCH_CHECK(next < at.size(), "bind: ", at.size(), " entry points are too few");
    entry = reinterpret_cast<std::remove_reference_t<decltype(entry)>>(at[next++]);
  };
  take(lib.bucket_context);
  take(lib.bucket_sums);
  take(lib.dropout_labels_last);
  take(lib.dropout_labels_first);
  take(lib.sample_labels);
  take(lib.norm_labels_last);
  take(lib.norm_labels_last_grad);
  take(lib.norm_workspace);
  take(lib.norm_stats);
  take(lib.best_labels);
  take(lib.distill_costs);
  take(lib.distill_costs_grad);
  take(lib.verify_labels);
  take(lib.last_error);
  TORCH_CHECK(next == at.size(), "bind: ", at.size(), " entry points are too many");
}

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check(int rc, const char* what) { TORCH_CHECK(rc == MPL_OK, what, " failed (", rc, "): ", lib.last_error()); }
// a size that the entry points take as an int
int small(int64_t size) {
  TORCH_CHECK(size <= std::numeric_limits<int>::max(), "a size of ", size, " is too large");
  return (int)size;
}
// whether a tensor carries a derivative of the forward mode, which the functions have none of: apply() refuses it, and what
// goes past apply() would lose it without a word
bool has_tangent(const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }
// whether autograd is to know of what is made of a tensor
bool recorded(const at::Tensor& t) { return (at::GradMode::is_enabled() && t.requires_grad()) || has_tangent(t); }

// ------------------------------------------------------------------------------------------------ bucketed tables
at::Tensor expand(const at::Tensor& table_in, const at::Tensor& starts, int64_t n, int64_t square) {
  const at::Tensor table = table_in.contiguous();
  std::vector<int64_t> size = table.sizes().vec();
  const int64_t buckets = size.back();
  size.back() = n;
  if (square) size.push_back(n);
  at::Tensor out = at::empty(size, table.options());
  if (out.numel() == 0) return out;
  const c10::DeviceGuard guard(table.device());
  check(lib.bucket_context(table.data_ptr<float>(), starts.data_ptr<int32_t>(), small(table.numel() / buckets),
                           (int)buckets, (int)n, (int)square, out.data_ptr<float>(), stream_of(table)),
        "bucket_context");
  return out;
}

at::Tensor sums(const at::Tensor& grad_in, const at::Tensor& starts, int64_t n, int64_t square) {
  const at::Tensor grad = grad_in.contiguous();
  std::vector<int64_t> size = grad.sizes().vec();
  const int64_t buckets = starts.numel() - 1;
  if (square) size.pop_back();
  size.back() = buckets;
  at::Tensor out = at::empty(size, grad.options());
  if (out.numel() == 0) return out;
  const c10::DeviceGuard guard(grad.device());
  check(lib.bucket_sums(grad.data_ptr<float>(), starts.data_ptr<int32_t>(), small(out.numel() / buckets), small(buckets),
                        (int)n, (int)square, out.data_ptr<float>(), stream_of(grad)),
        "bucket_sums");
  return out;
}

// Each is the other's gradient: the maps are linear.
struct BucketSums : Function<BucketSums> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& grad, const at::Tensor& starts, int64_t n, int64_t square);
  static variable_list backward(AutogradContext* ctx, const variable_list& grads);
};
struct BucketContext : Function<BucketContext> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& table, const at::Tensor& starts, int64_t n, int64_t square) {
    ctx->save_for_backward({starts});
    ctx->saved_data["n"] = n;
    ctx->saved_data["square"] = square;
    return expand(table, starts, n, square);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const at::Tensor starts = ctx->get_saved_variables()[0];
    const int64_t n = ctx->saved_data["n"].toInt(), square = ctx->saved_data["square"].toInt();
    return {recorded(grads[0]) ? BucketSums::apply(grads[0], starts, n, square) : sums(grads[0], starts, n, square), {}, {}, {}};
  }
};
at::Tensor BucketSums::forward(AutogradContext* ctx, const at::Tensor& grad, const at::Tensor& starts, int64_t n, int64_t square) {
  ctx->save_for_backward({starts});
  ctx->saved_data["n"] = n;
  ctx->saved_data["square"] = square;
  return sums(grad, starts, n, square);
}
variable_list BucketSums::backward(AutogradContext* ctx, const variable_list& grads) {
  const at::Tensor starts = ctx->get_saved_variables()[0];
  return {BucketContext::apply(grads[0], starts, ctx->saved_data["n"].toInt(), ctx->saved_data["square"].toInt()), {}, {}, {}};
}

at::Tensor bucket_context(const at::Tensor& table, const at::Tensor& starts, bool square, bool symmetric) {
  TORCH_CHECK(table.is_cuda(), "bucket_context: table must be a GPU tensor here");
  TORCH_CHECK(!starts.is_cuda() && starts.scalar_type() == at::kInt && starts.dim() == 1 && starts.is_contiguous(),
              "bucket_context: starts must be an int32 CPU tensor, as label_buckets returns it");
  TORCH_CHECK(table.scalar_type() == at::kFloat, "bucket_context: table must be float32, got ", table.scalar_type());
  TORCH_CHECK(table.dim() >= 1 && starts.numel() >= 2 && table.size(-1) == starts.numel() - 1, "bucket_context: table has ",
              table.dim() ? table.size(-1) : 0, " entries for ", starts.numel() - 1, " buckets");
  const int64_t n = starts.data_ptr<int32_t>()[starts.numel() - 1];
  TORCH_CHECK(n >= 1 && n <= MPL_MAX_LABELS, "bucket_context: 1 to 256 labels, got ", n);
  return BucketContext::apply(table, starts, n, (int64_t)(square ? symmetric ? 2 : 1 : 0));
}

// --------------------------------------------------------------------------------------------------------- dropout
int mpl_type(at::ScalarType type) {
  return type == at::kFloat ? MPL_F32 : type == at::kHalf ? MPL_F16 : type == at::kBFloat16 ? MPL_BF16 : -1;
}

at::Tensor dropout_last(const at::Tensor& x_in, const at::Tensor& state, double p, int64_t share) {
  const at::Tensor x = x_in.contiguous();
  const auto s = x.sizes();
  at::Tensor out = at::empty({s[0], s[1], s[3], s[4], s[2]}, x.options().dtype(at::kFloat));
  if (out.numel() == 0) return out;
  const c10::DeviceGuard guard(x.device());
  check(lib.dropout_labels_last(mpl_type(x.scalar_type()), (int)share, p, state.data_ptr<int64_t>(), x.data_ptr(),
                                out.data_ptr<float>(), small(s[0] * s[1]), (int)s[2], s[3] * s[4], stream_of(x)),
        "dropout_labels_last");
  return out;
}

at::Tensor dropout_first(const at::Tensor& grad_in, const at::Tensor& state, double p, int64_t share, at::ScalarType type) {
  const at::Tensor grad = grad_in.contiguous();
  const auto s = grad.sizes();
  at::Tensor out = at::empty({s[0], s[1], s[4], s[2], s[3]}, grad.options().dtype(type));
  if (out.numel() == 0) return out;
  const c10::DeviceGuard guard(grad.device());
  check(lib.dropout_labels_first(mpl_type(type), (int)share, p, state.data_ptr<int64_t>(), grad.data_ptr<float>(),
                                 out.data_ptr(), small(s[0] * s[1]), (int)s[4], s[2] * s[3], stream_of(grad)),
        "dropout_labels_first");
  return out;
}

struct DropoutFirst : Function<DropoutFirst> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& grad, const at::Tensor& state, double p, int64_t share,
                            int64_t type);
  static variable_list backward(AutogradContext* ctx, const variable_list& grads);
};
struct DropoutLast : Function<DropoutLast> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& state, double p, int64_t share) {
    ctx->save_for_backward({state});
    ctx->saved_data["p"] = p;
    ctx->saved_data["share"] = share;
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    return dropout_last(x, state, p, share);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const at::Tensor state = ctx->get_saved_variables()[0];
    const double p = ctx->saved_data["p"].toDouble();
    const int64_t share = ctx->saved_data["share"].toInt(), type = ctx->saved_data["type"].toInt();
    return {recorded(grads[0]) ? DropoutFirst::apply(grads[0], state, p, share, type)
                               : dropout_first(grads[0], state, p, share, (at::ScalarType)type),
            {}, {}, {}};
  }
};
at::Tensor DropoutFirst::forward(AutogradContext* ctx, const at::Tensor& grad, const at::Tensor& state, double p, int64_t share,
                                 int64_t type) {
  ctx->save_for_backward({state});
  ctx->saved_data["p"] = p;
  ctx->saved_data["share"] = share;
  return dropout_first(grad, state, p, share, (at::ScalarType)type);
}
variable_list DropoutFirst::backward(AutogradContext* ctx, const variable_list& grads) {
  const at::Tensor state = ctx->get_saved_variables()[0];
  return {DropoutLast::apply(grads[0], state, ctx->saved_data["p"].toDouble(), ctx->saved_data["share"].toInt()), {}, {}, {}, {}};
}

at::Tensor labels_last_dropout(const at::Tensor& x, double p, const at::Tensor& state, const std::string& share) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 5, "labels_last_dropout: x must be a (batch, cv, labels, H, W) GPU tensor");
  TORCH_CHECK(mpl_type(x.scalar_type()) >= 0, "labels_last_dropout: x must be float32, float16 or bfloat16, got ",
              x.scalar_type());
  TORCH_CHECK(x.size(2) >= 1 && x.size(2) <= MPL_MAX_LABELS, "labels_last_dropout: 1 to 256 labels, got ", x.size(2));
  TORCH_CHECK(state.device() == x.device() && state.scalar_type() == at::kLong && state.dim() == 1 && state.numel() == 2 &&
                  state.is_contiguous(),
              "labels_last_dropout: state must be two int64 numbers (seed, offset) on the device of x");
  TORCH_CHECK(p >= 0 && p <= 1, "labels_last_dropout: p must be in [0, 1], got ", p);
  const int64_t kind = share == "element" ? MPL_DROPOUT_ELEMENT : share == "pixel" ? MPL_DROPOUT_PIXEL
                       : share == "label" ? MPL_DROPOUT_LABEL : -1;
  TORCH_CHECK(kind >= 0, "labels_last_dropout: share must be 'element', 'pixel' or 'label', got '", share, "'");
  return DropoutLast::apply(x, state, p, kind);
}

// ------------------------------------------------------------------------------------------------------ layer norm
// (batch, cv, H, W, labels) of a tensor in either layout
struct Layout {
  int64_t batch, cv, n, height, width;
  Layout(const at::Tensor& t, bool labels_first) {
    const auto s = t.sizes();
    batch = s[0];
    cv = s[1];
    n = s[labels_first ? 2 : 4];
    height = s[labels_first ? 3 : 2];
    width = s[labels_first ? 4 : 3];
  }
  int64_t pixels() const { return height * width; }
};
template <typename T>
T* or_null(const at::Tensor& t) {
  return t.defined() ? t.data_ptr<T>() : nullptr;
}
void* data_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// y, and what its gradient takes (undefined where that is nothing, or not asked for)
std::pair<at::Tensor, at::Tensor> norm_last(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, double eps,
                                            bool labels_first, bool with_stats) {
  const Layout s(x, labels_first);
  const auto single = x.options().dtype(at::kFloat);
  at::Tensor y = at::empty({s.batch, s.cv, s.height, s.width, s.n}, single), stats;
  const int kept = with_stats ? lib.norm_stats((int)s.n) : 0;
  if (kept > 0) stats = at::empty({s.batch, s.cv, s.height, s.width, kept}, single);
  const c10::DeviceGuard guard(x.device());
  check(lib.norm_labels_last(mpl_type(x.scalar_type()), labels_first, x.data_ptr(), or_null<float>(weight), or_null<float>(bias),
                             (float)eps, y.data_ptr<float>(), or_null<float>(stats), small(s.batch * s.cv), (int)s.n, s.pixels(),
                             stream_of(x)),
        "labels_last_norm");
  return {y, stats};
}

// dx, dweight, dbias, undefined where they are not asked for
variable_list norm_grad(const at::Tensor& grad_in, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& stats, double eps,
                        bool labels_first, bool with_x, bool with_weight, bool with_bias) {
  const at::Tensor grad = grad_in.contiguous();
  const Layout s(x, labels_first);
  const c10::DeviceGuard guard(x.device());
  at::Tensor dx, dweight, dbias, workspace;
  if (with_x) dx = at::empty_like(x);
  if (with_weight) dweight = at::empty({s.n}, grad.options());
  if (with_bias) dbias = at::empty({s.n}, grad.options());
  const int items = small(s.batch * s.cv);
  if (with_weight || with_bias) workspace = at::empty({lib.norm_workspace(items, (int)s.n, s.pixels())}, grad.options());
  check(lib.norm_labels_last_grad(mpl_type(x.scalar_type()), labels_first, x.data_ptr(), or_null<float>(weight), (float)eps,
                                  or_null<float>(stats), grad.data_ptr<float>(), data_or_null(dx), or_null<float>(dweight), or_null<float>(dbias),
                                  or_null<float>(workspace), items, (int)s.n, s.pixels(), stream_of(x)),
        "labels_last_norm's gradient");
  return {dx, dweight, dbias};
}

// The gradient where it is recorded for another one, which there is none of: an error when that is asked for, not before.
struct NormGrad : Function<NormGrad> {
  static variable_list forward(AutogradContext*, const at::Tensor& grad, const at::Tensor& x, const std::optional<at::Tensor>& weight,
                               const std::optional<at::Tensor>& stats, double eps, bool labels_first, bool with_x, bool with_weight,
                               bool with_bias) {
    variable_list out = norm_grad(grad, x, weight.value_or(at::Tensor()), stats.value_or(at::Tensor()), eps, labels_first, with_x,
                                  with_weight, with_bias);
    for (at::Tensor& t : out)
      if (!t.defined()) t = at::empty({0}, grad.options());
    return out;
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "labels_last_norm cannot be differentiated twice");
  }
};
struct NormLast : Function<NormLast> {
  // (an input that is not there takes no place among those that may need a gradient)
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x_in, const std::optional<at::Tensor>& weight_in,
                            const std::optional<at::Tensor>& bias_in, double eps, bool labels_first) {
    const at::Tensor x = x_in.contiguous(), weight = weight_in ? weight_in->contiguous() : at::Tensor(),
                     bias = bias_in ? bias_in->contiguous() : at::Tensor();
    ctx->saved_data["weight"] = weight_in.has_value();
    ctx->saved_data["bias"] = bias_in.has_value();
    const auto [y, stats] = norm_last(x, weight, bias, eps, labels_first, true);
    ctx->save_for_backward({x, weight, stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["labels_first"] = labels_first;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const double eps = ctx->saved_data["eps"].toDouble();
    const bool labels_first = ctx->saved_data["labels_first"].toBool();
    const bool weighted = ctx->saved_data["weight"].toBool();
    const bool wanted[] = {ctx->needs_input_grad(0), weighted && ctx->needs_input_grad(1),
                           ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weighted ? 2 : 1)};
    variable_list out;
    if (at::GradMode::is_enabled() || has_tangent(grads[0])) {
      out = NormGrad::apply(grads[0], saved[0], weighted ? std::optional<at::Tensor>(saved[1]) : std::nullopt,
                            saved[2].defined() ? std::optional<at::Tensor>(saved[2]) : std::nullopt, eps, labels_first,
                            wanted[0], wanted[1], wanted[2]);
      for (int k = 0; k < 3; ++k)
        if (!wanted[k]) out[k] = at::Tensor();
    } else {
      out = norm_grad(grads[0], saved[0], saved[1], saved[2], eps, labels_first, wanted[0], wanted[1], wanted[2]);
    }
    return {out[0], out[1], out[2], {}, {}};
  }
};

at::Tensor labels_last_norm(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& bias,
                            double eps, bool labels_first) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 5, "labels_last_norm: x must be a (batch, cv, labels, H, W) or (batch, cv, H, W, labels) "
              "GPU tensor");
  TORCH_CHECK(mpl_type(x.scalar_type()) >= 0, "labels_last_norm: x must be float32, float16 or bfloat16, got ", x.scalar_type());
  const int64_t n = Layout(x, labels_first).n;
  TORCH_CHECK(n >= 1 && n <= MPL_MAX_LABELS, "labels_last_norm: 1 to 256 labels, got ", n);
  bool through_autograd = recorded(x);
  const std::pair<const char*, const std::optional<at::Tensor>*> given[] = {{"weight", &weight}, {"bias", &bias}};
  for (const auto& [name, t] : given) {
    if (!t->has_value()) continue;
    TORCH_CHECK((*t)->device() == x.device() && (*t)->scalar_type() == at::kFloat && (*t)->dim() == 1 && (*t)->size(0) == n,
                "labels_last_norm: ", name, " must be ", n, " float32 numbers on the device of x");
    through_autograd |= recorded(**t);
  }
  TORCH_CHECK(eps >= 0 && eps <= std::numeric_limits<float>::max(), "labels_last_norm: eps must be finite and not below 0, got ", eps);
  if (through_autograd) return NormLast::apply(x, weight, bias, eps, labels_first);
  return norm_last(x.contiguous(), weight ? weight->contiguous() : at::Tensor(), bias ? bias->contiguous() : at::Tensor(), eps,
                   labels_first, false).first;
}

// ---------------------------------------------------------------------------------------- a teacher's best labels
void check_costs(const char* what, const at::Tensor& cost, bool labels_first) {
  TORCH_CHECK(cost.is_cuda() && cost.dim() == 5, what, ": cost must be a (batch, cv, labels, H, W) or (batch, cv, H, W, labels) "
              "GPU tensor");
  TORCH_CHECK(mpl_type(cost.scalar_type()) >= 0, what, ": cost must be float32, float16 or bfloat16, got ", cost.scalar_type());
  const int64_t n = Layout(cost, labels_first).n;
  TORCH_CHECK(n >= 1 && n <= MPL_MAX_LABELS, what, ": 1 to 256 labels, got ", n);
}
void check_temperature(const char* what, double t) {
  const float single = (float)t;
  const float most = std::numeric_limits<float>::max();
  TORCH_CHECK(single > 0 && single <= most && (float)(1.4426950408889634 / (double)single) <= most, what,
              ": temperature must be finite and above 0 (and its inverse finite), got ", t);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> best_labels(const at::Tensor& cost_in, int64_t k, double temperature,
                                                           bool labels_first, at::ScalarType type) {
  check_costs("best_labels", cost_in, labels_first);
  TORCH_CHECK(mpl_type(type) >= 0, "best_labels: dtype must be float32, float16 or bfloat16, got ", type);
  check_temperature("best_labels", temperature);
  const Layout s(cost_in, labels_first);
  TORCH_CHECK(k >= 1 && k <= s.n, "best_labels: k must be in [1, ", s.n, "], got ", k);
  const c10::DeviceGuard guard(cost_in.device());
  const at::Tensor cost = cost_in.detach().contiguous();
  const std::vector<int64_t> size = labels_first ? std::vector<int64_t>{s.batch, s.cv, k, s.height, s.width}
                                                 : std::vector<int64_t>{s.batch, s.cv, s.height, s.width, k};
  const at::Tensor labels = at::empty(size, cost.options().dtype(at::kByte)), costs = at::empty(size, cost.options().dtype(type)),
                   rest = at::empty({s.batch, s.cv, s.height, s.width}, cost.options().dtype(at::kFloat));
  check(lib.best_labels(mpl_type(cost.scalar_type()), labels_first, cost.data_ptr(), (int)k, (float)temperature, mpl_type(type),
                        labels.data_ptr<uint8_t>(), costs.data_ptr(), rest.data_ptr<float>(), small(s.batch * s.cv), (int)s.n,
                        s.pixels(), stream_of(cost)),
        "best_labels");
  return {labels, costs, rest};
}

// ------------------------------------------------------------------------------------- the divergence from a teacher
// cost, labels, costs and rest are contiguous; rest may be undefined
at::Tensor distill_loss(const at::Tensor& cost, const at::Tensor& labels, const at::Tensor& costs, const at::Tensor& rest,
                        double temperature, bool labels_first) {
  const Layout s(cost, labels_first);
  const c10::DeviceGuard guard(cost.device());
  at::Tensor loss = at::empty({s.batch, s.cv, s.height, s.width}, cost.options().dtype(at::kFloat));
  check(lib.distill_costs(mpl_type(cost.scalar_type()), labels_first, cost.data_ptr(), mpl_type(costs.scalar_type()),
                          labels.data_ptr<uint8_t>(), costs.data_ptr(), or_null<float>(rest), (float)temperature,
                          loss.data_ptr<float>(), small(s.batch * s.cv), (int)s.n, (int)Layout(labels, labels_first).n, s.pixels(),
                          stream_of(cost)),
        "distill_costs");
  return loss;
}
at::Tensor distill_grad(const at::Tensor& grad_in, const at::Tensor& cost, const at::Tensor& labels, const at::Tensor& costs,
                        const at::Tensor& rest, double temperature, bool labels_first) {
  const Layout s(cost, labels_first);
  const c10::DeviceGuard guard(cost.device());
  const at::Tensor grad = grad_in.contiguous();
  at::Tensor out = at::empty_like(cost);
  check(lib.distill_costs_grad(mpl_type(cost.scalar_type()), labels_first, cost.data_ptr(), mpl_type(costs.scalar_type()),
                               labels.data_ptr<uint8_t>(), costs.data_ptr(), or_null<float>(rest), (float)temperature,
                               grad.data_ptr<float>(), out.data_ptr(), small(s.batch * s.cv), (int)s.n,
                               (int)Layout(labels, labels_first).n, s.pixels(), stream_of(cost)),
        "distill_costs' gradient");
  return out;
}

struct DistillGrad : Function<DistillGrad> {  // (as NormGrad)
  static at::Tensor forward(AutogradContext*, const at::Tensor& grad, const at::Tensor& cost, const at::Tensor& labels,
                            const at::Tensor& costs, const std::optional<at::Tensor>& rest, double temperature, bool labels_first) {
    return distill_grad(grad, cost, labels, costs, rest.value_or(at::Tensor()), temperature, labels_first);
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "distill_costs cannot be differentiated twice");
  }
};
struct Distill : Function<Distill> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& cost_in, const at::Tensor& labels_in, const at::Tensor& costs_in,
                            const std::optional<at::Tensor>& rest_in, double temperature, bool labels_first) {
    const at::Tensor cost = cost_in.contiguous(), labels = labels_in.contiguous(), costs = costs_in.contiguous(),
                     rest = rest_in ? rest_in->contiguous() : at::Tensor();
    ctx->save_for_backward({cost, labels, costs, rest});
    ctx->saved_data["rest"] = rest.defined();
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["labels_first"] = labels_first;
    return distill_loss(cost, labels, costs, rest, temperature, labels_first);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    const double temperature = ctx->saved_data["temperature"].toDouble();
    const bool labels_first = ctx->saved_data["labels_first"].toBool(), with_rest = ctx->saved_data["rest"].toBool();
    return {at::GradMode::is_enabled() || has_tangent(grads[0])
                ? DistillGrad::apply(grads[0], s[0], s[1], s[2], with_rest ? std::optional<at::Tensor>(s[3]) : std::nullopt,
                                     temperature, labels_first)
                : distill_grad(grads[0], s[0], s[1], s[2], s[3], temperature, labels_first),
            {}, {}, {}, {}, {}};
  }
};

at::Tensor distill_costs(const at::Tensor& cost, const at::Tensor& labels, const at::Tensor& costs,
                         const std::optional<at::Tensor>& rest, double temperature, bool labels_first) {
  check_costs("distill_costs", cost, labels_first);
  check_temperature("distill_costs", temperature);
  const Layout s(cost, labels_first);
  const std::pair<const char*, const at::Tensor*> lists[] = {{"labels", &labels}, {"costs", &costs}};
  for (const auto& [name, t] : lists) {
    TORCH_CHECK(t->device() == cost.device() && t->dim() == 5, "distill_costs: ", name, " must be a list for every pixel, in the layout "
                "of cost and on its device");
    const Layout l(*t, labels_first);
    TORCH_CHECK(l.batch == s.batch && l.cv == s.cv && l.height == s.height && l.width == s.width && l.n >= 1 && l.n <= MPL_MAX_LABELS,
                "distill_costs: ", name, " must have 1 to 256 entries for each of ", s.batch, "x", s.cv, "x", s.height, "x", s.width,
                " pixels");
    TORCH_CHECK(!recorded(*t), "distill_costs: the teacher's ", name, " have no gradient");
  }
  TORCH_CHECK(labels.scalar_type() == at::kByte, "distill_costs: labels must be uint8, got ", labels.scalar_type());
  TORCH_CHECK(mpl_type(costs.scalar_type()) >= 0, "distill_costs: costs must be float32, float16 or bfloat16, got ",
              costs.scalar_type());
  TORCH_CHECK(labels.sizes() == costs.sizes(), "distill_costs: labels and costs must be of the same size");
  if (rest) {
    TORCH_CHECK(rest->device() == cost.device() && rest->scalar_type() == at::kFloat && rest->dim() == 4 && rest->size(0) == s.batch &&
                    rest->size(1) == s.cv && rest->size(2) == s.height && rest->size(3) == s.width,
                "distill_costs: rest must be a float32 (batch, cv, H, W) tensor on the device of cost");
    TORCH_CHECK(!recorded(*rest), "distill_costs: the teacher's rest has no gradient");
  }
  if (recorded(cost)) return Distill::apply(cost, labels, costs, rest, temperature, labels_first);
  return distill_loss(cost.contiguous(), labels.contiguous(), costs.contiguous(), rest ? rest->contiguous() : at::Tensor(), temperature,
                      labels_first);
}

// -------------------------------------------------------------------------------------------------- sampled labels
// A parameter: a number, or a tensor of one per image (not looked at).
template <typename T>
struct Parameter {
  const T* each = nullptr;
  T all = 0;

  // name: with the call's, as errors give it
  Parameter(const char* name, const py::object& value, int64_t batch, const at::Tensor& cost, at::ScalarType type, double high) {
    if (THPVariable_Check(value.ptr())) {
      const at::Tensor& t = THPVariable_Unpack(value.ptr());
      TORCH_CHECK(t.device() == cost.device(), name, " must be on the device of the costs");
      TORCH_CHECK(t.scalar_type() == type && t.dim() == 1 && t.size(0) == batch && t.is_contiguous(), name,
                  " must be a number or a contiguous ", type, " tensor of one per image (", batch, ")");
      each = t.data_ptr<T>();
      return;
    }
    TORCH_CHECK(type != at::kInt || (PyIndex_Check(value.ptr()) && !PyBool_Check(value.ptr())), name, " must be a whole number");
    const double number = PyFloat_AsDouble(value.ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
    TORCH_CHECK(number >= 0 && number <= high, name, " must be in [0, ", high, "], got ", number);
    all = (T)number;
  }
};

at::Tensor sample_labels(const at::Tensor& cost, const at::Tensor& uniforms, const py::object& temperature,
                         const py::object& top_k, const py::object& top_p, const py::object& min_p, bool labels_first) {
  const std::pair<const char*, const at::Tensor*> both[] = {{"cost", &cost}, {"uniforms", &uniforms}};
  for (const auto& [name, t] : both) {
    TORCH_CHECK(t->is_cuda(), "sample_labels: ", name, " must be a GPU tensor");
    TORCH_CHECK(t->scalar_type() == at::kFloat, "sample_labels: ", name, " must be float32, got ", t->scalar_type());
    TORCH_CHECK(t->is_contiguous(), "sample_labels: ", name, " must be contiguous");
  }
  TORCH_CHECK(uniforms.device() == cost.device(), "sample_labels: uniforms must be on the device of the costs");
  TORCH_CHECK(cost.dim() == 5, "sample_labels: cost must be (batch, cv, labels, H, W) or (batch, cv, H, W, labels)");
  const int first = labels_first ? 3 : 2;  // of H and W
  const int64_t batch = cost.size(0), cv = cost.size(1), n = cost.size(labels_first ? 2 : 4), height = cost.size(first),
                width = cost.size(first + 1);
  const int64_t at = uniforms.dim() - 4;
  TORCH_CHECK((at == 0 || at == 1) && uniforms.size(at) == batch && uniforms.size(at + 1) == cv &&
                  uniforms.size(at + 2) == height && uniforms.size(at + 3) == width,
              "sample_labels: uniforms must be ([n,] ", batch, ", ", cv, ", ", height, ", ", width, ")");
  const double inf = std::numeric_limits<double>::infinity();
  const Parameter<float> t("sample_labels: temperature", temperature, batch, cost, at::kFloat, inf);
  const Parameter<int32_t> k("sample_labels: top_k", top_k, batch, cost, at::kInt, 2147483647.0);
  const Parameter<float> p("sample_labels: top_p", top_p, batch, cost, at::kFloat, 1), m("sample_labels: min_p", min_p, batch, cost, at::kFloat, 1);
  at::Tensor labels = at::empty(uniforms.sizes(), uniforms.options().dtype(at::kByte));
  const c10::DeviceGuard guard(cost.device());
  check(lib.sample_labels(labels_first, cost.data_ptr<float>(), uniforms.data_ptr<float>(), small(batch), small(cv), small(n),
                          height * width, at == 1 ? small(uniforms.size(0)) : 1, t.each, t.all, k.each, k.all, p.each, p.all,
                          m.each, m.all, labels.data_ptr<uint8_t>(), stream_of(cost)),
        "sample_labels");
  return labels;
}

// ------------------------------------------------------------------------------------------------- verified labels
std::pair<at::Tensor, at::Tensor> verify_labels(const at::Tensor& cost, const at::Tensor& draft, const at::Tensor& uniforms,
                                                const std::optional<at::Tensor>& draft_cost, const py::object& temperature,
                                                const py::object& draft_temperature, bool labels_first) {
  const std::tuple<const char*, const at::Tensor*, at::ScalarType> all[] = {
      {"cost", &cost, at::kFloat}, {"draft", &draft, at::kByte}, {"uniforms", &uniforms, at::kFloat},
      {"draft_cost", draft_cost ? &*draft_cost : nullptr, at::kFloat}};
  for (const auto& [name, t, type] : all) {
    if (t == nullptr) continue;
    TORCH_CHECK(t->is_cuda(), "verify_labels: ", name, " must be a GPU tensor");
    TORCH_CHECK(t->scalar_type() == type, "verify_labels: ", name, " must be ", type, ", got ", t->scalar_type());
    TORCH_CHECK(t->is_contiguous(), "verify_labels: ", name, " must be contiguous");
    TORCH_CHECK(t->device() == cost.device(), "verify_labels: ", name, " must be on the device of the costs");
  }
  TORCH_CHECK(cost.dim() == 5, "verify_labels: cost must be (batch, cv, labels, H, W) or (batch, cv, H, W, labels)");
  TORCH_CHECK(!draft_cost || draft_cost->sizes() == cost.sizes(), "verify_labels: draft_cost must be of the size of cost");
  const Layout s(cost, labels_first);
  const int64_t at = draft.dim() - 4;
  TORCH_CHECK((at == 0 || at == 1) && draft.size(at) == s.batch && draft.size(at + 1) == s.cv && draft.size(at + 2) == s.height &&
                  draft.size(at + 3) == s.width,
              "verify_labels: draft must be ([n,] ", s.batch, ", ", s.cv, ", ", s.height, ", ", s.width, ")");
  TORCH_CHECK(uniforms.dim() == draft.dim() + 1 && uniforms.size(0) == 2 && uniforms.sizes().slice(1) == draft.sizes(),
              "verify_labels: uniforms must be two for each drafted label, (2, ...) of draft's size");
  const double inf = std::numeric_limits<double>::infinity();
  const Parameter<float> t("verify_labels: temperature", temperature, s.batch, cost, at::kFloat, inf),
      dt("verify_labels: draft_temperature", draft_temperature.is_none() ? temperature : draft_temperature, s.batch, cost, at::kFloat,
         inf);
  at::Tensor labels = at::empty(draft.sizes(), draft.options()), kept = at::empty(draft.sizes(), draft.options().dtype(at::kBool));
  const c10::DeviceGuard guard(cost.device());
  check(lib.verify_labels(labels_first, cost.data_ptr<float>(), draft.data_ptr<uint8_t>(),
                          draft_cost ? draft_cost->data_ptr<float>() : nullptr, uniforms.data_ptr<float>(), small(s.batch), small(s.cv),
                          small(s.n), s.pixels(), at == 1 ? small(draft.size(0)) : 1, t.each, t.all, dt.each, dt.all,
                          labels.data_ptr<uint8_t>(), reinterpret_cast<uint8_t*>(kept.data_ptr<bool>()), stream_of(cost)),
        "verify_labels");
  return {labels, kept};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("bucket_context", &bucket_context);
  m.def("labels_last_dropout", &labels_last_dropout);
  m.def("labels_last_norm", &labels_last_norm);
  m.def("best_labels", [](const at::Tensor& cost, int64_t k, double temperature, bool labels_first, const py::object& dtype) {
    TORCH_CHECK(THPDtype_Check(dtype.ptr()), "best_labels: dtype must be a torch.dtype");
    return best_labels(cost, k, temperature, labels_first, reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type);
  });
  m.def("distill_costs", &distill_costs);
  m.def("sample_labels", &sample_labels);
  m.def("verify_labels", &verify_labels);
}
