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
  decltype(&mpl_last_error) last_error;
} lib;

void bind(const std::vector<uintptr_t>& at) {
  TORCH_CHECK(at.size() == 6, "bind: six entry points");
  lib.bucket_context = reinterpret_cast<decltype(lib.bucket_context)>(at[0]);
  lib.bucket_sums = reinterpret_cast<decltype(lib.bucket_sums)>(at[1]);
  lib.dropout_labels_last = reinterpret_cast<decltype(lib.dropout_labels_last)>(at[2]);
  lib.dropout_labels_first = reinterpret_cast<decltype(lib.dropout_labels_first)>(at[3]);
  lib.sample_labels = reinterpret_cast<decltype(lib.sample_labels)>(at[4]);
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at[5]);
}

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check(int rc, const char* what) { TORCH_CHECK(rc == MPL_OK, what, " failed (", rc, "): ", lib.last_error()); }
// a size that the entry points take as an int
int small(int64_t size) {
  TORCH_CHECK(size <= std::numeric_limits<int>::max(), "a size of ", size, " is too large");
  return (int)size;
}
// whether a gradient is itself to be differentiated
bool recorded(const at::Tensor& grad) { return at::GradMode::is_enabled() && grad.requires_grad(); }

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

// -------------------------------------------------------------------------------------------------- sampled labels
// A parameter: a number, or a tensor of one per image (not looked at).
template <typename T>
struct Parameter {
  const T* each = nullptr;
  T all = 0;

  Parameter(const char* name, const py::object& value, int64_t batch, const at::Tensor& cost, at::ScalarType type, double high) {
    if (THPVariable_Check(value.ptr())) {
      const at::Tensor& t = THPVariable_Unpack(value.ptr());
      TORCH_CHECK(t.device() == cost.device(), "sample_labels: ", name, " must be on the device of the costs");
      TORCH_CHECK(t.scalar_type() == type && t.dim() == 1 && t.size(0) == batch && t.is_contiguous(), "sample_labels: ", name,
                  " must be a number or a contiguous ", type, " tensor of one per image (", batch, ")");
      each = t.data_ptr<T>();
      return;
    }
    TORCH_CHECK(type != at::kInt || (PyIndex_Check(value.ptr()) && !PyBool_Check(value.ptr())), "sample_labels: ", name,
                " must be a whole number");
    const double number = PyFloat_AsDouble(value.ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
    TORCH_CHECK(number >= 0 && number <= high, "sample_labels: ", name, " must be in [0, ", high, "], got ", number);
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
  const Parameter<float> t("temperature", temperature, batch, cost, at::kFloat, inf);
  const Parameter<int32_t> k("top_k", top_k, batch, cost, at::kInt, 2147483647.0);
  const Parameter<float> p("top_p", top_p, batch, cost, at::kFloat, 1), m("min_p", min_p, batch, cost, at::kFloat, 1);
  at::Tensor labels = at::empty(uniforms.sizes(), uniforms.options().dtype(at::kByte));
  const c10::DeviceGuard guard(cost.device());
  check(lib.sample_labels(labels_first, cost.data_ptr<float>(), uniforms.data_ptr<float>(), small(batch), small(cv), small(n),
                          height * width, at == 1 ? small(uniforms.size(0)) : 1, t.each, t.all, k.each, k.all, p.each, p.all,
                          m.each, m.all, labels.data_ptr<uint8_t>(), stream_of(cost)),
        "sample_labels");
  return labels;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("bucket_context", &bucket_context);
  m.def("labels_last_dropout", &labels_last_dropout);
  m.def("sample_labels", &sample_labels);
}
