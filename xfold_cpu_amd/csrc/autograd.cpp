// Autograd nodes of the operators that have a backward pass: trainable_layer_norm and sequence_attention.
//
// The nodes take tensors that the Python front ends (fastnn/layer_norm.py, fastnn/sequence.py) have
// checked, allocate results and workspaces with torch's caching allocator and call the C ABI of
// libxfold_hip.so (include/xfold_hip.h) on the tensors' device and its current stream. They are in C++
// because a node in Python costs the host more than the kernels take on small inputs: forward and
// backward of a LayerNorm of 72 x 384, 12 us of GPU time, took 106 us of host time.
//
// The library is the one that fastnn/native_hip.py has loaded: bind() takes its functions' addresses.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cstring>
#include <map>
#include <string>
#include <vector>

#include "../../include/xfold_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
  decltype(&xfh_last_error) last_error = nullptr;
  decltype(&xfh_convert) convert = nullptr;
  decltype(&xfh_layer_norm_train) norm = nullptr;
  decltype(&xfh_layer_norm_backward_workspace_size) norm_backward_size = nullptr;
  decltype(&xfh_layer_norm_backward) norm_backward = nullptr;
  decltype(&xfh_sequence_attention_workspace_size) sequence_size = nullptr;
  decltype(&xfh_sequence_attention) sequence = nullptr;
  decltype(&xfh_sequence_attention_backward_workspace_size) sequence_backward_size = nullptr;
  decltype(&xfh_sequence_attention_backward) sequence_backward = nullptr;
} lib;

template <class F> void take(const std::map<std::string, uintptr_t> &at, const char *name, F &f) {
  f = reinterpret_cast<F>(at.at(name));
}
void bind(int abi_version, const std::map<std::string, uintptr_t> &at) {
  TORCH_CHECK(abi_version == XFH_ABI_VERSION, "xfold_autograd.so was built for ABI ", XFH_ABI_VERSION, ", not ", abi_version,
              "; rebuild it.");
  take(at, "xfh_last_error", lib.last_error);
  take(at, "xfh_convert", lib.convert);
  take(at, "xfh_layer_norm_train", lib.norm);
  take(at, "xfh_layer_norm_backward_workspace_size", lib.norm_backward_size);
  take(at, "xfh_layer_norm_backward", lib.norm_backward);
  take(at, "xfh_sequence_attention_workspace_size", lib.sequence_size);
  take(at, "xfh_sequence_attention", lib.sequence);
  take(at, "xfh_sequence_attention_backward_workspace_size", lib.sequence_backward_size);
  take(at, "xfh_sequence_attention_backward", lib.sequence_backward);
}

// A status as the exception that native_hip.call raises for it.
void check(int status, const char *name) {
  if (status == XFH_OK) return;
  const std::string message = lib.last_error();
  TORCH_CHECK_VALUE(status != XFH_EINVAL && status != XFH_EUNSUPPORTED, name, ": ", message);
  TORCH_CHECK(false, name, " failed (", status, "): ", message);
}

int code(at::ScalarType t) { return t == at::kFloat ? XFH_F32 : XFH_BF16; }
int code(const Tensor &t) { return t.defined() ? code(t.scalar_type()) : XFH_F32; }
void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *stream_of(const Tensor &t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}
Tensor workspace(int64_t bytes, const Tensor &like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
Tensor cast(const Tensor &t, at::ScalarType dtype) {
  if (t.scalar_type() == dtype) return t;
  const Tensor from = t.contiguous(), to = at::empty(t.sizes(), t.options().dtype(dtype));
  check(lib.convert(from.data_ptr(), code(from), to.data_ptr(), code(to), from.numel(), stream_of(t)), "xfh_convert");
  return to;
}

// Gradients that are to be differentiated again get a node that refuses it.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  std::vector<size_t> place;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) {
      some.push_back(grads[i].detach().set_requires_grad(true));
      place.push_back(i);
    }
  const auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "The backward passes of the 'hip' backend cannot be differentiated.", int64_t(some.size()));
  some = (*refuse)(std::move(some));
  for (size_t i = 0; i < place.size(); ++i) grads[place[i]] = some[i];
  return grads;
}

// ------------------------------------------------------------------------------ LayerNorm

// The rows of `cols` elements of t, or of a contiguous copy, and the stride between them.
std::pair<Tensor, int64_t> rows_of(const Tensor &t, int64_t cols) {
  if (t.is_contiguous()) return {t, cols};
  if (t.dim() == 2 && t.size(1) == cols && t.stride(1) == 1 && t.stride(0) >= cols) return {t, t.stride(0)};
  return {t.contiguous(), cols};
}

Tensor norm_forward(const Tensor &x, int64_t stride, int64_t cols, const Tensor &weight, const Tensor &bias, double eps,
                    at::ScalarType out_dtype, Tensor *stats) {
  const int64_t rows = cols ? x.numel() / cols : 0;
  const Tensor y = at::empty(x.sizes(), x.options().dtype(out_dtype));
  if (stats) *stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
  check(lib.norm(x.data_ptr(), code(x), stride, rows, cols, address(weight), code(weight), address(bias), code(bias), float(eps),
                 y.data_ptr(), code(y), stats ? stats->data_ptr<float>() : nullptr, stream_of(x)),
        "xfh_layer_norm_train");
  return y;
}

Tensor dense(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

using Maybe = std::optional<Tensor>;
Tensor get(const Maybe &t) { return t ? *t : Tensor(); }

struct TrainableLayerNorm : torch::autograd::Function<TrainableLayerNorm> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x_in, const Maybe &weight_in, const Maybe &bias_in, int64_t cols,
                        double eps, bool wide) {
    const c10::DeviceGuard guard(x_in.device());
    const Tensor weight = get(weight_in), bias = get(bias_in);
    const auto [x, stride] = rows_of(x_in, cols);
    const Tensor w = dense(weight);
    Tensor stats;
    const Tensor y = norm_forward(x, stride, cols, w, dense(bias), eps, wide ? at::kFloat : x.scalar_type(), &stats);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["cols"] = cols;
    if (bias.defined()) {
      ctx->saved_data["bias_shape"] = bias.sizes().vec();
      ctx->saved_data["bias_dtype"] = int64_t(bias.scalar_type());
    }
    return y;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &weight = saved[1], &stats = saved[2];
    const int64_t cols = ctx->saved_data["cols"].toInt();
    const c10::DeviceGuard guard(saved[0].device());
    const auto [x, stride] = rows_of(saved[0], cols);
    const auto [dy, dy_stride] = rows_of(grads[0], cols);
    const int64_t rows = stats.size(0);
    Tensor dx, dw, db, ws;
    if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), x.options());
    if (weight.defined() && ctx->needs_input_grad(1)) dw = at::empty_like(weight);
    if (ctx->saved_data.count("bias_dtype") && ctx->needs_input_grad(1 + weight.defined()))   // (counts the tensors that are there)
      db = at::empty(ctx->saved_data["bias_shape"].toIntVector(),
                     x.options().dtype(at::ScalarType(ctx->saved_data["bias_dtype"].toInt())));
    int64_t size = 0;
    if (dw.defined() || db.defined()) ws = workspace(size = lib.norm_backward_size(rows, cols), x);
    check(lib.norm_backward(dy.data_ptr(), code(dy), dy_stride, x.data_ptr(), code(x), stride, rows, cols, address(weight),
                            code(weight), stats.data_ptr<float>(), address(dx), address(dw), code(dw), address(db), code(db),
                            address(ws), size, stream_of(x)),
          "xfh_layer_norm_backward");
    return once({dx, dw, db, Tensor(), Tensor(), Tensor()});
  }
};

// (Tensors of which none needs a gradient are left to the forward call alone, which keeps no statistics.)
bool needs_gradient(std::initializer_list<Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor &t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

Tensor trainable_layer_norm(const Tensor &x, const Maybe &weight, const Maybe &bias, int64_t cols, double eps, bool wide) {
  const Tensor w = get(weight), b = get(bias);
  if (needs_gradient({x, w, b})) return TrainableLayerNorm::apply(x, weight, bias, cols, eps, wide);
  const c10::DeviceGuard guard(x.device());
  const auto [rows, stride] = rows_of(x, cols);
  return norm_forward(rows, stride, cols, dense(w), dense(b), eps, wide ? at::kFloat : x.scalar_type(), nullptr);
}

// ------------------------------------------------------------------------------ sequence attention

struct Options {
  bool causal;
  int64_t prefix_all;
  double softcap, scale;
};
struct Masks { Tensor prefix, documents, lengths; };

// t in `dtype`, its last dim contiguous.
Tensor heads_of(const Tensor &t, at::ScalarType dtype) {
  if (t.scalar_type() != dtype) return cast(t, dtype);
  return t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous();
}
// [B, heads, tokens, dim] in the memory order of `like`: token by token where its heads lie side by side.
Tensor empty_as(const Tensor &like, int64_t heads, int64_t tokens, int64_t dim) {
  if (like.stride(1) < like.stride(2)) return at::empty({like.size(0), tokens, heads, dim}, like.options()).transpose(1, 2);
  return at::empty({like.size(0), heads, tokens, dim}, like.options());
}
void strides(const Tensor &t, int64_t *to) {
  for (int i = 0; i < 3; ++i) to[i] = t.defined() ? t.stride(i) : 0;
}

XfhSequenceAttention arguments(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &out, const Tensor &lse,
                               const Tensor &low, const Tensor &slopes, const Masks &masks, const Options &o) {
  XfhSequenceAttention a;
  std::memset(&a, 0, sizeof(a));
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.out = out.data_ptr();
  a.lse = static_cast<float *>(address(lse));
  a.out_low = address(low);
  a.slopes = static_cast<const float *>(address(slopes));
  a.prefix = static_cast<const int32_t *>(address(masks.prefix));
  a.documents = static_cast<const int32_t *>(address(masks.documents));
  a.lengths = static_cast<const int32_t *>(address(masks.lengths));
  a.batch = q.size(0); a.heads = q.size(1); a.kv_heads = k.size(1); a.queries = q.size(2); a.keys = k.size(2);
  a.dim = q.size(3); a.value_dim = v.size(3);
  strides(q, a.q_strides); strides(k, a.k_strides); strides(v, a.v_strides); strides(out, a.out_strides);
  a.documents_stride = masks.documents.defined() ? masks.documents.stride(0) : 0;
  a.prefix_all = o.prefix_all;
  a.scale = float(o.scale);
  a.softcap = float(o.softcap);
  a.causal = o.causal;
  a.dtype = code(q);
  return a;
}

// Out; with `keep` what the backward pass needs besides.
Tensor sequence_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &slopes, const Masks &masks,
                        const Options &o, bool keep, Tensor *lse, Tensor *low) {
  const Tensor out = empty_as(q, q.size(1), q.size(2), v.size(3));
  if (keep) {
    const bool single = q.scalar_type() == at::kFloat;
    *lse = at::empty({1 + single, q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    if (!single) *low = at::empty({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options());
  }
  const XfhSequenceAttention a = arguments(q, k, v, out, keep ? *lse : Tensor(), keep ? *low : Tensor(), slopes, masks, o);
  const int64_t size = lib.sequence_size(&a);
  const Tensor ws = workspace(size, q);
  check(lib.sequence(&a, address(ws), size, stream_of(q)), "xfh_sequence_attention");
  return out;
}

Tensor slopes_of(const Tensor &slopes) { return slopes.defined() ? cast(slopes, at::kFloat).contiguous() : slopes; }

struct SequenceAttention : torch::autograd::Function<SequenceAttention> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q_in, const Tensor &k_in, const Tensor &v_in,
                        const Maybe &maybe_slopes, const Maybe &maybe_prefix, const Maybe &maybe_documents,
                        const Maybe &maybe_lengths, bool causal, int64_t prefix_all, double softcap, double scale,
                        at::ScalarType dtype) {
    const c10::DeviceGuard guard(q_in.device());
    const Tensor slopes_in = get(maybe_slopes), prefix = get(maybe_prefix), documents = get(maybe_documents),
                 lengths = get(maybe_lengths);
    const Tensor q = heads_of(q_in, dtype), k = heads_of(k_in, dtype), v = heads_of(v_in, dtype), slopes = slopes_of(slopes_in);
    Tensor lse, low;
    const Tensor out = sequence_forward(q, k, v, slopes, {prefix, documents, lengths}, {causal, prefix_all, softcap, scale}, true,
                                        &lse, &low);
    ctx->save_for_backward({q, k, v, slopes, out, lse, low, prefix, documents, lengths});
    ctx->saved_data["options"] = std::vector<double>{double(causal), softcap, scale};
    ctx->saved_data["prefix"] = prefix_all;
    ctx->saved_data["dtypes"] = std::vector<int64_t>{
        int64_t(q_in.scalar_type()), int64_t(k_in.scalar_type()), int64_t(v_in.scalar_type()),
        slopes_in.defined() ? int64_t(slopes_in.scalar_type()) : -1};
    return out;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &slopes = saved[3];
    const c10::DeviceGuard guard(q.device());
    const auto o = ctx->saved_data["options"].toDoubleVector();
    const auto dtypes = ctx->saved_data["dtypes"].toIntVector();
    const Tensor dout = heads_of(grads[0], q.scalar_type());
    Tensor d[4];
    d[0] = empty_as(q, q.size(1), q.size(2), q.size(3));
    if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
      d[1] = empty_as(k, k.size(1), k.size(2), k.size(3));
      d[2] = empty_as(v, v.size(1), v.size(2), v.size(3));
    }
    if (dtypes[3] >= 0 && ctx->needs_input_grad(3)) d[3] = at::empty_like(slopes);
    XfhSequenceAttention a = arguments(q, k, v, saved[4], saved[5], saved[6], slopes, {saved[7], saved[8], saved[9]},
                                       {o[0] != 0.0, ctx->saved_data["prefix"].toInt(), o[1], o[2]});
    a.dout = dout.data_ptr();
    a.dq = address(d[0]); a.dk = address(d[1]); a.dv = address(d[2]);
    a.dslopes = static_cast<float *>(address(d[3]));
    strides(dout, a.dout_strides); strides(d[0], a.dq_strides); strides(d[1], a.dk_strides); strides(d[2], a.dv_strides);
    const int64_t size = lib.sequence_backward_size(&a);
    const Tensor ws = workspace(size, q);
    check(lib.sequence_backward(&a, address(ws), size, stream_of(q)), "xfh_sequence_attention_backward");
    variable_list out(12);
    for (int i = 0; i < 4; ++i)
      if (dtypes[i] >= 0 && ctx->needs_input_grad(i)) out[i] = cast(d[i], at::ScalarType(dtypes[i]));
    return once(std::move(out));
  }
};

Tensor sequence_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Maybe &maybe_slopes, const Maybe &prefix,
                          const Maybe &documents, const Maybe &lengths, bool causal, int64_t prefix_all, double softcap,
                          double scale, bool low_precision) {
  const auto dtype = low_precision ? at::kBFloat16 : at::kFloat;
  const Tensor slopes = get(maybe_slopes);
  if (needs_gradient({q, k, v, slopes}))
    return SequenceAttention::apply(q, k, v, maybe_slopes, prefix, documents, lengths, causal, prefix_all, softcap, scale, dtype);
  const c10::DeviceGuard guard(q.device());
  return sequence_forward(heads_of(q, dtype), heads_of(k, dtype), heads_of(v, dtype), slopes_of(slopes),
                          {get(prefix), get(documents), get(lengths)},
                          {causal, prefix_all, softcap, scale}, false, nullptr, nullptr);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("trainable_layer_norm", &trainable_layer_norm, py::call_guard<py::gil_scoped_release>());
  m.def("sequence_attention", &sequence_attention, py::call_guard<py::gil_scoped_release>());
}
