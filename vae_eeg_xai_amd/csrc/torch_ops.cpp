// torch.ops.veex.dense / dropout / residual_norm: the dense-trunk operators of include/veex.h as dispatcher ops with autograd.
// In C++ because a small layer's training call is host time: forward and backward of a Dense layer cost about 130 us through
// Python autograd functions and ctypes, against about 20 us of kernels; so it is about 50 to 70 us, most of it torch's autograd
// engine (45 us a gradient call and some 6 us for each further leaf).
//
// The public ops check their arguments (ValueError) and take the differentiable or the plain path; the *_fwd / *_bwd ops under
// them have a kernel for the CUDA device type only, so a CPU tensor is refused by the dispatcher, and a fake implementation
// each (trunk_ops.py).  Memory comes from torch's allocator on the current stream, so that calls on several streams, and captured
// graphs, share no workspace.  No exception leaves the C-ABI below; errors of it arrive here as return codes.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/veex.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
const void* in_ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor contig(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
bool learns(const Tensor& t) { return t.defined() && t.requires_grad(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

veexStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (rc=", rc, "): ", veex_last_error()); }

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return VEEX_T_F32;
    case at::kBFloat16: return VEEX_T_BF16;
    case at::kHalf: return VEEX_T_F16;
    default: return -1;
  }
}

int64_t rows_of(const Tensor& x) { return x.size(-1) > 0 ? x.numel() / x.size(-1) : 0; }

void check_type(const char* what, const Tensor& x) {
  TORCH_CHECK_VALUE(dtype_code(x.scalar_type()) >= 0, what, ": float32, bfloat16 or float16 tensors, not ", x.scalar_type());
}
void check_same(const char* what, const Tensor& x, const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(!t.defined() || (t.scalar_type() == x.scalar_type() && t.device() == x.device()), what, ": ", name, " is ",
                    t.scalar_type(), " on ", t.device(), ", x is ", x.scalar_type(), " on ", x.device());
}
void check_drop(const char* what, const Tensor& x, double rate, int64_t first_row, const Tensor& counter) {
  TORCH_CHECK_VALUE(rate >= 0.0 && rate < 1.0 - 0x1p-17, what, ": rate ", rate, " is outside [0, 1 - 2^-17)");
  TORCH_CHECK_VALUE(first_row >= 0, what, ": first_row is negative");
  TORCH_CHECK_VALUE(!counter.defined() || (counter.scalar_type() == at::kLong && counter.numel() == 1 && counter.device() == x.device()),
                    what, ": counter has to be one int64 word on x's device");
}

// Forward-mode derivatives: no tangents are computed.  A dual tensor need not have requires_grad, and the ops under the public ones are
// called below autograd, where its tangent would go unnoticed and count as zero; so it is refused here, and in the backward passes.
void refuse_tangents(const char* what, at::ArrayRef<Tensor> tensors) {
  for (const Tensor& t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what, ": forward-mode derivatives are not implemented");
}

// the counter's word as a forward call saw it, for the backward pass: the caller may advance it in between
Tensor word_now(const Tensor& counter, bool used) { return counter.defined() && used ? counter.detach().add(0) : Tensor(); }

// Below autograd while a backward pass records none itself (its ops' autograd kernels, which only refuse, cost some microseconds)
struct BelowUnlessRecording {
  std::optional<at::AutoDispatchBelowADInplaceOrView> below;
  BelowUnlessRecording() { if (!at::GradMode::is_enabled()) below.emplace(); }
};

// ------------------------------------------------------------------------------------------------ dropout
// (the low-level ops check what keeps their kernels inside the tensors; the public ones run the same checks before autograd)
void check_dropout_args(const Tensor& x, const Tensor& residual, double rate, int64_t first_row, const Tensor& counter) {
  check_type("dropout", x);
  check_same("dropout", x, residual, "residual");
  check_drop("dropout", x, rate, first_row, counter);
  TORCH_CHECK_VALUE(x.dim() >= 1, "dropout: x has no columns");
  TORCH_CHECK_VALUE(x.size(-1) <= 1 << 30, "dropout: x ", x.sizes(), " has more than 2^30 columns");
  TORCH_CHECK_VALUE(!residual.defined() || residual.sizes() == x.sizes(), "dropout: residual ", residual.sizes(), " is not of x's shape ", x.sizes());
}

Tensor dropout_fwd(const Tensor& x_in, double rate, int64_t seed, int64_t first_row, const OptTensor& residual_in, const OptTensor& counter) {
  check_dropout_args(x_in, get(residual_in), rate, first_row, get(counter));
  const c10::DeviceGuard guard(x_in.device());
  const Tensor x = x_in.contiguous(), residual = contig(get(residual_in));
  Tensor y = at::empty_like(x);
  if (x.numel() > 0)
    check_rc(veex_dropout(in_ptr(x), in_ptr(residual), out_ptr(y), rows_of(x), (int)x.size(-1), dtype_code(x.scalar_type()), rate,
                          (unsigned long long)seed, (unsigned long long)first_row,
                          static_cast<const unsigned long long*>(in_ptr(get(counter))), stream_of(x)), "dropout");
  return y;
}

Tensor call_dropout_fwd(const Tensor& x, double rate, int64_t seed, int64_t first_row, const OptTensor& residual, const OptTensor& counter) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("veex::dropout_fwd", "").typed<decltype(dropout_fwd)>();
  at::AutoDispatchBelowADInplaceOrView below;      // (the caller is the op's autograd, or needs none)
  return op.call(x, rate, seed, first_row, residual, counter);
}

Tensor dropout(const Tensor&, double, int64_t, int64_t, const OptTensor&, const OptTensor&);

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double rate, int64_t seed, int64_t first_row, const OptTensor& residual,
                        const OptTensor& counter) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->saved_data["rate"] = rate;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["first_row"] = first_row;
    ctx->saved_data["residual"] = residual.has_value();
    ctx->save_for_backward({word_now(get(counter), x.requires_grad() && rate > 0.0)});
    return call_dropout_fwd(x, rate, seed, first_row, residual, counter);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dx, dr;
    if (ctx->needs_input_grad(0))
      dx = dropout(grads[0], ctx->saved_data["rate"].toDouble(), ctx->saved_data["seed"].toInt(), ctx->saved_data["first_row"].toInt(),
                   std::nullopt, opt(ctx->get_saved_variables()[0]));
    return {dx, Tensor(), Tensor(), Tensor(), ctx->saved_data["residual"].toBool() ? grads[0] : Tensor(), Tensor()};
  }
};

Tensor dropout(const Tensor& x, double rate, int64_t seed, int64_t first_row, const OptTensor& residual_in, const OptTensor& counter) {
  const Tensor residual = get(residual_in);
  check_dropout_args(x, residual, rate, first_row, get(counter));
  refuse_tangents("dropout", {x, residual});
  if (at::GradMode::is_enabled() && (learns(x) || learns(residual))) return Dropout::apply(x, rate, seed, first_row, residual_in, counter);
  return call_dropout_fwd(x, rate, seed, first_row, residual_in, counter);
}

// ------------------------------------------------------------------------------------------------ dense
int activation_code(const std::optional<std::string>& a) {
  if (!a.has_value() || *a == "linear") return VEEX_ACT_NONE;
  if (*a == "relu") return VEEX_ACT_RELU;
  if (*a == "gelu") return VEEX_ACT_GELU;
  if (*a == "silu") return VEEX_ACT_SILU;
  if (*a == "sigmoid") return VEEX_ACT_SIGMOID;
  TORCH_CHECK_VALUE(false, "dense: activation '", *a, "' is none of linear, relu, gelu, silu, sigmoid");
}

// x as (rows, K) with neighbouring columns next to each other: a view where its strides allow it
Tensor as_rows(const Tensor& x) {
  const Tensor r = x.dim() == 2 ? x : x.reshape({rows_of(x), x.size(-1)});
  if (r.size(0) <= 1) return r.contiguous();
  return (r.size(1) == 1 || r.stride(1) == 1) && r.stride(0) >= r.size(1) ? r : r.contiguous();
}

std::vector<int64_t> dense_shape(const Tensor& x, const Tensor& w) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = w.size(1);
  return s;
}

void check_dense_args(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual, double rate, int64_t first_row, const Tensor& counter) {
  check_type("dense", x);
  check_same("dense", x, w, "w");
  check_same("dense", x, bias, "bias");
  check_same("dense", x, residual, "residual");
  check_drop("dense", x, rate, first_row, counter);
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(0) && w.size(0) > 0 && w.size(1) > 0, "dense: x ", x.sizes(),
                    " is not (..., K) for w ", w.sizes(), " = (K, N) with K, N >= 1");
  TORCH_CHECK_VALUE(w.size(0) <= 1 << 30 && w.size(1) <= 1 << 30, "dense: w ", w.sizes(), " has more than 2^30 rows or columns");
  TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == w.size(1)), "dense: bias ", bias.sizes(), " is not (", w.size(1), ",)");
  TORCH_CHECK_VALUE(!residual.defined() || residual.sizes() == at::IntArrayRef(dense_shape(x, w)), "dense: residual ", residual.sizes(),
                    " is not of y's shape ", at::IntArrayRef(dense_shape(x, w)));
}

VeexDense dense_desc(const Tensor& x, const Tensor& w, int64_t activation, double rate, int64_t seed, int64_t first_row, const Tensor& counter) {
  VeexDense d = {};
  d.struct_size = sizeof(d);
  d.x = in_ptr(x); d.w = in_ptr(w);
  d.rows = x.size(0); d.k = (int32_t)w.size(0); d.n = (int32_t)w.size(1);
  d.ldx = d.rows > 1 ? x.stride(0) : d.k;
  d.dtype = dtype_code(x.scalar_type()); d.activation = (int32_t)activation;
  d.rate = rate; d.seed = (unsigned long long)seed; d.first_row = (unsigned long long)first_row;
  d.counter = static_cast<const unsigned long long*>(in_ptr(counter));
  return d;
}

Tensor workspace(VeexDense& d, long long bytes, const Tensor& x, const char* what) {
  TORCH_CHECK(bytes >= 0, what, " failed: ", veex_last_error());
  if (bytes == 0) return Tensor();
  Tensor w = at::empty({bytes}, x.options().dtype(at::kByte));
  d.workspace = out_ptr(w); d.workspace_bytes = bytes;
  return w;
}

std::tuple<Tensor, Tensor> dense_fwd(const Tensor& x_in, const Tensor& w_in, const OptTensor& bias_in, int64_t activation,
                                     const OptTensor& residual_in, double rate, int64_t seed, int64_t first_row, const OptTensor& counter, bool keep) {
  check_dense_args(x_in, w_in, get(bias_in), get(residual_in), rate, first_row, get(counter));
  const c10::DeviceGuard guard(x_in.device());
  const Tensor x = as_rows(x_in), w = w_in.contiguous(), bias = contig(get(bias_in)), residual = contig(get(residual_in));
  Tensor y = at::empty(dense_shape(x_in, w), x.options());
  Tensor pre = keep ? at::empty_like(y) : at::empty({0}, x.options());
  VeexDense d = dense_desc(x, w, activation, rate, seed, first_row, get(counter));
  d.bias = in_ptr(bias); d.residual = in_ptr(residual); d.y = out_ptr(y); d.pre = keep ? out_ptr(pre) : nullptr;
  if (d.rows > 0) {
    const Tensor ws = workspace(d, veex_dense_fwd_workspace_bytes(&d), x, "dense");
    check_rc(veex_dense_fwd(&d, stream_of(x)), "dense");
  }
  return {y, pre};
}

std::tuple<Tensor, Tensor, Tensor> dense_bwd(const Tensor& dy_in, const Tensor& x_in, const Tensor& w_in, const OptTensor& pre_in,
                                             int64_t activation, double rate, int64_t seed, int64_t first_row, const OptTensor& counter,
                                             bool need_x, bool need_w, bool need_b) {
  check_dense_args(x_in, w_in, Tensor(), dy_in, rate, first_row, get(counter));       // (dy is of the residual's shape)
  check_same("dense", x_in, get(pre_in), "pre");
  TORCH_CHECK_VALUE(activation == VEEX_ACT_NONE || (pre_in.has_value() && pre_in->sizes() == dy_in.sizes()), "dense backward: pre is not of dy's shape ", dy_in.sizes());
  const c10::DeviceGuard guard(x_in.device());
  const Tensor x = as_rows(x_in), w = w_in.contiguous(), dy = dy_in.contiguous(), pre = contig(get(pre_in));
  const bool rows = x.size(0) > 0;
  const auto make = [&](at::IntArrayRef shape, bool need) {
    return !need ? at::empty({0}, x.options()) : rows ? at::empty(shape, x.options()) : at::zeros(shape, x.options());
  };
  Tensor dx = make(x_in.sizes(), need_x), dw = make(w.sizes(), need_w), db = make({w.size(1)}, need_b);
  if (rows && (need_x || need_w || need_b)) {
    VeexDense d = dense_desc(x, w, activation, rate, seed, first_row, get(counter));
    d.dy = in_ptr(dy); d.pre = const_cast<void*>(in_ptr(pre));
    d.dx = need_x ? out_ptr(dx) : nullptr; d.dw = need_w ? out_ptr(dw) : nullptr; d.db = need_b ? out_ptr(db) : nullptr;
    const Tensor ws = workspace(d, veex_dense_bwd_workspace_bytes(&d), x, "dense backward");
    check_rc(veex_dense_bwd(&d, stream_of(x)), "dense backward");
  }
  return {dx, dw, db};
}

std::tuple<Tensor, Tensor> call_dense_fwd(const Tensor& x, const Tensor& w, const OptTensor& bias, int64_t activation, const OptTensor& residual,
                                          double rate, int64_t seed, int64_t first_row, const OptTensor& counter, bool keep) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("veex::dense_fwd", "").typed<decltype(dense_fwd)>();
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, w, bias, activation, residual, rate, seed, first_row, counter, keep);
}

struct Dense : torch::autograd::Function<Dense> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias, int64_t activation, const OptTensor& residual,
                        double rate, int64_t seed, int64_t first_row, const OptTensor& counter) {
    at::AutoDispatchBelowADInplaceOrView below;
    const bool need = learns(x) || learns(w) || learns(get(bias));
    // relu: y itself says where the gradient passes, unless a residual was added to it
    const bool by_output = activation == VEEX_ACT_RELU && !residual.has_value();
    auto [y, pre] = call_dense_fwd(x, w, bias, activation, residual, rate, seed, first_row, counter, need && activation != VEEX_ACT_NONE && !by_output);
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["rate"] = rate;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["first_row"] = first_row;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    if (need)
      ctx->save_for_backward({x, w, activation == VEEX_ACT_NONE ? Tensor() : by_output ? y : pre, word_now(get(counter), rate > 0.0)});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    // (needs_input_grad counts the tensors that were given, not the arguments)
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    if (need_x || need_w || need_b) {
      static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("veex::dense_bwd", "").typed<decltype(dense_bwd)>();
      const auto saved = ctx->get_saved_variables();
      refuse_tangents("dense backward", {grads[0], saved[0], saved[1]});
      const BelowUnlessRecording below;
      auto [dx, dw, db] = op.call(grads[0], saved[0], saved[1], opt(saved[2]), ctx->saved_data["activation"].toInt(), ctx->saved_data["rate"].toDouble(),
                                  ctx->saved_data["seed"].toInt(), ctx->saved_data["first_row"].toInt(), opt(saved[3]), need_x, need_w, need_b);
      if (need_x) out[0] = dx;
      if (need_w) out[1] = dw;
      if (need_b) out[2] = db;
    }
    if (ctx->saved_data["residual"].toBool()) out[4] = grads[0];
    return out;
  }
};

Tensor dense(const Tensor& x, const Tensor& w, const OptTensor& bias_in, std::optional<std::string> activation, const OptTensor& residual_in, double rate,
             int64_t seed, int64_t first_row, const OptTensor& counter) {
  const Tensor bias = get(bias_in), residual = get(residual_in);
  check_dense_args(x, w, bias, residual, rate, first_row, get(counter));
  const int act = activation_code(activation);
  refuse_tangents("dense", {x, w, bias, residual});
  if (at::GradMode::is_enabled() && (learns(x) || learns(w) || learns(bias) || learns(residual)))
    return Dense::apply(x, w, bias_in, (int64_t)act, residual_in, rate, seed, first_row, counter);
  return std::get<0>(call_dense_fwd(x, w, bias_in, act, residual_in, rate, seed, first_row, counter, false));
}

// ------------------------------------------------------------------------------------------------ residual_norm
void check_norm_args(const Tensor (&t)[8], int64_t groups, double eps) {
  static const char* const names[8] = {"x", "h", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias"};
  const Tensor& x = t[0];
  check_type("residual_norm", x);
  for (int i = 1; i < 8; ++i) check_same("residual_norm", x, t[i], names[i]);
  TORCH_CHECK_VALUE(eps >= 0.0, "residual_norm: eps has to be >= 0");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= VEEX_NORM_MAX_COLS, "residual_norm: rows of 1 to ", VEEX_NORM_MAX_COLS,
                    " columns, not x ", x.sizes());
  TORCH_CHECK_VALUE(t[1].defined() || !(t[2].defined() || t[3].defined() || t[4].defined() || t[5].defined()),
                    "residual_norm: gate, scale and the post norm's parameters go with h");
  TORCH_CHECK_VALUE(!t[1].defined() || t[1].sizes() == x.sizes(), "residual_norm: h (", t[1].sizes(), ") is not of x's shape ", x.sizes());
  for (int i = 3; i < 8; ++i)
    TORCH_CHECK_VALUE(!t[i].defined() || (t[i].dim() == 1 && t[i].size(0) == x.size(-1)), "residual_norm: ", names[i], " ", t[i].sizes(), " is not (", x.size(-1), ",)");
  TORCH_CHECK_VALUE(groups >= 1, "residual_norm: a gate of ", groups, " groups");
  TORCH_CHECK_VALUE(!t[2].defined() || rows_of(x) == 0 || (t[2].numel() == groups * x.size(-1) && rows_of(x) % groups == 0),
                    "residual_norm: gate ", t[2].sizes(), " does not go with x ", x.sizes());
}

VeexResidualNorm norm_desc(const Tensor (&t)[8], int64_t groups, int64_t kind, double eps) {
  VeexResidualNorm d = {};
  d.struct_size = sizeof(d);
  d.x = in_ptr(t[0]); d.h = in_ptr(t[1]); d.gate = in_ptr(t[2]); d.scale = in_ptr(t[3]);
  d.post_w = in_ptr(t[4]); d.post_b = in_ptr(t[5]); d.pre_w = in_ptr(t[6]); d.pre_b = in_ptr(t[7]);
  d.rows = rows_of(t[0]); d.cols = (int32_t)t[0].size(-1); d.groups = groups;
  d.dtype = dtype_code(t[0].scalar_type()); d.kind = (int32_t)kind; d.eps = (float)eps;
  return d;
}

std::tuple<Tensor, Tensor, Tensor> norm_fwd(const Tensor& x, const OptTensor& h, const OptTensor& gate, const OptTensor& scale, const OptTensor& post_w,
                                            const OptTensor& post_b, const OptTensor& pre_w, const OptTensor& pre_b, int64_t groups, int64_t kind,
                                            double eps, bool keep) {
  const c10::DeviceGuard guard(x.device());
  const Tensor t[8] = {x.contiguous(), contig(get(h)), contig(get(gate)), contig(get(scale)), contig(get(post_w)), contig(get(post_b)), contig(get(pre_w)), contig(get(pre_b))};
  check_norm_args(t, groups, eps);
  Tensor out = h.has_value() ? at::empty_like(t[0]) : at::empty({0}, x.options());
  Tensor u = at::empty_like(t[0]);
  Tensor stats = at::empty({keep ? rows_of(x) : 0, 4}, x.options().dtype(at::kFloat));
  if (x.numel() > 0) {
    VeexResidualNorm d = norm_desc(t, groups, kind, eps);
    d.x_out = h.has_value() ? out_ptr(out) : nullptr;
    d.u = out_ptr(u);
    d.stats = keep ? static_cast<float*>(out_ptr(stats)) : nullptr;
    check_rc(veex_residual_norm_fwd(&d, stream_of(x)), "residual_norm");
  }
  return {out, u, stats};
}

std::vector<Tensor> norm_bwd(const Tensor& x, const OptTensor& h, const OptTensor& gate, const OptTensor& scale, const OptTensor& post_w,
                             const OptTensor& post_b, const OptTensor& pre_w, const OptTensor& pre_b, int64_t groups, int64_t kind, double eps,
                             const Tensor& stats, const OptTensor& dx_out_in, const OptTensor& du_in, std::array<bool, 8> need) {
  const c10::DeviceGuard guard(x.device());
  const Tensor t[8] = {x.contiguous(), contig(get(h)), contig(get(gate)), contig(get(scale)), contig(get(post_w)), contig(get(post_b)), contig(get(pre_w)), contig(get(pre_b))};
  const Tensor dx_out = contig(get(dx_out_in)), du = contig(get(du_in));
  check_norm_args(t, groups, eps);
  check_same("residual_norm", x, dx_out, "dx_out");
  check_same("residual_norm", x, du, "du");
  TORCH_CHECK_VALUE((!dx_out.defined() || dx_out.sizes() == x.sizes()) && (!du.defined() || du.sizes() == x.sizes()) && stats.is_contiguous() &&
                        stats.scalar_type() == at::kFloat && stats.device() == x.device() && stats.numel() == rows_of(x) * 4,
                    "residual_norm backward: dx_out, du or stats do not go with x ", x.sizes());
  const bool rows = rows_of(x) > 0;
  std::vector<Tensor> g(8);
  void* out[8];
  for (int i = 0; i < 8; ++i) {
    const bool want = need[i] && t[i].defined();
    g[i] = !want ? at::empty({0}, x.options()) : rows ? at::empty(t[i].sizes(), x.options()) : at::zeros(t[i].sizes(), x.options());
    out[i] = want ? out_ptr(g[i]) : nullptr;
  }
  if (rows) {
    VeexResidualNorm d = norm_desc(t, groups, kind, eps);
    d.stats = const_cast<float*>(static_cast<const float*>(in_ptr(stats)));
    d.dx_out = in_ptr(dx_out); d.du = in_ptr(du);
    d.dx = out[0]; d.dh = out[1]; d.dgate = out[2]; d.dscale = out[3];
    d.dpost_w = out[4]; d.dpost_b = out[5]; d.dpre_w = out[6]; d.dpre_b = out[7];
    const long long floats = veex_residual_norm_bwd_workspace_floats(d.rows, d.cols, groups);
    TORCH_CHECK(floats >= 0, "residual_norm backward: the gate's groups do not divide the rows");
    Tensor ws = at::empty({floats}, x.options().dtype(at::kFloat));
    d.workspace = static_cast<float*>(out_ptr(ws)); d.workspace_floats = floats;
    check_rc(veex_residual_norm_bwd(&d, stream_of(x)), "residual_norm backward");
  }
  return g;
}

std::tuple<Tensor, Tensor, Tensor> call_norm_fwd(const Tensor& x, const OptTensor& h, const OptTensor& gate, const OptTensor& scale, const OptTensor& post_w,
                                                 const OptTensor& post_b, const OptTensor& pre_w, const OptTensor& pre_b, int64_t groups, int64_t kind,
                                                 double eps, bool keep) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("veex::residual_norm_fwd", "").typed<decltype(norm_fwd)>();
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps, keep);
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& h, const OptTensor& gate, const OptTensor& scale, const OptTensor& post_w,
                               const OptTensor& post_b, const OptTensor& pre_w, const OptTensor& pre_b, int64_t groups, int64_t kind, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    auto [out, u, stats] = call_norm_fwd(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps, true);
    ctx->save_for_backward({x, get(h), get(gate), get(scale), get(post_w), get(post_b), get(pre_w), get(pre_b), stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["eps"] = eps;
    if (h.has_value()) return {out, u};
    return {u};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(11);
    const Tensor dx_out = grads.size() == 2 ? grads[0] : Tensor(), du = grads.back();
    if (!dx_out.defined() && !du.defined()) return out;
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("veex::residual_norm_bwd", "").typed<decltype(norm_bwd)>();
    const auto s = ctx->get_saved_variables();
    refuse_tangents("residual_norm backward", {dx_out, du});
    refuse_tangents("residual_norm backward", s);
    std::array<bool, 8> need;
    for (int i = 0, given = 0; i < 8; ++i) need[i] = s[i].defined() && ctx->needs_input_grad(given++);   // (counts the tensors given)
    const BelowUnlessRecording below;
    const auto g = op.call(s[0], opt(s[1]), opt(s[2]), opt(s[3]), opt(s[4]), opt(s[5]), opt(s[6]), opt(s[7]), ctx->saved_data["groups"].toInt(),
                           ctx->saved_data["kind"].toInt(), ctx->saved_data["eps"].toDouble(), s[8], opt(dx_out), opt(du), need);
    for (int i = 0; i < 8; ++i)
      if (need[i]) out[i] = g[i];
    return out;
  }
};

// Rows of the gate: its leading indices are the first ones of x's, those left out (or 1) share a gate.
int64_t gate_groups(const Tensor& gate, const Tensor& x) {
  bool fits = gate.dim() >= 1 && gate.size(-1) == x.size(-1);
  if (fits) {
    int64_t lead = gate.dim() - 1;
    while (lead > 0 && gate.size(lead - 1) == 1) --lead;
    fits = lead < x.dim();
    for (int64_t i = 0; fits && i < lead; ++i) fits = gate.size(i) == x.size(i);
    if (!fits && x.dim() == 2 && lead == 1) fits = gate.size(0) > 0 && x.size(0) % gate.size(0) == 0;
  }
  TORCH_CHECK_VALUE(fits, "residual_norm: gate ", gate.sizes(), " does not go with x ", x.sizes());
  return std::max<int64_t>(rows_of(gate), 1);
}

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const OptTensor& h_in, const OptTensor& gate_in, const OptTensor& scale, const OptTensor& post_w,
                                         const OptTensor& post_b, const OptTensor& pre_w, const OptTensor& pre_b, std::string kind, double eps) {
  const Tensor t[8] = {x, get(h_in), get(gate_in), get(scale), get(post_w), get(post_b), get(pre_w), get(pre_b)};
  const Tensor &h = t[1], &gate = t[2];
  TORCH_CHECK_VALUE(kind == "layer" || kind == "rms", "residual_norm: kind '", kind, "' is neither 'layer' nor 'rms'");
  check_type("residual_norm", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "residual_norm: rows of 1 to ", VEEX_NORM_MAX_COLS, " columns, not x ", x.sizes());
  const int64_t groups = gate.defined() ? gate_groups(gate, x) : 1, code = kind == "layer" ? VEEX_NORM_LAYER : VEEX_NORM_RMS;
  check_norm_args(t, groups, eps);
  refuse_tangents("residual_norm", t);
  bool grad = false;
  for (const Tensor& v : t) grad = grad || learns(v);
  if (grad && at::GradMode::is_enabled()) {
    TORCH_CHECK_VALUE(groups < VEEX_NORM_MAX_GROUPS || groups == rows_of(x), "residual_norm: gate ", gate.sizes(), " for x ", x.sizes(),
                      " in training; it takes fewer than 2^22 groups, or one a row");
    const auto r = ResidualNorm::apply(x, h_in, gate_in, scale, post_w, post_b, pre_w, pre_b, groups, code, eps);
    return {h.defined() ? r[0] : x, r.back()};
  }
  auto [out, u, stats] = call_norm_fwd(x, h_in, gate_in, scale, post_w, post_b, pre_w, pre_b, groups, code, eps, false);
  return {h.defined() ? out : x, u};
}

#define NORM_ARGS "Tensor? h, Tensor? gate, Tensor? scale, Tensor? post_weight, Tensor? post_bias, Tensor? pre_weight, Tensor? pre_bias, int groups, int kind, float eps"

TORCH_LIBRARY_FRAGMENT(veex, m) {
  m.def("dropout_fwd(Tensor x, float rate, int seed, int first_row, Tensor? residual, Tensor? counter) -> Tensor");
  m.def("dropout(Tensor x, float rate, int seed, int first_row=0, Tensor? residual=None, Tensor? counter=None) -> Tensor");
  m.def("dense_fwd(Tensor x, Tensor w, Tensor? bias, int activation, Tensor? residual, float rate, int seed, int first_row, Tensor? counter, bool keep) -> (Tensor, Tensor)");
  m.def("dense_bwd(Tensor dy, Tensor x, Tensor w, Tensor? pre, int activation, float rate, int seed, int first_row, Tensor? counter, bool need_x, bool need_w, bool need_b) -> (Tensor, Tensor, Tensor)");
  m.def("dense(Tensor x, Tensor w, Tensor? bias=None, str? activation=None, Tensor? residual=None, float rate=0.0, int seed=0, int first_row=0, Tensor? counter=None) -> Tensor");
  m.def("residual_norm_fwd(Tensor x, " NORM_ARGS ", bool keep) -> (Tensor, Tensor, Tensor)");
  m.def("residual_norm_bwd(Tensor x, " NORM_ARGS ", Tensor stats, Tensor? dx_out, Tensor? du, bool[8] need) -> Tensor[]");
  m.def("residual_norm(Tensor x, Tensor? h=None, Tensor? gate=None, Tensor? scale=None, Tensor? post_weight=None, Tensor? post_bias=None, Tensor? pre_weight=None, Tensor? pre_bias=None, str kind='layer', float eps=0.001) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(veex, CUDA, m) {
  m.impl("dropout_fwd", dropout_fwd);
  m.impl("dense_fwd", dense_fwd);
  m.impl("dense_bwd", dense_bwd);
  m.impl("residual_norm_fwd", norm_fwd);
  m.impl("residual_norm_bwd", norm_bwd);
}

TORCH_LIBRARY_IMPL(veex, CompositeImplicitAutograd, m) {
  m.impl("dropout", dropout);
  m.impl("dense", dense);
  m.impl("residual_norm", residual_norm);
}

// differentiable once: a gradient of a gradient, or of a low-level op called by itself, raises
TORCH_LIBRARY_IMPL(veex, Autograd, m) {
  for (const char* name : {"dropout_fwd", "dense_fwd", "dense_bwd", "residual_norm_fwd", "residual_norm_bwd"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

}  // namespace
