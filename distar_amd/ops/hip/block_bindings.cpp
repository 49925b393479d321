// Python bindings of the kernels around the policy transformer: checks of the
// arguments, outputs and workspaces, the launch on the current stream of the
// tensors' own device, and the autograd nodes. The nodes are C++ so that a
// small call costs a few microseconds on the host instead of some fifty.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <array>
#include <cmath>

#include "block_ops.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

int dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return blk::kF32;
    case torch::kBFloat16: return blk::kBF16;
    case torch::kFloat16: return blk::kF16;
    default:
      TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16, not ",
                       t.scalar_type());
  }
}

void check_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(),
                    ", but the input is on ", like.device());
}

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// A tensor as rows of its last dimension with one stride between them; copied
// only where its strides are not of that form.
struct Rows {
  Tensor t;
  int64_t rows, stride;
};

Rows rows_of(const Tensor& in) {
  const int64_t width = in.size(-1);
  const int64_t rows = width ? in.numel() / width : 0;
  bool fits = in.stride(-1) == 1 || width == 1;
  int64_t stride = width, span = -1;
  bool first = true;
  for (int64_t d = in.dim() - 2; d >= 0 && fits; --d) {
    if (in.size(d) == 1) continue;
    if (first) {
      stride = in.stride(d);
      first = false;
    } else if (in.stride(d) != span) {
      fits = false;
    }
    span = in.stride(d) * in.size(d);
  }
  if (fits) return {in, rows, stride};
  return {in.contiguous(), rows, width};
}

void check_width(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name,
                    " needs a last dimension of at least one element");
  TORCH_CHECK_VALUE(t.size(-1) <= (1 << 30), name, " is wider than 2^30");
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(std::initializer_list<const OptTensor*> inputs) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const auto* t : inputs)
    if (t->has_value() && (*t)->requires_grad()) return true;
  return false;
}

// No kernel carries a forward-mode tangent on, and none may be lost in silence.
void refuse_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what,
                              " has no forward-mode derivative");
}

void refuse_tangents(std::initializer_list<const OptTensor*> inputs, const char* what) {
  for (const auto* t : inputs)
    if (t->has_value()) refuse_tangent(**t, what);
}

// Gradients come without a graph of their own: where one is being built, using
// it raises an error.
variable_list once(variable_list grads, const char* what) {
  if (!c10::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + " is not differentiable twice", (int64_t)grads.size());
  return (*error)(std::move(grads));
}

Tensor none_or(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// ------------------------------------------------------------ layer norm

int check_affine(const Tensor& x, const OptTensor& w, const OptTensor& b,
                 int dtype) {
  int wdtype = dtype;
  bool first = true;
  for (const auto* p : {&w, &b}) {
    if (!p->has_value()) continue;
    const Tensor& t = p->value();
    check_device(t, x, "weight or bias");
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1),
                      "weight and bias must have the row's width, ", x.size(-1));
    const int d = dtype_of(t, "weight or bias");
    TORCH_CHECK_TYPE(d == dtype || d == blk::kF32,
                     "weight and bias must be float32 or of the input's type");
    TORCH_CHECK_TYPE(first || d == wdtype, "weight and bias must be of one type");
    wdtype = d;
    first = false;
  }
  return wdtype;
}

const void* ptr(const OptTensor& t) {
  return t.has_value() ? t->data_ptr() : nullptr;
}

// -> y, s (x itself without a residual), stats (mean, rstd; undefined if unasked)
std::array<Tensor, 3> layer_norm_fwd(Tensor x, OptTensor residual, OptTensor weight,
                                   OptTensor bias, double eps, bool stats) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be on a GPU");
  check_width(x, "x");
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
  const int dtype = dtype_of(x, "x");
  const int wdtype = check_affine(x, weight, bias, dtype);
  if (residual.has_value()) {
    check_device(*residual, x, "residual");
    TORCH_CHECK_TYPE(residual->scalar_type() == x.scalar_type(),
                     "residual must be of x's type");
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "residual must be of x's shape");
  }
  const c10::DeviceGuard guard(x.device());
  if (weight.has_value()) weight = weight->contiguous();
  if (bias.has_value()) bias = bias->contiguous();
  const Rows xr = rows_of(x);
  const Rows rr = residual.has_value() ? rows_of(*residual) : Rows{x, 0, 0};
  Tensor y = torch::empty(x.sizes(), x.options());
  Tensor s = residual.has_value() ? torch::empty(x.sizes(), x.options()) : x;
  Tensor kept;
  if (stats) kept = torch::empty({2, xr.rows}, x.options().dtype(torch::kFloat32));
  if (xr.rows) {
    blk::LayerNormFwd a{};
    a.x = xr.t.data_ptr();
    a.residual = residual.has_value() ? rr.t.data_ptr() : nullptr;
    a.weight = ptr(weight);
    a.bias = ptr(bias);
    a.y = y.data_ptr();
    a.s = residual.has_value() ? s.data_ptr() : nullptr;
    a.mean = stats ? kept.data_ptr<float>() : nullptr;
    a.rstd = stats ? a.mean + xr.rows : nullptr;
    a.rows = xr.rows;
    a.x_stride = xr.stride;
    a.r_stride = rr.stride;
    a.width = (int)x.size(-1);
    a.eps = (float)eps;
    blk::layer_norm_fwd(a, dtype, wdtype, stream_of(x));
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {y, s, kept};
}

// -> dx, dweight, dbias (the last two undefined without `params`)
std::array<Tensor, 3> layer_norm_bwd(Tensor dy, OptTensor ds, Tensor s, Tensor stats,
                                     OptTensor weight, bool params,
                                     torch::ScalarType param_type) {
  const int dtype = dtype_of(s, "s");
  check_device(dy, s, "dy");
  TORCH_CHECK_VALUE(dy.sizes() == s.sizes(), "dy must be of s's shape");
  TORCH_CHECK_TYPE(dy.scalar_type() == s.scalar_type(), "dy must be of s's type");
  if (ds.has_value()) {
    check_device(*ds, s, "ds");
    TORCH_CHECK_VALUE(ds->sizes() == s.sizes(), "ds must be of s's shape");
    TORCH_CHECK_TYPE(ds->scalar_type() == s.scalar_type(), "ds must be of s's type");
  }
  const c10::DeviceGuard guard(s.device());
  const Rows yr = rows_of(dy), sr = rows_of(s);
  const Rows dr = ds.has_value() ? rows_of(*ds) : Rows{s, 0, 0};
  const int64_t width = s.size(-1);
  Tensor dx = torch::empty(s.sizes(), s.options());
  Tensor dw, db;
  if (params) {
    const auto options = s.options().dtype(param_type);
    dw = torch::empty({width}, options);
    db = torch::empty({width}, options);
  }
  if (!sr.rows) {
    if (params) dw.zero_(), db.zero_();
    return {dx, dw, db};
  }
  if (weight.has_value()) weight = weight->contiguous();
  blk::LayerNormBwd a{};
  a.blocks = blk::layer_norm_bwd_blocks(sr.rows, (int)width, dtype);
  Tensor partial;
  if (params)
    partial = torch::empty({a.blocks * 2 * width}, s.options().dtype(torch::kFloat32));
  a.dy = yr.t.data_ptr();
  a.ds = ds.has_value() ? dr.t.data_ptr() : nullptr;
  a.s = sr.t.data_ptr();
  a.weight = ptr(weight);
  a.mean = stats.data_ptr<float>();
  a.rstd = a.mean + sr.rows;
  a.dx = dx.data_ptr();
  a.dweight = params ? dw.data_ptr() : nullptr;
  a.dbias = params ? db.data_ptr() : nullptr;
  a.partial = params ? partial.data_ptr<float>() : nullptr;
  a.rows = sr.rows;
  a.dy_stride = yr.stride;
  a.ds_stride = dr.stride;
  a.s_stride = sr.stride;
  a.width = (int)width;
  blk::layer_norm_bwd(a, dtype, param_type == torch::kFloat32 ? (int)blk::kF32 : dtype,
                      stream_of(s));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {dx, dw, db};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  enum { kX = 1, kResidual = 2, kWeight = 4, kBias = 8 };

  static variable_list forward(AutogradContext* ctx, Tensor x, OptTensor residual,
                               OptTensor weight, OptTensor bias, double eps) {
    const auto r = layer_norm_fwd(x, residual, weight, bias, eps, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({r[1], r[2], none_or(weight)});
    int64_t need = x.requires_grad() ? kX : 0;
    if (residual.has_value() && residual->requires_grad()) need |= kResidual;
    if (weight.has_value() && weight->requires_grad()) need |= kWeight;
    if (bias.has_value() && bias->requires_grad()) need |= kBias;
    ctx->saved_data["need"] = need;
    ctx->saved_data["type"] = (int64_t)(weight.has_value() ? weight->scalar_type()
                                        : bias.has_value() ? bias->scalar_type()
                                                           : x.scalar_type());
    if (residual.has_value()) return {r[0], r[1]};
    return {r[0]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    const Tensor& s = saved[0];
    const Tensor dy = grads[0], ds = grads.size() > 1 ? grads[1] : Tensor();
    Tensor dx = ds, dw, db;                // where only the stream was used
    if (dy.defined()) {
      const auto r = layer_norm_bwd(dy, opt(ds), s, saved[1], opt(saved[2]),
                                    need & (kWeight | kBias),
                                    (torch::ScalarType)ctx->saved_data["type"].toInt());
      dx = r[0], dw = r[1], db = r[2];
    }
    return once({need & kX ? dx : Tensor(), need & kResidual ? dx : Tensor(),
                 need & kWeight ? dw : Tensor(), need & kBias ? db : Tensor(), Tensor()},
                "layer_norm");
  }
};

Tensor layer_norm(Tensor x, OptTensor weight, OptTensor bias, double eps) {
  const OptTensor leaf = x;
  refuse_tangents({&leaf, &weight, &bias}, "layer_norm");
  if (wants_grad({&leaf, &weight, &bias}))
    return LayerNorm::apply(x, OptTensor(), weight, bias, eps)[0];
  return layer_norm_fwd(x, {}, weight, bias, eps, false)[0];
}

std::pair<Tensor, Tensor> add_layer_norm(Tensor x, Tensor residual, OptTensor weight,
                                         OptTensor bias, double eps) {
  const OptTensor leaf = x, other = residual;
  refuse_tangents({&leaf, &other, &weight, &bias}, "add_layer_norm");
  if (wants_grad({&leaf, &other, &weight, &bias})) {
    const auto r = LayerNorm::apply(x, other, weight, bias, eps);
    return {r[0], r[1]};
  }
  const auto r = layer_norm_fwd(x, other, weight, bias, eps, false);
  return {r[0], r[1]};
}

// ------------------------------------------------- token log probabilities

struct LogitRows {
  Rows logits, mask;
  Tensor tokens;
  int dtype;
};

LogitRows check_logits(const Tensor& logits, const Tensor& tokens,
                       const OptTensor& mask) {
  TORCH_CHECK_VALUE(logits.is_cuda(), "logits must be on a GPU");
  check_width(logits, "logits");
  LogitRows r;
  r.dtype = dtype_of(logits, "logits");
  r.logits = rows_of(logits);
  check_device(tokens, logits, "tokens");
  switch (tokens.scalar_type()) {
    case torch::kLong: case torch::kInt: case torch::kShort: case torch::kByte: break;
    default: TORCH_CHECK_TYPE(false, "tokens must be integers, not ", tokens.scalar_type());
  }
  TORCH_CHECK_VALUE(tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                    "tokens must have the shape of logits without its last dimension");
  r.tokens = (tokens.scalar_type() == torch::kLong ? tokens : tokens.to(torch::kLong)).contiguous();
  if (mask.has_value()) {
    check_device(*mask, logits, "mask");
    TORCH_CHECK_TYPE(mask->scalar_type() == torch::kBool, "mask must be bool");
    bool fits = mask->dim() <= logits.dim();
    for (int64_t d = 1; fits && d <= mask->dim(); ++d)
      fits = mask->size(-d) == 1 || mask->size(-d) == logits.size(-d);
    TORCH_CHECK_VALUE(fits, "mask of shape ", mask->sizes(),
                      " does not broadcast to logits of shape ", logits.sizes());
    r.mask = rows_of(mask->sizes() == logits.sizes() ? *mask : mask->expand(logits.sizes()));
  }
  return r;
}

// -> logprob, entropy, top_logprobs, top_tokens (both of width 0 without top_k),
//    stats (maximum, log of the sum, entropy, token of each row; undefined if
//    unasked)
std::array<Tensor, 5> token_logprobs_fwd(Tensor logits, Tensor tokens, OptTensor mask,
                                       double temperature, int64_t top_k,
                                       int64_t ignore_index, bool stats) {
  const c10::OptionalDeviceGuard guard(
      logits.is_cuda() ? c10::optional<c10::Device>(logits.device()) : c10::nullopt);
  const LogitRows r = check_logits(logits, tokens, mask);
  const int64_t rows = r.logits.rows;
  const int64_t k = std::min<int64_t>(top_k, logits.size(-1));
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= 64, "top_k must be 0 to 64, got ", top_k);
  // beyond that the scaled logits or their scale leave the 32-bit range
  TORCH_CHECK_VALUE(temperature >= 1e-30 && temperature <= 1e30,
                    "temperature must be positive, 1e-30 to 1e30, got ", temperature);
  // a launch has at most 2^32 threads, and a thread of the gradient takes 32 bytes
  TORCH_CHECK_VALUE(!stats || logits.numel() < (int64_t)1 << 34, "logits of ",
                    logits.numel(), " elements are too large for a gradient");
  const auto f32 = logits.options().dtype(torch::kFloat32);
  Tensor logprob = torch::empty(tokens.sizes(), f32);
  Tensor entropy = torch::empty(tokens.sizes(), f32);
  Tensor kept, top_lp, top_t;
  if (stats) kept = torch::empty({rows, 4}, f32);
  if (top_k) {
    std::vector<int64_t> shape = tokens.sizes().vec();
    shape.push_back(k);
    top_lp = torch::empty(shape, f32);
    top_t = torch::empty(shape, logits.options().dtype(torch::kLong));
  }
  if (rows) {
    blk::LogProbs a{};
    a.logits = r.logits.t.data_ptr();
    a.tokens = r.tokens.data_ptr<int64_t>();
    a.mask = mask.has_value() ? (const uint8_t*)r.mask.t.data_ptr() : nullptr;
    a.logprob = logprob.data_ptr<float>();
    a.entropy = entropy.data_ptr<float>();
    a.stats = stats ? kept.data_ptr<float>() : nullptr;
    a.top_logprobs = k ? top_lp.data_ptr<float>() : nullptr;
    a.top_tokens = k ? top_t.data_ptr<int64_t>() : nullptr;
    a.rows = rows;
    a.stride = r.logits.stride;
    a.mask_stride = mask.has_value() ? r.mask.stride : 0;
    a.ignore_index = ignore_index;
    a.width = (int)logits.size(-1);
    a.top_k = (int)k;
    a.inv_temperature = (float)(1.0 / temperature);
    blk::token_logprobs_fwd(a, r.dtype, stream_of(logits));
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {logprob, entropy, top_lp, top_t, kept};
}

Tensor token_logprobs_bwd(const Tensor& logits, const OptTensor& mask,
                          const Tensor& stats, OptTensor dlogprob, OptTensor dentropy,
                          double temperature) {
  const c10::DeviceGuard guard(logits.device());
  const Rows l = rows_of(logits);
  Rows m;
  if (mask.has_value())
    m = rows_of(mask->sizes() == logits.sizes() ? *mask : mask->expand(logits.sizes()));
  for (OptTensor* t : {&dlogprob, &dentropy})
    if (t->has_value()) *t = (*t)->to(torch::kFloat32).contiguous();
  Tensor dlogits = torch::empty(logits.sizes(), logits.options());
  if (l.rows) {
    blk::LogProbsBwd a{};
    a.logits = l.t.data_ptr();
    a.mask = mask.has_value() ? (const uint8_t*)m.t.data_ptr() : nullptr;
    a.stats = stats.data_ptr<float>();
    a.dlogprob = (const float*)ptr(dlogprob);
    a.dentropy = (const float*)ptr(dentropy);
    a.dlogits = dlogits.data_ptr();
    a.rows = l.rows;
    a.stride = l.stride;
    a.mask_stride = mask.has_value() ? m.stride : 0;
    a.width = (int)logits.size(-1);
    a.inv_temperature = (float)(1.0 / temperature);
    blk::token_logprobs_bwd(a, dtype_of(logits, "logits"), stream_of(logits));
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return dlogits;
}

struct LogProbs : torch::autograd::Function<LogProbs> {
  static variable_list forward(AutogradContext* ctx, Tensor logits, Tensor tokens,
                               OptTensor mask, double temperature, int64_t top_k,
                               int64_t ignore_index) {
    const auto r = token_logprobs_fwd(logits, tokens, mask, temperature, top_k,
                                      ignore_index, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, none_or(mask), r[4]});
    ctx->saved_data["temperature"] = temperature;
    if (!top_k) return {r[0], r[1]};
    ctx->mark_non_differentiable({r[2], r[3]});
    return {r[0], r[1], r[2], r[3]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor d;
    if (grads[0].defined() || grads[1].defined())
      d = token_logprobs_bwd(saved[0], opt(saved[1]), saved[2], opt(grads[0]),
                             opt(grads[1]), ctx->saved_data["temperature"].toDouble());
    return once({d, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, "token_logprobs");
  }
};

// -> logprob, entropy, top_logprobs, top_tokens (None without top_k)
std::tuple<Tensor, Tensor, OptTensor, OptTensor> token_logprobs(
    Tensor logits, Tensor tokens, OptTensor mask, double temperature, int64_t top_k,
    int64_t ignore_index) {
  const OptTensor leaf = logits;
  refuse_tangents({&leaf}, "token_logprobs");
  if (wants_grad({&leaf})) {
    const auto r = LogProbs::apply(logits, tokens, mask, temperature, top_k, ignore_index);
    if (!top_k) return {r[0], r[1], OptTensor(), OptTensor()};
    return {r[0], r[1], r[2], r[3]};
  }
  const auto r = token_logprobs_fwd(logits, tokens, mask, temperature, top_k, ignore_index,
                                    false);
  return {r[0], r[1], opt(r[2]), opt(r[3])};
}

// ----------------------------------------------------------- linear layers

int linear_dtype(const Tensor& t, const char* name) {
  const int d = dtype_of(t, name);
  TORCH_CHECK_TYPE(d != blk::kF32, name, " must be bfloat16 or float16, not float32");
  return d;
}

// Rows as the products take them: of 8 elements at least, and with a stride that
// leaves a tile's offsets in 32 bits.
Rows product_rows_of(const Tensor& in) {
  if (in.size(-1) < 8) {
    // the padding keeps another order of the dimensions, such as channels-last
    const Tensor wide = torch::constant_pad_nd(in, {0, 8 - in.size(-1)}, 0).contiguous();
    return {wide, wide.numel() / 8, 8};
  }
  Rows r = rows_of(in);
  if (r.stride < 0 || r.stride >= (1 << 22)) r = {in.contiguous(), r.rows, in.size(-1)};
  return r;
}

bool chunked(const Rows& r) {
  return r.t.size(-1) % 8 == 0 && r.stride % 8 == 0 &&
         reinterpret_cast<uintptr_t>(r.t.data_ptr()) % 16 == 0;
}

// A weight's rows as whole aligned chunks of 8, with zeros behind them: a copy
// where they are not, so that the other operand alone decides how loads go.
Rows weight_rows_of(const Tensor& in) {
  const Rows r = product_rows_of(in);
  if (chunked(r)) return r;
  const Tensor wide = torch::constant_pad_nd(in, {0, (8 - in.size(-1) % 8) % 8}, 0).contiguous();
  return {wide, r.rows, wide.size(-1)};
}

void run_product(blk::Product& a, int dtype, const Tensor& like) {
  TORCH_CHECK_VALUE(a.i < (int64_t)1 << 32 && a.r < (int64_t)1 << 32,
                    "more than 2^32 rows");
  // a launch has at most 2^32 threads
  TORCH_CHECK_VALUE(((a.i + 127) / 128) * ((a.j + 127) / 128) < (int64_t)1 << 24,
                    "a product of ", a.i, " by ", a.j, " is too large");
  a.splits = blk::product_splits(a);
  Tensor partial;
  if (a.splits > 1) {
    a.partial_cols = (a.j + 7) / 8 * 8;
    partial = torch::empty({a.splits, a.i, a.partial_cols},
                           like.options().dtype(torch::kFloat32));
    a.partial = partial.data_ptr<float>();
  }
  blk::product(a, dtype, stream_of(like));
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

// -> y, z (undefined without `save`)
std::array<Tensor, 2> linear_act_fwd(Tensor x, Tensor weight, OptTensor bias,
                                   OptTensor residual, int64_t act, bool save) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be on a GPU");
  check_width(x, "x");
  const int dtype = linear_dtype(x, "x");
  check_device(weight, x, "weight");
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type() ||
                       weight.scalar_type() == torch::kFloat32,
                   "weight must be float32 or of x's type");
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.size(0) >= 1,
                    "weight must be (outputs, ", x.size(-1), ")");
  const int64_t n = weight.size(0);
  TORCH_CHECK_VALUE(n < (1 << 22) && x.size(-1) < (1 << 22),
                    "a layer's widths must be below 2^22");
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n;
  if (bias.has_value()) {
    check_device(*bias, x, "bias");
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == n, "bias must have ", n, " elements");
    TORCH_CHECK_TYPE(bias->scalar_type() == x.scalar_type() ||
                         bias->scalar_type() == torch::kFloat32,
                     "bias must be float32 or of x's type");
  }
  if (residual.has_value()) {
    check_device(*residual, x, "residual");
    TORCH_CHECK_TYPE(residual->scalar_type() == x.scalar_type(), "residual must be of x's type");
    TORCH_CHECK_VALUE(residual->sizes() == c10::IntArrayRef(shape),
                      "residual must be of the output's shape");
  }
  const c10::DeviceGuard guard(x.device());
  const Rows xr = product_rows_of(x);
  const Tensor w = weight.to(x.scalar_type());
  const Rows wr = chunked(xr) ? weight_rows_of(w) : product_rows_of(w);
  if (bias.has_value()) bias = bias->contiguous();
  const Rows rr = residual.has_value() ? rows_of(*residual) : Rows{x, 0, 0};
  Tensor y = torch::empty(shape, x.options());
  Tensor z;
  if (save)
    z = torch::empty(shape, act == blk::kRelu ? x.options()
                                              : x.options().dtype(torch::kFloat32));
  if (xr.rows) {
    blk::Product a{};
    a.p = xr.t.data_ptr();
    a.q = wr.t.data_ptr();
    a.p_stride = xr.stride;
    a.q_stride = wr.stride;
    a.p_cols = xr.t.size(-1);
    a.q_cols = wr.t.size(-1);
    a.i = xr.rows;
    a.j = n;
    a.r = x.size(-1);
    a.out = y.data_ptr();
    a.bias = ptr(bias);
    a.bias_f32 = bias.has_value() && bias->scalar_type() == torch::kFloat32;
    a.residual = residual.has_value() ? rr.t.data_ptr() : nullptr;
    a.residual_stride = rr.stride;
    a.z = save ? z.data_ptr() : nullptr;
    a.act = (int)act;
    run_product(a, dtype, x);
  }
  return {y, z};
}

// saved: z, or y of a relu; -> dx, dweight, dbias (undefined where not needed)
std::array<Tensor, 3> linear_act_bwd(Tensor dy, Tensor x, Tensor weight, Tensor saved,
                                     int64_t act, bool need_x, bool need_w, bool need_b,
                                     torch::ScalarType bias_type) {
  const int dtype = linear_dtype(x, "x");
  const int64_t n = weight.size(0), k = weight.size(1);
  const c10::DeviceGuard guard(x.device());
  const Rows yr = rows_of(dy);
  const int64_t rows = yr.rows;
  Tensor dx, dw, db;
  if (need_x) dx = torch::empty(x.sizes(), x.options());
  if (need_w) dw = torch::empty({n, k}, weight.options());
  if (need_b) db = torch::empty({n}, x.options().dtype(bias_type));
  if (!rows) {
    if (need_w) dw.zero_();
    if (need_b) db.zero_();
    return {dx, dw, db};
  }
  const hipStream_t stream = stream_of(x);
  Tensor dz = yr.t;
  if (act || need_b) {
    blk::ActBwd b{};
    b.blocks = blk::act_bwd_blocks(rows, n);
    Tensor partial;
    if (need_b && b.blocks > 1)
      partial = torch::empty({b.blocks * n}, x.options().dtype(torch::kFloat32));
    b.dy = yr.t.data_ptr();
    if (act) {
      dz = torch::empty({rows, n}, x.options());
      b.z = saved.data_ptr();
      b.dz = dz.data_ptr();
    }
    b.partial = partial.defined() ? partial.data_ptr<float>() : nullptr;
    b.dbias = need_b ? db.data_ptr() : nullptr;
    b.dbias_f32 = bias_type == torch::kFloat32;
    b.rows = rows;
    b.n = n;
    b.dy_stride = yr.stride;
    b.act = (int)act;
    blk::act_bwd(b, dtype, stream);
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  const Rows zr = need_x || need_w ? product_rows_of(dz) : Rows{dz, 0, 0};
  if (need_x) {
    const Tensor w = weight.to(x.scalar_type());
    const Rows wr = chunked(zr) ? weight_rows_of(w) : product_rows_of(w);
    blk::Product a{};
    a.p = zr.t.data_ptr();
    a.q = wr.t.data_ptr();
    a.p_stride = zr.stride;
    a.q_stride = wr.stride;
    a.p_cols = zr.t.size(-1);
    a.q_cols = wr.t.size(-1);
    a.i = rows;
    a.j = k;
    a.r = n;
    a.q_t = true;
    a.out = dx.data_ptr();
    run_product(a, dtype, x);
  }
  if (need_w) {
    const Rows xr = product_rows_of(x);
    blk::Product a{};
    a.p = zr.t.data_ptr();
    a.q = xr.t.data_ptr();
    a.p_stride = zr.stride;
    a.q_stride = xr.stride;
    a.p_cols = zr.t.size(-1);
    a.q_cols = xr.t.size(-1);
    a.i = n;
    a.j = k;
    a.r = rows;
    a.p_t = a.q_t = true;
    a.out = dw.data_ptr();
    a.out_f32 = weight.scalar_type() == torch::kFloat32;
    run_product(a, dtype, x);
  }
  return {dx, dw, db};
}

struct LinearAct : torch::autograd::Function<LinearAct> {
  enum { kX = 1, kWeight = 2, kBias = 4, kResidual = 8 };

  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor weight, OptTensor bias,
                        OptTensor residual, int64_t act) {
    // a relu's sign can be read off its output where no residual covers it
    const bool from_y = act == blk::kRelu && !residual.has_value();
    const auto r = linear_act_fwd(x, weight, bias, residual, act,
                                  act != blk::kNone && !from_y);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, from_y ? r[0] : r[1]});
    int64_t need = x.requires_grad() ? kX : 0;
    if (weight.requires_grad()) need |= kWeight;
    if (bias.has_value() && bias->requires_grad()) need |= kBias;
    if (residual.has_value() && residual->requires_grad()) need |= kResidual;
    ctx->saved_data["need"] = need;
    ctx->saved_data["act"] = act;
    ctx->saved_data["type"] = (int64_t)(bias.has_value() ? bias->scalar_type()
                                                         : x.scalar_type());
    return r[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    const Tensor dy = grads[0];
    std::array<Tensor, 3> r;
    if (dy.defined() && need & (kX | kWeight | kBias))
      r = linear_act_bwd(dy, saved[0], saved[1], saved[2],
                         ctx->saved_data["act"].toInt(), need & kX, need & kWeight,
                         need & kBias,
                         (torch::ScalarType)ctx->saved_data["type"].toInt());
    return once({r[0], r[1], r[2], need & kResidual ? dy : Tensor(), Tensor()},
                "linear_act");
  }
};

Tensor linear_act(Tensor x, Tensor weight, OptTensor bias, OptTensor residual, int64_t act) {
  const OptTensor leaf = x, w = weight;
  refuse_tangents({&leaf, &w, &bias, &residual}, "linear_act");
  if (wants_grad({&leaf, &w, &bias, &residual}))
    return LinearAct::apply(x, weight, bias, residual, act);
  return linear_act_fwd(x, weight, bias, residual, act, false)[0];
}

// ----------------------------------------------------------- gradient norm

struct Span {
  uintptr_t lo, hi;
  bool operator<(const Span& o) const { return lo < o.lo; }
};

Span span_of(const Tensor& t) {
  const auto lo = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {lo, lo + (uintptr_t)t.numel() * t.element_size()};
}

void sort_spans(std::vector<Span>& v) {
  if (!std::is_sorted(v.begin(), v.end())) std::sort(v.begin(), v.end());
}

// -> norm; scales into `outs`, or in place without them
Tensor clip_grad_norm(std::vector<Tensor> grads,
                      c10::optional<std::vector<Tensor>> outs, int64_t order,
                      double max_norm, double eps, bool scale) {
  TORCH_CHECK_VALUE(!grads.empty(), "no tensors were given");
  TORCH_CHECK_VALUE(!outs.has_value() || outs->size() == grads.size(),
                    "out must have as many tensors as the list");
  const Tensor first = grads[0];
  TORCH_CHECK_VALUE(first.is_cuda(), "the tensors must be on a GPU");
  const c10::DeviceGuard guard(first.device());
  static constexpr int kSize[3] = {4, 2, 2};
  const int listed = (int)grads.size();
  std::vector<blk::GradTensor> g(listed);
  std::vector<Tensor> kept;                         // copies that the kernels use
  std::vector<std::pair<Tensor, Tensor>> back;      // (where it belongs, copy)
  std::vector<Span> read, written;
  if (scale) written.reserve(listed);
  if (scale && outs.has_value()) read.reserve(listed);
  for (int i = 0; i < listed; ++i) {
    Tensor in = grads[i];
    TORCH_CHECK_TYPE(in.layout() == torch::kStrided, "sparse tensors are not taken");
    refuse_tangent(in, "a norm of gradients");
    check_device(in, first, "a tensor");
    g[i].in_dtype = dtype_of(in, "a tensor");
    g[i].numel = in.numel();
    const bool dense = in.is_non_overlapping_and_dense();
    Tensor out = in;
    if (scale && outs.has_value()) {
      out = (*outs)[i];
      refuse_tangent(out, "clipping");
      check_device(out, first, "an output");
      TORCH_CHECK_VALUE(out.sizes() == in.sizes(), "an output must be of its tensor's shape");
      const bool dense_out = out.is_non_overlapping_and_dense();
      TORCH_CHECK_VALUE(dense_out, "an output must be dense, without gaps or overlaps");
      if (g[i].numel) {
        written.push_back(span_of(out));
        const bool itself = out.data_ptr() == in.data_ptr() && out.strides() == in.strides() &&
                            out.scalar_type() == in.scalar_type();
        if (dense && !itself) read.push_back(span_of(in));
      }
      if (!dense || out.strides() != in.strides()) {
        Tensor same = torch::empty_strided(out.sizes(), out.strides(), in.options());
        same.copy_(in);
        in = same;
        kept.push_back(in);
      }
    } else if (!dense) {
      TORCH_CHECK_VALUE(!scale || !g[i].numel ||
                            at::has_internal_overlap(in) != at::MemOverlap::Yes,
                        "a tensor overlaps itself and cannot be scaled in place");
      in = in.contiguous();
      kept.push_back(in);
      if (scale) back.emplace_back(grads[i], in);
      out = in;
    } else if (scale && g[i].numel) {
      written.push_back(span_of(out));
    }
    g[i].out_dtype = dtype_of(out, "an output");
    g[i].in = in.data_ptr();
    g[i].out = out.data_ptr();
  }
  if (scale) {
    sort_spans(written);
    for (size_t i = 1; i < written.size(); ++i)
      TORCH_CHECK_VALUE(written[i - 1].hi <= written[i].lo,
                        "two of the tensors to be written share memory");
    sort_spans(read);
    for (size_t i = 0, j = 0; i < read.size() && j < written.size();) {
      TORCH_CHECK_VALUE(read[i].hi <= written[j].lo || written[j].hi <= read[i].lo,
                        "an output shares memory with a tensor of the list");
      if (read[i].hi <= written[j].lo) ++i; else ++j;
    }
  }
  for (size_t i = 0; i < back.size(); ++i)
    for (size_t j = 0; j < i; ++j)
      TORCH_CHECK_VALUE(back[i].first.data_ptr() != back[j].first.data_ptr(),
                        "two of the tensors to be written share memory");
  // autograd notices a change of what it has saved by the version: nothing behind here
  // refuses the call
  if (scale)
    for (const Tensor& t : outs.has_value() ? *outs : grads)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  // neighbours in memory are one tensor to the kernels: a bucket's views end to end
  // are one entry instead of a thousand
  int count = 0;
  for (int i = 0; i < listed; ++i) {
    if (!g[i].numel) continue;
    if (count) {
      blk::GradTensor& last = g[count - 1];
      if (last.in_dtype == g[i].in_dtype && last.out_dtype == g[i].out_dtype &&
          (const char*)last.in + last.numel * kSize[last.in_dtype] == g[i].in &&
          (char*)last.out + last.numel * kSize[last.out_dtype] == g[i].out) {
        last.numel += g[i].numel;
        continue;
      }
    }
    g[count++] = g[i];
  }
  int64_t chunk = 0;
  const int64_t blocks = blk::grad_norm_blocks(g.data(), count, &chunk);
  const auto f32 = first.options().dtype(torch::kFloat32).requires_grad(false);
  Tensor partial = torch::empty({blocks}, f32.dtype(torch::kFloat64));
  Tensor norm = torch::empty({}, f32), coef = torch::empty({}, f32);
  const hipStream_t stream = stream_of(first);
  blk::grad_norm(g.data(), count, chunk, (int)order, partial.data_ptr<double>(),
                 blocks, norm.data_ptr<float>(), coef.data_ptr<float>(),
                 (float)max_norm, (float)eps, stream);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  if (scale) {
    blk::grad_scale(g.data(), count, coef.data_ptr<float>(), stream);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    for (auto& p : back) p.first.copy_(p.second);
  }
  return norm;
}

}  // namespace

void register_block_ops(pybind11::module_& m) {
  m.def("layer_norm", &layer_norm, "layer norm of rows");
  m.def("add_layer_norm", &add_layer_norm,
        "residual sum and layer norm of rows -> (y, sum)");
  m.def("token_logprobs", &token_logprobs,
        "log probabilities of tokens, entropy and top alternatives");
  m.def("linear_act", &linear_act,
        "linear layer with bias, activation and residual (MFMA)");
  m.def("clip_grad_norm", &clip_grad_norm,
        "norm of a list of tensors, and their scaling to a largest norm");
}
