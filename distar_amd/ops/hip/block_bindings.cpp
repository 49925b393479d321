// Python bindings of the kernels around the policy transformer: checks of the
// arguments, outputs and workspaces, and the launch on the current stream of
// the tensors' own device.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <limits>

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

// -> y, s (x itself without a residual), mean, rstd (empty without `stats`)
std::vector<Tensor> layer_norm_fwd(Tensor x, OptTensor residual, OptTensor weight,
                                   OptTensor bias, double eps, bool stats) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be on a GPU");
  check_width(x, "x");
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
  const auto f32 = x.options().dtype(torch::kFloat32);
  Tensor mean = torch::empty({stats ? xr.rows : 0}, f32);
  Tensor rstd = torch::empty({stats ? xr.rows : 0}, f32);
  if (xr.rows) {
    blk::LayerNormFwd a{};
    a.x = xr.t.data_ptr();
    a.residual = residual.has_value() ? rr.t.data_ptr() : nullptr;
    a.weight = ptr(weight);
    a.bias = ptr(bias);
    a.y = y.data_ptr();
    a.s = residual.has_value() ? s.data_ptr() : nullptr;
    a.mean = stats ? mean.data_ptr<float>() : nullptr;
    a.rstd = stats ? rstd.data_ptr<float>() : nullptr;
    a.rows = xr.rows;
    a.x_stride = xr.stride;
    a.r_stride = rr.stride;
    a.width = (int)x.size(-1);
    a.eps = (float)eps;
    blk::layer_norm_fwd(a, dtype, wdtype, stream_of(x));
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return {y, s, mean, rstd};
}

// -> dx, dweight, dbias (empty without `params`)
std::vector<Tensor> layer_norm_bwd(Tensor dy, OptTensor ds, Tensor s, Tensor mean,
                                   Tensor rstd, OptTensor weight, bool params,
                                   torch::ScalarType param_type) {
  TORCH_CHECK_VALUE(s.is_cuda(), "s must be on a GPU");
  check_width(s, "s");
  const int dtype = dtype_of(s, "s");
  const OptTensor none;
  int wdtype = check_affine(s, weight, none, dtype);
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
  const auto f32 = s.options().dtype(torch::kFloat32);
  TORCH_CHECK_VALUE(mean.is_contiguous() && mean.numel() == sr.rows &&
                        mean.scalar_type() == torch::kFloat32 &&
                        rstd.is_contiguous() && rstd.numel() == sr.rows &&
                        rstd.scalar_type() == torch::kFloat32,
                    "mean and rstd must be the forward pass's own");
  check_device(mean, s, "mean");
  check_device(rstd, s, "rstd");
  Tensor dx = torch::empty(s.sizes(), s.options());
  const auto ptype = s.options().dtype(param_type);
  Tensor dw = torch::empty({params ? width : 0}, ptype);
  Tensor db = torch::empty({params ? width : 0}, ptype);
  if (params) {
    const int d = dtype_of(dw, "weight or bias");
    TORCH_CHECK_TYPE(d == dtype || d == blk::kF32,
                     "weight and bias must be float32 or of the input's type");
    TORCH_CHECK_TYPE(!weight.has_value() || d == wdtype,
                     "weight and bias must be of one type");
    wdtype = d;
  }
  if (!sr.rows) {
    dw.zero_();
    db.zero_();
    return {dx, dw, db};
  }
  if (weight.has_value()) weight = weight->contiguous();
  blk::LayerNormBwd a{};
  a.blocks = blk::layer_norm_bwd_blocks(sr.rows, (int)width, dtype);
  Tensor partial = torch::empty({params ? a.blocks * 2 * width : 0}, f32);
  a.dy = yr.t.data_ptr();
  a.ds = ds.has_value() ? dr.t.data_ptr() : nullptr;
  a.s = sr.t.data_ptr();
  a.weight = ptr(weight);
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.dx = dx.data_ptr();
  a.dweight = params ? dw.data_ptr() : nullptr;
  a.dbias = params ? db.data_ptr() : nullptr;
  a.partial = params ? partial.data_ptr<float>() : nullptr;
  a.rows = sr.rows;
  a.dy_stride = yr.stride;
  a.ds_stride = dr.stride;
  a.s_stride = sr.stride;
  a.width = (int)width;
  blk::layer_norm_bwd(a, dtype, wdtype, stream_of(s));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {dx, dw, db};
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
  TORCH_CHECK_TYPE(tokens.scalar_type() == torch::kLong, "tokens must be int64");
  TORCH_CHECK_VALUE(tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                    "tokens must have the shape of logits without its last dimension");
  r.tokens = tokens.contiguous();
  if (mask.has_value()) {
    check_device(*mask, logits, "mask");
    TORCH_CHECK_TYPE(mask->scalar_type() == torch::kBool, "mask must be bool");
    r.mask = rows_of(mask->expand(logits.sizes()));
  }
  return r;
}

// -> logprob, entropy, row_max, row_logsum (both empty without `stats`),
//    top_logprobs, top_tokens
std::vector<Tensor> token_logprobs_fwd(Tensor logits, Tensor tokens, OptTensor mask,
                                       double temperature, int64_t top_k,
                                       int64_t ignore_index, bool stats) {
  const c10::OptionalDeviceGuard guard(
      logits.is_cuda() ? c10::optional<c10::Device>(logits.device()) : c10::nullopt);
  const LogitRows r = check_logits(logits, tokens, mask);
  const int64_t rows = r.logits.rows;
  const int64_t k = std::min<int64_t>(top_k, logits.size(-1));
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= 64, "top_k must be 0 to 64");
  const auto f32 = logits.options().dtype(torch::kFloat32);
  Tensor logprob = torch::empty(tokens.sizes(), f32);
  Tensor entropy = torch::empty(tokens.sizes(), f32);
  Tensor row_max = torch::empty({stats ? rows : 0}, f32);
  Tensor row_logsum = torch::empty({stats ? rows : 0}, f32);
  std::vector<int64_t> shape = tokens.sizes().vec();
  shape.push_back(k);
  Tensor top_lp = torch::empty(shape, f32);
  Tensor top_t = torch::empty(shape, logits.options().dtype(torch::kLong));
  if (rows) {
    blk::LogProbs a{};
    a.logits = r.logits.t.data_ptr();
    a.tokens = r.tokens.data_ptr<int64_t>();
    a.mask = mask.has_value() ? (const uint8_t*)r.mask.t.data_ptr() : nullptr;
    a.logprob = logprob.data_ptr<float>();
    a.entropy = entropy.data_ptr<float>();
    a.row_max = stats ? row_max.data_ptr<float>() : nullptr;
    a.row_logsum = stats ? row_logsum.data_ptr<float>() : nullptr;
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
  return {logprob, entropy, row_max, row_logsum, top_lp, top_t};
}

Tensor token_logprobs_bwd(Tensor logits, Tensor tokens, OptTensor mask,
                          Tensor entropy, Tensor row_max, Tensor row_logsum,
                          OptTensor dlogprob, OptTensor dentropy,
                          double temperature, int64_t ignore_index) {
  const c10::OptionalDeviceGuard guard(
      logits.is_cuda() ? c10::optional<c10::Device>(logits.device()) : c10::nullopt);
  const LogitRows r = check_logits(logits, tokens, mask);
  const int64_t rows = r.logits.rows;
  for (const Tensor* t : {&entropy, &row_max, &row_logsum}) {
    check_device(*t, logits, "a row's statistics");
    TORCH_CHECK_VALUE(t->is_contiguous() && t->numel() == rows &&
                          t->scalar_type() == torch::kFloat32,
                      "a row's statistics must be the forward pass's own");
  }
  for (OptTensor* t : {&dlogprob, &dentropy}) {
    if (!t->has_value()) continue;
    check_device(**t, logits, "a gradient");
    TORCH_CHECK_VALUE((*t)->sizes() == tokens.sizes(), "a gradient must be of tokens' shape");
    *t = (*t)->to(torch::kFloat32).contiguous();
  }
  Tensor dlogits = torch::empty(logits.sizes(), logits.options());
  if (rows) {
    blk::LogProbsBwd a{};
    a.logits = r.logits.t.data_ptr();
    a.tokens = r.tokens.data_ptr<int64_t>();
    a.mask = mask.has_value() ? (const uint8_t*)r.mask.t.data_ptr() : nullptr;
    a.entropy = entropy.data_ptr<float>();
    a.row_max = row_max.data_ptr<float>();
    a.row_logsum = row_logsum.data_ptr<float>();
    a.dlogprob = (const float*)ptr(dlogprob);
    a.dentropy = (const float*)ptr(dentropy);
    a.dlogits = dlogits.data_ptr();
    a.rows = rows;
    a.stride = r.logits.stride;
    a.mask_stride = mask.has_value() ? r.mask.stride : 0;
    a.ignore_index = ignore_index;
    a.width = (int)logits.size(-1);
    a.inv_temperature = (float)(1.0 / temperature);
    blk::token_logprobs_bwd(a, r.dtype, stream_of(logits));
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return dlogits;
}

// ----------------------------------------------------------- linear layers

int linear_dtype(const Tensor& t, const char* name) {
  const int d = dtype_of(t, name);
  TORCH_CHECK_TYPE(d != blk::kF32, name, " must be bfloat16 or float16, not float32");
  return d;
}

void run_product(blk::Product& a, int dtype, const Tensor& like) {
  TORCH_CHECK_VALUE(a.i <= (int64_t)1 << 30 && a.j <= (int64_t)1 << 22,
                    "a product of ", a.i, " by ", a.j, " is too large");
  a.splits = blk::product_splits(a);
  Tensor partial;
  if (a.splits > 1) {
    partial = torch::empty({a.splits, a.i, a.j}, like.options().dtype(torch::kFloat32));
    a.partial = partial.data_ptr<float>();
  }
  blk::product(a, dtype, stream_of(like));
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

// -> y, z (empty without `save`)
std::vector<Tensor> linear_act_fwd(Tensor x, Tensor weight, OptTensor bias,
                                   OptTensor residual, int64_t act, bool save) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be on a GPU");
  check_width(x, "x");
  const int dtype = linear_dtype(x, "x");
  check_device(weight, x, "weight");
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type(), "weight must be of x's type");
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.size(0) >= 1,
                    "weight must be (outputs, ", x.size(-1), ")");
  const int64_t n = weight.size(0);
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
  const Rows xr = rows_of(x), wr = rows_of(weight);
  if (bias.has_value()) bias = bias->contiguous();
  const Rows rr = residual.has_value() ? rows_of(*residual) : Rows{x, 0, 0};
  Tensor y = torch::empty(shape, x.options());
  Tensor z = torch::empty(save ? shape : std::vector<int64_t>{0}, x.options());
  if (xr.rows) {
    blk::Product a{};
    a.p = xr.t.data_ptr();
    a.q = wr.t.data_ptr();
    a.p_stride = xr.stride;
    a.q_stride = wr.stride;
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

// saved: z, or y of a relu; -> dx, dweight, dbias (empty where not needed)
std::vector<Tensor> linear_act_bwd(Tensor dy, Tensor x, Tensor weight, OptTensor saved,
                                   int64_t act, bool need_x, bool need_w, bool need_b,
                                   torch::ScalarType weight_type,
                                   torch::ScalarType bias_type) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be on a GPU");
  const int dtype = linear_dtype(x, "x");
  const int64_t n = weight.size(0), k = weight.size(1);
  check_device(dy, x, "dy");
  check_device(weight, x, "weight");
  TORCH_CHECK_TYPE(dy.scalar_type() == x.scalar_type() &&
                       weight.scalar_type() == x.scalar_type(),
                   "dy and weight must be of x's type");
  TORCH_CHECK_VALUE(x.size(-1) == k && dy.size(-1) == n && dy.numel() / n == x.numel() / k,
                    "dy, x and weight do not fit together");
  TORCH_CHECK_VALUE(act == blk::kNone || (saved.has_value() && saved->is_contiguous() &&
                                          saved->numel() == dy.numel() &&
                                          saved->scalar_type() == x.scalar_type()),
                    "the forward pass's values are missing");
  const c10::DeviceGuard guard(x.device());
  const Rows yr = rows_of(dy), xr = rows_of(x), wr = rows_of(weight);
  const int64_t rows = xr.rows;
  Tensor dx = torch::empty(need_x ? x.sizes().vec() : std::vector<int64_t>{0}, x.options());
  Tensor dw = torch::empty({need_w ? n : 0, k}, x.options().dtype(weight_type));
  Tensor db = torch::empty({need_b ? n : 0}, x.options().dtype(bias_type));
  if (!rows) {
    dw.zero_();
    db.zero_();
    return {dx, dw, db};
  }
  const hipStream_t stream = stream_of(x);
  Tensor dz = yr.t;
  int64_t dz_stride = yr.stride;
  if (act || need_b) {
    blk::ActBwd b{};
    b.blocks = blk::act_bwd_blocks(rows, n);
    Tensor partial = torch::empty({need_b ? b.blocks * n : 0},
                                  x.options().dtype(torch::kFloat32));
    b.dy = yr.t.data_ptr();
    if (act) {
      dz = torch::empty({rows, n}, x.options());
      dz_stride = n;
      b.z = saved->data_ptr();
      b.dz = dz.data_ptr();
    }
    b.partial = need_b ? partial.data_ptr<float>() : nullptr;
    b.dbias = need_b ? db.data_ptr() : nullptr;
    b.dbias_f32 = bias_type == torch::kFloat32;
    b.rows = rows;
    b.n = n;
    b.dy_stride = yr.stride;
    b.act = (int)act;
    blk::act_bwd(b, dtype, stream);
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  if (need_x) {
    blk::Product a{};
    a.p = dz.data_ptr();
    a.q = wr.t.data_ptr();
    a.p_stride = dz_stride;
    a.q_stride = wr.stride;
    a.i = rows;
    a.j = k;
    a.r = n;
    a.q_t = true;
    a.out = dx.data_ptr();
    run_product(a, dtype, x);
  }
  if (need_w) {
    blk::Product a{};
    a.p = dz.data_ptr();
    a.q = xr.t.data_ptr();
    a.p_stride = dz_stride;
    a.q_stride = xr.stride;
    a.i = n;
    a.j = k;
    a.r = rows;
    a.p_t = a.q_t = true;
    a.out = dw.data_ptr();
    a.out_f32 = weight_type == torch::kFloat32;
    run_product(a, dtype, x);
  }
  return {dx, dw, db};
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

// -> norm, coefficient; scales into `outs`, or in place where that is `grads`
std::vector<Tensor> clip_grad_norm(std::vector<Tensor> grads,
                                   c10::optional<std::vector<Tensor>> outs,
                                   int64_t order, double max_norm, double eps,
                                   bool scale) {
  TORCH_CHECK_VALUE(!grads.empty(), "no tensors were given");
  TORCH_CHECK_VALUE(!outs.has_value() || outs->size() == grads.size(),
                    "out must have as many tensors as the list");
  const Tensor first = grads[0];
  TORCH_CHECK_VALUE(first.is_cuda(), "the tensors must be on a GPU");
  const c10::DeviceGuard guard(first.device());
  const int count = (int)grads.size();
  std::vector<blk::GradTensor> g(count);
  std::vector<Tensor> kept;                         // copies that the kernels use
  std::vector<std::pair<Tensor, Tensor>> back;      // (where it belongs, copy)
  std::vector<Span> read, written;
  if (scale) written.reserve(count);
  if (scale && outs.has_value()) read.reserve(count);
  for (int i = 0; i < count; ++i) {
    Tensor in = grads[i];
    TORCH_CHECK_TYPE(in.layout() == torch::kStrided, "sparse tensors are not taken");
    check_device(in, first, "a tensor");
    g[i].in_dtype = dtype_of(in, "a tensor");
    g[i].numel = in.numel();
    const bool dense = in.is_non_overlapping_and_dense();
    Tensor out = in;
    if (scale && outs.has_value()) {
      out = (*outs)[i];
      check_device(out, first, "an output");
      TORCH_CHECK_VALUE(out.sizes() == in.sizes(), "an output must be of its tensor's shape");
      const bool dense_out = out.is_non_overlapping_and_dense();
      TORCH_CHECK_VALUE(dense_out, "an output must be dense, without gaps or overlaps");
      if (g[i].numel) {
        written.push_back(span_of(out));
        if (dense) read.push_back(span_of(in));
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
    blk::grad_scale(g.data(), count, chunk, coef.data_ptr<float>(), stream);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    for (auto& p : back) p.first.copy_(p.second);
  }
  return {norm, coef};
}

}  // namespace

void register_block_ops(pybind11::module_& m) {
  m.def("layer_norm_fwd", &layer_norm_fwd,
        "layer norm of rows, behind an optional residual sum");
  m.def("layer_norm_bwd", &layer_norm_bwd, "layer norm backward");
  m.def("token_logprobs_fwd", &token_logprobs_fwd,
        "log probabilities of tokens, entropy and top alternatives");
  m.def("token_logprobs_bwd", &token_logprobs_bwd, "token log probabilities backward");
  m.def("linear_act_fwd", &linear_act_fwd,
        "linear layer with bias, activation and residual (MFMA)");
  m.def("linear_act_bwd", &linear_act_bwd, "linear layer with epilogue, backward");
  m.def("clip_grad_norm", &clip_grad_norm,
        "norm of a list of tensors, and their scaling to a largest norm");
}
