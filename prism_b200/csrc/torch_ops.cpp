// The torch side of the norm, rotary, 8-bit projection, clipping and packed and paged attention operators: argument checks,
// outputs and workspaces from torch's allocator, the current stream, autograd nodes, and the call of
// the C entry point.  In C++ because at one token the host's share of a call is longer than the
// kernel's (one row's norm: 14 us through Python attributes and ctypes), and a list of a thousand
// gradients costs microseconds here and hundreds of them there.
// Built against the installed torch and linked to libprism_bsa.so (prism_b200/build.py).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "prism_bsa.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Optional = std::optional<Tensor>;

// ------------------------------------------------------------------ errors
// A std::exception: autograd's threads carry those to the caller, and end the process on any other.
struct PrismFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(prism_status_t status, const char* name) {
  if (status != PRISM_OK)
    throw PrismFailure{std::string(name) + " failed (" + std::to_string((int)status) + "): " + prism_last_error()};
}

// ------------------------------------------------------------------ tensors
Tensor or_undefined(const Optional& t) { return t.has_value() ? *t : Tensor(); }
void* at(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

int dtype_code_or(const Tensor& t, int other) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return PRISM_BF16;
    case at::kHalf: return PRISM_FP16;
    case at::kFloat: return PRISM_FP32;
    default: return other;
  }
}
int dtype_code(const Tensor& t, const char* what) {
  const int code = dtype_code_or(t, -1);
  TORCH_CHECK_TYPE(code >= 0, what, " expects bf16, fp16 or fp32, got ", t.scalar_type());
  return code;
}

// The one CUDA device that every defined tensor is on.
int device_of(std::initializer_list<Tensor> tensors) {
  int device = -1;
  for (const Tensor& t : tensors) {
    if (!t.defined()) continue;
    if (!t.is_cuda()) throw PrismFailure{"prism_b200 ops require CUDA tensors (no CPU fallback)"};
    if (device < 0) device = t.get_device();
    TORCH_CHECK_VALUE(t.get_device() == device, "tensors on different devices: cuda:", device, " and ", t.device());
  }
  return device;
}

// Makes a device current for a launch on its current stream.
struct Launch {
  c10::cuda::CUDAGuard guard;
  cudaStream_t stream;
  explicit Launch(int device) : guard(device), stream(c10::cuda::getCurrentCUDAStream(device).stream()) {}
};

Tensor new_like(const Tensor& x, at::ScalarType type) {
  return at::empty(x.sizes(), x.options().dtype(type).requires_grad(false), at::MemoryFormat::Contiguous);
}
Tensor new_like(const Tensor& x) { return new_like(x, x.scalar_type()); }
Tensor fp32(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }

Tensor fp32_vector(const Tensor& w, int64_t n, const char* what) {
  if (!w.defined()) return w;
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == n, what, " must have shape [", n, "], got ", w.sizes());
  return w.to(at::kFloat).contiguous();
}

// [..., cols] -> a [rows, cols] view with unit column stride (a copy where there is none).
Tensor rows2d(const Tensor& t, int64_t cols) {
  if (!t.defined()) return t;
  const Tensor v = t.dim() == 2 ? t : t.reshape({-1, cols});
  return cols == 1 || v.stride(1) == 1 ? v : v.contiguous();
}
int64_t ld(const Tensor& t) { return t.defined() ? t.stride(0) : 0; }

bool wants_grad(std::initializer_list<Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// Forward-mode derivatives are not implemented: refused, since the kernels would drop the tangent.
void refuse_tangents(std::initializer_list<Tensor> tensors, const char* what) {
  for (const Tensor& t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, " has no forward-mode derivative");
}

// ------------------------------------------------------------------ RMS norm
struct Rows {
  int device, code;
  int64_t cols;
  Tensor x, r, w;
};

Rows rows_input(const Tensor& x, const Tensor& r, const Tensor& w, const char* what) {
  Rows in;
  in.device = device_of({x, r, w});
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, what, " needs at least one column");
  in.code = dtype_code(x, what);
  TORCH_CHECK_VALUE(!r.defined() || (r.sizes() == x.sizes() && r.scalar_type() == x.scalar_type()), what,
                    ": the residual must have the shape and type of x");
  in.cols = x.size(-1);
  TORCH_CHECK_VALUE(in.cols < (1 << 30), what, ": too many columns");
  in.x = rows2d(x, in.cols), in.r = rows2d(r, in.cols), in.w = fp32_vector(w, in.cols, "weight");
  return in;
}

// (y, h, rstd); h undefined without a residual.
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& r, const Tensor& w, double eps,
                                                bool want_rstd) {
  const Rows in = rows_input(x, r, w, "add_rms_norm");
  const int64_t rows = in.x.size(0);
  const Launch launch(in.device);
  Tensor y = new_like(x), h = r.defined() ? new_like(x) : Tensor(), rstd = want_rstd ? fp32({rows}, x) : Tensor();
  check(prism_add_rms_norm(at(in.x), ld(in.x), at(in.r), ld(in.r), (const float*)at(in.w), (float)eps, rows,
                           (int)in.cols, in.code, at(y), at(h), (float*)at(rstd), launch.stream),
        "prism_add_rms_norm");
  return {y, h, rstd};
}

// The gradients as parts of a graph that raises where it is differentiated.  `from`: what they depend on; the
// node leads there, or a derivative with respect to these alone would go past it.
variable_list without_derivative(const variable_list& grads, std::initializer_list<Tensor> from, const char* what) {
  const at::AutoGradMode grad(true);
  variable_list in;
  for (const Tensor& g : grads) in.push_back(g.defined() ? g.requires_grad_() : g);
  in.insert(in.end(), from);
  const auto node =
      std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": its gradient has no gradient", (int64_t)in.size());
  variable_list out = (*node)(std::move(in));
  out.resize(grads.size());
  return out;
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
  // absent tensors are empty optionals: they have no edge in the graph
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Optional& residual, const Optional& weight,
                               double eps) {
    const Tensor r = or_undefined(residual), w = or_undefined(weight);
    auto [y, h, rstd] = norm_forward(x, r, w, eps, true);
    ctx->save_for_backward({r.defined() ? h : x, rstd, w});
    ctx->saved_data["residual"] = r.defined();
    ctx->set_materialize_grads(false);
    return r.defined() ? variable_list{y, h} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &rstd = saved[1], &w = saved[2], &gy = grads[0];
    const Tensor gh = grads.size() > 1 ? grads[1] : Tensor();
    const bool has_r = ctx->saved_data["residual"].toBool();
    const bool want_w = w.defined() && ctx->needs_input_grad(has_r ? 2 : 1);
    Tensor dx = gh, dw;
    if (gy.defined()) {  // else h = x + r alone passes its gradient on
      const bool graph = at::GradMode::is_enabled();
      const at::NoGradGuard no_grad;
      const int64_t cols = h.size(-1);
      const Tensor g2 = rows2d(gy, cols), h2 = rows2d(h, cols), gh2 = rows2d(gh, cols);
      const Tensor w2 = fp32_vector(w, cols, "weight");
      const int64_t rows = h2.size(0);
      const Launch launch(h.get_device());
      dx = new_like(h);
      Tensor workspace;
      if (want_w) {
        dw = fp32({cols}, h);
        workspace = at::empty({(int64_t)prism_add_rms_norm_bwd_workspace_bytes(rows, (int)cols)},
                              h.options().dtype(at::kByte));
      }
      check(prism_add_rms_norm_bwd(at(g2), ld(g2), at(h2), ld(h2), at(gh2), ld(gh2), (const float*)at(w2),
                                   (const float*)at(rstd), rows, (int)cols, dtype_code(h, "add_rms_norm"), at(dx),
                                   at(workspace), (float*)at(dw), launch.stream),
            "prism_add_rms_norm_bwd");
      if (want_w) dw = dw.to(w.scalar_type());
      if (graph) {
        const variable_list out = without_derivative({dx, dw}, {gy, gh, h, w}, "add_rms_norm");
        dx = out[0], dw = out[1];
      }
    }
    const bool want_r = has_r && ctx->needs_input_grad(1);
    return {ctx->needs_input_grad(0) ? dx : Tensor(), want_r ? dx : Tensor(), dw, Tensor()};
  }
};

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const Optional& residual, const Optional& weight, double eps) {
  const Tensor r = or_undefined(residual), w = or_undefined(weight);
  refuse_tangents({x, r, w}, "add_rms_norm");
  if (wants_grad({x, r, w})) {
    const variable_list out = AddRmsNorm::apply(x, residual, weight, eps);
    return {out[0], r.defined() ? out[1] : x};
  }
  auto [y, h, rstd] = norm_forward(x, r, w, eps, false);
  return {y, r.defined() ? h : x};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_fp8(const Tensor& x, const Optional& residual, const Optional& weight,
                                                    double eps, bool normalize) {
  const char* what = normalize ? "add_rms_norm_fp8" : "quantize_rows_fp8";
  const Tensor r = or_undefined(residual), w = or_undefined(weight);
  refuse_tangents({x, r, w}, what);
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({x, r, w}), what, " is inference only: its 8-bit rounding has no gradient");
  const Rows in = rows_input(x, r, w, what);
  const Launch launch(in.device);
  Tensor y8 = new_like(x, at::kFloat8_e4m3fn), scale = fp32(x.sizes().slice(0, x.dim() - 1), x);
  Tensor h = r.defined() ? new_like(x) : Tensor();
  check(prism_add_rms_norm_fp8(at(in.x), ld(in.x), at(in.r), ld(in.r), (const float*)at(in.w), (float)eps, normalize,
                               in.x.size(0), (int)in.cols, in.code, at(y8), (float*)at(scale), at(h), launch.stream),
        "prism_add_rms_norm_fp8");
  return {y8, scale, r.defined() ? h : x};
}

// ------------------------------------------------------------------ rotary positions
// How a call turns: positions and their batch and token strides, the pairs' frequencies and axes.
struct Turn {
  Tensor positions, freqs;
  int64_t strides[2];
  int ends[2];
  bool interleaved;
  double scale;
  bool conjugate = false;  // the gradient's turn
};

// q [B, S, Hq, D], k [B, S, Hk, D] or undefined, unit column strides -> new (q, k).
std::pair<Tensor, Tensor> turn_heads(const Tensor& q, const Tensor& k, const Turn& t) {
  const Launch launch(device_of({q, k, t.positions, t.freqs}));
  const Tensor qo = new_like(q), ko = k.defined() ? new_like(k) : Tensor();
  const auto strides = [](const Tensor& x) { return x.defined() ? x.strides().data() : nullptr; };
  TORCH_CHECK_VALUE(q.size(2) < (1 << 30) && q.size(3) < (1 << 30) && (!k.defined() || k.size(2) < (1 << 30)),
                    "apply_rotary: too many heads or columns");
  check(prism_rotary(at(q), strides(q), (int)q.size(2), at(k), strides(k), k.defined() ? (int)k.size(2) : 0, q.size(0),
                     q.size(1), (int)q.size(3), 2 * (int)t.freqs.size(0), t.interleaved, at(t.positions),
                     t.positions.scalar_type() == at::kLong, t.strides, t.ends, (const double*)at(t.freqs),
                     (float)t.scale, t.conjugate, dtype_code(q, "apply_rotary"), at(qo), strides(qo), at(ko), strides(ko),
                     launch.stream),
        "prism_rotary");
  return {qo, ko};
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Optional& k_in, const Turn& t) {
    const Tensor k = or_undefined(k_in);
    ctx->save_for_backward({t.positions, t.freqs});
    ctx->saved_data["meta"] = std::vector<int64_t>{t.strides[0], t.strides[1],           t.ends[0],
                                                   t.ends[1],    (int64_t)t.interleaved, (int64_t)t.conjugate};
    ctx->saved_data["scale"] = t.scale;
    ctx->set_materialize_grads(false);
    auto [qo, ko] = turn_heads(q, k, t);
    return k.defined() ? variable_list{qo, ko} : variable_list{qo};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const auto meta = ctx->saved_data["meta"].toIntVector();
    const Turn t = {saved[0], saved[1], {meta[0], meta[1]}, {(int)meta[2], (int)meta[3]}, meta[4] != 0,
                    ctx->saved_data["scale"].toDouble(), meta[5] == 0};
    const auto unit = [](const Tensor& g) { return !g.defined() || g.stride(-1) == 1 ? g : g.contiguous(); };
    const Tensor gq = unit(grads[0]), gk = grads.size() > 1 ? unit(grads[1]) : Tensor();
    if (!gq.defined() && !gk.defined()) return {Tensor(), Tensor(), Tensor()};
    // linear, so its own gradient: a node of the graph where one is made of the gradients
    const auto turn = [&](const Tensor& a, const Tensor& b) {
      if (!at::GradMode::is_enabled()) return turn_heads(a, b, t);
      const variable_list out = apply(a, b.defined() ? Optional(b) : std::nullopt, t);
      return std::make_pair(out[0], b.defined() ? out[1] : Tensor());
    };
    if (!gq.defined()) return {Tensor(), turn(gk, Tensor()).first, Tensor()};  // k's alone
    auto [dq, dk] = turn(gq, gk);
    return {dq, dk, Tensor()};
  }
};

std::tuple<Tensor, Optional> apply_rotary(const Tensor& q_in, const Optional& k_in, const Tensor& positions_in,
                                          const Tensor& freqs, const std::string& layout,
                                          const std::optional<std::vector<int64_t>>& sections, double scale) {
  Tensor q = q_in, k = or_undefined(k_in), positions = positions_in;
  TORCH_CHECK_VALUE(layout == "interleaved" || layout == "half", "layout must be 'interleaved' or 'half', got '", layout,
                    "'");
  const int64_t dims = q.dim();
  TORCH_CHECK_VALUE(dims == 3 || dims == 4, "q must be [S, H, D] or [B, S, H, D], got ", q.sizes());
  dtype_code(q, "apply_rotary");
  const auto lead = q.sizes().slice(0, dims - 2);
  TORCH_CHECK_VALUE(!k.defined() || (k.dim() == dims && k.sizes().slice(0, dims - 2) == lead &&
                                     k.size(-1) == q.size(-1) && k.scalar_type() == q.scalar_type()),
                    "k must have q's batch, tokens, head dim and type");
  TORCH_CHECK_TYPE(freqs.scalar_type() == at::kDouble && freqs.dim() == 1,
                   "freqs must be a float64 vector (rotary_frequencies)");
  const int64_t pairs = freqs.size(0);
  TORCH_CHECK_VALUE(2 * pairs <= q.size(-1), pairs, " pairs do not fit a head of ", q.size(-1), " columns");
  TORCH_CHECK_TYPE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
                   "positions must be int32 or int64, got ", positions.scalar_type());
  Turn t;
  t.ends[0] = t.ends[1] = (int)pairs;
  std::vector<int64_t> want(lead.begin(), lead.end());
  if (sections.has_value()) {
    int64_t sum = 0;
    bool fine = sections->size() >= 1 && sections->size() <= 3;
    for (int64_t n : *sections) sum += n, fine = fine && n >= 0;
    TORCH_CHECK_VALUE(fine && sum == pairs, "sections must be 1 to 3 numbers of pairs that add up to ", pairs, ", got ",
                      *sections);
    const int64_t axes = (int64_t)sections->size();
    if (axes > 1) {
      t.ends[0] = (int)(*sections)[0], t.ends[1] = t.ends[0] + (int)(*sections)[1];
      if (positions.dim() > 0 && positions.stride(-1) != 1) positions = positions.contiguous();
    }
    want.push_back(axes);
  }
  // batch and token strides of the positions; the same row for every sequence without a batch
  const at::IntArrayRef whole(want), one = whole.slice(dims - 3);
  TORCH_CHECK_VALUE(positions.sizes() == whole || positions.sizes() == one, "positions must have shape ", whole,
                    " (the batch may be left out), got ", positions.sizes());
  const bool per_batch = dims == 4 && positions.sizes() == whole;
  t.strides[0] = per_batch ? positions.stride(0) : 0, t.strides[1] = positions.stride(per_batch ? 1 : 0);
  t.positions = positions, t.freqs = freqs.contiguous(), t.interleaved = layout == "interleaved", t.scale = scale;
  if (q.stride(-1) != 1) q = q.contiguous();
  if (k.defined() && k.stride(-1) != 1) k = k.contiguous();
  if (dims == 3) {
    q = q.unsqueeze(0);
    if (k.defined()) k = k.unsqueeze(0);
  }
  device_of({q, k, t.positions, t.freqs});
  refuse_tangents({q, k, t.freqs}, "apply_rotary");
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({freqs}), "apply_rotary has no gradient with respect to freqs");
  Tensor qo, ko;
  if (wants_grad({q, k})) {
    const variable_list out = Rotary::apply(q, k.defined() ? Optional(k) : std::nullopt, t);
    qo = out[0];
    if (k.defined()) ko = out[1];
  } else {
    std::tie(qo, ko) = turn_heads(q, k, t);
  }
  if (dims == 3) {
    qo = qo.squeeze(0);
    if (ko.defined()) ko = ko.squeeze(0);
  }
  return {qo, ko.defined() ? Optional(ko) : std::nullopt};
}

// ------------------------------------------------------------------ 8-bit projection
// t, or a contiguous copy where its 8-bit rows do not start on 16-byte boundaries.
Tensor rows16(const Tensor& t) {
  const bool fits = t.stride(1) == 1 && t.stride(0) % 16 == 0 && t.stride(0) >= t.size(1) &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

Tensor linear_fp8(const Tensor& x8, const Tensor& x_scale, const Tensor& w8, const Tensor& w_scale,
                  const Optional& bias_in) {
  const Tensor bias = or_undefined(bias_in);
  TORCH_CHECK_TYPE(x8.scalar_type() == at::kFloat8_e4m3fn && w8.scalar_type() == at::kFloat8_e4m3fn,
                   "linear_fp8 expects float8_e4m3fn operands, got ", x8.scalar_type(), " and ", w8.scalar_type());
  TORCH_CHECK_VALUE(x8.dim() >= 1 && w8.dim() == 2 && x8.size(-1) == w8.size(1) && w8.size(1) > 0, "linear_fp8: x ",
                    x8.sizes(), " and W ", w8.sizes(), " do not match");
  TORCH_CHECK_TYPE(x_scale.scalar_type() == at::kFloat && w_scale.scalar_type() == at::kFloat,
                   "linear_fp8 expects fp32 scales");
  TORCH_CHECK_VALUE(x_scale.sizes() == x8.sizes().slice(0, x8.dim() - 1) && w_scale.sizes() == w8.sizes().slice(0, 1),
                    "linear_fp8: one scale a row of x and of W");
  refuse_tangents({x8, x_scale, w8, w_scale, bias}, "linear_fp8");
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({x8, x_scale, w8, w_scale, bias}), "linear_fp8 is inference only");
  const Launch launch(device_of({x8, x_scale, w8, w_scale, bias}));
  const int64_t K = w8.size(1), N = w8.size(0);
  const Tensor x2 = x8.dim() == 2 ? x8 : x8.reshape({-1, K});
  const int64_t M = x2.size(0);
  TORCH_CHECK_VALUE(M < (1 << 30) && N < (1 << 30) && K < (1 << 30), "linear_fp8: sizes of 2^30 and more");
  const Tensor x = rows16(x2), w = rows16(w8), xs = x_scale.reshape({-1}).contiguous(), ws = w_scale.contiguous();
  const Tensor b = fp32_vector(bias, N, "bias"), out = at::empty({M, N}, x8.options().dtype(at::kBFloat16));
  check(prism_linear_fp8(at(x), x.stride(0), (const float*)at(xs), at(w), w.stride(0), (const float*)at(ws),
                         (const float*)at(b), (int)M, (int)N, (int)K, at(out), N, launch.stream),
        "prism_linear_fp8");
  if (x8.dim() == 2) return out;
  std::vector<int64_t> shape(x8.sizes().begin(), x8.sizes().end() - 1);
  shape.push_back(N);
  return out.view(shape);
}

// ------------------------------------------------------------------ attention over packed sequences
// t [rows, heads, D], or a contiguous copy where a tensor map does not take its strides.
Tensor mappable(const Tensor& t) {
  const auto fits = [&](int64_t d) { return t.size(d) <= 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0); };
  return t.stride(2) == 1 && fits(0) && fits(1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0
             ? t
             : t.clone(at::MemoryFormat::Contiguous);
}
// {row, head} strides; those of a dimension of one element are never used, but have to be fit for a map.
std::array<int64_t, 2> map_strides(const Tensor& t) {
  const int64_t head = t.size(1) > 1 ? t.stride(1) : t.size(2);
  return {t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2), head};
}

struct PackedCall {
  Tensor offsets, k_offsets;
  bool causal;
  double scale;
};

Tensor stats_like(const Tensor& q, const Tensor& k, const PackedCall& c) {
  const size_t bytes = prism_packed_attention_stats_bytes(q.size(0), c.offsets.size(0) - 1, (int)q.size(1), (int)k.size(1));
  return fp32({(int64_t)(bytes / sizeof(float))}, q);
}

// (o, lse, rest); the last two for the backward.
std::tuple<Tensor, Tensor, Tensor> packed_forward(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const PackedCall& c,
                                                  bool train) {
  const Launch launch(q_in.get_device());
  const Tensor q = mappable(q_in), k = mappable(k_in), v = mappable(v_in);
  Tensor o = new_like(q), lse = train ? stats_like(q, k, c) : Tensor(), rest = train ? new_like(q, at::kChar) : Tensor();
  const auto sq = map_strides(q), sk = map_strides(k), sv = map_strides(v);
  const int64_t bytes = train ? 0
                                 : (int64_t)prism_packed_attention_workspace_bytes(
                                       q.size(0), k.size(0), c.offsets.size(0) - 1, (int)q.size(1), (int)k.size(1), (int)q.size(2));
  const Tensor workspace = bytes > 0 ? at::empty({bytes}, q.options().dtype(at::kByte)) : Tensor();
  check(prism_packed_attention(at(q), sq.data(), at(k), sk.data(), at(v), sv.data(), at(c.offsets), at(c.k_offsets),
                               c.offsets.scalar_type() == at::kLong, c.offsets.size(0) - 1, q.size(0), k.size(0),
                               (int)q.size(1), (int)k.size(1), (int)q.size(2), c.causal, (float)c.scale,
                               dtype_code(q, "packed_attention"), at(o), (float*)at(lse), at(rest), at(workspace),
                               launch.stream),
        "prism_packed_attention");
  return {o, lse, rest};
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const PackedCall& c) {
    auto [o, lse, rest] = packed_forward(q, k, v, c, true);
    ctx->save_for_backward({q, k, v, o, lse, c.offsets, c.k_offsets, rest});
    ctx->saved_data["causal"] = c.causal;
    ctx->saved_data["scale"] = c.scale;
    ctx->set_materialize_grads(false);
    return o;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor& go_in = grads[0];
    if (!go_in.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const bool graph = at::GradMode::is_enabled();
    variable_list out(3);
    {
      const at::NoGradGuard no_grad;
      const Launch launch(saved[0].get_device());
      const Tensor q = mappable(saved[0]), k = mappable(saved[1]), v = mappable(saved[2]), go = mappable(go_in);
      const Tensor &o = saved[3], &lse = saved[4], &rest = saved[7];
      const PackedCall c = {saved[5], saved[6], ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble()};
      const bool want_q = ctx->needs_input_grad(0), want_k = ctx->needs_input_grad(1), want_v = ctx->needs_input_grad(2);
      const bool pair = want_k || want_v;
      if (q.size(0) == 0 || k.size(0) == 0) {
        out = {at::zeros_like(q), at::zeros_like(k), at::zeros_like(v)};
      } else {
        if (want_q) out[0] = new_like(q);
        if (pair) out[1] = new_like(k), out[2] = new_like(v);
        const Tensor workspace = at::empty({(int64_t)prism_packed_attention_bwd_workspace_bytes(
                                               q.size(0), k.size(0), c.offsets.size(0) - 1, (int)q.size(1), (int)k.size(1),
                                               (int)q.size(2))},
                                           q.options().dtype(at::kByte));
        const auto sq = map_strides(q), sk = map_strides(k), sv = map_strides(v), sg = map_strides(go);
        check(prism_packed_attention_bwd(at(q), sq.data(), at(k), sk.data(), at(v), sv.data(), at(o), at(rest), at(go), sg.data(),
                                         (const float*)at(lse), at(c.offsets), at(c.k_offsets),
                                         c.offsets.scalar_type() == at::kLong, c.offsets.size(0) - 1, q.size(0),
                                         k.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2), c.causal,
                                         (float)c.scale, at(workspace), at(out[0]), at(out[1]), at(out[2]),
                                         launch.stream),
              "prism_packed_attention_bwd");
      }
      if (!want_q) out[0] = Tensor();
      if (!want_k) out[1] = Tensor();
      if (!want_v) out[2] = Tensor();
    }
    if (graph) out = without_derivative(out, {go_in, saved[0], saved[1], saved[2]}, "packed_attention");
    return {out[0], out[1], out[2], Tensor()};
  }
};

void check_offsets(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64, got ",
                   t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) >= 1, name, " must hold one row number more than there are sequences, got shape ",
                    t.sizes());
}

void check_scale(const std::optional<double>& scale, const char* what) {
  TORCH_CHECK_VALUE(!scale.has_value() || (*scale > 0.0 && *scale < 1e30), what, ": scale must be positive and finite, got ",
                    scale.value_or(0.0));
}

Tensor packed_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets,
                        const Optional& k_offsets_in, bool causal, const std::optional<double>& scale) {
  constexpr const char* what = "packed_attention";
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && q.size(2) == k.size(2), what,
                    ": q must be [T, Hq, D], k and v [Tk, Hk, D], got ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_TYPE((q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) && k.scalar_type() == q.scalar_type() &&
                       v.scalar_type() == q.scalar_type(),
                   what, " expects q, k and v all bf16 or all fp16, got ", q.scalar_type(), ", ", k.scalar_type(), " and ",
                   v.scalar_type());
  TORCH_CHECK_VALUE(q.size(2) == 64 || q.size(2) == 128, what, ": head dim ", q.size(2), " not supported (64, 128)");
  TORCH_CHECK_VALUE(k.size(1) >= 1 && q.size(1) >= 1 && q.size(1) % k.size(1) == 0 && q.size(1) / k.size(1) <= 128, what, ": ",
                    q.size(1), " query heads do not share ", k.size(1), " key heads in equal groups of up to 128");
  TORCH_CHECK_VALUE(q.size(0) < (1 << 30) && k.size(0) < (1 << 30) && q.size(1) < (1 << 30), what, ": sizes of 2^30 and more");
  check_offsets(offsets, "offsets");
  const bool own_keys = k_offsets_in.has_value();
  if (own_keys) {
    check_offsets(*k_offsets_in, "k_offsets");
    TORCH_CHECK_VALUE(k_offsets_in->sizes() == offsets.sizes() && k_offsets_in->scalar_type() == offsets.scalar_type(),
                      "k_offsets must have the shape and type of offsets");
  } else {
    TORCH_CHECK_VALUE(k.size(0) == q.size(0), what, ": without k_offsets k must have q's rows, got ", k.size(0), " and ",
                      q.size(0));
  }
  check_scale(scale, what);
  refuse_tangents({q, k, v}, what);
  PackedCall c = {offsets.contiguous(), Tensor(), causal, scale.value_or(1.0 / std::sqrt((double)q.size(2)))};
  c.k_offsets = own_keys ? k_offsets_in->contiguous() : c.offsets;
  device_of({q, k, v, c.offsets, c.k_offsets});
  if (wants_grad({q, k, v})) {
    // fp16 holds p (dp - delta) down to 6e-8 only: gradients of long rows would be lost without a sign
    TORCH_CHECK_NOT_IMPLEMENTED(q.scalar_type() == at::kBFloat16, what, " has gradients in bf16 only");
    return PackedAttention::apply(q, k, v, c);
  }
  return std::get<0>(packed_forward(q, k, v, c, false));
}

// ------------------------------------------------------------------ paged cache
struct PagedCache {
  std::array<int64_t, 3> k_strides, v_strides;
  int pages, page_size;
};

// The caches [pages, page_size, Hk, D] and what addresses them: in place, so nothing here is copied into shape.
PagedCache check_cache(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths, const char* what) {
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && k.size(1) >= 1 && k.size(2) >= 1, what,
                    ": the caches must both be [pages, page_size, Hk, D], got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_TYPE((k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf) && v.scalar_type() == k.scalar_type(),
                   what, " expects caches both bf16 or both fp16, got ", k.scalar_type(), " and ", v.scalar_type());
  TORCH_CHECK_VALUE(k.stride(3) == 1 && v.stride(3) == 1, what, ": the caches' columns must be contiguous");
  TORCH_CHECK_TYPE(table.scalar_type() == at::kInt && lengths.scalar_type() == at::kInt, what,
                   " expects an int32 page_table and int32 lengths, got ", table.scalar_type(), " and ", lengths.scalar_type());
  TORCH_CHECK_VALUE(table.dim() == 2 && lengths.dim() == 1 && table.size(0) == lengths.size(0), what,
                    ": page_table must be [sequences, pages of each], lengths [sequences], got ", table.sizes(), " and ",
                    lengths.sizes());
  TORCH_CHECK_VALUE(k.size(0) < (1 << 30) && k.size(1) < (1 << 30) && k.size(2) < (1 << 20) && table.size(0) < (1 << 28) &&
                        table.size(1) * k.size(1) < (int64_t(1) << 31) - 64,
                    what, ": too many pages, heads, sequences or keys of a sequence");
  PagedCache c;
  for (int d = 0; d < 3; ++d) c.k_strides[d] = k.stride(d), c.v_strides[d] = v.stride(d);
  c.pages = (int)k.size(0), c.page_size = (int)k.size(1);
  return c;
}
// Whether elements of t share memory: by growing strides, a dimension has to step over all that lies within.
bool overlaps(const Tensor& t) {
  if (t.numel() == 0) return false;
  std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
  std::sort(dims.begin(), dims.end());
  int64_t extent = 1;
  for (const auto& [stride, size] : dims) {
    if (stride < extent) return true;
    extent += (size - 1) * stride;
  }
  return false;
}
Tensor unit_columns(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

// t [B, H, D] (one token a sequence) or [B, n, H, D] as rows [tokens, H, D], or [T, H, D] with offsets.
Tensor token_rows(const Tensor& t) { return unit_columns(t.dim() == 4 ? t.flatten(0, 1) : t); }

Optional append_paged(const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache, const Tensor& v_cache,
                      const Tensor& table_in, const Tensor& lengths_in, const Optional& offsets_in, const Optional& q_in,
                      const Optional& freqs_in, const std::string& layout, double scale) {
  constexpr const char* what = "append_paged";
  const Tensor q_given = or_undefined(q_in), offsets = or_undefined(offsets_in), freqs = or_undefined(freqs_in);
  TORCH_CHECK_VALUE(layout == "interleaved" || layout == "half", "layout must be 'interleaved' or 'half', got '", layout, "'");
  const PagedCache c = check_cache(k_cache, v_cache, table_in, lengths_in, what);
  TORCH_CHECK_VALUE(!overlaps(k_cache) && !overlaps(v_cache) && (k_cache.numel() == 0 || k_cache.data_ptr() != v_cache.data_ptr()),
                    what, ": places of the caches share memory");
  const int64_t dims = k_in.dim(), batch = lengths_in.size(0), D = k_cache.size(3);
  TORCH_CHECK_VALUE((dims == 3 || (dims == 4 && !offsets.defined())) && v_in.sizes() == k_in.sizes() && k_in.size(-1) == D &&
                        k_in.size(-2) == k_cache.size(2),
                    what, ": k and v must be [B, Hk, D] or [B, n, Hk, D], or [T, Hk, D] with offsets, of the caches' heads, got ",
                    k_in.sizes(), " and ", v_in.sizes(), " for caches ", k_cache.sizes());
  TORCH_CHECK_TYPE(k_in.scalar_type() == k_cache.scalar_type() && v_in.scalar_type() == k_cache.scalar_type(), what,
                   ": k and v must have the caches' type");
  TORCH_CHECK_VALUE(D <= 256, what, ": head dims up to 256, got ", D);
  if (q_given.defined()) {
    TORCH_CHECK_VALUE(q_given.dim() == dims && q_given.sizes().slice(0, dims - 2) == k_in.sizes().slice(0, dims - 2) &&
                          q_given.size(-1) == D && q_given.scalar_type() == k_cache.scalar_type(),
                      what, ": q must have k's tokens, head dim and type, got ", q_given.sizes());
    TORCH_CHECK_VALUE(q_given.size(-2) < (1 << 20), what, ": too many heads");
  }
  if (offsets.defined()) {
    check_offsets(offsets, "offsets");
    TORCH_CHECK_VALUE(offsets.size(0) == batch + 1, what, ": offsets must hold one row number more than there are sequences, got ",
                      offsets.size(0), " for ", batch);
  } else {
    TORCH_CHECK_VALUE(k_in.size(0) == batch, what, ": ", k_in.size(0), " sequences of k, ", batch, " of lengths");
  }
  if (freqs.defined()) {
    TORCH_CHECK_TYPE(freqs.scalar_type() == at::kDouble && freqs.dim() == 1, "freqs must be a float64 vector (rotary_frequencies)");
    TORCH_CHECK_VALUE(2 * freqs.size(0) <= D, freqs.size(0), " pairs do not fit a head of ", D, " columns");
  }
  refuse_tangents({k_in, v_in, q_given, k_cache, v_cache, freqs}, what);
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({k_in, v_in, q_given, k_cache, v_cache, freqs}), what, " is inference only");
  const Launch launch(device_of({k_in, v_in, k_cache, v_cache, table_in, lengths_in, offsets, q_given, freqs}));
  const Tensor k = token_rows(k_in), v = token_rows(v_in), q = q_given.defined() ? token_rows(q_given) : Tensor();
  const Tensor table = unit_columns(table_in), lengths = lengths_in.contiguous(), at_rows = offsets.defined() ? offsets.contiguous() : offsets;
  const Tensor f = freqs.defined() ? freqs.contiguous() : freqs;
  TORCH_CHECK_VALUE(k.size(0) < (1 << 30), what, ": too many tokens");
  const Tensor out = q.defined() ? new_like(q_given) : Tensor();
  const auto strides = [](const Tensor& t) { return t.defined() ? t.strides().data() : nullptr; };
  check(prism_append_paged(at(q), strides(q), q.defined() ? (int)q.size(1) : 0, at(k), strides(k), at(v), strides(v),
                           (int)k.size(1), k.size(0), (int)D, at(at_rows), at_rows.defined() && at_rows.scalar_type() == at::kLong,
                           (int)batch, at(k_cache), c.k_strides.data(), at(v_cache), c.v_strides.data(), c.pages, c.page_size,
                           (const int*)at(table), table.stride(0), (int)table.size(1), (const int*)at(lengths),
                           f.defined() ? 2 * (int)f.size(0) : 0, layout == "interleaved", (const double*)at(f), (float)scale,
                           dtype_code(k, what), at(out), launch.stream),
        "prism_append_paged");
  for (const Tensor& t : {k_cache, v_cache})
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return out.defined() ? Optional(out) : std::nullopt;
}

Tensor paged_attention(const Tensor& q_in, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table_in,
                       const Tensor& lengths_in, const std::optional<double>& scale) {
  constexpr const char* what = "paged_attention";
  const PagedCache c = check_cache(k_cache, v_cache, table_in, lengths_in, what);
  const int64_t D = k_cache.size(3), Hk = k_cache.size(2);
  TORCH_CHECK_VALUE((q_in.dim() == 3 || q_in.dim() == 4) && q_in.size(0) == lengths_in.size(0) && q_in.size(-1) == D, what,
                    ": q must be [B, Hq, D] or [B, n, Hq, D] with the sequences of lengths and the caches' head dim, got ",
                    q_in.sizes());
  TORCH_CHECK_TYPE(q_in.scalar_type() == k_cache.scalar_type(), what, ": q must have the caches' type, got ", q_in.scalar_type());
  TORCH_CHECK_VALUE(D == 64 || D == 128, what, ": head dim ", D, " not supported (64, 128)");
  TORCH_CHECK_VALUE(q_in.size(-2) >= 1 && q_in.size(-2) % Hk == 0, what, ": ", q_in.size(-2), " query heads do not share ", Hk,
                    " key heads in equal groups");
  TORCH_CHECK_VALUE(q_in.numel() / D < (1 << 28), what, ": too many rows");
  check_scale(scale, what);
  refuse_tangents({q_in, k_cache, v_cache}, what);
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({q_in, k_cache, v_cache}), what, " is inference only");
  const auto fits = [](const Tensor& t) {
    const auto whole = [&](int64_t d) { return t.size(d) <= 1 || t.stride(d) % 8 == 0; };
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && whole(0) && whole(1) && whole(2);
  };
  const Launch launch(device_of({q_in, k_cache, v_cache, table_in, lengths_in}));
  TORCH_CHECK_VALUE(fits(k_cache) && fits(v_cache), what, ": the caches' rows must start on 16 bytes");
  Tensor q = q_in.dim() == 4 ? q_in : q_in.unsqueeze(1);
  if (q.stride(3) != 1 || (q.stride(0) | q.stride(1) | q.stride(2)) % 2 != 0 || reinterpret_cast<uintptr_t>(q.data_ptr()) % 4 != 0)
    q = q.clone(at::MemoryFormat::Contiguous);
  const Tensor table = unit_columns(table_in), lengths = lengths_in.contiguous(), out = new_like(q_in);
  const int64_t bytes = (int64_t)prism_paged_attention_workspace_bytes((int)D, c.page_size, (int)table.size(1));
  const Tensor workspace = bytes > 0 ? at::empty({bytes}, q_in.options().dtype(at::kByte)) : Tensor();
  check(prism_paged_attention(at(q), q.strides().data(), (int)q.size(0), (int)q.size(1), (int)q.size(2), (int)Hk, (int)D,
                              at(k_cache), c.k_strides.data(), at(v_cache), c.v_strides.data(), c.pages, c.page_size,
                              (const int*)at(table), table.stride(0), (int)table.size(1), (const int*)at(lengths),
                              (float)scale.value_or(1.0 / std::sqrt((double)D)), dtype_code(q, what), at(out), at(workspace),
                              launch.stream),
        "prism_paged_attention");
  return out;
}

// ------------------------------------------------------------------ clipping
// Over lists of contiguous tensors (outs may be grads): the norm, 0-dim fp32.  None where the lists
// are not of contiguous CUDA tensors of the three types on one device, alike in type and number of
// elements; nothing has happened then.
Optional clip_grad_norm(const std::vector<Tensor>& grads, const std::vector<Tensor>& outs, double max_norm) {
  const size_t n = grads.size();
  if (n == 0 || outs.size() != n) return std::nullopt;
  std::vector<const void*> from(n);
  std::vector<void*> to(n);
  std::vector<int64_t> sizes(n);
  std::vector<int> codes(n);
  const auto plain = [](const Tensor& t) {
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous();
  };
  for (size_t i = 0; i < n; ++i) {
    const Tensor &g = grads[i], &o = outs[i];
    if (!plain(g) || !plain(o) || g.get_device() != grads[0].get_device() || o.get_device() != g.get_device() ||
        o.scalar_type() != g.scalar_type() || o.numel() != g.numel() || (codes[i] = dtype_code_or(g, -1)) < 0)
      return std::nullopt;
    from[i] = g.data_ptr(), to[i] = o.data_ptr(), sizes[i] = g.numel();
  }
  const Launch launch(grads[0].get_device());
  const auto options = grads[0].options().requires_grad(false);
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const Tensor workspace =
      at::empty({(int64_t)prism_clip_grad_norm_workspace_bytes((int64_t)n)}, options.dtype(at::kByte));
  check(prism_clip_grad_norm(from.data(), to.data(), sizes.data(), codes.data(), (int64_t)n, (float)max_norm,
                             at(workspace), (float*)at(norm), launch.stream),
        "prism_clip_grad_norm");
  // autograd sees that its saved tensors changed; an infinite max_norm writes nothing in place
  const bool measure = std::isinf((float)max_norm);
  for (size_t i = 0; i < n; ++i)
    if (!outs[i].is_inference() && !(measure && from[i] == to[i])) outs[i].unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

PYBIND11_MODULE(prism_torch_ops, m) {
  static PyObject* prism_error = nullptr;  // prism_b200._lib.PrismError
  m.attr("abi_version") = PRISM_ABI_VERSION;
  m.def("set_error", [](py::object type) { prism_error = type.inc_ref().ptr(); });
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const PrismFailure& e) {
      PyErr_SetString(prism_error ? prism_error : PyExc_RuntimeError, e.what());
    }
  });
  const auto free = py::call_guard<py::gil_scoped_release>();
  m.def("add_rms_norm", &add_rms_norm, free);
  m.def("add_rms_norm_fp8", &add_rms_norm_fp8, free);
  m.def("apply_rotary", &apply_rotary, free);
  m.def("linear_fp8", &linear_fp8, free);
  m.def("clip_grad_norm", &clip_grad_norm, free);
  m.def("packed_attention", &packed_attention, free);
  m.def("append_paged", &append_paged, free);
  m.def("paged_attention", &paged_attention, free);
}
