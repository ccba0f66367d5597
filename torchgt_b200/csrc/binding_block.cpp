// Autograd nodes of the operators around the attention of a pre-norm block: the root-mean-square norm
// (torchgt_b200/rms_norm.py), the learned relative position bias (torchgt_b200/position_bias.py) and the gated feed-forward
// block (torchgt_b200/gated_ffn.py).
#include "binding.h"

#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

namespace tgt_host {
namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// a CUDA tensor of the kernels' types, not a functorch wrapper, a dual number, a fake or a lazily negated view
bool plain(const at::Tensor& t, const at::Device& device, at::ScalarType type) {
  return t.defined() && !at::isTensorSubclassLike(t) && t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == type &&
         t.device() == device && !torch::autograd::isFwGradDefined(t) && !t.is_neg();
}
bool kernel_type(at::ScalarType type) { return type == at::kFloat || type == at::kBFloat16; }
int type_code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? TGT_F32 : TGT_BF16; }

// A backward pass is the formula as operations, not kernels: it is itself differentiated (create_graph), there are many gradients at once
// (is_grads_batched), or they carry tangents, which would be lost.
bool as_operations(const at::Tensor& grad) {
  return at::GradMode::is_enabled() || (grad.defined() && (at::isTensorSubclassLike(grad) || torch::autograd::isFwGradDefined(grad)));
}

// An uninitialised tensor next to `like`, straight from the allocator's function: the small calls are bound by the host, and on its
// way through the dispatcher at::empty takes twice the time.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}
at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor& like) { return fresh(sizes, like.scalar_type(), like); }
at::Tensor scratch_of(size_t bytes, const at::Tensor& like) { return fresh({int64_t(bytes < 16 ? 16 : bytes)}, at::kByte, like); }

// ---- root-mean-square norm, with the residual addition in front of it -----------------------------------------------
// Outputs: the normalised rows and, with a residual, x + residual.
struct RmsNormRowsBackward : public torch::autograd::Node {
  SavedVariable normalised, weight, rstd;   // the norm's input: x, or the output x + residual
  SavedVariable rest;                       // of a bf16 sum: what its rounding took
  bool with_residual = false;
  double eps = 0;

  variable_list recorded(const at::Tensor& dy_, const at::Tensor& ds, const at::Tensor& v_, const at::Tensor& w_,
                         const at::Tensor& rest_) {
    const at::Tensor w = w_.to(at::kFloat);
    at::Tensor v = v_.to(at::kFloat);
    if (rest_.defined()) {   // the sum before it was rounded, as the kernel takes it, with the rounded sum's derivative
      const at::Tensor rounded = v.detach(), whole = (rounded.view(at::kInt) + rest_.to(at::kInt) * 256).view(at::kFloat);
      v = whole + at::where(rounded.isfinite(), v - rounded, at::zeros_like(rounded));
    }
    const at::Tensor r = (v * v).mean(-1, true).add(eps).rsqrt(), u = v * r;
    at::Tensor dx, dw;
    if (dy_.defined()) {
      const at::Tensor dy = dy_.to(at::kFloat), g = dy * w;
      dx = r * (g - u * (g * u).mean(-1, true));
      dw = (dy * u).reshape({-1, w.numel()}).sum(0).to(w_.scalar_type());
    }
    if (ds.defined()) dx = dx.defined() ? dx + ds.to(at::kFloat) : ds;
    dx = dx.to(v_.scalar_type());
    return {dx, with_residual ? dx : at::Tensor(), dw};
  }

  variable_list apply(variable_list&& grads) override {
    return reporting([&] { return backward(grads); });
  }
  variable_list backward(const variable_list& grads) {
    const at::Tensor ds = with_residual ? grads[1] : at::Tensor();
    if (!grads[0].defined()) return {ds, ds, at::Tensor()};              // only x + residual was used, or nothing
    const at::Tensor v = with_residual ? normalised.unpack(shared_from_this()) : normalised.unpack();
    const at::Tensor w = weight.unpack(), rstd_ = rstd.unpack(), rest_ = rest.unpack();
    if (as_operations(grads[0]) || as_operations(ds))
      return recorded(grads[0], ds, v, w, rest_);
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(v.device());
    const at::Tensor dy = packed(grads[0]), vc = v.contiguous(), wc = w.contiguous();
    const at::Tensor dsum = ds.defined() ? packed(ds) : ds;
    const int64_t hidden = w.numel(), rows = v.numel() / hidden;
    const at::Tensor dx = fresh(v.sizes(), dy), dw = fresh(w.sizes(), dy);
    size_t bytes = 0;
    check(tgt_rms_norm_bwd_scratch_bytes(rows, int(hidden), type_code(v), &bytes));
    const at::Tensor scratch = scratch_of(bytes, dy);
    check(tgt_rms_norm_bwd(ptr(dy), ptr(dsum), ptr(vc), ptr(rest_), ptr(wc), fptr(rstd_), rows, int(hidden), type_code(v), ptr(dx), ptr(dw),
                           scratch.data_ptr(), scratch.numel(), stream_of(dy)));
    return {dx, with_residual ? dx : at::Tensor(), dw};
  }
  std::string name() const override { return "RmsNormRowsBackward"; }
  void release_variables() override {
    normalised.reset_data();
    weight.reset_data();
    rstd.reset_data();
    rest.reset_data();
  }
};

bool rms_norm_covers(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& residual) {
  constexpr int64_t kMostHidden = 16384;
  if (!x.defined() || at::isTensorSubclassLike(x) || !kernel_type(x.scalar_type())) return false;
  if (!plain(x, x.device(), x.scalar_type()) || !plain(w, x.device(), x.scalar_type())) return false;
  if (w.dim() != 1 || x.dim() < 1 || x.size(-1) != w.numel() || w.numel() < 1 || w.numel() > kMostHidden) return false;
  return !residual.has_value() || (plain(*residual, x.device(), x.scalar_type()) && residual->sizes() == x.sizes());
}

// {norm of x (+ residual), x + residual or nothing}; the sum is left out when nobody wants it.  Nothing, and nothing launched, for
// tensors that the kernels do not cover.
std::optional<std::pair<at::Tensor, std::optional<at::Tensor>>> add_rms_norm(const at::Tensor& x,
                                                                             const std::optional<at::Tensor>& residual_in,
                                                                             const at::Tensor& w, double eps, bool want_sum) {
  if (!rms_norm_covers(x, w, residual_in)) return std::nullopt;
  const at::Tensor residual = residual_in.value_or(at::Tensor());
  const c10::cuda::CUDAGuard guard(x.device());
  const bool record = torch::autograd::compute_requires_grad(x, residual, w);
  const int64_t hidden = w.numel(), rows = x.numel() / hidden;
  at::Tensor y, sum, rest, rstd;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor xc = x.contiguous(), wc = w.contiguous(), rc = residual.defined() ? residual.contiguous() : residual;
    y = fresh(x.sizes(), x);
    if (residual.defined() && (want_sum || record)) sum = fresh(x.sizes(), x);
    if (record && sum.defined() && x.scalar_type() == at::kBFloat16) rest = fresh(x.sizes(), at::kChar, x);
    if (record) rstd = fresh({rows}, at::kFloat, x);
    check(tgt_rms_norm_fwd(ptr(xc), ptr(rc), ptr(wc), float(eps), rows, int(hidden), type_code(x), ptr(sum), ptr(rest), ptr(y),
                           record ? fptr(rstd) : nullptr, stream_of(x)));
  }
  if (record) {
    auto node = std::shared_ptr<RmsNormRowsBackward>(new RmsNormRowsBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, residual, w));
    node->with_residual = residual.defined();
    node->eps = eps;
    node->rstd = SavedVariable(rstd, false);
    node->rest = SavedVariable(rest, false);
    node->weight = SavedVariable(w, false);
    if (residual.defined()) {
      torch::autograd::set_history(variable_list{y, sum}, node);
      node->normalised = SavedVariable(sum, true);
    } else {
      torch::autograd::set_history(y, node);
      node->normalised = SavedVariable(x, false);
    }
  }
  return std::make_pair(y, sum.defined() ? std::optional<at::Tensor>(sum) : std::nullopt);
}

// {values, scales, x + residual or nothing}; no gradients
std::tuple<at::Tensor, at::Tensor, std::optional<at::Tensor>> rms_norm_e4m3(const at::Tensor& x, const at::Tensor& w, double eps,
                                                                            const std::optional<at::Tensor>& residual_in) {
  TORCH_CHECK(rms_norm_covers(x, w, residual_in), "rms_norm_quantized: tensors that the kernels do not cover");
  const at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t hidden = w.numel(), rows = x.numel() / hidden;
  const at::Tensor xc = x.contiguous(), wc = w.contiguous();
  at::Tensor rc, sum;
  if (residual_in.has_value()) {
    rc = residual_in->contiguous();
    sum = fresh(x.sizes(), x);
  }
  const at::Tensor values = fresh(x.sizes(), at::kFloat8_e4m3fn, x);
  const at::Tensor scales = fresh(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
  check(tgt_rms_norm_e4m3(ptr(xc), ptr(rc), ptr(wc), float(eps), rows, int(hidden), type_code(x), ptr(sum), ptr(values),
                          fptr(scales), stream_of(x)));
  return {values, scales, sum.defined() ? std::optional<at::Tensor>(sum) : std::nullopt};
}

// ---- learned relative position bias ------------------------------------------------------------------------------------
struct EdgePositionBiasBackward : public torch::autograd::Node {
  SavedVariable buckets;      // int16, -1: an edge without one
  int64_t n_buckets = 0;

  variable_list apply(variable_list&& grads) override {
    return reporting([&] { return backward(grads); });
  }
  variable_list backward(const variable_list& grads) {
    if (!grads[0].defined()) return variable_list(1);
    const at::Tensor of = buckets.unpack();
    const int64_t edges = of.numel(), heads = grads[0].size(-1);
    if (as_operations(grads[0])) {
      const at::Tensor known = of.ge(0).unsqueeze(-1), d = at::where(known, grads[0], at::zeros_like(grads[0]));
      return {at::zeros({n_buckets, heads}, grads[0].options()).index_add(0, of.clamp_min(0).to(at::kLong), d)};
    }
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(of.device());
    const at::Tensor d = packed(grads[0]), dtable = fresh({n_buckets, heads}, d);
    size_t bytes = 0;
    check(tgt_edge_position_bias_grad_scratch_bytes(edges, int(n_buckets), int(heads), &bytes));
    const at::Tensor scratch = scratch_of(bytes, d);
    check(tgt_edge_position_bias_grad(fptr(d), static_cast<const uint16_t*>(ptr(of)), edges, int(n_buckets), int(heads),
                                      fptr(dtable), scratch.data_ptr(), scratch.numel(), stream_of(d)));
    return {dtable};
  }
  std::string name() const override { return "EdgePositionBiasBackward"; }
  void release_variables() override { buckets.reset_data(); }
};

// The caller has checked types, shapes and the borders; nothing, and nothing launched, for what is left: wrappers of torch.func, dual
// numbers and the like.
std::optional<at::Tensor> edge_position_bias(const at::Tensor& table, const at::Tensor& edge_index, const std::optional<at::Tensor>& positions,
                              const std::vector<int32_t>& borders, bool both_ways) {
  auto ids = [&](const at::Tensor& t) { return plain(t, table.device(), at::kLong) || plain(t, table.device(), at::kInt); };
  if (!table.defined() || !plain(table, table.device(), at::kFloat) || !ids(edge_index) || (positions.has_value() && !ids(*positions)))
    return std::nullopt;
  TORCH_CHECK(table.dim() == 2 && edge_index.dim() == 2 && edge_index.size(0) == 2 && (!positions.has_value() || positions->dim() == 1) &&
                  table.size(0) == int64_t(borders.size() + 1) * (both_ways ? 2 : 1),
              "edge_position_bias: shapes that do not fit one another");
  const at::Device device = table.device();
  const c10::cuda::CUDAGuard guard(device);
  const int64_t edges = edge_index.size(1), heads = table.size(1);
  const bool record = torch::autograd::compute_requires_grad(table);
  at::Tensor bias, buckets;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor tc = table.contiguous(), ec = edge_index.contiguous();
    const at::Tensor pc = positions.has_value() ? positions->contiguous() : at::Tensor();
    bias = fresh({edges, heads}, table);
    if (record) buckets = fresh({edges}, at::kShort, table);
    // no nodes: every id is outside, which takes a pointer to tell
    const void* where = pc.defined() ? (pc.numel() > 0 ? pc.data_ptr() : static_cast<const void*>(tc.data_ptr())) : nullptr;
    check(tgt_edge_position_bias(ptr(ec), edges, ec.scalar_type() == at::kLong, where, pc.defined() ? pc.numel() : 0,
                                 pc.defined() && pc.scalar_type() == at::kLong, borders.data(), int(borders.size()), both_ways,
                                 fptr(tc), int(heads), fptr(bias), static_cast<uint16_t*>(ptr(buckets)), stream_of(table)));
  }
  if (record) {
    auto node = std::shared_ptr<EdgePositionBiasBackward>(new EdgePositionBiasBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(table));
    node->buckets = SavedVariable(buckets, false);
    node->n_buckets = table.size(0);
    torch::autograd::set_history(bias, node);
  }
  return bias;
}

// ---- gated feed-forward block -------------------------------------------------------------------------------------------
// act(x w_gate^T) * (x w_up^T) times w_down^T, plus a residual.
int activation_code(const std::string& name) {
  TORCH_CHECK(name == "silu" || name == "gelu" || name == "relu", "gated_feed_forward knows silu, gelu and relu, not ", name);
  return name == "silu" ? TGT_ACT_SILU : name == "gelu" ? TGT_ACT_GELU : TGT_ACT_RELU;
}

// contiguous, and copied when it is a view that starts off a 16-byte boundary (the kernels move 16 bytes at a time)
at::Tensor kernel_ready(const at::Tensor& t) {
  const at::Tensor c = packed(t);
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) == 0 ? c : c.clone();
}

// Rows without gradients for which the kernels of gated_rows.cu are ahead of tiles of 128 rows.  us, weights not in the L2: 2,048 x
// 5,632 x 2,048, one row 14.5 / 35, 16 rows 17 / 29, 32 rows 22 / 24; 768 x 2,048 x 768, 32 rows 9 / 14; 4,096 x 11,008 x 4,096, one row
// 47 / 74, 32 rows 55 / 58; behind with 32 rows of 512 x 2,048 x 16,384 29 / 20, 4,096 x 14,336 x 4,096 82 / 70.  16 rows: 64 x 128 x 64
// 3.8 / 7.0, 768 x 2,048 x 768 7.5 / 14.6, 512 x 2,048 x 16,384 23 / 30, 1,024 x 4,096 x 16,384 37 / 40, 8,192 x 28,672 x 8,192 232 / 237,
// alike at 4,096 x 14,336 x 4,096 (70 / 69) and 5,120 x 13,824 x 5,120 (90 / 88), behind at 8,192 x 8,192 x 8,192 (86 / 78) and with
// middles of 64 outputs and more: 512 x 65,536 x 512 73 / 69, 128 x 65,536 x 128 65 / 47 (32 rows 82 / 47).
bool few_rows(int64_t rows, int64_t in, int64_t mid, int64_t out) {
  return rows <= 16 || (rows <= 32 && out <= 4096 && in * mid <= int64_t(48) << 20);
}

struct GatedFeedForwardBackward : public torch::autograd::Node {
  SavedVariable x, w_gate, w_up, w_down, hidden, gate, up, low;   // low: of bf16 (tgt_gated_hidden)
  int act = TGT_ACT_SILU;
  bool with_residual = false;

  variable_list apply(variable_list&& grads) override {
    return reporting([&] { return backward(grads); });
  }
  variable_list recorded(const at::Tensor& dy, const at::Tensor& x_, const at::Tensor& wg, const at::Tensor& wu,
                         const at::Tensor& wd) {
    const at::Tensor g = at::matmul(x_, wg.t()), u = at::matmul(x_, wu.t()), dh = at::matmul(dy, wd);
    at::Tensor a, slope;
    if (act == TGT_ACT_RELU) {
      a = at::relu(g);
      slope = (g > 0).to(g.scalar_type());
    } else if (act == TGT_ACT_GELU) {
      a = at::gelu(g);
      slope = at::gelu_backward(at::ones_like(g), g);
    } else {
      const at::Tensor s = at::sigmoid(g);
      a = g * s;
      slope = s * (1 + g * (1 - s));
    }
    auto flat = [](const at::Tensor& t) { return t.reshape({-1, t.size(-1)}); };
    const at::Tensor dg = dh * u * slope, du = dh * a;
    return {at::matmul(dg, wg) + at::matmul(du, wu), at::matmul(flat(dg).t(), flat(x_)), at::matmul(flat(du).t(), flat(x_)),
            at::matmul(flat(dy).t(), flat(a * u)), with_residual ? dy : at::Tensor()};
  }
  variable_list backward(const variable_list& grads) {
    variable_list result(5);
    if (!grads[0].defined()) return result;
    const at::Tensor x_ = x.unpack(), wg = w_gate.unpack(), wu = w_up.unpack(), wd = w_down.unpack();
    if (as_operations(grads[0])) return recorded(grads[0], x_, wg, wu, wd);
    if (with_residual) result[4] = grads[0];
    const at::Tensor h = hidden.unpack(), g = gate.unpack(), u = up.unpack(), l = low.unpack();
    const c10::cuda::CUDAGuard guard(x_.device());
    const at::AutoDispatchBelowADInplaceOrView below;
    const int64_t in = wg.size(1), mid = wg.size(0), out = wd.size(0), rows = x_.numel() / in;
    const int type = type_code(x_);
    const at::Tensor dy = kernel_ready(grads[0]);
    void* const stream = stream_of(x_);
    auto weight_gradients = [&](const std::vector<at::Tensor>& d, const at::Tensor& of, int64_t n, int64_t k, at::Tensor* dw) {
      const void* from[2];
      void* to[2];
      for (size_t i = 0; i < d.size(); ++i) {
        dw[i] = fresh({n, k}, x_);
        from[i] = ptr(d[i]);
        to[i] = dw[i].data_ptr();
      }
      size_t bytes = 0;
      check(tgt_gated_weight_grad_scratch_bytes(int(d.size()), rows, int(n), int(k), type, &bytes));
      const at::Tensor scratch = scratch_of(bytes, x_);
      check(tgt_gated_weight_grad(from, ptr(of), int(d.size()), rows, int(n), int(k), type, to, scratch.data_ptr(), scratch.numel(),
                                  stream));
    };
    if (task_should_compute_output(3)) weight_gradients({dy}, h, out, mid, &result[3]);
    const bool first = task_should_compute_output(1) || task_should_compute_output(2);
    if (!first && !task_should_compute_output(0)) return result;
    const at::Tensor dg = fresh(g.sizes(), g), du = fresh(u.sizes(), u);
    const at::Tensor wdc = kernel_ready(wd);
    check(tgt_gated_hidden_grad(ptr(dy), ptr(wdc), ptr(g), ptr(u), ptr(l), rows, int(out), int(mid), act, type, ptr(dg), ptr(du), stream));
    if (first) weight_gradients({dg, du}, kernel_ready(x_), mid, in, &result[1]);
    if (task_should_compute_output(0)) {
      const at::Tensor wgc = kernel_ready(wg), wuc = kernel_ready(wu);
      result[0] = fresh(x_.sizes(), x_);
      check(tgt_gated_input_grad(ptr(dg), ptr(du), ptr(wgc), ptr(wuc), rows, int(mid), int(in), type, ptr(result[0]), stream));
    }
    return result;
  }
  std::string name() const override { return "GatedFeedForwardBackward"; }
  void release_variables() override {
    for (SavedVariable* v : {&x, &w_gate, &w_up, &w_down, &hidden, &gate, &up, &low}) v->reset_data();
  }
};

bool gated_feed_forward_covers(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd,
                               const std::optional<at::Tensor>& residual) {
  if (!x.defined() || at::isTensorSubclassLike(x) || !kernel_type(x.scalar_type()) || x.dim() < 1) return false;
  for (const at::Tensor* t : {&x, &wg, &wu, &wd})
    if (!plain(*t, x.device(), x.scalar_type())) return false;
  if (wg.dim() != 2 || wd.dim() != 2 || wu.sizes() != wg.sizes() || wd.size(1) != wg.size(0) || x.size(-1) != wg.size(1)) return false;
  const int64_t in = wg.size(1), mid = wg.size(0), out = wd.size(0);
  if (in < 1 || mid < 1 || out < 1) return false;
  if (x.scalar_type() == at::kFloat) {
    if (in % 64 != 0 || mid % 64 != 0 || out % 4 != 0 || in > 1024 || mid > 1024 || out > 1024) return false;
  } else if (in % 8 != 0 || mid % 8 != 0 || out % 8 != 0 || in > 65536 || mid > 65536 || out > 65536 ||
             x.numel() / in > (int64_t(1) << 30)) {
    return false;
  }
  if (!residual.has_value()) return true;
  auto sizes = x.sizes().vec();
  sizes.back() = out;
  return plain(*residual, x.device(), x.scalar_type()) && residual->sizes() == at::IntArrayRef(sizes);
}

// Nothing, and nothing launched, for tensors that the kernels do not cover.
std::optional<at::Tensor> gated_feed_forward(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd,
                                             const std::string& activation, const std::optional<at::Tensor>& residual_in) {
  const int act = activation_code(activation);
  if (!gated_feed_forward_covers(x, wg, wu, wd, residual_in)) return std::nullopt;
  const at::Tensor residual = residual_in.value_or(at::Tensor());
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t in = wg.size(1), mid = wg.size(0), out = wd.size(0), rows = x.numel() / in;
  const int type = type_code(x);
  const bool record = torch::autograd::compute_requires_grad(x, wg, wu, wd, residual);
  at::Tensor y, h, g, u, l;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor xc = kernel_ready(x), wgc = kernel_ready(wg), wuc = kernel_ready(wu), wdc = kernel_ready(wd),
                     rc = residual.defined() ? kernel_ready(residual) : residual;
    auto sizes = x.sizes().vec();
    sizes.back() = mid;
    h = fresh(sizes, x);
    if (record || type == TGT_F32) {
      g = fresh(sizes, x);
      u = fresh(sizes, x);
      if (type == TGT_BF16) l = fresh(sizes, x);
    }
    sizes.back() = out;
    y = fresh(sizes, x);
    void* const stream = stream_of(x);
    if (type == TGT_BF16 && !record && few_rows(rows, in, mid, out)) {
      check(tgt_gated_few_rows(ptr(xc), ptr(wgc), ptr(wuc), ptr(wdc), ptr(rc), rows, int(in), int(mid), int(out), act, ptr(h), ptr(y),
                               stream));
      return y;
    }
    check(tgt_gated_block(ptr(xc), ptr(wgc), ptr(wuc), ptr(wdc), ptr(rc), rows, int(in), int(mid), int(out), act, type, ptr(h), ptr(g),
                          ptr(u), ptr(l), ptr(y), stream));
  }
  if (record) {
    auto node = std::shared_ptr<GatedFeedForwardBackward>(new GatedFeedForwardBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, wg, wu, wd, residual));
    node->act = act;
    node->with_residual = residual.defined();
    node->x = SavedVariable(x, false);
    node->w_gate = SavedVariable(wg, false);
    node->w_up = SavedVariable(wu, false);
    node->w_down = SavedVariable(wd, false);
    node->hidden = SavedVariable(h, false);
    node->gate = SavedVariable(g, false);
    node->up = SavedVariable(u, false);
    node->low = SavedVariable(l, false);
    torch::autograd::set_history(y, node);
  }
  return y;
}

}  // namespace

void bind_block(pybind11::module_& m) {
  m.def("add_rms_norm", &add_rms_norm, Unlocked());
  m.def("rms_norm_e4m3", &rms_norm_e4m3, Unlocked());
  m.def("edge_position_bias", &edge_position_bias, Unlocked());
  m.def("gated_feed_forward", &gated_feed_forward, Unlocked());
}

}  // namespace tgt_host
