// TorchScript operators on the features of the rows, and their gradients, on top of the
// C ABI in include/pca_features.h: torch.ops.pytorch_cluster_amd.{attention,
// norm_rotate, lookup}.  No counterpart in the reference.
//
// Checks of shapes and types come first, then those of devices.  Nothing waits for the
// device, so all of them (and their backward passes) may be captured into a graph.
// Workspaces come from PyTorch's caching allocator, call by call, on the current
// stream.
#include "ops_common.hpp"

#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <optional>
#include <vector>

#include "../../include/pca_features.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

Tensor or_none(const Maybe &t) { return t.has_value() ? *t : Tensor(); }
// (autograd takes a tensor that is not there in this form only)
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }

void check_type(const char *op, const Tensor &t, const char *name) {
  const auto type = t.scalar_type();
  TORCH_CHECK(type == at::kFloat || type == at::kHalf || type == at::kBFloat16,
              op, ": ", name, " has to be float32, float16 or bfloat16, got ",
              type);
}

// [rows, axes] fp32 positions; a vector counts as one axis.
Tensor positions(const char *op, const Tensor &pos, int64_t rows,
                 const char *name) {
  TORCH_CHECK(pos.scalar_type() == at::kFloat, op, ": ", name,
              " has to be float32, got ", pos.scalar_type());
  TORCH_CHECK(!pos.requires_grad(), op, ": ", name,
              " gets no gradient; pass ", name, ".detach()");
  TORCH_CHECK(pos.dim() == 1 || pos.dim() == 2, op, ": ", name,
              " has to be [rows, axes]");
  Tensor p = pos.dim() == 1 ? pos.view({-1, 1}) : pos;
  TORCH_CHECK(p.size(0) == rows, op, ": ", name, " has ", p.size(0),
              " rows for ", rows);
  TORCH_CHECK(p.size(1) >= 1 && p.size(1) <= 3, op, ": ", name,
              " has 1 to 3 axes, got ", p.size(1));
  return p;
}

// The kernels read the last dimension densely; the others by their strides.
Tensor dense_last(const Tensor &t) {
  return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

hipStream_t current_stream(const Tensor &t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

Tensor scratch(size_t bytes, const Tensor &like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

const void *data_or_null(const Tensor &t) {
  return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr;
}

// A second derivative would silently miss these operators.
void refuse_create_graph(const char *op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op,
              " cannot be differentiated twice (create_graph=True)");
}

// So would a forward-mode derivative, where no input wants a gradient.
void refuse_tangents(const char *op, std::initializer_list<Tensor> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode())
    return;
  for (const Tensor &t : tensors)
    TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), op,
                " has no forward-mode derivative");
}

// ---- attention ------------------------------------------------------------------

// Inputs after all checks, as the C ABI takes them.
struct Attention {
  Tensor q, k, v, pos_q, pos_k, slope, spans_q, spans_k;
  double scale = 1.0, cap = 0.0;

  pca_attention_args args() const {
    pca_attention_args a = {};
    a.q = data_or_null(q);
    a.k = data_or_null(k);
    a.v = data_or_null(v);
    a.q_row = q.stride(0);
    a.q_head = q.stride(1);
    a.k_row = k.stride(0);
    a.k_head = k.stride(1);
    a.v_row = v.stride(0);
    a.v_head = v.stride(1);
    a.spans_q = static_cast<const int32_t *>(data_or_null(spans_q));
    a.spans_k = static_cast<const int32_t *>(data_or_null(spans_k));
    if (slope.defined()) {
      a.slope = slope.data_ptr<float>();
      a.pos_q = static_cast<const float *>(data_or_null(pos_q));
      a.pos_k = static_cast<const float *>(data_or_null(pos_k));
      a.axes = (int32_t)pos_q.size(1);
    }
    a.dtype = dtype_code(q);
    a.nq = q.size(0);
    a.nk = k.size(0);
    a.hq = (int32_t)q.size(1);
    a.hk = (int32_t)k.size(1);
    a.d = (int32_t)q.size(2);
    a.scale = (float)scale;
    // (fp32 ends at both sides: a cap beyond bends nothing, one below leaves nothing)
    a.cap = cap > 0.0 ? (float)std::clamp(cap, (double)FLT_MIN, (double)FLT_MAX)
                      : 0.f;
    return a;
  }
  Tensor workspace(bool backward) const {
    const size_t bytes = pca_attention_workspace_bytes(
        q.size(0), k.size(0), (int32_t)q.size(1), (int32_t)k.size(1),
        (int32_t)q.size(2), backward);
    TORCH_CHECK(bytes > 0, "attention: problem size not supported");
    return scratch(bytes, q);
  }
};

Tensor spans_of(const Tensor &ids_a, const Tensor &ids_b) {
  auto spans =
      at::empty({ids_a.numel(), 2}, ids_a.options().dtype(at::kInt));
  check_status(pca_spans(
      static_cast<const int64_t *>(data_or_null(ids_a)), ids_a.numel(),
      static_cast<const int64_t *>(data_or_null(ids_b)), ids_b.numel(),
      static_cast<int32_t *>(const_cast<void *>(data_or_null(spans))),
      current_stream(ids_a)));
  return spans;
}

bool same_rows(const Tensor &a, const Tensor &b) {
  return a.data_ptr() == b.data_ptr() && a.numel() == b.numel();
}

// lse and rest: for the backward pass, or NULL.
Tensor attention_forward(const Attention &a, Tensor *lse, Tensor *rest) {
  auto out = at::empty(a.q.sizes(), a.q.options().memory_format(
                                        at::MemoryFormat::Contiguous));
  if (lse)
    *lse = at::empty({a.q.size(1), a.q.size(0)},
                     a.q.options().dtype(at::kFloat));
  if (rest && a.q.scalar_type() != at::kFloat)
    *rest = at::empty_like(out);
  const auto workspace = a.workspace(false);
  const auto args = a.args();
  check_status(pca_attention_forward(
      &args, const_cast<void *>(data_or_null(out)),
      rest ? const_cast<void *>(data_or_null(*rest)) : nullptr,
      lse ? static_cast<float *>(const_cast<void *>(data_or_null(*lse)))
          : nullptr,
      workspace.data_ptr(), (size_t)workspace.numel(), current_stream(a.q)));
  return out;
}

struct AttentionFunction
    : public torch::autograd::Function<AttentionFunction> {
  static Tensor forward(AutogradContext *ctx, Tensor q, Tensor k, Tensor v,
                        Maybe batch_q, Maybe batch_k, Maybe pos_q, Maybe pos_k,
                        Maybe slope, double scale, double cap) {
    DeviceScope scope(q.get_device());
    const Tensor ids_q = or_none(batch_q), ids_k = or_none(batch_k);
    Attention a;
    a.q = dense_last(q);
    a.k = dense_last(k);
    a.v = dense_last(v);
    a.pos_q = or_none(pos_q);
    a.pos_k = or_none(pos_k);
    a.slope = or_none(slope);
    a.scale = scale;
    a.cap = cap;
    if (ids_q.defined())
      a.spans_q = spans_of(ids_q, ids_k);
    Tensor lse, rest;
    auto out = attention_forward(a, &lse, &rest);
    ctx->save_for_backward({q, k, v, out, lse, ids_q, ids_k, a.pos_q, a.pos_k,
                            a.slope, a.spans_q, rest});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["cap"] = cap;
    return out;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    refuse_create_graph("attention");
    const auto saved = ctx->get_saved_variables();
    DeviceScope scope(saved[0].get_device());
    Attention a;
    a.q = dense_last(saved[0]);
    a.k = dense_last(saved[1]);
    a.v = dense_last(saved[2]);
    const Tensor &out = saved[3], &lse = saved[4];
    const Tensor &ids_q = saved[5], &ids_k = saved[6];
    a.pos_q = saved[7];
    a.pos_k = saved[8];
    a.slope = saved[9];
    a.spans_q = saved[10];
    a.scale = ctx->saved_data["scale"].toDouble();
    a.cap = ctx->saved_data["cap"].toDouble();
    if (ids_q.defined())
      a.spans_k =
          same_rows(ids_q, ids_k) ? a.spans_q : spans_of(ids_k, ids_q);
    const auto dout = dense_last(grads[0].to(a.q.scalar_type()));
    auto dense = a.q.options();
    auto dq = at::empty(a.q.sizes(), dense);
    auto dk = at::empty(a.k.sizes(), dense);
    auto dv = at::empty(a.v.sizes(), dense);
    const auto workspace = a.workspace(true);
    const auto args = a.args();
    check_status(pca_attention_backward(
        &args, data_or_null(out), data_or_null(saved[11]),
        static_cast<const float *>(data_or_null(lse)), data_or_null(dout),
        dout.stride(0), dout.stride(1), const_cast<void *>(data_or_null(dq)),
        const_cast<void *>(data_or_null(dk)),
        const_cast<void *>(data_or_null(dv)), workspace.data_ptr(),
        (size_t)workspace.numel(), current_stream(a.q)));
    return {dq,       dk,       dv,       Tensor(), Tensor(),
            Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor attention(const Tensor &q, const Tensor &k, const Tensor &v,
                 const Maybe &batch_q, const Maybe &batch_k,
                 const Maybe &pos_q, const Maybe &pos_k, const Maybe &slope,
                 std::optional<double> scale, double cap) {
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3,
              "attention: q, k and v have to be [rows, heads, channels]");
  check_type("attention", q, "q");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() &&
                  v.scalar_type() == q.scalar_type(),
              "attention: q, k and v have to be of one type");
  TORCH_CHECK(k.sizes() == v.sizes(),
              "attention: k and v have to be of one shape, got ", k.sizes(),
              " and ", v.sizes());
  TORCH_CHECK(q.size(2) == k.size(2),
              "attention: q and k differ in their channels, ", q.size(2),
              " and ", k.size(2));
  TORCH_CHECK(q.size(2) >= 1 && q.size(2) <= PCA_ATTENTION_MAX_D,
              "attention: heads have 1 to ", PCA_ATTENTION_MAX_D,
              " channels, got ", q.size(2));
  TORCH_CHECK(k.size(1) >= 1 && q.size(1) >= 1 && q.size(1) % k.size(1) == 0,
              "attention: the heads of q (", q.size(1),
              ") have to be a multiple of those of k (", k.size(1), ")");
  TORCH_CHECK(batch_q.has_value() == batch_k.has_value(),
              "attention: batch_q and batch_k go together");
  if (batch_q.has_value()) {
    TORCH_CHECK(batch_q->dim() == 1 && batch_q->numel() == q.size(0) &&
                    batch_k->dim() == 1 && batch_k->numel() == k.size(0),
                "attention: a batch vector needs one entry for each row");
    TORCH_CHECK(at::isIntegralType(batch_q->scalar_type(), false) &&
                    at::isIntegralType(batch_k->scalar_type(), false),
                "attention: batch vectors hold integers");
  }
  TORCH_CHECK(slope.has_value() == pos_q.has_value() &&
                  slope.has_value() == pos_k.has_value(),
              "attention: slope, pos_q and pos_k go together");
  Tensor at_q, at_k, slopes;
  if (slope.has_value()) {
    at_q = positions("attention", *pos_q, q.size(0), "pos_q");
    at_k = positions("attention", *pos_k, k.size(0), "pos_k");
    TORCH_CHECK(at_q.size(1) == at_k.size(1),
                "attention: pos_q and pos_k differ in their axes");
    TORCH_CHECK(slope->scalar_type() == at::kFloat && slope->dim() == 1 &&
                    slope->size(0) == q.size(1),
                "attention: slope has to be float32, one for each head of q");
    TORCH_CHECK(!slope->requires_grad(),
                "attention: slope gets no gradient; pass slope.detach()");
    slopes = *slope;
  }
  const double factor =
      scale.has_value() ? *scale : 1.0 / std::sqrt((double)q.size(2));
  TORCH_CHECK(std::isfinite(factor), "attention: scale has to be finite");
  TORCH_CHECK(std::isfinite(cap) && cap >= 0.0,
              "attention: cap has to be finite and not negative");
  refuse_tangents("attention", {q, k, v, at_q, at_k, slopes});

  PCA_CHECK_GPU(q);
  for (const Tensor &t :
       {k, v, or_none(batch_q), or_none(batch_k), at_q, at_k, slopes})
    TORCH_CHECK(!t.defined() || t.device() == q.device(),
                "attention: tensors on ", q.device(), " and ", t.device());
  Tensor ids_q, ids_k;
  {
    DeviceScope scope(q.get_device());
    if (batch_q.has_value()) {
      ids_q = batch_q->to(at::kLong).contiguous();
      ids_k = batch_k->is_same(*batch_q)
                  ? ids_q
                  : batch_k->to(at::kLong).contiguous();
    }
    if (slopes.defined()) {
      at_q = at_q.contiguous();
      at_k = at_k.contiguous();
      slopes = slopes.contiguous();
    }
  }
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return AttentionFunction::apply(q, k, v, maybe(ids_q), maybe(ids_k),
                                    maybe(at_q), maybe(at_k), maybe(slopes),
                                    factor, cap);
  DeviceScope scope(q.get_device());
  Attention a;
  a.q = dense_last(q);
  a.k = dense_last(k);
  a.v = dense_last(v);
  a.pos_q = at_q;
  a.pos_k = at_k;
  a.slope = slopes;
  a.scale = factor;
  a.cap = cap;
  if (ids_q.defined())
    a.spans_q = spans_of(ids_q, ids_k);
  return attention_forward(a, nullptr, nullptr);
}

// ---- norm_rotate ------------------------------------------------------------------

struct NormRotate {
  Tensor q, k, pos, freq, weight_q, weight_k;
  double eps = 0.0;

  pca_norm_rotate_args args() const {
    pca_norm_rotate_args a = {};
    a.q = data_or_null(q);
    a.q_row = q.stride(0);
    a.q_head = q.stride(1);
    a.hq = (int32_t)q.size(1);
    if (k.defined()) {
      a.k = data_or_null(k);
      a.k_row = k.stride(0);
      a.k_head = k.stride(1);
      a.hk = (int32_t)k.size(1);
    }
    a.weight_q = data_or_null(weight_q);
    a.weight_k = data_or_null(weight_k);
    a.pos = static_cast<const float *>(data_or_null(pos));
    a.freq = static_cast<const float *>(data_or_null(freq));
    a.rows = q.size(0);
    a.d = (int32_t)q.size(2);
    a.axes = (int32_t)pos.size(1);
    a.rotated = (int32_t)freq.size(1);
    a.dtype = dtype_code(q);
    a.weight_dtype = weight_q.defined()   ? dtype_code(weight_q)
                     : weight_k.defined() ? dtype_code(weight_k)
                                          : PCA_F32;
    a.eps = (float)eps;
    return a;
  }
};

Tensor dense_like(const Tensor &t) {
  return t.defined()
             ? at::empty(t.sizes(), t.options().memory_format(
                                        at::MemoryFormat::Contiguous))
             : Tensor();
}

variable_list norm_rotate_forward(const NormRotate &n) {
  auto out_q = dense_like(n.q), out_k = dense_like(n.k);
  const auto args = n.args();
  check_status(pca_norm_rotate_forward(
      &args, const_cast<void *>(data_or_null(out_q)),
      const_cast<void *>(data_or_null(out_k)), current_stream(n.q)));
  if (!out_k.defined())
    return {out_q};
  return {out_q, out_k};
}

struct NormRotateFunction
    : public torch::autograd::Function<NormRotateFunction> {
  static variable_list forward(AutogradContext *ctx, Tensor q, Maybe maybe_k,
                               Tensor pos, Tensor freq, Maybe maybe_weight_q,
                               Maybe maybe_weight_k, double eps) {
    DeviceScope scope(q.get_device());
    const Tensor k = or_none(maybe_k);
    const Tensor weight_q = or_none(maybe_weight_q);
    const Tensor weight_k = or_none(maybe_weight_k);
    NormRotate n;
    n.q = dense_last(q);
    n.k = k.defined() ? dense_last(k) : k;
    n.pos = pos;
    n.freq = freq;
    n.weight_q = weight_q.defined() ? weight_q.contiguous() : weight_q;
    n.weight_k = weight_k.defined() ? weight_k.contiguous() : weight_k;
    n.eps = eps;
    ctx->save_for_backward({q, k, pos, freq, weight_q, weight_k});
    ctx->saved_data["eps"] = eps;
    return norm_rotate_forward(n);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    refuse_create_graph("norm_rotate");
    const auto saved = ctx->get_saved_variables();
    DeviceScope scope(saved[0].get_device());
    NormRotate n;
    n.q = dense_last(saved[0]);
    n.k = saved[1].defined() ? dense_last(saved[1]) : saved[1];
    n.pos = saved[2];
    n.freq = saved[3];
    n.weight_q = saved[4].defined() ? saved[4].contiguous() : saved[4];
    n.weight_k = saved[5].defined() ? saved[5].contiguous() : saved[5];
    n.eps = ctx->saved_data["eps"].toDouble();
    const auto type = n.q.scalar_type();
    const auto dout_q = dense_last(grads[0].to(type));
    Tensor dout_k;
    if (n.k.defined())
      dout_k = dense_last(grads[1].to(type));
    auto dq = dense_like(n.q), dk = dense_like(n.k);
    Tensor dweight_q, dweight_k;
    if (n.weight_q.defined())
      dweight_q = at::empty_like(n.weight_q);
    if (n.weight_k.defined())
      dweight_k = at::empty_like(n.weight_k);
    const auto workspace = scratch(
        pca_norm_rotate_workspace_bytes(n.q.size(0), (int32_t)n.q.size(2)),
        n.q);
    const auto args = n.args();
    check_status(pca_norm_rotate_backward(
        &args, data_or_null(dout_q), dout_q.stride(0), dout_q.stride(1),
        data_or_null(dout_k), dout_k.defined() ? dout_k.stride(0) : 0,
        dout_k.defined() ? dout_k.stride(1) : 0,
        const_cast<void *>(data_or_null(dq)),
        const_cast<void *>(data_or_null(dk)),
        const_cast<void *>(data_or_null(dweight_q)),
        const_cast<void *>(data_or_null(dweight_k)), workspace.data_ptr(),
        (size_t)workspace.numel(), current_stream(n.q)));
    return {dq, dk, Tensor(), Tensor(), dweight_q, dweight_k, Tensor()};
  }
};

std::vector<Tensor> norm_rotate(const Tensor &q, const Maybe &k,
                                const Tensor &pos, const Tensor &freq,
                                const Maybe &weight_q, const Maybe &weight_k,
                                double eps) {
  TORCH_CHECK(q.dim() == 3, "norm_rotate: q has to be [rows, heads, channels]");
  check_type("norm_rotate", q, "q");
  TORCH_CHECK(q.size(1) >= 1 && q.size(2) >= 1 &&
                  q.size(2) <= PCA_NORM_ROTATE_MAX_D,
              "norm_rotate: heads have 1 to ", PCA_NORM_ROTATE_MAX_D,
              " channels, got ", q.size(2));
  if (k.has_value())
    TORCH_CHECK(k->dim() == 3 && k->scalar_type() == q.scalar_type() &&
                    k->size(0) == q.size(0) && k->size(1) >= 1 &&
                    k->size(2) == q.size(2),
                "norm_rotate: k has to be of q's type, rows and channels");
  const Tensor at = positions("norm_rotate", pos, q.size(0), "pos");
  TORCH_CHECK(freq.scalar_type() == at::kFloat && freq.dim() == 2 &&
                  freq.size(0) == at.size(1),
              "norm_rotate: freq has to be float32, [axes of pos, pairs]");
  TORCH_CHECK(!freq.requires_grad(),
              "norm_rotate: freq gets no gradient; pass freq.detach()");
  TORCH_CHECK(2 * freq.size(1) <= q.size(2), "norm_rotate: ", freq.size(1),
              " pairs do not fit ", q.size(2), " channels");
  TORCH_CHECK(k.has_value() || !weight_k.has_value(),
              "norm_rotate: weight_k without k");
  for (const Maybe &w : {weight_q, weight_k})
    if (w.has_value())
      TORCH_CHECK(w->dim() == 1 && w->size(0) == q.size(2) &&
                      (w->scalar_type() == at::kFloat ||
                       w->scalar_type() == q.scalar_type()),
                  "norm_rotate: a weight has to be [channels], of q's type or "
                  "float32");
  if (weight_q.has_value() && weight_k.has_value())
    TORCH_CHECK(weight_q->scalar_type() == weight_k->scalar_type(),
                "norm_rotate: weight_q and weight_k have to be of one type");
  TORCH_CHECK(std::isfinite(eps) && eps >= 0.0,
              "norm_rotate: eps has to be finite and not negative");
  refuse_tangents("norm_rotate", {q, or_none(k), pos, freq, or_none(weight_q),
                                  or_none(weight_k)});

  PCA_CHECK_GPU(q);
  for (const Tensor &t :
       {or_none(k), pos, freq, or_none(weight_q), or_none(weight_k)})
    TORCH_CHECK(!t.defined() || t.device() == q.device(),
                "norm_rotate: tensors on ", q.device(), " and ", t.device());
  NormRotate n;
  {
    DeviceScope scope(q.get_device());
    n.pos = at.contiguous();
    n.freq = freq.contiguous();
  }
  n.q = q;
  n.k = or_none(k);
  n.weight_q = or_none(weight_q);
  n.weight_k = or_none(weight_k);
  n.eps = eps;
  bool grad = false;
  for (const Tensor &t : {n.q, n.k, n.weight_q, n.weight_k})
    grad |= t.defined() && t.requires_grad();
  if (grad && at::GradMode::is_enabled())
    return NormRotateFunction::apply(n.q, maybe(n.k), n.pos, n.freq,
                                     maybe(n.weight_q), maybe(n.weight_k), eps);
  DeviceScope scope(q.get_device());
  n.q = dense_last(n.q);
  if (n.k.defined())
    n.k = dense_last(n.k);
  if (n.weight_q.defined())
    n.weight_q = n.weight_q.contiguous();
  if (n.weight_k.defined())
    n.weight_k = n.weight_k.contiguous();
  return norm_rotate_forward(n);
}

// ---- lookup -----------------------------------------------------------------------

// The C ABI wants tables that start on 16 bytes.
Tensor dense16(const Tensor &t) {
  const Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 ? c : c.clone();
}

Tensor lookup_rows(const Tensor &weight, const Tensor &index, double scale) {
  const Tensor table = dense16(weight);
  auto sizes = index.sizes().vec();
  sizes.push_back(table.size(1));
  auto out = at::empty(sizes, table.options());
  check_status(pca_lookup(
      data_or_null(table), data_or_null(index), (int32_t)index.element_size(),
      table.size(0), index.numel(), table.size(1), (float)scale,
      dtype_code(table), const_cast<void *>(data_or_null(out)),
      current_stream(table)));
  return out;
}

struct LookupFunction : public torch::autograd::Function<LookupFunction> {
  static Tensor forward(AutogradContext *ctx, Tensor weight, Tensor index,
                        double scale) {
    DeviceScope scope(weight.get_device());
    ctx->save_for_backward({index});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["rows"] = weight.size(0);
    return lookup_rows(weight, index, scale);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    refuse_create_graph("lookup");
    const auto index = ctx->get_saved_variables()[0];
    DeviceScope scope(index.get_device());
    const int64_t rows = ctx->saved_data["rows"].toInt();
    const Tensor dout = dense16(grads[0]);
    const int64_t width = dout.size(-1);
    auto dweight = at::empty({rows, width}, dout.options());
    const auto workspace = scratch(
        pca_lookup_grad_workspace_bytes(rows, index.numel(), width), dout);
    check_status(pca_lookup_grad(
        data_or_null(dout), data_or_null(index), (int32_t)index.element_size(),
        rows, index.numel(), width, (float)ctx->saved_data["scale"].toDouble(),
        dtype_code(dout), const_cast<void *>(data_or_null(dweight)),
        workspace.data_ptr(), (size_t)workspace.numel(),
        current_stream(dout)));
    return {dweight, Tensor(), Tensor()};
  }
};

Tensor lookup(const Tensor &weight, const Tensor &index, double scale) {
  TORCH_CHECK(weight.dim() == 2, "lookup: weight has to be [rows, channels]");
  check_type("lookup", weight, "weight");
  TORCH_CHECK(index.scalar_type() == at::kLong ||
                  index.scalar_type() == at::kInt,
              "lookup: index has to be int64 or int32, got ",
              index.scalar_type());
  TORCH_CHECK(std::isfinite(scale), "lookup: scale has to be finite");
  refuse_tangents("lookup", {weight});
  PCA_CHECK_GPU(weight);
  TORCH_CHECK(index.device() == weight.device(), "lookup: tensors on ",
              weight.device(), " and ", index.device());
  Tensor flat;
  {
    DeviceScope scope(weight.get_device());
    flat = index.contiguous();
  }
  if (at::GradMode::is_enabled() && weight.requires_grad())
    return LookupFunction::apply(weight, flat, scale);
  DeviceScope scope(weight.get_device());
  return lookup_rows(weight, flat, scale);
}

} // namespace

TORCH_LIBRARY_FRAGMENT(pytorch_cluster_amd, m) {
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? batch_q, "
        "Tensor? batch_k, Tensor? pos_q, Tensor? pos_k, Tensor? slope, "
        "float? scale, float cap) -> Tensor",
        &attention);
  m.def("norm_rotate(Tensor q, Tensor? k, Tensor pos, Tensor freq, "
        "Tensor? weight_q, Tensor? weight_k, float eps) -> Tensor[]",
        &norm_rotate);
  m.def("lookup(Tensor weight, Tensor index, float scale) -> Tensor",
        &lookup);
}
