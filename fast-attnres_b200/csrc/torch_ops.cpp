// torch operators of LayerNorm, embedding and vocabulary loss over the C ABI, with their autograd.
//
// These operators also run on a handful of rows, where the host's share of a call is most of its
// time.  layer_norm on eight rows, on a GPU host: 8.5 us a call, 18.9 through ctypes; forward and
// backward 77 us against 134 with a Python autograd function (60 of them are torch's engine, which
// takes 57 us for a multiplication and its gradient on that host).
//
// Per operator: `<name>_forward` and `<name>_backward` do the work (their fake kernels are in
// Python, so a compiled graph holds these two), `<name>` is the differentiable call.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include "../../include/attnres_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int status, const char* what) {
  TORCH_CHECK(status == ATTNRES_B200_OK, what, " failed: ", attnres_b200_status_string(status),
              " (status ", status, ")");
}

int64_t sized(int64_t value, const char* what) {
  if (value < 0) check((int)-value, what);
  return value;
}

int type_code(ScalarType type) {
  switch (type) {
    case at::kBFloat16: return ATTNRES_B200_BF16;
    case at::kHalf: return ATTNRES_B200_FP16;
    case at::kFloat: return ATTNRES_B200_FP32;
    default: TORCH_CHECK_TYPE(false, "BF16, FP16 or FP32 is required, got ", type);
  }
}

void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor unless_missing(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// Gradient slots of an operator's result are tensors; one that is not wanted has no elements.
Tensor or_nothing(const Tensor& t, const Tensor& like, ScalarType type) {
  return t.defined() ? t : at::empty({0}, like.options().dtype(type));
}

// `[..., D]` as rows of D neighbouring elements one stride apart: the tensor itself where its
// strides allow it (axes of one element never matter), else a contiguous copy.
struct Rows {
  Tensor kept;
  int64_t stride;
};

Rows rows_of(const Tensor& t) {
  const int64_t width = t.size(-1);
  if (t.is_contiguous()) return {t, width};
  if (t.stride(-1) == 1 || width == 1) {
    int64_t stride = 0, inside = 1;
    bool found = false, affine = true;
    for (int64_t axis = t.dim() - 2; axis >= 0 && affine; --axis) {
      if (t.size(axis) == 1) continue;
      if (!found) stride = t.stride(axis);
      else affine = t.stride(axis) == inside * stride;
      found = true;
      inside *= t.size(axis);
    }
    if (affine && stride >= 0) return {t, found ? stride : width};
  }
  return {t.contiguous(), width};
}

template <typename Signature>
auto operation(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

// Differentiating these gradients again is refused when it is tried, not when a graph of the
// first gradient is asked for.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (const Tensor& g : grads)
    if (g.defined()) {
      Tensor leaf = g.detach();
      leaf.set_requires_grad(true);
      defined.push_back(leaf);
    }
  const auto count = (int64_t)defined.size();
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "this operator is differentiable once", count);
  variable_list marked = (*refuse)(std::move(defined));
  size_t next = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = marked[next++];
  return grads;
}

bool needed(AutogradContext* ctx, const Tensor& t, size_t edge) {
  return t.defined() && ctx->needs_input_grad(edge);
}

// ------------------------------------------------------------------------------ LayerNorm

std::tuple<Tensor, Tensor> norm_forward(const Tensor& x, const optional<Tensor>& weight,
                                        const optional<Tensor>& bias, double eps, bool need_stats) {
  const int64_t width = x.size(-1), rows = x.numel() / width;
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor stats = at::empty({2, need_stats ? rows : 0}, x.options().dtype(at::kFloat));
  if (rows == 0) return {y, stats};
  c10::cuda::CUDAGuard guard(x.device());
  const Rows in = rows_of(x);
  const Tensor w = unless_missing(weight), b = unless_missing(bias);
  const ScalarType type = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat;
  check(attnres_b200_norm_forward(in.kept.data_ptr(), in.stride, pointer(w), pointer(b), rows,
                                  (int32_t)width, type_code(x.scalar_type()), type_code(type),
                                  (float)eps, y.data_ptr(),
                                  need_stats ? stats.data_ptr<float>() : nullptr, stream_of(x)),
        "attnres_b200_norm_forward");
  return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& grad, const Tensor& x,
                                                 const Tensor& stats, const optional<Tensor>& weight,
                                                 ScalarType param_type, bool need_x,
                                                 bool need_weight, bool need_bias) {
  const int64_t width = x.size(-1), rows = x.numel() / width;
  const auto params = x.options().dtype(param_type);
  Tensor dx, dweight, dbias;
  if (need_x) dx = at::empty(x.sizes(), x.options());
  if (need_weight) dweight = rows ? at::empty({width}, params) : at::zeros({width}, params);
  if (need_bias) dbias = rows ? at::empty({width}, params) : at::zeros({width}, params);
  if (rows != 0 && (need_x || need_weight || need_bias)) {
    c10::cuda::CUDAGuard guard(x.device());
    const Rows in = rows_of(x), up = rows_of(grad);
    const Tensor w = unless_missing(weight);
    Tensor partials;
    int32_t partial_rows = 0;
    if (need_weight || need_bias) {
      partial_rows = (int32_t)sized(
          attnres_b200_norm_workspace_rows(rows, (int32_t)width, x.device().index()),
          "attnres_b200_norm_workspace_rows");
      partials = at::empty({partial_rows, 2 * width}, x.options().dtype(at::kFloat));
    }
    check(attnres_b200_norm_backward(
              up.kept.data_ptr(), up.stride, in.kept.data_ptr(), in.stride, stats.data_ptr<float>(),
              pointer(w), rows, (int32_t)width, type_code(x.scalar_type()), type_code(param_type),
              pointer(dx), static_cast<float*>(pointer(partials)), partial_rows, pointer(dweight),
              pointer(dbias), stream_of(x)),
          "attnres_b200_norm_backward");
  }
  return {or_nothing(dx, x, x.scalar_type()), or_nothing(dweight, x, param_type),
          or_nothing(dbias, x, param_type)};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight,
                        const optional<Tensor>& bias, double eps) {
    static auto op = operation<decltype(norm_forward)>("attnres_b200::norm_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, stats] = op.call(x, weight, bias, eps, true);
    const Tensor w = unless_missing(weight), b = unless_missing(bias);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["type"] = (int64_t)(w.defined()   ? w.scalar_type()
                                        : b.defined() ? b.scalar_type()
                                                      : at::kFloat);
    ctx->saved_data["bias"] = b.defined();
    ctx->set_materialize_grads(false);
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(4);
    static auto op = operation<decltype(norm_backward)>("attnres_b200::norm_backward");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1];
    // edges follow the tensors that were given
    const bool nx = ctx->needs_input_grad(0), nw = needed(ctx, weight, 1);
    const bool nb = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weight.defined() ? 2 : 1);
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dx, dw, db] =
        op.call(grads[0], x, saved[2], weight.defined() ? optional<Tensor>(weight) : std::nullopt,
                (ScalarType)ctx->saved_data["type"].toInt(), nx, nw, nb);
    return once({nx ? dx : Tensor(), nw ? dw : Tensor(), nb ? db : Tensor(), Tensor()});
  }
};

// Whether a call has to leave a node behind.  Without one it goes straight to the device's (or the
// tracer's) kernel.
bool differentiated(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : inputs)
    if (t != nullptr && t->defined() && t->requires_grad()) return true;
  return false;
}

const Tensor* given(const optional<Tensor>& t) { return t.has_value() ? &*t : nullptr; }

Tensor layer_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                  double eps);

Tensor layer_norm_autograd(const Tensor& x, const optional<Tensor>& weight,
                           const optional<Tensor>& bias, double eps) {
  if (!differentiated({&x, given(weight), given(bias)})) {
    static auto op = operation<decltype(layer_norm)>("attnres_b200::layer_norm");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, weight, bias, eps);
  }
  return LayerNorm::apply(x, weight, bias, eps);
}

Tensor layer_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                  double eps) {
  return std::get<0>(norm_forward(x, weight, bias, eps, false));
}

// ------------------------------------------------------------------------------ embedding

int64_t period_of(const Tensor& tokens) { return tokens.dim() ? tokens.size(-1) : 1; }

Tensor embedding_forward(const Tensor& tokens, const Tensor& table, const optional<Tensor>& positions,
                         double scale, ScalarType type) {
  const int64_t width = table.size(1);
  auto shape = tokens.sizes().vec();
  shape.push_back(width);
  Tensor out = at::empty(shape, table.options().dtype(type));
  if (tokens.numel() == 0) return out;
  c10::cuda::CUDAGuard guard(table.device());
  const Tensor ids = tokens.contiguous();
  const Rows rows = rows_of(table);
  Rows added{Tensor(), 0};
  if (positions.has_value()) added = rows_of(*positions);
  check(attnres_b200_embedding_forward(
            ids.data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), period_of(ids),
            (int32_t)table.size(0), (int32_t)width, rows.kept.data_ptr(), rows.stride,
            type_code(table.scalar_type()), pointer(added.kept), added.stride,
            added.kept.defined() ? type_code(added.kept.scalar_type()) : ATTNRES_B200_FP32,
            (float)scale, out.data_ptr(), type_code(type), stream_of(table)),
        "attnres_b200_embedding_forward");
  return out;
}

std::tuple<Tensor, Tensor> embedding_backward(const Tensor& grad, const Tensor& tokens,
                                              int64_t vocabulary, ScalarType table_type,
                                              ScalarType position_type, double scale,
                                              int64_t padding, bool need_table, bool need_positions) {
  const int64_t width = grad.size(-1), count = tokens.numel(), period = period_of(tokens);
  Tensor dtable, dpositions;
  const auto table = grad.options().dtype(table_type), position = grad.options().dtype(position_type);
  if (need_table)
    dtable = count ? at::empty({vocabulary, width}, table) : at::zeros({vocabulary, width}, table);
  if (need_positions)
    dpositions = count ? at::empty({period, width}, position) : at::zeros({period, width}, position);
  if (count != 0 && (need_table || need_positions)) {
    c10::cuda::CUDAGuard guard(grad.device());
    const Tensor ids = tokens.contiguous();
    const Rows up = rows_of(grad);
    Tensor workspace;
    int64_t bytes = 0;
    if (need_table) {
      bytes = sized(attnres_b200_embedding_workspace_bytes(count, (int32_t)width),
                    "attnres_b200_embedding_workspace_bytes");
      workspace = at::empty({bytes}, grad.options().dtype(at::kByte));
    }
    check(attnres_b200_embedding_backward(
              ids.data_ptr(), ids.scalar_type() == at::kLong, count, period, (int32_t)vocabulary,
              (int32_t)width, padding, up.kept.data_ptr(), up.stride, type_code(grad.scalar_type()),
              (float)scale, pointer(dtable), type_code(table_type), pointer(dpositions),
              type_code(position_type), pointer(workspace), bytes, stream_of(grad)),
          "attnres_b200_embedding_backward");
  }
  return {or_nothing(dtable, grad, table_type), or_nothing(dpositions, grad, position_type)};
}

std::tuple<Tensor, Tensor> embedding_backward_sym(const Tensor& grad, const Tensor& tokens,
                                                  c10::SymInt vocabulary, ScalarType table_type,
                                                  ScalarType position_type, double scale,
                                                  int64_t padding, bool need_table,
                                                  bool need_positions) {
  return embedding_backward(grad, tokens, vocabulary.guard_int(__FILE__, __LINE__), table_type,
                            position_type, scale, padding, need_table, need_positions);
}

struct Embed : torch::autograd::Function<Embed> {
  static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& table,
                        const optional<Tensor>& positions, double scale, int64_t padding,
                        ScalarType type) {
    static auto op = operation<decltype(embedding_forward)>("attnres_b200::embedding_forward");
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({tokens});
    auto& data = ctx->saved_data;
    data["vocabulary"] = table.sym_size(0);
    data["table"] = (int64_t)table.scalar_type();
    data["given"] = positions.has_value();
    data["positions"] = (int64_t)(positions.has_value() ? positions->scalar_type() : at::kFloat);
    data["scale"] = scale;
    data["padding"] = padding;
    ctx->set_materialize_grads(false);
    return op.call(tokens, table, positions, scale, type);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(6);
    static auto op = operation<decltype(embedding_backward_sym)>("attnres_b200::embedding_backward");
    auto& data = ctx->saved_data;
    const bool nt = ctx->needs_input_grad(1);
    const bool np = data["given"].toBool() && ctx->needs_input_grad(2);
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dtable, dpositions] = op.call(
        grads[0], ctx->get_saved_variables()[0], data["vocabulary"].toSymInt(),
        (ScalarType)data["table"].toInt(), (ScalarType)data["positions"].toInt(),
        data["scale"].toDouble(), data["padding"].toInt(), nt, np);
    return once({Tensor(), nt ? dtable : Tensor(), np ? dpositions : Tensor(), Tensor(), Tensor(),
                 Tensor()});
  }
};

Tensor embed(const Tensor& tokens, const Tensor& table, const optional<Tensor>& positions,
             double scale, int64_t padding, ScalarType type);

Tensor embed_autograd(const Tensor& tokens, const Tensor& table, const optional<Tensor>& positions,
                      double scale, int64_t padding, ScalarType type) {
  if (!differentiated({&table, given(positions)})) {
    static auto op = operation<decltype(embed)>("attnres_b200::embed");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(tokens, table, positions, scale, padding, type);
  }
  return Embed::apply(tokens, table, positions, scale, padding, type);
}

Tensor embed(const Tensor& tokens, const Tensor& table, const optional<Tensor>& positions,
             double scale, int64_t, ScalarType type) {
  return embedding_forward(tokens, table, positions, scale, type);
}

// ------------------------------------------------------------------------------ vocabulary loss

constexpr int64_t kAlign = 64;  // elements between the arrays that share one allocation

struct LossForward {
  Tensor loss, kept, index, count, sums, dhidden, dweight;
};

LossForward run_loss(const Tensor& hidden, const Tensor& weight, const Tensor& targets,
                     int64_t ignored, int64_t reduction, double scale, bool gradients,
                     bool need_hidden, bool need_weight) {
  const int64_t width = hidden.size(-1), vocabulary = weight.size(0), rows = hidden.numel() / width;
  const auto floats = hidden.options().dtype(at::kFloat);
  const auto ints = hidden.options().dtype(at::kInt);
  const bool each = reduction == ATTNRES_B200_LOSS_NONE;
  LossForward r;
  r.kept = at::empty({rows, (width + 7) / 8 * 8}, hidden.options());
  r.index = at::empty({2, rows}, ints);
  r.count = at::empty({1}, ints);
  if (!gradients) r.sums = at::empty({rows}, floats);
  r.loss = each ? at::empty(targets.sizes(), floats) : at::empty({}, floats);
  if (gradients && need_hidden) r.dhidden = at::empty(hidden.sizes(), hidden.options());
  if (gradients && need_weight)
    r.dweight = rows ? at::empty({vocabulary, width}, hidden.options())
                     : at::zeros({vocabulary, width}, hidden.options());
  if (rows == 0) {
    r.count.zero_();
    if (!each)
      r.loss.fill_(reduction == ATTNRES_B200_LOSS_SUM ? 0.0
                                                      : std::numeric_limits<double>::quiet_NaN());
    return r;
  }
  c10::cuda::CUDAGuard guard(hidden.device());
  const Rows source = rows_of(hidden), head = rows_of(weight);
  const Tensor ids = targets.contiguous();
  const int64_t bytes = sized(
      attnres_b200_loss_workspace_bytes(
          rows, (int32_t)vocabulary, (int32_t)width,
          gradients ? ATTNRES_B200_LOSS_FORWARD_GRADIENTS : ATTNRES_B200_LOSS_FORWARD),
      "attnres_b200_loss_workspace_bytes");
  const int64_t losses_bytes = each ? 0 : (rows + kAlign) / kAlign * kAlign * 4;
  Tensor workspace = at::empty({bytes + losses_bytes}, hidden.options().dtype(at::kByte));
  char* space = static_cast<char*>(workspace.data_ptr());
  float* losses = each ? r.loss.data_ptr<float>() : reinterpret_cast<float*>(space);
  check(attnres_b200_loss_forward(
            source.kept.data_ptr(), source.stride, head.kept.data_ptr(), head.stride, ids.data_ptr(),
            ids.scalar_type() == at::kLong, rows, (int32_t)vocabulary, (int32_t)width,
            type_code(hidden.scalar_type()), ignored, (float)scale, (int32_t)reduction,
            r.kept.data_ptr(), r.index.data_ptr<int32_t>(), r.index.data_ptr<int32_t>() + rows,
            r.count.data_ptr<int32_t>(), static_cast<float*>(pointer(r.sums)), losses,
            each ? nullptr : r.loss.data_ptr<float>(), pointer(r.dhidden), pointer(r.dweight),
            space + losses_bytes, bytes, stream_of(hidden)),
        "attnres_b200_loss_forward");
  return r;
}

// -> loss, kept rows, their [2, N] indices and targets, their count, log2 of their sums
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> loss_forward(
    const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignored,
    int64_t reduction, double scale) {
  LossForward r = run_loss(hidden, weight, targets, ignored, reduction, scale, false, false, false);
  return {r.loss, r.kept, r.index, r.count, r.sums};
}

// -> loss, and the gradients of hidden and weight for an upstream gradient of one
std::tuple<Tensor, Tensor, Tensor> loss_with_gradients(const Tensor& hidden, const Tensor& weight,
                                                       const Tensor& targets, int64_t ignored,
                                                       int64_t reduction, double scale,
                                                       bool need_hidden, bool need_weight) {
  LossForward r = run_loss(hidden, weight, targets, ignored, reduction, scale, true, need_hidden,
                           need_weight);
  return {r.loss, or_nothing(r.dhidden, hidden, hidden.scalar_type()),
          or_nothing(r.dweight, hidden, hidden.scalar_type())};
}

Tensor loss_scale_gradient(const Tensor& gradient, const Tensor& upstream) {
  Tensor out = at::empty(gradient.sizes(), gradient.options());
  if (gradient.numel() == 0) return out;
  c10::cuda::CUDAGuard guard(gradient.device());
  check(attnres_b200_loss_scale_gradient(gradient.data_ptr(), upstream.data_ptr<float>(),
                                         gradient.numel(), out.data_ptr(), stream_of(gradient)),
        "attnres_b200_loss_scale_gradient");
  return out;
}

std::tuple<Tensor, Tensor> loss_backward(const Tensor& grad, const Tensor& weight,
                                         const Tensor& targets, const Tensor& kept,
                                         const Tensor& index, const Tensor& count, const Tensor& sums,
                                         int64_t ignored, int64_t reduction, double scale,
                                         bool need_hidden, bool need_weight) {
  const int64_t width = weight.size(1), vocabulary = weight.size(0), rows = targets.numel();
  Tensor dhidden, dweight;
  if (need_hidden) {
    auto shape = targets.sizes().vec();
    shape.push_back(width);
    dhidden = at::empty(shape, weight.options());
  }
  if (need_weight)
    dweight = rows ? at::empty({vocabulary, width}, weight.options())
                   : at::zeros({vocabulary, width}, weight.options());
  if (rows != 0 && (need_hidden || need_weight)) {
    c10::cuda::CUDAGuard guard(weight.device());
    const Rows head = rows_of(weight);
    const Tensor ids = targets.contiguous(), upstream = grad.contiguous();
    const int64_t bytes = sized(
        attnres_b200_loss_workspace_bytes(rows, (int32_t)vocabulary, (int32_t)width,
                                          ATTNRES_B200_LOSS_BACKWARD),
        "attnres_b200_loss_workspace_bytes");
    Tensor workspace = at::empty({bytes}, weight.options().dtype(at::kByte));
    check(attnres_b200_loss_backward(
              upstream.data_ptr<float>(), 1, head.kept.data_ptr(), head.stride, ids.data_ptr(),
              ids.scalar_type() == at::kLong, rows, (int32_t)vocabulary, (int32_t)width,
              type_code(weight.scalar_type()), ignored, (float)scale, (int32_t)reduction,
              kept.data_ptr(), index.data_ptr<int32_t>(), index.data_ptr<int32_t>() + rows,
              count.data_ptr<int32_t>(), sums.data_ptr<float>(), pointer(dhidden), pointer(dweight),
              workspace.data_ptr(), bytes, stream_of(weight)),
          "attnres_b200_loss_backward");
  }
  return {or_nothing(dhidden, weight, weight.scalar_type()),
          or_nothing(dweight, weight, weight.scalar_type())};
}

// Which of the two forwards serves a call that will be differentiated.
bool gradients_in_forward(const Tensor& hidden, int64_t reduction) {
  return attnres_b200_loss_gradients_in_forward((int32_t)hidden.size(-1),
                                                type_code(hidden.scalar_type()),
                                                (int32_t)reduction) != 0;
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                        const Tensor& targets, int64_t ignored, int64_t reduction, double scale) {
    const bool need_hidden = hidden.requires_grad(), need_weight = weight.requires_grad();
    ctx->set_materialize_grads(false);
    at::AutoDispatchBelowADInplaceOrView below;
    const bool early = (need_hidden || need_weight) && gradients_in_forward(hidden, reduction);
    ctx->saved_data["early"] = early;
    if (early) {
      static auto op = operation<decltype(loss_with_gradients)>(
          "attnres_b200::linear_cross_entropy_with_gradients");
      auto [loss, dhidden, dweight] =
          op.call(hidden, weight, targets, ignored, reduction, scale, need_hidden, need_weight);
      ctx->save_for_backward({dhidden, dweight});
      return loss;
    }
    static auto op =
        operation<decltype(loss_forward)>("attnres_b200::linear_cross_entropy_forward");
    auto [loss, kept, index, count, sums] =
        op.call(hidden, weight, targets, ignored, reduction, scale);
    ctx->save_for_backward({weight, targets, kept, index, count, sums});
    ctx->saved_data["ignored"] = ignored;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["scale"] = scale;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(6);
    const auto saved = ctx->get_saved_variables();
    auto& data = ctx->saved_data;
    const bool nh = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor dhidden, dweight;
    if (data["early"].toBool()) {
      static auto op = operation<decltype(loss_scale_gradient)>(
          "attnres_b200::linear_cross_entropy_scale_gradient");
      if (nh) dhidden = op.call(saved[0], grads[0]);
      if (nw) dweight = op.call(saved[1], grads[0]);
    } else {
      static auto op =
          operation<decltype(loss_backward)>("attnres_b200::linear_cross_entropy_backward");
      auto [dh, dw] = op.call(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4], saved[5],
                              data["ignored"].toInt(), data["reduction"].toInt(),
                              data["scale"].toDouble(), nh, nw);
      if (nh) dhidden = dh;
      if (nw) dweight = dw;
    }
    return once({dhidden, dweight, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor loss(const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignored,
            int64_t reduction, double scale);

Tensor loss_autograd(const Tensor& hidden, const Tensor& weight, const Tensor& targets,
                     int64_t ignored, int64_t reduction, double scale) {
  if (!differentiated({&hidden, &weight})) {
    static auto op = operation<decltype(loss)>("attnres_b200::linear_cross_entropy");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(hidden, weight, targets, ignored, reduction, scale);
  }
  return LinearCrossEntropy::apply(hidden, weight, targets, ignored, reduction, scale);
}

Tensor loss(const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignored,
            int64_t reduction, double scale) {
  return std::get<0>(loss_forward(hidden, weight, targets, ignored, reduction, scale));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(attnres_b200, m) {
  m.def("norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps, bool need_stats) -> (Tensor, Tensor)");
  m.def("norm_backward(Tensor grad, Tensor x, Tensor stats, Tensor? weight, ScalarType param_type, "
        "bool need_x, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)");
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("embedding_forward(Tensor tokens, Tensor table, Tensor? positions, float scale, "
        "ScalarType type) -> Tensor");
  m.def("embedding_backward(Tensor grad, Tensor tokens, SymInt vocabulary, ScalarType table_type, "
        "ScalarType position_type, float scale, int padding, bool need_table, bool need_positions) "
        "-> (Tensor, Tensor)");
  m.def("embed(Tensor tokens, Tensor table, Tensor? positions, float scale, int padding, "
        "ScalarType type) -> Tensor");
  m.def("linear_cross_entropy_forward(Tensor hidden, Tensor weight, Tensor targets, int ignored, "
        "int reduction, float scale) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("linear_cross_entropy_with_gradients(Tensor hidden, Tensor weight, Tensor targets, "
        "int ignored, int reduction, float scale, bool need_hidden, bool need_weight) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("linear_cross_entropy_scale_gradient(Tensor gradient, Tensor upstream) -> Tensor");
  m.def("linear_cross_entropy_backward(Tensor grad, Tensor weight, Tensor targets, Tensor kept, "
        "Tensor index, Tensor count, Tensor sums, int ignored, int reduction, float scale, "
        "bool need_hidden, bool need_weight) -> (Tensor, Tensor)");
  m.def("linear_cross_entropy(Tensor hidden, Tensor weight, Tensor targets, int ignored, "
        "int reduction, float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(attnres_b200, CUDA, m) {
  m.impl("norm_forward", norm_forward);
  m.impl("norm_backward", norm_backward);
  m.impl("layer_norm", layer_norm);
  m.impl("embedding_forward", embedding_forward);
  m.impl("embedding_backward", embedding_backward_sym);
  m.impl("embed", embed);
  m.impl("linear_cross_entropy_forward", loss_forward);
  m.impl("linear_cross_entropy_with_gradients", loss_with_gradients);
  m.impl("linear_cross_entropy_scale_gradient", loss_scale_gradient);
  m.impl("linear_cross_entropy_backward", loss_backward);
  m.impl("linear_cross_entropy", loss);
}

TORCH_LIBRARY_IMPL(attnres_b200, AutogradCUDA, m) {
  m.impl("layer_norm", layer_norm_autograd);
  m.impl("embed", embed_autograd);
  m.impl("linear_cross_entropy", loss_autograd);
}
