// The two ends of a language model as native torch operators, autograd included:
//   mmuon::linear_cross_entropy(x, weight, target, ignore_index, reduction, piece_tokens) -> loss
//   mmuon::embedding(index, weight, scale, padding_idx) -> out
// over the C ABI's mmuon_ce_* and mmuon_embedding_*.
//
// A loss that is a scalar makes its gradients in the forward, with the logits at hand, for a
// gradient of 1; the backward scales them by the one that arrives (on the device; nothing is
// touched where it is 1).  They are bf16 by then, so a factor that is no power of two rounds
// them a second time: kept in fp32 until the backward they would take twice the memory of dx
// and dw.  With a loss per token the backward knows each token's gradient only
// then, and makes the logits again.  The loss has no second derivative: what depends on its
// gradients raises when it is differentiated.  The table's gradient has one.
#include "torch_common.hpp"

#include <torch/csrc/autograd/engine.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include <tuple>

using namespace mmuon_torch;

namespace {

using Triple = std::tuple<Tensor, Tensor, Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void require_one_device(std::initializer_list<const Tensor*> ts) {
  const Tensor& first = **ts.begin();
  for (const Tensor* t : ts) {
    require_cuda(*t);
    TORCH_CHECK(t->device() == first.device(), "expected all tensors on one device, got ", first.device(), " and ",
                t->device());
  }
}

// Rows of 16-B chunks, not too far apart for the kernels' offsets: the tensor itself where its
// rows are such, else a copy
Tensor aligned_rows(const Tensor& t) {
  const bool rows = (t.size(1) <= 1 || t.stride(1) == 1) && t.stride(0) % 8 == 0 && t.stride(0) < (int64_t(1) << 22);
  return rows && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 ? t : dense_aligned(t);
}

// ---------------------------------------------------------------------------
// Cross entropy of a linear head
// ---------------------------------------------------------------------------
void check_head(const Tensor& x, const Tensor& w, const Tensor& target, int64_t reduction) {
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 2 && target.dim() == 1 && x.size(1) == w.size(1) &&
                        x.size(0) == target.size(0),
                    "expected x (T, D), weight (V, D) and target (T), got ", x.sizes(), ", ", w.sizes(), " and ",
                    target.sizes());
  TORCH_CHECK_VALUE(w.size(0) > 0 && w.size(1) > 0 && w.size(1) % 8 == 0,
                    "linear_cross_entropy needs a vocabulary of at least one token and a width that is a multiple of "
                    "8, got weight ", w.sizes());
  TORCH_CHECK_VALUE(reduction >= MMUON_CE_NONE && reduction <= MMUON_CE_SUM, "unknown reduction ", reduction);
  for (const Tensor* t : {&x, &w})
    TORCH_CHECK_TYPE(t->scalar_type() == at::kBFloat16, "linear_cross_entropy computes in bfloat16; ",
                     t == &x ? "x" : "weight", " is torch.", c10::getDtypeNames(t->scalar_type()).first,
                     " (run under torch.autocast(dtype=torch.bfloat16) or pass bf16 tensors)");
  TORCH_CHECK_TYPE(target.scalar_type() == at::kLong || target.scalar_type() == at::kInt,
                   "target must be int64 or int32, got torch.", c10::getDtypeNames(target.scalar_type()).first);
}

// Tokens of a piece: as asked, else as many as keep the codes of a piece (2 B per logit)
// within 1 GiB (256 at least), in whole 256-token tiles, and pieces of one size.  The loss
// alone has no codes: four times as many.  Several pieces keep fp32 sums of dw between them:
// where one piece of all tokens takes no more memory than those, it is one.
int64_t piece_of(int64_t tokens, int64_t width, int64_t vocab, int64_t asked, bool train, bool need_dw) {
  TORCH_CHECK_VALUE(asked >= 0, "piece_tokens must be positive, got ", asked);
  if (asked > 0) return std::min(asked, std::max<int64_t>(tokens, 1));
  const int64_t row = (vocab + 255) / 256 * 512;
  int64_t most = std::max<int64_t>(256, (int64_t(1) << 30) / row / 256 * 256);
  if (!train) most *= 4;
  if (tokens <= most) return std::max<int64_t>(tokens, 1);
  const int64_t pieces = (tokens + most - 1) / most;
  const int64_t piece = ((tokens + pieces - 1) / pieces + 255) / 256 * 256;
  // codes, gathered rows, statistics (8 B per 64 or 128 of the vocabulary)
  const int64_t each = row + 2 * width + row / 16;
  return train && need_dw && (tokens - piece) * each <= 4 * vocab * width ? tokens : piece;
}

struct HeadCall {
  Tensor x, w, target, grad, ws;
  mmuon_ce_args a{};
  HeadCall(const Tensor& x_, const Tensor& w_, const Tensor& target_, int64_t ignore_index, int64_t reduction,
           int64_t piece, bool train, bool need_dw)
      : x(aligned_rows(x_)), w(aligned_rows(w_)), target(target_.to(at::kLong).contiguous()) {
    a.tokens = x.size(0);
    a.vocab = w.size(0);
    TORCH_CHECK_VALUE(w.size(1) < (int64_t(1) << 22), "linear_cross_entropy: width ", w.size(1), " beyond 2^22");
    a.width = int32_t(w.size(1));
    a.dtype = MMUON_BF16;
    a.reduction = int32_t(reduction);
    a.ignore_index = ignore_index;
    a.x_stride = a.tokens > 1 ? x.stride(0) : a.width;
    a.w_stride = a.vocab > 1 ? w.stride(0) : a.width;
    a.piece_tokens = piece_of(a.tokens, a.width, a.vocab, piece, train, need_dw);
    a.x = x.const_data_ptr();
    a.w = w.const_data_ptr();
    a.target = static_cast<const int64_t*>(target.const_data_ptr());
  }
  void run(bool train) {
    ws = at::empty({std::max<int64_t>(int64_t(abi.ce_workspace(&a, train ? 1 : 0)), 256)}, x.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = size_t(ws.numel());
    check_rc(train ? abi.ce_fwd_bwd(&a, stream_of(x)) : abi.ce_fwd(&a, stream_of(x)),
             train ? "mmuon_ce_fwd_bwd" : "mmuon_ce_fwd");
  }
};

Tensor loss_impl(const Tensor& x, const Tensor& w, const Tensor& target, int64_t ignore_index, int64_t reduction,
                 int64_t piece) {
  check_head(x, w, target, reduction);
  require_one_device({&x, &w, &target});
  bind_library();
  const c10::DeviceGuard guard(x.device());
  HeadCall call(x, w, target, ignore_index, reduction, piece, false, false);
  const bool none = reduction == MMUON_CE_NONE;
  Tensor out = none ? at::empty({x.size(0)}, x.options().dtype(at::kFloat)) : at::empty({}, x.options().dtype(at::kFloat));
  (none ? call.a.nll : call.a.loss) = static_cast<float*>(out.data_ptr());
  call.run(false);
  return out;
}

// grad: d loss / d nll per token (fp32), or undefined: that of the reduction.
Triple grad_impl(const Tensor& x, const Tensor& w, const Tensor& target, const c10::optional<Tensor>& grad,
                 int64_t ignore_index, int64_t reduction, int64_t piece, bool need_dx, bool need_dw) {
  check_head(x, w, target, reduction);
  require_one_device({&x, &w, &target});
  TORCH_CHECK_VALUE(!grad.has_value() || (grad->dim() == 1 && grad->size(0) == x.size(0) &&
                                          grad->scalar_type() == at::kFloat && grad->device() == x.device()),
                    "grad must hold one float32 per token");
  bind_library();
  const c10::DeviceGuard guard(x.device());
  HeadCall call(x, w, target, ignore_index, reduction, piece, true, need_dw);
  const bool none = reduction == MMUON_CE_NONE;
  Tensor out = none ? at::empty({x.size(0)}, x.options().dtype(at::kFloat)) : at::empty({}, x.options().dtype(at::kFloat));
  (none ? call.a.nll : call.a.loss) = static_cast<float*>(out.data_ptr());
  Tensor dx = at::empty(need_dx ? x.sizes() : at::IntArrayRef{0}, x.options());
  Tensor dw = at::empty(need_dw ? w.sizes() : at::IntArrayRef{0}, w.options());
  if (grad.has_value()) {
    call.grad = grad->contiguous();
    call.a.grad = static_cast<const float*>(call.grad.const_data_ptr());
  }
  if (need_dx) call.a.dx = dx.data_ptr();
  if (need_dw) call.a.dw = dw.data_ptr();
  call.run(true);
  return {out, dx, dw};
}

// x and y *= factor (a float32 scalar on the device)
void scale_impl(const Tensor& x, const Tensor& y, const Tensor& factor) {
  for (const Tensor* t : {&x, &y}) {
    TORCH_CHECK_TYPE(t->scalar_type() == at::kBFloat16, "scale_ takes bfloat16 tensors");
    TORCH_CHECK_VALUE(t->is_contiguous() && t->numel() % 8 == 0, "scale_ takes contiguous tensors of whole 16-byte chunks");
  }
  TORCH_CHECK_VALUE(factor.numel() == 1 && factor.scalar_type() == at::kFloat, "scale_ takes one float32 factor");
  require_one_device({&x, &y, &factor});
  bind_library();
  const c10::DeviceGuard guard(x.device());
  check_rc(abi.scale(x.data_ptr(), x.numel(), y.data_ptr(), y.numel(),
                     static_cast<const float*>(factor.const_data_ptr()), stream_of(x)), "mmuon_scale_bf16");
}

Tensor call_loss(const Tensor& x, const Tensor& w, const Tensor& target, int64_t ignore_index, int64_t reduction,
                 int64_t piece) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::linear_cross_entropy", "")
                       .typed<Tensor(const Tensor&, const Tensor&, const Tensor&, int64_t, int64_t, int64_t)>();
  return op.call(x, w, target, ignore_index, reduction, piece);
}
Triple call_grad(const Tensor& x, const Tensor& w, const Tensor& target, const c10::optional<Tensor>& grad,
                 int64_t ignore_index, int64_t reduction, int64_t piece, bool need_dx, bool need_dw) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::linear_cross_entropy_grad", "")
                       .typed<Triple(const Tensor&, const Tensor&, const Tensor&, const c10::optional<Tensor>&, int64_t,
                                     int64_t, int64_t, bool, bool)>();
  return op.call(x, w, target, grad, ignore_index, reduction, piece, need_dx, need_dw);
}
void call_scale(const Tensor& x, const Tensor& y, const Tensor& factor) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::scale_", "")
                       .typed<void(const Tensor&, const Tensor&, const Tensor&)>();
  op.call(x, y, factor);
}

constexpr const char* NO_SECOND = "Trying to backward through mmuon.linear_cross_entropy_grad.default but no autograd "
                                  "formula was registered.";

// Gradients that the forward made, handed out by the current node of a graph that is kept
// (create_graph): they depend on the node's inputs and on the gradient that arrived, and a
// derivative along any of these raises.
void refuse_derivatives(std::initializer_list<Tensor*> made, const Tensor& arrived) {
  const std::shared_ptr<torch::autograd::Node> current = torch::autograd::get_current_node();
  TORCH_CHECK(current != nullptr, NO_SECOND);
  torch::autograd::edge_list edges = current->next_edges();
  edges.push_back(torch::autograd::impl::gradient_edge(arrived));
  const auto error = std::make_shared<torch::autograd::Error>(NO_SECOND, std::move(edges));
  for (Tensor* t : made) {
    if (t->numel() == 0) continue;  // not asked for
    *t = t->detach();
    torch::autograd::set_history(*t, error);
  }
}

struct LossFn : torch::autograd::Function<LossFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& target,
                        int64_t ignore_index, int64_t reduction, int64_t piece) {
    at::AutoDispatchBelowADInplaceOrView below;
    const bool dx = x.requires_grad(), dw = w.requires_grad();
    ctx->saved_data["dx"] = dx;
    ctx->saved_data["dw"] = dw;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["piece"] = piece;
    ctx->saved_data["spent"] = false;
    if (reduction == MMUON_CE_NONE) {
      ctx->save_for_backward({x, w, target});
      return call_loss(x, w, target, ignore_index, reduction, piece);
    }
    auto [loss, gx, gw] = call_grad(x, w, target, c10::nullopt, ignore_index, reduction, piece, dx, dw);
    ctx->save_for_backward({gx, gw});
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const bool dx = ctx->saved_data["dx"].toBool(), dw = ctx->saved_data["dw"].toBool();
    Tensor gx, gw;
    if (saved.size() == 3) {
      std::tie(std::ignore, gx, gw) =
          call_grad(saved[0], saved[1], saved[2], grads[0].to(at::kFloat), ctx->saved_data["ignore_index"].toInt(),
                    ctx->saved_data["reduction"].toInt(), ctx->saved_data["piece"].toInt(), dx, dw);
    } else {
      // the gradients were made by the forward and are handed over as they are
      TORCH_CHECK(!ctx->saved_data["spent"].toBool(),
                  "linear_cross_entropy hands its gradients over once: call it again for a second backward "
                  "(or use reduction=\"none\", whose backward computes them)");
      ctx->saved_data["spent"] = true;
      gx = saved[0];
      gw = saved[1];
      {
        at::AutoDispatchBelowADInplaceOrView below;
        call_scale(gx, gw, grads[0].to(at::kFloat));
      }
      if (at::GradMode::is_enabled()) refuse_derivatives({&gx, &gw}, grads[0]);
    }
    return {dx ? gx : Tensor(), dw ? gw : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// The gradient has no derivative of its own.
struct GradFn : torch::autograd::Function<GradFn> {
  static variable_list forward(AutogradContext*, const Tensor& x, const Tensor& w, const Tensor& target,
                               const c10::optional<Tensor>& grad, int64_t ignore_index, int64_t reduction,
                               int64_t piece, bool need_dx, bool need_dw) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, dx, dw] = call_grad(x, w, target, grad, ignore_index, reduction, piece, need_dx, need_dw);
    return {loss, dx, dw};
  }
  static variable_list backward(AutogradContext*, const variable_list&) { TORCH_CHECK(false, NO_SECOND); }
};

Triple grad_autograd(const Tensor& x, const Tensor& w, const Tensor& target, const c10::optional<Tensor>& grad,
                     int64_t ignore_index, int64_t reduction, int64_t piece, bool need_dx, bool need_dw) {
  if (any_requires_grad({&x, &w}) || (grad.has_value() && any_requires_grad({&*grad}))) {
    const variable_list r = GradFn::apply(x, w, target, grad, ignore_index, reduction, piece, need_dx, need_dw);
    return {r[0], r[1], r[2]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_grad(x, w, target, grad, ignore_index, reduction, piece, need_dx, need_dw);
}

Tensor loss_autograd(const Tensor& x, const Tensor& w, const Tensor& target, int64_t ignore_index, int64_t reduction,
                     int64_t piece) {
  if (any_requires_grad({&x, &w})) return LossFn::apply(x, w, target, ignore_index, reduction, piece);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_loss(x, w, target, ignore_index, reduction, piece);
}

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------
void check_ids(const Tensor& index) {
  TORCH_CHECK_TYPE(index.scalar_type() == at::kLong || index.scalar_type() == at::kInt,
                   "index must be int64 or int32, got torch.", c10::getDtypeNames(index.scalar_type()).first);
}
int32_t float_code(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, "embedding takes bfloat16 or "
                   "float32 tensors; ", name, " is torch.", c10::getDtypeNames(t.scalar_type()).first);
  return t.scalar_type() == at::kFloat ? MMUON_F32 : MMUON_BF16;
}
// Rows of consecutive elements
Tensor dense_rows(const Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }

Tensor embedding_impl(const Tensor& index, const Tensor& weight, double scale, int64_t padding_idx) {
  check_ids(index);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0 && weight.size(1) <= INT32_MAX,
                    "expected weight (V, D), got ", weight.sizes());
  TORCH_CHECK_VALUE(padding_idx < weight.size(0), "padding_idx ", padding_idx, " beyond ", weight.size(0), " rows");
  mmuon_embedding_args a{};
  a.dtype = float_code(weight, "weight");
  require_one_device({&weight, &index});
  bind_library();
  const c10::DeviceGuard guard(weight.device());
  const Tensor ids = index.to(at::kLong).contiguous(), w = dense_rows(weight);
  std::vector<int64_t> shape = index.sizes().vec();
  shape.push_back(w.size(1));
  Tensor out = at::empty(shape, w.options());
  a.tokens = ids.numel();
  a.vocab = w.size(0);
  a.width = int32_t(w.size(1));
  a.scale = float(scale);
  a.padding_idx = padding_idx;
  a.w_stride = a.vocab > 1 ? w.stride(0) : a.width;
  a.index = static_cast<const int64_t*>(ids.const_data_ptr());
  a.w = w.const_data_ptr();
  a.out = out.data_ptr();
  check_rc(abi.emb_fwd(&a, stream_of(w)), "mmuon_embedding_fwd");
  return out;
}

Tensor embedding_grad_impl(const Tensor& dout_, const Tensor& index, int64_t vocab, double scale, int64_t padding_idx) {
  check_ids(index);
  TORCH_CHECK_VALUE(vocab > 0 && padding_idx < vocab, "embedding: vocab ", vocab, ", padding_idx ", padding_idx);
  TORCH_CHECK_VALUE(dout_.dim() == index.dim() + 1 && dout_.sizes().slice(0, index.dim()) == index.sizes() &&
                        dout_.size(-1) > 0 && dout_.size(-1) <= INT32_MAX,
                    "dout ", dout_.sizes(), " does not match index ", index.sizes());
  mmuon_embedding_args a{};
  a.dtype = float_code(dout_, "dout");
  require_one_device({&dout_, &index});
  bind_library();
  const c10::DeviceGuard guard(dout_.device());
  const Tensor ids = index.to(at::kLong).contiguous();
  const Tensor dout = dense_rows(dout_.reshape({ids.numel(), dout_.size(-1)}));
  Tensor dw = at::empty({vocab, dout.size(1)}, dout.options());
  a.tokens = ids.numel();
  a.vocab = vocab;
  a.width = int32_t(dout.size(1));
  a.scale = float(scale);
  a.padding_idx = padding_idx;
  a.dout_stride = a.tokens > 1 ? dout.stride(0) : a.width;
  a.index = static_cast<const int64_t*>(ids.const_data_ptr());
  a.dout = dout.const_data_ptr();
  a.dw = dw.data_ptr();
  Tensor ws = at::empty({std::max<int64_t>(int64_t(abi.emb_workspace(&a)), 256)}, dout.options().dtype(at::kByte));
  a.workspace = ws.data_ptr();
  a.workspace_bytes = size_t(ws.numel());
  check_rc(abi.emb_bwd(&a, stream_of(dout)), "mmuon_embedding_bwd");
  return dw;
}

Tensor call_embedding(const Tensor& index, const Tensor& weight, double scale, int64_t padding_idx) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::embedding", "")
                       .typed<Tensor(const Tensor&, const Tensor&, double, int64_t)>();
  return op.call(index, weight, scale, padding_idx);
}
Tensor call_embedding_grad(const Tensor& dout, const Tensor& index, c10::SymInt vocab, double scale,
                           int64_t padding_idx) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::embedding_grad", "")
                       .typed<Tensor(const Tensor&, const Tensor&, c10::SymInt, double, int64_t)>();
  return op.call(dout, index, vocab, scale, padding_idx);
}
Tensor embedding_grad_sym(const Tensor& dout, const Tensor& index, c10::SymInt vocab, double scale,
                          int64_t padding_idx) {
  return embedding_grad_impl(dout, index, vocab.expect_int(), scale, padding_idx);
}

// The table's gradient is linear in the one that arrives: its derivative by that is the lookup
// in what arrives here, with zeros where a token took part in nothing.
struct EmbeddingGradFn : torch::autograd::Function<EmbeddingGradFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dout, const Tensor& index, c10::SymInt vocab, double scale,
                        int64_t padding_idx) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({index});
    ctx->saved_data["vocab"] = vocab;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding_idx"] = padding_idx;
    return call_embedding_grad(dout, index, vocab, scale, padding_idx);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const Tensor index = ctx->get_saved_variables()[0];
    const int64_t pad = ctx->saved_data["padding_idx"].toInt();
    const Tensor rows = call_embedding(index, grads[0], ctx->saved_data["scale"].toDouble(), -1);
    Tensor none = at::logical_or(index < 0, index >= at::Scalar(ctx->saved_data["vocab"].toSymInt()));
    if (pad >= 0) none = at::logical_or(none, index == pad);
    return {rows.masked_fill(none.unsqueeze(-1), 0), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor embedding_grad_autograd(const Tensor& dout, const Tensor& index, c10::SymInt vocab, double scale,
                               int64_t padding_idx) {
  if (any_requires_grad({&dout})) return EmbeddingGradFn::apply(dout, index, vocab, scale, padding_idx);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_embedding_grad(dout, index, std::move(vocab), scale, padding_idx);
}

struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& index, const Tensor& weight, double scale,
                        int64_t padding_idx) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({index});
    ctx->saved_data["vocab"] = weight.sym_size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding_idx"] = padding_idx;
    return call_embedding(index, weight, scale, padding_idx);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const Tensor index = ctx->get_saved_variables()[0];
    return {Tensor(),
            call_embedding_grad(grads[0], index, ctx->saved_data["vocab"].toSymInt(),
                                ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding_idx"].toInt()),
            Tensor(), Tensor()};
  }
};

Tensor embedding_autograd(const Tensor& index, const Tensor& weight, double scale, int64_t padding_idx) {
  if (any_requires_grad({&weight})) return EmbeddingFn::apply(index, weight, scale, padding_idx);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_embedding(index, weight, scale, padding_idx);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mmuon, m) {
  m.def("linear_cross_entropy(Tensor x, Tensor weight, Tensor target, int ignore_index, int reduction, int "
        "piece_tokens) -> Tensor", {at::Tag::pt2_compliant_tag});
  m.def("linear_cross_entropy_grad(Tensor x, Tensor weight, Tensor target, Tensor? grad, int ignore_index, int "
        "reduction, int piece_tokens, bool need_dx, bool need_dw) -> (Tensor, Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
  m.def("scale_(Tensor(a!) x, Tensor(b!) y, Tensor factor) -> ()", {at::Tag::pt2_compliant_tag});
  m.def("embedding(Tensor index, Tensor weight, float scale, int padding_idx) -> Tensor",
        {at::Tag::pt2_compliant_tag});
  m.def("embedding_grad(Tensor dout, Tensor index, SymInt vocab, float scale, int padding_idx) -> Tensor",
        {at::Tag::pt2_compliant_tag});
}
TORCH_LIBRARY_IMPL(mmuon, CompositeExplicitAutograd, m) {
  m.impl("linear_cross_entropy", loss_impl);
  m.impl("linear_cross_entropy_grad", grad_impl);
  m.impl("scale_", scale_impl);
  m.impl("embedding", embedding_impl);
  m.impl("embedding_grad", embedding_grad_sym);
}
TORCH_LIBRARY_IMPL(mmuon, Autograd, m) {
  m.impl("linear_cross_entropy", loss_autograd);
  m.impl("linear_cross_entropy_grad", grad_autograd);
  m.impl("embedding", embedding_autograd);
  m.impl("embedding_grad", embedding_grad_autograd);
}
