// What stands between a decoder layer's Monarch projections, as native torch operators, autograd
// included:
//   mmuon::rms_norm(x, residual, weight, eps) -> (y, h, inv)
//   mmuon::rms_norm_fp8(x, residual, weight, eps, dtype, group) -> (codes, scale, h)
//   mmuon::rotary(q, k, table, positions, interleaved, back) -> (q, k)
//   mmuon::differential_attention(q, k, v, lam, lengths, starts, causal, scale, save) -> (o, o1, o2, lse)
// over the C ABI's mmuon_norm_*, mmuon_rotary and mmuon_attention_*.
//
// The norm's and the attention's gradients have no derivative of their own; the rotation's is a
// rotation, to any order.
#include "torch_common.hpp"

#include <array>
#include <string>
#include <tuple>

using namespace mmuon_torch;

namespace {

using Pair = std::tuple<Tensor, Tensor>;
using Triple = std::tuple<Tensor, Tensor, Tensor>;
using OptionalTensor = c10::optional<Tensor>;
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

// The shape of a result that is not wanted
const std::array<int64_t, 1> NOTHING = {0};
const at::IntArrayRef NONE = NOTHING;

std::string name_of(const Tensor& t) { return c10::getDtypeNames(t.scalar_type()).first; }

int32_t float_code(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, op, " takes bfloat16 or float32 "
                   "tensors; ", name, " is torch.", name_of(t));
  return t.scalar_type() == at::kFloat ? MMUON_F32 : MMUON_BF16;
}

// ---------------------------------------------------------------------------
// Norm
// ---------------------------------------------------------------------------
// (rows, width), each row's elements side by side
Tensor rows_of(const Tensor& t) {
  const Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.size(1) <= 1 || r.stride(1) == 1 ? r : r.contiguous();
}
int64_t row_stride(const Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }

mmuon_norm_args norm_args(const char* op, const Tensor& x, const OptionalTensor& residual, const Tensor& w, double eps) {
  mmuon_norm_args a{};
  a.dtype = float_code(x, op, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0 && w.dim() == 1 && w.size(0) == x.size(-1),
                    "expected x (..., D) and weight (D), got ", x.sizes(), " and ", w.sizes());
  a.w_dtype = float_code(w, op, "weight");
  TORCH_CHECK_TYPE(a.w_dtype == a.dtype || a.w_dtype == MMUON_F32, op, ": weight must be float32 or x's type, got torch.",
                   name_of(w), " with torch.", name_of(x));
  if (residual.has_value()) {
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "residual ", residual->sizes(), " is not of x's shape ", x.sizes());
    TORCH_CHECK_TYPE(residual->scalar_type() == x.scalar_type(), op, ": residual must be of x's type, got torch.",
                     name_of(*residual), " with torch.", name_of(x));
  }
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
  TORCH_CHECK_VALUE(x.size(-1) <= (a.dtype == MMUON_BF16 ? 32768 : 16384), op, ": width ", x.size(-1), " beyond ",
                    a.dtype == MMUON_BF16 ? 32768 : 16384);
  require_one_device({&x, residual.has_value() ? &*residual : &x, &w});
  a.out_dtype = a.dtype;
  a.width = int32_t(x.size(-1));
  a.rows = x.numel() / a.width;
  a.eps = float(eps);
  return a;
}

Triple rms_norm_impl(const Tensor& x_, const OptionalTensor& residual, const Tensor& weight, double eps) {
  mmuon_norm_args a = norm_args("rms_norm", x_, residual, weight, eps);
  bind_library();
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows_of(x_), r = residual.has_value() ? rows_of(*residual) : Tensor(), w = weight.contiguous();
  Tensor y = at::empty(x_.sizes(), x.options());
  Tensor h = at::empty(residual.has_value() ? x_.sizes() : NONE, x.options());
  Tensor inv = at::empty({a.rows}, x.options().dtype(at::kFloat));
  a.x_stride = row_stride(x);
  a.x = x.const_data_ptr();
  a.w = w.const_data_ptr();
  if (r.defined()) {
    a.residual_stride = row_stride(r);
    a.residual = r.const_data_ptr();
    a.h = h.data_ptr();
  }
  a.y = y.data_ptr();
  a.inv = static_cast<float*>(inv.data_ptr());
  check_rc(abi.norm_fwd(&a, stream_of(x)), "mmuon_norm_fwd");
  return {y, h, inv};
}

// h: what was normalised; dh: the gradient of h beside that through y
Pair rms_norm_grad_impl(const Tensor& h_, const Tensor& inv, const Tensor& weight, const Tensor& dy_,
                        const OptionalTensor& dh_, bool need_dw) {
  mmuon_norm_args a = norm_args("rms_norm", h_, c10::nullopt, weight, 0.0);
  TORCH_CHECK_VALUE(inv.dim() == 1 && inv.size(0) == a.rows && inv.scalar_type() == at::kFloat && inv.is_contiguous(),
                    "inv must hold one float32 per row");
  for (const Tensor* t : {&dy_, dh_.has_value() ? &*dh_ : &dy_}) {
    TORCH_CHECK_VALUE(t->sizes() == h_.sizes() && t->scalar_type() == h_.scalar_type(), "the gradient of rms_norm's "
                      "output must be of its shape and type");
    require_one_device({&h_, &inv, t});
  }
  bind_library();
  const c10::DeviceGuard guard(h_.device());
  const Tensor h = rows_of(h_), dy = rows_of(dy_), dh = dh_.has_value() ? rows_of(*dh_) : Tensor(), w = weight.contiguous();
  Tensor dx = at::empty(h_.sizes(), h.options());
  Tensor dw = at::empty(need_dw ? weight.sizes() : NONE, w.options());
  a.x = h.const_data_ptr();
  a.x_stride = row_stride(h);
  a.w = w.const_data_ptr();
  a.inv = const_cast<float*>(static_cast<const float*>(inv.const_data_ptr()));
  a.dy = dy.const_data_ptr();
  a.dy_stride = row_stride(dy);
  if (dh.defined()) {
    a.dh = dh.const_data_ptr();
    a.dh_stride = row_stride(dh);
  }
  a.dx = dx.data_ptr();
  Tensor ws;
  if (need_dw) {
    a.dw = dw.data_ptr();
    ws = at::empty({std::max<int64_t>(int64_t(abi.norm_workspace(&a)), 256)}, h.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = size_t(ws.numel());
  }
  check_rc(abi.norm_bwd(&a, stream_of(h)), "mmuon_norm_bwd");
  return {dx, dw};
}

Triple rms_norm_fp8_impl(const Tensor& x_, const OptionalTensor& residual, const Tensor& weight, double eps,
                         at::ScalarType dtype, int64_t group) {
  TORCH_CHECK_TYPE(dtype == at::kFloat8_e4m3fn || dtype == at::kFloat8_e5m2, "rms_norm_fp8 gives float8_e4m3fn or "
                   "float8_e5m2, not torch.", c10::getDtypeNames(dtype).first);
  TORCH_CHECK_VALUE(group == 128 || group == 0, "group must be 128 columns or None, got ", group);
  mmuon_norm_args a = norm_args("rms_norm_fp8", x_, residual, weight, eps);
  bind_library();
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows_of(x_), r = residual.has_value() ? rows_of(*residual) : Tensor(), w = weight.contiguous();
  std::vector<int64_t> shape = x_.sizes().vec();
  shape.back() = group == 0 ? 1 : (a.width + 127) / 128;
  Tensor codes = at::empty(x_.sizes(), x.options().dtype(dtype));
  Tensor scale = at::empty(shape, x.options().dtype(at::kFloat));
  Tensor h = at::empty(residual.has_value() ? x_.sizes() : NONE, x.options());
  a.out_dtype = dtype == at::kFloat8_e4m3fn ? MMUON_F8E4M3 : MMUON_F8E5M2;
  a.group = int32_t(group);
  a.x_stride = row_stride(x);
  a.x = x.const_data_ptr();
  a.w = w.const_data_ptr();
  if (r.defined()) {
    a.residual_stride = row_stride(r);
    a.residual = r.const_data_ptr();
    a.h = h.data_ptr();
  }
  a.y = codes.data_ptr();
  a.scale = static_cast<float*>(scale.data_ptr());
  check_rc(abi.norm_fwd(&a, stream_of(x)), "mmuon_norm_fwd");
  return {codes, scale, h};
}

Triple call_norm(const Tensor& x, const OptionalTensor& residual, const Tensor& w, double eps) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::rms_norm", "")
                       .typed<Triple(const Tensor&, const OptionalTensor&, const Tensor&, double)>();
  return op.call(x, residual, w, eps);
}
Pair call_norm_grad(const Tensor& h, const Tensor& inv, const Tensor& w, const Tensor& dy, const OptionalTensor& dh,
                    bool need_dw) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::rms_norm_grad", "")
                       .typed<Pair(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptionalTensor&, bool)>();
  return op.call(h, inv, w, dy, dh, need_dw);
}
Triple call_norm_fp8(const Tensor& x, const OptionalTensor& residual, const Tensor& w, double eps, at::ScalarType dtype,
                     int64_t group) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::rms_norm_fp8", "")
                       .typed<Triple(const Tensor&, const OptionalTensor&, const Tensor&, double, at::ScalarType, int64_t)>();
  return op.call(x, residual, w, eps, dtype, group);
}

bool wants(const OptionalTensor& t) { return t.has_value() && any_requires_grad({&*t}); }

struct NormFn : torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptionalTensor& residual, const Tensor& w,
                               double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, h, inv] = call_norm(x, residual, w, eps);
    ctx->set_materialize_grads(false);
    ctx->saved_data["dx"] = x.requires_grad();
    ctx->saved_data["dr"] = residual.has_value() && residual->requires_grad();
    ctx->saved_data["dw"] = w.requires_grad();
    if (residual.has_value()) {
      ctx->mark_non_differentiable({inv});
      ctx->save_for_backward({h, inv, w});
    } else {
      ctx->mark_non_differentiable({h, inv});
      ctx->save_for_backward({x, inv, w});
    }
    return {y, h, inv};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const bool dx = ctx->saved_data["dx"].toBool(), dr = ctx->saved_data["dr"].toBool(), dw = ctx->saved_data["dw"].toBool();
    const Tensor dy = grads[0].defined() ? grads[0] : at::zeros_like(saved[0]);
    auto [gx, gw] = call_norm_grad(saved[0], saved[1], saved[2], dy, grads[1].defined() ? OptionalTensor(grads[1]) : c10::nullopt, dw);
    return {dx ? gx : Tensor(), dr ? gx : Tensor(), dw ? gw : Tensor(), Tensor()};
  }
};

struct NormGradFn : torch::autograd::Function<NormGradFn> {
  static variable_list forward(AutogradContext*, const Tensor& h, const Tensor& inv, const Tensor& w, const Tensor& dy,
                               const OptionalTensor& dh, bool need_dw) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dx, dw] = call_norm_grad(h, inv, w, dy, dh, need_dw);
    return {dx, dw};
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "Trying to backward through mmuon.rms_norm_grad.default but no autograd formula was registered.");
  }
};

Triple norm_autograd(const Tensor& x, const OptionalTensor& residual, const Tensor& w, double eps) {
  if (any_requires_grad({&x, &w}) || wants(residual)) {
    const variable_list r = NormFn::apply(x, residual, w, eps);
    return {r[0], r[1], r[2]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_norm(x, residual, w, eps);
}
Pair norm_grad_autograd(const Tensor& h, const Tensor& inv, const Tensor& w, const Tensor& dy, const OptionalTensor& dh,
                        bool need_dw) {
  if (any_requires_grad({&h, &inv, &w, &dy}) || wants(dh)) {
    const variable_list r = NormGradFn::apply(h, inv, w, dy, dh, need_dw);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_norm_grad(h, inv, w, dy, dh, need_dw);
}
Triple norm_fp8_autograd(const Tensor& x, const OptionalTensor& residual, const Tensor& w, double eps,
                         at::ScalarType dtype, int64_t group) {
  TORCH_CHECK(!any_requires_grad({&x, &w}) && !wants(residual), "rms_norm_fp8 has no gradient: call it under "
              "torch.no_grad(), or rms_norm where one is wanted");
  at::AutoDispatchBelowADInplaceOrView below;
  return call_norm_fp8(x, residual, w, eps, dtype, group);
}

// ---------------------------------------------------------------------------
// Rotary positions
// ---------------------------------------------------------------------------
Pair rotary_impl(const Tensor& q_, const Tensor& k_, const Tensor& table_, const OptionalTensor& positions,
                 bool interleaved, bool back) {
  mmuon_rotary_args a{};
  a.dtype = float_code(q_, "rotary", "q");
  TORCH_CHECK_TYPE(k_.scalar_type() == q_.scalar_type(), "rotary: q and k must be of one type, got torch.", name_of(q_),
                   " and torch.", name_of(k_));
  TORCH_CHECK_VALUE(q_.dim() == 4 && k_.dim() == 4 && q_.size(0) == k_.size(0) && q_.size(1) == k_.size(1) &&
                        q_.size(3) == k_.size(3),
                    "expected q (B, T, H, D) and k (B, T, K, D), got ", q_.sizes(), " and ", k_.sizes());
  TORCH_CHECK_TYPE(table_.scalar_type() == at::kFloat, "rotary: the table must be float32, got torch.", name_of(table_));
  TORCH_CHECK_VALUE(table_.dim() == 2 && table_.size(1) >= 2 && table_.size(1) % 2 == 0 && table_.size(1) <= q_.size(3) &&
                        q_.size(3) <= 65536,
                    "expected a table (positions, columns that are rotated) of an even number of at most ", q_.size(3),
                    " columns, got ", table_.sizes());
  TORCH_CHECK_VALUE(q_.numel() == 0 || table_.size(0) > 0, "rotary: a table of no positions");
  const int64_t B = q_.size(0), T = q_.size(1);
  Tensor at_;
  if (positions.has_value()) {
    TORCH_CHECK_TYPE(positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt,
                     "positions must be int64 or int32, got torch.", name_of(*positions));
    TORCH_CHECK_VALUE((positions->dim() == 1 && positions->size(0) == T) ||
                          (positions->dim() == 2 && positions->size(0) == B && positions->size(1) == T),
                      "positions must be (T) or (B, T) = (", B, ", ", T, "), got ", positions->sizes());
  }
  require_one_device({&q_, &k_, &table_, positions.has_value() ? &*positions : &table_});
  bind_library();
  const c10::DeviceGuard guard(q_.device());
  const auto heads = [](const Tensor& t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); };
  const Tensor q = heads(q_), k = heads(k_), table = table_.contiguous();
  if (positions.has_value()) at_ = positions->to(at::kLong).expand({B, T}).contiguous();
  Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
  a.batch = B;
  a.tokens = T;
  TORCH_CHECK_VALUE(q.size(2) <= INT32_MAX && k.size(2) <= INT32_MAX, "rotary: too many heads");
  a.q_heads = int32_t(q.size(2));
  a.k_heads = int32_t(k.size(2));
  a.dim = int32_t(q.size(3));
  a.part = int32_t(table.size(1));
  a.interleaved = interleaved;
  a.table_rows = table.size(0);
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = q.stride(i);
    a.k_stride[i] = k.stride(i);
  }
  a.q = q.const_data_ptr();
  a.k = k.const_data_ptr();
  a.table = static_cast<const float*>(table.const_data_ptr());
  if (at_.defined()) a.positions = static_cast<const int64_t*>(at_.const_data_ptr());
  a.q_out = qo.data_ptr();
  a.k_out = ko.data_ptr();
  check_rc(abi.rotary(&a, back ? 1 : 0, stream_of(q)), "mmuon_rotary");
  return {qo, ko};
}

Pair call_rotary(const Tensor& q, const Tensor& k, const Tensor& table, const OptionalTensor& positions, bool interleaved,
                 bool back) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::rotary", "")
                       .typed<Pair(const Tensor&, const Tensor&, const Tensor&, const OptionalTensor&, bool, bool)>();
  return op.call(q, k, table, positions, interleaved, back);
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& table,
                               const OptionalTensor& positions, bool interleaved, bool back) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->saved_data["q"] = q.requires_grad();
    ctx->saved_data["k"] = k.requires_grad();
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["back"] = back;
    if (positions.has_value()) ctx->save_for_backward({table, *positions});
    else ctx->save_for_backward({table});
    auto [qo, ko] = call_rotary(q, k, table, positions, interleaved, back);
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    auto [dq, dk] = call_rotary(grads[0], grads[1], saved[0], saved.size() > 1 ? OptionalTensor(saved[1]) : c10::nullopt,
                                ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["back"].toBool());
    return {ctx->saved_data["q"].toBool() ? dq : Tensor(), ctx->saved_data["k"].toBool() ? dk : Tensor(),
            Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Pair rotary_autograd(const Tensor& q, const Tensor& k, const Tensor& table, const OptionalTensor& positions,
                     bool interleaved, bool back) {
  TORCH_CHECK(!any_requires_grad({&table}), "rotary: the table has no gradient");
  if (any_requires_grad({&q, &k})) {
    const variable_list r = RotaryFn::apply(q, k, table, positions, interleaved, back);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_rotary(q, k, table, positions, interleaved, back);
}

// ---------------------------------------------------------------------------
// Differential attention
// ---------------------------------------------------------------------------
// Heads of 16-B chunks, tokens not too far apart for the kernels' offsets: the tensor itself where
// it is such, else a copy
Tensor aligned_heads(const Tensor& t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
  ok = ok && (t.size(1) <= 1 || t.stride(1) < (int64_t(1) << 22));
  return ok ? t : dense_aligned(t);
}
void take_strides(const Tensor& t, int64_t (&to)[3]) {
  for (int i = 0; i < 3; ++i) to[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

struct AttentionCall {
  Tensor q, k, v, lam, lengths, starts, ws;
  mmuon_attention_args a{};
  c10::DeviceGuard guard;
  AttentionCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& lam_, const OptionalTensor& lengths_,
                const OptionalTensor& starts_, bool causal, double scale)
      : guard((check(q_, k_, v_, lam_, lengths_, starts_, scale), q_.device())) {
    q = aligned_heads(q_), k = aligned_heads(k_), v = aligned_heads(v_);
    lam = lam_.size(0) <= 1 || lam_.stride(0) <= 1 ? lam_ : lam_.contiguous();
    a.batch = int32_t(q.size(0));
    a.queries = int32_t(q.size(1));
    a.keys = int32_t(k.size(1));
    a.heads = int32_t(q.size(2) / 2);
    a.kv_heads = int32_t(v.size(2));
    a.dim = int32_t(q.size(3));
    a.dtype = MMUON_BF16;
    a.causal = causal;
    a.scale = float(scale);
    a.lam_stride = a.heads > 1 ? int32_t(lam.stride(0)) : 0;
    take_strides(q, a.q_stride);
    take_strides(k, a.k_stride);
    take_strides(v, a.v_stride);
    a.q = q.const_data_ptr();
    a.k = k.const_data_ptr();
    a.v = v.const_data_ptr();
    a.lam = static_cast<const float*>(lam.const_data_ptr());
    if (lengths_.has_value()) {
      lengths = lengths_->to(at::kLong).contiguous();
      a.lengths = static_cast<const int64_t*>(lengths.const_data_ptr());
    }
    if (starts_.has_value()) {
      starts = starts_->to(at::kLong).contiguous();
      a.starts = static_cast<const int64_t*>(starts.const_data_ptr());
    }
  }
  static void check(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const OptionalTensor& lengths,
                    const OptionalTensor& starts, double scale) {
    const char* names[3] = {"q", "k", "v"};
    const Tensor* ts[3] = {&q, &k, &v};
    for (int i = 0; i < 3; ++i)
      TORCH_CHECK_TYPE(ts[i]->scalar_type() == at::kBFloat16, "differential_attention computes in bfloat16; ", names[i],
                       " is torch.", name_of(*ts[i]), " (run under torch.autocast(dtype=torch.bfloat16) or pass bf16 tensors)");
    TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4 && k.size(0) == q.size(0) && v.size(0) == q.size(0) &&
                          v.size(1) == k.size(1) && k.size(3) == q.size(3) && v.size(3) == 2 * q.size(3) &&
                          k.size(2) == 2 * v.size(2) && v.size(2) > 0 && q.size(2) % (2 * v.size(2)) == 0,
                      "expected q (B, T, 2 H, D), k (B, S, 2 K, D) and v (B, S, K, 2 D) with H a multiple of K, got ",
                      q.sizes(), ", ", k.sizes(), " and ", v.sizes());
    TORCH_CHECK_VALUE(q.size(3) >= 8 && q.size(3) <= 128 && q.size(3) % 8 == 0,
                      "differential_attention needs heads of a multiple of 8 columns, at most 128, got ", q.size(3));
    for (int i = 0; i < 3; ++i)
      TORCH_CHECK_VALUE(q.size(i) <= INT32_MAX && k.size(i) <= INT32_MAX, "differential_attention: sizes beyond 2^31");
    TORCH_CHECK_TYPE(lam.scalar_type() == at::kFloat, "lam must be float32, got torch.", name_of(lam));
    TORCH_CHECK_VALUE(lam.dim() == 1 && lam.size(0) == q.size(2) / 2, "lam must hold one value, or one for each of ",
                      q.size(2) / 2, " heads, got ", lam.sizes());
    TORCH_CHECK_VALUE(scale > 0 && scale <= 3.4e38, "scale must be positive and finite, got ", scale);
    for (const OptionalTensor* t : {&lengths, &starts}) {
      if (!t->has_value()) continue;
      const char* name = t == &lengths ? "lengths" : "starts";
      TORCH_CHECK_TYPE((*t)->scalar_type() == at::kLong || (*t)->scalar_type() == at::kInt, name,
                       " must be int64 or int32, got torch.", name_of(**t));
      TORCH_CHECK_VALUE((*t)->dim() == 1 && (*t)->size(0) == q.size(0), name, " must hold one value per sequence, got ",
                        (*t)->sizes());
    }
    require_one_device({&q, &k, &v, &lam, lengths.has_value() ? &*lengths : &q, starts.has_value() ? &*starts : &q});
    bind_library();
  }
  void workspace(bool backward) {
    ws = at::empty({std::max<int64_t>(int64_t(abi.attention_workspace(&a, backward ? 1 : 0)), 256)}, q.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = size_t(ws.numel());
  }
};

using Quad = std::tuple<Tensor, Tensor, Tensor, Tensor>;

Quad attention_impl(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const OptionalTensor& lengths,
                    const OptionalTensor& starts, bool causal, double scale, bool save) {
  AttentionCall call(q, k, v, lam, lengths, starts, causal, scale);
  mmuon_attention_args& a = call.a;
  const std::array<int64_t, 4> shape = {a.batch, a.queries, a.heads, 2 * a.dim};
  const at::IntArrayRef kept = save ? at::IntArrayRef(shape) : NONE;
  Tensor o = at::empty(shape, call.q.options()), o1 = at::empty(kept, call.q.options().dtype(at::kFloat)), o2 = at::empty(kept, o1.options());
  Tensor lse = save ? at::empty({a.batch, a.heads, a.queries, 4}, call.q.options().dtype(at::kFloat))
                    : at::empty(NONE, call.q.options().dtype(at::kFloat));
  a.o = o.data_ptr();
  if (save) {
    a.o1 = static_cast<float*>(o1.data_ptr());
    a.o2 = static_cast<float*>(o2.data_ptr());
    a.lse = static_cast<float*>(lse.data_ptr());
  }
  call.workspace(false);
  check_rc(abi.attention_fwd(&a, stream_of(call.q)), "mmuon_attention_fwd");
  return {o, o1, o2, lse};
}

// need_q: dq and dlam; need_kv: dk and dv
Quad attention_grad_impl(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const OptionalTensor& lengths,
                         const OptionalTensor& starts, const Tensor& o1, const Tensor& o2, const Tensor& lse,
                         const Tensor& dout_, bool causal, double scale, bool need_q, bool need_kv) {
  AttentionCall call(q, k, v, lam, lengths, starts, causal, scale);
  mmuon_attention_args& a = call.a;
  const std::array<int64_t, 4> shape = {a.batch, a.queries, a.heads, 2 * a.dim}, four = {a.batch, a.heads, a.queries, 4};
  TORCH_CHECK_VALUE(dout_.sizes() == at::IntArrayRef(shape) && dout_.scalar_type() == at::kBFloat16,
                    "the gradient of differential_attention's output must be bfloat16 and of its shape, got ", dout_.sizes());
  for (const Tensor* t : {&o1, &o2})
    TORCH_CHECK_VALUE(t->sizes() == at::IntArrayRef(shape) && t->scalar_type() == at::kFloat, "o1 and o2 must be the forward's");
  require_one_device({&q, &o1, &o2, &dout_});
  TORCH_CHECK_VALUE(lse.sizes() == at::IntArrayRef(four) && lse.scalar_type() == at::kFloat && lse.is_contiguous(),
                    "lse must be the forward's");
  require_one_device({&q, &lse});
  const Tensor dout = dense_aligned(dout_), p1 = dense_aligned(o1), p2 = dense_aligned(o2);
  Tensor dq = at::empty(need_q ? q.sizes() : NONE, call.q.options());
  Tensor dlam = at::empty(need_q ? lam.sizes() : NONE, lam.options());
  Tensor dk = at::empty(need_kv ? k.sizes() : NONE, call.q.options());
  Tensor dv = at::empty(need_kv ? v.sizes() : NONE, call.q.options());
  a.o1 = const_cast<float*>(static_cast<const float*>(p1.const_data_ptr()));
  a.o2 = const_cast<float*>(static_cast<const float*>(p2.const_data_ptr()));
  a.lse = const_cast<float*>(static_cast<const float*>(lse.const_data_ptr()));
  a.dout = dout.const_data_ptr();
  if (need_q) {
    a.dq = dq.data_ptr();
    a.dlam = static_cast<float*>(dlam.data_ptr());
  }
  if (need_kv) {
    a.dk = dk.data_ptr();
    a.dv = dv.data_ptr();
  }
  call.workspace(true);
  check_rc(abi.attention_bwd(&a, stream_of(call.q)), "mmuon_attention_bwd");
  return {dq, dk, dv, dlam};
}

Quad call_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const OptionalTensor& lengths,
                    const OptionalTensor& starts, bool causal, double scale, bool save) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::differential_attention", "")
                       .typed<Quad(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptionalTensor&,
                                   const OptionalTensor&, bool, double, bool)>();
  return op.call(q, k, v, lam, lengths, starts, causal, scale, save);
}
Quad call_attention_grad(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const OptionalTensor& lengths,
                         const OptionalTensor& starts, const Tensor& o1, const Tensor& o2, const Tensor& lse,
                         const Tensor& dout, bool causal, double scale, bool need_q, bool need_kv) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("mmuon::differential_attention_grad", "")
                       .typed<Quad(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptionalTensor&,
                                   const OptionalTensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, bool,
                                   double, bool, bool)>();
  return op.call(q, k, v, lam, lengths, starts, o1, o2, lse, dout, causal, scale, need_q, need_kv);
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam,
                               const OptionalTensor& lengths, const OptionalTensor& starts, bool causal, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, o1, o2, lse] = call_attention(q, k, v, lam, lengths, starts, causal, scale, true);
    ctx->saved_data["q"] = q.requires_grad();
    ctx->saved_data["k"] = k.requires_grad();
    ctx->saved_data["v"] = v.requires_grad();
    ctx->saved_data["lam"] = lam.requires_grad();
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->save_for_backward({q, k, v, lam, lengths.has_value() ? *lengths : Tensor(), starts.has_value() ? *starts : Tensor(),
                            o1, o2, lse});
    ctx->mark_non_differentiable({o1, o2, lse});
    return {o, o1, o2, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    const auto given = [](const Tensor& t) { return t.defined() ? OptionalTensor(t) : c10::nullopt; };
    const bool q = ctx->saved_data["q"].toBool(), k = ctx->saved_data["k"].toBool(), v = ctx->saved_data["v"].toBool(),
               lam = ctx->saved_data["lam"].toBool();
    auto [dq, dk, dv, dlam] = call_attention_grad(s[0], s[1], s[2], s[3], given(s[4]), given(s[5]), s[6], s[7], s[8], grads[0],
                                                  ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(),
                                                  q || lam, k || v);
    return {q ? dq : Tensor(), k ? dk : Tensor(), v ? dv : Tensor(), lam ? dlam : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct AttentionGradFn : torch::autograd::Function<AttentionGradFn> {
  static variable_list forward(AutogradContext*, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam,
                               const OptionalTensor& lengths, const OptionalTensor& starts, const Tensor& o1, const Tensor& o2,
                               const Tensor& lse, const Tensor& dout, bool causal, double scale, bool need_q, bool need_kv) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dq, dk, dv, dlam] = call_attention_grad(q, k, v, lam, lengths, starts, o1, o2, lse, dout, causal, scale, need_q, need_kv);
    return {dq, dk, dv, dlam};
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "Trying to backward through mmuon.differential_attention_grad.default but no autograd formula was "
                "registered.");
  }
};

Quad attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const OptionalTensor& lengths,
                        const OptionalTensor& starts, bool causal, double scale, bool save) {
  if (any_requires_grad({&q, &k, &v, &lam})) {
    const variable_list r = AttentionFn::apply(q, k, v, lam, lengths, starts, causal, scale);
    return {r[0], r[1], r[2], r[3]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_attention(q, k, v, lam, lengths, starts, causal, scale, save);
}
Quad attention_grad_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const OptionalTensor& lengths,
                             const OptionalTensor& starts, const Tensor& o1, const Tensor& o2, const Tensor& lse,
                             const Tensor& dout, bool causal, double scale, bool need_q, bool need_kv) {
  if (any_requires_grad({&q, &k, &v, &lam, &o1, &o2, &lse, &dout})) {
    const variable_list r = AttentionGradFn::apply(q, k, v, lam, lengths, starts, o1, o2, lse, dout, causal, scale, need_q, need_kv);
    return {r[0], r[1], r[2], r[3]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_attention_grad(q, k, v, lam, lengths, starts, o1, o2, lse, dout, causal, scale, need_q, need_kv);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mmuon, m) {
  m.def("rms_norm(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
  m.def("rms_norm_grad(Tensor h, Tensor inv, Tensor weight, Tensor dy, Tensor? dh, bool need_dw) -> (Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
  m.def("rms_norm_fp8(Tensor x, Tensor? residual, Tensor weight, float eps, ScalarType dtype, int group) -> (Tensor, "
        "Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
  m.def("rotary(Tensor q, Tensor k, Tensor table, Tensor? positions, bool interleaved, bool back) -> (Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
  m.def("differential_attention(Tensor q, Tensor k, Tensor v, Tensor lam, Tensor? lengths, Tensor? starts, bool causal, "
        "float scale, bool save) -> (Tensor, Tensor, Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
  m.def("differential_attention_grad(Tensor q, Tensor k, Tensor v, Tensor lam, Tensor? lengths, Tensor? starts, Tensor o1, "
        "Tensor o2, Tensor lse, Tensor dout, bool causal, float scale, bool need_q, bool need_kv) -> (Tensor, Tensor, "
        "Tensor, Tensor)", {at::Tag::pt2_compliant_tag});
}
TORCH_LIBRARY_IMPL(mmuon, CompositeExplicitAutograd, m) {
  m.impl("rms_norm", rms_norm_impl);
  m.impl("rms_norm_grad", rms_norm_grad_impl);
  m.impl("rms_norm_fp8", rms_norm_fp8_impl);
  m.impl("rotary", rotary_impl);
  m.impl("differential_attention", attention_impl);
  m.impl("differential_attention_grad", attention_grad_impl);
}
TORCH_LIBRARY_IMPL(mmuon, Autograd, m) {
  m.impl("rms_norm", norm_autograd);
  m.impl("rms_norm_grad", norm_grad_autograd);
  m.impl("rms_norm_fp8", norm_fp8_autograd);
  m.impl("rotary", rotary_autograd);
  m.impl("differential_attention", attention_autograd);
  m.impl("differential_attention_grad", attention_grad_autograd);
}
