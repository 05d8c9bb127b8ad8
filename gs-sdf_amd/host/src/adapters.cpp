// adapters.cpp — libtorch operators over the adapter entries of the C ABI (include/gsdf_hip.h: L1-L3).
#include "gsdf_adapters/gsdf_adapters.h"

#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "util.h"

namespace gsdf_adapters {
namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using gsdf_host::check;

int element_type(const Tensor &t, const char *name) {
  TORCH_CHECK(t.defined() && t.is_cuda(), name, ": expected a device tensor (the HIP path has no CPU fallback)");
  switch (t.scalar_type()) {
    case torch::kFloat32: return GSDF_F32;
    case torch::kFloat16: return GSDF_F16;
    case torch::kBFloat16: return GSDF_BF16;
    default: TORCH_CHECK(false, name, ": expected fp32, fp16 or bf16 elements, got ", t.scalar_type());
  }
}
void same_device(const Tensor &ref, const Tensor &t, const char *name) {
  TORCH_CHECK(t.defined() && t.device() == ref.device(), name, ": expected a tensor on ", ref.device());
}
void same(const Tensor &ref, const Tensor &t, const char *name, torch::ScalarType type) {
  same_device(ref, t, name);
  TORCH_CHECK(t.scalar_type() == type, name, ": expected ", type, " elements, got ", t.scalar_type());
}
// the tensor's memory holds what the tensor says (a lazily negated view, as conj().imag is one, holds the opposite)
Tensor plainly(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }
// a [rows, width] matrix whose rows are neighbours' elements: a view where the layout allows it
Tensor matrix(const Tensor &t) {
  Tensor m = plainly(t);
  if (m.dim() != 2) {
    const int64_t width = m.dim() ? m.size(-1) : 1;
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < m.dim(); ++i) rows *= m.size(i);
    m = m.reshape({rows, width});
  }
  return m.stride(1) == 1 || m.size(1) == 1 ? m : m.contiguous();
}
Tensor whole(const Tensor &t) {
  const Tensor p = plainly(t);
  return p.is_contiguous() ? p : p.contiguous();
}
Tensor index(const Tensor &ref, const Tensor &t, const char *name) {
  same_device(ref, t, name);
  TORCH_CHECK(t.scalar_type() == torch::kInt32 || t.scalar_type() == torch::kInt64, name, ": expected int32 or int64, got ", t.scalar_type());
  return whole(t);
}
void check_p(double p) { TORCH_CHECK(p >= 0.0 && p <= 1.0, "p: expected a probability in [0, 1], got ", p); }
void check_word(const Tensor &ref, const Offset &offset) {
  if (!offset.word) return;
  same(ref, *offset.word, "offset", torch::kInt64);
  TORCH_CHECK(offset.word->numel() == 1, "offset: expected one device word");
}
gsdf_stream_t stream_of(const Tensor &t) { return (gsdf_stream_t)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
bool wanted(const Tensor &t) { return t.defined() && t.requires_grad(); }
// a dual tensor asks for no gradient: its tangent would be lost without an error
void no_tangents(const char *name, std::initializer_list<const Tensor *> inputs) {
  for (const Tensor *t : inputs)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), name, ": no forward-mode derivatives (an input has a tangent)");
}
void *at_or_null(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes(const Tensor &ref, size_t n) { return torch::empty({(int64_t)n}, ref.options().dtype(torch::kUInt8).requires_grad(false)); }
Tensor plain(const Tensor &ref, at::IntArrayRef shape) { return torch::empty(shape, ref.options().requires_grad(false)); }

// A gradient that somebody wants to differentiate again (create_graph): that raises, instead of taking it for a constant.  `of`: what it depends on, so that the
// error lies on the way to every leaf behind it, also where torch.autograd.grad asks for that leaf alone.
Tensor once(const char *name, const Tensor &grad, variable_list of) {
  if (!torch::GradMode::is_enabled() || !grad.defined()) return grad;
  of.insert(of.begin(), grad.detach());
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + ": differentiable once only", (int64_t)of.size());
  return (*error)(std::move(of))[0];
}

// ---- L1 -------------------------------------------------------------------------------------------------------------------------------------
struct LowrankCall {
  Tensor ids, scales, word;
  int dtype;
  double p;
  uint64_t seed, offset;
};
gsdf_lowrank_args lowrank_args(const Tensor &x, const Tensor &a, const Tensor &b, const LowrankCall &c) {
  gsdf_lowrank_args r;
  r.rows = x.size(0); r.x_stride = x.stride(0);
  TORCH_CHECK(a.size(2) <= INT_MAX && b.size(1) <= INT_MAX, "lowrank_adapt: a projection ", a.size(2), " -> ", b.size(1), " is too wide");
  r.n_in = (int)a.size(2); r.n_out = (int)b.size(1); r.rank = (int)a.size(1); r.n_adapters = (int)a.size(0); r.dtype = c.dtype;
  r.ids_64 = c.ids.scalar_type() == torch::kInt64;
  r.x = x.data_ptr(); r.a = a.data_ptr(); r.b = b.data_ptr(); r.ids = c.ids.data_ptr();
  r.scales = (const float *)at_or_null(c.scales);
  r.p = c.p; r.seed = c.seed; r.offset = c.offset;
  r.offset_dev = (const uint64_t *)at_or_null(c.word);
  return r;
}
// -> the forward's saved buffer, if `training`
Tensor lowrank_run(const Tensor &x, const Tensor &a, const Tensor &b, const LowrankCall &c, const Tensor &base, const Tensor &y, bool training) {
  const c10::DeviceGuard guard(x.device());
  const gsdf_lowrank_args args = lowrank_args(x, a, b, c);
  const size_t n = gsdf_lowrank_fwd_ws_bytes(&args);
  TORCH_CHECK(n > 0, "lowrank_adapt: ", gsdf_last_error());
  const Tensor ws = bytes(x, n), save = training ? bytes(x, gsdf_lowrank_save_bytes(&args)) : Tensor();
  const Tensor m = base.defined() ? matrix(base) : Tensor();
  check(gsdf_lowrank_fwd(&args, at_or_null(m), m.defined() ? m.stride(0) : 0, y.data_ptr(), y.stride(0), at_or_null(save), ws.data_ptr(), stream_of(x)), "lowrank_adapt");
  return save;
}

struct LowrankFunction : public torch::autograd::Function<LowrankFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &a, const Tensor &b, const std::optional<Tensor> &base, const LowrankCall *c) {
    Tensor y = plain(x, {x.size(0), b.size(1)});
    const Tensor save = lowrank_run(x, a, b, *c, base.value_or(Tensor()), y, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, a, b, c->ids, c->scales, c->word, save});
    ctx->saved_data["dtype"] = (int64_t)c->dtype;
    ctx->saved_data["p"] = c->p;
    ctx->saved_data["seed"] = (int64_t)c->seed;
    ctx->saved_data["offset"] = (int64_t)c->offset;
    ctx->saved_data["base"] = base.has_value();
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &a = s[1], &b = s[2], &save = s[6], &dy = grads[0];
    if (!dy.defined()) return variable_list(5);
    LowrankCall c{s[3], s[4], s[5], (int)ctx->saved_data["dtype"].toInt(), ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
                  (uint64_t)ctx->saved_data["offset"].toInt()};
    no_tangents("lowrank_adapt's backward pass", {&dy});
    const bool need_x = ctx->needs_input_grad(0), need_a = ctx->needs_input_grad(1), need_b = ctx->needs_input_grad(2),
               need_base = ctx->saved_data["base"].toBool() && ctx->needs_input_grad(3);
    const Tensor dx = need_x ? plain(x, x.sizes()) : Tensor(), da = need_a ? plain(a, a.sizes()) : Tensor(), db = need_b ? plain(b, b.sizes()) : Tensor();
    if (need_x || need_a || need_b) {
      const c10::DeviceGuard guard(x.device());
      const gsdf_lowrank_args args = lowrank_args(x, a, b, c);
      const Tensor g = matrix(dy), ws = bytes(x, gsdf_lowrank_bwd_ws_bytes(&args));
      check(gsdf_lowrank_bwd(&args, g.data_ptr(), g.stride(0), save.data_ptr(), at_or_null(dx), need_x ? dx.stride(0) : 0, at_or_null(da), at_or_null(db),
                             ws.data_ptr(), stream_of(x)), "lowrank_adapt's backward pass");
    }
    return {once("lowrank_adapt", dx, {dy, a, b}), once("lowrank_adapt", da, {dy, x, b}), once("lowrank_adapt", db, {dy, x, a}), need_base ? dy : Tensor(), Tensor()};
  }
};

// checks what the C ABI cannot see; a, b become contiguous
LowrankCall lowrank_check(const Tensor &x, Tensor &a, Tensor &b, const Tensor &ids, const std::optional<Tensor> &scales, const Tensor &base, double p, uint64_t seed,
                          const Offset &offset) {
  LowrankCall c;
  c.dtype = element_type(x, "x");
  same(x, a, "a", x.scalar_type());
  same(x, b, "b", x.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && a.dim() == 3 && b.dim() == 3, "lowrank_adapt: expected x [..., k], a [g, r, k], b [g, n, r]");
  TORCH_CHECK(x.size(-1) == a.size(2) && b.size(0) == a.size(0) && b.size(2) == a.size(1), "lowrank_adapt: x ", x.sizes(), ", a ", a.sizes(), ", b ", b.sizes(),
              " do not fit (x [..., k], a [g, r, k], b [g, n, r])");
  TORCH_CHECK(a.size(1) >= 1 && a.size(1) <= GSDF_LOWRANK_MAX_RANK && a.size(0) >= 1 && a.size(0) <= GSDF_LOWRANK_MAX_ADAPTERS && a.size(2) >= 1 && b.size(1) >= 1,
              "lowrank_adapt: rank ", a.size(1), " outside [1, ", GSDF_LOWRANK_MAX_RANK, "], ", a.size(0), " adapters outside [1, ", GSDF_LOWRANK_MAX_ADAPTERS,
              "], or an empty projection ", a.size(2), " -> ", b.size(1));
  c.ids = index(x, ids, "ids");
  TORCH_CHECK(ids.sizes() == x.sizes().slice(0, x.dim() - 1), "ids: expected shape ", x.sizes().slice(0, x.dim() - 1), ", got ", ids.sizes());
  if (scales) {
    same(x, *scales, "scales", torch::kFloat32);
    TORCH_CHECK(scales->dim() == 1 && scales->size(0) == a.size(0), "scales: expected shape [", a.size(0), "], got ", scales->sizes());
    no_tangents("lowrank_adapt", {&*scales});
    TORCH_CHECK(!(scales->requires_grad() && torch::GradMode::is_enabled()), "scales: constants, no gradient is offered for them");
    c.scales = whole(*scales);
  }
  if (base.defined()) {
    same(x, base, "base", x.scalar_type());
    TORCH_CHECK(base.dim() == x.dim() && base.size(-1) == b.size(1) && base.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1), "base: shape ",
                base.sizes(), " does not fit x ", x.sizes(), " and b ", b.sizes());
  }
  check_p(p);
  check_word(x, offset);
  c.p = p; c.seed = seed; c.offset = offset.number;
  if (offset.word) c.word = *offset.word;
  no_tangents("lowrank_adapt", {&x, &a, &b, &base});
  a = whole(a);
  b = whole(b);
  return c;
}

// y, written in place, and something the call reads: apart, or columns of one buffer that do not meet (t's rows y's stride apart, or one row between two of y's)
void share_nothing(const Tensor &y, const Tensor &t, const char *name) {
  if (y.numel() == 0 || !t.defined() || t.numel() == 0) return;
  const int64_t es = (int64_t)y.element_size(), et = (int64_t)t.element_size(), rows = y.size(0), n = y.size(1) * es, stride = y.stride(0) * es;
  const bool matrix = t.dim() == 2;      // (anything else is contiguous)
  const int64_t rows_t = matrix ? t.size(0) : 1, k = (matrix ? t.size(1) : t.numel()) * et, stride_t = matrix ? t.stride(0) * et : 0;
  const char *py = (const char *)y.data_ptr(), *pt = (const char *)t.data_ptr();
  if (py + (rows - 1) * stride + n <= pt || pt + (rows_t - 1) * stride_t + k <= py) return;
  if (rows > 1 && (rows_t == 1 || stride_t == stride)) {
    const int64_t by = ((pt - py) % stride + stride) % stride;
    if (by >= n && by + k <= stride) return;
  }
  TORCH_CHECK(false, "lowrank_adapt_: y and ", name, " share memory");
}

// ---- L2 -------------------------------------------------------------------------------------------------------------------------------------
struct DropoutCall {
  Tensor word;
  int dtype;
  double p;
  uint64_t seed, offset;
};
Tensor dropout_run(const Tensor &x, const Tensor &residual, const DropoutCall &c) {
  const c10::DeviceGuard guard(x.device());
  Tensor y = plain(x, x.sizes());
  const Tensor m = matrix(x), r = residual.defined() ? matrix(residual) : Tensor();
  check(gsdf_dropout(m.size(0), m.size(1), c.dtype, m.data_ptr(), m.stride(0), at_or_null(r), r.defined() ? r.stride(0) : 0, c.p, c.seed, c.offset,
                     (const uint64_t *)at_or_null(c.word), y.data_ptr(), m.size(1), stream_of(x)), "dropout");
  return y;
}
struct DropoutFunction : public torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &residual, const DropoutCall *c) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({c->word});
    ctx->saved_data["dtype"] = (int64_t)c->dtype;
    ctx->saved_data["p"] = c->p;
    ctx->saved_data["seed"] = (int64_t)c->seed;
    ctx->saved_data["offset"] = (int64_t)c->offset;
    ctx->saved_data["residual"] = residual.has_value();
    return dropout_run(x, residual.value_or(Tensor()), *c);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const Tensor &dy = grads[0];
    if (!dy.defined()) return variable_list(3);
    no_tangents("dropout's backward pass", {&dy});
    const DropoutCall c{ctx->get_saved_variables()[0], (int)ctx->saved_data["dtype"].toInt(), ctx->saved_data["p"].toDouble(),
                        (uint64_t)ctx->saved_data["seed"].toInt(), (uint64_t)ctx->saved_data["offset"].toInt()};
    return {ctx->needs_input_grad(0) ? once("dropout", dropout_run(dy, Tensor(), c), {dy}) : Tensor(),
            ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1) ? dy : Tensor(), Tensor()};
  }
};

// ---- L3 -------------------------------------------------------------------------------------------------------------------------------------
struct BalanceCall {
  Tensor ids, mask;
  int64_t k;
  int dtype;
};
std::tuple<Tensor, Tensor, Tensor> balance_run(const Tensor &m, const BalanceCall &c) {
  const c10::DeviceGuard guard(m.device());
  const int64_t e = m.size(1);
  const auto options = m.options().requires_grad(false);
  Tensor loss = torch::empty({}, options.dtype(torch::kFloat32)), counts = torch::empty({e}, options.dtype(torch::kInt64)),
         pull = torch::empty({e}, options.dtype(torch::kFloat32));
  const Tensor ws = bytes(m, gsdf_router_balance_ws_bytes(m.size(0), (int)e));
  check(gsdf_router_balance_fwd(m.size(0), (int)e, (int)c.k, c.dtype, m.data_ptr(), m.stride(0), c.ids.data_ptr(), c.ids.scalar_type() == torch::kInt64,
                                (const uint8_t *)at_or_null(c.mask), loss.data_ptr<float>(), counts.data_ptr<int64_t>(), pull.data_ptr<float>(), ws.data_ptr(),
                                stream_of(m)), "router_balance");
  return {loss, counts, pull};
}
struct BalanceFunction : public torch::autograd::Function<BalanceFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &m, const BalanceCall *c) {
    auto [loss, counts, pull] = balance_run(m, *c);
    ctx->save_for_backward({m, c->mask, pull});
    ctx->saved_data["dtype"] = (int64_t)c->dtype;
    ctx->mark_non_differentiable({counts});
    ctx->set_materialize_grads(false);      // (of the counts neither: zeros that nobody reads)
    return {loss, counts};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &m = s[0], &mask = s[1], &pull = s[2];
    if (!grads[0].defined()) return variable_list(2);
    no_tangents("router_balance's backward pass", {&grads[0]});
    const c10::DeviceGuard guard(m.device());
    const Tensor v = whole(grads[0].to(torch::kFloat32)), out = plain(m, {m.size(0), m.size(1)});
    check(gsdf_router_balance_bwd(m.size(0), (int)m.size(1), (int)ctx->saved_data["dtype"].toInt(), m.data_ptr(), m.stride(0), (const uint8_t *)at_or_null(mask),
                                  pull.data_ptr<float>(), v.data_ptr<float>(), out.data_ptr(), stream_of(m)), "router_balance's backward pass");
    return {once("router_balance", out, {grads[0], m}), Tensor()};
  }
};

}  // namespace

Tensor lowrank_adapt(const Tensor &x, const Tensor &a_, const Tensor &b_, const Tensor &ids, const std::optional<Tensor> &scales, const std::optional<Tensor> &base_,
                     double p, uint64_t seed, const Offset &offset) {
  Tensor a = a_, b = b_, base = base_ ? *base_ : Tensor();
  const LowrankCall c = lowrank_check(x, a, b, ids, scales, base, p, seed, offset);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = b.size(1);
  if (torch::GradMode::is_enabled() && (wanted(x) || wanted(a) || wanted(b) || wanted(base))) {
    const Tensor m = matrix(x);      // (out here: what the node saves keeps its history)
    if (x.dim() == 2) return LowrankFunction::apply(m, a, b, base_, &c);
    return LowrankFunction::apply(m, a, b, base_ ? std::optional<Tensor>(matrix(base)) : base_, &c).view(shape);
  }
  const Tensor m = matrix(x), y = plain(x, shape);
  lowrank_run(m, a, b, c, base, y.dim() == 2 ? y : y.view({m.size(0), b.size(1)}), false);
  return y;
}

void lowrank_adapt_(const Tensor &y, const Tensor &x, const Tensor &a_, const Tensor &b_, const Tensor &ids, const std::optional<Tensor> &scales) {
  Tensor a = a_, b = b_;
  const LowrankCall c = lowrank_check(x, a, b, ids, scales, y, 0.0, 0, {});
  TORCH_CHECK(!(torch::GradMode::is_enabled() && (wanted(y) || wanted(x) || wanted(a) || wanted(b))), "lowrank_adapt_: no gradients in place; use lowrank_adapt");
  TORCH_CHECK(!y.is_neg(), "lowrank_adapt_: y is a lazily negated view");
  TORCH_CHECK(!y.is_inference() || c10::InferenceMode::is_enabled(), "lowrank_adapt_: y is an inference tensor, outside inference mode");
  const Tensor out = y.dim() == 2 ? y : y.view({c.ids.numel(), b.size(1)});
  TORCH_CHECK(out.stride(1) == 1 || out.size(1) == 1, "lowrank_adapt_: the elements of a row of y have to be neighbours");
  TORCH_CHECK(out.size(0) <= 1 || out.stride(0) >= out.size(1), "lowrank_adapt_: the rows of y overlap");
  const Tensor m = matrix(x);
  share_nothing(out, m, "x");
  share_nothing(out, a, "a");
  share_nothing(out, b, "b");
  share_nothing(out, c.ids, "ids");
  share_nothing(out, c.scales, "scales");
  lowrank_run(m, a, b, c, out, out, false);
  y.unsafeGetTensorImpl()->bump_version();
}

Tensor dropout(const Tensor &x, double p, uint64_t seed, const Offset &offset, const std::optional<Tensor> &residual_) {
  DropoutCall c;
  c.dtype = element_type(x, "x");
  check_p(p);
  check_word(x, offset);
  c.p = p; c.seed = seed; c.offset = offset.number;
  if (offset.word) c.word = *offset.word;
  const Tensor residual = residual_ ? *residual_ : Tensor();
  if (residual.defined()) {
    same(x, residual, "residual", x.scalar_type());
    TORCH_CHECK(residual.sizes() == x.sizes(), "residual: expected shape ", x.sizes(), ", got ", residual.sizes());
  }
  no_tangents("dropout", {&x, &residual});
  if (torch::GradMode::is_enabled() && (wanted(x) || wanted(residual))) return DropoutFunction::apply(x, residual_, &c);
  return dropout_run(x, residual, c);
}

std::tuple<Tensor, Tensor> router_balance(const Tensor &logits, const Tensor &ids, const std::optional<Tensor> &mask) {
  BalanceCall c;
  c.dtype = element_type(logits, "logits");
  no_tangents("router_balance", {&logits});
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) <= GSDF_ROUTER_MAX_EXPERTS, "logits: expected [..., e] with 1 to ", GSDF_ROUTER_MAX_EXPERTS,
              " experts, got ", logits.sizes());
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  c.ids = index(logits, ids, "ids");
  const bool one = ids.sizes() == lead;
  TORCH_CHECK(one || (ids.dim() == logits.dim() && ids.sizes().slice(0, ids.dim() - 1) == lead), "ids: expected shape ", lead, " or that and the choices of a row, got ",
              ids.sizes());
  c.k = one ? 1 : ids.size(-1);
  TORCH_CHECK(c.k >= 1 && c.k <= logits.size(-1), "ids: ", c.k, " choices of ", logits.size(-1), " experts");
  if (mask) {
    same_device(logits, *mask, "mask");
    TORCH_CHECK((mask->scalar_type() == torch::kBool || mask->scalar_type() == torch::kUInt8) && mask->sizes() == lead, "mask: expected bool or uint8 of shape ", lead,
                ", got ", mask->scalar_type(), " ", mask->sizes());
    c.mask = whole(*mask);
  }
  if (torch::GradMode::is_enabled() && wanted(logits)) {
    const variable_list r = BalanceFunction::apply(matrix(logits), &c);
    return {r[0], r[1]};
  }
  auto [loss, counts, pull] = balance_run(matrix(logits), c);
  return {loss, counts};
}

}  // namespace gsdf_adapters
