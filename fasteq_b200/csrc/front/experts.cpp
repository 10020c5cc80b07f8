// Dense layers with an epilogue, one matrix for all rows or one per expert, and the rows' way into the experts' order and back.
//
// Without its epilogue the layer is bilinear: with  P(x, w) = x w^T,  D(g, w) = g w,  W(g, x) = g^T x  (each over an expert's rows) the gradients of any of
// the three are the other two, so Product, ProductX and ProductW call one another and differentiate to every order.  The layer
// itself is one launch forward (which leaves act'(z) for the gradients) and one per gradient; where its gradients are to be differentiated
// it is taken apart into those and elementwise operations.
#include "front.h"

namespace front {
namespace {

enum Act : int64_t { kIdentity = 0, kSilu = 1, kTanh = 2, kSigmoid = 3, kAbs = 4 };

// Forward-mode differentiation is not offered.  Nodes refuse tangents by themselves; this is for where none is made, whatever the grad mode: no_grad does not
// switch it off.
void refuse_tangents(const char* name, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t && t->defined()) TORCH_CHECK(!t->_fw_grad(0).defined(), name, ": forward-mode differentiation is not supported");
}
const Tensor* pointer_of(const std::optional<Tensor>& t) { return t ? &*t : nullptr; }

// x [rows, K], w [experts, N, K]; offsets undefined: one matrix
fasteq_product_problem problem(const Tensor& x, const Tensor& w, int64_t inner, int64_t act) {
  fasteq_product_problem p{};
  p.dtype = w.scalar_type() == at::kDouble ? FASTEQ_F64 : FASTEQ_F32;
  p.experts = (int32_t)w.size(0); p.n = (int32_t)w.size(1); p.k = (int32_t)w.size(2);
  p.inner = (int32_t)inner; p.act = (int32_t)act; p.rows = x.size(0);
  return p;
}
const int32_t* offsets_of(const Tensor& offsets) { return offsets.defined() ? offsets.const_data_ptr<int32_t>() : nullptr; }

Tensor scratch_of(const fasteq_product_problem& p, bool backward, const Tensor& like) {
  int64_t need = 0;
  check(core.product_scratch(&p, backward, &need), "fasteq_product_scratch", core.last_cuda_error);
  return need ? at::empty({need}, like.options().dtype(at::kByte)) : Tensor();
}
int64_t bytes_of(const Tensor& t) { return t.defined() ? t.numel() : 0; }
// dense, and at an address the tensor-core kernels take
Tensor dense_rows(const Tensor& t) {
  if (!t.defined()) return t;
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 ? c.clone() : c;
}

// slope: receives act'(z) as the kernels keep it
Tensor run_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual, const Tensor& offsets, int64_t inner, int64_t act,
                   Tensor* slope) {
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor xc = dense_rows(x), wc = w.contiguous(), bc = defined_contiguous(bias), rc = defined_contiguous(residual);
  const auto p = problem(xc, wc, inner, act);
  const int64_t rows = xc.size(0), n = wc.size(1);
  Tensor y = at::empty({rows, n}, xc.options());
  if (slope) *slope = at::empty({rows, p.dtype == FASTEQ_F32 ? (n + 3) & ~(int64_t)3 : n}, xc.options());
  const Tensor scratch = scratch_of(p, false, xc);
  check(core.product_forward(&p, ptr(xc), ptr(wc), ptr(bc), ptr(rc), offsets_of(offsets), mptr(y), slope ? mptr(*slope) : nullptr, mptr(scratch),
                             bytes_of(scratch), stream_of(xc)),
        "fasteq_product_forward", core.last_cuda_error);
  return y;
}

// The gradients that are asked for, the others undefined.  w [experts, N, K] (only its extents without gx), x may be undefined without gw
variable_list run_backward(const Tensor& x, at::IntArrayRef shape, const Tensor& w, const Tensor& g, const Tensor& slope, const Tensor& offsets, int64_t inner,
                           bool need_x, bool need_w, bool need_b) {
  c10::cuda::CUDAGuard guard(g.device());
  const Tensor gc = dense_rows(g), xc = dense_rows(x), wc = defined_contiguous(w);
  fasteq_product_problem p{};
  p.dtype = gc.scalar_type() == at::kDouble ? FASTEQ_F64 : FASTEQ_F32;
  p.experts = (int32_t)shape[0]; p.n = (int32_t)shape[1]; p.k = (int32_t)shape[2]; p.inner = (int32_t)inner; p.rows = gc.size(0);
  p.act = slope.defined() ? (int32_t)kSilu : (int32_t)kIdentity;      // whether there is a slope is what counts here
  Tensor gx = need_x ? at::empty({gc.size(0), shape[2]}, gc.options()) : Tensor();
  Tensor gw = need_w || need_b ? at::empty(shape, gc.options()) : Tensor();
  Tensor gb = need_b ? at::empty({shape[0], shape[1]}, gc.options()) : Tensor();
  const Tensor scratch = scratch_of(p, true, gc);
  check(core.product_backward(&p, ptr(xc), ptr(wc), ptr(gc), ptr(slope), offsets_of(offsets), mptr(gx), mptr(gw), mptr(gb), mptr(scratch), bytes_of(scratch),
                              stream_of(gc)),
        "fasteq_product_backward", core.last_cuda_error);
  return {gx, need_w ? gw : Tensor(), gb};
}

Tensor product(const Tensor& x, const Tensor& w, const Tensor& offsets, int64_t inner);
Tensor product_x(const Tensor& g, const Tensor& w, const Tensor& offsets, int64_t inner);
Tensor product_w(const Tensor& g, const Tensor& x, const Tensor& offsets, int64_t inner, at::IntArrayRef shape);

// P(x, w), D(g, w), W(g, x) as nodes; which = 0, 1, 2
struct Bilinear : torch::autograd::Function<Bilinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& b, const std::optional<Tensor>& offsets, int64_t inner, int64_t which,
                        std::vector<int64_t> shape) {
    ctx->save_for_backward({a, b, offsets.value_or(Tensor())});
    ctx->saved_data["i"] = inner; ctx->saved_data["w"] = which;
    const Tensor o = offsets.value_or(Tensor());
    if (which == 0) return run_forward(a, b, Tensor(), Tensor(), o, inner, kIdentity, nullptr);
    if (which == 1) return run_backward(Tensor(), b.sizes(), b, a, Tensor(), o, inner, true, false, false)[0];
    return run_backward(b, shape, Tensor(), a, Tensor(), o, inner, false, true, false)[1];
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &a = saved[0], &b = saved[1], &o = saved[2], &h = go[0];
    const int64_t inner = ctx->saved_data["i"].toInt(), which = ctx->saved_data["w"].toInt();
    const bool need_a = ctx->needs_input_grad(0), need_b = ctx->needs_input_grad(1);
    Tensor da, db;
    if (which == 0) {                      // x, w
      if (need_a) da = product_x(h, b, o, inner);
      if (need_b) db = product_w(h, a, o, inner, b.sizes());
    } else if (which == 1) {               // g, w; h like x
      if (need_a) da = product(h, b, o, inner);
      if (need_b) db = product_w(a, h, o, inner, b.sizes());
    } else {                               // g, x; h like w
      if (need_a) da = product(b, h, o, inner);
      if (need_b) db = product_x(a, h, o, inner);
    }
    return {da, db, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
std::optional<Tensor> optional_of(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
Tensor product(const Tensor& x, const Tensor& w, const Tensor& offsets, int64_t inner) { return Bilinear::apply(x, w, optional_of(offsets), inner, (int64_t)0, std::vector<int64_t>()); }
Tensor product_x(const Tensor& g, const Tensor& w, const Tensor& offsets, int64_t inner) { return Bilinear::apply(g, w, optional_of(offsets), inner, (int64_t)1, std::vector<int64_t>()); }
Tensor product_w(const Tensor& g, const Tensor& x, const Tensor& offsets, int64_t inner, at::IntArrayRef shape) {
  return Bilinear::apply(g, x, optional_of(offsets), inner, (int64_t)2, shape.vec());
}

// The layer, in the caller's shapes: x [..., K], w [N, K] or [experts, N, K], bias [N] or [experts, N], residual like the result [..., N].  They are
// brought into the kernels' inside the node: views before it would be nodes of their own in the backward, a few microseconds each.
struct Layer : torch::autograd::Function<Layer> {
  static Tensor matrix(const Tensor& w) { return w.dim() == 2 ? w.unsqueeze(0) : w; }
  static Tensor vectors(const Tensor& b) { return b.defined() && b.dim() == 1 ? b.unsqueeze(0) : b; }
  static Tensor rows(const Tensor& t, int64_t width) {
    return !t.defined() || t.dim() == 2 ? t : t.reshape({c10::multiply_integers(t.sizes().begin(), t.sizes().end() - 1), width});
  }
  static Tensor run(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual, const Tensor& offsets, int64_t inner, int64_t act, Tensor* slope) {
    Tensor y = run_forward(rows(x, w.size(-1)), matrix(w), vectors(bias), rows(residual, w.size(-2)), offsets, inner, act, slope);
    if (x.dim() == 2) return y;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = w.size(-2);
    return y.view(shape);
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, const std::optional<Tensor>& residual,
                        const std::optional<Tensor>& offsets, int64_t inner, int64_t act, bool differentiated) {
    const Tensor b = bias.value_or(Tensor()), o = offsets.value_or(Tensor());
    Tensor slope;
    const Tensor y = run(x, w, b, residual.value_or(Tensor()), o, inner, act, differentiated && act != kIdentity ? &slope : nullptr);
    ctx->save_for_backward({x, w, b, o, slope});
    ctx->saved_data["i"] = inner; ctx->saved_data["a"] = act; ctx->saved_data["r"] = residual.has_value();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &o = saved[3], &slope = saved[4];
    const int64_t inner = ctx->saved_data["i"].toInt(), act = ctx->saved_data["a"].toInt();
    // the context numbers the tensors it was given, not the places they could have had
    const bool has_b = b.defined(), has_r = ctx->saved_data["r"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(2);
    refuse_tangents("dense layer", {&go[0]});
    Tensor gx, gw, gb;
    const Tensor gr = has_r && ctx->needs_input_grad(has_b ? 3 : 2) ? go[0] : Tensor();
    const Tensor g = rows(go[0], w.size(-2)), x2 = rows(x, w.size(-1)), w3 = matrix(w);
    if (at::GradMode::is_enabled()) {
      // to be differentiated again.  The bias and its gradient are products with a column of ones, which stay inside the experts' rows
      const Tensor b2 = vectors(b), ones = has_b ? at::ones({x2.size(0), 1}, x.options()) : Tensor();
      Tensor gz = g;
      if (act != kIdentity) {
        Tensor z = product(x2, w3, o, inner);
        if (has_b) z = z + product(ones, b2.unsqueeze(2), o, inner);
        if (act == kSilu) gz = silu_gradient(g.contiguous(), z.contiguous());
        else if (act == kTanh) gz = g * (1 - at::tanh(z).square());
        else if (act == kSigmoid) { const Tensor s = at::sigmoid(z); gz = g * (s * (1 - s)); }
        else gz = g * at::sgn(z).detach();
      }
      if (need_x) gx = product_x(gz, w3, o, inner);
      if (need_w) gw = product_w(gz, x2, o, inner, w3.sizes());
      if (need_b) gb = product_w(gz, ones, o, inner, {b2.size(0), b2.size(1), 1}).squeeze(2);
    } else {
      auto d = run_backward(x2, w3.sizes(), w3, g, slope, o, inner, need_x, need_w, need_b);
      gx = d[0]; gw = d[1]; gb = d[2];
    }
    auto shaped = [](const Tensor& t, const Tensor& like) { return t.defined() && t.dim() != like.dim() ? t.reshape(like.sizes()) : t; };
    return {shaped(gx, x), shaped(gw, w), shaped(gb, b), gr, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// CUDA tensors of one device and one type, float32 or float64
void check_operand(const char* name, const char* what, const Tensor& t, const Tensor& first) {
  if (!t.is_cuda()) TORCH_CHECK(false, name, ": ", what, " must be a CUDA tensor: fasteq_b200 has no CPU path");
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kDouble, name, ": only float32 and float64 are supported; ", what, " is ", t.scalar_type());
  TORCH_CHECK_VALUE(t.scalar_type() == first.scalar_type() && t.device() == first.device(), name, ": all operands must have one dtype and one device; ", what, " is ",
                    t.scalar_type(), " on ", t.device(), ", not ", first.scalar_type(), " on ", first.device());
}
void check_operand(const char* name, const char* what, const std::optional<Tensor>& t, const Tensor& first) {
  if (t) check_operand(name, what, *t, first);
}

// Whether a node is wanted of any of these.  Without one a call is about 2 us of host time shorter.
bool on_tape(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}

// extents that the C interface takes as 32-bit numbers
void check_extent(const char* name, const char* what, int64_t v, int64_t most = INT32_MAX) {
  TORCH_CHECK_VALUE(v <= most, name, ": ", what, " must be ", most, " at most, got ", v);
}

Tensor layer(const char* name, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, const std::optional<Tensor>& residual, const std::optional<Tensor>& offsets,
             int64_t inner, int64_t act) {
  check_extent(name, "channels", std::max(w.size(-1), w.size(-2)), FASTEQ_MAX_CHANNELS); check_extent(name, "rows of an entry", inner);
  refuse_tangents(name, {&x, &w, pointer_of(bias), pointer_of(residual)});
  if (!on_tape({&x, &w, pointer_of(bias), pointer_of(residual)}))
    return Layer::run(x, w, bias.value_or(Tensor()), residual.value_or(Tensor()), offsets.value_or(Tensor()), inner, act, nullptr);
  return Layer::apply(x, w, bias, residual, offsets, inner, act, on_tape({&x, &w, pointer_of(bias)}));
}

Tensor dense_act(const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, int64_t act, const std::optional<Tensor>& residual) {
  const char* name = "dense_act";
  check_operand(name, "x", x, x); check_operand(name, "weight", w, x); check_operand(name, "bias", bias, x); check_operand(name, "residual", residual, x);
  TORCH_CHECK_VALUE(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1), name, ": x [..., K] and weight [N, K] expected, got ", x.sizes(), " and ", w.sizes());
  TORCH_CHECK_VALUE(!bias || (bias->dim() == 1 && bias->size(0) == w.size(0)), name, ": bias must be [", w.size(0), "], got ", bias->sizes());
  if (residual) {
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = w.size(0);
    TORCH_CHECK_VALUE(residual->sizes() == shape, name, ": residual must have the result's shape ", shape, ", got ", residual->sizes());
  }
  return layer(name, x, w, bias, residual, std::nullopt, 1, act);
}

// ------------------------------------------------------------------------------------------------ experts' order
struct Order : torch::CustomClassHolder {
  Tensor position, offsets;              // [tokens, slots] and [experts + 1], int32
  int64_t experts, slots;
  uint32_t versions[2];
  Order(Tensor p, Tensor o)
      : position(std::move(p)), offsets(std::move(o)), experts(offsets.size(0) - 1), slots(position.size(1)), versions{position._version(), offsets._version()} {}
  // The kernels index with these, and a backward has to find them as its forward did; callers see them (as tensors of their own, which share the version).
  void check(const char* name) const {
    TORCH_CHECK(position._version() == versions[0] && offsets._version() == versions[1], name, ": the plan's position or offsets were changed in place since expert_plan made them");
  }
};
using OrderPtr = c10::intrusive_ptr<Order>;

int32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kDouble ? FASTEQ_F64 : FASTEQ_F32; }
int64_t width_of(const Tensor& t) { return c10::multiply_integers(t.sizes().begin() + 1, t.sizes().end()); }
std::vector<int64_t> with_rows(const Tensor& t, int64_t rows) {
  std::vector<int64_t> s = t.sizes().vec();
  s[0] = rows;
  return s;
}

Tensor run_gather(const Tensor& x, const Order& o) {
  o.check("expert_gather");
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor xc = x.contiguous();
  Tensor rows = at::empty(with_rows(x, x.size(0) * o.slots), xc.options());
  check(core.expert_gather(dtype_of(xc), ptr(xc), o.position.const_data_ptr<int32_t>(), o.offsets.const_data_ptr<int32_t>(), (int32_t)o.experts, xc.size(0),
                           (int32_t)o.slots, (int32_t)width_of(xc), mptr(rows), stream_of(xc)),
        "fasteq_expert_gather", core.last_cuda_error);
  return rows;
}
Tensor run_combine(const Tensor& rows, const Tensor& weight, const Order& o) {
  o.check("expert_combine");
  c10::cuda::CUDAGuard guard(rows.device());
  const Tensor rc = rows.contiguous(), wc = defined_contiguous(weight);
  const int64_t tokens = o.position.size(0);
  Tensor y = at::empty(with_rows(rows, tokens), rc.options());
  check(core.expert_combine(dtype_of(rc), ptr(rc), ptr(wc), o.position.const_data_ptr<int32_t>(), o.offsets.const_data_ptr<int32_t>(), (int32_t)o.experts, tokens,
                            (int32_t)o.slots, (int32_t)width_of(rc), mptr(y), stream_of(rc)),
        "fasteq_expert_combine", core.last_cuda_error);
  return y;
}
variable_list run_combine_backward(const Tensor& rows, const Tensor& weight, const Tensor& g, const Order& o, bool need_rows, bool need_weight) {
  o.check("expert_combine");
  c10::cuda::CUDAGuard guard(rows.device());
  const Tensor rc = rows.contiguous(), wc = defined_contiguous(weight), gc = g.contiguous();
  Tensor gr = need_rows ? at::empty_like(rc) : Tensor(), gw = need_weight ? at::empty(o.position.sizes(), rc.options()) : Tensor();
  check(core.expert_combine_backward(dtype_of(rc), ptr(rc), ptr(wc), ptr(gc), o.position.const_data_ptr<int32_t>(), o.offsets.const_data_ptr<int32_t>(),
                                     (int32_t)o.experts, o.position.size(0), (int32_t)o.slots, (int32_t)width_of(rc), mptr(gr), mptr(gw), stream_of(rc)),
        "fasteq_expert_combine_backward", core.last_cuda_error);
  return {gr, gw};
}

Tensor combine(const Tensor& rows, const std::optional<Tensor>& weight, const OrderPtr& o);

struct Gather : torch::autograd::Function<Gather> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OrderPtr& o) {
    ctx->saved_data["o"] = capsule(o);
    return run_gather(x, *o);
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    return {combine(go[0], std::nullopt, uncapsule<Order>(ctx->saved_data["o"])), Tensor()};
  }
};

// <rows[position[t, s]], g[t]>: bilinear as well
struct Dots : torch::autograd::Function<Dots> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& g, const OrderPtr& o) {
    ctx->save_for_backward({rows, g});
    ctx->saved_data["o"] = capsule(o);
    return run_combine_backward(rows, Tensor(), g, *o, false, true)[1];
  }
  static variable_list backward(AutogradContext* ctx, variable_list go);
};

// rows w[t, s] g[t], 0 for no expert
struct Spread : torch::autograd::Function<Spread> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& g, const OrderPtr& o) {
    o->check("expert_combine");
    ctx->save_for_backward({weight, g});
    ctx->saved_data["o"] = capsule(o);
    c10::cuda::CUDAGuard guard(g.device());
    const Tensor wc = weight.contiguous(), gc = g.contiguous();
    Tensor rows = at::empty(with_rows(g, o->position.numel()), gc.options());
    check(core.expert_combine_backward(dtype_of(gc), ptr(gc), ptr(wc), ptr(gc), o->position.const_data_ptr<int32_t>(), o->offsets.const_data_ptr<int32_t>(),
                                       (int32_t)o->experts, o->position.size(0), (int32_t)o->slots, (int32_t)width_of(gc), mptr(rows), nullptr, stream_of(gc)),
          "fasteq_expert_combine_backward", core.last_cuda_error);
    return rows;
  }
  static variable_list backward(AutogradContext* ctx, variable_list go);
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const std::optional<Tensor>& weight, const OrderPtr& o) {
    ctx->save_for_backward(weight ? variable_list{rows, *weight} : variable_list{});
    ctx->saved_data["o"] = capsule(o);
    return run_combine(rows, weight.value_or(Tensor()), *o);
  }
  static variable_list backward(AutogradContext* ctx, variable_list go) {
    const OrderPtr o = uncapsule<Order>(ctx->saved_data["o"]);
    const auto saved = ctx->get_saved_variables();
    const bool need_rows = ctx->needs_input_grad(0);
    if (saved.empty()) return {need_rows ? Tensor(Gather::apply(go[0], o)) : Tensor(), Tensor(), Tensor()};
    const Tensor &rows = saved[0], &weight = saved[1];
    const bool need_weight = ctx->needs_input_grad(1);
    if (at::GradMode::is_enabled())
      return {need_rows ? Tensor(Spread::apply(weight, go[0], o)) : Tensor(), need_weight ? Tensor(Dots::apply(rows, go[0], o)) : Tensor(), Tensor()};
    refuse_tangents("expert_combine", {&go[0]});
    auto d = run_combine_backward(rows, weight, go[0], *o, need_rows, need_weight);
    return {d[0], d[1], Tensor()};
  }
};
Tensor combine(const Tensor& rows, const std::optional<Tensor>& weight, const OrderPtr& o) { return Combine::apply(rows, weight, o); }

variable_list Dots::backward(AutogradContext* ctx, variable_list go) {
  const auto saved = ctx->get_saved_variables();
  const OrderPtr o = uncapsule<Order>(ctx->saved_data["o"]);
  return {ctx->needs_input_grad(0) ? Tensor(Spread::apply(go[0], saved[1], o)) : Tensor(),
          ctx->needs_input_grad(1) ? combine(saved[0], go[0], o) : Tensor(), Tensor()};
}
variable_list Spread::backward(AutogradContext* ctx, variable_list go) {
  const auto saved = ctx->get_saved_variables();
  const OrderPtr o = uncapsule<Order>(ctx->saved_data["o"]);
  return {ctx->needs_input_grad(0) ? Tensor(Dots::apply(go[0], saved[1], o)) : Tensor(),
          ctx->needs_input_grad(1) ? combine(go[0], saved[0], o) : Tensor(), Tensor()};
}

// expert [tokens, slots], int32 or int64, contiguous
OrderPtr make_order(const Tensor& expert, int64_t experts) {
  c10::cuda::CUDAGuard guard(expert.device());
  c10::InferenceMode ordinary(false);    // tensors made in inference mode have no version
  const auto ints = expert.options().dtype(at::kInt);
  Tensor position = at::empty(expert.sizes(), ints), offsets = at::empty({experts + 1}, ints);
  int64_t need = 0;
  check(core.expert_plan_scratch(expert.numel(), (int32_t)experts, &need), "fasteq_expert_plan_scratch", core.last_cuda_error);
  Tensor scratch = need ? at::empty({need}, expert.options().dtype(at::kByte)) : Tensor();
  check(core.expert_plan(ptr(expert), (int32_t)expert.element_size(), expert.numel(), (int32_t)experts, position.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(),
                         mptr(scratch), stream_of(expert)),
        "fasteq_expert_plan", core.last_cuda_error);
  return c10::make_intrusive<Order>(position, offsets);
}

// rows (or tokens) of a tensor that go with a plan
void check_rows(const char* name, const char* what, const Tensor& t, int64_t rows, const Order& o) {
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(0) == rows, name, ": ", what, " must have ", rows, " rows, got ", t.sizes());
  check_extent(name, "a row's values", width_of(t));
  TORCH_CHECK_VALUE(t.device() == o.offsets.device(), name, ": ", what, " is on ", t.device(), ", the plan on ", o.offsets.device());
}

Tensor expert_gather(const Tensor& x, const OrderPtr& o) {
  check_operand("expert_gather", "x", x, x);
  check_rows("expert_gather", "x", x, o->position.size(0), *o);
  refuse_tangents("expert_gather", {&x});
  return on_tape({&x}) ? Tensor(Gather::apply(x, o)) : run_gather(x, *o);
}

Tensor expert_combine(const Tensor& rows, const std::optional<Tensor>& weight, const OrderPtr& o) {
  const char* name = "expert_combine";
  check_operand(name, "rows", rows, rows); check_operand(name, "weight", weight, rows);
  check_rows(name, "rows", rows, o->position.numel(), *o);
  std::optional<Tensor> w = weight;
  if (w && w->dim() == 1 && o->slots == 1) w = w->unsqueeze(1);
  TORCH_CHECK_VALUE(!w || w->sizes() == o->position.sizes(), name, ": weight must be ", o->position.sizes(), ", got ", weight->sizes());
  refuse_tangents(name, {&rows, pointer_of(w)});
  return on_tape({&rows, pointer_of(w)}) ? combine(rows, w, o) : run_combine(rows, w.value_or(Tensor()), *o);
}

Tensor expert_dense(const Tensor& rows, const Tensor& w, const OrderPtr& o, const std::optional<Tensor>& bias, int64_t act) {
  const char* name = "expert_dense";
  o->check(name);
  check_operand(name, "rows", rows, rows); check_operand(name, "weight", w, rows); check_operand(name, "bias", bias, rows);
  check_rows(name, "rows", rows, o->position.numel(), *o);
  TORCH_CHECK_VALUE(rows.dim() >= 2 && w.dim() == 3 && w.size(0) == o->experts && w.size(2) == rows.size(-1), name, ": rows [rows, ..., K] and weight [", o->experts,
                    ", N, K] expected, got ", rows.sizes(), " and ", w.sizes());
  TORCH_CHECK_VALUE(!bias || (bias->dim() == 2 && bias->size(0) == w.size(0) && bias->size(1) == w.size(1)), name, ": bias must be [", w.size(0), ", ", w.size(1), "], got ",
                    bias->sizes());
  const int64_t inner = c10::multiply_integers(rows.sizes().begin() + 1, rows.sizes().end() - 1);
  return layer(name, rows, w, bias, std::nullopt, o->offsets, std::max<int64_t>(inner, 1), act);
}

OrderPtr expert_plan(const Tensor& expert, int64_t experts) {
  const char* name = "expert_plan";
  if (!expert.is_cuda()) TORCH_CHECK(false, name, ": expert must be a CUDA tensor: fasteq_b200 has no CPU path");
  TORCH_CHECK_VALUE(expert.scalar_type() == at::kInt || expert.scalar_type() == at::kLong, name, ": expert must be int32 or int64, got ", expert.scalar_type());
  TORCH_CHECK_VALUE(expert.dim() == 1 || (expert.dim() == 2 && expert.size(1) >= 1), name, ": expert must be [tokens] or [tokens, slots] with a slot at least, got ",
                    expert.sizes());
  TORCH_CHECK_VALUE(experts >= 1 && experts <= FASTEQ_MAX_EXPERTS, name, ": 1 to ", FASTEQ_MAX_EXPERTS, " experts are supported, got ", experts);
  return make_order((expert.dim() == 1 ? expert.unsqueeze(1) : expert).contiguous(), experts);
}

}  // namespace

void bind_experts(py::module_& m) {
  py::class_<Order, OrderPtr>(m, "ExpertOrder")
      .def_property_readonly("position", [](const Order& o) { return o.position.detach(); })
      .def_property_readonly("offsets", [](const Order& o) { return o.offsets.detach(); })
      .def_property_readonly("shape", [](const Order& o) { return std::make_tuple(o.position.size(0), o.slots, o.experts); });
  m.def("dense_act", &dense_act);
  m.def("expert_plan", &expert_plan);
  m.def("expert_gather", &expert_gather);
  m.def("expert_combine", &expert_combine);
  m.def("expert_dense", &expert_dense);
}

}  // namespace front
