// PyTorch side of the row operators: argument checks, output allocation and autograd nodes around the C entry points
// blh_layer_norm_*, blh_row_dropout and blh_residual_norm_* (host code only; bilinear_amd/row_ops.py loads it).
//
// Why C++ and not ctypes as the lifter's path: these calls are short — at a few hundred rows the kernels take 5-10 us —
// and autograd runs a backward node on its device thread, where a Python node starts with cold caches.  Measured with
// ctypes and a Python autograd.Function: forward + backward of a 64 x 1024 layer norm 143 us, without a gradient 12.6; with
// these nodes 56-62 us (23.3 with single-threaded autograd; the kernels are 8) and 4.3-5.  A node of three gradients that
// does nothing takes 41 (12.8).
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <optional>
#include <tuple>
#include <vector>

#include "../../include/bilinear_hip.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Optional;

// ---- checks ---------------------------------------------------------------------------------------------------------

const char* name_of(at::ScalarType t) { return c10::toString(t); }

int32_t code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return BLH_F32;
    case at::kBFloat16: return BLH_BF16;
    default: return BLH_F16;
  }
}

void check_rows(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), "bilinear_amd row operators run only on a HIP device (MI355X); ", what, " is on '", t.device(),
              "' and there is no CPU/ATen fallback.");
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::kFloat || s == at::kBFloat16 || s == at::kHalf, what, " must be float32, bfloat16 or float16, got ",
              name_of(s));
  TORCH_CHECK(t.layout() == at::kStrided, what, " must be a dense (strided) tensor");
  TORCH_CHECK(t.dim() >= 1 && t.size(-1) >= 1, what, " needs a last axis of at least one column, got shape ", t.sizes());
}

void check_like(const Tensor& t, const Tensor& x, const char* what, bool or_float) {
  TORCH_CHECK(t.device() == x.device(), what, " is on '", t.device(), "' where '", x.device(), "' is expected");
  TORCH_CHECK(t.sizes() == x.sizes(), what, " has shape ", t.sizes(), " where ", x.sizes(), " is expected");
  TORCH_CHECK(t.scalar_type() == x.scalar_type() || (or_float && t.scalar_type() == at::kFloat), what, " is ",
              name_of(t.scalar_type()), " where ", name_of(x.scalar_type()), or_float ? " or Float" : "", " is expected");
}

void check_param(const Tensor& x, const Optional& t, const char* what) {
  if (!t) return;
  TORCH_CHECK(t->device() == x.device(), what, " is on '", t->device(), "' where '", x.device(), "' is expected");
  TORCH_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), what, " has shape ", t->sizes(), " where [", x.size(-1),
              "] is expected");
  TORCH_CHECK(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat, what, " is ",
              name_of(t->scalar_type()), " where Float or ", name_of(x.scalar_type()), " is expected");
}

// the type of weight and bias (fp32 where neither is given)
int32_t check_params(const Tensor& x, const Optional& weight, const Optional& bias) {
  check_param(x, weight, "weight");
  check_param(x, bias, "bias");
  TORCH_CHECK(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "weight is ",
              weight ? name_of(weight->scalar_type()) : "", " and bias ", bias ? name_of(bias->scalar_type()) : "",
              ": one type for both is expected");
  return weight ? code_of(weight->scalar_type()) : bias ? code_of(bias->scalar_type()) : BLH_F32;
}

void check_eps(double eps) { TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative, got ", eps); }

struct Draws {
  double p;
  int64_t seed, step, layer, row_offset;
  Tensor device_step;      // undefined: none
};

void check_draws(const Draws& d, const Tensor& x) {
  TORCH_CHECK_VALUE(d.p >= 0.0 && d.p <= 1.0, "dropout probability has to be between 0 and 1, got ", d.p);
  TORCH_CHECK_VALUE(d.seed >= 0 && d.step >= 0, "seed and step must be in [0, 2^63), got ", d.seed, " and ", d.step);
  TORCH_CHECK_VALUE(d.layer >= 0 && d.layer < (int64_t(1) << 31), "layer must be in [0, 2^31), got ", d.layer);
  TORCH_CHECK_VALUE(d.row_offset >= 0 && d.row_offset < (int64_t(1) << 43), "row_offset must be in [0, 2^43), got ",
                    d.row_offset);
  if (d.device_step.defined())
    TORCH_CHECK(d.device_step.scalar_type() == at::kLong && d.device_step.numel() == 1 && d.device_step.device() == x.device(),
                "device_step must be one int64 on '", x.device(), "'");
}

void check_status(int status, const char* what) {
  if (status == BLH_OK) return;
  TORCH_CHECK(false, "bilinear_amd: ", what, " failed: ", blh_status_string(status),
              status == BLH_ERR_HIP ? " (hipError_t " + std::to_string(blh_last_hip_error()) + ")" : std::string());
}

// ---- native calls (checked tensors) ---------------------------------------------------------------------------------

// What a kernel may read: a lazily negated view (an imaginary part of a conjugate) is resolved first.
Tensor readable(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// NULL says that a tensor was left out: one whose storage has been freed (a sharded parameter, say) is not that.
const void* address(const Tensor& t) {
  if (!t.defined()) return nullptr;
  const void* p = t.const_data_ptr();           // (the offset alone where there is no storage)
  if ((!p || t.storage_offset() != 0) && t.numel() != 0)
    TORCH_CHECK(t.storage().nbytes() != 0, "bilinear_amd row operators: a tensor of shape ", t.sizes(), " has no storage");
  return p;
}

// Rows are read in place where the last axis is dense and the leading axes collapse to one, else from a dense copy.
struct Rows {
  Tensor t;
  int64_t ld;
  Rows() : ld(0) {}
  explicit Rows(const Tensor& given) : t(readable(given)), ld(given.size(-1)) {
    const Tensor x = t;
    if (x.is_contiguous()) return;
    const int64_t width = x.size(-1), n = x.dim();
    if (x.stride(-1) == 1 || width == 1) {
      // the step between consecutive rows, if all leading axes agree on one
      int64_t step = -1, next = 0;
      bool one = true;
      for (int64_t a = n - 2; a >= 0 && one; --a) {
        if (x.size(a) == 1) continue;
        if (step < 0) step = x.stride(a); else one = x.stride(a) == next;
        next = x.stride(a) * x.size(a);
      }
      if (one) {
        ld = step < 0 ? width : step;
        return;
      }
    }
    t = x.contiguous();
  }
  const void* ptr() const { return address(t); }
};

Tensor dense(const Tensor& t) { return t.defined() ? readable(t).contiguous() : t; }
Tensor plain(const Optional& t) { return t ? *t : Tensor(); }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
void* stream_of(const Tensor& x) { return (void*)c10::hip::getCurrentHIPStream(x.get_device()).stream(); }
int64_t rows_of(const Tensor& x) { return x.numel() / x.size(-1); }

blh_row_drop drop_of(const Draws& d, const Tensor& used) {
  return blh_row_drop{d.p, (uint64_t)d.seed, (uint64_t)d.step, d.row_offset,
                      (const uint64_t*)address(d.device_step), (uint64_t*)out_ptr(used), (int32_t)d.layer, 0};
}

// what the backward reads of the forward, [rows] each (both NULL: not kept)
struct Moments {
  float* mean = nullptr;
  float* rstd = nullptr;
  Moments() {}
  Moments(const Tensor& m, const Tensor& r) : mean(m.mutable_data_ptr<float>()), rstd(r.mutable_data_ptr<float>()) {}
  explicit Moments(const Tensor& both) : mean(both.mutable_data_ptr<float>()), rstd(mean + both.size(1)) {}   // [2, rows]
};

Tensor both_moments(const Tensor& x) { return at::empty({2, rows_of(x)}, x.options().dtype(at::kFloat)); }

// where the kernel leaves the step that it used (a call without rows launches none)
Tensor used_step(const Draws& d, const Tensor& x) {
  if (!d.device_step.defined()) return Tensor();
  return x.numel() ? at::empty({1}, d.device_step.options()) : d.device_step.add(d.step).reshape({1});
}

Tensor layer_norm_launch(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, int32_t param_code,
                         Moments m) {
  const c10::OptionalDeviceGuard guard(x.device());
  const Rows in(x);
  Tensor y = at::empty(x.sizes(), x.options());
  check_status(blh_layer_norm_forward(stream_of(x), in.ptr(), in.ld, address(weight), address(bias), eps, out_ptr(y), m.mean,
                                      m.rstd, rows_of(x), x.size(-1), code_of(x.scalar_type()), param_code),
               "blh_layer_norm_forward");
  return y;
}

struct ParamGrads {
  Tensor weight, bias, workspace;
  ParamGrads(const Tensor& x, bool need_weight, bool need_bias, int32_t code) {
    const auto o = x.options().dtype(code == BLH_F32 ? at::kFloat : x.scalar_type());
    if (need_weight) weight = at::empty({x.size(-1)}, o);
    if (need_bias) bias = at::empty({x.size(-1)}, o);
    if (need_weight || need_bias) {
      const int64_t need = blh_row_norm_workspace_bytes(rows_of(x), x.size(-1));
      if (need < 0) check_status((int)need, "blh_row_norm_workspace_bytes");
      if (need > 0) workspace = at::empty({need}, x.options().dtype(at::kByte));
    }
  }
  int64_t bytes() const { return workspace.defined() ? workspace.numel() : 0; }
};

variable_list layer_norm_backward_launch(const Tensor& dy, const Tensor& x, const Tensor& weight, Moments m,
                                         bool need_x, bool need_weight, bool need_bias, int32_t code) {
  const c10::OptionalDeviceGuard guard(x.device());
  const Rows gy(dy), in(x);
  Tensor dx = need_x ? at::empty(x.sizes(), x.options()) : Tensor();
  const ParamGrads g(x, need_weight, need_bias, code);
  check_status(blh_layer_norm_backward(stream_of(x), gy.ptr(), gy.ld, in.ptr(), in.ld, address(weight), m.mean, m.rstd,
                                       out_ptr(dx), out_ptr(g.weight), out_ptr(g.bias), out_ptr(g.workspace), g.bytes(),
                                       rows_of(x), x.size(-1), code_of(x.scalar_type()), code),
               "blh_layer_norm_backward");
  return {dx, g.weight, g.bias};
}

Tensor dropout_launch(const Tensor& x, const Draws& d, const Tensor& used) {
  const c10::OptionalDeviceGuard guard(x.device());
  const Rows in(x);
  Tensor y = at::empty(x.sizes(), x.options());
  const blh_row_drop drop = drop_of(d, used);
  check_status(blh_row_dropout(stream_of(x), in.ptr(), in.ld, out_ptr(y), &drop, rows_of(x), x.size(-1),
                               code_of(x.scalar_type())), "blh_row_dropout");
  return y;
}

std::tuple<Tensor, Tensor> residual_norm_launch(const Tensor& x, const Tensor& residual, const Tensor& weight,
                                                const Tensor& bias, double eps, const Draws& d, int32_t param_code,
                                                Moments m, const Tensor& used) {
  const c10::OptionalDeviceGuard guard(x.device());
  const Rows in(x), res(residual);
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor h = at::empty(x.sizes(), residual.options());
  const blh_row_drop drop = drop_of(d, used);
  check_status(blh_residual_norm_forward(stream_of(x), in.ptr(), in.ld, res.ptr(), res.ld, address(weight), address(bias), eps,
                                         d.p > 0.0 || used.defined() ? &drop : nullptr, out_ptr(y), out_ptr(h), m.mean, m.rstd,
                                         rows_of(x), x.size(-1), code_of(x.scalar_type()),
                                         code_of(residual.scalar_type()), param_code), "blh_residual_norm_forward");
  return {y, h};
}

// {dx, dresidual, dweight, dbias}
variable_list residual_norm_backward_launch(const Tensor& dy, const Tensor& dh, const Tensor& h, const Tensor& weight,
                                            Moments m, const Draws& d, bool need_x,
                                            bool need_residual, bool need_weight, bool need_bias, int32_t code) {
  const c10::OptionalDeviceGuard guard(h.device());
  const Rows gy(dy), in(h), gh = dh.defined() ? Rows(dh) : Rows();
  Tensor dx = need_x ? at::empty(h.sizes(), dy.options()) : Tensor();
  Tensor dres = need_residual ? at::empty(h.sizes(), h.options()) : Tensor();
  const ParamGrads g(dy, need_weight, need_bias, code);
  const blh_row_drop drop = drop_of(d, Tensor());
  check_status(blh_residual_norm_backward(stream_of(h), gy.ptr(), gy.ld, gh.ptr(), gh.ld, in.ptr(), in.ld, address(weight),
                                          m.mean, m.rstd, d.p > 0.0 ? &drop : nullptr, out_ptr(dx), out_ptr(dres),
                                          out_ptr(g.weight), out_ptr(g.bias), out_ptr(g.workspace), g.bytes(), rows_of(h),
                                          h.size(-1), code_of(dy.scalar_type()), code_of(h.scalar_type()), code),
               "blh_residual_norm_backward");
  return {dx, dres, g.weight, g.bias};
}

// ---- through the dispatcher -------------------------------------------------------------------------------------------
// A tracer, a dispatch mode or a tensor subclass sees what goes through torch's dispatcher.  Of the launches above that is an
// allocation and nothing that fills it, so where one is present the custom operators (row_ops.py) take their place, with
// their own autograd.

bool followed(std::initializer_list<const Tensor*> inputs) {
  const auto here = c10::impl::tls_local_dispatch_key_set();
  c10::DispatchKeySet keys = here.included_;           // (a dispatch mode sets the Python key, a tracer its own)
  for (const Tensor* t : inputs)
    if (t->defined()) keys = keys | t->key_set();
  return (keys - here.excluded_).has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Tracer}));
}

template <typename Signature> c10::TypedOperatorHandle<Signature> custom(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

Optional given(const Tensor& t) { return t.defined() ? Optional(t) : Optional(); }
Tensor wanted(bool need, const Tensor& t) { return need ? t : Tensor(); }

std::tuple<Tensor, Tensor, Tensor> custom_layer_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
  static const auto op = custom<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Optional&, const Optional&, double)>(
      "bilinear_hip::layer_norm");
  return op.call(x, given(w), given(b), eps);
}

variable_list custom_layer_norm_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& moments,
                                         bool need_x, bool need_weight, bool need_bias, int64_t code) {
  static const auto op = custom<std::tuple<Tensor, Tensor, Tensor>(
      const Tensor&, const Tensor&, const Optional&, const Tensor&, const Tensor&, bool, bool, bool, int64_t)>(
      "bilinear_hip::layer_norm_backward");
  const auto [dx, dw, db] = op.call(dy, x, given(w), moments.select(0, 0), moments.select(0, 1), need_x, need_weight,
                                    need_bias, code);
  return {wanted(need_x, dx), wanted(need_weight, dw), wanted(need_bias, db)};
}

Tensor custom_dropout(const Tensor& x, const Draws& d) {
  static const auto op = custom<std::tuple<Tensor, Tensor>(const Tensor&, double, c10::SymInt, c10::SymInt, c10::SymInt,
                                                           c10::SymInt, const Optional&)>("bilinear_hip::row_dropout");
  return std::get<0>(op.call(x, d.p, d.seed, d.step, d.layer, d.row_offset, given(d.device_step)));
}

std::tuple<Tensor, Tensor> custom_residual_norm(const Tensor& x, const Tensor& residual, const Tensor& w, const Tensor& b,
                                                double eps, const Draws& d) {
  static const auto op = custom<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>(
      const Tensor&, const Tensor&, const Optional&, const Optional&, double, double, c10::SymInt, c10::SymInt, c10::SymInt,
      c10::SymInt, const Optional&)>("bilinear_hip::residual_norm");
  const auto out = op.call(x, residual, given(w), given(b), eps, d.p, d.seed, d.step, d.layer, d.row_offset,
                           given(d.device_step));
  return {std::get<0>(out), std::get<1>(out)};
}

variable_list custom_residual_norm_backward(const Tensor& dy, const Tensor& dh, const Tensor& h, const Tensor& w,
                                            const Tensor& moments, const Draws& d, bool need_x, bool need_residual,
                                            bool need_weight, bool need_bias, int64_t code) {
  static const auto op = custom<std::tuple<Tensor, Tensor, Tensor, Tensor>(
      const Tensor&, const Optional&, const Tensor&, const Optional&, const Tensor&, const Tensor&, double, c10::SymInt,
      c10::SymInt, c10::SymInt, c10::SymInt, const Optional&, bool, bool, bool, bool, int64_t)>(
      "bilinear_hip::residual_norm_backward");
  const auto [dx, dres, dw, db] = op.call(dy, given(dh), h, given(w), moments.select(0, 0), moments.select(0, 1), d.p, d.seed,
                                          d.step, d.layer, d.row_offset, given(d.device_step), need_x, need_residual,
                                          need_weight, need_bias, code);
  return {wanted(need_x, dx), wanted(need_residual, dres), wanted(need_weight, dw), wanted(need_bias, db)};
}

// ---- autograd -------------------------------------------------------------------------------------------------------

// A leaf's gradient accumulator belongs to the stream it was made on.  One that an eager graph on the DEFAULT stream still
// holds cannot take part in a stream capture (that stream cannot be captured: the capture would break inside the autograd
// engine, where the error ends the process), so such a call is refused before anything is enqueued.  A view's leaf is its base.
template <typename L> void refuse_eager_leaves(const L& inputs) {
  c10::OptionalDeviceGuard guard;
  for (const Tensor* t : inputs) {
    if (!t->defined()) continue;
    guard.reset_device(t->device());      // (the inputs' one device, which need not be the current one)
    break;
  }
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad()) continue;
    const Tensor leaf = !t->is_leaf() && t->is_view() ? Tensor(t->_base()) : *t;
    if (!leaf.requires_grad() || !leaf.is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(leaf);
    if (!node) continue;
    const auto s = node->stream();
    TORCH_CHECK(!s || s->id() != 0,
                "bilinear_amd: a tensor that needs a gradient in this stream capture is still part of an eager autograd "
                "graph recorded on the default stream.  Drop that graph (its outputs and losses) before the capture, or "
                "run the eager steps on a side stream (torch.cuda.stream).");
  }
}

template <typename N> std::shared_ptr<N> make_node() {
  return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

void refuse_tangents(std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                "bilinear_amd row operators have no forward-mode derivative");
}

bool any_needs_grad(std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// The norms' formulas below are not themselves differentiable.  Under create_graph their results belong to a node that leads
// on to what they depend on and refuses to run: whoever differentiates them, towards whichever input, meets it.  (torch's own
// DelayedError leads nowhere: torch.autograd.grad would pass it by and leave the term out.)
struct SecondDerivative : public torch::autograd::Node {
  std::string name() const override { return "BilinearSecondDerivative"; }
  variable_list apply(variable_list&&) override {
    TORCH_CHECK(false, "bilinear_amd row operators: trying to differentiate the backward pass, which is not supported");
  }
};

variable_list once(variable_list grads, const variable_list& inputs) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::edge_list edges;
  for (const Tensor& t : inputs)
    if (t.defined() && t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
  if (edges.empty()) return grads;
  const auto node = make_node<SecondDerivative>();
  node->set_next_edges(std::move(edges));
  for (const Tensor& g : grads)
    if (g.defined()) torch::autograd::set_history(g, node);
  return grads;
}

// The custom backward operators under autograd: the same refusals.  (As a Python formula they cost 3 us a call.)
void autograd_of_backward(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  variable_list inputs;
  for (const c10::IValue& v : torch::jit::last(*stack, op.schema().arguments().size())) {
    if (!v.isTensor()) continue;
    const Tensor& t = v.toTensor();
    refuse_tangents({&t});
    if (t.requires_grad()) inputs.push_back(t);
  }
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
  if (inputs.empty() || !at::GradMode::is_enabled()) return;
  variable_list out;
  for (const c10::IValue& v : torch::jit::last(*stack, op.schema().returns().size())) out.push_back(v.toTensor());
  once(std::move(out), inputs);
}

struct LayerNormBackward : public torch::autograd::Node {
  SavedVariable x, weight;
  Tensor moments;           // mean and rstd, [2, rows]
  int32_t code = 0;
  std::string name() const override { return "BilinearLayerNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    moments.reset();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(3);
    const Tensor in = x.unpack(), w = weight.unpack();
    const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1),
               need_b = task_should_compute_output(2);
    if (followed({&grads[0], &in, &w}))
      return custom_layer_norm_backward(grads[0], in, w, moments, need_x, need_w, need_b, code);
    return once(layer_norm_backward_launch(grads[0], in, dense(w), Moments(moments), need_x, need_w, need_b, code),
                {grads[0], in, w});
  }
};

Tensor dropout(const Tensor& x, double p, int64_t seed, int64_t step, int64_t layer, int64_t row_offset,
               const Optional& device_step);

// dropout is linear: its backward is the same map, with the same derivative
Tensor dropped(const Tensor& dy, const Draws& d) {
  if (!at::GradMode::is_enabled() && !followed({&dy})) return dropout_launch(dy, d, Tensor());
  return dropout(dy, d.p, d.seed, d.step, d.layer, d.row_offset, given(d.device_step));
}

struct RowDropoutBackward : public torch::autograd::Node {
  Draws d;
  std::string name() const override { return "BilinearRowDropoutBackward"; }
  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined()) return variable_list(1);
    return {dropped(grads[0], d)};
  }
};

struct ResidualNormBackward : public torch::autograd::Node {
  SavedVariable h, weight;
  Tensor moments;
  Draws d;
  int32_t code = 0;
  at::ScalarType dtype = at::kFloat;
  std::string name() const override { return "BilinearResidualNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    h.reset_data();
    weight.reset_data();
    moments.reset();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(4);
    const bool need_x = task_should_compute_output(0), need_r = task_should_compute_output(1),
               need_w = task_should_compute_output(2), need_b = task_should_compute_output(3);
    const bool drops = (int64_t)(d.p * 65536.0 + 0.5) != 0;
    if (!grads[0].defined()) {
      // only the stream went on: the sum's gradients, whatever the rows' statistics are (a row may hold an infinity)
      const Tensor& dh = grads[1];
      const auto o = dh.options().dtype(code == BLH_F32 ? at::kFloat : dtype);
      return {need_x ? (drops ? dropped(dh, d) : dh).to(dtype) : Tensor(), wanted(need_r, dh),
              need_w ? at::zeros({dh.size(-1)}, o) : Tensor(), need_b ? at::zeros({dh.size(-1)}, o) : Tensor()};
    }
    const Tensor &dy = grads[0], stream = h.unpack(shared_from_this()), w = weight.unpack();
    if (followed({&dy, &grads[1], &stream, &w}))
      return custom_residual_norm_backward(dy, grads[1], stream, w, moments, d, need_x, need_r, need_w, need_b, code);
    // without dropout and with one type both branches of the sum get the same gradient: it is written once
    const bool same = need_x && need_r && stream.scalar_type() == dtype && !drops && !at::GradMode::is_enabled();
    variable_list out = residual_norm_backward_launch(dy, grads[1], stream, dense(w), Moments(moments), d, need_x && !same,
                                                      need_r, need_w, need_b, code);
    if (same) out[0] = out[1];
    return once(std::move(out), {dy, grads[1], stream, w});
  }
};

bool wants_grad(std::initializer_list<const Tensor*> inputs) {
  refuse_tangents(inputs);
  return at::GradMode::is_enabled() && any_needs_grad(inputs);
}

// ---- what Python calls ----------------------------------------------------------------------------------------------

Tensor layer_norm(const Tensor& x, const Optional& weight, const Optional& bias, double eps) {
  check_rows(x, "x");
  const int32_t code = check_params(x, weight, bias);
  check_eps(eps);
  const Tensor w = plain(weight), b = plain(bias);
  if (followed({&x, &w, &b})) return std::get<0>(custom_layer_norm(x, w, b, eps));
  if (!wants_grad({&x, &w, &b})) return layer_norm_launch(x, dense(w), dense(b), eps, code, Moments());
  refuse_eager_leaves(std::initializer_list<const Tensor*>{&x, &w, &b});
  const Tensor both = both_moments(x);
  Tensor y = layer_norm_launch(x, dense(w), dense(b), eps, code, Moments(both));
  auto node = make_node<LayerNormBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
  node->x = SavedVariable(x, false);
  node->weight = SavedVariable(w, false);
  node->moments = both;
  node->code = code;
  torch::autograd::set_history(y, node);
  return y;
}

Tensor dropout(const Tensor& x, double p, int64_t seed, int64_t step, int64_t layer, int64_t row_offset,
               const Optional& device_step) {
  check_rows(x, "x");
  Draws d{p, seed, step, layer, row_offset, plain(device_step)};
  check_draws(d, x);
  if (followed({&x, &d.device_step})) return custom_dropout(x, d);
  const bool grad = wants_grad({&x});
  if (grad) refuse_eager_leaves(std::initializer_list<const Tensor*>{&x});
  const Tensor used = grad ? used_step(d, x) : Tensor();
  Tensor y = dropout_launch(x, d, used);
  if (grad) {
    if (used.defined()) d.step = 0;
    d.device_step = used;
    auto node = make_node<RowDropoutBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->d = d;
    torch::autograd::set_history(y, node);
  }
  return y;
}

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const Tensor& residual, const Optional& weight,
                                         const Optional& bias, double eps, double p, int64_t seed, int64_t step,
                                         int64_t layer, int64_t row_offset, const Optional& device_step) {
  check_rows(x, "x");
  check_like(residual, x, "residual", true);
  const int32_t code = check_params(x, weight, bias);
  check_eps(eps);
  Draws d{p, seed, step, layer, row_offset, plain(device_step)};
  check_draws(d, x);
  const Tensor w = plain(weight), b = plain(bias);
  if (followed({&x, &residual, &w, &b, &d.device_step})) return custom_residual_norm(x, residual, w, b, eps, d);
  const bool grad = wants_grad({&x, &residual, &w, &b});
  if (!grad) return residual_norm_launch(x, residual, dense(w), dense(b), eps, d, code, Moments(), Tensor());
  refuse_eager_leaves(std::initializer_list<const Tensor*>{&x, &residual, &w, &b});
  const Tensor both = both_moments(x);
  const Tensor used = used_step(d, x);
  auto [y, h] = residual_norm_launch(x, residual, dense(w), dense(b), eps, d, code, Moments(both), used);
  if (used.defined()) d.step = 0;
  d.device_step = used;
  auto node = make_node<ResidualNormBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(x, residual, w, b));
  node->weight = SavedVariable(w, false);
  node->moments = both;
  node->d = d;
  node->code = code;
  node->dtype = x.scalar_type();
  torch::autograd::set_history({y, h}, node);
  node->h = SavedVariable(h, true);
  return {y, h};
}

// The custom operators' implementations: plain functions, outputs that were not asked for come back empty.

Tensor filled(const Tensor& t, const Tensor& x, at::ScalarType s) {
  return t.defined() ? t : at::empty({0}, x.options().dtype(s));
}

void check_stats(const Tensor& x, const Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == rows_of(x) && t.is_contiguous() && t.device() == x.device(), what,
              " must be ", rows_of(x), " dense float32 values on '", x.device(), "'");
}

int32_t check_code(const Tensor& x, const Optional& weight, int64_t code) {
  TORCH_CHECK(code == BLH_F32 || code == code_of(x.scalar_type()), "param_code must be 0 (float32) or that of ",
              name_of(x.scalar_type()));
  TORCH_CHECK(!weight || code_of(weight->scalar_type()) == code, "param_code is not the weight's type");
  return (int32_t)code;
}

std::tuple<Tensor, Tensor, Tensor> op_layer_norm(const Tensor& x, const Optional& weight, const Optional& bias, double eps) {
  check_rows(x, "x");
  const int32_t code = check_params(x, weight, bias);
  check_eps(eps);
  const auto o = x.options().dtype(at::kFloat);
  const Tensor mean = at::empty({rows_of(x)}, o), rstd = at::empty({rows_of(x)}, o);
  Tensor y = layer_norm_launch(x, dense(plain(weight)), dense(plain(bias)), eps, code, Moments(mean, rstd));
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> op_layer_norm_backward(const Tensor& dy, const Tensor& x, const Optional& weight,
                                                          const Tensor& mean, const Tensor& rstd, bool need_x,
                                                          bool need_weight, bool need_bias, int64_t param_code) {
  check_rows(x, "x");
  check_like(dy, x, "dy", false);
  check_param(x, weight, "weight");
  check_stats(x, mean, "mean");
  check_stats(x, rstd, "rstd");
  const int32_t code = check_code(x, weight, param_code);
  const auto g = layer_norm_backward_launch(dy, x, dense(plain(weight)), Moments(mean, rstd), need_x, need_weight,
                                            need_bias, code);
  const auto s = code == BLH_F32 ? at::kFloat : x.scalar_type();
  return {filled(g[0], x, x.scalar_type()), filled(g[1], x, s), filled(g[2], x, s)};
}

std::tuple<Tensor, Tensor> op_row_dropout(const Tensor& x, double p, int64_t seed, int64_t step, int64_t layer,
                                          int64_t row_offset, const Optional& device_step) {
  check_rows(x, "x");
  const Draws d{p, seed, step, layer, row_offset, plain(device_step)};
  check_draws(d, x);
  const Tensor used = used_step(d, x);
  Tensor y = dropout_launch(x, d, used);
  return {y, filled(used, x, at::kLong)};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> op_residual_norm(
    const Tensor& x, const Tensor& residual, const Optional& weight, const Optional& bias, double eps, double p,
    int64_t seed, int64_t step, int64_t layer, int64_t row_offset, const Optional& device_step) {
  check_rows(x, "x");
  check_like(residual, x, "residual", true);
  const int32_t code = check_params(x, weight, bias);
  check_eps(eps);
  const Draws d{p, seed, step, layer, row_offset, plain(device_step)};
  check_draws(d, x);
  const auto o = x.options().dtype(at::kFloat);
  const Tensor mean = at::empty({rows_of(x)}, o), rstd = at::empty({rows_of(x)}, o);
  const Tensor used = used_step(d, x);
  auto [y, h] = residual_norm_launch(x, residual, dense(plain(weight)), dense(plain(bias)), eps, d, code,
                                     Moments(mean, rstd), used);
  return {y, h, mean, rstd, filled(used, x, at::kLong)};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> op_residual_norm_backward(
    const Tensor& dy, const Optional& dh, const Tensor& h, const Optional& weight, const Tensor& mean, const Tensor& rstd,
    double p, int64_t seed, int64_t step, int64_t layer, int64_t row_offset, const Optional& device_step, bool need_x,
    bool need_residual, bool need_weight, bool need_bias, int64_t param_code) {
  check_rows(dy, "dy");
  check_like(h, dy, "h", true);
  if (dh) check_like(*dh, h, "dh", false);
  check_param(dy, weight, "weight");
  check_stats(h, mean, "mean");
  check_stats(h, rstd, "rstd");
  const int32_t code = check_code(dy, weight, param_code);
  const Draws d{p, seed, step, layer, row_offset, plain(device_step)};
  check_draws(d, dy);
  const auto g = residual_norm_backward_launch(dy, plain(dh), h, dense(plain(weight)), Moments(mean, rstd), d, need_x, need_residual, need_weight, need_bias,
                                               code);
  const auto s = code == BLH_F32 ? at::kFloat : dy.scalar_type();
  return {filled(g[0], dy, dy.scalar_type()), filled(g[1], h, h.scalar_type()), filled(g[2], dy, s), filled(g[3], dy, s)};
}

}  // namespace

TORCH_LIBRARY_IMPL(bilinear_hip, AutogradCUDA, m) {
  m.impl("layer_norm_backward", torch::CppFunction::makeFromBoxedFunction<&autograd_of_backward>());
  m.impl("residual_norm_backward", torch::CppFunction::makeFromBoxedFunction<&autograd_of_backward>());
}

PYBIND11_MODULE(_rows, m) {
  const auto release = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("layer_norm", &layer_norm, release);
  m.def("dropout", &dropout, release);
  m.def("residual_norm", &residual_norm, release);
  m.def("refuse_eager_leaves", [](const std::vector<Tensor>& tensors) {
    std::vector<const Tensor*> at;
    for (const Tensor& t : tensors) at.push_back(&t);
    refuse_eager_leaves(at);
  });
  m.def("op_layer_norm", &op_layer_norm, release);
  m.def("op_layer_norm_backward", &op_layer_norm_backward, release);
  m.def("op_row_dropout", &op_row_dropout, release);
  m.def("op_residual_norm", &op_residual_norm, release);
  m.def("op_residual_norm_backward", &op_residual_norm_backward, release);
}
