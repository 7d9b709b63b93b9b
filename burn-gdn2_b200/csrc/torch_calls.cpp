// The sequence operators on torch tensors: argument checks, outputs,
// workspaces, streams and autograd around the entry points of gdn2.h.  Native
// because a call of a decode step runs for 3 us on the device: the same work in
// Python took 15 to 20 us of the host, and 120 us with a gradient.
//
// Gradients are given once, in reverse: an output's gradient with create_graph
// = True raises when it is differentiated again (but for the norm of the
// training layer), a tangent of forward-mode differentiation is refused.
#include <torch/csrc/autograd/autograd.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/version.h>

#include <ATen/ATen.h>
#include <ATen/TensorUtils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "gdn2.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
namespace py = pybind11;

constexpr int64_t kCarry = 16;  // tokens between the states that gated_scan keeps for its backward
constexpr int64_t kTaps = 4, kCache = 3;
constexpr int64_t kMaxInt = 0x7fffffff;

// A status of the library; becomes burn_gdn2's Gdn2Error.
struct Failure : std::runtime_error {
  int status;
  Failure(int s, const char* text) : std::runtime_error(text), status(s) {}
};
void check(int status) {
  if (status != GDN2_OK) throw Failure(status, gdn2_last_error());
}

// The tensor's device as the current one, and the stream to launch on.
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* f32(const Tensor& t) { return static_cast<float*>(ptr(t)); }
const int32_t* i32(const Tensor& t) { return static_cast<const int32_t*>(ptr(t)); }
int32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? GDN2_DTYPE_F32 : GDN2_DTYPE_BF16; }
Tensor given(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
// An argument of a Function that has no gradient, and may be absent.
struct Plain {
  Tensor t;
};
// Which of these want a gradient, a bit each.
int64_t needs(std::initializer_list<Tensor> list) {
  int64_t bits = 0, bit = 1;
  for (const Tensor& t : list) {
    if (t.defined() && t.requires_grad()) bits |= bit;
    bit <<= 1;
  }
  return bits;
}

gdn2_view view(const Tensor& t) {  // [B,T,C] as [B,T,1,C]
  return t.defined() ? gdn2_view{t.data_ptr(), t.stride(0), t.stride(1), 0} : gdn2_view{};
}
Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor floats(at::IntArrayRef sizes, const Tensor& near) { return at::empty(sizes, near.options().dtype(at::kFloat)); }
Tensor workspace(size_t bytes, const Tensor& near) {
  return bytes ? at::empty({(int64_t)bytes}, near.options().dtype(at::kByte)) : Tensor();
}
// t with contiguous channels and no broadcast over them
Tensor rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

void check_input(const char* what, const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), what, " runs on the B200 CUDA kernels only; got a CPU tensor");
  TORCH_CHECK_TYPE(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, what, ": unsupported dtype ",
                   x.scalar_type(), "; use float32 or bfloat16");
}
void same_device(const char* what, const Tensor& x, const Tensor& t) {
  TORCH_CHECK_VALUE(!t.defined() || t.device() == x.device(), what, ": tensors on ", x.device(), " and ", t.device());
}
// An f32 argument of that shape, contiguous.
Tensor f32_argument(const char* what, const char* name, const Tensor& t, at::IntArrayRef sizes) {
  if (!t.defined()) return t;
  TORCH_CHECK_VALUE(t.sizes() == sizes, what, ": ", name, " must be ", sizes, ", got ", t.sizes());
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, what, ": ", name, " must be float32, got ", t.scalar_type());
  return t.contiguous();
}
void check_sizes(const char* what, const Tensor& x) {
  TORCH_CHECK_VALUE(x.size(0) <= kMaxInt && x.size(1) <= kMaxInt && x.size(2) <= kMaxInt, what, ": sizes ", x.sizes(),
                    " above 2^31 - 1");
}
bool wants_grad(std::initializer_list<Tensor> list) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : list)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// A dual tensor does not require a gradient, so its tangent would be lost.
void no_tangents(const char* what, std::initializer_list<Tensor> list) {
  for (const Tensor& t : list)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, " has no forward-mode derivative");
}

// What a second derivative meets.
struct Twice : torch::autograd::Node {
  const char* what;
  explicit Twice(const char* w) : what(w) {}
  variable_list apply(variable_list&&) override {
    TORCH_CHECK(false, what, ": trying to differentiate twice; its gradients are once_differentiable");
  }
};
// Gradients from a backward without a graph of its own: with create_graph they
// hang on all that they depend on (the incoming gradients, the inputs) by a
// node that refuses, else a penalty on a gradient would drop out in silence.
variable_list once(const char* what, const variable_list& incoming, const variable_list& inputs, variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  auto node = std::shared_ptr<Twice>(new Twice(what), torch::autograd::deleteNode);
  for (const variable_list* list : {&incoming, &inputs})
    for (const Tensor& t : *list)
      if (t.defined() && t.requires_grad()) node->add_next_edge(torch::autograd::impl::gradient_edge(t));
  if (!node->num_outputs()) return out;
  for (Tensor& t : out)
    if (t.defined()) {
      t = t.detach();
      torch::autograd::impl::set_gradient_edge(t, {node, node->add_input_metadata(t)});
    }
  return out;
}

// ---- gated scan ----

gdn2_scan_args scan_args(const Tensor& x, const Tensor& g, const Tensor& state, const Tensor& cu, bool complement,
                         const Tensor& carry) {
  gdn2_scan_args a{};
  a.batch = (int32_t)(cu.defined() ? cu.numel() - 1 : x.size(0));
  a.seq_len = (int32_t)x.size(1);
  a.channels = (int32_t)x.size(2);
  a.dtype = dtype_of(x);
  a.g_dtype = dtype_of(g);
  a.complement = complement;
  a.cu_seqlens = i32(cu);
  a.x = view(x);
  a.g = view(g);
  a.state_in = f32(state);
  a.carry = f32(carry);
  return a;
}

Tensor scan_forward(const Tensor& x, const Tensor& g, const Tensor& state, const Tensor& cu, bool complement,
                    const Tensor& last, const Tensor& carry) {
  On on(x);
  Tensor h = like(x);
  const gdn2_scan_args a = scan_args(x, g, state, cu, complement, carry);
  // up to 64 tokens are one block's and never cut into segments
  const size_t size = x.size(1) > 64 ? gdn2_gated_scan_workspace_bytes(&a, view(h)) : 0;
  const Tensor ws = workspace(size, x);
  check(gdn2_gated_scan(&a, view(h), f32(last), ptr(ws), size, on.stream));
  return h;
}

struct Scan : torch::autograd::Function<Scan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& g,
                               const std::optional<Tensor>& state_in, const Plain& packed, bool complement) {
    const Tensor state = given(state_in), cu = packed.t;
    Tensor last = floats({cu.defined() ? cu.numel() - 1 : x.size(0), x.size(2)}, x);
    Tensor carry = floats({x.size(0), (x.size(1) + kCarry - 1) / kCarry, x.size(2)}, x);
    Tensor h = scan_forward(x, g, state, cu, complement, last, carry);
    ctx->save_for_backward({x, g, state, cu, carry});
    ctx->saved_data["complement"] = complement;
    ctx->saved_data["needs"] = needs({state});
    ctx->set_materialize_grads(false);
    return {h, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &g = saved[1], &state = saved[2], &cu = saved[3], &carry = saved[4];
    variable_list out(5);
    {
      at::NoGradGuard none;
      On on(x);
      const Tensor d_h = grads[0].defined() ? rows(grads[0]) : at::zeros_like(x);
      const Tensor d_last = grads[1].defined() ? grads[1].contiguous() : Tensor();
      out[0] = like(x);
      out[1] = like(g);
      if (ctx->saved_data["needs"].toInt() & 1) out[2] = like(state);
      gdn2_scan_bwd_args a{};
      a.fwd = scan_args(x, g, state, cu, ctx->saved_data["complement"].toBool(), carry);
      a.d_h = view(d_h);
      a.d_state_out = f32(d_last);
      a.dx = view(out[0]);
      a.dg = view(out[1]);
      a.d_state_in = f32(out[2]);
      const size_t size = gdn2_gated_scan_bwd_workspace_bytes(&a);
      const Tensor ws = workspace(size, x);
      check(gdn2_gated_scan_bwd(&a, ptr(ws), size, on.stream));
    }
    return once("gated_scan", grads, {x, g, state}, std::move(out));
  }
};

std::tuple<Tensor, Tensor> gated_scan(Tensor x, Tensor g, const std::optional<Tensor>& state_in,
                                      const std::optional<Tensor>& cu_in, bool complement, bool inplace) {
  const char* what = "gated_scan";
  check_input(what, x);
  TORCH_CHECK_VALUE(x.dim() == 3 && x.sizes() == g.sizes(), what, ": x and g must both be [B,T,C], got ", x.sizes(),
                    " and ", g.sizes());
  TORCH_CHECK_TYPE(g.scalar_type() == at::kFloat || g.scalar_type() == x.scalar_type(), what,
                   ": g must be float32 or x's dtype ", x.scalar_type(), ", got ", g.scalar_type());
  check_sizes(what, x);
  const Tensor cu = given(cu_in), given_state = given(state_in);
  no_tangents(what, {x, g, given_state});
  same_device(what, x, g);
  same_device(what, x, given_state);
  const int64_t n = cu.defined() ? cu.numel() - 1 : x.size(0), T = x.size(1), C = x.size(2);
  Tensor state = f32_argument(what, "state", given_state, {n, C});
  x = rows(x);
  g = rows(g);
  const bool grads = wants_grad({x, g, state});
  if (inplace) {
    TORCH_CHECK_VALUE(state.defined(), what, ": inplace needs a state");
    TORCH_CHECK_VALUE(!grads, what, ": inplace does not go with gradients; detach the inputs or use torch.no_grad()");
    TORCH_CHECK_VALUE(state.is_same(given_state), what, ": inplace needs a contiguous state");
  }
  if (n == 0 || C == 0 || (T == 0 && !cu.defined())) {  // nothing to launch: no token, or nothing in it
    Tensor last = state.defined() ? state : at::zeros({n, C}, x.options().dtype(at::kFloat));
    return {x + g.to(x.scalar_type()), inplace ? last : last.clone()};
  }
  if (grads) {
    variable_list out = Scan::apply(x, g, maybe(state), Plain{cu}, complement);
    return {out[0], out[1]};
  }
  Tensor last = inplace ? state : floats({n, C}, x);
  Tensor h = scan_forward(x, g, state, cu, complement, last, Tensor());
  if (inplace && !state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return {h, last};
}

// ---- causal convolution ----

gdn2_conv_args conv_args(const Tensor& x, const Tensor& weight, const Tensor& cache, const Tensor& cu) {
  gdn2_conv_args a{};
  a.batch = (int32_t)(cu.defined() ? cu.numel() - 1 : x.size(0));
  a.seq_len = (int32_t)x.size(1);
  a.channels = (int32_t)x.size(2);
  a.dtype = dtype_of(x);
  a.cu_seqlens = i32(cu);
  a.x = view(x);
  a.weight = f32(weight);
  a.cache_in = f32(cache);
  return a;
}

variable_list conv_forward(const Tensor& x, const Tensor& weight, const Tensor& cache, const Tensor& cu) {
  On on(x);
  Tensor y = like(x), next = floats({cu.defined() ? cu.numel() - 1 : x.size(0), kCache, x.size(2)}, x);
  const gdn2_conv_args a = conv_args(x, weight, cache, cu);
  check(gdn2_causal_conv(&a, view(y), f32(next), on.stream));
  return {y, next};
}

struct Conv : torch::autograd::Function<Conv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                               const std::optional<Tensor>& cache_in, const Plain& packed) {
    const Tensor cache = given(cache_in), cu = packed.t;
    ctx->saved_data["needs"] = needs({weight, cache});
    ctx->save_for_backward({x, weight, cache, cu});
    ctx->set_materialize_grads(false);
    return conv_forward(x, weight, cache, cu);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &cache = saved[2], &cu = saved[3];
    variable_list out(4);
    {
      at::NoGradGuard none;
      On on(x);
      const Tensor d_y = grads[0].defined() ? rows(grads[0]) : at::zeros_like(x);
      const Tensor d_next = grads[1].defined() ? grads[1].contiguous() : Tensor();
      out[0] = like(x);
      const int64_t wanted = ctx->saved_data["needs"].toInt();
      if (wanted & 1) out[1] = like(weight);
      if (wanted & 2) out[2] = like(cache);
      gdn2_conv_bwd_args a{};
      a.fwd = conv_args(x, weight, cache, cu);
      a.d_y = view(d_y);
      a.d_cache_out = f32(d_next);
      a.dx = view(out[0]);
      a.d_weight = f32(out[1]);
      a.d_cache_in = f32(out[2]);
      const size_t size = gdn2_causal_conv_bwd_workspace_bytes(&a);
      const Tensor ws = workspace(size, x);
      check(gdn2_causal_conv_bwd(&a, ptr(ws), size, on.stream));
    }
    return once("causal_conv_silu", grads, {x, weight, cache}, std::move(out));
  }
};

std::tuple<Tensor, Tensor> causal_conv_silu(Tensor x, const Tensor& weight_in, const std::optional<Tensor>& cache_in,
                                            const std::optional<Tensor>& cu_in) {
  const char* what = "causal_conv_silu";
  check_input(what, x);
  TORCH_CHECK_VALUE(x.dim() == 3, what, ": x must be [B,T,C], got ", x.sizes());
  check_sizes(what, x);
  const Tensor cu = given(cu_in);
  no_tangents(what, {x, weight_in, given(cache_in)});
  same_device(what, x, weight_in);
  same_device(what, x, given(cache_in));
  const int64_t n = cu.defined() ? cu.numel() - 1 : x.size(0), T = x.size(1), C = x.size(2);
  const Tensor weight = f32_argument(what, "weight", weight_in, {C, kTaps});
  const Tensor cache = f32_argument(what, "cache", given(cache_in), {n, kCache, C});
  x = rows(x);
  if (n == 0 || C == 0 || (T == 0 && !cu.defined()))  // nothing to launch: no token, or nothing in it
    return {x * weight.select(1, 0).to(x.scalar_type()),
            cache.defined() ? cache.clone() : at::zeros({n, kCache, C}, x.options().dtype(at::kFloat))};
  variable_list out = wants_grad({x, weight, cache}) ? Conv::apply(x, weight, maybe(cache), Plain{cu}) : conv_forward(x, weight, cache, cu);
  return {out[0], out[1]};
}

// ---- group norm ----

struct NormRest {
  int64_t groups;
  double eps;
  bool center;
};

// The gradients of the inputs of which `wanted` has a bit, by the formula in
// torch operations and with a graph of their own.
variable_list norm_backward_again(const variable_list& saved, const Tensor& d_y, int64_t wanted, const NormRest& r) {
  const Tensor &x = saved[0], &gate = saved[1], &weight = saved[2], &bias = saved[3];
  const int64_t chan = x.size(-1), width = chan / r.groups;
  const auto split = [&](const Tensor& t) { return t.to(at::kFloat).reshape({-1, r.groups, width}); };
  const auto affine = [&](const Tensor& t) { return t.numel() == chan ? t.reshape({r.groups, width}) : t; };
  Tensor v = split(x);
  if (r.center) v = v - v.mean(-1, true);
  v = v * (v.square().mean(-1, true) + r.eps).rsqrt();
  if (weight.defined()) v = v * affine(weight);
  if (bias.defined()) v = v + affine(bias);
  const Tensor y = (gate.defined() ? v * at::silu(split(gate)) : at::silu(v)).reshape(x.sizes()).to(x.scalar_type());
  variable_list inputs, out(4);
  for (int k = 0; k < 4; ++k)
    if ((wanted >> k) & 1) inputs.push_back(saved[k]);
  variable_list grads = torch::autograd::grad({y}, inputs, {d_y}, true, true);
  for (int k = 0, at = 0; k < 4; ++k)
    if ((wanted >> k) & 1) out[k] = grads[at++];
  return out;
}

// [..., C] as rows; a copy where the rows are not evenly spaced or their channels not contiguous.
Tensor norm_rows(const Tensor& t, int64_t chan) {
  return t.defined() ? rows(t.dim() == 2 ? t : t.reshape({-1, chan})) : t;
}
// t such that norm_rows makes no copy of it: a copy made once, for forward and backward.
Tensor evenly(const Tensor& t, int64_t chan) {
  if (!t.defined() || t.is_contiguous()) return t;
  const bool lined = t.stride(-1) == 1 || t.size(-1) == 1;
  const int64_t sizes[] = {t.numel() / chan, chan};
  return lined && at::detail::computeStride(t.sizes(), t.strides(), at::IntArrayRef(sizes)) ? t : t.contiguous();
}

gdn2_group_norm_args norm_args(const Tensor& x, const Tensor& gate, const Tensor& weight, const Tensor& bias,
                               const NormRest& r) {
  const int64_t chan = x.size(1);
  gdn2_group_norm_args a{};
  a.rows = x.size(0);
  a.groups = (int32_t)r.groups;
  a.width = (int32_t)(chan / r.groups);
  a.dtype = dtype_of(x);
  a.center = r.center;
  a.weight_shared = weight.defined() && weight.numel() != chan;
  a.eps = (float)r.eps;
  a.x = ptr(x);
  a.ld_x = x.stride(0);
  a.gate = ptr(gate);
  a.ld_gate = gate.defined() ? gate.stride(0) : 0;
  a.weight = f32(weight);
  a.bias = f32(bias);
  return a;
}

Tensor norm_forward(const Tensor& x, const Tensor& gate, const Tensor& weight, const Tensor& bias, const NormRest& r) {
  On on(x);
  Tensor y = like(x);
  if (x.size(0)) {
    const gdn2_group_norm_args a = norm_args(x, gate, weight, bias, r);
    check(gdn2_group_norm_gate(&a, ptr(y), on.stream));
  }
  return y;
}

struct Norm : torch::autograd::Function<Norm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& gate_in,
                        const std::optional<Tensor>& weight_in, const std::optional<Tensor>& bias_in, int64_t groups,
                        double eps, bool center, bool twice) {
    const Tensor gate = given(gate_in), weight = given(weight_in), bias = given(bias_in);
    const int64_t chan = x.size(-1);
    ctx->save_for_backward({x, gate, weight, bias});
    ctx->saved_data["needs"] = needs({x, gate, weight, bias});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["center"] = center;
    ctx->saved_data["twice"] = twice;
    Tensor y = norm_forward(norm_rows(x, chan), norm_rows(gate, chan), weight, bias, {groups, eps, center});
    return x.dim() == 2 ? y : y.view(x.sizes());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &weight = saved[2], &bias = saved[3];
    const int64_t wanted = ctx->saved_data["needs"].toInt(), chan = saved[0].size(-1);
    const NormRest r{ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(),
                     ctx->saved_data["center"].toBool()};
    variable_list out(8);
    if (at::GradMode::is_enabled() && ctx->saved_data["twice"].toBool()) {
      variable_list again = norm_backward_again(saved, grads[0], wanted, r);
      std::copy(again.begin(), again.end(), out.begin());
      return out;
    }
    {
      at::NoGradGuard none;
      On on(saved[0]);
      const Tensor x = norm_rows(saved[0], chan), gate = norm_rows(saved[1], chan), d_y = norm_rows(grads[0], chan);
      const Tensor* of[] = {&x, &gate, &weight, &bias};
      for (int k = 0; k < 4; ++k)
        if ((wanted >> k) & 1) out[k] = like(*of[k]);
      if (x.size(0)) {
        gdn2_group_norm_bwd_args a{};
        a.fwd = norm_args(x, gate, weight, bias, r);
        a.d_y = ptr(d_y);
        a.ld_dy = d_y.stride(0);
        a.dx = ptr(out[0]);
        a.d_gate = ptr(out[1]);
        a.d_weight = f32(out[2]);
        a.d_bias = f32(out[3]);
        const size_t size = gdn2_group_norm_gate_bwd_workspace_bytes(&a);
        const Tensor ws = workspace(size, x);
        check(gdn2_group_norm_gate_bwd(&a, ptr(ws), size, on.stream));
      } else {
        for (int k = 2; k < 4; ++k)
          if (out[k].defined()) out[k].zero_();
      }
      for (int k = 0; k < 2; ++k)
        if (out[k].defined() && saved[0].dim() != 2) out[k] = out[k].view(saved[0].sizes());
    }
    return once("group_norm_gate", grads, {saved[0], saved[1], weight, bias}, std::move(out));
  }
};

// twice: a backward with create_graph takes norm_backward_again.
Tensor group_norm_gate(const Tensor& x, const std::optional<Tensor>& gate_in, const std::optional<Tensor>& weight_in,
                       const std::optional<Tensor>& bias_in, int64_t groups, double eps, bool center, bool twice) {
  const char* what = "group_norm_gate";
  check_input(what, x);
  const int64_t chan = x.dim() ? x.size(-1) : 0;
  TORCH_CHECK_VALUE(groups >= 1 && chan > 0 && chan % groups == 0, what, ": the ", chan, " channels do not split into ",
                    groups, " groups");
  TORCH_CHECK_VALUE(eps > 0, what, ": eps must be > 0, got ", eps);
  if (chan > kMaxInt) throw Failure(GDN2_EUNSUPPORTED, "group_norm_gate: more than 2^31 - 1 channels");
  const Tensor gate = given(gate_in);
  Tensor affine[2] = {given(weight_in), given(bias_in)};
  no_tangents(what, {x, gate, affine[0], affine[1]});
  same_device(what, x, gate);
  TORCH_CHECK_VALUE(!gate.defined() || (gate.sizes() == x.sizes() && gate.scalar_type() == x.scalar_type()), what,
                    ": gate must be ", x.sizes(), " ", x.scalar_type(), ", got ", gate.sizes(), " ", gate.scalar_type());
  for (int k = 0; k < 2; ++k) {
    Tensor& t = affine[k];
    if (!t.defined()) continue;
    const char* name = k ? "bias" : "weight";
    same_device(what, x, t);
    TORCH_CHECK_VALUE(t.dim() == 1 && (t.numel() == chan || t.numel() == chan / groups), what, ": ", name, " must be [",
                      chan, "] or [", chan / groups, "], got ", t.sizes());
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, what, ": ", name, " must be float32, got ", t.scalar_type());
    t = t.contiguous();
  }
  const Tensor &weight = affine[0], &bias = affine[1];
  TORCH_CHECK_VALUE(!bias.defined() || (weight.defined() && weight.sizes() == bias.sizes()), what,
                    ": a bias goes with a weight of its shape");
  if (wants_grad({x, gate, weight, bias}))
    return Norm::apply(evenly(x, chan), maybe(evenly(gate, chan)), maybe(weight), maybe(bias), groups, eps, center, twice);
  Tensor y = norm_forward(norm_rows(x, chan), norm_rows(gate, chan), weight, bias, {groups, eps, center});
  return x.dim() == 2 ? y : y.view(x.sizes());
}

// ---- state pools ----

void check_pool(const char* what, const std::vector<Tensor>& pool) {
  for (const Tensor& t : pool) {
    TORCH_CHECK(t.is_cuda(), what, " runs on the B200 CUDA kernels only; got a CPU tensor");
    TORCH_CHECK_VALUE(t.dim() && t.size(0) == pool[0].size(0), what, ": every tensor of a pool has its rows first and as "
                      "many, got ", t.sizes(), " beside ", pool[0].sizes());
    TORCH_CHECK_VALUE(t.is_contiguous(), what, ": the tensors of a pool must be contiguous");
    TORCH_CHECK_VALUE(!t.requires_grad(), what, ": the rows of a pool move without gradients; detach its tensors");
    no_tangents(what, {t});
    same_device(what, pool[0], t);
  }
  TORCH_CHECK_VALUE(pool[0].size(0) <= GDN2_MAX_STATE_ROWS, what, ": ", pool[0].size(0), " rows, at most ",
                    GDN2_MAX_STATE_ROWS);
}

// Row numbers on the device, int32; checked where they come from the host.
Tensor pool_index(const char* what, const Tensor& index, int64_t rows, const Tensor& near) {
  const auto type = index.scalar_type();
  TORCH_CHECK_VALUE(index.dim() == 1 && (type == at::kInt || type == at::kLong), what,
                    ": index must be a vector of int32 or int64, got ", type, " ", index.sizes());
  TORCH_CHECK_VALUE(index.size(0) <= GDN2_MAX_STATE_ROWS, what, ": ", index.size(0), " rows, at most ",
                    GDN2_MAX_STATE_ROWS);
  if (!index.is_cuda()) {
    const Tensor wide = index.to(at::kLong).contiguous();
    const int64_t* at = wide.data_ptr<int64_t>();
    for (int64_t i = 0; i < wide.numel(); ++i)
      TORCH_CHECK_VALUE(at[i] >= -1 && at[i] < rows, what, ": row numbers must be -1 to ", rows - 1, ", got ", at[i],
                        " for row ", i);
    return index.to(near.device(), at::kInt);
  }
  same_device(what, near, index);
  // int64: as far as 32 bits tell a number inside the pool from one outside
  return (type == at::kLong ? index.clamp(-2, rows).to(at::kInt) : index).contiguous();
}

void move_rows(const std::vector<Tensor>& from, const std::vector<Tensor>& to, const Tensor& index, int64_t src_rows) {
  On on(index);
  const int64_t n = index.size(0);
  c10::SmallVector<gdn2_state_rows, 16> list;
  for (size_t k = 0; k < to.size(); ++k)
    if (to[k].nbytes()) list.push_back({from[k].data_ptr(), to[k].data_ptr(), (int64_t)to[k].nbytes() / n});
  if (!list.empty())
    check(gdn2_move_state_rows(list.data(), (int32_t)list.size(), i32(index), (int32_t)src_rows, (int32_t)n, on.stream));
}

void reorder_states(const std::vector<Tensor>& pool, const Tensor& index_in) {
  const char* what = "reorder_states";
  check_pool(what, pool);
  const int64_t rows = pool[0].size(0);
  c10::SmallVector<std::pair<const char*, size_t>, 16> spans;
  for (const Tensor& t : pool) spans.push_back({static_cast<const char*>(t.data_ptr()), t.nbytes()});
  std::sort(spans.begin(), spans.end());
  for (size_t k = 1; k < spans.size(); ++k)
    TORCH_CHECK_VALUE(spans[k - 1].first + spans[k - 1].second <= spans[k].first, what,
                      ": a tensor (or a part of one) comes twice");
  const Tensor index = pool_index(what, index_in, rows, pool[0]);
  TORCH_CHECK_VALUE(index.size(0) == rows, what, ": ", index.size(0), " row numbers for ", rows, " rows");
  move_rows(pool, pool, index, rows);
  for (const Tensor& t : pool)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

std::vector<Tensor> select_states(const std::vector<Tensor>& pool, const Tensor& index_in) {
  const char* what = "select_states";
  check_pool(what, pool);
  const int64_t rows = pool[0].size(0);
  const Tensor index = pool_index(what, index_in, rows, pool[0]);
  std::vector<Tensor> out;
  for (const Tensor& t : pool) {
    auto sizes = t.sizes().vec();
    sizes[0] = index.size(0);
    out.push_back(at::empty(sizes, t.options()));
  }
  move_rows(pool, out, index, rows);
  return out;
}

}  // namespace

PYBIND11_MODULE(_torch_calls, m) {
  static py::handle error;  // burn_gdn2's Gdn2Error
  m.attr("torch_version") = TORCH_VERSION;
  m.def("set_error_class", [](py::object cls) { error = cls.release(); });
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure& f) {
      PyErr_SetObject(error.ptr(), py::object(error(f.status, f.what())).ptr());
    }
  });
  m.def("gated_scan", &gated_scan);
  m.def("causal_conv_silu", &causal_conv_silu);
  m.def("group_norm_gate", &group_norm_gate);
  m.def("reorder_states", &reorder_states);
  m.def("select_states", &select_states);
}
