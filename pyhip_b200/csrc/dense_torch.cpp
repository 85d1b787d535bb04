// torch side of the dense operators around the MoE layer (module pyhip_b200._dense): argument checks, output tensors,
// autograd nodes and the calls into libb200moe.so's C ABI, which knows nothing of torch.
//
// The MoE layer's own calls go through ctypes.  These operators take 3 to 10 us on the GPU at decode sizes, and their
// gradients run on autograd's device thread: a Python call that checks, allocates and launches costs 10 to 25 us, and a
// Python backward node another 40 to 80 us on top of autograd's own 40.  Here a call costs little more than its launches.
#include <torch/extension.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <initializer_list>
#include <optional>
#include <string>
#include <vector>

#include "../../include/b200moe.h"

// the torch and the Python that this file was built for, to be read without loading it
extern "C" __attribute__((visibility("default"), used)) const char b200moe_dense_tag[] = B200MOE_DENSE_TAG;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxRow = 16384;      // values of a row that the row-wise kernels hold in registers
constexpr int64_t kMaxExperts = 1024, kMaxTopk = 32;

struct B200Error : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void call_check(int rc, const char* what) {
  if (rc == 0) return;
  std::string kind = rc < 0 ? "argument error" : "CUDA error " + std::to_string(rc);
  throw B200Error(std::string(what) + ": " + kind + ": " + b200moe_last_error());
}
#define VALUE_CHECK(cond, ...) \
  do {                         \
    if (!(cond)) throw py::value_error(c10::str(__VA_ARGS__)); \
  } while (0)
#define TYPE_CHECK(cond, ...) \
  do {                        \
    if (!(cond)) throw py::type_error(c10::str(__VA_ARGS__)); \
  } while (0)
void need_cuda(const Tensor& x, const char* what) {
  if (!x.is_cuda()) throw std::runtime_error(std::string(what) + " runs on a CUDA device only (sm_100a); there is no CPU path");
}
void need_no_grad(bool requires_grad, const char* what) {
  if (requires_grad && at::GradMode::is_enabled())
    throw std::runtime_error(std::string(what) + ": call it under torch.no_grad() or on detached tensors");
}
// What torch may lay over a call and these kernels, which torch's dispatcher does not see, cannot take part in.  A dual tensor of
// forward-mode differentiation does not require a gradient: it would come back without its tangent.  A trace would record the
// empty outputs and none of the kernels that fill them.  `no_grad` ends neither.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
void need_no_tangent(bool any, const char* what) {
  if (any && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    throw std::runtime_error(std::string(what) + " has no forward-mode derivative: unpack the dual tensors first");
}
void need_eager(const char* what) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  bool traced = torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
  if (TorchDispatchModeTLS::any_modes_set())
    for (const auto mode : {TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FAKE, TorchDispatchModeKey::FUNCTIONAL})
      traced = traced || TorchDispatchModeTLS::get_mode(mode).has_value();
  if (traced) throw std::runtime_error(std::string(what) + " runs its own kernels and cannot be traced: call it outside of the traced function");
}

int row_type(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return B200MOE_T_BF16;
    case at::kHalf: return B200MOE_T_FP16;
    case at::kFloat: return B200MOE_T_FP32;
    default: return -1;
  }
}
// Null means an absent tensor to the C calls, so one that is there must not come as null: a wrapper around another tensor (a subclass
// without memory of its own) would be taken for none.
void* ptr(const Tensor& t) {
  if (!t.defined()) return nullptr;
  void* p = t.data_ptr();
  TYPE_CHECK(p != nullptr || t.numel() == 0, "a tensor of shape ", t.sizes(), " has no memory of its own: pass the tensor that it wraps");
  return p;
}
void* ptr(const OptTensor& t) { return t.has_value() ? ptr(*t) : nullptr; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
bool on(const OptTensor& t, const Tensor& like) { return !t.has_value() || t->device() == like.device(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }
Tensor empty_as(const Tensor& t, at::IntArrayRef shape, at::ScalarType dtype) { return at::empty(shape, t.options().dtype(dtype).requires_grad(false)); }

// The values as memory holds them: a negation that torch has put off (a view of a conjugate's imaginary part) is made first.
Tensor settled(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor packed(const Tensor& t) { return settled(t).contiguous(); }

// [..., H] as T rows of H neighbouring values, `stride` elements apart; a view wherever one exists
struct Rows {
  Tensor t;
  int64_t T, H, stride;
};
Rows rows_of(const Tensor& as_given) {
  const Tensor x = settled(as_given);
  Rows r{x, 0, x.size(-1), 0};
  r.T = r.H ? x.numel() / r.H : 0;
  if (x.is_contiguous()) {
    r.stride = r.H;
    return r;
  }
  if (x.dim() != 2) r.t = x.numel() ? x.reshape({-1, r.H}) : x.new_empty({r.T, r.H});
  if (r.H > 1 && r.t.stride(1) != 1) r.t = r.t.contiguous();
  r.stride = r.T > 1 ? r.t.stride(0) : r.H;
  return r;
}
// an upstream gradient as the kernels read it; one that is known to be zero has no memory and counts for none
Tensor upstream(const Tensor& g) { return g.defined() && !g._is_zerotensor() ? packed(g) : Tensor(); }
int32_t as_i32(int64_t v, const char* what) {
  VALUE_CHECK(v < (int64_t(1) << 31), what, " is too large: ", v);
  return (int32_t)v;
}

// ------------------------------------------------------------------------------------ 8-bit integers
std::tuple<Tensor, Tensor> quantize_int8(const Tensor& x) {
  need_cuda(x, "quantize_int8");
  need_eager("quantize_int8");
  need_no_tangent(has_tangent(x), "quantize_int8");
  const int dt = row_type(x.scalar_type());
  TYPE_CHECK(dt >= 0, "x must be bfloat16, float16 or float32");
  VALUE_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= kMaxRow, "rows of x must have 1 to ", kMaxRow, " values");
  need_no_grad(x.requires_grad(), "quantize_int8 has no gradient");
  c10::cuda::CUDAGuard guard(x.device());
  const Rows r = rows_of(x);
  Tensor q = empty_as(x, x.sizes(), at::kChar), scale = empty_as(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
  call_check(b200moe_quantize_int8(ptr(r.t), r.stride, as_i32(r.T, "the number of rows"), (int32_t)r.H, dt, ptr(q), scale.data_ptr<float>(),
                                   stream_of(x)), "quantize_int8");
  return {q, scale};
}

Tensor linear_int8(const Tensor& x, const Tensor& weight, const Tensor& weight_scale, const OptTensor& x_scale, const OptTensor& bias,
                   std::optional<at::ScalarType> out_dtype, int64_t variant) {
  need_cuda(x, "linear_int8");
  need_eager("linear_int8");
  need_no_tangent(has_tangent(x) || has_tangent(weight_scale) || has_tangent(x_scale) || has_tangent(bias), "linear_int8");
  TYPE_CHECK(weight.scalar_type() == at::kChar && weight.dim() == 2, "weight must be an int8 matrix [N, K]");
  const int64_t N = weight.size(0), K = weight.size(1);
  VALUE_CHECK(x.dim() >= 1 && x.size(-1) == K, "x has shape ", x.sizes(), ", the weight ", K, " columns");
  VALUE_CHECK(N >= 1 && K >= 16 && K % 16 == 0 && K < (1 << 17), "weight [", N, ", ", K, "]: K must be a multiple of 16 below 2**17");
  VALUE_CHECK(weight_scale.scalar_type() == at::kFloat && weight_scale.numel() == N, "weight_scale must hold one float32 scale per output channel");
  VALUE_CHECK(!bias || (bias->scalar_type() == at::kFloat && bias->numel() == N), "bias must hold one float32 value per output channel");
  int dt = row_type(x.scalar_type());
  if (dt >= 0) {
    VALUE_CHECK(!x_scale, "x_scale belongs to int8 rows");
    VALUE_CHECK(K <= kMaxRow, "rows that are quantised here have up to ", kMaxRow, " values");
  } else {
    TYPE_CHECK(x.scalar_type() == at::kChar, "x must be int8, bfloat16, float16 or float32");
    dt = B200MOE_T_INT8;
    VALUE_CHECK(x_scale && x_scale->scalar_type() == at::kFloat && x_scale->sizes() == x.sizes().slice(0, x.dim() - 1),
                "int8 rows need x_scale, one float32 per row");
  }
  VALUE_CHECK(weight.device() == x.device() && weight_scale.device() == x.device() && on(bias, x) && on(x_scale, x),
              "all tensors must be on one device");
  need_no_grad(x.requires_grad() || weight_scale.requires_grad() || wants_grad(bias) || wants_grad(x_scale), "linear_int8 has no gradient");
  const at::ScalarType out = out_dtype.value_or(dt < B200MOE_T_FP32 ? x.scalar_type() : at::kBFloat16);
  TYPE_CHECK(out == at::kBFloat16 || out == at::kHalf, "out_dtype must be bfloat16 or float16");
  VALUE_CHECK(variant >= 0 && variant <= 2, "variant=", variant, ": 0, 1 or 2");

  c10::cuda::CUDAGuard guard(x.device());
  void* stream = stream_of(x);
  Rows r = rows_of(x);
  const int32_t T = as_i32(r.T, "the number of rows"), n = as_i32(N, "the number of channels");
  auto shape = x.sizes().vec();
  shape.back() = N;
  Tensor y = empty_as(x, shape, out), ws, xs;
  int64_t bytes = 0;
  if (dt == B200MOE_T_INT8) {
    if (r.stride != K || ((uintptr_t)ptr(r.t) & 15)) {
      r.t = r.t.clone(at::MemoryFormat::Contiguous);
      r.stride = K;
    }
    xs = packed(*x_scale);
  } else {
    call_check(b200moe_linear_int8_workspace(T, n, (int32_t)K, (int32_t)variant, &bytes), "linear_int8_workspace");
    if (bytes) ws = empty_as(x, {bytes}, at::kByte);
  }
  Tensor w = packed(weight);
  if ((uintptr_t)ptr(w) & 15) w = w.clone();
  const Tensor sc = packed(weight_scale), b = bias ? packed(*bias) : Tensor();
  call_check(b200moe_linear_int8(ptr(r.t), r.stride, dt, (const float*)ptr(xs), ptr(w), (const float*)ptr(sc), (const float*)ptr(b), T, n,
                                 (int32_t)K, row_type(out), (int32_t)variant, ptr(ws), bytes, nullptr, ptr(y), stream),
             "linear_int8");
  return y;
}

// ------------------------------------------------------------------------------------ norms
// the inputs as the C calls take them; holds the tensors, some of which may be copies, until the launch
struct NormInputs {
  Rows y, r, g;
  Tensor w, wn;
  int32_t bits = 0, kind;
  int dt;
  NormInputs(const Tensor& y_, const OptTensor& residual, const OptTensor& weight, const OptTensor& gate, const OptTensor& next, int32_t kind_)
      : y(rows_of(y_)), r{}, g{}, kind(kind_), dt(row_type(y_.scalar_type())) {
    if (residual) r = rows_of(*residual);
    if (weight) w = packed(*weight);
    if (next) wn = packed(*next);
    if (gate) {
      if (kind == B200MOE_GATE_FULL) g = rows_of(*gate); else { g.t = packed(*gate); g.stride = 1; }
    }
    bits = (w.defined() && w.scalar_type() == at::kFloat) | (gate && gate->scalar_type() == at::kFloat) << 1 |
           (wn.defined() && wn.scalar_type() == at::kFloat) << 2;
  }
};

struct NormOutputs {
  Tensor h, n, q, scale, rstd;
};
NormOutputs norm_forward(const Tensor& y, const OptTensor& residual, const OptTensor& weight, const OptTensor& gate, const OptTensor& next,
                         int32_t kind, double alpha, double eps, bool want_h, bool quant, bool save) {
  c10::cuda::CUDAGuard guard(y.device());
  const NormInputs i(y, residual, weight, gate, next, kind);
  const int32_t T = as_i32(i.y.T, "the number of rows");
  NormOutputs o;
  if (want_h) o.h = empty_as(y, y.sizes(), y.scalar_type());
  if (quant) {
    o.q = empty_as(y, y.sizes(), at::kChar);
    o.scale = empty_as(y, y.sizes().slice(0, y.dim() - 1), at::kFloat);
  } else if (next) {
    o.n = empty_as(y, y.sizes(), y.scalar_type());
  }
  if (save) o.rstd = empty_as(y, {2 * i.y.T}, at::kFloat);
  call_check(b200moe_block_norm(ptr(i.y.t), i.y.stride, ptr(i.r.t), i.r.stride, ptr(i.w), ptr(i.g.t), i.g.stride, ptr(i.wn), T, (int32_t)i.y.H,
                                i.dt, i.bits, kind, (float)alpha, (float)eps, ptr(o.h), ptr(o.n), ptr(o.q), (float*)ptr(o.scale),
                                (float*)ptr(o.rstd), stream_of(y)), "block_norm");
  return o;
}

void need_first_order(const variable_list& up, const char* what) {
  need_eager(what);
  bool any = false;
  for (const Tensor& g : up) any = any || has_tangent(g);
  need_no_tangent(any, what);
}

// Gradients of a backward pass that is itself being recorded: nothing here can be differentiated again, and says so.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g.set_requires_grad(true);     // so that the node below stands behind them
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is not twice differentiable", (int64_t)grads.size());
  return (*node)(std::move(grads));
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& y, const OptTensor& residual, const OptTensor& weight, const OptTensor& gate,
                               const OptTensor& next, int64_t kind, double alpha, double eps, bool want_h) {
    NormOutputs o = norm_forward(y, residual, weight, gate, next, (int32_t)kind, alpha, eps, want_h, false, true);
    auto or_none = [](const OptTensor& t) { return t ? *t : Tensor(); };
    ctx->save_for_backward({y, or_none(residual), or_none(weight), or_none(gate), or_none(next), o.rstd});
    ctx->saved_data["how"] = std::make_tuple(kind, alpha, want_h);
    ctx->set_materialize_grads(false);
    variable_list out;
    if (want_h) out.push_back(o.h);
    if (next) out.push_back(o.n);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    need_first_order(up, "the block norm's backward pass");
    const auto s = ctx->get_saved_variables();
    const auto [kind, alpha, want_h] = ctx->saved_data["how"].to<std::tuple<int64_t, double, bool>>();
    const Tensor& y = s[0];
    auto opt = [&](int k) { return s[k].defined() ? OptTensor(s[k]) : OptTensor(); };
    variable_list grads(9);
    {
      at::NoGradGuard no_grad;
      c10::cuda::CUDAGuard guard(y.device());
      const NormInputs i(y, opt(1), opt(2), opt(3), opt(4), (int32_t)kind);
      const Tensor dh = want_h ? upstream(up[0]) : Tensor(), dn = s[4].defined() ? upstream(up[want_h ? 1 : 0]) : Tensor();
      size_t edge = 0;                       // edges are numbered over the tensors that are there
      for (int k = 0; k < 5; ++k)
        if (s[k].defined() && ctx->needs_input_grad(edge++)) grads[k] = empty_as(s[k], s[k].sizes(), s[k].scalar_type());
      Tensor ws;
      int64_t bytes = 0;
      const int32_t T = (int32_t)i.y.T, H = (int32_t)i.y.H;
      if (grads[2].defined() || grads[4].defined() || (grads[3].defined() && kind == B200MOE_GATE_CHANNEL)) {
        call_check(b200moe_block_norm_bwd_workspace(T, H, i.dt, &bytes), "block_norm_bwd_workspace");
        ws = empty_as(y, {bytes}, at::kByte);
      }
      call_check(b200moe_block_norm_bwd(ptr(i.y.t), i.y.stride, ptr(i.r.t), i.r.stride, ptr(i.w), ptr(i.g.t), i.g.stride, ptr(i.wn), T, H, i.dt,
                                        i.bits, (int32_t)kind, (float)alpha, (const float*)ptr(s[5]), ptr(dh), ptr(dn), ptr(grads[0]),
                                        ptr(grads[1]), ptr(grads[2]), ptr(grads[3]), ptr(grads[4]), ptr(ws), bytes, stream_of(y)),
                 "block_norm_bwd");
    }
    return once(std::move(grads), "the block norm");
  }
};

// -> [h] [n | q, scale]: h where want_h, n where next is given and not quant
variable_list block_norm(const Tensor& y, const OptTensor& residual, const OptTensor& weight, const OptTensor& gate, const OptTensor& next,
                         double alpha, double eps, bool want_h, bool quant, const std::string& what) {
  need_cuda(y, what.c_str());
  need_eager(what.c_str());
  need_no_tangent(has_tangent(y) || has_tangent(residual) || has_tangent(weight) || has_tangent(gate) || has_tangent(next), what.c_str());
  const auto dtype = y.scalar_type();
  TYPE_CHECK(row_type(dtype) >= 0, "rows must be bfloat16, float16 or float32");
  const int64_t H = y.dim() ? y.size(-1) : 0;
  VALUE_CHECK(H >= 1 && H <= kMaxRow, "rows must have 1 to ", kMaxRow, " values");
  VALUE_CHECK(!residual || (residual->scalar_type() == dtype && residual->sizes() == y.sizes()), "residual must have the rows' shape and type");
  for (const OptTensor* w : {&weight, &next})
    VALUE_CHECK(!*w || ((*w)->dim() == 1 && (*w)->size(0) == H && ((*w)->scalar_type() == dtype || (*w)->scalar_type() == at::kFloat)),
                "weights must hold ", H, " values of the rows' type or float32");
  int32_t kind = B200MOE_GATE_NONE;
  if (gate) {
    TYPE_CHECK(gate->scalar_type() == dtype || gate->scalar_type() == at::kFloat, "gate must be of the rows' type or float32");
    auto per_token = y.sizes().vec();
    per_token.back() = 1;
    if (gate->dim() == 1 && gate->size(0) == H) kind = B200MOE_GATE_CHANNEL;
    else if (gate->sizes() == y.sizes()) kind = B200MOE_GATE_FULL;
    else if (gate->sizes() == at::IntArrayRef(per_token)) kind = B200MOE_GATE_TOKEN;
    else VALUE_CHECK(false, "gate must be [", H, "], [..., 1] or [..., ", H, "] over the rows' leading sizes");
  }
  VALUE_CHECK(on(residual, y) && on(weight, y) && on(gate, y) && on(next, y), "all tensors must be on one device");
  const bool grad = at::GradMode::is_enabled() &&
                    (y.requires_grad() || wants_grad(residual) || wants_grad(weight) || wants_grad(gate) || wants_grad(next));
  if (quant) need_no_grad(grad, "8-bit rows have no gradient");
  if (grad) return BlockNorm::apply(y, residual, weight, gate, next, (int64_t)kind, alpha, eps, want_h);
  NormOutputs o = norm_forward(y, residual, weight, gate, next, kind, alpha, eps, want_h, quant, false);
  variable_list out;
  if (want_h) out.push_back(o.h);
  if (o.n.defined()) out.push_back(o.n);
  if (quant) {
    out.push_back(o.q);
    out.push_back(o.scale);
  }
  return out;
}

// ------------------------------------------------------------------------------------ router
// what the backward pass needs, in one allocation: lse [2, T], seg [T], coef [S, E], stats [2]
struct Saved {
  Tensor t;
  float* lse = nullptr;
  int32_t* seg = nullptr;
  float *coef = nullptr, *stats = nullptr;
  static int64_t words(int64_t T, int64_t S, int64_t E) { return 3 * T + S * E + 2; }
  Saved() = default;
  Saved(Tensor t_, int64_t T, int64_t S, int64_t E) : t(std::move(t_)) {
    lse = t.data_ptr<float>();
    seg = (int32_t*)(lse + 2 * T);
    coef = lse + 3 * T;
    stats = coef + S * E;
  }
};
struct RouterResult {
  variable_list out;      // weights, ids, counts, balance loss, z loss
  Tensor saved;
};
RouterResult router_forward(const Tensor& logits, int64_t K, int64_t scoring, bool renorm, const OptTensor& mask, const OptTensor& cu, bool save) {
  c10::cuda::CUDAGuard guard(logits.device());
  const Rows x = rows_of(logits);
  const int64_t T = x.T, E = x.H, S = cu ? cu->size(0) - 1 : 1;
  as_i32(T, "the number of tokens"), as_i32(S, "the number of sequences");
  const Tensor m = mask ? packed(*mask) : Tensor(), c = cu ? packed(*cu) : Tensor();
  int64_t bytes = 0;
  call_check(b200moe_router_workspace((int32_t)T, (int32_t)E, (int32_t)S, &bytes), "router_workspace");
  RouterResult r;
  Tensor weights = empty_as(logits, {T, K}, at::kFloat), ids = empty_as(logits, {T, K}, at::kInt);
  Tensor counts = cu ? empty_as(logits, {S, E}, at::kInt) : empty_as(logits, {E}, at::kInt);
  Tensor balance = empty_as(logits, {}, at::kFloat), z = empty_as(logits, {}, at::kFloat);
  Tensor ws = empty_as(logits, {bytes}, at::kByte);
  Saved s;
  if (save) s = Saved(empty_as(logits, {Saved::words(T, S, E)}, at::kFloat), T, S, E);
  call_check(b200moe_router_forward(ptr(x.t), x.stride, (int32_t)T, (int32_t)E, (int32_t)K, row_type(logits.scalar_type()), (int32_t)scoring,
                                    renorm, ptr(m), (const int32_t*)ptr(c), (int32_t)S, weights.data_ptr<float>(), ids.data_ptr<int32_t>(),
                                    counts.data_ptr<int32_t>(), balance.data_ptr<float>(), z.data_ptr<float>(), s.lse, s.seg, s.coef, s.stats,
                                    ptr(ws), bytes, stream_of(logits)), "router_forward");
  r.out = {weights, ids, counts, balance, z};
  r.saved = s.t;
  return r;
}

struct Router : torch::autograd::Function<Router> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t K, int64_t scoring, bool renorm, const OptTensor& mask,
                               const OptTensor& cu) {
    RouterResult r = router_forward(logits, K, scoring, renorm, mask, cu, true);
    // the logits are saved as such, so that a change in place is noticed
    ctx->save_for_backward({logits, r.out[0], r.out[1], r.saved});
    ctx->saved_data["how"] = std::make_tuple(K, scoring, renorm, cu ? cu->size(0) - 1 : int64_t(1));
    ctx->mark_non_differentiable({r.out[1], r.out[2]});
    ctx->set_materialize_grads(false);
    return r.out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    need_first_order(up, "fused_router's backward pass");
    const auto s = ctx->get_saved_variables();
    const auto [K, scoring, renorm, S] = ctx->saved_data["how"].to<std::tuple<int64_t, int64_t, bool, int64_t>>();
    const Tensor& logits = s[0];
    variable_list grads(6);
    {
      at::NoGradGuard no_grad;
      c10::cuda::CUDAGuard guard(logits.device());
      const Rows x = rows_of(logits);
      const Saved k(s[3], x.T, S, x.H);
      const Tensor dw = upstream(up[0]), db = upstream(up[3]), dz = upstream(up[4]);
      grads[0] = empty_as(logits, logits.sizes(), logits.scalar_type());
      call_check(b200moe_router_backward(ptr(x.t), x.stride, (int32_t)x.T, (int32_t)x.H, (int32_t)K, row_type(logits.scalar_type()),
                                         (int32_t)scoring, renorm, k.lse, k.seg, k.coef, k.stats, s[2].data_ptr<int32_t>(),
                                         s[1].data_ptr<float>(), (const float*)ptr(dw), (const float*)ptr(db), (const float*)ptr(dz),
                                         ptr(grads[0]), stream_of(logits)), "router_backward");
    }
    return once(std::move(grads), "fused_router");
  }
};

variable_list router(const Tensor& logits, int64_t K, bool renorm, const std::string& scoring, const OptTensor& mask, const OptTensor& cu) {
  need_cuda(logits, "fused_router");
  need_eager("fused_router");
  need_no_tangent(has_tangent(logits), "fused_router");
  TYPE_CHECK(row_type(logits.scalar_type()) >= 0, "gating_output must be bfloat16, float16 or float32");
  VALUE_CHECK(logits.dim() == 2, "gating_output must be [T, E]");
  const int64_t T = logits.size(0), E = logits.size(1);
  VALUE_CHECK(E >= 1 && E <= kMaxExperts, E, " experts: 1 to ", kMaxExperts, " are supported");
  VALUE_CHECK(K >= 1 && K <= std::min(E, kMaxTopk), "topk=", K, ": 1 to ", std::min(E, kMaxTopk), " for ", E, " experts");
  const int64_t how = scoring == "softmax" ? 0 : scoring == "sigmoid" ? 1 : -1;
  VALUE_CHECK(how >= 0, "scoring='", scoring, "': 'softmax' or 'sigmoid'");
  VALUE_CHECK(!mask || (mask->scalar_type() == at::kBool && mask->dim() == 1 && mask->size(0) == T && on(mask, logits)),
              "token_mask must be a bool tensor [T] on the logits' device");
  VALUE_CHECK(!cu || (cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->size(0) >= 2 && on(cu, logits)),
              "cu_seqlens must be an int32 tensor [S+1] on the logits' device");
  if (at::GradMode::is_enabled() && logits.requires_grad()) return Router::apply(logits, K, how, renorm, mask, cu);
  return router_forward(logits, K, how, renorm, mask, cu, false).out;
}

PyObject* error_class = nullptr;

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("set_error", [](py::object cls) { error_class = cls.release().ptr(); });      // held for good
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const B200Error& e) {
      PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
    }
  });
  // the interpreter is free while a call checks, allocates and launches
  using no_gil = py::call_guard<py::gil_scoped_release>;
  m.def("quantize_int8", &quantize_int8, no_gil());
  m.def("linear_int8", &linear_int8, no_gil());
  m.def("block_norm", &block_norm, no_gil());
  m.def("router", &router, no_gil());
}
