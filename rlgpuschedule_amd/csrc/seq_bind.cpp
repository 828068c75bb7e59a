// Torch bindings of the sequence operators: argument checks, output and
// scratch allocation, and autograd. Host code only; the kernels are in
// layer_norm.hip, gated_scan.hip and logprob.hip (seq_api.h).
//
// In C++ because the calls are short: a step of 256 x 256 values runs for a
// few microseconds, and a backward pass written in Python spends more than
// that on taking the interpreter's lock in autograd's thread.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <sstream>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "seq_api.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

namespace {

constexpr int64_t kMaxTopK = 64;  // logprob.hip

template <typename E, typename... A>
[[noreturn]] void fail(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw E(s.str());
}
#define VALUE_CHECK(ok, ...) \
  if (!(ok)) fail<py::value_error>(__VA_ARGS__)
#define TYPE_CHECK(ok, ...) \
  if (!(ok)) fail<py::type_error>(__VA_ARGS__)

void done_with(int rc, const char* what) {
  if (rc != 0) fail<std::runtime_error>(what, " failed: ", rc);
}

// element type codes of seq_common.h
int type_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default:
      fail<py::type_error>(name, " must be float32, bfloat16 or float16, got ",
                           t.scalar_type());
  }
}

bool is_flag(const Tensor& t) {
  return t.scalar_type() == at::kByte || t.scalar_type() == at::kBool;
}

void same_device(const Tensor& x, const Tensor& t, const char* name) {
  VALUE_CHECK(t.device() == x.device(), name, " is on ", t.device(),
              ", expected ", x.device());
}
void same_device(const Tensor& x, const MaybeTensor& t, const char* name) {
  if (t) same_device(x, *t, name);
}

// Whether a tensor's storage holds anything. Those of fake and wrapped tensors
// do not, and what is freed or shrunk keeps its views: torch hands out a
// pointer for each all the same.
bool has_memory(const Tensor& t) {
  return t.numel() == 0 || t.storage().data() != nullptr;
}

[[noreturn]] void no_memory(const Tensor& t, const char* name) {
  fail<std::runtime_error>(name, " of shape ", t.sizes(),
                           " has no memory on the GPU (it is fake, wrapped or "
                           "freed, or a fake mode is active)");
}

// An input whose storage reaches as far as its elements: asked before anything,
// a copy of torch's too, reads it.
const Tensor& held(const Tensor& t) {
  if (t.numel() == 0) return t;
  if (!has_memory(t)) no_memory(t, "an input");
  const auto sizes = t.sizes(), strides = t.strides();
  int64_t last = t.storage_offset();
  for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
  if ((last + 1) * (int64_t)t.element_size() > (int64_t)t.storage().nbytes())
    no_memory(t, "an input");
  return t;
}

void on_gpu(const Tensor& x, const char* name) {
  VALUE_CHECK(x.is_cuda(), name, " must be on a GPU, got ", x.device());
  if (!has_memory(x)) no_memory(x, name);
}

struct Place {
  int device;
  void* stream;
  explicit Place(const Tensor& x)
      : device(x.get_device()),
        stream(c10::hip::getCurrentHIPStream(x.get_device()).stream()) {}
};

const void* ptr(const Tensor& t) {
  if (!has_memory(t)) no_memory(t, "an input");
  return t.const_data_ptr();
}
const void* ptr(const MaybeTensor& t) {
  return t && t->defined() ? ptr(*t) : nullptr;
}
void* out_ptr(const Tensor& t) {
  if (!t.defined()) return nullptr;
  if (!has_memory(t)) no_memory(t, "an output");
  return t.mutable_data_ptr();
}
float* f32_ptr(const Tensor& t) { return (float*)out_ptr(t); }
MaybeTensor maybe(const Tensor& t) {
  return t.defined() ? MaybeTensor(t) : std::nullopt;
}
// Values as memory holds them: torch notes a conjugate's imaginary part as to
// be negated.
Tensor plain(const Tensor& t) {
  return held(t).is_neg() ? t.resolve_neg() : t;
}
MaybeTensor packed(const MaybeTensor& t) {
  return t && t->defined() ? MaybeTensor(plain(*t).contiguous())
                           : std::nullopt;
}

Tensor f32(const Tensor& x, at::IntArrayRef size) {
  return at::empty(size, x.options().dtype(at::kFloat).requires_grad(false));
}

// t [..., D] as rows of unit stride and the elements from one row to the
// next. Leading dims that no single stride walks, and last dims of another
// stride, are copied.
std::pair<Tensor, int64_t> rows_of(const Tensor& t_) {
  const Tensor t = plain(t_);
  const int64_t d = t.size(-1);
  if (t.is_contiguous()) return {t, d};
  Tensor r = t.reshape({-1, d});
  if (d > 1 && r.stride(1) != 1) r = r.contiguous();
  return {r, r.stride(0)};
}

// t [..., E, H] with neighbouring columns and environments within reach.
Tensor reachable(const Tensor& t_) {
  const Tensor t = plain(t_);
  const bool near = t.stride(-2) <= rlsched_scan_reach(t.size(-1));
  const bool unit = t.size(-1) == 1 || t.stride(-1) == 1;
  return near && unit ? t : t.contiguous();
}

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const MaybeTensor& t) { return t && t->requires_grad(); }

// A leaf's gradient is accumulated on the stream that was current when the
// leaf entered a graph that is still alive. Where that is another stream
// than the one being captured, the backward pass has to synchronise with it
// at its end, in the middle of the capture, and the process ends. Refused
// here, where a call is still refused: `t` leads to such a leaf.
void refuse_foreign_leaves(const Tensor& t, const c10::hip::HIPStream& s,
                           std::unordered_set<torch::autograd::Node*>& seen) {
  namespace ag = torch::autograd;
  std::vector<std::shared_ptr<ag::Node>> todo;
  if (t.grad_fn()) {
    todo.push_back(t.grad_fn());
  } else if (auto leaf = ag::impl::try_get_grad_accumulator(t)) {
    todo.push_back(leaf);
  }
  while (!todo.empty()) {
    auto node = todo.back();
    todo.pop_back();
    if (!seen.insert(node.get()).second) continue;
    for (const auto& e : node->next_edges())
      if (e.function) todo.push_back(e.function);
    if (node->num_outputs() != 0) continue;  // not a leaf's accumulation
    const auto at = node->stream();
    if (at && at->device_type() == c10::kCPU) continue;
    if (at && (at->id() != s.id() || at->device_index() != s.device_index()))
      fail<std::runtime_error>(
          "an autograd graph of the same leaves, made on another stream, is "
          "alive: a backward pass cannot be captured beside it. Release that "
          "graph (its outputs and losses) before the capture, or use the "
          "operator's _fwd and _bwd functions.");
  }
}

template <typename... T>
void check_capture(const Tensor& x, const T&... rest) {
  const auto s = c10::hip::getCurrentHIPStream(x.get_device());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s.stream(), &status) != hipSuccess ||
      status == hipStreamCaptureStatusNone)
    return;
  std::unordered_set<torch::autograd::Node*> seen;
  auto visit = [&](const MaybeTensor& t) {
    if (wants_grad(t)) refuse_foreign_leaves(*t, s, seen);
  };
  visit(x);
  (visit(MaybeTensor(rest)), ...);
}

// Forward-mode derivatives would be dropped where nothing requires a gradient.
void no_tangent(const char* name, std::initializer_list<const Tensor*> all) {
  for (const Tensor* t : all)
    if (t && t->_fw_grad(0).defined())
      fail<std::runtime_error>(name, " has no forward-mode derivative");
}
const Tensor* given(const MaybeTensor& t) { return t ? &*t : nullptr; }

void once(const char* name) {
  if (at::GradMode::is_enabled())
    fail<std::runtime_error>("the backward pass of ", name,
                             " cannot be differentiated (create_graph)");
}

// ------------------------------------------------------------- layer norm
struct NormTypes {
  int x, w;
};

NormTypes check_norm(const Tensor& x, const MaybeTensor& w,
                     const MaybeTensor& b) {
  VALUE_CHECK(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) < (1ll << 31),
              "x must have a last dimension of 1 to 2**31 - 1, got shape ",
              x.sizes());
  NormTypes t;
  t.x = t.w = type_code(x, "x");
  const Tensor* first = nullptr;
  const std::pair<const char*, const MaybeTensor*> both[] = {{"weight", &w},
                                                             {"bias", &b}};
  for (const auto& [name, p] : both) {
    if (!*p) continue;
    const Tensor& v = **p;
    VALUE_CHECK(v.dim() == 1 && v.size(0) == x.size(-1), name,
                " must have shape [", x.size(-1), "], got ", v.sizes());
    TYPE_CHECK(v.scalar_type() == x.scalar_type() ||
                   v.scalar_type() == at::kFloat,
               name, " must be ", x.scalar_type(), " or Float, got ",
               v.scalar_type());
    TYPE_CHECK(!first || first->scalar_type() == v.scalar_type(),
               "weight and bias must have one type, got ",
               first->scalar_type(), " and ", v.scalar_type());
    same_device(x, v, name);
    t.w = type_code(v, name);
    first = &v;
  }
  return t;
}

std::tuple<Tensor, Tensor, Tensor> norm_fwd(const Tensor& x,
                                            const MaybeTensor& weight,
                                            const MaybeTensor& bias,
                                            double eps, bool keep) {
  const NormTypes t = check_norm(x, weight, bias);
  on_gpu(x, "x");
  const int64_t d = x.size(-1), rows = x.numel() / d;
  Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
  Tensor mean, rstd;
  if (keep) {
    mean = f32(x, {rows});
    rstd = f32(x, {rows});
  }
  const auto [xr, stride] = rows_of(x);
  const MaybeTensor w = packed(weight), b = packed(bias);
  const Place at(x);
  done_with(rlsched_norm_fwd(at.device, at.stream, ptr(xr), ptr(w), ptr(b),
                             out_ptr(y), f32_ptr(mean), f32_ptr(rstd), rows, d,
                             stride, eps, t.x, t.w),
            "rlsched_norm_fwd");
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> norm_bwd(
    const Tensor& dy, const Tensor& x, const MaybeTensor& weight,
    const Tensor& mean, const Tensor& rstd,
    const std::optional<at::ScalarType>& wtype, bool need_dx, bool need_dw,
    bool need_db) {
  NormTypes t = check_norm(x, weight, std::nullopt);
  at::ScalarType wt = weight ? weight->scalar_type() : x.scalar_type();
  if (!weight && wtype) {
    wt = *wtype;
    TYPE_CHECK(wt == x.scalar_type() || wt == at::kFloat, "wdtype must be ",
               x.scalar_type(), " or Float, got ", wt);
    t.w = wt == x.scalar_type() ? t.x : 0;
  }
  VALUE_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(),
              "dy must have x's shape and type, got ", dy.sizes(), " ",
              dy.scalar_type());
  const int64_t d = x.size(-1), rows = x.numel() / d;
  const std::pair<const char*, const Tensor*> stats[] = {{"mean", &mean},
                                                         {"rstd", &rstd}};
  for (const auto& [name, s] : stats) {
    VALUE_CHECK(s->dim() == 1 && s->size(0) == rows &&
                    s->scalar_type() == at::kFloat && s->is_contiguous(),
                name, " must be contiguous float32 [", rows, "]");
    same_device(x, *s, name);
  }
  same_device(x, dy, "dy");
  on_gpu(x, "x");
  Tensor dx, dw, db, partial;
  const auto like_x = x.options().requires_grad(false);
  if (need_dx) dx = at::empty(x.sizes(), like_x);
  if (need_dw) dw = at::empty({d}, like_x.dtype(wt));
  if (need_db) db = at::empty({d}, like_x.dtype(wt));
  if (need_dw || need_db)
    partial = f32(x, {2 * rlsched_norm_parts(rows, d, t.x) * d});
  const auto [xr, xs] = rows_of(x);
  const auto [dyr, dys] = rows_of(dy);
  const MaybeTensor w = packed(weight);
  const Place at(x);
  done_with(
      rlsched_norm_bwd(at.device, at.stream, ptr(dyr), ptr(xr), ptr(w),
                       (const float*)ptr(held(mean)),
                       (const float*)ptr(held(rstd)),
                       out_ptr(dx), out_ptr(dw), out_ptr(db), f32_ptr(partial),
                       rows, d, xs, dys, t.x, t.w),
      "rlsched_norm_bwd");
  return {dx, dw, db};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const MaybeTensor& weight, const MaybeTensor& bias,
                        double eps) {
    auto [y, mean, rstd] = norm_fwd(x, weight, bias, eps, true);
    ctx->save_for_backward(
        {x, weight ? *weight : Tensor(), mean, rstd});
    ctx->saved_data["weight"] = weight.has_value();
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["type"] =
        (int64_t)(bias ? bias->scalar_type() : x.scalar_type());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("layer_norm");
    const auto saved = ctx->get_saved_variables();
    const bool has_w = ctx->saved_data["weight"].toBool();
    const bool has_b = ctx->saved_data["bias"].toBool();
    // gradients are numbered over the tensors that were given
    const bool need_dw = has_w && ctx->needs_input_grad(1);
    const bool need_db = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    auto [dx, dw, db] = norm_bwd(
        grads[0], saved[0], has_w ? MaybeTensor(saved[1]) : std::nullopt,
        saved[2], saved[3], type, ctx->needs_input_grad(0), need_dw, need_db);
    return {dx, dw, db, Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight,
                  const MaybeTensor& bias, double eps) {
  no_tangent("layer_norm", {&x, given(weight), given(bias)});
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(weight) || wants_grad(bias))) {
    check_norm(x, weight, bias);
    on_gpu(x, "x");
    check_capture(x, weight, bias);
    return LayerNorm::apply(x, weight, bias, eps);
  }
  return std::get<0>(norm_fwd(x, weight, bias, eps, false));
}

// ------------------------------------------------------------- gated scan
// gate, x of `dims` dimensions; h of the last two; done of all but the last.
int check_scan(const Tensor& gate, const Tensor& x, const MaybeTensor& h,
               const MaybeTensor& done, int64_t dims, const char* hname) {
  VALUE_CHECK(x.dim() == dims && gate.sizes() == x.sizes() &&
                  gate.scalar_type() == x.scalar_type(),
              "gate and x must have one type and one ", dims,
              "-dim shape, got ", gate.sizes(), " ", gate.scalar_type(),
              " and ", x.sizes(), " ", x.scalar_type());
  const int code = type_code(x, "x");
  const int64_t E = x.size(-2), H = x.size(-1);
  VALUE_CHECK(E == 0 || H < (1ll << 28) / E, E, " x ", H,
              " columns: fewer than 2**28 are supported");
  if (h) {
    VALUE_CHECK(h->dim() == 2 && h->size(0) == E && h->size(1) == H &&
                    h->scalar_type() == at::kFloat,
                hname, " must be float32 [", E, ", ", H, "], got ", h->sizes(),
                " ", h->scalar_type());
    same_device(x, *h, hname);
  }
  if (done) {
    VALUE_CHECK(done->sizes() == x.sizes().slice(0, dims - 1) &&
                    is_flag(*done),
                "done must be uint8 or bool ", x.sizes().slice(0, dims - 1),
                ", got ", done->sizes(), " ", done->scalar_type());
    same_device(x, *done, "done");
  }
  same_device(x, gate, "gate");
  return code;
}

std::tuple<Tensor, Tensor, Tensor> scan_fwd(const Tensor& gate_,
                                            const Tensor& x_,
                                            const MaybeTensor& h0_,
                                            const MaybeTensor& done_,
                                            bool keep) {
  const int type = check_scan(gate_, x_, h0_, done_, 3, "h0");
  on_gpu(x_, "x");
  const int64_t T = x_.size(0), E = x_.size(1), H = x_.size(2);
  Tensor hs = at::empty({T, E, H}, x_.options().requires_grad(false));
  Tensor h_last = f32(x_, {E, H}), states;
  if (keep) states = f32(x_, {rlsched_scan_states(T), E, H});
  Tensor scratch;
  if (const int64_t n = rlsched_scan_scratch(T, E, H, type, 0))
    scratch = f32(x_, {n});
  const Tensor gate = reachable(gate_), x = reachable(x_);
  const MaybeTensor h0 = packed(h0_), done = packed(done_);
  const Place at(x);
  done_with(
      rlsched_scan_fwd(at.device, at.stream, ptr(gate), ptr(x),
                       (const float*)ptr(h0), (const uint8_t*)ptr(done),
                       out_ptr(hs), f32_ptr(h_last), f32_ptr(states),
                       f32_ptr(scratch), T, E, H, gate.stride(0),
                       gate.stride(1), x.stride(0), x.stride(1), type),
      "rlsched_scan_fwd");
  return {hs, h_last, states};
}

std::tuple<Tensor, Tensor, Tensor> scan_bwd(
    const MaybeTensor& dhs_, const MaybeTensor& dh_last_, const Tensor& gate_,
    const Tensor& x_, const Tensor& states, const MaybeTensor& done_,
    bool need_dh0) {
  const int type = check_scan(gate_, x_, dh_last_, done_, 3, "dh_last");
  const int64_t T = x_.size(0), E = x_.size(1), H = x_.size(2);
  if (dhs_) {
    VALUE_CHECK(dhs_->sizes() == x_.sizes() &&
                    dhs_->scalar_type() == x_.scalar_type(),
                "dhs must have x's shape and type, got ", dhs_->sizes(), " ",
                dhs_->scalar_type());
    same_device(x_, *dhs_, "dhs");
  }
  VALUE_CHECK(states.dim() == 3 && states.size(0) == rlsched_scan_states(T) &&
                  states.size(1) == E && states.size(2) == H &&
                  states.is_contiguous() && states.scalar_type() == at::kFloat,
              "states must be gated_scan_fwd's, of these inputs");
  same_device(x_, states, "states");
  on_gpu(x_, "x");
  const auto like_x = x_.options().requires_grad(false);
  Tensor dgate = at::empty({T, E, H}, like_x);
  Tensor dx = at::empty({T, E, H}, like_x), dh0;
  if (need_dh0) dh0 = f32(x_, {E, H});
  Tensor scratch;
  if (const int64_t n = rlsched_scan_scratch(T, E, H, type, 1))
    scratch = f32(x_, {n});
  const Tensor gate = reachable(gate_), x = reachable(x_);
  MaybeTensor dhs;
  if (dhs_) dhs = reachable(*dhs_);
  const MaybeTensor dh_last = packed(dh_last_), done = packed(done_);
  const Place at(x);
  done_with(
      rlsched_scan_bwd(at.device, at.stream, ptr(dhs),
                       (const float*)ptr(dh_last), ptr(gate),
                       ptr(x), (const float*)ptr(held(states)),
                       (const uint8_t*)ptr(done), out_ptr(dgate), out_ptr(dx),
                       f32_ptr(dh0), f32_ptr(scratch), T, E, H,
                       gate.stride(0), gate.stride(1), x.stride(0),
                       x.stride(1), dhs ? dhs->stride(0) : 0,
                       dhs ? dhs->stride(1) : 0, type),
      "rlsched_scan_bwd");
  return {dgate, dx, dh0};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& gate,
                               const Tensor& x, const MaybeTensor& h0,
                               const MaybeTensor& done) {
    ctx->set_materialize_grads(false);
    auto [hs, h_last, states] = scan_fwd(gate, x, h0, done, true);
    ctx->save_for_backward({gate, x, states, done ? *done : Tensor()});
    ctx->saved_data["h0"] = h0.has_value();
    return {hs, h_last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("gated_scan");
    if (!grads[0].defined() && !grads[1].defined())
      return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    const bool need_dh0 =
        ctx->saved_data["h0"].toBool() && ctx->needs_input_grad(2);
    auto [dgate, dx, dh0] = scan_bwd(maybe(grads[0]), maybe(grads[1]), s[0],
                                     s[1], s[2], maybe(s[3]), need_dh0);
    return {dgate, dx, dh0, Tensor()};
  }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& gate, const Tensor& x,
                                      const MaybeTensor& h0,
                                      const MaybeTensor& done) {
  no_tangent("gated_scan", {&gate, &x, given(h0)});
  if (at::GradMode::is_enabled() &&
      (wants_grad(gate) || wants_grad(x) || wants_grad(h0))) {
    check_scan(gate, x, h0, done, 3, "h0");
    on_gpu(x, "x");
    check_capture(x, gate, h0);
    auto out = GatedScan::apply(gate, x, h0, done);
    return {out[0], out[1]};
  }
  auto [hs, h_last, states] = scan_fwd(gate, x, h0, done, false);
  return {hs, h_last};
}

Tensor scan_step(const Tensor& gate_, const Tensor& x_, Tensor h,
                 const MaybeTensor& done_) {
  const int type = check_scan(gate_, x_, h, done_, 2, "h");
  VALUE_CHECK(h.is_contiguous() && !h.is_neg(),
              "h is updated in place: it must be contiguous");
  no_tangent("gated_scan_step", {&gate_, &x_, &h});
  VALUE_CHECK(!at::GradMode::is_enabled() ||
                  !(wants_grad(gate_) || wants_grad(x_) || wants_grad(h)),
              "gated_scan_step has no derivative: gate, x and h must not "
              "require a gradient (call it under torch.no_grad())");
  for (const Tensor* t : {&gate_, &x_, given(done_)})
    VALUE_CHECK(!t || !h.is_alias_of(*t) ||
                    at::get_overlap_status(h, *t) == at::MemOverlapStatus::No,
                "h is updated in place: it must not share memory with gate, "
                "x or done");
  on_gpu(x_, "x");
  held(h);
  h.unsafeGetTensorImpl()->bump_version();
  const int64_t E = x_.size(0), H = x_.size(1);
  Tensor hs = at::empty({E, H}, x_.options().requires_grad(false));
  const Tensor gate = reachable(gate_), x = reachable(x_);
  const MaybeTensor done = packed(done_);
  const Place at(x);
  done_with(rlsched_scan_step(at.device, at.stream, ptr(gate), ptr(x),
                              (const uint8_t*)ptr(done), f32_ptr(h),
                              out_ptr(hs), E, H, gate.stride(0), x.stride(0),
                              type),
            "rlsched_scan_step");
  return hs;
}

// ------------------------------------------------------ log probabilities
int check_logp(const Tensor& logits, const Tensor& actions,
               const MaybeTensor& mask, int64_t top_k) {
  VALUE_CHECK(logits.dim() >= 1 && logits.size(-1) > 0 &&
                  logits.size(-1) <= (1ll << 30),
              "logits must have 1 to 2**30 actions, got shape ",
              logits.sizes());
  const int code = type_code(logits, "logits");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  VALUE_CHECK(actions.sizes() == lead && actions.scalar_type() == at::kLong,
              "actions must be int64 ", lead, ", got ", actions.sizes(), " ",
              actions.scalar_type());
  if (mask) {
    VALUE_CHECK(mask->sizes() == logits.sizes() && is_flag(*mask),
                "mask must be uint8 or bool ", logits.sizes(), ", got ",
                mask->sizes(), " ", mask->scalar_type());
    same_device(logits, *mask, "mask");
  }
  VALUE_CHECK(top_k >= 0 && top_k <= kMaxTopK && top_k <= logits.size(-1),
              "top_k must be 0 to ", kMaxTopK,
              " and at most the number of actions, got ", top_k);
  same_device(logits, actions, "actions");
  return code;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> logp_fwd(
    const Tensor& logits, const Tensor& actions_, const MaybeTensor& mask,
    int64_t top_k, bool keep) {
  const int type = check_logp(logits, actions_, mask, top_k);
  on_gpu(logits, "logits");
  const int64_t A = logits.size(-1), rows = logits.numel() / A;
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  Tensor logp = f32(logits, lead), entropy = f32(logits, lead);
  Tensor stats, top_logp, top_index;
  if (keep) stats = f32(logits, {rows, 3});
  if (top_k) {
    auto size = lead.vec();
    size.push_back(top_k);
    top_logp = f32(logits, size);
    top_index = at::empty(size, actions_.options().requires_grad(false));
  }
  Tensor scratch;
  if (const int64_t n = rlsched_logp_scratch(rows, A, (int)top_k, type))
    scratch = at::empty(
        {n}, logits.options().dtype(at::kByte).requires_grad(false));
  const auto [xr, xs] = rows_of(logits);
  Tensor mr;
  int64_t ms = 0;
  if (mask) std::tie(mr, ms) = rows_of(*mask);
  const Tensor actions = held(actions_).contiguous();
  const Place at(logits);
  done_with(
      rlsched_logp_fwd(at.device, at.stream, ptr(xr),
                       (const int64_t*)ptr(actions),
                       mask ? (const uint8_t*)ptr(mr) : nullptr,
                       f32_ptr(logp), f32_ptr(entropy), f32_ptr(stats),
                       f32_ptr(top_logp), (int64_t*)out_ptr(top_index),
                       out_ptr(scratch), rows, A, xs, ms, (int)top_k, type),
      "rlsched_logp_fwd");
  return {logp, entropy, stats, top_logp, top_index};
}

Tensor logp_bwd(const MaybeTensor& dlogp_, const MaybeTensor& dentropy_,
                const Tensor& logits, const Tensor& actions_,
                const MaybeTensor& mask, const Tensor& stats) {
  const int type = check_logp(logits, actions_, mask, 0);
  const int64_t A = logits.size(-1), rows = logits.numel() / A;
  const std::pair<const char*, const MaybeTensor*> given[] = {
      {"dlogp", &dlogp_}, {"dentropy", &dentropy_}};
  for (const auto& [name, p] : given) {
    const MaybeTensor& t = *p;
    if (!t) continue;
    VALUE_CHECK(t->sizes() == actions_.sizes() &&
                    t->scalar_type() == at::kFloat,
                name, " must be float32 ", actions_.sizes(), ", got ",
                t->sizes(), " ", t->scalar_type());
    same_device(logits, *t, name);
  }
  VALUE_CHECK(stats.dim() == 2 && stats.size(0) == rows &&
                  stats.size(1) == 3 && stats.scalar_type() == at::kFloat &&
                  stats.is_contiguous(),
              "stats must be action_logprobs_fwd's, of these inputs");
  same_device(logits, stats, "stats");
  on_gpu(logits, "logits");
  Tensor dlogits =
      at::empty(logits.sizes(), logits.options().requires_grad(false));
  const auto [xr, xs] = rows_of(logits);
  Tensor mr;
  int64_t ms = 0;
  if (mask) std::tie(mr, ms) = rows_of(*mask);
  const MaybeTensor dlogp = packed(dlogp_), dentropy = packed(dentropy_);
  const Tensor actions = held(actions_).contiguous();
  const Place at(logits);
  done_with(
      rlsched_logp_bwd(at.device, at.stream, (const float*)ptr(dlogp),
                       (const float*)ptr(dentropy), ptr(xr),
                       (const int64_t*)ptr(actions),
                       mask ? (const uint8_t*)ptr(mr) : nullptr,
                       (const float*)ptr(held(stats)), out_ptr(dlogits), rows,
                       A, xs, ms, type),
      "rlsched_logp_bwd");
  return dlogits;
}

struct ActionLogProbs : torch::autograd::Function<ActionLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits,
                               const Tensor& actions, const MaybeTensor& mask,
                               int64_t top_k) {
    ctx->set_materialize_grads(false);
    auto [logp, entropy, stats, top_logp, top_index] =
        logp_fwd(logits, actions, mask, top_k, true);
    // no output is among them: those are the caller's to change
    ctx->save_for_backward({logits, actions, mask ? *mask : Tensor(), stats});
    if (!top_k) return {logp, entropy};
    ctx->mark_non_differentiable({top_logp, top_index});
    return {logp, entropy, top_logp, top_index};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("action_logprobs");
    if (!grads[0].defined() && !grads[1].defined())
      return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    return {logp_bwd(maybe(grads[0]), maybe(grads[1]), s[0], s[1], maybe(s[2]),
                     s[3]),
            Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, MaybeTensor, MaybeTensor> action_logprobs(
    const Tensor& logits, const Tensor& actions, const MaybeTensor& mask,
    int64_t top_k) {
  no_tangent("action_logprobs", {&logits});
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    check_logp(logits, actions, mask, top_k);
    on_gpu(logits, "logits");
    check_capture(logits);
    auto out = ActionLogProbs::apply(logits, actions, mask, top_k);
    if (!top_k) return {out[0], out[1], std::nullopt, std::nullopt};
    return {out[0], out[1], out[2], out[3]};
  }
  auto [logp, entropy, stats, tl, ti] =
      logp_fwd(logits, actions, mask, top_k, false);
  if (!top_k) return {logp, entropy, std::nullopt, std::nullopt};
  return {logp, entropy, tl, ti};
}

}  // namespace

#ifndef RLS_SOURCE_HASH
#define RLS_SOURCE_HASH "unset"
#endif
extern "C" __attribute__((visibility("default"))) const char*
rlsched_source_hash() {
  return "RLSHASH:" RLS_SOURCE_HASH;
}

PYBIND11_MODULE(librlsched_seq, m) {
  // none of the calls touches Python objects
  using free_gil = py::call_guard<py::gil_scoped_release>;
  m.def("layer_norm", &layer_norm, free_gil());
  m.def("layer_norm_fwd",
        [](const Tensor& x, const MaybeTensor& w, const MaybeTensor& b,
           double eps) { return norm_fwd(x, w, b, eps, true); },
        free_gil());
  m.def("layer_norm_bwd",
        [](const Tensor& dy, const Tensor& x, const MaybeTensor& w,
           const Tensor& mean, const Tensor& rstd,
           const std::optional<at::ScalarType>& wtype, bool dx, bool dw,
           bool db) {
          auto [a, b, c] = norm_bwd(dy, x, w, mean, rstd, wtype, dx, dw, db);
          return std::make_tuple(maybe(a), maybe(b), maybe(c));
        },
        free_gil());
  m.def("gated_scan", &gated_scan, free_gil());
  m.def("gated_scan_fwd", [](const Tensor& gate, const Tensor& x,
                             const MaybeTensor& h0, const MaybeTensor& done,
                             bool keep) {
    auto [hs, last, states] = scan_fwd(gate, x, h0, done, keep);
    return std::make_tuple(hs, last, maybe(states));
  }, free_gil());
  m.def("gated_scan_bwd",
        [](const MaybeTensor& dhs, const MaybeTensor& dl, const Tensor& gate,
           const Tensor& x, const Tensor& states, const MaybeTensor& done,
           bool need_dh0) {
          auto [a, b, c] = scan_bwd(dhs, dl, gate, x, states, done, need_dh0);
          return std::make_tuple(a, b, maybe(c));
        },
        free_gil());
  m.def("gated_scan_step", &scan_step, free_gil());
  m.def("action_logprobs", &action_logprobs, free_gil());
  m.def("action_logprobs_fwd",
        [](const Tensor& logits, const Tensor& actions,
           const MaybeTensor& mask, int64_t top_k) {
          auto [a, b, c, d, e] = logp_fwd(logits, actions, mask, top_k, true);
          return std::make_tuple(a, b, c, maybe(d), maybe(e));
        },
        free_gil());
  m.def("action_logprobs_bwd", &logp_bwd, free_gil());
}
