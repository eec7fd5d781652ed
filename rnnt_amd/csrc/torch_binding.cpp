// The operators' path from torch to the C ABI: checks, outputs, workspaces, autograd nodes.  A decoder's step or a small layer
// is a few microseconds of GPU work; in Python its arguments alone cost more, and a backward pass in Python runs on
// autograd's thread with cold caches and the interpreter's lock.  Through ctypes and through this file: dense 8 x 250 x 62 10.8
// and 6.3 us a call, a beam step of one utterance 24 and 11.5, dropout of 1200 x 250 with its gradient 76 and 42, a training step of
// 6151 x 515 x 1030 in float16 139 and 87.  The entry points are those of the library that rnnt_amd._lib has loaded; their addresses come from there.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <unordered_set>

#include "../../include/rnnt_mi355x.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

#ifdef RNNT_BUILD_STAMP
__attribute__((used)) const char kBuildStamp[] = RNNT_BUILD_STAMP;  // the torch and Python this is for: build.py looks for it
#endif

struct Entries {
  decltype(&rnnt_mi355x_dropout) dropout;
  decltype(&rnnt_mi355x_layer_workspace_bytes) layer_workspace_bytes;
  decltype(&rnnt_mi355x_layer_forward) layer_forward;
  decltype(&rnnt_mi355x_layer_backward) layer_backward;
  decltype(&rnnt_mi355x_beam_select_workspace_bytes) beam_select_workspace_bytes;
  decltype(&rnnt_mi355x_beam_select) beam_select;
  decltype(&rnnt_mi355x_beam_reorder) beam_reorder;
  decltype(&rnnt_mi355x_status_string) status_string;
} C;

template <class F>
void bind_one(F& f, const py::dict& d, const char* name) {
  f = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}
void bind(const py::dict& d) {
  bind_one(C.dropout, d, "rnnt_mi355x_dropout");
  bind_one(C.layer_workspace_bytes, d, "rnnt_mi355x_layer_workspace_bytes");
  bind_one(C.layer_forward, d, "rnnt_mi355x_layer_forward");
  bind_one(C.layer_backward, d, "rnnt_mi355x_layer_backward");
  bind_one(C.beam_select_workspace_bytes, d, "rnnt_mi355x_beam_select_workspace_bytes");
  bind_one(C.beam_select, d, "rnnt_mi355x_beam_select");
  bind_one(C.beam_reorder, d, "rnnt_mi355x_beam_reorder");
  bind_one(C.status_string, d, "rnnt_mi355x_status_string");
}

[[noreturn]] void bad_value(const std::string& what) { throw py::value_error(what); }
[[noreturn]] void bad_type(const std::string& what) { throw py::type_error(what); }
void check(int rc, const char* what) {
  TORCH_CHECK(rc == RNNT_MI355X_OK, what, ": ", C.status_string(rc), " (status ", rc, ")");
}

std::string shape(const Tensor& t) { return c10::str(t.sizes()); }

void on_gpu(const char* op, const char* name, const Tensor& t) {
  if (t.device().type() != c10::kCUDA) bad_value(std::string(op) + ": " + name + " must live on an MI355X device (there is no CPU path)");
}
void same_device(const char* op, const char* name, const Tensor& t, const Tensor& first) {
  if (!t.defined() || t.device() == first.device()) return;
  on_gpu(op, name, t);
  bad_value(std::string(op) + ": " + name + " lives on " + t.device().str() + ", the others on " + first.device().str());
}
int code_of(const char* op, const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return RNNT_MI355X_FP32;
    case at::kBFloat16: return RNNT_MI355X_BF16;
    case at::kHalf: return RNNT_MI355X_FP16;
    default: bad_type(std::string(op) + ": float32, bfloat16 or float16 expected, got " + c10::toString(t.scalar_type()));
  }
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// Results are filled through raw pointers, past everything of torch that follows a computation; what would come out wrong without
// a word is refused.  A dual tensor of forward-mode differentiation would lose its tangent.
// What memory holds is what is read: a view that negates on access becomes a tensor that holds its values.
Tensor values(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// A trace would hold the allocation of the results and nothing of what is written to them.
void refuse_tracing(const char* op) {
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY), op,
              ": calls cannot be traced; trace what is around them");
}
void refuse_tangent(const char* op, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), op, ": forward-mode differentiation is not implemented");
}
void refuse_tangents(const char* op, std::initializer_list<const Tensor*> given) {
  for (const Tensor* t : given) refuse_tangent(op, *t);
}

// Where a backward pass is captured, autograd makes the stream of every node that it comes to wait for the stream captured.  A
// leaf that an eager graph still uses has its node on that graph's stream, and such a wait from outside the capture ends the
// process; it is refused before it happens, wherever behind the operator's node that leaf is.  (What does not lie behind an
// operator's node is not seen from here.)
void refuse_waits_outside_capture(const char* op) {
  const auto here = c10::hip::getCurrentHIPStream();
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  std::vector<torch::autograd::Node*> todo;
  std::unordered_set<torch::autograd::Node*> seen;
  if (const auto node = torch::autograd::get_current_node()) todo.push_back(node.get());
  while (!todo.empty()) {
    torch::autograd::Node* const node = todo.back();
    todo.pop_back();
    for (uint32_t i = 0; i < node->num_outputs(); ++i) {
      const auto& next = node->next_edge(i).function;
      if (!next || !node->task_should_compute_output(i) || !seen.insert(next.get()).second) continue;
      todo.push_back(next.get());
      const auto there = next->stream();
      if (!there || (there->id() == here.id() && there->device_index() == here.device_index())) continue;
      hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
      const hipStream_t other = c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *there).stream();
      const bool captured = other && hipStreamIsCapturing(other, &status) == hipSuccess && status == hipStreamCaptureStatusActive;
      TORCH_CHECK(captured, op, ": this backward pass is being captured, and goes on to a tensor that an eager graph on another stream still holds; "
                            "drop that graph and its results first, or give the captured pass leaves of its own");
    }
  }
}

constexpr int64_t kInt = 0x7fffffff;  // what an int of the C ABI holds

// ---- dropout ------------------------------------------------------------------------------------------------------------
struct Drop {
  int64_t drop16, seed, offset;  // seed and offset: the bits of unsigned values
};

Tensor run_dropout(const Tensor& given, const Drop& d, const Tensor& offset_given) {
  Tensor x = values(given);
  const Tensor offset_t = values(offset_given);
  const int64_t cols = x.size(-1);
  if (cols > kInt) bad_value("dropout: the last dimension holds 2^31 elements or more");
  int64_t stride = cols;
  if (!x.is_contiguous()) {
    // rows of a matrix may be any distance apart; anything else is made dense
    if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= cols) stride = x.stride(0);
    else x = x.contiguous();
  }
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  check(C.dropout(x.data_ptr(), stride, y.data_ptr(), x.numel() / cols, (int)cols, code_of("dropout", x), (int)d.drop16, (uint64_t)d.seed,
                  (uint64_t)d.offset, static_cast<const uint64_t*>(ptr(offset_t)), stream_of(x)),
        "rnnt_mi355x_dropout");
  return y;
}

struct DropoutNode : torch::autograd::Function<DropoutNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& offset_t_, int64_t drop16, int64_t seed, int64_t offset) {
    const Tensor offset_t = or_none(offset_t_);
    ctx->saved_data["drop16"] = drop16;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    if (offset_t.defined()) ctx->save_for_backward({offset_t});  // its version is checked: the backward pass needs the same offset
    return run_dropout(x, Drop{drop16, seed, offset}, offset_t);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
    refuse_waits_outside_capture("dropout");
    const auto saved = ctx->get_saved_variables();
    const OptTensor offset_t = saved.empty() ? OptTensor() : OptTensor(saved[0]);
    const Drop d{ctx->saved_data["drop16"].toInt(), ctx->saved_data["seed"].toInt(), ctx->saved_data["offset"].toInt()};
    // with a graph of the gradient wanted, the same linear map again
    Tensor dx = at::GradMode::is_enabled() ? apply(dy[0], offset_t, d.drop16, d.seed, d.offset) : run_dropout(dy[0], d, or_none(offset_t));
    return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor dropout(const Tensor& x, int64_t drop16, uint64_t seed, uint64_t offset, const OptTensor& offset_t) {
  refuse_tracing("dropout");
  refuse_tangent("dropout", x);
  on_gpu("dropout", "x", x);
  code_of("dropout", x);
  if (drop16 == 0 || x.numel() == 0) return x;
  if (at::GradMode::is_enabled() && x.requires_grad()) return DropoutNode::apply(x, offset_t, drop16, (int64_t)seed, (int64_t)offset);
  return run_dropout(x, Drop{drop16, (int64_t)seed, (int64_t)offset}, or_none(offset_t));
}

// ---- Dense layer --------------------------------------------------------------------------------------------------------
// t as [rows, last dimension] whose last dimension is contiguous, and the distance of its rows
Tensor as_rows(const Tensor& given, long long* stride) {
  Tensor t = values(given);
  const int64_t n = t.size(-1);
  if (t.is_contiguous()) {
    *stride = n;
    return t.dim() == 2 ? t : t.view({-1, n});
  }
  if (t.dim() != 2) t = t.reshape({-1, n});
  if ((n > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < n)) t = t.contiguous();
  *stride = t.size(0) > 1 ? std::max<int64_t>(t.stride(0), n) : n;
  return t;
}

struct LayerArgs {
  int64_t act;
  Drop d;
};

// the tensors whose addresses are in `layer` have to outlive it
rnnt_mi355x_layer layer_of(const Tensor& x, long long x_stride, const Tensor& kernel, long long kernel_stride, const LayerArgs& a, const Tensor& offset_t) {
  rnnt_mi355x_layer l{};
  l.x = x.data_ptr();
  l.kernel = kernel.data_ptr();
  l.x_stride = x_stride;
  l.kernel_stride = kernel_stride;
  l.rows = x.size(0);
  l.in = (int)kernel.size(0);
  l.out = (int)kernel.size(1);
  l.dtype = code_of("dense", x);
  l.act = (int)a.act;
  l.drop16 = (int)a.d.drop16;
  l.seed = (uint64_t)a.d.seed;
  l.offset = (uint64_t)a.d.offset;
  l.offset_dev = static_cast<const uint64_t*>(ptr(offset_t));
  return l;
}

// y, and the pre-activation where it is asked for
std::pair<Tensor, Tensor> run_layer(const Tensor& x_given, const Tensor& kernel_given, const Tensor& bias_given, const Tensor& residual_given,
                                    const Tensor& offset_given, const LayerArgs& a, bool want_aux) {
  const c10::DeviceGuard guard(x_given.device());
  at::DimVector size(x_given.sizes().begin(), x_given.sizes().end());
  size.back() = kernel_given.size(1);
  Tensor y = at::empty(size, x_given.options()), aux;
  if (want_aux) aux = at::empty(size, x_given.options().dtype(x_given.scalar_type() == at::kBFloat16 ? at::kHalf : at::kFloat));
  if (y.numel() == 0) return {y, aux};
  long long x_stride, kernel_stride;
  const Tensor x = as_rows(x_given, &x_stride), kernel = as_rows(kernel_given, &kernel_stride), offset_t = values(offset_given);
  rnnt_mi355x_layer l = layer_of(x, x_stride, kernel, kernel_stride, a, offset_t);
  Tensor bias, residual;
  if (bias_given.defined()) {
    bias = values(bias_given).contiguous();
    l.bias = bias.data_ptr();
  }
  if (residual_given.defined()) {
    residual = as_rows(residual_given, &l.residual_stride);
    l.residual = residual.data_ptr();
  }
  l.y = y.data_ptr();
  l.aux = ptr(aux);
  size_t bytes = 0;
  check(C.layer_workspace_bytes(&l, nullptr, 0, &bytes, nullptr), "rnnt_mi355x_layer_workspace_bytes");
  const Tensor ws = workspace(bytes, x);
  check(C.layer_forward(&l, ptr(ws), stream_of(x)), "rnnt_mi355x_layer_forward");
  return {y, aux};
}

struct LayerNode : torch::autograd::Function<LayerNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& kernel, const OptTensor& bias_, const OptTensor& residual_,
                        const OptTensor& offset_t_, int64_t act, int64_t drop16, int64_t seed, int64_t offset, bool wants) {
    const Tensor bias = or_none(bias_), residual = or_none(residual_), offset_t = or_none(offset_t_);
    const LayerArgs a{act, {drop16, seed, offset}};
    // what act' is computed from: the pre-activation, or the output where that is as good
    const bool from_y = !residual.defined() && (act == RNNT_MI355X_ACT_RELU || (act == RNNT_MI355X_ACT_TANH && x.scalar_type() == at::kFloat));
    const bool linear = act == RNNT_MI355X_ACT_LINEAR;
    auto [y, aux] = run_layer(x, kernel, bias, residual, offset_t, a, wants && !linear && !from_y);
    ctx->saved_data["act"] = act;
    ctx->saved_data["drop16"] = drop16;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["bias"] = bias.defined();
    ctx->saved_data["residual"] = residual.defined();
    ctx->save_for_backward({x, kernel, wants && !linear && from_y ? y : Tensor(), aux, offset_t});
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dys) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "dense: the gradient is not differentiable (create_graph)");
    refuse_waits_outside_capture("dense");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x_given = saved[0], &kernel_given = saved[1], &y = saved[2], &aux = saved[3], offset_t = values(saved[4]);
    // edges are counted over the tensors that were there
    const bool has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["residual"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_k = ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(2),
               need_r = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    torch::autograd::variable_list grads(10);
    if (need_r) grads[3] = dys[0];
    if (!(need_x || need_k || need_b)) return grads;
    const c10::DeviceGuard guard(x_given.device());
    Tensor dx, dk, db;
    if (need_x) grads[0] = dx = at::empty(x_given.sizes(), x_given.options());
    if (need_k) grads[1] = dk = at::empty(kernel_given.sizes(), x_given.options());
    if (need_b) grads[2] = db = at::empty({kernel_given.size(1)}, x_given.options());
    if (dys[0].numel() == 0) {
      for (auto& g : {dx, dk, db})
        if (g.defined()) g.zero_();
      return grads;
    }
    long long x_stride, kernel_stride, dy_stride;
    const Tensor x = as_rows(x_given, &x_stride), kernel = as_rows(kernel_given, &kernel_stride), dy = as_rows(dys[0], &dy_stride);
    const LayerArgs a{ctx->saved_data["act"].toInt(), {ctx->saved_data["drop16"].toInt(), ctx->saved_data["seed"].toInt(), ctx->saved_data["offset"].toInt()}};
    rnnt_mi355x_layer l = layer_of(x, x_stride, kernel, kernel_stride, a, offset_t);
    l.y = ptr(y);
    l.aux = ptr(aux);
    size_t bytes = 0;
    check(C.layer_workspace_bytes(&l, dy.data_ptr(), dy_stride, nullptr, &bytes), "rnnt_mi355x_layer_workspace_bytes");
    const Tensor ws = workspace(bytes, x);
    check(C.layer_backward(&l, dy.data_ptr(), dy_stride, ptr(dx), ptr(dk), ptr(db), ptr(ws), stream_of(x)), "rnnt_mi355x_layer_backward");
    return grads;
  }
};

Tensor dense(const Tensor& x, const Tensor& kernel, const OptTensor& bias_, const OptTensor& residual_, int64_t act, int64_t drop16, uint64_t seed,
             uint64_t offset, const OptTensor& offset_t) {
  const Tensor bias = or_none(bias_), residual = or_none(residual_);
  refuse_tracing("dense");
  refuse_tangents("dense", {&x, &kernel, &bias, &residual});
  on_gpu("dense", "x", x);
  same_device("dense", "kernel", kernel, x);
  same_device("dense", "bias", bias, x);
  same_device("dense", "residual", residual, x);
  code_of("dense", x);
  if (kernel.dim() != 2 || x.dim() < 1 || x.size(-1) != kernel.size(0) || kernel.numel() == 0)
    bad_value("dense: x" + shape(x) + " does not fit kernel" + shape(kernel));
  if (std::max(kernel.size(0), kernel.size(1)) > (1 << 24)) bad_value("dense: a layer is at most 2^24 wide, got kernel" + shape(kernel));
  if (bias.defined() && (bias.dim() != 1 || bias.size(0) != kernel.size(1))) bad_value("dense: bias" + shape(bias) + " does not fit kernel" + shape(kernel));
  if (residual.defined()) {
    at::DimVector want(x.sizes().begin(), x.sizes().end());
    want.back() = kernel.size(1);
    if (residual.sizes() != at::IntArrayRef(want)) bad_value("dense: residual" + shape(residual) + " is not of the result's shape");
  }
  for (const auto& [name, t] : {std::pair<const char*, const Tensor*>{"kernel", &kernel}, {"bias", &bias}, {"residual", &residual}})
    if (t->defined() && t->scalar_type() != x.scalar_type())
      bad_type(std::string("dense: ") + name + " is " + c10::toString(t->scalar_type()) + ", x is " + c10::toString(x.scalar_type()));
  if (at::GradMode::is_enabled()) {
    const bool wants = x.requires_grad() || kernel.requires_grad() || (bias.defined() && bias.requires_grad());
    if (wants || (residual.defined() && residual.requires_grad()))
      return LayerNode::apply(x, kernel, bias_, residual_, offset_t, act, drop16, (int64_t)seed, (int64_t)offset, wants);
  }
  return run_layer(x, kernel, bias, residual, or_none(offset_t), LayerArgs{act, {drop16, (int64_t)seed, (int64_t)offset}}, false).first;
}

// ---- beam step ----------------------------------------------------------------------------------------------------------
constexpr int64_t kMaxBeams = 64, kMaxWidth = 64;

std::tuple<Tensor, Tensor, Tensor> beam_select(const Tensor& logits_given, const Tensor& scores_given, int64_t width, const OptTensor& enc_,
                                               const OptTensor& allowed_, const OptTensor& finished_, int64_t end) {
  const char* op = "beam_select";
  Tensor logits = values(logits_given), scores = values(scores_given), enc = values(or_none(enc_)), allowed = or_none(allowed_), finished = or_none(finished_);
  refuse_tracing(op);
  refuse_tangents(op, {&logits, &scores, &enc});
  on_gpu(op, "logits", logits);
  same_device(op, "scores", scores, logits);
  same_device(op, "enc", enc, logits);
  same_device(op, "allowed", allowed, logits);
  same_device(op, "finished", finished, logits);
  const int code = code_of(op, logits);
  if (logits.dim() != 3 || logits.numel() == 0) bad_value("beam_select: expected logits[B,K,V], got " + shape(logits));
  const int64_t B = logits.size(0), K = logits.size(1), V = logits.size(2);
  if (width < 1 || width > kMaxWidth || K > kMaxBeams)
    bad_value("beam_select: 1 to " + std::to_string(kMaxWidth) + " continuations of at most " + std::to_string(kMaxBeams) + " beams, got " +
              std::to_string(width) + " of " + std::to_string(K));
  if (V > 0x7fff0000 / K || B > kInt) bad_value("beam_select: beams x vocabulary must not pass 2^31 - 2^16, got " + shape(logits));
  if (scores.dim() != 2 || scores.size(0) != B || scores.size(1) != K || scores.scalar_type() != at::kFloat)
    bad_value("beam_select: scores must be float32 [B, K]");
  if (enc.defined()) {
    if (enc.dim() != 2 || enc.size(0) != B || enc.size(1) != V || enc.scalar_type() != logits.scalar_type())
      bad_value("beam_select: enc must be [B, V] of the logits' type");
    if (V > 1 && enc.stride(1) != 1) enc = enc.contiguous();
  }
  if (allowed.defined()) {
    if (allowed.scalar_type() != at::kBool || allowed.dim() < 1 || allowed.dim() > 2 || allowed.size(-1) != V || (allowed.dim() == 2 && allowed.size(0) != B))
      bad_value("beam_select: allowed must be bool [V] or [B, V]");
    if (V > 1 && allowed.stride(-1) != 1) allowed = allowed.contiguous();
  }
  if (finished.defined()) {
    if (finished.scalar_type() != at::kBool || finished.dim() != 2 || finished.size(0) != B || finished.size(1) != K)
      bad_value("beam_select: finished must be bool [B, K]");
    if (end < 0 || end >= V) bad_value("beam_select: end " + std::to_string(end) + " outside [0, " + std::to_string(V) + ")");
    finished = finished.contiguous();
  }
  if (V > 1 && logits.stride(2) != 1) logits = logits.contiguous();
  scores = scores.contiguous();
  const c10::DeviceGuard guard(logits.device());
  const auto int32 = logits.options().dtype(at::kInt);
  Tensor out_scores = at::empty({B, width}, logits.options().dtype(at::kFloat)), parent = at::empty({B, width}, int32), token = at::empty({B, width}, int32);
  size_t bytes = 0;
  check(C.beam_select_workspace_bytes((int)B, (int)K, (int)V, (int)width, &bytes), "rnnt_mi355x_beam_select_workspace_bytes");
  const Tensor ws = workspace(bytes, logits);
  check(C.beam_select(logits.data_ptr(), logits.stride(0), logits.stride(1), code, ptr(enc), enc.defined() ? enc.stride(0) : 0, scores.data_ptr<float>(),
                      static_cast<const uint8_t*>(ptr(allowed)), allowed.defined() && allowed.dim() == 2 ? allowed.stride(0) : 0,
                      static_cast<const uint8_t*>(ptr(finished)), finished.defined() ? (int)end : 0, (int)B, (int)K, (int)V, (int)width,
                      out_scores.data_ptr<float>(), parent.data_ptr<int32_t>(), token.data_ptr<int32_t>(), ptr(ws), stream_of(logits)),
        "rnnt_mi355x_beam_select");
  return {out_scores, parent, token};
}

// [first, one past the last) byte a tensor covers
std::pair<uintptr_t, uintptr_t> bytes_of(const Tensor& t) {
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {p, p + (uintptr_t)((last + 1) * t.element_size())};
}

// A state as [outer, B, K, row], its row dense: outer, and the strides of the three leading dimensions in elements.  A dense
// tensor's come from its sizes: where a dimension has size 1 its own stride may be anything.
std::tuple<int64_t, int64_t, int64_t, int64_t> leading(const Tensor& s, int64_t d) {
  int64_t outer = 1, row = 1;
  for (int64_t j = 0; j < d; ++j) outer *= s.size(j);
  if (!s.is_contiguous()) return {outer, d ? s.stride(d - 1) : 0, s.stride(d), s.stride(d + 1)};
  for (int64_t j = d + 2; j < s.dim(); ++j) row *= s.size(j);
  return {outer, s.size(d) * s.size(d + 1) * row, s.size(d + 1) * row, row};
}

std::vector<Tensor> beam_reorder(const Tensor& parent_given, const std::vector<Tensor>& states, int64_t d, const std::optional<std::vector<Tensor>>& out_given) {
  const char* op = "beam_reorder";
  refuse_tracing(op);
  for (const Tensor& s : states) refuse_tangent(op, s);
  if (out_given)
    for (const Tensor& o : *out_given) refuse_tangent(op, o);
  if (parent_given.scalar_type() != at::kInt || parent_given.dim() != 2) bad_value("beam_reorder: parent must be int32 [B, W]");
  on_gpu(op, "parent", parent_given);
  if (d < 0) bad_value("beam_reorder: batch_dim counts from the first dimension");
  const int64_t B = parent_given.size(0), W = parent_given.size(1);
  int64_t K = -1;
  std::vector<Tensor> out;
  const c10::DeviceGuard guard(parent_given.device());
  for (size_t i = 0; i < states.size(); ++i) {
    const Tensor& s = states[i];
    const std::string name = "states[" + std::to_string(i) + "]";
    if (s.device() != parent_given.device()) same_device(op, name.c_str(), s, parent_given);
    if (s.dim() < d + 2 || s.size(d) != B)
      bad_value("beam_reorder: " + name + " has shape " + shape(s) + ", expected B=" + std::to_string(B) + " at dimension " + std::to_string(d) + " and the beams next");
    if (K < 0) K = s.size(d + 1);
    else if (s.size(d + 1) != K) bad_value("beam_reorder: the states differ in their number of beams");
    at::DimVector size(s.sizes().begin(), s.sizes().end());
    size[d + 1] = W;
    if (!out_given) {
      out.push_back(at::empty(size, s.options()));
    } else {
      if (out_given->size() != states.size()) bad_value("beam_reorder: out must be as many tensors as states");
      const Tensor& o = (*out_given)[i];
      same_device(op, ("out[" + std::to_string(i) + "]").c_str(), o, parent_given);
      if (o.sizes() != at::IntArrayRef(size) || o.scalar_type() != s.scalar_type() || !o.is_contiguous() || o.is_conj() || o.is_neg())
        bad_value("beam_reorder: out must be dense tensors of the results' shapes and types");
      out.push_back(o);
    }
  }
  if (out_given) {
    if (out_given->size() != states.size()) bad_value("beam_reorder: out must be as many tensors as states");
    std::vector<Tensor> all(out);
    all.insert(all.end(), states.begin(), states.end());
    all.push_back(parent_given);
    for (size_t i = 0; i < out.size(); ++i)
      for (size_t j = 0; j < all.size(); ++j) {
        if (i == j || !out[i].numel() || !all[j].numel()) continue;
        const auto a = bytes_of(out[i]), b = bytes_of(all[j]);
        if (a.first < b.second && b.first < a.second) bad_value("beam_reorder: out overlaps a state, another output or parent");
      }
    for (const Tensor& o : out)
      if (at::GradMode::is_enabled() && o.requires_grad()) bad_value("beam_reorder: out must not require gradients");
    // written in place: autograd has to see it where a graph keeps one of them
    for (const Tensor& o : out) torch::autograd::impl::bump_version(o);
  }
  if (states.empty()) return out;
  if (std::max(std::max(B, K), W) > kInt) bad_value("beam_reorder: more than 2^31 - 1 utterances or beams");
  if (K == 0) {
    for (Tensor& o : out) o.zero_();
    return out;
  }
  const Tensor parent = values(parent_given).contiguous();
  std::vector<rnnt_mi355x_reorder_tensor> table;
  std::vector<Tensor> keep;
  for (size_t i = 0; i < states.size(); ++i) {
    Tensor s = states[i];
    const Tensor& o = out[i];
    if (o.numel() == 0) continue;
    if (s.is_conj() || s.is_neg()) keep.push_back(s = s.resolve_conj().resolve_neg());  // what memory holds is not the value
    if (!s.is_contiguous()) {
      // [outer, B, K, row]: the row has to be dense, the three leading dimensions need one stride each
      bool dense_row = d <= 1;
      int64_t expect = 1;
      for (int64_t j = s.dim() - 1; j > d + 1; --j) {
        dense_row &= s.size(j) == 1 || s.stride(j) == expect;
        expect *= s.size(j);
      }
      if (!dense_row) s = s.contiguous();
      keep.push_back(s);
    }
    const auto [outer, outer_stride, batch_stride, beam_stride] = leading(s, d);
    const int64_t e = s.element_size();
    table.push_back({s.data_ptr(), o.data_ptr(), outer, outer_stride * e, batch_stride * e, beam_stride * e, o.numel() / (outer * B * W) * e});
  }
  for (size_t i = 0; i < table.size(); i += RNNT_MI355X_REORDER_MAX)
    check(C.beam_reorder(table.data() + i, (int)std::min<size_t>(RNNT_MI355X_REORDER_MAX, table.size() - i), parent.data_ptr<int32_t>(), (int)B, (int)K, (int)W,
                         stream_of(parent)),
          "rnnt_mi355x_beam_reorder");
  return out;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("bind", &bind);
  m.def("dropout", &dropout);
  m.def("dense", &dense);
  m.def("beam_select", &beam_select);
  m.def("beam_reorder", &beam_reorder);
  m.def("reorder_strides", &leading);  // of beam_reorder, for tests without a GPU
}
