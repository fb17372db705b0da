// cp_torch.cpp — the policy operators (include/contracts_policy.h) for torch tensors: allocates outputs and scratch memory, describes the tensors
// to the C-ABI, and takes gradients through nodes that need no interpreter.
//
// Host-side marshalling and the checks of arguments, because a call's latency is the host's: a forward call took 11-14 us through Python and
// ctypes, of which the launch is 3, and a forward and backward pass 120 us, most of it the interpreter in torch's backward thread.  What
// reaches the device is checked by the C-ABI once more.  policy_ops.py documents the calls.
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <ATen/TensorUtils.h>

#include <sstream>

#include "../../include/contracts_policy.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void check(int rc, const char* what) {
  if (rc == CE_OK) return;
  const char* name = rc == CE_EINVAL ? "CE_EINVAL" : rc == CE_ENODEV ? "CE_ENODEV" : "?";
  throw Refused(std::string(what) + " failed: " + name + " (" + std::to_string(rc) + ") " + ce_policy_error());
}

// ---- refusals: ValueError, as the engine's Python layer raises -------------------------------------------------------------------
template <class... A> [[noreturn]] void bad(const A&... parts) {
  std::ostringstream text;
  (text << ... << parts);
  throw py::value_error(text.str());
}
double number(const py::object& o) {
  const double v = PyFloat_AsDouble(o.ptr());
  if (v == -1 && PyErr_Occurred()) throw py::error_already_set();
  return v;
}
bool real(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
bool flag(at::ScalarType t) { return t == at::kBool || t == at::kByte; }
// Recorded as a graph, a call would leave nothing behind but the allocation of its outputs.
bool traced() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  return torch::jit::tracer::isTracing() || Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE);
}
// Tensors that stand for others: batched, traced or differentiated by a transform, of a subclass that dispatches, zeros that are nowhere.
bool wrapped(const Tensor& t) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet keys({DispatchKey::Python, DispatchKey::Batched, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper, DispatchKey::Functionalize, DispatchKey::ZeroTensor});
  return t.key_set().has_any(keys);
}
void memory(const char* op, const Tensor& t) {
  if (wrapped(t)) bad(op, ": a wrapped tensor (batched, traced, of a subclass) has no memory to read");
}
void on_gpu(const char* op, const Tensor& t) {
  if (traced()) bad(op, ": cannot be traced or recorded as a graph of operations");
  memory(op, t);
  if (!t.is_cuda()) bad(op, ": tensors must live on a GPU (there is no CPU path), got ", t.device());
}
// An incoming gradient as numbers that lie in memory; one that carries a forward-mode derivative, or is a batch in one, is refused.
Tensor incoming(const char* op, const Tensor& t) {
  if (traced()) throw Refused(std::string(op) + ": the backward pass cannot be traced or recorded as a graph of operations");
  if (!t.defined()) return t;
  if (wrapped(t)) throw Refused(std::string(op) + ": a gradient that is a wrapped tensor (batched, traced, of a subclass) has no memory to read");
  if (t._fw_grad(0).defined()) throw Refused(std::string(op) + ": has no forward-mode derivative");
  return t.resolve_neg();
}
// All on one device, and numbers as they lie in memory: not a lazily negated view, not carrying a forward-mode derivative, which a call would drop.
void same_device(const char* op, const Tensor& first, std::initializer_list<const Maybe*> rest) {
  auto plain = [&](const Tensor& t) {
    memory(op, t);
    if (t.is_neg()) bad(op, ": a lazily negated view; call resolve_neg() on it");
    if (t._fw_grad(0).defined()) bad(op, ": has no forward-mode derivative");
  };
  plain(first);
  for (const Maybe* t : rest)
    if (*t) {
      if ((*t)->device() != first.device()) bad(op, ": all tensors must live on one device");
      plain(**t);
    }
}
// The bytes a tensor reaches.
std::pair<const char*, const char*> span(const Tensor& t) {
  int64_t n = 1;
  for (int64_t d = 0; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
  const char* lo = (const char*)t.data_ptr();
  return {lo, lo + n * t.element_size()};
}
// An output may not overlap an input.
void apart(const char* op, const Maybe& out, const char* name, std::initializer_list<const Maybe*> inputs) {
  if (!out || out->numel() == 0) return;
  const auto o = span(*out);
  for (const Maybe* t : inputs)
    if (*t && (*t)->defined() && (*t)->numel()) {
      const auto i = span(**t);
      if (o.second > i.first && i.second > o.first) bad(op, ": ", name, " overlaps an input");
    }
}
// An output that is part of a graph would keep the gradients of what it held before (torch's own out= refuses it too).
void no_graph(const char* op, std::initializer_list<const Maybe*> outs) {
  if (!at::GradMode::is_enabled()) return;
  for (const Maybe* t : outs)
    if (*t && (*t)->requires_grad()) bad(op, ": an output wants a gradient, which this call would not keep; detach it");
}

uint32_t code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CE_F32;
    case at::kBFloat16: return CE_BF16;
    case at::kHalf: return CE_F16;
    case at::kDouble: return CE_F64;
    case at::kByte:
    case at::kBool: return CE_U8;
    case at::kInt: return CE_I32;
    default: return CE_I64;
  }
}
template <class T = void> T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
template <class T = void> T* ptr(const Maybe& t) { return t ? ptr<T>(*t) : nullptr; }
Tensor bytes(uint64_t n, const Tensor& like) { return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor(); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// A tensor of the caller's that a call wrote to: a graph that had saved it finds out, as after torch's own in-place operations.
void written(const Maybe& t) {
  if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// Gradients of these gradients do not exist: whoever asks for one is told so (and nobody else).
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& t : grads)
    if (t.defined()) t = t.detach().requires_grad_(true);
  return (*std::make_shared<torch::autograd::DelayedError>("the gradients of the policy operators have no gradients of their own", (int64_t)grads.size()))(std::move(grads));
}

// ---- linear_scan ----------------------------------------------------------------------------------------------------------------
ce_scan describe(const Tensor& x, const Tensor& gate, double decay, const Tensor& done, bool reverse) {
  ce_scan s = {};
  s.abi_version = CE_POLICY_ABI_VERSION;
  s.device = x.get_device();
  s.dtype = s.gate_dtype = code(x);
  s.flags = reverse ? CE_SCAN_REVERSE : 0;
  s.steps = x.size(0);
  s.rows = x.size(1);
  s.channels = s.heads = x.size(2);
  s.x_step = x.stride(0);
  s.x_row = x.stride(1);
  s.x = ptr(x);
  if (gate.defined()) {
    s.gate_dtype = code(gate);
    s.heads = gate.size(2);
    s.gate_step = gate.stride(0);
    s.gate_row = gate.stride(1);
    s.gate = ptr(gate);
  }
  s.decay = decay;
  if (done.defined()) {
    s.done_step = done.stride(0);
    s.done_row = done.stride(1);
    s.done = ptr<uint8_t>(done);
  }
  return s;
}

void scan_forward(const Tensor& x, const Tensor& gate, double decay, const Tensor& state, const Tensor& done, bool reverse, Tensor& y, Tensor& last, Tensor* saved) {
  const int64_t T = x.size(0), E = x.size(1), C = x.size(2);
  if (!y.defined()) y = at::empty({T, E, C}, x.options());
  if (!last.defined()) last = at::empty({E, C}, x.scalar_type() == at::kDouble ? x.options() : x.options().dtype(at::kFloat));
  ce_scan s = describe(x, gate, decay, done, reverse);
  s.state = ptr(state);
  s.y = ptr(y);
  s.last = ptr(last);
  if (saved) {
    *saved = at::empty({(T + CE_SCAN_SAVED_STEPS - 1) / CE_SCAN_SAVED_STEPS, E, C}, x.options().dtype(at::kFloat));
    s.saved = ptr<float>(*saved);
  }
  Tensor ws, before;
  if (T >= CE_SCAN_SPLIT_STEPS) {
    const bool in_place = s.state && s.state == s.last;
    if (in_place) s.state = nullptr;
    check(ce_linear_scan_workspace(&s, &s.workspace_bytes), "linear_scan");
    if (in_place) {  // a time axis that is to be split reads a copy: moved on in place it would stay whole ([65537, 1, 1024], 16 heads: 1426 us for 77)
      if (s.workspace_bytes) before = state.clone();
      s.state = ptr(s.workspace_bytes ? before : state);
    }
    ws = bytes(s.workspace_bytes, x);
    s.workspace = ptr(ws);
  }
  check(ce_linear_scan(&s, stream_of(x)), "linear_scan");
}

struct Scan : torch::autograd::Function<Scan> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Maybe gate, double decay, Maybe state, Maybe done, bool reverse) {
    ctx->set_materialize_grads(false);
    Tensor y, last, saved, a = gate.value_or(Tensor());
    scan_forward(x, a, decay, state.value_or(Tensor()), done.value_or(Tensor()), reverse, y, last, &saved);
    ctx->saved_data["decay"] = decay;
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["need"] = (int64_t)(x.requires_grad() | (a.defined() && a.requires_grad()) << 1 | (state && state->requires_grad()) << 2);
    ctx->save_for_backward({x, a, done.value_or(Tensor()), saved});
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto kept = ctx->get_saved_variables();
    const Tensor &x = kept[0], &gate = kept[1], &done = kept[2];
    const int64_t need = ctx->saved_data["need"].toInt(), T = x.size(0), E = x.size(1), C = x.size(2);
    Tensor dx = at::empty({T, E, C}, x.options()), dgate, dstate;
    if (gate.defined()) dgate = x.numel() ? at::empty(gate.sizes(), gate.options()) : at::zeros(gate.sizes(), gate.options());
    if (need & 4) dstate = at::empty({E, C}, x.options().dtype(at::kFloat));
    Tensor dy = incoming("linear_scan", grads[0]), dlast = incoming("linear_scan", grads[1]);
    dy = dy.defined() ? dy.contiguous() : at::zeros({T, E, C}, x.options());
    if (dlast.defined()) dlast = dlast.contiguous();
    ce_scan s = describe(x, gate, ctx->saved_data["decay"].toDouble(), done, ctx->saved_data["reverse"].toBool());
    s.saved = ptr<float>(kept[3]);
    const ce_scan_grad g = {ptr(dy), ptr(dlast), ptr(dx), ptr(dgate), ptr(dstate)};
    check(ce_linear_scan_backward_workspace(&s, &g, &s.workspace_bytes), "linear_scan_backward");
    const Tensor ws = bytes(s.workspace_bytes, x);
    s.workspace = ptr(ws);
    check(ce_linear_scan_backward(&s, &g, stream_of(x)), "linear_scan_backward");
    return once({need & 1 ? dx : Tensor(), need & 2 ? dgate : Tensor(), Tensor(), dstate, Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor> linear_scan(Tensor x, const py::object& gate_or_decay, Maybe state, const Maybe& done, bool reverse, const Maybe& out, const Maybe& state_out) {
  const char* op = "linear_scan";
  if (x.dim() != 3) bad("linear_scan: x must be [T, E, C]");
  on_gpu(op, x);
  Maybe gate;
  double decay = 0;
  if (THPVariable_Check(gate_or_decay.ptr())) gate = THPVariable_Unpack(gate_or_decay.ptr());
  else decay = number(gate_or_decay);
  same_device(op, x, {&gate, &state, &done, &out, &state_out});
  no_graph(op, {&out, &state_out});
  const auto type = x.scalar_type();
  const bool twice = type == at::kDouble;
  if (!real(type) && !twice) bad("linear_scan: x must be float32, bfloat16, float16 or float64, not ", type);
  const int64_t T = x.size(0), E = x.size(1), C = x.size(2);
  const auto acc = twice ? at::kDouble : at::kFloat;
  bool grad = x.requires_grad();
  int64_t head = 1;
  if (gate) {
    const int64_t H = gate->dim() == 3 ? gate->size(2) : -1;
    if (H < 0 || gate->size(0) != T || gate->size(1) != E || !(H == C || (H && C % H == 0)))
      bad("linear_scan: gate must be [T, E, H] with H dividing C, got ", gate->sizes(), " for x ", x.sizes());
    if (gate->scalar_type() != type && (gate->scalar_type() != at::kFloat || twice)) bad("linear_scan: gate must be of x's type or float32, not ", gate->scalar_type());
    grad |= gate->requires_grad();
    if (H) head = C / H;
  }
  // rows that far apart are more than a wave's 32-bit offsets, unless rows are whole waves
  const int64_t far = C % 256 == 0 && (head & (head - 1)) == 0 ? INT64_MAX : ((int64_t)1 << 28) / (255 / C + 1);
  if (gate && ((gate->stride(2) != 1 && gate->size(2) > 1) || gate->stride(1) >= far)) gate = gate->contiguous();
  if ((x.stride(2) != 1 && C > 1) || x.stride(1) >= far) x = x.contiguous();
  if (state) {
    if (state->dim() != 2 || state->size(0) != E || state->size(1) != C || state->scalar_type() != acc) bad("linear_scan: state must be ", acc, " [", E, ", ", C, "]");
    grad |= state->requires_grad();
  }
  if (done && (done->dim() != 2 || done->size(0) != T || done->size(1) != E || !flag(done->scalar_type()))) bad("linear_scan: done must be bool or uint8 [T, E]");
  grad = grad && at::GradMode::is_enabled();
  if (out || state_out) {
    if (grad) bad("linear_scan: out and state_out cannot be given where gradients are wanted");
    if (out && (out->sizes() != x.sizes() || out->scalar_type() != type || !out->is_contiguous())) bad("linear_scan: out must be a dense ", type, " ", x.sizes());
    if (state_out && (state_out->dim() != 2 || state_out->size(0) != E || state_out->size(1) != C || state_out->scalar_type() != acc || !state_out->is_contiguous()))
      bad("linear_scan: state_out must be a dense ", acc, " [", E, ", ", C, "]");
    const bool moved = state && state->is_contiguous() && state_out && state_out->data_ptr() == state->data_ptr();  // in place
    const Maybe none, mx = x;
    apart(op, out, "out", {&state, &state_out, &mx, &gate, &done});
    apart(op, state_out, "state_out", {moved ? &none : &state, &mx, &gate, &done});
  }
  if (state && !state->is_contiguous()) state = state->contiguous();
  if (grad) {
    if (twice) bad("linear_scan: float64 has no backward pass");
    variable_list r = Scan::apply(x, gate, decay, state, done, reverse);
    return {r[0], r[1]};
  }
  Tensor y = out.value_or(Tensor()), last = state_out.value_or(Tensor());
  scan_forward(x, gate.value_or(Tensor()), decay, state.value_or(Tensor()), done.value_or(Tensor()), reverse, y, last, nullptr);
  written(out);
  written(state_out);
  return {y, last};
}

// ---- advantages -----------------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> advantages(Tensor reward, Tensor value, Maybe last_value, Maybe done, double gamma, double lam, int64_t first, const std::optional<std::pair<Tensor, Tensor>>& out) {
  const char* op = "advantages";
  if (reward.dim() != 3) bad("advantages: reward must be [P, E, n]");
  on_gpu(op, reward);
  Maybe adv_out, ret_out;
  if (out) adv_out = out->first, ret_out = out->second;
  const Maybe mv = value;
  same_device(op, reward, {&mv, &last_value, &done, &adv_out, &ret_out});
  no_graph(op, {&adv_out, &ret_out});
  const int64_t P = reward.size(0), E = reward.size(1), n = reward.size(2);
  if (reward.scalar_type() != at::kDouble && reward.scalar_type() != at::kFloat) bad("advantages: reward must be float64 or float32, not ", reward.scalar_type());
  if (value.sizes() != reward.sizes() || !real(value.scalar_type())) bad("advantages: value must be float32, bfloat16 or float16 ", reward.sizes());
  if (last_value) {
    if (last_value->sizes() != reward.sizes().slice(1) || last_value->scalar_type() != value.scalar_type()) bad("advantages: last_value must be ", value.scalar_type(), " [", E, ", ", n, "]");
    last_value = last_value->contiguous();
  }
  if (done) {
    if (done->sizes() != reward.sizes().slice(0, done->dim() == 3 ? 3 : 2) || !flag(done->scalar_type())) bad("advantages: done must be bool or uint8 [P, E] or [P, E, n]");
    done = done->contiguous();
  }
  if (first < 0 || first >= std::max<int64_t>(P, 1)) bad("advantages: first_plane out of range");
  reward = reward.contiguous();
  value = value.contiguous();
  if (out) {
    for (const Maybe* t : {&adv_out, &ret_out})
      if ((*t)->sizes() != reward.sizes() || (*t)->scalar_type() != at::kFloat || !(*t)->is_contiguous()) bad("advantages: out must be two dense float32 ", reward.sizes());
    const Maybe mr = reward, mw = value;
    apart(op, adv_out, "out", {&mr, &mw, &last_value, &done, &ret_out});
    apart(op, ret_out, "out", {&mr, &mw, &last_value, &done});
  }
  const auto f32 = reward.options().dtype(at::kFloat);
  const Tensor adv = adv_out ? *adv_out : at::empty(reward.sizes(), f32), ret = ret_out ? *ret_out : at::empty(reward.sizes(), f32);
  ce_advantage a = {};
  a.abi_version = CE_POLICY_ABI_VERSION;
  a.device = reward.get_device();
  a.reward_dtype = code(reward);
  a.value_dtype = code(value);
  a.flags = done && done->dim() == 3 ? CE_ADV_DONE_PER_AGENT : 0;
  a.first_plane = (uint32_t)first;
  a.planes = reward.size(0);
  a.rows = reward.size(1);
  a.agents = reward.size(2);
  a.gamma = gamma;
  a.lam = lam;
  a.reward = ptr(reward);
  a.value = ptr(value);
  a.last_value = ptr(last_value);
  a.done = ptr<uint8_t>(done);
  a.advantage = ptr<float>(adv);
  a.ret = ptr<float>(ret);
  check(ce_advantages(&a, stream_of(reward)), "advantages");
  written(adv_out);
  written(ret_out);
  return {adv, ret};
}

// ---- process_logits -------------------------------------------------------------------------------------------------------------
struct Shaping {  // what scores are shaped with: everything of a ce_logits but the scores, the bias and the output
  Tensor tokens, lengths, prompt_lengths, mask, mask_index;
  Tensor penalty[3];  // repetition, presence, frequency; or the scalars
  double scalar[3];
};
ce_logits describe(const Tensor& logits, const Tensor& bias, const Shaping& h, uint32_t out_dtype) {
  ce_logits s = {};
  s.abi_version = CE_POLICY_ABI_VERSION;
  s.device = logits.get_device();
  s.dtype = code(logits);
  s.out_dtype = out_dtype;
  s.rows = logits.size(0);
  s.vocab = logits.size(1);
  s.logits_row = logits.stride(0);
  s.logits = ptr(logits);
  s.repetition_all = 1;
  if (h.tokens.defined() && h.tokens.numel()) {
    s.token_dtype = code(h.tokens);
    s.history = h.tokens.size(1);
    s.token_row = h.tokens.stride(0);
    s.token_step = h.tokens.stride(1);
    s.tokens = ptr(h.tokens);
    s.lengths = ptr<int32_t>(h.lengths);
    s.prompt_lengths = ptr<int32_t>(h.prompt_lengths);
    s.repetition = ptr<float>(h.penalty[0]);
    s.presence = ptr<float>(h.penalty[1]);
    s.frequency = ptr<float>(h.penalty[2]);
    s.repetition_all = h.scalar[0];
    s.presence_all = h.scalar[1];
    s.frequency_all = h.scalar[2];
  }
  if (h.mask.defined()) {
    s.mask_dtype = code(h.mask);
    s.mask_rows = h.mask.size(0);
    s.mask = ptr(h.mask);
    s.mask_index = ptr<int32_t>(h.mask_index);
  }
  if (bias.defined()) {
    s.bias_dtype = code(bias);
    s.bias_rows = bias.size(0);
    s.bias = ptr(bias);
  }
  return s;
}
void logits_forward(const Tensor& logits, const Tensor& bias, const Shaping& h, const Tensor& out) {
  ce_logits s = describe(logits, bias, h, code(out));
  s.out = ptr(out);
  s.out_row = out.stride(0);
  check(ce_process_logits(&s, stream_of(logits)), "process_logits");
}

struct Logits : torch::autograd::Function<Logits> {
  static Tensor forward(AutogradContext* ctx, Tensor logits, Maybe bias, const Shaping& h) {
    ctx->set_materialize_grads(false);
    const Tensor b = bias.value_or(Tensor()), out = at::empty(logits.sizes(), logits.options());
    logits_forward(logits, b, h, out);
    ctx->saved_data["need"] = (int64_t)(logits.requires_grad() | (b.defined() && b.requires_grad()) << 1);
    ctx->saved_data["scalars"] = std::vector<double>(h.scalar, h.scalar + 3);
    ctx->save_for_backward({logits, b, h.tokens, h.lengths, h.prompt_lengths, h.mask, h.mask_index, h.penalty[0], h.penalty[1], h.penalty[2]});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dz = incoming("process_logits", grads[0]);
    if (!dz.defined()) return {Tensor(), Tensor(), Tensor()};
    const auto kept = ctx->get_saved_variables();
    const Tensor &logits = kept[0], &bias = kept[1];
    Shaping h = {kept[2], kept[3], kept[4], kept[5], kept[6], {kept[7], kept[8], kept[9]}, {1, 0, 0}};
    const auto scalars = ctx->saved_data["scalars"].toDoubleVector();
    std::copy(scalars.begin(), scalars.end(), h.scalar);
    const int64_t need = ctx->saved_data["need"].toInt();
    if (dz.size(1) > 1 && dz.stride(1) != 1) dz = dz.contiguous();
    Tensor dlogits, dbias;
    if (need & 1) dlogits = at::empty(logits.sizes(), logits.options());
    if (need & 2) dbias = logits.numel() ? at::empty(bias.sizes(), bias.options()) : at::zeros(bias.sizes(), bias.options());
    ce_logits s = describe(logits, bias, h, code(dz));
    const ce_logits_grad g = {ptr(dz), dz.stride(0), ptr(dlogits), ptr(dbias)};
    check(ce_process_logits_backward_workspace(&s, &g, &s.workspace_bytes), "process_logits_backward");
    const Tensor ws = bytes(s.workspace_bytes, logits);
    s.workspace = ptr(ws);
    check(ce_process_logits_backward(&s, &g, stream_of(logits)), "process_logits_backward");
    return once({dlogits, dbias, Tensor()});
  }
};

// A [.., width] table whose rows repeat over the logits' rows, as a dense [B, width].
Tensor table(const char* name, const Tensor& t, at::IntArrayRef lead, int64_t width) {
  const int64_t k = t.dim() - 1;
  if (k < 0 || t.size(k) != width) bad("process_logits: ", name, " must end in ", width, " entries, got ", t.sizes());
  const auto axes = t.sizes().slice(0, k);
  const bool fits = k == 0 || (k == 1 && (lead.size() <= 1 || axes[0] == 1)) || (k <= (int64_t)lead.size() && axes == lead.slice(lead.size() - k));
  if (!fits) bad("process_logits: ", name, "'s leading axes ", axes, " must be the last of the logits' ", lead);
  return k == 1 ? t.contiguous() : t.reshape({c10::multiply_integers(axes), width}).contiguous();
}
// One entry a row, dense, in `type` (int64 is narrowed; what does not fit keeps its meaning: past every end, or before every start).
Maybe per_row(const char* name, const Maybe& t, at::IntArrayRef lead, at::ScalarType type) {
  if (!t) return t;
  if (t->sizes() != lead) bad("process_logits: ", name, " must hold one entry a row, ", lead, ", got ", t->sizes());
  if (t->scalar_type() == type) return t->contiguous();
  if (type != at::kInt || t->scalar_type() != at::kLong) bad("process_logits: ", name, " must be ", type, ", not ", t->scalar_type());
  return t->clamp(-1, INT32_MAX).to(at::kInt).contiguous();
}

Tensor process_logits(const Tensor& logits, Maybe tokens, Maybe lengths, Maybe prompt_lengths, const py::object& repetition, const py::object& presence, const py::object& frequency, Maybe bias, Maybe mask,
                      Maybe mask_index, const Maybe& out) {
  const char* op = "process_logits";
  if (logits.dim() < 1) bad("process_logits: logits must be [..., V]");
  if (!real(logits.scalar_type())) bad("process_logits: logits must be float32, bfloat16 or float16, not ", logits.scalar_type());
  on_gpu(op, logits);
  const char* names[3] = {"repetition", "presence", "frequency"};
  const py::object* given[3] = {&repetition, &presence, &frequency};
  Maybe penalty[3];
  Shaping h = {{}, {}, {}, {}, {}, {}, {1, 0, 0}};
  for (int k = 0; k < 3; ++k) {
    if (THPVariable_Check(given[k]->ptr())) penalty[k] = THPVariable_Unpack(given[k]->ptr());
    else h.scalar[k] = number(*given[k]);
  }
  same_device(op, logits, {&tokens, &lengths, &prompt_lengths, &penalty[0], &penalty[1], &penalty[2], &bias, &mask, &mask_index, &out});
  no_graph(op, {&out});
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const int64_t V = logits.size(-1), rows = c10::multiply_integers(lead);
  for (int k = 0; k < 3; ++k)
    if (penalty[k]) {
      if (penalty[k]->requires_grad() && at::GradMode::is_enabled()) bad("process_logits: ", names[k], " has no gradient here: detach it");
      penalty[k] = per_row(names[k], penalty[k], lead, at::kFloat);
    }
  if (tokens) {
    if (tokens->dim() != logits.dim() || tokens->sizes().slice(0, tokens->dim() - 1) != lead) bad("process_logits: tokens must be ", lead, " + [L], got ", tokens->sizes());
    const auto t = tokens->scalar_type();
    if (t != at::kByte && t != at::kInt && t != at::kLong) bad("process_logits: tokens must be uint8, int32 or int64, not ", t);
    if (tokens->dim() != 2) tokens = tokens->reshape({rows, tokens->size(-1)});
    lengths = per_row("lengths", lengths, lead, at::kInt);
    prompt_lengths = per_row("prompt_lengths", prompt_lengths, lead, at::kInt);
  } else if (lengths || prompt_lengths) {
    bad("process_logits: lengths without tokens");
  }
  if (mask) {
    const auto t = mask->scalar_type();
    if (!flag(t) && t != at::kInt) bad("process_logits: mask must be bool, uint8 or int32 words, not ", t);
    if (mask_index && mask->dim() != 2) bad("process_logits: an indexed mask must be a table [S, ..]");
    mask_index = per_row("mask_index", mask_index, lead, at::kInt);
    mask = table("mask", *mask, mask_index ? at::IntArrayRef() : lead, t == at::kInt ? (V + 31) / 32 : V);
  } else if (mask_index) {
    bad("process_logits: mask_index without a mask");
  }
  bool grad = logits.requires_grad();
  if (bias) {
    if (bias->scalar_type() != at::kFloat && bias->scalar_type() != logits.scalar_type()) bad("process_logits: bias must be float32 or of the logits' type, not ", bias->scalar_type());
    bias = table("bias", *bias, lead, V);
    grad |= bias->requires_grad();
  }
  grad = grad && at::GradMode::is_enabled();
  if (grad && out) bad("process_logits: out cannot be given where gradients are wanted");
  Tensor flat = logits.dim() == 2 ? logits : logits.reshape({rows, V});
  if (V > 1 && flat.stride(1) != 1) flat = flat.contiguous();
  const Tensor none;
  h.tokens = tokens.value_or(none);
  h.lengths = lengths.value_or(none);
  h.prompt_lengths = prompt_lengths.value_or(none);
  h.mask = mask.value_or(none);
  h.mask_index = mask_index.value_or(none);
  for (int k = 0; k < 3; ++k) h.penalty[k] = penalty[k].value_or(none);
  Tensor z;
  if (grad) {
    z = Logits::apply(flat, bias, h);
  } else if (!out) {
    z = at::empty({rows, V}, logits.options());
    logits_forward(flat, bias.value_or(none), h, z);
  } else {
    if (out->sizes() != logits.sizes() || (out->scalar_type() != at::kFloat && out->scalar_type() != logits.scalar_type()))
      bad("process_logits: out must be ", logits.sizes(), ", float32 or of the logits' type");
    const auto strides = at::detail::computeStride(out->sizes(), out->strides(), at::DimVector{rows, V});
    if (!strides || (V > 1 && (*strides)[1] != 1)) bad("process_logits: out's leading axes must collapse into one stride, its last be dense");
    const Maybe to = out->view({rows, V}), nothing, mf = flat;
    const bool same = to->data_ptr() == flat.data_ptr() && to->scalar_type() == flat.scalar_type() && to->strides() == flat.strides();
    apart(op, to, "out", {same ? &nothing : &mf, &tokens, &lengths, &prompt_lengths, &mask, &mask_index, &bias, &penalty[0], &penalty[1], &penalty[2]});
    logits_forward(flat, bias.value_or(none), h, *to);
    written(out);
    return *out;
  }
  return logits.dim() == 2 ? z : z.view(logits.sizes());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  static PyObject* error = nullptr;
  m.def("set_error", [](py::object cls) { error = cls.release().ptr(); }, "the exception class that a refusal of the C-ABI raises");
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Refused& e) {
      PyErr_SetString(error ? error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("linear_scan", &linear_scan);
  m.def("advantages", &advantages);
  m.def("process_logits", &process_logits);
}
