// cp_torch.cpp — the policy operators (include/contracts_policy.h) for torch tensors: allocates outputs and scratch memory, describes the tensors
// to the C-ABI, and takes gradients through nodes that need no interpreter.
//
// Host-side marshalling only, because a call's latency is the host's: a forward call took 11-14 us through ctypes, of which the
// launch is 3, and a forward and backward pass 120 us, most of it the interpreter in torch's backward thread.  What is checked about the
// arguments lies in policy_ops.py and, for everything that reaches the device, in the C-ABI itself.
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

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
  Tensor ws;
  if (T >= CE_SCAN_SPLIT_STEPS) {
    check(ce_linear_scan_workspace(&s, &s.workspace_bytes), "linear_scan");
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
    const Tensor dy = grads[0].defined() ? grads[0].contiguous() : at::zeros({T, E, C}, x.options());
    const Tensor dlast = grads[1].defined() ? grads[1].contiguous() : Tensor();
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

std::tuple<Tensor, Tensor> linear_scan(const Tensor& x, const Maybe& gate, double decay, const Maybe& state, const Maybe& done, bool reverse, const Maybe& out, const Maybe& state_out, bool grad) {
  if (grad) {
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
std::tuple<Tensor, Tensor> advantages(const Tensor& reward, const Tensor& value, const Maybe& last_value, const Maybe& done, double gamma, double lam, int64_t first, const Maybe& adv_out,
                                      const Maybe& ret_out) {
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
    Tensor dz = grads[0];
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

Tensor process_logits(const Tensor& logits, const Maybe& bias, const Maybe& tokens, const Maybe& lengths, const Maybe& prompt_lengths, const Maybe& mask, const Maybe& mask_index,
                      const Maybe& repetition, const Maybe& presence, const Maybe& frequency, double repetition_all, double presence_all, double frequency_all, const Maybe& out, bool grad) {
  const Tensor none;
  const Shaping h = {tokens.value_or(none), lengths.value_or(none), prompt_lengths.value_or(none), mask.value_or(none), mask_index.value_or(none),
                     {repetition.value_or(none), presence.value_or(none), frequency.value_or(none)}, {repetition_all, presence_all, frequency_all}};
  if (grad) return Logits::apply(logits, bias, h);
  const Tensor to = out ? *out : at::empty(logits.sizes(), logits.options());
  logits_forward(logits, bias.value_or(none), h, to);
  written(out);
  return to;
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
