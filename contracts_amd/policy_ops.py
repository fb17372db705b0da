"""The policy's own operators on either side of a rollout, over the engine's device layouts (include/contracts_policy.h).

The engine makes what a policy trains on — time-major trajectory planes with done flags (`engine.Trajectory`) — and takes what it
answers with — float scores, of which the step kernel takes the first maximum (`BatchedEnv.step_policy_device(.., "argmax")`).

* `linear_scan`: the gated linear recurrence along the time axis (a recurrent policy's memory, discounted returns), episodes ending
  inside the planes; differentiable; one step of it moves a sampler's state on.
* `advantages`: generalised advantage estimation over the planes of a (wrapped) ring.
* `process_logits`: penalties for repeated tokens, biases and masks on scores or logits, differentiable.

Tensors live on an MI355X (there is no CPU path) and a call is asynchronous on torch's current stream of their device; outputs
are new tensors unless `out=` names them, scratch memory comes from torch's allocator, nothing is kept between calls, and every call may
be captured into a graph.  Ordering against other streams (env slices on side streams) is the caller's, as for the engine's steps.
A tensor whose last axis is not dense, or whose leading axes do not collapse into one stride, is copied first."""
import ctypes as C

import torch

from . import _lib

_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float64: _lib.F64, torch.uint8: _lib.U8,
         torch.bool: _lib.U8, torch.int32: _lib.I32, torch.int64: _lib.I64}
_REAL = (torch.float32, torch.bfloat16, torch.float16)


def _need(cond, what, *args):
    if not cond:
        raise ValueError(what % args if args else what)


def _device(op, *tensors):
    """the one device that all of a call's tensors live on"""
    dev = tensors[0].device
    _need(dev.type == "cuda", "%s: tensors must live on a GPU (there is no CPU path), got %s", op, dev)
    for t in tensors[1:]:
        _need(t is None or t.device == dev, "%s: all tensors must live on one device", op)
    return dev


def _ptr(t):
    return None if t is None or t.numel() == 0 else t.data_ptr()


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


def _span(t):
    """first and last byte a tensor reaches"""
    lo = hi = t.data_ptr()
    for n, s in zip(t.shape, t.stride()):
        lo, hi = (lo + (n - 1) * s * t.element_size(), hi) if s < 0 else (lo, hi + (n - 1) * s * t.element_size())
    return lo, hi + t.element_size()


def _apart(op, out, name, *inputs):
    """an output may not overlap an input"""
    if out is None or out.numel() == 0:
        return
    lo, hi = _span(out)
    for t in inputs:
        if t is not None and t.numel() and t.device == out.device:
            a, b = _span(t)
            _need(hi <= a or b <= lo, "%s: %s overlaps an input", op, name)


def _workspace(fn, dev, *structs):
    nbytes = C.c_uint64()
    _lib.check_policy(fn(*[C.byref(s) for s in structs], C.byref(nbytes)), fn.__name__)
    return None if nbytes.value == 0 else torch.empty(nbytes.value, dtype=torch.uint8, device=dev)


# ---- linear_scan ---------------------------------------------------------------------------------------------------------------
def _scan_struct(x, gate, done, reverse):
    s = _lib.CeScan(abi_version=_lib.POLICY_ABI_VERSION, device=x.device.index, dtype=_CODE[x.dtype], flags=_lib.SCAN_REVERSE * bool(reverse))
    s.steps, s.rows, s.channels = x.shape
    s.x_step, s.x_row = x.stride(0), x.stride(1)
    s.x = _ptr(x)
    if isinstance(gate, torch.Tensor):
        s.gate_dtype, s.heads, s.gate_step, s.gate_row, s.gate = _CODE[gate.dtype], gate.shape[2], gate.stride(0), gate.stride(1), gate.data_ptr()
    else:
        s.gate_dtype, s.heads, s.decay = s.dtype, s.channels, gate
    if done is not None:
        s.done_step, s.done_row, s.done = done.stride(0), done.stride(1), _ptr(done)
    return s


def _scan_forward(x, gate, state, done, reverse, y, last, want_saved):
    L = _lib.load_policy()
    T, E, Ch = x.shape
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    y = torch.empty((T, E, Ch), dtype=x.dtype, device=x.device) if y is None else y
    last = torch.empty((E, Ch), dtype=acc, device=x.device) if last is None else last
    saved = torch.empty((-(-T // _lib.SCAN_SAVED_STEPS), E, Ch), dtype=torch.float32, device=x.device) if want_saved else None
    s = _scan_struct(x, gate, done, reverse)
    s.y, s.last, s.state, s.saved = _ptr(y), _ptr(last), _ptr(state), _ptr(saved)
    ws = _workspace(L.ce_linear_scan_workspace, x.device, s)
    s.workspace, s.workspace_bytes = _ptr(ws), 0 if ws is None else ws.numel()
    _lib.check_policy(L.ce_linear_scan(C.byref(s), _stream(x.device)), "linear_scan")
    return y, last, saved


def _scan_backward(x, gate, done, reverse, saved, dy, dlast, need_state):
    L = _lib.load_policy()
    T, E, Ch = x.shape
    dx = torch.empty((T, E, Ch), dtype=x.dtype, device=x.device)
    dgate = (torch.empty if x.numel() else torch.zeros)(gate.shape, dtype=gate.dtype, device=x.device) if isinstance(gate, torch.Tensor) else None
    dstate = torch.empty((E, Ch), dtype=torch.float32, device=x.device) if need_state else None
    s = _scan_struct(x, gate, done, reverse)
    s.saved = _ptr(saved)
    dy = torch.zeros((T, E, Ch), dtype=x.dtype, device=x.device) if dy is None else dy.contiguous()
    dlast = None if dlast is None else dlast.contiguous()
    g = _lib.CeScanGrad(dy=_ptr(dy), dlast=_ptr(dlast), dx=_ptr(dx), dgate=_ptr(dgate), dstate=_ptr(dstate))
    ws = _workspace(L.ce_linear_scan_backward_workspace, x.device, s, g)
    s.workspace, s.workspace_bytes = _ptr(ws), 0 if ws is None else ws.numel()
    _lib.check_policy(L.ce_linear_scan_backward(C.byref(s), C.byref(g), _stream(x.device)), "linear_scan_backward")
    return dx, dgate, dstate


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, done, reverse):
        ctx.set_materialize_grads(False)
        y, last, saved = _scan_forward(x, gate, state, done, reverse, None, None, True)
        ctx.reverse, ctx.const = reverse, None if isinstance(gate, torch.Tensor) else gate
        ctx.save_for_backward(x, gate if ctx.const is None else None, done, saved)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        x, gate, done, saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dgate, dstate = _scan_backward(x, gate if ctx.const is None else ctx.const, done, ctx.reverse, saved, dy, dlast, need[2])
        return dx if need[0] else None, dgate if need[1] else None, dstate, None, None


def linear_scan(x, gate, state=None, done=None, reverse=False, out=None, state_out=None):
    """The gated linear recurrence along the time axis: (y [T, E, C] in x's type, last [E, C] float32).

    Forward in time h_t = a_t h_{t-1} + x_t from h_{-1} = state, `last` = the state after step T - 1; with `reverse`
    h_t = a_t h_{t+1} + x_t from h_T = state, `last` = h_0.  done[t, e] says that an episode ended with step t: nothing crosses the border
    between t and t + 1, in either direction (going forward, `last` is 0 where done[T - 1]).  So `last` is the `state` of the next
    call: one of T = 1 moves a sampler's memory on, and a rollout may be scanned in pieces.

    x: [T, E, C] float32, bfloat16 or float16 (float64 without gradients).  gate: [T, E, H] of x's type or float32, H
    dividing C (channel c is under gate c // (C // H)); strides of 0 share it along time or rows; or a float, one constant.  A gate
    of exactly 0 forgets the state whatever it held, as done does.  state: [E, C] float32 (float64 with x).  done: [T, E] bool or uint8.
    The state is float32 throughout (float64 with x); y is rounded once.  Differentiable in x, gate and state (dy and dlast), from the
    unrounded states: one of every 16 is kept between the passes.  out / state_out: dense tensors to write to, without gradients;
    state_out may be `state`."""
    _need(isinstance(x, torch.Tensor) and x.dim() == 3, "linear_scan: x must be [T, E, C]")
    tensor_gate = isinstance(gate, torch.Tensor)
    dev = _device("linear_scan", x, gate if tensor_gate else None, state, done, out, state_out)
    _need(x.dtype in _REAL or x.dtype == torch.float64, "linear_scan: x must be float32, bfloat16, float16 or float64, not %s", x.dtype)
    T, E, Ch = x.shape
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    if tensor_gate:
        _need(gate.dim() == 3 and gate.shape[:2] == x.shape[:2] and (gate.shape[2] == Ch or (gate.shape[2] and Ch % gate.shape[2] == 0)),
              "linear_scan: gate must be [T, E, H] with H dividing C, got %s for x %s", tuple(gate.shape), tuple(x.shape))
        _need(gate.dtype == x.dtype or (gate.dtype == torch.float32 and x.dtype in _REAL), "linear_scan: gate must be of x's type or float32, not %s", gate.dtype)
    else:
        gate = float(gate)
    if state is not None:
        _need(tuple(state.shape) == (E, Ch) and state.dtype == acc, "linear_scan: state must be %s %s", acc, (E, Ch))
    if done is not None:
        _need(tuple(done.shape) == (T, E) and done.dtype in (torch.bool, torch.uint8), "linear_scan: done must be bool or uint8 [T, E]")
        done = done.view(torch.uint8) if done.dtype == torch.bool else done
    grad = torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, gate, state))
    for name, t, shape, dtype in (("out", out, (T, E, Ch), x.dtype), ("state_out", state_out, (E, Ch), acc)):
        if t is not None:
            _need(not grad, "linear_scan: %s cannot be given where gradients are wanted", name)
            _need(tuple(t.shape) == shape and t.dtype == dtype and t.is_contiguous(), "linear_scan: %s must be a dense %s %s", name, dtype, shape)
    far = (1 << 28) // (255 // max(Ch, 1) + 1)  # rows that far apart are more than a wave's 32-bit offsets
    if (x.stride(2) != 1 and Ch > 1) or x.stride(1) > far:
        x = x.contiguous()
    if tensor_gate and ((gate.stride(2) != 1 and gate.shape[2] > 1) or gate.stride(1) > far):
        gate = gate.contiguous()
    in_place = state_out is not None and state is not None and state_out.data_ptr() == state.data_ptr()
    _need(not in_place or state.is_contiguous(), "linear_scan: state_out overlaps an input")
    if state is not None:
        state = state.contiguous()
    _apart("linear_scan", out, "out", x, gate if tensor_gate else None, state, done, state_out)
    _apart("linear_scan", state_out, "state_out", x, gate if tensor_gate else None, None if in_place else state, done)
    if grad:
        _need(x.dtype != torch.float64, "linear_scan: float64 has no backward pass")
        return _Scan.apply(x, gate, state, done, bool(reverse))
    y, last, _ = _scan_forward(x, gate, state, done, reverse, out, state_out, False)
    return y, last


# ---- advantages -----------------------------------------------------------------------------------------------------------------
def advantages(reward, value, last_value=None, done=None, gamma=0.99, lam=0.95, first_plane=0, out=None):
    """Generalised advantage estimation over the planes of a rollout: (advantage, return), float32 [P, E, n] in the planes' order.

    delta_t = r_t + gamma V_{t+1} - V_t,  A_t = delta_t + gamma lam A_{t+1},  return_t = A_t + V_t; V_P = last_value (None: 0), and nothing crosses
    the border behind a step with done.  reward: [P, E, n] float64 (the engine's) or float32; value: [P, E, n] float32, bfloat16 or float16;
    last_value: [E, n] in value's type; done: [P, E] (the env's) or [P, E, n] (each agent's), bool or uint8.  Time t lies in plane
    (first_plane + t) % P, as a wrapped `Trajectory` holds it (its oldest plane is `traj.c.first_plane`).  Sums run in float64.
    out: a pair of dense float32 [P, E, n] tensors.  Not differentiable: targets are constants of a policy's loss."""
    _need(isinstance(reward, torch.Tensor) and reward.dim() == 3, "advantages: reward must be [P, E, n]")
    adv, ret = (None, None) if out is None else out
    dev = _device("advantages", reward, value, last_value, done, adv, ret)
    P, E, n = reward.shape
    _need(reward.dtype in (torch.float64, torch.float32), "advantages: reward must be float64 or float32, not %s", reward.dtype)
    _need(tuple(value.shape) == (P, E, n) and value.dtype in _REAL, "advantages: value must be float32, bfloat16 or float16 %s", (P, E, n))
    _need(last_value is None or (tuple(last_value.shape) == (E, n) and last_value.dtype == value.dtype), "advantages: last_value must be %s %s", value.dtype, (E, n))
    _need(done is None or (tuple(done.shape) in ((P, E), (P, E, n)) and done.dtype in (torch.bool, torch.uint8)), "advantages: done must be bool or uint8 [P, E] or [P, E, n]")
    _need(0 <= int(first_plane) < max(P, 1), "advantages: first_plane out of range")
    for t in (adv, ret):
        _need(t is None or (tuple(t.shape) == (P, E, n) and t.dtype == torch.float32 and t.is_contiguous()), "advantages: out must be two dense float32 %s", (P, E, n))
    reward, value = reward.detach().contiguous(), value.detach().contiguous()
    last_value = None if last_value is None else last_value.detach().contiguous()
    done = None if done is None else done.contiguous()
    _apart("advantages", adv, "out", reward, value, last_value, done, ret)
    _apart("advantages", ret, "out", reward, value, last_value, done)
    adv = torch.empty((P, E, n), dtype=torch.float32, device=dev) if adv is None else adv
    ret = torch.empty((P, E, n), dtype=torch.float32, device=dev) if ret is None else ret
    a = _lib.CeAdvantage(abi_version=_lib.POLICY_ABI_VERSION, device=dev.index, reward_dtype=_CODE[reward.dtype], value_dtype=_CODE[value.dtype],
                         flags=_lib.ADV_DONE_PER_AGENT * (done is not None and done.dim() == 3), first_plane=int(first_plane), planes=P, rows=E, agents=n,
                         gamma=float(gamma), lam=float(lam), reward=_ptr(reward), value=_ptr(value), last_value=_ptr(last_value), done=_ptr(done),
                         advantage=_ptr(adv), ret=_ptr(ret))
    L = _lib.load_policy()
    _lib.check_policy(L.ce_advantages(C.byref(a), _stream(dev)), "advantages")
    return adv, ret


# ---- process_logits ---------------------------------------------------------------------------------------------------------------
def pack_mask(allowed):
    """bool [..., V] -> the words of a packed mask, int32 [..., ceil(V / 32)]: bit v % 32 of word v // 32"""
    V = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed.to(torch.int64), (0, -V % 32)).unflatten(-1, (-1, 32))
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _logits_struct(logits, h, out_dtype):
    s = _lib.CeLogits(abi_version=_lib.POLICY_ABI_VERSION, device=logits.device.index, dtype=_CODE[logits.dtype], out_dtype=_CODE[out_dtype])
    s.rows, s.vocab = logits.shape
    s.logits_row, s.logits = logits.stride(0), _ptr(logits)
    if h["tokens"] is not None:
        t = h["tokens"]
        s.token_dtype, s.history, s.token_row, s.token_step, s.tokens = _CODE[t.dtype], t.shape[1], t.stride(0), t.stride(1), _ptr(t)
        s.lengths, s.prompt_lengths = (_ptr(h["lengths"]), _ptr(h["prompt_lengths"])) if s.tokens else (None, None)
        for name in ("repetition", "presence", "frequency"):
            v = h[name]
            if isinstance(v, torch.Tensor):
                setattr(s, name, _ptr(v))
            else:
                setattr(s, name + "_all", v)
    if h["mask"] is not None:
        s.mask_dtype, s.mask_rows, s.mask, s.mask_index = _CODE[h["mask"].dtype], h["mask"].shape[0], _ptr(h["mask"]), _ptr(h["mask_index"])
    return s


def _logits_bias(s, bias):
    if bias is not None:
        s.bias_dtype, s.bias_rows, s.bias = _CODE[bias.dtype], bias.shape[0], _ptr(bias)


class _Logits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, h):
        ctx.set_materialize_grads(False)
        ctx.h = {k: v for k, v in h.items() if not isinstance(v, torch.Tensor)}
        ctx.names = [k for k, v in h.items() if isinstance(v, torch.Tensor)]
        ctx.save_for_backward(logits, bias, *[h[k] for k in ctx.names])
        return _logits_forward(logits, bias, h, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dz):
        if dz is None:
            return None, None, None
        logits, bias, *rest = ctx.saved_tensors
        h = dict(ctx.h, **dict(zip(ctx.names, rest)))
        L = _lib.load_policy()
        dz = dz if dz.stride(1) == 1 or dz.shape[1] == 1 else dz.contiguous()
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if ctx.needs_input_grad[0] else None
        dbias = torch.zeros_like(bias) if ctx.needs_input_grad[1] and logits.numel() == 0 else torch.empty_like(bias) if ctx.needs_input_grad[1] else None
        s = _logits_struct(logits, h, dz.dtype)
        _logits_bias(s, bias)
        g = _lib.CeLogitsGrad(dout=_ptr(dz), dout_row=dz.stride(0), dlogits=_ptr(dlogits), dbias=_ptr(dbias))
        ws = _workspace(L.ce_process_logits_backward_workspace, logits.device, s, g)
        s.workspace, s.workspace_bytes = _ptr(ws), 0 if ws is None else ws.numel()
        _lib.check_policy(L.ce_process_logits_backward(C.byref(s), C.byref(g), _stream(logits.device)), "process_logits_backward")
        return dlogits, dbias, None


def _logits_forward(logits, bias, h, out):
    L = _lib.load_policy()
    out = torch.empty(logits.shape, dtype=h["out_dtype"], device=logits.device) if out is None else out
    s = _logits_struct(logits, h, out.dtype)
    _logits_bias(s, bias)
    s.out, s.out_row = _ptr(out), out.stride(0)
    _lib.check_policy(L.ce_process_logits(C.byref(s), _stream(logits.device)), "process_logits")
    return out


def _table(op, name, t, lead, width):
    """a [.., width] table whose rows repeat over the logits' rows, as [B, width]"""
    k = t.dim() - 1
    rows = 1
    for d in lead:
        rows *= d
    _need(k >= 0 and t.shape[-1] == width, "%s: %s must end in %d entries, got %s", op, name, width, tuple(t.shape))
    _need(k == 0 or (k == 1 and (len(lead) <= 1 or t.shape[0] == 1)) or tuple(t.shape[:-1]) == tuple(lead)[len(lead) - k:], "%s: %s's leading axes %s must be the last of the logits' %s", op, name, tuple(t.shape[:-1]), tuple(lead))
    t = t.reshape(-1, width) if t.numel() else t.reshape(t.shape[0] if k else 1, width)
    return t.contiguous()


def process_logits(logits, *, tokens=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, mask=None,
                   mask_index=None, out=None):
    """Scores or logits shaped ahead of a selection: penalties for repeated tokens (or past actions), biases, masks.

    logits: [..., V] float32, bfloat16 or float16; the leading axes are R rows (envs x agents, sequences).  In this order, in float32, rounded once:
      tokens      [..., L] uint8, int32 or int64 of any strides (`actions.permute(1, 2, 0)` of [T, E, n] action planes), a row's history; only its first
                  `lengths` [...] count, the first `prompt_lengths` [...] of these are its prompt; ids outside [0, V) are passed over
      repetition  > 0: l / repetition where l > 0, else l * repetition, for a token seen anywhere in the history
      presence    taken off a token that occurs behind the prompt;  frequency: taken off as often as it occurs there.
                  Each of the three is a float or a float32 [...] tensor, one for each row
      bias        added: [V], the last axes of the logits ([n, V] for [E, n, V]), or [B, V] for logits [R, V] with B dividing R (row r takes
                  row r mod B); float32 or the logits' type
      mask        -inf where it forbids, whatever stands there; bool / uint8 [.., V] (nonzero = allowed), or int32 [.., ceil(V / 32)] words
                  (`pack_mask`); rows as for bias, or `mask_index` int32 [...] names a row's row of a [S, ..] table (the state of its
                  grammar; negative: all is allowed, past the end: nothing).  A row whose mask leaves nothing is -inf throughout
                  (`step_policy_device(.., "argmax")` then takes action 0).
    out: float32 or the logits' type, rows dense; it may be `logits` itself; not where gradients are wanted.
    Differentiable in logits and bias: gradients scale as l was, vanish where forbidden; bias gradients sum over rows in float32."""
    op = "process_logits"
    _need(isinstance(logits, torch.Tensor) and logits.dim() >= 1, "process_logits: logits must be [..., V]")
    penal = [v for v in (repetition, presence, frequency) if isinstance(v, torch.Tensor)]
    dev = _device(op, logits, tokens, lengths, prompt_lengths, bias, mask, mask_index, out, *penal)
    _need(logits.dtype in _REAL, "process_logits: logits must be float32, bfloat16 or float16, not %s", logits.dtype)
    lead, V = tuple(logits.shape[:-1]), logits.shape[-1]
    rows = logits.shape[:-1].numel()
    h = dict(tokens=None, lengths=None, prompt_lengths=None, mask=None, mask_index=None, out_dtype=logits.dtype)

    def per_row(name, t, dtype):
        _need(tuple(t.shape) == lead, "process_logits: %s must hold one entry a row, %s, got %s", name, lead, tuple(t.shape))
        _need(t.dtype in dtype, "process_logits: %s must be %s, not %s", name, dtype[0], t.dtype)
        return t.detach().to(dtype[0]).reshape(-1).contiguous()

    for name, v in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        h[name] = per_row(name, v, (torch.float32,)) if isinstance(v, torch.Tensor) else float(v)
    _need(tokens is not None or (lengths is None and prompt_lengths is None), "process_logits: lengths without tokens")
    if tokens is not None:
        _need(tokens.dim() == logits.dim() and tuple(tokens.shape[:-1]) == lead, "process_logits: tokens must be %s + [L], got %s", lead, tuple(tokens.shape))
        _need(tokens.dtype in (torch.uint8, torch.int32, torch.int64), "process_logits: tokens must be uint8, int32 or int64, not %s", tokens.dtype)
        h["tokens"] = tokens.reshape(rows, tokens.shape[-1])
        if lengths is not None:
            h["lengths"] = per_row("lengths", lengths, (torch.int32, torch.int64))
        if prompt_lengths is not None:
            h["prompt_lengths"] = per_row("prompt_lengths", prompt_lengths, (torch.int32, torch.int64))
    if mask is not None:
        _need(mask.dtype in (torch.bool, torch.uint8, torch.int32), "process_logits: mask must be bool, uint8 or int32 words, not %s", mask.dtype)
        packed = mask.dtype == torch.int32
        if mask_index is not None:
            _need(mask.dim() == 2, "process_logits: an indexed mask must be a table [S, ..]")
            h["mask_index"] = per_row("mask_index", mask_index, (torch.int32, torch.int64))
        mask = mask.view(torch.uint8) if mask.dtype == torch.bool else mask
        h["mask"] = _table(op, "mask", mask, lead, -(-V // 32) if packed else V)
    else:
        _need(mask_index is None, "process_logits: mask_index without a mask")
    if bias is not None:
        _need(bias.dtype in (torch.float32, logits.dtype), "process_logits: bias must be float32 or of the logits' type, not %s", bias.dtype)
        bias = _table(op, "bias", bias, lead, V)
    flat = logits.reshape(rows, V)
    if V > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    grad = torch.is_grad_enabled() and (logits.requires_grad or (bias is not None and bias.requires_grad))
    if out is not None:
        _need(not grad, "process_logits: out cannot be given where gradients are wanted")
        _need(out.shape == logits.shape and out.dtype in (torch.float32, logits.dtype), "process_logits: out must be %s, float32 or of the logits' type", tuple(logits.shape))
        try:
            to = out.view(rows, V)
        except RuntimeError:
            to = None
        _need(to is not None and (V <= 1 or to.stride(1) == 1), "process_logits: out's leading axes must collapse into one stride, its last be dense")
        same = to.data_ptr() == flat.data_ptr() and to.dtype == flat.dtype and to.stride() == flat.stride()
        _apart(op, to, "out", None if same else flat, h["tokens"], h["lengths"], h["prompt_lengths"], h["mask"], h["mask_index"], bias,
               *[h[k] for k in ("repetition", "presence", "frequency") if isinstance(h[k], torch.Tensor)])
        _logits_forward(flat, bias, h, to)
        return out
    return (_Logits.apply(flat, bias, h) if grad else _logits_forward(flat, bias, h, None)).view(logits.shape)
