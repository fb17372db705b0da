"""The policy's own operators on either side of a rollout, over the engine's device layouts (include/contracts_policy.h).

The engine makes what a policy trains on — time-major trajectory planes with done flags (`engine.Trajectory`) — and takes what it
answers with — float scores, of which the step kernel takes the first maximum (`BatchedEnv.step_policy_device(.., "argmax")`).

* `linear_scan`: the gated linear recurrence along the time axis (a recurrent policy's memory, discounted returns), episodes ending
  inside the planes; differentiable; one step of it moves a sampler's state on.
* `advantages`: generalised advantage estimation over the planes of a (wrapped) ring.
* `process_logits`: penalties for repeated tokens, biases and masks on scores or logits, differentiable.

Tensors live on an MI355X (there is no CPU path) and a call is asynchronous on torch's current stream of their device; outputs
are new tensors unless `out=` names them, scratch memory comes from torch's allocator, nothing is kept between calls, and every call may
be captured into a graph (a backward pass together with its forward pass, and with leaves of its own: torch's engine ends the process where
a captured backward pass meets the nodes of an eager graph of the same leaves).  Ordering against other streams (env slices on side streams) is the caller's, as for the engine's steps.
A tensor whose last axis is not dense, or whose leading axes do not collapse into one stride, is copied first."""
import torch

from . import _lib

_REAL = (torch.float32, torch.bfloat16, torch.float16)
_loaded = None


def _ext():
    global _loaded
    if _loaded is None:
        _loaded = _lib.load_policy_torch()
    return _loaded


def _bad(what, *args):
    raise ValueError(what % args if args else what)


def _device(op, first, *tensors):
    """the one device that all of a call's tensors live on"""
    dev = first.device
    if dev.type != "cuda":
        _bad("%s: tensors must live on a GPU (there is no CPU path), got %s", op, dev)
    for t in tensors:
        if t is not None and t.device != dev:
            _bad("%s: all tensors must live on one device", op)
    return dev


def _span(t):
    """first and last byte a tensor reaches"""
    lo = t.data_ptr()
    return lo, lo + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _apart(op, out, name, *inputs):
    """an output may not overlap an input"""
    if out is None or out.numel() == 0:
        return
    lo, hi = _span(out)
    for t in inputs:
        if t is not None and t.numel() and t.device == out.device:
            a, b = _span(t)
            if not (hi <= a or b <= lo):
                _bad("%s: %s overlaps an input", op, name)


# ---- linear_scan ---------------------------------------------------------------------------------------------------------------
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
    if not isinstance(x, torch.Tensor) or x.dim() != 3:
        _bad("linear_scan: x must be [T, E, C]")
    tensor_gate = isinstance(gate, torch.Tensor)
    _device("linear_scan", x, gate if tensor_gate else None, state, done, out, state_out)
    dtype = x.dtype
    double = dtype == torch.float64
    if dtype not in _REAL and not double:
        _bad("linear_scan: x must be float32, bfloat16, float16 or float64, not %s", dtype)
    T, E, Ch = x.shape
    acc = torch.float64 if double else torch.float32
    head = Ch // gate.shape[2] if tensor_gate and gate.dim() == 3 and gate.shape[2] else 1
    # rows that far apart are more than a wave's 32-bit offsets, unless rows are whole waves
    far = 1 << 62 if Ch % 256 == 0 and head & (head - 1) == 0 else (1 << 28) // (255 // Ch + 1)
    strides = x.stride()
    grad = x.requires_grad
    if tensor_gate:
        if gate.dim() != 3 or gate.shape[0] != T or gate.shape[1] != E or not (gate.shape[2] == Ch or (gate.shape[2] and Ch % gate.shape[2] == 0)):
            _bad("linear_scan: gate must be [T, E, H] with H dividing C, got %s for x %s", tuple(gate.shape), tuple(x.shape))
        if gate.dtype != dtype and (gate.dtype != torch.float32 or double):
            _bad("linear_scan: gate must be of x's type or float32, not %s", gate.dtype)
        grad = grad or gate.requires_grad
        s = gate.stride()
        if (s[2] != 1 and gate.shape[2] > 1) or s[1] >= far:
            gate = gate.contiguous()
    else:
        gate = float(gate)
    if state is not None:
        if state.dim() != 2 or state.shape[0] != E or state.shape[1] != Ch or state.dtype != acc:
            _bad("linear_scan: state must be %s %s", acc, (E, Ch))
        grad = grad or state.requires_grad
    if done is not None:
        if done.dim() != 2 or done.shape[0] != T or done.shape[1] != E or done.dtype not in (torch.bool, torch.uint8):
            _bad("linear_scan: done must be bool or uint8 [T, E]")
    if (strides[2] != 1 and Ch > 1) or strides[1] >= far:
        x = x.contiguous()
    grad = grad and torch.is_grad_enabled()
    if out is not None or state_out is not None:
        if grad:
            _bad("linear_scan: out and state_out cannot be given where gradients are wanted")
        for name, t, shape, kind in (("out", out, (T, E, Ch), dtype), ("state_out", state_out, (E, Ch), acc)):
            if t is not None and (tuple(t.shape) != shape or t.dtype != kind or not t.is_contiguous()):
                _bad("linear_scan: %s must be a dense %s %s", name, kind, shape)
        moved = state is not None and state.is_contiguous() and state_out is not None and state_out.data_ptr() == state.data_ptr()  # in place
        others = (x, gate if tensor_gate else None, done)
        _apart("linear_scan", out, "out", state, state_out, *others)
        _apart("linear_scan", state_out, "state_out", None if moved else state, *others)
    if state is not None and not state.is_contiguous():
        state = state.contiguous()
    if grad and double:
        _bad("linear_scan: float64 has no backward pass")
    return _ext().linear_scan(x, gate if tensor_gate else None, 0.0 if tensor_gate else gate, state, done, bool(reverse), out, state_out, grad)


# ---- advantages -----------------------------------------------------------------------------------------------------------------
def advantages(reward, value, last_value=None, done=None, gamma=0.99, lam=0.95, first_plane=0, out=None):
    """Generalised advantage estimation over the planes of a rollout: (advantage, return), float32 [P, E, n] in the planes' order.

    delta_t = r_t + gamma V_{t+1} - V_t,  A_t = delta_t + gamma lam A_{t+1},  return_t = A_t + V_t; V_P = last_value (None: 0), and nothing crosses
    the border behind a step with done.  reward: [P, E, n] float64 (the engine's) or float32; value: [P, E, n] float32, bfloat16 or float16;
    last_value: [E, n] in value's type; done: [P, E] (the env's) or [P, E, n] (each agent's), bool or uint8.  Time t lies in plane
    (first_plane + t) % P, as a wrapped `Trajectory` holds it (its oldest plane is `traj.c.first_plane`).  Sums run in float64.
    out: a pair of dense float32 [P, E, n] tensors.  Not differentiable: targets are constants of a policy's loss."""
    if not isinstance(reward, torch.Tensor) or reward.dim() != 3:
        _bad("advantages: reward must be [P, E, n]")
    adv, ret = (None, None) if out is None else out
    _device("advantages", reward, value, last_value, done, adv, ret)
    shape = P, E, n = reward.shape
    if reward.dtype != torch.float64 and reward.dtype != torch.float32:
        _bad("advantages: reward must be float64 or float32, not %s", reward.dtype)
    if value.shape != shape or value.dtype not in _REAL:
        _bad("advantages: value must be float32, bfloat16 or float16 %s", tuple(shape))
    if last_value is not None:
        if last_value.shape != shape[1:] or last_value.dtype != value.dtype:
            _bad("advantages: last_value must be %s %s", value.dtype, (E, n))
        last_value = last_value.contiguous()
    if done is not None:
        per_agent = done.dim() == 3
        if done.shape != (shape if per_agent else shape[:2]) or done.dtype not in (torch.bool, torch.uint8):
            _bad("advantages: done must be bool or uint8 [P, E] or [P, E, n]")
        done = done.contiguous()
    first_plane = int(first_plane)
    if not 0 <= first_plane < max(P, 1):
        _bad("advantages: first_plane out of range")
    reward, value = reward.contiguous(), value.contiguous()
    if out is not None:
        for t in out:
            if t.shape != shape or t.dtype != torch.float32 or not t.is_contiguous():
                _bad("advantages: out must be two dense float32 %s", tuple(shape))
        _apart("advantages", adv, "out", reward, value, last_value, done, ret)
        _apart("advantages", ret, "out", reward, value, last_value, done)
    return _ext().advantages(reward, value, last_value, done, float(gamma), float(lam), first_plane, adv, ret)


# ---- process_logits ---------------------------------------------------------------------------------------------------------------
def pack_mask(allowed):
    """bool [..., V] -> the words of a packed mask, int32 [..., ceil(V / 32)]: bit v % 32 of word v // 32"""
    V = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed.to(torch.int64), (0, -V % 32)).unflatten(-1, (-1, 32))
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _table(name, t, lead, width):
    """a [.., width] table whose rows repeat over the logits' rows, as a dense [B, width]"""
    k = t.dim() - 1
    if k < 0 or t.shape[-1] != width:
        _bad("process_logits: %s must end in %d entries, got %s", name, width, tuple(t.shape))
    if k == 1:
        if len(lead) > 1 and t.shape[0] != 1 and t.shape[0] != lead[-1]:
            _bad("process_logits: %s's leading axes %s must be the last of the logits' %s", name, tuple(t.shape[:-1]), tuple(lead))
        return t if t.is_contiguous() else t.contiguous()
    if k > 1 and tuple(t.shape[:-1]) != tuple(lead)[len(lead) - k:]:
        _bad("process_logits: %s's leading axes %s must be the last of the logits' %s", name, tuple(t.shape[:-1]), tuple(lead))
    return t.reshape(t.shape[:-1].numel(), width).contiguous()


def _per_row(name, t, lead, dtype):
    """one entry a row, dense, in dtype (int64 is narrowed)"""
    if t.shape != lead:
        _bad("process_logits: %s must hold one entry a row, %s, got %s", name, tuple(lead), tuple(t.shape))
    if t.dtype != dtype:
        if dtype != torch.int32 or t.dtype != torch.int64:
            _bad("process_logits: %s must be %s, not %s", name, dtype, t.dtype)
        t = t.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


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
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1:
        _bad("process_logits: logits must be [..., V]")
    dtype = logits.dtype
    if dtype not in _REAL:
        _bad("process_logits: logits must be float32, bfloat16 or float16, not %s", dtype)
    dev = _device("process_logits", logits, tokens, lengths, prompt_lengths, bias, mask, mask_index, out)
    lead, V = logits.shape[:-1], logits.shape[-1]
    rows = lead.numel()
    tensors, scalars = [], []
    for name, v, none in (("repetition", repetition, 1.0), ("presence", presence, 0.0), ("frequency", frequency, 0.0)):
        if isinstance(v, torch.Tensor):
            if v.device != dev:
                _bad("process_logits: all tensors must live on one device")
            if v.requires_grad and torch.is_grad_enabled():
                _bad("process_logits: %s has no gradient here: detach it", name)
            tensors.append(_per_row(name, v, lead, torch.float32))
            scalars.append(none)
        else:
            tensors.append(None)
            scalars.append(float(v))
    if tokens is not None:
        if tokens.dim() != logits.dim() or tokens.shape[:-1] != lead:
            _bad("process_logits: tokens must be %s + [L], got %s", tuple(lead), tuple(tokens.shape))
        if tokens.dtype not in (torch.uint8, torch.int32, torch.int64):
            _bad("process_logits: tokens must be uint8, int32 or int64, not %s", tokens.dtype)
        if tokens.dim() != 2:
            tokens = tokens.reshape(rows, tokens.shape[-1])
        if lengths is not None:
            lengths = _per_row("lengths", lengths, lead, torch.int32)
        if prompt_lengths is not None:
            prompt_lengths = _per_row("prompt_lengths", prompt_lengths, lead, torch.int32)
    elif lengths is not None or prompt_lengths is not None:
        _bad("process_logits: lengths without tokens")
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8, torch.int32):
            _bad("process_logits: mask must be bool, uint8 or int32 words, not %s", mask.dtype)
        if mask_index is not None:
            if mask.dim() != 2:
                _bad("process_logits: an indexed mask must be a table [S, ..]")
            mask_index = _per_row("mask_index", mask_index, lead, torch.int32)
        mask = _table("mask", mask, () if mask_index is not None else lead, -(-V // 32) if mask.dtype == torch.int32 else V)
    elif mask_index is not None:
        _bad("process_logits: mask_index without a mask")
    grad = logits.requires_grad
    if bias is not None:
        if bias.dtype != torch.float32 and bias.dtype != dtype:
            _bad("process_logits: bias must be float32 or of the logits' type, not %s", bias.dtype)
        bias = _table("bias", bias, lead, V)
        grad = grad or bias.requires_grad
    grad = grad and torch.is_grad_enabled()
    if grad and out is not None:
        _bad("process_logits: out cannot be given where gradients are wanted")
    flat = logits if logits.dim() == 2 else logits.reshape(rows, V)
    if V > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    to = None
    if out is not None:
        if out.shape != logits.shape or (out.dtype != torch.float32 and out.dtype != dtype):
            _bad("process_logits: out must be %s, float32 or of the logits' type", tuple(logits.shape))
        try:
            to = out.view(rows, V)
        except RuntimeError:
            pass
        if to is None or (V > 1 and to.stride(1) != 1):
            _bad("process_logits: out's leading axes must collapse into one stride, its last be dense")
        same = to.data_ptr() == flat.data_ptr() and to.dtype == flat.dtype and to.stride() == flat.stride()
        _apart("process_logits", to, "out", None if same else flat, tokens, lengths, prompt_lengths, mask, mask_index, bias, *tensors)
    z = _ext().process_logits(flat, bias, tokens, lengths, prompt_lengths, mask, mask_index, *tensors, *scalars, to, grad)
    if out is not None:
        return out
    return z if logits.dim() == 2 else z.view(logits.shape)
