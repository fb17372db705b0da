"""The policy's own operators on either side of a rollout, over the engine's device layouts (include/contracts_policy.h).

The engine makes what a policy trains on — time-major trajectory planes with done flags (`engine.Trajectory`) — and takes what it
answers with — float scores, of which the step kernel takes the first maximum (`BatchedEnv.step_policy_device(.., "argmax")`).

* `linear_scan`: the gated linear recurrence along the time axis (a recurrent policy's memory, discounted returns), episodes ending
  inside the planes; differentiable; one step of it moves a sampler's state on.
* `advantages`: generalised advantage estimation over the planes of a (wrapped) ring.
* `process_logits`: penalties for repeated tokens, biases and masks on scores or logits, differentiable.

Tensors live on an MI355X (there is no CPU path) and a call is asynchronous on torch's current stream of their device; outputs
are new tensors unless `out=` names them (tensors that want no gradient), scratch memory comes from torch's allocator, nothing is kept between calls, and every call may
be captured into a graph (a backward pass together with its forward pass, and with leaves of its own: torch's engine ends the process where
a captured backward pass meets the nodes of an eager graph of the same leaves).  Ordering against other streams (env slices on side streams) is the caller's, as for the engine's steps.
A tensor whose last axis is not dense, or whose leading axes do not collapse into one stride, is copied first.
torch's tracers and transforms (jit.trace, fx, vmap, torch.func, fake tensors) are refused: calls are no operations of its dispatcher."""
import torch

from . import _lib

_loaded = None


def _ext():
    global _loaded
    if _loaded is None:
        _loaded = _lib.load_policy_torch()
    return _loaded


def linear_scan(x, gate, state=None, done=None, reverse=False, out=None, state_out=None):
    """The gated linear recurrence along the time axis: (y [T, E, C] in x's type, last [E, C] float32).

    Forward in time h_t = a_t h_{t-1} + x_t from h_{-1} = state, `last` = the state after step T - 1; with `reverse`
    h_t = a_t h_{t+1} + x_t from h_T = state, `last` = h_0.  done[t, e] says that an episode ended with step t: nothing crosses the border
    between t and t + 1, in either direction (going forward, `last` is 0 where done[T - 1]).  So `last` is the `state` of the next
    call: one of T = 1 moves a sampler's memory on, and a rollout may be scanned in pieces.  (A sampler that learns of done after the step clears
    the state of the rows that ended itself: state.masked_fill_(done[:, None] != 0, 0).)

    x: [T, E, C] float32, bfloat16 or float16 (float64 without gradients).  gate: [T, E, H] of x's type or float32, H
    dividing C (channel c is under gate c // (C // H)); strides of 0 share it along time or rows; or a float, one constant.  A gate
    of exactly 0 forgets the state whatever it held, as done does.  Gates over 1 are taken; their product over any stretch of steps without a
    border may not pass the state's range, for stretches are composed as maps h -> P h + H; one under that range takes nothing of a finite state,
    while an infinity or NaN shows until a border or a gate of 0, however small the gates.  state: [E, C] float32 (float64 with x).  done: [T, E] bool or uint8.
    The state is float32 throughout (float64 with x); y is rounded once.  Differentiable in x, gate and state (dy and dlast), from the
    unrounded states: one of every 16 is kept between the passes.  out / state_out: dense tensors to write to, without gradients;
    state_out may be `state`."""
    return (_loaded or _ext()).linear_scan(x, gate, state, done, reverse, out, state_out)


def advantages(reward, value, last_value=None, done=None, gamma=0.99, lam=0.95, first_plane=0, out=None):
    """Generalised advantage estimation over the planes of a rollout: (advantage, return), float32 [P, E, n] in the planes' order.

    delta_t = r_t + gamma V_{t+1} - V_t,  A_t = delta_t + gamma lam A_{t+1},  return_t = A_t + V_t; V_P = last_value (None: 0), and nothing crosses
    the border behind a step with done.  reward: [P, E, n] float64 (the engine's) or float32; value: [P, E, n] float32, bfloat16 or float16;
    last_value: [E, n] in value's type; done: [P, E] (the env's) or [P, E, n] (each agent's), bool or uint8.  Time t lies in plane
    (first_plane + t) % P, as a wrapped `Trajectory` holds it (its oldest plane is `traj.c.first_plane`).  Sums run in float64.
    out: a pair of dense float32 [P, E, n] tensors.  Not differentiable: targets are constants of a policy's loss."""
    return (_loaded or _ext()).advantages(reward, value, last_value, done, gamma, lam, first_plane, out)


def pack_mask(allowed):
    """bool or uint8 [..., V] (nonzero = allowed) -> the words of a packed mask, int32 [..., ceil(V / 32)]: bit v % 32 of word v // 32"""
    V = allowed.shape[-1]
    bits = torch.nn.functional.pad((allowed != 0).to(torch.int64), (0, -V % 32)).unflatten(-1, (-1, 32))
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def process_logits(logits, *, tokens=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, mask=None,
                   mask_index=None, out=None):
    """Scores or logits shaped ahead of a selection: penalties for repeated tokens (or past actions), biases, masks.

    logits: [..., V] float32, bfloat16 or float16; the leading axes are R rows (envs x agents, sequences), fewer than 2^24 in a call.  In this order, in float32, rounded once:
      tokens      [..., L] uint8, int32 or int64 of any strides (`actions.permute(1, 2, 0)` of [T, E, n] action planes), a row's history; only its first
                  `lengths` [...] count, the first `prompt_lengths` [...] of these are its prompt; ids outside [0, V) are passed over
      repetition  > 0: l / repetition where l > 0, else l * repetition, for a token seen anywhere in the history
      presence    taken off a token that occurs behind the prompt;  frequency: taken off as often as it occurs there.
                  Each of the three is a float or a float32 [...] tensor, one for each row; repetition lies between 2^-126 and 2^126 (a tensor's entries
                  are not checked), the others are finite
      bias        added: [V], the last axes of the logits ([n, V] for [E, n, V]), or [B, V] for logits [R, V] with B dividing R (row r takes
                  row r mod B); float32 or the logits' type
      mask        -inf where it forbids, whatever stands there; bool / uint8 [.., V] (nonzero = allowed), or int32 [.., ceil(V / 32)] words
                  (`pack_mask`); rows as for bias, or `mask_index` int32 [...] names a row's row of a [S, ..] table (the state of its
                  grammar; negative: all is allowed, past the end: nothing).  A row whose mask leaves nothing is -inf throughout
                  (`step_policy_device(.., "argmax")` then takes action 0).
    out: float32 or the logits' type, rows dense; it may be `logits` itself; not where gradients are wanted.
    Differentiable in logits and bias: gradients scale as l was, vanish where forbidden; bias gradients sum over rows in float32."""
    return (_loaded or _ext()).process_logits(logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias, mask, mask_index, out)
