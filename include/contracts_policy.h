/*
 * contracts_policy.h — C-ABI of the policy operators that stand on either side of a rollout (libcontracts_policy.so).
 *
 * The engine (contracts_engine.h) makes what a policy trains on and takes what it answers with.  These entry points are the
 * arithmetic in between that runs over the engine's own layouts on the device: the recurrence along the time axis of trajectory
 * planes (memories, discounted returns, advantages — with episodes that end inside the planes) and the shaping of scores
 * ahead of an arg-max (ce_step_policy, CE_POLICY_ARGMAX_F32).
 *
 * Conventions: as contracts_engine.h — plain pointers and sizes, 0 or a negative CE_E* code, no exceptions, no global state.
 * There is no handle: a call names its device, works on DEVICE pointers that the caller owns, and is asynchronous on `stream`
 * (hipStream_t, NULL = the device's null stream).  No call allocates, synchronises or keeps anything, so every call may be
 * captured into a hipGraph; a call that needs scratch memory says how much (ce_*_workspace), and two calls in flight at the
 * same time need a workspace each.  ce_policy_error() describes the last refusal of the calling thread.  All arguments are
 * checked on the host before anything is launched.  Strides are in elements.
 */
#ifndef CONTRACTS_POLICY_H
#define CONTRACTS_POLICY_H

#include <stdint.h>

#include "contracts_engine.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CE_POLICY_ABI_VERSION 1

enum ce_dtype { CE_F32 = 0, CE_BF16 = 1, CE_F16 = 2, CE_F64 = 3, CE_U8 = 4, CE_I32 = 5, CE_I64 = 6 };

int ce_policy_abi_version(void);
const char* ce_policy_error(void);

/* ---- the gated linear recurrence over time-major planes --------------------------------------------------------------------
 * x [T][E][C], gate [T][E][H] with H dividing C (channel c is under gate c / (C / H)), done [T][E], state [E][C]:
 *   forward in time:   h_t = a_t * k_t + x_t,  k_t = h_{t-1}, or 0 where done_{t-1};  k_0 = state;  last = h_{T-1}, or 0 where done_{T-1}
 *   CE_SCAN_REVERSE:   h_t = a_t * k_t + x_t,  k_t = h_{t+1}, or 0 where done_t;      k_{T-1} = state (0 where done_{T-1});  last = h_0
 * so that an episode that ends with step t hands nothing over the border between t and t + 1 in either direction, and cutting
 * the time axis into calls (`last` of one is `state` of the next) changes nothing.  A gate of exactly 0 forgets the
 * state whatever it held (infinities and NaN included), as done does.  The product of the gates over any stretch of steps without a
 * border may not pass the state's range (a stretch is composed as a map h -> P h + H); one under that range takes nothing of a finite
 * state, while an infinity or NaN shows until a border or a gate of 0, however small the gates.  The state is carried in float (double for CE_F64); each
 * y is rounded once to its own type and the rounded value is not used again.  T = 0 hands the state on.
 * Types: x and y dtype; gate dtype or CE_F32; state and last float (CE_F64: double throughout, and no backward pass).
 * gate == NULL: the constant `decay`, finite in the state's type.  state / done / last / saved may be NULL (zeros / none ended / not wanted).
 * `last` may be `state` itself (a state moved on in place; the time axis is then never split over blocks, however few); no other overlap of outputs with inputs.  x_row and gate_row are not
 * negative, and the rows that 256 channels span, min(E - 1, 255 / C + 1) of them (none where C is a
 * multiple of 256 and heads a power of two of channels), lie within 2^28 elements of each other. */
#define CE_SCAN_REVERSE 1u
#define CE_SCAN_SAVED_STEPS 16 /* saved: float [ceil(T / 16)][E][C], what ce_linear_scan_backward starts its tiles from */
#define CE_SCAN_SPLIT_STEPS 512 /* a call of fewer steps needs no workspace (its time axis is never split over blocks) */

typedef struct ce_scan {
  uint32_t abi_version; /* CE_POLICY_ABI_VERSION */
  int32_t device;
  uint32_t dtype, gate_dtype, flags, reserved;
  uint64_t steps, rows, channels, heads; /* T, E, C, H */
  int64_t x_step, x_row;       /* strides of x; channels lie next to each other                                       */
  int64_t gate_step, gate_row; /* strides of gate (0 = shared along that axis); heads lie next to each other           */
  int64_t done_step, done_row;
  double decay;
  const void* x;
  const void* gate;
  const uint8_t* done;
  const void* state; /* [E][C] dense */
  void* y;           /* [T][E][C] dense */
  void* last;        /* [E][C] dense */
  float* saved;
  void* workspace;
  uint64_t workspace_bytes;
} ce_scan;

int ce_linear_scan_workspace(const ce_scan* s, uint64_t* bytes);
int ce_linear_scan(const ce_scan* s, void* stream);

/* The gradients of y and last (dy [T][E][C] dense; dlast [E][C] dense, or NULL) taken back to x, gate and state.  `fwd` describes the
 * forward call: x, gate, done, strides, `saved` as it was filled (y, last and state are not read).
 *   g_t = dy_t + (the successor's a g, nothing over a border that done closes);  dx = g;  dgate = sum over a head's channels
 *   of g_t k_t;  dstate = a g of the first step
 * dx in dtype, dgate in gate_dtype ([T][E][H] dense, NULL with a constant gate), dstate float (or NULL).
 * Outputs overlap no input.  Sums run in float, in one fixed order: the same call gives the same bits. */
typedef struct ce_scan_grad {
  const void* dy;
  const void* dlast;
  void* dx;
  void* dgate;
  void* dstate;
} ce_scan_grad;

int ce_linear_scan_backward_workspace(const ce_scan* fwd, const ce_scan_grad* g, uint64_t* bytes);
int ce_linear_scan_backward(const ce_scan* fwd, const ce_scan_grad* g, void* stream);

/* ---- advantages and returns of a rollout (generalised advantage estimation) --------------------------------------------------
 *   delta_t = r_t + gamma V_{t+1} - V_t;  A_t = delta_t + gamma lam A_{t+1};  return_t = A_t + V_t;  V_T = last_value, A_T = 0;
 *   nothing crosses the border behind a step that ended the episode (done_t: V_{t+1} and A_{t+1} are not read).
 * reward [P][E][n] (CE_F64, the engine's, or CE_F32), value [P][E][n] (CE_F32 / CE_BF16 / CE_F16), last_value [E][n] in value's type,
 * done [P][E] or, with CE_ADV_DONE_PER_AGENT, [P][E][n]; advantage and return float [P][E][n].  All planes are a ring: time t
 * lies in plane (first_plane + t) % P, as ce_rollout_fused leaves a ce_traj behind.  Differences and sums run in double
 * and are rounded once.  advantage or ret may be NULL.  All arrays are dense; outputs overlap no input. */
#define CE_ADV_DONE_PER_AGENT 1u

typedef struct ce_advantage {
  uint32_t abi_version;
  int32_t device;
  uint32_t reward_dtype, value_dtype, flags, first_plane;
  uint64_t planes, rows, agents; /* P, E, n */
  double gamma, lam;
  const void* reward;
  const void* value;
  const void* last_value; /* NULL = zeros */
  const uint8_t* done;    /* NULL = none ended */
  float* advantage;
  float* ret;
} ce_advantage;

int ce_advantages(const ce_advantage* a, void* stream);

/* ---- scores shaped ahead of a selection: penalties for repeated tokens, biases, masks ----------------------------------------
 * For row r and token v, with `seen` = v occurs in the row's history and `count` = how often it occurs behind its prompt:
 *   z = l;  seen: z = l > 0 ? l / repetition : l * repetition;  count > 0: z -= presence;  z -= frequency * count;  z += bias;
 *   a token that the mask forbids: -inf, whatever l and bias hold (a row whose mask leaves nothing is -inf throughout)
 * Arithmetic in float, one rounding to the output's type.  Fewer than 2^24 rows, at most 2^28 tokens, histories shorter than 2^31.
 * History: tokens (CE_U8 / CE_I32 / CE_I64) at tokens[r * token_row + i * token_step], i < min(lengths[r], L) (lengths NULL: L;
 * a negative length counts as 0); those with i < prompt_lengths[r] (NULL: none) are the prompt.  A token outside [0, V) is
 * passed over.  repetition / presence / frequency: one float a row, or NULL with the scalar of that name (a finite float).  repetition lies between
 * 2^-126 and 2^126; a row's is not checked.
 * bias: [bias_rows][V] dense, float or the logits' type; row r takes row r mod bias_rows (bias_rows divides R).
 * mask: CE_U8 [mask_rows][V], nonzero = allowed, or CE_I32 [mask_rows][ceil(V / 32)], bit v % 32 of word v / 32.  Row r takes
 * row mask_index[r] — negative: everything is allowed; past the end: nothing is — or, without an index, row r mod mask_rows.
 * out: logits' type or CE_F32, [R][V] with row stride out_row (rows do not overlap); it may be `logits` itself (same type and stride). */
typedef struct ce_logits {
  uint32_t abi_version;
  int32_t device;
  uint32_t dtype, out_dtype, token_dtype, bias_dtype, mask_dtype, reserved;
  uint64_t rows, vocab, history; /* R, V, L */
  int64_t logits_row, out_row, token_row, token_step;
  uint64_t bias_rows, mask_rows;
  double repetition_all, presence_all, frequency_all;
  const void* logits;
  const void* tokens; /* NULL: no history, no penalties */
  const int32_t* lengths;
  const int32_t* prompt_lengths;
  const float* repetition;
  const float* presence;
  const float* frequency;
  const void* bias;
  const void* mask;
  const int32_t* mask_index;
  void* out;
  void* workspace; /* ce_process_logits_backward with dbias only */
  uint64_t workspace_bytes;
} ce_logits;

int ce_process_logits(const ce_logits* s, void* stream);

/* Gradient of the output (dout, in out_dtype, row stride dout_row) taken back: dlogits (logits' type, [R][V] dense) = dout scaled as l was, 0
 * where forbidden; dbias (bias_dtype, [bias_rows][V] dense) = the sum over the rows that share a bias row, in float and in one fixed order.
 * Either may be NULL.  dlogits overlaps neither dout nor the logits.  fwd->out is not read. */
typedef struct ce_logits_grad {
  const void* dout;
  int64_t dout_row;
  void* dlogits;
  void* dbias;
} ce_logits_grad;

int ce_process_logits_backward_workspace(const ce_logits* fwd, const ce_logits_grad* g, uint64_t* bytes);
int ce_process_logits_backward(const ce_logits* fwd, const ce_logits_grad* g, void* stream);

#ifdef __cplusplus
}
#endif
#endif
