// cp_api.hip — host side of the C-ABI in include/contracts_policy.h: checks every argument before anything is launched, names
// the launch's shape, never throws, never allocates and never synchronises.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "cp_common.h"

namespace {

thread_local char g_error[256] = "";

int refuse(const char* what, ...) {
  va_list ap;
  va_start(ap, what);
  vsnprintf(g_error, sizeof(g_error), what, ap);
  va_end(ap);
  return CE_EINVAL;
}

// The call's device while it is made; the caller's own is current again afterwards.  The thread's error state starts clean: what an earlier call of
// another library left there must not be blamed on the launches that follow.
struct OnDevice {
  int before = -1;
  hipError_t err;
  explicit OnDevice(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) err = hipSetDevice(device);
    else if (err == hipSuccess) before = -1;
    (void)hipGetLastError();
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

int launched(hipError_t e, const char* what) {
  if (e == hipSuccess) return CE_OK;
  snprintf(g_error, sizeof(g_error), "%s: %s", what, hipGetErrorString(e));
  return CE_ENODEV;
}

uint64_t size_of(uint32_t t) { return t == CE_U8 ? 1 : t == CE_BF16 || t == CE_F16 ? 2 : t == CE_F32 || t == CE_I32 ? 4 : 8; }
bool half_or_float(uint32_t t) { return t == CE_F32 || t == CE_BF16 || t == CE_F16; }
bool finite_float(double v) { return std::isfinite((float)v); }  // as the kernels hold it
bool aligned(const void* p, uint64_t to) { return (uintptr_t)p % to == 0; }

constexpr uint64_t kMost = 1ull << 28;   // columns of a scan: a launch has fewer than 2^32 threads
constexpr uint64_t kMostRows = (1ull << 24) - 1;  // rows of scores: short ones are packed, 8 and more to a block; long ones go in parts
constexpr uint64_t kFar = 1ull << 46;    // elements: products of sizes stay far inside 64 bits

// ---- the scan ---------------------------------------------------------------------------------------------------------------------
struct Plan {
  cp::ScanParams p;
  int mode, vec;
};

bool divides(int64_t vec, std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s % vec) return false;
  return true;
}

int check_scan(const ce_scan* s) {
  if (!s) return refuse("null ce_scan");
  if (s->abi_version != CE_POLICY_ABI_VERSION) return refuse("ce_scan.abi_version is %u, this library is %d", s->abi_version, CE_POLICY_ABI_VERSION);
  if (!half_or_float(s->dtype) && s->dtype != CE_F64) return refuse("linear_scan: x must be float, bfloat16, half or double");
  if (s->gate && s->gate_dtype != s->dtype && !(s->gate_dtype == CE_F32 && half_or_float(s->dtype)))
    return refuse("linear_scan: the gate must be of x's type or float");
  if (s->flags & ~CE_SCAN_REVERSE) return refuse("linear_scan: unknown flags %#x", s->flags);
  if (s->channels && s->gate && (s->heads == 0 || s->heads > s->channels || s->channels % s->heads)) return refuse("linear_scan: heads must divide channels");
  if (s->channels > kMost || s->rows > kMost || s->rows * s->channels > kMost) return refuse("linear_scan: more than 2^28 columns (rows x channels)");
  if (s->steps > kFar || (s->steps && s->rows * s->channels > kFar / s->steps)) return refuse("linear_scan: too many elements");
  if (s->rows * s->channels == 0) return CE_OK;
  if (s->steps && (!s->x || !s->y)) return refuse("linear_scan: null x or y");
  if (!s->gate && !(s->dtype == CE_F64 ? std::isfinite(s->decay) : finite_float(s->decay))) return refuse("linear_scan: decay must be finite in the state's type");
  const uint64_t b = size_of(s->dtype), a = s->dtype == CE_F64 ? 8 : 4;
  if (!aligned(s->x, b) || !aligned(s->y, b) || !aligned(s->state, a) || !aligned(s->last, a) || !aligned(s->saved, 4) || (s->gate && !aligned(s->gate, size_of(s->gate_dtype))))
    return refuse("linear_scan: a pointer is not aligned to its type");
  // a wave's lanes reach each other by 32-bit offsets: rows that far apart exist only where short rows are very long in time
  // (none where rows are whole waves: multiples of 256 channels, heads a power of two)
  const uint64_t head = s->gate ? s->channels / s->heads : 1;
  const bool whole = s->channels % 256 == 0 && (head & (head - 1)) == 0;
  const int64_t span = whole ? 0 : std::min<int64_t>((int64_t)s->rows - 1, 255 / (int64_t)s->channels + 1), reach = (int64_t)kMost;
  for (int64_t row : {s->x_row, s->gate ? s->gate_row : 0})
    if (row < 0 || (span && row >= reach / span)) return refuse("linear_scan: rows lie too far apart for a wave; lay x and gate out time-major");
  return CE_OK;
}

// Lanes, waves and chunks: what the columns leave of the chip is filled along the time axis.  Measured (us, fwd or bwd, done in 2 % of steps):
//  * 2048 waves of columns and more: a wave takes its columns' whole time axis, 8 bytes to a lane.  [128, 4096, 128] bfloat16 75 (floor 75).
//  * else the waves of a block share the time axis (a second walk in registers), 8 of them, and lanes take fewer channels as long as that
//    makes waves: [512, 256, 256] bfloat16 36 with 2 channels a lane, 43 with 4, 40 with 4 waves; the gradients' longer walks do better with 4
//    waves where 2048 can be had: 75 against 82.
//  * under 1536 waves that way, the time axis is cut into chunks too, which costs reading x and the gate twice, at least a tile each, up
//    to 4096 waves in all, in whole tiles: [65537, 1, 1024] bfloat16, 16 heads: 77 with 103 chunks (of 640 steps: 128 chunks would be of 513) and 4 channels a
//    lane, 168 with 16 chunks and 1 channel;
//    [1000, 37, 360] float keeps whole at 1672 waves: 31 against 36.  Gradients: [1000, 37, 360] float, 9 heads: 54 with 8 chunks of pairs of
//    channels, 60 whole with one; [1000, 64, 256] float 71 whole with one (2048 waves), 81 in chunks.
//  * a state moved on in place keeps the time axis whole (`split` is false), with the lanes and waves that suit that: its chunks would read the incoming
//    state while the last of them writes the outgoing one.
void share(cp::ScanParams& p, int* vec, bool grad, bool halves, bool split, uint64_t columns, uint64_t (*blocks)(const cp::ScanParams&, uint64_t columns, int vec)) {
  p.chunks = p.waves = 1;
  if (p.T <= CE_SCAN_SAVED_STEPS) return;
  const int widest = *vec;
  if (blocks(p, columns, widest) >= 2048) return;
  p.waves = p.T <= 4 * CE_SCAN_SAVED_STEPS || (grad && blocks(p, columns, widest) * 4 >= 2048) ? 4 : 8;
  if (grad) {
    if (!halves && *vec > 1 && blocks(p, columns, *vec) * p.waves < 1536 && columns / 64 * p.waves >= 2048) *vec = 1;
  } else {
    while (*vec > 1 && blocks(p, columns, *vec) * p.waves < 4096) *vec /= 2;
  }
  if (blocks(p, columns, *vec) * p.waves >= 1536 || p.T < CE_SCAN_SPLIT_STEPS || !split) return;
  *vec = widest;
  if (grad) p.waves = 4;
  const uint64_t have = blocks(p, columns, widest) * p.waves, tile = p.waves * CE_SCAN_SAVED_STEPS;
  const uint64_t want = std::min<uint64_t>((4096 + have - 1) / have, 128), each = ((p.T + want - 1) / want + tile - 1) / tile * tile;
  p.chunk = each;
  p.chunks = (uint32_t)((p.T + each - 1) / each);
}

// Waves side by side that a scan's columns make (with a head's gradient to add up, heads keep to a wave, or take several).
uint64_t flat_waves(const cp::ScanParams&, uint64_t columns, int vec) { return (columns / vec + 63) / 64; }
uint64_t head_waves(const cp::ScanParams& p, uint64_t columns, int vec) {
  const uint64_t lanes = p.head / vec, groups = columns / p.head;
  return lanes > 64 ? groups * ((lanes + 63) / 64) : (groups + 64 / lanes - 1) / (64 / lanes);
}

void plan_scan(const ce_scan* s, const ce_scan_grad* g, Plan* o) {
  cp::ScanParams& p = o->p;
  p = cp::ScanParams();
  const uint64_t T = s->steps, E = s->rows, C = s->channels, H = s->gate ? s->heads : C;
  o->mode = !s->gate ? cp::kGateConst : H == C ? cp::kGateChannel : cp::kGateHead;
  const uint64_t head = C / H, b = size_of(s->dtype), gb = size_of(s->gate_dtype);
  // 8 bytes of neighbouring channels to a lane, or less where the arrays' alignment or strides do not allow it
  auto fits = [&](int64_t v) {
    bool ok = (int64_t)C % v == 0 && divides(v, {s->x_step, s->x_row}) && aligned(s->x, v * b);
    if (o->mode == cp::kGateChannel) ok = ok && divides(v, {s->gate_step, s->gate_row}) && aligned(s->gate, v * gb);
    if (o->mode == cp::kGateHead) ok = ok && (int64_t)head % v == 0;
    if (!g) return ok && aligned(s->y, v * b);
    return ok && aligned(g->dy, v * b) && aligned(g->dx, v * b) && (o->mode != cp::kGateChannel || aligned(g->dgate, v * gb));
  };
  int vec = b == 8 ? 1 : (int)(8 / b);
  if (g) vec = std::min(vec, 2);
  while (vec > 1 && !fits(vec)) vec /= 2;
  p.T = T;
  p.head = (uint32_t)head;
  const bool sums = g && o->mode == cp::kGateHead;
  share(p, &vec, g != nullptr, b == 2, g || !s->last || s->last != s->state, E * C, sums ? head_waves : flat_waves);
  o->vec = vec;
  const bool rev = s->flags & CE_SCAN_REVERSE;
  const int64_t sign = rev ? -1 : 1, off = rev && T ? (int64_t)T - 1 : 0;
  p.cols = (uint32_t)(E * C / vec);
  p.row_cols = (uint32_t)(C / vec);
  p.heads = (uint32_t)H;
  p.rows = (uint32_t)E;
  p.cut_off = rev ? 0 : -1;
  p.x_step = sign * s->x_step;
  p.x_row = s->x_row;
  p.gate_step = sign * s->gate_step;
  p.gate_row = s->gate_row;
  p.done_step = sign * s->done_step;
  p.done_row = s->done_row;
  p.y_step = sign * (int64_t)(E * C);
  p.dgate_step = sign * (int64_t)(E * H);
  p.decay = s->decay;
  auto from = [&](const void* q, int64_t step, uint64_t bytes) -> char* { return q ? (char*)q + off * step * (int64_t)bytes : nullptr; };
  p.x = from(s->x, s->x_step, b);
  p.gate = from(s->gate, s->gate_step, gb);
  p.done = (const uint8_t*)from(s->done, s->done_step, 1);
  p.state = s->state;
  p.y = from(s->y, (int64_t)(E * C), b);
  p.last = s->last;
  p.saved = s->saved;
  p.slabs = 1;
  if (g) {
    p.dy = from(g->dy, (int64_t)(E * C), b);
    p.dlast = g->dlast;
    p.dx = from(g->dx, (int64_t)(E * C), b);
    p.dgate = from(g->dgate, (int64_t)(E * H), gb);
    p.dstate = g->dstate;
    if (sums) {
      p.lanes = (uint32_t)(head / vec);
      p.in_wave = p.lanes <= 64 ? 64 / p.lanes : 0;
      p.slabs = p.in_wave ? 1 : (p.lanes + 63) / 64;
    }
  }
  const uint32_t spanned = 62 / p.row_cols + 2;  // rows that 64 lanes can touch
  p.flags = !s->done ? cp::kFlagsNone : spanned <= 4 ? cp::kFlags4 : spanned <= 16 ? cp::kFlags16 : cp::kFlagsLane;
  if (p.chunks == 1) p.chunk = T;
}

uint64_t part_bytes(const Plan& o, uint32_t dtype) {
  return o.p.chunks > 1 ? (uint64_t)(o.p.chunks - 1) * 2 * o.p.cols * o.vec * (dtype == CE_F64 ? 8 : 4) : 0;
}
uint64_t slab_bytes(const Plan& o, const ce_scan* s, const ce_scan_grad* g) {
  return s->gate && o.p.slabs > 1 ? (uint64_t)o.p.slabs * s->steps * s->rows * s->heads * 4 : 0;
}

}  // namespace

extern "C" int ce_policy_abi_version(void) { return CE_POLICY_ABI_VERSION; }
extern "C" const char* ce_policy_error(void) { return g_error; }

extern "C" int ce_linear_scan_workspace(const ce_scan* s, uint64_t* bytes) {
  if (!bytes) return refuse("null bytes");
  if (int rc = check_scan(s)) return rc;
  *bytes = 0;
  if (s->rows * s->channels == 0) return CE_OK;
  Plan o;
  plan_scan(s, nullptr, &o);
  *bytes = part_bytes(o, s->dtype);
  return CE_OK;
}

extern "C" int ce_linear_scan(const ce_scan* s, void* stream) {
  if (int rc = check_scan(s)) return rc;
  if (s->saved && s->dtype == CE_F64) return refuse("linear_scan: double has no backward pass");
  if (s->rows * s->channels == 0 || (s->steps == 0 && !s->last)) return CE_OK;
  Plan o;
  plan_scan(s, nullptr, &o);
  const uint64_t need = part_bytes(o, s->dtype);
  if (need && (!s->workspace || s->workspace_bytes < need || !aligned(s->workspace, 8)))
    return refuse("linear_scan: workspace of %llu bytes needed, %llu given", (unsigned long long)need, (unsigned long long)(s->workspace ? s->workspace_bytes : 0));
  o.p.part = s->workspace;
  OnDevice dev(s->device);
  if (dev.err != hipSuccess) return launched(dev.err, "linear_scan: device");
  return launched(cp::launch_scan(o.p, s->dtype, s->gate ? s->gate_dtype : s->dtype, o.mode, o.vec, (hipStream_t)stream), "linear_scan");
}

static int check_scan_grad(const ce_scan* s, const ce_scan_grad* g) {
  if (!g) return refuse("null ce_scan_grad");
  if (!s) return refuse("null ce_scan");
  ce_scan t = *s;
  t.y = const_cast<void*>(t.x);  // the backward pass reads no y
  if (int rc = check_scan(&t)) return rc;
  if (s->dtype == CE_F64) return refuse("linear_scan: double has no backward pass");
  if (s->rows * s->channels == 0) return CE_OK;
  if (s->steps && !s->saved) return refuse("linear_scan_backward: the forward call's saved states are missing");
  if (s->steps && (!g->dy || !g->dx || (s->gate && !g->dgate))) return refuse("linear_scan_backward: null dy, dx or dgate");
  const uint64_t b = size_of(s->dtype);
  if (!aligned(g->dy, b) || !aligned(g->dx, b) || !aligned(g->dlast, 4) || !aligned(g->dstate, 4) || (s->gate && !aligned(g->dgate, size_of(s->gate_dtype))))
    return refuse("linear_scan_backward: a pointer is not aligned to its type");
  if (g->dgate && !s->gate) return refuse("linear_scan_backward: a constant gate has no gradient");
  return CE_OK;
}

extern "C" int ce_linear_scan_backward_workspace(const ce_scan* s, const ce_scan_grad* g, uint64_t* bytes) {
  if (!bytes) return refuse("null bytes");
  if (int rc = check_scan_grad(s, g)) return rc;
  *bytes = 0;
  if (s->rows * s->channels == 0) return CE_OK;
  Plan o;
  plan_scan(s, g, &o);
  *bytes = part_bytes(o, s->dtype) + slab_bytes(o, s, g);
  return CE_OK;
}

extern "C" int ce_linear_scan_backward(const ce_scan* s, const ce_scan_grad* g, void* stream) {
  if (int rc = check_scan_grad(s, g)) return rc;
  if (s->rows * s->channels == 0) return CE_OK;
  Plan o;
  plan_scan(s, g, &o);
  const uint64_t part = part_bytes(o, s->dtype), need = part + slab_bytes(o, s, g);
  if (need && (!s->workspace || s->workspace_bytes < need || !aligned(s->workspace, 8)))
    return refuse("linear_scan_backward: workspace of %llu bytes needed, %llu given", (unsigned long long)need, (unsigned long long)(s->workspace ? s->workspace_bytes : 0));
  o.p.part = s->workspace;
  o.p.slab = s->workspace ? (float*)((char*)s->workspace + part) : nullptr;
  OnDevice dev(s->device);
  if (dev.err != hipSuccess) return launched(dev.err, "linear_scan_backward: device");
  return launched(cp::launch_scan_grad(o.p, s->dtype, s->gate ? s->gate_dtype : s->dtype, o.mode, o.vec, (hipStream_t)stream), "linear_scan_backward");
}

// ---- advantages -------------------------------------------------------------------------------------------------------------------
extern "C" int ce_advantages(const ce_advantage* a, void* stream) {
  if (!a) return refuse("null ce_advantage");
  if (a->abi_version != CE_POLICY_ABI_VERSION) return refuse("ce_advantage.abi_version is %u, this library is %d", a->abi_version, CE_POLICY_ABI_VERSION);
  if (a->reward_dtype != CE_F64 && a->reward_dtype != CE_F32) return refuse("advantages: reward must be double or float");
  if (!half_or_float(a->value_dtype)) return refuse("advantages: value must be float, bfloat16 or half");
  if (a->flags & ~CE_ADV_DONE_PER_AGENT) return refuse("advantages: unknown flags %#x", a->flags);
  if (!std::isfinite(a->gamma) || !std::isfinite(a->lam) || !std::isfinite(a->gamma * a->lam)) return refuse("advantages: gamma, lam and their product must be finite");
  if (a->rows > kMost || a->agents > kMost || a->rows * a->agents > kMost) return refuse("advantages: more than 2^28 columns (rows x agents)");
  if (a->planes > kFar || (a->planes && a->rows * a->agents > kFar / a->planes)) return refuse("advantages: too many elements");
  if (a->planes * a->rows * a->agents == 0) return CE_OK;
  if (a->first_plane >= a->planes) return refuse("advantages: first_plane out of range");
  if (!a->reward || !a->value || (!a->advantage && !a->ret)) return refuse("advantages: null reward, value or outputs");
  if (!aligned(a->reward, size_of(a->reward_dtype)) || !aligned(a->value, size_of(a->value_dtype)) || !aligned(a->last_value, size_of(a->value_dtype)) ||
      !aligned(a->advantage, 4) || !aligned(a->ret, 4))
    return refuse("advantages: a pointer is not aligned to its type");
  OnDevice dev(a->device);
  if (dev.err != hipSuccess) return launched(dev.err, "advantages: device");
  return launched(cp::launch_advantages(*a, (hipStream_t)stream), "advantages");
}

// ---- scores -----------------------------------------------------------------------------------------------------------------------
static int check_logits(const ce_logits* s) {
  if (!s) return refuse("null ce_logits");
  if (s->abi_version != CE_POLICY_ABI_VERSION) return refuse("ce_logits.abi_version is %u, this library is %d", s->abi_version, CE_POLICY_ABI_VERSION);
  if (!half_or_float(s->dtype)) return refuse("process_logits: logits must be float, bfloat16 or half");
  if (s->out_dtype != s->dtype && s->out_dtype != CE_F32) return refuse("process_logits: the output must be of the logits' type or float");
  if (s->rows > kMostRows) return refuse("process_logits: 2^24 rows or more");
  if (s->vocab > (1ull << 28)) return refuse("process_logits: more than 2^28 tokens");
  if (s->history > (1ull << 31) - 1) return refuse("process_logits: a history of more than 2^31 - 1 tokens");
  if (s->rows * s->vocab == 0) return CE_OK;
  if (!s->logits) return refuse("process_logits: null logits");
  if (!aligned(s->logits, size_of(s->dtype)) || !aligned(s->out, size_of(s->out_dtype))) return refuse("process_logits: a pointer is not aligned to its type");
  if (s->tokens) {
    if (s->token_dtype != CE_U8 && s->token_dtype != CE_I32 && s->token_dtype != CE_I64) return refuse("process_logits: tokens must be uint8, int32 or int64");
    if (!aligned(s->tokens, size_of(s->token_dtype))) return refuse("process_logits: tokens are not aligned to their type");
    // the kernels take the reciprocal too: both are to be normal floats
    if (!s->repetition && !(s->repetition_all >= 0x1p-126 && s->repetition_all <= 0x1p126)) return refuse("process_logits: repetition must be positive, from 2^-126 to 2^126");
    if ((!s->presence && !finite_float(s->presence_all)) || (!s->frequency && !finite_float(s->frequency_all))) return refuse("process_logits: presence and frequency must be finite floats");
  } else if (s->lengths || s->prompt_lengths) {
    return refuse("process_logits: lengths without tokens");
  }
  if (s->bias) {
    if (s->bias_dtype != CE_F32 && s->bias_dtype != s->dtype) return refuse("process_logits: bias must be float or of the logits' type");
    if (!aligned(s->bias, size_of(s->bias_dtype))) return refuse("process_logits: bias is not aligned to its type");
    if (s->bias_rows == 0 || s->rows % s->bias_rows) return refuse("process_logits: bias_rows must divide the rows");
  }
  if (s->mask) {
    if (s->mask_dtype != CE_U8 && s->mask_dtype != CE_I32) return refuse("process_logits: a mask is uint8 tokens or int32 words");
    if (!aligned(s->mask, size_of(s->mask_dtype))) return refuse("process_logits: the mask is not aligned to its type");
    if (s->mask_rows == 0 || s->mask_rows > 0x7fffffffu || (!s->mask_index && s->rows % s->mask_rows)) return refuse("process_logits: mask_rows must divide the rows, or an index be given");
  } else if (s->mask_index) {
    return refuse("process_logits: mask_index without a mask");
  }
  return CE_OK;
}

extern "C" int ce_process_logits(const ce_logits* s, void* stream) {
  if (int rc = check_logits(s)) return rc;
  if (s->rows * s->vocab == 0) return CE_OK;
  if (!s->out) return refuse("process_logits: null output");
  if (s->rows > 1 && s->out_row < (int64_t)s->vocab && s->out_row > -(int64_t)s->vocab) return refuse("process_logits: the output's rows overlap");
  if (s->out == s->logits && (s->out_dtype != s->dtype || s->out_row != s->logits_row)) return refuse("process_logits: in place needs one type and one stride");
  OnDevice dev(s->device);
  if (dev.err != hipSuccess) return launched(dev.err, "process_logits: device");
  return launched(cp::launch_logits(*s, (hipStream_t)stream), "process_logits");
}

struct Reach {
  uintptr_t lo, hi;  // the bytes of [rows][width] elements, rows `row` elements apart
  bool meets(const Reach& o) const { return lo < o.hi && o.lo < hi; }
};
static Reach reach(const void* p, uint64_t rows, int64_t row, uint64_t width, uint64_t size) {
  const int64_t last = (int64_t)(rows - 1) * row, lo = std::min<int64_t>(last, 0), hi = std::max<int64_t>(last, 0) + (int64_t)width;
  return {(uintptr_t)p + (uintptr_t)(lo * (int64_t)size), (uintptr_t)p + (uintptr_t)(hi * (int64_t)size)};
}

static int check_logits_grad(const ce_logits* s, const ce_logits_grad* g) {
  if (!g) return refuse("null ce_logits_grad");
  if (int rc = check_logits(s)) return rc;
  if (s->rows * s->vocab == 0) return CE_OK;
  if (!g->dout) return refuse("process_logits_backward: null dout");
  if (g->dbias && !s->bias) return refuse("process_logits_backward: dbias without a bias");
  if (!aligned(g->dout, size_of(s->out_dtype)) || !aligned(g->dlogits, size_of(s->dtype)) || (g->dbias && !aligned(g->dbias, size_of(s->bias_dtype))))
    return refuse("process_logits_backward: a pointer is not aligned to its type");
  // the repeats' launch reads both again where the walk has written dlogits
  const Reach dl = reach(g->dlogits, s->rows, (int64_t)s->vocab, s->vocab, size_of(s->dtype));
  if (g->dlogits && (dl.meets(reach(g->dout, s->rows, g->dout_row, s->vocab, size_of(s->out_dtype))) || dl.meets(reach(s->logits, s->rows, s->logits_row, s->vocab, size_of(s->dtype)))))
    return refuse("process_logits_backward: dlogits overlaps dout or the logits");
  return CE_OK;
}

extern "C" int ce_process_logits_backward_workspace(const ce_logits* s, const ce_logits_grad* g, uint64_t* bytes) {
  if (!bytes) return refuse("null bytes");
  if (int rc = check_logits_grad(s, g)) return rc;
  *bytes = s->rows * s->vocab ? cp::logits_grad_workspace(*s, *g) : 0;
  return CE_OK;
}

extern "C" int ce_process_logits_backward(const ce_logits* s, const ce_logits_grad* g, void* stream) {
  if (int rc = check_logits_grad(s, g)) return rc;
  if (s->rows * s->vocab == 0 || (!g->dlogits && !g->dbias)) return CE_OK;
  const uint64_t need = cp::logits_grad_workspace(*s, *g);
  if (need && (!s->workspace || s->workspace_bytes < need || !aligned(s->workspace, 4)))
    return refuse("process_logits_backward: workspace of %llu bytes needed, %llu given", (unsigned long long)need, (unsigned long long)(s->workspace ? s->workspace_bytes : 0));
  OnDevice dev(s->device);
  if (dev.err != hipSuccess) return launched(dev.err, "process_logits_backward: device");
  return launched(cp::launch_logits_grad(*s, *g, (hipStream_t)stream), "process_logits_backward");
}
