// cp_logits.hip — scores shaped ahead of a selection (ce_process_logits): penalties for repeated tokens, biases, masks; and the
// gradients of logits and bias.
//
// A block takes a tile of kTile scores: a run of one row's vocabulary, or a whole number of short rows.  A table in LDS counts what the
// tile's histories hold (the prompt's tokens only as "seen", the top bit), then the tile streams through once, 8 neighbouring
// scores to a lane: read, penalise, bias, mask, write.  Bound by HBM: each score is read once and written once; a history is
// read once for every run of its row's vocabulary, from L2.
#include "cp_common.h"

namespace cp {

constexpr int kBlock = 256, kTile = 4096, kLane = 8;
constexpr uint32_t kSeen = 0x80000000u;  // of a 32-bit table entry
constexpr uint32_t kRowsMost = 512;  // short rows of a tile (their parameters lie in LDS too)

struct Row {  // what a row is penalised with
  float repetition, inverse, presence, frequency;
};
__device__ __forceinline__ Row row_of(const ce_logits& s, uint64_t r) {
  Row o;
  o.repetition = s.repetition ? s.repetition[r] : (float)s.repetition_all;
  o.inverse = 1.f / o.repetition;
  o.presence = s.presence ? s.presence[r] : (float)s.presence_all;
  o.frequency = s.frequency ? s.frequency[r] : (float)s.frequency_all;
  return o;
}
// How much of row r's history counts, and how much of that is its prompt.
__device__ __forceinline__ uint32_t used_of(const ce_logits& s, uint64_t r) {
  if (!s.tokens) return 0;
  if (!s.lengths) return (uint32_t)s.history;
  const int32_t l = s.lengths[r];
  return l < 0 ? 0u : (uint32_t)l < (uint32_t)s.history ? (uint32_t)l : (uint32_t)s.history;
}
__device__ __forceinline__ uint32_t prompt_of(const ce_logits& s, uint64_t r) {
  if (!s.prompt_lengths) return 0;
  const int32_t l = s.prompt_lengths[r];
  return l > 0 ? (uint32_t)l : 0u;
}
// kTokens places of a history at a time, all read before the first is looked at: i, i + stride, .. below end.
constexpr int kTokens = 8;
template <class K, class F> __device__ __forceinline__ void each_token(const ce_logits& s, uint64_t r, uint32_t from, uint32_t stride, uint32_t end, F&& f) {
  const K* p = (const K*)s.tokens + (int64_t)r * s.token_row;
  for (uint32_t i = from; i < end; i += kTokens * stride) {
    K t[kTokens];
#pragma unroll
    for (int u = 0; u < kTokens; ++u) t[u] = i + u * stride < end ? p[(int64_t)(i + u * stride) * s.token_step] : K(0);
#pragma unroll
    for (int u = 0; u < kTokens; ++u)
      if (i + u * stride < end) f(t[u], i + u * stride);
  }
}
// Where token t lies in a run of n from v0 on; n or more where it does not.
__device__ __forceinline__ uint32_t place(uint8_t t, uint32_t v0, uint32_t) { return (uint32_t)t - v0; }
__device__ __forceinline__ uint32_t place(int32_t t, uint32_t v0, uint32_t) { return (uint32_t)t - v0; }
__device__ __forceinline__ uint32_t place(int64_t t, uint32_t v0, uint32_t n) { return (uint64_t)t - v0 < n ? (uint32_t)((uint64_t)t - v0) : n; }
__device__ __forceinline__ int32_t indexed(const ce_logits& s, int32_t m) { return m < 0 ? -1 : (uint64_t)m < s.mask_rows ? m : -2; }
// The mask's row of row r: -1 = everything is allowed, -2 = nothing is.
__device__ __forceinline__ int32_t mask_row(const ce_logits& s, uint64_t r) {
  if (!s.mask) return -1;
  if (!s.mask_index) return s.mask_rows == s.rows ? (int32_t)r : (int32_t)((uint32_t)r % (uint32_t)s.mask_rows);
  return indexed(s, s.mask_index[r]);
}
__device__ __forceinline__ int32_t mask_row(const ce_logits& s, uint64_t r, int32_t index) {  // its index already read
  return s.mask_index ? indexed(s, index) : mask_row(s, r);
}
__device__ __forceinline__ bool allowed(const ce_logits& s, int32_t m, uint32_t v) {
  if (m < 0) return m == -1;
  if (s.mask_dtype == CE_U8) return ((const uint8_t*)s.mask)[(uint64_t)m * s.vocab + v] != 0;
  return (((const uint32_t*)s.mask)[(uint64_t)m * ((s.vocab + 31) / 32) + v / 32] >> (v % 32)) & 1u;
}
// 8 neighbouring tokens' permissions as bits; all 8 lie inside the row.
__device__ __forceinline__ uint32_t allowed8(const ce_logits& s, int32_t m, uint32_t v) {
  if (m < 0) return m == -1 ? 0xffu : 0u;
  if (s.mask_dtype == CE_U8) {
    uint64_t b;
    __builtin_memcpy(&b, (const uint8_t*)s.mask + (uint64_t)m * s.vocab + v, 8);
    uint32_t bits = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) bits |= ((b >> (8 * q)) & 0xff ? 1u : 0u) << q;
    return bits;
  }
  const uint32_t* words = (const uint32_t*)s.mask + (uint64_t)m * ((s.vocab + 31) / 32);
  uint32_t bits = words[v / 32] >> (v % 32);
  if (v % 32 > 24) bits |= words[v / 32 + 1] << (32 - v % 32);  // the 8 tokens reach into the next word, which the row has
  return bits & 0xffu;
}
// 8 neighbouring elements of any alignment as float.
template <class T> __device__ __forceinline__ void load8(const T* p, float (&o)[8]) {
  T t[8];
  __builtin_memcpy(t, __builtin_assume_aligned(p, alignof(T)), sizeof(t));
#pragma unroll
  for (int q = 0; q < 8; ++q) o[q] = (float)t[q];
}
template <class T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) t[q] = (T)v[q];
  __builtin_memcpy(__builtin_assume_aligned(p, alignof(T)), t, sizeof(t));
}
__device__ __forceinline__ float bias_at(const ce_logits& s, uint64_t at) {
  if (s.bias_dtype == CE_F32) return ((const float*)s.bias)[at];
  if (s.bias_dtype == CE_BF16) return (float)((const bf16*)s.bias)[at];
  return (float)((const f16*)s.bias)[at];
}
__device__ __forceinline__ void bias8(const ce_logits& s, uint64_t at, float (&o)[8]) {
  if (s.bias_dtype == CE_F32) load8((const float*)s.bias + at, o);
  else if (s.bias_dtype == CE_BF16) load8((const bf16*)s.bias + at, o);
  else load8((const f16*)s.bias + at, o);
}
// One score under its table entry, without branches: 11 operations a score, and every lane of a wave runs them where one lane has an
// entry, so a division (some 12 more) would cost as much as the reads: l / repetition is l times its reciprocal, half a step more off.
__device__ __forceinline__ float penalise(float l, uint32_t entry, const Row& row) {
  const float count = (float)(entry & ~kSeen), scaled = l * (l > 0.f ? row.inverse : row.repetition), z = entry ? scaled : l;
  return count > 0.f ? z - fma_(row.frequency, count, row.presence) : z;
}
// z where bit q says so, else -inf, in two operations
__device__ __forceinline__ float only(float z, uint32_t ok, int q) {
  const uint32_t keep = (uint32_t)((int32_t)(ok << (31 - q)) >> 31);
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, z) & keep) | (0xff800000u & ~keep));
}

// ---- a run of one row -----------------------------------------------------------------------------------------------------------
// What does not wait for something else is read first (a block is a chain of reads: the fewer links, the better): scores, the first tokens of the
// history whatever its length, the row's own numbers; then the mask, whose place one of these names.  (Scores taken apart where they are read, or
// read behind a branch, cost a wait of their own: 36 us against 33 at 256 x 131072 bfloat16, 160 against 153 for both passes at 2048 x 32000.)
// The table is 16 KB, 8 blocks a CU.  (Entries of 16 bits and runs of 8192 gain nothing: 2 % slower at 256 x 131072 bfloat16 with
// histories of up to 2048, 30 % at 1 x 50257 float; the first takes 32 us now, the second 5.2, and the first without a history 22, as a copy does.)
template <class X, class O, class K> __global__ __launch_bounds__(kBlock) void k_logits_run(ce_logits s, uint64_t row0, uint32_t runs) {
  constexpr int kGroups = kTile / kBlock / kLane, kFirst = 4;
  typedef Pack<X, kLane> Eight;
  __shared__ __attribute__((aligned(16))) uint32_t table[kTile];
  const uint64_t r = row0 + blockIdx.x / runs;
  const uint32_t v0 = blockIdx.x % runs * kTile, V = (uint32_t)s.vocab, n = V - v0 < kTile ? V - v0 : kTile;
  const X* x = (const X*)s.logits + (int64_t)r * s.logits_row + v0;
  O* o = (O*)s.out + (int64_t)r * s.out_row + v0;
  struct { uint32_t w[sizeof(Eight) / 4]; } raw[kGroups];  // taken apart behind the other reads only
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {  // lanes past the end read 8 scores of the row ahead of it (it has 8: shapes()), and drop them
    const int32_t k = (g * kBlock + threadIdx.x) * kLane, last = (int32_t)n - kLane;
    __builtin_memcpy(&raw[g], __builtin_assume_aligned(x + (k <= last ? k : last), alignof(X)), sizeof(Eight));
  }
  const uint32_t history = s.tokens ? (uint32_t)s.history : 0;
  const K* tokens = (const K*)s.tokens + (int64_t)r * s.token_row;
  K first[kFirst];
#pragma unroll
  for (int u = 0; u < kFirst; ++u) {
    const uint32_t i = u * kBlock + threadIdx.x;
    first[u] = i < history ? tokens[(int64_t)i * s.token_step] : K(0);
  }
  const uint32_t used = used_of(s, r), prompt = prompt_of(s, r);
  const int32_t m = mask_row(s, r);
  const Row row = row_of(s, r);
  uint32_t ok[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const uint32_t k = (g * kBlock + threadIdx.x) * kLane;
    ok[g] = k + kLane <= n ? allowed8(s, m, v0 + k) : 0;
  }
  if (used) {
    for (uint32_t k = threadIdx.x; k < kTile / 4; k += kBlock) ((uint4*)table)[k] = uint4{0, 0, 0, 0};
    __syncthreads();
    auto count = [&](K tok, uint32_t i) {
      const uint32_t t = place(tok, v0, n);
      if (t >= n) return;
      if (i < prompt) atomicOr(&table[t], kSeen);
      else atomicAdd(&table[t], 1u);
    };
#pragma unroll
    for (int u = 0; u < kFirst; ++u)
      if (u * kBlock + threadIdx.x < used) count(first[u], u * kBlock + threadIdx.x);
    each_token<K>(s, r, kFirst * kBlock + threadIdx.x, kBlock, used, count);
    __syncthreads();
  }
  const uint64_t b = s.bias ? (s.bias_rows == 1 ? 0 : r % s.bias_rows) * s.vocab + v0 : 0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const uint32_t k = (g * kBlock + threadIdx.x) * kLane;
    if (k + kLane <= n) {
      float l[kLane], add[kLane];
      if (s.bias) bias8(s, b + k, add);
#pragma unroll
      for (int q = 0; q < 8; ++q) l[q] = (float)__builtin_bit_cast(Eight, raw[g]).v[q];
      if (used) {
        const uint4 lo = ((const uint4*)table)[k / 4], hi = ((const uint4*)table)[k / 4 + 1];
        const uint32_t e[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        if (lo.x | lo.y | lo.z | lo.w | hi.x | hi.y | hi.z | hi.w)
#pragma unroll
          for (int q = 0; q < 8; ++q) l[q] = penalise(l[q], e[q], row);
      }
      if (s.bias)
#pragma unroll
        for (int q = 0; q < 8; ++q) l[q] += add[q];
#pragma unroll
      for (int q = 0; q < 8; ++q) l[q] = only(l[q], ok[g], q);
      store8(o + k, l);
    } else {
      for (uint32_t j = k; j < n; ++j) {  // the row's last scores
        float z = (float)x[j];
        if (used) z = penalise(z, table[j], row);
        if (s.bias) z += bias_at(s, b + j);
        o[j] = (O)(allowed(s, m, v0 + j) ? z : -__builtin_inff());
      }
    }
  }
}

// ---- short rows -----------------------------------------------------------------------------------------------------------------
// G rows (a power of two) of V < 512 scores each, G V <= kTile; dense rows are one run of memory, 8 scores a lane whatever row they are of.
template <class X, class O, class K> __global__ __launch_bounds__(kBlock) void k_logits_rows(ce_logits s, uint32_t G, uint32_t shift, int dense) {
  __shared__ __attribute__((aligned(16))) uint32_t table[kTile];
  __shared__ Row rows[kRowsMost];
  __shared__ uint32_t used[kRowsMost], prompt[kRowsMost];
  __shared__ int32_t masks[kRowsMost];
  const uint64_t r0 = (uint64_t)blockIdx.x * G;
  const uint32_t V = (uint32_t)s.vocab, have = s.rows - r0 < G ? (uint32_t)(s.rows - r0) : G, n = have * V;
  for (uint32_t j = threadIdx.x; j < have; j += kBlock) {
    rows[j] = row_of(s, r0 + j);
    used[j] = used_of(s, r0 + j);
    prompt[j] = prompt_of(s, r0 + j);
    masks[j] = mask_row(s, r0 + j);
  }
  if (s.tokens) {
    for (uint32_t k = threadIdx.x; k < (n + 3) / 4; k += kBlock) ((uint4*)table)[k] = uint4{0, 0, 0, 0};
    __syncthreads();
    auto count = [&](uint32_t j, uint32_t from, uint32_t stride) {
      each_token<K>(s, r0 + j, from, stride, used[j], [&](K tok, uint32_t i) {
        const uint32_t t = place(tok, 0, V);
        if (t >= V) return;
        if (i < prompt[j]) atomicOr(&table[j * V + t], kSeen);
        else atomicAdd(&table[j * V + t], 1u);
      });
    };
    if (s.token_row < s.token_step) {  // planes of actions: the same step of neighbouring rows lies together
      if (G >= kBlock) {
        for (uint32_t j = threadIdx.x; j < have; j += kBlock) count(j, 0, 1);
      } else if ((threadIdx.x & (G - 1)) < have) {
        count(threadIdx.x & (G - 1), threadIdx.x >> shift, kBlock >> shift);
      }
    } else {  // histories row by row: 16 lanes to a row
      for (uint32_t j = threadIdx.x / 16; j < have; j += kBlock / 16) count(j, threadIdx.x % 16, 16);
    }
  }
  __syncthreads();
  const X* x = (const X*)s.logits + (int64_t)r0 * s.logits_row;
  O* o = (O*)s.out + (int64_t)r0 * s.out_row;
  const uint32_t B = (uint32_t)s.bias_rows;
  for (uint32_t k = threadIdx.x * kLane; k < n; k += kBlock * kLane) {
    uint32_t j = k / V, v = k - j * V;
    const bool whole = k + kLane <= n;
    float l[8];
    if (dense && whole) load8(x + k, l);
    uint32_t jj = j, vv = v;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (k + q < n) {
        if (!(dense && whole)) l[q] = (float)x[(int64_t)jj * s.logits_row + vv];
        if (s.tokens) l[q] = penalise(l[q], table[k + q], rows[jj]);
        if (s.bias) l[q] += bias_at(s, (B == 1 ? 0 : (uint64_t)((uint32_t)(r0 + jj) % B) * V) + vv);
        if (!allowed(s, masks[jj], vv)) l[q] = -__builtin_inff();
        if (!(dense && whole)) o[(int64_t)jj * s.out_row + vv] = (O)l[q];
        if (++vv == V) ++jj, vv = 0;
      }
    }
    if (dense && whole) store8(o + k, l);
  }
}

template <class X, class O, class K> static void shapes(const ce_logits& s, hipStream_t st) {
  // A row is worth blocks of its own (which read 8 scores at a time, so it has to have 8) where it is long or there are no more of them than blocks in flight (8 a CU); otherwise a block takes as many rows
  // as fit and leave 1024 blocks.  us, own blocks against packed: 4.7 / 8.2 at 1000 x 32 float, 6.9 / 13.6 at 2048 x 600, 32.6 / 35.7 at 20000 x 512
  // bfloat16; 20.9 / 15.5 at 8192 x 300 float, 94 / 19 at 65536 x 64.  Packed, 131072 x 8: 9.4 with 1024 blocks, 10.2 with 512, 13.9 with 2048.
  if (s.vocab >= 512 || (s.rows <= 2048 && s.vocab >= kLane)) {
    const uint32_t runs = (uint32_t)((s.vocab + kTile - 1) / kTile);
    const uint64_t most = (1u << 23) / runs;  // rows of a launch: fewer than 2^32 threads
    for (uint64_t r = 0; r < s.rows; r += most)
      k_logits_run<X, O, K><<<(uint32_t)(s.rows - r < most ? s.rows - r : most) * runs, kBlock, 0, st>>>(s, r, runs);
    return;
  }
  uint32_t shift = 0;
  while ((2ull << shift) * s.vocab <= kTile && (2u << shift) <= kRowsMost && (s.rows >> shift) > 1024) ++shift;
  const uint32_t G = 1u << shift;
  const int dense = s.logits_row == (int64_t)s.vocab && s.out_row == (int64_t)s.vocab;
  k_logits_rows<X, O, K><<<(uint32_t)((s.rows + G - 1) / G), kBlock, 0, st>>>(s, G, shift, dense);
}

template <class X, class O> static void tokens_of(const ce_logits& s, hipStream_t st) {
  if (s.tokens && s.token_dtype == CE_I32) shapes<X, O, int32_t>(s, st);
  else if (s.tokens && s.token_dtype == CE_I64) shapes<X, O, int64_t>(s, st);
  else shapes<X, O, uint8_t>(s, st);
}
template <class X> static void outs(const ce_logits& s, hipStream_t st) {
  if (s.out_dtype == s.dtype) tokens_of<X, X>(s, st);
  else tokens_of<X, float>(s, st);
}

hipError_t launch_logits(const ce_logits& s, hipStream_t st) {
  if (s.dtype == CE_F32) outs<float>(s, st);
  else if (s.dtype == CE_BF16) outs<bf16>(s, st);
  else outs<f16>(s, st);
  return hipGetLastError();
}

// ---- gradients ------------------------------------------------------------------------------------------------------------------
// Where a bias wants a gradient, the B rows that its table covers in turn are one long row of B V columns, so that a lane keeps its 8
// columns while it walks down the R / B long rows and sums them in float; otherwise a long row is a row.  A block takes a run of
// 2048 columns, or as many whole long rows at a time as fill its lanes.  The long rows are cut into parts; a second launch adds
// their sums in a fixed order.
// The few scores that a repetition penalty scaled are put right behind that, one lane to a token of a history: a token that occurs twice
// is written twice, with the same value.  (Marking them in LDS ahead of the walk, as the forward pass does, took 113 us where the walk
// and this take 62 + 24, at 2048 x 32000 bfloat16 with histories of up to 512.)
constexpr int kCols = kBlock * kLane;

struct GradShape {
  uint64_t B, width, long_rows;  // rows of a long row, its columns, how many there are
  uint64_t chunks;               // runs of kCols columns
  uint32_t lanes, at_once;       // lanes of a long row (in a run), long rows a block walks side by side
  uint64_t parts;
};
static GradShape grad_shape(const ce_logits& s, const ce_logits_grad& g) {
  GradShape o;
  o.B = g.dbias ? s.bias_rows : 1;
  o.width = o.B * s.vocab;
  o.long_rows = s.rows / o.B;
  o.chunks = (o.width + kCols - 1) / kCols;
  o.lanes = o.width >= kCols ? kBlock : (uint32_t)((o.width + kLane - 1) / kLane);
  o.at_once = kBlock / o.lanes;
  const uint64_t passes = (o.long_rows + o.at_once - 1) / o.at_once;
  uint64_t parts = o.chunks >= 1024 ? 1 : 1024 / o.chunks;  // 4 blocks a CU, and sums of no more parts than that takes
  o.parts = parts < passes ? parts : passes;
  return o;
}

template <class X, class D> __global__ __launch_bounds__(kBlock, 4) void k_logits_grad(ce_logits s, ce_logits_grad g, GradShape w, uint64_t block0) {
  __shared__ float sums[kBlock][kLane + 1];
  const uint64_t block = block0 + blockIdx.x, chunk = block % w.chunks, part = block / w.chunks;
  const uint32_t V = (uint32_t)s.vocab, sub = threadIdx.x / w.lanes, t = threadIdx.x - sub * w.lanes;
  const uint64_t c = chunk * kCols + (uint64_t)t * kLane;
  const uint32_t cols = sub < w.at_once && c < w.width ? (uint32_t)(w.width - c < kLane ? w.width - c : kLane) : 0;  // 0: nothing to do
  const uint64_t b0 = c / V;
  const uint32_t v0 = (uint32_t)(c - b0 * V);
  const uint64_t passes = (w.long_rows + w.at_once - 1) / w.at_once;
  const uint64_t lr0 = passes * part / w.parts * w.at_once + sub, end = passes * (part + 1) / w.parts * w.at_once, lr1 = end < w.long_rows ? end : w.long_rows;
  float sum[kLane] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (cols == kLane && v0 + kLane <= V) {  // 8 columns of one row
    constexpr int kAhead = 8;  // long rows read before the first is written (the compiler could not: for all it knows, dlogits is dout)
    for (uint64_t lr = lr0; lr < lr1; lr += kAhead * w.at_once) {
      Pack<D, kLane> raw[kAhead];
      uint32_t ok[kAhead];
      int32_t m[kAhead];
      const uint32_t there = (uint32_t)((lr1 - lr + w.at_once - 1) / w.at_once);  // may be fewer: those past the end read the last one
      auto row = [&](uint32_t u) -> uint64_t { return (lr + (uint64_t)(u < there ? u : there - 1) * w.at_once) * w.B + b0; };
#pragma unroll
      for (int u = 0; u < kAhead; ++u) m[u] = mask_row(s, row(u));
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        __builtin_memcpy(&raw[u], __builtin_assume_aligned((const D*)g.dout + (int64_t)row(u) * g.dout_row + v0, alignof(D)), sizeof(raw[u]));
#pragma unroll
      for (int u = 0; u < kAhead; ++u) ok[u] = allowed8(s, m[u], v0);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u < (int)there) {
          float d[kLane];
#pragma unroll
          for (int j = 0; j < kLane; ++j) {
            d[j] = (ok[u] >> j) & 1 ? (float)raw[u].v[j] : 0.f;
            sum[j] += d[j];
          }
          if (g.dlogits) store8((X*)g.dlogits + row(u) * V + v0, d);
        }
    }
  } else if (cols) {  // columns of two rows and more, or a long row's last ones
    for (uint64_t lr = lr0; lr < lr1; lr += w.at_once) {
      uint64_t r = lr * w.B + b0;
      uint32_t v = v0;
      int32_t m = mask_row(s, r);
#pragma unroll
      for (int j = 0; j < kLane; ++j) {
        if (j >= (int)cols) continue;
        const float d = allowed(s, m, v) ? (float)((const D*)g.dout)[(int64_t)r * g.dout_row + v] : 0.f;
        sum[j] += d;
        if (g.dlogits) ((X*)g.dlogits)[lr * w.width + c + j] = (X)d;
        if (++v == V && j + 1 < (int)cols) {
          v = 0;
          m = mask_row(s, ++r);
        }
      }
    }
  }
  if (!g.dbias) return;
  if (w.at_once > 1) {  // the long rows walked side by side, in their order
#pragma unroll
    for (int j = 0; j < kLane; ++j) sums[threadIdx.x][j] = sum[j];
    __syncthreads();
    if (sub == 0)
      for (uint32_t k = 1; k < w.at_once; ++k)
#pragma unroll
        for (int j = 0; j < kLane; ++j) sum[j] += sums[k * w.lanes + t][j];
    if (sub != 0) return;
  }
  for (uint32_t j = 0; j < kLane; ++j)
    if (j < cols) ((float*)s.workspace)[part * w.width + c + j] = sum[j];
}

// The scores that a repetition penalty scaled.  kTokensBlock places of the histories to a block, neighbouring lanes where tokens lie together.
constexpr uint32_t kTokensBlock = kBlock * 4;
template <class X, class D, class K> __global__ __launch_bounds__(kBlock) void k_logits_repeats(ce_logits s, ce_logits_grad g, uint64_t block0) {
  const bool planes = s.token_row < s.token_step;
  const uint64_t inner = planes ? s.rows : s.history, outer = planes ? s.history : s.rows, n = inner * outer;
  const uint64_t first = (block0 + blockIdx.x) * kTokensBlock, o0 = first / inner;
  const uint32_t i0 = (uint32_t)(first - o0 * inner);
  // What depends on nothing is read for all four places, then what depends on that; places that do not count read another's.  A branch around a
  // read and its use would make each place wait for itself (28 us where it takes 24, 1 M places over 2048 x 32000 bfloat16).
  const uint32_t V = (uint32_t)s.vocab, history = (uint32_t)s.history;
  uint64_t r[4];
  uint32_t i[4], t[4], bits[4] = {0, 0, 0, 0};
  int32_t len[4], index[4], m[4];
  float rep[4];
  K tok[4];
  D d[4];
  X l[4];
  bool good[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const uint32_t k = u * kBlock + threadIdx.x;
    good[u] = first + k < n;
    const uint32_t at = good[u] ? i0 + k : i0, over = at / (uint32_t)inner, in = at - over * (uint32_t)inner;
    r[u] = planes ? in : o0 + over;
    i[u] = planes ? (uint32_t)o0 + over : in;
    len[u] = 0x7fffffff;
    index[u] = -1;
    rep[u] = (float)s.repetition_all;
    tok[u] = ((const K*)s.tokens)[(int64_t)r[u] * s.token_row + (int64_t)i[u] * s.token_step];
  }
  if (s.lengths)
#pragma unroll
    for (int u = 0; u < 4; ++u) len[u] = s.lengths[r[u]];
  if (s.mask_index)
#pragma unroll
    for (int u = 0; u < 4; ++u) index[u] = s.mask_index[r[u]];
  if (s.repetition)
#pragma unroll
    for (int u = 0; u < 4; ++u) rep[u] = s.repetition[r[u]];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    t[u] = place(tok[u], 0, V);
    good[u] = good[u] && i[u] < history && (int64_t)i[u] < len[u] && t[u] < V;
    if (!good[u]) t[u] = 0;
    m[u] = mask_row(s, r[u], index[u]);
    d[u] = ((const D*)g.dout)[(int64_t)r[u] * g.dout_row + t[u]];
    l[u] = ((const X*)s.logits)[(int64_t)r[u] * s.logits_row + t[u]];
  }
  if (s.mask) {
    const bool words = s.mask_dtype != CE_U8;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint64_t row = m[u] < 0 ? 0 : m[u];
      if (words) bits[u] = ((const uint32_t*)s.mask)[row * ((s.vocab + 31) / 32) + t[u] / 32];
      else bits[u] = ((const uint8_t*)s.mask)[row * s.vocab + t[u]];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) good[u] = good[u] && (m[u] < 0 ? m[u] == -1 : words ? (bits[u] >> (t[u] % 32)) & 1u : bits[u] != 0);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (good[u]) ((X*)g.dlogits)[r[u] * V + t[u]] = (X)((float)l[u] > 0.f ? (float)d[u] / rep[u] : (float)d[u] * rep[u]);
}

// 64 columns to a block, each 4th part to a wave, the waves' sums in their order
template <class T> __global__ __launch_bounds__(kBlock) void k_logits_bias(const float* part, T* dbias, uint64_t n, uint32_t parts, uint64_t block0) {
  __shared__ float sums[4][kWave];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t i = (block0 + blockIdx.x) * kWave + lane;
  float sum = 0.f;
  if (i < n)
#pragma unroll 8
    for (uint32_t k = w; k < parts; k += 4) sum += part[(uint64_t)k * n + i];
  sums[w][lane] = sum;
  __syncthreads();
  if (w == 0 && i < n) dbias[i] = (T)(((sums[0][lane] + sums[1][lane]) + sums[2][lane]) + sums[3][lane]);
}

uint64_t logits_grad_workspace(const ce_logits& s, const ce_logits_grad& g) {
  const GradShape w = grad_shape(s, g);
  return g.dbias ? w.parts * w.width * sizeof(float) : 0;
}

constexpr uint64_t kBlocksMost = 1u << 23;  // of a launch: fewer than 2^32 threads

template <class X, class D, class K> static void repeats_go(const ce_logits& s, const ce_logits_grad& g, hipStream_t st) {
  const uint64_t blocks = (s.rows * s.history + kTokensBlock - 1) / kTokensBlock;
  for (uint64_t b = 0; b < blocks; b += kBlocksMost)
    k_logits_repeats<X, D, K><<<(uint32_t)(blocks - b < kBlocksMost ? blocks - b : kBlocksMost), kBlock, 0, st>>>(s, g, b);
}
template <class X, class D> static void grad_go(const ce_logits& s, const ce_logits_grad& g, const GradShape& w, hipStream_t st) {
  const uint64_t blocks = w.chunks * w.parts;
  for (uint64_t b = 0; b < blocks; b += kBlocksMost)
    k_logits_grad<X, D><<<(uint32_t)(blocks - b < kBlocksMost ? blocks - b : kBlocksMost), kBlock, 0, st>>>(s, g, w, b);
  if (!s.tokens || !s.history || !g.dlogits || (!s.repetition && s.repetition_all == 1.0)) return;
  if (s.token_dtype == CE_I32) repeats_go<X, D, int32_t>(s, g, st);
  else if (s.token_dtype == CE_I64) repeats_go<X, D, int64_t>(s, g, st);
  else repeats_go<X, D, uint8_t>(s, g, st);
}
template <class X> static void grad_outs(const ce_logits& s, const ce_logits_grad& g, const GradShape& w, hipStream_t st) {
  if (s.out_dtype == s.dtype) grad_go<X, X>(s, g, w, st);
  else grad_go<X, float>(s, g, w, st);
}
template <class T> static void bias_go(const ce_logits& s, const ce_logits_grad& g, const GradShape& w, hipStream_t st) {
  const uint64_t blocks = (w.width + kWave - 1) / kWave;
  for (uint64_t b = 0; b < blocks; b += kBlocksMost)
    k_logits_bias<T><<<(uint32_t)(blocks - b < kBlocksMost ? blocks - b : kBlocksMost), kBlock, 0, st>>>((const float*)s.workspace, (T*)g.dbias, w.width, (uint32_t)w.parts, b);
}

hipError_t launch_logits_grad(const ce_logits& s, const ce_logits_grad& g, hipStream_t st) {
  const GradShape w = grad_shape(s, g);
  if (s.dtype == CE_F32) grad_outs<float>(s, g, w, st);
  else if (s.dtype == CE_BF16) grad_outs<bf16>(s, g, w, st);
  else grad_outs<f16>(s, g, w, st);
  if (hipError_t e = hipGetLastError()) return e;
  if (g.dbias) {
    if (s.bias_dtype == CE_F32) bias_go<float>(s, g, w, st);
    else if (s.bias_dtype == CE_BF16) bias_go<bf16>(s, g, w, st);
    else bias_go<f16>(s, g, w, st);
  }
  return hipGetLastError();
}

}  // namespace cp
