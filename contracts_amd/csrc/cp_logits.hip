// cp_logits.hip — scores shaped ahead of a selection (ce_process_logits): penalties for repeated tokens, biases, masks; and the
// gradients of logits and bias.
//
// A block takes a row's run of kChunk tokens: a table in LDS counts the history's tokens that fall into the run (the prompt's
// only as "seen", the top bit), then the run streams through once: read, penalise, bias, mask, write.
// Bound by HBM: each score is read once and written once.
#include "cp_common.h"

namespace cp {

constexpr int kBlock = 256, kChunk = 4096;
constexpr uint32_t kSeen = 0x80000000u;

struct Row {  // what a row is penalised with
  float repetition, presence, frequency;
  uint64_t used, prompt;  // how much of its history counts, and how much of that is its prompt
};
__device__ __forceinline__ Row row_of(const ce_logits& s, uint64_t r) {
  Row o;
  o.repetition = s.repetition ? s.repetition[r] : (float)s.repetition_all;
  o.presence = s.presence ? s.presence[r] : (float)s.presence_all;
  o.frequency = s.frequency ? s.frequency[r] : (float)s.frequency_all;
  o.used = s.tokens ? s.history : 0;
  if (s.lengths) {
    const int32_t l = s.lengths[r];
    if (l < 0) o.used = 0;
    else if ((uint64_t)l < o.used) o.used = l;
  }
  o.prompt = 0;
  if (s.prompt_lengths) {
    const int32_t l = s.prompt_lengths[r];
    o.prompt = l > 0 ? l : 0;
  }
  return o;
}
// The token at place i of row r's history, or a number past every vocabulary.
__device__ __forceinline__ uint64_t token(const ce_logits& s, uint64_t r, uint64_t i) {
  const int64_t at = (int64_t)r * s.token_row + (int64_t)i * s.token_step;
  if (s.token_dtype == CE_U8) return ((const uint8_t*)s.tokens)[at];
  if (s.token_dtype == CE_I32) return (uint64_t)(int64_t)((const int32_t*)s.tokens)[at];
  return (uint64_t)((const int64_t*)s.tokens)[at];
}
// The mask's row of row r: -1 = everything is allowed, -2 = nothing is.
__device__ __forceinline__ int64_t mask_row(const ce_logits& s, uint64_t r) {
  if (!s.mask) return -1;
  if (!s.mask_index) return (int64_t)(r % s.mask_rows);
  const int32_t m = s.mask_index[r];
  return m < 0 ? -1 : (uint64_t)m < s.mask_rows ? m : -2;
}
__device__ __forceinline__ bool allowed(const ce_logits& s, int64_t m, uint64_t v) {
  if (m < 0) return m == -1;
  if (s.mask_dtype == CE_U8) return ((const uint8_t*)s.mask)[(uint64_t)m * s.vocab + v] != 0;
  return (((const uint32_t*)s.mask)[(uint64_t)m * ((s.vocab + 31) / 32) + v / 32] >> (v % 32)) & 1u;
}
__device__ __forceinline__ float bias_at(const ce_logits& s, uint64_t at) {
  if (s.bias_dtype == CE_F32) return ((const float*)s.bias)[at];
  if (s.bias_dtype == CE_BF16) return (float)((const bf16*)s.bias)[at];
  return (float)((const f16*)s.bias)[at];
}

template <class X, class O> __global__ __launch_bounds__(kBlock) void k_logits(ce_logits s) {
  __shared__ uint32_t table[kChunk];
  const uint64_t r = blockIdx.x, v0 = (uint64_t)blockIdx.y * kChunk;
  const uint32_t n = (uint32_t)(s.vocab - v0 < kChunk ? s.vocab - v0 : kChunk);
  const Row row = row_of(s, r);
  const bool history = row.used > 0;
  if (history) {
    for (uint32_t k = threadIdx.x; k < n; k += kBlock) table[k] = 0;
    __syncthreads();
    for (uint64_t i = threadIdx.x; i < row.used; i += kBlock) {
      const uint64_t t = token(s, r, i) - v0;
      if (t < n) {
        if (i < row.prompt) atomicOr(&table[t], kSeen);
        else atomicAdd(&table[t], 1u);
      }
    }
    __syncthreads();
  }
  const int64_t m = mask_row(s, r);
  const X* x = (const X*)s.logits + (int64_t)r * s.logits_row;
  O* o = (O*)s.out + (int64_t)r * s.out_row;
  const uint64_t b = s.bias ? (r % s.bias_rows) * s.vocab : 0;
  for (uint32_t k = threadIdx.x; k < n; k += kBlock) {
    const uint64_t v = v0 + k;
    const float l = (float)x[v];
    float z = l;
    if (history && table[k]) {
      const uint32_t count = table[k] & ~kSeen;
      z = l > 0.f ? l / row.repetition : l * row.repetition;
      if (count) z = z - row.presence - row.frequency * (float)count;
    }
    if (s.bias) z += bias_at(s, b + v);
    if (!allowed(s, m, v)) z = -__builtin_inff();
    o[v] = (O)z;
  }
}

template <class X> static void outs(const ce_logits& s, dim3 grid, hipStream_t st) {
  if (s.out_dtype == s.dtype) k_logits<X, X><<<grid, kBlock, 0, st>>>(s);
  else k_logits<X, float><<<grid, kBlock, 0, st>>>(s);
}

hipError_t launch_logits(const ce_logits& s, hipStream_t st) {
  const dim3 grid((uint32_t)s.rows, (uint32_t)((s.vocab + kChunk - 1) / kChunk));
  if (s.dtype == CE_F32) outs<float>(s, grid, st);
  else if (s.dtype == CE_BF16) outs<bf16>(s, grid, st);
  else outs<f16>(s, grid, st);
  return hipGetLastError();
}

// ---- gradients ------------------------------------------------------------------------------------------------------------------
constexpr int kGradChunk = kBlock * 4;

// Rows that share a bias row are cut into `parts` runs; a block sums its run in float, row after row, and a second launch adds the
// parts in their order.
static uint32_t grad_parts(const ce_logits& s, const ce_logits_grad& g) {
  const uint64_t b = g.dbias ? s.bias_rows : 1, each = (s.rows + b - 1) / b, chunks = (s.vocab + kGradChunk - 1) / kGradChunk;
  uint64_t parts = 2048 / (b * chunks) + 1;
  if (parts > each) parts = each;
  return (uint32_t)parts;
}

template <class X, class D> __global__ __launch_bounds__(kBlock) void k_logits_grad(ce_logits s, ce_logits_grad g, uint32_t B, uint32_t parts) {
  __shared__ uint32_t bits[kGradChunk / 32];
  const uint32_t chunks = (uint32_t)((s.vocab + kGradChunk - 1) / kGradChunk), rest = blockIdx.x / chunks;
  const uint64_t v0 = (uint64_t)(blockIdx.x % chunks) * kGradChunk;
  const uint32_t b = rest % B, part = rest / B;
  const uint64_t each = (s.rows - b + B - 1) / B;  // rows b, b + B, ...
  const uint64_t k0 = each * part / parts, k1 = each * (part + 1) / parts;
  float sum[4] = {0, 0, 0, 0};
  for (uint64_t k = k0; k < k1; ++k) {
    const uint64_t r = b + k * B;
    const Row row = row_of(s, r);
    const bool history = g.dlogits && row.used > 0 && row.repetition != 1.f;
    if (history) {
      __syncthreads();
      if (threadIdx.x < kGradChunk / 32) bits[threadIdx.x] = 0;
      __syncthreads();
      for (uint64_t i = threadIdx.x; i < row.used; i += kBlock) {
        const uint64_t t = token(s, r, i), at = t - v0;
        if (at < kGradChunk && t < s.vocab) atomicOr(&bits[at / 32], 1u << (at % 32));
      }
      __syncthreads();
    }
    const int64_t m = mask_row(s, r);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t at = q * kBlock + threadIdx.x;
      const uint64_t v = v0 + at;
      if (v >= s.vocab) continue;
      float d = (float)((const D*)g.dout)[(int64_t)r * g.dout_row + v];
      if (!allowed(s, m, v)) d = 0.f;
      sum[q] += d;
      if (!g.dlogits) continue;
      if (history && ((bits[at / 32] >> (at % 32)) & 1u)) {
        const float l = (float)((const X*)s.logits)[(int64_t)r * s.logits_row + v];
        d = l > 0.f ? d / row.repetition : d * row.repetition;
      }
      ((X*)g.dlogits)[r * s.vocab + v] = (X)d;
    }
  }
  if (!g.dbias) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint64_t v = v0 + q * kBlock + threadIdx.x;
    if (v < s.vocab) ((float*)s.workspace)[((uint64_t)part * B + b) * s.vocab + v] = sum[q];
  }
}

template <class T> __global__ __launch_bounds__(kBlock) void k_logits_bias(const float* part, T* dbias, uint64_t n, uint32_t parts) {
  const uint64_t i = (uint64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= n) return;
  float sum = part[i];
  for (uint32_t k = 1; k < parts; ++k) sum += part[(uint64_t)k * n + i];
  dbias[i] = (T)sum;
}

uint64_t logits_grad_workspace(const ce_logits& s, const ce_logits_grad& g) {
  return g.dbias ? (uint64_t)grad_parts(s, g) * s.bias_rows * s.vocab * sizeof(float) : 0;
}

template <class X> static void douts(const ce_logits& s, const ce_logits_grad& g, dim3 grid, uint32_t B, uint32_t parts, hipStream_t st) {
  if (s.out_dtype == s.dtype) k_logits_grad<X, X><<<grid, kBlock, 0, st>>>(s, g, B, parts);
  else k_logits_grad<X, float><<<grid, kBlock, 0, st>>>(s, g, B, parts);
}

hipError_t launch_logits_grad(const ce_logits& s, const ce_logits_grad& g, hipStream_t st) {
  const uint32_t B = g.dbias ? (uint32_t)s.bias_rows : 1, parts = grad_parts(s, g);
  const dim3 grid((uint32_t)((s.vocab + kGradChunk - 1) / kGradChunk) * B * parts);
  if (s.dtype == CE_F32) douts<float>(s, g, grid, B, parts, st);
  else if (s.dtype == CE_BF16) douts<bf16>(s, g, grid, B, parts, st);
  else douts<f16>(s, g, grid, B, parts, st);
  if (hipError_t e = hipGetLastError()) return e;
  if (g.dbias) {
    const uint64_t n = (uint64_t)B * s.vocab;
    const uint32_t blocks = (uint32_t)((n + kBlock - 1) / kBlock);
    const float* part = (const float*)s.workspace;
    if (s.bias_dtype == CE_F32) k_logits_bias<float><<<blocks, kBlock, 0, st>>>(part, (float*)g.dbias, n, parts);
    else if (s.bias_dtype == CE_BF16) k_logits_bias<bf16><<<blocks, kBlock, 0, st>>>(part, (bf16*)g.dbias, n, parts);
    else k_logits_bias<f16><<<blocks, kBlock, 0, st>>>(part, (f16*)g.dbias, n, parts);
  }
  return hipGetLastError();
}

}  // namespace cp
