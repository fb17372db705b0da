// cp_scan_grad.hip — the gradients of the gated linear recurrence (ce_linear_scan_backward).
//
//   g_t = dy_t + R_t,  R_t = a_{t+1} g_{t+1} (what the successor hands back; nothing over a border that done closes);
//   dx_t = g_t;  da_t = sum over a head of g_t k_t, k_t the state that step t multiplied;  dstate = R ahead of the first step.
// The mirror image of cp_scan.hip: blocks of 64 lanes x VEC channels and W waves walk the time axis from its end, a wave's run of
// kSteps steps is the map R -> P R + Q, the waves exchange (P, Q) through LDS, and a time axis cut into chunks is reduced by a launch of
// its own first.  The states are not kept in y's rounded type: the forward pass left the float state ahead of every run (1 / 16
// of a float plane), and a wave walks its run forward again in registers.  Reads x, a, dy, writes dx and da, once each.
// A head's gate sums over its channels: lanes of a segment by butterflies, a head wider than a wave through partial sums that a
// second launch adds up in a fixed order (no atomics: the same call gives the same bits).
#include "cp_common.h"

namespace cp {

constexpr int kSteps = CE_SCAN_SAVED_STEPS;

template <class X, class G, int MODE, int VEC> struct GradTile {
  static constexpr int GV = MODE == kGateChannel ? VEC : 1;
  Pack<X, VEC> x[kSteps], dy[kSteps];
  Pack<G, GV> g[MODE == kGateConst ? 1 : kSteps];
  uint8_t d[kSteps];
};

template <class X, class G, int MODE, int VEC, int W, bool REDUCE> __global__ __launch_bounds__(kWave * W) void k_scan_grad(ScanParams p) {
  typedef GradTile<X, G, MODE, VEC> TileT;
  __shared__ float fold[W > 1 ? 2 : 1][W][2][VEC][kWave];
  const int lane = threadIdx.x & 63, w = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const uint32_t slot = blockIdx.x * kWave + lane;
  uint32_t e, c, head = 0;
  bool live;
  if (MODE == kGateHead) {  // `seg` lanes to a head of head / VEC columns
    const uint32_t group = slot / p.seg, in = (slot % p.seg) * VEC;
    live = in < p.head && group < p.cols / (p.head / VEC);
    e = group / p.heads;
    head = group % p.heads;
    c = head * p.head + in;
  } else {
    live = slot < p.cols;
    e = slot / p.row_cols;
    c = (slot % p.row_cols) * VEC;
  }
  if (!live) e = 0, c = 0, head = 0;  // lanes past the end read a column that exists, write nothing and add 0
  const X* x = (const X*)p.x + (int64_t)e * p.x_row + c;
  const G* gate = (const G*)p.gate;
  if (MODE != kGateConst) gate += (int64_t)e * p.gate_row + (MODE == kGateHead ? head : c);
  const uint8_t* done = p.done ? p.done + (int64_t)e * p.done_row + (int64_t)p.cut_off * p.done_step : nullptr;
  const uint64_t EC = (uint64_t)p.cols * VEC, ch = (uint64_t)e * p.row_cols * VEC + c;
  const X* dy = (const X*)p.dy + ch;
  X* dx = (X*)p.dx + ch;
  const uint32_t chunk = blockIdx.y + (REDUCE ? 1 : 0);  // nobody folds chunk 0
  const uint64_t i0 = chunk * p.chunk, i1 = i0 + p.chunk < p.T ? i0 + p.chunk : p.T;

  float R[VEC], P[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) R[v] = 0.f, P[v] = 1.f;
  if (!REDUCE) {
    const bool cut = done && p.cut_off < 0 && p.T > 0 && done[(int64_t)p.T * p.done_step];
    if (p.dlast && !cut)
#pragma unroll
      for (int v = 0; v < VEC; ++v) R[v] = ((const float*)p.dlast)[ch + v];
    const float* part = (const float*)p.part + ch;
    for (uint32_t k = p.chunks - 1; k > chunk; --k)
#pragma unroll
      for (int v = 0; v < VEC; ++v) R[v] = apply(part[(uint64_t)(k - 1) * 2 * EC + v], part[((uint64_t)(k - 1) * 2 + 1) * EC + v], R[v]);
  }

  auto take = [&](TileT& t, uint64_t i) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint64_t at = i + s;
      if (at < i1) {
        if (!REDUCE) t.x[s] = load<X, VEC>(x + (int64_t)at * p.x_step);
        if (p.dy) t.dy[s] = load<X, VEC>(dy + (int64_t)at * p.y_step);
        if (MODE != kGateConst) t.g[MODE == kGateConst ? 0 : s] = load<G, TileT::GV>(gate + (int64_t)at * p.gate_step);
        const uint64_t flag = at + p.cut_off;
        t.d[s] = done && flag < p.T ? done[(int64_t)at * p.done_step] : 0;
      }
    }
  };
  auto gate_of = [&](const TileT& t, int s, int v) -> float {
    const float a = MODE == kGateConst ? (float)p.decay : (float)t.g[MODE == kGateConst ? 0 : s].v[MODE == kGateChannel ? v : 0];
    return t.d[s] ? 0.f : a;
  };

  int buf = 0;
  const uint64_t span = (uint64_t)W * kSteps, tiles = i1 > i0 ? (i1 - i0 + span - 1) / span : 0;
  for (uint64_t n = tiles; n-- > 0;) {
    const uint64_t i = i0 + n * span + (uint64_t)w * kSteps;
    TileT t;
    take(t, i);
    if (W > 1 || REDUCE) {
      float rp[VEC], rq[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) rp[v] = 1.f, rq[v] = 0.f;
#pragma unroll
      for (int s = kSteps - 1; s >= 0; --s)
        if (i + s < i1)
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            const float a = gate_of(t, s, v), gt = (p.dy ? (float)t.dy[s].v[v] : 0.f) + rq[v];
            rp[v] *= a;
            rq[v] = a == 0.f ? 0.f : a * gt;
          }
#pragma unroll
      for (int v = 0; v < VEC; ++v) fold[buf][w][0][v][lane] = rp[v], fold[buf][w][1][v][lane] = rq[v];
      if (W > 1) __syncthreads();
    }
    float mine[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) mine[v] = R[v];
    if (W > 1 || REDUCE) {
#pragma unroll
      for (int k = W - 1; k >= 0; --k) {
        if (k == w)
#pragma unroll
          for (int v = 0; v < VEC; ++v) mine[v] = R[v];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          R[v] = apply(fold[buf][k][0][v][lane], fold[buf][k][1][v][lane], R[v]);
          if (REDUCE) P[v] *= fold[buf][k][0][v][lane];
        }
      }
      buf ^= W > 1;
    }
    if (REDUCE) continue;
    float k[kSteps][VEC];  // the state that each step multiplies
    if (i < i1) {
      float h[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[v] = p.saved[(i / kSteps) * EC + ch + v];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        if (i + s < i1)
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            k[s][v] = t.d[s] ? 0.f : h[v];
            h[v] = step(gate_of(t, s, v), h[v], (float)t.x[s].v[v]);
          }
    }
#pragma unroll
    for (int s = kSteps - 1; s >= 0; --s)
      if (i + s < i1) {
        Pack<X, VEC> o;
        float da[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float a = gate_of(t, s, v), gt = (p.dy ? (float)t.dy[s].v[v] : 0.f) + mine[v];
          mine[v] = a == 0.f ? 0.f : a * gt;
          o.v[v] = (X)gt;
          da[v] = live ? gt * k[s][v] : 0.f;
        }
        if (live && p.dx) store(dx + (int64_t)(i + s) * p.y_step, o);
        if (!p.dgate) continue;
        if (MODE == kGateChannel) {
          Pack<G, VEC> q;
#pragma unroll
          for (int v = 0; v < VEC; ++v) q.v[v] = (G)da[v];
          if (live) store((G*)p.dgate + ch + (int64_t)(i + s) * p.dgate_step, q);
        } else if (MODE == kGateHead) {
          float sum = da[0];
#pragma unroll
          for (int v = 1; v < VEC; ++v) sum += da[v];
          const uint32_t width = p.seg < kWave ? p.seg : kWave;
          for (uint32_t m = width / 2; m > 0; m >>= 1) sum += __shfl_xor(sum, (int)m);
          if (live && (lane & (width - 1)) == 0) {
            const uint64_t at = (uint64_t)e * p.heads + head;
            if (p.slabs == 1) {
              ((G*)p.dgate)[at + (int64_t)(i + s) * p.dgate_step] = (G)sum;
            } else {
              const uint64_t TEH = p.T * (uint64_t)(p.cols / p.row_cols) * p.heads;
              p.slab[((slot % p.seg) / kWave) * TEH + (i + s) * (uint64_t)(p.cols / p.row_cols) * p.heads + at] = sum;
            }
          }
        }
      }
    if (W == 1)
#pragma unroll
      for (int v = 0; v < VEC; ++v) R[v] = mine[v];
  }
  if (!live || w != 0) return;
  if (REDUCE) {
    float* part = (float*)p.part + (uint64_t)blockIdx.y * 2 * EC + ch;
#pragma unroll
    for (int v = 0; v < VEC; ++v) part[v] = P[v], part[EC + v] = R[v];
  } else if (p.dstate && chunk == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) ((float*)p.dstate)[ch + v] = R[v];
  }
}

// [slabs][T][E][H] partial sums -> dgate, in slab order; `i` counts processed steps
template <class G> __global__ __launch_bounds__(256) void k_scan_grad_slabs(ScanParams p) {
  const uint64_t EH = (uint64_t)(p.cols / p.row_cols) * p.heads, n = p.T * EH;
  for (uint64_t j = (uint64_t)blockIdx.x * 256 + threadIdx.x; j < n; j += (uint64_t)gridDim.x * 256) {
    float sum = p.slab[j];
    for (uint32_t s = 1; s < p.slabs; ++s) sum += p.slab[(uint64_t)s * n + j];
    ((G*)p.dgate)[j % EH + (int64_t)(j / EH) * p.dgate_step] = (G)sum;
  }
}

template <class X, class G, int MODE, int VEC> static hipError_t go(const ScanParams& p, hipStream_t stream) {
  const uint64_t slots = MODE == kGateHead ? (uint64_t)(p.cols / (p.head / VEC)) * p.seg : p.cols;
  const dim3 grid((uint32_t)((slots + kWave - 1) / kWave), p.chunks);
  if (p.T <= kSteps) {
    k_scan_grad<X, G, MODE, VEC, 1, false><<<grid, kWave, 0, stream>>>(p);
  } else {
    if (p.chunks > 1) {
      k_scan_grad<X, G, MODE, VEC, 4, true><<<dim3(grid.x, p.chunks - 1), 4 * kWave, 0, stream>>>(p);
      if (hipError_t e = hipGetLastError()) return e;
    }
    k_scan_grad<X, G, MODE, VEC, 4, false><<<grid, 4 * kWave, 0, stream>>>(p);
  }
  if (hipError_t e = hipGetLastError()) return e;
  if (MODE == kGateHead && p.dgate && p.slabs > 1 && p.T > 0) {
    const uint64_t n = p.T * (uint64_t)(p.cols / p.row_cols) * p.heads, blocks = (n + 255) / 256;
    k_scan_grad_slabs<G><<<(uint32_t)(blocks < 4096 ? blocks : 4096), 256, 0, stream>>>(p);
  }
  return hipGetLastError();
}

template <class X, class G, int MODE> static hipError_t vecs(const ScanParams& p, int vec, hipStream_t s) {
  if (vec == 2) return go<X, G, MODE, 2>(p, s);
  return go<X, G, MODE, 1>(p, s);
}
template <class X, class G> static hipError_t modes(const ScanParams& p, int mode, int vec, hipStream_t s) {
  if (mode == kGateConst) return vecs<X, X, kGateConst>(p, vec, s);
  if (mode == kGateChannel) return vecs<X, G, kGateChannel>(p, vec, s);
  return vecs<X, G, kGateHead>(p, vec, s);
}

hipError_t launch_scan_grad(const ScanParams& p, int dtype, int gate_dtype, int mode, int vec, hipStream_t s) {
  const bool wide = gate_dtype == CE_F32;
  if (dtype == CE_F32) return modes<float, float>(p, mode, vec, s);
  if (dtype == CE_BF16) return wide ? modes<bf16, float>(p, mode, vec, s) : modes<bf16, bf16>(p, mode, vec, s);
  return wide ? modes<f16, float>(p, mode, vec, s) : modes<f16, f16>(p, mode, vec, s);
}

}  // namespace cp
