// cp_scan_grad.hip — the gradients of the gated linear recurrence (ce_linear_scan_backward).
//
//   g_t = dy_t + R_t,  R_t = a_{t+1} g_{t+1} (what the successor hands back; nothing over a border that done closes);
//   dx_t = g_t;  da_t = sum over a head of g_t k_t, k_t the state that step t multiplied;  dstate = R ahead of the first step.
// The mirror image of cp_scan.hip: blocks of 64 lanes x VEC channels and W waves walk the time axis from its end, a wave's run of
// kSteps steps is the map R -> P R + Q, the waves exchange (P, Q) through LDS, and a time axis cut into chunks is reduced by a launch of
// its own first.  The states are not kept in y's rounded type: the forward pass left the float state ahead of every run (1 / 16
// of a float plane), and a wave walks its run forward again in registers.  Reads x, a, dy, writes dx and da, once each:
// [512, 256, 256] bfloat16 in 69 us, 4.9 TB/s.
// A head's gate sums over its channels: the run's terms go through LDS, where a lane adds up a step of a head (a butterfly in
// registers would take 6 exchanges a step: 178 us against 59 at [1000, 37, 360] float, 9 heads); a head wider than a wave leaves partial sums
// that a second launch adds up in a fixed order (no atomics: the same call gives the same bits).
#include "cp_common.h"

namespace cp {

constexpr int kSteps = CE_SCAN_SAVED_STEPS;

template <class X, class G, int MODE, int VEC, int W, bool REDUCE> __global__ __launch_bounds__(kWave * W) void k_scan_grad(ScanParams p) {
  constexpr int GV = MODE == kGateChannel ? VEC : 1;  // gates of a lane; its channels under one gate have one product P too
  __shared__ float fold[W > 1 ? 2 : 1][W][GV + VEC][kWave];  // P, then H
  // a run's terms of dgate, a row of lanes to a step; rows are 65 apart, so that lanes which add up different steps read different banks
  __shared__ float terms[MODE == kGateHead && !REDUCE ? W : 1][MODE == kGateHead && !REDUCE ? kSteps : 1][kWave + 1];
  const int lane = threadIdx.x & 63, w = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  uint32_t e, c, head = 0, group0 = 0;
  bool live;
  if (MODE == kGateHead) {
    // in_wave heads of `lanes` lanes side by side; or the blockIdx.x % slabs-th wave of a wider head
    group0 = p.in_wave ? blockIdx.x * p.in_wave : blockIdx.x / p.slabs;
    const uint32_t groups = p.rows * p.heads, own = p.in_wave ? lane / p.lanes : 0, in = p.in_wave ? lane - own * p.lanes : blockIdx.x % p.slabs * kWave + lane;
    live = p.in_wave ? own < p.in_wave && group0 + own < groups : in < p.lanes;
    const uint32_t g = group0 + own < groups && own < (p.in_wave ? p.in_wave : 1) ? group0 + own : group0;
    e = g / p.heads;
    head = g - e * p.heads;
    c = head * p.head + (live ? in : p.in_wave ? 0 : p.lanes - 1) * VEC;
  } else {
    const uint32_t slot = blockIdx.x * kWave + lane;
    live = slot < p.cols;
    const uint32_t col = live ? slot : p.cols - 1;
    e = col / p.row_cols;
    c = (col - e * p.row_cols) * VEC;
  }
  // lanes that are not live do what another one of their wave does and write the same; none lies ahead of the wave's first row e0, from which all
  // count
  const uint32_t e0 = __builtin_amdgcn_readfirstlane(e);
  const uint64_t EC = (uint64_t)p.cols * VEC, ch = (uint64_t)e * p.row_cols * VEC + c;
  // a lane's offsets from row e0
  const uint32_t x_off = (uint32_t)((int64_t)(e - e0) * p.x_row + c) * (uint32_t)sizeof(X), y_off = ((e - e0) * p.row_cols * VEC + c) * (uint32_t)sizeof(X);
  const uint32_t g_off = MODE == kGateConst ? 0 : (uint32_t)((int64_t)(e - e0) * p.gate_row + (MODE == kGateHead ? head : c)) * (uint32_t)sizeof(G);
  const uint32_t dg_off = ((e - e0) * p.row_cols * VEC + c) * (uint32_t)sizeof(G);
  const uint64_t x0 = (uint64_t)((const X*)p.x + (int64_t)e0 * p.x_row), g0 = (uint64_t)((const G*)p.gate + (int64_t)e0 * p.gate_row);
  const uint64_t row0 = (uint64_t)e0 * p.row_cols * VEC;
  const uint64_t dy0 = (uint64_t)((const X*)p.dy + row0), dx0 = (uint64_t)((X*)p.dx + row0), dg0 = (uint64_t)((G*)p.dgate + row0);
  const uint64_t x_step = (uint64_t)(p.x_step * (int64_t)sizeof(X)), g_step = (uint64_t)(p.gate_step * (int64_t)sizeof(G));
  const uint64_t y_step = (uint64_t)(p.y_step * (int64_t)sizeof(X)), dg_step = (uint64_t)(p.dgate_step * (int64_t)sizeof(G));
  const uint32_t chunk = blockIdx.y + (REDUCE ? 1 : 0);  // nobody folds chunk 0
  const uint64_t i0 = chunk * p.chunk, i1 = i0 + p.chunk < p.T ? i0 + p.chunk : p.T;

  float R[VEC], P[GV];
#pragma unroll
  for (int v = 0; v < VEC; ++v) R[v] = 0.f, P[v % GV] = 1.f;
  if (!REDUCE) {
    const bool cut = p.flags && p.cut_off < 0 && p.T > 0 && p.done[(int64_t)e * p.done_row + (int64_t)(p.T - 1) * p.done_step];
    if (p.dlast && !cut)
#pragma unroll
      for (int v = 0; v < VEC; ++v) R[v] = ((const float*)p.dlast)[ch + v];
  }
  int buf = 0;
  if (!REDUCE && W > 1 && chunk + 1 < p.chunks) {  // the chunks behind this one, last first: each wave composes its share, then all fold the shares
    const uint32_t behind = p.chunks - 1 - chunk, each = (behind + W - 1) / W, k0 = w * each, k1 = k0 + each < behind ? k0 + each : behind;
    auto part_of = [&](uint32_t k) { return (const float*)p.part + (uint64_t)(p.chunks - 2 - k) * 2 * EC + ch; };
    float cp[GV], cs[VEC];
    bool gone[GV], far = false;
#pragma unroll
    for (int v = 0; v < VEC; ++v) cp[v % GV] = 1.f, cs[v] = 0.f, gone[v % GV] = false;
#pragma unroll 8
    for (uint32_t k = k0; k < k1; ++k) {  // bare multiply-adds, as in a tile's fold
      const float* part = part_of(k);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        cs[v] = fma_(magnitude(part[v % GV]) <= kLeast<float> ? 0.f : part[v % GV], cs[v], part[EC + v]);
        if (v < GV) cp[v] *= part[v], gone[v] |= part[v] == 0.f;
      }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) far |= !finite(cs[v]);
#pragma unroll
    for (int v = 0; v < GV; ++v) cp[v] = product(cp[v], gone[v]);
    if (rare(far)) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) cs[v] = 0.f;
      for (uint32_t k = k0; k < k1; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) cs[v] = apply(part_of(k)[v % GV], part_of(k)[EC + v], cs[v]);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) fold[0][w][v % GV][lane] = cp[v % GV], fold[0][w][GV + v][lane] = cs[v];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int v = 0; v < VEC; ++v) R[v] = apply(fold[0][k][v % GV][lane], fold[0][k][GV + v][lane], R[v]);
    buf = 1;
  }

  const uint64_t span = (uint64_t)W * kSteps, tiles = i1 > i0 ? (i1 - i0 + span - 1) / span : 0;
  for (uint64_t m = tiles; m-- > 0;) {
    const uint64_t i = i0 + m * span + (uint64_t)w * kSteps;
    const int n = i >= i1 ? 0 : i1 - i < kSteps ? (int)(i1 - i) : kSteps;  // steps of this wave's run
    Pack<X, VEC> tx[kSteps], ty[kSteps];
    Pack<G, GV> tg[kSteps];
    float from[VEC];
    Flags flags(p, e0, lane, i, n);
    if (!REDUCE)
#pragma unroll
      for (int v = 0; v < VEC; ++v) from[v] = p.saved[((n ? i : i1 - 1) / kSteps) * EC + ch + v];
    {
      const uint64_t first = n ? i : i1 - 1;
      uint64_t xs = x0 + first * x_step, gs = g0 + first * g_step, ds = dy0 + first * y_step;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {  // steps past the end read the last one that exists
        if (!REDUCE) tx[s] = load<X, VEC>(xs, x_off);
        ty[s] = load<X, VEC>(ds, y_off);
        if (MODE != kGateConst) tg[s] = load<G, GV>(gs, g_off);
        xs += s + 1 < n ? x_step : 0;
        gs += s + 1 < n ? g_step : 0;
        ds += s + 1 < n ? y_step : 0;
        hold(xs);
        hold(gs);
        hold(ds);
      }
    }
    const uint32_t cut = flags.bits(p, e, e0, i, n);
    const bool plain = n == kSteps && !flags.any;
    auto gate_of = [&](int s, int v) -> float { return MODE == kGateConst ? (float)p.decay : (float)tg[s].v[GV > 1 ? v : 0]; };
    auto cut_gate = [&](int s, int v) -> float { return (cut >> s) & 1 ? 0.f : gate_of(s, v); };
    auto forgets = [&](int v) -> bool {
      bool f = cut != 0;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) f |= s < n && gate_of(s, v) == 0.f;
      return f;
    };
    float mine[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) mine[v] = R[v];
    // As in the forward pass: a quick walk that the careful one replaces where done cuts the run or a value is not finite.
    if (W > 1 || REDUCE) {
      float rp[GV], rq[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) rp[v % GV] = 1.f, rq[v] = 0.f;
      bool odd = !plain;
      if (plain) {
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s)
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            if (v < GV) rp[v] *= gate_of(s, v);
            rq[v] = gate_of(s, v) * ((float)ty[s].v[v] + rq[v]);
          }
        bool bad = false;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          bad |= !finite(rq[v]) || !finite(rp[v % GV]);
        }
        odd = __any(bad);
      }
      if (odd) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) rp[v % GV] = 1.f, rq[v] = 0.f;
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s)
          if (s < n)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
              const float a = cut_gate(s, v);
              if (v < GV) rp[v] *= a;
              rq[v] = a == 0.f ? 0.f : a * ((float)ty[s].v[v] + rq[v]);
            }
      }
      bool ask = false;  // a product that left the range forgets all the same; and of a chunk's it is not known yet what comes into it
#pragma unroll
      for (int v = 0; v < GV; ++v) ask |= !finite(rp[v]) || (REDUCE && rp[v] == 0 && cut == 0);
      if (rare(ask))
#pragma unroll
        for (int v = 0; v < GV; ++v)
          if (REDUCE || !finite(rp[v])) rp[v] = product(rp[v], forgets(v));
#pragma unroll
      for (int v = 0; v < VEC; ++v) fold[buf][w][v % GV][lane] = rp[v % GV], fold[buf][w][GV + v][lane] = rq[v];
      if (W > 1) __syncthreads();
      float at[VEC];  // the waves' maps in turn, as in the forward pass
      float Pt[GV];
      bool far = false;
#pragma unroll
      for (int v = 0; v < VEC; ++v) at[v] = R[v], Pt[v % GV] = P[v % GV];
#pragma unroll
      for (int k = W - 1; k >= 0; --k) {
        if (k == w)
#pragma unroll
          for (int v = 0; v < VEC; ++v) mine[v] = at[v];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float Pk = fold[buf][k][v % GV][lane];
          at[v] = fma_(REDUCE && magnitude(Pk) <= kLeast<float> ? 0.f : Pk, at[v], fold[buf][k][GV + v][lane]);
          if (REDUCE && v < GV) Pt[v] *= Pk;
        }
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) far |= !finite(at[v]);
      if (rare(far)) {
        if (W > 1) __syncthreads();
        if (!REDUCE)
#pragma unroll
          for (int v = 0; v < GV; ++v) {
            float& own = fold[buf][w][v][lane];
            if (own == 0) own = product(own, forgets(v));
          }
        if (W > 1) __syncthreads();
#pragma unroll 1
        for (int k = W - 1; k >= 0; --k) {
          if (k == w)
#pragma unroll
            for (int v = 0; v < VEC; ++v) mine[v] = R[v];
#pragma unroll
          for (int v = 0; v < VEC; ++v) R[v] = apply(fold[buf][k][v % GV][lane], fold[buf][k][GV + v][lane], R[v]);
        }
      } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) R[v] = at[v];
      }
      if (REDUCE) {  // a product that becomes 0, or leaves the range, in this tile is taken once more
        bool turns = false;
#pragma unroll
        for (int v = 0; v < GV; ++v) turns |= P[v] != 0 && (Pt[v] == 0 || !finite(Pt[v]));
        if (rare(turns)) {
#pragma unroll
          for (int v = 0; v < GV; ++v) Pt[v] = P[v];
#pragma unroll
          for (int k = W - 1; k >= 0; --k)
#pragma unroll
            for (int v = 0; v < GV; ++v) Pt[v] = both(Pt[v], fold[buf][k][v][lane]);
        }
#pragma unroll
        for (int v = 0; v < GV; ++v) P[v] = P[v] == 0 ? P[v] : Pt[v];
      }
      buf ^= W > 1;
    }
    if (REDUCE) continue;
    uint64_t os = 0, qs = 0;  // where dx and dgate of the step at hand go; the walk runs backwards
    auto emit = [&](int s, const float (&gt)[VEC], const float (&k)[VEC]) {
      Pack<X, VEC> o;
#pragma unroll
      for (int v = 0; v < VEC; ++v) o.v[v] = (X)gt[v];
      store(os, y_off, o);
      os -= y_step;
      hold(os);
      if (MODE == kGateChannel) {
        Pack<G, VEC> q;
#pragma unroll
        for (int v = 0; v < VEC; ++v) q.v[v] = (G)(gt[v] * k[v]);
        store(qs, dg_off, q);
        qs -= dg_step;
        hold(qs);
      } else if (MODE == kGateHead) {
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < VEC; ++v) sum = fma_(gt[v], k[v], sum);
        terms[w][s][lane] = sum;
      }
    };
    // dgate of the run's steps: each (step, head) is added up by one lane, or by 2 or 4 where there are fewer such sums than lanes
    auto add_up = [&]() {
      const uint32_t heads = p.in_wave ? p.in_wave : 1, each = p.in_wave ? p.lanes : p.lanes - blockIdx.x % p.slabs * kWave < kWave ? p.lanes - blockIdx.x % p.slabs * kWave : kWave;
      const uint32_t split = heads == 1 ? 4 : heads == 2 ? 2 : 1, share = (each + split - 1) / split;
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (uint32_t o = lane / split; o < heads * kSteps; o += kWave / split) {
        const uint32_t s = o % kSteps, own = o / kSteps, j0 = lane % split * share, j1 = j0 + share < each ? j0 + share : each;
        float sum = 0.f;
        for (uint32_t j = j0; j < j1; ++j) sum += terms[w][s][own * each + j];
        if (split >= 2) sum += __shfl_xor(sum, 1);
        if (split == 4) sum += __shfl_xor(sum, 2);
        if (lane % split || (int)s >= n || group0 + own >= p.rows * p.heads) continue;
        const uint64_t EH = (uint64_t)p.rows * p.heads;
        if (p.slabs == 1) ((G*)p.dgate)[group0 + own + (int64_t)(i + s) * p.dgate_step] = (G)sum;
        else p.slab[(blockIdx.x % p.slabs) * p.T * EH + (i + s) * EH + group0 + own] = sum;
      }
      __builtin_amdgcn_wave_barrier();
    };
    float k[kSteps][VEC];  // the state that each step multiplies
    bool odd = !plain;
    if (plain) {
      float h[VEC], r[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[v] = from[v], r[v] = mine[v];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          k[s][v] = h[v];
          h[v] = fma_(gate_of(s, v), h[v], (float)tx[s].v[v]);
        }
      os = dx0 + (i + kSteps - 1) * y_step;
      qs = dg0 + (i + kSteps - 1) * dg_step;
#pragma unroll
      for (int s = kSteps - 1; s >= 0; --s) {
        float gt[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          gt[v] = (float)ty[s].v[v] + r[v];
          r[v] = gate_of(s, v) * gt[v];
        }
        emit(s, gt, k[s]);
      }
      bool bad = false;
#pragma unroll
      for (int v = 0; v < VEC; ++v) bad |= !finite(h[v]) || !finite(r[v]);
      odd = __any(bad);
      if (W == 1 && !odd)
#pragma unroll
        for (int v = 0; v < VEC; ++v) R[v] = r[v];
    }
    if (odd) {
      float h[VEC], r[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[v] = from[v], r[v] = mine[v];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        if (s < n)
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            k[s][v] = (cut >> s) & 1 ? 0.f : h[v];
            h[v] = step(cut_gate(s, v), h[v], (float)tx[s].v[v]);
          }
      os = dx0 + (i + (n ? n - 1 : 0)) * y_step;
      qs = dg0 + (i + (n ? n - 1 : 0)) * dg_step;
#pragma unroll
      for (int s = kSteps - 1; s >= 0; --s)
        if (s < n) {
          float gt[VEC];
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            const float a = cut_gate(s, v);
            gt[v] = (float)ty[s].v[v] + r[v];
            r[v] = a == 0.f ? 0.f : a * gt[v];
          }
          emit(s, gt, k[s]);
        }
      if (W == 1)
#pragma unroll
        for (int v = 0; v < VEC; ++v) R[v] = r[v];
    }
    if (MODE == kGateHead) add_up();
  }
  if (!live || w != 0) return;
  if (REDUCE) {
    float* part = (float*)p.part + (uint64_t)blockIdx.y * 2 * EC + ch;
#pragma unroll
    for (int v = 0; v < VEC; ++v) part[v] = P[v % GV], part[EC + v] = R[v];
  } else if (p.dstate && chunk == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) ((float*)p.dstate)[ch + v] = R[v];
  }
}

// [slabs][T][E][H] partial sums -> dgate, in slab order; `i` counts processed steps
template <class G> __global__ __launch_bounds__(256) void k_scan_grad_slabs(ScanParams p) {
  const uint64_t EH = (uint64_t)p.rows * p.heads, n = p.T * EH;
  for (uint64_t j = (uint64_t)blockIdx.x * 256 + threadIdx.x; j < n; j += (uint64_t)gridDim.x * 256) {
    float sum = p.slab[j];
    for (uint32_t s = 1; s < p.slabs; ++s) sum += p.slab[(uint64_t)s * n + j];
    ((G*)p.dgate)[j % EH + (int64_t)(j / EH) * p.dgate_step] = (G)sum;
  }
}

template <class X, class G, int MODE, int VEC, int W> static hipError_t waves(const ScanParams& p, uint32_t x, hipStream_t stream) {
  if (p.chunks > 1) {
    k_scan_grad<X, G, MODE, VEC, W, true><<<dim3(x, p.chunks - 1), W * kWave, 0, stream>>>(p);
    if (hipError_t e = hipGetLastError()) return e;
  }
  k_scan_grad<X, G, MODE, VEC, W, false><<<dim3(x, p.chunks), W * kWave, 0, stream>>>(p);
  return hipGetLastError();
}

template <class X, class G, int MODE, int VEC> static hipError_t go(const ScanParams& p, hipStream_t stream) {
  // heads of a wave's lanes or fewer lie side by side in it, a wider one takes whole waves
  const uint64_t columns = MODE != kGateHead ? ((uint64_t)p.cols + kWave - 1) / kWave
                         : p.in_wave       ? ((uint64_t)p.rows * p.heads + p.in_wave - 1) / p.in_wave
                                           : (uint64_t)p.rows * p.heads * p.slabs;
  const uint32_t x = (uint32_t)columns;
  if (p.waves == 1) k_scan_grad<X, G, MODE, VEC, 1, false><<<x, kWave, 0, stream>>>(p);
  else if (hipError_t e = p.waves == 4 ? waves<X, G, MODE, VEC, 4>(p, x, stream) : waves<X, G, MODE, VEC, 8>(p, x, stream)) return e;
  if (hipError_t e = hipGetLastError()) return e;
  if (MODE == kGateHead && p.slabs > 1 && p.T > 0) {
    const uint64_t n = p.T * (uint64_t)p.rows * p.heads, blocks = (n + 255) / 256;
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
