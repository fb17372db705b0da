// cp_scan.hip — the gated linear recurrence h_t = a_t h_{t-1} + x_t along the time axis of [T][E][C] planes (ce_linear_scan).
//
// A run of steps is a map h -> P h + H (P the product of its gates, H its state from zero), and runs compose, so the time
// axis can be cut wherever that helps.  A block takes 64 lanes x VEC neighbouring channels (one coalesced access a step) and W
// waves, each W-th run of kSteps steps to a wave: a wave takes its run into registers, reduces it to (P, H), the waves exchange
// these through LDS, and each walks its run once more from the state it then knows — the data are read once, and the walk that
// writes y is the plain recurrence in float, whatever the cut.  Where E * C gives too few blocks for the 256 CUs, the time
// axis is cut into chunks too: a first launch reduces every chunk to (P, H), and a chunk of the second folds those before it.
// Bound by HBM: reads x and a, writes y, 2 flops an element.  [128, 4096, 128] bfloat16, a gate a channel, takes 75-80 us, 5.1-5.4 TB/s, the rate of
// a large copy; [65537, 1, 1024] bfloat16 under 16 heads 27 + 50 (chunks, then the walk: what is left is the second
// reading of x, and the chunks ahead that every block folds).  Addresses are a wave's base in scalar registers plus a lane's 32-bit
// offset: with 64-bit addresses a lane the compiler kept one for every step, spilled, and the gradient kernel took 208 us where it takes 70
// ([512, 256, 256] bfloat16).
#include "cp_common.h"

namespace cp {

constexpr int kSteps = CE_SCAN_SAVED_STEPS;

template <class X, class G, int MODE, int VEC, int W, bool REDUCE> __global__ __launch_bounds__(kWave * W) void k_scan(ScanParams p) {
  typedef typename AccOf<X>::type A;
  constexpr int GV = MODE == kGateChannel ? VEC : 1;  // gates of a lane; its channels under one gate have one product P too
  __shared__ A fold[W > 1 ? 2 : 1][W][GV + VEC][kWave];  // P, then H
  const int lane = threadIdx.x & 63, w = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const uint32_t col = blockIdx.x * kWave + lane;
  const uint32_t colc = col < p.cols ? col : p.cols - 1;  // lanes past the end do what the last one does, and write the same
  const uint32_t e = colc / p.row_cols, c = (colc % p.row_cols) * VEC, e0 = __builtin_amdgcn_readfirstlane(e);
  const uint64_t ch = (uint64_t)colc * VEC;  // index in the dense [E][C]
  // a lane's offsets from row e0 of the strided inputs, from the wave's first channel of the dense arrays
  const uint32_t x_off = (uint32_t)((int64_t)(e - e0) * p.x_row + c) * (uint32_t)sizeof(X), y_off = (colc - blockIdx.x * kWave) * (uint32_t)(VEC * sizeof(X));
  const uint32_t g_off = MODE == kGateConst ? 0 : (uint32_t)((int64_t)(e - e0) * p.gate_row + (MODE == kGateHead ? c / p.head : c)) * (uint32_t)sizeof(G);
  const uint64_t x0 = (uint64_t)((const X*)p.x + (int64_t)e0 * p.x_row), g0 = (uint64_t)((const G*)p.gate + (int64_t)e0 * p.gate_row);
  const uint64_t y0 = (uint64_t)((X*)p.y + (uint64_t)blockIdx.x * kWave * VEC);
  const uint64_t x_step = (uint64_t)(p.x_step * (int64_t)sizeof(X)), g_step = (uint64_t)(p.gate_step * (int64_t)sizeof(G)), y_step = (uint64_t)(p.y_step * (int64_t)sizeof(X));
  const uint64_t i0 = blockIdx.y * p.chunk, i1 = i0 + p.chunk < p.T ? i0 + p.chunk : p.T;

  A h[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) h[v] = A(0);
  if (!REDUCE) {
    if (p.state)
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[v] = ((const A*)p.state)[ch + v];
  }
  int buf = 0;
  if (!REDUCE && W > 1 && blockIdx.y > 0) {  // the chunks before this one: each wave composes its share of them, then all fold the shares
    const uint64_t EC = (uint64_t)p.cols * VEC;
    const uint32_t each = (blockIdx.y + W - 1) / W, k0 = w * each, k1 = k0 + each < blockIdx.y ? k0 + each : blockIdx.y;
    auto part_of = [&](uint32_t k) { return (const A*)p.part + (uint64_t)k * 2 * EC + ch; };
    A cp[GV], cs[VEC];
    bool gone[GV], far = false;
#pragma unroll
    for (int v = 0; v < VEC; ++v) cp[v % GV] = A(1), cs[v] = A(0), gone[v % GV] = false;
#pragma unroll 8
    for (uint32_t k = k0; k < k1; ++k) {  // bare multiply-adds, as in a tile's fold
      const A* part = part_of(k);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        cs[v] = fma_(magnitude(part[v % GV]) <= kLeast<A> ? A(0) : part[v % GV], cs[v], part[EC + v]);
        if (v < GV) cp[v] *= part[v], gone[v] |= part[v] == A(0);
      }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) far |= !finite(cs[v]);
#pragma unroll
    for (int v = 0; v < GV; ++v) cp[v] = product(cp[v], gone[v]);
    if (rare(far)) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) cs[v] = A(0);
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
      for (int v = 0; v < VEC; ++v) h[v] = apply(fold[0][k][v % GV][lane], fold[0][k][GV + v][lane], h[v]);
    buf = 1;
  }
  A P[GV];  // REDUCE: the chunk's product so far
#pragma unroll
  for (int v = 0; v < GV; ++v) P[v] = A(1);

  for (uint64_t tile = i0; tile < i1; tile += (uint64_t)W * kSteps) {
    const uint64_t i = tile + (uint64_t)w * kSteps;
    const int n = i >= i1 ? 0 : i1 - i < kSteps ? (int)(i1 - i) : kSteps;  // steps of this wave's run
    Pack<X, VEC> tx[kSteps];
    Pack<G, GV> tg[kSteps];
    Flags flags(p, e0, lane, i, n);
    {
      const uint64_t first = n ? i : i1 - 1;
      uint64_t xs = x0 + first * x_step, gs = g0 + first * g_step;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {  // steps past the end read the last one that exists: every load is issued, none is waited for
        tx[s] = load<X, VEC>(xs, x_off);
        if (MODE != kGateConst) tg[s] = load<G, GV>(gs, g_off);
        xs += s + 1 < n ? x_step : 0;
        gs += s + 1 < n ? g_step : 0;
        hold(xs);
        hold(gs);
      }
    }
    uint64_t ys = y0 + i * y_step;
    const uint32_t cut = flags.bits(p, e, e0, i, n);
    const bool plain = n == kSteps && !flags.any;  // uniform: a whole run that no border cuts
    auto gate_of = [&](int s, int v) -> A { return MODE == kGateConst ? A(p.decay) : A((typename AccOf<G>::type)tg[s].v[GV > 1 ? v : 0]); };
    // The state along a run.  The quick walk is the bare multiply-add: a state that is not finite stays so to the run's end under it, and
    // then, as where done cuts the run, the careful walk takes its place, which forgets at a gate of 0.
    auto careful = [&](int s, int v, A from) -> A {
      const A a = (cut >> s) & 1 ? A(0) : gate_of(s, v);
      return step(a, from, A(tx[s].v[v]));
    };
    // whether a gate of 0, or a border, is in the run
    auto forgets = [&](int v) -> bool {
      bool f = cut != 0;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) f |= s < n && gate_of(s, v) == A(0);
      return f;
    };
    A mine[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) mine[v] = h[v];
    if (W > 1 || REDUCE) {
      A rp[GV], rh[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) rp[v % GV] = A(1), rh[v] = A(0);
      bool odd = !plain;
      if (plain) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            if (v < GV) rp[v] *= gate_of(s, v);
            rh[v] = fma_(gate_of(s, v), rh[v], A(tx[s].v[v]));
          }
        bool bad = false;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          bad |= !finite(rh[v]) || !finite(rp[v % GV]);
        }
        odd = __any(bad);
      }
      if (odd) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) rp[v % GV] = A(1), rh[v] = A(0);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          if (s < n)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
              const A a = (cut >> s) & 1 ? A(0) : gate_of(s, v);
              if (v < GV) rp[v] *= a;
              rh[v] = step(a, rh[v], A(tx[s].v[v]));
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
      for (int v = 0; v < VEC; ++v) fold[buf][w][v % GV][lane] = rp[v % GV], fold[buf][w][GV + v][lane] = rh[v];
      if (W > 1) __syncthreads();
      // The waves' maps in turn, by bare multiply-adds: what is not finite stays so to the last of them, and then apply() takes their place, over products
      // of 0 that are told apart now.  All waves fold the same maps onto the same state, so all of them take this branch or none does.
      A at[VEC];
      A Pt[GV];
      bool far = false;
#pragma unroll
      for (int v = 0; v < VEC; ++v) at[v] = h[v], Pt[v % GV] = P[v % GV];
#pragma unroll
      for (int k = 0; k < W; ++k) {
        if (k == w)
#pragma unroll
          for (int v = 0; v < VEC; ++v) mine[v] = at[v];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const A Pk = fold[buf][k][v % GV][lane];
          at[v] = fma_(REDUCE && magnitude(Pk) <= kLeast<A> ? A(0) : Pk, at[v], fold[buf][k][GV + v][lane]);
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
            A& own = fold[buf][w][v][lane];
            if (own == 0) own = product(own, forgets(v));
          }
        if (W > 1) __syncthreads();
#pragma unroll 1
        for (int k = 0; k < W; ++k) {
          if (k == w)
#pragma unroll
            for (int v = 0; v < VEC; ++v) mine[v] = h[v];
#pragma unroll
          for (int v = 0; v < VEC; ++v) h[v] = apply(fold[buf][k][v % GV][lane], fold[buf][k][GV + v][lane], h[v]);
        }
      } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = at[v];
      }
      if (REDUCE) {  // a product that becomes 0, or leaves the range, in this tile is taken once more
        bool turns = false;
#pragma unroll
        for (int v = 0; v < GV; ++v) turns |= P[v] != 0 && (Pt[v] == 0 || !finite(Pt[v]));
        if (rare(turns)) {
#pragma unroll
          for (int v = 0; v < GV; ++v) Pt[v] = P[v];
#pragma unroll
          for (int k = 0; k < W; ++k)
#pragma unroll
            for (int v = 0; v < GV; ++v) Pt[v] = both(Pt[v], fold[buf][k][v][lane]);
        }
#pragma unroll
        for (int v = 0; v < GV; ++v) P[v] = P[v] == 0 ? P[v] : Pt[v];
      }
      buf ^= W > 1;
    }
    if (REDUCE) continue;
    if (p.saved && n > 0)
#pragma unroll
      for (int v = 0; v < VEC; ++v) p.saved[(i / kSteps) * (uint64_t)p.cols * VEC + ch + v] = (float)mine[v];
    A at[VEC];
    bool odd = !plain;
    if (plain) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) at[v] = mine[v];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        Pack<X, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          at[v] = fma_(gate_of(s, v), at[v], A(tx[s].v[v]));
          o.v[v] = (X)at[v];
        }
        store(ys, y_off, o);
        ys += y_step;
        hold(ys);
      }
      bool bad = false;
#pragma unroll
      for (int v = 0; v < VEC; ++v) bad |= !finite(at[v]);
      odd = __any(bad);
    }
    if (odd) {
      ys = y0 + i * y_step;
#pragma unroll
      for (int v = 0; v < VEC; ++v) at[v] = mine[v];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        if (s < n) {
          Pack<X, VEC> o;
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            at[v] = careful(s, v, at[v]);
            o.v[v] = (X)at[v];
          }
          store(ys, y_off, o);
          ys += y_step;
          hold(ys);
        }
    }
    if (W == 1)
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[v] = at[v];
  }
  if (w != 0) return;
  if (REDUCE) {
    A* part = (A*)p.part + (uint64_t)blockIdx.y * 2 * p.cols * VEC + ch;
#pragma unroll
    for (int v = 0; v < VEC; ++v) part[v] = P[v % GV], part[(uint64_t)p.cols * VEC + v] = h[v];
  } else if (p.last && blockIdx.y + 1 == gridDim.y) {
    // forward in time the flag of the last step closes the border behind it
    const bool cut = p.flags && p.cut_off < 0 && p.T > 0 && p.done[(int64_t)e * p.done_row + (int64_t)(p.T - 1) * p.done_step];
#pragma unroll
    for (int v = 0; v < VEC; ++v) ((A*)p.last)[ch + v] = cut ? A(0) : h[v];
  }
}

template <class X, class G, int MODE, int VEC, int W> static hipError_t waves(const ScanParams& p, uint32_t x, hipStream_t stream) {
  if (p.chunks > 1) {
    k_scan<X, G, MODE, VEC, W, true><<<dim3(x, p.chunks - 1), W * kWave, 0, stream>>>(p);
    if (hipError_t e = hipGetLastError()) return e;
  }
  k_scan<X, G, MODE, VEC, W, false><<<dim3(x, p.chunks), W * kWave, 0, stream>>>(p);
  return hipGetLastError();
}

template <class X, class G, int MODE, int VEC> static hipError_t go(const ScanParams& p, hipStream_t stream) {
  const uint32_t x = (p.cols + kWave - 1) / kWave;
  if (p.waves == 1) k_scan<X, G, MODE, VEC, 1, false><<<x, kWave, 0, stream>>>(p);
  else if (hipError_t e = p.waves == 4 ? waves<X, G, MODE, VEC, 4>(p, x, stream) : waves<X, G, MODE, VEC, 8>(p, x, stream)) return e;
  return hipGetLastError();
}

template <class X, class G, int MODE> static hipError_t vecs(const ScanParams& p, int vec, hipStream_t s) {
  if (sizeof(X) == 2 && vec == 4) return go<X, G, MODE, sizeof(X) == 2 ? 4 : 1>(p, s);
  if (sizeof(X) <= 4 && vec == 2) return go<X, G, MODE, sizeof(X) <= 4 ? 2 : 1>(p, s);
  return go<X, G, MODE, 1>(p, s);
}
template <class X, class G> static hipError_t modes(const ScanParams& p, int mode, int vec, hipStream_t s) {
  if (mode == kGateConst) return vecs<X, X, kGateConst>(p, vec, s);
  if (mode == kGateChannel) return vecs<X, G, kGateChannel>(p, vec, s);
  return vecs<X, G, kGateHead>(p, vec, s);
}

hipError_t launch_scan(const ScanParams& p, int dtype, int gate_dtype, int mode, int vec, hipStream_t s) {
  const bool wide = gate_dtype == CE_F32;
  if (dtype == CE_F32) return modes<float, float>(p, mode, vec, s);
  if (dtype == CE_F64) return modes<double, double>(p, mode, vec, s);
  if (dtype == CE_BF16) return wide ? modes<bf16, float>(p, mode, vec, s) : modes<bf16, bf16>(p, mode, vec, s);
  return wide ? modes<f16, float>(p, mode, vec, s) : modes<f16, f16>(p, mode, vec, s);
}

}  // namespace cp
