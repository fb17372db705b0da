// cp_advantage.hip — advantages and returns over the planes of a rollout (ce_advantages).
//
// A_t = delta_t + gamma lam A_{t+1}: the recurrence of cp_scan.hip run against time, its input delta_t made on the way from reward,
// value and done.  A lane owns one agent of one env (neighbouring lanes, neighbouring addresses), the W waves of a block share
// its time axis in runs of kSteps steps.  double throughout: the engine's rewards are, and V_{t+1} - V_t cancels; bound by HBM all the
// same: 64 planes of 16 384 envs x 8 agents in 34.5 us, 4.9 TB/s.  20 planes of 64 x 2 take 6.3 us, one run's chain of reads and the launch.
#include "cp_common.h"

namespace cp {

constexpr int kSteps = 16;

template <class R, class V, int W> __global__ __launch_bounds__(kWave * W) void k_advantages(ce_advantage a) {
  __shared__ double fold[2][W][2][kWave];
  const int lane = threadIdx.x & 63, w = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const uint64_t cols = a.rows * a.agents, col = (uint64_t)blockIdx.x * kWave + lane;
  const bool live = col < cols, per_agent = a.flags & CE_ADV_DONE_PER_AGENT;
  const uint64_t j = live ? col : cols - 1, dj = per_agent ? j : j / a.agents, dcols = per_agent ? cols : a.rows;
  const R* reward = (const R*)a.reward + j;
  const V* value = (const V*)a.value + j;
  const double end = a.last_value ? (double)(float)((const V*)a.last_value)[j] : 0.0, gl = a.gamma * a.lam;
  const uint64_t T = a.planes;
  auto plane = [&](uint64_t i) -> uint64_t {  // processed step i is time T - 1 - i
    const uint64_t t = a.first_plane + (T - 1 - i);
    return t < T ? t : t - T;
  };
  double h = 0;
  int buf = 0;
  for (uint64_t tile = 0; tile < T; tile += W * kSteps) {
    const uint64_t i = tile + (uint64_t)w * kSteps;
    R r[kSteps];
    V v[kSteps];
    uint8_t d[kSteps];
    double after = end;
    if (i > 0 && i < T) after = (double)(float)value[plane(i - 1) * cols];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      if (i + s < T) {
        const uint64_t pl = plane(i + s);
        r[s] = reward[pl * cols];
        v[s] = value[pl * cols];
        d[s] = a.done ? a.done[pl * dcols + dj] : 0;
      }
    double x[kSteps], rp = 1, rh = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      if (i + s < T) {
        const double now = (double)(float)v[s];
        x[s] = (double)r[s] - now + (d[s] ? 0.0 : a.gamma * after);
        after = now;
        const double g = d[s] ? 0.0 : gl;
        rp = both(rp, g);
        rh = step(g, rh, x[s]);
      }
    double mine = h;
    if (W > 1) {
      fold[buf][w][0][lane] = rp;
      fold[buf][w][1][lane] = rh;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < W; ++k) {
        if (k == w) mine = h;
        h = apply(fold[buf][k][0][lane], fold[buf][k][1][lane], h);
      }
      buf ^= 1;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      if (i + s < T) {
        mine = step(d[s] ? 0.0 : gl, mine, x[s]);
        const uint64_t at = plane(i + s) * cols + j;
        if (live && a.advantage) a.advantage[at] = (float)mine;
        if (live && a.ret) a.ret[at] = (float)(mine + (double)(float)v[s]);
      }
    if (W == 1) h = mine;
  }
}

template <class R, class V> static void go(const ce_advantage& a, hipStream_t s) {
  const uint32_t blocks = (uint32_t)((a.rows * a.agents + kWave - 1) / kWave);
  // Waves that share a block's time axis: as many as have a run, while blocks are too few to fill the chip by themselves.  us with 4 / 8 / 16 waves:
  // 64 planes x 512 blocks 12.7 / 13.3 / 19.5, 128 x 64 13.5 / 9.4 / 10.0, 187 x 256 40 / 31 / 20, 256 x 512 39 / 36 / 40, 187 x 616 53 / 64 / 57,
  // 927 x 1 92 / 55 / 40.
  if (a.planes <= kSteps) k_advantages<R, V, 1><<<blocks, kWave, 0, s>>>(a);
  else if (a.planes <= 4 * kSteps || blocks > 512) k_advantages<R, V, 4><<<blocks, 4 * kWave, 0, s>>>(a);
  else if (a.planes <= 8 * kSteps || blocks > 256) k_advantages<R, V, 8><<<blocks, 8 * kWave, 0, s>>>(a);
  else k_advantages<R, V, 16><<<blocks, 16 * kWave, 0, s>>>(a);
}
template <class R> static void values(const ce_advantage& a, hipStream_t s) {
  if (a.value_dtype == CE_F32) go<R, float>(a, s);
  else if (a.value_dtype == CE_BF16) go<R, bf16>(a, s);
  else go<R, f16>(a, s);
}

hipError_t launch_advantages(const ce_advantage& a, hipStream_t s) {
  if (a.reward_dtype == CE_F64) values<double>(a, s);
  else values<float>(a, s);
  return hipGetLastError();
}

}  // namespace cp
