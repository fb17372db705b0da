// cp_advantage.hip — advantages and returns over the planes of a rollout (ce_advantages).
//
// A_t = delta_t + gamma lam A_{t+1}: the recurrence of cp_scan.hip run against time, its input delta_t made on the way from reward,
// value and done.  A lane owns one agent of one env (neighbouring lanes, neighbouring addresses), the W waves of a block share
// its time axis in runs of kSteps steps.  double throughout: the engine's rewards are, and V_{t+1} - V_t cancels; bound by HBM all the
// same: 64 planes of 16 384 envs x 8 agents in 32 us, 5.4 TB/s.  20 planes of 64 x 2 take 6.1 us, one run's chain of reads and the launch.
#include "cp_common.h"

namespace cp {

constexpr int kSteps = 16;

template <class R, class V, int W> __global__ __launch_bounds__(kWave * W) void k_advantages(ce_advantage a) {
  __shared__ double fold[2][W][2][kWave];
  const int lane = threadIdx.x & 63, w = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const uint64_t cols = a.rows * a.agents, col = (uint64_t)blockIdx.x * kWave + lane;
  const bool per_agent = a.flags & CE_ADV_DONE_PER_AGENT;
  const uint64_t j = col < cols ? col : cols - 1, dj = per_agent ? j : j / a.agents, dcols = per_agent ? cols : a.rows;
  // A plane's base in scalar registers and a lane's 32-bit offset in it (2^28 columns of 8 bytes at most).  Without done flags the values' bytes
  // are read in their place, and dropped: a branch there made each step wait for its own read (187 planes of 616 blocks: 53 us, now
  // 33).
  const uint64_t reward = (uint64_t)a.reward, value = (uint64_t)a.value, done = (uint64_t)(a.done ? a.done : (const uint8_t*)a.value);
  const uint32_t r_off = (uint32_t)(j * sizeof(R)), v_off = (uint32_t)(j * sizeof(V)), o_off = (uint32_t)(j * sizeof(float)), ends = a.done ? 0xff : 0;
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
    const V before = load<V, 1>(value + plane(i > 0 && i < T ? i - 1 : 0) * cols * sizeof(V), v_off).v[0];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {  // steps past the end read the last one
      const uint64_t pl = plane(i + s < T ? i + s : T - 1);
      r[s] = load<R, 1>(reward + pl * cols * sizeof(R), r_off).v[0];
      v[s] = load<V, 1>(value + pl * cols * sizeof(V), v_off).v[0];
      d[s] = load<uint8_t, 1>(done + pl * dcols, (uint32_t)dj).v[0];
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) d[s] &= ends;
    float b = (float)before;
    asm volatile("" : "+v"(b));  // read with the rest, not behind a branch of its own
    if (i > 0) after = (double)b;
    double x[kSteps], rp = 1, rh = 0;
    bool ended = gl == 0;  // the run's map forgets what comes into it
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      if (i + s < T) {
        const double now = (double)(float)v[s];
        x[s] = (double)r[s] - now + (d[s] ? 0.0 : a.gamma * after);
        after = now;
        ended |= d[s] != 0;
        rp *= gl;
        rh = step(d[s] ? 0.0 : gl, rh, x[s]);
      }
    if (ended || rp == 0) rp = product(rp, ended);
    double mine = h;
    if (W > 1) {
      fold[buf][w][0][lane] = rp;
      fold[buf][w][1][lane] = rh;
      __syncthreads();
      // the waves' maps in turn, by bare multiply-adds: what is not finite stays so to the last of them, and then apply() takes their place
      double at = h;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        if (k == w) mine = at;
        const double P = fold[buf][k][0][lane];
        at = fma_(magnitude(P) <= kLeast<double> ? 0.0 : P, at, fold[buf][k][1][lane]);
      }
      if (rare(!finite(at))) {
#pragma unroll 1  // the maps are read again: kept, they would cost the 16 waves registers (187 x 16384: 14.7 us, 21.6 so)
        for (int k = 0; k < W; ++k) {
          if (k == w) mine = h;
          h = apply(fold[buf][k][0][lane], fold[buf][k][1][lane], h);
        }
      } else {
        h = at;
      }
      buf ^= 1;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      if (i + s < T) {
        mine = step(d[s] ? 0.0 : gl, mine, x[s]);
        const uint64_t at = plane(i + s) * cols * sizeof(float);  // lanes past the end do what the last one does, and write the same
        if (a.advantage) store<float, 1>((uint64_t)a.advantage + at, o_off, {(float)mine});
        if (a.ret) store<float, 1>((uint64_t)a.ret + at, o_off, {(float)(mine + (double)(float)v[s])});
      }
    if (W == 1) h = mine;
  }
}

template <class R, class V> static void go(const ce_advantage& a, hipStream_t s) {
  const uint32_t blocks = (uint32_t)((a.rows * a.agents + kWave - 1) / kWave);
  // Waves that share a block's time axis: as many as have a run, while blocks are too few to fill the chip by themselves.  us with 4 / 8 / 16 waves:
  // 64 planes x 512 blocks 13.0 / 17.2 / 20.2, 128 x 64 12.4 / 9.0 / 10.0, 187 x 256 18.2 / 15.5 / 13.6, 256 x 512 42 / 43 / 38,
  // 187 x 616 33 / 36 / 36, 927 x 1 74 / 47 / 36.
  if (a.planes <= kSteps) k_advantages<R, V, 1><<<blocks, kWave, 0, s>>>(a);
  else if (a.planes <= 4 * kSteps || blocks > 512) k_advantages<R, V, 4><<<blocks, 4 * kWave, 0, s>>>(a);
  else if (a.planes <= 8 * kSteps) k_advantages<R, V, 8><<<blocks, 8 * kWave, 0, s>>>(a);
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
