// cp_common.h — what the policy operators' kernels share: element types, the fold of a recurrence, launch parameters.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/contracts_policy.h"

namespace cp {

typedef __bf16 bf16;
typedef _Float16 f16;
constexpr int kWave = 64;

// A lane's run of N neighbouring elements, moved as one access (the host picks N by the alignment of every array involved).  Addresses are a
// base that the whole wave shares (scalar registers) and a lane's own 32-bit offset in bytes, so walking the time axis costs no
// vector arithmetic; `hold` keeps a running base a running base, where the compiler would rather keep one for every step.
template <class T, int N> struct alignas(sizeof(T) * N) Pack {
  T v[N];
};
template <int BYTES> struct Raw;
template <> struct Raw<1> { typedef uint8_t type; };
template <> struct Raw<2> { typedef uint16_t type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <> struct Raw<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };
#define CP_GLOBAL __attribute__((address_space(1)))

template <class T, int N> __device__ __forceinline__ Pack<T, N> load(uint64_t base, uint32_t off) {
  typedef typename Raw<sizeof(T) * N>::type R;
  return __builtin_bit_cast(Pack<T, N>, *(const CP_GLOBAL R*)(base + off));
}
template <class T, int N> __device__ __forceinline__ void store(uint64_t base, uint32_t off, const Pack<T, N>& v) {
  typedef typename Raw<sizeof(T) * N>::type R;
  *(CP_GLOBAL R*)(base + off) = __builtin_bit_cast(R, v);
}
__device__ __forceinline__ void hold(uint64_t& base) { asm volatile("" : "+s"(base)); }

template <class T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };

__device__ __forceinline__ float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Whether a lane asks for what hardly ever happens; its code lies out of the way.
__device__ __forceinline__ bool rare(bool lane) { return __builtin_expect(__any(lane) != 0, 0); }

// One step of the recurrence.  A gate of 0 (done flags arrive as one) forgets the state, infinities and NaN included, where a plain
// product would give NaN.
template <class A> __device__ __forceinline__ A step(A a, A h, A x) { return a == A(0) ? x : __builtin_fma(a, h, x); }
template <> __device__ __forceinline__ float step(float a, float h, float x) { return a == 0.f ? x : __builtin_fmaf(a, h, x); }

// A run of steps as a map of the state before it: h -> P h + H, P the product of its gates.  P = 0 says that a gate of the run is 0 (or done closed a
// border in it) and forgets the state, infinities and NaN included.  A product that merely falls under the type's range is held as the
// smallest number there is, with its sign: it takes nothing of a finite state, but an infinity or NaN shows behind the run as it would step by step.
// Folds run by bare multiply-adds first, which are right while everything is finite (a product of 0 and one under the range are then the same), and what is
// not finite stays so to their end; apply() takes their place then.  (Everywhere, it cost a split scan 5 %: [512, 256, 256] both passes 118 -> 124 us.)
template <class A> __device__ constexpr A kLeast = 0;
template <> __device__ constexpr float kLeast<float> = 0x1p-149f;
template <> __device__ constexpr double kLeast<double> = 0x1p-1074;
__device__ __forceinline__ float magnitude(float a) { return __builtin_fabsf(a); }
__device__ __forceinline__ double magnitude(double a) { return __builtin_fabs(a); }
__device__ __forceinline__ float least_of_sign(float a) { return __builtin_copysignf(kLeast<float>, a); }
__device__ __forceinline__ double least_of_sign(double a) { return __builtin_copysign(kLeast<double>, a); }
// A zero state takes no part, so that a product past the type's range (gates over 1) does not turn it into NaN.
template <class A> __device__ __forceinline__ A apply(A P, A H, A h) {
  const bool least = magnitude(P) <= kLeast<A>;  // 0 too
  const bool nothing = (h == A(0)) | (P == A(0)) | (least & __builtin_isfinite(h));
  return nothing ? H : fma_(P, h, H);
}
// P of a run whose gates' product is `r`, one of which was 0 (past the type's range too, where the product is NaN) or not.
template <class A> __device__ __forceinline__ A product(A r, bool forgets) { return forgets ? A(0) : r == A(0) ? least_of_sign(r) : r; }
// The product of two such P: one of 0 forgets whatever the other is, past the type's range too (0 times infinity would be NaN).
template <class A> __device__ __forceinline__ A both(A P, A Q) { return product(P * Q, P == A(0) || Q == A(0)); }

// Done flags of a wave's run of 16 steps as 16 bits a lane.  A wave spans at most 4 rows where a row has 21 lanes or more: then each
// quarter of the lanes reads one row's 16 flags with a single access and a ballot spreads them (kFlags4).  Up to 16 rows (5 lanes and more)
// take four such accesses of 4 steps (kFlags16), still shorter rows one a step in every lane (kFlagsLane).
enum FlagMode { kFlagsNone = 0, kFlags4 = 1, kFlags16 = 2, kFlagsLane = 3 };

struct ScanParams {
  uint64_t T;
  uint32_t cols;      // E * C / VEC: columns of VEC channels
  uint32_t row_cols;  // C / VEC
  uint64_t chunk;     // steps of one block (a multiple of every tile), T where the time axis is not split
  uint32_t chunks;
  uint32_t waves;     // waves of a block
  uint32_t head;      // channels under one gate
  uint32_t rows;      // E
  int32_t flags;      // FlagMode
  int32_t cut_off;    // the flag that cuts the state ahead of processed step i is done[i + cut_off]
  int64_t x_step, x_row, gate_step, gate_row, done_step, done_row, y_step;  // in processing order (steps may be negative)
  double decay;
  const void* x;
  const void* gate;
  const uint8_t* done;
  const void* state;
  void* y;
  void* last;
  float* saved;
  void* part;         // [chunks][2][E * C]: product and state of each chunk
  // backward pass
  const void* dy;
  const void* dlast;
  void* dx;
  void* dgate;
  void* dstate;
  int64_t dgate_step;
  uint32_t heads;
  uint32_t lanes;     // backward pass, gates shared by a head: lanes of a head (head / VEC)
  uint32_t in_wave;   // whole heads side by side in a wave (0: a head takes `slabs` waves)
  uint32_t slabs;     // partial sums a head's gradient is made of
  float* slab;        // [slabs][T][E][H] where slabs > 1
};

// The done flags that cut the state ahead of the n steps i, i + 1, .. of a wave's run; a flag ahead of the first step (index -1, forward
// in time) or past the run cuts nothing.  What ballots spread is read with the run's other loads, long before bits() asks.
struct Flags {
  uint8_t d[4] = {0, 0, 0, 0};
  bool any = false;
  static __device__ __forceinline__ uint8_t at(const ScanParams& p, uint32_t row, uint64_t i, int s, int n) {
    const uint64_t flag = i + s + (int64_t)p.cut_off;
    return s < n && flag < p.T && row < p.rows ? p.done[(int64_t)row * p.done_row + (int64_t)flag * p.done_step] : 0;
  }
  __device__ __forceinline__ Flags(const ScanParams& p, uint32_t e0, int lane, uint64_t i, int n) {
    if (p.flags == kFlags4) {
      d[0] = at(p, e0 + (lane >> 4), i, lane & 15, n);
    } else if (p.flags == kFlags16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = at(p, e0 + (lane >> 2), i, 4 * j + (lane & 3), n);
    }
  }
  __device__ __forceinline__ uint32_t bits(const ScanParams& p, uint32_t e, uint32_t e0, uint64_t i, int n) {
    uint32_t cut = 0;
    if (p.flags == kFlags4) {
      const uint64_t m = __ballot(d[0] != 0);
      any = m != 0;
      cut = (uint32_t)(m >> ((e - e0) * 16)) & 0xffffu;
    } else if (p.flags == kFlags16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t m = __ballot(d[j] != 0);
        any |= m != 0;
        cut |= ((uint32_t)(m >> ((e - e0) * 4)) & 0xfu) << (4 * j);
      }
    } else if (p.flags == kFlagsLane && n > 0) {
      const uint64_t row = (uint64_t)(p.done + (int64_t)e * p.done_row);
      uint8_t f[16];
#pragma unroll
      for (int s = 0; s < 16; ++s) {  // which flag is the same for the whole wave: one that does not count is another's, and dropped below
        const uint64_t flag = i + (s < n ? s : 0) + (int64_t)p.cut_off;
        uint64_t off = (flag < p.T ? flag : 0) * (uint64_t)p.done_step;
        hold(off);
        f[s] = *(const CP_GLOBAL uint8_t*)(row + off);
      }
#pragma unroll
      for (int s = 0; s < 16; ++s) cut |= (f[s] != 0 ? 1u : 0u) << s;
      const uint32_t ahead = i + (int64_t)p.cut_off < p.T ? 0u : 1u;  // the flag ahead of the first step
      cut &= ((1u << n) - 1u) & ~ahead;
      any = __any(cut != 0);
    }
    return cut;
  }
};

template <class A> __device__ __forceinline__ bool finite(A a) { return __builtin_isfinite(a); }

enum GateMode { kGateConst = 0, kGateChannel = 1, kGateHead = 2 };

hipError_t launch_scan(const ScanParams& p, int dtype, int gate_dtype, int mode, int vec, hipStream_t stream);
hipError_t launch_scan_grad(const ScanParams& p, int dtype, int gate_dtype, int mode, int vec, hipStream_t stream);
hipError_t launch_advantages(const ce_advantage& a, hipStream_t stream);
hipError_t launch_logits(const ce_logits& s, hipStream_t stream);
hipError_t launch_logits_grad(const ce_logits& s, const ce_logits_grad& g, hipStream_t stream);
uint64_t logits_grad_workspace(const ce_logits& s, const ce_logits_grad& g);

}  // namespace cp
