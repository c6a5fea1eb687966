// What the two families of decayed linear attention (flare_decay.cu, flare_decay_tc.cu) share: one kind of work,
//
//   out_t = scale * sum_{n <= t} lambda^(t-n) (a_t . b_n) c_n   (+ scale lambda^(t+1) a_t S_0)
//
// or its mirror image in time (n >= t).  The forward is that on (q, k, v); each gradient is the same sum with the roles
// exchanged: dq on (dy, v, k), dk mirrored on (v, dy, q), dv mirrored on (k, q, dy).
#pragma once
#include "common.cuh"

namespace flare {

constexpr int kDecayUnits = 3;

struct DecayUnit {
  const void *a, *b, *c;
  void* out;
  long long as[3], bs[3], cs[3], os[3];     // element strides of b, h, n
  int Da, Dc;
  int rev;                                  // 1: the mirror image (n >= t)
  float* seg;                               // [B*H][n_seg][Da][Dc]: the sums of the segments, then the states before them
  const float* state_in;                    // [B][H][Da][Dc] or null: empty
  float* state_out;                         // or null
};

struct DecayArgs {
  int B, H, N;
  int n_seg, seg_len;                       // the token axis in segments, each a CTA's
  float scale;
  const float* log_decay;                   // [H]
  const int* lengths;                       // [B] or null: all N tokens live
  int n_units;
  DecayUnit u[kDecayUnits];
};

__device__ __forceinline__ int decay_live(const DecayArgs& a, int b) {
  return a.lengths ? max(0, min(a.N, a.lengths[b])) : a.N;
}

// lambda^n.  A decay below 2^-200 is 0 for every n > 0 in 32 bits already; bounding it there keeps lambda^0 = 1 when
// log_decay is -inf.  A NaN stays one.
__device__ __forceinline__ float decay_log2(float log_decay) {
  const float g = log_decay * kLog2e;
  return g < -200.f ? -200.f : g;
}

// S <- lambda^n S.  Where lambda^n is near 1 its distance from 1 is what has to be exact: rounded to 32 bits itself it
// would be off by up to 2^-25 a step in the same direction each time, 3e-5 after a thousand steps.
struct DecayStep {
  float keep, mul;                          // S <- mul * S + keep * S
  __device__ __forceinline__ DecayStep(float log_decay, int n) {
    const float x = fmaxf(log_decay, -140.f) * (float)n;
    const bool near_one = x > -0.5f;
    keep = near_one ? 1.f : 0.f;
    mul = near_one ? expm1f(x) : expf(x);
    if (log_decay != log_decay) mul = log_decay;
  }
  __device__ __forceinline__ float operator()(float s) const { return fmaf(mul, s, keep * s); }
};

// How the tensor-core kernels spread a call: the CTAs of a sequence (a cluster), the segments of the token axis, and the sequences
// of the last wave, if they are launched by themselves.
struct DecaySpread { int cluster, segments, rest, rest_cluster; };
bool decay_tc_supported(const DecayArgs& a, int dtype);
DecaySpread decay_tc_spread(int B, int H, int N, int Da, int Dc, int n_units);
int decay_tc(const DecayArgs& a, int dtype, const DecaySpread& spread, cudaStream_t st);
// the sums of the segments into the states before them, in place; reads state_in
void launch_decay_prefix(const DecayArgs& a, cudaStream_t st);

}  // namespace flare
