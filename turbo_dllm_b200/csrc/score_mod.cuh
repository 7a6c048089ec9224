// Score transforms of attention and their derivative, shared by the forward and backward kernels:
//
//   z = scale * q.k                        (the accumulator of the tensor-core product holds q.k)
//   z = cap * tanh(z / cap)                MOD & CAP
//   z = z - slope_h * |q_pos - k_pos|      MOD & BIAS
//
// all in log2 units (z * log2 e), so that a probability is one exp2 of a difference.
//
// tanh(x) = 1 - 2 r with r = 1 / (1 + e^(2x)): no cancellation that matters here, since what counts is the absolute
// error of z (a relative error of the probability): 2^-23 of `cap` at most, also where tanh saturates (e = inf gives
// r = 0, e = 0 gives r = 1). The derivative of the capped score, 1 - tanh^2, is 4 r (1 - r).
//
// MOD & SAFE is set for every transformed kernel: query rows that see no key and keys that no row sees may hold
// anything (infinities and NaN of uninitialised padding): their rows of an operand tile are overwritten with zeros in
// shared memory before a product reads them, since a zero probability times NaN is NaN. MOD == 0 is the plain kernel.
#pragma once
#include "common.cuh"

namespace tdllm {
namespace score {

constexpr int CAP = 1, BIAS = 2, SAFE = 4;
constexpr int DEAD_KEY = -2147483647 - 1;   // code of a key that no row sees (also of padding behind the last key)

struct Mod {
  float in2;            // 2 log2(e) scale / cap
  float cap2;           // cap log2(e)
  const float* slope2;  // [Hq] slope_h log2(e)
  const float* q_pos;   // [nq_pad] positions as floats (exact: |position| < 2^24)
  const float* k_pos;   // [nk_pad]
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// r of tanh = 1 - 2 r for a raw product s
__device__ __forceinline__ float cap_r(float s, const Mod& m) { return rcp_approx(1.f + exp2_approx(s * m.in2)); }
__device__ __forceinline__ float cap_z(float r, const Mod& m) { return fmaf(-2.f * m.cap2, r, m.cap2); }
__device__ __forceinline__ float cap_slope(float r) { return 4.f * r * (1.f - r); }

}  // namespace score
}  // namespace tdllm

static inline tdllm::score::Mod score_mod_of(float scale, float softcap, const float* slope2, const float* q_pos,
                                             const float* k_pos) {
  const float log2e = 1.4426950408889634f;
  tdllm::score::Mod m;
  m.in2 = softcap > 0.f ? 2.f * log2e * scale / softcap : 0.f;
  m.cap2 = softcap * log2e;
  m.slope2 = slope2;
  m.q_pos = q_pos;
  m.k_pos = k_pos;
  return m;
}
