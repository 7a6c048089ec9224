// Score transforms of attention and their derivative, shared by the forward and backward kernels:
//
//   z = scale * q.k                        (the accumulator of the tensor-core product holds q.k)
//   z = cap * tanh(z / cap)                MOD & CAP
//   z = z - slope_h * |q_pos - k_pos|      MOD & BIAS
//
// all in log2 units (z * log2 e), so that a probability is one exp2 of a difference.
//
// What counts is the absolute error of z, which is a relative error of the probability; all forms below keep it under
// 2^-22 of the cap, the polynomials under 2^-22 of z too. The derivative of the capped score is 1 - tanh^2 = 1 - (z / cap)^2.
//
//   |x| <= 3/8:  tanh(x) = x Q(x^2), Q of degree 3 with the least largest error of x Q there (1.1e-8); cap and scale are in
//                the coefficients, so that five fp32 operations make z from the raw product, and no special-function one
//   |x| <= 3/4:  the same with degree 5 (1e-8), seven operations
//   beyond:      tanh(x) = 1 - 2 r with r = 1 / (1 + 2^y), y = 2 x log2 e clamped to +-60 (r is 0 or 1 to 32 bits there):
//                2^y = 2^n p(y - n) on the fp32 pipes, n the nearest integer, p of degree 5 with the least largest
//                relative error on [-1/2, 1/2] (7.5e-8), and one reciprocal
//
// A warp takes the first form that all the scores of its tile row allow (a cap of 50 leaves scores up to 18, then 37).
// With the special-function unit alone (exp2, reciprocal, and the softmax's exp2, at 16 a clock and SM) a 128 x 128 tile
// takes three times as long as its two products. Measured over the whole forward pass of 5000 rows, 16 / 8 heads, two
// documents with a prefix: 129 us without a transform, 160 with a cap, 173 with a bias, 201 with both (187, 195 and 244
// with degree 5 throughout, a loaded position and an absolute value for every score).
// NaN passes through all forms, and nothing crosses from one score to its neighbour, so masked scores, which may hold
// anything, are replaced behind the transform.
//
// MOD & SAFE is set for every transformed kernel: query rows that see no key and keys that no row sees may hold
// anything (infinities and NaN of uninitialised padding): their rows of an operand tile are overwritten with zeros in
// shared memory before a product reads them, since a zero probability times NaN is NaN. MOD == 0 is the plain kernel.
#pragma once
#include "common.cuh"

namespace tdllm {
namespace score {

constexpr int CAP = 1, BIAS = 2, SAFE = 4, REST = 8;   // REST: the forward form whose output a backward pass will use
constexpr int DEAD_KEY = -2147483647 - 1;   // code of a key that no row sees (also of padding behind the last key)

struct Mod {
  float in2;            // 2 log2(e) scale / cap
  float cap2;           // cap log2(e)
  float inv_cap2;       // 1 / cap2
  float near4, near6;   // 3/8 and 3/4 cap / scale: raw products up to here take the polynomials
  float poly4[4], poly6[6];   // z / s in powers of s^2
  const float* slope2;  // [Hq] slope_h log2(e)
  const float* q_pos;   // [nq_pad] positions as floats (exact: |position| < 2^24)
  const float* k_pos;   // [nk_pad]
};

// a position as the float that distances are taken with; one of 2^24 or more, which floats do not hold, becomes NaN, and with
// it what the rows that meet it get
__device__ __forceinline__ float position(int p) {
  return (unsigned)(p + 0xffffff) <= 2u * 0xffffff ? (float)p : __int_as_float(0x7fffffff);
}
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
__device__ __forceinline__ float clamp60(float y) {   // NaN stays NaN
  float r;
  asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, 0fC2700000;\n\tmin.NaN.f32 %0, t, 0f42700000;\n\t}" : "=f"(r) : "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t both(float v) { return pair_f32(v, v); }

// r of tanh = 1 - 2 r for two raw products
__device__ __forceinline__ void cap_r2(float s0, float s1, const Mod& m, float& r0, float& r1) {
  float y0, y1;
  unpair_f32(mul_f32x2(pair_f32(s0, s1), both(m.in2)), y0, y1);
  const uint64_t y = pair_f32(clamp60(y0), clamp60(y1));
  const uint64_t t = add_f32x2(y, both(12582912.f));              // 1.5 * 2^23: the low bits hold the integer
  const uint64_t f = fma_f32x2(add_f32x2(t, both(-12582912.f)), both(-1.f), y);
  uint64_t e = fma_f32x2(f, both(0.0013276409590616822f), both(0.009675540961325169f));
  e = fma_f32x2(e, f, both(0.05550713464617729f));
  e = fma_f32x2(e, f, both(0.24022120237350464f));
  e = fma_f32x2(e, f, both(0.6931469440460205f));
  e = fma_f32x2(e, f, both(1.0000001192092896f));
  float t0, t1, d0, d1;
  unpair_f32(t, t0, t1);
  const uint64_t p2 = pair_f32(__int_as_float((__float_as_int(t0) << 23) + 0x3f800000),
                               __int_as_float((__float_as_int(t1) << 23) + 0x3f800000));
  unpair_f32(fma_f32x2(e, p2, both(1.f)), d0, d1);
  r0 = rcp_approx(d0);
  r1 = rcp_approx(d1);
}
// A query row's side of the mask: key codes lo .. lo + range - 1, and the noisy block `grp` (a clean row has none: a
// code that no key carries). One unsigned comparison covers "code >= 0, lo <= code < hi": with lo raised to 0 at least, a
// negative code is further from it than any range reaches.
struct RowMask {
  int lo;
  unsigned range;
  int grp;
  __device__ __forceinline__ RowMask(int lo_, int hi_, int grp_)
      : lo(max(lo_, 0)), range(hi_ > max(lo_, 0) ? (unsigned)(hi_ - max(lo_, 0)) : 0u), grp(grp_ < 0 ? grp_ : DEAD_KEY + 1) {}
  __device__ __forceinline__ bool sees(int code) const { return (unsigned)code - (unsigned)lo < range || code == grp; }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// z = s P(s^2), two scores to an instruction
template <int N, int C>
__device__ __forceinline__ void cap_poly(uint32_t* s, const float* c) {
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    const uint64_t x = pair_f32(__uint_as_float(s[e]), __uint_as_float(s[e + 1]));
    const uint64_t u = mul_f32x2(x, x);
    uint64_t q = both(c[C - 1]);
#pragma unroll
    for (int i = C - 2; i >= 0; --i) q = fma_f32x2(q, u, both(c[i]));
    float z0, z1;
    unpair_f32(mul_f32x2(q, x), z0, z1);
    s[e] = __float_as_uint(z0);
    s[e + 1] = __float_as_uint(z1);
  }
}

// N raw products of one thread -> capped scores in log2 units, in place. All lanes of the warp take part.
template <int N>
__device__ __forceinline__ void cap_block(uint32_t* s, const Mod& m) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < N; e += 2) top = max3(top, fabsf(__uint_as_float(s[e])), fabsf(__uint_as_float(s[e + 1])));
  if (!__any_sync(0xffffffffu, top > m.near4)) {
    cap_poly<N, 4>(s, m.poly4);
  } else if (!__any_sync(0xffffffffu, top > m.near6)) {
    cap_poly<N, 6>(s, m.poly6);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      float r0, r1, z0, z1;
      cap_r2(__uint_as_float(s[e]), __uint_as_float(s[e + 1]), m, r0, r1);
      unpair_f32(fma_f32x2(pair_f32(r0, r1), both(-2.f * m.cap2), both(m.cap2)), z0, z1);
      s[e] = __float_as_uint(z0);
      s[e + 1] = __float_as_uint(z1);
    }
  }
}

// two scores of one head less slope * distance
__device__ __forceinline__ uint64_t less_distance(uint64_t z, float slope2, uint64_t qp, uint64_t kp) {
  float d0, d1;
  unpair_f32(fma_f32x2(kp, both(-1.f), qp), d0, d1);
  return fma_f32x2(pair_f32(fabsf(d0), fabsf(d1)), both(-slope2), z);
}

// The 64 raw products of one query row against consecutive keys -> transformed scores: in log2 units where they are capped,
// else still without the scale, which the exponent's subtraction applies; `slope` is in the same units. All lanes of the
// warp take part, with the same keys: `own` are the positions of keys lane and 32 + lane, kp(e) those of keys e .. e + 3.
//
// Positions mostly rise by one from key to key, and away from the diagonal all of a warp's rows lie behind all of the keys
// (or in front of them): then |distance| = +-(d0 - e), and no position is loaded and no absolute value taken.
template <int MOD, class KeyPos>
__device__ __forceinline__ void transform_row(uint32_t* s, const Mod& m, float slope, float qpos, float2 own, KeyPos kp) {
  constexpr int N = 64;
  if constexpr ((MOD & CAP) != 0) cap_block<N>(s, m);
  if constexpr ((MOD & BIAS) != 0) {
    const int lane = threadIdx.x & 31;
    const float k0 = __shfl_sync(0xffffffffu, own.x, 0), d0 = qpos - k0;
    const bool plain = own.x == k0 + lane && own.y == k0 + (32 + lane) && (d0 >= N - 1 || d0 <= 0.f);
    if (__all_sync(0xffffffffu, plain)) {
      const float f = d0 > 0.f ? -slope : slope;
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = __float_as_uint(fmaf(f, d0 - e, __uint_as_float(s[e])));
    } else {
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const float4 k = kp(e);
        s[e] = __float_as_uint(fmaf(-slope, fabsf(qpos - k.x), __uint_as_float(s[e])));
        s[e + 1] = __float_as_uint(fmaf(-slope, fabsf(qpos - k.y), __uint_as_float(s[e + 1])));
        s[e + 2] = __float_as_uint(fmaf(-slope, fabsf(qpos - k.z), __uint_as_float(s[e + 2])));
        s[e + 3] = __float_as_uint(fmaf(-slope, fabsf(qpos - k.w), __uint_as_float(s[e + 3])));
      }
    }
  }
}

}  // namespace score
}  // namespace tdllm

static inline tdllm::score::Mod score_mod_of(float scale, float softcap, const float* slope2, const float* q_pos,
                                             const float* k_pos) {
  const float log2e = 1.4426950408889634f;
  tdllm::score::Mod m;
  static const float q6[6] = {0.9999998211860657f, -0.33332470059394836f, 0.13320580124855042f,
                             -0.053149253129959106f, 0.01923721842467785f, -0.004493444226682186f};
  const bool cap = softcap > 0.f;
  const double in1 = cap ? (double)scale / softcap : 0.;
  m.in2 = (float)(2. * log2e * in1);
  m.cap2 = softcap * log2e;
  m.inv_cap2 = cap ? 1.f / m.cap2 : 0.f;
  // false: a coefficient is not an ordinary number of 32 bits
  auto powers = [&](const float* c, int n, float* out) {
    bool fine = cap;
    double f = m.cap2 * in1;
    for (int i = 0; i < n; ++i, f *= in1 * in1) {
      out[i] = (float)(f * c[i]);
      fine = fine && fabs(f * c[i]) > 1.2e-38 && fabs(f * c[i]) < 3.0e38;
    }
    return fine;
  };
  static const float q4[4] = {0.9999997615814209f, -0.3333083987236023f, 0.1326839178800583f, -0.04761846736073494f};
  double near4 = 0.375, near6 = 0.75;
  if (!powers(q4, 4, m.poly4)) {   // far beyond usual caps: tanh(x) = x - x^3 / 3 to 2^-26 up to 1/64, x itself up to 2^-13
    const float q2[2] = {1.f, -0.333333343f};
    const int n = powers(q2, 2, m.poly4) ? 2 : 1;
    for (int i = n; i < 4; ++i) m.poly4[i] = 0.f;
    near4 = n == 2 ? 0.015625 : 0.0001220703125;
  }
  if (!powers(q6, 6, m.poly6)) near6 = 0.;   // (never taken: near4 is larger)
  m.near4 = cap ? (float)(near4 / fabs(in1)) : 0.f;
  m.near6 = cap ? (float)(near6 / fabs(in1)) : 0.f;
  m.slope2 = slope2;
  m.q_pos = q_pos;
  m.k_pos = k_pos;
  return m;
}
