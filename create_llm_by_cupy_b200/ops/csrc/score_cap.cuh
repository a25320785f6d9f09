// Attention scores capped by a tanh: s -> c tanh(s scale / c), in log2 units (times log2 e).
//
// Exact everywhere, from an exponential: c tanh(y) = c - 2 c r with r = 1 / (1 + exp(2 y)); far out the exponential is 0 or infinite
// and the result -c or c. That takes two more special-function operations per score beside the softmax's own exponential, which
// already takes as long as the products; so where no score of a tile is beyond c itself (|y| <= 1) it is a polynomial on the FMA
// units instead: tanh(y) = y Q(y^2), Q of degree 6 fitted on [0, 1] by weighted least squares at Chebyshev nodes (Lawson's
// iteration: the largest error is the smallest), at most 2e-8 off in exact arithmetic, 9e-8 in fp32. Two scores per instruction.
#pragma once
#include <stdint.h>

namespace b200 {

struct ScoreCap {
  float2 q[7];          // Q's coefficients times c log2(e) (scale / c)^(2 i + 1), each twice
  float reach;          // c / scale: the polynomial holds for |s| up to there
  float kc, c2;         // 2 log2(e) scale / c, c log2(e)
  float inv_c2;
};

inline ScoreCap make_score_cap(float scale, float cap) {
  static const double kQ[7] = {0.999999693,   -0.333321293,   0.133195836,   -0.0532658323,
                               0.0199732783, -0.00595127725, 0.000963771265};
  const double kLog2e = 1.4426950408889634;
  ScoreCap c = {};
  if (!(cap > 0.f)) return c;
  double f = kLog2e * scale;                           // c log2(e) (scale / c)
  const double z = (double(scale) / cap) * (double(scale) / cap);
  for (int i = 0; i < 7; ++i, f *= z) c.q[i] = make_float2(float(kQ[i] * f), float(kQ[i] * f));
  c.reach = cap / scale;
  c.kc = float(2.0 * kLog2e * scale / cap);
  c.c2 = float(kLog2e * cap);
  c.inv_c2 = float(1.0 / (kLog2e * cap));
  return c;
}

#ifdef __CUDACC__
__device__ __forceinline__ uint64_t pair_of(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}

// The polynomial, for two scores in place.
__device__ __forceinline__ void cap_near(uint32_t& a, uint32_t& b, const ScoreCap& c) {
  uint64_t x, z, h;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "r"(a), "r"(b));
  asm("mul.rn.f32x2 %0, %1, %1;" : "=l"(z) : "l"(x));
  h = pair_of(c.q[6]);
#pragma unroll
  for (int i = 5; i >= 0; --i) asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(h) : "l"(h), "l"(z), "l"(pair_of(c.q[i])));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(x), "l"(h));
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(x));
}

// From the exponential, for any score.
__device__ __forceinline__ float cap_any(float s, const ScoreCap& c) {
  return fmaf(-2.f * c.c2, __fdividef(1.f, 1.f + exp2f(s * c.kc)), c.c2);
}

// max(m, |a|, |b|)
__device__ __forceinline__ float max_abs3(float m, float a, float b) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
  return r;
}

// N raw scores of a row in place; which way is one answer for the warp.
template <int N>
__device__ __forceinline__ void cap_scores(uint32_t (&s)[N], const ScoreCap& c) {
  float far[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < N; e += 2) far[(e >> 1) & 3] = max_abs3(far[(e >> 1) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
  // (a NaN among them is taken by either way)
  if (__all_sync(0xffffffffu, max_abs3(fmaxf(far[0], far[1]), far[2], far[3]) <= c.reach)) {
#pragma unroll
    for (int e = 0; e < N; e += 2) cap_near(s[e], s[e + 1], c);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] = __float_as_uint(cap_any(__uint_as_float(s[e]), c));
  }
}
#endif

}  // namespace b200
