// Attention scores capped by a tanh: s -> c tanh(s scale / c), in log2 units (times log2 e).
//
// From an exponential it is exact everywhere: c tanh(y) = c - 2 c r with r = 1 / (1 + exp(2 y)); far out the exponential is 0 or
// infinite and the result -c or c. But that takes two more special-function operations per score beside the softmax's own
// exponential, which already takes as long as the products. So where no score of a tile is far out it is a polynomial on the
// FMA units, two scores per instruction: tanh(y) = y Q(y^2), Q of degree 3 for |y| <= 0.4 and of degree 6 for |y| <= 1, fitted for the
// smallest largest relative error (weighted least squares at Chebyshev nodes, Lawson's iteration): 1.0e-7 and 5.0e-8 in exact
// arithmetic, 1.5e-7 both in fp32. The last multiply also subtracts the softmax's reference maximum. A model with a cap of 50 has
// nearly all scores below 20, the first form's reach.
#pragma once
#include <stdint.h>

#include <cmath>
#include <type_traits>

namespace b200 {

constexpr int kCapNear = 0, kCapMid = 1, kCapAny = 2;

struct ScoreCap {
  float2 near[4], mid[7];       // Q's coefficients times c log2(e) (scale / c)^(2 i + 1), each twice
  float reach_near, reach_mid;  // what |s| they hold for
  float kc, c2;                 // 2 log2(e) scale / c, c log2(e)
  float2 minus_inv2;            // -1 / (c log2 e)^2, twice
};

inline ScoreCap make_score_cap(float scale, float cap) {
  static const double kNear[4] = {0.999999902, -0.333313625, 0.132709768, -0.0475536037};
  static const double kMid[7] = {0.99999995, -0.333328392, 0.133252041, -0.0534570297, 0.0202899806, -0.00620337928, 0.00104102269};
  const double kLog2e = 1.4426950408889634;
  ScoreCap c = {};
  if (!(cap > 0.f)) return c;
  double f = kLog2e * scale;                           // c log2(e) (scale / c)
  const double z = (double(scale) / cap) * (double(scale) / cap);
  for (int i = 0; i < 7; ++i, f *= z) {
    if (i < 4) c.near[i] = make_float2(float(kNear[i] * f), float(kNear[i] * f));
    c.mid[i] = make_float2(float(kMid[i] * f), float(kMid[i] * f));
  }
  // a cap so small that a coefficient is no fp32 number: the exponential form alone
  c.reach_near = std::isfinite(c.near[3].x) ? float(0.4 * double(cap) / scale) : -1.f;
  c.reach_mid = std::isfinite(c.mid[6].x) ? float(double(cap) / scale) : -1.f;
  c.kc = float(2.0 * kLog2e * scale / cap);
  c.c2 = float(kLog2e * cap);
  const float inv2 = float(-1.0 / (kLog2e * cap) / (kLog2e * cap));
  c.minus_inv2 = make_float2(inv2, inv2);
  return c;
}

#ifdef __CUDACC__
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t pair_of(float2 v) { return pair_of(v.x, v.y); }
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The capped score of s is s times this (kTier: kCapNear or kCapMid).
template <int kTier>
__device__ __forceinline__ uint64_t cap_factor(uint64_t s, const ScoreCap& c) {
  const uint64_t z = mul2(s, s);
  if constexpr (kTier == kCapNear) {
    return fma2(fma2(fma2(pair_of(c.near[3]), z, pair_of(c.near[2])), z, pair_of(c.near[1])), z, pair_of(c.near[0]));
  } else {
    uint64_t h = pair_of(c.mid[6]);
#pragma unroll
    for (int i = 5; i >= 0; --i) h = fma2(h, z, pair_of(c.mid[i]));
    return h;
  }
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

// Which form the raw scores of a warp's rows need: one answer for the warp (rows that are not `live` do not count). A NaN stays one in
// any of them.
template <int N>
__device__ __forceinline__ int cap_tier(const uint32_t (&s)[N], const ScoreCap& c, bool live = true) {
  float far[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < N; e += 2) far[(e >> 1) & 3] = max_abs3(far[(e >> 1) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
  const float m = live ? max_abs3(fmaxf(far[0], far[1]), far[2], far[3]) : 0.f;
  if (__all_sync(0xffffffffu, m <= c.reach_near)) return kCapNear;
  return __all_sync(0xffffffffu, m <= c.reach_mid) ? kCapMid : kCapAny;
}

// P = exp2(capped s - m) for raw scores [kLo, kHi) of one row, none of them masked or far out, packed to bf16 pairs in place (pair
// e / 2 lands in register e / 2, which has been consumed by then); adds to the two partial row sums.
template <int kLo, int kHi>
__device__ __forceinline__ void cap_row_p(uint32_t (&sc)[128], const ScoreCap& c, float m, float& rs0, float& rs1) {
  const uint64_t minus_m = pair_of(-m, -m);
#pragma unroll
  for (int e = kLo; e < kHi; e += 2) {
    const uint64_t s = pair_of(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1]));
    const float2 a = unpair(fma2(s, cap_factor<kCapNear>(s, c), minus_m));
    const float p0 = exp2f(a.x), p1 = exp2f(a.y);
    rs0 += p0;
    rs1 += p1;
    const __nv_bfloat162 t = __floats2bfloat162_rn(p0, p1);
    sc[e >> 1] = *reinterpret_cast<const uint32_t*>(&t);
  }
}

// The scores of a row in place, in every other case (what is masked is masked behind this).
template <int N>
__device__ __forceinline__ void cap_scores(uint32_t (&sc)[N], const ScoreCap& c, int tier) {
  auto poly = [&](auto t) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const uint64_t s = pair_of(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1]));
      const float2 y = unpair(mul2(s, cap_factor<decltype(t)::value>(s, c)));
      sc[e] = __float_as_uint(y.x);
      sc[e + 1] = __float_as_uint(y.y);
    }
  };
  if (tier == kCapNear) {
    poly(std::integral_constant<int, kCapNear>{});
  } else if (tier == kCapMid) {
    poly(std::integral_constant<int, kCapMid>{});
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) sc[e] = __float_as_uint(cap_any(__uint_as_float(sc[e]), c));
  }
}
#endif

}  // namespace b200
