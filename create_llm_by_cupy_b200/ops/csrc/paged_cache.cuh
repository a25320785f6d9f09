// What the kernels of the paged cache share: how rows of K and V are held, and where they stand.
//
// A pool [pages, KV heads, page, D] per K and V; a sequence's tokens lie in the pages that its row of the table names, token t in row
// t % page of page table[t / page]. Rows are bf16, or 8 bits with one fp32 scale per token and head ([pages, KV heads, page]):
//   scale = max(largest |x| (1 / L), 2^-80), L = 127 (int8) or 448 (e4m3), 1 / L rounded; held = x / scale, rounded to nearest even.
// One scale per row is what a decoded token can be written with, without a look at its neighbours. The floor of the scale keeps
// reciprocals and logarithms of it finite; a row of zeros gets it.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace b200 {

constexpr int kHeldBf16 = 0, kHeldInt8 = 1, kHeldE4m3 = 2;
constexpr float kLeastScale = 8.2718061e-25f;      // 2^-80

struct PagedPool {
  void* k;
  void* v;
  float* ks;             // scales, null for bf16
  float* vs;
  const int* table;      // [B, width]
  int B, width, pages, KVH, log_page;
  __host__ __device__ int page() const { return 1 << log_page; }
  __host__ __device__ long long tokens() const { return (long long)width << log_page; }      // room of a sequence
};

#ifdef __CUDACC__
// Row (of all heads of all pages) in which token t of sequence b stands with KV head h; -1: its page is none of the pool.
__device__ __forceinline__ long long paged_row(const PagedPool& c, int b, int h, int t) {
  const int pg = c.table[(long long)b * c.width + (t >> c.log_page)];
  if (pg < 0 || pg >= c.pages) return -1;
  return (((long long)pg * c.KVH + h) << c.log_page) + (t & (c.page() - 1));
}

// One product with the rounded 1 / L, as every form of the framework takes it (and torch on a GPU, where it divides by a number): pools of
// all of them are the same bit for bit. A division differs from it in the last place of 5 % of int8 and 55 % of e4m3 scales, and in which
// of its two neighbours an e4m3 value halfway between them becomes, 1 in 1000; a row is represented equally well.
template <int kHeld>
__device__ __forceinline__ float held_scale(float largest) {
  return fmaxf(__fmul_rn(largest, kHeld == kHeldInt8 ? 1.f / 127.f : 1.f / 448.f), kLeastScale);
}

// x / s correctly rounded, given inv = 1 / s correctly rounded: Markstein's theorem (IBM J. Res. Dev. 34, 1990). A product with the
// reciprocal alone went the other way at one e4m3 value in 600 of rows that come from bf16, whose quotients often lie halfway.
__device__ __forceinline__ float quotient(float x, float s, float inv) {
  const float q = __fmul_rn(x, inv);
  return __fmaf_rn(__fmaf_rn(-q, s, x), inv, q);
}

// Four values as they are held, the first in the lowest byte, given the scale and its reciprocal.
template <int kHeld>
__device__ __forceinline__ uint32_t held_word(float a, float b, float c, float d, float s, float inv) {
  a = quotient(a, s, inv);
  b = quotient(b, s, inv);
  c = quotient(c, s, inv);
  d = quotient(d, s, inv);
  if constexpr (kHeld == kHeldInt8) {
    // from 2^23 + 2^22 on the last place of a float is 1: the sum rounds to the nearest even integer, whose low byte is the number
    const float big = 12582912.f;
    const uint32_t x = __float_as_uint(__fadd_rn(a, big)), y = __float_as_uint(__fadd_rn(b, big));
    const uint32_t z = __float_as_uint(__fadd_rn(c, big)), w = __float_as_uint(__fadd_rn(d, big));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
}

// Pairs of held bytes (the low two of `w`, or the high two) as exact fp16 pairs. int8 comes with its sign bit turned over: the byte
// u = x + 128 in the last bits of 1024, minus 1152.
template <int kHeld, bool kHigh>
__device__ __forceinline__ uint32_t half2_of(uint32_t w) {
  if constexpr (kHeld == kHeldInt8) {
    const uint32_t x = __byte_perm(w, 0x64646464u, kHigh ? 0x4342 : 0x4140);
    uint32_t y;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
    return y;
  } else {
    uint32_t y;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(y) : "h"(uint16_t(kHigh ? w >> 16 : w)));
    return y;
  }
}

__device__ __forceinline__ float2 float2_of_half2(uint32_t h) {
  float2 f;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
  return f;
}

__device__ __forceinline__ float2 float2_of_bf162(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

__device__ __forceinline__ uint32_t bf162_of(float a, float b) {
  const bf162 x = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&x);
}

// The two rotated values of a pair (x at d < D / 2, y at d + D / 2); each product is rounded, so that every kernel that writes a row
// writes the same.
__device__ __forceinline__ void rotate_pair(float& x, float& y, float c, float s) {
  const float a = x, b = y;
  x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  y = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}
#endif

// Why a pool is not one, or null.
inline const char* paged_pool_wrong(const PagedPool& c, int held, int D) {
  if (held < 0 || held > 2 || (D != 64 && D != 128)) return "type or head dimension";
  if (c.B < 0 || c.width < 1 || c.pages < 1 || c.KVH < 1 || c.log_page < 5 || c.log_page > 10) return "sizes";
  if (c.tokens() > 0x7fffffffLL) return "tokens";
  if (c.k == nullptr || c.v == nullptr || c.table == nullptr || (held != kHeldBf16) != (c.ks != nullptr && c.vs != nullptr))
    return "pointers";
  for (const void* x : {c.k, c.v, (void*)c.ks, (void*)c.vs})
    if ((reinterpret_cast<uintptr_t>(x) & 15) != 0) return "alignment";
  return nullptr;
}

}  // namespace b200
