// Rows of K and V into the pages of a cache, and tokens back out of it (paged_cache.cuh says how they are held).
//
// Both are one pass over the data with nothing to reuse, bound by HBM: 16 bytes of bf16 to a thread, all lanes of a row beside one
// another.
#include "paged_cache.cuh"

namespace b200 {

struct AppendParams {
  PagedPool c;
  const bf16* k;               // [M, KVH, D], pitches ldk and head D
  const bf16* v;
  const int* seq;              // [M]
  const int* pos;
  const float* cosr;           // [rows, D / 2], null: K as it is
  const float* sinr;
  long long ldk, ldv, M;
  int rows;
};

// One row of K or V for each D / 8 lanes. A row is left out when its sequence, position or page is none of the cache.
template <int D, int kHeld>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
  constexpr int kLanes = D / 8, kHalf = kLanes / 2;
  pdl_wait();
  pdl_trigger();
  const long long item = (long long)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const long long per = 2LL * p.c.KVH;
  const long long m = item / per;
  const int what = int(item - m * per), h = what >> 1;
  const bool is_v = what & 1;
  float x[8];
  long long row = -1;
  int t = 0;
  if (m < p.M) {
    const int b = p.seq[m];
    t = p.pos[m];
    if (b >= 0 && b < p.c.B && t >= 0 && t < p.c.tokens() && (p.cosr == nullptr || t < p.rows)) row = paged_row(p.c, b, h, t);
  }
  if (row >= 0) {
    const uint4 u = *reinterpret_cast<const uint4*>((is_v ? p.v + m * p.ldv : p.k + m * p.ldk) + h * D + lane * 8);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = float2_of_bf162(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
  }
  if (p.cosr != nullptr) {       // every lane takes part in the exchange; a lane holds one half of eight pairs
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl_xor_sync(0xffffffffu, x[i], kHalf);
    if (row >= 0 && !is_v) {
      const long long at = (long long)t * (D / 2) + (lane % kHalf) * 8;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float4 c = *reinterpret_cast<const float4*>(p.cosr + at + 4 * q), s = *reinterpret_cast<const float4*>(p.sinr + at + 4 * q);
        const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float lo = lane < kHalf ? x[4 * q + i] : y[4 * q + i], hi = lane < kHalf ? y[4 * q + i] : x[4 * q + i];
          rotate_pair(lo, hi, cs[i], sn[i]);
          x[4 * q + i] = lane < kHalf ? lo : hi;
        }
      }
    }
  }
  if constexpr (kHeld == kHeldBf16) {
    if (row >= 0)
      *reinterpret_cast<uint4*>(static_cast<bf16*>(is_v ? p.c.v : p.c.k) + row * D + lane * 8) =
          make_uint4(bf162_of(x[0], x[1]), bf162_of(x[2], x[3]), bf162_of(x[4], x[5]), bf162_of(x[6], x[7]));
  } else {
    float largest = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(x[i]));
#pragma unroll
    for (int o = kHalf; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    if (row >= 0) {
      const float scale = held_scale<kHeld>(largest), inv = __frcp_rn(scale);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_v ? p.c.v : p.c.k) + row * D + lane * 8) =
          make_uint2(held_word<kHeld>(x[0], x[1], x[2], x[3], scale, inv), held_word<kHeld>(x[4], x[5], x[6], x[7], scale, inv));
      if (lane == 0) (is_v ? p.c.vs : p.c.ks)[row] = scale;
    }
  }
}

struct ReadParams {
  PagedPool c;
  bf16* k;                     // [B, KVH, Tmax, D]
  bf16* v;
  const int* start;            // [B], null: 0
  const int* lens;             // [B]
  int Tmax;
};

// Eight values to a thread; grid (groups of rows, KVH, 2 B).
template <int D, int kHeld>
__global__ void __launch_bounds__(256) paged_read_kernel(const ReadParams p) {
  constexpr int kLanes = D / 8;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.z >> 1, h = blockIdx.y;
  const bool is_v = blockIdx.z & 1;
  const int i = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const long long from = p.start != nullptr ? max(p.start[b], 0) : 0, upto = min((long long)p.lens[b], p.c.tokens());
  if (i >= p.Tmax || from + i >= upto) return;
  const long long row = paged_row(p.c, b, h, int(from) + i);
  if (row < 0) return;
  uint4 out;
  if constexpr (kHeld == kHeldBf16) {
    out = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(is_v ? p.c.v : p.c.k) + row * D + lane * 8);
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(is_v ? p.c.v : p.c.k) + row * D + lane * 8);
    const float s = (is_v ? p.c.vs : p.c.ks)[row];
    uint32_t w[2] = {u.x, u.y}, o[4];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (kHeld == kHeldInt8) w[q] ^= 0x80808080u;
      const float2 lo = float2_of_half2(half2_of<kHeld, false>(w[q])), hi = float2_of_half2(half2_of<kHeld, true>(w[q]));
      o[2 * q] = bf162_of(lo.x * s, lo.y * s);
      o[2 * q + 1] = bf162_of(hi.x * s, hi.y * s);
    }
    out = make_uint4(o[0], o[1], o[2], o[3]);
  }
  *reinterpret_cast<uint4*>((is_v ? p.v : p.k) + ((long long)(b * p.c.KVH + h) * p.Tmax + i) * D + lane * 8) = out;
}

static PagedPool make_pool(void* k, void* v, void* ks, void* vs, const void* table, int B, int width, int pages, int KVH, int log_page) {
  PagedPool c;
  c.k = k;
  c.v = v;
  c.ks = static_cast<float*>(ks);
  c.vs = static_cast<float*>(vs);
  c.table = static_cast<const int*>(table);
  c.B = B; c.width = width; c.pages = pages; c.KVH = KVH; c.log_page = log_page;
  return c;
}

static bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

}  // namespace b200

using namespace b200;

// k, v [M] rows of [KVH, D] bf16, pitches ldk and ldv (multiples of 8); seq, pos [M]; cosr, sinr [rows, D / 2] or null. held: 0 bf16, 1
// int8, 2 e4m3.
B200_API int b200_paged_append(const void* k, const void* v, void* pk, void* pv, void* ks, void* vs, const void* table, const void* seq,
                               const void* pos, const void* cosr, const void* sinr, int rows, long long M, long long ldk, long long ldv,
                               int B, int width, int pages, int KVH, int log_page, int D, int held, cudaStream_t st) {
  AppendParams p;
  p.c = make_pool(pk, pv, ks, vs, table, B, width, pages, KVH, log_page);
  if (paged_pool_wrong(p.c, held, D) != nullptr || M < 0 || ldk % 8 != 0 || ldv % 8 != 0 || (cosr == nullptr) != (sinr == nullptr) ||
      !aligned16(k) || !aligned16(v) || !aligned16(cosr) || !aligned16(sinr) || (cosr != nullptr && rows < 1))
    return static_cast<int>(cudaErrorInvalidValue);
  if (M == 0 || B == 0) return 0;
  p.k = static_cast<const bf16*>(k);
  p.v = static_cast<const bf16*>(v);
  p.seq = static_cast<const int*>(seq);
  p.pos = static_cast<const int*>(pos);
  p.cosr = static_cast<const float*>(cosr);
  p.sinr = static_cast<const float*>(sinr);
  p.ldk = ldk; p.ldv = ldv; p.M = M; p.rows = rows;
  const long long per = 256 / (D / 8), blocks = (M * 2 * KVH + per - 1) / per;
  if (blocks > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
  auto go = [&](auto kern) { return static_cast<int>(launch_pdl(kern, dim3(unsigned(blocks)), dim3(256), 0, st, 0, p)); };
  if (D == 128)
    return held == kHeldBf16 ? go(paged_append_kernel<128, kHeldBf16>) : held == kHeldInt8 ? go(paged_append_kernel<128, kHeldInt8>)
                                                                                         : go(paged_append_kernel<128, kHeldE4m3>);
  return held == kHeldBf16 ? go(paged_append_kernel<64, kHeldBf16>) : held == kHeldInt8 ? go(paged_append_kernel<64, kHeldInt8>)
                                                                                      : go(paged_append_kernel<64, kHeldE4m3>);
}

// Tokens start[b] (null: 0) up to lens[b] of the pages into rows 0.. of k, v [B, KVH, Tmax, D]; other rows are left as they are.
B200_API int b200_paged_read(void* pk, void* pv, void* ks, void* vs, const void* table, const void* start, const void* lens, void* k,
                             void* v, int Tmax, int B, int width, int pages, int KVH, int log_page, int D, int held, cudaStream_t st) {
  ReadParams p;
  p.c = make_pool(pk, pv, ks, vs, table, B, width, pages, KVH, log_page);
  if (paged_pool_wrong(p.c, held, D) != nullptr || Tmax < 0 || !aligned16(k) || !aligned16(v) || B > 32767 || KVH > 65535)
    return static_cast<int>(cudaErrorInvalidValue);
  if (Tmax == 0 || B == 0) return 0;
  p.k = static_cast<bf16*>(k);
  p.v = static_cast<bf16*>(v);
  p.start = static_cast<const int*>(start);
  p.lens = static_cast<const int*>(lens);
  p.Tmax = Tmax;
  const int per = 256 / (D / 8);
  auto go = [&](auto kern) { return static_cast<int>(launch_pdl(kern, dim3((Tmax + per - 1) / per, KVH, 2 * B), dim3(256), 0, st, 0, p)); };
  if (D == 128)
    return held == kHeldBf16 ? go(paged_read_kernel<128, kHeldBf16>) : held == kHeldInt8 ? go(paged_read_kernel<128, kHeldInt8>)
                                                                                       : go(paged_read_kernel<128, kHeldE4m3>);
  return held == kHeldBf16 ? go(paged_read_kernel<64, kHeldBf16>) : held == kHeldInt8 ? go(paged_read_kernel<64, kHeldInt8>)
                                                                                    : go(paged_read_kernel<64, kHeldE4m3>);
}
