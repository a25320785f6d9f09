// Rows of K and V into the pages of a cache, and tokens back out of it (paged_cache.cuh says how they are held).
//
// Both are one pass over the data with nothing to reuse: 16 bytes to a load, all lanes of a row beside one another, two rows to a thread
// so that enough is on its way. Reading is bound by HBM, writing by the trips that follow one another (sequence and position, page,
// angles): it waits for its loads at 16 % of DRAM. int8, 8 KV heads of 128, 4096 tokens written and read back, in two launches: 20 us;
// with 8 bytes of one row to a thread 24.4, with four heads and four rows 22.5, with one head 24.3, with eight rows 23.9. 8 x 2000 to 4000
// e4m3 tokens read: 29.2 us, 5.1 TB/s (38.4, and 30.7 with four rows, 34.1 with eight).
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

// D / 8 lanes for a token's K (or V) of two heads, whose loads are all on their way before the first is used: its place and its angles are
// looked up once for them. A row is left out when its sequence, position or page is none of the cache.
constexpr int kAppendHeads = 2;

template <int D, int kHeld>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
  constexpr int kLanes = D / 8, kHalf = kLanes / 2;
  pdl_wait();
  pdl_trigger();
  const unsigned item = blockIdx.x * unsigned(256 / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const unsigned blocks = (p.c.KVH + kAppendHeads - 1) / kAppendHeads, per = 2 * blocks, m = item / per, what = item - m * per;
  const bool is_v = what >= blocks;
  const int h0 = int(is_v ? what - blocks : what) * kAppendHeads, heads = min(p.c.KVH - h0, kAppendHeads);
  uint4 in[kAppendHeads];
  int b = -1, t = 0;
  if (m < p.M) {
    const bf16* from = (is_v ? p.v + m * p.ldv : p.k + m * p.ldk) + h0 * D + lane * 8;
#pragma unroll
    for (int h = 0; h < kAppendHeads; ++h) in[h] = *reinterpret_cast<const uint4*>(from + (h < heads ? h : 0) * D);
    b = p.seq[m];
    t = p.pos[m];
  }
  const bool turns = p.cosr != nullptr && !is_v;
  long long row = -1;
  if (b >= 0 && b < p.c.B && t >= 0 && t < p.c.tokens() && (p.cosr == nullptr || t < p.rows)) row = paged_row(p.c, b, h0, t);
  float cs[8], sn[8];
  if (turns && row >= 0) {
    const long long at = (long long)t * (D / 2) + (lane % kHalf) * 8;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 c = *reinterpret_cast<const float4*>(p.cosr + at + 4 * q), s = *reinterpret_cast<const float4*>(p.sinr + at + 4 * q);
      cs[4 * q] = c.x; cs[4 * q + 1] = c.y; cs[4 * q + 2] = c.z; cs[4 * q + 3] = c.w;
      sn[4 * q] = s.x; sn[4 * q + 1] = s.y; sn[4 * q + 2] = s.z; sn[4 * q + 3] = s.w;
    }
  }
#pragma unroll
  for (int h = 0; h < kAppendHeads; ++h) {                   // all lanes take part in the exchanges
    const bool there = row >= 0 && h < heads;
    const long long at = row + ((long long)h << p.c.log_page);
    float x[8];
    const uint32_t w[4] = {in[h].x, in[h].y, in[h].z, in[h].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = there ? float2_of_bf162(w[i]) : make_float2(0.f, 0.f);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
    if (p.cosr != nullptr) {                                 // a lane holds one half of eight pairs
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __shfl_xor_sync(0xffffffffu, x[i], kHalf);
        float lo = lane < kHalf ? x[i] : y, hi = lane < kHalf ? y : x[i];
        if (turns && there) {
          rotate_pair(lo, hi, cs[i], sn[i]);
          x[i] = lane < kHalf ? lo : hi;
        }
      }
    }
    if constexpr (kHeld == kHeldBf16) {
      if (there)
        *reinterpret_cast<uint4*>(static_cast<bf16*>(is_v ? p.c.v : p.c.k) + at * D + lane * 8) =
            make_uint4(bf162_of(x[0], x[1]), bf162_of(x[2], x[3]), bf162_of(x[4], x[5]), bf162_of(x[6], x[7]));
    } else {
      float largest = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(x[i]));
#pragma unroll
      for (int o = kHalf; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
      if (there) {
        const float scale = held_scale<kHeld>(largest), inv = __frcp_rn(scale);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_v ? p.c.v : p.c.k) + at * D + lane * 8) =
            make_uint2(held_word<kHeld>(x[0], x[1], x[2], x[3], scale, inv), held_word<kHeld>(x[4], x[5], x[6], x[7], scale, inv));
        if (lane == 0) (is_v ? p.c.vs : p.c.ks)[at] = scale;
      }
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

// 16 bytes of two rows to a thread, both on their way before the first is used; grid (groups of rows, KVH, 2 B).
constexpr int kReadRows = 2;

template <int D, int kHeld>
__global__ void __launch_bounds__(256) paged_read_kernel(const ReadParams p) {
  constexpr int kRow = kHeld == kHeldBf16 ? 2 * D : D, kLanes = kRow / 16, kStep = 256 / kLanes;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.z >> 1, h = blockIdx.y;
  const bool is_v = blockIdx.z & 1;
  const int i0 = blockIdx.x * (kStep * kReadRows) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const long long from = p.start != nullptr ? max(p.start[b], 0) : 0, upto = min((long long)p.lens[b], p.c.tokens());
  const uint8_t* pool = static_cast<const uint8_t*>(is_v ? p.c.v : p.c.k) + lane * 16;
  bf16* to = (is_v ? p.v : p.k) + ((long long)b * p.c.KVH + h) * p.Tmax * D + lane * (kHeld == kHeldBf16 ? 8 : 16);
  long long row[kReadRows];
  uint4 u[kReadRows];
  float s[kReadRows];
#pragma unroll
  for (int r = 0; r < kReadRows; ++r) {
    const int i = i0 + r * kStep;
    row[r] = i < p.Tmax && from + i < upto ? paged_row(p.c, b, h, int(from) + i) : -1;
  }
#pragma unroll
  for (int r = 0; r < kReadRows; ++r) {
    if (row[r] < 0) continue;
    u[r] = *reinterpret_cast<const uint4*>(pool + row[r] * kRow);
    if (kHeld != kHeldBf16) s[r] = (is_v ? p.c.vs : p.c.ks)[row[r]];
  }
#pragma unroll
  for (int r = 0; r < kReadRows; ++r) {
    if (row[r] < 0) continue;
    uint4* out = reinterpret_cast<uint4*>(to + (long long)(i0 + r * kStep) * D);
    if constexpr (kHeld == kHeldBf16) {
      out[0] = u[r];
    } else {
      uint32_t w[4] = {u[r].x, u[r].y, u[r].z, u[r].w}, o[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (kHeld == kHeldInt8) w[q] ^= 0x80808080u;
        const float2 lo = float2_of_half2(half2_of<kHeld, false>(w[q])), hi = float2_of_half2(half2_of<kHeld, true>(w[q]));
        o[2 * q] = bf162_of(lo.x * s[r], lo.y * s[r]);
        o[2 * q + 1] = bf162_of(hi.x * s[r], hi.y * s[r]);
      }
      out[0] = make_uint4(o[0], o[1], o[2], o[3]);
      out[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
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
  const long long per = 256 / (D / 8), items = M * 2 * ((KVH + kAppendHeads - 1) / kAppendHeads), blocks = (items + per - 1) / per;
  if (items > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
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
  const int per = kReadRows * 256 / ((held == kHeldBf16 ? 2 * D : D) / 16);
  auto go = [&](auto kern) { return static_cast<int>(launch_pdl(kern, dim3((Tmax + per - 1) / per, KVH, 2 * B), dim3(256), 0, st, 0, p)); };
  if (D == 128)
    return held == kHeldBf16 ? go(paged_read_kernel<128, kHeldBf16>) : held == kHeldInt8 ? go(paged_read_kernel<128, kHeldInt8>)
                                                                                       : go(paged_read_kernel<128, kHeldE4m3>);
  return held == kHeldBf16 ? go(paged_read_kernel<64, kHeldBf16>) : held == kHeldInt8 ? go(paged_read_kernel<64, kHeldInt8>)
                                                                                    : go(paged_read_kernel<64, kHeldE4m3>);
}
