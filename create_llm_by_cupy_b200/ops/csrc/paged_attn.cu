// Attention of one new token of each sequence over a paged cache (paged_cache.cuh), with the token's rotation and append.
#include <cooperative_groups.h>

#include <atomic>

#include "paged_cache.cuh"
#include "ptx.cuh"
#include "score_cap.cuh"

namespace b200 {
namespace cg = cooperative_groups;

constexpr int PA_WARPS = 4;
constexpr int PA_HEADS = 8;          // query heads of a CTA: rows 0..7 of a product hold them, rows 8..15 what their rounding left
constexpr int kScorePlain = 0, kScoreCap = 1, kScoreBias = 2;
constexpr float kLog2e = 1.4426950408889634f;

struct PagedAttnParams {
  PagedPool c;
  const bf16* kqv;             // [B] rows K | Q | V, pitch ld
  const int* lens;             // [B] cached tokens, below 0: the row is none
  const float* cosr;           // [rows, D / 2]
  const float* sinr;
  const float* slopes;         // [QH]
  bf16* out;                   // [B, QH, D]
  long long ld;
  int QH, groups, rows;
  float scale;
  ScoreCap cap;
  int* status;
};

template <int D, int kHeld>
struct PA {
  static constexpr int kBytes = kHeld == kHeldBf16 ? 2 : 1;
  static constexpr int kRow = D * kBytes;                            // bytes of a token's row
  static constexpr int kTile = kHeld == kHeldBf16 ? 16 : 32;         // tokens of a warp's step
  static constexpr int kChunk = kHeld != kHeldBf16 && D == 128 ? 16 : 8;      // elements of K that a lane takes at once
  static constexpr int kChunks = D / (4 * kChunk);
  static constexpr int kWords = kChunk * kBytes / 4;                 // 32-bit words of a chunk
  static constexpr int kMat = kTile * kRow;                          // bytes of a tile of K, or of V
  static constexpr int kStage = 2 * kMat + 2 * kTile * 4;            // and the scales
  static constexpr int kStages = D == 128 ? 3 : 4;
  static constexpr int kWarp = kStages * kStage + kTile * 16 + 64;   // ring, numbers of a tile's tokens, barriers
  static constexpr int kSmem = PA_WARPS * kWarp + 256;
};

__device__ __forceinline__ void bulk_to_smem(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// Four bytes, or zeros in their place.
__device__ __forceinline__ void cp_async4(void* dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(__cvta_generic_to_global(src)), "r"(there ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int kHeld>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kHeld == kHeldBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two numbers as a pair of the products' type, and as another pair what that rounding left.
template <int kHeld>
__device__ __forceinline__ void two_parts(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (kHeld == kHeldBf16) {
    hi = bf162_of(x, y);
    const float2 f = float2_of_bf162(hi);
    lo = bf162_of(x - f.x, y - f.y);
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
    const float2 f = float2_of_half2(hi);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(y - f.y), "f"(x - f.x));
  }
}

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// N elements of bf16 from a 16-byte aligned address
template <int N>
__device__ __forceinline__ void load_bf16(const bf16* x, float* y) {
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    const uint4 u = reinterpret_cast<const uint4*>(x)[i];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = float2_of_bf162(w[e]);
      y[8 * i + 2 * e] = f.x;
      y[8 * i + 2 * e + 1] = f.y;
    }
  }
}

// The chunks of a head that a lane takes, rotated. The partner of an element is half the chunks away: in the same lane.
template <int D, int kHeld>
__device__ __forceinline__ void rotated_chunks(const bf16* x, int tq, const float* c, const float* s, float (&y)[D / 4]) {
  using L = PA<D, kHeld>;
#pragma unroll
  for (int i = 0; i < L::kChunks; ++i) load_bf16<L::kChunk>(x + (i * 4 + tq) * L::kChunk, y + i * L::kChunk);
#pragma unroll
  for (int i = 0; i < L::kChunks / 2; ++i)
#pragma unroll
    for (int e = 0; e < L::kChunk; e += 4) {
      const int at = (i * 4 + tq) * L::kChunk + e, j = i * L::kChunk + e;
      const float4 cv = *reinterpret_cast<const float4*>(c + at), sv = *reinterpret_cast<const float4*>(s + at);
      rotate_pair(y[j], y[j + D / 8], cv.x, sv.x);
      rotate_pair(y[j + 1], y[j + 1 + D / 8], cv.y, sv.y);
      rotate_pair(y[j + 2], y[j + 2 + D / 8], cv.z, sv.z);
      rotate_pair(y[j + 3], y[j + 3 + D / 8], cv.w, sv.w);
    }
}

// Grid (cluster, KVH * groups, B), cluster (size, 1, 1): the CTAs of a cluster share the tokens of one sequence and KV head, their warps
// take a tile in turn.
template <int D, int kHeld, int kScore>
__global__ void __launch_bounds__(PA_WARPS * 32, 2) paged_attn_kernel(const PagedAttnParams p) {
  using L = PA<D, kHeld>;
  constexpr int kTile = L::kTile, kRow = L::kRow, kNt = kTile / 8;
  constexpr float kUp = kHeld == kHeldBf16 ? 0.f : 14.f;       // log2 of what the largest weight of a row is held as
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  uint8_t* mine = smem + warp * L::kWarp;
  float4* numbers = reinterpret_cast<float4*>(mine + L::kStages * L::kStage);
  uint64_t* full = reinterpret_cast<uint64_t*>(mine + L::kStages * L::kStage + kTile * 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + PA_WARPS * L::kWarp);
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0) {
    for (int i = 0; i < L::kStages; ++i) mbar_init(&full[i], 1);
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  const int cs = gridDim.x, rank = blockIdx.x, b = blockIdx.z, kvh = blockIdx.y / p.groups, grp = blockIdx.y % p.groups;
  const int R = p.QH / p.c.KVH, heads = min(R - grp * PA_HEADS, PA_HEADS), h0 = kvh * R + grp * PA_HEADS;
  const int pos = p.lens[b], len = int(min((long long)max(pos, 0), p.c.tokens()));
  const int* table = p.c.table + (long long)b * p.c.width;
  const int nt = (len + kTile - 1) / kTile, step = cs * PA_WARPS, first = rank * PA_WARPS + warp;
  const int count = pos < 0 || first >= nt ? 0 : (nt - first + step - 1) / step;

  // Pages of 32 tiles of this warp at a time, a lane each; tiles are asked for ahead, and their pages with them.
  int pages = -1;
  auto page_of = [&](int i) {                                // all lanes; i goes up by one from call to call
    if ((i & 31) == 0) {
      const int t = first + (i + lane) * step;
      pages = i + lane < count ? table[(t * kTile) >> p.c.log_page] : -1;
    }
    return __shfl_sync(0xffffffffu, pages, i & 31);
  };
  uint32_t skipped = 0;                                      // bit i % 32: tile i has no page
  auto ask = [&](int i) {
    if (i < count) {
      const int pg = page_of(i), t0 = (first + i * step) * kTile, rows = min(kTile, len - t0);
      const bool there = pg >= 0 && pg < p.c.pages;
      uint8_t* st = mine + (i % L::kStages) * L::kStage;
      const long long row = there ? (((long long)pg * p.c.KVH + kvh) << p.c.log_page) + (t0 & (p.c.page() - 1)) : 0;
      skipped = (skipped & ~(1u << (i & 31))) | (there ? 0u : 1u << (i & 31));
      if (there && lane == 0) {
        mbar_expect_tx(&full[i % L::kStages], 2 * rows * kRow);
        bulk_to_smem(st, static_cast<const uint8_t*>(p.c.k) + row * kRow, rows * kRow, &full[i % L::kStages]);
        bulk_to_smem(st + L::kMat, static_cast<const uint8_t*>(p.c.v) + row * kRow, rows * kRow, &full[i % L::kStages]);
      } else if (lane == 0) {
        mbar_arrive(&full[i % L::kStages]);
      }
      if constexpr (kHeld != kHeldBf16) {
        const bool has = there && lane < rows;
        cp_async4(st + 2 * L::kMat + lane * 4, p.c.ks + (has ? row + lane : 0), has);
        cp_async4(st + 2 * L::kMat + kTile * 4 + lane * 4, p.c.vs + (has ? row + lane : 0), has);
      }
    }
    if constexpr (kHeld != kHeldBf16) cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < L::kStages; ++i) ask(i);

  // The queries as fragments. fp16 has room for little: each row is brought to a largest magnitude of 2^10 by a power of two.
  uint32_t qf[D / 16][4];
  float row_mul = 1.f;                                       // what a product is multiplied with, without the token's scale
  const int at = min(max(pos, 0), p.rows - 1);
  const float* cosr = p.cosr + (long long)at * (D / 2);
  const float* sinr = p.sinr + (long long)at * (D / 2);
  float q[D / 4];
  {
    const bf16* x = p.kqv + (long long)b * p.ld + ((long long)p.c.KVH + h0 + min(g, heads - 1)) * D;
    rotated_chunks<D, kHeld>(x, tq, cosr, sinr, q);
    if constexpr (kHeld != kHeldBf16) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < D / 4; ++i) m = fmaxf(m, fabsf(q[i]));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const int e = min(max(int(__float_as_uint(m) >> 23) - 127, -100), 100);
      const float up = __uint_as_float(uint32_t(127 + 10 - e) << 23);
      row_mul = __uint_as_float(uint32_t(127 - 10 + e) << 23);
#pragma unroll
      for (int i = 0; i < D / 4; ++i) q[i] *= up;
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      two_parts<kHeld>(q[4 * i], q[4 * i + 1], qf[i][0], qf[i][1]);
      two_parts<kHeld>(q[4 * i + 2], q[4 * i + 3], qf[i][2], qf[i][3]);
    }
  }
  float slope = 0.f;
  if (kScore == kScoreBias) slope = p.slopes[h0 + min(g, heads - 1)] * kLog2e;
  const float mul = kScore == kScoreCap ? row_mul : row_mul * p.scale * kLog2e;
  // log2-unit score of a product of row g with a token that is `dist` back
  auto score = [&](float s, float dist) {
    s *= mul;
    if (kScore == kScoreCap) return cap_any(s, p.cap);
    return kScore == kScoreBias ? fmaf(-slope, dist, s) : s;
  };

  float m_run = -INFINITY, l_run = 0.f;
  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

  // The new token: written to its page, and the first that its warp sees.
  if (warp == 0 && rank == 0 && pos >= 0 && pos < p.c.tokens() && pos < p.rows) {
    const long long row = paged_row(p.c, b, kvh, pos);
    if (row >= 0) {
      float k[D / 4], v[D / 4], ks = 1.f, vs = 1.f;
      rotated_chunks<D, kHeld>(p.kqv + (long long)b * p.ld + (long long)kvh * D, tq, cosr, sinr, k);
      load_bf16<D / 4>(p.kqv + (long long)b * p.ld + ((long long)p.c.KVH + p.QH + kvh) * D + tq * (D / 4), v);
      const bool writes = g == 0 && grp == 0;
      if constexpr (kHeld == kHeldBf16) {
#pragma unroll
        for (int i = 0; i < L::kChunks; ++i) {
          const float* x = k + 8 * i;
          const uint4 u = make_uint4(bf162_of(x[0], x[1]), bf162_of(x[2], x[3]), bf162_of(x[4], x[5]), bf162_of(x[6], x[7]));
          if (writes) *reinterpret_cast<uint4*>(static_cast<bf16*>(p.c.k) + row * D + (i * 4 + tq) * 8) = u;
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = float2_of_bf162(w[e]);
            k[8 * i + 2 * e] = f.x;
            k[8 * i + 2 * e + 1] = f.y;
          }
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const float* x = v + 8 * i;
          if (writes)
            *reinterpret_cast<uint4*>(static_cast<bf16*>(p.c.v) + row * D + tq * (D / 4) + 8 * i) =
                make_uint4(bf162_of(x[0], x[1]), bf162_of(x[2], x[3]), bf162_of(x[4], x[5]), bf162_of(x[6], x[7]));
        }
      } else {
        float mk = 0.f, mv = 0.f;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
          mk = fmaxf(mk, fabsf(k[i]));
          mv = fmaxf(mv, fabsf(v[i]));
        }
#pragma unroll
        for (int i = 1; i < 4; i <<= 1) {
          mk = fmaxf(mk, __shfl_xor_sync(0xffffffffu, mk, i));
          mv = fmaxf(mv, __shfl_xor_sync(0xffffffffu, mv, i));
        }
        ks = held_scale<kHeld>(mk);
        vs = held_scale<kHeld>(mv);
        const float ik = __frcp_rn(ks), iv = __frcp_rn(vs);
        uint8_t* wk = static_cast<uint8_t*>(p.c.k) + row * D;
        uint8_t* wv = static_cast<uint8_t*>(p.c.v) + row * D;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t x = held_word<kHeld>(k[4 * i], k[4 * i + 1], k[4 * i + 2], k[4 * i + 3], ks, ik);
          uint32_t y = held_word<kHeld>(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], vs, iv);
          const int j = 4 * i;
          if (writes) {
            *reinterpret_cast<uint32_t*>(wk + (j / L::kChunk * 4 + tq) * L::kChunk + j % L::kChunk) = x;
            *reinterpret_cast<uint32_t*>(wv + tq * (D / 4) + j) = y;
          }
          if (kHeld == kHeldInt8) {
            x ^= 0x80808080u;
            y ^= 0x80808080u;
          }
          const float2 a = float2_of_half2(half2_of<kHeld, false>(x)), c = float2_of_half2(half2_of<kHeld, true>(x));
          const float2 d = float2_of_half2(half2_of<kHeld, false>(y)), f = float2_of_half2(half2_of<kHeld, true>(y));
          k[j] = a.x; k[j + 1] = a.y; k[j + 2] = c.x; k[j + 3] = c.y;
          v[j] = d.x; v[j + 1] = d.y; v[j + 2] = f.x; v[j + 3] = f.y;
        }
        if (writes && tq == 0) {
          p.c.ks[row] = ks;
          p.c.vs[row] = vs;
        }
      }
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < D / 4; ++i) s = fmaf(q[i], k[i], s);
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      s = score(s * ks, 0.f);
      m_run = kHeld == kHeldBf16 ? s : s + __log2f(vs);
      const float w = exp2_of(kUp);
      l_run = tq == 0 ? w * (kHeld == kHeldBf16 ? 1.f : __frcp_rn(vs)) : 0.f;
#pragma unroll
      for (int i = 0; i < D / 4; ++i) o[i % (D / 8)][i / (D / 8)] = v[i] * w;
    }
  }

  bool ok = true;
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    const int slot = i % L::kStages, t0 = (first + i * step) * kTile, rows = min(kTile, len - t0);
    uint8_t* st = mine + slot * L::kStage;
    if constexpr (kHeld != kHeldBf16) cp_async_wait<L::kStages - 1>();
    ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], (i / L::kStages) & 1, abort_flag));
    if (!ok) break;
    if (!(skipped >> (i & 31) & 1)) {
      if constexpr (kHeld != kHeldBf16) {
        // a token's numbers: what its products are multiplied with, log2 of V's scale, and one over it
        const float* sc = reinterpret_cast<const float*>(st + 2 * L::kMat);
        const bool has = lane < rows;
        const float ks = sc[lane], vs = has ? sc[kTile + lane] : 1.f;
        numbers[lane] = make_float4(has ? ks : 0.f, has ? __log2f(vs) : 0.f, __fdividef(1.f, vs), 0.f);
      }
      if (rows < kTile)                                      // what lies behind the last token may be anything: its weight is 0, it shall be
        for (int x = rows * kRow + lane * 4; x < L::kMat; x += 128) *reinterpret_cast<uint32_t*>(st + L::kMat + x) = 0u;
      __syncwarp();
      float y[2 * kNt], rv[2 * kNt];
#pragma unroll
      for (int n = 0; n < kNt; ++n) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        const uint8_t* kr = st + (8 * n + g) * kRow + tq * L::kChunk * L::kBytes;
#pragma unroll
        for (int c = 0; c < L::kChunks; ++c) {
          uint32_t w[L::kWords];
          if constexpr (L::kWords == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(kr + c * 4 * L::kChunk * L::kBytes);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(kr + c * 4 * L::kChunk * L::kBytes);
            w[0] = u.x; w[1] = u.y;
          }
          if constexpr (kHeld == kHeldBf16) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t (&a)[4] = qf[2 * c + e];
              mma_16816<kHeld>(acc, a[0], a[1], a[2], a[3], w[2 * e], w[2 * e + 1]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < L::kWords; ++e) {
              const uint32_t (&a)[4] = qf[c * L::kWords + e];
              const uint32_t x = kHeld == kHeldInt8 ? w[e] ^ 0x80808080u : w[e];
              mma_16816<kHeld>(acc, a[0], a[1], a[2], a[3], half2_of<kHeld, false>(x), half2_of<kHeld, true>(x));
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = 8 * n + 2 * tq + e;
          float s = acc[e] + acc[2 + e], more = 0.f;
          rv[2 * n + e] = 1.f;
          if constexpr (kHeld != kHeldBf16) {
            const float4 u = numbers[tok];
            s *= u.x;
            more = u.y;
            rv[2 * n + e] = u.z;
          }
          s = score(s, float(pos - t0 - tok)) + more;
          y[2 * n + e] = tok < rows ? s : -INFINITY;
        }
      }
      float m = y[0];
#pragma unroll
      for (int e = 1; e < 2 * kNt; ++e) m = fmaxf(m, y[e]);
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const float m_new = fmaxf(m_run, m), ref = m_new == -INFINITY ? 0.f : m_new;
      const float f = exp2_of(m_run - ref);
      if (__any_sync(0xffffffffu, f != 1.f)) {
        l_run *= f;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[j][0] *= f; o[j][1] *= f; o[j][2] *= f; o[j][3] *= f;
        }
      }
      m_run = m_new;
      uint32_t hi[kNt], lo[kNt];
#pragma unroll
      for (int n = 0; n < kNt; ++n) {
        const float w0 = exp2_of(y[2 * n] - ref + kUp), w1 = exp2_of(y[2 * n + 1] - ref + kUp);
        l_run = fmaf(w0, rv[2 * n], l_run);
        l_run = fmaf(w1, rv[2 * n + 1], l_run);
        two_parts<kHeld>(w0, w1, hi[n], lo[n]);
      }
      const uint8_t* vr = st + L::kMat + 2 * tq * kRow + g * (kRow / 8);
#pragma unroll
      for (int n = 0; n < kNt; n += 2) {
        constexpr int kVw = kRow / 32;                       // words of a lane's piece of a row
        uint32_t r[4][kVw];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint8_t* from = vr + (8 * n + 8 * (x >> 1) + (x & 1)) * kRow;
          if constexpr (kVw >= 4) {
#pragma unroll
            for (int c = 0; c < kVw / 4; ++c) {
              const uint4 u = reinterpret_cast<const uint4*>(from)[c];
              r[x][4 * c] = u.x; r[x][4 * c + 1] = u.y; r[x][4 * c + 2] = u.z; r[x][4 * c + 3] = u.w;
            }
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(from);
            r[x][0] = u.x; r[x][1] = u.y;
          }
        }
#pragma unroll
        for (int w = 0; w < kVw; ++w) {
          if constexpr (kHeld == kHeldBf16) {
            mma_16816<kHeld>(o[2 * w], hi[n], lo[n], hi[n + 1], lo[n + 1], __byte_perm(r[0][w], r[1][w], 0x5410),
                             __byte_perm(r[2][w], r[3][w], 0x5410));
            mma_16816<kHeld>(o[2 * w + 1], hi[n], lo[n], hi[n + 1], lo[n + 1], __byte_perm(r[0][w], r[1][w], 0x7632),
                             __byte_perm(r[2][w], r[3][w], 0x7632));
          } else {
            uint32_t a = __byte_perm(r[0][w], r[1][w], 0x5140), c = __byte_perm(r[2][w], r[3][w], 0x5140);
            uint32_t d = __byte_perm(r[0][w], r[1][w], 0x7362), e = __byte_perm(r[2][w], r[3][w], 0x7362);
            if (kHeld == kHeldInt8) {
              a ^= 0x80808080u; c ^= 0x80808080u; d ^= 0x80808080u; e ^= 0x80808080u;
            }
            mma_16816<kHeld>(o[4 * w], hi[n], lo[n], hi[n + 1], lo[n + 1], half2_of<kHeld, false>(a), half2_of<kHeld, false>(c));
            mma_16816<kHeld>(o[4 * w + 1], hi[n], lo[n], hi[n + 1], lo[n + 1], half2_of<kHeld, true>(a), half2_of<kHeld, true>(c));
            mma_16816<kHeld>(o[4 * w + 2], hi[n], lo[n], hi[n + 1], lo[n + 1], half2_of<kHeld, false>(d), half2_of<kHeld, false>(e));
            mma_16816<kHeld>(o[4 * w + 3], hi[n], lo[n], hi[n + 1], lo[n + 1], half2_of<kHeld, true>(d), half2_of<kHeld, true>(e));
          }
        }
      }
    }
    __syncwarp();
    ask(i + L::kStages);
  }

  // Over the lanes, the warps and the CTAs of the cluster. The ring is free: every tile that was asked for has been waited for, or the
  // kernel gives up (then what still arrives may overwrite these numbers, which nobody uses, but not another kernel's memory).
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
  cg::cluster_group cluster = cg::this_cluster();
  float* wm = reinterpret_cast<float*>(mine);                // [8] maxima, [8] sums, [8][D] values of a warp
  float* wl = wm + PA_HEADS;
  float* wo = wl + PA_HEADS;
  if (tq == 0) {
    wm[g] = m_run;
    wl[g] = l_run;
  }
#pragma unroll
  for (int j = 0; j < D / 8; j += 4)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float4*>(wo + g * D + (2 * tq + e) * (D / 8) + j) =
          make_float4(o[j][e] + o[j][2 + e], o[j + 1][e] + o[j + 1][2 + e], o[j + 2][e] + o[j + 2][2 + e], o[j + 3][e] + o[j + 3][2 + e]);
  __syncthreads();
  constexpr int kPart = (2 + D) * PA_HEADS * 4;              // bytes of such a set
  float* cm = reinterpret_cast<float*>(smem + kPart);        // the CTA's, behind the first warp's
  float* cl = cm + PA_HEADS;
  float* co = cl + PA_HEADS;
  for (int i = threadIdx.x; i < heads * D; i += PA_WARPS * 32) {
    const int r = i / D, d = i % D;
    float m = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) m = fmaxf(m, *reinterpret_cast<const float*>(smem + w * L::kWarp + r * 4));
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) {
      const float* s = reinterpret_cast<const float*>(smem + w * L::kWarp);
      const float f = exp2_of(s[r] - ref);
      l = fmaf(s[PA_HEADS + r], f, l);
      x = fmaf(s[2 * PA_HEADS + r * D + d], f, x);
    }
    if (cs == 1) {
      p.out[((long long)b * p.QH + h0 + r) * D + d] = __float2bfloat16(l == 0.f ? 0.f : x / l);
    } else {
      co[r * D + d] = x;
      if (d == 0) {
        cm[r] = m;
        cl[r] = l;
      }
    }
  }
  if (cs > 1) {
    cluster.sync();
    for (int i = rank * PA_WARPS * 32 + threadIdx.x; i < heads * D; i += cs * PA_WARPS * 32) {
      const int r = i / D;
      float m = -INFINITY, l = 0.f, x = 0.f;
      for (int c = 0; c < cs; ++c) m = fmaxf(m, *cluster.map_shared_rank(cm + r, c));
      const float ref = m == -INFINITY ? 0.f : m;
      for (int c = 0; c < cs; ++c) {
        const float f = exp2_of(*cluster.map_shared_rank(cm + r, c) - ref);
        l = fmaf(*cluster.map_shared_rank(cl + r, c), f, l);
        x = fmaf(*cluster.map_shared_rank(co + i, c), f, x);
      }
      p.out[((long long)b * p.QH + h0) * D + i] = __float2bfloat16(l == 0.f ? 0.f : x / l);
    }
    cluster.sync();                                          // peers read this CTA's numbers until here
  }
  if (threadIdx.x == 0 && *abort_flag != 0 && p.status != nullptr && atomicCAS(p.status, 0, int(*abort_flag)) == 0) p.status[1] = 361;
}

template <int D, int kHeld, int kScore>
static int launch_paged(const PagedAttnParams& p, cudaStream_t st) {
  using L = PA<D, kHeld>;
  const auto kern = paged_attn_kernel<D, kHeld, kScore>;
  static std::atomic<bool> allowed[64];              // shared memory is asked for on every device of a process
  int dev = 0;
  B200_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !allowed[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return static_cast<int>(e);
    }
    if (dev >= 0 && dev < 64) allowed[dev].store(true, std::memory_order_release);
  }
  const long long units = (long long)p.c.B * p.c.KVH * p.groups;
  int cs = 1;
  while (cs < 8 && 2 * cs * units <= 2LL * num_sms() && 2LL * cs * PA_WARPS * L::kTile <= p.c.tokens() + L::kTile - 1) cs *= 2;
  return static_cast<int>(launch_pdl(kern, dim3(cs, p.c.KVH * p.groups, p.c.B), dim3(PA_WARPS * 32), L::kSmem, st, cs, p));
}

template <int D, int kHeld>
static int launch_paged_score(const PagedAttnParams& p, float cap, cudaStream_t st) {
  if (cap > 0.f) return launch_paged<D, kHeld, kScoreCap>(p, st);
  return p.slopes != nullptr ? launch_paged<D, kHeld, kScoreBias>(p, st) : launch_paged<D, kHeld, kScorePlain>(p, st);
}

}  // namespace b200

using namespace b200;

// kqv [B] rows K | Q | V (un-rotated, pitch ld), out [B, QH, D], lens [B], rotary tables [rows, D / 2]. cap > 0: scores c tanh(s / c);
// slopes [QH]: scores minus slope times distance (not both). held: 0 bf16, 1 int8, 2 e4m3.
B200_API int b200_paged_attn_append(const void* kqv, void* pk, void* pv, void* ks, void* vs, const void* table, const void* lens,
                                    const void* cosr, const void* sinr, const void* slopes, void* out, int rows, long long ld, int B,
                                    int width, int pages, int QH, int KVH, int log_page, int D, int held, float scale, float cap,
                                    cudaStream_t st) {
  PagedAttnParams p;
  p.c.k = pk;
  p.c.v = pv;
  p.c.ks = static_cast<float*>(ks);
  p.c.vs = static_cast<float*>(vs);
  p.c.table = static_cast<const int*>(table);
  p.c.B = B; p.c.width = width; p.c.pages = pages; p.c.KVH = KVH; p.c.log_page = log_page;
  if (paged_pool_wrong(p.c, held, D) != nullptr || QH < 1 || QH % KVH != 0 || rows < 1 || ld % 8 != 0 || cap < 0.f ||
      (cap > 0.f && slopes != nullptr) || lens == nullptr)
    return static_cast<int>(cudaErrorInvalidValue);
  for (const void* x : {kqv, cosr, sinr, (const void*)out})
    if (x == nullptr || (reinterpret_cast<uintptr_t>(x) & 15) != 0) return static_cast<int>(cudaErrorInvalidValue);
  p.groups = (QH / KVH + PA_HEADS - 1) / PA_HEADS;
  if (B > 65535 || (long long)KVH * p.groups > 65535) return static_cast<int>(cudaErrorInvalidValue);
  if (B == 0) return 0;
  p.kqv = static_cast<const bf16*>(kqv);
  p.lens = static_cast<const int*>(lens);
  p.cosr = static_cast<const float*>(cosr);
  p.sinr = static_cast<const float*>(sinr);
  p.slopes = static_cast<const float*>(slopes);
  p.out = static_cast<bf16*>(out);
  p.ld = ld; p.QH = QH; p.rows = rows; p.scale = scale;
  p.cap = make_score_cap(scale, cap);
  p.status = status_ptr();
  if (D == 128)
    return held == kHeldBf16   ? launch_paged_score<128, kHeldBf16>(p, cap, st)
           : held == kHeldInt8 ? launch_paged_score<128, kHeldInt8>(p, cap, st)
                               : launch_paged_score<128, kHeldE4m3>(p, cap, st);
  return held == kHeldBf16   ? launch_paged_score<64, kHeldBf16>(p, cap, st)
         : held == kHeldInt8 ? launch_paged_score<64, kHeldInt8>(p, cap, st)
                             : launch_paged_score<64, kHeldE4m3>(p, cap, st);
}
