// Attention of one new token of each sequence over a paged cache (paged_cache.cuh), with the token's rotation and append.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(s_j - m),   s_j = score(scale q . k_j) log2 e
//
// What bounds it: each cached row is read once, 2 D + 8 bytes a token and KV head in 8 bits, so HBM, if an SM gets through its tiles fast
// enough (it has 24 bytes of HBM a cycle). 64 x 1500 to 4000 tokens, 32 / 8 heads of 128, int8, with the append: 82 us, 4.6 TB/s; bytes to
// fp16 on the ALU and the last CTAs, which run alone, are the rest. Hence:
//   * products by mma.sync with the TOKENS (dims, for the values) as rows and the heads as columns. Columns 0 to 3 are the four query heads
//     of the CTA, columns 4 to 7 what rounding left of them: scores and weights go in as two parts at no further product. With the heads as
//     rows (8 and 8 of 16) it were twice the products and accumulators (107 -> 90 us). (A tcgen05 tile has 128 rows, of which four heads
//     would fill four.)
//   * int8 keys go in as they are held, with Q as whole numbers of four bytes, in two products of twice the depth that need no conversion
//     (88 -> 81 us; two bytes in one product 79, but off by up to 1.6e-2 where two dims of Q are 1000 times the others). Values and e4m3
//     become exact fp16 in registers. K's scale multiplies the score; V's joins the weight as a logarithm: w_j = 2^(s_j + log2 sv_j - M), M
//     the running maximum of that sum. The sum of the weights without it is that of 2^(s_j - M), up to 2^121 times smaller or 2^80 times
//     larger, and scaled in two half steps: a row of nothing beside large ones loses its weight, not its place in that sum. The largest
//     weight is held as 2^14, so that fp16 has 2^-38 of it to show for a small one.
//   * a dot product does not care in which order its dims are walked: a lane's 16-byte pieces of K are fragments as they stand. V needs
//     pairs of tokens: two byte permutations for four dims. Weights are turned over by movmatrix.
//   * tiles go through a ring per warp, so warps never wait for one another until the end. Three CTAs an SM.
//   * few sequences: clusters of up to eight CTAs share one or, where 8 leave SMs idle, pieces that a second kernel joins (one sequence of
//     60001 tokens 68 us with clusters of 8, 54 of 16, 41 with 55 pieces; 33 since four threads a dim join them, and Q went in as bytes).
// Tried and not kept: bulk copies by a warp of their own (no faster: the time is that of the arithmetic), one list of all tiles cut evenly
// over CTAs that stay (64 x 1500 to 4000 tokens 88 -> 93 us, 32 x 0 to 1980 21 -> 40: the start of a stretch takes as long as four tiles,
// and its state does not fit in the registers of three CTAs an SM).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged_cache.cuh"
#include "ptx.cuh"
#include "score_cap.cuh"

namespace b200 {
namespace cg = cooperative_groups;

constexpr int PA_CLUSTER = 8;        // CTAs of a cluster, at most
constexpr int PA_WARPS = 4, PA_THREADS = 32 * (PA_WARPS + 1);
constexpr int PA_HEADS = 4;          // query heads of a CTA: columns 0..3 of a product hold them, columns 4..7 what their rounding left
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
  int pieces;                  // more than 0: a sequence's tokens go to that many CTAs, which leave their parts to another kernel
  float2* part_ml;             // [B, QH, pieces] maximum and sum
  float* part_o;               // [B, QH, pieces, D]
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
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kWarp = kStages * kStage;                     // a warp's ring
  static constexpr int kPart = (2 + D) * PA_HEADS * 4;               // maxima, sums, values of the heads
  static constexpr int kOwn = PA_WARPS * kWarp;                      // those of the new token
  static constexpr int kSmem = kOwn + kPart;
  static_assert(2 * kPart <= kStages * kStage);
  // Where byte x of a tile stands: the 16-byte pieces of a 128-byte line in another order from line to line, so that neither the eight
  // lanes that read K together (two rows, four pieces) nor those that read V (four rows, two pieces) meet a bank twice (256-byte rows: V
  // twice). The order repeats every eight rows.
  __host__ __device__ static constexpr int place(int x) {
    const int line = x >> 7, r = kRow == 256 ? line >> 1 : line;
    return x ^ (kRow == 64 ? (line & 3) << 5 : ((r & 6) ^ (r & 1) << 2) << 4);
  }
};

// 16 or 4 bytes on their way to shared memory, or zeros in their place.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there = true) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool there = true) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(there ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int kHeld>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kHeld == kHeldBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 x 8 sums of products of 32 signed bytes.
__device__ __forceinline__ void mma_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// An 8 x 8 matrix of 16-bit elements, a row to four lanes, turned over.
__device__ __forceinline__ uint32_t turned(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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

// The chunks of a head that a lane takes, and their rotation. The partner of an element is half the chunks away: in the same lane.
template <int D, int kHeld>
__device__ __forceinline__ void load_chunks(const bf16* x, int tq, float (&y)[D / 4]) {
  using L = PA<D, kHeld>;
#pragma unroll
  for (int i = 0; i < L::kChunks; ++i) load_bf16<L::kChunk>(x + (i * 4 + tq) * L::kChunk, y + i * L::kChunk);
}
template <int D, int kHeld>
__device__ __forceinline__ void rotate_chunks(float (&y)[D / 4], int tq, const float* c, const float* s) {
  using L = PA<D, kHeld>;
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

// Grid (cluster or pieces, KVH * groups, B), cluster (size, 1, 1): the CTAs along x share the tokens of one sequence and KV head, their
// four warps take a tile in turn. A fifth warp deals with the new token. What they have is joined in the cluster, or by the next kernel.
template <int D, int kHeld, int kScore>
__global__ void __launch_bounds__(PA_THREADS, 3) paged_attn_kernel(const PagedAttnParams p) {
  using L = PA<D, kHeld>;
  constexpr int kTile = L::kTile, kRow = L::kRow, kStages = L::kStages;
  constexpr float kUp = kHeld == kHeldBf16 ? 0.f : 14.f;       // log2 of what the largest weight of a row is held as
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  uint8_t* mine = smem + warp * L::kWarp;
  pdl_wait();
  pdl_trigger();

  const int cs = gridDim.x, rank = blockIdx.x, b = blockIdx.z, kvh = blockIdx.y / p.groups, grp = blockIdx.y % p.groups;
  const int R = p.QH / p.c.KVH, heads = min(R - grp * PA_HEADS, PA_HEADS), h0 = kvh * R + grp * PA_HEADS;
  const bf16* row_in = p.kqv + (long long)b * p.ld;
  const int step = cs * PA_WARPS, first = rank * PA_WARPS + warp;
  const int* table = p.c.table + (long long)b * p.c.width;
  // Pages of 32 tiles at a time, a lane each; of the first ones while the length is still on its way.
  const auto page_at = [&](int i) {
    const long long at = ((long long)first + (long long)(i + lane) * step) * kTile >> p.c.log_page;
    return at < p.c.width ? table[at] : -1;
  };
  int pages = page_at(0);
  const int pos = p.lens[b];
  float q[D / 4];
  load_chunks<D, kHeld>(row_in + ((long long)p.c.KVH + h0 + min(g & 3, heads - 1)) * D, tq, q);
  const int len = int(min((long long)max(pos, 0), p.c.tokens()));
  const int nt = (len + kTile - 1) / kTile;
  const int count = warp == PA_WARPS || pos < 0 || first >= nt ? 0 : (nt - first + step - 1) / step;

  // Tiles are asked for kStages ahead, by the lanes themselves (bulk copies took as long, and leave the bytes in the order that they come
  // in).
  uint32_t lane_place[4];                                    // of this lane's 16 bytes of every 512
#pragma unroll
  for (int x = 0; x < 4; ++x) lane_place[x] = L::place(512 * x + lane * 16) - 512 * x;
  uint32_t skipped = 0;                                      // bit i % 32: tile i has no page
  auto ask = [&](int i) {
    if (i < count) {
      if ((i & 31) == 0 && i > 0) pages = page_at(i);
      const int pg = __shfl_sync(0xffffffffu, pages, i & 31), t0 = (first + i * step) * kTile, bytes = min(kTile, len - t0) * kRow;
      const bool there = pg >= 0 && pg < p.c.pages;
      skipped = (skipped & ~(1u << (i & 31))) | (there ? 0u : 1u << (i & 31));
      if (there) {
        const uint32_t st = smem_u32(mine) + (i % kStages) * L::kStage;
        const long long row = (((long long)pg * p.c.KVH + kvh) << p.c.log_page) + (t0 & (p.c.page() - 1));
        const uint8_t* k = static_cast<const uint8_t*>(p.c.k) + row * kRow + lane * 16;
        const uint8_t* v = static_cast<const uint8_t*>(p.c.v) + row * kRow + lane * 16;
        if (bytes == L::kMat) {
#pragma unroll
          for (int x = 0; x < L::kMat; x += 512) cp_async16(st + x + lane_place[x >> 9 & 3], k + x);
          if constexpr (kHeld != kHeldBf16) {
            cp_async4(st + 2 * L::kMat + lane * 4, p.c.ks + row + lane);
            cp_async4(st + 2 * L::kMat + kTile * 4 + lane * 4, p.c.vs + row + lane);
          }
#pragma unroll
          for (int x = 0; x < L::kMat; x += 512) cp_async16(st + L::kMat + x + lane_place[x >> 9 & 3], v + x);
        } else {                                             // zeros behind the last token
#pragma unroll
          for (int x = 0; x < L::kMat; x += 512) {
            const bool has = x + lane * 16 < bytes;
            cp_async16(st + x + lane_place[x >> 9 & 3], has ? k + x : k, has);
            cp_async16(st + L::kMat + x + lane_place[x >> 9 & 3], has ? v + x : v, has);
          }
          if constexpr (kHeld != kHeldBf16) {
            const bool has = lane * kRow < bytes;
            cp_async4(st + 2 * L::kMat + lane * 4, p.c.ks + row + (has ? lane : 0), has);
            cp_async4(st + 2 * L::kMat + kTile * 4 + lane * 4, p.c.vs + row + (has ? lane : 0), has);
          }
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) ask(i);

  // The queries as fragments: lanes g < 4 the rounded values of head g, the others what that left of head g - 4. Over 8-bit rows each head
  // is first brought to a largest magnitude of 2^10 by a power of two, whatever its numbers are. For e4m3 they go in as fp16, which has
  // room for little. For int8 as whole numbers of 2^-19, below 2^30, in four signed bytes: K goes into the products as it is held, their
  // sums are exact (at most 2^21, also as fp32), and a number is off by 2^-30 of its head's largest at most, not at all from a 64th of it
  // on. The upper two bytes are the eight columns of one product, the lower two of another. (Two bytes, off by 2^-16 of the largest, were
  // half of the products, but heads with a few dims 100 times the others lost what the others say.)
  constexpr bool kWhole = kHeld == kHeldInt8;
  uint32_t qf[D / 16][2];                                    // over int8 rows the upper bytes, then the lower ones
  float row_mul = 1.f, own_mul = 1.f;                        // what a product of head g & 3 is multiplied with, without the token's scale;
  const int at = min(max(pos, 0), p.rows - 1);               // and one of `q`
  const float* cosr = p.cosr + (long long)at * (D / 2);
  const float* sinr = p.sinr + (long long)at * (D / 2);
  rotate_chunks<D, kHeld>(q, tq, cosr, sinr);
  if constexpr (kHeld != kHeldBf16) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) m = fmaxf(m, fabsf(q[i]));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const int e = max(int(__float_as_uint(m) >> 23) - 127, -116);
    const float up = __uint_as_float(uint32_t(127 + 10 - e) << 23);
    own_mul = row_mul = __uint_as_float(uint32_t(127 - 10 + e) << 23);
#pragma unroll
    for (int i = 0; i < D / 4; ++i) q[i] *= up;
    if constexpr (kWhole) {
      row_mul *= 32.f;                                       // sums come in units of 2^5 of `q`'s
#pragma unroll
      for (int i = 0; i < D / 4; i += 4) {
        uint32_t n[4];                                       // bytes b3 b2 b1 b0 of a number (b3 2^24 + ..), b2 b1 b0 x in lanes g >= 4
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          n[x] = (uint32_t(__float2int_rn(q[i + x] * 524288.f)) + 0x808080u) ^ 0x808080u;
          if (g >= 4) n[x] <<= 8;
        }
        qf[i / 8][i / 4 % 2] = __byte_perm(__byte_perm(n[0], n[1], 0x0073), __byte_perm(n[2], n[3], 0x0073), 0x5410);
        qf[D / 32 + i / 8][i / 4 % 2] = __byte_perm(__byte_perm(n[0], n[1], 0x0051), __byte_perm(n[2], n[3], 0x0051), 0x5410);
      }
    }
  }
  if constexpr (!kWhole) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t hi, lo;
        two_parts<kHeld>(q[4 * i + 2 * e], q[4 * i + 2 * e + 1], hi, lo);
        qf[i][e] = g < 4 ? hi : lo;
      }
  }
  // Score in units of log2 of a product with a token that is `dist` back. `mul` has the token's scale in it: of large keys and small
  // queries the product times either alone could be infinite.
  auto score = [&](float s, float mul, float slope, float dist) {
    s *= mul;
    if (kScore == kScoreCap) return cap_any(s, p.cap);
    return kScore == kScoreBias ? fmaf(-slope, dist, s) : s;
  };
  const float unit = kScore == kScoreCap ? 1.f : p.scale * kLog2e;

  auto part = [&](int w) { return reinterpret_cast<float*>(smem + (w < PA_WARPS ? w * L::kWarp : L::kOwn)); };
  float* wm = part(warp);                                    // [4] maxima, [4] sums, [4][D] values of a warp
  float* wl = wm + PA_HEADS;
  float* wo = wl + PA_HEADS;
  // The new token: written to its page, and all that the fifth warp sees.
  if (warp == PA_WARPS && rank == 0) {
    float m_new = -INFINITY, l_new = 0.f, v[D / 4];
#pragma unroll
    for (int i = 0; i < D / 4; ++i) v[i] = 0.f;
    const long long row = pos >= 0 && pos < p.c.tokens() && pos < p.rows ? paged_row(p.c, b, kvh, pos) : -1;
    if (row >= 0) {
      float k[D / 4], ks = 1.f, vs = 1.f;
      load_chunks<D, kHeld>(row_in + (long long)kvh * D, tq, k);
      load_bf16<D / 4>(row_in + ((long long)p.c.KVH + p.QH + kvh) * D + tq * (D / 4), v);
      rotate_chunks<D, kHeld>(k, tq, cosr, sinr);
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
      s = score(s, ks * (own_mul * unit), 0.f, 0.f);
      m_new = kHeld == kHeldBf16 ? s : s + __log2f(vs);
      const float w = exp2_of(kUp);
      l_new = w * (kHeld == kHeldBf16 ? 1.f : __frcp_rn(vs));
#pragma unroll
      for (int i = 0; i < D / 4; ++i) v[i] *= w;
    }
    if (g < PA_HEADS) {
      if (tq == 0) {
        wm[g] = m_new;
        wl[g] = l_new;
      }
#pragma unroll
      for (int i = 0; i < D / 4; i += 4)
        *reinterpret_cast<float4*>(wo + g * D + tq * (D / 4) + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    }
  }

  // This lane's two columns of a tile's products: heads `ha` and `ha + 1`, or what is left of them; running maxima and sums of both.
  const int ha = 2 * (tq & 1);
  float mul[2], slope[2] = {0.f, 0.f}, m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    mul[e] = __shfl_sync(0xffffffffu, row_mul, 4 * (ha + e)) * unit;
    if (kScore == kScoreBias) slope[e] = p.slopes[h0 + min(ha + e, heads - 1)] * kLog2e;
  }
  float o[D / 16][4];                                        // dims (D / 8) g + 2 j of both heads, then the next dim of both
#pragma unroll
  for (int j = 0; j < D / 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    const int t0 = (first + i * step) * kTile, rows = min(kTile, len - t0);
    const uint8_t* st = mine + (i % kStages) * L::kStage;
    cp_async_wait<kStages - 1>();
    __syncwarp();
    if (!(skipped >> (i & 31) & 1)) {
      // Scores: tokens are the rows of the products, 16 at a time.
      constexpr int kMt = kTile / 16;
      std::conditional_t<kWhole, int, float> acc[kMt][4];
      int low[kWhole ? kMt : 1][4];                          // of the lower two bytes
#pragma unroll
      for (int t = 0; t < kMt; ++t) {
        acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0;
        if constexpr (kWhole) low[t][0] = low[t][1] = low[t][2] = low[t][3] = 0;
      }
      constexpr int kPiece = L::kChunk * L::kBytes;
      const uint8_t* kr = st + L::place(g * kRow + tq * kPiece);
      const int other = L::place(g * kRow + (tq + 4) * kPiece) - L::place(g * kRow + tq * kPiece);
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c) {
        uint32_t w[2 * kMt][L::kWords];
#pragma unroll
        for (int n = 0; n < 2 * kMt; ++n) {
          const uint8_t* from = kr + 8 * n * kRow + (c & 1) * other + (c >> 1) * 8 * kPiece;
          if constexpr (L::kWords == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(from);
            w[n][0] = u.x; w[n][1] = u.y; w[n][2] = u.z; w[n][3] = u.w;
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(from);
            w[n][0] = u.x; w[n][1] = u.y;
          }
        }
        if constexpr (kHeld == kHeldBf16) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int t = 0; t < kMt; ++t)
              mma_16816<kHeld>(acc[t], w[2 * t][2 * e], w[2 * t + 1][2 * e], w[2 * t][2 * e + 1], w[2 * t + 1][2 * e + 1], qf[2 * c + e][0],
                               qf[2 * c + e][1]);
        } else if constexpr (kWhole) {
#pragma unroll
          for (int e = 0; e < L::kWords / 2; ++e) {
            const uint32_t (&a)[2] = qf[c * (L::kWords / 2) + e], (&z)[2] = qf[D / 32 + c * (L::kWords / 2) + e];
#pragma unroll
            for (int t = 0; t < kMt; ++t) {
              mma_16832(acc[t], w[2 * t][2 * e], w[2 * t + 1][2 * e], w[2 * t][2 * e + 1], w[2 * t + 1][2 * e + 1], a[0], a[1]);
              mma_16832(low[t], w[2 * t][2 * e], w[2 * t + 1][2 * e], w[2 * t][2 * e + 1], w[2 * t + 1][2 * e + 1], z[0], z[1]);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < L::kWords; ++e) {
            const uint32_t (&a)[2] = qf[c * L::kWords + e];
#pragma unroll
            for (int t = 0; t < kMt; ++t) {
              const uint32_t x = w[2 * t][e], z = w[2 * t + 1][e];
              mma_16816<kHeld>(acc[t], half2_of<kHeld, false>(x), half2_of<kHeld, false>(z), half2_of<kHeld, true>(x),
                               half2_of<kHeld, true>(z), a[0], a[1]);
            }
          }
        }
      }
      // y[n][e]: token 8 n + g, head ha + e; what the rounding of Q left comes from the lane two further.
      float y[2 * kMt][2], lv[2 * kMt], m[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2 * kMt; ++n) {
        const int tok = 8 * n + g;
        float ks = 1.f;
        lv[n] = 0.f;
        if constexpr (kHeld != kHeldBf16) {
          // a token's scales: V's as its logarithm, which goes into the weight
          const float* scales = reinterpret_cast<const float*>(st + 2 * L::kMat);
          const float vs = fmaxf(scales[kTile + tok], kLeastScale);
          ks = scales[tok];
          lv[n] = __log2f(vs);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float part_s = float(acc[n >> 1][2 * (n & 1) + e]), s;
          if constexpr (kWhole) part_s = fmaf(float(low[n >> 1][2 * (n & 1) + e]), 1.f / 65536.f, part_s);  // bytes 3 and 1, or 2 and 0
          const float rest = __shfl_xor_sync(0xffffffffu, part_s, 2);
          if constexpr (kWhole) s = tq < 2 ? fmaf(rest, 1.f / 256.f, part_s) : fmaf(part_s, 1.f / 256.f, rest);
          else s = part_s + rest;
          s = score(s, ks * mul[e], slope[e], float(pos - t0 - tok)) + lv[n];
          y[n][e] = tok < rows ? s : -INFINITY;
          m[e] = fmaxf(m[e], y[n][e]);
        }
      }
      float ref[2], half[2], f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 4));
        m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 8));
        m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 16));
        m[e] = fmaxf(m_run[e], m[e]);
        ref[e] = m[e] == -INFINITY ? 0.f : m[e];
        half[e] = exp2_of(.5f * (m_run[e] - ref[e]));
        f[e] = half[e] * half[e];
        m_run[e] = m[e];
      }
      if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
        l_run[0] = l_run[0] * half[0] * half[0];
        l_run[1] = l_run[1] * half[1] * half[1];
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[j][0] *= f[0]; o[j][1] *= f[1]; o[j][2] *= f[0]; o[j][3] *= f[1];
        }
      }
      uint32_t pw[2 * kMt];                                  // weights, tokens along the lanes' pairs
#pragma unroll
      for (int n = 0; n < 2 * kMt; ++n) {
        const float w0 = exp2_of(y[n][0] - ref[0] + kUp), w1 = exp2_of(y[n][1] - ref[1] + kUp);
        if constexpr (kHeld == kHeldBf16) {
          l_run[0] += w0;
          l_run[1] += w1;
        } else {
          l_run[0] += exp2_of(y[n][0] - ref[0] - (lv[n] - kUp));
          l_run[1] += exp2_of(y[n][1] - ref[1] - (lv[n] - kUp));
        }
        uint32_t hi, lo;
        two_parts<kHeld>(w0, w1, hi, lo);
        pw[n] = turned(tq < 2 ? hi : lo);
      }
      // Values: dims are the rows of the products.
      constexpr int kVw = kRow / 32;                         // words of a lane's piece of a row; of 256-byte rows it is two places
      const uint8_t* vr[2];
      int next[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int from = (2 * tq + x) * kRow + g * (kRow / 8);
        vr[x] = st + L::kMat + L::place(from);
        next[x] = L::place(from + 16) - L::place(from);
      }
#pragma unroll
      for (int t = 0; t < kMt; ++t) {
        uint32_t r[4][kVw];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint8_t* from = vr[x & 1] + (16 * t + 8 * (x >> 1)) * kRow;
          if constexpr (kVw >= 4) {
#pragma unroll
            for (int c = 0; c < kVw / 4; ++c) {
              const uint4 u = *reinterpret_cast<const uint4*>(c == 0 ? from : from + next[x & 1]);
              r[x][4 * c] = u.x; r[x][4 * c + 1] = u.y; r[x][4 * c + 2] = u.z; r[x][4 * c + 3] = u.w;
            }
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(from);
            r[x][0] = u.x; r[x][1] = u.y;
          }
        }
        const uint32_t b0 = pw[2 * t], b1 = pw[2 * t + 1];
#pragma unroll
        for (int w = 0; w < kVw; ++w) {
          if constexpr (kHeld == kHeldBf16) {
            mma_16816<kHeld>(o[w], __byte_perm(r[0][w], r[1][w], 0x5410), __byte_perm(r[0][w], r[1][w], 0x7632),
                             __byte_perm(r[2][w], r[3][w], 0x5410), __byte_perm(r[2][w], r[3][w], 0x7632), b0, b1);
          } else {
            uint32_t a = __byte_perm(r[0][w], r[1][w], 0x5140), c = __byte_perm(r[2][w], r[3][w], 0x5140);
            uint32_t d = __byte_perm(r[0][w], r[1][w], 0x7362), e = __byte_perm(r[2][w], r[3][w], 0x7362);
            if (kHeld == kHeldInt8) {
              a ^= 0x80808080u; c ^= 0x80808080u; d ^= 0x80808080u; e ^= 0x80808080u;
            }
            mma_16816<kHeld>(o[2 * w], half2_of<kHeld, false>(a), half2_of<kHeld, true>(a), half2_of<kHeld, false>(c),
                             half2_of<kHeld, true>(c), b0, b1);
            mma_16816<kHeld>(o[2 * w + 1], half2_of<kHeld, false>(d), half2_of<kHeld, true>(d), half2_of<kHeld, false>(e),
                             half2_of<kHeld, true>(e), b0, b1);
          }
        }
      }
    }
    __syncwarp();
    ask(i + kStages);
  }

  // Over the lanes, the warps and the CTAs of the cluster. The ring is free: every tile that was asked for has arrived.
  cg::cluster_group cluster = cg::this_cluster();
  if (warp < PA_WARPS) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 4);
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 8);
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 16);
      if (g == 0 && tq < 2) {
        wm[ha + e] = m_run[e];
        wl[ha + e] = l_run[e];
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        float x = o[j][e], z = o[j][2 + e];
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        z += __shfl_xor_sync(0xffffffffu, z, 2);
        if (tq < 2) *reinterpret_cast<float2*>(wo + (ha + e) * D + g * (D / 8) + 2 * j) = make_float2(x, z);
      }
    }
  }
  __syncthreads();
  float* cm = reinterpret_cast<float*>(smem + L::kPart);        // the CTA's, behind the first warp's
  float* cl = cm + PA_HEADS;
  float* co = cl + PA_HEADS;
  for (int i = threadIdx.x; i < heads * D; i += PA_THREADS) {
    const int r = i / D, d = i % D;
    float m = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w <= PA_WARPS; ++w)
      if (w < PA_WARPS || rank == 0) m = fmaxf(m, part(w)[r]);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w <= PA_WARPS; ++w) {
      if (w == PA_WARPS && rank != 0) break;
      const float* s = part(w);
      const float half = exp2_of(.5f * (s[r] - ref));
      l = fmaf(s[PA_HEADS + r] * half, half, l);
      x = fmaf(s[2 * PA_HEADS + r * D + d], half * half, x);
    }
    if (p.pieces > 0) {
      const long long at = ((long long)b * p.QH + h0 + r) * p.pieces + rank;
      p.part_o[at * D + d] = x;
      if (d == 0) p.part_ml[at] = make_float2(m, l);
    } else if (cs == 1) {
      p.out[((long long)b * p.QH + h0 + r) * D + d] = __float2bfloat16(l == 0.f ? 0.f : x / l);
    } else {
      co[r * D + d] = x;
      if (d == 0) {
        cm[r] = m;
        cl[r] = l;
      }
    }
  }
  if (cs > 1 && p.pieces == 0) {
    cluster.sync();
    for (int i = rank * PA_THREADS + threadIdx.x; i < heads * D; i += cs * PA_THREADS) {
      const int r = i / D;
      float m = -INFINITY, l = 0.f, x = 0.f, ms[PA_CLUSTER], ls[PA_CLUSTER], xs[PA_CLUSTER];
#pragma unroll
      for (int c = 0; c < PA_CLUSTER; ++c) {                 // all reads on their way at a time: they take 700 cycles each
        const int from = min(c, cs - 1);
        ms[c] = *cluster.map_shared_rank(cm + r, from);
        ls[c] = *cluster.map_shared_rank(cl + r, from);
        xs[c] = *cluster.map_shared_rank(co + i, from);
      }
#pragma unroll
      for (int c = 0; c < PA_CLUSTER; ++c) m = fmaxf(m, ms[c]);
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int c = 0; c < PA_CLUSTER; ++c) {
        const float half = c < cs ? exp2_of(.5f * (ms[c] - ref)) : 0.f;
        l = fmaf(ls[c] * half, half, l);
        x = fmaf(xs[c], half * half, x);
      }
      p.out[((long long)b * p.QH + h0) * D + i] = __float2bfloat16(l == 0.f ? 0.f : x / l);
    }
    cluster.sync();                                          // peers read this CTA's numbers until here
  }
}

// The parts of a query head: grid B * QH, block (D, PA_JOIN): a thread for each dim takes every PA_JOIN-th part, four on their way at a
// time and the next four behind them (60001 tokens 33.1 us, 34.2 without those).
constexpr int PA_JOIN = 4;

template <int D>
__global__ void __launch_bounds__(D * PA_JOIN) paged_join_kernel(const PagedAttnParams p) {
  __shared__ float sm[PA_JOIN], sl[PA_JOIN], so[PA_JOIN][D];
  const int d = threadIdx.x, w = threadIdx.y;
  pdl_wait();
  pdl_trigger();
  const float2* ml = p.part_ml + (long long)blockIdx.x * p.pieces;
  const float* o = p.part_o + (long long)blockIdx.x * p.pieces * D + d;
  float m = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll 2
  for (int c0 = w; c0 < p.pieces; c0 += 4 * PA_JOIN) {
    float2 a[4];
    float y[4], m_new = m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = c0 + e * PA_JOIN, from = min(c, p.pieces - 1);
      a[e] = ml[from];
      y[e] = o[(long long)from * D];
      if (c != from) a[e] = make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) m_new = fmaxf(m_new, a[e].x);
    const float ref = m_new == -INFINITY ? 0.f : m_new, half0 = exp2_of(.5f * (m - ref));
    l = l * half0 * half0;
    x *= half0 * half0;
    float half[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) half[e] = exp2_of(.5f * (a[e].x - ref));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x = fmaf(y[e] * half[e], half[e], x);
      l = fmaf(a[e].y * half[e], half[e], l);
    }
    m = m_new;
  }
  so[w][d] = x;
  if (d == 0) {
    sm[w] = m;
    sl[w] = l;
  }
  __syncthreads();
  if (w != 0) return;
#pragma unroll
  for (int e = 1; e < PA_JOIN; ++e) m = fmaxf(m, sm[e]);
  const float ref = m == -INFINITY ? 0.f : m;
  l = x = 0.f;
#pragma unroll
  for (int e = 0; e < PA_JOIN; ++e) {
    const float half = exp2_of(.5f * (sm[e] - ref));
    l = fmaf(sl[e] * half, half, l);
    x = fmaf(so[e][d], half * half, x);
  }
  p.out[(long long)blockIdx.x * D + d] = __float2bfloat16(l == 0.f ? 0.f : x / l);
}

static int paged_groups(int QH, int KVH) { return (QH / KVH + PA_HEADS - 1) / PA_HEADS; }

// CTAs that share a sequence and KV head: {size of their cluster, 0}, or {1, pieces}. As many as still run at once, three CTAs an SM with a
// twentieth to spare for an uneven spread, and hold 256 tokens each: 32 x 0 to 1980 tokens, 16 / 4 heads, 25.8, 21.0, 18.8, 23.3, 28.5 us
// with clusters of 1, 2, 3, 4, 8; 16 x 900 to 2047 in bf16 28.5, 21.6, 18.5, 17.9, 22.4 with 1, 2, 4, 6, 8. Pieces where clusters of eight
// would fill less than half of the GPU; at other numbers of sequences they are no better (two of 64 x 1500 to 4000: 86 us for 88).
static int2 paged_split(int B, int QH, int KVH, int width, int log_page) {
  const long long units = (long long)B * KVH * paged_groups(QH, KVH), slots = 3LL * num_sms(), tokens = (long long)width << log_page;
  const long long most = std::max(1LL, tokens / 256);
  if (units * PA_CLUSTER <= slots / 2 && most > PA_CLUSTER) return make_int2(1, int(std::min(slots / units, most)));
  return make_int2(int(std::max(1LL, std::min({(long long)PA_CLUSTER, most, slots * 19 / (20 * units)}))), 0);
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
  const int cs = p.pieces > 0 ? 1 : paged_split(p.c.B, p.QH, p.c.KVH, p.c.width, p.c.log_page).x;
  B200_CHECK(launch_pdl(kern, dim3(p.pieces > 0 ? p.pieces : cs, p.c.KVH * p.groups, p.c.B), dim3(PA_THREADS), L::kSmem, st, cs, p));
  if (p.pieces == 0) return 0;
  return static_cast<int>(launch_pdl(paged_join_kernel<D>, dim3(unsigned(p.c.B * p.QH)), dim3(D, PA_JOIN), 0, st, 0, p));
}

template <int D, int kHeld>
static int launch_paged_score(const PagedAttnParams& p, float cap, cudaStream_t st) {
  if (cap > 0.f) return launch_paged<D, kHeld, kScoreCap>(p, st);
  return p.slopes != nullptr ? launch_paged<D, kHeld, kScoreBias>(p, st) : launch_paged<D, kHeld, kScorePlain>(p, st);
}

}  // namespace b200

using namespace b200;

// Bytes of the workspace that b200_paged_attn_append wants (16-byte aligned); 0: none, or sizes that it does not take.
B200_API long long b200_paged_attn_workspace(int B, int QH, int KVH, int width, int log_page, int D) {
  if (B < 1 || KVH < 1 || QH < 1 || QH % KVH != 0 || width < 1 || log_page < 5 || log_page > 10 || (D != 64 && D != 128)) return 0;
  return (long long)B * QH * paged_split(B, QH, KVH, width, log_page).y * (D + 2) * 4;
}

// kqv [B] rows K | Q | V (un-rotated, pitch ld), out [B, QH, D], lens [B], rotary tables [rows, D / 2]. cap > 0: scores c tanh(s / c);
// slopes [QH]: scores minus slope times distance (not both). held: 0 bf16, 1 int8, 2 e4m3.
B200_API int b200_paged_attn_append(const void* kqv, void* pk, void* pv, void* ks, void* vs, const void* table, const void* lens,
                                    const void* cosr, const void* sinr, const void* slopes, void* out, void* workspace, int rows,
                                    long long ld, int B,
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
  p.groups = paged_groups(QH, KVH);
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
  p.pieces = paged_split(B, QH, KVH, width, log_page).y;
  if (p.pieces > 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))
    return static_cast<int>(cudaErrorInvalidValue);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (long long)B * QH * p.pieces * D);
  if (D == 128)
    return held == kHeldBf16   ? launch_paged_score<128, kHeldBf16>(p, cap, st)
           : held == kHeldInt8 ? launch_paged_score<128, kHeldInt8>(p, cap, st)
                               : launch_paged_score<128, kHeldE4m3>(p, cap, st);
  return held == kHeldBf16   ? launch_paged_score<64, kHeldBf16>(p, cap, st)
         : held == kHeldInt8 ? launch_paged_score<64, kHeldInt8>(p, cap, st)
                             : launch_paged_score<64, kHeldE4m3>(p, cap, st);
}
