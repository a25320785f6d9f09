// GQA flash-attention forward under a span mask (span_mask.cu) on tcgen05, head_dim 128 or 64: query t sees the keys [lo, hi).
//
//   x = q k scale;  a cap: x = c tanh(x / c);  a bias: x = x - slope |t - s|;  o = softmax(x over the span) V;  lse = log sum exp x
//
// The arithmetic of a tile is that of the causal forward (flash_attn_tc3.cu): a query row per thread, scores and outputs in tensor
// memory, an online softmax whose reference maximum m moves only when a tile exceeds it by 2^8; P is rounded to bf16 for
// the tensor core, sums and statistics are fp32. What differs is the walk. Packed documents leave a query tile few key tiles (2.5 of
// 1024 / 128 at documents of 200 tokens), and a CTA's life was mostly its own start and end: 11.5 us of 26.7 at 4096 tokens, 32 / 8 heads
// of 128, documents of 700 - barriers and tensor memory, tables, Q, the output's way out. So the CTAs stay:
//
//   * one per SM (head_dim 128, two query tiles side by side) or two (64, one each); the grid has a CTA for every unit of work, those
//     with most to do first, and a CTA that is about to finish one takes the next that the grid has not started (with a fixed share of
//     the list for each the slowest took 20 to 30 % longer than the mean: what a tile costs is not its keys alone);
//   * loads of the next tile's Q, K and V start when the last scores of the present one are done, its first scores when the last P V
//     is, and the output leaves straight from tensor memory while they run.
//
// What bounds it then: the chain scores -> maximum -> exp2 -> P V of two warpgroups (2242 clocks a tile with both of them at it, 2048 of
// exponentials that they share a unit for; a masked tile 3100 to 3500), of which a CTA is in the middle only part of its life: over
// the whole kernel the exponential unit is at 37 %, the tensor core at 36, issue at 35. And masked parts of tiles (18 to 68 % of the pairs
// that are computed at the documents above). Measured, 32 / 8 heads
// of 128: 4096 tokens in documents of 700 97 us with the mask's tables; 16 / 4 heads, a cap, 8192 tokens in documents of 600 85 us.
//
// Roundings to bf16: P, for the tensor core (its sums are fp32), and the output.
//
//   tensor memory, head_dim 128: S_0, S_1 (P over them), O_0, O_1, 128 columns each;  64: S, O, P
#include <climits>

#include "common.cuh"
#include "ptx.cuh"
#include "score_cap.cuh"

namespace b200 {

constexpr float kFsLog2e = 1.4426950408889634f;
constexpr float kFsRescaleStep = 8.f;
// What is done to the scores beside the mask.
constexpr int kSpanOnly = 0, kSpanCap = 1, kSpanBias = 2;

struct FlashSpanParams {
  bf16* o;               // [B, T, QH, D] by element strides
  long long o_bs, o_ts, o_hs;
  float* lse;            // [B, QH, T]
  const int2* spans;     // [B, T]
  const int4* qtab;      // [B, n_tiles]
  const int* order;      // [B, n_units]: groups of kW query tiles, longest first
  int B, T, QH, KVH;
  int n_tiles, n_units;
  int bchunk;            // batch elements whose K and V stay in L2 together
  float scale;
  ScoreCap cap;          // kSpanCap
  const float* slopes;   // kSpanBias: [QH]
  int* status;
};

template <int kD>
struct FS {
  // Query tiles of a unit. (head_dim 128 with one, two CTAs to an SM and one tile of K and V each: documents of 600 tokens 57 -> 54 us, one
  // of 8192 251 -> 268, capped scores no different.)
  static constexpr int kW = kD == 128 ? 2 : 1;
  static constexpr int kCtas = 3 - kW;                                 // CTAs of an SM
  static constexpr int kRing = 2;                                      // tiles of K, and of V, in shared memory
  static constexpr int kFirst = 4;                                     // first softmax warp
  // A warpgroup for the two issuing warps, so that registers can be shared out: of 3 x 168 (2 x 128) at launch
  static constexpr int kRegsFew = kW == 2 ? 88 : 64, kRegsMany = kW == 2 ? 208 : 192;
  static constexpr int kThreads = 32 * kFirst + 128 * kW;
  static constexpr int kTile = 128 * kD * 2;
  static constexpr int kQ = 0;                                         // Q_w
  static constexpr int kK = kW * kTile;                                // K ring
  static constexpr int kV = kK + kRing * kTile;                        // V ring
  static constexpr int kBar = kV + kRing * kTile;
  // q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], early[2], p_full[2], pv_done[2], o_free[2], u_full, u_empty
  static constexpr int kSmem = kBar + 22 * 8 + 16 + 16 + 1024;
  static constexpr bool kOwnP = kD == 64;                              // P beside S, not over it
  static constexpr int kCols = kW == 2 ? 512 : 256;
  static constexpr int kColS = 0, kColO = kW * 128, kColP = kOwnP ? kColO + kD : 0;
};

// A unit of work: kW query tiles of one (batch element, head). Query tile w takes part in steps [st, nt) of the walk over key tiles
// j0, j0 + 1, ...; nt = 0: no row of it sees a key.
struct SpanItem {
  int b, h, unit, j0, steps, st[2], nt[2];
};

template <int kW>
__device__ __forceinline__ void span_item(const FlashSpanParams& p, unsigned i, SpanItem& it) {
  const unsigned per_chunk = p.n_units * p.QH * p.bchunk;
  const unsigned chunk = i / per_chunk, r = i - chunk * per_chunk;
  const unsigned hb = p.QH * min(p.bchunk, int(p.B - chunk * p.bchunk));
  const unsigned rank = r / hb, rest = r - rank * hb, in_chunk = rest / p.QH;
  it.h = rest - in_chunk * p.QH;
  it.b = chunk * p.bchunk + in_chunk;
  it.unit = p.order[size_t(it.b) * p.n_units + rank];
  it.j0 = 0;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    it.st[w] = it.nt[w] = 0;
    const int mt = kW * it.unit + w;
    if (w >= kW || mt >= p.n_tiles) continue;
    const int4 t = p.qtab[size_t(it.b) * p.n_tiles + mt];
    it.st[w] = t.x;
    it.nt[w] = t.y;
  }
  if (kW == 2 && it.nt[0] > 0 && it.nt[1] > 0) {
    // no step without a query tile: the rings of K and V go on only by products (the masked tiles weigh nothing)
    if (it.st[1] > it.nt[0]) it.nt[0] = it.st[1];
    else if (it.st[0] > it.nt[1]) it.nt[1] = it.st[0];
  }
  it.j0 = it.nt[0] > 0 ? (it.nt[1] > 0 ? min(it.st[0], it.st[1]) : it.st[0]) : it.st[1];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if (it.nt[w] == 0) continue;
    it.st[w] -= it.j0;
    it.nt[w] -= it.j0;
  }
  it.steps = max(it.nt[0], it.nt[1]);
}

// The units of a CTA: its own, then those that it takes over. One answer at a time stands in shared memory, until every role has read it.
struct SpanQueue {
  uint64_t* full;            // the answer is there
  uint64_t* empty;           // it has been read: by the MMA warp and every softmax warp
  uint4* answer;
  uint32_t asked;            // answers so far
  // The next unit, -1: there is none (or a wait ran out). The TMA thread asks when it has sent for all of the present one, which is then
  // two tiles from its end (asked at its start, a CTA sat on a second long unit while others ran out of work).
  __device__ __forceinline__ int ask(volatile int* abort_flag) {
    if (asked > 0 && !mbar_wait(empty, (asked - 1) & 1, abort_flag)) return -1;
    mbar_expect_tx(full, 16);
    take_cta(answer, full);
    if (!mbar_wait(full, asked & 1, abort_flag)) return -1;
    ++asked;
    return taken_cta(answer);
  }
  // By a whole warp of another role.
  __device__ __forceinline__ int next(volatile int* abort_flag) {
    if (!mbar_wait_warp(full, asked & 1, abort_flag)) return -1;
    ++asked;
    const int unit = taken_cta(answer);
    fence_proxy_async_smem();                        // read before the next answer is written over it
    __syncwarp();
    if (lane_id() == 0) mbar_arrive(empty);
    return unit;
  }
};

// 32 bytes, one sector, in one store.
__device__ __forceinline__ void fs_store32(void* at, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(__cvta_generic_to_global(at)), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ __forceinline__ float fs_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The keys that a thread's row sees, and those that every row of its warp sees: a tile inside the latter needs no mask, which costs a tile
// three operations per score (a masked tile keeps a warpgroup for 3100 to 3500 clocks, another for 2242). Skipping the 32-key
// blocks of a masked tile that no row of the warp sees was slower: its branches part the loads from the arithmetic.
struct RowSpans {
  int lo, hi, all_lo, all_hi;
};

// Maximum of 32 scores of one row from key `key` on; masked ones become -inf in place.
template <bool kMask>
__device__ __forceinline__ float fs_block_max(uint32_t (&sc)[32], int key, const RowSpans& s) {
  float mx[2] = {-INFINITY, -INFINITY};
  const uint32_t off = uint32_t(key - s.lo), n = uint32_t(s.hi - s.lo);
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    if (kMask) {
      if (off + e >= n) sc[e] = 0xff800000u;
      if (off + (e + 1) >= n) sc[e + 1] = 0xff800000u;
    }
    mx[(e >> 1) & 1] = fs_max3(mx[(e >> 1) & 1], __uint_as_float(sc[e]), __uint_as_float(sc[e + 1]));
  }
  return fmaxf(mx[0], mx[1]);
}

// P = exp2(s * sl2 - m) for scores [kLo, kHi) of one row, packed to bf16 pairs in place; adds to the two partial row sums.
template <int kLo, int kHi>
__device__ __forceinline__ void fs_row_p(uint32_t (&sc)[128], float sl2, float m, float& rs0, float& rs1) {
#pragma unroll
  for (int e = kLo; e < kHi; e += 2) {
    const float p0 = exp2f(fmaf(__uint_as_float(sc[e]), sl2, -m));
    const float p1 = exp2f(fmaf(__uint_as_float(sc[e + 1]), sl2, -m));
    rs0 += p0;
    rs1 += p1;
    const bf162 t = __floats2bfloat162_rn(p0, p1);
    sc[e >> 1] = *reinterpret_cast<const uint32_t*>(&t);
  }
}

template <int kD, int kMod>
__global__ void __launch_bounds__(FS<kD>::kThreads, FS<kD>::kCtas)
flash_fwd_span_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const FlashSpanParams p) {
  using L = FS<kD>;
  constexpr int kW = L::kW, kRing = L::kRing;
  constexpr bool kOwnP = L::kOwnP;
  constexpr uint32_t kTile = L::kTile;
  extern __shared__ uint8_t fs_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(fs_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* q_full = bars;           // Q of an item has arrived
  uint64_t* q_empty = bars + 1;      // every score product of it has read it
  uint64_t* k_full = bars + 2;       // [2]
  uint64_t* k_empty = bars + 4;
  uint64_t* v_full = bars + 6;
  uint64_t* v_empty = bars + 8;
  uint64_t* s_full = bars + 10;      // [w]: scores of the present key tile are in tensor memory
  uint64_t* early = bars + 12;       // [w]: head_dim 64: they have been read; 128: half of P_w has been written (128 arrivals)
  uint64_t* p_full = bars + 14;      // [w]: P_w has been written (128)
  uint64_t* pv_done = bars + 16;     // [w]: O_w includes the key tile whose P V was committed last
  uint64_t* o_free = bars + 18;      // [w]: O_w of an item has been read (128)
  uint64_t* u_full = bars + 20;      // the next unit's number has arrived
  uint64_t* u_empty = bars + 21;     // every role has read it
  uint4* answer = reinterpret_cast<uint4*>(bars + 22);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(u_full, 1);
    mbar_init(u_empty, 1 + 4 * kW);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&early[s], 128);
      mbar_init(&p_full[s], 128);
      mbar_init(&pv_done[s], 1);
      mbar_init(&o_free[s], 128);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) tmem_alloc(tmem_slot, L::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  constexpr uint32_t kColS = L::kColS, kColO = L::kColO, kColP = L::kColP;
  pdl_wait();                            // by every role: their bounded waits start counting behind it
  pdl_trigger();
  SpanItem it;
  SpanQueue queue = {u_full, u_empty, answer, 0};

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    setmaxnreg_dec<L::kRegsFew>();
    if (lane == 0) {
      int g = 0, active = 0;             // key tiles and items so far
      bool ok = true;
      for (int unit = blockIdx.x; ok && unit >= 0; unit = queue.ask(abort_flag)) {
        span_item<kW>(p, unit, it);
        if (it.steps == 0) continue;
        const int kvh = it.h / (p.QH / p.KVH);
        if (active > 0 && !mbar_wait(q_empty, (active - 1) & 1, abort_flag)) break;
        ++active;
        mbar_expect_tx(q_full, ((it.nt[0] > 0) + (it.nt[1] > 0)) * kTile);
        for (int w = 0; w < kW; ++w) {
          if (it.nt[w] == 0) continue;
          uint8_t* sQ = smem + L::kQ + w * kTile;
          tma_load_4d(sQ, &tmQ, q_full, 0, it.h, (kW * it.unit + w) * 128, it.b);
          if (kD == 128) tma_load_4d(sQ + 16384, &tmQ, q_full, 64, it.h, (kW * it.unit + w) * 128, it.b);
        }
        for (int j = 0; j < it.steps; ++j, ++g) {
          const int s = g % kRing, key = (it.j0 + j) * 128;
          const uint32_t par = ((g / kRing) & 1) ^ 1;
          if (!mbar_wait(&k_empty[s], par, abort_flag)) { ok = false; break; }
          uint8_t* sK = smem + L::kK + s * kTile;
          mbar_expect_tx(&k_full[s], kTile);
          tma_load_4d(sK, &tmK, &k_full[s], 0, kvh, key, it.b);
          if (kD == 128) tma_load_4d(sK + 16384, &tmK, &k_full[s], 64, kvh, key, it.b);
          if (!mbar_wait(&v_empty[s], par, abort_flag)) { ok = false; break; }
          uint8_t* sV = smem + L::kV + s * kTile;
          mbar_expect_tx(&v_full[s], kTile);
          tma_load_4d(sV, &tmV, &v_full[s], 0, kvh, key, it.b);
          if (kD == 128) tma_load_4d(sV + 16384, &tmV, &v_full[s], 64, kvh, key, it.b);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    setmaxnreg_dec<L::kRegsFew>();
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, 128, 0, 0);
    constexpr uint32_t idesc_pv = umma_idesc_bf16(128, kD, 0, 1);
    int g0 = 0, active = 0;
    int tiles0 = 0, tiles1 = 0, outs0 = 0, outs1 = 0;      // key tiles and outputs that each warpgroup has had
    bool ok = true;
    for (int unit = blockIdx.x; ok && unit >= 0; unit = queue.next(abort_flag)) {
      span_item<kW>(p, unit, it);
      if (it.steps == 0) continue;
      auto issue_s = [&](int w, int j) {
        const uint64_t dQ = umma_smem_desc(smem_u32(smem + L::kQ + w * kTile), 16, 1024);
        const uint64_t dK = umma_smem_desc(smem_u32(smem + L::kK + ((g0 + j) % kRing) * kTile), 16, 1024);
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;      // in the descriptors' 16-byte units
          umma_bf16_ss_warp(tmem_base + kColS + w * 128, dQ + off, dK + off, idesc_s, kk != 0);
        }
        umma_commit_warp(&s_full[w]);
      };
      // the scores of step j have been issued for every query tile
      auto k_used = [&](int j) {
        umma_commit_warp(&k_empty[(g0 + j) % kRing]);
        if (j + 1 == it.steps) umma_commit_warp(q_empty);
      };
      auto issue_pv = [&](int w, int j, int lo, int hi) {
        const uint64_t dV = umma_smem_desc(smem_u32(smem + L::kV + ((g0 + j) % kRing) * kTile), 16384, 1024);
        const uint32_t tP = tmem_base + kColP + w * 128;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          if (kk >= lo && kk < hi)
            umma_bf16_ts_warp(tmem_base + kColO + w * 128, tP + kk * 8, dV + kk * 128, idesc_pv, j != it.st[w] || kk != 0);
      };
      ok = mbar_wait_warp(q_full, active & 1, abort_flag) && mbar_wait_warp(&k_full[g0 % kRing], (g0 / kRing) & 1, abort_flag);
      // scores with a P beside them: the last ones of the item before have to have been read
      if (ok && kOwnP && tiles0 > 0) ok = mbar_wait_warp(&early[0], (tiles0 - 1) & 1, abort_flag);
      if (!ok) break;
      ++active;
      tc_fence_after();
      for (int w = 0; w < kW; ++w)
        if (it.nt[w] > 0 && it.st[w] == 0) issue_s(w, 0);
      k_used(0);
      for (int j = 0; j < it.steps && ok; ++j) {
        const int g = g0 + j;
        bool v_ready = false, k_ready = false;
        // The next scores of query tile w: with a P of its own as soon as the warpgroup has read the present ones, else behind the
        // P V whose P lies over them.
        auto next_s = [&](int w) {
          if (!k_ready && !mbar_wait_warp(&k_full[(g + 1) % kRing], ((g + 1) / kRing) & 1, abort_flag)) return false;
          k_ready = true;
          tc_fence_after();
          issue_s(w, j + 1);
          return true;
        };
        if (kOwnP && j + 1 < it.steps) {
          ok = mbar_wait_warp(&early[0], tiles0 & 1, abort_flag) && next_s(0);
          if (!ok) break;
          k_used(j + 1);
        }
        for (int w = 0; w < kW && ok; ++w) {
          if (j >= it.nt[w]) continue;
          if (!kOwnP && j < it.st[w]) {                      // its first scores come with this step's products
            if (j + 1 == it.st[w]) ok = next_s(w);
            continue;
          }
          const uint32_t ph = (w == 0 ? tiles0 : tiles1) & 1;
          const int outs = w == 0 ? outs0 : outs1;
          if (j == it.st[w] && outs > 0 && !mbar_wait_warp(&o_free[w], (outs - 1) & 1, abort_flag)) { ok = false; break; }
          if (!mbar_wait_warp(kOwnP ? &p_full[w] : &early[w], ph, abort_flag)) { ok = false; break; }
          if (!v_ready) {
            if (!mbar_wait_warp(&v_full[g % kRing], (g / kRing) & 1, abort_flag)) { ok = false; break; }
            v_ready = true;
          }
          tc_fence_after();
          if (kOwnP) {
            issue_pv(w, j, 0, 8);
          } else {
            issue_pv(w, j, 0, 4);
            if (!mbar_wait_warp(&p_full[w], ph, abort_flag)) { ok = false; break; }
            tc_fence_after();
            issue_pv(w, j, 4, 8);
          }
          umma_commit_warp(&pv_done[w]);
          if (w == 0) ++tiles0;
          else ++tiles1;
          if (!kOwnP && j + 1 < it.nt[w] && !next_s(w)) { ok = false; break; }
        }
        if (!ok) break;
        if (!kOwnP && j + 1 < it.steps) k_used(j + 1);
        umma_commit_warp(&v_empty[g % kRing]);
      }
      g0 += it.steps;
      outs0 += it.nt[0] > 0;
      outs1 += it.nt[1] > 0;
    }
  } else if (warp < L::kFirst) {
    setmaxnreg_dec<L::kRegsFew>();
  } else {
    // ---------------------------------------------------------------- softmax warpgroup w: one query tile
    setmaxnreg_inc<L::kRegsMany>();
    const int w = (warp - L::kFirst) >> 2;
    const int q = warp & 3;
    const int rloc = q * 32 + lane;
    const uint32_t lane_sel = uint32_t(q * 32) << 16;
    const uint32_t tS = tmem_base + lane_sel + kColS + w * 128;
    const uint32_t tO = tmem_base + lane_sel + kColO + w * 128;
    const uint32_t tP = tmem_base + lane_sel + kColP + w * 128;
    // log2 units per score; a bias leaves them in log2 units, a cap is taken on the way into the exponentials
    const float sl2 = kMod == kSpanCap || kMod == kSpanBias ? 1.f : p.scale * kFsLog2e;
    const float bias_sl2 = p.scale * kFsLog2e;
    const int T = p.T;
    int done = 0;                          // key tiles so far
    bool ok = true;
    // the next unit's tables and this row's keys in it are asked for before the present one's output is waited for
    int unit = blockIdx.x, b = 0, h = 0, mt = -1, first = 0, my_tiles = 0;      // mt < 0: nothing in the unit for this warpgroup
    int2 span = make_int2(0, 0);
    auto next_unit = [&]() {
      if (unit < 0) return false;
      SpanItem u;
      span_item<kW>(p, unit, u);
      mt = kW * u.unit + w;
      if (mt >= p.n_tiles) mt = -1;
      b = u.b;
      h = u.h;
      first = u.j0 + u.st[w];
      my_tiles = u.nt[w] - u.st[w];
      // (rows past the end as the last one: nobody stores them)
      if (mt >= 0) span = p.spans[size_t(b) * T + min(mt * 128 + rloc, T - 1)];
      return true;
    };
    bool more = next_unit();
    while (ok && more) {
      if (mt < 0) {
        unit = queue.next(abort_flag);
        more = next_unit();
        continue;
      }
      const int row = mt * 128 + rloc;
      RowSpans spans;
      {
        spans.lo = span.x;
        spans.hi = span.y;
        spans.all_lo = __reduce_max_sync(0xffffffffu, span.y <= span.x ? INT_MAX : span.x);
        spans.all_hi = __reduce_min_sync(0xffffffffu, span.y);
      }
      const float slope2 = kMod == kSpanBias ? p.slopes[h] * kFsLog2e : 0.f;
      float m_ref = -INFINITY, l_run = 0.f;          // reference maximum (log2 units) and the row sum relative to it
      for (int j = 0; j < my_tiles && ok; ++j, ++done) {
        if (!mbar_wait(&s_full[w], done & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const int key0 = (first + j) * 128;
        const bool full = key0 >= spans.all_lo && key0 + 128 <= spans.all_hi;
        // The whole row in one go: four loads, one wait.
        uint32_t sc[128];
        tmem_ld_32x32b_x32(tS, *reinterpret_cast<uint32_t(*)[32]>(&sc[0]));
        tmem_ld_32x32b_x32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&sc[32]));
        tmem_ld_32x32b_x32(tS + 64, *reinterpret_cast<uint32_t(*)[32]>(&sc[64]));
        tmem_ld_32x32b_x32(tS + 96, *reinterpret_cast<uint32_t(*)[32]>(&sc[96]));
        tmem_ld_wait();
        if (kOwnP) {                       // the tensor core may write the next scores over these
          tc_fence_before();
          mbar_arrive(&early[w]);
        }
        bool cap_now = false;              // kSpanCap: the exponentials take the cap
        if constexpr (kMod == kSpanCap) {
          const int tier = cap_tier(sc, p.cap);
          cap_now = tier == kCapNear && full;
          if (!cap_now) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
              cap_scores(*reinterpret_cast<uint32_t(*)[32]>(&sc[32 * b]), p.cap, tier);
          }
        } else if constexpr (kMod == kSpanBias) {
          const float dist = float(key0 - row);
#pragma unroll
          for (int e = 0; e < 128; ++e) sc[e] = __float_as_uint(fmaf(__uint_as_float(sc[e]), bias_sl2, -slope2 * fabsf(dist + float(e))));
        }
        float mx = -INFINITY;
        if (full) {
#pragma unroll
          for (int b = 0; b < 4; ++b) mx = fmaxf(mx, fs_block_max<false>(*reinterpret_cast<uint32_t(*)[32]>(&sc[32 * b]), 0, spans));
        } else {
#pragma unroll
          for (int b = 0; b < 4; ++b)
            mx = fmaxf(mx, fs_block_max<true>(*reinterpret_cast<uint32_t(*)[32]>(&sc[32 * b]), key0 + 32 * b, spans));
        }
        mx *= sl2;
        if (kMod == kSpanCap && cap_now) mx = cap_any(mx, p.cap);          // the cap keeps the order of the scores
        // A row that has seen nothing so far (its document begins behind the tile's first keys) has nothing to rescale: its weights
        // were 0. With the rescaling of such rows most tiles of packed documents took twice as long.
        if (m_ref == -INFINITY) m_ref = mx;
        if (j > 0) {
          const bool need = mx > m_ref + kFsRescaleStep;
          if (__any_sync(0xffffffffu, need)) {
            // O_w holds the key tiles up to j - 1 once their P V has completed
            if (!__all_sync(0xffffffffu, mbar_wait(&pv_done[w], (done - 1) & 1, abort_flag))) { ok = false; break; }
            tc_fence_after();
            const float corr = need ? exp2f(m_ref - mx) : 1.f;
            l_run *= corr;
#pragma unroll 1
            for (int c = 0; c < kD / 16; ++c) {
              uint32_t t[16];
              tmem_ld_32x32b_x16(tO + c * 16, t);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) t[e] = __float_as_uint(__uint_as_float(t[e]) * corr);
              tmem_st_32x32b_x16(tO + c * 16, t);
            }
            tmem_st_wait();
            if (need) m_ref = mx;
          }
        }
        // P = exp2(s - m) as bf16 pairs, packed in place over the first 64 registers, and its row sum
        float rs0 = 0.f, rs1 = 0.f;
        const float m_sub = m_ref == -INFINITY ? 0.f : m_ref;      // nothing seen yet: exp2(-inf) is 0
        if (kOwnP) {
          if (kMod == kSpanCap && cap_now) cap_row_p<0, 128>(sc, p.cap, m_sub, rs0, rs1);
          else fs_row_p<0, 128>(sc, sl2, m_sub, rs0, rs1);
          // P_w has been read (across items too: the output's way out waited for the last one)
          if (j > 0 && !__all_sync(0xffffffffu, mbar_wait(&pv_done[w], (done - 1) & 1, abort_flag))) { ok = false; break; }
          tc_fence_after();
        } else {
          // head_dim 128: the next scores wait for this P V, so its first half is handed over early
          if (kMod == kSpanCap && cap_now) cap_row_p<0, 64>(sc, p.cap, m_sub, rs0, rs1);
          else fs_row_p<0, 64>(sc, sl2, m_sub, rs0, rs1);
          tmem_st_32x32b_x16(tP, *reinterpret_cast<const uint32_t(*)[16]>(&sc[0]));
          tmem_st_32x32b_x16(tP + 16, *reinterpret_cast<const uint32_t(*)[16]>(&sc[16]));
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&early[w]);
          if (kMod == kSpanCap && cap_now) cap_row_p<64, 128>(sc, p.cap, m_sub, rs0, rs1);
          else fs_row_p<64, 128>(sc, sl2, m_sub, rs0, rs1);
        }
#pragma unroll
        for (int c = kOwnP ? 0 : 2; c < 4; ++c)
          tmem_st_32x32b_x16(tP + c * 16, *reinterpret_cast<const uint32_t(*)[16]>(&sc[16 * c]));
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[w]);
        l_run += rs0 + rs1;
      }
      if (!ok) break;
      // The output: a row's 32 columns at a time from tensor memory to bf16 to its place, a whole sector to a store (a tile through shared
      // memory and the copy engine kept the warpgroup for 4400 clocks, twice the time of a key tile).
      bf16* out = p.o + b * p.o_bs + (long long)min(row, T - 1) * p.o_ts + h * p.o_hs;
      float* lse = p.lse + (size_t(b) * p.QH + h) * T + min(row, T - 1);
      const bool any = my_tiles > 0, live = row < T;
      unit = queue.next(abort_flag);
      more = next_unit();
      if (any) {
        if (!__all_sync(0xffffffffu, mbar_wait(&pv_done[w], (done - 1) & 1, abort_flag))) { ok = false; break; }
        tc_fence_after();
      }
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
#pragma unroll
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t r[32];
        if (any) {
          tmem_ld_32x32b_x32(tO + c * 32, r);
          tmem_ld_wait();
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const bf162 t = __floats2bfloat162_rn(__uint_as_float(r[e]) * inv, __uint_as_float(r[e + 1]) * inv);
          r[e >> 1] = l_run == 0.f ? 0u : *reinterpret_cast<const uint32_t*>(&t);      // (nothing seen, or nothing in tensor memory)
        }
        if (live) {
          fs_store32(out + c * 32, &r[0]);
          fs_store32(out + c * 32 + 16, &r[8]);
        }
      }
      if (any) {
        tc_fence_before();
        mbar_arrive(&o_free[w]);
      }
      if (live)
        *lse = l_run != l_run ? l_run : l_run > 0.f ? m_ref * 0.6931471805599453f + logf(l_run) : -INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kCols);
  }
  if (threadIdx.x == 0 && *abort_flag != 0 && p.status != nullptr) {
    if (atomicCAS(p.status, 0, int(*abort_flag)) == 0) p.status[1] = 303;
  }
}

template <int kD, int kMod>
static int launch_fwd_span(FlashSpanParams p, const TensorMap (&m)[3], cudaStream_t st) {
  using L = FS<kD>;
  static bool configured = false;
  if (!configured) {
    B200_CHECK(cudaFuncSetAttribute(flash_fwd_span_kernel<kD, kMod>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem));
    configured = true;
  }
  p.n_units = (p.n_tiles + L::kW - 1) / L::kW;
  const long long items = (long long)p.n_units * p.QH * p.B;
  if (items > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
  if (L::kW == 2) p.order += (size_t)p.B * p.n_tiles;      // the orders of pairs stand behind those of single tiles
  return static_cast<int>(launch_pdl(flash_fwd_span_kernel<kD, kMod>, dim3(unsigned(items)), dim3(L::kThreads), L::kSmem, st, 0, *m[0],
                                     *m[1], *m[2], p));
}

}  // namespace b200

using namespace b200;

// q, k, v (already rotated) and o [B, T, heads, D] by element strides (batch, token, head each; of o multiples of 16), lse [B, QH, T];
// spans, qtab and order as b200_span_mask makes them. cap > 0: scores c tanh(s / c); slopes [QH]: scores minus slope times distance (not
// both).
B200_API int b200_flash_fwd_span(const void* q, const void* k, const void* v, void* o, void* lse, const void* spans, const void* qtab,
                                 const void* order, const long long* strides, int B, int T, int QH, int KVH, int D, float scale,
                                 float cap, const void* slopes, cudaStream_t st) {
  if (B <= 0 || T <= 0) return 0;
  if ((D != 128 && D != 64) || KVH <= 0 || QH % KVH != 0) return static_cast<int>(cudaErrorInvalidValue);
  if (cap < 0.f || (cap > 0.f && slopes != nullptr)) return static_cast<int>(cudaErrorInvalidValue);
  for (int i = 0; i < 12; ++i)
    if (strides[i] % (i < 9 ? 8 : 16) != 0) return static_cast<int>(cudaErrorInvalidValue);
  if ((reinterpret_cast<uintptr_t>(o) & 31) != 0) return static_cast<int>(cudaErrorInvalidValue);
  const TensorMap m[3] = {get_tensor_map_bthd(q, B, T, QH, D, strides[0], strides[1], strides[2], 128, 64),
                          get_tensor_map_bthd(k, B, T, KVH, D, strides[3], strides[4], strides[5], 128, 64),
                          get_tensor_map_bthd(v, B, T, KVH, D, strides[6], strides[7], strides[8], 128, 64)};
  for (const TensorMap& x : m)
    if (!x) return static_cast<int>(cudaErrorInvalidValue);
  FlashSpanParams p = {};
  p.o = static_cast<bf16*>(o);
  p.o_bs = strides[9]; p.o_ts = strides[10]; p.o_hs = strides[11];
  p.lse = static_cast<float*>(lse);
  p.spans = static_cast<const int2*>(spans);
  p.qtab = static_cast<const int4*>(qtab);
  p.order = static_cast<const int*>(order);
  p.B = B; p.T = T; p.QH = QH; p.KVH = KVH;
  p.n_tiles = (T + 127) / 128;
  {
    const double per_batch = 2.0 * T * D * 2.0 * KVH;             // K and V; about two thirds of the L2 is budgeted
    const int bc = int(80.0e6 / per_batch);
    p.bchunk = bc < 1 ? 1 : (bc > B ? B : bc);
  }
  p.scale = scale;
  p.cap = make_score_cap(scale, cap);
  p.slopes = static_cast<const float*>(slopes);
  p.status = status_ptr();
  if (D == 128) {
    if (cap > 0.f) return launch_fwd_span<128, kSpanCap>(p, m, st);
    return slopes != nullptr ? launch_fwd_span<128, kSpanBias>(p, m, st) : launch_fwd_span<128, kSpanOnly>(p, m, st);
  }
  if (cap > 0.f) return launch_fwd_span<64, kSpanCap>(p, m, st);
  return slopes != nullptr ? launch_fwd_span<64, kSpanBias>(p, m, st) : launch_fwd_span<64, kSpanOnly>(p, m, st);
}
