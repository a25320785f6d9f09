// Attention of drafted tokens over a KV cache (head_dim 128 or 64): n <= 64 drafts per sequence, a tree of them, one of them in
// the plain decoded step.
//
// Draft i of sequence b stands at position len + depth(i). It sees the len cached keys, its ancestors and itself. K, Q, V come
// packed from the projection, un-rotated: a first kernel rotates Q and K and appends K and V to the caches at len + i; a draft that
// has no room there is not seen by any, itself included.
//
//   x = q k scale, capped (c tanh(x / c)) or biased (x - slope |distance|);  o = softmax(x) V
//
// The rows of a tile are the drafts times the query heads that share a KV head: every key is read once for all of them, which is
// all that bounds the kernel while there are few (64 rows of head_dim 128 do 48 multiply-adds per byte read, two products for the scores
// and one for the values; the tensor core makes 96 of them, its tiles have 128 rows). The work is one list of 128-key tiles, over
// sequences, KV heads and groups of up to 256 rows, the drafts a tile of their own behind each sequence's cached ones; the list is cut into
// as many equal pieces as there are SMs, so sequences of any mix of lengths keep all of them busy. A piece that is not all of its rows'
// keys leaves its maximum, sum and values in a workspace, and a last kernel joins them in the order of the keys.
//
// Roles: warp 0 streams Q and the tiles of K and V by TMA, warp 1 issues the products (scores Q K^T into tensor memory, O += P V
// from it), and two warpgroups (warps 4..11) do the softmax, a row per thread, each with scores and an output of its own in tensor memory
// (columns S_0, S_1, O_0, O_1; P lies over S). A group of more than 128 rows gives each warpgroup a tile of rows; one of up to 128
// gives them the odd and the even key tiles, and the first one adds up what the two have. Either way the tensor core works for one
// while the other is in its exponentials: with one warpgroup, and Q as one part, a tile took 2.1 us at 128 rows of head_dim 128 where its
// 64 KiB arrive in 1.5. The whole call at 32 drafts, 32 / 8 heads of 128, one after the other on caches that are not in L2: 17.5 us at
// 1000 keys, 68 to 71 at 60000, 111 to 114 at 120000: 0.71 us per 1000 keys from there on, 5.8 TB/s, and 26 to 28 us of three launches,
// the ramp and the join (a tree of 32 over 60001 keys of a cache of 65536: 73 to 77).
//
// Roundings to bf16: rotated K and V, as the caches hold them; Q in two parts, which is 16 bits; P, for the tensor core (sums of P and
// the accumulators are fp32); the result.
// Cached rows past the length, which may hold anything, are masked as scores and cleared as values. Every wait is bounded (see
// ptx.cuh).
#include <algorithm>

#include "common.cuh"
#include "ptx.cuh"
#include "score_cap.cuh"

namespace b200 {

constexpr float kTaLog2e = 1.4426950408889634f;
constexpr float kTaRescaleStep = 8.f;
constexpr int TA_THREADS = 384;
// 384 x 168 registers at launch, shared out again: 88 for each thread of the first warpgroup, 208 for each of the other two (88 + 2 * 208 =
// 3 * 168): a row's 128 scores and the arithmetic on them stay in registers.
constexpr int TA_REGS_FEW = 88, TA_REGS_MANY = 208;
constexpr int TA_MAX_DRAFTS = 64;                        // the bits of a draft's mask
constexpr int kTreePlain = 0, kTreeCap = 1, kTreeBias = 2;

struct TreeParams {
  const bf16* kqv;          // [B * n][ld]: K | Q | V
  bf16* kc;                 // [B, KVH, Tmax, D]
  bf16* vc;
  bf16* q;                  // [2, B, n, QH, D]: rotated, as bf16 and what that leaves, as bf16 again
  bf16* out;                // [B, n, QH, D]
  const int* lens;          // [B]
  const unsigned long long* tree;   // [B, n]: bit j: draft i sees draft j
  const float* cosr;        // [rows, D / 2]
  const float* sinr;
  const float* slopes;      // kTreeBias: [QH]
  float4* part_o;           // [2 * CTAs][2][D / 4][128]: a CTA's first and last piece, row tile in the group; rows side by side
  float2* part_ml;          // [2 * CTAs][2][128]: maximum (log2 units), sum
  int B, n, QH, KVH, Tmax, table_rows;
  long long ld;
  int R, tok, groups;       // query heads of a KV head; drafts of a row tile (R tok <= 128); groups of two row tiles (or one)
  int ctas;                 // pieces of the list
  int* arrived;             // [B * KVH * groups]: pieces that are done, where the last of them joins them all; else null
  float scale;
  ScoreCap cap;             // kTreeCap
  int* status;
};

// kPair: there are groups of two row tiles.
template <int kD, bool kPair>
struct TA {
  static constexpr int kTile = 128 * kD * 2;
  // Rings of K and V. Two row tiles take more of the memory, and twice the time for a key tile.
  static constexpr int kStK = kD == 64 ? 4 : kPair ? 1 : 2, kStV = kD == 64 ? 4 : kPair ? 2 : 3;
  static constexpr int kQ = 0, kK = (kPair ? 4 : 2) * kTile, kV = kK + kStK * kTile;       // Q: the two parts of each row tile
  static constexpr int kBar = kV + kStV * kTile;
  // k_full, k_empty [kStK]; v_full, v_empty [kStV]; q_full, q_empty; s_full, p_half, p_full, pv_done, o_free [2]; ml_full, ml_empty;
  // part_out, last_known
  static constexpr int kBars = 2 * kStK + 2 * kStV + 2 + 10 + 2 + 2;
  static constexpr int kMl = kBar + kBars * 8 + 48;
  static constexpr int kSmem = kMl + 128 * 8 + 1024;
  static constexpr uint32_t kColS = 0, kColO = 256;                             // [2] each, 128 columns apart
};

// A stretch of one (sequence, KV head, row group): tiles [t0, t1) of its nt, the last of which are the drafts.
struct TreeSeg {
  int b, kvh, rg, t0, t1, nt, len;
  bool pair;                // two row tiles
};

__device__ __forceinline__ int tree_len(const TreeParams& p, int b) { return checked_index(p.lens[b], p.Tmax, p.status, 350); }
__device__ __forceinline__ int tree_tiles(int len) { return (len + 127) / 128 + 1; }

// The list's length, and the sequence that its tile `at` belongs to with that sequence's first tile; by a whole warp.
__device__ __forceinline__ long long tree_total(const TreeParams& p, int lane) {
  long long sum = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) sum += __reduce_add_sync(0xffffffffu, b0 + lane < p.B ? tree_tiles(tree_len(p, b0 + lane)) : 0);
  return sum * (p.KVH * p.groups);
}
__device__ __forceinline__ int tree_find(const TreeParams& p, long long at, int lane, long long& first) {
  const int per = p.KVH * p.groups;
  first = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int v = b0 + lane < p.B ? tree_tiles(tree_len(p, b0 + lane)) : 0;
    int before = v;                                      // of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, at < first + (long long)before * per);
    if (hit != 0) {
      const int l = __ffs(hit) - 1;
      first += (long long)__shfl_sync(0xffffffffu, before - v, l) * per;
      return b0 + l;
    }
    first += (long long)__shfl_sync(0xffffffffu, before, 31) * per;
  }
  return p.B;
}

// The list is cut into as many pieces as there are CTAs, or tiles if those are fewer: piece c has the tiles from c total / G on.
__device__ __forceinline__ long long tree_pieces_of(const TreeParams& p, long long total) { return total < p.ctas ? total : p.ctas; }

// Walks the pieces of one CTA.
struct TreeWalk {
  long long left;           // tiles that are left to it
  int b, idx, tile;         // where it stands: sequence, KV head * groups + group, tile
  __device__ __forceinline__ bool next(const TreeParams& p, TreeSeg& s) {
    if (left <= 0) return false;
    s.b = b;
    s.len = tree_len(p, b);
    s.nt = tree_tiles(s.len);
    s.kvh = idx / p.groups;
    s.rg = idx % p.groups;
    s.pair = p.n > (2 * s.rg + 1) * p.tok;        // (never where no group has two)
    s.t0 = tile;
    s.t1 = int(min((long long)s.nt, tile + left));
    left -= s.t1 - s.t0;
    tile = s.t1;
    if (tile == s.nt) {
      tile = 0;
      if (++idx == p.KVH * p.groups) {
        idx = 0;
        ++b;
      }
    }
    return true;
  }
};

__device__ __forceinline__ void ta_unpack(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// 8 elements from chunk `c` of the head at `x`, rotated by the table row of `pos` (half-split pairs) and rounded to bf16, the type of the
// cache and of the tensor core's operands; in `rest` what that leaves, as bf16.
template <int kD>
__device__ __forceinline__ uint4 ta_rotated(const TreeParams& p, const bf16* x, int c, int pos, uint4& rest) {
  constexpr int kHalf = kD / 16;
  float a[8], b[8];
  ta_unpack(reinterpret_cast<const uint4*>(x)[c], a);
  ta_unpack(reinterpret_cast<const uint4*>(x)[c ^ kHalf], b);
  const int j = (c % kHalf) * 8;
  const size_t row = size_t(min(max(pos, 0), p.table_rows - 1)) * (kD / 2) + j;
  uint4 u;
  uint32_t *w = reinterpret_cast<uint32_t*>(&u), *v = reinterpret_cast<uint32_t*>(&rest);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float4 cs = *reinterpret_cast<const float4*>(p.cosr + row + 4 * h), sn = *reinterpret_cast<const float4*>(p.sinr + row + 4 * h);
    const float cv[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = a[4 * h + e] * cv[e], z = b[4 * h + e] * sv[e];
      y[e] = c < kHalf ? x - z : x + z;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bf162 t = __floats2bfloat162_rn(y[2 * e], y[2 * e + 1]);
      const float2 f = __bfloat1622float2(t);
      const bf162 l = __floats2bfloat162_rn(y[2 * e] - f.x, y[2 * e + 1] - f.y);
      w[2 * h + e] = *reinterpret_cast<const uint32_t*>(&t);
      v[2 * h + e] = *reinterpret_cast<const uint32_t*>(&l);
    }
  }
  return u;
}

// Whom draft i of sequence b sees; bits of drafts that are not there count for nothing, neither here nor in its depth.
__device__ __forceinline__ unsigned long long tree_bits(const TreeParams& p, int b, int i) {
  return p.tree[size_t(b) * p.n + i] & (~0ull >> (64 - p.n));
}
__device__ __forceinline__ int tree_depth(unsigned long long bits) { return max(__popcll(bits) - 1, 0); }

// A thread per 16 bytes of the packed projection: K (rotated) and V to the caches, Q (rotated, in two parts) to its workspace.
template <int kD>
__global__ void __launch_bounds__(256)
tree_append_kernel(const TreeParams p) {
  constexpr int kChunks = kD / 8;
  pdl_wait();
  pdl_trigger();
  const int heads = p.QH + 2 * p.KVH;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (p.arrived != nullptr)
    for (long long c = i; c < (long long)p.B * p.KVH * p.groups; c += (long long)gridDim.x * 256) p.arrived[c] = 0;
  if (i >= (long long)p.B * p.n * heads * kChunks) return;
  const int c = int(i % kChunks), head = int(i / kChunks % heads);
  const long long row = i / kChunks / heads;
  const int b = int(row / p.n), d = int(row % p.n);
  const int len = tree_len(p, b), pos = len + tree_depth(tree_bits(p, b, d));
  const bf16* x = p.kqv + row * p.ld + head * kD;
  if (head >= p.KVH && head < p.KVH + p.QH) {
    uint4 rest;
    const uint4 u = ta_rotated<kD>(p, x, c, pos, rest);
    bf16* q = p.q + (row * p.QH + head - p.KVH) * kD;
    reinterpret_cast<uint4*>(q)[c] = u;
    reinterpret_cast<uint4*>(q + (size_t)p.B * p.n * p.QH * kD)[c] = rest;
    return;
  }
  const bool value = head >= p.KVH;
  if (len + d >= p.Tmax) return;
  uint4 rest;                                            // (the cache holds bf16)
  const uint4 u = value ? reinterpret_cast<const uint4*>(x)[c] : ta_rotated<kD>(p, x, c, pos, rest);
  const int kvh = value ? head - p.KVH - p.QH : head;
  reinterpret_cast<uint4*>((value ? p.vc : p.kc) + ((size_t(b) * p.KVH + kvh) * p.Tmax + len + d) * kD)[c] = u;
}

// 16-byte chunk `c` of row `r` in a tile of 128-byte rows (64 columns a box, 16 KiB apart), as TMA writes it.
__device__ __forceinline__ uint4* ta_chunk(uint8_t* tile, int r, int c) {
  return reinterpret_cast<uint4*>(tile + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Pieces [c0, c1] that a (sequence, KV head, row group) is cut into, whose tiles are [t0, t0 + nt) of the list: tile t is in piece
// ((t + 1) G - 1) / total. Nearly all lists are short enough for 32-bit division.
struct TreePieces {
  int c0, c1, late;         // late: the first one began with other rows
  // of row tile w in the group
  __device__ __forceinline__ int slot(int c, int w) const { return 4 * c + (c == c0 ? 2 * late : 0) + w; }
};

__device__ __forceinline__ TreePieces tree_pieces(const TreeParams& p, unsigned long long total, unsigned long long t0, int nt) {
  const unsigned G = unsigned(tree_pieces_of(p, total));
  TreePieces x;
  if ((total + 1) * (G + 1) < 0x100000000ull) {
    x.c0 = int((unsigned(t0 + 1) * G - 1) / unsigned(total));
    x.c1 = int((unsigned(t0 + nt) * G - 1) / unsigned(total));
    x.late = unsigned(x.c0) * unsigned(total) / G < unsigned(t0) ? 1 : 0;
  } else {
    x.c0 = int(((t0 + 1) * G - 1) / total);
    x.c1 = int(((t0 + nt) * G - 1) / total);
    x.late = (unsigned long long)x.c0 * total / G < t0 ? 1 : 0;
  }
  return x;
}

// First list position of a stretch's (sequence, KV head, row group).
__device__ __forceinline__ unsigned long long combo_first(const TreeParams& p, const TreeSeg& s) {
  unsigned long long before = 0;
  for (int b = 0; b < s.b; ++b) before += tree_tiles(tree_len(p, b));
  return before * (p.KVH * p.groups) + (unsigned long long)(s.kvh * p.groups + s.rg) * s.nt;
}

// 4 kQuads columns of one row's result from its pieces, in the order of the keys; some pieces' loads at a time.
template <int kD, int kQuads>
__device__ __forceinline__ void tree_join_task(const TreeParams& p, int b, int kvh, int rt, int w, int r, int part, const TreePieces& pc) {
  constexpr int kBatch = 8 / kQuads;
  float m = -INFINITY, l = 0.f, a[4 * kQuads];
#pragma unroll
  for (int e = 0; e < 4 * kQuads; ++e) a[e] = 0.f;
#pragma unroll 1
  for (int c = pc.c0; c <= pc.c1; c += kBatch) {
    float2 ml[kBatch];
    float4 o[kBatch][kQuads];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const unsigned slot = pc.slot(min(c + u, pc.c1), w);
      ml[u] = p.part_ml[slot * 128 + r];
      const float4* at = p.part_o + ((size_t)slot * (kD / 4) + kQuads * part) * 128 + r;
#pragma unroll
      for (int k = 0; k < kQuads; ++k) o[u][k] = at[128 * k];
    }
    float mx = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) mx = fmaxf(mx, ml[u].x);
    const float ref = mx == -INFINITY ? 0.f : mx, corr = exp2f(m - ref);
    m = mx;
    l *= corr;
#pragma unroll
    for (int e = 0; e < 4 * kQuads; ++e) a[e] *= corr;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float f = c + u <= pc.c1 ? exp2f(ml[u].x - ref) : 0.f;
      l += ml[u].y * f;
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        a[4 * k] += o[u][k].x * f;
        a[4 * k + 1] += o[u][k].y * f;
        a[4 * k + 2] += o[u][k].z * f;
        a[4 * k + 3] += o[u][k].w * f;
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int d = rt * p.tok + r / p.R, h = kvh * p.R + r % p.R;
  uint32_t u[2 * kQuads];
#pragma unroll
  for (int e = 0; e < 2 * kQuads; ++e) {
    const bf162 x = __floats2bfloat162_rn(a[2 * e] * inv, a[2 * e + 1] * inv);
    u[e] = *reinterpret_cast<const uint32_t*>(&x);
  }
  bf16* out = p.out + ((size_t(b) * p.n + d) * p.QH + h) * kD + part * 4 * kQuads;
  if constexpr (kQuads == 2) *reinterpret_cast<uint4*>(out) = make_uint4(u[0], u[1], u[2], u[3]);
  else *reinterpret_cast<uint2*>(out) = make_uint2(u[0], u[1]);
}

template <int kD, int kMod, bool kPair>
__global__ void __launch_bounds__(TA_THREADS, 1)
tree_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const TreeParams p) {
  using L = TA<kD, kPair>;
  constexpr int kStK = L::kStK, kStV = L::kStV;
  constexpr uint32_t kTile = L::kTile;
  extern __shared__ uint8_t ta_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ta_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* k_empty = k_full + kStK;
  uint64_t* v_full = k_empty + kStK;
  uint64_t* v_empty = v_full + kStV;
  uint64_t* q_full = v_empty + kStV;     // Q of a stretch has arrived
  uint64_t* q_empty = q_full + 1;        // every score product of a stretch has read it
  uint64_t* s_full = q_empty + 1;        // [w]: scores of warpgroup w's next tile are in tensor memory
  uint64_t* p_half = s_full + 2;         // [w]: it has written P of the first 64 keys (128 arrivals)
  uint64_t* p_full = p_half + 2;         // [w]: of all (128)
  uint64_t* pv_done = p_full + 2;        // [w]: O_w includes the tile
  uint64_t* o_free = pv_done + 2;        // [w]: O_w of a stretch has been read (128)
  uint64_t* ml_full = o_free + 2;        // the second warpgroup's maxima and sums of a stretch are in shared memory (128)
  uint64_t* ml_empty = ml_full + 1;      // the first has read them (128)
  uint64_t* part_out = ml_empty + 1;     // a piece's sums are in the workspace (128)
  uint64_t* last_known = part_out + 1;   // whether it was the last of its rows' pieces
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(last_known + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // [0] tiles of this CTA, [1] sequence, [2] place in it, [3] the list's
  long long* walk_at = reinterpret_cast<long long*>(tmem_slot + 2);
  volatile int* is_last = reinterpret_cast<volatile int*>(walk_at + 4);
  float2* s_ml = reinterpret_cast<float2*>(smem + L::kMl);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStK; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < kStV; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&p_half[w], 128);
      mbar_init(&p_full[w], 128);
      mbar_init(&pv_done[w], 1);
      mbar_init(&o_free[w], 128);
    }
    mbar_init(ml_full, 128);
    mbar_init(ml_empty, 128);
    mbar_init(part_out, 128);
    mbar_init(last_known, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  pdl_wait();
  if (warp == 0) {
    const long long total = tree_total(p, lane), G = tree_pieces_of(p, total);
    long long at, end, b_first;
    if ((total + 1) * (G + 1) < 0x100000000ll) {
      at = unsigned(blockIdx.x) * unsigned(total) / unsigned(G);
      end = (unsigned(blockIdx.x) + 1) * unsigned(total) / unsigned(G);
    } else {
      at = blockIdx.x * total / G;
      end = (blockIdx.x + 1) * total / G;
    }
    if (blockIdx.x >= G) at = end = 0;
    const int b_at = tree_find(p, at, lane, b_first);
    if (lane == 0) {
      walk_at[0] = end - at;
      walk_at[1] = b_at;
      walk_at[2] = at - b_first;
      walk_at[3] = total;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();                         // behind the allocation: a CTA of the next kernel must not take columns that this one waits for
  const uint32_t tmem_base = *tmem_slot;
  TreeWalk walk;
  walk.left = walk_at[0];
  walk.b = int(walk_at[1]);
  {
    const int nt = walk.left > 0 ? tree_tiles(tree_len(p, walk.b)) : 1;
    walk.idx = int(walk_at[2] / nt);
    walk.tile = int(walk_at[2] % nt);
  }
  TreeSeg s;

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    setmaxnreg_dec<TA_REGS_FEW>();
    if (lane == 0) {
      int g = 0, seg = 0;
      bool ok = true;
      while (ok && walk.next(p, s)) {
        if (seg > 0 && !mbar_wait(q_empty, (seg - 1) & 1, abort_flag)) break;
        ++seg;
        // (rows past the box: whatever, their results go nowhere)
        mbar_expect_tx(q_full, uint32_t((s.pair ? 4 : 2) * p.R * p.tok) * kD * 2);
        for (int i = 0; i < (s.pair ? 4 : 2); ++i) {                     // row tile i / 2, part i % 2
          const int d0 = (2 * s.rg + (i >> 1)) * p.tok, b = s.b + (i & 1) * p.B;
          uint8_t* sQ = smem + L::kQ + i * kTile;
          tma_load_4d(sQ, &tmQ, q_full, 0, s.kvh * p.R, d0, b);
          if (kD == 128) tma_load_4d(sQ + 16384, &tmQ, q_full, 64, s.kvh * p.R, d0, b);
        }
        for (int t = s.t0; t < s.t1; ++t, ++g) {
          const int row = t == s.nt - 1 ? s.len : t * 128;               // the drafts stand behind the cached keys
          if (!mbar_wait(&k_empty[g % kStK], ((g / kStK) & 1) ^ 1, abort_flag)) { ok = false; break; }
          uint8_t* sK = smem + L::kK + (g % kStK) * kTile;
          mbar_expect_tx(&k_full[g % kStK], kTile);
          tma_load_4d(sK, &tmK, &k_full[g % kStK], 0, s.kvh, row, s.b);
          if (kD == 128) tma_load_4d(sK + 16384, &tmK, &k_full[g % kStK], 64, s.kvh, row, s.b);
          if (!mbar_wait(&v_empty[g % kStV], ((g / kStV) & 1) ^ 1, abort_flag)) { ok = false; break; }
          uint8_t* sV = smem + L::kV + (g % kStV) * kTile;
          mbar_expect_tx(&v_full[g % kStV], kTile);
          tma_load_4d(sV, &tmV, &v_full[g % kStV], 0, s.kvh, row, s.b);
          if (kD == 128) tma_load_4d(sV + 16384, &tmV, &v_full[g % kStV], 64, s.kvh, row, s.b);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    setmaxnreg_dec<TA_REGS_FEW>();
    // Item u of a stretch is warpgroup u & 1's: with two row tiles both items of a key tile, else every key tile one item. The scores
    // of item u + 2 go out behind P V of item u, whose P they overwrite.
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, 128, 0, 0), idesc_s64 = umma_idesc_bf16(128, 64, 0, 0);
    constexpr uint32_t idesc_pv = umma_idesc_bf16(128, kD, 0, 1);
    int g0 = 0, seg = 0, done0 = 0, done1 = 0;           // tiles before the stretch; items that each warpgroup has had
    bool ok = true;
    while (ok && walk.next(p, s)) {
      const int sh = s.pair ? 1 : 0, items = (s.t1 - s.t0) << sh;
      auto scores = [&](int u) {
        const int t = u >> sh, g = g0 + t, w = u & 1;
        if ((!s.pair || w == 0) && !mbar_wait_warp(&k_full[g % kStK], (g / kStK) & 1, abort_flag)) return false;
        tc_fence_after();
        const uint64_t dQ = umma_smem_desc(smem_u32(smem + L::kQ + (s.pair ? 2 * w : 0) * kTile), 16, 1024);
        const uint64_t dK = umma_smem_desc(smem_u32(smem + L::kK + (g % kStK) * kTile), 16, 1024);
        const bool drafts = s.t0 + t == s.nt - 1;        // 64 keys are enough for them
        // Q's two parts, so that the scores are those of an unrounded rotation. Rounded to bf16 it was the largest error of the result:
        // 4.4e-3 of it at 60001 keys, 2.2e-3 like this, of which the result's own rounding is 1.7e-3. It costs 0 to 8 % of the whole call's
        // time at up to 3200 keys, 15 % at 60001 (67 -> 77 us, the header's last figure).
#pragma unroll
        for (int kk = 0; kk < kD / 8; ++kk) {
          const int k = kk % (kD / 16);
          const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
          umma_bf16_ss_warp(tmem_base + L::kColS + w * 128, dQ + (kk / (kD / 16)) * (kTile >> 4) + off, dK + off,
                            drafts ? idesc_s64 : idesc_s, kk != 0);
        }
        umma_commit_warp(&s_full[w]);
        if (!s.pair || w == 1) umma_commit_warp(&k_empty[g % kStK]);
        if (u + 1 == items) umma_commit_warp(q_empty);
        return true;
      };
      ok = mbar_wait_warp(q_full, seg & 1, abort_flag) && scores(0) && (items < 2 || scores(1));
      for (int u = 0; u < items && ok; ++u) {
        const int t = u >> sh, g = g0 + t, w = u & 1;
        const bool drafts = s.t0 + t == s.nt - 1;
        const uint32_t ph = (w == 0 ? done0 : done1) & 1;
        const uint64_t dV = umma_smem_desc(smem_u32(smem + L::kV + (g % kStV) * kTile), 16384, 1024);
        const uint32_t tO = tmem_base + L::kColO + w * 128, tP = tmem_base + L::kColS + w * 128;
        if (u < 2 && seg > 0) ok = mbar_wait_warp(&o_free[w], (seg - 1) & 1, abort_flag);
        ok = ok && mbar_wait_warp(&p_half[w], ph, abort_flag);
        if (ok && (!s.pair || w == 0)) ok = mbar_wait_warp(&v_full[g % kStV], (g / kStV) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) umma_bf16_ts_warp(tO, tP + kk * 8, dV + kk * 128, idesc_pv, u >= 2 || kk != 0);
        ok = mbar_wait_warp(&p_full[w], ph, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (!drafts) {
#pragma unroll
          for (int kk = 4; kk < 8; ++kk) umma_bf16_ts_warp(tO, tP + kk * 8, dV + kk * 128, idesc_pv, 1);
        }
        umma_commit_warp(&pv_done[w]);
        if (!s.pair || w == 1) umma_commit_warp(&v_empty[g % kStV]);
        if (w == 0) ++done0;
        else ++done1;
        if (u + 2 < items) ok = scores(u + 2);
      }
      g0 += s.t1 - s.t0;
      ++seg;
    }
  } else if (warp < 4) {
    setmaxnreg_dec<TA_REGS_FEW>();
  } else {
    // ---------------------------------------------------------------- softmax: a row per thread
    setmaxnreg_inc<TA_REGS_MANY>();
    // the quarter of tensor memory that a warp reaches is its number mod 4
    const int w = (warp - 4) >> 2, q = warp & 3, r = q * 32 + lane;
    const uint32_t lane_sel = uint32_t(q * 32) << 16;
    const uint32_t tS = tmem_base + lane_sel + L::kColS + w * 128, tO = tmem_base + lane_sel + L::kColO + w * 128;
    const float sl2 = kMod == kTreePlain ? p.scale * kTaLog2e : 1.f;
    // tiles before the stretch; items so far; sums handed from the second warpgroup; pieces
    int g0 = 0, seg = 0, done = 0, swaps = 0, parts = 0;
    bool ok = true;
    while (ok && walk.next(p, s)) {
      const int rt = 2 * s.rg + (s.pair ? w : 0);
      const int live = min(p.n - rt * p.tok, p.tok) * p.R;
      const bool work = q * 32 < live;                   // this warp has rows at all
      const int d = min(rt * p.tok + r / p.R, p.n - 1), h = s.kvh * p.R + r % p.R;
      const unsigned long long bits = tree_bits(p, s.b, d);
      const float slope2 = kMod == kTreeBias ? p.slopes[h] * kTaLog2e : 0.f, depth = float(tree_depth(bits));
      float m_ref = -INFINITY, l_run = 0.f;
      const int step = s.pair ? 1 : 2, first = s.t0 + (s.pair ? 0 : w);
      for (int t = first; t < s.t1 && ok; t += step, ++done) {
        if (!mbar_wait(&s_full[w], done & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const bool drafts = t == s.nt - 1;
        // keys of the tile: of the drafts those that the cache has room for (rows behind its end arrive as zeros, and would count)
        const int rem = drafts ? min(p.n, p.Tmax - s.len) : min(s.len - t * 128, 128);
        if (rem < (drafts ? 64 : 128) && (w == 0 || !s.pair)) {
          // values past the length may be anything, and 0 times that (two row tiles: P V of the first one comes first)
          const int g = g0 + t - s.t0, st = g % kStV;
          if (!__all_sync(0xffffffffu, mbar_wait(&v_full[st], (g / kStV) & 1, abort_flag))) { ok = false; break; }
          for (int i = r; i < ((drafts ? 64 : 128) - rem) * (kD / 8); i += 128)
            *ta_chunk(smem + L::kV + st * kTile, rem + i / (kD / 8), i % (kD / 8)) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
        }
        if (!work) {                                     // rows that nobody asked for: their P may be anything
          mbar_arrive(&p_half[w]);
          mbar_arrive(&p_full[w]);
          continue;
        }
        uint32_t sc[128];
        tmem_ld_32x32b_x32(tS, *reinterpret_cast<uint32_t(*)[32]>(&sc[0]));
        tmem_ld_32x32b_x32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&sc[32]));
        tmem_ld_32x32b_x32(tS + 64, *reinterpret_cast<uint32_t(*)[32]>(&sc[64]));
        tmem_ld_32x32b_x32(tS + 96, *reinterpret_cast<uint32_t(*)[32]>(&sc[96]));
        tmem_ld_wait();
        bool cap_now = false;                            // the exponentials take the cap
        if constexpr (kMod == kTreeCap) {
          const int tier = cap_tier(sc, p.cap, r < live);
          cap_now = tier == kCapNear && rem >= 128;
          if (!cap_now) cap_scores(sc, p.cap, tier);
        }
        if (drafts) {
#pragma unroll
          for (int e = 0; e < 64; ++e) {
            if constexpr (kMod == kTreeBias) {
              const float dj = e < p.n ? float(tree_depth(tree_bits(p, s.b, e))) : 0.f;
              sc[e] = __float_as_uint(fmaf(__uint_as_float(sc[e]), p.scale * kTaLog2e, -slope2 * fabsf(depth - dj)));
            }
            if (!((bits >> e) & 1) || e >= rem) sc[e] = 0xff800000u;
          }
#pragma unroll
          for (int e = 64; e < 128; ++e) sc[e] = 0xff800000u;
        } else {
          if constexpr (kMod == kTreeBias) {
            const float dist = float(s.len - t * 128) + depth;
#pragma unroll
            for (int e = 0; e < 128; ++e)
              sc[e] = __float_as_uint(fmaf(__uint_as_float(sc[e]), p.scale * kTaLog2e, -slope2 * (dist - float(e))));
          }
          if (rem < 128) {
#pragma unroll
            for (int e = 0; e < 128; ++e)
              if (e >= rem) sc[e] = 0xff800000u;
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 128; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], __uint_as_float(sc[e]));
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sl2;
        if (kMod == kTreeCap && cap_now) mx = cap_any(mx, p.cap);      // the cap keeps the order of the scores
        // the reference maximum moves when a tile exceeds it by more than 2^8, as in the attention forward
        const bool need = r < live && mx > m_ref + kTaRescaleStep;
        if (t == first) {
          m_ref = mx;
        } else if (__any_sync(0xffffffffu, need)) {
          if (!__all_sync(0xffffffffu, mbar_wait(&pv_done[w], (done - 1) & 1, abort_flag))) { ok = false; break; }
          tc_fence_after();
          const float corr = need ? exp2f(m_ref - mx) : 1.f;
          l_run *= corr;
#pragma unroll 1
          for (int c = 0; c < kD / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(tO + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = corr == 0.f ? 0u : __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st_32x32b_x16(tO + c * 16, o);
          }
          tmem_st_wait();
          if (need) m_ref = mx;
        }
        const float m_sub = m_ref == -INFINITY ? 0.f : m_ref;
        float rs0 = 0.f, rs1 = 0.f;
        auto half = [&](auto lo_tag) {                   // P of 64 keys, handed over as soon as it is there
          constexpr int kLo = decltype(lo_tag)::value;
          if (kMod == kTreeCap && cap_now) {
            cap_row_p<kLo, kLo + 64>(sc, p.cap, m_sub, rs0, rs1);
          } else {
#pragma unroll
            for (int e = kLo; e < kLo + 64; e += 2) {
              const float p0 = exp2f(fmaf(__uint_as_float(sc[e]), sl2, -m_sub)), p1 = exp2f(fmaf(__uint_as_float(sc[e + 1]), sl2, -m_sub));
              rs0 += p0;
              rs1 += p1;
              const bf162 x = __floats2bfloat162_rn(p0, p1);
              sc[e >> 1] = *reinterpret_cast<const uint32_t*>(&x);
            }
          }
          tmem_st_32x32b_x16(tS + kLo / 2, *reinterpret_cast<const uint32_t(*)[16]>(&sc[kLo / 2]));
          tmem_st_32x32b_x16(tS + kLo / 2 + 16, *reinterpret_cast<const uint32_t(*)[16]>(&sc[kLo / 2 + 16]));
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(kLo == 0 ? &p_half[w] : &p_full[w]);
        };
        half(std::integral_constant<int, 0>{});
        if (drafts) mbar_arrive(&p_full[w]);             // nothing behind the first 64
        else half(std::integral_constant<int, 64>{});
        l_run += rs0 + rs1;
      }
      if (!ok) break;
      // The stretch's end: with one row tile the second warpgroup hands its maximum and sum to the first, which reads both outputs.
      const bool any = first < s.t1, other = !s.pair && s.t1 - s.t0 > 1;
      if (any && !__all_sync(0xffffffffu, mbar_wait(&pv_done[w], (done - 1) & 1, abort_flag))) { ok = false; break; }
      tc_fence_after();
      g0 += s.t1 - s.t0;
      const int seg_now = seg++;
      if (!s.pair && w == 1) {
        if (other) {
          if (swaps > 0 && !__all_sync(0xffffffffu, mbar_wait(ml_empty, (swaps - 1) & 1, abort_flag))) { ok = false; break; }
          s_ml[r] = make_float2(m_ref, l_run);
          tc_fence_before();
          mbar_arrive(ml_full);
          ++swaps;
        }
        continue;
      }
      float f0 = 1.f, f1 = 0.f;                          // what the two outputs are multiplied with
      if (other) {
        if (!__all_sync(0xffffffffu, mbar_wait(ml_full, swaps & 1, abort_flag))) { ok = false; break; }
        tc_fence_after();
        const float2 ml = s_ml[r];
        mbar_arrive(ml_empty);
        ++swaps;
        const float m = fmaxf(m_ref, ml.x), m_sub = m == -INFINITY ? 0.f : m;
        f0 = exp2f(m_ref - m_sub);
        f1 = exp2f(ml.x - m_sub);
        l_run = l_run * f0 + ml.y * f1;
        m_ref = m;
      }
      const bool whole = s.t0 == 0 && s.t1 == s.nt;
      if (work) {
        const bool alive = r < live;
        const size_t slot = size_t((2 * int(blockIdx.x) + (seg_now == 0 ? 0 : 1)) * 2 + (s.pair ? w : 0));
        const float inv = whole ? (l_run == 0.f ? 0.f : 1.f / l_run) : 1.f;
        f0 = f0 == 0.f ? 0.f : f0 * inv;
        f1 *= inv;
        bf16* orow = p.out + ((size_t(s.b) * p.n + d) * p.QH + h) * kD;
        if (alive && !whole) p.part_ml[slot * 128 + r] = make_float2(m_ref, l_run);
#pragma unroll 1
        for (int c = 0; c < kD / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tO + c * 32, o);
          if (other) {
            uint32_t o1[32];
            tmem_ld_32x32b_x32(tO + 128 + c * 32, o1);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) {               // (what weighs nothing may be anything)
              const float x0 = f0 == 0.f ? 0.f : __uint_as_float(o[e]) * f0;
              o[e] = __float_as_uint(f1 == 0.f ? x0 : fmaf(__uint_as_float(o1[e]), f1, x0));
            }
          } else {
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = l_run == 0.f ? 0u : __float_as_uint(__uint_as_float(o[e]) * f0);
          }
          if (!alive) continue;
          if (whole) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint4 u;
              bf162* u2 = reinterpret_cast<bf162*>(&u);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                u2[e] = __floats2bfloat162_rn(__uint_as_float(o[8 * k + 2 * e]), __uint_as_float(o[8 * k + 2 * e + 1]));
              reinterpret_cast<uint4*>(orow + c * 32)[k] = u;
            }
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              reinterpret_cast<uint4*>(p.part_o)[(slot * (kD / 4) + c * 8 + k) * 128 + r] =
                  make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&o_free[w]);
      if (!s.pair) mbar_arrive(&o_free[1]);
      if (p.arrived != nullptr && !whole) {              // few rows: whoever comes last joins them
        const int combo = (s.b * p.KVH + s.kvh) * p.groups + s.rg;
        const TreePieces pc = tree_pieces(p, walk_at[3], combo_first(p, s), s.nt);
        __threadfence();
        mbar_arrive(part_out);
        if (r == 0 && mbar_wait(part_out, parts & 1, abort_flag)) {
          *is_last = atomicAdd(&p.arrived[combo], 1) == pc.c1 - pc.c0;
          mbar_arrive(last_known);
        }
        if (!__all_sync(0xffffffffu, mbar_wait(last_known, parts & 1, abort_flag))) { ok = false; break; }
        ++parts;
        if (*is_last != 0) {
          __threadfence();
          for (int i = r; i < live * (kD / 4); i += 128) tree_join_task<kD, 1>(p, s.b, s.kvh, 2 * s.rg, 0, i % live, i / live, pc);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  if (threadIdx.x == 0 && *abort_flag != 0 && p.status != nullptr) {
    if (atomicCAS(p.status, 0, int(*abort_flag)) == 0) p.status[1] = 351;
  }
}

// Joins the pieces of every (sequence, KV head, row group) that was cut: grid (those, rows * D / (4 kQuads) / 256).
template <int kD, int kQuads>
__global__ void __launch_bounds__(256)
tree_join_kernel(const TreeParams p) {
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const int per = p.KVH * p.groups, b = blockIdx.x / per, idx = blockIdx.x % per, kvh = idx / p.groups, rg = idx % p.groups;
  unsigned long long sum = 0, before = 0;
  int nt = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int v = b0 + lane < p.B ? tree_tiles(tree_len(p, b0 + lane)) : 0;
    sum += __reduce_add_sync(0xffffffffu, v);
    before += __reduce_add_sync(0xffffffffu, b0 + lane < b ? v : 0);
    if (b >= b0 && b < b0 + 32) nt = __shfl_sync(0xffffffffu, v, b - b0);
  }
  const TreePieces pc = tree_pieces(p, sum * per, before * per + (unsigned long long)idx * nt, nt);
  if (pc.c0 == pc.c1) return;
  const int rows = p.tok * p.R, all = p.n > p.tok ? 2 * rows : rows;
  const int task = blockIdx.y * 256 + threadIdx.x, row = task % all, part = task / all;
  const int w = row >= rows ? 1 : 0, r = row - w * rows, rt = 2 * rg + w;
  if (part < kD / (4 * kQuads) && r < min(p.n - rt * p.tok, p.tok) * p.R) tree_join_task<kD, kQuads>(p, b, kvh, rt, w, r, part, pc);
}

template <int kD, int kMod, bool kPair>
static int launch_tree_attn(const TreeParams& p, const TensorMap& tq, const TensorMap& tk, const TensorMap& tv, cudaStream_t st) {
  using L = TA<kD, kPair>;
  static bool configured = false;
  if (!configured) {
    B200_CHECK(cudaFuncSetAttribute(tree_attn_kernel<kD, kMod, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem));
    configured = true;
  }
  return static_cast<int>(launch_pdl(tree_attn_kernel<kD, kMod, kPair>, dim3(p.ctas), dim3(TA_THREADS), L::kSmem, st, 0, *tq, *tk, *tv, p));
}

template <int kD, int kMod>
static int launch_tree(const TreeParams& p, const TensorMap& tq, const TensorMap& tk, const TensorMap& tv, cudaStream_t st) {
  const long long chunks = (long long)p.B * p.n * (p.QH + 2 * p.KVH) * (kD / 8);
  B200_CHECK(launch_pdl(tree_append_kernel<kD>, dim3(unsigned((chunks + 255) / 256)), dim3(256), 0, st, 0, p));
  const int rc = p.n > p.tok ? launch_tree_attn<kD, kMod, true>(p, tq, tk, tv, st) : launch_tree_attn<kD, kMod, false>(p, tq, tk, tv, st);
  if (rc != 0) return rc;
  if (p.arrived != nullptr) return 0;
  // Eight columns to a thread where there are threads enough (the call at 8 x 3000 keys, 24 drafts, 32 / 8 heads of 128: 47.0 us with four,
  // 44.0 like this), four and more pieces at a time else (1 x 60001 keys, 32 drafts: 77.1, 77.5 with eight).
  const int combos = p.B * p.KVH * p.groups, rows = (p.n > p.tok ? 2 : 1) * p.tok * p.R;
  if ((long long)combos * rows * (kD / 8) >= 256LL * num_sms())
    return static_cast<int>(launch_pdl(tree_join_kernel<kD, 2>, dim3(combos, (rows * (kD / 8) + 255) / 256), dim3(256), 0, st, 0, p));
  return static_cast<int>(launch_pdl(tree_join_kernel<kD, 1>, dim3(combos, (rows * (kD / 4) + 255) / 256), dim3(256), 0, st, 0, p));
}

// Groups of two tiles of 128 / R drafts.
static int tree_groups(int n, int R) { return (n + 2 * (128 / R) - 1) / (2 * (128 / R)); }

// Pieces that the list of tiles is cut into: one for every SM, or every tile if there are fewer of full caches.
static int tree_ctas(int B, int n, int QH, int KVH, int Tmax) {
  const long long tiles = (long long)B * KVH * tree_groups(n, QH / KVH) * ((Tmax + 127) / 128 + 1);
  return int(tiles < num_sms() ? tiles : num_sms());
}

static bool tree_shape_ok(int B, int n, int QH, int KVH, int Tmax, int D) {
  return B >= 0 && n >= 1 && n <= TA_MAX_DRAFTS && (D == 64 || D == 128) && KVH > 0 && QH > 0 && QH % KVH == 0 && QH / KVH <= 128 &&
         Tmax > 0 && (long long)B * KVH * tree_groups(n, QH / KVH) <= 0x7fffffffLL;
}

}  // namespace b200

using namespace b200;

// Bytes of the workspace that b200_tree_attn_append wants (16-byte aligned); 0: sizes that it does not take.
B200_API long long b200_tree_attn_workspace(int B, int n, int QH, int KVH, int Tmax, int D) {
  if (!tree_shape_ok(B, n, QH, KVH, Tmax, D)) return 0;
  return 4LL * tree_ctas(B, n, QH, KVH, Tmax) * 128 * (D * 4 + 8) + 4LL * B * n * QH * D + 4LL * B * KVH * tree_groups(n, QH / KVH);
}

// kqv [B * n][ld] (K | Q | V, un-rotated), caches [B, KVH, Tmax, D], out [B, n, QH, D], lens [B], tree [B, n] (64 bits each), rotary
// tables [table_rows, D / 2]. cap > 0: scores c tanh(s / c); slopes [QH]: scores minus slope times distance (not both).
B200_API int b200_tree_attn_append(const void* kqv, void* kc, void* vc, void* out, const void* lens, const void* tree, const void* cosr,
                                   const void* sinr, const void* slopes, void* workspace, int B, int n, int QH, int KVH, int Tmax, int D,
                                   int table_rows, long long ld, float scale, float cap, cudaStream_t st) {
  if (!tree_shape_ok(B, n, QH, KVH, Tmax, D)) return static_cast<int>(cudaErrorInvalidValue);
  if (B == 0) return 0;
  if (cap < 0.f || (cap > 0.f && slopes != nullptr) || table_rows < 1 || ld % 8 != 0) return static_cast<int>(cudaErrorInvalidValue);
  for (const void* x : {kqv, (const void*)kc, (const void*)vc, (const void*)out, cosr, sinr, (const void*)workspace})
    if (x == nullptr || (reinterpret_cast<uintptr_t>(x) & 15) != 0) return static_cast<int>(cudaErrorInvalidValue);
  const unsigned long long hs = (unsigned long long)Tmax * D;
  const TensorMap tk = get_tensor_map_bthd(kc, B, Tmax, KVH, D, KVH * hs, D, hs, 128, 64);
  const TensorMap tv = get_tensor_map_bthd(vc, B, Tmax, KVH, D, KVH * hs, D, hs, 128, 64);
  TreeParams p;
  p.kqv = static_cast<const bf16*>(kqv);
  p.kc = static_cast<bf16*>(kc);
  p.vc = static_cast<bf16*>(vc);
  p.out = static_cast<bf16*>(out);
  p.lens = static_cast<const int*>(lens);
  p.tree = static_cast<const unsigned long long*>(tree);
  p.cosr = static_cast<const float*>(cosr);
  p.sinr = static_cast<const float*>(sinr);
  p.slopes = static_cast<const float*>(slopes);
  p.B = B; p.n = n; p.QH = QH; p.KVH = KVH; p.Tmax = Tmax; p.table_rows = table_rows; p.ld = ld;
  p.R = QH / KVH;
  p.tok = std::min(n, 128 / p.R);
  p.groups = tree_groups(n, p.R);
  p.ctas = tree_ctas(B, n, QH, KVH, Tmax);
  p.part_o = static_cast<float4*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + 4LL * p.ctas * 128 * (D / 4));
  p.q = reinterpret_cast<bf16*>(p.part_ml + 4LL * p.ctas * 128);
  // Few rows times few pieces: the CTA that finishes a (sequence, KV head) last joins its pieces (one token over 1801 keys, 16 / 4 heads of
  // 128: 15.6 us, 18.0 with a kernel of its own); more of them would keep that one SM busy for longer.
  const long long combos = (long long)B * KVH * p.groups;
  p.arrived = n * p.R <= 8 && (p.ctas / combos + 2) * n * p.R <= 512
                  ? reinterpret_cast<int*>(p.q + 2 * (size_t)B * n * QH * D) : nullptr;
  p.scale = scale;
  p.cap = make_score_cap(scale, cap);
  p.status = status_ptr();
  const unsigned long long qs = (unsigned long long)QH * D;
  const TensorMap tq = get_tensor_map_bthd(p.q, 2 * B, n, QH, D, n * qs, qs, D, p.tok, 64, p.R);
  if (!tq || !tk || !tv) return static_cast<int>(cudaErrorInvalidValue);
  if (D == 128) {
    if (cap > 0.f) return launch_tree<128, kTreeCap>(p, tq, tk, tv, st);
    return slopes != nullptr ? launch_tree<128, kTreeBias>(p, tq, tk, tv, st) : launch_tree<128, kTreePlain>(p, tq, tk, tv, st);
  }
  if (cap > 0.f) return launch_tree<64, kTreeCap>(p, tq, tk, tv, st);
  return slopes != nullptr ? launch_tree<64, kTreeBias>(p, tq, tk, tv, st) : launch_tree<64, kTreePlain>(p, tq, tk, tv, st);
}
