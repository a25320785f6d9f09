// Which keys each query of a batch sees, and which tiles of 128 queries and 128 keys meet.
//
// Query t of row b sees the keys [lo, hi): lo is the first position of its document, hi the position behind it, or the end
// of the document's leading prefix run if it is part of that; padding (a negative document) sees nothing. The attention
// kernels read, per query tile, the key tiles it meets and whether a key tile is seen whole by all its rows, and per key
// tile the query tiles that meet it.
//
// One CTA per row: lo is a running maximum over the starts of documents, the end of a prefix run a running minimum from
// behind. A warp holds 128 consecutive tokens, four to a lane, which are one tile of the tables. A step of a training
// run makes one mask for all its layers.
#include <climits>

#include "common.cuh"

namespace b200 {

constexpr int SM_THREADS = 1024;                      // at most: as many as there are tokens for
constexpr int SM_PER = 4;                             // tokens of a thread
constexpr int SM_MAX_TILES = 4000;                    // ranges and counts kept in shared memory: 47 KiB, 512000 tokens

struct SpanMaskParams {
  const int* docs;              // [B, T] or null: one document
  const unsigned char* prefix;  // [B, T] or null
  const int* valid_len;         // [B] or null
  const int* lo_in;             // [B, T]: spans as they are given, in place of all of the above
  const int* hi_in;
  int2* spans;                  // [B, T]
  int4* qtab;                   // [B, nt]: first key tile, end; largest lo, smallest hi of its rows
  int2* ktab;                   // [B, nt]: first query tile, end
  int* order;                   // [B, nt] query tiles, [B, (nt + 1) / 2] pairs of them, [B, nt] key tiles: those with most to do first
  int B, T, nt;
  int* status;
};

struct MaxOp {
  static constexpr int kNone = -1;
  __device__ static int of(int a, int b) { return max(a, b); }
  __device__ static int warp(int v) { return __reduce_max_sync(0xffffffffu, v); }
};
struct MinOp {
  static constexpr int kNone = INT_MAX;
  __device__ static int of(int a, int b) { return min(a, b); }
  __device__ static int warp(int v) { return __reduce_min_sync(0xffffffffu, v); }
};

// v over the threads before this one (kUp) or behind it, the carry first; `carry` leaves with the whole block in it.
template <class Op, bool kUp>
__device__ __forceinline__ int block_scan_excl(int v, int& carry, int* warp_v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = kUp ? __shfl_up_sync(0xffffffffu, x, o) : __shfl_down_sync(0xffffffffu, x, o);
    if (kUp ? lane >= o : lane + o < 32) x = Op::of(x, y);
  }
  int e = kUp ? __shfl_up_sync(0xffffffffu, x, 1) : __shfl_down_sync(0xffffffffu, x, 1);
  if (lane == (kUp ? 0 : 31)) e = Op::kNone;
  __syncthreads();                                    // the last scan's values have been read
  if (lane == (kUp ? 31 : 0)) warp_v[warp] = x;
  __syncthreads();
  const int y = lane < warps ? warp_v[lane] : Op::kNone;
  const int before = Op::warp((kUp ? lane < warp : lane > warp) ? y : Op::kNone);
  const int all = Op::warp(y), out = Op::of(Op::of(carry, before), e);
  carry = Op::of(carry, all);
  return out;
}

// Four tokens' values from `at` on: one load where the row allows it.
__device__ __forceinline__ void load4(const int* p, int at, int T, bool wide, int none, int (&v)[SM_PER]) {
  if (wide && at + 3 < T) {
    const int4 x = *reinterpret_cast<const int4*>(p + at);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < SM_PER; ++i) v[i] = at + i < T ? p[at + i] : none;
}
__device__ __forceinline__ void load4(const unsigned char* p, int at, int T, bool wide, int none, int (&v)[SM_PER]) {
  if (wide && at + 3 < T) {
    const uchar4 x = *reinterpret_cast<const uchar4*>(p + at);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < SM_PER; ++i) v[i] = at + i < T ? p[at + i] : none;
}

__device__ __forceinline__ int warp_min(int v) { return __reduce_min_sync(0xffffffffu, v); }
__device__ __forceinline__ int warp_max(int v) { return __reduce_max_sync(0xffffffffu, v); }

__global__ void __launch_bounds__(SM_THREADS)
span_mask_kernel(const SpanMaskParams p) {
  extern __shared__ int2 s_range[];                   // [nt]: key tiles of each query tile
  int* s_count = reinterpret_cast<int*>(s_range + p.nt);      // [nt]: query tiles of each key tile
  __shared__ int warp_v[SM_THREADS / 32];
  const int b = blockIdx.x, T = p.T;
  const size_t row0 = size_t(b) * T;
  pdl_wait();
  pdl_trigger();
  const int vlen = p.valid_len ? checked_index(p.valid_len[b], T, p.status, 340) : T;
  int2* spans = p.spans + row0;
  const int* docs = p.docs ? p.docs + row0 : nullptr;
  const unsigned char* pre = p.prefix ? p.prefix + row0 : nullptr;

  const int chunk = int(blockDim.x) * SM_PER;
  const bool wide_docs = (reinterpret_cast<uintptr_t>(docs) & 15) == 0, wide_pre = (reinterpret_cast<uintptr_t>(pre) & 3) == 0;
  // document, whether one starts here, and prefix flag of this thread's four tokens
  auto tokens = [&](int t0, int (&id)[SM_PER], bool (&start)[SM_PER], int (&flag)[SM_PER]) {
    int last = 0;
    if (docs != nullptr) {
      load4(docs, t0, T, wide_docs, 0, id);
      if (t0 > 0 && t0 < T) last = docs[t0 - 1];
    }
    if (pre != nullptr) load4(pre, t0, T, wide_pre, 0, flag);
#pragma unroll
    for (int i = 0; i < SM_PER; ++i) {
      if (docs == nullptr) id[i] = 0;
      if (pre == nullptr) flag[i] = 0;
      start[i] = t0 + i < T && (t0 + i == 0 || (docs != nullptr && id[i] != (i > 0 ? id[i - 1] : last)));
    }
  };

  // From behind: where the prefix run that a token may be part of ends (the first start or unflagged token behind it). Kept
  // in the spans' hi until the other pass has lo.
  if (pre != nullptr && p.lo_in == nullptr) {
    int carry = T;
    for (int c0 = (T - 1) / chunk * chunk; c0 >= 0; c0 -= chunk) {
      const int t0 = c0 + int(threadIdx.x) * SM_PER;
      int id[SM_PER], flag[SM_PER], stop[SM_PER], v = MinOp::kNone;
      bool start[SM_PER];
      tokens(t0, id, start, flag);
#pragma unroll
      for (int i = SM_PER - 1; i >= 0; --i) {
        stop[i] = v;                                  // the first stop of this thread behind it
        if (t0 + i < T && (flag[i] == 0 || start[i])) v = t0 + i;
      }
      const int behind = block_scan_excl<MinOp, false>(v, carry, warp_v);
#pragma unroll
      for (int i = 0; i < SM_PER; ++i)
        if (t0 + i < T) spans[t0 + i].y = min(stop[i], behind);
    }
    // (a thread reads back its own tokens' alone)
  }

  int carry_start = 0, carry_plain = -1;
  for (int c0 = 0; c0 < T; c0 += chunk) {
    const int t0 = c0 + int(threadIdx.x) * SM_PER;
    int lo[SM_PER], hi[SM_PER];
    if (p.lo_in != nullptr) {
#pragma unroll
      for (int i = 0; i < SM_PER; ++i) {
        lo[i] = t0 + i < T ? p.lo_in[row0 + t0 + i] : 0;
        hi[i] = t0 + i < T ? p.hi_in[row0 + t0 + i] : 0;
      }
    } else {
      int start_at[SM_PER], plain[SM_PER], id[SM_PER], flag[SM_PER], s = -1, u = -1;
      bool start[SM_PER];
      tokens(t0, id, start, flag);
#pragma unroll
      for (int i = 0; i < SM_PER; ++i) {
        const int t = t0 + i;
        if (start[i]) s = t;
        if (t < T && flag[i] == 0) u = t;
        start_at[i] = s;
        plain[i] = u;
      }
      const int s_before = block_scan_excl<MaxOp, true>(s, carry_start, warp_v);
      const int u_before = pre != nullptr ? block_scan_excl<MaxOp, true>(u, carry_plain, warp_v) : -1;
#pragma unroll
      for (int i = 0; i < SM_PER; ++i) {
        const int t = t0 + i;
        lo[i] = max(start_at[i], s_before);
        hi[i] = t + 1;
        if (pre != nullptr && t < T && max(plain[i], u_before) < lo[i]) hi[i] = spans[t].y;
        if (id[i] < 0 || t >= vlen) hi[i] = 0;
        hi[i] = min(hi[i], vlen);
      }
    }
    int lo_min = INT_MAX, lo_max = 0, hi_min = INT_MAX, hi_max = 0;
#pragma unroll
    for (int i = 0; i < SM_PER; ++i) {
      const int t = t0 + i;
      if (t >= T) continue;
      lo[i] = max(lo[i], 0);
      hi[i] = min(hi[i], T);
      const bool none = hi[i] <= lo[i];
      spans[t] = none ? make_int2(0, 0) : make_int2(lo[i], hi[i]);
      if (none) {
        lo_max = INT_MAX;                             // some row of the tile sees nothing: no key tile is seen by all
      } else {
        lo_min = min(lo_min, lo[i]);
        lo_max = max(lo_max, lo[i]);
        hi_min = min(hi_min, hi[i]);
        hi_max = max(hi_max, hi[i]);
      }
    }
    lo_min = warp_min(lo_min);
    lo_max = warp_max(lo_max);
    hi_min = warp_min(hi_min);
    hi_max = warp_max(hi_max);
    const int tile = t0 / 128;                        // the same for the warp
    if ((threadIdx.x & 31) == 0 && tile < p.nt) {
      const int2 r = hi_max > 0 ? make_int2(lo_min / 128, (hi_max + 127) / 128) : make_int2(0, 0);
      p.qtab[size_t(b) * p.nt + tile] = make_int4(r.x, r.y, lo_max, hi_min);
      s_range[tile] = r;
    }
  }
  __syncthreads();
  for (int n = threadIdx.x; n < p.nt; n += blockDim.x) {
    int first = INT_MAX, end = 0;
    for (int m = 0; m < p.nt; ++m) {
      const int2 r = s_range[m];
      if (n >= r.x && n < r.y) {
        first = min(first, m);
        end = m + 1;
      }
    }
    p.ktab[size_t(b) * p.nt + n] = end > 0 ? make_int2(first, end) : make_int2(0, 0);
    s_count[n] = end > 0 ? end - first : 0;
  }
  __syncthreads();
  // Places in the orders: how many have more to do (or as much, and a lower number).
  const int pairs = (p.nt + 1) / 2;
  int *order_q = p.order + size_t(b) * p.nt, *order_p = p.order + size_t(p.B) * p.nt + size_t(b) * pairs,
      *order_k = p.order + size_t(p.B) * (p.nt + pairs) + size_t(b) * p.nt;
  auto steps = [&](int u) {                           // of a pair: the walk that the two share
    const int2 x = s_range[2 * u], y = 2 * u + 1 < p.nt ? s_range[2 * u + 1] : make_int2(0, 0);
    return x.y == 0 ? y.y - y.x : y.y == 0 ? x.y - x.x : max(x.y, y.y) - min(x.x, y.x);
  };
  for (int n = threadIdx.x; n < p.nt; n += blockDim.x) {
    const int mine = s_range[n].y - s_range[n].x, count = s_count[n], both = n < pairs ? steps(n) : 0;
    int at_q = 0, at_k = 0, at_p = 0;
    for (int m = 0; m < p.nt; ++m) {
      const int other = s_range[m].y - s_range[m].x, c = s_count[m];
      at_q += other > mine || (other == mine && m < n);
      at_k += c > count || (c == count && m < n);
    }
    order_q[at_q] = n;
    order_k[at_k] = n;
    if (n < pairs) {
      for (int m = 0; m < pairs; ++m) {
        const int other = steps(m);
        at_p += other > both || (other == both && m < n);
      }
      order_p[at_p] = n;
    }
  }
}

}  // namespace b200

using namespace b200;

// Fills `spans` [B, T] (lo, hi), `qtab` [B, nt] (4 ints), `ktab` [B, nt] (2 ints) and `order` [B, nt], [B, (nt + 1) / 2], [B, nt] (query
// tiles, pairs of them, key tiles; most to do first), nt = tiles of 128 tokens, from documents,
// prefix flags and valid lengths (each may be null), or from the spans lo / hi [B, T].
B200_API int b200_span_mask(const void* docs, const void* prefix, const void* valid_len, const void* lo, const void* hi,
                            void* spans, void* qtab, void* ktab, void* order, int B, int T, cudaStream_t st) {
  if (B <= 0 || T <= 0) return 0;
  const int nt = (T + 127) / 128;
  if (nt > SM_MAX_TILES || (lo == nullptr) != (hi == nullptr)) return static_cast<int>(cudaErrorInvalidValue);
  SpanMaskParams p;
  p.docs = static_cast<const int*>(docs);
  p.prefix = static_cast<const unsigned char*>(prefix);
  p.valid_len = static_cast<const int*>(valid_len);
  p.lo_in = static_cast<const int*>(lo);
  p.hi_in = static_cast<const int*>(hi);
  p.spans = static_cast<int2*>(spans);
  p.qtab = static_cast<int4*>(qtab);
  p.ktab = static_cast<int2*>(ktab);
  p.order = static_cast<int*>(order);
  p.B = B; p.T = T; p.nt = nt;
  p.status = status_ptr();
  const int threads = nt * 32 < SM_THREADS ? nt * 32 : SM_THREADS;             // a warp to a tile
  return static_cast<int>(launch_pdl(span_mask_kernel, dim3(B), dim3(threads), size_t(nt) * (sizeof(int2) + sizeof(int)), st, 0, p));
}
