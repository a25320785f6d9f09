// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// A sequence has n nodes: node 0 is its last token, the others are drafts, each with a parent that stands before it. For node i, p is
// the softmax of its logits over the temperature, cut to its nucleus: the fewest tokens, taken by falling probability and rising index,
// whose mass reaches `top`. Without the drafts' probabilities a token is drawn from p, and the child that holds it is gone on to. With
// them (q, which the children of the node were drawn from, one after the other) children are tried in their order: child k, token x, is
// taken if accept u q(x) Z_k < r_k(x), where r_k = max(p - c_k q, 0), Z_k its sum, c_0 = 0, c_(k+1) = c_k + Z_k (each refusal leaves
// max(r_k / Z_k - q, 0), which is this up to a factor); if none is, the token comes from the last r_k.
//
// Every node is decided by itself, by a cluster of CTAs that share its row, the row in shared memory; a second kernel walks the trees.
// Weights are fp64, and sums are sums of integers (2^62 / columns to the largest weight): which token a number falls on depends on the
// whole row's sum, and integers add up to the same in any order.
//
// What bounds it: a row of 32000 logits is 128 KB, 3 us of an SM's share of HBM, and 32000 fp64 exponentials, which take 9; the chain of a
// node is longer: largest logit, weights, the bin, the tokens of the bin, the sums, the draw, each of them once over the CTA's slice and
// once through the cluster. A call with one node (no walk to speak of) takes 18 us with 4000 tokens to a CTA (a row in eight), 32 with
// 16000 (64 nodes in two CTAs each, one CTA an SM), 38 with two such CTAs an SM (148 nodes); without a nucleus 11 and, on full SMs, 23. So
// a row is cut into more CTAs while half of the SMs would be idle, and slices are else as large as two CTAs an SM hold, which is more
// nodes in a given time. Where there are more nodes than clusters, node 0 of all sequences comes first, then node 1: most of the later
// ones are out of question by then and passed over. Us, 6 nodes of one sequence (probabilities of the drafts, nucleus) / 8 x 24 (the same,
// no nucleus) / 16 x 63 (looked up, nucleus), 32000 tokens: bits of the nucleus' end one by one 267 / 122 / 1709, histogram 30 / 45 / 417,
// its search in two steps, weights remade and nodes passed over 20 to 25 / 54 to 63 / 72 to 104 (ten inputs, by how far their texts go;
// the second was faster with its weights kept in shared memory, which leaves an SM one row). (CTAs that read one another's whole
// histograms took 17000 cycles for it.)
#include <cooperative_groups.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "common.cuh"

namespace b200 {
namespace cg = cooperative_groups;

typedef unsigned long long u64;

constexpr int VD_THREADS = 512, VD_WARPS = VD_THREADS / 32, VD_SEG = 128, VD_MAX_SEGS = 376, VD_MAX_NODES = 64, VD_MAX_CLUSTER = 8;
constexpr int VD_BINS = 2048, VD_COARSE = VD_BINS / 32, VD_LIST = 512;      // bins of masses; tokens that are put in order one by one

struct VerifyParams {
  const void* logits;        // [B, n, V], fp32 or bf16
  const float* q;            // [B, n, V] or null
  const int* tokens;         // [B, n]
  const int* parents;
  const float* u;            // [B, n]: where in its row a node's token is drawn
  const float* accept;       // [B, n], with q: a draft's own number
  int* choice;               // workspace [B, n]: child that is gone on to, -1
  int* drawn;                // workspace [B, n]: token drawn, -1
  long long rows;
  int n, V, slice;
  double inv_temp;           // 0: the largest logit
  float reach;               // 699 temperatures
  u64 top;                   // the nucleus' mass is top 2^-top_shift; 0: everything
  int top_shift;
  u64 tail;                  // weights (as bits) below it cannot be where the nucleus ends
  int shift;                 // bits of a weight that the first histogram does not look at
  int lazy;                  // more nodes than clusters: nodes that are out of question are passed over
  int wide;                  // logits [node] start where four can be loaded at once
};

struct VerifyShared {
  u64 warp[32];
  u64 part[2];               // what this CTA adds to a sum over the row, two in turn
  u64 seg[VD_MAX_SEGS + 1];
  u64 above;                 // of the nucleus' search: mass above the bin, and the bin
  int bin, listed;
  int off[2];                // whether the node is passed over, in turn: peers may still read the one before
  u64 list_w[VD_LIST];
  int list_i[VD_LIST];
  u64 all_w[VD_LIST];
  int all_i[VD_LIST];
  u64 cut_w;
  int cut_i;
  u64 coarse[VD_COARSE];     // sums of 32 bins
  u64 bins[VD_BINS];
};
constexpr u64 kMostWeight = 0x3ff0000000000100ull;      // bits of 1 + 2^-44
enum : int { kUnknown = -2 };          // a node that is not decided yet
constexpr int kVerifyShared = int((sizeof(VerifyShared) + 15) / 16 * 16);

// What a logit counts as: NaN as -infinity, +infinity as the largest number.
__device__ __forceinline__ float tidy(float x) { return fminf(fmaxf(x, -CUDART_INF_F), 3.402823466e38f); }
// e^x for x <= 0 by Tang's table-driven method (ACM TOMS 15, 1989): x = (32 k + i) ln2 / 32 + r, |r| <= ln2 / 64, e^x = 2^k 2^(i / 32)
// e^r, e^r by its Taylor sum to r^5. `t` is x 32 / ln2 + 1.5 2^52, whose last place is 1. Off by at most 3e-13 (the sum's rest 2e-15, the
// argument's rounding the rest); below e^-693 what comes out is at most that. The table lies in the lanes of a warp, which all take part.
__device__ __forceinline__ double exp_of(double x, double t, double power) {
  const int n = __double2loint(t);
  const double r = fma(6755399441055744. - t, 0.021660849392498290, x);
  double p = fma(r, 1. / 120, 1. / 24);
  p = fma(p, r, 1. / 6);
  p = fma(p, r, .5);
  p = fma(p, r, 1.) * r;
  const int i = n & 31;
  const double T = __hiloint2double(__shfl_sync(0xffffffffu, __double2hiint(power), i), __shfl_sync(0xffffffffu, __double2loint(power), i));
  const double y = fma(T, p, T);
  return __hiloint2double(__double2hiint(y) + (max(n, -32000) >> 5) * (1 << 20), __double2loint(y));
}

// x * total for x = m 2^-k in [0, 1], rounded down or up: exact, so that masses that are equal are so here.
__device__ __forceinline__ u64 part_of(u64 m, int k, u64 total, bool up) {
  const u64 hi = __umul64hi(m, total), lo = m * total;
  if (k <= 0) return lo;                                     // x is 0 or 1
  if (k >= 128) return up && (hi | lo) != 0;
  const u64 whole = k < 64 ? hi << (64 - k) | lo >> k : k == 64 ? hi : hi >> (k - 64);
  const bool rest = k < 64 ? lo << (64 - k) != 0 : lo != 0 || (k > 64 && hi << (128 - k) != 0);
  return whole + (up && rest);
}
// The same for a number of any kind: what is not from [0, 1] counts as the nearest that is, NaN as 0.
__device__ __forceinline__ u64 part_of(float x, u64 total) {
  x = fminf(fmaxf(x, 0.f), 1.f);
  int e;
  const float f = frexpf(x, &e);                             // x = f 2^e, f of 24 bits
  return part_of(u64(f * 16777216.f), 24 - e, total, false);
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sums of the lanes up to and with this one.
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

// The same over the first eight lanes.
__device__ __forceinline__ u64 warp_scan8(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < VD_MAX_CLUSTER; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

template <bool kBf16>
__device__ __forceinline__ float logit_at(const VerifyParams& p, long long node, int j) {
  const long long at = node * p.V + j;
  return tidy(kBf16 ? __bfloat162float(static_cast<const bf16*>(p.logits)[at]) : static_cast<const float*>(p.logits)[at]);
}

// Four logits from an aligned place, as they are.
template <bool kBf16>
__device__ __forceinline__ float4 logits_at(const VerifyParams& p, long long node, int j) {
  const long long at = node * p.V + j;
  if (!kBf16) return *reinterpret_cast<const float4*>(static_cast<const float*>(p.logits) + at);
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const bf16*>(p.logits) + at);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}

// Grid (cluster, nodes), cluster (size, 1, 1).
//
// A CTA's slice of the row goes into shared memory once, in segments of 128 that belong to one warp throughout, four neighbouring tokens
// to a lane. One pass makes all weights and their sum; where the row's weights are needed again they are made again, of the segments alone
// that hold a logit in question. The nucleus' end is looked for in a histogram of masses over the weights' bits (an order of positive
// numbers), in finer ones while too many tokens share the bin, and then token by token.
template <bool kBf16>
__global__ void __launch_bounds__(VD_THREADS, 2) verify_rows_kernel(const VerifyParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  VerifyShared& sh = *reinterpret_cast<VerifyShared*>(smem);
  float* xs = reinterpret_cast<float*>(smem + kVerifyShared);
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = gridDim.x, rank = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int lo = min(rank * p.slice, p.V), size = min(p.slice, p.V - lo);
  const int segs = (size + VD_SEG - 1) / VD_SEG;
  const int bits = min(62 - (32 - __clz(p.V)), 51);
  const double unit = __hiloint2double((1023 + bits) << 20, 0);      // 2^bits
  const double kRest = 2251799813685248.;                    // 2^51, the same for what refusals leave
  const double power = exp2(double(lane) / 32.);
  pdl_wait();
  pdl_trigger();
  int phase = 0, parity = 0;
  auto meet = [&] {
    if (cs > 1) cluster.sync();
    else __syncthreads();
  };
  // Sum over the row, with what stands in front of this CTA; all threads.
  auto row_sum = [&](u64 v, u64* before) {
    v = warp_sum(v);
    if (lane == 0) sh.warp[warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = warp_sum(lane < VD_WARPS ? sh.warp[lane] : 0);
      if (lane == 0) sh.part[phase] = v;
    }
    meet();
    // a lane for each CTA: one after the other the reads would be eight times as long on their way
    const u64 x = lane < cs ? *cluster.map_shared_rank(&sh.part[phase], lane) : 0;
    phase ^= 1;
    const u64 upto = warp_scan8(x, lane);
    if (before != nullptr) *before = __shfl_sync(0xffffffffu, upto - x, rank);
    return __shfl_sync(0xffffffffu, upto, VD_MAX_CLUSTER - 1);
  };
  auto row_max = [&](uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (lane == 0) sh.warp[warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = __reduce_max_sync(0xffffffffu, lane < VD_WARPS ? uint32_t(sh.warp[lane]) : 0u);
      if (lane == 0) sh.part[phase] = v;
    }
    meet();
    const uint32_t x = lane < cs ? uint32_t(*cluster.map_shared_rank(&sh.part[phase], lane)) : 0u;
    phase ^= 1;
    return __reduce_max_sync(0xffffffffu, x);
  };
  // An integer number of units, rounded to nearest: the last bits of a sum with 2^52.
  auto fixed = [](double w, double u) { return u64(__double_as_longlong(fma(w, u, 4503599627370496.))) - 0x4330000000000000ull; };

  if (p.lazy && cs > 1) cluster.sync();                      // the first CTA writes into the others: they have to be there
  // Node 0 of all sequences, node 1 of all, ...: a parent is decided before its children begin, if they begin in a later round.
  const long long B = p.rows / p.n;
  for (long long turn = blockIdx.y; turn < p.rows; turn += gridDim.y) {
    const int i = int(turn / B);
    const long long first = turn % B * p.n, node = first + i;          // the sequence's node 0, this one
    const int up = i == 0 ? -1 : p.parents[node];
    if (i > 0 && (up < 0 || up >= i)) continue;              // not there (the same for the whole cluster)
    if (p.lazy) {                                            // a node that the text has not come to is not looked at: what one CTA sees
      __syncthreads();
      if (rank == 0 && warp == 0) {
        int above[2], chosen[2], off = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = 32 * e + lane;
          above[e] = j < p.n ? p.parents[first + j] : -1;
          chosen[e] = j < p.n ? *const_cast<volatile int*>(p.choice + first + j) : kUnknown;
        }
        for (int j = i; j > 0 && !off;) {                    // up to the root: each on the way is its parent's choice, or nobody knows
          const int a = j < 32 ? __shfl_sync(0xffffffffu, above[0], j) : __shfl_sync(0xffffffffu, above[1], j - 32);
          if (a < 0 || a >= j) {                             // below a node that is not there
            off = 1;
          } else {
            const int c = a < 32 ? __shfl_sync(0xffffffffu, chosen[0], a) : __shfl_sync(0xffffffffu, chosen[1], a - 32);
            off = c != kUnknown && c != j;
          }
          j = a;
        }
        if (lane < cs) *cluster.map_shared_rank(&sh.off[parity], lane) = off;
        if (off && lane == 0) p.choice[node] = -1;
      }
      meet();
      parity ^= 1;
      if (sh.off[parity ^ 1]) continue;
    }
    __syncthreads();
    // Which drafts are this node's children, and what the end will want to know of them: a lane holds drafts `lane` and 32 + lane.
    int tok[2];
    float child_x[2] = {0.f, 0.f}, child_q[2] = {0.f, 0.f}, child_a[2] = {0.f, 0.f};
    uint32_t kid[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 32 * e + lane;
      const bool mine = j > i && j < p.n && p.parents[first + j] == i;
      tok[e] = mine ? p.tokens[first + j] : -1;
      kid[e] = __ballot_sync(0xffffffffu, mine && tok[e] >= 0 && tok[e] < p.V);
      if (p.q != nullptr && (kid[e] >> lane & 1)) {
        child_x[e] = logit_at<kBf16>(p, node, tok[e]);
        child_q[e] = p.q[node * p.V + tok[e]];
        child_a[e] = p.accept[first + j];
      }
    }
    const u64 kids = u64(kid[1]) << 32 | kid[0];
    const float drawn_at = p.u[node];
    auto of = [&](const auto (&x)[2], int j) {
      const auto a = __shfl_sync(0xffffffffu, x[0], j & 31), c = __shfl_sync(0xffffffffu, x[1], j & 31);
      return j < 32 ? a : c;
    };
    float top = -CUDART_INF_F;
    for (int s0 = warp; s0 < segs; s0 += 4 * VD_WARPS) {     // four segments on their way at a time
      float4 x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = (s0 + c * VD_WARPS) * VD_SEG + 4 * lane;
        if (p.wide && j + 3 < size) {
          x[c] = logits_at<kBf16>(p, node, lo + j);
        } else {
          x[c].x = j < size ? logit_at<kBf16>(p, node, lo + j) : -CUDART_INF_F;
          x[c].y = j + 1 < size ? logit_at<kBf16>(p, node, lo + j + 1) : -CUDART_INF_F;
          x[c].z = j + 2 < size ? logit_at<kBf16>(p, node, lo + j + 2) : -CUDART_INF_F;
          x[c].w = j + 3 < size ? logit_at<kBf16>(p, node, lo + j + 3) : -CUDART_INF_F;
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (s0 + c * VD_WARPS >= segs) break;
        const float4 y = make_float4(tidy(x[c].x), tidy(x[c].y), tidy(x[c].z), tidy(x[c].w));
        reinterpret_cast<float4*>(xs)[(s0 + c * VD_WARPS) * 32 + lane] = y;
        top = fmaxf(fmaxf(fmaxf(top, y.x), fmaxf(y.y, y.z)), y.w);
      }
    }
    // fp32 numbers in the order of unsigned ones
    const uint32_t ub = __float_as_uint(top), most = row_max(ub & 0x80000000u ? ~ub : ub | 0x80000000u);
    const float largest = __uint_as_float(most & 0x80000000u ? most & 0x7fffffffu : ~most);
    if (largest == -CUDART_INF_F) {                          // nothing to choose
      if (rank == 0 && tid == 0) {
        p.choice[node] = -1;
        p.drawn[node] = -1;
      }
      continue;
    }
    int arg = -1;                                            // temperature 0: the first of the largest
    if (p.inv_temp == 0.) {
      uint32_t lowest = 0;
      for (int j = tid; j < size; j += VD_THREADS)
        if (xs[j] == largest) lowest = max(lowest, ~uint32_t(lo + j));
      arg = int(~row_max(lowest));
    }
    // The weight of token j, 1 for the largest; whole warps. What is more than 699 temperatures below has none (in fp32: up to twice that).
    const double per32 = p.inv_temp * 46.166241308446828;                               // 32 / ln2
    const float none = largest - p.reach;
    auto raw = [&](float x, int j) {
      if (p.inv_temp == 0.) return j == arg ? 1. : 0.;
      const double d = double(x < none ? largest : x) - double(largest);
      const double w = exp_of(d * p.inv_temp, fma(d, per32, 6755399441055744.), power);
      return x < none ? 0. : w;
    };
    const bool nucleus = p.top != 0 && p.inv_temp != 0.;
    // Bits of the four weights of a lane in segment s; false (and none) if no logit of the segment is `from` or more.
    auto weights = [&](int s, float from, u64 (&k)[4]) {
      const float4 x = reinterpret_cast<const float4*>(xs)[s * 32 + lane];
      const float y[4] = {x.x, x.y, x.z, x.w};
      if (!__any_sync(0xffffffffu, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) >= from)) return false;
#pragma unroll
      for (int e = 0; e < 4; ++e) k[e] = u64(__double_as_longlong(raw(y[e], lo + s * VD_SEG + 4 * lane + e)));
      return true;
    };
    // A logit that is at most that of a weight: from the logarithm in fp32, 2^-20 of what goes into it to spare.
    auto logit_of = [&](u64 k) {
      if (k == 0 || p.inv_temp == 0.) return -CUDART_INF_F;
      const float d = logf(float(__longlong_as_double((long long)k))) / float(p.inv_temp);
      return largest + d - 9.5e-7f * (fabsf(largest) + fabsf(d) + 1.f / float(p.inv_temp));
    };
    u64 cut_w = 0;                                           // weights below it are cut off, and those equal to it behind token cut_i
    int cut_i = 0x7fffffff;
    u64 khi = kMostWeight + 1, above = 0;              // the end lies in [klo, khi) (bits of weights), and this much above it
    u64 klo = p.tail;
    int shift = p.shift;
    if (nucleus) {
      for (int t = tid; t < VD_BINS; t += VD_THREADS) sh.bins[t] = 0;
      __syncthreads();
    }
    // All weights: sums of the segments, or the first histogram.
    u64 mine = 0;
    for (int s = warp; s < segs; s += VD_WARPS) {
      u64 k[4], v = 0;
      if (weights(s, -CUDART_INF_F, k)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u64 f = fixed(__longlong_as_double((long long)k[e]), unit);
          v += f;
          if (nucleus && k[e] >= klo) atomicAdd(&sh.bins[(khi - 1 - k[e]) >> shift], f);
        }
      }
      mine += v;
      if (!nucleus) {
        v = warp_sum(v);
        if (lane == 0) sh.seg[s] = v;
      }
    }
    auto coarse = [&] {                                      // all threads, the bins complete
      __syncthreads();
      for (int t = warp; t < VD_COARSE; t += VD_WARPS) {
        const u64 v = warp_sum(sh.bins[32 * t + lane]);
        if (lane == 0) sh.coarse[t] = v;
      }
    };
    if (nucleus) coarse();
    u64 before, total = row_sum(mine, &before);
    if (nucleus) {
      const u64 want = part_of(p.top, p.top_shift, total, true);
      while (true) {
        // The bin in which the masses of all CTAs reach `want`: among 64 sums of 32, then among those 32.
        if (warp == 0) {
          auto of_all = [&](const u64* at) {
            u64 x[VD_MAX_CLUSTER], v = 0;
#pragma unroll
            for (int c = 0; c < VD_MAX_CLUSTER; ++c) x[c] = c < cs ? *cluster.map_shared_rank(at, c) : 0;
#pragma unroll
            for (int c = 0; c < VD_MAX_CLUSTER; ++c) v += x[c];
            return v;
          };
          int bin = -1;
          u64 at = above;
          const u64 a = of_all(&sh.coarse[2 * lane]), c = of_all(&sh.coarse[2 * lane + 1]), scan = warp_scan(a + c, lane);
          const uint32_t over = __ballot_sync(0xffffffffu, at + scan >= want);
          if (over != 0) {
            const int l = __ffs(over) - 1;
            at += __shfl_sync(0xffffffffu, scan - a - c, l);
            const u64 low = __shfl_sync(0xffffffffu, a, l);
            const bool second = at + low < want;
            at += second ? low : 0;
            const int block = 2 * l + second;
            const u64 v = of_all(&sh.bins[32 * block + lane]), upto = warp_scan(v, lane);
            const uint32_t fine = __ballot_sync(0xffffffffu, at + upto >= want);
            const int f = fine != 0 ? __ffs(fine) - 1 : 31;
            at += __shfl_sync(0xffffffffu, upto - v, f);
            bin = 32 * block + f;
          }
          if (lane == 0) {
            sh.bin = bin;
            sh.above = at;
            sh.listed = 0;
          }
        }
        __syncthreads();
        if (sh.bin < 0) break;                               // (cannot be: everything is kept)
        above = sh.above;
        khi -= u64(sh.bin) << shift;
        klo = khi - klo > 1ull << shift ? khi - (1ull << shift) : klo;
        // Its tokens, if they are few.
        const float from = logit_of(klo);
        for (int s = warp; s < segs; s += VD_WARPS) {
          u64 k[4];
          if (!weights(s, from, k)) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k[e] >= klo && k[e] < khi && k[e] != 0) {
              const int n = atomicAdd(&sh.listed, 1);
              if (n < VD_LIST) {
                sh.list_w[n] = k[e];
                sh.list_i[n] = lo + s * VD_SEG + 4 * lane + e;
              }
            }
        }
        meet();
        const int found = lane < cs ? min(*cluster.map_shared_rank(&sh.listed, lane), 1 << 24) : 0;
        const int upto = int(warp_scan8(u64(found), lane));
        const int all = __shfl_sync(0xffffffffu, upto, VD_MAX_CLUSTER - 1);
        if (all <= VD_LIST) {
          int c = 0, at0 = 0;                                // token `tid` of all: whose it is, and how many stand before that CTA's
#pragma unroll
          for (int o = 0; o < VD_MAX_CLUSTER - 1; ++o) {
            const int n = __shfl_sync(0xffffffffu, upto, o);
            if (tid >= n && o + 1 < cs) {
              c = o + 1;
              at0 = n;
            }
          }
          if (tid < all) {
            sh.all_w[tid] = *cluster.map_shared_rank(&sh.list_w[tid - at0], c);
            sh.all_i[tid] = *cluster.map_shared_rank(&sh.list_i[tid - at0], c);
          }
          __syncthreads();
          if (tid < all) {
            const u64 k = sh.all_w[tid];
            const int j = sh.all_i[tid];
            u64 front = above;
            for (int o = 0; o < all; ++o) {
              const u64 ko = sh.all_w[o];
              if (ko > k || (ko == k && sh.all_i[o] < j)) front += fixed(__longlong_as_double((long long)ko), unit);
            }
            const u64 f = fixed(__longlong_as_double((long long)k), unit);
            if (front < want && front + f >= want) {
              sh.cut_w = k;
              sh.cut_i = j;
            }
          }
          __syncthreads();
          cut_w = sh.cut_w;
          cut_i = sh.cut_i;
          break;
        }
        if (shift == 0) {                                    // one weight, which many tokens have: the first of them that reach the mass
          const u64 each = fixed(__longlong_as_double((long long)klo), unit);
          u64 need = each == 0 || want <= above + each ? 1 : (want - above + each - 1) / each;
          mine = 0;
          for (int s = warp; s < segs; s += VD_WARPS) {
            u64 k[4], n = 0;
            if (weights(s, from, k)) n = (k[0] == klo) + (k[1] == klo) + (k[2] == klo) + (k[3] == klo);
            n = warp_sum(n);
            if (lane == 0) sh.seg[s] = n;
            mine += lane == 0 ? n : 0;
          }
          const u64 ties = row_sum(mine, &before);
          need = min(need, ties);
          cut_w = klo;
          if (tid == 0) sh.cut_i = -1;
          __syncthreads();
          if (warp == 0) {                                   // the owner of the last one: its segment, then its place
            u64 sum = before;
            for (int s = 0; s < segs; ++s) {
              u64 k[4];
              if (sum < need && sum + sh.seg[s] >= need && weights(s, from, k)) {
                const u64 n = (k[0] == klo) + (k[1] == klo) + (k[2] == klo) + (k[3] == klo);
                u64 at = sum + warp_scan(n, lane) - n;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (k[e] == klo && ++at == need) sh.cut_i = lo + s * VD_SEG + 4 * lane + e;
              }
              sum += sh.seg[s];
            }
          }
          __syncthreads();
          cut_i = int(row_max(tid == 0 ? uint32_t(sh.cut_i + 1) : 0u)) - 1;
          break;
        }
        // Too many: their masses in finer bins.
        shift = shift > 11 ? shift - 11 : 0;
        for (int t = tid; t < VD_BINS; t += VD_THREADS) sh.bins[t] = 0;
        __syncthreads();
        for (int s = warp; s < segs; s += VD_WARPS) {
          u64 k[4];
          if (!weights(s, from, k)) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k[e] >= klo && k[e] < khi)
              atomicAdd(&sh.bins[(khi - 1 - k[e]) >> shift], fixed(__longlong_as_double((long long)k[e]), unit));
        }
        coarse();
        meet();
      }
    }
    const float* q = p.q != nullptr ? p.q + node * p.V : nullptr;
    double used = 0., mass = 1., norm = 0.;
    auto kept = [&](double w, int j) {                       // of the nucleus
      const u64 k = u64(__double_as_longlong(w));
      return k > cut_w || (k == cut_w && j <= cut_i);
    };
    // What a lane adds to the sum of segment s: of w, or of max(p - used q, 0) in units of kRest.
    auto shares = [&](int s, bool rest, float from, u64 (&v)[4]) {
      u64 k[4];
      if (!weights(s, from, k)) return false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = lo + s * VD_SEG + 4 * lane + e;
        const double w = kept(__longlong_as_double((long long)k[e]), j) ? __longlong_as_double((long long)k[e]) : 0.;
        v[e] = !rest ? fixed(w, unit) : w > 0. ? fixed(fmax(w * norm - used * double(q[j]), 0.), kRest) : 0;
      }
      return true;
    };
    const float least = logit_of(cut_w);
    auto sum_up = [&](bool rest) {
      u64 sum = 0;
      for (int s = warp; s < segs; s += VD_WARPS) {
        u64 v[4], t = 0;
        if (shares(s, rest, least, v)) t = warp_sum(v[0] + v[1] + v[2] + v[3]);
        if (lane == 0) {
          sh.seg[s] = t;
          sum += t;
        }
      }
      return row_sum(sum, &before);
    };
    if (nucleus) total = sum_up(false);
    norm = unit / double(total);                             // weight -> probability
    int go = -1;
    u64 all = total;
    bool rest = false;
    if (q != nullptr) {
      for (u64 left = kids; left != 0 && go < 0; left &= left - 1) {
        const int j = __ffsll((long long)left) - 1, t = of(tok, j);
        const double w = raw(of(child_x, j), t);
        const double px = kept(w, t) ? w * norm : 0., qx = double(of(child_q, j));
        if (double(of(child_a, j)) * qx * mass < fmax(px - used * qx, 0.)) {
          go = j;
        } else {
          used += mass;
          rest = true;
          all = sum_up(true);
          mass = double(all) / kRest;
        }
      }
      if (go < 0 && rest && all == 0) {                      // nothing left: p itself
        rest = false;
        all = sum_up(false);
      }
    }
    if (go >= 0) {
      if (rank == 0 && tid == 0) {
        p.choice[node] = go;
        p.drawn[node] = -1;
      }
      continue;
    }
    // Where the number falls, in the order of the tokens: the CTA, the segment, the token.
    const u64 target = min(part_of(drawn_at, all), all - 1), own = sh.part[phase ^ 1];
    if (target >= before && target < before + own && warp == 0) {
      u64 sum = before;
      int s = 0;
      for (int s0 = 0; s0 < segs; s0 += 32) {
        const u64 v = warp_scan(s0 + lane < segs ? sh.seg[s0 + lane] : 0, lane);
        const uint32_t over = __ballot_sync(0xffffffffu, sum + v > target);
        if (over != 0) {
          const int l = __ffs(over) - 1;
          s = s0 + l;
          const u64 x = __shfl_sync(0xffffffffu, v, max(l - 1, 0));
          sum += l > 0 ? x : 0;
          break;
        }
        sum += __shfl_sync(0xffffffffu, v, 31);
      }
      u64 v[4] = {0, 0, 0, 0};
      shares(s, rest, least, v);
      const u64 here = v[0] + v[1] + v[2] + v[3];
      const u64 upto = warp_scan(here, lane);
      const uint32_t over = __ballot_sync(0xffffffffu, sum + upto > target);
      if (lane == __ffs(over) - 1) {
        u64 c = sum + upto - here;
        int e = 0;
#pragma unroll
        for (int x = 0; x < 3; ++x)
          if (e == x && c + v[x] <= target) {
            c += v[x];
            ++e;
          }
        sum = u64(lo + s * VD_SEG + 4 * lane + e);
      }
      const int token = __shfl_sync(0xffffffffu, int(sum), __ffs(over) - 1);
      if (q == nullptr) {                                    // the first child that holds it
        const uint32_t a = __ballot_sync(0xffffffffu, tok[0] == token) & kid[0], c = __ballot_sync(0xffffffffu, tok[1] == token) & kid[1];
        go = a != 0 ? __ffs(a) - 1 : c != 0 ? 31 + __ffs(c) : -1;
      }
      if (lane == 0) {
        p.choice[node] = go;
        p.drawn[node] = token;
      }
    }
  }
  if (cs > 1) cluster.sync();                                // peers read this CTA's numbers until here
}

// Nothing is decided yet.
__global__ void __launch_bounds__(256) verify_begin_kernel(int* choice, long long rows) {
  pdl_wait();
  pdl_trigger();
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i < rows) choice[i] = kUnknown;
}

struct WalkParams {
  const int* choice;
  const int* drawn;
  const int* tokens;
  int* out;              // [B, n]: the drafts that are kept, then the token behind them, then -1
  int* path;             // [B, n]: the nodes that are kept, then -1
  int* count;            // [B]
  int B, n;
};

// A warp per sequence, which holds up to 64 nodes in two registers.
__global__ void __launch_bounds__(128) verify_walk_kernel(const WalkParams p) {
  const int b = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  if (b >= p.B) return;
  const long long first = (long long)b * p.n;
  int next[2], draw[2], tok[2], out[2] = {-1, -1}, path[2] = {-1, -1};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 32 * e + lane;
    next[e] = i < p.n ? p.choice[first + i] : -1;
    draw[e] = i < p.n ? p.drawn[first + i] : -1;
    tok[e] = i < p.n ? p.tokens[first + i] : -1;
  }
  auto of = [&](const int (&x)[2], int i) {
    const int a = __shfl_sync(0xffffffffu, x[0], i & 31), c = __shfl_sync(0xffffffffu, x[1], i & 31);
    return i < 32 ? a : c;
  };
  int node = 0, count = 0;
  while (true) {
    const int go = of(next, node);
    const int t = go >= 0 ? of(tok, go) : of(draw, node);
    if (lane == (count & 31)) {
      if (count < 32) out[0] = t;
      else out[1] = t;
      if (go >= 0) (count < 32 ? path[0] : path[1]) = go;
    }
    if (go <= node) break;                                   // a child stands behind its parent, so this ends
    node = go;
    ++count;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 32 * e + lane;
    if (i >= p.n) continue;
    p.out[first + i] = out[e];
    p.path[first + i] = path[e];
  }
  if (lane == 0) p.count[b] = count;
}

// How many clusters of `cs` CTAs with `smem` bytes each run at the same time: registers allow two CTAs an SM, shared memory perhaps one,
// and a cluster lies within one GPC. The last answer is kept for each device, type of logits and size of clusters.
template <typename Kernel>
static long long clusters_at_once(Kernel kern, int dev, bool bf16_logits, int cs, int smem) {
  static std::atomic<u64> kept[64][2][4];                    // shared memory and count
  std::atomic<u64>* at = dev >= 0 && dev < 64 ? &kept[dev][bf16_logits][cs == 8 ? 3 : cs >> 1] : nullptr;
  const u64 known = at != nullptr ? at->load(std::memory_order_relaxed) : 0;
  if (known != 0 && int(known >> 32) == smem) return (long long)(known & 0xffffffffu);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cs);
  cfg.blockDim = dim3(VD_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return std::max(1, num_sms() / cs);
  }
  if (at != nullptr) at->store(u64(smem) << 32 | u64(n), std::memory_order_relaxed);
  return n;
}

}  // namespace b200

using namespace b200;

// logits [B, n, V] (bf16: is_bf16), tokens, parents [B, n], u [B, n]; q [B, n, V] with accept [B, n], or both null. temp 0: the largest
// logit. out, path [B, n], count [B]; workspace: 2 B n ints.
B200_API int b200_verify_drafts(const void* logits, const void* q, const void* tokens, const void* parents, const void* u,
                                const void* accept, void* out, void* path, void* count, void* workspace, int is_bf16, int B, int n, int V,
                                double temp, double top, cudaStream_t st) {
  if (B < 0 || n < 1 || n > VD_MAX_NODES || V < 1 || !(temp == 0. || (temp >= 1e-6 && temp <= 1e6)) || !(top > 0.) ||
      (q == nullptr) != (accept == nullptr))
    return static_cast<int>(cudaErrorInvalidValue);
  if (B == 0) return 0;
  VerifyParams p;
  p.logits = logits;
  p.q = static_cast<const float*>(q);
  p.tokens = static_cast<const int*>(tokens);
  p.parents = static_cast<const int*>(parents);
  p.u = static_cast<const float*>(u);
  p.accept = static_cast<const float*>(accept);
  p.choice = static_cast<int*>(workspace);
  p.drawn = p.choice + (long long)B * n;
  p.rows = (long long)B * n;
  p.n = n; p.V = V;
  p.inv_temp = temp > 0. ? 1. / temp : 0.;
  p.reach = float(699. * temp);
  p.top = 0;
  p.top_shift = 0;
  if (top < 1.) {
    int e;
    p.top = static_cast<u64>(std::ldexp(std::frexp(top, &e), 53));
    p.top_shift = 53 - e;
  }
  const double missing = 1. - top, tail = missing > 1e-6 ? 0.9 * missing / V : 0.;
  p.tail = 0;
  memcpy(&p.tail, &tail, 8);
  p.shift = 0;
  while ((kMostWeight - p.tail) >> p.shift >= VD_BINS) ++p.shift;
  p.wide = V % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & (is_bf16 ? 7 : 15)) == 0;
  constexpr int kMostSlice = VD_MAX_SEGS * VD_SEG;
  int cs = 1;
  while (cs < VD_MAX_CLUSTER && (cs * 16384LL < V || cs * p.rows * 2 <= num_sms())) cs *= 2;
  if ((long long)cs * kMostSlice < V) return static_cast<int>(cudaErrorInvalidValue);
  p.slice = ((V + cs - 1) / cs + VD_SEG - 1) / VD_SEG * VD_SEG;
  const int smem = kVerifyShared + p.slice * 4;
  static std::atomic<bool> allowed[2][64];
  const auto kern = is_bf16 ? verify_rows_kernel<true> : verify_rows_kernel<false>;
  std::atomic<bool>* known = allowed[is_bf16 != 0];
  int dev = 0;
  B200_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !known[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kVerifyShared + kMostSlice * 4);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return static_cast<int>(e);
    }
    if (dev >= 0 && dev < 64) known[dev].store(true, std::memory_order_release);
  }
  // CTAs that stay: a cluster takes node after node.
  const long long most = clusters_at_once(kern, dev, is_bf16 != 0, cs, smem);
  p.lazy = p.rows > most && n > 1;
  if (p.lazy) B200_CHECK(launch_pdl(verify_begin_kernel, dim3(unsigned((p.rows + 255) / 256)), dim3(256), 0, st, 0, p.choice, p.rows));
  B200_CHECK(launch_pdl(kern, dim3(cs, unsigned(std::min(p.rows, most))), dim3(VD_THREADS), smem, st, cs, p));
  WalkParams w;
  w.choice = p.choice; w.drawn = p.drawn; w.tokens = p.tokens;
  w.out = static_cast<int*>(out);
  w.path = static_cast<int*>(path);
  w.count = static_cast<int*>(count);
  w.B = B; w.n = n;
  return static_cast<int>(launch_pdl(verify_walk_kernel, dim3((B + 3) / 4), dim3(128), 0, st, 0, w));
}
