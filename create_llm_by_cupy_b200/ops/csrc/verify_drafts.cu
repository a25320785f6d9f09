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
#include <cooperative_groups.h>
#include <math_constants.h>

#include <atomic>
#include <cmath>

#include "common.cuh"

namespace b200 {
namespace cg = cooperative_groups;

typedef unsigned long long u64;

constexpr int VD_THREADS = 512, VD_WARPS = VD_THREADS / 32, VD_SEG = 128, VD_MAX_SEGS = 416, VD_MAX_NODES = 64, VD_MAX_CLUSTER = 8;

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
  u64 top;                   // the nucleus' mass is top 2^-top_shift; 0: everything
  int top_shift;
};

struct VerifyShared {
  u64 warp[VD_WARPS];
  u64 part[2][2];            // what this CTA adds to a sum over the row
  u64 seg[VD_MAX_SEGS];
  int first[VD_WARPS];
};

// Order of fp32 numbers as an order of unsigned ones; NaN has become -infinity, and +infinity the largest number, before.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float tidy(float x) { return x != x ? -CUDART_INF_F : fminf(x, 3.402823466e38f); }

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

template <bool kBf16>
__global__ void __launch_bounds__(VD_THREADS) verify_rows_kernel(const VerifyParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  VerifyShared& sh = *reinterpret_cast<VerifyShared*>(smem);
  float* xs = reinterpret_cast<float*>(smem + (sizeof(VerifyShared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = gridDim.x, rank = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int lo = min(rank * p.slice, p.V), size = min(p.slice, p.V - lo);
  const int segs = (size + VD_SEG - 1) / VD_SEG;
  const double unit = exp2(double(62 - (32 - __clz(p.V))));
  pdl_wait();
  pdl_trigger();
  int phase = 0;
  // Sum over the row, with what stands in front of this CTA; all threads.
  auto row_sum = [&](u64 v, u64* before) {
    v = warp_sum(v);
    if (lane == 0) sh.warp[warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = warp_sum(lane < VD_WARPS ? sh.warp[lane] : 0);
      if (lane == 0) sh.part[phase][0] = v;
    }
    cluster.sync();
    u64 all = 0, ahead = 0;
    for (int c = 0; c < cs; ++c) {
      const u64 x = *cluster.map_shared_rank(&sh.part[phase][0], c);
      if (c < rank) ahead += x;
      all += x;
    }
    phase ^= 1;
    if (before != nullptr) *before = ahead;
    return all;
  };
  auto row_max = [&](u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0) sh.warp[warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = lane < VD_WARPS ? sh.warp[lane] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
      if (lane == 0) sh.part[phase][0] = v;
    }
    cluster.sync();
    u64 all = 0;
    for (int c = 0; c < cs; ++c) all = max(all, *cluster.map_shared_rank(&sh.part[phase][0], c));
    phase ^= 1;
    return all;
  };

  for (long long node = blockIdx.y; node < p.rows; node += gridDim.y) {
    const int i = int(node % p.n);
    const long long first = node - i;                        // the sequence's node 0
    const int up = i == 0 ? -1 : p.parents[node];
    if (i > 0 && (up < 0 || up >= i)) continue;              // not there (the same for the whole cluster)
    auto at = [&](int j) {
      return tidy(kBf16 ? __bfloat162float(static_cast<const bf16*>(p.logits)[node * p.V + j]) : static_cast<const float*>(p.logits)[node * p.V + j]);
    };
    u64 best = 0;                                            // largest logit, lowest index
    __syncthreads();
    for (int j = tid; j < size; j += VD_THREADS) {
      const float x = at(lo + j);
      xs[j] = x;
      best = max(best, u64(order_key(x)) << 32 | uint32_t(~(lo + j)));
    }
    best = row_max(best);
    const int arg = int(~uint32_t(best));
    const float largest = tidy(at(arg));
    if (largest == -CUDART_INF_F) {                          // nothing to choose
      if (rank == 0 && tid == 0) {
        p.choice[node] = -1;
        p.drawn[node] = -1;
      }
      continue;
    }
    auto raw = [&](float x, int j) {                         // weight of token j, 1 for the largest
      return p.inv_temp == 0. ? (j == arg ? 1. : 0.) : exp((double(x) - double(largest)) * p.inv_temp);
    };
    auto fixed = [&](double w) { return u64(__double2ull_rn(w * unit)); };
    u64 mine = 0;
    for (int j = tid; j < size; j += VD_THREADS) mine += fixed(raw(xs[j], lo + j));
    u64 total = row_sum(mine, nullptr);
    uint32_t cut = 0;                                        // keys below it are cut off, and those equal to it behind `last`
    int last = 0x7fffffff;
    if (p.top != 0 && p.inv_temp != 0.) {
      // The largest key with which the tokens from it on reach the mass.
      const u64 want = part_of(p.top, p.top_shift, total, true);
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = cut | 1u << bit;
        mine = 0;
        for (int j = tid; j < size; j += VD_THREADS)
          if (order_key(xs[j]) >= trial) mine += fixed(raw(xs[j], lo + j));
        if (row_sum(mine, nullptr) >= want) cut = trial;
      }
      mine = 0;
      u64 same = 0;
      for (int j = tid; j < size; j += VD_THREADS) {
        const uint32_t k = order_key(xs[j]);
        if (k > cut) mine += fixed(raw(xs[j], lo + j));
        if (k == cut) ++same;
      }
      const u64 above = row_sum(mine, nullptr), ties = row_sum(same, nullptr);
      if (ties > 1) {
        const uint32_t ku = cut & 0x80000000u ? cut & 0x7fffffffu : ~cut;
        const u64 each = fixed(raw(__uint_as_float(ku), -1));
        // how many of the equal ones: the fewest that reach the mass
        const u64 need = each == 0 || want <= above + each ? 1 : (want - above + each - 1) / each;
        if (need < ties) {                                   // the index of the last one that is kept
          int low = 0, high = p.V - 1;
          while (low < high) {
            const int mid = low + (high - low) / 2;
            same = 0;
            for (int j = tid; j < size; j += VD_THREADS) same += order_key(xs[j]) == cut && lo + j <= mid;
            if (row_sum(same, nullptr) >= need) high = mid;
            else low = mid + 1;
          }
          last = low;
        }
      }
    }
    auto weight = [&](float x, int j) {
      const uint32_t k = order_key(x);
      return k > cut || (k == cut && j <= last) ? raw(x, j) : 0.;
    };
    if (cut != 0) {
      mine = 0;
      for (int j = tid; j < size; j += VD_THREADS) mine += fixed(weight(xs[j], lo + j));
      total = row_sum(mine, nullptr);
    }
    // Children, as bits.
    u64 kids = 0;
    for (int j = i + 1; j < p.n; ++j) kids |= u64(p.parents[first + j] == i) << j;
    int go = -1;
    double used = 0., mass = 1.;
    const double norm = unit / double(total);                // weight -> probability
    const double kUnit = 1152921504606846976.;               // 2^60
    const float* q = p.q != nullptr ? p.q + node * p.V : nullptr;
    if (q != nullptr) {
      for (u64 left = kids; left != 0 && go < 0; left &= left - 1) {
        const int j = __ffsll((long long)left) - 1, t = p.tokens[first + j];
        if (t < 0 || t >= p.V) continue;
        const double px = weight(at(t), t) * norm, qx = double(q[t]);
        if (double(p.accept[first + j]) * qx * mass < fmax(px - used * qx, 0.)) {
          go = j;
        } else {
          used += mass;
          mine = 0;
          for (int v = tid; v < size; v += VD_THREADS)
            mine += __double2ull_rn(fmax(weight(xs[v], lo + v) * norm - used * double(q[lo + v]), 0.) * kUnit);
          mass = double(row_sum(mine, nullptr)) / kUnit;
        }
      }
    }
    int token = -1;
    if (go < 0) {
      // Where the number falls, in the order of the tokens: the segment of 128, then the token.
      const bool rest = q != nullptr && used > 0. && mass > 0.;
      auto share = [&](int j) {                              // j: place in the slice
        if (j >= size) return u64(0);
        const double w = weight(xs[j], lo + j);
        return rest ? u64(__double2ull_rn(fmax(w * norm - used * double(q[lo + j]), 0.) * kUnit)) : fixed(w);
      };
      mine = 0;
      for (int s = warp; s < segs; s += VD_WARPS) {
        u64 v = 0;
#pragma unroll
        for (int e = 0; e < VD_SEG / 32; ++e) v += share(s * VD_SEG + lane * (VD_SEG / 32) + e);
        v = warp_sum(v);
        if (lane == 0) sh.seg[s] = v;
        mine += lane == 0 ? v : 0;
      }
      u64 before;
      const u64 all = row_sum(mine, &before);
      const u64 target = min(part_of(p.u[node], all), all - 1);
      const u64 own = sh.part[phase ^ 1][0];
      if (target >= before && target < before + own && warp == 0) {
        u64 sum = before;
        int s = 0;
        for (int s0 = 0; s0 < segs; s0 += 32) {              // 32 segments at a time
          u64 v = s0 + lane < segs ? sh.seg[s0 + lane] : 0;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const u64 x = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += x;
          }
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
        u64 v[VD_SEG / 32], here = 0;
#pragma unroll
        for (int e = 0; e < VD_SEG / 32; ++e) here += v[e] = share(s * VD_SEG + lane * (VD_SEG / 32) + e);
        u64 upto = here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 x = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += x;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, sum + upto > target);
        if (lane == __ffs(over) - 1) {
          u64 c = sum + upto - here;
          int e = 0;
          while (e < VD_SEG / 32 - 1 && c + v[e] <= target) c += v[e++];
          token = lo + s * VD_SEG + lane * (VD_SEG / 32) + e;
          if (q == nullptr)
            for (u64 left = kids; left != 0 && go < 0; left &= left - 1) {
              const int j = __ffsll((long long)left) - 1;
              if (p.tokens[first + j] == token) go = j;
            }
          p.choice[node] = go;
          p.drawn[node] = token;
        }
      }
    } else if (rank == 0 && tid == 0) {
      p.choice[node] = go;
      p.drawn[node] = -1;
    }
  }
  cluster.sync();                                            // peers read this CTA's sums until here
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

}  // namespace b200

using namespace b200;

// logits [B, n, V] (bf16: is_bf16), tokens, parents [B, n], u [B, n]; q [B, n, V] with accept [B, n], or both null. temp 0: the largest
// logit. out, path [B, n], count [B]; workspace: 2 B n ints.
B200_API int b200_verify_drafts(const void* logits, const void* q, const void* tokens, const void* parents, const void* u,
                                const void* accept, void* out, void* path, void* count, void* workspace, int is_bf16, int B, int n, int V,
                                double temp, double top, cudaStream_t st) {
  if (B < 0 || n < 1 || n > VD_MAX_NODES || V < 1 || !(temp >= 0.) || !(top > 0.) || (q == nullptr) != (accept == nullptr))
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
  p.top = 0;
  p.top_shift = 0;
  if (top < 1.) {
    int e;
    p.top = static_cast<u64>(std::ldexp(std::frexp(top, &e), 53));
    p.top_shift = 53 - e;
  }
  constexpr int kMostSlice = VD_MAX_SEGS * VD_SEG;
  int cs = 1;
  while (cs < VD_MAX_CLUSTER && (long long)cs * kMostSlice < V) cs *= 2;
  if ((long long)cs * kMostSlice < V) return static_cast<int>(cudaErrorInvalidValue);
  p.slice = ((V + cs - 1) / cs + VD_SEG - 1) / VD_SEG * VD_SEG;
  const int smem = int((sizeof(VerifyShared) + 15) / 16 * 16) + p.slice * 4;
  static std::atomic<bool> allowed[2][64];
  const auto kern = is_bf16 ? verify_rows_kernel<true> : verify_rows_kernel<false>;
  int dev = 0;
  B200_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !allowed[is_bf16 != 0][dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               int((sizeof(VerifyShared) + 15) / 16 * 16) + kMostSlice * 4);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return static_cast<int>(e);
    }
    if (dev >= 0 && dev < 64) allowed[is_bf16 != 0][dev].store(true, std::memory_order_release);
  }
  const long long rows = p.rows < 65535 ? p.rows : 65535;
  B200_CHECK(launch_pdl(kern, dim3(cs, unsigned(rows)), dim3(VD_THREADS), smem, st, cs, p));
  WalkParams w;
  w.choice = p.choice; w.drawn = p.drawn; w.tokens = p.tokens;
  w.out = static_cast<int*>(out);
  w.path = static_cast<int*>(path);
  w.count = static_cast<int*>(count);
  w.B = B; w.n = n;
  return static_cast<int>(launch_pdl(verify_walk_kernel, dim3((B + 3) / 4), dim3(128), 0, st, 0, w));
}
