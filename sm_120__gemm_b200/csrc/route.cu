// Routing to experts, the order of the routed rows, and their combination.
//
// Scores of a token: p_e = exp(x_e - max x) / sum (softmax) or
// 1 / (1 + exp(-x_e)) (sigmoid). Its choice score is c_e = p_e + bias_e, or the
// logit itself where nothing but the order of the p matters (no bias, no sum
// of group members): the scores rise with the logits, so the order is the
// same and exact. With groups, a group's score is its best member's c, or the
// sum of its best two; only members of the topk_group best groups stay. The
// top_k experts are those of the largest c, ties going to the lowest index;
// their weights are the p (without bias), renormalised to sum 1 if asked,
// times a factor. A logit of -infinity or NaN takes an expert out: its score
// is 0 and it is never chosen (nor is one whose bias is -infinity or NaN); a
// token with fewer than top_k experts left gets id -1 and weight 0 in the
// places that stay empty.
//
// Exactness of the choice. FP32 scores that differ by a few rounding errors
// may come out in either order, so a choice by scores is made in FP32 first
// and redone in FP64 (for that token alone) when two neighbours in the order,
// or the last group in and the first group out, are closer than the FP32
// error. Few tokens need it, so the choice costs FP32 and is the one the
// definition gives in FP64. The weights of a token with a chosen score below
// FP32's normal numbers are FP64's too. The FP64 parts are inlined and set the
// kernels' 46 to 64 registers; above 256 experts, 16 experts a lane, they spill
// (288 to 608 bytes of stores).
//
// One warp per token. Lane l holds experts l V .. l V + V - 1 (V = E / 32
// rounded up), so among equal scores the lowest lane, and in it the lowest
// register, is the lowest index. A round of the top-k is one warp-wide
// maximum of order-preserving integer keys and a ballot.
#include "route.h"

#include "gemm_tc.h"
#include "ptx.cuh"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

namespace i4g {
namespace route {

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kChunk = 128;       // tokens whose choices one bitmap holds
constexpr int kThreads = 1024;
constexpr int kOneBlock = 32;     // up to so many tokens one CTA does everything
// What two FP32 choice scores c <= 1 + |bias| can be off by against each other,
// relative to max(1, |c|). Sigmoid: p is off by p (1 - p) times exp's error
// (2 + 1.17 |x| units in the last place, at most 1e-7 so weighted), a
// reciprocal (1.2e-7) and the bias's addition (6e-8): 5e-7 for two. Softmax: a
// term's exp (3e-7 weighted by p), and the sum, of at most 16 additions in a
// lane and 5 across, whose error (21 x 6e-8) scales the difference of the two p.
constexpr float kSigmoidError = 1e-6f, kSoftmaxError = 2e-6f;

// Order-preserving keys: larger value, larger key; 0 is "not eligible".
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // -0 and 0 are equal
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double v) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
__device__ __forceinline__ double value_of(uint64_t k) {
  return __longlong_as_double(
      static_cast<long long>((k >> 63) ? (k ^ 0x8000000000000000ull) : ~k));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
  const uint32_t hi = static_cast<uint32_t>(k >> 32);
  const uint32_t top = __reduce_max_sync(kAll, hi);
  const uint32_t lo = __reduce_max_sync(kAll, hi == top ? static_cast<uint32_t>(k) : 0u);
  return (static_cast<uint64_t>(top) << 32) | lo;
}

// FP32: the choice's error bound allows for the fast forms; the weights are
// computed apart (weight_of).
__device__ __forceinline__ float exp_of(float x) { return __expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float reciprocal(float x) { return __fdividef(1.0f, x); }
__device__ __forceinline__ double reciprocal(double x) { return 1.0 / x; }
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}

template <typename F> struct Key;
template <> struct Key<float> { using type = uint32_t; };
template <> struct Key<double> { using type = uint64_t; };

// The scores p of this lane's experts (0 where not eligible); returns the
// softmax's sum of exp(x - top).
template <typename F, int V>
__device__ __forceinline__ F scores(const float (&x)[V], float top, int sigmoid, F (&p)[V]) {
  if (sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      p[v] = x[v] > -INFINITY ? reciprocal(F(1) + exp_of(-static_cast<F>(x[v]))) : F(0);
    return F(1);
  }
  F sum = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    // the largest logit's term is 1, an infinite one's too
    p[v] = x[v] > -INFINITY
               ? (x[v] == top ? F(1) : exp_of(static_cast<F>(x[v]) - static_cast<F>(top)))
               : F(0);
    sum += p[v];
  }
  sum = warp_sum(sum);
  const F r = sum > 0 ? F(1) / sum : F(0);
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] *= r;
  return sum;
}

// The score of a chosen expert, in full FP32 accuracy.
__device__ __forceinline__ float weight_of(float x, float top, int sigmoid, float sum) {
  if (sigmoid) return 1.0f / (1.0f + expf(-x));
  return (x == top ? 1.0f : expf(x - top)) / sum;
}
// The same in FP64, for scores near or below FP32's smallest normal number
// (e^-87.3), where the FP32 form has lost bits or is 0: a token whose chosen
// experts all lie there still has weights, divided by their sum.
constexpr float kSmallScore = -80.0f;  // of the logit, or of its distance to the largest
__device__ __forceinline__ bool small_score(float x, float top, int sigmoid) {
  return (sigmoid ? x : x - top) < kSmallScore;
}
__device__ __forceinline__ double small_weight_of(float x, float top, int sigmoid, float sum) {
  if (sigmoid) return 1.0 / (1.0 + exp(-static_cast<double>(x)));
  return (x == top ? 1.0 : exp(static_cast<double>(x) - top)) / sum;
}

// Lane's experts by falling key, the lower index first among equal keys:
// adjacent exchanges of strictly rising neighbours only, so ties keep their
// order. `order` holds the registers' first indices, four bits each.
template <int V>
using Order = std::conditional_t<(V <= 8), uint32_t, uint64_t>;

template <typename K, int V>
__device__ __forceinline__ Order<V> sort_keys(K (&key)[V]) {
  int at[V];
#pragma unroll
  for (int v = 0; v < V; ++v) at[v] = v;
#pragma unroll
  for (int pass = 0; pass < V; ++pass) {
#pragma unroll
    for (int v = pass & 1; v + 1 < V; v += 2) {
      const bool swap = key[v + 1] > key[v];
      const K k = swap ? key[v + 1] : key[v];
      key[v + 1] = swap ? key[v] : key[v + 1];
      key[v] = k;
      const int a = swap ? at[v + 1] : at[v];
      at[v + 1] = swap ? at[v] : at[v + 1];
      at[v] = a;
    }
  }
  Order<V> order = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) order |= static_cast<Order<V>>(at[v]) << (4 * v);
  return order;
}

// The choice of one token. On return lane i < top_k holds the i-th expert
// (or -1). Returns false when values closer than `tol` (relative to
// max(1, |value|)) decided it; tol = 0 accepts every order.
template <typename F, int V>
__device__ __forceinline__ bool choose(const Args& a, int lane, const float (&x)[V],
                                       const F (&p)[V], const float (&bias)[V], bool by_score,
                                       F tol, int& my_id) {
  using K = typename Key<F>::type;
  K key[V];
  const int e0 = lane * V;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const F c = by_score ? p[v] + static_cast<F>(bias[v]) : static_cast<F>(x[v]);
    key[v] = x[v] > -INFINITY && c > -INFINITY ? key_of(c) : K(0);
  }
  bool sure = true;
  if (a.n_group > 1) {
    const int size = a.E / a.n_group;
    const bool whole_lanes = a.E == 32 * V && 32 % a.n_group == 0;
    const int span = 32 / a.n_group;  // lanes of a group, if it is whole lanes
    F mine = -INFINITY;               // lane g: group g's score
    F largest = 0;                    // and the larger magnitude of its terms
    // the two terms of a sum may cancel, so its error goes by them
    const auto score_of = [&](K best, K second, F& size) {
      F score = best ? value_of(best) : -INFINITY;
      size = best ? fabs(score) : F(0);
      if (a.top2 && second) {
        const F next = value_of(second);
        size = fmax(size, fabs(next));
        score += next;
      }
      return score;
    };
    if (whole_lanes) {
      // the best two of a group's lanes meet in a few exchanges
      K best = 0, second = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        second = max(second, min(best, key[v]));
        best = max(best, key[v]);
      }
      for (int d = 1; d < span; d <<= 1) {
        const K ob = __shfl_xor_sync(kAll, best, d), os = __shfl_xor_sync(kAll, second, d);
        second = max(max(second, os), min(best, ob));
        best = max(best, ob);
      }
      F size_of;
      const F score = score_of(best, second, size_of);
      mine = __shfl_sync(kAll, score, (lane * span) & 31);
      if (tol > 0) largest = __shfl_sync(kAll, size_of, (lane * span) & 31);
    } else {
      // a group may start and end inside a lane: a pass over the warp for each
      for (int g = 0; g < a.n_group; ++g) {
        K best = 0, second = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int e = e0 + v;
          const K k = e >= g * size && e < (g + 1) * size ? key[v] : K(0);
          second = max(second, min(best, k));
          best = max(best, k);
        }
        const K top = warp_max(best);
        K next = 0;
        if (a.top2) {
          const unsigned holders = __ballot_sync(kAll, best == top);
          next = warp_max(lane == __ffs(holders) - 1 ? second : best);
        }
        F size_of;
        const F score = score_of(top, next, size_of);
        if (lane == g) {
          mine = score;
          largest = size_of;
        }
      }
    }
    int rank = 0;
    for (int g = 0; g < a.n_group; ++g) {
      const F other = __shfl_sync(kAll, mine, g);
      rank += other > mine || (other == mine && g < lane);
    }
    const bool kept = lane < a.n_group && rank < a.topk_group;
    const unsigned in = __ballot_sync(kAll, kept);
    if (tol > 0 && by_score && a.topk_group < a.n_group) {
      // what each group's score can be: the least of those in against the most
      // of those out (an infinite one is left to FP64; largest 0: no members)
      const F error = tol * fmax(F(1), largest);
      const bool finite = error < INFINITY && (fabs(mine) < INFINITY || largest == 0);
      const F least = kept ? (finite ? mine - error : -INFINITY) : INFINITY;
      const F most =
          lane < a.n_group && !kept ? (finite ? mine + error : INFINITY) : -INFINITY;
      const K lowest_in = ~warp_max(~key_of(least)), highest_out = warp_max(key_of(most));
      sure = lowest_in > highest_out || highest_out == key_of(F(-INFINITY));
    }
    int g = whole_lanes ? lane / span : e0 / size;
    int next = whole_lanes ? a.E : (g + 1) * size;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (e0 + v >= next) {
        ++g;
        next += size;
      }
      if (!((in >> (g & 31)) & 1)) key[v] = 0;
    }
  }
  Order<V> order = sort_keys(key);
  my_id = -1;
  K my_key = 0, past = 0;  // lane i: the i-th key chosen; the first one not chosen
  const int rounds = a.top_k + (tol > 0 && by_score ? 1 : 0);
  for (int i = 0; i < rounds; ++i) {
    const K top = warp_max(key[0]);
    if (top == 0) break;  // none left
    if (i == a.top_k) {
      past = top;
      break;
    }
    const int winner = __ffs(__ballot_sync(kAll, key[0] == top)) - 1;
    const int id = __shfl_sync(kAll, e0 + static_cast<int>(order & 15), winner);
    if (lane == i) {
      my_id = id;
      my_key = top;
    }
    if (lane == winner) {
#pragma unroll
      for (int v = 0; v + 1 < V; ++v) key[v] = key[v + 1];
      key[V - 1] = 0;
      order >>= 4;
    }
  }
  if (tol > 0 && by_score) {
    K next = __shfl_down_sync(kAll, my_key, 1);
    if (lane == a.top_k - 1 || lane == 31) next = past;
    bool close = false;
    if (my_key && next) {
      const F hi = value_of(my_key), lo = value_of(next);
      close = !(hi - lo > tol * fmax(F(1), fabs(hi)));
    }
    sure = sure && !__any_sync(kAll, close);
  }
  return sure;
}

// This lane's entries of a row of E (logits or bias); `none` past the last.
template <int V, typename T>
__device__ __forceinline__ void load_lane(const T* row, int E, int lane, float none,
                                          float (&x)[V]) {
  const int e0 = lane * V;
  if constexpr (V % 4 == 0 && sizeof(T) == 4) {
    if (E == 32 * V && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        const float4 f = reinterpret_cast<const float4*>(row + e0)[q];
        x[4 * q] = f.x;
        x[4 * q + 1] = f.y;
        x[4 * q + 2] = f.z;
        x[4 * q + 3] = f.w;
      }
      return;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = e0 + v < E ? static_cast<float>(row[e0 + v]) : none;
}

template <bool FP32>
__device__ __forceinline__ auto logits_of(const Args& a, int t) {
  using T = std::conditional_t<FP32, float, __half>;
  return static_cast<const T*>(a.logits) + static_cast<size_t>(t) * a.ld;
}

// Token t's experts and weights from this lane's logits x, by one warp; lane i < top_k returns expert i.
template <int V, bool FP32>
__device__ __forceinline__ int route_token(const Args& a, int t, int lane,
                                           const float (&bias)[V], const float (&x)[V]) {
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) top = x[v] > top ? x[v] : top;
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, d));
  float p[V];
  const float sum = scores(x, top, a.sigmoid, p);
  const bool by_score = a.bias || (a.n_group > 1 && a.top2);
  int id;
  if (!choose(a, lane, x, p, bias, by_score, a.sigmoid ? kSigmoidError : kSoftmaxError,
              id)) {
    double pd[V];
    scores(x, top, a.sigmoid, pd);
    choose(a, lane, x, pd, bias, by_score, 0.0, id);
  }
  float xi = 0.0f, w = 0.0f;  // lane i: expert id's logit and score
  if (id >= 0) {
    xi = static_cast<float>(logits_of<FP32>(a, t)[id]);
    w = weight_of(xi, top, a.sigmoid, sum);
  }
  if (__any_sync(kAll, id >= 0 && small_score(xi, top, a.sigmoid))) {
    double wd = id >= 0 ? small_weight_of(xi, top, a.sigmoid, sum) : 0.0;
    if (a.renormalize) {
      const double all = warp_sum(wd);
      wd = all > 0.0 ? wd / all : 0.0;
    }
    w = static_cast<float>(wd);
  } else if (a.renormalize) {
    const float all = warp_sum(w);
    w = all > 0.0f ? w / all : 0.0f;
  }
  if (lane < a.top_k) {
    const size_t at = static_cast<size_t>(t) * a.top_k + lane;
    a.ids[at] = id;
    a.weights[at] = w * a.scale;
  }
  return id;
}

// Tokens of block b of nb: [b T / nb, (b + 1) T / nb).
__device__ __forceinline__ int first_token(int T, int b, int nb) {
  return static_cast<int>(static_cast<long long>(b) * T / nb);
}

// A CTA's shared tables while it places pairs.
struct Place {
  int base[kMaxExperts];                      // next row of each expert
  alignas(16) uint32_t bits[kMaxExperts][kChunk / 32];  // tokens of the chunk that chose it
  int warp_total[32];
};

// Exclusive sum of v over the threads of the CTA (v = 0 past E); also the total.
__device__ __forceinline__ int block_scan(int v, int* warp_total, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(kAll, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31) warp_total[warp] = sum;
  __syncthreads();
  int mine = lane < static_cast<int>(blockDim.x) / 32 ? warp_total[lane] : 0;
  total = __reduce_add_sync(kAll, mine);
  const int before = __reduce_add_sync(kAll, lane < warp ? mine : 0);
  return before + sum - v;
}

// Gives the pairs of tokens [t0, t1) their rows: an expert's next row is
// base[e]; inside a chunk of kChunk tokens a pair's place is the number of
// earlier tokens that chose the same expert, counted in the expert's bitmap
// (a token chooses an expert once), so the order is by token and nothing
// depends on which thread comes first.
__device__ __forceinline__ void place_pairs(const Args& a, Place& s, int t0, int t1) {
  constexpr int kMost = kChunk * kMaxTopK / kThreads;  // pairs of a chunk per thread
  for (int c0 = t0; c0 < t1; c0 += kChunk) {
    const int pairs = min(kChunk, t1 - c0) * a.top_k;
    const size_t p0 = static_cast<size_t>(c0) * a.top_k;
    int e[kMost], t[kMost];
#pragma unroll
    for (int q = 0; q < kMost; ++q) {
      const int i = threadIdx.x + q * kThreads;
      e[q] = i < pairs ? a.ids[p0 + i] : -1;
      t[q] = i / a.top_k;
    }
    for (int i = threadIdx.x; i < a.E * (kChunk / 32); i += kThreads) (&s.bits[0][0])[i] = 0u;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kMost; ++q)
      if (e[q] >= 0) atomicOr(&s.bits[e[q]][t[q] >> 5], 1u << (t[q] & 31));
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kMost; ++q) {
      const int i = threadIdx.x + q * kThreads;
      if (i >= pairs) break;
      int row = -1;
      if (e[q] >= 0) {
        const uint4 b = *reinterpret_cast<const uint4*>(s.bits[e[q]]);
        const uint32_t word[4] = {b.x, b.y, b.z, b.w};
        const uint32_t below = (1u << (t[q] & 31)) - 1u;
        row = s.base[e[q]];
#pragma unroll
        for (int w = 0; w < 4; ++w)
          row += __popc(word[w] & (w < (t[q] >> 5) ? ~0u : (w == (t[q] >> 5) ? below : 0u)));
        a.rows[row] = static_cast<int>(p0) + i;
      }
      a.slots[p0 + i] = row;
    }
    if (c0 + kChunk >= t1) break;
    __syncthreads();
    for (int x = threadIdx.x; x < a.E; x += kThreads) {
      int count = 0;
#pragma unroll
      for (int q = 0; q < kChunk / 32; ++q) count += __popc(s.bits[x][q]);
      s.base[x] += count;
    }
    __syncthreads();
  }
}

// Everything in one CTA (T <= kOneBlock).
template <int V, bool FP32>
__global__ void __launch_bounds__(kThreads, 1) route_small_kernel(const Args a) {
  __shared__ Place s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < kMaxExperts; e += blockDim.x) s.base[e] = 0;
  grid_dependency_wait();
  if (threadIdx.x == 0) launch_dependents();
  __syncthreads();
  float bias[V] = {};
  if (a.bias) load_lane(a.bias, a.E, lane, 0.0f, bias);
  for (int t = warp; t < a.T; t += blockDim.x / 32) {
    float x[V];
    load_lane(logits_of<FP32>(a, t), a.E, lane, -INFINITY, x);
    const int e = route_token<V, FP32>(a, t, lane, bias, x);
    if (lane < a.top_k && e >= 0) atomicAdd(&s.base[e], 1);
  }
  __syncthreads();
  const int e = threadIdx.x;
  int total;
  const int before = block_scan(e < a.E ? s.base[e] : 0, s.warp_total, total);
  __syncthreads();
  if (e < a.E) {
    s.base[e] = before;
    a.offsets[e] = before;
  }
  if (e == 0) a.offsets[a.E] = total;
  __syncthreads();  // also orders the ids just written before they are read
  place_pairs(a, s, 0, a.T);
  for (int i = total + threadIdx.x; i < a.T * a.top_k; i += blockDim.x) a.rows[i] = -1;
}

// First of two kernels: choices, and how many of the block's pairs each
// expert got (counts [block][E rounded up to even], 16 bits each: a block has
// fewer tokens than that).
template <int V, bool FP32>
__global__ void __launch_bounds__(kThreads, 1)
    route_choose_kernel(const Args a, uint16_t* __restrict__ counts) {
  __shared__ int count[kMaxExperts];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < kMaxExperts; e += blockDim.x) count[e] = 0;
  grid_dependency_wait();
  if (threadIdx.x == 0) launch_dependents();
  __syncthreads();
  const int t0 = first_token(a.T, blockIdx.x, gridDim.x);
  const int t1 = first_token(a.T, blockIdx.x + 1, gridDim.x);
  float bias[V] = {};
  if (a.bias) load_lane(a.bias, a.E, lane, 0.0f, bias);
  float next[V];
  if (t0 + warp < t1) load_lane(logits_of<FP32>(a, t0 + warp), a.E, lane, -INFINITY, next);
  for (int t = t0 + warp; t < t1; t += kThreads / 32) {
    float x[V];
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = next[v];
    // the next token's logits arrive while this one's are sorted
    if (t + kThreads / 32 < t1)
      load_lane(logits_of<FP32>(a, t + kThreads / 32), a.E, lane, -INFINITY, next);
    const int e = route_token<V, FP32>(a, t, lane, bias, x);
    if (lane < a.top_k && e >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  const int width = (a.E + 1) & ~1;
  for (int e = threadIdx.x; e < width; e += blockDim.x)
    counts[static_cast<size_t>(blockIdx.x) * width + e] = static_cast<uint16_t>(count[e]);
}

// Second kernel: every block adds the counts up itself (all of them for the
// experts' offsets, those of earlier blocks for its own first rows), then
// places its tokens' pairs. The counts are a few tens of KB in L2.
__global__ void __launch_bounds__(kThreads, 1)
    route_place_kernel(const Args a, const uint16_t* __restrict__ counts) {
  __shared__ Place s;
  __shared__ int all[kMaxExperts];
  for (int e = threadIdx.x; e < kMaxExperts; e += blockDim.x) s.base[e] = all[e] = 0;
  grid_dependency_wait();
  if (threadIdx.x == 0) launch_dependents();
  __syncthreads();
  const int nb = gridDim.x, b = blockIdx.x;
  // two experts a thread, all its loads in flight together
  const int pairs_of = (a.E + 1) / 2;
  const int parts = static_cast<int>(blockDim.x) / pairs_of;
  const int e2 = threadIdx.x % pairs_of, part = threadIdx.x / pairs_of;
  if (part < parts) {
    const uint32_t* col = reinterpret_cast<const uint32_t*>(counts) + e2;
    int before0 = 0, before1 = 0, sum0 = 0, sum1 = 0;
#pragma unroll 20
    for (int i = part; i < nb; i += parts) {
      const uint32_t c = col[static_cast<size_t>(i) * pairs_of];
      const int c0 = static_cast<int>(c & 0xffffu), c1 = static_cast<int>(c >> 16);
      sum0 += c0;
      sum1 += c1;
      before0 += i < b ? c0 : 0;
      before1 += i < b ? c1 : 0;
    }
    // integers: the order of the additions does not matter
    atomicAdd(&all[2 * e2], sum0);
    atomicAdd(&s.base[2 * e2], before0);
    if (2 * e2 + 1 < a.E) {
      atomicAdd(&all[2 * e2 + 1], sum1);
      atomicAdd(&s.base[2 * e2 + 1], before1);
    }
  }
  __syncthreads();
  int total;
  const int mine = threadIdx.x;
  const int first = block_scan(mine < a.E ? all[mine] : 0, s.warp_total, total);
  if (mine < a.E) {
    s.base[mine] += first;
    if (b == 0) a.offsets[mine] = first;
  }
  if (b == 0 && mine == 0) a.offsets[a.E] = total;
  __syncthreads();
  place_pairs(a, s, first_token(a.T, b, nb), first_token(a.T, b + 1, nb));
  const size_t pairs = static_cast<size_t>(a.T) * a.top_k;
  for (size_t i = total + static_cast<size_t>(b) * blockDim.x + threadIdx.x; i < pairs;
       i += static_cast<size_t>(nb) * blockDim.x)
    a.rows[i] = -1;
}

int blocks_for(int T, int sm_count) {
  // one block per SM; more only so that a block's counts fit 16 bits
  const int most = std::max(sm_count, (T + 32767) / 32768);
  return std::min(most, (T + 31) / 32);
}

template <typename... KArgs, typename... AArgs>
cudaError_t launch_dependent(void (*kernel)(KArgs...), int grid, int threads, cudaStream_t stream,
                             AArgs... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int V, bool FP32>
cudaError_t launch_typed(const Args& a, int sm_count, void* workspace, cudaStream_t stream) {
  if (a.T <= kOneBlock)
    return launch_dependent(route_small_kernel<V, FP32>, 1, kThreads, stream, a);
  uint16_t* counts = static_cast<uint16_t*>(workspace);
  const int nb = blocks_for(a.T, sm_count);
  cudaError_t e = launch_dependent(route_choose_kernel<V, FP32>, nb, kThreads, stream, a, counts);
  if (e != cudaSuccess) return e;
  return launch_dependent(route_place_kernel, nb, kThreads, stream, a,
                          static_cast<const uint16_t*>(counts));
}

// out[t] = residual[t] + sum_s w[t, s] y[slots[t, s]]: a thread does eight
// columns of one token in FP32, in slot order, with the rows' loads issued
// together. Bound by the bytes of y.
constexpr int kCombineThreads = 128;

__global__ void __launch_bounds__(kCombineThreads)
    combine_kernel(const __half* __restrict__ y, int y_rows, const int* __restrict__ slots,
                   const float* __restrict__ weights, const __half* residual, __half* out,
                   int top_k, int N) {
  grid_dependency_wait();
  if (threadIdx.x == 0) launch_dependents();
  const int col = (blockIdx.y * kCombineThreads + threadIdx.x) * 8;
  const size_t t = blockIdx.x;
  if (col >= N) return;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  constexpr int BATCH = 8;
  for (int s0 = 0; s0 < top_k; s0 += BATCH) {
    uint4 v[BATCH];
    float w[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int slot = s0 + b < top_k ? slots[t * top_k + s0 + b] : -1;
      const bool has = static_cast<unsigned>(slot) < static_cast<unsigned>(y_rows);
      w[b] = has ? weights[t * top_k + s0 + b] : 0.0f;
      v[b] = has ? *reinterpret_cast<const uint4*>(y + static_cast<size_t>(slot) * N + col)
                 : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const uint32_t q[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(u32_as_half2(q[i]));
        acc[2 * i] = fmaf(w[b], f.x, acc[2 * i]);
        acc[2 * i + 1] = fmaf(w[b], f.y, acc[2 * i + 1]);
      }
    }
  }
  if (residual) {
    const uint4 r = *reinterpret_cast<const uint4*>(residual + t * N + col);
    const uint32_t q[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(u32_as_half2(q[i]));
      acc[2 * i] += f.x;
      acc[2 * i + 1] += f.y;
    }
  }
  uint4 o;
  o.x = half2_as_u32(__floats2half2_rn(acc[0], acc[1]));
  o.y = half2_as_u32(__floats2half2_rn(acc[2], acc[3]));
  o.z = half2_as_u32(__floats2half2_rn(acc[4], acc[5]));
  o.w = half2_as_u32(__floats2half2_rn(acc[6], acc[7]));
  *reinterpret_cast<uint4*>(out + t * N + col) = o;
}

}  // namespace

size_t workspace_bytes(int T, int E, int sm_count) {
  if (T <= kOneBlock) return 0;
  return static_cast<size_t>(blocks_for(T, sm_count)) * ((E + 1) & ~1) * sizeof(uint16_t);
}

cudaError_t launch(const Args& a, bool fp32_logits, int sm_count, void* workspace,
                   cudaStream_t stream) {
  const int v = (a.E + 31) / 32;
#define I4G_ROUTE_CASE(V)                                                          \
  if (v <= V)                                                                      \
    return fp32_logits ? launch_typed<V, true>(a, sm_count, workspace, stream)     \
                       : launch_typed<V, false>(a, sm_count, workspace, stream);
  I4G_ROUTE_CASE(1)
  I4G_ROUTE_CASE(2)
  I4G_ROUTE_CASE(4)
  I4G_ROUTE_CASE(8)
  I4G_ROUTE_CASE(16)
#undef I4G_ROUTE_CASE
  return cudaErrorInvalidValue;
}

cudaError_t combine(const __half* y, int y_rows, const int* slots, const float* weights,
                    const __half* residual, __half* out, int T, int top_k, int N,
                    cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(T, (N / 8 + kCombineThreads - 1) / kCombineThreads);
  cfg.blockDim = dim3(kCombineThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, combine_kernel, y, y_rows, slots, weights, residual, out, top_k,
                            N);
}

}  // namespace route
}  // namespace i4g
