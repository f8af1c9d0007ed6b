// Routing of tokens to experts, and the plan that groups the (token, expert) pairs by expert.
//
// Routing, per token: scores s = sigmoid(logit) or softmax(logits); values v = s + bias; the groups with the largest
// sum of two values (or largest value) stay; the top_k largest v of those are chosen, ties to the lowest index; weights are
// the scores without bias, normalised over the chosen ones where asked.  An expert whose logit is -inf or NaN, or whose bias is
// -inf or NaN, is never chosen.  +inf counts as the largest finite number, -0 as 0.
//
// One warp per token, a run of experts per lane.  Which experts come first is decided on fp32 scores wherever these lie further apart than
// they can be off, and in 64 bits in the rows where some do not (without a bias the logits themselves order the experts: exactly).
// 65536 tokens, 256 experts in 8 groups with a bias: 84 us (0.80 TB/s of logits), 192 with every row in 64 bits.
#include <math_constants.h>

#include "common.cuh"
#include "profile.cuh"

namespace mq {
namespace {

constexpr int ROUTE_WARPS = 8, EXTRA = 4, MAX_EXPERTS = 1024;
constexpr size_t SMEM_AS_IS = 47 * 1024;   // of the 48 KB that need no permission, beside what a kernel has of its own

struct RouteParams {
  int64_t T, ld;
  int E, k, groups, keep, group_size;
  bool sigmoid, top2, renormalise;
  float scale;
  const float* bias;
  int32_t* ids;
  float* weights;
  bool vec;               // rows of logits can be read 16 bytes at a time
  int lanes_per_group;    // lanes that hold a group, 0 where lanes and groups do not match
  int lanes_to_search;    // as many as there are to a group, a power of two of them
};

// NaN is -inf, +inf the largest number, -0 is +0 (the sum): keys order bits, and zeros of either sign have the same score
__device__ __forceinline__ float finite_logit(float l) { return fminf(fmaxf(l, -CUDART_INF_F), 3.402823466e38f) + 0.0f; }

template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename F>
__device__ __forceinline__ F warp_max(F v) {
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ uint64_t ordered64(double v) {
  const int64_t b = __double_as_longlong(v);
  return (uint64_t)(b ^ ((b >> 63) | (int64_t)0x8000000000000000ull));
}

// The choice in 64 bits, for one token.  `row` holds its logits (finite_logit), `value` is scratch of E doubles, both of this warp.
// Lane j < k gets the j-th expert, or -1.  Out of line: few tokens come here.
template <int VPL>
__device__ __noinline__ int choose(const RouteParams& p, const float* row, double* value, int lane) {
  const bool by_logit = p.bias == nullptr;   // sigmoid and softmax are increasing
  const bool by_score = !by_logit || (p.groups > 1 && p.top2);
  const int e0 = lane * VPL;
  double v[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) v[j] = e0 + j < p.E ? (double)row[e0 + j] : -CUDART_INF;
  if (by_score) {
    double top = 0.0, total = 1.0;
    if (!p.sigmoid) {
      top = v[0];
#pragma unroll
      for (int j = 1; j < VPL; ++j) top = max(top, v[j]);
      top = warp_max(top);
      total = 0.0;
#pragma unroll 1
      for (int j = 0; j < VPL; ++j) total += e0 + j < p.E && row[e0 + j] > -CUDART_INF_F ? exp((double)row[e0 + j] - top) : 0.0;
      total = warp_sum(total);
    }
#pragma unroll 4
    for (int j = 0; j < VPL; ++j) {
      const double e = exp(p.sigmoid ? -v[j] : v[j] - top);
      double s = p.sigmoid ? 1.0 / (1.0 + e) : e / total;
      if (!by_logit && e0 + j < p.E) s += (double)p.bias[e0 + j];
      v[j] = v[j] > -CUDART_INF && s == s ? s : -CUDART_INF;
    }
  }
  if (p.groups > 1) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (e0 + j < p.E) value[e0 + j] = v[j];
    __syncwarp();
    const int share = p.lanes_to_search;
    const int group = lane / share;
    double a = -CUDART_INF, b = -CUDART_INF;
    if (group < p.groups)
      for (int i = lane % share; i < p.group_size; i += share) {
        const double u = value[group * p.group_size + i];
        b = max(b, min(a, u));
        a = max(a, u);
      }
    for (int o = 1; o < share; o <<= 1) {
      const double a2 = __shfl_xor_sync(0xffffffffu, a, o), b2 = __shfl_xor_sync(0xffffffffu, b, o);
      b = max(min(a, a2), max(b, b2));
      a = max(a, a2);
    }
    const double mine = p.top2 && b > -CUDART_INF ? a + b : a;
    int better = 0;
    for (int g = 0; g < p.groups; ++g) {
      const double u = __shfl_sync(0xffffffffu, mine, g * share);
      better += u > mine || (u == mine && g < group);
    }
    const unsigned lanes = __ballot_sync(0xffffffffu, group < p.groups && better < p.keep);
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      if (e0 + j >= p.E) continue;
      if (!(lanes >> ((e0 + j) / p.group_size * share) & 1u)) v[j] = -CUDART_INF;
      else if (by_logit) v[j] = row[e0 + j];
    }
  }
  uint64_t key[VPL], largest = 0;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    key[j] = v[j] > -CUDART_INF ? ordered64(v[j]) : 0ull;
    largest = max(largest, key[j]);
  }
  int mine = -1;
  for (int r = 0; r < p.k; ++r) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(largest >> 32));
    const bool with_high = (uint32_t)(largest >> 32) == high;
    const uint32_t low = __reduce_max_sync(0xffffffffu, with_high ? (uint32_t)largest : 0u);
    if ((high | low) == 0) break;
    const int from = __ffs(__ballot_sync(0xffffffffu, with_high && (uint32_t)largest == low)) - 1;
    int j_of = 0;
    if (lane == from) {
      const uint64_t taken = largest;
      bool done = false;
      largest = 0;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        if (!done && key[j] == taken) {
          done = true;
          j_of = j;
          key[j] = 0;
        }
        largest = max(largest, key[j]);
      }
    }
    j_of = __shfl_sync(0xffffffffu, j_of, from);
    if (lane == r) mine = from * VPL + j_of;
  }
  return mine;
}

// Without a bias: whether a group whose two largest logits are a and b stays, by 64-bit sums of their scores (softmax without its common
// factor).  Groups are first_of lanes each.  16-bit logits come here often, since different groups have the same two: 28375 tokens of 332
// experts in 4 groups 93 us with all of the token's values formed anew.
__device__ __noinline__ bool stays_by_logits(const RouteParams& p, float a, float b, float top, int group, int first_of) {
  double sum = -CUDART_INF;
  if (a > -CUDART_INF_F) {
    sum = p.sigmoid ? 1.0 / (1.0 + exp(-(double)a)) : exp((double)a - top);
    if (b > -CUDART_INF_F) sum += p.sigmoid ? 1.0 / (1.0 + exp(-(double)b)) : exp((double)b - top);
  }
  int better = 0;
  for (int g = 0; g < p.groups; ++g) {
    const double u = __shfl_sync(0xffffffffu, sum, g * first_of);
    better += u > sum || (u == sum && g < group);
  }
  return better < p.keep;
}

// fp32 numbers as unsigned integers of the same order; 0 stands for an expert that cannot be chosen
__device__ __forceinline__ uint32_t ordered(float v) {
  const int b = __float_as_int(v);
  return (uint32_t)(b ^ ((b >> 31) | (int)0x80000000));
}
__device__ __forceinline__ float from_ordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// Scores for the choice: exponential and reciprocal as the hardware has them.
__device__ __forceinline__ float quick_exp(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.44269504f));
  return y;
}
__device__ __forceinline__ float quick_sigmoid(float l) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + quick_exp(-l)));
  return y;
}

// How far a value may be off.  quick_sigmoid by 4e-7 at most (the exponential by 2^-22 and by 9e-8 |l|, times s (1 - s); sum and reciprocal by
// 2^-23 each), a softmax score by 3.3e-6 of 1 / total, which no score exceeds (its sum over up to 1024 experts, 32 in a lane and five levels of
// lanes, and the exponentials; 3.3e-6 for all sizes of `total` left 27 us where 636 tokens of 260 experts with a bias take 14); the sum
// with the bias adds 2^-24 |v|.  So of two values the larger is certain where they are apart by 8e-7 (6.6e-6 / total) + 1.2e-7 |v|, and by
// 2^-23 VPL |v| more where low bits have given way to an index; of two sums of two values by 1.6e-6 (1.33e-5 / total) + 2.4e-7 of what was summed.
// (`total` is 1 for sigmoid.)
struct Margin {
  float fixed, per_size;
  __device__ __forceinline__ bool certain(float a, float b, float total, float size) const { return a - b > __fdividef(fixed, total) + per_size * size; }   // no for NaN
};

// Descending, by a network of compare-exchanges (odd-even merges of runs of P).  Steps by recursion: as loops, those of 16 and more keys are not
// unrolled as a whole, and keys that are indexed at run time live in memory (20000 tokens, 400 experts: 50 us instead of 37).
template <int N, int P = 1, int Q = P>
__device__ __forceinline__ void sort_descending(uint32_t (&k)[N]) {
  if constexpr (P < N) {
#pragma unroll
    for (int j = Q % P; j + Q < N; ++j)
      if ((j - Q % P) % (2 * Q) < Q && j / (2 * P) == (j + Q) / (2 * P)) {
        const uint32_t a = k[j], b = k[j + Q];
        k[j] = max(a, b);
        k[j + Q] = min(a, b);
      }
    if constexpr (Q > 1) sort_descending<N, P, Q / 2>(k);
    else sort_descending<N, 2 * P>(k);
  }
}

// VPL experts per lane: VPL lane .. VPL lane + VPL - 1.  A warp's next token's logits are on their way while it chooses.  Instructions
// bound it: 1085 a token at 256 experts, 8 groups and a choice of 8 (76 % of the issue slots; memory at 10 %).
constexpr int route_blocks(int vpl) { return vpl <= 4 ? 5 : vpl <= 8 ? 4 : vpl <= 16 ? 3 : 2; }   // per SM

template <int DT, int VPL>
__global__ void __launch_bounds__(ROUTE_WARPS * 32, route_blocks(VPL)) route_kernel(const void* __restrict__ logits, const __grid_constant__ RouteParams p) {
  using T = typename StorageOf<DT>::type;
  constexpr int WORD = VPL * sizeof(T) >= 16 ? 16 / sizeof(T) : 1;     // values per load
  struct alignas(WORD * sizeof(T)) Word { T v[WORD]; };
  extern __shared__ double route_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double* value = route_smem + (size_t)warp * p.E;
  float* row = reinterpret_cast<float*>(route_smem + (size_t)ROUTE_WARPS * p.E) + (size_t)warp * p.E;
  const int e0 = lane * VPL;
  const bool by_logit = p.bias == nullptr;   // sigmoid and softmax are increasing
  const bool by_sum = p.groups > 1 && p.top2;
  const bool by_score = !by_logit || by_sum;
  const Margin of_values = {p.sigmoid ? 1e-6f : 7e-6f, 1.4e-7f + 1.3e-7f * VPL}, of_sums = {p.sigmoid ? 2e-6f : 1.4e-5f, 3e-7f};
  // a block's tokens go to whichever of its warps is free: one that is in doubt about a token takes several times as long
  const int64_t begin = p.T / gridDim.x * blockIdx.x + min((int64_t)blockIdx.x, p.T % gridDim.x);
  const int64_t end = begin + p.T / gridDim.x + (blockIdx.x < p.T % gridDim.x);
  __shared__ int handed_out;
  if (threadIdx.x == 0) handed_out = ROUTE_WARPS;
  __syncthreads();
  chain_wait();
  chain_release();

  Word raw[VPL / WORD];      // experts behind the last one keep -inf
#pragma unroll
  for (int j = 0; j < VPL; ++j) raw[j / WORD].v[j % WORD] = from_float<T>(-CUDART_INF_F);
  auto load = [&](int64_t t) {
    const T* src = static_cast<const T*>(logits) + t * p.ld + e0;
#pragma unroll
    for (int j = 0; j < VPL / WORD; ++j) {
      if (WORD == 1 || p.vec) {     // (then E is a multiple of WORD)
        if (e0 + j * WORD < p.E) raw[j] = *reinterpret_cast<const Word*>(src + j * WORD);
      } else {
#pragma unroll
        for (int i = 0; i < WORD; ++i)
          if (e0 + j * WORD + i < p.E) raw[j].v[i] = src[j * WORD + i];
      }
    }
  };
  float bias[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) bias[j] = by_logit || e0 + j >= p.E ? 0.0f : fmaxf(p.bias[e0 + j], -CUDART_INF_F);   // NaN is -inf

  int64_t t = begin + warp, t_next = 0;
  if (t < end) load(t);
  for (; t < end; t = t_next) {
    int number = 0;
    if (lane == 0) number = atomicAdd(&handed_out, 1);
    t_next = begin + __shfl_sync(0xffffffffu, number, 0);
    float l[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) l[j] = finite_logit(to_float(raw[j / WORD].v[j % WORD]));
    if (t_next < end) load(t_next);

    // softmax: its largest logit and sum, where scores are needed
    float top = 0.0f, total = 1.0f;
    if (!p.sigmoid && (by_score || !p.renormalise)) {
      top = l[0];
#pragma unroll
      for (int j = 1; j < VPL; ++j) top = fmaxf(top, l[j]);
      top = warp_max(top);
      total = 0.0f;
#pragma unroll
      for (int j = 0; j < VPL; ++j) total += l[j] > -CUDART_INF_F ? expf(l[j] - top) : 0.0f;
      total = warp_sum(total);
    }
    // v: what experts are compared by, the score with its bias or the logit
    float v[VPL];
    auto score = [&](float logit, float inv) { return p.sigmoid ? quick_sigmoid(logit) : quick_exp(logit - top) * inv; };
    if (by_logit) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) v[j] = l[j];
    } else {
      const float inv = __fdividef(1.0f, total);
#pragma unroll
      for (int j = 0; j < VPL; ++j) v[j] = l[j] > -CUDART_INF_F ? score(l[j], inv) + bias[j] : -CUDART_INF_F;
    }
    bool near = false;
    bool whole_lane = true;           // groups keep or drop all of a lane's experts
    unsigned kept = 0xffffffffu;      // bit per lane, or per group
    if (p.groups > 1) {
      float a = -CUDART_INF_F, b = -CUDART_INF_F;     // the two largest of group `group`
      int group, first_of = 1;                        // group g is held by lane g * first_of
      if (p.lanes_per_group) {                        // whole lanes, 2^n of them, to a group
        first_of = p.lanes_per_group;
        group = lane / first_of;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
          b = fmaxf(b, fminf(a, v[j]));
          a = fmaxf(a, v[j]);
        }
      } else {
        first_of = p.lanes_to_search;
        group = lane / first_of;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
          if (e0 + j < p.E) row[e0 + j] = v[j];
        __syncwarp();
        if (group < p.groups) {
          const float* of_group = row + group * p.group_size;
#pragma unroll 4
          for (int i = lane % first_of; i < p.group_size; i += first_of) {
            const float u = of_group[i];
            b = fmaxf(b, fminf(a, u));
            a = fmaxf(a, u);
          }
        }
        __syncwarp();
      }
      for (int o = 1; o < first_of; o <<= 1) {
        const float a2 = __shfl_xor_sync(0xffffffffu, a, o), b2 = __shfl_xor_sync(0xffffffffu, b, o);
        b = fmaxf(fminf(a, a2), fmaxf(b, b2));
        a = fmaxf(a, a2);
      }
      float va = a, vb = b;
      if (by_logit && by_sum) {      // the largest logits have the largest scores
        const float inv = __fdividef(1.0f, total);
        if (a > -CUDART_INF_F) va = score(a, inv);
        if (b > -CUDART_INF_F) vb = score(b, inv);
      }
      const float mine = by_sum && vb > -CUDART_INF_F ? va + vb : va;
      int better = 0;
#pragma unroll 4
      for (int g = 0; g < p.groups; ++g) {
        const float u = __shfl_sync(0xffffffffu, mine, g * first_of);
        better += u > mine || (u == mine && g < group);
      }
      const bool real = group < p.groups, stays = real && better < p.keep;
      whole_lane = p.lanes_per_group != 0;
      kept = __ballot_sync(0xffffffffu, stays);
      if (by_score) {
        const float least = from_ordered(__reduce_min_sync(0xffffffffu, stays ? ordered(mine) : 0xffffffffu));
        const float most = from_ordered(__reduce_max_sync(0xffffffffu, real && !stays ? ordered(mine) : ordered(-CUDART_INF_F)));
        const float size = real && mine > -CUDART_INF_F ? fabsf(va) + (vb > -CUDART_INF_F ? fabsf(vb) : 0.0f) : 0.0f;
        near = most > -CUDART_INF_F && !of_sums.certain(least, most, total, __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(size))));
        if (near && by_logit) {
          const bool stays64 = stays_by_logits(p, a, b, top, group, first_of);     // (all lanes: it shuffles)
          kept = __ballot_sync(0xffffffffu, real && stays64);
          near = false;
        }
      }
    }
    // Keys: the number, its lowest bits replaced by which of the lane's experts it is, the first one highest.  Sorted, so that a lane offers its
    // largest and moves up once it is taken.
    constexpr uint32_t WHICH = VPL - 1;
    uint32_t key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      key[j] = v[j] > -CUDART_INF_F ? (ordered(v[j]) & ~WHICH) | (WHICH - (uint32_t)j) : 0u;
    }
    if (whole_lane) {
      if (!(kept >> lane & 1u))
#pragma unroll
        for (int j = 0; j < VPL; ++j) key[j] = 0;
    } else {
      int group = e0 / p.group_size, left = (group + 1) * p.group_size - e0;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        if (left == 0) {
          ++group;
          left = p.group_size;
        }
        --left;
        if (!(kept >> (group * p.lanes_to_search & 31) & 1u)) key[j] = 0;
      }
    }
    sort_descending(key);
    // The k largest, one by one, and where numbers may have lost what sets them apart the one behind them.  (The low bits of 16-bit logits
    // are empty.)  Lane r keeps the r-th.
    const bool exact = by_logit && sizeof(T) == 2;
    uint32_t my_key = 0, last = 0;     // `last`: of the last round
    int mine = -1;
    auto take = [&](int r) {
      const uint32_t head = key[0] & ~WHICH;
      const uint32_t m = __reduce_max_sync(0xffffffffu, head);
      const int from = __ffs(__ballot_sync(0xffffffffu, head == m)) - 1;
      const uint32_t taken = __shfl_sync(0xffffffffu, key[0], from);
      if (lane == r) {
        my_key = m;
        mine = m ? from * VPL + (int)(WHICH - (taken & WHICH)) : -1;
      }
      last = m;
      if (lane == from) {
#pragma unroll
        for (int j = 0; j + 1 < VPL; ++j) key[j] = key[j + 1];
        key[VPL - 1] = 0;
      }
    };
    auto apart = [&](uint32_t ka, uint32_t kb) {     // whether ka is larger for sure
      if (by_logit) return ka != kb;
      const float a = from_ordered(ka), b = from_ordered(kb);
      return of_values.certain(a, b, total, fmaxf(fabsf(a), fabsf(b)));
    };
#pragma unroll 2
    for (int r = 0; r < p.k + (exact ? 0 : 1); ++r) take(r);
    bool in_doubt = near;
    if (!exact) {
      uint32_t next = __shfl_down_sync(0xffffffffu, my_key, 1);
      if (lane == p.k - 1) next = last;     // (lane 32 of k = 32)
      in_doubt |= __any_sync(0xffffffffu, lane < p.k && next != 0 && !apart(my_key, next)) != 0;
    }
    if (in_doubt) {
      // A few more, as far as these have surely left the k-th behind: then the choice is among them, and a lane each finds their values in
      // 64 bits.  Otherwise (or where a group or a softmax's sum is in doubt, with a bias) all of the token's values are formed anew.
      const int n = p.k + EXTRA;
      bool among = !near && (by_logit || p.sigmoid) && n <= 32;
      if (among) {
#pragma unroll 1
        for (int r = p.k + 1; r < n; ++r) take(r);
        among = last == 0 || apart(__shfl_sync(0xffffffffu, my_key, p.k - 1), last);
      }
      if (among) {
        double d = -CUDART_INF;
        if (mine >= 0) {
          d = finite_logit(to_float(static_cast<const T*>(logits)[t * p.ld + mine]));
          if (!by_logit) d = 1.0 / (1.0 + exp(-d)) + (double)p.bias[mine];
        }
        int rank = 0;
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
          const double u = __shfl_sync(0xffffffffu, d, c);
          const int i = __shfl_sync(0xffffffffu, mine, c);
          rank += u > d || (u == d && i < mine);
        }
        if (mine < 0) rank = 32;
        const int found = mine;
        mine = -1;
#pragma unroll 1
        for (int c = 0; c < p.k; ++c) {
          const unsigned who = __ballot_sync(0xffffffffu, rank == c);
          const int i = __shfl_sync(0xffffffffu, found, who ? __ffs(who) - 1 : 0);
          if (lane == c && who) mine = i;
        }
      } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j)
          if (e0 + j < p.E) row[e0 + j] = l[j];
        __syncwarp();
        mine = choose<VPL>(p, row, value, lane);
        __syncwarp();
      }
    }
    if (lane >= p.k) mine = -1;
    // the weights, lane j the j-th: softmax over all experts, or without its common factor where the sum divides it out; sigmoid
    // times e^-m for m = min(0, largest chosen logit), which cannot underflow as a whole
    const float chosen = mine >= 0 ? finite_logit(to_float(static_cast<const T*>(logits)[t * p.ld + mine])) : -CUDART_INF_F;
    float w = 0.0f;
    if (p.sigmoid) {
      const float m = p.renormalise ? fminf(0.0f, from_ordered(__reduce_max_sync(0xffffffffu, ordered(chosen)))) : 0.0f;
      if (mine >= 0) w = 1.0f / (expf(m) + expf(m - chosen));
    } else {
      if (p.renormalise) top = from_ordered(__reduce_max_sync(0xffffffffu, ordered(chosen)));
      if (mine >= 0) w = expf(chosen - top);
      if (!p.renormalise && mine >= 0) w /= total;
    }
    if (p.renormalise) {
      const float sum = warp_sum(w);
      if (mine >= 0) w /= sum;
    }
    if (lane < p.k) {
      p.ids[t * p.k + lane] = mine;
      p.weights[t * p.k + lane] = w * p.scale;
    }
  }
}

template <int DT>
int launch_route(const void* logits, RouteParams p, cudaStream_t st) {
  const size_t smem = (size_t)ROUTE_WARPS * p.E * 12;
  const int64_t word = 16 / (int64_t)dtype_size(DT);
  p.lanes_to_search = 1;
  while (2 * p.lanes_to_search * p.groups <= 32) p.lanes_to_search *= 2;
  p.vec = aligned(logits, 16) && p.E % word == 0 && (p.ld % word == 0 || p.T == 1);
#define MQ_ROUTE(VPL)                                                                                                     \
  do {                                                                                                                    \
    const int lanes = p.group_size / VPL;                                                                                 \
    p.lanes_per_group = p.group_size % VPL == 0 && (lanes & (lanes - 1)) == 0 && lanes * p.groups <= 32 ? lanes : 0;      \
    if (smem > SMEM_AS_IS) MQ_TRY((allow_smem<route_kernel<DT, VPL>>((size_t)ROUTE_WARPS * 32 * VPL * 12)));               \
    const int64_t blocks = ceil_div(p.T, ROUTE_WARPS), most = 148 * route_blocks(VPL);                                    \
    MQ_CUDA(launch_chained(true, route_kernel<DT, VPL>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(ROUTE_WARPS * 32), smem, st, logits, p)); \
  } while (0)
  if (p.E <= 32) MQ_ROUTE(1);
  else if (p.E <= 64) MQ_ROUTE(2);
  else if (p.E <= 128) MQ_ROUTE(4);
  else if (p.E <= 256) MQ_ROUTE(8);
  else if (p.E <= 512) MQ_ROUTE(16);
  else MQ_ROUTE(32);
#undef MQ_ROUTE
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}

// ---------------------------------------------------------------- the plan
// A stable counting sort of the pairs by expert.  Every block takes a run of pairs; the first kernel counts them by expert, the
// second adds up the blocks in front and ranks its own.  Within a block each warp takes a run of its own, 32 pairs at a
// time; which of the 32 have the same expert comes from a vote per bit of its number (the match instruction takes some 100 cycles of the SM
// where all 32 differ: 3000 cycles for the 32 warps of a block, 25 us for 16384 pairs).
constexpr int PLAN_THREADS = 1024, PLAN_WARPS = PLAN_THREADS / 32, PLAN_KEEP = 8, PLAN_FETCH = 20, PLAN_BLOCKS = 148;

struct PlanParams {
  const int32_t* ids;
  int64_t pairs;
  int E, first;
  int run;      // pairs per block, a multiple of 32 * PLAN_WARPS
  int bits;     // 2^bits > E
  int32_t* counts;
  int32_t *offsets, *order, *place;
};

__device__ __forceinline__ int expert_of(const PlanParams& p, int64_t i, int64_t end) {
  if (i >= end) return -1;
  const int64_t e = (int64_t)p.ids[i] - p.first;
  return e >= 0 && e < p.E ? (int)e : -1;
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_count_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS) plan_smem[e] = 0;
  __syncthreads();
  chain_wait();
  chain_release();
  const int64_t begin = (int64_t)blockIdx.x * p.run, end = min(begin + p.run, p.pairs);
  for (int64_t i0 = begin + threadIdx.x; i0 < end; i0 += PLAN_THREADS * PLAN_KEEP) {
    int e[PLAN_KEEP];
#pragma unroll
    for (int i = 0; i < PLAN_KEEP; ++i) e[i] = expert_of(p, i0 + i * PLAN_THREADS, end);
#pragma unroll
    for (int i = 0; i < PLAN_KEEP; ++i)
      if (e[i] >= 0) atomicAdd(&plan_smem[e[i]], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS) p.counts[(int64_t)blockIdx.x * p.E + e] = plan_smem[e];
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_place_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];                 // next[warp][e]: where this warp's next pair of e goes; total[e], before[e]
  __shared__ int warp_total[PLAN_WARPS];
  __shared__ int all_pairs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t begin = (int64_t)blockIdx.x * p.run, end = min(begin + p.run, p.pairs);
  const int per_warp = p.run / PLAN_WARPS;
  const int64_t w_begin = begin + (int64_t)warp * per_warp, w_end = min(w_begin + per_warp, end);
  int* next = plan_smem + warp * p.E;
  int *totals = plan_smem + PLAN_WARPS * p.E, *befores = totals + p.E;
  for (int i = threadIdx.x; i < p.E * (PLAN_WARPS + 2); i += PLAN_THREADS) plan_smem[i] = 0;
  __syncthreads();
  chain_wait();
  chain_release();
  if (p.counts) {
    // All blocks' counts: a warp takes 32 experts and a share of the blocks, PLAN_FETCH loads at a time that do not wait for one another.  (One thread per
    // expert that walks through the blocks, or 32 experts after the other with all blocks' counts shared out, cost 18 and 6 us of latency
    // for 524288 pairs.)
    const int slices = (p.E + 31) / 32, shares = slices < PLAN_WARPS ? PLAN_WARPS / slices : 1;
    const int per_share = ((int)gridDim.x + shares - 1) / shares;
    for (int slice = warp % (slices < PLAN_WARPS ? slices : PLAN_WARPS); slice < slices; slice += PLAN_WARPS) {
      const int share = slices < PLAN_WARPS ? warp / slices : 0, e = slice * 32 + lane;
      if (share >= shares || e >= p.E) continue;
      const int first = share * per_share, last = min(first + per_share, (int)gridDim.x);
      int total = 0, before = 0;
      for (int b0 = first; b0 < last; b0 += PLAN_FETCH) {
        int c[PLAN_FETCH];
#pragma unroll
        for (int i = 0; i < PLAN_FETCH; ++i) c[i] = b0 + i < last ? __ldcg(p.counts + (int64_t)(b0 + i) * p.E + e) : 0;
#pragma unroll
        for (int i = 0; i < PLAN_FETCH; ++i) {
          total += c[i];
          before += b0 + i < (int)blockIdx.x ? c[i] : 0;
        }
      }
      atomicAdd(&totals[e], total);
      atomicAdd(&befores[e], before);
    }
  }
  // the experts of the warp's pairs, PLAN_KEEP at a time in registers; a run that is no longer stays there
  int mine[PLAN_KEEP];
  const bool all_kept = per_warp <= 32 * PLAN_KEEP;
  auto load = [&](int64_t i0) {
#pragma unroll
    for (int i = 0; i < PLAN_KEEP; ++i) mine[i] = expert_of(p, i0 + i * 32 + lane, w_end);
  };
  for (int64_t i0 = w_begin; i0 < w_end; i0 += 32 * PLAN_KEEP) {
    load(i0);
#pragma unroll
    for (int i = 0; i < PLAN_KEEP; ++i)
      if (mine[i] >= 0) atomicAdd(&next[mine[i]], 1);
  }
  __syncthreads();
  // experts in slices of PLAN_THREADS: pairs of all experts in front, of this one in the blocks in front, of this block's warps in front
  int in_front = 0;
  for (int e0 = 0; e0 < p.E; e0 += PLAN_THREADS) {
    const int e = e0 + threadIdx.x;
    int total = 0, before = 0;
    if (e < p.E) {
      if (p.counts) {
        total = totals[e];
        before = befores[e];
      } else {
        for (int w = 0; w < PLAN_WARPS; ++w) total += plan_smem[w * p.E + e];
      }
    }
    int sum = total;
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    if (lane == 31) warp_total[warp] = sum;
    __syncthreads();
    int base = in_front + sum - total;
    for (int w = 0; w < warp; ++w) base += warp_total[w];
    if (e < p.E) {
      if (blockIdx.x == 0) p.offsets[e] = base;
      int at = base + before;
      for (int w = 0; w < PLAN_WARPS; ++w) {
        const int c = plan_smem[w * p.E + e];
        plan_smem[w * p.E + e] = at;
        at += c;
      }
    }
    for (int w = 0; w < PLAN_WARPS; ++w) in_front += warp_total[w];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    all_pairs = in_front;
    if (blockIdx.x == 0) p.offsets[p.E] = in_front;
  }
  __syncthreads();
  for (int64_t i0 = w_begin; i0 < w_end; i0 += 32 * PLAN_KEEP) {
    if (!all_kept) load(i0);
#pragma unroll
    for (int b = 0; b < PLAN_KEEP; ++b) {
      const int64_t i = i0 + b * 32 + lane;
      if (i - lane >= w_end) break;
      const int e = mine[b];
      unsigned same = 0xffffffffu;      // lanes with the same expert; -1 has all bits set, as no expert's number has
      for (int bit = 0; bit < p.bits; ++bit) {
        const bool set = e >> bit & 1;
        const unsigned with = __ballot_sync(0xffffffffu, set);
        same &= set ? with : ~with;
      }
      const int rank = __popc(same & ((1u << lane) - 1u));
      int at = -1;
      if (e >= 0) at = next[e] + rank;
      __syncwarp();
      if (e >= 0) {
        if (rank == 0) next[e] = at + __popc(same);
        p.order[at] = (int32_t)i;
      }
      __syncwarp();
      if (i < w_end) {
        p.place[i] = at;
        if (i >= all_pairs) p.order[i] = -1;   // behind the last pair
      }
    }
  }
}

int plan_blocks(int64_t pairs) {
  // one block, and one launch, up to four pairs a thread (7.4 us for 4096 pairs, where two launches take 9); beyond, one a thread while there are
  // SMs: the scattered stores of `order` are what a block spends its time on
  if (pairs <= 4 * PLAN_THREADS) return 1;
  const int64_t b = ceil_div(pairs, PLAN_THREADS);
  return (int)(b > PLAN_BLOCKS ? PLAN_BLOCKS : b);
}

}  // namespace
}  // namespace mq

using namespace mq;

extern "C" int mq_route_tokens(const void* logits, int dtype, int64_t T, int64_t E, int64_t ld, int top_k, int score, const float* bias,
                               int groups, int keep_groups, int group_score, int renormalise, float scale, int32_t* ids, float* weights,
                               void* stream) {
  MQ_REQUIRE(valid_dtype(dtype), MQ_ERR_ARGUMENT, "mq_route_tokens: unknown dtype %d", dtype);
  MQ_REQUIRE(T >= 0 && E >= 1 && ld >= E, MQ_ERR_ARGUMENT, "mq_route_tokens: bad sizes T=%lld E=%lld ld=%lld", (long long)T, (long long)E,
             (long long)ld);
  MQ_REQUIRE(E <= MAX_EXPERTS, MQ_ERR_UNSUPPORTED, "mq_route_tokens: at most 1024 experts (got %lld)", (long long)E);
  MQ_REQUIRE(top_k >= 1 && top_k <= 32 && top_k <= E, MQ_ERR_ARGUMENT, "mq_route_tokens: top_k must be in [1, min(32, E)] (got %d)", top_k);
  MQ_REQUIRE((score == 0 || score == 1) && (group_score == 0 || group_score == 1), MQ_ERR_ARGUMENT,
             "mq_route_tokens: unknown score %d or group score %d", score, group_score);
  MQ_REQUIRE(groups >= 1 && groups <= 32 && E % groups == 0 && keep_groups >= 1 && keep_groups <= groups, MQ_ERR_ARGUMENT,
             "mq_route_tokens: groups must be in [1, 32] and divide E, keep_groups in [1, groups] (got %d of %d)", keep_groups, groups);
  if (T == 0) return MQ_OK;
  MQ_REQUIRE(logits && ids && weights, MQ_ERR_ARGUMENT, "mq_route_tokens: null pointer");
  MQ_REQUIRE(ceil_div(T, ROUTE_WARPS) < (1ll << 31), MQ_ERR_UNSUPPORTED, "mq_route_tokens: too many tokens");
  RouteParams p = {T, ld, (int)E, top_k, groups, keep_groups, (int)(E / groups), score == 1, group_score == 1, renormalise != 0, scale, bias, ids, weights, false, 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MQ_F32 ? launch_route<MQ_F32>(logits, p, st) : dtype == MQ_BF16 ? launch_route<MQ_BF16>(logits, p, st) : launch_route<MQ_F16>(logits, p, st);
}

extern "C" size_t mq_expert_plan_workspace_bytes(int64_t pairs, int64_t E) {
  const int blocks = plan_blocks(pairs);
  return blocks > 1 ? (size_t)blocks * (size_t)E * 4 : 0;
}

namespace mq {
int expert_plan(const int32_t* ids, int64_t pairs, int E, int first, int32_t* offsets, int32_t* order, int32_t* place, void* workspace,
                cudaStream_t st) {
  const int blocks = plan_blocks(pairs);
  const int64_t unit = 32 * PLAN_WARPS;
  PlanParams p = {ids, pairs, E, first, (int)(ceil_div(ceil_div(pairs > 0 ? pairs : 1, blocks), unit) * unit), 0, nullptr, offsets, order, place};
  while ((1 << p.bits) <= E) ++p.bits;
  if (blocks > 1) {
    p.counts = static_cast<int32_t*>(workspace);
    MQ_CUDA(launch_chained(true, plan_count_kernel, dim3(blocks), dim3(PLAN_THREADS), (size_t)E * 4, st, p));
    MQ_LAUNCH_CHECK();
  }
  const size_t smem = (size_t)E * (PLAN_WARPS + 2) * 4;
  if (smem > SMEM_AS_IS) MQ_TRY(allow_smem<plan_place_kernel>((size_t)MAX_EXPERTS * (PLAN_WARPS + 2) * 4));
  MQ_CUDA(launch_chained(true, plan_place_kernel, dim3(blocks), dim3(PLAN_THREADS), smem, st, p));
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}
}  // namespace mq

extern "C" int mq_expert_plan(const int32_t* ids, int64_t pairs, int64_t E, int64_t first, int32_t* offsets, int32_t* order, int32_t* place,
                              void* workspace, size_t workspace_bytes, void* stream) {
  // (2^31 - 1 is no expert: wider ids that are clamped to it stay without one)
  MQ_REQUIRE(pairs >= 0 && E >= 1 && first >= 0 && first < (1ll << 31) - E, MQ_ERR_ARGUMENT, "mq_expert_plan: bad sizes pairs=%lld E=%lld first=%lld",
             (long long)pairs, (long long)E, (long long)first);
  MQ_REQUIRE(E <= MAX_EXPERTS && pairs < (1ll << 31) - (1 << 20), MQ_ERR_UNSUPPORTED, "mq_expert_plan: at most 1024 experts and 2^31 - 2^20 pairs");
  MQ_REQUIRE(offsets && (pairs == 0 || (ids && order && place)), MQ_ERR_ARGUMENT, "mq_expert_plan: null pointer");
  MQ_REQUIRE(plan_blocks(pairs) == 1 || (workspace && workspace_bytes >= mq_expert_plan_workspace_bytes(pairs, E)), MQ_ERR_WORKSPACE,
             "mq_expert_plan: the workspace has %zu bytes and needs %zu", workspace_bytes, mq_expert_plan_workspace_bytes(pairs, E));
  return expert_plan(ids, pairs, (int)E, (int)first, offsets, order, place, workspace, static_cast<cudaStream_t>(stream));
}
