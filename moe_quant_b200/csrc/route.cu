// Routing of tokens to experts, and the plan that groups the (token, expert) pairs by expert.
//
// Routing, per token: scores s = sigmoid(logit) or softmax(logits); values v = s + bias; the groups with the largest
// sum of two values (or largest value) stay; the top_k largest v of those are chosen, ties to the lowest index; weights are
// the scores without bias, normalised over the chosen ones where asked.  An expert whose logit is -inf or NaN, or whose bias is
// -inf or NaN, is never chosen.  +inf counts as the largest finite number.
//
// One warp per token, the token's experts spread over its lanes.
#include <math_constants.h>

#include "common.cuh"
#include "profile.cuh"

namespace mq {
namespace {

constexpr int ROUTE_WARPS = 8;

struct RouteParams {
  int64_t T, ld;
  int E, k, groups, keep, group_size;
  bool sigmoid, top2, renormalise;
  float scale;
  const float* bias;
  int32_t* ids;
  float* weights;
};

__device__ __forceinline__ float finite_logit(float l) { return l != l ? -CUDART_INF_F : fminf(l, 3.402823466e38f); }

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
// the larger value, the lower index of equals; all lanes get it
__device__ __forceinline__ void warp_argmax(double& v, int& i) {
  for (int o = 16; o > 0; o >>= 1) {
    const double u = __shfl_xor_sync(0xffffffffu, v, o);
    const int j = __shfl_xor_sync(0xffffffffu, i, o);
    if (u > v || (u == v && j < i)) {
      v = u;
      i = j;
    }
  }
}

// The choice in 64 bits.  `row` holds the token's logits (finite_logit), `value` is scratch of E doubles, both of this warp.
// Lane j < k gets the j-th expert, or -1.
__device__ int choose(const RouteParams& p, const float* row, double* value, int lane) {
  const bool by_logit = p.bias == nullptr;   // sigmoid and softmax are increasing
  double top = -CUDART_INF, total = 0.0;
  if (!p.sigmoid && (p.groups > 1 || !by_logit)) {
    for (int e = lane; e < p.E; e += 32) top = max(top, (double)row[e]);
    top = warp_max(top);
    for (int e = lane; e < p.E; e += 32)
      if (row[e] > -CUDART_INF_F) total += exp((double)row[e] - top);
    total = warp_sum(total);
  }
  for (int e = lane; e < p.E; e += 32) {
    const double l = row[e];
    double v = -CUDART_INF;
    if (row[e] > -CUDART_INF_F) {
      if (by_logit && p.groups == 1) v = l;
      else v = p.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - top) / total;
      if (!by_logit) v += (double)p.bias[e];
      if (v != v) v = -CUDART_INF;
    }
    value[e] = v;
  }
  __syncwarp();
  if (p.groups > 1) {
    double of_group = -CUDART_INF;   // of group `lane`
    if (lane < p.groups) {
      double second = -CUDART_INF;
      for (int i = 0; i < p.group_size; ++i) {
        const double v = value[lane * p.group_size + i];
        if (v > of_group) {
          second = of_group;
          of_group = v;
        } else if (v > second) {
          second = v;
        }
      }
      if (p.top2 && second > -CUDART_INF) of_group += second;
    }
    int better = 0;
    for (int g = 0; g < p.groups; ++g) {
      const double u = __shfl_sync(0xffffffffu, of_group, g);
      better += u > of_group || (u == of_group && g < lane);
    }
    const unsigned kept = __ballot_sync(0xffffffffu, lane < p.groups && better < p.keep);
    __syncwarp();
    for (int e = lane; e < p.E; e += 32) {
      if (!(kept >> (e / p.group_size) & 1u)) value[e] = -CUDART_INF;
      else if (by_logit) value[e] = row[e];
    }
    __syncwarp();
  }
  int mine = -1;
  for (int r = 0; r < p.k; ++r) {
    double v = -CUDART_INF;
    int at = p.E;
    for (int e = lane; e < p.E; e += 32)
      if (value[e] > v) {
        v = value[e];
        at = e;
      }
    warp_argmax(v, at);
    if (!(v > -CUDART_INF)) break;
    if (lane == r) mine = at;
    if (lane == 0) value[at] = -CUDART_INF;
    __syncwarp();
  }
  return mine;
}

template <int DT>
__global__ void __launch_bounds__(ROUTE_WARPS * 32) route_kernel(const void* __restrict__ logits, const RouteParams p) {
  using T = typename StorageOf<DT>::type;
  extern __shared__ double route_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double* value = route_smem + (size_t)warp * p.E;
  float* row = reinterpret_cast<float*>(route_smem + (size_t)ROUTE_WARPS * p.E) + (size_t)warp * p.E;
  const int64_t t = (int64_t)blockIdx.x * ROUTE_WARPS + warp;
  if (t >= p.T) return;
  const T* src = static_cast<const T*>(logits) + t * p.ld;
  for (int e = lane; e < p.E; e += 32) row[e] = finite_logit(to_float(src[e]));
  __syncwarp();
  const int mine = choose(p, row, value, lane);
  // the weights, lane j the j-th: softmax over all experts, or without its common factor where the sum divides it out; sigmoid
  // times e^-m for m = min(0, largest chosen logit), which cannot underflow as a whole
  const float l = mine >= 0 ? row[mine] : -CUDART_INF_F;
  float w;
  if (p.sigmoid) {
    const float m = p.renormalise ? fminf(0.0f, warp_max(l)) : 0.0f;
    w = mine >= 0 ? 1.0f / (expf(m) + expf(m - l)) : 0.0f;
  } else {
    float top = l;
    if (!p.renormalise)
      for (int e = lane; e < p.E; e += 32) top = fmaxf(top, row[e]);
    top = warp_max(top);
    w = mine >= 0 ? expf(l - top) : 0.0f;
    if (!p.renormalise) {
      float total = 0.0f;
      for (int e = lane; e < p.E; e += 32)
        if (row[e] > -CUDART_INF_F) total += expf(row[e] - top);
      total = warp_sum(total);
      if (mine >= 0) w /= total;
    }
  }
  if (p.renormalise) {
    const float total = warp_sum(w);
    if (mine >= 0) w /= total;
  }
  if (lane < p.k) {
    p.ids[t * p.k + lane] = mine;
    p.weights[t * p.k + lane] = w * p.scale;
  }
}

// ---------------------------------------------------------------- the plan
// A stable counting sort of the pairs by expert.  Every block takes a run of pairs; the first kernel counts them by expert, the
// second adds up the blocks in front and ranks its own.  Within a block each warp takes a run of its own, 32 pairs at a
// time; equal experts among the 32 are ranked by a match.
constexpr int PLAN_THREADS = 512, PLAN_WARPS = PLAN_THREADS / 32;

struct PlanParams {
  const int32_t* ids;
  int64_t pairs;
  int E, first;
  int run;      // pairs per block, a multiple of 32 * PLAN_WARPS
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
  const int64_t begin = (int64_t)blockIdx.x * p.run, end = min(begin + p.run, p.pairs);
  for (int64_t i = begin + threadIdx.x; i < end; i += PLAN_THREADS) {
    const int e = expert_of(p, i, end);
    if (e >= 0) atomicAdd(&plan_smem[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += PLAN_THREADS) p.counts[(int64_t)blockIdx.x * p.E + e] = plan_smem[e];
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_place_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];                 // next[warp][e]: where this warp's next pair of e goes
  __shared__ int warp_total[PLAN_WARPS];
  __shared__ int all_pairs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t begin = (int64_t)blockIdx.x * p.run, end = min(begin + p.run, p.pairs);
  const int per_warp = p.run / PLAN_WARPS;
  const int64_t w_begin = begin + (int64_t)warp * per_warp, w_end = min(w_begin + per_warp, end);
  int* next = plan_smem + warp * p.E;
  for (int i = threadIdx.x; i < p.E * PLAN_WARPS; i += PLAN_THREADS) plan_smem[i] = 0;
  __syncthreads();
  for (int64_t i = w_begin + lane; i < w_end; i += 32) {
    const int e = expert_of(p, i, w_end);
    if (e >= 0) atomicAdd(&next[e], 1);
  }
  __syncthreads();
  // experts in slices of PLAN_THREADS: pairs of all experts in front, of this one in the blocks in front, of this block's warps in front
  int in_front = 0;
  for (int e0 = 0; e0 < p.E; e0 += PLAN_THREADS) {
    const int e = e0 + threadIdx.x;
    int total = 0, before = 0;
    if (e < p.E) {
      if (p.counts) {
        for (int b = 0; b < (int)gridDim.x; ++b) {
          const int c = p.counts[(int64_t)b * p.E + e];
          if (b < (int)blockIdx.x) before += c;
          total += c;
        }
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
  for (int64_t i0 = w_begin; i0 < w_end; i0 += 32) {
    const int64_t i = i0 + lane;
    const int e = expert_of(p, i, w_end);
    const unsigned same = __match_any_sync(0xffffffffu, e);
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

int plan_blocks(int64_t pairs) {
  const int64_t run = 32 * PLAN_WARPS;
  const int64_t b = ceil_div(pairs, 4 * run);
  return (int)(b < 1 ? 1 : b > 148 ? 148 : b);
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
  MQ_REQUIRE(E <= 1024, MQ_ERR_UNSUPPORTED, "mq_route_tokens: at most 1024 experts (got %lld)", (long long)E);
  MQ_REQUIRE(top_k >= 1 && top_k <= 32 && top_k <= E, MQ_ERR_ARGUMENT, "mq_route_tokens: top_k must be in [1, min(32, E)] (got %d)", top_k);
  MQ_REQUIRE((score == 0 || score == 1) && (group_score == 0 || group_score == 1), MQ_ERR_ARGUMENT,
             "mq_route_tokens: unknown score %d or group score %d", score, group_score);
  MQ_REQUIRE(groups >= 1 && groups <= 32 && E % groups == 0 && keep_groups >= 1 && keep_groups <= groups, MQ_ERR_ARGUMENT,
             "mq_route_tokens: groups must be in [1, 32] and divide E, keep_groups in [1, groups] (got %d of %d)", keep_groups, groups);
  if (T == 0) return MQ_OK;
  MQ_REQUIRE(logits && ids && weights, MQ_ERR_ARGUMENT, "mq_route_tokens: null pointer");
  MQ_REQUIRE(ceil_div(T, ROUTE_WARPS) < (1ll << 31), MQ_ERR_UNSUPPORTED, "mq_route_tokens: too many tokens");
  RouteParams p = {T, ld, (int)E, top_k, groups, keep_groups, (int)(E / groups), score == 1, group_score == 1, renormalise != 0, scale, bias, ids, weights};
  const size_t smem = (size_t)ROUTE_WARPS * E * 12;
  auto kernel = dtype == MQ_F32 ? route_kernel<MQ_F32> : dtype == MQ_BF16 ? route_kernel<MQ_BF16> : route_kernel<MQ_F16>;
  if (smem > 48 * 1024) MQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<(unsigned)ceil_div(T, ROUTE_WARPS), ROUTE_WARPS * 32, smem, static_cast<cudaStream_t>(stream)>>>(logits, p);
  MQ_LAUNCH_CHECK();
  return MQ_OK;
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
  PlanParams p = {ids, pairs, E, first, (int)(ceil_div(ceil_div(pairs > 0 ? pairs : 1, blocks), unit) * unit), nullptr, offsets, order, place};
  if (blocks > 1) {
    p.counts = static_cast<int32_t*>(workspace);
    plan_count_kernel<<<blocks, PLAN_THREADS, (size_t)E * 4, st>>>(p);
    MQ_LAUNCH_CHECK();
  }
  const size_t smem = (size_t)E * PLAN_WARPS * 4;
  if (smem > 48 * 1024) MQ_CUDA(cudaFuncSetAttribute(plan_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  plan_place_kernel<<<blocks, PLAN_THREADS, smem, st>>>(p);
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}
}  // namespace mq

extern "C" int mq_expert_plan(const int32_t* ids, int64_t pairs, int64_t E, int64_t first, int32_t* offsets, int32_t* order, int32_t* place,
                              void* workspace, size_t workspace_bytes, void* stream) {
  MQ_REQUIRE(pairs >= 0 && E >= 1 && first >= 0 && first < (1ll << 31), MQ_ERR_ARGUMENT, "mq_expert_plan: bad sizes pairs=%lld E=%lld first=%lld",
             (long long)pairs, (long long)E, (long long)first);
  MQ_REQUIRE(E <= 1024 && pairs < (1ll << 31) - (1 << 20), MQ_ERR_UNSUPPORTED, "mq_expert_plan: at most 1024 experts and 2^31 - 2^20 pairs");
  MQ_REQUIRE(offsets && (pairs == 0 || (ids && order && place)), MQ_ERR_ARGUMENT, "mq_expert_plan: null pointer");
  MQ_REQUIRE(plan_blocks(pairs) == 1 || (workspace && workspace_bytes >= mq_expert_plan_workspace_bytes(pairs, E)), MQ_ERR_WORKSPACE,
             "mq_expert_plan: the workspace has %zu bytes and needs %zu", workspace_bytes, mq_expert_plan_workspace_bytes(pairs, E));
  return expert_plan(ids, pairs, (int)E, (int)first, offsets, order, place, workspace, static_cast<cudaStream_t>(stream));
}
