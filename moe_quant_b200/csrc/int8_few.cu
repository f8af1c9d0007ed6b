// 8-bit integer products of a few tokens: the weights are read once, straight into registers, and bound the time.
//
// Every block holds the codes of all tokens in shared memory (it rounds them itself: they are few, and the first weights are on their way
// meanwhile) and takes a run of weight rows, a row per warp.  A lane multiplies 16 weights at a time with the tokens' codes (dp4a);
// the warp's sums come together in one reduction.  512 threads per block, one block per SM: sixteen warps with eight 16-byte loads per
// lane under way are 64 KB per SM, which is what the memory's latency wants.
#include <math_constants.h>

#include "int8.cuh"
#include "int8_codes.cuh"
#include "profile.cuh"

namespace mq {
namespace {

constexpr int FEW_THREADS = 512, FEW_WARPS = FEW_THREADS / 32, FEW_BLOCKS = 148, FEW_LOADS = 8;
constexpr int FEW_STEP = 512 * FEW_LOADS;   // bytes of a row that a warp loads at a time
constexpr size_t FEW_SMEM = 200 * 1024;

// bytes that a token's codes take: a whole number of steps, zeros behind the end
__host__ __device__ __forceinline__ int few_pitch(int K) { return (K + 511) / 512 * 512; }

// 16 codes of a weight row from byte k on; zeros behind its end
__device__ __forceinline__ int4 weights16(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return __ldcs(reinterpret_cast<const int4*>(row + k));
  int4 v = make_int4(0, 0, 0, 0);
  if (k < K) {
    uint32_t* p = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (k + j < K) p[j >> 2] |= (uint32_t)(uint8_t)row[k + j] << (8 * (j & 3));
  }
  return v;
}
__device__ __forceinline__ int dot16(int4 a, int4 b, int sum) {
  return __dp4a(a.w, b.w, __dp4a(a.z, b.z, __dp4a(a.y, b.y, __dp4a(a.x, b.x, sum))));
}

// a step of a row into registers: only the loads that lie in the row
__device__ __forceinline__ void load_step(int4 (&w)[FEW_LOADS], const int8_t* row, int k0, int K, int lane) {
#pragma unroll
  for (int i = 0; i < FEW_LOADS; ++i) {
    const int k = k0 + i * 512 + lane * 16;
    w[i] = k < K ? weights16(row, k, K) : make_int4(0, 0, 0, 0);
  }
}

// Rounds a row of numbers to codes in shared memory with `threads` threads (a multiple of 32, `id` of this one), whose warps leave their
// largest bits in `part` and meet in `meet`.  Returns the scale.
template <bool VEC, typename S, typename Meet>
__device__ __forceinline__ float round_row(const S* row, int K, int8_t* codes, int pitch, int id, int threads, uint32_t* part, Meet meet) {
  uint32_t bits = 0;
  for (int k = id * 8; k < K; k += threads * 8) bits = max(bits, largest_bits(eight_of<VEC>(row, k, K)));
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (threads > 32) {
    if ((id & 31) == 0) part[id >> 5] = bits;
    meet();
    for (int w = 0; w < threads / 32; ++w) bits = max(bits, part[w]);
  }
  const RowCodes code(bits);
  for (int k = id * 8; k < pitch; k += threads * 8) *reinterpret_cast<uint2*>(codes + k) = code.of(eight_of<VEC>(row, k, K));
  return code.scale;
}

struct FewParams {
  const void* x;
  const float* x_scale;   // MQ_I8
  int64_t ldx;
  int T, N, K;
  const int8_t* w;
  int64_t ldw;
  const float *w_scale, *bias;
  int out_dtype;
  void* y;
  int64_t ldy;
};

__device__ __forceinline__ void put(void* y, int dtype, int64_t at, float v) {
  if (dtype == MQ_F32) static_cast<float*>(y)[at] = v;
  else if (dtype == MQ_BF16) static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(y)[at] = __float2half_rn(v);
}

// NT tokens (T <= NT; the others' codes are zero), numbers or (MQ_I8) codes already
template <int DT, int NT, bool VEC>
__global__ void __launch_bounds__(FEW_THREADS, 1) int8_few_kernel(const FewParams p) {
  using S = typename StorageOf<DT == MQ_I8 ? MQ_F32 : DT>::type;
  extern __shared__ __align__(16) int8_t few_codes[];
  __shared__ uint32_t part[NT][FEW_WARPS];
  __shared__ float x_scale[NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pitch = few_pitch(p.K);
  const int begin = (int)((int64_t)p.N * blockIdx.x / gridDim.x), end = (int)((int64_t)p.N * (blockIdx.x + 1) / gridDim.x);
  chain_wait();
  chain_release();
  int4 w[FEW_LOADS];
  int n = begin + warp;
  if (n < end) load_step(w, p.w + (int64_t)n * p.ldw, 0, p.K, lane);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if constexpr (DT == MQ_I8) {
      const int8_t* row = static_cast<const int8_t*>(p.x) + t * p.ldx;
      for (int k = threadIdx.x * 16; k < pitch; k += FEW_THREADS * 16)
        *reinterpret_cast<int4*>(few_codes + t * pitch + k) = t < p.T ? weights16(row, k, p.K) : make_int4(0, 0, 0, 0);
      if (threadIdx.x == 0 && t < p.T) x_scale[t] = p.x_scale[t];
    } else if (t < p.T) {
      const float s = round_row<VEC>(static_cast<const S*>(p.x) + t * p.ldx, p.K, few_codes + t * pitch, pitch, (int)threadIdx.x, FEW_THREADS, part[t], [] { __syncthreads(); });
      if (threadIdx.x == 0) x_scale[t] = s;
    } else {
      for (int k = threadIdx.x * 8; k < pitch; k += FEW_THREADS * 8) *reinterpret_cast<uint2*>(few_codes + t * pitch + k) = make_uint2(0, 0);
    }
  }
  __syncthreads();
  for (; n < end; n += FEW_WARPS) {
    const int8_t* row = p.w + (int64_t)n * p.ldw;
    int sum[NT] = {};
    for (int k0 = 0; k0 < p.K; k0 += FEW_STEP) {
      int4 now[FEW_LOADS];
#pragma unroll
      for (int i = 0; i < FEW_LOADS; ++i) now[i] = w[i];
      // the next step, of this row or the next one, is under way while this one is multiplied
      if (k0 + FEW_STEP < p.K) load_step(w, row, k0 + FEW_STEP, p.K, lane);
      else if (n + FEW_WARPS < end) load_step(w, row + (int64_t)FEW_WARPS * p.ldw, 0, p.K, lane);
#pragma unroll
      for (int i = 0; i < FEW_LOADS; ++i) {
        const int k = k0 + i * 512;
        if (k >= p.K) break;
#pragma unroll
        for (int t = 0; t < NT; ++t) sum[t] = dot16(now[i], *reinterpret_cast<const int4*>(few_codes + t * pitch + k + lane * 16), sum[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) sum[t] = __reduce_add_sync(0xffffffffu, sum[t]);
    int mine = sum[0];
#pragma unroll
    for (int t = 1; t < NT; ++t) mine = lane == t ? sum[t] : mine;
    if (lane < p.T) {
      float v = (float)mine * x_scale[lane] * __ldg(p.w_scale + n);
      if (p.bias) v += __ldg(p.bias + n);
      put(p.y, p.out_dtype, lane * p.ldy + n, v);
    }
  }
}

// ---------------------------------------------------------------- the experts of one token
// Two launches: the first gives h = silu(gate) * up of every pair of the token and an expert here, a pair of weight rows per warp, the second
// rounds h to codes and sums the pairs' down products, a row of one expert per warp.  The pairs need no plan.
struct OneParams {
  const void* x;
  int K, I, E, top_k, first;
  const int32_t* ids;
  const float* weights;
  const int8_t *gate_up, *down;
  int64_t ld_gate_up, gate_up_expert, ld_down, down_expert;
  const float *gate_up_scale, *down_scale;
  float* h;      // (top_k, I)
  void* y;
};

__device__ __forceinline__ float gated(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// the pairs of the token with experts here, in the order of its slots; a whole warp
__device__ __forceinline__ int pairs_here(const OneParams& p, int lane, int* expert, int* slot) {
  int e = -1;
  if (lane < p.top_k) {
    const int64_t id = (int64_t)p.ids[lane] - p.first;
    if (id >= 0 && id < p.E) e = (int)id;
  }
  const unsigned have = __ballot_sync(0xffffffffu, e >= 0);
  if (e >= 0) {
    const int i = __popc(have & ((1u << lane) - 1u));
    expert[i] = e;
    slot[i] = lane;
  }
  return __popc(have);
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(FEW_THREADS, 1) one_token_gated_kernel(const OneParams p) {
  using S = typename StorageOf<DT>::type;
  extern __shared__ __align__(16) int8_t few_codes[];
  __shared__ uint32_t part[FEW_WARPS];
  __shared__ int expert[32], slot[32], found;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pitch = few_pitch(p.K);
  chain_wait();
  chain_release();
  if (warp == 0) {
    const int n = pairs_here(p, lane, expert, slot);
    if (lane == 0) found = n;
  }
  __syncthreads();
  const int64_t all = (int64_t)found * p.I;     // 32 * INT8_MAX_K at most
  const int begin = (int)(all * blockIdx.x / gridDim.x), end = (int)(all * (blockIdx.x + 1) / gridDim.x);
  // unit u: gate row and up row of result u % I of pair u / I
  auto row_of = [&](int u, int set) {
    const int pair = u / p.I, i = u % p.I;
    return p.gate_up + (int64_t)expert[pair] * p.gate_up_expert + ((int64_t)set * p.I + i) * p.ld_gate_up;
  };
  int4 w[FEW_LOADS];
  int u = begin + warp;
  if (u < end) load_step(w, row_of(u, 0), 0, p.K, lane);
  const float xs = round_row<VEC>(static_cast<const S*>(p.x), p.K, few_codes, pitch, (int)threadIdx.x, FEW_THREADS, part, [] { __syncthreads(); });
  __syncthreads();
  for (; u < end; u += FEW_WARPS) {
    int sum[2] = {0, 0};
#pragma unroll
    for (int set = 0; set < 2; ++set) {
      const int8_t* row = row_of(u, set);
      for (int k0 = 0; k0 < p.K; k0 += FEW_STEP) {
        int4 now[FEW_LOADS];
#pragma unroll
        for (int i = 0; i < FEW_LOADS; ++i) now[i] = w[i];
        if (k0 + FEW_STEP < p.K) load_step(w, row, k0 + FEW_STEP, p.K, lane);
        else if (set == 0) load_step(w, row_of(u, 1), 0, p.K, lane);
        else if (u + FEW_WARPS < end) load_step(w, row_of(u + FEW_WARPS, 0), 0, p.K, lane);
#pragma unroll
        for (int i = 0; i < FEW_LOADS; ++i) {
          const int k = k0 + i * 512;
          if (k >= p.K) break;
          sum[set] = dot16(now[i], *reinterpret_cast<const int4*>(few_codes + k + lane * 16), sum[set]);
        }
      }
    }
    const int g = __reduce_add_sync(0xffffffffu, sum[0]), up = __reduce_add_sync(0xffffffffu, sum[1]);
    if (lane == 0) {
      const int pair = u / p.I, i = u % p.I;
      const float* sc = p.gate_up_scale + (int64_t)expert[pair] * 2 * p.I;
      p.h[(int64_t)pair * p.I + i] = gated((float)g * xs * __ldg(sc + i), (float)up * xs * __ldg(sc + p.I + i));
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(FEW_THREADS, 1) one_token_down_kernel(const OneParams p) {
  extern __shared__ __align__(16) int8_t few_codes[];      // codes of h, then the products of the block's rows, (rows, pairs)
  __shared__ int expert[32], slot[32], found;
  __shared__ float factor[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pitch = few_pitch(p.I);
  float* products = reinterpret_cast<float*>(few_codes + (size_t)p.top_k * pitch);
  // (ids have been there since before the kernel in front began to write)
  if (warp == 0) {
    const int n = pairs_here(p, lane, expert, slot);
    if (lane == 0) found = n;
  }
  __syncthreads();
  const int n_pairs = found;
  const int begin = (int)((int64_t)p.K * blockIdx.x / gridDim.x), end = (int)((int64_t)p.K * (blockIdx.x + 1) / gridDim.x);
  // unit u: row begin + u / n_pairs of the expert of pair u % n_pairs
  const int units = (end - begin) * n_pairs;
  auto row_of = [&](int u) { return p.down + (int64_t)expert[u % n_pairs] * p.down_expert + (int64_t)(begin + u / n_pairs) * p.ld_down; };
  int4 w[FEW_LOADS];
  int u = warp;
  if (u < units) load_step(w, row_of(u), 0, p.I, lane);
  chain_wait();
  chain_release();
  for (int v = warp; v < n_pairs; v += FEW_WARPS) {
    const float s = p.I % 8 == 0 ? round_row<true>(p.h + (int64_t)v * p.I, p.I, few_codes + v * pitch, pitch, lane, 32, nullptr, [] {})
                                 : round_row<false>(p.h + (int64_t)v * p.I, p.I, few_codes + v * pitch, pitch, lane, 32, nullptr, [] {});
    if (lane == 0) factor[v] = s * p.weights[slot[v]];
  }
  __syncthreads();
  for (; u < units; u += FEW_WARPS) {
    const int v = u % n_pairs, n = begin + u / n_pairs;
    const int8_t* row = row_of(u);
    int sum = 0;
    for (int k0 = 0; k0 < p.I; k0 += FEW_STEP) {
      int4 now[FEW_LOADS];
#pragma unroll
      for (int i = 0; i < FEW_LOADS; ++i) now[i] = w[i];
      if (k0 + FEW_STEP < p.I) load_step(w, row, k0 + FEW_STEP, p.I, lane);
      else if (u + FEW_WARPS < units) load_step(w, row_of(u + FEW_WARPS), 0, p.I, lane);
#pragma unroll
      for (int i = 0; i < FEW_LOADS; ++i) {
        const int k = k0 + i * 512;
        if (k >= p.I) break;
        sum = dot16(now[i], *reinterpret_cast<const int4*>(few_codes + v * pitch + k + lane * 16), sum);
      }
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) products[u] = (float)sum * factor[v] * __ldg(p.down_scale + (int64_t)expert[v] * p.K + n);
  }
  __syncthreads();
  for (int r = threadIdx.x; r < end - begin; r += FEW_THREADS) {
    float sum = 0.0f;
    for (int v = 0; v < n_pairs; ++v) sum += products[r * n_pairs + v];
    put(p.y, DT, begin + r, sum);
  }
}

template <typename Params>
int launch_few(void (*kernel)(Params), size_t smem, const Params& p, cudaStream_t st) {
  if (smem > 48 * 1024) MQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FEW_SMEM));
  MQ_CUDA(launch_chained(true, kernel, dim3(FEW_BLOCKS), dim3(FEW_THREADS), smem, st, p));
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}

template <int DT>
bool rows_of_eight(const void* x, int64_t ldx, int64_t K, int64_t T) {
  return K % 8 == 0 && aligned(x, 8 * dtype_size(DT)) && (T == 1 || ldx % 8 == 0);
}

template <int DT, int NT>
int few(const FewParams& p, cudaStream_t st) {
  const size_t smem = (size_t)NT * few_pitch(p.K);
  if constexpr (DT == MQ_I8) return launch_few(int8_few_kernel<DT, NT, true>, smem, p, st);
  else return rows_of_eight<DT>(p.x, p.ldx, p.K, p.T) ? launch_few(int8_few_kernel<DT, NT, true>, smem, p, st) : launch_few(int8_few_kernel<DT, NT, false>, smem, p, st);
}
template <int DT>
int few_of(const FewParams& p, cudaStream_t st) {
  if (p.T == 1) return few<DT, 1>(p, st);
  if (p.T == 2) return few<DT, 2>(p, st);
  return few<DT, 4>(p, st);
}

size_t one_token_down_smem(int top_k, int64_t K, int64_t I) {
  return (size_t)top_k * few_pitch((int)I) + (size_t)(K / FEW_BLOCKS + 1) * top_k * 4;
}

template <int DT>
int one_token(const OneParams& p, cudaStream_t st) {
  const size_t smem = (size_t)few_pitch(p.K);
  MQ_TRY(rows_of_eight<DT>(p.x, 0, p.K, 1) ? launch_few(one_token_gated_kernel<DT, true>, smem, p, st) : launch_few(one_token_gated_kernel<DT, false>, smem, p, st));
  return launch_few(one_token_down_kernel<DT>, one_token_down_smem(p.top_k, p.K, p.I), p, st);
}

}  // namespace

bool int8_few_fits(int64_t T, int64_t K) { return T <= INT8_FEW_TOKENS && (T <= 2 ? T : 4) * few_pitch((int)K) <= (int64_t)FEW_SMEM; }

int int8_few(const void* x, int dtype, int64_t ldx, const Int8Product& q, const Int8Out& o, cudaStream_t st) {
  const FewParams p = {x, q.x_scale, ldx, (int)q.T, q.rows, q.K, q.w, q.ldw, q.w_scale, o.bias, o.dtype, o.y, o.ldy};
  if (dtype == MQ_I8) return few_of<MQ_I8>(p, st);
  if (dtype == MQ_F32) return few_of<MQ_F32>(p, st);
  if (dtype == MQ_BF16) return few_of<MQ_BF16>(p, st);
  return few_of<MQ_F16>(p, st);
}

bool int8_one_token_fits(int top_k, int64_t K, int64_t I) {
  return (size_t)few_pitch((int)K) <= FEW_SMEM && one_token_down_smem(top_k, K, I) <= FEW_SMEM;
}

int int8_one_token(const void* x, int dtype, const int32_t* ids, const float* weights, int top_k, int first, const Int8Product& up, const Int8Product& down,
                   float* h, void* y, cudaStream_t st) {
  const OneParams p = {x, up.K, up.rows, up.E, top_k, first, ids, weights, up.w, down.w, up.ldw, up.w_expert, down.ldw, down.w_expert,
                       up.w_scale, down.w_scale, h, y};
  return dtype == MQ_BF16 ? one_token<MQ_BF16>(p, st) : one_token<MQ_F16>(p, st);
}

}  // namespace mq
