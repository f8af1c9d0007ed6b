// Products in 8-bit integers with one scale per token and one per output channel, and the experts' gated MLPs made of them.
//
//   codes of a token  scale = max|x| / 127, code = round_half_even(127 x / max|x|);  a token with an infinity or a NaN has the scale
//                     NaN and codes of zero, so its whole result is NaN
//   product           y[t, n] = (sum_k code[t, k] w[n, k]) scale[t] w_scale[n] + bias[n], the sum in 32-bit integers: exact
//   experts           h = silu(gate product) * up product per pair of token and expert, codes of h as above, and
//                     y[t] = sum over the token's pairs of weight * down product
//
// Here: the codes (bound by memory and by instructions: 16384 x 2048 fp32 5.9 TB/s, 32768 x 2048 bf16 4.8, 16384 x 7168 bf16 4.3 to 4.5 with 16
// instructions a value and 70 % of the issue slots), the sum over a token's pairs (bound by memory: 6.4 TB/s), and the calls.  The products are in int8_umma.cu (tensor cores, bound by them) and int8_few.cu (up to four tokens,
// and the experts of one: bound by the weights' bytes).
#include <math_constants.h>

#include "int8.cuh"
#include "int8_codes.cuh"
#include "profile.cuh"

namespace mq {

int expert_plan(const int32_t* ids, int64_t pairs, int E, int first, int32_t* offsets, int32_t* order, int32_t* place, void* workspace,
                cudaStream_t st);

namespace {

// ---------------------------------------------------------------- codes of tokens
struct RowsParams {
  const void* x;
  int64_t ldx, T;
  const int32_t* rows_end;   // optional: rows from *rows_end on are left alone
  const int32_t* place;      // optional, (T, top_k): the codes of token t go to the rows place[t, :], but for those that are -1
  int top_k;
  int K;
  int8_t* codes;
  int64_t ldc;
  float* scale;
  // PLAN: the places are found on the way, and written with the offsets
  const int32_t* ids;
  int E, first;
  int32_t *place_out, *offsets;
};

// Up to so many pairs every block finds the places of its tokens by itself, counting the pairs that come in front: a launch less (experts
// of 64 tokens, 512 pairs: 9 us for the plan and the codes, 5 together).
constexpr int PLAN_PAIRS = 2048;

// G threads per row, CH * 8 values a thread at a time; a row of up to G * CH * 8 values stays in registers between the search for its
// largest and the rounding, and the block's next row is on its way meanwhile; a longer one is read twice (the second time from the L2).
// Blocks per SM: what a thread holds of a row, as values and as codes, beside what it needs anyway.
constexpr int rows_blocks(int dt, int ch) { return dt == MQ_F32 ? (ch >= 8 ? 1 : ch >= 4 ? 3 : 4) : (ch >= 8 ? 3 : ch >= 4 ? 4 : 5); }
template <int DT, int G, int CH, bool VEC, bool PLAN>
__global__ void __launch_bounds__(256, rows_blocks(DT, CH)) quantize_rows_kernel(const RowsParams p) {
  using S = typename StorageOf<DT>::type;
  __shared__ uint32_t part[2][8];
  __shared__ int expert[PLAN ? PLAN_PAIRS : 1], count[PLAN ? 1024 : 1];
  chain_wait();
  chain_release();
  const int n_pairs = PLAN ? (int)p.T * p.top_k : 0;
  if constexpr (PLAN) {
    for (int i = threadIdx.x; i < p.E; i += 256) count[i] = 0;
    for (int i = threadIdx.x; i < n_pairs; i += 256) {
      const int64_t e = (int64_t)p.ids[i] - p.first;
      expert[i] = e >= 0 && e < p.E ? (int)e : -1;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; i < n_pairs; i += 256)
        if (expert[i] >= 0) atomicAdd(&count[expert[i]], 1);
      __syncthreads();
      if (threadIdx.x < 32) {
        int before = 0;
        for (int e0 = 0; e0 < p.E; e0 += 32) {
          const int e = e0 + threadIdx.x, n = e < p.E ? count[e] : 0;
          int sum = n;
          for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum, o);
            if ((int)threadIdx.x >= o) sum += u;
          }
          if (e < p.E) p.offsets[e] = before + sum - n;
          before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (threadIdx.x == 0) p.offsets[p.E] = before;
      }
      __syncwarp();
    }
  }
  const int lane = threadIdx.x % G, warp_lane = threadIdx.x & 31;
  const int64_t end = p.rows_end ? min(p.T, (int64_t)__ldcg(p.rows_end)) : p.T;
  const int64_t stride = (int64_t)gridDim.x * (256 / G);
  const bool once = p.K <= G * CH * 8;
  // lane s of a warp: where the token's s-th copy goes
  auto places = [&](int64_t t) {
    if constexpr (PLAN) {
      int to = -1;
      for (int s = 0; s < p.top_k && t < end; ++s) {
        const int i = (int)t * p.top_k + s, e = expert[i];
        if (e < 0) continue;
        int n = 0;
        for (int j = warp_lane; j < n_pairs; j += 32) n += expert[j] >= 0 && (expert[j] < e || (expert[j] == e && j < i));
        n = __reduce_add_sync(0xffffffffu, n);
        if (warp_lane == s) to = n;
      }
      if (lane < p.top_k && t < end) p.place_out[t * p.top_k + lane] = to;
      return to;
    }
    return p.place ? (t < end && warp_lane < p.top_k ? p.place[t * p.top_k + warp_lane] : -1) : t < end ? 0 : -1;
  };
  const bool placed = PLAN || p.place;
  Eight<S> raw[CH];
  auto load = [&](int64_t t, int k0) {
    const S* row = static_cast<const S*>(p.x) + t * p.ldx;
#pragma unroll
    for (int c = 0; c < CH; ++c) raw[c] = eight_of<VEC>(row, k0 + (c * G + lane) * 8, p.K);
  };
  int turn = 0;
  int64_t t = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  int to = places(t), to_next = places(t + stride);
  unsigned copies = __ballot_sync(0xffffffffu, to >= 0);
  if (copies && once) load(t, 0);
  for (; t < end; t += stride) {
    const int to_after = places(t + 2 * stride);
    const unsigned copies_next = __ballot_sync(0xffffffffu, to_next >= 0);
    if (copies) {       // the same in all threads of the row
      uint32_t bits = 0;
      for (int k0 = 0; k0 < p.K; k0 += G * CH * 8) {
        if (!once) load(t, k0);
#pragma unroll
        for (int c = 0; c < CH; ++c) bits = max(bits, largest_bits(raw[c]));
      }
      bits = __reduce_max_sync(0xffffffffu, bits);
      if (G > 32) {
        constexpr int W = G / 32;
        if (warp_lane == 0) part[turn][threadIdx.x >> 5] = bits;
        asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.x / G + 1), "n"(G) : "memory");   // the row's threads
#pragma unroll
        for (int w = 0; w < W; ++w) bits = max(bits, part[turn][(int)threadIdx.x / G * W + w]);
        turn ^= 1;
      }
      const RowCodes code(bits);
      for (int k0 = 0; k0 < p.K; k0 += G * CH * 8) {
        if (!once) load(t, k0);
        uint2 word[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) word[c] = code.of(raw[c]);
        if (once && copies_next) load(t + stride, 0);
        for (unsigned left = copies; left; left &= left - 1) {
          const int64_t row = placed ? __shfl_sync(0xffffffffu, to, __ffs(left) - 1) : t;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const int k = k0 + (c * G + lane) * 8;
            int8_t* out = p.codes + row * p.ldc + k;
            if (VEC) {
              if (k < p.K) *reinterpret_cast<uint2*>(out) = word[c];
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (k + j < p.K) out[j] = (int8_t)((j < 4 ? word[c].x : word[c].y) >> (8 * (j & 3)));
            }
          }
          if (!placed) break;
        }
      }
      if (lane < 32) {
        if (placed) {
          if (to >= 0) p.scale[to] = code.scale;
        } else if (lane == 0) {
          p.scale[t] = code.scale;
        }
      }
    } else if (once && copies_next) {
      load(t + stride, 0);
    }
    to = to_next;
    to_next = to_after;
    copies = copies_next;
  }
}

template <int DT, bool PLAN>
int launch_rows(const RowsParams& p, bool vec, cudaStream_t st) {
#define MQ_ROWS(G, CH)                                                                                                      \
  do {                                                                                                                      \
    const int64_t blocks = ceil_div(p.T, 256 / G), most = 148 * rows_blocks(DT, CH);                                        \
    MQ_CUDA(launch_chained(true, vec ? quantize_rows_kernel<DT, G, CH, true, PLAN> : quantize_rows_kernel<DT, G, CH, false, PLAN>, \
                           dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, p));                          \
  } while (0)
  if (p.K <= 256) MQ_ROWS(32, 1);
  else if (p.K <= 512) MQ_ROWS(32, 2);
  else if (p.K <= 1024) MQ_ROWS(32, 4);
  else if (p.K <= 2048) MQ_ROWS(64, 4);
  else if (p.K <= 4096) MQ_ROWS(128, 4);
  else if (p.K <= 8192) MQ_ROWS(256, 4);
  else MQ_ROWS(256, 8);
#undef MQ_ROWS
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}

int quantize_rows(int dtype, RowsParams p, cudaStream_t st) {
  if (p.T == 0) return MQ_OK;
  const bool vec = p.K % 8 == 0 && aligned(p.x, 8 * dtype_size(dtype)) && p.ldx % 8 == 0 && aligned(p.codes, 8) && p.ldc % 8 == 0;
  if (p.ids) return dtype == MQ_BF16 ? launch_rows<MQ_BF16, true>(p, vec, st) : launch_rows<MQ_F16, true>(p, vec, st);
  if (dtype == MQ_F32) return launch_rows<MQ_F32, false>(p, vec, st);
  if (dtype == MQ_BF16) return launch_rows<MQ_BF16, false>(p, vec, st);
  return launch_rows<MQ_F16, false>(p, vec, st);
}

// ---------------------------------------------------------------- products
// y[t] = sum over the token's pairs, in the order of its slots, of weight * (the pair's down product).  The products are fp32 and short of the
// factor h_scale[pair] (INT8_PAIRS).  One block per token, eight columns a
// thread; smaller blocks for short rows (20000 tokens of 512, 2 of 8 experts: 115 us the whole call instead of 131 with 256 threads).
struct CombineParams {
  const float* pairs;
  int64_t ldp;
  const float *h_scale, *weights;
  const int32_t* place;
  int top_k, N;
  int64_t T;
  void* y;
  int64_t ldy;
};

template <int DT, bool VEC>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
  using S = typename StorageOf<DT>::type;
  __shared__ int row_of[2][32];
  __shared__ float factor_of[2][32];
  __shared__ int found[2];
  chain_wait();
  chain_release();
  int turn = 0;
  for (int64_t t = blockIdx.x; t < p.T; t += gridDim.x, turn ^= 1) {
    if (threadIdx.x < 32) {
      const int s = threadIdx.x;
      const int at = s < p.top_k ? __ldcg(p.place + t * p.top_k + s) : -1;
      const unsigned have = __ballot_sync(0xffffffffu, at >= 0);
      if (at >= 0) {
        const int i = __popc(have & ((1u << s) - 1u));
        row_of[turn][i] = at;
        factor_of[turn][i] = p.weights[t * p.top_k + s] * __ldcg(p.h_scale + at);
      }
      if (s == 0) found[turn] = __popc(have);
    }
    __syncthreads();
    const int n_pairs = found[turn];
    for (int n = threadIdx.x * 8; n < p.N; n += blockDim.x * 8) {
      float sum[8] = {};
#pragma unroll 2
      for (int i = 0; i < n_pairs; ++i) {
        const float f = factor_of[turn][i];
        // (rows of products have room for a multiple of sixteen)
        const Eight<float> a = *reinterpret_cast<const Eight<float>*>(p.pairs + (int64_t)row_of[turn][i] * p.ldp + n);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = fmaf(f, a.v[j], sum[j]);
      }
      S* out = static_cast<S*>(p.y) + t * p.ldy + n;
      if (VEC) {
        Eight<S> o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o.v[j] = from_float<S>(sum[j]);
        *reinterpret_cast<Eight<S>*>(out) = o;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (n + j < p.N) out[j] = from_float<S>(sum[j]);
      }
    }
  }
}

constexpr int64_t INT8_MAX_K = 131072;   // 127 * 128 * K stays below 2^31
constexpr int64_t ROWS_MAX_K = 1 << 30;  // quantize_rows_kernel counts columns in 32 bits, up to 32768 beyond the last

int64_t pitch_of(int64_t K) { return ceil_div(K, 16) * 16; }

}  // namespace
}  // namespace mq

using namespace mq;

extern "C" int mq_quantize_tokens(const void* x, int dtype, int64_t T, int64_t K, int64_t ldx, int8_t* codes, int64_t ldc, float* scale,
                                  void* stream) {
  MQ_REQUIRE(valid_dtype(dtype), MQ_ERR_ARGUMENT, "mq_quantize_tokens: unknown dtype %d", dtype);
  MQ_REQUIRE(T >= 0 && K >= 1 && ldx >= K && ldc >= K, MQ_ERR_ARGUMENT,
             "mq_quantize_tokens: bad sizes T=%lld K=%lld ldx=%lld ldc=%lld", (long long)T, (long long)K, (long long)ldx, (long long)ldc);
  MQ_REQUIRE(K <= ROWS_MAX_K, MQ_ERR_UNSUPPORTED, "mq_quantize_tokens: K is at most 2^30 (got %lld)", (long long)K);
  if (T == 0) return MQ_OK;
  MQ_REQUIRE(x && codes && scale, MQ_ERR_ARGUMENT, "mq_quantize_tokens: null pointer");
  return quantize_rows(dtype, RowsParams{x, ldx, T, nullptr, nullptr, 0, (int)K, codes, ldc, scale}, static_cast<cudaStream_t>(stream));
}

namespace mq {
namespace {
Int8Product dense_product(int64_t T, int64_t N, int64_t K) {
  Int8Product p = {};
  p.E = 1; p.rows = (int)N; p.K = (int)K; p.T = T;
  p.x_rows = T;
  return p;
}
}  // namespace
}  // namespace mq

extern "C" size_t mq_int8_matmul_workspace_bytes(int x_dtype, int64_t T, int64_t N, int64_t K) {
  if (T <= 0 || N <= 0 || K <= 0 || K > INT8_MAX_K || T >= (1ll << 31) - 256 || N >= (1ll << 31) - 256 || int8_few_fits(T, K)) return 0;
  const size_t codes = x_dtype == MQ_I8 ? 0 : align_up((size_t)T * (size_t)pitch_of(K), 256) + align_up((size_t)T * 4, 256);
  return codes + align_up(int8_umma_scratch_bytes(dense_product(T, N, K), INT8_Y), 256);
}

extern "C" int mq_int8_matmul(const void* x, int x_dtype, const float* x_scale, int64_t T, int64_t K, int64_t ldx, const int8_t* w, int64_t N,
                              int64_t ldw, const float* w_scale, const float* bias, int out_dtype, void* y, int64_t ldy, void* workspace,
                              size_t workspace_bytes, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  MQ_REQUIRE((valid_dtype(x_dtype) || x_dtype == MQ_I8) && valid_dtype(out_dtype), MQ_ERR_ARGUMENT, "mq_int8_matmul: unknown dtype %d or %d", x_dtype,
             out_dtype);
  MQ_REQUIRE(T >= 0 && N >= 0 && K >= 1 && ldx >= K && ldw >= K && ldy >= N, MQ_ERR_ARGUMENT,
             "mq_int8_matmul: bad sizes T=%lld N=%lld K=%lld ldx=%lld ldw=%lld ldy=%lld", (long long)T, (long long)N, (long long)K, (long long)ldx,
             (long long)ldw, (long long)ldy);
  // (codes of the caller's may all be -128)
  const int64_t most_k = x_dtype == MQ_I8 ? INT8_MAX_K - 1 : INT8_MAX_K;
  MQ_REQUIRE(K <= most_k, MQ_ERR_UNSUPPORTED, "mq_int8_matmul: K is at most %lld, so that a sum of products fits 32 bits (got %lld)",
             (long long)most_k, (long long)K);
  MQ_REQUIRE(T < (1ll << 31) - 256 && N < (1ll << 31) - 256, MQ_ERR_UNSUPPORTED, "mq_int8_matmul: too many tokens or rows");
  if (T == 0 || N == 0) return MQ_OK;
  MQ_REQUIRE(x && w && w_scale && y && (x_dtype != MQ_I8 || x_scale), MQ_ERR_ARGUMENT, "mq_int8_matmul: null pointer");
  MQ_REQUIRE(aligned(w, 16) && ldw % 16 == 0 && (x_dtype != MQ_I8 || (aligned(x, 16) && ldx % 16 == 0)), MQ_ERR_ALIGNMENT,
             "mq_int8_matmul: rows of 8-bit codes must start on 16-byte boundaries");
  const size_t need = mq_int8_matmul_workspace_bytes(x_dtype, T, N, K);
  MQ_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), MQ_ERR_WORKSPACE,
             "mq_int8_matmul: the workspace has %zu bytes and needs %zu", workspace_bytes, need);
  Int8Product p = dense_product(T, N, K);
  p.x_scale = x_scale;
  p.w = w; p.ldw = ldw; p.w_scale = w_scale;
  const Int8Out o = {INT8_Y, out_dtype, y, ldy, bias};
  if (int8_few_fits(T, K)) return int8_few(x, x_dtype, ldx, p, o, st);
  Workspace ws(workspace, workspace_bytes);
  const size_t n_sums = int8_umma_scratch_bytes(p, INT8_Y);
  char* sums = n_sums ? ws.take<char>(n_sums) : nullptr;
  if (x_dtype == MQ_I8) {
    p.x = static_cast<const int8_t*>(x);
    p.ldx = ldx;
  } else {
    int8_t* codes = ws.take<int8_t>((size_t)T * pitch_of(K));
    float* scale = ws.take<float>((size_t)T);
    MQ_TRY(quantize_rows(x_dtype, RowsParams{x, ldx, T, nullptr, nullptr, 0, (int)K, codes, pitch_of(K), scale}, st));
    p.x = codes;
    p.ldx = pitch_of(K);
    p.x_scale = scale;
  }
  return int8_product_umma(p, o, sums, st);
}

namespace mq {
namespace {
struct ExpertsBuffers {
  int32_t *offsets, *order, *place;
  void* plan;
  int8_t *x_codes, *h_codes;
  float *x_scale, *h_scale, *h, *pairs;
};
// Carves the buffers out of ws, or adds up their bytes where there is none.  The products of the pairs take the place of the tokens'
// codes and of the gated values, which have been read by then.
size_t experts_buffers(int64_t T, int k, int E, int64_t K, int64_t I, Workspace* ws, ExpertsBuffers* b) {
  const size_t P = (size_t)T * k;
  size_t total = 0;
  auto take = [&](size_t bytes) -> char* {
    bytes = align_up(bytes, 256);
    total += bytes;
    return ws ? ws->take<char>(bytes) : nullptr;
  };
  ExpertsBuffers x;
  x.offsets = reinterpret_cast<int32_t*>(take((size_t)(E + 1) * 4));
  x.order = reinterpret_cast<int32_t*>(take(P * 4));
  x.place = reinterpret_cast<int32_t*>(take(P * 4));
  x.plan = take(mq_expert_plan_workspace_bytes((int64_t)P, E));
  x.x_scale = reinterpret_cast<float*>(take(P * 4));
  x.h_scale = reinterpret_cast<float*>(take(P * 4));
  x.h_codes = reinterpret_cast<int8_t*>(take(P * (size_t)pitch_of(I)));
  const size_t codes = align_up(P * (size_t)pitch_of(K), 256), h = align_up(P * (size_t)pitch_of(I) * 4, 256), pairs = align_up(P * (size_t)pitch_of(K) * 4, 256);
  char* shared = take(codes + h > pairs ? codes + h : pairs);
  x.x_codes = reinterpret_cast<int8_t*>(shared);
  x.h = reinterpret_cast<float*>(shared + codes);
  x.pairs = reinterpret_cast<float*>(shared);
  if (b) *b = x;
  return total;
}

template <int DT>
int launch_combine(const CombineParams& p, cudaStream_t st) {
  const bool vec = p.N % 8 == 0 && p.ldy % 8 == 0 && aligned(p.y, 16);
  const int threads = p.N <= 512 ? 64 : p.N <= 1024 ? 128 : 256;
  const int64_t most = 148 * 4096 / threads;
  MQ_CUDA(launch_chained(true, vec ? combine_kernel<DT, true> : combine_kernel<DT, false>, dim3((unsigned)(p.T < most ? p.T : most)), dim3(threads), 0, st, p));
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}
}  // namespace
}  // namespace mq

extern "C" size_t mq_int8_experts_workspace_bytes(int /*dtype*/, int64_t T, int top_k, int64_t E, int64_t K, int64_t I) {
  return experts_buffers(T, top_k, (int)E, K, I, nullptr, nullptr);
}

extern "C" int mq_int8_experts(const void* x, int dtype, int64_t T, int64_t K, int64_t ldx, const int32_t* ids, const float* weights, int top_k,
                               int64_t first, int64_t E, int64_t I, const int8_t* gate_up, int64_t ld_gate_up, int64_t gate_up_expert,
                               const float* gate_up_scale, const int8_t* down, int64_t ld_down, int64_t down_expert, const float* down_scale,
                               void* y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  MQ_REQUIRE(dtype == MQ_BF16 || dtype == MQ_F16, MQ_ERR_ARGUMENT, "mq_int8_experts: tokens are bf16 or fp16 (got dtype %d)", dtype);
  MQ_REQUIRE(T >= 0 && K >= 1 && I >= 1 && E >= 1 && top_k >= 1 && top_k <= 32 && first >= 0 && first < (1ll << 31) - E && ldx >= K && ldy >= K &&
                 ld_gate_up >= K && ld_down >= I && gate_up_expert >= 0 && down_expert >= 0,
             MQ_ERR_ARGUMENT, "mq_int8_experts: bad sizes T=%lld K=%lld I=%lld E=%lld top_k=%d first=%lld", (long long)T, (long long)K, (long long)I,
             (long long)E, top_k, (long long)first);
  MQ_REQUIRE(K <= INT8_MAX_K && I <= INT8_MAX_K, MQ_ERR_UNSUPPORTED, "mq_int8_experts: K and I are at most %lld, so that a sum of products fits 32 bits",
             (long long)INT8_MAX_K);
  MQ_REQUIRE(E <= 1024 && T * top_k < (1ll << 31) - (1 << 20), MQ_ERR_UNSUPPORTED, "mq_int8_experts: at most 1024 experts and 2^31 - 2^20 pairs");
  if (T == 0) return MQ_OK;
  MQ_REQUIRE(x && ids && weights && gate_up && gate_up_scale && down && down_scale && y, MQ_ERR_ARGUMENT, "mq_int8_experts: null pointer");
  MQ_REQUIRE(aligned(gate_up, 16) && aligned(down, 16) && ld_gate_up % 16 == 0 && ld_down % 16 == 0 && gate_up_expert % 16 == 0 && down_expert % 16 == 0,
             MQ_ERR_ALIGNMENT, "mq_int8_experts: rows of 8-bit codes must start on 16-byte boundaries");
  const size_t need = mq_int8_experts_workspace_bytes(dtype, T, top_k, E, K, I);
  MQ_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= need, MQ_ERR_WORKSPACE, "mq_int8_experts: the workspace has %zu bytes and needs %zu",
             workspace_bytes, need);
  Workspace ws(workspace, workspace_bytes);
  ExpertsBuffers b;
  experts_buffers(T, top_k, (int)E, K, I, &ws, &b);
  const int64_t P = T * top_k;
  Int8Product up = {}, dn = {};
  up.w = gate_up; up.ldw = ld_gate_up; up.w_expert = gate_up_expert; up.w_scale = gate_up_scale;
  up.E = (int)E; up.rows = (int)I; up.K = (int)K; up.T = P;
  dn.w = down; dn.ldw = ld_down; dn.w_expert = down_expert; dn.w_scale = down_scale;
  dn.E = (int)E; dn.rows = (int)K; dn.K = (int)I; dn.T = P;
  if (T == 1 && int8_one_token_fits(top_k, K, I)) return int8_one_token(x, dtype, ids, weights, top_k, (int)first, up, dn, b.h, y, st);
  // the tokens' codes, once for each of their pairs, where the plan has them
  RowsParams rows = {x, ldx, T, nullptr, nullptr, top_k, (int)K, b.x_codes, pitch_of(K), b.x_scale};
  if (P <= PLAN_PAIRS) {
    rows.ids = ids;
    rows.E = (int)E;
    rows.first = (int)first;
    rows.place_out = b.place;
    rows.offsets = b.offsets;
  } else {
    MQ_TRY(expert_plan(ids, P, (int)E, (int)first, b.offsets, b.order, b.place, b.plan, st));
    rows.place = b.place;
  }
  MQ_TRY(quantize_rows(dtype, rows, st));
  up.x = b.x_codes; up.ldx = pitch_of(K); up.x_rows = P; up.x_scale = b.x_scale; up.offsets = b.offsets;
  MQ_TRY(int8_product_umma(up, Int8Out{INT8_GATED, MQ_F32, b.h, pitch_of(I), nullptr}, nullptr, st));
  MQ_TRY(quantize_rows(MQ_F32, RowsParams{b.h, pitch_of(I), P, b.offsets + E, nullptr, 0, (int)I, b.h_codes, pitch_of(I), b.h_scale}, st));
  dn.x = b.h_codes; dn.ldx = pitch_of(I); dn.x_rows = P; dn.x_scale = b.h_scale; dn.offsets = b.offsets;
  MQ_TRY(int8_product_umma(dn, Int8Out{INT8_PAIRS, MQ_F32, b.pairs, pitch_of(K), nullptr}, nullptr, st));
  const CombineParams c = {b.pairs, pitch_of(K), b.h_scale, weights, b.place, top_k, (int)K, T, y, ldy};
  return dtype == MQ_BF16 ? launch_combine<MQ_BF16>(c, st) : launch_combine<MQ_F16>(c, st);
}
