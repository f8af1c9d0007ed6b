// Products in 8-bit integers with one scale per token and one per output channel, and the experts' gated MLPs made of them.
//
//   codes of a token  scale = max|x| / 127, code = round_half_even(127 x / max|x|);  a token with an infinity or a NaN has the scale
//                     NaN and codes of zero, so its whole result is NaN
//   product           y[t, n] = (sum_k code[t, k] w[n, k]) scale[t] w_scale[n] + bias[n], the sum in 32-bit integers: exact
//   experts           h = silu(gate product) * up product per pair of token and expert, codes of h as above, and
//                     y[t] = sum over the token's pairs of weight * down product
#include <math_constants.h>

#include "int8.cuh"
#include "profile.cuh"

namespace mq {

int expert_plan(const int32_t* ids, int64_t pairs, int E, int first, int32_t* offsets, int32_t* order, int32_t* place, void* workspace,
                cudaStream_t st);

namespace {

// ---------------------------------------------------------------- codes of tokens
// code = round_half_even(127 x / top).  The product with 127 / top is off by less than 2.4e-5 of a code (three roundings of a number
// up to 127); where that could decide between two codes, the quotient is formed in 64 bits, whose error of 127 * 2^-53 is below
// the distance of any quotient of two fp32 numbers from a middle that it does not equal (at least 2^-25 / 254).
__device__ __forceinline__ float code_of(float x, float top, float inv) {
  const float q = x * inv;
  float r = rintf(q);
  if (fabsf(q - r) > 0.4999f) r = (float)rint(127.0 * (double)x / (double)top);
  return r;
}

template <typename T>
struct alignas(8 * sizeof(T)) Eight { T v[8]; };
struct alignas(8) EightCodes { int8_t v[8]; };

// G lanes per row (32, or the whole block), eight values per lane and step.  The row is read twice, the second time from the L1/L2.
template <int DT, int G, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int64_t T, const int32_t* __restrict__ rows_end,
                                                            int K, int8_t* __restrict__ codes, int64_t ldc, float* __restrict__ scale) {
  using S = typename StorageOf<DT>::type;
  __shared__ float part[8];
  const int64_t t = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const int lane = threadIdx.x % G;
  const int64_t end = rows_end ? min(T, (int64_t)*rows_end) : T;
  if (G == 256 ? t >= end : false) return;
  const bool in = t < end;
  const S* row = static_cast<const S*>(x) + (in ? t : 0) * ldx;
  float top = 0.0f;
  bool broken = false;
  if (in) {
    for (int k = lane * 8; k < K; k += G * 8) {
      float v[8];
      if (VEC) {
        const Eight<S> a = *reinterpret_cast<const Eight<S>*>(row + k);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_float(a.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < K ? to_float(row[k + j]) : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        broken |= !(fabsf(v[j]) < CUDART_INF_F);
        top = fmaxf(top, fabsf(v[j]));
      }
    }
  }
  if (broken) top = CUDART_INF_F;
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (G == 256) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, part[w]);
  }
  if (!in) return;
  if (lane == 0) scale[t] = top < CUDART_INF_F ? top / 127.0f : CUDART_NAN_F;
  // tiny rows are lifted (exactly) so that 127 / top stays finite
  const float lift = top < 0x1p-100f ? 0x1p60f : 1.0f;
  const bool plain = top > 0.0f && top < CUDART_INF_F;
  top *= lift;
  const float inv = plain ? 127.0f / top : 0.0f;
  int8_t* out = codes + t * ldc;
  for (int k = lane * 8; k < K; k += G * 8) {
    EightCodes c;
    if (VEC) {
      const Eight<S> a = *reinterpret_cast<const Eight<S>*>(row + k);
#pragma unroll
      for (int j = 0; j < 8; ++j) c.v[j] = plain ? (int8_t)code_of(to_float(a.v[j]) * lift, top, inv) : (int8_t)0;
      *reinterpret_cast<EightCodes*>(out + k) = c;
    } else {
      for (int j = 0; j < 8 && k + j < K; ++j) out[k + j] = plain ? (int8_t)code_of(to_float(row[k + j]) * lift, top, inv) : (int8_t)0;
    }
  }
}

int quantize_rows(const void* x, int dtype, int64_t T, const int32_t* rows_end, int64_t K, int64_t ldx, int8_t* codes, int64_t ldc, float* scale,
                  cudaStream_t st) {
  if (T == 0) return MQ_OK;
  const size_t size = dtype_size(dtype);
  const bool vec = K % 8 == 0 && aligned(x, 8 * size) && ldx % 8 == 0 && aligned(codes, 8) && ldc % 8 == 0;
  const bool warp_rows = K <= 1024;
  const int64_t blocks = warp_rows ? ceil_div(T, 8) : T;
  MQ_REQUIRE(blocks < (1ll << 31), MQ_ERR_UNSUPPORTED, "too many rows to quantize (%lld)", (long long)T);
#define MQ_ROWS(DT, G, V) quantize_rows_kernel<DT, G, V><<<(unsigned)blocks, 256, 0, st>>>(x, ldx, T, rows_end, (int)K, codes, ldc, scale)
#define MQ_ROWS_OF(DT)                                   \
  do {                                                   \
    if (warp_rows) { if (vec) MQ_ROWS(DT, 32, true); else MQ_ROWS(DT, 32, false); } \
    else { if (vec) MQ_ROWS(DT, 256, true); else MQ_ROWS(DT, 256, false); }         \
  } while (0)
  if (dtype == MQ_F32) MQ_ROWS_OF(MQ_F32);
  else if (dtype == MQ_BF16) MQ_ROWS_OF(MQ_BF16);
  else MQ_ROWS_OF(MQ_F16);
#undef MQ_ROWS_OF
#undef MQ_ROWS
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}

// ---------------------------------------------------------------- products
int int8_product(const Int8Product& p, const Int8Out& o, cudaStream_t st) {
  if (p.T == 0 || p.rows == 0) return MQ_OK;
  return int8_product_umma(p, o, st);
}

// y[t] = sum over the token's pairs, in the order of its slots, of weight * (the pair's down product)
template <int DT>
__global__ void __launch_bounds__(256) combine_kernel(const float* __restrict__ pairs, int64_t ldp, const int32_t* __restrict__ place,
                                                      const float* __restrict__ weights, int k, int N, void* __restrict__ y, int64_t ldy) {
  const int64_t t = blockIdx.x;
  auto* out = static_cast<typename StorageOf<DT>::type*>(y) + t * ldy;
  for (int n = threadIdx.x; n < N; n += 256) {
    float sum = 0.0f;
    for (int s = 0; s < k; ++s) {
      const int at = place[t * k + s];
      if (at >= 0) sum = fmaf(weights[t * k + s], pairs[(int64_t)at * ldp + n], sum);
    }
    out[n] = from_float<typename StorageOf<DT>::type>(sum);
  }
}

constexpr int64_t INT8_MAX_K = 131072;   // 127 * 128 * K stays below 2^31

int64_t pitch_of(int64_t K) { return ceil_div(K, 16) * 16; }

}  // namespace
}  // namespace mq

using namespace mq;

extern "C" int mq_quantize_tokens(const void* x, int dtype, int64_t T, int64_t K, int64_t ldx, int8_t* codes, int64_t ldc, float* scale,
                                  void* stream) {
  MQ_REQUIRE(valid_dtype(dtype), MQ_ERR_ARGUMENT, "mq_quantize_tokens: unknown dtype %d", dtype);
  MQ_REQUIRE(T >= 0 && K >= 1 && K < (1ll << 31) && ldx >= K && ldc >= K, MQ_ERR_ARGUMENT,
             "mq_quantize_tokens: bad sizes T=%lld K=%lld ldx=%lld ldc=%lld", (long long)T, (long long)K, (long long)ldx, (long long)ldc);
  if (T == 0) return MQ_OK;
  MQ_REQUIRE(x && codes && scale, MQ_ERR_ARGUMENT, "mq_quantize_tokens: null pointer");
  return quantize_rows(x, dtype, T, nullptr, K, ldx, codes, ldc, scale, static_cast<cudaStream_t>(stream));
}

extern "C" size_t mq_int8_matmul_workspace_bytes(int x_dtype, int64_t T, int64_t N, int64_t K) {
  (void)N;
  if (x_dtype == MQ_I8) return 0;
  return align_up((size_t)T * (size_t)pitch_of(K), 256) + align_up((size_t)T * 4, 256);
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
  MQ_REQUIRE(K <= INT8_MAX_K, MQ_ERR_UNSUPPORTED, "mq_int8_matmul: K is at most %lld, so that a sum of products fits 32 bits (got %lld)",
             (long long)INT8_MAX_K, (long long)K);
  MQ_REQUIRE(T < (1ll << 31) - 256 && N < (1ll << 31) - 256, MQ_ERR_UNSUPPORTED, "mq_int8_matmul: too many tokens or rows");
  if (T == 0 || N == 0) return MQ_OK;
  MQ_REQUIRE(x && w && w_scale && y && (x_dtype != MQ_I8 || x_scale), MQ_ERR_ARGUMENT, "mq_int8_matmul: null pointer");
  MQ_REQUIRE(aligned(w, 16) && ldw % 16 == 0 && (x_dtype != MQ_I8 || (aligned(x, 16) && ldx % 16 == 0)), MQ_ERR_ALIGNMENT,
             "mq_int8_matmul: rows of 8-bit codes must start on 16-byte boundaries");
  const size_t need = mq_int8_matmul_workspace_bytes(x_dtype, T, N, K);
  MQ_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), MQ_ERR_WORKSPACE,
             "mq_int8_matmul: the workspace has %zu bytes and needs %zu", workspace_bytes, need);
  Int8Product p = {};
  if (x_dtype == MQ_I8) {
    p.x = static_cast<const int8_t*>(x);
    p.ldx = ldx;
    p.x_scale = x_scale;
  } else {
    Workspace ws(workspace, workspace_bytes);
    int8_t* codes = ws.take<int8_t>((size_t)T * pitch_of(K));
    float* scale = ws.take<float>((size_t)T);
    MQ_TRY(quantize_rows(x, x_dtype, T, nullptr, K, ldx, codes, pitch_of(K), scale, st));
    p.x = codes;
    p.ldx = pitch_of(K);
    p.x_scale = scale;
  }
  p.x_rows = T;
  p.w = w; p.ldw = ldw; p.w_expert = 0; p.w_scale = w_scale;
  p.E = 1; p.rows = (int)N; p.K = (int)K; p.T = T; p.top_k = 1;
  return int8_product(p, Int8Out{INT8_Y, out_dtype, y, ldy, bias}, st);
}

namespace mq {
namespace {
struct ExpertsBuffers {
  int32_t *offsets, *order, *place;
  void* plan;
  int8_t *x_codes, *h_codes;
  float *x_scale, *h_scale, *h, *pairs;
};
// carves the buffers out of ws, or adds up their bytes where it has no base
size_t experts_buffers(int64_t T, int k, int E, int64_t K, int64_t I, Workspace* ws, ExpertsBuffers* b) {
  const size_t P = (size_t)T * k;
  size_t total = 0;
  auto take = [&](size_t bytes) -> void* {
    bytes = align_up(bytes, 256);
    total += bytes;
    return ws ? ws->take<char>(bytes) : nullptr;
  };
  ExpertsBuffers x;
  x.offsets = static_cast<int32_t*>(take((size_t)(E + 1) * 4));
  x.order = static_cast<int32_t*>(take(P * 4));
  x.place = static_cast<int32_t*>(take(P * 4));
  x.plan = take(mq_expert_plan_workspace_bytes((int64_t)P, E));
  x.x_codes = static_cast<int8_t*>(take((size_t)T * pitch_of(K)));
  x.x_scale = static_cast<float*>(take((size_t)T * 4));
  x.h = static_cast<float*>(take(P * (size_t)I * 4));
  x.h_codes = static_cast<int8_t*>(take(P * (size_t)pitch_of(I)));
  x.h_scale = static_cast<float*>(take(P * 4));
  x.pairs = static_cast<float*>(take(P * (size_t)K * 4));
  if (b) *b = x;
  return total;
}
}  // namespace
}  // namespace mq

extern "C" size_t mq_int8_experts_workspace_bytes(int64_t T, int top_k, int64_t E, int64_t K, int64_t I) {
  return experts_buffers(T, top_k, (int)E, K, I, nullptr, nullptr);
}

extern "C" int mq_int8_experts(const void* x, int dtype, int64_t T, int64_t K, int64_t ldx, const int32_t* ids, const float* weights, int top_k,
                               int64_t first, int64_t E, int64_t I, const int8_t* gate_up, int64_t ld_gate_up, int64_t gate_up_expert,
                               const float* gate_up_scale, const int8_t* down, int64_t ld_down, int64_t down_expert, const float* down_scale,
                               void* y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  MQ_REQUIRE(dtype == MQ_BF16 || dtype == MQ_F16, MQ_ERR_ARGUMENT, "mq_int8_experts: tokens are bf16 or fp16 (got dtype %d)", dtype);
  MQ_REQUIRE(T >= 0 && K >= 1 && I >= 1 && E >= 1 && top_k >= 1 && top_k <= 32 && first >= 0 && first < (1ll << 31) && ldx >= K && ldy >= K &&
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
  const size_t need = mq_int8_experts_workspace_bytes(T, top_k, E, K, I);
  MQ_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= need, MQ_ERR_WORKSPACE, "mq_int8_experts: the workspace has %zu bytes and needs %zu",
             workspace_bytes, need);
  Workspace ws(workspace, workspace_bytes);
  ExpertsBuffers b;
  experts_buffers(T, top_k, (int)E, K, I, &ws, &b);
  const int64_t P = T * top_k;
  MQ_TRY(expert_plan(ids, P, (int)E, (int)first, b.offsets, b.order, b.place, b.plan, st));
  MQ_TRY(quantize_rows(x, dtype, T, nullptr, K, ldx, b.x_codes, pitch_of(K), b.x_scale, st));
  Int8Product p = {};
  p.x = b.x_codes; p.ldx = pitch_of(K); p.x_rows = T; p.x_scale = b.x_scale;
  p.w = gate_up; p.ldw = ld_gate_up; p.w_expert = gate_up_expert; p.w_scale = gate_up_scale;
  p.E = (int)E; p.rows = (int)I; p.K = (int)K; p.T = P; p.offsets = b.offsets; p.order = b.order; p.top_k = top_k;
  MQ_TRY(int8_product(p, Int8Out{INT8_GATED, MQ_F32, b.h, I, nullptr}, st));
  MQ_TRY(quantize_rows(b.h, MQ_F32, P, b.offsets + E, I, I, b.h_codes, pitch_of(I), b.h_scale, st));
  p.x = b.h_codes; p.ldx = pitch_of(I); p.x_rows = P; p.x_scale = b.h_scale;
  p.w = down; p.ldw = ld_down; p.w_expert = down_expert; p.w_scale = down_scale;
  p.rows = (int)K; p.K = (int)I; p.order = nullptr;
  MQ_TRY(int8_product(p, Int8Out{INT8_PAIRS, MQ_F32, b.pairs, K, nullptr}, st));
  if (dtype == MQ_BF16) combine_kernel<MQ_BF16><<<(unsigned)T, 256, 0, st>>>(b.pairs, K, b.place, weights, top_k, (int)K, y, ldy);
  else combine_kernel<MQ_F16><<<(unsigned)T, 256, 0, st>>>(b.pairs, K, b.place, weights, top_k, (int)K, y, ldy);
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}
