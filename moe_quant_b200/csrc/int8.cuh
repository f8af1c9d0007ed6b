// What the kernels of the 8-bit integer products share (int8.cu).
#pragma once

#include "common.cuh"
#include "mbarrier.cuh"

namespace mq {

// One product of tokens with weights, both 8-bit codes, or one per expert.
//   dense   : E == 1, offsets == nullptr, rows 0 .. T - 1 of x
//   experts : rows offsets[e] .. offsets[e + 1] - 1 of x belong to expert e
// Weights are (E, rows, K) with strides w_expert and ldw (bytes), scales (E, rows); for INT8_GATED (E, 2 rows, K) and (E, 2 rows).
struct Int8Product {
  const int8_t* x;
  int64_t ldx;
  int64_t x_rows;          // rows that x has
  const float* x_scale;    // per row of x
  const int8_t* w;
  int64_t ldw, w_expert;
  const float* w_scale;
  int E, rows, K;
  int64_t T;               // rows of the result: tokens, or at most this many pairs
  const int32_t* offsets;
};

// where the sums go
enum Int8Result {
  INT8_Y = 0,      // y = sum * x_scale * w_scale + bias, in the result's type
  INT8_GATED = 1,  // weights are gate rows and up rows, `rows` of either: h = silu(gate) * up, fp32
  // The products of the pairs, short of x_scale: sum * w_scale in fp32.  (In fp16 they would be half the bytes, but their 11 bits
  // show beside the 8 of a bf16 result: they moved it by 1e-3 of its norm, its own rounding by 1.7e-3.)
  INT8_PAIRS = 2,
  INT8_SUMS = 3,   // the sums themselves, of a share of k (within int8_umma.cu)
};

struct Int8Out {
  int kind, dtype;
  void* y;
  int64_t ldy;
  const float* bias;
};

// The result with its bias, two roundings in every kernel (a fused sum in some of them would make a token's result depend on how many
// others are in the call).
__device__ __forceinline__ float plus_bias(float v, float bias) { return __fadd_rn(v, bias); }
// silu(g) u, the same in every kernel: a token's result does not depend on how many others are in the call.  (With __expf and __fdividef the exponential
// is off by 1.2 |g| steps more.)
__device__ __forceinline__ float gated(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// On the tensor cores (int8_umma.cu).  `scratch`: int8_umma_scratch_bytes bytes on a 16-byte boundary, or NULL (then no tile's k is shared
// among CTAs).
size_t int8_umma_scratch_bytes(const Int8Product& p, int kind);
int int8_product_umma(const Int8Product& p, const Int8Out& o, void* scratch, cudaStream_t st);

// A few tokens (int8_few.cu): x of any type, codes made on the way (p.x is not read; p.x_scale for MQ_I8 alone).
constexpr int64_t INT8_FEW_TOKENS = 4;
bool int8_few_fits(int64_t T, int64_t K);
int int8_few(const void* x, int dtype, int64_t ldx, const Int8Product& p, const Int8Out& o, cudaStream_t st);
// The experts of one token, without a plan; h holds top_k rows of up.rows numbers.
bool int8_one_token_fits(int top_k, int64_t K, int64_t I);
int int8_one_token(const void* x, int dtype, const int32_t* ids, const float* weights, int top_k, int first, const Int8Product& up,
                   const Int8Product& down, float* h, void* y, cudaStream_t st);

// Once per device: the word that waits record their codes in.  (Looking it up in every call, and asking for shared memory in each, cost 2 us
// of the 6 of a call.)
inline int fault_word(int** out) {
  static int* word[64] = {};
  int dev = 0;
  MQ_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return engine_fault_word(out);
  if (!word[dev]) MQ_TRY(engine_fault_word(&word[dev]));
  *out = word[dev];
  return MQ_OK;
}

}  // namespace mq
