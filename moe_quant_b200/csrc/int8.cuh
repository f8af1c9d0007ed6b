// What the kernels of the 8-bit integer products share (int8.cu).
#pragma once

#include "common.cuh"

namespace mq {

// One product of tokens with weights, both 8-bit codes, or one per expert.
//   dense   : E == 1, offsets == nullptr, rows of x are tokens 0 .. T - 1
//   experts : rows offsets[e] .. offsets[e + 1] - 1 belong to expert e; row i of x is row i itself, or, where `order` is given,
//             token order[i] / top_k
// Weights are (E, rows, K) with strides w_expert and ldw (bytes), scales (E, rows).
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
  const int32_t* order;
  int top_k;
};

// where the sums go
enum Int8Result {
  INT8_Y = 0,      // y = sum * x_scale * w_scale + bias, in the result's type
  INT8_GATED = 1,  // weights are gate rows and up rows, `rows` of either: h = silu(gate) * up, fp32
  INT8_PAIRS = 2,  // sum * x_scale * w_scale of each pair, fp32
};

struct Int8Out {
  int kind, dtype;
  void* y;
  int64_t ldy;
  const float* bias;
};

int int8_product_umma(const Int8Product& p, const Int8Out& o, cudaStream_t st);   // on the tensor cores (int8_umma.cu)

}  // namespace mq
