// 8-bit integer products of a few tokens: the weights are read once and bound the time.
//
// Every block holds the codes of all tokens in shared memory (it rounds them itself: they are few, and the first weights are on their way
// meanwhile) and takes a run of weight rows, a row per warp.  Rows come through a ring of pieces of 2 KB that each warp keeps by
// bulk copies: 128 KB per SM under way.  (Eight 16-byte loads per lane, 64 KB, gave 5.0 TB/s on the gate and up rows of one
// token's eight experts, and fetching rows into the L2 ahead of them less still.)  A lane multiplies 16 weights at a time with the tokens'
// codes (dp4a); the warp's sums come together in one reduction.
#include <math_constants.h>

#include "int8.cuh"
#include "int8_codes.cuh"
#include "mbarrier.cuh"
#include "profile.cuh"

namespace mq {
namespace {

// A layer's kernel has 16 warps of four slots each; the experts' kernels, which go through 20 times as many rows per SM, 32 of two: one
// token through 2048 x 7168 takes 4.8 / 5.3 us with 16 / 32 warps, its eight experts 68.5 / 63.4.
constexpr int FEW_THREADS = 512, FEW_WARPS = FEW_THREADS / 32, FEW_SLOTS = 4, FEW_BLOCKS = 148;
constexpr int ONE_THREADS = 1024, ONE_WARPS = ONE_THREADS / 32, ONE_SLOTS = 2;
constexpr int FEW_PIECE = 2048, FEW_RINGS = FEW_WARPS * FEW_SLOTS * FEW_PIECE;
static_assert(FEW_RINGS == ONE_WARPS * ONE_SLOTS * FEW_PIECE, "the same bytes under way");
constexpr size_t FEW_SMEM = 208 * 1024, FEW_CODES = FEW_SMEM - (size_t)FEW_RINGS;   // in front of the rings: codes

// bytes that a token's codes take: a whole number of steps of a warp, zeros behind the end
__host__ __device__ __forceinline__ int few_pitch(int K) { return (K + 511) / 512 * 512; }

// 16 codes of a row from byte k on; zeros behind its end
__device__ __forceinline__ int4 codes16(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return *reinterpret_cast<const int4*>(row + k);
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

// The weight rows of one warp, one after the other, through its ring.  Slots are refilled in the order in which they are emptied.
template <int SLOTS>
struct RowStream {
  uint32_t ring, bars;
  int lane, n_rows, K, whole;          // `whole`: bytes of a row that are copied, a multiple of 16; up to 15 more are read directly
  int next_row, next_at, next_slot;    // what is copied next, and where to
  const int8_t* from;                  // the row that is being copied
  int slot;
  uint32_t parity;
  int under_way;
  int* fault;
  bool ok;
  __device__ __forceinline__ RowStream(uint32_t ring_, uint32_t bars_, int lane_, int n_rows_, int K_, int* fault_)
      : ring(ring_), bars(bars_), lane(lane_), n_rows(n_rows_), K(K_), whole(K_ & ~15), next_row(0), next_at(0), next_slot(0), from(nullptr), slot(0), parity(0),
        under_way(0), fault(fault_), ok(true) {}
  template <typename RowOf>
  __device__ __forceinline__ void copy_next(RowOf row_of) {
    if (next_row >= n_rows || whole == 0) return;
    const int bytes = min(FEW_PIECE, whole - next_at);
    if (next_at == 0) from = row_of(next_row);
    if (lane == 0) {
      const uint32_t bar = bars + 8 * next_slot;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                   ::"r"(ring + (uint32_t)(next_slot * FEW_PIECE)), "l"(from + next_at), "r"(bytes), "r"(bar) : "memory");
    }
    ++under_way;
    next_slot = next_slot + 1 == SLOTS ? 0 : next_slot + 1;
    next_at += FEW_PIECE;
    if (next_at >= whole) {
      next_at = 0;
      ++next_row;
    }
  }
  template <typename RowOf>
  __device__ __forceinline__ void start(RowOf row_of) {
    for (int i = 0; i < SLOTS; ++i) copy_next(row_of);
  }
  // use(k, 16 weights from byte k on) for this lane's share of row r, the r-th call
  template <typename RowOf, typename Use>
  __device__ __forceinline__ void row(int r, RowOf row_of, Use use) {
    for (int at = 0; at < whole && ok; at += FEW_PIECE) {
      ok = mbar_wait(bars + 8 * slot, parity, fault, 97);
      if (!ok) return;
      --under_way;
      const uint32_t src = ring + (uint32_t)(slot * FEW_PIECE + lane * 16);
#pragma unroll
      for (int i = 0; i < FEW_PIECE / 512; ++i) {
        const int k = at + i * 512 + lane * 16;
        if (k < whole) {
          int4 w;
          asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(src + i * 512) : "memory");
          use(k, w);
        }
      }
      __syncwarp();      // all lanes have read the slot
      slot = slot + 1 == SLOTS ? 0 : slot + 1;
      if (slot == 0) parity ^= 1;
      copy_next(row_of);
    }
    if (whole < K && lane == 0) use(whole, codes16(row_of(r), whole, K));
  }
  // after a wait that ran out: the copies that are still under way come to their end first
  __device__ __forceinline__ void end() {
    if (ok) return;
    for (; under_way > 0; --under_way) {
      const uint64_t t0 = global_ns();
      while (!mbar_try(bars + 8 * slot, parity))
        if (global_ns() - t0 > 100000000ull) break;
      slot = slot + 1 == SLOTS ? 0 : slot + 1;
      if (slot == 0) parity ^= 1;
    }
  }
};

// by one thread of the block, before any warp's stream starts
template <int WARPS, int SLOTS>
__device__ __forceinline__ void init_bars(uint64_t (&bars)[WARPS][SLOTS]) {
  for (int w = 0; w < WARPS; ++w)
    for (int s = 0; s < SLOTS; ++s) mbar_init(smem_u32(&bars[w][s]), 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
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
  int* fault;
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
  extern __shared__ __align__(128) int8_t few_codes[];
  __shared__ uint64_t bars[FEW_WARPS][FEW_SLOTS];
  __shared__ uint32_t part[NT][FEW_WARPS];
  __shared__ float x_scale[NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pitch = few_pitch(p.K);
  const int begin = (int)((int64_t)p.N * blockIdx.x / gridDim.x), end = (int)((int64_t)p.N * (blockIdx.x + 1) / gridDim.x);
  if (threadIdx.x == 0) init_bars(bars);
  __syncthreads();
  chain_wait();
  chain_release();
  const int first = begin + warp;
  auto row_of = [&](int r) { return p.w + (int64_t)(first + r * FEW_WARPS) * p.ldw; };
  RowStream<FEW_SLOTS> stream(smem_u32(few_codes) + (uint32_t)(NT * pitch + warp * FEW_SLOTS * FEW_PIECE), smem_u32(&bars[warp][0]), lane,
                   first < end ? (end - first + FEW_WARPS - 1) / FEW_WARPS : 0, p.K, p.fault);
  stream.start(row_of);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if constexpr (DT == MQ_I8) {
      const int8_t* row = static_cast<const int8_t*>(p.x) + t * p.ldx;
      for (int k = threadIdx.x * 16; k < pitch; k += FEW_THREADS * 16)
        *reinterpret_cast<int4*>(few_codes + t * pitch + k) = t < p.T ? codes16(row, k, p.K) : make_int4(0, 0, 0, 0);
      if (threadIdx.x == 0 && t < p.T) x_scale[t] = p.x_scale[t];
    } else if (t < p.T) {
      const float s = round_row<VEC>(static_cast<const S*>(p.x) + t * p.ldx, p.K, few_codes + t * pitch, pitch, (int)threadIdx.x, FEW_THREADS, part[t], [] { __syncthreads(); });
      if (threadIdx.x == 0) x_scale[t] = s;
    } else {
      for (int k = threadIdx.x * 8; k < pitch; k += FEW_THREADS * 8) *reinterpret_cast<uint2*>(few_codes + t * pitch + k) = make_uint2(0, 0);
    }
  }
  __syncthreads();
  for (int r = 0; r < stream.n_rows; ++r) {
    int sum[NT] = {};
    stream.row(r, row_of, [&](int k, int4 w) {
#pragma unroll
      for (int t = 0; t < NT; ++t) sum[t] = dot16(w, *reinterpret_cast<const int4*>(few_codes + t * pitch + k), sum[t]);
    });
    if (!stream.ok) break;
    __syncwarp();
#pragma unroll
    for (int t = 0; t < NT; ++t) sum[t] = __reduce_add_sync(0xffffffffu, sum[t]);
    int mine = sum[0];
#pragma unroll
    for (int t = 1; t < NT; ++t) mine = lane == t ? sum[t] : mine;
    if (lane < p.T) {
      const int n = first + r * FEW_WARPS;
      float v = (float)mine * x_scale[lane] * __ldg(p.w_scale + n);
      if (p.bias) v = plus_bias(v, __ldg(p.bias + n));
      put(p.y, p.out_dtype, lane * p.ldy + n, v);
    }
  }
  stream.end();
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
  int* fault;
};

// bytes in front of the rings: codes of h and a product per row and pair
__host__ __device__ __forceinline__ size_t one_token_down_codes(int top_k, int64_t K, int64_t I) {
  return ((size_t)top_k * few_pitch((int)I) + (size_t)(K / FEW_BLOCKS + 1) * top_k * 4 + 127) / 128 * 128;
}

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
__global__ void __launch_bounds__(ONE_THREADS, 1) one_token_gated_kernel(const OneParams p) {
  using S = typename StorageOf<DT>::type;
  extern __shared__ __align__(128) int8_t few_codes[];
  __shared__ uint64_t bars[ONE_WARPS][ONE_SLOTS];
  __shared__ uint32_t part[ONE_WARPS];
  __shared__ int expert[32], slot[32], found;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pitch = few_pitch(p.K);
  if (threadIdx.x == 32) init_bars(bars);
  chain_wait();
  chain_release();
  if (warp == 0) {
    const int n = pairs_here(p, lane, expert, slot);
    if (lane == 0) found = n;
  }
  __syncthreads();
  const int64_t all = (int64_t)found * p.I;     // 32 * INT8_MAX_K at most
  const int begin = (int)(all * blockIdx.x / gridDim.x), end = (int)(all * (blockIdx.x + 1) / gridDim.x);
  // unit u: gate row and up row of result u % I of pair u / I; the warp's rows by turns
  const int first = begin + warp, units = first < end ? (end - first + ONE_WARPS - 1) / ONE_WARPS : 0;
  auto row_of = [&](int r) {
    const int u = first + (r >> 1) * ONE_WARPS, pair = u / p.I, i = u - pair * p.I;
    return p.gate_up + (int64_t)expert[pair] * p.gate_up_expert + ((int64_t)(r & 1) * p.I + i) * p.ld_gate_up;
  };
  RowStream<ONE_SLOTS> stream(smem_u32(few_codes) + (uint32_t)(pitch + warp * ONE_SLOTS * FEW_PIECE), smem_u32(&bars[warp][0]), lane, 2 * units, p.K, p.fault);
  stream.start(row_of);
  const float xs = round_row<VEC>(static_cast<const S*>(p.x), p.K, few_codes, pitch, (int)threadIdx.x, ONE_THREADS, part, [] { __syncthreads(); });
  __syncthreads();
  for (int n = 0; n < units; ++n) {
    int sum[2];
#pragma unroll
    for (int set = 0; set < 2; ++set) {
      int s = 0;
      stream.row(2 * n + set, row_of, [&](int k, int4 w) { s = dot16(w, *reinterpret_cast<const int4*>(few_codes + k), s); });
      sum[set] = s;
    }
    if (!stream.ok) break;
    __syncwarp();
    const int g = __reduce_add_sync(0xffffffffu, sum[0]), up = __reduce_add_sync(0xffffffffu, sum[1]);
    if (lane == 0) {
      const int u = first + n * ONE_WARPS, pair = u / p.I, i = u - pair * p.I;
      const float* sc = p.gate_up_scale + (int64_t)expert[pair] * 2 * p.I;
      p.h[(int64_t)pair * p.I + i] = gated((float)g * xs * __ldg(sc + i), (float)up * xs * __ldg(sc + p.I + i));
    }
  }
  stream.end();
}

template <int DT>
__global__ void __launch_bounds__(ONE_THREADS, 1) one_token_down_kernel(const OneParams p) {
  extern __shared__ __align__(128) int8_t few_codes[];      // codes of h, the products of the block's rows, (rows, pairs), and the rings
  __shared__ uint64_t bars[ONE_WARPS][ONE_SLOTS];
  __shared__ int expert[32], slot[32], found;
  __shared__ float factor[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pitch = few_pitch(p.I);
  float* products = reinterpret_cast<float*>(few_codes + (size_t)p.top_k * pitch);
  if (threadIdx.x == 32) init_bars(bars);
  // (ids and weights have been there since before the kernel in front began)
  if (warp == 0) {
    const int n = pairs_here(p, lane, expert, slot);
    if (lane == 0) found = n;
  }
  __syncthreads();
  const int n_pairs = found;
  const int begin = (int)((int64_t)p.K * blockIdx.x / gridDim.x), end = (int)((int64_t)p.K * (blockIdx.x + 1) / gridDim.x);
  // unit u: row begin + u / n_pairs of the expert of pair u % n_pairs
  const int units = (end - begin) * n_pairs;
  auto row_of = [&](int r) {
    const int u = warp + r * ONE_WARPS;
    return p.down + (int64_t)expert[u % n_pairs] * p.down_expert + (int64_t)(begin + u / n_pairs) * p.ld_down;
  };
  RowStream<ONE_SLOTS> stream(smem_u32(few_codes) + (uint32_t)(one_token_down_codes(p.top_k, p.K, p.I) + warp * ONE_SLOTS * FEW_PIECE), smem_u32(&bars[warp][0]), lane,
                   warp < units ? (units - warp + ONE_WARPS - 1) / ONE_WARPS : 0, p.I, p.fault);
  stream.start(row_of);
  chain_wait();
  chain_release();
  for (int v = warp; v < n_pairs; v += ONE_WARPS) {
    const float s = p.I % 8 == 0 ? round_row<true>(p.h + (int64_t)v * p.I, p.I, few_codes + v * pitch, pitch, lane, 32, nullptr, [] {})
                                 : round_row<false>(p.h + (int64_t)v * p.I, p.I, few_codes + v * pitch, pitch, lane, 32, nullptr, [] {});
    if (lane == 0) factor[v] = s * p.weights[slot[v]];
  }
  __syncthreads();
  for (int r = 0; r < stream.n_rows; ++r) {
    const int u = warp + r * ONE_WARPS, v = u % n_pairs, n = begin + u / n_pairs;
    int sum = 0;
    stream.row(r, row_of, [&](int k, int4 w) { sum = dot16(w, *reinterpret_cast<const int4*>(few_codes + v * pitch + k), sum); });
    if (!stream.ok) break;
    __syncwarp();
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) products[u] = (float)sum * __ldg(p.down_scale + (int64_t)expert[v] * p.K + n);
  }
  stream.end();
  __syncthreads();
  for (int r = threadIdx.x; r < end - begin; r += ONE_THREADS) {
    float sum = 0.0f;
    for (int v = 0; v < n_pairs; ++v) sum = fmaf(factor[v], products[r * n_pairs + v], sum);      // as combine_kernel does
    put(p.y, DT, begin + r, sum);
  }
}

template <auto KERNEL, typename Params>
int launch_few(int threads, size_t smem, const Params& p, cudaStream_t st) {
  MQ_TRY(allow_smem<KERNEL>(FEW_SMEM));
  MQ_CUDA(launch_chained(true, KERNEL, dim3(FEW_BLOCKS), dim3((unsigned)threads), smem, st, p));
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}

template <int DT>
bool rows_of_eight(const void* x, int64_t ldx, int64_t K, int64_t T) {
  return K % 8 == 0 && aligned(x, 8 * dtype_size(DT)) && (T == 1 || ldx % 8 == 0);
}

template <int DT, int NT>
int few(const FewParams& p, cudaStream_t st) {
  const size_t smem = (size_t)NT * few_pitch(p.K) + FEW_RINGS;
  if constexpr (DT == MQ_I8) return launch_few<int8_few_kernel<DT, NT, true>>(FEW_THREADS, smem, p, st);
  else return rows_of_eight<DT>(p.x, p.ldx, p.K, p.T) ? launch_few<int8_few_kernel<DT, NT, true>>(FEW_THREADS, smem, p, st) : launch_few<int8_few_kernel<DT, NT, false>>(FEW_THREADS, smem, p, st);
}
template <int DT>
int few_of(const FewParams& p, cudaStream_t st) {
  if (p.T == 1) return few<DT, 1>(p, st);
  if (p.T == 2) return few<DT, 2>(p, st);
  return few<DT, 4>(p, st);
}

template <int DT>
int one_token(const OneParams& p, cudaStream_t st) {
  const size_t smem = (size_t)few_pitch(p.K) + FEW_RINGS;
  int status;
  if (rows_of_eight<DT>(p.x, 0, p.K, 1)) status = launch_few<one_token_gated_kernel<DT, true>>(ONE_THREADS, smem, p, st);
  else status = launch_few<one_token_gated_kernel<DT, false>>(ONE_THREADS, smem, p, st);
  MQ_TRY(status);
  return launch_few<one_token_down_kernel<DT>>(ONE_THREADS, one_token_down_codes(p.top_k, p.K, p.I) + FEW_RINGS, p, st);
}

}  // namespace

bool int8_few_fits(int64_t T, int64_t K) { return T <= INT8_FEW_TOKENS && (T <= 2 ? T : 4) * few_pitch((int)K) <= (int64_t)FEW_CODES; }

int int8_few(const void* x, int dtype, int64_t ldx, const Int8Product& q, const Int8Out& o, cudaStream_t st) {
  FewParams p = {x, q.x_scale, ldx, (int)q.T, q.rows, q.K, q.w, q.ldw, q.w_scale, o.bias, o.dtype, o.y, o.ldy, nullptr};
  MQ_TRY(fault_word(&p.fault));
  if (dtype == MQ_I8) return few_of<MQ_I8>(p, st);
  if (dtype == MQ_F32) return few_of<MQ_F32>(p, st);
  if (dtype == MQ_BF16) return few_of<MQ_BF16>(p, st);
  return few_of<MQ_F16>(p, st);
}

bool int8_one_token_fits(int top_k, int64_t K, int64_t I) {
  return (size_t)few_pitch((int)K) <= FEW_CODES && one_token_down_codes(top_k, K, I) <= FEW_CODES;
}

int int8_one_token(const void* x, int dtype, const int32_t* ids, const float* weights, int top_k, int first, const Int8Product& up, const Int8Product& down,
                   float* h, void* y, cudaStream_t st) {
  OneParams p = {x, up.K, up.rows, up.E, top_k, first, ids, weights, up.w, down.w, up.ldw, up.w_expert, down.ldw, down.w_expert,
                       up.w_scale, down.w_scale, h, y, nullptr};
  MQ_TRY(fault_word(&p.fault));
  return dtype == MQ_BF16 ? one_token<MQ_BF16>(p, st) : one_token<MQ_F16>(p, st);
}

}  // namespace mq
