// The 8-bit integer product on the fifth-generation tensor cores (tcgen05.mma kind::i8, sums in 32-bit integers in tensor
// memory: exact).
//
// The weights are the operand of 128 rows per CTA, the tokens the one of up to 256 columns, so a tile can be as narrow as the tokens
// that there are (32 and up in steps of 32) while weights fill the tensor core.  Two CTAs of a cluster share a tile of 256 weight
// rows (cta_group::2): each keeps 128 of them and half of the tokens, 32 KB per 128 of k instead of 48.
//   warp 0 of either CTA : TMA, 192 KB of stages (six where tiles are 256 tokens wide, nine of 20 KB where they are up to 64: a load takes
//                          about two microseconds from the wait for its stage to the end of its MMAs, and that many bytes must be under
//                          way meanwhile); the bytes of both CTAs count on the leader's barrier
//   warp 1 of the leader : tcgen05.mma for both SMs, two accumulators of 256 columns by turns
//   warps 4 .. 11        : epilogue, a quarter of the CTA's weight rows each, chunks of 32 tokens by turns
// What bounds it: 8192 tokens through 7168 x 7168 take 259 us, 3.25 PFLOP/s (bf16 by cuBLAS 1.66); the tensor pipe is busy 95.4 % of
// the SMs' active cycles, and 86.4 % of all: 896 tiles are 12.1 rounds of 74, so the thirteenth is nearly empty.
// Persistent: a pair of CTAs takes every 74th tile.  Eight tiles of weight rows at a time go with all tiles of tokens, so that the
// SMs that run side by side share rows of either in the L2.
// Where there are fewer tiles than pairs of CTAs, several take a share of k each (`splits`) and store their sums as integers; a second kernel
// on all SMs adds these up and does what the epilogue does.  (Adding them up in place by atomics, with the last CTA to arrive doing the
// epilogue, made it 39 us instead of 29 for 512 tokens through 2048 x 7168, codes included.)
#include "int8.cuh"
#include "profile.cuh"
#include "umma_pair.cuh"

namespace mq {
namespace {

constexpr int I8_MAX_STAGES = 9, I8_THREADS = 384, I8_K = 128, I8_TILE_BYTES = 128 * I8_K, I8_MAX_WIDTH = 256, I8_ROW_GROUP = 8;
constexpr int I8_PAIRS = 74;
constexpr int I8_RING_BYTES = 192 * 1024;
constexpr int I8_MAX_EXPERTS = 1024;
constexpr int I8_STAGING = 2048;   // of an epilogue warp
constexpr size_t kInt8Smem = (size_t)I8_RING_BYTES + 8 * I8_STAGING + 1024;

struct PairArgs {
  Int8Product p;
  Int8Out o;
  int max_width, m_tiles;
  int stages, stage_bytes;
  int gated_box;   // gate and up rows of a CTA come in one box (rows in whole sixteens), otherwise in four
  int packed;      // rows of results can be stored 16 bytes at a time
  int splits;      // CTA pairs that share a tile's k
  int* sums;       // INT8_SUMS: (splits, T, ld_sums)
  int64_t ld_sums;
  int* fault;
};

__device__ __forceinline__ void load_weights_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int k, int row, int set, int e) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(row), "r"(set), "r"(e)
      : "memory");
}
__device__ __forceinline__ void load_gated_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int k, int group, int e) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(0), "r"(group), "r"(e)
      : "memory");
}
__device__ __forceinline__ void load_tokens_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int k, int row) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(row)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32_int(uint32_t taddr, int (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Tiles of tokens of an expert with `count` rows, and their width: as few as the widest tile allows, all of one width.
__host__ __device__ __forceinline__ int token_tiles(int64_t count, int max_width) { return (int)((count + max_width - 1) / max_width); }
__host__ __device__ __forceinline__ int tile_width(int64_t count, int tiles) { return (int)((((count + tiles - 1) / tiles) + 31) / 32 * 32); }

// The tile that comes `unit`-th: which expert, which weight rows, which of its tokens, which share of k.
struct Unit {
  int e, m, width;
  int share, slab0, slab1;
  int t0, t_end;     // rows of the result
  __device__ __forceinline__ bool seek(int64_t unit, const PairArgs& a, const int* offsets, const int* tiles_before) {
    const int slabs = (a.p.K + I8_K - 1) / I8_K;
    share = 0;
    slab0 = 0;
    slab1 = slabs;
    if (a.splits > 1) {
      share = (int)(unit % a.splits);
      unit /= a.splits;
      slab0 = slabs * share / a.splits;
      slab1 = slabs * (share + 1) / a.splits;
    }
    if (unit >= (int64_t)tiles_before[a.p.E] * a.m_tiles) return false;
    int lo = 0, hi = a.p.E;      // the last expert whose tiles begin at or in front of this one
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int64_t)tiles_before[mid] * a.m_tiles <= unit) lo = mid;
      else hi = mid;
    }
    e = lo;
    const int begin = offsets[e], end = offsets[e + 1], n_tiles = tiles_before[e + 1] - tiles_before[e];
    const int i = (int)(unit - (int64_t)tiles_before[e] * a.m_tiles);
    const int g = i / (I8_ROW_GROUP * n_tiles), r = i - g * I8_ROW_GROUP * n_tiles;
    const int in_group = min(I8_ROW_GROUP, a.m_tiles - g * I8_ROW_GROUP);
    m = g * I8_ROW_GROUP + r % in_group;
    width = tile_width(end - begin, n_tiles);
    t0 = begin + r / in_group * width;
    t_end = min(t0 + width, end);
    return true;
  }
};

__device__ __forceinline__ uint16_t bits16(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ uint16_t bits16(__half v) { return __half_as_ushort(v); }

// Results of 32 columns (a lane each) for `TOKENS` tokens leave in 16-byte pieces of rows, through a tile in shared memory (2 KB, this
// warp's).  Stored by the lanes as they come, in pieces of 64 bytes, an epilogue of 256 tokens took 6 us.
template <int TOKENS, typename S, typename Of>
__device__ __forceinline__ void store_rows(uint32_t tile, int lane, S* out, int64_t ld, int left, int cols, Of value) {
  constexpr int PITCH = 32 * sizeof(S), PER = 16 / sizeof(S), LANES = 32 / PER;     // bytes of a row; values per piece; lanes per row
  static_assert(TOKENS * PITCH == 2048, "the tile has 2 KB");
#pragma unroll
  for (int j = 0; j < TOKENS; ++j) {
    if constexpr (sizeof(S) == 4) asm volatile("st.shared.f32 [%0], %1;" ::"r"(tile + j * PITCH + lane * 4), "f"(value(j)) : "memory");
    else asm volatile("st.shared.u16 [%0], %1;" ::"r"(tile + j * PITCH + lane * 2), "h"(bits16(from_float<S>(value(j)))) : "memory");
  }
  __syncwarp();
  const int row = lane / LANES, piece = lane % LANES;
  S* to = out + (int64_t)row * ld + piece * PER;
  const bool in = piece * PER < cols;
#pragma unroll
  for (int i = 0; i < TOKENS * LANES / 32; ++i) {
    uint4 w;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(tile + i * 512 + lane * 16) : "memory");
    if (in && i * (32 / LANES) + row < left) *reinterpret_cast<uint4*>(to) = w;
    to += (int64_t)(32 / LANES) * ld;
  }
  __syncwarp();
}

// The same, each lane its column: rows that cannot be stored 16 bytes at a time.  (A comparison in front of every store costs more than the
// stores: 2914 x 9508 x 120, bf16 results, 46 us instead of 25.5; in 16-byte pieces 2914 x 9504 x 120 takes 21.5.)
template <typename S, typename Of>
__device__ __forceinline__ void store_columns(S* to, int64_t ld, int left, Of value) {
  if (left >= 32) {
#pragma unroll
    for (int j = 0; j < 32; ++j, to += ld) *to = value(j);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j, to += ld)
      if (j < left) *to = value(j);
  }
}

// The tokens' rows in boxes of 32, 64 and 128. A box costs the TMA unit time beside its bytes: 16384 pairs, 32 experts, 7168 to 2048 and back,
// gate and up 364 us against 386 with boxes of 32 rows and of 16 gate and up rows, down 209 against 217 (with products stored in fp16).
struct TokenMaps {
  CUtensorMap rows32, rows64, rows128;
};

// DT: type of what is stored (INT8_Y)
template <int KIND, int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8_THREADS, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ TokenMaps maps, const PairArgs a) {
  constexpr int SETS = KIND == INT8_GATED ? 2 : 1;
  constexpr int TILE_ROWS = 256 / SETS;            // result columns of a tile
  const Int8Product& p = a.p;
  const int rank = (int)(blockIdx.x & 1), pair = (int)(blockIdx.x >> 1), n_pairs = (int)(gridDim.x >> 1);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  __shared__ __align__(8) uint64_t bars[2 * I8_MAX_STAGES + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ PairEnd end;
  __shared__ int offsets[I8_MAX_EXPERTS + 1], tiles_before[I8_MAX_EXPERTS + 1];
  __shared__ __align__(16) float token_scale[8][32];
  const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[I8_MAX_STAGES]);
  const uint32_t acc_full = smem_u32(&bars[2 * I8_MAX_STAGES]), acc_empty = smem_u32(&bars[2 * I8_MAX_STAGES + 2]);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(full0 + 8 * s, 1);    // the leader's: its producer's arrival, then the bytes of both CTAs
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + 8 * b, 1);
      mbar_init(acc_empty + 8 * b, 16);  // the leader's: eight epilogue warps of either CTA
    }
    end.reset();
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(&tmem_slot));
  chain_wait();
  chain_release();
  if (warp == 2) {   // where each expert's rows and tiles begin
    int before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      int tiles = 0;
      if (e < p.E) {
        const int begin = p.offsets ? __ldcg(p.offsets + e) : 0, last = p.offsets ? __ldcg(p.offsets + e + 1) : (int)p.T;
        offsets[e] = begin;
        if (e == p.E - 1) offsets[p.E] = last;
        tiles = token_tiles(last - begin, a.max_width);
      }
      int sum = tiles;
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += u;
      }
      if (e < p.E) tiles_before[e] = before + sum - tiles;
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) tiles_before[p.E] = before;
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // either CTA's barriers and tensor memory exist before the other signals or writes them
  tc_fence_after();
  const uint32_t tmem_acc = tmem_slot;

  // Producer and MMA run in one thread each: with warps that wait and issue together a slab cost 680 cycles of issue, more than the MMAs of any
  // width take (8192 tokens through 7168 x 7168: 382 us).
  if (warp == 0) {
    if (elect_one()) {
      const uint32_t full_leader = leader_addr(full0);
      int it = 0, st = 0;
      uint32_t round = 0;
      bool ok = true;
      Unit u;
      for (int64_t unit = pair; ok && u.seek(unit, a, offsets, tiles_before); unit += n_pairs) {
        const int half = u.width >> 1;
        const int b_row = u.t0 + rank * half;
        const int n_boxes = (half + 31) / 32;
        const uint32_t bytes = 2 * (I8_TILE_BYTES + (uint32_t)n_boxes * 32 * I8_K);
        for (int s = u.slab0; s < u.slab1; ++s, ++it) {
          if (it >= a.stages && !mbar_wait_elected(empty0 + 8 * st, (round - 1) & 1, a.fault, 91)) { ok = false; break; }
          const uint32_t dst = smem_base + (uint32_t)(st * a.stage_bytes), bar = full_leader + 8 * st;
          if (rank == 0) mbar_expect_tx(full0 + 8 * st, bytes);
          if constexpr (KIND == INT8_GATED) {
            // sixteen gate rows, then the sixteen up rows of the same results, for each quarter of the CTA's rows
            if (a.gated_box) {
              load_gated_pair(dst, &map_w, bar, s * I8_K, u.m * (TILE_ROWS / 16) + rank * 4, u.e);
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q)
                load_weights_pair(dst + q * (I8_TILE_BYTES / 4), &map_w, bar, s * I8_K, u.m * TILE_ROWS + rank * 64 + q * 16, 0, u.e);
            }
          } else {
            load_weights_pair(dst, &map_w, bar, s * I8_K, u.m * TILE_ROWS + rank * 128, 0, u.e);
          }
          const uint32_t tokens = dst + I8_TILE_BYTES;
          if (n_boxes == 4) {
            load_tokens_pair(tokens, &maps.rows128, bar, s * I8_K, b_row);
          } else {
            if (n_boxes >= 2) load_tokens_pair(tokens, &maps.rows64, bar, s * I8_K, b_row);
            if (n_boxes & 1) load_tokens_pair(tokens + (n_boxes & 2) * 32 * I8_K, &maps.rows32, bar, s * I8_K, b_row + (n_boxes & 2) * 32);
          }
          if (++st == a.stages) {
            st = 0;
            ++round;
          }
        }
      }
      // the last use of every stage has been read (so its copies had landed)
      for (int j = it > a.stages ? it - a.stages : 0; j < it && ok; ++j) ok = mbar_wait_elected(empty0 + 8 * (j % a.stages), (j / a.stages) & 1, a.fault, 95);
      end.copied_by(rank, it);
      if (!ok) end.give_up();
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      int it = 0, n = 0, st = 0;
      uint32_t round = 0;
      bool ok = true;
      Unit u;
      const uint64_t desc0 = kmajor_sw128_desc(smem_base);
      for (int64_t unit = pair; ok && u.seek(unit, a, offsets, tiles_before); unit += n_pairs, ++n) {
        const int b = n & 1;
        // sums of 32 bits, signed 8-bit operands, 256 rows, `width` columns
        const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(u.width >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
        const uint32_t acc = tmem_acc + (uint32_t)(b * I8_MAX_WIDTH);
        if (n >= 2) ok = mbar_wait_elected(acc_empty + 8 * b, ((n >> 1) - 1) & 1, a.fault, 93);
        tc_fence_after();
        for (int s = u.slab0; s < u.slab1 && ok; ++s) {
          ok = mbar_wait_elected(full0 + 8 * st, round & 1, a.fault, 92);
          if (!ok) break;
          tc_fence_after();
          const uint64_t a0 = desc0 + (uint64_t)((uint32_t)(st * a.stage_bytes) >> 4), b0 = a0 + (I8_TILE_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < I8_K / 32; ++kk)
            umma_i8_pair(acc, a0 + (uint64_t)((kk * 32) >> 4), b0 + (uint64_t)((kk * 32) >> 4), idesc, s > u.slab0 || kk > 0 ? 1u : 0u);
          umma_commit_pair(empty0 + 8 * st);
          if (s == u.slab1 - 1) umma_commit_pair(acc_full + 8 * b);
          ++it;
          if (++st == a.stages) {
            st = 0;
            ++round;
          }
        }
        if (!ok) break;
      }
      end.multiplied(it, n);
      if (!ok) end.give_up();
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int h = (warp - 4) >> 2, q = warp & 3;   // which chunks of 32 tokens, TMEM lane quadrant
    const uint32_t empty_leader = leader_addr(acc_empty);
    const uint32_t t_lane = tmem_acc + ((uint32_t)(q * 32) << 16);
    float* my_scale = token_scale[warp - 4];
    const uint32_t tile = smem_base + (uint32_t)I8_RING_BYTES + (uint32_t)(warp - 4) * I8_STAGING;
    bool ok = true;
    int n = 0;
    Unit u;
    for (int64_t unit = pair; ok && u.seek(unit, a, offsets, tiles_before); unit += n_pairs, ++n) {
      const int b = n & 1;
      const int col = KIND == INT8_GATED ? u.m * TILE_ROWS + rank * 64 + q * 16 + (lane & 15) : u.m * TILE_ROWS + rank * 128 + q * 32 + lane;
      const bool col_in = col < p.rows;
      const int w_row = KIND == INT8_GATED ? (lane >> 4) * p.rows + col : col;
      const float ws = col_in ? __ldg(p.w_scale + (int64_t)u.e * SETS * p.rows + w_row) : 0.0f;
      const float bias = KIND == INT8_Y && a.o.bias && col_in ? __ldg(a.o.bias + col) : 0.0f;
      const int chunks = u.width >> 5;
      float xs[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = u.t0 + (2 * i + h) * 32 + lane;
        xs[i] = 0.0f;
        if (2 * i + h < chunks && t < u.t_end) xs[i] = KIND == INT8_PAIRS || KIND == INT8_SUMS ? 1.0f : __ldcg(p.x_scale + t);
      }
      ok = mbar_wait(acc_full + 8 * b, (n >> 1) & 1, a.fault, 94);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 2 * i + h;
        if (c >= chunks) break;
        int r[32];
        tmem_ld32_int(t_lane + (uint32_t)(b * I8_MAX_WIDTH + c * 32), r);
        const int t = u.t0 + c * 32, left = u.t_end - t;     // tokens of this chunk that exist
        if constexpr (KIND == INT8_SUMS) {
          store_columns(a.sums + ((int64_t)u.share * p.T + t) * a.ld_sums + col, a.ld_sums, col_in ? left : 0, [&](int j) { return r[j]; });
          continue;
        }
        float v[32];
        if constexpr (KIND == INT8_PAIRS) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = (float)r[j] * ws;
        } else {
          __syncwarp();
          my_scale[lane] = xs[i];
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(my_scale + j);
            v[j] = (float)r[j] * s4.x * ws;
            v[j + 1] = (float)r[j + 1] * s4.y * ws;
            v[j + 2] = (float)r[j + 2] * s4.z * ws;
            v[j + 3] = (float)r[j + 3] * s4.w * ws;
          }
        }
        if constexpr (KIND == INT8_GATED) {
          // lanes 0 .. 15 hold the gate, 16 .. 31 the up of the same results: the former take the even tokens, the latter the odd; 32 tokens
          // of 16 results lie in the tile as 16 rows of two tokens each
          const bool up = lane >= 16;
          float hv[16];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + 1], 16);
            hv[j / 2] = up ? gated(other, v[j + 1]) : gated(v[j], other);
          }
          float* out = static_cast<float*>(a.o.y) + (int64_t)t * a.o.ldy + (col - (lane & 15));
          const int cols = p.rows - (col - (lane & 15));
#pragma unroll
          for (int j = 0; j < 16; ++j)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(tile + j * 128 + lane * 4), "f"(hv[j]) : "memory");
          __syncwarp();
          const int token = lane >> 2, piece = lane & 3;
          float* to = out + (int64_t)token * a.o.ldy + piece * 4;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint4 w;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(tile + k * 512 + lane * 16) : "memory");
            // (rows of h have room for a multiple of sixteen results)
            if (piece * 4 < cols && k * 8 + token < left) *reinterpret_cast<uint4*>(to) = w;
            to += 8 * a.o.ldy;
          }
          __syncwarp();
        } else {
          using S = typename StorageOf<DT>::type;
          if constexpr (KIND == INT8_Y) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = plus_bias(v[j], bias);
          }
          S* out = static_cast<S*>(a.o.y) + (int64_t)t * a.o.ldy + (col - lane);
          if (a.packed) {
            constexpr int TOKENS = 64 / sizeof(S);
            store_rows<TOKENS>(tile, lane, out, a.o.ldy, left, p.rows - (col - lane), [&](int j) { return v[j]; });
            if constexpr (TOKENS < 32)
              store_rows<TOKENS>(tile, lane, out + (int64_t)TOKENS * a.o.ldy, a.o.ldy, left - TOKENS, p.rows - (col - lane), [&](int j) { return v[TOKENS + j]; });
          } else {
            store_columns(out + lane, a.o.ldy, col_in ? left : 0, [&](int j) { return from_float<S>(v[j]); });
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(empty_leader + 8 * b);
    }
    if (lane == 0 && !ok) end.give_up();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // neither CTA issues a copy, an MMA or an arrival any more
  if (end.given_up) {   // the same in both CTAs
    if (warp == 0) end.drain(a.stages, rank, full0, empty0, acc_full);
    __syncthreads();
    cluster_sync();   // the other CTA's copies signal the leader's barriers
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_acc);
  }
}

// y from the sums of `splits` shares of k: four results of a token a thread
__global__ void __launch_bounds__(256) finish_kernel(const PairArgs a) {
  const Int8Product& p = a.p;
  chain_wait();
  chain_release();
  const int words = (int)(a.ld_sums >> 2);
  const int64_t all = p.T * words;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / words;
    const int n = (int)(i - t * words) * 4;
    const int4* src = reinterpret_cast<const int4*>(a.sums + t * a.ld_sums + n);
    int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
      const int4 v = __ldcg(src + s * (p.T * words));
      sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    }
    const float xs = __ldcg(p.x_scale + t);
    const int r[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (n + j >= p.rows) break;
      float v = (float)r[j] * xs * __ldg(p.w_scale + n + j);
      if (a.o.bias) v = plus_bias(v, __ldg(a.o.bias + n + j));
      const int64_t at = t * a.o.ldy + n + j;
      if (a.o.dtype == MQ_F32) static_cast<float*>(a.o.y)[at] = v;
      else if (a.o.dtype == MQ_BF16) static_cast<__nv_bfloat16*>(a.o.y)[at] = __float2bfloat16_rn(v);
      else static_cast<__half*>(a.o.y)[at] = __float2half_rn(v);
    }
  }
}

int encode(EncodeTiledFn enc, CUtensorMap* map, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, ones,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  MQ_REQUIRE(r == CUDA_SUCCESS, MQ_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d for codes of %llu x %llu", (int)r, (unsigned long long)dims[1],
             (unsigned long long)dims[0]);
  return MQ_OK;
}

template <int KIND, int DT = MQ_F32>
int launch(const CUtensorMap& map_w, const TokenMaps& map_x, const PairArgs& a, int pairs, cudaStream_t st) {
  MQ_TRY((allow_smem<int8_pair_kernel<KIND, DT>>(kInt8Smem)));
  MQ_CUDA(launch_chained(true, int8_pair_kernel<KIND, DT>, dim3((unsigned)(2 * pairs)), dim3(I8_THREADS), kInt8Smem, st, map_w, map_x, a));
  MQ_LAUNCH_CHECK();
  return MQ_OK;
}

}  // namespace

namespace {
// How wide a tile of tokens is at most and how many pairs of CTAs share its k, from what a tile costs (us, measured over 2048 to 7168 rows of
// 1024 to 16384): a slab of 128 of k 0.225 up to 64 columns and 0.20 + 0.00035 a column above, 4.9 + 0.008 a column beside the slabs; where k
// is shared, 3.3 for the second kernel and 10 MB/us for the sums' way through the L2.  Picked / best of all shapes tried: 16 tokens
// through 2048 x 7168 9.7 / 9.6 (not shared 16.3), 512 tokens 16.1 / 15.5, 2048 tokens 23.9 / 23.8 (128 wide 31.0), 1011 x 1008 x 1072 7.1 / 7.1 (256
// wide 9.6).
struct Shape {
  int width, splits;
};
constexpr int I8_MOST_SPLITS = 16;
Shape best_shape(int64_t rows_of_tiles, int64_t T, int slabs, bool shared) {
  Shape best = {I8_MAX_WIDTH, 1};
  double best_us = 1e30;
  for (int width = I8_MAX_WIDTH; width >= 32; width -= 32) {
    const int64_t n_tiles = token_tiles(T, width), tiles = rows_of_tiles * n_tiles;
    const int w = tile_width(T, (int)n_tiles);
    const double slab_us = w <= 64 ? 0.225 : 0.20 + 0.00035 * w;
    const int fit = shared && tiles < I8_PAIRS ? (int)(I8_PAIRS / tiles) : 1;
    for (int splits = 1; splits <= fit && splits <= I8_MOST_SPLITS && splits * 2 <= slabs; ++splits) {
      const double us = (double)ceil_div(tiles * splits, I8_PAIRS) * (double)ceil_div(slabs, splits) * slab_us + 4.9 + 0.008 * w +
                        (splits > 1 ? 3.3 + 8.0 * splits * (double)T * (double)rows_of_tiles * 256 / 1e7 : 0.0);
      if (us < best_us * 0.98) {
        best_us = us;
        best = {width, splits};
      }
    }
  }
  return best;
}
int64_t row_tiles(const Int8Product& p, int kind) { return ceil_div(p.rows, kind == INT8_GATED ? 128 : 256); }
Shape shape_of(const Int8Product& p, int kind, bool shared) {
  // several experts, whose rows the host does not know: a tile need not be wider than there are rows
  if (p.offsets || kind != INT8_Y) return Shape{p.T < I8_MAX_WIDTH ? tile_width(p.T, 1) : I8_MAX_WIDTH, 1};
  return best_shape(row_tiles(p, kind), p.T, (int)ceil_div(p.K, I8_K), shared);
}
}  // namespace

size_t int8_umma_scratch_bytes(const Int8Product& p, int kind) {
  const Shape s = shape_of(p, kind, true);
  return s.splits == 1 ? 0 : (size_t)s.splits * (size_t)p.T * (size_t)align_up(p.rows, 4) * 4;
}

int int8_product_umma(const Int8Product& p, const Int8Out& o, void* scratch, cudaStream_t st) {
  EncodeTiledFn enc;
  MQ_TRY(get_encoder(&enc));
  PairArgs a = {};
  a.p = p;
  a.o = o;
  MQ_TRY(fault_word(&a.fault));
  const int sets = o.kind == INT8_GATED ? 2 : 1;
  CUtensorMap map_w;
  TokenMaps map_x;
  a.gated_box = sets == 2 && p.rows % 16 == 0;
  if (a.gated_box) {
    // sixteen rows, gate and up, groups of sixteen rows: four groups of a tile land as its epilogue wants them
    const cuuint64_t dims[5] = {(cuuint64_t)p.K, 16, 2, (cuuint64_t)p.rows / 16, (cuuint64_t)p.E};
    const cuuint64_t set = (cuuint64_t)p.ldw * p.rows, expert = p.E > 1 ? (cuuint64_t)p.w_expert : 2 * set;
    const cuuint64_t strides[4] = {(cuuint64_t)p.ldw, set, 16 * (cuuint64_t)p.ldw, expert};
    const cuuint32_t box[5] = {I8_K, 16, 2, 4, 1};
    MQ_TRY(encode(enc, &map_w, 5, p.w, dims, strides, box));
  } else {
    const cuuint64_t dims[4] = {(cuuint64_t)p.K, (cuuint64_t)p.rows, (cuuint64_t)sets, (cuuint64_t)p.E};
    const cuuint64_t set = (cuuint64_t)p.ldw * p.rows, expert = p.E > 1 ? (cuuint64_t)p.w_expert : set * sets;
    const cuuint64_t strides[3] = {(cuuint64_t)p.ldw, set, expert};
    const cuuint32_t box[4] = {I8_K, sets == 2 ? 16u : 128u, (cuuint32_t)sets, 1};
    MQ_TRY(encode(enc, &map_w, 4, p.w, dims, strides, box));
  }
  {
    const cuuint64_t dims[2] = {(cuuint64_t)p.K, (cuuint64_t)p.x_rows};
    const cuuint64_t strides[1] = {(cuuint64_t)p.ldx};
    CUtensorMap* map[3] = {&map_x.rows32, &map_x.rows64, &map_x.rows128};
    for (int i = 0; i < 3; ++i) {
      const cuuint32_t box[2] = {I8_K, 32u << i};
      MQ_TRY(encode(enc, map[i], 2, p.x, dims, strides, box));
    }
  }
  a.m_tiles = (int)row_tiles(p, o.kind);
  const Shape shape = shape_of(p, o.kind, scratch != nullptr);
  a.max_width = shape.width;
  a.splits = shape.splits;
  a.stage_bytes = I8_TILE_BYTES + (a.max_width / 2 + 31) / 32 * 32 * I8_K;
  a.stages = I8_RING_BYTES / a.stage_bytes < I8_MAX_STAGES ? I8_RING_BYTES / a.stage_bytes : I8_MAX_STAGES;
  a.sums = static_cast<int*>(scratch);
  a.ld_sums = (int64_t)align_up(p.rows, 4);
  const int64_t most = a.m_tiles * (ceil_div(p.T, a.max_width) + (p.offsets ? p.E : 0)) * a.splits;
  const int pairs = (int)(most < I8_PAIRS ? most : I8_PAIRS);
  if (a.splits > 1) {
    MQ_TRY(launch<INT8_SUMS>(map_w, map_x, a, pairs, st));
    const int64_t blocks = ceil_div(p.T * (a.ld_sums >> 2), 256);
    MQ_CUDA(launch_chained(true, finish_kernel, dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8)), dim3(256), 0, st, a));
    MQ_LAUNCH_CHECK();
    return MQ_OK;
  }
  const int64_t piece = o.kind == INT8_GATED ? 4 : 16 / (int64_t)dtype_size(o.dtype);
  a.packed = p.rows % piece == 0 && o.ldy % piece == 0 && aligned(o.y, 16);
  if (o.kind == INT8_GATED) return launch<INT8_GATED>(map_w, map_x, a, pairs, st);
  if (o.kind == INT8_PAIRS) return launch<INT8_PAIRS>(map_w, map_x, a, pairs, st);
  if (o.dtype == MQ_F32) return launch<INT8_Y, MQ_F32>(map_w, map_x, a, pairs, st);
  if (o.dtype == MQ_BF16) return launch<INT8_Y, MQ_BF16>(map_w, map_x, a, pairs, st);
  return launch<INT8_Y, MQ_F16>(map_w, map_x, a, pairs, st);
}

}  // namespace mq
