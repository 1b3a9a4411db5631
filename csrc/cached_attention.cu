// Attention over the block-wise 8-bit KV cache (kv_format.cuh) for few query rows per request: single tokens, drafted
// tokens, short pieces, and every shape that the tcgen05 kernel (cached_attention_tc.cu) does not take.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp2(s_ij - m_i),   s_ij = (q_i . k_j) * scale * log2(e)
//   over the keys j <= context - new + i of the request's own blocks.
//
// The query heads that share a kv head, and the new tokens, are rows of one tile (8 to 32 rows), so the cache is read once
// for all of them. Bound by HBM: 2 D bytes per cached token and kv head against 4 D flops per row.
//
// Codes go from global memory into the registers of the tensor-core fragments: the contraction indices of an MMA may be
// permuted as long as both operands agree, so a lane's fragments are consecutive bytes of a row (16 bytes of the key it
// holds the column of, 16 bytes of each of the four values that it holds the contraction rows of). They are widened to
// f16, which holds every code exactly, next to the MMA; the block's scales are applied in 32 bits, the key's to the
// scores and the value's to the probabilities (relative to the largest value scale so far, in steps of two, so that the
// f16 probabilities keep their 11 bits). That they are f16 is a choice: the second product then runs at the tensor cores' f16
// rate beside exact codes, and 11 bits are eight times finer than the bf16 result (error against 64 bits 0.0016 of the
// result's norm, as with 32-bit probabilities; the two differ by 0.0005 to 0.0009, in last bits of bf16). Sums of the
// probabilities are of the unrounded ones.
//
// The work is the list of all (request, row tile, kv head) items times their 64-key units. It is cut into equal
// consecutive ranges, one per resident block of threads, so ragged lengths cost nothing; a range that ends inside an item
// leaves a partial result (at most two per block), which the join kernel adds up in a fixed order. Where there is little
// work (cluster_parts), a cluster of blocks takes each (request, kv head) instead and adds its results up itself.
//
// Measured on a B200, single tokens, 32 heads on 8 of 128, fp8: 64 requests of every length up to 16384 tokens 111-118 us,
// 5.3-5.7 TB/s, 82-87% of the measured copy rate; one of 600 tokens 7.5-7.9 us, latency alone (the launch, then lengths, table,
// codes and products one after another). 32 requests of up to 2047 tokens, 16 kv heads of 64: 25 us, where the two launches
// and the pieces' ends (512 items, two ends per range) take most of it.
#include <algorithm>
#include <type_traits>

#include "cached_attention.cuh"
#include "common.cuh"
#include "kv_format.cuh"
#include "launch.cuh"
#include "launchers.h"

namespace qw {
namespace {

constexpr int kUnit = 64;    // keys of a unit: 16 per warp
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -3e38f;      // running maximum of a row that has seen no key
constexpr float kLazy = 6.f;        // the running maximum moves when a row grows by more than 2^6
constexpr float kWeightUp = 256.f;  // probabilities (<= 2^6) times value scale over the largest: at most 2^14 in f16

// c (16 x 8) += a (16 x 16) b (16 x 8), f16 operands
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 x 8 transpose of 16-bit numbers, two per lane
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float quad_max(float v) {  // over the four lanes that hold one row of q
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float column_max(float v) {  // over the eight lanes that hold one column of an MMA tile
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// The items of a request: row tiles x kv heads, each `units` long. The first `kLead` units of an item stand for what a
// piece costs apart from its keys (query rows, the sum over the warps): without them the ranges that hold many short
// requests took 1.3 times as long as the others.
struct Shape {
  int units, tiles;
};
constexpr int kLead = 3;
constexpr int kMaxParts = 16;  // blocks of a cluster
__device__ __forceinline__ Shape shape_of(const CachedAttn& p, int b, int rows_per_tile) {
  const int n = new_rows(p, b).n;
  const int ctx = min(p.context[b], p.max_table_tokens);
  Shape s;
  s.tiles = n > 0 ? (n * p.group + rows_per_tile - 1) / rows_per_tile : 0;
  s.units = ctx > 0 ? (ctx + kUnit - 1) / kUnit + kLead : 0;
  return s;
}
__device__ __forceinline__ int64_t work_of(const CachedAttn& p, int b, int rows_per_tile) {
  const Shape s = shape_of(p, b, rows_per_tile);
  return static_cast<int64_t>(s.units) * s.tiles * p.Hkv;
}
// Ranges: worker i has the units [i W / N, (i + 1) W / N).
__device__ __forceinline__ int worker_of(int64_t unit, int64_t total, int workers) {
  return static_cast<int>(((unit + 1) * workers - 1) / total);
}

// Bytes of shared memory.
template <int D, int ROWS>
struct Layout {
  static constexpr int kStages = D == 128 ? 3 : D == 64 ? 4 : 6;
  static constexpr int kStep = 16 * 2 * D;                       // one 16-key step: keys, then values
  static constexpr int kJoinRows = 8;                            // rows that the warps add up at a time
  static constexpr int kRing = kWarps * kStages * kStep;
  static constexpr int kJoin = kWarps * kJoinRows * D * 4;
  static constexpr int kQ = ROWS > 16 ? ROWS / 8 * (D / 16) * 32 * 8 : 0;  // query fragments (fewer: in registers)
  static constexpr int kTotal = kRing + kJoin + kQ;
  static constexpr int kPart = kJoinRows * (D + 2) * 4;          // a cluster's block: its result of those rows
  // blocks of threads per SM: registers and shared memory allow no more
  static constexpr int kPerSm = D == 128 ? (ROWS > 16 ? 2 : 3) : ROWS > 16 ? 3 : ROWS > 8 ? 4 : 5;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Where the 16-byte piece c of row r (of 16) of a step lies. The lanes that read shared memory together hold the rows
// g, g + 1 (keys) or the rows 0, 2, 4, 6 (values); the order of the pieces keeps them on different banks. Row r + 8 lies
// 8 D bytes after row r.
template <int D>
__device__ __forceinline__ int piece_at(int r, int c) {
  if constexpr (D == 128) return r * 128 + ((c ^ ((((r >> 1) & 3) << 1) ^ ((r & 1) << 2))) * 16);
  else if constexpr (D == 64) return (r >> 1) * 128 + ((r ^ (r >> 1)) & 1) * 64 + ((c ^ (((r >> 2) & 1) << 1)) * 16);
  else return r * 32 + c * 16;
}

// N bytes of shared memory as 32-bit words
template <int N>
__device__ __forceinline__ void lds(uint32_t* w, const uint8_t* p) {
  if constexpr (N == 16) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (N == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x; w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// shared memory of the cluster's block `rank`, at the place that this block calls `at`
__device__ __forceinline__ float4 ld_cluster4(uint32_t at, int rank) {
  float4 x;
  asm volatile(
      "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
      : "r"(at), "r"(rank));
  return x;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t at, int rank) {
  float2 x;
  asm volatile(
      "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %2, %3;\n\t"
      "ld.shared::cluster.v2.f32 {%0, %1}, [a];\n\t}"
      : "=f"(x.x), "=f"(x.y)
      : "r"(at), "r"(rank));
  return x;
}

// Rows that belong to no request are zero.
template <int D>
__device__ void zero_free_rows(const CachedAttn& p) {
  const int first = p.B > 0 ? min(max(p.query_start[0], 0), p.T) : p.T;
  const int last = p.B > 0 ? min(max(p.query_start[p.B], first), p.T) : p.T;
  const int64_t per = static_cast<int64_t>(p.Hkv) * p.group * (D / 8);
  for (int64_t i = threadIdx.x; i < (first + p.T - last) * per; i += kThreads) {
    const int r = static_cast<int>(i / per), c = static_cast<int>(i % per);
    const int64_t tok = r < first ? r : last + (r - first);
    *reinterpret_cast<uint4*>(p.out + tok * p.o_token + c / (D / 8) * p.o_head + (c % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
  }
}

// Walks the pieces (one item's consecutive units) of a range.
struct Walk {
  int64_t u, at;  // next unit; first unit of request b
  int b;
  Shape shape;
  // the piece
  int h, tile, u0, units, first_key, q0, n, ctx, row0, rows;

  template <int R>
  __device__ __forceinline__ void next(const CachedAttn& p, int64_t end) {
    int64_t size = static_cast<int64_t>(shape.units) * shape.tiles * p.Hkv;
    while (u >= at + size) {  // ends: u < end <= the sum of all requests' units
      at += size;
      shape = shape_of(p, ++b, R);
      size = static_cast<int64_t>(shape.units) * shape.tiles * p.Hkv;
    }
    const int64_t local = u - at;
    const int item = (local >> 32) == 0 ? static_cast<int>(static_cast<uint32_t>(local) / static_cast<uint32_t>(shape.units))
                                        : static_cast<int>(local / shape.units);
    u0 = static_cast<int>(local - static_cast<int64_t>(item) * shape.units);
    units = static_cast<int>(min(static_cast<int64_t>(shape.units - u0), end - u));
    u += units;
    first_key = max(u0 - kLead, 0) * kUnit;
    tile = item / p.Hkv;
    h = item - tile * p.Hkv;
    rows_of<R>(p);
  }
  // Part `rank` of `parts` of the keys of the next row tile of (b, h). u counts the row tiles.
  template <int R>
  __device__ __forceinline__ void next_tile(const CachedAttn& p, int rank, int parts) {
    tile = static_cast<int>(u++);
    rows_of<R>(p);
    const int all = max(shape.units - kLead, 0), from = static_cast<int>(static_cast<int64_t>(all) * rank / parts);
    u0 = from + kLead;
    units = static_cast<int>(static_cast<int64_t>(all) * (rank + 1) / parts) - from;
    first_key = from * kUnit;
  }
  template <int R>
  __device__ __forceinline__ void rows_of(const CachedAttn& p) {
    const NewRows fresh = new_rows(p, b);
    q0 = fresh.first;
    n = fresh.n;
    ctx = min(p.context[b], p.max_table_tokens);
    row0 = tile * R;
    rows = min(R, n * p.group - row0);
  }
  // keys that a row of the piece's tile sees: [0, lim)
  __device__ __forceinline__ int lim_of(const CachedAttn& p, int row) const {
    return min(ctx, p.context[b] - n + p.by_group.quotient(row0 + min(row, rows - 1)) + 1);
  }
  __device__ __forceinline__ int key_end(const CachedAttn& p) const { return min(lim_of(p, rows - 1), (u0 + units - kLead) * kUnit); }
};

// CLUSTERS: a cluster of blocks for each (request, kv head) instead of equal ranges of all work. Its blocks share the keys and
// add their results over distributed shared memory, without a second kernel.
template <int FMT, int D, int ROWS, bool CLUSTERS>
__global__ void __launch_bounds__(kThreads, Layout<D, ROWS>::kPerSm) cached_attn_kernel(CachedAttn p, int parts) {
  using L = Layout<D, ROWS>;
  constexpr int R = ROWS;                         // rows of a tile
  constexpr int N = ROWS / 8;                     // 8-row tiles of queries
  constexpr int VB = D / 4 < 16 ? D / 4 : 16;     // bytes of a key that a lane reads at a time
  constexpr int CH = D / 4 / VB;
  constexpr int NT = D / 16;                      // 16-wide output tiles
  constexpr bool kQInSmem = L::kQ > 0;
  constexpr int S = L::kStages;
  extern __shared__ __align__(16) uint8_t smem[];
  float* s_o = reinterpret_cast<float*>(smem + L::kRing);  // [kWarps][kJoinRows][D]
  uint2* s_q = reinterpret_cast<uint2*>(smem + L::kRing + L::kJoin);  // [N][D / 16][32]
  __shared__ __align__(8) float s_scale[kWarps][S][2];
  __shared__ float s_unit[R];
  __shared__ float s_mlv[kWarps][R][3];       // maximum, sum, largest value scale
  __shared__ int s_poison[D];                 // the first key whose value is NaN in this dim, among masked steps
  __shared__ int64_t s_find[3];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, t = lane % 4;
  griddep_wait();
  int64_t begin = 0, end;
  Walk ahead;
  const int rank = CLUSTERS ? static_cast<int>(blockIdx.x) % parts : 0;
  if constexpr (CLUSTERS) {
    for (int i = threadIdx.x; i < D; i += kThreads) s_poison[i] = 0x7fffffff;
    if (blockIdx.x == 0) zero_free_rows<D>(p);
    const int item = static_cast<int>(blockIdx.x) / parts;
    ahead.b = item / p.Hkv;
    ahead.h = item - ahead.b * p.Hkv;
    ahead.shape = shape_of(p, ahead.b, R);
    end = ahead.shape.tiles;
    __syncthreads();
    if (end == 0) {  // the same in the whole cluster
      griddep_launch();
      return;
    }
  } else {
    // ---- the range of this block of threads, and the request that it begins in
    if (warp == 0) {
      // the first 32 requests stay in registers between the two passes
      const int64_t mine = lane < p.B ? work_of(p, lane, R) : 0;
      int64_t total = mine;
      for (int b = lane + 32; b < p.B; b += 32) total += work_of(p, b, R);
  #pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      const int64_t workers = min(static_cast<int64_t>(gridDim.x), total);
      const int64_t first = blockIdx.x < workers ? blockIdx.x * total / workers : total;
      int64_t before = 0;
      const bool publish = blockIdx.x == 0;  // the join kernel reads the prefix sums
      if (lane == 0) s_find[0] = total;
      for (int b0 = 0; b0 < p.B && (publish || before <= first); b0 += 32) {
        const int b = b0 + lane;
        const int64_t w = b0 == 0 ? mine : b < p.B ? work_of(p, b, R) : 0;
        int64_t x = w;
  #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        const int64_t at = before + x - w;
        if (w > 0 && first >= at && first < at + w) {
          s_find[1] = b;
          s_find[2] = at;
        }
        if (publish && b < p.B) p.prefix[b] = at;
        before += __shfl_sync(0xffffffffu, x, 31);
      }
      if (publish && lane == 0) p.prefix[p.B] = total;
    }
    for (int i = threadIdx.x; i < D; i += kThreads) s_poison[i] = 0x7fffffff;
    __syncthreads();
    const int64_t total = s_find[0];
    const int workers = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total));
    if (static_cast<int>(blockIdx.x) >= workers) {
      griddep_launch();
      return;
    }
    begin = blockIdx.x * total / workers;
    end = (blockIdx.x + 1) * total / workers;
    ahead.b = static_cast<int>(s_find[1]);
    ahead.at = s_find[2];
    ahead.shape = shape_of(p, ahead.b, R);
  }
  ahead.u = begin;
  auto next_piece = [&](Walk& x) {
    if constexpr (CLUSTERS) x.next_tile<R>(p, rank, parts);
    else x.next<R>(p, end);
  };

  // ---- the warp's 16-key steps, fetched S - 1 steps ahead across the pieces
  uint8_t* ring = smem + warp * S * L::kStep;
  const uint32_t ring_u32 = smem_u32(ring), scale_u32 = smem_u32(&s_scale[warp][0][0]);
  Walk now = ahead;
  constexpr int CPR = D / 16;                         // 16-byte pieces of a row
  constexpr int RPI = 32 / CPR < 16 ? 32 / CPR : 16;  // rows per instruction
  // Shared-memory offsets of a step that the lane needs; the others differ by constants (see piece_at). Kept in registers:
  // worked out again in every step they cost as much as the arithmetic.
  const int put[2] = {piece_at<D>(lane / CPR, lane % CPR), piece_at<D>(RPI < 16 ? RPI + lane / CPR : 0, lane % CPR)};
  int key_at[CH], val_at[2];
#pragma unroll
  for (int c = 0; c < CH; ++c) key_at[c] = piece_at<D>(g, (c * 4 * VB + t * VB) / 16) + (t * VB) % 16;
#pragma unroll
  for (int x = 0; x < 2; ++x) val_at[x] = 16 * D + piece_at<D>(2 * t + x, g * (D / 8) / 16) + (g * (D / 8)) % 16;
  // row r + 8 lies 8 rows further
  const uint32_t k_lane = (lane / CPR) * p.k.token_stride + (lane % CPR) * 16;
  const uint32_t v_lane = (lane / CPR) * p.v.token_stride + (lane % CPR) * 16;
  const float* const my_scale = lane == 0 ? p.k.scale : p.v.scale;  // lane 0 fetches the key scale, lane 1 the value's
  const uint32_t my_scale_stride = lane == 0 ? p.k.scale_stride : p.v.scale_stride;
  int a_j = -kUnit, a_end = 0, a_stage = 0;
  int a_id = -1, a_in = 0;              // the step's block, and where in it the step begins
  const int* a_entry = p.table;         // its table entry
  const uint8_t *a_k = nullptr, *a_v = nullptr;  // the lane's first byte in block 0
  bool a_done = false;
  auto a_next = [&]() {  // to the next step
    a_j += kUnit;
    a_in += kUnit;
    if (a_j >= a_end) {
      do {
        if (ahead.u >= end) {
          a_done = true;
          return;
        }
        next_piece(ahead);
        a_j = ahead.first_key + warp * 16;
        a_end = ahead.key_end(p);
      } while (a_j >= a_end);
      a_entry = p.table + static_cast<int64_t>(ahead.b) * p.table_stride + p.by_block.quotient(a_j);
      a_in = p.by_block.remainder(a_j, p.by_block.quotient(a_j));
      a_k = p.k.codes + static_cast<int64_t>(ahead.h) * p.k.head_stride + k_lane;
      a_v = p.v.codes + static_cast<int64_t>(ahead.h) * p.v.head_stride + v_lane;
    }
    while (a_in >= p.block) {
      a_in -= p.block;
      ++a_entry;
    }
    a_id = __ldg(a_entry);
  };
  auto fetch = [&]() {
    if (!a_done) {
      const uint32_t dst = ring_u32 + a_stage * L::kStep;
      if (static_cast<uint32_t>(a_id) < static_cast<uint32_t>(p.blocks)) {
        const uint32_t id = a_id;
        const uint8_t* kp = a_k + static_cast<uint64_t>(id) * p.k.block_stride + a_in * p.k.token_stride;
        const uint8_t* vp = a_v + static_cast<uint64_t>(id) * p.v.block_stride + a_in * p.v.token_stride;
#pragma unroll
        for (int i = 0; i < 16 / RPI; ++i) {
          const int at = put[i & 1] + (i >> 1) * (2 * RPI * D);
          cp_async16(dst + at, kp);
          cp_async16(dst + 16 * D + at, vp);
          kp += RPI * p.k.token_stride;
          vp += RPI * p.v.token_stride;
        }
        if (lane < 2) cp_async4(scale_u32 + a_stage * 8 + lane * 4, my_scale + static_cast<uint64_t>(id) * my_scale_stride + ahead.h);
      } else if (lane == 0) {  // a key without a block (none given, or outside the cache) counts as masked
        s_scale[warp][a_stage][0] = -1.f;
      }
      a_stage = a_stage + 1 == S ? 0 : a_stage + 1;
      a_next();
    }
    cp_async_commit();
  };
  a_next();
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch();
  int stage = 0;

  while (now.u < end) {
    next_piece(now);
    const int rows = now.rows;
    const int lim_first = now.lim_of(p, 0), lim_last = now.lim_of(p, rows - 1);
    const int key_end = now.key_end(p);

    // ---- query rows as f16 fragments, each divided by a power of two (kQueryTop)
    uint32_t q[kQInSmem ? 1 : N][D / 16][2];
    float unit[N][2];  // of the rows 2t, 2t + 1: what a product of codes and fragments is worth, but for the key's scale
    auto load_q = [&](int n, uint32_t (*frag)[2]) {  // row g of tile n; returns the row's unit
      const int row = n * 8 + g;
      float x[D / 4];
      float m = 0.f;
      if (row < rows) {
        const int r = now.row0 + row;
        const int rt = p.by_group.quotient(r);
        const bf16* src = p.q + static_cast<int64_t>(now.q0 + rt) * p.q_token + (now.h * p.group + p.by_group.remainder(r, rt)) * p.q_head;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int i = 0; i < VB; i += 8) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(src + c * 4 * VB + t * VB + i));
            const __nv_bfloat162* y = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = __bfloat1622float2(y[e]);
              x[c * VB + i + 2 * e] = f.x;
              x[c * VB + i + 2 * e + 1] = f.y;
            }
          }
#pragma unroll
        for (int i = 0; i < D / 4; ++i) m = fmaxf(m, fabsf(x[i]));
      } else {
#pragma unroll
        for (int i = 0; i < D / 4; ++i) x[i] = 0.f;
      }
      m = quad_max(m);
      const int e = min(max(static_cast<int>(__float_as_uint(m) >> 23) - 127, -100), 127);
      const bool fine = m > 0.f && m <= 3.4028234e38f;  // zero or infinite rows as they are
      const float inv = fine ? exp2i(kQueryTop - e) : 1.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        frag[s][0] = pack_f16(x[4 * s] * inv, x[4 * s + 1] * inv);
        frag[s][1] = pack_f16(x[4 * s + 2] * inv, x[4 * s + 3] * inv);
      }
      return (fine ? exp2i(e - kQueryTop) : 1.f) * p.scale * kLog2e;
    };
    if constexpr (!kQInSmem) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float u = load_q(n, q[n]);
        unit[n][0] = __shfl_sync(0xffffffffu, u, 8 * t);
        unit[n][1] = __shfl_sync(0xffffffffu, u, 8 * t + 4);
      }
    } else {  // a warp makes each tile's fragments, all read them from shared memory
      if (warp < N) {
        uint32_t frag[D / 16][2];
        const float u = load_q(warp, frag);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) s_q[(warp * (D / 16) + s) * 32 + lane] = make_uint2(frag[s][0], frag[s][1]);
        if (t == 0) s_unit[warp * 8 + g] = u;
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < N; ++n) {
        unit[n][0] = s_unit[n * 8 + 2 * t];
        unit[n][1] = s_unit[n * 8 + 2 * t + 1];
      }
    }

    // o[n][i]: dims g * D / 8 + 2i (first two: rows 2t, 2t + 1) and + 2i + 1 (last two)
    float o[N][NT][4];
    float m_run[N][2], l_run[N][2];
    float v_ref[N][2], v_up[N][2];  // the largest value scale that the row has seen, and kWeightUp over it
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int i = 0; i < NT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m_run[n][e] = kNone;
        l_run[n][e] = v_ref[n][e] = v_up[n][e] = 0.f;
      }
    }

    for (int j = now.first_key + warp * 16; j < key_end; j += kUnit) {
      cp_async_wait<S - 2>();
      __syncwarp();
      const uint8_t* step = ring + stage * L::kStep;
      const float2 sc = *reinterpret_cast<const float2*>(s_scale[warp][stage]);
      const float ks = sc.x, vs = sc.y;
      if (ks >= 0.f) {
        const bool edge = j + 16 > lim_first;
        // ---- scores: 16 keys x rows. Keys g, 8 + g are the rows of the MMA, queries its columns
        float s[N][4];
#pragma unroll
        for (int n = 0; n < N; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          uint32_t kw[2][VB / 4];  // dims c * 4 VB + t * VB ...
#pragma unroll
          for (int x = 0; x < 2; ++x) lds<VB>(kw[x], step + key_at[c] + x * 8 * D);
#pragma unroll
          for (int i = 0; i < VB / 4; ++i) {
            uint32_t lo[2], hi[2];
            Kv<FMT>::decode4(kw[0][i], lo[0], hi[0]);
            Kv<FMT>::decode4(kw[1][i], lo[1], hi[1]);
#pragma unroll
            for (int n = 0; n < N; ++n) {
              if constexpr (kQInSmem) {
                const uint2 w = s_q[(n * (D / 16) + c * (VB / 4) + i) * 32 + lane];
                mma_f16(s[n], lo[0], lo[1], hi[0], hi[1], w.x, w.y);
              } else {
                mma_f16(s[n], lo[0], lo[1], hi[0], hi[1], q[n][c * (VB / 4) + i][0], q[n][c * (VB / 4) + i][1]);
              }
            }
          }
        }
        // ---- probabilities of the rows 2t, 2t + 1 (e) and the keys j + g, j + g + 8
        bool moved = false;
        float top[N][2], v_top[N][2];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = unit[n][e] * ks;
            s[n][e] *= f;
            s[n][2 + e] *= f;
            v_top[n][e] = vs;
            if (edge) {
              const int lim = now.lim_of(p, n * 8 + 2 * t + e) - j;
              if (lim <= g) s[n][e] = -INFINITY;
              if (lim <= g + 8) s[n][2 + e] = -INFINITY;
              if (lim <= 0) v_top[n][e] = 0.f;
            }
            top[n][e] = fmaxf(s[n][e], s[n][2 + e]);
            moved = moved || top[n][e] > m_run[n][e] + kLazy || v_top[n][e] > v_ref[n][e];
          }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float v_new = fmaxf(v_ref[n][e], v_top[n][e]);
              const float m_new = fmaxf(m_run[n][e], column_max(top[n][e]));
              const float f = exp2f_approx(m_run[n][e] - m_new);
              const float fo = v_ref[n][e] > 0.f ? f * (v_ref[n][e] / v_new) : 0.f;
              m_run[n][e] = m_new;
              l_run[n][e] *= f;
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                o[n][i][e] *= fo;
                o[n][i][2 + e] *= fo;
              }
              v_ref[n][e] = v_new;
              v_up[n][e] = v_new > 0.f ? kWeightUp / v_new : 0.f;
            }
        }
        uint32_t w[N][2];  // weights as the second operand: keys 2t, 2t + 1 (and + 8) of row g
#pragma unroll
        for (int n = 0; n < N; ++n) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) pr[e] = exp2f_approx(s[n][e] - m_run[n][e & 1]);
          l_run[n][0] += pr[0] + pr[2];
          l_run[n][1] += pr[1] + pr[3];
          const float u0 = v_up[n][0] * vs, u1 = v_up[n][1] * vs;
          w[n][0] = transpose8(pack_f16(pr[0] * u0, pr[1] * u1));
          w[n][1] = transpose8(pack_f16(pr[2] * u0, pr[3] * u1));
        }
        // ---- output: values 2t, 2t + 1, 2t + 8, 2t + 9, dims g * D / 8 ..., four dims at a time
        uint32_t vw[4][D / 32];
#pragma unroll
        for (int x = 0; x < 4; ++x) lds<D / 8>(vw[x], step + val_at[x & 1] + (x >> 1) * 8 * D);
        if (edge) {  // values past the last row's limit may be anything: they count as zero
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = j + 2 * t + (x & 1) + (x >> 1) * 8;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
              if (key >= lim_last) {
                vw[x][i] = 0;
              } else if (key >= lim_first) {  // seen by some rows only: a NaN must not reach the others
                const uint32_t bad = Kv<FMT>::nan_bytes(vw[x][i]);
                if (bad)
                  for (int e = 0; e < 4; ++e)
                    if ((bad >> (8 * e + 7)) & 1) {
                      atomicMin(&s_poison[g * (D / 8) + 4 * i + e], key);
                      vw[x][i] &= ~(0xffu << (8 * e));
                    }
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t b0[4], b1[4];
          Kv<FMT>::decode4(__byte_perm(vw[0][i], vw[1][i], 0x5140), b0[0], b0[1]);
          Kv<FMT>::decode4(__byte_perm(vw[0][i], vw[1][i], 0x7362), b0[2], b0[3]);
          Kv<FMT>::decode4(__byte_perm(vw[2][i], vw[3][i], 0x5140), b1[0], b1[1]);
          Kv<FMT>::decode4(__byte_perm(vw[2][i], vw[3][i], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int n = 0; n < N; ++n)
              mma_f16(o[n][2 * i + e], b0[2 * e], b0[2 * e + 1], b1[2 * e], b1[2 * e + 1], w[n][0], w[n][1]);
        }
      }
      stage = stage + 1 == S ? 0 : stage + 1;
      __syncwarp();  // every lane has read the stage that is filled next
      fetch();
    }

    // ---- the four warps' results of this piece into one, a few rows at a time
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float l = column_sum(l_run[n][e]);
        if (g == 0) {
          float* dst = s_mlv[warp][n * 8 + 2 * t + e];
          dst[0] = m_run[n][e];
          dst[1] = l;
          dst[2] = v_ref[n][e];
        }
      }
    const bool whole = CLUSTERS ? parts == 1 : now.units == now.shape.units;
    float* const s_part = reinterpret_cast<float*>(smem + L::kTotal);  // with CLUSTERS: [8][D], then [8] maximum and sum
    auto store_row4 = [&](int row, int d, const float4& x, float f) {
      const int r = now.row0 + row;
      const int rt = p.by_group.quotient(r);
      bf16* dst = p.out + static_cast<int64_t>(now.q0 + rt) * p.o_token + (now.h * p.group + p.by_group.remainder(r, rt)) * p.o_head + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(x.x * f, x.y * f), pack_bf16(x.z * f, x.w * f));
    };
    const int64_t slot = now.u0 > 0 ? 2 * static_cast<int64_t>(blockIdx.x) : 2 * static_cast<int64_t>(blockIdx.x) + 1;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int first = n * 8;  // rows of this turn
      if (first < rows) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (first + 2 * t + e < rows) {
            float* dst = s_o + (warp * 8 + 2 * t + e) * D + g * (D / 8);
#pragma unroll
            for (int i = 0; i < NT; i += 2)
              *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[n][i][e], o[n][i][2 + e], o[n][i + 1][e], o[n][i + 1][2 + e]);
          }
        __syncthreads();
        for (int i = threadIdx.x; i < min(8, rows - first) * (D / 4); i += kThreads) {
          const int in = i / (D / 4), row = first + in, d = (i % (D / 4)) * 4;
          float m = kNone;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_mlv[w][row][0]);
          float l = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float mw = s_mlv[w][row][0];
            const float f = exp2f_approx(mw - m);
            const float fv = f * s_mlv[w][row][2] * (1.f / kWeightUp);
            l += s_mlv[w][row][1] * f;
            const float4 x = *reinterpret_cast<const float4*>(s_o + (w * 8 + in) * D + d);
            acc.x += x.x * fv; acc.y += x.y * fv; acc.z += x.z * fv; acc.w += x.w * fv;
          }
          const int lim = now.lim_of(p, row);
          if (s_poison[d] < lim) acc.x = __int_as_float(0x7fffffff);
          if (s_poison[d + 1] < lim) acc.y = __int_as_float(0x7fffffff);
          if (s_poison[d + 2] < lim) acc.z = __int_as_float(0x7fffffff);
          if (s_poison[d + 3] < lim) acc.w = __int_as_float(0x7fffffff);
          if (whole) {
            const float inv = m == kNone ? 0.f : 1.f / l;  // a row that sees no key is zero
            store_row4(row, d, acc, inv);
          } else if constexpr (CLUSTERS) {
            *reinterpret_cast<float4*>(s_part + in * D + d) = acc;
            if (d == 0) *reinterpret_cast<float2*>(s_part + 8 * D + in * 2) = make_float2(m, l);
          } else {
            *reinterpret_cast<float4*>(p.part_o + (slot * R + row) * D + d) = acc;
            if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * R + row) * 2) = make_float2(m, l);
          }
        }
        if (CLUSTERS && parts > 1) {
          cluster_sync();
          for (int i = rank * kThreads + threadIdx.x; i < min(8, rows - first) * (D / 4); i += parts * kThreads) {
            const int in = i / (D / 4), d = (i % (D / 4)) * 4;
            const uint32_t at = smem_u32(s_part + in * D + d), at_ml = smem_u32(s_part + 8 * D + in * 2);
            float m = kNone;
#pragma unroll 8
            for (int c = 0; c < parts; ++c) m = fmaxf(m, ld_cluster2(at_ml, c).x);
            float l = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (int c = 0; c < parts; ++c) {
              const float2 ml = ld_cluster2(at_ml, c);
              const float4 x = ld_cluster4(at, c);
              const float f = exp2f_approx(ml.x - m);
              l += ml.y * f;
              acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
            }
            const float inv = l != 0.f ? 1.f / l : 0.f;
            store_row4(in + first, d, acc, inv);
          }
          cluster_sync();  // the others have read this block's rows
        } else {
          __syncthreads();
        }
      }
    }
    if (FMT == kKvFp8 && key_end > lim_first) {  // uniform: only then a NaN may have been noted
      for (int i = threadIdx.x; i < D; i += kThreads) s_poison[i] = 0x7fffffff;
      __syncthreads();
    }
  }
  cp_async_wait<0>();
  griddep_launch();
}

// One warp per (token, query head): adds up the partial results of its item in the order of the ranges, and zeroes the
// rows that no range has (requests without cached tokens, tokens of no request).
template <int D>
__global__ void __launch_bounds__(128) cached_attn_join_kernel(CachedAttn p, int workers_max, int R) {
  const int lane = threadIdx.x % 32;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 32;
  griddep_wait();
  griddep_launch();
  if (i >= static_cast<int64_t>(p.T) * p.Hkv * p.group) return;
  const int tok = static_cast<int>(i / (p.Hkv * p.group)), hq = static_cast<int>(i % (p.Hkv * p.group));
  constexpr int PER = D / 32;
  bf16* dst = p.out + static_cast<int64_t>(tok) * p.o_token + hq * p.o_head + lane * PER;
  float acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  const int b = request_of(p, tok);
  float l = 0.f;
  const NewRows fresh = p.B > 0 ? new_rows(p, b) : NewRows{0, 0};
  if (tok >= fresh.first && tok < fresh.first + fresh.n) {
    const int64_t total = p.prefix[p.B], at0 = p.prefix[b];
    const Shape s = shape_of(p, b, R);
    if (s.units > 0) {
      const int row_all = (tok - fresh.first) * p.group + hq % p.group;
      const int h = hq / p.group, tile = row_all / R, row = row_all % R;
      const int64_t u0 = at0 + (static_cast<int64_t>(tile) * p.Hkv + h) * s.units;
      const int workers = static_cast<int>(min(static_cast<int64_t>(workers_max), total));
      const int w0 = worker_of(u0, total, workers), w1 = worker_of(u0 + s.units - 1, total, workers);
      if (w0 == w1) return;  // one range had the whole item
      auto place = [&](int w) { return (2 * static_cast<int64_t>(w) + (w == w0)) * R + row; };
      // each lane holds one range's maximum and sum, 32 ranges at a time
      float m = kNone;
      for (int w = w0 + lane; w <= w1; w += 32) m = fmaxf(m, p.part_ml[place(w) * 2]);
      m = warp_max(m);
      for (int w32 = w0; w32 <= w1; w32 += 32) {
        float f = 0.f;
        if (w32 + lane <= w1) {
          const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + place(w32 + lane) * 2);
          f = exp2f_approx(ml.x - m);
          l += ml.y * f;
        }
        const int n = min(32, w1 - w32 + 1);
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
          const float fi = __shfl_sync(0xffffffffu, f, i);
          const float* src = p.part_o + place(w32 + i) * D + lane * PER;
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] += src[e] * fi;
        }
      }
      l = warp_sum(l);
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) dst[e] = __float2bfloat16(acc[e] * inv);
}

template <typename F>
auto with_shape(int D, int rows, F&& f) {
  using std::integral_constant;
  auto by_rows = [&](auto d) {
    if (rows <= 8) return f(d, integral_constant<int, 8>{});
    if (rows <= 16) return f(d, integral_constant<int, 16>{});
    if (rows <= 24) return f(d, integral_constant<int, 24>{});
    return f(d, integral_constant<int, 32>{});
  };
  if (D == 32) return by_rows(integral_constant<int, 32>{});
  if (D == 64) return by_rows(integral_constant<int, 64>{});
  return by_rows(integral_constant<int, 128>{});
}

int workers_of(int D, int rows) {
  return 148 * with_shape(D, rows, [](auto d, auto r) { return Layout<d(), r()>::kPerSm; });
}

template <int FMT, int D, int ROWS, bool CLUSTERS>
void launch(const CachedAttn& p, int parts, cudaStream_t stream) {
  auto kernel = cached_attn_kernel<FMT, D, ROWS, CLUSTERS>;
  constexpr int smem = Layout<D, ROWS>::kTotal + (CLUSTERS ? Layout<D, ROWS>::kPart : 0);
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, current_device(), [&] {
    check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cached_attention smem");
    if (CLUSTERS) check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cached_attention cluster");
  });
  if constexpr (CLUSTERS) {
    launch_pdl_clusters(kernel, dim3(static_cast<unsigned>(p.B) * p.Hkv * parts), dim3(kThreads), parts, smem, stream,
                        "cached_attention", p, parts);
  } else {
    const int workers = 148 * Layout<D, ROWS>::kPerSm;
    launch_pdl(kernel, dim3(workers), dim3(kThreads), smem, stream, "cached_attention", p, 0);
    const int64_t rows = static_cast<int64_t>(p.T) * p.Hkv * p.group;
    launch_pdl(cached_attn_join_kernel<D>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, stream,
               "cached_attention join", p, workers, ROWS);
  }
}

void cached_attention_rows(const CachedAttn& p, int D, int fmt, int rows, int parts, cudaStream_t stream) {
  with_shape(D, rows, [&](auto d, auto r) {
    auto run = [&](auto f) {
      if (parts > 0) launch<f(), d(), r(), true>(p, parts, stream);
      else launch<f(), d(), r(), false>(p, 0, stream);
    };
    if (fmt == kKvFp8) run(std::integral_constant<int, kKvFp8>{});
    else run(std::integral_constant<int, kKvInt8>{});
  });
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Which kernel, and how its work is split.
struct Way {
  bool prompt;
  int tile, parts;          // few rows: rows of a tile, blocks of a cluster (0: equal ranges)
  int tiles_max, splits;    // prompts
  int64_t part_o, part_ml, bytes;  // of the workspace; the prefix sums are at its beginning
};

// Few rows, little work: the blocks of a cluster that each (request, kv head) gets, or 0 for equal ranges of all work. Equal
// ranges leave no SM idle, but a second kernel has to add their results, and finding them takes time: about 5 us. Measured
// (us, clusters against ranges, 8 kv heads of 128 dims, 4 rows each): 1 request of 600 tokens 6.4 / 11.0, of 2400 8.8 / 16.5,
// of 16000 (16 blocks) 19.6 / 22.6; 4 of 4800 tokens 14.6 / 18.2; 64 of up to 400 tokens 13.1 / 16.5, of up to 1600 28.8 / 22.8.
// 20 rows: 1 request of 4800 tokens 21.0 / 23.1, of 16000 33.4 / 28.3. So a block of a cluster gets at most `longest` units of
// 64 keys, fewer where lengths may differ (B > 1) and where a unit takes longer. More blocks than the SMs hold at a time cost
// more than the ranges do, but for clusters of one; the largest clusters need some room to be placed. A block without a unit
// only costs barriers (27 requests of up to 5 tokens: 4.7 us, 6.8 with eight blocks).
int cluster_parts(int64_t B, int Hkv, int tile, int resident, int max_context) {
  const int64_t items = B * Hkv, units = (static_cast<int64_t>(max_context) + kUnit - 1) / kUnit;
  if (items == 0) return 0;
  int parts = 1;
  if (units > 48 && items * kMaxParts * 10 <= resident * 7) {
    parts = kMaxParts;
  } else {
    while (parts < 8 && parts < units && items * parts * 2 * 8 <= resident * 7) parts *= 2;
  }
  const int64_t longest = parts == 1 ? 13 : tile > 8 ? 9 : B == 1 ? 20 : 12;
  return units <= parts * longest ? parts : 0;
}

Way way_of(int T, int B, int Hq, int Hkv, int D, int max_query, int max_context) {
  Way w{};
  const int group = Hq / Hkv;
  const int64_t rows = static_cast<int64_t>(std::min(max_query, T)) * group;
  w.prompt = D != 32 && rows > 32;
  w.tile = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 24 ? 24 : 32;
  int64_t slots;
  if (w.prompt) {
    const int64_t R = prompt_rows(D);  // sum of ceil(rows / R) over B requests is at most:
    w.tiles_max = static_cast<int>(std::max<int64_t>(1, (static_cast<int64_t>(T) * group + B * (R - 1)) / R));
    // too few row tiles for the SMs: split the keys, two tiles of 128 at least for each part
    const int64_t blocks = static_cast<int64_t>(w.tiles_max) * Hkv;
    w.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(148 * prompt_per_sm(D) / blocks, max_context / 256)));
    slots = w.splits > 1 ? blocks * w.splits * prompt_rows(D) : 0;
  } else {
    const int resident = workers_of(D, w.tile);
    w.parts = rows <= w.tile ? cluster_parts(B, Hkv, w.tile, resident, max_context) : 0;  // a request is one row tile
    slots = w.parts > 0 ? 0 : 2 * static_cast<int64_t>(resident) * w.tile;
  }
  w.part_o = align256((static_cast<int64_t>(B) + 1) * sizeof(int64_t));
  w.part_ml = w.part_o + align256(slots * D * sizeof(float));
  w.bytes = w.part_ml + align256(slots * 2 * sizeof(float));
  return w;
}

}  // namespace

int64_t cached_attention_workspace(int T, int B, int Hq, int Hkv, int D, int max_query, int max_context) {
  return way_of(T, B, Hq, Hkv, D, max_query, max_context).bytes;
}

void cached_attention(const bf16* q, int64_t q_token, int64_t q_head, bf16* out, int64_t o_token, int64_t o_head,
                      const KvPages& k, const KvPages& v, const int* table, int64_t table_stride, const int* context,
                      const int* query_start, int T, int B, int Hq, int Hkv, int D, int block, int blocks, int width,
                      int max_query, int max_context, float scale, int fmt, void* workspace, cudaStream_t stream) {
  if (T == 0) return;
  const Way w = way_of(T, B, Hq, Hkv, D, max_query, max_context);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  CachedAttn p{};
  p.q = q;
  p.q_token = q_token;
  p.q_head = q_head;
  p.out = out;
  p.o_token = o_token;
  p.o_head = o_head;
  auto pages = [](const KvPages& x) {
    return CachedPages{static_cast<const uint8_t*>(x.codes), static_cast<uint32_t>(x.block_stride),
                       static_cast<uint32_t>(x.head_stride), static_cast<uint32_t>(x.token_stride), x.scale,
                       static_cast<uint32_t>(x.scale_stride)};
  };
  p.k = pages(k);
  p.v = pages(v);
  p.table = table;
  p.table_stride = table_stride;
  p.context = context;
  p.query_start = query_start;
  p.T = T;
  p.B = B;
  p.Hkv = Hkv;
  p.group = Hq / Hkv;
  p.block = block;
  p.by_group = Divisor(p.group);
  p.by_block = Divisor(block);
  p.blocks = blocks;
  p.max_table_tokens = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(width) * block, 0x7fffffff));
  p.scale = scale;
  p.prefix = reinterpret_cast<int64_t*>(base);
  p.part_o = reinterpret_cast<float*>(base + w.part_o);
  p.part_ml = reinterpret_cast<float*>(base + w.part_ml);
  if (w.prompt) cached_attention_prompt(p, D, fmt, w.tiles_max, w.splits, stream);
  else cached_attention_rows(p, D, fmt, w.tile, w.parts, stream);
}

int cached_attention_status(bool clear) { return read_status_word(clear); }

}  // namespace qw
