// The block-wise KV cache's bookkeeping and its quantising write.
//
//  * plan_blocks: block tables, slot maps, positions and query offsets of a step from the requests' lengths. The block
//    pool lives on the device (a stack of free block ids and its height), so a captured step allocates its own blocks.
//  * release_blocks: blocks of finished (or cut) requests back onto the stack.
//  * append_kv: new keys and values into their slots in 8 bits (kv_format.cuh), one scale per block and head.
#include <algorithm>

#include "common.cuh"
#include "divisor.cuh"
#include "kv_format.cuh"
#include "launch.cuh"
#include "launchers.h"

namespace qw {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = 1024;  // tokens of a block of threads

// Exclusive sums of two numbers (below 2^31 in all) over the block's threads; `total` gets both sums.
struct Two {
  int tokens, blocks;
};
__device__ __forceinline__ Two block_scan(Two v, uint64_t* warp_sums, Two& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint64_t own = (static_cast<uint64_t>(static_cast<uint32_t>(v.tokens)) << 32) | static_cast<uint32_t>(v.blocks);
  uint64_t x = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {  // eight reads of shared memory instead of a second scan and its barriers
    const uint64_t s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  total = {static_cast<int>(all >> 32), static_cast<int>(all & 0xffffffffu)};
  const uint64_t at = before + x - own;
  return {static_cast<int>(at >> 32), static_cast<int>(at & 0xffffffffu)};
}

struct PlanArgs {
  const int* cached;
  const int* fresh;
  const int* state;  // [1 + B]: free blocks, then the blocks that each request holds
  int* table;
  int64_t table_stride;
  const int* free_blocks;
  int capacity;  // of free_blocks
  int B, width, block, tokens;
  int* query_start;
  int* context;
  int* positions;
  int* slots;
  int* state_out;
  int* missing;
};

struct Need {
  int cached, fresh, context;
  int held, fits, wanted;  // blocks
};

__device__ __forceinline__ Need need_of(const PlanArgs& a, int b) {
  Need n;
  n.cached = max(a.cached[b], 0);
  n.fresh = max(a.fresh[b], 0);
  const uint32_t total = min(static_cast<uint32_t>(n.cached) + static_cast<uint32_t>(n.fresh), 0x7fffffffu);
  n.context = static_cast<int>(total);
  // without new tokens: none, whatever length a caller leaves beside a row that it does not use
  n.wanted = n.fresh > 0 ? static_cast<int>((total + static_cast<uint32_t>(a.block) - 1) / static_cast<uint32_t>(a.block)) : 0;
  n.fits = min(n.wanted, a.width);
  n.held = min(max(a.state[1 + b], 0), a.width);
  return n;
}

// Two prefix sums over the requests (tokens, and blocks to take), which every block of threads does for itself: at a
// few hundred requests they cost less than a second launch. Then the work is spread over the blocks: the tokens' slots
// and positions by ranges, the tables' new entries by requests. A token's slot in a new block comes from the free list
// itself, not from the table, so that no block reads an entry that another one writes.
// Bound by the latency of the dependent reads (lengths, then tables, then slots), not by its few bytes: what the later parts
// need of a request is kept in shared memory.
// Measured on a B200: 256 decode requests or 64 prompts of up to 2048 tokens 9.4 us a call, of which the kernel is 3.4; the
// rest is the host's work for a call with six results.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanArgs a) {
  extern __shared__ int plan_smem[];
  int* start = plan_smem;           // [B + 1]
  int* rank = start + a.B + 1;      // [B]
  int* cached = rank + a.B;         // [B]
  int* held = cached + a.B;         // [B]
  int* fits = held + a.B;           // [B]
  __shared__ uint64_t sums[kPlanThreads / 32];
  __shared__ int s_short[kPlanThreads / 32];
  griddep_wait();
  griddep_launch();
  const int per = (a.B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(static_cast<int>(threadIdx.x) * per, a.B), b1 = min(b0 + per, a.B);
  const int free = min(max(a.state[0], 0), a.capacity);
  Two mine{0, 0}, all;
  int narrow = 0;
  for (int b = b0; b < b1; ++b) {
    const Need n = need_of(a, b);
    start[b] = n.fresh;
    rank[b] = max(n.fits - n.held, 0);
    cached[b] = n.cached;
    held[b] = n.held;
    fits[b] = n.fits;
    if (blockIdx.x == 0) a.context[b] = n.context;
    mine.tokens += n.fresh;
    mine.blocks += rank[b];
    narrow += n.wanted - n.fits;
  }
  Two at = block_scan(mine, sums, all);
  for (int b = b0; b < b1; ++b) {
    const int tokens = start[b], blocks = rank[b];
    start[b] = at.tokens;
    rank[b] = at.blocks;
    if (blockIdx.x == 0) {
      a.query_start[b] = at.tokens;
      a.state_out[1 + b] = held[b] + min(blocks, max(free - at.blocks, 0));
    }
    at.tokens += tokens;
    at.blocks += blocks;
  }
  if (threadIdx.x == 0) start[a.B] = all.tokens;
  if (blockIdx.x == 0) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) narrow += __shfl_xor_sync(0xffffffffu, narrow, o);
    if (threadIdx.x % 32 == 0) s_short[threadIdx.x / 32] = narrow;
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    int m = all.blocks - min(all.blocks, free);
    for (int w = 0; w < kPlanThreads / 32; ++w) m += s_short[w];
    a.query_start[a.B] = all.tokens;
    a.state_out[0] = free - min(all.blocks, free);
    a.missing[0] = m;
  }
  // slots and positions: kPlanTokens consecutive tokens per turn, neighbouring threads on neighbouring tokens
  for (int base = blockIdx.x * kPlanTokens; base < a.tokens; base += gridDim.x * kPlanTokens) {
#pragma unroll
    for (int i = 0; i < kPlanTokens / kPlanThreads; ++i) {
      const int tok = base + i * kPlanThreads + static_cast<int>(threadIdx.x);
      if (tok >= a.tokens) break;
      int slot = -1, pos = 0;
      if (tok < all.tokens) {
        int lo = 0, hi = a.B;  // the last request whose start is <= tok
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (start[mid] <= tok) lo = mid;
          else hi = mid;
        }
        const uint32_t p = min(static_cast<uint32_t>(tok - start[lo]) + static_cast<uint32_t>(cached[lo]), 0x7fffffffu);
        const uint32_t e = p / static_cast<uint32_t>(a.block), in = p - e * a.block;
        pos = static_cast<int>(p);
        int id = -1;
        if (static_cast<int>(e) < held[lo]) {
          id = a.table[lo * a.table_stride + e];
        } else if (static_cast<int>(e) < fits[lo]) {
          const int k = rank[lo] + static_cast<int>(e) - held[lo];
          if (k < free) id = a.free_blocks[free - 1 - k];
        }
        if (id >= 0) slot = id * a.block + static_cast<int>(in);
      }
      a.positions[tok] = pos;
      a.slots[tok] = slot;
    }
  }
  // new table entries: a warp per request
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int b = blockIdx.x * (kPlanThreads / 32) + warp; b < a.B; b += gridDim.x * (kPlanThreads / 32))
    for (int e = held[b] + lane; e < fits[b]; e += 32) {
      const int k = rank[b] + e - held[b];
      a.table[b * a.table_stride + e] = k < free ? a.free_blocks[free - 1 - k] : -1;
    }
}

// One block of threads: a request's entries past its kept tokens go onto the stack, requests in order.
__global__ void __launch_bounds__(kPlanThreads) release_kernel(const int* keep, int* state, int* table,
                                                               int64_t table_stride, int* free_blocks, int capacity,
                                                               int B, int width, int block) {
  __shared__ uint64_t sums[kPlanThreads / 32];
  griddep_wait();
  griddep_launch();
  const int per = (B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(static_cast<int>(threadIdx.x) * per, B), b1 = min(b0 + per, B);
  auto kept = [&](int b, int held) {
    return keep[b] < 0 ? held : min(held, static_cast<int>((static_cast<int64_t>(keep[b]) + block - 1) / block));
  };
  int n = 0;
  for (int b = b0; b < b1; ++b) {
    const int held = min(max(state[1 + b], 0), width);
    n += held - kept(b, held);
  }
  Two total;
  int at = block_scan(Two{0, n}, sums, total).blocks + min(max(state[0], 0), capacity);
  for (int b = b0; b < b1; ++b) {
    const int held = min(max(state[1 + b], 0), width), k = kept(b, held);
    for (int e = k; e < held; ++e, ++at) {
      if (at < capacity) free_blocks[at] = table[b * table_stride + e];
      table[b * table_stride + e] = -1;
    }
    state[1 + b] = k;
  }
  __syncthreads();  // every thread has read state[0]
  if (threadIdx.x == 0) state[0] = min(min(max(state[0], 0), capacity) + total.blocks, capacity);
}

// ------------------------------------------------------------------------------------------------ append
struct AppendArgs {
  const bf16* x[2];  // keys, values: [T, Hkv, D]
  int64_t token_stride[2], head_stride[2];
  const int* slots;
  uint8_t* cache[2];  // [blocks, Hkv, block, D]
  int64_t c_block[2], c_head[2], c_token[2];
  float* scale[2];  // [blocks, Hkv]
  int64_t s_block[2];
  int T, Hkv, block, blocks;
  Divisor by_block;
  int rows;   // tokens of a block of threads
  int turns;  // (head, keys or values) pairs of a team
};

constexpr int kAppendThreads = 256;
constexpr int kAppendRows = 128;  // most tokens of a block of threads
constexpr int kKeep = 8;          // 16-byte pieces of a run that a thread keeps between its two passes

// Largest magnitude of eight numbers as bf16 bits, two at a time: without the sign they order like unsigned integers.
// Infinities and NaN come out as 0x7f80 and above.
__device__ __forceinline__ uint32_t amax_bits(const uint4& w) {
  const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
  return max(m & 0xffffu, m >> 16);
}
constexpr uint32_t kInfBits = 0x7f80u;

// The same without infinities and NaN: neither sets a block's scale.
__device__ __forceinline__ uint32_t amax_bits_finite(const uint4& w) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = x[i] & 0x7fffu, hi = (x[i] >> 16) & 0x7fffu;
    m = max(m, max(lo < kInfBits ? lo : 0u, hi < kInfBits ? hi : 0u));
  }
  return m;
}

template <int FMT, bool FINITE>
__device__ __forceinline__ uint2 encode8(const uint4& w, float inv) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(x[i] << 16);
    f[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
  }
  if constexpr (FINITE && FMT == kKvInt8) {
    // |f * inv| <= 127: added to 1.5 * 2^23 the number is rounded to the nearest integer, ties to even, whose low byte is the
    // code
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(fmaf(f[i], inv, 12582912.f));
    return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
  } else {
    return make_uint2(Kv<FMT>::encode4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                      Kv<FMT>::encode4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
  }
}

// The tokens [t0, t0 + n) of one (block, head), written by a team of NT threads: into the block from token `first` on where
// the slots ascend one by one (`straight`).
template <int FMT, int D, int NT>
__device__ __forceinline__ void append_run(const AppendArgs& a, int kv, int h, int t0, int n, int64_t id, int first,
                                           bool straight, int team, int me, float* red) {
  constexpr int PPR = D / 8;  // 16-byte pieces of a token's row
  const bf16* x = (kv ? a.x[1] : a.x[0]) + h * (kv ? a.head_stride[1] : a.head_stride[0]);
  const int64_t ts = kv ? a.token_stride[1] : a.token_stride[0];
  const int64_t ct = kv ? a.c_token[1] : a.c_token[0];
  uint8_t* rows = (kv ? a.cache[1] : a.cache[0]) + id * (kv ? a.c_block[1] : a.c_block[0]) + h * (kv ? a.c_head[1] : a.c_head[0]);
  float* sp = (kv ? a.scale[1] : a.scale[0]) + id * (kv ? a.s_block[1] : a.s_block[0]) + h;
  const float old = first > 0 ? *sp : 0.f;
  // the thread's pieces: column `me % PPR` of the rows row0, row0 + RS, ... (one 64-bit step each, no products)
  constexpr int RS = NT / PPR;
  const int row0 = me / PPR;
  const bf16* const src = x + static_cast<int64_t>(t0 + row0) * ts + (me % PPR) * 8;
  const int64_t src_step = RS * ts;
  uint4 keep[kKeep];
  uint32_t bits = 0;
  const bool all = n >= kKeep * RS;  // every thread keeps kKeep pieces: no branch for each
  {
    const bf16* q = src;
    if (all) {
#pragma unroll
      for (int k = 0; k < kKeep; ++k, q += src_step) keep[k] = __ldg(reinterpret_cast<const uint4*>(q));
#pragma unroll
      for (int k = 0; k < kKeep; ++k) bits = max(bits, amax_bits(keep[k]));
    } else {
#pragma unroll
      for (int k = 0; k < kKeep; ++k, q += src_step) {
        keep[k] = make_uint4(0, 0, 0, 0);
        if (row0 + k * RS < n) keep[k] = __ldg(reinterpret_cast<const uint4*>(q));
      }
#pragma unroll
      for (int k = 0; k < kKeep; ++k) bits = max(bits, amax_bits(keep[k]));
    }
    for (int r = row0 + kKeep * RS; r < n; r += RS, q += src_step) bits = max(bits, amax_bits(__ldg(reinterpret_cast<const uint4*>(q))));
  }
  const bool finite = bits < kInfBits;
  if (!finite) {
    bits = 0;
    for (int r = row0; r < n; r += RS)
      bits = max(bits, amax_bits_finite(__ldg(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(r - row0) * ts))));
  }
  float m = __uint_as_float(__reduce_max_sync(0xffffffffu, bits) << 16);
  auto team_sync = [&]() {
    if constexpr (NT > 32) asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(NT) : "memory");
    else __syncwarp();
  };
  if constexpr (NT > 32) {
    if (me % 32 == 0) red[me / 32] = m;
    team_sync();
    m = red[0];
#pragma unroll
    for (int w = 1; w < NT / 32; ++w) m = fmaxf(m, red[w]);
  }
  int e = scale_exponent<FMT>(m);
  if (old > 0.f && old <= 3.4028234e38f) {  // a held scale stays unless the new tokens need a larger one (a scale that is no power of two: the next)
    int xo;
    const float mo = frexpf(old, &xo);
    e = max(e, mo == 0.5f ? xo - 1 : xo);
  }
  e = min(e, 126);
  const float scale = exp2i(e), inv = exp2i(-e);
  if (first > 0 && old != scale) {  // the tokens that the block holds, onto the new scale
    const float ratio = old * inv;
    for (int i = me; i < first * (D / 4); i += NT) {
      uint32_t* p = reinterpret_cast<uint32_t*>(rows + (i / (D / 4)) * ct + (i % (D / 4)) * 4);
      uint32_t lo, hi;
      Kv<FMT>::decode4(*p, lo, hi);
      const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&lo));
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hi));
      *p = Kv<FMT>::encode4(u.x * ratio, u.y * ratio, v.x * ratio, v.y * ratio);
    }
  }
  uint8_t* const dst = rows + static_cast<int64_t>(first + row0) * ct + (me % PPR) * 8;
  auto put = [&](int r, uint8_t* to, const uint4& w) {
    if (!straight) to = rows + static_cast<int64_t>(a.slots[t0 + r] - static_cast<int>(id) * a.block) * ct + (me % PPR) * 8;
    *reinterpret_cast<uint2*>(to) = finite ? encode8<FMT, true>(w, inv) : encode8<FMT, false>(w, inv);
  };
  {
    uint8_t* q = dst;
    if (all && straight && finite) {
#pragma unroll
      for (int k = 0; k < kKeep; ++k, q += RS * ct) *reinterpret_cast<uint2*>(q) = encode8<FMT, true>(keep[k], inv);
    } else {
#pragma unroll
      for (int k = 0; k < kKeep; ++k, q += RS * ct)
        if (row0 + k * RS < n) put(row0 + k * RS, q, keep[k]);
    }
    for (int r = row0 + kKeep * RS; r < n; r += RS, q += RS * ct)
      put(r, q, __ldg(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(r - row0) * ts)));
  }
  team_sync();  // `red` and the old scale have been read
  if (me == 0) *sp = scale;
}

// A block of threads owns the runs (neighbouring tokens of one cache block) that begin in its `rows` tokens; each of its
// teams writes them for `turns` (head, keys or values) pairs. So every (cache block, head) has one owner and the scale needs
// no atomics. A run is read once: a thread keeps its pieces in registers between the search for the largest magnitude and
// the rounding, which sets the team's size (NT = block * D / 64 threads; a longer run's rest is read again, from L2).
// Bound by HBM for prompts (2 bytes read, 1 written per number), by the latency of dependent reads for decode. With a block
// of threads per (run, head) and 4 KB of each run in flight, prompts ran at 16% of HBM; with a warp per pair the runs are
// looked for once per eight pairs.
// Measured on a B200: 24 prompts of 14900 tokens in all, bf16 to int8, 16 heads of 64 each for keys and values: 24.2 us,
// 3.8 TB/s, 58% of the measured copy rate. No unit is full: the issue slots are busy for 49%, a third of the warps is resident
// (80 registers a thread), so too few bytes are on their way; and the pairs do not divide evenly (there, half of the blocks
// take three turns and half one). 32 single tokens 4.4 us, one launch's latency.
template <int FMT, int D, int NT>
__global__ void __launch_bounds__(kAppendThreads, 3) append_kernel(AppendArgs a) {
  constexpr int kTeams = kAppendThreads / NT;
  __shared__ float s_red[kAppendThreads / 32];
  const int lane = threadIdx.x % 32, team = threadIdx.x / NT, me = threadIdx.x % NT;
  griddep_wait();
  griddep_launch();
  const int r0 = blockIdx.x * a.rows, r1 = min(r0 + a.rows, a.T);
  // a token's slot; -1: none (padding, or a slot that the cache does not have)
  auto slot_of = [&](int t) {
    const int s = t >= 0 && t < a.T ? a.slots[t] : -1;
    return s >= 0 && a.by_block.quotient(s) < a.blocks ? s : -1;
  };
  auto block_of = [&](int s) { return s < 0 ? -1 : a.by_block.quotient(s); };
  // Every warp looks for the runs itself: they are few, and nothing has to be waited for. The slots of 64 tokens are read at
  // once, so that what most runs need to be found is there after one latency.
  for (int base = r0; base < r1; base += 32) {
    const int slots[2] = {slot_of(base + lane), slot_of(base + 32 + lane)};
    const int before = block_of(slot_of(base + lane - 1));
    const int ids[2] = {block_of(slots[0]), block_of(slots[1])};
    unsigned heads = __ballot_sync(0xffffffffu, base + lane < r1 && ids[0] >= 0 && ids[0] != before);
    while (heads) {
      const int at = __ffs(heads) - 1;
      heads &= heads - 1;
      const int t0 = base + at, id = __shfl_sync(0xffffffffu, ids[0], at), slot0 = __shfl_sync(0xffffffffu, slots[0], at);
      const unsigned others[2] = {~(__ballot_sync(0xffffffffu, ids[0] == id) >> at), ~__ballot_sync(0xffffffffu, ids[1] == id)};
      int n = __ffs(others[0]) - 1;  // a shift leaves zeros at the top; none for at = 0
      if (others[0] == 0) n = 32;
      if (at + n == 32) n += others[1] ? __ffs(others[1]) - 1 : 32;
      if (at + n == 64) {
        while (n < a.block) {
          const unsigned other = __ballot_sync(0xffffffffu, block_of(slot_of(t0 + n + lane)) != id);
          n += other ? __ffs(other) - 1 : 32;
          if (other) break;
        }
      }
      n = min(n, a.block);
      // Ascending slots as many as their span are consecutive; others (a plan never makes them) are looked up one by one.
      const int last = at + n - 1, in = __shfl_sync(0xffffffffu, last < 32 ? slots[0] : slots[1], last & 31);
      const bool straight = (last < 64 ? in : a.slots[t0 + n - 1]) - slot0 == n - 1;
      const int first = a.by_block.remainder(slot0, id);
      for (int k = 0; k < a.turns; ++k) {
        const int pair = (blockIdx.y * a.turns + k) * kTeams + team;
        if (pair < 2 * a.Hkv)
          append_run<FMT, D, NT>(a, pair & 1, pair >> 1, t0, n, id, first, straight, team, me, s_red + team * (NT / 32));
      }
    }
  }
}

template <int FMT, int D, int NT>
void append_launch(AppendArgs a, cudaStream_t stream) {
  constexpr int kTeams = kAppendThreads / NT;
  const int groups = (2 * a.Hkv + kTeams - 1) / kTeams;
  // few tokens: one per block of threads and one pair per team, for latency; many: a cache block of tokens, so that a
  // prompt's runs have one owner each, and all pairs of a few hundred blocks per SM in one
  a.rows = std::max(1, std::min({a.block, kAppendRows, static_cast<int>(static_cast<int64_t>(a.T) * groups / (148 * 4))}));
  const int64_t tiles = (a.T + a.rows - 1) / a.rows;
  a.turns = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(groups, tiles * groups / (148 * 4))));
  const dim3 grid(static_cast<unsigned>(tiles), (groups + a.turns - 1) / a.turns);
  launch_pdl(append_kernel<FMT, D, NT>, grid, dim3(kAppendThreads), 0, stream, "append_kv", a);
}

template <int FMT, int D>
void append_team(const AppendArgs& a, cudaStream_t stream) {
  const int pieces = a.block * (D / 8);
  if (pieces <= 32 * kKeep) append_launch<FMT, D, 32>(a, stream);
  else if (pieces <= 64 * kKeep) append_launch<FMT, D, 64>(a, stream);
  else append_launch<FMT, D, 128>(a, stream);
}

template <int FMT>
void append_dim(const AppendArgs& a, int D, cudaStream_t stream) {
  if (D == 32) append_team<FMT, 32>(a, stream);
  else if (D == 64) append_team<FMT, 64>(a, stream);
  else append_team<FMT, 128>(a, stream);
}

}  // namespace

int plan_max_requests() { return 4096; }

void plan_blocks(const int* cached, const int* fresh, const int* state, int* table, int64_t table_stride,
                 const int* free_blocks, int capacity, int B, int width, int block, int tokens, int* query_start,
                 int* context, int* positions, int* slots, int* state_out, int* missing, cudaStream_t stream) {
  PlanArgs a{cached, fresh, state, table, table_stride, free_blocks, capacity, B, width, block, tokens,
             query_start, context, positions, slots, state_out, missing};
  const int grid = std::min(148, std::max((tokens + kPlanTokens - 1) / kPlanTokens, (B + 63) / 64));
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, current_device(), [] {
    check_cuda(cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>((5 * plan_max_requests() + 1) * sizeof(int))),
               "plan_blocks smem");
  });
  launch_pdl(plan_kernel, dim3(std::max(grid, 1)), dim3(kPlanThreads), static_cast<size_t>(5 * B + 1) * sizeof(int), stream,
             "plan_blocks", a);
}

void release_blocks(const int* keep, int* state, int* table, int64_t table_stride, int* free_blocks, int capacity, int B,
                    int width, int block, cudaStream_t stream) {
  if (B == 0) return;
  launch_pdl(release_kernel, dim3(1), dim3(kPlanThreads), 0, stream, "release_blocks", keep, state, table, table_stride,
             free_blocks, capacity, B, width, block);
}

void append_kv(const KvSource& k, const KvSource& v, const int* slots, const KvPages& kc, const KvPages& vc, int T, int Hkv,
               int D, int block, int blocks, int fmt, cudaStream_t stream) {
  if (T == 0) return;
  AppendArgs a{};
  a.by_block = Divisor(block);
  const KvSource* src[2] = {&k, &v};
  const KvPages* dst[2] = {&kc, &vc};
  for (int i = 0; i < 2; ++i) {
    a.x[i] = src[i]->x;
    a.token_stride[i] = src[i]->token_stride;
    a.head_stride[i] = src[i]->head_stride;
    a.cache[i] = static_cast<uint8_t*>(const_cast<void*>(dst[i]->codes));
    a.c_block[i] = dst[i]->block_stride;
    a.c_head[i] = dst[i]->head_stride;
    a.c_token[i] = dst[i]->token_stride;
    a.scale[i] = const_cast<float*>(dst[i]->scale);
    a.s_block[i] = dst[i]->scale_stride;
  }
  a.slots = slots;
  a.T = T;
  a.Hkv = Hkv;
  a.block = block;
  a.blocks = blocks;
  if (fmt == kKvFp8) append_dim<kKvFp8>(a, D, stream);
  else append_dim<kKvInt8>(a, D, stream);
}

}  // namespace qw
