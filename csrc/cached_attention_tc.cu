// Attention over the block-wise 8-bit KV cache for prompts: tcgen05.mma with TMEM accumulators (head_dim 64 and 128).
//
//   S_g  = Q_g K_j^T        TMEM, 128 rows x 128 keys per group; Q and K (f16) from shared memory
//   P_g  = exp2(S_g * scale * k_scale - m_g) * v_scale / v_ref     softmax warps, f16, TMEM
//   O_g += P_g V_j          TMEM, 128 x D; P_g from TMEM, V_j from shared memory
//
// A block of threads owns query rows (new tokens x the query heads of one kv head) of one request and walks the request's
// cache in tiles of 128 keys. With head_dim 128 it has 256 rows as two groups of 128, so that the tensor core works on one
// group's tiles while the other's scores become probabilities, and the widening is shared by 256 rows (about 2 instructions
// per code against 256 x 4 flops). With head_dim 64 it has one group, and two blocks share an SM: prompts of a few hundred
// tokens have few tiles per block, and the second block works while the first begins or ends. Where the row
// tiles are fewer than the SMs hold, the keys are split as well and a second kernel adds up.
//
// No TMA: the operands are not in memory as the tensor core wants them. Four warps fetch the codes of each tile by the block
// table (cp.async, a whole tile ahead), widen them to f16 (every code is one) and store them in the 128-byte-swizzled layout;
// the scales of the tile's 16-key groups go beside it and are applied in 32 bits, as in the kernel for few rows
// (cached_attention.cu), whose rules for masks, row factors and value scales hold here too.
//
// Probabilities come from 32-bit exponentials: f16x2 ones would halve the special-function work, but the rounding of
// their argument costs 2^-8 relative at arguments of 8.
//
// TMEM: S_g, then O_g (D columns each). head_dim 64 (256 columns) has room for P behind them; head_dim 128 (512 columns) has
// none, so P_g lies in S_g (each half of the weights in the columns of its own keys), and the next S_g is issued only once
// P_g V has completed. A thread reads its scores twice (maximum, then exponentials, 32 columns at a time): kept in between,
// they cost the registers that a second block (or the second group) needs, and took longer.
//
// Warps: 0-3 widen; then eight softmax warps per group, two threads per row; then one warp per group that issues its MMAs,
// converged (from a single diverged thread an N = 128 MMA took 93 to 105 cycles instead of 64). Every wait is bounded
// (common.cuh); on a timeout all roles stop, MMAs in flight are waited for, TMEM is freed and the status word records the
// cause.
//
// Measured on a B200: 2048 new tokens after 14337, 32 heads on 8 of 128, fp8: 581-593 us, 870-890 TFLOP/s, 53% of the
// measured bf16 rate. Bound by the chain S -> maximum -> exponentials -> P V of two groups that share the tensor core (its pipe
// is busy for 47% of the active cycles, the special-function units for 51%) and by the last wave: 256 row tiles on 148 SMs. Splitting the tiles of that wave
// over the keys gave back in partial results what it won. 16 ragged prompts of up to 2048 tokens, 16 heads of 64, int8:
// 128 us, 268 TFLOP/s: a block has five tiles on average, so its beginning and end and the masked tile on the diagonal count
// as much as the tiles; 57% of the issue slots are busy.
#include <algorithm>
#include <type_traits>

#include "cached_attention.cuh"
#include "common.cuh"
#include "kv_format.cuh"
#include "launch.cuh"
#include "launchers.h"

namespace qw {
namespace {

constexpr int KT = 128;        // keys of a tile
constexpr int kGroupRows = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -3e38f;       // running maximum of a row that has seen no key
constexpr float kLazy = 6.f;          // the running maximum moves when a row grows by more than 2^6
constexpr float kWeightUpLog2 = 8.f;  // weights in f16: at most 2^14

template <int D>
struct Layout {
  static constexpr int kGroups = D == 64 ? 1 : 2;
  static constexpr int kRows = kGroups * kGroupRows;         // rows of a block of threads
  static constexpr int kIssuer = 4 + 8 * kGroups;            // first of the issuing warps
  static constexpr int kThreads = (kIssuer + kGroups) * 32;
  static constexpr bool kAlias = D == 128;                   // P_g in S_g's columns
  static constexpr int kStages = 2;
  static constexpr int kBoxes = D / 64;                      // 64-wide (128-byte) column boxes
  static constexpr int kQBytes = kBoxes * kGroupRows * 128;  // one group's rows
  static constexpr int kTileBytes = kBoxes * KT * 128;       // one K or V tile
  static constexpr int kKV = kGroups * kQBytes;              // stages of [K | V]
  static constexpr int kScale = kKV + kStages * 2 * kTileBytes;  // stages of k_scale[8], v_scale[8]
  static constexpr int kRaw = kScale + kStages * 64;         // codes of one K and one V tile on their way
  static constexpr int kPoison = kRaw + 2 * KT * D;
  static constexpr int kJoin = kPoison + D * 4;              // [groups][2 halves][128 rows]: maxima, at the end sums
  static constexpr int kBar = kJoin + kGroups * 1024;
  static constexpr int kBarriers = 21 + 3 * kStages;         // at most (see the pointers in the kernel)
  static constexpr int kTotal = kBar + kBarriers * 8 + 32;   // and eight words
  static constexpr int kTmemO = kGroups * KT;
  static constexpr int kTmemP = kAlias ? 0 : kTmemO + kGroups * D;  // 128 columns apart where P_g lies in S_g
  static constexpr int kTmemCols = kGroups * 256;
  static constexpr int kPHalf = kAlias ? 64 : 32;            // columns from the first 64 keys' weights to the others'
  static_assert(kTotal <= (kGroups == 1 ? 113 : 227) * 1024, "shared memory per block");
  static_assert(kRows == prompt_rows(D) && prompt_per_sm(D) == 3 - kGroups, "what the host counts on");
  static_assert(kAlias || kTmemP + kGroups * KT / 2 <= kTmemCols, "tensor memory");
};

// Instruction descriptor, kind::f16 with f16 operands and fp32 accumulators.
constexpr uint32_t idesc_f16(int n, bool b_mn_major) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 32 lanes x 32 bit, 16 consecutive columns per thread, raw words.
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// 16 bytes of global memory into shared memory, or zeros.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const uint8_t* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

struct TcArgs {
  CachedAttn p;
  int splits;
};

template <int FMT, int D>
__global__ void __launch_bounds__(Layout<D>::kThreads, 3 - Layout<D>::kGroups) cached_attn_tc_kernel(const __grid_constant__ TcArgs args) {
  using L = Layout<D>;
  constexpr int kStages = L::kStages;
  constexpr int G = L::kGroups;
  constexpr int kRows = L::kRows;
  constexpr int kIssuer = L::kIssuer;
  constexpr int kThreads = L::kThreads;
  const CachedAttn& p = args.p;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;  // the swizzle wants 1 KB; checked below
  float* s_scale = reinterpret_cast<float*>(smem + L::kScale);  // [stage][2][8]
  int* s_poison = reinterpret_cast<int*>(smem + L::kPoison);
  float* s_join = reinterpret_cast<float*>(smem + L::kJoin);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* k_full = q_full + 1;
  uint64_t* v_full = k_full + kStages;
  uint64_t* kv_empty = v_full + kStages;
  uint64_t* s_full = kv_empty + kStages;  // [2] S_g of the next tile is in TMEM
  uint64_t* p_full = s_full + 2;          // [2][2] P_g's keys 0-31, 64-95 (then the others) are written, O_g rescaled
  uint64_t* o_full = p_full + 4;          // [2] O_g += P_g V has completed
  uint64_t* met = o_full + 2;             // [8] the two warps of 32 rows meet
  uint64_t* turn = met + 8;               // [2]
  uint64_t* teardown = turn + 2;          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(teardown + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_item = reinterpret_cast<int*>(tmem_slot + 2);  // request, row tile, all row tiles, first row, new rows, context

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (smem_u32(smem) & 1023) {  // never with dynamic shared memory alone
    if (threadIdx.x == 0) set_status(kBoundsError);
    return;
  }
  griddep_wait();

  // ---- which request and row tile: the last tiles, which see the most keys, come first
  if (warp == 0) {
    auto tiles_of = [&](const NewRows& x) {
      return x.n > 0 ? static_cast<int>((static_cast<int64_t>(x.n) * p.group + kRows - 1) / kRows) : 0;
    };
    // the first 32 requests stay in registers between the two passes
    const NewRows mine = lane < p.B ? new_rows(p, lane) : NewRows{0, 0};
    const int my_ctx = lane < p.B ? p.context[lane] : 0;
    int total = tiles_of(mine);
    for (int b = lane + 32; b < p.B; b += 32) total += tiles_of(new_rows(p, b));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    // Requests whose rows overlap (offsets that do not ascend) could have more tiles than the grid and the partial results have
    // room for: those past the bound are left out, and the status word says so.
    const int most = static_cast<int>(gridDim.x) / p.Hkv;
    if (total < 0 || total > most) {
      if (lane == 0) set_status(kBoundsError);
      total = total < 0 ? 0 : most;
    }
    const int want = total - 1 - static_cast<int>(blockIdx.x) / p.Hkv;
    const bool publish = args.splits > 1 && blockIdx.x == 0 && blockIdx.y == 0;  // for the join kernel
    if (lane == 0) {
      s_item[0] = -1;
      s_item[2] = total;
    }
    __syncwarp();
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int b = b0 + lane;
      const NewRows rows_b = b0 == 0 ? mine : b < p.B ? new_rows(p, b) : NewRows{0, 0};
      const int w = tiles_of(rows_b);
      int x = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const int at = before + x - w;
      if (want >= max(at, 0) && want < at + w) {
        s_item[0] = b;
        s_item[1] = want - at;
        s_item[3] = rows_b.first;
        s_item[4] = rows_b.n;
        s_item[5] = b0 == 0 ? my_ctx : p.context[b];
      }
      if (publish && b < p.B) p.prefix[b] = at;
      before += __shfl_sync(0xffffffffu, x, 31);
    }
  } else if (warp == kIssuer) {
    tmem_alloc(tmem_slot, L::kTmemCols);  // freed below where the block has nothing to do
  }
  for (int i = threadIdx.x; i < D; i += kThreads) s_poison[i] = 0x7fffffff;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 8 * G);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&v_full[s], 4);
      mbar_init(&kv_empty[s], G);
    }
    for (int g = 0; g < G; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[2 * g], 8);
      mbar_init(&p_full[2 * g + 1], 8);
      mbar_init(&o_full[g], 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&met[i], 2);
    mbar_init(&turn[0], 8);
    mbar_init(&turn[1], 8);
    mbar_init(&teardown[0], 1);
    mbar_init(&teardown[1], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  const int b = s_item[0], row_tile = s_item[1];
  const int h = static_cast<int>(blockIdx.x) % p.Hkv;

  // rows that belong to no request are zero
  if (blockIdx.x < static_cast<unsigned>(p.Hkv) && blockIdx.y == 0) {
    const int first = p.B > 0 ? min(max(p.query_start[0], 0), p.T) : p.T;
    const int last = p.B > 0 ? min(max(p.query_start[p.B], first), p.T) : p.T;
    const int rows = first + p.T - last;
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(rows) * p.group * (D / 8); i += kThreads) {
      const int r = static_cast<int>(i / (p.group * (D / 8))), c = static_cast<int>(i % (p.group * (D / 8)));
      const int64_t tok = r < first ? r : last + (r - first);
      *reinterpret_cast<uint4*>(p.out + tok * p.o_token + (h * p.group + c / (D / 8)) * p.o_head + (c % (D / 8)) * 8) =
          make_uint4(0, 0, 0, 0);
    }
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (b < 0) {  // the grid is an upper bound
    if (warp == kIssuer) tmem_dealloc(tmem, L::kTmemCols);
    griddep_launch();
    return;
  }

  const int q0 = s_item[3], n = s_item[4], all_ctx = s_item[5];
  const int ctx = min(all_ctx, p.max_table_tokens);
  const int row0 = row_tile * kRows;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kRows), static_cast<int64_t>(n) * p.group - row0));
  // keys that a row of the tile sees: [0, lim)
  auto lim_of = [&](int row) { return min(ctx, all_ctx - n + p.by_group.quotient(row0 + min(row, rows - 1)) + 1); };
  const int lim_all = lim_of(0), lim_any = lim_of(rows - 1);
  const int tiles = lim_any > 0 ? (lim_any + KT - 1) / KT : 0;
  const int per = (tiles + args.splits - 1) / args.splits;
  const int t0 = min(tiles, static_cast<int>(blockIdx.y) * per), t1 = min(tiles, t0 + per);
  auto tiles_of_group = [&](int g) {
    if (rows <= g * kGroupRows) return 0;
    const int lim = lim_of(min(rows, (g + 1) * kGroupRows) - 1);
    return max(0, min(t1, lim > 0 ? (lim + KT - 1) / KT : 0) - t0);
  };
  const int n0 = tiles_of_group(0), n1 = G == 2 ? tiles_of_group(1) : 0;
  const int nk = max(n0, n1);

  if (warp < 4) {
    // ------------------------------------------------------------------ codes -> f16 tiles in shared memory
    // A thread widens one 16-byte piece of every KPP-th key. Four lanes hold a key's pieces of one 64-column box and the next
    // four the next key's: their f16 halves, swizzled, fall on different banks.
    constexpr int KPP = 128 / (D / 16);
    constexpr int NP = 64 / KPP;         // keys per thread of a half tile (64 keys)
    const int key_in = (threadIdx.x / 4) % KPP, box = threadIdx.x / (4 * KPP);
    const int piece = box * 4 + threadIdx.x % 4;
    const int* table = p.table + static_cast<int64_t>(b) * p.table_stride;
    // the thread's byte in a 16-key group, and its places in a tile (they repeat every 8 keys)
    const uint8_t* base[2] = {p.k.codes + static_cast<int64_t>(h) * p.k.head_stride + (key_in % 16) * p.k.token_stride + piece * 16,
                              p.v.codes + static_cast<int64_t>(h) * p.v.head_stride + (key_in % 16) * p.v.token_stride + piece * 16};
    const int put = box * (KT * 128) + key_in * 128;
    const int put0 = put + (((piece % 4) * 2) ^ (key_in & 7)) * 16, put1 = put + (((piece % 4) * 2 + 1) ^ (key_in & 7)) * 16;
    // Lanes 0-7 look up the tile's 16-key groups: where the keys and values begin (-1: masked, without a block or past the
    // last key that a row sees) and their scales. The block's id is read three tiles ahead and used two ahead, so that no
    // thread waits for the dependent reads.
    struct Groups {
      int64_t at[2];
      float scale[2];
    };
    auto id_of = [&](int j) {
      const int key = (t0 + j) * KT + lane * 16;
      return lane < 8 && j < nk && key < lim_any ? __ldg(table + p.by_block.quotient(key)) : -1;
    };
    auto groups_of = [&](int j, int id) {
      Groups x{{-1, -1}, {-1.f, 0.f}};
      if (static_cast<unsigned>(id) < static_cast<unsigned>(p.blocks)) {
        const int key = (t0 + j) * KT + lane * 16;
        const uint32_t in = p.by_block.remainder(key, p.by_block.quotient(key));
        const uint64_t u = static_cast<uint32_t>(id);
        x.at[0] = static_cast<int64_t>(u * p.k.block_stride + in * p.k.token_stride);
        x.at[1] = static_cast<int64_t>(u * p.v.block_stride + in * p.v.token_stride);
        if (warp == 0) {
          x.scale[0] = __ldg(p.k.scale + u * p.k.scale_stride + h);
          x.scale[1] = __ldg(p.v.scale + u * p.v.scale_stride + h);
        }
      }
      return x;
    };
    // The half tiles K lower, K upper, V lower, V upper: each fetched a whole tile before it is widened, into places of
    // the thread's own (loads into registers wait for one another: a warp has few scoreboards).
    uint8_t* raw = smem + L::kRaw + threadIdx.x * 16;
    const uint32_t raw_u32 = smem_u32(raw);
    auto fetch = [&](auto which, int half, const Groups& x) {
      constexpr int kv = decltype(which)::value;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, x.at[kv], half * 4 + (key_in + i * KPP) / 16);
        cp_async16_or_zero(raw_u32 + ((2 * kv + half) * NP + i) * 2048, at >= 0 ? base[kv] + at : base[kv], at >= 0);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto store = [&](auto which, int half, int j) {
      constexpr int kv = decltype(which)::value;
      asm volatile("cp.async.wait_group 3;" ::: "memory");  // four groups are on their way: the oldest has come
      uint4 r[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) r[i] = *reinterpret_cast<const uint4*>(raw + ((2 * kv + half) * NP + i) * 2048);
      uint8_t* dst = smem + L::kKV + (j % kStages) * 2 * L::kTileBytes + kv * L::kTileBytes + half * 64 * 128;
      if (kv == 1 && (t0 + j + 1) * KT > lim_all) {
        // Keys that only some rows see: values past the last one may be anything and count as zero, and a NaN must not
        // reach the rows that do not see it.
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int key = (t0 + j) * KT + half * 64 + key_in + i * KPP;
          if (key >= lim_any) r[i] = make_uint4(0, 0, 0, 0);
          if (key >= lim_all) {
            uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t bad = Kv<FMT>::nan_bytes(w[c]);
              if (bad)
                for (int e = 0; e < 4; ++e)
                  if ((bad >> (8 * e + 7)) & 1) {
                    atomicMin(&s_poison[piece * 16 + c * 4 + e], key);
                    w[c] &= ~(0xffu << (8 * e));
                  }
            }
            r[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        uint4 lo, hi;
        Kv<FMT>::decode4(r[i].x, lo.x, lo.y);
        Kv<FMT>::decode4(r[i].y, lo.z, lo.w);
        Kv<FMT>::decode4(r[i].z, hi.x, hi.y);
        Kv<FMT>::decode4(r[i].w, hi.z, hi.w);
        *reinterpret_cast<uint4*>(dst + put0 + i * KPP * 128) = lo;
        *reinterpret_cast<uint4*>(dst + put1 + i * KPP * 128) = hi;
      }
    };
    auto arrive = [&](uint64_t* bar) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    using K_ = std::integral_constant<int, 0>;
    using V_ = std::integral_constant<int, 1>;
    Groups now = groups_of(0, id_of(0)), next = groups_of(1, id_of(1));
    int id = id_of(2);
    fetch(K_{}, 0, now);
    fetch(K_{}, 1, now);
    fetch(V_{}, 0, now);
    fetch(V_{}, 1, now);
    for (int j = 0; j < nk; ++j) {
      const int st = j % kStages;
      const bool ok = mbar_wait(&kv_empty[st], ((j / kStages) & 1) ^ 1, kTimeoutEmpty);
      if (!__all_sync(0xffffffffu, ok)) {
        *abort_flag = 1;
        break;
      }
      if (warp == 0 && lane < 8) {
        s_scale[st * 16 + lane] = now.scale[0];
        s_scale[st * 16 + 8 + lane] = __log2f(now.scale[1]);
      }
      store(K_{}, 0, j);
      fetch(K_{}, 0, next);
      store(K_{}, 1, j);
      fetch(K_{}, 1, next);
      arrive(&k_full[st]);
      store(V_{}, 0, j);
      fetch(V_{}, 0, next);
      store(V_{}, 1, j);
      fetch(V_{}, 1, next);
      arrive(&v_full[st]);
      now = next;
      next = groups_of(j + 2, id);
      id = id_of(j + 3);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= kIssuer) {
    // ------------------------------------------------------------------ MMA issuers, one warp per group
    // The whole warp runs this, converged (umma_f16_warp); one lane issues. A warp of its own for each group waits for
    // exactly the next thing that the group needs; one that polled for both took 500 cycles to notice.
    constexpr uint32_t kAll = 0xffffffffu;
    constexpr uint32_t id_s = idesc_f16(KT, false);
    constexpr uint32_t id_o = idesc_f16(D, true);
    const uint32_t elect = elect_one();
    const int g = __shfl_sync(kAll, warp, 0) - kIssuer;
    const int count = __shfl_sync(kAll, g == 0 ? n0 : n1, 0), all = __shfl_sync(kAll, nk, 0);
    const uint32_t acc = __shfl_sync(kAll, tmem, 0);
    const uint32_t t_s = acc + g * KT, t_o = acc + L::kTmemO + g * D, t_p = acc + L::kTmemP + g * KT;
    const uint64_t dq = smem_desc_sw128(smem_u32(smem) + g * L::kQBytes, 16, 1024);
    const uint64_t dk0 = smem_desc_sw128(smem_u32(smem + L::kKV), 16, 1024);
    const uint64_t dv0 = smem_desc_sw128(smem_u32(smem + L::kKV + L::kTileBytes), KT * 128, 1024);
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase, int code) {
      ok = ok && __all_sync(kAll, mbar_wait(bar, phase & 1, code)) != 0;
      return ok;
    };
    auto issue_s = [&](int j) {
      const uint64_t dk = dk0 + static_cast<uint32_t>((j % kStages) * ((2 * L::kTileBytes) >> 4));
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        umma_f16_warp(t_s, dq + (((k / 4) * (kGroupRows * 128) + (k % 4) * 32) >> 4),
                      dk + (((k / 4) * (KT * 128) + (k % 4) * 32) >> 4), id_s, k > 0 ? 1u : 0u, elect);
      umma_commit_warp(&s_full[g], elect);
    };
    auto issue_o = [&](int j, int part) {
      const uint64_t dv = dv0 + static_cast<uint32_t>((j % kStages) * ((2 * L::kTileBytes) >> 4));
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = (i & 1) + (i >> 1) * 4 + part * 2;
        umma_f16_ts_warp(t_o, t_p + (k / 4) * L::kPHalf + (k % 4) * 8, dv + ((k * 2048) >> 4), id_o,
                         i > 0 || part > 0 || j > 0 ? 1u : 0u, elect);
      }
    };
    if (count > 0 && wait(q_full, 0, kTimeoutFull) && wait(&k_full[0], 0, kTimeoutFull)) issue_s(0);
    for (int j = 0; ok && j < count; ++j) {
      const bool more = j + 1 < count;
      if (!wait(&v_full[j % kStages], j / kStages, kTimeoutFull)) break;
      if (!wait(&p_full[2 * g], j, kTimeoutAccum)) break;
      issue_o(j, 0);
      if (more && !wait(&k_full[(j + 1) % kStages], (j + 1) / kStages, kTimeoutFull)) break;
      if (!wait(&p_full[2 * g + 1], j, kTimeoutAccum)) break;
      if (!L::kAlias && more) issue_s(j + 1);  // S_g has been read when all weights are written
      issue_o(j, 1);
      umma_commit_warp(&o_full[g], elect);
      umma_commit_warp(&kv_empty[j % kStages], elect);
      if (L::kAlias && more) {
        if (!wait(&o_full[g], j, kTimeoutAccum)) break;
        issue_s(j + 1);
      }
    }
    if (!ok) *abort_flag = 1;
    for (int j = count; ok && j < all; ++j) {  // tiles that only the other group needs
      if (!wait(&v_full[j % kStages], j / kStages, kTimeoutFull)) break;
      if (elect) mbar_arrive(&kv_empty[j % kStages]);
    }
    umma_commit_warp(&teardown[g], elect);  // fires once every MMA issued above has completed
    mbar_wait(&teardown[g], 0, kTimeoutAccum);
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax
    // Two threads share a row: each makes the weights of 64 of a tile's keys and rescales and writes half of the row's output.
    // Four such warps on a sub-partition hide each other's latencies; two took 1.5 times as long for a tile.
    const int g = (warp - 4) / 8, half = (warp - 4) / 4 % 2;
    const int row = (warp % 4) * 32 + lane;     // of the group = TMEM lane
    const int r = g * kGroupRows + row;         // of the tile
    const int n_g = g == 0 ? n0 : n1;
    const bool real = r < rows;
    const int row_tok = p.by_group.quotient(row0 + r);
    const int tok = q0 + row_tok, head = h * p.group + p.by_group.remainder(row0 + r, row_tok);
    const uint32_t lane_off = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t ts = tmem + lane_off + g * KT + half * 64;
    const uint32_t to = tmem + lane_off + L::kTmemO + g * D + half * (D / 2);
    const uint32_t tp = tmem + lane_off + L::kTmemP + g * KT + half * L::kPHalf;
    float* const s_mine = s_join + (g * 2 + half) * kGroupRows + row;
    const float* const s_other = s_join + (g * 2 + 1 - half) * kGroupRows + row;
    // the two warps of the same 32 rows (a barrier whose wait is bounded)
    uint64_t* const my_met = &met[g * 4 + warp % 4];
    auto meet = [&](int phase) {
      __syncwarp();
      if (lane == 0) mbar_arrive(my_met);
      return __all_sync(0xffffffffu, mbar_wait(my_met, phase & 1, kTimeoutAccum)) != 0;
    };
    {
      // Query rows in f16, each divided by a power of two (kQueryTop). D / 8 lanes read a row.
      constexpr int LPR = D / 8, RPI = 32 / LPR, NI = 16 / RPI;  // a warp has 16 rows
      const int c = lane % LPR, w16 = (warp - 4) % 8;
      uint4 w[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int rr = g * kGroupRows + w16 * 16 + i * RPI + lane / LPR, rt = p.by_group.quotient(row0 + rr);
        w[i] = make_uint4(0, 0, 0, 0);
        if (rr < rows)
          w[i] = __ldg(reinterpret_cast<const uint4*>(p.q + static_cast<int64_t>(q0 + rt) * p.q_token +
                                                      (h * p.group + p.by_group.remainder(row0 + rr, rt)) * p.q_head) + c);
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int in = w16 * 16 + i * RPI + lane / LPR;  // row of the group
        const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&w[i]);
        const float2 f0 = __bfloat1622float2(x[0]), f1 = __bfloat1622float2(x[1]), f2 = __bfloat1622float2(x[2]),
                     f3 = __bfloat1622float2(x[3]);
        float m = fmaxf(fmaxf(fmaxf(fabsf(f0.x), fabsf(f0.y)), fmaxf(fabsf(f1.x), fabsf(f1.y))),
                        fmaxf(fmaxf(fabsf(f2.x), fabsf(f2.y)), fmaxf(fabsf(f3.x), fabsf(f3.y))));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int e = min(max(static_cast<int>(__float_as_uint(m) >> 23) - 127, -100), 127);
        const bool fine = m > 0.f && m <= 3.4028234e38f;  // zero or infinite rows as they are
        const float inv = fine ? exp2i(kQueryTop - e) : 1.f;
        *reinterpret_cast<uint4*>(smem + g * L::kQBytes + (c / 8) * (kGroupRows * 128) + in * 128 + ((c % 8) ^ (in & 7)) * 16) =
            make_uint4(pack_f16(f0.x * inv, f0.y * inv), pack_f16(f1.x * inv, f1.y * inv), pack_f16(f2.x * inv, f2.y * inv),
                       pack_f16(f3.x * inv, f3.y * inv));
        if (c < 2)  // for the two threads of the row
          s_join[(g * 2 + c) * kGroupRows + in] = (fine ? exp2i(e - kQueryTop) : 1.f) * p.scale * kLog2e;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, kTimeoutFull)) != 0;
    const float unit = *s_mine;  // what a product of codes and fragments is worth, but for the key's scale
    const int lim = lim_of(r);
    const int lim_group = lim_of(g * kGroupRows);  // the group's first row sees the fewest keys
    // running maximum, sum (of this thread's keys), and log2 of the largest value scale that the row has seen
    float m_run = kNone, l_run = 0.f, v_ref = -INFINITY;
    for (int j = 0; ok && j < n_g; ++j) {
      const int st = j % kStages;
      // the scales are written before k_full completes; S_g comes after it
      if (!__all_sync(0xffffffffu, mbar_wait(&k_full[st], (j / kStages) & 1, kTimeoutFull) &&
                                       mbar_wait(&s_full[g], j & 1, kTimeoutAccum))) { ok = false; break; }
      tc_fence_after();
      const int k0 = (t0 + j) * KT;
      const int lim_tile = lim - k0 - half * 64;       // of this thread's 64 keys
      const float* sc = s_scale + st * 16;             // [8] key scales, [8] log2 of value scales
      const float* my_sc = sc + half * 4;
      bool plain = k0 + KT <= lim_group;               // the same for the whole warp: all rows see all 128 keys
      float v_top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 a = *reinterpret_cast<const float4*>(sc + i), c = *reinterpret_cast<const float4*>(sc + 8 + i);
        plain = plain && fminf(fminf(a.x, a.y), fminf(a.z, a.w)) >= 0.f;
        v_top = fmaxf(fmax3(v_top, c.x, c.y), fmaxf(c.z, c.w));
      }
      // ---- the row's maximum
      float mx = -INFINITY;
      if (plain) {
        float v[64];
        tmem_ld32_pair(ts, ts + 32, v, v + 32);
#pragma unroll
        for (int i = 0; i < 64; i += 16) {
          float a = fmax3(v[i], v[i + 1], v[i + 2]), d = fmax3(v[i + 3], v[i + 4], v[i + 5]);
          a = fmax3(a, v[i + 6], v[i + 7]);
          d = fmax3(d, v[i + 8], v[i + 9]);
          a = fmax3(a, v[i + 10], v[i + 11]);
          d = fmax3(d, v[i + 12], v[i + 13]);
          mx = fmaxf(mx, fmaxf(fmax3(a, v[i + 14], v[i + 15]), d) * my_sc[i / 16]);
        }
      } else {
        v_top = -INFINITY;
#pragma unroll 1
        for (int i = 0; i < 8; ++i)
          if (sc[i] >= 0.f && i * 16 < lim - k0) v_top = fmaxf(v_top, sc[8 + i]);
#pragma unroll 1
        for (int c = 0; c < 64; c += 16) {
          float v[16];
          tmem_ld16(ts + c, v);
          const float f = my_sc[c / 16];
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, f >= 0.f && c + i < lim_tile ? v[i] * f : -INFINITY);
        }
      }
      *s_mine = mx * unit;
      if (!meet(j)) { ok = false; break; }
      mx = fmaxf(mx * unit, *s_other);
      float factor = 1.f;
      bool rescale = false;
      if (__any_sync(0xffffffffu, mx > m_run + kLazy || v_top > v_ref)) {  // the same in both warps
        const float m_new = fmaxf(m_run, mx), v_new = fmaxf(v_ref, v_top);
        const float f = exp2f_approx(m_run - m_new);
        factor = v_ref == -INFINITY ? 0.f : f * exp2f_approx(v_ref - v_new);
        l_run *= f;
        m_run = m_new;
        v_ref = v_new;
        rescale = j > 0;
      }
      // O_g += P_g V of the tile before has to be complete before P_g (head_dim 64) or O_g is written
      // (head_dim 128: S_g came after it)
      if constexpr (!L::kAlias) {
        if (j > 0 && !__all_sync(0xffffffffu, mbar_wait(&o_full[g], (j - 1) & 1, kTimeoutAccum))) { ok = false; break; }
        tc_fence_after();
      }
      if (rescale) {
#pragma unroll 1
        for (int c = 0; c < D / 2; c += 32) {
          float o[32];
          tmem_ld32(to + c, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= factor;
          tmem_st32(to + c, o);
        }
      }
      if (G == 2 && (g == 0 ? j > 0 && j - 1 < n1 : j < n0)) {
        if (!__all_sync(0xffffffffu, mbar_wait(&turn[1 - g], (g == 0 ? j - 1 : j) & 1, kTimeoutAccum))) { ok = false; break; }
      }
      // ---- weights. A group's value scale goes into the exponent (at most 2^8 up, and not below 2^-60, where an f16 weight
      // is zero and the sum would lose it), so that the sum takes it out again once per 16 keys.
      auto hand_on = [&](int part) {
        if (part == 1 && lane == 0) mbar_arrive(&turn[g]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * g + part]);
      };
      const float neg_m = -m_run, v_off = kWeightUpLog2 - v_ref;
      if (plain) {
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          float v[32];
          uint32_t w[16];
          tmem_ld32(ts + c, v);
#pragma unroll
          for (int i = 0; i < 32; i += 16) {
            const float f = unit * my_sc[(c + i) / 16], up = fmaxf(my_sc[8 + (c + i) / 16] + v_off, -60.f);
            const float2 f2 = make_float2(f, f), off = make_float2(neg_m + up, neg_m + up);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = i; k < i + 16; k += 2) {
              const float2 x = fma_f32x2(make_float2(v[k], v[k + 1]), f2, off);
              const float2 e = make_float2(exp2f_approx(x.x), exp2f_approx(x.y));
              sum = k == i ? e : add_f32x2(sum, e);
              w[k / 2] = pack_f16(e.x, e.y);
            }
            l_run = fmaf(sum.x + sum.y, exp2f_approx(-up), l_run);
          }
          tmem_st16u(tp + c / 2, w);
          hand_on(c / 32);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          float v[32];
          uint32_t w[16];
          tmem_ld32(ts + c, v);
#pragma unroll
          for (int i = 0; i < 32; i += 16) {
            const float ks = my_sc[(c + i) / 16], up = fmaxf(my_sc[8 + (c + i) / 16] + v_off, -60.f);
            const float f = unit * ks;
            float sum = 0.f;
#pragma unroll
            for (int k = i; k < i + 16; k += 2) {
              const float e0 = ks >= 0.f && c + k < lim_tile ? exp2f_approx(fmaf(v[k], f, neg_m + up)) : 0.f;
              const float e1 = ks >= 0.f && c + k + 1 < lim_tile ? exp2f_approx(fmaf(v[k + 1], f, neg_m + up)) : 0.f;
              sum += e0 + e1;
              w[k / 2] = pack_f16(e0, e1);
            }
            l_run = fmaf(sum, exp2f_approx(-up), l_run);
          }
          tmem_st16u(tp + c / 2, w);
          hand_on(c / 32);
        }
      }
    }
    if (ok && n_g > 0 && !__all_sync(0xffffffffu, mbar_wait(&o_full[g], (n_g - 1) & 1, kTimeoutAccum))) ok = false;
    if (ok) {
      *s_mine = l_run;
      ok = meet(n_g);
    }
    if (!ok) {
      *abort_flag = 1;
    } else {
      tc_fence_after();
      l_run += *s_other;
      const bool part = args.splits > 1;
      const float up = exp2f_approx(v_ref - kWeightUpLog2);
      const float inv = part ? up : (m_run == kNone ? 0.f : up / l_run);  // a row that sees no key is zero
      const int64_t slot = ((static_cast<int64_t>(s_item[2]) - 1 - blockIdx.x / p.Hkv) * p.Hkv + h) * args.splits + blockIdx.y;
      bf16* out = p.out + static_cast<int64_t>(tok) * p.o_token + head * p.o_head + half * (D / 2);
      float* part_o = p.part_o + (slot * kRows + r) * D + half * (D / 2);
#pragma unroll
      for (int c = 0; c < D / 2; c += 32) {
        float o[32];
        if (n_g > 0) {
          tmem_ld32(to + c, o);  // by whole warps
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        }
        if (real) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            o[i] *= inv;
            if (s_poison[half * (D / 2) + c + i] < lim) o[i] = __int_as_float(0x7fffffff);
          }
          if (part) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(part_o + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(out + c + i) = make_uint4(pack_bf16(o[i], o[i + 1]), pack_bf16(o[i + 2], o[i + 3]),
                                                                  pack_bf16(o[i + 4], o[i + 5]), pack_bf16(o[i + 6], o[i + 7]));
          }
        }
      }
      if (part && real && half == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * kRows + r) * 2) = make_float2(m_run, l_run);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer) tmem_dealloc(tmem, L::kTmemCols);
  griddep_launch();
}

// One warp per (token, query head): adds the splits' results in their order.
template <int D>
__global__ void __launch_bounds__(128) cached_attn_tc_join_kernel(CachedAttn p, int tiles_max, int splits) {
  constexpr int kRows = Layout<D>::kRows;
  const int lane = threadIdx.x % 32;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 32;
  griddep_wait();
  griddep_launch();
  if (i >= static_cast<int64_t>(p.T) * p.Hkv * p.group) return;
  const int tok = static_cast<int>(i / (p.Hkv * p.group)), hq = static_cast<int>(i % (p.Hkv * p.group));
  const int lo = request_of(p, tok);
  const NewRows fresh = p.B > 0 ? new_rows(p, lo) : NewRows{0, 0};
  if (tok < fresh.first || tok >= fresh.first + fresh.n) return;  // zeroed by the attention kernel
  const int r = (tok - fresh.first) * p.group + hq % p.group;
  const int64_t tile = p.prefix[lo] + r / kRows;
  if (tile < 0 || tile >= tiles_max) return;  // overlapping requests: left out (see the other kernel)
  const int64_t slot0 = (tile * p.Hkv + hq / p.group) * splits;
  float m = kNone;
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, p.part_ml[((slot0 + s) * kRows + r % kRows) * 2]);
  m = warp_max(m);
  constexpr int PER = D / 32;
  float acc[PER], l = 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const int64_t at = (slot0 + s) * kRows + r % kRows;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
    const float f = exp2f_approx(ml.x - m);
    l += ml.y * f;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] += p.part_o[at * D + lane * PER + e] * f;
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  bf16* dst = p.out + static_cast<int64_t>(tok) * p.o_token + hq * p.o_head + lane * PER;
#pragma unroll
  for (int e = 0; e < PER; ++e) dst[e] = __float2bfloat16(acc[e] * inv);
}

template <int FMT, int D>
void launch(const CachedAttn& p, int tiles_max, int splits, cudaStream_t stream) {
  auto kernel = cached_attn_tc_kernel<FMT, D>;
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, current_device(), [&] {
    check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kTotal),
               "cached_attention tc smem");
  });
  launch_pdl(kernel, dim3(static_cast<unsigned>(tiles_max) * p.Hkv, splits), dim3(Layout<D>::kThreads), Layout<D>::kTotal, stream,
             "cached_attention tc", TcArgs{p, splits});
  if (splits > 1) {
    const int64_t rows = static_cast<int64_t>(p.T) * p.Hkv * p.group;
    launch_pdl(cached_attn_tc_join_kernel<D>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, stream,
               "cached_attention tc join", p, tiles_max, splits);
  }
}

}  // namespace

void cached_attention_prompt(const CachedAttn& p, int D, int fmt, int tiles_max, int splits, cudaStream_t stream) {
  if (fmt == kKvFp8) {
    if (D == 64) launch<kKvFp8, 64>(p, tiles_max, splits, stream);
    else launch<kKvFp8, 128>(p, tiles_max, splits, stream);
  } else {
    if (D == 64) launch<kKvInt8, 64>(p, tiles_max, splits, stream);
    else launch<kKvInt8, 128>(p, tiles_max, splits, stream);
  }
}

int cached_attention_tc_status(bool clear) { return read_status_word(clear); }

}  // namespace qw
