// Attention over the block-wise 8-bit KV cache (kv_format.cuh) for few query rows per request: single tokens, drafted
// tokens, short pieces, and every shape that the tcgen05 kernel (cached_attention_tc.cu) does not take.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp2(s_ij - m_i),   s_ij = (q_i . k_j) * scale * log2(e)
//   over the keys j <= context - new + i of the request's own blocks.
//
// The query heads that share a kv head, and the new tokens, are rows of one tile (16 MT rows), so the cache is read once
// for all of them. Bound by HBM: 2 D bytes per cached token and kv head against 4 D flops per row.
//
// Codes go from global memory into the registers of the tensor-core fragments: the contraction indices of an MMA may be
// permuted as long as both operands agree, so a lane's fragments are consecutive bytes of a row (16 bytes of the key it
// holds the column of, 16 bytes of each of the four values that it holds the contraction rows of). They are widened to
// f16, which holds every code exactly, next to the MMA; the block's scales are applied in 32 bits, the key's to the
// scores and the value's to the probabilities (relative to the largest value scale so far, in steps of two, so that the
// f16 probabilities keep their 11 bits).
//
// The work is the list of all (request, row tile, kv head) items times their 64-key units. It is cut into equal
// consecutive ranges, one per resident block of threads, so ragged lengths cost nothing; a range that ends inside an item
// leaves a partial result (at most two per block), which the join kernel adds up in a fixed order.
#include <algorithm>

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
constexpr float kLazy = 6.f;        // the running maximum moves when a row grows by more than 2^6
constexpr float kWeightUp = 256.f;  // probabilities (<= 2^6) times value scale over the largest: at most 2^14 in f16

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// N bytes per lane as 32-bit words
template <int N>
struct Bytes {
  uint32_t w[N / 4];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (N == 16) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else if constexpr (N == 8) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = x.x; w[1] = x.y;
    } else {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = 0;
  }
};

// The items of a request: row tiles x kv heads, each `units` long.
struct Shape {
  int units, tiles;
};
__device__ __forceinline__ Shape shape_of(const CachedAttn& p, int b, int rows_per_tile) {
  const int n = new_rows(p, b).n;
  const int ctx = min(p.context[b], p.max_table_tokens);
  Shape s;
  s.tiles = n > 0 ? (n * p.group + rows_per_tile - 1) / rows_per_tile : 0;
  s.units = ctx > 0 ? (ctx + kUnit - 1) / kUnit : 0;
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

// One 16-key step of a warp, as loaded: codes, scales, and whether the keys have a block at all.
template <int D>
struct Raw {
  static constexpr int VB = D / 4 < 16 ? D / 4 : 16;  // bytes of a key that a lane loads at a time
  static constexpr int CH = D / 4 / VB;
  Bytes<VB> k[2][CH];    // key n of the two 8-key halves: dims c * 4 VB + t * VB ...
  Bytes<D / 8> v[4];     // values 2t, 2t + 1, 2t + 8, 2t + 9: dims g * D / 8 ...
  float ks, vs;
};

template <int FMT, int D, int MT>
__global__ void __launch_bounds__(kThreads, MT == 1 ? 2 : 1) cached_attn_kernel(CachedAttn p) {
  constexpr int R = 16 * MT;      // rows of a tile
  constexpr int VB = Raw<D>::VB;
  constexpr int CH = Raw<D>::CH;
  constexpr int NT = D / 8;       // 8-wide output tiles
  extern __shared__ float attn_smem[];
  float* s_o = attn_smem;                     // [kWarps][R][D]
  __shared__ float s_mlv[kWarps][R][3];      // maximum, sum, largest value scale
  __shared__ int s_poison[D];                 // the first key whose value is NaN in this dim, among masked steps
  __shared__ int64_t s_find[3];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, t = lane % 4;
  griddep_wait();

  // ---- the range of this block of threads, and the request that it begins in
  if (warp == 0) {
    int64_t total = 0;
    for (int b = lane; b < p.B; b += 32) total += work_of(p, b, R);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const int64_t workers = min(static_cast<int64_t>(gridDim.x), total);
    const int64_t begin = blockIdx.x < workers ? blockIdx.x * total / workers : total;
    int64_t before = 0;
    const bool publish = blockIdx.x == 0;  // the join kernel reads the prefix sums
    if (lane == 0) s_find[0] = total;
    for (int b0 = 0; b0 < p.B && (publish || before <= begin); b0 += 32) {
      const int b = b0 + lane;
      const int64_t w = b < p.B ? work_of(p, b, R) : 0;
      int64_t x = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const int64_t at = before + x - w;
      if (w > 0 && begin >= at && begin < at + w) {
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
  const int64_t begin = blockIdx.x * total / workers, end = (blockIdx.x + 1) * total / workers;
  int b = static_cast<int>(s_find[1]);
  int64_t at = s_find[2];
  Shape shape = shape_of(p, b, R);

  for (int64_t u = begin; u < end;) {
    while (u >= at + static_cast<int64_t>(shape.units) * shape.tiles * p.Hkv) {  // ends: u < end <= total
      at += static_cast<int64_t>(shape.units) * shape.tiles * p.Hkv;
      shape = shape_of(p, ++b, R);
    }
    const int64_t local = u - at;
    const int item = static_cast<int>(local / shape.units), u0 = static_cast<int>(local % shape.units);
    const int n_units = static_cast<int>(min(static_cast<int64_t>(shape.units - u0), end - u));
    u += n_units;
    const int h = item % p.Hkv, tile = item / p.Hkv;
    const NewRows fresh = new_rows(p, b);
    const int q0 = fresh.first, n = fresh.n;
    const int ctx = min(p.context[b], p.max_table_tokens);
    const int row0 = tile * R, rows = min(R, n * p.group - row0);
    // keys that a row sees: [0, lim)
    auto lim_of = [&](int row) { return min(ctx, p.context[b] - n + (row0 + min(row, rows - 1)) / p.group + 1); };
    const int lim_first = lim_of(0), lim_last = lim_of(rows - 1);
    const int* table = p.table + static_cast<int64_t>(b) * p.table_stride;
    const uint8_t* kbase = p.k.codes + h * p.k.head_stride + t * VB;
    const uint8_t* vbase = p.v.codes + h * p.v.head_stride + g * (D / 8);
    const int key_end = min(lim_last, (u0 + n_units) * kUnit);
    const int step0 = u0 * kUnit + warp * 16;

    auto block_of = [&](int j) { return j < key_end ? __ldg(table + j / p.block) : -1; };
    auto load = [&](Raw<D>& r, int j, int id) {
      // a key without a block (none given, or outside the cache) counts as masked: nothing is read for it
      if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.blocks)) {
        r.ks = -1.f;
        return;
      }
      const int in = j % p.block;
      r.ks = __ldg(p.k.scale + static_cast<int64_t>(id) * p.k.scale_stride + h);
      r.vs = __ldg(p.v.scale + static_cast<int64_t>(id) * p.v.scale_stride + h);
      const uint8_t* kp = kbase + static_cast<int64_t>(id) * p.k.block_stride + (in + g) * p.k.token_stride;
      const uint8_t* vp = vbase + static_cast<int64_t>(id) * p.v.block_stride + (in + 2 * t) * p.v.token_stride;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int c = 0; c < CH; ++c) r.k[x][c].load(kp + x * 8 * p.k.token_stride + c * 4 * VB);
#pragma unroll
      for (int x = 0; x < 4; ++x) r.v[x].load(vp + ((x & 1) + (x >> 1) * 8) * p.v.token_stride);
    };
    Raw<D> cur, next;
    int id_next = block_of(step0 + kUnit);
    if (step0 < key_end) load(cur, step0, block_of(step0));

    // ---- query rows as f16 fragments: each row divided by a power of two that brings its largest number to [1, 2)
    uint32_t q[MT][D / 16][4];
    float unit[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = mt * 16 + half * 8 + g;
        float x[D / 4];
        float m = 0.f;
        if (row < rows) {
          const int r = row0 + row;
          const bf16* src = p.q + static_cast<int64_t>(q0 + r / p.group) * p.q_token + (h * p.group + r % p.group) * p.q_head;
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < VB; i += 4) {
              const uint2 w = *reinterpret_cast<const uint2*>(src + c * 4 * VB + t * VB + i);
              const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.x));
              const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.y));
              float* y = x + c * VB + i;
              y[0] = lo.x; y[1] = lo.y; y[2] = hi.x; y[3] = hi.y;
            }
#pragma unroll
          for (int i = 0; i < D / 4; ++i) m = fmaxf(m, fabsf(x[i]));
        } else {
#pragma unroll
          for (int i = 0; i < D / 4; ++i) x[i] = 0.f;
        }
        m = quad_max(m);
        const uint32_t bits = __float_as_uint(m);
        const int e = min(max(static_cast<int>(bits >> 23) - 127, -100), 126);
        const bool fine = m > 0.f && m <= 3.4028234e38f;  // zero or infinite rows as they are
        const float inv = fine ? exp2i(-e) : 1.f;
        unit[mt][half] = (fine ? exp2i(e) : 1.f) * p.scale * kLog2e;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          q[mt][s][half] = pack_f16(x[4 * s] * inv, x[4 * s + 1] * inv);
          q[mt][s][2 + half] = pack_f16(x[4 * s + 2] * inv, x[4 * s + 3] * inv);
        }
      }

    float o[MT][NT][4];
    float m_run[MT][2], l_run[MT][2];
    float v_ref[MT][2], v_up[MT][2];  // the largest value scale that the row has seen, and kWeightUp over it
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][i][e] = 0.f;
      m_run[mt][0] = m_run[mt][1] = -INFINITY;
      l_run[mt][0] = l_run[mt][1] = 0.f;
      v_ref[mt][0] = v_ref[mt][1] = v_up[mt][0] = v_up[mt][1] = 0.f;
    }

    for (int j = step0; j < key_end; j += kUnit) {
      const int id_after = block_of(j + 2 * kUnit);
      if (j + kUnit < key_end) load(next, j + kUnit, id_next);
      if (cur.ks >= 0.f) {
        const bool edge = j + 16 > lim_first;
        if (edge) {  // values past the last row's limit may be anything: they count as zero
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = j + 2 * t + (x & 1) + (x >> 1) * 8;
            if (key >= lim_last) {
              cur.v[x].zero();
            } else if (key >= lim_first) {  // seen by some rows only: a NaN must not reach the others
#pragma unroll
              for (int i = 0; i < D / 32; ++i) {
                const uint32_t bad = Kv<FMT>::nan_bytes(cur.v[x].w[i]);
                if (bad) {
                  for (int e = 0; e < 4; ++e)
                    if ((bad >> (8 * e + 7)) & 1) {
                      atomicMin(&s_poison[g * (D / 8) + 4 * i + e], key);
                      cur.v[x].w[i] &= ~(0xffu << (8 * e));
                    }
                }
              }
            }
          }
        }
        // ---- scores: rows x 16 keys
        float s[MT][2][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[mt][x][e] = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int i = 0; i < VB / 4; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              uint32_t b0, b1;
              Kv<FMT>::decode4(cur.k[x][c].w[i], b0, b1);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) mma_f16(s[mt][x], q[mt][c * (VB / 4) + i], b0, b1);
            }
        // ---- probabilities
        bool moved = false;
        float top[MT][2], v_top[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float f = unit[mt][half] * cur.ks;
            const int lim = edge ? lim_of(mt * 16 + half * 8 + g) - j : 16;
            float mx = -INFINITY;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& y = s[mt][x][half * 2 + e];
                y = x * 8 + 2 * t + e < lim ? y * f : -INFINITY;
                mx = fmaxf(mx, y);
              }
            top[mt][half] = mx;
            v_top[mt][half] = lim > 0 ? cur.vs : 0.f;
            moved = moved || mx > m_run[mt][half] + kLazy || v_top[mt][half] > v_ref[mt][half];
          }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float v_new = fmaxf(v_ref[mt][half], v_top[mt][half]);
              const float vf = v_ref[mt][half] > 0.f ? v_ref[mt][half] / v_new : 0.f;
              const float m_new = fmaxf(m_run[mt][half], quad_max(top[mt][half]));
              const float f = m_run[mt][half] == -INFINITY ? 0.f : exp2f_approx(m_run[mt][half] - m_new);
              m_run[mt][half] = m_new;
              l_run[mt][half] *= f;
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                o[mt][i][half * 2] *= f * vf;
                o[mt][i][half * 2 + 1] *= f * vf;
              }
              v_ref[mt][half] = v_new;
              v_up[mt][half] = v_new > 0.f ? kWeightUp / v_new : 0.f;
            }
        }
        uint32_t w[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float m = m_run[mt][half] == -INFINITY ? 0.f : m_run[mt][half];
            const float up = v_up[mt][half] * cur.vs;
            float pr[2][2];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int e = 0; e < 2; ++e) pr[x][e] = exp2f_approx(s[mt][x][half * 2 + e] - m);
            l_run[mt][half] += (pr[0][0] + pr[0][1]) + (pr[1][0] + pr[1][1]);
            w[mt][half] = pack_f16(pr[0][0] * up, pr[0][1] * up);
            w[mt][2 + half] = pack_f16(pr[1][0] * up, pr[1][1] * up);
          }
        // ---- output: four dims of the lane's values at a time
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t b0[4], b1[4];
          Kv<FMT>::decode4(__byte_perm(cur.v[0].w[i], cur.v[1].w[i], 0x5140), b0[0], b0[1]);
          Kv<FMT>::decode4(__byte_perm(cur.v[0].w[i], cur.v[1].w[i], 0x7362), b0[2], b0[3]);
          Kv<FMT>::decode4(__byte_perm(cur.v[2].w[i], cur.v[3].w[i], 0x5140), b1[0], b1[1]);
          Kv<FMT>::decode4(__byte_perm(cur.v[2].w[i], cur.v[3].w[i], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma_f16(o[mt][4 * i + e], w[mt], b0[e], b1[e]);
        }
      }
      cur = next;
      id_next = id_after;
    }

    // ---- the four warps' results of this piece into one
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = mt * 16 + half * 8 + g;
        const float l = quad_sum(l_run[mt][half]);
        if (t == 0) {
          s_mlv[warp][row][0] = m_run[mt][half];
          s_mlv[warp][row][1] = l;
          s_mlv[warp][row][2] = v_ref[mt][half];
        }
        if (row < rows) {
          float* dst = s_o + (warp * R + row) * D;
#pragma unroll
          for (int i = 0; i < NT; ++i) {  // lane t holds the dims (2t) D/8 + i and (2t + 1) D/8 + i
            dst[2 * t * (D / 8) + i] = o[mt][i][half * 2];
            dst[(2 * t + 1) * (D / 8) + i] = o[mt][i][half * 2 + 1];
          }
        }
      }
    __syncthreads();
    const bool whole = n_units == shape.units;
    const int64_t slot = u0 > 0 ? 2 * static_cast<int64_t>(blockIdx.x) : 2 * static_cast<int64_t>(blockIdx.x) + 1;
    for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
      const int row = i / (D / 4), d = (i % (D / 4)) * 4;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_mlv[w][row][0]);
      float l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = s_mlv[w][row][0];
        const float f = mw == -INFINITY ? 0.f : exp2f_approx(mw - m);
        const float fv = f * s_mlv[w][row][2] * (1.f / kWeightUp);
        l += s_mlv[w][row][1] * f;
        const float4 x = *reinterpret_cast<const float4*>(s_o + (w * R + row) * D + d);
        acc.x += x.x * fv; acc.y += x.y * fv; acc.z += x.z * fv; acc.w += x.w * fv;
      }
      const int lim = lim_of(row);
      if (s_poison[d] < lim) acc.x = __int_as_float(0x7fffffff);
      if (s_poison[d + 1] < lim) acc.y = __int_as_float(0x7fffffff);
      if (s_poison[d + 2] < lim) acc.z = __int_as_float(0x7fffffff);
      if (s_poison[d + 3] < lim) acc.w = __int_as_float(0x7fffffff);
      if (whole) {
        const float inv = m == -INFINITY ? 0.f : 1.f / l;  // a row that sees no key is zero
        const int r = row0 + row;
        bf16* dst = p.out + static_cast<int64_t>(q0 + r / p.group) * p.o_token + (h * p.group + r % p.group) * p.o_head + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
      } else {
        *reinterpret_cast<float4*>(p.part_o + (slot * R + row) * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * R + row) * 2) = make_float2(m, l);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += kThreads) s_poison[i] = 0x7fffffff;
    __syncthreads();
  }
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
  int lo = 0, hi = p.B;  // the last request whose start is <= tok
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.query_start[mid] <= tok) lo = mid;
    else hi = mid;
  }
  const int b = lo;
  float l = 0.f;
  const NewRows fresh = p.B > 0 ? new_rows(p, b) : NewRows{0, 0};
  if (tok >= fresh.first && tok < fresh.first + fresh.n) {
    const int64_t total = p.prefix[p.B];
    const Shape s = shape_of(p, b, R);
    if (s.units > 0) {
      const int row_all = (tok - fresh.first) * p.group + hq % p.group;
      const int h = hq / p.group, tile = row_all / R, row = row_all % R;
      const int64_t u0 = p.prefix[b] + (static_cast<int64_t>(tile) * p.Hkv + h) * s.units;
      const int workers = static_cast<int>(min(static_cast<int64_t>(workers_max), total));
      const int w0 = worker_of(u0, total, workers), w1 = worker_of(u0 + s.units - 1, total, workers);
      if (w0 == w1) return;  // one range had the whole item
      float m = -INFINITY;
      for (int w = w0 + lane; w <= w1; w += 32)
        m = fmaxf(m, p.part_ml[((2 * static_cast<int64_t>(w) + (w == w0)) * R + row) * 2]);
      m = warp_max(m);
      if (m > -INFINITY) {
#pragma unroll 4
        for (int w = w0; w <= w1; ++w) {
          const int64_t at = (2 * static_cast<int64_t>(w) + (w == w0)) * R + row;
          const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
          const float f = ml.x == -INFINITY ? 0.f : exp2f_approx(ml.x - m);
          l += ml.y * f;
          const float* src = p.part_o + at * D + lane * PER;
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] += src[e] * f;
        }
      }
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) dst[e] = __float2bfloat16(acc[e] * inv);
}

// Resident blocks of threads on 148 SMs: two per SM with one row tile (the registers), one with two.
int cached_attn_workers(int mt) { return 148 * (mt == 1 ? 2 : 1); }

template <int FMT, int D, int MT>
void launch(const CachedAttn& p, cudaStream_t stream) {
  auto kernel = cached_attn_kernel<FMT, D, MT>;
  constexpr int smem = kWarps * 16 * MT * D * static_cast<int>(sizeof(float));
  static const bool configured = [&] {
    check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cached_attention smem");
    return true;
  }();
  (void)configured;
  const int workers = cached_attn_workers(MT);
  launch_pdl(kernel, dim3(workers), dim3(kThreads), smem, stream, "cached_attention", p);
  const int64_t rows = static_cast<int64_t>(p.T) * p.Hkv * p.group;
  launch_pdl(cached_attn_join_kernel<D>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, stream,
             "cached_attention join", p, workers, 16 * MT);
}

template <int FMT>
void dispatch(const CachedAttn& p, int D, int mt, cudaStream_t stream) {
  if (mt == 1) {
    if (D == 32) launch<FMT, 32, 1>(p, stream);
    else if (D == 64) launch<FMT, 64, 1>(p, stream);
    else launch<FMT, 128, 1>(p, stream);
  } else {
    if (D == 32) launch<FMT, 32, 2>(p, stream);
    else if (D == 64) launch<FMT, 64, 2>(p, stream);
    else launch<FMT, 128, 2>(p, stream);
  }
}

void cached_attention_rows(const CachedAttn& p, int D, int fmt, int mt, cudaStream_t stream) {
  if (fmt == kKvFp8) dispatch<kKvFp8>(p, D, mt, stream);
  else dispatch<kKvInt8>(p, D, mt, stream);
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Which kernel, and how its work is split.
struct Way {
  bool prompt;
  int mt;                   // few rows: 16-row tiles per block of threads
  int tiles_max, splits;    // prompts
  int64_t part_o, part_ml, bytes;  // of the workspace; the prefix sums are at its beginning
};

Way way_of(int T, int B, int Hq, int Hkv, int D, int max_query, int max_context) {
  Way w{};
  const int group = Hq / Hkv;
  const int64_t rows = static_cast<int64_t>(std::min(max_query, T)) * group;
  w.prompt = D != 32 && rows > 32;
  w.mt = rows <= 16 ? 1 : 2;
  int64_t slots;
  if (w.prompt) {
    w.tiles_max = static_cast<int>(static_cast<int64_t>(T) * group / kPromptRows + B);
    // too few row tiles for the SMs: split the keys, two tiles of 128 at least for each part
    const int64_t blocks = static_cast<int64_t>(w.tiles_max) * Hkv;
    w.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(148 / std::max<int64_t>(blocks, 1), max_context / 256)));
    slots = w.splits > 1 ? blocks * w.splits * kPromptRows : 0;
  } else {
    slots = 2 * static_cast<int64_t>(cached_attn_workers(w.mt)) * 16 * w.mt;
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
  p.k = {static_cast<const uint8_t*>(k.codes), k.block_stride, k.head_stride, k.token_stride, k.scale, k.scale_stride};
  p.v = {static_cast<const uint8_t*>(v.codes), v.block_stride, v.head_stride, v.token_stride, v.scale, v.scale_stride};
  p.table = table;
  p.table_stride = table_stride;
  p.context = context;
  p.query_start = query_start;
  p.T = T;
  p.B = B;
  p.Hkv = Hkv;
  p.group = Hq / Hkv;
  p.block = block;
  p.blocks = blocks;
  p.max_table_tokens = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(width) * block, 0x7fffffff));
  p.scale = scale;
  p.prefix = reinterpret_cast<int64_t*>(base);
  p.part_o = reinterpret_cast<float*>(base + w.part_o);
  p.part_ml = reinterpret_cast<float*>(base + w.part_ml);
  if (w.prompt) cached_attention_prompt(p, D, fmt, w.tiles_max, w.splits, stream);
  else cached_attention_rows(p, D, fmt, w.mt, stream);
}

int cached_attention_status(bool clear) { return read_status_word(clear); }

}  // namespace qw
