// Logits before sampling: penalties for repeated tokens, biases, grammar masks.
//
//   x = logit;  x > 0 ? x / repetition : x * repetition   for every id of the row's history (prompt and generated)
//   x -= frequency * count;  x -= presence                for the ids generated `count` > 0 times
//   x += bias;  -inf where the mask's bit is 0
//
// A block of threads owns a range of one row's ids and keeps their counts in shared memory: it scans the row's history
// (a few thousand ids, from L2) and counts those of its range, then reads and writes each logit once, 16 bytes at a
// time (at most four pieces per thread, fetched before the history). That needs no count tables in memory, no sort and no
// second launch. Counts are integers, so the order of the atomics does not matter. A thread's ids are on a 16-byte boundary
// of the logits, not of the bias row: it reads the two or three aligned pieces that hold their biases and shifts (one by one,
// eight numbers apart from lane to lane, the biases kept L1 busy for 79% of the time). Bound by HBM for many rows, by latency
// for one.
//
// Measured on a B200: 256 rows of 50257 bf16 logits with histories of up to 4096 ids, biases and masks for some rows: 23.4 us,
// 2.4 TB/s, 37% of the measured copy rate: the parts of a block follow one another (clear the counts, count, then the
// logits), and each block scans its row's history anew. One row of 32000 fp32 logits: 6 us a call, of which 3.1 on the
// device.
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "launchers.h"

namespace qw {
namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 4;  // 16-byte pieces of a thread
constexpr uint32_t kPrompt = 0x80000000u;  // in the prompt; the other bits count generated occurrences

template <typename T>
struct Num;
template <>
struct Num<float> {
  __device__ static __forceinline__ float get(float v) { return v; }
  __device__ static __forceinline__ float put(float v) { return v; }
};
template <>
struct Num<bf16> {
  __device__ static __forceinline__ float get(bf16 v) { return __bfloat162float(v); }
  __device__ static __forceinline__ bf16 put(float v) { return __float2bfloat16(v); }
};
template <>
struct Num<__half> {
  __device__ static __forceinline__ float get(__half v) { return __half2float(v); }
  __device__ static __forceinline__ __half put(float v) { return __float2half(v); }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) logits_kernel(LogitsArgs a, int range) {
  constexpr int VE = 16 / static_cast<int>(sizeof(T));
  extern __shared__ __align__(16) uint32_t counts[];  // [range + 2 VE]
  griddep_wait();
  griddep_launch();
  const int row = blockIdx.y;
  const T* src = static_cast<const T*>(a.logits) + row * a.ld;
  T* dst = static_cast<T*>(a.out) + row * a.ldo;
  // ids before the row's first 16-byte boundary go to the first range; where the output's boundaries are elsewhere, all
  // ids go one by one
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
  const bool wide = off == static_cast<int>((reinterpret_cast<uintptr_t>(dst) & 15) / sizeof(T));
  const int lead = off ? VE - off : 0;
  const int lo = blockIdx.x ? min(a.vocab, lead + static_cast<int>(blockIdx.x) * range) : 0;
  const int hi = min(a.vocab, lead + static_cast<int>(blockIdx.x + 1) * range);
  if (lo >= hi) return;
  const int body = wide ? min(hi, blockIdx.x ? lo : lead) : hi;  // first id of the 16-byte pieces
  // id `first` is entry 0: the pieces' entries begin on 16-byte boundaries
  const int first = lo - (VE - (body - lo) % VE) % VE;

  // Everything that depends on nothing else is read first: a block of threads lives for a few memory latencies.
  const bool penalised = a.history != nullptr;
  int bias_row = -1, mask_row = -1, used = 0, prompt = 0;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (a.bias) bias_row = a.bias_rows ? a.bias_rows[row] : row;
  if (a.mask) mask_row = a.mask_rows ? a.mask_rows[row] : row;
  const int pieces = (hi - body) / VE;  // at most kThreads * kPieces
  uint4 w[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int p = threadIdx.x + k * kThreads;
    if (p < pieces) w[k] = *reinterpret_cast<const uint4*>(src + body + p * VE);
  }
  const int* ids = a.history + (penalised ? row * a.history_stride : 0);
  // by fours where the row begins on a 16-byte boundary; the first four of a thread before it knows how many there are
  const int fours = penalised && (reinterpret_cast<uintptr_t>(ids) & 15) == 0 ? a.history_width / 4 : 0;
  int4 early = make_int4(-1, -1, -1, -1);
  if (penalised) {
    used = min(max(a.history_lens[row], 0), a.history_width);
    prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
    rep = a.repetition ? a.repetition[row] : 1.f;
    freq = a.frequency ? a.frequency[row] : 0.f;
    pres = a.presence ? a.presence[row] : 0.f;
    if (static_cast<int>(threadIdx.x) < fours) early = __ldg(reinterpret_cast<const int4*>(ids) + threadIdx.x);
    for (int i = threadIdx.x * 4; i < hi - first; i += kThreads * 4) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
  }
  const float* bias = bias_row >= 0 && bias_row < a.biases ? a.bias + bias_row * a.bias_stride : nullptr;
  const uint32_t* mask = mask_row >= 0 && mask_row < a.masks ? a.mask + mask_row * a.mask_stride : nullptr;
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int id = body + (threadIdx.x + k * kThreads) * VE;
    if (id < hi && bias) asm volatile("prefetch.global.L1 [%0];" ::"l"(bias + id));
    if (id < hi && mask) asm volatile("prefetch.global.L1 [%0];" ::"l"(mask + (id >> 5)));
  }
  if (penalised) {
    __syncthreads();
    const uint32_t span = hi - lo;
    auto count = [&](int i, int id) {
      if (static_cast<uint32_t>(id - lo) < span && i < used) {
        if (i < prompt) atomicOr(&counts[id - first], kPrompt);
        else atomicAdd(&counts[id - first], 1u);
      }
    };
    auto count4 = [&](int i, const int4& x) {
      count(i, x.x);
      count(i + 1, x.y);
      count(i + 2, x.z);
      count(i + 3, x.w);
    };
    count4(threadIdx.x * 4, early);
    const int full = min(fours, (used + 3) / 4);
#pragma unroll 2
    for (int i = threadIdx.x + kThreads; i < full; i += kThreads) count4(4 * i, __ldg(reinterpret_cast<const int4*>(ids) + i));
    for (int i = 4 * fours + threadIdx.x; i < used; i += kThreads) count(i, ids[i]);
    __syncthreads();
  }

  // A division, although most warps have a penalised id among their numbers: a product with the reciprocal would round once
  // more.
  auto penalty = [&](float x, uint32_t c) {
    if (!c) return x;
    x = x > 0.f ? x / rep : x * rep;
    const uint32_t made = c & ~kPrompt;
    return made ? x - static_cast<float>(made) * freq - pres : x;
  };
  auto one = [&](float x, int id) {
    if (penalised) x = penalty(x, counts[id - first]);
    if (bias) x += bias[id];
    return !mask || ((mask[id >> 5] >> (id & 31)) & 1u) ? x : -INFINITY;
  };
  for (int i = lo + threadIdx.x; i < body; i += kThreads) dst[i] = Num<T>::put(one(Num<T>::get(src[i]), i));
  // numbers from an aligned piece of the bias row's memory to the bias of a thread's first id
  const int shift = bias ? static_cast<int>((reinterpret_cast<uintptr_t>(bias + body) & 15) / 4) : 0;
  auto biased = [&](auto by, float* x, const float* b) {
    constexpr int S = decltype(by)::value;
    float f[VE + 4];
#pragma unroll
    for (int i = 0; i < VE + (S ? 4 : 0); i += 4) {  // each holds at least one of the VE biases
      const float4 y = __ldg(reinterpret_cast<const float4*>(b - S + i));
      f[i] = y.x; f[i + 1] = y.y; f[i + 2] = y.z; f[i + 3] = y.w;
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] += f[e + S];
  };
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int p = threadIdx.x + k * kThreads;
    if (p >= pieces) break;
    const int id = body + p * VE;
    T* v = reinterpret_cast<T*>(&w[k]);
    uint32_t allowed = 0xffffffffu;
    if (mask) {
      const int at = id >> 5, sh = id & 31;
      const uint32_t next = sh + VE > 32 ? mask[at + 1] : 0u;  // the piece's last id is below vocab: the word exists
      allowed = __funnelshift_r(mask[at], next, sh);
    }
    float x[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = Num<T>::get(v[e]);
    if (penalised) {
      uint32_t c[VE], any = 0;
#pragma unroll
      for (int e = 0; e < VE; e += 4) {
        const uint4 y = *reinterpret_cast<const uint4*>(counts + id - first + e);
        c[e] = y.x; c[e + 1] = y.y; c[e + 2] = y.z; c[e + 3] = y.w;
        any |= y.x | y.y | y.z | y.w;
      }
      if (any) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[e] = penalty(x[e], c[e]);
      }
    }
    if (bias) {
      if (shift == 0) biased(std::integral_constant<int, 0>{}, x, bias + id);
      else if (shift == 1) biased(std::integral_constant<int, 1>{}, x, bias + id);
      else if (shift == 2) biased(std::integral_constant<int, 2>{}, x, bias + id);
      else biased(std::integral_constant<int, 3>{}, x, bias + id);
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = Num<T>::put((allowed >> e) & 1u ? x[e] : -INFINITY);
    *reinterpret_cast<uint4*>(dst + id) = w[k];
  }
  for (int i = body + pieces * VE + threadIdx.x; i < hi; i += kThreads) dst[i] = Num<T>::put(one(Num<T>::get(src[i]), i));
}

template <typename T>
void launch(const LogitsArgs& a, cudaStream_t stream) {
  // Equal ranges of at most four pieces per thread: each range scans the row's history anew (256 rows of 32000 fp32 logits:
  // 13.9 us, 17.1 with two; 256 of 50257 bf16: 23.4 and 22.1). Of two or one where that leaves fewer than two blocks for an SM
  // (16 rows of 50257 bf16: 6.0 us, 8.4 with four; one row 5.2 and 9.2).
  constexpr int VE = 16 / static_cast<int>(sizeof(T));
  int most = kThreads * kPieces * VE;
  while (most > kThreads * VE && static_cast<int64_t>(a.rows) * ((a.vocab + most - 1) / most) < 148 * 2) most /= 2;
  const int ranges = (a.vocab + most - 1) / most;
  const int range = ((a.vocab + ranges - 1) / ranges + 32 * VE - 1) / (32 * VE) * (32 * VE);
  const dim3 grid(ranges, a.rows);  // the ids before the first boundary come on top of the first range
  const size_t smem = a.history ? (range + 2 * VE + 4) * sizeof(uint32_t) : 0;
  launch_pdl(logits_kernel<T>, grid, dim3(kThreads), smem, stream, "process_logits", a, range);
}

}  // namespace

void process_logits(const LogitsArgs& a, cudaStream_t stream) {
  if (a.rows == 0 || a.vocab == 0) return;
  if (a.dtype == 0) launch<float>(a, stream);
  else if (a.dtype == 1) launch<bf16>(a, stream);
  else launch<__half>(a, stream);
}

}  // namespace qw
