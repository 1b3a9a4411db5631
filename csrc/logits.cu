// Logits before sampling: penalties for repeated tokens, biases, grammar masks.
//
//   x = logit;  x > 0 ? x / repetition : x * repetition   for every id of the row's history (prompt and generated)
//   x -= frequency * count;  x -= presence                for the ids generated `count` > 0 times
//   x += bias;  -inf where the mask's bit is 0
//
// A block of threads owns a range of one row's ids. It scans the row's history (a few thousand ids, from L2), counts those
// of its range in shared memory, and turns the counts, with the bias row, into one number to add and one bit (penalised or
// not) per id. Then it reads and writes each logit once, 16 bytes at a time. That needs no count tables in memory, no sort
// and no second launch. Counts are integers, so the order of the atomics does not matter. The bias goes through shared
// memory because a thread's eight ids are not on a 16-byte boundary of its row: read next to the logits, eight numbers apart
// from lane to lane, it kept L1 busy for 79% of the time. Bound by HBM for many rows, by latency for one.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "launch.cuh"
#include "launchers.h"

namespace qw {
namespace {

constexpr int kThreads = 256;
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
  extern __shared__ __align__(16) uint32_t counts[];  // [range + 2 VE], then the bits
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
  uint32_t* const seen_bits = counts + range + 2 * VE;

  int bias_row = -1, mask_row = -1;
  if (a.bias) bias_row = a.bias_rows ? a.bias_rows[row] : row;
  if (a.mask) mask_row = a.mask_rows ? a.mask_rows[row] : row;
  const float* bias = bias_row >= 0 && bias_row < a.biases ? a.bias + bias_row * a.bias_stride : nullptr;
  const uint32_t* mask = mask_row >= 0 && mask_row < a.masks ? a.mask + mask_row * a.mask_stride : nullptr;
  const bool penalised = a.history != nullptr, adds = penalised || bias;
  float rep = 1.f;
  if (adds) {
    float freq = 0.f, pres = 0.f;
    if (penalised) {
      rep = a.repetition ? a.repetition[row] : 1.f;
      freq = a.frequency ? a.frequency[row] : 0.f;
      pres = a.presence ? a.presence[row] : 0.f;
      for (int i = threadIdx.x * 4; i < hi - first; i += kThreads * 4) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
      __syncthreads();
      const int n = min(max(a.history_lens[row], 0), a.history_width);
      const int prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
      const int* ids = a.history + row * a.history_stride;
#pragma unroll 4
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const int id = ids[i];
        if (id >= lo && id < hi) {
          if (i < prompt) atomicOr(&counts[id - first], kPrompt);
          else atomicAdd(&counts[id - first], 1u);
        }
      }
      __syncthreads();
    }
#pragma unroll 4
    for (int i = threadIdx.x; i < (hi - first + 31) / 32 * 32; i += kThreads) {
      const bool there = i >= lo - first && i < hi - first;
      const uint32_t c = penalised && there ? counts[i] : 0;
      float add = bias && there ? bias[first + i] : 0.f;
      const uint32_t made = c & ~kPrompt;
      if (made) add -= static_cast<float>(made) * freq + pres;
      if (there) counts[i] = __float_as_uint(add);
      const uint32_t bits = __ballot_sync(0xffffffffu, c != 0);
      if (threadIdx.x % 32 == 0) seen_bits[i / 32] = bits;
    }
    __syncthreads();
  }

  auto penalty = [&](float x, bool seen) { return seen ? (x > 0.f ? x / rep : x * rep) : x; };
  auto one = [&](float x, int id) {
    const int i = id - first;
    if (adds) x = penalty(x, (seen_bits[i >> 5] >> (i & 31)) & 1u) + __uint_as_float(counts[i]);
    return !mask || ((mask[id >> 5] >> (id & 31)) & 1u) ? x : -INFINITY;
  };
  const int pieces = (hi - body) / VE;
  for (int i = lo + threadIdx.x; i < body; i += kThreads) dst[i] = Num<T>::put(one(Num<T>::get(src[i]), i));
#pragma unroll 4
  for (int p = threadIdx.x; p < pieces; p += kThreads) {
    const int id = body + p * VE;
    uint4 w = *reinterpret_cast<const uint4*>(src + id);
    T* v = reinterpret_cast<T*>(&w);
    uint32_t allowed = 0xffffffffu;
    if (mask) {
      const int at = id >> 5, sh = id & 31;
      const uint32_t next = sh + VE > 32 ? mask[at + 1] : 0u;  // the piece's last id is below vocab: the word exists
      allowed = __funnelshift_r(mask[at], next, sh);
    }
    float x[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = Num<T>::get(v[e]);
    if (adds) {
      const int i = id - first;
      const uint32_t seen = seen_bits[i >> 5] >> (i & 31);  // VE divides 32 and i
      if (seen & ((1u << VE) - 1)) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[e] = penalty(x[e], (seen >> e) & 1u);
      }
#pragma unroll
      for (int e = 0; e < VE; e += 4) {
        const float4 add = *reinterpret_cast<const float4*>(counts + i + e);
        x[e] += add.x; x[e + 1] += add.y; x[e + 2] += add.z; x[e + 3] += add.w;
      }
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = Num<T>::put((allowed >> e) & 1u ? x[e] : -INFINITY);
    *reinterpret_cast<uint4*>(dst + id) = w;
  }
  for (int i = body + pieces * VE + threadIdx.x; i < hi; i += kThreads) dst[i] = Num<T>::put(one(Num<T>::get(src[i]), i));
}

template <typename T>
void launch(const LogitsArgs& a, cudaStream_t stream) {
  // one row: short ranges, so that all SMs share it; many rows: 8192 ids (32 KB of counts, six blocks on an SM), so that
  // the history is scanned few times
  int range = 8192;
  while (range > 1024 && static_cast<int64_t>(a.rows) * ((a.vocab + range - 1) / range) < 296) range /= 2;
  constexpr int VE = 16 / static_cast<int>(sizeof(T));
  const dim3 grid((a.vocab + range - 1) / range + 1, a.rows);  // the ids before the first boundary can shift the last range
  const size_t smem = a.history || a.bias ? (range + 2 * VE + range / 32 + 2) * sizeof(uint32_t) : 0;
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
