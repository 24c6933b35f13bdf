// sequence.cuh - what the packed and paged operators share: the two 16-bit element types, the
// clamped bounds of a packed sequence, the search for a row's sequence and the page lookup.
#pragma once

#include <cuda_bf16.h>

#include "kernels.h"
#include "sm100.cuh"

namespace dv3 {

// Two 16-bit elements in one word <-> two floats; pack rounds to nearest even, once.
template <bool kBf16>
struct Elem;
template <>
struct Elem<false> {
  __device__ static __forceinline__ float2 unpack(uint32_t v) { return unpack_half2(v); }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
};
template <>
struct Elem<true> {
  __device__ static __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
  }
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The softmax's weights are rounded to the element type, as which the tensor cores take them; their sum is
// of the unrounded ones. bf16 has f32's range. In f16 a weight 17 e-folds below the largest would
// be lost if that were 1 (one strong key before 2^17 weak ones: results 16 to 20 % off), so weights and
// sum carry a factor 2^shift that leaves the largest 2^15: f16 ends at 65504, `slack` is how far (log2) a
// weight may pass its reference, and the factor drops out of their quotient.
template <bool kBf16>
__host__ __device__ constexpr int weight_shift(int slack) {
  return kBf16 ? 0 : 15 - slack;
}
// log of the unshifted sum: reference (log2 units) and sum of such weights.
template <bool kBf16>
__device__ __forceinline__ float log_sum(float reference, float sum, int slack) {
  return (reference + log2f(sum * (1.f / (1 << weight_shift<kBf16>(slack))))) * kLn2;
}

// Rows [begin, end) of packed sequence s, clamped to the tensor's rows whatever cu holds (NULL:
// one row per sequence).
__device__ __forceinline__ void sequence_rows(const int32_t *cu, uint32_t s, uint32_t total,
                                              uint32_t *begin, uint32_t *end) {
  if (!cu) {
    *begin = min(s, total);
    *end = min(s + 1, total);
    return;
  }
  const int64_t b = min(max(static_cast<int64_t>(cu[s]), int64_t{0}), static_cast<int64_t>(total));
  const int64_t e = min(max(static_cast<int64_t>(cu[s + 1]), b), static_cast<int64_t>(total));
  *begin = static_cast<uint32_t>(b);
  *end = static_cast<uint32_t>(e);
}

// The last sequence s < n whose first row cu[s] is at or before row t, found by the whole warp 32
// probes at a time (two rounds up to 1024 sequences); -1 if none. Every lane passes the same t.
__device__ __forceinline__ int warp_find_sequence(const int32_t *cu, uint32_t n, uint32_t t) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t lo = 0, count = n;
  while (true) {
    const uint32_t step = (count + 31) / 32;
    const bool in = lane * step < count;
    const bool le = in && static_cast<int64_t>(cu[lo + lane * step]) <= static_cast<int64_t>(t);
    const uint32_t b = __ballot_sync(0xffffffffu, le);
    if (b == 0) return -1;
    const uint32_t last = 31u - __clz(b);
    lo += last * step;
    count = min(step, count - last * step);
    if (step <= 1) return static_cast<int>(lo);
  }
}

// The page that holds position pos < 2^31.
__device__ __forceinline__ uint32_t page_of(PageDiv d, uint32_t pos) {
  return static_cast<uint32_t>(static_cast<uint64_t>(pos) * d.magic >> d.shift);
}

}  // namespace dv3
