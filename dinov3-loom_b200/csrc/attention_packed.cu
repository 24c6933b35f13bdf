// attention_packed.cu - attention over packed sequences of different lengths, grouped heads, full
// or causal.
//
// For query row i of a sequence with a queries and b keys, and query head h reading key-value head
// h / (q_heads / kv_heads): o = sum_j w_j v_j / sum_j w_j, w_j = exp(scale (q . k_j - max)), over
// the keys j < b, and j <= i + b - a where causal (the last query sees the last key). A row that
// sees no key gives 0 (and -inf as its log-sum).
//
// One warp per (row, query head): the running maximum and sum of the softmax, in f32, one pass
// over the keys.
#include "sequence.cuh"

namespace dv3 {

namespace {
constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
}  // namespace

template <bool kBf16, int kDim>
__global__ void __launch_bounds__(kWarps * 32) attention_packed_kernel(const PackedAttention p) {
  constexpr int kWords = kDim / 64;  // 32-bit words of a row per lane
  const uint32_t lane = threadIdx.x % 32;
  const uint64_t work = static_cast<uint64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  const uint32_t t = static_cast<uint32_t>(work / p.q_heads), h = static_cast<uint32_t>(work % p.q_heads);
  if (t >= p.total_q) return;
  const int s = warp_find_sequence(p.cu_q, p.n_seq, t);
  if (s < 0) return;
  uint32_t q0, q1, k0, k1;
  sequence_rows(p.cu_q, s, p.total_q, &q0, &q1);
  sequence_rows(p.cu_k, s, p.total_k, &k0, &k1);
  if (t < q0 || t >= q1) return;
  int64_t visible = k1 - k0;
  if (p.causal) visible = min(visible, visible - (q1 - q0) + (t - q0) + 1);
  const uint32_t g = h / (p.q_heads / p.kv_heads);
  float q[2 * kWords], o[2 * kWords] = {};
  const uint32_t *qr = reinterpret_cast<const uint32_t *>(p.q + t * p.q_token + h * p.q_head) + lane * kWords;
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const float2 x = Elem<kBf16>::unpack(qr[i]);
    q[2 * i] = x.x * p.scale * kLog2e;
    q[2 * i + 1] = x.y * p.scale * kLog2e;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < visible; ++j) {
    const uint32_t *kr = reinterpret_cast<const uint32_t *>(p.k + (k0 + j) * p.k_token + g * p.k_head) + lane * kWords;
    const uint32_t *vr = reinterpret_cast<const uint32_t *>(p.v + (k0 + j) * p.v_token + g * p.v_head) + lane * kWords;
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const float2 x = Elem<kBf16>::unpack(kr[i]);
      d = fmaf(q[2 * i], x.x, fmaf(q[2 * i + 1], x.y, d));
    }
#pragma unroll
    for (int i = 16; i > 0; i /= 2) d += __shfl_xor_sync(0xffffffffu, d, i);
    const float top = fmaxf(m, d), base = top == -INFINITY ? 0.f : top;
    const float keep = exp2f(m - base), w = exp2f(d - base);
    l = fmaf(l, keep, w);
    m = top;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const float2 x = Elem<kBf16>::unpack(vr[i]);
      o[2 * i] = fmaf(o[2 * i], keep, w * x.x);
      o[2 * i + 1] = fmaf(o[2 * i + 1], keep, w * x.y);
    }
  }
  const float inv = visible > 0 ? 1.f / l : 0.f;
  uint32_t *out = reinterpret_cast<uint32_t *>(p.out + t * p.out_token + h * p.out_head) + lane * kWords;
#pragma unroll
  for (int i = 0; i < kWords; ++i) out[i] = Elem<kBf16>::pack(o[2 * i] * inv, o[2 * i + 1] * inv);
  if (p.lse && lane == 0)
    p.lse[static_cast<int64_t>(t) * p.q_heads + h] = visible > 0 ? (m + log2f(l)) * kLn2 : -INFINITY;
}

cudaError_t launch_attention_packed(const PackedAttention &p, bool bf16, cudaStream_t stream) {
  const uint64_t work = static_cast<uint64_t>(p.total_q) * p.q_heads;
  if (work == 0 || p.n_seq == 0) return cudaSuccess;
  const uint64_t grid = (work + kWarps - 1) / kWarps;
  if (grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  const dim3 g(static_cast<uint32_t>(grid)), b(kWarps * 32);
  if (p.head_dim == 64) {
    if (bf16)
      attention_packed_kernel<true, 64><<<g, b, 0, stream>>>(p);
    else
      attention_packed_kernel<false, 64><<<g, b, 0, stream>>>(p);
  } else {
    if (bf16)
      attention_packed_kernel<true, 128><<<g, b, 0, stream>>>(p);
    else
      attention_packed_kernel<false, 128><<<g, b, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace dv3
