// attention_paged.cu - attention of one new token per sequence over a paged key-value cache.
//
// For sequence s of n = lens[s] cached tokens and query head h reading key-value head
// h / (q_heads / kv_heads): o = sum_j w_j v_j / sum_j w_j, w_j = exp(scale (q . k_j - max)), over
// j < n. Key j lies in slot j % page_size of page page_table[s][j / page_size]. No tokens give 0
// (and -inf as the log-sum). A page id outside the pool, or a length past the table, is reported in
// `status` and its tokens count as absent.
//
// One warp per (sequence, query head): the running maximum and sum of the softmax, in f32, one
// pass over the keys.
#include "sequence.cuh"

namespace dv3 {

namespace {
constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
}  // namespace

template <bool kBf16, int kDim>
__global__ void __launch_bounds__(kWarps * 32) attention_paged_kernel(const PagedAttention p) {
  constexpr int kWords = kDim / 64;
  const uint32_t lane = threadIdx.x % 32;
  const uint64_t work = static_cast<uint64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  const uint32_t s = static_cast<uint32_t>(work / p.q_heads), h = static_cast<uint32_t>(work % p.q_heads);
  if (s >= p.n_seq) return;
  const uint32_t g = h / (p.q_heads / p.kv_heads);
  const int64_t room = static_cast<int64_t>(p.max_pages) * p.page.size;
  int64_t n = max(p.lens[s], 0);
  if (n > room) {
    if (lane == 0) report(p.status, kErrPage);
    n = room;
  }
  float q[2 * kWords], o[2 * kWords] = {};
  const uint32_t *qr = reinterpret_cast<const uint32_t *>(p.q + s * p.q_seq + h * p.q_head) + lane * kWords;
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const float2 x = Elem<kBf16>::unpack(qr[i]);
    q[2 * i] = x.x * p.scale * kLog2e;
    q[2 * i + 1] = x.y * p.scale * kLog2e;
  }
  float m = -INFINITY, l = 0.f;
  bool any = false;
  for (int64_t j = 0; j < n; ++j) {
    const uint32_t page = page_of(p.page, static_cast<uint32_t>(j));
    const int32_t id = p.page_table[s * p.table_stride + page];
    if (id < 0 || static_cast<uint32_t>(id) >= p.n_pages) {
      if (lane == 0) report(p.status, kErrPage);
      continue;
    }
    any = true;
    const int64_t row = (static_cast<int64_t>(g) * p.page.size + (j - static_cast<int64_t>(page) * p.page.size)) * kDim;
    const uint32_t *kr = reinterpret_cast<const uint32_t *>(p.k_cache + id * p.k_page + row) + lane * kWords;
    const uint32_t *vr = reinterpret_cast<const uint32_t *>(p.v_cache + id * p.v_page + row) + lane * kWords;
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
  const float inv = any ? 1.f / l : 0.f;
  uint32_t *out = reinterpret_cast<uint32_t *>(p.out + s * p.out_seq + h * p.out_head) + lane * kWords;
#pragma unroll
  for (int i = 0; i < kWords; ++i) out[i] = Elem<kBf16>::pack(o[2 * i] * inv, o[2 * i + 1] * inv);
  if (p.lse && lane == 0)
    p.lse[static_cast<int64_t>(s) * p.q_heads + h] = any ? (m + log2f(l)) * kLn2 : -INFINITY;
}

size_t attention_paged_workspace(const PagedAttention &) { return 0; }

cudaError_t launch_attention_paged(const PagedAttention &p, bool bf16, cudaStream_t stream) {
  const uint64_t work = static_cast<uint64_t>(p.n_seq) * p.q_heads;
  if (work == 0) return cudaSuccess;
  const uint64_t grid = (work + kWarps - 1) / kWarps;
  if (grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  const dim3 g(static_cast<uint32_t>(grid)), b(kWarps * 32);
  if (p.head_dim == 64) {
    if (bf16)
      attention_paged_kernel<true, 64><<<g, b, 0, stream>>>(p);
    else
      attention_paged_kernel<false, 64><<<g, b, 0, stream>>>(p);
  } else {
    if (bf16)
      attention_paged_kernel<true, 128><<<g, b, 0, stream>>>(p);
    else
      attention_paged_kernel<false, 128><<<g, b, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace dv3
