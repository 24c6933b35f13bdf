// rope_append.cu - rotates the new queries and keys of packed sequences by their positions and
// appends the keys and values to a paged cache, in one launch.
//
// Row t of sequence s stands at position p = lens[s] - new(s) + (t - first row of s) (lens counts
// the appended rows already). Channels c < rot/2 and c + rot/2 of each head turn together:
// (a, b) -> (a cos[p][c] - b sin[p][c], b cos[p][c] + a sin[p][c]), in f32 from the 16-bit inputs
// and the f32 tables, rounded once. K and V go to slot p % page_size of page
// page_table[s][p / page_size].
//
// Bound by bandwidth: every element is read once and written once, the arithmetic is three
// operations an element. One thread moves one unit of 16 channels as two 16-byte chunks: the two
// halves of 8 rotated pairs, or 32 contiguous bytes where nothing turns; a unit's row and head come from
// products by a precomputed reciprocal (64-bit divisions kept the kernel issue-bound: 66 us for 375 MB,
// 58 without: 6.4 TB/s, 98 % of a plain copy's rate).
#include "sequence.cuh"

namespace dv3 {

namespace {
constexpr int kAppendThreads = 256;

template <bool kBf16>
__device__ __forceinline__ void rotate(uint4 &a, uint4 &b, const float *cs, const float *sn) {
  uint32_t *aw = reinterpret_cast<uint32_t *>(&a), *bw = reinterpret_cast<uint32_t *>(&b);
  float c[8], s[8];
  *reinterpret_cast<float4 *>(c) = __ldg(reinterpret_cast<const float4 *>(cs));
  *reinterpret_cast<float4 *>(c + 4) = __ldg(reinterpret_cast<const float4 *>(cs) + 1);
  *reinterpret_cast<float4 *>(s) = __ldg(reinterpret_cast<const float4 *>(sn));
  *reinterpret_cast<float4 *>(s + 4) = __ldg(reinterpret_cast<const float4 *>(sn) + 1);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = Elem<kBf16>::unpack(aw[i]), y = Elem<kBf16>::unpack(bw[i]);
    aw[i] = Elem<kBf16>::pack(x.x * c[2 * i] - y.x * s[2 * i], x.y * c[2 * i + 1] - y.y * s[2 * i + 1]);
    bw[i] = Elem<kBf16>::pack(y.x * c[2 * i] + x.x * s[2 * i], y.y * c[2 * i + 1] + x.y * s[2 * i + 1]);
  }
}
}  // namespace

template <bool kBf16>
__global__ void __launch_bounds__(kAppendThreads) rope_append_kernel(
    const RopeAppend p, uint32_t row0, uint32_t rows) {
  pdl_wait();  // what the kernel before wrote is there from here on
  pdl_trigger();
  const uint32_t units = p.units.size;
  const uint32_t total_units = rows * units;  // below 2^31
  const uint32_t base = blockIdx.x * kAppendThreads;
  const uint32_t warp_first = base + (threadIdx.x & ~31u);
  if (warp_first >= total_units) return;
  const uint32_t at = min(base + threadIdx.x, total_units - 1);
  const uint32_t of = page_of(p.units, at), t = row0 + of, u = at - of * units;
  const uint32_t shift = p.head_dim == 64 ? 2 : 3, head = u >> shift, w = u & ((1u << shift) - 1);
  const bool is_q = head < p.q_heads;
  const bool is_k = !is_q && head < p.q_heads + p.kv_heads;
  const uint32_t h = is_q ? head : head - p.q_heads - (is_k ? 0 : p.kv_heads);
  // the unit's two chunks: the halves of 8 turned pairs, or 16 channels that stay as they are
  const uint32_t turned = is_q || is_k ? p.rot_dim / 16 : 0;
  const uint32_t ca = w < turned ? 8 * w : 16 * w;
  const uint32_t cb = w < turned ? ca + p.rot_dim / 2 : ca + 8;
  const uint16_t *src = is_q ? p.q + t * p.q_token + h * p.q_head
                        : is_k ? p.k + t * p.k_token + h * p.k_head
                               : p.v + t * p.v_token + h * p.v_head;
  // The data first: where it goes takes a chain of loads (sequence, length, page) that they overlap.
  uint4 a = *reinterpret_cast<const uint4 *>(src + ca), b = *reinterpret_cast<const uint4 *>(src + cb);
  int s = static_cast<int>(t);
  if (p.cu_new) {
    s = warp_find_sequence(p.cu_new, p.n_seq, row0 + page_of(p.units, warp_first));
    // A later row of the warp may belong to a later sequence, mostly the next; empty ones may lie between,
    // however many: steps that double while they land at or before the row, then halve.
    auto before = [&](uint32_t step) {
      const int64_t to = static_cast<int64_t>(s) + step;
      return to < p.n_seq && static_cast<int64_t>(p.cu_new[to]) <= t;
    };
    uint32_t step = 1;
    for (; before(step); step *= 2) s += step;
    while (step /= 2)
      if (before(step)) s += step;
  }
  if (base + threadIdx.x >= total_units || s < 0 || s >= static_cast<int>(p.n_seq)) return;
  uint32_t first, end;
  sequence_rows(p.cu_new, s, p.total, &first, &end);
  if (t < first || t >= end) return;  // before the first or behind the last sequence
  const int64_t pos = static_cast<int64_t>(p.lens[s]) - (end - first) + (t - first);
  if (pos < 0 || (p.rot_dim && pos >= p.positions)) {
    report(p.status, kErrPosition);
    return;
  }
  uint16_t *dst;
  if (is_q) {
    dst = p.q_out + t * p.qo_token + h * p.qo_head;
  } else {
    const uint32_t page = page_of(p.page, static_cast<uint32_t>(pos));
    const int32_t id = page < p.max_pages ? p.page_table[s * p.table_stride + page] : -1;
    if (id < 0 || static_cast<uint32_t>(id) >= p.n_pages) {
      report(p.status, kErrPage);
      return;
    }
    const uint32_t slot = static_cast<uint32_t>(pos) - page * p.page.size;
    dst = (is_k ? p.k_cache + id * p.k_page : p.v_cache + id * p.v_page) +
          (static_cast<int64_t>(h) * p.page.size + slot) * p.head_dim;
  }
  if (w < turned) {
    const int64_t row = pos * (p.rot_dim / 2) + ca;
    rotate<kBf16>(a, b, p.cos + row, p.sin + row);
  }
  *reinterpret_cast<uint4 *>(dst + ca) = a;
  *reinterpret_cast<uint4 *>(dst + cb) = b;
}

cudaError_t launch_rope_append(const RopeAppend &args, bool bf16, cudaStream_t stream) {
  RopeAppend p = args;
  p.units = page_div((p.q_heads + 2 * p.kv_heads) * (p.head_dim / 16));
  // one launch, but for more units than 31 bits count
  const uint32_t most = 0x7fffff00u / p.units.size;
  for (uint32_t row0 = 0; row0 < p.total; row0 += most) {
    const uint32_t rows = p.total - row0 < most ? p.total - row0 : most;
    const dim3 g((rows * p.units.size + kAppendThreads - 1) / kAppendThreads), b(kAppendThreads);
    const cudaError_t e = bf16 ? launch_pdl(rope_append_kernel<true>, g, b, 0, stream, p, row0, rows)
                               : launch_pdl(rope_append_kernel<false>, g, b, 0, stream, p, row0, rows);
    if (e != cudaSuccess || rows < most) return e;
  }
  return cudaSuccess;
}

}  // namespace dv3
