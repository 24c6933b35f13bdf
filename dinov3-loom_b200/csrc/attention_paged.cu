// attention_paged.cu - attention of one new token per sequence over a paged key-value cache.
//
// For sequence s of n = lens[s] cached tokens and query head h reading key-value head
// h / (q_heads / kv_heads): o = sum_j w_j v_j / sum_j w_j, w_j = exp(scale (q . k_j - max)), over
// j < n. Key j lies in slot j % page_size of page page_table[s][j / page_size]. No tokens give 0
// (and -inf as the log-sum). A page id outside the pool, or a length past the table, is reported in
// `status` and its tokens count as absent.
//
// Bound by the one read of K and V: a key costs 4 head_dim bytes and 4 head_dim flops for each of
// the group's query heads, far below the tensor cores' rate. So the kernel is a stream: a CTA takes
// one (sequence, key-value head, split of the length), and 64-key tiles of K and V run through a
// ring of shared-memory stages by 16-byte cp.async (any page size; a tile's row addresses are looked
// up one tile ahead). Each of the four warps owns 16 keys of a tile and its own running maximum,
// sum and output, so warps meet only at the ring's barrier: S = Q K^T and O += P V are m16n8k16
// tensor-core products with the group's up to 16 query heads as M (rows past the group are zero),
// P stays in registers. Groups of more than 16 heads take one CTA per 16.
//
// A sequence is cut into chunks of whole tiles, dealt round-robin to the grid's splits, so that a
// long sequence fills the GPU and a long one among short ones does not end last. With more than
// one split each CTA leaves (max, sum, unnormalised output) in the workspace, and a second launch
// joins them in split order; nothing depends on the order in which CTAs end.
#include <atomic>

#include "sequence.cuh"

namespace dv3 {

namespace {
constexpr int kThreads = 128;
constexpr int kTile = 64;     // keys per stage, 16 per warp
constexpr int kStages = 3;
constexpr int kRing = 4;      // tiles whose row addresses are kept: kStages + the one being looked up
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int kDim>
constexpr int smem_bytes() {
  return kStages * 2 * kTile * kDim * 2 + kRing * kTile * 2 * 8;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// How the lengths are cut: chunks of `chunk` tiles dealt round-robin to `splits` CTAs.
struct Split {
  uint32_t splits, chunk, head_blocks;
};

// A chunk is 4 tiles (256 keys) to 16, so that the grid has about four waves of CTAs: less than
// four leave a ragged tail, and chunks under 256 keys spend more on their start than on the
// stream. The splits are capped so that the partial results stay small beside the cache, whatever
// bound of the lengths the caller gave: beyond 32 waves the chunks go round.
Split split_of(const PagedAttention &p) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t slots = static_cast<uint64_t>(sm_count(dev)) * (p.head_dim == 64 ? 4 : 2);
  const uint32_t group = p.q_heads / p.kv_heads;
  Split s;
  s.head_blocks = p.kv_heads * ((group + 15) / 16);
  const uint64_t units = static_cast<uint64_t>(p.n_seq) * s.head_blocks;
  const uint64_t tiles = p.max_len > 0 ? (static_cast<uint64_t>(p.max_len) + kTile - 1) / kTile : 1;
  uint64_t chunk = (tiles * units + 4 * slots - 1) / (4 * slots);
  chunk = chunk < 4 ? 4 : chunk > 16 ? 16 : chunk;
  uint64_t splits = (tiles + chunk - 1) / chunk;
  const uint64_t most = (32 * slots + units - 1) / units;
  if (splits > most) splits = most;
  if (splits > 1024) splits = 1024;
  s.splits = static_cast<uint32_t>(splits);
  s.chunk = static_cast<uint32_t>(chunk);
  return s;
}

// Tokens of sequence s that the page table has room for.
__device__ __forceinline__ uint32_t cached_tokens(const PagedAttention &p, uint32_t s, bool tell) {
  const uint32_t room = p.max_pages * p.page.size;  // < 2^31
  const int32_t n = p.lens[s];
  if (n <= 0) return 0;
  if (static_cast<uint32_t>(n) > room) {
    if (tell) report(p.status, kErrPage);
    return room;
  }
  return static_cast<uint32_t>(n);
}
}  // namespace

template <bool kBf16, int kDim>
__global__ void __launch_bounds__(kThreads)
    attention_paged_kernel(const PagedAttention p, const Split sp) {
  constexpr int kChunks = kDim / 8;            // 16-byte chunks of a row
  constexpr int kRowsPass = kThreads / kChunks;
  constexpr int kTileBytes = kTile * kDim * 2;  // of K or of V
  constexpr int kSteps = kDim / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  int64_t(*rows)[kTile][2] = reinterpret_cast<int64_t(*)[kTile][2]>(smem + kStages * 2 * kTileBytes);
  const uint32_t smem0 = smem_u32(smem);
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

  const uint32_t split = blockIdx.x % sp.splits;
  const uint32_t hb = blockIdx.x / sp.splits % sp.head_blocks;
  const uint32_t s = blockIdx.x / sp.splits / sp.head_blocks;
  const uint32_t group = p.q_heads / p.kv_heads, blocks = sp.head_blocks / p.kv_heads;
  const uint32_t g = hb / blocks, h0 = g * group + hb % blocks * 16;
  const uint32_t heads = min(16u, (g + 1) * group - h0);

  const uint32_t len = cached_tokens(p, s, tid == 0 && split == 0 && hb == 0);
  const uint32_t tiles = (len + kTile - 1) / kTile;
  const uint32_t n_chunks = (tiles + sp.chunk - 1) / sp.chunk;
  if (split >= n_chunks && !(split == 0 && sp.splits == 1)) return;
  // This CTA's tiles: chunks split, split + splits, ...; the last chunk of the sequence may be short.
  const uint32_t mine = split < n_chunks ? (n_chunks - 1 - split) / sp.splits + 1 : 0;
  uint32_t count = mine * sp.chunk;
  if (mine > 0 && (n_chunks - 1) % sp.splits == split) count -= n_chunks * sp.chunk - tiles;
  auto tile_at = [&](uint32_t i) {
    return (split + i / sp.chunk * sp.splits) * sp.chunk + i % sp.chunk;
  };

  // The element offset of each row of a tile in the two caches, -1 where there is none.
  const int32_t *table = p.page_table + static_cast<int64_t>(s) * p.table_stride;
  auto look_up = [&](uint32_t i, uint32_t r, int64_t &k_at, int64_t &v_at) {
    k_at = v_at = -1;
    if (i >= count) return;
    const uint32_t j = tile_at(i) * kTile + r;
    if (j >= len) return;
    const uint32_t page = page_of(p.page, j);
    const int32_t id = __ldg(table + page);
    if (id < 0 || static_cast<uint32_t>(id) >= p.n_pages) {
      report(p.status, kErrPage);
      return;
    }
    const int64_t row = (static_cast<int64_t>(g) * p.page.size + (j - page * p.page.size)) * kDim;
    k_at = id * p.k_page + row;
    v_at = id * p.v_page + row;
  };
  const uint32_t c = tid % kChunks, r0 = tid / kChunks;
  auto load_tile = [&](uint32_t i) {
    if (i < count) {
      const uint32_t kb = smem0 + i % kStages * 2 * kTileBytes;
#pragma unroll
      for (int r = r0, n = 0; n < kTile / kRowsPass; ++n, r += kRowsPass) {
        const int64_t k_at = rows[i % kRing][r][0], v_at = rows[i % kRing][r][1];
        const uint32_t dst = kb + r * kDim * 2 + ((c ^ (r & 7)) * 16);
        cp_async16(dst, p.k_cache + (k_at < 0 ? 0 : k_at + c * 8), k_at >= 0);
        cp_async16(dst + kTileBytes, p.v_cache + (v_at < 0 ? 0 : v_at + c * 8), v_at >= 0);
      }
    }
    cp_async_commit();
  };

  for (uint32_t x = tid; x < kStages * kTile; x += kThreads) {
    int64_t k_at, v_at;
    look_up(x / kTile, x % kTile, k_at, v_at);
    rows[x / kTile][x % kTile][0] = k_at;
    rows[x / kTile][x % kTile][1] = v_at;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load_tile(i);

  // Q as the products' A operand: rows lane / 4 and lane / 4 + 8, columns 2 (lane % 4) of each half
  const uint32_t ra = lane / 4, cq = 2 * (lane % 4);
  uint32_t q[kSteps][4];
  {
    const uint16_t *qa = p.q + static_cast<int64_t>(s) * p.q_seq + static_cast<int64_t>(h0 + ra) * p.q_head + cq;
    const uint16_t *qb = qa + 8 * p.q_head;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      q[k][0] = ra < heads ? *reinterpret_cast<const uint32_t *>(qa + 16 * k) : 0u;
      q[k][1] = ra + 8 < heads ? *reinterpret_cast<const uint32_t *>(qb + 16 * k) : 0u;
      q[k][2] = ra < heads ? *reinterpret_cast<const uint32_t *>(qa + 16 * k + 8) : 0u;
      q[k][3] = ra + 8 < heads ? *reinterpret_cast<const uint32_t *>(qb + 16 * k + 8) : 0u;
    }
  }
  float o[kDim / 8][4];
#pragma unroll
  for (int n = 0; n < kDim / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const float c2 = p.scale * kLog2e;

  const uint32_t key0 = warp * 16;
  for (uint32_t i = 0; i < count; ++i) {
    cp_async_wait<kStages - 2>();
    __syncthreads();  // tile i is in; tile i - 1's stage and the oldest addresses are free
    load_tile(i + kStages - 1);
    int64_t k_at, v_at;
    if (tid < kTile) look_up(i + kStages, tid, k_at, v_at);

    const uint32_t kb = smem0 + i % kStages * 2 * kTileBytes, vb = kb + kTileBytes;
    float sc[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
    {
      // four 8x8 matrices: keys 0-7 and 8-15 of the warp, both halves of 16 channels
      const uint32_t r = key0 + (lane / 16) * 8 + lane % 8;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t b[4];
        ldsm4(kb + r * kDim * 2 + (((2 * k + (lane / 8 & 1)) ^ (r & 7)) * 16), b);
        mma16816<kBf16>(sc[0], q[k], b[0], b[1]);
        mma16816<kBf16>(sc[1], q[k], b[2], b[3]);
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int64_t *at = rows[i % kRing][key0 + n * 8 + cq];
      if (at[0] < 0) sc[n][0] = sc[n][2] = -INFINITY;
      if (at[2] < 0) sc[n][1] = sc[n][3] = -INFINITY;
    }
    uint32_t pa[4];
    float keep[2];
    bool moved = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(top, m[h]);
      const float base = top == -INFINITY ? 0.f : top * c2;
      keep[h] = ex2_approx(m[h] * c2 - base);
      moved |= top != m[h];
      m[h] = top;
      const float p0 = ex2_approx(fmaf(sc[0][2 * h], c2, -base)), p1 = ex2_approx(fmaf(sc[0][2 * h + 1], c2, -base));
      const float p2 = ex2_approx(fmaf(sc[1][2 * h], c2, -base)), p3 = ex2_approx(fmaf(sc[1][2 * h + 1], c2, -base));
      l[h] = fmaf(l[h], keep[h], (p0 + p1) + (p2 + p3));
      pa[h] = Elem<kBf16>::pack(p0, p1);
      pa[2 + h] = Elem<kBf16>::pack(p2, p3);
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < kDim / 8; ++n) {
        o[n][0] *= keep[0];
        o[n][1] *= keep[0];
        o[n][2] *= keep[1];
        o[n][3] *= keep[1];
      }
    }
    {
      // keys 0-7 and 8-15 of the warp, two 8-channel columns
      const uint32_t r = key0 + lane % 16;
#pragma unroll
      for (int n = 0; n < kDim / 16; ++n) {
        uint32_t b[4];
        ldsm4t(vb + r * kDim * 2 + (((2 * n + lane / 16) ^ (r & 7)) * 16), b);
        mma16816<kBf16>(o[2 * n], pa, b[0], b[1]);
        mma16816<kBf16>(o[2 * n + 1], pa, b[2], b[3]);
      }
    }
    if (tid < kTile) {
      rows[(i + kStages) % kRing][tid][0] = k_at;
      rows[(i + kStages) % kRing][tid][1] = v_at;
    }
  }
  pdl_trigger();

  // Join the four warps: their maxima and sums, then the outputs scaled to the common maximum.
  cp_async_wait<0>();
  __syncthreads();
  float *wo = reinterpret_cast<float *>(smem);                      // [4][16][kDim]
  float(*wml)[16][2] = reinterpret_cast<float(*)[16][2]>(rows);     // [4][16] (max, sum)
  static_assert(4 * 16 * kDim * 4 <= kStages * 2 * kTileBytes && 4 * 16 * 2 * 4 <= kRing * kTile * 16, "reuse");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (lane % 4 == 0) {
      wml[warp][ra + 8 * h][0] = m[h];
      wml[warp][ra + 8 * h][1] = l[h];
    }
#pragma unroll
    for (int n = 0; n < kDim / 8; ++n)
      *reinterpret_cast<float2 *>(wo + (warp * 16 + ra + 8 * h) * kDim + n * 8 + cq) =
          make_float2(o[n][2 * h], o[n][2 * h + 1]);
  }
  __syncthreads();
  constexpr int kQuads = kDim / 4;
  for (uint32_t x = tid; x < heads * kQuads; x += kThreads) {
    const uint32_t h = x / kQuads, d = x % kQuads * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, wml[w][h][0]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = top == -INFINITY ? 1.f : ex2_approx((wml[w][h][0] - top) * c2);
      const float4 v = *reinterpret_cast<const float4 *>(wo + (w * 16 + h) * kDim + d);
      sum = fmaf(wml[w][h][1], f, sum);
      acc.x = fmaf(v.x, f, acc.x);
      acc.y = fmaf(v.y, f, acc.y);
      acc.z = fmaf(v.z, f, acc.z);
      acc.w = fmaf(v.w, f, acc.w);
    }
    const int64_t row = static_cast<int64_t>(s) * p.q_heads + h0 + h;
    if (sp.splits == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2 *>(p.out + static_cast<int64_t>(s) * p.out_seq + (h0 + h) * p.out_head + d) =
          make_uint2(Elem<kBf16>::pack(acc.x * inv, acc.y * inv), Elem<kBf16>::pack(acc.z * inv, acc.w * inv));
      if (p.lse && d == 0) p.lse[row] = (top * c2 + log2f(sum)) * kLn2;
    } else {
      const int64_t rows_total = static_cast<int64_t>(p.n_seq) * p.q_heads;
      float *part = static_cast<float *>(p.workspace);
      *reinterpret_cast<float4 *>(part + (row * sp.splits + split) * kDim + d) = acc;
      if (d == 0)
        reinterpret_cast<float2 *>(part + rows_total * sp.splits * kDim)[row * sp.splits + split] =
            make_float2(top * c2, sum);
    }
  }
}

// Joins the splits of one (sequence, query head): out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
// Eight warps take every eighth split, then meet in shared memory, always in the same order.
template <bool kBf16, int kDim>
__global__ void __launch_bounds__(256) attention_paged_join_kernel(const PagedAttention p, const Split sp) {
  constexpr int kWarps = 8;
  constexpr int kLane = kDim / 32;  // channels per lane
  __shared__ float po[kWarps][kDim];
  __shared__ float2 pml[kWarps];
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t row = blockIdx.x;
  const uint32_t s = blockIdx.x / p.q_heads, h = blockIdx.x % p.q_heads;
  pdl_wait();
  const uint32_t tiles = (cached_tokens(p, s, false) + kTile - 1) / kTile;
  const uint32_t n = min((tiles + sp.chunk - 1) / sp.chunk, sp.splits);  // splits that wrote
  const float *part = static_cast<const float *>(p.workspace) + row * sp.splits * kDim;
  const float2 *ml = reinterpret_cast<const float2 *>(
                         static_cast<const float *>(p.workspace) +
                         static_cast<int64_t>(p.n_seq) * p.q_heads * sp.splits * kDim) + row * sp.splits;
  float top = -INFINITY;
  for (uint32_t i = lane; i < n; i += 32) top = fmaxf(top, ml[i].x);
#pragma unroll
  for (int i = 16; i > 0; i /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
  float sum = 0.f, acc[kLane] = {};
#pragma unroll 4
  for (uint32_t i = warp; i < n; i += kWarps) {
    const float2 x = ml[i];
    const float f = top == -INFINITY ? 1.f : ex2_approx(x.x - top);
    sum = fmaf(x.y, f, sum);
#pragma unroll
    for (int e = 0; e < kLane; e += 2) {
      const float2 v = *reinterpret_cast<const float2 *>(part + static_cast<int64_t>(i) * kDim + lane * kLane + e);
      acc[e] = fmaf(v.x, f, acc[e]);
      acc[e + 1] = fmaf(v.y, f, acc[e + 1]);
    }
  }
#pragma unroll
  for (int e = 0; e < kLane; ++e) po[warp][lane * kLane + e] = acc[e];
  if (lane == 0) pml[warp] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.x < kDim / 2) {
    const uint32_t d = threadIdx.x * 2;
    float a = 0.f, b = 0.f;
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      a += po[w][d];
      b += po[w][d + 1];
      sum += pml[w].y;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint32_t *>(p.out + static_cast<int64_t>(s) * p.out_seq + h * p.out_head + d) =
        Elem<kBf16>::pack(a * inv, b * inv);
    if (p.lse && d == 0) p.lse[row] = (top + log2f(sum)) * kLn2;
  }
}

size_t attention_paged_workspace(const PagedAttention &p) {
  const Split s = split_of(p);
  if (s.splits <= 1) return 0;
  return static_cast<size_t>(p.n_seq) * p.q_heads * s.splits * (p.head_dim + 2) * sizeof(float);
}

namespace {
template <bool kBf16, int kDim>
cudaError_t launch(const PagedAttention &p, cudaStream_t stream) {
  static std::atomic<bool> configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev].load(std::memory_order_acquire)) {
    // setting the attribute twice (two threads racing here) is harmless
    const cudaError_t e = cudaFuncSetAttribute(attention_paged_kernel<kBf16, kDim>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               smem_bytes<kDim>());
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  const Split s = split_of(p);
  const uint64_t grid = static_cast<uint64_t>(p.n_seq) * s.head_blocks * s.splits;
  const uint64_t join = static_cast<uint64_t>(p.n_seq) * p.q_heads;
  if (grid > 0x7fffffffull || join > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  attention_paged_kernel<kBf16, kDim>
      <<<dim3(static_cast<uint32_t>(grid)), dim3(kThreads), smem_bytes<kDim>(), stream>>>(p, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || s.splits == 1) return e;
  return launch_pdl(attention_paged_join_kernel<kBf16, kDim>, dim3(static_cast<uint32_t>(join)),
                    dim3(256), 0, stream, p, s);
}
}  // namespace

cudaError_t launch_attention_paged(const PagedAttention &p, bool bf16, cudaStream_t stream) {
  if (p.n_seq == 0) return cudaSuccess;
  if (p.head_dim == 64) return bf16 ? launch<true, 64>(p, stream) : launch<false, 64>(p, stream);
  return bf16 ? launch<true, 128>(p, stream) : launch<false, 128>(p, stream);
}

}  // namespace dv3
