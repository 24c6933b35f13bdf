// attention_paged.cu - attention of one new token per sequence over a paged key-value cache.
//
// For sequence s of n = lens[s] cached tokens and query head h reading key-value head
// h / (q_heads / kv_heads): o = sum_j w_j v_j / sum_j w_j, w_j = exp(scale (q . k_j - max)), over
// j < n. Key j lies in slot j % page_size of page page_table[s][j / page_size]. No tokens give 0
// (and -inf as the log-sum). A page id outside the pool, or a length past the table, is reported in
// `status` and its tokens count as absent.
//
// Bound by the one read of K and V: a key costs 4 head_dim bytes and 4 head_dim flops for each of
// the group's query heads, far below the tensor cores' rate. So the kernel is a stream of 64-key
// tiles of K and V through a ring of shared-memory stages by 16-byte cp.async (any page size; a
// tile's row addresses are looked up a tile before its loads are issued), and the CTAs (four an SM
// at 64 channels, two at 128) run on without a break:
//   - A unit is one (sequence, key-value head); groups of more than 16 query heads make one for
//     each 16. The tiles of all units stand in one row, and each CTA takes an equal stretch of
//     it, whatever the lengths: the loads of a stretch's next unit are under way while this one is
//     finished. A unit that lies in one stretch is written out; of one that does not each CTA
//     leaves (max, sum, unnormalised output) in the workspace, at most two a CTA, and a second
//     launch joins them in order. Nothing depends on the order in which CTAs end.
//   - Where no sequence passes 256 keys, stretches are whole units and there is nothing to join.
// Within a tile each of the four warps computes the scores of 16 keys for the group's up to 16
// query heads (m16n8k16 tensor-core products, rows past the group zero), the warps agree on the
// running maximum in shared memory, and each then multiplies all 64 weights with its quarter of V's
// channels: no warp's output has to be added to another's at a unit's end, which for short
// sequences cost more than the keys (26.6 us against NNNN for 256 images of 201 tokens).
#include <atomic>

#include "sequence.cuh"

namespace dv3 {

namespace {
constexpr int kThreads = 128;
constexpr int kTile = 64;     // keys per stage, 16 per warp
constexpr int kStages = 3;
constexpr int kRing = 4;      // tiles whose row addresses are kept: kStages + the one being looked up
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

constexpr uint32_t kLeast = 4;  // tiles that a CTA takes at least

// Stages | row addresses | weights of a tile [16][64], 128-byte rows
template <int kDim>
constexpr int smem_bytes() {
  return kStages * 2 * kTile * kDim * 2 + kRing * kTile * 2 * 8 + 16 * kTile * 2;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
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

// The grid, and how it cuts the work.
struct Plan {
  uint32_t grid, head_blocks, rows;  // rows: query heads of a unit at most
  bool units;                        // stretches are whole units
};

Plan plan_of(const PagedAttention &p) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t slots = static_cast<uint64_t>(sm_count(dev)) * (p.head_dim == 64 ? 4 : 2);
  const uint32_t group = p.q_heads / p.kv_heads;
  Plan s;
  s.head_blocks = p.kv_heads * ((group + 15) / 16);
  s.rows = group < 16 ? group : 16;
  const uint64_t units = static_cast<uint64_t>(p.n_seq) * s.head_blocks;
  const uint64_t tiles = (static_cast<uint64_t>(p.max_len) + kTile - 1) / kTile;
  s.units = tiles <= kLeast;
  // as many CTAs as run at once, but none for less than a unit or kLeast tiles
  const uint64_t most = s.units ? units : units * ((tiles + kLeast - 1) / kLeast);
  s.grid = static_cast<uint32_t>(most < slots ? most : slots);
  return s;
}

// Workspace: the first tile of each sequence in the row of all tiles [n_seq + 1] (u64, written by
// CTA 0), then (max, sum) and the output of [grid][2][rows] partial results.
__host__ __device__ inline size_t starts_bytes(uint32_t n_seq) {
  return ((static_cast<size_t>(n_seq) + 1) * 8 + 15) / 16 * 16;
}
struct Partials {
  uint64_t *starts;
  float2 *ml;
  float *o;
};
__device__ __forceinline__ Partials partials_of(const PagedAttention &p, const Plan &pl) {
  Partials w;
  uint8_t *at = static_cast<uint8_t *>(p.workspace);
  w.starts = reinterpret_cast<uint64_t *>(at);
  w.ml = reinterpret_cast<float2 *>(at + starts_bytes(p.n_seq));
  const size_t n = (static_cast<size_t>(pl.grid) * 2 * pl.rows + 1) / 2 * 2;
  w.o = reinterpret_cast<float *>(w.ml + n);
  return w;
}
// Tiles of a stretch.
__device__ __forceinline__ uint64_t stretch_of(uint64_t total, uint32_t grid) {
  const uint64_t n = (total + grid - 1) / grid;
  return n < kLeast ? kLeast : n;
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
__global__ void __launch_bounds__(kThreads, kDim == 64 ? 4 : 2)
    attention_paged_kernel(const PagedAttention p, const Plan pl) {
  constexpr int kChunks = kDim / 8;            // 16-byte chunks of a row
  constexpr int kRowsPass = kThreads / kChunks;
  constexpr int kTileBytes = kTile * kDim * 2;  // of K or of V
  constexpr int kSteps = kDim / 16;
  constexpr int kCols = kDim / 4 / 16;  // 16-channel columns of a warp's quarter
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float tops[4][16], sums[4][16];
  __shared__ uint64_t found[2][3];  // the stretch's two ends: sequence, head block, tile
  __shared__ uint64_t scan[4];
  int64_t(*rows)[kTile][2] = reinterpret_cast<int64_t(*)[kTile][2]>(smem + kStages * 2 * kTileBytes);
  const uint32_t smem0 = smem_u32(smem), w_at = smem0 + kStages * 2 * kTileBytes + kRing * kTile * 16;
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t group = p.q_heads / p.kv_heads, blocks = pl.head_blocks / p.kv_heads;
  auto tiles_of = [&](uint32_t s) { return (cached_tokens(p, s, false) + kTile - 1) / kTile; };

  // The stretch of this CTA: from (s, hb, t) up to but without (end_s, end_hb, end_t).
  uint64_t per = 0;  // tiles of a stretch
  if (pl.units) {
    const uint64_t n = static_cast<uint64_t>(p.n_seq) * pl.head_blocks;
    if (tid < 2) {
      const uint64_t u = n * (blockIdx.x + tid) / pl.grid;
      found[tid][0] = u / pl.head_blocks;
      found[tid][1] = u % pl.head_blocks;
      found[tid][2] = 0;
    }
  } else {
    const uint32_t each = (p.n_seq + kThreads - 1) / kThreads;
    const uint32_t from = min(tid * each, p.n_seq), to = min(from + each, p.n_seq);
    uint64_t mine = 0;
    for (uint32_t s = from; s < to; ++s) mine += tiles_of(s);
    mine *= pl.head_blocks;
    uint64_t sum = mine;
#pragma unroll
    for (int i = 1; i < 32; i *= 2) {
      const uint64_t x = __shfl_up_sync(0xffffffffu, sum, i);
      if (lane >= static_cast<uint32_t>(i)) sum += x;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    uint64_t total = 0, before = sum - mine;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    per = stretch_of(total, pl.grid);
    const uint64_t first = per * blockIdx.x, beyond = first + per;
    const uint64_t ends[2] = {first < total ? first : total, beyond < total ? beyond : total};
    if (tid < 2 && ends[tid] == total) {
      found[tid][0] = p.n_seq;
      found[tid][1] = found[tid][2] = 0;
    }
    uint64_t *starts = static_cast<uint64_t *>(p.workspace);
    uint64_t at = before;
    for (uint32_t s = from; s < to; ++s) {
      if (blockIdx.x == 0) starts[s] = at;
      const uint64_t n = tiles_of(s), next = at + n * pl.head_blocks;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (ends[e] >= at && ends[e] < next) {
          found[e][0] = s;
          found[e][1] = (ends[e] - at) / n;
          found[e][2] = (ends[e] - at) % n;
        }
      at = next;
    }
    if (blockIdx.x == 0 && tid == 0) starts[p.n_seq] = total;
  }
  __syncthreads();
  const uint32_t end_s = static_cast<uint32_t>(found[1][0]), end_hb = static_cast<uint32_t>(found[1][1]),
                 end_t = static_cast<uint32_t>(found[1][2]);

  // A place in the row of tiles; the loads run ahead of the products with a place of their own.
  struct Place {
    uint32_t s, hb, t, len, tiles, end;  // end: tiles of this unit up to the stretch's end
  };
  auto enter = [&](Place &x) {  // the unit at (s, hb); its end, 0 past the stretch
    x.end = 0;
    if (x.s >= p.n_seq || (x.s == end_s && x.hb > end_hb) || x.s > end_s) return;
    x.len = cached_tokens(p, x.s, false);
    x.tiles = (x.len + kTile - 1) / kTile;
    x.end = x.s == end_s && x.hb == end_hb ? end_t : x.tiles;
  };
  auto past = [&](const Place &x) {  // the unit is not of the stretch any more
    return x.s >= p.n_seq || x.s > end_s || (x.s == end_s && (x.hb > end_hb || (x.hb == end_hb && end_t == 0)));
  };
  auto next_unit = [&](Place &x) {
    x.t = 0;
    if (++x.hb == pl.head_blocks) {
      x.hb = 0;
      ++x.s;
    }
    enter(x);
  };
  Place ld = {static_cast<uint32_t>(found[0][0]), static_cast<uint32_t>(found[0][1]),
              static_cast<uint32_t>(found[0][2]), 0, 0, 0};
  enter(ld);
  Place at = ld;
  auto settle = [&] {  // to the next tile there is
    while (ld.t >= ld.end && !past(ld)) next_unit(ld);
  };
  settle();

  // The element offsets of row r of the tile at `ld` in the two caches, -1 where there is none.
  auto look_up = [&](uint32_t r, int64_t &k_at, int64_t &v_at) {
    k_at = v_at = -1;
    if (ld.t >= ld.end) return;
    const uint32_t j = ld.t * kTile + r;
    if (j >= ld.len) return;
    const uint32_t page = page_of(p.page, j);
    const int32_t id = __ldg(p.page_table + static_cast<int64_t>(ld.s) * p.table_stride + page);
    if (id < 0 || static_cast<uint32_t>(id) >= p.n_pages) {
      report(p.status, kErrPage);
      return;
    }
    const int64_t row = (static_cast<int64_t>(ld.hb / blocks) * p.page.size + (j - page * p.page.size)) * kDim;
    k_at = id * p.k_page + row;
    v_at = id * p.v_page + row;
  };
  uint32_t known = 0;  // tiles looked up
  auto advance = [&] {
    if (ld.t >= ld.end) return;
    ++known;
    ++ld.t;
    settle();
  };
  const uint32_t c = tid % kChunks, r0 = tid / kChunks;
  auto load_tile = [&](uint32_t i) {
    if (i < known) {
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

#pragma unroll 1
  for (int i = 0; i < kStages; ++i) {
    int64_t k_at, v_at;
    if (tid < kTile) {
      look_up(tid, k_at, v_at);
      rows[i][tid][0] = k_at;
      rows[i][tid][1] = v_at;
    }
    advance();
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load_tile(i);

  const uint32_t ra = lane / 4, cq = 2 * (lane % 4), key0 = warp * 16;
  const float c2 = p.scale * kLog2e;
  uint32_t i = 0;  // tiles done
  while (!past(at)) {
    const uint32_t g = at.hb / blocks, h0 = g * group + at.hb % blocks * 16;
    const uint32_t heads = min(16u, (g + 1) * group - h0);
    const bool whole = at.t == 0 && at.end == at.tiles;
    const uint32_t slot = i == 0 ? 0 : 1;  // the stretch's first unit, or its last
    if (tid == 0 && at.hb == 0) cached_tokens(p, at.s, true);  // tells of a length past the table
    if (at.t >= at.end) __syncthreads();                       // `sums` may still be read

    // Q as the products' A operand: rows lane / 4 and lane / 4 + 8, columns 2 (lane % 4) of each half
    uint32_t q[kSteps][4];
    {
      const uint16_t *qa = p.q + static_cast<int64_t>(at.s) * p.q_seq + static_cast<int64_t>(h0 + ra) * p.q_head + cq;
      const uint16_t *qb = qa + 8 * p.q_head;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        q[k][0] = ra < heads ? *reinterpret_cast<const uint32_t *>(qa + 16 * k) : 0u;
        q[k][1] = ra + 8 < heads ? *reinterpret_cast<const uint32_t *>(qb + 16 * k) : 0u;
        q[k][2] = ra < heads ? *reinterpret_cast<const uint32_t *>(qa + 16 * k + 8) : 0u;
        q[k][3] = ra + 8 < heads ? *reinterpret_cast<const uint32_t *>(qb + 16 * k + 8) : 0u;
      }
    }
    float o[2 * kCols][4];
#pragma unroll
    for (int n = 0; n < 2 * kCols; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (; at.t < at.end; ++at.t, ++i) {
      cp_async_wait<kStages - 2>();
      __syncthreads();  // tile i is in; tile i - 1's stage, weights and the oldest addresses are free
      load_tile(i + kStages - 1);
      int64_t k_at, v_at;
      if (tid < kTile) look_up(tid, k_at, v_at);
      advance();

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
        const int64_t *row = rows[i % kRing][key0 + n * 8 + cq];
        if (row[0] < 0) sc[n][0] = sc[n][2] = -INFINITY;
        if (row[2] < 0) sc[n][1] = sc[n][3] = -INFINITY;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (lane % 4 == 0) tops[warp][ra + 8 * h] = top;
      }
      __syncthreads();
      float keep[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t r = ra + 8 * h;
        const float top = fmaxf(m[h], fmaxf(fmaxf(tops[0][r], tops[1][r]), fmaxf(tops[2][r], tops[3][r])));
        const float base = top == -INFINITY ? 0.f : top * c2;
        keep[h] = ex2_approx(fmaf(m[h], c2, -base));
        m[h] = top;
        const float p0 = ex2_approx(fmaf(sc[0][2 * h], c2, -base)), p1 = ex2_approx(fmaf(sc[0][2 * h + 1], c2, -base));
        const float p2 = ex2_approx(fmaf(sc[1][2 * h], c2, -base)), p3 = ex2_approx(fmaf(sc[1][2 * h + 1], c2, -base));
        l[h] = fmaf(l[h], keep[h], (p0 + p1) + (p2 + p3));
        const uint32_t row = w_at + r * (kTile * 2) + (cq * 2);
        sts32(row + (((2 * warp) ^ (r & 7)) * 16), Elem<kBf16>::pack(p0, p1));
        sts32(row + (((2 * warp + 1) ^ (r & 7)) * 16), Elem<kBf16>::pack(p2, p3));
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < 2 * kCols; ++n) {
        o[n][0] *= keep[0];
        o[n][1] *= keep[0];
        o[n][2] *= keep[1];
        o[n][3] *= keep[1];
      }
      {
        const uint32_t r = lane % 16;
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k) {
          uint32_t w[4];
          ldsm4(w_at + r * (kTile * 2) + (((2 * k + lane / 16) ^ (r & 7)) * 16), w);
#pragma unroll
          for (int n = 0; n < kCols; ++n) {
            // keys 0-7 and 8-15 of the step, two 8-channel columns
            uint32_t b[4];
            ldsm4t(vb + (k * 16 + r) * kDim * 2 + (((warp * (kDim / 32) + 2 * n + lane / 16) ^ (r & 7)) * 16), b);
            mma16816<kBf16>(o[2 * n], w, b[0], b[1]);
            mma16816<kBf16>(o[2 * n + 1], w, b[2], b[3]);
          }
        }
      }
      if (tid < kTile) {
        rows[(i + kStages) % kRing][tid][0] = k_at;
        rows[(i + kStages) % kRing][tid][1] = v_at;
      }
    }

    // The unit's end: the row sums of the four warps, then this warp's quarter of the channels.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (lane % 4 == 0) sums[warp][ra + 8 * h] = l[h];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t r = ra + 8 * h;
      if (r >= heads) continue;
      const float sum = (sums[0][r] + sums[1][r]) + (sums[2][r] + sums[3][r]);
      const uint32_t col = warp * (kDim / 4) + cq;
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint16_t *dst = p.out + static_cast<int64_t>(at.s) * p.out_seq + (h0 + r) * p.out_head + col;
#pragma unroll
        for (int n = 0; n < 2 * kCols; ++n)
          *reinterpret_cast<uint32_t *>(dst + 8 * n) = Elem<kBf16>::pack(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
        if (p.lse && col == 0)
          p.lse[static_cast<int64_t>(at.s) * p.q_heads + h0 + r] = (m[h] * c2 + log2f(sum)) * kLn2;
      } else {
        const Partials w = partials_of(p, pl);
        const size_t row = (static_cast<size_t>(blockIdx.x) * 2 + slot) * pl.rows + r;
#pragma unroll
        for (int n = 0; n < 2 * kCols; ++n)
          *reinterpret_cast<float2 *>(w.o + row * kDim + col + 8 * n) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if (col == 0) w.ml[row] = make_float2(m[h] * c2, sum);
      }
    }
    next_unit(at);
  }
  pdl_trigger();
  cp_async_wait<0>();
}

// Joins the units that several stretches share, a CTA for each (sequence, query head):
// out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the CTAs i in order; and writes the rows
// of empty sequences. Four warps take every fourth, then meet in shared memory.
template <bool kBf16, int kDim>
__global__ void __launch_bounds__(128) attention_paged_join_kernel(const PagedAttention p, const Plan pl) {
  constexpr int kLane = kDim / 32;  // channels per lane
  __shared__ float po[4][kDim];
  __shared__ float pl4[4];
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t row = blockIdx.x;
  const uint32_t s = blockIdx.x / p.q_heads, h = blockIdx.x % p.q_heads;
  const uint32_t group = p.q_heads / p.kv_heads, blocks = pl.head_blocks / p.kv_heads;
  const uint32_t hb = h / group * blocks + h % group / 16, r = h % group % 16;
  pdl_wait();
  const Partials w = partials_of(p, pl);
  const uint64_t per = stretch_of(w.starts[p.n_seq], pl.grid);
  const uint64_t tiles = (w.starts[s + 1] - w.starts[s]) / pl.head_blocks;
  const uint64_t from = w.starts[s] + hb * tiles, to = from + tiles;
  const uint32_t c0 = static_cast<uint32_t>(from / per);
  const uint32_t n = tiles ? static_cast<uint32_t>((to - 1) / per) - c0 + 1 : 0;
  if (n == 1) return;  // one CTA's: written
  auto slot_of = [&](uint32_t i) {  // the unit is the first of that CTA's stretch, or its last
    return (static_cast<size_t>(c0 + i) * 2 + (per * (c0 + i) >= from ? 0 : 1)) * pl.rows + r;
  };
  float top = -INFINITY;
  for (uint32_t i = lane; i < n; i += 32) top = fmaxf(top, w.ml[slot_of(i)].x);
#pragma unroll
  for (int i = 16; i > 0; i /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
  float sum = 0.f, acc[kLane] = {};
#pragma unroll 4
  for (uint32_t i = warp; i < n; i += 4) {
    const size_t at = slot_of(i);
    const float2 x = w.ml[at];
    const float f = top == -INFINITY ? 1.f : ex2_approx(x.x - top);
    sum = fmaf(x.y, f, sum);
#pragma unroll
    for (int e = 0; e < kLane; e += 2) {
      const float2 v = *reinterpret_cast<const float2 *>(w.o + at * kDim + lane * kLane + e);
      acc[e] = fmaf(v.x, f, acc[e]);
      acc[e + 1] = fmaf(v.y, f, acc[e + 1]);
    }
  }
#pragma unroll
  for (int e = 0; e < kLane; ++e) po[warp][lane * kLane + e] = acc[e];
  if (lane == 0) pl4[warp] = sum;
  __syncthreads();
  if (threadIdx.x < kDim / 2) {
    const uint32_t d = threadIdx.x * 2;
    sum = (pl4[0] + pl4[1]) + (pl4[2] + pl4[3]);
    const float a = (po[0][d] + po[1][d]) + (po[2][d] + po[3][d]);
    const float b = (po[0][d + 1] + po[1][d + 1]) + (po[2][d + 1] + po[3][d + 1]);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint32_t *>(p.out + static_cast<int64_t>(s) * p.out_seq + h * p.out_head + d) =
        Elem<kBf16>::pack(a * inv, b * inv);
    if (p.lse && d == 0) p.lse[row] = (top + log2f(sum)) * kLn2;
  }
}

size_t attention_paged_workspace(const PagedAttention &p) {
  const Plan pl = plan_of(p);
  if (pl.units) return 0;
  const size_t n = (static_cast<size_t>(pl.grid) * 2 * pl.rows + 1) / 2 * 2;
  return starts_bytes(p.n_seq) + n * (p.head_dim + 2) * sizeof(float);
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
  const Plan pl = plan_of(p);
  const uint64_t join = static_cast<uint64_t>(p.n_seq) * p.q_heads;
  if (join > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  attention_paged_kernel<kBf16, kDim><<<dim3(pl.grid), dim3(kThreads), smem_bytes<kDim>(), stream>>>(p, pl);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || pl.units) return e;
  return launch_pdl(attention_paged_join_kernel<kBf16, kDim>, dim3(static_cast<uint32_t>(join)),
                    dim3(128), 0, stream, p, pl);
}
}  // namespace

cudaError_t launch_attention_paged(const PagedAttention &p, bool bf16, cudaStream_t stream) {
  if (p.n_seq == 0) return cudaSuccess;
  if (p.head_dim == 64) return bf16 ? launch<true, 64>(p, stream) : launch<false, 64>(p, stream);
  return bf16 ? launch<true, 128>(p, stream) : launch<false, 128>(p, stream);
}

}  // namespace dv3
