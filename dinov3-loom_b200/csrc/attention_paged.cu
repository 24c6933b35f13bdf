// attention_paged.cu - attention of one new token per sequence over a paged key-value cache.
//
// For sequence s of n = lens[s] cached tokens and query head h reading key-value head
// h / (q_heads / kv_heads): o = sum_j w_j v_j / sum_j w_j, w_j = exp(scale (q . k_j - max)), over
// j < n. Key j lies in slot j % page_size of page page_table[s][j / page_size]. No tokens give 0
// (and -inf as the log-sum). A page id outside the pool, or a length past the table, is reported in
// `status` and its tokens count as absent.
//
// Bound by the one read of K and V: a key costs 4 head_dim bytes and 4 head_dim flops for each of
// the group's query heads, far below the tensor cores' rate. So the kernel is a stream of 16-key
// tiles, and every warp is a stream of its own, without a barrier: its tiles of K and V run
// through its own ring of shared-memory stages by 16-byte cp.async (any page size; a tile's row
// addresses are looked up a tile before its loads are issued), and its scores S^T = K Q^T and its
// O^T += V^T P^T are m16n8k16 tensor-core products: the 16 keys, then 16 channels, are M, and the
// query heads of the group, 8 or 16 (those past the group zero), are N, which leaves the registers
// half of what heads as M take. P, the running maximum, the sum and O stay in registers; the next
// unit's Q is under way while this one runs.
//   - A unit is one (sequence, key-value head); groups of more than 16 query heads make one for
//     each 16. The tiles of all units stand in one row, kUnit more for each unit's start and end,
//     and each warp of the grid (eight an SM at 128 channels, twelve at 64) takes an equal
//     stretch of it, whatever the lengths: the loads of
//     a stretch's next unit are under way while this one is finished. A unit that lies in one
//     stretch is written out; of one that does not each warp leaves (max, sum, unnormalised
//     output) in the workspace, at most two a warp, and a second launch joins them in order.
//     Nothing depends on the order in which warps end.
//   - Where no sequence passes 256 keys, stretches are whole units and there is nothing to join; with
//     no more units than CTAs, the four warps of a CTA share one and join in shared memory. So do
//     the warps of a cluster of 2 to 8 CTAs where units are few and not so long that the rest of the
//     SMs is missed: that spares the second launch (one sequence of 1000 keys, 32/8 heads of 128: 8.1 us,
//     11.4 with it; 2500 keys 11.0 and 11.8; 5000 keys would take 15.9 and not 13.2).
// Four warps on one 64-key tile, meeting at barriers, took 24.8 us for 256 images of 201 tokens and
// 51.5 us for 64 sequences of 1..4096 (32/8 heads of 128); these take 18 and 39. One sequence of 131072 tokens takes 98 us (5.5 TB/s with its join). Groups of more than 16
// query heads read the cache once for every 16: 16 sequences of 32768 keys of one head of 128 take 60 us with 16 query
// heads, 106 with 32 and 293 with 128 (one read: 41).
#include <atomic>
#include <type_traits>

#include "sequence.cuh"

namespace dv3 {

namespace {
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16;  // keys
// Times in us at 32/8 heads of 128 unless said. Tiles that a warp takes at least: 32 sequences of 1..300 keys
// take 10.9 with 4, 14.2 with 8; 9.9 with 2, which gains nowhere else.
constexpr uint32_t kLeast = 4;
// Tiles up to which a unit is not split. 256 sequences of 201 keys, 6 heads of 64, take 17.9 with 16 and 24.4 split (8);
// with 32 they would take 23.6 and not 30.4 at 300 keys each, but 64 of 1..512 keys 29.6 and not 12.8.
constexpr uint32_t kShort = 16;
// What a unit's start and end cost, in tiles: 64 sequences of 1..4096 keys take 39.2 with 2 or 4, 55 with 0.
constexpr uint32_t kUnit = 2;
constexpr uint32_t kJoinTiles = 4;  // what the joining launch costs, in a warp's tiles

// A warp's shared memory: stages of K and V, and the addresses of the rows of the tiles in flight
// and the next (8-byte pointers into K and V; 0: no such row).
template <int kDim>
struct Ring {
  static constexpr int kStages = kDim == 64 ? 4 : 3;
  static constexpr int kAhead = kDim == 64 ? 8 : 4;  // kStages + 1, to a power of two
  static constexpr int kTileBytes = kTile * kDim * 2;  // of K or of V
  static constexpr int kRowsOff = kStages * 2 * kTileBytes;
  static constexpr int kBytes = kRowsOff + kAhead * kTile * 16;
  static constexpr int kPerSm = kDim == 64 ? 3 : 2;  // CTAs
};

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared memory location in the cluster's CTA `rank`, and a load from there.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(addr), "r"(rank));
  return to;
}
__device__ __forceinline__ float2 load_cta(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void sts_zero16(uint32_t dst) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
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
// The transposed 8x8 matrix of 16-bit elements.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
  bool team;                         // the warps of a cluster of CTAs share one unit, a tile each in turn
  uint32_t cluster, log;             // its CTAs, and their number's logarithm
  bool crowd;                        // many stretches share a unit
};

// CTAs that run at once.
uint32_t cta_slots(const PagedAttention &p) {
  int dev = 0;
  cudaGetDevice(&dev);
  return static_cast<uint32_t>(sm_count(dev)) * (p.head_dim == 64 ? Ring<64>::kPerSm : Ring<128>::kPerSm);
}

Plan plan_of(const PagedAttention &p) {
  const uint64_t slots = cta_slots(p);
  const uint32_t group = p.q_heads / p.kv_heads;
  Plan s;
  s.head_blocks = p.kv_heads * ((group + 15) / 16);
  s.rows = group < 16 ? group : 16;
  const uint64_t units = static_cast<uint64_t>(p.n_seq) * s.head_blocks;
  const uint64_t tiles = (static_cast<uint64_t>(p.max_len) + kTile - 1) / kTile;
  // Few long units: a cluster each, whose warps take tiles in turn and meet in its shared memory, where
  // that costs a warp less than kJoinTiles more than an equal share of all tiles.
  s.cluster = 1;
  s.log = 0;
  if (tiles > kShort)
    for (uint32_t log = 3, c = 8; c > 1; c /= 2, --log)
      if (units * c <= slots && tiles / (c * kWarps) <= tiles * units / (slots * kWarps) + kJoinTiles) {
        s.cluster = c;
        s.log = log;
        break;
      }
  s.units = tiles <= kShort || s.cluster > 1;
  s.team = s.cluster > 1 || (s.units && units <= slots);
  // as many CTAs as run at once, but no warp for less than a unit or kLeast tiles
  const uint64_t warps = s.units ? units : units * ((tiles + kLeast - 1) / kLeast);
  const uint64_t most = s.team ? units * s.cluster : (warps + kWarps - 1) / kWarps;
  s.grid = static_cast<uint32_t>(most < slots ? most : slots);
  s.crowd = !s.units && static_cast<uint64_t>(s.grid) * kWarps > 16 * units;
  return s;
}

// Workspace: for each unit with tokens the first warp that has part of it, and how many have (the top
// bit: it is that warp's last unit, not its first), written by that warp; then (max, sum) and the
// output of [warps][2][rows] partial results.
struct Share {
  uint32_t first, parts;
};
constexpr uint32_t kLastUnit = 0x80000000u;
__host__ __device__ inline size_t shares_bytes(const PagedAttention &p, const Plan &pl) {
  return (static_cast<size_t>(p.n_seq) * pl.head_blocks * sizeof(Share) + 15) / 16 * 16;
}
struct Partials {
  Share *shares;
  float2 *ml;
  float *o;
};
__device__ __forceinline__ Partials partials_of(const PagedAttention &p, const Plan &pl) {
  Partials w;
  uint8_t *at = static_cast<uint8_t *>(p.workspace);
  w.shares = reinterpret_cast<Share *>(at);
  w.ml = reinterpret_cast<float2 *>(at + shares_bytes(p, pl));
  const size_t n = (static_cast<size_t>(pl.grid) * kWarps * 2 * pl.rows + 1) / 2 * 2;
  w.o = reinterpret_cast<float *>(w.ml + n);
  return w;
}
// What a unit of that many tiles counts in the row, and the stretches' length in the same measure.
// The cost of its start and end stands before its tiles: an end that falls on it is the unit's
// first tile.
__device__ __forceinline__ uint64_t cost_of(uint32_t tiles) { return tiles ? tiles + kUnit : 0; }
__device__ __forceinline__ uint64_t stretch_of(uint64_t total, uint32_t grid) {
  const uint64_t warps = static_cast<uint64_t>(grid) * kWarps, n = (total + warps - 1) / warps;
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

template <bool kBf16, int kDim, int kHeads8>
__global__ void __launch_bounds__(kThreads, Ring<kDim>::kPerSm)
    attention_paged_kernel(const PagedAttention p, const Plan pl) {
  using R = Ring<kDim>;
  constexpr int kStages = R::kStages, kAhead = R::kAhead, kTileBytes = R::kTileBytes;
  constexpr int kChunks = kDim / 8;  // 16-byte chunks of a row
  constexpr int kRowsPass = 32 / kChunks;
  constexpr int kSteps = kDim / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t found[kWarps + 1][3];  // the stretches' ends: sequence, head block, tile
  __shared__ uint64_t scan[kWarps];
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t group = p.q_heads / p.kv_heads, blocks = pl.head_blocks / p.kv_heads;
  pdl_wait();  // what the kernel before wrote is there from here on
  pdl_trigger();
  auto tiles_of = [&](uint32_t s) { return (cached_tokens(p, s, false) + kTile - 1) / kTile; };

  uint64_t per = 0;  // tiles of a stretch
  // The stretches of this CTA's warps: each from (s, hb, t) up to but without the next one's.
  const uint64_t warp0 = static_cast<uint64_t>(blockIdx.x) * kWarps;
  if (pl.units) {
    const uint64_t n = static_cast<uint64_t>(p.n_seq) * pl.head_blocks, warps = static_cast<uint64_t>(pl.grid) * kWarps;
    if (tid <= kWarps) {
      const uint64_t u = pl.team ? (blockIdx.x >> pl.log) + (tid == kWarps) : n * (warp0 + tid) / warps;
      found[tid][0] = u / pl.head_blocks;
      found[tid][1] = u % pl.head_blocks;
      found[tid][2] = 0;
    }
  } else {
    const uint32_t each = (p.n_seq + kThreads - 1) / kThreads;
    const uint32_t from = min(tid * each, p.n_seq), to = min(from + each, p.n_seq);
    uint64_t mine = 0;
    for (uint32_t s = from; s < to; ++s) mine += cost_of(tiles_of(s));
    mine *= pl.head_blocks;
    uint64_t sum = mine;
#pragma unroll
    for (int i = 1; i < 32; i *= 2) {
      const uint64_t x = __shfl_up_sync(0xffffffffu, sum, i);
      if (lane >= static_cast<uint32_t>(i)) sum += x;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    uint64_t total = 0, at = sum - mine;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      if (w < warp) at += scan[w];
      total += scan[w];
    }
    per = stretch_of(total, pl.grid);
    if (tid <= kWarps && per * (warp0 + tid) >= total) {
      found[tid][0] = p.n_seq;
      found[tid][1] = found[tid][2] = 0;
    }
    for (uint32_t s = from; s < to; ++s) {
      const uint64_t n = cost_of(tiles_of(s)), next = at + n * pl.head_blocks;
#pragma unroll 1
      for (int e = 0; e <= kWarps; ++e) {
        const uint64_t end = per * (warp0 + e);
        if (end >= at && end < next) {
          found[e][0] = s;
          const uint64_t in = (end - at) % n;
          found[e][1] = (end - at) / n;
          found[e][2] = in > kUnit ? in - kUnit : 0;
        }
      }
      at = next;
    }
  }
  __syncthreads();
  const uint32_t to = pl.team ? kWarps : warp + 1, step = pl.team ? kWarps * pl.cluster : 1;
  const uint32_t rank = blockIdx.x & (pl.cluster - 1);  // in the cluster
  const uint32_t end_s = static_cast<uint32_t>(found[to][0]), end_hb = static_cast<uint32_t>(found[to][1]),
                 end_t = static_cast<uint32_t>(found[to][2]);

  // A place in the row of tiles; the loads run ahead of the products with a place of their own.
  struct Place {
    uint32_t s, hb, t, len, tiles, end;  // end: tiles of this unit up to the stretch's end
    uint32_t head;                       // key-value head
  };
  auto past = [&](const Place &x) {  // the unit is not of the stretch any more
    return x.s >= p.n_seq || x.s > end_s || (x.s == end_s && (x.hb > end_hb || (x.hb == end_hb && end_t == 0)));
  };
  auto enter = [&](Place &x) {
    x.end = 0;
    if (past(x)) return;
    x.len = cached_tokens(p, x.s, false);
    x.tiles = (x.len + kTile - 1) / kTile;
    x.head = blocks == 1 ? x.hb : x.hb / blocks;
    x.end = x.s == end_s && x.hb == end_hb ? end_t : x.tiles;
  };
  // The next sequence to visit, s or a later one. Of cut units the first with tokens, as far as the stretch
  // goes: a batch may be mostly empty (the unused slots of a captured step), and visiting 63 empty sequences beside
  // one of 4000 tokens (32/8 heads of 128) one by one took 534 us and not 14. Their rows are the join's. Of whole
  // units every one, an empty one's zeros among them.
  auto visit = [&](uint32_t s) {
    if (pl.units) return s;
    for (; s < p.n_seq && s <= end_s; s += 32) {
      const uint32_t some = __ballot_sync(0xffffffffu, s + lane < p.n_seq && p.lens[s + lane] > 0);
      if (some) return s + __ffs(some) - 1;
    }
    return p.n_seq;
  };
  auto next_of = [&](const Place &x) { return x.hb + 1 < pl.head_blocks ? x.s : visit(x.s + 1); };
  auto go_to = [&](Place &x, uint32_t s) {  // s = next_of(x)
    x.t = 0;
    x.hb = s == x.s ? x.hb + 1 : 0;
    x.s = s;
    enter(x);
  };
  Place ld = {static_cast<uint32_t>(found[warp][0]), static_cast<uint32_t>(found[warp][1]),
              static_cast<uint32_t>(found[warp][2]) + (pl.team ? rank * kWarps + warp : 0), 0, 0, 0, 0};
  enter(ld);
  Place at = ld;
  auto settle = [&] {  // to the next tile there is
    while (ld.t >= ld.end && !past(ld)) go_to(ld, next_of(ld));
  };
  settle();

  uint8_t *mine = smem + warp * R::kBytes;
  const uint32_t ring = smem_u32(mine);
  ulonglong2 *rows = reinterpret_cast<ulonglong2 *>(mine + R::kRowsOff);  // [kAhead][kTile]
  // The rows of the tile at `ld`, one for each of the first 16 lanes, and on to the next tile. What
  // it loads is first used in keep_rows, a tile's products later.
  ulonglong2 row = {0, 0};
  auto look_up = [&] {
    row = {0, 0};
    if (ld.t >= ld.end) return;
    const uint32_t j = ld.t * kTile + lane;
    if (lane < kTile && j < ld.len) {
      const uint32_t page = page_of(p.page, j);
      const int32_t id = __ldg(p.page_table + static_cast<int64_t>(ld.s) * p.table_stride + page);
      if (id < 0 || static_cast<uint32_t>(id) >= p.n_pages) {
        report(p.status, kErrPage);
      } else {
        const int64_t off = (static_cast<int64_t>(ld.head) * p.page.size + (j - page * p.page.size)) * kDim;
        row.x = reinterpret_cast<uint64_t>(p.k_cache + (id * p.k_page + off));
        row.y = reinterpret_cast<uint64_t>(p.v_cache + (id * p.v_page + off));
      }
    }
    ld.t += step;
    settle();
  };
  auto keep_rows = [&](uint32_t i) -> uint32_t {  // of tile i; returns which rows there are
    if (lane < kTile) rows[i % kAhead * kTile + lane] = row;
    return __ballot_sync(0xffffffffu, row.x != 0);
  };
  const uint32_t c = lane % kChunks, r0 = lane / kChunks;
  // Start tile i (rows `which`) into the stage at `kb`.
  auto load_tile = [&](uint32_t i, uint32_t which, uint32_t kb) {
    const ulonglong2 *from = rows + i % kAhead * kTile + r0;
    if (which == 0xffffu) {
#pragma unroll
      for (int n = 0; n < kTile / kRowsPass; ++n) {
        const uint32_t r = r0 + n * kRowsPass;
        const ulonglong2 a = from[n * kRowsPass];
        const uint32_t dst = kb + r * kDim * 2 + ((c ^ (r & 7)) * 16);
        cp_async16(dst, reinterpret_cast<const uint8_t *>(a.x) + c * 16);
        cp_async16(dst + kTileBytes, reinterpret_cast<const uint8_t *>(a.y) + c * 16);
      }
    } else if (which) {  // a last tile, or one with bad pages: absent rows are zeros
#pragma unroll 1
      for (int n = 0; n < kTile / kRowsPass; ++n) {
        const uint32_t r = r0 + n * kRowsPass;
        const ulonglong2 a = from[n * kRowsPass];
        const uint32_t dst = kb + r * kDim * 2 + ((c ^ (r & 7)) * 16);
        if (a.x) {
          cp_async16(dst, reinterpret_cast<const uint8_t *>(a.x) + c * 16);
          cp_async16(dst + kTileBytes, reinterpret_cast<const uint8_t *>(a.y) + c * 16);
        } else {
          sts_zero16(dst);
          sts_zero16(dst + kTileBytes);
        }
      }
    }
    cp_async_commit();
  };

  const uint32_t ra = lane / 4, cq = 2 * (lane % 4);
  const float c2 = p.scale * kLog2e;
  constexpr float kShift = weight_shift<kBf16>(0);
  // Q^T as the products' B operand: head lane / 4 of each 8, channels 2 (lane % 4) of each half step
  uint32_t q[kHeads8][kSteps][2], qn[kHeads8][kSteps][2];
  auto load_q = [&](uint32_t s, uint32_t hb) {
    const uint32_t head = blocks == 1 ? hb : hb / blocks, first = head * group + (hb - head * blocks) * 16;
#pragma unroll
    for (int n = 0; n < kHeads8; ++n) {
      const uint32_t h = first + 8 * n + ra;
      const bool in = s < p.n_seq && h < (head + 1) * group;
      const uint16_t *from = p.q + static_cast<int64_t>(s) * p.q_seq + static_cast<int64_t>(h) * p.q_head + cq;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        qn[n][k][0] = in ? __ldg(reinterpret_cast<const uint32_t *>(from + 16 * k)) : 0u;
        qn[n][k][1] = in ? __ldg(reinterpret_cast<const uint32_t *>(from + 16 * k + 8)) : 0u;
      }
    }
  };
  load_q(at.s, at.hb);
  uint32_t there[kStages + 1];  // rows of tile i, i + 1, ...
#pragma unroll
  for (int i = 0; i < kStages; ++i) {
    look_up();
    there[i] = keep_rows(i);
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load_tile(i, there[i], ring + i * 2 * kTileBytes);

  uint32_t i = 0;  // tiles done
  uint32_t kb = ring, lb = ring + (kStages - 1) * 2 * kTileBytes;  // stages of tile i, and of the one to load
  auto next_stage = [&](uint32_t x) {
    x += 2 * kTileBytes;
    return x == ring + kStages * 2 * kTileBytes ? ring : x;
  };
  for (uint32_t next = 0; !past(at); go_to(at, next)) {
    const uint32_t h0 = at.head * group + (at.hb - at.head * blocks) * 16;
    const uint32_t heads = min(16u, (at.head + 1) * group - h0);
    const bool whole = at.t == 0 && at.end == at.tiles;
    const uint32_t slot = i == 0 ? 0 : 1;                      // the stretch's first unit, or its last
    if (!pl.units && lane == 0 && at.t == 0 && at.tiles > 0) {
      // the warps after this one start within the unit and take `per` tiles of it each
      const uint32_t after = at.tiles - at.end;
      Share share = {static_cast<uint32_t>(warp0) + warp, 1 + static_cast<uint32_t>((after + per - 1) / per)};
      if (slot) share.parts |= kLastUnit;
      partials_of(p, pl).shares[static_cast<size_t>(at.s) * pl.head_blocks + at.hb] = share;
    }
    if (lane == 0 && at.hb == 0) cached_tokens(p, at.s, true);  // tells of a length past the table

#pragma unroll
    for (int n = 0; n < kHeads8; ++n)
#pragma unroll
      for (int k = 0; k < kSteps; ++k) q[n][k][0] = qn[n][k][0], q[n][k][1] = qn[n][k][1];
    if (!pl.team) {
      next = next_of(at);
      load_q(next, next == at.s ? at.hb + 1 : 0);
    }
    // O^T: channels 16 n + lane / 4 and 8 more, heads 2 (lane % 4) and the next
    float o[kHeads8][kSteps][4];
    float m[kHeads8][2], l[kHeads8][2];
#pragma unroll
    for (int h = 0; h < kHeads8; ++h) {
#pragma unroll
      for (int n = 0; n < kSteps; ++n) o[h][n][0] = o[h][n][1] = o[h][n][2] = o[h][n][3] = 0.f;
      m[h][0] = m[h][1] = -INFINITY;
      l[h][0] = l[h][1] = 0.f;
    }

    for (; at.t < at.end; at.t += step, ++i) {
      cp_async_wait<kStages - 2>();
      __syncwarp();  // tile i is in; tile i - 1's stage and the oldest addresses are free
      load_tile(i + kStages - 1, there[kStages - 1], lb);
      look_up();

      if (there[0]) {  // a tile without any row was not loaded
        const uint32_t vb = kb + kTileBytes;
        float sc[kHeads8][2][4];  // the even and the odd steps: shorter chains
#pragma unroll
        for (int h = 0; h < kHeads8; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[h][0][e] = sc[h][1][e] = 0.f;
        {
          const uint32_t r = lane % 16;  // key
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            uint32_t a[4];
            ldsm4(kb + r * kDim * 2 + (((2 * k + lane / 16) ^ (r & 7)) * 16), a);
#pragma unroll
            for (int h = 0; h < kHeads8; ++h) mma16816<kBf16>(sc[h][k & 1], a, q[h][k][0], q[h][k][1]);
          }
        }
        // keys lane / 4 and 8 more; the same heads as in O^T
        uint32_t w[kHeads8][2];
        float keep[kHeads8][2];
        bool moved = false;
#pragma unroll
        for (int h = 0; h < kHeads8; ++h) {
          float s4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) s4[e] = sc[h][0][e] + sc[h][1][e];
          if (there[0] != 0xffffu) {
            if (!(there[0] >> ra & 1)) s4[0] = s4[1] = -INFINITY;
            if (!(there[0] >> (ra + 8) & 1)) s4[2] = s4[3] = -INFINITY;
          }
          float p4[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s4[e], s4[2 + e]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(top, m[h][e]);
            // differences before the scale: a rounded top c2 may be off by more than the exponent's range
            const float from = top == -INFINITY ? 0.f : top;
            keep[h][e] = ex2_approx((m[h][e] - from) * c2);
            moved |= top != m[h][e];
            m[h][e] = top;
            p4[e] = ex2_approx(fmaf(s4[e] - from, c2, kShift));
            p4[2 + e] = ex2_approx(fmaf(s4[2 + e] - from, c2, kShift));
            l[h][e] = fmaf(l[h][e], keep[h][e], p4[e] + p4[2 + e]);
          }
          w[h][0] = transposed(Elem<kBf16>::pack(p4[0], p4[1]));
          w[h][1] = transposed(Elem<kBf16>::pack(p4[2], p4[3]));
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int h = 0; h < kHeads8; ++h)
#pragma unroll
            for (int n = 0; n < kSteps; ++n) {
              o[h][n][0] *= keep[h][0];
              o[h][n][1] *= keep[h][1];
              o[h][n][2] *= keep[h][0];
              o[h][n][3] *= keep[h][1];
            }
        }
        {
          const uint32_t r = (lane / 16) * 8 + lane % 8;  // key
#pragma unroll
          for (int n = 0; n < kSteps; ++n) {
            uint32_t a[4];
            ldsm4t(vb + r * kDim * 2 + (((2 * n + (lane / 8 & 1)) ^ (r & 7)) * 16), a);
#pragma unroll
            for (int h = 0; h < kHeads8; ++h) mma16816<kBf16>(o[h][n], a, w[h][0], w[h][1]);
          }
        }
      }
      kb = next_stage(kb);
      lb = next_stage(lb);
      there[kStages] = keep_rows(i + kStages);
#pragma unroll
      for (int n = 0; n < kStages; ++n) there[n] = there[n + 1];
    }

    // The unit's end.
#pragma unroll
    for (int h = 0; h < kHeads8; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], 4);
        l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], 8);
        l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], 16);
      }
    if (pl.team) {  // meet in the rings' memory; every warp comes here once
      cp_async_wait<0>();
      __syncthreads();
      float *to = reinterpret_cast<float *>(smem);                          // [kWarps][16][kDim]
      float2 *ml = reinterpret_cast<float2 *>(to + kWarps * 16 * kDim);     // [kWarps][16]
      static_assert(kWarps * 16 * (kDim * 4 + 8) <= kWarps * R::kBytes, "the rings hold the outputs");
#pragma unroll
      for (int h = 0; h < kHeads8; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t r = warp * 16 + 8 * h + cq + e;
          if (ra == 0) ml[r] = make_float2(m[h][e], l[h][e]);
#pragma unroll
          for (int n = 0; n < kSteps; ++n) {
            to[r * kDim + 16 * n + ra] = o[h][n][e];
            to[r * kDim + 16 * n + ra + 8] = o[h][n][2 + e];
          }
        }
      auto join = [&](auto many) {
        // a partial result of the cluster's CTA c
        auto part_of = [&](const void *here, uint32_t c) {
          if constexpr (decltype(many)::value)
            return load_cta(in_cta(smem_u32(here), c));
          else
            return *static_cast<const float2 *>(here);
        };
        const uint32_t ctas = decltype(many)::value ? pl.cluster : 1;
        constexpr uint32_t kPairs = kDim / 2;
        for (uint32_t x = rank * kThreads + tid; x < heads * kPairs; x += ctas * kThreads) {
          const uint32_t r = x / kPairs, d = x % kPairs * 2;
          float top = -INFINITY, sum = 0.f, a = 0.f, b = 0.f;
#pragma unroll 2
          for (uint32_t c = 0; c < ctas; ++c)
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_of(ml + w * 16 + r, c).x);
#pragma unroll 2
          for (uint32_t c = 0; c < ctas; ++c)
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              const float2 part = part_of(ml + w * 16 + r, c), v = part_of(to + (w * 16 + r) * kDim + d, c);
              const float f = top == -INFINITY ? 1.f : ex2_approx((part.x - top) * c2);
              sum = fmaf(part.y, f, sum);
              a = fmaf(v.x, f, a);
              b = fmaf(v.y, f, b);
            }
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          *reinterpret_cast<uint32_t *>(p.out + static_cast<int64_t>(at.s) * p.out_seq + (h0 + r) * p.out_head + d) =
              Elem<kBf16>::pack(a * inv, b * inv);
          if (p.lse && d == 0) p.lse[static_cast<int64_t>(at.s) * p.q_heads + h0 + r] = log_sum<kBf16>(top * c2, sum, 0);
        }
      };
      if (pl.cluster > 1) {
        cluster_sync();
        join(std::true_type{});
        cluster_sync();  // the others have read this CTA's shared memory
      } else {
        __syncthreads();
        join(std::false_type{});
      }
      break;
    }
    if (whole) {
#pragma unroll
      for (int h = 0; h < kHeads8; ++h) {
        float inv[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          inv[e] = l[h][e] == 0.f ? 0.f : 1.f / l[h][e];
          if (p.lse && ra == 0 && 8 * h + cq + e < heads)
            p.lse[static_cast<int64_t>(at.s) * p.q_heads + h0 + 8 * h + cq + e] = log_sum<kBf16>(m[h][e] * c2, l[h][e], 0);
        }
        uint16_t *dst = p.out + static_cast<int64_t>(at.s) * p.out_seq + (h0 + 8 * h + ra) * p.out_head + cq;
#pragma unroll
        for (int n = 0; n < kSteps; ++n) {
          const uint32_t lo = transposed(Elem<kBf16>::pack(o[h][n][0] * inv[0], o[h][n][1] * inv[1]));
          const uint32_t hi = transposed(Elem<kBf16>::pack(o[h][n][2] * inv[0], o[h][n][3] * inv[1]));
          if (8 * h + ra < heads) {
            *reinterpret_cast<uint32_t *>(dst + 16 * n) = lo;
            *reinterpret_cast<uint32_t *>(dst + 16 * n + 8) = hi;
          }
        }
      }
    } else {
      const Partials part = partials_of(p, pl);
#pragma unroll
      for (int h = 0; h < kHeads8; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t r = 8 * h + cq + e;
          if (r >= heads) continue;
          const size_t to = ((warp0 + warp) * 2 + slot) * pl.rows + r;
          if (ra == 0) part.ml[to] = make_float2(m[h][e], l[h][e]);
#pragma unroll
          for (int n = 0; n < kSteps; ++n) {
            part.o[to * kDim + 16 * n + ra] = o[h][n][e];
            part.o[to * kDim + 16 * n + ra + 8] = o[h][n][2 + e];
          }
        }
    }
  }
  cp_async_wait<0>();
}

// Joins the units that several stretches share: out = sum_i f_i o_i / sum_i f_i l_i, f_i =
// 2^(c (m_i - M)), over the stretches i in order; and writes the rows of empty sequences. kJoin warps take every kJoin-th
// part of a (sequence, query head), then meet in shared memory: 4 where units have few parts, 32
// where they have more than 16 (4 warps took 20 us for 148 parts; 32, or a single one, 2 to 4 us
// more than 4 for the few parts of 64 sequences of 1..4096 tokens). What a unit's parts are the first
// launch has left in the workspace: summing the lengths before s again, as it was, kept the join's
// loads waiting (42.0 us in all for those 64 sequences; 39.6 so).
template <bool kBf16, int kDim, int kJoin>
__global__ void __launch_bounds__(kJoin * 32)
    attention_paged_join_kernel(const PagedAttention p, const Plan pl) {
  constexpr int kLane = kDim / 32;  // channels per lane
  __shared__ float po[kJoin][kDim];
  __shared__ float ps[kJoin];
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = blockIdx.x;
  const uint32_t s = row / p.q_heads, h = row % p.q_heads;
  const uint32_t group = p.q_heads / p.kv_heads, blocks = pl.head_blocks / p.kv_heads;
  const uint32_t hb = h / group * blocks + h % group / 16, r = h % group % 16;
  pdl_wait();
  pdl_trigger();
  const float c2 = p.scale * kLog2e;
  const Partials w = partials_of(p, pl);
  Share share = w.shares[static_cast<size_t>(s) * pl.head_blocks + hb];  // of an empty one: not read
  if (cached_tokens(p, s, false) == 0) share = {0, 0};
  const uint32_t n = share.parts & ~kLastUnit;
  if (n == 1) return;  // one warp's: written
  auto slot_of = [&](uint32_t i) {
    return ((static_cast<size_t>(share.first) + i) * 2 + (i == 0 && share.parts != n)) * pl.rows + r;
  };
  // The first of this warp's parts on their way under the search for the largest maximum.
  constexpr int kEarly = 4;
  float2 ml[kEarly];
  float v[kEarly][kLane];
  auto load = [&](uint32_t i, float2 &x, float(&o)[kLane]) {
    const size_t at = slot_of(i);
    x = w.ml[at];
#pragma unroll
    for (int e = 0; e < kLane; e += 2) {
      const float2 y = *reinterpret_cast<const float2 *>(w.o + at * kDim + lane * kLane + e);
      o[e] = y.x;
      o[e + 1] = y.y;
    }
  };
#pragma unroll
  for (int k = 0; k < kEarly; ++k)
    if (warp + k * kJoin < n) load(warp + k * kJoin, ml[k], v[k]);
  float top = -INFINITY;
  for (uint32_t i = lane; i < n; i += 32) top = fmaxf(top, w.ml[slot_of(i)].x);
#pragma unroll
  for (int i = 16; i > 0; i /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
  float sum = 0.f, acc[kLane] = {};
  auto add = [&](const float2 &x, const float(&o)[kLane]) {
    const float f = top == -INFINITY ? 1.f : ex2_approx((x.x - top) * c2);
    sum = fmaf(x.y, f, sum);
#pragma unroll
    for (int e = 0; e < kLane; ++e) acc[e] = fmaf(o[e], f, acc[e]);
  };
#pragma unroll
  for (int k = 0; k < kEarly; ++k)
    if (warp + k * kJoin < n) add(ml[k], v[k]);
#pragma unroll 4
  for (uint32_t i = warp + kEarly * kJoin; i < n; i += kJoin) {
    load(i, ml[0], v[0]);
    add(ml[0], v[0]);
  }
#pragma unroll
  for (int e = 0; e < kLane; ++e) po[warp][lane * kLane + e] = acc[e];
  if (lane == 0) ps[warp] = sum;
  __syncthreads();
  if (warp > 0) return;
  sum = 0.f;
#pragma unroll
  for (int e = 0; e < kLane; ++e) acc[e] = 0.f;
#pragma unroll 8
  for (int i = 0; i < kJoin; ++i) {
    sum += ps[i];
#pragma unroll
    for (int e = 0; e < kLane; ++e) acc[e] += po[i][lane * kLane + e];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t *dst = p.out + static_cast<int64_t>(s) * p.out_seq + h * p.out_head + lane * kLane;
#pragma unroll
  for (int e = 0; e < kLane; e += 2)
    *reinterpret_cast<uint32_t *>(dst + e) = Elem<kBf16>::pack(acc[e] * inv, acc[e + 1] * inv);
  if (p.lse && lane == 0) p.lse[row] = log_sum<kBf16>(top * c2, sum, 0);
}

namespace {
size_t workspace_of(const PagedAttention &p, const Plan &pl) {
  const size_t n = (static_cast<size_t>(pl.grid) * kWarps * 2 * pl.rows + 1) / 2 * 2;
  return shares_bytes(p, pl) + n * (p.head_dim + 2) * sizeof(float);
}
}  // namespace

size_t attention_paged_workspace(const PagedAttention &p) {
  const Plan pl = plan_of(p);
  return pl.units ? 0 : workspace_of(p, pl);
}

size_t attention_paged_workspace_bound(const PagedAttention &p) {
  Plan pl = plan_of(p);
  pl.grid = cta_slots(p);  // of any plan at most, and the shares grow with the sequences
  return workspace_of(p, pl);
}

namespace {
template <bool kBf16, int kDim, int kHeads8>
cudaError_t launch(const PagedAttention &p, const Plan &pl, cudaStream_t stream) {
  static std::atomic<bool> configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev].load(std::memory_order_acquire)) {
    // setting the attribute twice (two threads racing here) is harmless
    const cudaError_t e = cudaFuncSetAttribute(attention_paged_kernel<kBf16, kDim, kHeads8>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kWarps * Ring<kDim>::kBytes);
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {pl.cluster, 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kWarps * Ring<kDim>::kBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pl.cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, attention_paged_kernel<kBf16, kDim, kHeads8>, p, pl);
  if (e != cudaSuccess || pl.units) return e;
  const uint32_t rows = p.n_seq * p.q_heads;  // below 2^31
  return pl.crowd ? launch_pdl(attention_paged_join_kernel<kBf16, kDim, 32>, dim3(rows), dim3(1024), 0, stream, p, pl)
                  : launch_pdl(attention_paged_join_kernel<kBf16, kDim, 4>, dim3(rows), dim3(128), 0, stream, p, pl);
}
}  // namespace

cudaError_t launch_attention_paged(const PagedAttention &p, bool bf16, cudaStream_t stream) {
  if (p.n_seq == 0) return cudaSuccess;
  const Plan pl = plan_of(p);
  auto run = [&](auto b, auto dim) {
    return pl.rows <= 8 ? launch<decltype(b)::value, decltype(dim)::value, 1>(p, pl, stream)
                        : launch<decltype(b)::value, decltype(dim)::value, 2>(p, pl, stream);
  };
  using std::integral_constant;
  if (p.head_dim == 64)
    return bf16 ? run(std::true_type{}, integral_constant<int, 64>{}) : run(std::false_type{}, integral_constant<int, 64>{});
  return bf16 ? run(std::true_type{}, integral_constant<int, 128>{}) : run(std::false_type{}, integral_constant<int, 128>{});
}

}  // namespace dv3
