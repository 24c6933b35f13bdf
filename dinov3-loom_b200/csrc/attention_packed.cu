// attention_packed.cu - attention over packed sequences of different lengths, grouped heads, full
// or causal, on tcgen05 tensor cores.
//
// For query row i of a sequence with a queries and b keys, and query head h reading key-value head
// h / (q_heads / kv_heads): o = sum_j w_j v_j / sum_j w_j, w_j = exp(scale (q . k_j - max)), over
// the keys j < b, and j <= i + b - a where causal (the last query sees the last key). A row that
// sees no key gives 0 (and -inf as its log-sum).
//
// Tiles. A 128-row query tile holds 128 / group tokens with all `group` query heads that read one
// key-value head (one TMA box of group heads x tokens), so grouped heads share every K and V tile
// and a short sequence still fills its rows; a work item is two such tiles of one sequence and
// key-value head against that sequence's visible keys, 128 at a time. Persistent CTAs, one per
// SM, walk the items longest first (below).
//
// Roles (384 threads):
//   warps 0-3  softmax and output of tile 0, warps 4-7 of tile 1: one query row per thread (its
//              TMEM lane). All 128 scores of a step are held in registers: running maximum, w =
//              2^(s c - m c) with c = scale log2(e), f32 sum of the unrounded weights, P (rounded to
//              the element type) back to TMEM over the consumed scores. The reference m only moves
//              when the maximum has grown by more than 2^8 over it: any m gives the same quotient,
//              and sums and weights up to 2^8 too large lose nothing in f32, f16 or bf16; the row's
//              output is then rescaled in TMEM. At an item's end O / sum goes through a staging
//              tile to global memory. Of a last, partly visible step only the blocks of 32 keys
//              that some row sees are computed.
//   warp 8     TMA producer: Q tiles, then K and V tiles in turn through one ring of stages.
//   warps 9/10 MMA issuers of tile 0 / tile 1: S_t = Q_t K^T (M = N = 128), and O_t += P_t V with P
//              from TMEM and V as the MN-major B operand, one tile at a time.
//   warp 11    scheduler (publishes items one ahead), and guard of V: a key that a row does not see has weight 0, but 0 times
//              an infinity or NaN is NaN. Only the tiles at an item's end (from the first that some
//              row sees in part) can hold such keys; there it tests V in shared memory, sets what
//              is not finite to 0 and leaves a note, and the rows that do see those keys add them
//              at the end from global memory.
// TMEM: S_0 | S_1 | O_0 | O_1, 128 columns each.
//
// Every wait is bounded; on a timeout the kernel records kErrAttentionWait, raises the CTA's
// abort flag, lets its own copies and MMAs in flight land, frees TMEM and returns.
#include <atomic>

#include "sequence.cuh"

namespace dv3 {

namespace {
constexpr int kThreads = 384;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;  // TMEM allocator; issues tile 0's MMAs, warp 10 tile 1's
constexpr int kGuardWarp = 11;
constexpr int kKeys = 128;      // keys per step
constexpr int kBuckets = 64;    // of the scheduler's order
constexpr int kTmemCols = 512;
constexpr int kTmemO = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.f;   // log2 units by which a row's maximum may pass its reference

// One work item as the scheduler publishes it (two 16-byte words).
struct __align__(16) Item {
  int32_t q_row;    // first query row
  int32_t q_count;  // its tokens (0: nothing to do)
  int32_t k_row;    // first key row of the sequence
  int32_t k_len;
  int32_t visible;  // keys the first token sees, less than 1 if none; a later one sees one more if causal
  int32_t head;     // key-value head
  int32_t last;     // 1: no more items
  int32_t fix;      // set by the guard: V held something that is not finite
};

__device__ __forceinline__ Item read_item(const Item *slot) {
  Item it;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(it.q_row), "=r"(it.q_count), "=r"(it.k_row), "=r"(it.k_len)
               : "r"(smem_u32(slot))
               : "memory");
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(it.visible), "=r"(it.head), "=r"(it.last), "=r"(it.fix)
               : "r"(smem_u32(slot) + 16)
               : "memory");
  return it;
}

template <int kDim>
struct Layout {
  static constexpr int kHalves = kDim / 64;         // 64-channel (128-byte) columns of a tile
  static constexpr int kHalfBytes = 128 * 128;      // 128 rows of one
  static constexpr int kTileBytes = kHalves * kHalfBytes;
  static constexpr int kStages = kDim == 128 ? 4 : 6;
  static constexpr int kRingOff = 2 * kTileBytes;   // Q_0 | Q_1 | stages | output staging
  static constexpr int kOutOff = kRingOff + kStages * kTileBytes;
  static constexpr int kOutBytes = 32 * 128;        // a softmax warp's: 32 rows of 64 channels
  static constexpr int kBarOff = kOutOff + 8 * kOutBytes;
  // barriers: q_full[2] q_empty[2] s_full[2] p_full[4] (first halves, second halves) o_full[2]
  // drain[2] sched_full[3] sched_empty[3] kv_full[stages] kv_empty[stages] v_ok[stages] (by V tile, not by stage: a stage
  // of an odd ring holds K and V in turn)
  static constexpr int kBars = 20 + 3 * kStages;
  static constexpr int kItemOff = (kBarOff + kBars * 8 + 15) / 16 * 16;
  static constexpr int kMiscOff = kItemOff + 3 * static_cast<int>(sizeof(Item));  // TMEM slot, abort, turn
  static constexpr int kOrderOff = kMiscOff + 16;
  static constexpr int kBytes = 1024 + kOrderOff + (kBuckets + 1) * 4;
  static_assert(kBytes <= 227 * 1024, "shared memory budget");
};

// Instruction descriptor with the element type (see idesc_f16_f32): bf16 is format 1.
__host__ __device__ constexpr uint32_t idesc_f32(bool bf16, uint32_t m, uint32_t n, bool b_mn_major) {
  return idesc_f16_f32(m, n, b_mn_major) | (bf16 ? (1u << 7) | (1u << 10) : 0u);
}
// MN-major 128-byte-swizzle tile whose 64-element columns lie `column_bytes` apart (the leading
// byte offset); 8-row groups of K are 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t smem_addr, uint32_t column_bytes) {
  return (sw128_desc(smem_addr) & ~(0x3FFFull << 16)) | (static_cast<uint64_t>(column_bytes >> 4) << 16);
}

// Two f32 at once (Blackwell's packed f32 operations, one issue slot for both).
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  return pair(__float_as_uint(lo), __float_as_uint(hi));
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  uint32_t lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
  return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Registers of a warpgroup: the kernel starts with 168 a thread (384 x 168 = 64512); the softmax
// warps hold a step's 128 scores and take 216, the other four keep 72 (256 x 216 + 128 x 72 = 64512).
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 216;"); }
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The items stand in an order that ends evenly: most visible keys first, in kBuckets classes of
// `width` keys; by sequence within a class, later items of a sequence first.
struct Order {
  uint32_t *starts;  // first item of each class, top class first; [kBuckets]
  uint32_t total;    // items
  uint32_t width;
  // where the last search stood
  int bucket;
  uint32_t seq, before;
};
}  // namespace

struct PackedArgs {
  const uint16_t *v;
  uint16_t *out;
  float *lse;
  const int32_t *cu_q, *cu_k;
  int64_t v_token, v_head, out_token, out_head;
  uint32_t *status;
  uint32_t n_seq, total_q, total_k, q_heads, kv_heads, group;
  uint32_t tokens;  // per tile
  PageDiv item;     // division by an item's 2 tokens
  uint32_t boxed;   // 32 rows of a tile are whole tokens: one TMA box of the output
  bool causal;
  float scale_log2;
};

namespace {
// A sequence as the scheduler sees it: `n` items of 2 p.tokens query tokens for one key-value head.
struct Sequence {
  uint32_t q0, a, k0, b, n;  // first rows, lengths
};
__device__ __forceinline__ Sequence sequence_of(const PackedArgs &p, uint32_t s) {
  Sequence x;
  uint32_t q1, k1;
  sequence_rows(p.cu_q, s, p.total_q, &x.q0, &q1);
  sequence_rows(p.cu_k, s, p.total_k, &x.k0, &k1);
  x.a = q1 - x.q0;
  x.b = k1 - x.k0;
  x.n = page_of(p.item, x.a + 2 * p.tokens - 1);
  return x;
}
// Items of the sequence whose last token sees more than `keys` keys: the last so many.
__device__ __forceinline__ uint32_t items_above(const PackedArgs &p, const Sequence &x, uint32_t keys) {
  if (x.n == 0 || x.b <= keys) return 0;
  if (!p.causal) return x.n;
  // item l's last token sees b - a + min(a, (l + 1) 2 tokens) of them
  const int32_t beyond = static_cast<int32_t>(keys - x.b + x.a);
  const uint32_t first = beyond < 0 ? 0u : page_of(p.item, static_cast<uint32_t>(beyond));
  return x.n - min(first, x.n - 1);
}
// Items of the sequence in class c (`width` keys each; the lowest also holds those that see none).
__device__ __forceinline__ uint32_t items_in(const PackedArgs &p, const Sequence &x, uint32_t c, uint32_t width) {
  return (c == 0 ? x.n : items_above(p, x, c * width)) - items_above(p, x, (c + 1) * width);
}

// Item `index` in the order, for key-value head `head`; whole warp.
__device__ __forceinline__ Item find_item(const PackedArgs &p, Order &o, uint32_t index, uint32_t head) {
  const uint32_t lane = threadIdx.x & 31u;
  Item it = {};
  it.head = static_cast<int32_t>(head);
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < kBuckets / 32; ++i) mine += o.starts[lane * (kBuckets / 32) + i] <= index;
  const int at = static_cast<int>(__reduce_add_sync(0xffffffffu, mine)) - 1;
  const uint32_t rest = index - o.starts[at], c = kBuckets - 1 - at;
  if (at != o.bucket || rest < o.before) {
    o.bucket = at;
    o.seq = 0;
    o.before = 0;
  }
  for (; o.seq < p.n_seq; o.seq += 32) {
    const uint32_t s = o.seq + lane;
    Sequence x = {};
    if (s < p.n_seq) x = sequence_of(p, s);
    const uint32_t count = items_in(p, x, c, o.width);
    uint32_t sum = count;
#pragma unroll
    for (int i = 1; i < 32; i *= 2) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, sum, i);
      if (lane >= static_cast<uint32_t>(i)) sum += y;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, rest < o.before + sum);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const uint32_t within = rest - (o.before + sum - count);  // of this lane's sequence
      const uint32_t t0 = (x.n - items_above(p, x, (c + 1) * o.width) - 1 - within) * 2 * p.tokens;
      it.q_row = static_cast<int32_t>(__shfl_sync(0xffffffffu, x.q0 + t0, src));
      it.q_count = static_cast<int32_t>(__shfl_sync(0xffffffffu, min(x.a - t0, 2 * p.tokens), src));
      it.k_row = static_cast<int32_t>(__shfl_sync(0xffffffffu, x.k0, src));
      it.k_len = static_cast<int32_t>(__shfl_sync(0xffffffffu, x.b, src));
      it.visible = static_cast<int32_t>(__shfl_sync(0xffffffffu, p.causal ? x.b - x.a + t0 + 1 : x.b, src));
      return it;
    }
    o.before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return it;  // not reached while cu is ascending
}

// What a tile's rows see.
struct Reach {
  int steps;  // of 128 keys
  int first;  // keys that its first token sees (at least 0)
  int most;   // keys that its last token sees
};
// Blocks of 32 keys in step j that some row of the tile sees.
__device__ __forceinline__ int blocks_of(const Reach &r, int j) {
  return min(kKeys / 32, (r.most - j * kKeys + 31) / 32);
}
__device__ __forceinline__ Reach reach_of(const Item &it, int tile, int tokens, bool causal) {
  const int begin = tile * tokens, end = min(it.q_count, begin + tokens);
  Reach r = {0, 0, 0};
  if (begin >= end) return r;
  r.most = causal ? min(it.k_len, it.visible + end - 1) : it.k_len;
  r.first = max(0, causal ? min(it.k_len, it.visible + begin) : it.k_len);
  r.steps = r.most > 0 ? (r.most + kKeys - 1) / kKeys : 0;
  return r;
}

// Whether 16 bytes of 16-bit floats are all finite: x * 0 summed is NaN otherwise.
template <bool kBf16>
__device__ __forceinline__ uint32_t times_zero(uint32_t x, uint32_t acc) {
  if constexpr (kBf16)
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(x), "r"(0u));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(x), "r"(0u));
  return acc;
}
template <bool kBf16>
__device__ __forceinline__ bool finite16(uint32_t half) {
  const uint32_t e = kBf16 ? 0x7f80u : 0x7c00u;
  return (half & e) != e;
}

// A row's reference, moved to the step's maximum `now` (log2 units) where that passes it by more than
// kSlack; the row's sum and output so far follow. The previous product is done: the thread that
// issued it issued these scores after it.
__device__ __forceinline__ void move_reference(uint32_t to, int dim, float now, bool first, float &m,
                                               float &sum) {
  if (first) {
    m = now;
    return;
  }
  const bool grown = now > m + kSlack;
  if (!__any_sync(0xffffffffu, grown)) return;
  const float next = grown ? now : m;
  const float f = grown ? ex2_approx(m - next) : 1.f;
  sum *= f;
  m = next;
#pragma unroll 1
  for (int d = 0; d < dim; d += 16) {
    uint32_t x[16];
    tmem_ld16(to + d, x);
    tmem_ld_wait();
    tmem_regs_ready16(x);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
    tmem_st16(to + d, x);
  }
}

// The weights of 32 scores, 2^(s c - base), stored over consumed scores and added to (s0, s1).
template <bool kBf16>
__device__ __forceinline__ void weigh(uint32_t to, const uint32_t (&v)[32], uint64_t c2,
                                      uint64_t base2, uint64_t &s0, uint64_t &s1) {
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float2 x = unpair(fma2(pair(v[2 * e], v[2 * e + 1]), c2, base2));
    const uint64_t w2 = pair(ex2_approx(x.x), ex2_approx(x.y));
    if (e & 1)
      s1 = add2(s1, w2);
    else
      s0 = add2(s0, w2);
    const float2 f = unpair(w2);
    w[e] = Elem<kBf16>::pack(f.x, f.y);
  }
  tmem_st16(to, w);
}

__device__ __forceinline__ void hand_over_weights(uint64_t *p_full) {
  tmem_st_wait();
  tc_fence_before();
  __syncwarp();
  if (threadIdx.x % 32 == 0) mbar_arrive(p_full);
}

// Scores, weights and sums of one step for this thread's row, through m (reference, log2 units) and
// sum. Where some row sees the step in part (kMasked), this one sees `vis` keys of it and the tile
// `blocks` blocks of 32; the products skip the others. The weights are handed over in two halves
// (p_full[0], p_full[2]), so that the product with V starts under the second.
template <bool kBf16, bool kMasked>
__device__ __forceinline__ void softmax_step(uint32_t tl, uint32_t to, int dim, float c, int vis,
                                             int blocks, bool first, float &m, float &sum,
                                             uint64_t *p_full) {
  uint32_t v[4][32];
#pragma unroll
  for (int i = 0; i < 4; ++i) tmem_ld32(tl + 32 * i, v[i]);  // past `blocks`: old values, not used
  tmem_wait_ld(v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) tmem_regs_ready(v[i]);
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (kMasked && i >= blocks) break;
    if constexpr (kMasked) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (32 * i + e >= vis) v[i][e] = 0xff800000u;  // -inf
    }
#pragma unroll
    for (int e = 0; e < 32; e += 2)
      top[i] = max3(top[i], __uint_as_float(v[i][e]), __uint_as_float(v[i][e + 1]));
  }
  move_reference(to, dim, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c, first, m, sum);
  const float base = m == -INFINITY ? 0.f : m;
  const uint64_t c2 = pair(c, c), base2 = pair(-base, -base);
  uint64_t s0 = 0, s1 = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!kMasked || i < blocks) weigh<kBf16>(tl + 16 * i, v[i], c2, base2, s0, s1);
    if (i & 1) hand_over_weights(p_full + i - 1);
  }
  const float2 part = unpair(add2(s0, s1));
  sum += part.x + part.y;
}
}  // namespace

template <bool kBf16, int kDim>
__global__ void __launch_bounds__(kThreads, 1)
    attention_packed_kernel(const __grid_constant__ CUtensorMap tmq,
                            const __grid_constant__ CUtensorMap tmk,
                            const __grid_constant__ CUtensorMap tmv,
                            const __grid_constant__ CUtensorMap tmo,
                            const __grid_constant__ PackedArgs p) {
  using L = Layout<kDim>;
  constexpr int kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t *q_full = reinterpret_cast<uint64_t *>(smem + L::kBarOff);
  uint64_t *q_empty = q_full + 2, *s_full = q_full + 4, *p_full = q_full + 6, *o_full = q_full + 10;
  uint64_t *drain = q_full + 12, *sched_full = q_full + 14, *sched_empty = q_full + 17;
  uint64_t *kv_full = q_full + 20, *kv_empty = kv_full + kStages, *v_ok = kv_empty + kStages;
  Item *items = reinterpret_cast<Item *>(smem + L::kItemOff);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::kMiscOff);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  uint32_t *turn = tmem_slot + 2;
  uint32_t *order = reinterpret_cast<uint32_t *>(smem + L::kOrderOff);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);  // the tile's softmax warps
      mbar_init(&p_full[2 + i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&drain[i], 1);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&sched_full[i], 1);
      mbar_init(&sched_empty[i], 8 + 3);  // softmax warps, producer, issuers
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 2);  // both tiles
      mbar_init(&v_ok[i], 1);
    }
    *abort_flag = 0;
    *turn = 0;
    fence_mbar_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_map(&tmq);
    tma_prefetch_map(&tmk);
    tma_prefetch_map(&tmv);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  for (int i = threadIdx.x; i <= kBuckets; i += kThreads) order[i] = 0;
  __syncthreads();
  // The longest sequence sets the classes' width; then each sequence's items in them.
  uint32_t longest = 0;
  for (uint32_t s = threadIdx.x; s < p.n_seq; s += kThreads) {
    const Sequence x = sequence_of(p, s);
    if (x.n) longest = max(longest, x.b);
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 0) atomicMax(&order[kBuckets], longest);
  __syncthreads();
  const uint32_t width = max(1u, (order[kBuckets] + kBuckets - 1) / kBuckets);
  // Few sequences: a warp for each, the classes over its lanes; else a thread, over its own classes.
  if (p.n_seq <= 96) {
    for (uint32_t s = warp; s < p.n_seq; s += kThreads / 32) {
      const Sequence x = sequence_of(p, s);
#pragma unroll
      for (int i = lane; i < kBuckets; i += 32)
        if (const uint32_t n = items_in(p, x, i, width)) atomicAdd(&order[kBuckets - 1 - i], n);
    }
  } else {
    for (uint32_t s = threadIdx.x; s < p.n_seq; s += kThreads) {
      const Sequence x = sequence_of(p, s);
      uint32_t left = x.n;
      for (int i = min(kBuckets - 1, static_cast<int>(x.b ? (x.b - 1) / width : 0)); left > 0; --i) {
        const uint32_t n = items_in(p, x, i, width);
        if (n) atomicAdd(&order[kBuckets - 1 - i], n);
        left = i > 0 ? left - n : 0;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int tokens = static_cast<int>(p.tokens);

  if (warp == kGuardWarp) {
    fewer_registers();
    Order o = {order, 0, width, -1, 0, 0};
    {  // counts to starts
      const uint32_t n0 = order[2 * lane], n1 = order[2 * lane + 1];
      static_assert(kBuckets == 64, "two classes a lane");
      uint32_t sum = n0 + n1;
#pragma unroll
      for (int i = 1; i < 32; i *= 2) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, sum, i);
        if (lane >= i) sum += x;
      }
      o.total = __shfl_sync(0xffffffffu, sum, 31);
      __syncwarp();
      order[2 * lane] = sum - n0 - n1;
      order[2 * lane + 1] = sum - n1;
      __syncwarp();
    }
    const uint64_t n_items = static_cast<uint64_t>(o.total) * p.kv_heads;
    bool ok = true;
    // Publish item k of this CTA: up the order and down again in turn, so that no CTA always gets
    // the longest of each round.
    auto publish = [&](uint32_t k) {
      const uint64_t at = static_cast<uint64_t>(k) * gridDim.x +
                          (k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      Item it = {};
      if (at < n_items)
        it = find_item(p, o, static_cast<uint32_t>(at / p.kv_heads), static_cast<uint32_t>(at % p.kv_heads));
      // the up-and-down order may leave one CTA an item in a round in which others have none
      it.last = static_cast<uint64_t>(k) * gridDim.x >= n_items;
      ok = __all_sync(0xffffffffu, mbar_wait(&sched_empty[k % 3], ((k / 3) & 1) ^ 1u, abort_flag));
      if (ok && lane == 0) {
        volatile Item *d = &items[k % 3];
        d->q_row = it.q_row;
        d->q_count = it.q_count;
        d->k_row = it.k_row;
        d->k_len = it.k_len;
        d->visible = it.visible;
        d->head = it.head;
        d->last = it.last;
        d->fix = 0;
        mbar_arrive(&sched_full[k % 3]);
      }
      return it;
    };
    if (!ok && lane == 0) {
      report(p.status, kErrAttentionWait);
      *abort_flag = 1;
    }
    uint32_t ring = 0, phase = 0, v_ring = 0;
    Item it = publish(0);
    for (uint32_t k = 0; ok && !it.last; ++k) {
      const Item next = publish(k + 1);
      if (!ok) break;
      const Reach r0 = reach_of(it, 0, tokens, p.causal), r1 = reach_of(it, 1, tokens, p.causal);
      const int steps = max(r0.steps, r1.steps), partial = r0.first / kKeys;
      for (int j = 0; j < steps; ++j) {
        if (++ring == kStages) ring = 0, phase ^= 1;  // the step's K stage
        ok = __all_sync(0xffffffffu, mbar_wait(&kv_full[ring], phase, abort_flag));
        if (!ok) break;
        if (j >= partial) {
          uint4 *x = reinterpret_cast<uint4 *>(smem + L::kRingOff + ring * L::kTileBytes);
          uint32_t acc = 0;
#pragma unroll 8
          for (int i = lane; i < L::kTileBytes / 16; i += 32) {
            const uint4 w = x[i];
            acc = times_zero<kBf16>(w.x, acc);
            acc = times_zero<kBf16>(w.y, acc);
            acc = times_zero<kBf16>(w.z, acc);
            acc = times_zero<kBf16>(w.w, acc);
          }
          if (__any_sync(0xffffffffu, !finite16<kBf16>(acc & 0xffffu) || !finite16<kBf16>(acc >> 16))) {
            for (int i = lane; i < L::kTileBytes / 16; i += 32) {
              uint4 w = x[i];
              uint32_t *u = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (!finite16<kBf16>(u[e] & 0xffffu)) u[e] &= 0xffff0000u;
                if (!finite16<kBf16>(u[e] >> 16)) u[e] &= 0x0000ffffu;
              }
              x[i] = w;
            }
            *reinterpret_cast<volatile int32_t *>(&items[k % 3].fix) = 1;
            fence_proxy_async_smem();
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ok[v_ring]);
        if (++v_ring == kStages) v_ring = 0;
        if (++ring == kStages) ring = 0, phase ^= 1;
      }
      it = next;
    }
    if (!ok && lane == 0) {
      report(p.status, kErrAttentionWait);
      *abort_flag = 1;
    }
  } else if (warp == kProducerWarp) {
    fewer_registers();
    if (lane == 0) {
      uint32_t ring = 0, phase = 0, armed = 0, parity = 0;
      uint32_t q_phase[2] = {0, 0};
      bool q_armed[2] = {false, false}, q_due[2] = {false, false}, ok = true;
      Item it = {};
      // Q tiles go out as soon as the item before has used them up, between the K and V loads.
      auto load_q = [&] {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!q_due[t] || !mbar_test(&q_empty[t], q_phase[t] ^ 1u)) continue;
          mbar_arrive_expect_tx(&q_full[t], p.tokens * p.group * 128u * L::kHalves);
#pragma unroll
          for (int h = 0; h < L::kHalves; ++h)
            tma_load_3d(smem + t * L::kTileBytes + h * L::kHalfBytes, &tmq, &q_full[t], 64 * h,
                        it.head * static_cast<int>(p.group), it.q_row + t * tokens);
          q_armed[t] = true;
          q_due[t] = false;
          q_phase[t] ^= 1;
        }
      };
      auto wait = [&](auto &&done) {
        if (done()) return true;
        const uint64_t t0 = globaltimer();
        while (true) {
#pragma unroll 1
          for (int i = 0; i < 64; ++i) {
            load_q();
            if (done()) return true;
          }
          if (*abort_flag || globaltimer() - t0 > kWaitTimeoutNs) return false;
        }
      };
      auto load_kv = [&](const CUtensorMap *map, int row, int head) {
        if (!wait([&] { return mbar_test(&kv_empty[ring], phase ^ 1u); })) return false;
        uint8_t *dst = smem + L::kRingOff + ring * L::kTileBytes;
        mbar_arrive_expect_tx(&kv_full[ring], L::kTileBytes);
#pragma unroll
        for (int h = 0; h < L::kHalves; ++h)
          tma_load_3d(dst + h * L::kHalfBytes, map, &kv_full[ring], 64 * h, head, row);
        armed |= 1u << ring;
        parity = (parity & ~(1u << ring)) | (phase << ring);
        if (++ring == kStages) ring = 0, phase ^= 1;
        return true;
      };
      for (uint32_t k = 0; ok; ++k) {
        ok = mbar_wait(&sched_full[k % 3], (k / 3) & 1, abort_flag);
        if (!ok) break;
        it = read_item(&items[k % 3]);
        mbar_arrive(&sched_empty[k % 3]);
        if (it.last) break;
        const Reach r[2] = {reach_of(it, 0, tokens, p.causal), reach_of(it, 1, tokens, p.causal)};
        const int steps = max(r[0].steps, r[1].steps);
        q_due[0] = r[0].steps > 0;
        q_due[1] = r[1].steps > 0;
        for (int j = 0; ok && j < steps; ++j) {
          ok = load_kv(&tmk, it.k_row + j * kKeys, it.head);
          load_q();
          ok = ok && load_kv(&tmv, it.k_row + j * kKeys, it.head);
        }
        ok = ok && wait([&] { return !q_due[0] && !q_due[1]; });
      }
      if (!ok) {
        report(p.status, kErrAttentionWait);
        *abort_flag = 1;
      }
      // Copies still in flight (only after an abort) land before shared memory is released.
      for (int i = 0; i < kStages; ++i)
        if ((armed >> i) & 1u) mbar_drain(&kv_full[i], (parity >> i) & 1u);
      for (int t = 0; t < 2; ++t)
        if (q_armed[t]) mbar_drain(&q_full[t], q_phase[t] ^ 1u);
    }
  } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    fewer_registers();
    if (lane == 0) {
      const int t = warp - kMmaWarp;
      constexpr uint32_t idesc_s = idesc_f32(kBf16, 128, 0, false);  // N to come: 32 a block
      constexpr uint32_t idesc_o = idesc_f32(kBf16, 128, kDim, true);
      const uint32_t d_s = tmem + t * 128, d_o = tmem + kTmemO + t * 128;
      const uint32_t q_at = smem_u32(smem + t * L::kTileBytes);
      uint32_t ring = 0, phase = 0, v_ring = 0, v_phase = 0, p_phase = 0, q_phase = 0;
      bool ok = true;
      // One tile at a time puts its products on the tensor cores. Left to interleave, both tiles'
      // would end together, both softmaxes would start together, and the tiles would stay in step,
      // the tensor cores idle under the softmax and the other way round (2.30 ms for 16384 causal
      // tokens against 2.12); taken in turn, one falls half a step behind the other by itself.
      auto take = [&] {
        if (atomicCAS(turn, 0u, 1u) == 0u) return true;
        const uint64_t t0 = globaltimer();
        while (true) {
#pragma unroll 1
          for (int i = 0; i < 64; ++i)
            if (atomicCAS(turn, 0u, 1u) == 0u) return true;
          if (*abort_flag || globaltimer() - t0 > kWaitTimeoutNs) return false;
        }
      };
      auto give = [&] { *reinterpret_cast<volatile uint32_t *>(turn) = 0u; };
      // S = Q K^T of stage `stage`, the last of a turn.
      auto scores = [&](uint32_t stage, int blocks) {
        const uint32_t idesc = idesc_s | static_cast<uint32_t>(blocks * 32 / 8) << 17;
        tc_fence_after();
        const uint32_t k_at = smem_u32(smem + L::kRingOff + stage * L::kTileBytes);
#pragma unroll
        for (int kk = 0; kk < kDim / 16; ++kk) {
          const uint32_t off = (kk / 4) * L::kHalfBytes + (kk % 4) * 32;
          umma_f16(d_s, sw128_desc(q_at + off), sw128_desc(k_at + off), idesc, kk > 0);
        }
        give();
      };
      // One commit, for the softmax, covers the scores and all before: the softmax releases the
      // stages when it sees it (a commit holds the issuing thread about 100 cycles).
      auto hand_over = [&](bool last) {
        umma_commit(&s_full[t]);
        if (last) umma_commit(&q_empty[t]);
      };
      // Half of O += P V; of a step with fewer than four blocks of 32 keys only theirs.
      auto product = [&](uint32_t v_at, int half, bool first, int blocks) {
        tc_fence_after();
        if (blocks == 4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kk = half * 4 + i;
            umma_f16_ts(d_o, d_s + 8 * kk, sw128_mn_desc(v_at + kk * 2048, L::kHalfBytes), idesc_o,
                        !first || kk > 0);
          }
        } else {
#pragma unroll 1
          for (int kk = half * 4; kk < min(2 * blocks, half * 4 + 4); ++kk)
            umma_f16_ts(d_o, d_s + 8 * kk, sw128_mn_desc(v_at + kk * 2048, L::kHalfBytes), idesc_o,
                        !first || kk > 0);
        }
      };
      for (uint32_t k = 0; ok; ++k) {
        ok = mbar_wait(&sched_full[k % 3], (k / 3) & 1, abort_flag);
        if (!ok) break;
        const Item it = read_item(&items[k % 3]);
        mbar_arrive(&sched_empty[k % 3]);
        if (it.last) break;
        const Reach reach = reach_of(it, t, tokens, p.causal);
        const int mine = reach.steps;
        const int steps = max(mine, reach_of(it, 1 - t, tokens, p.causal).steps);
        if (steps == 0) continue;
        uint32_t k_stage = ring;
        ok = mbar_wait(&kv_full[ring], phase, abort_flag);
        if (!ok) break;
        if (++ring == kStages) ring = 0, phase ^= 1;
        if (mine > 0) {
          ok = mbar_wait(&q_full[t], q_phase, abort_flag) && take();
          if (!ok) break;
          q_phase ^= 1;
          scores(k_stage, blocks_of(reach, 0));
          hand_over(mine == 1);
        } else {
          mbar_arrive(&kv_empty[k_stage]);
        }
        for (int j = 0; j < steps; ++j) {
          // this step's V, and the next step's K behind it
          const uint32_t v_stage = ring;
          ok = mbar_wait(&kv_full[ring], phase, abort_flag) && mbar_wait(&v_ok[v_ring], v_phase, abort_flag);
          if (!ok) break;
          if (++v_ring == kStages) v_ring = 0, v_phase ^= 1;
          if (++ring == kStages) ring = 0, phase ^= 1;
          const bool more = j + 1 < steps;
          if (more) {
            k_stage = ring;
            ok = mbar_wait(&kv_full[ring], phase, abort_flag);
            if (!ok) break;
            if (++ring == kStages) ring = 0, phase ^= 1;
          }
          if (j >= mine) {
            mbar_arrive(&kv_empty[v_stage]);
            if (more) mbar_arrive(&kv_empty[k_stage]);
            continue;
          }
          const uint32_t v_at = smem_u32(smem + L::kRingOff + v_stage * L::kTileBytes);
          ok = mbar_wait(&p_full[t], p_phase, abort_flag) && take();
          if (!ok) break;
          const int blocks = blocks_of(reach, j);
          product(v_at, 0, j == 0, blocks);
          // where the second half is there by now, the turn is kept
          if (!mbar_test(&p_full[2 + t], p_phase)) {
            give();
            ok = mbar_wait(&p_full[2 + t], p_phase, abort_flag) && take();
            if (!ok) break;
          }
          p_phase ^= 1;
          product(v_at, 1, j == 0, blocks);
          if (j + 1 < mine) {
            scores(k_stage, blocks_of(reach, j + 1));
            hand_over(j + 2 == mine);
          } else {
            give();
            umma_commit(&o_full[t]);
            if (more) mbar_arrive(&kv_empty[k_stage]);
          }
        }
      }
      if (!ok) {
        report(p.status, kErrAttentionWait);
        *abort_flag = 1;
      }
      umma_commit(&drain[t]);  // every MMA this thread issued has completed before TMEM is freed
      mbar_drain(&drain[t], 0);
    }
  } else {
    more_registers();
    const int t = warp >> 2, q = warp & 3;
    const int row = q * 32 + lane;
    const int token = row / static_cast<int>(p.group), sub = row % static_cast<int>(p.group);
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t tl = tmem + lanes + t * 128, to = tmem + lanes + kTmemO + t * 128;
    const float c = p.scale_log2;
    uint8_t *stage = smem + L::kOutOff + warp * L::kOutBytes;
    uint32_t s_phase = 0, o_phase = 0, ring = 0;
    // Release the stage at `ring`, for this tile, once its last product with it is known to be done.
    auto release = [&] {
      if (q == 0 && lane == 0) mbar_arrive(&kv_empty[ring]);
      if (++ring == kStages) ring = 0;
    };
    bool ok = true;
    for (uint32_t k = 0; ok; ++k) {
      ok = __all_sync(0xffffffffu, mbar_wait(&sched_full[k % 3], (k / 3) & 1, abort_flag));
      if (!ok) break;
      const Item it = read_item(&items[k % 3]);
      __syncwarp();
      const Reach r = reach_of(it, t, tokens, p.causal);
      const int whole = r.first / kKeys;  // steps that every row of the tile sees in full
      const int mine = t * tokens + token;  // token within the item
      const int sees = p.causal ? min(it.k_len, it.visible + mine) : it.k_len;
      float m = -INFINITY, sum = 0.f;
      for (int j = 0; j < r.steps; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], s_phase, abort_flag));
        if (!ok) break;
        s_phase ^= 1;
        tc_fence_after();
        if (j > 0) release();  // the previous step's V
        release();             // this step's K
        if (j < whole)
          softmax_step<kBf16, false>(tl, to, kDim, c, kKeys, 4, j == 0, m, sum, &p_full[t]);
        else
          softmax_step<kBf16, true>(tl, to, kDim, c, sees - j * kKeys, blocks_of(r, j), j == 0, m, sum,
                                    &p_full[t]);
      }
      if (!ok) break;
      // Where the row goes, worked out under the last product.
      const bool live = token < tokens && mine < it.q_count;
      const uint32_t rows_live = __ballot_sync(0xffffffffu, live);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t out_row = static_cast<int64_t>(it.q_row) + mine;
      const uint32_t head = static_cast<uint32_t>(it.head) * p.group + sub;
      uint16_t *dst = p.out + out_row * p.out_token + head * p.out_head;
      if (live && p.lse) p.lse[out_row * p.q_heads + head] = (m + log2f(sum)) * kLn2;
      if (r.steps > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&o_full[t], o_phase, abort_flag));
        if (!ok) break;
        o_phase ^= 1;
        tc_fence_after();
        release();
      }
      // the issuer releases the stages of steps that only the other tile has
      ring = (ring + 2 * (max(r.steps, reach_of(it, 1 - t, tokens, p.causal).steps) - r.steps)) % kStages;
      const int fix = r.steps > 0 ? *reinterpret_cast<volatile int32_t *>(&items[k % 3].fix) : 0;
      __syncwarp();
      // From here on the slot is not read again; the next item but two may be written into it.
      if (lane == 0) mbar_arrive(&sched_empty[k % 3]);
      if (it.last) break;
      // 64 channels at a time through this warp's staging (16-byte chunk c of row r at c ^ (r & 7)):
      // by one TMA store where all 32 rows are of the sequence and whole tokens, else 8 lanes to a
      // row of 128 bytes.
      const bool boxed = p.boxed && rows_live == 0xffffffffu;
#pragma unroll 1
      for (int d = 0; d < kDim; d += 64) {
        if (lane == 0) bulk_wait_read<0>();  // the store before has read the staging
        __syncwarp();
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t x[32];
          if (r.steps > 0) {
            tmem_load32(to + d + 32 * half, x);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = 0;
          }
          if (fix && live) {
            // what the guard took out of the steps that are seen in part
            const int from = reach_of(it, 0, tokens, p.causal).first / kKeys * kKeys;
#pragma unroll 1
            for (int kk = from; kk < sees; ++kk) {
              const uint32_t *v = reinterpret_cast<const uint32_t *>(
                  p.v + (static_cast<int64_t>(it.k_row) + kk) * p.v_token + it.head * p.v_head + d + 32 * half);
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const uint32_t w = v[e];
                const float2 f = Elem<kBf16>::unpack(w);
                if (!finite16<kBf16>(w & 0xffffu)) x[2 * e] = __float_as_uint(__uint_as_float(x[2 * e]) + f.x);
                if (!finite16<kBf16>(w >> 16)) x[2 * e + 1] = __float_as_uint(__uint_as_float(x[2 * e + 1]) + f.y);
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = Elem<kBf16>::pack(__uint_as_float(x[8 * e + 2 * i]) * inv, __uint_as_float(x[8 * e + 2 * i + 1]) * inv);
            *reinterpret_cast<uint4 *>(stage + lane * 128 + (((4 * half + e) ^ (lane & 7)) * 16)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        if (boxed) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&tmo, stage, d, it.head * static_cast<int>(p.group), it.q_row + t * tokens + q * (32 / static_cast<int>(p.group)));
            bulk_commit();
          }
        } else {
          __syncwarp();
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {
            const int from = 4 * i + lane / 8;  // row of this warp
            const uint64_t at = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(dst), from);
            if (rows_live >> from & 1)
              *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(at) + d + 8 * (lane % 8)) =
                  *reinterpret_cast<const uint4 *>(stage + from * 128 + (((lane % 8) ^ (from & 7)) * 16));
          }
          __syncwarp();
        }
      }
      tc_fence_before();
    }
    if (!ok && lane == 0) {
      report(p.status, kErrAttentionWait);
      *abort_flag = 1;
    }
    if (lane == 0) bulk_wait<0>();  // output stores complete before the CTA retires
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

namespace {
template <bool kBf16, int kDim>
cudaError_t launch(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v,
                   const CUtensorMap &o, const PackedArgs &a, int dev, uint32_t grid, cudaStream_t stream) {
  static std::atomic<bool> configured[64] = {};
  if (dev >= 0 && dev < 64 && !configured[dev].load(std::memory_order_acquire)) {
    // setting the attribute twice (two threads racing here) is harmless
    const cudaError_t e = cudaFuncSetAttribute(attention_packed_kernel<kBf16, kDim>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               Layout<kDim>::kBytes);
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  attention_packed_kernel<kBf16, kDim>
      <<<dim3(grid), dim3(kThreads), Layout<kDim>::kBytes, stream>>>(q, k, v, o, a);
  return cudaGetLastError();
}
}  // namespace

cudaError_t launch_attention_packed(const PackedAttention &p, bool bf16, cudaStream_t stream,
                                    std::string *err) {
  if (p.total_q == 0 || p.n_seq == 0) return cudaSuccess;
  const uint32_t group = p.q_heads / p.kv_heads, tokens = 128 / group;
  CUtensorMap q, k, v, o;
  const bool boxed = 32 % group == 0;
  const bool maps =
      encode_map_rows(&q, p.q, bf16, p.head_dim, p.q_heads, p.total_q, p.q_head, p.q_token, group, tokens, err) &&
      // without keys the maps stand on q: no load reads through them
      encode_map_rows(&k, p.total_k ? p.k : p.q, bf16, p.head_dim, p.kv_heads, p.total_k ? p.total_k : 1, p.k_head,
                      p.k_token, 1, kKeys, err) &&
      encode_map_rows(&v, p.total_k ? p.v : p.q, bf16, p.head_dim, p.kv_heads, p.total_k ? p.total_k : 1, p.v_head,
                      p.v_token, 1, kKeys, err) &&
      encode_map_rows(&o, p.out, bf16, p.head_dim, p.q_heads, p.total_q, p.out_head, p.out_token,
                      boxed ? group : 1, boxed ? 32 / group : 1, err);
  if (!maps) return cudaErrorInvalidValue;
  PackedArgs a = {};
  a.v = p.v;
  a.out = p.out;
  a.lse = p.lse;
  a.cu_q = p.cu_q;
  a.cu_k = p.cu_k;
  a.v_token = p.v_token;
  a.v_head = p.v_head;
  a.out_token = p.out_token;
  a.out_head = p.out_head;
  a.status = p.status;
  a.n_seq = p.n_seq;
  a.total_q = p.total_q;
  a.total_k = p.total_k;
  a.q_heads = p.q_heads;
  a.kv_heads = p.kv_heads;
  a.group = group;
  a.tokens = tokens;
  a.item = page_div(2 * tokens);
  a.boxed = boxed;
  a.causal = p.causal;
  a.scale_log2 = p.scale * kLog2e;
  const uint64_t levels = (static_cast<uint64_t>(p.total_q) + 2 * tokens - 1) / (2 * tokens);
  int dev = 0;
  cudaGetDevice(&dev);
  // at most one partly filled item per sequence
  const uint64_t most = (levels + p.n_seq) * p.kv_heads;
  const uint32_t sms = static_cast<uint32_t>(sm_count(dev));
  const uint32_t grid = most < sms ? static_cast<uint32_t>(most) : sms;
  if (p.head_dim == 64)
    return bf16 ? launch<true, 64>(q, k, v, o, a, dev, grid, stream) : launch<false, 64>(q, k, v, o, a, dev, grid, stream);
  return bf16 ? launch<true, 128>(q, k, v, o, a, dev, grid, stream) : launch<false, 128>(q, k, v, o, a, dev, grid, stream);
}

}  // namespace dv3
