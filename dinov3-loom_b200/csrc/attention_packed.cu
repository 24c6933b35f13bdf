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
//              TMEM lane). All scores of a step are held in registers: running maximum, w =
//              2^(c (s - m)) with c = scale log2(e), f32 sum of the unrounded weights, P (rounded to
//              the element type) back to TMEM over the consumed scores. The reference m only moves
//              when the maximum has grown by more than 2^8 over it: any m gives the same quotient,
//              and sums and weights up to 2^8 too large lose nothing in f32, bf16 or f16 (whose
//              weights end at 2^15, see sequence.cuh); the row's output is then rescaled in TMEM. At an item's end O / sum goes through a staging
//              tile to global memory. Of a last, partly visible step only the blocks of 32 keys
//              that some row sees are computed.
//   warp 8     TMA producer: Q tiles, then K and V tiles in turn through one ring of stages.
//   warps 9/10 MMA issuers of tile 0 / tile 1: S_t = Q_t K^T (M = 128, N = a step's keys), and
//              O_t += P_t V with P from TMEM and V as the MN-major B operand, one tile at a time.
//   warp 11    scheduler (publishes items one ahead), and guard of V: a key that a row does not see
//              has weight 0, but 0 times an infinity or NaN is NaN. Only the tiles at an item's end (from the first that some
//              row sees in part) can hold such keys; there it tests V in shared memory, sets what
//              is not finite to 0 and leaves a note, and the rows that do see those keys add them
//              at the end from global memory.
//
// Bound by the exp2 unit and the tensor cores together where sequences are long (each busy 56 % of the
// time, one tile's softmax under the other's products), by the chain of a tile's steps and its
// items' starts and ends where they are short. Measured: 16384 causal tokens, 32/8 heads of 128, bf16,
// 2.13 ms (1030 TFLOP/s, at the power cap); 24 such sequences of 1..2048 tokens 83 us; 64 of 201
// tokens, 6 heads of 64, f16, 23.0 us (14.9 as an eighth of a batch of 512).
//
// Every wait is bounded; on a timeout the kernel records kErrAttentionWait, raises the CTA's
// abort flag, lets its own copies and MMAs in flight land, frees TMEM and returns; the join then leaves
// the cut items' rows as they were.
#include <atomic>

#include "packed_parts.h"
#include "sequence.cuh"

namespace dv3 {

namespace {
constexpr int kThreads = 384;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;  // TMEM allocator; issues tile 0's MMAs, warp 10 tile 1's
constexpr int kGuardWarp = 11;
constexpr int kBuckets = 64;    // of the scheduler's order
// Log2 units by which a row's maximum may pass its reference. 4 would leave f16 weights four bits more
// below the largest, but moved the references of 8192 causal tokens (32/8 heads of 128) so much more
// often that they took 665 us and not 569.
constexpr int kSlack = 8;
constexpr float kFar = 4096.f;  // log2 units from which on a reference is subtracted before the scale

// One work item as the scheduler publishes it (two 16-byte words).
struct __align__(16) Item {
  int32_t q_row;    // first query row
  int32_t q_count;  // its tokens (0: nothing to do)
  int32_t k_row;    // first key row of the sequence
  int32_t k_len;
  int32_t visible;  // keys the first token sees, less than 1 if none; a later one sees one more if causal
  int32_t head;     // key-value head
  int32_t part;     // -1: no more items; 0: the whole of it; else 1 + the place of its partial result
  int32_t fix;      // set by the guard: V held something that is not finite
};

__device__ __forceinline__ Item read_item(const Item *slot) {
  Item it;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(it.q_row), "=r"(it.q_count), "=r"(it.k_row), "=r"(it.k_len)
               : "r"(smem_u32(slot))
               : "memory");
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(it.visible), "=r"(it.head), "=r"(it.part), "=r"(it.fix)
               : "r"(smem_u32(slot) + 16)
               : "memory");
  return it;
}

// At 64 channels the outputs leave TMEM columns for P, so that a step's scores need not wait for the
// step before to be done with its weights: they are issued when the softmax has the previous ones in
// registers, and the next softmax starts at once.
template <int kDim>
struct Layout {
  static constexpr int kKeys = 128;  // a step
  static constexpr int kBlocks = kKeys / 32;
  static constexpr bool kOwnP = kDim == 64;
  static constexpr int kTmemO = 2 * kKeys;              // S_0 | S_1 | O_0 | O_1 | P_0 | P_1
  static constexpr int kTmemP = kOwnP ? kTmemO + 2 * kDim : 0;
  static constexpr int kTmemPStep = kOwnP ? kKeys / 2 : kKeys;  // from P_0 to P_1
  static constexpr int kHalves = kDim / 64;             // 64-channel (128-byte) columns of a tile
  static constexpr int kQHalf = 128 * 128, kQBytes = kHalves * kQHalf;
  static constexpr int kTileHalf = kKeys * 128, kTileBytes = kHalves * kTileHalf;  // of K or V
  static constexpr int kStages = kDim == 128 ? 4 : 6;
  static constexpr int kRingOff = 2 * kQBytes;          // Q_0 | Q_1 | stages | output staging
  static constexpr int kOutOff = kRingOff + kStages * kTileBytes;
  static constexpr int kOutBytes = 32 * 128;            // a softmax warp's: 32 rows of 64 channels
  static constexpr int kBarOff = kOutOff + 8 * kOutBytes;
  // barriers: q_full[2] q_empty[2] s_full[2] s_free[2] p_full[4] (first halves, second halves) o_full[2]
  // drain[2] sched_full[3] sched_empty[3] kv_full[stages] kv_empty[stages] v_ok[stages] (by V tile, not by stage: a stage
  // of an odd ring holds K and V in turn)
  static constexpr int kBars = 22 + 3 * kStages;
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
// `width` keys; by sequence within a class, later items of a sequence first. Where there are few items
// and some have more steps than 1.5 times what the average CTA has in all, those are cut into parts of
// at most so many (`part`), by class, that other CTAs take (300 queries behind 16000 keys: 253 us uncut,
// 148 cut at the average, 106 so; choosing the parts by estimated rounds of the CTAs took 1.8 us for
// the choice and gave 4096 causal tokens 147 us, not 134); a part leaves (max, sum, unnormalised
// output) in the workspace and a second launch joins them. The classes that are cut are the first in the order,
// so that a part's place in it is also its place in the workspace.
struct Order {
  uint32_t *starts;  // first entry (item, or part) of each class, top class first; [kBuckets]
  uint32_t total;    // entries
  uint32_t width;
  uint32_t part;     // steps; 0: nothing is cut
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
  bool flat;           // no CTA gets more than one item: their order does not matter
  uint32_t parts_max;  // partial results that the workspace holds; 0: nothing is cut
  void *workspace;
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

// Steps of 128 keys in the items of a class, and the parts that each is cut into.
__device__ __forceinline__ uint32_t steps_of(uint32_t c, uint32_t width) {
  return ((c + 1) * width + 127) / 128;
}
__device__ __forceinline__ uint32_t parts_of(uint32_t c, uint32_t width, uint32_t part) {
  return part ? (steps_of(c, width) + part - 1) / part : 1;
}

// Entry `index` of the order, for key-value head `head`; whole warp.
template <int kDim>
__device__ __forceinline__ Item find_item(const PackedArgs &p, Order &o, uint32_t index, uint32_t head) {
  const uint32_t lane = threadIdx.x & 31u;
  Item it = {};
  it.head = static_cast<int32_t>(head);
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < kBuckets / 32; ++i) mine += o.starts[lane * (kBuckets / 32) + i] <= index;
  const int at = static_cast<int>(__reduce_add_sync(0xffffffffu, mine)) - 1;
  const uint32_t c = kBuckets - 1 - at, parts = parts_of(c, o.width, o.part);
  const uint32_t entry = index - o.starts[at], rest = parts > 1 ? entry / parts : entry;
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
      if (parts > 1) {
        // this part's steps, as an item of its own over their keys
        const int which = static_cast<int>(entry % parts), n = static_cast<int>(parts);
        const int most = p.causal ? min(it.k_len, it.visible + it.q_count - 1) : it.k_len;
        const int steps = (max(most, 0) + 127) / 128, from = steps * which / n * 128;
        const int to = which + 1 == n ? it.k_len : min(it.k_len, steps * (which + 1) / n * 128);
        it.k_row += from;
        it.k_len = to - from;
        it.visible -= from;
        const uint32_t place = index * p.kv_heads + head;
        it.part = static_cast<int32_t>(place) + 1;
        if (lane == 0) {
          Part *w = Parts<kDim>::of(p.workspace, p.parts_max).what + place;
          w->q_row = it.q_row;
          w->q_count = it.q_count;
          w->head = it.head;
          w->index = which;
          w->parts = n;
        }
      }
      return it;
    }
    o.before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return it;  // not reached while cu is ascending
}

// What a tile's rows see.
template <int kKeys>
struct Reach {
  int steps;  // of kKeys keys
  int first;  // keys that its first token sees (at least 0)
  int most;   // keys that its last token sees
};
// Blocks of 32 keys in step j that some row of the tile sees.
template <int kKeys>
__device__ __forceinline__ int blocks_of(const Reach<kKeys> &r, int j) {
  return min(kKeys / 32, (r.most - j * kKeys + 31) / 32);
}
template <int kKeys>
__device__ __forceinline__ Reach<kKeys> reach_of(const Item &it, int tile, int tokens, bool causal) {
  const int begin = tile * tokens, end = min(it.q_count, begin + tokens);
  Reach<kKeys> r = {0, 0, 0};
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

// A row's reference m, a score, moved to the step's maximum `top` where that passes it by more than kSlack
// after the scale c; the row's sum and output so far follow. The previous product is done: the thread
// that issued it issued these scores after it.
__device__ __forceinline__ void move_reference(uint32_t to, int dim, float c, float top, bool first,
                                               float &m, float &sum) {
  const float rise = (top - m) * c;  // rounded products of the two might not differ
  const bool grown = rise > kSlack;
  if (!first && !__any_sync(0xffffffffu, grown)) return;
  if (first || grown) m = top;
  if (first) return;
  const float f = grown ? ex2_approx(-rise) : 1.f;
  sum *= f;
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

// The weights of 32 scores, 2^(s c + base), stored over consumed scores and added to (s0, s1).
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

// Scores, weights and sums of one step for this thread's row, through its reference m and sum; c is
// scale log2(e). Where some row of the tile sees the step in part (`masked`), this one sees `vis` keys of it
// and the tile `blocks` blocks of 32; the products skip the others. The weights are handed over in
// two halves (p_full[0], p_full[2]), so that the product with V starts under the second. One form for
// both kinds of step: two thrashed the instruction cache. loaded() is called when the scores are in
// registers, before() before the output or the weights' columns (at tp) are touched.
template <bool kBf16, int kBlocks, class Loaded, class Before>
__device__ __forceinline__ bool softmax_step(uint32_t tl, uint32_t to, int dim, float c, bool masked,
                                             int vis, int blocks, bool first, float &m, float &sum,
                                             uint32_t tp, uint64_t *p_full, Loaded &&loaded,
                                             Before &&before) {
  if (masked) {
    // what a row does not see becomes -inf in TMEM, in the blocks that some row of the warp sees in part
    const int least = __reduce_min_sync(0xffffffffu, vis);
#pragma unroll 1
    for (int i = max(least, 0) / 32; i < blocks; ++i) {
      uint32_t x[32];
      tmem_load32(tl + 32 * i, x);
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (e >= vis - 32 * i) x[e] = 0xff800000u;
      tmem_st32(tl + 32 * i, x);
    }
    tmem_st_wait();
  }
  uint32_t v[kBlocks][32];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) tmem_ld32(tl + 32 * i, v[i]);  // past `blocks`: old values, not used
  tmem_wait_ld(v[0]);
#pragma unroll
  for (int i = 1; i < kBlocks; ++i) tmem_regs_ready(v[i]);
  loaded();
  float tops[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) {
    tops[i] = max3(__uint_as_float(v[i][0]), __uint_as_float(v[i][1]), __uint_as_float(v[i][2]));
#pragma unroll
    for (int e = 3; e + 1 < 32; e += 2)
      tops[i] = max3(tops[i], __uint_as_float(v[i][e]), __uint_as_float(v[i][e + 1]));
    tops[i] = fmaxf(tops[i], __uint_as_float(v[i][31]));
    if (i >= blocks) tops[i] = -INFINITY;
  }
  float top = tops[0];
#pragma unroll
  for (int i = 1; i < kBlocks; ++i) top = fmaxf(top, tops[i]);
  if (!before()) return false;
  move_reference(to, dim, c, top, first, m, sum);
  // The weights are 2^(s c - m c). The rounding of m c is a factor of all of a row's weights that its sum
  // has too, below 2^(2^-12) where it is less than kFar; it grows with m c, past the exponent's range at
  // 2^32. From kFar on the difference s - m comes before the scale (for every score it took 3 to 4 % of the
  // long prompts' time).
  float base = m == -INFINITY ? 0.f : m * c;
  if (__builtin_expect(fabsf(base) >= kFar, 0)) {
    const uint64_t from2 = pair(-m, -m);
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 x = unpair(add2(pair(v[i][e], v[i][e + 1]), from2));
        v[i][e] = __float_as_uint(x.x);
        v[i][e + 1] = __float_as_uint(x.y);
      }
    base = 0.f;
  }
  base = weight_shift<kBf16>(kSlack) - base;
  const uint64_t c2 = pair(c, c), base2 = pair(base, base);
  uint64_t s0 = 0, s1 = 0;
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) {
    if (i < blocks) weigh<kBf16>(tp + 16 * i, v[i], c2, base2, s0, s1);
    if (i == kBlocks / 2 - 1) hand_over_weights(p_full);
    if (i == kBlocks - 1) hand_over_weights(p_full + 2);
  }
  const float2 part = unpair(add2(s0, s1));
  sum += part.x + part.y;
  return true;
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
  constexpr int kStages = L::kStages, kKeys = L::kKeys, kTmemO = L::kTmemO, kTmemCols = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t *q_full = reinterpret_cast<uint64_t *>(smem + L::kBarOff);
  uint64_t *q_empty = q_full + 2, *s_full = q_full + 4, *s_free = q_full + 6, *p_full = q_full + 8;
  uint64_t *o_full = q_full + 12, *drain = q_full + 14, *sched_full = q_full + 16, *sched_empty = q_full + 19;
  uint64_t *kv_full = q_full + 22, *kv_empty = kv_full + kStages, *v_ok = kv_empty + kStages;
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
      mbar_init(&s_free[i], 4);  // the tile's softmax warps
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
  for (int i = threadIdx.x; i <= kBuckets; i += kThreads) order[i] = 0;
  // All before is under the end of the kernel before. TMEM after the wait: all its columns are taken, and
  // a kernel that is not done may still want some on this SM. This kernel does not let the next one in
  // early: its CTAs would take the SMs in the order they fall free, and 24 prompts of 1..2048 tokens, each
  // call behind the last, then took 90 us and not 84.
  pdl_wait();
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  uint32_t width = 0x7fffff00u;  // one class
  if (!p.flat) {
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
    // Few sequences: a warp for each, the classes over its lanes; else a thread, over its own classes
    // (24 of 1..2048 tokens, 16/8 heads of 64: 79 us with warps, 89 with threads; 256 of them 408 and 410, 256 of 1..16
    // 66 and 59). Of many, a class is a step wide at least: the search walks all sequences once for
    // each class that there is (4096 of 1..16 tokens 830 us, 1250 with classes of one key).
    const bool few = p.n_seq <= 96;
    width = max(few ? 1u : static_cast<uint32_t>(kKeys), (order[kBuckets] + kBuckets - 1) / kBuckets);
    if (few) {
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
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int tokens = static_cast<int>(p.tokens);

  if (warp == kGuardWarp) {
    fewer_registers();
    Order o = {order, 0, width, 0, -1, 0, 0};
    if (!p.flat) {  // counts to starts
      static_assert(kBuckets == 64, "two classes a lane");
      uint32_t n0 = order[2 * lane], n1 = order[2 * lane + 1];
      const uint32_t c0 = kBuckets - 1 - 2 * lane, c1 = c0 - 1;
      auto sum_of = [](uint64_t x) {
#pragma unroll
        for (int i = 16; i > 0; i /= 2) x += __shfl_xor_sync(0xffffffffu, x, i);
        return x;
      };
      if (p.parts_max) {
        const uint64_t steps = sum_of(static_cast<uint64_t>(n0) * steps_of(c0, width) +
                                      static_cast<uint64_t>(n1) * steps_of(c1, width)) * p.kv_heads;
        uint64_t cut;
        // 4 steps at least: 2 take 16.0 us and not 17.9 for one query behind 1100 keys, but 28.8 and not 23.9
        // where one sequence of 8000 keys stands among sixteen
        o.part = max(4u, static_cast<uint32_t>((steps * 3 / 2 + gridDim.x - 1) / gridDim.x));
        while (true) {  // until the parts fit the workspace
          const uint32_t p0 = parts_of(c0, width, o.part), p1 = parts_of(c1, width, o.part);
          cut = sum_of((p0 > 1 ? static_cast<uint64_t>(n0) * p0 : 0) + (p1 > 1 ? static_cast<uint64_t>(n1) * p1 : 0)) * p.kv_heads;
          if (cut <= p.parts_max) break;
          o.part += o.part / 4 + 1;
        }
        if (blockIdx.x == 0 && lane == 0) *Parts<kDim>::of(p.workspace, p.parts_max).count = static_cast<uint32_t>(cut);
        n0 *= parts_of(c0, width, o.part);
        n1 *= parts_of(c1, width, o.part);
      }
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
    // flat: as many items as CTAs at most, whatever their number
    const uint64_t n_items = p.flat ? gridDim.x : static_cast<uint64_t>(o.total) * p.kv_heads;
    bool ok = true;
    // Publish item k of this CTA: up the order and down again in turn, so that no CTA always gets
    // the longest of each round.
    auto publish = [&](uint32_t k) {
      const uint64_t at = static_cast<uint64_t>(k) * gridDim.x +
                          (k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      Item it = {};
      if (at < n_items)
        it = find_item<kDim>(p, o, static_cast<uint32_t>(at / p.kv_heads), static_cast<uint32_t>(at % p.kv_heads));
      // the up-and-down order may leave one CTA an item in a round in which others have none
      if (static_cast<uint64_t>(k) * gridDim.x >= n_items) it.part = -1;
      ok = __all_sync(0xffffffffu, mbar_wait(&sched_empty[k % 3], ((k / 3) & 1) ^ 1u, abort_flag));
      if (ok && lane == 0) {
        volatile Item *d = &items[k % 3];
        d->q_row = it.q_row;
        d->q_count = it.q_count;
        d->k_row = it.k_row;
        d->k_len = it.k_len;
        d->visible = it.visible;
        d->head = it.head;
        d->part = it.part;
        d->fix = 0;
        mbar_arrive(&sched_full[k % 3]);
      }
      return it;
    };
    uint32_t ring = 0, phase = 0, v_ring = 0;
    Item it = {};  // nothing before the first
    for (uint32_t k = 0; ok && it.part >= 0; ++k) {
      const Item next = publish(k);
      if (!ok) break;
      const Reach<kKeys> r0 = reach_of<kKeys>(it, 0, tokens, p.causal), r1 = reach_of<kKeys>(it, 1, tokens, p.causal);
      const int steps = max(r0.steps, r1.steps), partial = r0.first / kKeys;
      for (int j = 0; j < steps; ++j) {
        if (++ring == kStages) ring = 0, phase ^= 1;  // the step's K stage
        ok = __all_sync(0xffffffffu, mbar_wait(&kv_full[ring], phase, abort_flag));
        if (!ok) break;
        if (j >= partial) {
          uint4 *x = reinterpret_cast<uint4 *>(smem + L::kRingOff + ring * L::kTileBytes);
          uint32_t acc = 0;
#pragma unroll 4
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
            *reinterpret_cast<volatile int32_t *>(&items[(k - 1) % 3].fix) = 1;
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
            tma_load_3d(smem + t * L::kQBytes + h * L::kQHalf, &tmq, &q_full[t], 64 * h,
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
          tma_load_3d(dst + h * L::kTileHalf, map, &kv_full[ring], 64 * h, head, row);
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
        if (it.part < 0) break;
        const Reach<kKeys> r[2] = {reach_of<kKeys>(it, 0, tokens, p.causal), reach_of<kKeys>(it, 1, tokens, p.causal)};
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
      const uint32_t d_s = tmem + t * kKeys, d_o = tmem + kTmemO + t * kDim, p_at = tmem + L::kTmemP + t * L::kTmemPStep;
      const uint32_t q_at = smem_u32(smem + t * L::kQBytes);
      uint32_t ring = 0, phase = 0, v_ring = 0, v_phase = 0, p_phase = 0, q_phase = 0;
      bool ok = true;
      // One tile at a time puts its products on the tensor cores. Left to interleave, both tiles'
      // would end together, both softmaxes would start together, and the tiles would stay in step,
      // the tensor cores idle under the softmax and the other way round (2.30 ms for 16384 causal
      // tokens of 32/8 heads of 128 against 2.07); taken in turn, one falls half a step behind the other by itself.
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
      // S = Q K^T of stage `stage`.
      auto scores = [&](uint32_t stage, int blocks) {
        const uint32_t idesc = idesc_s | static_cast<uint32_t>(blocks * 32 / 8) << 17;
        tc_fence_after();
        const uint32_t k_at = smem_u32(smem + L::kRingOff + stage * L::kTileBytes);
#pragma unroll
        for (int kk = 0; kk < kDim / 16; ++kk) {
          const uint32_t in = (kk % 4) * 32;
          umma_f16(d_s, sw128_desc(q_at + (kk / 4) * L::kQHalf + in),
                   sw128_desc(k_at + (kk / 4) * L::kTileHalf + in), idesc, kk > 0);
        }
      };
      // One commit, for the softmax, covers the scores and all before: the softmax releases the
      // stages when it sees it (a commit holds the issuing thread about 100 cycles).
      auto hand_over = [&](bool last) {
        umma_commit(&s_full[t]);
        if (last) umma_commit(&q_empty[t]);
      };
      // Half of O += P V; of a step that is seen in part only the blocks of 32 keys that are.
      auto product = [&](uint32_t v_at, int half, bool first, int blocks) {
        tc_fence_after();
        constexpr int kHalf = kKeys / 32;  // products of 16 keys in half a step
        if (blocks == L::kBlocks) {
#pragma unroll
          for (int i = 0; i < kHalf; ++i) {
            const int kk = half * kHalf + i;
            umma_f16_ts(d_o, p_at + 8 * kk, sw128_mn_desc(v_at + kk * 2048, L::kTileHalf), idesc_o,
                        !first || kk > 0);
          }
        } else {
#pragma unroll 1
          for (int kk = half * kHalf; kk < min(2 * blocks, half * kHalf + kHalf); ++kk)
            umma_f16_ts(d_o, p_at + 8 * kk, sw128_mn_desc(v_at + kk * 2048, L::kTileHalf), idesc_o,
                        !first || kk > 0);
        }
      };
      for (uint32_t k = 0; ok; ++k) {
        ok = mbar_wait(&sched_full[k % 3], (k / 3) & 1, abort_flag);
        if (!ok) break;
        const Item it = read_item(&items[k % 3]);
        mbar_arrive(&sched_empty[k % 3]);
        if (it.part < 0) break;
        const Reach<kKeys> reach = reach_of<kKeys>(it, t, tokens, p.causal);
        const int mine = reach.steps;
        const int steps = max(mine, reach_of<kKeys>(it, 1 - t, tokens, p.causal).steps);
        if (steps == 0) continue;
        if constexpr (L::kOwnP) {
          // The item's nth stage, K and V in turn, counted over all items.
          auto wait_stage = [&](uint32_t n) {
            return mbar_wait(&kv_full[n % kStages], n / kStages & 1, abort_flag);
          };
          for (int j = -1; j < steps; ++j) {
            // the next step's scores, once the softmax has this one's in registers
            if (j + 1 < steps) {
              const uint32_t n = ring + 2 * (j + 1);
              ok = wait_stage(n);
              if (!ok) break;
              if (j + 1 < mine) {
                if (j < 0) {
                  ok = mbar_wait(&q_full[t], q_phase, abort_flag);
                  q_phase ^= 1;
                }
                ok = ok && mbar_wait(&s_free[t], phase ^ 1u, abort_flag);
                if (!ok) break;
                phase ^= 1;
                scores(n % kStages, blocks_of(reach, j + 1));
                hand_over(j + 2 == mine);
              } else {
                mbar_arrive(&kv_empty[n % kStages]);
              }
            }
            if (j < 0) continue;
            const uint32_t n = ring + 2 * j + 1;
            ok = wait_stage(n) && mbar_wait(&v_ok[v_ring], v_phase, abort_flag);
            if (!ok) break;
            if (++v_ring == kStages) v_ring = 0, v_phase ^= 1;
            if (j >= mine) {
              mbar_arrive(&kv_empty[n % kStages]);
              continue;
            }
            const uint32_t v_at = smem_u32(smem + L::kRingOff + n % kStages * L::kTileBytes);
            const int blocks = blocks_of(reach, j);
            ok = mbar_wait(&p_full[t], p_phase, abort_flag);
            if (!ok) break;
            product(v_at, 0, j == 0, blocks);
            ok = mbar_wait(&p_full[2 + t], p_phase, abort_flag);
            if (!ok) break;
            p_phase ^= 1;
            product(v_at, 1, j == 0, blocks);
            umma_commit(&o_full[t]);
          }
          ring += 2 * steps;
        } else {
          uint32_t k_stage = ring;
          ok = mbar_wait(&kv_full[ring], phase, abort_flag);
          if (!ok) break;
          if (++ring == kStages) ring = 0, phase ^= 1;
          if (mine > 0) {
            ok = mbar_wait(&q_full[t], q_phase, abort_flag) && take();
            if (!ok) break;
            q_phase ^= 1;
            scores(k_stage, blocks_of(reach, 0));
            give();
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
            ok = mbar_wait(&p_full[2 + t], p_phase, abort_flag);
            if (!ok) break;
            p_phase ^= 1;
            product(v_at, 1, j == 0, blocks);
            if (j + 1 < mine) {
              scores(k_stage, blocks_of(reach, j + 1));
              give();
              hand_over(j + 2 == mine);
            } else {
              give();
              umma_commit(&o_full[t]);
              if (more) mbar_arrive(&kv_empty[k_stage]);
            }
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
    const uint32_t tl = tmem + lanes + t * kKeys, to = tmem + lanes + kTmemO + t * kDim;
    const float c = p.scale_log2;
    uint8_t *stage = smem + L::kOutOff + warp * L::kOutBytes;
    const uint32_t tp = L::kOwnP ? tmem + lanes + L::kTmemP + t * L::kTmemPStep : tl;
    uint32_t s_phase = 0, o_phase = 0, ring = 0;
    // Release the item's nth stage (K and V in turn), for this tile, when its last product with it is
    // known to be done.
    auto release = [&](int n) {
      if (q == 0 && lane == 0) mbar_arrive(&kv_empty[(ring + n) % kStages]);
    };
    bool ok = true;
    for (uint32_t k = 0; ok; ++k) {
      ok = __all_sync(0xffffffffu, mbar_wait(&sched_full[k % 3], (k / 3) & 1, abort_flag));
      if (!ok) break;
      const Item seen = read_item(&items[k % 3]);
      __syncwarp();
      const Reach<kKeys> r = reach_of<kKeys>(seen, t, tokens, p.causal);
      const int whole = r.first / kKeys;  // steps that every row of the tile sees in full
      const int mine = t * tokens + token;  // token within the item
      const int sees = p.causal ? min(seen.k_len, seen.visible + mine) : seen.k_len;
      float m = -INFINITY, sum = 0.f;
      for (int j = 0; j < r.steps; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], s_phase, abort_flag));
        if (!ok) break;
        s_phase ^= 1;
        tc_fence_after();
        const bool masked = j >= whole;
        auto step = [&](auto &&loaded, auto &&before) {
          return softmax_step<kBf16, L::kBlocks>(tl, to, kDim, c, masked, sees - j * kKeys,
                                                 masked ? blocks_of(r, j) : L::kBlocks, j == 0, m, sum,
                                                 tp, &p_full[t], loaded, before);
        };
        if constexpr (L::kOwnP) {
          release(2 * j);  // this step's K
          ok = step(
              [&] {  // S may be overwritten
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_free[t]);
              },
              [&] {  // the product of the step before is done: its V, P and O are free
                if (j == 0) return true;
                if (!__all_sync(0xffffffffu, mbar_wait(&o_full[t], o_phase, abort_flag))) return false;
                o_phase ^= 1;
                tc_fence_after();
                release(2 * j - 1);
                return true;
              });
          if (!ok) break;
        } else {
          if (j > 0) release(2 * j - 1);  // the previous step's V
          release(2 * j);                 // this step's K
          step([] {}, [] { return true; });
        }
      }
      if (!ok) break;
      // Where the row goes, worked out under the last product (the item read again: its registers are
      // the scores' meanwhile).
      const Item it = read_item(&items[k % 3]);
      const bool live = token < tokens && mine < it.q_count;
      const uint32_t rows_live = __ballot_sync(0xffffffffu, live);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t out_row = static_cast<int64_t>(it.q_row) + mine;
      const uint32_t head = static_cast<uint32_t>(it.head) * p.group + sub;
      uint16_t *dst = p.out + out_row * p.out_token + head * p.out_head;
      if (live && p.lse && it.part == 0) p.lse[out_row * p.q_heads + head] = log_sum<kBf16>(m * c, sum, kSlack);
      if (r.steps > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&o_full[t], o_phase, abort_flag));
        if (!ok) break;
        o_phase ^= 1;
        tc_fence_after();
        release(2 * r.steps - 1);
      }
      // the issuer releases the stages of steps that only the other tile has
      ring = (ring + 2 * max(r.steps, reach_of<kKeys>(it, 1 - t, tokens, p.causal).steps)) % kStages;
      const int fix = r.steps > 0 ? *reinterpret_cast<volatile int32_t *>(&items[k % 3].fix) : 0;
      __syncwarp();
      // From here on the slot is not read again; the next item but two may be written into it.
      if (lane == 0) mbar_arrive(&sched_empty[k % 3]);
      if (it.part < 0) break;
      if (rows_live == 0) continue;
      if (fix) {
        // what the guard took out of the steps that are seen in part
        const int from = reach_of<kKeys>(it, 0, tokens, p.causal).first / kKeys * kKeys;
#pragma unroll 1
        for (int d = 0; d < kDim; d += 16) {
          uint32_t x[16];
          tmem_ld16(to + d, x);
          tmem_ld_wait();
          tmem_regs_ready16(x);
#pragma unroll 1
          for (int kk = from; live && kk < sees; ++kk) {
            const uint32_t *v = reinterpret_cast<const uint32_t *>(
                p.v + (static_cast<int64_t>(it.k_row) + kk) * p.v_token + it.head * p.v_head + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t w = v[e];
              const float2 f = Elem<kBf16>::unpack(w);
              if (!finite16<kBf16>(w & 0xffffu)) x[2 * e] = __float_as_uint(__uint_as_float(x[2 * e]) + f.x);
              if (!finite16<kBf16>(w >> 16)) x[2 * e + 1] = __float_as_uint(__uint_as_float(x[2 * e + 1]) + f.y);
            }
          }
          __syncwarp();
          tmem_st16(to + d, x);
        }
        tmem_st_wait();
      }
      // 64 channels at a time through this warp's staging (16-byte chunk c of row r at c ^ (r & 7)):
      // by one TMA store where all 32 rows are of the sequence and whole tokens, else 8 lanes to a
      // row of 128 bytes. The next 64 are read and rounded while the store before reads the staging.
      const bool boxed = p.boxed && rows_live == 0xffffffffu;
#pragma unroll 1
      for (int d = 0; d < kDim; d += 64) {
        uint32_t x[2][32];
        if (r.steps > 0) {
          tmem_ld32(to + d, x[0]);
          tmem_ld32(to + d + 32, x[1]);
          tmem_wait_ld(x[0]);
          tmem_regs_ready(x[1]);
        } else {
#pragma unroll
          for (int e = 0; e < 64; ++e) x[e / 32][e % 32] = 0;
        }
        if (it.part > 0) {  // a part: as it is
          const Parts<kDim> to_join = Parts<kDim>::of(p.workspace, p.parts_max);
          const size_t tile = static_cast<size_t>(it.part - 1) * 2 + t;
          if (live) {
            if (d == 0) reinterpret_cast<float2 *>(to_join.ml)[tile * 128 + row] = make_float2(m, sum);
            float4 *o = reinterpret_cast<float4 *>(to_join.o) + (tile * (kDim / 4) + d / 4) * 128 + row;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e * 128] = make_float4(__uint_as_float(x[e / 8][4 * e % 32]), __uint_as_float(x[e / 8][4 * e % 32 + 1]),
                                       __uint_as_float(x[e / 8][4 * e % 32 + 2]), __uint_as_float(x[e / 8][4 * e % 32 + 3]));
          }
          continue;
        }
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 32; ++e)
          w[e] = Elem<kBf16>::pack(__uint_as_float(x[e / 16][2 * e % 32]) * inv, __uint_as_float(x[e / 16][2 * e % 32 + 1]) * inv);
        if (lane == 0) bulk_wait_read<0>();  // the store before has read the staging
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4 *>(stage + lane * 128 + ((e ^ (lane & 7)) * 16)) =
              make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
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
  if (p.parts_max && threadIdx.x == 0)
    Parts<kDim>::of(p.workspace, p.parts_max).done[blockIdx.x] = *abort_flag ? Parts<kDim>::kGaveUp : Parts<kDim>::kDone;
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the parts of the cut items: out = sum_i f_i o_i / sum_i f_i l_i, f_i = 2^(c (m_i - M)), over the
// parts in order. The CTAs of a part take its share of the item's rows, 16 channels each: a thread for a row and
// four channels, rows next to one another.
template <bool kBf16, int kDim>
__global__ void __launch_bounds__(256) attention_packed_join_kernel(const PackedArgs p) {
  pdl_wait();
  const Parts<kDim> w = Parts<kDim>::of(p.workspace, p.parts_max);
  // loaded together; what is not a part's is not used
  const uint32_t count = *w.count;
  const Part part = w.what[blockIdx.x];
  if (!__syncthreads_and(w.finished(p.parts_max, threadIdx.x, 256)) || blockIdx.x >= count) return;
  const float2 *mls = reinterpret_cast<const float2 *>(w.ml);
  const float4 *os = reinterpret_cast<const float4 *>(w.o);
  // the item's parts stand kv_heads apart
  const uint32_t first = blockIdx.x - part.index * p.kv_heads;
  const int from = 256 * part.index / part.parts, rows = 256 * (part.index + 1) / part.parts - from;
  for (int x = threadIdx.x; x < rows * 4; x += 256) {
    const int row = from + x % rows, d4 = blockIdx.y * 4 + x / rows;
    const int t = row / 128, in = row % 128, token = in / static_cast<int>(p.group);
    const int mine = t * static_cast<int>(p.tokens) + token;
    if (token >= static_cast<int>(p.tokens) || mine >= part.q_count) continue;
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int i = 0; i < part.parts; ++i)
      top = fmaxf(top, mls[(static_cast<size_t>(first) + i * p.kv_heads) * 256 + row].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < part.parts; ++i) {
      const size_t at = static_cast<size_t>(first) + i * p.kv_heads;
      const float2 ml = mls[at * 256 + row];
      if (ml.x == -INFINITY && ml.y == 0.f) continue;  // sees none of the part's keys
      const float f = top == -INFINITY ? 1.f : ex2_approx((ml.x - top) * p.scale_log2);
      const float4 v = os[((at * 2 + t) * (kDim / 4) + d4) * 128 + in];
      sum = fmaf(ml.y, f, sum);
      acc.x = fmaf(v.x, f, acc.x);
      acc.y = fmaf(v.y, f, acc.y);
      acc.z = fmaf(v.z, f, acc.z);
      acc.w = fmaf(v.w, f, acc.w);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t out_row = static_cast<int64_t>(part.q_row) + mine;
    const uint32_t head = part.head * p.group + in % p.group;
    *reinterpret_cast<uint2 *>(p.out + out_row * p.out_token + head * p.out_head + 4 * d4) =
        make_uint2(Elem<kBf16>::pack(acc.x * inv, acc.y * inv), Elem<kBf16>::pack(acc.z * inv, acc.w * inv));
    if (p.lse && d4 == 0) p.lse[out_row * p.q_heads + head] = log_sum<kBf16>(top * p.scale_log2, sum, kSlack);
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
  const cudaError_t e = launch_pdl(attention_packed_kernel<kBf16, kDim>, dim3(grid), dim3(kThreads), Layout<kDim>::kBytes,
                                   stream, q, k, v, o, a);
  if (e != cudaSuccess || a.parts_max == 0) return e;
  return launch_pdl(attention_packed_join_kernel<kBf16, kDim>, dim3(a.parts_max, kDim / 16), dim3(256), 0, stream, a);
}

// What the host can tell of a call's items.
struct Items {
  uint32_t tokens;     // of a tile
  uint64_t most;       // items at most: one partly filled one per sequence
  uint32_t parts_max;  // see PackedArgs
};
uint32_t most_parts(uint32_t sms) { return 2 * sms; }
Items items_of(const PackedAttention &p, uint32_t sms) {
  Items x;
  x.tokens = 128 / (p.q_heads / p.kv_heads);
  x.most = ((static_cast<uint64_t>(p.total_q) + 2 * x.tokens - 1) / (2 * x.tokens) + p.n_seq) * p.kv_heads;
  // Items are cut where they may be few (fewer than four a CTA: beyond, an uneven end is short beside
  // the whole) and long: more than 8 steps in all (one query, 32/8 heads of 128: 900 keys 18.9 us cut and 20.2
  // uncut, 1100 17.9 and 22.6, 8000 25 and 120), more than 4 on average. The average hides how uneven
  // the lengths are: four sequences of 64 queries lose up to 7 us behind 600 keys each (24.6 and 17.6), 4 behind
  // 800, nothing behind 1200, and gain 16 where one of them has 2000 and the others 100 (22.7 and 38.5). A part
  // costs its own start and end and 133 KB of partial results at 128 channels, so there are two for each
  // CTA at most.
  x.parts_max = x.most < 4ull * sms && p.total_k > 8 * 128 && p.total_k / p.n_seq > 4 * 128 ? most_parts(sms) : 0;
  return x;
}
}  // namespace

size_t attention_packed_workspace(const PackedAttention &p) {
  if (p.total_q == 0 || p.n_seq == 0) return 0;
  int dev = 0;
  cudaGetDevice(&dev);
  const uint32_t parts = items_of(p, static_cast<uint32_t>(sm_count(dev))).parts_max;
  if (parts == 0) return 0;
  return p.head_dim == 64 ? Parts<64>::bytes(parts) : Parts<128>::bytes(parts);
}

size_t attention_packed_workspace_bound(uint32_t head_dim) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint32_t parts = most_parts(static_cast<uint32_t>(sm_count(dev)));
  return head_dim == 64 ? Parts<64>::bytes(parts) : Parts<128>::bytes(parts);
}

cudaError_t launch_attention_packed(const PackedAttention &p, bool bf16, cudaStream_t stream,
                                    std::string *err) {
  if (p.total_q == 0 || p.n_seq == 0) return cudaSuccess;
  int dev = 0;
  cudaGetDevice(&dev);
  const uint32_t sms = static_cast<uint32_t>(sm_count(dev));
  const Items items = items_of(p, sms);
  const uint32_t group = p.q_heads / p.kv_heads, tokens = items.tokens;
  CUtensorMap q, k, v, o;
  const bool boxed = 32 % group == 0;
  constexpr uint32_t keys = Layout<64>::kKeys;
  static_assert(Layout<64>::kKeys == Layout<128>::kKeys, "one box");
  const bool maps =
      encode_map_rows(&q, p.q, bf16, p.head_dim, p.q_heads, p.total_q, p.q_head, p.q_token, group, tokens, err) &&
      // without keys the maps stand on q: no load reads through them
      encode_map_rows(&k, p.total_k ? p.k : p.q, bf16, p.head_dim, p.kv_heads, p.total_k ? p.total_k : 1, p.k_head,
                      p.k_token, 1, keys, err) &&
      encode_map_rows(&v, p.total_k ? p.v : p.q, bf16, p.head_dim, p.kv_heads, p.total_k ? p.total_k : 1, p.v_head,
                      p.v_token, 1, keys, err) &&
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
  a.parts_max = items.parts_max;
  a.workspace = p.workspace;
  a.flat = !items.parts_max && items.most <= sms;
  const uint32_t grid = items.parts_max || items.most > sms ? sms : static_cast<uint32_t>(items.most);
  if (p.head_dim == 64)
    return bf16 ? launch<true, 64>(q, k, v, o, a, dev, grid, stream) : launch<false, 64>(q, k, v, o, a, dev, grid, stream);
  return bf16 ? launch<true, 128>(q, k, v, o, a, dev, grid, stream) : launch<false, 128>(q, k, v, o, a, dev, grid, stream);
}

}  // namespace dv3
