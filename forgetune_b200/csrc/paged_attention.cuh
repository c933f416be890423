// Attention of new tokens over a paged cache on the tensor cores.
//
//   S = scale Q K^T (masked),  P = exp(S - m),  O = P V / sum P
//
// in one pass over the keys: a row keeps its reference m and its sum, and O
// lies in tensor memory.  m is raised (and O rescaled) only where a tile's
// largest weight would be above 2^7 times the reference's: any reference gives
// the same quotient, and weights up to 2^7 are as exact as weights up to 1.
// Scores, m, sums and O are fp32; a weight is rounded once, to the type of the
// values that the tensor cores multiply it by, while the sum takes it as it was.
//
// Rows.  The queries that share a kv head are the rows of one matrix, row r =
// (token r / G, head r % G), so that one token of G heads costs one row of
// loads, not G.  A unit of work is up to 256 rows of one sequence and kv head
// (two tiles of 128 that share every tile of keys and values), or, where the
// sequence has at most 128, all of its rows, with the tiles of keys going to
// the two halves of the block in turn and the halves joined at the end.
//
// Work.  Every unit's cost is a formula of its sequence's numbers, so each
// block sums them up and takes its equal share, from an offset in the middle
// of one unit to one in the middle of another: long contexts are split over
// blocks as finely as needed and short ones gathered, by the device's own
// numbers, without a plan from the host.  A block has at most two parts of
// units that others share; they go to the workspace (O, m and the sum), and
// paged_join_kernel joins them in order.  No atomics: the same bits each time.
//
// Block: twenty warps.
//   warps 0-7, 8-15  softmax of the two halves: a thread has 64 of a row's 128
//                    scores, the other 64 are four warps on.  S from tensor
//                    memory, mask, maximum (exchanged by the two), exponentials,
//                    P back over S as the A operand of P V; at the end O to
//                    global memory
//   warp 16          units of the block; keys and values by TMA, boxes of as
//                    many tokens as lie in one page, into a ring of tiles
//   warp 17          tensor memory and the products (one elected lane): while
//                    one half is in its softmax, the other's run
//   warps 18-19      Q of the next unit; tiles that some row sees in part:
//                    values outside of the unit's keys become 0, and so do
//                    values that are not finite (0 weights would make them
//                    NaN); rows that do see one get it added at the end
//
// Shared memory: Q of two tiles, and a ring of 128-token tiles of K or V,
// 128-byte swizzle, in columns of 64.  Tensor memory: S and P of both halves at
// [0, 256), O at [256, 512).
//
// What bounds it.  Few rows: the cache's bytes; a tile of 64 KB takes an SM 1.38
// us (47 GB/s, 7.0 TB/s over all).  Many rows: a pair of tiles takes 2.20 us, of
// which the tensor cores are busy 42 % and the exponentials' unit 42 % (prompt of
// 4096); neither is full because a half's next S waits for its P V, since P lies
// over S.  Tiles of 80 keys leave room for S beside P, and S and P V then had
// threads of their own; but an N = 80 product takes about 97 cycles (N = 128: 82), and
// 128 keys took 2.5 us.  A row's scores in one thread had spilled registers, for
// which 227 KB of shared memory leave little L1: 262 us for a prompt of 4096 where
// two threads a row took 218 (171 now).  A unit costs 4 to 4.5 us beside its
// tiles: Q, the first tile, the last P V and O (1480 units against 296: 6.7 us for
// each further unit of 256 rows and one tile, 5.4 for one of a single token).  A
// group that does not divide 128 has its Q by 16-byte copies, which the two warps
// wait for: 14 heads take 73 us where 16, with more work, take 61 (chunks of up to
// 1000 tokens, heads of 80).  Times of a graph of ten calls; calls for longer run
// at the power limit (a prompt of 8192 617 to 634 us, in a graph 561).
#pragma once

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "paged_rows.cuh"
#include "tc_ptx.cuh"

namespace ftb {

constexpr int kPagedThreads = 640;
constexpr int kPagedProducer = 16, kPagedProducts = 17, kPagedQueries = 18;  // warps
constexpr int kPagedTile = 128;      // keys of a tile, rows of a half
// A unit's own cost, in keys; twice that where it is all of a sequence's rows, whose keys cost less (160, 256, 512 and
// 700 for all: 64 sequences of one token 191, 184, 172 and 174 us, a prompt of 8192 586, 552, 562 and 573).
constexpr int kPagedUnitOver = 256;
constexpr int kPagedLeast = 512;     // keys (with it) that are worth a block
constexpr float kPagedRaise = 7.0f;  // log2
// The exponent score scale - m is one fused product, of which m is rounded: the difference of the largest score itself is
// up to half a step of float32 at m, from 2^28 on more than float16's weights hold and from 2^31 on more than any.  Rows
// whose m is beyond this round the product as m was, before the difference.  (A prompt of 8192 takes 617 us with it, 606
// without, and 650 with the scale in a register that such rows set to 1; out of line on tensor memory 618 to 643.)
__device__ __forceinline__ bool paged_far(float m) { return fabsf(m) > 16777216.0f && m != -INFINITY; }
// float16 weights are taken relative to 2^-7 of a row's reference (sums and O alike, so that the factor cancels): up to
// 2^15, below the largest number, and off by at most 2^-32 of the reference's where they are below the smallest normal
// number.  Relative to the reference itself, what lay 2^-25 below it became 0 in P V and counted in the sum: of 4096 keys
// 17.5 nats below one nothing was left, and 17 nats below came out 44 % too large.  bfloat16 has float32's exponents.
template <typename T>
constexpr float kPagedLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;  // log2
constexpr int kPagedBlocks = 148;    // at most: B200's SMs

// What the blocks leave for the join: for each block whose last unit others go on with.
struct PagedMeta {
  int open, last, kvh, r0, rows, tok0, pos0, pad;
};

struct PagedTensorParams {
  PagedAttentionParams a;
  int group;         // query heads of a kv head
  FastDiv by_group;
  int capacity;      // tokens that a row of the page table has places for
  int cost_shift, cost_step, cost_over, window_cap;  // see PagedCost
  int q_tma;         // Q has a TMA map: the group divides a tile's rows
  int box;           // tokens of a TMA box: in one page
  int negative;      // the scale is below 0 (a.scale is its absolute value)
  int rows_bound;    // rows of a part in the workspace
  PagedMeta* meta;   // [blocks]
  float* parts;      // [2 blocks][rows_bound] of (m, sum), then O [DH]
  int* err;
  int stall_test;    // failure-detection tests: the MMA warp first waits for what nothing completes
};

struct PagedUnit {
  int seq, kvh, r0, rows, tok0, pos0;
  int tb, te;          // tiles of keys of this part
  int lo, hi;          // keys that some row sees and the table has places for
  int first, last;     // positions of the first and the last row
  int alternate;       // the halves take the tiles in turn
  int count0, count1;  // tiles that the halves take
  int slot;            // part of the workspace, -1: the whole unit
  int done;
  volatile int bad;    // a page outside of the pool, in tiles that have come
  volatile int dirty;  // a value that is not finite in a tile seen in part
};

// Cost of the first n tiles of rows of a sequence, in keys (or, where the sum
// over all sequences might not fit 31 bits, in 2^cost_shift of them): tile i sees
// about base + step (i + 1) of them, at most `cap`.
struct PagedCost {
  int base, step, cap, over;
  __device__ __forceinline__ int first(int n) const {
    int k = n;  // about the tiles below the cap
    if (cap - base < step * n) k = cap <= base ? 0 : min(n, (int)__fdividef((float)(cap - base), (float)step));
    return k * base + step * (k * (k + 1) / 2) + (n - k) * cap + n * over;
  }
};

struct PagedSequence {
  int tok0, n, len, tiles;
  PagedCost cost;
  int head, whole;  // cost of a kv head, of all
};

__device__ __forceinline__ PagedSequence paged_sequence(const PagedTensorParams& p, int b) {
  const PagedBatchParams& t = p.a.batch;
  PagedSequence s;
  const int start = t.starts[b], stop = t.starts[b + 1];
  s.len = t.lengths[b];
  s.tok0 = max(0, min(start, p.a.tokens));
  s.n = max(0, min(stop, p.a.tokens) - s.tok0);
  // rows = n G below 2^27 2^12: tiles by the number of tokens
  s.tiles = s.n == 0 ? 0 : (int64_t)s.n * p.group <= kPagedTile ? 1 : (int)(((int64_t)s.n * p.group + 255) >> 8);
  const int len = max(0, min(s.len, p.capacity));
  s.cost.base = max(0, len - s.n) >> p.cost_shift;
  s.cost.step = p.cost_step;
  s.cost.cap = (p.a.window ? min(len, p.window_cap) : len) >> p.cost_shift;
  s.cost.over = s.tiles == 1 ? 2 * p.cost_over : p.cost_over;
  s.head = s.cost.first(s.tiles);
  s.whole = s.head * p.a.kv_heads;
  return s;
}

// A bounded wait by a whole warp, with one outcome.  The long form is apart: the roles are many and what they do
// between waits is short, so that instructions have to come from near (a prompt of 4096: 218 us with 129 KB of code,
// 171 with 78).
__device__ __noinline__ bool paged_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
  return mbar_wait_warp(bar, parity, abort_flag, err, code & 0xFF, (code & 0x100) != 0);
}
// ... by a thread for itself.
__device__ __noinline__ bool paged_wait_one_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
  return mbar_wait(bar, parity, abort_flag, err, code & 0xFF, (code & 0x100) != 0);
}
__device__ __forceinline__ bool paged_wait_one(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
  return mbar_try_wait(bar, parity) || paged_wait_one_long(bar, parity, abort_flag, err, code);
}
__device__ __forceinline__ bool paged_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return paged_wait_long(bar, parity, abort_flag, err, code);
}

template <int DH>
struct PagedSmem {
  static constexpr int HALVES = DH / 64;
  static constexpr int TILE = kPagedTile * DH * 2;
  static constexpr int STAGES = DH == 128 ? 5 : 10;
  static constexpr int Q_OFF = STAGES * TILE;
  static constexpr int ROW_OFF = Q_OFF + 2 * TILE;  // [16 softmax warps][32]: a row's maximum or sum
  static constexpr int UNIT_OFF = ROW_OFF + 16 * 32 * 4;
  static constexpr int UNITS = 4;
  static constexpr int BAR_OFF = (UNIT_OFF + UNITS * (int)sizeof(PagedUnit) + 15) / 16 * 16;
  static constexpr int NBAR = 2 * STAGES + 2 * UNITS + 2 + 2 * 4 + 13;
  static constexpr int TOTAL = BAR_OFF + 8 * NBAR + 16;
  static_assert(TOTAL <= 227 * 1024, "shared memory budget");
};

template <typename T>
__device__ __forceinline__ uint32_t paged_idesc(int n, bool b_by_rows) {
  constexpr uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | (b_by_rows ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kPagedTile >> 4) << 24);
}

// Operand tiles of 128-byte rows in the 128-byte swizzle, 8-row groups 1024
// bytes apart: K-major (Q, K: rows are M or N, 64 of the depth side by side) and
// MN-major (V: rows are the depth, 64 of N side by side, the next 64 a tile of
// 128 rows further).  The descriptor's upper word is the same for all; the lower has
// the address and `lead`, both in units of 16 bytes.
constexpr uint32_t kPagedDesc = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t paged_desc(uint32_t saddr, uint32_t lead) { return (saddr >> 4) | ((lead >> 4) << 16); }

__device__ __forceinline__ void umma_f16(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kPagedDesc)
      : "memory");
}
// A in tensor memory: a lane a row, eight columns 16 values of the depth
__device__ __forceinline__ void umma_f16_tmem_a(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kPagedDesc)
      : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

// Whether some row of the unit sees tile t in part.
__device__ __forceinline__ bool paged_masked(const PagedUnit& u, int t, int window) {
  return (t + 1) * kPagedTile > u.first + 1 || (window && t * kPagedTile <= u.last - window);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Top bit of each half of a word: an infinity or a NaN (the exponent's last bit
// carries into it; the other bits mean nothing).
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return std::is_same<T, __half>::value ? (w & 0x7C007C00u) + 0x04000400u : (w & 0x7F807F80u) + 0x00800080u;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
  const uint32_t m = not_finite<T>(w);
  return w & ~((m & 0x8000u ? 0xFFFFu : 0u) | (m & 0x80000000u ? 0xFFFF0000u : 0u));
}

// (x, y) = (x, y) a + b
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %2};\n\tmov.b64 r, {%3, %3};\n\t"
      "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// (x, y) += (a, b) f
__device__ __forceinline__ void fma2_to(float& x, float& y, float a, float b, float f) {
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %4};\n\t"
      "fma.rn.f32x2 p, q, r, p;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b), "f"(f));
}

// Transposes four pieces of four neighbouring lanes: lane l of them gets piece l of each, in order of the lanes.
__device__ __forceinline__ void swap_pieces(uint4& a, uint4& b, uint4& c, uint4& d, int lane) {
  auto swap = [&](uint4& x, uint4& y, int by) {  // lanes apart by `by`: the lower keeps x and gets the other's x as y
    const bool upper = lane & by;
    uint4 give = upper ? x : y;
    give.x = __shfl_xor_sync(0xffffffffu, give.x, by);
    give.y = __shfl_xor_sync(0xffffffffu, give.y, by);
    give.z = __shfl_xor_sync(0xffffffffu, give.z, by);
    give.w = __shfl_xor_sync(0xffffffffu, give.w, by);
    (upper ? x : y) = give;
  };
  swap(a, b, 1);
  swap(c, d, 1);
  swap(a, c, 2);
  swap(b, d, 2);
}

// Of 32 elements from c on of a row's output, a bit for each in which a value of
// a tile seen in part is +inf or -inf (NaN: both) and the row, at `position`,
// sees it.  Such values were left out of the products.
struct PagedMarks {
  uint32_t plus, minus;
};
template <typename T>
__device__ __forceinline__ PagedMarks paged_marks(const PagedTensorParams& p, const PagedUnit& u, int position, int c) {
  const PagedAttentionParams& a = p.a;
  PagedMarks bits{0, 0};
  const int64_t from = a.window ? (int64_t)position - a.window + 1 : 0;
  const int end = min(min(position + 1, u.hi), u.te * kPagedTile);  // within the table
#pragma unroll 1
  for (int key = (int)max((int64_t)u.tb * kPagedTile, from); key < end; ++key) {
    if (!paged_masked(u, key / kPagedTile, a.window)) continue;
    const int page = a.batch.page_table[u.seq * a.batch.table_ld + a.batch.by_page.of(key)];
    if (page < 0 || page >= a.batch.pages) continue;
    const T* x = static_cast<const T*>(a.values) + page * a.v_page + key % a.batch.page_size * a.v_token +
                 (int64_t)u.kvh * a.v_head + c;
#pragma unroll 1
    for (int k = 0; k < 32 && c + k < a.dim; ++k) {
      const float v = to_f32(x[k]);
      if (!(v < INFINITY)) bits.plus |= 1u << k;
      if (!(v > -INFINITY)) bits.minus |= 1u << k;
    }
  }
  return bits;
}

// Whether the row at `position` sees a key of this part whose page is outside of the pool.  By the table and not by what
// the block has come to: the answer is the same for any split and at any time.  (In a tile that other rows see in part
// such keys have a weight of 0 for the rows that do not see them, and finite values: cleaned.)
__device__ __forceinline__ bool paged_lost(const PagedTensorParams& p, const PagedUnit& u, int position) {
  const PagedAttentionParams& a = p.a;
  const int64_t from = a.window ? (int64_t)position - a.window + 1 : 0;
  const int end = min(min(position + 1, u.hi), u.te * kPagedTile);
#pragma unroll 1
  for (int64_t key = max((int64_t)u.tb * kPagedTile, from); key < end;) {
    const int n = a.batch.by_page.of((int)key), page = a.batch.page_table[u.seq * a.batch.table_ld + n];
    if (page < 0 || page >= a.batch.pages) return true;
    key = (int64_t)(n + 1) * a.batch.page_size;
  }
  return false;
}

template <typename T, int DH>
__global__ void __launch_bounds__(kPagedThreads, 1)
    paged_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const __grid_constant__ CUtensorMap map_q, const PagedTensorParams p) {
  using L = PagedSmem<DH>;
  constexpr int STAGES = L::STAGES, HALVES = L::HALVES, UNITS = L::UNITS;
  extern __shared__ __align__(1024) uint8_t paged_smem[];  // the swizzle's unit
  uint8_t* smem = paged_smem;
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, 40);
    return;
  }
  PagedUnit* units = reinterpret_cast<PagedUnit*>(smem + L::UNIT_OFF);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);  // a tile of K or V landed
  uint64_t* empty = full + STAGES;       // the products are done with it
  uint64_t* u_full = empty + STAGES;     // a unit is described
  uint64_t* u_empty = u_full + UNITS;    // every role is done with it
  uint64_t* q_full = u_empty + UNITS;    // its Q landed
  uint64_t* q_empty = q_full + 1;        // its last S = Q K^T is done
  uint64_t* s_full = q_empty + 1;        // [2] S of a half
  uint64_t* p_full = s_full + 2;         // [2] its P is in tensor memory, O rescaled
  uint64_t* pv_done = p_full + 2;        // [2] P V is done
  uint64_t* o_free = pv_done + 2;        // [2] O was read (in units where the half had tiles)
  uint64_t* v_seen = o_free + 2;         // a tile of V seen in part is there
  uint64_t* v_clean = v_seen + 1;        // ... and clean
  uint64_t* ml_full = v_clean + 1;       // m and sum of the second half
  uint64_t* ml_free = ml_full + 1;       // ... read
  uint64_t* pairs = ml_free + 1;         // [8] the two warps of 32 rows have met
  uint64_t* drain = pairs + 8;           // products retired after an abort
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(drain + 1) + 1;

  const PagedAttentionParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.group;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < UNITS; ++s) {
      mbar_init(&u_full[s], 1);
      mbar_init(&u_empty[s], 19);  // sixteen softmax warps, the products, two of Q
    }
    mbar_init(q_full, 2);
    mbar_init(q_empty, 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&p_full[w], 8);
      mbar_init(&pv_done[w], 1);
      mbar_init(&o_free[w], 8);
    }
    mbar_init(v_seen, 1);
    mbar_init(v_clean, 2);
    mbar_init(ml_full, 8);
    mbar_init(ml_free, 8);
    for (int s = 0; s < 8; ++s) mbar_init(&pairs[s], 2);
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kPagedProducts) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(const_cast<uint32_t*>(tmem_slot))),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kPagedQueries && elect_one()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dep_wait();
  grid_dep_trigger();
  // Costs of many sequences: each warp sums a run of them, in chunks of 32.
  const int chunks = (a.batch.seqs + 31) / 32, run = (chunks + kPagedThreads / 32 - 1) / (kPagedThreads / 32);
  int* warp_cost = reinterpret_cast<int*>(smem + L::ROW_OFF);
  if (chunks > 2) {
    int sum = 0;
#pragma unroll 1
    for (int c = warp * run; c < min(chunks, (warp + 1) * run); ++c)
      sum += c * 32 + lane < a.batch.seqs ? paged_sequence(p, c * 32 + lane).whole : 0;
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) warp_cost[warp] = sum;
    __syncthreads();
  }
  const uint32_t tmem = *tmem_slot;
  const uint32_t ring = smem_u32(smem), q_smem = smem_u32(smem + L::Q_OFF);

  if (warp == kPagedProducer) {
    // ---- units, keys and values ----
    bool ok = true;
    uint32_t it = 0, uc = 0;
    const PagedBatchParams& bt = a.batch;
    // all sequences' cost, then the sequence that this block's share begins in
    int total = 0, begin = 0, end = 0, share = 1, at = 0;  // at: offset of sequence seq
    int seq = 0;
#pragma unroll 1
    for (int pass = 0; pass < 2 && (pass == 0 || begin < end); ++pass) {
      int sum = 0, c = 0;
      if (chunks > 2) {
        const int mine = lane < kPagedThreads / 32 ? warp_cost[lane] : 0;
        int upto = mine;
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += o;
        }
        total = __shfl_sync(0xffffffffu, upto, 31);
        if (pass) {  // the run that `begin` lies in
          const int w = __ffs(__ballot_sync(0xffffffffu, upto > begin)) - 1;
          sum = __shfl_sync(0xffffffffu, upto - mine, max(w, 0));
          c = max(w, 0) * run;
        } else {
          c = chunks;
          sum = total;
        }
      }
#pragma unroll 1
      for (; c < chunks; ++c) {
        const int mine = c * 32 + lane < bt.seqs ? paged_sequence(p, c * 32 + lane).whole : 0;
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += o;
        }
        if (pass) {
          const uint32_t beyond = __ballot_sync(0xffffffffu, sum + upto > begin);
          if (beyond) {
            const int l = __ffs(beyond) - 1;
            seq = c * 32 + l;
            at = sum + __shfl_sync(0xffffffffu, upto - mine, l);
            break;
          }
        }
        sum += __shfl_sync(0xffffffffu, upto, 31);
      }
      if (pass == 0) {
        total = sum;
        const int blocks = max(1, min((int)gridDim.x, total / (p.cost_over * kPagedLeast / kPagedUnitOver)));
        share = total / blocks + 1;
        begin = min((int64_t)total, (int64_t)blockIdx.x * share);
        end = min((int64_t)total, (int64_t)begin + share);
      }
    }
    PagedMeta meta{};
    PagedSequence s{};
    bool known = false;  // s is sequence seq
    int now = begin;     // offset of the next part
    while (ok) {
      // the unit at `now`
      PagedUnit u{};
      u.done = 1;
      if (now < end) {
#pragma unroll 1
        while (!known || s.whole <= now - at) {
          if (known) {
            at += s.whole;
            ++seq;
          }
          if (seq >= bt.seqs) break;  // starts that fall may let the sum overflow
          s = paged_sequence(p, seq);
          known = true;
        }
        if (seq >= bt.seqs || s.head <= 0) {
          now = end;
          continue;
        }
        u.done = 0;
        u.seq = seq;
        int rest = now - at;
        u.kvh = min(rest / s.head, a.kv_heads - 1);
        rest -= u.kvh * s.head;
        int lo = 0, hi = s.tiles - 1;  // the tile of rows: first(i) <= rest < first(i + 1)
#pragma unroll 1
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (s.cost.first(mid) <= rest) lo = mid;
          else hi = mid - 1;
        }
        const int before = s.cost.first(lo), cost = s.cost.first(lo + 1) - before, u0 = now - (rest - before), u1 = u0 + cost;
        u.r0 = lo * 256;
        u.rows = (int)min((int64_t)256, (int64_t)s.n * G - u.r0);
        u.alternate = lo == 0 && u.rows <= kPagedTile;
        u.tok0 = s.tok0;
        u.pos0 = max(s.len, -(1 << 30)) - s.n;
        u.first = u.pos0 + p.by_group.of(u.r0);
        u.last = u.pos0 + p.by_group.of(u.r0 + u.rows - 1);
        u.hi = max(0, min(u.last + 1, p.capacity));
        u.lo = a.window ? (int)max((int64_t)0, (int64_t)u.first - a.window + 1) : 0;
        const int tb = u.lo / kPagedTile, n = max(0, (u.hi + kPagedTile - 1) / kPagedTile - tb);
        // where a share's border cuts the unit, the same for the blocks on either side; not within two tiles of its ends
        const float per = __fdividef((float)n, (float)cost);
        auto cut = [&](int x) {
          const int c = (int)((float)(x - u0) * per + 0.5f);
          return c < 2 ? 0 : n - c < 2 ? n : c;
        };
        const int c1 = now > u0 ? cut(now) : 0, c2 = u1 > end ? cut(end) : n;
        if (c1 == n && n > 0) {  // the block before took all of it
          now = min(u1, end);
          continue;
        }
        if (u1 > end && c2 == 0) {  // the block behind does
          u.done = 1;
        } else {
        u.tb = tb + c1;
          u.te = tb + c2;
          if (u.alternate) {
            u.count0 = (c2 - c1 + 1) >> 1;
            u.count1 = (c2 - c1) >> 1;
          } else {  // the first half's last row may see fewer
            const int seen = u.pos0 + p.by_group.of(u.r0 + min(u.rows, kPagedTile) - 1);
            u.count0 = max(0, min(u.te, seen < 0 ? 0 : seen / kPagedTile + 1) - u.tb);
            u.count1 = u.rows <= kPagedTile ? 0 : c2 - c1;
          }
          u.slot = c1 > 0 ? 2 * (int)blockIdx.x : c2 < n ? 2 * (int)blockIdx.x + 1 : -1;
          if (c1 == 0 && c2 < n) {
            int last = (u1 - 1) / share;
#pragma unroll 1
            while (cut(last * share) == n) --last;
            meta = PagedMeta{1, last, u.kvh, u.r0, u.rows, u.tok0, u.pos0, 0};
          }
        }
        now = min(u1, end);
      }
      const uint32_t us = uc % UNITS;
      if (!(ok = paged_wait(&u_empty[us], ((uc / UNITS) & 1u) ^ 1u, abort_flag, p.err, 41))) break;
      if (lane == 0) {
        PagedUnit& d = units[us];
        d.seq = u.seq, d.kvh = u.kvh, d.r0 = u.r0, d.rows = u.rows, d.tok0 = u.tok0, d.pos0 = u.pos0;
        d.first = u.first, d.last = u.last, d.count0 = u.count0, d.count1 = u.count1;
        d.tb = u.tb, d.te = u.te, d.lo = u.lo, d.hi = u.hi, d.alternate = u.alternate, d.slot = u.slot;
        d.done = u.done, d.bad = 0, d.dirty = 0;
        mbar_arrive(&u_full[us]);
      }
      __syncwarp();
      ++uc;
      if (u.done) break;
      // K and V in the order of their products: K0 [K(i + 1)] V(i) where the
      // halves alternate, K0 V(i) [K(i + 1)] where they share
      const int n = u.te - u.tb;
      const int* table = bt.page_table + u.seq * bt.table_ld;
      // number j of them: its tile, and this lane's key and page (-1: none wanted, -2: none there)
      auto tile_of = [&](int j) {
        if (j == 0) return 0;
        if (j == 2 * n - 1) return n - 1;
        return u.alternate && !(j & 1) ? j / 2 - 1 : u.alternate ? (j + 1) / 2 : j / 2;
      };
      auto key_of = [&](int j) { return (u.tb + tile_of(j)) * kPagedTile + lane * p.box; };
      auto page_of = [&](int j) {
        const int key = key_of(j);
        if (j >= 2 * n || lane * p.box >= kPagedTile || key >= u.hi || key + p.box <= u.lo) return -1;
        const int page = table[bt.by_page.of(key)];
        return page < 0 || page >= bt.pages ? -2 : page;
      };
      int ahead = page_of(0);
      for (int j = 0; j < 2 * n; ++j, ++it) {
        const bool is_v = j == 2 * n - 1 || (j > 0 && (u.alternate ? !(j & 1) : (j & 1)));
        const int key = key_of(j), page = ahead;
        ahead = page_of(j + 1);
        if (__any_sync(0xffffffffu, page == -2) && lane == 0) units[us].bad = 1;
        const uint32_t s = it % STAGES;
        if (!(ok = paged_wait(&empty[s], ((it / STAGES) & 1u) ^ 1u, abort_flag, p.err, 42))) break;
        const uint32_t boxes = (uint32_t)__popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) mbar_arrive_expect_tx(&full[s], boxes * (uint32_t)p.box * DH * 2);
        __syncwarp();
        if (page >= 0) {
          const CUtensorMap* map = is_v ? &map_v : &map_k;
          const uint32_t dst = ring + s * L::TILE + (uint32_t)(lane * p.box) * 128u;
          const int in = key - bt.by_page.of(key) * bt.page_size;
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
            tma_load_4d(dst + h * (kPagedTile * 128), map, h * 64, in, u.kvh, page, &full[s]);
        }
        __syncwarp();
      }
    }
    if (lane == 0) p.meta[blockIdx.x] = meta;
    if (!ok)  // the copies in flight land before the block leaves
      for (uint32_t j = it > STAGES ? it - STAGES : 0; j < it; ++j)
        paged_wait(&full[j % STAGES], (j / STAGES) & 1u, abort_flag, p.err, 0x100 | 43);
  } else if (warp == kPagedProducts) {
    // ---- products, by one thread ----
    if (elect_one()) {
      bool ok = true;
      uint32_t it = 0, uc = 0, vc = 0;
      uint32_t p_phase = 0, o_phase = 3u;  // a bit of each half
      const uint32_t idesc_s = paged_idesc<T>(kPagedTile, false), idesc_o = paged_idesc<T>((a.dim + 15) / 16 * 16, true);
      const int steps = (a.dim + 15) / 16;
      const uint32_t q_desc = paged_desc(q_smem, 16), k_desc = paged_desc(ring, 16), v_desc = paged_desc(ring, kPagedTile * 128);
      if (p.stall_test) ok = paged_wait_one(drain, 0, abort_flag, p.err, 44);
      while (ok) {
        const uint32_t us = uc % UNITS;
        if (!(ok = paged_wait_one(&u_full[us], (uc / UNITS) & 1u, abort_flag, p.err, 46))) break;
        const PagedUnit& u = units[us];
        if (u.done) break;
        const int n = u.te - u.tb, alternate = u.alternate, count0 = u.count0, count1 = u.count1;
        // tiles from here on are seen in part, and those before that
        const int masked_from = (u.first + 1) / kPagedTile - u.tb;
        const int masked_to = a.window ? (int)min((int64_t)n, ((int64_t)u.last - a.window + kPagedTile) / kPagedTile - u.tb) : 0;
        if (!(ok = paged_wait_one(q_full, uc & 1u, abort_flag, p.err, 47))) break;
        if (n == 0) umma_commit(q_empty);
        // Step q is P V of half w = q & 1 with its tile i, then its next S; the first
        // two are the halves' first S.  Tiles of the unit: i, or 2 i + w.
        int k_seen = 0, v_seen_to = 0;  // tiles of K and V that were waited for
#pragma unroll 1
        for (int q = -2; q < (alternate ? n : 2 * n) && ok; ++q) {
          const int w = q & 1, i = q >> 1, count = w ? count1 : count0;
          const int t = alternate ? q : i, ahead = t + (alternate ? 2 : 1);  // tile of P V, of the next S
          const bool last_of_tile = alternate || w == 1;
          if (q >= 0) {
            const uint32_t v = it + (alternate ? (t == n - 1 ? 2 * n - 1 : 2 * t + 2) : 2 * t + 1), s = v % STAGES;
            if (t >= v_seen_to) {
              v_seen_to = t + 1;
              if (!(ok = paged_wait_one(&full[s], (v / STAGES) & 1u, abort_flag, p.err, 45))) break;
              if (t >= masked_from || t < masked_to) {
                mbar_arrive(v_seen);
                if (!(ok = paged_wait_one(v_clean, vc & 1u, abort_flag, p.err, 48))) break;
                ++vc;
              }
            }
            if (i < count) {
              if (i == 0) {
                if (!(ok = paged_wait_one(&o_free[w], (o_phase >> w) & 1u, abort_flag, p.err, 49))) break;
                o_phase ^= 1u << w;
              }
              const uint32_t vs = v_desc + s * (L::TILE / 16), d = tmem + w * 128;
              if (!(ok = paged_wait_one(&p_full[w], (p_phase >> w) & 1u, abort_flag, p.err, 50))) break;
              p_phase ^= 1u << w;
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < kPagedTile / 16; ++k)
                umma_f16_tmem_a(d + 256, d + (k >> 2) * 64 + (k & 3) * 8, vs + k * (2048 / 16), idesc_o, i > 0 || k > 0 ? 1u : 0u);
              umma_commit(&pv_done[w]);
            }
            if (last_of_tile) umma_commit(&empty[s]);
          }
          if (ahead >= n) continue;
          const uint32_t k = it + (alternate ? (ahead == 0 ? 0 : 2 * ahead - 1) : 2 * ahead), s = k % STAGES;
          if (ahead >= k_seen) {
            k_seen = ahead + 1;
            if (!(ok = paged_wait_one(&full[s], (k / STAGES) & 1u, abort_flag, p.err, 45))) break;
          }
          if (i + 1 < count) {
            const uint32_t qs = q_desc + (alternate ? 0 : w * (L::TILE / 16)), ks = k_desc + s * (L::TILE / 16);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < DH / 16; ++c)
              if (c < steps)
                umma_f16(tmem + w * 128, qs + ((c >> 2) * (kPagedTile * 128) + (c & 3) * 32) / 16,
                         ks + ((c >> 2) * (kPagedTile * 128) + (c & 3) * 32) / 16, idesc_s, c > 0 ? 1u : 0u);
            umma_commit(&s_full[w]);
          }
          if (last_of_tile) {
            umma_commit(&empty[s]);
            if (ahead == n - 1) umma_commit(q_empty);
          }
        }
        if (!ok) break;
        it += 2 * n;
        mbar_arrive(&u_empty[us]);
        ++uc;
      }
      if (!ok) {
        umma_commit(drain);
        paged_wait_one(drain, 0, abort_flag, p.err, 0x100 | 52);
      }
    }
    __syncwarp();
  } else if (warp >= kPagedQueries) {
    // ---- Q, and values of tiles that are seen in part ----
    const int me = warp - kPagedQueries;
    bool ok = true;
    uint32_t it = 0, uc = 0, vc = 0, sent = 0;  // sent: Q on its way by TMA, of so many units
    while (ok) {
      const uint32_t us = uc % UNITS;
      if (!(ok = paged_wait(&u_full[us], (uc / UNITS) & 1u, abort_flag, p.err, 53))) break;
      PagedUnit& u = units[us];
      if (u.done) break;
      if (!(ok = paged_wait(q_empty, (uc & 1u) ^ 1u, abort_flag, p.err, 54))) break;
      if (p.q_tma) {  // G heads by 128 / G tokens: rows behind the unit's are other tokens', of which nothing is used
        sent = uc + 1;
        if (elect_one()) {
          const int tiles = u.rows > kPagedTile ? 2 : 1;
          if (me == 0) {
            mbar_arrive_expect_tx(q_full, (uint32_t)(tiles * L::TILE));
            const int per = kPagedTile / G, tok = u.tok0 + p.by_group.of(u.r0);
            for (int i = 0; i < tiles; ++i)
#pragma unroll
              for (int h = 0; h < HALVES; ++h)
                tma_load_4d(q_smem + i * L::TILE + h * (kPagedTile * 128), &map_q, h * 64, 0, tok + i * per, u.kvh, q_full);
          } else {
            mbar_arrive(q_full);
          }
        }
        __syncwarp();
      } else {
        constexpr int CH = DH / 8;  // 16-byte pieces of a row
        const int c = lane % CH, rows = u.rows;
        const T* q = static_cast<const T*>(a.q) + (int64_t)u.tok0 * a.q_token + (int64_t)u.kvh * G * a.q_head + c * 8;
#pragma unroll 2
        for (int r = me * (32 / CH) + lane / CH; r < rows; r += 2 * (32 / CH)) {
          const int row = u.r0 + r, tok = p.by_group.of(row), g = row - tok * G;
          const uint32_t dst = q_smem + (r >> 7) * L::TILE + (c >> 3) * (kPagedTile * 128) + (r & 127) * 128 +
                               (((c & 7) ^ (r & 7)) << 4);
          const bool real = c * 8 < a.dim;
          cp_async16(dst, real ? static_cast<const void*>(q + (int64_t)tok * a.q_token + (int64_t)g * a.q_head) : a.q, real);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        __syncwarp();
      }
      const int n = u.te - u.tb;
      for (int t = 0; t < n && ok; ++t) {
        if (!paged_masked(u, u.tb + t, a.window)) continue;
        const uint32_t v = it + (u.alternate ? (t == n - 1 ? 2 * n - 1 : 2 * t + 2) : 2 * t + 1), s = v % STAGES;
        // the products wait at this tile: it has landed, and stays until it is clean
        if (!(ok = paged_wait(v_seen, vc & 1u, abort_flag, p.err, 51))) break;
        ++vc;
        if (!(ok = paged_wait(&full[s], (v / STAGES) & 1u, abort_flag, p.err, 55))) break;
        const int key0 = (u.tb + t) * kPagedTile;
        constexpr int CH = DH / 8;
        uint8_t* tile = smem + s * L::TILE;
        auto piece = [&](int row, int c) { return reinterpret_cast<uint4*>(tile + (c >> 3) * (kPagedTile * 128) + row * 128 + (c & 7) * 16); };
        const int c = lane % CH, r_first = me * (32 / CH) + lane / CH;
        constexpr int STEP = 2 * (32 / CH);
        // keys outside of the unit's
#pragma unroll 1
        for (int row = r_first; row < min(kPagedTile, u.lo - key0); row += STEP) *piece(row, c) = make_uint4(0, 0, 0, 0);
#pragma unroll 2
        for (int row = max(r_first, r_first + (u.hi - key0 - r_first + STEP - 1) / STEP * STEP); row < kPagedTile; row += STEP)
          *piece(row, c) = make_uint4(0, 0, 0, 0);
        // keys that some rows see and others do not: the last ones, and those before the last row's window
        uint32_t found = 0;
        const int late = u.first + 1 - key0;
#pragma unroll 1
        for (int part = a.window ? 0 : 1; part < 2; ++part) {
          const int from = max(part ? late : 0, max(0, u.lo - key0));
          const int to = min(part ? kPagedTile : (int)min((int64_t)late, (int64_t)u.last - a.window - key0 + 1),
                             min(kPagedTile, u.hi - key0));
#pragma unroll 1
          for (int row0 = from + r_first; row0 < to; row0 += 4 * STEP) {
            uint4 x[4];
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x[i] = row0 + i * STEP < to ? *piece(row0 + i * STEP, c) : make_uint4(0, 0, 0, 0);
              any |= not_finite<T>(x[i].x) | not_finite<T>(x[i].y) | not_finite<T>(x[i].z) | not_finite<T>(x[i].w);
            }
            if (!(any & 0x80008000u)) continue;
            found = 1;
#pragma unroll 1
            for (int row = row0; row < min(to, row0 + 4 * STEP); row += STEP) {
              const uint4 w = *piece(row, c);
              *piece(row, c) = make_uint4(finite_or_zero<T>(w.x), finite_or_zero<T>(w.y), finite_or_zero<T>(w.z), finite_or_zero<T>(w.w));
            }
          }
        }
        if (found) u.dirty = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_clean);
        __syncwarp();
      }
      it += 2 * n;
      if (!ok) break;
      if (lane == 0) mbar_arrive(&u_empty[us]);
      __syncwarp();
      ++uc;
    }
    if (!ok && sent > 0 && me == 0) paged_wait(q_full, (sent - 1) & 1u, abort_flag, p.err, 0x100 | 54);  // it lands before the block leaves
  } else {
    // ---- softmax ----
    const int w = warp >> 3, side = (warp >> 2) & 1, quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tmem = tmem + w * 128 + lanes;
    // the warp with the other scores of the same rows, and where the two leave theirs
    float* rows = reinterpret_cast<float*>(smem + L::ROW_OFF) + lane;
    // What the two warps of a row have, for both.  A place is written again only when its
    // reader is known to be past this: behind a meeting of theirs or the next S.  Meetings
    // are bounded waits too: one warp may have given up where the other went on.
    uint64_t* pair = pairs + w * 4 + quarter;
    uint32_t met = 0;
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(pair);
      __syncwarp();
      const bool both_here = paged_wait(pair, met & 1u, abort_flag, p.err, 62);
      ++met;
      return both_here;
    };
    auto exchange = [&](float x, float* y) {
      rows[warp * 32] = x;
      const bool both_here = meet();
      *y = rows[(warp ^ 4) * 32];
      return both_here;
    };
    bool ok = true;
    uint32_t uc = 0, cnt0 = 0, cnt1 = 0, mc = 0;
    while (ok) {
      const uint32_t us = uc % UNITS;
      if (!(ok = paged_wait(&u_full[us], (uc / UNITS) & 1u, abort_flag, p.err, 56))) break;
      const PagedUnit& u = units[us];
      if (u.done) break;
      const int alternate = u.alternate, tb = u.tb;
      const int count0 = u.count0, count1 = u.count1, count = w ? count1 : count0;
      const uint32_t done = w ? cnt1 : cnt0;  // tiles of this half so far
      const int r = (alternate ? 0 : w * kPagedTile) + quarter * 32 + lane;  // row of the unit
      const bool real = r < u.rows, active = (alternate ? 0 : w * kPagedTile) + quarter * 32 < u.rows;
      const int tok = p.by_group.of(u.r0 + r), position = u.pos0 + tok;
      float m = -INFINITY, sum = 0.0f;
      bool far = false;  // some row's m is far
      for (int i = 0; i < count && ok; ++i) {
        const int t = tb + (alternate ? 2 * i + w : i);
        if (!(ok = paged_wait(&s_full[w], (done + i) & 1u, abort_flag, p.err, 57))) break;
        tc_fence_after();
        if (active) {
          // columns that this row sees: low < column <= high
          const int high = position - t * kPagedTile - side * 64;
          const int low = a.window ? (int)max((int64_t)high - a.window, (int64_t)-1) : -1;
          const bool partly = __any_sync(0xffffffffu, real && (high < 63 || low >= 0));
          // The second 32 of the thread's scores, the first, and the second again: all 64 and what else a thread
          // keeps do not fit its registers, and what is spilled goes to L2.  P of 32 goes over the first 16 columns
          // of the scores, when both are done with.
          float high_s = -INFINITY, base = 0.0f, part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll  // rolled up: 578 us for a prompt of 8192 where it took 545
          for (int pass = 0; pass < 3; ++pass) {
            const int c = (pass & 1) ^ 1;
            uint32_t x[32];
            __syncwarp();
            FTB_TMEM_LD32(s_tmem + side * 64 + c * 32, x);
            FTB_TMEM_WAIT_LD32(x);
            if (p.negative) {
#pragma unroll
              for (int k = 0; k < 32; ++k) x[k] ^= 0x80000000u;
            }
            if (partly) {
              const int h = min(high - c * 32, 31), l = max(low - c * 32, -1);
              const uint32_t seen = h < 0 || l > 30 ? 0u : (0xFFFFFFFFu >> (31 - h)) & (0xFFFFFFFFu << (l + 1));
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!(seen & (1u << k))) x[k] = 0xFF800000u;
            }
            if (pass < 2) {
              float top[2];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                top[k] = fmaxf(__uint_as_float(x[16 * k]), __uint_as_float(x[16 * k + 1]));
#pragma unroll
                for (int e = 2; e < 16; e += 2)
                  top[k] = max3(top[k], __uint_as_float(x[16 * k + e]), __uint_as_float(x[16 * k + e + 1]));
              }
              high_s = max3(high_s, top[0], top[1]);
            }
            if (pass == 0) continue;
            if (pass == 1) {
              float other;
              if (!(ok = exchange(high_s, &other))) break;
              high_s = fmaxf(high_s, other) * a.scale;
              const bool raise = real && high_s - m > kPagedRaise;  // (their sum might round up to high_s)
              if (__any_sync(0xffffffffu, raise)) {
                float keep = 1.0f;
                if (raise) {
                  keep = ex2(m - high_s);
                  sum *= keep;
                  m = high_s;
                }
                far = __any_sync(0xffffffffu, paged_far(m));
                // this S followed the last P V, so O is complete; each of a row's warps has half of its columns
#pragma unroll 1
                for (int d = i > 0 ? side * (DH / 2) : a.dim; d < (side + 1) * (DH / 2) && d < a.dim; d += 16) {
                  uint32_t o[16];
                  __syncwarp();
                  FTB_TMEM_LD16(tmem + 256 + w * 128 + lanes + d, o);
#pragma unroll
                  for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                  FTB_TMEM_ST16(tmem + 256 + w * 128 + lanes + d, o);
                }
              }
              base = m == -INFINITY ? 0.0f : m - kPagedLift<T>;
            }
            if (far) [[unlikely]] {
              if (paged_far(m)) {  // of this row alone: other rows' scores do not change its bits
                const float back = __frcp_rn(a.scale);
                base = -kPagedLift<T>;
#pragma unroll
                for (int k = 0; k < 32; ++k)  // (a packed product and sum were made one operation again)
                  x[k] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(x[k]), a.scale), m) * back);
              }
              __syncwarp();
            }
            uint32_t o[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float u = __uint_as_float(x[2 * k]), v = __uint_as_float(x[2 * k + 1]);
              fma2(u, v, a.scale, -base);
              u = ex2(u);
              v = ex2(v);
              add2(part[2 * (k & 1)], part[2 * (k & 1) + 1], u, v);
              o[k] = pack2<T>(u, v);
            }
            FTB_TMEM_ST16(s_tmem + side * 64 + c * 16, o);
          }
          if (!ok) break;
          sum += (part[0] + part[1]) + (part[2] + part[3]);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[w]);
        __syncwarp();
      }
      if (!ok) break;
      // ---- O ----
      cnt0 += count0;
      cnt1 += count1;
      const bool both = alternate && count0 > 0, mine = !alternate || w == 0;
      float f0 = 1.0f, f1 = 1.0f;  // factors of the halves' O
      if (count > 0) {
        if (!(ok = paged_wait(&pv_done[w], (done + count - 1) & 1u, abort_flag, p.err, 60))) break;
        float other;
        if (!(ok = exchange(sum, &other))) break;
        sum += other;
        if (!(ok = meet())) break;
      }
      if (both && w == 1) {
        rows[warp * 32] = side ? sum : m;
        __syncwarp();
        if (lane == 0) mbar_arrive(ml_full);
        __syncwarp();
        if (!(ok = paged_wait(ml_free, mc & 1u, abort_flag, p.err, 61))) break;
      }
      if (both && w == 0) {
        if (!(ok = paged_wait(ml_full, mc & 1u, abort_flag, p.err, 59))) break;
        const float m1 = rows[(8 + quarter) * 32], sum1 = rows[(12 + quarter) * 32];
        __syncwarp();
        if (lane == 0) mbar_arrive(ml_free);
        __syncwarp();
        const float top = fmaxf(m, m1), base = top == -INFINITY ? 0.0f : top;
        f0 = ex2(m - base);
        f1 = ex2(m1 - base);
        sum = sum * f0 + sum1 * f1;
        m = top;
      }
      if (both) ++mc;
      if (mine) {
        if (both && count1 > 0 && !(ok = paged_wait(&pv_done[1], (cnt1 - 1) & 1u, abort_flag, p.err, 63))) break;
        tc_fence_after();
        const bool dirty = u.dirty, bad = position >= p.capacity || (u.bad && real && paged_lost(p, u, position));
        const int g = u.r0 + r - tok * G;
        // a part of the workspace: (m, sum) of each row, then O in quads of columns, each of them of all rows
        float* part = p.parts + (int64_t)max(u.slot, 0) * p.rows_bound * (2 + DH);
        if (u.slot >= 0 && real && side == 0) *reinterpret_cast<float2*>(part + 2 * r) = make_float2(m, bad ? NAN : sum);
        const float by = u.slot >= 0 ? 1.0f : bad ? NAN : position < 0 ? 0.0f : 1.0f / sum;
        f0 *= by;
        f1 *= by;
        const int64_t out = (int64_t)(u.tok0 + tok) * a.o_token + (int64_t)(u.kvh * G + g) * a.o_head;
        if (active) {
#pragma unroll 1
          for (int c = side * (DH / 2); c < (side + 1) * (DH / 2) && c < a.dim; c += 32) {
            float v[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = by != by ? NAN : 0.0f;
#pragma unroll 1
            for (int h = both ? 0 : w; h < (both ? 2 : w + 1); ++h) {
              if ((h ? count1 : count0) == 0) continue;
              const float f = h && both ? f1 : f0;
              uint32_t o[32];
              __syncwarp();
              FTB_TMEM_LD32(tmem + 256 + h * 128 + lanes + c, o);
              FTB_TMEM_WAIT_LD32(o);
#pragma unroll
              for (int k = 0; k < 32; k += 2) fma2_to(v[k], v[k + 1], __uint_as_float(o[k]), __uint_as_float(o[k + 1]), f);
            }
            if (dirty && real) {
              const PagedMarks bits = paged_marks<T>(p, u, position, c);
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                if (bits.plus & (1u << k)) v[k] += INFINITY;
                if (bits.minus & (1u << k)) v[k] -= INFINITY;
              }
            }
            if (u.slot >= 0) {
              if (real) {
#pragma unroll
                for (int k = 0; k < 32; k += 4)
                  *reinterpret_cast<float4*>(part + 2 * p.rows_bound + ((int64_t)((c + k) / 4) * p.rows_bound + r) * 4) =
                      make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
              }
              continue;
            }
            // Four lanes exchange the 16-byte pieces of their rows, so that they store 64 bytes of one row at a time:
            // a store of 32 rows takes as many turns of the memory pipe as it has lines.
            uint4 o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              o[k] = make_uint4(pack2<T>(v[8 * k], v[8 * k + 1]), pack2<T>(v[8 * k + 2], v[8 * k + 3]),
                                pack2<T>(v[8 * k + 4], v[8 * k + 5]), pack2<T>(v[8 * k + 6], v[8 * k + 7]));
            swap_pieces(o[0], o[1], o[2], o[3], lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // row 4 (lane / 4) + k, piece lane % 4
              const int64_t to = __shfl_sync(0xffffffffu, real ? out : (int64_t)-1, (lane & 28) + k);
              const int e = c + 8 * (lane & 3);
              if (to >= 0 && e < a.dim) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + to + e) = o[k];
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          for (int h = 0; h < 2; ++h)
            if ((both || h == w) && (h ? count1 : count0) > 0) mbar_arrive(&o_free[h]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&u_empty[us]);
      __syncwarp();
      ++uc;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kPagedProducts) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// Units that several blocks worked on: block x of the grid joins the one that
// block x of paged_attention_kernel began and did not finish; a thread has four
// columns of a row, the rows side by side.
// O = sum_k O_k 2^(m_k - m) / sum_k sum_k 2^(m_k - m), parts in order.
constexpr int kPagedJoinThreads = 256;

template <typename T, int DH>
__global__ void __launch_bounds__(kPagedJoinThreads) paged_join_kernel(const PagedTensorParams p) {
  grid_dep_wait();
  grid_dep_trigger();
  const PagedMeta u = p.meta[blockIdx.x];
  if (!u.open) return;
  const PagedAttentionParams& a = p.a;
  const int rows = min(32, p.rows_bound), at = (int)(blockIdx.y * kPagedJoinThreads + threadIdx.x);
  const int r = at % rows + at / (rows * (DH / 4)) * 32, quad = at / rows % (DH / 4);
  if (r >= u.rows || 4 * quad >= a.dim) return;
  const int parts = u.last - (int)blockIdx.x + 1;
  const int64_t stride = (int64_t)p.rows_bound * (2 + DH);
  auto part = [&](int k) { return p.parts + (k == 0 ? 2 * (int64_t)blockIdx.x + 1 : 2 * ((int64_t)blockIdx.x + k)) * stride; };
  float m = -INFINITY, sum = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int k = 0; k < parts; ++k) {
    const float2 x = *reinterpret_cast<const float2*>(part(k) + 2 * r);
    const float4 v = *reinterpret_cast<const float4*>(part(k) + 2 * p.rows_bound + ((int64_t)quad * p.rows_bound + r) * 4);
    const float top = fmaxf(m, x.x), base = top == -INFINITY ? 0.0f : top, f = ex2(m - base), g = ex2(x.x - base);
    m = top;
    sum = sum * f + x.y * g;
    o.x = o.x * f + v.x * g;
    o.y = o.y * f + v.y * g;
    o.z = o.z * f + v.z * g;
    o.w = o.w * f + v.w * g;
  }
  const int tok = p.by_group.of(u.r0 + r), g = u.r0 + r - tok * p.group;
  const float by = 1.0f / sum;
  if (u.pos0 + tok < 0) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  else o = make_float4(o.x * by, o.y * by, o.z * by, o.w * by);
  T* out = static_cast<T*>(a.out) + (int64_t)(u.tok0 + tok) * a.o_token + (int64_t)(u.kvh * p.group + g) * a.o_head + 4 * quad;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(o.x, o.y), pack2<T>(o.z, o.w));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Heads as the kernel reads them: [n3][n2][n1][dim] with strides in elements, in boxes of 64 elements by b1 by b2.
inline bool make_map_heads(CUtensorMap* map, const void* base, int type, int64_t dim, int64_t n1, int64_t n2, int64_t n3,
                           int64_t s1, int64_t s2, int64_t s3, int b1, int b2) {
  PFN_encodeTiled enc = tma_encoder();
  if (!enc) return false;
  auto bytes = [&](int64_t n, int64_t stride) { return (cuuint64_t)(n > 1 ? stride * 2 : (dim * 2 + 15) / 16 * 16); };
  cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)n1, (cuuint64_t)n2, (cuuint64_t)n3};
  cuuint64_t strides[3] = {bytes(n1, s1), bytes(n2, s2), bytes(n3, s3)};
  cuuint32_t boxes[4] = {64, (cuuint32_t)b1, (cuuint32_t)b2, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(map, type == FTB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
             const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether the tensor-core kernel takes a call: 16-bit types, heads of up to 128
// in eights, pages of whole 16 tokens, and 16-byte boundaries throughout.  (A
// pool that repeats itself, with strides of 0, has no TMA map.)
inline bool paged_on_tensor_cores(const PagedAttentionParams& p, int type) {
  if (type == FTB_F32 || p.dim > 128 || p.dim % 8 || p.batch.page_size % 16) return false;
  for (const void* x : {p.q, (const void*)p.out, p.keys, p.values})
    if (reinterpret_cast<uintptr_t>(x) & 15) return false;
  for (int64_t s : {p.q_token, p.q_head, p.o_token, p.o_head, p.k_page, p.k_token, p.k_head, p.v_page, p.v_token, p.v_head})
    if (s % 8) return false;
  if ((p.batch.pages > 1 && !(p.k_page && p.v_page)) || (p.batch.page_size > 1 && !(p.k_token && p.v_token)) ||
      (p.kv_heads > 1 && !(p.k_head && p.v_head)))
    return false;
  return true;
}

inline int paged_rows_bound(const PagedAttentionParams& p) {
  return (int)std::min<int64_t>(256, ((int64_t)p.tokens * (p.heads / p.kv_heads) + 3) / 4 * 4);
}
constexpr int64_t kPagedMetaBytes = (int64_t)kPagedBlocks * (int64_t)sizeof(PagedMeta);
inline int64_t paged_workspace(const PagedAttentionParams& p) {
  return kPagedMetaBytes + 2 * (int64_t)kPagedBlocks * paged_rows_bound(p) * (2 + (p.dim <= 64 ? 64 : 128)) * 4;
}

inline cudaError_t paged_attention_prepare() {
  cudaError_t e = cudaSuccess;
  auto set = [&](auto kernel, int bytes) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  };
  set(paged_attention_kernel<__half, 64>, PagedSmem<64>::TOTAL);
  set(paged_attention_kernel<__half, 128>, PagedSmem<128>::TOTAL);
  set(paged_attention_kernel<__nv_bfloat16, 64>, PagedSmem<64>::TOTAL);
  set(paged_attention_kernel<__nv_bfloat16, 128>, PagedSmem<128>::TOTAL);
  return e;
}

template <typename T, int DH>
cudaError_t launch_paged_as(PagedTensorParams& p, int type, int blocks, cudaStream_t s) {
  const PagedAttentionParams& a = p.a;
  CUtensorMap map_k, map_v, map_q;
  // tokens of a page, kv heads, pages
  if (!make_map_heads(&map_k, a.keys, type, a.dim, a.batch.page_size, a.kv_heads, a.batch.pages, a.k_token, a.k_head,
                      a.k_page, p.box, 1) ||
      !make_map_heads(&map_v, a.values, type, a.dim, a.batch.page_size, a.kv_heads, a.batch.pages, a.v_token, a.v_head,
                      a.v_page, p.box, 1))
    return cudaErrorInvalidValue;
  // heads of a group, tokens, groups
  std::memset(&map_q, 0, sizeof(map_q));
  p.q_tma = kPagedTile % p.group == 0 &&
            make_map_heads(&map_q, a.q, type, a.dim, p.group, a.tokens, a.kv_heads, a.q_head, a.q_token, a.q_head * p.group,
                           p.group, kPagedTile / p.group);
  cudaError_t e = pdl_launch(paged_attention_kernel<T, DH>, dim3((unsigned)blocks), dim3(kPagedThreads), PagedSmem<DH>::TOTAL, s,
                             map_k, map_v, map_q, p);
  if (e == cudaSuccess) {
    const int rows = std::min(32, p.rows_bound), threads = (p.rows_bound + rows - 1) / rows * rows * (DH / 4);
    e = pdl_launch(paged_join_kernel<T, DH>, dim3((unsigned)blocks, (unsigned)((threads + kPagedJoinThreads - 1) / kPagedJoinThreads)),
                   dim3(kPagedJoinThreads), 0, s, p);
  }
  return e;
}

inline cudaError_t launch_paged_attention(const PagedAttentionParams& a, int type, void* workspace, int sm_count, int* err,
                                          int stall, cudaStream_t s) {
  const int blocks = std::min(sm_count, kPagedBlocks);
  PagedTensorParams p{};
  p.a = a;
  p.a.scale = std::fabs(a.scale);
  if (p.a.scale == 0.0f) p.a.scale = 1e-30f;  // equal weights either way, and a masked score stays -inf
  p.negative = a.scale < 0.0f;
  p.group = a.heads / a.kv_heads;
  p.by_group = FastDiv((uint32_t)p.group);
  // the largest sum of costs that tokens and page table allow fits 31 bits
  p.capacity = (int)std::min<int64_t>((int64_t)a.batch.most_pages * a.batch.page_size, 0x7fffffff);
  const int step = std::max(1, 256 / p.group);
  const double tiles = (double)a.kv_heads * ((double)a.tokens * p.group / 256 + std::min(a.batch.seqs, a.tokens));
  const double most = a.window ? std::min<double>(p.capacity, (double)a.window + step) : p.capacity;
  while (tiles * (most / (1 << p.cost_shift) + 2 * std::max(1, kPagedUnitOver >> p.cost_shift) + 1) > 0x3fffffff && p.cost_shift < 20)
    ++p.cost_shift;
  p.cost_step = step >> p.cost_shift;
  p.cost_over = std::max(1, kPagedUnitOver >> p.cost_shift);
  p.window_cap = (int)std::min<int64_t>((int64_t)a.window + step, 0x7fffffff);
  p.box = 16;
  while (p.box < kPagedTile && a.batch.page_size % (2 * p.box) == 0) p.box *= 2;
  p.rows_bound = paged_rows_bound(a);
  p.meta = static_cast<PagedMeta*>(workspace);
  p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + kPagedMetaBytes);
  p.err = err;
  p.stall_test = stall;
  if (type == FTB_F16) return a.dim <= 64 ? launch_paged_as<__half, 64>(p, type, blocks, s) : launch_paged_as<__half, 128>(p, type, blocks, s);
  return a.dim <= 64 ? launch_paged_as<__nv_bfloat16, 64>(p, type, blocks, s) : launch_paged_as<__nv_bfloat16, 128>(p, type, blocks, s);
}

}  // namespace ftb
