// Block-scaled 8-bit matrix product on SM pairs, for many tokens: the
// arithmetic of fp8_gemm.cuh on 256 x 256 tiles (tcgen05 cta_group::2).
//
// CTA r of a pair holds token rows [128 r, 128 r + 128) and weight rows
// [128 r, 128 r + 128) of the tile, so each SM loads 32 KB per k-block of 128
// for 128 x 256 x 128 products, half of what two separate 128 x 256 tiles
// would load; its tensor memory receives its 128 token rows.  Both CTAs need
// the scales of their own tokens and of all 256 outputs.
//
// Tensor memory: accumulators at columns [0, 256) and [224, 480), scale
// factors at [480, 512).  The two accumulators share columns 224 .. 255, so
// that both fit beside the scale factors: the epilogue reads the shared
// columns of a tile first, and the next tile's products wait for that alone.
//
// Persistent pairs walk the tiles in bands of 16 row blocks (74 pairs at work
// then share 16 + 5 operand blocks of 256 rows through L2, not 2 + 37;
// 8192^3: 385 us, with bands of 8 390, of 4 401).
// Warps per CTA:
//   warp 0     TMA producer of this CTA's rows (its own barriers);
//   warp 1     tensor memory; in the leader CTA the MMAs of the pair;
//   warp 2     scale factors of this CTA, four k-blocks at a time;
//   warp 3     passes this CTA's landed stages on to the leader;
//   warps 4-19 epilogue: a lane quarter and 64 columns each; a lane is a token.
//              32 columns at a time go out through the warp's box in shared
//              memory and a TMA store, or by rows where the output's rows are
//              not 16-byte aligned or the box ends outside; the residual comes
//              in through the same box.  Bias is staged while the products
//              run.  For a quantised output the two warps of a block of 128
//              columns exchange each token's largest value; the 64 values that
//              a lane holds meanwhile spill 66 bytes at 96 registers.
// Short depths are bound by the epilogue, its instructions and its turns
// through the box: 8192 x 8192 outputs of depth 64 take 36 us in bf16, 50 in
// f32, 43 quantised, 61 with a bf16 residual (floors by bytes 21, 41, 10 and
// 41 us; with 8 warps of 128 columns 48, 64, 57 and 79).  Long depths are bound
// by the operands' way through L2 and by power: 8192^3 takes 388 us in a burst,
// 454 when repeated for seconds at the 1 kW limit (314 in a burst without
// loads and stores).
#pragma once

#include "fp8_gemm.cuh"

namespace ftb {

constexpr int kFp8Band = 16;

constexpr int kFp8EpiWarps = 16;
constexpr int kFp8EpiColumns = 64;  // of an epilogue warp

struct Fp8PairShape {
  static constexpr int THREADS = 128 + 32 * kFp8EpiWarps;
  static constexpr int STAGES = 5;
  static constexpr int OPERAND_BYTES = 128 * 128;
  static constexpr int STAGE_BYTES = 2 * OPERAND_BYTES;
  static constexpr int SF_BYTES = 512 + 1024;
  static constexpr int BOXES = kFp8EpiWarps * 2048;
  static constexpr int BIAS_OFF = STAGES * STAGE_BYTES + BOXES;
  static constexpr int AMAX_OFF = BIAS_OFF + kFp8EpiWarps * kFp8EpiColumns * 4;
  static constexpr int SF_OFF = AMAX_OFF + 2 * kFp8EpiWarps * 32 * 4;  // of two tiles
  static constexpr int BAR_OFF = SF_OFF + 2 * SF_BYTES;
  static constexpr int NBAR = 3 * STAGES + 4 + 4 + 2 + 2 * kFp8EpiWarps;
  static constexpr int TOTAL = 1024 + BAR_OFF + 8 * NBAR + 16;
  static_assert(TOTAL <= 227 * 1024, "shared memory budget");
};

struct Fp8PairParams {
  Fp8Params p;
  int y_tma;     // the output has a TMA map
  int res_tma;   // the residual has one
  int bias_vec;  // bias is 16-byte aligned
};

__device__ __forceinline__ void umma2_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
      : "memory");
}

// In both CTAs: 512 bytes of this CTA's scale factors into its tensor memory.
__device__ __forceinline__ void tmem2_copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

__device__ __forceinline__ void tma_load_2d_at(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int c0, int c1, uint32_t smem) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(smem)
               : "memory");
}

// Tile number -> token and output block, in bands of kFp8Band token blocks.
struct Fp8Tiles {
  int tm, tn;
  __device__ __forceinline__ void at(int t, int& m0, int& n0) const {
    const int band = t / (kFp8Band * tn), in = t - band * kFp8Band * tn;
    const int h = min(kFp8Band, tm - band * kFp8Band);
    m0 = (band * kFp8Band + in % h) * 256;
    n0 = in / h * 256;
  }
};

__device__ __forceinline__ uint4 ld_shared4(uint32_t addr) {
  uint4 u;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(addr));
  return u;
}

// Max that keeps NaN: ReLU in one instruction.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 16-byte piece `i` of this lane's row in a box of 32 rows x 64 bytes, 64-byte
// swizzle.
__device__ __forceinline__ uint32_t box_at(uint32_t box, int lane, int i) {
  return box + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4);
}

// A box from or to a matrix without TMA: its rows are not 16-byte aligned, or
// the box reaches past the last column (a TMA store clips columns in units of
// 16 bytes only).  Lanes take consecutive columns of a row.
template <typename U>
__device__ __noinline__ void load_box_rows(uint32_t box, const U* x, int64_t ld, int m0, int n, int M, int N,
                                              int lane) {
  constexpr int E = (int)sizeof(U), C = 64 / E, R = 32 / C, B = 8;  // R rows at a time, B times in flight
  const int c = lane % C;
  const U* src = x + (int64_t)(m0 + lane / C) * ld + n + c;
  for (int r0 = lane / C; r0 < 32; r0 += R * B) {
    U u[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      u[i] = m0 + r0 + i * R < M && n + c < N ? *src : (U)0;
      src += R * ld;
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const uint32_t at = box_at(box, r0 + i * R, (c * E) >> 4) + ((c * E) & 15);
      if constexpr (E == 4) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(u[i]) : "memory");
      else asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(u[i]) : "memory");
    }
  }
  __syncwarp();
}

template <typename U>
__device__ __noinline__ void store_box_rows(uint32_t box, U* y, int64_t ld, int m0, int n, int M, int N, int lane) {
  constexpr int E = (int)sizeof(U), C = E == 1 ? 32 : 64 / E, R = 32 / C, B = 8;
  __syncwarp();
#pragma unroll
  for (int c0 = 0; c0 < 64 / E; c0 += C) {
    const int c = c0 + lane % C;
    U* dst = y + (int64_t)(m0 + lane / C) * ld + n + c;
    for (int r0 = lane / C; r0 < 32; r0 += R * B) {
      uint32_t u[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const uint32_t at = box_at(box, r0 + i * R, (c * E) >> 4) + ((c * E) & 15);
        if constexpr (E == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u[i]) : "r"(at));
        else if constexpr (E == 2)
          asm volatile("{ .reg .u16 t; ld.shared.u16 t, [%1]; cvt.u32.u16 %0, t; }" : "=r"(u[i]) : "r"(at));
        else asm volatile("ld.shared.u8 %0, [%1];" : "=r"(u[i]) : "r"(at));
      }
#pragma unroll
      for (int i = 0; i < B; ++i) {
        if (m0 + r0 + i * R < M && n + c < N) *dst = (U)u[i];
        dst += R * ld;
      }
    }
  }
  // the box next receives a residual by TMA: after these ordinary accesses
  fence_proxy_async_smem();
  __syncwarp();
}

// One epilogue warp: its box, bias and residual loads.
struct Fp8EpilogueWarp {
  static constexpr int CHUNKS = kFp8EpiColumns / 32;
  const Fp8PairParams& q;
  const CUtensorMap *map_y, *map_r;
  uint32_t box;         // shared address of its 2 KB
  const float4* bias4;  // its columns
  uint64_t* res_bar;    // residual box landed
  uint64_t* amax_bar;   // both warps of a block have its largest values (quantised output)
  uint32_t* amax;       // [2][warps][32] largest |value| of 64 columns, this warp's
  int lane;
  int group;            // its columns begin at 64 group
  int m0, n0;           // its tokens and columns of this tile
  uint32_t res_phase;   // parity of res_bar
  bool res_open;        // a load has not been waited for
  volatile int* abort_flag;
  uint32_t peer_abort;

  // the chunk that holds the columns that the accumulators share comes first:
  // the last of accumulator 0, the first of accumulator 1
  __device__ __forceinline__ int chunk(int j) const { return group >= 2 ? CHUNKS - 1 - j : j; }
  __device__ __forceinline__ int column(int j) const { return n0 + 32 * chunk(j); }
  __device__ __forceinline__ bool inside(int n) const { return n < q.p.N && m0 < q.p.M; }
  __device__ __forceinline__ int res_cols() const { return q.p.e.res_type == FTB_F32 ? 16 : 32; }

  // Residual columns from n into the box, once the stores from it have read it.
  __device__ __forceinline__ void res_load(int n) {
    if (lane == 0) {
      bulk_wait_read();
      mbar_arrive_expect_tx(res_bar, 2048);
      tma_load_2d_at(box, map_r, n, m0, res_bar);
    }
    res_open = true;
  }
  __device__ __forceinline__ bool res_wait(bool ignore_abort = false) {
    const bool ok = pair_wait_warp(res_bar, res_phase, abort_flag, peer_abort, q.p.err, 22, ignore_abort);
    res_phase ^= 1u;
    res_open = false;
    return ok;
  }
  // The first residual box of the first chunk from j on that is inside.
  __device__ __forceinline__ void res_next(int j) {
    for (; j < CHUNKS; ++j)
      if (inside(column(j))) {
        __syncwarp();
        res_load(column(j));
        return;
      }
  }

  __device__ __forceinline__ void begin_tile() {
    if (q.p.e.bias) {
      const int n = n0 + 4 * lane, N = 4 * lane < kFp8EpiColumns ? q.p.N : 0;
      float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (q.bias_vec && n + 4 <= N) {
        f = *reinterpret_cast<const float4*>(q.p.e.bias + n);
      } else {
        if (n < N) f.x = q.p.e.bias[n];
        if (n + 1 < N) f.y = q.p.e.bias[n + 1];
        if (n + 2 < N) f.z = q.p.e.bias[n + 2];
        if (n + 3 < N) f.w = q.p.e.bias[n + 3];
      }
      __syncwarp();
      if (4 * lane < kFp8EpiColumns) const_cast<float4*>(bias4)[lane] = f;
      __syncwarp();
    }
    if (q.res_tma) res_next(0);
  }

  // bias, ReLU and residual on chunk j of this lane's token; false on a timeout
  __device__ __forceinline__ bool finish(int j, float (&v)[32]) {
    const Fp8Epilogue& e = q.p.e;
    const int n = column(j);
    if (!inside(n)) return true;
    if (e.bias) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 b = bias4[8 * chunk(j) + i];
        v[4 * i] = __fadd_rn(v[4 * i], b.x);
        v[4 * i + 1] = __fadd_rn(v[4 * i + 1], b.y);
        v[4 * i + 2] = __fadd_rn(v[4 * i + 2], b.z);
        v[4 * i + 3] = __fadd_rn(v[4 * i + 3], b.w);
      }
    }
    if (e.relu) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = max_nan(v[i], 0.0f);
    }
    if (!e.residual) return true;
    if (e.res_type == FTB_F32) return add_boxes<float>(j, v);
    if (e.res_type == FTB_F16) return add_boxes<__half>(j, v);
    return add_boxes<__nv_bfloat16>(j, v);
  }
  template <typename T>
  __device__ __forceinline__ bool add_boxes(int j, float (&v)[32]) {
    constexpr int C = 64 / (int)sizeof(T), E = 16 / (int)sizeof(T);
#pragma unroll
    for (int b = 0; b < 32 / C; ++b) {
      const int n = column(j) + b * C;
      if (!inside(n)) break;
      if (q.res_tma) {
        if (b > 0) {
          __syncwarp();
          res_load(n);
        }
        if (!res_wait()) return false;
      } else {
        box_begin();
        using U = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
        load_box_rows(box, static_cast<const U*>(q.p.e.residual), q.p.e.res_ld, m0, n, q.p.M, q.p.N, lane);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 u = ld_shared4(box_at(box, lane, i));
        T t[E];
        memcpy(t, &u, 16);
#pragma unroll
        for (int k = 0; k < E; ++k) v[b * C + i * E + k] = __fadd_rn(v[b * C + i * E + k], to_f32(t[k]));
      }
    }
    return true;
  }

  // The box, once the store before has read it and every lane its residual.
  __device__ __forceinline__ void box_begin() const {
    if (lane == 0) bulk_wait_read();
    __syncwarp();
  }
  __device__ __forceinline__ void box_store(int n) const {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(map_y, n, m0, box);
      bulk_commit();
    }
  }
};

// 32 finished columns (from n) of a warp's tokens into a plain output.
template <typename T>
__device__ __forceinline__ void store_plain32(const Fp8EpilogueWarp& w, int n, const float (&v)[32]) {
  constexpr int C = 64 / (int)sizeof(T);  // columns per box
  const Fp8Params& p = w.q.p;
#pragma unroll
  for (int b = 0; b < 32 / C; ++b) {
    if (n + b * C >= p.N) break;
    w.box_begin();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T t[C / 4];
#pragma unroll
      for (int j = 0; j < C / 4; ++j) t[j] = from_f32<T>(v[b * C + i * (C / 4) + j]);
      uint32_t u[4];
      memcpy(u, t, 16);
      st_shared4(box_at(w.box, w.lane, i), u[0], u[1], u[2], u[3]);
    }
    if (w.q.y_tma && n + (b + 1) * C <= p.N) {
      w.box_store(n + b * C);
    } else {
      using U = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
      store_box_rows(w.box, static_cast<U*>(p.e.y), p.e.y_ld, w.m0, n + b * C, p.M, p.N, w.lane);
    }
  }
}

// A lane's 64 columns, half of a block, in chunk order, into a quantised
// output; `buf` alternates between tiles.  False on a timeout.
__device__ __forceinline__ bool store_quantized(const Fp8EpilogueWarp& w, uint32_t buf, uint32_t phase,
                                                float (&v)[2][32]) {
  const Fp8Params& p = w.q.p;
  float top = 0.0f;  // NaN is passed over
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(v[j][i]));
  uint32_t amax = __float_as_uint(top);
  if (amax >= 0x7F800000u) {  // an infinity: the scale comes from the finite values
    amax = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        amax = max(amax, finite_abs_bits(v[j][i]));
        v[j][i] = nan_unless_finite(v[j][i]);
      }
  }
  // the other half of the block is four warps on (or back): columns 64 apart
  uint32_t* mine = w.amax + buf * (kFp8EpiWarps * 32) + w.lane;
  *mine = amax;
  __syncwarp();
  if (w.lane == 0) mbar_arrive(w.amax_bar);
  if (!pair_wait_warp(w.amax_bar, phase, w.abort_flag, w.peer_abort, p.err, 23)) return false;
  amax = max(amax, *(volatile uint32_t*)(w.group & 1 ? mine - 4 * 32 : mine + 4 * 32));
  if (!w.inside(w.n0)) return true;
  const uint32_t byte = fp8_scale_byte(amax);
  const float inv = fp8_inv_scale(byte);
  const int64_t m = (int64_t)w.m0 + w.lane;
  if (!(w.group & 1) && m < p.M) p.e.ys[m * p.e.ys_ld + w.n0 / kFp8Block] = (uint8_t)byte;
  w.box_begin();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int first = 2 * w.chunk(j);
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      u[i] = fp8_pack4(v[j][4 * i], v[j][4 * i + 1], v[j][4 * i + 2], v[j][4 * i + 3], inv);
    st_shared4(box_at(w.box, w.lane, first), u[0], u[1], u[2], u[3]);
    st_shared4(box_at(w.box, w.lane, first + 1), u[4], u[5], u[6], u[7]);
  }
  if (w.n0 + 64 <= p.N) w.box_store(w.n0);
  else store_box_rows(w.box, static_cast<uint8_t*>(p.e.y), p.e.y_ld, w.m0, w.n0, p.M, p.N, w.lane);
  return true;
}

template <bool QUANT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Fp8PairShape::THREADS, 1)
    fp8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                    const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_r,
                    const Fp8PairParams q) {
  using L = Fp8PairShape;
  constexpr int STAGES = L::STAGES;
  constexpr uint32_t kAcc1 = 224, kSf = 480;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* boxes = smem + STAGES * L::STAGE_BYTES;
  uint8_t* sf = smem + L::SF_OFF;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);  // this CTA's loads landed
  uint64_t* ready = full + STAGES;      // leader: both CTAs' loads landed
  uint64_t* empty = ready + STAGES;     // the pair's MMAs done with the stage
  uint64_t* sf_full = empty + STAGES;   // [2] leader: both CTAs' scale factors staged
  uint64_t* sf_empty = sf_full + 2;     // [2] the pair's MMAs done with them
  uint64_t* accf = sf_empty + 2;        // [2] accumulator complete
  uint64_t* acce = accf + 2;            // [2] leader: accumulator read (both CTAs' epilogue warps)
  uint64_t* shared_cols = acce + 2;     // leader: the shared columns read (the same), once per tile
  uint64_t* drain = shared_cols + 1;    // leader: MMAs retired after an abort
  uint64_t* res_bar = drain + 1;        // [warps] an epilogue warp's residual box landed
  uint64_t* amax_bar = res_bar + kFp8EpiWarps;  // [warps] the two warps of a block share its first one's
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(amax_bar + kFp8EpiWarps);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(amax_bar + kFp8EpiWarps) + 1;

  const Fp8Params& p = q.p;
  const uint32_t rank = cluster_ctarank(), peer = rank ^ 1u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nk = (p.K + kFp8Block - 1) / kFp8Block;
  Fp8Tiles tiles{(p.M + 255) / 256, (p.N + 255) / 256};
  const int ntiles = tiles.tm * tiles.tn;
  const int pair = (int)cluster_index(), npairs = (int)cluster_count();

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&ready[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sf_full[s], 2);
      mbar_init(&sf_empty[s], 1);
      mbar_init(&accf[s], 1);
      mbar_init(&acce[s], 2 * kFp8EpiWarps);
    }
    mbar_init(shared_cols, 2 * kFp8EpiWarps);
    mbar_init(drain, 1);
    for (int s = 0; s < kFp8EpiWarps; ++s) {
      mbar_init(&res_bar[s], 1);
      mbar_init(&amax_bar[s], 2);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(const_cast<uint32_t*>(tmem_slot))),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 3 && elect_one()) {
    prefetch_map(&map_a);
    prefetch_map(&map_w);
    if (q.y_tma) prefetch_map(&map_y);
    if (q.res_tma) prefetch_map(&map_r);
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  grid_dep_wait();
  grid_dep_trigger();
  const uint32_t tmem = *tmem_slot;
  const uint32_t peer_abort = cluster_addr(const_cast<int*>(abort_flag), peer);

  if (warp == 0) {
    bool ok = true;
    uint32_t it = 0;
    for (int t = pair; t < ntiles && ok; t += npairs) {
      int m0, n0;
      tiles.at(t, m0, n0);
      m0 += (int)rank * 128;
      n0 += (int)rank * 128;
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const uint32_t s = it % STAGES;
        if (!(ok = pair_wait_warp(&empty[s], ((it / STAGES) & 1u) ^ 1u, abort_flag, peer_abort, p.err, 11))) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&full[s], L::STAGE_BYTES);
          tma_load_2d(smem + s * L::STAGE_BYTES, &map_a, kb * kFp8Block, m0, &full[s]);
          tma_load_2d(smem + s * L::STAGE_BYTES + L::OPERAND_BYTES, &map_w, kb * kFp8Block, n0, &full[s]);
        }
        __syncwarp();
      }
    }
    if (!ok)  // the copies in flight land before the CTA leaves
      for (uint32_t j = it > STAGES ? it - STAGES : 0; j < it; ++j)
        pair_wait_warp(&full[j % STAGES], (j / STAGES) & 1u, abort_flag, peer_abort, p.err, 12, /*ignore_abort=*/true);
  } else if (warp == 1) {
    if (rank == 0) {
      bool ok = true;
      uint32_t it = 0, sg = 0, tc = 0;
      if (p.stall_test) ok = pair_wait_warp(drain, 0, abort_flag, peer_abort, p.err, 13);
      for (int t = pair; t < ntiles && ok; t += npairs, ++tc) {
        const uint32_t b = tc & 1u;
        if (!(ok = pair_wait_warp(&acce[b], ((tc >> 1) & 1u) ^ 1u, abort_flag, peer_abort, p.err, 14))) break;
        if (tc > 0 &&
            !(ok = pair_wait_warp(shared_cols, (tc - 1) & 1u, abort_flag, peer_abort, p.err, 15)))
          break;
        tc_fence_after();
        const uint32_t d = tmem + b * kAcc1;
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const uint32_t slot = sg & 1u, byte = (uint32_t)kb & 3u;
          const uint32_t sfa = tmem + kSf + slot * 16, sfb = sfa + 4;
          if (byte == 0) {
            if (!(ok = pair_wait_warp(&sf_full[slot], (sg >> 1) & 1u, abort_flag, peer_abort, p.err, 16))) break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t at = smem_u32(sf + slot * L::SF_BYTES);
              tmem2_copy_scales(sfa, fp8_scale_desc(at));
              tmem2_copy_scales(sfb, fp8_scale_desc(at + 512));
              tmem2_copy_scales(sfb + 4, fp8_scale_desc(at + 1024));
            }
            __syncwarp();
          }
          const uint32_t s = it % STAGES;
          if (!(ok = pair_wait_warp(&ready[s], (it / STAGES) & 1u, abort_flag, peer_abort, p.err, 17))) break;
          tc_fence_after();
          const bool last = kb + 1 == nk, group_end = byte == 3u || last;
          const uint32_t empty_peer = cluster_addr(&empty[s], peer);
          const uint32_t sf_empty_peer = cluster_addr(&sf_empty[slot], peer);
          const uint32_t accf_peer = cluster_addr(&accf[b], peer);
          if (elect_one()) {
            const uint32_t a = smem_u32(smem + s * L::STAGE_BYTES), w = a + L::OPERAND_BYTES;
            const uint32_t idesc = fp8_idesc(256, 256, (int)byte);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              umma2_fp8(d, fp8_operand_desc(a + j * 32), fp8_operand_desc(w + j * 32), idesc, sfa, sfb,
                        (kb > 0 || j > 0) ? 1u : 0u);
            umma2_commit(smem_u32(&empty[s]));
            umma2_commit(empty_peer);
            if (group_end) {
              umma2_commit(smem_u32(&sf_empty[slot]));
              umma2_commit(sf_empty_peer);
            }
            if (last) {
              umma2_commit(smem_u32(&accf[b]));
              umma2_commit(accf_peer);
            }
          }
          __syncwarp();
          if (group_end) ++sg;
        }
      }
      if (!ok) {
        if (elect_one()) umma2_commit(smem_u32(drain));
        __syncwarp();
        pair_wait_warp(drain, 0, abort_flag, peer_abort, p.err, 18, /*ignore_abort=*/true);
      }
    }
  } else if (warp == 2) {
    bool ok = true;
    uint32_t sg = 0;
    const int groups = (nk + 3) >> 2, nb = (p.N + kFp8Block - 1) / kFp8Block;
    for (int t = pair; t < ntiles && ok; t += npairs) {
      int m0, n0;
      tiles.at(t, m0, n0);
      const int r0 = m0 + (int)rank * 128 + lane, b0 = n0 / kFp8Block;
      const uint8_t* w0 = p.sw + (int64_t)b0 * p.sw_ld;
      const uint8_t* w1 = p.sw + (int64_t)min(b0 + 1, nb - 1) * p.sw_ld;
      for (int g = 0; g < groups; ++g, ++sg) {
        const uint32_t slot = sg & 1u;
        const uint32_t x = fp8_scale_word(w0, g, nk), y = fp8_scale_word(w1, g, nk);
        uint32_t a[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          a[j] = r0 + 32 * j < p.M ? fp8_scale_word(p.sa + (int64_t)(r0 + 32 * j) * p.sa_ld, g, nk) : 0u;
        if (!(ok = pair_wait_warp(&sf_empty[slot], ((sg >> 1) & 1u) ^ 1u, abort_flag, peer_abort, p.err, 19))) break;
        const uint32_t at = smem_u32(sf + slot * L::SF_BYTES) + lane * 16;
        st_shared4(at, a[0], a[1], a[2], a[3]);
        st_shared4(at + 512, x, x, x, x);
        st_shared4(at + 1024, y, y, y, y);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_addr(&sf_full[slot], 0));
      }
    }
  } else if (warp == 3) {
    bool ok = true;
    uint32_t it = 0;
    for (int t = pair; t < ntiles && ok; t += npairs) {
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const uint32_t s = it % STAGES;
        if (!(ok = pair_wait_warp(&full[s], (it / STAGES) & 1u, abort_flag, peer_abort, p.err, 20))) break;
        if (lane == 0) mbar_arrive_cluster(cluster_addr(&ready[s], 0));
      }
    }
  } else {
    const int quarter = warp & 3, e = warp - 4;
    Fp8EpilogueWarp w{q, &map_y, &map_r, smem_u32(boxes) + (uint32_t)e * 2048u,
                      reinterpret_cast<const float4*>(smem + L::BIAS_OFF + e * kFp8EpiColumns * 4), res_bar + e,
                      amax_bar + (e & ~4), reinterpret_cast<uint32_t*>(smem + L::AMAX_OFF) + e * 32, lane, e >> 2, 0,
                      0, 0u, false, abort_flag, peer_abort};
    const uint32_t shared_leader = cluster_addr(shared_cols, 0);
    uint32_t tc = 0;
    bool ok = true;
    for (int t = pair; t < ntiles && ok; t += npairs, ++tc) {
      const uint32_t b = tc & 1u;
      tiles.at(t, w.m0, w.n0);
      w.m0 += (int)rank * 128 + quarter * 32;
      w.n0 += w.group * kFp8EpiColumns;
      w.begin_tile();
      if (!(ok = pair_wait_warp(&accf[b], (tc >> 1) & 1u, abort_flag, peer_abort, p.err, 21))) break;
      tc_fence_after();
      const uint32_t acc = tmem + b * kAcc1 + (uint32_t)(w.group * kFp8EpiColumns) + ((uint32_t)(quarter * 32) << 16);
      const uint32_t acce_leader = cluster_addr(&acce[b], 0);
      auto load = [&](int j, float (&v)[32]) {
        uint32_t r[32];
        __syncwarp();  // warp-collective, and one lane has sent a box or arrived since
        FTB_TMEM_LD32(acc + 32 * w.chunk(j), r);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        if (j == 0 || j + 1 == Fp8EpilogueWarp::CHUNKS) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(j == 0 ? shared_leader : acce_leader);
        }
      };
      if constexpr (!QUANT) {
#pragma unroll 1
        for (int j = 0; j < Fp8EpilogueWarp::CHUNKS; ++j) {
          float v[32];
          load(j, v);
          const int n = w.column(j);
          if (!ok || !w.inside(n)) continue;
          if (!(ok = w.finish(j, v))) continue;
          if (p.e.y_type == FTB_F32) store_plain32<float>(w, n, v);
          else if (p.e.y_type == FTB_F16) store_plain32<__half>(w, n, v);
          else store_plain32<__nv_bfloat16>(w, n, v);
          if (q.res_tma) w.res_next(j + 1);
        }
      } else {
        float v[2][32];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          load(j, v[j]);
          const int n = w.column(j);
          if (ok && w.inside(n)) {
            ok = w.finish(j, v[j]);
            if (ok && q.res_tma) w.res_next(j + 1);
          }
          if (n + 32 > p.N) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (n + i >= p.N) v[j][i] = 0.0f;
          }
        }
        if (ok) ok = store_quantized(w, b, (tc & 1u), v);
      }
    }
    if (w.res_open) w.res_wait(/*ignore_abort=*/true);  // a load in flight lands before the CTA leaves
    if (lane == 0) bulk_wait_all();  // this warp's stores are complete before the CTA leaves
  }
  tc_fence_before();
  cluster_sync_all();  // no MMA of the pair and no remote arrival is still in flight
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Shared-memory attributes and the number of pairs that are resident at once.
inline cudaError_t fp8_pair_prepare(int* pairs) {
  using L = Fp8PairShape;
  cudaError_t e = cudaFuncSetAttribute(fp8_pair_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(fp8_pair_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2, 1, 1);
  cfg.blockDim = dim3(L::THREADS, 1, 1);
  cfg.dynamicSmemBytes = L::TOTAL;
  e = cudaOccupancyMaxActiveClusters(pairs, fp8_pair_kernel<false>, &cfg);
  if (e == cudaSuccess && *pairs <= 0) e = cudaErrorInvalidConfiguration;
  return e;
}

// An output or residual as the epilogue moves it: boxes of 32 rows x 64 bytes,
// 64-byte swizzle.  False where its rows are not 16-byte aligned.
inline bool make_map_fp8_box(CUtensorMap* map, void* base, int type, int64_t ld, int64_t m, int64_t n) {
  const int size = type == FTB_F32 ? 4 : type == kFp8Type ? 1 : 2;
  if (!base || (reinterpret_cast<uintptr_t>(base) & 15) || (ld * size) % 16) return false;
  PFN_encodeTiled enc = tma_encoder();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)n, (cuuint64_t)m};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * size)};
  cuuint32_t box[2] = {(cuuint32_t)(64 / size), 32};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType dtype = size == 4   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                    : size == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                                : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  return enc(map, dtype, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline cudaError_t launch_fp8_pair(const Fp8Operands& o, const Fp8Params& p, int max_pairs, cudaStream_t s) {
  CUtensorMap map_a, map_w, map_y, map_r;
  if (!make_map_fp8(&map_a, o.a, p.M, p.K, o.a_ld, 128) || !make_map_fp8(&map_w, o.w, p.N, p.K, o.w_ld, 128))
    return cudaErrorInvalidValue;
  Fp8PairParams q{};
  q.p = p;
  memset(&map_y, 0, sizeof(map_y));
  memset(&map_r, 0, sizeof(map_r));
  q.y_tma = make_map_fp8_box(&map_y, p.e.y, p.e.y_type, p.e.y_ld, p.M, p.N);
  if (!q.y_tma && p.e.y_type == kFp8Type) return cudaErrorInvalidValue;
  q.res_tma = make_map_fp8_box(&map_r, const_cast<void*>(p.e.residual), p.e.res_type, p.e.res_ld, p.M, p.N);
  q.bias_vec = (reinterpret_cast<uintptr_t>(p.e.bias) & 15) == 0;
  const int64_t tiles = (((int64_t)p.M + 255) / 256) * (((int64_t)p.N + 255) / 256);
  if (tiles > 0x3fffffff) return cudaErrorInvalidConfiguration;
  const unsigned pairs = (unsigned)std::min<int64_t>(tiles, max_pairs);
  return pdl_launch(p.e.y_type == kFp8Type ? fp8_pair_kernel<true> : fp8_pair_kernel<false>, dim3(2 * pairs),
                    dim3(Fp8PairShape::THREADS), Fp8PairShape::TOTAL, s, map_a, map_w, map_y, map_r, q);
}

}  // namespace ftb
