// Matrix product of block-scaled 8-bit operands on the tensor cores.
//
//   y[m, n] = epi( sum_b sa[m, b] sw[n / 128, b] sum_{k in block b} a[m, k] w[n, k] )
//   epi(v) = relu(v + bias[n]) + residual[m, n], each part optional
//
// tcgen05.mma kind::mxf8f6f4.block_scale multiplies each product of 32 k by
// the two operands' ue8m0 scales itself and accumulates in fp32, so a block of
// 128 is four such steps that use the same scale byte: the scale factors lie
// in tensor memory as one word per row, its four bytes the scales of four
// consecutive blocks, and the instruction descriptor names the byte.
//
// fp8_tile_kernel: 128 weight rows are the MMA's M side and NT tokens its N
// side, so few tokens waste no tensor rows, a lane of tensor memory is an
// output column and 32 lanes store consecutive outputs.  Eight warps:
//   warp 0     TMA producer: a 128 x 128 weight block and an NT x 128 token
//              block per k-block, 128-byte swizzle, into a ring;
//   warp 1     tensor memory and the MMAs (one elected lane);
//   warp 2     scale factors: one group (four k-blocks) at a time from global
//              memory into the layout that tcgen05.cp takes;
//   warps 4-7  the accumulator into shared memory as [token][output];
// then every warp finishes tokens: a lane has four consecutive outputs of one
// token, a warp the 128 of a quantisation block.
// Every wait is bounded, as in the other tensor-core kernels.
#pragma once

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "fp8_format.cuh"
#include "tc_ptx.cuh"

namespace ftb {

constexpr int kFp8Threads = 256;

// What an epilogue reads and writes.
struct Fp8Epilogue {
  const float* bias;      // [N], or null
  const void* residual;   // [M, N] of res_type, or null
  int64_t res_ld;
  int res_type;
  int relu;
  void* y;                // [M, N] of y_type (kFp8Type: quantised)
  int64_t y_ld;
  int y_type;
  uint8_t* ys;            // scales of a quantised output
  int64_t ys_ld;
  int res_vec, y_vec;     // residual and plain output: bases and rows are aligned to 16 bytes
};

struct Fp8Params {
  int M, N, K;            // tokens, outputs, depth
  const uint8_t* sa;      // [M, K / 128], rows sa_ld apart
  int64_t sa_ld;
  const uint8_t* sw;      // [N / 128, K / 128]
  int64_t sw_ld;
  Fp8Epilogue e;
  int* err;        // set when a bounded wait gives up
  int stall_test;  // failure-detection tests: the MMA warp first waits for what nothing completes
};

// The four scale bytes of k-blocks 4 g .. 4 g + 3 as one word; bytes past the
// last block are not read (rows start on multiples of four bytes).
__device__ __forceinline__ uint32_t fp8_scale_word(const uint8_t* row, int g, int kblocks) {
  if (4 * g + 3 < kblocks) return *reinterpret_cast<const uint32_t*>(row + 4 * g);
  uint32_t w = 0;
  for (int i = 0; i < 3; ++i)
    if (4 * g + i < kblocks) w |= (uint32_t)row[4 * g + i] << (8 * i);
  return w;
}

// K-major operand tile of 128-byte rows in the 128-byte swizzle: 8-row groups
// 1024 bytes apart.
__device__ __forceinline__ uint64_t fp8_operand_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Scale factors as tcgen05.cp 32x128b reads them: 32 rows of 16 bytes, no
// swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t fp8_scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(128 >> 4) << 32) |
         ((uint64_t)1 << 46);
}

// Instruction descriptor: e4m3 x e4m3 (formats 0), ue8m0 scales, K-major, D of
// m x n; `byte` selects the scale byte of both operands.
__device__ __forceinline__ uint32_t fp8_idesc(int m, int n, int byte) {
  return ((uint32_t)byte << 4) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27) |
         ((uint32_t)byte << 29);
}

__device__ __forceinline__ void umma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                         uint32_t sfb, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
      : "memory");
}

// 512 bytes of scale factors (128 rows) into four columns of tensor memory.
__device__ __forceinline__ void tmem_copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// A box into L2 only.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}

__device__ __forceinline__ void st_shared4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Four consecutive values of a plain type, of which `cnt` exist; `vec`: rows
// and bases are aligned to four elements.
template <typename T>
__device__ __forceinline__ void fp8_load4(const T* src, int cnt, bool vec, float (&v)[4]) {
  if (vec && cnt >= 4) {
    T t[4];
    if constexpr (sizeof(T) == 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(src);
      memcpy(t, &u, 16);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(src);
      memcpy(t, &u, 8);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f32(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < cnt ? to_f32(src[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void fp8_store4(T* dst, int cnt, bool vec, const float (&v)[4]) {
  if (vec && cnt >= 4) {
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = from_f32<T>(v[i]);
    if constexpr (sizeof(T) == 4) {
      uint4 u;
      memcpy(&u, t, 16);
      *reinterpret_cast<uint4*>(dst) = u;
    } else {
      uint2 u;
      memcpy(&u, t, 8);
      *reinterpret_cast<uint2*>(dst) = u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < cnt) dst[i] = from_f32<T>(v[i]);
  }
}

// A warp finishes 128 outputs of token m: lane l has columns n .. n + 3,
// n = n0 + 4 l, their bias and residual; `cnt` = N - n columns exist from there.
__device__ __forceinline__ void fp8_residual(const Fp8Epilogue& e, int64_t m, int n, int cnt, float (&r)[4]) {
  const int64_t at = m * e.res_ld + n;
  if (e.res_type == FTB_F32) fp8_load4(static_cast<const float*>(e.residual) + at, cnt, e.res_vec, r);
  else if (e.res_type == FTB_F16) fp8_load4(static_cast<const __half*>(e.residual) + at, cnt, e.res_vec, r);
  else fp8_load4(static_cast<const __nv_bfloat16*>(e.residual) + at, cnt, e.res_vec, r);
}

__device__ __forceinline__ void fp8_finish(const Fp8Epilogue& e, int64_t m, int n0, int N, int lane,
                                           const float (&bias)[4], const float (&res)[4], float (&v)[4]) {
  const int n = n0 + 4 * lane;
  const int cnt = N - n;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (e.bias) v[i] = __fadd_rn(v[i], bias[i]);
    if (e.relu) v[i] = (v[i] != v[i] || v[i] > 0.0f) ? v[i] : 0.0f;  // keeps NaN
    if (e.residual) v[i] = __fadd_rn(v[i], res[i]);
  }
  if (e.y_type == kFp8Type) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < cnt) a = max(a, finite_abs_bits(v[i]));
      v[i] = nan_unless_finite(v[i]);
    }
    const uint32_t byte = fp8_scale_byte(__reduce_max_sync(0xffffffffu, a));
    const uint32_t w = fp8_pack4(v[0], v[1], v[2], v[3], fp8_inv_scale(byte));
    uint8_t* q = static_cast<uint8_t*>(e.y) + m * e.y_ld + n;
    if (cnt >= 4) {
      *reinterpret_cast<uint32_t*>(q) = w;
    } else {
      for (int i = 0; i < cnt; ++i) q[i] = (uint8_t)(w >> (8 * i));
    }
    if (lane == 0) e.ys[m * e.ys_ld + n0 / kFp8Block] = (uint8_t)byte;
    return;
  }
  if (cnt < 1) return;
  const int64_t at = m * e.y_ld + n;
  if (e.y_type == FTB_F32) fp8_store4(static_cast<float*>(e.y) + at, cnt, e.y_vec, v);
  else if (e.y_type == FTB_F16) fp8_store4(static_cast<__half*>(e.y) + at, cnt, e.y_vec, v);
  else fp8_store4(static_cast<__nv_bfloat16*>(e.y) + at, cnt, e.y_vec, v);
}

// The address in CTA `rank` of the cluster of the shared variable at `addr`.
__device__ __forceinline__ uint32_t cluster_map(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void ld_cluster4(uint32_t addr, float (&v)[4]) {
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
               : "r"(addr)
               : "memory");
}

template <int NT>
struct Fp8TileSmem {
  static constexpr int W_BYTES = 128 * 128;
  static constexpr int A_BYTES = NT * 128;
  static constexpr int STAGE_BYTES = W_BYTES + A_BYTES;
  // Three stages of few tokens, and the first weights sent for ahead of the
  // launch's turn: a chain of norm and two layers of 4096 x 8192 at 16 tokens
  // takes 20.5 us a layer; with five stages 21.5, without those weights 21.2,
  // with neither change 22.6.  One product of 16 x 8192 x 4096 with its weights
  // in HBM: 8.9, 9.4, 9.2 and 9.9.  Registers (118 to 128) hold the split forms
  // to two CTAs per SM with either ring, so it is not room for a third that the
  // shorter one gains by; what it is has not been found.
  static constexpr int STAGES = NT == 64 ? 4 : 3;
  static constexpr int SF_SLOTS = 2;
  static constexpr int SF_BYTES = 1024;  // 512 of each operand
  static constexpr int BAR_OFF = STAGES * STAGE_BYTES + SF_SLOTS * SF_BYTES;
  static constexpr int TOTAL = 1024 + BAR_OFF + 8 * (2 * STAGES + 2 * SF_SLOTS + 2) + 16;
  static constexpr int D_COLS = NT < 32 ? 32 : NT;
  static constexpr int TMEM_COLS = D_COLS <= 32 ? 64 : D_COLS == 64 ? 128 : 256;  // D, then 8 columns per slot
  static_assert(NT * 128 * 4 <= STAGES * STAGE_BYTES, "the result tile reuses the ring");
};

template <int NT, int SPLIT>
__global__ void __launch_bounds__(kFp8Threads) fp8_tile_kernel(const __grid_constant__ CUtensorMap map_w,
                                                               const __grid_constant__ CUtensorMap map_a,
                                                               const Fp8Params p) {
  using L = Fp8TileSmem<NT>;
  constexpr int STAGES = L::STAGES, SLOTS = L::SF_SLOTS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sf = smem + STAGES * L::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* empty = full + STAGES;
  uint64_t* sf_full = empty + STAGES;
  uint64_t* sf_empty = sf_full + SLOTS;
  uint64_t* done = sf_empty + SLOTS;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(done + 1) + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned n_tiles = (unsigned)(p.N + 127) / 128u;
  const unsigned tile_id = blockIdx.x / SPLIT;
  const int n0 = (int)(tile_id % n_tiles) * 128;
  const int m0 = (int)(tile_id / n_tiles) * NT;
  const int nk = (p.K + kFp8Block - 1) / kFp8Block;
  // this CTA's k-blocks: whole groups of four, so that its scale words start
  // at byte 0; the last CTAs of a cluster may have none
  const int rank = SPLIT > 1 ? (int)cluster_ctarank() : 0;
  const int per = ((nk + 3) / 4 + SPLIT - 1) / SPLIT * 4;
  const int kb0 = min(nk, rank * per), kb1 = min(nk, kb0 + per);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&sf_full[s], 1);
      mbar_init(&sf_empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(const_cast<uint32_t*>(tmem_slot))),
                 "r"((uint32_t)L::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 3 && elect_one()) {
    prefetch_map(&map_w);
    prefetch_map(&map_a);
    // the first weight blocks on their way to L2 while kernels before this one
    // still run; nothing is read before grid_dep_wait
    for (int kb = kb0; kb < min(kb1, kb0 + STAGES); ++kb) tma_prefetch_2d(&map_w, kb * kFp8Block, n0);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dep_wait();
  grid_dep_trigger();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_sf = tmem + L::D_COLS;
  // of this lane's outputs; plain loads: a kernel before this one may have
  // written them after this one began (see grid_dep_wait)
  float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.e.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n0 + 4 * lane + i < p.N) bias[i] = p.e.bias[n0 + 4 * lane + i];
  }

  if (warp == 0) {
    bool ok = true;
    int it = 0;
    for (int kb = kb0; kb < kb1; ++kb, ++it) {
      const int s = it % STAGES;
      if (!(ok = mbar_wait_warp(&empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, p.err, 1))) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&full[s], L::STAGE_BYTES);
        tma_load_2d(smem + s * L::STAGE_BYTES, &map_w, kb * kFp8Block, n0, &full[s]);
        tma_load_2d(smem + s * L::STAGE_BYTES + L::W_BYTES, &map_a, kb * kFp8Block, m0, &full[s]);
      }
      __syncwarp();
    }
    if (!ok)  // the copies in flight land before the CTA leaves
      for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j)
        mbar_wait_warp(&full[j % STAGES], (j / STAGES) & 1, abort_flag, p.err, 2, /*ignore_abort=*/true);
  } else if (warp == 1) {
    bool ok = true;
    int it = 0;
    if (p.stall_test) ok = mbar_wait_warp(done, 0, abort_flag, p.err, 8);
    for (int kb = kb0; kb < kb1 && ok; ++kb, ++it) {
      const int g = (kb - kb0) >> 2, slot = g % SLOTS, byte = kb & 3;
      const uint32_t sfa = tmem_sf + slot * 8, sfb = sfa + 4;
      if (byte == 0) {
        if (!(ok = mbar_wait_warp(&sf_full[slot], (g / SLOTS) & 1, abort_flag, p.err, 3))) break;
        tc_fence_after();
        if (elect_one()) {
          tmem_copy_scales(sfa, fp8_scale_desc(smem_u32(sf + slot * L::SF_BYTES)));
          tmem_copy_scales(sfb, fp8_scale_desc(smem_u32(sf + slot * L::SF_BYTES + 512)));
        }
        __syncwarp();
      }
      const int s = it % STAGES;
      if (!(ok = mbar_wait_warp(&full[s], (it / STAGES) & 1, abort_flag, p.err, 4))) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t w = smem_u32(smem + s * L::STAGE_BYTES), a = w + L::W_BYTES;
        const uint32_t idesc = fp8_idesc(128, NT, byte);
#pragma unroll
        for (int j = 0; j < 4; ++j)  // K = 32 (32 bytes) per MMA
          umma_fp8(tmem, fp8_operand_desc(w + j * 32), fp8_operand_desc(a + j * 32), idesc, sfa, sfb,
                   (kb > kb0 || j > 0) ? 1u : 0u);
        umma_commit(&empty[s]);
        if (byte == 3 || kb + 1 == kb1) umma_commit(&sf_empty[slot]);
        if (kb + 1 == kb1) umma_commit(done);
      }
      __syncwarp();
    }
    if (!ok) {  // what was issued retires before tensor memory is released
      if (elect_one()) umma_commit(done);
      __syncwarp();
      mbar_wait_warp(done, 0, abort_flag, p.err, 5, /*ignore_abort=*/true);
    }
  } else if (warp == 2) {
    const uint8_t* wrow = p.sw + (int64_t)(n0 / kFp8Block) * p.sw_ld;
    const int groups = (kb1 - kb0 + 3) >> 2;
    for (int g = 0; g < groups; ++g) {
      const int slot = g % SLOTS, kg = (kb0 >> 2) + g;
      const uint32_t w = fp8_scale_word(wrow, kg, nk);
      uint32_t t[4];  // tokens lane, lane + 32, ...: the words of one 16-byte row
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 32 * j + lane;
        t[j] = r < NT && m0 + r < p.M ? fp8_scale_word(p.sa + (int64_t)(m0 + r) * p.sa_ld, kg, nk) : 0u;
      }
      if (!mbar_wait_warp(&sf_empty[slot], ((g / SLOTS) & 1) ^ 1, abort_flag, p.err, 6)) break;
      const uint32_t at = smem_u32(sf + slot * L::SF_BYTES) + lane * 16;
      st_shared4(at, w, w, w, w);
      st_shared4(at + 512, t[0], t[1], t[2], t[3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sf_full[slot]);
    }
  }
  __syncwarp();
  float* tile = reinterpret_cast<float*>(smem);  // [NT][128]
  const int tokens = min(NT, p.M - m0);
  if (warp >= 4 && kb0 < kb1) {
    const bool ok = mbar_wait_warp(done, 0, abort_flag, p.err, 7);
    tc_fence_after();
    if (ok) {
      const int q = warp & 3;
#pragma unroll 1
      for (int c0 = 0; c0 < tokens; c0 += 32) {
        uint32_t r[32];
        __syncwarp();  // warp-collective
        FTB_TMEM_LD32(tmem + c0 + ((uint32_t)(q * 32) << 16), r);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c0 + j < NT) tile[(c0 + j) * 128 + q * 32 + lane] = __uint_as_float(r[j]);
      }
    }
    tc_fence_before();
  }
  if (SPLIT > 1) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::TMEM_COLS)
                 : "memory");
  }
  // each CTA finishes its share of the tokens, U per warp at a time (all
  // their loads in flight together): the partial sums in rank order, of the
  // CTAs that had k-blocks
  constexpr int U = SPLIT <= 2 ? 8 : 16 / SPLIT, STEP = SPLIT * (kFp8Threads / 32);
  const int parts = (nk + per - 1) / per;
  const int n = n0 + 4 * lane;
  for (int t0 = rank + SPLIT * warp; t0 < tokens; t0 += U * STEP) {
    float v[U][SPLIT][4], res[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * STEP;
      if (t >= tokens) break;
      const float* at = tile + t * 128 + lane * 4;
      if constexpr (SPLIT == 1) {
        const float4 f = *reinterpret_cast<const float4*>(at);
        v[u][0][0] = f.x, v[u][0][1] = f.y, v[u][0][2] = f.z, v[u][0][3] = f.w;
      } else {
#pragma unroll
        for (int r = 0; r < SPLIT; ++r)
          if (r < parts) ld_cluster4(cluster_map(smem_u32(at), r), v[u][r]);
      }
      if (p.e.residual) fp8_residual(p.e, m0 + t, n, p.N - n, res[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * STEP;
      if (t >= tokens) break;
#pragma unroll
      for (int r = 1; r < SPLIT; ++r)
        if (r < parts) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[u][0][i] = __fadd_rn(v[u][0][i], v[u][r][i]);
        }
      fp8_finish(p.e, m0 + t, n0, p.N, lane, bias, res[u], v[u][0]);
    }
  }
  if (SPLIT > 1) cluster_sync_all();  // no CTA leaves while another reads its sums
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// [rows, cols] bytes with rows `ld` apart, boxes of box_rows x 128, zero fill.
inline bool make_map_fp8(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  PFN_encodeTiled enc = tma_encoder();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Fp8Operands {
  const uint8_t* a;
  int64_t a_ld;
  const uint8_t* w;
  int64_t w_ld;
};

template <int NT, int SPLIT>
inline cudaError_t launch_fp8_tile(const Fp8Operands& o, const Fp8Params& p, cudaStream_t s) {
  CUtensorMap map_w, map_a;
  if (!make_map_fp8(&map_w, o.w, p.N, p.K, o.w_ld, 128) || !make_map_fp8(&map_a, o.a, p.M, p.K, o.a_ld, NT))
    return cudaErrorInvalidValue;
  const int64_t ctas = (((int64_t)p.N + 127) / 128) * (((int64_t)p.M + NT - 1) / NT) * SPLIT;
  if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kFp8Threads);
  cfg.dynamicSmemBytes = Fp8TileSmem<NT>::TOTAL;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = SPLIT;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fp8_tile_kernel<NT, SPLIT>, map_w, map_a, p);
}

// NT tokens per tile; `split` CTAs (1, 2, 4 or 8: a cluster) share its k-blocks.
template <int NT>
inline cudaError_t launch_fp8_tile(const Fp8Operands& o, const Fp8Params& p, int split, cudaStream_t s) {
  switch (split) {
    case 1: return launch_fp8_tile<NT, 1>(o, p, s);
    case 2: return launch_fp8_tile<NT, 2>(o, p, s);
    case 4: return launch_fp8_tile<NT, 4>(o, p, s);
    default: return launch_fp8_tile<NT, 8>(o, p, s);
  }
}

template <int NT, int SPLIT>
inline cudaError_t fp8_tile_attribute() {
  return cudaFuncSetAttribute(fp8_tile_kernel<NT, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Fp8TileSmem<NT>::TOTAL);
}
template <int NT>
inline cudaError_t fp8_tile_attributes() {
  cudaError_t e = fp8_tile_attribute<NT, 1>();
  if (e == cudaSuccess) e = fp8_tile_attribute<NT, 2>();
  if (e == cudaSuccess) e = fp8_tile_attribute<NT, 4>();
  if (e == cudaSuccess) e = fp8_tile_attribute<NT, 8>();
  return e;
}

}  // namespace ftb
