// W8A8 linears: y[t, n] = (sum_k q[t, k] w[n, k]) * scale[t] * row_scale[n], int32 sums.
//
// Every kernel here takes the weight rows as the tensor core's M operand and the tokens as its N
// operand, so an accumulator's lane is an output feature: 32 lanes write 32 neighbouring outputs of
// one token, whatever the row stride and however many outputs there are, and the channel scale is
// one register per lane. The int32 sum does not depend on the order of its terms and the two
// scales are applied in one order (i8_value), so a row's result is the same bits in every kernel,
// batch and split.
//
//   gemm_i8_pair_kernel   CTA pairs, 256 features x 256 or 192 tokens, persistent (large products)
//   gemm_i8_split_kernel  one CTA per 128 features x up to 128 tokens and K range; the K ranges of
//                         a tile are a cluster that adds its sums through distributed shared memory
//   gemm_i8_reg_kernel    at most 16 tokens: weights through registers into mma.sync, up to 32 MB of
//                         them (26 from 9 tokens on, fewer for the SwiGLU), or for at most 8 tokens and
//                         K <= 2048 as many as there are once the outputs pass 256 a SM (i8_few_tokens)
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace sdb {

struct I8Args {
  const int8_t* q;      // [m, ldx]
  const float* xs;      // [m]
  const int8_t* w;      // [n, k]
  const float* ws;      // [n]
  b200_linear_out o;
  int m, n, k, ldx;
  int ngroup;           // pair kernel: feature tiles per group
  int bt;               // pair and split kernel: tokens per tile
  int stages;           // split kernel: ring depth
  int vec;              // split kernel: every fourth output of a row is aligned to four outputs
};

constexpr int I8_BK = 128;  // bytes (= codes) of K per stage: one 128-byte swizzled row

__device__ __forceinline__ float i8_value(int acc, float xs, float ws) {
  return __fmul_rn(__fmul_rn(__int2float_rn(acc), xs), ws);
}

// silu(g) u = g u / (1 + 2^(-g log2 e)), flushing what underflows: 2^x to 0 where 1 + 2^x is 1
// anyway, 1 / (1 + 2^x) to 0 from 2^126 on, where the quotient is below 2^-119 (a NaN stays one).
__device__ __forceinline__ float swiglu(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(g, -1.4426950408889634f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return __fmul_rn(__fmul_rn(g, r), u);
}
// The SwiGLU's output at element idx of the planes: silu(g) * u as the bf16 hi plane and, with LO,
// the low plane.
template <bool LO>
__device__ __forceinline__ void store_swiglu(const b200_linear_out& o, size_t idx, float g, float u) {
  const float h = swiglu(g, u);
  const uint16_t hb = f32_to_bf16_rn(h);
  uint16_t* dst = static_cast<uint16_t*>(o.out);
  dst[idx] = hb;
  if constexpr (LO) {
    if (o.lo_format == B200_LO_E4M3)
      reinterpret_cast<uint8_t*>(dst + o.lo_offset)[idx] = uint8_t(f32x2_to_e4m3x2(lo8_value(h, hb), 0.0f));
    else
      dst[o.lo_offset + idx] = f32_to_bf16_rn(h - bf16_to_f32(hb));
  }
}

// Instruction descriptor, kind::i8: D s32, A and B signed bytes, both K-major, M x N.
__host__ __device__ constexpr uint32_t umma_idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_pair_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Waits for this warp's tcgen05.ld's; the registers they fill pass through, so that nothing that
// uses them moves ahead of the wait.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                 "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                 "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld_32x32b_x16(taddr, r); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_32x32b_x32(taddr, r); }
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}

// 5-D form of tma_load_2d_pair_hint, from the start of dimensions 1 to 3 (the SwiGLU's weight tile).
__device__ __forceinline__ void tma_load_5d_pair_hint(void* dst, const CUtensorMap* map, uint32_t bar_cluster, int x,
                                                      int v, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
      "[%1, {%3, %4, %4, %4, %5}], [%2], %6;" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(0), "r"(v), "l"(policy)
      : "memory");
}
// umma_pair_commit for the barrier at this offset in both CTAs of the pair: one instruction of the
// issuing thread instead of two (8192 x 12288 x 2048 SwiGLU 148.0 -> 144.8 us).
__device__ __forceinline__ void umma_pair_commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_addr(bar)),
      "h"(uint16_t(3))
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_addr(src)), "r"(x), "r"(y)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// All but the newest N of this thread's stores have read their shared memory.
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tma_store_wait_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ----------------------------------------------------------------------------- CTA pairs
// Tile: 256 features (128 per CTA) x bt tokens (256, or 192), K in stages of 128 codes (four MMAs of K = 32).
// Each CTA loads its 128 weight rows and its half of the tokens; the pair's MMA reads both halves.
//   warp 0      TMA ring (both CTAs; bytes signalled on the leader's full barrier)
//   warp 1      the leader's lane 0 issues the MMAs into one of two 256-column accumulators
//   warps 2..9  epilogue: TMEM lane quarter warp % 4, token half (warp - 2) / 4
//               (bt / 2 tokens, 16 or 32 at a time; the next ones leave TMEM while these are finished)
// 256 x 256 is the largest tile that leaves room for a second accumulator, which the next tile's
// products need while this one is finished: the main loop alone runs at 3425-3496 Tops/s (8192 and
// 18944 x 12288 x 2048), and with it 13 TB/s of operands cross from L2. What is lost on top is
// the epilogue's instructions and bytes: 8192 x 12288 x 2048 SwiGLU 143 us = 2.88 Pops/s, 65536
// tokens 1130 us; in a seconds-long run the 1000 W cap sets 1.47 GHz and 1325 us = 2.49 Pops/s.
// 65536 x 2048 x 6144 with the residual: 567 us = 2.91 Pops/s; x 2048: 262 us = 4.6 TB/s.
constexpr int I8P_THREADS = 320;
constexpr int I8P_EPI_WARPS = 8;
// How the pair kernel writes: from registers (the fp32 store, where 32 lanes write 128 bytes of a row;
// any alignment), the SwiGLU with a low plane, or through shared memory (rows aligned to 16 bytes).
// The SwiGLU's 32 tokens x 16 features go out by TMA: stores of 2 bytes and their addresses were the
// longest part of its epilogue. A residual's 16 tokens x 32 features are turned, so that it is read
// and written 16 bytes a lane (65536 x 2048 x 2048 262 us, from registers 320; by TMA 289, its small
// copies queued with the operands'; only a K of 512 went faster so, 16384 x 2048 61.5 us against 65.1).
enum I8Out { I8_DIRECT = 0, I8_PLANES = 1, I8_STAGED = 2 };

template <int EP, int OUT>
struct I8PairSmem {
  static constexpr int OP = 128 * I8_BK;                    // one operand of a stage
  static constexpr int STAGE = 2 * OP;
  static constexpr int STAGES = 6;
  static constexpr int TILES = OUT == I8_STAGED ? 2048 : 0;  // each epilogue warp's: one in fp32 or two in bf16
  static constexpr int XS = I8P_EPI_WARPS * 128 * 4;        // each epilogue warp's token scales
  static constexpr int BARS = 2 * STAGES + 4;
  static constexpr int TOTAL = 1024 + STAGES * STAGE + I8P_EPI_WARPS * TILES + XS + BARS * 8 + 16;
  static_assert(TOTAL <= 227 * 1024, "shared memory");
  static_assert(TOTAL >= kWholeTmemSmem, "a pair that takes all tensor memory columns has the SM to itself");
};

// CW neighbouring columns (tokens) of one accumulator lane (feature), stored at p and ldo apart.
// FULL: all of them are inside the batch.
template <int EP, bool FULL, int CW>
__device__ __forceinline__ void i8_finish(const I8Args& a, const uint32_t (&v)[CW], const float* xs, float ws, float* p,
                                          const float (&r)[CW], int left) {
#pragma unroll
  for (int j = 0; j < CW; j += 4) {
    const float4 x4 = *reinterpret_cast<const float4*>(xs + j);
    const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float y = i8_value(int(v[j + e]), x[e], ws);
      if constexpr (EP == B200_EP_RESID_ADD) y = __fadd_rn(r[j + e], y);
      if (FULL || j + e < left) p[size_t(j + e) * a.o.ldo] = y;
    }
  }
}

template <int EP, int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8P_THREADS, 1)
    gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                        const __grid_constant__ CUtensorMap tmO, const I8Args a) {
  using SM = I8PairSmem<EP, OUT>;
  extern __shared__ uint8_t i8_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = sW + SM::STAGES * SM::OP;
  uint8_t* sO = sX + SM::STAGES * SM::OP;  // [epilogue warp] tiles
  float* sxs = reinterpret_cast<float*>(sO + I8P_EPI_WARPS * SM::TILES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sxs + SM::XS / 4);
  uint64_t* full = bars;                            // the leader's are used
  uint64_t* empty = bars + SM::STAGES;              // both CTAs'
  uint64_t* acc_full = bars + 2 * SM::STAGES;       // [2], both CTAs'
  uint64_t* acc_empty = bars + 2 * SM::STAGES + 2;  // [2], the leader's are used
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + SM::BARS);

  const uint32_t rank = cluster_ctarank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nk = (a.k + I8_BK - 1) / I8_BK;
  const int bt = a.bt, th = bt / 2;
  const int n_tiles = (a.o.n_valid + 255) / 256, m_tiles = (a.m + bt - 1) / bt;
  const int n_units = n_tiles * m_tiles;
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  // groups of ngroup feature tiles; token tiles within a group, so that the weights a group
  // re-reads stay in L2 while the activations stream past
  const int G = a.ngroup;
  auto tile_of = [&](int u, int& mt, int& nt) {
    const int g = u / (G * m_tiles), r = u - g * G * m_tiles;
    const int gs = min(G, n_tiles - g * G);
    mt = r / gs;
    nt = g * G + r % gs;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < SM::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * I8P_EPI_WARPS);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers initialised and tensor memory allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  if (n_units <= n_pairs) pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tmW);
      tma_prefetch_desc(&tmX);
      const uint32_t full0 = mapa_shared(smem_addr(full), 0);
      const uint64_t keep = l2_evict_last_policy();  // weight tiles: re-read for every token tile
      int s = 0;
      uint32_t ph = 0;
      for (int u = pair; u < n_units; u += n_pairs) {
        int mt, nt;
        tile_of(u, mt, nt);
        const int n0 = nt * 256 + int(rank) * 128, t0 = mt * bt + int(rank) * th;
        for (int kt = 0; kt < nk; ++kt) {
          mbar_wait(&empty[s], ph ^ 1, FAULT_GEMM_WAIT_EMPTY);
          const uint32_t fb = full0 + 8u * s;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * (SM::OP + th * I8_BK));
          if constexpr (EP == B200_EP_SWIGLU)
            tma_load_5d_pair_hint(sW + s * SM::OP, &tmW, fb, kt * (I8_BK / 2), n0 / 128, keep);
          else
            tma_load_2d_pair_hint(sW + s * SM::OP, &tmW, fb, kt * (I8_BK / 2), n0, keep);
          tma_load_2d_pair(sX + s * SM::OP, &tmX, fb, kt * (I8_BK / 2), t0);
          if (++s == SM::STAGES) s = 0, ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      const uint32_t idesc = umma_idesc_i8(256, bt);
      int s = 0;
      uint32_t ph = 0, local = 0;
      for (int u = pair; u < n_units; u += n_pairs, ++local) {
        const uint32_t ab = local & 1, aph = (local >> 1) & 1;
        mbar_wait(&acc_empty[ab], aph ^ 1, FAULT_GEMM_WAIT_ACCUM);
        tc_fence_after();
        const uint32_t acc = tmem + ab * 256;
        for (int kt = 0; kt < nk; ++kt) {
          mbar_wait(&full[s], ph, FAULT_GEMM_WAIT_FULL_A);
          tc_fence_after();
          const uint64_t ad = umma_desc_sw128(smem_addr(sW + s * SM::OP));
          const uint64_t bd = umma_desc_sw128(smem_addr(sX + s * SM::OP));
#pragma unroll
          for (int j = 0; j < I8_BK / 32; ++j)  // 32 bytes of K per MMA = +2 in 16-byte units
            umma_pair_i8(acc, ad + 2 * j, bd + 2 * j, idesc, (kt != 0 || j != 0) ? 1u : 0u);
          umma_pair_commit_both(&empty[s]);  // both CTAs may refill stage s
          if (++s == SM::STAGES) s = 0, ph ^= 1;
        }
        umma_pair_commit_both(&acc_full[ab]);
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, hf = (warp - 2) >> 2;
    const uint32_t acc_empty0 = mapa_shared(smem_addr(acc_empty), 0);
    float* xs = sxs + (warp - 2) * 128;  // scales of this warp's 128 tokens
    uint8_t* tiles = sO + (warp - 2) * SM::TILES;
    // Store tiles: the g-th tile that this warp stores (tiles with nothing to store are left out, and
    // not written either) lies in buffer g % 2, free once the store before the last has read it.
    uint32_t sg = 0;
    auto free_tile = [&]() {
      if (lane == 0) tma_store_wait_read<1>();
      __syncwarp();
      return tiles + (sg++ & 1) * 1024;
    };
    auto tile_store = [&](const void* tile, int x, int y) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tma_store_2d(&tmO, tile, x, y);
    };
    // this lane's feature of a tile: its row, or in the SwiGLU's order of rows (i8_swiglu_map) gate
    // feature 16 q + lane % 16 in the lower lanes and the matching up feature in the upper ones
    const bool up = lane >= 16;
    const int row = EP == B200_EP_SWIGLU ? 16 * q + (lane & 15) + (up ? 64 : 0) : 32 * q + lane;
    // the channel scale and token scales of a unit, read while the unit before is finished
    float ws_next = 0.0f, xs_next[4] = {};
    auto scales = [&](int u) {
      int mt, nt;
      tile_of(u, mt, nt);
      const int n = nt * 256 + int(rank) * 128 + row, t0 = mt * bt + th * hf;
      ws_next = n < a.n ? a.ws[n] : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) xs_next[i] = t0 + 32 * i + lane < a.m ? a.xs[t0 + 32 * i + lane] : 0.0f;
    };
    if (pair < n_units) scales(pair);
    // Sums that a residual is added to go through a [16 tokens][32 features] tile, after which this
    // lane has four features, lf .. lf + 3, of every fourth token from lr on. Their residuals are read
    // three chunks of 16 tokens ahead, over the end of a unit too (two ahead: 1200 x 2048 x 2048 13.1 us
    // against 12.2).
    constexpr bool RES = OUT == I8_STAGED && EP == B200_EP_RESID_ADD;
    const int lr = lane >> 3, lf = 4 * (lane & 7);
    auto out_at = [&](int u, int& left) {
      int mt, nt;
      tile_of(u, mt, nt);
      const int t0 = mt * bt + th * hf, f = nt * 256 + int(rank) * 128 + 32 * q + lf;
      left = f < a.o.n_valid ? min(th, a.m - t0) - lr : 0;
      return static_cast<float*>(a.o.out) + size_t(t0 + lr) * a.o.ldo + f;
    };
    float4 res[4][4];
    auto residuals = [&](int c, float* p, int left) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (16 * c + 4 * i < left) res[c & 3][i] = *reinterpret_cast<const float4*>(p + size_t(16 * c + 4 * i) * a.o.ldo);
    };
    float* pn = nullptr;
    int ln = 0;
    if constexpr (RES) {
      if (pair < n_units) {
        pn = out_at(pair, ln);
        residuals(0, pn, ln);
        residuals(1, pn, ln);
        residuals(2, pn, ln);
      }
    }
    // The warp has an accumulator's sums in registers: the next products may overwrite it. Relaxed: no
    // memory is handed over, and a release would wait for this warp's stores.
    auto acc_read = [&](uint32_t ab) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(acc_empty0 + 8u * ab) : "memory");
    };
    uint32_t local = 0;
    for (int u = pair; u < n_units; u += n_pairs, ++local) {
      int mt, nt;
      tile_of(u, mt, nt);
      const int n0 = nt * 256 + int(rank) * 128, n = n0 + row;
      const int t0 = mt * bt + th * hf, left = min(th, a.m - t0);  // this warp's first token, and how many
      const uint32_t ab = local & 1, aph = (local >> 1) & 1;
      const uint32_t tl = tmem + ab * 256 + th * hf + (uint32_t(q * 32) << 16);
      const float ws = ws_next;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) xs[32 * i + lane] = xs_next[i];
      __syncwarp();
      if (u + n_pairs < n_units) scales(u + n_pairs);
      if constexpr (EP == B200_EP_SWIGLU) {
        // of two tokens the gate lane finishes the first and its up lane the second: each sends the
        // other the value it lacks
        const bool valid = n0 < a.o.n_valid;
        const size_t idx0 = size_t(t0 + (up ? 1 : 0)) * a.o.ldo + n0 / 2 + 16 * q + (lane & 15);
        uint32_t v[2][32];
        mbar_wait(&acc_full[ab], aph, FAULT_GEMM_WAIT_ACCUM);
        tc_fence_after();
        tmem_ld(tl, v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld_wait_for(v[c & 1]);
          if (c < 3) tmem_ld(tl + 32 * (c + 1), v[(c + 1) & 1]);
          else acc_read(ab);
          const int l = left - 32 * c;
          const size_t idx = idx0 + size_t(32 * c) * a.o.ldo;
          if (!valid || l <= 0) continue;  // the whole warp
          uint8_t* tile = nullptr;
          if constexpr (OUT == I8_STAGED) tile = free_tile();
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 x = *reinterpret_cast<const float4*>(xs + 32 * c + j);
            const float xe[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float y0 = i8_value(int(v[c & 1][j + e]), xe[e], ws);
              const float y1 = i8_value(int(v[c & 1][j + e + 1]), xe[e + 1], ws);
              const float other = __shfl_xor_sync(0xffffffffu, up ? y0 : y1, 16);
              const float g = up ? other : y0, uv = up ? y1 : other;
              if constexpr (OUT == I8_STAGED)
                reinterpret_cast<uint16_t*>(tile)[16 * (j + e) + lane] = f32_to_bf16_rn(swiglu(g, uv));
              else if (j + e + (up ? 1 : 0) < l)
                store_swiglu<OUT == I8_PLANES>(a.o, idx + size_t(j + e) * a.o.ldo, g, uv);
            }
          }
          if constexpr (OUT == I8_STAGED) tile_store(tile, n0 / 2 + 16 * q, t0 + 32 * c);
        }
      } else {
        float* p = static_cast<float*>(a.o.out) + size_t(t0) * a.o.ldo + n;
        const bool valid = n < a.o.n_valid;
        float* const po = pn;
        const int lo = ln;
        if constexpr (RES) {
          ln = 0;
          if (u + n_pairs < n_units) pn = out_at(u + n_pairs, ln);
        }
        // columns in hand (and as many ahead)
        constexpr int CW = EP == B200_EP_RESID_ADD ? 16 : 32;
        float r[2][CW];
        auto residual = [&](int c) {  // chunk c's residual, read while the chunk before is finished
          if constexpr (EP == B200_EP_RESID_ADD && OUT == I8_DIRECT) {
#pragma unroll
            for (int j = 0; j < CW; ++j)
              r[c & 1][j] = valid && CW * c + j < left ? p[size_t(CW * c + j) * a.o.ldo] : 0.0f;
          }
        };
        residual(0);
        uint32_t v[2][CW];
        mbar_wait(&acc_full[ab], aph, FAULT_GEMM_WAIT_ACCUM);
        tc_fence_after();
        tmem_ld(tl, v[0]);
#pragma unroll
        for (int c = 0; c < 128 / CW; ++c) {
          tmem_ld_wait_for(v[c & 1]);
          if (c + 1 < 128 / CW) {
            tmem_ld(tl + CW * (c + 1), v[(c + 1) & 1]);
            residual(c + 1);
          } else {
            acc_read(ab);
          }
          const int l = left - CW * c;
          if constexpr (RES) {
            if (c < 5) residuals(c + 3, po, lo);
            else residuals(c - 5, pn, ln);
            if (l > 0) {  // the whole warp
              float* const dst = reinterpret_cast<float*>(tiles);
              float* tile = dst + lane;
#pragma unroll
              for (int j = 0; j < CW; j += 4) {
                const float4 x = *reinterpret_cast<const float4*>(xs + CW * c + j);
                tile[32 * j] = i8_value(int(v[c & 1][j]), x.x, ws);
                tile[32 * (j + 1)] = i8_value(int(v[c & 1][j + 1]), x.y, ws);
                tile[32 * (j + 2)] = i8_value(int(v[c & 1][j + 2]), x.z, ws);
                tile[32 * (j + 3)] = i8_value(int(v[c & 1][j + 3]), x.w, ws);
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float4 y = *reinterpret_cast<const float4*>(dst + 32 * (4 * i + lr) + lf);
                const float4 r4 = res[c & 3][i];
                y = make_float4(__fadd_rn(r4.x, y.x), __fadd_rn(r4.y, y.y), __fadd_rn(r4.z, y.z), __fadd_rn(r4.w, y.w));
                if (16 * c + 4 * i < lo) *reinterpret_cast<float4*>(po + size_t(16 * c + 4 * i) * a.o.ldo) = y;
              }
            }
          } else if (valid) {
            float* pc = p + size_t(CW * c) * a.o.ldo;
            if (l >= CW) i8_finish<EP, true>(a, v[c & 1], xs + CW * c, ws, pc, r[c & 1], l);
            else i8_finish<EP, false>(a, v[c & 1], xs + CW * c, ws, pc, r[c & 1], l);
          }
          __syncwarp();
        }
      }
    }
  }

  if constexpr (OUT == I8_STAGED && EP == B200_EP_SWIGLU) {
    if (warp >= 2 && lane == 0) tma_store_wait_done();
  }
  tc_fence_before();
  cluster_sync_all();  // neither CTA leaves while the other may still read or signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ----------------------------------------------------------------------------- K split over a cluster
// One CTA = 128 features x bt tokens (a multiple of 16, at most 128) over its share of the K
// stages; the SPLIT CTAs of a tile form a cluster. Each turns its int32 sums around in shared
// memory ([token][feature], where its operands were), and after one cluster barrier CTA r adds the
// cluster's sums of tokens r * bt / SPLIT .. and finishes them. No partial sum reaches global
// memory and none is added atomically.
//   warp 0  TMA ring; warps 1 and 2  MMAs; then all warps drain the accumulators and finish outputs.
// Two threads issue MMAs. To issue one costs a thread 35 to 40 ns, more than the tensor cores need for
// 128 tokens or fewer, so each of two takes every second k-block, with an accumulator of its own (the
// sums are whole numbers: their order changes nothing). 96 x 8224 x 2048 on clusters of 2 8.4 us, with
// one issuer 9.1; 1021 x 2048 x 6144 17.8 : 21.2. (Half of every k-block each: 8.8 and 18.4 us.)
// At these sizes a launch is a chain of latencies. 96 x 8224 x 2048 on clusters of 2, 8.4 us in a row
// of launches, of which one takes 7.2: 0.5 set-up, 3 until the last MMA (8 k-blocks of 28 KB),
// 0.4 sums to shared memory, 0.7 cluster barrier, 1.3 outputs, 0.8 last barrier. In two token tiles
// of 48 instead, without a cluster, it takes 7.6.
// Warps per CTA. Without a cluster a CTA takes 16 (1021 x 2048 x 2048: 10.3 us against 11.3), with
// registers for two of them an SM (1 x 32768 x 2048 residual: 12.8 us against 17.1); CTAs of
// a cluster take 8, and the next launch's clusters find room beside them (32 x 2048 x 6144 on
// clusters of 8: 7.7 us against 12.6).
constexpr int i8s_warps(int split) { return split == 1 ? 16 : 8; }
constexpr int I8S_OP_W = 128 * I8_BK;
constexpr int I8S_MAX_STAGES = 12;
constexpr int I8S_RING = 220 * 1024;       // bytes of stages: one CTA per SM
constexpr int I8S_RING_HALF = 104 * 1024;  // two CTAs per SM
// Columns of tensor memory: the two accumulators.
__host__ __device__ constexpr int i8s_cols(int bt) { return bt <= 32 ? 64 : bt <= 64 ? 128 : 256; }
// Shared memory: what the CTA uses, and at least as large a share of the SM's as its columns are of
// 512. So whatever CTAs of this kernel an SM takes in, of several streams too, its tensor memory serves
// them all, and no cluster waits for columns that another holds while it waits for the first; nor
// beside a cluster kernel that takes all columns (kWholeTmemSmem).
constexpr int i8s_smem(int stages, int bt) {
  const int used = 1024 + stages * (I8S_OP_W + bt * I8_BK) + 128 * 4 + (4 * I8S_MAX_STAGES + 1) * 8 + 16;
  const int share = kSmSmem / 512 * i8s_cols(bt) - kCtaSmem;
  return used > share ? used : share;
}
static_assert(i8s_smem(2, 16) >= kClusterSmemMin, "two stages of 16 tokens are the least that a CTA asks for");

__device__ __forceinline__ int4 ld_cluster_s32x4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ int4 add4(int4 a, int4 b) { return make_int4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }

template <int EP, bool LO, int SPLIT>
__global__ void __launch_bounds__(32 * i8s_warps(SPLIT), SPLIT == 1 ? 2 : 1)
    gemm_i8_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                         const I8Args a) {
  extern __shared__ uint8_t i8_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8_smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int W = i8s_warps(SPLIT);
  const int bt = a.bt, stages = a.stages, x_op = bt * I8_BK;
  uint8_t* sW = smem;
  uint8_t* sX = sW + stages * I8S_OP_W;
  float* sxs = reinterpret_cast<float*>(sX + stages * x_op);  // [bt] token scales
  uint64_t* full = reinterpret_cast<uint64_t*>(sxs + 128);
  uint64_t* empty = full + 2 * I8S_MAX_STAGES;
  uint64_t* acc_full = empty + 2 * I8S_MAX_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  int* sP = reinterpret_cast<int*>(smem);  // [bt][128], once the operands are consumed

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % SPLIT, n0 = blockIdx.x / SPLIT * 128, t0 = blockIdx.y * bt;
  const int nk = (a.k + I8_BK - 1) / I8_BK;
  const int kb0 = int(int64_t(rank) * nk / SPLIT), kb1 = int(int64_t(rank + 1) * nk / SPLIT);
  const uint32_t cols = i8s_cols(bt) / 2;  // of one accumulator

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2 * stages; ++b) {
      mbar_init(&full[b], 1);
      mbar_init(&empty[b], 1);
    }
    mbar_init(acc_full, 2);
    mbar_fence_init();
    // weights that lie in HBM start for L2 before the wait for the kernel ahead (a prefetch:
    // nothing is read that it may still write)
    for (int kt = kb0; kt < min(kb1, kb0 + 2 * stages); ++kt) tma_prefetch_2d(&tmW, kt * (I8_BK / 2), n0);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x >= 128 && int(threadIdx.x) - 128 < bt)
    sxs[threadIdx.x - 128] = t0 + int(threadIdx.x) - 128 < a.m ? a.xs[t0 + threadIdx.x - 128] : 0.0f;

  if (warp == 0) {
    // k-block i of this CTA lies in stage i % stages; its barriers are number i % (2 stages), so that
    // a barrier always belongs to the same issuing thread, with an odd number of stages too
    if (lane == 0) {
      int s = 0, b = 0, be = 0;
      uint32_t ph = 0;
      for (int kt = kb0; kt < kb1; ++kt) {
        if (kt - kb0 >= stages) {
          mbar_wait(&empty[be], ph, FAULT_GEMM_WAIT_EMPTY);
          if (++be == 2 * stages) be = 0, ph ^= 1;
        }
        mbar_arrive_expect_tx(&full[b], I8S_OP_W + x_op);
        tma_load_2d(sW + s * I8S_OP_W, &tmW, &full[b], kt * (I8_BK / 2), n0);
        tma_load_2d(sX + s * x_op, &tmX, &full[b], kt * (I8_BK / 2), t0);
        if (++s == stages) s = 0;
        if (++b == 2 * stages) b = 0;
      }
    }
    __syncwarp();
  } else if (warp <= 2) {
    if (lane == 0) {  // issuer h: every second k-block, into its own accumulator
      const uint32_t idesc = umma_idesc_i8(128, bt), h = warp - 1, acc = tmem + h * cols;
      int b = h;
      uint32_t ph = 0;
      for (int kt = kb0 + h; kt < kb1; kt += 2) {
        const int s = b >= stages ? b - stages : b;
        mbar_wait(&full[b], ph, FAULT_GEMM_WAIT_FULL_A);
        tc_fence_after();
        const uint64_t ad = umma_desc_sw128(smem_addr(sW + s * I8S_OP_W));
        const uint64_t bd = umma_desc_sw128(smem_addr(sX + s * x_op));
#pragma unroll
        for (int j = 0; j < I8_BK / 32; ++j)
          umma_i8(acc, ad + 2 * j, bd + 2 * j, idesc, (kt >= kb0 + 2 || j != 0) ? 1u : 0u);
        umma_commit(&empty[b]);
        if ((b += 2) >= 2 * stages) b -= 2 * stages, ph ^= 1;
      }
      umma_commit(acc_full);
    }
    __syncwarp();
  }

  // what the outputs need besides the sums, read while the sums are formed: the channel scales of
  // this lane's four features, and the residual of the warp's first TB tokens
  const int cnt = bt / SPLIT, c0 = rank * cnt;
  const int c_end = min(c0 + cnt, a.m - t0);
  const int f = n0 + 4 * lane;
  constexpr int TB = SPLIT == 8 ? 2 : 4;  // tokens per batch: its loads are all issued before its first store
  float ws[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) ws[e] = f + e < a.n ? a.ws[f + e] : 0.0f;
  float4 r[TB];
  auto residual = [&](int cb) {
    if constexpr (EP == B200_EP_RESID_ADD) {
#pragma unroll
      for (int i = 0; i < TB; ++i) {
        const int c = cb + W * i;
        const float* p = static_cast<const float*>(a.o.out) + size_t(t0 + c) * a.o.ldo + f;
        r[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < c_end && f < a.o.n_valid) {
          if (a.vec && f + 4 <= a.o.n_valid) {
            r[i] = *reinterpret_cast<const float4*>(p);
          } else {
            r[i].x = p[0];
            if (f + 1 < a.o.n_valid) r[i].y = p[1];
            if (f + 2 < a.o.n_valid) r[i].z = p[2];
            if (f + 3 < a.o.n_valid) r[i].w = p[3];
          }
        }
      }
    }
  };
  residual(c0 + warp);
  mbar_wait(acc_full, 0, FAULT_GEMM_WAIT_ACCUM);
  tc_fence_after();
  __syncwarp();

  // ---- sums to shared memory: warp -> lane quarter warp % 4, every second 16 tokens
  const int q = warp & 3;
  for (int c = 16 * (warp >> 2); c < bt; c += 4 * W) {
    uint32_t v[16], v2[16] = {};
    tmem_ld(tmem + c + (uint32_t(q * 32) << 16), v);
    if (kb1 - kb0 > 1) tmem_ld(tmem + cols + c + (uint32_t(q * 32) << 16), v2);
    tmem_ld_wait_for(v);
    tmem_ld_wait_for(v2);
#pragma unroll
    for (int j = 0; j < 16; ++j) sP[(c + j) * 128 + 32 * q + lane] = int(v[j] + v2[j]);
  }
  tc_fence_before();
  if (SPLIT > 1) cluster_sync_all();
  else __syncthreads();

  // ---- this CTA's tokens: the cluster's sums, scaled and finished. A warp takes whole tokens,
  // four features per lane: 16-byte reads of each CTA's sums (4-byte ones through distributed
  // shared memory took the most of the kernel) and 16-byte stores where the output is aligned.
  const uint32_t base = smem_addr(sP);
  for (int cb = c0 + warp; cb < c_end; cb += W * TB) {
    if (cb != c0 + warp) residual(cb);
    int4 v[TB], part[TB][SPLIT];
#pragma unroll
    for (int i = 0; i < TB; ++i) {
      const int c = min(cb + W * i, c_end - 1);
#pragma unroll
      for (int s = 0; s < SPLIT; ++s) {
        if constexpr (SPLIT == 1) part[i][s] = *reinterpret_cast<const int4*>(sP + c * 128 + 4 * lane);
        else part[i][s] = ld_cluster_s32x4(mapa_shared(base + uint32_t(c * 128 + 4 * lane) * 4, s));
      }
    }
#pragma unroll
    for (int i = 0; i < TB; ++i) {
      v[i] = part[i][0];
#pragma unroll
      for (int s = 1; s < SPLIT; ++s) v[i] = add4(v[i], part[i][s]);
    }
#pragma unroll
    for (int i = 0; i < TB; ++i) {
      const int c = cb + W * i;
      if (c >= c_end) break;  // the whole warp
      const float xs = sxs[c];
      float y[4] = {i8_value(v[i].x, xs, ws[0]), i8_value(v[i].y, xs, ws[1]), i8_value(v[i].z, xs, ws[2]),
                    i8_value(v[i].w, xs, ws[3])};
      if constexpr (EP == B200_EP_SWIGLU) {
        // Lanes 0..15 hold gate features 4 l .. 4 l + 3, lanes 16..31 the up features of the same
        // outputs: the lower lane finishes the first two, the upper one the other two.
        const bool up = lane >= 16;
        const float a0 = __shfl_xor_sync(0xffffffffu, up ? y[0] : y[2], 16);
        const float a1 = __shfl_xor_sync(0xffffffffu, up ? y[1] : y[3], 16);
        if (n0 < a.o.n_valid) {
          const float g0 = up ? a0 : y[0], g1 = up ? a1 : y[1], u0 = up ? y[2] : a0, u1 = up ? y[3] : a1;
          const size_t idx = size_t(t0 + c) * a.o.ldo + n0 / 2 + 4 * (lane & 15) + (up ? 2 : 0);
          if (!LO && a.vec) {
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o.out) + idx) = pack_bf16x2(swiglu(g0, u0), swiglu(g1, u1));
          } else {
            store_swiglu<LO>(a.o, idx, g0, u0);
            store_swiglu<LO>(a.o, idx + 1, g1, u1);
          }
        }
      } else if (f < a.o.n_valid) {
        if constexpr (EP == B200_EP_RESID_ADD) {
          y[0] = __fadd_rn(r[i].x, y[0]);
          y[1] = __fadd_rn(r[i].y, y[1]);
          y[2] = __fadd_rn(r[i].z, y[2]);
          y[3] = __fadd_rn(r[i].w, y[3]);
        }
        float* p = static_cast<float*>(a.o.out) + size_t(t0 + c) * a.o.ldo + f;
        if (a.vec && f + 4 <= a.o.n_valid) {
          *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (f + e < a.o.n_valid) p[e] = y[e];
        }
      }
    }
  }
  if (SPLIT > 1) cluster_sync_all();  // no CTA leaves while its sums may still be read
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * cols);
  }
}

// ----------------------------------------------------------------------------- at most 16 tokens
// A matrix-vector product reads each weight once: no ring, barrier or tensor memory before the
// first MMA. A CTA owns RT 16-feature tiles (the SwiGLU: a gate tile and its up tile) over all of
// K; its W warps take the 64-code k-blocks warp, warp + W, ..., D of them in flight, and add their
// int32 sums through shared memory. Bound by HBM where there are weights enough (1 token, 98304 x
// 2048: 30.6 us = 6.6 TB/s; 12288 x 2048 SwiGLU 6.0 us = 4.2 TB/s), by the launch's chain of
// latencies below (2048 x 2048: 2.3 us).
// Lane (g, t) = (lane / 4, lane % 4) loads codes 16 t .. 16 t + 15 of its k-block of rows g and
// g + 8 (a quad reads 64 neighbouring bytes), and of tokens g and g + 8. mma.sync m16n8k32 takes 4
// codes of each row per register: MMA j = 0, 1 is given the words 2 j and 2 j + 1 of both operands,
// so its k-slots are the same columns on both sides, in an order the sum does not see.
constexpr int I8R_MAX_M = 16;

__device__ __forceinline__ void mma_s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 weight bytes, read once per call: no L1 allocation
__device__ __forceinline__ uint4 ld_stream_u4(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <int EP, int RT, int NT8, int W, int D, int CTAS>
__global__ void __launch_bounds__(32 * W, CTAS) gemm_i8_reg_kernel(const I8Args a) {
  static_assert(EP != B200_EP_SWIGLU || RT == 2, "a SwiGLU CTA holds a gate tile and its up tile");
  __shared__ int4 red[W][RT][NT8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int nkb = (a.k + 63) / 64;
  int row0[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if constexpr (EP == B200_EP_SWIGLU) row0[rt] = (blockIdx.x >> 2) * 128 + rt * 64 + (blockIdx.x & 3) * 16;
    else row0[rt] = (blockIdx.x * RT + rt) * 16;
  }
  // weights that lie in HBM start for L2 before the wait for the kernel ahead
  if (threadIdx.x == 0) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
      if (row0[rt] < a.n) bulk_prefetch_l2(a.w + size_t(row0[rt]) * a.k, uint32_t(min(16, a.n - row0[rt])) * a.k);
  }
  pdl_wait();
  pdl_trigger();

  const int ns = warp < nkb ? (nkb - warp + W - 1) / W : 0;
  uint4 wr[D][RT][2], xr[D][NT8];
  int acc[RT][NT8][4] = {};
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  auto load = [&](int d, int s) {
    const int k0 = (warp + W * s) * 64 + 16 * t;
    const bool in = k0 < a.k;  // k is a multiple of 16: a lane's 16 codes are all inside or all outside
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = row0[rt] + g + 8 * h;
        wr[d][rt][h] = in && row < a.n ? ld_stream_u4(a.w + size_t(row) * a.k + k0) : zero;
      }
#pragma unroll
    for (int i = 0; i < NT8; ++i) {
      const int tok = 8 * i + g;
      xr[d][i] = in && tok < a.m ? *reinterpret_cast<const uint4*>(a.q + size_t(tok) * a.ldx + k0) : zero;
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < ns) load(d, d);
  // what a finishing warp needs besides the sums: lane (g, t) finishes row g (e = 0, 1) and g + 8
  // (e = 2, 3) of tile rt for tokens 2 t (e = 0, 2) and 2 t + 1 of token tile i
  constexpr int SETS = (EP == B200_EP_SWIGLU ? 1 : RT) * NT8;  // (tile, 8 tokens) finished by a warp each
  const int rt = warp < SETS ? warp / NT8 : 0, i = warp % NT8;
  const int first = rt ? row0[RT - 1] : row0[0];
  float xs[2] = {}, ws[2] = {}, wu[2] = {}, res[4] = {};
  if (warp < SETS) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int tok = 8 * i + 2 * t + e, n = first + g + 8 * e;
      xs[e] = tok < a.m ? a.xs[tok] : 0.0f;
      ws[e] = n < a.n ? a.ws[n] : 0.0f;
      if constexpr (EP == B200_EP_SWIGLU) wu[e] = a.ws[row0[RT - 1] + g + 8 * e];
    }
    if constexpr (EP == B200_EP_RESID_ADD) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = 8 * i + 2 * t + (e & 1), n = first + g + 8 * (e >> 1);
        if (tok < a.m && n < a.o.n_valid) res[e] = static_cast<const float*>(a.o.out)[size_t(tok) * a.o.ldo + n];
      }
    }
  }
  for (int s0 = 0; s0 < ns; s0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (s0 + d < ns) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int i = 0; i < NT8; ++i) {
            const uint4 &u = wr[d][rt][0], &v = wr[d][rt][1], &x = xr[d][i];
            mma_s8_16832(acc[rt][i], u.x, v.x, u.y, v.y, x.x, x.y);
            mma_s8_16832(acc[rt][i], u.z, v.z, u.w, v.w, x.z, x.w);
          }
        if (s0 + d + D < ns) load(d, s0 + d + D);
      }
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int i = 0; i < NT8; ++i)
      red[warp][rt][i][lane] = make_int4(acc[rt][i][0], acc[rt][i][1], acc[rt][i][2], acc[rt][i][3]);
  __syncthreads();
  if (warp >= SETS) return;
  auto sums = [&](int r, int (&v)[4]) {
    v[0] = v[1] = v[2] = v[3] = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int4 p = red[w][r][i][lane];
      v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
    }
  };
  int v[4];
  sums(rt, v);
  if constexpr (EP == B200_EP_SWIGLU) {
    int u[4];
    sums(1, u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = 8 * i + 2 * t + (e & 1), l = g + 8 * (e >> 1);
      if (tok >= a.m) continue;
      const float gv = i8_value(v[e], xs[e & 1], ws[e >> 1]), uv = i8_value(u[e], xs[e & 1], wu[e >> 1]);
      const size_t idx = size_t(tok) * a.o.ldo + (blockIdx.x >> 2) * 64 + (blockIdx.x & 3) * 16 + l;
      if (a.o.lo_offset) store_swiglu<true>(a.o, idx, gv, uv);
      else store_swiglu<false>(a.o, idx, gv, uv);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = 8 * i + 2 * t + (e & 1), n = first + g + 8 * (e >> 1);
      if (tok >= a.m || n >= a.o.n_valid) continue;
      float y = i8_value(v[e], xs[e & 1], ws[e >> 1]);
      if constexpr (EP == B200_EP_RESID_ADD) y = __fadd_rn(res[e], y);
      static_cast<float*>(a.o.out)[size_t(tok) * a.o.ldo + n] = y;
    }
  }
}

// ----------------------------------------------------------------------------- host side
// Codes [rows, k] of ld bytes per row as 128-byte swizzled tiles of 128 codes x box_rows (two
// codes to a 16-bit element; columns and rows past the end read as zero).
static int i8_map(CUtensorMap* map, const void* base, int rows, int k, int ld, int box_rows) {
  const uint64_t dims[2] = {uint64_t(k) / 2, uint64_t(rows)};
  const uint64_t strides[1] = {uint64_t(ld)};
  const uint32_t box[2] = {I8_BK / 2, uint32_t(box_rows)};
  return encode_bf16_sw128(map, base, 2, dims, strides, box);
}

// The pair kernel's SwiGLU weight tile: a block's 64 gate and 64 up rows in the order 16 gate, the
// matching 16 up, the next 16 gate, ..., so that a warp's 32 accumulator lanes hold both values of
// its 16 outputs. Dimensions: code, row of 16, gate / up, 16s of the 64, block of 128 rows.
static int i8_swiglu_map(CUtensorMap* map, const void* base, int blocks, int k) {
  const uint64_t kk = uint64_t(k);
  const uint64_t dims[5] = {kk / 2, 16, 2, 4, uint64_t(blocks)};
  const uint64_t strides[4] = {kk, 64 * kk, 16 * kk, 128 * kk};
  const uint32_t box[5] = {I8_BK / 2, 16, 2, 4, 1};
  return encode_bf16_sw128(map, base, 5, dims, strides, box);
}

// CTA pairs of a pair kernel that the current device holds at once (and the kernel's attributes).
template <int EP, int OUT>
static int i8_device_pairs(int& pairs) {
  constexpr int smem = I8PairSmem<EP, OUT>::TOTAL;
  static DeviceOnce attr;
  static int max_pairs_dev[kMaxDevices] = {};  // written under attr's lock, once per device
  const int r = once_per_device(attr, [](int dev) -> int {
    SDB_CUDA(cudaFuncSetAttribute(gemm_i8_pair_kernel<EP, OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sm_count() & ~1);
    cfg.blockDim = dim3(I8P_THREADS);
    cfg.dynamicSmemBytes = smem;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, gemm_i8_pair_kernel<EP, OUT>, &cfg) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = sm_count() / 2;
    }
    max_pairs_dev[dev] = n;
    return B200_OK;
  });
  if (r != B200_OK) return r;
  int dev = 0;
  SDB_CUDA(cudaGetDevice(&dev));
  pairs = max_pairs_dev[dev];
  return B200_OK;
}

// The pair kernel's launch where the device holds `pairs` pairs at once.
template <int EP, int OUT>
static b200_launch_plan plan_i8_pair(const I8Args& a, int pairs) {
  using SM = I8PairSmem<EP, OUT>;
  // Tiles of 192 tokens where the pairs need no more rounds of them: a k-block takes 0.32 us instead of
  // 0.34 and the outputs less (1536 x 2048 x 2048 15.7 -> 14.3 us, 2560 x 2048 x 6144 43.9 -> 41.8); with
  // another round they lose (4096 x 2048 x 2048: 29.2 us against 25.6).
  const int n_tiles = (a.o.n_valid + 255) / 256;
  auto rounds = [&](int bt) {
    const int64_t units = int64_t(n_tiles) * ((a.m + bt - 1) / bt);
    return (units + pairs - 1) / pairs;
  };
  const int bt = rounds(192) == rounds(256) ? 192 : 256;
  // weights beyond what L2 keeps beside the activation stream: groups of about 40 MB
  const double tile_bytes = 256.0 * a.k;
  const int groups = n_tiles * tile_bytes <= 48e6 ? 1 : int(std::ceil(n_tiles * tile_bytes / 40e6));
  b200_launch_plan p = {};
  p.kernel = B200_KERNEL_INT8_PAIR;
  p.tile_n = 256;
  p.tile_m = bt;
  p.tiles = n_tiles * ((a.m + bt - 1) / bt);
  p.ctas = 2 * std::min(p.tiles, pairs);
  p.cluster = 2;
  p.threads = I8P_THREADS;
  p.smem_bytes = SM::TOTAL;
  p.tmem_cols = 512;
  p.stages = SM::STAGES;
  p.k_blocks = (a.k + I8_BK - 1) / I8_BK;
  p.group_tiles = (n_tiles + groups - 1) / groups;
  return p;
}

template <int EP, int OUT>
static int launch_i8_pair(I8Args a, cudaStream_t st) {
  int pairs = 0;
  if (int rc = i8_device_pairs<EP, OUT>(pairs)) return rc;
  const b200_launch_plan p = plan_i8_pair<EP, OUT>(a, pairs);
  a.bt = p.tile_m;
  a.ngroup = p.group_tiles;
  CUtensorMap mw, mx, mo;
  constexpr bool SW = EP == B200_EP_SWIGLU;
  if (int rc = SW ? i8_swiglu_map(&mw, a.w, a.o.n_valid / 128, a.k) : i8_map(&mw, a.w, a.n, a.k, a.k, 128)) return rc;
  if (int rc = i8_map(&mx, a.q, a.m, a.k, a.ldx, a.bt / 2)) return rc;
  mo = mw;  // not read
  if constexpr (SW && OUT == I8_STAGED) {
    if (int rc = encode_store_tile(&mo, a.o.out, a.m, a.o.n_valid / 2, a.o.ldo, 32, 16)) return rc;
  }
  SDB_CUDA(launch_pdl(gemm_i8_pair_kernel<EP, OUT>, dim3(p.ctas), dim3(I8P_THREADS), p.smem_bytes, st, mw, mx, mo, a));
  return B200_OK;
}

// How the pair kernel writes these outputs: f(its I8Out).
template <int EP, typename F>
static int with_i8_out(const b200_linear_out& o, F f) {
  constexpr bool SW = EP == B200_EP_SWIGLU;
  if constexpr (SW) {
    if (o.lo_offset) return f(std::integral_constant<int, I8_PLANES>{});
  }
  if constexpr (EP != B200_EP_STORE) {
    if (int64_t(o.ldo) * (SW ? 2 : 4) % 16 == 0 && (reinterpret_cast<uintptr_t>(o.out) & 15) == 0 &&
        (SW || o.n_valid % 4 == 0))
      return f(std::integral_constant<int, I8_STAGED>{});
  }
  return f(std::integral_constant<int, I8_DIRECT>{});
}

// The split kernel's launch on a device of `sms` SMs.
static b200_launch_plan plan_i8_split(const I8Args& a, int sms) {
  const int nk = (a.k + I8_BK - 1) / I8_BK, n_tiles = (a.o.n_valid + 127) / 128;
  // Tokens of a tile, at most: 128, or with 16 k-blocks or fewer the fewest of 32, 64 and 128 whose
  // tiles each have an SM. Where K is short, splitting the tokens is cheaper than splitting K, whose
  // sums cross the cluster (128 x 1024 x 1024 4.6 us against 5.7, 128 x 2048 x 2048 6.6 : 7.3, 96 x
  // 8224 x 2048 7.6 : 8.3; K 6144, 200 x 2048: 14.4 : 10.2).
  const bool shallow = nk <= 16;
  int most = shallow ? 32 : 128;
  while (most < 128 && int64_t(n_tiles) * ((a.m + most - 1) / most) > sms) most *= 2;
  int m_tiles = (a.m + most - 1) / most;
  const int bt = ((a.m + m_tiles - 1) / m_tiles + 15) / 16 * 16;
  m_tiles = (a.m + bt - 1) / bt;
  const int tiles = n_tiles * m_tiles;
  // K split over a cluster while SMs would idle and every CTA has two k-blocks. Clusters of 8 only
  // for at most 32 tokens: they wait longest for their SMs, and each of their CTAs reads as many sums
  // as one of 4 (2048 x 6144: 32 tokens 7.7 us against 8.3 on clusters of 4, 128 tokens 15.3 : 9.4).
  // At most 2 with 16 k-blocks or fewer (64 x 2048 x 2048 in tiles of 32: 5.8 us against 6.7 on 4).
  int split = 1;
  while (split < (shallow ? 2 : bt <= 32 ? 8 : 4) && 2 * split * tiles <= sms && 4 * split <= nk) split *= 2;
  // Half the shared memory per CTA when there are more CTAs than SMs (two run side by side: 300
  // x 12288 x 2048 17.8 -> 13.2 us), or when that ring holds most of the CTA's K anyway (the next
  // launch's CTAs then set up beside this one's: 32 x 2048 x 6144 12.1 -> 7.7 us), or for clusters of
  // 8 on most SMs, which else wait for one another's end (32 x 2048 x 8192 13.2 -> 8.7 us; on 64 SMs,
  // 1024 x 8192, 6.6 : 6.9); else the deeper ring (96 x 12288 x 2048: 8.9 us against 11.7).
  const int stage = I8S_OP_W + bt * I8_BK, nkb = (nk + split - 1) / split;
  const bool half = tiles * split > sms || 3 * (I8S_RING_HALF / stage) >= 2 * nkb ||
                    (split == 8 && 2 * tiles * split > sms);
  b200_launch_plan p = {};
  p.kernel = B200_KERNEL_INT8_SPLIT;
  p.tile_n = 128;
  p.tile_m = bt;
  p.tiles = tiles;
  p.ctas = tiles * split;
  p.cluster = split;
  p.threads = 32 * i8s_warps(split);
  // Two stages at least: the sums take their room.
  p.stages = std::min({I8S_MAX_STAGES, (half ? I8S_RING_HALF : I8S_RING) / stage, std::max(2, nkb)});
  p.k_blocks = nkb;
  p.smem_bytes = i8s_smem(p.stages, bt);
  p.tmem_cols = i8s_cols(bt);
  return p;
}

template <int EP, bool LO, int SPLIT>
static int launch_i8_cluster(const I8Args& a, const b200_launch_plan& p, cudaStream_t st) {
  static DeviceOnce attr;
  const int r = once_per_device(attr, [](int) -> int {
    SDB_CUDA(cudaFuncSetAttribute(gemm_i8_split_kernel<EP, LO, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  227 * 1024));
    return B200_OK;
  });
  if (r != B200_OK) return r;
  CUtensorMap mw, mx;
  if (int rc = i8_map(&mw, a.w, a.n, a.k, a.k, 128)) return rc;
  if (int rc = i8_map(&mx, a.q, a.m, a.k, a.ldx, a.bt)) return rc;
  const int n_tiles = (a.o.n_valid + 127) / 128;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(SPLIT * n_tiles, p.tiles / n_tiles);
  cfg.blockDim = dim3(p.threads);
  cfg.dynamicSmemBytes = p.smem_bytes;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = SPLIT;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = SPLIT > 1 ? 2 : 1;
  SDB_CUDA(cudaLaunchKernelEx(&cfg, gemm_i8_split_kernel<EP, LO, SPLIT>, mw, mx, a));
  return B200_OK;
}

template <int EP, bool LO>
static int launch_i8_split(I8Args a, cudaStream_t st) {
  const b200_launch_plan p = plan_i8_split(a, sm_count());
  a.bt = p.tile_m;
  a.stages = p.stages;
  switch (p.cluster) {
    case 1: return launch_i8_cluster<EP, LO, 1>(a, p, st);
    case 2: return launch_i8_cluster<EP, LO, 2>(a, p, st);
    case 4: return launch_i8_cluster<EP, LO, 4>(a, p, st);
    default: return launch_i8_cluster<EP, LO, 8>(a, p, st);
  }
}

template <int EP, int RT, int NT8, int W, int D, int CTAS>
static int launch_i8_reg(const I8Args& a, cudaStream_t st) {
  const int grid = (a.o.n_valid + 16 * RT - 1) / (16 * RT);
  SDB_CUDA(launch_pdl(gemm_i8_reg_kernel<EP, RT, NT8, W, D, CTAS>, dim3(grid), dim3(32 * W), 0, st, a));
  return B200_OK;
}
// Warps per CTA, depth and CTAs per SM, each the best of the shapes measured beside it (us, the
// others in brackets; all before the finishing operands were read early, which took 0.4 - 0.8 more
// off each):
//   SwiGLU, 12288 x 2048: 1 token 6.4 (7.7 - 9.9), 16 tokens 8.8 (10.2 - 11.0)
//   few tiles (about one CTA per SM), deep K: 16 warps share it (2048 x 6144, 1 token 4.0 against
//   6.9 on 8 warps); shallow K: 8 warps (2048 x 2048, 13 tokens 3.2 against 3.9 on 16)
//   many tiles, 8224 x 2048: 1 token 4.5 with four CTAs per SM (4.8 - 8.6), 16 tokens two tiles per
//   CTA 5.8 (6.9 - 9.6)
template <int EP, int NT8>
static int dispatch_i8_reg(const I8Args& a, cudaStream_t st) {
  if constexpr (EP == B200_EP_SWIGLU) {
    if constexpr (NT8 == 1) return launch_i8_reg<EP, 2, NT8, 8, 2, 3>(a, st);
    else return launch_i8_reg<EP, 2, NT8, 4, 3, 4>(a, st);
  } else {
    if ((a.o.n_valid + 15) / 16 <= 2 * sm_count())
      return a.k >= 4096 ? launch_i8_reg<EP, 1, NT8, 16, NT8 == 1 ? 6 : 4, 1>(a, st)
                         : launch_i8_reg<EP, 1, NT8, 8, 4, 2>(a, st);
    if constexpr (NT8 == 1) return launch_i8_reg<EP, 1, NT8, 8, 2, 4>(a, st);
    else return launch_i8_reg<EP, 2, NT8, 8, 2, 2>(a, st);
  }
}

// Whether the register kernel takes the product. It starts sooner, but loads through registers, and
// few CTAs share a long K: beyond some weight bytes, or some K, the split kernel's copies are faster.
// us, registers : split - 1 token, 12288 x 2048 SwiGLU 6.0 : 7.2, 24576 x 1024 6.1 : 7.0, 32768 x 2048
// store 15.0 : 12.4, 8192 x 3088 residual 7.1 : 8.4, 1024 x 16384 10.3 : 7.3, 1024 x 8192 4.2 : 4.9;
// SwiGLU of K 4096, 2048 outputs 5.4 : 4.6, 6144 9.4 : 8.0, K 3088 8.5 : 8.5; 16 tokens, SwiGLU 12288 x
// 1024 4.5 : 4.7, 8192 x 2048 7.4 : 6.6, 4096 x 3088 8.3 : 6.7, 4096 x 2048 5.1 : 5.6; residual 8192 x
// 3088 8.6 : 10.1, 32768 x 1024 10.1 : 8.0. With more feature tiles than two a SM, where the split
// kernel takes more than a round, 1 token 98304 x 2048 30.6 : 36.2, 49152 x 1024 10.0 : 12.5, 49152 x
// 6144 64 : 57; 16 tokens 98304 x 2048 39.8 : 37.6.
static bool i8_few_tokens(const I8Args& a, bool swiglu, int sms) {
  if (a.m > I8R_MAX_M) return false;
  const double bytes = double(a.o.n_valid) * a.k;
  if (a.m <= 8 && a.o.n_valid > 256 * sms) return a.k <= 2048;
  if (swiglu) return a.m <= 8 ? a.k < 4096 && bytes <= 32e6 : a.k <= 2048 && bytes <= 14e6;
  return a.k < 16384 && bytes <= (a.m <= 8 ? 32e6 : 26e6);
}

// The kernel that runs the product on a device of `sms` SMs.
static b200_linear_kernel i8_kernel(const I8Args& a, bool swiglu, int sms) {
  if (i8_few_tokens(a, swiglu, sms)) return B200_KERNEL_INT8_REG;
  // Single CTAs while each 128 x 128 tile has an SM (1021 x 2048 x 6144: 17.8 us, pairs 25). With two
  // of them to an SM, pairs if one round of them does (2000 x 2048 x 6144: 27.2 us against 46.2; 300 x
  // 8224 x 2048: 11.7 : 13.1), unless K is short, where two CTAs hide each other's set-up and outputs
  // (200 x 16384 x 512: 9.2 : 7.5; at K = 1024 both are within 8 %). Where pairs would take two
  // rounds, single CTAs (300 x 12288 x 2048: 13.0 us against 17.7). Pairs beyond (512 x 12288 x 2048:
  // 18.6 us against 22), but not for 32 tokens or fewer, of which a pair's tile would be almost empty
  // (32 x 98304 x 2048: 37.8 us in single CTAs, several rounds of them, against 43.6; 64 tokens 41 : 43,
  // 100 tokens 46 : 44).
  const int64_t tiles = int64_t((a.o.n_valid + 127) / 128) * ((a.m + 127) / 128);
  const int64_t pair_tiles = int64_t((a.o.n_valid + 255) / 256) * ((a.m + 255) / 256);
  return tiles <= sms || a.m <= 32 || (tiles <= 2 * sms && (2 * pair_tiles > sms || a.k <= 1024))
             ? B200_KERNEL_INT8_SPLIT
             : B200_KERNEL_INT8_PAIR;
}

template <int EP>
static int launch_int8(const I8Args& a, cudaStream_t st) {
  constexpr bool SW = EP == B200_EP_SWIGLU;
  switch (i8_kernel(a, SW, sm_count())) {
    case B200_KERNEL_INT8_REG: return a.m <= 8 ? dispatch_i8_reg<EP, 1>(a, st) : dispatch_i8_reg<EP, 2>(a, st);
    case B200_KERNEL_INT8_SPLIT:
      if constexpr (SW) {
        if (a.o.lo_offset) return launch_i8_split<EP, true>(a, st);
      }
      return launch_i8_split<EP, false>(a, st);
    default: return with_i8_out<EP>(a.o, [&](auto out) { return launch_i8_pair<EP, decltype(out)::value>(a, st); });
  }
}

// launch_int8's choices on a device of `sms` SMs (0: the current one).
template <int EP>
static int plan_int8(const I8Args& a, int sms, b200_launch_plan& p) {
  const int n_sm = sms ? sms : sm_count();
  p = {};
  switch (i8_kernel(a, EP == B200_EP_SWIGLU, n_sm)) {
    case B200_KERNEL_INT8_REG:
      p.kernel = B200_KERNEL_INT8_REG;
      p.cluster = 1;
      return B200_OK;
    case B200_KERNEL_INT8_SPLIT: p = plan_i8_split(a, n_sm); return B200_OK;
    default:
      return with_i8_out<EP>(a.o, [&](auto out) -> int {
        int pairs = std::max(1, sms / 2);
        if (!sms) {
          if (int rc = i8_device_pairs<EP, decltype(out)::value>(pairs)) return rc;
        }
        p = plan_i8_pair<EP, decltype(out)::value>(a, pairs);
        return B200_OK;
      });
  }
}

// The arguments of b200_linear_int8, checked.
static int i8_args(const int8_t* q, const float* x_scale, int32_t m, int32_t k, int32_t ldx, const b200_qweight* w,
                   const b200_linear_out* out, I8Args& a) {
  if (!q || !x_scale || !w || !out || !w->data || !out->out)
    return sdb_fail(B200_ERR_ARG, "b200_linear_int8: null pointer");
  if (w->format != B200_W_INT8) return sdb_fail(B200_ERR_FORMAT, "b200_linear_int8: needs a B200_W_INT8 weight");
  if (!w->row_scale) return sdb_fail(B200_ERR_ARG, "b200_linear_int8: missing row_scale");
  if (m <= 0 || k <= 0 || w->n <= 0) return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: empty shape");
  if (m > 1 << 30 || w->n > 1 << 30) return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: more than 2^30 rows");
  if (w->k != k) return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: q and W disagree on k");
  if (k % 16 != 0 || k > 65536)
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: k must be a multiple of 16, at most 65536");
  if (ldx < k || ldx % 16 != 0 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(w->data)) & 15))
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: q and W must be 16-byte aligned with ldx a multiple of 16");
  if (out->epilogue < 0 || out->epilogue > 2) return sdb_fail(B200_ERR_ARG, "b200_linear_int8: unknown epilogue");
  if (out->n_valid <= 0 || out->n_valid > w->n)
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: n_valid must be in (0, n]");
  const bool swiglu = out->epilogue == B200_EP_SWIGLU;
  if (swiglu && out->n_valid % 128 != 0)
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: SwiGLU needs n_valid % 128 == 0");
  if (out->ldo < (swiglu ? out->n_valid / 2 : out->n_valid))
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: ldo does not hold a row");
  if (reinterpret_cast<uintptr_t>(out->out) & (swiglu ? 1 : 3))
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: out is not aligned to its elements");
  if (out->lo_format != B200_LO_BF16 && out->lo_format != B200_LO_E4M3)
    return sdb_fail(B200_ERR_ARG, "b200_linear_int8: unknown lo_format");
  if ((reinterpret_cast<uintptr_t>(x_scale) | reinterpret_cast<uintptr_t>(w->row_scale)) & 3)
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: scales are not aligned to their elements");
  a = I8Args{q, x_scale, static_cast<const int8_t*>(w->data), w->row_scale, *out, m, w->n, k, ldx, 1, 0, 0, 0};
  a.vec = out->ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out->out) & (swiglu ? 7 : 15)) == 0;
  return B200_OK;
}

int sdb_linear_int8(const int8_t* q, const float* x_scale, int32_t m, int32_t k, int32_t ldx, const b200_qweight* w,
                    const b200_linear_out* out, cudaStream_t st) {
  I8Args a;
  if (int rc = i8_args(q, x_scale, m, k, ldx, w, out, a)) return rc;
  switch (out->epilogue) {
    case B200_EP_STORE: return launch_int8<B200_EP_STORE>(a, st);
    case B200_EP_RESID_ADD: return launch_int8<B200_EP_RESID_ADD>(a, st);
    default: return launch_int8<B200_EP_SWIGLU>(a, st);
  }
}

}  // namespace sdb

extern "C" int b200_linear_int8(const int8_t* q, const float* x_scale, int32_t m, int32_t k, int32_t ldx,
                                const b200_qweight* w, const b200_linear_out* out, b200_stream stream) {
  return sdb::sdb_linear_int8(q, x_scale, m, k, ldx, w, out, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int b200_linear_int8_plan(const int8_t* q, const float* x_scale, int32_t m, int32_t k, int32_t ldx,
                                     const b200_qweight* w, const b200_linear_out* out, int32_t sms,
                                     b200_launch_plan* plan) {
  using namespace sdb;
  if (!plan || sms < 0) return sdb_fail(B200_ERR_ARG, "b200_linear_int8_plan: no plan, or a negative number of SMs");
  I8Args a;
  if (int rc = i8_args(q, x_scale, m, k, ldx, w, out, a)) return rc;
  switch (out->epilogue) {
    case B200_EP_STORE: return plan_int8<B200_EP_STORE>(a, sms, *plan);
    case B200_EP_RESID_ADD: return plan_int8<B200_EP_RESID_ADD>(a, sms, *plan);
    default: return plan_int8<B200_EP_SWIGLU>(a, sms, *plan);
  }
}
