// Persistent tcgen05 GEMM with a choice of operand layouts and a fused epilogue, for the
// training operators:
//
//   D[r, c] = sum_k A(r, k) B(c, k)
//
// Each operand is either K-major (rows of contiguous k) or MN-major (rows of contiguous r or
// c, one row per k), so a gradient product reads its operands as they lie in memory:
//   dX = dY W      A = dY K-major,  B = W MN-major
//   dW = dY^T X    A = dY MN-major, B = X MN-major
// and no transposed copy is made. B is loaded as two halves of BN / 2 rows whose distance is
// an argument: BN / 2 for one matrix, F for the two stacked projections of a gated block, so
// gate and up columns of the same features meet in one accumulator tile.
//
// Roles: TMA warp, MMA warp, TMEM warp, and eight epilogue warps (two for each quarter of the
// accumulator's lanes, taking its columns in turn, because the epilogues here are more than a
// store); two TMEM accumulators, so that the epilogue of tile i runs beside the products of tile
// i+1.
// What bounds it: 128 x 256 tiles read 12 KB of shared memory per 16-deep MMA step (96 of its
// 128 cycles), so the tensor pipe, not shared memory, is the limit for BN = 256; BN = 64 and
// 128 are for grids that would otherwise leave SMs idle.
//
// Results leave through shared memory: an epilogue warp lays 32 rows x 128 bytes into its 4 KB
// buffer (128-byte swizzle, no bank conflicts) and a TMA store writes whole lines, while the warp
// goes on with the next columns. (Direct 16-byte stores, one row a lane, touch 32 lines an
// instruction.)
//
// The tensor cores add in fp32 but cut off instead of rounding, which over thousands of additions
// is a bias of 1e-6 relative and more. An Epi whose results are kept in fp32 asks for segments
// (SEG steps of 64): each is accumulated apart, and the epilogue adds them in registers, rounded.
//
// Epi is a functor type with Args, SEG and
//   static Row row(const GemmX&, const Args&, int r)
//   SEG == 0: template <int BN> static void tile(const GemmX&, const Args&, const Row&, const OutMaps&,
//                                 RowStage&, uint32_t tbase, int r, int tc, int sp, int half)
//   SEG > 0:  template <int BN> static void finish(const GemmX&, const Args&, const Row&,
//                                 float (&z)[BN / 2], int r, int tc, int half)
// called by every epilogue thread (accumulator row r, TMEM lane address tbase); `half` takes the
// 32- or 64-column pieces half, half + 2, ... of the tile.
#pragma once
#include <cuda.h>
#include "../common/om_ptx.cuh"

namespace om {

struct GemmX {
  int rows, cols;    // extents of D (for a gated pair: cols = F)
  int num_kb;        // 64-deep steps of the whole contraction
  int splits, kb_per_split;
  int tiles_r, tiles_c;
  int b_step;        // rows of B per column tile (K-major B): BN, or for a gated pair the features of a tile
  int b_box;         // rows of B that one of the two loads of a step brings (K-major B): BN / 2 or fewer
  int b_second;      // distance of the second half's rows (K-major B): BN / 2, or F
  int* status;
};

struct OutMaps {
  CUtensorMap m[3];  // what an Epi stores through; unused ones are zero
};

// The buffer of one epilogue warp.
struct RowStage {
  uint8_t* base;  // 4096 bytes, 1024-byte aligned
  int lane;
  __device__ __forceinline__ uint8_t* begin() const {  // its last store has been read
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
    return base;
  }
  // 32 bf16 columns into half `h` of the lane's 64-column row / 32 fp32 columns
  __device__ __forceinline__ void put(uint8_t* b, int h, const float (&f)[32]) const {
    const uint32_t row = smem_u32(b) + lane * 128;
#pragma unroll
    for (int j = 0; j < 4; ++j) sts128(row + (((h * 4 + j) ^ (lane & 7)) << 4), pack8(f + 8 * j));
  }
  // 32 bf16 columns as rows of 64 bytes (64-byte swizzle)
  __device__ __forceinline__ void put32(uint8_t* b, const float (&f)[32]) const {
    const uint32_t row = smem_u32(b) + lane * 64;
#pragma unroll
    for (int j = 0; j < 4; ++j) sts128(row + ((j ^ ((lane >> 1) & 3)) << 4), pack8(f + 8 * j));
  }
  __device__ __forceinline__ void put_f32(uint8_t* b, const float (&f)[32]) const {
    const uint32_t row = smem_u32(b) + lane * 128;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      sts128(row + ((j ^ (lane & 7)) << 4), make_uint4(__float_as_uint(f[4 * j]), __float_as_uint(f[4 * j + 1]),
                                                       __float_as_uint(f[4 * j + 2]), __float_as_uint(f[4 * j + 3])));
  }
  template <class F>
  __device__ __forceinline__ void end(F&& store) const {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      store();
      bulk_commit();
    }
  }
};

constexpr int GX_THREADS = 384;
constexpr int GX_GROUP = 16;  // row tiles walked before the next column tile: 16 x 9 tiles in flight share L2 lines

__device__ __forceinline__ void gx_coords(const GemmX& g, int u, int& tr, int& tc, int& sp) {
  sp = u % g.splits;
  const int t = u / g.splits;
  const int per = GX_GROUP * g.tiles_c;
  const int first = (t / per) * GX_GROUP;
  const int n = min(GX_GROUP, g.tiles_r - first);
  const int in = t % per;
  tr = first + in % n;
  tc = in / n;
}

// kind::f16, bf16 operands, fp32 accumulator; bit 15 / 16 select an MN-major A / B
__host__ __device__ constexpr uint32_t idesc_bf16_x(int M, int N, bool amn, bool bmn) {
  return idesc_bf16_f32(M, N) | (amn ? 1u << 15 : 0u) | (bmn ? 1u << 16 : 0u);
}

// AR: rows of A that are loaded, and the row tile. For a few tokens (32) the MMA has 64 rows, of which
// the last 32 are whatever follows in shared memory; they end in accumulator rows that are never
// read, and the room goes to stages. A 64-row accumulator has 16 rows in each quarter of the lanes.
template <int BN, int AR = 128>
struct GemmXCfg {
  static constexpr int BK = 64;
  static constexpr int MM = AR <= 64 ? 64 : 128;  // rows of the MMA
  static constexpr int A_BYTES = AR * BK * 2;
  static constexpr int B_BYTES = BN * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = (192 * 1024) / STAGE_BYTES > 16 ? 16 : (192 * 1024) / STAGE_BYTES;
  static constexpr int TMEM_COLS = BN <= 128 ? 2 * BN : 512;  // a power of two
  static constexpr int OUT_BYTES = 8 * 4096;  // eight epilogue warps; also what lies behind a short A
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + OUT_BYTES + 1024 /*align slack*/ + 512;
  static_assert((MM - AR) * BK * 2 <= B_BYTES + OUT_BYTES, "the MMA reads MM rows of A");
};

// Steps of one segment: the whole contraction (`kb1` is past its end) unless the Epi wants shorter ones.
template <class Epi>
__device__ __forceinline__ int gx_seg(int kb1) {
  return Epi::SEG ? Epi::SEG : kb1;
}

template <int BN, int AR, bool AMN, bool BMN, class Epi>
__global__ void __launch_bounds__(GX_THREADS, 1)
    gemm_ex_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ OutMaps outs, const GemmX g, const typename Epi::Args e) {
  using C = GemmXCfg<BN, AR>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* out_bytes = smem + C::STAGES * C::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(out_bytes + C::OUT_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drained = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = g.tiles_r * g.tiles_c * g.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 256);
    }
    mbar_init(drained, 1);
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 2) tmem_alloc(tmem_slot, C::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_wait();
  grid_release();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        int tr, tc, sp;
        gx_coords(g, u, tr, tc, sp);
        const int kb0 = sp * g.kb_per_split, kb1 = min(g.num_kb, kb0 + g.kb_per_split);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&empty[s], ((it / C::STAGES) & 1) ^ 1, g.status, OM_ERR_WAIT_EMPTY)) { ok = false; break; }
          uint8_t* a_dst = smem + s * C::STAGE_BYTES;
          uint8_t* b_dst = a_dst + C::A_BYTES;
          mbar_arrive_expect_tx(&full[s], C::A_BYTES + (BMN ? C::B_BYTES : 2 * g.b_box * 128));
          if constexpr (AMN) {
            tma_load_2d(a_dst, &tmA, &full[s], tr * 128, kb * 64);
            tma_load_2d(a_dst + 8192, &tmA, &full[s], tr * 128 + 64, kb * 64);
          } else {
            tma_load_2d(a_dst, &tmA, &full[s], kb * 64, tr * 128);
          }
          if constexpr (BMN) {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) tma_load_2d(b_dst + j * 8192, &tmB, &full[s], tc * BN + j * 64, kb * 64);
          } else {
            tma_load_2d(b_dst, &tmB, &full[s], kb * 64, tc * g.b_step);
            tma_load_2d(b_dst + C::B_BYTES / 2, &tmB, &full[s], kb * 64, tc * g.b_step + g.b_second);
          }
        }
      }
      if (!ok)  // wait (bounded) for the loads that may still be in flight
        for (int j = max(0, it - C::STAGES); j < it; ++j)
          mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, nullptr, 0);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t IDESC = idesc_bf16_x(C::MM, BN, AMN, BMN);
      int it = 0, local = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        int tr, tc, sp;
        gx_coords(g, u, tr, tc, sp);
        const int kb0 = sp * g.kb_per_split, kb1 = min(g.num_kb, kb0 + g.kb_per_split);
        for (int s0 = kb0; s0 < kb1 && ok; s0 += gx_seg<Epi>(kb1), ++local) {
          const int acc = local & 1, s1 = min(kb1, s0 + gx_seg<Epi>(kb1));
          if (!mbar_wait(&tempty[acc], ((local >> 1) & 1) ^ 1, g.status, OM_ERR_WAIT_ACCUM)) { ok = false; break; }
          tc_fence_after();
          for (int kb = s0; kb < s1; ++kb, ++it) {
            const int s = it % C::STAGES;
            if (!mbar_wait(&full[s], (it / C::STAGES) & 1, g.status, OM_ERR_WAIT_FULL)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a_addr = smem_u32(smem + s * C::STAGE_BYTES), b_addr = a_addr + C::A_BYTES;
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // 16 deep: 32 bytes of a K-major row, two 8-row atoms MN-major
              const uint64_t ad = AMN ? smem_desc_sw128_mn(a_addr + k * 2048, 8192, 1024)
                                      : smem_desc_sw128(a_addr + k * 32, 1024);
              const uint64_t bd = BMN ? smem_desc_sw128_mn(b_addr + k * 2048, 8192, 1024)
                                      : smem_desc_sw128(b_addr + k * 32, 1024);
              tc_mma_f16(tmem + acc * BN, ad, bd, IDESC, (kb > s0 || k > 0) ? 1u : 0u);
            }
            tc_commit(&empty[s]);
          }
          if (ok) tc_commit(&tfull[acc]);
        }
      }
      if (!ok) {  // wait (bounded) for the products that may still be running
        tc_commit(drained);
        mbar_wait(drained, 0, nullptr, 0);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - 4) >> 2;
    const RowStage stage{out_bytes + (warp - 4) * 4096, lane};
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    int local = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      int tr, tc, sp;
      gx_coords(g, u, tr, tc, sp);
      const int r = C::MM == 128 ? tr * 128 + q * 32 + lane : lane < 16 ? tr * 64 + q * 16 + lane : g.rows;
      const auto row = Epi::row(g, e, r);  // the row's own inputs, read while the products run
      if constexpr (Epi::SEG == 0) {
        const int acc = local & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&tfull[acc], (local >> 1) & 1, g.status, OM_ERR_WAIT_ACCUM));
        if (!ok) break;
        ++local;
        tc_fence_after();
        Epi::template tile<BN>(g, e, row, outs, stage, lanes + acc * BN, r, tc, sp, half);
        tc_fence_before();
        mbar_arrive(&tempty[acc]);
      } else {
        float z[BN / 2];
        const int kb0 = sp * g.kb_per_split, kb1 = min(g.num_kb, kb0 + g.kb_per_split);
        for (int s0 = kb0; s0 < kb1; s0 += gx_seg<Epi>(kb1), ++local) {
          const int acc = local & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&tfull[acc], (local >> 1) & 1, g.status, OM_ERR_WAIT_ACCUM));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < BN / 32; ++i) {  // 16 columns at a time: z takes most of the registers
            uint32_t v[16];
            tmem_ld_32x32b_x16(lanes + acc * BN + (2 * (i >> 1) + half) * 32 + (i & 1) * 16, v);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) z[i * 16 + j] = (s0 == kb0 ? 0.f : z[i * 16 + j]) + __uint_as_float(v[j]);
          }
          tc_fence_before();
          mbar_arrive(&tempty[acc]);
        }
        if (ok) Epi::template finish<BN>(g, e, row, z, r, tc, half);
      }
    }
    if (lane == 0) bulk_wait<0>();  // the stores are complete before the CTA's memory goes
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// The same GEMM on CTA pairs: one 256 x 256 tile a pair, half of A's and of B's rows in each CTA.
// A CTA brings 32 KB a 64-deep step instead of 48 and reads 8 KB of shared memory an MMA instead of
// 12: a third less traffic from L2 (where a 1-CTA grid draws 18 TB/s) and six stages instead of
// four to cover the memory's latency. For grids with enough 256 x 256 tiles. Measured: 4096 x 30464 x
// 5120 with the cross entropy's epilogue 770 us, tensor cores busy 95 % of the cycles (single CTAs 807 us,
// 89 %); a plain product 30464 x 5120 x 4096 808 us (852).
// B's halves are b_second rows apart (K-major B), as above: CTA 0 has the first, CTA 1 the second.
struct GemmPairCfg {
  static constexpr int BN = 256;
  static constexpr int A_BYTES = 128 * 64 * 2;
  static constexpr int STAGE_BYTES = 2 * A_BYTES;
  static constexpr int STAGES = 6;
  static constexpr int OUT_BYTES = 8 * 4096;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + OUT_BYTES + 1024 + 256;
};

template <bool AMN, bool BMN, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GX_THREADS, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ OutMaps outs, const GemmX g, const typename Epi::Args e) {
  using C = GemmPairCfg;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // both CTAs have the same layout: a location is the same offset in either
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* out_bytes = smem + C::STAGES * C::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(out_bytes + C::OUT_BYTES);  // the leader's count both CTAs' bytes
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;  // the leader's count both CTAs' epilogue warps
  uint64_t* drained = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = pair_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int units = g.tiles_r * g.tiles_c * g.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 16);
    }
    mbar_init(drained, 1);
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 2) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  pair_sync();
  tc_fence_after();
  grid_wait();
  grid_release();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer (each CTA its halves)
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      for (int u = pair; u < units && ok; u += pairs) {
        int tr, tc, sp;
        gx_coords(g, u, tr, tc, sp);
        const int kb0 = sp * g.kb_per_split, kb1 = min(g.num_kb, kb0 + g.kb_per_split);
        const int ra = tr * 256 + (int)rank * 128;
        const int rb = BMN ? tc * 256 + (int)rank * 128 : tc * g.b_step + (int)rank * g.b_second;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&empty[s], ((it / C::STAGES) & 1) ^ 1, g.status, OM_ERR_WAIT_EMPTY)) { ok = false; break; }
          uint8_t* a_dst = smem + s * C::STAGE_BYTES;
          uint8_t* b_dst = a_dst + C::A_BYTES;
          const uint32_t bar = pair_addr(&full[s], 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::STAGE_BYTES);
          if constexpr (AMN) {
            tma_load_2d_pair(a_dst, &tmA, bar, ra, kb * 64);
            tma_load_2d_pair(a_dst + 8192, &tmA, bar, ra + 64, kb * 64);
          } else {
            tma_load_2d_pair(a_dst, &tmA, bar, kb * 64, ra);
          }
          if constexpr (BMN) {
            tma_load_2d_pair(b_dst, &tmB, bar, rb, kb * 64);
            tma_load_2d_pair(b_dst + 8192, &tmB, bar, rb + 64, kb * 64);
          } else {
            tma_load_2d_pair(b_dst, &tmB, bar, kb * 64, rb);
          }
        }
      }
      if (!ok) {  // wait (bounded) for the loads that may still be in flight; only the leader can see them land
        if (rank == 0) {
          for (int j = max(0, it - C::STAGES); j < it; ++j)
            mbar_wait(&full[j % C::STAGES], (j / C::STAGES) & 1, nullptr, 0);
        } else {
          const uint64_t t0 = globaltimer();
          while (globaltimer() - t0 < 1000000ull) {
          }
        }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------ MMA issuer (the leader)
    if (elect_one()) {
      constexpr uint32_t IDESC = idesc_bf16_x(256, 256, AMN, BMN);
      int it = 0, local = 0;
      bool ok = true;
      for (int u = pair; u < units && ok; u += pairs) {
        int tr, tc, sp;
        gx_coords(g, u, tr, tc, sp);
        const int kb0 = sp * g.kb_per_split, kb1 = min(g.num_kb, kb0 + g.kb_per_split);
        for (int s0 = kb0; s0 < kb1 && ok; s0 += gx_seg<Epi>(kb1), ++local) {
          const int acc = local & 1, s1 = min(kb1, s0 + gx_seg<Epi>(kb1));
          if (!mbar_wait(&tempty[acc], ((local >> 1) & 1) ^ 1, g.status, OM_ERR_WAIT_ACCUM)) { ok = false; break; }
          tc_fence_after();
          for (int kb = s0; kb < s1; ++kb, ++it) {
            const int s = it % C::STAGES;
            if (!mbar_wait(&full[s], (it / C::STAGES) & 1, g.status, OM_ERR_WAIT_FULL)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a_addr = smem_u32(smem + s * C::STAGE_BYTES), b_addr = a_addr + C::A_BYTES;
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // 16 deep: 32 bytes of a K-major row, two 8-row atoms MN-major
              const uint64_t ad = AMN ? smem_desc_sw128_mn(a_addr + k * 2048, 8192, 1024)
                                      : smem_desc_sw128(a_addr + k * 32, 1024);
              const uint64_t bd = BMN ? smem_desc_sw128_mn(b_addr + k * 2048, 8192, 1024)
                                      : smem_desc_sw128(b_addr + k * 32, 1024);
              tc_mma_f16_pair(tmem + acc * 256, ad, bd, IDESC, (kb > s0 || k > 0) ? 1u : 0u);
            }
            tc_commit_pair(&empty[s]);
          }
          if (ok) tc_commit_pair(&tfull[acc]);
        }
      }
      if (!ok) {  // wait (bounded) for the products that may still be running
        tc_commit_pair(drained, 1);
        mbar_wait(drained, 0, nullptr, 0);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue (each CTA its 128 rows)
    const int q = warp & 3, half = (warp - 4) >> 2;
    const RowStage stage{out_bytes + (warp - 4) * 4096, lane};
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    int local = 0;
    bool ok = true;
    for (int u = pair; u < units && ok; u += pairs) {
      int tr, tc, sp;
      gx_coords(g, u, tr, tc, sp);
      const int r = tr * 256 + (int)rank * 128 + q * 32 + lane;
      const auto row = Epi::row(g, e, r);  // the row's own inputs, read while the products run
      if constexpr (Epi::SEG == 0) {
        const int acc = local & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&tfull[acc], (local >> 1) & 1, g.status, OM_ERR_WAIT_ACCUM));
        if (!ok) break;
        ++local;
        tc_fence_after();
        Epi::template tile<256>(g, e, row, outs, stage, lanes + acc * 256, r, tc, sp, half);
        tc_fence_before();
        __syncwarp();
          if (lane == 0) mbar_arrive_cluster(pair_addr(&tempty[acc], 0));
      } else {
        float z[256 / 2];
        const int kb0 = sp * g.kb_per_split, kb1 = min(g.num_kb, kb0 + g.kb_per_split);
        for (int s0 = kb0; s0 < kb1; s0 += gx_seg<Epi>(kb1), ++local) {
          const int acc = local & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&tfull[acc], (local >> 1) & 1, g.status, OM_ERR_WAIT_ACCUM));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < 256 / 32; ++i) {  // 16 columns at a time: z takes most of the registers
            uint32_t v[16];
            tmem_ld_32x32b_x16(lanes + acc * 256 + (2 * (i >> 1) + half) * 32 + (i & 1) * 16, v);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) z[i * 16 + j] = (s0 == kb0 ? 0.f : z[i * 16 + j]) + __uint_as_float(v[j]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(pair_addr(&tempty[acc], 0));
        }
        if (ok) Epi::template finish<256>(g, e, row, z, r, tc, half);
      }
    }
    if (lane == 0) bulk_wait<0>();
  }

  tc_fence_before();
  __syncthreads();
  pair_sync();  // neither CTA's memory goes while the other may still use it
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// n of 32 columns of one accumulator row, in 16-byte stores where they are whole.
__device__ __forceinline__ void store_row32(__nv_bfloat16* dst, const float (&f)[32], int n, bool vec) {
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    if (j + 8 <= n && vec) {
      *reinterpret_cast<uint4*>(dst + j) = pack8(f + j);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j + i < n) dst[j + i] = __float2bfloat16_rn(f[j + i]);
    }
  }
}
__device__ __forceinline__ void store_row32(float* dst, const float (&f)[32], int n, bool vec) {
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    if (j + 4 <= n && vec) {
      *reinterpret_cast<float4*>(dst + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i < n) dst[j + i] = f[j + i];
    }
  }
}

struct NoRow {};

// A factor of a whole product, applied in fp32 before its one rounding: mul times the mantissa (1 to
// 2) of *ref, where there is one. An operand that carries a value common to all its rows divides it
// out first, so that the value's rounding does not become a bias of every term.
struct Factor {
  const float* ref;
  float mul;
};
__device__ __forceinline__ float mantissa_of(float v) {
  const uint32_t u = __float_as_uint(v), e = (u >> 23) & 255u;
  return e == 0u || e == 255u ? 1.f : __uint_as_float((u & 0x007fffffu) | 0x3f800000u);
}
__device__ __forceinline__ float factor_of(const Factor& f) {
  return f.ref != nullptr ? f.mul * mantissa_of(*f.ref) : f.mul;
}

// bf16 rows through map 0, 64 columns a store.
struct EpiStore {
  struct Args {
    Factor factor;
  };
  static constexpr int SEG = 0;
  static __device__ __forceinline__ float row(const GemmX&, const Args& e, int) { return factor_of(e.factor); }
  template <int BN>
  static __device__ __forceinline__ void tile(const GemmX& g, const Args&, const float& factor, const OutMaps& o,
                                              const RowStage& st, uint32_t tbase, int r, int tc, int, int half) {
#pragma unroll 1
    for (int cc = half; cc < BN / 64; cc += 2) {
      const int c0 = tc * BN + cc * 64;
      if (c0 >= g.cols || r - st.lane >= g.rows) break;  // the same for the whole warp
      uint8_t* b = st.begin();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tbase + cc * 64 + h * 32, v);
        tc_wait_ld();
        float f[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]) * factor;
        st.put(b, h, f);
      }
      st.end([&] { tma_store_2d(&o.m[0], b, c0, r - st.lane); });
    }
  }
};

// fp32 sums [splits][rows][cols] through map 0: pieces of a long contraction (`add`: launches after
// the first) and splits are added up here. Every element has one writer a launch, so the order of
// the sum is the launches' order.
struct EpiSum {
  struct Args {
    int add;
  };
  static constexpr int SEG = 0;
  static __device__ __forceinline__ NoRow row(const GemmX&, const Args&, int) { return {}; }
  template <int BN>
  static __device__ __forceinline__ void tile(const GemmX& g, const Args& e, const NoRow&, const OutMaps& o,
                                              const RowStage& st, uint32_t tbase, int r, int tc, int sp, int half) {
#pragma unroll 1
    for (int cc = half; cc < BN / 32; cc += 2) {
      const int c0 = tc * BN + cc * 32;
      if (c0 >= g.cols || r - st.lane >= g.rows) break;
      uint8_t* b = st.begin();
      uint32_t v[32];
      tmem_ld_32x32b_x32(tbase + cc * 32, v);
      tc_wait_ld();
      float f[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
      st.put_f32(b, f);
      st.end([&] {
        if (e.add)
          tma_add_3d(&o.m[0], b, c0, r - st.lane, sp);
        else
          tma_store_3d(&o.m[0], b, c0, r - st.lane, sp);
      });
    }
  }
};

}  // namespace om
