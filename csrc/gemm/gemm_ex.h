// Host side of gemm_ex.cuh: tensor maps, launch and the plain products of the training
// operators.
#pragma once
#include "../common/om_host.h"
#include "gemm_ex.cuh"

namespace om {

inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Operand of logical extent [rows, K]: K-major (`ld` elements between rows), or MN-major (`ld`
// elements between k). A K-major box has `box` rows and 64 k, an MN-major one 64 x 64.
inline CUtensorMap gx_map(const void* p, bool mn, uint64_t rows, uint64_t K, uint64_t ld, uint32_t box) {
  return mn ? make_tmap_2d(p, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rows, K, ld, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B)
            : make_tmap_2d(p, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, K, rows, ld, 64, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Output maps of RowStage: boxes of 32 rows x 128 bytes. Rows start on 16 bytes.
inline CUtensorMap gx_out(__nv_bfloat16* p, uint64_t rows, uint64_t cols, uint64_t ld) {
  return make_tmap_2d(p, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, cols, rows, ld, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
}
// 32 columns a store (RowStage::put32)
inline CUtensorMap gx_out32(__nv_bfloat16* p, uint64_t rows, uint64_t cols, uint64_t ld) {
  return make_tmap_2d(p, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, cols, rows, ld, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}
inline CUtensorMap gx_out(float* p, uint64_t rows, uint64_t cols, uint64_t ld) {
  return make_tmap_2d(p, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, cols, rows, ld, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int BN, bool AMN, bool BMN, class Epi, int AR = 128>
void gx_launch(const CUtensorMap& ta, const CUtensorMap& tb, const OutMaps& outs, const GemmX& g,
               const typename Epi::Args& e, cudaStream_t st) {
  using C = GemmXCfg<BN, AR>;
  static std::atomic<bool> attr_set[64];
  int dev;
  OM_CUDA_CHECK(cudaGetDevice(&dev));
  if (!attr_set[dev].load()) {
    OM_CUDA_CHECK(cudaFuncSetAttribute(gemm_ex_kernel<BN, AR, AMN, BMN, Epi>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
    attr_set[dev].store(true);
  }
  const long long units = (long long)g.tiles_r * g.tiles_c * g.splits;
  TORCH_CHECK(units < (1ll << 31), "gemm: too many tiles");
  const int grid = (int)std::min<long long>(units, num_sms());
  launch_dependent(gemm_ex_kernel<BN, AR, AMN, BMN, Epi>, grid, GX_THREADS, C::SMEM_BYTES, st, ta, tb, outs, g, e);
}

// On CTA pairs; g.tiles_r counts 256-row tiles, K-major operands have boxes of 128 rows.
template <bool AMN, bool BMN, class Epi>
void gx_launch_pair(const CUtensorMap& ta, const CUtensorMap& tb, const OutMaps& outs, const GemmX& g,
                    const typename Epi::Args& e, cudaStream_t st) {
  static std::atomic<bool> attr_set[64];
  int dev;
  OM_CUDA_CHECK(cudaGetDevice(&dev));
  if (!attr_set[dev].load()) {
    OM_CUDA_CHECK(cudaFuncSetAttribute(gemm_pair_kernel<AMN, BMN, Epi>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       GemmPairCfg::SMEM_BYTES));
    attr_set[dev].store(true);
  }
  const long long units = (long long)g.tiles_r * g.tiles_c * g.splits;
  TORCH_CHECK(units < (1ll << 30), "gemm: too many tiles");
  const int pairs = (int)std::min<long long>(units, num_sms() / 2);
  launch_dependent(gemm_pair_kernel<AMN, BMN, Epi>, 2 * pairs, GX_THREADS, GemmPairCfg::SMEM_BYTES, st, ta, tb, outs, g, e);
}

// Whether a product goes to pairs: a 256 x 256 tile for every pair of SMs, rows that fill more than
// one half of a tile, and a contraction long enough for the setting up of a pair's tile (4096 rows,
// gated projection of 8192 / cross entropy of 32000, us on pairs and on single CTAs: K = 256 46 and 37 /
// 108 and 94; K = 512 58 and 56 / 120 and 109; K = 1024 89 and 102 / 175 and 190).
inline bool gx_pairs(int64_t rows, int64_t cols, int64_t K) {
  return rows > 128 && K >= 768 && (int64_t)ceil_div(rows, 256) * ceil_div(cols, 256) >= num_sms() / 2;
}

struct GxOperand {
  const void* p;
  bool mn;
  int64_t ld;
};

// out[rows, cols] (+)= A . B over K, split over K where the tiles alone leave SMs idle.
// `acc` (from gx_acc_floats) carries fp32 sums from piece to piece; first / last tell the piece's place.
struct GxPlan {
  int bn, splits, pair;
};
GxPlan gx_plan(int64_t rows, int64_t cols, int64_t K);
int64_t gx_acc_floats(const GxPlan& p, int64_t rows, int64_t cols, bool pieces);
void gx_product(const GxPlan& p, GxOperand a, GxOperand b, int64_t rows, int64_t cols, int64_t K,
                __nv_bfloat16* out, int64_t ldo, float* acc, bool first, bool last, int* status, cudaStream_t st,
                Factor factor = {nullptr, 1.f});

}  // namespace om
