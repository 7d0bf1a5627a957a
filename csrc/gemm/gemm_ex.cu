// Plain products of the training operators on gemm_ex.cuh (dX = dY W, dW = dY^T X).
#include "gemm_ex.h"

namespace om {

// Sums the fp32 planes of a split contraction and rounds once. SUB lanes share four columns: lane
// group s adds planes s, s + SUB, ..., and the groups are added in order (one order, whatever the
// grid). SUB = 8 from 16 planes on, where the walk over the planes is what takes the time.
template <int SUB>
__global__ void __launch_bounds__(256) planes_to_bf16_kernel(const float* __restrict__ P, int splits, long long rows,
                                                             int cols, int ldacc, __nv_bfloat16* __restrict__ out,
                                                             long long ldo, int vec, Factor factor) {
  __shared__ float4 sh[SUB > 1 ? 256 : 1];
  grid_wait();
  grid_release();
  const float mul = factor_of(factor);
  const int nv = ldacc >> 2, lanes = 256 / SUB, sub = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const long long plane = rows * ldacc, n = rows * nv;
  for (long long i0 = blockIdx.x * (long long)lanes; i0 < n; i0 += gridDim.x * (long long)lanes) {
    const long long i = i0 + lane;
    const long long r = i / nv;
    const int c = (int)(i - r * nv) * 4;
    const bool live = i < n && c < cols;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
#pragma unroll 8
      for (int s = sub; s < splits; s += SUB) {
        const float4 b = *reinterpret_cast<const float4*>(P + s * plane + r * ldacc + c);
        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
      }
    }
    if constexpr (SUB > 1) {
      __syncthreads();
      sh[threadIdx.x] = a;
      __syncthreads();
      if (sub != 0) continue;
#pragma unroll
      for (int s = 1; s < SUB; ++s) {
        const float4 b = sh[s * lanes + lane];
        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
      }
    }
    if (!live) continue;
    a.x *= mul; a.y *= mul; a.z *= mul; a.w *= mul;
    __nv_bfloat16* o = out + r * ldo + c;
    if (vec && c + 4 <= cols) {
      uint2 w;
      w.x = pack_bf16x2(a.x, a.y);
      w.y = pack_bf16x2(a.z, a.w);
      *reinterpret_cast<uint2*>(o) = w;
    } else {
      const float f[4] = {a.x, a.y, a.z, a.w};
      for (int j = 0; j < 4 && c + j < cols; ++j) o[j] = __float2bfloat16_rn(f[j]);
    }
  }
}

GxPlan gx_plan(int64_t rows, int64_t cols, int64_t K) {
  const int sms = num_sms();
  const int64_t tr = ceil_div(rows, 128);
  const int kb = ceil_div(K, 64);
  // The launch lasts as long as its fullest SM: waves of tiles x the time of one. A 128-wide tile
  // takes 64 of the MMA's cycles a step, a 192-wide one 96 and a 256-wide one 128; shared memory
  // (A is read again for each) leaves the narrow ones 4 and 2 % behind.
  GxPlan p{256, 1, 0};
  if (gx_pairs(rows, cols, K)) {
    p.pair = 1;
    // Not split where the last wave leaves pairs idle: under the power limit the others run faster
    // meanwhile, and the fp32 planes cost more (4096 x 4096 x 22016: 519 us whole, 560 in two).
    return p;
  }
  double best = 1e300;
  for (int bn : {256, 192, 128}) {
    const int64_t tiles = tr * ceil_div(cols, bn);
    const double t = (double)ceil_div(tiles, sms) * bn * (bn == 128 ? 1.04 : bn == 192 ? 1.02 : 1.0);
    if (t < best) {
      best = t;
      p.bn = bn;
    }
  }
  const int64_t tiles = tr * ceil_div(cols, p.bn);
  // Split over K where that saves more steps than its fp32 planes (written and read once) and a second launch
  // take: at least 8 steps of 64 a split, and 16 saved in all and 2 more for each MB of planes. Split and not, us:
  // 688 x 256 x 1024 9.2 and 8.1, x 1536 9.9 and 9.9, x 2048 10.6 and 11.7, x 4096 12.1 and 18.9; 2048 x 512 (8.4 MB)
  // x 2048 14.2 and 12.5, x 4096 21.4 and 20.9, x 8192 41.7 and 46.9; 1024 x 512 x 2048 12.1 and 11.5, x 4096 14.9
  // and 17.3; 688 x 1024 x 2048 11.9 and 12.1, x 4096 15.2 and 19.1.
  const int s = (int)std::max<int64_t>(1, std::min<int64_t>(sms / tiles, kb / 8));
  const int per = ceil_div(kb, s), splits = ceil_div(kb, per);
  const double plane_mb = (double)rows * cols * 4e-6;
  if (splits > 1 && kb - per >= 16 + 2 * splits * plane_mb) p.splits = splits;
  return p;
}

int64_t gx_acc_floats(const GxPlan& p, int64_t rows, int64_t cols, bool pieces) {
  return p.splits > 1 || pieces ? (int64_t)p.splits * rows * ceil_div(cols, 32) * 32 : 0;
}

template <int BN, class Epi>
static void product_bn(GxOperand a, GxOperand b, const OutMaps& o, GemmX g, const typename Epi::Args& e, int64_t K,
                       cudaStream_t st) {
  g.tiles_c = ceil_div(g.cols, BN);
  const CUtensorMap ta = gx_map(a.p, a.mn, g.rows, K, a.ld, 128);
  const CUtensorMap tb = gx_map(b.p, true, g.cols, K, b.ld, 64);
  if (a.mn)
    gx_launch<BN, true, true, Epi>(ta, tb, o, g, e, st);
  else
    gx_launch<BN, false, true, Epi>(ta, tb, o, g, e, st);
}

template <class Epi>
static void product_pair(GxOperand a, GxOperand b, const OutMaps& o, GemmX g, const typename Epi::Args& e, int64_t K,
                         cudaStream_t st) {
  g.tiles_r = ceil_div(g.rows, 256);
  g.tiles_c = ceil_div(g.cols, 256);
  const CUtensorMap ta = gx_map(a.p, a.mn, g.rows, K, a.ld, 128);
  const CUtensorMap tb = gx_map(b.p, true, g.cols, K, b.ld, 64);
  if (a.mn)
    gx_launch_pair<true, true, Epi>(ta, tb, o, g, e, st);
  else
    gx_launch_pair<false, true, Epi>(ta, tb, o, g, e, st);
}

template <class Epi>
static void product(const GxPlan& p, GxOperand a, GxOperand b, const OutMaps& o, const GemmX& g,
                    const typename Epi::Args& e, int64_t K, cudaStream_t st) {
  if (p.pair)
    product_pair<Epi>(a, b, o, g, e, K, st);
  else if (p.bn == 128)
    product_bn<128, Epi>(a, b, o, g, e, K, st);
  else if (p.bn == 192)
    product_bn<192, Epi>(a, b, o, g, e, K, st);
  else
    product_bn<256, Epi>(a, b, o, g, e, K, st);
}

void gx_product(const GxPlan& p, GxOperand a, GxOperand b, int64_t rows, int64_t cols, int64_t K,
                __nv_bfloat16* out, int64_t ldo, float* acc, bool first, bool last, int* status, cudaStream_t st,
                Factor factor) {
  TORCH_CHECK(b.mn, "gx_product: B is MN-major");
  GemmX g{};
  g.rows = (int)rows;
  g.cols = (int)cols;
  g.num_kb = ceil_div(K, 64);
  g.kb_per_split = ceil_div(g.num_kb, p.splits);
  // a piece shorter than the planned one may have fewer splits: the planes it leaves out keep
  // the sums of the pieces before it (the first piece is never shorter than the plan's K)
  g.splits = ceil_div(g.num_kb, g.kb_per_split);
  TORCH_CHECK(!first || g.splits == p.splits, "gx_product: the first piece is shorter than planned");
  g.tiles_r = ceil_div(rows, 128);
  g.status = status;
  OutMaps o{};
  if (p.splits == 1 && first && last) {
    o.m[0] = gx_out(out, rows, cols, ldo);
    product<EpiStore>(p, a, b, o, g, {factor}, K, st);
    return;
  }
  const int ldacc = ceil_div(cols, 32) * 32;
  o.m[0] = make_tmap_3d(acc, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, cols, rows, p.splits, ldacc,
                        (uint64_t)rows * ldacc, 32, 32, 1, CU_TENSOR_MAP_SWIZZLE_128B);
  product<EpiSum>(p, a, b, o, g, {first ? 0 : 1}, K, st);
  if (last) {
    const bool many = p.splits >= 16;
    const long long work = (long long)rows * (ldacc / 4), lanes = many ? 32 : 256;
    const int blocks = (int)std::min<long long>((work + lanes - 1) / lanes, (long long)num_sms() * 8);
    launch_dependent(many ? planes_to_bf16_kernel<8> : planes_to_bf16_kernel<1>, blocks, 256, 0, st, acc, p.splits,
                     (long long)rows, (int)cols, ldacc, out, (long long)ldo,
                     (int)(ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0), factor);
  }
}

}  // namespace om
