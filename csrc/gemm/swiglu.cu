// Gated feed-forward projection and its gradient.
//
//   h = silu(g) * u,  g = x Wg^T,  u = x Wu^T,  W = [Wg; Wu]  [2F, K]
//
// Forward: one GEMM whose column tile holds BN / 2 gate columns beside the BN / 2 up columns of
// the same features (gemm_ex.cuh loads B in two halves F rows apart), so the activation and the
// product happen on the fp32 accumulators as they leave tensor memory; h is rounded once. For
// training, g and u are also stored, in 32 bits: dg and du are then rounded once, as operands of
// their products, and keeping them saves the gradient a third of its products.
//
// Gradient: s = 1 / (1 + exp(-g))
//   dg = dh u s (1 + g (1 - s)),  du = dh g s      one pass over g, u, dh
//   dx = [dg du] W,  dW = [dg du]^T x              two GEMMs that read both operands in place
//
// What bounds it: the tensor cores for M of a few hundred and more; the weight's bytes below
// (2 F K * 2 bytes for a single token). Measured (B200, back to back): 4096 x 4096 -> 11008, forward and
// gradient 1.85 to 1.90 ms, its three products at 1230 to 1270 TFLOP/s; one token, 8192 -> 28672 185 us (5.1 TB/s).
#include <c10/cuda/CUDAGuard.h>
#include "gemm_ex.h"

namespace om {

// exp(-g) = inf gives 0, as it should
__device__ __forceinline__ float sigmoid_f(float g) { return fast_rcp(1.f + fast_exp2(-1.4426950408889634f * g)); }

// Rows of h, g and u are laid out a multiple of 8 elements apart (ld: F rounded up), whatever F is.
// Maps: 0 h, 1 g, 2 u; without `maps` (narrow tiles) plain stores.
struct EpiSwiglu {
  struct Args {
    __nv_bfloat16* h;
    float* gu;  // optional [M, 2 ld]: g at column f, u at column ld + f
    int ld, maps;
  };
  static constexpr int SEG = 0;
  static __device__ __forceinline__ NoRow row(const GemmX&, const Args&, int) { return {}; }
  template <int BN>
  static __device__ __forceinline__ void tile(const GemmX& g, const Args& e, const NoRow&, const OutMaps& o,
                                              const RowStage& st, uint32_t tbase, int r, int tc, int, int half) {
    constexpr int HALF = BN / 2;
    const int F = g.cols, r0 = __shfl_sync(0xffffffffu, r, 0);
#pragma unroll 1
    for (int cc = half; cc < HALF / 32; cc += 2) {
      const int c0 = tc * g.b_step + cc * 32;
      if (c0 >= F || r0 >= g.rows) break;
      uint32_t gv[32], uv[32];
      tmem_ld_32x32b_x32(tbase + cc * 32, gv);
      tmem_ld_32x32b_x32(tbase + HALF + cc * 32, uv);
      tc_wait_ld();
      float gf[32], uf[32], hf[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        gf[j] = __uint_as_float(gv[j]);
        uf[j] = __uint_as_float(uv[j]);
        hf[j] = gf[j] * sigmoid_f(gf[j]) * uf[j];
      }
      if (HALF >= 64 && e.maps) {
        if (e.gu != nullptr) {
          uint8_t* b = st.begin();
          st.put_f32(b, gf);
          st.end([&] { tma_store_2d(&o.m[1], b, c0, r0); });
          b = st.begin();
          st.put_f32(b, uf);
          st.end([&] { tma_store_2d(&o.m[2], b, c0, r0); });
        }
        uint8_t* b = st.begin();
        st.put32(b, hf);
        st.end([&] { tma_store_2d(&o.m[0], b, c0, r0); });
        continue;
      }
      if (r >= g.rows) continue;
      const int n = min(min(32, g.b_step - cc * 32), F - c0);
      const bool vec = (c0 & 7) == 0;
      store_row32(e.h + (size_t)r * e.ld + c0, hf, n, vec);
      if (e.gu != nullptr) {
        store_row32(e.gu + (size_t)r * 2 * e.ld + c0, gf, n, vec);
        store_row32(e.gu + ((size_t)r * 2 + 1) * e.ld + c0, uf, n, vec);
      }
    }
  }
};

// dg, du, V columns a thread: 8 where dh's and the result's rows start on 16 bytes, else 1. The block
// is blockDim.x columns' worth by blockDim.y rows.
template <int V>
__global__ void __launch_bounds__(256) swiglu_grad_kernel(const float* __restrict__ gu, int ld,
                                                          const __nv_bfloat16* __restrict__ dh, long long lddh,
                                                          __nv_bfloat16* __restrict__ dgu, long long lddgu,
                                                          long long M, int F) {
  grid_wait();
  grid_release();
  const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V;
  if (c >= F) return;
  for (long long r = blockIdx.y * (long long)blockDim.y + threadIdx.y; r < M; r += gridDim.y * (long long)blockDim.y) {
    float g[V], u[V], d[V];
    const float* pg = gu + r * 2 * ld + c;
    if constexpr (V == 8) {
      const float4 g0 = reinterpret_cast<const float4*>(pg)[0], g1 = reinterpret_cast<const float4*>(pg)[1];
      const float4 u0 = reinterpret_cast<const float4*>(pg + ld)[0], u1 = reinterpret_cast<const float4*>(pg + ld)[1];
      unpack8(*reinterpret_cast<const uint4*>(dh + r * lddh + c), d);
      g[0] = g0.x; g[1] = g0.y; g[2] = g0.z; g[3] = g0.w; g[4] = g1.x; g[5] = g1.y; g[6] = g1.z; g[7] = g1.w;
      u[0] = u0.x; u[1] = u0.y; u[2] = u0.z; u[3] = u0.w; u[4] = u1.x; u[5] = u1.y; u[6] = u1.z; u[7] = u1.w;
    } else {
      g[0] = pg[0];
      u[0] = pg[ld];
      d[0] = __bfloat162float(dh[r * lddh + c]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float s = sigmoid_f(g[j]);
      const float dg = d[j] * u[j] * s * (1.f + g[j] * (1.f - s));
      u[j] = d[j] * g[j] * s;
      g[j] = dg;
    }
    __nv_bfloat16* o = dgu + r * lddgu + c;
    if constexpr (V == 8) {
      *reinterpret_cast<uint4*>(o) = pack8(g);
      *reinterpret_cast<uint4*>(o + F) = pack8(u);
    } else {
      o[0] = __float2bfloat16_rn(g[0]);
      o[F] = __float2bfloat16_rn(u[0]);
    }
  }
}

}  // namespace om

using om::GemmX;

namespace {

void check_swiglu(const char* op, const torch::Tensor& x, const torch::Tensor& w) {
  for (const auto& t : {x, w})
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() >= 1, op,
                ": x and w must be bf16 CUDA tensors");
  const int64_t K = x.size(-1);
  TORCH_CHECK(w.dim() == 2 && w.size(0) % 2 == 0 && w.size(1) == K, op, ": w must be [2F, K]");
  TORCH_CHECK(K > 0 && K % 8 == 0, op, ": K must be a positive multiple of 8");
  // a tile may reach 255 rows past the last one, whose index is 32 bits
  TORCH_CHECK(x.numel() / K < (1ll << 31) - 256 && w.size(0) < (1ll << 31) - 256 && K < (1ll << 30), op,
              ": too large");
}

}  // namespace

// (h [..., F] = silu(x Wg^T) * (x Wu^T), gu fp32 [rows, 2 Fp] if saved). Fp is F rounded up to 8: rows
// of h are Fp apart, so that F need not be a multiple of anything for whole-line stores.
std::pair<torch::Tensor, c10::optional<torch::Tensor>> om_swiglu(torch::Tensor x, torch::Tensor w, bool save,
                                                                 torch::Tensor status) {
  check_swiglu("swiglu", x, w);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t K = x.size(x.dim() - 1), F = w.size(0) / 2, M = x.numel() / K;
  const int64_t Fp = (F + 7) / 8 * 8;
  auto shape = x.sizes().vec();
  shape.back() = Fp;
  auto h = torch::empty(shape, x.options());
  if (Fp != F) h = h.narrow(-1, 0, F);
  c10::optional<torch::Tensor> gu;
  if (save) gu = torch::empty({M, 2 * Fp}, x.options().dtype(at::kFloat));
  if (M == 0 || F == 0) return {h, gu};
  const torch::Tensor x2 = om::tma_rows(x), w2 = om::tma_rows(w);
  auto st = at::cuda::getCurrentCUDAStream().stream();
  om::EpiSwiglu::Args e{};
  e.h = reinterpret_cast<__nv_bfloat16*>(h.data_ptr());
  e.ld = (int)Fp;
  if (save) e.gu = gu->data_ptr<float>();
  GemmX g{};
  g.rows = (int)M;
  g.cols = (int)F;
  g.num_kb = om::ceil_div(K, 64);
  g.splits = 1;
  g.kb_per_split = g.num_kb;
  g.tiles_r = om::ceil_div(M, 128);
  g.status = status.data_ptr<int>();
  const int sms = om::num_sms();
  g.b_second = (int)F;
  om::OutMaps o{};
  // 128 features a tile once those tiles fill the SMs and there is more than one row tile's worth of
  // work for each weight byte
  if (M > 128 && (int64_t)g.tiles_r * om::ceil_div(F, 128) >= sms) {
    const CUtensorMap ta = om::gx_map(x2.data_ptr(), false, M, K, x2.stride(0), 128);
    const CUtensorMap tb = om::gx_map(w2.data_ptr(), false, 2 * F, K, w2.stride(0), 128);
    g.b_step = g.b_box = 128;
    g.tiles_c = om::ceil_div(F, 128);
    e.maps = 1;
    o.m[0] = om::gx_out32(e.h, M, F, Fp);
    if (save) {
      o.m[1] = om::gx_out(e.gu, M, F, 2 * Fp);
      o.m[2] = om::gx_out(e.gu + Fp, M, F, 2 * Fp);
    }
    if (om::gx_pairs(M, 2 * F, K)) {
      g.tiles_r = om::ceil_div(M, 256);
      om::gx_launch_pair<false, false, om::EpiSwiglu>(ta, tb, o, g, e, st);
    } else {
      om::gx_launch<256, false, false, om::EpiSwiglu>(ta, tb, o, g, e, st);
    }
    return {h, gu};
  }
  // Few tokens, or a small layer: bound by the weight's bytes or by latency. At most 32 features a
  // tile, and as many (not a multiple of anything) as give every SM the same number of tiles:
  // 28672 features are 7 tiles of 28 on each of 148 SMs, where 32 each would leave a seventh idle.
  // With 32 tokens or fewer, A is loaded 32 rows high and the room is 16 stages of weights.
  const int waves = om::ceil_div((int64_t)g.tiles_r * om::ceil_div(F, 32), sms);
  const int64_t tiles = std::max<int64_t>(1, (int64_t)waves * sms / g.tiles_r);
  int64_t step = std::min<int64_t>(32, std::max<int64_t>(8, om::ceil_div(F, tiles)));
  if (M > 32) step = (step + 7) / 8 * 8;  // many rows: whole 16-byte stores matter more
  g.b_step = g.b_box = (int)step;
  g.tiles_c = om::ceil_div(F, g.b_step);
  const CUtensorMap ta = om::gx_map(x2.data_ptr(), false, M, K, x2.stride(0), M <= 32 ? 32 : 128);
  const CUtensorMap tb = om::gx_map(w2.data_ptr(), false, 2 * F, K, w2.stride(0), g.b_box);
  if (M <= 32)
    om::gx_launch<64, false, false, om::EpiSwiglu, 32>(ta, tb, o, g, e, st);
  else
    om::gx_launch<64, false, false, om::EpiSwiglu>(ta, tb, o, g, e, st);
  return {h, gu};
}

// (dx [..., K], dw [2F, K]) from x, w, gu (as the forward stored it) and dh [..., F].
std::pair<c10::optional<torch::Tensor>, c10::optional<torch::Tensor>> om_swiglu_bwd(torch::Tensor x, torch::Tensor w,
                                                                                    torch::Tensor gu, torch::Tensor dh,
                                                                                    bool need_dx, bool need_dw,
                                                                                    torch::Tensor status) {
  check_swiglu("swiglu_bwd", x, w);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t K = x.size(x.dim() - 1), F = w.size(0) / 2, M = x.numel() / K;
  const int64_t Fp = (F + 7) / 8 * 8;
  TORCH_CHECK(gu.is_cuda() && gu.scalar_type() == at::kFloat && gu.dim() == 2 && gu.size(0) == M &&
                  gu.size(1) == 2 * Fp && gu.is_contiguous() && (reinterpret_cast<uintptr_t>(gu.data_ptr()) & 15) == 0,
              "swiglu_bwd: gu must be the fp32 projections that swiglu saved");
  TORCH_CHECK(dh.is_cuda() && dh.numel() == M * F && (F == 0 || dh.size(-1) == F), "swiglu_bwd: dh must be [..., F]");
  c10::optional<torch::Tensor> dx, dw;
  if (need_dx) dx = torch::empty(x.sizes(), x.options());
  if (need_dw) dw = torch::empty(w.sizes(), w.options());
  if (M == 0 || F == 0) {
    if (need_dx) dx->zero_();
    if (need_dw) dw->zero_();
    return {dx, dw};
  }
  const torch::Tensor x2 = om::tma_rows(x), w2 = om::tma_rows(w), d2 = om::rows_view(dh.to(at::kBFloat16));
  auto st = at::cuda::getCurrentCUDAStream().stream();
  const int64_t ld = (2 * F + 7) / 8 * 8;
  auto dgu = torch::empty({M, ld}, x.options());
  auto ptr = [](const torch::Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); };
  const bool v8 = F % 8 == 0 && d2.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(d2.data_ptr()) & 15) == 0;
  const int cols = (int)(v8 ? F / 8 : F);
  int bx = 32;
  while (bx < 256 && bx < cols) bx *= 2;
  const dim3 block(bx, 256 / bx);
  const dim3 blocks(om::ceil_div(cols, bx), (unsigned)std::min<int64_t>(om::ceil_div(M, block.y), 65535));
  om::launch_dependent(v8 ? om::swiglu_grad_kernel<8> : om::swiglu_grad_kernel<1>, blocks, block, 0, st,
                       (const float*)gu.data_ptr<float>(), (int)Fp, (const __nv_bfloat16*)ptr(d2),
                       (long long)d2.stride(0), ptr(dgu), (long long)ld, (long long)M, (int)F);
  auto product = [&](om::GxOperand a, om::GxOperand b, int64_t rows, int64_t cols, int64_t k, torch::Tensor& out) {
    const om::GxPlan p = om::gx_plan(rows, cols, k);
    const int64_t n = om::gx_acc_floats(p, rows, cols, false);
    torch::Tensor acc;
    if (n) acc = torch::empty({n}, gu.options());
    om::gx_product(p, a, b, rows, cols, k, ptr(out), cols, n ? acc.data_ptr<float>() : nullptr, true, true,
                   status.data_ptr<int>(), st);
  };
  if (need_dx) product({dgu.data_ptr(), false, ld}, {w2.data_ptr(), true, w2.stride(0)}, M, K, 2 * F, *dx);
  if (need_dw) product({dgu.data_ptr(), true, ld}, {x2.data_ptr(), true, x2.stride(0)}, 2 * F, K, M, *dw);
  return {dx, dw};
}
