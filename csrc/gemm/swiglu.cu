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
// (2 F K * 2 bytes for a single token).
#include <c10/cuda/CUDAGuard.h>
#include "gemm_ex.h"

namespace om {

// exp(-g) = inf gives 0, as it should
__device__ __forceinline__ float sigmoid_f(float g) { return fast_rcp(1.f + fast_exp2(-1.4426950408889634f * g)); }

// n of 32 fp32 columns
__device__ __forceinline__ void store_row32(float* dst, const float (&f)[32], int n, bool vec) {
  if (n >= 32 && vec) {
#pragma unroll
    for (int j = 0; j < 32; j += 4)
      *reinterpret_cast<float4*>(dst + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < n) dst[j] = f[j];
  }
}

struct EpiSwiglu {
  struct Args {
    __nv_bfloat16* h;
    float* gu;  // optional [M, ldgu]: g at column f, u at column F + f
    int ldh, ldgu, vec_h, vec_gu;
  };
  template <int BN>
  static __device__ __forceinline__ void tile(const GemmX& g, const Args& e, uint32_t tbase, int r, int tc, int) {
    constexpr int HALF = BN / 2;
    constexpr int CH = HALF < 32 ? HALF : 32;
    const int F = g.cols;
#pragma unroll 1
    for (int cc = 0; cc < HALF / CH; ++cc) {
      const int c0 = tc * HALF + cc * CH;
      if (c0 >= F) break;
      uint32_t gv[32], uv[32];
      tmem_ld_32x32b_x32(tbase + cc * CH, gv);
      tmem_ld_32x32b_x32(tbase + HALF + cc * CH, uv);
      tc_wait_ld();
      if (r >= g.rows) continue;
      const int n = min(CH, F - c0);
      float gf[32], uf[32], hf[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        gf[j] = __uint_as_float(gv[j]);
        uf[j] = __uint_as_float(uv[j]);
        hf[j] = gf[j] * sigmoid_f(gf[j]) * uf[j];
      }
      store_row32(e.h + (size_t)r * e.ldh + c0, hf, n, e.vec_h);
      if (e.gu != nullptr) {
        store_row32(e.gu + (size_t)r * e.ldgu + c0, gf, n, e.vec_gu);
        store_row32(e.gu + (size_t)r * e.ldgu + F + c0, uf, n, e.vec_gu && (F & 3) == 0);
      }
    }
  }
};

// dg, du of one row block; V = 8 where every row start and F allow 16-byte accesses, else 1.
template <int V>
__global__ void __launch_bounds__(256) swiglu_grad_kernel(const float* __restrict__ gu, long long ldgu,
                                                          const __nv_bfloat16* __restrict__ dh, long long lddh,
                                                          __nv_bfloat16* __restrict__ dgu, long long lddgu,
                                                          long long M, int F) {
  const int nv = F / V;
  const long long n = M * nv;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const long long r = i / nv;
    const int c = (int)(i - r * nv) * V;
    float g[V], u[V], d[V];
    if constexpr (V == 8) {
      const float4* pg = reinterpret_cast<const float4*>(gu + r * ldgu + c);
      const float4* pu = reinterpret_cast<const float4*>(gu + r * ldgu + F + c);
      const float4 g0 = pg[0], g1 = pg[1], u0 = pu[0], u1 = pu[1];
      g[0] = g0.x; g[1] = g0.y; g[2] = g0.z; g[3] = g0.w; g[4] = g1.x; g[5] = g1.y; g[6] = g1.z; g[7] = g1.w;
      u[0] = u0.x; u[1] = u0.y; u[2] = u0.z; u[3] = u0.w; u[4] = u1.x; u[5] = u1.y; u[6] = u1.z; u[7] = u1.w;
      unpack8(*reinterpret_cast<const uint4*>(dh + r * lddh + c), d);
    } else {
      g[0] = gu[r * ldgu + c];
      u[0] = gu[r * ldgu + F + c];
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

template <int BN>
static void swiglu_fwd_bn(const CUtensorMap& ta, const void* w, int64_t ldw, GemmX g, const EpiSwiglu::Args& e,
                          int64_t F, int64_t K, cudaStream_t st) {
  g.tiles_c = ceil_div(F, BN / 2);
  g.b_step = BN / 2;
  g.b_second = (int)F;
  gx_launch<BN, false, false, EpiSwiglu>(ta, gx_map(w, false, 2 * F, K, ldw, BN / 2), g, e, st);
}

}  // namespace om

using om::GemmX;

static void check_bf16_rows(const torch::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1, op, ": ", name,
              " must be a 2-D bf16 CUDA tensor with contiguous rows");
  TORCH_CHECK(t.size(0) < (1ll << 31) && t.size(1) < (1ll << 31) && t.stride(0) < (1ll << 31), op, ": ", name,
              " is too large");
}

static void check_gu(const torch::Tensor& t, const char* op, int64_t M, int64_t F) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == M && t.size(1) == 2 * F &&
                  t.is_contiguous() && 2 * F < (1ll << 31),
              op, ": gu must be fp32 [M, 2F]");
}

// h [M, F] = silu(x Wg^T) * (x Wu^T); gu fp32 [M, 2F] optional.
void om_swiglu(torch::Tensor x, torch::Tensor w, torch::Tensor h, c10::optional<torch::Tensor> gu,
               torch::Tensor status) {
  check_bf16_rows(x, "swiglu", "x");
  check_bf16_rows(w, "swiglu", "w");
  check_bf16_rows(h, "swiglu", "h");
  const int64_t M = x.size(0), K = x.size(1), F = w.size(0) / 2;
  TORCH_CHECK(w.size(0) == 2 * F && w.size(1) == K, "swiglu: w must be [2F, K]");
  TORCH_CHECK(h.size(0) == M && h.size(1) == F, "swiglu: h must be [M, F]");
  TORCH_CHECK(K > 0 && K % 8 == 0, "swiglu: K must be a positive multiple of 8");
  if (M == 0 || F == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  auto st = at::cuda::getCurrentCUDAStream().stream();
  om::EpiSwiglu::Args e{};
  e.h = reinterpret_cast<__nv_bfloat16*>(h.data_ptr());
  e.ldh = (int)h.stride(0);
  e.vec_h = h.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(e.h) & 15) == 0;
  if (gu.has_value()) {
    check_gu(*gu, "swiglu", M, F);
    e.gu = gu->data_ptr<float>();
    e.ldgu = (int)(2 * F);
    e.vec_gu = F % 2 == 0 && (reinterpret_cast<uintptr_t>(e.gu) & 15) == 0;
  }
  GemmX g{};
  g.rows = (int)M;
  g.cols = (int)F;
  g.num_kb = om::ceil_div(K, 64);
  g.splits = 1;
  g.kb_per_split = g.num_kb;
  g.tiles_r = om::ceil_div(M, 128);
  g.status = status.data_ptr<int>();
  const CUtensorMap ta = om::gx_map(x.data_ptr(), false, M, K, x.stride(0), 128);
  // 128 features a tile once those tiles fill the SMs; fewer tiles than SMs: 32 features a tile
  if ((int64_t)g.tiles_r * om::ceil_div(F, 128) >= om::num_sms())
    om::swiglu_fwd_bn<256>(ta, w.data_ptr(), w.stride(0), g, e, F, K, st);
  else
    om::swiglu_fwd_bn<64>(ta, w.data_ptr(), w.stride(0), g, e, F, K, st);
}

// dx [M, K], dw [2F, K] from x, w, gu (as the forward stored it) and dh [M, F].
void om_swiglu_bwd(torch::Tensor x, torch::Tensor w, torch::Tensor gu, torch::Tensor dh,
                   c10::optional<torch::Tensor> dx, c10::optional<torch::Tensor> dw, torch::Tensor status) {
  check_bf16_rows(x, "swiglu_bwd", "x");
  check_bf16_rows(w, "swiglu_bwd", "w");
  check_bf16_rows(dh, "swiglu_bwd", "dh");
  const int64_t M = x.size(0), K = x.size(1), F = w.size(0) / 2;
  TORCH_CHECK(w.size(0) == 2 * F && w.size(1) == K, "swiglu_bwd: w must be [2F, K]");
  check_gu(gu, "swiglu_bwd", M, F);
  TORCH_CHECK(dh.size(0) == M && dh.size(1) == F, "swiglu_bwd: dh must be [M, F]");
  TORCH_CHECK(K > 0 && K % 8 == 0, "swiglu_bwd: K must be a positive multiple of 8");
  const c10::cuda::CUDAGuard guard(x.device());
  auto st = at::cuda::getCurrentCUDAStream().stream();
  if (M == 0 || F == 0) {
    if (dx.has_value()) dx->zero_();
    if (dw.has_value()) dw->zero_();
    return;
  }
  const int64_t ld = (2 * F + 7) / 8 * 8;
  auto dgu = torch::empty({M, ld}, x.options());
  auto ptr = [](const torch::Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); };
  auto al = [](const torch::Tensor& t) {
    return t.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  };
  const bool v8 = F % 8 == 0 && (reinterpret_cast<uintptr_t>(gu.data_ptr()) & 15) == 0 && al(dh);
  const long long work = M * (v8 ? F / 8 : F);
  const int blocks = (int)std::min<long long>((work + 255) / 256, (long long)om::num_sms() * 16);
  if (v8)
    om::swiglu_grad_kernel<8><<<blocks, 256, 0, st>>>(gu.data_ptr<float>(), 2 * F, ptr(dh), dh.stride(0), ptr(dgu), ld, M,
                                                      (int)F);
  else
    om::swiglu_grad_kernel<1><<<blocks, 256, 0, st>>>(gu.data_ptr<float>(), 2 * F, ptr(dh), dh.stride(0), ptr(dgu), ld, M,
                                                      (int)F);
  OM_LAUNCH_CHECK();
  auto product = [&](om::GxOperand a, om::GxOperand b, int64_t rows, int64_t cols, int64_t k, torch::Tensor& out,
                     const char* name) {
    check_bf16_rows(out, "swiglu_bwd", name);
    TORCH_CHECK(out.size(0) == rows && out.size(1) == cols, "swiglu_bwd: ", name, " has the wrong shape");
    const om::GxPlan p = om::gx_plan(rows, cols, k);
    const int64_t n = om::gx_acc_floats(p, rows, cols, false);
    torch::Tensor acc;
    if (n) acc = torch::empty({n}, x.options().dtype(at::kFloat));
    om::gx_product(p, a, b, rows, cols, k, ptr(out), out.stride(0), n ? acc.data_ptr<float>() : nullptr, true, true,
                   status.data_ptr<int>(), st);
  };
  if (dx.has_value())
    product({dgu.data_ptr(), false, ld}, {w.data_ptr(), true, w.stride(0)}, M, K, 2 * F, *dx, "dx");
  if (dw.has_value())
    product({dgu.data_ptr(), true, ld}, {x.data_ptr(), true, x.stride(0)}, 2 * F, K, M, *dw, "dw");
}
