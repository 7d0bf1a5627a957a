// Cross entropy of x W^T over a large vocabulary without the logits, and its gradient.
//
//   z = c x W^T            (columns that the keep mask leaves out are -inf)
//   lse = log sum_j exp z_j
//   loss = (1 - e) (lse - z_t) + e (lse - mean_j z_j)
//   dz_j = gloss (exp(z_j - lse) - e / V - (1 - e) [j = t]),   dx = c dz W,  dW = c dz^T x
//
// Forward: the GEMM's epilogue reduces each 128 x 256 tile of logits to one (max, sum of
// exponentials) pair a row, in base 2 and fp32, and picks z_t; a second kernel joins the pairs of
// a row in tile order. What leaves the chip is M V / 32 bytes instead of 4 M V.
//
// Gradient: the vocabulary is walked in pieces. Each piece's logits are computed again, and the
// epilogue turns them into dz (16 bits: its rounding is 2^-9 relative per entry and independent,
// like that of a stored activation) in a workspace of one piece; dx takes the piece's product
// into fp32 sums, dW's rows of the piece are finished at once. Four products instead of three is
// the price of not keeping M V values.
//
// What bounds it: the tensor cores (2 M K V flops a product). The epilogue's exponentials take
// 2048 cycles a tile beside 8 K cycles of products, on other warps.
#include <c10/cuda/CUDAGuard.h>
#include "gemm_ex.h"

namespace om {

constexpr float XE_LOG2E = 1.4426950408889634f;
constexpr float XE_LN2 = 0.6931471805599453f;

struct XentRows {
  const long long* targets;  // [M]
  const int* keep;           // optional [M, ldk] words, bit j of word i = column 32 i + j
  long long ldk;
  long long ignore;
  float scale;               // c
  int V;
};

// Fwd partials of row r and column tile tc: (max, sum 2^(z2 - max)) with z2 = z log2 e.
template <bool SMOOTH>
struct EpiXentFwd {
  struct Args {
    XentRows x;
    float2* part;   // [tiles_c][M]
    float* sumz;    // [tiles_c][M] sums of z (SMOOTH)
    float* zt;      // [M] z of the target, -inf if masked
  };
  template <int BN>
  static __device__ __forceinline__ void tile(const GemmX& g, const Args& e, uint32_t tbase, int r, int tc, int) {
    const bool row = r < g.rows;
    const int t0 = tc * BN;
    // the target's column within this tile, or a value no column has
    int tcol = -1;
    if (row) {
      const long long t = e.x.targets[r] - t0;
      tcol = t >= 0 && t < BN ? (int)t : -1;
    }
    const float c2 = e.x.scale * XE_LOG2E;
    float m = -INFINITY, s = 0.f, zs = 0.f;
#pragma unroll 1
    for (int cc = 0; cc < BN / 32; ++cc) {
      const int c0 = t0 + cc * 32;
      if (c0 >= g.cols) break;
      uint32_t v[32];
      tmem_ld_32x32b_x32(tbase + cc * 32, v);
      uint32_t bits = 0xffffffffu;
      if (g.cols - c0 < 32) bits = (1u << (g.cols - c0)) - 1u;
      if (e.x.keep != nullptr && row) bits &= (uint32_t)e.x.keep[r * e.x.ldk + (c0 >> 5)];
      tc_wait_ld();
      float f[32], mx = -INFINITY;
      if (bits == 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]) * c2;
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = (bits >> j) & 1u ? __uint_as_float(v[j]) * c2 : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) mx = fmaxf(mx, f[j]);
      if constexpr (SMOOTH) {
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) a += (bits >> j) & 1u ? __uint_as_float(v[j]) : 0.f;
        zs += a;
      }
      const float mn = fmaxf(m, mx);
      const float ref = mn == -INFINITY ? 0.f : mn;  // nothing kept so far: every term is 2^-inf = 0
      float a0 = 0.f, a1 = 0.f;
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        a0 += fast_exp2(f[j] - ref);
        a1 += fast_exp2(f[j + 1] - ref);
      }
      s = s * fast_exp2(m - ref) + (a0 + a1);
      m = mn;
      if ((tcol >> 5) == cc) {  // tcol = -1 matches no chunk
        const int j = tcol & 31;
        float z = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i == j && ((bits >> i) & 1u)) z = __uint_as_float(v[i]) * e.x.scale;
        e.zt[r] = z;
      }
    }
    if (row) {
      const size_t at = (size_t)tc * g.rows + r;
      e.part[at] = make_float2(m, s);
      if constexpr (SMOOTH) e.sumz[at] = zs * e.x.scale;
    }
  }
};

// Joins the column tiles of 32 rows: warp w takes tiles w, w + 8, ...; the eight partial results
// are joined in warp order (fixed order: the same result on every run).
__global__ void __launch_bounds__(256) xent_join_kernel(const float2* __restrict__ part, const float* __restrict__ sumz,
                                                        const float* __restrict__ zt, XentRows x, int M, int tiles,
                                                        float smoothing, float* __restrict__ loss,
                                                        float* __restrict__ lse, int* status) {
  __shared__ float sm[8][32], ss[8][32], sz[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f, z = 0.f;
  if (r < M) {
#pragma unroll 4
    for (int t = warp; t < tiles; t += 8) {
      const float2 p = part[(size_t)t * M + r];
      const float mn = fmaxf(m, p.x), ref = mn == -INFINITY ? 0.f : mn;
      s = s * exp2f(m - ref) + p.y * exp2f(p.x - ref);
      m = mn;
      if (sumz != nullptr) z += sumz[(size_t)t * M + r];
    }
  }
  sm[warp][lane] = m;
  ss[warp][lane] = s;
  sz[warp][lane] = z;
  __syncthreads();
  if (warp != 0 || r >= M) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) {
    const float mn = fmaxf(m, sm[w][lane]), ref = mn == -INFINITY ? 0.f : mn;
    s = s * exp2f(m - ref) + ss[w][lane] * exp2f(sm[w][lane] - ref);
    m = mn;
    z += sz[w][lane];
  }
  const float l = m == -INFINITY ? -INFINITY : (m + log2f(s)) * XE_LN2;
  lse[r] = l;
  const long long t = x.targets[r];
  float out = 0.f;
  if (t >= 0 && t < x.V && t != x.ignore) {
    const float a = zt[r];
    out = a == -INFINITY ? INFINITY : l - a;  // a target that the mask leaves out has probability 0
    if (smoothing != 0.f) out = (1.f - smoothing) * out + smoothing * (l - z / (float)x.V);
  } else if (t != x.ignore) {
    record_error(status, OM_ERR_BOUNDS);
  }
  loss[r] = out;
}

// dz of one vocabulary piece, 16 bits.
struct EpiXentBwd {
  struct Args {
    XentRows x;
    const float* lse;    // [M]
    const float* dloss;  // [M]
    float smoothing;
    int v0;              // the piece's first column
    __nv_bfloat16* dz;   // [M, ld], ld a multiple of 32
    int ld;
  };
  template <int BN>
  static __device__ __forceinline__ void tile(const GemmX& g, const Args& e, uint32_t tbase, int r, int tc, int) {
    const int t0 = tc * BN;
    float gz = 0.f, l2 = 0.f;
    int tcol = -1;
    if (r < g.rows) {
      const long long t = e.x.targets[r];
      if (t >= 0 && t < e.x.V && t != e.x.ignore) {
        gz = e.dloss[r] * e.x.scale;
        l2 = e.lse[r] * XE_LOG2E;
        const long long tt = t - e.v0 - t0;
        tcol = tt >= 0 && tt < BN ? (int)tt : -1;
      }
    }
    const float c2 = e.x.scale * XE_LOG2E;
    const float base = e.smoothing / (float)e.x.V;
#pragma unroll 1
    for (int cc = 0; cc < BN / 32; ++cc) {
      const int c0 = t0 + cc * 32;
      if (c0 >= g.cols) break;
      uint32_t v[32];
      tmem_ld_32x32b_x32(tbase + cc * 32, v);
      uint32_t bits = 0xffffffffu;
      if (e.x.keep != nullptr && r < g.rows) bits = (uint32_t)e.x.keep[r * e.x.ldk + ((e.v0 + c0) >> 5)];
      tc_wait_ld();
      if (r >= g.rows) continue;
      float f[32];
      if (gz == 0.f) {  // an ignored row: nothing, whatever its logits are
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = 0.f;
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = fast_exp2(__uint_as_float(v[j]) * c2 - l2) - base;
        if ((tcol >> 5) == cc) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j == (tcol & 31)) f[j] -= 1.f - e.smoothing;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = (bits >> j) & 1u ? f[j] * gz : 0.f;
      }
      // ld is a multiple of 32 and the workspace has whole rows: a short last chunk may fill its row's end
      store_row32(e.dz + (size_t)r * e.ld + c0, f, 32, true);
    }
  }
};

// Columns of one piece: dz of a piece stays within 256 MiB, in whole 256-column tiles.
static int64_t piece_columns(int64_t M, int64_t V) {
  const int64_t cap = std::max<int64_t>(2048, (256ll << 20) / (2 * M) / 256 * 256);
  const int64_t n = (V + cap - 1) / cap;
  return ((V + n - 1) / n + 255) / 256 * 256;
}

}  // namespace om

namespace {

void check_xent(const char* op, const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& targets,
                const c10::optional<torch::Tensor>& keep, double smoothing, om::XentRows& rows, double scale,
                int64_t ignore) {
  auto mat = [&](const torch::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1, op, ": ", name,
                " must be a 2-D bf16 CUDA tensor with contiguous rows");
    TORCH_CHECK(t.size(0) < (1ll << 31) && t.stride(0) < (1ll << 31), op, ": ", name, " is too large");
  };
  mat(x, "x");
  mat(w, "w");
  const int64_t M = x.size(0), K = x.size(1), V = w.size(0);
  TORCH_CHECK(w.size(1) == K && V > 0, op, ": w must be [V, K] with V > 0");
  TORCH_CHECK(K > 0 && K % 8 == 0, op, ": K must be a positive multiple of 8");
  TORCH_CHECK(targets.is_cuda() && targets.scalar_type() == at::kLong && targets.is_contiguous() &&
                  targets.dim() == 1 && targets.size(0) == M,
              op, ": targets must be int64 [M]");
  rows = om::XentRows{};
  rows.targets = reinterpret_cast<const long long*>(targets.data_ptr<int64_t>());
  rows.ignore = ignore;
  rows.scale = (float)scale;
  rows.V = (int)V;
  if (keep.has_value()) {
    TORCH_CHECK(smoothing == 0.0, op, ": label smoothing over a keep mask is not defined");
    TORCH_CHECK(keep->is_cuda() && keep->scalar_type() == at::kInt && keep->dim() == 2 && keep->size(0) == M &&
                    keep->size(1) >= (V + 31) / 32 && keep->stride(1) == 1,
                op, ": keep must be int32 [M, ceil(V / 32)] words");
    rows.keep = keep->data_ptr<int>();
    rows.ldk = keep->stride(0);
  }
}

}  // namespace

void om_linear_xent(torch::Tensor x, torch::Tensor w, torch::Tensor targets, c10::optional<torch::Tensor> keep,
                    double scale, double smoothing, int64_t ignore, torch::Tensor loss, torch::Tensor lse,
                    torch::Tensor status) {
  om::XentRows rows;
  check_xent("linear_xent", x, w, targets, keep, smoothing, rows, scale, ignore);
  const int64_t M = x.size(0), K = x.size(1), V = w.size(0);
  for (const auto& t : {loss, lse})
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == M,
                "linear_xent: loss and lse must be fp32 [M]");
  if (M == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  auto st = at::cuda::getCurrentCUDAStream().stream();
  om::GemmX g{};
  g.rows = (int)M;
  g.cols = (int)V;
  g.num_kb = om::ceil_div(K, 64);
  g.splits = 1;
  g.kb_per_split = g.num_kb;
  g.tiles_r = om::ceil_div(M, 128);
  g.tiles_c = om::ceil_div(V, 256);
  g.b_step = 256;
  g.b_second = 128;
  g.status = status.data_ptr<int>();
  const int64_t n = (int64_t)g.tiles_c * M;
  const bool smooth = smoothing != 0.0;
  auto ws = torch::empty({n * (smooth ? 3 : 2) + M}, loss.options());
  float* p = ws.data_ptr<float>();
  const CUtensorMap ta = om::gx_map(x.data_ptr(), false, M, K, x.stride(0), 128);
  const CUtensorMap tb = om::gx_map(w.data_ptr(), false, V, K, w.stride(0), 128);
  auto run = [&](auto epi) {
    using E = decltype(epi);
    typename E::Args e{rows, reinterpret_cast<float2*>(p), smooth ? p + 2 * n + M : nullptr, p + 2 * n};
    om::gx_launch<256, false, false, E>(ta, tb, g, e, st);
  };
  if (smooth)
    run(om::EpiXentFwd<true>{});
  else
    run(om::EpiXentFwd<false>{});
  om::xent_join_kernel<<<om::ceil_div(M, 32), 256, 0, st>>>(
      reinterpret_cast<float2*>(p), smooth ? p + 2 * n + M : nullptr, p + 2 * n, rows, (int)M, g.tiles_c,
      (float)smoothing, loss.data_ptr<float>(), lse.data_ptr<float>(), g.status);
  OM_LAUNCH_CHECK();
}

void om_linear_xent_bwd(torch::Tensor x, torch::Tensor w, torch::Tensor targets, c10::optional<torch::Tensor> keep,
                        double scale, double smoothing, int64_t ignore, torch::Tensor lse, torch::Tensor dloss,
                        c10::optional<torch::Tensor> dx, c10::optional<torch::Tensor> dw, torch::Tensor status) {
  om::XentRows rows;
  check_xent("linear_xent_bwd", x, w, targets, keep, smoothing, rows, scale, ignore);
  const int64_t M = x.size(0), K = x.size(1), V = w.size(0);
  for (const auto& t : {lse, dloss})
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == M,
                "linear_xent_bwd: lse and dloss must be fp32 [M]");
  auto grad = [&](const c10::optional<torch::Tensor>& t, int64_t r, const char* name) -> __nv_bfloat16* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kBFloat16 && t->dim() == 2 && t->size(0) == r &&
                    t->size(1) == K && t->is_contiguous(),
                "linear_xent_bwd: ", name, " has the wrong shape or type");
    return reinterpret_cast<__nv_bfloat16*>(t->data_ptr());
  };
  __nv_bfloat16* dxp = grad(dx, M, "dx");
  __nv_bfloat16* dwp = grad(dw, V, "dw");
  const c10::cuda::CUDAGuard guard(x.device());
  auto st = at::cuda::getCurrentCUDAStream().stream();
  if (M == 0) {
    if (dwp) dw->zero_();
    return;
  }
  if (!dxp && !dwp) return;
  const int64_t C = om::piece_columns(M, V);
  const int64_t ld = std::min(C, (V + 31) / 32 * 32);
  auto dz = torch::empty({M, ld}, x.options());
  const bool pieces = C < V;
  const om::GxPlan px = om::gx_plan(M, K, std::min(C, V));
  const om::GxPlan pw = om::gx_plan(std::min(C, V), K, M);
  const int64_t nx = dxp ? om::gx_acc_floats(px, M, K, pieces) : 0;
  const int64_t nw = dwp ? om::gx_acc_floats(pw, std::min(C, V), K, false) : 0;
  torch::Tensor ax, aw;
  if (nx) ax = torch::empty({nx}, lse.options());
  if (nw) aw = torch::empty({nw}, lse.options());
  om::GemmX g{};
  g.rows = (int)M;
  g.num_kb = om::ceil_div(K, 64);
  g.splits = 1;
  g.kb_per_split = g.num_kb;
  g.tiles_r = om::ceil_div(M, 128);
  g.b_step = 256;
  g.b_second = 128;
  g.status = status.data_ptr<int>();
  const CUtensorMap ta = om::gx_map(x.data_ptr(), false, M, K, x.stride(0), 128);
  const __nv_bfloat16* wp = reinterpret_cast<const __nv_bfloat16*>(w.data_ptr());
  for (int64_t v0 = 0; v0 < V; v0 += C) {
    const int64_t n = std::min(C, V - v0);
    const __nv_bfloat16* wv = wp + v0 * w.stride(0);
    g.cols = (int)n;
    g.tiles_c = om::ceil_div(n, 256);
    om::EpiXentBwd::Args e{rows,      lse.data_ptr<float>(), dloss.data_ptr<float>(),
                           (float)smoothing, (int)v0, reinterpret_cast<__nv_bfloat16*>(dz.data_ptr()), (int)ld};
    om::gx_launch<256, false, false, om::EpiXentBwd>(ta, om::gx_map(wv, false, n, K, w.stride(0), 128), g, e, st);
    if (dxp)
      om::gx_product(px, {dz.data_ptr(), false, ld}, {wv, true, w.stride(0)}, M, K, n, dxp, K,
                     nx ? ax.data_ptr<float>() : nullptr, v0 == 0, v0 + n == V, g.status, st);
    if (dwp)
      om::gx_product(pw, {dz.data_ptr(), true, ld}, {x.data_ptr(), true, x.stride(0)}, n, K, M, dwp + v0 * K, K,
                     nw ? aw.data_ptr<float>() : nullptr, true, true, g.status, st);
  }
}
