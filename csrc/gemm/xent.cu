// Cross entropy of x W^T over a large vocabulary without the logits, and its gradient.
//
//   z = c x W^T            (columns that the keep mask leaves out are -inf)
//   lse = log sum_j exp z_j
//   loss = (1 - e) (lse - z_t) + e (lse - mean_j z_j)
//   dz_j = gloss (exp(z_j - lse) - e / V - (1 - e) [j = t]),   dx = c dz W,  dW = c dz^T x
//
// Forward: the GEMM's epilogue reduces each 128 x 256 tile of logits to one (max, sum of
// exponentials) pair a row and half tile, in base 2 and fp32, and picks z_t; a second kernel joins
// the pairs of a row in a fixed order. What leaves the chip is M V / 16 bytes instead of 4 M V.
//
// Gradient: the vocabulary is walked in pieces. Each piece's logits are computed again, and the
// epilogue turns them into dz (16 bits) in a workspace of one piece; dx takes the piece's product
// into fp32 sums, dW's rows of the piece are finished at once. Four products instead of three is
// the price of not keeping M V values.
// What is rounded is dz without what all rows share: gloss / m ((p - e / V) / (1 - e) - [j = t]), m the
// mantissa of the first row's gloss. Under a mean loss every target's entry is then within p_t of
// -2^k and takes at most p_t from its rounding; with the common factor c (1 - e) m inside, all of
// them would be off by the same amount of up to 2^-9, the whole of an output's own rounding again.
// The factor is applied to the sums. Weights that differ by row keep the rounding of their own target's
// entry (up to 2^-9 of the row's dx): the weight has to be inside dz, over whose rows dW sums.
//
// What bounds it: the tensor cores (2 M K V flops a product). The epilogue's exponentials take
// 2048 cycles a tile beside 8 K cycles of products, on other warps. Measured (B200, back to back): 4096 x
// 5120 -> 152064, forward and gradient 18.8 to 19.2 ms, its four products at 1330 to 1360 TFLOP/s (the library GEMM's
// sustained rate is 1395); forward alone of 4000 x 2048 -> 32000 with a keep mask 397 us, 1320 TFLOP/s.
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

// Fwd partials of row r and half of column tile tc: (max, sum 2^(z2 - max)) with z2 = z log2 e. The
// logits are summed in segments of 1024: loss and lse stay in fp32, where the tensor cores' cutting
// off shows (K = 5120: 8e-7 of lse in one piece; the segments are added with rounding).
template <bool SMOOTH>
struct EpiXentFwd {
  struct Args {
    XentRows x;
    float2* part;   // [2 tiles_c][M]
    float* sumz;    // [2 tiles_c][M] sums of z (SMOOTH)
    float* zt;      // [M] z of the target, -inf if masked
  };
  static constexpr int SEG = 16;
  static __device__ __forceinline__ long long row(const GemmX& g, const Args& e, int r) {
    return r < g.rows ? e.x.targets[r] : -1;
  }
  template <int BN>
  static __device__ __forceinline__ void finish(const GemmX& g, const Args& e, const long long& target,
                                                float (&z)[BN / 2], int r, int tc, int half) {
    const bool row = r < g.rows;
    const float c2 = e.x.scale * XE_LOG2E;
    float m = -INFINITY, s = 0.f, zs = 0.f;
#pragma unroll
    for (int i = 0; i < BN / 64; ++i) {
      const int c0 = tc * BN + (2 * i + half) * 32;
      uint32_t bits = g.cols - c0 >= 32 ? 0xffffffffu : g.cols > c0 ? (1u << (g.cols - c0)) - 1u : 0u;
      if (e.x.keep != nullptr && row && bits) bits &= (uint32_t)e.x.keep[r * e.x.ldk + (c0 >> 5)];
      float* f = z + i * 32;  // z2 in place; masked columns -inf
#pragma unroll
      for (int j = 0; j < 32; ++j) f[j] *= c2;
      if constexpr (SMOOTH) {
#pragma unroll
        for (int j = 0; j < 32; ++j) zs += (bits >> j) & 1u ? f[j] : 0.f;
      }
      const long long in = target - c0;
      if (target >= 0 && in >= 0 && in < 32) {
        const uint32_t hit = bits & (1u << (int)in);  // a mask, not an index: registers stay registers
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) t += (hit >> j) & 1u ? f[j] : 0.f;
        e.zt[r] = hit ? t * XE_LN2 : -INFINITY;
      }
      if (bits != 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = (bits >> j) & 1u ? f[j] : -INFINITY;
      }
      float mn = m;
#pragma unroll
      for (int j = 0; j < 32; ++j) mn = fmaxf(mn, f[j]);
      const float ref = mn == -INFINITY ? 0.f : mn;  // nothing kept so far: every term is 2^-inf = 0
      float a0 = 0.f, a1 = 0.f;
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        a0 += fast_exp2(f[j] - ref);
        a1 += fast_exp2(f[j + 1] - ref);
      }
      s = s * fast_exp2(m - ref) + (a0 + a1);
      m = mn;
    }
    if (row) {
      const size_t at = (size_t)(2 * tc + half) * g.rows + r;
      e.part[at] = make_float2(m, s);
      if constexpr (SMOOTH) e.sumz[at] = zs * XE_LN2;
    }
  }
};

// Joins the column tiles of 32 rows: warp w takes tiles w, w + 16, ...; the sixteen partial results
// are joined in warp order (fixed order: the same result on every run).
constexpr int XE_JOIN = 16;
__global__ void __launch_bounds__(32 * XE_JOIN) xent_join_kernel(const float2* __restrict__ part,
                                                                 const float* __restrict__ sumz,
                                                                 const float* __restrict__ zt, XentRows x, int M,
                                                                 int tiles, float smoothing, float* __restrict__ loss,
                                                                 float* __restrict__ lse, int* status) {
  __shared__ float sm[XE_JOIN][32], ss[XE_JOIN][32], sz[XE_JOIN][32];
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f, z = 0.f;
  if (r < M) {
#pragma unroll 8
    for (int t = warp; t < tiles; t += XE_JOIN) {
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
  const long long t = x.targets[r];
#pragma unroll
  for (int w = 1; w < XE_JOIN; ++w) {
    const float mn = fmaxf(m, sm[w][lane]), ref = mn == -INFINITY ? 0.f : mn;
    s = s * exp2f(m - ref) + ss[w][lane] * exp2f(sm[w][lane] - ref);
    m = mn;
    z += sz[w][lane];
  }
  const float l = s == 0.f ? -INFINITY : (m + log2f(s)) * XE_LN2;  // no column: -inf; a NaN logit: NaN
  lse[r] = l;
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

// dz of one vocabulary piece, 16 bits, through map 0 ([M, piece], rows a multiple of 64 bytes).
struct EpiXentBwd {
  struct Args {
    XentRows x;
    const float* lse;    // [M]
    const float* dloss;  // [M]
    float smoothing;
    int v0;              // the piece's first column
  };
  static constexpr int SEG = 0;
  struct Row {
    float gz, l2;  // gloss / m (0: ignored), lse log2 e
    int tcol;      // the target's column in the piece, or -1
  };
  static __device__ __forceinline__ Row row(const GemmX& g, const Args& e, int r) {
    Row o{0.f, 0.f, -1};
    if (r >= g.rows) return o;
    const long long t = e.x.targets[r];
    if (t < 0 || t >= e.x.V || t == e.x.ignore) return o;
    o.gz = e.dloss[r] / mantissa_of(e.dloss[0]);
    o.l2 = e.lse[r] * XE_LOG2E;
    if (t >= e.v0 && t < e.v0 + (long long)g.cols) o.tcol = (int)(t - e.v0);
    return o;
  }
  template <int BN>
  static __device__ __forceinline__ void tile(const GemmX& g, const Args& e, const Row& w, const OutMaps& o,
                                              const RowStage& st, uint32_t tbase, int r, int tc, int, int half) {
    const float c2 = e.x.scale * XE_LOG2E;
    const float inv = 1.f / (1.f - e.smoothing), base = inv * e.smoothing / (float)e.x.V;
#pragma unroll 1
    for (int cc = half; cc < BN / 64; cc += 2) {
      const int c64 = tc * BN + cc * 64;
      if (c64 >= g.cols || r - st.lane >= g.rows) break;
      uint8_t* b = st.begin();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c0 = c64 + h * 32;
        uint32_t v[32];
        tmem_ld_32x32b_x32(tbase + cc * 64 + h * 32, v);
        uint32_t bits = 0xffffffffu;
        if (e.x.keep != nullptr && r < g.rows && c0 < g.cols)
          bits = (uint32_t)e.x.keep[r * e.x.ldk + ((e.v0 + c0) >> 5)];
        tc_wait_ld();
        float f[32];
        if (w.gz == 0.f) {  // an ignored row: nothing, whatever its logits are
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = 0.f;
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = fmaf(fast_exp2(__uint_as_float(v[j]) * c2 - w.l2), inv, -base);
          // tcol = -1 matches no column; a mask, not an index: registers stay registers
          const uint32_t hit = (w.tcol >> 5) == (c0 >> 5) ? 1u << (w.tcol & 31) : 0u;
          if (hit) {
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] -= (hit >> j) & 1u ? 1.f : 0.f;
          }
          if (bits == 0xffffffffu) {
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] *= w.gz;
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = (bits >> j) & 1u ? f[j] * w.gz : 0.f;
          }
        }
        st.put(b, h, f);
      }
      st.end([&] { tma_store_2d(&o.m[0], b, c64, r - st.lane); });
    }
  }
};

// Columns of one piece, in whole 256-column tiles: dz of a piece stays within 256 MiB, or takes 4096 M bytes
// where that is more (from 65536 rows on): narrower pieces would be launches of few tiles.
static int64_t piece_columns(int64_t M, int64_t V) {
  const int64_t cap = std::max<int64_t>(2048, (256ll << 20) / (2 * M) / 256 * 256);
  const int64_t n = (V + cap - 1) / cap;
  return ((V + n - 1) / n + 255) / 256 * 256;
}

}  // namespace om

namespace {

struct XentIn {
  torch::Tensor x, w, targets, keep;  // as the kernels read them
  int64_t M, K, V;
  om::XentRows rows{};
};

XentIn check_xent(const char* op, const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& targets,
                  const c10::optional<torch::Tensor>& keep, double smoothing, double scale, int64_t ignore) {
  for (const auto& t : {x, w})
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() >= 1, op,
                ": x and w must be bf16 CUDA tensors");
  XentIn in;
  in.K = x.size(x.dim() - 1);
  TORCH_CHECK(w.dim() == 2 && w.size(1) == in.K && w.size(0) > 0, op, ": w must be [V, K] with V > 0");
  TORCH_CHECK(in.K > 0 && in.K % 8 == 0, op, ": K must be a positive multiple of 8");
  in.M = x.numel() / in.K;
  in.V = w.size(0);
  TORCH_CHECK(in.M < (1ll << 31) - 256 && in.V < (1ll << 31) - 256 && in.K < (1ll << 30), op, ": too large");
  TORCH_CHECK(targets.is_cuda() && targets.numel() == in.M, op, ": targets must have one entry a row");
  in.x = om::tma_rows(x);
  in.w = om::tma_rows(w);
  in.targets = targets.to(at::kLong).contiguous();
  in.rows.targets = reinterpret_cast<const long long*>(in.targets.data_ptr<int64_t>());
  in.rows.ignore = ignore;
  in.rows.scale = (float)scale;
  in.rows.V = (int)in.V;
  if (keep.has_value()) {
    TORCH_CHECK(smoothing == 0.0, op, ": label smoothing over a keep mask is not defined");
    TORCH_CHECK(keep->is_cuda() && keep->scalar_type() == at::kInt && keep->dim() == 2 && keep->size(0) == in.M &&
                    keep->size(1) >= (in.V + 31) / 32 && keep->stride(1) == 1,
                op, ": keep must be int32 [rows, ceil(V / 32)] words");
    in.keep = *keep;
    in.rows.keep = keep->data_ptr<int>();
    in.rows.ldk = keep->stride(0);
  }
  return in;
}

// Column tile of the product x W^T: 256 on CTA pairs or single CTAs; half of that while its tiles are at most half
// of the SMs, and 64 for the fewest. Forward with 64, 128 and 256 columns, us: 8 tiles of 256 (127 x 2048 -> 2048)
// 11.4, 11.4, 15.9 (its gradient 17.0, 17.4, 22.7); 24 (500 x 1024 -> 1500) 8.7, 8.9, 11.9; 36 (128 x 2048 -> 9000)
// 13.4, 12.4, 17.1; 72 (300 x 2048 -> 6000) 20.6, 13.5, 17.3; 118 (60 x 1024 -> 30000) 31.3, 22.0, 17.2.
struct XentTile {
  int bn, pair;
};
XentTile xent_tile(const XentIn& in, int64_t cols) {
  if (om::gx_pairs(in.M, cols, in.K)) return {256, 1};
  const int64_t tiles = (int64_t)om::ceil_div(in.M, 128) * om::ceil_div(cols, 256), sms = om::num_sms();
  return {tiles * 6 <= sms ? 64 : tiles * 2 <= sms ? 128 : 256, 0};
}

// The product with `cols` vocabulary rows from wv and either logits epilogue.
template <class Epi>
void xent_logits(const XentIn& in, const XentTile& t, const void* wv, int64_t cols, const om::OutMaps& o,
                 const typename Epi::Args& e, int* status, cudaStream_t st) {
  om::GemmX g{};
  g.rows = (int)in.M;
  g.cols = (int)cols;
  g.num_kb = om::ceil_div(in.K, 64);
  g.splits = 1;
  g.kb_per_split = g.num_kb;
  g.tiles_r = om::ceil_div(in.M, t.pair ? 256 : 128);
  g.tiles_c = om::ceil_div(cols, t.bn);
  g.b_step = t.bn;
  g.b_second = g.b_box = t.bn / 2;
  g.status = status;
  const CUtensorMap ta = om::gx_map(in.x.data_ptr(), false, in.M, in.K, in.x.stride(0), 128);
  const CUtensorMap tb = om::gx_map(wv, false, cols, in.K, in.w.stride(0), t.bn / 2);
  if (t.pair)
    om::gx_launch_pair<false, false, Epi>(ta, tb, o, g, e, st);
  else if (t.bn == 64)
    om::gx_launch<64, false, false, Epi>(ta, tb, o, g, e, st);
  else if (t.bn == 128)
    om::gx_launch<128, false, false, Epi>(ta, tb, o, g, e, st);
  else
    om::gx_launch<256, false, false, Epi>(ta, tb, o, g, e, st);
}

}  // namespace

// (loss, lse) fp32 in targets' shape
std::pair<torch::Tensor, torch::Tensor> om_linear_xent(torch::Tensor x, torch::Tensor w, torch::Tensor targets,
                                                       c10::optional<torch::Tensor> keep, double scale,
                                                       double smoothing, int64_t ignore, torch::Tensor status) {
  const c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::make_optional(x.device()) : c10::nullopt);
  const XentIn in = check_xent("linear_xent", x, w, targets, keep, smoothing, scale, ignore);
  const auto f32 = x.options().dtype(at::kFloat);
  auto loss = torch::empty(targets.sizes(), f32), lse = torch::empty(targets.sizes(), f32);
  const int64_t M = in.M;
  if (M == 0) return {loss, lse};
  auto st = at::cuda::getCurrentCUDAStream().stream();
  const XentTile tile = xent_tile(in, in.V);
  const int tiles = 2 * om::ceil_div(in.V, tile.bn);  // halves of column tiles
  const int64_t n = (int64_t)tiles * M;
  const bool smooth = smoothing != 0.0;
  auto ws = torch::empty({n * (smooth ? 3 : 2) + M}, f32);
  float* p = ws.data_ptr<float>();
  auto run = [&](auto epi) {
    using E = decltype(epi);
    typename E::Args e{in.rows, reinterpret_cast<float2*>(p), smooth ? p + 2 * n + M : nullptr, p + 2 * n};
    xent_logits<E>(in, tile, in.w.data_ptr(), in.V, om::OutMaps{}, e, status.data_ptr<int>(), st);
  };
  if (smooth)
    run(om::EpiXentFwd<true>{});
  else
    run(om::EpiXentFwd<false>{});
  om::launch_dependent(om::xent_join_kernel, om::ceil_div(M, 32), 32 * om::XE_JOIN, 0, st, (const float2*)p,
                       (const float*)(smooth ? p + 2 * n + M : nullptr), (const float*)(p + 2 * n), in.rows, (int)M,
                       tiles, (float)smoothing, loss.data_ptr<float>(), lse.data_ptr<float>(), status.data_ptr<int>());
  return {loss, lse};
}

// (dx [..., K], dw [V, K])
std::pair<c10::optional<torch::Tensor>, c10::optional<torch::Tensor>> om_linear_xent_bwd(
    torch::Tensor x, torch::Tensor w, torch::Tensor targets, c10::optional<torch::Tensor> keep, double scale,
    double smoothing, int64_t ignore, torch::Tensor lse, torch::Tensor dloss, bool need_dx, bool need_dw,
    torch::Tensor status) {
  const c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::make_optional(x.device()) : c10::nullopt);
  const XentIn in = check_xent("linear_xent_bwd", x, w, targets, keep, smoothing, scale, ignore);
  const int64_t M = in.M, K = in.K, V = in.V;
  TORCH_CHECK(lse.is_cuda() && lse.scalar_type() == at::kFloat && lse.numel() == M,
              "linear_xent_bwd: lse must be fp32 with one entry a row");
  TORCH_CHECK(dloss.is_cuda() && dloss.numel() == M, "linear_xent_bwd: dloss must have one entry a row");
  lse = lse.contiguous();
  dloss = dloss.to(at::kFloat).contiguous();
  c10::optional<torch::Tensor> dx, dw;
  if (need_dx) dx = torch::empty(x.sizes(), x.options());
  if (need_dw) dw = torch::empty(w.sizes(), w.options());
  if (M == 0) {
    if (need_dw) dw->zero_();
    return {dx, dw};
  }
  if (!need_dx && !need_dw) return {dx, dw};
  auto ptr = [](const torch::Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); };
  auto st = at::cuda::getCurrentCUDAStream().stream();
  const int64_t C = om::piece_columns(M, V);
  const int64_t ld = std::min(C, (V + 31) / 32 * 32);
  auto dz = torch::empty({M, ld}, x.options());
  const om::GxPlan px = om::gx_plan(M, K, std::min(C, V));
  const om::GxPlan pw = om::gx_plan(std::min(C, V), K, M);
  const int64_t nx = need_dx ? om::gx_acc_floats(px, M, K, C < V) : 0;
  const int64_t nw = need_dw ? om::gx_acc_floats(pw, std::min(C, V), K, false) : 0;
  torch::Tensor acc;
  if (nx + nw) acc = torch::empty({nx + nw}, lse.options());
  float* ax = nx ? acc.data_ptr<float>() : nullptr;
  float* aw = nw ? acc.data_ptr<float>() + nx : nullptr;  // nx is a multiple of 32
  const om::Factor factor{dloss.data_ptr<float>(), (float)(scale * (1.0 - smoothing))};
  for (int64_t v0 = 0; v0 < V; v0 += C) {
    const int64_t n = std::min(C, V - v0);
    const __nv_bfloat16* wv = ptr(in.w) + v0 * in.w.stride(0);
    const om::EpiXentBwd::Args e{in.rows, lse.data_ptr<float>(), dloss.data_ptr<float>(), (float)smoothing, (int)v0};
    om::OutMaps o{};
    o.m[0] = om::gx_out(ptr(dz), M, n, ld);
    xent_logits<om::EpiXentBwd>(in, xent_tile(in, n), wv, n, o, e, status.data_ptr<int>(), st);
    if (need_dx)
      om::gx_product(px, {dz.data_ptr(), false, ld}, {wv, true, in.w.stride(0)}, M, K, n, ptr(*dx), K, ax, v0 == 0,
                     v0 + n == V, status.data_ptr<int>(), st, factor);
    if (need_dw)
      om::gx_product(pw, {dz.data_ptr(), true, ld}, {in.x.data_ptr(), true, in.x.stride(0)}, n, K, M,
                     ptr(*dw) + v0 * K, K, aw, true, true, status.data_ptr<int>(), st, factor);
  }
  return {dx, dw};
}
