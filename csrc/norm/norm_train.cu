// RMSNorm / LayerNorm for training: forward with the residual add fused and the row statistics
// kept, and the gradient with the reduction of the weight's (and bias's) gradient.
//
//   h = x (+ delta, rounded to the stream's type)     n = (h - mu) r,  y = n w (+ b)
//   r = 1 / sqrt(mean((h - mu)^2) + eps),  mu = mean(h) (RMSNorm: 0)
//   a = dy w;  dx = r (a - n mean(a n) - [mean(a)]) (+ dh);  dw = sum_rows dy n;  db = sum_rows dy
//
// What bounds it: the rows' bytes, each read once and written once (4 or 7 values a column).
// A row is held in the registers of G threads (16 elements each with 16-byte accesses), so the
// two passes of the variance and of the gradient cost no second read. In the gradient every
// group of threads walks rows grid-strided and keeps its columns' dw and db in registers; the
// partial sums of the blocks are joined in block order by a second kernel: fp32, no atomics,
// the same result on every run. The next row's loads are issued before the current row's
// reductions, so the reductions' latency is hidden behind the loads.
#include <c10/cuda/CUDAGuard.h>
#include "../common/om_host.h"
#include "../common/om_ptx.cuh"

namespace om {

// V elements (1, or 16 bytes' worth) from / to memory as fp32
template <typename T, int V>
struct Vec {
  uint32_t u[V * sizeof(T) / 4 > 0 ? V * sizeof(T) / 4 : 1];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
      for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) {
        const uint4 q = reinterpret_cast<const uint4*>(p)[i];
        u[4 * i] = q.x; u[4 * i + 1] = q.y; u[4 * i + 2] = q.z; u[4 * i + 3] = q.w;
      }
    } else if constexpr (sizeof(T) == 2) {
      u[0] = *reinterpret_cast<const unsigned short*>(p);
    } else {
      u[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(u) / 4); ++i) u[i] = 0u;
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[j]);
    return (j & 1) ? bf16hi(u[j >> 1]) : bf16lo(u[j >> 1]);
  }
};
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  if constexpr (sizeof(T) == 2 && V == 8) {
    *reinterpret_cast<uint4*>(p) = pack8(f);
  } else if constexpr (sizeof(T) == 4 && V == 8) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else if constexpr (sizeof(T) == 2) {
    p[0] = __float2bfloat16_rn(f[0]);
  } else {
    p[0] = f[0];
  }
}
template <typename T>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(__float2bfloat16_rn(v));
  return v;
}

// Sums of N values over the G threads of a row; `sh` has 2 * N * (threads / 32) floats and is
// used by halves in turn (`flip`), so that one barrier a reduction is enough.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* sh, int& flip) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (G > 32) {
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
    float* s = sh + flip * N * warps;
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[i * warps + warp] = v[i];
    }
    __syncthreads();
    const int w0 = threadIdx.x / G * (G / 32);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < G / 32; ++w) t += s[i * warps + w0 + w];
      v[i] = t;
    }
  }
}

template <int G>
constexpr int norm_threads() { return G < 256 ? 256 : G; }

struct NormFwd {
  const void *x, *delta, *w, *b;
  void *y, *h;
  float* stats;  // [M, 2]: mu, r
  long long M, ldx, ldd;
  int D;
  float eps;
};

template <typename T, typename W, bool LAYER, int G, int V, int P>
__global__ void __launch_bounds__(norm_threads<G>()) norm_fwd_kernel(const NormFwd a) {
  __shared__ float sh[2 * (norm_threads<G>() / 32)];
  constexpr int RPB = norm_threads<G>() / G;
  const int lane = threadIdx.x % G;
  const long long row = (long long)blockIdx.x * RPB + threadIdx.x / G;
  const bool live = row < a.M;
  int flip = 0;
  float f[P][V];
  float sum[1] = {0.f};
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (lane + i * G) * V;
    Vec<T, V> v, d;
    v.zero();
    d.zero();
    if (live && c < a.D) {
      v.load(static_cast<const T*>(a.x) + row * a.ldx + c);
      if (a.delta) d.load(static_cast<const T*>(a.delta) + row * a.ldd + c);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      // the stream's rounded value is what is normalised, as the gradient will read it
      f[i][j] = a.delta ? round_to<T>(v.get(j) + d.get(j)) : v.get(j);
      sum[0] += LAYER ? f[i][j] : f[i][j] * f[i][j];
    }
    if (live && c < a.D && a.h) store_vec<T, V>(static_cast<T*>(a.h) + row * a.D + c, f[i]);
  }
  group_sum<G, 1>(sum, sh, flip);
  float mu = 0.f;
  if constexpr (LAYER) {
    mu = sum[0] / a.D;
    sum[0] = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float t = (lane + i * G) * V < a.D ? f[i][j] - mu : 0.f;
        sum[0] += t * t;
      }
    group_sum<G, 1>(sum, sh, flip);
  }
  const float r = rsqrtf(sum[0] / a.D + a.eps);
  if (!live) return;
  if (lane == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(mu, r);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (lane + i * G) * V;
    if (c >= a.D) continue;
    Vec<W, V> w, b;
    w.load(static_cast<const W*>(a.w) + c);
    b.zero();
    if (a.b) b.load(static_cast<const W*>(a.b) + c);
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = (f[i][j] - mu) * r * w.get(j) + b.get(j);
    store_vec<T, V>(static_cast<T*>(a.y) + row * a.D + c, o);
  }
}

struct NormBwd {
  const void *dy, *h, *w, *dh;
  void* dx;
  const float* stats;
  float* part;  // [blocks][1 or 2][D]: dw, db
  long long M, ldy, ldh, lddh;
  int D;
};

template <typename T, typename W, bool LAYER, int G, int V, int P>
__global__ void __launch_bounds__(norm_threads<G>()) norm_bwd_kernel(const NormBwd a) {
  constexpr int NT = norm_threads<G>(), RPB = NT / G, N = LAYER ? 2 : 1;
  __shared__ float sh[2 * N * (NT / 32)];
  const int lane = threadIdx.x % G;
  const long long step = (long long)gridDim.x * RPB;
  int flip = 0;
  float dw[P][V], db[LAYER ? P : 1][V];
  Vec<W, V> w[P];
  Vec<T, V> hv[P], yv[P];
  float2 st = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (lane + i * G) * V;
    w[i].zero();
    if (c < a.D) w[i].load(static_cast<const W*>(a.w) + c);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      dw[i][j] = 0.f;
      if constexpr (LAYER) db[i][j] = 0.f;
    }
  }
  auto fetch = [&](long long row) {
    const bool live = row < a.M;
    if (live) st = *reinterpret_cast<const float2*>(a.stats + 2 * row);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + i * G) * V;
      if (live && c < a.D) {
        hv[i].load(static_cast<const T*>(a.h) + row * a.ldh + c);
        yv[i].load(static_cast<const T*>(a.dy) + row * a.ldy + c);
      } else {
        hv[i].zero();
        yv[i].zero();
      }
    }
  };
  const long long row0 = (long long)blockIdx.x * RPB;
  fetch(row0 + threadIdx.x / G);
  // every thread of the block takes the same number of turns (the reductions have barriers)
  for (long long base = row0; base < a.M; base += step) {
    const long long row = base + threadIdx.x / G;
    const float mu = st.x, r = row < a.M ? st.y : 0.f;
    float n[P][V], ga[P][V];
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float y = yv[i].get(j);
        n[i][j] = (hv[i].get(j) - mu) * r;
        ga[i][j] = y * w[i].get(j);   // 0 beyond the row's end: w and dy are 0 there
        s[0] += ga[i][j] * n[i][j];
        dw[i][j] += y * n[i][j];
        if constexpr (LAYER) {
          s[N - 1] += ga[i][j];
          db[i][j] += y;
        }
      }
    }
    fetch(row + step);
    group_sum<G, N>(s, sh, flip);
    if (row >= a.M) continue;  // no barrier below
    const float c1 = s[0] / a.D, c2 = LAYER ? s[N - 1] / a.D : 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + i * G) * V;
      if (c >= a.D) continue;
      Vec<T, V> d;
      d.zero();
      if (a.dh) d.load(static_cast<const T*>(a.dh) + row * a.lddh + c);
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = r * (ga[i][j] - n[i][j] * c1 - c2) + d.get(j);
      store_vec<T, V>(static_cast<T*>(a.dx) + row * a.D + c, o);
    }
  }
  // the block's row groups are added up in group order through shared memory
  extern __shared__ float acc[];  // [D] when RPB > 1
#pragma unroll
  for (int k = 0; k < N; ++k) {
    float* out = a.part + ((size_t)blockIdx.x * N + k) * a.D;
    if constexpr (RPB == 1) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = (lane + i * G) * V;
        if (c >= a.D) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) out[c + j] = k == 0 ? dw[i][j] : db[LAYER ? i : 0][j];
      }
    } else {
      for (int grp = 0; grp < RPB; ++grp) {
        __syncthreads();
        if ((int)threadIdx.x / G == grp) {
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const int c = (lane + i * G) * V;
            if (c >= a.D) continue;
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float t = k == 0 ? dw[i][j] : db[LAYER ? i : 0][j];
              if (grp == 0)
                acc[c + j] = t;
              else if (grp < RPB - 1)
                acc[c + j] += t;
              else
                out[c + j] = acc[c + j] + t;
            }
          }
        }
      }
      __syncthreads();
    }
  }
}

// dw (db) = sum over blocks, in block order: 32 columns a block, 8 warps each take every eighth
// partial row, joined in warp order.
template <typename W>
__global__ void __launch_bounds__(256) norm_join_kernel(const float* __restrict__ part, int blocks, int n, int D,
                                                        W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float sh[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, k = blockIdx.y;
  float t = 0.f;
  if (c < D) {
#pragma unroll 4
    for (int b = warp; b < blocks; b += 8) t += part[((size_t)b * n + k) * D + c];
  }
  sh[warp][lane] = t;
  __syncthreads();
  if (warp != 0 || c >= D) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) t += sh[w][lane];
  W* out = k == 0 ? dw : db;
  if constexpr (sizeof(W) == 2)
    out[c] = __float2bfloat16_rn(t);
  else
    out[c] = t;
}

// Threads of a row: 16 elements a thread with 16-byte accesses, single elements otherwise
// (16 each from 512 columns on).
template <typename F>
static void norm_shape(const char* op, int D, bool vec, F&& f) {
  using std::integral_constant;
#define OM_NORM_CASE(G_, V_, P_) \
  return f(integral_constant<int, G_>{}, integral_constant<int, V_>{}, integral_constant<int, P_>{})
  if (vec) {
    if (D <= 256) OM_NORM_CASE(32, 8, 1);
    if (D <= 512) OM_NORM_CASE(32, 8, 2);
    if (D <= 1024) OM_NORM_CASE(64, 8, 2);
    if (D <= 2048) OM_NORM_CASE(128, 8, 2);
    if (D <= 4096) OM_NORM_CASE(256, 8, 2);
    if (D <= 8192) OM_NORM_CASE(512, 8, 2);
    if (D <= 16384) OM_NORM_CASE(1024, 8, 2);
  } else {
    if (D <= 128) OM_NORM_CASE(32, 1, 4);
    if (D <= 1024) OM_NORM_CASE(128, 1, 8);
    if (D <= 4096) OM_NORM_CASE(512, 1, 8);
    if (D <= 16384) OM_NORM_CASE(1024, 1, 16);
  }
#undef OM_NORM_CASE
  TORCH_CHECK(false, op, ": rows of more than 16384 elements are not supported (got ", num(D), ")");
}

template <typename F>
static void norm_types(const char* op, at::ScalarType t, at::ScalarType w, F&& f) {
  const bool tb = t == at::kBFloat16, wb = w == at::kBFloat16;
  TORCH_CHECK((tb || t == at::kFloat) && (wb || w == at::kFloat), op, ": bf16 or fp32 tensors required");
  if (tb && wb) return f(__nv_bfloat16{}, __nv_bfloat16{});
  if (tb) return f(__nv_bfloat16{}, 0.f);
  TORCH_CHECK(!wb, op, ": fp32 rows take fp32 weights");
  return f(0.f, 0.f);
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace om

namespace {

// [..., D] as [M, D] rows of the expected type
torch::Tensor norm_rows(const char* op, const char* name, const torch::Tensor& t, int64_t M, int64_t D,
                        at::ScalarType ty) {
  TORCH_CHECK(t.is_cuda() && t.dim() >= 1 && t.size(t.dim() - 1) == D && t.numel() == M * D && t.scalar_type() == ty,
              op, ": ", name, " must be a CUDA tensor of the rows' shape and type");
  return om::rows_view(t);
}
torch::Tensor norm_cols(const char* op, const char* name, const torch::Tensor& t, int64_t D, at::ScalarType ty) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 1 && t.size(0) == D && t.scalar_type() == ty, op, ": ", name,
              " must be a CUDA [D] tensor of the weight's type");
  return t.contiguous();
}
bool norm_vec(const torch::Tensor& t) {
  return (t.dim() == 1 || t.stride(0) % 8 == 0) && om::aligned16(t.data_ptr());
}

}  // namespace

// (y [..., D], h (x itself without delta), stats fp32 [M, 2])
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> om_norm_train(torch::Tensor x, torch::Tensor w,
                                                                      c10::optional<torch::Tensor> b, double eps,
                                                                      bool layer, c10::optional<torch::Tensor> delta) {
  const char* op = "norm_train";
  TORCH_CHECK(x.dim() >= 1 && x.is_cuda(), "norm_train: x must be a CUDA tensor [..., D]");
  const int64_t D = x.size(x.dim() - 1);
  TORCH_CHECK(D > 0, "norm_train: empty rows");
  const int64_t M = x.numel() / D;
  const c10::cuda::CUDAGuard guard(x.device());
  om::NormFwd a{};
  const auto ty = x.scalar_type(), wt = w.scalar_type();
  const torch::Tensor x2 = norm_rows(op, "x", x, M, D, ty), w2 = norm_cols(op, "w", w, D, wt);
  torch::Tensor d2, b2, h;
  bool vec = D % 8 == 0 && norm_vec(x2) && norm_vec(w2);
  if (delta.has_value()) {
    d2 = norm_rows(op, "delta", *delta, M, D, ty);
    a.ldd = d2.stride(0);
    a.delta = d2.data_ptr();
    vec = vec && norm_vec(d2);
  }
  if (b.has_value()) {
    TORCH_CHECK(layer, "norm_train: RMSNorm takes no bias");
    b2 = norm_cols(op, "b", *b, D, wt);
    a.b = b2.data_ptr();
    vec = vec && norm_vec(b2);
  }
  auto y = torch::empty(x.sizes(), x.options());
  h = delta.has_value() ? torch::empty(x.sizes(), x.options()) : x;
  auto stats = torch::empty({M, 2}, x.options().dtype(at::kFloat));
  a.x = x2.data_ptr();
  a.ldx = x2.stride(0);
  a.w = w2.data_ptr();
  a.y = y.data_ptr();
  a.h = delta.has_value() ? h.data_ptr() : nullptr;
  a.stats = stats.data_ptr<float>();
  a.M = M;
  a.D = (int)std::min<int64_t>(D, INT32_MAX);
  a.eps = (float)eps;
  auto st = at::cuda::getCurrentCUDAStream().stream();
  om::norm_types(op, ty, wt, [&](auto t0, auto w0) {
    om::norm_shape(op, a.D, vec, [&](auto G, auto V, auto P) {
      using T = decltype(t0);
      using W = decltype(w0);
      constexpr int g = decltype(G)::value, v = decltype(V)::value, p = decltype(P)::value;
      constexpr int NT = om::norm_threads<g>();
      const long long blocks = (M + NT / g - 1) / (NT / g);
      TORCH_CHECK(blocks < (1ll << 31), "norm_train: too many rows");
      if (M == 0) return;
      if (layer)
        om::norm_fwd_kernel<T, W, true, g, v, p><<<(unsigned)blocks, NT, 0, st>>>(a);
      else
        om::norm_fwd_kernel<T, W, false, g, v, p><<<(unsigned)blocks, NT, 0, st>>>(a);
      OM_LAUNCH_CHECK();
    });
  });
  return {y, h, stats};
}

// (dx [..., D], dw [D], db [D] (LayerNorm with bias))
std::tuple<torch::Tensor, torch::Tensor, c10::optional<torch::Tensor>> om_norm_train_bwd(
    torch::Tensor dy, torch::Tensor h, torch::Tensor w, torch::Tensor stats, bool layer, bool bias,
    c10::optional<torch::Tensor> dh) {
  const char* op = "norm_train_bwd";
  TORCH_CHECK(h.dim() >= 1 && h.is_cuda(), "norm_train_bwd: h must be a CUDA tensor [..., D]");
  const int64_t D = h.size(h.dim() - 1);
  TORCH_CHECK(D > 0, "norm_train_bwd: empty rows");
  TORCH_CHECK(layer || !bias, "norm_train_bwd: RMSNorm has no bias");
  const int64_t M = h.numel() / D;
  const c10::cuda::CUDAGuard guard(h.device());
  const auto ty = h.scalar_type(), wt = w.scalar_type();
  om::NormBwd a{};
  const torch::Tensor h2 = norm_rows(op, "h", h, M, D, ty), y2 = norm_rows(op, "dy", dy.to(ty), M, D, ty);
  const torch::Tensor w2 = norm_cols(op, "w", w, D, wt);
  torch::Tensor d2;
  bool vec = D % 8 == 0 && norm_vec(h2) && norm_vec(y2) && norm_vec(w2);
  if (dh.has_value()) {
    d2 = norm_rows(op, "dh", dh->to(ty), M, D, ty);
    a.lddh = d2.stride(0);
    a.dh = d2.data_ptr();
    vec = vec && norm_vec(d2);
  }
  TORCH_CHECK(stats.is_cuda() && stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == 2 * M,
              "norm_train_bwd: stats must be fp32 [M, 2]");
  auto dx = torch::empty(h.sizes(), h.options());
  auto dw = torch::empty({D}, w.options());
  c10::optional<torch::Tensor> db;
  if (bias) db = torch::empty({D}, w.options());
  if (M == 0) {
    dw.zero_();
    if (bias) db->zero_();
    return {dx, dw, db};
  }
  a.dy = y2.data_ptr();
  a.ldy = y2.stride(0);
  a.h = h2.data_ptr();
  a.ldh = h2.stride(0);
  a.w = w2.data_ptr();
  a.dx = dx.data_ptr();
  a.stats = stats.data_ptr<float>();
  a.M = M;
  a.D = (int)std::min<int64_t>(D, INT32_MAX);
  const int n = layer ? 2 : 1;
  auto st = at::cuda::getCurrentCUDAStream().stream();
  om::norm_types(op, ty, wt, [&](auto t0, auto w0) {
    om::norm_shape(op, a.D, vec, [&](auto G, auto V, auto P) {
      using T = decltype(t0);
      using W = decltype(w0);
      constexpr int g = decltype(G)::value, v = decltype(V)::value, p = decltype(P)::value;
      constexpr int NT = om::norm_threads<g>(), RPB = NT / g;
      auto go = [&](auto kernel, std::atomic<int>& resident) {
        const size_t smem = RPB > 1 ? (size_t)a.D * sizeof(float) : 0;
        int per_sm = resident.load();  // the same for every call of this instance (smem is at most 8 KB)
        if (per_sm == 0) {
          OM_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, NT, smem));
          per_sm = std::max(1, per_sm);
          resident.store(per_sm);
        }
        const long long most = (M + RPB - 1) / RPB;
        const int blocks = (int)std::min<long long>(most, (long long)om::num_sms() * per_sm);
        auto part = torch::empty({(int64_t)blocks * n * a.D}, stats.options());
        a.part = part.data_ptr<float>();
        kernel<<<blocks, NT, smem, st>>>(a);
        OM_LAUNCH_CHECK();
        om::norm_join_kernel<W><<<dim3((a.D + 31) / 32, bias ? 2 : 1), 256, 0, st>>>(
            a.part, blocks, n, a.D, reinterpret_cast<W*>(dw.data_ptr()),
            bias ? reinterpret_cast<W*>(db->data_ptr()) : nullptr);
        OM_LAUNCH_CHECK();
      };
      static std::atomic<int> resident[2];
      if (layer)
        go(om::norm_bwd_kernel<T, W, true, g, v, p>, resident[1]);
      else
        go(om::norm_bwd_kernel<T, W, false, g, v, p>, resident[0]);
    });
  });
  return {dx, dw, db};
}
