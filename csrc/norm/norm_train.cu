// RMSNorm / LayerNorm for training: forward with the residual add fused and the row statistics
// kept, and the gradient with the reduction of the weight's (and bias's) gradient.
//
//   h = x (+ delta, rounded to the stream's type)     n = (h - mu) r,  y = n w (+ b)
//   r = 1 / sqrt(mean((h - mu)^2) + eps),  mu = mean(h) (RMSNorm: 0)
//   a = dy w;  dx = r (a - n mean(a n) - [mean(a)]) (+ dh);  dw = sum_rows dy n;  db = sum_rows dy
//
// What bounds it: the rows' bytes, each read once and written once (4 or 7 values a column). A row
// is held in the registers of G threads, so the two passes of the variance and of the gradient
// cost no second read, and every group of threads walks rows grid-strided with the weights (and
// its columns' dw and db) in registers. Rows come into a ring in shared memory by bulk copies,
// several rows ahead: registers alone could hold one row ahead, which left the memory idle during
// the reductions. Rows that do not start on 16 bytes take a ring of their own, from which they are
// read element by element; rows of which two stages do not fit into shared memory (the longest fp32
// ones) are read straight into registers.
// The partial dw, db of the blocks are joined in a fixed order by a second kernel: fp32, no atomics,
// the same result on every run.
// Measured (B200): 8192 x 4096 bf16 with residual, forward 40 us (5.3 TB/s to and from memory), gradient
// 44 us (5.6 TB/s); 19600 x 1024 LayerNorm with fp32 gain 21 and 30 us (3.8 and 4.0 TB/s): a 2 KB row is the
// work of two warps, which meet at a barrier for each of its two sums (one in the gradient), and the
// issue slots are half used.
#include <c10/cuda/CUDAGuard.h>
#include "../common/om_host.h"
#include "../common/om_ptx.cuh"

namespace om {

// V elements (1 or 8) from / to memory as fp32
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
    } else if constexpr (V * sizeof(T) == 2) {
      u[0] = *reinterpret_cast<const unsigned short*>(p);
    } else {
      u[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(u) / 4); ++i) u[i] = 0u;
  }
  __device__ __forceinline__ uint64_t pair(int j) const {  // elements 2 j, 2 j + 1
    if constexpr (sizeof(T) == 4) return pair_f32(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1]));
    return pair_f32(bf16lo(u[j]), bf16hi(u[j]));
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
__device__ __forceinline__ void store_pairs(T* p, const uint64_t (&f)[4]) {
  const float2 a = unpair_f32(f[0]), b = unpair_f32(f[1]), c = unpair_f32(f[2]), d = unpair_f32(f[3]);
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(b.x, b.y), pack_bf16x2(c.x, c.y), pack_bf16x2(d.x, d.y));
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(a.x, a.y, b.x, b.y);
    reinterpret_cast<float4*>(p)[1] = make_float4(c.x, c.y, d.x, d.y);
  }
}
__device__ __forceinline__ float pair_sum(uint64_t v) {
  const float2 a = unpair_f32(v);
  return a.x + a.y;
}
template <typename T>
__device__ __forceinline__ uint64_t round_pair(uint64_t v) {
  if constexpr (sizeof(T) == 2) {
    const float2 a = unpair_f32(v);
    const uint32_t u = pack_bf16x2(a.x, a.y);
    return pair_f32(bf16lo(u), bf16hi(u));
  }
  return v;
}
template <typename T>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(__float2bfloat16_rn(v));
  return v;
}

// Sums of N values over the G threads of a row, which meet at a barrier of their own; `sh` has
// 2 * N * (threads / 32) floats and is used by halves in turn (`flip`), so that one barrier a
// reduction is enough.
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
    if (G == (int)blockDim.x)
      __syncthreads();
    else
      named_bar_sync(1 + threadIdx.x / G, G);
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

// A ring of rows in shared memory, one per group of G threads: NA arrays a stage, filled by bulk
// copies that the group's first thread starts. Only arrival is signalled: a stage is filled again
// after a barrier of the group that follows its last read. ODD: rows may start anywhere; the
// 16-byte blocks that hold a row are copied whole, and it is read at its offset in them.
template <typename T, int G, int NA, bool ODD = false>
struct RowRing {
  uint8_t* base;      // this group's stages
  uint64_t* full;     // this group's barriers
  const T* src[NA];
  long long ld[NA];
  int stages;
  uint32_t bytes;     // of a row's place in a stage
  uint32_t len;       // ODD: bytes of a row
  int s;              // the stage in turn and the phase of its barrier
  uint32_t phase;
  __device__ __forceinline__ uint32_t off(int i, long long row) const {
    return ODD ? (uint32_t)(reinterpret_cast<uintptr_t>(src[i] + row * ld[i]) & 15) : 0u;
  }
  __device__ __forceinline__ void fill(int stage, long long row) const {  // one thread
    uint32_t n[NA], all = 0;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      n[i] = ODD ? (src[i] != nullptr ? (off(i, row) + len + 15) & ~15u : 0u) : bytes;
      all += n[i];
    }
    mbar_arrive_expect_tx(&full[stage], all);
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (n[i])
        bulk_load(base + (size_t)(stage * NA + i) * bytes,
                  reinterpret_cast<const uint8_t*>(src[i] + row * ld[i]) - off(i, row), n[i], &full[stage]);
  }
  // Not stopped by another wait that gave up: a group's copies depend on nobody, and leaving early would
  // leave them in flight.
  __device__ __forceinline__ bool wait(int* status) const {
    if (mbar_wait(&full[s], phase, nullptr, 0)) return true;
    record_error(status, OM_ERR_WAIT_FULL);
    return false;
  }
  __device__ __forceinline__ const T* row(int i) const {
    return reinterpret_cast<const T*>(base + (size_t)(s * NA + i) * bytes);
  }
  __device__ __forceinline__ const T* row_at(int i, long long r) const {  // ODD
    return reinterpret_cast<const T*>(base + (size_t)(s * NA + i) * bytes + off(i, r));
  }
  __device__ __forceinline__ void next() {
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
};

constexpr int RING_MAX = 8;  // stages
// place of a row that may start anywhere in its first 16-byte block
__host__ __device__ constexpr uint32_t odd_place(uint32_t len) { return (len + 30u) & ~15u; }

struct NormFwd {
  const void *x, *delta, *w, *b;
  void *y, *h;
  float* stats;  // [M, 2]: mu, r
  long long M, ldx, ldd;
  int D;
  float eps;
  int stages;  // of the ring
  int* status;
};

template <typename T, typename W, bool LAYER, int G, int V, int P>
__global__ void __launch_bounds__(norm_threads<G>()) norm_fwd_kernel(const NormFwd a) {
  __shared__ float sh[2 * (norm_threads<G>() / 32)];
  constexpr int RPB = norm_threads<G>() / G;
  grid_wait();
  grid_release();
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

// The same with the rows in a ring and the weights in registers.
template <typename T, typename W, bool LAYER, bool DELTA, int G, int P>
__global__ void __launch_bounds__(norm_threads<G>()) norm_fwd_ring_kernel(const NormFwd a) {
  constexpr int NT = norm_threads<G>(), RPB = NT / G, V = 8, NA = DELTA ? 2 : 1;
  extern __shared__ __align__(128) uint8_t ring_mem[];
  __shared__ float sh[2 * (NT / 32)];
  __shared__ uint64_t bars[RPB * RING_MAX];
  const int grp = threadIdx.x / G, lane = threadIdx.x % G;
  const long long step = (long long)gridDim.x * RPB, row0 = (long long)blockIdx.x * RPB;
  RowRing<T, G, NA> ring;
  ring.stages = a.stages;
  ring.s = 0;
  ring.phase = 0;
  ring.bytes = a.D * sizeof(T);
  ring.base = ring_mem + (size_t)grp * a.stages * NA * ring.bytes;
  ring.full = bars + grp * RING_MAX;
  ring.src[0] = static_cast<const T*>(a.x);
  ring.ld[0] = a.ldx;
  if constexpr (DELTA) {
    ring.src[1] = static_cast<const T*>(a.delta);
    ring.ld[1] = a.ldd;
  }
  if (lane == 0) {
    for (int i = 0; i < a.stages; ++i) mbar_init(&ring.full[i], 1);
    fence_barrier_init();
  }
  grid_wait();
  grid_release();
  if (lane == 0) {
    for (int k = 0; k < a.stages; ++k)
      if (row0 + grp + k * step < a.M) ring.fill(k, row0 + grp + k * step);
  }
  uint64_t w[P][4], b[LAYER ? P : 1][4];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (lane + i * G) * V;
    Vec<W, V> wv, bv;
    wv.zero();
    bv.zero();
    if (c < a.D) wv.load(static_cast<const W*>(a.w) + c);
    if (LAYER && a.b && c < a.D) bv.load(static_cast<const W*>(a.b) + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[i][j] = wv.pair(j);
      if constexpr (LAYER) b[i][j] = bv.pair(j);
    }
  }
  __syncthreads();
  int flip = 0;
  // every group takes the same number of turns
  for (long long base = row0; base < a.M; base += step) {
    const long long row = base + grp;
    const bool live = row < a.M && ring.wait(a.status);
    uint64_t f[P][4], acc = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + i * G) * V;
      Vec<T, V> v, d;
      v.zero();
      d.zero();
      if (live && c < a.D) {
        v.load(ring.row(0) + c);
        if constexpr (DELTA) d.load(ring.row(1) + c);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[i][j] = DELTA ? round_pair<T>(add_f32x2(v.pair(j), d.pair(j))) : v.pair(j);
        acc = LAYER ? add_f32x2(acc, f[i][j]) : fma_f32x2(f[i][j], f[i][j], acc);
      }
      if (DELTA && live && c < a.D) store_pairs(static_cast<T*>(a.h) + row * a.D + c, f[i]);
    }
    float sum[1] = {pair_sum(acc)};
    group_sum<G, 1>(sum, sh, flip);
    if constexpr (G == 32) __syncwarp();
    if (lane == 0 && row + a.stages * step < a.M) ring.fill(ring.s, row + a.stages * step);
    ring.next();
    float mu = 0.f;
    if constexpr (LAYER) {
      mu = sum[0] / a.D;
      acc = 0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const bool in = (lane + i * G) * V < a.D;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[i][j] = add_f32x2(f[i][j], pair_f32(-mu, -mu));
          if (in) acc = fma_f32x2(f[i][j], f[i][j], acc);
        }
      }
      sum[0] = pair_sum(acc);
      group_sum<G, 1>(sum, sh, flip);
    }
    if (!live) continue;
    const float r = rsqrtf(sum[0] / a.D + a.eps);
    if (lane == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(mu, r);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + i * G) * V;
      if (c >= a.D) continue;
      uint64_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = mul_f32x2(f[i][j], pair_f32(r, r));
        o[j] = LAYER ? fma_f32x2(o[j], w[i][j], b[LAYER ? i : 0][j]) : mul_f32x2(o[j], w[i][j]);
      }
      store_pairs(static_cast<T*>(a.y) + row * a.D + c, o);
    }
  }
}

struct NormBwd {
  const void *dy, *h, *w, *dh;
  void* dx;
  const float* stats;
  float* part;  // [blocks][1 or 2][D]: dw, db
  void *dw, *db;  // of the weight's type: written straight by a single block
  long long M, ldy, ldh, lddh;
  int D;
  int stages;
  int* status;
};

// The block's row groups are added up in group order through shared memory (acc: [D]); the sum goes to
// the block's partial, or is the result if there is no other block.
template <typename W, int G, int V, int P, int N, int RPB>
__device__ __forceinline__ void write_partials(const NormBwd& a, const float (&dw)[P][V],
                                               const float (&db)[N == 2 ? P : 1][V], float* acc) {
  const int lane = threadIdx.x % G;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    float* part = a.part + ((size_t)blockIdx.x * N + k) * a.D;
    W* out = static_cast<W*>(k == 0 ? a.dw : a.db);
    auto put = [&](int c, float v) {
      if (gridDim.x > 1)
        part[c] = v;
      else if (out != nullptr)
        store_vec<W, 1>(out + c, &v);
    };
    if constexpr (RPB == 1) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = (lane + i * G) * V;
        if (c >= a.D) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) put(c + j, k == 0 ? dw[i][j] : db[N == 2 ? i : 0][j]);
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
              const float t = k == 0 ? dw[i][j] : db[N == 2 ? i : 0][j];
              if (grp == 0)
                acc[c + j] = t;
              else if (grp < RPB - 1)
                acc[c + j] += t;
              else
                put(c + j, acc[c + j] + t);
            }
          }
        }
      }
      __syncthreads();
    }
  }
}

template <typename T, typename W, bool LAYER, int G, int V, int P>
__global__ void __launch_bounds__(norm_threads<G>()) norm_bwd_kernel(const NormBwd a) {
  constexpr int NT = norm_threads<G>(), RPB = NT / G, N = LAYER ? 2 : 1;
  __shared__ float sh[2 * N * (NT / 32)];
  const int lane = threadIdx.x % G;
  const long long step = (long long)gridDim.x * RPB;
  int flip = 0;
  grid_wait();
  grid_release();
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
  extern __shared__ float acc[];  // [D] when RPB > 1
  write_partials<W, G, V, P, N, RPB>(a, dw, db, acc);
}

// The same with the rows in a ring.
template <typename T, typename W, bool LAYER, bool DH, int G, int P>
__global__ void __launch_bounds__(norm_threads<G>()) norm_bwd_ring_kernel(const NormBwd a) {
  constexpr int NT = norm_threads<G>(), RPB = NT / G, N = LAYER ? 2 : 1, V = 8, NA = DH ? 3 : 2;
  extern __shared__ __align__(128) uint8_t ring_mem[];
  __shared__ float sh[2 * N * (NT / 32)];
  __shared__ uint64_t bars[RPB * RING_MAX];
  const int grp = threadIdx.x / G, lane = threadIdx.x % G;
  const long long step = (long long)gridDim.x * RPB, row0 = (long long)blockIdx.x * RPB;
  RowRing<T, G, NA> ring;
  ring.stages = a.stages;
  ring.s = 0;
  ring.phase = 0;
  ring.bytes = a.D * sizeof(T);
  ring.base = ring_mem + (size_t)grp * a.stages * NA * ring.bytes;
  ring.full = bars + grp * RING_MAX;
  ring.src[0] = static_cast<const T*>(a.h);
  ring.ld[0] = a.ldh;
  ring.src[1] = static_cast<const T*>(a.dy);
  ring.ld[1] = a.ldy;
  if constexpr (DH) {
    ring.src[2] = static_cast<const T*>(a.dh);
    ring.ld[2] = a.lddh;
  }
  if (lane == 0) {
    for (int i = 0; i < a.stages; ++i) mbar_init(&ring.full[i], 1);
    fence_barrier_init();
  }
  grid_wait();
  grid_release();
  if (lane == 0) {
    for (int k = 0; k < a.stages; ++k)
      if (row0 + grp + k * step < a.M) ring.fill(k, row0 + grp + k * step);
  }
  uint64_t dw2[P][4], db2[LAYER ? P : 1][4], w[P][4];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = (lane + i * G) * V;
    Vec<W, V> wv;
    wv.zero();
    if (c < a.D) wv.load(static_cast<const W*>(a.w) + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[i][j] = wv.pair(j);
      dw2[i][j] = 0;
      if constexpr (LAYER) db2[i][j] = 0;
    }
  }
  float2 next = make_float2(0.f, 0.f);
  if (row0 + grp < a.M) next = *reinterpret_cast<const float2*>(a.stats + 2 * (row0 + grp));
  __syncthreads();
  int flip = 0;
  for (long long base = row0; base < a.M; base += step) {
    const long long row = base + grp;
    const bool live = row < a.M && ring.wait(a.status);
    const float mu = next.x, r = live ? next.y : 0.f;
    if (row + step < a.M) next = *reinterpret_cast<const float2*>(a.stats + 2 * (row + step));
    uint64_t n[P][4], ga[P][4], s0 = 0, s1 = 0;
    Vec<T, V> d[DH ? P : 1];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + i * G) * V;
      Vec<T, V> hv, yv;
      hv.zero();
      yv.zero();
      if constexpr (DH) d[i].zero();
      if (live && c < a.D) {
        hv.load(ring.row(0) + c);
        yv.load(ring.row(1) + c);
        if constexpr (DH) d[i].load(ring.row(2) + c);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t y = yv.pair(j);
        n[i][j] = LAYER ? add_f32x2(hv.pair(j), pair_f32(-mu, -mu)) : hv.pair(j);
        n[i][j] = mul_f32x2(n[i][j], pair_f32(r, r));
        ga[i][j] = mul_f32x2(y, w[i][j]);  // 0 beyond the row's end: w and dy are 0 there
        s0 = fma_f32x2(ga[i][j], n[i][j], s0);
        dw2[i][j] = fma_f32x2(y, n[i][j], dw2[i][j]);
        if constexpr (LAYER) {
          s1 = add_f32x2(s1, ga[i][j]);
          db2[i][j] = add_f32x2(db2[i][j], y);
        }
      }
    }
    float s[N];
    s[0] = pair_sum(s0);
    if constexpr (LAYER) s[N - 1] = pair_sum(s1);
    group_sum<G, N>(s, sh, flip);
    if constexpr (G == 32) __syncwarp();
    if (lane == 0 && row + a.stages * step < a.M) ring.fill(ring.s, row + a.stages * step);
    ring.next();
    if (!live) continue;  // no barrier below
    const float c1 = -s[0] / a.D, c2 = LAYER ? -s[N - 1] / a.D : 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + i * G) * V;
      if (c >= a.D) continue;
      uint64_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = fma_f32x2(n[i][j], pair_f32(c1, c1), ga[i][j]);
        if constexpr (LAYER) o[j] = add_f32x2(o[j], pair_f32(c2, c2));
        o[j] = DH ? fma_f32x2(o[j], pair_f32(r, r), d[DH ? i : 0].pair(j)) : mul_f32x2(o[j], pair_f32(r, r));
      }
      store_pairs(static_cast<T*>(a.dx) + row * a.D + c, o);
    }
  }
  float dw[P][V], db[LAYER ? P : 1][V];
#pragma unroll
  for (int i = 0; i < P; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = unpair_f32(dw2[i][j]);
      dw[i][2 * j] = t.x;
      dw[i][2 * j + 1] = t.y;
      if constexpr (LAYER) {
        const float2 q = unpair_f32(db2[LAYER ? i : 0][j]);
        db[i][2 * j] = q.x;
        db[i][2 * j + 1] = q.y;
      }
    }
  __syncthreads();  // every copy has been waited for and read: the ring's memory is free
  write_partials<W, G, V, P, N, RPB>(a, dw, db, reinterpret_cast<float*>(ring_mem));
}

// Rows that do not start on 16 bytes (an odd length, an offset view): the same ring, read element by
// element, 16 a thread, in the order of the lanes, so that shared memory and the stores are whole
// lines.
template <typename T>
__device__ __forceinline__ float elem(const T* p) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(*p);
  return *p;
}

template <typename T, typename W, bool LAYER, int G>
__global__ void __launch_bounds__(norm_threads<G>()) norm_fwd_odd_kernel(const NormFwd a) {
  constexpr int NT = norm_threads<G>(), RPB = NT / G, P = 16;
  extern __shared__ __align__(128) uint8_t ring_mem[];
  __shared__ float sh[2 * (NT / 32)];
  __shared__ uint64_t bars[RPB * RING_MAX];
  const int grp = threadIdx.x / G, lane = threadIdx.x % G;
  const long long step = (long long)gridDim.x * RPB, row0 = (long long)blockIdx.x * RPB;
  RowRing<T, G, 2, true> ring;
  ring.stages = a.stages;
  ring.s = 0;
  ring.phase = 0;
  ring.len = a.D * sizeof(T);
  ring.bytes = odd_place(ring.len);
  ring.base = ring_mem + (size_t)grp * a.stages * 2 * ring.bytes;
  ring.full = bars + grp * RING_MAX;
  ring.src[0] = static_cast<const T*>(a.x);
  ring.ld[0] = a.ldx;
  ring.src[1] = static_cast<const T*>(a.delta);
  ring.ld[1] = a.ldd;
  if (lane == 0) {
    for (int i = 0; i < a.stages; ++i) mbar_init(&ring.full[i], 1);
    fence_barrier_init();
  }
  grid_wait();
  grid_release();
  if (lane == 0) {
    for (int k = 0; k < a.stages; ++k)
      if (row0 + grp + k * step < a.M) ring.fill(k, row0 + grp + k * step);
  }
  __syncthreads();
  int flip = 0;
  for (long long base = row0; base < a.M; base += step) {
    const long long row = base + grp;
    const bool live = row < a.M && ring.wait(a.status);
    const T* x = ring.row_at(0, row);
    const T* d = ring.row_at(1, row);
    float f[P], sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = lane + i * G;
      f[i] = 0.f;
      if (live && c < a.D) {
        f[i] = elem(x + c);
        if (a.delta) {
          f[i] = round_to<T>(f[i] + elem(d + c));
          store_vec<T, 1>(static_cast<T*>(a.h) + row * a.D + c, &f[i]);
        }
      }
      sum[0] += LAYER ? f[i] : f[i] * f[i];
    }
    group_sum<G, 1>(sum, sh, flip);
    if constexpr (G == 32) __syncwarp();
    if (lane == 0 && row + a.stages * step < a.M) ring.fill(ring.s, row + a.stages * step);
    ring.next();
    float mu = 0.f;
    if constexpr (LAYER) {
      mu = sum[0] / a.D;
      sum[0] = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float t = lane + i * G < a.D ? f[i] - mu : 0.f;
        sum[0] += t * t;
      }
      group_sum<G, 1>(sum, sh, flip);
    }
    if (!live) continue;
    const float r = rsqrtf(sum[0] / a.D + a.eps);
    if (lane == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(mu, r);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = lane + i * G;
      if (c >= a.D) continue;
      float o = (f[i] - mu) * r * elem(static_cast<const W*>(a.w) + c);
      if (LAYER && a.b) o += elem(static_cast<const W*>(a.b) + c);
      store_vec<T, 1>(static_cast<T*>(a.y) + row * a.D + c, &o);
    }
  }
}

// The row is read from the ring twice, for the sums and for dx, instead of being held; its stage is
// filled again after the next row's reduction, when every thread is past it.
template <typename T, typename W, bool LAYER, int G>
__global__ void __launch_bounds__(norm_threads<G>()) norm_bwd_odd_kernel(const NormBwd a) {
  constexpr int NT = norm_threads<G>(), RPB = NT / G, N = LAYER ? 2 : 1, P = 16;
  extern __shared__ __align__(128) uint8_t ring_mem[];
  __shared__ float sh[2 * N * (NT / 32)];
  __shared__ uint64_t bars[RPB * RING_MAX];
  const int grp = threadIdx.x / G, lane = threadIdx.x % G;
  const long long step = (long long)gridDim.x * RPB, row0 = (long long)blockIdx.x * RPB;
  RowRing<T, G, 3, true> ring;
  ring.stages = a.stages;
  ring.s = 0;
  ring.phase = 0;
  ring.len = a.D * sizeof(T);
  ring.bytes = odd_place(ring.len);
  ring.base = ring_mem + (size_t)grp * a.stages * 3 * ring.bytes;
  ring.full = bars + grp * RING_MAX;
  ring.src[0] = static_cast<const T*>(a.h);
  ring.ld[0] = a.ldh;
  ring.src[1] = static_cast<const T*>(a.dy);
  ring.ld[1] = a.ldy;
  ring.src[2] = static_cast<const T*>(a.dh);
  ring.ld[2] = a.lddh;
  if (lane == 0) {
    for (int i = 0; i < a.stages; ++i) mbar_init(&ring.full[i], 1);
    fence_barrier_init();
  }
  grid_wait();
  grid_release();
  if (lane == 0) {
    for (int k = 0; k < a.stages; ++k)
      if (row0 + grp + k * step < a.M) ring.fill(k, row0 + grp + k * step);
  }
  float dw[P][1], db[LAYER ? P : 1][1], w[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = lane + i * G;
    w[i] = c < a.D ? elem(static_cast<const W*>(a.w) + c) : 0.f;
    dw[i][0] = 0.f;
    if constexpr (LAYER) db[i][0] = 0.f;
  }
  __syncthreads();
  int flip = 0;
  for (long long base = row0; base < a.M; base += step) {
    const long long row = base + grp;
    const bool live = row < a.M && ring.wait(a.status);
    float2 st = make_float2(0.f, 0.f);
    if (live) st = *reinterpret_cast<const float2*>(a.stats + 2 * row);
    const T* h = ring.row_at(0, row);
    const T* y = ring.row_at(1, row);
    const T* dh = ring.row_at(2, row);
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = lane + i * G;
      if (live && c < a.D) {
        const float v = elem(y + c), n = (elem(h + c) - st.x) * st.y, g = v * w[i];
        s[0] += g * n;
        dw[i][0] += v * n;
        if constexpr (LAYER) {
          s[N - 1] += g;
          db[i][0] += v;
        }
      }
    }
    group_sum<G, N>(s, sh, flip);
    if constexpr (G == 32) __syncwarp();
    if (lane == 0 && row >= row0 + grp + step && row + (a.stages - 1) * step < a.M)
      ring.fill(ring.s == 0 ? a.stages - 1 : ring.s - 1, row + (a.stages - 1) * step);
    if (live) {
      const float c1 = s[0] / a.D, c2 = LAYER ? s[N - 1] / a.D : 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = lane + i * G;
        if (c >= a.D) continue;
        const float n = (elem(h + c) - st.x) * st.y;
        float o = st.y * (elem(y + c) * w[i] - n * c1 - c2);
        if (a.dh) o += elem(dh + c);
        store_vec<T, 1>(static_cast<T*>(a.dx) + row * a.D + c, &o);
      }
    }
    ring.next();
  }
  __syncthreads();  // every copy has been waited for and read: the ring's memory is free
  write_partials<W, G, 1, P, N, RPB>(a, dw, db, reinterpret_cast<float*>(ring_mem));
}

// dw (db) = sum over blocks, in a fixed order: 32 columns a block, each of 16 warps takes every
// sixteenth partial row, joined in warp order.
constexpr int NORM_JOIN = 16;
template <typename W>
__global__ void __launch_bounds__(32 * NORM_JOIN) norm_join_kernel(const float* __restrict__ part, int blocks, int n, int D,
                                                        W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float sh[NORM_JOIN][32];
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, k = blockIdx.y;
  float t = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int b = warp; b < blocks; b += NORM_JOIN) t += part[((size_t)b * n + k) * D + c];
  }
  sh[warp][lane] = t;
  __syncthreads();
  if (warp != 0 || c >= D) return;
#pragma unroll
  for (int w = 1; w < NORM_JOIN; ++w) t += sh[w][lane];
  W* out = k == 0 ? dw : db;
  if constexpr (sizeof(W) == 2)
    out[c] = __float2bfloat16_rn(t);
  else
    out[c] = t;
}

// Threads of a row: 16 elements each where the row is long enough, with 16-byte accesses or one by one.
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
    if (D <= 512) OM_NORM_CASE(32, 1, 16);
    if (D <= 2048) OM_NORM_CASE(128, 1, 16);
    if (D <= 8192) OM_NORM_CASE(512, 1, 16);
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

// Stages of a ring: what makes about 64 KB a block, at least two; fewer than two: no ring.
static int ring_stages(size_t stage_bytes) {
  const size_t two = 2 * stage_bytes;
  if (two > 200 * 1024) return 0;
  return (int)std::min<size_t>(RING_MAX, std::max<size_t>(2, (64 * 1024) / stage_bytes));
}

// Blocks of a kernel that an SM holds, for the shared memory last asked for (a program runs few
// row lengths). The kernel is allowed that much first.
struct Residents {
  std::mutex lock;
  size_t smem = (size_t)-1, allowed = 40 * 1024;
  int dev = -1, blocks = 0;
  template <typename K>
  int get(K kernel, int threads, size_t bytes) {
    std::lock_guard<std::mutex> hold(lock);
    int d;
    OM_CUDA_CHECK(cudaGetDevice(&d));
    if (d != dev) allowed = 40 * 1024;
    if (d == dev && bytes == smem) return blocks;
    if (bytes > allowed) {
      OM_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
      allowed = bytes;
    }
    OM_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, threads, bytes));
    blocks = std::max(1, blocks);
    dev = d;
    smem = bytes;
    return blocks;
  }
};

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
// Whether every row of `t` is whole 16-byte blocks
bool norm_vec(const torch::Tensor& t) {
  return t.size(t.dim() - 1) % 8 == 0 && (t.dim() == 1 || t.stride(0) % 8 == 0) &&
         (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

}  // namespace

// (y [..., D], h (x itself without delta), stats fp32 [M, 2])
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> om_norm_train(torch::Tensor x, torch::Tensor w,
                                                                      c10::optional<torch::Tensor> b, double eps,
                                                                      bool layer, c10::optional<torch::Tensor> delta,
                                                                      torch::Tensor status) {
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
  bool vec = norm_vec(x2) && norm_vec(w2);
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
  a.status = status.data_ptr<int>();
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
      if constexpr (v == 8) {
        constexpr int RPB = NT / g;
        const size_t stage = (size_t)RPB * (delta.has_value() ? 2 : 1) * D * sizeof(T);
        a.stages = om::ring_stages(stage);
        if (a.stages >= 2) {
          auto go = [&](auto kernel, om::Residents& res) {
            const size_t smem = a.stages * stage;
            const int grid = (int)std::min<long long>(blocks, om::num_sms() * res.get(kernel, NT, smem));
            om::launch_dependent(kernel, grid, NT, smem, st, a);
          };
          static om::Residents res[4];
          if (layer && a.delta)
            go(om::norm_fwd_ring_kernel<T, W, true, true, g, p>, res[0]);
          else if (layer)
            go(om::norm_fwd_ring_kernel<T, W, true, false, g, p>, res[1]);
          else if (a.delta)
            go(om::norm_fwd_ring_kernel<T, W, false, true, g, p>, res[2]);
          else
            go(om::norm_fwd_ring_kernel<T, W, false, false, g, p>, res[3]);
          return;
        }
      } else {
        const size_t stage = (size_t)(NT / g) * 2 * om::odd_place((uint32_t)(D * sizeof(T)));
        a.stages = om::ring_stages(stage);
        if (a.stages >= 2) {
          static om::Residents res[2];
          auto kernel = layer ? om::norm_fwd_odd_kernel<T, W, true, g> : om::norm_fwd_odd_kernel<T, W, false, g>;
          const size_t smem = a.stages * stage;
          const int grid = (int)std::min<long long>(blocks, om::num_sms() * res[layer].get(kernel, NT, smem));
          om::launch_dependent(kernel, grid, NT, smem, st, a);
          return;
        }
      }
      om::launch_dependent(layer ? om::norm_fwd_kernel<T, W, true, g, v, p> : om::norm_fwd_kernel<T, W, false, g, v, p>,
                           (unsigned)blocks, NT, 0, st, a);
    });
  });
  return {y, h, stats};
}

// (dx [..., D], dw [D], db [D] (LayerNorm with bias))
std::tuple<torch::Tensor, torch::Tensor, c10::optional<torch::Tensor>> om_norm_train_bwd(
    torch::Tensor dy, torch::Tensor h, torch::Tensor w, torch::Tensor stats, bool layer, bool bias,
    c10::optional<torch::Tensor> dh, torch::Tensor status) {
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
  bool vec = norm_vec(h2) && norm_vec(y2) && norm_vec(w2);
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
  a.status = status.data_ptr<int>();
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
      auto go = [&](auto kernel, om::Residents& res, size_t smem) {
        const long long most = (M + RPB - 1) / RPB;
        int blocks = (int)std::min<long long>(most, om::num_sms() * res.get(kernel, NT, smem));
        // Few rows: one block walks them and writes dw itself. That saves a launch, 3 us of the caller's time, and
        // costs the GPU a turn's time for each: 0.5 to 0.9 us, but 2 to 3 us where rows are read element by
        // element or have more than 8192 elements. Forward and gradient, one block and several, us by the
        // caller's clock and the GPU's alone: rows of 256 (eight a turn) in 8 turns 14.3 and 17.6, 11.1 and 8.4;
        // in 16 turns 16.4 and 17.5, 15.8 and 8.6; 8192: 8 rows 14.6 and 17.7, 13.0 and 9.6, 16 rows 21.0 and
        // 17.8, 20.5 and 9.9; 16384: 2 rows 15.4 and 18.0, 14.6 and 17.3, 4 rows 20.1 and 18.1, 19.0 and 17.6;
        // 4097: 2 rows 14.5 and 17.6, 12.1 and 10.5, 4 rows 19.1 and 17.8, 18.1 and 10.7.
        if (most <= (v == 8 && a.D <= 8192 ? 8 : 2)) blocks = 1;
        torch::Tensor part;
        if (blocks > 1) {
          part = torch::empty({(int64_t)blocks * n * a.D}, stats.options());
          a.part = part.data_ptr<float>();
        }
        a.dw = dw.data_ptr();
        a.db = bias ? db->data_ptr() : nullptr;
        om::launch_dependent(kernel, blocks, NT, smem, st, a);
        if (blocks > 1)
          om::launch_dependent(om::norm_join_kernel<W>, dim3((a.D + 31) / 32, bias ? 2 : 1), 32 * om::NORM_JOIN, 0, st,
                               (const float*)a.part, blocks, n, a.D, static_cast<W*>(a.dw), static_cast<W*>(a.db));
      };
      const size_t joined = RPB > 1 ? (size_t)a.D * sizeof(float) : 0;
      if constexpr (v == 8) {
        const size_t stage = (size_t)RPB * (a.dh ? 3 : 2) * D * sizeof(T);
        a.stages = om::ring_stages(stage);
        if (a.stages >= 2) {
          const size_t smem = std::max(a.stages * stage, joined);
          static om::Residents res[4];
          if (layer && a.dh)
            go(om::norm_bwd_ring_kernel<T, W, true, true, g, p>, res[0], smem);
          else if (layer)
            go(om::norm_bwd_ring_kernel<T, W, true, false, g, p>, res[1], smem);
          else if (a.dh)
            go(om::norm_bwd_ring_kernel<T, W, false, true, g, p>, res[2], smem);
          else
            go(om::norm_bwd_ring_kernel<T, W, false, false, g, p>, res[3], smem);
          return;
        }
      } else {
        const size_t stage = (size_t)RPB * 3 * om::odd_place((uint32_t)(D * sizeof(T)));
        a.stages = om::ring_stages(stage);
        if (a.stages >= 2) {
          const size_t smem = std::max(a.stages * stage, joined);
          static om::Residents res[2];
          if (layer)
            go(om::norm_bwd_odd_kernel<T, W, true, g>, res[1], smem);
          else
            go(om::norm_bwd_odd_kernel<T, W, false, g>, res[0], smem);
          return;
        }
      }
      static om::Residents res[2];
      if (layer)
        go(om::norm_bwd_kernel<T, W, true, g, v, p>, res[1], joined);
      else
        go(om::norm_bwd_kernel<T, W, false, g, v, p>, res[0], joined);
    });
  });
  return {dx, dw, db};
}
