// Attention's backward pass on the 5th-generation tensor cores, with the probabilities computed
// again from the forward's log-sum-exp (head_dim <= 128, GQA, causal or full, padded batches).
//
//   P  = exp(c Q K^T - L)  (0 where the mask leaves a pair out)
//   dV = P^T dO                         summed over the query heads of a KV head
//   dS = P * (dO V^T - rowsum(dO * O))
//   dQ = c dS K,   dK = c dS^T Q
//
// No gradient is summed by atomics (the same result on every run). Two kinds of work items:
//   kv  128 keys of a KV head walk the 64-query tiles of its query heads: dK, dV
//   q   128 queries of a head walk the 64-key tiles: dQ
// One CTA an SM stays and takes the next item off a counter, the heavy ones first; the next item's
// rows are loaded and its first scores computed while the last one's results are written, because
// setting up a CTA and filling its pipeline (about 5 us) is more than a short item's work.
// Both keep their rows (keys, or queries) in the MMA's 128 lanes and compute S and dP of a
// 64-column tile from shared memory; the softmax threads turn the tile into P and dS and write
// them, as 16-bit pairs, over S and dP in tensor memory, from where they are the A operand of the
// accumulating products. P and dS therefore never touch shared memory, and the transposed form
// (S^T) needs no transposition. Rounding P and dS to 16 bits enters each gradient at 2^-8
// relative per term at the most, independently; sums are fp32 in tensor memory.
//
// Tensor memory of a kv item: dV 128 + dK 128 + two stages of (S 64 + dP 64) = 512 columns, all
// there are; this is what sets the 64-query tile. Eight softmax warps work on one tile, 32 columns
// a thread, and two such groups take the tiles in turn: a tile's exponentials (512 cycles at the
// SM's 16 a cycle) and its loads and stores of tensor memory have to fit beside the 1280 cycles of
// products of the tile before and after.
//
// Seven products instead of the five of a single loop is the price of the fixed summation order
// (and of no fp32 dQ in memory).
//
// What bounds it: the tensor cores take 1280 + 1024 cycles for a pair of tiles at head_dim 128 (kv + q) and are
// busy for half of the time; the rest is a tile's way through S, P, dP and dS, two tiles at once.
// Measured (B200, back to back): 1 x 8192, 40 / 8 heads of 128, causal 2.35 ms, 731 TFLOP/s of the five
// products, 1023 of the seven; 4 x <= 1499 padded, 16 / 4 heads 122 us; head_dim 64, 1 x 8192, 32 / 8 heads
// 1.27 ms, where the exponentials bound it.
//
// Padded batches: rows of Q, dO (or K) at and beyond a sequence's length are cleared in shared
// memory before a product contracts over them, so that whatever padding holds (NaN too) adds 0.
//
// Work split: where the items would leave SMs idle, the query heads of a KV head are divided among
// `nsplit` items, which leave fp32 partials that a last kernel adds in order.
#include <c10/cuda/CUDAGuard.h>
#include <type_traits>
#include "../common/om_host.h"
#include "../common/om_ptx.cuh"

namespace om {

namespace fa_bw {
constexpr float LOG2E = 1.4426950408889634f;
constexpr int NSTAGE = 4;
constexpr int THREADS = 640;  // copy, MMA, TMEM and one idle warp; two groups of eight softmax warps
template <int D>
struct Cfg {
  static constexpr int H = D / 64;               // 64-wide halves of the head dimension
  static constexpr int BIG = 128 * 64 * 2;       // one half of 128 rows
  static constexpr int SMALL = 64 * 64 * 2;      // one half of 64 rows
  static constexpr int FIX_BYTES = 2 * H * BIG;  // the two resident operands (K, V or Q, dO)
  static constexpr int ST_BYTES = 2 * H * SMALL; // the two streamed ones
  static constexpr int STAT = 64 * 8;            // -lse log2 e and -delta of 64 queries
  static constexpr int STAT_OFF = FIX_BYTES + NSTAGE * ST_BYTES;
  static constexpr int BAR_OFF = STAT_OFF + NSTAGE * STAT;
  static constexpr int SMEM = BAR_OFF + 256 + 1024;
};
}  // namespace fa_bw

struct AttnBwdArgs {
  const float* stat;    // [B, H, Tp / 64][2][64]: -lse log2 e (or -inf), -delta
  const int* lens;      // optional [B] valid tokens
  __nv_bfloat16 *dq, *dk, *dv;  // contiguous [B, T, H, D], [B, S, Hkv, D]
  float* part;          // nsplit > 1: [nsplit][2][B, S, Hkv, D]
  int B, T, S, H, Hkv, G, hd;
  int Tp;               // T rounded up to 64
  int causal, off;      // key j visible to query i when j <= i + off
  int nsplit, gper;     // kv items of a KV head and key tile, and the query heads of one
  int kv_items, items;  // kv items come first
  int* next;            // the next item
  float scale, scale_log2;
  int* status;
};

__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// -lse log2 e and -rowsum(dO * O) of every query row, 64 of each side by side for a tile of the
// kernel below. Rows without a visible key (lse = -inf), beyond the length or beyond T get
// (-inf, 0): P = 0.
// 16 lanes a row, 8 elements each; blockIdx.y is the sequence. Bound by reading out and dout.
__global__ void __launch_bounds__(256) attn_bwd_stat_kernel(const __nv_bfloat16* __restrict__ o,
                                                            const __nv_bfloat16* __restrict__ go,
                                                            const float* __restrict__ lse, const int* lens,
                                                            float* __restrict__ stat, int* next, int T, int Tp, int H,
                                                            int hd,
                                                            long long ob, long long ot, long long oh, long long gb,
                                                            long long gt, long long gh) {
  grid_wait();
  grid_release();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *next = 0;
  const int sub = threadIdx.x & 15, b = blockIdx.y;
  const unsigned n = (unsigned)Tp * H;  // below 2^31
  const int len = lens ? min(lens[b], T) : T;
  // Tp is a multiple of 64, so both halves of a warp take the same number of turns
  for (unsigned i = blockIdx.x * 16 + (threadIdx.x >> 4); i < n; i += gridDim.x * 16) {
    const int t = (int)(i / (unsigned)H), h = (int)(i - (unsigned)t * H);
    float d = 0.f, l = -INFINITY;
    if (t < len) {
      l = lse[((long long)b * T + t) * H + h];
      if (sub * 8 < hd) {
        float x[8], y[8];
        unpack8(*reinterpret_cast<const uint4*>(o + b * ob + t * ot + h * oh + sub * 8), x);
        unpack8(*reinterpret_cast<const uint4*>(go + b * gb + t * gt + h * gh + sub * 8), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) d += x[j] * y[j];
      }
    }
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
    if (sub == 0) {
      float* p = stat + (((long long)b * H + h) * Tp + (t & ~63)) * 2 + (t & 63);
      p[0] = l == -INFINITY ? -INFINITY : -l * fa_bw::LOG2E;
      p[64] = l == -INFINITY ? 0.f : -d;
    }
  }
}

// Clears rows [from, 64) of one streamed operand (H halves of 64 rows x 128 bytes).
template <int HALVES>
__device__ __forceinline__ void clear_rows(uint8_t* p, int from, int lane) {
  for (int i = lane; i < HALVES * (64 - from) * 8; i += 32) {
    const int half = i / ((64 - from) * 8), in = i % ((64 - from) * 8);
    sts128(smem_u32(p + half * fa_bw::Cfg<64>::SMALL + from * 128 + in * 16), make_uint4(0, 0, 0, 0));
  }
}

// Where tile i keeps its S (which = 0) and dP (1): 64 columns each, for both parities of i. P is written
// over S and dS over dP; the tile after the next takes both places, each when the products that read
// it are complete. (Products of one shape into one accumulator run in order by themselves, others have
// to be waited for.) The issue order dV(t), dP(t + 1), dK(t), S(t + 2) has two products between each and
// the one whose end it waits for: 1 x 8192, 40 / 8 heads of 128 2.35 ms; dK, S, dP in one go 2.40; P and dS
// both over S, so that dP waits for both products, 2.45; S as soon as dV is complete 2.66.
__device__ __forceinline__ uint32_t tile_region(int i, int which) {
  return (uint32_t)((i & 1) * 128 + which * 64);
}

// A thread's 32 columns of S -> P, kept in fp32 pairs; COLQ: also written in 16 bits over the
// first 16 of these columns. COLQ: columns are queries (S^T),
// their -lse come from shared memory; else the thread's row has one. MASK: column j is visible
// when lo <= j < hi; selected, not multiplied: what lies under a mask may be anything.
template <bool COLQ, bool MASK>
__device__ __forceinline__ void tile_p(uint32_t s_at, uint32_t stat, float own, float c2, int lo, int hi,
                                       uint64_t (&p)[16]) {
  uint32_t sv[32];
  tmem_ld_32x32b_x32(s_at, sv);
  tc_wait_ld();
  const uint64_t c = pair_f32(c2, c2);
  uint32_t pk[16];
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    uint4 u;
    if constexpr (COLQ) u = lds128(stat + j * 4);
#pragma unroll
    for (int e = j; e < j + 4; e += 2) {
      const uint64_t l = COLQ ? pair_f32(__uint_as_float(e > j ? u.z : u.x), __uint_as_float(e > j ? u.w : u.y))
                              : pair_f32(own, own);
      const float2 x = unpair_f32(fma_f32x2(pair_f32(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), c, l));
      float p0 = fast_exp2(x.x), p1 = fast_exp2(x.y);
      if constexpr (MASK) {
        p0 = e >= lo && e < hi ? p0 : 0.f;
        p1 = e + 1 >= lo && e + 1 < hi ? p1 : 0.f;
      }
      p[e / 2] = pair_f32(p0, p1);
      if constexpr (COLQ) pk[e / 2] = pack_bf16x2(p0, p1);
    }
  }
  if constexpr (COLQ) {
    tmem_st_32x32b_x16(s_at, pk);
    tc_wait_st();
  }
}

// dS = P (dP - delta) of the same columns, in 16 bits over the first 16 of them. stat / own: -delta.
template <bool COLQ, bool MASK>
__device__ __forceinline__ void tile_ds(uint32_t dp_at, uint32_t stat, float own, int lo, int hi,
                                        const uint64_t (&p)[16]) {
  uint32_t dv[32];
  tmem_ld_32x32b_x32(dp_at, dv);
  tc_wait_ld();
  uint32_t dk[16];
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    uint4 u;
    if constexpr (COLQ) u = lds128(stat + j * 4);
#pragma unroll
    for (int e = j; e < j + 4; e += 2) {
      const uint64_t l = COLQ ? pair_f32(__uint_as_float(e > j ? u.z : u.x), __uint_as_float(e > j ? u.w : u.y))
                              : pair_f32(own, own);
      float2 d = unpair_f32(
          mul_f32x2(p[e / 2], add_f32x2(pair_f32(__uint_as_float(dv[e]), __uint_as_float(dv[e + 1])), l)));
      if constexpr (MASK) {
        d.x = e >= lo && e < hi ? d.x : 0.f;
        d.y = e + 1 >= lo && e + 1 < hi ? d.y : 0.f;
      }
      dk[e / 2] = pack_bf16x2(d.x, d.y);
    }
  }
  tmem_st_32x32b_x16(dp_at, dk);
  tc_wait_st();
}

// 128 accumulator rows (lane = row) of D columns, times `f`, to global rows; rows >= `rows` are
// not there. OUT is bf16 or fp32.
template <int D, typename OUT>
__device__ __forceinline__ void write_acc(uint32_t tmem, OUT* dst, bool live, bool zero, float f, int hd) {
#pragma unroll 1
  for (int q = 0; q < D / 32; ++q) {
    uint32_t v[32];
    tmem_ld_32x32b_x32(tmem + q * 32, v);
    tc_wait_ld();
    if (!live) continue;
    float x[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = zero ? 0.f : __uint_as_float(v[j]) * f;
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      if (q * 32 + j >= hd) continue;  // hd is a multiple of 8
      if constexpr (sizeof(OUT) == 2) {
        *reinterpret_cast<uint4*>(dst + q * 32 + j) = pack8(x + j);
      } else {
        reinterpret_cast<float4*>(dst + q * 32 + j)[0] = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        reinterpret_cast<float4*>(dst + q * 32 + j)[1] = make_float4(x[j + 4], x[j + 5], x[j + 6], x[j + 7]);
      }
    }
  }
}

// Zeros for the 128 rows of an item that has no tile to walk; `t` of `n` threads.
__device__ __forceinline__ void write_zero(const AttnBwdArgs& a, bool kv, int b, int kvh, int head, int split, int row0,
                                           int t, int n) {
  const int vecs = a.hd / 8, rows = min(128, (kv ? a.S : a.T) - row0);
  const uint4 z = make_uint4(0, 0, 0, 0);
  for (int i = t; i < rows * vecs; i += n) {
    const int row = row0 + i / vecs, c = i % vecs * 8;
    if (kv) {
      const size_t at = (((size_t)b * a.S + row) * a.Hkv + kvh) * a.hd + c;
      if (a.nsplit > 1) {
        const size_t plane = (size_t)a.B * a.S * a.Hkv * a.hd;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint4* p = reinterpret_cast<uint4*>(a.part + (split * 2 + k) * plane + at);
          p[0] = z;
          p[1] = z;
        }
      } else {
        *reinterpret_cast<uint4*>(a.dk + at) = z;
        *reinterpret_cast<uint4*>(a.dv + at) = z;
      }
    } else {
      *reinterpret_cast<uint4*>(a.dq + (((size_t)b * a.T + row) * a.H + head) * a.hd + c) = z;
    }
  }
}

// A work item: its rows, heads and tiles.
struct Item {
  bool kv;
  int b, kvh, head, split, row0, first, ntile, total;
  int nstream, nrow;  // valid rows of the streamed and of the resident operands
  __device__ __forceinline__ Item(const AttnBwdArgs& a, int i) {
    kv = i < a.kv_items;
    if (!kv) i -= a.kv_items;
    const int heads = kv ? a.Hkv * a.nsplit : a.H;
    const int per = a.B * heads;
    const int tile = i / per, rest = i % per;
    b = rest / heads;
    head = rest % heads;
    split = 0;
    const int nk = a.lens ? max(0, min(a.lens[b], a.S)) : a.S;
    const int nq = a.lens ? max(0, min(a.lens[b], a.T)) : a.T;
    if (kv) {  // the heaviest are the first keys, under a causal mask
      split = head % a.nsplit;
      kvh = head / a.nsplit;
      row0 = tile * 128;
      head = kvh * a.G + split * a.gper;
      first = a.causal ? max(0, row0 - a.off) / 64 : 0;
      ntile = row0 < nk ? max(0, (nq + 63) / 64 - first) : 0;
      total = ntile * max(0, min(a.G - split * a.gper, a.gper));
      nstream = nq;
      nrow = nk;
    } else {  // and the last queries
      kvh = head / a.G;
      row0 = ((a.T + 127) / 128 - 1 - tile) * 128;
      const int last = min(nq, row0 + 128) - 1;
      const int kend = last < row0 ? 0 : (a.causal ? min(nk, last + a.off + 1) : nk);
      first = 0;
      total = ntile = kend > 0 ? (kend + 63) / 64 : 0;
      nstream = nk;
      nrow = nq;
    }
  }
};

// kv: resident K, V; streamed Q, dO (and their stats); accumulates dV, dK.
// q:  resident Q, dO; streamed K, V; accumulates dQ.
// Counters run over all items of a CTA: `tile` numbers the streamed tiles (ring stage, S / dP
// region and barrier phases go by it), `done` the items that had any.
template <int D>
__global__ void __launch_bounds__(fa_bw::THREADS, 1)
    attn_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmG,
                    const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const AttnBwdArgs a) {
  using C = fa_bw::Cfg<D>;
  constexpr int NS = fa_bw::NSTAGE;
  constexpr int STAGE0 = 256;  // tensor memory: dV [0, D), dK [128, 128 + D) / dQ [0, D), then S and dP
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* fix_full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* fix_empty = fix_full + 1;  // the item's last scores are computed
  uint64_t* full = fix_empty + 1;      // [NS]
  uint64_t* empty = full + NS;         // [NS]
  uint64_t* land = empty + NS;         // a padded tile before its rows are cleared
  uint64_t* s_full = land + 1;         // [2] S of a tile is there
  uint64_t* dp_full = s_full + 2;      // [2] dP is
  uint64_t* p_full = dp_full + 2;      // [2] P is (q items: S has been read)
  uint64_t* p_used = p_full + 2;       // [2] the products that read P are complete
  uint64_t* ds_full = p_used + 2;      // [2] dS is there
  uint64_t* acc_full = ds_full + 2;    // the item's sums are
  uint64_t* acc_empty = acc_full + 1;  // and have been read
  uint64_t* item_full = acc_empty + 1; // [2] the next item's number
  uint64_t* item_empty = item_full + 2;  // [2]
  uint64_t* drained = item_empty + 2;
  int* items = reinterpret_cast<int*>(drained + 1);  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(fix_full, 1);
    mbar_init(fix_empty, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(land, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&dp_full[s], 1);
      mbar_init(&p_full[s], 256);
      mbar_init(&p_used[s], 1);
      mbar_init(&ds_full[s], 256);
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], 17);
    }
    mbar_init(drained, 1);
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 16);
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_wait();
  grid_release();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer (the whole warp)
    bool ok = true;
    int tile = 0, landed = 0, done = 0;
    for (int k = 0; ok; ++k) {
      int n = 0;
      if (lane == 0) n = atomicAdd(a.next, 1);
      n = __shfl_sync(0xffffffffu, n, 0);
      ok = __all_sync(0xffffffffu, mbar_wait(&item_empty[k & 1], ((k >> 1) & 1) ^ 1, a.status, OM_ERR_WAIT_EMPTY));
      if (!ok) break;
      if (lane == 0) {
        items[k & 1] = n < a.items ? n : -1;
        mbar_arrive(&item_full[k & 1]);
      }
      if (n >= a.items) break;
      const Item w(a, n);
      if (w.total == 0) continue;
      const CUtensorMap* r0 = w.kv ? &tmK : &tmQ;
      const CUtensorMap* r1 = w.kv ? &tmV : &tmG;
      const CUtensorMap* x0 = w.kv ? &tmQ : &tmK;
      const CUtensorMap* x1 = w.kv ? &tmG : &tmV;
      ok = __all_sync(0xffffffffu, mbar_wait(fix_empty, (done & 1) ^ 1, a.status, OM_ERR_WAIT_EMPTY));
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(fix_full, C::FIX_BYTES);
        for (int h = 0; h < C::H; ++h)
          for (int r = 0; r < 2; ++r) {
            const int off = h * C::BIG + r * C::SMALL;
            tma_load_4d(smem + off, r0, fix_full, h * 64, w.kv ? w.kvh : w.head, w.row0 + r * 64, w.b);
            tma_load_4d(smem + C::H * C::BIG + off, r1, fix_full, h * 64, w.kv ? w.kvh : w.head, w.row0 + r * 64, w.b);
          }
      }
      __syncwarp();
      ++done;
      const bool may_pad = a.lens != nullptr && w.nstream < a.S;  // beyond T the copies fill zeros themselves
      int t = 0, hd = w.head;
      for (int i = 0; i < w.total; ++i, ++tile) {
        const int s = tile % NS, row = (w.first + t) * 64;
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((tile / NS) & 1) ^ 1, a.status, OM_ERR_WAIT_EMPTY));
        if (!ok) break;
        uint8_t* st = smem + C::FIX_BYTES + s * C::ST_BYTES;
        const bool pad = may_pad && w.nstream - row < 64;
        uint64_t* bar = pad ? land : &full[s];
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, C::ST_BYTES + (w.kv ? C::STAT : 0));
          for (int h = 0; h < C::H; ++h) {
            tma_load_4d(st + h * C::SMALL, x0, bar, h * 64, w.kv ? hd : w.kvh, row, w.b);
            tma_load_4d(st + (C::H + h) * C::SMALL, x1, bar, h * 64, w.kv ? hd : w.kvh, row, w.b);
          }
          if (w.kv)
            bulk_load(smem + C::STAT_OFF + s * C::STAT, a.stat + (((size_t)w.b * a.H + hd) * a.Tp + row) * 2, C::STAT,
                      bar);
        }
        __syncwarp();
        if (pad) {
          ok = __all_sync(0xffffffffu, mbar_wait(land, landed & 1, a.status, OM_ERR_WAIT_FULL));
          ++landed;
          if (!ok) {
            mbar_wait(land, (landed - 1) & 1, nullptr, 0);
            break;
          }
          clear_rows<2 * C::H>(st, w.nstream - row, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
        }
        if (++t == w.ntile) {
          t = 0;
          ++hd;
        }
      }
    }
    if (!ok) {  // wait (bounded) for the loads that may still be in flight
      for (int j = max(0, tile - NS); j < tile; ++j) mbar_wait(&full[j % NS], (j / NS) & 1, nullptr, 0);
      if (done > 0) mbar_wait(fix_full, (done - 1) & 1, nullptr, 0);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t IDESC_S = idesc_bf16_f32(128, 64);
      constexpr uint32_t IDESC_A = idesc_bf16_f32_bmn(128, D);
      // descriptors by their low words: this thread's instructions are what the tensor pipe waits for
      const uint32_t r_lo = smem_desc_lo(smem_u32(smem), 16);                  // K, V or Q, dO
      const uint32_t x_lo = smem_desc_lo(smem_u32(smem + C::FIX_BYTES), 16);   // streamed, K-major
      const uint32_t m_lo = smem_desc_lo(smem_u32(smem + C::FIX_BYTES), C::SMALL);  // streamed, MN-major
      // S (which = 0) or dP (1) of a tile, from the resident rows and the tile's 64
      auto scores = [&](int tile, auto which_c) {
        constexpr int which = decltype(which_c)::value;
        const uint32_t x = x_lo + (tile % NS) * (C::ST_BYTES / 16);
        const uint32_t d = tmem + STAGE0 + tile_region(tile, which);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc_mma_f16_lo(d, r_lo + (which * C::H * C::BIG + (k >> 2) * C::BIG + (k & 3) * 32) / 16,
                        x + (which * C::H * C::SMALL + (k >> 2) * C::SMALL + (k & 3) * 32) / 16, IDESC_S, k > 0);
        tc_commit(which ? &dp_full[tile & 1] : &s_full[tile & 1]);
      };
      const std::integral_constant<int, 0> S{};
      const std::integral_constant<int, 1> DP{};
      auto loaded = [&](int tile) {
        const bool there = mbar_poll(&full[tile % NS], (tile / NS) & 1, a.status, OM_ERR_WAIT_FULL);
        tc_fence_after();
        return there;
      };
      auto p_gone = [&](int tile) {  // the products that read P of a tile are complete
        const bool so = mbar_poll(&p_used[tile & 1], (tile >> 1) & 1, a.status, OM_ERR_WAIT_ACCUM);
        tc_fence_after();
        return so;
      };
      auto ds_gone = [&](int tile) {  // those that read its dS are
        const bool so = mbar_poll(&empty[tile % NS], (tile / NS) & 1, a.status, OM_ERR_WAIT_ACCUM);
        tc_fence_after();
        return so;
      };
      // S and dP of a tile in the place of the tile two before
      auto both = [&](int tile) {
        if (!loaded(tile) || !(tile < 2 || p_gone(tile - 2))) return false;
        scores(tile, S);
        if (!(tile < 2 || ds_gone(tile - 2))) return false;
        scores(tile, DP);
        return true;
      };
      int tile = 0, done = 0;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        ok = mbar_poll(&item_full[k & 1], (k >> 1) & 1, a.status, OM_ERR_WAIT_FULL);
        if (!ok) break;
        const int n = items[k & 1];
        mbar_arrive(&item_empty[k & 1]);
        if (n < 0) break;
        const Item w(a, n);
        if (w.total == 0) continue;
        ok = mbar_poll(fix_full, done & 1, a.status, OM_ERR_WAIT_FULL);
        for (int i = 0; i < 2 && i < w.total && ok; ++i) ok = both(tile + i);
        if (ok && w.total <= 2) tc_commit(fix_empty);
        for (int i = 0; i < w.total && ok; ++i, ++tile) {
          const uint32_t x = m_lo + (tile % NS) * (C::ST_BYTES / 16);
          const uint32_t p = tmem + STAGE0 + tile_region(tile, 0), ds = tmem + STAGE0 + tile_region(tile, 1);
          ok = mbar_poll(&p_full[tile & 1], (tile >> 1) & 1, a.status, OM_ERR_WAIT_ACCUM) &&
               // the sums of the item before have been read
               (i > 0 || mbar_poll(acc_empty, (done & 1) ^ 1, a.status, OM_ERR_WAIT_ACCUM));
          if (!ok) break;
          tc_fence_after();
          if (w.kv) {
#pragma unroll
            for (int j = 0; j < 4; ++j)  // dV += P^T dO, 16 queries a step
              tc_mma_f16_ts_lo(tmem, p + (j >> 1) * 32 + (j & 1) * 8, x + (C::H * C::SMALL + j * 2048) / 16, IDESC_A,
                               j > 0 ? 1 : i);
          }
          tc_commit(&p_used[tile & 1]);
          if (i > 0 && i + 1 < w.total) {
            ok = ds_gone(tile - 1);
            if (!ok) break;
            scores(tile + 1, DP);
            if (i + 2 == w.total) tc_commit(fix_empty);  // the item's last scores
          }
          ok = mbar_poll(&ds_full[tile & 1], (tile >> 1) & 1, a.status, OM_ERR_WAIT_ACCUM);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + (w.kv ? 128 : 0);
#pragma unroll
          for (int j = 0; j < 4; ++j)  // dK += dS^T Q, or dQ += dS K
            tc_mma_f16_ts_lo(d, ds + (j >> 1) * 32 + (j & 1) * 8, x + j * 2048 / 16, IDESC_A, j > 0 ? 1 : i);
          tc_commit(&empty[tile % NS]);
          if (i + 2 < w.total) {
            ok = loaded(tile + 2) && p_gone(tile);
            if (!ok) break;
            scores(tile + 2, S);
          }
        }
        if (ok) tc_commit(acc_full);
        ++done;
      }
      if (!ok) {  // wait (bounded) for the products that may still be running
        tc_commit(drained);
        mbar_wait(drained, 0, nullptr, 0);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax and output
    const int group = (warp - 4) >> 3;           // tiles of one parity
    const int half = ((warp - 4) >> 2) & 1;      // columns 32 half .. of a tile
    const int t = (warp & 3) * 32 + lane;        // row == TMEM lane
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    int tile = 0, done = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      ok = __all_sync(0xffffffffu, mbar_wait(&item_full[k & 1], (k >> 1) & 1, a.status, OM_ERR_WAIT_FULL));
      if (!ok) break;
      const int n = items[k & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[k & 1]);
      if (n < 0) break;
      const Item w(a, n);
      if (w.total == 0) {
        write_zero(a, w.kv, w.b, w.kvh, w.head, w.split, w.row0, threadIdx.x - 128, 512);
        continue;
      }
      const int row = w.row0 + t;
      float2 own = make_float2(0.f, 0.f);
      bool zero = false;
      if (!w.kv) {
        own.x = -INFINITY;
        if (row < w.nrow) {
          const float* p = a.stat + (((size_t)w.b * a.H + w.head) * a.Tp + (row & ~63)) * 2 + (row & 63);
          own = make_float2(p[0], p[64]);
        }
        zero = own.x == -INFINITY;               // padding, or no visible key: gradient 0
      }
      auto walk = [&](auto kv_c) {
        constexpr bool KV = decltype(kv_c)::value;
        const int skip = (group ^ tile) & 1;     // this group's first tile of the item
        int q = skip % w.ntile;
        for (int i = skip; i < w.total; i += 2) {
          const int it = tile + i, x0 = (w.first + q) * 64;
          q += 2;
          while (q >= w.ntile) q -= w.ntile;
          // whoever reads a tile's statistics waits for their copy as well
          if constexpr (KV) ok = mbar_wait(&full[it % NS], (it / NS) & 1, a.status, OM_ERR_WAIT_FULL);
          ok = ok && mbar_wait(&s_full[it & 1], (it >> 1) & 1, a.status, OM_ERR_WAIT_ACCUM);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) return;
          tc_fence_after();
          const uint32_t s_at = lanes + STAGE0 + tile_region(it, 0) + half * 32;
          const uint32_t dp_at = lanes + STAGE0 + tile_region(it, 1) + half * 32;
          const uint32_t stat = smem_u32(smem + C::STAT_OFF + (it % NS) * C::STAT) + half * 128;
          const bool masked = KV ? w.row0 + 128 > w.nrow || (a.causal && w.row0 + 127 > x0 + a.off)
                                 : x0 + 64 > w.nstream || (a.causal && x0 + 63 > w.row0 + a.off);
          const int lo = (!KV ? 0 : row >= w.nrow ? 64 : (a.causal ? row - a.off - x0 : 0)) - half * 32;
          const int hi = (KV ? 64 : min(w.nstream - x0, a.causal ? row + a.off + 1 - x0 : 64)) - half * 32;
          uint64_t p[16];
          if (masked)
            tile_p<KV, true>(s_at, stat, own.x, a.scale_log2, lo, hi, p);
          else
            tile_p<KV, false>(s_at, stat, own.x, a.scale_log2, lo, hi, p);
          tc_fence_before();
          mbar_arrive(&p_full[it & 1]);
          ok = __all_sync(0xffffffffu, mbar_wait(&dp_full[it & 1], (it >> 1) & 1, a.status, OM_ERR_WAIT_ACCUM));
          if (!ok) return;
          tc_fence_after();
          if (masked)
            tile_ds<KV, true>(dp_at, stat + 256, own.y, lo, hi, p);
          else
            tile_ds<KV, false>(dp_at, stat + 256, own.y, lo, hi, p);
          tc_fence_before();
          mbar_arrive(&ds_full[it & 1]);
        }
      };
      if (w.kv)
        walk(std::true_type{});
      else
        walk(std::false_type{});
      if (!ok) break;
      tile += w.total;
      ok = __all_sync(0xffffffffu, mbar_wait(acc_full, done & 1, a.status, OM_ERR_WAIT_ACCUM));
      if (!ok) break;
      ++done;
      tc_fence_after();
      const int col0 = half * (D / 2);  // each half writes half of the columns
      if (w.kv) {                       // group 0 writes dV, group 1 dK
        const bool live = row < a.S;
        const size_t at = (((size_t)w.b * a.S + row) * a.Hkv + w.kvh) * a.hd + col0;
        const float f = group ? a.scale : 1.f;
        const uint32_t acc = lanes + group * 128 + col0;
        if (a.nsplit > 1) {
          const size_t plane = (size_t)a.B * a.S * a.Hkv * a.hd;
          write_acc<D / 2>(acc, a.part + (w.split * 2 + group) * plane + at, live, zero, f, a.hd - col0);
        } else {
          write_acc<D / 2>(acc, (group ? a.dk : a.dv) + at, live, zero, f, a.hd - col0);
        }
      } else if (group == 0) {
        write_acc<D / 2>(lanes + col0, a.dq + (((size_t)w.b * a.T + row) * a.H + w.head) * a.hd + col0, row < a.T, zero,
                         a.scale, a.hd - col0);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds the query-head splits' fp32 partials in split order.
__global__ void __launch_bounds__(256) attn_bwd_join_kernel(const float* __restrict__ part, int nsplit, long long n,
                                                            __nv_bfloat16* __restrict__ dv,
                                                            __nv_bfloat16* __restrict__ dk) {
  grid_wait();
  grid_release();
  for (long long i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < 2 * n; i += gridDim.x * 1024ll) {
    const int k = i >= n;
    const long long at = i - k * n;  // n is a multiple of 8
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < nsplit; ++j) {
      const float4 p = *reinterpret_cast<const float4*>(part + (2 * j + k) * n + at);
      s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
    }
    uint2 o;
    o.x = pack_bf16x2(s.x, s.y);
    o.y = pack_bf16x2(s.z, s.w);
    *reinterpret_cast<uint2*>((k ? dk : dv) + at) = o;
  }
}

// [B, T, H, D] rows (D contiguous) as a 4-D map with boxes of 64 tokens x 64 elements
static CUtensorMap map_bthd(const torch::Tensor& x) {
  const uint64_t B = x.size(0), T = x.size(1), H = x.size(2), D = x.size(3);
  CUtensorMap m;
  cuuint64_t dims[4] = {D, H, T, B};
  // the stride of a dimension of one element is never used: give it a legal value
  const uint64_t sh = H > 1 ? x.stride(2) : D, st = T > 1 ? x.stride(1) : H * D, sb = B > 1 ? x.stride(0) : T * H * D;
  cuuint64_t strides[3] = {sh * 2, st * 2, sb * 2};
  cuuint32_t box[4] = {64, 1, 64, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  CUresult r = encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, x.data_ptr(), dims, strides, box, es,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "attention_bwd: cuTensorMapEncodeTiled failed: ", num((int)r));
  return m;
}

template <int D>
static void attn_bwd_launch(const AttnBwdArgs& a, const CUtensorMap& q, const CUtensorMap& g, const CUtensorMap& k,
                            const CUtensorMap& v, cudaStream_t st) {
  using C = fa_bw::Cfg<D>;
  static std::atomic<bool> attr_set[64];
  int dev;
  OM_CUDA_CHECK(cudaGetDevice(&dev));
  if (!attr_set[dev].load()) {
    OM_CUDA_CHECK(cudaFuncSetAttribute(attn_bwd_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr_set[dev].store(true);
  }
  launch_dependent(attn_bwd_kernel<D>, std::min(a.items, num_sms()), fa_bw::THREADS, C::SMEM, st, q, g, k, v, a);
  if (a.nsplit > 1) {
    const long long n = (long long)a.B * a.S * a.Hkv * a.hd;
    const int jb = (int)std::min<long long>((2 * n + 1023) / 1024, (long long)num_sms() * 8);
    launch_dependent(attn_bwd_join_kernel, jb, 256, 0, st, (const float*)a.part, a.nsplit, n, a.dv, a.dk);
  }
}

}  // namespace om

namespace {

// [B, T, H, D] bf16 as the kernels read it: D contiguous, every other stride a positive multiple
// of 8 (16 bytes). Anything else is copied.
torch::Tensor read_rows(const torch::Tensor& t, const char* name, int64_t b, int64_t n, int64_t h, int64_t d) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 4 && t.size(0) == b && t.size(1) == n && t.size(2) == h && t.size(3) == d,
              "attention_bwd: ", name, " must be a CUDA tensor [", om::num(b), ", ", om::num(n), ", ", om::num(h),
              ", ", om::num(d), "]");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, "attention_bwd: ", name, " must be bf16");
  if (t.numel() == 0) return t;
  bool ok = t.stride(3) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) % 8 == 0 && t.stride(i) > 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

}  // namespace

// (dq, dk, dv) of q, out, dout [B, T, H, D] and k, v [B, S, Hkv, D], lse fp32 [B, T, H] natural log,
// lens int32 [B] (T == S).
std::vector<torch::Tensor> om_attention_bwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor out,
                                            torch::Tensor lse, torch::Tensor dout, c10::optional<torch::Tensor> lens,
                                            double scale, bool causal, torch::Tensor status) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4, "attention_bwd: q [B, T, H, D], k / v [B, S, Hkv, D]");
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3), S = k.size(1), Hkv = k.size(2);
  TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "attention_bwd: head_dim must be a multiple of 8 up to 128 (got ",
              om::num(D), ")");
  TORCH_CHECK(Hkv > 0 && H % Hkv == 0, "attention_bwd: query heads must be a multiple of KV heads");
  TORCH_CHECK(T < (1 << 30) && S < (1 << 30) && ((T + 63) / 64 * 64) * H < (1ll << 31) && B < 65536,
              "attention_bwd: batch, sequence or head count too large");
  TORCH_CHECK(q.is_cuda(), "attention_bwd: CUDA tensors required");
  const c10::cuda::CUDAGuard guard(q.device());
  q = read_rows(q, "q", B, T, H, D);
  k = read_rows(k, "k", B, S, Hkv, D);
  v = read_rows(v, "v", B, S, Hkv, D);
  out = read_rows(out, "out", B, T, H, D);
  dout = read_rows(dout, "dout", B, T, H, D);
  TORCH_CHECK(lse.is_cuda() && lse.scalar_type() == at::kFloat && lse.dim() == 3 && lse.size(0) == B &&
                  lse.size(1) == T && lse.size(2) == H,
              "attention_bwd: lse must be fp32 [B, T, H]");
  lse = lse.contiguous();
  om::AttnBwdArgs a{};
  if (lens.has_value()) {
    TORCH_CHECK(T == S, "attention_bwd: lens needs as many queries as keys");
    TORCH_CHECK(lens->is_cuda() && lens->dim() == 1 && lens->size(0) == B, "attention_bwd: lens must be int32 [B]");
    lens = lens->to(at::kInt).contiguous();
    a.lens = lens->data_ptr<int>();
  }
  auto dq = torch::empty({B, T, H, D}, q.options());
  auto dk = torch::empty({B, S, Hkv, D}, q.options());
  auto dv = torch::empty({B, S, Hkv, D}, q.options());
  if (B == 0 || T == 0 || S == 0 || H == 0) {
    dq.zero_();
    dk.zero_();
    dv.zero_();
    return {dq, dk, dv};
  }
  auto st = at::cuda::getCurrentCUDAStream().stream();
  auto ptr = [](const torch::Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); };
  a.B = (int)B; a.T = (int)T; a.S = (int)S; a.H = (int)H; a.Hkv = (int)Hkv; a.G = (int)(H / Hkv); a.hd = (int)D;
  a.Tp = (int)((T + 63) / 64 * 64);
  a.causal = causal;
  a.off = (int)(S - T);
  a.scale = (float)scale;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.dq = ptr(dq);
  a.dk = ptr(dk);
  a.dv = ptr(dv);
  a.status = status.data_ptr<int>();
  // A kv item with all query heads of its KV head walks up to G T / 64 tiles. The launch ends about
  // when the longest item or the average SM does, so an item gets as many heads as fit into the
  // average (a q tile counts 0.75 of a kv tile), and all of them where that is a few tiles anyway
  // (a join costs more). Split and not, 16 / 4 heads of 128: 1 x 2048 92 and 123 us; 1 x 512 (32 tiles) 25.6
  // and 39.2; 1 x 256 (16 tiles) 23.5 and 24.5; 1 x 128 23.3 and 19.7. 1 x 4096, 16 / 2 heads 236 and 449.
  const int64_t qt = (T + 63) / 64, kt = (S + 127) / 128;
  const double average = (double)B * H * qt * kt * (causal ? 0.5 : 1.0) * 1.75 / om::num_sms();
  a.gper = a.G * qt < 16 ? a.G : (int)std::min<double>(a.G, std::max(1.0, average / qt));
  a.nsplit = (a.G + a.gper - 1) / a.gper;
  const int64_t kv_items = kt * B * Hkv * a.nsplit, q_items = (T + 127) / 128 * B * H;
  TORCH_CHECK(kv_items + q_items < (1ll << 30), "attention_bwd: too many tiles");
  a.kv_items = (int)kv_items;
  a.items = (int)(kv_items + q_items);
  // scratch: the rows' statistics, then the split heads' partials, then the item counter
  const int64_t stat_floats = B * H * a.Tp * 2, plane = B * S * Hkv * D;
  auto ws = torch::empty({stat_floats + (a.nsplit > 1 ? 2 * a.nsplit * plane : 0) + 1}, lse.options());
  float* stat = ws.data_ptr<float>();
  a.stat = stat;
  a.part = a.nsplit > 1 ? ws.data_ptr<float>() + stat_floats : nullptr;
  a.next = reinterpret_cast<int*>(ws.data_ptr<float>() + ws.numel() - 1);
  const int64_t rows = (int64_t)a.Tp * H;
  const int blocks = (int)std::min<int64_t>((rows + 15) / 16, std::max<int64_t>(1, om::num_sms() * 16 / B));
  om::launch_dependent(om::attn_bwd_stat_kernel, dim3(blocks, (unsigned)B), 256, 0, st, ptr(out), ptr(dout),
                       lse.data_ptr<float>(), a.lens, stat, a.next, a.T, a.Tp, a.H, a.hd, (long long)out.stride(0),
                       (long long)out.stride(1), (long long)out.stride(2), (long long)dout.stride(0),
                       (long long)dout.stride(1), (long long)dout.stride(2));
  const CUtensorMap mq = om::map_bthd(q), mg = om::map_bthd(dout), mk = om::map_bthd(k), mv = om::map_bthd(v);
  if (D <= 64)
    om::attn_bwd_launch<64>(a, mq, mg, mk, mv, st);
  else
    om::attn_bwd_launch<128>(a, mq, mg, mk, mv, st);
  return {dq, dk, dv};
}
