// Dense attention over key intervals, backward, on sm_100a (tcgen05 + TMA + TMEM).
//
// With s = sm_scale q.k, z = s or cap tanh(s / cap), p_ij = e^(z_ij - lse_i):
//   delta_i = do_i . o_i,   dz_ij = p_ij (do_i . v_j - delta_i),   ds_ij = dz_ij (1 - (z_ij / cap)^2)
//   dv_j = sum_i p_ij do_i,   dk_j = sm_scale sum_i ds_ij q_i,   dq_i = sm_scale sum_j ds_ij k_j
// Nothing of size Sq x Sk is kept: the scores are computed again from q, k and lse.
//
// Two kernels of their own for (dk, dv) and for dq.  The scores and do.v are computed in both, 7 products where one
// kernel would need 5, but neither adds into memory that another CTA adds into: no atomics, the same bits every
// time, fp32 accumulators from the first product to the one rounding of the result.
//   dkv_kernel: a CTA owns 128 keys of one key head and walks the query tiles that see them, over every query
//               head that shares the key head.   S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//   dq_kernel : a CTA owns 128 queries and walks their key tiles.  S = Q K^T, dP = dO V^T, dQ += dS K
// P^T and dS^T (dS) are rounded to 16 bits into tensor memory, over the scores they came from, as the A operands of
// the second products.  TMEM: S, dP, dV, dK, or S, dP twice, dQ, 128 columns each.
//
// Roles (320 threads, one CTA to an SM): warps 0-7 compute, warps 0-3 on columns 0-63 of a score tile and 4-7 on
// 64-127; warp 8 issues the products; warp 9 loads.  The products' order lets each phase of the arithmetic run beside
// products that do not need it:
//   dkv: S(0) dP(0) [P(i) ready] dV(i) S(i+1) [dS(i) ready] dK(i) dP(i+1) ...
//   dq : S(0) dP(0) [S(j) read] S(j+1) dP(j+1) [dS(j) ready] dQ(j) ...
//
// Where key tiles are few, the query heads of a key head are shared by the CTAs of a cluster, which add up their sums over
// distributed shared memory, in the order of the CTAs.
//
// Measured, forward and backward: 9,360 rows x 8 heads, D 128, 1,560 of conditioning, 1.49 to 1.52 ms (920 TFLOP/s of
// what is computed); 4,680 rows of 9 documents, 16 heads on 4, 0.32 ms (0.05 more without clusters).  fp16's scaling costs
// 0.7 % of 9,360 causal rows, and 5 % of 5 rows over 100,000 keys, whose values are read once more.  Bound by the port of
// the shared memory, which the operands of the products pass, and by the arithmetic between the products.
//
// Masked places: p and ds are set to 0 by comparison, whatever the scores hold; rows of empty queries (dkv) and keys
// in front of or behind all of the tile's intervals (dq) are zeroed in shared memory, since 0 * NaN would be NaN.
// Every wait is bounded (bsa_ptx.cuh).
#include <climits>
#include <type_traits>
#include "bsa_dense.cuh"
#include "bsa_rows.cuh"

namespace bsa {
namespace dense {

__device__ int g_dense_bwd_err;

constexpr int kBwdThreads = 320;
constexpr uint32_t kColA = 0, kColB = 128, kColC = 256, kColD = 384;  // tensor memory, 128 columns each
// Up to this many steps of a CTA, p and ds go through the second products as their rounding and what it left over, so
// that a gradient carries no error but its own rounding's.  Beyond, the one rounding of p and ds to the tensors' type adds
// as much again (1.4 times the error).  4 steps cost nothing measurable, 8 would cost 4,680 rows of 9 documents 1 % and
// 1,000 rows x 32 heads 8 %, 16 would cost 3 % and, at 2,000 rows x 16 heads, 9 %.
constexpr int kFineSteps = 4;

struct BwdParams {
  const int2* ranges;   // [Bm][Sq], null: all keys
  const int4* table;
  int Bm, H, Hk, G, Sq, Sk, D;
  int q_tiles, k_tiles, Sq_pad;
  int cluster;          // CTAs that share the query heads of a key tile (dkv)
  float scale_log2, sm_scale;
  Cap cap;
  float* lse2;          // [B * H][Sq_pad]: lse in log2 (+inf: no keys)
  float* delta;         // [B * H][Sq_pad]
  int* up;              // fp16: [B * H][Sq_pad] powers of two above |do|, then of 16 rows each the most of those and of delta's
  int* v_up;            // fp16: [B * Hk][kBins] powers of two above |v| of the keys that are seen, v_bin of them each
  int v_bin, v_bins;
  Tensor4 v;
  int heads;            // B * H
  float cap_inv, cap_mask;  // 1 / cap.log2, and a score below every capped one by 2^300
  float cap_mask_rest;      // a rest with such a score
  int2* rng;            // [Bm][Sq_pad]: ranges, padded with empty ones
  const float* lse;
  Tensor4 o, g;         // forward output, its gradient
  const void* o_lo;     // what the output's rounding left over, contiguous
  Tensor4 d0, d1;       // dk, dv or dq
};

// ------------------------------------------------------------------------- row statistics
// 16 lanes to a row.  delta in fp32 from o to twice its type's bits: do.v - delta is a difference of near values where
// few keys share a row, and with the rounded o alone dq and dk came out with twice the error of their own rounding
// (0.0034 against 0.0017 on causal documents in bf16).
//
// fp16 keeps 11 bits only between 2^-14 and 2^16, and ds is a product of p, which falls with the number of keys, of do and
// of v, which may be small or large altogether.  So p and ds are multiplied by powers of two, which their sums are divided
// by again: p by 2^kUp, ds by 2^n, n <= kUp, such that 2^n |ds_ij| <= 2^n (|do_i| |v_j| + |delta_i|) < 2^15 by the
// norms of the rows.  dq, whose rows are queries, takes n for each query, with the largest |v_j| of the keys that its tile
// sees; dk, whose rows are keys, for each key, with the largest |do_i| and |delta_i| of its CTA's queries.  Rows that are
// not finite choose nothing: what they touch is not finite either.
constexpr int kUp = 15, kBelow = 14;
constexpr int kBins = 128;  // runs of keys of a head, at least 64 keys each

// The least e with |x| < 2^e; -126 for 0 and for what is not finite
__device__ __forceinline__ int log2_above(float x) {
  const int e = static_cast<int>((__float_as_uint(x) >> 23) & 255u);
  return e == 255 ? -126 : e - 126;
}
// ... of a vector whose square is x
__device__ __forceinline__ int log2_above_root(float x) { return (log2_above(x) + 1) >> 1; }
__device__ __forceinline__ int pack_most(int g, int d) { return (g + 256) << 16 | (d + 256); }
__device__ __forceinline__ int most_g(int m) { return (m >> 16) - 256; }
__device__ __forceinline__ int most_d(int m) { return (m & 0xffff) - 256; }

// The power of two above |v| of the keys of run blockIdx.x that some row may see (that lie between the first and the last key
// of some 128 rows: what lies elsewhere must not choose anything).  16 lanes to a key, all threads of the CTA.
__device__ __forceinline__ void values_above(const BwdParams& p, int b, int hk, uint32_t (*top)[8]) {
  const int first = blockIdx.x * p.v_bin, end = min(p.Sk, first + p.v_bin);
  const int lane = threadIdx.x & 15;
  __shared__ uint32_t seen[2];
  float most = 0.f;
  for (int base = first; base < end; base += 64) {
    uint64_t mask = ~0ull;
    if (p.table) {
      if (threadIdx.x < 2) seen[threadIdx.x] = 0u;
      __syncthreads();
      uint64_t mine = 0ull;
      for (int i = threadIdx.x; i < p.q_tiles; i += 256) {
        const int4 t = p.table[static_cast<long long>(p.Bm > 1 ? b : 0) * p.q_tiles + i];
        const int lo = max(t.x, base), hi = min(t.y, base + 64);
        if (lo < hi) mine |= (~0ull >> (64 - (hi - lo))) << (lo - base);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t any = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(mine >> (32 * w)));
        if ((threadIdx.x & 31) == 0 && any) atomicOr(&seen[w], any);
      }
      __syncthreads();
      mask = static_cast<uint64_t>(seen[1]) << 32 | seen[0];
      __syncthreads();
    }
    float n2[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = 16 * u + (threadIdx.x >> 4);
      n2[u] = 0.f;
      if (base + at < end && 8 * lane < p.D && (mask >> at & 1u)) {
        Row8<__half> v;
        v.load(static_cast<const __half*>(p.v.p) + b * p.v.sb + hk * p.v.sh + (base + at) * p.v.ss + 8 * lane);
        float f[8];
        v.get(f);
#pragma unroll
        for (int e = 0; e < 8; ++e) n2[u] = fmaf(f[e], f[e], n2[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) n2[u] += __shfl_xor_sync(0xffffffffu, n2[u], o);
      if (n2[u] < INFINITY) most = fmaxf(most, n2[u]);
    }
  }
  const uint32_t warp = __reduce_max_sync(0xffffffffu, __float_as_uint(most));  // >= 0: ordered as its bits
  if ((threadIdx.x & 31) == 0) (*top)[threadIdx.x >> 5] = warp;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t m = (*top)[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) m = max(m, (*top)[w]);
    p.v_up[(static_cast<long long>(b) * p.Hk + hk) * kBins + blockIdx.x] = log2_above_root(__uint_as_float(m));
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(256) stats_kernel(const BwdParams p) {
  constexpr int kLanes = 16;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  const int row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool on = row < p.Sq;
  __shared__ uint32_t most[8];
  for (int bh = blockIdx.y; bh < p.heads; bh += gridDim.y) {
    const int b = bh / p.H, h = bh - b * p.H;
    if constexpr (kHalf) {
      if (static_cast<int>(blockIdx.x) < p.v_bins && h % p.G == 0) values_above(p, b, h / p.G, &most);
      if (static_cast<int>(blockIdx.x) >= p.Sq_pad / 16) continue;
    }
    const long long at = static_cast<long long>(bh) * p.Sq_pad + row;
    float dot = 0.f, norm2 = 0.f;
    if (on && 8 * lane < p.D) {
      Row8<T> o, g, r;
      r.load(static_cast<const T*>(p.o_lo) + (static_cast<long long>(bh) * p.Sq + row) * p.D + 8 * lane);
      o.load(static_cast<const T*>(p.o.p) + b * p.o.sb + h * p.o.sh + row * p.o.ss + 8 * lane);
      g.load(static_cast<const T*>(p.g.p) + b * p.g.sb + h * p.g.sh + row * p.g.ss + 8 * lane);
      float a[8], c[8], d[8];
      o.get(a);
      g.get(c);
      r.get(d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dot = fmaf(a[e] + d[e], c[e], dot);
        norm2 = fmaf(c[e], c[e], norm2);
      }
    }
#pragma unroll
    for (int s = kLanes / 2; s > 0; s >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, s);
      if constexpr (kHalf) norm2 += __shfl_xor_sync(0xffffffffu, norm2, s);
    }
    float l = INFINITY;
    if (on) l = p.lse[static_cast<long long>(bh) * p.Sq + row] * 1.4426950408889634f;
    const bool keys = on && l != -INFINITY;
    if (!keys) l = INFINITY;  // e^(z - lse) is 0 then
    if (lane == 0) {
      p.lse2[at] = kHalf ? l - kUp : l;
      p.delta[at] = keys ? dot : 0.f;
      if (h == 0 && b < p.Bm && p.rng)
        p.rng[static_cast<long long>(b) * p.Sq_pad + row] =
            on ? p.ranges[static_cast<long long>(b) * p.Sq + row] : make_int2(0, 0);
    }
    if constexpr (kHalf) {
      const int eg = keys ? log2_above_root(norm2) : -126, ed = keys ? log2_above(dot) : -126;
      if (lane == 0) p.up[at] = eg;
      const int mg = __reduce_max_sync(0xffffffffu, eg), md = __reduce_max_sync(0xffffffffu, ed);
      if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = pack_most(mg, md);
      __syncthreads();
      if (threadIdx.x == 0) {
        int g = -126, d = -126;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          g = max(g, most_g(most[w]));
          d = max(d, most_d(most[w]));
        }
        (p.up + static_cast<long long>(p.heads) * p.Sq_pad)[static_cast<long long>(bh) * (p.Sq_pad / 16) + blockIdx.x] =
            pack_most(g, d);
      }
      __syncthreads();
    }
  }
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void put_masked(uint32_t* r, const uint32_t* seen, uint32_t v) {
#pragma unroll
  for (int e = 0; e < 64; ++e)
    if (!(seen[e >> 5] & (1u << (e & 31)))) r[e] = v;
}

template <int N>
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// Products of a 128 x N accumulator: A and B along d (K-major both), or A in tensor memory (two runs of 32 columns at
// `a` and `a` + 64, 64 values of K each) and B by rows.
template <int DP>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t b, uint32_t id) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) umma_ss(d, desc_d(a, kk), desc_d(b, kk), id, kk > 0);
}
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t id, bool add) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    umma_ts(d, a + (kk >> 2) * 64 + (kk & 3) * 8, desc_rows(b, kk), id, add || kk > 0);
}

// What the 16-bit roundings of two values leave over, as a pair
template <bool kBF16>
__device__ __forceinline__ uint32_t rest16(uint32_t pair, float x0, float x1) {
  float lo, hi;
  unpack16<kBF16>(pair, lo, hi);
  return pack16<kBF16>(x0 - lo, x1 - hi);
}

// One warp's 32 rows x (DP / 2) columns of an accumulator, times f, to 16-bit rows of a tensor.
template <int DP, bool kBF16>
__device__ __forceinline__ void store_acc(uint32_t addr, int col0, float f, void* out, long long off, int D, bool live,
                                          bool some) {
#pragma unroll 1
  for (int c = 0; c < DP / 64; ++c) {
    uint32_t r[32];
    if (some) {
      tmem_ld32(addr + col0 + 32 * c, r);
      tmem_ld_wait();
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) r[e] = 0u;
    }
    float v[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]) * f;
    if (live) {
#pragma unroll
      for (int e8 = 0; e8 < 4; ++e8) {
        const int d0 = col0 + 32 * c + 8 * e8;
        if (d0 < D) store8<kBF16>(out, off + d0, v + 8 * e8);
      }
    }
  }
}

// One warp's 32 rows x (DP / 2) columns of an accumulator to shared memory as fp32, [4 columns][row][4], so that lanes
// write side by side.
template <int DP>
__device__ __forceinline__ void to_shared(uint32_t addr, int half, int row, float f, uint8_t* dst, bool some) {
#pragma unroll 1
  for (int c = 0; c < DP / 64; ++c) {
    const int c0 = half * (DP / 2) + 32 * c;
    uint32_t r[32];
    if (some) {
      tmem_read32(addr + c0, r);
#pragma unroll
      for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) r[e] = 0u;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      *reinterpret_cast<uint4*>(dst + ((c0 / 4 + e) * kTile + row) * 16) =
          make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
  }
}

// All threads of all CTAs of the cluster; every CTA comes here whatever happened before.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 load_peer(uint32_t addr, int rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

// ------------------------------------------------------------------------- dk, dv
template <int DP>
struct DkvSmem {
  static constexpr int kQ = DP == 128 ? 2 : 4;   // query tiles in flight
  static constexpr int kG = DP == 128 ? 2 : 4;   // tiles of do in flight
  static constexpr int kTiles = (2 + kQ + kG) * tile_bytes<DP>();
  alignas(16) float lse2[kQ][kTile], delta[kQ][kTile];
  alignas(16) int2 rng[kQ][kTile];
  uint64_t kv_full;
  uint64_t q_full[kQ], q_empty[kQ], g_full[kG], g_empty[kG];
  uint64_t fix;
  uint64_t s_full, dp_full, p_full, ds_full, done, drain;
  uint32_t tmem;
  int abort_flag;
  int first, last;
  int most[2];  // fp16: powers of two above |do| and |delta| of the CTA's queries
};
template <int DP>
constexpr int dkv_smem_bytes() { return DkvSmem<DP>::kTiles + static_cast<int>(sizeof(DkvSmem<DP>)) + 1024; }

template <int DP, bool kBF16, bool kCap>
__global__ void __launch_bounds__(kBwdThreads, 1)
    dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_g, const BwdParams p) {
  using S = DkvSmem<DP>;
  constexpr int kBytes = tile_bytes<DP>();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sK = smem, *sV = smem + kBytes, *sQ = smem + 2 * kBytes, *sG = sQ + S::kQ * kBytes;
  S& ss = *reinterpret_cast<S*>(smem + S::kTiles);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // key tiles ascending: under a causal mask the first are seen by the most queries
  const int item = blockIdx.x / p.cluster, rank = blockIdx.x - item * p.cluster;
  const int bhk = item / p.k_tiles;
  const int kt = item - bhk * p.k_tiles;
  const int g_count = p.G / p.cluster, g_first = rank * g_count;
  const int b = bhk / p.Hk, hk = bhk - b * p.Hk;
  const int bm = p.Bm > 1 ? b : 0;
  const int key0 = kt * kTile;
  const int4* table = p.table ? p.table + static_cast<long long>(bm) * p.q_tiles : nullptr;
  auto sees = [&](const int4& t) { return t.x < t.y && t.x < key0 + kTile && t.y > key0; };

  if (tid == 0) {
    mbar_init(&ss.kv_full, 1);
    for (int i = 0; i < S::kQ; ++i) {
      mbar_init(&ss.q_full[i], 1);
      mbar_init(&ss.q_empty[i], 1);
    }
    for (int i = 0; i < S::kG; ++i) {
      mbar_init(&ss.g_full[i], 1);
      mbar_init(&ss.g_empty[i], 1);
    }
    mbar_init(&ss.fix, 1);
    mbar_init(&ss.s_full, 1);
    mbar_init(&ss.dp_full, 1);
    mbar_init(&ss.p_full, 8);
    mbar_init(&ss.ds_full, 8);
    mbar_init(&ss.done, 1);
    mbar_init(&ss.drain, 1);
    ss.abort_flag = 0;
    ss.first = table ? INT_MAX : 0;
    ss.last = table ? -1 : p.q_tiles - 1;
    ss.most[0] = ss.most[1] = -126;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(&ss.tmem, 512);
    tmem_relinquish();
  }
  __syncthreads();
  if (table) {  // first and last query tile that sees a key of this tile
    int lo = INT_MAX, hi = -1;
    for (int i = tid; i < p.q_tiles; i += kBwdThreads)
      if (sees(table[i])) {
        lo = min(lo, i);
        hi = i;
      }
    if (hi >= 0) {
      atomicMin(&ss.first, lo);
      atomicMax(&ss.last, hi);
    }
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem = ss.tmem;
  const int first = ss.first, last = ss.last;
  const bool some = first <= last;
  if constexpr (!kBF16) {
    if (some) {
      const int runs = 8 * (last - first + 1);
      const int* from = p.up + static_cast<long long>(p.heads) * p.Sq_pad +
                        (static_cast<long long>(b) * p.H + hk * p.G + g_first) * (p.Sq_pad / 16) + 8 * first;
      int mg = -126, md = -126;
      for (int g = 0; g < g_count; ++g)
        for (int i = tid; i < runs; i += kBwdThreads) {
          const int m = from[g * static_cast<long long>(p.Sq_pad / 16) + i];
          mg = max(mg, most_g(m));
          md = max(md, most_d(m));
        }
      atomicMax(&ss.most[0], mg);
      atomicMax(&ss.most[1], md);
    }
    __syncthreads();
  }
  const bool fine = some && static_cast<long long>(g_count) * (last - first + 1) <= kFineSteps;
  volatile int* abort_flag = &ss.abort_flag;
  int* err = &g_dense_bwd_err;
  // every role walks the same tiles: `step(g, i, tab)` returns false to stop
  auto walk = [&](auto&& step) {
    for (int g = g_first; g < g_first + g_count; ++g)
      for (int i = first; i <= last; ++i) {
        const int4 t = table ? __ldg(table + i) : make_int4(0, p.Sk, 0, p.Sk);
        if (!sees(t)) continue;
        if (!step(g, i, t)) return false;
      }
    return true;
  };

  if (warp == 9) {
    // ------------------------------------------------------------------ loads
    if (some) {
      if (elect_one()) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_g);
        mbar_arrive_expect_tx(&ss.kv_full, 2 * kBytes);
        load_tile<DP>(sK, &tm_k, &ss.kv_full, key0, hk, b);
        load_tile<DP>(sV, &tm_v, &ss.kv_full, key0, hk, b);
      }
      Ring<S::kQ> rq;
      Ring<S::kG> rg;
      int nq = 0, ng = 0, fixes = 0;
      bool fixing = false;
      walk([&](int g, int i, const int4& t) {
        const int h = hk * p.G + g;
        bool w = true;
        if (nq >= S::kQ) w = bar_wait(&ss.q_empty[rq.slot], rq.phase ^ 1u, abort_flag, err, 401);
        if (!__all_sync(0xffffffffu, w)) return false;
        const bool fix = t.w <= 0;  // rows without keys, whose q and do may hold anything
        uint8_t* q = sQ + rq.slot * kBytes;
        const uint32_t extra = 2 * kTile * sizeof(float) + (p.rng ? kTile * sizeof(int2) : 0);
        if (elect_one()) {
          uint64_t* bar = fix ? &ss.fix : &ss.q_full[rq.slot];
          mbar_arrive_expect_tx(bar, kBytes + extra);
          load_tile<DP>(q, &tm_q, bar, i * kTile, h, b);
          const long long at = (static_cast<long long>(b) * p.H + h) * p.Sq_pad + i * kTile;
          bulk_load(ss.lse2[rq.slot], p.lse2 + at, kTile * sizeof(float), bar);
          bulk_load(ss.delta[rq.slot], p.delta + at, kTile * sizeof(float), bar);
          if (p.rng)
            bulk_load(ss.rng[rq.slot], p.rng + static_cast<long long>(bm) * p.Sq_pad + i * kTile, kTile * sizeof(int2),
                      bar);
        }
        if (fix) {
          __syncwarp();
          w = bar_wait(&ss.fix, static_cast<uint32_t>(fixes & 1), abort_flag, err, 402);
          fixing = !__all_sync(0xffffffffu, w);
          if (fixing) return false;
          ++fixes;
          for (int r = 0; r < kTile; ++r)
            if (ss.rng[rq.slot][r].x >= ss.rng[rq.slot][r].y) zero_row<DP>(q, r, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ss.q_full[rq.slot]);
        }
        ++nq;
        if (ng >= S::kG) w = bar_wait(&ss.g_empty[rg.slot], rg.phase ^ 1u, abort_flag, err, 403);
        if (!__all_sync(0xffffffffu, w)) return false;
        uint8_t* go = sG + rg.slot * kBytes;
        if (elect_one()) {
          uint64_t* bar = fix ? &ss.fix : &ss.g_full[rg.slot];
          mbar_arrive_expect_tx(bar, kBytes);
          load_tile<DP>(go, &tm_g, bar, i * kTile, h, b);
        }
        if (fix) {
          __syncwarp();
          w = bar_wait(&ss.fix, static_cast<uint32_t>(fixes & 1), abort_flag, err, 404);
          fixing = !__all_sync(0xffffffffu, w);
          if (fixing) return false;
          ++fixes;
          for (int r = 0; r < kTile; ++r)
            if (ss.rng[rq.slot][r].x >= ss.rng[rq.slot][r].y) zero_row<DP>(go, r, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ss.g_full[rg.slot]);
        }
        ++ng;
        rq.next();
        rg.next();
        return true;
      });
      if (lane == 0) {
        drain(&ss.kv_full, 0);
        drain_ring(ss.q_full, S::kQ, nq);
        drain_ring(ss.g_full, S::kG, ng);
        if (fixing) drain(&ss.fix, static_cast<uint32_t>(fixes & 1));
      }
    }
    __syncwarp();
  } else if (warp == 8) {
    // ------------------------------------------------------------------ products
    if (some && elect_one()) {
      constexpr uint32_t kIdS = idesc_f16(128, 128, kBF16 ? 1 : 0, 0, 0);
      constexpr uint32_t kIdR = idesc_f16(128, DP, kBF16 ? 1 : 0, 0, 1);
      const uint32_t kb = smem_u32(sK), vb = smem_u32(sV), qb = smem_u32(sQ), gb = smem_u32(sG);
      Ring<S::kQ> rq;
      Ring<S::kG> rg;
      int n = 0;
      int q_prev = 0;
      // dK of the step before: its dS, then the step's own dP
      auto finish = [&](int m) {
        if (!bar_wait(&ss.ds_full, static_cast<uint32_t>(m & 1), abort_flag, err, 411)) return false;
        tc_fence_after();
        mma_rows(tmem + kColD, tmem + kColB, qb + q_prev * kBytes, kIdR, m > 0);
        if (fine) mma_rows(tmem + kColD, tmem + kColB + 32, qb + q_prev * kBytes, kIdR, true);
        umma_commit(&ss.q_empty[q_prev]);
        return true;
      };
      bool ok = bar_wait(&ss.kv_full, 0, abort_flag, err, 412);
      int g_prev = 0;
      if (ok)
        ok = walk([&](int, int, const int4&) {
          if (n > 0) {  // dV(n - 1)
            if (!bar_wait(&ss.p_full, static_cast<uint32_t>((n - 1) & 1), abort_flag, err, 413)) return false;
            tc_fence_after();
            mma_rows(tmem + kColC, tmem + kColA, gb + g_prev * kBytes, kIdR, n > 1);
            if (fine) mma_rows(tmem + kColC, tmem + kColA + 32, gb + g_prev * kBytes, kIdR, true);
            umma_commit(&ss.g_empty[g_prev]);
          }
          if (!bar_wait(&ss.q_full[rq.slot], rq.phase, abort_flag, err, 414)) return false;
          tc_fence_after();
          mma_scores<DP>(tmem + kColA, kb, qb + rq.slot * kBytes, kIdS);
          umma_commit(&ss.s_full);
          if (n > 0 && !finish(n - 1)) return false;
          if (!bar_wait(&ss.g_full[rg.slot], rg.phase, abort_flag, err, 415)) return false;
          tc_fence_after();
          mma_scores<DP>(tmem + kColB, vb, gb + rg.slot * kBytes, kIdS);
          umma_commit(&ss.dp_full);
          q_prev = rq.slot;
          g_prev = rg.slot;
          rq.next();
          rg.next();
          ++n;
          return true;
        });
      if (ok) ok = bar_wait(&ss.p_full, static_cast<uint32_t>((n - 1) & 1), abort_flag, err, 416);
      if (ok) {
        tc_fence_after();
        mma_rows(tmem + kColC, tmem + kColA, gb + g_prev * kBytes, kIdR, n > 1);
        if (fine) mma_rows(tmem + kColC, tmem + kColA + 32, gb + g_prev * kBytes, kIdR, true);
        ok = finish(n - 1);
      }
      if (ok) umma_commit(&ss.done);
      umma_commit(&ss.drain);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&ss.drain, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ p and ds
    const int half = warp >> 2;
    const uint32_t la = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const int key = key0 + 32 * (warp & 3) + lane;
    bool ok = true;
    int up = kUp;  // what ds is raised by (log2), and by which factor over p's
    float raise = 1.f;
    if constexpr (!kBF16) {
      if (some) {
        ok = bar_wait(&ss.kv_full, 0, abort_flag, err, 425);
        ok = __all_sync(0xffffffffu, ok);
        float n2 = 0.f;
#pragma unroll 4
        for (int c = 0; c < DP / 8; ++c) {
          const uint4 u = *reinterpret_cast<const uint4*>(
              sV + (c >> 3) * kHalfBytes + sw128_offset(static_cast<uint32_t>(32 * (warp & 3) + lane), c & 7));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x0, x1;
            unpack16<false>(w[e], x0, x1);
            n2 = fmaf(x0, x0, fmaf(x1, x1, n2));
          }
        }
        up = min(kUp, kBelow - max(ss.most[0] + log2_above_root(n2), ss.most[1]));
        raise = __uint_as_float(static_cast<uint32_t>(127 + up - kUp) << 23);
      }
    }
    if (some && ok) {
      Ring<S::kQ> rq;
      int n = 0;
      ok = walk([&](int, int, const int4& t) {
        bool w = bar_wait(&ss.q_full[rq.slot], rq.phase, abort_flag, err, 421);  // the tile's statistics
        w = w && bar_wait(&ss.s_full, static_cast<uint32_t>(n & 1), abort_flag, err, 422);
        if (!__all_sync(0xffffffffu, w)) return false;
        tc_fence_after();
        uint32_t r[64];
        tmem_read32(la + kColA + 64 * half, r);
        tmem_read32(la + kColA + 64 * half + 32, r + 32);
        // p = 2^(z - lse), in pairs of 16 bits for the product and as r = p (1 - tanh^2) for ds.  The queries' statistics
        // come four to a load: what a load returns to 32 lanes passes the same port as the tiles.
        const float4* ls = reinterpret_cast<const float4*>(ss.lse2[rq.slot] + 64 * half);
        const bool border = table && (t.z > key0 || t.w < key0 + kTile);
        uint32_t seen[2] = {0xffffffffu, 0xffffffffu};  // one bit for each of the thread's 64 queries
        if (border) {
          const int4* rg = reinterpret_cast<const int4*>(ss.rng[rq.slot] + 64 * half);
          seen[0] = seen[1] = 0u;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int4 b2 = rg[e];
            if (key >= b2.x && key < b2.y) seen[e >> 4] |= 1u << (2 * (e & 15));
            if (key >= b2.z && key < b2.w) seen[e >> 4] |= 2u << (2 * (e & 15));
          }
          // what a masked place holds must not choose the form of tanh, nor reach anything else
          if constexpr (kCap) put_masked(r, seen, 0u);
        }
        bool far = false;  // scores beyond the cap's polynomials
        if constexpr (kCap) far = !capped_near<64>(r, p.cap);
        uint32_t pk[32];
        auto weights = [&](auto split, auto far) {
          uint32_t lo[32];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float4 l4 = ls[e];
            const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
            float x[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float s = __uint_as_float(r[4 * e + c]);
              if constexpr (far.value) {
                float slope;
                x[c] = ex2_approx(capped_of(s, p.cap, slope) - lv[c]);
                r[4 * e + c] = __float_as_uint(x[c] * slope);
              } else {
                x[c] = ex2_approx(kCap ? s - lv[c] : fmaf(s, p.scale_log2, -lv[c]));
                const float u = s * p.cap_inv;  // tanh, at most tanh(1) in size
                r[4 * e + c] = __float_as_uint(kCap ? x[c] * fmaf(-u, u, 1.f) : x[c]);
              }
            }
            pk[2 * e] = pack16<kBF16>(x[0], x[1]);
            pk[2 * e + 1] = pack16<kBF16>(x[2], x[3]);
            if constexpr (split.value) {
              lo[2 * e] = rest16<kBF16>(pk[2 * e], x[0], x[1]);
              lo[2 * e + 1] = rest16<kBF16>(pk[2 * e + 1], x[2], x[3]);
            }
          }
          if constexpr (split.value) tmem_st32(la + kColA + 64 * half + 32, lo);
        };
        if (kCap && far) [[unlikely]] {
          capped_rest<64>(r, p.cap);
          if (border) put_masked(r, seen, __float_as_uint(p.cap_mask_rest));
          weights(std::true_type(), std::bool_constant<kCap>());  // what is left over is used where `fine`
        } else {
          if (border) put_masked(r, seen, __float_as_uint(kCap ? p.cap_mask : -INFINITY));
          if (fine) weights(std::true_type(), std::false_type()); else weights(std::false_type(), std::false_type());
        }
        tmem_st32(la + kColA + 64 * half, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ss.p_full);
        w = bar_wait(&ss.dp_full, static_cast<uint32_t>(n & 1), abort_flag, err, 423);
        if (!__all_sync(0xffffffffu, w)) return false;
        tc_fence_after();
        const float4* dl = reinterpret_cast<const float4*>(ss.delta[rq.slot] + 64 * half);
        auto slopes = [&](auto split) {
          uint32_t lo[32];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t g[32];
            tmem_read32(la + kColB + 64 * half + 32 * c, g);
            if (border) {  // 0 * NaN
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (__uint_as_float(r[32 * c + e]) == 0.f) g[e] = 0u;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 d4 = dl[8 * c + e];
              const float dv[4] = {d4.x, d4.y, d4.z, d4.w};
              float x[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                float f = __uint_as_float(r[32 * c + 4 * e + y]);
                if constexpr (!kBF16) f *= raise;
                x[y] = f * (__uint_as_float(g[4 * e + y]) - dv[y]);
              }
              const int at = 16 * c + 2 * e;
              pk[at] = pack16<kBF16>(x[0], x[1]);
              pk[at + 1] = pack16<kBF16>(x[2], x[3]);
              if constexpr (split.value) {
                lo[at] = rest16<kBF16>(pk[at], x[0], x[1]);
                lo[at + 1] = rest16<kBF16>(pk[at + 1], x[2], x[3]);
              }
            }
          }
          if constexpr (split.value) tmem_st32(la + kColB + 64 * half + 32, lo);
        };
        if (fine) slopes(std::true_type()); else slopes(std::false_type());
        tmem_st32(la + kColB + 64 * half, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ss.ds_full);
        rq.next();
        ++n;
        return true;
      });
      if (ok) {
        ok = bar_wait(&ss.done, 0, abort_flag, err, 424);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
    }
    // what p and ds were raised by
    const float lower_p = kBF16 ? 1.f : __uint_as_float((127u - kUp) << 23);
    const float lower_ds = kBF16 ? 1.f : __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
    if (p.cluster > 1) {  // this CTA's sums to shared memory: its tiles are done with
      to_shared<DP>(la + kColD, half, 32 * (warp & 3) + lane, lower_ds, smem, ok && some);
      to_shared<DP>(la + kColC, half, 32 * (warp & 3) + lane, lower_p, smem + kTile * DP * 4, ok && some);
    } else if (ok) {
      const bool live = key < p.Sk;
      const long long ok0 = b * p.d0.sb + hk * p.d0.sh + static_cast<long long>(key) * p.d0.ss;
      const long long ov0 = b * p.d1.sb + hk * p.d1.sh + static_cast<long long>(key) * p.d1.ss;
      store_acc<DP, kBF16>(la + kColD, half * (DP / 2), p.sm_scale * lower_ds, p.d0.p, ok0, p.D, live, some);
      store_acc<DP, kBF16>(la + kColC, half * (DP / 2), lower_p, p.d1.p, ov0, p.D, live, some);
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
  if (p.cluster > 1) {
    // The CTAs of a cluster took a part of the query heads each.  Each now adds up a share of the columns, in the order of
    // the CTAs, from everybody's shared memory.
    cluster_sync();
    constexpr int kEights = DP / 8;  // runs of 8 columns of dk, then of dv
    for (int t = tid; t < 2 * kEights * kTile; t += kBwdThreads) {
      const int run = t / kTile, row = t - run * kTile;
      if (run % p.cluster != rank) continue;
      const int which = run / kEights, d = 8 * (run - which * kEights);
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const uint32_t at = smem_u32(smem) + which * kTile * DP * 4 + ((d >> 2) * kTile + row) * 16;
      for (int c = 0; c < p.cluster; ++c) {
        const float4 a = load_peer(at, c), e = load_peer(at + kTile * 16, c);
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += e.x; v[5] += e.y; v[6] += e.z; v[7] += e.w;
      }
      if (key0 + row >= p.Sk || d >= p.D) continue;
      const Tensor4& o = which ? p.d1 : p.d0;
      const float f = which ? 1.f : p.sm_scale;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= f;
      store8<kBF16>(o.p, b * o.sb + hk * o.sh + static_cast<long long>(key0 + row) * o.ss + d, v);
    }
    cluster_sync();  // nobody leaves while its sums are read
  }
}

// ------------------------------------------------------------------------- dq
template <int DP>
struct DqSmem {
  static constexpr int kK = DP == 128 ? 3 : 5;
  static constexpr int kV = DP == 128 ? 2 : 4;
  static constexpr int kTiles = (2 + kK + kV) * tile_bytes<DP>();
  uint64_t qg_full;
  uint64_t k_full[kK], k_empty[kK], v_full[kV], v_empty[kV];
  uint64_t fix;
  uint64_t s_full, s_read;
  uint64_t dp_full[2], ds_full[2];  // of step n in [n % 2]: the arithmetic may be a step ahead of who issues the products
  uint64_t done, drain;
  uint32_t tmem;
  int abort_flag;
};
template <int DP>
constexpr int dq_smem_bytes() { return DqSmem<DP>::kTiles + static_cast<int>(sizeof(DqSmem<DP>)) + 1024; }

template <int DP, bool kBF16, bool kCap>
__global__ void __launch_bounds__(kBwdThreads, 1)
    dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
              const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_g, const BwdParams p) {
  using S = DqSmem<DP>;
  constexpr int kBytes = tile_bytes<DP>();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sQ = smem, *sG = smem + kBytes, *sK = smem + 2 * kBytes, *sV = sK + S::kK * kBytes;
  S& ss = *reinterpret_cast<S*>(smem + S::kTiles);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // the last query tiles first: under a causal mask they see the most keys
  const int bh = blockIdx.x / p.q_tiles;
  const int qt = p.q_tiles - 1 - (blockIdx.x - bh * p.q_tiles);
  const int b = bh / p.H, h = bh - b * p.H;
  const int hk = h / p.G;
  const int bm = p.Bm > 1 ? b : 0;
  const int4 tab = p.table ? p.table[static_cast<long long>(bm) * p.q_tiles + qt] : make_int4(0, p.Sk, 0, p.Sk);
  const int n0 = tab.x < tab.y ? tab.x / kTile : 0;
  const int n1 = tab.x < tab.y ? (tab.y + kTile - 1) / kTile : 0;
  const int steps = n1 - n0;
  const bool fine = steps <= kFineSteps;

  if (tid == 0) {
    mbar_init(&ss.qg_full, 1);
    for (int i = 0; i < S::kK; ++i) {
      mbar_init(&ss.k_full[i], 1);
      mbar_init(&ss.k_empty[i], 1);
    }
    for (int i = 0; i < S::kV; ++i) {
      mbar_init(&ss.v_full[i], 1);
      mbar_init(&ss.v_empty[i], 1);
    }
    mbar_init(&ss.fix, 1);
    mbar_init(&ss.s_full, 1);
    mbar_init(&ss.s_read, 8);
    mbar_init(&ss.dp_full[0], 1);
    mbar_init(&ss.dp_full[1], 1);
    mbar_init(&ss.ds_full[0], 8);
    mbar_init(&ss.ds_full[1], 8);
    mbar_init(&ss.done, 1);
    mbar_init(&ss.drain, 1);
    ss.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(&ss.tmem, 512);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ss.tmem;
  volatile int* abort_flag = &ss.abort_flag;
  int* err = &g_dense_bwd_err;

  if (warp == 9) {
    // ------------------------------------------------------------------ loads
    if (steps > 0) {
      if (elect_one()) {
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        mbar_arrive_expect_tx(&ss.qg_full, 2 * kBytes);
        load_tile<DP>(sQ, &tm_q, &ss.qg_full, qt * kTile, h, b);
        load_tile<DP>(sG, &tm_g, &ss.qg_full, qt * kTile, h, b);
      }
      Ring<S::kK> rk;
      Ring<S::kV> rv;
      int nk = 0, nv = 0, fixes = 0;
      bool ok = true, fixing = false;
      for (int n = 0; n < steps; ++n) {
        if (n >= S::kK) ok = bar_wait(&ss.k_empty[rk.slot], rk.phase ^ 1u, abort_flag, err, 451);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int row = (n0 + n) * kTile;
        uint8_t* dst = sK + rk.slot * kBytes;
        const bool fix = row < tab.x || min(row + kTile, p.Sk) > tab.y;  // keys of the tile that no row sees
        if (elect_one()) {
          uint64_t* bar = fix ? &ss.fix : &ss.k_full[rk.slot];
          mbar_arrive_expect_tx(bar, kBytes);
          load_tile<DP>(dst, &tm_k, bar, row, hk, b);
        }
        if (fix) {
          __syncwarp();
          ok = bar_wait(&ss.fix, static_cast<uint32_t>(fixes & 1), abort_flag, err, 452);
          ok = __all_sync(0xffffffffu, ok);
          fixing = !ok;
          if (!ok) break;
          ++fixes;
          for (int r = 0; r < kTile; ++r)
            if (row + r < tab.x || row + r >= tab.y) zero_row<DP>(dst, r, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ss.k_full[rk.slot]);
        }
        ++nk;
        if (n >= S::kV) ok = bar_wait(&ss.v_empty[rv.slot], rv.phase ^ 1u, abort_flag, err, 453);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&ss.v_full[rv.slot], kBytes);
          load_tile<DP>(sV + rv.slot * kBytes, &tm_v, &ss.v_full[rv.slot], row, hk, b);
        }
        ++nv;
        rk.next();
        rv.next();
      }
      if (lane == 0) {
        drain(&ss.qg_full, 0);
        drain_ring(ss.k_full, S::kK, nk);
        drain_ring(ss.v_full, S::kV, nv);
        if (fixing) drain(&ss.fix, static_cast<uint32_t>(fixes & 1));
      }
    }
    __syncwarp();
  } else if (warp == 8) {
    // ------------------------------------------------------------------ products
    if (steps > 0 && elect_one()) {
      constexpr uint32_t kIdS = idesc_f16(128, 128, kBF16 ? 1 : 0, 0, 0);
      constexpr uint32_t kIdR = idesc_f16(128, DP, kBF16 ? 1 : 0, 0, 1);
      const uint32_t qb = smem_u32(sQ), gb = smem_u32(sG), kb = smem_u32(sK), vb = smem_u32(sV);
      Ring<S::kK> rk;
      Ring<S::kV> rv;
      auto scores = [&](int n) {  // S(n) and dP(n)
        if (!bar_wait(&ss.k_full[rk.slot], rk.phase, abort_flag, err, 461)) return false;
        tc_fence_after();
        mma_scores<DP>(tmem + kColA, qb, kb + rk.slot * kBytes, kIdS);
        umma_commit(&ss.s_full);
        if (!bar_wait(&ss.v_full[rv.slot], rv.phase, abort_flag, err, 462)) return false;
        tc_fence_after();
        mma_scores<DP>(tmem + ((n & 1) ? kColC : kColB), gb, vb + rv.slot * kBytes, kIdS);
        umma_commit(&ss.dp_full[n & 1]);
        umma_commit(&ss.v_empty[rv.slot]);
        rk.next();
        rv.next();
        return true;
      };
      bool ok = bar_wait(&ss.qg_full, 0, abort_flag, err, 463) && scores(0);
      int k_used = 0;
      for (int n = 0; n < steps && ok; ++n) {
        if (n + 1 < steps) {
          ok = bar_wait(&ss.s_read, static_cast<uint32_t>(n & 1), abort_flag, err, 464);
          if (!ok) break;
          tc_fence_after();
          ok = scores(n + 1);
          if (!ok) break;
        }
        ok = bar_wait(&ss.ds_full[n & 1], static_cast<uint32_t>((n >> 1) & 1), abort_flag, err, 465);
        if (!ok) break;
        tc_fence_after();
        mma_rows(tmem + kColD, tmem + ((n & 1) ? kColC : kColB), kb + k_used * kBytes, kIdR, n > 0);
        if (fine) mma_rows(tmem + kColD, tmem + ((n & 1) ? kColC : kColB) + 32, kb + k_used * kBytes, kIdR, true);
        umma_commit(&ss.k_empty[k_used]);
        if (++k_used == S::kK) k_used = 0;
      }
      if (ok) umma_commit(&ss.done);
      umma_commit(&ss.drain);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&ss.drain, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ ds
    const int half = warp >> 2;
    const uint32_t la = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const int row = qt * kTile + 32 * (warp & 3) + lane;
    const bool live = row < p.Sq;
    bool ok = true;
    float lower = 1.f;
    if (steps > 0) {
      float lse2 = p.lse2[static_cast<long long>(bh) * p.Sq_pad + row];
      const float delta = p.delta[static_cast<long long>(bh) * p.Sq_pad + row];
      if constexpr (!kBF16) {  // p raised by 2^kUp there; here p, and so ds, by what the row allows
        const int* bins = p.v_up + (static_cast<long long>(b) * p.Hk + hk) * kBins;
        int above = -126;
        for (int i = tab.x / p.v_bin + lane; i <= (tab.y - 1) / p.v_bin; i += 32) above = max(above, bins[i]);
        above = __reduce_max_sync(0xffffffffu, above);
        const int n = min(kUp, kBelow - max(p.up[static_cast<long long>(bh) * p.Sq_pad + row] + above, log2_above(delta)));
        lse2 += static_cast<float>(kUp - n);
        lower = __uint_as_float(static_cast<uint32_t>(127 - n) << 23);
      }
      int lo = 0, hi = live ? p.Sk : 0;  // rows behind the last see nothing, and choose nothing
      if (p.ranges && live) {
        const int2 r = p.ranges[static_cast<long long>(bm) * p.Sq + row];
        lo = r.x;
        hi = r.y;
      }
      const uint32_t len = static_cast<uint32_t>(hi - lo);
      for (int n = 0; n < steps; ++n) {
        ok = bar_wait(&ss.s_full, static_cast<uint32_t>(n & 1), abort_flag, err, 471);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t r[64];
        tmem_read32(la + kColA + 64 * half, r);
        tmem_read32(la + kColA + 64 * half + 32, r + 32);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ss.s_read);
        const int key0 = (n0 + n) * kTile;
        const bool border = key0 < tab.z || key0 + kTile > tab.w;
        const uint32_t d = static_cast<uint32_t>(key0 + 64 * half - lo);
        auto mask = [&](float v) {
          if (border) {
#pragma unroll
            for (int e = 0; e < 64; ++e)
              if (d + e >= len) r[e] = __float_as_uint(v);
          }
        };
        bool far = false;  // scores beyond the cap's polynomials
        if constexpr (kCap) {
          mask(0.f);  // what a masked place holds must not choose the form of tanh
          far = !capped_near<64>(r, p.cap);
        }
        if (kCap && far) [[unlikely]] {
          capped_rest<64>(r, p.cap);
          mask(p.cap_mask_rest);
#pragma unroll
          for (int e = 0; e < 64; ++e) {
            float slope;
            const float x = ex2_approx(capped_of(__uint_as_float(r[e]), p.cap, slope) - lse2);
            r[e] = __float_as_uint(x * slope);
          }
        } else {
          mask(kCap ? p.cap_mask : -INFINITY);
#pragma unroll
          for (int e = 0; e < 64; ++e) {
            const float s = __uint_as_float(r[e]);
            const float x = ex2_approx(kCap ? s - lse2 : fmaf(s, p.scale_log2, -lse2));
            const float u = s * p.cap_inv;  // tanh, at most tanh(1) in size
            r[e] = __float_as_uint(kCap ? x * fmaf(-u, u, 1.f) : x);
          }
        }
        const uint32_t col = (n & 1) ? kColC : kColB;
        ok = bar_wait(&ss.dp_full[n & 1], static_cast<uint32_t>((n >> 1) & 1), abort_flag, err, 472);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t pk[32];
        auto slopes = [&](auto split) {
          uint32_t lo[32];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t g[32];
            tmem_read32(la + col + 64 * half + 32 * c, g);
            if (border) {  // 0 * NaN
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (__uint_as_float(r[32 * c + e]) == 0.f) g[e] = 0u;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float x0 = __uint_as_float(r[32 * c + 2 * e]) * (__uint_as_float(g[2 * e]) - delta);
              const float x1 = __uint_as_float(r[32 * c + 2 * e + 1]) * (__uint_as_float(g[2 * e + 1]) - delta);
              pk[16 * c + e] = pack16<kBF16>(x0, x1);
              if constexpr (split.value) lo[16 * c + e] = rest16<kBF16>(pk[16 * c + e], x0, x1);
            }
          }
          if constexpr (split.value) tmem_st32(la + col + 64 * half + 32, lo);
        };
        if (fine) slopes(std::true_type()); else slopes(std::false_type());
        tmem_st32(la + col + 64 * half, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ss.ds_full[n & 1]);
      }
      if (ok) {
        ok = bar_wait(&ss.done, 0, abort_flag, err, 473);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
    }
    if (ok) {
      const bool empty = p.ranges && live && [&] {
        const int2 r = p.ranges[static_cast<long long>(bm) * p.Sq + row];
        return r.x >= r.y;
      }();
      const long long off = b * p.d0.sb + h * p.d0.sh + static_cast<long long>(row) * p.d0.ss;
      store_acc<DP, kBF16>(la + kColD, half * (DP / 2), p.sm_scale * lower, p.d0.p, off, p.D, live && !empty,
                           steps > 0);
      if (live && empty) {
        const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int d0 = half * (DP / 2); d0 < min(p.D, (half + 1) * (DP / 2)); d0 += 8)
          store8<kBF16>(p.d0.p, off + d0, z);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

template <int DP, bool kBF16, bool kCap>
int launch_bwd(const CUtensorMap* m, BwdParams p, const DenseArgs& a, cudaStream_t stream) {
  auto* kv = dkv_kernel<DP, kBF16, kCap>;
  auto* qk = dq_kernel<DP, kBF16, kCap>;
  if (cudaFuncSetAttribute(kv, cudaFuncAttributeMaxDynamicSharedMemorySize, dkv_smem_bytes<DP>()) != cudaSuccess ||
      cudaFuncSetAttribute(qk, cudaFuncAttributeMaxDynamicSharedMemorySize, dq_smem_bytes<DP>()) != cudaSuccess)
    return BSA_ERR_CUDA;
  if (a.dk.p) {
    p.d0 = a.dk;
    p.d1 = a.dv;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.B * a.Hk * p.k_tiles * p.cluster);
    cfg.blockDim = dim3(kBwdThreads);
    cfg.dynamicSmemBytes = dkv_smem_bytes<DP>();
    cfg.stream = stream;
    cfg.attrs = at;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kv, m[0], m[1], m[2], m[3], p) != cudaSuccess) return BSA_ERR_CUDA;
  }
  if (!a.dq.p) return BSA_OK;
  p.d0 = a.dq;
  qk<<<a.B * a.H * p.q_tiles, kBwdThreads, dq_smem_bytes<DP>(), stream>>>(m[0], m[1], m[2], m[3], p);
  return cudaGetLastError() == cudaSuccess ? BSA_OK : BSA_ERR_CUDA;
}

}  // namespace dense

long long dense_backward_stats_bytes(int B, int H, int Sq, int Bm) {
  const long long rows = (static_cast<long long>(Sq) + dense::kTile - 1) / dense::kTile * dense::kTile;
  const long long heads = static_cast<long long>(B) * H;
  return (3 * heads + 2ll * Bm) * rows * 4 + heads * (rows / 16) * 4 + heads * dense::kBins * 4;
}

int launch_dense_backward(const DenseArgs& a, int sms, cudaStream_t stream) {
  using namespace dense;
  CUtensorMap m[4];
  int rc;
  if ((rc = make_map4(&m[0], a.q, a.dtype, a.B, a.H, a.Sq, a.D, "q"))) return rc;
  if ((rc = make_map4(&m[1], a.k, a.dtype, a.B, a.Hk, a.Sk, a.D, "k"))) return rc;
  if ((rc = make_map4(&m[2], a.v, a.dtype, a.B, a.Hk, a.Sk, a.D, "v"))) return rc;
  if ((rc = make_map4(&m[3], a.g, a.dtype, a.B, a.H, a.Sq, a.D, "gradient of out"))) return rc;
  BwdParams p = {};
  p.ranges = a.ranges; p.table = a.table; p.Bm = a.Bm;
  p.H = a.H; p.Hk = a.Hk; p.G = a.H / a.Hk; p.Sq = a.Sq; p.Sk = a.Sk; p.D = a.D;
  p.q_tiles = (a.Sq + kTile - 1) / kTile;
  p.k_tiles = (a.Sk + kTile - 1) / kTile;
  p.Sq_pad = p.q_tiles * kTile;
  // Key tiles alone may be few and uneven (4,680 rows of 9 documents, 4 key heads: 148 tiles that see 8 to 44 query
  // tiles): then the query heads of a key head are shared among the CTAs of a cluster, 8 at most.
  p.cluster = 1;
  if (static_cast<long long>(a.B) * a.Hk * p.k_tiles < 4ll * sms)
    for (int c = 2; c <= 8; ++c)
      if (p.G % c == 0) p.cluster = c;
  p.scale_log2 = a.sm_scale * 1.4426950408889634f;
  p.sm_scale = a.sm_scale;
  if (a.softcap > 0.f) {
    p.cap = make_cap(p.scale_log2, a.softcap);
    p.cap_inv = 1.f / p.cap.log2;
    p.cap_mask = -p.cap.log2 - 300.f;
    p.cap_mask_rest = 4.f + 300.f * p.cap_inv;
  }
  p.lse2 = a.stats;
  p.delta = a.stats + static_cast<long long>(a.B) * a.H * p.Sq_pad;
  p.rng = a.ranges ? reinterpret_cast<int2*>(a.stats + 2 * static_cast<long long>(a.B) * a.H * p.Sq_pad) : nullptr;
  p.heads = a.B * a.H;
  p.up = reinterpret_cast<int*>(a.stats + (2ll * p.heads + (a.ranges ? 2ll * a.Bm : 0)) * p.Sq_pad);
  p.v_up = p.up + static_cast<long long>(p.heads) * (p.Sq_pad + p.Sq_pad / 16);
  p.v_bin = 64 * ((a.Sk + 64 * kBins - 1) / (64 * kBins));
  p.v_bins = a.dq.p ? (a.Sk + p.v_bin - 1) / p.v_bin : 0;  // only dq reads them
  p.v = a.v;
  p.lse = a.lse;
  p.o = a.o;
  p.o_lo = a.o_lo;
  p.g = a.g;
  if (static_cast<long long>(a.B) * a.H * p.q_tiles > INT_MAX || static_cast<long long>(a.B) * a.Hk * p.k_tiles > INT_MAX / 8)
    return set_error(BSA_ERR_SHAPE, "too many row tiles for one launch");
  const bool bf = a.dtype == BSA_DTYPE_BF16, cap = a.softcap > 0.f;
  const int runs = p.Sq_pad / 16;
  const dim3 sgrid(bf || runs > p.v_bins ? runs : p.v_bins, p.heads < 65535 ? p.heads : 65535);
  if (bf) stats_kernel<__nv_bfloat16><<<sgrid, 256, 0, stream>>>(p);
  else stats_kernel<__half><<<sgrid, 256, 0, stream>>>(p);
  rc = cudaGetLastError() == cudaSuccess ? BSA_OK : BSA_ERR_CUDA;
  if (!rc) {
    if (a.D > 64)
      rc = bf ? (cap ? launch_bwd<128, true, true>(m, p, a, stream) : launch_bwd<128, true, false>(m, p, a, stream))
              : (cap ? launch_bwd<128, false, true>(m, p, a, stream) : launch_bwd<128, false, false>(m, p, a, stream));
    else
      rc = bf ? (cap ? launch_bwd<64, true, true>(m, p, a, stream) : launch_bwd<64, true, false>(m, p, a, stream))
              : (cap ? launch_bwd<64, false, true>(m, p, a, stream) : launch_bwd<64, false, false>(m, p, a, stream));
  }
  if (rc) return set_error(rc, "dense attention backward launch: %s", cudaGetErrorString(cudaGetLastError()));
  return BSA_OK;
}

int dense_bwd_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, dense::g_dense_bwd_err, sizeof(int)) != cudaSuccess) return BSA_ERR_CUDA;
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(dense::g_dense_bwd_err, &z, sizeof(int));
  }
  return v;
}

}  // namespace bsa
