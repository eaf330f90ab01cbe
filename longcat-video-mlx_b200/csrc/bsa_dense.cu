// Dense attention over key intervals, forward, on sm_100a (tcgen05 + TMA + TMEM).
//
//   z_ij = s_ij = sm_scale q_i . k_j, or cap tanh(s_ij / cap);   p_ij = 2^(z_ij log2(e) - m_i) for j in [lo_i, hi_i)
//   o_i = sum_j p_ij v_j / l_i,  l_i = sum_j p_ij,  lse_i = ln sum_j e^z_ij        (0 and -inf for an empty row)
//
// One pass over the keys with a running maximum and sum, scores and output accumulator in tensor memory.  A CTA takes one
// query tile of 128 rows of one head:
//     S(j)[128 x 128] = Q K_j^T        A = Q in tensor memory, B = K in shared memory
//     O[128 x D]     += P(j) V_j       A = P in tensor memory, B = V in shared memory
// TMEM: two S buffers and O of 128 columns each, Q and P of 64 (16-bit pairs).  With Q in tensor memory the operands of
// both products and the loads of K and V move 128 KB a step through shared memory, 160 KB with Q there too.  S(j+3)
// is issued when S(j+1) has been read, behind P(j) V, two steps before it is needed.
//
// Roles (320 threads, one CTA to an SM):
//   warps 0-7 : softmax, warps 0-3 on the keys 0-63 of a step, 4-7 on 64-127, a thread on half a row.  The two threads
//               of a row need one maximum only when one of them finds it exceeded (below), which a barrier with a vote
//               tells; their sums join at the end.  Of its 64 scores a thread reads the next step's first 32 before
//               it computes the exponentials of this step's last 32, so their maximum is found beside those
//   warp 8    : issues the products: P(j) V first, which the next step's P waits for, then S(j+3)
//   warp 9    : loads; one ring for K and V tiles in the order of their use
// The maximum is raised, and O and l rescaled, only when a score exceeds it by more than 2^8 (log2 8): P stays within
// fp16's range and rounding is relative, so the result is as exact as with the true maximum.  fp16's P is multiplied by 2^7
// (and so is l), up to 2^15: weights keep their bits down to 2^-21 of the largest and vanish below 2^-32, where 2^-25 without
// it would cost a row with a few heavy keys the sum of a long tail.
// P is rounded to the input type for the tensor cores, and o is divided by the sum of the rounded values: the weights
// then sum to 1 and their rounding errors count against v_j - o_i instead of v_j.  lse comes from the fp32 values.
//
// Masked places never reach a result: scores are replaced by -inf whatever they hold, and V rows in front of or behind
// all of the CTA's intervals are zeroed in shared memory (0 * NaN would be NaN).  Tiles there are not loaded; tiles
// inside all of the intervals are not compared.
//
// Measured: 20,280 rows x 8 heads, D 128, 6,240 of conditioning in front, 1.46 ms, 910 TFLOP/s of the visible pairs.
// The card is then at its power limit (SM clock 1.65 of 1.97 GHz), and without the loads of K and V, which a tile of 128
// rows makes for each step, it would take a tenth less.  Short calls are bound by their start: 2 us for one tile.
// Tried and not faster (1.49 to 1.60 ms): two query tiles to a CTA with 8 or 16 softmax warps, three S buffers, two
// issuing threads, half of the exponentials as polynomials.
// Every wait is bounded (bsa_ptx.cuh).
#include <climits>
#include "bsa_dense.cuh"

namespace bsa {
namespace dense {

__device__ int g_dense_err;

constexpr int kThreads = 320;
constexpr int kSoftmaxWarps = 8;
constexpr int kIssue = kSoftmaxWarps, kLoad = kSoftmaxWarps + 1;  // warps
constexpr float kRescale = 8.f;  // log2
template <bool kBF16>
constexpr float kRaise = kBF16 ? 0.f : 7.f;  // log2: of P
constexpr uint32_t kTmemCols = 512;
__host__ __device__ constexpr uint32_t col_s(int b) { return 128u * static_cast<uint32_t>(b); }
constexpr uint32_t kColO = 256, kColQ = 384, kColP = 448;
template <int DP>
struct Smem {
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr int kTiles = (1 + kStages) * tile_bytes<DP>();
  uint64_t q_full;
  uint64_t full[kStages], empty[kStages];
  uint64_t fix;
  uint64_t q_ready;              // Q copied into tensor memory
  uint64_t s_full[2], s_read[2];  // S(j) in buffer j % 2
  // of step j in [j % 2]; a waiter may be one step behind or ahead of the others, so one barrier each would not tell
  uint64_t p_full[2];  // P(j) written, O rescaled where it had to be (one arrival for each softmax warp)
  uint64_t o_full[2];  // P(j) V done
  uint64_t drain;
  uint32_t tmem;
  int abort_flag;
  float join[2][2][kTile];  // [half][maximum or sum, fp32 sum][row]
};
template <int DP>
constexpr int smem_bytes() { return Smem<DP>::kTiles + static_cast<int>(sizeof(Smem<DP>)) + 1024; }

struct Params {
  const int2* ranges;  // [Bm][Sq], null: all keys
  const int4* table;   // [Bm][q_tiles]
  int Bm, H, G, Sq, Sk, D;
  int q_tiles;         // tiles of 128 rows
  int heads;           // B * H
  int group;           // heads that run side by side
  int splits;          // CTAs along the keys
  float scale_log2;    // sm_scale log2(e)
  Cap cap;
  void* out;
  long long ob, oh, os;
  void* out_lo;        // nullable: [B, H, Sq, D] contiguous, o - out in 16 bits
  float* lse;
  float* part;         // splits > 1: [splits][rows][D] of o, then [splits][rows] of lse in log2
  long long rows;      // B * H * Sq
};

template <int DP, bool kBF16, bool kCap>
__global__ void __launch_bounds__(kThreads, 1)
    dense_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using S = Smem<DP>;
  constexpr int kStages = S::kStages;
  constexpr int kBytes = tile_bytes<DP>();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + kBytes;
  S& ss = *reinterpret_cast<S*>(smem + S::kTiles);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    mbar_init(&ss.q_full, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&ss.full[i], 1);
      mbar_init(&ss.empty[i], 1);
    }
    mbar_init(&ss.fix, 1);
    mbar_init(&ss.q_ready, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ss.s_full[i], 1);
      mbar_init(&ss.s_read[i], kSoftmaxWarps);
      mbar_init(&ss.p_full[i], kSoftmaxWarps);
      mbar_init(&ss.o_full[i], 1);
    }
    mbar_init(&ss.drain, 1);
    ss.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kIssue) {
    tmem_alloc(&ss.tmem, kTmemCols);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ss.tmem;
  after_previous();
  let_next_start();

  // Heads in groups whose K and V fit in L2 together; within a group the last rows of every head first: under causal
  // and prefix masks they see the most keys, and what is left for the end is short.  (4,096 rows of 7 documents,
  // 12 heads: 80 us head by head, 60 like this; 14,040 rows x 8 heads, 10 MB of K and V a head, all
  // heads as one group: 1.33 ms, head by head 1.27.)
  int item = blockIdx.x;
  const int split = item % p.splits;
  item /= p.splits;
  const int grp = item / (p.group * p.q_tiles);
  item -= grp * p.group * p.q_tiles;
  const int in_grp = min(p.group, p.heads - grp * p.group);
  const int bh = grp * p.group + item % in_grp;
  const int tile = p.q_tiles - 1 - item / in_grp;
  const int b = bh / p.H, h = bh - b * p.H;
  const int hk = h / p.G;
  const int bm = p.Bm > 1 ? b : 0;
  const int4 tab = p.table ? p.table[static_cast<long long>(bm) * p.q_tiles + tile] : make_int4(0, p.Sk, 0, p.Sk);
  const int lo_u = tab.x, hi_u = tab.y;
  int n0 = 0, n1 = 0;
  if (lo_u < hi_u) {
    n0 = lo_u / kTile;
    n1 = (hi_u + kTile - 1) / kTile;
    if (p.splits > 1) {
      const int per = (n1 - n0 + p.splits - 1) / p.splits;
      n0 = min(n1, n0 + split * per);
      n1 = min(n1, n0 + per);
    }
  }
  const int steps = n1 - n0;

  volatile int* abort_flag = &ss.abort_flag;
  int* err = &g_dense_err;

  if (warp == kLoad) {
    // ------------------------------------------------------------------ loads
    if (steps > 0) {
      if (elect_one()) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        mbar_arrive_expect_tx(&ss.q_full, kBytes);
        load_tile<DP>(sQ, &tm_q, &ss.q_full, tile * kTile, h, b);
      }
      int slot = 0, issued = 0, fixes = 0;
      uint32_t phase = 0;
      bool ok = true, fixing = false;
      // in the order of use: K(0) K(1) K(2), then V(j) K(j+3)
      int ik = 0, iv = 0;
      for (int i = 0; i < 2 * steps && ok; ++i) {
        const bool is_v = ik == steps || ik > iv + 2;
        const int step = is_v ? iv++ : ik++;
        if (issued >= kStages) {
          ok = bar_wait(&ss.empty[slot], phase ^ 1u, abort_flag, err, 301);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        const int row = (n0 + step) * kTile;
        uint8_t* dst = sKV + slot * kBytes;
        // V rows of this tile that no row of the CTA sees, but the tensor holds
        const bool fix = is_v && (row < lo_u || min(row + kTile, p.Sk) > hi_u);
        if (!fix) {
          if (elect_one()) {
            mbar_arrive_expect_tx(&ss.full[slot], kBytes);
            load_tile<DP>(dst, is_v ? &tm_v : &tm_k, &ss.full[slot], row, hk, b);
          }
        } else {
          if (lane == 0) {
            mbar_arrive_expect_tx(&ss.fix, kBytes);
            load_tile<DP>(dst, &tm_v, &ss.fix, row, hk, b);
          }
          __syncwarp();
          ok = bar_wait(&ss.fix, static_cast<uint32_t>(fixes & 1), abort_flag, err, 302);
          ok = __all_sync(0xffffffffu, ok);
          fixing = !ok;
          if (!ok) break;
          ++fixes;
          for (int r = 0; r < kTile; ++r)
            if (row + r < lo_u || row + r >= hi_u) zero_row<DP>(dst, r, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ss.full[slot]);
        }
        ++issued;
        if (++slot == kStages) {
          slot = 0;
          phase ^= 1u;
        }
      }
      if (lane == 0) {
        drain(&ss.q_full, 0);
        drain_ring(ss.full, kStages, issued);
        if (fixing) drain(&ss.fix, static_cast<uint32_t>(fixes & 1));
      }
    }
    __syncwarp();
  } else if (warp == kIssue) {
    // ------------------------------------------------------------------ products
    if (steps > 0 && elect_one()) {
      constexpr uint32_t kIdQK = idesc_f16(128, 128, kBF16 ? 1 : 0, 0, 0);
      constexpr uint32_t kIdPV = idesc_f16(128, DP, kBF16 ? 1 : 0, 0, 1);
      const uint32_t kvb = smem_u32(sKV);
      int slot = 0;
      uint32_t phase = 0;
      auto next = [&] {
        if (++slot == kStages) {
          slot = 0;
          phase ^= 1u;
        }
      };
      auto qk = [&](int j) {  // S(j) of the ring's next tile, once S(j - 2) has been read
        if (j >= 2 &&
            !bar_wait(&ss.s_read[j & 1], static_cast<uint32_t>(((j - 2) >> 1) & 1), abort_flag, err, 314))
          return false;
        if (!bar_wait(&ss.full[slot], phase, abort_flag, err, 312)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          umma_ts(tmem + col_s(j & 1), tmem + kColQ + 8 * kk, desc_d(kvb + slot * kBytes, kk), kIdQK, kk > 0);
        umma_commit(&ss.s_full[j & 1]);
        umma_commit(&ss.empty[slot]);
        next();
        return true;
      };
      bool ok = bar_wait(&ss.q_ready, 0, abort_flag, err, 311);
      for (int j = 0; j < 3 && j < steps && ok; ++j) ok = qk(j);
      for (int j = 0; j < steps && ok; ++j) {
        ok = bar_wait(&ss.full[slot], phase, abort_flag, err, 313) &&
             bar_wait(&ss.p_full[j & 1], static_cast<uint32_t>((j >> 1) & 1), abort_flag, err, 315);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_ts(tmem + kColO, tmem + kColP + 8 * kk, desc_rows(kvb + slot * kBytes, kk), kIdPV, j > 0 || kk > 0);
        umma_commit(&ss.o_full[j & 1]);
        umma_commit(&ss.empty[slot]);
        next();
        if (j + 3 < steps) ok = qk(j + 3);
      }
      // teardown: this thread's products complete before the tensor memory is released
      umma_commit(&ss.drain);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&ss.drain, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    }
    __syncwarp();
  } else if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------------ softmax
    const int half = warp >> 2;
    const int r_tile = 32 * (warp & 3) + lane;
    const int row = tile * kTile + r_tile;
    const uint32_t la = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const int pair = 1 + (warp & 3);  // named barrier of the two warps that share 32 rows
    const bool live = row < p.Sq;
    {
      int lo = 0, hi = live ? p.Sk : 0;  // rows behind the last see nothing, and choose nothing
      if (p.ranges && live) {
        const int2 r = p.ranges[static_cast<long long>(bm) * p.Sq + row];
        lo = r.x;
        hi = r.y;
      }
      const uint32_t seen = static_cast<uint32_t>(hi - lo);
      const int lo_max = tab.z, hi_min = tab.w;
      const float scale = kCap ? 1.f : p.scale_log2;
      float m = -INFINITY;
      uint64_t l2 = f2_pack(0.f, 0.f);  // sum of the rounded weights, two partial sums
      uint64_t t2 = l2;                 // of the fp32 ones
      bool ok = true;
      uint32_t rx[32], ry[32];  // scores of this step's first and last 32 keys
      // the cap and the mask on 32 scores of keys from `key` on
      auto prepare = [&](uint32_t* r, int key, bool border) {
        const uint32_t first = static_cast<uint32_t>(key - lo);
        if constexpr (kCap) {
          if (border) {  // what a masked place holds must not choose the form of tanh
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (first + e >= seen) r[e] = 0u;
          }
          capped<32>(r, p.cap);
        }
        if (border) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (first + e >= seen) r[e] = 0xff800000u;
        }
      };
      auto top_of = [&](const uint32_t* r) {
        float mv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) mv[e] = max3(__uint_as_float(r[e]), __uint_as_float(r[e + 4]), __uint_as_float(r[e + 8]));
#pragma unroll
        for (int c = 12; c < 28; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mv[e] = max3(mv[e], __uint_as_float(r[c + e]), __uint_as_float(r[c + 4 + e]));
#pragma unroll
        for (int e = 0; e < 4; ++e) mv[e] = max3(mv[e], mv[e], __uint_as_float(r[28 + e]));
        return max3(max3(mv[0], mv[1], mv[2]), mv[3], mv[3]);
      };
      // exponentials of 32 scores: their sums and, in pairs, their 16-bit roundings
      auto weights = [&](const uint32_t* r, uint64_t sc2, uint64_t nm2, uint32_t* pk) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), sc2, nm2), x0, x1);
          x0 = ex2_approx(x0);
          x1 = ex2_approx(x1);
          t2 = f2_add(t2, f2_pack(x0, x1));
          pk[e] = pack16<kBF16>(x0, x1);
          unpack16<kBF16>(pk[e], x0, x1);
          l2 = f2_add(l2, f2_pack(x0, x1));
        }
      };
      float mx = -INFINITY;
      if (steps > 0) {
        if (half == 0) {  // Q into tensor memory: row r_tile, 16-bit pairs along d
          ok = bar_wait(&ss.q_full, 0, abort_flag, err, 324);
          ok = __all_sync(0xffffffffu, ok);
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint4 u = *reinterpret_cast<const uint4*>(sQ + (c >> 1) * kHalfBytes +
                                                              sw128_offset(static_cast<uint32_t>(r_tile), 4 * (c & 1) + x));
              w[4 * x] = u.x;
              w[4 * x + 1] = u.y;
              w[4 * x + 2] = u.z;
              w[4 * x + 3] = u.w;
            }
            tmem_st16(la + kColQ + 16 * c, w);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ss.q_ready);
        }
        if (ok) ok = bar_wait(&ss.s_full[0], 0, abort_flag, err, 321);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          tc_fence_after();
          tmem_read32(la + col_s(0) + 64 * half, rx);
          tmem_read32(la + col_s(0) + 64 * half + 32, ry);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ss.s_read[0]);
          const int key = n0 * kTile;
          const bool border = key < lo_max || key + kTile > hi_min;
          prepare(rx, key + 64 * half, border);
          prepare(ry, key + 64 * half + 32, border);
          mx = max3(top_of(rx), top_of(ry), -INFINITY) * scale;
        }
      }
      // After an expired wait the loop goes on without work: both warps of a pair pass the same barriers.
      for (int j = 0; j < steps; ++j) {
        if (pair_any(pair, !(mx <= m + kRescale))) {  // a NaN raises too, and stays
          ss.join[half][0][r_tile] = mx;
          pair_sync(pair);
          mx = max3(mx, ss.join[half ^ 1][0][r_tile], mx);
          float f = 1.f;
          if (!(mx <= m + kRescale)) {
            f = ex2_approx(m - mx);  // 0 for the first maximum
            m = mx;
            l2 = f2_mul(l2, f2_pack(f, f));
            t2 = f2_mul(t2, f2_pack(f, f));
          }
          if (j > 0 && ok) {
            // O holds P V up to step j - 1 once that step's products are done; the next ones wait for this step's P
            ok = bar_wait(&ss.o_full[(j - 1) & 1], static_cast<uint32_t>(((j - 1) >> 1) & 1), abort_flag, err, 323);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
          }
          if (j > 0 && ok) {
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
              uint32_t o[16];
              const uint32_t at = la + kColO + half * (DP / 2) + 16 * c;
              tmem_read16(at, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(at, o);
            }
          }
        }
        if (!ok) continue;
        const float nm = m == -INFINITY ? 0.f : kRaise<kBF16> - m;
        const uint64_t sc2 = f2_pack(scale, scale), nm2 = f2_pack(nm, nm);
        const bool more = j + 1 < steps;
        uint32_t pk[16];
        const uint32_t o_phase = static_cast<uint32_t>(((j - 1) >> 1) & 1), s_phase = static_cast<uint32_t>(((j + 1) >> 1) & 1);
        uint64_t *o_bar = &ss.o_full[(j - 1) & 1], *s_bar = &ss.s_full[(j + 1) & 1];
        const bool o_done = j == 0 || bar_test(o_bar, o_phase);
        const bool s_done = !more || bar_test(s_bar, s_phase);
        weights(rx, sc2, nm2, pk);
        if (!o_done) ok = bar_wait(o_bar, o_phase, abort_flag, err, 325);  // P(j - 1) has been read
        if (ok && !s_done) ok = bar_wait(s_bar, s_phase, abort_flag, err, 326);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) continue;
        tc_fence_after();
        tmem_st16(la + kColP + 32 * half, pk);
        const uint32_t s_next = la + col_s((j + 1) & 1) + 64 * half;
        const int key = (n0 + j + 1) * kTile;
        const bool border = key < lo_max || key + kTile > hi_min;
        float top = -INFINITY;
        if (more) {
          tmem_read32(s_next, rx);
          if (kCap || border) prepare(rx, key + 64 * half, border);
          weights(ry, sc2, nm2, pk);
          tmem_st16(la + kColP + 32 * half + 16, pk);
          tmem_read32(s_next + 32, ry);  // beside the store
          top = top_of(rx);
        } else {
          weights(ry, sc2, nm2, pk);
          tmem_st16(la + kColP + 32 * half + 16, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ss.p_full[j & 1]);
          if (more) mbar_arrive(&ss.s_read[(j + 1) & 1]);
        }
        if (more) {
          if (kCap || border) prepare(ry, key + 64 * half + 32, border);
          mx = max3(top, top_of(ry), top) * scale;
        }
      }
      // ---- join the halves' sums; o / l and the row's log sum, half of the columns to a thread
      float l, lt, other;
      f2_unpack(l2, l, other);
      l += other;
      f2_unpack(t2, lt, other);
      lt += other;
      pair_sync(pair);  // the last maximum has been read
      ss.join[half][0][r_tile] = l;
      ss.join[half][1][r_tile] = lt;
      pair_sync(pair);
      l += ss.join[half ^ 1][0][r_tile];
      lt += ss.join[half ^ 1][1][r_tile];
      if (ok && steps > 0) {
        ok = bar_wait(&ss.o_full[(steps - 1) & 1], static_cast<uint32_t>(((steps - 1) >> 1) & 1), abort_flag, err, 322);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (ok) {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays NaN
        const float lse2 = lt == 0.f ? -INFINITY : log2f(lt) - (kRaise<kBF16> - m);
        const long long flat = static_cast<long long>(bh) * p.Sq + row;
        float* part = p.splits > 1 ? p.part + (split * p.rows + flat) * p.D : nullptr;
        const long long off = b * p.ob + h * p.oh + static_cast<long long>(row) * p.os;
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          const int c0 = half * (DP / 2) + 16 * c;
          uint32_t o[16];
          if (steps > 0) {
            tmem_read16(la + kColO + c0, o);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0u;
          }
          float v[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = l == 0.f ? 0.f : __uint_as_float(o[e]) * inv;
          if (live) {
#pragma unroll
            for (int e8 = 0; e8 < 2; ++e8) {
              const int d0 = c0 + 8 * e8;
              if (d0 < p.D) {
                if (part) {
                  reinterpret_cast<float4*>(part + d0)[0] = make_float4(v[8 * e8], v[8 * e8 + 1], v[8 * e8 + 2], v[8 * e8 + 3]);
                  reinterpret_cast<float4*>(part + d0)[1] =
                      make_float4(v[8 * e8 + 4], v[8 * e8 + 5], v[8 * e8 + 6], v[8 * e8 + 7]);
                } else {
                  store8<kBF16>(p.out, off + d0, v + 8 * e8);
                  if (p.out_lo) store_rest8<kBF16>(p.out_lo, flat * p.D + d0, v + 8 * e8);
                }
              }
            }
          }
        }
        if (live && half == 0) {
          if (part) p.part[(p.splits * p.D + split) * p.rows + flat] = lse2;
          else if (p.lse) p.lse[flat] = lse2 * 0.6931471805599453f;
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == kIssue) tmem_dealloc(tmem, kTmemCols);
}

// Joins the key splits of a row, always in their order: o = sum 2^(lse_s - m) o_s / sum 2^(lse_s - m).  A CTA takes 8
// rows, 16 lanes of 8 columns to each.
template <bool kBF16>
__global__ void __launch_bounds__(128) dense_join_kernel(const Params p) {
  constexpr int kLanes = 16;
  after_previous();
  const long long row = static_cast<long long>(blockIdx.x) * (128 / kLanes) + threadIdx.x / kLanes;
  const int d0 = 8 * (threadIdx.x % kLanes);
  if (row >= p.rows || d0 >= p.D) return;
  const float* lse = p.part + p.splits * p.rows * p.D + row;
  float m = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, lse[s * p.rows]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const float* src = p.part + row * p.D + d0;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float f = ex2_approx(lse[s * p.rows] - base);
    const float4 a = reinterpret_cast<const float4*>(src + s * p.rows * p.D)[0];
    const float4 c = reinterpret_cast<const float4*>(src + s * p.rows * p.D)[1];
    l += f;
    v[0] = fmaf(f, a.x, v[0]); v[1] = fmaf(f, a.y, v[1]); v[2] = fmaf(f, a.z, v[2]); v[3] = fmaf(f, a.w, v[3]);
    v[4] = fmaf(f, c.x, v[4]); v[5] = fmaf(f, c.y, v[5]); v[6] = fmaf(f, c.z, v[6]); v[7] = fmaf(f, c.w, v[7]);
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= inv;
  const int i = static_cast<int>(row % p.Sq);
  const long long bh = row / p.Sq;
  const int h = static_cast<int>(bh % p.H);
  store8<kBF16>(p.out, (bh / p.H) * p.ob + h * p.oh + static_cast<long long>(i) * p.os + d0, v);
  if (p.out_lo) store_rest8<kBF16>(p.out_lo, row * p.D + d0, v);
  if (p.lse && d0 == 0) p.lse[row] = l == 0.f ? -INFINITY : (base + log2f(l)) * 0.6931471805599453f;
}

template <int DP, bool kBF16, bool kCap>
int launch(const CUtensorMap* maps, const Params& p, long long grid, cudaStream_t stream) {
  auto* k = dense_fwd_kernel<DP, kBF16, kCap>;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<DP>()) != cudaSuccess)
    return BSA_ERR_CUDA;
  return launch_behind(k, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem_bytes<DP>(), stream, maps[0], maps[1],
                       maps[2], p) == cudaSuccess
             ? BSA_OK
             : BSA_ERR_CUDA;
}

}  // namespace dense

int make_map4(CUtensorMap* m, const Tensor4& t, int dtype, int B, int H, int S, int D, const char* name) {
  auto enc = reinterpret_cast<CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                           const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                           CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                           CUtensorMapFloatOOBfill)>(tensor_map_encoder());
  if (!enc) return set_error(BSA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  // an axis of one element may carry any stride: it is given one that every map accepts
  const long long ss = S > 1 ? t.ss : D, sh = H > 1 ? t.sh : ss * S, sb = B > 1 ? t.sb : sh * H;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(S), static_cast<cuuint64_t>(H),
                              static_cast<cuuint64_t>(B)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(ss) * 2, static_cast<cuuint64_t>(sh) * 2,
                                 static_cast<cuuint64_t>(sb) * 2};
  const cuuint32_t box[4] = {64, dense::kTile, 1, 1}, es[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, dtype == BSA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         4, t.p, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(BSA_ERR_ARG, "%s: cuTensorMapEncodeTiled failed (%d)", name, static_cast<int>(r));
  return BSA_OK;
}

// Key splits of a call: 1 where the row tiles alone give half of the SMs a CTA; else as many as give each SM one, with
// at least 4 key tiles to a split, since each costs a start and a partial output (128 queries x 16,384 keys, 1 head: 1
// tile 43 us, 2 28, 4 21; 77 queries x 1,001 keys, 16 heads: 12.3, 12.1, 13.4).
constexpr int kSplitTiles = 4;
int dense_pick_splits(int sms, int B, int H, int Sq, int Sk) {
  const long long ctas = static_cast<long long>(B) * H * ((Sq + dense::kTile - 1) / dense::kTile);
  if (ctas <= 0 || ctas * 2 > sms) return 1;
  const int most = (Sk + kSplitTiles * dense::kTile - 1) / (kSplitTiles * dense::kTile);
  const int want = static_cast<int>(sms / ctas);
  return want < most ? want : (most > 1 ? most : 1);
}

int launch_dense(const DenseArgs& a, int sms, cudaStream_t stream) {
  using namespace dense;
  CUtensorMap maps[3];
  int rc;
  if ((rc = make_map4(&maps[0], a.q, a.dtype, a.B, a.H, a.Sq, a.D, "q"))) return rc;
  if ((rc = make_map4(&maps[1], a.k, a.dtype, a.B, a.Hk, a.Sk, a.D, "k"))) return rc;
  if ((rc = make_map4(&maps[2], a.v, a.dtype, a.B, a.Hk, a.Sk, a.D, "v"))) return rc;
  Params p = {};
  p.ranges = a.ranges; p.table = a.table; p.Bm = a.Bm;
  p.H = a.H; p.G = a.H / a.Hk; p.Sq = a.Sq; p.Sk = a.Sk; p.D = a.D;
  p.q_tiles = (a.Sq + kTile - 1) / kTile;
  const long long bh = static_cast<long long>(a.B) * a.H;
  p.splits = a.splits;
  p.heads = static_cast<int>(bh);
  // a third of the 126 MB of L2 for K and V of a group: each of the two dies keeps its own copy of what both read
  const long long kv_bytes = 4ll * a.Sk * a.D;
  const long long group = (40ll << 20) / kv_bytes * p.G;
  p.group = static_cast<int>(group < 1 ? 1 : (group < bh ? group : bh));
  p.scale_log2 = a.sm_scale * 1.4426950408889634f;
  if (a.softcap > 0.f) p.cap = make_cap(p.scale_log2, a.softcap);
  p.out = a.o.p; p.ob = a.o.sb; p.oh = a.o.sh; p.os = a.o.ss;
  p.out_lo = a.o_lo;
  p.lse = a.lse;
  p.part = a.part;
  p.rows = bh * a.Sq;
  const long long grid = bh * p.q_tiles * p.splits;
  if (grid > INT_MAX) return set_error(BSA_ERR_SHAPE, "too many row tiles for one launch");
  const bool bf = a.dtype == BSA_DTYPE_BF16, cap = a.softcap > 0.f;
  if (a.D > 64)
    rc = bf ? (cap ? launch<128, true, true>(maps, p, grid, stream) : launch<128, true, false>(maps, p, grid, stream))
            : (cap ? launch<128, false, true>(maps, p, grid, stream) : launch<128, false, false>(maps, p, grid, stream));
  else
    rc = bf ? (cap ? launch<64, true, true>(maps, p, grid, stream) : launch<64, true, false>(maps, p, grid, stream))
            : (cap ? launch<64, false, true>(maps, p, grid, stream) : launch<64, false, false>(maps, p, grid, stream));
  if (rc) return set_error(rc, "dense attention kernel launch: %s", cudaGetErrorString(cudaGetLastError()));
  if (a.splits > 1) {
    const int jg = static_cast<int>((p.rows + 7) / 8);
    if (launch_behind(bf ? dense_join_kernel<true> : dense_join_kernel<false>, dim3(jg), dim3(128), 0, stream, p) != cudaSuccess)
      return set_error(BSA_ERR_CUDA, "dense attention join launch");
  }
  return BSA_OK;
}

int dense_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, dense::g_dense_err, sizeof(int)) != cudaSuccess) return BSA_ERR_CUDA;
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(dense::g_dense_err, &z, sizeof(int));
  }
  return v;
}

}  // namespace bsa
