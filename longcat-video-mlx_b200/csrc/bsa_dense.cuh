// What the dense attention's forward and backward kernels share: tile geometry, tile loads, the tanh cap.
#pragma once
#include <cmath>
#include <type_traits>
#include "bsa_dense.h"
#include "bsa_ptx.cuh"

namespace bsa {
namespace dense {

constexpr int kTile = 128;  // rows of a query tile and of a key tile

// Bounded wait like mbar_wait, wholly inline: a call would spill what the softmax warps hold in registers.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int site) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  uint32_t spins = 0;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if ((++spins & 63u) == 0 && globaltimer_ns() - t0 > kWaitLimitNs) {
      *abort_flag = 1;
      atomicCAS(err, 0, site);
      return false;
    }
  }
}

// Whether the phase is over, without waiting: asked early, the answer is there when it is needed
__device__ __forceinline__ bool bar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// 4-D tiled load (d, token, head, batch), completion counted in bytes on `bar`.
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                                            int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// A tile of 128 rows in shared memory: one 16 KB half for each 64 columns of d, rows of 128 bytes in the
// 128-byte swizzle.  Rows past the tensor's end and columns past D arrive as zeros.
template <int DP>
__host__ __device__ constexpr int tile_bytes() { return kTile * DP * 2; }
constexpr int kHalfBytes = kTile * 128;

template <int DP>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int row, int h, int b) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) tma_load_4d(dst + c * kHalfBytes, m, bar, 64 * c, row, h, b);
}

// The loading warp's end, by one lane: every load that it issued has landed before the CTA may end and its shared memory go to
// another, whether or not their readers are still there.  `issued` tiles of a ring of `stages` have signalled, or will, on
// `full`; a load of a tile that this warp mends before it hands it on signals on a barrier of its own.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 < kWaitLimitNs) {
  }
}
__device__ __forceinline__ void drain_ring(uint64_t* full, int stages, int issued) {
  for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
    drain(&full[i % stages], static_cast<uint32_t>((i / stages) & 1));
}

// Zeros in row r of a tile, by the 32 lanes of a warp: lanes split the row's 16-byte chunks.
template <int DP>
__device__ __forceinline__ void zero_row(uint8_t* tile, int r, int lane) {
  constexpr int kChunks = DP / 8;
  for (int c = lane; c < kChunks; c += 32)
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kHalfBytes + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
}

// Operand descriptors of a tile for k-step kk: 16 values along d (K-major), or 16 rows (rows are K).  The step adds to
// the address field, which a tile in shared memory cannot carry out of.
__device__ __forceinline__ uint64_t desc_d(uint32_t tile, int kk) {
  return sdesc_sw128(tile, 16, 1024) + static_cast<uint64_t>(((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4);
}
__device__ __forceinline__ uint64_t desc_rows(uint32_t tile, int kk) {
  return sdesc_sw128(tile, kHalfBytes, 1024) + static_cast<uint64_t>((kk * 2048) >> 4);
}

// One lane of a whole warp, as a predicate the compiler knows to be one lane: issuing a product takes 14 to 26 cycles
// then, behind `lane == 0` 46 to 56 (its operands go through registers that a whole warp shares), where the tensor
// cores take 64 for it.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh(a) for a2 = 2 a log2(e): 1 - 2 / (1 + e^(2a)); exact at both infinities, absolute error of an ulp of 1
__device__ __forceinline__ float tanh_of(float a2) { return fmaf(-2.f, rcp_approx(1.f + ex2_approx(a2)), 1.f); }

template <bool kBF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return kBF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}

template <bool kBF16>
__device__ __forceinline__ void unpack16(uint32_t u, float& lo, float& hi) {
  if constexpr (kBF16) {
    lo = __uint_as_float(u << 16);
    hi = __uint_as_float(u & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    lo = f.x;
    hi = f.y;
  }
}

// 32 lanes x 32 (16) columns, complete on return: the wait belongs to the load, so no use of the registers can be
// moved between the two
__device__ __forceinline__ void tmem_read32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
      "}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_read16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Named barriers of two warps (64 threads); both warps must reach each of them whatever happens.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pair_any(int id, bool v) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(v)), "r"(id)
      : "memory");
  return any != 0;
}

// NaN wins: a row with a NaN score has a NaN maximum
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) { return max3(a, fabsf(b), fabsf(c)); }

// The cap: z log2(e) = cap log2(e) tanh(s / cap) of s = sm_scale q.k.  With x = q.k and a = s / cap, odd polynomials in a,
// fitted here for the smallest relative error (5.5e-7 for |a| <= 1/2, 6.1e-7 for |a| <= 1), the factors of a and of the
// result taken into their coefficients: x (c0 + c1 x^2 + ...).
struct Cap {
  float in;          // 2 sm_scale log2(e) / cap, of x
  float log2;        // cap log2(e)
  float near, most;  // |x| up to which |a| <= 1/2, and 1 (< 0: a coefficient would overflow)
  float n[4], m[6];  // coefficients
};
inline Cap make_cap(float scale_log2, float cap) {
  Cap c = {};
  c.in = 2.f * scale_log2 / cap;
  c.log2 = cap * 1.4426950408889634f;
  const float n[4] = {0.999999464f, -0.333263189f, 0.131902963f, -0.0444022231f};
  const float m[6] = {0.999999404f, -0.333290428f, 0.132814333f, -0.0516056716f, 0.0167431086f, -0.00306705665f};
  const double a = c.in * 0.34657359027997264;  // in / (2 log2(e)): a = a x
  double f = a * c.log2;
  float largest = 0.f;
  for (int i = 0; i < 6; ++i, f *= a * a) {
    c.m[i] = static_cast<float>(m[i] * f);
    if (i < 4) c.n[i] = static_cast<float>(n[i] * f);
    largest = fmaxf(largest, fabsf(static_cast<float>(f)));
  }
  const float square = 1.2e18f;  // x^2 stays finite
  c.most = largest < 1e37f ? fminf(static_cast<float>(1. / a), square) : -1.f;
  c.near = 0.5f * c.most;
  return c;
}
// N products q.k of a row through the cap where a polynomial serves all of the warp's rows, 5 or 7 packed operations a pair;
// else they stay as they are, and false.
template <int N>
__device__ __forceinline__ bool capped_near(uint32_t* r, const Cap& c) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < N; e += 2) top = max3_abs(top, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
  auto series = [&](const float* k, auto terms) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const uint64_t x = f2_pack(__uint_as_float(r[e]), __uint_as_float(r[e + 1]));
      const uint64_t v = f2_mul(x, x);
      uint64_t y = f2_pack(k[terms.value - 1], k[terms.value - 1]);
#pragma unroll
      for (int i = terms.value - 2; i >= 0; --i) y = f2_fma(y, v, f2_pack(k[i], k[i]));
      float a, b;
      f2_unpack(f2_mul(y, x), a, b);
      r[e] = __float_as_uint(a);
      r[e + 1] = __float_as_uint(b);
    }
  };
  if (__all_sync(0xffffffffu, top <= c.near)) {
    series(c.n, std::integral_constant<int, 4>());
  } else if (__all_sync(0xffffffffu, top <= c.most)) {
    series(c.m, std::integral_constant<int, 6>());
  } else {
    return false;
  }
  return true;
}
// ... or through the exponential: two operations of its unit a score, of which a step's exponentials take one each.
template <int N>
__device__ __forceinline__ void capped(uint32_t* r, const Cap& c) {
  if (capped_near<N>(r, c)) return;
#pragma unroll
  for (int e = 0; e < N; ++e) r[e] = __float_as_uint(c.log2 * tanh_of(__uint_as_float(r[e]) * c.in));
}
// ... or, where the slope is wanted too, as w = 1 - |tanh| with the product's sign, which keeps its digits where tanh rounds
// to 1: with e = 2^-|2 a log2(e)|, w = 2 e / (1 + e), z = +-(1 - w) and 1 - tanh^2 = w (2 - w).
template <int N>
__device__ __forceinline__ void capped_rest(uint32_t* r, const Cap& c) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float a2 = __uint_as_float(r[e]) * c.in, x = ex2_approx(-fabsf(a2));
    r[e] = __float_as_uint(copysignf(2.f * x * rcp_approx(1.f + x), a2));
  }
}
// z log2(e) of a rest, and the slope (0 for a masked place, which is a rest above 2)
__device__ __forceinline__ float capped_of(float w, const Cap& c, float& slope) {
  slope = fmaxf(fabsf(w) * (2.f - fabsf(w)), 0.f);
  return fmaf(-c.log2, w, copysignf(c.log2, w));
}

// 32 lanes x 32 columns store, counterpart of tmem_ld32
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Eight fp32 values as 16-bit ones in one 16-byte store
template <bool kBF16>
__device__ __forceinline__ void store8(void* out, long long off, const float* v) {
  uint4 u;
  u.x = pack16<kBF16>(v[0], v[1]);
  u.y = pack16<kBF16>(v[2], v[3]);
  u.z = pack16<kBF16>(v[4], v[5]);
  u.w = pack16<kBF16>(v[6], v[7]);
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + off) = u;
}

// What the rounding of store8 leaves over, in 16 bits: hi + lo holds a value to twice the bits
template <bool kBF16>
__device__ __forceinline__ void store_rest8(void* out, long long off, const float* v) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float lo, hi;
    unpack16<kBF16>(pack16<kBF16>(v[e], v[e + 1]), lo, hi);
    r[e] = v[e] - lo;
    r[e + 1] = v[e + 1] - hi;
  }
  store8<kBF16>(out, off, r);
}

}  // namespace dense
}  // namespace bsa
