// q/k RMSNorm + rotary positions over three axes (time, height, width), forward and backward.
//
//   r = (mean(x^2) + eps)^(-1/2),  z = w * x * r,  y = R(s) z
// R(s) turns each adjacent pair of z by the angle of its axis at token s's grid place (rope_3d.py:65-128).
// Backward, with dz = R(s)^T dy and g = w * dz:
//   dx = r g - x r^3 mean(g x),   dw = sum over tokens and heads of dz * x * r
// Everything is fp32 from the loaded value to the one rounding of the stored one.  r is computed again in
// the backward pass: it costs nothing beside the read of x, which the pass needs anyway.
//
// Bound: HBM.  One read and one write of the tensors forward, two reads and one write backward.  A group of lanes (16
// for D > 64, else 8) holds one row, 8 values (16 bytes of bf16) to a lane, as pairs for the packed fp32
// instructions.  A CTA keeps to one group of kHeads heads and walks over tokens, so that the weights, and what a lane
// needs of the angle tables, stay in registers, and a token's angles are used for all heads of the group:
// with w folded into them a row costs 3 packed operations a pair.  86,400 tokens x 32 heads: 5.4 TB/s of 6.54 measured (with
// the addresses worked out for each token and 4 heads, and scalar arithmetic, 240 instructions a row and warp: 4.1).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "bsa_dense.h"
#include "bsa_ptx.cuh"
#include "bsa_rows.cuh"

namespace bsa {
namespace nrope {

constexpr int kThreads = 256;
constexpr int kHeads = 8;  // of a group

struct Side {
  const void* x;
  long long xb, xh, xs;
  const void* g;
  long long gb, gh, gs;
  void* y;
  const void* w;
  int H, groups;  // groups of kHeads heads
};
// n / d by a multiplication, for n < 2^31: m = ceil(2^(31 + k) / d) with 2^k >= d
struct Divisor {
  unsigned m;
  int k;
  __device__ __forceinline__ int of(int n) const {
    return k < 0 ? n : static_cast<int>(__umulhi(static_cast<unsigned>(n), m) >> (k - 1));
  }
};
Divisor divisor(int d) {
  if (d == 1) return {0u, -1};
  int k = 0;
  while ((1ll << k) < d) ++k;
  return {static_cast<unsigned>(((1ull << (31 + k)) + d - 1) / d), k};
}

struct Params {
  Side side[2];
  int sides, S, D, w_dtype;
  int tiles;          // token tiles of a batch entry
  int chunk, chunks;  // token tiles of a CTA, CTAs of a head group
  long long total;    // token tiles of the batch
  float eps, inv_d;
  const float* rope;
  int nt, nh, nw;     // rotated pairs of each axis
  int gT, gH, gW, start;
  Divisor by_tiles, by_hw, by_w;
  float* partial;
};

__device__ __forceinline__ void load_weight(const void* w, int w_dtype, int d0, float* f) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (w_dtype == BSA_DTYPE_F32)
      f[e] = static_cast<const float*>(w)[d0 + e];
    else if (w_dtype == BSA_DTYPE_F16)
      f[e] = __half2float(static_cast<const __half*>(w)[d0 + e]);
    else
      f[e] = __bfloat162float(static_cast<const __nv_bfloat16*>(w)[d0 + e]);
  }
}

__device__ __forceinline__ uint64_t swapped(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return f2_pack(b, a);
}
__device__ __forceinline__ float sum_of(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Rows in flight: 4 forward (8: 306 us at 720p x 16 heads, 4: 263, 2: 301); 2 backward, where they leave registers
// for 4 CTAs to an SM (6 frames x 32 heads, both passes: 2 rows and 2 CTAs 174 us, 2 and 4 162 to 167, 4 and 2 162).  Reading
// the next rows before this step's arithmetic costs more registers than it hides (the same: 9 to 58 us more).
template <typename T, int kLanes, bool kBackward>
__global__ void __launch_bounds__(kThreads, kBackward && sizeof(T) == 2 ? 4 : 0) norm_rope_kernel(const Params p) {
  constexpr int kBatch = kBackward ? 2 : 4;
  constexpr int kRows = kThreads / kLanes;  // tokens of a tile
  after_previous();
  let_next_start();
  const int sub = threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int d0 = 8 * lane;
  const bool live = d0 < p.D;
  int grp = blockIdx.x / p.chunks;
  const int chunk = blockIdx.x - grp * p.chunks;
  const int which = grp >= p.side[0].groups ? 1 : 0;
  if (which) grp -= p.side[0].groups;
  const Side& sd = p.side[which];
  const int h0 = grp * kHeads;
  const int heads = min(kHeads, sd.H - h0);
  const bool norm = sd.w != nullptr;
  uint64_t w2[4];
  {
    float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (norm && live) load_weight(sd.w, p.w_dtype, d0, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) w2[e] = f2_pack(w[2 * e], w[2 * e + 1]);
  }
  // where the lane's 4 angles of a place (t, h, w) are: column `col` of axis `axis`'s table
  const float* cos_at[4];
  int axis[4], step[4], sin_off[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = (d0 >> 1) + e;
    if (i < p.nt) {
      axis[e] = 0;
      step[e] = p.nt;
      sin_off[e] = p.gT * p.nt;
      cos_at[e] = p.rope + i;
    } else if (i < p.nt + p.nh) {
      axis[e] = 1;
      step[e] = p.nh;
      sin_off[e] = p.gH * p.nh;
      cos_at[e] = p.rope + 2ll * p.gT * p.nt + (i - p.nt);
    } else {
      axis[e] = 2;
      step[e] = p.nw;
      sin_off[e] = p.gW * p.nw;
      cos_at[e] = p.rope + 2ll * p.gT * p.nt + 2ll * p.gH * p.nh + (i - p.nt - p.nh);
    }
  }
  uint64_t acc[4];  // this lane's share of dw
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = f2_pack(0.f, 0.f);
  const long long tile_end = min(p.total, (chunk + 1ll) * p.chunk);
  for (long long tile = static_cast<long long>(chunk) * p.chunk; tile < tile_end; ++tile) {
    const int b = p.by_tiles.of(static_cast<int>(tile));
    const int s = (static_cast<int>(tile) - b * p.tiles) * kRows + sub;
    const bool row = s < p.S;
    const bool on = row && live;
    // cos and sin of the pairs, with w folded in forward: y = (a, b) * cw + (b, a) * sw
    uint64_t cw[4], sw[4];
    if (p.rope && on) {
      const int place = p.start + s;
      const int t = p.by_hw.of(place);
      const int rem = place - t * p.gH * p.gW;
      const int h = p.by_w.of(rem);
      const int w = rem - h * p.gW;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float* at = cos_at[e] + (axis[e] == 0 ? t : axis[e] == 1 ? h : w) * step[e];
        const float c = at[0], sn = at[sin_off[e]];
        cw[e] = f2_pack(c, c);
        sw[e] = kBackward ? f2_pack(sn, -sn) : f2_pack(-sn, sn);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        cw[e] = f2_pack(1.f, 1.f);
        sw[e] = f2_pack(0.f, 0.f);
      }
    }
    if constexpr (!kBackward) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        cw[e] = f2_mul(cw[e], w2[e]);
        sw[e] = f2_mul(sw[e], swapped(w2[e]));
      }
    }
    const T* x = static_cast<const T*>(sd.x) + b * sd.xb + h0 * sd.xh + s * sd.xs + d0;
    const T* g = kBackward ? static_cast<const T*>(sd.g) + b * sd.gb + h0 * sd.gh + s * sd.gs + d0 : nullptr;
    T* y = static_cast<T*>(sd.y) + ((static_cast<long long>(b) * sd.H + h0) * p.S + s) * p.D + d0;
    const long long y_step = static_cast<long long>(p.S) * p.D;
#pragma unroll 1
    for (int i0 = 0; i0 < heads; i0 += kBatch) {
      Row8<T> xv[kBatch], gv[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        xv[i].zero();
        if constexpr (kBackward) gv[i].zero();
        if (on && i0 + i < heads) {
          xv[i].load(x + i * sd.xh);
          if constexpr (kBackward) gv[i].load(g + i * sd.gh);
        }
      }
      // the row's lanes share `row`, and the shuffles below are reached by the whole warp
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        uint64_t v[4];
        xv[i].get2(v);
        float r = 1.f;
        if (norm) {
          uint64_t q = f2_mul(v[0], v[0]);
#pragma unroll
          for (int e = 1; e < 4; ++e) q = f2_fma(v[e], v[e], q);
          r = rsqrtf(fmaf(row_sum<kLanes>(sum_of(q)), p.inv_d, p.eps));
          if (!row || i0 + i >= heads) r = 0.f;  // no row here: with eps = 0 its r would be infinite
        }
        const uint64_t r2 = f2_pack(r, r);
        uint64_t out[4];
        if constexpr (!kBackward) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint64_t u = f2_mul(v[e], r2);
            out[e] = f2_fma(swapped(u), sw[e], f2_mul(u, cw[e]));
          }
        } else {
          uint64_t gr[4], dot = f2_pack(0.f, 0.f);
          gv[i].get2(gr);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint64_t dz = f2_fma(swapped(gr[e]), sw[e], f2_mul(gr[e], cw[e]));
            acc[e] = f2_fma(dz, f2_mul(v[e], r2), acc[e]);
            out[e] = f2_mul(dz, w2[e]);
            dot = f2_fma(out[e], v[e], dot);
          }
          if (norm) {
            const float f = -row_sum<kLanes>(sum_of(dot)) * p.inv_d * r * r * r;
            const uint64_t f2 = f2_pack(f, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = f2_fma(v[e], f2, f2_mul(out[e], r2));
          }
        }
        if (on && i0 + i < heads) Row8<T>::store2(y + i * y_step, out);
      }
      x += kBatch * sd.xh;
      if constexpr (kBackward) g += kBatch * sd.gh;
      y += kBatch * y_step;
    }
  }
  if constexpr (kBackward) {
    if (p.partial) {
      // fixed order: lanes of a warp that hold the same columns, then the CTA's warps
      __shared__ float red[kThreads / 32][128];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v[2];
        f2_unpack(acc[e], v[0], v[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int o = 16; o >= kLanes; o >>= 1) v[c] += __shfl_xor_sync(0xffffffffu, v[c], o);
          if ((threadIdx.x & 31) < kLanes) red[threadIdx.x >> 5][d0 + 2 * e + c] = v[c];
        }
      }
      __syncthreads();
      for (int d = threadIdx.x; d < p.D; d += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kThreads / 32; ++k) v += red[k][d];
        p.partial[static_cast<long long>(blockIdx.x) * p.D + d] = v;
      }
    }
  }
}

// Column sums of the partial rows of one side, in a fixed order: 32 row strides of a column, then their sum.
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* partial, int rows0, int rows1, int D, float* dw0,
                                                           float* dw1) {
  __shared__ float red[32][33];
  after_previous();
  float* dst = blockIdx.y ? dw1 : dw0;
  if (!dst) return;
  const int c = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c;
  const int first = blockIdx.y ? rows0 : 0, rows = blockIdx.y ? rows1 : rows0;
  float v = 0.f;
  if (col < D)
#pragma unroll 8
    for (int r = part; r < rows; r += 32) v += partial[static_cast<long long>(first + r) * D + col];
  red[part][c] = v;
  __syncthreads();
  if (part == 0 && col < D) {
#pragma unroll
    for (int k = 1; k < 32; ++k) v += red[k][c];
    dst[col] = v;
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// CTAs of a launch: `most` at most where the work allows, each head group with the same number of them
Params make_params(const NormRopeArgs& a, int rows, int most) {
  Params p = {};
  p.sides = a.sides;
  p.S = a.S;
  p.D = a.D;
  p.w_dtype = a.w_dtype;
  int groups = 0;
  for (int i = 0; i < a.sides; ++i) {
    const NormRopeSide& s = a.side[i];
    Side& d = p.side[i];
    d.x = s.x.p; d.xb = s.x.sb; d.xh = s.x.sh; d.xs = s.x.ss;
    d.g = s.g.p; d.gb = s.g.sb; d.gh = s.g.sh; d.gs = s.g.ss;
    d.y = s.y; d.w = s.w; d.H = s.H;
    d.groups = (s.H + kHeads - 1) / kHeads;
    groups += d.groups;
  }
  p.tiles = (a.S + rows - 1) / rows;
  p.total = static_cast<long long>(a.B) * p.tiles;
  const long long per = most / groups > 0 ? most / groups : 1;
  p.chunk = static_cast<int>((p.total + per - 1) / per);
  p.chunks = static_cast<int>((p.total + p.chunk - 1) / p.chunk);
  p.by_tiles = divisor(p.tiles);
  p.eps = a.eps;
  p.inv_d = 1.f / static_cast<float>(a.D);
  p.rope = a.rope;
  p.nt = a.dt / 2; p.nh = a.dh / 2; p.nw = a.dw / 2;
  p.gT = a.gT; p.gH = a.gH; p.gW = a.gW;
  p.start = a.start;
  if (a.rope) {
    p.by_hw = divisor(a.gH * a.gW);
    p.by_w = divisor(a.gW);
  }
  p.partial = a.partial;
  return p;
}

template <typename T, bool kBackward>
int launch(const NormRopeArgs& a, int most, cudaStream_t stream, int* rows_out) {
  const bool wide = a.D > 64;
  const Params p = make_params(a, kThreads / (wide ? 16 : 8), most);
  const int grid = (p.side[0].groups + p.side[1].groups) * p.chunks;
  if (rows_out) {
    rows_out[0] = p.side[0].groups * p.chunks;
    rows_out[1] = p.side[1].groups * p.chunks;
  }
  auto* kernel = wide ? norm_rope_kernel<T, 16, kBackward> : norm_rope_kernel<T, 8, kBackward>;
  return launch_behind(kernel, dim3(grid), dim3(kThreads), 0, stream, p) == cudaSuccess ? BSA_OK : BSA_ERR_CUDA;
}

}  // namespace nrope

// CTAs: several waves forward, so that the last ones are short; one wave backward, where each leaves a row of weight
// gradients to add up (a head group has one at least)
constexpr int kForwardCtas = 64, kBackwardCtas = 4;  // for each SM

int norm_rope_partials(int groups) {
  const int most = kBackwardCtas * nrope::sm_count();
  return most > groups ? most : groups;
}

int launch_norm_rope(const NormRopeArgs& a, cudaStream_t stream) {
  const int most = kForwardCtas * nrope::sm_count();
  if (a.dtype == BSA_DTYPE_F32) return nrope::launch<float, false>(a, most, stream, nullptr);
  if (a.dtype == BSA_DTYPE_F16) return nrope::launch<__half, false>(a, most, stream, nullptr);
  return nrope::launch<__nv_bfloat16, false>(a, most, stream, nullptr);
}

int launch_norm_rope_backward(const NormRopeArgs& a, cudaStream_t stream) {
  int rows[2] = {0, 0};
  const int most = kBackwardCtas * nrope::sm_count();
  const int rc = a.dtype == BSA_DTYPE_F32   ? nrope::launch<float, true>(a, most, stream, rows)
                 : a.dtype == BSA_DTYPE_F16 ? nrope::launch<__half, true>(a, most, stream, rows)
                                            : nrope::launch<__nv_bfloat16, true>(a, most, stream, rows);
  if (rc || !a.partial) return rc;
  return launch_behind(nrope::weight_grad_kernel, dim3((a.D + 31) / 32, a.sides), dim3(1024), 0, stream, a.partial, rows[0],
                       rows[1], a.D, a.side[0].dw, a.sides > 1 ? a.side[1].dw : nullptr) == cudaSuccess
             ? BSA_OK
             : BSA_ERR_CUDA;
}

}  // namespace bsa
