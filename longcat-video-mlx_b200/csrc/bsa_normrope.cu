// q/k RMSNorm + rotary positions over three axes (time, height, width), forward and backward.
//
//   r = (mean(x^2) + eps)^(-1/2),  z = w * x * r,  y = R(s) z
// R(s) turns each adjacent pair of z by the angle of its axis at token s's grid place (rope_3d.py:65-128).
// Backward, with dz = R(s)^T dy and g = w * dz:
//   dx = r g - x r^3 mean(g x),   dw = sum over tokens and heads of dz * x * r
// Everything is fp32 from the loaded value to the one rounding of the stored one.  r is computed again in
// the backward pass: it costs nothing beside the read of x, which the pass needs anyway.
//
// Bound: HBM.  One read and one write of the tensors forward, two reads and one write backward.  A group of
// lanes (16 for D > 64, else 8) holds one row, 8 values (16 bytes of bf16) to a lane, and takes kHeads heads
// of one token, so the token's angles are loaded once for them and their rows are in flight together.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "bsa_dense.h"
#include "bsa_rows.cuh"

namespace bsa {
namespace nrope {

constexpr int kThreads = 256;
constexpr int kHeads = 4;

struct Side {
  const void* x;
  long long xb, xh, xs;
  const void* g;
  long long gb, gh, gs;
  void* y;
  const void* w;
  int H, groups;  // groups of kHeads heads
};
struct Params {
  Side side[2];
  int sides, S, D, w_dtype;
  long long items;  // (batch, token tile, head group), token tiles inside
  int tiles;        // token tiles of a batch entry
  float eps, inv_d;
  const float* rope;
  int nt, nh, nw;   // rotated pairs of each axis
  int gT, gH, gW, start;
  float* partial;
};

// cos and sin of the 4 pairs from `pair` on at grid token `tok`
__device__ __forceinline__ void load_angles(const Params& p, int tok, int pair, float* c, float* s) {
  const int hw = p.gH * p.gW;
  const int t = tok / hw;
  const int rem = tok - t * hw;
  const int h = rem / p.gW;
  const int w = rem - h * p.gW;
  const float* base_h = p.rope + 2ll * p.gT * p.nt;
  const float* base_w = base_h + 2ll * p.gH * p.nh;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = pair + e;
    const float *cp, *sp;
    if (i < p.nt) {
      cp = p.rope + static_cast<long long>(t) * p.nt + i;
      sp = cp + static_cast<long long>(p.gT) * p.nt;
    } else if (i < p.nt + p.nh) {
      cp = base_h + static_cast<long long>(h) * p.nh + (i - p.nt);
      sp = cp + static_cast<long long>(p.gH) * p.nh;
    } else {
      cp = base_w + static_cast<long long>(w) * p.nw + (i - p.nt - p.nh);
      sp = cp + static_cast<long long>(p.gW) * p.nw;
    }
    c[e] = __ldg(cp);
    s[e] = __ldg(sp);
  }
}

__device__ __forceinline__ void load_weight(const void* w, int w_dtype, int d0, float* f) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (w_dtype == BSA_DTYPE_F32)
      f[e] = __ldg(static_cast<const float*>(w) + d0 + e);
    else if (w_dtype == BSA_DTYPE_F16)
      f[e] = __half2float(static_cast<const __half*>(w)[d0 + e]);
    else
      f[e] = __bfloat162float(static_cast<const __nv_bfloat16*>(w)[d0 + e]);
  }
}

template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int kLanes, bool kBackward>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const Params p) {
  constexpr int kRows = kThreads / kLanes;  // tokens of a CTA's tile
  const int sub = threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int d0 = 8 * lane;
  const bool live = d0 < p.D;
  float acc[2][8];
  if constexpr (kBackward) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[i][e] = 0.f;
  }
  const int groups = p.side[0].groups + (p.sides > 1 ? p.side[1].groups : 0);
  for (long long item = blockIdx.x; item < p.items; item += gridDim.x) {
    int grp = static_cast<int>(item % groups);
    const long long bt = item / groups;
    const int b = static_cast<int>(bt / p.tiles);
    const int s = static_cast<int>(bt % p.tiles) * kRows + sub;
    const int which = grp >= p.side[0].groups ? 1 : 0;
    if (which) grp -= p.side[0].groups;
    const Side& sd = p.side[which];
    const int h0 = grp * kHeads;
    const int nh = min(kHeads, sd.H - h0);
    const bool row = s < p.S;
    const bool on = row && live;
    Row8<T> xv[kHeads], gv[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (on && i < nh) {
        xv[i].load(static_cast<const T*>(sd.x) + b * sd.xb + (h0 + i) * sd.xh + s * sd.xs + d0);
        if constexpr (kBackward)
          gv[i].load(static_cast<const T*>(sd.g) + b * sd.gb + (h0 + i) * sd.gh + s * sd.gs + d0);
      } else {
        xv[i].zero();
        if constexpr (kBackward) gv[i].zero();
      }
    }
    float c[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.rope && on) load_angles(p, p.start + s, d0 >> 1, c, sn);
    float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (sd.w && live) load_weight(sd.w, p.w_dtype, d0, w);
    // the row's kLanes lanes share `row`, and the shuffles below are reached by the whole warp
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      float x[8];
      xv[i].get(x);
      float r = 1.f;
      if (sd.w) {
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) q = fmaf(x[e], x[e], q);
        r = rsqrtf(fmaf(row_sum<kLanes>(q), p.inv_d, p.eps));
        if (!row || i >= nh) r = 0.f;  // no row here: with eps = 0 its r would be infinite
      }
      float y[8];
      if constexpr (!kBackward) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = x[2 * e] * r * w[2 * e], bb = x[2 * e + 1] * r * w[2 * e + 1];
          y[2 * e] = a * c[e] - bb * sn[e];
          y[2 * e + 1] = bb * c[e] + a * sn[e];
        }
      } else {
        float gr[8];
        gv[i].get(gr);
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = gr[2 * e] * c[e] + gr[2 * e + 1] * sn[e];
          const float bb = gr[2 * e + 1] * c[e] - gr[2 * e] * sn[e];
          if (sd.w) {
            const float ua = x[2 * e] * r, ub = x[2 * e + 1] * r;
            if (which) {
              acc[1][2 * e] = fmaf(a, ua, acc[1][2 * e]);
              acc[1][2 * e + 1] = fmaf(bb, ub, acc[1][2 * e + 1]);
            } else {
              acc[0][2 * e] = fmaf(a, ua, acc[0][2 * e]);
              acc[0][2 * e + 1] = fmaf(bb, ub, acc[0][2 * e + 1]);
            }
          }
          y[2 * e] = a * w[2 * e];
          y[2 * e + 1] = bb * w[2 * e + 1];
          dot = fmaf(y[2 * e], x[2 * e], fmaf(y[2 * e + 1], x[2 * e + 1], dot));
        }
        if (sd.w) {
          const float f = row_sum<kLanes>(dot) * p.inv_d * r * r;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = r * (y[e] - x[e] * f);
        }
      }
      if (on && i < nh) {
        T* out = static_cast<T*>(sd.y) + ((static_cast<long long>(b) * sd.H + h0 + i) * p.S + s) * p.D + d0;
        Row8<T>::store(out, y);
      }
    }
  }
  if constexpr (kBackward) {
    if (p.partial) {
      // fixed order: lanes of a warp that hold the same columns, then the CTA's warps
      __shared__ float red[2][kThreads / 32][128];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v = acc[i][e];
#pragma unroll
          for (int o = 16; o >= kLanes; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
          if ((threadIdx.x & 31) < kLanes) red[i][threadIdx.x >> 5][d0 + e] = v;
        }
      __syncthreads();
      for (int j = threadIdx.x; j < p.sides * p.D; j += kThreads) {
        const int i = j / p.D, d = j - i * p.D;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kThreads / 32; ++k) v += red[i][k][d];
        p.partial[(static_cast<long long>(blockIdx.x) * p.sides + i) * p.D + d] = v;
      }
    }
  }
}

// Column sums of the partial rows in a fixed order: 8 row strides of a column, then their sum.
__global__ void __launch_bounds__(256) weight_grad_kernel(const float* partial, int rows, int sides, int D, float* dw0,
                                                          float* dw1) {
  __shared__ float red[8][32];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31);
  const int part = threadIdx.x >> 5;
  float v = 0.f;
  if (col < sides * D)
    for (int r = part; r < rows; r += 8) v += partial[static_cast<long long>(r) * sides * D + col];
  red[part][threadIdx.x & 31] = v;
  __syncthreads();
  if (part == 0 && col < sides * D) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += red[k][threadIdx.x & 31];
    float* dst = col < D ? dw0 : dw1;
    if (dst) dst[col < D ? col : col - D] = v;
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

Params make_params(const NormRopeArgs& a, int rows) {
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
  p.items = static_cast<long long>(a.B) * p.tiles * groups;
  p.eps = a.eps;
  p.inv_d = 1.f / static_cast<float>(a.D);
  p.rope = a.rope;
  p.nt = a.dt / 2; p.nh = a.dh / 2; p.nw = a.dw / 2;
  p.gT = a.gT; p.gH = a.gH; p.gW = a.gW;
  p.start = a.start;
  p.partial = a.partial;
  return p;
}

template <typename T, bool kBackward>
int launch(const NormRopeArgs& a, int grid_most, cudaStream_t stream, int* grid_out) {
  const bool wide = a.D > 64;
  const Params p = make_params(a, kThreads / (wide ? 16 : 8));
  const int grid = static_cast<int>(p.items < grid_most ? p.items : grid_most);
  if (grid_out) *grid_out = grid;
  if (wide)
    norm_rope_kernel<T, 16, kBackward><<<grid, kThreads, 0, stream>>>(p);
  else
    norm_rope_kernel<T, 8, kBackward><<<grid, kThreads, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? BSA_OK : BSA_ERR_CUDA;
}

}  // namespace nrope

int norm_rope_partials() { return 4 * nrope::sm_count(); }

int launch_norm_rope(const NormRopeArgs& a, cudaStream_t stream) {
  const int most = 1 << 30;  // one item for each CTA: the hardware's scheduler balances them
  if (a.dtype == BSA_DTYPE_F32) return nrope::launch<float, false>(a, most, stream, nullptr);
  if (a.dtype == BSA_DTYPE_F16) return nrope::launch<__half, false>(a, most, stream, nullptr);
  return nrope::launch<__nv_bfloat16, false>(a, most, stream, nullptr);
}

int launch_norm_rope_backward(const NormRopeArgs& a, cudaStream_t stream) {
  int grid = 0;
  const int most = norm_rope_partials();
  const int rc = a.dtype == BSA_DTYPE_F32   ? nrope::launch<float, true>(a, most, stream, &grid)
                 : a.dtype == BSA_DTYPE_F16 ? nrope::launch<__half, true>(a, most, stream, &grid)
                                            : nrope::launch<__nv_bfloat16, true>(a, most, stream, &grid);
  if (rc || !a.partial) return rc;
  const int cols = a.sides * a.D;
  nrope::weight_grad_kernel<<<(cols + 31) / 32, 256, 0, stream>>>(a.partial, grid, a.sides, a.D, a.side[0].dw,
                                                                  a.sides > 1 ? a.side[1].dw : nullptr);
  return cudaGetLastError() == cudaSuccess ? BSA_OK : BSA_ERR_CUDA;
}

}  // namespace bsa
