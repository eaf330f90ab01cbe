// Internal interface of the operators around dense attention: q/k norm + rotary positions, attention over
// key intervals, and the 8-bit key/value cache (argument checks in bsa_dense_capi.cu).
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>
#include "../../include/bsa_b200.h"

namespace bsa {

// A launch that may begin while the stream's kernel before it ends: its kernel calls after_previous() before it touches
// global memory, and the one before it may call let_next_start() to say that its own CTAs have all begun.
template <typename... P, typename... A>
inline cudaError_t launch_behind(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                 A... args) {
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
#ifdef __CUDACC__
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif

// From bsa_capi.cu.
int set_error(int code, const char* fmt, ...);
void* tensor_map_encoder();  // cuTensorMapEncodeTiled, or null

// A [B, H, S, D] tensor with element strides and d contiguous.
struct Tensor4 {
  void* p = nullptr;
  long long sb = 0, sh = 0, ss = 0;
};

// ------------------------------------------------------------------ q/k norm + rotary positions
struct NormRopeSide {
  Tensor4 x;               // input
  Tensor4 g;               // backward: gradient of the output
  void* y = nullptr;       // forward: output, backward: gradient of x; contiguous [B, H, S, D]
  const void* w = nullptr; // [D] norm weight; null: no norm
  float* dw = nullptr;     // backward: [D], nullable
  int H = 0;
};
struct NormRopeArgs {
  NormRopeSide side[2];
  int sides = 1;
  int dtype = 0, w_dtype = 0;
  int B = 0, S = 0, D = 0;
  float eps = 0.f;
  const float* rope = nullptr;  // nullable: [cos_t | sin_t | cos_h | sin_h | cos_w | sin_w]
  int dt = 0, dh = 0, dw = 0, gT = 0, gH = 0, gW = 0, start = 0;
  float* partial = nullptr;     // backward: norm_rope_partials() rows of D
};
int launch_norm_rope(const NormRopeArgs& a, cudaStream_t stream);
int norm_rope_partials(int head_groups);  // most rows of `partial` on the current device
int launch_norm_rope_backward(const NormRopeArgs& a, cudaStream_t stream);

// ------------------------------------------------------------------ key intervals
// Row i of batch b sees the keys [lo, hi).  ranges: [Bm][Sq] int2; table: [Bm][tiles of 128 rows] int4
// (lowest lo and highest hi over the rows that see a key, highest lo and lowest hi over all rows).
struct RangesArgs {
  int2* ranges = nullptr;
  int4* table = nullptr;
  int Bm = 0, Sq = 0, Sk = 0;
  const int2* given = nullptr;         // intervals of the caller, clamped to [0, Sk]
  int causal = 0;
  int prefix = 0;
  const int32_t* prefixes = nullptr;   // one for each document (or batch entry)
  const int32_t* q_offsets = nullptr;  // [docs + 1]
  const int32_t* k_offsets = nullptr;
  int docs = 0;
  const int32_t* q_lengths = nullptr;  // [Bm]
  const int32_t* k_lengths = nullptr;  // [Bm]
  int k_add = 0;                       // added to every key length
};
int launch_ranges(const RangesArgs& a, cudaStream_t stream);

// ------------------------------------------------------------------ 8-bit cache
constexpr int kCacheBlock = 64;        // tokens that share a scale
constexpr int kMostSplits = 256;       // of the few-row attention along the tokens
struct CacheView {
  uint8_t* k = nullptr;                // [B, Hk, cap, D] e4m3 codes, contiguous
  uint8_t* v = nullptr;
  float* ks = nullptr;                 // [B, Hk, cap / 64] scales, powers of two
  float* vs = nullptr;
  int32_t* lengths = nullptr;          // [B] tokens held
  int B = 0, Hk = 0, cap = 0, D = 0;
};
struct AppendArgs {
  CacheView c;
  Tensor4 k, v;
  const int32_t* counts = nullptr;     // [B], nullable: n
  int dtype = 0, n = 0;
};
int launch_cache_append(const AppendArgs& a, cudaStream_t stream);
struct UnpackArgs {
  CacheView c;
  Tensor4 k, v;                        // fresh keys and values (n of them), nullable
  int dtype = 0, n = 0;
  void* ko = nullptr;                  // [B, Hk, rows, D] in dtype: held tokens, fresh tokens, zeros
  void* vo = nullptr;
  int rows = 0, zeros = 1;             // zeros 0: nothing is written behind the fresh tokens
};
int launch_cache_unpack(const UnpackArgs& a, cudaStream_t stream);
struct CacheAttnArgs {
  CacheView c;
  Tensor4 q;                           // [B, H, Sq, D]
  Tensor4 o;
  int dtype = 0, H = 0, Sq = 0, causal = 0, splits = 1;
  float sm_scale = 1.f;
  float* part = nullptr;               // splits > 1: [splits][B * H * Sq] rows of D + 2
};
int launch_cache_attention(const CacheAttnArgs& a, cudaStream_t stream);
int cache_device_error(int clear);

// ------------------------------------------------------------------ dense attention over key intervals
struct DenseArgs {
  int dtype = 0;
  int B = 0, H = 0, Hk = 0, Sq = 0, Sk = 0, D = 0;
  const int2* ranges = nullptr;        // null: every key
  const int4* table = nullptr;
  int Bm = 1;                          // 1: one set of intervals for every batch entry
  float sm_scale = 1.f, softcap = 0.f;
  Tensor4 q, k, v, o, g;               // g: gradient of o
  void* o_lo = nullptr;                // [B, H, Sq, D] contiguous: what o's rounding left over, nullable in the forward
  float* lse = nullptr;                // [B, H, Sq], nullable in the forward
  int splits = 1;
  float* part = nullptr;               // splits > 1: [splits][B * H * Sq][D + 1]
  Tensor4 dq, dk, dv;
  float* stats = nullptr;              // backward: dense_backward_stats_bytes()
};
int dense_pick_splits(int sms, int B, int H, int Sq, int Sk);
int launch_dense(const DenseArgs& a, int sms, cudaStream_t stream);
int make_map4(CUtensorMap* m, const Tensor4& t, int dtype, int B, int H, int S, int D, const char* name);
long long dense_backward_stats_bytes(int B, int H, int Sq, int Bm);
int launch_dense_backward(const DenseArgs& a, int sms, cudaStream_t stream);
int dense_bwd_device_error(int clear);
int dense_device_error(int clear);

}  // namespace bsa
