// Eight consecutive values of a row: 16-byte loads and stores, fp32 in registers.  The loads are plain ones: a kernel that
// begins before the one in front of it has ended (bsa_dense.h) may read what that one writes.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace bsa {

__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __nv_bfloat16) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __half) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void unpack_pair(uint32_t u, float& lo, float& hi, __nv_bfloat16) {
  lo = __uint_as_float(u << 16);
  hi = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ void unpack_pair(uint32_t u, float& lo, float& hi, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  lo = f.x;
  hi = f.y;
}

template <typename T>
struct Row8 {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float* f) const {
    unpack_pair(u.x, f[0], f[1], T());
    unpack_pair(u.y, f[2], f[3], T());
    unpack_pair(u.z, f[4], f[5], T());
    unpack_pair(u.w, f[6], f[7], T());
  }
  // as four packed pairs
  __device__ __forceinline__ void get2(uint64_t* v) const {
    float f[8];
    get(f);
#pragma unroll
    for (int e = 0; e < 4; ++e) asm("mov.b64 %0, {%1, %2};" : "=l"(v[e]) : "f"(f[2 * e]), "f"(f[2 * e + 1]));
  }
  static __device__ __forceinline__ void store2(T* p, const uint64_t* v) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) asm("mov.b64 {%0, %1}, %2;" : "=f"(f[2 * e]), "=f"(f[2 * e + 1]) : "l"(v[e]));
    store(p, f);
  }
  static __device__ __forceinline__ void store(T* p, const float* f) {
    uint4 o;
    o.x = pack_pair(f[0], f[1], T());
    o.y = pack_pair(f[2], f[3], T());
    o.z = pack_pair(f[4], f[5], T());
    o.w = pack_pair(f[6], f[7], T());
    *reinterpret_cast<uint4*>(p) = o;
  }
};

template <>
struct Row8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  __device__ __forceinline__ void get2(uint64_t* v) const {
    float f[8];
    get(f);
#pragma unroll
    for (int e = 0; e < 4; ++e) asm("mov.b64 %0, {%1, %2};" : "=l"(v[e]) : "f"(f[2 * e]), "f"(f[2 * e + 1]));
  }
  static __device__ __forceinline__ void store2(float* p, const uint64_t* v) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) asm("mov.b64 {%0, %1}, %2;" : "=f"(f[2 * e]), "=f"(f[2 * e + 1]) : "l"(v[e]));
    store(p, f);
  }
  static __device__ __forceinline__ void store(float* p, const float* f) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};

}  // namespace bsa
