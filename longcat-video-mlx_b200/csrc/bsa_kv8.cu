// Key/value cache in 8 bits: e4m3 codes with one power-of-two scale for each 64 tokens of a head.
//
//   s = the smallest 2^n with max|x| / s <= 448,   code = e4m3(x / s) to nearest even,   x ~ code * s
// A floating-point code loses no precision by a power-of-two scale (only the codes' subnormals move), and
// the scale makes three steps exact: x / s, the rescaling of a block whose largest value grew (up to codes
// that become subnormal), and code * s in 16 bits within the type's range: fp16 holds every code exactly for s >= 2^-15 (the
// last place of a code is 2^-9 s, fp16's 2^-24), bf16 for s >= 2^-124 (2^-133), up to the type's largest value.  Outside,
// unpacking rounds and clamps where the lookup of few rows, which takes s in fp32, does not.
//
// Append: 256 threads for each touched block of one head and tensor.  Bound: HBM (2 bytes read, 1 written for a
// value), at few tokens the launch.  A block that already holds tokens keeps its scale unless the new ones
// need a larger one; then its codes are decoded and rounded again at the new scale.  6,240 tokens x 32 heads: 35 us,
// 4.4 TB/s of 6.5; the maximum and the conversion, about 100 instructions for 8 values, are what is left.
//
// Attention for few rows (kernel `cache_attn_kernel`): the H / Hk query heads of a key head times the query
// tokens are the rows of one mma tile of 16, so each code is read once for all of them.  Bound: HBM, one byte
// for a value of K and V.  A warp takes every fourth block of 64 tokens, brings its codes to shared memory by
// cp.async (K and V of a block are separate groups in a ring of three, so loads run behind the arithmetic),
// and widens them to fp16 in registers, which is exact, for mma.m16n8k16 with fp32 sums.  The queries go
// through fp16 too: bf16's 8 bits fit fp16's 11, and each row is scaled by a power of two to its largest
// value, so only elements 2^-14 below it lose bits.  P, at most 1, is multiplied by 2^15 in fp16, so that a long tail of
// small weights keeps its bits (2^-29 of the largest) and its sum.  The scales of the blocks are applied in fp32: K's to the
// scores, V's, with P's 2^-15, where a block's P V is added to the output.  The tensor cores' newer path does not pay here:
// 16 rows fill an eighth of its smallest tile, and its operands would have to pass through shared memory.
// One token, 8 sequences of up to 32,000 tokens, 32 heads on 8: 78 us, 4.7 TB/s of 6.5.
#include <climits>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "bsa_dense.h"
#include "bsa_rows.cuh"

namespace bsa {
namespace kv8 {

__device__ int g_cache_err;

// The smallest power of two s with amax / s <= 448 (448 = 1.75 * 2^8); 0 for 0, never below 2^-126.
__device__ __forceinline__ float scale_of(float amax) {
  if (!(amax > 0.f)) return 0.f;
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) + ((u & 0x7fffffu) > 0x600000u ? 1 : 0) - 8;
  return __uint_as_float(static_cast<uint32_t>(e < 1 ? 1 : e) << 23);
}
__device__ __forceinline__ float inverse_of(float s) {  // of a power of two or 0, exact (0 for 0)
  return s > 0.f ? 1.f / s : 0.f;
}
__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}
__device__ __forceinline__ uint2 encode8(const float* f, float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = static_cast<uint32_t>(to_e4m3x2(f[4 * i] * inv, f[4 * i + 1] * inv)) |
           (static_cast<uint32_t>(to_e4m3x2(f[4 * i + 2] * inv, f[4 * i + 3] * inv)) << 16);
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void decode8(uint2 u, float* f) {
  const uint32_t w[2] = {u.x, u.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t a = e4m3x2_to_f16x2(static_cast<uint16_t>(w[i]));
    const uint32_t b = e4m3x2_to_f16x2(static_cast<uint16_t>(w[i] >> 16));
    unpack_pair(a, f[4 * i], f[4 * i + 1], __half());
    unpack_pair(b, f[4 * i + 2], f[4 * i + 3], __half());
  }
}

// ------------------------------------------------------------------------------------------ append
constexpr int kAppendThreads = 256;

struct AppendParams {
  CacheView c;
  const void* x[2];
  long long sb[2], sh[2], ss[2];
  const int32_t* counts;
  int n, blocks;  // tokens, and the most blocks that they touch
};

// 256 threads on one touched block of one head of K or V; `sync` is a barrier of theirs, `red` of 2 x 8 words
template <typename T, typename Sync>
__device__ __forceinline__ void append_block(const AppendParams& p, int b, int h, int which, int block, int held, int tid,
                                             uint32_t (*red)[kAppendThreads / 32], Sync&& sync) {
  const int bh = b * p.c.Hk + h;
  const int room = p.c.cap - held;
  int n = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
  if (held < 0 || n > room) {  // a device-side length the host could not check: keep what fits
    if (tid == 0) atomicCAS(&g_cache_err, 0, BSA_ERR_INDEX);
    n = held < 0 ? 0 : max(room, 0);
  }
  if (n <= 0) return;
  const int blk = held / kCacheBlock + block;
  const int t0 = blk * kCacheBlock;
  if (t0 >= held + n) return;
  const int lanes = p.c.D >> 3;                // 8 values to a thread
  const int per = kAppendThreads / 16;         // rows of a pass (16 thread columns, D / 8 of them used)
  const int col = tid & 15, row0 = tid >> 4;
  const bool live = col < lanes;
  const int nblk = p.c.cap / kCacheBlock;
  uint8_t* codes = (which ? p.c.v : p.c.k) + (static_cast<long long>(bh) * p.c.cap + t0) * p.c.D + 8 * col;
  float* sp = (which ? p.c.vs : p.c.ks) + static_cast<long long>(bh) * nblk + blk;
  const T* x = static_cast<const T*>(p.x[which]) + b * p.sb[which] + h * p.sh[which] + 8 * col;
  Row8<T> v[kCacheBlock / per];
  uint32_t top = 0u;  // largest magnitude bits of the low and the high halves: their order is the values' order
#pragma unroll
  for (int i = 0; i < kCacheBlock / per; ++i) {
    const int t = t0 + row0 + i * per - held;  // place among the new tokens
    if (live && t >= 0 && t < n) {
      v[i].load(x + static_cast<long long>(t) * p.ss[which]);
      const uint32_t w[4] = {v[i].u.x, v[i].u.y, v[i].u.z, v[i].u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __vmaxu2(top, w[e] & 0x7fff7fffu);
    } else {
      v[i].zero();
    }
  }
  constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  auto block_max = [&](uint32_t m, int k) {
    uint32_t one = max(m & 0xffffu, m >> 16);
    one = __reduce_max_sync(0xffffffffu, one);
    if ((tid & 31) == 0) red[k][tid >> 5] = one;
    sync();
#pragma unroll
    for (int i = 0; i < kAppendThreads / 32; ++i) one = max(one, red[k][i]);
    return one;
  };
  const float was = *sp;
  uint32_t largest = block_max(top, 0);
  float least = 0.f;
  if (largest >= kInf) {  // neither infinity nor NaN sets a scale: once more without them
    least = 1.17549435e-38f;  // 2^-126, so that infinity * (1 / s) is infinity where there is nothing but zeros beside it
    top = 0u;
#pragma unroll
    for (int i = 0; i < kCacheBlock / per; ++i) {
      const uint32_t w[4] = {v[i].u.x, v[i].u.y, v[i].u.z, v[i].u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = w[e] & 0x7fffu, hi = (w[e] >> 16) & 0x7fffu;
        top = max(top, max(lo < kInf ? lo : 0u, hi < kInf ? hi : 0u));
      }
    }
    largest = block_max(top, 1);
  }
  float amax, none;
  unpack_pair(largest, amax, none, T());
  const float old = t0 < held ? was : 0.f;     // a block without tokens has no scale to keep
  const float s = fmaxf(fmaxf(old, least), scale_of(amax));
  const float inv = inverse_of(s);
#pragma unroll
  for (int i = 0; i < kCacheBlock / per; ++i) {
    const int r = row0 + i * per;
    const int t = t0 + r - held;
    if (!live || t >= n) continue;
    uint2* dst = reinterpret_cast<uint2*>(codes + static_cast<long long>(r) * p.c.D);
    float f[8];
    if (t >= 0) {
      v[i].get(f);
      *dst = encode8(f, inv);
    } else if (s != old) {
      decode8(*dst, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= old;
      *dst = encode8(f, inv);
    }
  }
  if (tid == 0) *sp = s;
}

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendParams p) {
  __shared__ uint32_t red[2][kAppendThreads / 32];
  after_previous();
  let_next_start();
  const int b = blockIdx.y / p.c.Hk, h = blockIdx.y - b * p.c.Hk;
  append_block<T>(p, b, h, blockIdx.z, blockIdx.x, p.c.lengths[b], threadIdx.x, red, [] { __syncthreads(); });
}

// lengths[b] += what append_kernel wrote; a launch of its own, since every CTA above reads the old lengths
__global__ void advance_kernel(int32_t* lengths, const int32_t* counts, int n, int cap, int B) {
  after_previous();
  for (int b = threadIdx.x; b < B; b += blockDim.x) {
    const int held = lengths[b];
    const int add = counts ? min(max(counts[b], 0), n) : n;
    if (held >= 0) lengths[b] = min(held + add, max(cap, held));
  }
}

// Both in one launch where a batch entry's blocks fit a cluster of 8 CTAs of four blocks each (a token on up to 16 heads):
// the length advances when all of the cluster has read it.  A second launch costs more there than the work does (a token
// of 16 x 8 heads: 12.5 us a call with two, 10.7 with one).
constexpr int kSide = 4, kMostCluster = 8;
template <typename T>
__global__ void __launch_bounds__(kSide * kAppendThreads) append_few_kernel(const AppendParams p, int cluster) {
  __shared__ uint32_t red[kSide][2][kAppendThreads / 32];
  after_previous();
  const int b = blockIdx.x / cluster, rank = blockIdx.x - b * cluster;
  const int side = threadIdx.x / kAppendThreads;
  const int held = p.c.lengths[b];
  const int item = rank * kSide + side;
  if (item < p.blocks * p.c.Hk * 2) {
    const int block = item / (2 * p.c.Hk), head = item - block * 2 * p.c.Hk;
    append_block<T>(p, b, head >> 1, head & 1, block, held, threadIdx.x % kAppendThreads, red[side],
                    [&] {
                      __syncwarp();
                      asm volatile("bar.sync %0, %1;" ::"r"(1 + side), "n"(kAppendThreads) : "memory");
                    });
  }
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0 && threadIdx.x == 0 && held >= 0) {
    const int add = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    p.c.lengths[b] = min(held + add, max(p.c.cap, held));
  }
}

// ------------------------------------------------------------------------------------------ unpack
struct UnpackParams {
  CacheView c;
  const void* x[2];
  long long sb[2], sh[2], ss[2];
  void* out[2];
  int n, rows, zeros;
};

template <typename T>
__global__ void __launch_bounds__(256) unpack_kernel(const UnpackParams p) {
  const int bh = blockIdx.y;
  const int b = bh / p.c.Hk, h = bh - b * p.c.Hk;
  const int which = blockIdx.z;
  const int held = min(max(p.c.lengths[b], 0), p.c.cap);
  const int rows = p.zeros ? p.rows : min(p.rows, held + (p.x[0] ? p.n : 0));
  const int lanes = p.c.D >> 3;
  const int nblk = p.c.cap / kCacheBlock;
  const uint8_t* codes = (which ? p.c.v : p.c.k) + static_cast<long long>(bh) * p.c.cap * p.c.D;
  const float* sp = (which ? p.c.vs : p.c.ks) + static_cast<long long>(bh) * nblk;
  const T* x = static_cast<const T*>(p.x[which]);
  if (x) x += b * p.sb[which] + h * p.sh[which];
  T* out = static_cast<T*>(p.out[which]) + static_cast<long long>(bh) * p.rows * p.c.D;
  const float most = std::is_same<T, __half>::value ? 65504.f : 3.3895314e38f;  // the type's largest value
  const int j0 = blockIdx.x * 64 * lanes;
#pragma unroll 2
  for (int j = j0 + threadIdx.x; j < min(j0 + 64 * lanes, rows * lanes); j += 256) {
    const int r = j / lanes, d0 = 8 * (j - r * lanes);
    float f[8];
    if (r < held) {
      decode8(*reinterpret_cast<const uint2*>(codes + static_cast<long long>(r) * p.c.D + d0), f);
      const float s = sp[r / kCacheBlock];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] *= s;
        // the code nearest to a value just below the type's largest may lie above it
        f[e] = f[e] != f[e] ? f[e] : fminf(fmaxf(f[e], -most), most);
      }
      Row8<T>::store(out + static_cast<long long>(r) * p.c.D + d0, f);
    } else if (x && r < held + p.n) {
      Row8<T> v;
      v.load(x + static_cast<long long>(r - held) * p.ss[which] + d0);
      *reinterpret_cast<uint4*>(out + static_cast<long long>(r) * p.c.D + d0) = v.u;
    } else {
      *reinterpret_cast<uint4*>(out + static_cast<long long>(r) * p.c.D + d0) = make_uint4(0, 0, 0, 0);
    }
  }
}

// ------------------------------------------------------------------------- attention for few rows
constexpr int kWarps = 4;
constexpr int kAttnThreads = 32 * kWarps;
constexpr int kRowBytes = 128;                       // a token's codes in shared memory, zero-filled behind D
constexpr int kSlotBytes = kCacheBlock * kRowBytes;  // K or V of one block
constexpr int kSlots = 3;
constexpr int kAttnSmem = kWarps * kSlots * kSlotBytes;
constexpr float kRaise = 15.f, kLower = 1.f / 32768.f;  // of P: log2, and what its sums are multiplied by

__device__ __forceinline__ void store1(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

struct AttnParams {
  CacheView c;
  const void* q;
  long long qb, qh, qs;
  void* o;
  long long ob, oh, os;
  int H, G, Sq, rows, row_tiles, splits, causal;
  float scale_log2;
  long long total;  // B * H * Sq
  float* part;      // splits > 1: [splits][total][D] sums, then [splits][total][2] of (maximum, sum)
};

// 16-byte chunk `chunk` of token row `r`, exchanged by the row's low bits: the fragments below read one
// chunk of 4 tokens, or two of 8, without two lanes on one bank
__device__ __forceinline__ uint32_t chunk_at(int r, int chunk) {
  return static_cast<uint32_t>(r * kRowBytes + ((chunk ^ (r & 7)) << 4));
}

// The codes of a block (64 token rows of D bytes, `held` of them of tokens) into a slot; the rows behind arrive as
// zeros.  kPieces: D / kPiece where it is known (D = 128: a lane keeps its column and steps 4 rows), 0: as it comes.
template <int kPiece, int kPieces>
__device__ __forceinline__ void load_block(uint8_t* slot, const uint8_t* src, int D, int held, int lane) {
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(slot));
  auto copy = [&](uint32_t dst, const uint8_t* from, bool token) {
    const int bytes = token ? kPiece : 0;
    if constexpr (kPiece == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
  };
  if constexpr (kPieces == 8) {
    const int r = lane >> 3, c = lane & 7;
    const uint8_t* from = src + lane * 16;
    const uint32_t even = base + chunk_at(r, c), odd = base + chunk_at(r + 4, c);
    if (held >= kCacheBlock) {
#pragma unroll
      for (int i = 0; i < kCacheBlock / 8; ++i) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(even + i * 8 * kRowBytes), "l"(from + i * 1024)
                     : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(odd + i * 8 * kRowBytes), "l"(from + i * 1024 + 512)
                     : "memory");
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCacheBlock / 8; ++i) {
        copy(even + i * 8 * kRowBytes, from + i * 1024, 8 * i + r < held);
        copy(odd + i * 8 * kRowBytes, from + i * 1024 + 512, 8 * i + 4 + r < held);
      }
    }
  } else {
    const int pieces = D / kPiece;
    int r = lane / pieces, c = lane - r * pieces;
    const int dr = 32 / pieces, dc = 32 - dr * pieces;
    for (; r < kCacheBlock;) {
      const int byte = c * kPiece;
      copy(base + chunk_at(r, byte >> 4) + (byte & 15), src + r * D + byte, r < held);
      r += dr;
      c += dc;
      if (c >= pieces) {
        c -= pieces;
        ++r;
      }
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t byte_pair(uint32_t a, uint32_t b, int sel) { return __byte_perm(a, b, sel); }

template <typename T, bool kFull>  // kFull: D = 128
__global__ void __launch_bounds__(kAttnThreads, 2) cache_attn_kernel(const AttnParams p) {
  after_previous();
  let_next_start();
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float st_m[kWarps][16], st_l[kWarps][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int bh = blockIdx.y / p.row_tiles;
  const int r0 = (blockIdx.y - bh * p.row_tiles) * 16;
  const int b = bh / p.c.Hk, hk = bh - b * p.c.Hk;
  const int held = min(max(p.c.lengths[b], 0), p.c.cap);
  const int D = kFull ? 128 : p.c.D;
  uint8_t* ring = smem + warp * kSlots * kSlotBytes;
  if (!kFull) {  // columns behind D stay zero: the copies never write them
    for (int i = threadIdx.x * 16; i < kAttnSmem; i += kAttnThreads * 16)
      *reinterpret_cast<uint4*>(smem + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  // the split's blocks; the tile's last row sees the most keys
  int seen = held;
  if (p.causal) {
    int last = 0;  // latest token among the tile's rows: rows go token by token within a head
    const int r_end = min(r0 + 16, p.rows) - 1;
    last = r0 / p.Sq != r_end / p.Sq ? p.Sq - 1 : r_end % p.Sq;
    seen = min(max(held - p.Sq + last + 1, 0), held);
  }
  const int blocks = (seen + kCacheBlock - 1) / kCacheBlock;
  const int per = (blocks + p.splits - 1) / p.splits;
  const int blk_end = min(blocks, (static_cast<int>(blockIdx.x) + 1) * per);
  const int nblk = p.c.cap / kCacheBlock;
  const uint8_t* kc = p.c.k + static_cast<long long>(bh) * p.c.cap * D;
  const uint8_t* vc = p.c.v + static_cast<long long>(bh) * p.c.cap * D;
  const float* ksc = p.c.ks + static_cast<long long>(bh) * nblk;
  const float* vsc = p.c.vs + static_cast<long long>(bh) * nblk;
  int blk = blockIdx.x * per + warp;
  const bool wide = (D & 15) == 0;
  int slot_load = 0;
  auto fetch = [&](const uint8_t* codes, int k) {
    uint8_t* slot = ring + slot_load * kSlotBytes;
    if (k < blk_end) {
      const uint8_t* src = codes + static_cast<long long>(k) * kCacheBlock * D;
      const int n = held - k * kCacheBlock;
      if (kFull) load_block<16, 8>(slot, src, D, n, lane);
      else if (wide) load_block<16, 0>(slot, src, D, n, lane);
      else load_block<8, 0>(slot, src, D, n, lane);
    } else {
      asm volatile("cp.async.commit_group;" ::: "memory");  // empty: the group count stays in step
    }
    if (++slot_load == kSlots) slot_load = 0;
  };
  fetch(kc, blk);
  fetch(vc, blk);

  // the tile's queries as mma A fragments: k-step t covers, for lane column c, the four values
  // d = (2c + t / 4) * 16 + (t % 4) * 4 + 0..3, so that a lane's K bytes are 16-byte runs
  uint32_t qa[8][4];
  int last_key[2];  // keys [0, last_key) are seen by rows g and g + 8
  float row_scale[2];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int r = r0 + g + 8 * hf;
    const bool on = r < p.rows;
    const int head = on ? r / p.Sq : 0, tok = on ? r - head * p.Sq : 0;
    const T* src = static_cast<const T*>(p.q) + b * p.qb + (hk * p.G + head) * p.qh + tok * p.qs;
    float f[32];
    float amax = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int d0 = (2 * c + (t >> 1)) * 16 + (t & 1) * 8;
      Row8<T> v;
      if (on && d0 < D) v.load(src + d0); else v.zero();
      v.get(f + 8 * t);
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) amax = fmaxf(amax, fabsf(f[e]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // 2^-e brings the row's largest value into [1, 2); rows of 0, infinity or subnormals keep their values
    const uint32_t ex = __float_as_uint(amax) >> 23;
    const float up = ex > 2 && ex < 253 ? __uint_as_float((254u - ex) << 23) : 1.f;
    row_scale[hf] = (ex > 2 && ex < 253 ? __uint_as_float(ex << 23) : 1.f) * p.scale_log2;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      qa[t][hf] = pack_pair(f[4 * t] * up, f[4 * t + 1] * up, __half());
      qa[t][hf + 2] = pack_pair(f[4 * t + 2] * up, f[4 * t + 3] * up, __half());
    }
    last_key[hf] = !on ? 0 : p.causal ? min(held, held - p.Sq + tok + 1) : held;
  }

  float o[16][4];
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  int slot = 0;
  for (; blk < blk_end; blk += kWarps) {
    const float kscale = ksc[blk], vscale = vsc[blk] * kLower;
    fetch(kc, blk + kWarps);  // into the slot of the last V read
    asm volatile("cp.async.wait_group 2;" ::: "memory");
    __syncwarp();
    const uint8_t* ks = ring + slot * kSlotBytes;
    if (++slot == kSlots) slot = 0;
    float s[8][4];
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
    // the eight token groups' products side by side: one after the other each would wait for the one before
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint4 u[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) u[t] = *reinterpret_cast<const uint4*>(ks + chunk_at(8 * t + g, 2 * c + i));
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const uint32_t w = (&u[t].x)[x];
          mma_f16(s[t], qa[4 * i + x], e4m3x2_to_f16x2(static_cast<uint16_t>(w)),
                  e4m3x2_to_f16x2(static_cast<uint16_t>(w >> 16)));
        }
    }
    const int key0 = blk * kCacheBlock + 2 * c;
    float alpha[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const float f = row_scale[hf] * kscale;
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& v = s[t][2 * hf + e];
          v = key0 + 8 * t + e < last_key[hf] ? v * f : -INFINITY;
          mx = fmaxf(mx, v);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[hf], mx);
      const float base = mn == -INFINITY ? 0.f : mn;
      alpha[hf] = ex2(m[hf] - base);
      m[hf] = mn;
      const float below = base - kRaise;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& v = s[t][2 * hf + e];
          v = ex2(v - below);
          sum += v;
        }
      l[hf] = l[hf] * alpha[hf] + sum * kLower;
    }
    // P as A fragments: the scores' layout is the A layout of k-steps of 16 tokens
    uint32_t pa[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      pa[t][0] = pack_pair(s[2 * t][0], s[2 * t][1], __half());
      pa[t][1] = pack_pair(s[2 * t][2], s[2 * t][3], __half());
      pa[t][2] = pack_pair(s[2 * t + 1][0], s[2 * t + 1][1], __half());
      pa[t][3] = pack_pair(s[2 * t + 1][2], s[2 * t + 1][3], __half());
    }
    __syncwarp();
    fetch(vc, blk + kWarps);  // into the slot of the K just read
    asm volatile("cp.async.wait_group 2;" ::: "memory");
    __syncwarp();
    const uint8_t* vs = ring + slot * kSlotBytes;
    if (++slot == kSlots) slot = 0;
    // lane group g holds the columns d = 16 g + j, one n-tile for each j
    uint4 vw[16];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        vw[4 * t + e] = *reinterpret_cast<const uint4*>(vs + chunk_at(16 * t + 2 * c + (e & 1) + 8 * (e >> 1), g));
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      float acc[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t w0 = (&vw[4 * t].x)[x], w1 = (&vw[4 * t + 1].x)[x];
        const uint32_t w2 = (&vw[4 * t + 2].x)[x], w3 = (&vw[4 * t + 3].x)[x];
        const uint32_t lo01 = byte_pair(w0, w1, 0x5140), hi01 = byte_pair(w0, w1, 0x7362);
        const uint32_t lo23 = byte_pair(w2, w3, 0x5140), hi23 = byte_pair(w2, w3, 0x7362);
        mma_f16(acc[0], pa[t], e4m3x2_to_f16x2(static_cast<uint16_t>(lo01)), e4m3x2_to_f16x2(static_cast<uint16_t>(lo23)));
        mma_f16(acc[1], pa[t], e4m3x2_to_f16x2(static_cast<uint16_t>(lo01 >> 16)),
                e4m3x2_to_f16x2(static_cast<uint16_t>(lo23 >> 16)));
        mma_f16(acc[2], pa[t], e4m3x2_to_f16x2(static_cast<uint16_t>(hi01)), e4m3x2_to_f16x2(static_cast<uint16_t>(hi23)));
        mma_f16(acc[3], pa[t], e4m3x2_to_f16x2(static_cast<uint16_t>(hi01 >> 16)),
                e4m3x2_to_f16x2(static_cast<uint16_t>(hi23 >> 16)));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * x + j][e] = fmaf(o[4 * x + j][e], alpha[e >> 1], acc[j][e] * vscale);
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
    l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
  }
  // ---- join the warps: their sums go to shared memory (16 x 128 fp32 each, in the warp's own ring)
  __syncwarp();
  float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int j = 0; j < 16; ++j)  // accumulator (row g / g + 8, n = 2c, 2c + 1) of n-tile j: columns 16 n + j
#pragma unroll
    for (int e = 0; e < 4; ++e) mine[(g + 8 * (e >> 1)) * 128 + 16 * (2 * c + (e & 1)) + j] = o[j][e];
  if (c == 0) {
    st_m[warp][g] = m[0];
    st_m[warp][g + 8] = m[1];
    st_l[warp][g] = l[0];
    st_l[warp][g + 8] = l[1];
  }
  __syncthreads();
  const int tpr = kAttnThreads / 16;  // threads of a row
  const int r = threadIdx.x / tpr;
  if (r0 + r >= p.rows) return;
  float mm = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, st_m[w][r]);
  const float base = mm == -INFINITY ? 0.f : mm;
  float f[kWarps], ll = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    f[w] = ex2(st_m[w][r] - base);
    ll += f[w] * st_l[w][r];
  }
  const int head = (r0 + r) / p.Sq, tok = (r0 + r) - head * p.Sq;
  const int h = hk * p.G + head;
  const float inv = p.splits > 1 ? 1.f : (ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll));
  float* part = nullptr;
  if (p.splits > 1) {
    const long long row = blockIdx.x * p.total + (static_cast<long long>(b) * p.H + h) * p.Sq + tok;
    part = p.part + row * D;
    if (threadIdx.x % tpr == 0)
      reinterpret_cast<float2*>(p.part + p.splits * p.total * D)[row] = make_float2(mm, ll);
  }
  T* out = static_cast<T*>(p.o) + b * p.ob + h * p.oh + tok * p.os;
  for (int d0 = 8 * (threadIdx.x % tpr); d0 < D; d0 += 8 * tpr) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        v[e] = fmaf(f[w], reinterpret_cast<const float*>(smem + w * kSlots * kSlotBytes)[r * 128 + d0 + e], v[e]);
      v[e] *= inv;
    }
    if (part) {
      reinterpret_cast<float4*>(part + d0)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(part + d0)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      Row8<T>::store(out + d0, v);
    }
  }
}

// Joins the splits of a row: o = sum 2^(m_s - m) o_s / sum 2^(m_s - m) l_s, always in the splits' order.  A CTA a row: a
// thread holds a column, and the splits' weights are worked out once.
template <typename T>
__global__ void __launch_bounds__(128) cache_join_kernel(const AttnParams p) {
  __shared__ float weight[kMostSplits];
  after_previous();
  const long long row = blockIdx.x;
  const int D = p.c.D, d = threadIdx.x;
  if (threadIdx.x < 32) {
    const float2* ml = reinterpret_cast<const float2*>(p.part + p.splits * p.total * D) + row;
    float m = -INFINITY;
    for (int s = threadIdx.x; s < p.splits; s += 32) m = fmaxf(m, ml[s * p.total].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = threadIdx.x; s < p.splits; s += 32) {
      const float2 v = ml[s * p.total];
      const float f = ex2(v.x - base);
      weight[s] = f;
      l = fmaf(f, v.y, l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    for (int s = threadIdx.x; s < p.splits; s += 32) weight[s] *= inv;
  }
  __syncthreads();
  if (d >= D) return;
  const float* src = p.part + row * D + d;
  float v = 0.f;
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) v = fmaf(weight[s], src[s * p.total * D], v);
  const int tok = static_cast<int>(row % p.Sq);
  const long long bh = row / p.Sq;
  const int h = static_cast<int>(bh % p.H);
  store1(static_cast<T*>(p.o) + (bh / p.H) * p.ob + h * p.oh + tok * p.os + d, v);
}

template <typename T>
int attention(const CacheAttnArgs& a, cudaStream_t stream) {
  AttnParams p = {};
  p.c = a.c;
  p.q = a.q.p; p.qb = a.q.sb; p.qh = a.q.sh; p.qs = a.q.ss;
  p.o = a.o.p; p.ob = a.o.sb; p.oh = a.o.sh; p.os = a.o.ss;
  p.H = a.H;
  p.G = a.H / a.c.Hk;
  p.Sq = a.Sq;
  p.rows = p.G * a.Sq;
  p.row_tiles = (p.rows + 15) / 16;
  p.splits = a.splits;
  p.causal = a.causal;
  p.scale_log2 = a.sm_scale * 1.4426950408889634f;
  p.part = a.part;
  p.total = static_cast<long long>(a.c.B) * a.H * a.Sq;
  auto* kernel = a.c.D == 128 ? cache_attn_kernel<T, true> : cache_attn_kernel<T, false>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kAttnSmem) != cudaSuccess)
    return BSA_ERR_CUDA;
  if (launch_behind(kernel, dim3(a.splits, a.c.B * a.c.Hk * p.row_tiles), dim3(kAttnThreads), kAttnSmem, stream, p) !=
      cudaSuccess)
    return BSA_ERR_CUDA;
  if (a.splits > 1 && launch_behind(cache_join_kernel<T>, dim3(static_cast<unsigned>(p.total)), dim3(128), 0, stream, p) !=
                          cudaSuccess)
    return BSA_ERR_CUDA;
  return BSA_OK;
}

template <typename P>
void set_pair(P& p, const Tensor4& k, const Tensor4& v) {
  p.x[0] = k.p; p.sb[0] = k.sb; p.sh[0] = k.sh; p.ss[0] = k.ss;
  p.x[1] = v.p; p.sb[1] = v.sb; p.sh[1] = v.sh; p.ss[1] = v.ss;
}

}  // namespace kv8

int launch_cache_append(const AppendArgs& a, cudaStream_t stream) {
  kv8::AppendParams p = {};
  p.c = a.c;
  kv8::set_pair(p, a.k, a.v);
  p.counts = a.counts;
  p.n = a.n;
  p.blocks = (a.n + kCacheBlock - 2) / kCacheBlock + 1;  // from any place in a block
  const int cluster = (p.blocks * a.c.Hk * 2 + kv8::kSide - 1) / kv8::kSide;
  if (p.blocks <= kv8::kMostCluster * kv8::kSide && cluster <= kv8::kMostCluster) {
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.c.B * cluster);
    cfg.blockDim = dim3(kv8::kSide * kv8::kAppendThreads);
    cfg.stream = stream;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    auto* few = a.dtype == BSA_DTYPE_F16 ? kv8::append_few_kernel<__half> : kv8::append_few_kernel<__nv_bfloat16>;
    return cudaLaunchKernelEx(&cfg, few, p, cluster) == cudaSuccess ? BSA_OK : BSA_ERR_CUDA;
  }
  const dim3 grid(p.blocks, a.c.B * a.c.Hk, 2);
  auto* kernel = a.dtype == BSA_DTYPE_F16 ? kv8::append_kernel<__half> : kv8::append_kernel<__nv_bfloat16>;
  if (launch_behind(kernel, grid, dim3(kv8::kAppendThreads), 0, stream, p) != cudaSuccess ||
      launch_behind(kv8::advance_kernel, dim3(1), dim3(128), 0, stream, a.c.lengths, a.counts, a.n, a.c.cap, a.c.B) !=
          cudaSuccess)
    return BSA_ERR_CUDA;
  return BSA_OK;
}

int launch_cache_unpack(const UnpackArgs& a, cudaStream_t stream) {
  kv8::UnpackParams p = {};
  p.c = a.c;
  kv8::set_pair(p, a.k, a.v);
  p.out[0] = a.ko;
  p.out[1] = a.vo;
  p.n = a.n;
  p.rows = a.rows;
  p.zeros = a.zeros;
  const dim3 grid((a.rows + 63) / 64, a.c.B * a.c.Hk, 2);
  if (a.dtype == BSA_DTYPE_F16)
    kv8::unpack_kernel<__half><<<grid, 256, 0, stream>>>(p);
  else
    kv8::unpack_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? BSA_OK : BSA_ERR_CUDA;
}

int launch_cache_attention(const CacheAttnArgs& a, cudaStream_t stream) {
  return a.dtype == BSA_DTYPE_F16 ? kv8::attention<__half>(a, stream) : kv8::attention<__nv_bfloat16>(a, stream);
}

int cache_device_error(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, kv8::g_cache_err, sizeof(int)) != cudaSuccess) return BSA_ERR_CUDA;
  if (clear && v) {
    const int z = 0;
    cudaMemcpyToSymbol(kv8::g_cache_err, &z, sizeof(int));
  }
  return v;
}

}  // namespace bsa
