// C ABI of the operators around dense attention (declared in include/bsa_b200.h): argument checks and
// launches.  As everywhere in this library, a call that returns an argument error has launched nothing, and
// nothing allocates device memory.
#include <climits>
#include <cmath>
#include "bsa_dense.h"

namespace {

using bsa::set_error;
using bsa::Tensor4;

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

Tensor4 tensor(const void* p, const int64_t* st) {
  Tensor4 t;
  t.p = const_cast<void*>(p);
  if (st) {
    t.sb = st[0];
    t.sh = st[1];
    t.ss = st[2];
  }
  return t;
}

constexpr int kMostRows = 1 << 30;  // tokens of a sequence: places and tile borders stay within 32 bits

int elt(int dtype) { return dtype == BSA_DTYPE_F32 ? 4 : 2; }

// base and strides (of axes that are walked) in multiples of 16 bytes
int check_tensor(const Tensor4& t, int dtype, int B, int H, int S, const char* name) {
  if (!t.p) return set_error(BSA_ERR_ARG, "%s: null pointer", name);
  const int e = elt(dtype);
  if (!aligned(t.p, 16) || (S > 1 && (t.ss * e) % 16) || (H > 1 && (t.sh * e) % 16) || (B > 1 && (t.sb * e) % 16))
    return set_error(BSA_ERR_ALIGN, "%s: base and strides must be multiples of 16 bytes", name);
  return BSA_OK;
}

int check_head_dim(int D) {
  if (D <= 0 || D % 8 || D > 128) return set_error(BSA_ERR_SHAPE, "head_dim D=%d must be a multiple of 8 and <= 128", D);
  return BSA_OK;
}

int check_16bit(int dtype) {
  if (dtype != BSA_DTYPE_F16 && dtype != BSA_DTYPE_BF16)
    return set_error(BSA_ERR_DTYPE, "unsupported dtype code %d (fp16 or bf16)", dtype);
  return BSA_OK;
}

// The kernels take sm_scale log2(e), twice its quotient by the cap, and cap log2(e) in fp32
int check_scales(float sm_scale, float softcap) {
  if (!(sm_scale > 0.f) || std::isinf(sm_scale)) return set_error(BSA_ERR_ARG, "sm_scale must be positive and finite");
  if (!(softcap >= 0.f) || std::isinf(softcap)) return set_error(BSA_ERR_ARG, "softcap must be finite and >= 0");
  const float log2e = 1.4426950408889634f, scale_log2 = sm_scale * log2e;
  if (std::isinf(scale_log2) || (softcap > 0.f && (std::isinf(2.f * scale_log2 / softcap) || std::isinf(softcap * log2e))))
    return set_error(BSA_ERR_ARG, "sm_scale %g with softcap %g is out of fp32's range", sm_scale, softcap);
  return BSA_OK;
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaGetLastError();
  return sms;
}

int launched(int rc, const char* what) {
  if (rc == BSA_ERR_CUDA) return set_error(rc, "%s launch: %s", what, cudaGetErrorString(cudaGetLastError()));
  return rc;
}

// ------------------------------------------------------------------ q/k norm + rotary positions
int norm_rope_plan(bsa::NormRopeArgs& a, int dtype, int w_dtype, int B, int S, int D, float eps, const float* rope,
                   int rope_dt, int rope_dh, int rope_dw, int rope_T, int rope_H, int rope_W, int start) {
  if (dtype != BSA_DTYPE_F32 && dtype != BSA_DTYPE_F16 && dtype != BSA_DTYPE_BF16)
    return set_error(BSA_ERR_DTYPE, "unsupported dtype code %d", dtype);
  if (w_dtype != BSA_DTYPE_F32 && w_dtype != BSA_DTYPE_F16 && w_dtype != BSA_DTYPE_BF16)
    return set_error(BSA_ERR_DTYPE, "unsupported weight dtype code %d", w_dtype);
  if (B <= 0 || S <= 0) return set_error(BSA_ERR_SHAPE, "empty tensor");
  if (S > INT_MAX - 64 || static_cast<long long>(B) * (S / 16 + 1) >= INT_MAX)  // a tile's rows go past the last token
    return set_error(BSA_ERR_SHAPE, "too many tokens for one launch");
  int rc = check_head_dim(D);
  if (rc) return rc;
  if (!(eps >= 0.f)) return set_error(BSA_ERR_ARG, "norm eps must be >= 0");
  if (rope) {
    if (rope_dt + rope_dh + rope_dw != D || (rope_dt | rope_dh | rope_dw) & 1 || rope_dt < 0 || rope_dh < 0 ||
        rope_dw < 0)
      return set_error(BSA_ERR_SHAPE, "rope dims (%d, %d, %d) must be even and sum to D=%d", rope_dt, rope_dh, rope_dw, D);
    if (rope_T <= 0 || rope_H <= 0 || rope_W <= 0 || start < 0 ||
        static_cast<long long>(rope_H) * rope_W > INT_MAX ||
        static_cast<long long>(start) + S > static_cast<long long>(rope_T) * rope_H * rope_W)
      return set_error(BSA_ERR_SHAPE, "rope grid (%d, %d, %d) does not cover tokens %d to %lld", rope_T, rope_H, rope_W,
                       start, static_cast<long long>(start) + S);
    if (static_cast<long long>(start) + S > INT_MAX)
      return set_error(BSA_ERR_SHAPE, "places %d to %lld do not fit 32 bits", start, static_cast<long long>(start) + S);
    // an axis's cosines are indexed in 32 bits
    const int n[3] = {rope_T, rope_H, rope_W}, d[3] = {rope_dt, rope_dh, rope_dw};
    for (int i = 0; i < 3; ++i)
      if (static_cast<long long>(n[i]) * (d[i] / 2) > INT_MAX)
        return set_error(BSA_ERR_SHAPE, "a rope table of %d places of %d angles is too large", n[i], d[i] / 2);
  }
  a.dtype = dtype; a.w_dtype = w_dtype; a.B = B; a.S = S; a.D = D; a.eps = eps;
  a.rope = rope; a.dt = rope_dt; a.dh = rope_dh; a.dw = rope_dw;
  a.gT = rope_T; a.gH = rope_H; a.gW = rope_W; a.start = start;
  return BSA_OK;
}

// ------------------------------------------------------------------ cache
int cache_view(bsa::CacheView& c, void* k_codes, float* k_scale, void* v_codes, float* v_scale, int32_t* lengths, int B,
               int Hk, int capacity, int D) {
  if (!k_codes || !k_scale || !v_codes || !v_scale || !lengths) return set_error(BSA_ERR_ARG, "null pointer");
  if (B <= 0 || Hk <= 0 || capacity <= 0) return set_error(BSA_ERR_SHAPE, "empty cache");
  if (capacity % bsa::kCacheBlock)
    return set_error(BSA_ERR_SHAPE, "cache capacity %d must be a multiple of %d", capacity, bsa::kCacheBlock);
  int rc = check_head_dim(D);
  if (rc) return rc;
  if (static_cast<long long>(B) * Hk > 65535) return set_error(BSA_ERR_SHAPE, "more than 65535 cache heads");
  if (!aligned(k_codes, 16) || !aligned(v_codes, 16))
    return set_error(BSA_ERR_ALIGN, "cache codes must be 16-byte aligned");
  c.k = static_cast<uint8_t*>(k_codes);
  c.v = static_cast<uint8_t*>(v_codes);
  c.ks = k_scale; c.vs = v_scale; c.lengths = lengths;
  c.B = B; c.Hk = Hk; c.cap = capacity; c.D = D;
  return BSA_OK;
}

// Splits of the cache along its tokens: about three CTAs for each of an SM's two places, so that ragged lengths even
// out, and at least two blocks for each of a CTA's four warps (8 sequences of 16 to 32 thousand tokens: 3 for each SM
// 79 us, 6 79, 8 83, 12 91).
int cache_splits(int sms, int B, int Hk, int rows, int capacity) {
  const long long units = static_cast<long long>(B) * Hk * ((rows + 15) / 16);
  const long long want = (6ll * sms + units - 1) / units;
  long long most = (capacity / bsa::kCacheBlock + 7) / 8;
  if (most > bsa::kMostSplits) most = bsa::kMostSplits;
  return static_cast<int>(want < most ? want : (most > 1 ? most : 1));
}

// ------------------------------------------------------------------ dense attention
int dense_plan(bsa::DenseArgs& a, const void* q, const void* k, const void* v, int dtype, int B, int H, int Hk, int Sq,
               int Sk, int D, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
               const int32_t* ranges, const int32_t* table, int ranges_batch, float sm_scale, float softcap) {
  if (!q_strides || !k_strides || !v_strides) return set_error(BSA_ERR_ARG, "null pointer");
  int rc = check_16bit(dtype);
  if (rc) return rc;
  if (B <= 0 || H <= 0 || Hk <= 0 || Sq <= 0 || Sk <= 0) return set_error(BSA_ERR_SHAPE, "empty tensor");
  if (Sq > kMostRows || Sk > kMostRows) return set_error(BSA_ERR_SHAPE, "more than %d tokens", kMostRows);
  if (H % Hk) return set_error(BSA_ERR_SHAPE, "%d query heads are no multiple of %d key heads", H, Hk);
  if ((rc = check_head_dim(D))) return rc;
  if ((rc = check_scales(sm_scale, softcap))) return rc;
  if ((ranges == nullptr) != (table == nullptr)) return set_error(BSA_ERR_ARG, "ranges come with their table");
  if (ranges && ranges_batch != 1 && ranges_batch != B)
    return set_error(BSA_ERR_SHAPE, "ranges of %d batch entries for a batch of %d", ranges_batch, B);
  if (!aligned(ranges, 8) || !aligned(table, 16)) return set_error(BSA_ERR_ALIGN, "ranges: 8 bytes, table: 16 bytes");
  a.q = tensor(q, q_strides);
  a.k = tensor(k, k_strides);
  a.v = tensor(v, v_strides);
  if ((rc = check_tensor(a.q, dtype, B, H, Sq, "q"))) return rc;
  if ((rc = check_tensor(a.k, dtype, B, Hk, Sk, "k"))) return rc;
  if ((rc = check_tensor(a.v, dtype, B, Hk, Sk, "v"))) return rc;
  a.dtype = dtype; a.B = B; a.H = H; a.Hk = Hk; a.Sq = Sq; a.Sk = Sk; a.D = D;
  a.ranges = reinterpret_cast<const int2*>(ranges);
  a.table = reinterpret_cast<const int4*>(table);
  a.Bm = ranges ? ranges_batch : 1;
  a.sm_scale = sm_scale;
  a.softcap = softcap;
  return BSA_OK;
}

}  // namespace

extern "C" {

int bsa_norm_rope(const void* x0, const int64_t* x0_strides, int H0, const void* w0, void* y0, const void* x1,
                  const int64_t* x1_strides, int H1, const void* w1, void* y1, int dtype, int w_dtype, int B, int S,
                  int D, float eps, const float* rope, int rope_dt, int rope_dh, int rope_dw, int rope_T, int rope_H,
                  int rope_W, int start, void* stream) {
  bsa::NormRopeArgs a;
  int rc = norm_rope_plan(a, dtype, w_dtype, B, S, D, eps, rope, rope_dt, rope_dh, rope_dw, rope_T, rope_H, rope_W, start);
  if (rc) return rc;
  if (!x0_strides || !y0 || (x1 && (!x1_strides || !y1))) return set_error(BSA_ERR_ARG, "null pointer");
  a.sides = x1 ? 2 : 1;
  for (int i = 0; i < a.sides; ++i) {
    bsa::NormRopeSide& s = a.side[i];
    s.x = i ? tensor(x1, x1_strides) : tensor(x0, x0_strides);
    s.H = i ? H1 : H0;
    s.w = i ? w1 : w0;
    s.y = i ? y1 : y0;
    if (s.H <= 0) return set_error(BSA_ERR_SHAPE, "empty tensor");
    if ((rc = check_tensor(s.x, dtype, B, s.H, S, i ? "x1" : "x0"))) return rc;
    if (!aligned(s.y, 16)) return set_error(BSA_ERR_ALIGN, "outputs must be 16-byte aligned");
  }
  return launched(bsa::launch_norm_rope(a, static_cast<cudaStream_t>(stream)), "norm + rope");
}

int64_t bsa_norm_rope_backward_scratch_bytes(int H0, int H1, int D) {
  if (H0 <= 0 || H1 < 0 || D <= 0) return 0;
  return static_cast<int64_t>(bsa::norm_rope_partials((H0 + 7) / 8 + (H1 + 7) / 8)) * D *
         static_cast<int64_t>(sizeof(float));
}

int bsa_norm_rope_backward(const void* x0, const int64_t* x0_strides, const void* g0, const int64_t* g0_strides, int H0,
                           const void* w0, void* dx0, float* dw0, const void* x1, const int64_t* x1_strides,
                           const void* g1, const int64_t* g1_strides, int H1, const void* w1, void* dx1, float* dw1,
                           int dtype, int w_dtype, int B, int S, int D, float eps, const float* rope, int rope_dt,
                           int rope_dh, int rope_dw, int rope_T, int rope_H, int rope_W, int start, void* scratch,
                           void* stream) {
  bsa::NormRopeArgs a;
  int rc = norm_rope_plan(a, dtype, w_dtype, B, S, D, eps, rope, rope_dt, rope_dh, rope_dw, rope_T, rope_H, rope_W, start);
  if (rc) return rc;
  if (!x0_strides || !g0_strides || !dx0 || (x1 && (!x1_strides || !g1_strides || !dx1)))
    return set_error(BSA_ERR_ARG, "null pointer");
  if (!aligned(scratch, 4)) return set_error(BSA_ERR_ALIGN, "scratch must be 4-byte aligned");
  if ((dw0 || dw1) && !scratch) return set_error(BSA_ERR_ARG, "weight gradients need scratch");
  a.sides = x1 ? 2 : 1;
  for (int i = 0; i < a.sides; ++i) {
    bsa::NormRopeSide& s = a.side[i];
    s.x = i ? tensor(x1, x1_strides) : tensor(x0, x0_strides);
    s.g = i ? tensor(g1, g1_strides) : tensor(g0, g0_strides);
    s.H = i ? H1 : H0;
    s.w = i ? w1 : w0;
    s.y = i ? dx1 : dx0;
    s.dw = i ? dw1 : dw0;
    if (s.H <= 0) return set_error(BSA_ERR_SHAPE, "empty tensor");
    if (s.dw && !s.w) return set_error(BSA_ERR_ARG, "a weight gradient without a weight");
    if ((rc = check_tensor(s.x, dtype, B, s.H, S, i ? "x1" : "x0"))) return rc;
    if ((rc = check_tensor(s.g, dtype, B, s.H, S, i ? "g1" : "g0"))) return rc;
    if (!aligned(s.y, 16)) return set_error(BSA_ERR_ALIGN, "outputs must be 16-byte aligned");
  }
  a.partial = dw0 || dw1 ? static_cast<float*>(scratch) : nullptr;
  return launched(bsa::launch_norm_rope_backward(a, static_cast<cudaStream_t>(stream)), "norm + rope backward");
}

int bsa_attention_ranges(int32_t* ranges, int32_t* table, int batch, int Sq, int Sk, const int32_t* given, int causal,
                         int prefix, const int32_t* prefixes, const int32_t* q_offsets, const int32_t* k_offsets,
                         int documents, const int32_t* q_lengths, const int32_t* k_lengths, int k_add, void* stream) {
  if (!ranges || !table) return set_error(BSA_ERR_ARG, "null pointer");
  if (batch <= 0 || Sq <= 0 || Sk < 0) return set_error(BSA_ERR_SHAPE, "empty ranges");
  if (Sq > kMostRows || Sk > kMostRows) return set_error(BSA_ERR_SHAPE, "more than %d tokens", kMostRows);
  if (static_cast<long long>(batch) * ((Sq + 127) / 128) > INT_MAX)
    return set_error(BSA_ERR_SHAPE, "too many rows for one launch");
  if ((q_offsets == nullptr) != (k_offsets == nullptr)) return set_error(BSA_ERR_ARG, "q_offsets come with k_offsets");
  if (q_offsets && documents <= 0) return set_error(BSA_ERR_SHAPE, "no documents");
  if (q_offsets && (q_lengths || k_lengths)) return set_error(BSA_ERR_ARG, "documents or lengths, not both");
  if (prefix < 0) return set_error(BSA_ERR_ARG, "prefix must be >= 0");
  if (!aligned(ranges, 8) || !aligned(given, 8) || !aligned(table, 16))
    return set_error(BSA_ERR_ALIGN, "ranges: 8 bytes, table: 16 bytes");
  bsa::RangesArgs a;
  a.ranges = reinterpret_cast<int2*>(ranges);
  a.table = reinterpret_cast<int4*>(table);
  a.given = reinterpret_cast<const int2*>(given);
  a.Bm = batch; a.Sq = Sq; a.Sk = Sk;
  a.causal = causal; a.prefix = prefix; a.prefixes = prefixes;
  a.q_offsets = q_offsets; a.k_offsets = k_offsets; a.docs = documents;
  a.q_lengths = q_lengths; a.k_lengths = k_lengths; a.k_add = k_add;
  return launched(bsa::launch_ranges(a, static_cast<cudaStream_t>(stream)), "attention ranges");
}

int64_t bsa_masked_attention_scratch_bytes(int B, int H, int Sq, int Sk, int D) {
  if (B <= 0 || H <= 0 || Sq <= 0 || Sk <= 0 || D <= 0) return 0;
  const int splits = bsa::dense_pick_splits(sm_count(), B, H, Sq, Sk);
  return splits > 1 ? static_cast<int64_t>(splits) * B * H * Sq * (D + 1) * static_cast<int64_t>(sizeof(float)) : 0;
}

int bsa_masked_attention(const void* q, const void* k, const void* v, int dtype, int B, int H, int Hk, int Sq, int Sk,
                         int D, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                         const int32_t* ranges, const int32_t* table, int ranges_batch, float sm_scale, float softcap,
                         void* out, const int64_t* out_strides, void* out_rest, float* lse, void* scratch,
                         void* stream) {
  bsa::DenseArgs a;
  int rc = dense_plan(a, q, k, v, dtype, B, H, Hk, Sq, Sk, D, q_strides, k_strides, v_strides, ranges, table,
                      ranges_batch, sm_scale, softcap);
  if (rc) return rc;
  if (!out_strides) return set_error(BSA_ERR_ARG, "null pointer");
  a.o = tensor(out, out_strides);
  if ((rc = check_tensor(a.o, dtype, B, H, Sq, "out"))) return rc;
  if (!aligned(out_rest, 16)) return set_error(BSA_ERR_ALIGN, "out_rest must be 16-byte aligned");
  a.o_lo = out_rest;
  a.lse = lse;
  const int sms = sm_count();
  a.splits = bsa::dense_pick_splits(sms, B, H, Sq, Sk);
  if (a.splits > 1) {
    if (!scratch) return set_error(BSA_ERR_ARG, "scratch is required (bsa_masked_attention_scratch_bytes)");
    if (!aligned(scratch, 16)) return set_error(BSA_ERR_ALIGN, "scratch must be 16-byte aligned");
    a.part = static_cast<float*>(scratch);
  }
  return bsa::launch_dense(a, sms, static_cast<cudaStream_t>(stream));
}

int64_t bsa_masked_attention_backward_scratch_bytes(int B, int H, int Sq, int ranges_batch) {
  if (B <= 0 || H <= 0 || Sq <= 0 || ranges_batch < 0) return 0;
  return bsa::dense_backward_stats_bytes(B, H, Sq, ranges_batch);
}

int bsa_masked_attention_backward(const void* q, const void* k, const void* v, const void* out, const void* out_rest,
                                  const void* grad, const float* lse, int dtype, int B, int H, int Hk, int Sq, int Sk, int D,
                                  const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                  const int64_t* out_strides, const int64_t* grad_strides, const int32_t* ranges,
                                  const int32_t* table, int ranges_batch, float sm_scale, float softcap, void* dq,
                                  void* dk, void* dv, void* scratch, void* stream) {
  bsa::DenseArgs a;
  int rc = dense_plan(a, q, k, v, dtype, B, H, Hk, Sq, Sk, D, q_strides, k_strides, v_strides, ranges, table,
                      ranges_batch, sm_scale, softcap);
  if (rc) return rc;
  if (!out_strides || !grad_strides || !out_rest || !lse || !scratch || (dk == nullptr) != (dv == nullptr))
    return set_error(BSA_ERR_ARG, "null pointer");
  a.o = tensor(out, out_strides);
  a.g = tensor(grad, grad_strides);
  if ((rc = check_tensor(a.o, dtype, B, H, Sq, "out"))) return rc;
  if ((rc = check_tensor(a.g, dtype, B, H, Sq, "gradient of out"))) return rc;
  a.o_lo = const_cast<void*>(out_rest);
  if (!aligned(out_rest, 16) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16) || !aligned(scratch, 16))
    return set_error(BSA_ERR_ALIGN, "out_rest, gradients and scratch must be 16-byte aligned");
  const int64_t qs[3] = {static_cast<int64_t>(H) * Sq * D, static_cast<int64_t>(Sq) * D, D};
  const int64_t ks[3] = {static_cast<int64_t>(Hk) * Sk * D, static_cast<int64_t>(Sk) * D, D};
  a.dq = tensor(dq, qs);
  a.dk = tensor(dk, ks);
  a.dv = tensor(dv, ks);
  a.lse = const_cast<float*>(lse);
  a.stats = static_cast<float*>(scratch);
  return bsa::launch_dense_backward(a, sm_count(), static_cast<cudaStream_t>(stream));
}

int bsa_kv8_append(void* k_codes, float* k_scale, void* v_codes, float* v_scale, int32_t* lengths, int B, int Hk,
                   int capacity, int D, const void* k, const void* v, int dtype, int n, const int64_t* k_strides,
                   const int64_t* v_strides, const int32_t* counts, void* stream) {
  bsa::AppendArgs a;
  int rc = cache_view(a.c, k_codes, k_scale, v_codes, v_scale, lengths, B, Hk, capacity, D);
  if (rc) return rc;
  if ((rc = check_16bit(dtype))) return rc;
  if (!k_strides || !v_strides) return set_error(BSA_ERR_ARG, "null pointer");
  if (n <= 0 || n > capacity) return set_error(BSA_ERR_SHAPE, "%d new tokens for a capacity of %d", n, capacity);
  a.k = tensor(k, k_strides);
  a.v = tensor(v, v_strides);
  if ((rc = check_tensor(a.k, dtype, B, Hk, n, "k"))) return rc;
  if ((rc = check_tensor(a.v, dtype, B, Hk, n, "v"))) return rc;
  a.counts = counts;
  a.dtype = dtype;
  a.n = n;
  return launched(bsa::launch_cache_append(a, static_cast<cudaStream_t>(stream)), "cache append");
}

int bsa_kv8_unpack(void* k_codes, float* k_scale, void* v_codes, float* v_scale, int32_t* lengths, int B, int Hk,
                   int capacity, int D, const void* k, const void* v, int dtype, int n, const int64_t* k_strides,
                   const int64_t* v_strides, void* k_out, void* v_out, int rows, int zeros, void* stream) {
  bsa::UnpackArgs a;
  int rc = cache_view(a.c, k_codes, k_scale, v_codes, v_scale, lengths, B, Hk, capacity, D);
  if (rc) return rc;
  if ((rc = check_16bit(dtype))) return rc;
  if (!k_out || !v_out) return set_error(BSA_ERR_ARG, "null pointer");
  if (rows <= 0 || rows > (1 << 26)) return set_error(BSA_ERR_SHAPE, "%d rows to unpack", rows);
  if (n < 0 || (n > 0 && (!k_strides || !v_strides))) return set_error(BSA_ERR_ARG, "null pointer");
  if (n > 0) {
    a.k = tensor(k, k_strides);
    a.v = tensor(v, v_strides);
    if ((rc = check_tensor(a.k, dtype, B, Hk, n, "k"))) return rc;
    if ((rc = check_tensor(a.v, dtype, B, Hk, n, "v"))) return rc;
  }
  if (!aligned(k_out, 16) || !aligned(v_out, 16)) return set_error(BSA_ERR_ALIGN, "outputs must be 16-byte aligned");
  a.dtype = dtype; a.n = n; a.ko = k_out; a.vo = v_out; a.rows = rows; a.zeros = zeros;
  return launched(bsa::launch_cache_unpack(a, static_cast<cudaStream_t>(stream)), "cache unpack");
}

int64_t bsa_kv8_attention_scratch_bytes(int B, int H, int Hk, int Sq, int capacity, int D) {
  if (B <= 0 || H <= 0 || Hk <= 0 || Sq <= 0 || capacity <= 0 || D <= 0 || H % Hk) return 0;
  const int splits = cache_splits(sm_count(), B, Hk, H / Hk * Sq, capacity);
  return splits > 1 ? static_cast<int64_t>(splits) * B * H * Sq * (D + 2) * static_cast<int64_t>(sizeof(float)) : 0;
}

int bsa_kv8_attention(const void* q, int dtype, int B, int H, int Sq, const int64_t* q_strides, const void* k_codes,
                      const float* k_scale, const void* v_codes, const float* v_scale, const int32_t* lengths, int Hk,
                      int capacity, int D, int causal, float sm_scale, void* out, const int64_t* out_strides,
                      void* scratch, void* stream) {
  bsa::CacheAttnArgs a;
  int rc = cache_view(a.c, const_cast<void*>(k_codes), const_cast<float*>(k_scale), const_cast<void*>(v_codes),
                      const_cast<float*>(v_scale), const_cast<int32_t*>(lengths), B, Hk, capacity, D);
  if (rc) return rc;
  if ((rc = check_16bit(dtype))) return rc;
  if (!q_strides || !out_strides) return set_error(BSA_ERR_ARG, "null pointer");
  if (H <= 0 || Sq <= 0) return set_error(BSA_ERR_SHAPE, "empty tensor");
  if (H % Hk) return set_error(BSA_ERR_SHAPE, "%d query heads are no multiple of %d key heads", H, Hk);
  if ((rc = check_scales(sm_scale, 0.f))) return rc;
  const long long rows = static_cast<long long>(H / Hk) * Sq;
  if (rows > INT_MAX || static_cast<long long>(B) * Hk * ((rows + 15) / 16) > 65535)
    return set_error(BSA_ERR_SHAPE, "too many query rows for the cache's few-row kernel");
  a.q = tensor(q, q_strides);
  a.o = tensor(out, out_strides);
  if ((rc = check_tensor(a.q, dtype, B, H, Sq, "q"))) return rc;
  if ((rc = check_tensor(a.o, dtype, B, H, Sq, "out"))) return rc;
  a.dtype = dtype; a.H = H; a.Sq = Sq; a.causal = causal; a.sm_scale = sm_scale;
  a.splits = cache_splits(sm_count(), B, Hk, static_cast<int>(rows), capacity);
  if (a.splits > 1) {
    if (!scratch) return set_error(BSA_ERR_ARG, "scratch is required (bsa_kv8_attention_scratch_bytes)");
    if (!aligned(scratch, 16)) return set_error(BSA_ERR_ALIGN, "scratch must be 16-byte aligned");
    a.part = static_cast<float*>(scratch);
  }
  return launched(bsa::launch_cache_attention(a, static_cast<cudaStream_t>(stream)), "cache attention");
}

}  // extern "C"
