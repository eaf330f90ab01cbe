// Key intervals of the dense attention: row i of a batch entry sees the keys [lo, hi).
//
// Document, padding, causal and prefix masks over contiguous documents all have this form.  With a document's
// qn queries and kn keys, query i' of it stands at key place a = i' + kn - qn (the last query lines up with
// the last key), and sees
//   causal: a + 1 keys,  else kn keys;   a < prefix: the prefix and nothing else;   a >= prefix: at least it
// clamped to the document's keys.  A row outside every document, or behind its entry's length, sees none.
// Two ints for a row replace a mask of Sq x Sk truth values, and the table of 128-row tiles tells the
// attention kernels which key tiles a query tile reaches and which of those need no comparison.
#include <climits>
#include "bsa_dense.h"

namespace bsa {
namespace ranges {

constexpr int kTile = 128;

struct Params {
  int2* ranges;
  int4* table;
  const int2* given;
  const int32_t *prefixes, *q_offsets, *k_offsets, *q_lengths, *k_lengths;
  int Sq, Sk, causal, prefix, docs, k_add, tiles;
};

__global__ void __launch_bounds__(kTile) ranges_kernel(const Params p) {
  let_next_start();
  const int b = blockIdx.x / p.tiles;
  const int tile = blockIdx.x - b * p.tiles;
  const int i = tile * kTile + threadIdx.x;
  const bool row = i < p.Sq;
  int lo = 0, hi = 0;
  if (row) {
    if (p.given) {
      const int2 r = p.given[static_cast<long long>(b) * p.Sq + i];
      lo = min(max(r.x, 0), p.Sk);
      hi = min(max(r.y, 0), p.Sk);
    } else {
      int qs = 0, qe = p.Sq, ks = 0, ke = p.Sk, doc = b;
      if (p.q_offsets) {
        // the last document that starts at or before row i (an empty one before it never holds the row)
        int lower = 0, upper = p.docs;  // q_offsets[lower] <= i < q_offsets[upper] where there is such a pair
        while (upper - lower > 1) {
          const int mid = (lower + upper) >> 1;
          if (p.q_offsets[mid] <= i) lower = mid; else upper = mid;
        }
        doc = lower;
        qs = p.q_offsets[doc];
        qe = p.q_offsets[doc + 1];
        ks = min(max(p.k_offsets[doc], 0), p.Sk);
        ke = min(max(p.k_offsets[doc + 1], ks), p.Sk);
      } else {
        if (p.q_lengths) qe = min(max(p.q_lengths[b], 0), p.Sq);
        if (p.k_lengths) ke = min(max(p.k_lengths[b] + p.k_add, 0), p.Sk);
      }
      if (i >= qs && i < qe) {
        const int prefix = p.prefixes ? p.prefixes[doc] : p.prefix;
        const int n = ke - ks;
        const int at = i - qs + n - (qe - qs);
        int seen = p.causal ? at + 1 : n;
        if (prefix > 0 && at < prefix) seen = prefix;
        lo = ks;
        hi = ks + min(max(seen, 0), n);
      }
    }
    if (lo >= hi) lo = hi = 0;
    p.ranges[static_cast<long long>(b) * p.Sq + i] = make_int2(lo, hi);
  }
  const bool some = row && lo < hi;
  int lo_min = some ? lo : INT_MAX, hi_max = some ? hi : 0;
  int lo_max = row ? lo : 0, hi_min = row ? hi : INT_MAX;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo_min = min(lo_min, __shfl_xor_sync(0xffffffffu, lo_min, o));
    hi_max = max(hi_max, __shfl_xor_sync(0xffffffffu, hi_max, o));
    lo_max = max(lo_max, __shfl_xor_sync(0xffffffffu, lo_max, o));
    hi_min = min(hi_min, __shfl_xor_sync(0xffffffffu, hi_min, o));
  }
  __shared__ int4 part[kTile / 32];
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_int4(lo_min, hi_max, lo_max, hi_min);
  __syncthreads();
  if (threadIdx.x == 0) {
    int4 t = part[0];
    for (int k = 1; k < kTile / 32; ++k)
      t = make_int4(min(t.x, part[k].x), max(t.y, part[k].y), max(t.z, part[k].z), min(t.w, part[k].w));
    p.table[blockIdx.x] = t;
  }
}

}  // namespace ranges

int launch_ranges(const RangesArgs& a, cudaStream_t stream) {
  ranges::Params p = {};
  p.ranges = a.ranges; p.table = a.table; p.given = a.given;
  p.prefixes = a.prefixes; p.q_offsets = a.q_offsets; p.k_offsets = a.k_offsets;
  p.q_lengths = a.q_lengths; p.k_lengths = a.k_lengths;
  p.Sq = a.Sq; p.Sk = a.Sk; p.causal = a.causal; p.prefix = a.prefix; p.docs = a.docs; p.k_add = a.k_add;
  p.tiles = (a.Sq + ranges::kTile - 1) / ranges::kTile;
  const long long grid = static_cast<long long>(a.Bm) * p.tiles;
  ranges::ranges_kernel<<<static_cast<int>(grid), ranges::kTile, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? BSA_OK : BSA_ERR_CUDA;
}

}  // namespace bsa
