// Attention over a sliding window and the first tokens ("sinks"), forward and backward: the
// parameters and the mask that the kernels of sink_attn.hip and sink_attn_bf16.hip share.
//
// Query i stands at position p = i + Tk - Tq and sees key s where
//   s <= p  and  (s > p - window  or  s < sinks)  and  p, s < length of the sequence.
//   P = exp(scale q.k - m) / l over the visible keys,  out = P v  (0 for a query without keys)
//   D = dout . out,  dV = P^T dout,  dS = P (dout v^T - D),  dQ = scale dS K,  dK = scale dS^T Q
// with dK and dV summed over the query heads of a KV head.
#pragma once

#include "fsi_common.h"

namespace fsi_sink {

constexpr int SK_T = 64;  // queries / keys per tile

struct SkParams {
  const void* q;
  int64_t qs_b, qs_h, qs_t;
  const void* k;
  int64_t ks_b, ks_h, ks_t;
  const void* v;
  int64_t vs_b, vs_h, vs_t;
  void* o;  // forward: written
  int64_t os_b, os_h, os_t;
  void* olo;  // bf16, laid out as o: what rounding took from it, so that D keeps 16 bits; or null
  const void* dout;
  int64_t ds_b, ds_h, ds_t;
  int B, Hq, Hkv, Tq, Tk, hd, window, sinks;
  const int32_t* lengths;
  float scale;
  float* lse;  // (B, Hq, Tq): log2 of the softmax denominator of scale log2(e) q.k; +inf without keys
  float* dd;   // (B, Hq, Tq): D
  void* dq;    // contiguous gradients of the operands' type
  void* dk;
  void* dv;
  // Key tiles of a query block cut into ksplit workgroups (forward, dQ): fp32 rows of
  // sk_part_stride(hd) floats, (ksplit, B, Hq, Tq), that sk_join_kernel combines.
  int ksplit;
  float* kpart;
  // Query heads of a KV head cut into hsplit workgroups (dK, dV): fp32 rows (hsplit, B, Hkv, Tk, [dK,
  // dV], hd), added by sk_kv_sum_kernel.
  int hsplit;
  float* hpart;
  bool vec;    // sink_attn.hip's kernels: 4 elements at a time can be read from the tiles' rows
};

__device__ __forceinline__ int sk_length(const SkParams& P, int b) {
  if (!P.lengths) return P.Tk;
  const int n = P.lengths[b];
  return n < 0 ? 0 : (n > P.Tk ? P.Tk : n);
}

// Key tiles that the queries at positions [p0, p1] reach: [0, n_sink) and [w0, w1].
struct SkTiles {
  int n_sink, w0, w1;
  __device__ __forceinline__ int count() const { return n_sink + (w1 >= w0 ? w1 - w0 + 1 : 0); }
  __device__ __forceinline__ int tile(int i) const { return i < n_sink ? i : w0 + i - n_sink; }
};
__device__ __forceinline__ SkTiles sk_key_tiles(const SkParams& P, int p0, int p1) {
  SkTiles t;
  if (p1 < p0) return {0, 0, -1};
  const int wlo = p0 - P.window + 1 > 0 ? p0 - P.window + 1 : 0;  // first key of the first query's window
  const int se = P.sinks < wlo ? P.sinks : wlo;                   // sinks before it
  t.n_sink = (se + SK_T - 1) / SK_T;
  t.w0 = wlo / SK_T > t.n_sink ? wlo / SK_T : t.n_sink;
  t.w1 = P.window > 0 || P.sinks > wlo ? p1 / SK_T : -1;
  return t;
}

// A tile of sink keys is seen by every later query, far more than a window's: its queries beyond
// the window are cut into `parts` of `span` queries (a multiple of the tile), each a workgroup of
// its own that leaves fp32 sums of the sink rows in `sums` (B, Hkv, hsplit, parts + 1, sinks, [dK, dV],
// hd), the window's own queries as the last part; sk_kv_sum_kernel adds them in that order.
// parts 0: no such split, a sink tile's workgroup takes all of its queries.
struct SkSinkSplit {
  int tiles, parts, span;
  float* sums;
};

// A partial row: the accumulated dims, then (forward) the maximum, the sum that divides the output and
// the sum that makes lse.
__host__ __device__ __forceinline__ int sk_part_stride(int hd) { return (hd + 3) / 4 * 4 + 4; }
__device__ __forceinline__ float* sk_part_row(const SkParams& P, int z, int b, int h, int i) {
  return P.kpart + (((static_cast<int64_t>(z) * P.B + b) * P.Hq + h) * P.Tq + i) * sk_part_stride(P.hd);
}

// Tiles [lo, hi) of part z of a query block's n key tiles.
struct SkRange {
  int lo, hi;
};
__device__ __forceinline__ SkRange sk_key_part(const SkParams& P, int n, int z) {
  const int per = (n + P.ksplit - 1) / P.ksplit, lo = min(n, z * per);
  return {lo, min(n, lo + per)};
}
// Query heads [lo, hi) of part z of a KV head's group.
__device__ __forceinline__ SkRange sk_head_part(const SkParams& P, int z) {
  const int G = P.Hq / P.Hkv, per = (G + P.hsplit - 1) / P.hsplit, lo = min(G, z * per);
  return {lo, min(G, lo + per)};
}

// Where key row s of (b, g) goes to as fp32 (dK, then dV at + hd): a term of a split sum, or null for
// a row that is stored as it is.  far: the part of a split sink tile (-1: the window's queries).
__device__ __forceinline__ float* sk_kv_term(const SkParams& P, const SkSinkSplit& S, int64_t head, int s, int z,
                                             int far) {
  if (S.parts > 0 && s < P.sinks)
    return S.sums +
           ((((head * P.hsplit + z) * (S.parts + 1) + (far < 0 ? S.parts : far)) * P.sinks + s) * 2) * P.hd;
  if (P.hsplit == 1) return nullptr;
  const int64_t heads = static_cast<int64_t>(P.B) * P.Hkv;
  return P.hpart + (((z * heads + head) * P.Tk + s) * 2) * P.hd;
}

__device__ __forceinline__ bool sk_visible(const SkParams& P, int len, int p, int s) {
  return s <= p && (s > p - P.window || s < P.sinks) && p < len;
}

// The key of a query at position p that sees one key only, else -1.  Its P is 1 and its dS is 0: with
// D = dout . v, summed as dP is, the kernels' dP - D is 0 to the bit, whatever out was rounded to.
__device__ __forceinline__ int sk_only_key(const SkParams& P, int p) {
  if (P.window > 0) return p == 0 || (P.window == 1 && P.sinks == 0) ? p : -1;
  return P.sinks > 0 && (p == 0 || P.sinks == 1) ? 0 : -1;
}

// Column r's element (r, r) of a 16 x 16 product, in every lane of the column.
__device__ __forceinline__ float sk_diagonal(fsi::f32x4_t x, int r, int kg) {
  const float lo = r & 1 ? x[1] : x[0], hi = r & 1 ? x[3] : x[2];
  return fsi::sum_rows4(kg == r >> 2 ? (r & 2 ? hi : lo) : 0.f);
}

// End of the queries that reach key tile s0 before the split's parts begin, in whole query tiles.
__device__ __forceinline__ int sk_near_end(const SkParams& P, const SkSinkSplit& S, int s0) {
  if (s0 < P.sinks && S.parts == 0) return P.Tq;
  const int64_t end = static_cast<int64_t>(s0) + SK_T - 1 + P.window - (P.Tk - P.Tq);
  if (end <= 0) return 0;
  return static_cast<int>(end < P.Tq ? (end + SK_T - 1) / SK_T * SK_T : P.Tq);
}

// The bf16 kernels of sink_attn_bf16.hip: whether they take the call, and their launches.
// sb_query_blocks: the workgroups of the forward (dQ) without a split of the keys.
bool sb_takes(const SkParams& P, int dtype, bool backward);
int64_t sb_query_blocks(const SkParams& P, bool backward);
void sb_forward(const SkParams& P, hipStream_t st);
void sb_backward(const SkParams& P, const SkSinkSplit& S, hipStream_t st);

}  // namespace fsi_sink
