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

__device__ __forceinline__ bool sk_visible(const SkParams& P, int len, int p, int s) {
  return s <= p && (s > p - P.window || s < P.sinks) && p < len;
}

// A tile of sink keys is seen by every later query, far more than a window's: its queries beyond
// the window are cut into `parts` of `span` queries (a multiple of the tile), each a workgroup of
// its own that leaves fp32 sums of the sink rows in `sums` (B, Hkv, parts + 1, sinks, [dK, dV], hd),
// the window's own queries as the last part; sk_sink_sum_kernel adds them in that order.
// parts 0: no such split, a sink tile's workgroup takes all of its queries.
struct SkSinkSplit {
  int tiles, parts, span;
  float* sums;
};

// End of the queries that reach key tile s0 before the split's parts begin, in whole query tiles.
__device__ __forceinline__ int sk_near_end(const SkParams& P, const SkSinkSplit& S, int s0) {
  if (s0 < P.sinks && S.parts == 0) return P.Tq;
  const int64_t end = static_cast<int64_t>(s0) + SK_T - 1 + P.window - (P.Tk - P.Tq);
  if (end <= 0) return 0;
  return static_cast<int>(end < P.Tq ? (end + SK_T - 1) / SK_T * SK_T : P.Tq);
}

// The bf16 kernels of sink_attn_bf16.hip: whether they take the call, and their launches.
bool sb_takes(const SkParams& P, int dtype, bool backward);
void sb_forward(const SkParams& P, hipStream_t st);
void sb_backward(const SkParams& P, const SkSinkSplit& S, hipStream_t st);

}  // namespace fsi_sink
