// Attention over a sliding window and sinks (sink_attn.h): the C ABI, and the kernels for every
// type, head size and alignment, on fp32 MFMA (v_mfma_f32_16x16x4_f32) over LDS tiles of 64 keys
// (or queries) in fp32.  A wave owns 16 queries (or keys); a score tile's accumulators hold, per
// lane, rows 4 kg + j of column r, and step j of the next product takes rows {4 kg + j} as its
// four contraction indices, so P and dS enter it where they are.
#include <algorithm>
#include <type_traits>

#include "sink_attn.h"

using namespace fsi;
using namespace fsi_sink;

namespace {

constexpr int SK_THREADS = 256;
constexpr float SK_LOG2E = 1.4426950408889634f;

template <typename T>
__device__ __forceinline__ float sk_ld(const T* p, int64_t i);
template <>
__device__ __forceinline__ float sk_ld<float>(const float* p, int64_t i) { return p[i]; }
template <>
__device__ __forceinline__ float sk_ld<bf16_t>(const bf16_t* p, int64_t i) { return bf16_to_f32(p[i]); }
__device__ __forceinline__ void sk_st(float* p, float x) { *p = x; }
__device__ __forceinline__ void sk_st(bf16_t* p, float x) { *p = f32_to_bf16(x); }

__device__ __forceinline__ f32x4_t mfma4(float a, float b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Rows [r0, r0 + 64) of a (n, hd) matrix on their way into an LDS tile of row stride HD + 4 (the
// pad puts the 16 rows of a column read on distinct banks): fetched into registers while the tile
// before is computed, stored after it.  Rows from n on and dims from hd on are 0.  vec: hd and every
// row's start are multiples of 4 elements.
template <typename T, int HD>
struct SkFetch {
  static constexpr int PIECES = SK_T * HD / 4 / SK_THREADS, PPR = HD / 4;
  f32x4_t x[PIECES];
  __device__ __forceinline__ void load(const T* base, int64_t rs, int r0, int n, int hd, bool vec) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int i = p * SK_THREADS + threadIdx.x, row = r0 + i / PPR, d = i % PPR * 4;
      x[p] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (row >= n || d >= hd) continue;
      const T* src = base + row * rs + d;
      if (!vec) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[p][j] = d + j < hd ? sk_ld(src, j) : 0.f;
      } else if constexpr (sizeof(T) == 4) {
        x[p] = *reinterpret_cast<const f32x4_t*>(src);
      } else {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(src);
        x[p] = f32x4_t{lo_bf16(w[0]), hi_bf16(w[0]), lo_bf16(w[1]), hi_bf16(w[1])};
      }
    }
  }
  __device__ __forceinline__ void store(float* tile) const {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int i = p * SK_THREADS + threadIdx.x;
      *reinterpret_cast<f32x4_t*>(tile + i / PPR * (HD + 4) + i % PPR * 4) = x[p];
    }
  }
};

// Row `row` of a (., hd) matrix as an operand: dims 4 s + kg; 0 where !ok.
template <typename T, int HD>
__device__ __forceinline__ void sk_frag(const T* base, int64_t rs, int row, bool ok, int hd, int kg, float (&f)[HD / 4]) {
#pragma unroll
  for (int s = 0; s < HD / 4; ++s) f[s] = ok && 4 * s + kg < hd ? sk_ld(base, row * rs + 4 * s + kg) : 0.f;
}

// X^T (16 rows of the tile from 16 t) against the wave's operand.
template <int HD>
__device__ __forceinline__ f32x4_t sk_scores(const float* tile, int t, int r, int kg, const float (&f)[HD / 4]) {
  f32x4_t s = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float* row = tile + (16 * t + r) * (HD + 4) + kg;
#pragma unroll
  for (int i = 0; i < HD / 4; ++i) s = mfma4(row[4 * i], f[i], s);
  return s;
}

// acc[dim][col] += sum over NT 16-row parts of the tile from part t0, X[row][dim] w[row][col]; w holds
// rows 16 (t0 + t) + 4 kg + j.  A tile is summed by itself and then added: one chain over all of a
// key's queries rounds once per 4 of them (fp32, 2 x 1448 queries a key: dk off by 1.3e-6 of its norm,
// 5e-7 this way; times within 2 % either way).
template <int HD, int NT>
__device__ __forceinline__ void sk_accumulate(const float* tile, int t0, int r, int kg, const f32x4_t (&w)[NT],
                                              f32x4_t (&acc)[HD / 16]) {
  constexpr int N = HD % 64 == 0 ? 4 : HD / 32;  // 16-dim parts at a time: enough chains side by side
#pragma unroll
  for (int d0 = 0; d0 < HD / 16; d0 += N) {
    f32x4_t sum[N];
#pragma unroll
    for (int d = 0; d < N; ++d) sum[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float* row = tile + (16 * (t0 + t) + 4 * kg + j) * (HD + 4) + r + 16 * d0;
#pragma unroll
        for (int d = 0; d < N; ++d) sum[d] = mfma4(row[16 * d], w[t][j], sum[d]);
      }
#pragma unroll
    for (int d = 0; d < N; ++d) acc[d0 + d] += sum[d];
  }
}

// Column r of acc (dims 16 dt + 4 kg + j) times f into a row.
template <typename T, int HD>
__device__ __forceinline__ void sk_store(T* row, int hd, int kg, const f32x4_t (&acc)[HD / 16], float f) {
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (16 * dt + 4 * kg + j < hd) sk_st(row + 16 * dt + 4 * kg + j, acc[dt][j] * f);
}

// One output value, and what rounding took from it where that is kept.
template <typename T>
__device__ __forceinline__ void sk_out(const SkParams& P, int64_t at, float x) {
  sk_st(static_cast<T*>(P.o) + at, x);
  if constexpr (sizeof(T) == 2)
    if (P.olo) static_cast<bf16_t*>(P.olo)[at] = f32_to_bf16(x - round_bf16(x));
}

// SPLIT kernels: the four waves own the same 16 columns and a 16-row part of every tile each, and
// their sums meet in LDS at the end.  Taken where workgroups of 64 columns would leave CUs without
// one (rule and figures at sk_split_waves): a quarter of the work behind one another, in four times
// the workgroups.
//
// Sum of the waves' accumulators, each times its wave's factor f, in wave 0.
template <int HD>
__device__ __forceinline__ void sk_merge(float* lds, int wave, int lane, float f, f32x4_t (&acc)[HD / 16]) {
  f32x4_t* slot = reinterpret_cast<f32x4_t*>(lds) + lane;
  __syncthreads();
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) {
    acc[dt] *= f;
    if (wave > 0) slot[((wave - 1) * (HD / 16) + dt) * 64] = acc[dt];
  }
  __syncthreads();
  if (wave == 0)
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt)
#pragma unroll
      for (int w = 0; w < 3; ++w) acc[dt] += slot[(w * (HD / 16) + dt) * 64];
}

template <typename T, int HD, bool SPLIT>
__global__ __launch_bounds__(SK_THREADS) void sk_fwd_kernel(SkParams P) {
  constexpr int UN = SPLIT ? 16 : SK_T, NT = SPLIT ? 1 : 4;  // queries of a workgroup, tile parts of a wave
  extern __shared__ __attribute__((aligned(16))) float sk_smem[];
  float *kt = sk_smem, *vt = sk_smem + SK_T * (HD + 4);
  const int h = blockIdx.x % P.Hq, b = blockIdx.y, g = h / (P.Hq / P.Hkv);
  const int i0 = (gridDim.x / P.Hq - 1 - blockIdx.x / P.Hq) * UN;  // most keys first
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kg = lane >> 4;
  const int off = P.Tk - P.Tq, len = sk_length(P, b);
  const int i = i0 + (SPLIT ? 0 : 16 * wave) + r, p = off + i, part = SPLIT ? wave : 0;
  const bool live = i < P.Tq && p < len;
  const T* k = static_cast<const T*>(P.k) + b * P.ks_b + g * P.ks_h;
  const T* v = static_cast<const T*>(P.v) + b * P.vs_b + g * P.vs_h;
  float qf[HD / 4];
  sk_frag<T, HD>(static_cast<const T*>(P.q) + b * P.qs_b + h * P.qs_h, P.qs_t, i, live, P.hd, kg, qf);
  f32x4_t acc[HD / 16];
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const float sl2 = P.scale * SK_LOG2E;
  const SkTiles tiles = sk_key_tiles(P, off + i0, min(off + min(i0 + UN, P.Tq), len) - 1);
  const SkRange range = sk_key_part(P, tiles.count(), blockIdx.z);
  SkFetch<T, HD> fk, fv;
  auto fetch = [&](int c) {
    if (c >= range.hi) return;
    fk.load(k, P.ks_t, tiles.tile(c) * SK_T, len, P.hd, P.vec);
    fv.load(v, P.vs_t, tiles.tile(c) * SK_T, len, P.hd, P.vec);
  };
  fetch(range.lo);
  for (int c = range.lo; c < range.hi; ++c) {
    const int s0 = tiles.tile(c) * SK_T;
    __syncthreads();
    fk.store(kt);
    fv.store(vt);
    __syncthreads();
    fetch(c + 1);
    f32x4_t st[NT];
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      st[t] = sk_scores<HD>(kt, part + t, r, kg, qf);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        st[t][j] = live && sk_visible(P, len, p, s0 + 16 * (part + t) + 4 * kg + j) ? st[t][j] * sl2 : -INFINITY;
        mx = fmaxf(mx, st[t][j]);
      }
    }
    const float m_new = fmaxf(m, max_rows4(mx));
    const float ref = m_new == -INFINITY ? 0.f : m_new;  // nothing visible yet: every p is 0
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = m_new;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        st[t][j] = __builtin_amdgcn_exp2f(st[t][j] - ref);
        sum += st[t][j];
      }
    l = l * alpha + sum_rows4(sum);
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) acc[dt] *= alpha;
    sk_accumulate<HD, NT>(vt, part, r, kg, st, acc);
  }
  if constexpr (SPLIT) {  // the waves' maxima and sums, then their accumulators at the common maximum
    __syncthreads();
    if (kg == 0) {
      sk_smem[wave * 32 + r] = m;
      sk_smem[wave * 32 + 16 + r] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, sk_smem[w * 32 + r]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum = fmaf(sk_smem[w * 32 + 16 + r], __builtin_amdgcn_exp2f(sk_smem[w * 32 + r] - ref), sum);
    sk_merge<HD>(sk_smem, wave, lane, __builtin_amdgcn_exp2f(m - ref), acc);
    m = top;
    l = sum;
    if (wave > 0) return;
  }
  if (i >= P.Tq) return;
  if (P.ksplit > 1) {
    float* row = sk_part_row(P, blockIdx.z, b, h, i);
    sk_store<float, HD>(row, P.hd, kg, acc, 1.f);
    if (kg == 0) *reinterpret_cast<f32x4_t*>(row + sk_part_stride(P.hd) - 4) = f32x4_t{m, l, l, 0.f};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t at = b * P.os_b + h * P.os_h + i * P.os_t;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (16 * dt + 4 * kg + j < P.hd) sk_out<T>(P, at + 16 * dt + 4 * kg + j, acc[dt][j] * inv);
  if (P.lse && kg == 0)
    P.lse[(static_cast<int64_t>(b) * P.Hq + h) * P.Tq + i] = l == 0.f ? INFINITY : m + __log2f(l);
}

// dQ of 16 queries a wave, and D.
template <typename T, int HD, bool SPLIT>
__global__ __launch_bounds__(SK_THREADS) void sk_dq_kernel(SkParams P) {
  constexpr int UN = SPLIT ? 16 : SK_T, NT = SPLIT ? 1 : 4;  // queries of a workgroup, tile parts of a wave
  extern __shared__ __attribute__((aligned(16))) float sk_smem[];
  float *kt = sk_smem, *vt = sk_smem + SK_T * (HD + 4);
  const int h = blockIdx.x % P.Hq, b = blockIdx.y, g = h / (P.Hq / P.Hkv);
  const int i0 = (gridDim.x / P.Hq - 1 - blockIdx.x / P.Hq) * UN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kg = lane >> 4;
  const int off = P.Tk - P.Tq, len = sk_length(P, b);
  const int i = i0 + (SPLIT ? 0 : 16 * wave) + r, p = off + i, part = SPLIT ? wave : 0;
  const bool live = i < P.Tq && p < len;
  const T* k = static_cast<const T*>(P.k) + b * P.ks_b + g * P.ks_h;
  const T* v = static_cast<const T*>(P.v) + b * P.vs_b + g * P.vs_h;
  const int64_t stat = (static_cast<int64_t>(b) * P.Hq + h) * P.Tq + i;
  float qf[HD / 4], df[HD / 4];
  sk_frag<T, HD>(static_cast<const T*>(P.q) + b * P.qs_b + h * P.qs_h, P.qs_t, i, live, P.hd, kg, qf);
  sk_frag<T, HD>(static_cast<const T*>(P.dout) + b * P.ds_b + h * P.ds_h, P.ds_t, i, live, P.hd, kg, df);
  // D, as the diagonal of dout . out
  const int only = live ? sk_only_key(P, p) : -1;
  const int64_t at = only < 0 ? b * P.os_b + h * P.os_h + i * P.os_t : only * P.vs_t;
  const T* o = only < 0 ? static_cast<const T*>(P.o) : v;
  f32x4_t d4 = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < HD / 4; ++s) {
    float x = 0.f;
    if (live && 4 * s + kg < P.hd) {
      x = sk_ld(o, at + 4 * s + kg);
      if (sizeof(T) == 2 && P.olo && only < 0) x += bf16_to_f32(static_cast<const bf16_t*>(P.olo)[at + 4 * s + kg]);
    }
    d4 = mfma4(x, df[s], d4);
  }
  const float dd = sk_diagonal(d4, r, kg);
  if (i < P.Tq && kg == 0 && part == 0 && blockIdx.z == 0) P.dd[stat] = dd;
  const float lse = live ? P.lse[stat] : INFINITY, sl2 = P.scale * SK_LOG2E;
  f32x4_t acc[HD / 16];
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const SkTiles tiles = sk_key_tiles(P, off + i0, min(off + min(i0 + UN, P.Tq), len) - 1);
  const SkRange range = sk_key_part(P, tiles.count(), blockIdx.z);
  SkFetch<T, HD> fk, fv;
  auto fetch = [&](int c) {
    if (c >= range.hi) return;
    fk.load(k, P.ks_t, tiles.tile(c) * SK_T, len, P.hd, P.vec);
    fv.load(v, P.vs_t, tiles.tile(c) * SK_T, len, P.hd, P.vec);
  };
  fetch(range.lo);
  for (int c = range.lo; c < range.hi; ++c) {
    const int s0 = tiles.tile(c) * SK_T;
    __syncthreads();
    fk.store(kt);
    fv.store(vt);
    __syncthreads();
    fetch(c + 1);
    f32x4_t ds[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const f32x4_t s = sk_scores<HD>(kt, part + t, r, kg, qf), dp = sk_scores<HD>(vt, part + t, r, kg, df);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool ok = live && sk_visible(P, len, p, s0 + 16 * (part + t) + 4 * kg + j);
        ds[t][j] = ok ? __builtin_amdgcn_exp2f(fmaf(s[j], sl2, -lse)) * (dp[j] - dd) : 0.f;
      }
    }
    sk_accumulate<HD, NT>(kt, part, r, kg, ds, acc);
  }
  if constexpr (SPLIT) {
    sk_merge<HD>(sk_smem, wave, lane, 1.f, acc);
    if (wave > 0) return;
  }
  if (i >= P.Tq) return;
  if (P.ksplit > 1)
    sk_store<float, HD>(sk_part_row(P, blockIdx.z, b, h, i), P.hd, kg, acc, P.scale);
  else
    sk_store<T, HD>(static_cast<T*>(P.dq) + ((static_cast<int64_t>(b) * P.Hq + h) * P.Tq + i) * P.hd, P.hd, kg, acc,
                    P.scale);
}

// dK and dV of 16 keys a wave: every query tile that reaches the 64 keys, every query head.
template <typename T, int HD, bool SPLIT>
__global__ __launch_bounds__(SK_THREADS, 1) void sk_dkv_kernel(SkParams P, SkSinkSplit S) {
  constexpr int UN = SPLIT ? 16 : SK_T, NT = SPLIT ? 1 : 4;  // keys of a workgroup, tile parts of a wave
  extern __shared__ __attribute__((aligned(16))) float sk_smem[];
  float *qt = sk_smem, *gt = sk_smem + SK_T * (HD + 4), *stats = sk_smem + 2 * SK_T * (HD + 4);
  const int g = static_cast<int>(blockIdx.x) % P.Hkv, b = blockIdx.y;
  // the parts of the split sink tiles come first: they are the longest
  const int x = static_cast<int>(blockIdx.x) / P.Hkv, n_far = S.tiles * S.parts;
  const int tile = x < n_far ? x / S.parts : x - n_far, part = x < n_far ? x % S.parts : -1;
  const int s0 = tile * UN, G = P.Hq / P.Hkv;
  const SkRange heads = sk_head_part(P, blockIdx.z);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kg = lane >> 4;
  const int off = P.Tk - P.Tq, len = sk_length(P, b);
  const int s = s0 + (SPLIT ? 0 : 16 * wave) + r, tp = SPLIT ? wave : 0;
  float kf[HD / 4], vf[HD / 4];
  sk_frag<T, HD>(static_cast<const T*>(P.k) + b * P.ks_b + g * P.ks_h, P.ks_t, s, s < len, P.hd, kg, kf);
  sk_frag<T, HD>(static_cast<const T*>(P.v) + b * P.vs_b + g * P.vs_h, P.vs_t, s, s < len, P.hd, kg, vf);
  f32x4_t dk[HD / 16], dv[HD / 16];
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) dk[dt] = dv[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float sl2 = P.scale * SK_LOG2E;
  // queries that reach the keys through the window, or the part's beyond it
  const int q_end = min(P.Tq, len - off), near_hi = sk_near_end(P, S, s0);
  const int i_lo = part < 0 ? max(0, s0 - off) / SK_T * SK_T : near_hi + part * S.span;
  const int i_hi = min(q_end, part < 0 ? near_hi : i_lo + S.span);
  SkFetch<T, HD> fq, fg;
  float stat = 0.f;  // threads 0..63: lse of a row, 64..127: D
  auto fetch = [&](int i0, int hh) {
    if (i0 >= i_hi || hh >= heads.hi) return;
    const int h = g * G + hh;
    fq.load(static_cast<const T*>(P.q) + b * P.qs_b + h * P.qs_h, P.qs_t, i0, q_end, P.hd, P.vec);
    fg.load(static_cast<const T*>(P.dout) + b * P.ds_b + h * P.ds_h, P.ds_t, i0, q_end, P.hd, P.vec);
    const int i = i0 + (threadIdx.x & 63);
    if (threadIdx.x < 2 * SK_T && i < q_end)
      stat = (threadIdx.x < SK_T ? P.lse : P.dd)[(static_cast<int64_t>(b) * P.Hq + h) * P.Tq + i];
  };
  fetch(i_lo, heads.lo);
  for (int i0 = i_lo; i0 < i_hi; i0 += SK_T)
    for (int hh = heads.lo; hh < heads.hi; ++hh) {
      __syncthreads();
      fq.store(qt);
      fg.store(gt);
      if (threadIdx.x < 2 * SK_T) stats[threadIdx.x] = stat;
      __syncthreads();
      fetch(hh + 1 < heads.hi ? i0 : i0 + SK_T, hh + 1 < heads.hi ? hh + 1 : heads.lo);
      f32x4_t pw[NT], ds[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f32x4_t sc = sk_scores<HD>(qt, tp + t, r, kg, kf), dp = sk_scores<HD>(gt, tp + t, r, kg, vf);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 16 * (tp + t) + 4 * kg + j, i = i0 + row;
          const bool ok = i < q_end && sk_visible(P, len, off + i, s);
          pw[t][j] = ok ? __builtin_amdgcn_exp2f(fmaf(sc[j], sl2, -stats[row])) : 0.f;
          ds[t][j] = ok ? pw[t][j] * (dp[j] - stats[SK_T + row]) : 0.f;
        }
      }
      sk_accumulate<HD, NT>(gt, tp, r, kg, pw, dv);
      sk_accumulate<HD, NT>(qt, tp, r, kg, ds, dk);
    }
  if constexpr (SPLIT) {
    sk_merge<HD>(sk_smem, wave, lane, 1.f, dk);
    sk_merge<HD>(sk_smem, wave, lane, 1.f, dv);
    if (wave > 0) return;
  }
  if (s >= P.Tk) return;
  const int64_t head = static_cast<int64_t>(b) * P.Hkv + g;
  if (float* t = sk_kv_term(P, S, head, s, blockIdx.z, part)) {
    if (part >= 0 && s >= P.sinks) return;
    sk_store<float, HD>(t, P.hd, kg, dk, P.scale);
    sk_store<float, HD>(t + P.hd, P.hd, kg, dv, 1.f);
  } else if (part < 0) {
    const int64_t row = (head * P.Tk + s) * P.hd;
    sk_store<T, HD>(static_cast<T*>(P.dk) + row, P.hd, kg, dk, P.scale);
    sk_store<T, HD>(static_cast<T*>(P.dv) + row, P.hd, kg, dv, 1.f);
  }
}

// dK and dV rows that come in terms (sk_kv_term), added in order: one workgroup per (head, row); the
// first `rows` rows of every head.
template <typename T>
__global__ __launch_bounds__(SK_THREADS) void sk_kv_sum_kernel(SkParams P, SkSinkSplit S, int rows) {
  const int s = static_cast<int>(blockIdx.x % rows);
  const int64_t head = blockIdx.x / rows;
  const int far = S.parts > 0 && s < P.sinks ? S.parts + 1 : 1;
  for (int d = threadIdx.x; d < 2 * P.hd; d += SK_THREADS) {
    float sum = 0.f;
    for (int z = 0; z < P.hsplit; ++z)
      for (int part = 0; part < far; ++part) sum += sk_kv_term(P, S, head, s, z, far > 1 && part < S.parts ? part : -1)[d];
    T* out = static_cast<T*>(d < P.hd ? P.dk : P.dv) + (head * P.Tk + s) * P.hd + (d < P.hd ? d : d - P.hd);
    sk_st(out, sum);
  }
}

// Output rows from the parts of their keys, one wave per (sequence, head, query): forward (out, lse),
// or dQ.
template <typename T, bool FWD>
__global__ __launch_bounds__(64) void sk_join_kernel(SkParams P) {
  const int64_t row = blockIdx.x;
  const int i = static_cast<int>(row % P.Tq), h = static_cast<int>(row / P.Tq % P.Hq);
  const int b = static_cast<int>(row / P.Tq / P.Hq), last = sk_part_stride(P.hd) - 4;
  float m = -INFINITY, l = 0.f, lf = 0.f;
  if constexpr (FWD) {
    for (int z = 0; z < P.ksplit; ++z) m = fmaxf(m, sk_part_row(P, z, b, h, i)[last]);
    const float ref = m == -INFINITY ? 0.f : m;
    for (int z = 0; z < P.ksplit; ++z) {
      const f32x4_t st = *reinterpret_cast<const f32x4_t*>(sk_part_row(P, z, b, h, i) + last);
      const float w = __builtin_amdgcn_exp2f(st[0] - ref);
      l = fmaf(st[1], w, l);
      lf = fmaf(st[2], w, lf);
    }
    if (P.lse && threadIdx.x == 0) P.lse[row] = l == 0.f ? INFINITY : m + __log2f(lf);
  }
  const float ref = m == -INFINITY ? 0.f : m, inv = l == 0.f ? 0.f : 1.f / l;
  for (int d = threadIdx.x; d < P.hd; d += 64) {
    float x = 0.f;
    for (int z = 0; z < P.ksplit; ++z) {
      const float* p = sk_part_row(P, z, b, h, i);
      x = FWD ? fmaf(p[d], __builtin_amdgcn_exp2f(p[last] - ref), x) : x + p[d];
    }
    if constexpr (FWD) sk_out<T>(P, b * P.os_b + h * P.os_h + i * P.os_t + d, x * inv);
    else sk_st(static_cast<T*>(P.dq) + row * P.hd + d, x);
  }
}

// A part has about a window tile's queries, and no fewer than 512 (a short part's start and sum
// cost more than it saves).  More than 1024 sinks are tiles enough to fill the chip by themselves.
SkSinkSplit sk_split(int64_t Tq, int64_t Tk, int64_t window, int64_t sinks) {
  SkSinkSplit S{};
  window = std::min(window, Tk);
  sinks = std::min(sinks, Tk);
  if (sinks <= 0 || sinks > 1024) return S;
  const int64_t span = std::max<int64_t>(512, (window + 2 * SK_T - 1) / SK_T * SK_T);
  const int64_t near_hi = std::max<int64_t>((SK_T - 1 + window - (Tk - Tq) + SK_T - 1) / SK_T * SK_T, 0);
  if (Tq - near_hi <= span) return S;
  S.tiles = static_cast<int>((sinks + SK_T - 1) / SK_T);
  S.parts = static_cast<int>((Tq - near_hi + span - 1) / span);
  S.span = static_cast<int>(span);
  return S;
}

// Whether `cols` columns of `heads` (sequence, head) pairs go to SPLIT workgroups: where workgroups
// of 64 are fewer than the chip's CUs.  fp32, 3 sequences of 333, 6 / 3 heads of 64, with gradients:
// 261 us in workgroups of 64, 159 split (of which the kernels 17 + 26 + 31, the rest is the host).
bool sk_split_waves(int64_t cols, int64_t heads) { return (cols + SK_T - 1) / SK_T * heads < 256; }

// Parts that the keys of `blocks` workgroups are cut into: as many as two workgroups a CU hold, each
// of 4 key tiles at least.  32 / 8 heads, 1 query over 8192 keys, forward us in one part / cut: bf16
// 199 / 39, fp32 410 / 68.
constexpr int64_t SK_SLOTS = 512;
int sk_key_splits(const SkParams& P, int64_t blocks, int64_t columns) {
  const int64_t span = std::min<int64_t>(P.Tk, static_cast<int64_t>(P.window) + columns);
  const int64_t tiles = (span + SK_T - 1) / SK_T + 1 + (P.sinks + SK_T - 1) / SK_T;
  return static_cast<int>(std::max<int64_t>(std::min(SK_SLOTS / std::max<int64_t>(blocks, 1), tiles / 4), 1));
}
// Workgroups of the fp32 kernels' forward (dQ), and their queries.
int64_t sk_query_blocks(const SkParams& P) {
  const int64_t heads = static_cast<int64_t>(P.B) * P.Hq;
  return (P.Tq + (sk_split_waves(P.Tq, heads) ? 15 : 63)) / (sk_split_waves(P.Tq, heads) ? 16 : 64) * heads;
}
size_t sk_part_bytes(const SkParams& P, int splits) {
  return splits > 1 ? fsi_host::align_up(sizeof(float) * static_cast<size_t>(splits) * P.B * P.Hq * P.Tq *
                                             sk_part_stride(P.hd),
                                         256)
                    : 0;
}
// Parts that the query heads of a KV head are cut into for dK and dV: while the key tiles leave CUs
// without a workgroup.  unit: keys of a workgroup.  8 heads on one KV head, 2048 tokens, window 1024,
// bf16, forward and gradients: 508 us in one part, 174 cut.
int sk_head_splits(const SkParams& P, const SkSinkSplit& S, int64_t unit, int64_t slots) {
  const int64_t far = S.parts ? (P.sinks + unit - 1) / unit * S.parts : 0;
  const int64_t blocks = ((P.Tk + unit - 1) / unit + far) * P.Hkv * P.B;
  return static_cast<int>(std::max<int64_t>(std::min<int64_t>(slots / blocks, P.Hq / P.Hkv), 1));
}
size_t sk_head_bytes(const SkParams& P, int splits) {
  return splits > 1 ? fsi_host::align_up(sizeof(float) * 2 * static_cast<size_t>(splits) * P.B * P.Hkv * P.Tk * P.hd, 256)
                    : 0;
}
size_t sk_sums_bytes(const SkParams& P, const SkSinkSplit& S, int hsplit) {
  return S.parts ? fsi_host::align_up(sizeof(float) * 2 * static_cast<size_t>(hsplit) * P.B * P.Hkv * (S.parts + 1) *
                                          P.sinks * P.hd,
                                      256)
                 : 0;
}
// How a backward is cut, for the bf16 kernels or the fp32 ones.
struct SkPlan {
  int ksplit, hsplit;
  size_t bytes(const SkParams& P, const SkSinkSplit& S) const {
    return fsi_host::align_up(sizeof(float) * static_cast<size_t>(P.B) * P.Hq * P.Tq, 256) + sk_part_bytes(P, ksplit) +
           sk_head_bytes(P, hsplit) + sk_sums_bytes(P, S, hsplit);
  }
};
SkPlan sk_plan(const SkParams& P, const SkSinkSplit& S, bool bf16) {
  if (bf16) return {sk_key_splits(P, sb_query_blocks(P, true), 2 * SK_T), sk_head_splits(P, S, SK_T, SK_SLOTS)};
  return {sk_key_splits(P, sk_query_blocks(P), SK_T),
          sk_head_splits(P, S, sk_split_waves(P.Tk, static_cast<int64_t>(P.B) * P.Hkv) ? 16 : SK_T, SK_SLOTS / 2)};
}

// LDS above 64 KiB a workgroup has to be asked for.
template <typename K, typename... A>
void sk_launch(K* kern, dim3 grid, size_t lds, hipStream_t st, const A&... args) {
  if (lds > 65536)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(lds));
  kern<<<grid, SK_THREADS, lds, st>>>(args...);
}

template <typename F>
void sk_by_width(int64_t hd, F&& f) {
  if (hd <= 32) f(std::integral_constant<int, 32>{});
  else if (hd <= 64) f(std::integral_constant<int, 64>{});
  else if (hd <= 96) f(std::integral_constant<int, 96>{});
  else if (hd <= 128) f(std::integral_constant<int, 128>{});
  else f(std::integral_constant<int, 256>{});
}

template <bool FWD>
void sk_join(const SkParams& P, int dtype, hipStream_t st) {
  if (P.ksplit == 1) return;
  const unsigned rows = static_cast<unsigned>(static_cast<int64_t>(P.B) * P.Hq * P.Tq);
  if (dtype == FSI_DTYPE_F32) sk_join_kernel<float, FWD><<<rows, 64, 0, st>>>(P);
  else sk_join_kernel<bf16_t, FWD><<<rows, 64, 0, st>>>(P);
}

// f(type tag, SPLIT tag).
template <typename F>
void sk_by_form(int dtype, bool split, F&& f) {
  auto by_type = [&](auto t) {
    if (split) f(t, std::true_type{});
    else f(t, std::false_type{});
  };
  if (dtype == FSI_DTYPE_F32) by_type(float{});
  else by_type(bf16_t{});
}

// Whether 4 elements at a time can be read from every row of a (B, H, T, hd) operand.
bool sk_vec(const void* p, int64_t sb, int64_t sh, int64_t st, int64_t hd, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % (dtype == FSI_DTYPE_F32 ? 16 : 8) == 0 && (sb | sh | st | hd) % 4 == 0;
}

int sk_check(const char* what, int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t hd, int64_t window,
             int64_t sinks, int dtype) {
  FSI_CHECK_ARG(dtype == FSI_DTYPE_F32 || dtype == FSI_DTYPE_BF16, FSI_ERR_DTYPE, "%s: dtype %d", what, dtype);
  FSI_CHECK_ARG(hd >= 1 && hd <= 256, FSI_ERR_SHAPE, "%s: head_dim %lld (1..256)", what, (long long)hd);
  FSI_CHECK_ARG(B >= 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Tq >= 0 && Tk >= Tq, FSI_ERR_SHAPE,
                "%s: B %lld, Hq %lld, Hkv %lld, Tq %lld, Tk %lld (Hkv divides Hq, Tq <= Tk)", what, (long long)B,
                (long long)Hq, (long long)Hkv, (long long)Tq, (long long)Tk);
  FSI_CHECK_ARG(window >= 0 && sinks >= 0, FSI_ERR_SHAPE, "%s: window %lld, sinks %lld", what, (long long)window,
                (long long)sinks);
  FSI_CHECK_ARG(Tk <= (int64_t(1) << 30) && B <= 65535 && (Tk + 15) / 16 * Hq <= 0x7fffffff, FSI_ERR_SHAPE,
                "%s: sizes beyond range", what);
  return FSI_OK;
}

SkParams sk_params(const void* q, int64_t qs_b, int64_t qs_h, int64_t qs_t, const void* k, int64_t ks_b, int64_t ks_h,
                   int64_t ks_t, const void* v, int64_t vs_b, int64_t vs_h, int64_t vs_t, const void* o, int64_t os_b,
                   int64_t os_h, int64_t os_t, int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t hd,
                   int64_t window, int64_t sinks, const int32_t* lengths, float scale) {
  SkParams P{};
  P.q = q;
  P.qs_b = qs_b;
  P.qs_h = qs_h;
  P.qs_t = qs_t;
  P.k = k;
  P.ks_b = ks_b;
  P.ks_h = ks_h;
  P.ks_t = ks_t;
  P.v = v;
  P.vs_b = vs_b;
  P.vs_h = vs_h;
  P.vs_t = vs_t;
  P.o = const_cast<void*>(o);
  P.os_b = os_b;
  P.os_h = os_h;
  P.os_t = os_t;
  P.B = (int)B;
  P.Hq = (int)Hq;
  P.Hkv = (int)Hkv;
  P.Tq = (int)Tq;
  P.Tk = (int)Tk;
  P.hd = (int)hd;
  // a window or sinks past the sequence see all of it
  P.window = (int)std::min<int64_t>(window, Tk);
  P.sinks = (int)std::min<int64_t>(sinks, Tk);
  P.lengths = lengths;
  P.scale = scale;
  P.ksplit = P.hsplit = 1;
  return P;
}

}  // namespace

extern "C" {

FSI_API size_t fsi_sink_attn_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t Tk,
                                            int64_t head_dim, int64_t window, int64_t sinks) {
  if (sk_check("sink_attn", B, Hq, Hkv, Tq, Tk, head_dim, window, sinks, FSI_DTYPE_F32) != FSI_OK || B == 0 || Tq == 0)
    return 0;
  const SkParams P = sk_params(nullptr, 0, 0, 0, nullptr, 0, 0, 0, nullptr, 0, 0, 0, nullptr, 0, 0, 0, B, Hq, Hkv, Tq,
                               Tk, head_dim, window, sinks, nullptr, 1.f);
  return std::max(sk_part_bytes(P, sk_key_splits(P, sk_query_blocks(P), SK_T)),
                  sk_part_bytes(P, sk_key_splits(P, sb_query_blocks(P, false), 2 * SK_T)));
}

FSI_API int fsi_sink_attn(const void* q, int64_t qs_b, int64_t qs_h, int64_t qs_t, const void* k, int64_t ks_b,
                          int64_t ks_h, int64_t ks_t, const void* v, int64_t vs_b, int64_t vs_h, int64_t vs_t,
                          int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t head_dim, int64_t window,
                          int64_t sinks, const int32_t* lengths, float scale, int dtype, void* out, int64_t os_b,
                          int64_t os_h, int64_t os_t, void* out_lo, float* lse, void* workspace,
                          size_t workspace_bytes, void* stream) {
  using namespace fsi_host;
  const int c = sk_check("sink_attn", B, Hq, Hkv, Tq, Tk, head_dim, window, sinks, dtype);
  if (c != FSI_OK || B == 0 || Tq == 0) return c;
  FSI_CHECK_ARG(q && k && v && out, FSI_ERR_INVALID_ARG, "sink_attn: null pointer");
  const size_t need = fsi_sink_attn_workspace_size(B, Hq, Hkv, Tq, Tk, head_dim, window, sinks);
  FSI_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                FSI_ERR_WORKSPACE, "sink_attn: workspace %zu < %zu bytes (or misaligned)", workspace_bytes, need);
  SkParams P = sk_params(q, qs_b, qs_h, qs_t, k, ks_b, ks_h, ks_t, v, vs_b, vs_h, vs_t, out, os_b, os_h, os_t, B, Hq,
                         Hkv, Tq, Tk, head_dim, window, sinks, lengths, scale);
  P.olo = dtype == FSI_DTYPE_BF16 ? out_lo : nullptr;
  P.lse = lse;
  P.kpart = static_cast<float*>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (sb_takes(P, dtype, false)) {
    P.ksplit = sk_key_splits(P, sb_query_blocks(P, false), 2 * SK_T);
    sb_forward(P, st);
  } else {
    P.ksplit = sk_key_splits(P, sk_query_blocks(P), SK_T);
    P.vec = sk_vec(k, ks_b, ks_h, ks_t, head_dim, dtype) && sk_vec(v, vs_b, vs_h, vs_t, head_dim, dtype);
    auto run = [&](auto t, auto w, auto sp) {
      using T = decltype(t);
      constexpr int HD = decltype(w)::value, UN = decltype(sp)::value ? 16 : SK_T;
      const dim3 grid(static_cast<unsigned>((Tq + UN - 1) / UN * Hq), static_cast<unsigned>(B), P.ksplit);
      sk_launch(&sk_fwd_kernel<T, HD, decltype(sp)::value>, grid, sizeof(float) * 2 * SK_T * (HD + 4), st, P);
    };
    sk_by_width(head_dim, [&](auto w) {
      sk_by_form(dtype, sk_split_waves(Tq, B * Hq), [&](auto t, auto sp) { run(t, w, sp); });
    });
  }
  sk_join<true>(P, dtype, st);
  FSI_HIP_LAUNCH_CHECK("sink_attn");
  return FSI_OK;
}

FSI_API size_t fsi_sink_attn_bwd_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t Tk,
                                                int64_t head_dim, int64_t window, int64_t sinks) {
  if (sk_check("sink_attn_bwd", B, Hq, Hkv, Tq, Tk, head_dim, window, sinks, FSI_DTYPE_F32) != FSI_OK || B == 0 ||
      Tq == 0)
    return 0;
  const SkParams P = sk_params(nullptr, 0, 0, 0, nullptr, 0, 0, 0, nullptr, 0, 0, 0, nullptr, 0, 0, 0, B, Hq, Hkv, Tq,
                               Tk, head_dim, window, sinks, nullptr, 1.f);
  const SkSinkSplit S = sk_split(Tq, Tk, window, sinks);
  return std::max(sk_plan(P, S, false).bytes(P, S), sk_plan(P, S, true).bytes(P, S));
}

FSI_API int fsi_sink_attn_bwd(const void* q, int64_t qs_b, int64_t qs_h, int64_t qs_t, const void* k, int64_t ks_b,
                              int64_t ks_h, int64_t ks_t, const void* v, int64_t vs_b, int64_t vs_h, int64_t vs_t,
                              const void* out, int64_t os_b, int64_t os_h, int64_t os_t, const void* out_lo,
                              const void* dout, int64_t ds_b, int64_t ds_h, int64_t ds_t, const float* lse,
                              int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t head_dim,
                              int64_t window, int64_t sinks,
                              const int32_t* lengths, float scale, int dtype, void* dq, void* dk, void* dv,
                              void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fsi_host;
  const int c = sk_check("sink_attn_bwd", B, Hq, Hkv, Tq, Tk, head_dim, window, sinks, dtype);
  if (c != FSI_OK || B == 0 || Tk == 0) return c;
  FSI_CHECK_ARG(dk && dv && (Tq == 0 || (q && k && v && out && dout && lse && dq)), FSI_ERR_INVALID_ARG,
                "sink_attn_bwd: null pointer");
  const size_t need = fsi_sink_attn_bwd_workspace_size(B, Hq, Hkv, Tq, Tk, head_dim, window, sinks);
  FSI_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                FSI_ERR_WORKSPACE, "sink_attn_bwd: workspace %zu < %zu bytes (or misaligned)", workspace_bytes, need);
  SkParams P = sk_params(q, qs_b, qs_h, qs_t, k, ks_b, ks_h, ks_t, v, vs_b, vs_h, vs_t, out, os_b, os_h, os_t, B, Hq,
                         Hkv, Tq, Tk, head_dim, window, sinks, lengths, scale);
  P.olo = dtype == FSI_DTYPE_BF16 ? const_cast<void*>(out_lo) : nullptr;
  P.dout = dout;
  P.ds_b = ds_b;
  P.ds_h = ds_h;
  P.ds_t = ds_t;
  P.lse = const_cast<float*>(lse);
  P.dq = dq;
  P.dk = dk;
  P.dv = dv;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  SkSinkSplit S = sk_split(Tq, Tk, window, sinks);
  FSI_CHECK_ARG(B * Hkv * Tk <= 0x7fffffff && ((Tk + 15) / 16 + 4 * S.tiles * S.parts) * Hkv <= 0x7fffffff,
                FSI_ERR_SHAPE, "sink_attn_bwd: sizes beyond range");
  const bool bf16 = sb_takes(P, dtype, true);
  if (Tq > 0) {  // D, the parts of dQ, of dK / dV, and of the sink rows
    const SkPlan plan = sk_plan(P, S, bf16);
    P.ksplit = plan.ksplit;
    P.hsplit = plan.hsplit;
    char* ws = static_cast<char*>(workspace);
    P.dd = reinterpret_cast<float*>(ws);
    ws += align_up(sizeof(float) * static_cast<size_t>(B * Hq * Tq), 256);
    P.kpart = reinterpret_cast<float*>(ws);
    ws += sk_part_bytes(P, P.ksplit);
    P.hpart = reinterpret_cast<float*>(ws);
    ws += sk_head_bytes(P, P.hsplit);
    S.sums = reinterpret_cast<float*>(ws);
  }
  if (bf16) {
    sb_backward(P, S, st);
  } else {
    P.vec = sk_vec(q, qs_b, qs_h, qs_t, head_dim, dtype) && sk_vec(k, ks_b, ks_h, ks_t, head_dim, dtype) &&
            sk_vec(v, vs_b, vs_h, vs_t, head_dim, dtype) && sk_vec(dout, ds_b, ds_h, ds_t, head_dim, dtype);
    auto run_q = [&](auto t, auto w, auto sp) {
      using T = decltype(t);
      constexpr int HD = decltype(w)::value, UN = decltype(sp)::value ? 16 : SK_T;
      const dim3 grid(static_cast<unsigned>((Tq + UN - 1) / UN * Hq), static_cast<unsigned>(B), P.ksplit);
      sk_launch(&sk_dq_kernel<T, HD, decltype(sp)::value>, grid, sizeof(float) * 2 * SK_T * (HD + 4), st, P);
    };
    auto run_kv = [&](auto t, auto w, auto sp) {
      using T = decltype(t);
      constexpr int HD = decltype(w)::value, UN = decltype(sp)::value ? 16 : SK_T;
      SkSinkSplit SU = S;
      if (S.parts) SU.tiles = (P.sinks + UN - 1) / UN;
      const dim3 grid(static_cast<unsigned>(((Tk + UN - 1) / UN + SU.tiles * SU.parts) * Hkv), static_cast<unsigned>(B),
                      P.hsplit);
      sk_launch(&sk_dkv_kernel<T, HD, decltype(sp)::value>, grid, sizeof(float) * (2 * SK_T * (HD + 4) + 2 * SK_T), st,
                P, SU);
    };
    sk_by_width(head_dim, [&](auto w) {
      if (Tq > 0) sk_by_form(dtype, sk_split_waves(Tq, B * Hq), [&](auto t, auto sp) { run_q(t, w, sp); });
      sk_by_form(dtype, sk_split_waves(Tk, B * Hkv), [&](auto t, auto sp) { run_kv(t, w, sp); });
    });
  }
  sk_join<false>(P, dtype, st);
  const int rows = P.hsplit > 1 ? P.Tk : (S.parts ? P.sinks : 0);
  if (rows > 0) {
    const unsigned blocks = static_cast<unsigned>(B * Hkv * rows);
    if (dtype == FSI_DTYPE_F32) sk_kv_sum_kernel<float><<<blocks, SK_THREADS, 0, st>>>(P, S, rows);
    else sk_kv_sum_kernel<bf16_t><<<blocks, SK_THREADS, 0, st>>>(P, S, rows);
  }
  FSI_HIP_LAUNCH_CHECK("sink_attn_bwd");
  return FSI_OK;
}

}  // extern "C"
