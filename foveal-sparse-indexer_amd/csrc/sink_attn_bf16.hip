// Windowed attention with sinks (sink_attn.h) for bf16 with head_dim 64, 128 or 256: forward, dQ, and
// dK / dV, every product on v_mfma_f32_16x16x32_bf16 over 64-row LDS tiles (attn_tiles_bf16.h)
// that direct-to-LDS loads fill one step ahead.
//
// The score tiles are formed transposed (keys as rows), so a lane's accumulators hold 4 keys
// times the tiles of one query: the softmax reduces inside the lane and over 4 lanes, and P^T
// (dS^T) is already the next product's operand.  P and (but for few tiles, sb_fine) dS are
// rounded once to bf16 for those products (8 bits, as the outputs themselves are rounded); the
// output's denominator is the sum of the same rounded P, formed by one more MFMA against ones, so
// that P's rounding leaves no bias.  The denominator that the backward takes (lse) is the sum
// before rounding, which forms P again to fp32 precision, and D = dout . out takes out with the
// remainder of its rounding: with out alone, rows of few keys have dq and dk up to 3.6e-3 of
// their norm off, with it 2.4e-3, and 1.75e-3 with dS in two terms (their own rounding: 1.66e-3).
#include <algorithm>
#include <type_traits>

#include "attn_tiles_bf16.h"
#include "sink_attn.h"

using namespace fsi_sink;

namespace {

static_assert(SK_T == AB_T, "one tile size");
constexpr float SB_LOG2E = 1.4426950408889634f;

// dims 32 s + 8 kg .. of row `row` of a (., HD) matrix; 0 where !ok (row is then any row that exists)
template <int HD>
__device__ __forceinline__ void sb_frag(const bf16_t* base, int64_t rs, int row, bool ok, int kg,
                                        u32x4_t (&f)[HD / 32]) {
#pragma unroll
  for (int s = 0; s < HD / 32; ++s) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(base + row * rs + 32 * s + 8 * kg);
    f[s] = ok ? x : u32x4_t{0u, 0u, 0u, 0u};
  }
}

// 8 values, as bf16 and, LO, what that rounding took from them
template <bool LO>
__device__ __forceinline__ void sb_round(const f32x4_t& a, const f32x4_t& b, u32x4_t& hi, u32x4_t& lo) {
  const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    hi[w] = bf_cvt2(x[2 * w], x[2 * w + 1]);
    if (LO) lo[w] = bf_cvt2(x[2 * w] - lo_bf16(hi[w]), x[2 * w + 1] - hi_bf16(hi[w]));
  }
}

// How the keys [a, a + n) of a tile meet the queries at positions [p0, p1] (both uniform).
enum SbKeys : int { SB_NONE = 0, SB_SOME = 1, SB_ALL = 2 };
__device__ __forceinline__ SbKeys sb_keys(const SkParams& P, int len, int a, int n, int p0, int p1) {
  const int z = a + n - 1;
  if (p1 < p0 || a > p1 || p0 >= len || (z <= p0 - P.window && a >= P.sinks)) return SB_NONE;
  return z <= p0 && p1 < len && (a > p1 - P.window || z < P.sinks) ? SB_ALL : SB_SOME;
}

// ---------------------------------------------------------------------------
// Forward.  A workgroup of 4 waves is HPW query heads of one KV head (they share the K / V
// tiles) at 32 * 4 / HPW queries; a wave is one head's 32 queries (two 16-query tiles, so a K or
// V fragment read from LDS enters two MFMAs).  Two workgroups a CU: the two waves of a SIMD then
// meet no common barrier, and one's products run beside the other's softmax (8 waves a workgroup
// over a ring of four tiles: 2 x 4096 tokens 190 against 168 us, 16384 tokens 2 % slower).
// The running maximum moves only when a score exceeds it by more than 2^8: P then stays below
// 2^8, most tiles need one compare instead of the row maxima, and the accumulators are rescaled
// rarely.
// Bound: issue of the matrix pipe (0.48 busy) and the vector units (0.4), whose phases of a tile
// overlap with the other wave's only.  16384 tokens, window 4096, 32 / 8 heads of 128 (963 GFLOP): 902
// - 952 us card by card, 1010 - 1067 TFLOP/s; 2 x 4096, window 1024, with lse and remainder 167 - 179.
// One test of both query tiles' maxima and the copies' offsets in registers: 943 -> 902, 178 -> 167.
// Slower: 32 keys of a tile at a time 1045, the next tile's scores before
// this one's softmax (spills) 7000, every K fragment read first 985.
// ---------------------------------------------------------------------------
constexpr int SB_THREADS = 256;
constexpr int SB_WAVES = SB_THREADS / 64;
// Workgroups a CU that a kernel's registers and LDS are kept to: head_dim 256 takes all of one.
constexpr int sb_blocks(int hd) { return hd > 128 ? 1 : 2; }

// sab_dma's copy of rows [r0, r0 + 64) by the workgroup, with what it needs of a thread kept in
// registers: lo, the thread's byte offset from a row of its group of ROWS rows, and the wave's share of
// the tile.  Bases are scalars of their own per group (opaque, or the compiler chains 64-bit vector
// additions from one to the next).
template <int HD>
struct SbLoad {
  static constexpr int PC = HD / 8, ROWS = SB_THREADS / PC, N = SK_T / ROWS;
  int row, piece, wave;
  __device__ __forceinline__ SbLoad() {
    row = static_cast<int>(threadIdx.x) / PC;
    piece = 16 * ((static_cast<int>(threadIdx.x) % PC) ^ sab_swz<HD>(row));
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  }
  __device__ __forceinline__ void operator()(const bf16_t* base, int64_t rs, int r0, int T, char* tile) const {
    const uint32_t rsb = static_cast<uint32_t>(rs) * 2u;
    const char* rb = reinterpret_cast<const char*>(base + static_cast<int64_t>(r0) * rs);
    char* dst = tile + wave * 1024;
    if (r0 + SK_T <= T) {
      const uint32_t lo = static_cast<uint32_t>(row) * rsb + static_cast<uint32_t>(piece);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const char* p = rb + static_cast<uint64_t>(j * ROWS) * rsb;
        asm volatile("" : "+s"(p));
        __builtin_amdgcn_global_load_lds((ab_glb_t*)(p + lo), (ab_lds_t*)(dst + j * SB_THREADS * 16), 16, 0, 0);
      }
    } else {
      const int last = T - 1 - r0;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t lo = static_cast<uint32_t>(min(j * ROWS + row, last)) * rsb + static_cast<uint32_t>(piece);
        __builtin_amdgcn_global_load_lds((ab_glb_t*)(rb + lo), (ab_lds_t*)(dst + j * SB_THREADS * 16), 16, 0, 0);
      }
    }
  }
};

template <int HD, int HPW, bool LSE>
__global__ __launch_bounds__(SB_THREADS, sb_blocks(HD)) void sb_fwd_kernel(SkParams P) {
  constexpr int KS = HD / 32, DT = HD / 16, TB = sab_tile_bytes<HD>();
  constexpr int QW = SB_WAVES / HPW * 32;  // queries of a workgroup
  __shared__ __attribute__((aligned(1024))) char smem[2 * 2 * TB];  // [stage][K, V]
  const int per = P.Hq / HPW;  // workgroups a query range takes
  const int hp = static_cast<int>(blockIdx.x) % per, b = blockIdx.y;
  const int i0 = (static_cast<int>(gridDim.x) / per - 1 - static_cast<int>(blockIdx.x) / per) * QW;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, kg = lane >> 4;
  // consecutive workgroups are consecutive KV heads: one XCD's L2 each where there are eight
  const int g = hp % P.Hkv, h = g * (P.Hq / P.Hkv) + hp / P.Hkv * HPW + wave % HPW;
  const int off = P.Tk - P.Tq, len = sk_length(P, b);
  const int iw = i0 + 32 * (wave / HPW), pw = off + iw;  // this wave's queries
  const int pw1 = off + min(iw + 32, P.Tq) - 1;
  const bf16_t* k = static_cast<const bf16_t*>(P.k) + b * P.ks_b + g * P.ks_h;
  const bf16_t* v = static_cast<const bf16_t*>(P.v) + b * P.vs_b + g * P.vs_h;
  const SkTiles tiles = sk_key_tiles(P, off + i0, min(off + min(i0 + QW, P.Tq), len) - 1);
  const SkRange range = sk_key_part(P, tiles.count(), blockIdx.z);
  const SbLoad<HD> copy;
  auto load = [&](int c) {
    if (c >= range.hi) return;
    char* dst = smem + (c & 1) * (2 * TB);
    copy(k, P.ks_t, tiles.tile(c) * SK_T, len, dst);
    copy(v, P.vs_t, tiles.tile(c) * SK_T, len, dst + TB);
  };
  load(range.lo);
  u32x4_t q[2][KS];
  int hi[2];  // last visible key of query iw + 16 i + r
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int qi = iw + 16 * i + r;
    const bool live = qi < P.Tq && off + qi < len;
    sb_frag<HD>(static_cast<const bf16_t*>(P.q) + b * P.qs_b + h * P.qs_h, P.qs_t, qi < P.Tq ? qi : P.Tq - 1, live, kg,
                q[i]);
    hi[i] = live ? off + qi : -1;
  }
  const float sl2 = P.scale * SB_LOG2E, inv_sl2 = 1.f / sl2;
  f32x4_t acc[2][DT], lsum[2];
  float m[2], thr[2], l_full[2] = {0.f, 0.f};  // thr: raw score whose scaled value is m + 8
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    m[i] = -3.0e38f;  // finite: a masked score gives exp2(-inf) = 0 without a special case
    thr[i] = -INFINITY;
    lsum[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[i][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t row_off = sab_row_off<HD>(r, kg), tr_off = sab_tr_off<HD>(r, kg);
  const u32x4_t ones = u32x4_t{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  auto step = [&](int c) {
    const int s0 = tiles.tile(c) * SK_T;
    const uint32_t at = (c & 1) * (2 * TB);
    const SbKeys all = sb_keys(P, len, s0, SK_T, pw, pw1);
    if (all == SB_NONE) return;
    f32x4_t st[2][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      st[0][t] = st[1][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4_t a = sab_row(smem, row_off + at, ks, 16 * t * HD * 2);
        st[0][t] = mfma16x16x32(a, q[0][ks], st[0][t]);
        st[1][t] = mfma16x16x32(a, q[1][ks], st[1][t]);
      }
    }
    if (all != SB_ALL) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int lo = hi[i] - P.window;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int s = s0 + 16 * t + 4 * kg + j;
            st[i][t][j] = s <= hi[i] && (s > lo || s < P.sinks) ? st[i][t][j] : -INFINITY;
          }
      }
    }
    float mx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float a = max3_raw(st[i][0][0], st[i][0][1], st[i][0][2]), c2 = max3_raw(st[i][2][0], st[i][2][1], st[i][2][2]);
      a = max3_raw(a, st[i][0][3], st[i][1][0]);
      c2 = max3_raw(c2, st[i][2][3], st[i][3][0]);
      a = max3_raw(a, st[i][1][1], st[i][1][2]);
      c2 = max3_raw(c2, st[i][3][1], st[i][3][2]);
      mx[i] = max3_raw(max3_raw(a, st[i][1][3], c2), st[i][3][3], st[i][3][3]);
    }
    if (__ballot(mx[0] > thr[0] || mx[1] > thr[1]) != 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float cand = max_rows4(mx[i]) * sl2;
        const bool bump = cand > m[i] + 8.f;
        const float m_new = bump ? cand : m[i];
        const float alpha = bump ? __builtin_amdgcn_exp2f(m[i] - m_new) : 1.f;
        m[i] = m_new;
        thr[i] = (m_new + 8.f) * inv_sl2;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[i][dt] *= alpha;
        lsum[i] *= alpha;
        l_full[i] *= alpha;
      }
    }
    u32x4_t pb[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float add[2] = {0.f, 0.f};
#pragma unroll
      for (int hc = 0; hc < 2; ++hc)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const f32x4_t& x = st[i][2 * hc + (w >> 1)];
          const float pa = __builtin_amdgcn_exp2f(fmaf(x[2 * (w & 1)], sl2, -m[i]));
          const float pc = __builtin_amdgcn_exp2f(fmaf(x[2 * (w & 1) + 1], sl2, -m[i]));
          pb[i][hc][w] = bf_cvt2(pa, pc);
          if (LSE) add[w & 1] += pa + pc;
        }
      if (LSE) l_full[i] += add[0] + add[1];
    }
#pragma unroll
    for (int hc = 0; hc < 2; ++hc) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x4_t a = sab_trow<HD>(smem, tr_off + at, dt, TB + 32 * hc * HD * 2);
        acc[0][dt] = mfma16x16x32(a, pb[0][hc], acc[0][dt]);
        acc[1][dt] = mfma16x16x32(a, pb[1][hc], acc[1][dt]);
      }
      lsum[0] = mfma16x16x32(ones, pb[0][hc], lsum[0]);
      lsum[1] = mfma16x16x32(ones, pb[1][hc], lsum[1]);
    }
  };

  __syncthreads();  // the first tile is there
  for (int c = range.lo; c < range.hi; ++c) {
    load(c + 1);
    step(c);
    __syncthreads();
  }

  if (LSE) {
#pragma unroll
    for (int i = 0; i < 2; ++i) l_full[i] = sum_rows4(l_full[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int qi = iw + 16 * i + r;
    if (qi >= P.Tq) continue;
    if (P.ksplit > 1) {
      float* row = sk_part_row(P, blockIdx.z, b, h, qi);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(row + 16 * dt + 4 * kg) = acc[i][dt];
      if (kg == 0) *reinterpret_cast<f32x4_t*>(row + HD) = f32x4_t{m[i], lsum[i][0], l_full[i], 0.f};
      continue;
    }
    const float l = lsum[i][0], inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = b * P.os_b + h * P.os_h + qi * P.os_t + 4 * kg;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const f32x4_t x = acc[i][dt] * inv;
      const u32x2_t w = u32x2_t{bf_cvt2(x[0], x[1]), bf_cvt2(x[2], x[3])};
      *reinterpret_cast<u32x2_t*>(static_cast<bf16_t*>(P.o) + at + 16 * dt) = w;
      if (LSE && P.olo) {
        const u32x2_t e = u32x2_t{bf_cvt2(x[0] - lo_bf16(w[0]), x[1] - hi_bf16(w[0])),
                                  bf_cvt2(x[2] - lo_bf16(w[1]), x[3] - hi_bf16(w[1]))};
        *reinterpret_cast<u32x2_t*>(static_cast<bf16_t*>(P.olo) + at + 16 * dt) = e;
      }
    }
    if (LSE && kg == 0)
      P.lse[(static_cast<int64_t>(b) * P.Hq + h) * P.Tq + qi] = l == 0.f ? INFINITY : m[i] + __log2f(l_full[i]);
  }
}

// ---------------------------------------------------------------------------
// dQ, and D for the key kernel.  A workgroup of 4 waves is HPW query heads of one KV head at
// 64 * 2 / HPW queries; a wave is one head's 32 queries over 32 keys at a time.  2 x 4096 tokens, window
// 1024, 32 / 8 heads of 128: 201 us for 6 hd flops a pair (900 TFLOP/s); dS in two terms 235.  The
// next 32 keys' scores beside this half's exponents (whole tiles, in one block): 219 - 231 us.
// ---------------------------------------------------------------------------
template <int HD, int HPW, bool FINE>
__global__ __launch_bounds__(SB_THREADS, sb_blocks(HD)) void sb_dq_kernel(SkParams P) {
  constexpr int KS = HD / 32, DT = HD / 16, TB = sab_tile_bytes<HD>();
  constexpr int QW = SB_WAVES / HPW * 32;
  __shared__ __attribute__((aligned(1024))) char smem[2 * 2 * TB];  // [stage][K, V]
  const int per = P.Hq / HPW;
  const int hp = static_cast<int>(blockIdx.x) % per, b = blockIdx.y;
  const int i0 = (static_cast<int>(gridDim.x) / per - 1 - static_cast<int>(blockIdx.x) / per) * QW;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, kg = lane >> 4;
  const int g = hp % P.Hkv, h = g * (P.Hq / P.Hkv) + hp / P.Hkv * HPW + wave % HPW;
  const int off = P.Tk - P.Tq, len = sk_length(P, b);
  const int iw = i0 + 32 * (wave / HPW), pw = off + iw, pw1 = off + min(iw + 32, P.Tq) - 1;
  const bf16_t* k = static_cast<const bf16_t*>(P.k) + b * P.ks_b + g * P.ks_h;
  const bf16_t* v = static_cast<const bf16_t*>(P.v) + b * P.vs_b + g * P.vs_h;
  const SkTiles tiles = sk_key_tiles(P, off + i0, min(off + min(i0 + QW, P.Tq), len) - 1);
  const SkRange range = sk_key_part(P, tiles.count(), blockIdx.z);
  const SbLoad<HD> copy;
  auto load = [&](int c) {
    if (c >= range.hi) return;
    char* dst = smem + (c & 1) * (2 * TB);
    copy(k, P.ks_t, tiles.tile(c) * SK_T, len, dst);
    copy(v, P.vs_t, tiles.tile(c) * SK_T, len, dst + TB);
  };
  load(range.lo);
  u32x4_t q[2][KS], gr[2][KS];
  float lse[2], dd[2];
  int hi[2];
  const int64_t stat = (static_cast<int64_t>(b) * P.Hq + h) * P.Tq;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int qi = iw + 16 * i + r, ql = qi < P.Tq ? qi : P.Tq - 1;
    const bool live = qi < P.Tq && off + qi < len;
    sb_frag<HD>(static_cast<const bf16_t*>(P.q) + b * P.qs_b + h * P.qs_h, P.qs_t, ql, live, kg, q[i]);
    sb_frag<HD>(static_cast<const bf16_t*>(P.dout) + b * P.ds_b + h * P.ds_h, P.ds_t, ql, live, kg,
                gr[i]);
    u32x4_t of[KS], ol[KS];
    const int64_t head = b * P.os_b + h * P.os_h;
    const int only = live ? sk_only_key(P, off + qi) : -1;
    sb_frag<HD>(only < 0 ? static_cast<const bf16_t*>(P.o) + head : v, only < 0 ? P.os_t : P.vs_t, only < 0 ? ql : only,
                live, kg, of);
    sb_frag<HD>(static_cast<const bf16_t*>(P.olo ? P.olo : P.o) + head, P.os_t, ql, live && P.olo && only < 0, kg, ol);
    f32x4_t d = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) d = mfma16x16x32(of[s], gr[i][s], d);
#pragma unroll
    for (int s = 0; s < KS; ++s) d = mfma16x16x32(ol[s], gr[i][s], d);
    dd[i] = sk_diagonal(d, r, kg);
    lse[i] = live ? P.lse[stat + qi] : INFINITY;
    hi[i] = live ? off + qi : -1;
    if (qi < P.Tq && kg == 0 && blockIdx.z == 0) P.dd[stat + qi] = dd[i];
  }
  const float sl2 = P.scale * SB_LOG2E;
  f32x4_t acc[2][DT];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[i][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const uint32_t row_off = sab_row_off<HD>(r, kg), tr_off = sab_tr_off<HD>(r, kg);
  __syncthreads();
  for (int c = range.lo; c < range.hi; ++c) {
    load(c + 1);
    const int s0 = tiles.tile(c) * SK_T;
#pragma unroll 1
    for (int hc = 0; hc < 2; ++hc) {  // 32 keys at a time (not unrolled: register budget)
      const int a0 = s0 + 32 * hc;
      const SbKeys all = sb_keys(P, len, a0, 32, pw, pw1);
      if (all == SB_NONE) continue;
      const uint32_t at = (c & 1) * (2 * TB) + 32 * hc * HD * 2;
      f32x4_t st[2][2], dp[2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        st[0][t] = st[1][t] = dp[0][t] = dp[1][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4_t a = sab_row(smem, row_off + at, ks, 16 * t * HD * 2);
          const u32x4_t e = sab_row(smem, row_off + at, ks, 16 * t * HD * 2 + TB);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            st[i][t] = mfma16x16x32(a, q[i][ks], st[i][t]);
            dp[i][t] = mfma16x16x32(e, gr[i][ks], dp[i][t]);
          }
        }
      }
      // the mask is a loop of its own, so that whole tiles run without branches
      if (all != SB_ALL) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int lo = hi[i] - P.window;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int s = a0 + 16 * t + 4 * kg + j;
              st[i][t][j] = s <= hi[i] && (s > lo || s < P.sinks) ? st[i][t][j] : -INFINITY;
            }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)  // dS^T
            dp[i][t][j] = __builtin_amdgcn_exp2f(fmaf(st[i][t][j], sl2, -lse[i])) * (dp[i][t][j] - dd[i]);
      __builtin_amdgcn_iglp_opt(0);  // LDS reads spread between the products: 207 -> 201 us (the case above)
      u32x4_t ds[2], dl[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) sb_round<FINE>(dp[i][0], dp[i][1], ds[i], dl[i]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x4_t a = sab_trow<HD>(smem, tr_off + at, dt, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (FINE) acc[i][dt] = mfma16x16x32(a, dl[i], acc[i][dt]);
          acc[i][dt] = mfma16x16x32(a, ds[i], acc[i][dt]);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int qi = iw + 16 * i + r;
    if (qi >= P.Tq) continue;
    if (P.ksplit > 1) {
      float* row = sk_part_row(P, blockIdx.z, b, h, qi);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(row + 16 * dt + 4 * kg) = acc[i][dt] * P.scale;
      continue;
    }
    bf16_t* o = static_cast<bf16_t*>(P.dq) + (stat + qi) * HD + 4 * kg;
    const float f = P.scale;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<u32x2_t*>(o + 16 * dt) =
          u32x2_t{bf_cvt2(acc[i][dt][0] * f, acc[i][dt][1] * f), bf_cvt2(acc[i][dt][2] * f, acc[i][dt][3] * f)};
  }
}

// ---------------------------------------------------------------------------
// dK and dV of 64 keys: wave (query half, key half) owns 32 keys and, of every query tile, 32
// queries; the two query halves' sums meet in LDS at the end.  The same case: 270 us for 8 hd
// flops a pair (895 TFLOP/s); dS in two terms 367 at best, the registers then hold no more.
// The first S.tiles * S.parts workgroups of a KV head are the split sink tiles' (SkSinkSplit).
// ---------------------------------------------------------------------------
template <int HD, bool FINE>
__global__ __launch_bounds__(SB_THREADS, sb_blocks(HD)) void sb_dkv_kernel(SkParams P, SkSinkSplit S) {
  constexpr int KS = HD / 32, DT = HD / 16, TB = sab_tile_bytes<HD>();
  constexpr int STAGE = 2 * TB + 2 * AB_T * 4;    // Q, dout, then lse and D of the rows
  constexpr int SUMS = 2 * 2 * 2 * DT * 64 * 16;  // two waves' dK and dV accumulators
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE > SUMS ? 2 * STAGE : SUMS];
  const int b = blockIdx.y, g = static_cast<int>(blockIdx.x) % P.Hkv;
  // the parts of the sink tiles come first: they are the longest
  const int x = static_cast<int>(blockIdx.x) / P.Hkv, n_far = S.tiles * S.parts;
  const int tile = x < n_far ? x / S.parts : x - n_far, part = x < n_far ? x % S.parts : -1;
  const int s0 = tile * SK_T;
  const int G = P.Hq / P.Hkv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, kg = lane >> 4;
  const int wq = wave >> 1, sw = s0 + 32 * (wave & 1);  // this wave's keys sw + 16 kt + r
  const int off = P.Tk - P.Tq, len = sk_length(P, b), q_end = min(P.Tq, len - off);
  const bf16_t* k = static_cast<const bf16_t*>(P.k) + b * P.ks_b + g * P.ks_h;
  const bf16_t* v = static_cast<const bf16_t*>(P.v) + b * P.vs_b + g * P.vs_h;
  // queries [i_lo, i_hi) that reach the keys through the window, or the part's beyond it
  const int near_hi = sk_near_end(P, S, s0);
  const int i_lo = part < 0 ? max(0, s0 - off) / SK_T * SK_T : near_hi + part * S.span;
  const int i_hi = min(q_end, part < 0 ? near_hi : i_lo + S.span);
  u32x4_t kb[2][KS], vb[2][KS];
  f32x4_t dka[2][DT], dva[2][DT];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const int s = sw + 16 * kt + r, sl = s < P.Tk ? s : P.Tk - 1;
    sb_frag<HD>(k, P.ks_t, sl, s < len, kg, kb[kt]);
    sb_frag<HD>(v, P.vs_t, sl, s < len, kg, vb[kt]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dka[kt][dt] = dva[kt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t row_off = sab_row_off<HD>(r, kg) + 32 * wq * HD * 2;
  const uint32_t tr_off = sab_tr_off<HD>(r, kg) + 32 * wq * HD * 2;
  const float sl2 = P.scale * SB_LOG2E;
  const SbLoad<HD> copy;
  auto load = [&](int i, int hh, int stage) {
    char* dst = smem + stage * STAGE;
    const int h = g * G + hh;
    copy(static_cast<const bf16_t*>(P.q) + b * P.qs_b + h * P.qs_h, P.qs_t, i, q_end, dst);
    copy(static_cast<const bf16_t*>(P.dout) + b * P.ds_b + h * P.ds_h, P.ds_t, i, q_end, dst + TB);
    if (wave < 2) {
      const float* st = (wave ? P.dd : P.lse) + (static_cast<int64_t>(b) * P.Hq + h) * P.Tq + min(i + lane, q_end - 1);
      __builtin_amdgcn_global_load_lds((ab_glb_t*)st, (ab_lds_t*)(dst + 2 * TB + wave * AB_T * 4), 4, 0, 0);
    }
  };
  const SkRange heads = sk_head_part(P, blockIdx.z);
  int i = heads.lo < heads.hi ? i_lo : i_hi, hh = heads.lo, stage = 0;
  if (i < i_hi) load(i, hh, 0);
  __syncthreads();
  while (i < i_hi) {
    const int t0 = i, cur = stage * STAGE;
    stage ^= 1;
    if (++hh == heads.hi) {
      hh = heads.lo;
      i += SK_T;
    }
    if (i < i_hi) load(i, hh, stage);
    const int p0 = off + t0 + 32 * wq, p1 = off + min(t0 + 32 * wq + 32, q_end) - 1;
    const SbKeys all = sb_keys(P, len, sw, 32, p0, p1);
    if (all != SB_NONE) {
      f32x4_t s[2][2], dp[2][2];  // [key half][16-query part]: query 32 wq + 16 i + 4 kg + e, key r
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        s[0][qt] = s[1][qt] = dp[0][qt] = dp[1][qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4_t aq = sab_row(smem, row_off + cur, ks, 16 * qt * HD * 2);
          const u32x4_t ad = sab_row(smem, row_off + cur, ks, 16 * qt * HD * 2 + TB);
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            s[kt][qt] = mfma16x16x32(aq, kb[kt][ks], s[kt][qt]);
            dp[kt][qt] = mfma16x16x32(ad, vb[kt][ks], dp[kt][qt]);
          }
        }
      }
      // the mask is a loop of its own, so that whole tiles run without branches
      if (all != SB_ALL || t0 + 32 * wq + 32 > q_end) {
#pragma unroll
        for (int qt = 0; qt < 2; ++qt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = t0 + 32 * wq + 16 * qt + 4 * kg + e;
            const int last = t < q_end ? off + t : -1, lo = last - P.window;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
              const int key = sw + 16 * kt + r;
              s[kt][qt][e] = key <= last && (key > lo || key < P.sinks) ? s[kt][qt][e] : -INFINITY;
            }
          }
      }
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        const int rq = 32 * wq + 16 * qt + 4 * kg;
        const float* rows = reinterpret_cast<const float*>(smem + cur + 2 * TB) + rq;
        const f32x4_t lse = *reinterpret_cast<const f32x4_t*>(rows);
        const f32x4_t rd = *reinterpret_cast<const f32x4_t*>(rows + AB_T);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[kt][qt][e], sl2, -lse[e]));
            dp[kt][qt][e] = p * (dp[kt][qt][e] - rd[e]);  // dS
            s[kt][qt][e] = p;
          }
      }
      u32x4_t ph[2], dh[2], dl[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        sb_round<false>(s[kt][0], s[kt][1], ph[kt], dl[kt]);
        sb_round<FINE>(dp[kt][0], dp[kt][1], dh[kt], dl[kt]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x4_t ad = sab_trow<HD>(smem, tr_off + cur, dt, TB);
        const u32x4_t aq = sab_trow<HD>(smem, tr_off + cur, dt, 0);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          dva[kt][dt] = mfma16x16x32(ad, ph[kt], dva[kt][dt]);
          if (FINE) dka[kt][dt] = mfma16x16x32(aq, dl[kt], dka[kt][dt]);
          dka[kt][dt] = mfma16x16x32(aq, dh[kt], dka[kt][dt]);
        }
      }
    }
    __syncthreads();
  }
  // the second query half hands its sums over, the first stores
  f32x4_t* sums = reinterpret_cast<f32x4_t*>(smem) + (wave & 1) * (4 * DT * 64) + lane;
  if (wq == 1) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        sums[(2 * (kt * DT + dt)) * 64] = dka[kt][dt];
        sums[(2 * (kt * DT + dt) + 1) * 64] = dva[kt][dt];
      }
  }
  __syncthreads();
  if (wq == 1) return;
  const int64_t head = static_cast<int64_t>(b) * P.Hkv + g;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const int s = sw + 16 * kt + r;
    if (s >= P.Tk) continue;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const f32x4_t ka = (dka[kt][dt] + sums[(2 * (kt * DT + dt)) * 64]) * P.scale;
      const f32x4_t va = dva[kt][dt] + sums[(2 * (kt * DT + dt) + 1) * 64];
      if (float* t = sk_kv_term(P, S, head, s, blockIdx.z, part)) {
        if (part >= 0 && s >= P.sinks) continue;
        *reinterpret_cast<f32x4_t*>(t + 16 * dt + 4 * kg) = ka;
        *reinterpret_cast<f32x4_t*>(t + HD + 16 * dt + 4 * kg) = va;
      } else if (part < 0) {
        const int64_t at = (head * P.Tk + s) * HD + 16 * dt + 4 * kg;
        *reinterpret_cast<u32x2_t*>(static_cast<bf16_t*>(P.dk) + at) = u32x2_t{bf_cvt2(ka[0], ka[1]), bf_cvt2(ka[2], ka[3])};
        *reinterpret_cast<u32x2_t*>(static_cast<bf16_t*>(P.dv) + at) = u32x2_t{bf_cvt2(va[0], va[1]), bf_cvt2(va[2], va[3])};
      }
    }
  }
}

}  // namespace

namespace fsi_sink {

bool sb_takes(const SkParams& P, int dtype, bool backward) {
  auto rows = [](const void* p, int64_t sb, int64_t sh, int64_t st) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && sb % 8 == 0 && sh % 8 == 0 && st % 8 == 0 && st >= 0 &&
           st < (int64_t(1) << 24);
  };
  return dtype == FSI_DTYPE_BF16 && (P.hd == 64 || P.hd == 128 || P.hd == 256) && P.scale > 0.f && P.Tq > 0 &&
         rows(P.q, P.qs_b, P.qs_h, P.qs_t) && rows(P.k, P.ks_b, P.ks_h, P.ks_t) && rows(P.v, P.vs_b, P.vs_h, P.vs_t) &&
         rows(P.o, P.os_b, P.os_h, P.os_t) && reinterpret_cast<uintptr_t>(P.olo) % 16 == 0 &&
         (!backward || (rows(P.dout, P.ds_b, P.ds_h, P.ds_t) &&
                        (reinterpret_cast<uintptr_t>(P.dq) | reinterpret_cast<uintptr_t>(P.dk) |
                         reinterpret_cast<uintptr_t>(P.dv)) % 8 == 0));
}

// Query heads that share a workgroup's K / V tiles: as many as divide the group.
static int sb_heads(const SkParams& P, int most) {
  const int G = P.Hq / P.Hkv;
  for (int n = most; n > 1; n /= 2)
    if (G % n == 0) return n;
  return 1;
}

int64_t sb_query_blocks(const SkParams& P, bool backward) {
  const int64_t heads = sb_heads(P, backward ? 2 : 4), queries = SB_WAVES / heads * 32;
  return (P.Tq + queries - 1) / queries * (P.Hq / heads) * P.B;
}

void sb_forward(const SkParams& P, hipStream_t st) {
  auto run = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    auto launch = [&](auto heads) {
      constexpr int HPW = decltype(heads)::value, QW = SB_WAVES / HPW * 32;
      const dim3 grid(static_cast<unsigned>((P.Tq + QW - 1) / QW * (P.Hq / HPW)), static_cast<unsigned>(P.B),
                      P.ksplit);
      if (P.lse) sb_fwd_kernel<HD, HPW, true><<<grid, SB_THREADS, 0, st>>>(P);
      else sb_fwd_kernel<HD, HPW, false><<<grid, SB_THREADS, 0, st>>>(P);
    };
    switch (sb_heads(P, 4)) {
      case 4: launch(std::integral_constant<int, 4>{}); break;
      case 2: launch(std::integral_constant<int, 2>{}); break;
      default: launch(std::integral_constant<int, 1>{});
    }
  };
  if (P.hd == 256) run(std::integral_constant<int, 256>{});
  else if (P.hd == 128) run(std::integral_constant<int, 128>{});
  else run(std::integral_constant<int, 64>{});
}

// Up to this many key tiles a launch leaves most of the card idle, and dS enters its products as two
// bf16 terms: with few keys a row, rounding it once is most of dq's and dk's error (2.4e-3 of their norm
// against 1.7e-3, which is their own rounding).  us of the backward, one term / two: heads of 64, 8
// heads of 512 tokens (64 tiles) 27.8 / 29.8; heads of 128, (4, 4 heads, 27) 13.6 / 14.6, 8 heads of 512
// 39.7 / 46.7.  Beyond, the product would be paid for in full: (1, 16 / 4 heads, 2048, 128) 151 / 190.
constexpr int SB_FINE_TILES = 64;
// Queries of up to SB_FINE_KEYS keys are too: the roundings of few terms do not average out (1 + 4 keys,
// 21 heads of 3160: 2.5e-3 against 1.8e-3), for a third more time (2 x 4096, 32 / 8 heads of 128, window
// 32: 179 / 247 us).
constexpr int SB_FINE_KEYS = 16;
static bool sb_fine(const SkParams& P) {
  return SB_FINE_TILES >= static_cast<int64_t>(P.B) * P.Hkv * ((P.Tk + SK_T - 1) / SK_T) ||
         SB_FINE_KEYS >= P.window + P.sinks;
}

void sb_backward(const SkParams& P, const SkSinkSplit& S, hipStream_t st) {
  auto run = [&](auto hd, auto fine) {
    constexpr int HD = decltype(hd)::value;
    constexpr bool FINE = decltype(fine)::value;
    auto launch = [&](auto heads) {
      constexpr int HPW = decltype(heads)::value, QW = SB_WAVES / HPW * 32;
      const dim3 grid(static_cast<unsigned>((P.Tq + QW - 1) / QW * (P.Hq / HPW)), static_cast<unsigned>(P.B),
                      P.ksplit);
      sb_dq_kernel<HD, HPW, FINE><<<grid, SB_THREADS, 0, st>>>(P);
    };
    if (sb_heads(P, 2) == 2) launch(std::integral_constant<int, 2>{});
    else launch(std::integral_constant<int, 1>{});
    const unsigned tiles = static_cast<unsigned>((P.Tk + SK_T - 1) / SK_T + S.tiles * S.parts);
    sb_dkv_kernel<HD, FINE><<<dim3(tiles * static_cast<unsigned>(P.Hkv), static_cast<unsigned>(P.B), P.hsplit),
                              SB_THREADS, 0, st>>>(P, S);
  };
  auto by_width = [&](auto fine) {
    if (P.hd == 256) run(std::integral_constant<int, 256>{}, fine);
    else if (P.hd == 128) run(std::integral_constant<int, 128>{}, fine);
    else run(std::integral_constant<int, 64>{}, fine);
  };
  if (sb_fine(P)) by_width(std::true_type{});
  else by_width(std::false_type{});
}

}  // namespace fsi_sink
