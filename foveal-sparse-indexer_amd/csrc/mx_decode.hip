// Decode attention over pages held in bf16, 8 or 4 bits (mx_cache.h): one query token per
// sequence, over the first `sinks` tokens, the last `window` tokens and listed pages.
//
//   ls = max(0, pos + 1 - window), se = min(sinks, ls)
//   support = [0, se) u [ls, pos] u the tokens of the listed pages inside [se, ls)
//   out = softmax(scale q K^T) V over the support
//
// Work split: a sequence's support is a list of chunks of TOK tokens (sinks, window, pages).
// Wave w of a workgroup takes a contiguous share of them for one KV head and up to 16 of its
// query heads (the MFMA N dimension), with a running maximum and sum:
//   S^T[t][h] = sum_d K[t][d] Q[h][d]       (A = K tile, B = Q^T)
//   O^T[d][h] += sum_t V^T[d][t] P^T[t][h]  (A = V^T tile, B = P^T from S^T's accumulators)
// Elements are widened to bf16 with their scale by v_cvt_scalef32_pk_bf16_{fp4,fp8}, which is
// exact; V's dim pairs are regrouped to token pairs by v_perm.  The contraction's dims may come
// in any order that Q follows, so a lane takes HD / 4 consecutive dims of its token.
// bf16 queries: P as a bf16 hi + lo pair (16 bits of P).  fp32 queries: Q and P as three
// bf16 parts (24 bits), the other operand exact, fp32 sums: an fp32 result.
// The workgroup's waves merge in LDS; several workgroups of a pair leave partials that a
// second kernel merges.
#include <algorithm>

#include "mx_cache.h"

using namespace fsi;
using namespace fsi_mx;

namespace {

constexpr int MD_MAX_WAVES = 8;
constexpr float MD_LOG2E = 1.4426950408889634f;

struct MdParams {
  const void* q;  // (B, Hq, HD)
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const int32_t* page_table;
  const int32_t* pos_rows;
  const int32_t* remote;
  const int32_t* counts;
  float* part;  // (B, Hkv, heads/16, wgs, 16 or G: max, sum) then (.., G, HD)
  void* out;
  int* err;
  int64_t n_phys;
  int B, Hq, Hkv, G, n_sub, wgs, waves, max_pages, cap, pos, window, sinks;
  float scale_log2;
};

typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2v_t;

template <int FMT, int SEL>
__device__ __forceinline__ uint32_t widen(uint32_t w, float s) {
  if constexpr (FMT == FMT_FP4)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, SEL != 0));
}

// N consecutive dwords at p (aligned to the largest power of two in 4 N bytes, at most 16), each
// read once per step: non-temporal.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const u32x2_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(p) + i);
      w[2 * i] = x[0];
      w[2 * i + 1] = x[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p) + i);
  }
}

__device__ __forceinline__ uint32_t pk_bf16(float a, float b) {
  const bf16x2v_t v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}

// Tokens of a chunk: as many as keep the chunk's K and V within 32 registers a lane.
constexpr int md_tok(int fmt, int hd) { return mx_bits(fmt) * hd <= 512 ? 64 : 32; }

// A chunk's operands as they lie in memory.
template <int FMT, int HD>
struct MdChunk {
  static constexpr int TOK = md_tok(FMT, HD), NT = TOK / 16, HALVES = TOK / 32, NG = HD / 32, KS = HD / 32;
  static constexpr bool MX = FMT != FMT_BF16;
  // the next chunk's loads run ahead of this one's products, where two chunks fit the registers
  static constexpr bool AHEAD = TOK * HD * mx_bits(FMT) <= 32 * 1024 || !MX;
  static constexpr int KW = HD * mx_bits(FMT) / 128;  // dwords of a lane's dims of one K tile
  // distinct scale dwords of a lane's dims: 8-dim step ks lies in group (grp HD / 4 + 8 ks) / 32
  static constexpr int SG = HD == 96 ? 3 : (HD <= 128 ? 1 : HD / 128);
  static constexpr int VW = MX ? HALVES * 4 * mx_bits(FMT) / 8 : 4;  // dwords of a lane's V piece of one group
  static constexpr int VP = MX ? NG : HALVES * (HD / 16);            // V pieces
  uint32_t k[NT][KW];
  uint32_t ksc[MX ? SG : 1];
  uint32_t v[VP][VW];
  uint32_t vsc[MX ? NG : 1][MX ? HALVES * 2 : 1];

  // blk_k / blk_v: the (page, head) blocks; first: the chunk's first token in the page
  __device__ __forceinline__ void load(const uint8_t* blk_k, const uint8_t* blk_v, int first) {
    const int lane = threadIdx.x & 63, r = lane & 15, grp = lane >> 4;
    if constexpr (MX) {
      constexpr int ROWB = HD * mx_bits(FMT) / 8;
#pragma unroll
      for (int t = 0; t < NT; ++t) load_words<KW>(blk_k + (first + 16 * t + r) * ROWB + grp * (ROWB / 4), k[t]);
      const uint8_t* sk = blk_k + mx_codes_bytes(FMT, HD);
#pragma unroll
      for (int i = 0; i < SG; ++i) {
        const int group = HD == 96 ? (grp * 24 + 8 * i) / 32 : (grp * HD / 4) / 32 + i;
        ksc[i] = *reinterpret_cast<const uint32_t*>(sk + (group * 16 + r) * 4);
      }
      const int half = first / 32;
#pragma unroll
      for (int i = 0; i < NG; ++i)
        load_words<VW>(blk_v + ((i * 64 + lane) * 2 + half) * (2 * mx_bits(FMT)), v[i]);
      const uint8_t* sv = blk_v + mx_codes_bytes(FMT, HD) + grp * NG * 16 + half * 8;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        if constexpr (HALVES == 2) {
          const u32x4_t x = *reinterpret_cast<const u32x4_t*>(sv + i * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) vsc[i][j] = x[j];
        } else {
          const u32x2_t x = *reinterpret_cast<const u32x2_t*>(sv + i * 16);
          vsc[i][0] = x[0];
          vsc[i][1] = x[1];
        }
      }
    } else {
      // K [HD/32][64 tokens][32 dims], V [half][HD dims][32 slots], bf16
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t w[4];
          load_words<4>(blk_k + ((ks * 64 + first + 16 * t + r) * 32 + 8 * grp) * 2, w);
#pragma unroll
          for (int j = 0; j < 4; ++j) k[t][4 * ks + j] = w[j];
        }
#pragma unroll
      for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt)
          load_words<4>(blk_v + (((first / 32 + hf) * HD + 16 * dt + r) * 32 + 8 * grp) * 2, v[hf * (HD / 16) + dt]);
    }
  }

  // A operand of 16-token tile t (tile t0 + t of the page), 32-dim step ks.
  template <int T, int KSI>
  __device__ __forceinline__ u32x4_t k_op(int t0) const {
    if constexpr (!MX) {
      return u32x4_t{k[T][4 * KSI], k[T][4 * KSI + 1], k[T][4 * KSI + 2], k[T][4 * KSI + 3]};
    } else {
      const uint32_t sw = ksc[SG == 1 ? 0 : (HD == 96 ? KSI : KSI / 4)];
      const float s = __uint_as_float(((sw >> (8 * (t0 + T))) & 0xffu) << 23);
      if constexpr (FMT == FMT_FP4) {
        const uint32_t w = k[T][KSI];
        return u32x4_t{widen<FMT, 0>(w, s), widen<FMT, 1>(w, s), widen<FMT, 2>(w, s), widen<FMT, 3>(w, s)};
      } else {
        const uint32_t a = k[T][2 * KSI], b = k[T][2 * KSI + 1];
        return u32x4_t{widen<FMT, 0>(a, s), widen<FMT, 1>(a, s), widen<FMT, 0>(b, s), widen<FMT, 1>(b, s)};
      }
    }
  }

  // A operands of dims 32 i + 2 r (x) and the next (y), the 8 tokens of half hf that the lane holds.
  template <int I, int HF>
  __device__ __forceinline__ void v_pair(u32x4_t& x, u32x4_t& y) const {
    uint32_t p[8];  // token e: (dim, dim + 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = __uint_as_float(((vsc[I][2 * HF + e / 4] >> (8 * (e & 3))) & 0xffu) << 23);
      if constexpr (FMT == FMT_FP4) {
        const uint32_t w = v[I][2 * HF + e / 4];
        switch (e & 3) {
          case 0: p[e] = widen<FMT, 0>(w, s); break;
          case 1: p[e] = widen<FMT, 1>(w, s); break;
          case 2: p[e] = widen<FMT, 2>(w, s); break;
          default: p[e] = widen<FMT, 3>(w, s); break;
        }
      } else {
        const uint32_t w = v[I][4 * HF + e / 2];
        p[e] = e & 1 ? widen<FMT, 1>(w, s) : widen<FMT, 0>(w, s);
      }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      x[w] = __builtin_amdgcn_perm(p[2 * w + 1], p[2 * w], 0x05040100u);
      y[w] = __builtin_amdgcn_perm(p[2 * w + 1], p[2 * w], 0x07060302u);
    }
  }
};

// Q^T operands of a lane's head, in PARTS bf16 parts whose sum is the query.
template <int FMT, int HD, int PARTS>
__device__ __forceinline__ void md_load_q(const MdParams& P, int b, int g, int sub, u32x4_t (&q)[PARTS][HD / 32]) {
  const int lane = threadIdx.x & 63, r = lane & 15, grp = lane >> 4;
  const int h = 16 * sub + r;
  const int64_t row = (static_cast<int64_t>(b) * P.Hq + g * P.G + h) * HD;
#pragma unroll
  for (int ks = 0; ks < HD / 32; ++ks) {
    const int d0 = FMT == FMT_BF16 ? 32 * ks + 8 * grp : grp * (HD / 4) + 8 * ks;
#pragma unroll
    for (int pt = 0; pt < PARTS; ++pt) q[pt][ks] = u32x4_t{0u, 0u, 0u, 0u};
    if (h >= P.G) continue;
    if constexpr (PARTS == 1) {
      q[0][ks] = *reinterpret_cast<const u32x4_t*>(static_cast<const bf16_t*>(P.q) + row + d0);
    } else {
      const f32x4_t* src = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(P.q) + row + d0);
      const f32x4_t x0 = src[0], x1 = src[1];
      float x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
#pragma unroll
      for (int pt = 0; pt < PARTS; ++pt)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t hi = pk_bf16(x[2 * w], x[2 * w + 1]);
          q[pt][ks][w] = hi;
          x[2 * w] -= lo_bf16(hi);
          x[2 * w + 1] -= hi_bf16(hi);
        }
    }
  }
}

template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

// PP parts of P beside the query's PARTS: 2 for bf16 outputs, 3 for fp32.  Bound by bytes where
// every CU has work: 8 x 65536 tokens of 8 heads of 128 in 4 bits (570 MB) take 107 us, 5.3 TB/s;
// 64 ragged sequences of bf16 pages (271 MB) 48.8 us, 5.5 TB/s.
template <int FMT, int HD, int PARTS>
__global__ __launch_bounds__(64 * MD_MAX_WAVES) void md_partial_kernel(MdParams P) {
  using Chunk = MdChunk<FMT, HD>;
  constexpr int TOK = Chunk::TOK, NT = Chunk::NT, HALVES = Chunk::HALVES, KS = HD / 32, DT = HD / 16;
  constexpr int PP = PARTS == 1 ? 2 : 3;
  extern __shared__ __attribute__((aligned(16))) float md_smem[];  // [wave][16] max, sum; [wave][G][HD]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, grp = lane >> 4;
  int y = blockIdx.x;
  const int wg = y % P.wgs;
  y /= P.wgs;
  const int sub = y % P.n_sub;
  y /= P.n_sub;
  const int g = y % P.Hkv, b = y / P.Hkv;

  int pos = P.pos_rows ? P.pos_rows[b] : P.pos;
  if (pos >= P.max_pages * MX_PAGE) {  // only from pos_rows: the host checks a shared position
    if (lane == 0) set_error(P.err, FSI_ERR_INDEX_RANGE);
    pos = P.max_pages * MX_PAGE - 1;
  }
  const int end = pos < 0 ? 0 : pos + 1;
  const int ls = end - P.window > 0 ? end - P.window : 0;
  const int se = P.sinks < ls ? P.sinks : ls;
  // chunks: sinks, window, then the listed pages' pieces
  const int n_sink = (se + TOK - 1) / TOK;
  const int c_lo = ls / TOK;
  const int n_loc = end > ls ? (end - 1) / TOK - c_lo + 1 : 0;
  int cnt = P.cap > 0 ? P.counts[b] : 0;
  cnt = cnt < 0 ? 0 : (cnt > P.cap ? P.cap : cnt);
  constexpr int PIECES = MX_PAGE / TOK;
  const int n_chunks = n_sink + n_loc + PIECES * cnt;
  const int n_waves = P.wgs * P.waves;
  const int per = (n_chunks + n_waves - 1) / n_waves;
  const int c0 = (wg * P.waves + wave) * per;
  const int c1 = c0 + per < n_chunks ? c0 + per : n_chunks;

  u32x4_t q[PARTS][KS];
  md_load_q<FMT, HD, PARTS>(P, b, g, sub, q);
  f32x4_t acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  const int64_t blk_bytes = mx_block_bytes(FMT, HD);

  for (int base = c0; base < c1; base += 64) {
    // chunk base + lane: its block, first token in the page, attended tokens [lo, hi) of the chunk
    int64_t blk = 0;
    int first = 0, lo = 0, hi = 0;
    const int c = base + lane;
    if (c < c1) {
      int page, t_lo, t_hi;
      if (c < n_sink + n_loc) {
        const int ca = c < n_sink ? c : c_lo + (c - n_sink);
        page = ca / PIECES;
        first = (ca % PIECES) * TOK;
        t_lo = c < n_sink ? 0 : ls;
        t_hi = c < n_sink ? se : end;
      } else {
        const int j = c - n_sink - n_loc;
        page = P.remote[static_cast<int64_t>(b) * P.cap + j / PIECES];
        first = (j % PIECES) * TOK;
        t_lo = se;
        t_hi = ls;
      }
      int64_t phys = -1;
      if (page >= 0 && page < P.max_pages) phys = P.page_table[static_cast<int64_t>(b) * P.max_pages + page];
      if (phys < 0 || phys >= P.n_phys) {
        set_error(P.err, FSI_ERR_INDEX_RANGE);
        phys = 0;  // read, but no token of it is attended
      } else {
        const int t0 = page * MX_PAGE + first;
        lo = t_lo - t0 > 0 ? t_lo - t0 : 0;
        hi = t_hi - t0 < TOK ? t_hi - t0 : TOK;
      }
      blk = (phys * P.Hkv + g) * blk_bytes;
    }
    const int n = c1 - base < 64 ? c1 - base : 64;
    auto at = [&](int i, int& f) {
      const uint32_t a = __builtin_amdgcn_readlane(static_cast<uint32_t>(blk), i);
      const uint32_t h = __builtin_amdgcn_readlane(static_cast<uint32_t>(blk >> 32), i);
      f = __builtin_amdgcn_readlane(first, i);
      return static_cast<int64_t>((static_cast<uint64_t>(h) << 32) | a);
    };
    auto load = [&](Chunk& ch, int i) {
      int f;
      const int64_t o = at(i, f);
      ch.load(P.k_pool + o, P.v_pool + o, f);
    };
    Chunk cur, nxt;
    if (Chunk::AHEAD) load(cur, 0);
    for (int i = 0; i < n; ++i) {
      int f_cur;
      at(i, f_cur);
      if (Chunk::AHEAD) load(nxt, i + 1 < n ? i + 1 : i);  // the last one re-reads
      else load(cur, i);
      const int lo_t = __builtin_amdgcn_readlane(lo, i), hi_t = __builtin_amdgcn_readlane(hi, i);

      f32x4_t st[NT];
      const int t0 = TOK == 64 ? 0 : f_cur / 16;
      static_for<NT>([&](auto t) {
        st[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        static_for<KS>([&](auto ks) {
          const u32x4_t a = cur.template k_op<t, ks>(t0);
#pragma unroll
          for (int pt = 0; pt < PARTS; ++pt) st[t] = mfma16x16x32(a, q[PARTS - 1 - pt][ks], st[t]);
        });
      });
      // lane: tokens 16 t + 4 grp + j for head r
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tau = 16 * t + 4 * grp + j;
          st[t][j] = tau >= lo_t && tau < hi_t ? st[t][j] * P.scale_log2 : -INFINITY;
          mx = fmaxf(mx, st[t][j]);
        }
      mx = max_rows4(mx);
      const float m_new = fmaxf(m_run, mx);
      // nothing attended yet: exponents against 0 give p = 0 (and keep a NaN score's NaN)
      const float m_ref = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_ref);
      m_run = m_new;
      float psum = 0.f;
      u32x4_t pb[PP][HALVES];
#pragma unroll
      for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int t = 2 * hf + (w >> 1), j = 2 * (w & 1);
          float a = __builtin_amdgcn_exp2f(st[t][j] - m_ref), c2 = __builtin_amdgcn_exp2f(st[t][j + 1] - m_ref);
          psum += a + c2;
#pragma unroll
          for (int pp = 0; pp < PP; ++pp) {
            const uint32_t h = pk_bf16(a, c2);
            pb[pp][hf][w] = h;
            a -= lo_bf16(h);
            c2 -= hi_bf16(h);
          }
        }
      l_run = l_run * alpha + sum_rows4(psum);
      if (__ballot(alpha != 1.f) != 0) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
      }
      // slots of tokens that are not attended hold anything: zero them
      const bool part = lo_t > 0 || hi_t < TOK;
      auto mask = [&](u32x4_t& a, int hf) {
        if (!part) return;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int tau = 32 * hf + 16 * (w >> 1) + 4 * grp + 2 * (w & 1);
          const uint32_t m0 = tau >= lo_t && tau < hi_t ? 0x0000ffffu : 0u;
          const uint32_t m1 = tau + 1 >= lo_t && tau + 1 < hi_t ? 0xffff0000u : 0u;
          a[w] &= m0 | m1;
        }
      };
      static_for<HALVES>([&](auto hf) {
        if constexpr (FMT == FMT_BF16) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const uint32_t(&w)[4] = cur.v[hf * DT + dt];
            u32x4_t a = u32x4_t{w[0], w[1], w[2], w[3]};
            mask(a, hf);
#pragma unroll
            for (int pp = 0; pp < PP; ++pp) acc[dt] = mfma16x16x32(a, pb[PP - 1 - pp][hf], acc[dt]);
          }
        } else {
          static_for<KS>([&](auto gi) {
            u32x4_t x, z;
            cur.template v_pair<gi, hf>(x, z);
            mask(x, hf);
            mask(z, hf);
#pragma unroll
            for (int pp = 0; pp < PP; ++pp) {
              acc[2 * gi] = mfma16x16x32(x, pb[PP - 1 - pp][hf], acc[2 * gi]);
              acc[2 * gi + 1] = mfma16x16x32(z, pb[PP - 1 - pp][hf], acc[2 * gi + 1]);
            }
          });
        }
      });
      if (Chunk::AHEAD) cur = nxt;
    }
  }

  // merge the workgroup's waves
  const int Gs = P.G - 16 * sub < 16 ? P.G - 16 * sub : 16;
  float* ml = md_smem;                           // [wave][2][16]
  float* ov = md_smem + MD_MAX_WAVES * 2 * 16;   // [wave][Gs][HD]
  if (grp == 0) {
    ml[wave * 32 + r] = m_run;
    ml[wave * 32 + 16 + r] = l_run;
  }
  if (r < Gs) {
    float* o = ov + (wave * Gs + r) * HD;
    if constexpr (FMT == FMT_BF16) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(o + 16 * dt + 4 * grp) = acc[dt];
    } else {
      // dims 32 i + 8 grp + 2 j (even tile) and the next (odd tile)
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const f32x4_t a = acc[2 * i], c2 = acc[2 * i + 1];
        *reinterpret_cast<f32x4_t*>(o + 32 * i + 8 * grp) = f32x4_t{a[0], c2[0], a[1], c2[1]};
        *reinterpret_cast<f32x4_t*>(o + 32 * i + 8 * grp + 4) = f32x4_t{a[2], c2[2], a[3], c2[3]};
      }
    }
  }
  __syncthreads();
  const int64_t pair = (static_cast<int64_t>(b) * P.Hkv + g) * P.n_sub + sub;
  for (int idx = threadIdx.x; idx < Gs * HD; idx += blockDim.x) {
    const int h = idx / HD, d = idx % HD;
    float M = -INFINITY;
    for (int w = 0; w < P.waves; ++w) M = fmaxf(M, ml[w * 32 + h]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, o = 0.f;
    for (int w = 0; w < P.waves; ++w) {
      const float wt = __builtin_amdgcn_exp2f(ml[w * 32 + h] - ref);
      L = fmaf(ml[w * 32 + 16 + h], wt, L);
      o = fmaf(ov[(w * Gs + h) * HD + d], wt, o);
    }
    if (P.wgs == 1) {
      const int64_t at = (static_cast<int64_t>(b) * P.Hq + g * P.G + 16 * sub + h) * HD + d;
      const float x = L == 0.f ? 0.f : o / L;
      if constexpr (PARTS == 1) static_cast<bf16_t*>(P.out)[at] = f32_to_bf16(x);
      else static_cast<float*>(P.out)[at] = x;
    } else {
      float* p = P.part + (pair * P.wgs + wg) * (16 * (HD + 2));
      p[h * (HD + 2) + d] = o;
      if (d == 0) {
        p[h * (HD + 2) + HD] = M;
        p[h * (HD + 2) + HD + 1] = L;
      }
    }
  }
}

// The workgroups' partials of each (sequence, query head): one workgroup of HD threads.
template <typename T>
__global__ void md_merge_kernel(MdParams P, int hd) {
  const int b = blockIdx.x / P.Hq, hq = blockIdx.x % P.Hq;
  const int g = hq / P.G, hh = hq % P.G, sub = hh / 16, h = hh % 16;
  const int64_t pair = (static_cast<int64_t>(b) * P.Hkv + g) * P.n_sub + sub;
  const float* p0 = P.part + pair * P.wgs * (16 * (hd + 2)) + h * (hd + 2);
  const int64_t step = 16 * (hd + 2);
  float M = -INFINITY;
  for (int w = 0; w < P.wgs; ++w) M = fmaxf(M, p0[w * step + hd]);
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f, o = 0.f;
  for (int w = 0; w < P.wgs; ++w) {
    const float* p = p0 + w * step;
    const float wt = __builtin_amdgcn_exp2f(p[hd] - ref);
    L = fmaf(p[hd + 1], wt, L);
    o = fmaf(p[threadIdx.x], wt, o);
  }
  const float x = L == 0.f ? 0.f : o / L;
  const int64_t at = (static_cast<int64_t>(b) * P.Hq + hq) * hd + threadIdx.x;
  if constexpr (sizeof(T) == 2) static_cast<bf16_t*>(P.out)[at] = f32_to_bf16(x);
  else static_cast<float*>(P.out)[at] = x;
}

// Waves per workgroup and workgroups per (sequence, KV head, 16 query heads), a pair below.
// Eight waves a CU stream with enough loads in flight, so one round of workgroups holds
// MD_SLOTS = 256 CUs x 8 waves.  Where the pairs alone give that, a pair is one workgroup of up
// to 8 waves and needs no merge; fewer pairs are cut into workgroups of 4 waves, as many as one
// round holds (a second round of a few workgroups would double the time), and no more than the
// chunks per wave that results needs.  us at 2048 / 1536 / 4096 slots: 32 sequences of 1024 + 32
// pages, 4 bits, 24.8 / 29.2 / 29.9; 48 ragged ones to 4096, 8 bits, 16.8 / 19.1 / 19.4; 8 of 65536
// tokens 108.8 / 126 / 108.
struct MdSplit {
  int waves, wgs;
};
constexpr int64_t MD_SLOTS = 2048;
MdSplit md_split(int64_t pairs, int64_t hd, int format, int64_t window, int64_t sinks, int64_t cap,
                 int64_t max_pages) {
  const int64_t tok = md_tok(format, hd), most_int = 0x7fffffff;
  window = std::min(window, most_int);
  sinks = std::min(sinks, most_int);
  cap = std::min(cap, most_int);
  max_pages = std::min(max_pages, most_int / MX_PAGE);
  const int64_t all = max_pages * (MX_PAGE / tok);
  const int64_t local = std::min<int64_t>(window / tok + 2, all);
  const int64_t chunks = std::min<int64_t>((sinks + tok - 1) / tok, all) + local + cap * (MX_PAGE / tok);
  const int64_t most = std::max<int64_t>(MD_SLOTS / pairs, 1);  // waves a pair may have
  if (chunks <= MD_MAX_WAVES || most <= MD_MAX_WAVES)
    return {static_cast<int>(std::min<int64_t>({chunks, most, MD_MAX_WAVES})), 1};
  const int64_t wgs = std::min<int64_t>(most / 4, (chunks + 3) / 4);
  const int64_t per = (chunks + 4 * wgs - 1) / (4 * wgs);
  const int64_t need = (chunks + 4 * per - 1) / (4 * per);
  return need <= 2 ? MdSplit{MD_MAX_WAVES, 1} : MdSplit{4, static_cast<int>(need)};
}

int64_t md_subs(int64_t Hq, int64_t Hkv) { return (Hq / Hkv + 15) / 16; }

}  // namespace

extern "C" {

FSI_API size_t fsi_decode_attn_sinks_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t head_dim, int format,
                                                    int64_t window, int64_t sinks, int64_t capacity,
                                                    int64_t max_pages) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || head_dim <= 0 || head_dim > 256 || max_pages <= 0 ||
      window < 0 || sinks < 0 || capacity < 0 || B > 0x7fffffff / Hkv || format < FSI_KV_BF16 || format > FSI_KV_MXFP4)
    return 0;
  const int64_t pairs = B * Hkv * md_subs(Hq, Hkv);
  const MdSplit s = md_split(pairs, head_dim, format, window, sinks, capacity, max_pages);
  return s.wgs == 1 ? 0 : sizeof(float) * static_cast<size_t>(pairs * s.wgs * 16 * (head_dim + 2));
}

FSI_API int fsi_decode_attn_sinks(const void* q, int dtype, const void* k_pool, const void* v_pool, int format,
                                  const int32_t* page_table, int64_t max_pages, int64_t n_phys_pages,
                                  const int32_t* pos_rows, int64_t pos, int64_t window, int64_t sinks,
                                  const int32_t* remote_pages, const int32_t* remote_counts, int64_t capacity,
                                  int64_t B, int64_t Hq, int64_t Hkv, int64_t head_dim, float scale, void* out,
                                  void* workspace, size_t workspace_bytes, int* err, void* stream) {
  using namespace fsi_host;
  FSI_CHECK_ARG(format == FSI_KV_BF16 || format == FSI_KV_MXFP8 || format == FSI_KV_MXFP4, FSI_ERR_INVALID_ARG,
                "decode_attn_sinks: format %d", format);
  FSI_CHECK_ARG(dtype == FSI_DTYPE_BF16 || (dtype == FSI_DTYPE_F32 && format != FSI_KV_BF16), FSI_ERR_DTYPE,
                "decode_attn_sinks: dtype %d (bf16 pages take bf16 queries)", dtype);
  const bool hd_ok = format == FSI_KV_BF16 ? head_dim == 64 || head_dim == 128
                                           : fsi_kv_mx_block_bytes(head_dim, format) > 0;
  FSI_CHECK_ARG(hd_ok, FSI_ERR_SHAPE, "decode_attn_sinks: head_dim %lld (bf16 pages 64 or 128, else 64, 96, 128, 256)",
                (long long)head_dim);
  FSI_CHECK_ARG(B >= 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0, FSI_ERR_SHAPE,
                "decode_attn_sinks: B %lld, Hq %lld, Hkv %lld", (long long)B, (long long)Hq, (long long)Hkv);
  FSI_CHECK_ARG(B <= 0x7fffffff / Hq, FSI_ERR_SHAPE, "decode_attn_sinks: B * Hq beyond int32");
  FSI_CHECK_ARG(max_pages > 0 && n_phys_pages > 0 && window >= 0 && sinks >= 0 && pos >= 0 && capacity >= 0,
                FSI_ERR_SHAPE, "decode_attn_sinks: bad sizes");
  FSI_CHECK_ARG(max_pages <= 0x7fffffff / MX_PAGE && B <= 0x7fffffff && Hq <= 0x7fffffff && capacity <= 0x1000000,
                FSI_ERR_SHAPE, "decode_attn_sinks: sizes beyond int32");
  FSI_CHECK_ARG(pos_rows || pos < max_pages * MX_PAGE, FSI_ERR_INDEX_RANGE,
                "decode_attn_sinks: position %lld beyond the page table (%lld pages)", (long long)pos,
                (long long)max_pages);
  if (B == 0) return FSI_OK;
  FSI_CHECK_ARG(q && k_pool && v_pool && page_table && out, FSI_ERR_INVALID_ARG, "decode_attn_sinks: null pointer");
  FSI_CHECK_ARG(capacity == 0 || (remote_pages && remote_counts), FSI_ERR_INVALID_ARG,
                "decode_attn_sinks: remote page list or counts missing");
  FSI_CHECK_ARG((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) |
                 reinterpret_cast<uintptr_t>(v_pool)) % 16 == 0,
                FSI_ERR_ALIGN, "decode_attn_sinks: q and pools must be 16-byte aligned");
  const size_t need = fsi_decode_attn_sinks_workspace_size(B, Hq, Hkv, head_dim, format, window, sinks, capacity,
                                                           max_pages);
  FSI_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                FSI_ERR_WORKSPACE, "decode_attn_sinks: workspace %zu < %zu bytes (or misaligned)", workspace_bytes,
                need);
  const int64_t subs = md_subs(Hq, Hkv), pairs = B * Hkv * subs;
  const MdSplit s = md_split(pairs, head_dim, format, window, sinks, capacity, max_pages);
  FSI_CHECK_ARG(pairs * s.wgs <= 0x7fffffff && B * Hq <= 0x7fffffff, FSI_ERR_SHAPE,
                "decode_attn_sinks: %lld workgroups beyond the grid", (long long)(pairs * s.wgs));
  MdParams P{};
  P.q = q;
  P.k_pool = static_cast<const uint8_t*>(k_pool);
  P.v_pool = static_cast<const uint8_t*>(v_pool);
  P.page_table = page_table;
  P.pos_rows = pos_rows;
  P.remote = remote_pages;
  P.counts = remote_counts;
  P.part = static_cast<float*>(workspace);
  P.out = out;
  P.err = err;
  P.n_phys = n_phys_pages;
  P.B = (int)B;
  P.Hq = (int)Hq;
  P.Hkv = (int)Hkv;
  P.G = (int)(Hq / Hkv);
  P.n_sub = (int)subs;
  P.wgs = s.wgs;
  P.waves = s.waves;
  P.max_pages = (int)max_pages;
  P.cap = (int)capacity;
  P.pos = (int)pos;
  P.window = (int)std::min<int64_t>(window, 0x7fffffff);
  P.sinks = (int)std::min<int64_t>(sinks, 0x7fffffff);
  P.scale_log2 = scale * MD_LOG2E;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(pairs * s.wgs), threads = static_cast<unsigned>(64 * s.waves);
  const int gs = P.G < 16 ? P.G : 16;
  const size_t lds = sizeof(float) * (MD_MAX_WAVES * 32 + static_cast<size_t>(s.waves) * gs * head_dim);
  auto run = [&](auto fmt, auto hd, auto parts) {
    auto* kern = &md_partial_kernel<decltype(fmt)::value, decltype(hd)::value, decltype(parts)::value>;
    if (lds > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    kern<<<grid, threads, lds, st>>>(P);
  };
  auto by_dtype = [&](auto fmt, auto hd) {
    if (dtype == FSI_DTYPE_BF16) run(fmt, hd, std::integral_constant<int, 1>{});
    else run(fmt, hd, std::integral_constant<int, 3>{});
  };
  auto by_hd = [&](auto fmt) {
    switch (head_dim) {
      case 64: by_dtype(fmt, std::integral_constant<int, 64>{}); break;
      case 96: by_dtype(fmt, std::integral_constant<int, 96>{}); break;
      case 128: by_dtype(fmt, std::integral_constant<int, 128>{}); break;
      default: by_dtype(fmt, std::integral_constant<int, 256>{}); break;
    }
  };
  if (format == FSI_KV_MXFP4) by_hd(std::integral_constant<int, FMT_FP4>{});
  else if (format == FSI_KV_MXFP8) by_hd(std::integral_constant<int, FMT_FP8>{});
  else if (head_dim == 64) run(std::integral_constant<int, FMT_BF16>{}, std::integral_constant<int, 64>{},
                               std::integral_constant<int, 1>{});
  else run(std::integral_constant<int, FMT_BF16>{}, std::integral_constant<int, 128>{},
           std::integral_constant<int, 1>{});
  FSI_HIP_LAUNCH_CHECK("decode_attn_sinks");
  if (s.wgs > 1) {
    const unsigned mg = static_cast<unsigned>(B * Hq);
    if (dtype == FSI_DTYPE_BF16) md_merge_kernel<bf16_t><<<mg, (unsigned)head_dim, 0, st>>>(P, (int)head_dim);
    else md_merge_kernel<float><<<mg, (unsigned)head_dim, 0, st>>>(P, (int)head_dim);
    FSI_HIP_LAUNCH_CHECK("decode_attn_sinks merge");
  }
  return FSI_OK;
}

}  // extern "C"
