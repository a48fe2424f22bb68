// K/V pages held in 8 or 4 bits: element formats, scales and memory layout.
//
// 32 consecutive dims of one token and head form a group x = value * 2^e: the values are
// e4m3 (|value| <= 448) or e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6), the scale is one byte e + 127.
//   e = the smallest integer with max|x| <= L 2^e, L = 464 or 7: the largest value plus half
//       a step, so clamping the largest element costs no more than a rounding does; kept in
//       [E_MIN, E_MAX], so 2^e and every value 2^e are zero or normal finite numbers of fp32
//       and bf16 (a value has at most 4 significant bits: bf16 holds the product exactly);
//   value = x 2^-e rounded to the nearest element, ties to even, clamped to the largest.
// A group with an infinity or a NaN has scale byte 255 and reads back as NaN.
//
// One block of a pool holds one (page of 64 tokens, KV head), W = bits / 8 bytes an element:
//   K: [64 tokens][HD W] element bytes, then scale bytes [HD/32 groups][16 r][4 tiles] of
//      token 16 tile + r.  Lane (r, grp) of a 16-token MFMA tile reads HD / 4 consecutive dims
//      of token r, and one dword holds a group's scales of token r in all four tiles.
//   V: [HD/32 groups][64 lanes][2 halves][8 slots] dim pairs (2 W bytes: dims 32 i + 2 r and
//      the next, lane = r + 16 grp; slot 8 grp + idx of half t / 32 is v_slot(t % 32)),
//      then scale bytes [4 grp][HD/32 groups][2 halves][8 slots].  Lane (r, grp) reads its
//      tokens' pairs of a group as one piece; a pair has one token, so one scale.
#pragma once

#include "fsi_common.h"

namespace fsi_mx {

constexpr int MX_PAGE = 64;
constexpr int MX_GROUP = 32;

enum Fmt : int { FMT_BF16 = FSI_KV_BF16, FMT_FP8 = FSI_KV_MXFP8, FMT_FP4 = FSI_KV_MXFP4 };

// Element bits, exponent of the largest element, mantissa field of the scale limit L, bounds of e.
template <int FMT>
struct MxFmt;
template <>
struct MxFmt<FMT_FP8> {
  static constexpr int BITS = 8, TOP = 8, E_MAX = 119;
  static constexpr uint32_t LIMIT_MANT = 0x680000u;  // 464 = 1.8125 * 2^8
};
template <>
struct MxFmt<FMT_FP4> {
  static constexpr int BITS = 4, TOP = 2, E_MAX = 125;
  static constexpr uint32_t LIMIT_MANT = 0x600000u;  // 7 = 1.75 * 2^2
};
constexpr int E_MIN = -116;
constexpr int SCALE_NAN = 255;

__host__ __device__ constexpr int mx_bits(int fmt) { return fmt == FMT_FP4 ? 4 : (fmt == FMT_FP8 ? 8 : 16); }
__host__ __device__ constexpr int64_t mx_codes_bytes(int fmt, int64_t hd) { return MX_PAGE * hd * mx_bits(fmt) / 8; }
// Bytes of one (page, head) block of a pool.
__host__ __device__ constexpr int64_t mx_block_bytes(int fmt, int64_t hd) {
  return mx_codes_bytes(fmt, hd) + (fmt == FMT_BF16 ? 0 : MX_PAGE * hd / MX_GROUP);
}

// MFMA k slot of token tau within a 32-token half (the order in which the two 16-token score
// tiles' accumulators hold the tokens).
__host__ __device__ __forceinline__ int mx_slot(int tau) { return 8 * ((tau & 15) >> 2) + 4 * (tau >> 4) + (tau & 3); }

// Byte offsets inside a block.
__device__ __forceinline__ int k_scale_off(int group, int t) { return (group * 16 + (t & 15)) * 4 + (t >> 4); }
template <int W2>  // bytes of a dim pair
__device__ __forceinline__ int v_pair_off(int group, int r, int t) {
  const int s = mx_slot(t & 31);
  return (((group * 64 + r + 16 * (s >> 3)) * 2 + (t >> 5)) * 8 + (s & 7)) * W2;
}
__device__ __forceinline__ int v_scale_off(int n_groups, int group, int t) {
  const int s = mx_slot(t & 31);
  return (((s >> 3) * n_groups + group) * 2 + (t >> 5)) * 8 + (s & 7);
}

// Scale byte of a group whose largest |x| has the fp32 bits `amax` (0 for an empty group; the
// fp32 bit patterns of non-negative numbers are ordered as the numbers, NaN above infinity).
// Adding the distance from L's mantissa to the next power of two carries into the exponent
// field exactly where the mantissa passes L's.
template <int FMT>
__device__ __forceinline__ int mx_scale_byte(uint32_t amax) {
  using F = MxFmt<FMT>;
  if (amax >= 0x7f800000u) return SCALE_NAN;
  int e = static_cast<int>((amax + (0x7fffffu - F::LIMIT_MANT)) >> 23) - 127 - F::TOP;
  e = e < E_MIN ? E_MIN : (e > F::E_MAX ? F::E_MAX : e);
  return e + 127;
}

// 2^(byte - 127), exact for bytes of finite groups.
__device__ __forceinline__ float mx_scale(int byte) { return __uint_as_float(static_cast<uint32_t>(byte) << 23); }

}  // namespace fsi_mx
