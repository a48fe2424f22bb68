// K/V pages held in 8 or 4 bits (mx_cache.h): writing tokens into the pools and reading
// them back.
#include <algorithm>

#include "mx_cache.h"

using namespace fsi;
using namespace fsi_mx;

namespace {

struct MxParams {
  const void* k;  // write: (B, Hkv, n_tok, HD) with element strides; read: unused
  const void* v;
  int64_t ks_b, ks_g, ks_t, vs_b, vs_g, vs_t;
  int B, Hkv, n_tok, hd;
  const int32_t* start_rows;
  int start;
  const int32_t* page_table;
  int max_pages;
  int64_t n_phys;
  uint8_t* k_pool;
  uint8_t* v_pool;
  void* k_out;  // read: contiguous (B, Hkv, n_tok, HD)
  void* v_out;
  int* err;
  unsigned pages;  // workgroups per (sequence, head)
  bool vec;  // write: every row of K and V starts 16-byte aligned
};

template <typename T>
__device__ __forceinline__ float mx_ld(const T* p);
template <>
__device__ __forceinline__ float mx_ld<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float mx_ld<bf16_t>(const bf16_t* p) { return bf16_to_f32(*p); }
// Largest of a lane quad (DPP, no LDS).
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  const uint32_t y = __builtin_amdgcn_mov_dpp(x, 0xB1, 0xF, 0xF, true);  // lane ^ 1
  x = x > y ? x : y;
  const uint32_t z = __builtin_amdgcn_mov_dpp(x, 0x4E, 0xF, 0xF, true);  // lane ^ 2
  return x > z ? x : z;
}

// 8 consecutive elements as fp32; vec: 16-byte aligned.
template <typename T>
__device__ __forceinline__ void mx_ld8(const T* p, bool vec, float (&x)[8]) {
  if (!vec) {
#pragma unroll
    for (int d = 0; d < 8; ++d) x[d] = mx_ld(p + d);
  } else if constexpr (sizeof(T) == 4) {
    const f32x4_t a = reinterpret_cast<const f32x4_t*>(p)[0], c = reinterpret_cast<const f32x4_t*>(p)[1];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      x[d] = a[d];
      x[4 + d] = c[d];
    }
  } else {
    const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      x[2 * w] = lo_bf16(a[w]);
      x[2 * w + 1] = hi_bf16(a[w]);
    }
  }
}
// Quantise the lane's 8 dims of a group whose other dims the lanes of its quad hold: the codes of
// dim pair e (2 bits / 8 bytes each), the scale byte returned.  v_cvt_scalef32_pk_{fp4,fp8}_f32
// divides by the scale and rounds to the nearest element, ties to even; the clamp before it takes
// what lies above the largest.  (Rounding in integer code instead, 10 instructions an element, made
// the vector units the bound: 8192-token prompts of 4 sequences written in 44 against 31 us, read
// back in 42 against 26.)
template <int FMT>
__device__ __forceinline__ int mx_quantise8(const float (&x)[8], uint32_t (&pair)[4]) {
  uint32_t amax = 0;
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    const uint32_t a = __float_as_uint(x[d]) & 0x7fffffffu;
    amax = a > amax ? a : amax;
  }
  const int byte = mx_scale_byte<FMT>(quad_max(amax));
  const float scale = mx_scale(byte), top = (FMT == FMT_FP4 ? 6.f : 448.f) * scale;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = __builtin_amdgcn_fmed3f(x[2 * e], -top, top), c = __builtin_amdgcn_fmed3f(x[2 * e + 1], -top, top);
    if constexpr (FMT == FMT_FP4) {
      pair[e] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, c, scale, 0) & 0xffu;
    } else {
      typedef short s16x2_t __attribute__((ext_vector_type(2)));
      const s16x2_t w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2_t{0, 0}, a, c, scale, false);
      pair[e] = static_cast<uint16_t>(w[0]);
    }
    if (byte == SCALE_NAN) pair[e] = 0u;
  }
  return byte;
}

// The values of 4 dim pairs' codes (pair e in the low bits of c[e]) at the scale byte.
template <typename T, int FMT>
__device__ __forceinline__ void mx_widen8(const uint32_t (&c)[4], int byte, T* dst) {
  const float scale = mx_scale(byte);
  const bool nan = byte == SCALE_NAN;
  if constexpr (sizeof(T) == 2) {
    u32x4_t w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (FMT == FMT_FP4)
        w[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[e], scale, 0));
      else
        w[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[e], scale, false));
      w[e] = nan ? 0x7fc07fc0u : w[e];
    }
    *reinterpret_cast<u32x4_t*>(dst) = w;
  } else {
    f32x4_t w[2];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      typedef float f32x2v_t __attribute__((ext_vector_type(2)));
      f32x2v_t y;
      if constexpr (FMT == FMT_FP4) y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[e], scale, 0);
      else y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[e], scale, false);
      w[e / 2][2 * (e & 1)] = nan ? __uint_as_float(0x7fc00000u) : y[0];
      w[e / 2][2 * (e & 1) + 1] = nan ? __uint_as_float(0x7fc00000u) : y[1];
    }
    reinterpret_cast<f32x4_t*>(dst)[0] = w[0];
    reinterpret_cast<f32x4_t*>(dst)[1] = w[1];
  }
}

constexpr int MX_THREADS = 256;

// A workgroup writes its share of one (page, head): a thread takes 8 dims of a token, a lane quad
// a group.  K's codes go straight to memory (a token's row is contiguous); V's codes and both
// scales are laid out in LDS, and leave as 16-byte pieces of a page that is written whole, as
// single pairs and bytes otherwise.  Bound by bytes: 4 x 8192 tokens, 8 heads of 128, bf16 to 4 bits
// (170 MB) take 31 - 35 us, 4.9 - 5.5 TB/s (with the read back 62 - 70; 364 with a wave per token and
// single pairs for every page).
template <typename T, int FMT, int HD>
__global__ __launch_bounds__(MX_THREADS) void mx_write_kernel(MxParams P) {
  constexpr int BITS = MxFmt<FMT>::BITS, W2 = 2 * BITS / 8, NG = HD / MX_GROUP, TPT = HD / 8;
  constexpr int CODES = MX_PAGE * HD * BITS / 8, SCALES = MX_PAGE * NG;
  __shared__ __attribute__((aligned(16))) uint8_t vimg[CODES + SCALES];
  __shared__ __attribute__((aligned(16))) uint8_t kscale[SCALES];
  const int bh = static_cast<int>(blockIdx.x / P.pages), g = bh % P.Hkv, b = bh / P.Hkv;
  const int64_t start = P.start_rows ? P.start_rows[b] : P.start;
  // the page that holds position start (rounded down for negative ones), then the later ones
  const int64_t page = (start >= 0 ? start / MX_PAGE : -((MX_PAGE - 1 - start) / MX_PAGE)) + blockIdx.x % P.pages;
  const int64_t t_base = page * MX_PAGE - start;  // input token of the page's first slot
  const int lo = t_base < 0 ? static_cast<int>(-t_base) : 0;
  const int hi = P.n_tok - t_base < MX_PAGE ? static_cast<int>(P.n_tok - t_base) : MX_PAGE;
  if (hi <= lo) return;
  int64_t phys = -1;
  if (page >= 0 && page < P.max_pages) phys = P.page_table[static_cast<int64_t>(b) * P.max_pages + page];
  if (phys < 0 || phys >= P.n_phys) {
    if (threadIdx.x == 0) set_error(P.err, FSI_ERR_INDEX_RANGE);
    return;
  }
  const int64_t base = (phys * P.Hkv + g) * (CODES + SCALES);
  const T* k = static_cast<const T*>(P.k) + b * P.ks_b + g * P.ks_g;
  const T* v = static_cast<const T*>(P.v) + b * P.vs_b + g * P.vs_g;
  const int piece = threadIdx.x % TPT, d0 = 8 * piece, group = piece / 4;
  // hd 96: 21 tokens of 12 threads a round; the last 4 threads idle
  for (int t = lo + static_cast<int>(threadIdx.x) / TPT; t < hi; t += MX_THREADS / TPT) {
    if (threadIdx.x >= MX_THREADS / TPT * TPT) break;
    const int64_t src = t_base + t;
    float x[8], y[8];
    mx_ld8(k + src * P.ks_t + d0, P.vec, x);
    mx_ld8(v + src * P.vs_t + d0, P.vec, y);
    uint32_t pair[4];
    const int kb = mx_quantise8<FMT>(x, pair);
    uint8_t* kd = P.k_pool + base + (t * HD + d0) * BITS / 8;
    if constexpr (FMT == FMT_FP4) {
      *reinterpret_cast<uint32_t*>(kd) = pair[0] | (pair[1] << 8) | (pair[2] << 16) | (pair[3] << 24);
    } else {
      *reinterpret_cast<u32x2_t*>(kd) = u32x2_t{pair[0] | (pair[1] << 16), pair[2] | (pair[3] << 16)};
    }
    const int vb = mx_quantise8<FMT>(y, pair);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint8_t* vd = vimg + v_pair_off<W2>(group, (piece % 4) * 4 + e, t);
      if constexpr (FMT == FMT_FP4) *vd = static_cast<uint8_t>(pair[e]);
      else *reinterpret_cast<uint16_t*>(vd) = static_cast<uint16_t>(pair[e]);
    }
    if (piece % 4 == 0) {
      kscale[k_scale_off(group, t)] = static_cast<uint8_t>(kb);
      vimg[CODES + v_scale_off(NG, group, t)] = static_cast<uint8_t>(vb);
    }
  }
  __syncthreads();
  uint8_t* kdst = P.k_pool + base + CODES;
  uint8_t* vdst = P.v_pool + base;
  if (lo == 0 && hi == MX_PAGE) {
    for (int i = threadIdx.x; i < (CODES + SCALES) / 16; i += MX_THREADS)
      reinterpret_cast<u32x4_t*>(vdst)[i] = reinterpret_cast<const u32x4_t*>(vimg)[i];
    for (int i = threadIdx.x; i < SCALES / 16; i += MX_THREADS)
      reinterpret_cast<u32x4_t*>(kdst)[i] = reinterpret_cast<const u32x4_t*>(kscale)[i];
    return;
  }
  for (int i = threadIdx.x; i < (hi - lo) * (HD / 2); i += MX_THREADS) {
    const int t = lo + i / (HD / 2), pr = i % (HD / 2), at = v_pair_off<W2>(pr / 16, pr % 16, t);
    if constexpr (FMT == FMT_FP4) vdst[at] = vimg[at];
    else *reinterpret_cast<uint16_t*>(vdst + at) = *reinterpret_cast<const uint16_t*>(vimg + at);
  }
  for (int i = threadIdx.x; i < (hi - lo) * NG; i += MX_THREADS) {
    const int t = lo + i / NG, gi = i % NG;
    kdst[k_scale_off(gi, t)] = kscale[k_scale_off(gi, t)];
    vdst[CODES + v_scale_off(NG, gi, t)] = vimg[CODES + v_scale_off(NG, gi, t)];
  }
}

// One page of a head back to rows: V's block through LDS, 8 dims of a token a thread.  0 where
// the page is not there.  The same 170 MB back take 26 - 27 us, 6.3 - 6.5 TB/s (the pages still lie
// in the cache after the write).
template <typename T, int FMT, int HD>
__global__ __launch_bounds__(MX_THREADS) void mx_read_kernel(MxParams P) {
  constexpr int BITS = MxFmt<FMT>::BITS, W2 = 2 * BITS / 8, NG = HD / MX_GROUP, TPT = HD / 8;
  constexpr int CODES = MX_PAGE * HD * BITS / 8, SCALES = MX_PAGE * NG;
  __shared__ __attribute__((aligned(16))) uint8_t vimg[CODES + SCALES];
  const int bh = static_cast<int>(blockIdx.x / P.pages), g = bh % P.Hkv, b = bh / P.Hkv;
  const int page = static_cast<int>(blockIdx.x % P.pages);
  const int hi = P.n_tok - page * MX_PAGE < MX_PAGE ? P.n_tok - page * MX_PAGE : MX_PAGE;
  int64_t phys = page < P.max_pages ? P.page_table[static_cast<int64_t>(b) * P.max_pages + page] : -1;
  if (phys >= P.n_phys) phys = -1;
  const int64_t base = (phys * P.Hkv + g) * (CODES + SCALES);
  if (phys >= 0) {
    for (int i = threadIdx.x; i < (CODES + SCALES) / 16; i += MX_THREADS)
      reinterpret_cast<u32x4_t*>(vimg)[i] = reinterpret_cast<const u32x4_t*>(P.v_pool + base)[i];
  }
  __syncthreads();
  const int piece = threadIdx.x % TPT, d0 = 8 * piece, group = piece / 4;
  const int64_t row0 = (static_cast<int64_t>(b) * P.Hkv + g) * P.n_tok + static_cast<int64_t>(page) * MX_PAGE;
  for (int t = static_cast<int>(threadIdx.x) / TPT; t < hi; t += MX_THREADS / TPT) {
    if (threadIdx.x >= MX_THREADS / TPT * TPT) break;
    T* kd = static_cast<T*>(P.k_out) + (row0 + t) * HD + d0;
    T* vd = static_cast<T*>(P.v_out) + (row0 + t) * HD + d0;
    uint32_t ck[4] = {0u, 0u, 0u, 0u}, cv[4] = {0u, 0u, 0u, 0u};
    int ks = 0, vs = 0;
    if (phys >= 0) {
      const uint8_t* kb = P.k_pool + base;
      const uint8_t* ksrc = kb + (t * HD + d0) * BITS / 8;
      ks = kb[CODES + k_scale_off(group, t)];
      vs = vimg[CODES + v_scale_off(NG, group, t)];
      u32x2_t w;
      if constexpr (FMT == FMT_FP4) w[0] = *reinterpret_cast<const uint32_t*>(ksrc);
      else w = *reinterpret_cast<const u32x2_t*>(ksrc);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ck[e] = FMT == FMT_FP4 ? w[0] >> (8 * e) : w[e >> 1] >> (16 * (e & 1));
        const uint8_t* vsrc = vimg + v_pair_off<W2>(group, (piece % 4) * 4 + e, t);
        cv[e] = FMT == FMT_FP4 ? *vsrc : *reinterpret_cast<const uint16_t*>(vsrc);
      }
    }
    mx_widen8<T, FMT>(ck, ks, kd);
    mx_widen8<T, FMT>(cv, vs, vd);
  }
}

int mx_check(const char* what, int64_t B, int64_t Hkv, int64_t n_tok, int64_t head_dim, int dtype, int format,
             int64_t max_pages, int64_t n_phys_pages) {
  FSI_CHECK_ARG(format == FSI_KV_MXFP8 || format == FSI_KV_MXFP4, FSI_ERR_INVALID_ARG, "%s: format %d", what, format);
  FSI_CHECK_ARG(dtype == FSI_DTYPE_F32 || dtype == FSI_DTYPE_BF16, FSI_ERR_DTYPE, "%s: dtype %d", what, dtype);
  FSI_CHECK_ARG(fsi_kv_mx_block_bytes(head_dim, format) > 0, FSI_ERR_SHAPE, "%s: head_dim %lld not 64, 96, 128 or 256",
                what, (long long)head_dim);
  FSI_CHECK_ARG(B >= 0 && Hkv > 0 && n_tok >= 0 && max_pages > 0 && n_phys_pages > 0, FSI_ERR_SHAPE, "%s: bad sizes",
                what);
  FSI_CHECK_ARG(max_pages <= 0x7fffffff / MX_PAGE && B <= 0x7fffffff && Hkv <= 0x7fffffff && n_tok <= 0x7fffff00,
                FSI_ERR_SHAPE, "%s: sizes beyond int32", what);
  return FSI_OK;
}

// f(type tag, format tag, head size tag) for the call's type, format and head size.
template <typename F>
void mx_dispatch(int dtype, int format, int64_t hd, F&& f) {
  auto by_hd = [&](auto t, auto fm) {
    switch (hd) {
      case 64: f(t, fm, std::integral_constant<int, 64>{}); break;
      case 96: f(t, fm, std::integral_constant<int, 96>{}); break;
      case 128: f(t, fm, std::integral_constant<int, 128>{}); break;
      default: f(t, fm, std::integral_constant<int, 256>{});
    }
  };
  auto by_format = [&](auto t) {
    if (format == FSI_KV_MXFP4) by_hd(t, std::integral_constant<int, FMT_FP4>{});
    else by_hd(t, std::integral_constant<int, FMT_FP8>{});
  };
  if (dtype == FSI_DTYPE_F32) by_format(float{});
  else by_format(bf16_t{});
}

}  // namespace

extern "C" {

FSI_API int64_t fsi_kv_mx_block_bytes(int64_t head_dim, int format) {
  const bool hd_ok = head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256;
  if (!hd_ok || (format != FSI_KV_MXFP8 && format != FSI_KV_MXFP4)) return 0;
  return mx_block_bytes(format, head_dim);
}

FSI_API int fsi_kv_mx_write(const void* k, const void* v, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t,
                            int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_t, int64_t B, int64_t Hkv,
                            int64_t n_tok, int64_t head_dim, int dtype, int format, const int32_t* start_rows,
                            int64_t start, const int32_t* page_table, int64_t max_pages, int64_t n_phys_pages,
                            void* k_pool, void* v_pool, int* err, void* stream) {
  const int c = mx_check("kv_mx_write", B, Hkv, n_tok, head_dim, dtype, format, max_pages, n_phys_pages);
  if (c != FSI_OK) return c;
  FSI_CHECK_ARG(start >= 0 && start <= 0x7fffffff, FSI_ERR_SHAPE, "kv_mx_write: start %lld", (long long)start);
  if (B == 0 || n_tok == 0) return FSI_OK;
  FSI_CHECK_ARG(k && v && page_table && k_pool && v_pool, FSI_ERR_INVALID_ARG, "kv_mx_write: null pointer");
  FSI_CHECK_ARG((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) % 16 == 0, FSI_ERR_ALIGN,
                "kv_mx_write: pools must be 16-byte aligned");
  MxParams P{};
  P.k = k;
  P.v = v;
  P.ks_b = k_stride_b;
  P.ks_g = k_stride_h;
  P.ks_t = k_stride_t;
  P.vs_b = v_stride_b;
  P.vs_g = v_stride_h;
  P.vs_t = v_stride_t;
  P.B = (int)B;
  P.Hkv = (int)Hkv;
  P.n_tok = (int)n_tok;
  P.hd = (int)head_dim;
  P.start_rows = start_rows;
  P.start = (int)start;
  P.page_table = page_table;
  P.max_pages = (int)max_pages;
  P.n_phys = n_phys_pages;
  P.k_pool = static_cast<uint8_t*>(k_pool);
  P.v_pool = static_cast<uint8_t*>(v_pool);
  P.err = err;
  const int64_t esz = dtype == FSI_DTYPE_F32 ? 4 : 2;
  P.vec = (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 &&
          ((k_stride_b | k_stride_h | k_stride_t | v_stride_b | v_stride_h | v_stride_t) * esz) % 16 == 0;
  // the pages that n_tok tokens touch at most, from any start
  P.pages = static_cast<unsigned>((n_tok + MX_PAGE - 2) / MX_PAGE + 1);
  FSI_CHECK_ARG(B * Hkv <= 0x7fffffff / P.pages, FSI_ERR_SHAPE, "kv_mx_write: B * Hkv * tokens beyond the grid");
  const unsigned grid = static_cast<unsigned>(B * Hkv) * P.pages;
  mx_dispatch(dtype, format, head_dim, [&](auto t, auto f, auto hd) {
    mx_write_kernel<decltype(t), decltype(f)::value, decltype(hd)::value>
        <<<grid, MX_THREADS, 0, reinterpret_cast<hipStream_t>(stream)>>>(P);
  });
  FSI_HIP_LAUNCH_CHECK("kv_mx_write");
  return FSI_OK;
}

FSI_API int fsi_kv_mx_read(const void* k_pool, const void* v_pool, int format, int64_t B, int64_t Hkv, int64_t n_tok,
                           int64_t head_dim, const int32_t* page_table, int64_t max_pages, int64_t n_phys_pages,
                           int dtype, void* k_out, void* v_out, void* stream) {
  const int c = mx_check("kv_mx_read", B, Hkv, n_tok, head_dim, dtype, format, max_pages, n_phys_pages);
  if (c != FSI_OK) return c;
  if (B == 0 || n_tok == 0) return FSI_OK;
  FSI_CHECK_ARG(k_pool && v_pool && page_table && k_out && v_out, FSI_ERR_INVALID_ARG, "kv_mx_read: null pointer");
  FSI_CHECK_ARG((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool) |
                 reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16 == 0,
                FSI_ERR_ALIGN, "kv_mx_read: pools and outputs must be 16-byte aligned");
  MxParams P{};
  P.B = (int)B;
  P.Hkv = (int)Hkv;
  P.n_tok = (int)n_tok;
  P.hd = (int)head_dim;
  P.page_table = page_table;
  P.max_pages = (int)max_pages;
  P.n_phys = n_phys_pages;
  P.k_pool = static_cast<uint8_t*>(const_cast<void*>(k_pool));
  P.v_pool = static_cast<uint8_t*>(const_cast<void*>(v_pool));
  P.k_out = k_out;
  P.v_out = v_out;
  P.pages = static_cast<unsigned>((n_tok + MX_PAGE - 1) / MX_PAGE);
  FSI_CHECK_ARG(B * Hkv <= 0x7fffffff / P.pages, FSI_ERR_SHAPE, "kv_mx_read: B * Hkv * tokens beyond the grid");
  const unsigned grid = static_cast<unsigned>(B * Hkv) * P.pages;
  mx_dispatch(dtype, format, head_dim, [&](auto t, auto f, auto hd) {
    mx_read_kernel<decltype(t), decltype(f)::value, decltype(hd)::value>
        <<<grid, MX_THREADS, 0, reinterpret_cast<hipStream_t>(stream)>>>(P);
  });
  FSI_HIP_LAUNCH_CHECK("kv_mx_read");
  return FSI_OK;
}

}  // extern "C"
