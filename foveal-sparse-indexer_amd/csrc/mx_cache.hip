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
};

template <typename T>
__device__ __forceinline__ float mx_ld(const T* p);
template <>
__device__ __forceinline__ float mx_ld<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float mx_ld<bf16_t>(const bf16_t* p) { return bf16_to_f32(*p); }
template <typename T>
__device__ __forceinline__ void mx_st(T* p, float x);
template <>
__device__ __forceinline__ void mx_st<float>(float* p, float x) { *p = x; }
template <>
__device__ __forceinline__ void mx_st<bf16_t>(bf16_t* p, float x) { *p = f32_to_bf16(x); }

// Physical page of sequence b's token p, or -1 outside the table or the pool.
__device__ __forceinline__ int64_t mx_phys(const MxParams& P, int b, int p) {
  if (p < 0 || p / MX_PAGE >= P.max_pages) return -1;
  const int64_t phys = P.page_table[static_cast<int64_t>(b) * P.max_pages + p / MX_PAGE];
  return phys >= 0 && phys < P.n_phys ? phys : -1;
}

// One thread per (sequence, head, token, group).
template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_write_kernel(MxParams P) {
  constexpr int W2 = 2 * MxFmt<FMT>::BITS / 8;
  const int ng = P.hd / MX_GROUP;
  const int64_t total = static_cast<int64_t>(P.B) * P.Hkv * P.n_tok * ng;
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < total;
       id += static_cast<int64_t>(gridDim.x) * 256) {
    const int i = static_cast<int>(id % ng);
    int64_t rest = id / ng;
    const int t = static_cast<int>(rest % P.n_tok);
    rest /= P.n_tok;
    const int g = static_cast<int>(rest % P.Hkv), b = static_cast<int>(rest / P.Hkv);
    const int64_t p = static_cast<int64_t>(P.start_rows ? P.start_rows[b] : P.start) + t;
    const int64_t phys = p > 0x7fffffff ? -1 : mx_phys(P, b, static_cast<int>(p));
    if (phys < 0) {
      set_error(P.err, FSI_ERR_INDEX_RANGE);
      continue;
    }
    const int off = static_cast<int>(p) % MX_PAGE;
    const int64_t base = (phys * P.Hkv + g) * mx_block_bytes(FMT, P.hd);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const T* src = (kv ? static_cast<const T*>(P.v) + b * P.vs_b + g * P.vs_g + t * P.vs_t
                         : static_cast<const T*>(P.k) + b * P.ks_b + g * P.ks_g + t * P.ks_t) + MX_GROUP * i;
      float x[MX_GROUP];
      uint32_t amax = 0;
#pragma unroll
      for (int d = 0; d < MX_GROUP; ++d) {
        x[d] = mx_ld(src + d);
        const uint32_t a = __float_as_uint(x[d]) & 0x7fffffffu;
        amax = a > amax ? a : amax;
      }
      const int byte = mx_scale_byte<FMT>(amax);
      const float inv = byte == SCALE_NAN ? 0.f : mx_inv_scale(byte);
      uint8_t* blk = (kv ? P.v_pool : P.k_pool) + base;
      uint8_t* scales = blk + mx_codes_bytes(FMT, P.hd);
      scales[kv ? v_scale_off(ng, i, off) : k_scale_off(i, off)] = static_cast<uint8_t>(byte);
#pragma unroll
      for (int r = 0; r < MX_GROUP / 2; ++r) {
        const uint32_t c0 = byte == SCALE_NAN ? 0u : mx_code<FMT>(x[2 * r] * inv);
        const uint32_t c1 = byte == SCALE_NAN ? 0u : mx_code<FMT>(x[2 * r + 1] * inv);
        uint8_t* dst = blk + (kv ? v_pair_off<W2>(i, r, off) : (off * P.hd + MX_GROUP * i + 2 * r) * W2 / 2);
        if (FMT == FMT_FP4) *dst = static_cast<uint8_t>(c0 | (c1 << 4));
        else *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(c0 | (c1 << 8));
      }
    }
  }
}

// One thread per (sequence, head, token, group): tokens [0, n_tok) of every sequence; 0 where the
// page is not there.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_read_kernel(MxParams P) {
  constexpr int W2 = 2 * MxFmt<FMT>::BITS / 8;
  const int ng = P.hd / MX_GROUP;
  const int64_t total = static_cast<int64_t>(P.B) * P.Hkv * P.n_tok * ng;
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < total;
       id += static_cast<int64_t>(gridDim.x) * 256) {
    const int i = static_cast<int>(id % ng);
    int64_t rest = id / ng;
    const int t = static_cast<int>(rest % P.n_tok);
    rest /= P.n_tok;
    const int g = static_cast<int>(rest % P.Hkv), b = static_cast<int>(rest / P.Hkv);
    const int64_t phys = mx_phys(P, b, t);
    const int off = t % MX_PAGE;
    const int64_t base = (phys * P.Hkv + g) * mx_block_bytes(FMT, P.hd);
    const int64_t at = (id / ng) * P.hd + MX_GROUP * i;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      T* dst = static_cast<T*>(kv ? P.v_out : P.k_out) + at;
      if (phys < 0) {
#pragma unroll
        for (int d = 0; d < MX_GROUP; ++d) mx_st(dst + d, 0.f);
        continue;
      }
      const uint8_t* blk = (kv ? P.v_pool : P.k_pool) + base;
      const int byte = blk[mx_codes_bytes(FMT, P.hd) + (kv ? v_scale_off(ng, i, off) : k_scale_off(i, off))];
      const float s = byte == SCALE_NAN ? __uint_as_float(0x7fc00000u) : mx_scale(byte);
#pragma unroll
      for (int r = 0; r < MX_GROUP / 2; ++r) {
        const uint8_t* src = blk + (kv ? v_pair_off<W2>(i, r, off) : (off * P.hd + MX_GROUP * i + 2 * r) * W2 / 2);
        const uint32_t c = FMT == FMT_FP4 ? *src : *reinterpret_cast<const uint16_t*>(src);
        const uint32_t c0 = FMT == FMT_FP4 ? c & 15u : c & 255u, c1 = FMT == FMT_FP4 ? c >> 4 : c >> 8;
        mx_st(dst + 2 * r, mx_value<FMT>(c0) * s);
        mx_st(dst + 2 * r + 1, mx_value<FMT>(c1) * s);
      }
    }
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
  FSI_CHECK_ARG(max_pages <= 0x7fffffff / MX_PAGE && B <= 0x7fffffff && Hkv <= 0x7fffffff && n_tok <= 0x7fffffff,
                FSI_ERR_SHAPE, "%s: sizes beyond int32", what);
  return FSI_OK;
}

// f(type tag, format tag) for the call's type and format.
template <typename F>
void mx_dispatch(int dtype, int format, F&& f) {
  if (dtype == FSI_DTYPE_F32) {
    if (format == FSI_KV_MXFP4) f(float{}, std::integral_constant<int, FMT_FP4>{});
    else f(float{}, std::integral_constant<int, FMT_FP8>{});
  } else {
    if (format == FSI_KV_MXFP4) f(bf16_t{}, std::integral_constant<int, FMT_FP4>{});
    else f(bf16_t{}, std::integral_constant<int, FMT_FP8>{});
  }
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
  const int64_t total = B * Hkv * n_tok * (head_dim / MX_GROUP);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((total + 255) / 256, 1 << 20));
  mx_dispatch(dtype, format, [&](auto t, auto f) {
    mx_write_kernel<decltype(t), decltype(f)::value><<<grid, 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(P);
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
  const int64_t total = B * Hkv * n_tok * (head_dim / MX_GROUP);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((total + 255) / 256, 1 << 20));
  mx_dispatch(dtype, format, [&](auto t, auto f) {
    mx_read_kernel<decltype(t), decltype(f)::value><<<grid, 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(P);
  });
  FSI_HIP_LAUNCH_CHECK("kv_mx_read");
  return FSI_OK;
}

}  // extern "C"
