// 64-row bf16 tiles in LDS, shared by the attention backward (attn_bwd.hip) and windowed attention
// with sinks (sink_attn_bf16.hip): direct-to-LDS loads, and the MFMA operands read from them.
// The tiles are row-major; products that contract over a tile's rows read it with
// ds_read_b64_tr_b16, so no transposed copy is written.
//
// 16-byte piece p of row r sits at piece p ^ sab_swz(r): the 8 rows a 128-bit read serves
// at once fall on distinct bank quads, and the 4 rows x 32 bytes that 16 lanes of a
// transposing read cover fill one bank period (head_dim 32: two rows share a period and
// the transposing reads conflict pairwise).
//
// A lane's k slots of a 32-row product: rows 4 kg + e (e < 4) and 16 + 4 kg + e - 4
// (e >= 4), i.e. the rows its two 16 x 16 accumulators of P / dS hold, so those enter the
// MFMA where they are; the transposing reads take the same rows.
#pragma once

#include "fsi_common.h"

namespace {

using namespace fsi;

constexpr int AB_T = 64;  // rows (queries / keys) per tile

typedef __attribute__((address_space(3))) void ab_lds_t;
typedef __attribute__((address_space(1))) void ab_glb_t;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4_t;
typedef __attribute__((address_space(3))) s16x4_t ab_tr_t;

template <int HD>
__device__ __forceinline__ int sab_swz(int row) {
  return HD >= 64 ? ((row & 3) << 1) | ((row >> 2) & 1) : (row >> 1) & 3;
}

template <int HD>
constexpr int sab_tile_bytes() { return AB_T * HD * 2; }

// Rows [r0, r0 + 64) of a (T, HD) bf16 matrix at row stride rs into the LDS tile, by NT
// threads; rows past T re-read row T - 1 (every product that uses them is multiplied by a
// zero P / dS or never stored, so they only need to be finite).  Row strides are below
// 2^24 elements (host-checked): a scalar row base and 32-bit lane offsets.
template <int HD, int NT>
__device__ __forceinline__ void sab_dma(const bf16_t* base, int64_t rs, int r0, int T, char* tile) {
  constexpr int PC = HD / 8, ROWS = NT / PC, N = AB_T / ROWS > 0 ? AB_T / ROWS : 1;
  static_assert(ROWS % 8 == 0, "a thread's rows share their swizzle");
  if (NT > AB_T * PC && threadIdx.x >= AB_T * PC) return;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // offsets are formed here, not kept in registers over the caller's loop
  const int row = tid / PC, lp = (tid % PC) ^ sab_swz<HD>(row);
  const uint32_t rsb = static_cast<uint32_t>(rs) * 2u;
  const char* rb = reinterpret_cast<const char*>(base + static_cast<int64_t>(r0) * rs);
  char* dst = tile + (threadIdx.x & ~63u) * 16;
  if (r0 + AB_T <= T) {
    // scalar bases and one lane offset: nothing else is kept in registers over the loop
    const uint32_t lo = static_cast<uint32_t>(row) * rsb + 16u * static_cast<uint32_t>(lp);
#pragma unroll
    for (int j = 0; j < N; ++j)
      __builtin_amdgcn_global_load_lds((ab_glb_t*)(rb + static_cast<uint64_t>(j * ROWS) * rsb + lo),
                                       (ab_lds_t*)(dst + j * NT * 16), 16, 0, 0);
  } else {
    const int last = T - 1 - r0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint32_t lo = static_cast<uint32_t>(min(j * ROWS + row, last)) * rsb + 16u * static_cast<uint32_t>(lp);
      __builtin_amdgcn_global_load_lds((ab_glb_t*)(rb + lo), (ab_lds_t*)(dst + j * NT * 16), 16, 0, 0);
    }
  }
}

// LDS byte offsets of a lane's reads inside a tile: every fragment's address is one of
// these plus the tile's, xored with its step's piece, plus a constant, so a loop keeps two
// registers of them and not one per fragment.
//   row: row (lane & 15) of the 128-bit operand reads (32-dim step ks in bits 6 and up);
//   tr: row 4 kg + r / 4, 4-dim group r % 4 of the transposing reads (dims 16 dt in bits 5 and up).
template <int HD>
__device__ __forceinline__ uint32_t sab_row_off(int r, int kg) {
  return r * (HD * 2) + 16 * (kg ^ sab_swz<HD>(r));
}
template <int HD>
__device__ __forceinline__ uint32_t sab_tr_off(int r, int kg) {
  const int row = 4 * kg + (r >> 2);
  return row * (HD * 2) + 16 * (((r >> 1) & 1) ^ sab_swz<HD>(row)) + 8 * (r & 1);
}
// The operand at a row offset (16 rows from a multiple of 16, `at` the constant part) for step ks.
__device__ __forceinline__ u32x4_t sab_row(const char* smem, uint32_t off, int ks, int at) {
  typedef __attribute__((address_space(3))) const u32x4_t lds_u32x4_t;
  typedef __attribute__((address_space(3))) const char lds_char_t;
  return *(lds_u32x4_t*)((lds_char_t*)smem + ((off ^ (64u * (ks & 1))) + 128 * (ks >> 1) + at));
}
// Dims 16 dt + (lane & 15) at the lane's k slots of 32 rows.
template <int HD>
__device__ __forceinline__ u32x4_t sab_trow(char* smem, uint32_t off, int dt, int at) {
  typedef __attribute__((address_space(3))) char lds_char_t;
  lds_char_t* p = (lds_char_t*)smem + ((off ^ (32u * (dt & 3))) + 128 * (dt >> 2) + at);
  const u32x2_t x = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ab_tr_t*)p));
  const u32x2_t y = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ab_tr_t*)(p + 16 * HD * 2)));
  return u32x4_t{x[0], x[1], y[0], y[1]};
}

__device__ __forceinline__ uint32_t bf_cvt2(float a, float b) {
  typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2_t;
  const bf16x2_t v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}

}  // namespace
