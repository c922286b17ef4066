// Building blocks of the matrix-core kernels over sequences (tsg_attn.hip, tsg_xent.hip): element types, operand
// fragments of v_mfma_f32_32x32x16 (bf16 / f16) and v_mfma_f32_16x16x4 (f32), tiles in LDS, direct loads into LDS.
//
// A product covers W x W results: W = 32 for the 16-bit types, 16 for f32 (where an operand takes twice the registers).
// Lane l has column l % W of it and is part h = l / W of 64 / W; the accumulator's register i is row (i & 3) + 8 (i >> 2) + 4 h.
// A tile in LDS is [rows][CH] chunks of 16 bytes (8 elements of 16 bits or 4 of 32).  Chunk c of row r lies at
// position c ^ swz(r) of its row, which spreads both kinds of read over the banks:
//   row fragment  lane l takes chunk (64 / W) s + h of row l % W: the k index of the product runs along the row
//   col fragment  lane l takes column l % W of eight (f32: one) rows: the k index runs down the rows
// A sum does not care how its k index is numbered as long as both operands agree, so an accumulator is
// fed back as the B operand of the next product without moving data between lanes: the col fragment of the A operand
// is read from exactly the rows that the lane's accumulator registers stand for.
#pragma once
#include "tsg_common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

typedef _Float16 tsg_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 tsg_b8 __attribute__((ext_vector_type(8)));
typedef short tsg_s4 __attribute__((ext_vector_type(4)));
typedef unsigned tsg_u4 __attribute__((ext_vector_type(4)));
typedef float tsg_f4 __attribute__((ext_vector_type(4)));

struct TsgF32 { typedef float type; };
struct TsgBf16 { typedef __bf16 type; };
struct TsgF16 { typedef _Float16 type; };

template <typename D> struct TsgElem {  // bf16 / f16
  typedef typename D::type T;
  typedef tsg_f32x16 Acc;
  static constexpr int BYTES = 2, EPC = 8, W = 32, REGS = 16;  // bytes, elements per chunk, width of a product, accumulator registers
};
template <> struct TsgElem<TsgF32> {
  typedef float T;
  typedef tsg_f4 Acc;
  static constexpr int BYTES = 4, EPC = 4, W = 16, REGS = 4;
};

template <typename T> __device__ __forceinline__ float tsg_to_f32(T v) { return (float)v; }

// two f32 -> two 16-bit values in one register, rounded to nearest even (v_cvt_pk_bf16_f32 / two v_cvt_f16_f32)
template <typename D> __device__ __forceinline__ unsigned tsg_pack2(float a, float b) {
  typedef typename D::type T;
  typedef T T2 __attribute__((ext_vector_type(2)));
  T2 v;
  v.x = (T)a;
  v.y = (T)b;
  return __builtin_bit_cast(unsigned, v);
}

// acc += A . B for one row-fragment pair: k = 16 (16-bit types), or four products of k = 4 (f32)
template <typename D> __device__ __forceinline__ void tsg_mma(tsg_u4 a, tsg_u4 b, typename TsgElem<D>::Acc& acc);
template <> __device__ __forceinline__ void tsg_mma<TsgBf16>(tsg_u4 a, tsg_u4 b, tsg_f32x16& acc) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(tsg_b8, a), __builtin_bit_cast(tsg_b8, b), acc, 0, 0, 0);
}
template <> __device__ __forceinline__ void tsg_mma<TsgF16>(tsg_u4 a, tsg_u4 b, tsg_f32x16& acc) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(tsg_h8, a), __builtin_bit_cast(tsg_h8, b), acc, 0, 0, 0);
}
template <> __device__ __forceinline__ void tsg_mma<TsgF32>(tsg_u4 a, tsg_u4 b, tsg_f4& acc) {
  const tsg_f4 x = __builtin_bit_cast(tsg_f4, a), y = __builtin_bit_cast(tsg_f4, b);
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
}

// swz(r) for rows of CH chunks (see the top): a bijection of 16 neighbouring rows (CH < 16: eight pairs of them) onto the bank
// groups.  The transposing loads of the 16-bit types take four neighbouring rows at once, the f32 ones rows four apart:
// those get the positions that lie furthest from each other.
template <int CH, bool F32 = false> __device__ __forceinline__ int tsg_swz(int r) {
  if (F32) return r & 15;
  if (CH >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

typedef __attribute__((address_space(3))) char tsg_lds_char;
__device__ __forceinline__ unsigned tsg_lds_addr(const void* p) { return (unsigned)(uintptr_t)(tsg_lds_char*)p; }

template <int CH, bool F32 = false> __device__ __forceinline__ tsg_u4 tsg_row_frag(const char* tile, int row, int chunk) {
  return *reinterpret_cast<const tsg_u4*>(tile + ((size_t)row * CH + (chunk ^ tsg_swz<CH, F32>(row))) * 16);
}

// acc[m][n] += sum over the 32 rows row0.. of tile: tile[row][col0 + m] * p(row, n), p in accumulator layout
template <typename D, int CH>
__device__ __forceinline__ void tsg_mma_cols(const char* tile, int row0, int col0, const tsg_u4 (&p)[2], tsg_f32x16& acc, int lane) {
  const int h = lane >> 5, i = lane & 15, part = (lane >> 4) & 1;
  const int col = col0 + 16 * part + 4 * (i & 3);  // ds_read_b64_tr_b16: 16 lanes hand in 4 rows x 16 columns
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    tsg_s4 v[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int row = row0 + 16 * t + 8 * g + 4 * h + (i >> 2);
      const char* at = tile + ((size_t)row * CH + ((col >> 3) ^ tsg_swz<CH>(row))) * 16 + (col & 7) * 2;
      v[g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tsg_s4*)at);
    }
    typedef short s8 __attribute__((ext_vector_type(8)));
    const s8 a = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    tsg_mma<D>(__builtin_bit_cast(tsg_u4, a), p[t], acc);
  }
}
template <int CH>
__device__ __forceinline__ void tsg_mma_cols_f32(const char* tile, int row0, int col0, const tsg_f4& p, tsg_f4& acc, int lane) {
  const int col = col0 + (lane & 15);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 4 * (lane >> 4) + i;
    const float a = *reinterpret_cast<const float*>(tile + ((size_t)row * CH + ((col >> 2) ^ tsg_swz<CH, true>(row))) * 16 + (col & 3) * 4);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a, p[i], acc, 0, 0, 0);
  }
}
// the accumulator as the B operand: rounded to the operand type (nearest even)
template <typename D> struct TsgAccB {
  tsg_u4 v[2];
  __device__ __forceinline__ void set(const tsg_f32x16& p) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int w = 0; w < 4; ++w) v[t][w] = tsg_pack2<D>(p[8 * t + 2 * w], p[8 * t + 2 * w + 1]);
  }
  template <int CH>
  __device__ __forceinline__ void mma(const char* tile, int row0, int col0, tsg_f32x16& acc, int lane) const {
    tsg_mma_cols<D, CH>(tile, row0, col0, v, acc, lane);
  }
};
template <> struct TsgAccB<TsgF32> {
  tsg_f4 v;
  __device__ __forceinline__ void set(const tsg_f4& p) { v = p; }
  template <int CH>
  __device__ __forceinline__ void mma(const char* tile, int row0, int col0, tsg_f4& acc, int lane) const {
    tsg_mma_cols_f32<CH>(tile, row0, col0, v, acc, lane);
  }
};

// 16 bytes per lane straight into LDS at lds + 16 * lane (lds wave-uniform).  The compiler does not see these loads:
// tsg_dma_wait() before the barrier that hands the tile over.
static __device__ const tsg_u4 tsg_zero_chunk = {0u, 0u, 0u, 0u};  // what chunks outside an operand are read from
__device__ __forceinline__ void tsg_dma16(const void* g, unsigned lds) {
  unsigned keep;  // m0 holds the LDS base of such a load; what the compiler has in it is put back
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(g)
               : "memory");
}
__device__ __forceinline__ void tsg_dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Tile [ROWS][CH] of a row-major operand: row r of the tile is src + r * stride bytes for r < r1 and zeros from there on,
// chunks from `chunks` on are zeros.  All WAVES waves take part.
// MASKED: row r is zeros also where bit r of `used` is clear.
template <int ROWS, int CH, int WAVES, bool MASKED = false, bool F32 = false>
__device__ __forceinline__ void tsg_load_tile(char* tile, const char* src, long stride, int r1, int chunks, int wave, int lane,
                                              unsigned long long used = 0) {
  constexpr int N = ROWS * CH / 64;  // instructions of 64 chunks
  static_assert(ROWS * CH % 64 == 0, "whole wave loads");
#pragma unroll
  for (int n = 0; n < (N + WAVES - 1) / WAVES; ++n) {
    const int ins = n * WAVES + wave;
    if (N % WAVES == 0 || ins < N) {
      const int at = ins * 64 + lane, r = at / CH, c = (at % CH) ^ tsg_swz<CH, F32>(r);
      const char* g = src + (long)r * stride + c * 16;
      if (r >= r1 || c >= chunks || (MASKED && !(used >> r & 1))) g = reinterpret_cast<const char*>(&tsg_zero_chunk);
      tsg_dma16(g, tsg_lds_addr(tile) + ins * 1024);
    }
  }
}
