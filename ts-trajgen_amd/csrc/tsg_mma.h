// Building blocks of the matrix-core kernels over sequences (tsg_attn.hip, tsg_xent.hip): element types, operand
// fragments of v_mfma_f32_32x32x16 (bf16 / f16) and v_mfma_f32_16x16x4 (f32), tiles in LDS, direct loads into LDS.
//
// A product covers W x W results: W = 32 for the 16-bit types, 16 for f32 (where an operand takes twice the registers).
// Lane l has column l % W of it and is part h = l / W of 64 / W; the accumulator's register i is row (i & 3) + 8 (i >> 2) + 4 h.
//   row fragment  lane l takes chunk (64 / W) s + h (16 bytes) of row l % W: the k index of the product runs along the row
//   col fragment  lane l takes column l % W of eight (f32: one) rows: the k index runs down the rows
// A tile of 16-bit elements in LDS is [rows][CH] chunks of 16 bytes; chunk c of row r lies at position c ^ swz(r) of its row,
// which spreads both kinds of read over the banks (the col fragment is a transposing load, ds_read_b64_tr_b16).
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
// groups, with four neighbouring rows, which the transposing loads take at once, as far apart as can be.
template <int CH> __device__ __forceinline__ int tsg_swz(int r) {
  if (CH >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

typedef __attribute__((address_space(3))) char tsg_lds_char;
__device__ __forceinline__ unsigned tsg_lds_addr(const void* p) { return (unsigned)(uintptr_t)(tsg_lds_char*)p; }

// Where a lane's fragments lie, as LDS byte addresses.  A row takes CH * 16 bytes, a power of two, and tiles start at
// multiples of that, so the swizzle is an exclusive-or on the address: a fragment's address is the lane's own start, `^` a
// constant of the k step or column block, plus an offset the load instruction carries.  tsg_opaque() inside a loop keeps the
// compiler from holding every such address in a register of its own (which costs more than the one operation).
__device__ __forceinline__ unsigned tsg_opaque(unsigned v) {
  asm volatile("" : "+v"(v));
  return v;
}
template <typename D, int CH> struct TsgLane {
  static constexpr int W = TsgElem<D>::W, PARTS = 64 / W, ROW = CH * 16;
  // first row fragment of row l % W of the tile
  static __device__ __forceinline__ unsigned row(int lane) {
    const int r = lane % W, h = lane / W;
    return r * ROW + ((h ^ tsg_swz<CH>(r)) << 4);
  }
  // first column fragment of the W rows from the tile's start, numbered as an accumulator's registers number them
  static __device__ __forceinline__ unsigned col(int lane) {
    const int i = lane & 15, r = 4 * (lane >> 5) + (i >> 2);  // ds_read_b64_tr_b16: 16 lanes hand in 4 rows x 16 columns
    return r * ROW + (((2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ tsg_swz<CH>(r)) << 4) + 8 * (i & 1);
  }
  // the same with k = 8 (l / 32) + 0..7: the order that a row fragment has
  static __device__ __forceinline__ unsigned col_in_order(int lane) {
    const int i = lane & 15, r = 8 * (lane >> 5) + (i >> 2);
    return r * ROW + (((2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ tsg_swz<CH>(r)) << 4) + 8 * (i & 1);
  }
};
typedef __attribute__((address_space(3))) const tsg_u4 tsg_lds_u4;
typedef __attribute__((address_space(3))) tsg_s4 tsg_lds_s4;
// row fragment of k step s; offset: of the tile and the row block
template <typename D> __device__ __forceinline__ tsg_u4 tsg_row_frag(unsigned row, int s, int offset) {
  return *reinterpret_cast<tsg_lds_u4*>((uintptr_t)((row ^ (s * (64 / TsgElem<D>::W) * 16)) + offset));
}
__device__ __forceinline__ tsg_u4 tsg_join4(tsg_s4 x, tsg_s4 y) {
  typedef short s8 __attribute__((ext_vector_type(8)));
  const s8 a = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(tsg_u4, a);
}
// 16 rows x 32 columns from row fragment order (TsgLane::col_in_order); block: 32-column block
template <int CH> __device__ __forceinline__ tsg_u4 tsg_col_frag(unsigned col, int block, int offset) {
  const unsigned at = col ^ (block * 64);
  const tsg_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<tsg_lds_s4*>((uintptr_t)(at + offset)));
  const tsg_s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<tsg_lds_s4*>((uintptr_t)((at ^ 16) + offset + 4 * CH * 16)));
  return tsg_join4(x, y);
}

// acc[m][n] += sum over W rows of a tile: tile[row][W block + m] * p(row, n), p in accumulator layout, rounded to the
// operand type (nearest even)
template <typename D> struct TsgAccB {
  tsg_u4 v[2];
  __device__ __forceinline__ void set(const tsg_f32x16& p) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int w = 0; w < 4; ++w) v[t][w] = tsg_pack2<D>(p[8 * t + 2 * w], p[8 * t + 2 * w + 1]);
  }
  // what set() rounded off p
  __device__ __forceinline__ void set_rest(tsg_f32x16 p) {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] -= (float)(typename D::type)p[i];
    set(p);
  }
  template <int CH> __device__ __forceinline__ void mma(unsigned col, int block, int offset, tsg_f32x16& acc) const {
    const unsigned at = col ^ (block * 64);
#pragma unroll
    for (int t = 0; t < 2; ++t) tsg_mma<D>(frag<CH>(at, offset, t), v[t], acc);
  }
  template <int CH> static __device__ __forceinline__ tsg_u4 frag(unsigned at, int offset, int t) {
    const tsg_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<tsg_lds_s4*>((uintptr_t)(at + offset + 16 * t * CH * 16)));
    const tsg_s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<tsg_lds_s4*>((uintptr_t)((at ^ 32) + offset + (16 * t + 8) * CH * 16)));
    return tsg_join4(x, y);
  }
};
// ---- tiles from memory straight into LDS (buffer_load_dwordx4 ... lds: lane l's 16 bytes go to m0 + 16 l).
// The compiler does not see these loads: tsg_dma_wait() before the barrier that hands the tile over, and no load of its
// own left in flight across a tile loop (tsg_settle), or its waits would drain these too.
// A buffer descriptor bounds the operand: what lies behind its last valid byte is written to LDS as zeros.
__device__ __forceinline__ void tsg_dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
template <int N> __device__ __forceinline__ void tsg_settle(tsg_u4 (&f)[N]) {
#pragma unroll
  for (int s = 0; s < N; ++s) asm volatile("" : "+v"(f[s]));
}

__device__ __forceinline__ tsg_u4 tsg_descriptor(const char* base, unsigned bytes) {
  const unsigned long long p = reinterpret_cast<unsigned long long>(base);
  tsg_u4 d;
  d[0] = __builtin_amdgcn_readfirstlane((unsigned)p);
  d[1] = __builtin_amdgcn_readfirstlane((unsigned)(p >> 32)) & 0xffffu;
  d[2] = __builtin_amdgcn_readfirstlane(bytes);
  d[3] = 0x00020000u;  // raw buffer, no stride
  return d;
}
// m0 holds the LDS address of such a load; what the compiler has in it is put back
__device__ __forceinline__ void tsg_dma(tsg_u4 d, unsigned off, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "s"(lds), "v"(off), "s"(d)
               : "memory");
}
template <int STEP> __device__ __forceinline__ void tsg_dma2(tsg_u4 d, unsigned o0, unsigned o1, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds\n\ts_add_u32 m0, m0, %5\n\ts_nop 0\n\t"
               "buffer_load_dwordx4 %3, %4, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "s"(lds), "v"(o0), "v"(o1), "s"(d), "n"(STEP)
               : "memory", "scc");
}
template <int STEP> __device__ __forceinline__ void tsg_dma4(tsg_u4 d, unsigned o0, unsigned o1, unsigned o2, unsigned o3, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %6, 0 offen lds\n\ts_add_u32 m0, m0, %7\n\ts_nop 0\n\t"
               "buffer_load_dwordx4 %3, %6, 0 offen lds\n\ts_add_u32 m0, m0, %7\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %6, 0 offen lds\n\t"
               "s_add_u32 m0, m0, %7\n\ts_nop 0\n\tbuffer_load_dwordx4 %5, %6, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "s"(lds), "v"(o0), "v"(o1), "v"(o2), "v"(o3), "s"(d), "n"(STEP)
               : "memory", "scc");
}

// The loads of a [ROWS][CH] tile by WAVES waves: a lane's byte offsets within the operand's rows, kept over the tile loop.
// ROWS * stride must stay below 2^31 bytes.
template <int ROWS, int CH, int WAVES> struct TsgLoader {
  static constexpr int N = ROWS * CH / 64 / WAVES, DOWN = 64 * WAVES / CH;  // loads per wave; rows from one to the next
  static constexpr bool EVEN = DOWN % 16 == 0;  // the swizzle repeats: one offset serves all
  static_assert(N >= 1 && ROWS * CH % (64 * WAVES) == 0, "whole wave loads");
  unsigned off[EVEN ? 1 : N], stride, lds;
  int row;  // of the first load
  __device__ __forceinline__ void init(long row_bytes, int chunks, unsigned tile, int wave, int lane) {
    stride = __builtin_amdgcn_readfirstlane((unsigned)row_bytes);
    lds = __builtin_amdgcn_readfirstlane(tile + wave * 1024);
    row = (wave * 64 + lane) / CH;
#pragma unroll
    for (int n = 0; n < (EVEN ? 1 : N); ++n) {
      const int r = row + n * DOWN, c = ((wave * 64 + lane) % CH) ^ tsg_swz<CH>(r);
      off[n] = c < chunks ? r * stride + c * 16 : 0x80000000u;  // behind every bound
    }
  }
  __device__ __forceinline__ unsigned at(int n) const { return EVEN ? off[0] + n * DOWN * stride : off[EVEN ? 0 : n]; }
  __device__ __forceinline__ unsigned at(int n, unsigned long long used) const { return used >> (row + n * DOWN) & 1 ? at(n) : 0x80000000u; }
  // rows [0, left) of the operand at base exist, `width` bytes each; shift: of the LDS address, for the buffer
  __device__ __forceinline__ tsg_u4 bound(const char* base, long left, int width) const {
    const int rows = left < ROWS ? (int)left : ROWS;
    return tsg_descriptor(base, rows > 0 ? (rows - 1) * stride + width : 0u);
  }
  __device__ __forceinline__ void load(const char* base, long left, int width, int shift) const {
    const tsg_u4 d = bound(base, left, width);
    issue(d, shift, [&](int n) { return at(n); });
  }
  __device__ __forceinline__ void load(const char* base, long left, int width, int shift, unsigned long long used) const {
    const tsg_u4 d = bound(base, left, width);
    issue(d, shift, [&](int n) { return at(n, used); });
  }
  template <typename F> __device__ __forceinline__ void issue(tsg_u4 d, int shift, F off_of) const {
    const unsigned to = __builtin_amdgcn_readfirstlane(lds + shift);
    if constexpr (N == 1) tsg_dma(d, off_of(0), to);
    else if constexpr (N == 2) tsg_dma2<WAVES * 1024>(d, off_of(0), off_of(1), to);
    else {
      static_assert(N % 4 == 0, "");
#pragma unroll
      for (int n = 0; n < N; n += 4) tsg_dma4<WAVES * 1024>(d, off_of(n), off_of(n + 1), off_of(n + 2), off_of(n + 3), to + n * WAVES * 1024);
    }
  }
};

// Order of the instructions of a block: `first` LDS reads, then one matrix product for every `per` more, so that a product never
// waits for the read just before it.
template <int READS, int PRODUCTS, int FIRST, int PER> __device__ __forceinline__ void tsg_interleave() {
  __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
#pragma unroll
  for (int n = 0; n < PRODUCTS; ++n) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (FIRST + n * PER < READS) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
  }
}
