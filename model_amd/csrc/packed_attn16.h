// Tiles of fp16 and bf16 rows in LDS for the attention's products on
// v_mfma_f32_32x32x16_{f16,bf16}.
//
// A stage is [row][HD] as it comes from memory by LDS DMA, 16 bytes a lane.  It is
// read two ways: rows (a lane's 16 bytes are 8 neighbouring elements of its row,
// ds_read_b128) and columns (a lane's 8 elements are one column of 8 rows, two
// ds_read_b64_tr_b16), so no operand is transposed in memory.
//
// A tile of scores leaves its product with 16 rows of the lane's column in the
// registers: of each 32, rows 8 (r / 4) + 4 (lane / 32) + r % 4.  The next product
// contracts over these rows, and the order of a contraction is free: registers 8 c
// to 8 c + 7 are its operand as they are, when the other operand's elements are read
// in the same order: rows 16 c + 4 h + [0, 4) and 16 c + 8 + 4 h + [0, 4).
//
// Banks: DMA writes lane after lane, so places are permuted at the source.  The
// 16-byte piece p of row r lies at p ^ f(r), f a permutation of r's low bits by
// which 8 neighbouring rows' pieces fall on all banks, and so do the 32-byte
// granules of 4 rows that 16 lanes read transposed.
#pragma once

#include "mfma.h"
#include "packed_attn.h"

namespace mpl {

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v lds_short4;

template <class T>
__device__ __forceinline__ f32x16 mma16(short8v a, short8v b, f32x16 c) {
  if constexpr (sizeof(T) == 2 && !__is_same(T, _Float16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// Eight accumulators rounded to T: the operand of a contraction over them.
template <class T>
__device__ __forceinline__ short8v round8(const float* x) {
  typedef T v8 __attribute__((ext_vector_type(8)));
  v8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (T)x[i];
  return __builtin_bit_cast(short8v, y);
}

template <int HD>
struct Stage {
  static constexpr int kRow = 2 * HD, kPieces = HD / 8;       // bytes, 16-byte pieces of a row
  static constexpr int kPer = 1024 / kRow;                    // rows of one load
  static constexpr int kSteps = HD / 16, kTiles = HD / 32;

  __device__ static __forceinline__ int f(int r) {
    return HD >= 64 ? (r & 3) << 1 | (r >> 2 & 1) : (r & 2) | (r >> 2 & 1);
  }

  uint32_t row[4], col[2];
  __device__ __forceinline__ Stage() {
    const int lane = threadIdx.x & 63, h = lane >> 5, r = lane & 31;
#pragma unroll
    for (int c = 0; c < 4; ++c) row[c] = r * kRow + (((2 * c + h) ^ f(r)) & (kPieces - 1)) * 16;
    const int kr = (lane & 15) >> 2, q = lane >> 4 & 1, cr = 4 * h + kr;
#pragma unroll
    for (int d = 0; d < 2; ++d)
      col[d] = cr * kRow + (((4 * d + 2 * q + ((lane & 3) >> 1)) ^ f(cr)) & (kPieces - 1)) * 16 + (lane & 1) * 8;
  }
  // Row 32 b + lane % 32, elements 16 c + 8 (lane / 32) + [0, 8).
  __device__ __forceinline__ short8v rows(const char* lds, int b, int c) const {
    return *(const short8v*)(lds + row[c & 3] + (c >> 2) * 128 + b * 32 * kRow);
  }
  // Column 32 d + lane % 32 of rows 16 c + 4 (lane / 32) + [0, 4) and 8 further.
  __device__ __forceinline__ short8v cols(const char* lds, int c, int d) const {
    const char* at = lds + col[d & 1] + (d >> 1) * 128 + 16 * c * kRow;
    const short4v u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
    const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + 8 * kRow));
    return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // Sends load i of a stage: rows i kPer to (i + 1) kPer - 1 of it; `at(row)` gives a
  // row's address.
  template <class F>
  __device__ static __forceinline__ void load(char* lds, int i, F&& at) {
    const int lane = threadIdx.x & 63, r = i * kPer + lane / kPieces;
    const char* p = at(r) + (((lane % kPieces) ^ f(r)) << 4);
    __builtin_amdgcn_global_load_lds((const void*)p, (lds_void*)(lds + i * 1024), 16, 0, 0);
  }
};

// All of this wave's LDS reads are done: what it read may be written over.
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

}  // namespace mpl
