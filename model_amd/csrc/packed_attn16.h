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
// Banks: DMA writes lane after lane, so places are permuted at the source: the
// 16-byte piece p of row r lies at p ^ f(r).  f spreads the pieces that 16 lanes read
// of 16 neighbouring rows over all 64 banks, and the 64 bytes each that 32 lanes read
// transposed of 4 rows as well.  (With 8 and 16 lanes and half the banks, as 128 bytes
// a cycle would have it, every read took twice its cycles: SQ_LDS_BANK_CONFLICT half of
// SQ_LDS_IDX_ACTIVE, now 0.)
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
    return HD >= 128 ? (r & 3) << 2 | (r >> 2 & 3) : HD == 64 ? (r & 2) << 1 | (r >> 2 & 3) : r >> 2 & 3;
  }

  uint32_t row, col0, col1;
  __device__ __forceinline__ Stage() {
    const int lane = threadIdx.x & 63, h = lane >> 5, r = lane & 31;
    row = r * kRow + ((h ^ f(r)) << 4);
    const int cr = 4 * h + ((lane & 15) >> 2), piece = (lane >> 3 & 2) | (lane >> 1 & 1), e = (lane & 1) * 8;
    col0 = cr * kRow + ((piece ^ f(cr)) << 4) + e;
    col1 = (cr + 8) * kRow + ((piece ^ f(cr + 8)) << 4) + e;
  }
  // Row 32 b + lane % 32, elements 16 c + 8 (lane / 32) + [0, 8).
  __device__ __forceinline__ short8v rows(const char* lds, int b, int c) const {
    return *(const short8v*)(lds + (row ^ (c << 5)) + b * 32 * kRow);
  }
  // Column 32 d + lane % 32 of rows 16 c + 4 (lane / 32) + [0, 4) and 8 further.
  __device__ __forceinline__ short8v cols(const char* lds, int c, int d) const {
    const short4v u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(lds + (col0 ^ (d << 6)) + 16 * c * kRow));
    const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(lds + (col1 ^ (d << 6)) + 16 * c * kRow));
    return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // Sends load n of a stage: its rows n kPer to (n + 1) kPer - 1, of which the lane
  // brings 16 bytes of load_row(n), at `base` (the same for the wave) + `row_at`.
  __device__ static __forceinline__ int load_row(int n) { return n * kPer + (threadIdx.x & 63) / kPieces; }
  //
  // In assembly, because the compiler makes every transposing read wait for all loads
  // under way, those of the next stage among them (it does not know what either
  // touches).  The instruction has no register for a result; whoever reads the stage
  // waits for it with wait_vmcnt_le and a barrier.
  //
  // The compiler does not look for hazards inside the statement either.  An address in
  // scalar registers that a vector instruction wrote (v_readfirstlane, here or wherever
  // the base comes from) may be read by a vector-memory instruction five wait states
  // later at the earliest, so the statement copies it: a scalar read waits for the
  // vector write, and what a scalar instruction wrote may be read at once.  The copy is
  // the wait state, too, that m0 needs.
  __device__ static __forceinline__ void load(char* lds, int n, const char* base, uint32_t row_at) {
    const uint32_t piece = (threadIdx.x & 63) % kPieces ^ f(load_row(n));
    const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void*)(lds + n * 1024));
    const uint64_t from = (uint64_t)base;
    const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(from >> 32)) << 32 |
                        (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)from);
    uint64_t copy;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: declared all the same, so that no value of it is kept across
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
                 : "=&s"(copy)
                 : "s"(to), "v"(row_at + (piece << 4)), "s"(at)
                 : "memory", "m0");
#pragma clang diagnostic pop
  }
  // N loads, every BY-th from n0 on, of rows `pitch` bytes apart from `base` on, the
  // stage's first; rows behind `last` are read as the last.
  template <int N, int BY>
  __device__ static __forceinline__ void load_rows(char* lds, int n0, const char* base, uint32_t pitch, int last) {
    if (last >= N * BY * kPer - 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) load(lds, n0 + i * BY, base + i * BY * kPer * pitch, load_row(n0) * pitch);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) load(lds, n0 + i * BY, base, min(load_row(n0 + i * BY), last) * pitch);
    }
  }
};

// All of this wave's LDS reads are done: what it read may be written over.
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

}  // namespace mpl
