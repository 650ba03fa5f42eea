// A workgroup's tile of a matrix product over 16-bit operands,
//
//   acc[i][j] = sum_k A[i][k] B[j][k],   a WM TM 32 x WN TN 32 tile,
//
// for the vocabulary's products (cross_entropy.hip): operands come from memory
// by LDS DMA through two LDS stages and feed v_mfma_f32_32x32x16_{f16,bf16}.
//
// An operand lies in memory either way round:
//   rows (ST = 0)   the contraction runs along the rows of the array;
//   columns (ST = 1) the contraction runs down its rows.
// Either way a stage is 128 bytes of contraction for each of the tile's rows
// or columns, brought by 16 bytes a lane.  A stage of rows is [row][128 bytes]
// and a lane reads its 16 bytes of operand with one ds_read_b128; a stage of
// columns is [k][columns] and a lane reads them with two transposing reads
// (ds_read_b64_tr_b16: 16 lanes read a 4 x 16 block and each gets a column of
// it), so no array is ever transposed in memory.
//
// fp32 operands (S = 2) are split: x = hi + lo, both fp16, after a power of
// two that brings the largest of the array to [2^14, 2^15); 11 + 11 bits and
// lo's sign hold x to 2^-23 of it (and to 2^-39 of the array's largest, where
// fp16's own range ends).  A row is then 32 hi, 32 lo, 32 hi, ... and a
// product is hi hi + hi lo + lo hi; lo lo is below 2^-22 of the product.
// Three fp16 products run at 5 times the rate of one fp32 product.
//
// LDS banks: DMA writes lanes one after the other, so the places are permuted
// at the source.  In a stage of rows the 16-byte piece c of row r lies at
// c ^ (r % 8): 8 lanes of a read cover all banks.  In a stage of columns
// 32-byte granule g of contraction row k lies at g ^ 2 (k % 4): the 4 rows
// that 16 lanes read transposed, and their neighbours' next granule, fall on
// different banks.
#pragma once

#include "common.h"
#include "mfma.h"

namespace mpl {

typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v lds_short4;

// One operand array: `pitch` bytes from row to row.  ST = 0: `rows` rows may be
// read (the tile's rows past them are read clamped).  ST = 1: `rows` rows of
// the contraction, and the first `width` bytes of a row.
struct TileOperand {
  const char* base;
  int64_t pitch;
  int64_t rows;
  int64_t width;
};

template <int S_, bool BF_, bool AST_, bool BST_, int WM_, int WN_, int TM_, int TN_>
struct TileMma {
  static constexpr int S = S_, WM = WM_, WN = WN_, TM = TM_, TN = TN_;
  static constexpr bool BF = BF_, AST = AST_, BST = BST_;
  static constexpr int NW = WM * WN, kThreads = NW * 64;
  static constexpr int BM = WM * TM * 32, BN = WN * TN * 32;
  static constexpr int KI = 64 / S;  // contraction of a stage
  static constexpr int kSteps = KI / 16;
  static constexpr int kStageA = BM * 128, kStageB = BN * 128;

  template <int B>
  static constexpr int instrs() { return B * 128 / 1024 / NW; }
  static_assert(BM * 128 % (1024 * NW) == 0 && BN * 128 % (1024 * NW) == 0, "a stage splits evenly over the waves");

  // Sends the loads of stage `it` (from contraction row it * KI) of one operand.
  template <bool ST, int B>
  __device__ static __forceinline__ void issue(const TileOperand& o, int64_t origin, int it, char* lds, int wave,
                                               int lane) {
#pragma unroll
    for (int i = 0; i < instrs<B>(); ++i) {
      const int n = wave * instrs<B>() + i;
      const char* src;
      if constexpr (!ST) {
        const int64_t row = min(origin + n * 8 + (lane >> 3), o.rows - 1);
        src = o.base + row * o.pitch + (int64_t)it * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
      } else {
        constexpr int L = B * 2 * S;  // bytes of a contraction row in the stage
        static_assert(L <= 1024 && L >= 128, "");
        const int at = n * 1024 + lane * 16;
        const int k = at / L;
        const int piece = ((at % L) >> 4) ^ ((4 * (k & 3)) & (L / 16 - 1));
        const int64_t row = min((int64_t)it * KI + k, o.rows - 1);
        const int64_t col = min(origin * (2 * S) + piece * 16, o.width - 16);
        src = o.base + row * o.pitch + col;
      }
      __builtin_amdgcn_global_load_lds((const void*)src, (lds_void*)(lds + n * 1024), 16, 0, 0);
    }
  }

  // The operand of 32 rows or columns `t` (of the tile), plane p, step s.
  template <bool ST, int B>
  __device__ static __forceinline__ short8v frag(const char* lds, int t, int p, int s, int lane) {
    if constexpr (!ST) {
      const int c = (S == 1 ? 2 * s : 4 * p + 2 * s) + (lane >> 5);
      return *(const short8v*)(lds + (t * 32 + (lane & 31)) * 128 + ((c ^ (lane & 7)) << 4));
    } else {
      constexpr int L = B * 2 * S;
      const int kr = (lane & 15) >> 2;
      const int g = (S == 1 ? 2 * t : 4 * t + 2 * p) + ((lane >> 4) & 1);
      const int k = 16 * s + 8 * (lane >> 5) + kr;
      const char* at = lds + k * L + ((g ^ ((2 * kr) & (L / 32 - 1))) << 5) + ((lane & 3) << 3);
      const short4v u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
      const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + 4 * L));
      return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }

  __device__ static __forceinline__ f32x16 mma(short8v a, short8v b, f32x16 c) {
    if constexpr (BF)
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c,
                                                     0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0,
                                                    0, 0);
  }

  __device__ static __forceinline__ void compute(const char* la, const char* lb, int wm, int wn, int lane,
                                                 f32x16 (&acc)[TM][TN]) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      short8v a[S][TM], b[S][TN];
#pragma unroll
      for (int p = 0; p < S; ++p) {
#pragma unroll
        for (int j = 0; j < TN; ++j) b[p][j] = frag<BST, BN>(lb, wn * TN + j, p, s, lane);
#pragma unroll
        for (int i = 0; i < TM; ++i) a[p][i] = frag<AST, BM>(la, wm * TM + i, p, s, lane);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mma(a[0][i], b[0][j], acc[i][j]);
      if constexpr (S == 2) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mma(a[0][i], b[1][j], acc[i][j]);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mma(a[1][i], b[0][j], acc[i][j]);
      }
    }
  }

  // The tile whose first row of A is m0 and of B n0, over the stages [it0, it1).
  // Between the barrier of a stage and the next one's, its operands are read
  // and the next stage's loads fly; a wave passes a barrier only with its loads
  // landed and its reads done.
  __device__ static __forceinline__ void run(const TileOperand& A, const TileOperand& B, int64_t m0, int64_t n0, int it0,
                                             int it1, char* a0, char* b0, char* a1, char* b1, f32x16 (&acc)[TM][TN]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};
    if (it0 >= it1) return;
    auto sync = [&]() __attribute__((always_inline)) {
      wait_vmcnt_le<0>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    issue<AST, BM>(A, m0, it0, a0, wave, lane);
    issue<BST, BN>(B, n0, it0, b0, wave, lane);
    for (int it = it0; it < it1; it += 2) {
      sync();
      if (it + 1 < it1) {
        issue<AST, BM>(A, m0, it + 1, a1, wave, lane);
        issue<BST, BN>(B, n0, it + 1, b1, wave, lane);
      }
      compute(a0, b0, wm, wn, lane, acc);
      if (it + 1 >= it1) break;
      sync();
      if (it + 2 < it1) {
        issue<AST, BM>(A, m0, it + 2, a0, wave, lane);
        issue<BST, BN>(B, n0, it + 2, b0, wave, lane);
      }
      compute(a1, b1, wm, wn, lane, acc);
    }
  }
};

// Workgroups go to the 8 XCDs in turn: each XCD gets a run of neighbouring
// tiles, walked `group` row tiles deep, so that what its workgroups read
// together stays in its L2.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t total, uint32_t tm, uint32_t tn, uint32_t group,
                                        uint32_t& m, uint32_t& n) {
  const uint32_t full = total / 8 * 8;
  const uint32_t at = id < full ? (id & 7) * (full / 8) + (id >> 3) : id;
  const uint32_t band = at / (group * tn), first = band * group;
  const uint32_t deep = min(group, tm - first), in = at - band * group * tn;
  m = first + in % deep;
  n = in / deep;
}

}  // namespace mpl
