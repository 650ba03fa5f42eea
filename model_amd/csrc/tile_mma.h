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

  // Sends the loads of stage `it` (from contraction row it * KI) of one operand:
  // a scalar address of the stage and 32-bit places of the lanes in it.
  template <bool ST, int B>
  __device__ static __forceinline__ void issue(const TileOperand& o, int64_t origin, int it, char* lds, int wave,
                                               int lane) {
    const char* base;
    int last;
    // a tile or a stage that lies behind the array reads its last row
    if constexpr (!ST) {
      const int64_t first = min(origin, o.rows - 1);
      base = o.base + first * o.pitch + (int64_t)it * 128;
      last = (int)min(o.rows - 1 - first, (int64_t)(B - 1));
    } else {
      const int64_t first = min((int64_t)it * KI, o.rows - 1);
      base = o.base + first * o.pitch + origin * (2 * S);
      last = (int)min(o.rows - 1 - first, (int64_t)(KI - 1));
    }
    const uint32_t pitch = (uint32_t)o.pitch;
#pragma unroll
    for (int i = 0; i < instrs<B>(); ++i) {
      const int n = wave * instrs<B>() + i;
      uint32_t at;
      if constexpr (!ST) {
        const int row = min(n * 8 + (lane >> 3), last);
        at = row * pitch + (((lane & 7) ^ (lane >> 3)) << 4);
      } else {
        constexpr int L = B * 2 * S;  // bytes of a contraction row in the stage
        static_assert(L <= 1024 && L >= 128, "");
        const int k = (n * 1024 + lane * 16) / L;
        const int piece = ((lane * 16 % L) >> 4) ^ ((4 * (k & 3)) & (L / 16 - 1));
        at = min(k, last) * pitch + (uint32_t)min(piece * 16, (int)(o.width - 16 - origin * (2 * S)));
      }
      __builtin_amdgcn_global_load_lds((const void*)(base + at), (lds_void*)(lds + n * 1024), 16, 0, 0);
    }
  }

  // A lane's places in a stage of one operand: what differs between its
  // fragments by more than a constant.
  template <bool ST, int B, int T>
  struct Places {
    uint32_t o[4];
    __device__ __forceinline__ Places(int w, int lane) {
      const int h = lane >> 5, kr = (lane & 15) >> 2, q = (lane >> 4) & 1;
      constexpr int L = B * 2 * S;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        if constexpr (!ST) {
          o[v] = (w * T * 32 + (lane & 31)) * 128 + (((2 * v + h) ^ (lane & 7)) << 4);
        } else {
          const int g = (S == 1 ? 2 * (w * T + v) : 4 * (w * T) + 2 * v) + q;
          o[v] = (8 * h + kr) * L + ((g ^ ((2 * kr) & (L / 32 - 1))) << 5) + ((lane & 3) << 3);
        }
      }
    }
    // The operand of 32 rows or columns `t` of the wave, plane p, step s.
    __device__ __forceinline__ short8v read(const char* lds, int t, int p, int s) const {
      if constexpr (!ST) {
        return *(const short8v*)(lds + o[S == 1 ? s : 2 * p + s] + t * 4096);
      } else {
        static_assert(S == 1 ? T <= 4 : T % 2 == 0, "a wave's tiles must keep to the places");
        constexpr int L = B * 2 * S;
        const char* at = lds + (S == 1 ? o[t] : o[2 * (t & 1) + p] + (t >> 1) * 256) + 16 * s * L;
        const short4v u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
        const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + 4 * L));
        return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    }
  };
  typedef Places<AST, BM, TM> PlacesA;
  typedef Places<BST, BN, TN> PlacesB;

  __device__ static __forceinline__ f32x16 mma(short8v a, short8v b, f32x16 c) {
    if constexpr (BF)
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c,
                                                     0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0,
                                                    0, 0);
  }

  template <int N>
  __device__ static __forceinline__ void products(const short8v (&a)[TM], const short8v (&b)[N][TN],
                                                  f32x16 (&acc)[TM][TN]) {
#pragma unroll
    for (int p = 0; p < N; ++p)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mma(a[i], b[p][j], acc[i][j]);
  }

  // A stage's products.  The reads of the next fragments are sent before the
  // products of these, and the scheduler is kept from sending more (it would
  // spill).  fp32: a step is hi hi + hi lo, then lo hi.
  __device__ static __forceinline__ void compute(const char* la, const char* lb, const PlacesA& pa, const PlacesB& pb,
                                                 f32x16 (&acc)[TM][TN]) {
    short8v b[2][S][TN];
    auto read_b = [&](int s) __attribute__((always_inline)) {
#pragma unroll
      for (int p = 0; p < S; ++p)
#pragma unroll
        for (int j = 0; j < TN; ++j) b[s & 1][p][j] = pb.read(lb, j, p, s);
    };
    auto read_a = [&](short8v(&a)[TM], int p, int s) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < TM; ++i) a[i] = pa.read(la, i, p, s);
    };
    short8v a[2][TM];
    read_b(0);
    read_a(a[0], 0, 0);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if constexpr (S == 1) {
        if (s + 1 < kSteps) {
          read_b(s + 1);
          read_a(a[(s + 1) & 1], 0, s + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        products(a[s & 1], b[s & 1], acc);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        read_a(a[1], 1, s);
        __builtin_amdgcn_sched_barrier(0);
        products(a[0], b[s & 1], acc);
        __builtin_amdgcn_sched_barrier(0);
        if (s + 1 < kSteps) {
          read_b(s + 1);
          read_a(a[0], 0, s + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        short8v hi[1][TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) hi[0][j] = b[s & 1][0][j];
        products(a[1], hi, acc);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // The tile whose first row of A is m0 and of B n0, over the stages [it0, it1),
  // it0 < it1.
  // Between the barrier of a stage and the next one's, its operands are read
  // and the next stage's loads fly; a wave passes a barrier only with its loads
  // landed and its reads done.
  __device__ static __forceinline__ void run(const TileOperand& A, const TileOperand& B, int64_t m0, int64_t n0, int it0,
                                             int it1, char* a0, char* b0, char* a1, char* b1, f32x16 (&acc)[TM][TN]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PlacesA pa(wave / WN, lane);
    const PlacesB pb(wave % WN, lane);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};
    auto sync = [&]() __attribute__((always_inline)) {
      wait_vmcnt_le<0>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    issue<AST, BM>(A, m0, it0, a0, wave, lane);
    issue<BST, BN>(B, n0, it0, b0, wave, lane);
    // One exit, so that the accumulators are not copied at its edges; the last
    // stages are sent twice rather than under a branch.
    int it = it0;
    for (; it + 1 < it1; it += 2) {
      sync();
      issue<AST, BM>(A, m0, it + 1, a1, wave, lane);
      issue<BST, BN>(B, n0, it + 1, b1, wave, lane);
      compute(a0, b0, pa, pb, acc);
      sync();
      const int next = min(it + 2, it1 - 1);
      issue<AST, BM>(A, m0, next, a0, wave, lane);
      issue<BST, BN>(B, n0, next, b0, wave, lane);
      compute(a1, b1, pa, pb, acc);
    }
    sync();
    if (it < it1) compute(a0, b0, pa, pb, acc);
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
