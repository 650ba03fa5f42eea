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
// two that brings the largest of those that share it (a row, or the array) to
// [2^14, 2^15); 11 + 11 bits and lo's sign hold x to 2^-23 of it (and to 2^-39 of
// that largest, where fp16's own range ends).  A row is then 32 hi, 32 lo, 32 hi, ... and a
// product is hi hi + hi lo + lo hi; lo lo is below 2^-22 of the product.
// Three fp16 products run at 5 times the rate of one fp32 product.
//
// LDS banks: DMA writes lanes one after the other, so the places are permuted
// at the source.  In a stage of rows the 16-byte piece c of row r lies at
// c ^ (r % 8): 8 lanes of a read cover all banks.  In a stage of columns
// 32-byte granule g of contraction row k lies at g ^ 2 (k % 4): the 4 rows
// that 16 lanes read transposed, and their neighbours' next granule, fall on
// different banks.
//
// Tiles: 256 x 256 of 8 waves (128 x 64 each: 128 accumulators a lane, two waves
// a SIMD, 128 KB of LDS, one workgroup a CU) where 256 of them exist, else
// 128 x 128 of 4 waves, two workgroups a CU, which read LDS and memory half as
// much again for a product.  Measured on fp16 operands of random mantissas,
// TFLOP/s, large / small tiles: rows x rows of 8,192 x 8,192 x 4,096 1,265 / 1,128,
// 16,384 x 16,384 x 1,024 1,030 / 1,070; rows x columns of 16,384 x 1,024 x 8,192
// 1,190 / 1,020; fp32 split 8,192 x 16,384 x 256 1,284 / 1,170 of its three products.
// Bound: the same loop without its LDS loads makes 1,435 and without its LDS
// reads as well 1,508, about what the MFMAs reach here at all; loads sent in one
// burst after the barrier held the wave's products up (1,043), so they lie
// between them.
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

  // Sends load i of the wave's instrs<B>() of stage `it` (from contraction row
  // it * KI) of one operand: a scalar address of the stage and 32-bit places of
  // the lanes in it.
  template <bool ST, int B>
  __device__ static __forceinline__ void issue(const TileOperand& o, int64_t origin, int it, char* lds, int wave,
                                               int lane, int i) {
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

  // The fragments of a step in registers: A's (fp32: hi, then lo), B's of this
  // step and the next.
  struct Frags {
    short8v a[2][TM], b[2][S][TN];
  };

  // Products of all of a with N planes of b.  `slot(n)` comes after product n;
  // the scheduler keeps what it sends there.
  template <int N, class F>
  __device__ static __forceinline__ void products(const short8v (&a)[TM], const short8v (&b)[S][TN],
                                                  f32x16 (&acc)[TM][TN], F&& slot) {
#pragma unroll
    for (int p = 0; p < N; ++p)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          acc[i][j] = mma(a[i], b[p][j], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
          slot((p * TM + i) * TN + j);
          __builtin_amdgcn_sched_barrier(0);
        }
  }

  // Loads of a stage that one wave sends, and how many of them in the last
  // group of products of the stage before the one in flight.
  static constexpr int kLoads = instrs<BM>() + instrs<BN>(), kEarly = kLoads / 2;
  // A load after every kEvery products.
  static constexpr int kEvery = TM * TN >= kLoads ? TM * TN / kEarly : 1;
  static_assert(kEarly * kEvery <= TM * TN, "the loads must fit between the products");

  // A stage's products, from the stage la, lb, whose first fragments are in
  // registers.  Between any two products at most one fragment of the next step
  // is read and every few products one load is sent: a wave issues in order, so
  // a burst of either would hold its products up until the queues drain.  The
  // barrier comes before the last group: by then the wave has read all of the
  // stage, so behind it the loads of the stage after next go over it (`fresh`,
  // the first kEarly; the next stage's first products send the rest, `old`), and
  // the first fragments of the next stage, na and nb, are read.
  template <class OLD, class NEW>
  __device__ static __forceinline__ void stage(const char* la, const char* lb, const char* na, const char* nb,
                                               const PlacesA& pa, const PlacesB& pb, Frags& f, f32x16 (&acc)[TM][TN],
                                               OLD&& old, NEW&& fresh) {
    int sent = kEarly;
    auto turn = [&]() __attribute__((always_inline)) {
      wait_vmcnt_le<0>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    auto load = [&](int n, bool last) __attribute__((always_inline)) {
      if (n % kEvery != kEvery - 1) return;
      if (last) {
        if (n / kEvery < kEarly) fresh(n / kEvery);
      } else if (sent < kLoads) {
        old(sent++);
      }
    };
    // reads fragments [from, to) of step s + 1: B's planes, then A's first plane
    auto read_next = [&](int s, int from, int to) __attribute__((always_inline)) {
      const bool last = s + 1 == kSteps;
#pragma unroll
      for (int q = from; q < to; ++q) {
        if (q < S * TN) f.b[(s + 1) & 1][q / TN % S][q % TN] = pb.read(last ? nb : lb, q % TN, q / TN % S, (s + 1) % kSteps);
        else if (q < S * TN + TM)
          f.a[S == 1 ? (s + 1) & 1 : 0][(q - S * TN) % TM] = pa.read(last ? na : la, (q - S * TN) % TM, 0, (s + 1) % kSteps);
      }
    };
    constexpr int kRead = (S * TN + TM + TM * TN - 1) / (TM * TN);  // fragments after a product
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const bool last = s + 1 == kSteps;
      if constexpr (S == 1) {
        if (last) turn();
        products<1>(f.a[s & 1], f.b[s & 1], acc, [&](int n) __attribute__((always_inline)) {
          read_next(s, n * kRead, (n + 1) * kRead);
          load(n, last);
        });
      } else {
        products<2>(f.a[0], f.b[s & 1], acc, [&](int n) __attribute__((always_inline)) {
          if (n < TM) f.a[1][n % TM] = pa.read(la, n % TM, 1, s);
          load(n, false);
        });
        if (last) turn();
        products<1>(f.a[1], f.b[s & 1], acc, [&](int n) __attribute__((always_inline)) {
          read_next(s, n * kRead, (n + 1) * kRead);
          load(n, last);
        });
      }
    }
  }

  // The tile whose first row of A is m0 and of B n0, over the stages [it0, it1),
  // it0 < it1.  One exit of the loop, so that the accumulators are not copied at
  // its edges; past the last stage it is sent again rather than under a branch.
  __device__ static __forceinline__ void run(const TileOperand& A, const TileOperand& B, int64_t m0, int64_t n0, int it0,
                                             int it1, char* a0, char* b0, char* a1, char* b1, f32x16 (&acc)[TM][TN]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PlacesA pa(wave / WN, lane);
    const PlacesB pb(wave % WN, lane);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};
    auto send = [&](int it, char* a, char* b, int n) __attribute__((always_inline)) {
      it = min(it, it1 - 1);
      if (n < instrs<BM>()) issue<AST, BM>(A, m0, it, a, wave, lane, n);
      else issue<BST, BN>(B, n0, it, b, wave, lane, n - instrs<BM>());
    };
#pragma unroll
    for (int n = 0; n < kLoads; ++n) send(it0, a0, b0, n);
#pragma unroll
    for (int n = 0; n < kEarly; ++n) send(it0 + 1, a1, b1, n);
    wait_vmcnt_le<kEarly>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    Frags f;
#pragma unroll
    for (int p = 0; p < S; ++p)
#pragma unroll
      for (int j = 0; j < TN; ++j) f.b[0][p][j] = pb.read(b0, j, p, 0);
#pragma unroll
    for (int i = 0; i < TM; ++i) f.a[0][i] = pa.read(a0, i, 0, 0);
    int it = it0;
    for (; it + 1 < it1; it += 2) {
      stage(a0, b0, a1, b1, pa, pb, f, acc, [&](int n) __attribute__((always_inline)) { send(it + 1, a1, b1, n); },
            [&](int n) __attribute__((always_inline)) { send(it + 2, a0, b0, n); });
      stage(a1, b1, a0, b0, pa, pb, f, acc, [&](int n) __attribute__((always_inline)) { send(it + 2, a0, b0, n); },
            [&](int n) __attribute__((always_inline)) { send(it + 3, a1, b1, n); });
    }
    if (it < it1) stage(a0, b0, a1, b1, pa, pb, f, acc, [](int) {}, [](int) {});
    wait_vmcnt_le<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
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
