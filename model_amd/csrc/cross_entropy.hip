// Softmax cross entropy of tokens over a vocabulary, from the hidden rows and
// the embedding table, without the logits in memory, and its gradients:
//
//   z_rv   = hidden_r . embedding_v
//   lse_r  = log sum_v exp(z_rv),      loss_r = lse_r - z_r,target (0 where ignored)
//   dz_rv  = (g_r + gl_r) exp(z_rv - lse_r) - g_r [v = target_r]
//   d hidden = dz . embedding,         d embedding = dz^T . hidden
//
// with g_r the loss's gradient (0 where ignored) and gl_r the logsumexp's.
//
// Forward: tiles of z (tile_mma.h: the vocabulary down, tokens across, so a
// lane's accumulators are one token's and its maximum and sum stay in
// registers) end in one (maximum, sum of 2^) pair a token and vocabulary tile;
// a second launch joins the pairs in a fixed order.  Few tokens have a kernel of
// their own (xent_rows_kernel).
//
// Backward: the vocabulary goes in pieces of up to 512 MiB of dz.  A piece's
// tiles of z are formed again from the same products and written as dz, fp16
// under a power of two a token (fp32 calls: hi and lo); two products read it from
// there, dz . embedding with its sums kept over the pieces, dz^T . hidden piece by
// piece.  Forming z again is the fourth product of size rows x vocab x d where
// three would do with the logits in memory.  dz is fp16 for bf16 calls too (the
// other operand of its products goes through fp16 under a power of two, exact
// above 2^-29 of the largest there): 8 bits of dz would put an error of bf16's own
// rounding into the gradients before they are rounded (2-norm error 1.45 times that
// of fp32 sums rounded once; 1.0 so).  In fp16 calls dz's rounding is of the
// result's size: 2-norm error 2.8e-4 where fp32 sums rounded once have 2.1e-4
// (1,001 x 50,021 x 500); hi and lo would double two of the four products.  Few
// tokens keep dz in fp32, by the same kernel as their forward, and one pass over
// the table makes both gradients (xent_few_kernel).
//
// Bound: the MFMAs.  At 16,384 x 131,072 x 1,024 bf16 the four products take 3.75,
// 4.62, 3.72 and 3.41 ms (1,175, 950, 1,185 and 1,290 TFLOP/s; a library product
// without the softmax reaches 1,210 there), the rest 0.29 (the table's largest
// magnitude, the copies of the operands, d hidden's sums): 15.8 ms in all, 105.5 the
// formula in fp32 tensors on the same machine.  What they lose is the epilogues at
// the end of each tile, which no other wave of the CU covers (128 exp a lane, 3 us
// beside 26 us of a tile at d = 1,024, and dz's bytes).  fp32 calls run three fp16
// products for one: 8,192 x 16,384 x 256 in 0.906 ms (200, 265, 194 and 169 us the
// products, 78 the operands, powers and sums), 2.71 in fp32 tensors.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "tile_mma.h"

namespace mpl {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Powers of two.  z's fp32 operands are split row by row: a hidden row and a word
// each under a power of its own, which z's tile undoes, so that no row's size costs
// another's logits bits.  dz has a power a token, 2^c, undone in d hidden's rows;
// in d embedding, which sums over tokens, the hidden rows carry 2^-c (and one power
// for all): they come weighted by their tokens' coefficients, and tokens without
// any as zeros, whatever their rows hold.  The table of dz . embedding, summed over
// words, has one power for the array.
//
// Device scalars of a call: the powers that undo those of the table and of the
// weighted hidden rows.
enum { kUndoE = 0, kUndoH, kScalars = 16 };

// The power that brings the largest magnitude, given by its bits, to [2^top,
// 2^(top + 1)); 0 for 0.
__device__ __forceinline__ int power_for(uint32_t bits, int top) {
  return bits == 0 ? 0 : max(-126, min(126, top + 127 - (int)(bits >> 23)));
}
// Magnitude bits of x, 0 if it is not finite.
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}

// ---------------------------------------------------------------- operands
// One array.  The fields that kernels choose by array stand in one struct of a
// size and alignment that scalar loads take whole: with bool vec[2] beside
// pointer arrays the compiler split the index of a scalar load into parts that
// are no multiples of 4, which those loads ignore the low bits of.
struct PackOne {
  const void* src;
  char* dst;
  int64_t rows, pitch;  // pitch in elements
  int64_t blocks;
  int64_t vec;  // rows are 16-byte aligned
};
struct PackArgs {
  PackOne e, h;  // embedding, hidden
  int d, dpad, width;  // width: lanes of a team
  int* undo_e;         // of the rows (z's fp32 operands)
  int* undo_h;
  int* scal;
  uint32_t* part;    // [kParts] of the table: largest magnitudes; of the weighted rows: their exponents
  const int* power;  // of dz's rows
};
constexpr int kParts = 512;
constexpr int kNoWeight = 1 << 16;  // the power of a token without coefficients

// i / n in 32 bits where i allows it (wave-uniform branch mostly): a 64-bit
// division is some hundred instructions.
__device__ __forceinline__ int64_t divide(int64_t i, int n) {
  return (uint64_t)i >> 32 ? i / n : (int64_t)((uint32_t)i / (uint32_t)n);
}

// Types of rows and what becomes of them: 16-bit rows that are only filled up;
// 16-bit rows as fp16 under a power of two; fp32 rows as hi and lo under one.
enum { kCopy16 = 0, kBf16ToF16, kF16, kSplit };

// 8 elements from element c of row r, zero past d.
template <int MODE>
__device__ __forceinline__ void load8(const PackOne& o, int64_t r, int64_t c, int64_t d, float (&v)[8]) {
  if constexpr (MODE == kSplit) {
    const float* x = (const float*)o.src + r * o.pitch + c;
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      if (o.vec && c + k + 4 <= d) {
        *(float4*)(v + k) = *(const float4*)(x + k);
      } else {
#pragma unroll
        for (int j = k; j < k + 4; ++j) v[j] = c + j < d ? x[j] : 0.f;
      }
    }
  } else {
    const uint16_t* x = (const uint16_t*)o.src + r * o.pitch + c;
    uint16_t u[8] __attribute__((aligned(16)));
    if (o.vec && c + 8 <= d) {
      *(uint4*)u = *(const uint4*)x;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = c + j < d ? x[j] : (uint16_t)0;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = MODE == kBf16ToF16 ? __uint_as_float((uint32_t)u[j] << 16) : (float)__builtin_bit_cast(_Float16, u[j]);
  }
}
__device__ __forceinline__ uint32_t most_of(const float (&v)[8], uint32_t most) {
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, finite_bits(v[j]));
  return most;
}
// ... and what is written of them, under a power of two.
template <int MODE>
__device__ __forceinline__ void store8(char* dst, int64_t r, int64_t dpad, int c, const float (&v)[8], int power) {
  half8 hi, lo;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float y = ldexpf(v[j], power);
    hi[j] = (_Float16)y;
    lo[j] = (_Float16)(y - (float)hi[j]);
  }
  if constexpr (MODE == kSplit) {
    char* q = dst + (r * dpad + c / 32 * 32) * 4 + (c % 32) * 2;
    *(half8*)q = hi;
    *(half8*)(q + 64) = lo;
  } else {
    *(half8*)(dst + (r * dpad + c) * 2) = hi;
  }
}

// A token's coefficients, under a power of two that leaves |dz| <= |g + gl| + |g|
// below 2^15: zeros for rows of dz that only fill it up (i >= R).  Returns the
// exponent of the hidden row's largest magnitude (its bits `most`) times the
// coefficients, from 1 on, 0 for none.
struct CoefArgs {
  const int64_t* target;
  int64_t R, rows_p, V, ignore;
  const float* g_loss;
  const float* g_lse;
  const float* lse;
  float* coef;  // [3][rows_p]: (g + gl) 2^c, g 2^c, lse
  int* power;   // [rows_p]: c
};
constexpr int kExponents = 512;  // what makes those exponents positive
__device__ __forceinline__ uint32_t coefficients(const CoefArgs& p, int64_t i, uint32_t most) {
  float all = 0.f, g = 0.f, l = 0.f;
  if (i < p.R) {
    const int64_t at = p.target[i];
    g = at == p.ignore || !p.g_loss ? 0.f : p.g_loss[i];
    if (at != p.ignore && (at < 0 || at >= p.V)) g = NAN;
    all = g + (p.g_lse ? p.g_lse[i] : 0.f);
    l = p.lse[i];
  }
  const int c = power_for(max(finite_bits(all), finite_bits(g)), 13);
  const bool weighs = all != 0.f || g != 0.f;
  p.coef[i] = ldexpf(all, c);
  p.coef[p.rows_p + i] = ldexpf(g, c);
  p.coef[2 * p.rows_p + i] = l;
  p.power[i] = weighs ? c : kNoWeight;
  return weighs && most ? kExponents + (int)(most >> 23) - c : 0;
}

// The largest of a workgroup's values, in every thread.
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
  __shared__ uint32_t s[4];
  for (int h = 32; h; h >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, h));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, s[i]);
  return m;
}

// The largest of a value that a team's lanes hold.
__device__ __forceinline__ uint32_t team_max(uint32_t m, int width) {
  for (int h = width / 2; h; h >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, h));
  return m;
}

// 16-bit calls' backward: the coefficients with the exponents of the weighted
// hidden rows (blockIdx.y = 0; a team of `width` lanes a row), and for bf16 the
// table's largest magnitude (1).
template <int MODE>
__global__ __launch_bounds__(256) void weigh_kernel(PackArgs p, CoefArgs q) {
  const PackOne o = blockIdx.y ? p.e : p.h;
  const int vecs = (p.d + 7) / 8;
  uint32_t m = 0;
  if (blockIdx.y == 0) {
    const int lane = threadIdx.x & (p.width - 1);
    const int64_t teams = (int64_t)gridDim.x * (256 / p.width);
    for (int64_t r = (int64_t)blockIdx.x * (256 / p.width) + threadIdx.x / p.width; r < q.rows_p; r += teams) {
      uint32_t most = 0;
      for (int c = r < o.rows ? lane : vecs; c < vecs; c += p.width) {
        float v[8];
        load8<MODE>(o, r, 8 * c, p.d, v);
        most = most_of(v, most);
      }
      most = team_max(most, p.width);
      if (lane == 0) m = max(m, coefficients(q, r, most));
    }
  } else {
    const int64_t n = o.rows * vecs, step = 256 * (int64_t)gridDim.x;
    auto take = [&](int64_t r, int64_t c, int64_t d) __attribute__((always_inline)) {
      float v[8];
      load8<MODE>(o, r, c, d, v);
      m = most_of(v, m);
    };
    int64_t i = blockIdx.x * 256 + threadIdx.x;
    if (o.vec && o.pitch == p.d && p.d % 8 == 0) {  // one long row
      for (; i + 7 * step < n; i += 8 * step) {  // 8 loads in flight
#pragma unroll
        for (int k = 0; k < 8; ++k) take(0, 8 * (i + k * step), 8 * n);
      }
      for (; i < n; i += step) take(0, 8 * i, 8 * n);
    } else {
      for (; i < n; i += step) {
        const int64_t r = divide(i, vecs);
        take(r, 8 * (i - r * vecs), p.d);
      }
    }
  }
  m = block_max(m);
  if (threadIdx.x == 0) p.part[blockIdx.y * kParts + blockIdx.x] = m;
}

// fp32 rows of both arrays as z's operands: hi and lo under a power of two a row,
// whose undoing power is written beside.  Of a group of 32 words those whose largest
// is within 2^-kNear of the group's take the group's power (at the cost of that many
// of 39 bits): z's tiles then undo one power a fragment.  A workgroup takes 32 rows,
// 8 lanes each, which hold their first kHold vectors of 8.  BWD: with weigh_kernel's
// part.
constexpr int kNear = 6;
template <bool BWD>
__global__ __launch_bounds__(256) void split_rows_kernel(PackArgs p, CoefArgs q) {
  constexpr int kHold = 4;
  __shared__ uint32_t largest[32];
  const bool hidden = blockIdx.y == 0;
  const PackOne o = hidden ? p.h : p.e;
  int* undo = hidden ? p.undo_h : p.undo_e;
  const int lane = threadIdx.x & 7, row = threadIdx.x >> 3, vecs = p.dpad / 8;
  const int64_t rows = BWD && hidden ? q.rows_p : o.rows;
  uint32_t m = 0;
  for (int64_t r0 = 32 * (int64_t)blockIdx.x; r0 < rows; r0 += 32 * (int64_t)gridDim.x) {
    const int64_t r = r0 + row;
    const int all = r < o.rows ? vecs : 0;
    float v[kHold][8];
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      const int c = lane + 8 * k;
      if (c >= all) continue;
      load8<kSplit>(o, r, 8 * c, p.d, v[k]);
      most = most_of(v[k], most);
    }
    for (int c = lane + 8 * kHold; c < all; c += 8) {
      float u[8];
      load8<kSplit>(o, r, 8 * c, p.d, u);
      most = most_of(u, most);
    }
    most = team_max(most, 8);
    uint32_t shared = most;
    if (!hidden) {
      if (lane == 0) largest[row] = most;
      __syncthreads();
      uint32_t group = largest[threadIdx.x & 31];
      group = team_max(group, 32);
      if (most == 0 || (most >> 23) + kNear >= group >> 23) shared = group;
      __syncthreads();
    }
    const int power = power_for(shared, 14);
    if (lane == 0 && all) undo[r] = -power;
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (lane + 8 * k < all) store8<kSplit>(o.dst, r, p.dpad, 8 * (lane + 8 * k), v[k], power);
    for (int c = lane + 8 * kHold; c < all; c += 8) {
      float u[8];
      load8<kSplit>(o, r, 8 * c, p.d, u);
      store8<kSplit>(o.dst, r, p.dpad, 8 * c, u, power);
    }
    if (BWD && !hidden) m = max(m, most);
    if (BWD && hidden && lane == 0 && r < rows) m = max(m, coefficients(q, r, most));
  }
  if (!BWD) return;
  m = block_max(m);
  if (threadIdx.x == 0) p.part[blockIdx.y * kParts + blockIdx.x] = m;
}

// Rows of an array as a tile product's operand, zero-filled to whole stages: z's
// (kCopy16), or the gradients' products'.  A thread writes 8 elements.
template <int MODE>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs p) {
  const bool hidden = blockIdx.x >= p.e.blocks;
  const PackOne o = hidden ? p.h : p.e;
  int power = 0;
  if constexpr (MODE != kCopy16) {
    const uint32_t* q = p.part + (hidden ? 0 : kParts) + threadIdx.x;
    const uint32_t most = block_max(max(q[0], q[256]));
    power = !hidden ? power_for(most, 14) : most ? 14 + 127 + kExponents - (int)most : 0;
    if (threadIdx.x == 0 && (blockIdx.x == 0 || blockIdx.x == p.e.blocks)) p.scal[hidden ? kUndoH : kUndoE] = -power;
  }
  const int per = p.dpad / 8;
  const int64_t i = (int64_t)(blockIdx.x - (hidden ? p.e.blocks : 0)) * 256 + threadIdx.x;
  if (i >= o.rows * per) return;
  const int64_t r = divide(i, per);
  const int c = 8 * (int)(i - r * per);
  if constexpr (MODE != kCopy16) {
    float v[8];
    load8<MODE>(o, r, c, p.d, v);
    if (hidden) {
      const int weight = p.power[r];
      power -= weight;
      if (weight == kNoWeight) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
      }
    }
    store8<MODE>(o.dst, r, p.dpad, c, v, power);
  } else {
    const uint16_t* x = (const uint16_t*)o.src + r * o.pitch + c;
    uint16_t v[8] __attribute__((aligned(16)));
    if (o.vec && c + 8 <= p.d) {
      *(uint4*)v = *(const uint4*)x;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < p.d ? x[j] : (uint16_t)0;
    }
    *(uint4*)(o.dst + (r * p.dpad + c) * 2) = *(const uint4*)v;
  }
}

// The words of a piece, which z no longer needs, as the operand of dz . embedding in
// fp32 calls: their rows' powers become the table's, in place.  Groups of 32 whose
// largest lies in the binade of the table's have it already and are left.
__global__ __launch_bounds__(256) void rescale_kernel(char* __restrict__ words, const int* __restrict__ undo, int64_t n,
                                                      int dpad, const uint32_t* __restrict__ part,
                                                      int* __restrict__ scal) {
  const int power = power_for(block_max(max(part[threadIdx.x], part[256 + threadIdx.x])), 14);
  if (blockIdx.x == 0 && threadIdx.x == 0) scal[kUndoE] = -power;
  const int per = dpad / 8;
  for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < n * per; i += 256 * (int64_t)gridDim.x) {
    const int64_t r = divide(i, per);
    const int by = power + undo[r];
    if (by == 0) continue;
    const int c = 8 * (int)(i - r * per);
    const char* q = words + (r * dpad + c / 32 * 32) * 4 + (c % 32) * 2;
    const half8 hi = *(const half8*)q, lo = *(const half8*)(q + 64);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)hi[j] + (float)lo[j];
    store8<kSplit>(words, r, dpad, c, v, by);
  }
}

// ------------------------------------------------------------------ forward
struct LogitArgs {
  TileOperand E, H;
  int64_t R, V;
  int iters;
  uint32_t tiles_v, tiles_t;
  const int* undo_e;  // fp32 calls: the powers that undo those of the words and of the hidden rows
  const int* undo_h;
  const int64_t* target;
  // forward
  float2* part;  // [tiles_v][R]: maximum of z, sum of exp(z - maximum)
  float* z_target;
  // backward: the piece starts at row v0 of the table
  int64_t v0, rows_p, pitch_p;  // rows_p: rows of dz that exist (zero past R); pitch in bytes
  const float* coef;            // [3][rows_p]: (g + gl) 2^c, g 2^c, lse
  char* P;
  bool stream;  // dz is written past the caches
};

// exp(z - at) for z <= at: exactly 1 at z = at, whatever their size (the powers
// are of the difference; z log2(e) - at log2(e) by a fused multiply-add leaves the
// rounding of at log2(e), 4e-6 at 100 and infinite powers from 1e9 on).
__device__ __forceinline__ float exp_below(float z, float at) {
  return __builtin_amdgcn_exp2f((z - at) * kLog2e);
}

#define MPL_TILE_LDS(C)                                      \
  __shared__ __attribute__((aligned(1024))) char a0[C::kStageA]; \
  __shared__ __attribute__((aligned(1024))) char b0[C::kStageB]; \
  __shared__ __attribute__((aligned(1024))) char a1[C::kStageA]; \
  __shared__ __attribute__((aligned(1024))) char b1[C::kStageB];

// What undoes the powers of a tile's words and of a lane's tokens (S = 2): z is an
// accumulator times 2^(word's + token's), no product of two powers, which may pass
// fp32's range on the way.  The 32 words of a fragment nearly always share one
// (kNear), and then the factor is one for all of a lane's accumulators there and
// costs no operation: it makes the difference in exp_below a fused multiply-add.
// 8,192 x 16,384 x 256 fp32, z's two kernels with one power an array 198 and 259 us,
// so 203 and 268 (on one machine; by v_ldexp of every word's own the calls of 4,096
// rows took 117 us for 109).  The words' lie in LDS since
// before the tile's product, whose barriers show them to all waves.
__device__ __forceinline__ float power_of_2(int e) {
  return __uint_as_float((uint32_t)(127 + max(-126, min(127, e))) << 23);
}
template <class C>
__device__ __forceinline__ void hold_undo(const int* undo_e, int64_t v0, int64_t V, int* undo) {
  if (C::S == 2)
    for (int i = threadIdx.x; i < C::BM; i += C::kThreads) undo[i] = undo_e[min(v0 + i, V - 1)];
}
// The tokens' powers are read before the product too: behind it a tile would wait
// for them.
template <class C>
struct Undo {
  const int* words;  // of acc[0][.][0]
  int first[C::TM], token[C::TN];
  bool shared;  // by the words of each fragment
  __device__ __forceinline__ Undo(const int* undo_h, int64_t tok, int64_t R) {
    if constexpr (C::S == 2) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) token[j] = undo_h[min(tok + 32 * j, R - 1)];
    }
  }
  __device__ __forceinline__ void behind_product(const int* undo, int lane) {
    shared = true;
    if constexpr (C::S == 2) {
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        const int u = undo[32 * i + (lane & 31)];
        first[i] = __builtin_amdgcn_readfirstlane(u);
        shared = shared && __all(u == first[i]);
      }
      words = undo + 4 * (lane >> 5);
    }
  }
  // of accumulator r (SHARED: of all) of fragment i, j
  template <bool SHARED>
  __device__ __forceinline__ float factor(int i, int j, int r) const {
    if constexpr (C::S == 1) return 1.f;
    else if constexpr (SHARED) return power_of_2(first[i] + token[j]);
    else return power_of_2(words[32 * i + 8 * (r >> 2) + (r & 3)] + token[j]);
  }
};

template <class C>
__global__ __launch_bounds__(C::kThreads) void xent_lse_kernel(LogitArgs p) {
  MPL_TILE_LDS(C)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  uint32_t tv, tt;
  tile_of(blockIdx.x, gridDim.x, p.tiles_v, p.tiles_t, 8, tv, tt);
  const int64_t v0 = (int64_t)tv * C::BM, t0 = (int64_t)tt * C::BN;
  f32x16 acc[C::TM][C::TN];
  __shared__ int undo[C::S == 2 ? C::BM : 1];
  hold_undo<C>(p.undo_e, v0, p.V, undo);
  Undo<C> z_of(p.undo_h, t0 + wn * C::TN * 32 + (lane & 31), p.R);
  C::run(p.E, p.H, v0, t0, 0, p.iters, a0, b0, a1, b1, acc);
  const int64_t vw = v0 + wm * C::TM * 32 + 4 * (lane >> 5);  // of acc[0][.][0]
  z_of.behind_product(undo + wm * C::TM * 32, lane);
  float2* pair = (float2*)a0;  // [WM][BN]: the stages are free
#pragma unroll
  for (int j = 0; j < C::TN; ++j) {
    const int64_t tok = t0 + (wn * C::TN + j) * 32 + (lane & 31);
    const int64_t at = tok < p.R ? p.target[tok] - vw : -1;  // place of the target among the lane's, if it is there
    const int place = at >= 0 && at < C::TM * 32 && !(at & 4) ? (int)at : -1;
    if (__any(place >= 0)) {
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) z = place == 32 * i + 8 * (r >> 2) + (r & 3) ? acc[i][j][r] : z;
      if (place >= 0) p.z_target[tok] = C::S == 2 ? z * power_of_2(z_of.words[place] + z_of.token[j]) : z;
    }
    if (v0 + C::BM > p.V) {
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (vw + 32 * i + 8 * (r >> 2) + (r & 3) >= p.V) acc[i][j][r] = -INFINITY;
    }
    float m = -INFINITY, s = 0.f, x, y;
    auto sums = [&](auto shared) __attribute__((always_inline)) {
      constexpr bool SHARED = decltype(shared)::value;
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        float most = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          most = fmaxf(most, SHARED ? acc[i][j][r] : acc[i][j][r] * z_of.template factor<false>(i, j, r));
        m = fmaxf(m, SHARED ? most * z_of.template factor<true>(i, j, 0) : most);
      }
      x = m, y = m;
      half_swap(x, y);
      m = fmaxf(x, y);
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s += exp_below(acc[i][j][r] * z_of.template factor<SHARED>(i, j, r), ref);
    };
    if (C::S == 1 || z_of.shared) sums(std::true_type{});
    else sums(std::false_type{});
    x = s, y = s;
    half_swap(x, y);
    if (lane < 32) pair[wm * C::BN + (wn * C::TN + j) * 32 + lane] = make_float2(m, x + y);
  }
  __syncthreads();
  for (int t = tid; t < C::BN; t += C::kThreads) {
    if (t0 + t >= p.R) continue;
    float m = pair[t].x;
#pragma unroll
    for (int w = 1; w < C::WM; ++w) m = fmaxf(m, pair[w * C::BN + t].x);
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < C::WM; ++w)
      s += pair[w * C::BN + t].y * exp_below(pair[w * C::BN + t].x, ref);
    p.part[(int64_t)tv * p.R + t0 + t] = make_float2(m, s);
  }
}

// Joins a token's pairs: a workgroup takes TOK tokens, 256 / TOK threads a
// token, each every so-manieth pair in order, then the threads in order.
template <int TOK>
__global__ __launch_bounds__(256) void xent_join_kernel(const float2* __restrict__ part, int tiles, int64_t R, int64_t V,
                                                        const int64_t* __restrict__ target, int64_t ignore,
                                                        const float* __restrict__ z_target, float* __restrict__ loss,
                                                        float* __restrict__ lse) {
  constexpr int N = 256 / TOK;
  __shared__ float2 s[N][TOK];
  const int t = threadIdx.x % TOK, g = threadIdx.x / TOK;
  const int64_t tok = (int64_t)blockIdx.x * TOK + t, at = min(tok, R - 1);
  float m = -INFINITY, l = 0.f;
  auto add = [&](float2 v) __attribute__((always_inline)) {
    const float n = fmaxf(m, v.x), ref = n == -INFINITY ? 0.f : n;
    l = l * exp_below(m, ref) + v.y * exp_below(v.x, ref);
    m = n;
  };
  int i = g;
  for (; i + 7 * N < tiles; i += 8 * N) {
    float2 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = part[(int64_t)(i + k * N) * R + at];
#pragma unroll
    for (int k = 0; k < 8; ++k) add(v[k]);
  }
  for (; i < tiles; i += N) add(part[(int64_t)i * R + at]);
  s[g][t] = make_float2(m, l);
  __syncthreads();
  if (g || tok >= R) return;
  for (int k = 1; k < N; ++k) add(s[k][t]);
  // l >= 1 and m >= the target's z, both exact where the target is the largest: the
  // loss of a learned token is log(l), not a difference of two numbers of m's size
  const float rest = log2f(l) * kLn2;
  const int64_t to = target[tok];
  lse[tok] = m + rest;
  loss[tok] = to == ignore ? 0.f : (to < 0 || to >= V) ? NAN : rest + (m - z_target[tok]);
}

// Few tokens: the table is read once, straight into the operands (no copy of
// it, no LDS), as rows of 16 bytes a lane.  A workgroup takes 32 words at a
// time; its 4 waves split d, so that a wave's loads are all in flight, and
// their sums of z meet in LDS, from where each wave keeps the running maximum
// and sum of 8 of the words.  fp32 rows go to v_mfma_f32_32x32x2_f32 as they
// are: 4 products a vector, for which lanes of half h take dims 4h .. 4h + 3 of
// each 8.  Two blocks of 32 tokens share the table's vectors (64 tokens of
// 131,072 x 1,024 fp32 406 -> 260 us), and LDS with a second barrier.  Bound: the
// table's bytes, and the fp32 products from some 100 tokens on.  One token of 16,384 x 256 fp32 6.5 us and 3.8 to join (tiles, with the
// table's copy: 30 in all); of 131,072 x 1,024 143 us, 3.7 TB/s of the table.
struct RowsArgs {
  const void* E;
  const void* H;
  int64_t e_pitch, h_pitch, R, V;
  int d;
  const int64_t* target;
  float2* part;  // [workgroups][R]
  float* z_target;
  // backward
  const float* lse;
  const float* g_loss;
  const float* g_lse;
  int64_t ignore;
  float* dz;  // [group][32 words][TOK tokens], then as much of [group][TOK tokens][32 words]
  void* rows;  // [R][d]: the hidden rows, zeros for tokens without coefficients (their dz is 0, but they may hold NaN)
};

template <typename T>
__device__ __forceinline__ uint4 row_vector(const T* row, int at, int d) {
  constexpr int VE = 16 / sizeof(T);
  typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
  if (at + VE <= d) return __builtin_bit_cast(uint4, (any4)(*(const any4*)(row + at)));
  T v[VE] __attribute__((aligned(16)));
#pragma unroll
  for (int e = 0; e < VE; ++e) v[e] = at + e < d ? row[at + e] : (T)0.f;
  return *(const uint4*)v;
}

// BWD: z becomes dz, in both orders that the products with it read.  NT: blocks
// of 32 tokens.
template <typename T, int NT, bool BWD>
__global__ __launch_bounds__(256) void xent_rows_kernel(RowsArgs p) {
  constexpr int VE = 16 / sizeof(T), TOK = 32 * NT, kBuffers = NT == 1 ? 2 : 1;
  constexpr int kAhead = NT == 1 ? 8 : 4;
  __shared__ float s[kBuffers][NT][4][16][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const T* h[NT];
  int64_t to[NT];
  float m[NT], l[NT], all[NT], gt[NT], lse[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int64_t tok = 32 * n + col, at = min(tok, p.R - 1);
    h[n] = (const T*)p.H + at * p.h_pitch;
    to[n] = p.target[at];
    m[n] = -INFINITY, l[n] = 0.f;
    if constexpr (BWD) {
      gt[n] = to[n] == p.ignore || !p.g_loss ? 0.f : p.g_loss[at];
      if (to[n] != p.ignore && (to[n] < 0 || to[n] >= p.V)) gt[n] = NAN;
      all[n] = gt[n] + (p.g_lse ? p.g_lse[at] : 0.f);
      lse[n] = p.lse[at];
      if (tok >= p.R) all[n] = gt[n] = 0.f;
    }
  }
  if constexpr (BWD) {
    __shared__ int weighs[TOK];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      if (threadIdx.x < 32) weighs[32 * n + col] = all[n] != 0.f || gt[n] != 0.f;
    __syncthreads();
    for (int i = blockIdx.x * 256 + threadIdx.x; i < (int)p.R * p.d; i += 256 * gridDim.x) {
      const int r = i / p.d;
      ((T*)p.rows)[i] = weighs[r] ? ((const T*)p.H)[r * p.h_pitch + (i - r * p.d)] : (T)0.f;
    }
  }
  const int chunks = (p.d + 2 * VE - 1) / (2 * VE);
  const int c0 = chunks * wave / 4, c1 = chunks * (wave + 1) / 4;
  const int64_t groups = (p.V + 31) / 32;
  int turn = 0;
  for (int64_t g = blockIdx.x; g < groups; g += gridDim.x, turn = kBuffers - 1 - turn) {
    const T* e = (const T*)p.E + min(32 * g + col, p.V - 1) * p.e_pitch;
    f32x16 acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = f32x16{};
    auto product = [&](uint4 a, uint4 b, f32x16& acc) __attribute__((always_inline)) {
      if constexpr (sizeof(T) == 4) {
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), acc, 0, 0, 0);
      } else if constexpr (__is_same(T, _Float16)) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), acc, 0,
                                                     0, 0);
      } else {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), acc,
                                                      0, 0, 0);
      }
    };
    int c = c0;
    for (; c + kAhead <= c1 && (c + kAhead) * 2 * VE <= p.d; c += kAhead) {
      uint4 a[kAhead], b[NT][kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) a[k] = row_vector(e, VE * (2 * (c + k) + half), 0x7FFFFFFF);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) b[n][k] = row_vector(h[n], VE * (2 * (c + k) + half), 0x7FFFFFFF);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) product(a[k], b[n][k], acc[n]);
    }
    for (; c < c1; ++c) {
      const uint4 a = row_vector(e, VE * (2 * c + half), p.d);
#pragma unroll
      for (int n = 0; n < NT; ++n) product(a, row_vector(h[n], VE * (2 * c + half), p.d), acc[n]);
    }
    if (kBuffers == 1) __syncthreads();  // with two, the other one is written next
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[turn][n][wave][r][lane] = acc[n][r];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int64_t tok = 32 * n + col;
      const float (*z4)[16][64] = s[turn][n];
      float z[4], most = m[n];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * wave + i;
        z[i] = ((z4[0][r][lane] + z4[1][r][lane]) + z4[2][r][lane]) + z4[3][r][lane];
        const int64_t v = 32 * g + 8 * wave + 4 * half + i;
        if constexpr (BWD) {
          z[i] = all[n] * exp_below(z[i], lse[n]) - (v == to[n] ? gt[n] : 0.f);
          z[i] = v < p.V && (all[n] != 0.f || gt[n] != 0.f) ? z[i] : 0.f;
          p.dz[(g * 32 + 8 * wave + 4 * half + i) * TOK + tok] = z[i];
        } else {
          if (v == to[n] && tok < p.R) p.z_target[tok] = z[i];
          z[i] = v < p.V ? z[i] : -INFINITY;
          most = fmaxf(most, z[i]);
        }
      }
      if constexpr (BWD) {
        *(float4*)(p.dz + (groups * 32 + g * 32) * TOK + tok * 32 + 8 * wave + 4 * half) =
            make_float4(z[0], z[1], z[2], z[3]);
      } else {
        const float ref = most == -INFINITY ? 0.f : most;
        l[n] *= exp_below(m[n], ref);
#pragma unroll
        for (int i = 0; i < 4; ++i) l[n] += exp_below(z[i], ref);
        m[n] = most;
      }
    }
  }
  if constexpr (!BWD) {
    // a token's 8 pairs: two halves of four waves
    __shared__ float2 pair[4][NT][64];
#pragma unroll
    for (int n = 0; n < NT; ++n) pair[wave][n][lane] = make_float2(m[n], l[n]);
    __syncthreads();
    const int n = threadIdx.x >> 5, tok = threadIdx.x;
    if (n >= NT || tok >= p.R) return;
    float most = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) most = fmaxf(most, fmaxf(pair[w][n][col].x, pair[w][n][col + 32].x));
    const float ref = most == -INFINITY ? 0.f : most;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      sum += pair[w][n][col].y * exp_below(pair[w][n][col].x, ref) +
             pair[w][n][col + 32].y * exp_below(pair[w][n][col + 32].x, ref);
    p.part[(int64_t)blockIdx.x * p.R + tok] = make_float2(most, sum);
  }
}

// ----------------------------------------------------------------- backward
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

template <class C>
__global__ __launch_bounds__(C::kThreads) void xent_dz_kernel(LogitArgs p) {
  MPL_TILE_LDS(C)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  uint32_t tv, tt;
  tile_of(blockIdx.x, gridDim.x, p.tiles_v, p.tiles_t, 8, tv, tt);
  const int64_t v0 = (int64_t)tv * C::BM, t0 = (int64_t)tt * C::BN;
  f32x16 acc[C::TM][C::TN];
  __shared__ int undo[C::S == 2 ? C::BM : 1];
  hold_undo<C>(p.undo_e, p.v0 + v0, p.V, undo);
  Undo<C> z_of(p.undo_h, t0 + wn * C::TN * 32 + (lane & 31), p.R);
  C::run(p.E, p.H, p.v0 + v0, t0, 0, p.iters, a0, b0, a1, b1, acc);
  const int half = lane >> 5;
  const int64_t vw = v0 + wm * C::TM * 32;  // the wave's first column of the piece
  // 32 tokens' rows of the wave go through LDS (the stages are free), so that a
  // row leaves as one run of ROW bytes: straight from the registers it would
  // leave by 32 bytes at a time.  16-byte piece c of row t lies at c ^ (t % 16).
  constexpr int ROW = C::TM * 32 * 2 * C::S, kPieces = ROW / 16, kWaves = C::NW / 4;
  static_assert(kWaves * 32 * ROW <= C::kStageA && kWaves * 32 * ROW <= C::kStageB, "");
  const int place = wave / kWaves;
  char* rows = (place == 0 ? a0 : place == 1 ? b0 : place == 2 ? a1 : b1) + wave % kWaves * 32 * ROW;
  z_of.behind_product(undo + wm * C::TM * 32, lane);
  auto piece = [&](int t, int c) __attribute__((always_inline)) {
    return (uint4*)(rows + t * ROW + ((c ^ (t & 15 & (kPieces - 1))) << 4));
  };
#pragma unroll
  for (int j = 0; j < C::TN; ++j) {
    const int64_t tok = t0 + (wn * C::TN + j) * 32 + (lane & 31);
    const int64_t row = min(tok, p.rows_p - 1);
    const float ga = p.coef[row], gb = p.coef[p.rows_p + row], lse = p.coef[2 * p.rows_p + row];
    const bool there = tok < p.R && (ga != 0.f || gb != 0.f);  // else dz is 0, whatever z is
    const int64_t at = (there ? p.target[tok] - p.v0 : -1) - (vw + 4 * half);
    const int to = at >= 0 && at < C::TM * 32 ? (int)at : -1;
    const bool hit = __any(to >= 0);
    const bool edge = p.v0 + v0 + C::BM > p.V;
#pragma unroll
    for (int i = 0; i < C::TM; ++i) {
      float x[16];
      auto soft = [&](auto shared) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          x[r] = ga * exp_below(acc[i][j][r] * z_of.template factor<decltype(shared)::value>(i, j, r), lse);
      };
      if (C::S == 1 || z_of.shared) soft(std::true_type{});
      else soft(std::false_type{});
      if (hit) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          x[r] -= to == 32 * i + 8 * (r >> 2) + (r & 3) ? gb : 0.f;
      }
      if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (p.v0 + vw + 4 * half + 32 * i + 8 * (r >> 2) + (r & 3) >= p.V) x[r] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = there ? x[r] : 0.f;
      // 4 neighbours a group of registers; the lane's other half holds the next 4:
      // after the exchange a lane has 8 neighbours, 16 bytes
#pragma unroll
      for (int pl = 0; pl < C::S; ++pl) {
        uint32_t u[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          half2v v;
          v[0] = (_Float16)x[2 * r];
          v[1] = (_Float16)x[2 * r + 1];
          u[r] = __builtin_bit_cast(uint32_t, v);
          if (C::S == 2 && pl == 0) {
            x[2 * r] -= (float)v[0];
            x[2 * r + 1] -= (float)v[1];
          }
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const auto sw = __builtin_amdgcn_permlane32_swap(u[4 * q + e], u[4 * q + 2 + e], false, false);
            w[e] = sw[0];
            w[2 + e] = sw[1];
          }
          *piece(lane & 31, (32 * i * 2 * C::S + 64 * pl + 32 * q) / 16 + half) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own rows: no barrier
    char* out = p.P + (t0 + (wn * C::TN + j) * 32) * p.pitch_p + vw * (2 * C::S);
    const int last = (int)min(p.rows_p - (t0 + (wn * C::TN + j) * 32), (int64_t)32);
#pragma unroll
    for (int n = 0; n < 32 * kPieces / 64; ++n) {
      const int t = (n * 64 + lane) / kPieces, c = (n * 64 + lane) % kPieces;
      const uint4 v = *piece(t, c);
      u4v* to = (u4v*)(out + t * (uint32_t)p.pitch_p + c * 16);
      if (t >= last) continue;
      if (p.stream) __builtin_nontemporal_store((u4v){v.x, v.y, v.z, v.w}, to);
      else *to = (u4v){v.x, v.y, v.z, v.w};
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// The two products with dz.  Output rows below `rows` and columns below `cols`.
struct GradArgs {
  TileOperand A, B;
  int64_t rows;
  int cols, iters, splits;
  uint32_t tiles_m, tiles_n;
  const int* undo;   // device scalar: the power that undoes the operands', or null
  const int* power;  // those of dz's rows, where they are the output's, or null
  float* part;  // [splits][rows][cols] sums, or null: the result goes to out
  bool add;     // onto what part holds
  void* out;
  int dtype;  // of out
};

__device__ __forceinline__ void store_as(void* out, int64_t i, float x, int dtype) {
  if (dtype == MPL_F32) ((float*)out)[i] = x;
  else if (dtype == MPL_F16) ((_Float16*)out)[i] = (_Float16)x;
  else ((__bf16*)out)[i] = (__bf16)x;
}

// DTYPE: of what is stored, fp32 sums or the result; ADD: onto the sums there.
template <class C, int DTYPE, bool ADD>
__device__ __forceinline__ void grad_store(const GradArgs& p, const f32x16 (&acc)[C::TM][C::TN], int64_t m0, int n0,
                                           int wm, int wn, int lane, const int* powers, void* out, bool whole) {
  constexpr int size = DTYPE == MPL_F32 ? 4 : 2;
  const int undo = p.undo ? *p.undo : 0;
  // the tile's rows from a scalar address, the lane's place in 32 bits
  char* base = (char*)out + m0 * p.cols * size;
  const int last = (int)min(p.rows - m0, (int64_t)C::BM);
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      const int col = n0 + (wn * C::TN + j) * 32 + (lane & 31);
      const int row0 = (wm * C::TM + i) * 32 + 4 * (lane >> 5);
      const uint32_t at = (uint32_t)(row0 * p.cols + col) * size;
      const int rows = col < p.cols ? last - row0 : 0;  // below it there are rows
      int power[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int4 w = p.power ? *(const int4*)(powers + row0 + 8 * q) : int4{};
        power[4 * q] = undo - w.x, power[4 * q + 1] = undo - w.y;
        power[4 * q + 2] = undo - w.z, power[4 * q + 3] = undo - w.w;
      }
      float old[16];
      if (ADD) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int step = 8 * (r >> 2) + (r & 3);
          old[r] = whole || step < rows ? *(const float*)(base + (int64_t)step * p.cols * size + at) : 0.f;
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int step = 8 * (r >> 2) + (r & 3);
        float x = ldexpf(acc[i][j][r], power[r]);
        if (ADD) x += old[r];
        char* q = base + (int64_t)step * p.cols * size + at;
        if (whole || step < rows) store_as(q, 0, x, DTYPE);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
}

template <class C>
__global__ __launch_bounds__(C::kThreads) void xent_grad_kernel(GradArgs p) {
  MPL_TILE_LDS(C)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  uint32_t tm, tn;
  tile_of(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, 8, tm, tn);
  const int64_t m0 = (int64_t)tm * C::BM;
  const int n0 = (int)tn * C::BN;
  const int split = blockIdx.y;
  const int it0 = (int)((int64_t)p.iters * split / p.splits), it1 = (int)((int64_t)p.iters * (split + 1) / p.splits);
  f32x16 acc[C::TM][C::TN];
  // dz's powers, shown to all waves by the product's barriers
  __shared__ __attribute__((aligned(16))) int powers[C::BM];
  if (p.power)
    for (int i = tid; i < C::BM; i += C::kThreads) powers[i] = p.power[min(m0 + i, p.rows - 1)];
  C::run(p.A, p.B, m0, n0, it0, it1, a0, b0, a1, b1, acc);
  float* part = p.part + (int64_t)split * p.rows * p.cols;
  const bool whole = m0 + C::BM <= p.rows && n0 + C::BN <= p.cols;
#define MPL_STORE(DTYPE, ADD, out)                                                      \
  do {                                                                                  \
    if (whole) grad_store<C, DTYPE, ADD>(p, acc, m0, n0, wm, wn, lane, powers, out, true);      \
    else grad_store<C, DTYPE, ADD>(p, acc, m0, n0, wm, wn, lane, powers, out, false);           \
  } while (0)
  if (p.part && p.add) MPL_STORE(MPL_F32, true, part);
  else if (p.part) MPL_STORE(MPL_F32, false, part);
  else if (p.dtype == MPL_F32) MPL_STORE(MPL_F32, false, p.out);
  else if (p.dtype == MPL_F16) MPL_STORE(MPL_F16, false, p.out);
  else MPL_STORE(MPL_BF16, false, p.out);
#undef MPL_STORE
}

// Few tokens' gradients: the table is read once more, and its gradient written,
// in one pass with v_mfma_f32_32x32x2_f32.  A wave has 128 columns, 4 next to
// each other a lane: their hidden rows stay in registers, and so do its sums of
// d hidden over the groups of 32 words that it walks.  Lanes of half h take words
// (and tokens) 8 m + 4 h + t at step (m, t) of a contraction.  At the end of a
// ragged row lanes take the last 4 columns again, and the same values.  Parts of
// d hidden are added by the next launch, in a fixed order.
//
// Bound: the table read and its gradient written; 1 and 32 tokens of 131,072 x
// 1,024 fp32 210 and 202 us (5.1 TB/s, what a large copy reaches), 64 tokens 306;
// 16 bits 137, 198 (2.7 TB/s: the fp32 products, at one wave a SIMD).  Two columns
// a lane and two waves a SIMD were slower (fp32, 1 and 32 tokens 265 and 298), as
// were two waves with rows widened at each use (16 bits 303 and 368: spills).
struct FewArgs {
  const void* E;
  const void* H;  // RowsArgs' rows
  int64_t e_pitch, R, V;
  int d;
  const float* dz;  // as RowsArgs
  void* de;         // or null
  float* part;      // [workgroups.x][R][d], or null
};

// 4 elements of any alignment, kept as they are until a product takes them.
template <typename T>
struct Four {
  typedef T vec __attribute__((ext_vector_type(4)));
  typedef T any __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  vec v;
  __device__ __forceinline__ void load(const T* q) { v = *(const any*)q; }
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
  __device__ static __forceinline__ void store(T* q, f4 x) { *(any*)q = __builtin_convertvector(x, vec); }
};

template <typename T, int NT>
__global__ __launch_bounds__(64) void xent_few_kernel(FewArgs p) {
  constexpr int TOK = 32 * NT;
  const int lane = threadIdx.x, col = lane & 31, half = lane >> 5;
  const int c0 = min((int)blockIdx.y * 128 + 4 * col, p.d - 4);
  const bool owns = (int)blockIdx.y * 128 + 4 * col < p.d;
  const int64_t groups = (p.V + 31) / 32;
  const int64_t g0 = groups * blockIdx.x / gridDim.x, g1 = groups * (blockIdx.x + 1) / gridDim.x;
  const float* turned = p.dz + groups * 32 * TOK;
  Four<T> h[4 * NT][4];
#pragma unroll
  for (int m = 0; m < 4 * NT; ++m)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t tok = 8 * m + 4 * half + t;
      h[m][t].load((const T*)p.H + min(tok, p.R - 1) * p.d + c0);
    }
  f32x16 dh[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) dh[n][j] = f32x16{};
  struct Group {  // of 32 words: their rows, and their dz by tokens
    Four<T> e[4][4];
    f4 at[NT][4];
  };
  auto load = [&](int64_t g, Group& x) __attribute__((always_inline)) {
    g = min(g, groups - 1);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int n = 0; n < NT; ++n) x.at[n][m] = *(const f4*)(turned + (g * TOK + 32 * n + col) * 32 + 8 * m + 4 * half);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        x.e[m][t].load((const T*)p.E + min(32 * g + 8 * m + 4 * half + t, p.V - 1) * p.e_pitch + c0);
    }
  };
  // The next group is on the way during both products, or (two blocks of tokens
  // have no registers for that) the second.
  constexpr bool kBoth = NT == 1;
  auto step = [&](int64_t g, Group& x, Group& next) __attribute__((always_inline)) {
    if (kBoth) load(g + 1, next);
    f4 a[4 * NT];
#pragma unroll
    for (int m = 0; m < 4 * NT; ++m) a[m] = *(const f4*)(p.dz + (g * 32 + col) * TOK + 8 * m + 4 * half);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            dh[n][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.at[n][m][t], x.e[m][t][j], dh[n][j], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    if (!kBoth) load(g + 1, next);
    __builtin_amdgcn_sched_barrier(0);
    if (!p.de) return;
    f32x16 o[4] = {f32x16{}, f32x16{}, f32x16{}, f32x16{}};
#pragma unroll
    for (int m = 0; m < 4 * NT; ++m) {
      if (8 * m >= p.R) break;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[m][t], h[m][t][j], o[j], 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t v = 32 * g + 8 * (r >> 2) + 4 * half + (r & 3);
      if (owns && v < p.V) Four<T>::store((T*)p.de + v * p.d + c0, (f4){o[0][r], o[1][r], o[2][r], o[3][r]});
    }
  };
  Group x[kBoth ? 2 : 1];
  load(g0, x[0]);
  int64_t g = g0;
  if constexpr (kBoth) {
    for (; g + 1 < g1; g += 2) {
      step(g, x[0], x[1]);
      step(g + 1, x[1], x[0]);
    }
    if (g < g1) step(g, x[0], x[1]);
  } else {
    for (; g < g1; ++g) step(g, x[0], x[0]);
  }
  if (!p.part) return;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t tok = 32 * n + 8 * (r >> 2) + 4 * half + (r & 3);
      if (owns && tok < p.R)
        Four<float>::store(p.part + (blockIdx.x * p.R + tok) * p.d + c0,
                           (f4){dh[n][0][r], dh[n][1][r], dh[n][2][r], dh[n][3][r]});
    }
}

// Adds many parts of few values: 32 values a workgroup, 32 threads a value, each
// every 32nd part in order, then the 32 in order.
__global__ __launch_bounds__(1024) void xent_sum_parts_kernel(const float* __restrict__ part, int parts, int64_t n,
                                                              void* __restrict__ out, int dtype) {
  __shared__ float s[32][33];
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int64_t i = blockIdx.x * 32 + (int64_t)c;
  float sum = 0.f;
  if (i < n) {
    int g = k;
    for (; g + 7 * 32 < parts; g += 8 * 32) {  // 8 loads in flight
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = part[(int64_t)(g + 32 * e) * n + i];
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += v[e];
    }
    for (; g < parts; g += 32) sum += part[(int64_t)g * n + i];
  }
  s[k][c] = sum;
  __syncthreads();
  if (k || i >= n) return;
  float all = 0.f;
#pragma unroll
  for (int g = 0; g < 32; ++g) all += s[g][c];
  store_as(out, i, all, dtype);
}

// Adds the splits' sums in order; VE values a thread (1 where n is no multiple
// of 4, or small).
template <int VE>
__global__ __launch_bounds__(256) void xent_sum_kernel(const float* __restrict__ part, int splits, int64_t n,
                                                       void* __restrict__ out, int dtype) {
  typedef float vec __attribute__((ext_vector_type(VE)));
  for (int64_t i = VE * (blockIdx.x * 256 + (int64_t)threadIdx.x); i < n; i += VE * 256 * (int64_t)gridDim.x) {
    vec s = 0.f;
    int k = 0;
    for (; k + 8 <= splits; k += 8) {  // 8 loads in flight
      vec v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = *(const vec*)(part + (k + e) * n + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e];
    }
    for (; k < splits; ++k) s += *(const vec*)(part + k * n + i);
#pragma unroll
    for (int e = 0; e < VE; ++e) store_as(out, i + e, s[e], dtype);
  }
}

void sum_splits(const float* part, int splits, int64_t n, void* out, int dtype, hipStream_t s) {
  if (n % 4 == 0 && n >= (1 << 19))
    xent_sum_kernel<4><<<(unsigned)cdiv(n, 1024), 256, 0, s>>>(part, splits, n, out, dtype);
  else
    xent_sum_kernel<1><<<(unsigned)std::min<int64_t>(cdiv(n, 256), 1 << 20), 256, 0, s>>>(part, splits, n, out, dtype);
}

// --------------------------------------------------------------------- host
template <int S, bool BF, bool AST, bool BST> using Big = TileMma<S, BF, AST, BST, 2, 4, 4, 2>;    // 256 x 256
template <int S, bool BF, bool AST, bool BST> using Mid = TileMma<S, BF, AST, BST, 2, 2, 2, 2>;    // 128 x 128

struct Plan {
  int64_t rows_p, v_piece, pieces;
  int dpad;
  int mode_z, mode;  // what the operands of z need (-1: nothing), and those of the gradients
  bool split;
  bool big_z, big_h, big_e;
  uint32_t tiles_v;    // of the forward
  uint32_t rows_grid;  // workgroups of the few-token forward, and of the backward's dz; 0: tiles
  int few, parts;      // few-token backward: blocks of 32 tokens, parts of d hidden's sums
  int splits_h, splits_e;
  // offsets into the workspace
  size_t scal, maxima, ze, zh, undo_e, undo_h, e, h, power, part, zt, coef, P, ph, pe, bytes;
};

constexpr int64_t kPieceBytes = 512ll << 20;

inline int64_t up(int64_t x, int64_t to) { return cdiv(x, to) * to; }

// Tokens up to which the table is read into the operands: the tiles read a copy
// of it that has to be made first (fp32, bf16's gradients, and 16-bit rows of
// d % 64 != 0), or go over it with mostly empty columns.  The backward has to
// take the forward's way: other kernels add z's products in another order, and
// exp(z - lse) of a learned token turns the difference, 2^-24 of z, into an error
// of p.  The few tokens' backward holds 8 bytes of dz a word and token, at most
// kFewBytes.
//
// Measured, us, few tokens / tiles, of forward and of forward with backward:
//                                  1 token              16                   32                   64
//   fp32 16,384 x 256        10 / 30  30 / 82    11 / 31  34 / 82    12 / 31  39 / 85    15 / 31  60 / 89
//        131,072 x 1,024   137 / 483 508 / 1,338 171 / 482 568 / 1,339 205 / 482 630 / 1,356 257 / 485 844 / 1,396
//   bf16 16,384 x 256         10 / 11  27 / 50    10 / 11  31 / 49    10 / 11  38 / 51    12 / 11  52 / 57
//        37,484 x 640         19 / 18  69 / 118   21 / 19  79 / 121   24 / 20  93 / 124   31 / 20 143 / 130
//        131,072 x 1,024      53 / 61 276 / 487   67 / 62 329 / 494   80 / 63 405 / 496  113 / 65 656 / 510
//        50,021 x 500         22 / 43  79 / 193   25 / 44  91 / 195   28 / 45 106 / 198   38 / 45 167 / 202
//   fp16 16,384 x 256         10 / 11  27 / 43    10 / 11  31 / 46    10 / 11  37 / 47    12 / 12  50 / 52
//        37,484 x 640         19 / 18  69 / 92    21 / 19  79 / 96    24 / 20  93 / 98    31 / 20 140 / 103
//        131,072 x 1,024      53 / 64 276 / 303   66 / 64 329 / 307   80 / 64 405 / 310  113 / 66 649 / 322
//        50,021 x 500         22 / 44  79 / 141   25 / 44  90 / 144   28 / 45 106 / 147   38 / 45 163 / 153
// 8 tokens of fp16 131,072 x 1,024: 59 / 62 and 293 / 304.  So fp32 and ragged 16-bit
// rows take it as far as the kernels go, bf16 up to 32 tokens for its gradients'
// sake (the forward alone pays up to 17 us from 16 tokens on), fp16 the same up to
// 2^26 elements of the table and 8 tokens of larger ones.
constexpr int64_t kFewBytes = 4ll << 30;
inline bool few_tokens(int64_t R, int64_t V, int d, int dtype) {
  const int64_t most = dtype == MPL_F32 || d % 64 ? 64 : dtype == MPL_BF16 || V * d < (1 << 26) ? 32 : 8;
  return d >= 4 && R <= most && up(V, 32) * up(R, 32) * 8 <= kFewBytes;
}

Plan make_plan(int64_t R, int64_t V, int d, int dtype, bool backward) {
  Plan p{};
  p.split = dtype == MPL_F32;
  const int S = p.split ? 2 : 1;
  p.mode_z = p.split ? kSplit : d % 64 ? kCopy16 : -1;
  p.mode = p.split ? kSplit : dtype == MPL_BF16 ? kBf16ToF16 : kF16;
  p.dpad = (int)up(d, 64);
  p.rows_p = up(R, 64);
  p.big_z = cdiv(R, 256) * cdiv(V, 256) >= 256;
  p.tiles_v = (uint32_t)cdiv(V, p.big_z ? 256 : 128);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at = (at + bytes + 1023) / 1024 * 1024;
    return o;
  };
  if (!backward && few_tokens(R, V, d, dtype)) {
    p.rows_grid = (uint32_t)std::min<int64_t>(cdiv(V, 32), 2048);
    p.part = take((size_t)p.rows_grid * R * 8);
    p.zt = take((size_t)R * 4);
    p.bytes = at;
    return p;
  }
  if (backward && few_tokens(R, V, d, dtype)) {
    const int64_t groups = cdiv(V, 32), waves = std::max<int64_t>(8, 1024 / cdiv(d, 128) / 8 * 8);
    p.few = R <= 32 ? 1 : 2;
    p.rows_grid = (uint32_t)std::min<int64_t>(groups, 2048);
    p.parts = (int)std::min(groups, waves);
    p.P = take((size_t)groups * 32 * p.few * 32 * 8);
    p.h = take((size_t)R * d * (dtype == MPL_F32 ? 4 : 2));
    p.ph = take((size_t)p.parts * R * d * 4);
    p.bytes = at;
    return p;
  }
  p.ze = take(p.mode_z >= 0 ? (size_t)V * p.dpad * 2 * S : 0);
  p.zh = take(p.mode_z >= 0 ? (size_t)R * p.dpad * 2 * S : 0);
  p.undo_e = take(p.split ? (size_t)V * 4 : 0);
  p.undo_h = take(p.split ? (size_t)R * 4 : 0);
  if (!backward) {
    p.part = take((size_t)p.tiles_v * R * 8);
    p.zt = take((size_t)R * 4);
    p.bytes = at;
    return p;
  }
  p.scal = take(kScalars * 4);
  p.maxima = take(2 * kParts * 4);
  p.h = take((size_t)R * p.dpad * 2 * S);
  p.power = take((size_t)p.rows_p * 4);
  // Pieces of the vocabulary: as few as their dz's bytes allow, and where the
  // table's gradient has 256 tiles in a piece, whole multiples of that: each
  // product of a piece then fills the 256 CUs evenly.
  const int64_t col = p.rows_p * 2 * S, even = 256 * cdiv(256, cdiv(d, 256));
  int64_t most = std::max<int64_t>(kPieceBytes / col / 256, 1) * 256;
  if (most >= even && most < V) most = most / even * even;
  p.pieces = cdiv(V, most);
  p.v_piece = p.pieces == 1 ? up(V, 256) : most;
  // Products with few tiles split their contraction, at least 16 stages a part
  // (8 of the small tiles).  Up to d = 128 half of a large tile would be empty
  // (8,192 x 16,384 x 128 bf16 with gradients: 361 us, 323 with small ones).
  auto pick = [&](int64_t M, int64_t K, bool& big, int& splits) {
    const int64_t tiles = cdiv(M, 256) * cdiv(d, 256), iters = K * S / 64;
    big = d > 128 && tiles * std::max<int64_t>(1, iters / 16) >= 256;
    const int64_t n = big ? tiles : cdiv(M, 128) * cdiv(d, 128), want = big ? 256 : 512;
    splits = (int)std::max<int64_t>(1, std::min(cdiv(want, n), iters / (big ? 16 : 8)));
    if (n * 4 >= want * 3) splits = 1;
  };
  pick(R, p.v_piece, p.big_h, p.splits_h);
  pick(p.v_piece, p.rows_p, p.big_e, p.splits_e);
  p.e = take(p.mode == kBf16ToF16 ? (size_t)std::min(V, p.v_piece) * p.dpad * 2 : 0);  // else z's serves
  p.coef = take((size_t)p.rows_p * 12);
  p.P = take((size_t)p.v_piece * col);
  p.ph = take(p.splits_h > 1 || p.pieces > 1 ? (size_t)p.splits_h * R * d * 4 : 0);
  p.pe = take(p.splits_e > 1 ? (size_t)p.splits_e * p.v_piece * d * 4 : 0);
  p.bytes = at;
  return p;
}

struct Call {
  const void* hidden;
  int64_t hidden_pitch;
  const void* embedding;
  int64_t embedding_pitch;
  int dtype;
  int64_t R, V;
  int d;
};

// A grid has less than 2^32 threads: 512 for a tile of 256 x 256, one for 8
// elements of a copy, for 4 of the sums (or for one, in turns), 8 for a token of
// the join.
bool sizes_ok(int64_t R, int64_t V, int d, int dtype) {
  return R >= 0 && V > 0 && d > 0 && d <= 65536 && R <= (1ll << 31) && V <= (1ll << 31) &&
         cdiv(R, 256) * cdiv(V, 256) < (1ll << 23) && (R + V) * up(d, 64) < (1ll << 34) &&
         (dtype == MPL_F32 || dtype == MPL_F16 || dtype == MPL_BF16);
}

int check_call(const char* what, const Call& c, const void* ws, size_t ws_bytes, size_t need) {
  MPL_REQUIRE(c.hidden && c.embedding, MPL_EINVAL, "%s: null buffer", what);
  MPL_REQUIRE(c.hidden_pitch >= c.d && c.embedding_pitch >= c.d, MPL_EINVAL, "%s: a pitch is below d = %d", what, c.d);
  const int size = c.dtype == MPL_F32 ? 4 : 2;
  for (const void* q : {c.hidden, c.embedding})
    MPL_REQUIRE(((uintptr_t)q & (size - 1)) == 0, MPL_EINVAL, "%s: an array is not aligned to its elements", what);
  if (c.dtype != MPL_F32 && c.d % 64 == 0)  // read as they lie
    MPL_REQUIRE(((uintptr_t)c.hidden & 15) == 0 && ((uintptr_t)c.embedding & 15) == 0 && c.hidden_pitch % 8 == 0 &&
                    c.embedding_pitch % 8 == 0,
                MPL_EINVAL, "%s: 16-bit rows of d %% 64 == 0 must be 16-byte aligned", what);
  if (c.dtype != MPL_F32 && c.d % 64 == 0)  // 256 rows of a tile in 32 bits
    MPL_REQUIRE(c.hidden_pitch < (1 << 23) && c.embedding_pitch < (1 << 23), MPL_EUNSUPPORTED,
                "%s: 16-bit rows of d %% 64 == 0 must be less than 2^23 elements apart", what);
  MPL_REQUIRE(ws && ((uintptr_t)ws & 255) == 0, MPL_EINVAL, "%s: the workspace must be 256-byte aligned", what);
  MPL_REQUIRE(ws_bytes >= need, MPL_EWORKSPACE, "%s: workspace %zu < %zu bytes", what, ws_bytes, need);
  return MPL_OK;
}

// Both arrays on their way to operands at e and h.
PackArgs pack_args(const Call& c, const Plan& p, char* ws, char* e, char* h) {
  auto one = [&](const void* src, char* dst, int64_t rows, int64_t pitch) {
    const bool vec = ((uintptr_t)src & 15) == 0 && pitch % (p.split ? 4 : 8) == 0;
    return PackOne{src, dst, rows, pitch, cdiv(rows * (p.dpad / 8), 256), vec};
  };
  PackArgs a{};
  a.e = one(c.embedding, e, c.V, c.embedding_pitch);
  a.h = one(c.hidden, h, c.R, c.hidden_pitch);
  a.d = c.d, a.dpad = p.dpad;
  for (a.width = 8; a.width < 64 && a.width < p.dpad / 8;) a.width *= 2;
  a.undo_e = (int*)(ws + p.undo_e), a.undo_h = (int*)(ws + p.undo_h);
  a.scal = (int*)(ws + p.scal);
  a.part = (uint32_t*)(ws + p.maxima);
  a.power = (const int*)(ws + p.power);
  return a;
}

// Both arrays as z's operands, the forward's and the backward's, in rows form.  In
// the backward (q) fp32 calls form the coefficients in the same launch.
void z_operands(const Call& c, const Plan& p, char* ws, const CoefArgs* q, hipStream_t s, LogitArgs& a) {
  const int64_t row = (int64_t)p.dpad * (p.split ? 4 : 2);
  if (p.mode_z < 0) {
    a.E = {(const char*)c.embedding, c.embedding_pitch * 2, c.V, row};
    a.H = {(const char*)c.hidden, c.hidden_pitch * 2, c.R, row};
    return;
  }
  a.E = {ws + p.ze, row, c.V, row};
  a.H = {ws + p.zh, row, c.R, row};
  PackArgs g = pack_args(c, p, ws, ws + p.ze, ws + p.zh);
  if (p.mode_z == kSplit) {
    a.undo_e = g.undo_e, a.undo_h = g.undo_h;
    const int64_t groups = cdiv(std::max(c.V, c.R), 32);
    if (q) split_rows_kernel<true><<<dim3(kParts, 2), 256, 0, s>>>(g, *q);
    else split_rows_kernel<false><<<dim3((unsigned)std::min<int64_t>(groups, 1 << 20), 2), 256, 0, s>>>(g, CoefArgs{});
  } else {
    pack_kernel<kCopy16><<<(unsigned)(g.e.blocks + g.h.blocks), 256, 0, s>>>(g);
  }
}

// The operands of the gradients' products of a piece of the table, rows v0 to v0 +
// nv: those for d hidden, and with the first piece the weighted hidden rows for d
// embedding, each if it is wanted; 16-bit calls form the coefficients before the
// first.  fp16 calls' table is z's as it is, fp32 calls' once it is rescaled.
void grad_operands(const Call& c, const Plan& p, char* ws, const CoefArgs& q, const LogitArgs& z, int64_t v0,
                   int64_t nv, bool want_h, bool want_e, hipStream_t s, TileOperand& E, TileOperand& H) {
  const int64_t row = (int64_t)p.dpad * (p.split ? 4 : 2);
  const bool table = want_h && p.mode == kBf16ToF16, rows = want_e && v0 == 0;
  PackArgs g = pack_args(c, p, ws, ws + p.e, ws + p.h);
  if (v0 == 0 && p.mode == kBf16ToF16) weigh_kernel<kBf16ToF16><<<dim3(kParts, table ? 2 : 1), 256, 0, s>>>(g, q);
  else if (v0 == 0 && p.mode == kF16) weigh_kernel<kF16><<<dim3(kParts, 1), 256, 0, s>>>(g, q);
  g.e.src = (const char*)g.e.src + v0 * g.e.pitch * 2;
  g.e.rows = nv;
  g.e.blocks = table ? cdiv(nv * (p.dpad / 8), 256) : 0;
  if (!rows) g.h.blocks = 0;
  const unsigned grid = (unsigned)(g.e.blocks + g.h.blocks);
  if (grid) {
    if (p.mode == kSplit) pack_kernel<kSplit><<<grid, 256, 0, s>>>(g);
    else if (p.mode == kBf16ToF16) pack_kernel<kBf16ToF16><<<grid, 256, 0, s>>>(g);
    else pack_kernel<kF16><<<grid, 256, 0, s>>>(g);
  }
  E = p.mode == kBf16ToF16 ? TileOperand{ws + p.e, row, nv, row}
                           : TileOperand{z.E.base + v0 * z.E.pitch, z.E.pitch, nv, z.E.width};
  H = {ws + p.h, row, c.R, row};
}

template <typename T, bool BWD>
void rows_kernel(unsigned grid, hipStream_t s, const RowsArgs& a) {
  if (a.R <= 32) xent_rows_kernel<T, 1, BWD><<<grid, 256, 0, s>>>(a);
  else xent_rows_kernel<T, 2, BWD><<<grid, 256, 0, s>>>(a);
}

template <bool BWD>
void rows_kernel(int dtype, unsigned grid, hipStream_t s, const RowsArgs& a) {
  if (dtype == MPL_F32) rows_kernel<float, BWD>(grid, s, a);
  else if (dtype == MPL_F16) rows_kernel<_Float16, BWD>(grid, s, a);
  else rows_kernel<__bf16, BWD>(grid, s, a);
}

template <typename T>
void few_kernel(int blocks, dim3 grid, hipStream_t s, const FewArgs& a) {
  if (blocks == 1) xent_few_kernel<T, 1><<<grid, 64, 0, s>>>(a);
  else xent_few_kernel<T, 2><<<grid, 64, 0, s>>>(a);
}

// The instantiation of one product for the operands' type and the tile.
#define MPL_TILE(KERNEL, S, BF, AST, BST, big, grid, s, args)                                           \
  do {                                                                                                  \
    if (big) KERNEL<Big<S, BF, AST, BST>><<<grid, Big<S, BF, AST, BST>::kThreads, 0, s>>>(args);        \
    else KERNEL<Mid<S, BF, AST, BST>><<<grid, Mid<S, BF, AST, BST>::kThreads, 0, s>>>(args);            \
  } while (0)

}  // namespace
}  // namespace mpl

using namespace mpl;

extern "C" size_t mpl_vocab_cross_entropy_workspace_bytes(int64_t rows, int64_t vocab, int d, int dtype, int backward) {
  if (!sizes_ok(rows, vocab, d, dtype)) return 0;
  return make_plan(rows, vocab, d, dtype, backward != 0).bytes;
}

extern "C" int mpl_vocab_cross_entropy(const void* hidden, int64_t hidden_pitch, const void* embedding,
                                       int64_t embedding_pitch, int dtype, const int64_t* target, int64_t rows,
                                       int64_t vocab, int d, int64_t ignore_index, void* workspace,
                                       size_t workspace_bytes, float* loss, float* lse, void* stream) {
  clear_error();
  const char* what = "mpl_vocab_cross_entropy";
  MPL_REQUIRE(sizes_ok(rows, vocab, d, dtype), MPL_EINVAL, "%s: bad sizes or type: rows=%lld vocab=%lld d=%d dtype=%d",
              what, (long long)rows, (long long)vocab, d, dtype);
  if (rows == 0) return MPL_OK;
  const Call c{hidden, hidden_pitch, embedding, embedding_pitch, dtype, rows, vocab, d};
  const Plan p = make_plan(rows, vocab, d, dtype, false);
  if (const int rc = check_call(what, c, workspace, workspace_bytes, p.bytes)) return rc;
  MPL_REQUIRE(target && loss && lse, MPL_EINVAL, "%s: null buffer", what);
  char* ws = (char*)workspace;
  hipStream_t s = (hipStream_t)stream;
  float2* part = (float2*)(ws + p.part);
  float* z_target = (float*)(ws + p.zt);
  auto join = [&](int pairs) {
    if (rows <= 2048)
      xent_join_kernel<4><<<(unsigned)cdiv(rows, 4), 256, 0, s>>>(part, pairs, rows, vocab, target, ignore_index,
                                                               z_target, loss, lse);
    else
      xent_join_kernel<32><<<(unsigned)cdiv(rows, 32), 256, 0, s>>>(part, pairs, rows, vocab, target, ignore_index,
                                                                 z_target, loss, lse);
    return check_launch(what);
  };
  if (p.rows_grid) {
    RowsArgs a{embedding, hidden, embedding_pitch, hidden_pitch, rows, vocab, d, target};
    a.part = part, a.z_target = z_target;
    rows_kernel<false>(dtype, p.rows_grid, s, a);
    return join((int)p.rows_grid);
  }
  LogitArgs a{};
  z_operands(c, p, ws, nullptr, s, a);
  a.R = rows, a.V = vocab;
  a.iters = p.dpad * (p.split ? 2 : 1) / 64;
  a.tiles_v = p.tiles_v;
  a.tiles_t = (uint32_t)cdiv(rows, p.big_z ? 256 : 128);
  a.target = target;
  a.part = part;
  a.z_target = z_target;
  const unsigned grid = a.tiles_v * a.tiles_t;
  if (dtype == MPL_F32) MPL_TILE(xent_lse_kernel, 2, false, false, false, p.big_z, grid, s, a);
  else if (dtype == MPL_F16) MPL_TILE(xent_lse_kernel, 1, false, false, false, p.big_z, grid, s, a);
  else MPL_TILE(xent_lse_kernel, 1, true, false, false, p.big_z, grid, s, a);
  return join((int)p.tiles_v);
}

extern "C" int mpl_vocab_cross_entropy_bwd(const void* hidden, int64_t hidden_pitch, const void* embedding,
                                           int64_t embedding_pitch, int dtype, const int64_t* target, int64_t rows,
                                           int64_t vocab, int d, int64_t ignore_index, const float* lse,
                                           const float* g_loss, const float* g_lse, void* workspace,
                                           size_t workspace_bytes, void* d_hidden, void* d_embedding, void* stream) {
  clear_error();
  const char* what = "mpl_vocab_cross_entropy_bwd";
  MPL_REQUIRE(sizes_ok(rows, vocab, d, dtype) && rows > 0, MPL_EINVAL,
              "%s: bad sizes or type: rows=%lld vocab=%lld d=%d dtype=%d", what, (long long)rows, (long long)vocab, d,
              dtype);
  const Call c{hidden, hidden_pitch, embedding, embedding_pitch, dtype, rows, vocab, d};
  const Plan p = make_plan(rows, vocab, d, dtype, true);
  if (const int rc = check_call(what, c, workspace, workspace_bytes, p.bytes)) return rc;
  MPL_REQUIRE(target && lse && (g_loss || g_lse) && (d_hidden || d_embedding), MPL_EINVAL, "%s: null buffer", what);
  char* ws = (char*)workspace;
  hipStream_t s = (hipStream_t)stream;
  if (p.few) {
    RowsArgs r{embedding, hidden, embedding_pitch, hidden_pitch, rows, vocab, d, target};
    r.lse = lse, r.g_loss = g_loss, r.g_lse = g_lse, r.ignore = ignore_index;
    r.dz = (float*)(ws + p.P), r.rows = ws + p.h;
    rows_kernel<true>(dtype, p.rows_grid, s, r);
    FewArgs f{embedding, r.rows, embedding_pitch, rows, vocab, d, r.dz, d_embedding};
    f.part = d_hidden ? (float*)(ws + p.ph) : nullptr;
    const dim3 grid(p.parts, (unsigned)cdiv(d, 128));
    if (dtype == MPL_F32) few_kernel<float>(p.few, grid, s, f);
    else if (dtype == MPL_F16) few_kernel<_Float16>(p.few, grid, s, f);
    else few_kernel<__bf16>(p.few, grid, s, f);
    if (d_hidden)
      xent_sum_parts_kernel<<<(unsigned)cdiv(rows * d, 32), 1024, 0, s>>>(f.part, p.parts, rows * d, d_hidden, dtype);
    return check_launch(what);
  }
  const int S = p.split ? 2 : 1;
  LogitArgs a{};
  const int* scal = (const int*)(ws + p.scal);
  float* coef = (float*)(ws + p.coef);
  int* power = (int*)(ws + p.power);
  const CoefArgs q{target, rows, p.rows_p, vocab, ignore_index, g_loss, g_lse, lse, coef, power};
  TileOperand E, H;
  z_operands(c, p, ws, &q, s, a);
  a.R = rows, a.V = vocab;
  a.iters = p.dpad * S / 64;
  const int bz = p.big_z ? 256 : 128;
  a.tiles_t = (uint32_t)cdiv(rows, bz);
  a.target = target;
  a.rows_p = p.rows_p;
  a.pitch_p = p.v_piece * 2 * S;
  a.coef = coef;
  a.P = ws + p.P;
  // A piece that fills the Infinity Cache (256 MiB) is written past it, so that
  // the operands stay there: 16,384 x 50,000 x 1,024 bf16 6.18 -> 6.06 ms, 8,192 x
  // 16,384 x 512 639 -> 617 us; a smaller one is read from it again: 1,024 x
  // 16,384 x 256 fp32 186 us, 194 past it.
  a.stream = p.rows_p * p.v_piece * 2 * S >= (256ll << 20);
  for (int64_t i = 0; i < p.pieces; ++i) {
    a.v0 = i * p.v_piece;
    const int64_t nv = p.v_piece < vocab - a.v0 ? p.v_piece : vocab - a.v0;  // rows of the table in the piece
    const int64_t nvp = up(nv, 256);
    grad_operands(c, p, ws, q, a, a.v0, nv, d_hidden, d_embedding, s, E, H);
    a.tiles_v = (uint32_t)(nvp / bz);
    if (p.split) MPL_TILE(xent_dz_kernel, 2, false, false, false, p.big_z, a.tiles_v * a.tiles_t, s, a);
    else if (dtype == MPL_BF16) MPL_TILE(xent_dz_kernel, 1, true, false, false, p.big_z, a.tiles_v * a.tiles_t, s, a);
    else MPL_TILE(xent_dz_kernel, 1, false, false, false, p.big_z, a.tiles_v * a.tiles_t, s, a);
    if (p.split && d_hidden)
      rescale_kernel<<<(unsigned)std::min<int64_t>(cdiv(nv * (p.dpad / 8), 256), 8192), 256, 0, s>>>(
          ws + p.ze + a.v0 * a.E.pitch, a.undo_e + a.v0, nv, p.dpad, (const uint32_t*)(ws + p.maxima) + kParts,
          (int*)(ws + p.scal));
    if (d_hidden) {
      GradArgs g{};
      g.A = {a.P, a.pitch_p, p.rows_p, a.pitch_p};
      g.B = E;
      g.rows = rows, g.cols = d;
      g.iters = (int)(nvp * S / 64);
      // a short last piece has fewer stages than parts: the others' sums stand
      g.splits = std::min(p.splits_h, g.iters);
      const int b = p.big_h ? 256 : 128;
      g.tiles_m = (uint32_t)cdiv(rows, b), g.tiles_n = (uint32_t)cdiv(d, b);
      g.undo = p.mode == kF16 ? nullptr : scal + kUndoE, g.power = power;
      g.part = p.splits_h > 1 || p.pieces > 1 ? (float*)(ws + p.ph) : nullptr;
      g.add = i > 0;
      g.out = d_hidden, g.dtype = dtype;
      const dim3 grid(g.tiles_m * g.tiles_n, g.splits);
      if (p.split) MPL_TILE(xent_grad_kernel, 2, false, false, true, p.big_h, grid, s, g);
      else MPL_TILE(xent_grad_kernel, 1, false, false, true, p.big_h, grid, s, g);
    }
    if (d_embedding) {
      GradArgs g{};
      g.A = {a.P, a.pitch_p, p.rows_p, nvp * 2 * S};
      g.B = H;
      g.rows = nv, g.cols = d;
      g.iters = (int)(p.rows_p * S / 64);
      g.splits = p.splits_e;
      const int b = p.big_e ? 256 : 128;
      g.tiles_m = (uint32_t)cdiv(nv, b), g.tiles_n = (uint32_t)cdiv(d, b);
      g.undo = scal + kUndoH;
      g.part = p.splits_e > 1 ? (float*)(ws + p.pe) : nullptr;
      g.out = (char*)d_embedding + a.v0 * d * (dtype == MPL_F32 ? 4 : 2);
      g.dtype = dtype;
      const dim3 grid(g.tiles_m * g.tiles_n, g.splits);
      if (p.split) MPL_TILE(xent_grad_kernel, 2, false, true, true, p.big_e, grid, s, g);
      else MPL_TILE(xent_grad_kernel, 1, false, true, true, p.big_e, grid, s, g);
      if (g.part) sum_splits(g.part, g.splits, nv * d, g.out, dtype, s);
    }
  }
  if (d_hidden && (p.splits_h > 1 || p.pieces > 1))
    sum_splits((const float*)(ws + p.ph), p.splits_h, rows * d, d_hidden, dtype, s);
  return check_launch(what);
}
