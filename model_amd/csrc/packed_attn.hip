// Causal attention over packed sequences of unlike lengths with grouped heads
// (the backbone's attention, model.py:88-95, for sequences of lengths of their
// own), and its gradients:
//
//   z = scale q . k over the keys s <= j + Lk - Lq of query j,  lse = log sum exp z,
//   out = sum_s exp(z - lse) v_s;
//   delta = g_out . out - g_lse,  p = exp(z - lse),  dz = p (g_out . v - delta),
//   dq = scale sum_s dz k_s,  dk = scale sum_rows dz q,  dv = sum_rows p g_out.
//
// A tile of scores is formed transposed or not so that a lane holds one column of it
// and its registers are directly an operand of the next product: no score goes through
// LDS or memory.  fp32 runs on v_mfma_f32_32x32x2_f32, 16 bits on the 32x32x16
// products, both with operands staged in LDS (packed_attn16.h).  The
// backward pass forms the scores twice, for dq by rows and for dk and dv by keys: seven
// products instead of five, and no atomics.
//
// Measured (MI355X; a large bf16 product makes 1,247 TFLOP/s, an fp32 one 154), us:
//   forward, one prompt of 16,384, 16 heads over 4 of 128, bf16      1,138   966 TFLOP/s
//     the same of 16 heads of 64                                       673   817
//   backward of the latter: delta 22, dq 816 (1,010), dk and dv 1,115 (986 of its four products);
//     in fp16 2,250 for 1,945, for dz's powers of two
//   24 documents, 16,384 tokens, 16 heads over 4 of 128, bf16: forward 148, delta 40, dq 197,
//     dk and dv 324: the longest document's first tiles are most of the time
//   40 documents, 8,192 tokens, 4 heads of 64, fp32: forward 47, delta 5, dq 63, dk and dv 88
//   4,096 tokens, 8 heads of 64, fp32: forward 178 (96 TFLOP/s), backward 557 (108 of its seven products);
//     of 128: 359 (96), 1,268 (95)
//   64 single tokens over caches of up to 8,192, 32 heads over 8 of 128, bf16: 266, 5.2 TB/s
// Bound: the matrix units of large 16-bit calls (half of their cycles; the vector units
// 60 to 85 % of theirs: exponentials and conversions), memory for single tokens, for
// short sequences the chain of loads that each workgroup begins with.
#include <math.h>

#include <type_traits>

#include "packed_attn.h"
#include "packed_attn16.h"

namespace mpl {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave;

// Tokens are at most this many elements apart, and the heads that share a key head lie
// within 32 times that.  So the places of a stage of `rows` rows, of as many tokens where
// a token is one row, and of its heads are offsets of 32 bits.
constexpr int64_t kMostStride = 1 << 23;
constexpr bool far_rows_fit(int64_t rows, int64_t size) { return (rows + 32) * kMostStride * size < (int64_t)1 << 32; }

// Register r of a 32 x 32 tile holds this row of it.
__device__ __forceinline__ int tile_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

template <int HD, class T>
__device__ __forceinline__ void load_operand(float4 (&x)[HD / 8], const T* row, int half) {
#pragma unroll
  for (int g = 0; g < HD / 8; ++g) x[g] = load4(row + 8 * g + 4 * half);
}

template <class T>
__device__ __forceinline__ const T* row_at(const char* base, int64_t tok, int64_t head, int t, int h) {
  return (const T*)(base + t * tok + h * head);
}

// A wave's stage of 32 fp32 rows in LDS, by DMA: from the caches straight, a lane's own
// row costs a line a lane and a scalar load an element of a column (40 documents of
// 8,192 tokens, 4 heads of 64, with gradients: 264 us so, 191 with the stages).
template <int HD>
struct Stage32 : Stage<2 * HD> {
  typedef Stage<2 * HD> Base;
  static constexpr int kBytes = 128 * HD, kLoads = kBytes / 1024;
  static_assert(far_rows_fit(32, 4), "32-bit places");
  // The operand of the lane's row: elements 8 g + 4 (lane / 32) + [0, 4).
  __device__ __forceinline__ float4 operand(const char* lds, int g) const {
    return __builtin_bit_cast(float4, this->rows(lds, 0, g));
  }
  // Element 32 d + lane % 32 of row tile_row(r, lane / 32).
  __device__ __forceinline__ float column(const char* lds, int r, int d) const {
    const int lane = threadIdx.x & 63, half = lane >> 5, row = tile_row(r, half);
    const int piece = (8 * d + (lane >> 2 & 7)) ^ Base::f(row);
    return *(const float*)(lds + row * Base::kRow + piece * 16 + (lane & 3) * 4);
  }
};

// One operand of a product in registers, the other a stage.
template <int HD>
__device__ __forceinline__ f32x16 staged_products(const Stage32<HD>& st, const char* lds, const float4 (&y)[HD / 8]) {
  f32x16 s = f32x16{};
#pragma unroll
  for (int g = 0; g < HD / 8; ++g) {
    const float4 x = st.operand(lds, g);
    s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, y[g].x, s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, y[g].y, s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, y[g].z, s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, y[g].w, s, 0, 0, 0);
  }
  return s;
}

// The waves' results of 32 rows in LDS: sums of weighted values, the maximum (base 2)
// that was taken off and the sum of the weights.
template <int HD>
struct Join {
  float so[kWaves][32][HD + 4];
  float sm[kWaves][32], sl[kWaves][32];

  __device__ __forceinline__ void put(int wave, int col, int half, float m, float l, const f32x16 (&acc)[HD / 32]) {
    float l0 = l, l1 = l;
    half_swap(l0, l1);
    if (half == 0) {
      sm[wave][col] = m;
      sl[wave][col] = l0 + l1;
    }
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(float4*)&so[wave][col][32 * d + tile_row(r, half)] =
            make_float4(acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]);
  }

  template <class T>
  __device__ __forceinline__ void write(const Packed& a, int splits, const Segment& seg, int group, int row0, int rows,
                                        T* out, float* lse, float* part, float2* stats) const {
    for (int i = threadIdx.x; i < 32 * HD / 4; i += kThreads) {
      const int t = i / (HD / 4), d = 4 * (i % (HD / 4));
      if (row0 + t >= rows) continue;
      float mm = sm[0][t];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, sm[w][t]);
      const float ref = mm == -INFINITY ? 0.f : mm;
      float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm[w][t] - ref);  // 0 for a wave that had no block
        const float4 x = *(const float4*)&so[w][t][d];
        num.x += f * x.x; num.y += f * x.y; num.z += f * x.z; num.w += f * x.w;
        den += f * sl[w][t];
      }
      if (splits > 1) {
        const int64_t at =
            ((int64_t)blockIdx.y * a.G + group) * ((int64_t)a.T * a.R) + (int64_t)seg.first * a.R + row0 + t;
        *(float4*)(part + at * HD + d) = num;
        if (d == 0) stats[at] = make_float2(mm, den);
        continue;
      }
      const int tk = div_r(a, row0 + t);
      const int64_t at = (int64_t)(seg.first + tk) * a.H + group * a.R + row0 + t - tk * a.R;
      const float inv = den == 0.f ? 0.f : 1.f / den;  // a row without keys gives 0
      store4(out + at * HD + d, make_float4(num.x * inv, num.y * inv, num.z * inv, num.w * inv));
      if (d == 0 && lse) lse[at] = (mm + __builtin_amdgcn_logf(den)) * kLn2;
    }
  }
};

// ------------------------------------------------------------------ forward
// A workgroup of 32 rows of one group; `splits` > 1: of one part of their keys,
// whose sums go to `part` [split][group][T R][HD] and `stats` [..][2] (the running
// maximum in base 2, the sum).
template <int HD>
__global__ __launch_bounds__(kThreads) void packed_forward_kernel(const Packed a, int splits, float* __restrict__ out,
                                                                  float* __restrict__ lse, float* __restrict__ part,
                                                                  float2* __restrict__ stats) {
  typedef float T;
  constexpr int DT = HD / 32;
  constexpr int kStages = 2 * Stage32<HD>::kBytes * kWaves, kJoin = sizeof(Join<HD>);
  __shared__ __attribute__((aligned(1024))) char lds[kStages > kJoin ? kStages : kJoin];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int group = blockIdx.x % a.G;
  const Segment seg = segment_of<5>(a.starts, a.wide, a.n, a.T, a.R, blockIdx.x / a.G);
  const int rows = seg.len * a.R, tiles = (rows + 31) >> 5;
  if (seg.tile >= tiles) return;
  const int row0 = 32 * (tiles - 1 - seg.tile);  // the rows with the most keys first
  const Keys keys = keys_of(a, seg.seq);
  const int ri = min(row0 + col, rows - 1), tok = div_r(a, ri);
  const int sees = min(tok + 1 + keys.len - seg.len, keys.len);  // keys of this lane's row; <= 0 for none
  const int most = min(div_r(a, min(row0 + 31, rows - 1)) + 1 + keys.len - seg.len, keys.len);
  const int least = min(div_r(a, row0) + 1 + keys.len - seg.len, keys.len);

  float4 q[HD / 8];
  load_operand<HD>(q, row_at<T>(a.q, a.qt, a.qh, seg.first + tok, group * a.R + ri - tok * a.R), half);
  float m = -INFINITY, l = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};

  const int blocks = most > 0 ? (most + 31) >> 5 : 0, per = (blocks + splits - 1) / splits;
  const int j1 = min(blocks, ((int)blockIdx.y + 1) * per);
  const char* kb = a.k + group * a.kh + keys.first * a.kt;
  const char* vb = a.v + group * a.vh + keys.first * a.vt;
  // keys and values of a block arrive in the wave's own stages, the next block's keys
  // once this one's scores are formed, its values behind its last product
  typedef Stage32<HD> St;
  const St st;
  char* ks = lds + 2 * St::kBytes * wave;
  char* vs = ks + St::kBytes;
  auto send = [&](const char* base, int64_t pitch, int j, char* to) __attribute__((always_inline)) {
    St::template load_rows<St::kLoads, 1>(to, 0, base + 32 * j * pitch, (uint32_t)pitch, keys.len - 1 - 32 * j);
  };
  const int j0 = blockIdx.y * per + wave;
  wait_vmcnt_le<0>();  // q: the compiler does not count the stages' loads
  if (j0 < j1) {
    send(kb, a.kt, j0, ks);
    send(vb, a.vt, j0, vs);
  }
  for (int j = j0; j < j1; j += kWaves) {
    const int k0 = 32 * j;
    const bool more = j + kWaves < j1;
    wait_vmcnt_le<St::kLoads>();
    asm volatile("" ::: "memory");
    f32x16 s = staged_products<HD>(st, ks, q);
    reads_done();
    if (more) send(kb, a.kt, j + kWaves, ks);
    if (k0 + 32 > least) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (k0 + tile_row(r, half) >= sees) s[r] = -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    float a0 = mx, a1 = mx;
    half_swap(a0, a1);
    mx = fmaxf(m, fmaxf(a0, a1) * a.c);
    const float ref = mx == -INFINITY ? 0.f : mx;  // no key of the row yet
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mx;
    float sum = 0.f, p[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -ref));
      sum += p[r];
    }
    l = l * alpha + sum;
    if (more) wait_vmcnt_le<St::kLoads>();
    else wait_vmcnt_le<0>();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(st.column(vs, r, d), p[r], acc[d], 0, 0, 0);
    }
    reads_done();
    if (more) send(vb, a.vt, j + kWaves, vs);
  }
  reads_done();
  __syncthreads();  // the stages become the waves' results
  Join<HD>& join = *(Join<HD>*)lds;

  join.put(wave, col, half, m, l, acc);
  __syncthreads();
  join.write(a, splits, seg, group, row0, rows, out, lse, part, stats);
}

// ------------------------------------------------- forward, fp16 and bf16
// The running softmax of a wave's 32 rows, one a lane (both halves of the wave hold
// the same rows and different keys).  The maximum that is taken off, m, moves only
// when a row's scores pass it by 2^8 or more: until then the weights stay below
// 2^8, exact in fp32 and of the same relative error in 16 bits, and the
// accumulators need no scaling.
// fp16's weights are 2^6 times as large, which the division takes out again: with
// 2^8 that is 2^14, and those down to 2^-20 of the largest keep all their bits.
template <class T>
constexpr float kLift = __is_same(T, _Float16) ? 6.f : 0.f;

template <class T, int HD>
struct Softmax {
  static constexpr int DT = HD / 32;
  float m = -INFINITY, l = 0.f;
  f32x16 acc[DT];
  __device__ __forceinline__ Softmax() {
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  }
  // Takes in the scores of 32 keys, of which the row sees those below `sees` (counted
  // from the first; `masked`: some row of the wave does not see them all): the maximum.
  __device__ __forceinline__ void top(f32x16& s, float c, int sees, bool masked) {
    const int half = (threadIdx.x >> 5) & 1;
    if (masked) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (tile_row(r, half) >= sees) s[r] = -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    float a0 = mx, a1 = mx;
    half_swap(a0, a1);
    mx = fmaxf(a0, a1) * c;
    if (__any(mx > m + 8.f)) {
      mx = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.f : mx));
      m = mx;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
    }
  }
  // Their weights, as operands of the product with the values.
  __device__ __forceinline__ void weights(const f32x16& s, float c, short8v (&w)[2]) {
    const float ref = (m == -INFINITY ? 0.f : m) - kLift<T>;  // no key of the row yet: weights 0
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(s[8 * i + e], c, -ref));
        sum += p[e];
      }
      w[i] = round8<T>(p);
    }
    l += sum;
  }
  __device__ __forceinline__ void values(const Stage<HD>& st, const char* v, int b, const short8v (&w)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] = mma16<T>(st.cols(v, 2 * b + i, d), w[i], acc[d]);
  }
};

// Many rows: 128 a workgroup, 32 a wave, 64 keys a stage that all four waves read.  Two
// waves a SIMD of heads of 128 (225 registers, 80 KB of LDS a workgroup).
//
// The scores of the next 32 keys are formed while the softmax of these 32 runs: the
// products need the matrix unit and the softmax the vector unit, and a wave that
// alternated them would leave one or the other idle (one prompt of 16,384: 1,164 us
// without this, 1,110 with).  So keys run half a stage ahead of values, and values have
// one stage more.
constexpr int kWideRows = 128, kWideKeys = 64;
template <class T, int HD>
__global__ __launch_bounds__(kThreads, 2) void packed_forward16_kernel(const Packed a, T* __restrict__ out,
                                                                       float* __restrict__ lse) {
  typedef Stage<HD> St;
  constexpr int kBytes = kWideKeys * St::kRow, kLoads = kBytes / 1024 / kWaves;
  static_assert(far_rows_fit(kWideKeys, 2), "32-bit places");
  __shared__ __attribute__((aligned(1024))) char lds[5 * kBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int group = blockIdx.x % a.G;
  const Segment seg = segment_of<7>(a.starts, a.wide, a.n, a.T, a.R, blockIdx.x / a.G);
  const int rows = seg.len * a.R, tiles = (rows + kWideRows - 1) / kWideRows;
  if (seg.tile >= tiles) return;
  const int row0 = kWideRows * (tiles - 1 - seg.tile);  // the rows with the most keys first
  const Keys keys = keys_of(a, seg.seq);
  const int behind = keys.len - seg.len;
  const int w0 = row0 + 32 * wave, ri = min(w0 + col, rows - 1), tok = div_r(a, ri);
  const int sees = min(tok + 1 + behind, keys.len);
  const int most = min(div_r(a, min(row0 + kWideRows, rows) - 1) + 1 + behind, keys.len);
  const int wave_most = w0 < rows ? min(div_r(a, min(w0 + 32, rows) - 1) + 1 + behind, keys.len) : 0;
  const int least = min(div_r(a, min(w0, rows - 1)) + 1 + behind, keys.len);
  const char* kb = a.k + group * a.kh + keys.first * a.kt;
  const char* vb = a.v + group * a.vh + keys.first * a.vt;
  const char* qrow = a.q + (seg.first + tok) * a.qt + (group * a.R + ri - tok * a.R) * a.qh;
  auto send = [&](int it, int slot) __attribute__((always_inline)) {
    const int k0 = it * kWideKeys, last = keys.len - 1 - k0;
    St::template load_rows<kLoads, kWaves>(lds + (it & 1) * kBytes, wave, kb + k0 * a.kt, (uint32_t)a.kt, last);
    St::template load_rows<kLoads, kWaves>(lds + (2 + slot) * kBytes, wave, vb + k0 * a.vt, (uint32_t)a.vt, last);
  };
  const St st;
  const int stages = most > 0 ? (most + kWideKeys - 1) / kWideKeys : 0;
  if (stages) send(0, 0);
  short8v q[HD / 16], kf[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) q[i] = *(const short8v*)(qrow + 32 * i + 16 * half);
  Softmax<T, HD> sm;
  f32x16 s[2] = {f32x16{}, f32x16{}};
  auto turn = [&]() __attribute__((always_inline)) {
    reads_done();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto fetch = [&](const char* k, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) kf[i] = st.rows(k, b, i);
  };
  auto scores = [&](f32x16& to) __attribute__((always_inline)) {
    to = f32x16{};
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) to = mma16<T>(kf[i], q[i], to);
  };
  wait_vmcnt_le<0>();  // q too: the compiler does not count the stages' loads, and would wait for all of them
  if (stages) {
    turn();
    if (stages > 1) send(1, 1);
    fetch(lds, 0);
    scores(s[0]);
  }
  // block j of the wave: its scores are there, the next one's are formed
  auto block = [&](f32x16& now, f32x16& next, const char* v, int b, int j) __attribute__((always_inline)) {
    sm.top(now, a.c, sees - 32 * j, 32 * j + 32 > least);
    short8v w[2];
    scores(next);
    sm.weights(now, a.c, w);
    sm.values(st, v, b, w);
  };
  int slot = 0;  // it % 3
  for (int it = 0; it < stages; ++it) {
    const char* k = lds + (it & 1) * kBytes;
    const char* v = lds + (2 + slot) * kBytes;
    const bool first = it * kWideKeys < wave_most, second = it * kWideKeys + 32 < wave_most;
    if (first) {
      fetch(k, 1);
      block(s[0], s[1], v, 0, 2 * it);
    }
    if (it + 1 < stages) {
      // behind the barrier the next stage has arrived; every wave is done with this
      // one's keys and with the values before, over which the stage after next goes
      wait_vmcnt_le<0>();
      turn();
      if (it + 2 < stages) send(it + 2, slot == 0 ? 2 : slot - 1);
    }
    if (second) {
      fetch(lds + ((it + 1) & 1) * kBytes, 0);  // past the last stage: not used
      block(s[1], s[0], v, 1, 2 * it + 1);
    }
    slot = slot == 2 ? 0 : slot + 1;
  }
  float l0 = sm.l, l1 = sm.l;
  half_swap(l0, l1);
  const float l = l0 + l1, inv = l == 0.f ? 0.f : 1.f / l;  // a row without keys gives 0
  if (w0 + col >= rows) return;
  const int64_t at = (int64_t)(seg.first + tok) * a.H + group * a.R + ri - tok * a.R;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      store4(out + at * HD + 32 * d + tile_row(r, half), make_float4(sm.acc[d][r] * inv, sm.acc[d][r + 1] * inv,
                                                                    sm.acc[d][r + 2] * inv, sm.acc[d][r + 3] * inv));
  if (lse && half == 0) lse[at] = (sm.m - kLift<T> + __builtin_amdgcn_logf(l)) * kLn2;
}

// Few rows: 32 a workgroup; every wave has keys, and stages of 32 of them, of its own,
// two under way: with single tokens over a cache 64 KB a CU (heads of 128).
template <class T, int HD>
__global__ __launch_bounds__(kThreads) void packed_forward16_few_kernel(const Packed a, int splits, T* __restrict__ out,
                                                                        float* __restrict__ lse, float* __restrict__ part,
                                                                        float2* __restrict__ stats) {
  typedef Stage<HD> St;
  constexpr int kBytes = 32 * St::kRow, kLoads = kBytes / 1024;
  constexpr int kStages = 4 * kBytes * kWaves, kJoin = sizeof(Join<HD>);
  __shared__ __attribute__((aligned(1024))) char lds[kStages > kJoin ? kStages : kJoin];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int group = blockIdx.x % a.G;
  const Segment seg = segment_of<5>(a.starts, a.wide, a.n, a.T, a.R, blockIdx.x / a.G);
  const int rows = seg.len * a.R, tiles = (rows + 31) >> 5;
  if (seg.tile >= tiles) return;
  const int row0 = 32 * (tiles - 1 - seg.tile);
  const Keys keys = keys_of(a, seg.seq);
  const int behind = keys.len - seg.len;
  const int ri = min(row0 + col, rows - 1), tok = div_r(a, ri);
  const int sees = min(tok + 1 + behind, keys.len);
  const int most = min(div_r(a, min(row0 + 32, rows) - 1) + 1 + behind, keys.len);
  const int least = min(div_r(a, row0) + 1 + behind, keys.len);
  const char* kb = a.k + group * a.kh + keys.first * a.kt;
  const char* vb = a.v + group * a.vh + keys.first * a.vt;
  const char* qrow = a.q + (seg.first + tok) * a.qt + (group * a.R + ri - tok * a.R) * a.qh;
  const int blocks = most > 0 ? (most + 31) >> 5 : 0, per = (blocks + splits - 1) / splits;
  const int j0 = blockIdx.y * per + wave, j1 = min(blocks, ((int)blockIdx.y + 1) * per);
  char* mine = lds + 4 * kBytes * wave;
  auto send = [&](int j, char* to) __attribute__((always_inline)) {
    const int last = keys.len - 1 - 32 * j;
    St::template load_rows<kLoads, 1>(to, 0, kb + 32 * j * a.kt, (uint32_t)a.kt, last);
    St::template load_rows<kLoads, 1>(to + kBytes, 0, vb + 32 * j * a.vt, (uint32_t)a.vt, last);
  };
  const St st;
  short8v q[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) q[i] = *(const short8v*)(qrow + 32 * i + 16 * half);
  Softmax<T, HD> sm;
  if (j0 < j1) send(j0, mine);
  wait_vmcnt_le<0>();  // q too: the compiler does not count the stages' loads, and would wait for all of them
  int turn = 0;
  for (int j = j0; j < j1; j += kWaves, turn ^= 1) {
    reads_done();  // of the stage before, over which the next is sent
    if (j + kWaves < j1) {
      send(j + kWaves, mine + 2 * kBytes * (turn ^ 1));
      wait_vmcnt_le<2 * kLoads>();
    } else {
      wait_vmcnt_le<0>();
    }
    asm volatile("" ::: "memory");
    const char* at = mine + 2 * kBytes * turn;
    f32x16 s = f32x16{};
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) s = mma16<T>(st.rows(at, 0, i), q[i], s);
    short8v w[2];
    sm.top(s, a.c, sees - 32 * j, 32 * j + 32 > least);
    sm.weights(s, a.c, w);
    sm.values(st, at + kBytes, 0, w);
  }
  reads_done();
  __syncthreads();  // the stages become the waves' results
  Join<HD>& join = *(Join<HD>*)lds;
  join.put(wave, col, half, sm.m - kLift<T>, sm.l, sm.acc);
  __syncthreads();
  join.write(a, splits, seg, group, row0, rows, out, lse, part, stats);
}

// Joins the parts of the keys: HD / 4 lanes a row.
template <class T, int HD>
__global__ __launch_bounds__(256) void packed_join_kernel(const Packed a, int splits, const float* __restrict__ part,
                                                          const float2* __restrict__ stats, T* __restrict__ out,
                                                          float* __restrict__ lse) {
  const uint32_t rows = (uint32_t)a.T * a.R;
  const int64_t all = (int64_t)rows * a.G;
  const uint32_t at = (blockIdx.x * 256u + threadIdx.x) / (HD / 4);  // below 2^29 for all rows
  const int d = 4 * (threadIdx.x % (HD / 4));
  if (at >= all) return;
  float mm = -INFINITY;
  for (int s = 0; s < splits; ++s) mm = fmaxf(mm, stats[s * all + at].x);
  const float ref = mm == -INFINITY ? 0.f : mm;
  float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float2 st = stats[s * all + at];
    const float f = __builtin_amdgcn_exp2f(st.x - ref);
    const float4 x = *(const float4*)(part + (s * all + at) * HD + d);
    num.x += f * x.x; num.y += f * x.y; num.z += f * x.z; num.w += f * x.w;
    den += f * st.y;
  }
  const int group = at / rows, row = at % rows, tk = div_r(a, row);
  const int64_t to = (int64_t)tk * a.H + group * a.R + row - tk * a.R;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  store4(out + to * HD + d, make_float4(num.x * inv, num.y * inv, num.z * inv, num.w * inv));
  if (d == 0 && lse) lse[to] = (mm + __builtin_amdgcn_logf(den)) * kLn2;
}

// ----------------------------------------------------------------- backward
struct Grads {
  const char* g_out;
  int64_t gt, gh;  // bytes
  const float* lse2;  // [group][T R]: base 2, +inf for a row without keys
  float* delta;       // [group][T R]
  const float* g_lse;
  float scale;
};

// lse2 and delta of every row, HD / 4 lanes a row.
constexpr int kDeltaBlocks = 1024;
template <int L>
__device__ __forceinline__ float sum_lanes(float x) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

template <class T, int HD>
__global__ __launch_bounds__(256) void packed_delta_kernel(const Packed a, const char* __restrict__ g_out, int64_t gt,
                                                           int64_t gh, const T* __restrict__ out,
                                                           const float* __restrict__ lse,
                                                           const float* __restrict__ g_lse, float* __restrict__ lse2,
                                                           float* __restrict__ delta) {
  constexpr int L = HD / 4;
  const int d = 4 * (threadIdx.x % L);
  const uint32_t rows = (uint32_t)a.T * a.H;  // below 2^29
  for (uint32_t first = blockIdx.x * (256 / L); first < rows; first += gridDim.x * (256 / L)) {
    const uint32_t at = first + threadIdx.x / L, row = min(at, rows - 1);
    const int t = row / (uint32_t)a.H, h = row % (uint32_t)a.H;
    const float4 x = load4(row_at<T>(g_out, gt, gh, t, h) + d), y = load4(out + (int64_t)row * HD + d);
    const float s = sum_lanes<L>(x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w);
    if (at < rows && d == 0) {
      const int g = div_r(a, h);
      const int64_t to = (int64_t)g * a.T * a.R + (int64_t)t * a.R + h - g * a.R;
      const float z = lse[row];
      lse2[to] = z == -INFINITY ? INFINITY : z * kLog2e;
      delta[to] = s - (g_lse ? g_lse[row] : 0.f);
    }
  }
}

// The sums of N sets of RW waves, 32 rows each, joined in LDS and written.
template <int HD, int N, int RW>
struct Sums {
  float so[N][RW][32][HD + 4];
  __device__ __forceinline__ void put(int n, int rw, int col, int half, const f32x16 (&acc)[HD / 32], float f) {
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(float4*)&so[n][rw][col][32 * d + tile_row(r, half)] =
            make_float4(acc[d][r] * f, acc[d][r + 1] * f, acc[d][r + 2] * f, acc[d][r + 3] * f);
  }
  // `place(t)`: where row t goes, null for nowhere; those from `kept` on are 0.
  template <class F>
  __device__ __forceinline__ void write(int kept, F&& place) const {
    for (int i = threadIdx.x; i < N * 32 * HD / 4; i += 64 * N * RW) {
      const int t = i / (HD / 4), d = 4 * (i % (HD / 4));
      auto* to = place(t);
      if (!to) continue;
      float4 x = *(const float4*)&so[t >> 5][0][t & 31][d];
#pragma unroll
      for (int w = 1; w < RW; ++w) {
        const float4 y = *(const float4*)&so[t >> 5][w][t & 31][d];
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
      store4(to + d, t < kept ? x : make_float4(0.f, 0.f, 0.f, 0.f));
    }
  }
};

// dq: 32 rows a workgroup, tiles of scores transposed (the lane's column a row).
template <int HD>
__global__ __launch_bounds__(kThreads) void packed_dq_kernel(const Packed a, const Grads g, float* __restrict__ dq) {
  typedef float T;
  constexpr int DT = HD / 32;
  constexpr int kStages = 2 * Stage32<HD>::kBytes * kWaves, kJoin = sizeof(Sums<HD, 1, kWaves>);
  __shared__ __attribute__((aligned(1024))) char lds[kStages > kJoin ? kStages : kJoin];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int group = blockIdx.x % a.G;
  const Segment seg = segment_of<5>(a.starts, a.wide, a.n, a.T, a.R, blockIdx.x / a.G);
  const int rows = seg.len * a.R, tiles = (rows + 31) >> 5;
  if (seg.tile >= tiles) return;
  const int row0 = 32 * (tiles - 1 - seg.tile);
  const Keys keys = keys_of(a, seg.seq);
  const int ri = min(row0 + col, rows - 1), tok = div_r(a, ri);
  const int sees = min(tok + 1 + keys.len - seg.len, keys.len);
  const int most = min(div_r(a, min(row0 + 31, rows - 1)) + 1 + keys.len - seg.len, keys.len);
  const int least = min(div_r(a, row0) + 1 + keys.len - seg.len, keys.len);
  const int head = group * a.R + ri - tok * a.R;

  float4 q[HD / 8], go[HD / 8];
  load_operand<HD>(q, row_at<T>(a.q, a.qt, a.qh, seg.first + tok, head), half);
  load_operand<HD>(go, row_at<T>(g.g_out, g.gt, g.gh, seg.first + tok, head), half);
  const int64_t st = (int64_t)group * a.T * a.R + (int64_t)seg.first * a.R + ri;
  const float lse2 = g.lse2[st], delta = g.delta[st];
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  const int blocks = most > 0 ? (most + 31) >> 5 : 0;
  const char* kb = a.k + group * a.kh + keys.first * a.kt;
  const char* vb = a.v + group * a.vh + keys.first * a.vt;
  // as in the forward pass: values first, whose stage is free again after one product
  typedef Stage32<HD> St;
  const St stage;
  char* ks = lds + 2 * St::kBytes * wave;
  char* vs = ks + St::kBytes;
  auto send = [&](const char* base, int64_t pitch, int j, char* to) __attribute__((always_inline)) {
    St::template load_rows<St::kLoads, 1>(to, 0, base + 32 * j * pitch, (uint32_t)pitch, keys.len - 1 - 32 * j);
  };
  wait_vmcnt_le<0>();  // the rows: the compiler does not count the stages' loads
  if (wave < blocks) {
    send(vb, a.vt, wave, vs);
    send(kb, a.kt, wave, ks);
  }
  for (int j = wave; j < blocks; j += kWaves) {
    const int k0 = 32 * j;
    const bool more = j + kWaves < blocks;
    wait_vmcnt_le<St::kLoads>();
    asm volatile("" ::: "memory");
    f32x16 ds = staged_products<HD>(stage, vs, go);
    reads_done();
    if (more) {
      send(vb, a.vt, j + kWaves, vs);
      wait_vmcnt_le<St::kLoads>();
    } else {
      wait_vmcnt_le<0>();
    }
    asm volatile("" ::: "memory");
    const f32x16 s = staged_products<HD>(stage, ks, q);
    const bool masked = k0 + 32 > least;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lse2)) * (ds[r] - delta);
      if (masked && k0 + tile_row(r, half) >= sees) ds[r] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(stage.column(ks, r, d), ds[r], acc[d], 0, 0, 0);
      }
    reads_done();
    if (more) send(kb, a.kt, j + kWaves, ks);
  }
  reads_done();
  __syncthreads();  // the stages become the waves' sums
  Sums<HD, 1, kWaves>& sums = *(Sums<HD, 1, kWaves>*)lds;
  sums.put(0, wave, col, half, acc, g.scale);
  __syncthreads();
  sums.write(32, [&](int t) -> T* {
    if (row0 + t >= rows) return nullptr;
    const int tk = div_r(a, row0 + t);
    return dq + ((int64_t)(seg.first + tk) * a.H + group * a.R + row0 + t - tk * a.R) * HD;
  });
}

// dk and dv: 32 keys a workgroup, the lane's column a key, rows in the registers.
template <int HD>
__global__ __launch_bounds__(kThreads, HD <= 64 ? 2 : 1) void packed_dkv_kernel(const Packed a, const Grads g,
                                                                               float* __restrict__ dk,
                                                                               float* __restrict__ dv) {
  typedef float T;
  constexpr int DT = HD / 32;
  constexpr int kStages = 2 * Stage32<HD>::kBytes * kWaves, kJoin = sizeof(Sums<HD, 1, kWaves>);
  __shared__ __attribute__((aligned(1024))) char lds[kStages > kJoin ? kStages : kJoin];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int group = blockIdx.x % a.G;
  const Segment seg = segment_of<5>(a.key_starts, a.wide, a.n, a.S, 1, blockIdx.x / a.G);
  if (32 * seg.tile >= seg.len) return;
  const int k0 = 32 * seg.tile;
  const bool real = seg.seq >= 0 && seg.seq < a.n;
  const int len = real ? keys_of(a, seg.seq).len : 0;  // of the segment's keys those in use
  int first = 0, rows = 0, behind = 0;
  if (real) {
    first = __builtin_amdgcn_readfirstlane(segment_start(a.starts, a.wide, a.n, a.T, seg.seq + 1));
    const int end = __builtin_amdgcn_readfirstlane(segment_start(a.starts, a.wide, a.n, a.T, seg.seq + 2));
    const int tokens = max(end - first, 0);
    rows = tokens * a.R;
    behind = len - tokens;  // token j sees the keys below j + 1 + behind
  }
  f32x16 ak[DT], av[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) ak[d] = av[d] = f32x16{};
  if (k0 < len) {
    const int key = min(k0 + col, len - 1);
    const T* krow = row_at<T>(a.k, a.kt, a.kh, seg.first + key, group);
    const T* vrow = row_at<T>(a.v, a.vt, a.vh, seg.first + key, group);
    float4 k[HD / 8], v[HD / 8];
    load_operand<HD>(k, krow, half);
    load_operand<HD>(v, vrow, half);
    const int64_t st = (int64_t)group * a.T * a.R + (int64_t)first * a.R;
    const int row_from = max(k0 - behind, 0) * a.R, blocks = (rows + 31) >> 5;
    const int row_min = max(k0 + col - behind, 0) * a.R;  // the first row that sees the lane's key
    // rows of g_out and q in the wave's own stages, each sent again behind its last product
    typedef Stage32<HD> St;
    const St stage;
    char* gs = lds + 2 * St::kBytes * wave;
    char* qs = gs + St::kBytes;
    auto send = [&](const char* base, int64_t tok, int64_t head, int j, char* to) __attribute__((always_inline)) {
      const int t0 = div_r(a, 32 * j);
      const char* at = base + (int64_t)(first + t0) * tok + group * a.R * head;
#pragma unroll
      for (int i = 0; i < St::kLoads; ++i) {
        const int row = min(32 * j + St::load_row(i), rows - 1), tk = div_r(a, row);
        St::load(to, i, at, (uint32_t)(tk - t0) * (uint32_t)tok + (row - tk * a.R) * (uint32_t)head);
      }
    };
    const int from = (row_from >> 5) + wave;
    float next = 0.f;
    // the rows' lse2 and delta by two lanes a row, and from them by shuffles
    auto stat = [&](int j) __attribute__((always_inline)) {
      next = (half ? g.delta : g.lse2)[st + min(32 * j + col, rows - 1)];
    };
    if (from < blocks) stat(from);
    wait_vmcnt_le<0>();  // the keys too: the compiler does not count the stages' loads
    if (from < blocks) {
      send(g.g_out, g.gt, g.gh, from, gs);
      send(a.q, a.qt, a.qh, from, qs);
    }
    for (int j = from; j < blocks; j += kWaves) {
      const int r0 = 32 * j;
      const bool more = j + kWaves < blocks;
      const float mine = next;
      wait_vmcnt_le<St::kLoads>();
      asm volatile("" ::: "memory");
      f32x16 ds = staged_products<HD>(stage, gs, v);
      wait_vmcnt_le<0>();
      asm volatile("" ::: "memory");
      f32x16 s = staged_products<HD>(stage, qs, k);
      if (more) stat(j + kWaves);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = r0 + tile_row(r, half), at = min(row, rows - 1);
        const bool off = row >= rows || at < row_min || k0 + col >= len;
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -__shfl(mine, tile_row(r, half))));
        const float e = __shfl(mine, 32 + tile_row(r, half));
        s[r] = off ? 0.f : p;
        ds[r] = off ? 0.f : p * (ds[r] - e);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          av[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(stage.column(gs, r, d), s[r], av[d], 0, 0, 0);
      reads_done();
      if (more) {
        wait_vmcnt_le<0>();  // the next rows' lse2, before loads that the compiler does not count
        send(g.g_out, g.gt, g.gh, j + kWaves, gs);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          ak[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(stage.column(qs, r, d), ds[r], ak[d], 0, 0, 0);
      reads_done();
      if (more) send(a.q, a.qt, a.qh, j + kWaves, qs);
    }
  }
  Sums<HD, 1, kWaves>& sums = *(Sums<HD, 1, kWaves>*)lds;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    T* to = which ? dv : dk;
    if (!to) continue;
    reads_done();
    __syncthreads();  // the stages become the waves' sums
    sums.put(0, wave, col, half, which ? av : ak, which ? 1.f : g.scale);
    __syncthreads();
    sums.write(len - k0, [&](int t) -> T* {  // places not in use have gradients 0
      return k0 + t < seg.len ? to + ((int64_t)(seg.first + k0 + t) * a.G + group) * HD : nullptr;
    });
  }
}

// ------------------------------------------------ backward, fp16 and bf16
// dz is rounded to fp16 under a power of two of the lane's column (a row in dq, a key
// in dk and dv; both halves of the wave hold the same ones): the largest |dz| so far goes
// to [2^13, 2^14) when it is found and stays below 2^15, else the power falls, and the
// accumulators with it.  So nothing overflows, and dz keeps all its bits down to 2^-27 of
// the column's largest, whatever the other rows and keys, sequences or places not in use
// hold.  (One power for the whole call, of its largest |g_out| and |v|, cost a sequence
// its bits for another's size, and a pass over all of v.)  What is not finite takes its
// own column along.  bf16 has fp32's range and takes none.
template <class T, int HD>
struct Unit {
  static constexpr bool kNone = !__is_same(T, _Float16);
  uint32_t e = 227;  // of the power, biased by 127: at most 2^100, so that the inverse is finite
  // x, the column's next 16 dz, times the power; acc is in the power's measure
  __device__ __forceinline__ void scale(f32x16& x, f32x16 (&acc)[HD / 32]) {
    if constexpr (kNone) return;
    float top = fabsf(x[0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
    float t0 = top, t1 = top;
    half_swap(t0, t1);
    top = fmaxf(t0, t1);
    if (__any(top * power() >= 32768.f)) {
      const uint32_t now = top * power() >= 32768.f ? 127 + 13 + 127 - (__float_as_uint(top) >> 23) : e;
      const float f = __uint_as_float((uint32_t)max(127 + (int)now - (int)e, 0) << 23);  // 0 below 2^-126
      e = now;
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= f;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= power();
  }
  __device__ __forceinline__ float power() const { return __uint_as_float(e << 23); }
  __device__ __forceinline__ float inverse() const { return kNone ? 1.f : __uint_as_float((254 - e) << 23); }
};

// fp16's weights in dv, at most 1, are 2^14 times as large.
template <class T>
constexpr float kLiftP = __is_same(T, _Float16) ? 16384.f : 1.f;

// dq.  WIDE: 128 rows a workgroup, 32 a wave, 64 keys a stage that all waves read;
// else 32 rows, and every wave has keys and stages of its own.
//
// delta = g_out . out is as good as out, which was rounded to 16 bits; where a row's
// weights lie on few keys, out is as large as v, and that error shows in dq and dk.  The
// exact one is sum p dp - g_lse, known once all keys have been seen.  Tiles of up to
// kExactKeys keys form it in a sweep of their own, two thirds of dq once more; with more
// keys out is an average more often.  Heads of 32 are the ones that lose most, and have
// registers left: they take g_out . out as they go, sum p k beside dz k, and add
// (g_out . out - sum p dp) sum p k at the end, one product instead of the sweep's two and
// its exponentials.  Either way delta goes to memory for dk.
//
// Error of dq by its norm, in errors of the exact value rounded once, and us of the
// backward pass (bf16, 4,096 tokens, scores of standard deviation 1.7), sequences of
//                                            512           1,024         4,096
//   16 heads of 64, sweep up to 256 keys:    1.467   68    1.487   86    1.499  194
//     512:                                   1.432   73    1.463   87    1.485  196
//     all:                                   1.432   73    1.439  104    1.446  245
//   16 over 4 of 128, sweep up to 256:       1.451   90    1.460  143    1.457  422
//     512:                                   1.427  103    1.443  145    1.447  424
//     all:                                   1.427  103    1.427  168    1.427  507
//   16 of 32, sweep up to 512:               1.466   49    1.514   56    1.554  115
//     beside dz k, all:                      1.463   44    1.470   55    1.480  120
// (Two roundings, dz's and dq's own, make 1.414.)
constexpr int kExactKeys = 512;
template <class T, int HD, bool WIDE>
__global__ __launch_bounds__(kThreads, WIDE ? 2 : 1) void packed_dq16_kernel(const Packed a, const Grads g,
                                                                            T* __restrict__ dq) {
  typedef Stage<HD> St;
  constexpr int B = WIDE ? 2 : 1, kKeys = 32 * B, kRows = WIDE ? 128 : 32;
  static_assert(far_rows_fit(kKeys, 2), "32-bit places");
  constexpr int kBytes = kKeys * St::kRow, kLoads = kBytes / 1024 / (WIDE ? kWaves : 1);
  constexpr int kStages = 4 * kBytes * (WIDE ? 1 : kWaves), kJoin = WIDE ? 0 : sizeof(Sums<HD, 1, kWaves>);
  __shared__ __attribute__((aligned(1024))) char lds[kStages > kJoin ? kStages : kJoin];
  __shared__ float sigma[kWaves][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int group = blockIdx.x % a.G;
  const Segment seg = segment_of<WIDE ? 7 : 5>(a.starts, a.wide, a.n, a.T, a.R, blockIdx.x / a.G);
  const int rows = seg.len * a.R, tiles = (rows + kRows - 1) / kRows;
  if (seg.tile >= tiles) return;
  const int row0 = kRows * (tiles - 1 - seg.tile);
  const Keys keys = keys_of(a, seg.seq);
  const int behind = keys.len - seg.len;
  const int w0 = row0 + (WIDE ? 32 * wave : 0), ri = min(w0 + col, rows - 1), tok = div_r(a, ri);
  const int sees = min(tok + 1 + behind, keys.len);
  const int most = min(div_r(a, min(row0 + kRows, rows) - 1) + 1 + behind, keys.len);
  const int wave_most = w0 < rows ? min(div_r(a, min(w0 + 32, rows) - 1) + 1 + behind, keys.len) : 0;
  const int least = min(div_r(a, min(w0, rows - 1)) + 1 + behind, keys.len);
  const char* kb = a.k + group * a.kh + keys.first * a.kt;
  const char* vb = a.v + group * a.vh + keys.first * a.vt;
  const int head = group * a.R + ri - tok * a.R;
  const char* qrow = a.q + (seg.first + tok) * a.qt + head * a.qh;
  const char* grow = g.g_out + (seg.first + tok) * g.gt + head * g.gh;
  char* mine = lds + (WIDE ? 0 : 4 * kBytes * wave);
  auto send = [&](int it, char* to) __attribute__((always_inline)) {
    constexpr int BY = WIDE ? kWaves : 1;
    const int from = it * kKeys, last = keys.len - 1 - from, n0 = WIDE ? wave : 0;
    St::template load_rows<kLoads, BY>(to, n0, kb + from * a.kt, (uint32_t)a.kt, last);
    St::template load_rows<kLoads, BY>(to + kBytes, n0, vb + from * a.vt, (uint32_t)a.vt, last);
  };
  const St st;
  const int stages = most > 0 ? (most + kKeys - 1) / kKeys : 0;
  const int from = WIDE ? 0 : wave, by = WIDE ? 1 : kWaves;
  short8v q[HD / 16], go[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) {
    q[i] = *(const short8v*)(qrow + 32 * i + 16 * half);
    go[i] = *(const short8v*)(grow + 32 * i + 16 * half);
  }
  const int64_t at = (int64_t)group * a.T * a.R + (int64_t)seg.first * a.R + ri;
  const float lse2 = g.lse2[at];
  float delta = g.delta[at];
  // use(p, dp, k, b): the weights of 32 keys (0 where not seen) and g_out . v, transposed,
  // and where block b of keys lies
  auto sweep = [&](auto&& use) __attribute__((always_inline)) {
    reads_done();
    if (WIDE) __builtin_amdgcn_s_barrier();  // of a sweep before
    asm volatile("" ::: "memory");
    if (from < stages) send(from, mine);
    wait_vmcnt_le<0>();  // q and the rest too: the compiler does not count the stages' loads
    int turn = 0;
    for (int it = from; it < stages; it += by, turn ^= 1) {
      if (WIDE) wait_vmcnt_le<0>();
      reads_done();
      if (WIDE) __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (it + by < stages) {
        send(it + by, mine + 2 * kBytes * (turn ^ 1));
        if (!WIDE) wait_vmcnt_le<2 * kLoads>();
      } else if (!WIDE) {
        wait_vmcnt_le<0>();
      }
      asm volatile("" ::: "memory");
      const int k0 = it * kKeys;
      if (k0 >= wave_most) continue;
      const char* k = mine + 2 * kBytes * turn;
      const char* v = k + kBytes;
#pragma unroll
      for (int b = 0; b < B; ++b) {
        f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          s = mma16<T>(st.rows(k, b, i), q[i], s);
          dp = mma16<T>(st.rows(v, b, i), go[i], dp);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lse2));
        if (k0 + kKeys > least) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (k0 + 32 * b + tile_row(r, half) >= sees) s[r] = dp[r] = 0.f;
        }
        use(s, dp, k, b);
      }
    }
  };
  // The lane's sum of p dp becomes the row's exact delta, which goes to memory too.
  auto exact = [&](float sum) __attribute__((always_inline)) {
    float other = sum;
    half_swap(sum, other);
    sum += other;
    if constexpr (!WIDE) {
      if (half == 0) sigma[wave][col] = sum;
      __syncthreads();
      sum = (sigma[0][col] + sigma[1][col]) + (sigma[2][col] + sigma[3][col]);
    }
    sum -= g.g_lse ? g.g_lse[(int64_t)(seg.first + tok) * a.H + head] : 0.f;
    if (half == 0 && w0 + col < rows && (WIDE || wave == 0)) g.delta[at] = sum;
    return sees <= 0 ? 0.f : sum;
  };
  constexpr bool kBeside = HD == 32;
  if (sees <= 0) delta = 0.f;  // a row without keys, whose weights are 0: g_lse may be anything
  if (!kBeside && most <= kExactKeys) {
    float sum = 0.f;
    sweep([&](const f32x16& p, const f32x16& dp, const char*, int) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sum = fmaf(p[r], dp[r], sum);
    });
    delta = exact(sum);
  }
  if (!kBeside && !dq) return;
  f32x16 acc[HD / 32];
#pragma unroll
  for (int d = 0; d < HD / 32; ++d) acc[d] = f32x16{};
  Unit<T, HD> unit;
  f32x16 mean = f32x16{};  // sum p k
  float sum = 0.f;
  sweep([&](const f32x16& p, const f32x16& dp, const char* k, int b) __attribute__((always_inline)) {
    f32x16 dz;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dz[r] = p[r] * (dp[r] - delta);
      if (kBeside) sum = fmaf(p[r], dp[r], sum);
    }
    unit.scale(dz, acc);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = dz[8 * i + e];
      const short8v w = round8<T>(x);
#pragma unroll
      for (int d = 0; d < HD / 32; ++d) acc[d] = mma16<T>(st.cols(k, 2 * b + i, d), w, acc[d]);
      if constexpr (kBeside) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p[8 * i + e] * kLiftP<T>;
        mean = mma16<T>(st.cols(k, 2 * b + i, 0), round8<T>(x), mean);
      }
    }
  });
  float f = g.scale * unit.inverse();
  if constexpr (kBeside) {
    const float off = (delta - exact(sum)) * (g.scale / kLiftP<T>);
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[0][r] = fmaf(mean[r], off, acc[0][r] * f);
    f = 1.f;
    if (!dq) return;
  }
  if constexpr (WIDE) {
    if (w0 + col >= rows) return;
    T* to = dq + ((int64_t)(seg.first + tok) * a.H + head) * HD;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        store4(to + 32 * d + tile_row(r, half),
               make_float4(acc[d][r] * f, acc[d][r + 1] * f, acc[d][r + 2] * f, acc[d][r + 3] * f));
  } else {
    reads_done();
    __syncthreads();  // the stages become the waves' sums
    Sums<HD, 1, kWaves>& sums = *(Sums<HD, 1, kWaves>*)lds;
    sums.put(0, wave, col, half, acc, f);
    __syncthreads();
    sums.write(32, [&](int t) -> T* {
      if (row0 + t >= rows) return nullptr;
      const int tk = div_r(a, row0 + t);
      return dq + ((int64_t)(seg.first + tk) * a.H + group * a.R + row0 + t - tk * a.R) * HD;
    });
  }
}

// dk and dv.  A workgroup of KW x RW waves has 32 KW keys, 32 a wave, and its rows in
// stages (8 KB of q and of g_out, or 32 rows) that RW sets of KW waves take in turn, each set
// with stages of its own, and join at the end.  us of the backward pass, bf16 (T tokens in
// n sequences of one length, H heads over G):
//   KW, RW                               2, 3     4, 2     2, 2     4, 1
//   heads of 128:  2,048, 4, 8, 8        47.1     51.1     48.5
//                  4,096, 1, 16 over 4   416      527      455
//                  16,384, 24, 16 over 4 346      322      361
//                  16,384, 16, 16, 16    465      416      474
//   of 64:         8,192, 8, 16, 16               132      129      128
//                  16,384, 1, 16, 16              1,958    1,976    1,920
//                  32,768, 16, 16 over 4          663      648      687
//                  16,384, 16, 16, 16             236      225      214
//   of 32:         16,384, 16, 8, 8               83.9     88.4     83.6
//                  65,536, 64, 16 over 4          452      466      459
//                  16,384, 16, 32, 32             258      297      244
// Heads of 128 take 2, 3: documents of unlike lengths are nearer to the calls with few
// tiles (24 of them 323 us for dk and dv, 356 with 4, 2), for the first keys of a long one
// with the heads that share them are the longest way through.  The others take 4, 1.
template <class T, int HD, int KW, int RW>
__global__ __launch_bounds__(64 * KW * RW) void packed_dkv16_kernel(const Packed a, const Grads g, T* __restrict__ dk,
                                                                   T* __restrict__ dv) {
  typedef Stage<HD> St;
  constexpr int kKeys = 32 * KW, W = KW * RW;
  constexpr int kBytes = KW == 1 ? 32 * St::kRow : 8192, kLoads = kBytes / 1024;
  constexpr int kRows = kBytes / St::kRow, NB = kRows / 32;
  static_assert(far_rows_fit(kRows, 2) && far_rows_fit(kKeys, 2), "32-bit places");
  // heads of 128 leave no registers for the wave's keys and values as operands: they
  // lie in LDS, behind the stages
  constexpr bool kHeld = HD < 128 || KW == 1;
  constexpr int kKV = kHeld ? 0 : kKeys * St::kRow;
  constexpr int kStages = 4 * kBytes * RW + 2 * kKV, kJoin = sizeof(Sums<HD, KW, RW>);
  // a stage: rows of q, then of g_out; each wave's own copy of the rows' lse2 and delta
  __shared__ __attribute__((aligned(1024))) char lds[kStages > kJoin ? kStages : kJoin];
  __shared__ __attribute__((aligned(16))) float row_stats[W][2 * kRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = wave % KW, rw = wave / KW;
  const int col = lane & 31, half = lane >> 5;
  const int group = blockIdx.x % a.G;
  const Segment seg = segment_of<KW == 1 ? 5 : KW == 2 ? 6 : 7>(a.key_starts, a.wide, a.n, a.S, 1, blockIdx.x / a.G);
  const int k0 = kKeys * seg.tile;
  if (k0 >= seg.len) return;
  const bool real = seg.seq >= 0 && seg.seq < a.n;
  const int len = real ? keys_of(a, seg.seq).len : 0;  // of the segment's keys those in use
  int first = 0, tokens = 0;
  if (real) {
    first = __builtin_amdgcn_readfirstlane(segment_start(a.starts, a.wide, a.n, a.T, seg.seq + 1));
    const int end = __builtin_amdgcn_readfirstlane(segment_start(a.starts, a.wide, a.n, a.T, seg.seq + 2));
    tokens = max(end - first, 0);
  }
  const int rows = tokens * a.R, behind = len - tokens;  // token j sees the keys below j + 1 + behind
  const int w0 = k0 + 32 * kw, key = w0 + col;
  f32x16 ak[HD / 32], av[HD / 32];
#pragma unroll
  for (int d = 0; d < HD / 32; ++d) ak[d] = av[d] = f32x16{};
  Unit<T, HD> unit;
  char* mine = lds + 4 * kBytes * rw;
  if (k0 < len && rows > 0) {
    const int held = min(key, len - 1);
    const char* krow = a.k + (seg.first + held) * a.kt + group * a.kh;
    const char* vrow = a.v + (seg.first + held) * a.vt + group * a.vh;
    const int64_t st0 = (int64_t)group * a.T * a.R + (int64_t)first * a.R;
    // the first row that sees the lane's key, the wave's first key and the workgroup's
    const int row_min = max(key - behind, 0) * a.R, wave_min = max(w0 - behind, 0) * a.R;
    const int all_see = max(min(w0 + 31, len - 1) - behind, 0) * a.R;  // from here on a row sees all keys of the wave
    const int stages = (rows + kRows - 1) / kRows, from = max(k0 - behind, 0) * a.R / kRows;
    uint32_t q_at[kLoads / KW], g_at[kLoads / KW];
#pragma unroll
    for (int i = 0; i < kLoads / KW; ++i) {
      const int row = St::load_row(kw + i * KW), tk = div_r(a, row), h = row - tk * a.R;
      q_at[i] = tk * (uint32_t)a.qt + h * (uint32_t)a.qh;
      g_at[i] = tk * (uint32_t)g.gt + h * (uint32_t)g.gh;
    }
    auto send = [&](int it, char* to) __attribute__((always_inline)) {
      // a stage is whole tokens where R divides 32: a lane's rows lie alike in every
      // one.  Else, and in the last stage, each row's token is looked for.
      constexpr int N = kLoads / KW;
      const bool alike = (a.R & (a.R - 1)) == 0 && a.R <= 32 && kRows * (it + 1) <= rows;
      const int t0 = div_r(a, kRows * it);
      const char* qb = a.q + (int64_t)(first + t0) * a.qt + group * a.R * a.qh;
      const char* gb = g.g_out + (int64_t)(first + t0) * g.gt + group * a.R * g.gh;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int n = kw + i * KW;
        uint32_t qat = q_at[i], gat = g_at[i];
        if (!alike) {
          const int row = min(kRows * it + St::load_row(n), rows - 1), tk = div_r(a, row), h = row - tk * a.R;
          qat = (uint32_t)(tk - t0) * (uint32_t)a.qt + h * (uint32_t)a.qh;
          gat = (uint32_t)(tk - t0) * (uint32_t)g.gt + h * (uint32_t)g.gh;
        }
        St::load(to, n, qb, qat);
        St::load(to + kBytes, n, gb, gat);
      }
    };
    // a stage's lse2, then its deltas, NB a lane; rows behind the last weigh nothing
    float next[NB];
    auto stat = [&](int it) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int e = lane + 64 * i, row = kRows * it + (e & (kRows - 1));
        const float x = (e >= kRows ? g.delta : g.lse2)[st0 + min(row, rows - 1)];
        next[i] = row < rows ? x : e >= kRows ? 0.f : INFINITY;
      }
    };
    const St st;
#pragma unroll
    for (int i = 0; i < NB; ++i) next[i] = 0.f;
    if (from + rw < stages) {
      send(from + rw, mine);
      stat(from + rw);
    }
    short8v k[HD / 16], v[HD / 16];
    char* kv = lds + 4 * kBytes * RW;
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        k[i] = *(const short8v*)(krow + 32 * i + 16 * half);
        v[i] = *(const short8v*)(vrow + 32 * i + 16 * half);
      }
    } else {
      if (rw < 2) {  // two sets of waves bring them
        St::template load_rows<kKV / 2048 / KW, 2 * KW>(kv, wave, a.k + (int64_t)(seg.first + k0) * a.kt + group * a.kh,
                                                        (uint32_t)a.kt, len - 1 - k0);
        St::template load_rows<kKV / 2048 / KW, 2 * KW>(
            kv + kKV, wave, a.v + (int64_t)(seg.first + k0) * a.vt + group * a.vh, (uint32_t)a.vt, len - 1 - k0);
      }
    }
    int turn = 0;
    for (int base = from; base < stages; base += RW, turn ^= 1) {
      const int it = base + rw;
      wait_vmcnt_le<0>();
      reads_done();
#pragma unroll
      for (int i = 0; i < NB; ++i) row_stats[wave][lane + 64 * i] = next[i];
      if (KW > 1) __builtin_amdgcn_s_barrier();  // every wave comes by here as often
      asm volatile("" ::: "memory");
      if (it + RW < stages) {
        send(it + RW, mine + 2 * kBytes * (turn ^ 1));
        stat(it + RW);
      }
      if (it >= stages) continue;
      const char* q = mine + 2 * kBytes * turn;
      const char* go = q + kBytes;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int r0 = kRows * it + 32 * b;
        if (r0 + 32 <= wave_min || r0 >= rows) continue;
        f32x16 s = f32x16{}, ds = f32x16{};
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          s = mma16<T>(st.rows(q, b, i), kHeld ? k[i] : st.rows(kv, kw, i), s);
          ds = mma16<T>(st.rows(go, b, i), kHeld ? v[i] : st.rows(kv + kKV, kw, i), ds);
        }
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const float4 z = *(const float4*)&row_stats[wave][32 * b + tile_row(r, half)];
          const float4 e = *(const float4*)&row_stats[wave][kRows + 32 * b + tile_row(r, half)];
          const float zs[4] = {z.x, z.y, z.z, z.w}, es[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[r + i] = __builtin_amdgcn_exp2f(fmaf(s[r + i], a.c, -zs[i]));
            ds[r + i] = s[r + i] * (ds[r + i] - es[i]);
          }
        }
        if (r0 < all_see) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (r0 + tile_row(r, half) < row_min) s[r] = ds[r] = 0.f;
        }
        unit.scale(ds, ak);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x[8], y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = s[8 * i + e] * kLiftP<T>;
            y[e] = ds[8 * i + e];
          }
          const short8v p = round8<T>(x), w = round8<T>(y);
#pragma unroll
          for (int d = 0; d < HD / 32; ++d) {
            av[d] = mma16<T>(st.cols(go, 2 * b + i, d), p, av[d]);
            ak[d] = mma16<T>(st.cols(q, 2 * b + i, d), w, ak[d]);
          }
        }
      }
    }
  }
  const float fk = g.scale * unit.inverse(), fv = 1.f / kLiftP<T>;
  const bool in = key < len;  // places not in use have gradients 0
  Sums<HD, KW, RW>& sums = *(Sums<HD, KW, RW>*)lds;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    T* to = which ? dv : dk;
    if (!to) continue;
    f32x16 (&x)[HD / 32] = which ? av : ak;
    if (!in) {
#pragma unroll
      for (int d = 0; d < HD / 32; ++d) x[d] = f32x16{};
    }
    reads_done();
    __syncthreads();  // the stages become the waves' sums
    sums.put(kw, rw, col, half, x, which ? fv : fk);
    __syncthreads();
    sums.write(kKeys, [&](int t) -> T* {
      return k0 + t < seg.len ? to + ((int64_t)(seg.first + k0 + t) * a.G + group) * HD : nullptr;
    });
  }
}

// --------------------------------------------------------------------- host
typedef mpl_packed_attention_args Args;

int element_size(int dtype) { return dtype == MPL_F32 ? 4 : 2; }

// What does not depend on the buffers.
int check_sizes(const Args* p, const char* what) {
  MPL_REQUIRE(p, MPL_EINVAL, "%s: null arguments", what);
  MPL_REQUIRE(p->dtype == MPL_F32 || p->dtype == MPL_F16 || p->dtype == MPL_BF16, MPL_EINVAL, "%s: dtype %d", what,
              p->dtype);
  MPL_REQUIRE(p->heads > 0 && p->groups > 0 && p->heads % p->groups == 0, MPL_EINVAL,
              "%s: %d heads for %d key heads", what, p->heads, p->groups);
  MPL_REQUIRE(p->head_dim == 32 || p->head_dim == 64 || p->head_dim == 128, MPL_EUNSUPPORTED,
              "%s: head_dim %d (32, 64 or 128)", what, p->head_dim);
  MPL_REQUIRE(p->tokens >= 0 && p->keys >= 0 && p->sequences >= 0, MPL_EINVAL,
              "%s: bad sizes tokens=%lld keys=%lld sequences=%lld", what, (long long)p->tokens, (long long)p->keys,
              (long long)p->sequences);
  MPL_REQUIRE(p->index_bytes == 4 || p->index_bytes == 8, MPL_EINVAL, "%s: index_bytes %d (4 or 8)", what,
              p->index_bytes);
  // rows are counted in 32 bits, and a grid's threads too
  constexpr int64_t kMost = (int64_t)1 << 30;
  MPL_REQUIRE(p->heads <= 65536 && p->tokens <= kMost && p->keys <= kMost && p->sequences <= kMost &&
                  p->tokens * (p->heads / p->groups) <= kMost &&
                  (p->tokens * (p->heads / p->groups) / 32 + p->sequences + 2) * p->groups < ((int64_t)1 << 24) &&
                  (p->keys / 32 + p->sequences + 2) * p->groups < ((int64_t)1 << 24) &&
                  p->tokens * p->heads * (p->head_dim / 4) < ((int64_t)1 << 32),
              MPL_EUNSUPPORTED, "%s: %lld tokens and %lld keys in %lld sequences of %d and %d heads are too many", what,
              (long long)p->tokens, (long long)p->keys, (long long)p->sequences, p->heads, p->groups);
  return MPL_OK;
}

// `shared`: of k and v, whose heads lie where they like.
int check_rows(const Args* p, const void* x, int64_t tok, int64_t head, bool shared, const char* name,
               const char* what) {
  const int64_t unit = 16 / element_size(p->dtype);
  MPL_REQUIRE(x, MPL_EINVAL, "%s: null %s", what, name);
  MPL_REQUIRE(((uintptr_t)x & 15) == 0 && tok >= 0 && head >= 0 && tok % unit == 0 && head % unit == 0, MPL_EINVAL,
              "%s: the rows of %s must be 16-byte aligned (token %lld, head %lld)", what, name, (long long)tok,
              (long long)head);
  // places within a stage of rows are 32-bit (far_rows_fit)
  const int64_t r = p->heads / p->groups;
  MPL_REQUIRE(tok <= kMostStride && (shared || (head <= kMostStride && head * (r < 32 ? 32 : r) <= 32 * kMostStride)),
              MPL_EUNSUPPORTED, "%s: the rows of %s lie too far apart (token %lld, head %lld)", what, name,
              (long long)tok, (long long)head);
  return MPL_OK;
}

int check_inputs(const Args* p, const char* what) {
  if (int rc = check_sizes(p, what)) return rc;
  MPL_REQUIRE(p->scale > 0.f && p->scale < INFINITY, MPL_EINVAL, "%s: scale must be positive and finite", what);
  MPL_REQUIRE(p->starts && p->key_starts, MPL_EINVAL, "%s: null starts", what);
  MPL_REQUIRE((((uintptr_t)p->starts | (uintptr_t)p->key_starts | (uintptr_t)p->key_lengths) & (p->index_bytes - 1)) == 0,
              MPL_EINVAL, "%s: starts must be aligned", what);
  if (p->tokens)
    if (int rc = check_rows(p, p->q, p->q_token, p->q_head, false, "q", what)) return rc;
  if (p->keys) {
    if (int rc = check_rows(p, p->k, p->k_token, p->k_head, true, "k", what)) return rc;
    if (int rc = check_rows(p, p->v, p->v_token, p->v_head, true, "v", what)) return rc;
  }
  return MPL_OK;
}

Packed device_args(const Args* p) {
  Packed a;
  const int64_t e = element_size(p->dtype);
  a.q = (const char*)p->q; a.k = (const char*)p->k; a.v = (const char*)p->v;
  a.qt = p->q_token * e; a.qh = p->q_head * e;
  a.kt = p->k_token * e; a.kh = p->k_head * e;
  a.vt = p->v_token * e; a.vh = p->v_head * e;
  a.starts = p->starts; a.key_starts = p->key_starts; a.key_lengths = p->key_lengths;
  a.n = (int)p->sequences;
  a.wide = p->index_bytes == 8;
  a.T = (int)p->tokens; a.S = (int)p->keys;
  a.H = p->heads; a.G = p->groups; a.R = p->heads / p->groups;
  a.shift = 0;
  while (((int64_t)1 << a.shift) < a.R) ++a.shift;
  a.magic = (uint32_t)((((uint64_t)1 << (31 + a.shift)) + a.R - 1) / a.R);
  a.c = p->scale * kLog2e;
  return a;
}

// Whether the 16-bit forward and dq take tiles of 128 rows: where there are enough of
// them, more of narrower heads, whose tiles are less work.  us, tiles of 32 / of 128 rows
// (bf16, forward; T tokens in n sequences, H heads over G):
//   heads of 128:  T 2,048 n 4 H 8 G 8 (128 tiles): 17.2 / 16.8;  4,096, 8 (256): 29.5 / 19.4;
//                  2,048, 1, 16 over 4 (256): 48.3 / 49.3;  16,384, 16, 16 over 4 (2,048): 267 / 109
//   of 64:         4,096, 8, 8, 8 (256): 15.2 / 14.2;  2,048, 1, 16 over 4 (256): 23.1 / 35.7;
//                  8,192, 8, 8, 8 (512): 31.9 / 29.0;  4,096, 16, 16 over 4 (512): 22.3 / 13.3
//   of 32:         8,192, 8, 8, 8 (512): 19.3 / 24.5;  8,192, 16, 16 over 4 (1,024): 22.9 / 17.3
bool wide_of(const Args* p) {
  const int64_t r = p->heads / p->groups;
  return p->dtype != MPL_F32 && p->tokens * r / kWideRows * p->groups >= 256 * (128 / p->head_dim);
}

// Whether dk and dv in 16 bits take tiles of more keys, which read the rows less often.
// us of the backward pass, tiles of 32 keys / of 64 (heads of 128) or 128:
//   heads of 128:  2,048, 4, 8, 8 (128 tiles of 128): 53.8 / 44.7;  4,096, 16, 16 over 4 (128): 124 / 112;
//                  2,048, 1, 16 over 4 (64): 189 / 206
//                  16,384, 24, 16 over 4 (512): 433 / 357
//   of 64:         4,096, 8, 8, 8 (256): 44.2 / 44.6;  8,192, 8, 8, 8 (512): 89.0 / 80.1;
//                  8,192, 64, 32 over 8 (512): 96.8 / 106;  8,192, 8, 16, 16 (1,024): 151 / 132;
//                  32,768, 16, 16 over 4 (1,024): 682 / 702;  65,536, 64, 16 over 4 (2,048): 834 / 786;
//                  dk and dv of 16,384, 1, 16, 16 (2,048): 1,353 / 1,129
//   of 32:         8,192, 8, 8, 8 (512): 51.3 / 54.4;  16,384, 16, 16 over 4 (512): 140 / 165;
//                  16,384, 1, 8, 8 (1,024): 708 / 684;  32,768, 16, 16 over 4 (1,024): 407 / 410;
//                  16,384, 1, 16, 16 (2,048): 1,327 / 1,194;  65,536, 64, 16 over 4 (2,048): 469 / 468;
//                  16,384, 16, 32, 32 (4,096): 294 / 252
//
// Heads of 128 have 384 threads a workgroup then: with more than some 11 million tiles
// (sequences times key heads) the grid's threads would pass 32 bits, where 256 do not.
bool wide_keys_of(const Args* p) {
  const int64_t tiles = p->keys / 128 * p->groups;
  if (p->head_dim == 128 && (p->keys / 64 + p->sequences + 2) * p->groups * 384 >= (int64_t)1 << 32) return false;
  return tiles >= (p->head_dim == 128 ? 128 : 1024);
}

// Parts of the keys: where the tiles of rows do not fill the chip and the keys of
// a sequence are many.  Only sums over the sequences are known here, of a cache its
// places and not how many are in use.  A part is worth its share of the join's launch and
// memory from some keys on; fp32's products take longer, and want more workgroups.  Of
// heads of 128 a CU holds one of them (128 KB of LDS), and some more than 256 take twice
// as long: there the tiles are counted from below (as for single tokens).  us by number of
// parts, single tokens of B streams over `cap` places each, all in use / a quarter of
// them; * what the rule takes:
//   fp32, B 1, 4 heads of 64, cap 256:        1: 8.7 / 6.3 *   2: 8.2 / 8.3
//     512:                                    1: 13.4 / 6.3    2: 10.7 / 8.3 *   4: 8.9 / 9.4
//     1,024:                                  1: 23.1 / 8.6    2: 15.7 / 8.6   4: 11.3 / 8.8 *   8: 10.4 / 10.9
//     2,048:                                  1: 42.1 / 13.4   4: 16.5 / 9.5   8: 12.7 / 10.5 *
//   fp32, 16, 32 over 8 of 128, cap 512:      1: 26.5 / 10.5   2: 22.3 / 13.9 *   4: 29.0 / 24.3
//     1,024:                                  1: 46.7 / 16.2   2: 32.5 / 16.7 *   3: 46.5 / 24.4   4: 39.2 / 24.8
//     4,096:                                  1: 170 / 47.0    2: 107 / 32.5 *   3: 130 / 47.0   4: 110 / 40.0
//   fp32, 4, 32 over 8 of 128, cap 4,096:     1: 166 / 45.6    4: 50.7 / 20.8   8: 35.9 / 18.8 *   16: 45.7 / 32.0
//   bf16, 1, 4 of 64, cap 512:                1: 5.9 / 4.2 *   2: 7.2 / 6.2
//     1,024:                                  1: 8.3 / 4.8    2: 8.0 / 6.2 *   4: 7.2 / 7.3
//     2,048:                                  1: 13.1 / 6.0   4: 9.1 / 7.2 *   8: 9.0 / 8.5
//   bf16, 1, 32 over 8 of 128, cap 4,096:     1: 31.0 / 10.8   4: 15.0 / 9.7   8: 13.9 / 11.1 *
//     32,768, all in use:                     1: 215    8: 38.1   16: 33.9 *  32: 47.6   64: 64.8
//   bf16, 16, 32 over 8 of 128, cap 4,096:    1: 44.3 / 15.2 *   2: 43.3 / 17.1   4: 47.1 / 20.9
// Caches that are full at their end gain more than those that are not lose: with fp32's
// 512 places and up to half of them in use one part would be up to 2 us shorter.
int splits_of(const Args* p) {
  const bool f32 = p->dtype == MPL_F32;
  const int64_t r = p->heads / p->groups, n = p->sequences ? p->sequences : 1;
  const int64_t full = p->tokens * r / 32, some = p->tokens < n ? p->tokens : n;
  const bool single = f32 && p->head_dim == 128;  // workgroup a CU
  const int64_t tiles = (single ? (full > some ? full : some) : full + some) * p->groups;
  const int64_t want = tiles ? (single ? 256 : f32 ? 512 : 128) / tiles : 1, most = p->keys / n / (f32 ? 256 : 512);
  const int64_t s = want < most ? want : most;
  return s < 1 ? 1 : s > 16 ? 16 : (int)s;
}

size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

size_t workspace_bytes(const Args* p, bool backward) {
  const size_t rows = (size_t)p->tokens * p->heads;
  if (backward) return 2 * round256(rows * 4);
  const int s = wide_of(p) ? 1 : splits_of(p);
  return s > 1 ? round256(s * rows * p->head_dim * 4) + round256(s * rows * 8) : 0;
}

template <class T, int HD>
void forward(const Args* p, void* out, float* lse, void* ws, hipStream_t s) {
  const Packed a = device_args(p);
  const int splits = splits_of(p);
  const size_t rows = (size_t)p->tokens * p->heads;
  float* part = (float*)ws;
  float2* stats = (float2*)((char*)ws + round256(splits * rows * HD * 4));
  const int64_t tiles = ((int64_t)a.T * a.R / 32 + a.n + 2) * a.G;
  if constexpr (sizeof(T) == 2) {
    if (wide_of(p)) {
      const int64_t wide = ((int64_t)a.T * a.R / kWideRows + a.n + 2) * a.G;
      packed_forward16_kernel<T, HD><<<(unsigned)wide, kThreads, 0, s>>>(a, (T*)out, lse);
      return;
    }
    packed_forward16_few_kernel<T, HD><<<dim3((unsigned)tiles, splits), kThreads, 0, s>>>(a, splits, (T*)out, lse, part,
                                                                                        stats);
  } else {
    packed_forward_kernel<HD><<<dim3((unsigned)tiles, splits), kThreads, 0, s>>>(a, splits, (T*)out, lse, part, stats);
  }
  if (splits > 1)
    packed_join_kernel<T, HD><<<(unsigned)cdiv(rows * (HD / 4), 256), 256, 0, s>>>(a, splits, part, stats, (T*)out, lse);
}

template <class T, int HD>
void backward(const Args* p, const void* g_out, int64_t gt, int64_t gh, const void* out, const float* lse,
              const float* g_lse, void* ws, void* dq, void* dk, void* dv, hipStream_t s) {
  const Packed a = device_args(p);
  const size_t rows = (size_t)p->tokens * p->heads;
  float* lse2 = (float*)ws;
  float* delta = (float*)((char*)ws + round256(rows * 4));
  const int64_t blocks = cdiv(rows * (HD / 4), 256);
  const int used = (int)(blocks < kDeltaBlocks ? blocks : kDeltaBlocks);
  const Grads g{(const char*)g_out, gt * (int64_t)sizeof(T), gh * (int64_t)sizeof(T), lse2, delta, g_lse, p->scale};
  if (rows)
    packed_delta_kernel<T, HD><<<used, 256, 0, s>>>(a, g.g_out, g.gt, g.gh, (const T*)out, lse, g_lse, lse2, delta);
  auto tiles = [&](int64_t x, int unit) { return (unsigned)((x / unit + a.n + 2) * a.G); };
  if constexpr (sizeof(T) == 2) {
    if (rows) {  // for delta, too
      if (wide_of(p)) packed_dq16_kernel<T, HD, true><<<tiles((int64_t)a.T * a.R, 128), kThreads, 0, s>>>(a, g, (T*)dq);
      else packed_dq16_kernel<T, HD, false><<<tiles((int64_t)a.T * a.R, 32), kThreads, 0, s>>>(a, g, (T*)dq);
    }
    if (a.S && (dk || dv)) {
      constexpr int KW = HD == 128 ? 2 : 4, RW = HD == 128 ? 3 : 1;
      if (wide_keys_of(p))
        packed_dkv16_kernel<T, HD, KW, RW><<<tiles(a.S, 32 * KW), 64 * KW * RW, 0, s>>>(a, g, (T*)dk, (T*)dv);
      else
        packed_dkv16_kernel<T, HD, 1, 4><<<tiles(a.S, 32), kThreads, 0, s>>>(a, g, (T*)dk, (T*)dv);
    }
  } else {
    if (rows && dq) packed_dq_kernel<HD><<<tiles((int64_t)a.T * a.R, 32), kThreads, 0, s>>>(a, g, (T*)dq);
    if (a.S && (dk || dv)) packed_dkv_kernel<HD><<<tiles(a.S, 32), kThreads, 0, s>>>(a, g, (T*)dk, (T*)dv);
  }
}

template <class F>
void with_types(const Args* p, F&& f) {
  auto width = [&](auto t) {
    if (p->head_dim == 32) f(t, std::integral_constant<int, 32>{});
    else if (p->head_dim == 64) f(t, std::integral_constant<int, 64>{});
    else f(t, std::integral_constant<int, 128>{});
  };
  if (p->dtype == MPL_F32) width(float{});
  else if (p->dtype == MPL_F16) width(_Float16{});
  else width(__bf16{});
}

}  // namespace
}  // namespace mpl

using namespace mpl;

extern "C" size_t mpl_packed_attention_workspace_bytes(const mpl_packed_attention_args* args, int backward) {
  clear_error();
  if (check_sizes(args, "mpl_packed_attention_workspace_bytes")) return 0;
  const size_t n = workspace_bytes(args, backward != 0);
  return n ? n : 256;
}

extern "C" int mpl_packed_attention(const mpl_packed_attention_args* args, void* workspace, size_t workspace_bytes_,
                                    void* out, float* lse, void* stream) {
  clear_error();
  if (int rc = check_inputs(args, "mpl_packed_attention")) return rc;
  if (!args->tokens) return MPL_OK;
  MPL_REQUIRE(out && ((uintptr_t)out & 15) == 0, MPL_EINVAL, "mpl_packed_attention: out must be 16-byte aligned");
  const size_t need = workspace_bytes(args, false);
  MPL_REQUIRE(!need || (workspace && ((uintptr_t)workspace & 255) == 0), MPL_EINVAL,
              "mpl_packed_attention: a 256-byte aligned workspace is needed");
  MPL_REQUIRE(workspace_bytes_ >= need, MPL_EWORKSPACE, "mpl_packed_attention: workspace of %zu bytes needed", need);
  with_types(args, [&](auto t, auto hd) {
    forward<decltype(t), decltype(hd)::value>(args, out, lse, workspace, (hipStream_t)stream);
  });
  return check_launch("mpl_packed_attention");
}

extern "C" int mpl_packed_attention_bwd(const mpl_packed_attention_args* args, const void* g_out, int64_t g_token,
                                        int64_t g_head, const void* out, const float* lse, const float* g_lse,
                                        void* workspace, size_t workspace_bytes_, void* dq, void* dk, void* dv,
                                        void* stream) {
  clear_error();
  if (int rc = check_inputs(args, "mpl_packed_attention_bwd")) return rc;
  MPL_REQUIRE(dq || dk || dv, MPL_EINVAL, "mpl_packed_attention_bwd: no gradient is asked for");
  MPL_REQUIRE((((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) == 0, MPL_EINVAL,
              "mpl_packed_attention_bwd: gradients must be 16-byte aligned");
  if (args->tokens) {
    if (int rc = check_rows(args, g_out, g_token, g_head, false, "g_out", "mpl_packed_attention_bwd")) return rc;
    MPL_REQUIRE(out && ((uintptr_t)out & 15) == 0 && lse, MPL_EINVAL,
                "mpl_packed_attention_bwd: out (16-byte aligned) and lse are needed");
    const size_t need = workspace_bytes(args, true);
    MPL_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, MPL_EINVAL,
                "mpl_packed_attention_bwd: a 256-byte aligned workspace is needed");
    MPL_REQUIRE(workspace_bytes_ >= need, MPL_EWORKSPACE, "mpl_packed_attention_bwd: workspace of %zu bytes needed", need);
  }
  with_types(args, [&](auto t, auto hd) {
    backward<decltype(t), decltype(hd)::value>(args, g_out, g_token, g_head, out, lse, g_lse, workspace, dq, dk, dv,
                                               (hipStream_t)stream);
  });
  return check_launch("mpl_packed_attention_bwd");
}
