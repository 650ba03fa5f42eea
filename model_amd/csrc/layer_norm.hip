// LayerNorm of rows and its backward pass (model.py:86-125, nn.LayerNorm), with
// the residual add before it:
//
//   s = x + r (rounded to the rows' type),  x_hat = (s - mean) rstd,
//   y = x_hat scale + bias,  rstd = 1 / sqrt(mean((s - mean)^2) + eps)
//
//   dx = rstd (g - mean(g) - x_hat mean(g x_hat)) + g_s,  g = dy scale
//   d scale = sum_rows dy x_hat,   d bias = sum_rows dy
//
// A row stays in the registers of a team of lanes from its one read to its one
// write: up to 64 lanes of a wave (as few as the row has 16-byte vectors, so
// narrow rows share a wave), or a workgroup for rows of more than 256 vectors.
// The variance is of the centred values, so it does not cancel.  Teams walk the
// rows; in the backward each lane sums d scale and d bias of its own columns in
// registers on the way, a workgroup writes one partial row of each, and a
// second launch adds the partial rows in a fixed order: no atomics, and the
// same bits in every call.
//
// Rows of any width and alignment are read by 16-byte vectors (gfx950 takes
// them unaligned); the last vector of a ragged row is read from its end and the
// elements that it shares with the one before are masked out of the sums.
//
// Bound: memory.  16,384 x 4,096 bf16 with the residual: forward 4 arrays in 88 us
// (6.1 TB/s; a large copy 5.1), backward 4 arrays and 512 partial rows in 120 us
// (4.5 TB/s) and 4.7 for the second launch.  Small calls: 64 x 256 fp32 3.4 us,
// 8,192 x 256 5.9, and 7.5 and 2.9; 4,001 x 1,283 fp16 with the residual 12.5, and
// 18.8 and 4.9.  Few wide rows leave CUs idle: 300 x 16,384 12.6, and 22.9 and 6.1
// (3.1 and 2.6 TB/s).  512 workgroups of the backward are two a CU; 768 or 1,024 were
// slower (87 and 96 us for 69 at 4,096 x 8,192 bf16): a CU's share is uneven and the
// partial rows more.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "topk.h"

namespace mpl {
namespace {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Row;
template <>
struct Row<float> {
  static constexpr int VE = 4;
  __device__ static void widen(u32x4 u, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  }
  __device__ static u32x4 narrow(const float (&v)[4]) {
    u32x4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(v[i]);
    return u;
  }
};
template <>
struct Row<_Float16> {
  static constexpr int VE = 8;
  __device__ static void widen(u32x4 u, float (&v)[8]) {
    const half8 h = __builtin_bit_cast(half8, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
  }
  __device__ static u32x4 narrow(const float (&v)[8]) {
    half8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)v[i];
    return __builtin_bit_cast(u32x4, h);
  }
};
template <>
struct Row<__bf16> {
  static constexpr int VE = 8;
  typedef __bf16 b8 __attribute__((ext_vector_type(8)));
  __device__ static void widen(u32x4 u, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
  __device__ static u32x4 narrow(const float (&v)[8]) {
    b8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (__bf16)v[i];
    return __builtin_bit_cast(u32x4, h);
  }
};

// The place of a lane's vector in a row of d elements: `off`, and which of its
// elements count (bits): all, or those that the vector before does not hold.
template <int VE>
struct Place {
  int off;
  uint32_t mask;
  __device__ __forceinline__ Place(int vec, int d) {
    const int at = vec * VE;
    off = max(min(at, d - VE), 0);
    const int skip = at - off;
    mask = at >= d ? 0u : d < VE ? (1u << d) - 1 : ((1u << VE) - 1) & ~((1u << skip) - 1);
    if (at >= d) off = 0;
  }
};

// SMALL: the row may have not one whole vector, d < VE.
template <bool SMALL, typename T>
__device__ __forceinline__ void load_vec(const T* row, int off, int d, float (&v)[Row<T>::VE]) {
  constexpr int VE = Row<T>::VE;
  if (!SMALL || d >= VE) {
    Row<T>::widen((u32x4)(*(const u32x4_any*)(row + off)), v);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = (float)row[min(e, d - 1)];
  }
}
template <bool SMALL, typename T>
__device__ __forceinline__ void store_vec(T* row, int off, int d, const float (&v)[Row<T>::VE]) {
  constexpr int VE = Row<T>::VE;
  if (!SMALL || d >= VE) {
    *(u32x4_any*)(row + off) = Row<T>::narrow(v);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (e < d) row[e] = (T)v[e];
  }
}
// A vector's worth of a parameter, fp32 or of the rows' type.
template <bool SMALL, typename T>
__device__ __forceinline__ void load_param(const void* p, bool f32, int off, int d, float (&v)[Row<T>::VE]) {
  constexpr int VE = Row<T>::VE;
  if (!f32) {
    load_vec<SMALL>((const T*)p, off, d, v);
  } else if (!SMALL || d >= VE) {
#pragma unroll
    for (int i = 0; i < VE / 4; ++i) {
      float u[4];
      load_vec<false>((const float*)p, off + 4 * i, 4, u);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * i + e] = u[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = ((const float*)p)[min(e, d - 1)];
  }
}

template <int S>
__device__ __forceinline__ float add_xor(float v, int lane) {
  return v + __uint_as_float(w64::xr<S>(__float_as_uint(v), lane));
}

// Sums of N values over a team.  TL = 64: `width` lanes of a wave; else the
// workgroup, through `s`, whose two halves alternate so that one barrier a sum
// is enough.
template <int TL, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], int width, int lane, int wave, float (*s)[TL / 64][N],
                                         int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (TL > 64 || width > 1) v[i] = add_xor<1>(v[i], lane);
    if (TL > 64 || width > 2) v[i] = add_xor<2>(v[i], lane);
    if (TL > 64 || width > 4) v[i] = add_xor<4>(v[i], lane);
    if (TL > 64 || width > 8) v[i] = add_xor<8>(v[i], lane);
    if (TL > 64 || width > 16) v[i] = add_xor<16>(v[i], lane);
    if (TL > 64 || width > 32) v[i] = add_xor<32>(v[i], lane);
  }
  if constexpr (TL > 64) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[turn][wave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = s[turn][0][i];
#pragma unroll
      for (int w = 1; w < TL / 64; ++w) t += s[turn][w][i];
      v[i] = t;
    }
    turn ^= 1;
  }
}

struct LnArgs {
  const void* x;
  int64_t x_pitch;
  const void* r;
  int64_t r_pitch;
  const void* scale;
  const void* bias;
  int param_f32;
  int64_t rows;
  int d, width;
  float eps;
  void* y;
  void* s;
  float* mean;
  float* rstd;
  // backward: x is the normalised rows' input, r the gradient that joins dx
  const void* dy;
  int64_t dy_pitch;
  void* dx;
  float* part;  // [workgroups][2][d]
};

// Threads of a workgroup whose teams have TL lanes, and how a lane finds its
// team: its index, the lane's place in it and the number of teams.
template <int TL>
constexpr int ln_threads() { return TL > 256 ? TL : 256; }

template <int TL>
struct Team {
  int lane, wave, at, width;
  int64_t id, count;
  __device__ __forceinline__ Team(int w) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (TL == 64) {
      width = w;
      at = lane & (w - 1);
      const int per = 256 / w;  // teams of a workgroup
      id = (int64_t)blockIdx.x * per + threadIdx.x / w;
      count = (int64_t)gridDim.x * per;
    } else {
      width = TL;
      at = threadIdx.x;
      id = blockIdx.x;
      count = gridDim.x;
    }
  }
};

// MASK: the lanes' vectors do not fill the row exactly.
template <typename T, int TL, int NV, int NR, bool MASK>
__global__ __launch_bounds__(ln_threads<TL>()) void ln_fwd_kernel(LnArgs p) {
  constexpr int VE = Row<T>::VE;
  constexpr bool SMALL = MASK && TL == 64 && NV == 1;
  __shared__ float red[2][TL / 64][NR];
  const Team<TL> t(p.width);
  const int d = p.d;
  int turn = 0;
  int off[NV];
  uint32_t mask[NV];
  float g[NV][VE], b[NV][VE];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Place<VE> at(t.at + i * t.width, d);
    off[i] = at.off, mask[i] = at.mask;
    load_param<SMALL, T>(p.scale, p.param_f32, off[i], d, g[i]);
    load_param<SMALL, T>(p.bias, p.param_f32, off[i], d, b[i]);
  }
  const float inv = 1.f / (float)d;
  // teams of one wave run as many turns as its first: the waves of a workgroup
  // need no barrier with each other then, and a workgroup has one team
  const int64_t first = TL == 64 ? t.id - t.lane / t.width : t.id;
  for (int64_t at = 0; (first + at) * NR < p.rows; at += t.count) {
    float v[NR][NV][VE], m[NR], q[NR];
    int64_t row[NR];
    bool live[NR];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      row[k] = (t.id + at) * NR + k;
      live[k] = row[k] < p.rows;
      row[k] = min(row[k], p.rows - 1);
#pragma unroll
      for (int i = 0; i < NV; ++i) load_vec<SMALL>((const T*)p.x + row[k] * p.x_pitch, off[i], d, v[k][i]);
    }
    if (p.r) {
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        float r[NV][VE];
#pragma unroll
        for (int i = 0; i < NV; ++i) load_vec<SMALL>((const T*)p.r + row[k] * p.r_pitch, off[i], d, r[i]);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
          for (int e = 0; e < VE; ++e) v[k][i][e] = v[k][i][e] + r[i][e];
          Row<T>::widen(Row<T>::narrow(v[k][i]), v[k][i]);  // the norm is that of the rounded sum
          if (p.s && live[k] && (!MASK || mask[i])) store_vec<SMALL>((T*)p.s + row[k] * d, off[i], d, v[k][i]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      m[k] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) m[k] += !MASK || (mask[i] >> e & 1) ? v[k][i][e] : 0.f;
    }
    team_sum<TL, NR>(m, t.width, t.lane, t.wave, red, turn);
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      m[k] *= inv;
      q[k] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          v[k][i][e] -= m[k];
          q[k] = fmaf(!MASK || (mask[i] >> e & 1) ? v[k][i][e] : 0.f, v[k][i][e], q[k]);
        }
    }
    team_sum<TL, NR>(q, t.width, t.lane, t.wave, red, turn);
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const float rstd = 1.f / sqrtf(fmaf(q[k], inv, p.eps));
      if (!live[k]) continue;
      if (p.mean && t.at == 0) {
        p.mean[row[k]] = m[k];
        p.rstd[row[k]] = rstd;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float y[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) y[e] = fmaf(v[k][i][e] * rstd, g[i][e], b[i][e]);
        if (!MASK || mask[i]) store_vec<SMALL>((T*)p.y + row[k] * d, off[i], d, y);
      }
    }
  }
}

template <typename T, int TL, int NV, int NR, bool MASK>
__global__ __launch_bounds__(ln_threads<TL>()) void ln_bwd_kernel(LnArgs p) {
  constexpr int VE = Row<T>::VE;
  constexpr bool SMALL = MASK && TL == 64 && NV == 1;
  __shared__ float red[2][TL / 64][2 * NR];
  const Team<TL> t(p.width);
  const int d = p.d;
  int turn = 0;
  int off[NV];
  uint32_t mask[NV];
  // the widest workgroups read their scale again for each row: registers
  constexpr bool HOLD = TL < 1024 || NV * VE < 16;
  float g[NV][VE], ds[NV][VE], db[NV][VE];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Place<VE> at(t.at + i * t.width, d);
    off[i] = at.off, mask[i] = at.mask;
    if (HOLD) load_param<SMALL, T>(p.scale, p.param_f32, off[i], d, g[i]);
#pragma unroll
    for (int e = 0; e < VE; ++e) ds[i][e] = db[i][e] = 0.f;
  }
  const float inv = 1.f / (float)d;
  const int64_t first = TL == 64 ? t.id - t.lane / t.width : t.id;
  // a workgroup of 256 has its next row on the way while it sums this one (wider
  // ones have no registers for it: 69 -> 77 us at 4,096 x 8,192 bf16)
  constexpr bool AHEAD = TL == 256;
  u32x4 nx[AHEAD ? NV : 1], ny[AHEAD ? NV : 1];
  auto send = [&](int64_t r) __attribute__((always_inline)) {
    r = min(r, p.rows - 1);
#pragma unroll
    for (int i = 0; i < (AHEAD ? NV : 0); ++i) {
      nx[i] = (u32x4)(*(const u32x4_any*)((const T*)p.x + r * p.x_pitch + off[i]));
      ny[i] = (u32x4)(*(const u32x4_any*)((const T*)p.dy + r * p.dy_pitch + off[i]));
    }
  };
  if (AHEAD) send(t.id);
  for (int64_t at = 0; (first + at) * NR < p.rows; at += t.count) {
    float x[NR][NV][VE], y[NR][NV][VE], sums[2 * NR], rstd[NR];
    int64_t row[NR];
    bool live[NR];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      row[k] = (t.id + at) * NR + k;
      live[k] = row[k] < p.rows;
      row[k] = min(row[k], p.rows - 1);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (AHEAD) {
          Row<T>::widen(nx[i], x[k][i]);
          Row<T>::widen(ny[i], y[k][i]);
        } else {
          load_vec<SMALL>((const T*)p.x + row[k] * p.x_pitch, off[i], d, x[k][i]);
          load_vec<SMALL>((const T*)p.dy + row[k] * p.dy_pitch, off[i], d, y[k][i]);
        }
      }
    }
    if (AHEAD) send(t.id + at + t.count);
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const float m = p.mean[row[k]];
      rstd[k] = p.rstd[row[k]];
      float a = 0.f, c = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!HOLD) load_param<SMALL, T>(p.scale, p.param_f32, off[i], d, g[i]);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const bool on = !MASK || (mask[i] >> e & 1);
          const float hat = (x[k][i][e] - m) * rstd[k], dy = y[k][i][e], gy = dy * g[i][e];
          if (live[k] && on) {
            ds[i][e] = fmaf(dy, hat, ds[i][e]);
            db[i][e] += dy;
          }
          a += on ? gy : 0.f;
          c = fmaf(on ? gy : 0.f, hat, c);
          x[k][i][e] = hat;
          y[k][i][e] = gy;
        }
      }
      sums[2 * k] = a, sums[2 * k + 1] = c;
    }
    team_sum<TL, 2 * NR>(sums, t.width, t.lane, t.wave, red, turn);
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      if (!live[k] || !p.dx) continue;
      const float a = sums[2 * k] * inv, c = sums[2 * k + 1] * inv;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (MASK && !mask[i]) continue;
        float o[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) o[e] = rstd[k] * (y[k][i][e] - a - x[k][i][e] * c);
        if (p.r) {
          float u[VE];
          load_vec<SMALL>((const T*)p.r + row[k] * p.r_pitch, off[i], d, u);
#pragma unroll
          for (int e = 0; e < VE; ++e) o[e] += u[e];
        }
        store_vec<SMALL>((T*)p.dx + row[k] * d, off[i], d, o);
      }
    }
  }
  if (!p.part) return;
  // one partial row of each sum from the workgroup
  float* out = p.part + (int64_t)blockIdx.x * 2 * d;
  if constexpr (TL > 64) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (!MASK || (mask[i] >> e & 1)) {
          out[off[i] + e] = ds[i][e];
          out[d + off[i] + e] = db[i][e];
        }
  } else {
    // teams of a wave by exchanges, waves through LDS
    __shared__ float s[4][2][NV * 64 * VE];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        float u = ds[i][e], w = db[i][e];
#define MPL_JOIN(W) \
  if (t.width <= W) u = add_xor<W>(u, t.lane), w = add_xor<W>(w, t.lane);
        MPL_JOIN(32) MPL_JOIN(16) MPL_JOIN(8) MPL_JOIN(4) MPL_JOIN(2) MPL_JOIN(1)
#undef MPL_JOIN
        s[t.wave][0][(i * 64 + t.lane) * VE + e] = u;
        s[t.wave][1][(i * 64 + t.lane) * VE + e] = w;
      }
    __syncthreads();
    // thread -> (which sum, vector, element): the vector's place as its lanes had it
    for (int n = threadIdx.x; n < 2 * NV * t.width * VE; n += 256) {
      const int e = n % VE, l = n / VE % t.width, i = n / (VE * t.width) % NV, which = n / (VE * t.width * NV);
      const Place<VE> at(l + i * t.width, d);
      if (!(at.mask >> e & 1)) continue;
      float u = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) u += s[w][which][(i * 64 + l) * VE + e];
      out[which * d + at.off + e] = u;
    }
  }
}

// d scale and d bias from the partial rows: 32 columns a workgroup, 32 threads
// a column, each every 32nd partial row in order, then the 32 in order.
__global__ __launch_bounds__(1024) void ln_params_kernel(const float* __restrict__ part, int groups, int d, int f32,
                                                        int bf16, void* __restrict__ d_scale,
                                                        void* __restrict__ d_bias) {
  __shared__ float s[32][33];
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c;
  const int which = blockIdx.y;
  float sum = 0.f;
  if (col < d) {
    int g = k;
    for (; g + 7 * 32 < groups; g += 8 * 32) {  // 8 loads in flight
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = part[((int64_t)(g + 32 * i) * 2 + which) * d + col];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += v[i];
    }
    for (; g < groups; g += 32) sum += part[((int64_t)g * 2 + which) * d + col];
  }
  s[k][c] = sum;
  __syncthreads();
  if (k || col >= d) return;
  float out = 0.f;
#pragma unroll
  for (int g = 0; g < 32; ++g) out += s[g][c];
  void* q = which ? d_bias : d_scale;
  if (q == nullptr) return;
  if (f32) ((float*)q)[col] = out;
  else if (bf16) ((__bf16*)q)[col] = (__bf16)out;
  else ((_Float16*)q)[col] = (_Float16)out;
}

// --------------------------------------------------------------------- host
constexpr int kMaxWidth = 16384;

inline int elems(int dtype) { return dtype == MPL_F32 ? 4 : 8; }
inline int64_t vecs_of(int d, int dtype) { return cdiv(d, elems(dtype)); }

// Lanes of a team for rows of `vecs` vectors; from d alone, so that a row's
// result does not depend on the others of its call.
inline int width_of(int64_t vecs) {
  int w = 1;
  while (w < 64 && w < vecs) w *= 2;
  return w;
}

// Workgroups of the backward: as many as fill the card, but each sums at least
// 4 rows a team before it writes its partial rows.
int64_t bwd_groups(int64_t rows, int d, int dtype) {
  const int64_t vecs = vecs_of(d, dtype);
  const bool wave = vecs <= (dtype == MPL_F32 ? 256 : 192);  // a team is at most a wave
  const int64_t teams = wave ? 256 / width_of(vecs) : 1;
  return std::max<int64_t>(1, std::min<int64_t>(512, cdiv(rows, teams * (vecs <= 64 ? 4 : 2))));
}

template <typename T, bool BWD>
void launch(const LnArgs& p, int64_t groups, hipStream_t s) {
  constexpr int VE = Row<T>::VE;
  const int64_t vecs = cdiv(p.d, VE);
#define MPL_LN(TL, NV, NR)                                                                                           \
  do {                                                                                                               \
    const int64_t per = (TL == 64 ? 256 / p.width : 1) * (int64_t)(NR);                                              \
    const unsigned grid = (unsigned)(BWD ? groups : std::min<int64_t>(cdiv(p.rows, per), 4096));                     \
    const bool exact = p.d == (int64_t)VE * (NV) * (TL == 64 ? p.width : TL);                                        \
    if (BWD) {                                                                                                       \
      if (exact) ln_bwd_kernel<T, TL, NV, NR, false><<<grid, ln_threads<TL>(), 0, s>>>(p);                           \
      else ln_bwd_kernel<T, TL, NV, NR, true><<<grid, ln_threads<TL>(), 0, s>>>(p);                                  \
    } else {                                                                                                         \
      if (exact) ln_fwd_kernel<T, TL, NV, NR, false><<<grid, ln_threads<TL>(), 0, s>>>(p);                           \
      else ln_fwd_kernel<T, TL, NV, NR, true><<<grid, ln_threads<TL>(), 0, s>>>(p);                                  \
    }                                                                                                                \
  } while (0)
  if (vecs <= 64) MPL_LN(64, 1, (BWD ? 4 : 2));
  else if (vecs <= 128) MPL_LN(64, 2, (BWD ? 2 : 1));
  else if constexpr (VE == 4) {
    if (vecs <= 256) MPL_LN(64, 4, 1);
    else if (vecs <= 512) MPL_LN(256, 2, 1);
    else if (vecs <= 1024) MPL_LN(256, 4, 1);
    else if (vecs <= 2048) MPL_LN(512, 4, 1);
    else MPL_LN(1024, 4, 1);
  } else {
    if (vecs <= 192) MPL_LN(64, 3, 1);
    else if (vecs <= 256) MPL_LN(256, 1, 1);
    else if (vecs <= 512) MPL_LN(256, 2, 1);
    else if (vecs <= 1024) MPL_LN(512, 2, 1);
    else MPL_LN(1024, 2, 1);
  }
#undef MPL_LN
}

template <bool BWD>
void launch_of(int dtype, const LnArgs& p, int64_t groups, hipStream_t s) {
  if (dtype == MPL_F32) launch<float, BWD>(p, groups, s);
  else if (dtype == MPL_F16) launch<_Float16, BWD>(p, groups, s);
  else launch<__bf16, BWD>(p, groups, s);
}

int check(const char* what, int64_t rows, int d, int dtype, int param_dtype) {
  MPL_REQUIRE(rows >= 0 && d > 0, MPL_EINVAL, "%s: bad sizes rows=%lld d=%d", what, (long long)rows, d);
  MPL_REQUIRE(dtype == MPL_F32 || dtype == MPL_F16 || dtype == MPL_BF16, MPL_EINVAL, "%s: bad dtype %d", what, dtype);
  MPL_REQUIRE(param_dtype == MPL_F32 || param_dtype == dtype, MPL_EINVAL,
              "%s: parameters are fp32 or of the rows' type, got %d for %d", what, param_dtype, dtype);
  MPL_REQUIRE(d <= kMaxWidth, MPL_EUNSUPPORTED, "%s: d = %d above %d", what, d, kMaxWidth);
  return MPL_OK;
}

bool aligned_to(const void* q, int dtype) { return ((uintptr_t)q & (dtype == MPL_F32 ? 3 : 1)) == 0; }

}  // namespace
}  // namespace mpl

using namespace mpl;

extern "C" int mpl_layer_norm(const void* x, int64_t x_pitch, const void* residual, int64_t residual_pitch, int dtype,
                              const void* scale, const void* bias, int param_dtype, int64_t rows, int d, float eps,
                              void* y, void* sum, float* mean, float* rstd, void* stream) {
  clear_error();
  const char* what = "mpl_layer_norm";
  if (const int rc = check(what, rows, d, dtype, param_dtype)) return rc;
  if (rows == 0) return MPL_OK;
  MPL_REQUIRE(x && scale && bias && y && (mean == nullptr) == (rstd == nullptr), MPL_EINVAL, "%s: null buffer", what);
  MPL_REQUIRE(x_pitch >= d && (!residual || residual_pitch >= d), MPL_EINVAL, "%s: a pitch is below d = %d", what, d);
  MPL_REQUIRE(residual || !sum, MPL_EINVAL, "%s: sum without residual", what);
  for (const void* q : {x, residual, (const void*)y, (const void*)sum})
    MPL_REQUIRE(aligned_to(q, dtype), MPL_EINVAL, "%s: an array is not aligned to its elements", what);
  for (const void* q : {scale, bias})
    MPL_REQUIRE(aligned_to(q, param_dtype), MPL_EINVAL, "%s: a parameter is not aligned to its elements", what);
  LnArgs p{};
  p.x = x, p.x_pitch = x_pitch, p.r = residual, p.r_pitch = residual_pitch;
  p.scale = scale, p.bias = bias, p.param_f32 = param_dtype == MPL_F32;
  p.rows = rows, p.d = d, p.width = width_of(vecs_of(d, dtype)), p.eps = eps;
  p.y = y, p.s = sum, p.mean = mean, p.rstd = rstd;
  launch_of<false>(dtype, p, 0, (hipStream_t)stream);
  return check_launch(what);
}

extern "C" size_t mpl_layer_norm_bwd_workspace_bytes(int64_t rows, int d, int dtype) {
  if (rows <= 0 || d <= 0 || (dtype != MPL_F32 && dtype != MPL_F16 && dtype != MPL_BF16) ||
      d > kMaxWidth)
    return 0;
  return (size_t)bwd_groups(rows, d, dtype) * 2 * d * sizeof(float);
}

extern "C" int mpl_layer_norm_bwd(const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch,
                                  const void* g_residual, int64_t g_residual_pitch, int dtype, const void* scale,
                                  int param_dtype, const float* mean, const float* rstd, int64_t rows, int d, void* dx,
                                  void* d_scale, void* d_bias, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* what = "mpl_layer_norm_bwd";
  if (const int rc = check(what, rows, d, dtype, param_dtype)) return rc;
  MPL_REQUIRE(rows > 0, MPL_EINVAL, "%s: no rows", what);
  MPL_REQUIRE(dy && x && scale && mean && rstd && (dx || d_scale || d_bias), MPL_EINVAL, "%s: null buffer", what);
  MPL_REQUIRE(x_pitch >= d && dy_pitch >= d && (!g_residual || g_residual_pitch >= d), MPL_EINVAL,
              "%s: a pitch is below d = %d", what, d);
  for (const void* q : {dy, x, g_residual, (const void*)dx})
    MPL_REQUIRE(aligned_to(q, dtype), MPL_EINVAL, "%s: an array is not aligned to its elements", what);
  for (const void* q : {scale, (const void*)d_scale, (const void*)d_bias})
    MPL_REQUIRE(aligned_to(q, param_dtype), MPL_EINVAL, "%s: a parameter is not aligned to its elements", what);
  const bool params = d_scale || d_bias;
  const size_t need = params ? mpl_layer_norm_bwd_workspace_bytes(rows, d, dtype) : 0;
  MPL_REQUIRE(!params || (workspace && ((uintptr_t)workspace & 3) == 0), MPL_EINVAL, "%s: no workspace", what);
  MPL_REQUIRE(workspace_bytes >= need, MPL_EWORKSPACE, "%s: workspace %zu < %zu bytes", what, workspace_bytes, need);
  LnArgs p{};
  p.x = x, p.x_pitch = x_pitch, p.r = g_residual, p.r_pitch = g_residual_pitch;
  p.scale = scale, p.param_f32 = param_dtype == MPL_F32;
  p.rows = rows, p.d = d, p.width = width_of(vecs_of(d, dtype));
  p.mean = (float*)mean, p.rstd = (float*)rstd;
  p.dy = dy, p.dy_pitch = dy_pitch, p.dx = dx;
  p.part = params ? (float*)workspace : nullptr;
  hipStream_t s = (hipStream_t)stream;
  const int64_t groups = bwd_groups(rows, d, dtype);
  launch_of<true>(dtype, p, groups, s);
  if (params)
    ln_params_kernel<<<dim3((unsigned)cdiv(d, 32), 2), 1024, 0, s>>>(p.part, (int)groups, d, param_dtype == MPL_F32,
                                                                    param_dtype == MPL_BF16, d_scale, d_bias);
  return check_launch(what);
}
