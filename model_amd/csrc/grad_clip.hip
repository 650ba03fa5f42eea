// The global norm of many gradients, and the gradients scaled in place
// (train.py:395-399, optax.global_norm and the clip, over every dense gradient of a
// model beside the sparse rows):
//
//   norm = sqrt(sum_t sum x^2 + sum row_sq),  scale = min(1, clip / (norm + 1e-6)),
//   x = x scale.
//
// Three passes: sums of squares in fp64 by workgroups over the tensors' tiles, one
// workgroup that joins them in a fixed order, and the scaling, which ends at once
// where scale is 1.  The tensors' places come as kernel arguments, kTable of them a
// launch: nothing is copied to the device, and a captured call keeps its table.
//
// Bound: memory.
#include <math.h>

#include "common.h"

namespace mpl {
namespace {

constexpr int kTable = 192;   // 3.9 KB of arguments
constexpr int kTile = 4096;   // elements
constexpr int kThreads = 256;
constexpr int kSum = 3;       // a tensor of squares (fp32): summed, not scaled
constexpr int kMostBlocks = 1024;

struct Table {
  void* x[kTable];
  int64_t n[kTable];         // elements; the type in the upper 8 bits
  uint32_t first[kTable + 1];  // tiles before the tensor
  int count;
  int blocks;  // workgroups of the launch
};
static_assert(sizeof(Table) <= 3960, "kernel arguments are 4 KB");

__device__ __forceinline__ float from16(uint32_t u, int type) {
  if (type == MPL_BF16) return __uint_as_float(u << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}
__device__ __forceinline__ uint32_t to16(float x, int type) {
  if (type == MPL_BF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
  return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// The tensor that a tile lies in.
__device__ __forceinline__ int tensor_of(const Table& t, uint32_t tile) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= tile) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double s, double* lds) {
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  const int waves = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  double all = 0;
  for (int w = 0; w < waves; ++w) all += lds[w];
  return all;
}

__device__ __forceinline__ void add_square(double& s, float x) { s = fma((double)x, (double)x, s); }

__global__ __launch_bounds__(kThreads) void grad_sums_kernel(const Table t, double* __restrict__ sums) {
  __shared__ double lds[kThreads / 64];
  const uint32_t tiles = t.first[t.count];
  double s = 0;
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int i = tensor_of(t, tile);
    const int type = (int)(t.n[i] >> 56);
    const int64_t n = t.n[i] & (((int64_t)1 << 56) - 1), from = (int64_t)(tile - t.first[i]) * kTile;
    const int m = (int)min(n - from, (int64_t)kTile);
    if (type == MPL_F32 || type == kSum) {
      const float* x = (const float*)t.x[i] + from;
      if (m == kTile && ((uintptr_t)x & 15) == 0) {
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ((const float4*)x)[k * kThreads + threadIdx.x];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (type == kSum) {
            s += (double)v[k].x + (double)v[k].y + (double)v[k].z + (double)v[k].w;
          } else {
            add_square(s, v[k].x); add_square(s, v[k].y); add_square(s, v[k].z); add_square(s, v[k].w);
          }
        }
      } else {
        for (int k = threadIdx.x; k < m; k += kThreads) {
          if (type == kSum) s += (double)x[k];
          else add_square(s, x[k]);
        }
      }
    } else {
      const uint16_t* x = (const uint16_t*)t.x[i] + from;
      if (m == kTile && ((uintptr_t)x & 15) == 0) {
        uint4 v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) v[k] = ((const uint4*)x)[k * kThreads + threadIdx.x];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            add_square(s, from16(u[e] & 0xffff, type));
            add_square(s, from16(u[e] >> 16, type));
          }
        }
      } else {
        for (int k = threadIdx.x; k < m; k += kThreads) add_square(s, from16(x[k], type));
      }
    }
  }
  s = block_sum(s, lds);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void grad_norm_kernel(const double* __restrict__ sums, int count, float clip,
                                                         float* __restrict__ scale_norm) {
  __shared__ double lds[16];
  double s = 0;
  for (int i = threadIdx.x; i < count; i += 1024) s += sums[i];
  s = block_sum(s, lds);
  if (threadIdx.x == 0) {
    const float norm = (float)sqrt(s), f = clip / (norm + 1e-6f);
    scale_norm[0] = f > 1.f ? 1.f : f;  // NaN stays
    scale_norm[1] = norm;
  }
}

__global__ __launch_bounds__(kThreads) void grad_scale_kernel(const Table t, const float* __restrict__ scale_norm) {
  const float f = scale_norm[0];
  if (f == 1.f) return;
  const uint32_t tiles = t.first[t.count];
  // from the end on: what the sums read last may still lie in the last-level cache
  for (uint32_t at = blockIdx.x; at < tiles; at += gridDim.x) {
    const uint32_t tile = tiles - 1 - at;
    const int i = tensor_of(t, tile);
    const int type = (int)(t.n[i] >> 56);
    if (type == kSum) continue;
    const int64_t n = t.n[i] & (((int64_t)1 << 56) - 1), from = (int64_t)(tile - t.first[i]) * kTile;
    const int m = (int)min(n - from, (int64_t)kTile);
    if (type == MPL_F32) {
      float* x = (float*)t.x[i] + from;
      if (m == kTile && ((uintptr_t)x & 15) == 0) {
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ((const float4*)x)[k * kThreads + threadIdx.x];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          ((float4*)x)[k * kThreads + threadIdx.x] = make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f);
      } else {
        for (int k = threadIdx.x; k < m; k += kThreads) x[k] *= f;
      }
    } else {
      uint16_t* x = (uint16_t*)t.x[i] + from;
      if (m == kTile && ((uintptr_t)x & 15) == 0) {
        uint4 v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) v[k] = ((const uint4*)x)[k * kThreads + threadIdx.x];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            u[e] = to16(from16(u[e] & 0xffff, type) * f, type) | to16(from16(u[e] >> 16, type) * f, type) << 16;
          ((uint4*)x)[k * kThreads + threadIdx.x] = make_uint4(u[0], u[1], u[2], u[3]);
        }
      } else {
        for (int k = threadIdx.x; k < m; k += kThreads) x[k] = (uint16_t)to16(from16(x[k], type) * f, type);
      }
    }
  }
}

// The launches' tables, from the tensors in turn; f(table).
template <class F>
void tables(void* const* x, const int64_t* n, const int* dtype, int64_t count, const float* row_sq, int64_t rows, F&& f) {
  Table t;
  t.count = 0;
  t.first[0] = 0;
  auto flush = [&] {
    if (!t.count) return;
    const uint32_t tiles = t.first[t.count];
    t.blocks = tiles < (uint32_t)kMostBlocks ? (int)tiles : kMostBlocks;
    f(t);
    t.count = 0;
  };
  auto add = [&](void* p, int64_t m, int type) {
    // tiles are counted in 32 bits: a launch of its own where they would not fit
    const int64_t tiles = cdiv(m, kTile);
    if (t.count == kTable || (int64_t)t.first[t.count] + tiles > 0x7fffffff) flush();
    t.x[t.count] = p;
    t.n[t.count] = m | (int64_t)type << 56;
    t.first[t.count + 1] = t.first[t.count] + (uint32_t)tiles;
    ++t.count;
  };
  if (rows) add((void*)row_sq, rows, kSum);
  for (int64_t i = 0; i < count; ++i)
    if (n[i]) add(x[i], n[i], dtype[i]);
  flush();
}

}  // namespace
}  // namespace mpl

using namespace mpl;

extern "C" size_t mpl_clip_grads_workspace_bytes(int64_t count) {
  // a launch for each table's worth of tensors and row_sq
  return count < 0 || count > (1 << 24) ? 0 : (size_t)(cdiv(count + 1, kTable) + 1) * kMostBlocks * sizeof(double);
}

extern "C" int mpl_clip_grads(void* const* x, const int64_t* n, const int* dtype, int64_t count, const float* row_sq,
                              int64_t rows, float grad_clip, int apply, float* scale_gnorm, void* workspace,
                              size_t workspace_bytes, void* stream) {
  clear_error();
  MPL_REQUIRE(count >= 0 && count <= (1 << 24) && rows >= 0, MPL_EINVAL, "mpl_clip_grads: bad sizes count=%lld rows=%lld",
              (long long)count, (long long)rows);
  MPL_REQUIRE((!count || (x && n && dtype)) && (!rows || row_sq) && scale_gnorm, MPL_EINVAL, "mpl_clip_grads: null buffer");
  MPL_REQUIRE(((uintptr_t)row_sq & 3) == 0, MPL_EINVAL, "mpl_clip_grads: row_sq must be aligned");
  constexpr int64_t kMost = (int64_t)1 << 40;  // elements of a tensor
  MPL_REQUIRE(rows <= kMost, MPL_EUNSUPPORTED, "mpl_clip_grads: %lld rows", (long long)rows);
  for (int64_t i = 0; i < count; ++i) {
    MPL_REQUIRE(dtype[i] == MPL_F32 || dtype[i] == MPL_F16 || dtype[i] == MPL_BF16, MPL_EINVAL,
                "mpl_clip_grads: tensor %lld: dtype %d", (long long)i, dtype[i]);
    MPL_REQUIRE(n[i] >= 0 && n[i] <= kMost && (!n[i] || x[i]), MPL_EINVAL, "mpl_clip_grads: tensor %lld: bad size or null",
                (long long)i);
    MPL_REQUIRE(((uintptr_t)x[i] & (dtype[i] == MPL_F32 ? 3 : 1)) == 0, MPL_EINVAL,
                "mpl_clip_grads: tensor %lld must be aligned to its elements", (long long)i);
  }
  int64_t sums = 0;
  tables(x, n, dtype, count, row_sq, rows, [&](const Table& t) { sums += t.blocks; });
  MPL_REQUIRE(!sums || (workspace && ((uintptr_t)workspace & 7) == 0), MPL_EINVAL,
              "mpl_clip_grads: an 8-byte aligned workspace is needed");
  MPL_REQUIRE(workspace_bytes >= sums * sizeof(double), MPL_EWORKSPACE, "mpl_clip_grads: workspace of %zu bytes needed",
              (size_t)sums * sizeof(double));
  hipStream_t s = (hipStream_t)stream;
  double* to = (double*)workspace;
  tables(x, n, dtype, count, row_sq, rows, [&](const Table& t) {
    grad_sums_kernel<<<t.blocks, kThreads, 0, s>>>(t, to);
    to += t.blocks;
  });
  grad_norm_kernel<<<1, 1024, 0, s>>>((const double*)workspace, (int)sums, grad_clip, scale_gnorm);
  if (apply)
    tables(x, n, dtype, count, nullptr, 0, [&](const Table& t) {
      grad_scale_kernel<<<t.blocks, kThreads, 0, s>>>(t, scale_gnorm);
    });
  return check_launch("mpl_clip_grads");
}
