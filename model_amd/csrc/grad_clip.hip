// The global norm of many gradients, and the gradients scaled in place
// (train.py:395-399, optax.global_norm and the clip, over every dense gradient of a
// model beside the sparse rows):
//
//   norm = sqrt(sum_t sum x^2 + sum row_sq),  scale = min(1, clip / (norm + 1e-6)),
//   x = x scale.
//
// Two passes over the tensors' tiles: sums of squares in fp64 by workgroup, and the
// scaling, each workgroup of which joins the same sums in the same order first, and
// ends at once where scale is 1.  The tensors' places come as kernel arguments; more
// than kTable of them are written to the workspace by small launches of kTable each
// before, so nothing is copied from the host and a captured call keeps its table.
//
// A workgroup has neighbouring tiles, so that it looks for a tensor once; the scaling
// goes from the end on, where what was read last may still lie in the last-level
// cache.  Bound: memory; of small sets the two launches' latency, of a thousand tensors
// the host (65 ns each).  Measured: 1.2 G elements (bf16 matrices, fp32 vectors, 2.4 GB
// read twice and written) 1,540 us, sums 513 to 521 and the scaling 1,017, against 1,497 at
// a large copy's 4.85 TB/s; where the scale is 1 the scaling ends at once, and the call
// takes 522; 32 fp32 tensors of 6.3 MB 9 to 11 us, kernels 5.3 + 3.2;
// 1,500 fp16 tensors of 65 MB below the clip 118 us, of which 39 on the GPU (eight lists
// of 1.7, sums 21, the end 4).  A launch of each kernel for every 192 tensors instead
// of the list took 218 us, a third launch for the norm 15.4 where two take 10.
#include <math.h>

#include "common.h"

namespace mpl {
namespace {

constexpr int kTable = 192;   // 3.9 KB of arguments
constexpr int kTile = 4096;   // elements
constexpr int kThreads = 256;
constexpr int kSum = 3;       // a tensor of squares (fp32): summed, not scaled
constexpr int kMostBlocks = 1024;

struct Entries {
  void* x[kTable];
  int64_t n[kTable];           // elements; the type in the upper 8 bits
  uint32_t first[kTable + 1];  // tiles before the tensor
};
static_assert(sizeof(Entries) <= 3960, "kernel arguments are 4 KB");

// The table in the workspace.
struct Listed {
  void** x;
  int64_t* n;
  uint32_t* first;
};

__device__ __forceinline__ float from16(uint32_t u, int type) {
  if (type == MPL_BF16) return __uint_as_float(u << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}
__device__ __forceinline__ uint32_t to16(float x, int type) {
  if (type == MPL_BF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
  return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// The last tensor that begins no later than a tile, 64 of them a step.
template <class Tab>
__device__ __forceinline__ int tensor_of(const Tab& t, int count, uint32_t tile) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = count;
  while (len > 1) {
    const int step = (len + 63) >> 6, i = lo + min(lane * step, len - 1);
    const int before = 63 - __clzll((long long)(__ballot(lane * step < len && t.first[i] <= tile) | 1));
    lo += before * step;
    len = min(step, len - before * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The tiles [from, to) of a workgroup, in turn (or, BACK, from the last on):
// use(tensor, elements before the tile, elements of it).
template <bool BACK, class Tab, class F>
__device__ __forceinline__ void walk(const Tab& t, int count, F&& use) {
  const uint32_t tiles = t.first[count], per = (tiles + gridDim.x - 1) / gridDim.x;
  const uint32_t block = BACK ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const uint32_t from = min(block * per, tiles), to = min(from + per, tiles);
  if (from == to) return;
  int i = tensor_of(t, count, BACK ? to - 1 : from);
  for (uint32_t k = from; k < to; ++k) {
    const uint32_t tile = BACK ? to - 1 - (k - from) : k;
    if (BACK) {
      while (t.first[i] > tile) --i;
    } else {
      while (t.first[i + 1] <= tile) ++i;
    }
    const int64_t n = t.n[i] & (((int64_t)1 << 56) - 1), before = (int64_t)(tile - t.first[i]) * kTile;
    use(t.x[i], (int)(t.n[i] >> 56), before, (int)min(n - before, (int64_t)kTile));
  }
}

// m elements from x on, E of them 16 bytes: the whole 16 bytes among them by vec(place),
// up to 1,024 of them, and those before and behind one by one.
template <class T, class V, class S>
__device__ __forceinline__ void pieces(T* x, int m, V&& vec, S&& single) {
  constexpr int E = 16 / sizeof(T);
  const int head = min((int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T), m);
  const int whole = (m - head) / E, tail = m - head - whole * E;
  vec((uint4*)(x + head), whole);
  if ((int)threadIdx.x < head) single(x + threadIdx.x);
  if ((int)threadIdx.x < tail) single(x + head + whole * E + threadIdx.x);
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

template <class Tab>
__global__ __launch_bounds__(kThreads) void grad_sums_kernel(const Tab t, int count, double* __restrict__ sums) {
  __shared__ double lds[kThreads / 64];
  double s = 0;
  walk<false>(t, count, [&](void* p, int type, int64_t before, int m) __attribute__((always_inline)) {
    if (type == MPL_F32 || type == kSum) {
      auto add = [&](float x) __attribute__((always_inline)) {
        if (type == kSum) s += (double)x;
        else add_square(s, x);
      };
      pieces((float*)p + before, m, [&](const uint4* x, int n) __attribute__((always_inline)) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int at = k * kThreads + threadIdx.x;
          v[k] = at < n ? x[at] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          add(__uint_as_float(v[k].x)); add(__uint_as_float(v[k].y));
          add(__uint_as_float(v[k].z)); add(__uint_as_float(v[k].w));
        }
      }, [&](const float* x) __attribute__((always_inline)) { add(*x); });
    } else {
      pieces((uint16_t*)p + before, m, [&](const uint4* x, int n) __attribute__((always_inline)) {
        uint4 v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = k * kThreads + threadIdx.x;
          v[k] = at < n ? x[at] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            add_square(s, from16(u[e] & 0xffff, type));
            add_square(s, from16(u[e] >> 16, type));
          }
        }
      }, [&](const uint16_t* x) __attribute__((always_inline)) { add_square(s, from16(*x, type)); });
    }
  });
  s = block_sum(s, lds);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// [scale, norm] from the sums, in one order wherever it is done.
__device__ __forceinline__ float2 scale_and_norm(const double* sums, int count, float clip, double* lds) {
  double s = 0;
  for (int i = threadIdx.x; i < count; i += kThreads) s += sums[i];
  s = block_sum(s, lds);
  const float norm = (float)sqrt(s), f = clip / (norm + 1e-6f);
  return make_float2(f > 1.f ? 1.f : f, norm);  // NaN stays
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const double* __restrict__ sums, int count, float clip,
                                                             float* __restrict__ scale_norm) {
  __shared__ double lds[kThreads / 64];
  const float2 r = scale_and_norm(sums, count, clip, lds);
  if (threadIdx.x == 0) {
    scale_norm[0] = r.x;
    scale_norm[1] = r.y;
  }
}

template <class Tab>
__global__ __launch_bounds__(kThreads) void grad_scale_kernel(const Tab t, int count, const double* __restrict__ sums,
                                                              int blocks, float clip, float* __restrict__ scale_norm) {
  __shared__ double lds[kThreads / 64];
  const float2 r = scale_and_norm(sums, blocks, clip, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    scale_norm[0] = r.x;
    scale_norm[1] = r.y;
  }
  const float f = r.x;
  if (f == 1.f) return;
  walk<true>(t, count, [&](void* p, int type, int64_t before, int m) __attribute__((always_inline)) {
    if (type == kSum) return;
    if (type == MPL_F32) {
      pieces((float*)p + before, m, [&](uint4* to, int n) __attribute__((always_inline)) {
        float4* x = (float4*)to;
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int at = k * kThreads + threadIdx.x;
          if (at < n) v[k] = x[at];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int at = k * kThreads + threadIdx.x;
          if (at < n) x[at] = make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f);
        }
      }, [&](float* x) __attribute__((always_inline)) { *x *= f; });
    } else {
      pieces((uint16_t*)p + before, m, [&](uint4* x, int n) __attribute__((always_inline)) {
        uint4 v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = k * kThreads + threadIdx.x;
          if (at < n) v[k] = x[at];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = k * kThreads + threadIdx.x;
          uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            u[e] = to16(from16(u[e] & 0xffff, type) * f, type) | to16(from16(u[e] >> 16, type) * f, type) << 16;
          if (at < n) x[at] = make_uint4(u[0], u[1], u[2], u[3]);
        }
      }, [&](uint16_t* x) __attribute__((always_inline)) { *x = (uint16_t)to16(from16(*x, type) * f, type); });
    }
  });
}

// Entries [at, at + count) of the table in the workspace, and the end behind them.
__global__ __launch_bounds__(kThreads) void grad_list_kernel(const Entries e, int count, Listed to, int64_t at) {
  const int i = threadIdx.x;
  if (i < count) {
    to.x[at + i] = e.x[i];
    to.n[at + i] = e.n[i];
  }
  if (i <= count) to.first[at + i] = e.first[i];
}

// The tensors in groups of kTable: f(entries, their number, entries before them).
template <class F>
void groups(void* const* x, const int64_t* n, const int* dtype, int64_t count, const float* row_sq, int64_t rows, F&& f) {
  Entries e;
  int used = 0;
  int64_t before = 0;
  e.first[0] = 0;
  auto add = [&](void* p, int64_t m, int type) {
    if (used == kTable) {
      f(e, used, before);
      before += used;
      e.first[0] = e.first[used];
      used = 0;
    }
    e.x[used] = p;
    e.n[used] = m | (int64_t)type << 56;
    e.first[used + 1] = e.first[used] + (uint32_t)cdiv(m, kTile);
    ++used;
  };
  if (rows) add((void*)row_sq, rows, kSum);
  for (int64_t i = 0; i < count; ++i)
    if (n[i]) add(x[i], n[i], dtype[i]);
  if (used) f(e, used, before);
}

constexpr size_t kSumBytes = kMostBlocks * sizeof(double);
int64_t list_places(int64_t count) { return (count + 1 + 31) / 32 * 32 + 32; }  // and the end

}  // namespace
}  // namespace mpl

using namespace mpl;

extern "C" size_t mpl_clip_grads_workspace_bytes(int64_t count) {
  if (count < 0 || count > (1 << 24)) return 0;
  return kSumBytes + (count + 1 > kTable ? (size_t)list_places(count) * 20 : 0);
}

extern "C" int mpl_clip_grads(void* const* x, const int64_t* n, const int* dtype, int64_t count, const float* row_sq,
                              int64_t rows, float grad_clip, int apply, float* scale_gnorm, void* workspace,
                              size_t workspace_bytes, void* stream) {
  clear_error();
  MPL_REQUIRE(count >= 0 && count <= (1 << 24) && rows >= 0, MPL_EINVAL, "mpl_clip_grads: bad sizes count=%lld rows=%lld",
              (long long)count, (long long)rows);
  MPL_REQUIRE((!count || (x && n && dtype)) && (!rows || row_sq) && scale_gnorm, MPL_EINVAL, "mpl_clip_grads: null buffer");
  MPL_REQUIRE(((uintptr_t)row_sq & 3) == 0, MPL_EINVAL, "mpl_clip_grads: row_sq must be aligned");
  constexpr int64_t kMost = (int64_t)1 << 40;  // elements in all
  int64_t tiles = cdiv(rows <= kMost ? rows : 0, kTile), all = rows, entries = rows ? 1 : 0;
  for (int64_t i = 0; i < count; ++i) {
    MPL_REQUIRE(dtype[i] == MPL_F32 || dtype[i] == MPL_F16 || dtype[i] == MPL_BF16, MPL_EINVAL,
                "mpl_clip_grads: tensor %lld: dtype %d", (long long)i, dtype[i]);
    MPL_REQUIRE(n[i] >= 0 && (!n[i] || x[i]), MPL_EINVAL, "mpl_clip_grads: tensor %lld: bad size or null", (long long)i);
    MPL_REQUIRE(((uintptr_t)x[i] & (dtype[i] == MPL_F32 ? 3 : 1)) == 0, MPL_EINVAL,
                "mpl_clip_grads: tensor %lld must be aligned to its elements", (long long)i);
    MPL_REQUIRE(all <= kMost && n[i] <= kMost, MPL_EUNSUPPORTED, "mpl_clip_grads: too many elements");
    all += n[i];
    tiles += cdiv(n[i], kTile);
    entries += n[i] ? 1 : 0;
  }
  MPL_REQUIRE(all <= kMost, MPL_EUNSUPPORTED, "mpl_clip_grads: too many elements");
  MPL_REQUIRE(workspace && ((uintptr_t)workspace & 7) == 0, MPL_EINVAL,
              "mpl_clip_grads: an 8-byte aligned workspace is needed");
  const size_t need = mpl_clip_grads_workspace_bytes(count);
  MPL_REQUIRE(workspace_bytes >= need, MPL_EWORKSPACE, "mpl_clip_grads: workspace of %zu bytes needed", need);
  hipStream_t s = (hipStream_t)stream;
  double* sums = (double*)workspace;
  const int blocks = (int)(tiles < kMostBlocks ? tiles : kMostBlocks);
  auto run = [&](const auto& table) {
    if (blocks) grad_sums_kernel<<<blocks, kThreads, 0, s>>>(table, (int)entries, sums);
    if (apply && blocks)
      grad_scale_kernel<<<blocks, kThreads, 0, s>>>(table, (int)entries, sums, blocks, grad_clip, scale_gnorm);
    else
      grad_norm_kernel<<<1, kThreads, 0, s>>>(sums, blocks, grad_clip, scale_gnorm);
  };
  if (entries <= kTable) {
    Entries only;
    only.first[0] = 0;
    groups(x, n, dtype, count, row_sq, rows, [&](const Entries& e, int, int64_t) { only = e; });
    run(only);
  } else {
    const int64_t places = list_places(count);
    char* at = (char*)workspace + kSumBytes;
    const Listed list{(void**)at, (int64_t*)(at + 8 * places), (uint32_t*)(at + 16 * places)};
    groups(x, n, dtype, count, row_sq, rows, [&](const Entries& e, int used, int64_t before) {
      grad_list_kernel<<<1, kThreads, 0, s>>>(e, used, list, before);
    });
    run(list);
  }
  return check_launch("mpl_clip_grads");
}
