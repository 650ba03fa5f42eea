// What the kernels of the attention over packed sequences share: the arguments
// as the device sees them, which sequence a workgroup's tile lies in, and where
// its rows are.
//
// Rows.  The R = heads / groups query heads that share a key head are rows of one
// matrix: row t R + r of a group is head r of token t.  A tile of rows then reads
// its keys and values once for all of them, and a single new token is R rows.
//
// Tiles.  A sequence of `len` tokens from token `first` has len R rows, from row
// first R, and at most floor(end R / BM) - floor(first R / BM) + 1 tiles of BM
// rows.  So tile id b belongs to the last sequence i with
// floor(first_i R / BM) + i <= b: the grid's size follows from the number of tokens
// and of sequences alone, without the lengths, which only the device knows.  The
// tokens before the first sequence and behind the last are two more segments,
// without keys.
#pragma once

#include "common.h"

namespace mpl {

typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));

struct Packed {
  const char *q, *k, *v;
  int64_t qt, qh, kt, kh, vt, vh;  // bytes from token to token and from head to head
  const void *starts, *key_starts, *key_lengths;
  int n, wide;  // sequences; 64-bit places
  int T, S, H, G, R;
  uint32_t magic, shift;  // x / R = umulhi(2 x, magic) >> shift for x < 2^31
  float c;                // scale log2(e)
};

__device__ __forceinline__ int div_r(const Packed& a, int x) { return __umulhi(2u * x, a.magic) >> a.shift; }

__device__ __forceinline__ int64_t place_at(const void* p, int wide, int i) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int*)p)[i];
}

// The first token of segment i in 0 .. n + 2, held to [0, total].
__device__ __forceinline__ int segment_start(const void* starts, int wide, int n, int total, int i) {
  const int64_t v = place_at(starts, wide, min(max(i - 1, 0), n));
  const int held = (int)min(max(v, (int64_t)0), (int64_t)total);
  return i <= 0 ? 0 : i >= n + 2 ? total : held;
}

struct Segment {
  int seq;         // -1 and n: tokens of no sequence
  int first, len;  // tokens (keys)
  int tile;        // the id's tile of the segment, >= 0; it may lie behind the segment's end
};

// The segment of tile id b, for tiles of 2^LOG rows and `per` rows a token.  Every
// lane of the wave calls it.  64 segments a step, of which the last that begins no
// later than b is kept (the first one does), so that tile >= 0 whatever the starts:
// such as do not ascend give some segment within the arrays.
template <int LOG>
__device__ __forceinline__ Segment segment_of(const void* starts, int wide, int n, int total, int per, int b) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = n + 2, first, end;
  do {
    const int step = (len + 63) >> 6, i = lo + lane * step;
    const int begins = segment_start(starts, wide, n, total, i);
    const int64_t at = ((int64_t)begins * per >> LOG) + i;
    const int before = 63 - __clzll((long long)(__ballot(lane * step < len && at <= b) | 1));
    lo += before * step;
    len = min(step, len - before * step);
    // a step of neighbouring segments: the lanes hold where they begin
    first = __shfl(begins, before);
    end = step == 1 && before < 63 ? __shfl(begins, before + 1) : segment_start(starts, wide, n, total, lo + 1);
  } while (len > 1);
  Segment s;
  s.seq = __builtin_amdgcn_readfirstlane(lo - 1);
  s.first = __builtin_amdgcn_readfirstlane(first);
  s.len = __builtin_amdgcn_readfirstlane(max(end - first, 0));
  s.tile = __builtin_amdgcn_readfirstlane(max(b - (int)(((int64_t)first * per >> LOG) + lo), 0));
  return s;
}

// The keys of sequence seq: the first of them and their number.
struct Keys {
  int first, len;
};
__device__ __forceinline__ Keys keys_of(const Packed& a, int seq) {
  if (seq < 0 || seq >= a.n) return {0, 0};
  const int first = segment_start(a.key_starts, a.wide, a.n, a.S, seq + 1);
  int len = max(segment_start(a.key_starts, a.wide, a.n, a.S, seq + 2) - first, 0);
  if (a.key_lengths) len = (int)min(max(place_at(a.key_lengths, a.wide, seq), (int64_t)0), (int64_t)len);
  return {__builtin_amdgcn_readfirstlane(first), __builtin_amdgcn_readfirstlane(len)};
}

// Loads of one to four neighbouring elements as fp32.
__device__ __forceinline__ float4 load4(const float* p) { return *(const float4*)p; }
__device__ __forceinline__ float4 load4(const _Float16* p) {
  typedef _Float16 half4v __attribute__((ext_vector_type(4)));
  const half4v x = *(const half4v*)p;
  return make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
}
__device__ __forceinline__ float4 load4(const __bf16* p) {
  const uint2 u = *(const uint2*)p;
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(float* p, float4 x) { *(float4*)p = x; }
__device__ __forceinline__ void store4(_Float16* p, float4 x) {
  typedef _Float16 half4v __attribute__((ext_vector_type(4)));
  *(half4v*)p = half4v{(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
}
__device__ __forceinline__ void store4(__bf16* p, float4 x) {
  typedef __bf16 bhalf4v __attribute__((ext_vector_type(4)));
  *(bhalf4v*)p = bhalf4v{(__bf16)x.x, (__bf16)x.y, (__bf16)x.z, (__bf16)x.w};
}

constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.442695040888963407f;

}  // namespace mpl
