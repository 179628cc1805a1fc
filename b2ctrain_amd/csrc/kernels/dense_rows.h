// How the operators of a few rows read theirs: pieces of sixteen bytes whatever their alignment, and what becomes of a row's end.
#pragma once
#include "dense.h"

namespace b2c {
namespace dev {

// N values of a row from i on; zeros beyond its last, at whose place the last is read: loads without conditions go out together, where one
// that waits for its condition holds up the next.
template <typename E, int N>
__device__ __forceinline__ vec<E, N> some(const E* row, int i, int count) {
  vec<E, N> v{};
  if (i + N <= count) {
    __builtin_memcpy(&v, row + i, sizeof(E) * N);
  } else {
#pragma unroll
    for (int j = 0; j < N; j++)
      v[j] = row[i + j < count ? i + j : count - 1];
#pragma unroll
    for (int j = 0; j < N; j++) v[j] = i + j < count ? v[j] : (E)0;
  }
  return v;
}

// Sixteen bytes moved down by n, zeros behind them.
__device__ __forceinline__ vec<uint32_t, 4> moved_down(vec<uint32_t, 4> v, int n) {
  uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
  if (n >= 8) lo = hi, hi = 0, n -= 8;
  if (n >= 8) lo = 0;
  else if (n > 0) lo = lo >> (8 * n) | hi << (64 - 8 * n), hi >>= 8 * n;
  return {(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// The eight 16-bit values from k on where a row of K >= 8 ends: its last sixteen bytes, moved to their place, and zeros behind them; no load
// waits for a condition.
template <typename T>
__device__ __forceinline__ vec<T, 8> end8(const T* row, int k, int K) {
  const int from = k < K - 8 ? k : K - 8;
  vec<uint32_t, 4> v;
  __builtin_memcpy(&v, row + from, 16);
  return __builtin_bit_cast(vec<T, 8>, moved_down(v, 2 * (k - from)));
}

// c + a.lo b.lo + a.hi b.hi of two 16-bit values each, in single precision.
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c, bf16) {
  using V = vec<bf16, 2>;
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, false);
}
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c, f16) {
  using V = vec<f16, 2>;
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, false);
}
// How far apart rows may lie that are addressed by 32 bits from a tile's first.
constexpr int64_t kFarRows = 1 << 25;

}  // namespace dev
}  // namespace b2c
