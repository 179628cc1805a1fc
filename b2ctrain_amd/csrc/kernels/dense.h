// What the dense operators' kernels share: element types, vector loads and stores, the activations, and the
// epilogues that finish a tile of a matrix product.
//
// Every product is out[m][n] = sum_k Q[m][k] P[n][k]. A matrix instruction is issued with P as its first
// operand, so that a lane's accumulators lie along n, the direction in which out is contiguous: it stores
// several neighbouring values at once.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <algorithm>
#include <type_traits>

#include "b2c_kernels.h"
#include "philox.h"

namespace b2c {
namespace dev {

using bf16 = __bf16;
using f16 = _Float16;
template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));
using f32x4 = vec<float, 4>;
using i32x4 = vec<int, 4>;

// 16x16 tiles: 32 values of k a step in 16 bits, 64 in 8 bits; lane l gives row l % 16, sixteen bytes of k at
// 16 (l / 16); accumulator r of lane l is row (l / 16) 4 + r of P, row l % 16 of Q.
__device__ __forceinline__ f32x4 mfma(vec<bf16, 8> p, vec<bf16, 8> q, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, q, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(vec<f16, 8> p, vec<f16, 8> q, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(p, q, c, 0, 0, 0);
}
__device__ __forceinline__ i32x4 mfma(vec<int8_t, 16> p, vec<int8_t, 16> q, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, p), __builtin_bit_cast(i32x4, q), c, 0, 0, 0);
}

template <typename T>
struct Elem {  // sixteen bytes of T, and the accumulator of its products
  static constexpr int N = 16 / sizeof(T);
  using Acc = f32x4;
};
template <>
struct Elem<int8_t> {
  static constexpr int N = 16;
  using Acc = i32x4;
};

// The normal distribution function in `cdf` and e^(-g^2 / 2) in `bell`. erfc by M. Abramowitz and I. Stegun, Handbook of
// Mathematical Functions, 7.1.26 (off by at most 1.5e-7), taken at -|g| so that nothing cancels in the lower tail: one
// exponential and one reciprocal, and the slope of gelu needs the same exponential.
__device__ __forceinline__ void normal(float g, float& cdf, float& bell) {
  const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(g), 0.3275911f * 0.70710678f, 1.f));
  bell = __expf(-0.5f * g * g);
  const float p = fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
  const float tail = 0.5f * t * p * bell;
  cdf = g > 0.f ? 1.f - tail : tail;
}
template <int ACT>
__device__ __forceinline__ float act(float g) {
  if constexpr (ACT == B2C_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.f + __expf(-g));
  if constexpr (ACT == B2C_ACT_GELU) {
    float cdf, bell;
    normal(g, cdf, bell);
    return g * cdf;
  }
  return g > 0.f ? g : (g <= 0.f ? 0.f : g);  // a NaN stays one
}
// act(g) in `a` and its derivative in `d`.
template <int ACT>
__device__ __forceinline__ void act_grad(float g, float& a, float& d) {
  if constexpr (ACT == B2C_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-g));
    a = g * s;
    d = fmaf(a, 1.f - s, s);
  } else if constexpr (ACT == B2C_ACT_GELU) {
    float cdf, bell;
    normal(g, cdf, bell);
    a = g * cdf;
    d = fmaf(g * 0.39894228f, bell, cdf);
  } else {
    a = g > 0.f ? g : (g <= 0.f ? 0.f : g);
    d = g > 0.f ? 1.f : 0.f;
  }
}

// W neighbouring values of row m from column n on, of which those from `cols` on do not exist. Whole vectors go in
// one access whatever their alignment, which costs the device nothing but the extra line that they may touch.
template <int W, typename T>
__device__ __forceinline__ void put(T* base, int64_t ld, int64_t m, int n, int cols, const float (&v)[W]) {
  T* p = base + m * ld + n;
  if (n + W <= cols) {
    vec<T, W> t;
#pragma unroll
    for (int j = 0; j < W; j++) t[j] = (T)v[j];
    __builtin_memcpy(p, &t, sizeof(t));
  } else {
#pragma unroll
    for (int j = 0; j < W; j++)
      if (n + j < cols) p[j] = (T)v[j];
  }
}
template <int W, typename T>
__device__ __forceinline__ void get(const T* base, int64_t ld, int64_t m, int n, int cols, float (&v)[W]) {
  const T* p = base + m * ld + n;
  if (n + W <= cols) {
    vec<T, W> t;
    __builtin_memcpy(&t, p, sizeof(t));
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = (float)t[j];
  } else {
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = n + j < cols ? (float)p[j] : 0.f;
  }
}

// ---- epilogues: row m of out, columns n .. n + W - 1 (the first argument is a part, see Parts) ------------------------------------------------------
// The block's inner widths are stored at a pitch of fp columns, a multiple of 64 >= f; columns f .. fp - 1 hold
// zeros, so that a later product may run over them.

// h = act(g) u, and the factors of the backward pass: du = dh act(g), dg = dh u act'(g). act(g) at column n of `saved`,
// u act'(g) at column fp + n, in single precision, since their products with dh are rounded for the matrix instructions anyway:
// kept in T they left the gradients of a 8192 x 2048-5632 step 2.9e-3 off in bf16, where this way they are 2.3e-3 off, as y is; the
// step takes 1551 us so, 1495 with them in T. Factors instead of g and u, so that the backward pass need not take act again.
template <typename T, int ACT>
struct GateOut {
  T* h;
  float* saved;  // [m][2 fp] or null
  int64_t fp;
  int f;
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t, int64_t m, int n, const float (&g)[W], const float (&u)[W]) const {
    float v[W];
    if (!saved) {
#pragma unroll
      for (int j = 0; j < W; j++) v[j] = n + j < f ? act<ACT>(g[j]) * u[j] : 0.f;
    } else {
      float a[W], b[W];
#pragma unroll
      for (int j = 0; j < W; j++) {
        float d;
        act_grad<ACT>(g[j], a[j], d);
        const bool in = n + j < f;
        a[j] = in ? a[j] : 0.f;
        b[j] = in ? u[j] * d : 0.f;
        v[j] = in ? a[j] * u[j] : 0.f;
      }
      put<W>(saved, 2 * fp, m, n, (int)fp, a);
      put<W>(saved + fp, 2 * fp, m, n, (int)fp, b);
    }
    put<W>(h, fp, m, n, (int)fp, v);
  }
};

// y = residual + dropout(v)
template <typename T>
struct RowsOut {
  T* y;
  int64_t ldy;
  const T* r;  // or null
  int64_t ldr;
  int cols;
  Drop drop;
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t, int64_t m, int n, const float (&acc)[W]) const {
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = acc[j];
    if (drop.threshold) {
      static_assert(W == 4 || W == 8);
      const uint64_t e = (uint64_t)m * cols + n;
      const uint32_t k = kept_bits<W>(drop, e);
#pragma unroll
      for (int j = 0; j < W; j++) v[j] = k >> j & 1 ? v[j] * drop.scale : 0.f;
    }
    if (r) {
      float t[W];
      get<W>(r, ldr, m, n, cols, t);
#pragma unroll
      for (int j = 0; j < W; j++) v[j] += t[j];
    }
    put<W>(y, ldy, m, n, cols, v);
  }
};

// dg and du from dh and the factors that the forward pass kept, rounded to T once for the products that follow: relative errors of
// half a unit in the last place, independent from value to value, that average out in the sums.
template <typename T>
struct GateBack {
  const float* saved;  // [m][2 fp]
  T* dgu;          // [m][2 fp]: dg, then du
  int64_t fp;
  int f;
  float scale;  // dropout's: dz enters the products as dy where it is kept, which needs no rounding
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t, int64_t m, int n, const float (&dh)[W]) const {
    float a[W], b[W];
    get<W>(saved, 2 * fp, m, n, (int)fp, a);
    get<W>(saved + fp, 2 * fp, m, n, (int)fp, b);
#pragma unroll
    for (int j = 0; j < W; j++) {
      const bool in = n + j < f;
      const float s = dh[j] * scale;
      a[j] = in ? s * a[j] : 0.f;
      b[j] = in ? s * b[j] : 0.f;
    }
    put<W>(dgu, 2 * fp, m, n, (int)fp, b);
    put<W>(dgu + fp, 2 * fp, m, n, (int)fp, a);
  }
};

// A weight's gradient, in T or single precision. Rows 0 .. rows - 1 go to `a`, rows second .. second + rows - 1
// to `b` (null: there is one).
template <typename T>
struct WeightOut {
  void* a;
  void* b;
  int64_t ld;
  int rows, second, cols;
  bool f32, add;
  float scale;
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t, int64_t m, int n, const float (&acc)[W]) const {
    void* to = m < rows ? a : (m >= second && m < second + rows ? b : nullptr);
    if (!to) return;
    if (m >= rows) m -= second;
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = acc[j] * scale;
    if (f32) {
      if (add) {
        float t[W];
        get<W>((const float*)to, ld, m, n, cols, t);
#pragma unroll
        for (int j = 0; j < W; j++) v[j] += t[j];
      }
      put<W>((float*)to, ld, m, n, cols, v);
    } else {
      put<W>((T*)to, ld, m, n, cols, v);
    }
  }
};

// 8-bit products: y = acc sx[m] sw[n]
template <typename T>
struct ScaledOut {
  T* y;
  int64_t ldy;
  const float *sx, *sw;
  int cols;
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t, int64_t m, int n, const int (&acc)[W]) const {
    const float s = sx[m];
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = (float)acc[j] * s * sw[n + j < cols ? n + j : cols - 1];
    put<W>(y, ldy, m, n, cols, v);
  }
};
// and h = act(g) u from them, in single precision: its rounding to 8 bits, which follows, goes by the row's
// largest value, and a rounding in between would move values across the 8-bit steps.
template <int ACT>
struct ScaledGate {
  float* h;  // [m][fp]
  const float *sx, *sg, *su;
  int64_t fp;
  int f;
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t, int64_t m, int n, const int (&g)[W], const int (&u)[W]) const {
    const float s = sx[m];
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) {
      const int c = n + j < f ? n + j : f - 1;
      v[j] = n + j < f ? act<ACT>((float)g[j] * s * sg[c]) * ((float)u[j] * s * su[c]) : 0.f;
    }
    put<W>(h, fp, m, n, (int)fp, v);
  }
};

// ---- launches ----------------------------------------------------------------------------------------------

// A dimension of a launch holds fewer than 2^32 threads; with more, only the remainder runs and nothing is reported. So many
// workgroups of up to 512 threads go into two dimensions, where the last ones may have no work.
constexpr int64_t kMostInRow = 1 << 22;
inline dim3 grid_of(int64_t blocks) {
  return blocks <= kMostInRow ? dim3((unsigned)blocks) : dim3((unsigned)kMostInRow, (unsigned)((blocks + kMostInRow - 1) / kMostInRow));
}
__device__ __forceinline__ uint32_t block_index() { return blockIdx.y * (uint32_t)kMostInRow + blockIdx.x; }

// ---- host checks -------------------------------------------------------------------------------------------

// A matrix that a call reads or writes: present, on its element's alignment, rows at least as far apart as wide.
inline bool good(const void* p, int64_t ld, int64_t cols, size_t size) {
  return p && reinterpret_cast<uintptr_t>(p) % size == 0 && ld >= cols;
}
// Dropout's constants from p; false where p is outside its range.
inline bool drop_of(float p, uint64_t seed, uint64_t stream, Drop* d) {
  if (!(p >= 0.f && p < 1.f)) return false;
  const uint32_t t = (uint32_t)((double)p * 65536.0 + 0.5);
  if (t >= 65536) return false;
  *d = {seed, stream, t, (float)(65536.0 / (65536.0 - t))};
  return true;
}

// One operand of a product over k: element (i, k) is p[i ld + k], or p[k ld + i] where it is transposed.
template <typename T>
struct Side {
  const T* p;
  int64_t ld;
};

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// A workspace handed out in pieces; without a base it only counts.
struct Room {
  char* base;
  size_t used = 0;
  template <typename T>
  T* take(int64_t n) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += (size_t)up(n * (int64_t)sizeof(T), 256);
    return p;
  }
};

}  // namespace dev
}  // namespace b2c
