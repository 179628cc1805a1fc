// What the dense operators' kernels share: element types, vector loads and stores, the activations, and the
// epilogues that finish a tile of a matrix product.
//
// Every product is out[m][n] = sum_k Q[m][k] P[n][k]. A matrix instruction is issued with P as its first
// operand, so that a lane's accumulators lie along n, the direction in which out is contiguous: it stores
// several neighbouring values at once.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
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

template <int ACT>
__device__ __forceinline__ float act(float g) {
  if constexpr (ACT == B2C_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.f + __expf(-g));
  if constexpr (ACT == B2C_ACT_GELU) return g * (0.5f + 0.5f * erff(g * 0.70710678f));
  return g > 0.f ? g : (g <= 0.f ? 0.f : g);  // a NaN stays one
}
// act(g) in `a` and its derivative in `d`.
template <int ACT>
__device__ __forceinline__ void act_grad(float g, float& a, float& d) {
  if constexpr (ACT == B2C_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-g));
    a = g * s;
    d = s * (1.f + g * (1.f - s));
  } else if constexpr (ACT == B2C_ACT_GELU) {
    const float phi = 0.5f + 0.5f * erff(g * 0.70710678f);
    a = g * phi;
    d = phi + g * __expf(-0.5f * g * g) * 0.39894228f;
  } else {
    a = g > 0.f ? g : (g <= 0.f ? 0.f : g);
    d = g > 0.f ? 1.f : 0.f;
  }
}

// W neighbouring values of row m from column n on, of which those from `cols` on do not exist. `wide`: rows
// start on 16 bytes.
template <int W, typename T>
__device__ __forceinline__ void put(T* base, int64_t ld, int64_t m, int n, int cols, bool wide, const float (&v)[W]) {
  T* p = base + m * ld + n;
  if (wide && n + W <= cols) {
    vec<T, W> t;
#pragma unroll
    for (int j = 0; j < W; j++) t[j] = (T)v[j];
    *reinterpret_cast<vec<T, W>*>(p) = t;
  } else {
#pragma unroll
    for (int j = 0; j < W; j++)
      if (n + j < cols) p[j] = (T)v[j];
  }
}
template <int W, typename T>
__device__ __forceinline__ void get(const T* base, int64_t ld, int64_t m, int n, int cols, bool wide, float (&v)[W]) {
  const T* p = base + m * ld + n;
  if (wide && n + W <= cols) {
    const vec<T, W> t = *reinterpret_cast<const vec<T, W>*>(p);
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = (float)t[j];
  } else {
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = n + j < cols ? (float)p[j] : 0.f;
  }
}

// ---- epilogues: row m of out, columns n .. n + W - 1 ------------------------------------------------------
// The block's inner widths are stored at a pitch of fp columns, a multiple of 64 >= f; columns f .. fp - 1 hold
// zeros, so that a later product may run over them.

// h = act(g) u, and g, u for the backward pass: g at column n of `saved`, u at column fp + n.
template <typename T, int ACT>
struct GateOut {
  T* h;
  T* saved;  // [m][2 fp] or null
  int64_t fp;
  int f;
  template <int W>
  __device__ __forceinline__ void operator()(int64_t m, int n, const float (&g)[W], const float (&u)[W]) const {
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = n + j < f ? act<ACT>(g[j]) * u[j] : 0.f;
    put<W>(h, fp, m, n, (int)fp, true, v);
    if (saved) {
      float a[W], b[W];
#pragma unroll
      for (int j = 0; j < W; j++) a[j] = n + j < f ? g[j] : 0.f, b[j] = n + j < f ? u[j] : 0.f;
      put<W>(saved, 2 * fp, m, n, (int)fp, true, a);
      put<W>(saved + fp, 2 * fp, m, n, (int)fp, true, b);
    }
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
  bool wide_y, wide_r;
  Drop drop;
  template <int W>
  __device__ __forceinline__ void operator()(int64_t m, int n, const float (&acc)[W]) const {
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = acc[j];
    if (drop.threshold) {
#pragma unroll
      for (int j = 0; j < W; j += 4) {
        const uint32_t k = kept4(drop, (uint64_t)m * cols + n + j);
#pragma unroll
        for (int i = 0; i < 4; i++) v[j + i] = k >> i & 1 ? v[j + i] * drop.scale : 0.f;
      }
    }
    if (r) {
      float t[W];
      get<W>(r, ldr, m, n, cols, wide_r, t);
#pragma unroll
      for (int j = 0; j < W; j++) v[j] += t[j];
    }
    put<W>(y, ldy, m, n, cols, wide_y, v);
  }
};

// From dh and the saved g, u: h = act(g) u (for the down weights' gradient), dg = dh u act'(g), du = dh act(g).
// g, u, and so h, dg and du, are rounded to T: each enters the gradients with a relative error of half a unit
// in the last place, which is independent from value to value and averages out in the sums that follow.
template <typename T, int ACT>
struct GateBack {
  const T* saved;  // [m][2 fp]
  T* h;            // [m][fp] or null
  T* dgu;          // [m][2 fp]: dg, then du
  int64_t fp;
  int f;
  template <int W>
  __device__ __forceinline__ void operator()(int64_t m, int n, const float (&dh)[W]) const {
    float g[W], u[W], v[W];
    get<W>(saved, 2 * fp, m, n, (int)fp, true, g);
    get<W>(saved + fp, 2 * fp, m, n, (int)fp, true, u);
#pragma unroll
    for (int j = 0; j < W; j++) {
      float a, d;
      act_grad<ACT>(g[j], a, d);
      const bool in = n + j < f;
      v[j] = in ? a * u[j] : 0.f;
      g[j] = in ? dh[j] * u[j] * d : 0.f;
      u[j] = in ? dh[j] * a : 0.f;
    }
    if (h) put<W>(h, fp, m, n, (int)fp, true, v);
    put<W>(dgu, 2 * fp, m, n, (int)fp, true, g);
    put<W>(dgu + fp, 2 * fp, m, n, (int)fp, true, u);
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
  bool f32, add, wide;
  template <int W>
  __device__ __forceinline__ void operator()(int64_t m, int n, const float (&acc)[W]) const {
    void* to = m < rows ? a : (m >= second && m < second + rows ? b : nullptr);
    if (!to) return;
    if (m >= rows) m -= second;
    if (f32) {
      float v[W];
#pragma unroll
      for (int j = 0; j < W; j++) v[j] = acc[j];
      if (add) {
        float t[W];
        get<W>((const float*)to, ld, m, n, cols, wide, t);
#pragma unroll
        for (int j = 0; j < W; j++) v[j] += t[j];
      }
      put<W>((float*)to, ld, m, n, cols, wide, v);
    } else {
      put<W>((T*)to, ld, m, n, cols, wide, acc);
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
  bool wide;
  template <int W>
  __device__ __forceinline__ void operator()(int64_t m, int n, const int (&acc)[W]) const {
    const float s = sx[m];
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = (float)acc[j] * s * sw[n + j < cols ? n + j : cols - 1];
    put<W>(y, ldy, m, n, cols, wide, v);
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
  __device__ __forceinline__ void operator()(int64_t m, int n, const int (&g)[W], const int (&u)[W]) const {
    const float s = sx[m];
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) {
      const int c = n + j < f ? n + j : f - 1;
      v[j] = n + j < f ? act<ACT>((float)g[j] * s * sg[c]) * ((float)u[j] * s * su[c]) : 0.f;
    }
    put<W>(h, fp, m, n, (int)fp, true, v);
  }
};

// ---- host checks -------------------------------------------------------------------------------------------

// A matrix that a call reads or writes: present, on its element's alignment, rows at least as far apart as wide.
inline bool good(const void* p, int64_t ld, int64_t cols, size_t size) {
  return p && reinterpret_cast<uintptr_t>(p) % size == 0 && ld >= cols;
}
inline bool wide(const void* p, int64_t ld, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (int64_t)size % 16 == 0;
}
// Dropout's constants from p; false where p is outside its range.
inline bool drop_of(float p, uint64_t seed, uint64_t stream, Drop* d) {
  if (!(p >= 0.f && p < 1.f)) return false;
  const uint32_t t = (uint32_t)((double)p * 65536.0 + 0.5);
  if (t >= 65536) return false;
  *d = {seed, stream, t, (float)(65536.0 / (65536.0 - t))};
  return true;
}

// ---- a product ---------------------------------------------------------------------------------------------

// One operand of a product over k: element (i, k) is p[i ld + k], or p[k ld + i] where it is transposed.
template <typename T>
struct Side {
  const T* p;
  int64_t ld;
};

// out[m][n] = sum_k Q[m][k] P[n][k] by 64x64 tiles, 32 bytes x 2 of k a step, any alignment. DUAL: P2 runs beside
// P with the same Q (gate and up). A second segment (q2, p2, k2 > 0) continues the sum.
template <typename T, bool PT, bool QT, bool DUAL, typename Epi>
__global__ __launch_bounds__(256) void product_kernel(Side<T> q, Side<T> p, Side<T> q2, Side<T> p2, int64_t M, int N,
                                                      int64_t K, int64_t K2, int tiles_n, Epi epi) {
  constexpr int V = Elem<T>::N, BK = 4 * V, PAD = V, BM = 64, BN = 64;
  using Acc = typename Elem<T>::Acc;
  using A = vec<T, V>;
  __shared__ alignas(16) T sq[BM][BK + PAD];
  __shared__ alignas(16) T sp[DUAL ? 2 : 1][BN][BK + PAD];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * BM;
  const int n0 = (int)(blockIdx.x % tiles_n) * BN;
  Acc acc[DUAL ? 2 : 1][2][2] = {};
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;

  auto stage = [&](const Side<T>& s, bool trans, int64_t i0, int64_t I, int64_t k0, int64_t kn, T(*dst)[BK + PAD]) {
    if (!trans) {
      const int r = t >> 2, c = (t & 3) * V;
      const int64_t i = i0 + r;
#pragma unroll
      for (int j = 0; j < V; j++) dst[r][c + j] = i < I && k0 + c + j < kn ? s.p[i * s.ld + k0 + c + j] : (T)0;
    } else {
      const int r = t & 63;
      const int64_t i = i0 + r;
#pragma unroll
      for (int j = 0; j < V; j++) {
        const int c = (t >> 6) * V + j;
        dst[r][c] = i < I && k0 + c < kn ? s.p[(k0 + c) * s.ld + i] : (T)0;
      }
    }
  };
  for (int seg = 0; seg < 2; seg++) {
    const Side<T>&Q = seg ? q2 : q, &P = seg && !DUAL ? p2 : p;
    const int64_t kn = seg ? K2 : K;
    for (int64_t k0 = 0; k0 < kn; k0 += BK) {
      __syncthreads();
      stage(Q, QT, m0, M, k0, kn, sq);
      stage(P, PT, n0, N, k0, kn, sp[0]);
      if constexpr (DUAL) stage(p2, PT, n0, N, k0, kn, sp[1]);
      __syncthreads();
      const int row = lane & 15, kk = (lane >> 4) * V;
      A fq[2];
#pragma unroll
      for (int i = 0; i < 2; i++) fq[i] = *reinterpret_cast<const A*>(&sq[wm + i * 16 + row][kk]);
#pragma unroll
      for (int d = 0; d < (DUAL ? 2 : 1); d++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const A fp = *reinterpret_cast<const A*>(&sp[d][wn + j * 16 + row][kk]);
#pragma unroll
          for (int i = 0; i < 2; i++) acc[d][i][j] = mfma(fp, fq[i], acc[d][i][j]);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int64_t m = m0 + wm + i * 16 + (lane & 15);
      const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
      if (m >= M || n >= N) continue;
      using S = std::remove_reference_t<decltype(acc[0][0][0][0])>;
      S a[4], b[4];
#pragma unroll
      for (int r = 0; r < 4; r++) a[r] = acc[0][i][j][r], b[r] = acc[DUAL ? 1 : 0][i][j][r];
      if constexpr (DUAL) epi.template operator()<4>(m, n, a, b);
      else epi.template operator()<4>(m, n, a);
    }
}

template <typename T, bool PT, bool QT, bool DUAL, typename Epi>
int product(Side<T> q, Side<T> p, Side<T> q2, Side<T> p2, int64_t M, int64_t N, int64_t K, int64_t K2, const Epi& epi,
            hipStream_t stream) {
  if (M <= 0 || N <= 0) return hipSuccess;
  const int64_t tn = (N + 63) / 64, tm = (M + 63) / 64;
  if (tn * tm > 0x7fffffff) return hipErrorInvalidValue;
  product_kernel<T, PT, QT, DUAL, Epi>
      <<<dim3((unsigned)(tm * tn)), 256, 0, stream>>>(q, p, q2, p2, M, (int)N, K, K2, (int)tn, epi);
  return hipGetLastError();
}

}  // namespace dev
}  // namespace b2c
