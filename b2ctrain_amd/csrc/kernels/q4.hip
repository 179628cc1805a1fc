// Weights in 4 bits with a scale, and a zero point where there are any, for each group of columns (b2c_hip_quantize4,
// b2c_hip_q4_linear).
#include "dense_product.h"
#include "dense_rows.h"

namespace b2c {
namespace dev {
namespace {

// ---- to 4 bits ---------------------------------------------------------------------------------------------

// The largest of the values that N neighbouring lanes hold, to all of them.
template <int N, typename Better>
__device__ __forceinline__ uint32_t among(uint32_t v, Better better) {
#define B2C_STEP(CTRL) v = better(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true))
  if constexpr (N >= 2) B2C_STEP(0xB1);   // quad_perm:[1,0,3,2]
  if constexpr (N >= 4) B2C_STEP(0x4E);   // quad_perm:[2,3,0,1]
  if constexpr (N >= 8) B2C_STEP(0x141);  // row_half_mirror
  if constexpr (N >= 16) B2C_STEP(0x140); // row_mirror
#undef B2C_STEP
  if constexpr (N >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = better((uint32_t)r[0], (uint32_t)r[1]);
  }
  return v;
}

struct PackArgs {
  int64_t rows;
  int cols, groups;
  uint32_t pieces;  // of eight columns, in a row's groups
  const void* x;
  uint8_t *q, *zero;
  void *scale, *values;
  int64_t ldx, ldq, lds, ldz, ldv;
};

// A thread takes eight columns, so a group is GROUP / 8 neighbouring lanes, which find its scale among themselves: x is read once. Bound by
// memory, with the arithmetic close behind: 11264 x 4096 in bf16 by 128 with `values` (208 MB) 41.5 us, 5.0 TB/s, VALU 92%; 5001 x 2049
// in f32 by 32 with zero points and `values` (88 MB) 16.6 us, 5.3 TB/s.
template <typename T, typename S, int GROUP, bool ZERO>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a) {
  constexpr int LANES = GROUP / 8;
  const int64_t first = (int64_t)block_index() * 256, m0 = first / a.pieces;
  const uint32_t at = (uint32_t)(first - m0 * a.pieces) + threadIdx.x, down = at / a.pieces, piece = at - down * a.pieces;
  const int64_t m = m0 + down;
  const bool there = m < a.rows;
  const int n = (int)piece * 8;
  float x[8] = {};
  if (there && n < a.cols) get<8>((const T*)a.x, a.ldx, m, n, a.cols, x);
  uint32_t top = 0;  // magnitudes as bits, in which an infinity or NaN orders last
  float lo = 0.f, hi = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu;
    top = b > top ? b : top;
    lo = fminf(lo, x[j]);
    hi = fmaxf(hi, x[j]);
  }
  top = among<LANES>(top, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
  float reach = __builtin_bit_cast(float, top) / 7.f;
  if constexpr (ZERO) {
    lo = __builtin_bit_cast(float, among<LANES>(__builtin_bit_cast(uint32_t, lo), [](uint32_t p, uint32_t q) {
      return __builtin_bit_cast(uint32_t, fminf(__builtin_bit_cast(float, p), __builtin_bit_cast(float, q)));
    }));
    hi = __builtin_bit_cast(float, among<LANES>(__builtin_bit_cast(uint32_t, hi), [](uint32_t p, uint32_t q) {
      return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, p), __builtin_bit_cast(float, q)));
    }));
    reach = (hi - lo) / 15.f;
  }
  const S held = (S)(top < 0x7f800000u ? reach : __builtin_nanf(""));
  const float scale = (float)held;
  const bool fine = scale > 0.f && scale < __builtin_inff();
  // x / scale, correctly rounded: with the correctly rounded inverse y, q = x y and its remainder x - q scale (exact in one fused operation),
  // q + remainder y is it (Markstein 1990), three operations in place of a division's ten, where nothing under- or overflows. With divisions
  // the arithmetic takes longer than the memory: 47 us for 11264 x 4096.
  const bool plain = scale > 1e-30f && scale < 1e30f;
  const float inverse = plain ? 1.f / scale : 0.f;
  auto over = [&](float v) {
    if (!plain) return v / scale;
    const float q = v * inverse;
    return fmaf(fmaf(-q, scale, v), inverse, q);
  };
  const float zero = !ZERO ? 8.f : fine ? fminf(fmaxf(rintf(over(-lo)), 0.f), 15.f) : 0.f;
  if (!there || n >= a.cols) return;
  uint32_t word = 0;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float code = fine ? __builtin_amdgcn_fmed3f(rintf(over(x[j])) + zero, 0.f, 15.f) : zero;
    v[j] = (code - zero) * scale;
    word |= (uint32_t)(n + j < a.cols ? code : 0.f) << (4 * j);
  }
  uint8_t* q = a.q + m * a.ldq + piece * 4;
  if (n + 8 <= a.cols) {
    __builtin_memcpy(q, &word, 4);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (n + 2 * j < a.cols) q[j] = (uint8_t)(word >> (8 * j));
  }
  if (a.values) put<8>((T*)a.values, a.ldv, m, n, a.cols, v);
  if (piece % LANES == 0) {
    const int64_t g = piece / LANES;
    ((S*)a.scale)[m * a.lds + g] = held;
    if constexpr (ZERO) a.zero[m * a.ldz + g] = (uint8_t)zero;
  }
}

// ---- products ----------------------------------------------------------------------------------------------

// A code c of 4 bits becomes the 16-bit float (BASE + c) UNIT by taking its place among the mantissa's bits of BASE UNIT, two to a register: no
// conversion. UNIT is a power of two small enough that a group's sum of up to 128 (BASE + c) x, c up to 15, stays within single precision's
// range whatever numbers x holds. The eight codes of a word, in their order.
template <typename T>
struct Codes;
template <>
struct Codes<bf16> {
  static constexpr float BASE = 128.f, UNIT = 0x1p-15f;  // 0x3b80: the lowest mantissa bit counts 1 UNIT
  static __device__ __forceinline__ uint32_t two(uint32_t t) { return (t & 0x000f000fu) | 0x3b803b80u; }
  static __device__ __forceinline__ uint32_t spread(uint32_t a) { return a << 12 | a; }
};
template <>
struct Codes<f16> {
  static constexpr float BASE = 64.f, UNIT = 1.f;  // 0x5400: bit 4 counts 1
  static __device__ __forceinline__ uint32_t two(uint32_t t) { return (t & 0x00f000f0u) | 0x54005400u; }
  static __device__ __forceinline__ uint32_t spread(uint32_t a) { return a << 16 | a << 4; }
};
template <typename T>
__device__ __forceinline__ vec<T, 8> codes(uint32_t w) {
  using D = Codes<T>;
  const uint32_t a = D::spread(w & 0xffffu), b = D::spread(w >> 16);
  const vec<uint32_t, 4> v = {D::two(a), D::two(a >> 8), D::two(b), D::two(b >> 8)};
  return __builtin_bit_cast(vec<T, 8>, v);
}

// The same in the order 0, 4, 1, 5, 2, 6, 3, 7, which takes seven operations in place of ten.
template <typename T>
__device__ __forceinline__ vec<uint32_t, 4> codes_apart(uint32_t w) {
  using D = Codes<T>;
  constexpr int down = std::is_same_v<T, bf16> ? 0 : 4;  // where the lowest bit of a code counts 1
  return {D::two(w << down), D::two(down ? w : w >> 4), D::two(w >> (8 - down)), D::two(w >> (12 - down))};
}

template <typename T>
struct Weights4 {
  const uint8_t* q;
  int64_t ldq;
  const T* scale;
  int64_t lds;
  const uint8_t* zero;
  int64_t ldz;
  int rows, cols, groups;
};

// Sixteen bytes of a row from byte b on; zeros beyond the row's last, at whose place the last is read: loads without conditions go out
// together, where one that waits for its condition holds up the next.
__device__ __forceinline__ vec<uint32_t, 4> bytes16(const uint8_t* row, int b, int bytes) {
  vec<uint32_t, 4> v{};
  if (b + 16 <= bytes) {
    __builtin_memcpy(&v, row + b, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 16; j++)
      v[j / 4] |= (b + j < bytes ? (uint32_t)row[b + j < bytes ? b + j : bytes - 1] : 0u) << (j % 4 * 8);
  }
  return v;
}
// The four words that lanes l, l + 16, l + 32, l + 48 hold, turned: word i of lane 16 j + l becomes word j of lane 16 i + l.
__device__ __forceinline__ void turn4(vec<uint32_t, 4>& v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false), b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  v = {(uint32_t)c[0], (uint32_t)c[1], (uint32_t)d[0], (uint32_t)d[1]};
}
// At most 16 MT rows of x. A workgroup takes 16 NT outputs, its eight waves every eighth run of 128 values of k: sixteen bytes of a row a
// lane, turned so that each matrix instruction meets 32 neighbouring values of k, which are of one group. With c the code and B its base, a
// group's sum is s (sum (B + c) x - (B + z) sum x), and sum x comes from the same instruction against ones, in the same lanes, all of it in
// units of UNIT. B is at most 128, so that the difference costs four bits of the 24 that the sums are held in. Rows beyond the last read
// the last one's values, which nobody stores; in the run at the end of k (not the first: LONG) every load that would pass a row's end reads
// its last bytes, which are then moved to their place, so that no load waits for a condition (7 rows of 2050-5001: 3 us less). The waves'
// sums meet in LDS and are added in a fixed order. Bound by the latency of two to four round trips where there are few runs: 7 rows of
// 2050-5001 (f16, by 32, zero points; 6 MB) take 10.1 us, 9.7 with rows on even bytes and 6.3 on sixteen; of 2048 9.0, 8.5 and 5.8; 16 of
// 4096-11264 13.9.
template <typename T, int GROUP, bool ZERO, int MT, int NT, bool LONG>
__global__ __launch_bounds__(512, MT == 4 ? 2 : 4) void q4_few_kernel(Weights4<T> w, int shift, Side<T> all, int64_t all_rows, T* all_y,
                                                                      int64_t ldy) {
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const Side<T> x{all.p + m0 * all.ld, all.ld};
  T* y = all_y + m0 * ldy;
  const int M = all_rows - m0 < 16 * MT ? (int)(all_rows - m0) : 16 * MT;
  constexpr int NG = GROUP >= 128 ? 1 : 128 / GROUP, PER = 4 / NG;  // groups of a run, matrix instructions of a group
  constexpr int U = MT == 4 ? 1 : MT == 1 ? (NT == 1 ? 4 : 2) : (NT == 4 ? 1 : 2);  // runs in flight
  __shared__ f32x4 sums[8][NT][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & 15, q4 = lane >> 4;
  const int n0 = (int)blockIdx.x * 16 * NT, rows = w.rows - n0;
  const int K = w.cols, bytes = (K + 1) >> 1, whole = K >> 7, runs = (K + 127) >> 7;
  const uint8_t* q = w.q + n0 * w.ldq;
  const T* scale = w.scale + n0 * w.lds;
  const uint8_t* zero = ZERO ? w.zero + n0 * w.ldz : nullptr;
  uint32_t q_at[NT], s_at[NT], z_at[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    const uint32_t r = n * 16 + row < rows ? n * 16 + row : rows - 1;
    q_at[n] = r * (uint32_t)w.ldq;
    s_at[n] = r * (uint32_t)w.lds;
    z_at[n] = ZERO ? r * (uint32_t)w.ldz : 0;
  }
  const T* px[MT];
#pragma unroll
  for (int t = 0; t < MT; t++) px[t] = x.p + (t * 16 + row < M ? t * 16 + row : M - 1) * x.ld;
  const T one = (T)Codes<T>::UNIT;
  const vec<T, 8> ones = {one, one, one, one, one, one, one, one};
  struct Run {
    vec<uint32_t, 4> q[NT];
    vec<T, NG> s[NT];
    vec<uint8_t, NG> z[NT];
    vec<T, 8> x[MT][4];
  };
  auto fetch = [&](Run& r, int run) {
    const int k = run * 128;
#pragma unroll
    for (int n = 0; n < NT; n++) {
      __builtin_memcpy(&r.q[n], q + (q_at[n] + (uint32_t)(run * 64 + q4 * 16)), 16);
      __builtin_memcpy(&r.s[n], scale + (s_at[n] + (uint32_t)(k >> shift)), sizeof(T) * NG);
      if constexpr (ZERO) __builtin_memcpy(&r.z[n], zero + (z_at[n] + (uint32_t)(k >> shift)), NG);
    }
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) __builtin_memcpy(&r.x[t][i], px[t] + k + i * 32 + q4 * 8, 16);
  };
  auto fetch_end = [&](Run& r) {  // the run in which a long k ends
    const int k = whole * 128, b = whole * 64 + q4 * 16, at = b < bytes - 16 ? b : bytes - 16;
    const int g = k >> shift, first = g < w.groups - NG ? g : w.groups - NG;
#pragma unroll
    for (int n = 0; n < NT; n++) {
      __builtin_memcpy(&r.q[n], q + (q_at[n] + (uint32_t)at), 16);
      __builtin_memcpy(&r.s[n], scale + (s_at[n] + (uint32_t)first), sizeof(T) * NG);
      if constexpr (ZERO) __builtin_memcpy(&r.z[n], zero + (z_at[n] + (uint32_t)first), NG);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int j = k + i * 32 + q4 * 8, from = j < K - 8 ? j : K - 8;
#pragma unroll
      for (int t = 0; t < MT; t++) __builtin_memcpy(&r.x[t][i], px[t] + from, 16);
    }
  };
  auto settle = [&](Run& r) {  // and everything of it to its place, zeros behind the last
    const int k = whole * 128, b = whole * 64 + q4 * 16, g = k >> shift, off = g - (g < w.groups - NG ? g : w.groups - NG);
#pragma unroll
    for (int n = 0; n < NT; n++) {
      r.q[n] = moved_down(r.q[n], b - (bytes - 16));
      vec<T, NG> s = r.s[n];
      vec<uint8_t, NG> z = r.z[n];
#pragma unroll
      for (int j = 0; j < NG; j++) {
        r.s[n][j] = (T)0.f;
#pragma unroll
        for (int i = 0; i < NG; i++)
          if (j + off == i) r.s[n][j] = s[i], r.z[n][j] = z[i];
      }
    }
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        r.x[t][i] = __builtin_bit_cast(vec<T, 8>, moved_down(__builtin_bit_cast(vec<uint32_t, 4>, r.x[t][i]), 2 * (k + i * 32 + q4 * 8 - (K - 8))));
  };
  auto fetch_only = [&](Run& r) {  // the only run of a short k
#pragma unroll
    for (int n = 0; n < NT; n++) {
      r.q[n] = bytes16(q + q_at[n], q4 * 16, bytes);
      r.s[n] = some<T, NG>(scale + s_at[n], 0, w.groups);
      if constexpr (ZERO) r.z[n] = some<uint8_t, NG>(zero + z_at[n], 0, w.groups);
    }
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) r.x[t][i] = some<T, 8>(px[t], i * 32 + q4 * 8, K);
  };
  f32x4 total[NT][MT] = {};
  auto multiply = [&](Run& r) {
#pragma unroll
    for (int n = 0; n < NT; n++) turn4(r.q[n]);
#pragma unroll
    for (int g = 0; g < NG; g++) {
      f32x4 sum[MT] = {};
#pragma unroll
      for (int i = g * PER; i < (g + 1) * PER; i++)
#pragma unroll
        for (int t = 0; t < MT; t++) sum[t] = mfma(r.x[t][i], ones, sum[t]);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        f32x4 acc[MT] = {};
#pragma unroll
        for (int i = g * PER; i < (g + 1) * PER; i++) {
          const vec<T, 8> p = codes<T>(r.q[n][i]);
#pragma unroll
          for (int t = 0; t < MT; t++) acc[t] = mfma(r.x[t][i], p, acc[t]);
        }
        const float s = (float)r.s[n][g], b = Codes<T>::BASE + (ZERO ? (float)r.z[n][g] : 8.f);
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int j = 0; j < 4; j++) total[n][t][j] = fmaf(s, fmaf(-b, sum[t][j], acc[t][j]), total[n][t][j]);
      }
    }
  };
  if constexpr (LONG) {
    if (whole < runs && wave == 0) {
      Run r;
      fetch_end(r);
      settle(r);
      multiply(r);
    }
    for (int run = wave + 7 & 7; run < whole; run += U * 8) {  // the first wave last, which has had the end
      Run r[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (run + u * 8 < whole) fetch(r[u], run + u * 8);
#pragma unroll
      for (int u = 0; u < U; u++)
        if (run + u * 8 < whole) multiply(r[u]);
    }
  } else if (wave == 0) {
    Run r;
    fetch_only(r);
    multiply(r);
  }
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int t = 0; t < MT; t++) sums[wave][n][t][lane] = total[n][t];
  __syncthreads();
  for (int tile = wave; tile < NT * MT; tile += 8) {
    const int tn = tile % NT, tm = tile / NT, n = n0 + tn * 16 + row;
    f32x4 v = sums[0][tn][tm][lane];
#pragma unroll
    for (int i = 1; i < 8; i++) v += sums[i][tn][tm][lane];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int m = tm * 16 + q4 * 4 + j;
      if (m < M && n < w.rows) y[m * ldy + n] = (T)(v[j] * (1.f / Codes<T>::UNIT));
    }
  }
}

// One row of x. Where a matrix instruction would multiply mostly nothing, a lane multiplies by pairs: 32 values of k of each of its
// wave's four outputs at a time, sixteen bytes that are all of one group, against the same 32 of x, which wait in LDS with their sums, in
// the order in which the codes come apart most cheaply. So a wave reads a kilobyte of a row at once, a slab of 2048 values, and two slabs of
// four rows are on their way together. Where there are few outputs, `split` waves share four of them and take every split-th slab.
// 4096-11264 takes 9.5 us, 2.5 TB/s of weights: one round of workgroups, in which x to LDS, then two steps of loads, follow each other.
template <typename T, bool ZERO>
__global__ __launch_bounds__(256, 4) void q4_one_kernel(Weights4<T> w, int shift, const T* x, T* y, int split) {
  constexpr int SLABS = 4, STEPS = 2;  // slabs of x in LDS; of weights on their way
  __shared__ __attribute__((aligned(16))) vec<uint32_t, 4> held[SLABS * 256];
  __shared__ float sums[SLABS * 64];
  __shared__ float parts[4][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int K = w.cols, bytes = (K + 1) >> 1, slabs = (K + 2047) >> 11;
  const int part = wave % split, n0 = ((int)blockIdx.x * (4 / split) + wave / split) * 4;
  float total[4] = {};
  struct Slab {
    vec<uint32_t, 4> q[4];
    T s[4];
    uint8_t z[4];
  };
  auto fetch = [&](Slab& r, int slab) {
    const int b = slab * 1024 + lane * 16, at = b < bytes - 16 ? b : bytes - 16;
    const int k = slab * 2048 + lane * 32, g = (k < K ? k : K - 1) >> shift;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t n = n0 + i < w.rows ? n0 + i : w.rows - 1;
      __builtin_memcpy(&r.q[i], w.q + n * w.ldq + at, 16);
      r.s[i] = w.scale[n * w.lds + g];
      if constexpr (ZERO) r.z[i] = w.zero[n * w.ldz + g];
    }
  };
  auto multiply = [&](Slab& r, int slab, int i0) {
    if ((slab + 1) * 2048 > K) {  // k ends in this slab
#pragma unroll
      for (int i = 0; i < 4; i++) r.q[i] = moved_down(r.q[i], slab * 1024 + lane * 16 - (bytes - 16));
    }
    vec<uint32_t, 4> p[4];
#pragma unroll
    for (int j = 0; j < 4; j++) p[j] = held[i0 * 4 + (j ^ (i0 >> 2 & 3))];
    const float sum = sums[i0];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float acc[2] = {};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const vec<uint32_t, 4> c = codes_apart<T>(r.q[i][j]);
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e & 1] = dot2(c[e], p[j][e], acc[e & 1], T{});
      }
      const float b = Codes<T>::BASE + (ZERO ? (float)r.z[i] : 8.f);
      total[i] = fmaf((float)r.s[i], fmaf(-b, sum, acc[0] + acc[1]), total[i]);
    }
  };
  for (int base = 0; base < slabs; base += SLABS) {  // as much of x as LDS holds; `split` and STEPS divide it
    if (base) __syncthreads();
    for (int i = threadIdx.x; i < SLABS * 64; i += 256) {
      const int k = base * 2048 + i * 32;
      float s = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        vec<T, 8> v{};
        if (k + j * 8 < K) v = some<T, 8>(x, k + j * 8, K);
#pragma unroll
        for (int e = 0; e < 8; e++) s = fmaf((float)v[e], Codes<T>::UNIT, s);
        const vec<T, 8> apart = {v[0], v[4], v[1], v[5], v[2], v[6], v[3], v[7]};
        held[i * 4 + (j ^ (i >> 2 & 3))] = __builtin_bit_cast(vec<uint32_t, 4>, apart);  // turned: eight lanes' pieces in different banks
      }
      sums[i] = s;
    }
    __syncthreads();
    const int end = slabs < base + SLABS ? slabs : base + SLABS;
    for (int slab = base + part; slab < end; slab += STEPS * split) {
      Slab r[STEPS];
#pragma unroll
      for (int u = 0; u < STEPS; u++)
        if (slab + u * split < end) fetch(r[u], slab + u * split);
#pragma unroll
      for (int u = 0; u < STEPS; u++)
        if (slab + u * split < end) multiply(r[u], slab + u * split, (slab + u * split - base) * 64 + lane);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
#pragma unroll
    for (int o = 32; o; o >>= 1) total[i] += __shfl_xor(total[i], o);
    if (lane == i) parts[wave][i] = total[i];
  }
  __syncthreads();
  if (part || lane >= 4 || n0 + lane >= w.rows) return;
  float v = parts[wave][lane];
  for (int p = 1; p < split; p++) v += parts[wave + p][lane];
  y[n0 + lane] = (T)(v * (1.f / Codes<T>::UNIT));
}

// What the whole numbers code - zero count in the tiles' weights, a power of two, so that 16 bits hold them exactly: as little as keeps the sum
// of a group's 256 products with the largest value of T, up to 15 each, in single precision's range.
template <typename T>
constexpr float kWhole = std::is_same_v<T, bf16> ? 0x1p-12f : 1.f;

// The weights less their scales in T, for the tiles, their scales in single precision and turned, one group's next to each other, and x where
// its rows have to be copied to ones that start on 16 bytes: `own`, the next `scaling` and all other workgroups. There are M rows of x to copy:
// none where x is read in place, and none for the workgroups that a launch of more than 2^22 has too many. A thread takes AT pieces of eight
// values, whose loads are on their way together. Bound by memory: 4096-11264 (116 MB) 25.5 us, 4.5 TB/s.
template <typename T, bool ZERO, int AT>
__global__ __launch_bounds__(256) void unpack_kernel(Weights4<T> w, int shift, T* to, int64_t pitch, float* scale_to, uint32_t scale_pitch,
                                                     uint32_t groups, uint32_t own, uint32_t scaling, Side<T> x, int64_t M, T* x_to) {
  uint32_t block = block_index();
  if (block >= own && block - own < scaling) {
    const int64_t first = (int64_t)(block - own) * 256, g0 = first / scale_pitch;
    const uint32_t at = (uint32_t)(first - g0 * scale_pitch) + threadIdx.x, down = at / scale_pitch;
    const int64_t g = g0 + down, m = at - down * scale_pitch;
    if (g < w.groups && m < w.rows) scale_to[g * scale_pitch + m] = (float)w.scale[m * w.lds + g];
    return;
  }
  const bool copies = block >= own;
  if (copies) block -= own + scaling;
  const int64_t first = (int64_t)block * (256 * AT) + threadIdx.x, m0 = first / groups;
  const uint32_t start = (uint32_t)(first - m0 * groups);
  if (copies) {
#pragma unroll
    for (int i = 0; i < AT; i++) {
      const uint32_t at = start + i * 256, down = i ? at / groups : 0;
      const int64_t m = m0 + down;
      const int n = (int)(at - down * groups) * 8;
      if (m < M) *reinterpret_cast<vec<T, 8>*>(x_to + m * pitch + n) = some<T, 8>(x.p + m * x.ld, n, w.cols);
    }
    return;
  }
  uint32_t word[AT];
  float z[AT];
  int64_t to_at[AT];
  int left[AT];
#pragma unroll
  for (int i = 0; i < AT; i++) {
    const uint32_t at = start + i * 256, down = i ? at / groups : 0;
    const bool there = m0 + down < w.rows;
    const int64_t m = there ? m0 + down : w.rows - 1;
    const int n = (int)(at - down * groups) * 8;
    const uint8_t* q = w.q + m * w.ldq + n / 2;
    word[i] = 0;
    if (n + 8 <= w.cols) {
      __builtin_memcpy(&word[i], q, 4);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (n + 2 * j < w.cols) word[i] |= (uint32_t)q[j] << (8 * j);
    }
    z[i] = ZERO ? (float)w.zero[m * w.ldz + (n >> shift)] : 8.f;
    to_at[i] = m * pitch + n;
    left[i] = there ? w.cols - n : 0;
  }
#pragma unroll
  for (int i = 0; i < AT; i++) {
    vec<T, 8> v;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = j < left[i] ? (T)(((float)(word[i] >> (4 * j) & 15) - z[i]) * kWhole<T>) : (T)0.f;
    if (left[i] > 0) *reinterpret_cast<vec<T, 8>*>(to + to_at[i]) = v;
  }
}

// y from the tiles' sums
template <typename T, int N>
struct Q4Out {
  static constexpr int GROUPS = N;
  GroupScales scales;
  T* y;
  int64_t ldy;
  int cols;
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t, int64_t m, int n, const float (&acc)[W]) const {
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = acc[j] * (1.f / kWhole<T>);
    put<W>(y, ldy, m, n, cols, v);
  }
};

// ---- host --------------------------------------------------------------------------------------------------

bool group_ok(int g) { return g == 32 || g == 64 || g == 128 || g == 256; }
int groups_of(int cols, int group) { return (cols + group - 1) / group; }

template <typename F>
int with_group(int group, F f) {
  using std::integral_constant;
  if (group == 32) return f(integral_constant<int, 32>{});
  if (group == 64) return f(integral_constant<int, 64>{});
  if (group == 128) return f(integral_constant<int, 128>{});
  return f(integral_constant<int, 256>{});
}

template <typename T, typename S>
int pack(const b2c_quantize4_args* a, hipStream_t stream) {
  const int groups = groups_of(a->cols, a->group);
  const PackArgs d{a->rows, a->cols, groups, (uint32_t)(groups * (a->group / 8)), a->x, a->q, a->zero, a->scale, a->values,
                   a->ldx, a->ldq, a->lds, a->ldz, a->ldv};
  const int64_t blocks = up(a->rows * (int64_t)d.pieces, 256) / 256;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  return with_group(a->group, [&](auto group) -> int {
    constexpr int G = decltype(group)::value;
    if (a->zero) pack_kernel<T, S, G, true><<<grid_of(blocks), 256, 0, stream>>>(d);
    else pack_kernel<T, S, G, false><<<grid_of(blocks), 256, 0, stream>>>(d);
    return hipGetLastError();
  });
}
template <typename T>
int pack(const b2c_quantize4_args* a, hipStream_t stream) {
  return a->scale_dtype == B2C_F16 ? pack<T, f16>(a, stream) : pack<T, bf16>(a, stream);
}

bool sizes_ok(const b2c_q4_linear_args* a) {
  const int most = 1 << 20;
  return a && a->rows >= 0 && a->rows <= (1 << 30) && a->d_in >= 1 && a->d_in <= most && a->d_out >= 1 && a->d_out <= most &&
         group_ok(a->group) && (a->dtype == B2C_F16 || a->dtype == B2C_BF16);
}
bool direct(const b2c_q4_linear_args* a) {
  return reinterpret_cast<uintptr_t>(a->x) % 16 == 0 && a->ldx % 8 == 0 && a->d_in % 8 == 0 && a->ldx < ((int64_t)1 << 21);
}

// Outputs of a workgroup of the kernel for a few rows, in sixteens: one round of workgroups, one to a compute unit, with as few each as that
// takes; but for three sixteens of more than one row tile, which spill. 16 rows of 4096 -> 4096, 8192 and 11264: 8.7, 11.4 and 13.9 us this
// way, 11.0, 14.0 and 16.2 with the next fewer or more outputs.
int outputs_of(const b2c_q4_linear_args* a) {
  const int64_t tiles = up(a->d_out, 16) / 16;
  if (a->d_in < 128 || tiles <= 256) return 1;
  if (tiles <= 512) return 2;
  return tiles <= 768 && a->rows <= 16 ? 3 : 4;
}
// Whether the weights are multiplied as codes: up to 32 rows; with more, 64 to a workgroup, where that takes less time than to unpack them for
// the tiles, from 64 products timed both ways. A workgroup reads all of its rows of x, and what a compute unit may have on its way from the
// die's cache bounds that: 128 rows of 1024 -> 8192 and 256 of 2048 -> 2048 and 1024 -> 8192 take 13, 20 and 24 us this way, 18, 27 and 29 by
// tiles; but 128 of 4096 -> 4096 35 and 31, 256 of 4096 -> 11264 78 and 62, 512 of 2048 -> 2048 36 and 28.
bool few(const b2c_q4_linear_args* a) {
  if (a->rows <= 32) return true;
  if (a->rows > 512) return false;
  const int n = outputs_of(a);
  const int64_t blocks = up(a->rows, 64) / 64 * (up(a->d_out, 16 * n) / (16 * n));
  const double weights = (double)a->d_in * a->d_out;
  const double codes = 3 + (double)(up(blocks, 256) / 256) * a->d_in * (0.0033 + 0.0007 * n);
  return codes < 19 + weights * 0.45e-6 + weights * (double)a->rows * 2e-9;
}

template <typename T>
struct Q4Plan {
  T *w = nullptr, *x = nullptr;
  float* scales = nullptr;
  int64_t pitch = 0, scale_pitch = 0;
  Way way{};
  void* sums = nullptr;
  Q4Plan(const b2c_q4_linear_args* a, Room& room) {
    if (few(a)) return;
    pitch = up(a->d_in, 64);
    w = room.take<T>(a->d_out * pitch);
    scale_pitch = up(a->d_out, 128);
    scales = room.take<float>(groups_of(a->d_in, a->group) * scale_pitch);
    if (!direct(a)) x = room.take<T>(a->rows * pitch);
    way = choose({{a->rows, a->d_out}}, pitch / 64, false, false, 2, TILE_128);
    sums = room.take<char>(way.sums);
  }
};

// One row takes a kernel of its own where its slabs are at least nine tenths full: 4096 -> 11264 9.6 us and 8192 -> 1024 5.1, by the kernel
// for a few 12.1 and 8.4; 2600 -> 11264 9.2 and 7.8, and below one slab 1024 -> 1024 4.7 and 3.2. Its waves share outputs until there
// are 2048 of them: 8192 -> 1024 takes 6.7, 5.5 and 5.0 us with one, two and four waves, 4096 -> 11264 9.7, 10.9 and 14.8.
bool one_row(const b2c_q4_linear_args* a) {
  const int64_t slabs = up(a->d_in, 2048) / 2048;
  return a->rows == 1 && a->d_in >= 2048 && a->d_in * 10 >= slabs * 2048 * 9;
}
int split_of(const b2c_q4_linear_args* a) {
  const int64_t slabs = up(a->d_in, 2048) / 2048;
  int split = 1;
  while (split < 4 && split * 2 <= slabs && (int64_t)split * a->d_out < 8192) split *= 2;
  return split;
}

template <typename T>
int linear(const b2c_q4_linear_args* a, hipStream_t stream) {
  const Weights4<T> w{a->w, a->ldw, (const T*)a->scale, a->lds, a->zero, a->ldz, a->d_out, a->d_in, groups_of(a->d_in, a->group)};
  Side<T> x{(const T*)a->x, a->ldx};
  const int shift = a->group == 32 ? 5 : a->group == 64 ? 6 : a->group == 128 ? 7 : 8;
  if (few(a)) {
    using std::integral_constant;
    if (one_row(a)) {
      const int split = split_of(a);
      const dim3 grid((unsigned)(up(a->d_out, 16 / split) / (16 / split)));
      if (a->zero) q4_one_kernel<T, true><<<grid, 256, 0, stream>>>(w, shift, x.p, (T*)a->y, split);
      else q4_one_kernel<T, false><<<grid, 256, 0, stream>>>(w, shift, x.p, (T*)a->y, split);
      return hipGetLastError();
    }
    auto run = [&](auto group, auto zero, auto rows, auto outputs, auto far) -> int {
      constexpr int NT = decltype(outputs)::value, MT = decltype(rows)::value;
      q4_few_kernel<T, decltype(group)::value, decltype(zero)::value, MT, NT, decltype(far)::value>
          <<<dim3((unsigned)(up(a->d_out, 16 * NT) / (16 * NT)), (unsigned)(up(a->rows, 16 * MT) / (16 * MT))), 512, 0, stream>>>(
              w, shift, x, a->rows, (T*)a->y, a->ldy);
      return hipGetLastError();
    };
    auto with_rows = [&](auto group, auto zero) {
      auto with_outputs = [&](auto rows) {
        if (a->d_in < 128) return run(group, zero, rows, integral_constant<int, 1>{}, std::false_type{});
        const int n = outputs_of(a);
        if (n == 1) return run(group, zero, rows, integral_constant<int, 1>{}, std::true_type{});
        if (n == 2) return run(group, zero, rows, integral_constant<int, 2>{}, std::true_type{});
        if constexpr (decltype(rows)::value == 1)
          if (n == 3) return run(group, zero, rows, integral_constant<int, 3>{}, std::true_type{});
        return run(group, zero, rows, integral_constant<int, 4>{}, std::true_type{});
      };
      if (a->rows > 32) return with_outputs(integral_constant<int, 4>{});
      return a->rows <= 16 ? with_outputs(integral_constant<int, 1>{}) : with_outputs(integral_constant<int, 2>{});
    };
    auto with_zero = [&](auto group) { return a->zero ? with_rows(group, std::true_type{}) : with_rows(group, std::false_type{}); };
    if (a->group == 32) return with_zero(integral_constant<int, 32>{});
    if (a->group == 64) return with_zero(integral_constant<int, 64>{});
    return with_zero(integral_constant<int, 128>{});
  }
  Room room{(char*)a->workspace};
  const Q4Plan<T> p(a, room);
  const uint32_t pieces = (uint32_t)(up(a->d_in, 8) / 8);
  auto unpack = [&](auto zero, auto at) -> int {
    const int64_t block = 256 * at.value, own = up((int64_t)a->d_out * pieces, block) / block, copies = p.x ? up(a->rows * pieces, block) / block : 0;
    const int64_t scaling = up(w.groups * p.scale_pitch, 256) / 256;
    if (own + scaling + copies > 0x7fffffff) return hipErrorInvalidValue;
    unpack_kernel<T, zero.value, at.value>
        <<<grid_of(own + scaling + copies), 256, 0, stream>>>(w, shift, p.w, p.pitch, p.scales, (uint32_t)p.scale_pitch, pieces,
                                                              (uint32_t)own, (uint32_t)scaling, x, p.x ? a->rows : 0, p.x);
    return hipGetLastError();
  };
  // Four pieces a thread where that leaves workgroups enough: 4096-11264 25.5 us, 30 with one; 1000-1000 5.1 and 4.0, 2050-5001 9.9 and 9.0.
  auto with_zero = [&](auto zero) {
    if ((int64_t)a->d_out * pieces >= 1 << 21) return unpack(zero, std::integral_constant<int, 4>{});
    return unpack(zero, std::integral_constant<int, 1>{});
  };
  const int rc = a->zero ? with_zero(std::true_type{}) : with_zero(std::false_type{});
  if (rc) return rc;
  if (p.x) x = {p.x, p.pitch};
  const Product<T> product_of{x, {p.w, p.pitch}, {}, {}, a->rows, a->d_out, a->d_in, 0, a->rows, a->d_out};
  const GroupScales scales{p.scales, p.scale_pitch, shift};
  auto tiles = [&](auto groups) {
    return product<T, false, false, false, false>(product_of, p.way, p.sums, Q4Out<T, groups.value>{scales, (T*)a->y, a->ldy, a->d_out}, stream);
  };
  return a->group == 32 ? tiles(std::integral_constant<int, 2>{}) : tiles(std::integral_constant<int, 1>{});
}

}  // namespace
}  // namespace dev
}  // namespace b2c

using namespace b2c::dev;

extern "C" int b2c_hip_quantize4(const b2c_quantize4_args* a, hipStream_t stream) {
  if (!a || a->rows < 0 || a->rows > (1 << 30) || a->cols < 1 || a->cols > (1 << 20) || !group_ok(a->group) || a->dtype < B2C_F32 ||
      a->dtype > B2C_BF16 || (a->scale_dtype != B2C_F16 && a->scale_dtype != B2C_BF16))
    return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  const size_t s = a->dtype == B2C_F32 ? 4 : 2;
  const int groups = groups_of(a->cols, a->group);
  if (!good(a->x, a->ldx, a->cols, s) || !good(a->q, a->ldq, (a->cols + 1) / 2, 1) || !good(a->scale, a->lds, groups, 2) ||
      (a->zero && !good(a->zero, a->ldz, groups, 1)) || (a->values && !good(a->values, a->ldv, a->cols, s)))
    return hipErrorInvalidValue;
  if (a->dtype == B2C_F32) return pack<float>(a, stream);
  if (a->dtype == B2C_F16) return pack<f16>(a, stream);
  return pack<bf16>(a, stream);
}

extern "C" size_t b2c_q4_linear_workspace_bytes(const b2c_q4_linear_args* a) {
  if (!sizes_ok(a) || a->rows == 0) return 0;
  Room room{nullptr};
  Q4Plan<bf16>(a, room);  // both types have the same size
  return room.used;
}
extern "C" int b2c_hip_q4_linear(const b2c_q4_linear_args* a, hipStream_t stream) {
  if (!sizes_ok(a)) return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  const int groups = groups_of(a->d_in, a->group);
  const size_t need = b2c_q4_linear_workspace_bytes(a);
  if (!good(a->x, a->ldx, a->d_in, 2) || !good(a->w, a->ldw, (a->d_in + 1) / 2, 1) || !good(a->scale, a->lds, groups, 2) ||
      (a->zero && !good(a->zero, a->ldz, groups, 1)) || !good(a->y, a->ldy, a->d_out, 2) ||
      a->ldw > kFarRows || a->lds > kFarRows || (a->zero && a->ldz > kFarRows) ||
      (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_bytes < need)))
    return hipErrorInvalidValue;
  return a->dtype == B2C_F16 ? linear<f16>(a, stream) : linear<bf16>(a, stream);
}
