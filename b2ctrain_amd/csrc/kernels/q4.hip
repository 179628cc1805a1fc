// Weights in 4 bits with a scale, and a zero point where there are any, for each group of columns (b2c_hip_quantize4,
// b2c_hip_q4_linear).
#include "dense_product.h"

namespace b2c {
namespace dev {
namespace {

constexpr int64_t kFewRows = 32;  // up to here the weights are multiplied as codes

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

// A thread takes eight columns, so a group is GROUP / 8 neighbouring lanes, which find its scale among themselves: x is read once.
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
  const float zero = !ZERO ? 8.f : fine ? fminf(fmaxf(rintf(-lo / scale), 0.f), 15.f) : 0.f;
  if (!there || n >= a.cols) return;
  uint32_t word = 0;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float code = fine ? fminf(fmaxf(rintf(x[j] / scale) + zero, 0.f), 15.f) : zero;
    v[j] = (code - zero) * scale;
    if (n + j < a.cols) word |= (uint32_t)code << (4 * j);
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

// A code c of 4 bits becomes the 16-bit float BASE + c by taking its place among the mantissa's bits of BASE, two to a register: no
// conversion. The eight codes of a word, in their order.
template <typename T>
struct Codes;
template <>
struct Codes<bf16> {
  static constexpr float BASE = 128.f;  // 0x4300: the lowest mantissa bit counts 1
  static __device__ __forceinline__ uint32_t two(uint32_t t) { return (t & 0x000f000fu) | 0x43004300u; }
  static __device__ __forceinline__ uint32_t spread(uint32_t a) { return a << 12 | a; }
};
template <>
struct Codes<f16> {
  static constexpr float BASE = 64.f;  // 0x5400: bit 4 counts 1
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

// Sixteen bytes of a row from byte b on; zeros beyond the row's last.
__device__ __forceinline__ vec<uint32_t, 4> bytes16(const uint8_t* row, int b, int bytes, bool there) {
  vec<uint32_t, 4> v{};
  if (!there || b >= bytes) return v;
  if (b + 16 <= bytes) {
    __builtin_memcpy(&v, row + b, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 16; j++)
      if (b + j < bytes) v[j / 4] |= (uint32_t)row[b + j] << (j % 4 * 8);
  }
  return v;
}
// The four words that lanes l, l + 16, l + 32, l + 48 hold, turned: word i of lane 16 j + l becomes word j of lane 16 i + l.
__device__ __forceinline__ void turn4(vec<uint32_t, 4>& v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false), b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  v = {(uint32_t)c[0], (uint32_t)c[1], (uint32_t)d[0], (uint32_t)d[1]};
}
template <typename E, int N>
__device__ __forceinline__ vec<E, N> some(const E* row, int i, int count, bool there) {
  vec<E, N> v{};
  if (!there) return v;
  if (i + N <= count) {
    __builtin_memcpy(&v, row + i, sizeof(E) * N);
  } else {
#pragma unroll
    for (int j = 0; j < N; j++)
      if (i + j < count) v[j] = row[i + j];
  }
  return v;
}

// At most 16 MT rows of x. A workgroup takes 16 outputs, its eight waves every eighth run of 128 values of k: sixteen bytes of a row
// a lane, turned so that each matrix instruction meets 32 neighbouring values of k, which are of one group. With c the code and B its
// base, a group's sum is s (sum (B + c) x - (B + z) sum x), and sum x comes from the same instruction against ones, in the same lanes.
// B is at most 128, so that the difference costs four bits of the 24 that the sums are held in. The eight sums meet in LDS and are
// added in a fixed order.
template <typename T, int GROUP, bool ZERO, int MT>
__global__ __launch_bounds__(512) void q4_few_kernel(Weights4<T> w, Side<T> x, int64_t M, T* y, int64_t ldy) {
  constexpr int NG = GROUP >= 128 ? 1 : 128 / GROUP, PER = 4 / NG;  // groups of a run, matrix instructions of a group
  constexpr int U = 4;
  __shared__ f32x4 sums[8][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q4 = lane >> 4;
  const int64_t n = (int64_t)blockIdx.x * 16 + row;
  const bool there = n < w.rows;
  const int K = w.cols, bytes = (K + 1) / 2;
  const uint8_t* q = w.q + (there ? n : 0) * w.ldq;
  const T* scale = w.scale + (there ? n : 0) * w.lds;
  const uint8_t* zero = ZERO ? w.zero + (there ? n : 0) * w.ldz : nullptr;
  const T one = (T)1.f;
  const vec<T, 8> ones = {one, one, one, one, one, one, one, one};
  struct Run {
    vec<uint32_t, 4> q;
    vec<T, NG> s;
    vec<uint8_t, NG> z;
  };
  auto fetch = [&](int k0) {
    Run r;
    r.q = bytes16(q, k0 / 2 + q4 * 16, bytes, there && k0 < K);
    r.s = some<T, NG>(scale, k0 / GROUP, w.groups, there && k0 < K);
    if constexpr (ZERO) r.z = some<uint8_t, NG>(zero, k0 / GROUP, w.groups, there && k0 < K);
    return r;
  };
  f32x4 total[MT] = {};
  Run next[U];
#pragma unroll
  for (int u = 0; u < U; u++) next[u] = fetch((u * 8 + wave) * 128);
  for (int k0 = wave * 128; k0 < K; k0 += U * 1024) {
    Run now[U];
#pragma unroll
    for (int u = 0; u < U; u++) now[u] = next[u];
    if (k0 + U * 1024 < K) {
#pragma unroll
      for (int u = 0; u < U; u++) next[u] = fetch(k0 + (U + u) * 1024);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int k = k0 + u * 1024;
      if (k >= K) break;
      turn4(now[u].q);
#pragma unroll
      for (int g = 0; g < NG; g++) {
        f32x4 acc[MT] = {}, sum[MT] = {};
#pragma unroll
        for (int i = 0; i < PER; i++) {
          const vec<T, 8> p = codes<T>(now[u].q[g * PER + i]);
#pragma unroll
          for (int t = 0; t < MT; t++) {
            const int64_t m = t * 16 + row;
            const int at = k + (g * PER + i) * 32 + q4 * 8;
            const vec<T, 8> v = some<T, 8>(x.p + m * x.ld, at, K, m < M);
            acc[t] = mfma(v, p, acc[t]);
            sum[t] = mfma(v, ones, sum[t]);
          }
        }
        const float s = (float)now[u].s[g], b = Codes<T>::BASE + (ZERO ? (float)now[u].z[g] : 8.f);
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int j = 0; j < 4; j++) total[t][j] = fmaf(s, fmaf(-b, sum[t][j], acc[t][j]), total[t][j]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; t++) sums[wave][t][lane] = total[t];
  __syncthreads();
  if (wave >= MT) return;
  f32x4 v = sums[0][wave][lane];
#pragma unroll
  for (int i = 1; i < 8; i++) v += sums[i][wave][lane];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int64_t m = wave * 16 + q4 * 4 + j;
    if (m < M && there) y[m * ldy + n] = (T)v[j];
  }
}

// The weights in T, for the tiles, and x where its rows have to be copied to ones that start on 16 bytes. (code - zero) scale is formed in
// single precision and rounded once. Eight values a thread.
template <typename T, bool ZERO>
__global__ __launch_bounds__(256) void unpack_kernel(Weights4<T> w, int shift, T* to, int64_t pitch, uint32_t groups, uint32_t own,
                                                     Side<T> x, int64_t M, T* x_to) {
  uint32_t block = block_index();
  const bool copies = block >= own;
  if (copies) block -= own;
  const int64_t t = (int64_t)block * 256 + threadIdx.x, m = t / groups;
  const int n = (int)(t - m * groups) * 8;
  if (copies) {
    if (m >= M) return;
    *reinterpret_cast<vec<T, 8>*>(x_to + m * pitch + n) = some<T, 8>(x.p + m * x.ld, n, w.cols, true);
    return;
  }
  if (m >= w.rows) return;
  uint32_t word = 0;
  const uint8_t* q = w.q + m * w.ldq + n / 2;
  if (n + 8 <= w.cols) {
    __builtin_memcpy(&word, q, 4);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (n + 2 * j < w.cols) word |= (uint32_t)q[j] << (8 * j);
  }
  const int g = n >> shift;
  const float s = (float)w.scale[m * w.lds + g], z = ZERO ? (float)w.zero[m * w.ldz + g] : 8.f;
  vec<T, 8> v;
#pragma unroll
  for (int j = 0; j < 8; j++) v[j] = n + j < w.cols ? (T)(((float)(word >> (4 * j) & 15) - z) * s) : (T)0.f;
  *reinterpret_cast<vec<T, 8>*>(to + m * pitch + n) = v;
}

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

template <typename T>
struct Q4Plan {
  T *w = nullptr, *x = nullptr;
  int64_t pitch = 0;
  Way way{};
  void* sums = nullptr;
  Q4Plan(const b2c_q4_linear_args* a, Room& room) {
    if (a->rows <= kFewRows) return;
    pitch = up(a->d_in, 64);
    w = room.take<T>(a->d_out * pitch);
    if (!direct(a)) x = room.take<T>(a->rows * pitch);
    way = choose({{a->rows, a->d_out}}, pitch / 64, false, false);
    sums = room.take<char>(way.sums);
  }
};

template <typename T>
int linear(const b2c_q4_linear_args* a, hipStream_t stream) {
  const Weights4<T> w{a->w, a->ldw, (const T*)a->scale, a->lds, a->zero, a->ldz, a->d_out, a->d_in, groups_of(a->d_in, a->group)};
  Side<T> x{(const T*)a->x, a->ldx};
  if (a->rows <= kFewRows) {
    const dim3 grid((unsigned)(up(a->d_out, 16) / 16));
    return with_group(a->group, [&](auto group) -> int {
      constexpr int G = decltype(group)::value;
      auto run = [&](auto zero, auto tiles) {
        q4_few_kernel<T, G, decltype(zero)::value, decltype(tiles)::value><<<grid, 512, 0, stream>>>(w, x, a->rows, (T*)a->y, a->ldy);
      };
      using One = std::integral_constant<int, 1>;
      using Two = std::integral_constant<int, 2>;
      if (a->zero) a->rows <= 16 ? run(std::true_type{}, One{}) : run(std::true_type{}, Two{});
      else a->rows <= 16 ? run(std::false_type{}, One{}) : run(std::false_type{}, Two{});
      return hipGetLastError();
    });
  }
  Room room{(char*)a->workspace};
  const Q4Plan<T> p(a, room);
  const uint32_t pieces = (uint32_t)(up(a->d_in, 8) / 8);
  const int64_t own = up((int64_t)a->d_out * pieces, 256) / 256, copies = p.x ? up(a->rows * pieces, 256) / 256 : 0;
  if (own + copies > 0x7fffffff) return hipErrorInvalidValue;
  const int shift = a->group == 32 ? 5 : a->group == 64 ? 6 : a->group == 128 ? 7 : 8;
  if (a->zero) unpack_kernel<T, true><<<grid_of(own + copies), 256, 0, stream>>>(w, shift, p.w, p.pitch, pieces, (uint32_t)own, x, a->rows, p.x);
  else unpack_kernel<T, false><<<grid_of(own + copies), 256, 0, stream>>>(w, shift, p.w, p.pitch, pieces, (uint32_t)own, x, a->rows, p.x);
  int rc = hipGetLastError();
  if (rc) return rc;
  if (p.x) x = {p.x, p.pitch};
  const RowsOut<T> out{(T*)a->y, a->ldy, nullptr, 0, a->d_out, {}};
  const Product<T> product_of{x, {p.w, p.pitch}, {}, {}, a->rows, a->d_out, a->d_in, 0, a->rows, a->d_out};
  return product<T, false, false, false, false>(product_of, p.way, p.sums, out, stream);
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
      (need && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_bytes < need)))
    return hipErrorInvalidValue;
  return a->dtype == B2C_F16 ? linear<f16>(a, stream) : linear<bf16>(a, stream);
}
