// Products in 8-bit integers with a scale for each row and each channel (b2c_hip_quantize_rows, b2c_hip_i8_linear,
// b2c_hip_i8_ffn).
#include "dense_product.h"
#include "i8_head.h"
#include "i8_quant.h"

namespace b2c {
namespace dev {
namespace {

// Weights in 8 bits as the products read them: in place where rows start on 16 bytes (columns beyond the last meet zeros of
// the quantised rows), else copied to rows that do, in the launch that quantises x. A few rows read them anywhere.
struct Copy {
  const int8_t* from;
  int64_t ld, rows, pitch;
  int8_t* to;
  int cols;
  uint32_t groups, blocks;
};
struct Copies {
  Copy of[3]{};
  int n = 0;
  uint32_t blocks = 0;
};
__device__ __forceinline__ void copy_block(const Copy& c, uint32_t block) {
  const int64_t t = (int64_t)block * 256 + threadIdx.x, m = t / c.groups;
  if (m >= c.rows) return;
  const int n = (int)(t - m * c.groups) * 16;
  const int8_t* p = c.from + m * c.ld + n;
  vec<int8_t, 16> v{};
  if (n + 16 <= c.cols) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 16; j++)
      if (n + j < c.cols) v[j] = p[j];
  }
  *reinterpret_cast<vec<int8_t, 16>*>(c.to + m * c.pitch + n) = v;
}

// THREADS threads to a row, sixteen values each at a time. What they read first they keep (up to HELD times sixteen), so that a
// row is read once; the rest of a longer row is read again. A row's columns from cols to the next multiple of 16 become 0.
// Bound by memory: 4096 x 11264 in single precision 39 us, 5.9 TB/s, most of which the last-level cache gives.
// The workgroups from `own` on make a call's copies of weights: in a launch of their own they cost 1333 rows of 2050 -> 5001
// three of 33 us. Where there are none, a kernel that takes Nothing: each launch with the larger arguments costs half a
// microsecond more (1000 rows of 1024-2816: 37.2 us with two of them, 36.6 without).
struct Nothing {};
template <typename T, int THREADS, int HELD, typename With>
__global__ __launch_bounds__(256) void quantize_kernel(const T* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* q,
                                                       int64_t ldq, float* scale, uint32_t own, With copies) {
  __shared__ uint32_t part[4];
  const uint32_t block = block_index();
  if constexpr (std::is_same_v<With, Copies>) {
    if (block >= own) {  // each with an index of its own: for a variable one the compiler puts them into scratch memory
      const uint32_t b = block - own, b1 = copies.of[0].blocks, b2 = b1 + copies.of[1].blocks;
      if (b >= copies.blocks) return;
      if (b < b1) copy_block(copies.of[0], b);
      else if (b < b2) copy_block(copies.of[1], b - b1);
      else copy_block(copies.of[2], b - b2);
      return;
    }
  }
  const int t = threadIdx.x % THREADS;
  const int64_t m = (int64_t)block * (256 / THREADS) + threadIdx.x / THREADS;
  const bool there = m < rows;
  const T* row = x + (there ? m : 0) * ldx;
  auto load = [&](int64_t k) {
    vec<T, 16> v{};
    if (there && k + 16 <= cols) {
      __builtin_memcpy(&v, row + k, sizeof(v));
    } else if (there && k < cols) {
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (k + j < cols) v[j] = row[k + j];
    }
    return v;
  };
  uint32_t top = 0;
  auto highest = [&](const vec<T, 16>& v) {
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const uint32_t b = magnitude((float)v[j]);
      top = b > top ? b : top;
    }
  };
  vec<T, 16> held[HELD];
#pragma unroll
  for (int h = 0; h < HELD; h++) {
    held[h] = load((int64_t)(h * THREADS + t) * 16);
    highest(held[h]);
  }
  for (int64_t k = (int64_t)(HELD * THREADS + t) * 16; k < cols; k += THREADS * 16) highest(load(k));
#pragma unroll
  for (int o = 1; o < THREADS && o < 64; o *= 2) {
    const uint32_t b = __shfl_xor(top, o);
    top = b > top ? b : top;
  }
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; w++) top = part[w] > top ? part[w] : top;
  }
  const RowScale s(top);
  if (there && t == 0) scale[m] = s.scale;
  auto write = [&](int64_t k, const vec<T, 16>& v) {
    if (!there || k >= cols) return;
    vec<uint32_t, 4> b;
#pragma unroll
    for (int j = 0; j < 4; j++)
      b[j] = bytes4(s((float)v[4 * j]), s((float)v[4 * j + 1]), s((float)v[4 * j + 2]), s((float)v[4 * j + 3]));
    int8_t* to = q + m * ldq + k;
    if (k + 16 <= ldq) {
      __builtin_memcpy(to, &b, 16);
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (k + j < ldq) to[j] = (int8_t)(b[j / 4] >> (j % 4 * 8));
    }
  };
#pragma unroll
  for (int h = 0; h < HELD; h++) write((int64_t)(h * THREADS + t) * 16, held[h]);
  for (int64_t k = (int64_t)(HELD * THREADS + t) * 16; k < cols; k += THREADS * 16) write(k, load(k));
}

// Four lanes a row up to 128 columns, sixteen up to 1024, a wave or a workgroup beyond: whole rows in registers, and as few idle
// lanes as that allows (four waves a row of 64 took 600 us for a million of them).
template <typename T>
int quantize(const T* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* q, int64_t ldq, float* scale, const Copies& copies,
             hipStream_t stream) {
  constexpr int H = sizeof(T) == 4 ? 2 : 4;
  auto run = [&](auto threads, auto held) {
    constexpr int N = decltype(threads)::value;
    const uint32_t own = (uint32_t)(up(rows, 256 / N) / (256 / N));
    constexpr int HELD = decltype(held)::value;
    if (copies.blocks) quantize_kernel<T, N, HELD><<<grid_of((int64_t)own + copies.blocks), 256, 0, stream>>>(x, ldx, rows, cols, q, ldq, scale, own, copies);
    else quantize_kernel<T, N, HELD><<<grid_of(own), 256, 0, stream>>>(x, ldx, rows, cols, q, ldq, scale, own, Nothing{});
    return hipGetLastError();
  };
  using std::integral_constant;
  if (cols <= 128) return run(integral_constant<int, 4>{}, integral_constant<int, 2>{});
  if (cols <= 1024) return run(integral_constant<int, 16>{}, integral_constant<int, H>{});
  if (cols <= 4096 && rows >= 2048) return run(integral_constant<int, 64>{}, integral_constant<int, H>{});
  return run(integral_constant<int, 256>{}, integral_constant<int, H>{});
}
int quantize(const void* x, int64_t ldx, int dtype, int64_t rows, int64_t cols, int8_t* q, int64_t ldq, float* scale,
             hipStream_t stream, const Copies& copies = {}) {
  if (dtype == B2C_F32) return quantize((const float*)x, ldx, rows, cols, q, ldq, scale, copies, stream);
  if (dtype == B2C_F16) return quantize((const f16*)x, ldx, rows, cols, q, ldq, scale, copies, stream);
  return quantize((const bf16*)x, ldx, rows, cols, q, ldq, scale, copies, stream);
}

// A few rows of a product, quantised on the way: every workgroup takes all of x (at most kHeld values, which the caches hand
// out) to LDS in 8 bits, while the first of its weights are on their way, and then streams 16 rows of the weights (DUAL: of
// each of the two), every eighth 256-byte run a wave. One launch less than quantising first: 4096 -> 4096 for one row takes
// 7 us where two launches take 10.
constexpr int kHeld = 32768, kHeldRows = 8;
inline bool held(int64_t rows, int64_t cols) { return rows <= kHeldRows && rows * up(cols, 16) <= kHeld; }

template <typename TX, bool DUAL, typename Epi>
__global__ __launch_bounds__(512) void quantised_rows_kernel(const TX* x, int64_t ldx, Product<int8_t> a, Epi epi) {
  constexpr int PL = DUAL ? 2 : 1, RUN = 256;
  using A = vec<int8_t, 16>;
  __shared__ __attribute__((aligned(16))) int8_t qx[kHeld];
  __shared__ uint32_t tops[8][kHeldRows];
  __shared__ float scales[kHeldRows];
  __shared__ i32x4 sums[8][PL][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q4 = lane >> 4;
  const int64_t n = (int64_t)blockIdx.x * 16 + row;
  const int K = (int)a.K, M = (int)a.M, pitch = (K + 15) / 16 * 16;
  auto load = [&](const Side<int8_t>& s, int k) {
    A v{};
    if (n >= a.p_lim || k >= K) return v;
    const int8_t* p = s.p + n * s.ld + k;
    if (k + 16 <= K) {
      __builtin_memcpy(&v, p, 16);
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (k + j < K) v[j] = p[j];
    }
    return v;
  };
  A p[2][PL][4];
  auto fetch = [&](int b, int k0) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
      p[b][0][c] = load(a.p, k0 + (c * 4 + q4) * 16);
      if constexpr (DUAL) p[b][1][c] = load(a.p2, k0 + (c * 4 + q4) * 16);
    }
  };
  fetch(0, wave * RUN);

  auto values = [&](int m, int k) {
    vec<TX, 16> v{};
    const TX* from = x + m * ldx + k;
    if (k + 16 <= K) {
      __builtin_memcpy(&v, from, sizeof(v));
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (k + j < K) v[j] = from[j];
    }
    return v;
  };
  for (int m = 0; m < M; m++) {
    uint32_t top = 0;
    for (int k = (int)threadIdx.x * 16; k < K; k += 512 * 16) {
      const vec<TX, 16> v = values(m, k);
#pragma unroll
      for (int j = 0; j < 16; j++) top = magnitude((float)v[j]) > top ? magnitude((float)v[j]) : top;
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const uint32_t b = __shfl_xor(top, o);
      top = b > top ? b : top;
    }
    if (lane == 0) tops[wave][m] = top;
  }
  __syncthreads();
  for (int m = 0; m < M; m++) {
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < 8; w++) top = tops[w][m] > top ? tops[w][m] : top;
    const RowScale s(top);
    if (threadIdx.x == 0) scales[m] = s.scale;
    for (int k = (int)threadIdx.x * 16; k < K; k += 512 * 16) {
      const vec<TX, 16> v = values(m, k);
      vec<uint32_t, 4> b;
#pragma unroll
      for (int j = 0; j < 4; j++)
        b[j] = bytes4(s((float)v[4 * j]), s((float)v[4 * j + 1]), s((float)v[4 * j + 2]), s((float)v[4 * j + 3]));
      *reinterpret_cast<vec<uint32_t, 4>*>(qx + m * pitch + k) = b;
    }
  }
  __syncthreads();

  i32x4 acc[PL] = {};
  auto multiply = [&](int b, int k0) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int k = k0 + (c * 4 + q4) * 16;
      const A v = row < M && k < K ? *reinterpret_cast<const A*>(qx + row * pitch + k) : A{};
#pragma unroll
      for (int d = 0; d < PL; d++) acc[d] = mfma(p[b][d][c], v, acc[d]);
    }
  };
  for (int k0 = wave * RUN; k0 < K; k0 += 16 * RUN) {
    fetch(1, k0 + 8 * RUN);
    multiply(0, k0);
    fetch(0, k0 + 16 * RUN);
    multiply(1, k0 + 8 * RUN);
  }
#pragma unroll
  for (int d = 0; d < PL; d++) sums[wave][d][lane] = acc[d];
  __syncthreads();
  if (wave) return;
  i32x4 v[PL];
#pragma unroll
  for (int d = 0; d < PL; d++) {
    v[d] = sums[0][d][lane];
#pragma unroll
    for (int w = 1; w < 8; w++) v[d] += sums[w][d][lane];
  }
  const int n4 = (int)blockIdx.x * 16 + q4 * 4;
  if (row >= M || n4 >= a.N) return;
  epi.sx = scales;
  int g[4], u[4];
#pragma unroll
  for (int j = 0; j < 4; j++) g[j] = v[0][j], u[j] = v[PL - 1][j];
  if constexpr (DUAL) epi.template operator()<4>(0u, row, n4, g, u);
  else epi.template operator()<4>(0u, row, n4, g);
}
template <bool DUAL, typename Epi>
int quantised_rows(const void* x, int64_t ldx, int dtype, const Product<int8_t>& a, const Epi& epi, hipStream_t stream) {
  const dim3 grid((unsigned)(up(a.N, 16) / 16));
  if (dtype == B2C_F32) quantised_rows_kernel<float, DUAL><<<grid, 512, 0, stream>>>((const float*)x, ldx, a, epi);
  else if (dtype == B2C_F16) quantised_rows_kernel<f16, DUAL><<<grid, 512, 0, stream>>>((const f16*)x, ldx, a, epi);
  else quantised_rows_kernel<bf16, DUAL><<<grid, 512, 0, stream>>>((const bf16*)x, ldx, a, epi);
  return hipGetLastError();
}

bool type_ok(int t) { return t == B2C_F32 || t == B2C_F16 || t == B2C_BF16; }
size_t size_of(int t) { return t == B2C_F32 ? 4 : 2; }
bool room_ok(const void* p, size_t have, size_t need) {
  return have >= need && (need == 0 || (p && reinterpret_cast<uintptr_t>(p) % 16 == 0));
}
constexpr int MOST = 131072;  // 131072 products of at most 127 * 127 stay below 2^31
bool sizes_ok(const b2c_i8_linear_args* a) {
  return a && a->rows >= 0 && a->rows <= 0x7fffffff && a->d_in >= 1 && a->d_in <= MOST && a->d_out >= 1 && a->d_out <= (1 << 24) && type_ok(a->dtype);
}
bool sizes_ok(const b2c_i8_ffn_args* a) {
  return a && a->rows >= 0 && a->rows <= 0x7fffffff && a->d_in >= 1 && a->d_in <= MOST && a->d_hidden >= 1 && a->d_hidden <= MOST && a->d_out >= 1 &&
         a->d_out <= (1 << 24) && type_ok(a->dtype) && a->act >= B2C_ACT_SILU && a->act <= B2C_ACT_RELU;
}

struct Weights {
  Side<int8_t> from;
  int64_t rows;
  int cols;
  int8_t* copy = nullptr;
  int64_t pitch = 0;
  bool straight() const {
    return reinterpret_cast<uintptr_t>(from.p) % 16 == 0 && from.ld % 16 == 0 && cols % 16 == 0 && from.ld < (1 << 22);
  }
  void place(Room& room, bool stay) {
    if (stay) return;
    pitch = up(cols, 128);
    copy = room.take<int8_t>(rows * pitch);
  }
  Side<int8_t> side() const { return pitch ? Side<int8_t>{copy, pitch} : from; }
  void add_to(Copies& all) const {
    if (!pitch) return;
    const int64_t groups = up(cols, 16) / 16, blocks = up(rows * groups, 256) / 256;  // at most 2^24 rows of 8192 groups
    all.of[all.n++] = {from.p, from.ld, rows, pitch, copy, cols, (uint32_t)groups, (uint32_t)blocks};
    all.blocks += (uint32_t)blocks;
  }
};
int64_t steps_of(int64_t k) { return up(k, 128) / 128; }

struct LinearPlan {
  int64_t kp;
  int8_t* q;
  float* sx;
  Weights w;
  Way way;
  void* sums;
  LinearPlan(const b2c_i8_linear_args* a, Room& room) {
    kp = up(a->d_in, 128);
    q = room.take<int8_t>(a->rows * kp);
    sx = room.take<float>(a->rows);
    w = {{a->w, a->ldw}, a->d_out, a->d_in};
    const bool few = few_rows(a->rows, w.straight());
    way = choose({{a->rows, a->d_out}}, steps_of(a->d_in), false, few);
    w.place(room, few || w.straight());
    sums = room.take<char>(way.sums);
  }
};
struct BlockPlan {
  int64_t kp, fp;
  float *h, *s;  // s: of x's rows, then of h's
  int8_t *qx, *qh;
  Weights wg, wu, wd;
  Way gate, down;
  void* sums;
  BlockPlan(const b2c_i8_ffn_args* a, Room& room) {
    kp = up(a->d_in, 128);
    fp = up(a->d_hidden, 128);
    h = room.take<float>(a->rows * fp);
    qh = room.take<int8_t>(a->rows * fp);
    qx = room.take<int8_t>(a->rows * kp);
    s = room.take<float>(a->rows);
    wg = {{a->w_gate, a->ld_in}, a->d_hidden, a->d_in};
    wu = {{a->w_up, a->ld_in}, a->d_hidden, a->d_in};
    wd = {{a->w_down, a->ld_out}, a->d_out, a->d_hidden};
    const bool in = wg.straight() && wu.straight();  // both or none: the tiles read them with one distance between rows
    const bool few = few_rows(a->rows, in && wd.straight());
    gate = choose({{a->rows, a->d_hidden}}, steps_of(a->d_in), true, few, 4);
    down = choose({{a->rows, a->d_out}}, steps_of(a->d_hidden), false, few);
    wg.place(room, few || in);
    wu.place(room, few || in);
    wd.place(room, few || wd.straight());
    sums = room.take<char>(std::max(gate.sums, down.sums));
  }
};

// x, ldx, type: where the rows still have to be quantised (held()), else null
struct Raw {
  const void* x;
  int64_t ldx;
  int dtype;
};
template <typename T>
int scaled(const Product<int8_t>& p, const Way& way, void* sums, const float* sx, const float* sw, void* y, int64_t ldy,
           const Raw& raw, hipStream_t stream) {
  const ScaledOut<T> out{(T*)y, ldy, sx, sw, (int)p.N};
  if (raw.x) return quantised_rows<false>(raw.x, raw.ldx, raw.dtype, p, out, stream);
  return product<int8_t, false, false, false, false>(p, way, sums, out, stream);
}
int scaled(const Product<int8_t>& p, const Way& way, void* sums, const float* sx, const float* sw, int dtype, void* y,
           int64_t ldy, const Raw& raw, hipStream_t stream) {
  if (dtype == B2C_F32) return scaled<float>(p, way, sums, sx, sw, y, ldy, raw, stream);
  if (dtype == B2C_F16) return scaled<f16>(p, way, sums, sx, sw, y, ldy, raw, stream);
  return scaled<bf16>(p, way, sums, sx, sw, y, ldy, raw, stream);
}
template <int ACT>
int gated(const BlockPlan& p, const b2c_i8_ffn_args* a, const Raw& raw, hipStream_t stream) {
  const ScaledGate<ACT> out{p.h, p.s, a->s_gate, a->s_up, p.fp, a->d_hidden};
  const Product<int8_t> in{{p.qx, p.kp}, p.wg.side(), {}, p.wu.side(), a->rows, a->d_hidden, a->d_in, 0, a->rows, a->d_hidden};
  if (raw.x) return quantised_rows<true>(raw.x, raw.ldx, raw.dtype, in, out, stream);
  return product<int8_t, false, false, true, false>(in, p.gate, p.sums, out, stream);
}

}  // namespace
}  // namespace dev
}  // namespace b2c

using namespace b2c::dev;

extern "C" int b2c_hip_quantize_rows(const b2c_quantize_args* a, hipStream_t stream) {
  if (!a || a->rows < 0 || a->rows > 0x7fffffff || a->cols < 1 || !type_ok(a->dtype)) return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  if (!good(a->x, a->ldx, a->cols, size_of(a->dtype)) || !good(a->q, a->ldq, a->cols, 1) || !good(a->scale, 1, 1, 4))
    return hipErrorInvalidValue;
  return quantize(a->x, a->ldx, a->dtype, a->rows, a->cols, a->q, a->ldq, a->scale, stream);
}

extern "C" size_t b2c_i8_linear_workspace_bytes(const b2c_i8_linear_args* a) {
  if (!sizes_ok(a) || a->rows == 0 || is_i8_narrow(a)) return 0;
  Room room{nullptr};
  LinearPlan(a, room);
  return room.used;
}
extern "C" int b2c_hip_i8_linear(const b2c_i8_linear_args* a, hipStream_t stream) {
  if (!sizes_ok(a)) return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  if (!good(a->x, a->ldx, a->d_in, size_of(a->dtype)) || !good(a->w, a->ldw, a->d_in, 1) || !good(a->w_scale, 1, 1, 4) ||
      !good(a->y, a->ldy, a->d_out, size_of(a->dtype)) ||
      !room_ok(a->workspace, a->workspace_bytes, b2c_i8_linear_workspace_bytes(a)))
    return hipErrorInvalidValue;
  if (is_i8_narrow(a)) return i8_narrow(a, stream);
  Room room{(char*)a->workspace};
  const LinearPlan p(a, room);
  const Product<int8_t> out{{p.q, p.kp}, p.w.side(), {}, {}, a->rows, a->d_out, a->d_in, 0, a->rows, a->d_out};
  Raw raw{};
  if (p.way.tile == FEW_ROWS && held(a->rows, a->d_in)) {
    raw = {a->x, a->ldx, a->dtype};
  } else {
    Copies copies;
    p.w.add_to(copies);
    const int rc = quantize(a->x, a->ldx, a->dtype, a->rows, a->d_in, p.q, p.kp, p.sx, stream, copies);
    if (rc) return rc;
  }
  return scaled(out, p.way, p.sums, p.sx, a->w_scale, a->dtype, a->y, a->ldy, raw, stream);
}

extern "C" size_t b2c_i8_ffn_workspace_bytes(const b2c_i8_ffn_args* a) {
  if (!sizes_ok(a) || a->rows == 0) return 0;
  if (is_i8_head(a)) return i8_head_bytes(a);
  Room room{nullptr};
  BlockPlan(a, room);
  return room.used;
}
extern "C" int b2c_hip_i8_ffn(const b2c_i8_ffn_args* a, hipStream_t stream) {
  if (!sizes_ok(a)) return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  if (!good(a->x, a->ldx, a->d_in, size_of(a->dtype)) || !good(a->w_gate, a->ld_in, a->d_in, 1) ||
      !good(a->w_up, a->ld_in, a->d_in, 1) || !good(a->w_down, a->ld_out, a->d_hidden, 1) || !good(a->s_gate, 1, 1, 4) ||
      !good(a->s_up, 1, 1, 4) || !good(a->s_down, 1, 1, 4) || !good(a->y, a->ldy, a->d_out, size_of(a->dtype)) ||
      !room_ok(a->workspace, a->workspace_bytes, b2c_i8_ffn_workspace_bytes(a)))
    return hipErrorInvalidValue;
  if (is_i8_head(a)) return i8_head(a, stream);
  Room room{(char*)a->workspace};
  const BlockPlan p(a, room);
  int rc = hipSuccess;
  Raw raw{};
  if (p.gate.tile == FEW_ROWS && held(a->rows, a->d_in)) {
    raw = {a->x, a->ldx, a->dtype};
  } else {
    Copies copies;
    for (const Weights* w : {&p.wg, &p.wu, &p.wd}) w->add_to(copies);
    rc = quantize(a->x, a->ldx, a->dtype, a->rows, a->d_in, p.qx, p.kp, p.s, stream, copies);
    if (rc) return rc;
  }
  if (a->act == B2C_ACT_SILU) rc = gated<B2C_ACT_SILU>(p, a, raw, stream);
  else if (a->act == B2C_ACT_GELU) rc = gated<B2C_ACT_GELU>(p, a, raw, stream);
  else rc = gated<B2C_ACT_RELU>(p, a, raw, stream);
  if (rc) return rc;
  raw = {};
  if (p.down.tile == FEW_ROWS && held(a->rows, a->d_hidden)) raw = {p.h, p.fp, B2C_F32};
  else if ((rc = quantize(p.h, p.fp, B2C_F32, a->rows, a->d_hidden, p.qh, p.fp, p.s, stream))) return rc;
  const Product<int8_t> out{{p.qh, p.fp}, p.wd.side(), {}, {}, a->rows, a->d_out, a->d_hidden, 0, a->rows, a->d_out};
  return scaled(out, p.down, p.sums, p.s, a->s_down, a->dtype, a->y, a->ldy, raw, stream);
}
