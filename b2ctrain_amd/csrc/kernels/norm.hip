// The norms, gate and residual sum between two blocks, and their gradients (b2c_hip_block_norm, b2c_hip_block_norm_backward).
#include "dense_rows.h"

namespace b2c {
namespace dev {
namespace {

// A team of LANES threads holds a row in registers, C pieces of sixteen bytes each, so that every matrix is read once, whatever
// statistics the row needs: thread t has columns (c LANES + t) E .. + E - 1. Teams of up to 64 threads share a wave, larger ones are a
// workgroup.
template <int LANES>
struct Team {
  static constexpr int THREADS = LANES > 64 ? LANES : 256, TEAMS = THREADS / LANES, WAVES = THREADS / 64;
  int flip = 0;

  template <int CTRL>
  static __device__ __forceinline__ float add_dpp(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
  }
  // The sum over the team, to all of it. Every thread of a workgroup takes part. `room`: two rows of 16 values, used in turn, so that one
  // barrier a sum is enough.
  __device__ __forceinline__ float sum(float v, float (&room)[2][16]) {
    if constexpr (LANES >= 2) v = add_dpp<0xB1>(v);   // quad_perm:[1,0,3,2]
    if constexpr (LANES >= 4) v = add_dpp<0x4E>(v);   // quad_perm:[2,3,0,1]
    if constexpr (LANES >= 8) v = add_dpp<0x141>(v);  // row_half_mirror
    if constexpr (LANES >= 16) v = add_dpp<0x140>(v); // row_mirror
    if constexpr (LANES >= 32) {
      const uint32_t b = __builtin_bit_cast(uint32_t, v);
      const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
      v = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    }
    if constexpr (LANES >= 64) {
      const uint32_t b = __builtin_bit_cast(uint32_t, v);
      const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
      v = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    }
    if constexpr (LANES > 64) {
      if ((threadIdx.x & 63) == 0) room[flip][threadIdx.x >> 6] = v;
      __syncthreads();
      v = room[flip][0];
#pragma unroll
      for (int w = 1; w < WAVES; w++) v += room[flip][w];
      flip ^= 1;
    }
    return v;
  }
};

// How rows end: at a piece's end, inside a piece, or before the first one's.
enum { WHOLE, RAGGED, SHORT };

// E neighbouring values of a row as they are held in memory: first what a load without conditions gives, and by settle() when it is used,
// since a use would wait for the load, those that are there and zeros. A piece that is not there reads the row's first in its place, one
// inside which the row ends the row's last E values.
template <int E, int END, typename T>
__device__ __forceinline__ vec<T, E> piece(const T* row, int n, int cols) {
  vec<T, E> v{};
  if constexpr (END == SHORT) {
    if (n == 0) {
#pragma unroll
      for (int j = 0; j < E; j++) v[j] = row[j < cols ? j : 0];
    }
  } else {
    __builtin_memcpy(&v, row + (END == WHOLE ? (n < cols ? n : 0) : (n < cols - E ? n : cols - E)), sizeof(v));
  }
  return v;
}
template <int E, int END, typename T>
__device__ __forceinline__ void settle(vec<T, E>& v, int n, int cols, bool there) {
  if constexpr (END == RAGGED) {
    const int by = (n - (n < cols - E ? n : cols - E)) * (int)sizeof(T);
    if constexpr (sizeof(v) == 16) {
      v = __builtin_bit_cast(vec<T, E>, moved_down(__builtin_bit_cast(vec<uint32_t, 4>, v), by));
    } else {
      const uint64_t w = __builtin_bit_cast(uint64_t, v);
      v = __builtin_bit_cast(vec<T, E>, by < 8 ? w >> (8 * by) : 0);
    }
    if (!there) v = vec<T, E>{};
  } else {
#pragma unroll
    for (int j = 0; j < E; j++) v[j] = there && (END == WHOLE ? n : n + j) < cols ? v[j] : (T)0.f;
  }
}
template <int E, int END, typename T>
__device__ __forceinline__ void put_piece(T* row, int n, int cols, bool there, const float (&v)[E]) {
  if constexpr (END == WHOLE) {
    vec<T, E> t;
#pragma unroll
    for (int j = 0; j < E; j++) t[j] = (T)v[j];
    if (there && n < cols) __builtin_memcpy(row + n, &t, sizeof(t));
  } else if (there) {
    put<E>(row, 0, 0, n, cols, v);
  }
}
// A norm's weights: ones without any, zeros beyond the last column.
template <int E, typename T>
__device__ __forceinline__ void weights(const void* w, bool f32, int n, int cols, float (&v)[E]) {
#pragma unroll
  for (int j = 0; j < E; j++) v[j] = n + j < cols ? 1.f : 0.f;
  if (!w) return;
  if (f32) get<E>((const float*)w, 0, 0, n, cols, v);
  else get<E>((const T*)w, 0, 0, n, cols, v);
}

struct NormArgs {
  int64_t rows;
  int cols;
  bool centre, post, sigmoid, w_f32;
  float eps, scale, inv_cols, part, of_parts;  // part: a power of two of at most one over the columns; of_parts part = inv_cols
  const void *x, *r, *g, *w_post, *w_pre;
  int64_t ldx, ldr, ldg;
  uint32_t per_gate;
  void *y, *n;
  int64_t ldy, ldn;
};

// norm(v) in `u`; returns one over its size. The sums for a mean are of the values times `part`, so that they stay in range as the row does.
// Rows whose squares pass single precision's range, and small ones with next to no eps, are multiplied by a power of two and summed again: TIGHT
// in a loop, whose code stands once, else behind a branch. The loop keeps the largest teams' gradients from spilling (bf16 2048 x 8192 takes
// 82 us with the branch, 53 with the loop, 1000 x 16384 153 and 120), and costs others time (forward a million rows of 64 99 and 105).
template <bool TIGHT, int LANES, int C, int E>
__device__ __forceinline__ float normalise(const NormArgs& a, Team<LANES>& team, float (&room)[2][16], int first, float (&u)[C][E]) {
  if (a.centre) {
    float s = 0;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int j = 0; j < E; j++) s = fmaf(u[c][j], a.part, s);
    const float mean = team.sum(s, room) * a.of_parts;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int j = 0; j < E; j++) u[c][j] = first + c * LANES * E + j < a.cols ? u[c][j] - mean : 0.f;
  }
  auto squares = [&] {
    float s = 0;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int j = 0; j < E; j++) s = fmaf(u[c][j], u[c][j], s);
    return team.sum(s, room);
  };
  auto times = [&](float by) {
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int j = 0; j < E; j++) u[c][j] *= by;
  };
  float s, by = 1.f, eps = a.eps;
  auto beyond = [&] { return !(s < __builtin_inff()) || (s < 0x1p-96f && eps < 0x1p-80f); };  // the whole team's answer
  auto scale = [&] {
    by = s < 1.f ? 0x1p100f : 0x1p-72f;
    eps = eps * by * by;
    times(by);
  };
  if constexpr (TIGHT) {
#pragma unroll 1
    for (;;) {
      s = squares();
      if (by != 1.f || !beyond()) break;
      scale();
    }
  } else {
    s = squares();
    if (beyond()) {
      scale();
      s = squares();
    }
  }
  const float size = rsqrtf(fmaf(s, a.inv_cols, eps));
  times(size);
  return size * by;
}

// A row's pieces, where the matrix is given.
template <int E, int END, int LANES, typename T, int C>
__device__ __forceinline__ void read(vec<T, E> (&v)[C], const void* p, int64_t at, int first, int cols) {
  if (!p) return;
#pragma unroll
  for (int c = 0; c < C; c++) v[c] = piece<E, END>((const T*)p + at, first + c * LANES * E, cols);
}
// act(gate). Of 16-bit gates by the hardware's approximations, which are off by 2^-22, and by |g| 2^-24 for the exponential's argument.
template <typename T>
__device__ __forceinline__ float act_of(bool sigmoid, float g) {
  if (!sigmoid) return g;
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-g));
  return __builtin_amdgcn_rcpf(1.f + __expf(-g));
}
// A gate as the gradients keep it: itself, or, of a sigmoid, the smaller of it and what it is short of one, with a sign bit where that is the
// second, so that neither cancels in its slope, their product.
template <typename T>
__device__ __forceinline__ float kept_gate(bool sigmoid, float g) {
  if (!sigmoid) return g;
  const float small = act_of<T>(true, -fabsf(g));
  return g < 0.f ? small : -small;
}
__device__ __forceinline__ float gate_of(bool sigmoid, float kept) {
  return sigmoid && __builtin_bit_cast(int, kept) < 0 ? 1.f + kept : kept;
}
__device__ __forceinline__ float slope_of(bool sigmoid, float kept) { return sigmoid ? fabsf(kept) * (1.f - fabsf(kept)) : 1.f; }

// Both norms of a row from registers: t = u / size(u), y = r + scale gate t w_post, n = y / size(y) w_pre, with y as it was before it was
// rounded; the sums of layer norms are of differences from the mean, in a second pass over registers. Bound by memory: 8192 rows of 4096
// with a gate a row (bf16, 336 MB) take 63 to 66 us, 5.1 TB/s, a million rows of 64 (512 MB) 92 us, 5.5 TB/s, one row of 4096 2.8 us.
template <typename T, int E, int LANES, int C, int END>
__global__ __launch_bounds__(Team<LANES>::THREADS) void norm_kernel(NormArgs a) {
  constexpr int TEAMS = Team<LANES>::TEAMS;
  __shared__ float room[2][16];
  Team<LANES> team;
  const int first = (threadIdx.x % LANES) * E, mine = threadIdx.x / LANES;
  float wa[C][E], wb[C][E];
#pragma unroll
  for (int c = 0; c < C; c++) {
    weights<E, T>(a.w_post, a.w_f32, first + c * LANES * E, a.cols, wa[c]);
    weights<E, T>(a.w_pre, a.w_f32, first + c * LANES * E, a.cols, wb[c]);
  }
  for (int64_t base = (int64_t)blockIdx.x * TEAMS; base < a.rows; base += (int64_t)gridDim.x * TEAMS) {
    const bool there = base + mine < a.rows;
    const int64_t m = there ? base + mine : a.rows - 1;  // rows behind the last take its values, and are not stored
    vec<T, E> x[C] = {}, r[C] = {}, g[C] = {};
    read<E, END, LANES, T>(x, a.x, m * a.ldx, first, a.cols);
    read<E, END, LANES, T>(r, a.r, m * a.ldr, first, a.cols);
    if (a.g) read<E, END, LANES, T>(g, a.g, (uint32_t)m / a.per_gate * a.ldg, first, a.cols);
#pragma unroll
    for (int c = 0; c < C; c++) {
      settle<E, END>(x[c], first + c * LANES * E, a.cols, true);
      settle<E, END>(r[c], first + c * LANES * E, a.cols, true);
      if (END != RAGGED || a.g) settle<E, END>(g[c], first + c * LANES * E, a.cols, true);  // an infinity times no x would be a NaN
    }
    float u[C][E];
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int j = 0; j < E; j++) u[c][j] = (float)x[c][j];
    if (a.post) normalise<false>(a, team, room, first, u);
#pragma unroll
    for (int c = 0; c < C; c++) {
#pragma unroll
      for (int j = 0; j < E; j++) {
        const float gate = a.g ? act_of<T>(a.sigmoid, (float)g[c][j]) : 1.f;
        u[c][j] = fmaf(a.scale * gate, u[c][j] * wa[c][j], (float)r[c][j]);  // without x: the residual, since u is 0
      }
      if (a.y) put_piece<E, END>((T*)a.y + m * a.ldy, first + c * LANES * E, a.cols, there, u[c]);
    }
    if (!a.n) continue;
    normalise<false>(a, team, room, first, u);
#pragma unroll
    for (int c = 0; c < C; c++) {
#pragma unroll
      for (int j = 0; j < E; j++) u[c][j] *= wb[c][j];
      put_piece<E, END>((T*)a.n + m * a.ldn, first + c * LANES * E, a.cols, there, u[c]);
    }
  }
}

// How the backward pass walks the rows: `groups` of `per` rows, each in `segments` of `rows`, one unit after the other in steps of the
// grid. A gate row that several rows share is a group; else all rows are one.
struct Walk {
  uint32_t groups, per, segments, rows, blocks;
};
struct NormGradArgs {
  NormArgs f;
  Walk walk;
  const void *dy, *dn;
  int64_t lddy, lddn;
  void *dx, *dr, *dg;
  int64_t lddx, lddr, lddg;
  float* w_parts;     // [blocks][2][cols]: of w_post, of w_pre; null: neither is wanted
  float* gate_parts;  // [units][cols]; null: a unit is a group, and writes its sum itself
  bool shared;        // the gate's gradient is summed over a unit's rows
};

// The sums of a workgroup's teams, which wave 0 (or, with one team, every thread) has afterwards. In a fixed order.
template <int LANES, int C, int E>
__device__ __forceinline__ void gather(float (&v)[C][E], float* lds) {
  if constexpr (LANES <= 64) {
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int j = 0; j < E; j++)
#pragma unroll
        for (int o = LANES; o < 64; o *= 2) v[c][j] += __shfl_xor(v[c][j], o);
    constexpr int W = LANES * C * E;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    if (wave > 0 && lane < LANES) {
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int j = 0; j < E; j++) lds[(wave - 1) * W + (c * E + j) * LANES + lane] = v[c][j];
    }
    __syncthreads();
    if (wave == 0 && lane < LANES) {
#pragma unroll
      for (int w = 0; w < 3; w++)
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int j = 0; j < E; j++) v[c][j] += lds[w * W + (c * E + j) * LANES + lane];
    }
  }
}

// With yh = y / size(y) and a = dn w_pre, the gradient of y is dy + (a - [mean a] - yh mean(a yh)) / size(y), and that of x the same of
// scale act(gate) times it, with w_post and size(x). y is formed again from x and the residual: to keep it and both sizes would save
// arithmetic that memory hides and cost the forward pass a write where y is not wanted. A thread sums its columns' weight gradients over
// all rows of its workgroup, in registers. A row's values are on their way while the one before is at work (AHEAD) where a compute unit
// has one workgroup, whose waves wait for each other at every sum. Bound by memory: 8192 rows of 4096 with a gate a row
// (bf16, 537 MB) take 114 us, 4.7 TB/s; a million rows of 64 (768 MB) 168 to 178 us, 4.5 TB/s, VALU 73%.
template <typename T, int E, int LANES, int C, int END>
__global__ __launch_bounds__(Team<LANES>::THREADS) void norm_back_kernel(NormGradArgs b) {
  constexpr bool AHEAD = LANES > 64 && LANES <= 512;
  constexpr int TEAMS = Team<LANES>::TEAMS;
  __shared__ float room[2][16];
  __shared__ float lds[LANES <= 64 ? 3 * LANES * C * E : 1];
  const NormArgs& a = b.f;
  Team<LANES> team;
  const int first = (threadIdx.x % LANES) * E, mine = threadIdx.x / LANES;
  const bool writes = LANES > 64 || threadIdx.x < LANES;  // what gather() leaves
  // The largest teams have 128 registers a thread. Where it holds sixteen of a row's values, they take all of them: the weights are read again
  // for each row, and the sums of their gradients stay in LDS, each thread's own (us so and in registers: bf16 1000 x 16384 120 and 155, f32
  // 600 x 16384 122 and 143; with eight values bf16 2048 x 8192 64 and 53, 2000 x 5001 60 and 57, f32 2048 x 8192 101 and 94).
  constexpr bool WIDE = C * E > 8;
  __shared__ float held[2][WIDE ? C * E * LANES : 1];
  float wa[C][E], wb[C][E], sa[C][E] = {}, sb[C][E] = {};
  if constexpr (WIDE) {
    for (int i = 0; i < C * E; i++) held[0][i * LANES + threadIdx.x] = held[1][i * LANES + threadIdx.x] = 0.f;
  } else {
#pragma unroll
    for (int c = 0; c < C; c++) {
      weights<E, T>(a.w_post, a.w_f32, first + c * LANES * E, a.cols, wa[c]);
      weights<E, T>(a.w_pre, a.w_f32, first + c * LANES * E, a.cols, wb[c]);
    }
  }
  const uint32_t units = b.walk.groups * b.walk.segments;
  struct Raw {
    vec<T, E> x[C], r[C], g[C], dy[C], dn[C];
  };
  // Rows behind the last take its values with gradients of zero, which add nothing to any sum.
  auto fetch = [&](Raw& w, int64_t base, int64_t end) {
    const bool there = base + mine < end;
    const int64_t m = there ? base + mine : end - 1;
    read<E, END, LANES, T>(w.x, a.x, m * a.ldx, first, a.cols);
    read<E, END, LANES, T>(w.r, a.r, m * a.ldr, first, a.cols);
    if (a.g) read<E, END, LANES, T>(w.g, a.g, (uint32_t)m / a.per_gate * a.ldg, first, a.cols);
    read<E, END, LANES, T>(w.dy, b.dy, m * b.lddy, first, a.cols);
    read<E, END, LANES, T>(w.dn, b.dn, m * b.lddn, first, a.cols);
  };
  for (uint32_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const uint32_t group = unit / b.walk.segments, segment = unit - group * b.walk.segments;
    const int64_t start = (int64_t)group * b.walk.per, last = start + b.walk.per < a.rows ? start + b.walk.per : a.rows;
    const int64_t begin = start + (int64_t)segment * b.walk.rows, end = begin + b.walk.rows < last ? begin + b.walk.rows : last;
    float sg[C][E] = {};
    Raw next{};
    if (AHEAD && begin < end) fetch(next, begin, end);
    for (int64_t base = begin; base < end; base += TEAMS) {
      const int64_t m = base + mine;
      const bool there = m < end;
      Raw w{};
      if constexpr (AHEAD) {
        w = next;
        if (base + TEAMS < end) fetch(next, base + TEAMS, end);
      } else {
        fetch(w, base, end);
      }
#pragma unroll
      for (int c = 0; c < C; c++) {
        const int n = first + c * LANES * E;
        settle<E, END>(w.x[c], n, a.cols, true);
        settle<E, END>(w.r[c], n, a.cols, true);
        if (END != RAGGED || a.g) settle<E, END>(w.g[c], n, a.cols, true);
        settle<E, END>(w.dy[c], n, a.cols, there);
        settle<E, END>(w.dn[c], n, a.cols, there);
      }
      float u[C][E], d[C][E];
      float size_x = 1.f;
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int j = 0; j < E; j++) {
          u[c][j] = (float)w.x[c][j];
          d[c][j] = (float)w.dy[c][j];
        }
      if (a.post) size_x = normalise<LANES == 1024>(a, team, room, first, u);
      if constexpr (WIDE) {
#pragma unroll
        for (int c = 0; c < C; c++) weights<E, T>(a.w_post, a.w_f32, first + c * LANES * E, a.cols, wa[c]);
      }
      float gate[C][E];
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int j = 0; j < E; j++) gate[c][j] = a.g ? kept_gate<T>(a.sigmoid, (float)w.g[c][j]) : 1.f;
      if (b.dn) {
        float v[C][E];
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int j = 0; j < E; j++) v[c][j] = fmaf(a.scale * gate_of(a.sigmoid, gate[c][j]), u[c][j] * wa[c][j], (float)w.r[c][j]);
        const float size = normalise<LANES == 1024>(a, team, room, first, v);
        if constexpr (WIDE) {
#pragma unroll
          for (int c = 0; c < C; c++) weights<E, T>(a.w_pre, a.w_f32, first + c * LANES * E, a.cols, wb[c]);
        }
        float along = 0, mean = 0;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int j = 0; j < E; j++) {
            const float n = (float)w.dn[c][j];
            float& sum = WIDE ? held[1][WIDE ? (c * E + j) * LANES + threadIdx.x : 0] : sb[c][j];
            sum = fmaf(n, v[c][j], sum);
            along = fmaf(n * wb[c][j], v[c][j], along);
            mean = fmaf(n, wb[c][j], mean);
          }
        along = team.sum(along, room) * a.inv_cols;
        mean = a.centre ? team.sum(mean, room) * a.inv_cols : 0.f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int j = 0; j < E; j++)
            d[c][j] = fmaf(size, fmaf(-v[c][j], along, fmaf((float)w.dn[c][j], wb[c][j], -mean)), d[c][j]);
      }
      if (b.dr) {
#pragma unroll
        for (int c = 0; c < C; c++) put_piece<E, END>((T*)b.dr + m * b.lddr, first + c * LANES * E, a.cols, there, d[c]);
      }
      if (!a.x) continue;
      if (b.dg) {
        float dg[C][E];
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int j = 0; j < E; j++) dg[c][j] = a.scale * d[c][j] * (u[c][j] * wa[c][j]) * slope_of(a.sigmoid, gate[c][j]);
#pragma unroll
        for (int c = 0; c < C; c++) {
          if (b.shared) {
#pragma unroll
            for (int j = 0; j < E; j++) sg[c][j] += dg[c][j];
          } else {
            put_piece<E, END>((T*)b.dg + m * b.lddg, first + c * LANES * E, a.cols, there, dg[c]);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int j = 0; j < E; j++) {
          float kept = gate[c][j];
          asm("" : "+v"(kept));  // formed again: the compiler would hold the gate from its first use on, beside what it is kept as
          d[c][j] *= a.scale * gate_of(a.sigmoid, kept);
        }
      if (a.post) {
        float along = 0, mean = 0;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int j = 0; j < E; j++) {
            float& sum = WIDE ? held[0][WIDE ? (c * E + j) * LANES + threadIdx.x : 0] : sa[c][j];
            sum = fmaf(d[c][j], u[c][j], sum);
            d[c][j] *= wa[c][j];
            along = fmaf(d[c][j], u[c][j], along);
            mean += d[c][j];
          }
        along = team.sum(along, room) * a.inv_cols;
        mean = a.centre ? team.sum(mean, room) * a.inv_cols : 0.f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int j = 0; j < E; j++) d[c][j] = size_x * (fmaf(-u[c][j], along, d[c][j]) - mean);
      }
      if (b.dx) {
#pragma unroll
        for (int c = 0; c < C; c++) put_piece<E, END>((T*)b.dx + m * b.lddx, first + c * LANES * E, a.cols, there, d[c]);
      }
    }
    if (b.shared) {
      gather<LANES, C, E>(sg, lds);
      if (writes) {
#pragma unroll
        for (int c = 0; c < C; c++) {
          const int n = first + c * LANES * E;
          if (b.gate_parts) put_piece<E, END>(b.gate_parts + (int64_t)unit * a.cols, n, a.cols, true, sg[c]);
          else put_piece<E, END>((T*)b.dg + (int64_t)group * b.lddg, n, a.cols, true, sg[c]);
        }
      }
    }
  }
  if (!b.w_parts) return;
  if constexpr (WIDE) {
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int j = 0; j < E; j++) {
        sa[c][j] = held[0][(c * E + j) * LANES + threadIdx.x];
        sb[c][j] = held[1][(c * E + j) * LANES + threadIdx.x];
      }
  }
  gather<LANES, C, E>(sa, lds);
  gather<LANES, C, E>(sb, lds);
  if (writes) {
    float* to = b.w_parts + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int c = 0; c < C; c++) {
      put_piece<E, END>(to, first + c * LANES * E, a.cols, true, sa[c]);
      put_piece<E, END>(to + a.cols, first + c * LANES * E, a.cols, true, sb[c]);
    }
  }
}

// out[job][n] = the sum of `parts` rows of single-precision sums, which lie `step` apart, in 64 bits and a fixed order: 32 columns a workgroup, a
// thirty-second of the parts a thread. Jobs 0 and 1 are the weights, the others the gate's rows. Adding in a launch of its own keeps the
// order, which atomics would not; it takes 5 us for 256 workgroups' sums of 4096 columns (8 MB), most of it the launch and two round trips.
struct JoinArgs {
  const float *w_parts, *gate_parts;
  int cols;
  uint32_t tiles, w_count, g_count, w_jobs;
  void *dw[2], *dg;
  int64_t lddg;
  bool w_f32, accumulate;
};
template <typename T>
__global__ __launch_bounds__(1024) void norm_join_kernel(JoinArgs a) {
  __shared__ double sums[32][33];
  const uint32_t block = block_index(), job = block / a.tiles;
  const int col = threadIdx.x & 31, part = threadIdx.x >> 5, n = (int)(block - job * a.tiles) * 32 + col;
  const bool weight = job < a.w_jobs;
  if (weight && !a.dw[job]) return;
  if (!weight && !a.dg) return;
  const uint32_t count = weight ? a.w_count : a.g_count;
  const int64_t step = weight ? 2 * (int64_t)a.cols : a.cols;
  const float* from = weight ? a.w_parts + job * (int64_t)a.cols : a.gate_parts + (int64_t)(job - a.w_jobs) * a.g_count * a.cols;
  double s = 0;
  if (n < a.cols) {
    uint32_t p = part;
    for (; p + 7 * 32 < count; p += 8 * 32) {  // eight loads on their way
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = from[(p + i * 32) * step + n];
#pragma unroll
      for (int i = 0; i < 8; i++) s += v[i];
    }
    for (; p < count; p += 32) s += from[p * step + n];
  }
  sums[part][col] = s;
  __syncthreads();
  if (part || n >= a.cols) return;
#pragma unroll
  for (int p = 1; p < 32; p++) s += sums[p][col];
  if (!weight) {
    ((T*)a.dg)[(int64_t)(job - a.w_jobs) * a.lddg + n] = (T)(float)s;
  } else if (a.w_f32) {
    float* to = (float*)a.dw[job] + n;
    *to = (float)(a.accumulate ? *to + s : s);
  } else {
    ((T*)a.dw[job])[n] = (T)(float)s;
  }
}

// ---- host --------------------------------------------------------------------------------------------------

size_t size_of(int dtype) { return dtype == B2C_F32 ? 4 : 2; }

bool sizes_ok(const b2c_block_norm_args* a) {
  return a && a->rows >= 0 && a->rows <= (1 << 30) && a->cols >= 1 && a->cols <= 16384 && a->dtype >= B2C_F32 && a->dtype <= B2C_BF16 &&
         (a->w_dtype == a->dtype || a->w_dtype == B2C_F32) && (a->kind == B2C_NORM_RMS || a->kind == B2C_NORM_LAYER) &&
         (a->gate_act == B2C_GATE_NONE || a->gate_act == B2C_GATE_SIGMOID) && a->eps >= 0 && a->eps < __builtin_inff() &&
         (!a->gate || a->rows_per_gate >= 1) && (a->post || !a->w_post);
}
bool inputs_ok(const b2c_block_norm_args* a) {  // of some rows: those of none have no address
  const size_t s = size_of(a->dtype), w = size_of(a->w_dtype);
  return (a->x || a->residual) && (a->x || (!a->post && !a->gate)) && (!a->x || good(a->x, a->ldx, a->cols, s)) &&
         (!a->residual || good(a->residual, a->ldr, a->cols, s)) &&
         (!a->gate || good(a->gate, a->ldg, a->cols, s)) && reinterpret_cast<uintptr_t>(a->w_post) % w == 0 &&
         reinterpret_cast<uintptr_t>(a->w_pre) % w == 0;
}

NormArgs to_device(const b2c_block_norm_args* a) {
  const int64_t per = a->gate ? std::min<int64_t>(a->rows_per_gate, 1 << 30) : 1;
  float part = 1.f;
  while (part * (float)a->cols > 1.f) part *= 0.5f;
  return {a->rows, a->cols, a->kind == B2C_NORM_LAYER, a->post != 0, a->gate && a->gate_act == B2C_GATE_SIGMOID, a->w_dtype == B2C_F32,
          a->eps, a->x ? a->scale : 0.f, 1.f / (float)a->cols, part, 1.f / (part * (float)a->cols), a->x, a->residual, a->gate, a->w_post,
          a->w_pre, a->ldx, a->ldr, a->ldg, (uint32_t)per, a->y, a->n, a->ldy, a->ldn};
}

// Calls f(lanes, pieces) with the team that a row of `cols` values takes, E to a piece.
template <int E, typename F>
int with_team(int cols, F f) {
  using std::integral_constant;
  const int pieces = (cols + E - 1) / E;
  if (pieces <= 8) return f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  if (pieces <= 16) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  if (pieces <= 32) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  if (pieces <= 64) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  if (pieces <= 128) return f(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  if (pieces <= 256) return f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  if (pieces <= 512) return f(integral_constant<int, 512>{}, integral_constant<int, 1>{});
  if (pieces <= 1024) return f(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
  if (pieces <= 2048) return f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
  if constexpr (E == 4) return f(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
  return hipErrorInvalidValue;
}

// Calls f(values of a piece, lanes, pieces, how rows end). Of 16-bit values a piece holds eight, or four where that keeps more rows on
// their way: in the backward pass up to 2048 columns (a million rows of 64: 168 us in place of 195 with 100 registers for 160; 4096 rows
// of 1024: 16.5 and 19.7; but 8192 rows of 4096 144 and 114), and where only four divide the columns.
template <typename T, typename F>
int with_rows(int cols, bool back, F f) {
  using std::integral_constant;
  auto with = [&](auto values) {
    constexpr int E = decltype(values)::value;
    return with_team<E>(cols, [&](auto lanes, auto pieces) -> int {
      if (cols % E == 0) return f(values, lanes, pieces, integral_constant<int, WHOLE>{});
      if (cols > E) return f(values, lanes, pieces, integral_constant<int, RAGGED>{});
      if constexpr (decltype(lanes)::value == 8) return f(values, lanes, pieces, integral_constant<int, SHORT>{});
      return hipErrorInvalidValue;
    });
  };
  if constexpr (sizeof(T) == 2) {
    if (cols <= 2048 && (back || (cols % 8 && cols % 4 == 0))) return with(integral_constant<int, 4>{});
  }
  return with(integral_constant<int, 16 / sizeof(T)>{});
}
template <typename T>
int forward(const b2c_block_norm_args* a, hipStream_t stream) {
  const NormArgs d = to_device(a);
  return with_rows<T>(a->cols, false, [&](auto values, auto lanes, auto pieces, auto ends) -> int {
    using L = Team<decltype(lanes)::value>;
    const int64_t blocks = std::min<int64_t>(up(a->rows, L::TEAMS) / L::TEAMS, 256 * (2048 / L::THREADS));
    norm_kernel<T, decltype(values)::value, decltype(lanes)::value, decltype(pieces)::value, decltype(ends)::value>
        <<<dim3((unsigned)blocks), L::THREADS, 0, stream>>>(d);
    return hipGetLastError();
  });
}

bool shared_gate(const b2c_block_norm_grad_args* b) { return b->dgate && b->fwd.rows_per_gate > 1; }

struct NormGradPlan {
  Walk walk;
  float *w_parts = nullptr, *gate_parts = nullptr;
  bool w, g;
  NormGradPlan(const b2c_block_norm_grad_args* b, Room& room) {
    const b2c_block_norm_args* a = &b->fwd;
    const int64_t most = [&] {
      int threads = 256, teams = 1;
      auto look = [&](auto values, auto lanes, auto, auto) -> int {
        using L = Team<decltype(lanes)::value>;
        threads = decltype(values)::value == 8 ? 1024 : L::THREADS, teams = L::TEAMS;
        return 0;
      };
      a->dtype == B2C_F32 ? with_rows<float>(a->cols, true, look) : with_rows<f16>(a->cols, true, look);
      walk.rows = (uint32_t)teams;
      return 256 * (1024 / threads);  // workgroups, as many as are at work at once: 2048 rows of 4096 take 26 us with 256, 31 with 512
    }();
    const int64_t teams = walk.rows, rows = std::max<int64_t>(a->rows, 1);
    const bool shared = shared_gate(b);
    const int64_t per = shared ? std::min(a->rows_per_gate, rows) : rows, groups = up(rows, per) / per;
    const int64_t steps = up(per, teams) / teams, segments = std::max<int64_t>(1, std::min(steps, up(most, groups) / groups));
    const int64_t each = up(up(per, segments) / segments, teams);
    walk = {(uint32_t)groups, (uint32_t)per, (uint32_t)(up(per, each) / each), (uint32_t)each, 0};
    walk.blocks = (uint32_t)std::min<int64_t>(most, groups * walk.segments);
    w = (b->dw_post && a->post && a->x) || (b->dw_pre && b->dn);
    g = shared && walk.segments > 1;
    if (w) w_parts = room.take<float>((int64_t)walk.blocks * 2 * a->cols);
    if (g) gate_parts = room.take<float>(groups * walk.segments * a->cols);
  }
};

template <typename T>
int backward(const b2c_block_norm_grad_args* b, hipStream_t stream) {
  const b2c_block_norm_args* a = &b->fwd;
  Room room{(char*)b->workspace};
  const NormGradPlan p(b, room);
  NormGradArgs d{to_device(a), p.walk, b->dy, b->dn, b->lddy, b->lddn, b->dx, b->dresidual, b->dgate, b->lddx, b->lddr, b->lddg,
                 p.w_parts, p.gate_parts, shared_gate(b)};
  int rc = with_rows<T>(a->cols, true, [&](auto values, auto lanes, auto pieces, auto ends) -> int {
    constexpr int L = decltype(lanes)::value;
    norm_back_kernel<T, decltype(values)::value, L, decltype(pieces)::value, decltype(ends)::value>
        <<<dim3(p.walk.blocks), Team<L>::THREADS, 0, stream>>>(d);
    return hipGetLastError();
  });
  if (rc || (!p.w && !p.g)) return rc;
  const uint32_t tiles = (uint32_t)(up(a->cols, 32) / 32);
  JoinArgs j{p.w_parts, p.gate_parts, a->cols, tiles, p.walk.blocks, p.walk.segments, p.w ? 2u : 0u, {b->dw_post, b->dw_pre},
             p.g ? b->dgate : nullptr, b->lddg, b->grad_dtype == B2C_F32, b->accumulate != 0};
  const int64_t blocks = (int64_t)tiles * (j.w_jobs + (p.g ? p.walk.groups : 0));
  norm_join_kernel<T><<<grid_of(blocks), 1024, 0, stream>>>(j);
  return hipGetLastError();
}

// The weights' gradients of no rows.
__global__ __launch_bounds__(256) void clear_kernel(void* a, void* b, int n, bool f32) {
  const int i = (int)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  for (void* p : {a, b}) {
    if (p && f32) ((float*)p)[i] = 0.f;
    else if (p) ((uint16_t*)p)[i] = 0;
  }
}

}  // namespace
}  // namespace dev
}  // namespace b2c

using namespace b2c::dev;

extern "C" int b2c_hip_block_norm(const b2c_block_norm_args* a, hipStream_t stream) {
  if (!sizes_ok(a)) return hipErrorInvalidValue;
  const size_t s = size_of(a->dtype);
  if (a->rows == 0) return hipSuccess;
  if (!inputs_ok(a) || (!a->y && !a->n) || (!a->x && a->y) || (a->y && !good(a->y, a->ldy, a->cols, s)) ||
      (a->n && !good(a->n, a->ldn, a->cols, s)))
    return hipErrorInvalidValue;
  if (a->dtype == B2C_F32) return forward<float>(a, stream);
  if (a->dtype == B2C_F16) return forward<f16>(a, stream);
  return forward<bf16>(a, stream);
}

extern "C" size_t b2c_block_norm_grad_workspace_bytes(const b2c_block_norm_grad_args* b) {
  if (!b || !sizes_ok(&b->fwd) || b->fwd.rows == 0) return 0;
  Room room{nullptr};
  NormGradPlan(b, room);
  return room.used;
}

extern "C" int b2c_hip_block_norm_backward(const b2c_block_norm_grad_args* b, hipStream_t stream) {
  if (!b || !sizes_ok(&b->fwd)) return hipErrorInvalidValue;
  const b2c_block_norm_args* a = &b->fwd;
  const size_t s = size_of(a->dtype), gs = size_of(b->grad_dtype);
  if ((b->grad_dtype != a->w_dtype && b->grad_dtype != B2C_F32) || (b->accumulate && b->grad_dtype != B2C_F32) || (b->dw_post && !a->post) ||
      reinterpret_cast<uintptr_t>(b->dw_post) % gs || reinterpret_cast<uintptr_t>(b->dw_pre) % gs)
    return hipErrorInvalidValue;
  if (a->rows == 0) {
    if (b->accumulate || (!b->dw_post && !b->dw_pre)) return hipSuccess;
    clear_kernel<<<dim3((unsigned)(up(a->cols, 256) / 256)), 256, 0, stream>>>(b->dw_post, b->dw_pre, a->cols, gs == 4);
    return hipGetLastError();
  }
  if (!inputs_ok(a) || (b->dw_post && !a->x) || (b->dw_pre && !b->dn) || (b->dx && !a->x) || (b->dgate && !a->gate) ||
      (!b->dy && !b->dn) || (b->dy && !good(b->dy, b->lddy, a->cols, s)) || (b->dn && !good(b->dn, b->lddn, a->cols, s)) ||
      (b->dx && !good(b->dx, b->lddx, a->cols, s)) || (b->dresidual && !good(b->dresidual, b->lddr, a->cols, s)) ||
      (b->dgate && !good(b->dgate, b->lddg, a->cols, s)))
    return hipErrorInvalidValue;
  const size_t need = b2c_block_norm_grad_workspace_bytes(b);
  if (need && (!b->workspace || reinterpret_cast<uintptr_t>(b->workspace) % 16 || b->workspace_bytes < need)) return hipErrorInvalidValue;
  if (!b->dx && !b->dresidual && !b->dgate && !b->dw_post && !b->dw_pre) return hipSuccess;
  if (a->dtype == B2C_F32) return backward<float>(b, stream);
  if (a->dtype == B2C_F16) return backward<f16>(b, stream);
  return backward<bf16>(b, stream);
}
