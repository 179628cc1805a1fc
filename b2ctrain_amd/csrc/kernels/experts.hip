// A mixture-of-experts layer for a few tokens (b2c_hip_experts): the router, the chosen experts' gate and up projections, their down
// projections, and the weighted sum.
#include "dense_rows.h"

#include <cmath>

namespace b2c {
namespace dev {
namespace {

constexpr int kMostExperts = 1024, kMostChosen = 64;
constexpr int kLot = 1024;  // pairs of a token and an expert that one set of launches carries out

// ---- the router --------------------------------------------------------------------------------------------

struct RouteArgs {
  int D, E, K;
  bool normalize;
  int32_t *to, *index;
  float *share, *weight;
  int64_t ldi, ldw;
};

// x . w in 64 bits, by a wave, for AT rows of w that lie `step` apart; those from `left` on are not there. Products of 16-bit floats are
// exact in 64 bits and their sums nearly so: two experts are told apart where the numbers do it.
template <typename T, int AT>
__device__ __forceinline__ void wide_dots(const T* x, const T* w, int64_t step, int left, int D, double (&s)[AT]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < AT; i++) s[i] = 0;
  auto add = [&](auto read, int k) {
    const vec<T, 8> v = read(x, k);
    vec<T, 8> u[AT];
#pragma unroll
    for (int i = 0; i < AT; i++) u[i] = read(w + (i < left ? i : 0) * step, k);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double d = (double)(float)v[j];
#pragma unroll
      for (int i = 0; i < AT; i++) s[i] = fma(d, (double)(float)u[i][j], s[i]);
    }
  };
  const int whole = D / 512 * 512;
#pragma unroll 4
  for (int k = 0; k < whole; k += 512)
    add([](const T* p, int k) {
      vec<T, 8> v;
      __builtin_memcpy(&v, p + k, 16);
      return v;
    }, k + lane * 8);
  if (D < 8) {
    if (lane == 0) add([D](const T* p, int k) { return some<T, 8>(p, k, D); }, 0);
  } else if (whole < D) {
    add([D](const T* p, int k) { return end8<T>(p, k, D); }, whole + lane * 8);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < AT; i++) s[i] += __shfl_xor(s[i], o);
}

// Chooses among the logits of one token, which a workgroup of THREADS has in LDS: an expert's place is how many are before it, so that the
// order takes no rounds of maxima.
template <int MOST, int THREADS>
struct Choice {
  double logits[MOST];
  uint64_t keys[MOST + 8];
  int chosen[kMostChosen];
  float parts[THREADS / 64], share[kMostChosen];
  __device__ __forceinline__ void set(int e, double l) {
    l += 0.0;  // no negative zero
    const uint64_t b = l != l ? 0x7fffffffffffffffull : __builtin_bit_cast(uint64_t, l);
    logits[e] = l;
    keys[e] = b >> 63 ? ~b : b | 1ull << 63;  // in the order of the numbers, a NaN above them
  }
  // After a barrier; leaves `chosen` and `share`, behind one.
  __device__ __forceinline__ void choose(const RouteArgs& a) {
    const int t = threadIdx.x;
    if (t < 8) keys[a.E + t] = 0;  // below every number
    __syncthreads();
    for (int e = t; e < a.E; e += THREADS) {
      const uint64_t mine = keys[e];
      int before = 0;
      for (int i = 0; i < a.E; i += 8)
#pragma unroll
        for (int j = 0; j < 8; j++) before += keys[i + j] > mine || (keys[i + j] == mine && i + j < e);
      if (before < a.K) chosen[before] = e;
    }
    __syncthreads();
    const double top = logits[chosen[0]];
    float all = 0;
    if (a.normalize) {
      for (int j = 0; j < a.K; j++) all += expf((float)(logits[chosen[j]] - top));
    } else {
      float s = 0;
      for (int e = t; e < a.E; e += THREADS) s += expf((float)(logits[e] - top));
#pragma unroll
      for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
      if ((t & 63) == 0) parts[t >> 6] = s;
      __syncthreads();
      for (int i = 0; i < THREADS / 64; i++) all += parts[i];
    }
    if (t < a.K) share[t] = expf((float)(logits[chosen[t]] - top)) / all;
    __syncthreads();
  }
  __device__ __forceinline__ void write(const RouteArgs& a, int64_t m) const {
    const int t = threadIdx.x;
    if (t >= a.K) return;
    a.to[m * a.K + t] = chosen[t];
    a.share[m * a.K + t] = share[t];
    if (a.index) a.index[m * a.ldi + t] = chosen[t];
    if (a.weight) a.weight[m * a.ldw + t] = share[t];
  }
};

// A workgroup a token, AT experts of a wave at a time, so that a piece of x is converted once for them. Latency and arithmetic in 64 bits: 16
// tokens of 2048 with 16 experts take 5.0 us, with 64 experts 10.7.
template <typename T, int AT>
__global__ __launch_bounds__(1024) void route_kernel(Side<T> x, Side<T> w, RouteArgs a) {
  __shared__ Choice<kMostExperts, 1024> choice;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m = blockIdx.x;
  for (int e0 = wave * AT; e0 < a.E; e0 += 16 * AT) {
    double s[AT];
    wide_dots<T, AT>(x.p + m * x.ld, w.p + e0 * w.ld, w.ld, a.E - e0, a.D, s);
#pragma unroll
    for (int i = 0; i < AT; i++)
      if (lane == i && e0 + i < a.E) choice.set(e0 + i, s[i]);
  }
  choice.choose(a);
  choice.write(a, m);
}

// ---- one token ---------------------------------------------------------------------------------------------

// The logits of one token by more than one workgroup; every workgroup of the kernel that follows chooses for itself. 64 experts of 2048: 2.9
// us, where one workgroup takes 10.7.
template <typename T>
__global__ __launch_bounds__(256) void logits_kernel(const T* x, Side<T> w, int E, int D, double* logits) {
  const int e = (int)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (e >= E) return;
  double s[1];
  wide_dots<T, 1>(x, w.p + e * w.ld, 0, 1, D, s);
  if ((threadIdx.x & 63) == 0) logits[e] = s[0];
}

// An inner activation as a value of T and what that is off by. The first stays within T's largest, so that the second takes what is beyond.
template <typename T>
__device__ __forceinline__ void halves(float v, T& first, T& second) {
  constexpr float most = std::is_same_v<T, f16> ? 65504.f : 0x1.fep127f;
  first = (T)__builtin_amdgcn_fmed3f(v, -most, most);
  second = (T)(v - (float)first);
}

constexpr int kChooseOften = 256;  // experts among which every workgroup of a launch may choose again

// A row's slab of 512 values is a kilobyte, sixteen bytes a lane. Values begin .. end - 1 of four rows (a wave's) against those of the sum of X
// vectors that lie `next` apart, SLABS slabs at a time; each row's sum stays spread over the lanes. `end` is the rows' end K or a multiple
// of 512.
template <typename T, int SLABS, int X>
__device__ __forceinline__ void four_rows(const T* const (&rows)[4], const T* x, int64_t next, int K, int begin, int end, float (&sum)[4]) {
  const int lane = threadIdx.x & 63;
  using V = vec<uint32_t, 4>;
  auto add = [&](const V& w, const V (&v)[X], float& to) {
#pragma unroll
    for (int p = 0; p < X; p++)
#pragma unroll
      for (int j = 0; j < 4; j++) to = dot2(w[j], v[p][j], to, T{});
  };
  int k0 = begin;
  for (; k0 + 512 <= end; k0 += SLABS * 512) {
    V w[SLABS][4], v[SLABS][X];
#pragma unroll
    for (int s = 0; s < SLABS; s++)
      if (k0 + s * 512 + 512 <= end) {
#pragma unroll
        for (int p = 0; p < X; p++) __builtin_memcpy(&v[s][p], x + p * next + k0 + s * 512 + lane * 8, 16);
#pragma unroll
        for (int i = 0; i < 4; i++) __builtin_memcpy(&w[s][i], rows[i] + k0 + s * 512 + lane * 8, 16);
      }
#pragma unroll
    for (int s = 0; s < SLABS; s++)
      if (k0 + s * 512 + 512 <= end)
#pragma unroll
        for (int i = 0; i < 4; i++) add(w[s][i], v[s], sum[i]);
  }
  const int k = begin + (end - begin) / 512 * 512;  // what a slab holds of the end
  if (k >= end) return;
  V v[X];
  if (K < 8) {
    if (lane) return;
#pragma unroll
    for (int p = 0; p < X; p++) v[p] = __builtin_bit_cast(V, some<T, 8>(x + p * next, 0, K));
#pragma unroll
    for (int i = 0; i < 4; i++) add(__builtin_bit_cast(V, some<T, 8>(rows[i], 0, K)), v, sum[i]);
    return;
  }
#pragma unroll
  for (int p = 0; p < X; p++) v[p] = __builtin_bit_cast(V, end8<T>(x + p * next, k + lane * 8, K));
#pragma unroll
  for (int i = 0; i < 4; i++) add(__builtin_bit_cast(V, end8<T>(rows[i], k + lane * 8, K)), v, sum[i]);
}
__device__ __forceinline__ float over_wave(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// h[choice] = act(w_gate x) (w_up x), as a value of T and what it is off by, hp behind it: one rounding to T would leave y half as far off
// again as its own does (2.5e-3 for 1.7e-3 in bf16), and the second product costs the down projection, which waits for memory, nothing.
// Two hidden units a wave, eight a workgroup, so that a few experts' rows fill the device, and a wave's 16 kilobytes are on their way
// together. Eight experts of 2048-1024 (67 MB) take 14.7 us, 4.6 TB/s, in one round of workgroups.
template <typename T, int ACT, bool CHOOSE>
__global__ __launch_bounds__(256) void gate_up_one_kernel(const T* x, Side<T> wg, Side<T> wu, int F, const double* logits, T* h, int64_t hp, RouteArgs a) {
  __shared__ Choice<CHOOSE ? kChooseOften : 1, 256> choice;
  const int wave = threadIdx.x >> 6, slot = (int)blockIdx.y, n = (int)blockIdx.x * 8 + wave * 2;
  int e;
  if constexpr (CHOOSE) {
    for (int i = threadIdx.x; i < a.E; i += 256) choice.set(i, logits[i]);
    choice.choose(a);
    e = choice.chosen[slot];
    if (blockIdx.x == 0 && slot == 0) choice.write(a, 0);
  } else {
    e = a.to[slot];
  }
  if (n >= F) return;
  const int64_t row = (int64_t)e * F + n;
  const int next = n + 1 < F ? 1 : 0;
  const T* const rows[4] = {wg.p + row * wg.ld, wg.p + (row + next) * wg.ld, wu.p + row * wu.ld, wu.p + (row + next) * wu.ld};
  float sum[4] = {};
  four_rows<T, 4, 1>(rows, x, 0, a.D, 0, a.D, sum);
#pragma unroll
  for (int i = 0; i < 4; i++) sum[i] = over_wave(sum[i]);
  const int lane = threadIdx.x & 63;
  if (lane > next) return;
  const float v = act<ACT>(lane ? sum[1] : sum[0]) * (lane ? sum[3] : sum[2]);
  T* to = h + slot * 2 * hp + n + lane;
  halves(v, to[0], to[hp]);
}

// y = residual + the weighted sum over the choices of w_down h: four outputs a workgroup, its eight waves a choice each, or a part of one's k
// where there are fewer. Eight experts of 1024-2048 (34 MB): 7.9 us, 4.2 TB/s.
template <typename T>
__global__ __launch_bounds__(512) void down_one_kernel(const T* h, int64_t hp, Side<T> w, int F, int O, const T* residual, T* y, RouteArgs a) {
  __shared__ float sums[8][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = (int)blockIdx.x * 4;
  int parts = 1;
  while (parts * 2 * a.K <= 8 && parts * 1024 <= F) parts *= 2;
  const int each = ((F + parts - 1) / parts + 511) / 512 * 512;
  float total[4] = {};
  for (int unit = wave; unit < a.K * parts; unit += 8) {
    const int slot = unit / parts, begin = (unit - slot * parts) * each, end = begin + each < F ? begin + each : F;
    const int e = a.to[slot];
    const float p = a.share[slot];
    const T* rows[4];
#pragma unroll
    for (int i = 0; i < 4; i++) rows[i] = w.p + ((int64_t)e * O + (n0 + i < O ? n0 + i : O - 1)) * w.ld;
    float sum[4] = {};
    four_rows<T, 2, 2>(rows, h + slot * 2 * hp, hp, F, begin, end, sum);
#pragma unroll
    for (int i = 0; i < 4; i++) total[i] = fmaf(p, sum[i], total[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float v = over_wave(total[i]);
    if (lane == i) sums[wave][i] = v;
  }
  __syncthreads();
  const int n = n0 + (int)threadIdx.x;
  if (threadIdx.x >= 4 || n >= O) return;
  float v = residual ? (float)residual[n] : 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) v += sums[i][threadIdx.x];
  y[n] = (T)v;
}

// ---- who goes where ----------------------------------------------------------------------------------------

// Which experts the pairs of a lot (token t's j-th choice is pair t K + j) name, as bits in LDS.
struct Taken {
  uint32_t bits[kMostExperts / 32];
  __device__ __forceinline__ void find(const int32_t* to, int pairs) {
    for (int i = threadIdx.x; i < kMostExperts / 32; i += blockDim.x) bits[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) atomicOr(&bits[to[i] >> 5], 1u << (to[i] & 31));
    __syncthreads();
  }
  // The expert with `before` taken ones below it, or -1.
  __device__ __forceinline__ int at(int before, int E) const {
    for (int i = 0; i < (E + 31) / 32; i++) {
      uint32_t b = bits[i];
      const int n = __builtin_popcount(b);
      if (before < n) {
        while (before--) b &= b - 1;
        return i * 32 + __builtin_ctz(b);
      }
      before -= n;
    }
    return -1;
  }
};
// A wave writes the pairs that name expert e to `list`, in their order, and returns how many there are.
__device__ __forceinline__ int pairs_of(const int32_t* to, int pairs, int e, uint16_t* list) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int base = 0; base < pairs; base += 64) {
    const bool mine = base + lane < pairs && to[base + lane] == e;
    const uint64_t all = __ballot(mine);
    if (mine) list[n + __builtin_popcountll(all & ((1ull << lane) - 1))] = (uint16_t)(base + lane);
    n += __builtin_popcountll(all);
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");  // the wave's other lanes read them
  __builtin_amdgcn_wave_barrier();
  return n;
}

// ---- products ----------------------------------------------------------------------------------------------

struct ExpertArgs {
  int pairs, K, E;   // of the lot, choices a token, experts
  int cols, rows;    // of an expert's matrix
  int shared;        // waves that share a tile's k: 1, 2, 4 or 8
  const int32_t* to;
};

// Products of an expert's rows with its pairs' vectors, PL = 2 of them with the same (gate and up) or one (down): 16 rows a tile, 16 MT vectors
// at a time. With HALVES a pair's vector is the sum of two that lie `next` apart; a matrix instruction's 16 columns are then eight pairs
// twice, since an expert of few tokens has less than eight as a rule, and the two sums are added at the end (with two instructions for 16
// pairs the down projection of 16 tokens, two of 16 of 2048-5632, took 92 us where it takes 80: it waits for what the die's cache gives).
// `shared` waves take every shared-th run of 128 values of k of a tile. The weights go from memory straight to the matrix instructions'
// registers: each is used by one wave, once, so LDS would add a copy. Rows beyond the last read the last one's values, which nobody stores.
// LONG: K >= 8. Those 16 tokens: gate and up (681 MB) 148 us, 4.6 TB/s, down (341 MB) 80, 4.3; bound by memory.
// 61 tokens, three of 10 of 1000-1365 in f16: 24 and 28 us, 2.5 and 1.3 TB/s, bound by the vectors, which every tile reads from the die's cache.
template <typename T, int PL, bool HALVES, int MT, bool LONG, typename In, typename Out>
__device__ __forceinline__ void expert_product(const Side<T> (&w)[PL], int64_t next, const ExpertArgs& a, In in, Out out) {
  __shared__ Taken taken;
  __shared__ uint16_t list[kLot];
  __shared__ int count;
  __shared__ f32x4 sums[8][PL * MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & 15, q4 = lane >> 4;
  taken.find(a.to, a.pairs);
  const int e = taken.at((int)blockIdx.y, a.E);
  if (e < 0) return;
  if (wave == 0) {
    const int n = pairs_of(a.to, a.pairs, e, list);
    if (lane == 0) count = n;
  }
  __syncthreads();
  const int all = count, K = a.cols, whole = K >> 7, runs = (K + 127) >> 7;
  const int part = wave & (a.shared - 1), n0 = ((int)blockIdx.x * (8 / a.shared) + wave / a.shared) * 16;
  const int left = a.rows - n0;  // none: the wave has no tile
  const T* base[PL];
  uint32_t at[PL];
#pragma unroll
  for (int d = 0; d < PL; d++) {
    base[d] = w[d].p + ((int64_t)e * a.rows + (left > 0 ? n0 : 0)) * w[d].ld;
    at[d] = (uint32_t)(left > 0 ? (row < left ? row : left - 1) : 0) * (uint32_t)w[d].ld;
  }
  constexpr int PAIRS = HALVES ? 8 : 16;  // of a tile
  const int column = HALVES ? row & 7 : row;
  for (int first = 0; first < all; first += PAIRS * MT) {
    const T* px[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) {
      const int i = first + t * PAIRS + column;
      px[t] = in(list[i < all ? i : all - 1]) + (HALVES ? (row >> 3) * next : 0);
    }
    struct Run {
      vec<T, 8> w[PL][4], x[MT][4];
    };
    f32x4 acc[PL][MT] = {};
    auto fetch = [&](Run& r, int run) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int k = run * 128 + c * 32 + q4 * 8;
#pragma unroll
        for (int d = 0; d < PL; d++) __builtin_memcpy(&r.w[d][c], base[d] + (at[d] + (uint32_t)k), 16);
#pragma unroll
        for (int t = 0; t < MT; t++) __builtin_memcpy(&r.x[t][c], px[t] + k, 16);
      }
    };
    auto fetch_end = [&](Run& r) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int k = whole * 128 + c * 32 + q4 * 8;
#pragma unroll
        for (int d = 0; d < PL; d++) r.w[d][c] = end8<T>(base[d] + at[d], k, K);
#pragma unroll
        for (int t = 0; t < MT; t++) r.x[t][c] = end8<T>(px[t], k, K);
      }
    };
    auto fetch_only = [&](Run& r) {  // a row shorter than a piece
      r = {};
      if (q4 == 0) {
#pragma unroll
        for (int d = 0; d < PL; d++) r.w[d][0] = some<T, 8>(base[d] + at[d], 0, K);
#pragma unroll
        for (int t = 0; t < MT; t++) r.x[t][0] = some<T, 8>(px[t], 0, K);
      }
    };
    auto multiply = [&](const Run& r) {
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int d = 0; d < PL; d++) acc[d][t] = mfma(r.w[d][c], r.x[t][c], acc[d][t]);
    };
    if (left > 0) {
      if constexpr (LONG) {
        if (whole < runs && part == 0) {
          Run r;
          fetch_end(r);
          multiply(r);
        }
        // From a run on that differs from tile to tile, and around: rows are often a multiple of 4 KB apart, and waves that read the same
        // columns of theirs at the same time ask the same channels of the memory (168 us for 148).
        const int mine = (part + a.shared - 1) & (a.shared - 1), steps = whole > mine ? (whole - 1 - mine) / a.shared + 1 : 0;
        const int start = steps ? (n0 >> 4) % steps : 0;
        for (int i = 0; i < steps; i++) {
          Run r;
          const int step = start + i;
          fetch(r, mine + (step < steps ? step : step - steps) * a.shared);
          multiply(r);
        }
      } else if (part == 0) {
        Run r;
        fetch_only(r);
        multiply(r);
      }
    }
    auto finish = [&](int t, f32x4 (&v)[PL]) {
      if constexpr (HALVES) {
#pragma unroll
        for (int d = 0; d < PL; d++)
#pragma unroll
          for (int j = 0; j < 4; j++) {  // row_ror:8
            const float mine = v[d][j];
            v[d][j] = mine + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, mine), 0x128, 0xF, 0xF, true));
          }
      }
      const int i = first + t * PAIRS + column;
      if (i >= all || q4 * 4 >= left || (HALVES && row >= 8)) return;
      float o[PL][4];
#pragma unroll
      for (int d = 0; d < PL; d++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[d][j] = v[d][j];
      out(list[i], n0 + q4 * 4, o);
    };
    if (a.shared == 1) {
#pragma unroll
      for (int t = 0; t < MT; t++) {
        f32x4 v[PL];
#pragma unroll
        for (int d = 0; d < PL; d++) v[d] = acc[d][t];
        finish(t, v);
      }
      continue;
    }
    // The sums of the waves that share a tile, in their order; each finishes every shared-th of its column tiles.
    if (first) __syncthreads();
#pragma unroll
    for (int d = 0; d < PL; d++)
#pragma unroll
      for (int t = 0; t < MT; t++) sums[wave][d * MT + t][lane] = acc[d][t];
    __syncthreads();
    for (int t = part; t < MT; t += a.shared) {
      f32x4 v[PL];
#pragma unroll
      for (int d = 0; d < PL; d++) {
        v[d] = sums[wave - part][d * MT + t][lane];
        for (int i = 1; i < a.shared; i++) v[d] += sums[wave - part + i][d * MT + t][lane];
      }
      finish(t, v);
    }
  }
}

// h[pair] = act(w_gate x) (w_up x), as a value of T and what it is off by
template <typename T, int ACT, int MT, bool LONG>
__global__ __launch_bounds__(512, 4) void gate_up_kernel(Side<T> x, Side<T> wg, Side<T> wu, T* h, int64_t hp, ExpertArgs a) {
  const Side<T> w[2] = {wg, wu};
  expert_product<T, 2, false, MT, LONG>(
      w, 0, a, [&](int pair) { return x.p + (int64_t)(pair / a.K) * x.ld; },
      [&](int pair, int n, const float (&v)[2][4]) {
        float o[4], rest[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          T first, second;
          halves(act<ACT>(v[0][j]) * v[1][j], first, second);
          o[j] = (float)first, rest[j] = (float)second;
        }
        put<4>(h, 2 * hp, pair, n, a.rows, o);
        put<4>(h + hp, 2 * hp, pair, n, a.rows, rest);
      });
}
// parts[pair] = w_down h
template <typename T, int MT, bool LONG>
__global__ __launch_bounds__(512, 4) void down_kernel(const T* h, int64_t hp, Side<T> wd, float* parts, int64_t pp, ExpertArgs a) {
  const Side<T> w[1] = {wd};
  expert_product<T, 1, true, MT, LONG>(
      w, hp, a, [&](int pair) { return h + pair * 2 * hp; },
      [&](int pair, int n, const float (&v)[1][4]) { put<4>(parts, pp, pair, n, a.rows, v[0]); });
}
// y = residual + the weighted sum of a token's parts, in the order of its choices; four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const float* parts, int64_t pp, const float* share, const T* residual, int64_t ldr, T* y,
                                                      int64_t ldy, int K, int O) {
  const int64_t m = blockIdx.y;
  const int n = ((int)blockIdx.x * 256 + threadIdx.x) * 4;
  if (n >= O) return;
  float v[4] = {};
  if (residual) get<4>(residual, ldr, m, n, O, v);
  for (int j = 0; j < K; j++) {
    const f32x4 s = *reinterpret_cast<const f32x4*>(parts + (m * K + j) * pp + n);
    const float p = share[m * K + j];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = fmaf(p, s[i], v[i]);
  }
  put<4>(y, ldy, m, n, O, v);
}

// ---- host --------------------------------------------------------------------------------------------------

bool sizes_ok(const b2c_experts_args* a) {
  const int most = 1 << 20;
  return a && a->rows >= 0 && a->rows <= most && a->d_in >= 1 && a->d_in <= most && a->d_hidden >= 1 && a->d_hidden <= most &&
         a->d_out >= 1 && a->d_out <= most && a->experts >= 1 && a->experts <= kMostExperts && a->top_k >= 1 && a->top_k <= a->experts &&
         a->top_k <= kMostChosen && (int64_t)a->experts * std::max(a->d_hidden, a->d_out) <= 0x7fffffff &&
         (a->dtype == B2C_F16 || a->dtype == B2C_BF16) && a->act >= B2C_ACT_SILU && a->act <= B2C_ACT_RELU;
}

template <typename T>
struct ExpertsPlan {
  int64_t lot, hp, pp;
  int32_t* to;
  float *share, *parts = nullptr;
  double* logits = nullptr;
  T* h;
  ExpertsPlan(const b2c_experts_args* a, Room& room) {
    lot = std::min<int64_t>(a->rows, kLot / a->top_k);
    hp = up(a->d_hidden, 8);
    pp = up(a->d_out, 4);
    to = room.take<int32_t>(lot * a->top_k);
    share = room.take<float>(lot * a->top_k);
    h = room.take<T>(lot * a->top_k * 2 * hp);
    if (a->rows == 1) logits = room.take<double>(a->experts);
    else parts = room.take<float>(lot * a->top_k * pp);
  }
};

template <typename T, int ACT>
int one_token(const b2c_experts_args* a, const ExpertsPlan<T>& p, const RouteArgs& r, hipStream_t stream) {
  const T *x = (const T*)a->x, *residual = (const T*)a->residual;
  const Side<T> wr{(const T*)a->w_router, a->ld_router}, wg{(const T*)a->w_gate, a->ld_in}, wu{(const T*)a->w_up, a->ld_in},
      wd{(const T*)a->w_down, a->ld_out};
  const dim3 units((unsigned)(up(a->d_hidden, 8) / 8), (unsigned)a->top_k), outputs((unsigned)(up(a->d_out, 4) / 4));
  int rc;
  if (a->experts <= kChooseOften) {
    logits_kernel<T><<<dim3((unsigned)(up(a->experts, 4) / 4)), 256, 0, stream>>>(x, wr, a->experts, a->d_in, p.logits);
    if ((rc = hipGetLastError())) return rc;
    gate_up_one_kernel<T, ACT, true><<<units, 256, 0, stream>>>(x, wg, wu, a->d_hidden, p.logits, p.h, p.hp, r);
    if ((rc = hipGetLastError())) return rc;
  } else {
    route_kernel<T, 4><<<dim3(1), 1024, 0, stream>>>(Side<T>{x, a->ldx}, wr, r);
    if ((rc = hipGetLastError())) return rc;
    gate_up_one_kernel<T, ACT, false><<<units, 256, 0, stream>>>(x, wg, wu, a->d_hidden, p.logits, p.h, p.hp, r);
    if ((rc = hipGetLastError())) return rc;
  }
  down_one_kernel<T><<<outputs, 512, 0, stream>>>(p.h, p.hp, wd, a->d_hidden, a->d_out, residual, (T*)a->y, r);
  return hipGetLastError();
}

// Waves that share a tile's k, from how many rounds of 4096 waves (four to a SIMD) the tiles of the experts that are expected to be met take:
// 16 tokens, two of 16 experts of 2048-5632: gate and up take 182 us with one wave to a tile, 148, 158 and 201 with two, four and eight;
// two tokens, eight of 64 of 2048-1024: 59, 33, 28 and 35.
int sharing(double tiles, int cols) {
  constexpr double more[] = {1, 1.07, 1.3, 1.45};
  int best = 1;
  double least = 1e30;
  for (int i = 0; i < 4 && (i == 0 || cols >= 128 << i); i++) {
    const double cost = std::ceil(tiles * (1 << i) / 4096) / (1 << i) * more[i];
    if (cost < least) least = cost, best = 1 << i;
  }
  return best;
}

template <typename T, int ACT>
int run(const b2c_experts_args* a, hipStream_t stream) {
  Room room{(char*)a->workspace};
  const ExpertsPlan<T> p(a, room);
  const Side<T> wr{(const T*)a->w_router, a->ld_router}, wg{(const T*)a->w_gate, a->ld_in}, wu{(const T*)a->w_up, a->ld_in},
      wd{(const T*)a->w_down, a->ld_out};
  const int K = a->top_k, E = a->experts;
  for (int64_t m = 0; m < a->rows; m += p.lot) {
    const int64_t rows = std::min(p.lot, a->rows - m);
    const Side<T> x{(const T*)a->x + m * a->ldx, a->ldx};
    const RouteArgs r{a->d_in, E, K, a->normalize != 0, p.to, a->index ? a->index + m * a->ldi : nullptr, p.share,
                      a->weight ? a->weight + m * a->ldw : nullptr, a->ldi, a->ldw};
    if (a->rows == 1) return one_token<T, ACT>(a, p, r, stream);
    if (E <= 16) route_kernel<T, 1><<<dim3((unsigned)rows), 1024, 0, stream>>>(x, wr, r);
    else if (E <= 32) route_kernel<T, 2><<<dim3((unsigned)rows), 1024, 0, stream>>>(x, wr, r);
    else route_kernel<T, 4><<<dim3((unsigned)rows), 1024, 0, stream>>>(x, wr, r);
    int rc = hipGetLastError();
    if (rc) return rc;
    const int pairs = (int)rows * K;
    const int64_t slots = std::min(pairs, E);
    const double met = std::max(1.0, E * (1 - std::pow(1 - (double)K / E, (double)rows)));  // experts, where any are as likely
    ExpertArgs up_args{pairs, K, E, a->d_in, a->d_hidden, 0, p.to}, down_args{pairs, K, E, a->d_hidden, a->d_out, 0, p.to};
    // One tile of columns, or as many as an expert's vectors, of which the down projection has two for each pair, mostly fill: 64 tokens, eight
    // of 64 of 2048-1024: down 115, 89 and 107 us with one, two and four; 61 tokens, three of 10 of 1000-1365: 43, 32 and 27, and gate and up
    // 24, 18 and 24.
    auto launch = [&](ExpertArgs& args, double vectors, auto most, auto with) -> int {
      const int64_t tiles = up(args.rows, 16) / 16;
      args.shared = sharing((double)tiles * met, args.cols);
      const dim3 grid((unsigned)(up(tiles * args.shared, 8) / 8), (unsigned)slots);
      using std::integral_constant;
      if (args.cols < 8) with(grid, integral_constant<int, 1>{}, std::false_type{});
      else if (vectors <= 14) with(grid, integral_constant<int, 1>{}, std::true_type{});
      else if (vectors <= 32 || decltype(most)::value == 2) with(grid, integral_constant<int, 2>{}, std::true_type{});
      else with(grid, most, std::true_type{});
      return hipGetLastError();
    };
    rc = launch(up_args, pairs / met, std::integral_constant<int, 2>{}, [&](dim3 grid, auto mt, auto far) {
      gate_up_kernel<T, ACT, decltype(mt)::value, decltype(far)::value><<<grid, 512, 0, stream>>>(x, wg, wu, p.h, p.hp, up_args);
    });
    if (rc) return rc;
    rc = launch(down_args, 2 * pairs / met, std::integral_constant<int, 4>{}, [&](dim3 grid, auto mt, auto far) {
      down_kernel<T, decltype(mt)::value, decltype(far)::value><<<grid, 512, 0, stream>>>(p.h, p.hp, wd, p.parts, p.pp, down_args);
    });
    if (rc) return rc;
    const dim3 grid((unsigned)(up(a->d_out, 1024) / 1024), (unsigned)rows);
    combine_kernel<T><<<grid, 256, 0, stream>>>(p.parts, p.pp, p.share, a->residual ? (const T*)a->residual + m * a->ldr : nullptr, a->ldr,
                                                (T*)a->y + m * a->ldy, a->ldy, K, a->d_out);
    if ((rc = hipGetLastError())) return rc;
  }
  return hipSuccess;
}
template <typename T>
int run(const b2c_experts_args* a, hipStream_t stream) {
  if (a->act == B2C_ACT_SILU) return run<T, B2C_ACT_SILU>(a, stream);
  if (a->act == B2C_ACT_GELU) return run<T, B2C_ACT_GELU>(a, stream);
  return run<T, B2C_ACT_RELU>(a, stream);
}

}  // namespace
}  // namespace dev
}  // namespace b2c

using namespace b2c::dev;

extern "C" size_t b2c_experts_workspace_bytes(const b2c_experts_args* a) {
  if (!sizes_ok(a) || a->rows == 0) return 0;
  Room room{nullptr};
  ExpertsPlan<bf16>(a, room);  // both types have the same size
  return room.used;
}
extern "C" int b2c_hip_experts(const b2c_experts_args* a, hipStream_t stream) {
  if (!sizes_ok(a)) return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  if (!good(a->x, a->ldx, a->d_in, 2) || !good(a->w_router, a->ld_router, a->d_in, 2) || !good(a->w_gate, a->ld_in, a->d_in, 2) ||
      !good(a->w_up, a->ld_in, a->d_in, 2) || !good(a->w_down, a->ld_out, a->d_hidden, 2) || !good(a->y, a->ldy, a->d_out, 2) ||
      (a->residual && !good(a->residual, a->ldr, a->d_out, 2)) || (a->index && !good(a->index, a->ldi, a->top_k, 4)) ||
      (a->weight && !good(a->weight, a->ldw, a->top_k, 4)) || !a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 ||
      a->workspace_bytes < b2c_experts_workspace_bytes(a) || a->ld_in > kFarRows || a->ld_out > kFarRows)
    return hipErrorInvalidValue;
  return a->dtype == B2C_F16 ? run<f16>(a, stream) : run<bf16>(a, stream);
}
