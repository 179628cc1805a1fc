// How a product is carried out: the tile's size and the number of parts that k is split into are chosen by its shape;
// a few rows take a kernel of their own, which streams the weights.
#pragma once
#include "dense_tile.h"

namespace b2c {
namespace dev {

// ---- a long k in parts -------------------------------------------------------------------------------------

// Sums of a part of k, kept whole: value (part, plane, m, n) at ((part planes + plane) M + m) ld + n.
template <typename S>
struct Parts {
  S* sums;
  int64_t M, ld;
  int planes;
  template <int W>
  __device__ __forceinline__ void store(int64_t plane, int64_t m, int n, const S (&v)[W]) const {
    vec<S, W> t;
#pragma unroll
    for (int j = 0; j < W; j++) t[j] = v[j];
    *reinterpret_cast<vec<S, W>*>(sums + (plane * M + m) * ld + n) = t;
  }
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t part, int64_t m, int n, const S (&v)[W]) const {
    store<W>((int64_t)part * planes, m, n, v);
  }
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t part, int64_t m, int n, const S (&g)[W], const S (&u)[W]) const {
    store<W>((int64_t)part * planes, m, n, g);
    store<W>((int64_t)part * planes + 1, m, n, u);
  }
};

// Adds the parts in their order and finishes them with the product's epilogue, eight columns a thread.
template <typename S, bool DUAL, typename Epi>
__global__ __launch_bounds__(256) void join_kernel(Parts<S> p, int64_t M, uint32_t groups, int N, int parts, Epi epi) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, m = t / groups;
  if (m >= M) return;
  const int n = (int)(t - m * groups) * 8;
  S v[DUAL ? 2 : 1][8] = {};
  for (int part = 0; part < parts; part++)
#pragma unroll
    for (int d = 0; d < (DUAL ? 2 : 1); d++) {
      const S* from = p.sums + (((int64_t)part * p.planes + d) * p.M + m) * p.ld + n;
#pragma unroll
      for (int j = 0; j < 8; j++) v[d][j] += from[j];
    }
  if constexpr (DUAL) epi.template operator()<8>(0u, m, n, v[0], v[1]);
  else epi.template operator()<8>(0u, m, n, v[0]);
}

// ---- a few rows --------------------------------------------------------------------------------------------

// At most 16 MT rows of q against P: bound by reading P once. A workgroup takes 16 rows of P (DUAL: of each of the
// two), its eight waves every eighth 256-byte run of k; P goes from memory straight into the matrix instruction's
// registers, sixteen bytes of a row a lane, and q, which every workgroup reads again, comes from the caches. The
// eight sums meet in LDS and are added in a fixed order. No alignment is asked for.
template <typename T, bool DUAL, int MT, typename Epi>
__global__ __launch_bounds__(512) void few_rows_kernel(Product<T> a, Epi epi) {
  constexpr int V = Elem<T>::N, PL = DUAL ? 2 : 1, RUN = 16 * V;
  using Acc = typename Elem<T>::Acc;
  using A = vec<T, V>;
  __shared__ Acc sums[8][PL * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q4 = lane >> 4;
  const int64_t n = (int64_t)blockIdx.x * 16 + row;
  const int K = (int)a.K;
  Acc acc[PL][MT] = {};
  auto load = [&](const Side<T>& s, int64_t i, bool there, int k) {
    A v{};
    if (!there || k >= K) return v;
    const T* p = s.p + i * s.ld + k;
    if (k + V <= K) {
      __builtin_memcpy(&v, p, 16);
    } else {
#pragma unroll
      for (int j = 0; j < V; j++) v[j] = k + j < K ? p[j] : (T)0;
    }
    return v;
  };
  A p[2][PL][4], x[2][MT][4];
  auto fetch = [&](int b, int k0) {  // the run from k0 on; beyond K it is zeros and reads nothing
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int k = k0 + (c * 4 + q4) * V;
      p[b][0][c] = load(a.p, n, n < a.p_lim, k);
      if constexpr (DUAL) p[b][1][c] = load(a.p2, n, n < a.p_lim, k);
#pragma unroll
      for (int i = 0; i < MT; i++) x[b][i][c] = load(a.q, i * 16 + row, i * 16 + row < a.M, k);
    }
  };
  auto multiply = [&](int b) {
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int d = 0; d < PL; d++) acc[d][i] = mfma(p[b][d][c], x[b][i][c], acc[d][i]);
  };
  fetch(0, wave * RUN);
  for (int k0 = wave * RUN; k0 < K; k0 += 16 * RUN) {  // a run ahead of the one at work
    fetch(1, k0 + 8 * RUN);
    multiply(0);
    fetch(0, k0 + 16 * RUN);
    multiply(1);
  }
#pragma unroll
  for (int d = 0; d < PL; d++)
#pragma unroll
    for (int i = 0; i < MT; i++) sums[wave][d * MT + i][lane] = acc[d][i];
  __syncthreads();
  if (wave >= MT) return;
  using S = std::remove_reference_t<decltype(acc[0][0][0])>;
  Acc v[PL];
#pragma unroll
  for (int d = 0; d < PL; d++) {
    v[d] = sums[0][d * MT + wave][lane];
#pragma unroll
    for (int w = 1; w < 8; w++) v[d] += sums[w][d * MT + wave][lane];
  }
  const int64_t m = wave * 16 + row;
  const int n4 = (int)blockIdx.x * 16 + q4 * 4;
  if (m >= a.M || n4 >= a.N) return;
  S g[4], u[4];
#pragma unroll
  for (int j = 0; j < 4; j++) g[j] = v[0][j], u[j] = v[PL - 1][j];
  if constexpr (DUAL) epi.template operator()<4>(0u, m, n4, g, u);
  else epi.template operator()<4>(0u, m, n4, g);
}

// ---- the choice --------------------------------------------------------------------------------------------

enum { TILE_256, TILE_128, TILE_64, FEW_ROWS };
constexpr int64_t kFewRows = 32;

struct Way {
  int tile;
  int parts;
  size_t sums;  // bytes of workspace for the parts
};

// What a product of these sizes costs by each tile, in microseconds, from measured times: a step of 128 bytes of k takes a
// compute unit 1.58 us for a 256x256 tile, 0.51 each for two of 128x128 side by side (0.82 for one alone), 0.2 each for five of 64x64
// (0.51 alone), beside a launch, a first copy and an epilogue of 6, 3.7 and 2.9. A large tile reads less, small ones keep
// more compute units at work when there are few: 4096 x 4096 x 4096 takes 106, 133 and 210 us, 1037 x 2752 x 1000 takes 28, 14
// and 14, 512 x 512 x 512 takes 16, 7 and 5. Where even the small ones leave the device idle, k is split, for a write and a
// read of the sums.
inline Way choose(int64_t M, int64_t N, int64_t steps, bool dual, bool may_be_few) {
  if (may_be_few && M <= kFewRows) return {FEW_ROWS, 1, 0};
  static const struct { int side; double wide, alone, fixed; int held; } tiles[3] = {
      {256, 1.58, 1.45, 6.0, 1}, {128, 0.51, 0.82, 3.7, 2}, {64, 0.2, 0.51, 2.9, 5}};
  Way best{TILE_64, 1, 0};
  double least = 1e30;
  const int64_t ld = up(N, 8);
  for (int t = 0; t < 3; t++) {
    const int64_t cols = dual ? tiles[t].side / 2 : tiles[t].side;
    const int64_t count = up(M, tiles[t].side) / tiles[t].side * (up(N, cols) / cols);
    for (int parts = 1; parts <= 64; parts *= 2) {
      const double sums = 4.0 * parts * (dual ? 2 : 1) * M * ld;
      if (parts > 1 && (steps / parts < 4 || sums > 256e6)) break;
      const int64_t all = count * parts;
      const double step = std::max(tiles[t].wide * (double)up(all, 256) / 256, tiles[t].alone * (double)up(all, 256 * tiles[t].held) / (256 * tiles[t].held));
      const double us = tiles[t].fixed + step * std::max(1.0, (double)steps / parts) + (parts > 1 ? 4 + 2 * sums / 3.5e6 : 0);
      if (us < least) least = us, best = {t, parts, parts > 1 ? (size_t)sums : 0};
    }
  }
  return best;
}

template <typename T, bool PT, bool QT, bool DUAL, bool TWO, int SIDE, typename Epi>
int launch_tiles(const Product<T>& a, int parts, const Epi& epi, hipStream_t stream) {
  constexpr int COLS = DUAL ? SIDE / 2 : SIDE;
  const int64_t tm = up(a.M, SIDE) / SIDE, tn = up(a.N, COLS) / COLS;
  if (tm * tn * parts > 0x7fffffff) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(tm * tn * parts));
  if constexpr (SIDE == 256)
    tile_kernel<T, PT, QT, DUAL, TWO, 2, 4, 128, 64><<<grid, 512, 0, stream>>>(a, (int)tm, (int)tn, parts, epi);
  else if constexpr (SIDE == 128)
    tile_kernel<T, PT, QT, DUAL, TWO, 2, 4, 64, 32><<<grid, 512, 0, stream>>>(a, (int)tm, (int)tn, parts, epi);
  else
    tile_kernel<T, PT, QT, DUAL, TWO, 2, 2, 32, 32><<<grid, 256, 0, stream>>>(a, (int)tm, (int)tn, parts, epi);
  return hipGetLastError();
}

template <typename T, bool PT, bool QT, bool DUAL, bool TWO, typename Epi>
int tiles(const Product<T>& a, int tile, int parts, const Epi& epi, hipStream_t stream) {
  if (tile == TILE_256) return launch_tiles<T, PT, QT, DUAL, TWO, 256>(a, parts, epi, stream);
  if (tile == TILE_128) return launch_tiles<T, PT, QT, DUAL, TWO, 128>(a, parts, epi, stream);
  return launch_tiles<T, PT, QT, DUAL, TWO, 64>(a, parts, epi, stream);
}

// Carries out `a` the way that choose() gave; `sums`: its workspace.
template <typename T, bool PT, bool QT, bool DUAL, bool TWO, typename Epi>
int product(const Product<T>& a, const Way& way, void* sums, const Epi& epi, hipStream_t stream) {
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  if constexpr (!PT && !QT && !TWO) {
    if (way.tile == FEW_ROWS) {
      const dim3 grid((unsigned)(up(a.N, 16) / 16));
      if (a.M <= 16) few_rows_kernel<T, DUAL, 1><<<grid, 512, 0, stream>>>(a, epi);
      else few_rows_kernel<T, DUAL, 2><<<grid, 512, 0, stream>>>(a, epi);
      return hipGetLastError();
    }
  }
  if (way.parts == 1) return tiles<T, PT, QT, DUAL, TWO>(a, way.tile, 1, epi, stream);
  using S = std::conditional_t<std::is_same_v<T, int8_t>, int, float>;
  const Parts<S> p{(S*)sums, a.M, up(a.N, 8), DUAL ? 2 : 1};
  const int rc = tiles<T, PT, QT, DUAL, TWO>(a, way.tile, way.parts, p, stream);
  if (rc) return rc;
  const int64_t groups = up(a.N, 8) / 8, blocks = up(a.M * groups, 256) / 256;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  join_kernel<S, DUAL><<<dim3((unsigned)blocks), 256, 0, stream>>>(p, a.M, (uint32_t)groups, (int)a.N, way.parts, epi);
  return hipGetLastError();
}

}  // namespace dev
}  // namespace b2c
