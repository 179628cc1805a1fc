// How a product is carried out: the tile's size and the number of parts that k is split into are chosen by its shape;
// a few rows take a kernel of their own, which streams the weights.
#pragma once
#include "dense_tile.h"

#include <cmath>
#include <initializer_list>

namespace b2c {
namespace dev {

// ---- a long k in parts -------------------------------------------------------------------------------------

// Sums of parts of k, tile by tile: value (plane, m, n) of workgroup w at ((w planes + plane) rows + m % rows) cols + n % cols,
// in single precision, or in integers, which stay exact.
template <typename S, int ROWS, int COLS, int PLANES>
struct Parts {
  S* sums;
  __device__ __forceinline__ S* at(uint32_t w, int plane, int64_t m, int n) const {
    return sums + (((int64_t)w * PLANES + plane) * ROWS + m % ROWS) * COLS + n % COLS;
  }
  template <int W>
  __device__ __forceinline__ void store(S* to, const S (&v)[W]) const {
    vec<S, W> t;
#pragma unroll
    for (int j = 0; j < W; j++) t[j] = v[j];
    *reinterpret_cast<vec<S, W>*>(to) = t;
  }
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t w, int64_t m, int n, const S (&v)[W]) const {
    store<W>(at(w, 0, m, n), v);
  }
  template <int W>
  __device__ __forceinline__ void operator()(uint32_t w, int64_t m, int n, const S (&g)[W], const S (&u)[W]) const {
    store<W>(at(w, 0, m, n), g);
    store<W>(at(w, 1, m, n), u);
  }
};

// Adds the parts in their order and finishes them with the product's epilogue, eight columns a thread.
template <typename T, bool DUAL, int ROWS, int COLS, typename S, typename Epi, int NJ>
__global__ __launch_bounds__(256) void join_kernel(Jobs<T, Epi, NJ> jobs, uint32_t first, uint32_t count, int parts, S* sums) {
  constexpr int PL = DUAL ? 2 : 1, BLOCKS = ROWS * COLS / 2048;
  const Parts<S, ROWS, COLS, PL> p{sums};
  const uint32_t slot = blockIdx.x / BLOCKS, v0 = (blockIdx.x % BLOCKS * 256 + threadIdx.x) * 8;
  uint32_t tm, tn;
  const int job = find<Jobs<T, Epi, NJ>, NJ>(jobs, first + tile_of(slot, count), tm, tn);
  const int64_t m = (int64_t)tm * ROWS + v0 / COLS, n = (int64_t)tn * COLS + v0 % COLS;
  if (m >= jobs.product[job].M || n >= jobs.product[job].N) return;
  S v[PL][8] = {};
  for (int part = 0; part < parts; part++)
#pragma unroll
    for (int d = 0; d < PL; d++) {
      const vec<S, 8> t = *reinterpret_cast<const vec<S, 8>*>(p.at(part * count + slot, d, m, (int)n));
#pragma unroll
      for (int j = 0; j < 8; j++) v[d][j] += t[j];
    }
  if constexpr (DUAL) jobs.epi[job].template operator()<8>(0u, m, (int)n, v[0], v[1]);
  else jobs.epi[job].template operator()<8>(0u, m, (int)n, v[0]);
}

// ---- a few rows --------------------------------------------------------------------------------------------

// At most 16 MT rows of q against P: bound by reading P once. A workgroup takes 16 rows of P (DUAL: of each of the
// two), its eight waves every eighth 256-byte run of k; P goes from memory straight into the matrix instruction's
// registers, sixteen bytes of a row a lane, and q, which every workgroup reads again, comes from the caches. The
// eight sums meet in LDS and are added in a fixed order. No alignment is asked for. One row of a 4096-11264 block: gate and up
// 37 us (4.9 TB/s of weights), down 21 (4.4).
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
// Up to 8 rows by the kernel for a few, up to 32 where the tiles would need the weights copied first: 16 rows of a 4096-11264
// block take 78 us that way and 66 by tiles, one row 54.
inline bool few_rows(int64_t M, bool straight) { return M <= 8 || (M <= 32 && !straight); }

// Tiles of one size; the first `whole` of them each by one workgroup, the rest by `parts`, through `sums` bytes of workspace.
struct Way {
  int tile;
  int64_t whole, rest;
  int parts;
  size_t sums;
};
struct Extent {
  int64_t M, N;
};

// What `n` tiles of a size cost over `steps` steps of 128 bytes of k, in microseconds, fitted to 360 products of 64 to 8000 rows,
// 256 to 5504 columns and 256 to 5504 values of k, timed warm:
//   256x256, one a compute unit: a step takes 1.04 with half of them busy, 1.43 with all; 8 a round for its start and end.
//   128x128: 0.36 where a compute unit has one (four buffers), 0.9 for a round of two in each.
//   64x64: 0.27 up to one each, 0.4 up to two (three buffers), then 0.2 for each of several side by side.
// A large tile reads less, small ones keep more compute units at work when there are few: 4096 x 4096 x 4096 takes 100, 125 and
// 191 us, 1000 x 1024 x 1024 takes 25, 10 and 10.
inline double tile_time(int tile, int64_t n, double steps) {
  const double each = (double)n / 256;
  if (tile == TILE_256) {
    const double part = each - std::floor(each);
    return (1.43 * std::floor(each) + (part > 0 ? 1.04 + 0.39 * std::max(0.0, 2 * part - 1) : 0)) * steps + 8 * std::ceil(each);
  }
  if (tile == TILE_128) {
    if (n <= 256) return 0.365 * steps + 4.4;
    const double part = (each / 2 - std::floor(each / 2)) * 2;
    return (0.9 * std::floor(each / 2) + (part > 0 ? 0.64 + 0.26 * std::max(0.0, part - 1) : 0)) * steps + 3 + 3.2 * std::ceil(each / 2);
  }
  return (n <= 512 ? 0.265 + 0.14 * std::max(0.0, each - 1) : 0.2 * each) * steps + 3.1 + 0.35 * each;
}

// The cheapest way for products of these extents, `steps` long. Tiles beyond the last full round of compute units, or all of them
// where there are too few, may be split over k, for a write and a read of their sums at 5 TB/s. `moved`: bytes that the
// epilogue reads and writes for each value of out; several tiles in a compute unit hide a little of them.
inline Way choose(std::initializer_list<Extent> jobs, int64_t steps, bool dual, bool few, int moved = 2) {
  if (few) return {FEW_ROWS, 0, 0, 1, 0};
  Way best{TILE_64, 0, 0, 1, 0};
  double least = 1e30;
  for (int t = 0; t < 3; t++) {
    const int64_t side = t == TILE_256 ? 256 : t == TILE_128 ? 128 : 64, cols = dual ? side / 2 : side;
    const int64_t full = t == TILE_256 ? 256 : t == TILE_128 ? 512 : 1280;
    int64_t count = 0;
    double values = 0;
    for (const Extent& e : jobs) {
      count += up(e.M, side) / side * (up(e.N, cols) / cols);
      values += (double)e.M * (double)e.N;
    }
    const double end = values * (moved - 2) / 4.5e6 * (t == TILE_256 ? 0.55 : t == TILE_128 ? 0.5 : 0.4);
    const double all = tile_time(t, count, (double)steps) + end;
    if (all < least) least = all, best = {t, count, 0, 1, 0};
    for (const int64_t whole : {(int64_t)0, count / full * full}) {
      const int64_t rest = count - whole;
      for (int parts = 2; parts <= 64 && rest > 0; parts++) {
        const double sums = 4.0 * parts * (double)rest * (double)(side * side);
        if (steps / parts < 3 || sums > 256e6) break;
        const double us = (whole ? tile_time(t, whole, (double)steps) : 0) + tile_time(t, rest * parts, (double)((steps + parts - 1) / parts)) + 3 + 2 * sums / 5e6 + end;
        if (us < least) least = us, best = {t, whole, rest, parts, (size_t)sums};
      }
    }
  }
  return best;
}

template <typename T, bool PT, bool QT, bool DUAL, bool TWO, int SIDE, typename Epi, int NJ>
int launch_tiles(const Jobs<T, Epi, NJ>& jobs, int64_t first, int64_t count, int parts, hipStream_t stream) {
  if (count <= 0) return hipSuccess;
  if (count * parts * (SIDE == 64 ? 256 : 512) >= (int64_t)1 << 32) return hipErrorInvalidValue;  // no device memory holds that much
  const dim3 grid((unsigned)(count * parts));
  if constexpr (SIDE == 256)
    tile_kernel<T, PT, QT, DUAL, TWO, 2, 4, 128, 64, 2><<<grid, 512, 0, stream>>>(jobs, (uint32_t)first, (uint32_t)count, parts);
  else if constexpr (SIDE == 128) {
    if (count * parts <= 256)
      tile_kernel<T, PT, QT, DUAL, TWO, 2, 4, 64, 32, 4><<<grid, 512, 0, stream>>>(jobs, (uint32_t)first, (uint32_t)count, parts);
    else
      tile_kernel<T, PT, QT, DUAL, TWO, 2, 4, 64, 32, 2><<<grid, 512, 0, stream>>>(jobs, (uint32_t)first, (uint32_t)count, parts);
  } else {
    if (count * parts <= 512)
      tile_kernel<T, PT, QT, DUAL, TWO, 2, 2, 32, 32, 3><<<grid, 256, 0, stream>>>(jobs, (uint32_t)first, (uint32_t)count, parts);
    else
      tile_kernel<T, PT, QT, DUAL, TWO, 2, 2, 32, 32, 2><<<grid, 256, 0, stream>>>(jobs, (uint32_t)first, (uint32_t)count, parts);
  }
  return hipGetLastError();
}

template <typename T, bool PT, bool QT, bool DUAL, bool TWO, int SIDE, typename Epi, int NJ>
int run_tiles(Jobs<T, Epi, NJ>& jobs, const Way& way, void* sums, hipStream_t stream) {
  constexpr int COLS = DUAL ? SIDE / 2 : SIDE;
  for (int j = 0; j < NJ; j++) {
    jobs.tiles_m[j] = (uint32_t)(up(jobs.product[j].M, SIDE) / SIDE);
    jobs.tiles_n[j] = (uint32_t)(up(jobs.product[j].N, COLS) / COLS);
  }
  int rc = launch_tiles<T, PT, QT, DUAL, TWO, SIDE>(jobs, 0, way.whole, 1, stream);
  if (rc || way.rest == 0) return rc;
  using S = std::conditional_t<std::is_same_v<T, int8_t>, int, float>;
  using P = Parts<S, SIDE, COLS, DUAL ? 2 : 1>;
  Jobs<T, P, NJ> parts{};
  for (int j = 0; j < NJ; j++) {
    parts.product[j] = jobs.product[j];
    parts.epi[j] = P{(S*)sums};
    parts.tiles_m[j] = jobs.tiles_m[j];
    parts.tiles_n[j] = jobs.tiles_n[j];
  }
  rc = launch_tiles<T, PT, QT, DUAL, TWO, SIDE>(parts, way.whole, way.rest, way.parts, stream);
  if (rc) return rc;
  join_kernel<T, DUAL, SIDE, COLS, S><<<dim3((unsigned)(way.rest * (SIDE * COLS / 2048))), 256, 0, stream>>>(
      jobs, (uint32_t)way.whole, (uint32_t)way.rest, way.parts, (S*)sums);
  return hipGetLastError();
}

// Carries the jobs out the way that choose() gave for their extents; `sums`: its workspace.
template <typename T, bool PT, bool QT, bool DUAL, bool TWO, typename Epi, int NJ>
int products(Jobs<T, Epi, NJ>& jobs, const Way& way, void* sums, hipStream_t stream) {
  for (int j = 0; j < NJ; j++)
    if (jobs.product[j].M <= 0 || jobs.product[j].N <= 0) return hipSuccess;
  if constexpr (!PT && !QT && !TWO) {
    if (way.tile == FEW_ROWS) {
      const Product<T>& a = jobs.product[0];
      const dim3 grid((unsigned)(up(a.N, 16) / 16));
      if (a.M <= 16) few_rows_kernel<T, DUAL, 1><<<grid, 512, 0, stream>>>(a, jobs.epi[0]);
      else few_rows_kernel<T, DUAL, 2><<<grid, 512, 0, stream>>>(a, jobs.epi[0]);
      return hipGetLastError();
    }
  }
  if (way.tile == TILE_256) return run_tiles<T, PT, QT, DUAL, TWO, 256>(jobs, way, sums, stream);
  if (way.tile == TILE_128) return run_tiles<T, PT, QT, DUAL, TWO, 128>(jobs, way, sums, stream);
  return run_tiles<T, PT, QT, DUAL, TWO, 64>(jobs, way, sums, stream);
}
template <typename T, bool PT, bool QT, bool DUAL, bool TWO, typename Epi>
int product(const Product<T>& a, const Way& way, void* sums, const Epi& epi, hipStream_t stream) {
  Jobs<T, Epi, 1> one{{a}, {epi}, {0}, {0}};
  return products<T, PT, QT, DUAL, TWO>(one, way, sums, stream);
}

}  // namespace dev
}  // namespace b2c
