// The feed-forward block where its input and output are narrow (at most 128) and its rows many (is_head): a head over the splats
// of a scene. Written to memory and read back, the inner activations would be most of the traffic (g, u, h, dg, du of a
// 64-256-64 head: 2.5 KB a row beside 128 bytes of x), so they never leave the registers: the forward pass and the two
// halves of the backward pass each form g and u again from x. What bounds them then is the activation's arithmetic.
//
//   forward, input gradient: a wave owns rows. Hidden units come in chunks of 32: g^T = Wg x^T puts row l % 16 in lane l,
//     and with the rows of Wg dealt out as 8 (i / 4) + 4 t + i % 4 lane group l / 16 holds eight neighbouring hidden units
//     of two tiles t, which is the layout that the next product wants of its second operand. So h^T goes from one matrix
//     instruction to the next through arithmetic alone.
//   weight gradients: a wave owns hidden units, whose weights it keeps in registers with the sums of their gradients, and
//     passes over rows. g = x Wg^T then has hidden unit l % 16 in lane l and rows along the registers, the layout of an
//     operand that is summed over rows; the other operand, x by rows, is read from LDS transposed.
//
// Weights are first put in the order in which lanes read them ("fragments": 64 lanes x 16 bytes), zeros where a width ends.
#pragma once
#include "dense_product.h"

namespace b2c {
namespace dev {

enum { FOR_Y, FOR_DX, FOR_DW };

template <typename T>
struct HeadWeights {
  const T *wg, *wu, *wd;
  int64_t ld_in, ld_out;
  int D, F, O;
};

// Fragments of 32 hidden units (FOR_DW: of 16), KS x 32 values of input or output wide:
//   FOR_Y   g (t, k), u (t, k), down (o tile)
//   FOR_DX  g, u, down transposed (t, k), g transposed (d tile), u transposed (d tile)
//   FOR_DW  g (k), u (k), down transposed (k)
constexpr int fragments(int use, int ks) { return use == FOR_Y ? 6 * ks : use == FOR_DX ? 10 * ks : 3 * ks; }

template <typename T, int USE, int KS>
__device__ __forceinline__ vec<T, 8> fragment(const HeadWeights<T>& w, int c, int f, int lane) {
  const int i = lane & 15, q = lane >> 4;
  constexpr int WIDE = 8 * KS;  // neighbouring columns of an output that a lane holds
  vec<T, 8> v{};
  auto row_of = [&](const T* p, int64_t ld, int r, int R, int k, int K) {  // eight values along a row
    if (r >= R) return;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (k + j < K) v[j] = p[r * ld + k + j];
  };
  auto column_of = [&](const T* p, int64_t ld, int col, int C, int r, int R) {  // eight values down a column
    if (col >= C) return;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (r + j < R) v[j] = p[(int64_t)(r + j) * ld + col];
  };
  if constexpr (USE == FOR_DW) {
    const int h = c * 16 + i, k = f % KS * 32 + q * 8;
    if (f < KS) row_of(w.wg, w.ld_in, h, w.F, k, w.D);
    else if (f < 2 * KS) row_of(w.wu, w.ld_in, h, w.F, k, w.D);
    else column_of(w.wd, w.ld_out, h, w.F, k, w.O);
  } else {
    const int two = f % (2 * KS), t = two / KS, k = two % KS * 32 + q * 8;  // of the tiles whose rows are hidden units
    const int h = c * 32 + (i >> 2) * 8 + t * 4 + (i & 3);
    const int n = (i >> 2) * WIDE + two * 4 + (i & 3), hk = c * 32 + q * 8;  // of those whose rows are columns of the output
    const int s = f / (2 * KS);
    if (s == 0) row_of(w.wg, w.ld_in, h, w.F, k, w.D);
    else if (s == 1) row_of(w.wu, w.ld_in, h, w.F, k, w.D);
    else if (USE == FOR_Y) row_of(w.wd, w.ld_out, n, w.O, hk, w.F);
    else if (s == 2) column_of(w.wd, w.ld_out, h, w.F, k, w.O);
    else column_of(s == 3 ? w.wg : w.wu, w.ld_in, n, w.D, hk, w.F);
  }
  return v;
}

// A use's fragments, and with BOTH also those of FOR_DW, behind them.
template <typename T, int USE, bool BOTH, int KS>
__global__ __launch_bounds__(256) void fragments_kernel(HeadWeights<T> w, int chunks, T* out, int chunks_dw, T* out_dw) {
  const int lane = threadIdx.x & 63, n = fragments(USE, KS), all = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (all < chunks * n) {
    *reinterpret_cast<vec<T, 8>*>(out + ((int64_t)all * 64 + lane) * 8) = fragment<T, USE, KS>(w, all / n, all % n, lane);
  } else if constexpr (BOTH) {
    const int f = all - chunks * n, nd = fragments(FOR_DW, KS);
    if (f < chunks_dw * nd)
      *reinterpret_cast<vec<T, 8>*>(out_dw + ((int64_t)f * 64 + lane) * 8) = fragment<T, FOR_DW, KS>(w, f / nd, f % nd, lane);
  }
}

// Eight values of a row from column k on, zeros beyond the row's or the matrix's end.
template <typename T>
__device__ __forceinline__ vec<T, 8> eight(const T* p, int64_t ld, int64_t m, int64_t M, int k, int K) {
  vec<T, 8> v{};
  if (m >= M) return v;
  p += m * ld + k;
  if (k + 8 <= K) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (k + j < K) v[j] = p[j];
  }
  return v;
}
// The same of dy, zeros where dropout takes them.
template <typename T>
__device__ __forceinline__ vec<T, 8> eight_kept(const T* p, int64_t ld, int64_t m, int64_t M, int k, int K, const Drop& d) {
  vec<T, 8> v = eight(p, ld, m, M, k, K);
  if (d.threshold && m < M && k < K) {
    const uint32_t keep = kept_bits<8>(d, (uint64_t)m * K + k);
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (!(keep >> j & 1)) v[j] = (T)0.f;
  }
  return v;
}

template <typename T>
struct HeadRows {
  const T* x;
  int64_t ldx;
  const T* dy;
  int64_t lddy;
  int64_t M;
  int D, F, O;
  Drop drop;
  T* kept;  // FOR_DX: dy with dropout's zeros is left here for the weights' gradients, rows 32 KS apart; or null
};

// Rows by waves: y (USE = FOR_Y), or the gradient of x. RT tiles of 16 rows a wave; the chunks' fragments pass through two
// LDS buffers, copied there by the buffer unit while the chunk before is at work. 1M rows of 64-256-64: 153 us for y, 235 for
// dx; the vector unit issues for about two thirds of that, the matrix instructions take a quarter, and the two add up.
template <typename T, int ACT, int USE, int KS, int RT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void head_rows_kernel(HeadRows<T> a, const T* frags, int chunks, RowsOut<T> out) {
  constexpr int N = fragments(USE, KS), OT = 2 * KS;
  using F8 = vec<T, 8>;
  __shared__ __attribute__((aligned(1024))) F8 lds[2][N][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q4 = lane >> 4;
  const int64_t m0 = ((int64_t)block_index() * WAVES + wave) * (16 * RT) + (lane & 15);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)(char*)lds;

  auto start = [&](int c) {
#pragma unroll
    for (int j = 0; j < (N + WAVES - 1) / WAVES; j++) {
      const int f = j * WAVES + wave;
      if (f < N) copy_to_lds(frags + ((int64_t)c * N + f) * 512, lane * 16, lds0 + ((c & 1) * N + f) * 1024);
    }
  };
  start(0);
  F8 x[RT][KS], dz[USE == FOR_DX ? RT : 1][KS];
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int k = 0; k < KS; k++) {
      x[r][k] = eight(a.x, a.ldx, m0 + r * 16, a.M, k * 32 + q4 * 8, a.D);
      if constexpr (USE == FOR_DX) dz[r][k] = eight_kept(a.dy, a.lddy, m0 + r * 16, a.M, k * 32 + q4 * 8, a.O, a.drop);
    }
  if constexpr (USE == FOR_DX) {
    if (a.kept)
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int k = 0; k < KS; k++)
          if (m0 + r * 16 < a.M) *reinterpret_cast<F8*>(a.kept + (m0 + r * 16) * (32 * KS) + k * 32 + q4 * 8) = dz[r][k];
  }
  f32x4 acc[RT][OT] = {};
  for (int c = 0; c < chunks; c++) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (c + 1 < chunks) start(c + 1);
    const F8(&w)[N][64] = lds[c & 1];
    // Two row tiles to each read of the weights; the fence keeps the compiler from holding all of them in registers.
    constexpr int RG = RT < 2 ? RT : 2;
#pragma unroll
    for (int r0 = 0; r0 < RT; r0 += RG) {
      if (r0) asm volatile("" ::: "memory");
      f32x4 g[RG][2] = {}, u[RG][2] = {}, dh[RG][2] = {};
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
          for (int r = 0; r < RG; r++) {
            g[r][t] = mfma(w[t * KS + k][lane], x[r0 + r][k], g[r][t]);
            u[r][t] = mfma(w[(2 + t) * KS + k][lane], x[r0 + r][k], u[r][t]);
            if constexpr (USE == FOR_DX) dh[r][t] = mfma(w[(4 + t) * KS + k][lane], dz[r0 + r][k], dh[r][t]);
          }
      F8 h[RG], du[RG];  // FOR_DX: dg in h
#pragma unroll
      for (int r = 0; r < RG; r++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float gv = g[r][j / 4][j % 4], uv = u[r][j / 4][j % 4];
          if constexpr (USE == FOR_Y) {
            h[r][j] = (T)(act<ACT>(gv) * uv);
          } else {
            float av, dv;
            act_grad<ACT>(gv, av, dv);
            const float s = dh[r][j / 4][j % 4];  // dropout's scale follows at the end
            h[r][j] = (T)(s * uv * dv);
            du[r][j] = (T)(s * av);
          }
        }
#pragma unroll
      for (int t = 0; t < OT; t++)
#pragma unroll
        for (int r = 0; r < RG; r++) {
          if constexpr (USE == FOR_Y) {
            acc[r0 + r][t] = mfma(w[4 * KS + t][lane], h[r], acc[r0 + r][t]);
          } else {
            acc[r0 + r][t] = mfma(w[6 * KS + t][lane], h[r], acc[r0 + r][t]);
            acc[r0 + r][t] = mfma(w[8 * KS + t][lane], du[r], acc[r0 + r][t]);
          }
        }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; r++) {
    const int64_t m = m0 + r * 16;
    if (m >= a.M) continue;
#pragma unroll
    for (int h = 0; h < KS; h++) {
      const int n = q4 * 8 * KS + h * 8;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = USE == FOR_DX ? acc[r][2 * h + j / 4][j % 4] * a.drop.scale : acc[r][2 * h + j / 4][j % 4];
      if (n < out.cols) out.template operator()<8>(0u, m, n, v);
    }
  }
}

// Hidden units by waves, HT tiles of 16 each: the weights' gradients of part blockIdx.y of the rows. Rows pass through LDS in
// tiles of 64, x beside dz (dropout applied), each row's 16-byte pieces at (piece ^ row & 7) of its 128-byte blocks.
// sums: [part][3][chunks 16][32 KS]: dWg, dWu, dWd transposed. 1M rows of 64-256-64: 219 us, bound as the rows' kernel.
template <typename T, int ACT, int KS, int HT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, KS == 1 && WAVES == 4 ? 4 : 1) void head_weights_kernel(HeadRows<T> a, const T* frags,
                                                                                                int chunks, float* sums) {
  constexpr int KB = (KS + 1) / 2, R = 64, PIECES = R * 8 * KB / (WAVES * 64), OT = 2 * KS;
  static_assert(PIECES * WAVES * 64 == R * 8 * KB);
  using F8 = vec<T, 8>;
  __shared__ __attribute__((aligned(1024))) F8 lds[2][2][KB][R][8];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q4 = lane >> 4, i = lane & 15;
  const int c0 = (blockIdx.x * WAVES + wave) * HT;
  F8 wg[HT][KS], wu[HT][KS], wd[HT][KS];
#pragma unroll
  for (int t = 0; t < HT; t++)
#pragma unroll
    for (int k = 0; k < KS; k++) {
      const T* f = frags + ((int64_t)(c0 + t) * 3 * KS + k) * 512 + lane * 8;
      const bool there = c0 + t < chunks;
      wg[t][k] = there ? *reinterpret_cast<const F8*>(f) : F8{};
      wu[t][k] = there ? *reinterpret_cast<const F8*>(f + KS * 512) : F8{};
      wd[t][k] = there ? *reinterpret_cast<const F8*>(f + 2 * KS * 512) : F8{};
    }
  const int64_t tiles = (a.M + R - 1) / R;
  const int64_t first = tiles * blockIdx.y / gridDim.y, last = tiles * (blockIdx.y + 1) / gridDim.y;
  f32x4 sg[HT][OT] = {}, su[HT][OT] = {}, sd[HT][OT] = {};

  F8 next_x[PIECES], next_dz[PIECES];
  auto fetch = [&](int64_t tile) {
#pragma unroll
    for (int j = 0; j < PIECES; j++) {
      const int s = (int)threadIdx.x + j * WAVES * 64, piece = s % (8 * KB);
      const int64_t m = tile * R + s / (8 * KB);
      next_x[j] = eight(a.x, a.ldx, m, a.M, piece * 8, a.D);
      next_dz[j] = eight_kept(a.dy, a.lddy, m, a.M, piece * 8, a.O, a.drop);
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int j = 0; j < PIECES; j++) {
      const int s = (int)threadIdx.x + j * WAVES * 64, piece = s % (8 * KB), row = s / (8 * KB);
      lds[buf][0][piece / 8][row][(piece & 7) ^ (row & 7)] = next_x[j];
      lds[buf][1][piece / 8][row][(piece & 7) ^ (row & 7)] = next_dz[j];
    }
  };
  // rows row0 + i, piece q4 of k step k
  auto along = [&](int buf, int side, int row0, int k) {
    const int row = row0 + i, piece = k * 4 + q4;
    return lds[buf][side][piece / 8][row][(piece & 7) ^ (row & 7)];
  };
  // column 16 t + i, rows row0 + 4 q4 .. + 3 and 16 further
  auto down = [&](int buf, int side, int row0, int t) {
    const int piece = t * 2 + (i >> 1 & 1), row = row0 + q4 * 4 + (i >> 2);
    const char* p = (const char*)&lds[buf][side][piece / 8][row][(piece & 7) ^ (row & 7)] + (i & 1) * 8;
    return join<T>(read_transposed(p), read_transposed(p + 16 * 128));
  };

  if (first < last) fetch(first);
  for (int64_t tile = first; tile < last; tile++) {
    const int buf = (int)(tile - first) & 1;
    store(buf);
    __syncthreads();
    if (tile + 1 < last) fetch(tile + 1);
    if (c0 >= chunks) continue;  // a wave without hidden units only helps to move rows
#pragma unroll 1
    for (int row0 = 0; row0 < R; row0 += 32) {
      F8 h[HT], dg[HT], du[HT];
      f32x4 g[2][HT] = {}, u[2][HT] = {}, dh[2][HT] = {};
#pragma unroll
      for (int r = 0; r < 2; r++)
#pragma unroll
        for (int k = 0; k < KS; k++) {
          const F8 x = along(buf, 0, row0 + r * 16, k), dz = along(buf, 1, row0 + r * 16, k);
#pragma unroll
          for (int t = 0; t < HT; t++) {
            g[r][t] = mfma(x, wg[t][k], g[r][t]);
            u[r][t] = mfma(x, wu[t][k], u[r][t]);
            dh[r][t] = mfma(dz, wd[t][k], dh[r][t]);
          }
        }
#pragma unroll
      for (int t = 0; t < HT; t++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float uv = u[j / 4][t][j % 4];
          float av, dv;
          act_grad<ACT>(g[j / 4][t][j % 4], av, dv);
          const float s = dh[j / 4][t][j % 4];  // dropout's scale follows when the parts are added
          h[t][j] = (T)(av * uv);
          dg[t][j] = (T)(s * uv * dv);
          du[t][j] = (T)(s * av);
        }
#pragma unroll
      for (int o = 0; o < OT; o++) {
        const F8 x = down(buf, 0, row0, o), dz = down(buf, 1, row0, o);
#pragma unroll
        for (int t = 0; t < HT; t++) {
          sg[t][o] = mfma(x, dg[t], sg[t][o]);
          su[t][o] = mfma(x, du[t], su[t][o]);
          sd[t][o] = mfma(dz, h[t], sd[t][o]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < HT; t++) {
    if (c0 + t >= chunks) continue;
    const int64_t hid = (int64_t)(c0 + t) * 16 + i, plane = (int64_t)chunks * 16 * (32 * KS);
    float* to = sums + (int64_t)blockIdx.y * 3 * plane + hid * (32 * KS) + q4 * 4;
#pragma unroll
    for (int o = 0; o < OT; o++) {
      *reinterpret_cast<f32x4*>(to + o * 16) = sg[t][o];
      *reinterpret_cast<f32x4*>(to + plane + o * 16) = su[t][o];
      *reinterpret_cast<f32x4*>(to + 2 * plane + o * 16) = sd[t][o];
    }
  }
}

// Adds the parts in a fixed order and writes the gradients: four columns a thread, 32 threads to them, each for every 32nd
// part (12 us for the 50 MB of 256 parts of 64-256-64).
template <typename T>
__global__ __launch_bounds__(256) void head_join_kernel(const float* sums, int64_t hidden, int wide, int parts, int F, int D, int O,
                                                        WeightOut<T> in, WeightOut<T> down) {
  __shared__ f32x4 some[32][8];
  const int64_t plane = hidden * wide, at = ((int64_t)blockIdx.x * 8 + (threadIdx.x & 7)) * 4;
  const int g = threadIdx.x >> 3;
  f32x4 v = {};
#pragma unroll 8
  for (int p = g; p < parts; p += 32) v += *reinterpret_cast<const f32x4*>(sums + (int64_t)p * 3 * plane + at);
  some[g][threadIdx.x & 7] = v;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int j = 1; j < 32; j++) v += some[j][threadIdx.x];
  const int which = (int)(at / plane), h = (int)((at - which * plane) / wide), n = (int)((at - which * plane) % wide);
  if (h >= F) return;
  float o[4] = {v[0], v[1], v[2], v[3]};
  if (which < 2) {
    if (n < D) in.template operator()<4>(0u, which == 0 ? h : in.second + h, n, o);
  } else if (down.a) {  // transposed: one value of four rows
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (n + j < O) {
        const float one[1] = {o[j]};
        down.template operator()<1>(0u, n + j, h, one);
      }
  }
}

// ---- host --------------------------------------------------------------------------------------------------

// Whether a block is such a head: narrow, and its rows, 64 to a workgroup, give every compute unit one, since a workgroup passes over
// the whole hidden width by itself. Steps in microseconds, this way and by tiles through memory: 16384 rows of 64-512-64 69 and
// 64, of 64-2048-64 167 and 236, of 128-2048-128 244 and 251; 4096 rows of 64-512-64 65 and 43, of 64-2048-64 147 and 68; 40 rows
// of 96-8192-96 696 and 57; 32768 rows of 64-512-64 77 and 110. Up to 64 hidden units the two are alike for fewer rows (1024
// rows of 64-64-64: 24 and 25), and this one keeps nothing between its passes; but the weights are rearranged in each call, which a few rows do not pay for.
inline bool is_head(const b2c_ffn_args* a) {
  return a->d_in <= 128 && a->d_out <= 128 && (a->rows >= 64 * 256 || (a->rows > 32 && a->d_hidden <= 64));
}
inline int head_steps(const b2c_ffn_args* a) {
  const int n = (int)(up(std::max(a->d_in, a->d_out), 32) / 32);
  return n == 3 ? 4 : n;
}

// How the weights' gradients are shared out: tiles of 16 hidden units a wave (two where the registers take them), workgroups
// of eight waves along the hidden units (four where there are few), parts of the rows: as many workgroups as the compute
// units hold: one of eight waves (a step of 1M rows of 64-256-64 took 679 us with 512 where 256 take 661), four of four waves
// (600k rows of 16-32-16 took 93 us with 768 of them, 84 with 1024).
struct HeadSplit {
  int ht, waves, blocks, parts;
  int64_t chunks;
  HeadSplit(const b2c_ffn_args* a) {
    chunks = up(a->d_hidden, 16) / 16;
    ht = head_steps(a) <= 2 && up(a->d_hidden, 256) == up(a->d_hidden, 128) ? 2 : 1;
    waves = chunks <= 4 ? 4 : 8;
    blocks = (int)(up(chunks, waves * ht) / (waves * ht));
    parts = (int)std::max<int64_t>(1, std::min<int64_t>(up(a->rows, 64) / 64, (waves == 4 ? 1024 : 256) / blocks));
  }
  int64_t sums(int ks) const { return (int64_t)parts * 3 * chunks * 16 * 32 * ks; }
};

template <typename T>
struct HeadPlan {
  int ks, chunks;  // of 32 hidden units
  T *for_y = nullptr, *for_dx = nullptr, *for_dw = nullptr, *kept = nullptr;
  float* sums = nullptr;
  HeadPlan(const b2c_ffn_args* a, const b2c_ffn_grad_args* b, Room& room) {
    ks = head_steps(a);
    chunks = (int)(up(a->d_hidden, 32) / 32);
    const HeadSplit split(a);
    if (!b) {
      for_y = room.take<T>((int64_t)chunks * fragments(FOR_Y, ks) * 512);
      return;
    }
    if (b->dx) for_dx = room.take<T>((int64_t)chunks * fragments(FOR_DX, ks) * 512);
    if (b->dw_gate || b->dw_up || b->dw_down) {
      for_dw = room.take<T>(split.chunks * fragments(FOR_DW, ks) * 512);
      sums = room.take<float>(split.sums(ks));
      if (b->dx && b->fwd.p > 0.f) kept = room.take<T>(a->rows * 32 * ks);
    }
  }
};

template <typename T, int USE, bool BOTH, int KS>
int make_fragments(const b2c_ffn_args* a, int64_t chunks, T* to, int64_t chunks_dw, T* to_dw, hipStream_t stream) {
  const HeadWeights<T> w{(const T*)a->w_gate, (const T*)a->w_up, (const T*)a->w_down, a->ld_in, a->ld_out, a->d_in, a->d_hidden, a->d_out};
  const int64_t blocks = up(chunks * fragments(USE, KS) + (BOTH ? chunks_dw * fragments(FOR_DW, KS) : 0), 4) / 4;
  if (blocks > 0x7fffff) return hipErrorInvalidValue;
  fragments_kernel<T, USE, BOTH, KS><<<dim3((unsigned)blocks), 256, 0, stream>>>(w, (int)chunks, to, (int)chunks_dw, to_dw);
  return hipGetLastError();
}

// Four waves of two row tiles each (of one where the widths fill the registers) where that gives every compute unit its three
// workgroups, else of one. A training step of 1M rows of 64-256-64 took 756 us with eight waves of four tiles, 729 with four of
// four, 690 with four of two: what counts is that a compute unit's workgroups are out of step, so that one's matrix
// instructions meet another's arithmetic.
template <typename T, int ACT, int USE, int KS>
int head_rows(const HeadRows<T>& rows, const T* frags, int chunks, const RowsOut<T>& out, hipStream_t stream) {
  constexpr int RT = KS == 4 ? 1 : 2;
  const int64_t many = up(rows.M, 64 * RT) / (64 * RT), few = up(rows.M, 64) / 64;
  if (RT == 1 || many < 768) head_rows_kernel<T, ACT, USE, KS, 1, 4><<<grid_of(few), 256, 0, stream>>>(rows, frags, chunks, out);
  else head_rows_kernel<T, ACT, USE, KS, RT, 4><<<grid_of(many), 256, 0, stream>>>(rows, frags, chunks, out);
  return hipGetLastError();
}

template <typename T, int ACT, int KS>
int head_forward(const b2c_ffn_args* a, const Drop& d, hipStream_t stream) {
  Room room{(char*)a->workspace};
  const HeadPlan<T> p(a, nullptr, room);
  const int rc = make_fragments<T, FOR_Y, false, KS>(a, p.chunks, p.for_y, 0, nullptr, stream);
  if (rc) return rc;
  const HeadRows<T> rows{(const T*)a->x, a->ldx, nullptr, 0, a->rows, a->d_in, a->d_hidden, a->d_out, {}, nullptr};
  const RowsOut<T> out{(T*)a->y, a->ldy, (const T*)a->residual, a->ldr, a->d_out, d};
  return head_rows<T, ACT, FOR_Y, KS>(rows, p.for_y, p.chunks, out, stream);
}

template <typename T, int ACT, int KS>
int head_backward(const b2c_ffn_grad_args* b, const Drop& d, hipStream_t stream) {
  const b2c_ffn_args* a = &b->fwd;
  Room room{(char*)b->workspace};
  const HeadPlan<T> p(a, b, room);
  HeadRows<T> rows{(const T*)a->x, a->ldx, (const T*)b->dy, b->lddy, a->rows, a->d_in, a->d_hidden, a->d_out, d, p.kept};
  rows.drop.scale = d.threshold ? d.scale : 1.f;
  const bool weights = b->dw_gate || b->dw_up || b->dw_down;
  const HeadSplit split(a);
  int rc = hipSuccess;
  if (b->dx) {
    rc = weights ? make_fragments<T, FOR_DX, true, KS>(a, p.chunks, p.for_dx, split.chunks, p.for_dw, stream)
                 : make_fragments<T, FOR_DX, false, KS>(a, p.chunks, p.for_dx, 0, nullptr, stream);
    if (rc) return rc;
    const RowsOut<T> out{(T*)b->dx, b->lddx, nullptr, 0, a->d_in, {}};
    if ((rc = head_rows<T, ACT, FOR_DX, KS>(rows, p.for_dx, p.chunks, out, stream))) return rc;
  } else if (weights) {
    if ((rc = make_fragments<T, FOR_DW, false, KS>(a, split.chunks, p.for_dw, 0, nullptr, stream))) return rc;
  }
  if (!weights) return hipSuccess;
  if (p.kept) {  // dropout's bits cost as much as a third of a pass over the rows
    rows.dy = p.kept;
    rows.lddy = 32 * KS;
    rows.drop.threshold = 0;
  }
  const dim3 grid((unsigned)split.blocks, (unsigned)split.parts);
  const int chunks = (int)split.chunks;
  if (split.waves == 4) {
    head_weights_kernel<T, ACT, KS, 1, 4><<<grid, 256, 0, stream>>>(rows, p.for_dw, chunks, p.sums);
  } else if constexpr (KS <= 2) {
    if (split.ht == 2) head_weights_kernel<T, ACT, KS, 2, 8><<<grid, 512, 0, stream>>>(rows, p.for_dw, chunks, p.sums);
    else head_weights_kernel<T, ACT, KS, 1, 8><<<grid, 512, 0, stream>>>(rows, p.for_dw, chunks, p.sums);
  } else {
    head_weights_kernel<T, ACT, KS, 1, 8><<<grid, 512, 0, stream>>>(rows, p.for_dw, chunks, p.sums);
  }
  if ((rc = hipGetLastError())) return rc;
  const bool f32 = b->grad_dtype == B2C_F32, add = b->accumulate != 0;
  const WeightOut<T> in{b->dw_gate, b->dw_up, b->ld_din, a->d_hidden, a->d_hidden, a->d_in, f32, add, rows.drop.scale};
  const WeightOut<T> down{b->dw_down, nullptr, b->ld_dout, a->d_out, 0, a->d_hidden, f32, add, rows.drop.scale};
  const int64_t hidden = split.chunks * 16, blocks = 3 * hidden * KS;
  head_join_kernel<T><<<dim3((unsigned)blocks), 256, 0, stream>>>(p.sums, hidden, 32 * KS, split.parts, a->d_hidden, a->d_in, a->d_out, in,
                                                                  down);
  return hipGetLastError();
}

// One instance for each type, each in a file of its own.
template <typename T>
int head_forward(const b2c_ffn_args* a, const Drop& d, hipStream_t stream);
template <typename T>
int head_backward(const b2c_ffn_grad_args* b, const Drop& d, hipStream_t stream);

template <typename T, int ACT>
int head_forward_by_width(const b2c_ffn_args* a, const Drop& d, hipStream_t s) {
  const int ks = head_steps(a);
  return ks == 1 ? head_forward<T, ACT, 1>(a, d, s) : ks == 2 ? head_forward<T, ACT, 2>(a, d, s) : head_forward<T, ACT, 4>(a, d, s);
}
template <typename T, int ACT>
int head_backward_by_width(const b2c_ffn_grad_args* b, const Drop& d, hipStream_t s) {
  const int ks = head_steps(&b->fwd);
  return ks == 1 ? head_backward<T, ACT, 1>(b, d, s) : ks == 2 ? head_backward<T, ACT, 2>(b, d, s) : head_backward<T, ACT, 4>(b, d, s);
}

}  // namespace dev
}  // namespace b2c
