// The tiled matrix product behind the dense operators: out[m][n] = sum_k Q[m][k] P[n][k], with an epilogue.
//
// A workgroup computes BM x BN of out in steps of 128 bytes of k (64 values of 16 bits, 128 of 8). Both operands'
// next step is copied from memory to LDS by the buffer unit itself while the current one is multiplied: two
// to four buffers, one barrier a step, no registers in between. A copy instruction writes 64 pieces of 16 bytes in lane order,
// so any rearrangement is done on the side of the addresses it reads:
//   - rows along k ("plain" operand, element (i, k) at p[i ld + k]): row i's eight pieces are stored at
//     (piece ^ i & 7), so that the sixteen rows that a matrix instruction's lanes read lie in different banks;
//   - rows along i ("transposed", element (i, k) at p[k ld + i]): stored as they are, the pieces of row k at
//     (piece ^ 2 key(k)), and read with the transposing LDS load, which hands lane l of each sixteen the four
//     values that column l has in four rows.
// Pieces beyond an operand's edge are read as zeros: their lanes are given an offset outside the buffer's range.
//
// Bound by the matrix instructions and, over a long run, by the clock that their power leaves: 4096 x 4096 x 11264 with tiles
// of 256x256 takes 257 us in bfloat16 (1.47 PFLOP/s), 138 in 8 bits (2.73 POP/s); 272 within a 4096-11264 block's pass.
#pragma once
#include "dense.h"

namespace b2c {
namespace dev {

constexpr uint32_t kOutside = 0x80000000u;  // an offset beyond every buffer range used here (2 GiB)

// 16 bytes a lane from base + offset to LDS at `lds` + 16 lane. In assembly, since the compiler would wait for
// every copy in flight before each LDS read; the kernel waits once a step.
__device__ __forceinline__ void copy_to_lds(const void* base, uint32_t offset, uint32_t lds) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const vec<uint32_t, 4> rsrc = {(uint32_t)b, (uint32_t)(b >> 32) & 0xffffu, kOutside, 0x00020000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rsrc)
               : "m0", "memory");
}

template <typename T>
__device__ __forceinline__ vec<T, 8> join(vec<short, 4> a, vec<short, 4> b) {
  return __builtin_bit_cast(vec<T, 8>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ vec<short, 4> read_transposed(const char* lds) {
  using L = __attribute__((address_space(3))) vec<short, 4>;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(lds));
}

// Operand of a tile: R rows of i from i0 on, of I; `trans` as above. Rows k of K.
template <typename T, int R, int THREADS, bool TRANS>
struct Tile {
  static constexpr int V = Elem<T>::N, BK = 128 / sizeof(T);
  static constexpr int BYTES = R * 128, COPIES = BYTES / (THREADS * 16);
  static constexpr int PIECES = TRANS ? R / V : 8;  // of a stored row
  static constexpr int key_of(int k) { return k & (PIECES / 2 - 1); }
  static_assert(COPIES >= 1 && COPIES * THREADS * 16 == BYTES);
  uint32_t off[COPIES];
  int kpos[TRANS ? COPIES : 1];  // this lane's k within a step

  // `row_of`: which row of the operand is stored at LDS row r (plain operands)
  template <typename RowOf>
  __device__ __forceinline__ void init(int64_t ld, int64_t i0, int64_t I, int wave, int lane, RowOf row_of) {
#pragma unroll
    for (int j = 0; j < COPIES; j++) {
      const uint32_t piece = (uint32_t)((wave * COPIES + j) * 64 + lane);
      const int r = (int)(piece / PIECES), s = (int)(piece % PIECES);
      if constexpr (!TRANS) {
        const int64_t i = (int64_t)row_of(r);
        kpos[0] = (s ^ (r & 7)) * V;
        off[j] = i0 + i < I ? (uint32_t)((i * ld + kpos[0]) * (int64_t)sizeof(T)) : kOutside;
      } else {
        const int key = key_of(r & 3 | (r >> 3 & 1) << 2), c = (s ^ key << 1) * V;
        kpos[j] = r;
        off[j] = i0 + c < I ? (uint32_t)(((int64_t)r * ld + c) * (int64_t)sizeof(T)) : kOutside;
      }
    }
  }
  // Starts the copies of the step whose first k is k0; `base`: element (i0, k0).
  __device__ __forceinline__ void copy(int j, const void* base, uint32_t lds, int wave, int left) const {
    const uint32_t o = kpos[TRANS ? j : 0] < left ? off[j] : kOutside;
    copy_to_lds(base, o, lds + (uint32_t)((wave * COPIES + j) * 1024));
  }
};

// The 16 x (16 bytes of k) fragments of a wave's rows w0 .. in an operand's LDS tile.
template <typename T, int R, bool TRANS>
struct Fragments {
  static constexpr int V = Elem<T>::N;
  int base;       // plain: byte offset of (row l % 16, piece 0)
  int sw;         // plain: this lane's row & 7
  int q, key, col;
  __device__ __forceinline__ void init(int w0, int lane) {
    q = lane >> 4;
    if constexpr (!TRANS) {
      base = (w0 + (lane & 15)) * 128;
      sw = lane & 7;
    } else {
      const int i = lane & 15;
      key = ((i >> 2) | (q & 1) << 2) & (R / V / 2 - 1);
      base = (q * 8 + (i >> 2)) * (R * 2) + (i & 1) * 8;
      col = w0 / 8 + (i >> 1 & 1);
    }
  }
  // Tile t (16 rows), half kk of the step.
  __device__ __forceinline__ vec<T, V> get(const char* lds, int t, int kk) const {
    if constexpr (!TRANS) {
      return *reinterpret_cast<const vec<T, V>*>(lds + base + t * 2048 + ((kk * 4 + q) ^ sw) * 16);
    } else {
      const char* p = lds + base + ((col + t * 2) ^ key << 1) * 16 + kk * 32 * (R * 2);
      return join<T>(read_transposed(p), read_transposed(p + 4 * (R * 2)));
    }
  }
};

// Which of `count` neighbouring tiles workgroup `slot` takes: workgroups go to the eight dies in turn, and each die takes a run.
__device__ __forceinline__ uint32_t tile_of(uint32_t slot, uint32_t count) {
  const uint32_t die = slot % 8, per = count / 8, more = count % 8;
  return die * per + (die < more ? die : more) + slot / 8;
}
// Tile t -> (m tile, n tile): down four m tiles before the next n tile, so that a die's cache holds both operands' rows for a
// while.
__device__ __forceinline__ void place(uint32_t t, uint32_t tiles_m, uint32_t tiles_n, uint32_t& tm, uint32_t& tn) {
  constexpr uint32_t group = 4;
  const uint32_t g = t / (group * tiles_n), first = g * group;
  const uint32_t rows = tiles_m - first < group ? tiles_m - first : group, r = t - g * group * tiles_n;
  tn = r / rows;
  tm = first + r - tn * rows;
}

// A product: operands p, q (and with TWO, after K values of k, p2, q2 for K2 more, rows as far apart), or with DUAL two
// products that share q (p the gate's weights, p2 the up projection's, rows as far apart; the epilogue gets both).
template <typename T>
struct Product {
  Side<T> q, p, q2, p2;
  int64_t M, N, K, K2;
  int64_t q_lim, p_lim;  // how far m and n may be read in the operands; what lies beyond counts as zeros
};

// One or two products of a kind, to be carried out together; the second's tiles follow the first's.
template <typename T, typename Epi, int N>
struct Jobs {
  Product<T> product[N];
  Epi epi[N];
  uint32_t tiles_m[N], tiles_n[N];
};

// Tile t of the jobs: which job's, and where in it.
template <typename J, int N>
__device__ __forceinline__ int find(const J& jobs, uint32_t t, uint32_t& tm, uint32_t& tn) {
  int job = 0;
  if constexpr (N == 2) {
    const uint32_t first = jobs.tiles_m[0] * jobs.tiles_n[0];
    if (t >= first) job = 1, t -= first;
  }
  place(t, jobs.tiles_m[job], jobs.tiles_n[job], tm, tn);
  return job;
}

// A product whose P has a scale for every row and group of 2^shift values of k: out[m][n] = sum_g scale[g][n] sum_(k in g) Q[m][k] P[n][k],
// so that P may hold whole numbers, which 16 bits hold exactly. Such a product's epilogue has a member `scales`. Each group's sum is added to
// the whole one when the group ends, in a second set of accumulators, for which tiles of 256x256 have no registers. The scales come to LDS
// beside the step's values. 2048 x 4096-11264 takes 187 us with groups of 128, 214 with groups of 32, and 171 without scales in
// tiles of 256x256.
struct GroupScales {
  const float* p;  // [ceil(K / 2^shift)][pitch], pitch a multiple of the tile's width
  int64_t pitch;
  int shift;
};
template <typename Epi>
constexpr int groups_of_step() {  // 0: a product without
  if constexpr (requires(Epi e) { e.scales; }) return Epi::GROUPS;
  else return 0;
}

// Waves that a SIMD has to hold: what a workgroup of `waves` needs, and two of eight waves where a product has scales, whose second accumulators
// would leave room for one.
template <typename Epi>
constexpr int least_waves(int waves, int stages) {
  return waves / 4 * (groups_of_step<Epi>() && waves == 8 && stages == 2 ? 2 : 1);
}

// Tiles first .. first + count - 1 of the jobs, each in `parts` parts of its k: workgroup part count + slot. The epilogue is
// told the workgroup too.
template <typename T, bool PT, bool QT, bool DUAL, bool TWO, int WAVES_M, int WAVES_N, int WM, int WN, int STAGES, typename Epi, int NJ>
__global__ __launch_bounds__(WAVES_M* WAVES_N * 64, least_waves<Epi>(WAVES_M * WAVES_N, STAGES)) void tile_kernel(
    Jobs<T, Epi, NJ> jobs, uint32_t first, uint32_t count, int parts) {
  constexpr int THREADS = WAVES_M * WAVES_N * 64, BM = WAVES_M * WM, BN = WAVES_N * WN;
  constexpr bool AHEAD = WAVES_M * WAVES_N == 8;
  constexpr int MT = WM / 16, NT = WN / 16, COLS = DUAL ? BN / 2 : BN;  // columns of out in a tile
  using Acc = typename Elem<T>::Acc;
  using TQ = Tile<T, BM, THREADS, QT>;
  using TP = Tile<T, BN, THREADS, PT>;
  static_assert(!DUAL || (!PT && !TWO));
  constexpr int STEP = TQ::BYTES + TP::BYTES, BK = TQ::BK;
  constexpr int GROUPS = groups_of_step<Epi>();  // of a step: 2 where they have half its length, 1 where one or more steps make a group
  static_assert(GROUPS * BN <= 256 && !(GROUPS && (DUAL || TWO)));
  constexpr int RING = 2 * STAGES;  // steps whose scales are held, so that they are read after the step
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * STEP + (GROUPS ? RING * 1024 : 0)];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t part = blockIdx.x / count;
  uint32_t tm, tn;
  const int job = find<Jobs<T, Epi, NJ>, NJ>(jobs, first + tile_of(blockIdx.x - part * count, count), tm, tn);
  const Product<T>& a = jobs.product[job];
  const Epi& epi = jobs.epi[job];
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * COLS;
  const int wm = wave % WAVES_M * WM, wb = wave / WAVES_M, wn = wb * WN;

  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const int steps1 = (int)((a.K + BK - 1) / BK), all = steps1 + (TWO ? (int)((a.K2 + BK - 1) / BK) : 0);
  const int begin = (int)((int64_t)all * part / parts), steps = (int)((int64_t)all * (part + 1) / parts) - begin;

  TQ cq;
  TP cp;
  auto q_row = [](uint32_t r) { return r; };
  auto p_row = [](uint32_t r) {  // DUAL: a wave's block of rows is half gate, half up
    if constexpr (DUAL) return r / WN * (WN / 2) + r % (WN / 2);
    else return r;
  };
  const T *pq = nullptr, *pp = nullptr, *pu = nullptr;
  int left = 0;
  auto enter = [&](int seg, int step) {  // a segment's step
    const Side<T>&Q = seg ? a.q2 : a.q, &P = seg && !DUAL ? a.p2 : a.p;
    pq = Q.p + (QT ? m0 : m0 * Q.ld);
    pp = P.p + (PT ? n0 : n0 * P.ld);
    if constexpr (DUAL) pu = a.p2.p + n0 * a.p2.ld;
    left = (int)(seg ? a.K2 : a.K) - step * BK;
    pq += QT ? (int64_t)step * BK * a.q.ld : step * BK;
    pp += PT ? (int64_t)step * BK * a.p.ld : step * BK;
    if constexpr (DUAL) pu += step * BK;
    cq.init(Q.ld, m0, a.q_lim, wave, lane, q_row);
    cp.init(P.ld, n0, a.p_lim, wave, lane, p_row);
  };
  constexpr int COPIES = TQ::COPIES + TP::COPIES;
  // The scales of the groups of the step that is copied, a copy of one wave: it waits for one copy more than it has to.
  auto copy_scales = [&](int s) {
    if constexpr (GROUPS > 0) {
      if (wave != 0) return;
      constexpr int LANES = BN / 4;
      const GroupScales& g = epi.scales;
      const int k = (int)a.K - left + lane / LANES * (BK / GROUPS);
      const bool there = lane < GROUPS * LANES && k < a.K;
      const uint32_t o = there ? (uint32_t)(((int64_t)(lane / LANES) * g.pitch + lane % LANES * 4) * (int64_t)sizeof(float)) : kOutside;
      copy_to_lds(g.p + n0 + (((int)a.K - left) >> g.shift) * g.pitch, o, lds0 + STAGES * STEP + (uint32_t)s % RING * 1024);
    }
  };
  auto copy = [&](int s, int j) {  // copy j of step s; beyond the last step `left` makes it one of zeros
    const uint32_t to = lds0 + (uint32_t)s % STAGES * STEP;
    if (j < TQ::COPIES) {
      cq.copy(j, pq, to, wave, left);
    } else {
      j -= TQ::COPIES;
      const T* base = pp;
      if constexpr (DUAL) {  // eight LDS rows a copy, all of one of the two
        const int r = (wave * TP::COPIES + j) * 8;
        base = r % WN >= WN / 2 ? pu : pp;
      }
      cp.copy(j, base, to + TQ::BYTES, wave, left);
    }
  };
  auto advance = [&](int s) {  // from step s to the next
    left -= BK;
    if (TWO && begin + s + 1 == steps1) {
      enter(1, 0);
    } else {
      pq += QT ? BK * a.q.ld : BK;
      pp += PT ? BK * a.p.ld : BK;
      if constexpr (DUAL) pu += BK;
    }
  };
  auto start = [&](int s) {
    copy_scales(s);
#pragma unroll
    for (int j = 0; j < COPIES; j++) copy(s, j);
    advance(s);
  };

  Fragments<T, BM, QT> fq;
  Fragments<T, BN, PT> fp;
  fq.init(wm, lane);
  fp.init(wn, lane);
  Acc acc[NT][MT] = {}, sum[GROUPS ? NT : 1][GROUPS ? MT : 1] = {};
  // Adds the group's sums that end with half g of step s (GROUPS: 2), or with the step, if one ends there or the part does.
  auto add_group = [&](int s, int g) {
    if constexpr (GROUPS > 0) {
      if (GROUPS == 1 && ((begin + s + 1) * BK & ((1 << epi.scales.shift) - 1)) && s != steps - 1) return;
      const char* at = lds + STAGES * STEP + (uint32_t)s % RING * 1024 + (g * BN + wn + (lane >> 4) * 4) * 4;
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const Acc scale = *reinterpret_cast<const Acc*>(at + j * 64);
#pragma unroll
        for (int i = 0; i < MT; i++) {
#pragma unroll
          for (int e = 0; e < 4; e++) sum[j][i][e] = fmaf(scale[e], acc[j][i][e], sum[j][i][e]);
          acc[j][i] = Acc{};
        }
      }
    }
  };
  using F = vec<T, TQ::V>;
  F q0[MT], p0[NT], q1[MT], p1[NT];
  auto read = [&](int s, int kk, F(&q)[MT], F(&p)[NT]) {
    const char* at = lds + (uint32_t)s % STAGES * STEP;
#pragma unroll
    for (int t = 0; t < NT; t++) p[t] = fp.get(at + TQ::BYTES, t, kk);
#pragma unroll
    for (int t = 0; t < MT; t++) q[t] = fq.get(at, t, kk);
  };
  auto multiply = [&](const F(&q)[MT], const F(&p)[NT]) {
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) acc[j][i] = mfma(p[j], q[i], acc[j][i]);
  };
  // This wave's copies are in LDS, but for those of the last LATER steps, and its reads done; then everybody's.
  auto landed = [](auto later) {
    constexpr int n = decltype(later)::value * COPIES;
    static_assert(n < 64);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(n) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  using All = std::integral_constant<int, 0>;
  // Multiplies one half's fragments while those of another are read from buffer `at`, spread over the first three
  // quarters, and with COPY the copies of step s are started, spread too: a wave issues in order, and the address unit
  // takes 16 cycles for each copy, so eight waves' copies in a row would hold up all of them for a thousand cycles.
  auto half = [&](const F(&q)[MT], const F(&p)[NT], F(&qn)[MT], F(&pn)[NT], const char* at, int kk, auto with_copies, int s) {
    constexpr int READS = MT + NT, SLOTS = MT * 3 / 4;
#pragma unroll
    for (int i = 0; i < MT; i++) {
      if constexpr (decltype(with_copies)::value) {
        if (i == 0) copy_scales(s);
#pragma unroll
        for (int j = COPIES * i / MT; j < COPIES * (i + 1) / MT; j++) copy(s, j);
      }
      if (i < SLOTS) {
#pragma unroll
        for (int j = READS * i / SLOTS; j < READS * (i + 1) / SLOTS; j++) {
          if (j < NT) pn[j] = fp.get(at + TQ::BYTES, j, kk);
          else qn[j - NT] = fq.get(at, j - NT, kk);
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j++) acc[j][i] = mfma(p[j], q[i], acc[j][i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (steps) TWO && begin >= steps1 ? enter(1, begin - steps1) : enter(0, begin);
  // Where a compute unit has several workgroups they fill each other's waits, and one step ahead is enough; where it has one,
  // what a step reads comes from beyond the die's cache and takes longer than a step, so two steps are on their way. The number
  // of copies on their way is counted, so beyond the last step they go on, reading nothing.
  if constexpr (AHEAD) {
    // A step in two halves of k. While one half is multiplied the next is read into registers, across the steps too: the
    // barrier stands between the halves, where nothing of the current buffer is left to read, so the copies of the step
    // that will use it next can start there.
    if (steps) {
#pragma unroll
      for (int s = 0; s < STAGES; s++) start(s);
      landed(std::integral_constant<int, STAGES - 1>{});
      read(0, 0, q0, p0);
    }
    for (int s = 0; s < steps; s++) {
      half(q0, p0, q1, p1, lds + (uint32_t)s % STAGES * STEP, 1, std::false_type{}, 0);
      if constexpr (GROUPS == 2) add_group(s, 0);
      landed(std::integral_constant<int, STAGES - 2>{});
      // after the last step the reads get what is there, unused
      half(q1, p1, q0, p0, lds + (uint32_t)(s + 1) % STAGES * STEP, 0, std::true_type{}, s + STAGES);
      advance(s + STAGES);
      add_group(s, GROUPS - 1);
    }
  } else {
    // The copies of step s + STAGES - 1 go where step s - 1 was, which everybody has left at the barrier.
    if (steps)
#pragma unroll
      for (int s = 0; s < STAGES - 1; s++) start(s);
    for (int s = 0; s < steps; s++) {
      landed(std::integral_constant<int, STAGES - 2>{});
      start(s + STAGES - 1);
      read(s, 0, q0, p0);
      multiply(q0, p0);
      if constexpr (GROUPS == 2) add_group(s, 0);
      read(s, 1, q1, p1);
      multiply(q1, p1);
      add_group(s, GROUPS - 1);
    }
  }
  landed(All{});  // no copy may outlive the workgroup, and everybody's reads are done

  // The epilogue's values pass through LDS, 16 rows of a wave at a time, so that it gets eight neighbouring columns a lane and
  // eight lanes a row: whole lines where it reads and writes. A wave has its own piece of LDS and waits for nobody.
  using S = std::remove_reference_t<decltype(acc[0][0][0])>;
  constexpr int PITCH = WN + 4;  // values between rows: sixteen rows' pieces in different banks
  constexpr int LANES = (DUAL ? WN / 2 : WN) / 8, ROWS = 64 / LANES;
  static_assert(sizeof(S) * PITCH * 16 * WAVES_M * WAVES_N <= STAGES * STEP && ROWS * LANES == 64);
  S* turn = reinterpret_cast<S*>(lds) + wave * (16 * PITCH);
  const int lq = lane >> 4;
#pragma unroll
  for (int i = 0; i < MT; i++) {
#pragma unroll
    for (int t = 0; t < NT; t++) {
      Acc v = acc[t][i];
      if constexpr (GROUPS > 0) v = sum[t][i];
      *reinterpret_cast<Acc*>(turn + (lane & 15) * PITCH + t * 16 + lq * 4) = v;
    }
#pragma unroll 1
    for (int h = 0; h < 16; h += ROWS) {
      const int row = h + lane / LANES, col = lane % LANES * 8;
      const int64_t m = m0 + wm + i * 16 + row;
      if (row >= 16 || m >= a.M) continue;
      const S* v = turn + row * PITCH + col;
      S g[8], u[8];
#pragma unroll
      for (int j = 0; j < 8; j++) g[j] = v[j], u[j] = DUAL ? v[WN / 2 + j] : S(0);
      if constexpr (DUAL) {
        const int64_t n = n0 + wb * (WN / 2) + col;
        if (n < a.N) epi.template operator()<8>(blockIdx.x, m, (int)n, g, u);
      } else {
        const int64_t n = n0 + wn + col;
        if (n < a.N) epi.template operator()<8>(blockIdx.x, m, (int)n, g);
      }
    }
  }
}

}  // namespace dev
}  // namespace b2c
