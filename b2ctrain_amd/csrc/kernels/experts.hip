// A mixture-of-experts layer for a few tokens (b2c_hip_experts): the router, the chosen experts' gate and up projections, their down
// projections with the weighted sum, a launch each.
#include "dense.h"

namespace b2c {
namespace dev {
namespace {

constexpr int kMostExperts = 1024, kMostChosen = 64;
constexpr int kLot = 1024;  // pairs of a token and an expert that one set of launches carries out

template <int N, typename T>
__device__ __forceinline__ vec<T, N> run_of(const T* row, int k, int K, bool there) {
  vec<T, N> v{};
  if (!there || k >= K) return v;
  if (k + N <= K) {
    __builtin_memcpy(&v, row + k, sizeof(v));
  } else {
#pragma unroll
    for (int j = 0; j < N; j++)
      if (k + j < K) v[j] = row[k + j];
  }
  return v;
}

// ---- the router --------------------------------------------------------------------------------------------

struct RouteArgs {
  int D, E, K;
  bool normalize;
  int32_t *to, *index;
  float *share, *weight;
  int64_t ldi, ldw;
};

// A workgroup a token. Products of 16-bit floats are exact in 64 bits and their sums nearly so: two experts are told apart where the numbers
// do it. An expert's place is how many are before it, so that the order takes no rounds of maxima.
template <typename T>
__global__ __launch_bounds__(1024) void route_kernel(Side<T> x, Side<T> w, RouteArgs a) {
  __shared__ double logits[kMostExperts];
  __shared__ uint64_t keys[kMostExperts];
  __shared__ int chosen[kMostChosen];
  __shared__ float parts[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m = blockIdx.x;
  const T* row = x.p + m * x.ld;
  constexpr int AT = 4;  // experts of a wave at a time
  for (int e0 = wave; e0 < a.E; e0 += 16 * AT) {
    double s[AT] = {};
    for (int k = lane * 8; k < a.D; k += 512) {
      const vec<T, 8> v = run_of<8>(row, k, a.D, true);
      vec<T, 8> u[AT];
#pragma unroll
      for (int i = 0; i < AT; i++) u[i] = run_of<8>(w.p + (int64_t)(e0 + 16 * i) * w.ld, k, a.D, e0 + 16 * i < a.E);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const double d = (double)(float)v[j];
#pragma unroll
        for (int i = 0; i < AT; i++) s[i] = fma(d, (double)(float)u[i][j], s[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < AT; i++) {
#pragma unroll
      for (int o = 32; o; o >>= 1) s[i] += __shfl_xor(s[i], o);
      const int e = e0 + 16 * i;
      if (lane == 0 && e < a.E) {
        const double l = s[i] + 0.0;  // no negative zero
        const uint64_t b = l != l ? 0x7fffffffffffffffull : __builtin_bit_cast(uint64_t, l);
        logits[e] = l;
        keys[e] = b >> 63 ? ~b : b | 1ull << 63;  // in the order of the numbers, a NaN above them
      }
    }
  }
  __syncthreads();
  const int e = threadIdx.x;
  if (e < a.E) {
    const uint64_t mine = keys[e];
    int before = 0;
    for (int i = 0; i < a.E; i++) before += keys[i] > mine || (keys[i] == mine && i < e);
    if (before < a.K) chosen[before] = e;
  }
  __syncthreads();
  const double top = logits[chosen[0]];
  float all = 0;
  if (a.normalize) {
    for (int j = 0; j < a.K; j++) all += expf((float)(logits[chosen[j]] - top));
  } else {
    float s = e < a.E ? expf((float)(logits[e] - top)) : 0.f;
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) parts[wave] = s;
    __syncthreads();
    for (int i = 0; i < 16; i++) all += parts[i];
  }
  if (e >= a.K) return;
  const float p = expf((float)(logits[chosen[e]] - top)) / all;
  a.to[m * a.K + e] = chosen[e];
  a.share[m * a.K + e] = p;
  if (a.index) a.index[m * a.ldi + e] = chosen[e];
  if (a.weight) a.weight[m * a.ldw + e] = p;
}

// ---- who goes where ----------------------------------------------------------------------------------------

// Which experts the pairs of a lot (token t's j-th choice is pair t K + j) name, as bits in LDS.
struct Taken {
  uint32_t bits[kMostExperts / 32];
  __device__ __forceinline__ void find(const int32_t* to, int pairs, int E) {
    for (int i = threadIdx.x; i < kMostExperts / 32; i += blockDim.x) bits[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) atomicOr(&bits[to[i] >> 5], 1u << (to[i] & 31));
    __syncthreads();
  }
  __device__ __forceinline__ int count(int E) const {
    int n = 0;
    for (int i = 0; i < (E + 31) / 32; i++) n += __builtin_popcount(bits[i]);
    return n;
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
  int64_t rows;
  int D, F, O, E, K;
  int64_t hp;  // between rows of h
  const int32_t* to;
  const float* share;
};

// h[pair] = act(w_gate x) (w_up x) for one expert's pairs: 16 hidden units a workgroup, its eight waves every eighth run of 128 values of
// k, 16 MT pairs at a time. The weights go from memory straight to the matrix instructions' registers.
template <typename T, int ACT, int MT>
__global__ __launch_bounds__(512) void gate_up_kernel(Side<T> x, Side<T> wg, Side<T> wu, T* h, ExpertArgs a) {
  __shared__ Taken taken;
  __shared__ uint16_t list[kLot];
  __shared__ int count;
  __shared__ f32x4 sums[8][2 * MT][64];
  const int pairs = (int)a.rows * a.K, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q4 = lane >> 4;
  taken.find(a.to, pairs, a.E);
  const int e = taken.at((int)blockIdx.y, a.E);
  if (e < 0) return;
  if (wave == 0) {
    const int n = pairs_of(a.to, pairs, e, list);
    if (lane == 0) count = n;
  }
  __syncthreads();
  const int n = (int)blockIdx.x * 16 + row, all = count;
  const bool there = n < a.F;
  const T* pg = wg.p + ((int64_t)e * a.F + (there ? n : 0)) * wg.ld;
  const T* pu = wu.p + ((int64_t)e * a.F + (there ? n : 0)) * wu.ld;
  for (int first = 0; first < all; first += 16 * MT) {
    const T* px[MT];
    bool has[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) {
      const int i = first + t * 16 + row;
      has[t] = i < all;
      px[t] = x.p + (int64_t)(has[t] ? list[i] / a.K : 0) * x.ld;
    }
    f32x4 acc[2][MT] = {};
    using A = vec<T, 8>;
    A g[2][4], u[2][4], v[2][MT][4];
    auto fetch = [&](int b, int k0) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int k = k0 + (c * 4 + q4) * 8;
        g[b][c] = run_of<8>(pg, k, a.D, there);
        u[b][c] = run_of<8>(pu, k, a.D, there);
#pragma unroll
        for (int t = 0; t < MT; t++) v[b][t][c] = run_of<8>(px[t], k, a.D, has[t]);
      }
    };
    auto multiply = [&](int b) {
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int t = 0; t < MT; t++) {
          acc[0][t] = mfma(g[b][c], v[b][t][c], acc[0][t]);
          acc[1][t] = mfma(u[b][c], v[b][t][c], acc[1][t]);
        }
    };
    fetch(0, wave * 128);
    for (int k0 = wave * 128; k0 < a.D; k0 += 2048) {
      fetch(1, k0 + 1024);
      multiply(0);
      fetch(0, k0 + 2048);
      multiply(1);
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < 2; d++)
#pragma unroll
      for (int t = 0; t < MT; t++) sums[wave][d * MT + t][lane] = acc[d][t];
    __syncthreads();
    if (wave < MT) {
      f32x4 s[2];
#pragma unroll
      for (int d = 0; d < 2; d++) {
        s[d] = sums[0][d * MT + wave][lane];
#pragma unroll
        for (int i = 1; i < 8; i++) s[d] += sums[i][d * MT + wave][lane];
      }
      const int i = first + wave * 16 + row, to = (int)blockIdx.x * 16 + q4 * 4;
      if (i < all && to < a.F) {
        float o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = act<ACT>(s[0][j]) * s[1][j];
        put<4>(h, a.hp, list[i], to, a.F, o);
      }
    }
  }
}

// y = residual + the weighted sum over a token's choices of w_down h: 16 outputs a workgroup, its sixteen waves an expert each, or a part of
// one's k where there are fewer. Every pair's sums stand in LDS before they are added, in the order of the choices.
template <typename T, int MT>
__global__ __launch_bounds__(1024) void down_kernel(const T* h, Side<T> w, const T* residual, int64_t ldr, T* y, int64_t ldy, ExpertArgs a) {
  __shared__ Taken taken;
  __shared__ uint16_t lists[16][kLot];
  __shared__ __attribute__((aligned(16))) float sums[kLot][16];
  const int pairs = (int)a.rows * a.K, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q4 = lane >> 4;
  taken.find(a.to, pairs, a.E);
  const int experts = taken.count(a.E), steps = (a.F + 127) / 128;
  int parts = 16 / experts;  // of an expert's k
  parts = parts < steps ? parts : steps;
  parts = parts < kLot / pairs ? parts : kLot / pairs;
  parts = parts < 1 ? 1 : parts;
  const int n = (int)blockIdx.x * 16 + row;
  const bool there = n < a.O;
  for (int unit = wave; unit < experts * parts; unit += 16) {
    const int i = unit / parts, part = unit - i * parts, e = taken.at(i, a.E);
    uint16_t* list = lists[wave];
    const int all = pairs_of(a.to, pairs, e, list);
    const int begin = steps * part / parts, end = steps * (part + 1) / parts;
    const T* p = w.p + ((int64_t)e * a.O + (there ? n : 0)) * w.ld;
    for (int first = 0; first < all; first += 16 * MT) {
      const T* ph[MT];
      bool has[MT];
#pragma unroll
      for (int t = 0; t < MT; t++) {
        const int j = first + t * 16 + row;
        has[t] = j < all;
        ph[t] = h + (int64_t)(has[t] ? list[j] : 0) * a.hp;
      }
      f32x4 acc[MT] = {};
      vec<T, 8> g[2][4], v[2][MT][4];
      auto fetch = [&](int b, int step) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const int k = step * 128 + (c * 4 + q4) * 8;
          g[b][c] = run_of<8>(p, k, a.F, there && step < end);
#pragma unroll
          for (int t = 0; t < MT; t++) v[b][t][c] = run_of<8>(ph[t], k, a.F, has[t] && step < end);
        }
      };
      auto multiply = [&](int b) {
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
          for (int t = 0; t < MT; t++) acc[t] = mfma(g[b][c], v[b][t][c], acc[t]);
      };
      fetch(0, begin);
      for (int s = begin; s < end; s += 2) {
        fetch(1, s + 1);
        multiply(0);
        fetch(0, s + 2);
        multiply(1);
      }
#pragma unroll
      for (int t = 0; t < MT; t++) {
        const int j = first + t * 16 + row;
        if (j < all) *reinterpret_cast<f32x4*>(&sums[part * pairs + list[j]][q4 * 4]) = acc[t];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < (int)a.rows * 16; i += 1024) {
    const int64_t m = i >> 4;
    const int c = i & 15, to = (int)blockIdx.x * 16 + c;
    if (to >= a.O) continue;
    float v = residual ? (float)residual[m * ldr + to] : 0.f;
    for (int j = 0; j < a.K; j++) {
      const int p = (int)m * a.K + j;
      float s = 0;
      for (int q = 0; q < parts; q++) s += sums[q * pairs + p][c];
      v = fmaf(a.share[p], s, v);
    }
    y[m * ldy + to] = (T)v;
  }
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
  int64_t lot, hp;
  int32_t* to;
  float* share;
  T* h;
  ExpertsPlan(const b2c_experts_args* a, Room& room) {
    lot = std::min<int64_t>(a->rows, kLot / a->top_k);
    hp = up(a->d_hidden, 8);
    to = room.take<int32_t>(lot * a->top_k);
    share = room.take<float>(lot * a->top_k);
    h = room.take<T>(lot * a->top_k * hp);
  }
};

template <typename T, int ACT>
int run(const b2c_experts_args* a, hipStream_t stream) {
  Room room{(char*)a->workspace};
  const ExpertsPlan<T> p(a, room);
  const Side<T> wr{(const T*)a->w_router, a->ld_router}, wg{(const T*)a->w_gate, a->ld_in}, wu{(const T*)a->w_up, a->ld_in},
      wd{(const T*)a->w_down, a->ld_out};
  for (int64_t m = 0; m < a->rows; m += p.lot) {
    const int64_t rows = std::min(p.lot, a->rows - m);
    const Side<T> x{(const T*)a->x + m * a->ldx, a->ldx};
    const RouteArgs r{a->d_in, a->experts, a->top_k, a->normalize != 0, p.to, a->index ? a->index + m * a->ldi : nullptr, p.share,
                      a->weight ? a->weight + m * a->ldw : nullptr, a->ldi, a->ldw};
    route_kernel<T><<<dim3((unsigned)rows), 1024, 0, stream>>>(x, wr, r);
    int rc = hipGetLastError();
    if (rc) return rc;
    const ExpertArgs e{rows, a->d_in, a->d_hidden, a->d_out, a->experts, a->top_k, p.hp, p.to, p.share};
    const dim3 grid((unsigned)(up(a->d_hidden, 16) / 16), (unsigned)std::min<int64_t>(rows * a->top_k, a->experts));
    if (rows <= 16) gate_up_kernel<T, ACT, 1><<<grid, 512, 0, stream>>>(x, wg, wu, p.h, e);
    else gate_up_kernel<T, ACT, 2><<<grid, 512, 0, stream>>>(x, wg, wu, p.h, e);
    if ((rc = hipGetLastError())) return rc;
    const T* residual = a->residual ? (const T*)a->residual + m * a->ldr : nullptr;
    T* y = (T*)a->y + m * a->ldy;
    const dim3 tiles((unsigned)(up(a->d_out, 16) / 16));
    if (rows <= 16) down_kernel<T, 1><<<tiles, 1024, 0, stream>>>(p.h, wd, residual, a->ldr, y, a->ldy, e);
    else down_kernel<T, 2><<<tiles, 1024, 0, stream>>>(p.h, wd, residual, a->ldr, y, a->ldy, e);
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
      a->workspace_bytes < b2c_experts_workspace_bytes(a))
    return hipErrorInvalidValue;
  return a->dtype == B2C_F16 ? run<f16>(a, stream) : run<bf16>(a, stream);
}
