// The 8-bit block where it is narrow (at most 128 wide, all weights in LDS) and its rows many: a trained head over the
// splats of a scene, in one pass over x. A wave takes 16 rows from x to y: it quantises them, multiplies them by the
// gate's and the up projection's weights from LDS, keeps the whole row of h in registers (its largest value is needed
// before the first of them can be rounded), rounds it and multiplies it by the down weights. As in the 16-bit head, the rows
// of the weights are dealt out so that a lane's accumulators are the next instruction's operand: hidden unit
// 16 (l / 16) + 4 t + r of each 64 for accumulator r of tile t. Bound by the arithmetic on h, about 20 instructions a value: 1M
// rows of 64-256-64 take 156 us.
#include "i8_head.h"
#include "i8_quant.h"

namespace b2c {
namespace dev {
namespace {

constexpr int head_fragments(int ki) { return 12 * ki; }  // of 64 hidden units: g (t, k), u (t, k), down (o tile)

template <int KI>
__global__ __launch_bounds__(256) void fragments_kernel(b2c_i8_ffn_args a, int chunks, int8_t* out) {
  const int t = blockIdx.x * 256 + threadIdx.x, lane = t & 63, i = lane & 15, q = lane >> 4, all = t >> 6;
  const int c = all / head_fragments(KI), f = all % head_fragments(KI);
  if (c >= chunks) return;
  vec<int8_t, 16> v{};
  if (f < 8 * KI) {
    const int8_t* w = f < 4 * KI ? a.w_gate : a.w_up;
    const int tile = f % (4 * KI) / KI, h = c * 64 + (i >> 2) * 16 + tile * 4 + (i & 3), k = f % KI * 64 + q * 16;
    if (h < a.d_hidden)
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (k + j < a.d_in) v[j] = w[h * a.ld_in + k + j];
  } else {
    const int o = (i >> 2) * (16 * KI) + (f - 8 * KI) * 4 + (i & 3), k = c * 64 + q * 16;
    if (o < a.d_out)
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (k + j < a.d_hidden) v[j] = a.w_down[o * a.ld_out + k + j];
  }
  *reinterpret_cast<vec<int8_t, 16>*>(out + (int64_t)t * 16) = v;
}

// Sixteen values of row m from column k on, as floats; zeros beyond the ends.
template <typename T>
__device__ __forceinline__ void sixteen(const void* x, int64_t ld, int64_t m, int64_t M, int k, int K, float (&v)[16]) {
  const T* p = (const T*)x + m * ld + k;
  if (m < M && k + 16 <= K) {
    vec<T, 16> t;
    __builtin_memcpy(&t, p, sizeof(t));
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = (float)t[j];
  } else {
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = m < M && k + j < K ? (float)p[j] : 0.f;
  }
}

__device__ __forceinline__ uint32_t over_row(uint32_t top) {  // of the four lanes that share a row
  const uint32_t a = __shfl_xor(top, 16), b = top > a ? top : a, c = __shfl_xor(b, 32);
  return b > c ? b : c;
}

// Row m of x in 8 bits, as the matrix instruction's operand (lane group q4 holds values 16 q4 .. of each 64), and its scale.
template <int KI>
__device__ __forceinline__ RowScale row_in_bytes(const void* x, int64_t ldx, int dtype, int64_t m, int64_t M, int K, int q4,
                                                 i32x4 (&q)[KI]) {
  float v[KI][16];
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < KI; k++) {
    if (dtype == B2C_BF16) sixteen<bf16>(x, ldx, m, M, k * 64 + q4 * 16, K, v[k]);
    else if (dtype == B2C_F16) sixteen<f16>(x, ldx, m, M, k * 64 + q4 * 16, K, v[k]);
    else sixteen<float>(x, ldx, m, M, k * 64 + q4 * 16, K, v[k]);
#pragma unroll
    for (int j = 0; j < 16; j++) top = magnitude(v[k][j]) > top ? magnitude(v[k][j]) : top;
  }
  const RowScale s(over_row(top));
#pragma unroll
  for (int k = 0; k < KI; k++)
#pragma unroll
    for (int j = 0; j < 4; j++) q[k][j] = (int)bytes4(s(v[k][4 * j]), s(v[k][4 * j + 1]), s(v[k][4 * j + 2]), s(v[k][4 * j + 3]));
  return s;
}
__device__ __forceinline__ void put_as(int dtype, void* y, int64_t ldy, int64_t m, int n, int cols, const float (&v)[8]) {
  if (dtype == B2C_BF16) put<8>((bf16*)y, ldy, m, n, cols, v);
  else if (dtype == B2C_F16) put<8>((f16*)y, ldy, m, n, cols, v);
  else put<8>((float*)y, ldy, m, n, cols, v);
}

template <int ACT, int KI, int NC>
__global__ __launch_bounds__(512) void head_kernel(b2c_i8_ffn_args a, const int8_t* frags, int chunks) {
  constexpr int N = head_fragments(KI), OT = 4 * KI;
  static_assert(NC >= KI);  // the loop over hidden units' scales covers the outputs'
  using A = vec<int8_t, 16>;
  __shared__ A w[NC * N][64];
  __shared__ f32x4 sg[NC * 16], su[NC * 16], sd[KI * 16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q4 = lane >> 4;
  for (int f = wave; f < NC * N; f += 8) w[f][lane] = f < chunks * N ? *reinterpret_cast<const A*>(frags + ((int64_t)f * 64 + lane) * 16) : A{};
  for (int j = threadIdx.x; j < NC * 64; j += 512) {
    ((float*)sg)[j] = j < a.d_hidden ? a.s_gate[j] : 0.f;
    ((float*)su)[j] = j < a.d_hidden ? a.s_up[j] : 0.f;
    if (j < KI * 64) ((float*)sd)[j] = j < a.d_out ? a.s_down[j] : 0.f;
  }
  __syncthreads();
  const int64_t M = a.rows, tiles = (M + 15) / 16;
  for (int64_t tile = (int64_t)blockIdx.x * 8 + wave; tile < tiles; tile += (int64_t)gridDim.x * 8) {
    const int64_t m = tile * 16 + (lane & 15);
    i32x4 qx[KI];
    const RowScale rx = row_in_bytes<KI>(a.x, a.ldx, a.dtype, m, M, a.d_in, q4, qx);

    float h[NC][16];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < NC; c++) {
      asm volatile("" ::: "memory");  // the weights stay in LDS: held over the loop, they would fill the registers
#pragma unroll
      for (int t = 0; t < 4; t++) {
        i32x4 g = {}, u = {};
#pragma unroll
        for (int k = 0; k < KI; k++) {
          g = mfma(w[c * N + t * KI + k][lane], __builtin_bit_cast(A, qx[k]), g);
          u = mfma(w[c * N + (4 + t) * KI + k][lane], __builtin_bit_cast(A, qx[k]), u);
        }
        const f32x4 a4 = sg[c * 16 + q4 * 4 + t], b4 = su[c * 16 + q4 * 4 + t];
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float v = act<ACT>((float)g[r] * (rx.scale * a4[r])) * ((float)u[r] * b4[r]);  // x's scale of u follows below
          h[c][t * 4 + r] = v;
          top = magnitude(v) > top ? magnitude(v) : top;
        }
      }
    }
    top = over_row(top);
    RowScale rh(top);
    float sh = rh.scale * rx.scale;
    if (!rh.plain && rh.scale > 0.f) {  // a row whose scale is too small for an inverse: the same 8 bits from 2^100 h
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 16; j++) h[c][j] *= 0x1p100f;
      rh = RowScale(__builtin_bit_cast(uint32_t, __builtin_bit_cast(float, top) * 0x1p100f));
      sh = rh.scale * rx.scale * 0x1p-100f;
    }
    i32x4 y[OT] = {};
#pragma unroll
    for (int c = 0; c < NC; c++) {
      asm volatile("" ::: "memory");
      i32x4 qh;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t b[4];
#pragma unroll
        for (int r = 0; r < 4; r++) b[r] = rh.near(h[c][4 * j + r]);
        qh[j] = (int)bytes4(b[0], b[1], b[2], b[3]);
      }
#pragma unroll
      for (int t = 0; t < OT; t++) y[t] = mfma(w[c * N + 8 * KI + t][lane], __builtin_bit_cast(A, qh), y[t]);
    }
    if (m >= M) continue;
#pragma unroll
    for (int t = 0; t < OT; t += 2) {
      const int n = q4 * (16 * KI) + t * 4;
      if (n >= a.d_out) continue;
      const f32x4 a4 = sd[n / 4], b4 = sd[n / 4 + 1];
      float v[8];
#pragma unroll
      for (int r = 0; r < 4; r++) v[r] = (float)y[t][r] * sh * a4[r], v[4 + r] = (float)y[t + 1][r] * sh * b4[r];
      put_as(a.dtype, a.y, a.ldy, m, n, a.d_out, v);
    }
  }
}

// The same for one layer: 16 rows of x to a wave, quantised in registers, times weights that all lie in LDS. Bound by memory: what
// a tile of 128 outputs would do in one step of k is over before its copies could be hidden. 500k rows of 64 -> 256: 86 us, 163
// by quantising first and 128-wide tiles.
template <int KI>
__global__ __launch_bounds__(512) void linear_kernel(b2c_i8_linear_args a, int chunks) {
  using A = vec<int8_t, 16>;
  extern __shared__ __attribute__((aligned(1024))) char room[];
  A(*w)[64] = reinterpret_cast<A(*)[64]>(room);  // fragment 4 KI c + KI t + k: outputs 64 c + 16 (i / 4) + 4 t + i % 4
  float* sw = reinterpret_cast<float*>(room + (size_t)chunks * 4 * KI * 1024);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q4 = lane >> 4, i = lane & 15;
  for (int f = wave; f < chunks * 4 * KI; f += 8) {
    const int o = f / (4 * KI) * 64 + (i >> 2) * 16 + f % (4 * KI) / KI * 4 + (i & 3), k = f % KI * 64 + q4 * 16;
    A v{};
    if (o < a.d_out) {
      const int8_t* p = a.w + o * a.ldw + k;
      if (k + 16 <= a.d_in) {
        __builtin_memcpy(&v, p, 16);
      } else {
#pragma unroll
        for (int j = 0; j < 16; j++)
          if (k + j < a.d_in) v[j] = p[j];
      }
    }
    w[f][lane] = v;
  }
  for (int j = threadIdx.x; j < chunks * 64; j += 512) sw[j] = j < a.d_out ? a.w_scale[j] : 0.f;
  __syncthreads();
  const int64_t M = a.rows, tiles = (M + 15) / 16;
  for (int64_t tile = (int64_t)blockIdx.x * 8 + wave; tile < tiles; tile += (int64_t)gridDim.x * 8) {
    const int64_t m = tile * 16 + i;
    i32x4 qx[KI];
    const RowScale rx = row_in_bytes<KI>(a.x, a.ldx, a.dtype, m, M, a.d_in, q4, qx);
    for (int c = 0; c < chunks; c++) {
      i32x4 y[4] = {};
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int k = 0; k < KI; k++) y[t] = mfma(w[c * 4 * KI + t * KI + k][lane], __builtin_bit_cast(A, qx[k]), y[t]);
      const int n = c * 64 + q4 * 16;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (m >= M || n + h * 8 >= a.d_out) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (float)y[h * 2 + j / 4][j % 4] * (rx.scale * sw[n + h * 8 + j]);
        put_as(a.dtype, a.y, a.ldy, m, n + h * 8, a.d_out, v);
      }
    }
  }
}

int chunks_of(const b2c_i8_ffn_args* a) { return (int)up(a->d_hidden, 64) / 64; }
int width_of(const b2c_i8_ffn_args* a) { return std::max(a->d_in, a->d_out) <= 64 ? 1 : 2; }

template <int ACT, int KI, int NC>
int launch(const b2c_i8_ffn_args* a, const int8_t* frags, hipStream_t stream) {
  const int64_t groups = up(a->rows, 128) / 128;
  const int held = NC * KI <= 4 ? 2 : 1;  // workgroups that a compute unit holds, by LDS and registers
  head_kernel<ACT, KI, NC><<<dim3((unsigned)std::min<int64_t>(groups, 256 * held)), 512, 0, stream>>>(*a, frags, chunks_of(a));
  return hipGetLastError();
}
template <int ACT, int KI>
int launch(const b2c_i8_ffn_args* a, const int8_t* frags, hipStream_t stream) {
  const int c = chunks_of(a);
  if (c <= 2) return launch<ACT, KI, 2>(a, frags, stream);
  if (c <= 4) return launch<ACT, KI, 4>(a, frags, stream);
  if (KI == 2 || c <= 6) return launch<ACT, KI, 6>(a, frags, stream);
  if constexpr (KI == 1) return launch<ACT, 1, 8>(a, frags, stream);
  return hipErrorInvalidValue;
}
template <int KI>
int run(const b2c_i8_ffn_args* a, int8_t* frags, hipStream_t stream) {
  const int n = chunks_of(a) * head_fragments(KI);
  fragments_kernel<KI><<<dim3((unsigned)up(n, 4) / 4), 256, 0, stream>>>(*a, chunks_of(a), frags);
  const int rc = hipGetLastError();
  if (rc) return rc;
  if (a->act == B2C_ACT_SILU) return launch<B2C_ACT_SILU, KI>(a, frags, stream);
  if (a->act == B2C_ACT_GELU) return launch<B2C_ACT_GELU, KI>(a, frags, stream);
  return launch<B2C_ACT_RELU, KI>(a, frags, stream);
}

constexpr int64_t kRoom = 64 << 10;  // of LDS for a layer's weights, so that a compute unit holds two workgroups
int64_t linear_room(const b2c_i8_linear_args* a) {
  return up(a->d_out, 64) / 64 * (4 * (a->d_in <= 64 ? 1 : 2) * 1024 + 256);
}

}  // namespace

bool is_i8_head(const b2c_i8_ffn_args* a) {
  return a->rows > kI8HeadRows && a->d_in <= 128 && a->d_out <= 128 && chunks_of(a) <= (width_of(a) == 1 ? 8 : 6);
}
size_t i8_head_bytes(const b2c_i8_ffn_args* a) { return (size_t)chunks_of(a) * head_fragments(width_of(a)) * 1024; }
int i8_head(const b2c_i8_ffn_args* a, hipStream_t stream) {
  return width_of(a) == 1 ? run<1>(a, (int8_t*)a->workspace, stream) : run<2>(a, (int8_t*)a->workspace, stream);
}


bool is_i8_narrow(const b2c_i8_linear_args* a) { return a->rows > kI8HeadRows && a->d_in <= 128 && linear_room(a) <= kRoom; }
int i8_narrow(const b2c_i8_linear_args* a, hipStream_t stream) {
  const int chunks = (int)(up(a->d_out, 64) / 64);
  const dim3 grid((unsigned)std::min<int64_t>(up(a->rows, 128) / 128, 512));
  if (a->d_in <= 64) linear_kernel<1><<<grid, 512, (size_t)linear_room(a), stream>>>(*a, chunks);
  else linear_kernel<2><<<grid, 512, (size_t)linear_room(a), stream>>>(*a, chunks);
  return hipGetLastError();
}

}  // namespace dev
}  // namespace b2c
