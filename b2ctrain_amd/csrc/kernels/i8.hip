// Products in 8-bit integers with a scale for each row and each channel (b2c_hip_quantize_rows, b2c_hip_i8_linear,
// b2c_hip_i8_ffn).
#include "dense_product.h"

namespace b2c {
namespace dev {
namespace {

// A row to a workgroup, in two passes over it: the largest magnitude, then the values. A row's columns from
// cols to `pad` become 0.
template <typename T>
__global__ __launch_bounds__(256) void quantize_kernel(const T* x, int64_t ldx, int64_t cols, int8_t* q, int64_t ldq,
                                                       int64_t pad, float* scale) {
  __shared__ float part[4];
  const int64_t m = blockIdx.x;
  const T* row = x + m * ldx;
  float top = 0.f;
  for (int64_t j = threadIdx.x; j < cols; j += 256) {
    const float v = fabsf((float)row[j]);
    top = v <= top ? top : v;  // a NaN stays in `top`: it is not <= anything
    if (v != v) top = INFINITY;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  const bool fine = top < INFINITY;
  const float s = fine ? top / 127.f : NAN;
  if (threadIdx.x == 0) scale[m] = s;
  for (int64_t j = threadIdx.x; j < pad; j += 256) {
    int v = 0;
    if (j < cols && fine && s > 0.f) v = (int)rintf((float)row[j] / s);
    q[m * ldq + j] = (int8_t)(v > 127 ? 127 : (v < -127 ? -127 : v));
  }
}

int quantize(const void* x, int64_t ldx, int dtype, int64_t rows, int64_t cols, int8_t* q, int64_t ldq, float* scale,
             hipStream_t stream) {
  const int64_t pad = ldq < (cols + 15) / 16 * 16 ? ldq : (cols + 15) / 16 * 16;
  const dim3 grid((unsigned)rows);
  if (dtype == B2C_F32) quantize_kernel<float><<<grid, 256, 0, stream>>>((const float*)x, ldx, cols, q, ldq, pad, scale);
  else if (dtype == B2C_F16) quantize_kernel<f16><<<grid, 256, 0, stream>>>((const f16*)x, ldx, cols, q, ldq, pad, scale);
  else quantize_kernel<bf16><<<grid, 256, 0, stream>>>((const bf16*)x, ldx, cols, q, ldq, pad, scale);
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

// Weights in 8 bits as the products read them: in place where rows start on 16 bytes (columns beyond the last meet zeros of
// the quantised rows), else copied to rows that do. A few rows read them anywhere.
__global__ __launch_bounds__(256) void pack_kernel(const int8_t* w, int64_t ldw, int64_t rows, int cols, int8_t* to,
                                                   int64_t pitch, uint32_t groups) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, m = t / groups;
  if (m >= rows) return;
  const int n = (int)(t - m * groups) * 16;
  const int8_t* p = w + m * ldw + n;
  vec<int8_t, 16> v{};
  if (n + 16 <= cols) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 16; j++)
      if (n + j < cols) v[j] = p[j];
  }
  *reinterpret_cast<vec<int8_t, 16>*>(to + m * pitch + n) = v;
}
struct Weights {
  Side<int8_t> from;
  int64_t rows;
  int cols;
  int8_t* copy = nullptr;
  int64_t pitch = 0;
  void place(Room& room, bool few) {
    if (few || (reinterpret_cast<uintptr_t>(from.p) % 16 == 0 && from.ld % 16 == 0 && cols % 16 == 0 && from.ld < (1 << 22))) return;
    pitch = up(cols, 128);
    copy = room.take<int8_t>(rows * pitch);
  }
  Side<int8_t> side() const { return pitch ? Side<int8_t>{copy, pitch} : from; }
  int make(hipStream_t stream) const {
    if (!pitch) return hipSuccess;
    const int64_t groups = up(cols, 16) / 16, blocks = up(rows * groups, 256) / 256;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    pack_kernel<<<dim3((unsigned)blocks), 256, 0, stream>>>(from.p, from.ld, rows, cols, copy, pitch, (uint32_t)groups);
    return hipGetLastError();
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
    way = choose(a->rows, a->d_out, steps_of(a->d_in), false, true);
    w = {{a->w, a->ldw}, a->d_out, a->d_in};
    w.place(room, way.tile == FEW_ROWS);
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
    gate = choose(a->rows, a->d_hidden, steps_of(a->d_in), true, true);
    down = choose(a->rows, a->d_out, steps_of(a->d_hidden), false, true);
    const bool few = gate.tile == FEW_ROWS;
    wg = {{a->w_gate, a->ld_in}, a->d_hidden, a->d_in};
    wu = {{a->w_up, a->ld_in}, a->d_hidden, a->d_in};
    wd = {{a->w_down, a->ld_out}, a->d_out, a->d_hidden};
    wg.place(room, few);
    wu.place(room, few);
    wd.place(room, few);
    sums = room.take<char>(std::max(gate.sums, down.sums));
  }
};

template <typename T>
int scaled(const Product<int8_t>& p, const Way& way, void* sums, const float* sx, const float* sw, void* y, int64_t ldy,
           hipStream_t stream) {
  const ScaledOut<T> out{(T*)y, ldy, sx, sw, (int)p.N};
  return product<int8_t, false, false, false, false>(p, way, sums, out, stream);
}
int scaled(const Product<int8_t>& p, const Way& way, void* sums, const float* sx, const float* sw, int dtype, void* y,
           int64_t ldy, hipStream_t stream) {
  if (dtype == B2C_F32) return scaled<float>(p, way, sums, sx, sw, y, ldy, stream);
  if (dtype == B2C_F16) return scaled<f16>(p, way, sums, sx, sw, y, ldy, stream);
  return scaled<bf16>(p, way, sums, sx, sw, y, ldy, stream);
}
template <int ACT>
int gated(const BlockPlan& p, const b2c_i8_ffn_args* a, hipStream_t stream) {
  const ScaledGate<ACT> out{p.h, p.s, a->s_gate, a->s_up, p.fp, a->d_hidden};
  const Product<int8_t> in{{p.qx, p.kp}, p.wg.side(), {}, p.wu.side(), a->rows, a->d_hidden, a->d_in, 0, a->rows, a->d_hidden};
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
  if (!sizes_ok(a) || a->rows == 0) return 0;
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
  Room room{(char*)a->workspace};
  const LinearPlan p(a, room);
  int rc = quantize(a->x, a->ldx, a->dtype, a->rows, a->d_in, p.q, p.kp, p.sx, stream);
  if (rc || (rc = p.w.make(stream))) return rc;
  const Product<int8_t> out{{p.q, p.kp}, p.w.side(), {}, {}, a->rows, a->d_out, a->d_in, 0, a->rows, a->d_out};
  return scaled(out, p.way, p.sums, p.sx, a->w_scale, a->dtype, a->y, a->ldy, stream);
}

extern "C" size_t b2c_i8_ffn_workspace_bytes(const b2c_i8_ffn_args* a) {
  if (!sizes_ok(a) || a->rows == 0) return 0;
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
  Room room{(char*)a->workspace};
  const BlockPlan p(a, room);
  int rc = quantize(a->x, a->ldx, a->dtype, a->rows, a->d_in, p.qx, p.kp, p.s, stream);
  if (rc || (rc = p.wg.make(stream)) || (rc = p.wu.make(stream)) || (rc = p.wd.make(stream))) return rc;
  if (a->act == B2C_ACT_SILU) rc = gated<B2C_ACT_SILU>(p, a, stream);
  else if (a->act == B2C_ACT_GELU) rc = gated<B2C_ACT_GELU>(p, a, stream);
  else rc = gated<B2C_ACT_RELU>(p, a, stream);
  if (rc) return rc;
  if ((rc = quantize(p.h, p.fp, B2C_F32, a->rows, a->d_hidden, p.qh, p.fp, p.s, stream))) return rc;
  const Product<int8_t> out{{p.qh, p.fp}, p.wd.side(), {}, {}, a->rows, a->d_out, a->d_hidden, 0, a->rows, a->d_out};
  return scaled(out, p.down, p.sums, p.s, a->s_down, a->dtype, a->y, a->ldy, stream);
}
