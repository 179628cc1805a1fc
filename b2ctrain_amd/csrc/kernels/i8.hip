// Products in 8-bit integers with a scale for each row and each channel (b2c_hip_quantize_rows, b2c_hip_i8_linear,
// b2c_hip_i8_ffn).
#include "dense.h"

namespace b2c {
namespace dev {
namespace {

int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }

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
size_t up16(size_t v) { return (v + 15) / 16 * 16; }

template <typename T>
int linear_out(const int8_t* q, int64_t ldq, const float* sx, const int8_t* w, int64_t ldw, const float* sw, int64_t rows,
               int d_out, int d_in, void* y, int64_t ldy, hipStream_t stream) {
  ScaledOut<T> out{(T*)y, ldy, sx, sw, d_out, wide(y, ldy, sizeof(T))};
  return product<int8_t, false, false, false>(Side<int8_t>{q, ldq}, Side<int8_t>{w, ldw}, {}, {}, rows, d_out, d_in, 0, out,
                                              stream);
}
int linear(const int8_t* q, int64_t ldq, const float* sx, const int8_t* w, int64_t ldw, const float* sw, int64_t rows,
           int d_out, int d_in, int dtype, void* y, int64_t ldy, hipStream_t stream) {
  if (dtype == B2C_F32) return linear_out<float>(q, ldq, sx, w, ldw, sw, rows, d_out, d_in, y, ldy, stream);
  if (dtype == B2C_F16) return linear_out<f16>(q, ldq, sx, w, ldw, sw, rows, d_out, d_in, y, ldy, stream);
  return linear_out<bf16>(q, ldq, sx, w, ldw, sw, rows, d_out, d_in, y, ldy, stream);
}
template <int ACT>
int gated(const int8_t* q, int64_t ldq, const float* sx, const b2c_i8_ffn_args* a, float* h, int64_t fp, hipStream_t stream) {
  ScaledGate<ACT> out{h, sx, a->s_gate, a->s_up, fp, a->d_hidden};
  const Side<int8_t> x{q, ldq};
  return product<int8_t, false, false, true>(x, {a->w_gate, a->ld_in}, x, {a->w_up, a->ld_in}, a->rows, a->d_hidden, a->d_in,
                                             0, out, stream);
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
  return sizes_ok(a) ? (size_t)a->rows * up64(a->d_in) + up16((size_t)a->rows * 4) : 0;
}
extern "C" int b2c_hip_i8_linear(const b2c_i8_linear_args* a, hipStream_t stream) {
  if (!sizes_ok(a)) return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  if (!good(a->x, a->ldx, a->d_in, size_of(a->dtype)) || !good(a->w, a->ldw, a->d_in, 1) || !good(a->w_scale, 1, 1, 4) ||
      !good(a->y, a->ldy, a->d_out, size_of(a->dtype)) ||
      !room_ok(a->workspace, a->workspace_bytes, b2c_i8_linear_workspace_bytes(a)))
    return hipErrorInvalidValue;
  const int64_t kp = up64(a->d_in);
  int8_t* q = (int8_t*)a->workspace;
  float* sx = (float*)(q + a->rows * kp);
  const int rc = quantize(a->x, a->ldx, a->dtype, a->rows, a->d_in, q, kp, sx, stream);
  if (rc) return rc;
  return linear(q, kp, sx, a->w, a->ldw, a->w_scale, a->rows, a->d_out, a->d_in, a->dtype, a->y, a->ldy, stream);
}

extern "C" size_t b2c_i8_ffn_workspace_bytes(const b2c_i8_ffn_args* a) {
  if (!sizes_ok(a)) return 0;
  return (size_t)a->rows * (up64(a->d_in) + up64(a->d_hidden) * 5) + up16((size_t)a->rows * 4);
}
extern "C" int b2c_hip_i8_ffn(const b2c_i8_ffn_args* a, hipStream_t stream) {
  if (!sizes_ok(a)) return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  if (!good(a->x, a->ldx, a->d_in, size_of(a->dtype)) || !good(a->w_gate, a->ld_in, a->d_in, 1) ||
      !good(a->w_up, a->ld_in, a->d_in, 1) || !good(a->w_down, a->ld_out, a->d_hidden, 1) || !good(a->s_gate, 1, 1, 4) ||
      !good(a->s_up, 1, 1, 4) || !good(a->s_down, 1, 1, 4) || !good(a->y, a->ldy, a->d_out, size_of(a->dtype)) ||
      !room_ok(a->workspace, a->workspace_bytes, b2c_i8_ffn_workspace_bytes(a)))
    return hipErrorInvalidValue;
  const int64_t kp = up64(a->d_in), fp = up64(a->d_hidden);
  float* h = (float*)a->workspace;
  int8_t* qh = (int8_t*)(h + a->rows * fp);
  int8_t* qx = qh + a->rows * fp;
  float* s = (float*)(qx + a->rows * kp);  // of x's rows, then of h's
  int rc = quantize(a->x, a->ldx, a->dtype, a->rows, a->d_in, qx, kp, s, stream);
  if (rc) return rc;
  if (a->act == B2C_ACT_SILU) rc = gated<B2C_ACT_SILU>(qx, kp, s, a, h, fp, stream);
  else if (a->act == B2C_ACT_GELU) rc = gated<B2C_ACT_GELU>(qx, kp, s, a, h, fp, stream);
  else rc = gated<B2C_ACT_RELU>(qx, kp, s, a, h, fp, stream);
  if (rc) return rc;
  rc = quantize(h, fp, B2C_F32, a->rows, a->d_hidden, qh, fp, s, stream);
  if (rc) return rc;
  return linear(qh, fp, s, a->w_down, a->ld_out, a->s_down, a->rows, a->d_out, a->d_hidden, a->dtype, a->y, a->ldy, stream);
}
