// The gated feed-forward block and its gradients (b2c_hip_ffn_forward, b2c_hip_ffn_backward).
#include "dense.h"

namespace b2c {
namespace dev {
namespace {

int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }

bool sizes_ok(const b2c_ffn_args* a, Drop* d) {
  const int most = 1 << 24;
  return a && a->rows >= 0 && a->rows <= ((int64_t)1 << 31) && a->d_in >= 1 && a->d_in <= most && a->d_hidden >= 1 &&
         a->d_hidden <= most && a->d_out >= 1 && a->d_out <= most && (a->dtype == B2C_F16 || a->dtype == B2C_BF16) &&
         a->act >= B2C_ACT_SILU && a->act <= B2C_ACT_RELU && drop_of(a->p, a->seed, a->stream, d);
}
bool room_ok(const void* p, size_t have, size_t need) {
  return have >= need && (need == 0 || (p && reinterpret_cast<uintptr_t>(p) % 16 == 0));
}

template <typename T, int ACT>
int forward(const b2c_ffn_args* a, const Drop& d, hipStream_t stream) {
  const int64_t fp = up64(a->d_hidden);
  T* h = (T*)a->workspace;
  GateOut<T, ACT> gate{h, (T*)a->saved, fp, a->d_hidden};
  const Side<T> x{(const T*)a->x, a->ldx};
  int rc = product<T, false, false, true>(x, {(const T*)a->w_gate, a->ld_in}, x, {(const T*)a->w_up, a->ld_in}, a->rows,
                                          a->d_hidden, a->d_in, 0, gate, stream);
  if (rc) return rc;
  RowsOut<T> out{(T*)a->y, a->ldy, (const T*)a->residual, a->ldr, a->d_out, wide(a->y, a->ldy, 2),
                 wide(a->residual, a->ldr, 2), d};
  return product<T, false, false, false>(Side<T>{h, fp}, {(const T*)a->w_down, a->ld_out}, {}, {}, a->rows, a->d_out,
                                         a->d_hidden, 0, out, stream);
}

template <typename T, int ACT>
int backward(const b2c_ffn_grad_args* b, const Drop& d, hipStream_t stream) {
  const b2c_ffn_args* a = &b->fwd;
  const int64_t fp = up64(a->d_hidden), op = up64(a->d_out), M = a->rows;
  T* dgu = (T*)b->workspace;
  T* h = dgu + M * 2 * fp;
  T* dz = h + M * fp;
  Side<T> dy{(const T*)b->dy, b->lddy};
  int rc;
  if (d.threshold && M) {
    b2c_dropout_args da{M, a->d_out, a->dtype, a->p, a->seed, a->stream, b->dy, b->lddy, nullptr, 0, dz, op};
    if ((rc = b2c_hip_dropout(&da, stream))) return rc;
    dy = {dz, op};
  }
  const bool inner = b->dx || b->dw_gate || b->dw_up;
  const Side<T> wd{(const T*)a->w_down, a->ld_out};
  if (inner || b->dw_down) {
    GateBack<T, ACT> back{(const T*)a->saved, b->dw_down ? h : nullptr, dgu, fp, a->d_hidden};
    if ((rc = product<T, true, false, false>(dy, wd, {}, {}, M, a->d_hidden, a->d_out, 0, back, stream))) return rc;
  }
  const size_t gs = b->grad_dtype == B2C_F32 ? 4 : 2;
  const bool f32 = b->grad_dtype == B2C_F32, add = b->accumulate != 0;
  if (b->dw_down) {
    WeightOut<T> out{b->dw_down, nullptr, b->ld_dout, a->d_out, 0, a->d_hidden, f32, add, wide(b->dw_down, b->ld_dout, gs)};
    if ((rc = product<T, true, true, false>(dy, Side<T>{h, fp}, {}, {}, a->d_out, a->d_hidden, M, 0, out, stream))) return rc;
  }
  if (b->dw_gate || b->dw_up) {
    WeightOut<T> out{b->dw_gate, b->dw_up, b->ld_din, a->d_hidden, (int)fp, a->d_in, f32, add,
                     wide(b->dw_gate, b->ld_din, gs) && wide(b->dw_up, b->ld_din, gs)};
    if ((rc = product<T, true, true, false>(Side<T>{dgu, 2 * fp}, Side<T>{(const T*)a->x, a->ldx}, {}, {}, fp + a->d_hidden,
                                            a->d_in, M, 0, out, stream)))
      return rc;
  }
  if (b->dx) {
    RowsOut<T> out{(T*)b->dx, b->lddx, nullptr, 0, a->d_in, wide(b->dx, b->lddx, 2), false, {}};
    if ((rc = product<T, true, false, false>(Side<T>{dgu, 2 * fp}, Side<T>{(const T*)a->w_gate, a->ld_in},
                                             Side<T>{dgu + fp, 2 * fp}, Side<T>{(const T*)a->w_up, a->ld_in}, M, a->d_in,
                                             a->d_hidden, a->d_hidden, out, stream)))
      return rc;
  }
  return hipSuccess;
}

template <typename T>
int forward(const b2c_ffn_args* a, const Drop& d, hipStream_t s) {
  if (a->act == B2C_ACT_SILU) return forward<T, B2C_ACT_SILU>(a, d, s);
  if (a->act == B2C_ACT_GELU) return forward<T, B2C_ACT_GELU>(a, d, s);
  return forward<T, B2C_ACT_RELU>(a, d, s);
}
template <typename T>
int backward(const b2c_ffn_grad_args* a, const Drop& d, hipStream_t s) {
  if (a->fwd.act == B2C_ACT_SILU) return backward<T, B2C_ACT_SILU>(a, d, s);
  if (a->fwd.act == B2C_ACT_GELU) return backward<T, B2C_ACT_GELU>(a, d, s);
  return backward<T, B2C_ACT_RELU>(a, d, s);
}

}  // namespace
}  // namespace dev
}  // namespace b2c

using namespace b2c::dev;

extern "C" size_t b2c_ffn_saved_bytes(const b2c_ffn_args* a) {
  Drop d;
  return sizes_ok(a, &d) ? (size_t)a->rows * 2 * up64(a->d_hidden) * 2 : 0;
}
extern "C" size_t b2c_ffn_workspace_bytes(const b2c_ffn_args* a) {
  Drop d;
  return sizes_ok(a, &d) ? (size_t)a->rows * up64(a->d_hidden) * 2 : 0;
}
extern "C" int b2c_hip_ffn_forward(const b2c_ffn_args* a, hipStream_t stream) {
  Drop d;
  if (!sizes_ok(a, &d)) return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  if (!good(a->x, a->ldx, a->d_in, 2) || !good(a->w_gate, a->ld_in, a->d_in, 2) || !good(a->w_up, a->ld_in, a->d_in, 2) ||
      !good(a->w_down, a->ld_out, a->d_hidden, 2) || !good(a->y, a->ldy, a->d_out, 2) ||
      (a->residual && !good(a->residual, a->ldr, a->d_out, 2)) || reinterpret_cast<uintptr_t>(a->saved) % 16 ||
      !room_ok(a->workspace, a->workspace_bytes, b2c_ffn_workspace_bytes(a)))
    return hipErrorInvalidValue;
  return a->dtype == B2C_F16 ? forward<f16>(a, d, stream) : forward<bf16>(a, d, stream);
}

extern "C" size_t b2c_ffn_grad_workspace_bytes(const b2c_ffn_grad_args* b) {
  Drop d;
  if (!b || !sizes_ok(&b->fwd, &d)) return 0;
  return (size_t)b->fwd.rows * (3 * up64(b->fwd.d_hidden) + (d.threshold ? up64(b->fwd.d_out) : 0)) * 2;
}
extern "C" int b2c_hip_ffn_backward(const b2c_ffn_grad_args* b, hipStream_t stream) {
  Drop d;
  if (!b || !sizes_ok(&b->fwd, &d)) return hipErrorInvalidValue;
  const b2c_ffn_args* a = &b->fwd;
  if ((b->grad_dtype != a->dtype && b->grad_dtype != B2C_F32) || (b->accumulate && b->grad_dtype != B2C_F32))
    return hipErrorInvalidValue;
  const size_t gs = b->grad_dtype == B2C_F32 ? 4 : 2;
  if ((b->dw_gate && !good(b->dw_gate, b->ld_din, a->d_in, gs)) || (b->dw_up && !good(b->dw_up, b->ld_din, a->d_in, gs)) ||
      (b->dw_down && !good(b->dw_down, b->ld_dout, a->d_hidden, gs)))
    return hipErrorInvalidValue;
  if (a->rows) {
    if (!good(a->x, a->ldx, a->d_in, 2) || !good(a->w_gate, a->ld_in, a->d_in, 2) || !good(a->w_up, a->ld_in, a->d_in, 2) ||
        !good(a->w_down, a->ld_out, a->d_hidden, 2) || !good(b->dy, b->lddy, a->d_out, 2) ||
        (b->dx && !good(b->dx, b->lddx, a->d_in, 2)) || !a->saved || reinterpret_cast<uintptr_t>(a->saved) % 16 ||
        !room_ok(b->workspace, b->workspace_bytes, b2c_ffn_grad_workspace_bytes(b)))
      return hipErrorInvalidValue;
  }
  return a->dtype == B2C_F16 ? backward<f16>(b, d, stream) : backward<bf16>(b, d, stream);
}
