// The gated feed-forward block and its gradients (b2c_hip_ffn_forward, b2c_hip_ffn_backward).
#include "ffn_head.h"

namespace b2c {
namespace dev {

template <>
int head_forward<f16>(const b2c_ffn_args*, const Drop&, hipStream_t);
template <>
int head_forward<bf16>(const b2c_ffn_args*, const Drop&, hipStream_t);
template <>
int head_backward<f16>(const b2c_ffn_grad_args*, const Drop&, hipStream_t);
template <>
int head_backward<bf16>(const b2c_ffn_grad_args*, const Drop&, hipStream_t);

namespace {

bool sizes_ok(const b2c_ffn_args* a, Drop* d) {
  const int most = 1 << 20;  // 256 rows of two such widths span 1 GiB: the copies to LDS have offsets of 31 bits
  return a && a->rows >= 0 && a->rows <= (1 << 30) && a->d_in >= 1 && a->d_in <= most && a->d_hidden >= 1 &&
         a->d_hidden <= most && a->d_out >= 1 && a->d_out <= most && (a->dtype == B2C_F16 || a->dtype == B2C_BF16) &&
         a->act >= B2C_ACT_SILU && a->act <= B2C_ACT_RELU && drop_of(a->p, a->seed, a->stream, d);
}
bool room_ok(const void* p, size_t have, size_t need) {
  return have >= need && (need == 0 || (p && reinterpret_cast<uintptr_t>(p) % 16 == 0));
}

// Matrices copied to rows that start on 16 bytes, `pitch` values apart, zeros in the columns from `cols` up to the next
// multiple of 8; where dropout is given, zeros in the place of what it drops too. Eight values a thread; all of a call's
// copies in one launch.
template <typename T>
struct Pack {
  Side<T> from;
  T* to;
  int64_t rows, pitch;
  int cols;
  uint32_t groups, blocks;
  Drop drop;
};
template <typename T>
struct Packs {
  Pack<T> of[5];
  int n = 0;
  uint32_t blocks = 0;
  void add(const Side<T>& from, int64_t rows, int cols, T* to, int64_t pitch, const Drop& d) {
    const int64_t groups = up(cols, 8) / 8;
    of[n++] = {from, to, rows, pitch, cols, (uint32_t)groups, (uint32_t)(up(rows * groups, 256) / 256), d};
  }
};
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(Packs<T> all) {
  uint32_t block = block_index();
  int i = 0;
  if (block >= all.blocks) return;
  while (block >= all.of[i].blocks) block -= all.of[i++].blocks;
  const Pack<T>& p = all.of[i];
  const int64_t t = (int64_t)block * 256 + threadIdx.x, m = t / p.groups;
  if (m >= p.rows) return;
  const int n = (int)(t - m * p.groups) * 8;
  const T* from = p.from.p + m * p.from.ld + n;
  vec<T, 8> v{};
  if (n + 8 <= p.cols) {
    __builtin_memcpy(&v, from, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (n + j < p.cols) v[j] = from[j];
  }
  if (p.drop.threshold) {
    const uint32_t keep = kept_bits<8>(p.drop, (uint64_t)m * p.cols + n);
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (!(keep >> j & 1)) v[j] = (T)0.f;
  }
  *reinterpret_cast<vec<T, 8>*>(p.to + m * p.pitch + n) = v;
}
template <typename T>
int make(Packs<T>& all, hipStream_t stream) {
  int64_t blocks = 0;
  for (int i = 0; i < all.n; i++) {
    blocks += all.of[i].blocks;
    if (up(all.of[i].rows * all.of[i].groups, 256) / 256 > 0x7fffffff) return hipErrorInvalidValue;
  }
  if (blocks == 0) return hipSuccess;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  all.blocks = (uint32_t)blocks;
  pack_kernel<T><<<grid_of(blocks), 256, 0, stream>>>(all);
  return hipGetLastError();
}

// Whether the tiles' copies can read a matrix where it is: rows on 16 bytes, whole pieces of 8 columns, and 256 rows
// within the 2 GiB that a copy's offset spans.
bool direct(const void* p, int64_t ld, int64_t cols) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && cols % 8 == 0 && ld < ((int64_t)1 << 21);
}

// An operand: where it is, or its packed copy.
template <typename T>
struct Operand {
  Side<T> from;
  int64_t rows;
  int cols;
  T* copy = nullptr;
  int64_t pitch = 0;
  Drop drop{};
  void place(Room& room, bool straight) {
    if (straight) return;
    pitch = up(cols, 64);
    copy = room.take<T>(rows * pitch);
  }
  Side<T> side() const { return pitch ? Side<T>{copy, pitch} : from; }
  void add_to(Packs<T>& all) const {
    if (pitch) all.add(from, rows, cols, copy, pitch, drop);
  }
};

// The steps of 64 values that a sum over k takes.
int64_t steps_of(int64_t k) { return up(k, 64) / 64; }

// The inner activations that a forward pass keeps for the down weights' gradient: behind its factors.
template <typename T>
T* kept_h(const b2c_ffn_args* a) {
  return (T*)((float*)a->saved + a->rows * 2 * up(a->d_hidden, 64));
}

// What a forward pass needs beside its matrices.
template <typename T>
struct ForwardPlan {
  int64_t fp;
  T* h;
  Operand<T> x, wg, wu, wd;
  Way gate, down;
  void* sums;
  ForwardPlan(const b2c_ffn_args* a, Room& room) {
    const int64_t M = a->rows;
    fp = up(a->d_hidden, 64);
    h = room.take<T>(M * fp);  // with `saved` too, where it stays unused: a call without it may follow in the same workspace
    if (a->saved) h = kept_h<T>(a);
    const bool in = direct(a->w_gate, a->ld_in, a->d_in) && direct(a->w_up, a->ld_in, a->d_in);
    const bool out = direct(a->w_down, a->ld_out, a->d_hidden), few = few_rows(M, in && out);
    const Way plain = choose({{M, fp}}, steps_of(a->d_in), true, few, 2), keeping = choose({{M, fp}}, steps_of(a->d_in), true, few, 10);
    gate = a->saved ? keeping : plain;
    down = choose({{M, a->d_out}}, steps_of(a->d_hidden), false, few);
    x = {{(const T*)a->x, a->ldx}, M, a->d_in};
    wg = {{(const T*)a->w_gate, a->ld_in}, a->d_hidden, a->d_in};
    wu = {{(const T*)a->w_up, a->ld_in}, a->d_hidden, a->d_in};
    wd = {{(const T*)a->w_down, a->ld_out}, a->d_out, a->d_hidden};
    if (!few) {  // all or none along d_in: a copy's zeros beyond the last column meet zeros
      x.place(room, direct(a->x, a->ldx, a->d_in));
      wg.place(room, in);
      wu.place(room, in);
      wd.place(room, out);
    }
    sums = room.take<char>(std::max({plain.sums, keeping.sums, down.sums}));  // either call may follow the other in the same workspace
  }
};

template <typename T, int ACT>
int forward(const b2c_ffn_args* a, const Drop& d, hipStream_t stream) {
  Room room{(char*)a->workspace};
  const ForwardPlan<T> p(a, room);
  int rc;
  Packs<T> packs;
  for (const Operand<T>* o : {&p.x, &p.wg, &p.wu, &p.wd}) o->add_to(packs);
  if ((rc = make(packs, stream))) return rc;
  const GateOut<T, ACT> gate{p.h, (float*)a->saved, p.fp, a->d_hidden};
  Product<T> in{p.x.side(), p.wg.side(), {}, p.wu.side(), a->rows, p.fp, a->d_in, 0, a->rows, a->d_hidden};
  if ((rc = product<T, false, false, true, false>(in, p.gate, p.sums, gate, stream))) return rc;
  const RowsOut<T> out{(T*)a->y, a->ldy, (const T*)a->residual, a->ldr, a->d_out, d};
  Product<T> down{{p.h, p.fp}, p.wd.side(), {}, {}, a->rows, a->d_out, a->d_hidden, 0, a->rows, a->d_out};
  return product<T, false, false, false, false>(down, p.down, p.sums, out, stream);
}

template <typename T>
struct BackwardPlan {
  int64_t fp;
  T* dgu;
  Operand<T> x, wg, wu, wd, dz;
  Way back, dw, dx;
  void* sums;
  BackwardPlan(const b2c_ffn_grad_args* b, const Drop& d, Room& room) {
    const b2c_ffn_args* a = &b->fwd;
    const int64_t M = a->rows;
    fp = up(a->d_hidden, 64);
    dgu = room.take<T>(M * 2 * fp);
    back = choose({{M, fp}}, steps_of(a->d_out), false, false, 12);
    const Extent in{fp + a->d_hidden, a->d_in}, down{a->d_out, a->d_hidden};
    const int64_t k = steps_of(M);
    dw = b->dw_down && (b->dw_gate || b->dw_up) ? choose({in, down}, k, false, false)
         : b->dw_down                           ? choose({down}, k, false, false)
                                                : choose({in}, k, false, false);
    dx = choose({{M, a->d_in}}, 2 * steps_of(a->d_hidden), false, false);
    x = {{(const T*)a->x, a->ldx}, M, a->d_in};
    wg = {{(const T*)a->w_gate, a->ld_in}, a->d_hidden, a->d_in};
    wu = {{(const T*)a->w_up, a->ld_in}, a->d_hidden, a->d_in};
    wd = {{(const T*)a->w_down, a->ld_out}, a->d_out, a->d_hidden};
    dz = {{(const T*)b->dy, b->lddy}, M, a->d_out};
    dz.drop = d;
    if (b->dw_gate || b->dw_up) x.place(room, direct(a->x, a->ldx, a->d_in));
    if (b->dx) {
      const bool in = direct(a->w_gate, a->ld_in, a->d_in) && direct(a->w_up, a->ld_in, a->d_in);
      wg.place(room, in);
      wu.place(room, in);
    }
    wd.place(room, direct(a->w_down, a->ld_out, a->d_hidden));
    dz.place(room, !d.threshold && direct(b->dy, b->lddy, a->d_out));
    sums = room.take<char>(std::max(back.sums, std::max(dw.sums, dx.sums)));
  }
};

template <typename T>
int block_backward(const b2c_ffn_grad_args* b, const Drop& d, hipStream_t stream) {
  const b2c_ffn_args* a = &b->fwd;
  Room room{(char*)b->workspace};
  const BackwardPlan<T> p(b, d, room);
  const int64_t fp = p.fp, M = a->rows;
  const float scale = d.threshold ? d.scale : 1.f;
  int rc;
  if (!b->dx && !b->dw_gate && !b->dw_up && !b->dw_down) return hipSuccess;
  if (M) {
    Packs<T> packs;
    for (const Operand<T>* o : {&p.x, &p.wg, &p.wu, &p.wd, &p.dz}) o->add_to(packs);
    if ((rc = make(packs, stream))) return rc;
  }
  const Side<T> dz = p.dz.side(), x = p.x.side(), dgu{p.dgu, 2 * fp};
  const GateBack<T> back{(const float*)a->saved, p.dgu, fp, a->d_hidden, scale};
  const Product<T> dh{dz, p.wd.side(), {}, {}, M, fp, a->d_out, 0, M, a->d_hidden};
  if ((rc = product<T, true, false, false, false>(dh, p.back, p.sums, back, stream))) return rc;
  const bool f32 = b->grad_dtype == B2C_F32, add = b->accumulate != 0;
  const bool in = b->dw_gate || b->dw_up;
  const WeightOut<T> to_in{b->dw_gate, b->dw_up, b->ld_din, a->d_hidden, (int)fp, a->d_in, f32, add, 1.f};
  const WeightOut<T> to_down{b->dw_down, nullptr, b->ld_dout, a->d_out, 0, a->d_hidden, f32, add, scale};
  const Product<T> dwi{dgu, x, {}, {}, fp + a->d_hidden, a->d_in, M, 0, fp + a->d_hidden, a->d_in};
  const Product<T> dwd{dz, {kept_h<T>(a), fp}, {}, {}, a->d_out, a->d_hidden, M, 0, a->d_out, a->d_hidden};
  if (in && b->dw_down) {  // together: one launch, and fewer compute units without work in its last round
    Jobs<T, WeightOut<T>, 2> both{{dwi, dwd}, {to_in, to_down}, {}, {}};
    rc = products<T, true, true, false, false>(both, p.dw, p.sums, stream);
  } else if (in) {
    rc = product<T, true, true, false, false>(dwi, p.dw, p.sums, to_in, stream);
  } else if (b->dw_down) {
    rc = product<T, true, true, false, false>(dwd, p.dw, p.sums, to_down, stream);
  }
  if (rc) return rc;
  if (b->dx) {
    const RowsOut<T> out{(T*)b->dx, b->lddx, nullptr, 0, a->d_in, {}};
    const Product<T> dx{dgu, p.wg.side(), {p.dgu + fp, 2 * fp}, p.wu.side(), M, a->d_in, a->d_hidden, a->d_hidden, M, a->d_in};
    if ((rc = product<T, true, false, false, true>(dx, p.dx, p.sums, out, stream))) return rc;
  }
  return hipSuccess;
}

template <typename T>
int forward(const b2c_ffn_args* a, const Drop& d, hipStream_t s) {
  if (is_head(a)) return head_forward<T>(a, d, s);
  if (a->act == B2C_ACT_SILU) return forward<T, B2C_ACT_SILU>(a, d, s);
  if (a->act == B2C_ACT_GELU) return forward<T, B2C_ACT_GELU>(a, d, s);
  return forward<T, B2C_ACT_RELU>(a, d, s);
}
template <typename T>
int backward(const b2c_ffn_grad_args* a, const Drop& d, hipStream_t s) {
  if (is_head(&a->fwd)) return head_backward<T>(a, d, s);
  return block_backward<T>(a, d, s);
}

}  // namespace
}  // namespace dev
}  // namespace b2c

using namespace b2c::dev;

extern "C" size_t b2c_ffn_saved_bytes(const b2c_ffn_args* a) {
  Drop d;
  return sizes_ok(a, &d) && !is_head(a) ? (size_t)a->rows * up(a->d_hidden, 64) * (2 * sizeof(float) + 2) : 0;
}
extern "C" size_t b2c_ffn_workspace_bytes(const b2c_ffn_args* a) {
  Drop d;
  if (!sizes_ok(a, &d) || a->rows == 0) return 0;
  Room room{nullptr};
  if (is_head(a)) HeadPlan<bf16>(a, nullptr, room);  // both types have the same size
  else ForwardPlan<bf16>(a, room);
  return room.used;
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
  Room room{nullptr};
  if (is_head(&b->fwd)) HeadPlan<bf16>(&b->fwd, b, room);
  else BackwardPlan<bf16>(b, d, room);
  return room.used;
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
        (b->dx && !good(b->dx, b->lddx, a->d_in, 2)) || (!a->saved && !is_head(a)) ||
        reinterpret_cast<uintptr_t>(a->saved) % 16)
      return hipErrorInvalidValue;
  }
  if (!room_ok(b->workspace, b->workspace_bytes, b2c_ffn_grad_workspace_bytes(b))) return hipErrorInvalidValue;
  return a->dtype == B2C_F16 ? backward<f16>(b, d, stream) : backward<bf16>(b, d, stream);
}
