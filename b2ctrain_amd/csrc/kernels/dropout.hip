// Dropout with a mask that is formed from a counter and never stored (b2c_hip_dropout).
#include "dense.h"

namespace b2c {
namespace dev {
namespace {

// Rows that follow each other without a gap in every matrix, all on 16 bytes: a thread takes the eight elements of a counter
// in one access. Bound by memory: 8192 x 4096 in bfloat16 with a residual, and its gradient, 62 us, 5.4 TB/s; a copy
// of 0.5 GiB reaches 5.3.
template <typename T>
__global__ __launch_bounds__(256) void flat_kernel(const T* x, const T* r, T* y, uint64_t n, Drop d) {
  const uint64_t q = (uint64_t)block_index() * 256 + threadIdx.x, e = q * 8;
  if (e >= n) return;
  Philox4 w{};
  if (d.threshold) w = philox(q, d.stream, d.seed);
  if (e + 8 <= n) {
    const vec<T, 8> a = *reinterpret_cast<const vec<T, 8>*>(x + e);
    vec<T, 8> b{};
    if (r) b = *reinterpret_cast<const vec<T, 8>*>(r + e);
    vec<T, 8> o;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float v = kept(w, j, d.threshold) ? (float)a[j] * d.scale : 0.f;
      if (r) v += (float)b[j];
      o[j] = (T)v;
    }
    *reinterpret_cast<vec<T, 8>*>(y + e) = o;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; j++) {
    if (e + j >= n) break;
    float v = kept(w, j, d.threshold) ? (float)x[e + j] * d.scale : 0.f;
    if (r) v += (float)r[e + j];
    y[e + j] = (T)v;
  }
}

// Any rows: a wave takes 512 elements in their order, lane l first forms the bits of the l-th counter of them and then
// moves elements l, l + 64, ..., neighbouring lanes neighbouring elements, fetching their bits from the lane that has them. Bound by
// memory: 333333 x 45 in single precision, rows three apart, and its gradient, 50 us, 4.8 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void rows_kernel(const T* x, int64_t ldx, const T* r, int64_t ldr, T* y, int64_t ldy, uint64_t n,
                                                   uint32_t cols, Drop d) {
  const int lane = threadIdx.x & 63;
  const uint64_t first = ((uint64_t)block_index() * 4 + (threadIdx.x >> 6)) * 512;
  if (first >= n) return;
  uint32_t bits = 255;
  if (d.threshold) {
    const Philox4 w = philox(first / 8 + lane, d.stream, d.seed);
    bits = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) bits |= (uint32_t)kept(w, j, d.threshold) << j;
  }
  const uint32_t down = 64 / cols, right = 64 % cols;
  const uint64_t m = (first + lane) / cols;
  uint32_t c = (uint32_t)((first + lane) - m * cols);
  // Places advance by sums: a product m ld for each element took longer than the memory does.
  int64_t px = (int64_t)m * ldx + c, pr = (int64_t)m * ldr + c, py = (int64_t)m * ldy + c;
  const int64_t dx = (int64_t)down * ldx + right, dr = (int64_t)down * ldr + right, dy = (int64_t)down * ldy + right;
  // All loads first and without conditions (a last, partial wave reads its first element again for those that are not there): one
  // at a time, each store holds up the next load, which it might be the source of.
  const bool whole = first + 512 <= n;
  float v[8], add[8];
  int64_t to[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const bool there = whole || first + j * 64 + lane < n;
    const int64_t m0 = (int64_t)(first / cols), c0 = (int64_t)(first - (uint64_t)m0 * cols);
    v[j] = (float)x[there ? px : m0 * ldx + c0];
    add[j] = r ? (float)r[there ? pr : m0 * ldr + c0] : 0.f;
    to[j] = there ? py : -1;
    c += right;
    px += dx;
    pr += dr;
    py += dy;
    if (c >= cols) {
      c -= cols;
      px += ldx - (int64_t)cols;
      pr += ldr - (int64_t)cols;
      py += ldy - (int64_t)cols;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const bool keep = __shfl(bits, j * 8 + (lane >> 3)) >> (lane & 7) & 1;
    float o = keep ? v[j] * d.scale : 0.f;
    if (r) o += add[j];
    if (to[j] >= 0) y[to[j]] = (T)o;
  }
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T>
int launch(const b2c_dropout_args* a, const Drop& d, hipStream_t stream) {
  const uint64_t n = (uint64_t)a->rows * (uint64_t)a->cols, blocks = (n + 2047) / 2048;
  const bool flat = (a->rows == 1 || (a->ldx == a->cols && a->ldy == a->cols && (!a->residual || a->ldr == a->cols))) &&
                    on16(a->x) && on16(a->y) && on16(a->residual);
  const T *x = (const T*)a->x, *r = (const T*)a->residual;
  if (flat) flat_kernel<T><<<grid_of((int64_t)blocks), 256, 0, stream>>>(x, r, (T*)a->y, n, d);
  else rows_kernel<T><<<grid_of((int64_t)blocks), 256, 0, stream>>>(x, a->ldx, r, a->ldr, (T*)a->y, a->ldy, n, (uint32_t)a->cols, d);
  return hipGetLastError();
}

}  // namespace
}  // namespace dev
}  // namespace b2c

extern "C" int b2c_hip_dropout(const b2c_dropout_args* a, hipStream_t stream) {
  using namespace b2c::dev;
  Drop d;
  if (!a || a->rows < 0 || a->cols < 1 || a->cols > 0x7fffffff || !drop_of(a->p, a->seed, a->stream, &d))
    return hipErrorInvalidValue;
  if (a->rows && (uint64_t)a->rows > ((uint64_t)1 << 41) / (uint64_t)a->cols) return hipErrorInvalidValue;
  const size_t size = a->dtype == B2C_F32 ? 4 : 2;
  if (a->dtype != B2C_F32 && a->dtype != B2C_F16 && a->dtype != B2C_BF16) return hipErrorInvalidValue;
  if (a->rows == 0) return hipSuccess;
  if (!good(a->x, a->ldx, a->cols, size) || !good(a->y, a->ldy, a->cols, size) ||
      (a->residual && !good(a->residual, a->ldr, a->cols, size)))
    return hipErrorInvalidValue;
  if (a->dtype == B2C_F32) return launch<float>(a, d, stream);
  if (a->dtype == B2C_F16) return launch<f16>(a, d, stream);
  return launch<bf16>(a, d, stream);
}
