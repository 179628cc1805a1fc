#include "dense.h"

namespace b2c {

namespace {

// The launchers refuse arguments with hipErrorInvalidValue before they touch the device.
void done(int rc, const char* what) {
  if (rc == hipErrorInvalidValue)
    throw std::runtime_error(std::string(what) + ": invalid arguments (sizes, type, a null or unaligned pointer, or rows that overlap)");
  LAUNCH_CHECK(rc);
}

template <typename Args>
void give_workspace(DenseCtx& ctx, Args& a, size_t bytes, hipStream_t stream) {
  ctx.workspace.reserve(bytes, false, stream);
  a.workspace = ctx.workspace.ptr;
  a.workspace_bytes = ctx.workspace.bytes();
}

// Whether what a forward pass kept is what the gradients of `b` need.
bool same_call(const b2c_ffn_args& a, const b2c_ffn_args& b) {
  return a.rows == b.rows && a.d_in == b.d_in && a.d_hidden == b.d_hidden && a.d_out == b.d_out && a.dtype == b.dtype && a.act == b.act &&
         a.p == b.p && (a.p == 0 || (a.seed == b.seed && a.stream == b.stream));
}

}  // namespace

void dropout(const b2c_dropout_args& a, hipStream_t stream) { done(b2c_hip_dropout(&a, stream), "dropout"); }

void feed_forward(DenseCtx& ctx, b2c_ffn_args a, bool train, hipStream_t stream) {
  a.saved = nullptr;
  if (train) {
    ctx.kept.rows = -1;  // until the call has succeeded
    ctx.saved.reserve(b2c_ffn_saved_bytes(&a), false, stream);
    a.saved = ctx.saved.ptr;
  }
  give_workspace(ctx, a, b2c_ffn_workspace_bytes(&a), stream);
  done(b2c_hip_ffn_forward(&a, stream), "feed_forward");
  if (train) ctx.kept = a;
}

void feed_forward_backward(DenseCtx& ctx, b2c_ffn_grad_args a, hipStream_t stream) {
  if (b2c_ffn_saved_bytes(&a.fwd) && !same_call(ctx.kept, a.fwd))
    throw std::runtime_error("feed_forward_backward: no forward pass of these sizes, type, activation and mask was kept on this context");
  a.fwd.saved = ctx.saved.ptr;
  give_workspace(ctx, a, b2c_ffn_grad_workspace_bytes(&a), stream);
  done(b2c_hip_ffn_backward(&a, stream), "feed_forward_backward");
}

void quantize_rows(const b2c_quantize_args& a, hipStream_t stream) { done(b2c_hip_quantize_rows(&a, stream), "quantize_rows"); }

void i8_linear(DenseCtx& ctx, b2c_i8_linear_args a, hipStream_t stream) {
  give_workspace(ctx, a, b2c_i8_linear_workspace_bytes(&a), stream);
  done(b2c_hip_i8_linear(&a, stream), "i8_linear");
}

void i8_feed_forward(DenseCtx& ctx, b2c_i8_ffn_args a, hipStream_t stream) {
  give_workspace(ctx, a, b2c_i8_ffn_workspace_bytes(&a), stream);
  done(b2c_hip_i8_ffn(&a, stream), "i8_feed_forward");
}

}  // namespace b2c
