// Dense operators of a learned head (no reference counterpart): the launchers of b2c_kernels.h with their buffers kept and
// their errors thrown. The argument structs are the launchers'; their workspace, workspace_bytes and saved fields are filled
// in here. Nothing is copied or synchronised except where a buffer grows.
#pragma once
#include "util.h"

namespace b2c {

// The buffers of one block: what its last forward pass with `train` left for its backward pass, that call's arguments, and
// workspace. Blocks whose passes are interleaved need one each; calls on one are ordered by their stream.
struct DenseCtx {
  DevBuf<char> saved, workspace;
  b2c_ffn_args kept{};  // rows = -1: nothing is kept
  DenseCtx() { kept.rows = -1; }
};

// y = residual + dropout(x), and on the gradient with the same p, seed and stream the backward pass (b2c_hip_dropout).
void dropout(const b2c_dropout_args& a, hipStream_t stream);

// The gated feed-forward block; with `train`, what feed_forward_backward needs stays in ctx.saved.
void feed_forward(DenseCtx& ctx, b2c_ffn_args a, bool train, hipStream_t stream);
// Its gradients: a.fwd as given to the forward pass on the same context. Throws where kept values are needed (b2c_ffn_saved_bytes is
// not 0) and what is kept is not of a call with these sizes, type, activation and mask.
void feed_forward_backward(DenseCtx& ctx, b2c_ffn_grad_args a, hipStream_t stream);

// Rows to 8 bits with a scale each (weights: rows are output channels), and products of what they give.
void quantize_rows(const b2c_quantize_args& a, hipStream_t stream);
void i8_linear(DenseCtx& ctx, b2c_i8_linear_args a, hipStream_t stream);
void i8_feed_forward(DenseCtx& ctx, b2c_i8_ffn_args a, hipStream_t stream);

// The norms, gate and residual sum between two blocks, and their gradients.
void block_norm(const b2c_block_norm_args& a, hipStream_t stream);
void block_norm_backward(DenseCtx& ctx, b2c_block_norm_grad_args a, hipStream_t stream);

// Groups of columns to 4 bits with a scale each, and products with weights held that way.
void quantize4(const b2c_quantize4_args& a, hipStream_t stream);
void q4_linear(DenseCtx& ctx, b2c_q4_linear_args a, hipStream_t stream);

// A mixture-of-experts layer for a few tokens.
void experts(DenseCtx& ctx, b2c_experts_args a, hipStream_t stream);

}  // namespace b2c
