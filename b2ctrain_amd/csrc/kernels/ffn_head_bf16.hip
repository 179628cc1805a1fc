// The narrow feed-forward block's kernels in bfloat16.
#include "ffn_head.h"

namespace b2c {
namespace dev {

template <>
int head_forward<bf16>(const b2c_ffn_args* a, const Drop& d, hipStream_t s) {
  if (a->act == B2C_ACT_SILU) return head_forward_by_width<bf16, B2C_ACT_SILU>(a, d, s);
  if (a->act == B2C_ACT_GELU) return head_forward_by_width<bf16, B2C_ACT_GELU>(a, d, s);
  return head_forward_by_width<bf16, B2C_ACT_RELU>(a, d, s);
}
template <>
int head_backward<bf16>(const b2c_ffn_grad_args* b, const Drop& d, hipStream_t s) {
  if (b->fwd.act == B2C_ACT_SILU) return head_backward_by_width<bf16, B2C_ACT_SILU>(b, d, s);
  if (b->fwd.act == B2C_ACT_GELU) return head_backward_by_width<bf16, B2C_ACT_GELU>(b, d, s);
  return head_backward_by_width<bf16, B2C_ACT_RELU>(b, d, s);
}

}  // namespace dev
}  // namespace b2c
