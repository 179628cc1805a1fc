// The narrow 8-bit block and layer in one kernel each (i8_head.hip).
#pragma once
#include "dense.h"

namespace b2c {
namespace dev {

constexpr int64_t kI8HeadRows = 32;  // above these: the weights are rearranged in each call

bool is_i8_head(const b2c_i8_ffn_args* a);
size_t i8_head_bytes(const b2c_i8_ffn_args* a);  // workspace
int i8_head(const b2c_i8_ffn_args* a, hipStream_t stream);

bool is_i8_narrow(const b2c_i8_linear_args* a);  // a narrow layer, likewise; needs no workspace
int i8_narrow(const b2c_i8_linear_args* a, hipStream_t stream);

}  // namespace dev
}  // namespace b2c
