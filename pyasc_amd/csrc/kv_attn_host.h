// Host checks that the attention entries over other keys than the queries' share.
#pragma once

#include "common.h"

namespace asc {
namespace kv {

// The arguments' types, shapes and scale.
int32_t check_shape(const asc_attention_t* a, const char* what);

// Whether rows can be read and written in 16-byte pieces.
bool row_operand(const asc_rows_t& r);

}  // namespace kv
}  // namespace asc
