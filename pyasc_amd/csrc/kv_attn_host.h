// Host checks that the attention entries over other keys than the queries' share.
#pragma once

#include "common.h"
#include "kv_attn_kernels.h"
#include "overlap.h"

namespace asc {
namespace kv {

// The arguments' types, shapes and scale.
int32_t check_shape(const asc_attention_t* a, const char* what);

// Keys' or values' strides in units of 16 bytes, checked so that a row's place fits 32 bits.
int32_t strides_of(const asc_rows_t& r, int64_t batch, int64_t heads, int64_t rows, int head_dim, const char* what,
                   Strides& s);

// Whether rows can be read and written in 16-byte pieces.
bool row_operand(const asc_rows_t& r);

// Every result shares no byte with an operand nor with another result.
template <int kResults, int kOperands>
int32_t check_places(const char* what, const Region (&results)[kResults], const Region (&operands)[kOperands]) {
  for (int i = 0; i < kResults; ++i) {
    for (const Region& x : operands) {
      ASC_REQUIRE(!overlap(results[i], x), ASC_ERR_INVALID_ARG, "%s: '%s' overlaps '%s'", what, results[i].name, x.name);
    }
    for (int j = 0; j < i; ++j) {
      ASC_REQUIRE(!overlap(results[i], results[j]), ASC_ERR_INVALID_ARG, "%s: '%s' overlaps '%s'", what,
                  results[i].name, results[j].name);
    }
  }
  return ASC_OK;
}

}  // namespace kv
}  // namespace asc
