// How the rows of asc_process_logits are cut into slices, one for each workgroup.
#pragma once

#include <stdint.h>

namespace asc {

// Slices of `size` tokens for a row of `vocab`.  Slices begin at 16 bytes, up to 16 / element - 1 tokens before a row that does
// not (aligned: all rows do); the last ones of a row that begins nearer may be empty.
constexpr int64_t slices_of(int64_t vocab, int size, int element, bool aligned) {
  return (vocab + (aligned ? 0 : 16 / element - 1) + size - 1) / size;
}

// The token that a slice begins at, `lead` before the row's first in slice 0.
constexpr int slice_first(int slice, int size, int lead) { return slice * size - lead; }

// Places of the slice up to the row's end, none where it begins behind that.
constexpr uint32_t slice_places(int first, int size, int vocab) {
  return first >= vocab ? 0 : (size < vocab - first ? size : vocab - first);
}

}  // namespace asc
