// A cache held in 8 bits: where its rows and scales lie, and its codes (asc_cache8_t).
#pragma once

#include "common.h"
#include "divisor.h"
#include "numeric.h"
#include "overlap.h"

namespace asc {
namespace c8 {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// In units of 16 bytes (codes) or of elements (scales).
struct Strides {
  uint32_t page, head, row;
};

struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  Strides ks, vs, kss, vss;
  const int32_t* table;  // null: sequence b's rows in page b
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* news;  // null: n
  Divisor page, block;  // rows
  uint32_t pages;
  int32_t capacity, n, kv_heads;
};

// The page of key `key` of sequence b, and its row there; false where the page lies outside the cache.
__device__ __forceinline__ bool place(const Cache& c, int b, uint32_t key, uint32_t& page, uint32_t& row) {
  const uint32_t column = c.page.divide(key);
  row = key - column * c.page.d;
  page = c.table ? static_cast<uint32_t>(c.table[b * c.table_stride + column]) : static_cast<uint32_t>(b);
  return page < c.pages;
}
__device__ __forceinline__ uint64_t row_at(const Strides& s, uint32_t page, uint32_t head, uint32_t row) {
  return static_cast<uint64_t>(page * s.page + head * s.head + row * s.row) * 16;
}
__device__ __forceinline__ uint32_t scale_at(const Cache& c, const Strides& s, uint32_t page, uint32_t head, uint32_t row) {
  return page * s.page + head * s.head + c.block.divide(row) * s.row;
}

// The formats.  kMost: the largest value of a code; kMantissa: its mantissa's bits in fp32; kExponent: its
// exponent's.
struct Int8 {
  static constexpr float kMost = 127.0f;
  static constexpr uint32_t kMantissa = 0x7e0000u;  // 127 = 1.984375 * 2^6
  static constexpr int kExponent = 6;
  // value k (0..3) of a word of codes
  static __device__ __forceinline__ float value(uint32_t w, int k) {
    return static_cast<float>(static_cast<int8_t>(w >> (8 * k)));
  }
  // codes of four values times `inverse`, a power of two, within the format's range: to nearest even, as the sum with
  // 1.5 * 2^23 is rounded, whose lowest byte is the code
  static __device__ __forceinline__ uint32_t pack(const float (&x)[4], float inverse) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __float_as_uint(fmaf(x[k], inverse, 12582912.0f));
    const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(w[3], w[2], 0x04000c0cu);
    return lo | hi;
  }
  static __device__ __forceinline__ float of_nan(float) { return 0.0f; }
};
struct E4m3 {
  static constexpr float kMost = 448.0f;
  static constexpr uint32_t kMantissa = 0x600000u;  // 448 = 1.75 * 2^8
  static constexpr int kExponent = 8;
  static __device__ __forceinline__ float value(uint32_t w, int k) {
    const f32x2 v = k < 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false)
                          : __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    return v[k & 1];
  }
  static __device__ __forceinline__ uint32_t pack(const float (&x)[4], float inverse) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inverse, x[1] * inverse, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inverse, x[3] * inverse, w, true));
  }
  static __device__ __forceinline__ float of_nan(float x) { return x; }
};

// Checks of the cache itself.
int32_t make_cache(const asc_cache8_t* a, const char* what, Cache& c);

// Checks that rows of 16-bit elements (32-bit where `element` is 4) can be moved 16 bytes at a time.
bool row_operand(const asc_rows_t& r, int64_t element);

// The cache's regions, for checks against results: k, v, k_scales, v_scales, lengths, new_lengths, block_table.
constexpr int kRegions = 7;
void regions_of(const asc_cache8_t& a, Region (&r)[kRegions]);

}  // namespace c8
}  // namespace asc
