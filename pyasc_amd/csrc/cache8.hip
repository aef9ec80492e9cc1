// The append to a cache held in 8 bits, and the read that gives its values back.
//
// append: a group of waves owns one head's block of rows.  It loads the block's new rows into registers, takes the
// largest of them, and stores their codes under the scale that the block then has.  Where the
// scale of earlier rows has to grow it rewrites their codes.  Scales are powers of two, so x / s is exact, and
// codes of e4m3 are rescaled without a rounding but below its normal range.
#include <cmath>

#include "cache8.h"

namespace {

using asc::c8::Cache;
using asc::c8::u32x2;
using asc::c8::u32x4;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct RowsArgs {
  Cache c;
  uint8_t* k_new;
  uint8_t* v_new;
  int64_t k_batch, k_head, k_seq, v_batch, v_head, v_seq;  // elements
  asc::Divisor heads, blocks;  // blocks that n tokens can reach (append), or runs of tokens (read)
  int32_t batch;
};

template <bool kBf16>
__device__ __forceinline__ float to_f32(uint16_t x) {
  return kBf16 ? asc::bf16_to_f32(x) : asc::f16_to_f32(x);
}

// The least 2^e >= 2^-126 with amax <= kMost 2^e, for a finite amax >= 0.
template <class Q>
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = static_cast<int>(bits >> 23) - Q::kExponent + ((bits & 0x7fffffu) > Q::kMantissa ? 1 : 0);
  e = e < 1 ? 1 : e;  // biased: 2^-126
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}

template <int kWaves>
__device__ __forceinline__ float group_max(float v, float (&waves)[kWaves]) {
  v = asc::wave_max(v);
  if (kWaves == 1) return v;
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v = fmaxf(v, waves[w]);
  return v;
}

// kVecs: vectors of eight values that a thread holds.  A block of more goes through them twice, for its largest
// value and for its codes.
template <int D, class Q, bool kBf16, int kWaves, int kVecs>
__global__ void __launch_bounds__(kWaves * 64) append(RowsArgs p) {
  constexpr int kThreads = kWaves * 64, kPerRow = D / 8, kChunk = kThreads * kVecs;
  __shared__ float waves[kWaves], waves_special[kWaves], waves_finite[kWaves];
  const Cache& c = p.c;
  uint32_t id = blockIdx.x;
  const bool is_v = id & 1;
  id >>= 1;
  const uint32_t pair = p.blocks.divide(id);
  const int slot = static_cast<int>(id - pair * p.blocks.d);
  const int b = static_cast<int>(p.heads.divide(pair)), head = static_cast<int>(pair - b * p.heads.d);
  const int length = c.lengths[b], n = c.news ? c.news[b] : c.n;
  if (length < 0 || n <= 0 || n > c.n || length > c.capacity - n) return;
  const int size = static_cast<int>(c.block.d);
  const int start = (static_cast<int>(c.block.divide(length)) + slot) * size;  // the block's first key
  if (start >= length + n) return;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(is_v ? p.v_new : p.k_new) +
                      b * (is_v ? p.v_batch : p.k_batch) + head * (is_v ? p.v_head : p.k_head);
  const int64_t step = is_v ? p.v_seq : p.k_seq;
  const int old = length - start;  // rows before it are there already
  const int end = min(size, length + n - start);
  const int first_vec = max(old, 0) * kPerRow, end_vec = end * kPerRow;

  u32x4 held[kVecs];
  const auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int vec = base + i * kThreads + static_cast<int>(threadIdx.x);
      held[i] = u32x4{0, 0, 0, 0};
      if (vec < end_vec) held[i] = *reinterpret_cast<const u32x4*>(x + (vec / kPerRow - old) * step + vec % kPerRow * 8);
    }
  };
  // the new rows, the page and the held scale are under way together
  load(first_vec);
  uint32_t page, row;
  const bool good = asc::c8::place(c, b, start, page, row);
  const auto& strides = is_v ? c.vs : c.ks;
  float* scale_place = (is_v ? c.v_scale : c.k_scale) + asc::c8::scale_at(c, is_v ? c.vss : c.kss, good ? page : 0, head, row);
  float before = 0.0f;
  if (old > 0) before = *scale_place;
  if (!good) return;
  uint8_t* codes = (is_v ? c.v : c.k) + asc::c8::row_at(strides, page, head, row);
  const uint64_t row_bytes = static_cast<uint64_t>(strides.row) * 16;  // a block's rows may span more than 4 GiB

  // magnitudes are ordered as the integers of their bits, infinities and NaN above all
  const bool once = end_vec - first_vec <= kChunk;
  u16x2 most = {0, 0};
  for (int base = first_vec; base < end_vec; base += kChunk) {
    if (!once) load(base);
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, held[i][w] & 0x7fff7fffu));
      }
  }
  const uint16_t top = most[0] > most[1] ? most[0] : most[1];
  const float largest = group_max(kBf16 ? asc::bf16_to_f32(top) : (top >= 0x7c00u ? INFINITY : asc::f16_to_f32(top)), waves);
  // a bf16 NaN is lost in group_max, but not that a lane had one
  const bool special = group_max(top >= (kBf16 ? 0x7f80u : 0x7c00u) ? 1.0f : 0.0f, waves_special) != 0.0f;
  float amax = largest;
  if (special) {  // of the finite ones
    amax = 0.0f;
    for (int base = first_vec; base < end_vec; base += kChunk) {
      if (!once) load(base);
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = fabsf(to_f32<kBf16>(static_cast<uint16_t>(held[i][e / 2] >> (e % 2 * 16))));
          amax = v < INFINITY ? fmaxf(amax, v) : amax;
        }
    }
    amax = group_max(amax, waves_finite);
  }
  float scale = scale_for<Q>(amax);
  if (!(before > 0.0f && before < INFINITY)) before = 0.0f;
  const bool grows = before < scale;
  if (!grows) scale = before;

  const auto in_range = [&](float v) {
    if (v != v) return Q::of_nan(v);
    return fminf(fmaxf(v, -Q::kMost), Q::kMost);
  };
  // By a power of two the quotient is a product, and finite values need no bounds.
  const bool power = (__float_as_uint(scale) & 0x7fffffu) == 0 && scale >= 0x1p-126f && scale <= 0x1p126f;
  const bool plain = power && !special;
  const float inverse = power ? 1.0f / scale : 0.0f;
  for (int base = first_vec; base < end_vec; base += kChunk) {
    if (!once) load(base);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int vec = base + i * kThreads + static_cast<int>(threadIdx.x);
      u32x2 w;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = to_f32<kBf16>(static_cast<uint16_t>(held[i][half * 2 + e / 2] >> (e % 2 * 16)));
        if (plain) {
          w[half] = Q::pack(q, inverse);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = in_range(power ? q[e] * inverse : q[e] / scale);
          w[half] = Q::pack(q, 1.0f);
        }
      }
      if (vec < end_vec) *reinterpret_cast<u32x2*>(codes + (vec / kPerRow) * row_bytes + vec % kPerRow * 8) = w;
    }
  }
  if (old > 0 && grows) {
    __syncthreads();  // all have read the scale
    const float ratio = before / scale;  // by a power of two; a code times `before` may lie outside fp32
    for (int vec = threadIdx.x; vec < first_vec; vec += kThreads) {
      u32x2* at = reinterpret_cast<u32x2*>(codes + (vec / kPerRow) * row_bytes + vec % kPerRow * 8);
      u32x2 w = *at;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = in_range(Q::value(w[half], e) * ratio);
        w[half] = Q::pack(q, 1.0f);
      }
      *at = w;
    }
  }
  if (threadIdx.x == 0 && (old <= 0 || grows)) *scale_place = scale;
}

// A workgroup reads a run of tokens of one head, kVecs vectors of eight values per thread, whose pages, codes and scales are
// under way together.  Results are written past the caches.  50 MB (8 sequences of 500 to 1999 tokens from int8 to fp16) in 11.4 us:
// with four vectors 15.9, with one 13.2, with stores through the caches 13.3.
constexpr int kReadVecs = 2;
template <int D>
constexpr int kReadTokens = 256 * kReadVecs / (D / 8);

template <int D, class Q, class T>
__global__ void __launch_bounds__(256) read(RowsArgs p) {
  constexpr int kPerRow = D / 8, kStep = 256 / kPerRow;
  const Cache& c = p.c;
  uint32_t pair = p.blocks.divide(blockIdx.x);
  const int first = static_cast<int>(blockIdx.x - pair * p.blocks.d) * kReadTokens<D> + static_cast<int>(threadIdx.x) / kPerRow;
  const bool is_v = p.k_new == nullptr || pair >= p.heads.d * p.batch;
  if (is_v && p.k_new) pair -= p.heads.d * p.batch;
  const int b = static_cast<int>(p.heads.divide(pair)), head = static_cast<int>(pair - b * p.heads.d);
  const int ch = static_cast<int>(threadIdx.x) % kPerRow;
  const int start = c.lengths[b], n = c.news ? c.news[b] : c.n;
  const bool fits = start >= 0 && n <= c.n && start <= c.capacity - n;
  const auto& strides = is_v ? c.vs : c.ks;
  const uint8_t* codes = is_v ? c.v : c.k;
  const float* scales = is_v ? c.v_scale : c.k_scale;
  T* to = reinterpret_cast<T*>(is_v ? p.v_new : p.k_new) + b * (is_v ? p.v_batch : p.k_batch) + head * (is_v ? p.v_head : p.k_head) +
          ch * 8;
  const int64_t step = is_v ? p.v_seq : p.k_seq;
  const int most = min(n, c.n);  // written, whatever the lengths are
  uint32_t page[kReadVecs], row[kReadVecs];
  bool good[kReadVecs];
#pragma unroll
  for (int i = 0; i < kReadVecs; ++i) {
    const int token = first + i * kStep;
    page[i] = row[i] = 0;
    good[i] = fits && token < most;
    if (good[i]) good[i] = asc::c8::place(c, b, start + token, page[i], row[i]);
  }
  u32x2 w[kReadVecs];
  float scale[kReadVecs];
#pragma unroll
  for (int i = 0; i < kReadVecs; ++i) {
    w[i] = u32x2{0, 0};
    scale[i] = __builtin_nanf("");
    if (good[i]) {
      w[i] = *reinterpret_cast<const u32x2*>(codes + asc::c8::row_at(strides, page[i], head, row[i]) + ch * 8);
      scale[i] = scales[asc::c8::scale_at(c, is_v ? c.vss : c.kss, page[i], head, row[i])];
    }
  }
#pragma unroll
  for (int i = 0; i < kReadVecs; ++i) {
    const int token = first + i * kStep;
    if (token >= most) continue;
    T packed[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) packed[e] = static_cast<T>(Q::value(w[i][e / 4], e % 4) * scale[i]);
#pragma unroll
    for (int e = 0; e < static_cast<int>(sizeof(T)) / 2; ++e) {
      __builtin_nontemporal_store(reinterpret_cast<const u32x4*>(packed)[e], reinterpret_cast<u32x4*>(to + token * step) + e);
    }
  }
}

struct Launch {
  RowsArgs p{};
  int tensors = 0;
};

int32_t make(const asc_cache8_t* a, bool reads, const char* what, Launch& L) {
  int32_t rc = asc::c8::make_cache(a, what, L.p.c);
  if (rc != ASC_OK) return rc;
  const bool wide = reads && a->dtype == ASC_DT_FLOAT32;
  ASC_REQUIRE(a->dtype == ASC_DT_FLOAT16 || a->dtype == ASC_DT_BFLOAT16 || wide, ASC_ERR_UNSUPPORTED,
              "%s: dtype %d not supported", what, a->dtype);
  if (a->batch == 0 || a->kv_heads == 0 || a->n == 0) return ASC_OK;
  // a block's vectors of eight values and a step of a workgroup behind them are numbered in 32 bits
  ASC_REQUIRE(reads || static_cast<int64_t>(a->scale_block) * (a->head_dim / 8) < int64_t{1} << 30, ASC_ERR_UNSUPPORTED,
              "%s: scale_block %d is too large (below 2^27 rows of 64 values, 2^26 of 128)", what, a->scale_block);
  ASC_REQUIRE(reads ? a->k_new.data || a->v_new.data : a->k_new.data && a->v_new.data, ASC_ERR_INVALID_ARG,
              "%s: null buffer", what);
  const int64_t element = wide ? 4 : 2;
  ASC_REQUIRE(asc::c8::row_operand(a->k_new, element) && asc::c8::row_operand(a->v_new, element), ASC_ERR_ALIGNMENT,
              "%s: k_new and v_new must be 16-byte aligned, with strides that are multiples of %d", what,
              static_cast<int>(16 / element));
  RowsArgs& p = L.p;
  p.k_new = static_cast<uint8_t*>(a->k_new.data);
  p.v_new = static_cast<uint8_t*>(a->v_new.data);
  p.k_batch = a->k_new.batch_stride;
  p.k_head = a->k_new.head_stride;
  p.k_seq = a->k_new.seq_stride;
  p.v_batch = a->v_new.batch_stride;
  p.v_head = a->v_new.head_stride;
  p.v_seq = a->v_new.seq_stride;
  p.batch = static_cast<int32_t>(a->batch);
  p.heads = asc::divisor_of(static_cast<uint32_t>(a->kv_heads));
  L.tensors = (p.k_new != nullptr) + (p.v_new != nullptr);
  asc::Region cache[asc::c8::kRegions];
  asc::c8::regions_of(*a, cache);
  const asc::Region rows[] = {
      asc::region_of("k_new", a->k_new, a->batch, a->kv_heads, a->n, a->head_dim, element),
      asc::region_of("v_new", a->v_new, a->batch, a->kv_heads, a->n, a->head_dim, element)};
  // what is written: the rows (read), or the cache's codes and scales (append)
  for (const asc::Region& r : rows) {
    for (int i = 0; i < (reads ? asc::c8::kRegions : 4); ++i) {
      ASC_REQUIRE(!asc::overlap(r, cache[i]), ASC_ERR_INVALID_ARG, "%s: '%s' overlaps '%s'", what, r.name, cache[i].name);
    }
  }
  if (reads) {
    ASC_REQUIRE(!asc::overlap(rows[0], rows[1]), ASC_ERR_INVALID_ARG, "%s: 'k_new' overlaps 'v_new'", what);
  } else {
    for (int i = 0; i < 4; ++i) {
      for (int j = i + 1; j < asc::c8::kRegions; ++j) {
        ASC_REQUIRE(!asc::overlap(cache[i], cache[j]), ASC_ERR_INVALID_ARG, "%s: '%s' overlaps '%s'", what,
                    cache[i].name, cache[j].name);
      }
    }
  }
  return ASC_OK;
}

template <int D, class Q, bool kBf16>
int32_t launch_append(const Launch& L, int64_t units, hipStream_t s) {
  const int64_t vecs = std::min<int64_t>(L.p.c.block.d, L.p.c.n) * (D / 8);
  const dim3 grid(static_cast<uint32_t>(units));
  if (vecs <= 64) {
    hipLaunchKernelGGL((append<D, Q, kBf16, 1, 1>), grid, dim3(64), 0, s, L.p);
  } else if (vecs <= 256) {
    hipLaunchKernelGGL((append<D, Q, kBf16, 1, 4>), grid, dim3(64), 0, s, L.p);
  } else if (vecs <= 1024) {
    hipLaunchKernelGGL((append<D, Q, kBf16, 4, 4>), grid, dim3(256), 0, s, L.p);
  } else {
    hipLaunchKernelGGL((append<D, Q, kBf16, 4, 16>), grid, dim3(256), 0, s, L.p);
  }
  return ASC_OK;
}

template <int D, class Q>
void launch_read(const Launch& L, int32_t dtype, int64_t groups, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(groups));
  if (dtype == ASC_DT_FLOAT32) {
    hipLaunchKernelGGL((read<D, Q, float>), grid, dim3(256), 0, s, L.p);
  } else if (dtype == ASC_DT_FLOAT16) {
    hipLaunchKernelGGL((read<D, Q, _Float16>), grid, dim3(256), 0, s, L.p);
  } else {
    hipLaunchKernelGGL((read<D, Q, __bf16>), grid, dim3(256), 0, s, L.p);
  }
}

}  // namespace

namespace asc {
namespace c8 {

bool row_operand(const asc_rows_t& r, int64_t element) {
  return aligned16(r.data) && (((r.batch_stride | r.head_stride | r.seq_stride) * element) & 15) == 0;
}

namespace {

// Offsets of rows in units of `unit` elements, which have to fit 32 bits.
int32_t strides_of(const asc_rows_t& r, int64_t pages, int64_t heads, int64_t rows, int64_t unit, int64_t row,
                   const char* what, const char* name, Strides& s) {
  ASC_REQUIRE(r.batch_stride >= 0 && r.head_stride >= 0 && r.seq_stride >= 0, ASC_ERR_INVALID_ARG,
              "%s: negative stride of '%s'", what, name);
  constexpr int64_t limit = (int64_t{1} << 32) - 64;
  const auto term = [&](int64_t n, int64_t stride) {
    return n <= 1 || stride == 0 ? 0 : (stride / unit > limit / (n - 1) ? limit : (n - 1) * (stride / unit));
  };
  ASC_REQUIRE(term(pages, r.batch_stride) + term(heads, r.head_stride) + term(rows, r.seq_stride) + row <= limit,
              ASC_ERR_UNSUPPORTED, "%s: '%s' spans more than 2^32 units", what, name);
  s.page = pages > 1 ? static_cast<uint32_t>(r.batch_stride / unit) : 0;
  s.head = heads > 1 ? static_cast<uint32_t>(r.head_stride / unit) : 0;
  s.row = rows > 1 ? static_cast<uint32_t>(r.seq_stride / unit) : 0;
  return ASC_OK;
}

}  // namespace

int32_t make_cache(const asc_cache8_t* a, const char* what, Cache& c) {
  ASC_REQUIRE(a, ASC_ERR_INVALID_ARG, "%s: null arguments", what);
  ASC_REQUIRE(a->cache_dtype == ASC_DT_INT8 || a->cache_dtype == ASC_DT_FLOAT8_E4M3, ASC_ERR_UNSUPPORTED,
              "%s: cache dtype %d not supported (int8, float8 e4m3)", what, a->cache_dtype);
  ASC_REQUIRE(a->head_dim == 64 || a->head_dim == 128, ASC_ERR_UNSUPPORTED, "%s: head_dim %d not supported (64, 128)",
              what, a->head_dim);
  ASC_REQUIRE(a->batch >= 0 && a->kv_heads >= 0 && a->n >= 0 && a->kv_len >= 0, ASC_ERR_INVALID_ARG,
              "%s: negative shape", what);
  const bool paged = a->block_table != nullptr;
  const int64_t rows = paged ? a->page_size : a->kv_len, pages = paged ? a->num_pages : a->batch;
  ASC_REQUIRE(a->batch < 1 << 20 && a->kv_heads < 1 << 20 && a->batch * a->kv_heads < 1 << 20 && a->n < 1 << 30 &&
                  a->kv_len < 1 << 30,
              ASC_ERR_UNSUPPORTED, "%s: shape too large", what);
  ASC_REQUIRE(!paged || (a->page_size >= 1 && a->page_size < 1 << 30 && a->num_pages >= 0 &&
                         a->num_pages < int64_t{1} << 31 && a->table_stride >= 0),
              ASC_ERR_INVALID_ARG, "%s: invalid pages (%d rows, %lld pages)", what, a->page_size,
              static_cast<long long>(a->num_pages));
  ASC_REQUIRE(a->scale_block >= 16 && a->scale_block % 16 == 0 && rows % a->scale_block == 0, ASC_ERR_INVALID_ARG,
              "%s: scale_block %d must be a multiple of 16 that divides the %lld rows of a page", what, a->scale_block,
              static_cast<long long>(rows));
  if (a->batch == 0 || a->kv_heads == 0) return ASC_OK;
  ASC_REQUIRE(a->lengths, ASC_ERR_INVALID_ARG, "%s: null buffer", what);
  c.lengths = a->lengths;
  c.news = a->new_lengths;
  c.table = a->block_table;
  c.table_stride = a->table_stride;
  c.pages = static_cast<uint32_t>(pages);
  c.capacity = static_cast<int32_t>(pages > 0 ? a->kv_len : 0);
  c.n = static_cast<int32_t>(a->n);
  c.kv_heads = static_cast<int32_t>(a->kv_heads);
  c.page = divisor_of(rows > 0 ? static_cast<uint32_t>(rows) : 16);
  c.block = divisor_of(static_cast<uint32_t>(a->scale_block));
  if (c.capacity == 0) return ASC_OK;  // nothing of it is touched
  ASC_REQUIRE(a->k.data && a->v.data && a->k_scales.data && a->v_scales.data, ASC_ERR_INVALID_ARG, "%s: null buffer",
              what);
  ASC_REQUIRE(row_operand(a->k, 1) && row_operand(a->v, 1), ASC_ERR_ALIGNMENT,
              "%s: the cache must be 16-byte aligned, with strides that are multiples of 16", what);
  c.k = static_cast<uint8_t*>(a->k.data);
  c.v = static_cast<uint8_t*>(a->v.data);
  c.k_scale = static_cast<float*>(a->k_scales.data);
  c.v_scale = static_cast<float*>(a->v_scales.data);
  const int64_t blocks = rows / a->scale_block;
  int32_t rc = strides_of(a->k, pages, a->kv_heads, rows, 16, a->head_dim / 16, what, "k", c.ks);
  if (rc == ASC_OK) rc = strides_of(a->v, pages, a->kv_heads, rows, 16, a->head_dim / 16, what, "v", c.vs);
  if (rc == ASC_OK) rc = strides_of(a->k_scales, pages, a->kv_heads, blocks, 1, 1, what, "k_scales", c.kss);
  if (rc == ASC_OK) rc = strides_of(a->v_scales, pages, a->kv_heads, blocks, 1, 1, what, "v_scales", c.vss);
  return rc;
}

void regions_of(const asc_cache8_t& a, Region (&r)[kRegions]) {
  const bool paged = a.block_table != nullptr;
  const int64_t rows = paged ? a.page_size : a.kv_len, pages = paged ? a.num_pages : a.batch;
  const int64_t blocks = rows / a.scale_block;
  const asc_rows_t table{const_cast<int32_t*>(a.block_table), a.table_stride, 0, 0};
  r[0] = region_of("k", a.k, pages, a.kv_heads, rows, a.head_dim, 1);
  r[1] = region_of("v", a.v, pages, a.kv_heads, rows, a.head_dim, 1);
  r[2] = region_of("k_scales", a.k_scales, pages, a.kv_heads, blocks, 1, 4);
  r[3] = region_of("v_scales", a.v_scales, pages, a.kv_heads, blocks, 1, 4);
  r[4] = region_of("lengths", a.lengths, a.batch * 4);
  r[5] = region_of("new_lengths", a.new_lengths, a.batch * 4);
  r[6] = region_of("block_table", table, a.batch, 1, 1, paged ? ceil_div(a.kv_len, a.page_size) : 0, 4);
}

}  // namespace c8
}  // namespace asc

extern "C" int32_t asc_quantized_cache_append(const asc_cache8_t* a, asc_stream_t stream) {
  const char* what = "asc_quantized_cache_append";
  Launch L;
  const int32_t rc = make(a, false, what, L);
  if (rc != ASC_OK || L.tensors == 0 || L.p.c.capacity == 0) return rc;
  const int64_t block = a->scale_block;
  const int64_t blocks = (a->n + block - 2) / block + 1;
  L.p.blocks = asc::divisor_of(static_cast<uint32_t>(blocks));
  const int64_t units = 2 * a->batch * a->kv_heads * blocks;
  ASC_REQUIRE(units < int64_t{1} << 24, ASC_ERR_UNSUPPORTED, "%s: %lld workgroups exceed the launch grid limit", what,
              static_cast<long long>(units));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool small = a->head_dim == 64, bf16 = a->dtype == ASC_DT_BFLOAT16;
  if (a->cache_dtype == ASC_DT_INT8) {
    using Q = asc::c8::Int8;
    small ? (bf16 ? launch_append<64, Q, true>(L, units, s) : launch_append<64, Q, false>(L, units, s))
          : (bf16 ? launch_append<128, Q, true>(L, units, s) : launch_append<128, Q, false>(L, units, s));
  } else {
    using Q = asc::c8::E4m3;
    small ? (bf16 ? launch_append<64, Q, true>(L, units, s) : launch_append<64, Q, false>(L, units, s))
          : (bf16 ? launch_append<128, Q, true>(L, units, s) : launch_append<128, Q, false>(L, units, s));
  }
  return asc::check_launch(what);
}

extern "C" int32_t asc_quantized_cache_read(const asc_cache8_t* a, asc_stream_t stream) {
  const char* what = "asc_quantized_cache_read";
  Launch L;
  const int32_t rc = make(a, true, what, L);
  if (rc != ASC_OK || L.tensors == 0) return rc;
  const int64_t runs = asc::ceil_div(a->n, a->head_dim == 64 ? kReadTokens<64> : kReadTokens<128>);
  const int64_t groups = L.tensors * a->batch * a->kv_heads * runs;
  ASC_REQUIRE(groups < int64_t{1} << 24, ASC_ERR_UNSUPPORTED, "%s: %lld workgroups exceed the launch grid limit", what,
              static_cast<long long>(groups));
  L.p.blocks = asc::divisor_of(static_cast<uint32_t>(runs));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->cache_dtype == ASC_DT_INT8) {
    a->head_dim == 64 ? launch_read<64, asc::c8::Int8>(L, a->dtype, groups, s)
                      : launch_read<128, asc::c8::Int8>(L, a->dtype, groups, s);
  } else {
    a->head_dim == 64 ? launch_read<64, asc::c8::E4m3>(L, a->dtype, groups, s)
                      : launch_read<128, asc::c8::E4m3>(L, a->dtype, groups, s);
  }
  return asc::check_launch(what);
}
