// Pages of a cache: copies between caches, the fork of sequences that share pages, and compaction.
//
// What a fork does to the pages is worked out by one workgroup, with the reference counts in LDS (64 sequences of 4096
// tokens to 256: 15 us, bound by its instructions over counts and table: with all its first loads asked for together 15.2),
// what a compaction does by as many as the pages need (8192: 5.7 us).  A second launch moves the data and writes the
// tables (8192 pages of 65.5 KB, two fifths used: 258 MB in 45.6 us, 5.7 TB/s).  Nothing comes back to the host, so all of
// them can be captured.  Ranks of free and moving pages are prefix sums and counts are integers: the same result on every
// call.
#include "common.h"
#include "divisor.h"
#include "overlap.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTensors = ASC_MAX_PAGE_TENSORS;
constexpr int kThreads = 256;
constexpr int kPiece = 8192;  // bytes of a page that a workgroup copies at a time, where it lies in one piece

// One tensor's share of a page's move: `pieces` parts, of kPiece bytes (flat) or of a head each.
struct Tensor {
  const uint8_t* from;
  uint8_t* to;
  int64_t from_stride, to_stride;
  int64_t head_stride, row_stride;
  int64_t bytes;  // flat: of a page
  int32_t rows, row_bytes;
  int32_t flat, pieces;
  int32_t width;  // bytes that its addresses and sizes are multiples of: 1, 2, 4 or 16
};

// A kernel's first argument: the tensors are read from where the arguments lie (tensor_of).
struct CopyArgs {
  Tensor t[kTensors];
  asc::Divisor per_move;  // pieces of a move
  asc::Divisor page_size;
  int32_t n_tensors;
  int32_t moves;              // at most
  const int32_t* count;       // null: moves
  const int32_t* from;        // pages
  const int32_t* to;
  const int32_t* used;        // rows of a page that are copied, null: all
  int64_t from_pages, to_pages;
};

// Bytes that are not looked at again soon: 268 MB in 53.6 us (5.0 TB/s; a plain copy of 1 GiB: 6.1), 57.3 with loads and stores that
// stay in the caches.
template <class T>
__device__ __forceinline__ void copy_run(const uint8_t* from, uint8_t* to, int64_t bytes) {
  const T* src = reinterpret_cast<const T*>(from);
  T* dst = reinterpret_cast<T*>(to);
  const int n = static_cast<int>(bytes / static_cast<int64_t>(sizeof(T)));
  int i = threadIdx.x;
  for (; i + kThreads < n; i += 2 * kThreads) {
    const T a = __builtin_nontemporal_load(src + i), b = __builtin_nontemporal_load(src + i + kThreads);
    __builtin_nontemporal_store(a, dst + i);
    __builtin_nontemporal_store(b, dst + i + kThreads);
  }
  if (i < n) dst[i] = src[i];
}

template <class T>
__device__ __forceinline__ void copy_rows(const uint8_t* from, uint8_t* to, int rows, int row_bytes, int64_t stride) {
  const int per = row_bytes / static_cast<int>(sizeof(T));
  const int64_t n = static_cast<int64_t>(rows) * per;
  for (int64_t i = threadIdx.x; i < n; i += kThreads) {
    const int64_t row = i / per;
    const int64_t at = row * stride + (i - row * per) * static_cast<int64_t>(sizeof(T));
    *reinterpret_cast<T*>(to + at) = *reinterpret_cast<const T*>(from + at);
  }
}

// Tensor k.  An array of an argument's struct that is indexed at run time would be copied to scratch memory first:
// 120 us for copies of 268 MB that take 51.
typedef const __attribute__((address_space(4))) Tensor* TensorAt;
__device__ __forceinline__ TensorAt tensor_of(int k) {
  return (TensorAt)__builtin_amdgcn_kernarg_segment_ptr() + k;
}

// Item `item` of all: a move, one of its tensors, a piece of that.
__device__ __forceinline__ void copy_item(const CopyArgs& p, uint32_t item) {
  const uint32_t move = p.per_move.divide(item);
  int piece = static_cast<int>(item - move * p.per_move.d);
  const int64_t from_page = p.from[move], to_page = p.to[move];
  int used = 0;
  if (p.used) used = p.used[move];
  if (from_page < 0 || from_page >= p.from_pages || to_page < 0 || to_page >= p.to_pages) return;
  TensorAt t = tensor_of(0);
  while (piece >= t->pieces) {
    piece -= t->pieces;
    ++t;
  }
  const uint8_t* from = t->from + from_page * t->from_stride;
  uint8_t* to = t->to + to_page * t->to_stride;
  const int width = t->width;
  int64_t bytes;
  if (t->flat) {
    const int64_t at = static_cast<int64_t>(piece) * kPiece;
    bytes = t->bytes - at < kPiece ? t->bytes - at : kPiece;
    from += at;
    to += at;
  } else {
    from += piece * t->head_stride;
    to += piece * t->head_stride;
    int rows = t->rows;
    if (p.used) {
      rows = rows == static_cast<int>(p.page_size.d)
                 ? used
                 : static_cast<int>(p.page_size.divide(static_cast<uint32_t>(used * rows + p.page_size.d - 1)));
    }
    if (t->row_stride != t->row_bytes) {
      if (width == 16) return copy_rows<u32x4>(from, to, rows, t->row_bytes, t->row_stride);
      if (width == 4) return copy_rows<uint32_t>(from, to, rows, t->row_bytes, t->row_stride);
      if (width == 2) return copy_rows<uint16_t>(from, to, rows, t->row_bytes, t->row_stride);
      return copy_rows<uint8_t>(from, to, rows, t->row_bytes, t->row_stride);
    }
    bytes = static_cast<int64_t>(rows) * t->row_bytes;
  }
  if (width == 16) return copy_run<u32x4>(from, to, bytes);
  if (width == 4) return copy_run<uint32_t>(from, to, bytes);
  if (width == 2) return copy_run<uint16_t>(from, to, bytes);
  copy_run<uint8_t>(from, to, bytes);
}

__device__ __forceinline__ void copy_items(const CopyArgs& p, uint32_t first, uint32_t step) {
  const uint32_t items = static_cast<uint32_t>(p.count ? *p.count : p.moves) * p.per_move.d;
  for (uint32_t item = first; item < items; item += step) copy_item(p, item);
}

__global__ void __launch_bounds__(kThreads) page_copy(CopyArgs p) { copy_items(p, blockIdx.x, gridDim.x); }

// ------------------------------------------------------------------------------------ plans

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / asc::kWave;
constexpr int kMostSequences = 4096;

// Sum of v over the lower threads of the workgroup; total: over all.  `waves`: LDS of its own.
__device__ __forceinline__ int prefix(int v, int (&waves)[kPlanWaves], int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = v;
#pragma unroll
  for (int d = 1; d < asc::kWave; d *= 2) {
    const int up = __shfl_up(sum, d, asc::kWave);
    if (lane >= d) sum += up;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = sum;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w < wave) before += waves[w];
    total += waves[w];
  }
  return before + sum - v;
}

// Ranks of the flagged i = k * kPlanThreads + thread < n, in their order, and how many there are.  Neighbouring threads have
// neighbouring i, and rounds behind n are left out by all of them.
template <int kPer>
__device__ __forceinline__ int ranks_of(const bool (&flag)[kPer], int n, int (&rank)[kPer], int* sums,
                                        int (&waves)[kPlanWaves]) {
  static_assert(kPer * kPlanWaves <= kPlanThreads, "a sum for each thread at most");
  const int tid = threadIdx.x, wave = tid >> 6;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (k * kPlanThreads >= n) break;
    const uint64_t set = __builtin_amdgcn_ballot_w64(flag[k]);
    rank[k] = __popcll(set & ((uint64_t{1} << (tid & 63)) - 1));
    if ((tid & 63) == 0) sums[k * kPlanWaves + wave] = __popcll(set);
  }
  __syncthreads();
  const int used = (n + kPlanThreads - 1) / kPlanThreads * kPlanWaves;
  const int mine = tid < used ? sums[tid] : 0;
  int total;
  const int sum = prefix(mine, waves, total);
  if (tid < used) sums[tid] = sum;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (k * kPlanThreads >= n) break;
    rank[k] += sums[k * kPlanWaves + wave];
  }
  return total;
}

struct PlanArgs {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* parents;
  const int32_t* refcounts;
  int32_t* table_out;
  int64_t table_out_stride;
  int32_t* lengths_out;
  int32_t* refcounts_out;
  int32_t* page_map;
  int32_t* count;  // workspace: moves, and where they go
  int32_t* from;
  int32_t* to;
  int32_t* used;
  int32_t page_size, pages, batch, new_batch, width;
  asc::Divisor by_page, by_width;
};

// Pages that sequence b's row holds, 0 where its length does not fit the table.
__device__ __forceinline__ int held_of(const PlanArgs& p, int64_t length) {
  if (length < 0 || length > static_cast<int64_t>(p.width) * p.page_size) return 0;
  return length == 0 ? 0 : static_cast<int>(p.by_page.divide(static_cast<uint32_t>(length - 1))) + 1;
}

// The counts change by (children - 1) for a parent's full pages; its last page, partly filled, is given up only
// by a parent without children.  They go through LDS kCountChunk pages at a time; a page that is
// free after that has a rank, and goes to the child in need of that rank.
__global__ void __launch_bounds__(kPlanThreads) fork_plan(PlanArgs p) {
  constexpr int kCountChunk = 16384, kPer = kCountChunk / kPlanThreads, kRows = kMostSequences / kPlanThreads;
  __shared__ int counts[kCountChunk];
  __shared__ int children[kMostSequences];
  __shared__ int first[kMostSequences];  // child; later 2 * full pages + whether another is partly filled
  __shared__ int fresh[kMostSequences];  // free page of each rank
  __shared__ int sums[kPer * kPlanWaves];
  __shared__ int waves[kPlanWaves];
  const int tid = threadIdx.x;
  int parent[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (k * kPlanThreads >= p.new_batch) break;
    const int i = k * kPlanThreads + tid;
    parent[k] = i < p.new_batch ? p.parents[i] : -1;
    if (parent[k] >= p.batch) parent[k] = -1;
  }
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    children[b] = 0;
    first[b] = p.new_batch;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (k * kPlanThreads >= p.new_batch) break;
    if (parent[k] < 0) continue;
    atomicAdd(&children[parent[k]], 1);
    atomicMin(&first[parent[k]], k * kPlanThreads + tid);
  }
  __syncthreads();
  // children in need of a page
  bool need[kRows] = {};
  int rank[kRows], rows[kRows], held[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (k * kPlanThreads >= p.new_batch) break;
    const int i = k * kPlanThreads + tid;
    const int length = parent[k] >= 0 ? p.lengths[parent[k]] : 0;
    if (i < p.new_batch) p.lengths_out[i] = length;
    held[k] = held_of(p, length);
    rows[k] = held[k] ? length - static_cast<int>(p.by_page.divide(length)) * p.page_size : 0;
    need[k] = rows[k] != 0 && first[parent[k]] != i;
  }
  const int needs = ranks_of(need, p.new_batch, rank, sums, waves);
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    const int length = p.lengths[b], pages = held_of(p, length);
    const int full = pages ? static_cast<int>(p.by_page.divide(length)) : 0;
    first[b] = 2 * full + (pages != full);
  }
  int given = 0;
  for (int base = 0; base < p.pages; base += kCountChunk) {
    const int here = min(kCountChunk, p.pages - base);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (k * kPlanThreads >= here) break;
      const int i = k * kPlanThreads + tid;
      if (i < here) counts[i] = p.refcounts[base + i];
    }
    __syncthreads();
    // eight entries of the table at a time: one by one, each waits for memory alone
    const int entries = p.batch * p.width;
    for (int e0 = tid; e0 < entries; e0 += 8 * kPlanThreads) {
      int change[8], page[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = e0 + k * kPlanThreads;
        change[k] = 0;
        page[k] = -1;
        if (e >= entries) continue;
        const int b = static_cast<int>(p.by_width.divide(e)), j = e - b * p.width;
        const int full = first[b] >> 1, c = children[b];
        change[k] = j < full ? c - 1 : (j == full && (first[b] & 1) && c == 0 ? -1 : 0);
        if (change[k] != 0) page[k] = p.table[b * p.table_stride + j];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t at = static_cast<uint32_t>(page[k]) - static_cast<uint32_t>(base);
        if (page[k] >= 0 && at < static_cast<uint32_t>(here)) atomicAdd(&counts[at], change[k]);
      }
    }
    __syncthreads();
    bool free[kPer] = {};
    int r[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (k * kPlanThreads >= here) break;
      const int i = k * kPlanThreads + tid;
      free[k] = i < here && counts[i] == 0;
    }
    const int all = ranks_of(free, here, r, sums, waves);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (k * kPlanThreads >= here) break;
      const int i = k * kPlanThreads + tid;
      const bool taken = free[k] && given + r[k] < needs;
      if (taken) fresh[given + r[k]] = base + i;
      if (i < here) p.refcounts_out[base + i] = taken ? 1 : counts[i];
    }
    given += all;
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (k * kPlanThreads >= p.new_batch) break;
    const int i = k * kPlanThreads + tid;
    if (i >= p.new_batch) break;
    p.from[i] = need[k] ? p.table[parent[k] * p.table_stride + held[k] - 1] : -1;
    p.to[i] = need[k] ? (rank[k] < given ? fresh[rank[k]] : -1) : -2;  // -2: the parent's own
    p.used[i] = rows[k];
  }
}

// The copies, and the new rows of the table.
__global__ void __launch_bounds__(kThreads) fork_move(CopyArgs c, PlanArgs p, int row_groups) {
  if (static_cast<int>(blockIdx.x) >= row_groups) {
    copy_items(c, blockIdx.x - row_groups, gridDim.x - row_groups);
    return;
  }
  for (int i = blockIdx.x; i < p.new_batch; i += row_groups) {
    const int parent = p.parents[i];
    const bool any = parent >= 0 && parent < p.batch;
    const int held = any ? held_of(p, p.lengths[parent]) : 0;
    const int to = p.to[i];
    for (int j = threadIdx.x; j < p.width; j += kThreads) {
      int page = -1;
      if (j < held) page = j == held - 1 && to != -2 ? to : p.table[parent * p.table_stride + j];
      p.table_out[i * p.table_out_stride + j] = page;
    }
  }
}

// Each workgroup lists the free pages and the used ones of its run of pages, and counts the used pages of all by itself: with one
// workgroup for all of them, its instructions take 17 us for 8192 pages.  What a page is then: its own place (>= 0), kFree, or
// the place in the list of those that move, as kMoves - place.
constexpr int kFree = -1, kMoves = -2;

__global__ void __launch_bounds__(kPlanThreads) compact_plan(PlanArgs p, int run) {
  __shared__ int waves[kPlanWaves], sums[kPlanWaves], more[kPlanWaves];
  const int tid = threadIdx.x, begin = blockIdx.x * run, end = min(begin + run, p.pages);
  int mine = 0, below = 0;
#pragma unroll 8
  for (int i = tid; i < p.pages; i += kPlanThreads) {
    const int in_use = p.refcounts[i] > 0;
    mine += in_use;
    below += i < begin ? in_use : 0;
  }
  int used, used_before;
  prefix(mine, waves, used);
  prefix(below, more, used_before);
  // of the pages before this run: those that are free below `used`, and used from there on
  int used_low = 0;
  if (begin > used) {
#pragma unroll 8
    for (int i = tid; i < used; i += kPlanThreads) used_low += p.refcounts[i] > 0;
  }
  int low;
  prefix(used_low, waves, low);
  int holes = begin <= used ? begin - used_before : 0, movers = begin > used ? used_before - low : 0;
  for (int base = begin; base < end; base += kPlanThreads) {
    const int i = base + tid;
    const int refs = i < end ? p.refcounts[i] : 0;
    const bool hole = i < end && i < used && refs <= 0, moves = i < end && i >= used && refs > 0;
    const bool flag_hole[1] = {hole}, flag_moves[1] = {moves};
    int at_hole[1], at_move[1];
    const int all_holes = ranks_of(flag_hole, 1, at_hole, sums, waves);
    __syncthreads();
    const int all_moves = ranks_of(flag_moves, 1, at_move, sums, waves);
    __syncthreads();
    if (hole) p.to[holes + at_hole[0]] = i;
    if (moves) p.from[movers + at_move[0]] = i;
    if (i < end) p.used[i] = moves ? kMoves - (movers + at_move[0]) : (refs > 0 ? i : kFree);
    holes += all_holes;
    movers += all_moves;
  }
  if (end == p.pages && tid == 0) {
    *p.count = movers;
    p.count[1] = used;
  }
}

// The copies, the pages' new places and counts, and the rows of the table.
__global__ void __launch_bounds__(kThreads) compact_move(CopyArgs c, PlanArgs p, int row_groups, int page_groups) {
  const auto place = [&](int page) {
    const int x = p.used[page];
    return x <= kMoves ? p.to[kMoves - x] : x;
  };
  int group = blockIdx.x;
  if (group < row_groups) {
    for (int b = group; b < p.batch; b += row_groups) {
      const int held = held_of(p, p.lengths[b]);
      for (int j = threadIdx.x; j < p.width; j += kThreads) {
        const int page = j < held ? p.table[b * p.table_stride + j] : -1;
        p.table_out[b * p.table_out_stride + j] = page >= 0 && page < p.pages ? place(page) : -1;
      }
    }
    return;
  }
  group -= row_groups;
  if (group < page_groups) {
    const int used = p.count[1];
    for (int i = group * kThreads + threadIdx.x; i < p.pages; i += page_groups * kThreads) {
      const int refs = p.refcounts[i], to = place(i);
      p.page_map[i] = to;
      if (to >= 0 && to != i) {
        p.refcounts_out[to] = refs;
        p.refcounts_out[i] = 0;
      } else if (to >= 0 || i >= used) {
        p.refcounts_out[i] = refs;
      }  // else a free page that another moves to
    }
    return;
  }
  copy_items(c, group - page_groups, gridDim.x - row_groups - page_groups);
}

// ------------------------------------------------------------------------------------ host

constexpr int64_t kPlanRuns = 256;  // workgroups of a compaction's plan, at most
constexpr int64_t kMostGroups = 1 << 16;  // a piece for each, as far as that goes (2048 that go on: 55.5 us for 53.6)

int width_of(uintptr_t bits) { return (bits & 15) == 0 ? 16 : ((bits & 3) == 0 ? 4 : ((bits & 1) == 0 ? 2 : 1)); }

asc::Region pages_region(const char* name, const void* data, int64_t pages, int64_t stride, const asc_page_tensor_t& t) {
  const bool any = pages > 0 && t.heads > 0 && t.rows > 0;
  return asc::spanned({name,
                       reinterpret_cast<uintptr_t>(data),
                       {pages, t.heads, t.rows},
                       {pages > 1 ? stride : 0, t.heads > 1 ? t.head_stride : 0, t.rows > 1 ? t.row_stride : 0},
                       any ? t.row_bytes : 0,
                       0,
                       0});
}

// The tensors' checks, and their pieces.  partial: a part of a page's rows may be copied.
int32_t make_copy(const asc_pages_t& a, int64_t moves, bool within, bool partial, const char* what, CopyArgs& c) {
  ASC_REQUIRE(a.n_tensors >= 0 && a.n_tensors <= kTensors, ASC_ERR_INVALID_ARG, "%s: %lld tensors (at most %d)", what,
              static_cast<long long>(a.n_tensors), kTensors);
  c.n_tensors = static_cast<int32_t>(a.n_tensors);
  c.page_size = asc::divisor_of(partial ? static_cast<uint32_t>(a.page_size) : 1);
  int64_t per_move = 0;
  c.from_pages = a.num_pages;
  c.to_pages = within ? a.num_pages : a.to_num_pages;
  for (int i = 0; i < c.n_tensors; ++i) {
    const asc_page_tensor_t& x = a.tensors[i];
    ASC_REQUIRE(x.from && x.to, ASC_ERR_INVALID_ARG, "%s: null tensor", what);
    ASC_REQUIRE(!within || (x.from == x.to && x.from_stride == x.to_stride), ASC_ERR_INVALID_ARG,
                "%s: pages move within a tensor", what);
    ASC_REQUIRE(x.heads >= 1 && x.rows >= 1 && x.row_bytes >= 1 && x.heads < 1 << 20 && x.rows < 1 << 30 &&
                    x.row_bytes < 1 << 30 && x.from_stride >= 0 && x.to_stride >= 0 && x.head_stride >= 0 &&
                    x.row_stride >= 0,
                ASC_ERR_INVALID_ARG, "%s: invalid shape or stride of a tensor", what);
    ASC_REQUIRE(!partial || (x.rows <= a.page_size && a.page_size % x.rows == 0), ASC_ERR_INVALID_ARG,
                "%s: %lld rows of a page of %lld", what, static_cast<long long>(x.rows),
                static_cast<long long>(a.page_size));
    ASC_REQUIRE(!partial || x.rows == a.page_size || x.rows * a.page_size < int64_t{1} << 30, ASC_ERR_UNSUPPORTED,
                "%s: pages too large", what);
    Tensor& t = c.t[i];
    t.from = static_cast<const uint8_t*>(x.from);
    t.to = static_cast<uint8_t*>(x.to);
    t.from_stride = x.from_stride;
    t.to_stride = x.to_stride;
    t.head_stride = x.heads > 1 ? x.head_stride : 0;
    t.row_stride = x.rows > 1 ? x.row_stride : x.row_bytes;
    t.rows = static_cast<int32_t>(x.rows);
    t.row_bytes = static_cast<int32_t>(x.row_bytes);
    const bool heads_outside = t.row_stride == x.row_bytes && (x.heads == 1 || x.head_stride == x.rows * x.row_bytes);
    const bool rows_outside = t.head_stride == x.row_bytes && (x.rows == 1 || x.row_stride == x.heads * x.row_bytes);
    t.bytes = x.heads * x.rows * x.row_bytes;
    t.flat = !partial && (heads_outside || rows_outside);
    const int64_t pieces = t.flat ? asc::ceil_div(t.bytes, kPiece) : x.heads;
    // copy_run numbers a head's bytes, and a step of its threads behind them, in 31 bits
    ASC_REQUIRE(t.bytes < int64_t{1} << 40 && pieces < 1 << 24 &&
                    (t.flat || x.rows * x.row_bytes <= (int64_t{1} << 31) - 2 * kThreads),
                ASC_ERR_UNSUPPORTED, "%s: pages too large", what);
    t.pieces = static_cast<int32_t>(pieces);
    per_move += t.pieces;
    uintptr_t bits = reinterpret_cast<uintptr_t>(x.from) | reinterpret_cast<uintptr_t>(x.to) |
                     static_cast<uintptr_t>(x.from_stride | x.to_stride | x.row_bytes);
    if (!t.flat) bits |= static_cast<uintptr_t>(t.head_stride | t.row_stride);
    t.width = width_of(bits);
    // results lie apart from each other and from what is read, unless they are it
    const asc::Region to = pages_region("a result", x.to, c.to_pages, x.to_stride, x);
    for (int j = 0; j < c.n_tensors; ++j) {
      const asc_page_tensor_t& y = a.tensors[j];
      const asc::Region from = pages_region("a cache", y.from, c.from_pages, y.from_stride, y);
      const bool same = i == j && x.from == x.to && x.from_stride == x.to_stride;
      ASC_REQUIRE(same || !asc::overlap(to, from), ASC_ERR_INVALID_ARG, "%s: 'a result' overlaps 'a cache'", what);
      if (j < i) {
        ASC_REQUIRE(!asc::overlap(to, pages_region("a result", y.to, c.to_pages, y.to_stride, y)), ASC_ERR_INVALID_ARG,
                    "%s: two results overlap", what);
      }
    }
  }
  // the last item plus a grid's step stays below 2^31
  ASC_REQUIRE(moves < int64_t{1} << 30 && moves * per_move < int64_t{1} << 30, ASC_ERR_UNSUPPORTED,
              "%s: more than 2^30 pieces of pages to copy", what);
  c.moves = static_cast<int32_t>(moves);
  c.per_move = asc::divisor_of(per_move > 0 ? static_cast<uint32_t>(per_move) : 1);
  return ASC_OK;
}

int32_t check_apart(const asc::Region& r, const asc_pages_t& a, const CopyArgs& c, bool written, const char* what) {
  for (int i = 0; i < c.n_tensors; ++i) {
    const asc_page_tensor_t& x = a.tensors[i];
    ASC_REQUIRE(!asc::overlap(r, pages_region("a cache", x.to, c.to_pages, x.to_stride, x)) &&
                    (!written || !asc::overlap(r, pages_region("a cache", x.from, c.from_pages, x.from_stride, x))),
                ASC_ERR_INVALID_ARG, "%s: '%s' overlaps '%s'", what, r.name, "a cache");
  }
  return ASC_OK;
}

int64_t items_of(const CopyArgs& c) { return c.n_tensors > 0 ? static_cast<int64_t>(c.moves) * c.per_move.d : 0; }
int64_t groups_of(int64_t items) { return items < kMostGroups ? items : kMostGroups; }

struct Plan {
  CopyArgs c{};
  PlanArgs p{};
};

int64_t fork_workspace(const asc_pages_t& a) { return 16 + 3 * asc::ceil_div(a.new_batch, 4) * 16; }
int64_t compact_workspace(const asc_pages_t& a) { return 16 + 3 * asc::ceil_div(a.num_pages, 4) * 16; }

int32_t make_plan(const asc_pages_t* a, bool fork, const char* what, Plan& plan) {
  ASC_REQUIRE(a, ASC_ERR_INVALID_ARG, "%s: null arguments", what);
  ASC_REQUIRE(a->page_size >= 1 && a->page_size < 1 << 30 && a->num_pages >= 0 && a->num_pages < 1 << 30 &&
                  a->width >= 0 && a->width < 1 << 30 && a->batch >= 0 && a->table_stride >= 0 &&
                  a->table_out_stride >= 0,
              ASC_ERR_INVALID_ARG, "%s: invalid shape", what);
  ASC_REQUIRE(a->width * a->page_size < int64_t{1} << 40 && a->width * a->batch < int64_t{1} << 30, ASC_ERR_UNSUPPORTED,
              "%s: shape too large", what);
  const int64_t rows = fork ? a->new_batch : a->batch;
  ASC_REQUIRE(rows >= 0, ASC_ERR_INVALID_ARG, "%s: invalid shape", what);
  ASC_REQUIRE((!fork && a->batch < 1 << 20) || (a->batch <= kMostSequences && a->new_batch <= kMostSequences),
              ASC_ERR_UNSUPPORTED, "%s: more than %d sequences", what, fork ? kMostSequences : 1 << 20);
  const bool table = a->batch > 0 && a->width > 0, counts = a->num_pages > 0;
  ASC_REQUIRE((!table || a->block_table) && (a->batch == 0 || a->lengths) && (!counts || (a->refcounts && a->refcounts_out)) &&
                  (rows == 0 || a->width == 0 || a->table_out),
              ASC_ERR_INVALID_ARG, "%s: null buffer", what);
  ASC_REQUIRE(fork ? rows == 0 || (a->parents && a->lengths_out) : !counts || a->page_map, ASC_ERR_INVALID_ARG,
              "%s: null buffer", what);
  int32_t rc = make_copy(*a, fork ? a->new_batch : a->num_pages / 2, true, fork, what, plan.c);
  if (rc != ASC_OK) return rc;
  const auto table_rows = [&](const char* name, const int32_t* data, int64_t stride, int64_t n) {
    return asc::region_of(name, asc_rows_t{const_cast<int32_t*>(data), stride, 0, 0}, n, 1, 1, a->width, 4);
  };
  const asc::Region block_table = table_rows("block_table", a->block_table, a->table_stride, a->batch);
  const asc::Region refcounts = asc::region_of("refcounts", a->refcounts, a->num_pages * 4);
  const asc::Region results[] = {
      table_rows("table_out", a->table_out, a->table_out_stride, rows),
      asc::region_of("refcounts_out", a->refcounts_out, a->num_pages * 4),
      fork ? asc::region_of("lengths_out", a->lengths_out, a->new_batch * 4)
           : asc::region_of("page_map", a->page_map, a->num_pages * 4)};
  const asc::Region operands[] = {block_table, refcounts, asc::region_of("lengths", a->lengths, a->batch * 4),
                                  asc::region_of("parents", fork ? a->parents : nullptr, a->new_batch * 4)};
  for (int i = 0; i < 3; ++i) {
    for (const asc::Region& x : operands) {
      const bool in_place = (i == 1 && &x == &operands[1]) || (i == 0 && !fork && &x == &operands[0]);
      ASC_REQUIRE(!asc::overlap(results[i], x) || (in_place && asc::same_place(results[i], x)), ASC_ERR_INVALID_ARG,
                  "%s: '%s' overlaps '%s'", what, results[i].name, x.name);
    }
    for (int j = 0; j < i; ++j) {
      ASC_REQUIRE(!asc::overlap(results[i], results[j]), ASC_ERR_INVALID_ARG, "%s: '%s' overlaps '%s'", what,
                  results[i].name, results[j].name);
    }
    rc = check_apart(results[i], *a, plan.c, true, what);
    if (rc != ASC_OK) return rc;
  }
  for (const asc::Region& x : operands) {
    rc = check_apart(x, *a, plan.c, false, what);
    if (rc != ASC_OK) return rc;
  }
  PlanArgs& p = plan.p;
  p.table = a->block_table;
  p.table_stride = a->table_stride;
  p.lengths = a->lengths;
  p.parents = a->parents;
  p.refcounts = a->refcounts;
  p.table_out = a->table_out;
  p.table_out_stride = a->table_out_stride;
  p.lengths_out = a->lengths_out;
  p.refcounts_out = a->refcounts_out;
  p.page_map = a->page_map;
  p.page_size = static_cast<int32_t>(a->page_size);
  p.pages = static_cast<int32_t>(a->num_pages);
  p.batch = static_cast<int32_t>(a->batch);
  p.new_batch = static_cast<int32_t>(a->new_batch);
  p.width = static_cast<int32_t>(a->width);
  p.by_page = asc::divisor_of(static_cast<uint32_t>(p.page_size));
  p.by_width = asc::divisor_of(p.width > 0 ? static_cast<uint32_t>(p.width) : 1);
  return ASC_OK;
}

int32_t check_workspace(const void* workspace, int64_t bytes, int64_t need, const char* what) {
  ASC_REQUIRE(workspace && bytes >= need && asc::aligned16(workspace), ASC_ERR_INVALID_ARG,
              "%s: the workspace must hold %lld bytes, 16-byte aligned", what, static_cast<long long>(need));
  return ASC_OK;
}

}  // namespace

extern "C" int32_t asc_cache_copy_pages(const asc_pages_t* a, asc_stream_t stream) {
  const char* what = "asc_cache_copy_pages";
  ASC_REQUIRE(a, ASC_ERR_INVALID_ARG, "%s: null arguments", what);
  ASC_REQUIRE(a->pairs >= 0 && a->num_pages >= 0 && a->to_num_pages >= 0, ASC_ERR_INVALID_ARG, "%s: negative shape", what);
  CopyArgs c{};
  int32_t rc = make_copy(*a, a->pairs, false, false, what, c);
  if (rc != ASC_OK || a->pairs == 0 || c.n_tensors == 0) return rc;
  ASC_REQUIRE(a->from_pages && a->to_pages, ASC_ERR_INVALID_ARG, "%s: null buffer", what);
  for (const asc::Region& x : {asc::region_of("from_pages", a->from_pages, a->pairs * 4),
                               asc::region_of("to_pages", a->to_pages, a->pairs * 4)}) {
    rc = check_apart(x, *a, c, false, what);
    if (rc != ASC_OK) return rc;
  }
  c.from = a->from_pages;
  c.to = a->to_pages;
  hipLaunchKernelGGL(page_copy, dim3(static_cast<uint32_t>(groups_of(items_of(c)))), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), c);
  return asc::check_launch(what);
}

extern "C" int64_t asc_cache_fork_workspace(const asc_pages_t* a) {
  Plan plan;
  return make_plan(a, true, "asc_cache_fork_workspace", plan) == ASC_OK ? fork_workspace(*a) : 0;
}

extern "C" int32_t asc_cache_fork(const asc_pages_t* a, void* workspace, int64_t workspace_bytes, asc_stream_t stream) {
  const char* what = "asc_cache_fork";
  Plan plan;
  int32_t rc = make_plan(a, true, what, plan);
  if (rc == ASC_OK) rc = check_workspace(workspace, workspace_bytes, fork_workspace(*a), what);
  if (rc != ASC_OK) return rc;
  const int64_t n = asc::ceil_div(a->new_batch, 4) * 4;
  plan.p.count = static_cast<int32_t*>(workspace);
  plan.p.from = plan.p.count + 4;
  plan.p.to = plan.p.from + n;
  plan.p.used = plan.p.to + n;
  CopyArgs& c = plan.c;
  c.from = plan.p.from;
  c.to = plan.p.to;
  c.used = plan.p.used;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(fork_plan, dim3(1), dim3(kPlanThreads), 0, s, plan.p);
  if (a->new_batch > 0) {
    const int rows = static_cast<int>(a->new_batch < 256 ? a->new_batch : 256);
    const int64_t groups = rows + groups_of(items_of(c));
    hipLaunchKernelGGL(fork_move, dim3(static_cast<uint32_t>(groups)), dim3(kThreads), 0, s, c, plan.p, rows);
  }
  return asc::check_launch(what);
}

extern "C" int64_t asc_cache_compact_workspace(const asc_pages_t* a) {
  Plan plan;
  return make_plan(a, false, "asc_cache_compact_workspace", plan) == ASC_OK ? compact_workspace(*a) : 0;
}

extern "C" int32_t asc_cache_compact(const asc_pages_t* a, void* workspace, int64_t workspace_bytes,
                                     asc_stream_t stream) {
  const char* what = "asc_cache_compact";
  Plan plan;
  int32_t rc = make_plan(a, false, what, plan);
  if (rc == ASC_OK) rc = check_workspace(workspace, workspace_bytes, compact_workspace(*a), what);
  if (rc != ASC_OK) return rc;
  plan.p.count = static_cast<int32_t*>(workspace);
  plan.p.from = plan.p.count + 4;
  plan.p.to = plan.p.from + asc::ceil_div(a->num_pages, 4) * 4;
  plan.p.used = plan.p.to + asc::ceil_div(a->num_pages, 4) * 4;
  CopyArgs& c = plan.c;
  c.count = plan.p.count;
  c.from = plan.p.from;
  c.to = plan.p.to;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->num_pages > 0) {
    const int run = static_cast<int>(asc::ceil_div(asc::ceil_div(a->num_pages, kPlanRuns), kPlanThreads) * kPlanThreads);
    hipLaunchKernelGGL(compact_plan, dim3(static_cast<uint32_t>(asc::ceil_div(a->num_pages, run))), dim3(kPlanThreads), 0, s, plan.p,
                       run);
  }
  const int rows = static_cast<int>(a->batch < 256 ? a->batch : 256);
  const int64_t per_group = asc::ceil_div(a->num_pages, kThreads);
  const int pages = static_cast<int>(per_group < 256 ? per_group : 256);
  const int64_t groups = rows + pages + groups_of(items_of(c));
  if (groups > 0) {
    hipLaunchKernelGGL(compact_move, dim3(static_cast<uint32_t>(groups)), dim3(kThreads), 0, s, c, plan.p, rows, pages);
  }
  return asc::check_launch(what);
}
