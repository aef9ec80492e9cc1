// Attention over cached keys: asc_cross_attention_fwd (an encoder's states, of another length than
// the queries) and asc_tree_attention (a cache in pages or in one piece, and drafted tokens behind
// it).  The device code is kv_attn_kernels.h; here are the checks, the choice of the kernel and of
// the split of the keys, and the workspace of the splits.
#include <cmath>
#include <cstdio>

#include "kv_attn_host.h"
#include "kv_attn_kernels.h"

namespace {

using asc::kv::KvArgs;
using asc::kv::Narrow;
using asc::kv::Wide;

// Each kernel for a head_dim, an element type, and with (tree) or without pages and drafted keys.
template <int D, class E, bool kTree>
__global__ void __launch_bounds__(Wide<D>::kWaves * 64, Wide<D>::kWgPerCu) kv_wide(KvArgs p) {
  asc::kv::kv_wide_body<D, E, kTree>(p);
}
template <int D, class E, bool kTree>
__global__ void __launch_bounds__(Narrow<D>::kWaves * 64, Narrow<D>::kWgPerCu) kv_narrow(KvArgs p) {
  asc::kv::kv_narrow_body<D, E, kTree>(p);
}
template <int D, class E>
__global__ void __launch_bounds__(256) kv_join(KvArgs p) {
  asc::kv::kv_join_body<D, E>(p);
}

struct Launch {
  KvArgs p{};
  bool wide = false;
  int64_t blocks = 0;  // 0: nothing to launch
  int64_t rows_all = 0;
};

constexpr int kMaxSplits = 64;
constexpr int64_t kCus = 256;

// One way to launch.
struct Way {
  int64_t row_blocks, splits;
  double us;
};

// A way's split of the keys, where its workgroups are too few to fill the chip, and its time: rounds
// of workgroups, each with its start and end and its longest chain of tiles, and the join.
Way way_of(int64_t heads, int64_t row_blocks, int64_t tiles, int64_t slots, int fill, int64_t least, int waves,
           double start, double tile) {
  Way w{row_blocks, 1, 0.0};
  const int64_t shares = heads * row_blocks;
  if (shares < slots) w.splits = fill * slots / shares;
  if (w.splits > tiles / least) w.splits = tiles / least;
  if (w.splits > kMaxSplits) w.splits = kMaxSplits;
  if (w.splits < 1) w.splits = 1;
  const int64_t chain = asc::ceil_div(asc::ceil_div(tiles, w.splits), waves);
  w.us = static_cast<double>(asc::ceil_div(shares * w.splits, slots)) * (start + tile * static_cast<double>(chain)) +
         (w.splits > 1 ? 3.5 : 0.0);
  return w;
}

// kv_narrow for up to 32 rows; above that, kv_narrow (whose four waves share a tile's time, but
// which reads the keys once per 32 rows) or kv_wide, whichever the times above say is clearly shorter.
// They were taken from kernels of 1 to 4 rounds.  kv_wide, kv_narrow (us): 128 heads, 64 rows, 500
// keys, head_dim 64: 13.7, 7.0; 64 heads, 333 rows, 777 keys, head_dim 64: 24.0, 18.1; 8 heads, 333
// rows, 777 keys, head_dim 128: 22.4, 13.0; 128 heads, 128 rows, 500 keys: 22.3, 19.9; 32 heads, 200
// rows, 2000 keys: 31.8, 32.0; 64 heads, 48 rows, 4000 keys: 32.7, 36.2.
// kv_wide's keys are split to fill the chip once (twice: 70 against 60 us for 8 sequences of 4096
// down to 1024 keys, 64 drafted tokens, 32 / 8 heads), kv_narrow's, which HBM bounds, twice.
void plan(Launch& L, const asc_attention_t& a) {
  KvArgs& p = L.p;
  const bool small = a.head_dim == 64;
  const int64_t heads = a.batch * a.kv_heads, slots = small ? 2 * kCus : kCus;
  const int64_t tiles = asc::ceil_div(p.capacity, asc::fa::BKV) + (p.k_draft ? asc::ceil_div(p.n_q, asc::fa::BKV) : 0);
  const Way narrow = way_of(heads, asc::ceil_div(p.rows, Narrow<64>::kRows), tiles, slots, 2, 8, Narrow<64>::kWaves,
                            small ? 4.5 : 5.5, small ? 1.2 : 2.0);
  const Way wide = way_of(heads, asc::ceil_div(p.rows, small ? Wide<64>::kRows : Wide<128>::kRows), tiles, slots, 1, 4,
                          1, small ? 8.0 : 9.0, small ? 1.6 : 2.2);
  L.wide = p.rows > Narrow<64>::kRows && narrow.us > 0.9 * wide.us;
  const Way& w = L.wide ? wide : narrow;
  p.row_blocks = static_cast<int>(w.row_blocks);
  p.splits = static_cast<int>(w.splits);
  p.units = static_cast<uint32_t>(heads * p.splits);
  L.rows_all = heads * p.rows;
  p.join_groups = small ? asc::kv::JoinLanes<64>::groups_of(L.rows_all, p.splits)
                        : asc::kv::JoinLanes<128>::groups_of(L.rows_all, p.splits);
  L.blocks = asc::ceil_div(p.units, 8) * 8 * p.row_blocks;
}

// Bytes of the parts: their values, statistics and flags.
int64_t workspace_of(const Launch& L, int head_dim) {
  if (L.blocks == 0 || L.p.splits == 1) return 0;
  return L.p.units * (static_cast<int64_t>(L.p.rows) * (head_dim + 2) + 1) * static_cast<int64_t>(sizeof(float));
}

int32_t make(const asc_attention_t* a, bool tree, const char* what, Launch& L) {
  int32_t rc = asc::kv::check_shape(a, what);
  if (rc != ASC_OK) return rc;
  if (a->batch == 0 || a->q_heads == 0 || a->q_len == 0) return ASC_OK;
  ASC_REQUIRE(asc::kv::row_operand(a->q) && asc::kv::row_operand(a->o), ASC_ERR_ALIGNMENT,
              "%s: q and o must be 16-byte aligned, with strides that are multiples of 8", what);
  ASC_REQUIRE(a->q.data && a->o.data, ASC_ERR_INVALID_ARG, "%s: null buffer", what);
  KvArgs& p = L.p;
  p.q = static_cast<const uint16_t*>(a->q.data);
  p.o = static_cast<uint16_t*>(a->o.data);
  p.lse = a->lse;
  p.q_batch = a->q.batch_stride;
  p.q_head = a->q.head_stride;
  p.q_seq = a->q.seq_stride;
  p.o_batch = a->o.batch_stride;
  p.o_head = a->o.head_stride;
  p.o_seq = a->o.seq_stride;
  p.batch = static_cast<int32_t>(a->batch);
  p.kv_heads = static_cast<int32_t>(a->kv_heads);
  p.group = static_cast<int32_t>(a->q_heads / a->kv_heads);
  p.n_q = static_cast<int32_t>(a->q_len);
  p.rows = p.group * p.n_q;
  p.capacity = static_cast<int32_t>(a->kv_len);
  p.lengths = a->kv_lengths;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  const bool paged = tree && a->block_table != nullptr;
  if (a->kv_len > 0) {
    ASC_REQUIRE(a->k.data && a->v.data, ASC_ERR_INVALID_ARG, "%s: null buffer", what);
    p.k = static_cast<const uint8_t*>(a->k.data);
    p.v = static_cast<const uint8_t*>(a->v.data);
    const int64_t batch = paged ? a->num_pages : a->batch, rows = paged ? a->page_size : a->kv_len;
    if (paged) {
      ASC_REQUIRE(a->page_size >= 1 && a->page_size < 1 << 30 && a->num_pages >= 1 &&
                      a->num_pages < int64_t{1} << 31 && a->table_stride >= 0,
                  ASC_ERR_INVALID_ARG, "%s: invalid pages (%d rows, %lld pages)", what, a->page_size,
                  static_cast<long long>(a->num_pages));
      p.table = a->block_table;
      p.table_stride = a->table_stride;
      p.num_pages = static_cast<uint32_t>(a->num_pages);
      p.page_size = static_cast<uint32_t>(a->page_size);
      // key / page_size = key * magic >> (31 + shift) for keys below 2^31, 2^shift >= page_size
      while ((uint32_t{1} << p.page_shift) < p.page_size) ++p.page_shift;
      p.page_magic = static_cast<uint32_t>(((uint64_t{1} << (31 + p.page_shift)) + p.page_size - 1) / p.page_size);
    }
    rc = asc::kv::strides_of(a->k, batch, a->kv_heads, rows, a->head_dim, what, p.ks);
    if (rc == ASC_OK) rc = asc::kv::strides_of(a->v, batch, a->kv_heads, rows, a->head_dim, what, p.vs);
    if (rc != ASC_OK) return rc;
  }
  if (tree) {
    ASC_REQUIRE(a->k_draft.data && a->v_draft.data, ASC_ERR_INVALID_ARG, "%s: null drafted keys or values", what);
    p.k_draft = static_cast<const uint8_t*>(a->k_draft.data);
    p.v_draft = static_cast<const uint8_t*>(a->v_draft.data);
    rc = asc::kv::strides_of(a->k_draft, a->batch, a->kv_heads, a->q_len, a->head_dim, what, p.kds);
    if (rc == ASC_OK) rc = asc::kv::strides_of(a->v_draft, a->batch, a->kv_heads, a->q_len, a->head_dim, what, p.vds);
    if (rc != ASC_OK) return rc;
    p.draft_lengths = a->draft_lengths;
    p.mask = a->tree_mask;
    p.mask_batch = a->mask_batch_stride;
    p.mask_row = a->mask_row_stride;
    p.mask_words = a->q_len % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.mask) | p.mask_batch | p.mask_row) & 3) == 0;
  }
  plan(L, *a);
  ASC_REQUIRE(L.blocks < int64_t{1} << 22, ASC_ERR_UNSUPPORTED,
              "%s: %lld workgroups exceed the launch grid limit", what, static_cast<long long>(L.blocks));
  return ASC_OK;
}

int32_t check_places(const asc_attention_t& a, bool tree, const char* what) {
  const bool paged = tree && a.block_table != nullptr && a.kv_len > 0;
  const auto rows = [&](const char* name, const asc_rows_t& r, int64_t batch, int64_t heads, int64_t length) {
    return asc::region_of(name, r, batch, heads, length, a.head_dim, 2);
  };
  const int64_t kv_batch = paged ? a.num_pages : a.batch, kv_rows = paged ? a.page_size : a.kv_len;
  const asc_rows_t none{};
  const asc_rows_t table{const_cast<int32_t*>(paged ? a.block_table : nullptr), a.table_stride, 0, 0};
  const asc_rows_t mask{const_cast<uint8_t*>(tree ? a.tree_mask : nullptr), a.mask_batch_stride, 0, a.mask_row_stride};
  const int64_t lengths = a.batch * static_cast<int64_t>(sizeof(int32_t));
  const asc::Region results[] = {
      rows("o", a.o, a.batch, a.q_heads, a.q_len),
      asc::region_of("lse", a.lse, a.batch * a.q_heads * a.q_len * static_cast<int64_t>(sizeof(float)))};
  const asc::Region operands[] = {
      rows("q", a.q, a.batch, a.q_heads, a.q_len),
      rows("k", a.k, kv_batch, a.kv_heads, kv_rows),
      rows("v", a.v, kv_batch, a.kv_heads, kv_rows),
      rows("k_draft", tree ? a.k_draft : none, a.batch, a.kv_heads, a.q_len),
      rows("v_draft", tree ? a.v_draft : none, a.batch, a.kv_heads, a.q_len),
      asc::region_of("kv_lengths", a.kv_lengths, lengths),
      asc::region_of("draft_lengths", tree ? a.draft_lengths : nullptr, lengths),
      asc::region_of("block_table", table, a.batch, 1, 1, paged ? asc::ceil_div(a.kv_len, a.page_size) : 0,
                     sizeof(int32_t)),
      asc::region_of("tree_mask", mask, a.batch, 1, a.q_len, a.q_len, 1)};
  return asc::kv::check_places(what, results, operands);
}

template <int D, class E>
void launch(const Launch& L, bool tree, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(L.blocks));
  if (L.wide) {
    hipLaunchKernelGGL((tree ? kv_wide<D, E, true> : kv_wide<D, E, false>), grid, dim3(Wide<D>::kWaves * 64), 0, stream,
                       L.p);
  } else {
    hipLaunchKernelGGL((tree ? kv_narrow<D, E, true> : kv_narrow<D, E, false>), grid, dim3(Narrow<D>::kWaves * 64), 0,
                       stream, L.p);
  }
  if (L.p.splits == 1) return;
  const int64_t threads = L.rows_all * (D / 8) * L.p.join_groups;
  hipLaunchKernelGGL((kv_join<D, E>), dim3(static_cast<uint32_t>(asc::ceil_div(threads, 256))), dim3(256), 0, stream,
                     L.p);
}

int32_t run(const asc_attention_t* a, bool tree, const char* what, void* workspace, int64_t workspace_bytes,
            asc_stream_t stream) {
  Launch L;
  int32_t rc = make(a, tree, what, L);
  if (rc != ASC_OK || L.blocks == 0) return rc;
  const int64_t need = workspace_of(L, a->head_dim);
  ASC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && asc::aligned16(workspace)), ASC_ERR_INVALID_ARG,
              "%s: the workspace must hold %lld bytes, 16-byte aligned", what, static_cast<long long>(need));
  rc = check_places(*a, tree, what);
  if (rc != ASC_OK) return rc;
  if (need != 0) {
    L.p.part_o = static_cast<float*>(workspace);
    L.p.part_ml = L.p.part_o + L.p.units * static_cast<int64_t>(L.p.rows) * a->head_dim;
    L.p.infinite = reinterpret_cast<int32_t*>(L.p.part_ml + L.p.units * static_cast<int64_t>(L.p.rows) * 2);
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f16 = a->dtype == ASC_DT_FLOAT16;
  if (a->head_dim == 64) {
    f16 ? launch<64, asc::fa::F16>(L, tree, s) : launch<64, asc::fa::Bf16>(L, tree, s);
  } else {
    f16 ? launch<128, asc::fa::F16>(L, tree, s) : launch<128, asc::fa::Bf16>(L, tree, s);
  }
  return asc::check_launch(what);
}

int64_t workspace(const asc_attention_t* a, bool tree, const char* what) {
  Launch L;
  return make(a, tree, what, L) == ASC_OK ? workspace_of(L, a->head_dim) : 0;
}

}  // namespace

namespace asc {
namespace kv {

bool row_operand(const asc_rows_t& r) {
  return aligned16(r.data) && ((r.batch_stride | r.head_stride | r.seq_stride) & 7) == 0;
}

int32_t strides_of(const asc_rows_t& r, int64_t batch, int64_t heads, int64_t rows, int head_dim, const char* what,
                   Strides& s) {
  ASC_REQUIRE(((r.batch_stride | r.head_stride | r.seq_stride) & 7) == 0 && asc::aligned16(r.data), ASC_ERR_ALIGNMENT,
              "%s: keys and values must be 16-byte aligned, with strides that are multiples of 8", what);
  ASC_REQUIRE(r.batch_stride >= 0 && r.head_stride >= 0 && r.seq_stride >= 0, ASC_ERR_INVALID_ARG,
              "%s: negative stride", what);
  // the place of a row in 32 bits of 16 bytes; the last value marks none.  Each term is checked
  // before they are added: none overflows 64 bits
  constexpr int64_t limit = (int64_t{1} << 32) - 64;
  const auto term = [](int64_t n, int64_t stride) {
    return n <= 1 || stride == 0 ? 0 : (stride / 8 > limit / (n - 1) ? limit : (n - 1) * (stride / 8));
  };
  ASC_REQUIRE(term(batch, r.batch_stride) + term(heads, r.head_stride) + term(rows, r.seq_stride) + head_dim / 8 <= limit,
              ASC_ERR_UNSUPPORTED, "%s: keys and values span more than 64 GiB", what);
  // a dimension of one element is not stepped over, whatever its stride
  s.batch = batch > 1 ? static_cast<uint32_t>(r.batch_stride / 8) : 0;
  s.head = heads > 1 ? static_cast<uint32_t>(r.head_stride / 8) : 0;
  s.seq = rows > 1 ? static_cast<uint32_t>(r.seq_stride / 8) : 0;
  return ASC_OK;
}

int32_t check_shape(const asc_attention_t* a, const char* what) {
  ASC_REQUIRE(a, ASC_ERR_INVALID_ARG, "%s: null arguments", what);
  ASC_REQUIRE(a->dtype == ASC_DT_FLOAT16 || a->dtype == ASC_DT_BFLOAT16, ASC_ERR_UNSUPPORTED,
              "%s: dtype %d not supported (float16, bfloat16)", what, a->dtype);
  ASC_REQUIRE(a->head_dim == 64 || a->head_dim == 128, ASC_ERR_UNSUPPORTED, "%s: head_dim %d not supported (64, 128)",
              what, a->head_dim);
  ASC_REQUIRE(a->batch >= 0 && a->q_heads >= 0 && a->kv_heads >= 0 && a->q_len >= 0 && a->kv_len >= 0,
              ASC_ERR_INVALID_ARG, "%s: negative shape", what);
  ASC_REQUIRE(a->q_heads == 0 || (a->kv_heads > 0 && a->q_heads % a->kv_heads == 0), ASC_ERR_INVALID_ARG,
              "%s: %lld query heads cannot share %lld key / value heads", what, static_cast<long long>(a->q_heads),
              static_cast<long long>(a->kv_heads));
  ASC_REQUIRE(a->sm_scale > 0.f && a->sm_scale < INFINITY, ASC_ERR_INVALID_ARG,
              "%s: sm_scale must be positive and finite", what);
  // rows of one key / value head, keys of one sequence and workgroups stay below 2^30, 2^30 and 2^22
  ASC_REQUIRE(a->batch < 1 << 20 && a->q_heads < 1 << 20 && a->q_len < 1 << 30 && a->kv_len < 1 << 30 &&
                  a->batch * a->q_heads < 1 << 20 &&
                  (a->kv_heads == 0 || a->q_heads / a->kv_heads * a->q_len < 1 << 30),
              ASC_ERR_UNSUPPORTED, "%s: shape too large", what);
  return ASC_OK;
}

}  // namespace kv
}  // namespace asc

extern "C" int64_t asc_cross_attention_fwd_workspace(const asc_attention_t* args) {
  return workspace(args, false, "asc_cross_attention_fwd_workspace");
}
extern "C" int32_t asc_cross_attention_fwd(const asc_attention_t* args, void* ws, int64_t ws_bytes,
                                           asc_stream_t stream) {
  return run(args, false, "asc_cross_attention_fwd", ws, ws_bytes, stream);
}
extern "C" int64_t asc_tree_attention_workspace(const asc_attention_t* args) {
  return workspace(args, true, "asc_tree_attention_workspace");
}
extern "C" int32_t asc_tree_attention(const asc_attention_t* args, void* ws, int64_t ws_bytes, asc_stream_t stream) {
  return run(args, true, "asc_tree_attention", ws, ws_bytes, stream);
}
extern "C" int32_t asc_attention_plan(const asc_attention_t* args, int32_t tree, asc_attention_plan_t* plan) {
  ASC_REQUIRE(plan, ASC_ERR_INVALID_ARG, "asc_attention_plan: null plan");
  *plan = asc_attention_plan_t{};
  Launch L;
  const int32_t rc = make(args, tree != 0, "asc_attention_plan", L);
  if (rc != ASC_OK || L.blocks == 0) return rc;
  snprintf(plan->kernel, sizeof(plan->kernel), "%s", L.wide ? "kv_wide" : "kv_narrow");
  plan->row_blocks = L.p.row_blocks;
  plan->splits = L.p.splits;
  return ASC_OK;
}
