// Attention over a cache held in 8 bits (asc_quantized_cache_attention).  The device code is cache8_attn_kernels.h;
// here are the checks, the choice of the kernel and of the split of the keys, and the workspace of the splits.
#include <cmath>
#include <cstdio>

#include "cache8_attn_kernels.h"

namespace {

using asc::c8::AttnArgs;
using asc::c8::E4m3;
using asc::c8::Int8;
using asc::c8::Narrow;
using asc::c8::Wide;

template <int D, class E, class Q>
__global__ void __launch_bounds__(Wide<D>::kWaves * 64, Wide<D>::kWgPerCu) cache8_wide(AttnArgs p) {
  asc::c8::wide_body<D, E, Q>(p);
}
template <int D, class E, class Q>
__global__ void __launch_bounds__(Narrow<D>::kWaves * 64, Narrow<D>::kWgPerCu) cache8_narrow(AttnArgs p) {
  asc::c8::narrow_body<D, E, Q>(p);
}
template <int D, class E>
__global__ void __launch_bounds__(256) cache8_join(AttnArgs p) {
  asc::c8::join_body<D, E>(p);
}

struct Launch {
  AttnArgs p{};
  bool wide = false;
  int64_t blocks = 0;  // 0: nothing to launch
  int64_t rows_all = 0;
};

constexpr int kMaxSplits = 64;
constexpr int kCus = 256;

struct Way {
  int64_t row_blocks, splits;
  double us;
};

// What a kernel takes, in us: `start`, and then the longest of its workgroups' chains of tiles (`chain` for each round of
// `waves` tiles), of what the busiest CU works on (`tile` for each), and of the average CU's work and a part (`last`) of
// a workgroup's chain where sequences of several lengths end one by one.  A split's parts cost `join` and their bytes.
// Fitted to 240 shapes of 4 to 2048 rows, 8 heads, 1 to 40 sequences and 512 to 32768 keys, with 1 to 64 splits in either
// kernel: off by 6 to 19% (root mean square).  The choice from it is 2% slower than the best of each shape on average
// where the caches were read just before, 4% where they come from memory; as many splits as fill the card's slots
// twice: 8% and 13%.  8 sequences of 15000 to 32768 keys get their best (16 splits: 72 us, 4: 80, 64: 95).
struct Cost {
  int rows, slots, waves;  // slots: workgroups that the card holds
  double start, chain, tile, last;
};
constexpr double kJoinUs = 4.5, kPartBytesPerUs = 3e6;
template <int D>
constexpr Cost kNarrowCost{Narrow<D>::kRows, kCus * Narrow<D>::kWgPerCu, Narrow<D>::kWaves, D == 128 ? 7.4 : 6.2,
                           D == 128 ? 1.85 : 1.28, D == 128 ? 0.48 : 0.28, 0.3};
template <int D>
constexpr Cost kWideCost{Wide<D>::kRows, kCus * Wide<D>::kWgPerCu, 1, D == 128 ? 9.2 : 7.2, D == 128 ? 1.75 : 1.03,
                         D == 128 ? 2.0 : 0.77, 0.0};

// The fastest split: more than another only where they save 3%.
Way way_of(const Cost& c, int64_t batch, int64_t heads, int64_t rows, int64_t tiles, int head_dim) {
  Way best{asc::ceil_div(rows, c.rows), 1, INFINITY};
  heads *= batch;
  const int64_t shares = heads * best.row_blocks;
  const double last = batch > 1 ? c.last : 0.0;
  const auto consider = [&](int64_t splits) {
    const int64_t all = shares * splits, per = asc::ceil_div(tiles, splits);
    const double chain = c.chain * static_cast<double>(asc::ceil_div(per, c.waves)), work = c.tile * static_cast<double>(per);
    const double average = work * static_cast<double>(all) / kCus;
    const double busiest = all < kCus ? average : work * static_cast<double>(asc::ceil_div(all, kCus));
    const double chains = chain * static_cast<double>(asc::ceil_div(all, c.slots));
    double us = c.start + std::fmax(std::fmax(chains, busiest), average + last * chain);
    if (splits > 1) us += kJoinUs + static_cast<double>(heads * rows * splits * head_dim * 8) / kPartBytesPerUs;
    if (us < 0.97 * best.us) best = {best.row_blocks, splits, us};
  };
  consider(1);
  if (shares >= 8 * kCus) return best;
  const int64_t most = tiles / 2 < kMaxSplits ? tiles / 2 : kMaxSplits;
  for (int64_t splits = 2, step = 1; splits <= most; splits += step) {  // 2, 3, 4, 6, 8, 12, ...
    if ((splits & (splits - 1)) == 0) step = splits / 2;
    consider(splits);
  }
  for (int64_t fill = kCus; fill <= 2 * kCus; fill += kCus) {  // as many as the CUs hold at a time
    if (fill / shares > 1 && fill / shares <= most) consider(fill / shares);
  }
  return best;
}

void plan(Launch& L, const asc_cache8_t& a) {
  AttnArgs& p = L.p;
  const bool small = a.head_dim == 64;
  const int64_t heads = a.batch * a.kv_heads, tiles = asc::ceil_div(p.c.capacity, asc::fa::BKV);
  const Way narrow = way_of(small ? kNarrowCost<64> : kNarrowCost<128>, a.batch, a.kv_heads, p.rows, tiles, a.head_dim);
  const Way wide = way_of(small ? kWideCost<64> : kWideCost<128>, a.batch, a.kv_heads, p.rows, tiles, a.head_dim);
  L.wide = p.rows > Narrow<128>::kRows && wide.us < 0.95 * narrow.us;
  const Way& w = L.wide ? wide : narrow;
  p.row_blocks = static_cast<int>(w.row_blocks);
  p.splits = static_cast<int>(w.splits);
  p.by_n = asc::divisor_of(static_cast<uint32_t>(p.c.n));
  p.by_heads = asc::divisor_of(static_cast<uint32_t>(p.c.kv_heads));
  p.by_splits = asc::divisor_of(static_cast<uint32_t>(p.splits));
  p.lanes = p.causal && p.row_blocks >= 2 * p.group ? p.group : 1;
  p.per_lane = asc::ceil_div(p.row_blocks, p.lanes);
  p.by_lanes = asc::divisor_of(static_cast<uint32_t>(p.lanes));
  p.by_slots = asc::divisor_of(static_cast<uint32_t>(p.lanes * p.per_lane));
  p.units = static_cast<uint32_t>(heads * p.splits);
  L.rows_all = heads * p.rows;
  p.join_groups = small ? asc::kv::JoinLanes<64>::groups_of(L.rows_all, p.splits)
                        : asc::kv::JoinLanes<128>::groups_of(L.rows_all, p.splits);
  L.blocks = asc::ceil_div(p.units, 8) * 8 * p.lanes * p.per_lane;
}

// Bytes of the parts: their values and statistics.
int64_t workspace_of(const Launch& L, int head_dim) {
  if (L.blocks == 0 || L.p.splits == 1) return 0;
  return L.p.units * static_cast<int64_t>(L.p.rows) * (head_dim + 4) * static_cast<int64_t>(sizeof(float));
}

int32_t make(const asc_cache8_t* a, const char* what, Launch& L) {
  AttnArgs& p = L.p;
  int32_t rc = asc::c8::make_cache(a, what, p.c);
  if (rc != ASC_OK) return rc;
  ASC_REQUIRE(a->dtype == ASC_DT_FLOAT16 || a->dtype == ASC_DT_BFLOAT16, ASC_ERR_UNSUPPORTED,
              "%s: dtype %d not supported (float16, bfloat16)", what, a->dtype);
  ASC_REQUIRE(a->q_heads >= 0 && (a->q_heads == 0 || (a->kv_heads > 0 && a->q_heads % a->kv_heads == 0)),
              ASC_ERR_INVALID_ARG, "%s: %lld query heads cannot share %lld key / value heads", what,
              static_cast<long long>(a->q_heads), static_cast<long long>(a->kv_heads));
  ASC_REQUIRE(a->sm_scale > 0.f && a->sm_scale < INFINITY, ASC_ERR_INVALID_ARG,
              "%s: sm_scale must be positive and finite", what);
  if (a->batch == 0 || a->q_heads == 0 || a->n == 0) return ASC_OK;
  ASC_REQUIRE(a->q_heads < 1 << 20 && a->batch * a->q_heads < 1 << 20 && a->q_heads / a->kv_heads * a->n < 1 << 30,
              ASC_ERR_UNSUPPORTED, "%s: shape too large", what);
  ASC_REQUIRE(a->q.data && a->o.data, ASC_ERR_INVALID_ARG, "%s: null buffer", what);
  ASC_REQUIRE(asc::c8::row_operand(a->q, 2) && asc::c8::row_operand(a->o, 2), ASC_ERR_ALIGNMENT,
              "%s: q and o must be 16-byte aligned, with strides that are multiples of 8", what);
  // offsets within a group of 16 rows fit 32 bits
  ASC_REQUIRE(p.c.ks.row < 1 << 22 && p.c.vs.row < 1 << 22, ASC_ERR_UNSUPPORTED, "%s: rows of the cache lie 64 MiB apart",
              what);
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
  p.group = static_cast<int32_t>(a->q_heads / a->kv_heads);
  p.rows = p.group * p.c.n;
  p.causal = a->causal != 0;
  p.scale_mantissa = static_cast<float>(std::frexp(a->sm_scale * 1.4426950408889634, &p.scale_power));
  plan(L, *a);
  ASC_REQUIRE(L.blocks < int64_t{1} << 22, ASC_ERR_UNSUPPORTED, "%s: %lld workgroups exceed the launch grid limit", what,
              static_cast<long long>(L.blocks));
  return ASC_OK;
}

int32_t check_places(const asc_cache8_t& a, const char* what) {
  asc::Region operands[asc::c8::kRegions + 1];
  asc::c8::regions_of(a, reinterpret_cast<asc::Region(&)[asc::c8::kRegions]>(operands));
  operands[asc::c8::kRegions] = asc::region_of("q", a.q, a.batch, a.q_heads, a.n, a.head_dim, 2);
  const asc::Region results[] = {asc::region_of("o", a.o, a.batch, a.q_heads, a.n, a.head_dim, 2),
                                 asc::region_of("lse", a.lse, a.batch * a.q_heads * a.n * static_cast<int64_t>(sizeof(float)))};
  for (const asc::Region& r : results) {
    for (const asc::Region& x : operands) {
      ASC_REQUIRE(!asc::overlap(r, x), ASC_ERR_INVALID_ARG, "%s: '%s' overlaps '%s'", what, r.name, x.name);
    }
  }
  ASC_REQUIRE(!asc::overlap(results[0], results[1]), ASC_ERR_INVALID_ARG, "%s: '%s' overlaps '%s'", what, "o", "lse");
  return ASC_OK;
}

template <int D, class E, class Q>
void launch(const Launch& L, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(L.blocks));
  if (L.wide) {
    hipLaunchKernelGGL((cache8_wide<D, E, Q>), grid, dim3(Wide<D>::kWaves * 64), 0, stream, L.p);
  } else {
    hipLaunchKernelGGL((cache8_narrow<D, E, Q>), grid, dim3(Narrow<D>::kWaves * 64), 0, stream, L.p);
  }
  if (L.p.splits == 1) return;
  const int64_t threads = L.rows_all * (D / 8) * L.p.join_groups;
  hipLaunchKernelGGL((cache8_join<D, E>), dim3(static_cast<uint32_t>(asc::ceil_div(threads, 256))), dim3(256), 0, stream, L.p);
}

template <int D, class E>
void launch_format(const Launch& L, int32_t cache_dtype, hipStream_t stream) {
  cache_dtype == ASC_DT_INT8 ? launch<D, E, Int8>(L, stream) : launch<D, E, E4m3>(L, stream);
}

}  // namespace

extern "C" int64_t asc_quantized_cache_attention_workspace(const asc_cache8_t* a) {
  Launch L;
  return make(a, "asc_quantized_cache_attention_workspace", L) == ASC_OK ? workspace_of(L, a->head_dim) : 0;
}

extern "C" int32_t asc_quantized_cache_attention(const asc_cache8_t* a, void* workspace, int64_t workspace_bytes,
                                                 asc_stream_t stream) {
  const char* what = "asc_quantized_cache_attention";
  Launch L;
  int32_t rc = make(a, what, L);
  if (rc != ASC_OK || L.blocks == 0) return rc;
  const int64_t need = workspace_of(L, a->head_dim);
  ASC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && asc::aligned16(workspace)), ASC_ERR_INVALID_ARG,
              "%s: the workspace must hold %lld bytes, 16-byte aligned", what, static_cast<long long>(need));
  rc = check_places(*a, what);
  if (rc != ASC_OK) return rc;
  if (need != 0) {
    L.p.part_o = static_cast<float*>(workspace);
    L.p.part_ml = L.p.part_o + L.p.units * static_cast<int64_t>(L.p.rows) * a->head_dim;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f16 = a->dtype == ASC_DT_FLOAT16;
  if (a->head_dim == 64) {
    f16 ? launch_format<64, asc::fa::F16>(L, a->cache_dtype, s) : launch_format<64, asc::fa::Bf16>(L, a->cache_dtype, s);
  } else {
    f16 ? launch_format<128, asc::fa::F16>(L, a->cache_dtype, s) : launch_format<128, asc::fa::Bf16>(L, a->cache_dtype, s);
  }
  return asc::check_launch(what);
}

extern "C" int32_t asc_quantized_cache_attention_plan(const asc_cache8_t* a, asc_attention_plan_t* plan) {
  ASC_REQUIRE(plan, ASC_ERR_INVALID_ARG, "asc_quantized_cache_attention_plan: null plan");
  *plan = asc_attention_plan_t{};
  Launch L;
  const int32_t rc = make(a, "asc_quantized_cache_attention_plan", L);
  if (rc != ASC_OK || L.blocks == 0) return rc;
  snprintf(plan->kernel, sizeof(plan->kernel), "%s", L.wide ? "cache8_wide" : "cache8_narrow");
  plan->row_blocks = L.p.row_blocks;
  plan->splits = L.p.splits;
  return ASC_OK;
}
