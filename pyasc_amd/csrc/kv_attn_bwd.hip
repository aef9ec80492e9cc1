// asc_cross_attention_bwd: the checks, the splits, the workspace and the launches of the gradients in
// kv_attn_bwd_kernels.h.
#include "kv_attn_bwd_kernels.h"
#include "kv_attn_host.h"

namespace {

using asc::kv::GradArgs;
using asc::kv::GradKv;
using asc::kv::GradQ;

template <int D, class E>
__global__ void __launch_bounds__(GradQ<D>::kWaves * 64, GradQ<D>::kWgPerCu) grad_q(GradArgs p) {
  asc::kv::grad_q_body<D, E>(p);
}
template <int D, class E, bool kPacked>
__global__ void __launch_bounds__(GradKv<D>::kWaves * 64, GradKv<D>::kWgPerCu) grad_kv(GradArgs p) {
  asc::kv::grad_kv_body<D, E, kPacked>(p);
}
template <int D, class E>
__global__ void __launch_bounds__(256) join_grad(GradArgs p) {
  asc::kv::join_grad_body<D, E>(p);
}

constexpr int kMaxSplits = 32;
constexpr int64_t kSlots = 512;  // workgroups of four waves that fill 256 CUs

struct Launch {
  GradArgs p{};
  bool keys = false;  // there is something to sum over
  int64_t q_rows = 0, kv_rows = 0;  // of all heads
  int64_t q_grid = 0, kv_grid = 0;
  int64_t values = 0, parts_q = 0, parts_kv = 0;  // floats of the workspace
};

int32_t splits_of(int64_t shares, int64_t slots, int64_t tiles, int64_t least) {
  int64_t n = shares >= slots || shares == 0 ? 1 : slots / shares;
  if (n > tiles / least) n = tiles / least;
  if (n > kMaxSplits) n = kMaxSplits;
  return n < 1 ? 1 : static_cast<int32_t>(n);
}

void plan(Launch& L, const asc_attention_t& a) {
  GradArgs& p = L.p;
  const bool small = a.head_dim == 64;
  const int64_t heads = a.batch * a.kv_heads;
  L.q_rows = heads * p.rows;
  L.kv_rows = heads * a.kv_len;
  p.q_blocks = static_cast<int32_t>(asc::ceil_div(p.rows, small ? GradQ<64>::kRows : GradQ<128>::kRows));
  p.kv_blocks = static_cast<int32_t>(asc::ceil_div(a.kv_len, GradKv<64>::kKeys));
  p.q_splits = splits_of(heads * p.q_blocks, small ? kSlots : kSlots / 2, asc::ceil_div(a.kv_len, GradQ<64>::kKeys), 4);
  // at least 8 tiles of rows in a part (4: 80.6 against 75.8 us for 8 / 2 heads of 128, 300 queries, 2000
  // keys, forward and gradients; 55.5 against 50.0 for 2 x 16 / 4 heads of 64, 64 queries, 4000 keys: the
  // parts' bytes outweigh the shorter chains)
  p.kv_splits = splits_of(heads * p.kv_blocks, kSlots,
                          p.n_q < GradKv<64>::kRows ? asc::ceil_div(p.rows, GradKv<64>::kRows)
                                                    : p.group * asc::ceil_div(p.n_q, GradKv<64>::kRows),
                          8);
  p.q_units = static_cast<uint32_t>(heads * p.q_splits);
  p.kv_units = static_cast<uint32_t>(heads * p.kv_splits);
  L.q_grid = asc::ceil_div(p.q_units, 8) * 8 * p.q_blocks;
  L.kv_grid = asc::ceil_div(p.kv_units, 8) * 8 * p.kv_blocks;
  L.values = L.q_rows;
  L.parts_q = p.q_splits > 1 ? L.q_rows * p.q_splits * a.head_dim : 0;
  L.parts_kv = p.kv_splits > 1 ? L.kv_rows * p.kv_splits * a.head_dim : 0;
  const auto groups = [&](int64_t n, int splits) {
    return small ? asc::kv::JoinLanes<64>::groups_of(n, splits) : asc::kv::JoinLanes<128>::groups_of(n, splits);
  };
  p.q_join_groups = groups(L.q_rows, p.q_splits);
  p.kv_join_groups = groups(L.kv_rows, p.kv_splits);
  const int64_t lanes = a.head_dim / 8;
  if (L.parts_q > 0) p.q_join = static_cast<uint32_t>(asc::ceil_div(L.q_rows * lanes * p.q_join_groups, 256));
  if (L.parts_kv > 0) p.kv_join = static_cast<uint32_t>(asc::ceil_div(L.kv_rows * lanes * p.kv_join_groups, 256));
}

// Floats of a workspace region, so that the next one is 16-byte aligned.
int64_t region(int64_t n) { return (n + 3) / 4 * 4; }

int64_t workspace_of(const Launch& L) {
  if (!L.keys) return 0;
  return (2 * region(L.values) + region(L.parts_q) + 2 * region(L.parts_kv)) * static_cast<int64_t>(sizeof(float));
}

int32_t make(const asc_attention_t* a, const char* what, Launch& L) {
  int32_t rc = asc::kv::check_shape(a, what);
  if (rc != ASC_OK) return rc;
  // lse / sm_scale has to stay finite: the logarithm of a count of keys is below 2^5
  ASC_REQUIRE(a->sm_scale >= 0x1p-100f, ASC_ERR_UNSUPPORTED, "%s: sm_scale %g is below 2^-100", what, a->sm_scale);
  const bool queries = a->batch > 0 && a->q_heads > 0 && a->q_len > 0;
  const bool keys = a->batch > 0 && a->kv_heads > 0 && a->kv_len > 0;
  GradArgs& p = L.p;
  const asc_rows_t* rows[] = {&a->q, &a->o, &a->d_o, &a->dq, &a->k, &a->v, &a->dk, &a->dv};
  for (int i = 0; i < 8; ++i) {
    if (!(i < 4 ? queries : keys)) continue;
    ASC_REQUIRE(rows[i]->data, ASC_ERR_INVALID_ARG, "%s: null buffer", what);
    ASC_REQUIRE(asc::kv::row_operand(*rows[i]), ASC_ERR_ALIGNMENT,
                "%s: buffers must be 16-byte aligned, with strides that are multiples of 8", what);
  }
  ASC_REQUIRE(!queries || a->lse, ASC_ERR_INVALID_ARG, "%s: null lse", what);
  p.kv_heads = static_cast<int32_t>(a->kv_heads > 0 ? a->kv_heads : 1);
  p.group = static_cast<int32_t>(a->q_heads / p.kv_heads);
  p.n_q = static_cast<int32_t>(a->q_len);
  p.rows = p.group * p.n_q;
  p.capacity = static_cast<int32_t>(a->kv_len);
  p.lengths = a->kv_lengths;
  p.scale = a->sm_scale;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  p.inv_scale = 1.0f / a->sm_scale;
  const auto in = [&](const asc_rows_t& r, bool q, const uint8_t*& base, asc::kv::Strides& s) {
    base = static_cast<const uint8_t*>(r.data);
    return asc::kv::strides_of(r, a->batch, q ? a->q_heads : a->kv_heads, q ? a->q_len : a->kv_len, a->head_dim, what,
                               s);
  };
  if (queries) {
    if ((rc = in(a->q, true, p.q, p.qs)) != ASC_OK) return rc;
    if ((rc = in(a->o, true, p.o, p.os)) != ASC_OK) return rc;
    if ((rc = in(a->d_o, true, p.d_o, p.dos)) != ASC_OK) return rc;
    p.lse = a->lse;
    p.dq = static_cast<uint16_t*>(a->dq.data);
    p.dq_batch = a->dq.batch_stride;
    p.dq_head = a->dq.head_stride;
    p.dq_seq = a->dq.seq_stride;
  }
  if (keys) {
    if ((rc = in(a->k, false, p.k, p.ks)) != ASC_OK) return rc;
    if ((rc = in(a->v, false, p.v, p.vs)) != ASC_OK) return rc;
    p.dk = static_cast<uint16_t*>(a->dk.data);
    p.dk_batch = a->dk.batch_stride;
    p.dk_head = a->dk.head_stride;
    p.dk_seq = a->dk.seq_stride;
    p.dv = static_cast<uint16_t*>(a->dv.data);
    p.dv_batch = a->dv.batch_stride;
    p.dv_head = a->dv.head_stride;
    p.dv_seq = a->dv.seq_stride;
  }
  L.keys = queries || keys;
  if (!L.keys) return ASC_OK;
  plan(L, *a);
  ASC_REQUIRE(L.q_grid < int64_t{1} << 22 && L.kv_grid < int64_t{1} << 22, ASC_ERR_UNSUPPORTED,
              "%s: the launch exceeds the grid limit", what);
  return ASC_OK;
}

int32_t check_places(const asc_attention_t& a, const char* what) {
  const auto rows = [&](const char* name, const asc_rows_t& r, bool q) {
    return asc::region_of(name, r, a.batch, q ? a.q_heads : a.kv_heads, q ? a.q_len : a.kv_len, a.head_dim, 2);
  };
  const asc::Region results[] = {rows("dq", a.dq, true), rows("dk", a.dk, false), rows("dv", a.dv, false)};
  const asc::Region operands[] = {
      rows("do", a.d_o, true), rows("q", a.q, true), rows("k", a.k, false), rows("v", a.v, false), rows("o", a.o, true),
      asc::region_of("lse", a.lse, a.batch * a.q_heads * a.q_len * static_cast<int64_t>(sizeof(float))),
      asc::region_of("kv_lengths", a.kv_lengths, a.batch * static_cast<int64_t>(sizeof(int32_t)))};
  return asc::kv::check_places(what, results, operands);
}

template <int D, class E>
int32_t launch(const Launch& L, const char* what, hipStream_t stream) {
  const auto grid = [](int64_t n) { return dim3(static_cast<uint32_t>(n)); };
  if (L.q_grid > 0) {
    hipLaunchKernelGGL((grad_q<D, E>), grid(L.q_grid), dim3(GradQ<D>::kWaves * 64), 0, stream, L.p);
    const int32_t rc = asc::check_launch(what);
    if (rc != ASC_OK) return rc;
  }
  if (L.kv_grid > 0) {
    const auto kernel = L.p.n_q < GradKv<D>::kRows ? grad_kv<D, E, true> : grad_kv<D, E, false>;
    hipLaunchKernelGGL(kernel, grid(L.kv_grid), dim3(GradKv<D>::kWaves * 64), 0, stream, L.p);
    const int32_t rc = asc::check_launch(what);
    if (rc != ASC_OK) return rc;
  }
  const int64_t joins = int64_t{L.p.q_join} + 2 * int64_t{L.p.kv_join};
  if (joins > 0) hipLaunchKernelGGL((join_grad<D, E>), grid(joins), dim3(256), 0, stream, L.p);
  return asc::check_launch(what);
}

}  // namespace

extern "C" int64_t asc_cross_attention_bwd_workspace(const asc_attention_t* args) {
  Launch L;
  return make(args, "asc_cross_attention_bwd_workspace", L) == ASC_OK ? workspace_of(L) : 0;
}

extern "C" int32_t asc_cross_attention_bwd(const asc_attention_t* args, void* workspace, int64_t workspace_bytes,
                                           asc_stream_t stream) {
  const char* what = "asc_cross_attention_bwd";
  Launch L;
  int32_t rc = make(args, what, L);
  if (rc != ASC_OK || !L.keys) return rc;
  const int64_t need = workspace_of(L);
  ASC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && asc::aligned16(workspace)), ASC_ERR_INVALID_ARG,
              "%s: the workspace must hold %lld bytes, 16-byte aligned", what, static_cast<long long>(need));
  rc = check_places(*args, what);
  if (rc != ASC_OK) return rc;
  float* at = static_cast<float*>(workspace);
  const auto take = [&at](int64_t n) {
    float* r = at;
    at += region(n);
    return r;
  };
  L.p.neg_a = take(L.values);
  L.p.neg_d = take(L.values);
  L.p.part_q = take(L.parts_q);
  L.p.part_k = take(L.parts_kv);
  L.p.part_v = take(L.parts_kv);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f16 = args->dtype == ASC_DT_FLOAT16;
  if (args->head_dim == 64) {
    return f16 ? launch<64, asc::fa::F16>(L, what, s) : launch<64, asc::fa::Bf16>(L, what, s);
  }
  return f16 ? launch<128, asc::fa::F16>(L, what, s) : launch<128, asc::fa::Bf16>(L, what, s);
}
