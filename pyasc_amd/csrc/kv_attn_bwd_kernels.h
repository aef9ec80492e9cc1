// Gradients of attention over other keys than the queries' own: the device code of
// asc_cross_attention_bwd.
//
// With s = q k^T c, p = exp(s - lse), o = p v:
//   delta = rowsum(do * o),  ds = p * (do v^T - delta),
//   dq = c ds k,  dk = c ds^T q,  dv = p^T do.
// s and do v^T are taken again from the tiles (nothing of size queries x keys is kept): two kernels,
// each owning the rows that it sums into, so the sums have a fixed order and need no atomics:
//
//  - grad_q: a wave owns 32 rows (a query of one of the heads that share a key / value head) and
//    streams the keys: S^T = K Q^T and dP^T = V dO^T hold one row per lane, dQ^T += K^T dS^T takes
//    dS^T straight from those registers.  It also leaves -lse / sm_scale and -delta of its rows
//    for the other kernel.
//  - grad_kv: a wave owns 32 keys and streams the rows of every query head that shares them:
//    S = Q K^T and dP = dO V^T hold one key per lane, with -lse / sm_scale and -delta of the rows
//    as the products' initial values; dV^T += dO^T P and dK^T += Q^T dS.
//
// A tile is read from LDS as rows (an operand of S or dP) and transposed (of the sums), so its
// 16-byte chunks are placed for both: chunk c of row r at c ^ place(r).
// Where rows or keys are few, keys (grad_q) or rows (grad_kv) are split over workgroups, whose fp32
// parts join_grad adds in order.
//
// Two things bound both.  A wave's products, exp2, packing and sums follow one another, so the matrix units
// are busy 40 to 47% of the time; and the board is at its power: 1372 to 1400 W of 1400, at 2.0 to 2.1
// GHz.  4 sequences, 32 / 8 heads of 128, 2048 queries, 1024 keys, bf16: grad_q (three products) 225 us,
// 0.92 PFLOP/s, matrix units busy 40%; grad_kv (four) 266 us, 1.03 PFLOP/s, 47%; join_grad 15 us for dk and
// dv in two parts each (84 MB).
#pragma once

#include "kv_attn_kernels.h"

namespace asc {
namespace kv {

struct GradArgs {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* o;
  const uint8_t* d_o;
  const float* lse;  // [batch, q_heads, n_q]
  Strides qs, ks, vs, os, dos;
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  int64_t dq_batch, dq_head, dq_seq, dk_batch, dk_head, dk_seq, dv_batch, dv_head, dv_seq;  // elements
  const int32_t* lengths;
  float* neg_a;  // -lse / sm_scale of every row, [batch, q_heads, n_q]
  float* neg_d;  // -delta
  float* part_q;  // [batch, kv_heads, rows][splits][D]
  float* part_k;  // [batch, kv_heads, capacity][splits][D]
  float* part_v;
  int32_t capacity, kv_heads, group, n_q, rows;
  int32_t q_blocks, q_splits, kv_blocks, kv_splits;
  uint32_t q_units, kv_units;  // batch * kv_heads * splits
  uint32_t q_join, kv_join;    // workgroups that add up the parts of dq, of dk and of dv
  int32_t q_join_groups, kv_join_groups;
  float scale, scale_log2, inv_scale;
};

// One workgroup's share: a sequence's key / value head, a block of the rows (keys) that it sums into,
// and which split of what it streams.
struct GradShare {
  int b, head, row0, split;
  bool live;
};
// As share_of: the blocks of one split run on one XCD one after the other.
__device__ __forceinline__ GradShare grad_share(uint32_t blocks, uint32_t splits, uint32_t units, uint32_t kv_heads) {
  const uint32_t slot = blockIdx.x >> 3;
  const uint32_t per = slot / blocks;
  const uint32_t unit = per * 8 + (blockIdx.x & 7);
  GradShare s;
  s.live = unit < units;
  const uint32_t bh = unit / splits;
  s.split = static_cast<int>(unit - bh * splits);
  s.b = static_cast<int>(bh / kv_heads);
  s.head = static_cast<int>(bh - static_cast<uint32_t>(s.b) * kv_heads);
  s.row0 = static_cast<int>(slot - per * blocks);
  return s;
}

// Sixteen rows that read one chunk (a row operand) hit all banks, and so do four rows of 64 bytes
// (a transposed one).
template <int D>
__device__ __forceinline__ int place(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}
template <int D>
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
  return static_cast<uint32_t>(row * (D * 2) + ((chunk ^ place<D>(row)) << 4));
}

template <int D, int kWaves, class E>
struct Tiles {
  static constexpr int kKSteps = D / 16, kDBlocks = D / 32;
  static constexpr int kRowsPerLoad = 1024 / (D * 2), kLanesPerRow = 64 / kRowsPerLoad;

  int lane, wave, col, h;
  // One address per kind of operand; other chunks and rows are some of its bits flipped, as the
  // places only flip bits and a block of 32 rows starts at a multiple of its size.
  uint32_t raddr;  // row operand: row col, chunk h (k-step kk: 2 kk chunks away)
  uint32_t taddr;  // transposed operand: rows 4 h + 0..3 (w: 8 rows, db: 4 chunks away)

  __device__ __forceinline__ void init(int tid) {
    lane = tid & 63;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    col = lane & 31;
    h = lane >> 5;
    raddr = tile_off<D>(col, h);
    const int g_lane = lane & 15;
    const int tr_col = ((lane >> 4) & 1) * 16 + (g_lane & 3) * 4;
    taddr = tile_off<D>(4 * h + (g_lane >> 2), tr_col >> 3) + (tr_col & 7) * 2;
  }

  // Rows row0 .. row0 + kRows - 1 of `base` (`stride` 16-byte units apart) into an LDS tile; rows
  // >= n are zeros.  kPacked: row r is row r % per_head of head r / per_head.
  template <int kRows, bool kPacked = false>
  __device__ __forceinline__ void load(uint8_t* dst, const uint8_t* base, uint32_t stride, int row0, int n,
                                       int per_head = 0, uint32_t head_stride = 0) const {
    constexpr int kLoads = kRows / kRowsPerLoad / kWaves;
    static_assert(kLoads >= 1, "a load per wave");
    int wave_lds = wave * (kLoads * 1024);
    asm volatile("" : "+s"(wave_lds));
    const int rr = lane / kLanesPerRow, pos = lane % kLanesPerRow;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = kRowsPerLoad * (wave * kLoads + i) + rr;
      const uint8_t* src = base + static_cast<uint64_t>(row0 + row) * (static_cast<uint64_t>(stride) * 16);
      if constexpr (kPacked) {
        const uint32_t g = static_cast<uint32_t>(row0 + row) / static_cast<uint32_t>(per_head);
        const uint32_t s = static_cast<uint32_t>(row0 + row) - g * static_cast<uint32_t>(per_head);
        src = base + (static_cast<uint64_t>(g) * head_stride + static_cast<uint64_t>(s) * stride) * 16;
      }
      if (row0 + row >= n) src = reinterpret_cast<const uint8_t*>(kZeroRow);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(src + ((pos ^ place<D>(row)) << 4)),
          (__attribute__((address_space(3))) void*)(dst + wave_lds + i * 1024), 16, 0, 0);
    }
  }

  // x += A bx and y += B by for 32 rows of two tiles (A, B: row operands).
  __device__ __forceinline__ void products(uint32_t a_base, uint32_t b_base, const u32x4 (&bx)[kKSteps],
                                           const u32x4 (&by)[kKSteps], f32x16& x, f32x16& y) const {
    constexpr int kWin = 3, kReads = 2 * kKSteps;  // 4: 1% slower, for the registers
    u32x4 a[kReads];
    const auto read = [&](int r) {
      return fa::lds_read_b128(((r < kKSteps ? a_base : b_base) + raddr) ^ (r % kKSteps << 5), 0);
    };
#pragma unroll
    for (int r = 0; r < kWin; ++r) a[r] = read(r);
#pragma unroll
    for (int r = 0; r < kReads; ++r) {
      fa::lds_wait(a[r], r + kWin <= kReads ? kWin - 1 : kReads - 1 - r);
      if (r < kKSteps) {
        x = E::mfma(a[r], bx[r % kKSteps], x);
      } else {
        y = E::mfma(a[r], by[r % kKSteps], y);
      }
      if (r + kWin < kReads) a[r + kWin] = read(r + kWin);
    }
  }

  // Operand (db, u) of a transposed tile: rows 16 u + 4 h + 0..3 and 16 u + 8 + 4 h + 0..3.
  __device__ __forceinline__ u32x4 transposed(uint32_t base, int db, int u) const {
    const uint32_t at = (base + taddr) ^ (db << 6);
    const u32x2 lo = fa::lds_read_tr16_b64(at, u * 16 * (D * 2));
    const u32x2 hi = fa::lds_read_tr16_b64(at ^ (8 * D * 2 + 32), u * 16 * (D * 2));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
  // acc += A^T b for 32 rows of the tile at base, b[u] holding rows 16 u ..
  __device__ __forceinline__ void add_transposed(uint32_t base, const u32x4 (&b)[2], f32x16 (&acc)[kDBlocks]) const {
    constexpr int kWin = 4, kOps = 2 * kDBlocks;
    u32x4 a[kOps];
#pragma unroll
    for (int r = 0; r < kWin; ++r) a[r] = transposed(base, r >> 1, r & 1);
#pragma unroll
    for (int r = 0; r < kOps; ++r) {
      fa::lds_wait(a[r], 2 * (r + kWin <= kOps ? kWin - 1 : kOps - 1 - r));
      acc[r >> 1] = E::mfma(a[r], b[r & 1], acc[r >> 1]);
      if (r + kWin < kOps) a[r + kWin] = transposed(base, (r + kWin) >> 1, (r + kWin) & 1);
    }
  }

  // This lane's row as the other operand of products(): d = 16 ks + 8 h + 0..7.
  __device__ __forceinline__ void own_row(const uint8_t* row, bool live, u32x4 (&x)[kKSteps]) const {
#pragma unroll
    for (int ks = 0; ks < kKSteps; ++ks) {
      x[ks] = u32x4{0, 0, 0, 0};
      if (live) x[ks] = *reinterpret_cast<const u32x4*>(row + ks * 32 + h * 16);
    }
  }

  // Registers of products() rounded and packed as the operand of add_transposed().
  static __device__ __forceinline__ void pack(const f32x16& x, u32x4 (&b)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int w = 0; w < 4; ++w) b[u][w] = E::pack(x[8 * u + 2 * w], x[8 * u + 2 * w + 1]);
  }

  // As pack, of the scores' gradients whose products acc sums up for this lane's row (or key).  bf16 has
  // fp32's range.  fp16 has not: 8192 keys and gradients of 2^-10 leave nothing of ds but its last
  // bits, and 2^16 is soon passed.  So its ds come here at `up`, a power of two of the row's own, times
  // their value: the first tile, or one with a value above 2^15, puts its largest between 2^7 and 2^8
  // (both halves of the lanes hold the row) and acc follows.  Values down to 2^-22 of the largest keep all
  // their bits.  Finite rows of 128 values give ds of at most 2^40, 2^114 at the first `up` and kProbUp.  4
  // sequences, 32 / 8 heads, 2048 queries, 1024 keys, fp16: 536 us for 518 at head_dim 128, 305 for 288 at 64.
  static constexpr bool kMoves = __is_same(E, fa::F16);
  static constexpr float kFirstUp = kMoves ? 0x1p60f : 1.0f;
  static __device__ __forceinline__ void pack_moving(f32x16& x, float& up, f32x16 (&acc)[kDBlocks], u32x4 (&b)[2]) {
    if constexpr (kMoves) {
      float most = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(x[r]));
      if (__builtin_amdgcn_ballot_w64(most > 0x1p15f && most < INFINITY) != 0) {
        most = fmaxf(most, other_half(most));
        // 2^7 over the power of two below most, by the exponents as stored
        const uint32_t e = __builtin_bit_cast(uint32_t, most) >> 23;
        const float by =
            most > 0x1p15f && most < INFINITY ? __builtin_bit_cast(float, (127 + 7 + 127 - e) << 23) : 1.0f;
        up *= by;
        x *= by;
#pragma unroll
        for (int i = 0; i < kDBlocks; ++i) acc[i] *= by;
      }
    }
    pack(x, b);
  }
  // What takes `up` from a sum again: 1 / up.
  static __device__ __forceinline__ float back(float up) {
    return kMoves ? __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, up)) : 1.0f;
  }
  // The probabilities' operand of dv: at most 1, held at 2^14 times their value in fp16, so that they keep
  // all bits down to 2^-28 (1 / keys reaches 2^-14 at 16384 keys).
  static constexpr float kProbUp = kMoves ? 14.0f : 0.0f, kProbBack = kMoves ? 0x1p-14f : 1.0f;

  // acc^T (d = 32 db + 8 rq + 4 h + 0..3 of this lane's row) to rows, as values, through 32 rows of LDS of
  // this wave: a lane's own 8 bytes of a row at a time would be 32 pieces of 16 bytes per store.  out(r):
  // where the wave's row r goes, null: nowhere.
  template <class Out>
  __device__ __forceinline__ void store(uint8_t* mine, const f32x16 (&acc)[kDBlocks], float scale, bool zero,
                                        Out out) const {
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        u32x2 w;
        w[0] = E::pack(acc[db][rq * 4] * scale, acc[db][rq * 4 + 1] * scale);
        w[1] = E::pack(acc[db][rq * 4 + 2] * scale, acc[db][rq * 4 + 3] * scale);
        *reinterpret_cast<u32x2*>(mine + tile_off<D>(col, db * 4 + rq) + h * 8) = zero ? u32x2{0, 0} : w;
      }
    constexpr int kChunks = D / 8;
#pragma unroll
    for (int i = 0; i < 32 * kChunks / 64; ++i) {
      const int at = i * 64 + lane, r = at / kChunks, ch = at % kChunks;
      uint16_t* row = out(r);
      if (row != nullptr) {
        *reinterpret_cast<u32x4*>(row + ch * 8) = *reinterpret_cast<const u32x4*>(mine + tile_off<D>(r, ch));
      }
    }
  }
  __device__ __forceinline__ void store_part(const f32x16 (&acc)[kDBlocks], float* row) const {
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        *reinterpret_cast<f32x4*>(row + db * 32 + rq * 8 + h * 4) =
            f32x4{acc[db][rq * 4], acc[db][rq * 4 + 1], acc[db][rq * 4 + 2], acc[db][rq * 4 + 3]};
      }
  }
};

// Keys of sequence b; bad: a length outside [0, capacity].
__device__ __forceinline__ int keys_of(const GradArgs& p, int b, bool& bad) {
  const int n = p.lengths ? p.lengths[b] : p.capacity;
  bad = n < 0 || n > p.capacity;
  return n < 0 ? 0 : (n > p.capacity ? p.capacity : n);
}

template <int D>
struct GradQ {
  static constexpr int kWaves = D == 128 ? 8 : 4, kWgPerCu = D == 128 ? 1 : 2;
  static constexpr int kRows = 32 * kWaves;
  static constexpr int kKeys = 64;  // of a tile
};
constexpr int kExactTiles = 3;  // up to as many, as the ring has stages, delta is exact (see grad_q_body)

template <int D, class E>
__device__ __forceinline__ void grad_q_body(const GradArgs& p) {
  constexpr int kWaves = GradQ<D>::kWaves, kKeys = GradQ<D>::kKeys;
  using T = Tiles<D, kWaves, E>;
  constexpr int kTile = kKeys * D * 2;
  constexpr int kLoads = 2 * (kKeys / T::kRowsPerLoad / kWaves);  // of K and V, per wave and tile
  __shared__ __attribute__((aligned(8192))) uint8_t ring[6 * kTile];  // K stages 0-2, V stages 3-5

  const GradShare s = grad_share(p.q_blocks, p.q_splits, p.q_units, p.kv_heads);
  if (!s.live) return;
  T t;
  t.init(threadIdx.x);
  bool bad;
  const int len = keys_of(p, s.b, bad);
  const int row = (s.row0 * kWaves + t.wave) * 32 + t.col;
  const bool live = row < p.rows;
  const bool act = (s.row0 * kWaves + t.wave) * 32 < p.rows;  // of the wave; others only load and wait
  const int g = live ? row / p.n_q : 0, query = live ? row - g * p.n_q : 0;
  const uint32_t head = s.head * p.group + g;
  const auto at = [&](const uint8_t* base, const Strides& st) {
    return base + (static_cast<uint64_t>(s.b) * st.batch + static_cast<uint64_t>(head) * st.head +
                   static_cast<uint64_t>(query) * st.seq) * 16;
  };

  const int total = (len + kKeys - 1) / kKeys;
  // few keys are not split, however many there could be: the first split sees all of them
  const int per = total <= kExactTiles ? total : (total + p.q_splits - 1) / p.q_splits;
  const int begin = min(total, s.split * per), end = min(total, begin + per);
  const uint8_t* kbase = p.k + (static_cast<uint64_t>(s.b) * p.ks.batch + static_cast<uint64_t>(s.head) * p.ks.head) * 16;
  const uint8_t* vbase = p.v + (static_cast<uint64_t>(s.b) * p.vs.batch + static_cast<uint64_t>(s.head) * p.vs.head) * 16;
  const auto load = [&](int j, int stage) {
    t.template load<kKeys>(ring + stage * kTile, kbase, p.ks.seq, j * kKeys, len);
    t.template load<kKeys>(ring + (3 + stage) * kTile, vbase, p.vs.seq, j * kKeys, len);
  };
  if (begin < end) load(begin, 0);
  if (begin + 1 < end) load(begin + 1, 1);

  u32x4 q[T::kKSteps], d_o[T::kKSteps];
  t.own_row(at(p.q, p.qs), live, q);
  t.own_row(at(p.d_o, p.dos), live, d_o);
  // delta: this lane has half of its row's values, the other half of the lanes the rest
  float delta = 0.f;
  {
    u32x4 o[T::kKSteps];
    t.own_row(at(p.o, p.os), live, o);
#pragma unroll
    for (int ks = 0; ks < T::kKSteps; ++ks)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const auto val = [](uint32_t bits, int half) {
          const uint16_t b = static_cast<uint16_t>(half ? bits >> 16 : bits);
          return __is_same(E, fa::Bf16) ? bf16_to_f32(b) : f16_to_f32(b);
        };
        delta = fmaf(val(o[ks][w], 0), val(d_o[ks][w], 0), delta);
        delta = fmaf(val(o[ks][w], 1), val(d_o[ks][w], 1), delta);
      }
    delta += other_half(delta);
  }
  const int64_t row_at = (static_cast<int64_t>(s.b) * p.kv_heads * p.group + head) * p.n_q + query;
  // a row without keys: its probabilities are 0
  const float lse = live ? p.lse[row_at] : -INFINITY;
  const float a = lse == -INFINITY ? INFINITY : lse * p.inv_scale;
  const float neg_l2 = lse == -INFINITY ? -INFINITY : -lse * 1.4426950408889634f;

  // body(tile, x, y) for every 32 keys: x the probabilities, y = dP; loaded: the tiles are in the ring
  const auto stream = [&](bool loaded, auto body) {
    int c = 0;
    for (int j = begin; j < end; ++j) {
      if (!loaded) {
        // every wave has read the stage that the tile after the next goes to: it was tile j-1's
        if (j + 1 < end) {
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLoads) : "memory");
        } else {
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        }
        asm volatile("s_barrier" ::: "memory");
        if (j + 2 < end) load(j + 2, c == 0 ? 2 : c - 1);
      }
      const int at = c;
      c = c == 2 ? 0 : c + 1;
      if (!act) continue;
      const uint32_t kt = fa::lds_addr(ring + at * kTile), vt = fa::lds_addr(ring + (3 + at) * kTile);
#pragma unroll
      for (int kb = 0; kb < kKeys / 32; ++kb) {
        const uint32_t off = kb * 32 * D * 2;
        f32x16 x = {}, y = {};
        t.products(kt + off, vt + off, q, d_o, x, y);
        if (j * kKeys + kb * 32 + 32 > len) {  // keys behind the length
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            if (j * kKeys + kb * 32 + (r >> 2) * 8 + t.h * 4 + (r & 3) >= len) x[r] = -INFINITY;
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], p.scale_log2, neg_l2));
        body(kt + off, x, y);
      }
    }
  };

  // o is rounded to its type, and delta with it.  Over few keys, where o is as large as the values,
  // that shows in the gradients (0.0026 against 0.0024 relative, bf16, 10 keys), and delta is taken
  // as the sum of p dP in a pass of its own; over many it is left to o: the pass would add two products
  // to the nine.  It shows there too where rows give few of the keys most of their probability: 256 rows,
  // 1024 keys, bf16, dq off by 0.0024 of its norm with a largest probability of 0.02, 0.0033 of
  // 0.42 and 0.0054 of 0.70 (0.0016 where only the result is rounded).
  if (total <= kExactTiles) {
    delta = 0.f;
    stream(false, [&](uint32_t, const f32x16& x, const f32x16& y) {
#pragma unroll
      for (int r = 0; r < 16; ++r) delta = fmaf(x[r], y[r], delta);
    });
    delta += other_half(delta);
  }

  f32x16 acc[T::kDBlocks];
#pragma unroll
  for (int i = 0; i < T::kDBlocks; ++i) acc[i] = f32x16{};
  float up = T::kFirstUp;
  if (live && t.h == 0 && s.split == 0) {
    p.neg_a[row_at] = -a;
    p.neg_d[row_at] = -delta;
  }
  stream(total <= kExactTiles, [&](uint32_t kt, f32x16& x, const f32x16& y) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= T::kMoves ? fmaf(y[r], up, -delta * up) : y[r] - delta;
    u32x4 ds[2];
    T::pack_moving(x, up, acc, ds);
    t.add_transposed(kt, ds, acc);
  });
  if constexpr (T::kMoves) {
#pragma unroll
    for (int i = 0; i < T::kDBlocks; ++i) acc[i] *= T::back(up);
  }
  const float scale = bad ? __builtin_nanf("") : p.scale;
  if (p.q_splits > 1) {
    if (!live) return;
    const int64_t part = ((static_cast<int64_t>(s.b) * p.kv_heads + s.head) * p.rows + row) * p.q_splits + s.split;
    if (bad) {
#pragma unroll
      for (int i = 0; i < T::kDBlocks; ++i) acc[i] += scale;
    }
    t.store_part(acc, p.part_q + part * D);
    return;
  }
  // the rows go where another wave may still read a tile
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  asm volatile("s_barrier" ::: "memory");
  const int row0 = (s.row0 * kWaves + t.wave) * 32;
  t.store(ring + t.wave * (32 * D * 2), acc, scale, false, [&](int r) -> uint16_t* {
    if (row0 + r >= p.rows) return nullptr;
    const int g = (row0 + r) / p.n_q, query = row0 + r - g * p.n_q;
    return p.dq + s.b * p.dq_batch + static_cast<int64_t>(s.head * p.group + g) * p.dq_head + query * p.dq_seq;
  });
}

template <int D>
struct GradKv {
  static constexpr int kWaves = 4, kWgPerCu = 2;
  static constexpr int kKeys = 32 * kWaves;
  static constexpr int kRows = 32;  // of a tile
};

// kPacked: fewer queries than a tile has rows, so those of several heads share one.
template <int D, class E, bool kPacked>
__device__ __forceinline__ void grad_kv_body(const GradArgs& p) {
  constexpr int kWaves = GradKv<D>::kWaves, kRows = GradKv<D>::kRows;
  using T = Tiles<D, kWaves, E>;
  constexpr int kTile = kRows * D * 2;
  constexpr int kLoads = 2 * (kRows / T::kRowsPerLoad / kWaves);
  __shared__ __attribute__((aligned(8192))) uint8_t ring[6 * kTile];  // Q stages 0-2, dO stages 3-5
  __shared__ __attribute__((aligned(16))) float values[3][2 * kRows];  // -lse / scale and -delta of a tile

  const GradShare s = grad_share(p.kv_blocks, p.kv_splits, p.kv_units, p.kv_heads);
  if (!s.live) return;
  T t;
  t.init(threadIdx.x);
  bool bad;
  const int len = keys_of(p, s.b, bad);
  const int key0 = s.row0 * GradKv<D>::kKeys;
  const int key = key0 + t.wave * 32 + t.col;
  const bool live = key < len;
  const bool act = key0 + t.wave * 32 < len;  // of the wave; others only load and wait

  // tiles of rows: every query head of the group, its queries in tiles
  const int per_head = ((kPacked ? p.rows : p.n_q) + kRows - 1) / kRows;
  const int total = key0 < len ? (kPacked ? per_head : per_head * p.group) : 0;
  const int per = (total + p.kv_splits - 1) / p.kv_splits;
  const int begin = min(total, s.split * per), end = min(total, begin + per);
  int next_head = per_head && !kPacked ? begin / per_head : 0, next_tile = begin - next_head * per_head;  // of the next load
  float value = 0.f;  // loaded for a tile, not yet in LDS
  const auto load = [&](int stage) {
    const uint64_t head = static_cast<uint64_t>(s.head) * p.group + next_head;
    const int row0 = next_tile * kRows;
    const int n = kPacked ? p.rows : p.n_q;
    if (t.wave == 0) {
      const int row = row0 + t.col;
      const float* from = t.h ? p.neg_d : p.neg_a;
      value = t.h ? 0.f : -INFINITY;  // behind the queries: probability 0
      // the heads of a group follow each other
      if (row < n) value = from[(static_cast<int64_t>(s.b) * p.kv_heads * p.group + head) * p.n_q + row];
    }
    const uint8_t* q = p.q + (static_cast<uint64_t>(s.b) * p.qs.batch + head * p.qs.head) * 16;
    const uint8_t* d_o = p.d_o + (static_cast<uint64_t>(s.b) * p.dos.batch + head * p.dos.head) * 16;
    t.template load<kRows, kPacked>(ring + stage * kTile, q, p.qs.seq, row0, n, p.n_q, p.qs.head);
    t.template load<kRows, kPacked>(ring + (3 + stage) * kTile, d_o, p.dos.seq, row0, n, p.n_q, p.dos.head);
    if (++next_tile == per_head) {
      next_tile = 0;
      ++next_head;
    }
  };
  const auto put_values = [&](int stage) {
    if (t.wave == 0) values[stage][t.lane] = value;
  };
  if (begin < end) {
    load(0);
    put_values(0);
  }
  if (begin + 1 < end) load(1);

  u32x4 k[T::kKSteps], v[T::kKSteps];
  const uint64_t at_key = live ? key : 0;
  t.own_row(p.k + (static_cast<uint64_t>(s.b) * p.ks.batch + static_cast<uint64_t>(s.head) * p.ks.head +
                   at_key * p.ks.seq) * 16, live, k);
  t.own_row(p.v + (static_cast<uint64_t>(s.b) * p.vs.batch + static_cast<uint64_t>(s.head) * p.vs.head +
                   at_key * p.vs.seq) * 16, live, v);
  f32x16 dk[T::kDBlocks], dv[T::kDBlocks];
#pragma unroll
  for (int i = 0; i < T::kDBlocks; ++i) dk[i] = dv[i] = f32x16{};
  float up = T::kFirstUp;

  int c = 0;
  for (int j = begin; j < end; ++j) {
    const int c1 = c == 2 ? 0 : c + 1, c2 = c == 0 ? 2 : c - 1;
    if (j + 1 < end) {
      put_values(c1);
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLoads) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }
    asm volatile("s_barrier" ::: "memory");
    if (j + 2 < end) load(c2);
    const int at = c;
    c = c1;
    if (!act) continue;
    const uint32_t qt = fa::lds_addr(ring + at * kTile), dt = fa::lds_addr(ring + (3 + at) * kTile);
    const uint32_t vals = fa::lds_addr(reinterpret_cast<const uint8_t*>(values[at])) + t.h * 16;
    u32x4 ia[4], id[4];  // rows 8 i + 4 h + 0..3
#pragma unroll
    for (int i = 0; i < 4; ++i) ia[i] = fa::lds_read_b128(vals, i * 32);
#pragma unroll
    for (int i = 0; i < 4; ++i) id[i] = fa::lds_read_b128(vals, kRows * 4 + i * 32);
    fa::lds_wait(ia, 0);
    fa::lds_wait(id, 0);
    f32x16 x, y;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = __builtin_bit_cast(float, static_cast<uint32_t>(ia[r >> 2][r & 3]));
      y[r] = __builtin_bit_cast(float, static_cast<uint32_t>(id[r >> 2][r & 3]));
    }
    t.products(qt, dt, k, v, x, y);
    u32x4 pb[2], ds[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = __builtin_amdgcn_exp2f(T::kMoves ? fmaf(x[r], p.scale_log2, T::kProbUp) : x[r] * p.scale_log2);
      y[r] *= T::kMoves ? x[r] * up : x[r];
    }
    T::pack(x, pb);
    T::pack_moving(y, up, dk, ds);
    t.add_transposed(dt, pb, dv);
    t.add_transposed(qt, ds, dk);
  }
  if constexpr (T::kMoves) {  // dk's terms hold the probabilities' factor too
#pragma unroll
    for (int i = 0; i < T::kDBlocks; ++i) {
      dk[i] *= T::back(up) * T::kProbBack;
      dv[i] *= T::kProbBack;
    }
  }
  const float nan = __builtin_nanf("");
  if (p.kv_splits > 1) {
    if (key >= p.capacity) return;
    const int64_t part = ((static_cast<int64_t>(s.b) * p.kv_heads + s.head) * p.capacity + key) * p.kv_splits + s.split;
#pragma unroll
    for (int i = 0; i < T::kDBlocks; ++i) {
      if (!live) dk[i] = dv[i] = f32x16{};
      if (bad) {
        dk[i] += nan;
        dv[i] += nan;
      }
    }
    t.store_part(dk, p.part_k + part * D);
    t.store_part(dv, p.part_v + part * D);
    return;
  }
  // keys behind the length have no part in the results
  const bool zero = !live && !bad;
  // the rows go where another wave may still read a tile
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  asm volatile("s_barrier" ::: "memory");
  uint8_t* mine = ring + t.wave * (32 * D * 2);
  const auto rows_of = [&](uint16_t* base, int64_t seq) {
    return [=](int r) -> uint16_t* {
      const int at = key0 + t.wave * 32 + r;
      return at < p.capacity ? base + at * seq : nullptr;
    };
  };
  t.store(mine, dk, bad ? nan : p.scale, zero, rows_of(p.dk + s.b * p.dk_batch + s.head * p.dk_head, p.dk_seq));
  t.store(mine, dv, bad ? nan : 1.0f, zero, rows_of(p.dv + s.b * p.dv_batch + s.head * p.dv_head, p.dv_seq));
}

// Adds up the parts of rows.  kind 0: dq, 1: dk, 2: dv, in q_join, kv_join and kv_join workgroups of one
// launch.
template <int D, class E>
__device__ __forceinline__ void join_grad_body(const GradArgs& p) {
  const int kind = blockIdx.x < p.q_join ? 0 : (blockIdx.x < p.q_join + p.kv_join ? 1 : 2);
  const uint32_t block = blockIdx.x - (kind == 0 ? 0 : p.q_join + (kind - 1) * p.kv_join);
  const int per_head = kind == 0 ? p.rows : p.capacity, splits = kind == 0 ? p.q_splits : p.kv_splits;
  const JoinLanes<D> at(block, kind == 0 ? p.q_join_groups : p.kv_join_groups);
  const int64_t bh = at.row / per_head;
  if (bh >= static_cast<int64_t>((kind == 0 ? p.q_units : p.kv_units) / splits)) return;
  const int row = static_cast<int>(at.row - bh * per_head);
  const int64_t b = bh / p.kv_heads, head = bh - b * p.kv_heads;
  const float* part = (kind == 0 ? p.part_q : kind == 1 ? p.part_k : p.part_v) + at.row * splits * D + at.ch * 8;
  float o[8] = {};
#pragma unroll 4
  for (int k = at.group; k < splits; k += at.groups) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(part + k * D);
    const f32x4 hi = *reinterpret_cast<const f32x4*>(part + k * D + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] += lo[e];
      o[4 + e] += hi[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = at.reduce(o[e], [](float x, float y) { return x + y; });
  if (at.group != 0) return;
  uint16_t* out;
  if (kind == 0) {
    const int g = row / p.n_q;
    out = p.dq + b * p.dq_batch + (head * p.group + g) * p.dq_head + static_cast<int64_t>(row - g * p.n_q) * p.dq_seq;
  } else if (kind == 1) {
    out = p.dk + b * p.dk_batch + head * p.dk_head + row * p.dk_seq;
  } else {
    out = p.dv + b * p.dv_batch + head * p.dv_head + row * p.dv_seq;
  }
  *reinterpret_cast<u32x4*>(out + at.ch * 8) = pack8<E>(o, kind == 2 ? 1.0f : p.scale);
}

}  // namespace kv
}  // namespace asc
