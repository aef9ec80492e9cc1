// Rotary positions of queries and keys, with or without an RMS norm of each head in the same
// pass, and the gradient of both.
//
// Pair (a, b) of frequency f in a token of position p turns by t = p f:
//   a' = m (a cos t - b sin t),  b' = m (b cos t + a sin t),
// which is linear in (a, b); its gradient is the turn by -t times m.  With the norm, r =
// 1 / sqrt(mean(x^2) + eps) and y = turn(x r w); with g = turn^T(dy) the gradients are
//   dw = sum over rows of g x r,   dx = r (g w - x r mean(g w x r)).
//
// Each value is read and written once, so HBM bounds it.  A workgroup takes a few tokens and all
// (or a chunk of) their heads: the angles of its tokens go into LDS once, from the product of
// position and frequency in fp64 (a far position keeps its fraction of a turn).  A row (one head of
// one token) belongs to neighbouring lanes of a wave; a lane holds both values of V pairs, so the
// turn needs no exchange and the norm one butterfly.  A lane stays with its token: cos and sin,
// weights and the steps of its addresses are registers over all heads (with addresses worked out
// row by row, the norm took 74 us where it takes 63).
//
// Contiguous heads, more bytes than the caches hold: bf16, 4 x 4096 tokens, 32 + 8 heads of 128 (336 MB):
// positions 64 us (5.2 TB/s), with the norm 66 (5.1), a copy of the same bytes 65; the gradient (503 MB)
// 106 (4.8), its conversions and sums beside the loads.  fp32 (671 and 1007 MB): 126, 130, a copy 130,
// and 197 us (5.1 to 5.3 TB/s).  Heads whose slots are no power of two leave lanes idle, and a rotated part that
// is not a multiple of 16 values narrows the loads: bf16, head_dim 80, 50 us, 52 and 87 (a copy 43);
// 20 of 80 rotated, 70, 70 and 110; head_dim 130, 121, 127 and 173 (66).
#include <type_traits>

#include "common.h"
#include "numeric.h"
#include "overlap.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;     // of a workgroup at a time
constexpr int kMinTokens = 4;     // where there are many: a row has at most 64 lanes
constexpr int kMaxHeadDim = 512;  // kSlots lanes' slots and the LDS tables cover it
constexpr int kMaxParts = 1024;   // workgroups of a gradient launch: partial sums of its weights

struct Rows {  // [batch, heads, seq, head_dim], the last dimension contiguous
  const void* p;
  int64_t batch, head, seq;
};

struct RotaryArgs {
  Rows x[2];   // queries and keys (gradient: of the forward pass)
  Rows dy[2];  // gradient: of the results
  Rows out[2];
  const float* weight[2];
  float* parts;  // gradient: [workgroup][2][head_dim] sums of g x r
  const void* positions;
  int64_t pos_batch, pos_seq;
  const double* freqs;
  int64_t seq;
  uint32_t units;  // batch * tiles * chunks < 2^31
  uint32_t tiles;  // of tokens per sequence
  uint32_t chunks;  // of heads
  int32_t q_heads, heads, chunk_heads;
  int32_t head_dim, pairs, tokens;
  int32_t lanes;  // of a row, a power of two
  int32_t pos64;
  float sign, magnitude, epsilon, inv_dim;
};

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<_Float16>(_Float16 v) { return static_cast<float>(v); }
template <>
__device__ __forceinline__ float widen<__bf16>(__bf16 v) { return static_cast<float>(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void widen(const Vec<T, V>& w, float (&x)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = widen<T>(w.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&x)[V]) {
  Vec<T, V> w;
#pragma unroll
  for (int i = 0; i < V; ++i) w.v[i] = static_cast<T>(x[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = w;
}

// Sum over the `lanes` (a power of two) neighbouring lanes of a row, by wave_sum's steps.
__device__ __forceinline__ float row_sum(float v, int lanes) {
  if (lanes > 1) v += asc::dpp_mov<asc::kDppQuadXor1>(v);
  if (lanes > 2) v += asc::dpp_mov<asc::kDppQuadXor2>(v);
  if (lanes > 4) v += asc::dpp_mov<asc::kDppRowHalfMirror>(v);
  if (lanes > 8) v += asc::dpp_mov<asc::kDppRowMirror>(v);
  if (lanes > 16) v += asc::lane_xor16(v);
  if (lanes > 32) v += asc::lane_xor32(v);
  return v;
}

// cos and sin of `rev` turns.  The fraction of a quarter turn is exact in fp64 before it is
// rounded to fp32: the angle is off by at most 2^-27.
__device__ __forceinline__ float2 turn_of(double rev, float sign, float magnitude) {
  const double f = rev - rint(rev);
  const double q = rint(f * 4.0);
  float s, c;
  sincospif(2.0f * static_cast<float>(f - 0.25 * q), &s, &c);
  const int quarter = static_cast<int>(q) & 3;
  if (quarter & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  if (quarter & 2) {
    c = -c;
    s = -s;
  }
  return make_float2(c * magnitude, s * sign * magnitude);
}

enum Mode { kTurn, kNorm, kNormGrad };

// Slots of a lane: a row has head_dim / (2 kV) of them on at most 64 lanes.
template <int V>
constexpr int slots_per_lane() { return V >= 4 ? 1 : (V == 2 ? 2 : 4); }

template <typename T, int V, bool kInterleaved, Mode kMode>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(RotaryArgs p) {
  constexpr int kSlots = slots_per_lane<V>();
  __shared__ float2 table[kMaxTokens * kMaxHeadDim / 2];
  __shared__ float weights[kMode != kTurn ? 2 * kMaxHeadDim : 1];

  const int tid = threadIdx.x;
  const int lane = tid & (p.lanes - 1);
  // rows of a pass: tokens fastest, so that neighbours lie together in both orders of heads and
  // tokens; at least as many as tokens, so a lane stays with its token and steps over heads
  const int row0 = tid / p.lanes, rows_per_pass = kThreads / p.lanes;
  const int t = row0 & (p.tokens - 1), head0 = row0 / p.tokens, head_step = rows_per_pass / p.tokens;
  const int pair_slots = p.pairs / V, slots = p.head_dim / (2 * V);

  // the two vectors of each slot: the pairs' first and second values, or two neighbours of
  // the values behind the rotated ones
  int c0[kSlots], c1[kSlots], at[kSlots];
  bool live[kSlots], turned[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int slot = lane + i * p.lanes;
    live[i] = slot < slots;
    turned[i] = slot < pair_slots;
    at[i] = slot * V;
    c0[i] = kInterleaved || !turned[i] ? slot * 2 * V : slot * V;
    c1[i] = kInterleaved || !turned[i] ? c0[i] + V : c0[i] + p.pairs;
  }
  float dw[2][kSlots][2][V] = {};
  if (kMode != kTurn) {
    for (int i = tid; i < 2 * p.head_dim; i += kThreads) {
      const float* w = p.weight[i >= p.head_dim];
      weights[i] = w ? w[i >= p.head_dim ? i - p.head_dim : i] : 0.f;
    }
  }

  for (uint32_t unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
    const uint32_t tile = unit / p.chunks;
    const int chunk = static_cast<int>(unit - tile * p.chunks);
    const int64_t b = tile / p.tiles;
    const int64_t s0 = static_cast<int64_t>(tile % p.tiles) * p.tokens;
    const int tokens = static_cast<int>(p.seq - s0 < p.tokens ? p.seq - s0 : p.tokens);
    const int h0 = chunk * p.chunk_heads;
    const int n_heads = p.heads - h0 < p.chunk_heads ? p.heads - h0 : p.chunk_heads;
    struct Row {
      bool live;
      Vec<T, V> a0[kSlots], a1[kSlots], g0[kSlots], g1[kSlots];
    };
    struct Heads {   // of queries or keys
      const T* x;    // of the next row to fetch, and dy
      const T* dy;
      T* out;  // of the next row to work on
      int64_t x_step, dy_step, out_step;
      int count, left;  // of the unit; from the next row to fetch on
    };
    const auto heads_of = [&](auto which) {
      constexpr int kKind = decltype(which)::value;  // 0: queries, 1: keys
      const int first = kKind == 0 ? h0 : (h0 > p.q_heads ? h0 : p.q_heads) - p.q_heads;
      const int last = kKind == 0 ? (h0 + n_heads < p.q_heads ? h0 + n_heads : p.q_heads) : h0 + n_heads - p.q_heads;
      const auto at_row = [&](const Rows& rows) {
        return static_cast<const T*>(rows.p) + b * rows.batch + (first + head0) * rows.head + (s0 + t) * rows.seq;
      };
      Heads m;
      m.x = at_row(p.x[kKind]);
      m.dy = kMode == kNormGrad ? at_row(p.dy[kKind]) : nullptr;
      m.out = const_cast<T*>(at_row(p.out[kKind]));
      m.x_step = head_step * p.x[kKind].head;
      m.dy_step = head_step * p.dy[kKind].head;
      m.out_step = head_step * p.out[kKind].head;
      m.count = last - first;
      m.left = t < tokens ? m.count - head0 : 0;
      return m;
    };
    const auto fetch = [&](Heads& h, Row& m) {
      m.live = h.left > 0;
      h.left -= head_step;
      if (!m.live) return;
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        if (!live[i]) continue;
        m.a0[i] = load<T, V>(h.x + c0[i]);
        m.a1[i] = load<T, V>(h.x + c1[i]);
      }
      h.x += h.x_step;
      if (kMode == kNormGrad) {
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
          if (!live[i]) continue;
          m.g0[i] = load<T, V>(h.dy + c0[i]);
          m.g1[i] = load<T, V>(h.dy + c1[i]);
        }
        h.dy += h.dy_step;
      }
    };
    // The first rows are asked for ahead of the table; of the gradient's, whose registers are full, the
    // queries' alone and only in four 16-bit values (8 x 2047 tokens of 32 + 8 heads of 64: 53.4 to 51.3 us).
    constexpr bool kAhead = kMode != kNormGrad, kQueriesAhead = kAhead || (sizeof(T) == 2 && V == 4);
    Heads heads[2];
    Row first[2];
    if constexpr (kQueriesAhead) {
      heads[0] = heads_of(std::integral_constant<int, 0>{});
      fetch(heads[0], first[0]);
    }
    if constexpr (kAhead) {
      heads[1] = heads_of(std::integral_constant<int, 1>{});
      fetch(heads[1], first[1]);
    }
    __syncthreads();  // the table's last readers
    for (int i = tid; i < tokens * p.pairs; i += kThreads) {
      const int of = i / p.pairs, j = i - of * p.pairs;
      const int64_t o = b * p.pos_batch + (s0 + of) * p.pos_seq;
      const double pos = p.pos64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[o])
                                 : static_cast<double>(static_cast<const int32_t*>(p.positions)[o]);
      table[of * p.pairs + j] = turn_of(pos * (p.freqs[j] * 0.15915494309189533577), p.sign, p.magnitude);
    }
    __syncthreads();
    float2 cs[kSlots][V];  // of this lane's token and pairs, for every head
#pragma unroll
    for (int i = 0; i < kSlots; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        cs[i][e] = t < tokens && turned[i] ? table[t * p.pairs + at[i] + e] : make_float2(1.f, 0.f);
      }
    // Queries and keys one after the other, so that a row's weights and sums are fixed registers.
    // The next row is asked for before this one is worked on.
    const auto rows_of = [&](auto which, Heads& h, Row& first) {
      constexpr int kKind = decltype(which)::value;
      if (h.count <= 0) return;
      float w[kSlots][2][V];
      if (kMode != kTurn) {
#pragma unroll
        for (int i = 0; i < kSlots; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            w[i][0][e] = live[i] ? weights[kKind * p.head_dim + c0[i] + e] : 0.f;
            w[i][1][e] = live[i] ? weights[kKind * p.head_dim + c1[i] + e] : 0.f;
          }
      }
      const auto work = [&](Row& m) {
        if (!m.live) return;  // all lanes of the row
        float a0[kSlots][V], a1[kSlots][V], g0[kSlots][V], g1[kSlots][V];
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
          if (!live[i]) continue;
          widen<T, V>(m.a0[i], a0[i]);
          widen<T, V>(m.a1[i], a1[i]);
          if (kMode != kNormGrad) continue;
          widen<T, V>(m.g0[i], g0[i]);
          widen<T, V>(m.g1[i], g1[i]);
        }
        float rms = 1.f;
        if (kMode != kTurn) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < kSlots; ++i) {
            if (!live[i]) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) ss += a0[i][e] * a0[i][e] + a1[i][e] * a1[i][e];
          }
          rms = rsqrtf(row_sum(ss, p.lanes) * p.inv_dim + p.epsilon);
        }
        // turn of one slot's vectors in place; the pairs' values lie in y0, y1, or alternate
        const auto turn = [&](int i, float (&y0)[V], float (&y1)[V]) {
          if (!turned[i]) return;
          if (kInterleaved && V > 1) {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
              const float2 u = cs[i][e / 2], v = cs[i][V / 2 + e / 2];
              const float u0 = y0[e], u1 = y0[e + 1], v0 = y1[e], v1 = y1[e + 1];
              y0[e] = u0 * u.x - u1 * u.y;
              y0[e + 1] = u1 * u.x + u0 * u.y;
              y1[e] = v0 * v.x - v1 * v.y;
              y1[e + 1] = v1 * v.x + v0 * v.y;
            }
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float2 c = cs[i][e];
              const float u = y0[e], v = y1[e];
              y0[e] = u * c.x - v * c.y;
              y1[e] = v * c.x + u * c.y;
            }
          }
        };
        if (kMode == kNormGrad) {
          float along = 0.f;  // sum of g w x r
#pragma unroll
          for (int i = 0; i < kSlots; ++i) {
            if (!live[i]) continue;
            turn(i, g0[i], g1[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              a0[i][e] *= rms;
              a1[i][e] *= rms;
              const float d0 = g0[i][e] * a0[i][e], d1 = g1[i][e] * a1[i][e];
              dw[kKind][i][0][e] += d0;
              dw[kKind][i][1][e] += d1;
              g0[i][e] *= w[i][0][e];
              g1[i][e] *= w[i][1][e];
              along += g0[i][e] * a0[i][e] + g1[i][e] * a1[i][e];
            }
          }
          along = row_sum(along, p.lanes) * p.inv_dim;
#pragma unroll
          for (int i = 0; i < kSlots; ++i) {
            if (!live[i]) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
              a0[i][e] = rms * (g0[i][e] - a0[i][e] * along);
              a1[i][e] = rms * (g1[i][e] - a1[i][e] * along);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < kSlots; ++i) {
            if (!live[i]) continue;
            if (kMode == kNorm) {
#pragma unroll
              for (int e = 0; e < V; ++e) {
                a0[i][e] = a0[i][e] * rms * w[i][0][e];
                a1[i][e] = a1[i][e] * rms * w[i][1][e];
              }
            }
            turn(i, a0[i], a1[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
          if (!live[i]) continue;
          store<T, V>(h.out + c0[i], a0[i]);
          store<T, V>(h.out + c1[i], a1[i]);
        }
        h.out += h.out_step;
      };
      Row second;
      for (int n = 0; n < h.count; n += 2 * head_step) {
        fetch(h, second);
        work(first);
        fetch(h, first);
        work(second);
      }
    };
    const auto fetch_and_work = [&](auto which) {
      Heads h = heads_of(which);
      Row m;
      fetch(h, m);
      rows_of(which, h, m);
    };
    if constexpr (kQueriesAhead) {
      rows_of(std::integral_constant<int, 0>{}, heads[0], first[0]);
    } else {
      fetch_and_work(std::integral_constant<int, 0>{});
    }
    if constexpr (kAhead) {
      rows_of(std::integral_constant<int, 1>{}, heads[1], first[1]);
    } else {
      fetch_and_work(std::integral_constant<int, 1>{});
    }
  }

  if (kMode == kNormGrad) {
    // the workgroup's sums: rows of one wave by a butterfly over the lanes above the row's, then
    // the four waves, always in the same order
    float* sums = reinterpret_cast<float*>(table);  // [wave][2][head_dim]
    constexpr int kWaves = kThreads / 64;
    static_assert(sizeof(table) >= kWaves * 2 * kMaxHeadDim * sizeof(float), "the sums fit the table");
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < kSlots; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            for (int d = p.lanes; d < 64; d <<= 1) dw[k][i][c][e] += __shfl_xor(dw[k][i][c][e], d, 64);
          }
    __syncthreads();  // the table's last readers
    if ((tid & 63) < p.lanes) {
      float* mine = sums + (tid >> 6) * 2 * p.head_dim;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
          if (!live[i]) continue;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            mine[k * p.head_dim + c0[i] + e] = dw[k][i][0][e];
            mine[k * p.head_dim + c1[i] + e] = dw[k][i][1][e];
          }
        }
    }
    __syncthreads();
    for (int i = tid; i < 2 * p.head_dim; i += kThreads) {
      float sum = sums[i];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += sums[w * 2 * p.head_dim + i];
      p.parts[static_cast<int64_t>(blockIdx.x) * 2 * p.head_dim + i] = sum;
    }
  }
}

// dw[t][c] = sum over workgroups of parts[.][t][c], in fp64 (the sum itself is short).  One
// workgroup per 16 columns; 64 rows of threads take every 64th part, four loads in flight each, and
// are added up in pairs: 4 us for 1024 parts of 2 x 64, the latency of sixteen loads in a chain of four.
constexpr int kSumRows = 64;
__global__ void __launch_bounds__(1024) weight_sums_kernel(const float* parts, int n_parts, int head_dim, float* dq,
                                                           float* dk) {
  __shared__ double acc[kSumRows][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;
  const int64_t step = 2 * head_dim;
  double s = 0.0;
  if (col < 2 * head_dim) {
    int i = r;
    for (; i + 3 * kSumRows < n_parts; i += 4 * kSumRows) {
      float x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = parts[(i + k * kSumRows) * step + col];
#pragma unroll
      for (int k = 0; k < 4; ++k) s += x[k];
    }
    for (; i < n_parts; i += kSumRows) s += parts[i * step + col];
  }
  acc[r][c] = s;
  __syncthreads();
  for (int half = kSumRows / 2; half > 0; half /= 2) {
    if (r < half) acc[r][c] += acc[r + half][c];
    __syncthreads();
  }
  if (r != 0 || col >= 2 * head_dim) return;
  float* out = col < head_dim ? dq : dk;
  if (out != nullptr) out[col < head_dim ? col : col - head_dim] = static_cast<float>(acc[0][c]);
}

template <typename T, int V, Mode kMode>
void launch(bool interleaved, dim3 grid, hipStream_t stream, const RotaryArgs& p) {
  if (interleaved) {
    hipLaunchKernelGGL((rotary_kernel<T, V, true, kMode>), grid, dim3(kThreads), 0, stream, p);
  } else {
    hipLaunchKernelGGL((rotary_kernel<T, V, false, kMode>), grid, dim3(kThreads), 0, stream, p);
  }
}

template <typename T, Mode kMode>
void launch_vec(int vec, bool interleaved, dim3 grid, hipStream_t stream, const RotaryArgs& p) {
  if constexpr (sizeof(T) == 2 && kMode != kNormGrad) {
    if (vec == 8) return launch<T, 8, kMode>(interleaved, grid, stream, p);
  }
  if (vec == 4) return launch<T, 4, kMode>(interleaved, grid, stream, p);
  if (vec == 2) return launch<T, 2, kMode>(interleaved, grid, stream, p);
  return launch<T, 1, kMode>(interleaved, grid, stream, p);
}

// Tokens of a workgroup at a time, a power of two of at most the rows of its pass: as many as leave
// the chip four workgroups per CU, or one where fewer tokens would leave lanes without a head (24
// sequences of 78 tokens, 4 and 4 heads of 128: 7.5 us, always four per CU 19.7).
int tokens_of(const asc_rotary_t& a, int rows_per_pass) {
  const int64_t heads = a.q_heads > a.k_heads ? a.q_heads : a.k_heads;
  int n = rows_per_pass < kMaxTokens ? rows_per_pass : kMaxTokens;
  while (n > 1 && (a.seq <= n / 2 || a.batch * asc::ceil_div(a.seq, n) < (n * heads <= rows_per_pass ? 256 : 1024))) {
    n /= 2;
  }
  return n;
}

// Workgroups of a gradient launch, as its workspace counts them: each has a share of the tokens.
int64_t grad_parts(const asc_rotary_t& a) {
  return a.seq >= kMaxParts || a.batch * a.seq >= kMaxParts ? kMaxParts : a.batch * a.seq;
}

int32_t check(const asc_rotary_t* a, const char* what, Mode mode) {
  ASC_REQUIRE(a, ASC_ERR_INVALID_ARG, "%s: null arguments", what);
  ASC_REQUIRE(a->dtype == ASC_DT_FLOAT32 || a->dtype == ASC_DT_FLOAT16 || a->dtype == ASC_DT_BFLOAT16,
              ASC_ERR_UNSUPPORTED, "%s: dtype %d not supported (float32, float16, bfloat16)", what, a->dtype);
  ASC_REQUIRE(a->batch >= 0 && a->q_heads >= 0 && a->k_heads >= 0 && a->seq >= 0, ASC_ERR_INVALID_ARG,
              "%s: negative shape", what);
  ASC_REQUIRE(a->head_dim > 0 && a->head_dim % 2 == 0 && a->head_dim <= kMaxHeadDim, ASC_ERR_UNSUPPORTED,
              "%s: head_dim %d not supported (even, at most %d)", what, a->head_dim, kMaxHeadDim);
  ASC_REQUIRE(a->rotary_dim >= 0 && a->rotary_dim % 2 == 0 && a->rotary_dim <= a->head_dim, ASC_ERR_INVALID_ARG,
              "%s: rotary_dim %d must be even and at most head_dim %d", what, a->rotary_dim, a->head_dim);
  ASC_REQUIRE(a->q_heads <= 1 << 20 && a->k_heads <= 1 << 20, ASC_ERR_UNSUPPORTED, "%s: too many heads", what);
  ASC_REQUIRE(a->seq < int64_t{1} << 31 && a->batch < int64_t{1} << 31 &&
                  a->batch * asc::ceil_div(a->seq, kMinTokens) < int64_t{1} << 31,
              ASC_ERR_UNSUPPORTED, "%s: batch %lld x seq %lld too large", what, static_cast<long long>(a->batch),
              static_cast<long long>(a->seq));
  ASC_REQUIRE(mode == kTurn || a->epsilon >= 0.f, ASC_ERR_INVALID_ARG, "%s: epsilon must not be negative", what);
  if (a->batch == 0 || a->seq == 0 || a->q_heads + a->k_heads == 0) return ASC_OK;
  ASC_REQUIRE(a->rotary_dim == 0 || (a->positions && a->freqs), ASC_ERR_INVALID_ARG, "%s: null positions or freqs",
              what);
  for (int t = 0; t < 2; ++t) {
    if ((t ? a->k_heads : a->q_heads) == 0) continue;
    ASC_REQUIRE((t ? a->k.data : a->q.data) && (t ? a->k_out.data : a->q_out.data), ASC_ERR_INVALID_ARG,
                "%s: null buffer", what);
    if (mode == kTurn) continue;
    ASC_REQUIRE(t ? a->k_weight : a->q_weight, ASC_ERR_INVALID_ARG, "%s: null weight", what);
    ASC_REQUIRE(mode != kNormGrad || ((t ? a->dk_out.data : a->dq_out.data) && (t ? a->dk_weight : a->dq_weight)),
                ASC_ERR_INVALID_ARG, "%s: null gradient", what);
  }
  return ASC_OK;
}

// A result may lie in place of its own input, row by row (a lane reads its values of a row before it
// writes them), and shares no byte with another operand or result.  The weights' gradients are written by a
// launch of their own behind the one that reads the operands, so only other results are in their way.
int32_t check_places(const asc_rotary_t& a, const char* what, Mode mode) {
  const int64_t element = a.dtype == ASC_DT_FLOAT32 ? 4 : 2, weight = a.head_dim * static_cast<int64_t>(sizeof(float));
  const auto rows = [&](const char* name, const asc_rows_t& r, bool key) {
    return asc::region_of(name, r, a.batch, key ? a.k_heads : a.q_heads, a.seq, a.head_dim, element);
  };
  const bool grad = mode == kNormGrad;
  const asc_rows_t none{};
  const asc::Region results[] = {rows(grad ? "dq" : "q_out", a.q_out, false), rows(grad ? "dk" : "k_out", a.k_out, true)};
  const asc::Region of_q[] = {rows("q", a.q, false), rows("dq_out", grad ? a.dq_out : none, false)};
  const asc::Region of_k[] = {rows("k", a.k, true), rows("dk_out", grad ? a.dk_out : none, true)};
  const int64_t position = a.positions_int64 ? 8 : 4;
  const asc_rows_t at{const_cast<void*>(a.rotary_dim ? a.positions : nullptr), a.position_batch_stride, 0,
                      a.position_seq_stride};
  const asc::Region shared[] = {
      asc::region_of("positions", at, a.batch, 1, a.seq, 1, position),
      asc::region_of("freqs", a.freqs, a.rotary_dim / 2 * 8),
      asc::region_of("q_weight", mode != kTurn && a.q_heads ? a.q_weight : nullptr, weight),
      asc::region_of("k_weight", mode != kTurn && a.k_heads ? a.k_weight : nullptr, weight)};
  const asc::Region sums[] = {asc::region_of("dq_weight", grad ? a.dq_weight : nullptr, weight),
                              asc::region_of("dk_weight", grad ? a.dk_weight : nullptr, weight)};
  const auto apart = [&](const asc::Region& result, const asc::Region& other) {
    ASC_REQUIRE(!asc::overlap(result, other), ASC_ERR_INVALID_ARG, "%s: '%s' overlaps '%s'", what, result.name,
                other.name);
    return static_cast<int32_t>(ASC_OK);
  };
  int32_t rc = ASC_OK;
  for (int t = 0; t < 2; ++t) {
    const asc::Region& result = results[t];
    for (const asc::Region& x : t ? of_k : of_q) {
      if (!asc::same_place(result, x) && (rc = apart(result, x)) != ASC_OK) return rc;
    }
    for (const asc::Region& x : t ? of_q : of_k) {
      if ((rc = apart(result, x)) != ASC_OK) return rc;
    }
    for (const asc::Region& x : shared) {
      if ((rc = apart(result, x)) != ASC_OK) return rc;
    }
    for (const asc::Region& x : sums) {
      if ((rc = apart(result, x)) != ASC_OK) return rc;
    }
  }
  if ((rc = apart(results[0], results[1])) != ASC_OK) return rc;
  return apart(sums[0], sums[1]);
}

// The widest vector (16 bytes at most; four values in a gradient launch, whose two rows in flight and
// sums would not fit the registers of four waves per SIMD otherwise: 127 us against 105 at 4 x 4096 tokens of
// 32 + 8 heads, bf16) that
// every row's slots allow: both halves of a pair slot and every stride and address are multiples of it.
int vector_width(const asc_rotary_t& a, Mode mode) {
  const int64_t size = a.dtype == ASC_DT_FLOAT32 ? 4 : 2;
  const asc_rows_t* rows[] = {&a.q, &a.q_out, &a.dq_out, &a.k, &a.k_out, &a.dk_out};
  for (int v = mode == kNormGrad ? 4 : static_cast<int>(16 / size); v > 1; v /= 2) {
    bool ok = a.rotary_dim % (2 * v) == 0 && a.head_dim % (2 * v) == 0;
    for (int i = 0; i < 6; ++i) {
      if ((i < 3 ? a.q_heads : a.k_heads) == 0 || (i % 3 == 2 && mode != kNormGrad)) continue;
      ok = ok && reinterpret_cast<uintptr_t>(rows[i]->data) % (v * size) == 0 && rows[i]->batch_stride % v == 0 &&
           rows[i]->head_stride % v == 0 && rows[i]->seq_stride % v == 0;
    }
    if (ok) return v;
  }
  return 1;
}

void sum_weights(const asc_rotary_t& a, const float* parts, int n_parts, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(asc::ceil_div(2 * a.head_dim, 16)));
  hipLaunchKernelGGL(weight_sums_kernel, grid, dim3(1024), 0, stream, parts, n_parts, a.head_dim, a.dq_weight, a.dk_weight);
}

int32_t run(const asc_rotary_t* a, const char* what, Mode mode, float* parts, asc_stream_t stream) {
  const int32_t places = check_places(*a, what, mode);
  if (places != ASC_OK) return places;
  RotaryArgs p{};
  const auto rows = [](const asc_rows_t& r) { return Rows{r.data, r.batch_stride, r.head_stride, r.seq_stride}; };
  p.x[0] = rows(a->q);
  p.x[1] = rows(a->k);
  p.dy[0] = rows(a->dq_out);
  p.dy[1] = rows(a->dk_out);
  p.out[0] = rows(a->q_out);
  p.out[1] = rows(a->k_out);
  p.weight[0] = a->q_weight;
  p.weight[1] = a->k_weight;
  p.parts = parts;
  p.positions = a->positions;
  p.pos64 = a->positions_int64;
  p.pos_batch = a->position_batch_stride;
  p.pos_seq = a->position_seq_stride;
  p.freqs = a->freqs;
  p.seq = a->seq;
  p.q_heads = static_cast<int32_t>(a->q_heads);
  p.heads = static_cast<int32_t>(a->q_heads + a->k_heads);
  p.head_dim = a->head_dim;
  p.pairs = a->rotary_dim / 2;
  p.sign = mode == kNormGrad || (mode == kTurn && a->backward) ? -1.f : 1.f;
  p.magnitude = a->magnitude;
  p.epsilon = a->epsilon;
  p.inv_dim = 1.0f / static_cast<float>(a->head_dim);
  const int vec = vector_width(*a, mode);
  const int per_lane = vec >= 4 ? 1 : (vec == 2 ? 2 : 4);
  const int slots = static_cast<int>(asc::ceil_div(a->head_dim / (2 * vec), per_lane));
  p.lanes = 1;
  while (p.lanes < slots) p.lanes *= 2;  // at most 64: head_dim <= 512
  p.tokens = tokens_of(*a, kThreads / p.lanes);
  p.tiles = static_cast<uint32_t>(asc::ceil_div(a->seq, p.tokens));
  const int64_t n_tiles = a->batch * p.tiles;
  // Few tokens: their heads spread over workgroups of one pass each; else one workgroup for all.
  p.chunk_heads = p.heads;
  if (mode != kNormGrad && n_tiles < 2 * 256) {
    const int per_pass = kThreads / p.lanes / p.tokens;
    p.chunk_heads = per_pass < 1 ? 1 : (per_pass < p.heads ? per_pass : p.heads);
  }
  p.chunks = static_cast<uint32_t>(asc::ceil_div(p.heads, p.chunk_heads));
  p.units = static_cast<uint32_t>(n_tiles * p.chunks);  // chunks > 1 only where n_tiles is small
  int64_t blocks = p.units;
  const int64_t most = mode == kNormGrad ? grad_parts(*a) : int64_t{1} << 23;  // the kernel strides over the rest
  if (blocks > most) blocks = most;
  const dim3 grid(static_cast<uint32_t>(blocks));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool inter = a->interleaved != 0;
  const auto go = [&](auto tag) {
    using T = decltype(tag);
    if (mode == kTurn) return launch_vec<T, kTurn>(vec, inter, grid, s, p);
    if (mode == kNorm) return launch_vec<T, kNorm>(vec, inter, grid, s, p);
    return launch_vec<T, kNormGrad>(vec, inter, grid, s, p);
  };
  if (a->dtype == ASC_DT_FLOAT32) {
    go(float{});
  } else if (a->dtype == ASC_DT_FLOAT16) {
    go(_Float16{});
  } else {
    go(__bf16{});
  }
  if (mode == kNormGrad) {
    const int32_t rc = asc::check_launch(what);
    if (rc != ASC_OK) return rc;
    sum_weights(*a, parts, static_cast<int>(blocks), s);
  }
  return asc::check_launch(what);
}

bool empty(const asc_rotary_t& a) { return a.batch == 0 || a.seq == 0 || a.q_heads + a.k_heads == 0; }

}  // namespace

extern "C" int32_t asc_rotary(const asc_rotary_t* args, asc_stream_t stream) {
  const int32_t rc = check(args, "asc_rotary", kTurn);
  if (rc != ASC_OK || empty(*args)) return rc;
  return run(args, "asc_rotary", kTurn, nullptr, stream);
}

extern "C" int32_t asc_qk_norm_rotary(const asc_rotary_t* args, asc_stream_t stream) {
  const int32_t rc = check(args, "asc_qk_norm_rotary", kNorm);
  if (rc != ASC_OK || empty(*args)) return rc;
  return run(args, "asc_qk_norm_rotary", kNorm, nullptr, stream);
}

extern "C" int64_t asc_qk_norm_rotary_bwd_workspace(const asc_rotary_t* args) {
  if (check(args, "asc_qk_norm_rotary_bwd_workspace", kTurn) != ASC_OK || empty(*args)) return 0;
  return grad_parts(*args) * 2 * args->head_dim * static_cast<int64_t>(sizeof(float));
}

extern "C" int32_t asc_qk_norm_rotary_bwd(const asc_rotary_t* args, void* workspace, int64_t workspace_bytes,
                                          asc_stream_t stream) {
  const int32_t rc = check(args, "asc_qk_norm_rotary_bwd", kNormGrad);
  if (rc != ASC_OK) return rc;
  if (empty(*args)) {  // no rows: the weights' gradients are zeros
    if (args->dq_weight == nullptr && args->dk_weight == nullptr) return ASC_OK;
    const int32_t places = check_places(*args, "asc_qk_norm_rotary_bwd", kNormGrad);
    if (places != ASC_OK) return places;
    sum_weights(*args, nullptr, 0, static_cast<hipStream_t>(stream));
    return asc::check_launch("asc_qk_norm_rotary_bwd");
  }
  const int64_t need = grad_parts(*args) * 2 * args->head_dim * static_cast<int64_t>(sizeof(float));
  ASC_REQUIRE(workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 4 == 0,
              ASC_ERR_INVALID_ARG, "asc_qk_norm_rotary_bwd: the workspace must hold %lld bytes",
              static_cast<long long>(need));
  return run(args, "asc_qk_norm_rotary_bwd", kNormGrad, static_cast<float*>(workspace), stream);
}
