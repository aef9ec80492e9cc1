// Logits before a token is chosen: penalties for tokens of the row's history, a bias, a grammar's
// mask (asc_process_logits).
//
// A workgroup owns a slice of one row's vocabulary.  It counts the history's tokens that fall into the
// slice in LDS (integers: the order does not matter), then takes the slice through the formula.  The
// whole history is read for every slice, from L2 after the first.  HBM bounds large calls: 64 rows of 131072 fp32
// logits with masks: 70.7 MB in 14.1 us (5.0 TB/s), in 16 to 17.3 us with 8000 tokens of history; the launch small ones (4 us).
#include "common.h"
#include "logits_slices.h"
#include "numeric.h"
#include "overlap.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct LogitsArgs {
  const void* logits;
  void* out;
  int64_t logits_stride, out_stride;
  const void* history;
  int64_t history_stride;
  const int32_t* lengths;
  const int32_t* prompts;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const float* bias;
  int64_t bias_stride;
  const uint32_t* mask;
  int64_t mask_stride;
  int32_t history_int64, vocab, width, slices;
};

struct F32 {
  typedef float Stored;
  static __device__ __forceinline__ float load(float x) { return x; }
  static __device__ __forceinline__ float store(float x) { return x; }
};
struct F16 {
  typedef uint16_t Stored;
  static __device__ __forceinline__ float load(uint16_t x) { return asc::f16_to_f32(x); }
  static __device__ __forceinline__ uint16_t store(float x) { return asc::f32_to_f16_rne(x); }
};
struct Bf16 {
  typedef uint16_t Stored;
  static __device__ __forceinline__ float load(uint16_t x) { return asc::bf16_to_f32(x); }
  static __device__ __forceinline__ uint16_t store(float x) { return asc::f32_to_bf16_rne(x); }
};

constexpr uint32_t kInPrompt = 0x80000000u;  // beside the count of a token behind the prompt

// Tokens of the history that a thread has under way: one at a time, each waits for memory alone.
constexpr int kAhead = 8;

// add(i, token) for the history's first n tokens; what is no uint32 becomes one that no vocabulary has.
template <int kThreads, class T, class F>
__device__ __forceinline__ void for_history(const T* history, int n, const F& add) {
  for (int base = threadIdx.x; base < n; base += kThreads * kAhead) {
    T token[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = base + k * kThreads;
      token[k] = history[i < n ? i : base];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = base + k * kThreads;
      const bool fits = sizeof(T) == 4 || static_cast<uint64_t>(token[k]) >> 32 == 0;
      if (i < n) add(i, fits ? static_cast<uint32_t>(token[k]) : ~0u);
    }
  }
}

// kPerThread tokens per thread.  kVec: the rows of logits and out lie at the same offset from 16
// bytes, so vectors of the slice do, `lead` elements before the row's first; else element by element.
template <class E, bool kVec, int kThreads, int kPerThread>
__global__ void __launch_bounds__(kThreads) process_logits(LogitsArgs p) {
  typedef typename E::Stored S;
  constexpr int V = kVec ? 16 / sizeof(S) : 1;
  constexpr int kSlice = kThreads * kPerThread;
  constexpr int kVecs = kPerThread / V;
  __shared__ uint32_t counts[kSlice];
  const int tid = threadIdx.x;
  const uint32_t row = blockIdx.x / p.slices, slice = blockIdx.x - row * p.slices;
  const S* x = static_cast<const S*>(p.logits) + row * p.logits_stride;
  S* y = static_cast<S*>(p.out) + row * p.out_stride;
  const int lead = kVec ? static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(S)) : 0;
  const int first = asc::slice_first(static_cast<int>(slice), kSlice, lead);  // token of counts[0]
  const uint32_t here = asc::slice_places(first, kSlice, p.vocab);
  if (here == 0) return;  // all of the workgroup
  // vectors that lie in the row are taken whole; `some`, the row's first, is read in place of the others
  const int some = lead == 0 ? 0 : V - lead;
  const bool vectors = kVec && some + V <= p.vocab;
  const auto inside = [&](int token) { return token >= 0 && token + V <= p.vocab; };

  const float* bias = p.bias ? p.bias + row * p.bias_stride : nullptr;
  const uint32_t* mask = p.mask ? p.mask + row * p.mask_stride : nullptr;

  const int length = p.lengths[row];
  const bool bad = length < 0 || length > p.width;
  const int n = bad ? 0 : length;
  const int prompt = p.prompts ? p.prompts[row] : 0;

#pragma unroll
  for (int i = 0; i < kSlice / 4 / kThreads; ++i) {
    reinterpret_cast<u32x4*>(counts)[tid + i * kThreads] = u32x4{0, 0, 0, 0};
  }
  __syncthreads();
  const auto count = [&](int i, uint32_t token) {
    // what is counted before the row's first token is looked at by nobody
    const uint32_t at = token - static_cast<uint32_t>(first);
    if (at >= here) return;
    if (i < prompt) {
      atomicOr(&counts[at], kInPrompt);
    } else {
      atomicAdd(&counts[at], 1u);
    }
  };
  if (p.history_int64) {
    for_history<kThreads>(static_cast<const int64_t*>(p.history) + row * p.history_stride, n, count);
  } else {
    for_history<kThreads>(static_cast<const int32_t*>(p.history) + row * p.history_stride, n, count);
  }
  __syncthreads();

  const float repetition = p.repetition ? p.repetition[row] : 1.0f;
  const float frequency = p.frequency ? p.frequency[row] : 0.0f;
  const float presence = p.presence ? p.presence[row] : 0.0f;
  const auto process = [&](uint32_t c, float v, float add, bool allowed) {
    if (c != 0) {
      v = v > 0.0f ? v / repetition : v * repetition;
      const float times = static_cast<float>(c & ~kInPrompt);
      v = v - frequency * times;
      if (times > 0.0f) v = v - presence;
    }
    if (bias) v = v + add;
    if (bad) v = __builtin_nanf("");
    return allowed ? v : -INFINITY;
  };
  const auto allowed = [&](int token) { return !mask || ((mask[token >> 5] >> (token & 31)) & 1); };
  if constexpr (kVec) {
    if (vectors) {
      u32x4 held[kVecs];
      float add[kVecs][V];
      uint64_t bits[kVecs];
      const bool bias_vec = ((reinterpret_cast<uintptr_t>(bias) >> 2) + some) % 4 == 0;
#pragma unroll
      for (int it = 0; it < kVecs; ++it) {
        int token = first + (tid + it * kThreads) * V;
        token = inside(token) ? token : some;
        held[it] = *reinterpret_cast<const u32x4*>(x + token);
        if (bias) {
          if (bias_vec) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
              *reinterpret_cast<f32x4*>(&add[it][e]) = *reinterpret_cast<const f32x4*>(bias + token + e);
            }
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) add[it][e] = bias[token + e];
          }
        }
        bits[it] = ~0ull;
        if (mask) {
          // both words are the same one, unless the vector lies across two
          bits[it] = (static_cast<uint64_t>(mask[(token + V - 1) >> 5]) << 32 | mask[token >> 5]) >> (token & 31);
        }
      }
#pragma unroll
      for (int it = 0; it < kVecs; ++it) {
        const int at = (tid + it * kThreads) * V;
        S in[V], out[V];
        uint32_t c[V];
        *reinterpret_cast<u32x4*>(in) = held[it];
#pragma unroll
        for (int e = 0; e < V; e += 4) *reinterpret_cast<u32x4*>(&c[e]) = *reinterpret_cast<const u32x4*>(&counts[at + e]);
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = E::store(process(c[e], E::load(in[e]), add[it][e], bits[it] >> e & 1));
        if (inside(first + at)) *reinterpret_cast<u32x4*>(y + first + at) = *reinterpret_cast<u32x4*>(out);
      }
    }
  }
  // element by element: the row's ends, or all of it
  for (int at = tid * V; at < kSlice; at += kThreads * V) {
    const int token = first + at;
    if (token >= p.vocab) break;
    if (vectors && inside(token)) continue;
    for (int e = 0; e < V; ++e) {
      const int t = token + e;
      if (t < 0 || t >= p.vocab) continue;
      y[t] = E::store(process(counts[at + e], E::load(x[t]), bias ? bias[t] : 0.0f, allowed(t)));
    }
  }
}

// Workgroups of many threads read the history in few rounds and few times: 64 rows of 131072 fp32 logits with 8000 tokens
// of history 17.3 us with 1024 threads and 16384 tokens, 18.8 with 256 and 4096, 21.3 with 256 and 2048.  The last where
// the large would not fill the chip (16 rows: 9.3 us, 10.4 large; 32 rows: 13.2, 12.0) and the history is no longer than what
// reading it that often costs (4 rows, 30000 tokens: 13.1, 11.1 large).
constexpr int kLargeThreads = 1024, kLarge = 16384, kSmallThreads = 256, kSmall = 2048;
constexpr int64_t kFewGroups = 256, kLongHistory = 16384;

template <class E, bool kVec>
void launch(const LogitsArgs& p, int64_t rows, bool small, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(rows * p.slices));
  if (small) {
    hipLaunchKernelGGL((process_logits<E, kVec, kSmallThreads, kSmall / kSmallThreads>), grid, dim3(kSmallThreads), 0, stream,
                       p);
  } else {
    hipLaunchKernelGGL((process_logits<E, kVec, kLargeThreads, kLarge / kLargeThreads>), grid, dim3(kLargeThreads), 0, stream,
                       p);
  }
}

}  // namespace

extern "C" int32_t asc_process_logits(const asc_logits_t* a, asc_stream_t stream) {
  const char* what = "asc_process_logits";
  ASC_REQUIRE(a, ASC_ERR_INVALID_ARG, "%s: null arguments", what);
  ASC_REQUIRE(a->dtype == ASC_DT_FLOAT32 || a->dtype == ASC_DT_FLOAT16 || a->dtype == ASC_DT_BFLOAT16,
              ASC_ERR_UNSUPPORTED, "%s: dtype %d not supported (float32, float16, bfloat16)", what, a->dtype);
  ASC_REQUIRE(a->rows >= 0 && a->vocab >= 0 && a->history_width >= 0, ASC_ERR_INVALID_ARG, "%s: negative shape", what);
  if (a->rows == 0 || a->vocab == 0) return ASC_OK;
  ASC_REQUIRE(a->vocab < 1 << 30 && a->history_width < 1 << 30, ASC_ERR_UNSUPPORTED, "%s: shape too large", what);
  ASC_REQUIRE(a->logits && a->out && a->history_lengths && (a->history || a->history_width == 0), ASC_ERR_INVALID_ARG,
              "%s: null buffer", what);
  const int64_t size = a->dtype == ASC_DT_FLOAT32 ? 4 : 2;
  ASC_REQUIRE(((reinterpret_cast<uintptr_t>(a->logits) | reinterpret_cast<uintptr_t>(a->out)) & (size - 1)) == 0,
              ASC_ERR_ALIGNMENT, "%s: logits and out must be aligned to their elements", what);
  const auto rows = [&](const char* name, const void* data, int64_t stride, int64_t row, int64_t element) {
    return asc::region_of(name, asc_rows_t{const_cast<void*>(data), stride, 0, 0}, a->rows, 1, 1, row, element);
  };
  const asc::Region out = rows("out", a->out, a->out_stride, a->vocab, size);
  const asc::Region logits = rows("logits", a->logits, a->logits_stride, a->vocab, size);
  const asc::Region operands[] = {
      rows("history", a->history, a->history_stride, a->history_width, a->history_int64 ? 8 : 4),
      asc::region_of("history_lengths", a->history_lengths, a->rows * 4),
      asc::region_of("prompt_lengths", a->prompt_lengths, a->rows * 4),
      asc::region_of("repetition", a->repetition, a->rows * 4),
      asc::region_of("frequency", a->frequency, a->rows * 4),
      asc::region_of("presence", a->presence, a->rows * 4),
      rows("bias", a->bias, a->bias_stride, a->vocab, 4),
      rows("mask", a->mask, a->mask_stride, asc::ceil_div(a->vocab, 32), 4)};
  ASC_REQUIRE(asc::same_place(out, logits) || !asc::overlap(out, logits), ASC_ERR_INVALID_ARG, "%s: 'out' overlaps '%s'",
              what, "logits");
  for (const asc::Region& r : operands) {
    ASC_REQUIRE(!asc::overlap(out, r), ASC_ERR_INVALID_ARG, "%s: 'out' overlaps '%s'", what, r.name);
  }
  LogitsArgs p{};
  p.logits = a->logits;
  p.out = a->out;
  p.logits_stride = a->logits_stride;
  p.out_stride = a->out_stride;
  p.history = a->history;
  p.history_stride = a->history_stride;
  p.history_int64 = a->history_int64;
  p.lengths = a->history_lengths;
  p.prompts = a->prompt_lengths;
  p.repetition = a->repetition;
  p.frequency = a->frequency;
  p.presence = a->presence;
  p.bias = a->bias;
  p.bias_stride = a->bias_stride;
  p.mask = reinterpret_cast<const uint32_t*>(a->mask);
  p.mask_stride = a->mask_stride;
  p.vocab = static_cast<int32_t>(a->vocab);
  p.width = static_cast<int32_t>(a->history_width);
  // room for the lead of rows that do not begin at 16 bytes
  const bool aligned = asc::aligned16(a->logits) && (a->rows == 1 || a->logits_stride * size % 16 == 0);
  const auto slices = [&](int of) { return asc::slices_of(a->vocab, of, static_cast<int>(size), aligned); };
  const bool small = a->rows * slices(kLarge) < kFewGroups && a->history_width <= kLongHistory;
  p.slices = static_cast<int32_t>(slices(small ? kSmall : kLarge));
  ASC_REQUIRE(a->rows * p.slices < int64_t{1} << 22, ASC_ERR_UNSUPPORTED, "%s: %lld workgroups exceed the launch grid limit",
              what, static_cast<long long>(a->rows * p.slices));
  const uintptr_t apart = reinterpret_cast<uintptr_t>(a->logits) ^ reinterpret_cast<uintptr_t>(a->out);
  const int64_t steps = a->rows > 1 ? (a->logits_stride - a->out_stride) * size : 0;
  const bool vec = ((apart | static_cast<uintptr_t>(steps)) & 15) == 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == ASC_DT_FLOAT32) {
    vec ? launch<F32, true>(p, a->rows, small, s) : launch<F32, false>(p, a->rows, small, s);
  } else if (a->dtype == ASC_DT_FLOAT16) {
    vec ? launch<F16, true>(p, a->rows, small, s) : launch<F16, false>(p, a->rows, small, s);
  } else {
    vec ? launch<Bf16, true>(p, a->rows, small, s) : launch<Bf16, false>(p, a->rows, small, s);
  }
  return asc::check_launch(what);
}
