// What a sampler does to the logits of a step before it picks a token: penalties for tokens that were seen, biases of
// single tokens, a grammar's mask.  Per row and token
//   x = x > 0 ? x / r : x r   if the token occurs in the row's history,
//   x = x - f c - [c > 0] p   c: its occurrences behind the prompt,
//   x = x + (sum of its biases, in list order),   x = -inf unless the mask allows it.
//
// Bound by HBM: the logits are read once and written once (64 rows of 151936 in fp32, 8192 ids each: 25 us = 3.4 TB/s, of which
// the walk over the ids, before the first store, is about a third); a launch at few rows (1 row: kernel 4.6 us).  A workgroup takes a slice of one row's
// vocabulary and keeps what it has to know of a token - seen, has a bias, occurrences - in one LDS word per token,
// filled by a walk over the row's history with integer LDS atomics (whatever their order, the counts are the same), so the
// dense pass touches LDS and the logits only, and no table of counts travels through memory.  Every slice of a row
// walks the whole history: slices are made as large as LDS and an even spread over the device allow.
#include "common.hpp"

#include <type_traits>

namespace axhip {
namespace {

constexpr int kThreads = 1024;
constexpr int kAhead = 4;        // loads of a thread on their way at a time
constexpr int kMostLds = 96 * 1024;
constexpr int kMostBias = 16384;  // every biased token walks the list

struct LogitsArgs {
  const void *x;
  void *out;
  int64_t x_stride, out_stride;
  const void *history;
  int64_t hist_row, hist_token;  // strides in elements
  int max_history;
  const int32_t *hist_len, *prompt_len;
  const float *repetition, *presence, *frequency;
  const int32_t *bias_ids;
  const float *bias;
  int bias_count;
  const uint32_t *allowed;
  int64_t allowed_stride;
  int vocab, slice;  // tokens per workgroup, a multiple of 64
};

extern __shared__ __attribute__((aligned(16))) unsigned char logits_smem[];

// The word of a token: the two highest bits say that it was seen and that it has a bias, the others count it.
template <typename CT>
struct Word {
  static constexpr uint32_t kBits = sizeof(CT) * 8;
  static constexpr uint32_t kSeen = 1u << (kBits - 1), kBias = 1u << (kBits - 2), kCount = kBias - 1;
  static __device__ __forceinline__ void set(int i, uint32_t bit) {
    uint32_t *w = reinterpret_cast<uint32_t *>(logits_smem);
    if constexpr (sizeof(CT) == 2) atomicOr(w + (i >> 1), bit << ((i & 1) * 16));
    else atomicOr(w + i, bit);
  }
  static __device__ __forceinline__ void count(int i) {
    uint32_t *w = reinterpret_cast<uint32_t *>(logits_smem);
    if constexpr (sizeof(CT) == 2) atomicAdd(w + (i >> 1), 1u << ((i & 1) * 16));
    else atomicAdd(w + i, 1u);
  }
};

// The biases of token `id` of a row in list order: 64 entries a step over the lanes of the wavefront.
__device__ __forceinline__ float bias_of(const int32_t *ids, const float *values, int n, int id, int lane) {
  float sum = 0.f;
  for (int j = 0; j < n; j += 64) {
    const int at = j + lane;
    const bool hit = at < n && ids[at] == id;
    const float v = hit ? values[at] : 0.f;
    for (uint64_t m = __ballot(hit); m; m &= m - 1)
      sum += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), __ffsll(static_cast<unsigned long long>(m)) - 1));
  }
  return sum;
}

template <typename T, typename I, typename CT, int V>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a) {
  using W = Word<CT>;
  using S = typename std::conditional<sizeof(T) == 2, _Float16, float>::type;
  typedef S vec __attribute__((ext_vector_type(V)));
  const int tid = threadIdx.x, lane = tid & 63;
  const int row = blockIdx.y, v0 = blockIdx.x * a.slice, v1 = min(v0 + a.slice, a.vocab);
  const int n = v1 - v0;
  const bool marked = a.history || a.bias_count > 0;  // uniform
  if (marked) {
    u32x4_t *w = reinterpret_cast<u32x4_t *>(logits_smem);
    for (int i = tid; i < a.slice * static_cast<int>(sizeof(CT)) / 16; i += kThreads) w[i] = u32x4_t{0, 0, 0, 0};
    __syncthreads();
    if (a.history) {
      const int len = a.hist_len ? min(max(a.hist_len[row], 0), a.max_history) : a.max_history;
      const int prompt = a.prompt_len ? max(a.prompt_len[row], 0) : 0;
      const I *ids = static_cast<const I *>(a.history) + row * a.hist_row;
      for (int t0 = tid; t0 < len; t0 += kThreads * kAhead) {
        int64_t id[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) id[u] = ids[min(t0 + u * kThreads, len - 1) * a.hist_token];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int t = t0 + u * kThreads;
          const int64_t at = id[u] - v0;
          if (t < len && at >= 0 && at < n) {
            if (t >= prompt) W::count(static_cast<int>(at));  // (a count says that the token was seen, too)
            else W::set(static_cast<int>(at), W::kSeen);
          }
        }
      }
    }
    const int32_t *bids = a.bias_ids + static_cast<int64_t>(row) * a.bias_count;
    for (int j = tid; j < a.bias_count; j += kThreads) {
      const int64_t id = static_cast<int64_t>(bids[j]) - v0;
      if (id >= 0 && id < n) W::set(static_cast<int>(id), W::kBias);
    }
    __syncthreads();
  }
  const float r = a.repetition ? a.repetition[row] : 1.f;
  const float f = a.frequency ? a.frequency[row] : 0.f;
  const float p = a.presence ? a.presence[row] : 0.f;
  const S *x = static_cast<const S *>(a.x) + row * a.x_stride;
  S *y = static_cast<S *>(a.out) + row * a.out_stride;
  const CT *words = reinterpret_cast<const CT *>(logits_smem);
  const uint32_t *allowed = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  // Whole wavefronts stay in the loop: the search for a bias is theirs together.
  for (int i0 = 0; i0 < n; i0 += kThreads * V * kAhead) {
    vec in[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + (u * kThreads + tid) * V;  // (a slice ends on a multiple of V, and so does the vocabulary where V > 1)
      in[u] = {};
      if (i < n) in[u] = *reinterpret_cast<const vec *>(x + v0 + i);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + (u * kThreads + tid) * V;
      const bool on = i < n;
      float val[V];
      uint32_t word[V];
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        val[j] = static_cast<float>(in[u][j]);
        word[j] = marked && on ? words[i + j] : 0u;
        any |= word[j];
      }
      if (__any(any != 0)) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const uint32_t c = word[j] & W::kCount;
          if (word[j] & (W::kSeen | W::kCount)) val[j] = val[j] > 0.f ? val[j] / r : val[j] * r;
          if (c) val[j] = (val[j] - f * static_cast<float>(c)) - p;
          for (uint64_t m = __ballot((word[j] & W::kBias) != 0); m; m &= m - 1) {
            const int l = __ffsll(static_cast<unsigned long long>(m)) - 1;
            const float b = bias_of(a.bias_ids + static_cast<int64_t>(row) * a.bias_count,
                                    a.bias + static_cast<int64_t>(row) * a.bias_count, a.bias_count,
                                    v0 + __builtin_amdgcn_readlane(i, l) + j, lane);
            if (lane == l) val[j] += b;
          }
        }
      }
      if (on) {
        if (allowed) {
          const uint32_t bits = allowed[(v0 + i) >> 5] >> ((v0 + i) & 31);
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (!((bits >> j) & 1u)) val[j] = -__builtin_inff();
        }
        vec o;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = static_cast<S>(val[j]);
        *reinterpret_cast<vec *>(y + v0 + i) = o;
      }
    }
  }
}

template <typename T, typename I, typename CT>
int launch(LogitsArgs a, int rows, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = a.vocab % V == 0 && a.x_stride % V == 0 && a.out_stride % V == 0 &&
                    ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0;
  // Slices: about one workgroup per CU over all rows, at least 2048 tokens each, at most what 96 KB of words hold.  (64 rows,
  // 8192 int64 ids each in a [steps, rows] log: 26 us; two workgroups per CU 29 us, since every slice walks the history.)
  const int most = kMostLds / static_cast<int>(sizeof(CT)), least = 2048;
  const int64_t want = (device_cu_count() + rows - 1) / rows;
  int64_t slice = (a.vocab + want - 1) / want;
  slice = slice < least ? least : (slice > most ? most : slice);
  a.slice = static_cast<int>((slice + 63) / 64 * 64);
  const dim3 grid(static_cast<unsigned>((a.vocab + a.slice - 1) / a.slice), static_cast<unsigned>(rows));
  const unsigned lds = static_cast<unsigned>(a.slice) * sizeof(CT);
  static std::atomic<uint64_t> raised[2];
  const void *kernel = wide ? reinterpret_cast<const void *>(&logits_kernel<T, I, CT, V>) : reinterpret_cast<const void *>(&logits_kernel<T, I, CT, 1>);
  const int rc = raise_dynamic_lds(kernel, kMostLds, raised[wide]);
  if (rc != AXHIP_OK) return rc;
  if (wide) hipLaunchKernelGGL((logits_kernel<T, I, CT, V>), grid, dim3(kThreads), lds, st, a);
  else hipLaunchKernelGGL((logits_kernel<T, I, CT, 1>), grid, dim3(kThreads), lds, st, a);
  return launch_status();
}

template <typename T, typename I>
int launch(const LogitsArgs &a, int rows, hipStream_t st) {
  // 14 bits of a 16-bit word count the occurrences
  return a.max_history < (1 << 14) ? launch<T, I, uint16_t>(a, rows, st) : launch<T, I, uint32_t>(a, rows, st);
}

}  // namespace
}  // namespace axhip

using namespace axhip;

extern "C" {

AXHIP_API int axhip_logits_process(const void *logits, int64_t logits_stride, int dtype, const void *history,
                                   int history_dtype, int64_t history_row_stride, int64_t history_token_stride,
                                   int max_history, const int32_t *history_len, const int32_t *prompt_len,
                                   const float *repetition, const float *presence, const float *frequency,
                                   const int32_t *bias_ids, const float *bias, int bias_count, const uint32_t *allowed,
                                   int64_t allowed_stride, void *out, int64_t out_stride, int rows, int vocab,
                                   axhip_stream stream) {
  if (!is_float_dtype(dtype)) return AXHIP_UNSUPPORTED_TYPE;
  if (history && history_dtype != AXHIP_INT32 && history_dtype != AXHIP_INT64) return AXHIP_UNSUPPORTED_TYPE;
  if (rows < 0 || rows > 65535 || vocab < 0 || vocab > (1 << 30) || max_history < 0 || max_history >= (1 << 30) || bias_count < 0 ||
      bias_count > kMostBias)
    return AXHIP_INVALID_ARGUMENT;
  if (logits_stride < vocab || out_stride < vocab || history_row_stride < 0 || history_token_stride < 0) return AXHIP_INVALID_ARGUMENT;
  if (allowed && allowed_stride < (static_cast<int64_t>(vocab) + 31) / 32) return AXHIP_INVALID_ARGUMENT;
  if (rows == 0 || vocab == 0) return AXHIP_OK;
  if (!logits || !out || (bias_count > 0 && (!bias_ids || !bias))) return AXHIP_INVALID_PTR;
  if (logits == out && logits_stride != out_stride) return AXHIP_INVALID_ARGUMENT;
  const uintptr_t esz = dtype == AXHIP_FLOAT16 ? 2 : 4, hsz = history_dtype == AXHIP_INT64 ? 8 : 4;
  const auto at = [](const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (!at(logits, esz) || !at(out, esz) || (history && !at(history, hsz)) || !at(history_len, 4) || !at(prompt_len, 4) ||
      !at(repetition, 4) || !at(presence, 4) || !at(frequency, 4) || !at(bias_ids, 4) || !at(bias, 4) || !at(allowed, 4))
    return AXHIP_INVALID_PTR;
  LogitsArgs a{};
  a.x = logits;
  a.out = out;
  a.x_stride = logits_stride;
  a.out_stride = out_stride;
  a.history = max_history > 0 ? history : nullptr;
  a.hist_row = history_row_stride;
  a.hist_token = history_token_stride;
  a.max_history = max_history;
  a.hist_len = history_len;
  a.prompt_len = prompt_len;
  a.repetition = repetition;
  a.presence = presence;
  a.frequency = frequency;
  a.bias_ids = bias_ids;
  a.bias = bias;
  a.bias_count = bias_count;
  a.allowed = allowed;
  a.allowed_stride = allowed_stride;
  a.vocab = vocab;
  hipStream_t st = as_stream(stream);
  const bool wide_ids = history_dtype == AXHIP_INT64;
  if (dtype == AXHIP_FLOAT16) return wide_ids ? launch<__half, int64_t>(a, rows, st) : launch<__half, int32_t>(a, rows, st);
  return wide_ids ? launch<float, int64_t>(a, rows, st) : launch<float, int32_t>(a, rows, st);
}

}  // extern "C"
