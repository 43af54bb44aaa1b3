// Rotary position embedding by a frequency table, alone (axhip_rotary_qk) and on the way into a paged KV cache
// (axhip_rotary_append_paged: norm of each q / k head, rotation, k and v rows into their pages, for a ragged batch).
//
// Pair i (i < rotary_dim / 2) of a head is (x_i, x_{i + rotary_dim/2}) or, interleaved, (x_{2i}, x_{2i+1}); it turns by
// a = pos * f_i:  y0 = s (x0 cos a - x1 sin a), y1 = s (x1 cos a + x0 sin a); elements behind rotary_dim are copied.
//
// The angle of a far position needs more than 32 bits: pos * f in fp32 is off by pos * 2^-24 radians (0.03 at 2^19).
// It is formed in fp64 as a number of turns, whole turns are dropped, and what is left - below half a turn - goes to sincosf in
// fp32; the r that this cuts off (up to 2^-23) comes back as cos a - r sin a, sin a + r cos a.  One angle per (token, pair), shared by
// the heads: a few fp64 instructions per token and lane.
//
// Both kernels are bound by HBM (every element is read once and written once: 33001 rows of 24 heads of 128 in fp32 136 us =
// 6.0 TB/s, 65536 such rows with norm into fp16 pages 285 us = 5.7 TB/s, a plain copy 5.1 TB/s), by the launch when rows are
// few (kernels of 4 to 6 us up to some hundred rows).
// One wavefront takes one token and a run of its heads.  A lane holds V elements of a head and their V partners, V * esz =
// 16 bytes where sizes and alignment allow: both loads of a wavefront are then contiguous over the lanes of a head, and
// the partner never has to cross lanes.  Its cosines and sines stay in registers for all heads of the token; they are
// computed one pair per lane and spread through a strip of LDS that only this wavefront uses.
#include "common.hpp"

#include <cmath>
#include <type_traits>

namespace axhip {
namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
constexpr int kMaxPairs = 256;   // rotary_dim <= 512
constexpr int kPageShift = 7;    // 128 keys per page
constexpr int64_t kMostRows = int64_t(1) << 25;  // of a launch: 2^32 threads are too many

struct RotaryArgs {
  const void *x[3];       // q, k, v rows
  int64_t stride[3];      // elements between rows
  void *out[3];           // q_out [rows, heads, D]; k_out likewise, or the pools [n_pages, Hkv, 128, D]
  int heads[3];           // heads[2] = 0 without a cache
  const int64_t *pos;     // [rows] or [3, rows], null: the position in the cache
  const float *inv_freq;  // [rotary_dim / 2]
  const void *w[2];       // norm weights of q and k heads [D] or null
  int w_f16, norm;
  float eps, scale;
  int64_t first, end, rows;  // rows of this launch; all rows
  int dim, rotary_dim, interleaved, axes, h_lim, w_lim;
  int lanes_shift;        // log2 of the lanes a head is spread over
  int groups, heads_per_group;
  // paged form
  const int32_t *cu, *start, *page_table;
  int B, max_pages, n_pages;
};

template <typename T>
using Elem = typename std::conditional<sizeof(T) == 2, _Float16, float>::type;

template <typename T, int V>
__device__ __forceinline__ void load_v(const T *p, float (&f)[V]) {
  typedef Elem<T> vec __attribute__((ext_vector_type(V)));
  const vec x = __builtin_nontemporal_load(reinterpret_cast<const vec *>(p));
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = static_cast<float>(x[j]);
}
template <bool STREAM, typename T, int V>
__device__ __forceinline__ void store_v(T *p, const float (&f)[V]) {
  typedef Elem<T> vec __attribute__((ext_vector_type(V)));
  vec x;
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = static_cast<Elem<T>>(f[j]);
  if constexpr (STREAM) __builtin_nontemporal_store(x, reinterpret_cast<vec *>(p));
  else *reinterpret_cast<vec *>(p) = x;
}

// Sum over the 1 << shift lanes of a head.
__device__ __forceinline__ float head_sum(float x, int shift) {
  if (shift >= 1) x += dpp_f32<0xB1>(x);
  if (shift >= 2) x += dpp_f32<0x4E>(x);
  if (shift >= 3) x += dpp_f32<0x141>(x);
  if (shift >= 4) x += dpp_f32<0x140>(x);
  if (shift >= 5) x = sum_xor16(x);
  if (shift >= 6) x = sum_xor32(x);
  return x;
}

__device__ __forceinline__ float weight_at(const void *w, int f16, int i) {
  return f16 ? __half2float(static_cast<const __half *>(w)[i]) : static_cast<const float *>(w)[i];
}

// The sequence that holds row t: how many sequences end at or before it.  64 sequences a load.
__device__ __forceinline__ int sequence_of(const int32_t *cu, int B, int64_t t, int lane) {
  int b = 0;
  for (int j = 0; j < B; j += 64) {
    const bool before = j + lane < B && cu[j + lane + 1] <= t;
    const int n = __popcll(__ballot(before));
    b += n;
    if (n < 64) break;
  }
  return b;
}

// V: elements per load; REP: units of 2 V elements a lane takes of a head (more than one only where V is 1 or 2).
// STREAM: the results are stored past the caches.
template <typename TI, typename TO, int V, int REP, bool PAGED, bool STREAM = false>
__global__ __launch_bounds__(kBlock) void rotary_kernel(RotaryArgs a) {
  __shared__ float s_cos[kWaves][kMaxPairs], s_sin[kWaves][kMaxPairs];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWaves + wave;
  const int64_t t = a.first + unit / a.groups;
  if (t >= a.end) return;  // whole wavefronts leave; nothing below waits for another wavefront
  const int group = static_cast<int>(unit % a.groups);

  int64_t cache_row = -1, cache_pos = t;  // element offset / D of head 0 of the token's row in its page; -1: not stored
  if constexpr (PAGED) {
    const int b = sequence_of(a.cu, a.B, t, lane);
    if (b >= a.B) return;  // behind the last sequence: left as it was
    cache_pos = static_cast<int64_t>(a.start[b]) + (t - a.cu[b]);
    if (cache_pos >= 0 && (cache_pos >> kPageShift) < a.max_pages) {
      const int page = a.page_table[static_cast<int64_t>(b) * a.max_pages + (cache_pos >> kPageShift)];
      if (page >= 0 && page < a.n_pages)
        cache_row = (static_cast<int64_t>(page) * a.heads[1] << kPageShift) + (cache_pos & ((1 << kPageShift) - 1));
    }
  }

  // this lane's elements of a head: V from e0[r] on and V from e1[r] on
  const int units = a.dim / (2 * V), turned = a.rotary_dim / (2 * V), pairs = a.rotary_dim / 2;
  const int sub = lane & ((1 << a.lanes_shift) - 1);
  int e0[REP], e1[REP];
  bool rot[REP], rot1[REP];
#pragma unroll
  for (int r = 0; r < REP; ++r) {
    const int u = sub + 64 * r;
    if (a.interleaved) {  // chunks u and u + units of the head, V / 2 pairs in each
      e0[r] = u * V;
      e1[r] = (u + units) * V;
      rot[r] = u < units && e0[r] < a.rotary_dim;
      rot1[r] = u < units && e1[r] < a.rotary_dim;
    } else {
      rot[r] = rot1[r] = u < turned;
      // behind the rotated part the remaining chunks are paired the same way, for the sake of the loads
      e0[r] = rot[r] ? u * V : a.rotary_dim + (u - turned) * V;
      e1[r] = rot[r] ? e0[r] + pairs : e0[r] + (units - turned) * V;
    }
  }

  const int step = 64 >> a.lanes_shift;
  const int all = a.heads[0] + a.heads[1] + a.heads[2];
  const int h_first = group * a.heads_per_group, h_end = min(h_first + a.heads_per_group, all);
  auto which_of = [&](int h) { return h < a.heads[0] ? 0 : (h < a.heads[0] + a.heads[1] ? 1 : 2); };
  auto head_in = [&](int h, int which) { return h - (which == 0 ? 0 : (which == 1 ? a.heads[0] : a.heads[0] + a.heads[1])); };
  // the elements of head h; a head that is not this wavefront's, or has no place to go, reads as zeros
  auto load = [&](int h, float (&x0)[REP][V], float (&x1)[REP][V]) {
    const int which = which_of(h), hh = head_in(h, which);
    const bool live = h < h_end && (!PAGED || which == 0 || cache_row >= 0);
    const TI *src = static_cast<const TI *>(which == 0 ? a.x[0] : (which == 1 ? a.x[1] : a.x[2])) +
                    t * (which == 0 ? a.stride[0] : (which == 1 ? a.stride[1] : a.stride[2])) + static_cast<int64_t>(hh) * a.dim;
#pragma unroll
    for (int r = 0; r < REP; ++r) {
#pragma unroll
      for (int j = 0; j < V; ++j) x0[r][j] = x1[r][j] = 0.f;
      if (live && sub + 64 * r < units) {
        load_v<TI, V>(src + e0[r], x0[r]);
        load_v<TI, V>(src + e1[r], x1[r]);
      }
    }
  };
  // the first heads, and the weights, are on their way while the angles are made; each next round of heads while one is rotated
  // (65536 rows into the pages 361 -> 317 us; without norm and pages there is less to wait for, and the registers cost more
  // wavefronts than the loads ahead bring: 33001 rows 149 us, 159 us with them.)
  constexpr bool kLoadsAhead = PAGED;
  float x0[REP][V], x1[REP][V];
  if constexpr (kLoadsAhead) load(h_first + (lane >> a.lanes_shift), x0, x1);
  float w0[2][REP][V], w1[2][REP][V];
  if constexpr (PAGED) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < REP; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const bool on = a.norm && a.w[k] && sub + 64 * r < units;
          w0[k][r][j] = on ? weight_at(a.w[k], a.w_f16, e0[r] + j) : 1.f;
          w1[k][r][j] = on ? weight_at(a.w[k], a.w_f16, e1[r] + j) : 1.f;
        }
  }

  // angles: one pair per lane and pass
  for (int i = lane; i < pairs; i += 64) {
    int64_t p = cache_pos;
    if (a.pos) {
      int axis = 0;
      if (a.axes == 3) axis = i % 3 == 1 && i < a.h_lim ? 1 : (i % 3 == 2 && i < a.w_lim ? 2 : 0);
      p = a.pos[axis * a.rows + t];
    }
    const double turns = static_cast<double>(p) * static_cast<double>(a.inv_freq[i]) * 0.15915494309189533577;  // 1 / 2 pi
    const double angle = (turns - rint(turns)) * 6.283185307179586477;
    const float ang = static_cast<float>(angle), rest = static_cast<float>(angle - static_cast<double>(ang));
    float sn, cs;
    sincosf(ang, &sn, &cs);
    s_cos[wave][i] = __builtin_fmaf(-rest, sn, cs) * a.scale;
    s_sin[wave][i] = __builtin_fmaf(rest, cs, sn) * a.scale;
  }
  // LDS accesses of one wavefront complete in order; the compiler must keep them in order too
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();

  float c0[REP][V], n0[REP][V];  // interleaved: of the first chunk's pairs, then of the second's
#pragma unroll
  for (int r = 0; r < REP; ++r)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool second = a.interleaved && j >= V / 2;
      const int pair = a.interleaved ? (second ? e1[r] / 2 + j - V / 2 : e0[r] / 2 + j) : e0[r] + j;
      const bool on = second ? rot1[r] : rot[r];
      c0[r][j] = on ? s_cos[wave][pair] : 1.f;
      n0[r][j] = on ? s_sin[wave][pair] : 0.f;
    }

  // (every lane stays in the loop: the sums below run over whole rows of lanes)
  for (int h0 = h_first; h0 < h_end; h0 += step) {
    const int h = h0 + (lane >> a.lanes_shift), which = which_of(h), hh = head_in(h, which);
    const bool live = h < h_end && (!PAGED || which == 0 || cache_row >= 0);
    TO *dst = static_cast<TO *>(which == 0 ? a.out[0] : (which == 1 ? a.out[1] : a.out[2]));
    if (PAGED && which != 0)
      dst += (cache_row + (static_cast<int64_t>(hh) << kPageShift)) * a.dim;
    else
      dst += (t * (which == 0 ? a.heads[0] : a.heads[1]) + hh) * a.dim;
    float y0[REP][V], y1[REP][V];
    if constexpr (!kLoadsAhead) load(h, x0, x1);
    else if (h0 + step < h_end) load(h + step, y0, y1);
    if (PAGED && a.norm) {
      float ss = 0.f;
#pragma unroll
      for (int r = 0; r < REP; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) ss = __builtin_fmaf(x0[r][j], x0[r][j], __builtin_fmaf(x1[r][j], x1[r][j], ss));
      ss = head_sum(ss, a.lanes_shift);
      if (which < 2) {
        const float inv = 1.0f / sqrtf(ss / static_cast<float>(a.dim) + a.eps);
#pragma unroll
        for (int r = 0; r < REP; ++r)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            x0[r][j] = x0[r][j] * inv * (which == 0 ? w0[0][r][j] : w0[1][r][j]);
            x1[r][j] = x1[r][j] * inv * (which == 0 ? w1[0][r][j] : w1[1][r][j]);
          }
      }
    }
#pragma unroll
    for (int r = 0; r < REP; ++r) {
      if (!live || sub + 64 * r >= units) continue;
      if (which < 2) {
        if (a.interleaved) {
          if constexpr (V >= 2) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
              const float p = x0[r][2 * j], q = x0[r][2 * j + 1], u = x1[r][2 * j], v = x1[r][2 * j + 1];
              if (rot[r]) {
                x0[r][2 * j] = p * c0[r][j] - q * n0[r][j];
                x0[r][2 * j + 1] = q * c0[r][j] + p * n0[r][j];
              }
              if (rot1[r]) {
                x1[r][2 * j] = u * c0[r][j + V / 2] - v * n0[r][j + V / 2];
                x1[r][2 * j + 1] = v * c0[r][j + V / 2] + u * n0[r][j + V / 2];
              }
            }
          }
        } else if (rot[r]) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float p = x0[r][j], q = x1[r][j];
            x0[r][j] = p * c0[r][j] - q * n0[r][j];
            x1[r][j] = q * c0[r][j] + p * n0[r][j];
          }
        }
      }
      store_v<STREAM>(dst + e0[r], x0[r]);
      store_v<STREAM>(dst + e1[r], x1[r]);
    }
    if constexpr (kLoadsAhead) {
#pragma unroll
      for (int r = 0; r < REP; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x0[r][j] = y0[r][j];
          x1[r][j] = y1[r][j];
        }
    }
  }
}

// Elements per load: the widest V of at most 16 bytes for which the chunks of a head, its rotated part and the rows of
// every tensor start on multiples of V elements (V * esz bytes for the pointers).  0: none (interleaved pairs need V >= 2).
int pick_v(const RotaryArgs &a, int in_size, int out_size) {
  for (int v = 16 / in_size; v >= 1; v /= 2) {
    bool ok = a.dim % (2 * v) == 0 && (a.interleaved ? v >= 2 && a.rotary_dim % v == 0 : a.rotary_dim % (2 * v) == 0);
    ok = ok && (v <= 2 || a.dim / (2 * v) <= 64);
    for (int i = 0; i < 3 && ok; ++i) {
      if (a.heads[i] == 0) continue;
      const uintptr_t in = reinterpret_cast<uintptr_t>(a.x[i]), out = reinterpret_cast<uintptr_t>(a.out[i]);
      const uintptr_t oa = static_cast<uintptr_t>(v * out_size < 16 ? v * out_size : 16);
      ok = in % (v * in_size) == 0 && a.stride[i] % v == 0 && out % oa == 0;
    }
    if (ok) return v;
  }
  return 0;
}

template <typename TI, typename TO, bool PAGED>
int launch(RotaryArgs a, hipStream_t st) {
  const int v = pick_v(a, sizeof(TI), sizeof(TO));
  if (v == 0) return AXHIP_INVALID_ARGUMENT;
  const int units = a.dim / (2 * v);
  a.lanes_shift = 0;
  while ((1 << a.lanes_shift) < units && a.lanes_shift < 6) ++a.lanes_shift;
  // heads of a token: all in one wavefront when there are tokens enough to fill the device, else one round of heads each
  const int all = a.heads[0] + a.heads[1] + a.heads[2], step = 64 >> a.lanes_shift;
  const int rounds = (all + step - 1) / step;
  int64_t per = a.rows >= 16384 ? rounds : (a.rows * rounds) / 16384;
  if (per < 1) per = 1;
  if (per > rounds) per = rounds;
  a.heads_per_group = static_cast<int>(per) * step;
  a.groups = (all + a.heads_per_group - 1) / a.heads_per_group;
  // Results that would push the input of the next operators out of the 256 MB memory-side cache are stored past it (33001 rows
  // in fp32 150 -> 135 us, 65536 rows into the pages 317 -> 286 us); smaller ones are about to be read again.
  const bool stream = a.rows * all * a.dim * static_cast<int64_t>(sizeof(TO)) >= (int64_t(64) << 20);
  constexpr int kWide = 16 / sizeof(TI);
  for (a.first = 0; a.first < a.rows; a.first = a.end) {
    a.end = a.rows - a.first < kMostRows ? a.rows : a.first + kMostRows;  // (that many only where a.groups is 1)
    const dim3 g(static_cast<unsigned>(((a.end - a.first) * a.groups + kWaves - 1) / kWaves)), b(kBlock);
    if (v == kWide) {
      if (stream) hipLaunchKernelGGL((rotary_kernel<TI, TO, kWide, 1, PAGED, true>), g, b, 0, st, a);
      else hipLaunchKernelGGL((rotary_kernel<TI, TO, kWide, 1, PAGED>), g, b, 0, st, a);
    } else if (v == 4) {
      if constexpr (kWide > 4) hipLaunchKernelGGL((rotary_kernel<TI, TO, 4, 1, PAGED>), g, b, 0, st, a);
    } else if (v == 2) {
      hipLaunchKernelGGL((rotary_kernel<TI, TO, 2, 2, PAGED>), g, b, 0, st, a);
    } else {
      hipLaunchKernelGGL((rotary_kernel<TI, TO, 1, 4, PAGED>), g, b, 0, st, a);
    }
    const int rc = launch_status();
    if (rc != AXHIP_OK) return rc;
  }
  return AXHIP_OK;
}

bool aligned_to(const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace axhip

using namespace axhip;

extern "C" {

AXHIP_API int axhip_rotary_inv_freq(int kind, double theta, int rotary_dim, double factor, int64_t trained_len,
                                    double fast_turns, double slow_turns, float *inv_freq, float *scale) {
  if (kind < AXHIP_ROTARY_PLAIN || kind > AXHIP_ROTARY_YARN || rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > 2 * kMaxPairs)
    return AXHIP_INVALID_ARGUMENT;
  if (!(theta > 0.0) || (kind != AXHIP_ROTARY_PLAIN && !(factor > 0.0))) return AXHIP_INVALID_ARGUMENT;
  if (kind == AXHIP_ROTARY_YARN && (trained_len <= 0 || !(fast_turns > slow_turns))) return AXHIP_INVALID_ARGUMENT;
  if (!inv_freq) return AXHIP_INVALID_PTR;
  const double two_pi = 6.283185307179586477;
  double base = theta;
  if (kind == AXHIP_ROTARY_NTK && rotary_dim > 2) base = theta * pow(factor, static_cast<double>(rotary_dim) / (rotary_dim - 2));
  for (int i = 0; i < rotary_dim / 2; ++i) {
    double f = pow(base, -2.0 * i / rotary_dim);
    if (kind == AXHIP_ROTARY_LINEAR) f /= factor;
    if (kind == AXHIP_ROTARY_YARN) {
      double keep = (static_cast<double>(trained_len) * f / two_pi - slow_turns) / (fast_turns - slow_turns);
      keep = keep < 0.0 ? 0.0 : (keep > 1.0 ? 1.0 : keep);
      f = f * keep + f / factor * (1.0 - keep);
    }
    inv_freq[i] = static_cast<float>(f);
  }
  if (scale) *scale = kind == AXHIP_ROTARY_YARN && factor > 1.0 ? static_cast<float>(0.1 * log(factor) + 1.0) : 1.0f;
  return AXHIP_OK;
}

AXHIP_API int axhip_rotary_qk(const void *q, int64_t q_stride, const void *k, int64_t k_stride, const int64_t *pos,
                              const float *inv_freq, float scale, int interleaved, int rotary_dim, void *q_out,
                              void *k_out, int dtype, int64_t rows, int q_heads, int k_heads, int dim,
                              axhip_stream stream) {
  if (!is_float_dtype(dtype)) return AXHIP_UNSUPPORTED_TYPE;
  if (rows < 0 || q_heads < 0 || k_heads < 0 || q_heads + static_cast<int64_t>(k_heads) > 65535) return AXHIP_INVALID_ARGUMENT;
  if (dim <= 0 || dim > 512 || dim % 8 != 0 || rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > dim)
    return AXHIP_INVALID_ARGUMENT;
  if (rows > INT32_MAX) return AXHIP_INVALID_ARGUMENT;
  if ((q_heads && q_stride < static_cast<int64_t>(q_heads) * dim) || (k_heads && k_stride < static_cast<int64_t>(k_heads) * dim))
    return AXHIP_INVALID_ARGUMENT;
  if ((q_heads && q == q_out && q_stride != static_cast<int64_t>(q_heads) * dim) ||
      (k_heads && k == k_out && k_stride != static_cast<int64_t>(k_heads) * dim))
    return AXHIP_INVALID_ARGUMENT;  // results would be written over rows that are still to be read
  if (rows == 0 || q_heads + k_heads == 0) return AXHIP_OK;
  if (!pos || !inv_freq || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return AXHIP_INVALID_PTR;
  const int esz = dtype == AXHIP_FLOAT16 ? 2 : 4;
  if (!aligned_to(q, esz) || !aligned_to(k, esz) || !aligned_to(q_out, esz) || !aligned_to(k_out, esz) ||
      !aligned_to(pos, 8) || !aligned_to(inv_freq, 4))
    return AXHIP_INVALID_PTR;
  RotaryArgs a{};
  a.x[0] = q;
  a.x[1] = k;
  a.stride[0] = q_stride;
  a.stride[1] = k_stride;
  a.out[0] = q_out;
  a.out[1] = k_out;
  a.heads[0] = q_heads;
  a.heads[1] = k_heads;
  a.pos = pos;
  a.inv_freq = inv_freq;
  a.scale = scale;
  a.rows = rows;
  a.dim = dim;
  a.rotary_dim = rotary_dim;
  a.interleaved = interleaved ? 1 : 0;
  a.axes = 1;
  return dtype == AXHIP_FLOAT16 ? launch<__half, __half, false>(a, as_stream(stream))
                                : launch<float, float, false>(a, as_stream(stream));
}

AXHIP_API int axhip_rotary_append_paged(const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v,
                                        int64_t v_stride, int dtype, const void *q_weight, const void *k_weight,
                                        int w_dtype, float eps, int norm, const int64_t *pos, int pos_axes,
                                        const float *inv_freq, float scale, int interleaved, int rotary_dim, int h_sec,
                                        int w_sec, const int32_t *cu_tokens, const int32_t *start,
                                        const int32_t *page_table, void *q_out, void *k_pool, void *v_pool,
                                        int cache_dtype, int tokens, int B, int Hq, int Hkv, int D, int max_pages,
                                        int n_pages, axhip_stream stream) {
  if (!is_float_dtype(dtype) || !is_float_dtype(cache_dtype)) return AXHIP_UNSUPPORTED_TYPE;
  if (norm && (q_weight || k_weight) && !is_float_dtype(w_dtype)) return AXHIP_UNSUPPORTED_TYPE;
  if (tokens < 0 || B < 0 || Hq <= 0 || Hkv <= 0 || max_pages <= 0 || n_pages <= 0) return AXHIP_INVALID_ARGUMENT;
  if (Hq > 32767 || Hkv > 16383 || B > (1 << 20)) return AXHIP_INVALID_ARGUMENT;
  if (D <= 0 || D > 512 || D % 8 != 0 || rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > D) return AXHIP_INVALID_ARGUMENT;
  if (pos_axes != 1 && pos_axes != 3) return AXHIP_INVALID_ARGUMENT;
  if (!pos && pos_axes != 1) return AXHIP_INVALID_ARGUMENT;
  if (h_sec < 0 || w_sec < 0 || h_sec > D || w_sec > D) return AXHIP_INVALID_ARGUMENT;
  if (q_stride < static_cast<int64_t>(Hq) * D || k_stride < static_cast<int64_t>(Hkv) * D || v_stride < static_cast<int64_t>(Hkv) * D)
    return AXHIP_INVALID_ARGUMENT;
  if (tokens == 0 || B == 0) return AXHIP_OK;
  if (!q || !k || !v || !inv_freq || !cu_tokens || !start || !page_table || !q_out || !k_pool || !v_pool) return AXHIP_INVALID_PTR;
  const int esz = dtype == AXHIP_FLOAT16 ? 2 : 4, csz = cache_dtype == AXHIP_FLOAT16 ? 2 : 4;
  const int wsz = w_dtype == AXHIP_FLOAT16 ? 2 : 4;
  if (!aligned_to(q, esz) || !aligned_to(k, esz) || !aligned_to(v, esz) || !aligned_to(q_out, csz) || !aligned_to(k_pool, 16) ||
      !aligned_to(v_pool, 16) || !aligned_to(pos, 8) || !aligned_to(inv_freq, 4) || !aligned_to(cu_tokens, 4) ||
      !aligned_to(start, 4) || !aligned_to(page_table, 4) || (norm && (!aligned_to(q_weight, wsz) || !aligned_to(k_weight, wsz))))
    return AXHIP_INVALID_PTR;
  RotaryArgs a{};
  a.x[0] = q;
  a.x[1] = k;
  a.x[2] = v;
  a.stride[0] = q_stride;
  a.stride[1] = k_stride;
  a.stride[2] = v_stride;
  a.out[0] = q_out;
  a.out[1] = k_pool;
  a.out[2] = v_pool;
  a.heads[0] = Hq;
  a.heads[1] = a.heads[2] = Hkv;
  a.pos = pos;
  a.axes = pos_axes;
  a.inv_freq = inv_freq;
  a.scale = scale;
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.w_f16 = w_dtype == AXHIP_FLOAT16;
  a.norm = norm ? 1 : 0;
  a.eps = eps;
  a.rows = tokens;
  a.dim = D;
  a.rotary_dim = rotary_dim;
  a.interleaved = interleaved ? 1 : 0;
  a.h_lim = 3 * h_sec;
  a.w_lim = 3 * w_sec;
  a.cu = cu_tokens;
  a.start = start;
  a.page_table = page_table;
  a.B = B;
  a.max_pages = max_pages;
  a.n_pages = n_pages;
  hipStream_t st = as_stream(stream);
  if (dtype == AXHIP_FLOAT16)
    return cache_dtype == AXHIP_FLOAT16 ? launch<__half, __half, true>(a, st) : launch<__half, float, true>(a, st);
  return cache_dtype == AXHIP_FLOAT16 ? launch<float, __half, true>(a, st) : launch<float, float, true>(a, st);
}

}  // extern "C"
