// Attention of a ragged batch of new tokens over a paged KV cache that already holds their keys and values.
//
//   out_i = sum_{j <= p_i} softmax_j(q_i . k_j / sqrt(D)) v_j,   p_i = start[b] + i the position of the i-th new token of b.
//
// Work decomposition.  The G = Hq / Hkv query heads of a kv head see the same keys, so the new tokens of a sequence give
// n G "rows" per kv head, row r = (token r / G, head r % G): any G, and positions that grow with r.  A workgroup of four
// wavefronts takes a tile of up to 64 NT rows of one (sequence, kv head) and a piece of the keys they see; a wavefront
// takes NT column tiles of 16 rows.  In a tile with few rows (at most 16 NT: decoding sequences, drafts, the last rows of
// a chunk) all wavefronts take the same rows and deal the 32-key blocks of a stage among themselves; their states are
// added up at the end.
//
// Everything is computed transposed, so that no operand changes its layout in registers (see the products below):
//   S^T = K . Q^T  (16 keys x 16 rows), O^T += V^T . P^T  (16 d x 16 rows); a lane owns the row lane % 16 in both.
// K and V travel through LDS in stages of KS keys (double-buffered, 16-byte units XOR-swizzled by key).  A stage lies
// inside one page of 128 keys, so its address is one page number (read a stage ahead) and fixed lane offsets, and every
// address of a stage is inside the pool whatever the lengths are.
//
// Few tiles over many keys would leave the device idle: the keys of a tile are cut into pieces so that the launch has
// about two workgroups per CU of equal work.  The cut is made on the device from cu_tokens and start (every workgroup
// derives it with a few wave operations), so a captured launch follows lengths that change.  A piece of a cut tile leaves
// an unnormalised state in the workspace; a second kernel adds the pieces of a tile in a fixed order.  No counters, no
// state between launches: launches with workspaces of their own may overlap.
//
// fp32 statistics throughout.  fp16: probabilities are rounded to fp16 for the second product (2^-12 of their value at
// most, random in sign), numerator and denominator from the same rounded values.  fp32: fp32 matrix instructions.
#include "common.hpp"

#include <type_traits>

namespace axhip {
namespace {

constexpr int kThreads = 256;
constexpr int kWavesWg = 4;
constexpr int kPageKeys = 128, kPageShift = 7;
constexpr int kBlockKeys = 32;      // keys of one softmax step
constexpr float kMasked = -1.0e30f;
typedef float float8_t __attribute__((ext_vector_type(8)));
constexpr int kMinPieceUnits = 2;   // a piece has at least 2 units of 128 keys

struct ChunkArgs {
  const void *q, *k, *v;
  const int32_t *page_table, *cu, *start;
  void *out;
  float *part_o;   // [slots][slot_rows][D]
  float *part_ml;  // [slots][slot_rows][2]: maximum (log2 units), sum
  int tokens, B, Hq, Hkv, group, max_q, max_len, max_pages, n_pages;
  int slots, slot_rows, target;  // target: pieces the launch aims at
  float scale_log2e;
};

template <typename T, int D>
struct Cfg {
  static constexpr int NT = D == 256 || (sizeof(T) == 4 && D == 128) ? 1 : 2;  // column tiles per wavefront
  static constexpr int TR = kWavesWg * 16 * NT;                        // rows per tile
  static constexpr int FEW = 16 * NT;                                  // rows up to which wavefronts deal the keys
  static constexpr int KS = (D == 256 || (sizeof(T) == 4 && D == 128)) ? 32 : 64;  // keys per stage
  static constexpr int E = 16 / sizeof(T);                             // elements per 16-byte unit
  static constexpr int UPR = D / E;                                    // units per row
  static constexpr int SW = (UPR < 16 ? UPR : 16) - 1;                 // swizzle mask
  static constexpr int VEC = KS * UPR / kThreads;                      // units per thread, tensor and stage
  static constexpr int STATE = D + 4;                                  // row stride of the states added up in LDS
  static constexpr int kStageBytes = 4 * KS * D * static_cast<int>(sizeof(T));
  // wavefronts with keys of their own in a tile of few rows
  static constexpr int kDealt = sizeof(T) == 2 && D <= 128 ? kWavesWg : (KS / kBlockKeys < kWavesWg ? KS / kBlockKeys : kWavesWg);
  static constexpr int kStateBytes = kDealt * FEW * (STATE + 2) * 4;
  static constexpr int kLdsBytes = (kStageBytes > kStateBytes ? kStageBytes : kStateBytes) + 16;
};

// ---- the cut -------------------------------------------------------------------------------------------------------
struct Seq {
  int c0, rows, tiles, units, pieces;  // first token, rows per kv head, tiles, 128-key units of the last tile, pieces a tile
};
template <int TR>
__device__ __forceinline__ Seq load_seq(const ChunkArgs &a, int b) {
  Seq s{0, 0, 0, 0, 1};
  if (b < a.B) {
    s.c0 = min(max(a.cu[b], 0), a.tokens);
    const int c1 = min(max(a.cu[b + 1], s.c0), a.tokens);
    const int n = min(c1 - s.c0, a.max_q);
    const int64_t last = static_cast<int64_t>(a.start[b]) + n;  // keys the last token sees
    const int keys = static_cast<int>(last < 0 ? 0 : (last > a.max_len ? a.max_len : last));
    s.rows = n * a.group;
    s.tiles = (s.rows + TR - 1) / TR;
    s.units = (keys + 127) >> 7;
  }
  return s;
}
// Units per piece: the work of the launch (every tile taken as long as its sequence's last) over the pieces aimed at.
template <int TR>
__device__ __forceinline__ int units_per_piece(const ChunkArgs &a, int lane) {
  float work = 0.f;
  for (int j = 0; j < a.B; j += 64) {
    const Seq s = load_seq<TR>(a, j + lane);
    work += group_sum<64>(static_cast<float>(s.tiles) * static_cast<float>(s.units));
  }
  const float q = ceilf(work * static_cast<float>(a.Hkv) / static_cast<float>(a.target));
  return max(kMinPieceUnits, static_cast<int>(fminf(q, 1.0e9f)));
}
__device__ __forceinline__ int pieces_of(int units, int per) { return max(1, (units + per - 1) / per); }

struct Piece {
  int b, tile, piece, pieces, slot, c0, rows, units;
  bool found;
};
// The `flat`-th piece (MERGE: the `flat`-th cut tile) of the launch, per kv head.  slot: number of the piece (MERGE: of the
// tile's first piece) among the pieces of cut tiles.
template <int TR, bool MERGE>
__device__ __forceinline__ Piece find_piece(const ChunkArgs &a, int flat, int lane) {
  const int per = units_per_piece<TR>(a, lane);
  int done = 0, slots = 0;
  Piece p{};
  p.found = false;
  for (int j = 0; j < a.B; j += 64) {
    Seq s = load_seq<TR>(a, j + lane);
    s.pieces = pieces_of(s.units, per);
    const bool cut = s.pieces > 1;
    const int mine = MERGE ? (cut ? s.tiles : 0) : s.tiles * s.pieces;
    const int upto = done + wave_prefix_i32(mine);
    const int my_slots = cut ? s.tiles * s.pieces : 0;
    const int slots_upto = slots + wave_prefix_i32(my_slots);
    const uint64_t hit = __ballot(flat < upto);
    if (hit) {
      const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      auto at = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int rest = flat - at(upto - mine);
      p.b = j + l;
      p.c0 = at(s.c0);
      p.rows = at(s.rows);
      p.units = at(s.units);
      p.pieces = at(s.pieces);
      const int tiles = at(s.tiles);
      const int order = MERGE ? rest : rest / p.pieces;
      p.piece = MERGE ? 0 : rest - order * p.pieces;
      p.tile = tiles - 1 - order;  // the tiles that see most keys first
      p.slot = at(slots_upto - my_slots) + p.tile * p.pieces + p.piece;
      p.found = true;
      return p;
    }
    done = __builtin_amdgcn_readlane(upto, 63);
    slots = __builtin_amdgcn_readlane(slots_upto, 63);
  }
  return p;
}

// ---- LDS reads of the products' operands -----------------------------------------------------------------------------
typedef unsigned char __attribute__((address_space(3))) lds_byte;

template <typename V>
__device__ __forceinline__ V lds_at(const lds_byte *base, int offset) {
  return *reinterpret_cast<const V __attribute__((address_space(3))) *>(base + offset);
}
// 4 keys x 16 d of row-major V, transposed on the way: within 16 lanes, lane i names 4 consecutive elements and receives
// element i of each of the 4 rows.
__device__ __forceinline__ half4_t lds_tr(const lds_byte *base, int offset) {
  typedef __fp16 fp16x4_t __attribute__((__vector_size__(4 * sizeof(__fp16))));
  return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((fp16x4_t __attribute__((address_space(3))) *)(base + offset)));
}

// 16 bytes a lane from memory (base, uniform, + off) straight to LDS: lane l's to dst + 16 l.  AUX 2: a non-temporal load.
template <typename T, int AUX = 0>
__device__ __forceinline__ void load_lds16(const T *base, unsigned off, lds_byte *dst) {
  const unsigned char *src = reinterpret_cast<const unsigned char *>(base) + off;
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                   (__attribute__((address_space(3))) void *)dst, 16, 0, AUX);
}

// Whether a 16-byte unit holds an infinity or a NaN, and the unit without them.
template <typename T>
__device__ __forceinline__ bool unit_bad(const u32x4_t &u) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2)
      bad |= (u[i] & 0x7c00u) == 0x7c00u || (u[i] & 0x7c000000u) == 0x7c000000u;
    else
      bad |= (u[i] & 0x7f800000u) == 0x7f800000u;
  }
  return bad;
}
template <typename T>
__device__ __forceinline__ u32x4_t unit_finite(u32x4_t u) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      if ((u[i] & 0x7c00u) == 0x7c00u) u[i] &= 0xffff0000u;
      if ((u[i] & 0x7c000000u) == 0x7c000000u) u[i] &= 0x0000ffffu;
    } else {
      if ((u[i] & 0x7f800000u) == 0x7f800000u) u[i] = 0u;
    }
  }
  return u;
}

// w * o added to a sum of pieces; a weight that underflowed to 0 must not turn an infinity into a NaN.
__device__ __forceinline__ float add_weighted(float sum, float w, float o) {
  return w > 0.f || fabsf(o) < __builtin_inff() ? __builtin_fmaf(w, o, sum) : sum + o;
}

extern __shared__ __attribute__((aligned(16))) unsigned char chunk_smem[];

template <typename T, int D>
__global__ __launch_bounds__(kThreads, (Cfg<T, D>::kLdsBytes <= 80 * 1024 ? 2 : 1)) void chunk_attn_kernel(ChunkArgs a) {
  using C = Cfg<T, D>;
  using S = typename std::conditional<sizeof(T) == 2, _Float16, float>::type;
  constexpr int NT = C::NT, KS = C::KS, UPR = C::UPR, VEC = C::VEC, SW = C::SW;
  constexpr int DT = D / 16;
  constexpr int QF = sizeof(T) == 2 ? D / 32 : D / 4;  // operand registers of a column tile (8 halves or 1 float each)
  constexpr bool kHalf = sizeof(T) == 2;
  constexpr int kRow = D * static_cast<int>(sizeof(T)), kTensor = 2 * KS * kRow;  // bytes: a row, both stages of K (V behind)
  lds_byte *smem = (lds_byte *)chunk_smem;
  int *s_flag = reinterpret_cast<int *>(chunk_smem + C::kLdsBytes - 16);

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c = lane & 15, g = lane >> 4;
  const int hk = blockIdx.x % a.Hkv;
  const Piece pc = find_piece<C::TR, false>(a, blockIdx.x / a.Hkv, lane);
  if (!pc.found) return;
  const int start = a.start[pc.b];
  const int row0 = pc.tile * C::TR, n_rows = min(pc.rows - row0, C::TR);
  const bool few = n_rows <= C::FEW;
  if (tid == 0) *s_flag = 0;

  // this wavefront's rows (positions never fall with the row); rows past the tile repeat its last one and are not stored
  auto position = [&](int r) {  // last key row r of the tile sees, -1: none
    const int64_t p = static_cast<int64_t>(start) + (row0 + r) / a.group;
    return static_cast<int>(p < -1 ? -1 : (p > a.max_len - 1 ? a.max_len - 1 : p));
  };
  const int wrow = few ? 0 : wave * 16 * NT;
  int pos[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) pos[t] = position(min(wrow + t * 16 + c, n_rows - 1));
  const int wave_first = position(min(wrow, n_rows - 1)), wave_last = position(min(wrow + 16 * NT, n_rows) - 1);
  const bool idle = wrow >= n_rows;  // a wavefront without rows only loads
  const int tile_first = position(0), k_all = position(n_rows - 1) + 1;  // keys the tile sees: [0, k_all)
  const int tile_units = (k_all + 127) >> 7;
  const int k0 = static_cast<int>(static_cast<int64_t>(tile_units) * pc.piece / pc.pieces) << 7;
  const int k_end = min(static_cast<int>(static_cast<int64_t>(tile_units) * (pc.piece + 1) / pc.pieces) << 7, k_all);
  const int n_stages = k_end > k0 ? (k_end - k0 + KS - 1) / KS : 0;
  // V rows past the tile's last key are stored as zeros, and in stages that some row of the tile must not see whole,
  // infinities and NaN of V are stored as zeros too (0 * inf is NaN) and added at the end to the rows that see them
  const int mixed_from = tile_first < 0 ? 0 : (tile_first + 1) / KS * KS;

  // K and V go from memory to LDS directly (16 bytes a lane; a wavefront fills 1 KiB in lane order, so the swizzle is made on
  // the side of memory: the lane of place u of a row fetches unit u ^ (row & SW)).  Load p of a thread covers row
  // p kStep + tid / UPR of the stage; its offset within the page differs by constants from load 0's.
  constexpr int kStep = kThreads / UPR;
  const unsigned voff = tid / UPR * kRow + ((tid % UPR) ^ ((tid / UPR) & SW)) * 16;
  // Where this lane reads its operands, as byte offsets into a stage of K / V; the steps of the products flip or add constant
  // bits of them.  Made opaque in every block, or the compiler keeps every one of the flipped offsets in registers.
  const int kaddr = c * kRow + (kHalf ? (g ^ (c & SW)) * 16 : (c & SW) * 16 + g * 4);
  const int vkey = kHalf ? 4 * g + (c >> 2) : 4 * g;
  const int vaddr = vkey * kRow + (kHalf ? ((((c & 3) >> 1) ^ (vkey & SW)) * 16 + (c & 1) * 8) : (((c >> 2) ^ (vkey & SW)) * 16 + (c & 3) * 4));
  // page numbers by scalar loads: a vector load would have to be waited for behind the stage on its way
  typedef const int32_t __attribute__((address_space(4))) *scalar_ptr;
  const scalar_ptr table = (scalar_ptr)(a.page_table + static_cast<int64_t>(pc.b) * a.max_pages);
  const int64_t page_elems = static_cast<int64_t>(a.Hkv) * kPageKeys * D;
  const T *kbase = static_cast<const T *>(a.k) + static_cast<int64_t>(hk) * kPageKeys * D;
  const T *vbase = static_cast<const T *>(a.v) + static_cast<int64_t>(hk) * kPageKeys * D;
  auto in_pool = [&](int page) { return min(max(page, 0), a.n_pages - 1); };
  auto load_stage = [&](int page, int key0, int buf) __attribute__((always_inline)) {
    const int64_t base = in_pool(page) * page_elems + static_cast<int64_t>(key0 & (kPageKeys - 1)) * D;
    const unsigned place = buf * (KS * kRow) + wave * 1024;
#pragma unroll
    for (int p = 0; p < VEC; ++p) {
      const unsigned off = (voff ^ ((p * kStep & SW) * 16)) + p * kStep * kRow;
      load_lds16(kbase + base, off, smem + place + p * kThreads * 16);
      load_lds16(vbase + base, off, smem + kTensor + place + p * kThreads * 16);
    }
  };
  // V of key `key` in LDS: zeros behind the piece, no infinities and NaN; whether there were any.
  auto clean_unit = [&](lds_byte *place, int key) __attribute__((always_inline)) {
    typedef u32x4_t __attribute__((address_space(3))) lds_unit;
    lds_unit *at = reinterpret_cast<lds_unit *>(place);
    const u32x4_t u = *at;
    if (key >= k_end) {
      *at = u32x4_t{0, 0, 0, 0};
    } else if (unit_bad<T>(u)) {
      *at = unit_finite<T>(u);
      return true;
    }
    return false;
  };
  // The units that this thread has fetched are in LDS.  (In its own order: the barrier behind this call makes them everybody's.)
  auto stage_arrived = [&](int key0, int buf) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (key0 + KS > mixed_from) {  // uniform; also every stage that reaches past k_end, for mixed_from <= k_all
      bool bad = false;
#pragma unroll 1
      for (int p = 0; p < VEC; ++p)
        bad |= clean_unit(smem + kTensor + buf * (KS * kRow) + (p * kThreads + tid) * 16, key0 + p * kStep + tid / UPR);
      if (bad) *s_flag = 1;
    }
  };

  const bool own_blocks = few && kHalf && D <= 128;
  if (n_stages > 0 && !own_blocks) load_stage(table[k0 >> kPageShift], k0, 0);

  // Q as the right operand of the first product, for the whole kernel
  typename std::conditional<kHalf, half8_t, float>::type qf[NT][QF];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = row0 + min(wrow + t * 16 + c, n_rows - 1), i = r / a.group;
    const S *qrow = static_cast<const S *>(a.q) +
                    (static_cast<int64_t>(pc.c0 + i) * a.Hq + hk * a.group + (r - i * a.group)) * D;
#pragma unroll
    for (int kk = 0; kk < QF; ++kk) {
      if constexpr (kHalf) qf[t][kk] = *reinterpret_cast<const half8_t *>(qrow + kk * 32 + g * 8);
      else qf[t][kk] = qrow[kk * 4 + g];
    }
  }

  float4_t o[NT][DT], lsum[NT];
  float m[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = kMasked;
    lsum[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[t][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
  }

  // ---- a block of 32 keys for this wavefront, in four parts ------------------------------------------------------------
  using KFrag = typename std::conditional<kHalf, half8_t, float>::type;
  using Probs = typename std::conditional<kHalf, half8_t, float8_t>::type;
  auto read_k = [&](int buf, int sub, KFrag (&kf)[2][QF]) __attribute__((always_inline)) {
    const lds_byte *k_l = smem + sub * (kBlockKeys * kRow);
    int ka = kaddr + buf * (KS * kRow);
    asm volatile("" : "+v"(ka));
#pragma unroll
    for (int tk = 0; tk < 2; ++tk)
#pragma unroll
      for (int kk = 0; kk < QF; ++kk) kf[tk][kk] = lds_at<KFrag>(k_l, (ka ^ (kk * (kHalf ? 64 : 16))) + tk * 16 * kRow);
  };
  auto scores = [&](const KFrag (&kf)[2][QF], float4_t (&sc)[NT][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < QF; ++kk)
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (kHalf) sc[t][tk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[tk][kk], qf[t][kk], sc[t][tk], 0, 0, 0);
          else sc[t][tk] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[tk][kk], qf[t][kk], sc[t][tk], 0, 0, 0);
        }
  };
  // Probabilities against the running maximum as it stands: it is moved, and everything rescaled, only when one of them
  // passes 2^8 (the first block of a row always does).  Until then p <= 256, which fp16 holds to the same 11 bits, and a
  // block needs no maximum over its row at all.  (The maximum never runs ahead, so no p is smaller than against the true one.)
  // MASK: some key of the block at kb is behind some row's position.
  auto softmax = [&](const float4_t (&sc)[NT][2], Probs (&pf)[NT], int kb, auto mask_c) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_c)::value;
    float p[NT][8];
    auto x_at = [&](int t, int j) __attribute__((always_inline)) {
      float v = sc[t][j >> 2][j & 3];
      if (MASK && kb + (j >> 2) * 16 + 4 * g + (j & 3) > pos[t]) v = kMasked;
      return v;
    };
    auto exps = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = x_at(t, j);
          p[t][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.scale_log2e, -m[t]));
          if (MASK && x <= kMasked) p[t][j] = 0.f;
        }
    };
    exps();
    float top = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, p[t][j]);
    if (__builtin_expect(__any(top > 256.f), 0)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float mx = x_at(t, 0);
#pragma unroll
        for (int j = 1; j < 8; ++j) mx = fmaxf(mx, x_at(t, j));
        const float mnew = fmaxf(m[t], max_xor32(max_xor16(mx)) * a.scale_log2e);
        const float corr = __builtin_amdgcn_exp2f(m[t] - mnew);
        m[t] = mnew;
        lsum[t] *= corr;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[t][dt] *= corr;
      }
      exps();
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (kHalf) pf[t][j] = static_cast<_Float16>(p[t][j]);
        else pf[t][j] = p[t][j];
      }
  };
  // fp16: V^T fragments of the block, d tile by d tile
  auto read_v = [&](int buf, int sub, half8_t (&vf)[DT]) __attribute__((always_inline)) {
    const lds_byte *v_l = smem + sub * (kBlockKeys * kRow) + kTensor;
    int va = vaddr + buf * (KS * kRow);
    asm volatile("" : "+v"(va));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const half4_t lo = lds_tr(v_l, va ^ (dt * 32)), hi = lds_tr(v_l, (va ^ (dt * 32)) + 16 * kRow);
      vf[dt] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  };
  auto add_values = [&](const half8_t (&vf)[DT], const Probs (&pf)[NT]) __attribute__((always_inline)) {
    if constexpr (kHalf) {
      const half8_t ones = {1, 1, 1, 1, 1, 1, 1, 1};
      // the row sums as a product with ones: every register of the result holds the row's sum
#pragma unroll
      for (int t = 0; t < NT; ++t) lsum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[t], lsum[t], 0, 0, 0);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[dt], pf[t], o[t][dt], 0, 0, 0);
    }
  };
  // fp32: product step (tk, e) takes keys tk * 16 + 4 g + e, g = 0 .. 3, so that a lane's score register e is its right operand
  auto add_values_f32 = [&](int buf, int sub, const Probs (&pf)[NT]) __attribute__((always_inline)) {
    if constexpr (!kHalf) {
      const lds_byte *v_l = smem + sub * (kBlockKeys * kRow) + kTensor;
      int va = vaddr + buf * (KS * kRow);
      asm volatile("" : "+v"(va));
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int t = 0; t < NT; ++t) lsum[t][0] += pf[t][tk * 4 + e];
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const float vf = lds_at<float>(v_l, (va ^ (dt * 64) ^ (e * 16)) + (tk * 16 + e) * kRow);
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf, pf[t][tk * 4 + e], o[t][dt], 0, 0, 0);
          }
        }
    }
  };
  auto block = [&](int buf, int sub, int kb, auto mask_c) __attribute__((always_inline)) {
    KFrag kf[2][QF];
    float4_t sc[NT][2];
    Probs pf[NT];
    read_k(buf, sub, kf);
    scores(kf, sc);
    softmax(sc, pf, kb, mask_c);
    if constexpr (kHalf) {
      half8_t vf[DT];
      read_v(buf, sub, vf);
      add_values(vf, pf);
    } else {
      add_values_f32(buf, sub, pf);
    }
  };

  // ---- a tile with few rows, fp16 ------------------------------------------------------------------------------------------
  // Bound by the stream of keys, so every wavefront takes blocks of its own (block i of the piece goes to wavefront i % 4) and
  // waits for nobody: K goes to registers in operand order (16 rows x 64 bytes a load), V through a strip of LDS of the
  // wavefront's own, both a block ahead, read once and therefore past the caches.
  constexpr bool kOwnBlocks = kHalf && D <= 128;
  auto few_rows = [&]() __attribute__((always_inline)) {
    constexpr int kVBytes = kBlockKeys * kRow, kLoads = kVBytes / 1024;  // V of a block; loads of a lane for it, as many for K
    constexpr int kRowsALoad = 1024 / kRow;
    static_assert(!kOwnBlocks || 2 * kWavesWg * kVBytes <= C::kStageBytes, "two blocks of V per wavefront fit the stages' LDS");
    auto fetch = [&](int page, int kb, int buf, KFrag (&kf)[2][QF]) __attribute__((always_inline)) {
      const int64_t base = in_pool(page) * page_elems + static_cast<int64_t>(kb & (kPageKeys - 1)) * D;
      int l = lane;
      asm volatile("" : "+v"(l));  // offsets are made here, not kept
      const unsigned v_row = static_cast<unsigned>(l) / UPR, v_off = v_row * kRow + ((l % UPR) ^ (v_row & SW)) * 16;
#pragma unroll
      for (int p = 0; p < kLoads; ++p)
        load_lds16<T, 2>(vbase + base, (v_off ^ ((p * kRowsALoad & SW) * 16)) + p * 1024, smem + (wave * 2 + buf) * kVBytes + p * 1024);
      const T *kb_ = kbase + base + (l & 15) * D + (l >> 4) * 8;
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
#pragma unroll
        for (int kk = 0; kk < QF; ++kk)
          if constexpr (kHalf)
            kf[tk][kk] = __builtin_bit_cast(half8_t, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(kb_ + tk * 16 * D + kk * 32)));
    };
    auto use = [&](int kb, int buf, const KFrag (&kf)[2][QF]) __attribute__((always_inline)) {
      float4_t sc[NT][2];
      Probs pf[NT];
      scores(kf, sc);
      __builtin_amdgcn_sched_barrier(0);
      if (kb + kBlockKeys > mixed_from) {
#pragma unroll 1
        for (int p = 0; p < kLoads; ++p)
          if (clean_unit(smem + (wave * 2 + buf) * kVBytes + p * 1024 + lane * 16, kb + static_cast<int>(lane / UPR) + p * kRowsALoad)) *s_flag = 1;
      }
      softmax(sc, pf, kb, std::true_type{});
      __builtin_amdgcn_sched_barrier(0);
      half8_t vf[DT];
      int va = vaddr + (wave * 2 + buf) * kVBytes;
      asm volatile("" : "+v"(va));
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const half4_t lo = lds_tr(smem, va ^ (dt * 32)), hi = lds_tr(smem, (va ^ (dt * 32)) + 16 * kRow);
        vf[dt] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
      add_values(vf, pf);
    };
    constexpr int kHop = kWavesWg * kBlockKeys;  // 128 keys: the wavefront's next block lies in the next page
    KFrag k_a[2][QF], k_b[2][QF];
    int kb = k0 + wave * kBlockKeys;
    if (kb >= k_end) return;
    auto page_of = [&](int key) { return table[min(key, k_end - 1) >> kPageShift]; };
    fetch(page_of(kb), kb, 0, k_a);
    int page = page_of(kb + kHop);
    // the loads of the block in use have arrived when no more than the next block's are under way (loads return in order)
    while (true) {
      if (kb + kHop < k_end) {
        fetch(page, kb + kHop, 1, k_b);
        page = page_of(kb + 2 * kHop);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kLoads) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      use(kb, 0, k_a);
      kb += kHop;
      if (kb >= k_end) break;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V of the block just used is in registers: its strip is free
      if (kb + kHop < k_end) {
        fetch(page, kb + kHop, 0, k_a);
        page = page_of(kb + 2 * kHop);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kLoads) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      use(kb, 1, k_b);
      kb += kHop;
      if (kb >= k_end) break;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  };

  // ---- the stages -------------------------------------------------------------------------------------------------------
  // At the top of stage s its keys are in buffer s & 1 for everybody and stage s + 1 is on its way into the other buffer.
  if (own_blocks) {
    __syncthreads();  // the flag is cleared
    if constexpr (kOwnBlocks) few_rows();
  } else if (n_stages > 0) {
    __syncthreads();  // the flag is cleared
    stage_arrived(k0, 0);
    lds_barrier();
    if (n_stages > 1) load_stage(table[(k0 + KS) >> kPageShift], k0 + KS, 1);
    auto page_after = [&](int s) { return table[min(k0 + (s + 2) * KS, k_end - 1) >> kPageShift]; };
    int s = 0, page = page_after(0);
    // Stages that every row of the tile sees whole run as a software pipeline: while one block's scores and values are
    // multiplied, the next operands come from LDS, so a wavefront never waits for an LDS read that it has just made.  The
    // barrier that ends a stage stands in the middle of its last block, behind that block's last LDS read.
    if constexpr (kHalf && KS == 2 * kBlockKeys) {
      const int n_fast = few || tile_first < k0 ? 0 : min((tile_first + 1 - k0) / KS, n_stages);
      if (n_fast > 0) {
        KFrag kf[2][QF];
        if (!idle) read_k(0, 0, kf);
        for (; s < n_fast; ++s) {
          const int buf = s & 1, key0 = k0 + s * KS;
          const bool more = s + 1 < n_stages;
          half8_t vf[DT];
          float4_t sc[NT][2];
          Probs pf[NT];
          if (!idle) {
            scores(kf, sc);
            read_v(buf, 0, vf);
            read_k(buf, 1, kf);
            __builtin_amdgcn_sched_barrier(0);
            softmax(sc, pf, key0, std::false_type{});
            add_values(vf, pf);
            __builtin_amdgcn_sched_barrier(0);
            scores(kf, sc);
            read_v(buf, 1, vf);
          }
          if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            stage_arrived(key0 + KS, buf ^ 1);
            lds_barrier();
            if (s + 2 < n_stages) load_stage(page, key0 + 2 * KS, buf);
            page = page_after(s + 1);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (!idle) {
            if (s + 1 < n_fast) read_k(buf ^ 1, 0, kf);
            softmax(sc, pf, key0, std::false_type{});
            add_values(vf, pf);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    for (; s < n_stages; ++s) {
      const int buf = s & 1, key0 = k0 + s * KS;
#pragma unroll
      for (int sub = 0; sub < KS / kBlockKeys; ++sub) {
        const int kb = key0 + sub * kBlockKeys;
        const bool mine = few ? sub == wave : !idle;
        if (mine && kb <= wave_last && kb < k_end) {  // wave-uniform
          if (kb + kBlockKeys - 1 > wave_first) block(buf, sub, kb, std::true_type{});
          else block(buf, sub, kb, std::false_type{});
        }
      }
      if (s + 1 < n_stages) {
        stage_arrived(key0 + KS, buf ^ 1);
        lds_barrier();
        if (s + 2 < n_stages) load_stage(page, key0 + 2 * KS, buf);
        page = page_after(s + 1);
      }
    }
  }
  if constexpr (!kHalf) {
#pragma unroll
    for (int t = 0; t < NT; ++t) lsum[t][0] = sum_xor32(sum_xor16(lsum[t][0]));
  }
  __syncthreads();
  const bool repair = *s_flag != 0;  // uniform

  const bool cut = pc.pieces > 1;
  const int64_t slot = static_cast<int64_t>(pc.slot) * a.Hkv + hk;
  if (cut && (slot >= a.slots || n_rows > a.slot_rows)) return;  // (cannot happen: the cut is bounded by both)
  auto out_row = [&](int r) -> T * {
    const int rr = row0 + r, i = rr / a.group;
    return static_cast<T *>(a.out) + (static_cast<int64_t>(pc.c0 + i) * a.Hq + hk * a.group + (rr - i * a.group)) * D;
  };

  // Infinities and NaN of V that were stored as zeros are added at the end, to element d of every row that sees their key
  // (a positive weight does not change them): rare, so through memory and without a thought for speed.
  auto finish = [&]() {
    if (!repair) return;
    __threadfence_block();
    __syncthreads();
    for (int x = tid; x < n_rows * D; x += kThreads) {
      const int r = x / D, d = x % D, last = position(r);
      float sum = 0.f;
      for (int key = max(k0, mixed_from); key < k_end && key <= last; ++key) {
        const float v = ldf(vbase + in_pool(table[key >> kPageShift]) * page_elems + static_cast<int64_t>(key & (kPageKeys - 1)) * D + d);
        if (!(fabsf(v) < __builtin_inff())) sum += v;
      }
      if (sum == 0.f) continue;
      if (cut) a.part_o[(slot * a.slot_rows + r) * D + d] += sum;
      else stf(out_row(r) + d, ldf(out_row(r) + d) + sum);
    }
  };

  if (!few) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = wrow + t * 16 + c;
      if (r >= n_rows) continue;
      const float l = lsum[t][0];
      if (cut) {
        float *po = a.part_o + (slot * a.slot_rows + r) * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4_t *>(po + dt * 16 + 4 * g) = o[t][dt];
        if (g == 0) {
          a.part_ml[(slot * a.slot_rows + r) * 2] = m[t];
          a.part_ml[(slot * a.slot_rows + r) * 2 + 1] = l;
        }
      } else {
        const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);  // no key: zeros; a NaN stays one
        S *orow = reinterpret_cast<S *>(out_row(r));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          typedef S vec4 __attribute__((ext_vector_type(4)));
          vec4 h;
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = static_cast<S>(o[t][dt][e] * inv);
          *reinterpret_cast<vec4 *>(orow + dt * 16 + 4 * g) = h;
        }
      }
    }
    finish();
    return;
  }

  // few rows: the states of the wavefronts that had keys, through LDS
  float *so = reinterpret_cast<float *>(chunk_smem);
  float *sml = so + C::kDealt * C::FEW * C::STATE;
  if (wave < C::kDealt) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = wave * C::FEW + t * 16 + c;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4_t *>(so + r * C::STATE + dt * 16 + 4 * g) = o[t][dt];
      if (g == 0) {
        sml[2 * r] = m[t];
        sml[2 * r + 1] = lsum[t][0];
      }
    }
  }
  __syncthreads();
  for (int x = tid; x < n_rows * D; x += kThreads) {
    const int r = x / D, d = x % D;
    float mx = kMasked;
#pragma unroll
    for (int w = 0; w < C::kDealt; ++w) mx = fmaxf(mx, sml[2 * (w * C::FEW + r)]);
    float l = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < C::kDealt; ++w) {
      const float f = __builtin_amdgcn_exp2f(sml[2 * (w * C::FEW + r)] - mx);
      l = __builtin_fmaf(f, sml[2 * (w * C::FEW + r) + 1], l);
      acc = add_weighted(acc, f, so[(w * C::FEW + r) * C::STATE + d]);
    }
    if (cut) {
      a.part_o[(slot * a.slot_rows + r) * D + d] = acc;
      if (d == 0) {
        a.part_ml[(slot * a.slot_rows + r) * 2] = mx;
        a.part_ml[(slot * a.slot_rows + r) * 2 + 1] = l;
      }
    } else {
      const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
      stf(out_row(r) + d, acc * inv);
    }
  }
  finish();
}

// Adds the pieces of a cut tile: out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), in the order of the keys.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void chunk_merge_kernel(ChunkArgs a) {
  using C = Cfg<T, D>;
  const int lane = threadIdx.x & 63;
  const int hk = blockIdx.x % a.Hkv;
  const Piece pc = find_piece<C::TR, true>(a, blockIdx.x / a.Hkv, lane);
  if (!pc.found) return;
  const int row0 = pc.tile * C::TR, n_rows = min(pc.rows - row0, C::TR);
  if ((static_cast<int64_t>(pc.slot) + pc.pieces - 1) * a.Hkv + hk >= a.slots || n_rows > a.slot_rows) return;
  const int64_t step = static_cast<int64_t>(a.Hkv) * a.slot_rows;
  for (int x = threadIdx.x; x < n_rows * (D / 4); x += kThreads) {
    const int r = x / (D / 4), d = x % (D / 4) * 4;
    const int64_t base = (static_cast<int64_t>(pc.slot) * a.Hkv + hk) * a.slot_rows + r;
    float mx = kMasked;
    for (int s = 0; s < pc.pieces; ++s) mx = fmaxf(mx, a.part_ml[(base + s * step) * 2]);
    float l = 0.f;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < pc.pieces; ++s) {
      const float f = __builtin_amdgcn_exp2f(a.part_ml[(base + s * step) * 2] - mx);
      l = __builtin_fmaf(f, a.part_ml[(base + s * step) * 2 + 1], l);
      const float4_t o = *reinterpret_cast<const float4_t *>(a.part_o + (base + s * step) * D + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = add_weighted(acc[e], f, o[e]);
    }
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
    const int rr = row0 + r, i = rr / a.group;
    T *out = static_cast<T *>(a.out) + (static_cast<int64_t>(pc.c0 + i) * a.Hq + hk * a.group + (rr - i * a.group)) * D + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) stf(out + e, acc[e] * inv);
  }
}

struct Sizes {
  int64_t tiles;      // at most, per kv head
  int64_t grid;       // pieces at most, per kv head
  int64_t slots;      // pieces of cut tiles at most, over the kv heads
  int64_t cut_tiles;  // cut tiles at most, per kv head
  int slot_rows, target;
};
// Bounds of the cut for any cu_tokens and start within tokens, B, max_q and max_len.  With q units per piece, q >= work / target
// and pieces = ceil(units / q) > 1 for a cut tile: its pieces are at most 2 units / q, all cut tiles' together at most
// 2 work / q <= 2 target.
Sizes sizes_for(int tile_rows, int tokens, int B, int Hkv, int group, int max_q, int max_len) {
  Sizes z{};
  const int64_t rows = static_cast<int64_t>(tokens) * group;
  z.tiles = rows / tile_rows + B;
  const int64_t per_seq = (static_cast<int64_t>(max_q) * group + tile_rows - 1) / tile_rows;
  if (z.tiles > per_seq * B) z.tiles = per_seq * B;
  z.target = 2 * device_cu_count();
  const int64_t units = (static_cast<int64_t>(max_len) + 127) / 128;
  const int64_t most = (units + kMinPieceUnits - 1) / kMinPieceUnits;  // pieces of one tile
  const int64_t cut = 2 * static_cast<int64_t>(z.target) / Hkv + 1;    // pieces of cut tiles, per kv head
  if (most <= 1) {
    z.grid = z.tiles;
  } else {
    const int64_t all = z.tiles * most < cut ? z.tiles * most : cut;
    z.grid = z.tiles + all < z.tiles * most ? z.tiles + all : z.tiles * most;
    z.slots = all * Hkv;
    z.cut_tiles = all / 2 < z.tiles ? (all / 2 > 0 ? all / 2 : 1) : z.tiles;
    const int64_t rows_seq = static_cast<int64_t>(max_q) * group;
    z.slot_rows = static_cast<int>(rows_seq < tile_rows ? (rows_seq + 15) / 16 * 16 : tile_rows);
  }
  return z;
}
int tile_rows_of(int dtype, int D) { return D == 256 || (dtype == AXHIP_FLOAT32 && D == 128) ? 64 : 128; }

template <typename T, int D>
int launch(const ChunkArgs &a, const Sizes &z, hipStream_t st) {
  using C = Cfg<T, D>;
  static std::atomic<uint64_t> raised{0};
  const int rc = raise_dynamic_lds(reinterpret_cast<const void *>(&chunk_attn_kernel<T, D>), C::kLdsBytes, raised);
  if (rc != AXHIP_OK) return rc;
  hipLaunchKernelGGL((chunk_attn_kernel<T, D>), dim3(static_cast<unsigned>(z.grid * a.Hkv)), dim3(kThreads), C::kLdsBytes, st, a);
  if (z.cut_tiles > 0)
    hipLaunchKernelGGL((chunk_merge_kernel<T, D>), dim3(static_cast<unsigned>(z.cut_tiles * a.Hkv)), dim3(kThreads), 0, st, a);
  return launch_status();
}

bool aligned_to(const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The checks that both entry points make.
int check_sizes(int dtype, int tokens, int B, int Hq, int Hkv, int D, int max_q, int max_len) {
  if (!is_float_dtype(dtype)) return AXHIP_UNSUPPORTED_TYPE;
  if (tokens < 0 || B < 0 || Hq <= 0 || Hkv <= 0 || max_q < 0 || max_len < 0) return AXHIP_INVALID_ARGUMENT;
  if (Hq % Hkv != 0) return AXHIP_SHAPE_MISMATCH;
  if (D != 64 && D != 128 && D != 256) return AXHIP_INVALID_ARGUMENT;
  if (B > (1 << 20) || Hkv > 1024 || static_cast<int64_t>(tokens) * Hq > (int64_t(1) << 30) || max_len > (1 << 30))
    return AXHIP_INVALID_ARGUMENT;
  return AXHIP_OK;
}

}  // namespace
}  // namespace axhip

using namespace axhip;

extern "C" {

AXHIP_API size_t axhip_chunk_attention_paged_workspace_bytes(int dtype, int tokens, int B, int Hq, int Hkv, int D, int max_q,
                                                             int max_len) {
  if (check_sizes(dtype, tokens, B, Hq, Hkv, D, max_q, max_len) != AXHIP_OK) return 0;
  if (max_q > tokens) max_q = tokens;
  const Sizes z = sizes_for(tile_rows_of(dtype, D), tokens, B, Hkv, Hq / Hkv, max_q, max_len);
  return static_cast<size_t>(z.slots) * z.slot_rows * (D + 2) * sizeof(float);
}

AXHIP_API int axhip_chunk_attention_paged(const void *q, const void *k_pool, const void *v_pool, const int32_t *page_table,
                                          const int32_t *cu_tokens, const int32_t *start, void *out, void *workspace,
                                          size_t workspace_bytes, int dtype, int tokens, int B, int Hq, int Hkv, int D,
                                          int max_q, int max_len, int max_pages, int n_pages, axhip_stream stream) {
  const int rc = check_sizes(dtype, tokens, B, Hq, Hkv, D, max_q, max_len);
  if (rc != AXHIP_OK) return rc;
  if (max_pages <= 0 || n_pages <= 0 || static_cast<int64_t>(max_pages) * kPageKeys < max_len) return AXHIP_INVALID_ARGUMENT;
  if (tokens == 0 || B == 0 || max_q == 0) return AXHIP_OK;
  if (!q || !k_pool || !v_pool || !page_table || !cu_tokens || !start || !out) return AXHIP_INVALID_PTR;
  if (!aligned_to(q, 16) || !aligned_to(k_pool, 16) || !aligned_to(v_pool, 16) || !aligned_to(out, 16) ||
      !aligned_to(page_table, 4) || !aligned_to(cu_tokens, 4) || !aligned_to(start, 4))
    return AXHIP_INVALID_PTR;
  if (max_q > tokens) max_q = tokens;
  const int group = Hq / Hkv;
  const Sizes z = sizes_for(tile_rows_of(dtype, D), tokens, B, Hkv, group, max_q, max_len);
  const size_t need = static_cast<size_t>(z.slots) * z.slot_rows * (D + 2) * sizeof(float);
  if (need && (!workspace || !aligned_to(workspace, 16))) return AXHIP_INVALID_PTR;
  if (workspace_bytes < need) return AXHIP_OUT_OF_MEMORY;
  if (z.grid * Hkv > INT32_MAX) return AXHIP_INVALID_ARGUMENT;
  ChunkArgs a{};
  a.q = q;
  a.k = k_pool;
  a.v = v_pool;
  a.page_table = page_table;
  a.cu = cu_tokens;
  a.start = start;
  a.out = out;
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = a.part_o + static_cast<size_t>(z.slots) * z.slot_rows * D;
  a.tokens = tokens;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.group = group;
  a.max_q = max_q;
  a.max_len = max_len;
  a.max_pages = max_pages;
  a.n_pages = n_pages;
  a.slots = static_cast<int>(z.slots);
  a.slot_rows = z.slot_rows;
  a.target = z.target;
  a.scale_log2e = 1.4426950408889634f / sqrtf(static_cast<float>(D));
  hipStream_t st = as_stream(stream);
  if (dtype == AXHIP_FLOAT16) {
    if (D == 64) return launch<__half, 64>(a, z, st);
    if (D == 128) return launch<__half, 128>(a, z, st);
    return launch<__half, 256>(a, z, st);
  }
  if (D == 64) return launch<float, 64>(a, z, st);
  if (D == 128) return launch<float, 128>(a, z, st);
  return launch<float, 256>(a, z, st);
}

}  // extern "C"
