// Attention of a ragged batch of new tokens over a paged KV cache that already holds their keys and values.
//
//   out_i = sum_{j <= p_i} softmax_j(q_i . k_j / sqrt(D)) v_j,   p_i = start[b] + i the position of the i-th new token of b.
//
// Work decomposition.  The G = Hq / Hkv query heads of a kv head see the same keys, so the new tokens of a sequence give
// n G "rows" per kv head, row r = (token r / G, head r % G): any G, and positions that grow with r.  A workgroup of four
// wavefronts takes a tile of up to 64 NT rows of one (sequence, kv head) and a piece of the keys they see; a wavefront
// takes NT column tiles of 16 rows.  In a tile with few rows (at most 16 NT: decoding sequences, drafts, the last rows of
// a chunk) all wavefronts take the same rows and deal the keys among themselves in blocks of 32; their states are added up at
// the end.  (D = 256: a stage is one block, so one wavefront multiplies there and the others only load.)
//
// Everything is computed transposed, so that no operand changes its layout in registers (see the products below):
//   S^T = K . Q^T  (16 keys x 16 rows), O^T += V^T . P^T  (16 d x 16 rows); a lane owns the row lane % 16 in both.
// K and V travel through LDS in stages of KS keys (double-buffered, 16-byte units XOR-swizzled by key).  A stage lies
// inside one page of 128 keys, so its address is one page number (read a stage ahead) and fixed lane offsets, and every
// address of a stage is inside the pool whatever the lengths are.
//
// Few tiles over many keys would leave the device idle: the keys of a tile are cut into pieces so that the launch has
// about two workgroups per CU (fp32 with D = 64: three) of equal work.  The cut is made on the device from cu_tokens and start
// (every workgroup derives it with a few wave operations), so a captured launch follows lengths that change.  A piece of a cut tile leaves
// an unnormalised state in the workspace; a second kernel adds the pieces of a tile in a fixed order.  No counters, no
// state between launches: launches with workspaces of their own may overlap.
//
// What bounds it, fp16 D = 128 (figures here and below: Hq / Hkv behind the tokens): from about 32 rows of a kv head on the matrix cores
// beside the exponentials (16 x 4096 tokens, 16 / 8: 1145 us = 960 TFLOP/s, 2048 tokens at 129024 keys, 16 / 8: 1940 us =
// 1125 TFLOP/s, where a large library product reaches 1144); below that the stream of keys (4 tokens each of 32 sequences of up to
// 8192 keys, 32 / 8: 537 MB read in 97 us = 5.5 TB/s, with the merge 110 to 128 us, box to box) and, where there are few keys
// too, the plan, the merge and the two launches (about 5 us).
//
// fp32 statistics throughout.  fp16: probabilities are rounded to fp16 for the second product (2^-11 of their value at
// most; see softmax()), numerator and denominator from the same rounded values.  fp32: fp32 matrix instructions.
#include "common.hpp"

#include <type_traits>

namespace axhip {
namespace {

constexpr int kThreads = 256;
constexpr int kWavesWg = 4;
constexpr int kPageKeys = 128, kPageShift = 7;
constexpr int kBlockKeys = 32;      // keys of one softmax step
constexpr int64_t kMostWorkgroups = (1 << 24) - 1;  // a launch has less than 2^32 threads
constexpr float kMasked = -3.40282347e38f;  // below every finite score
typedef float float8_t __attribute__((ext_vector_type(8)));

struct ChunkArgs {
  const void *q, *k, *v;
  const int32_t *page_table, *cu, *start;
  void *out;
  float *part_o;   // [slots][slot_rows][D]
  float *part_ml;  // [slots][slot_rows][2]: level (log2 units), sum
  int tokens, B, Hq, Hkv, group, max_q, max_len, max_pages, n_pages;
  int slots, slot_rows, target;  // target: pieces the launch aims at
  int merge_rows;                // rows per workgroup of the merge
  float scale_log2e;
};

template <typename T, int D>
struct Cfg {
  // Column tiles per wavefront, the fewest units of 128 keys of a piece, and the workgroups per CU that the cut aims at.
  // fp32 products take long enough for one column tile, and with half the rows in a tile and pieces of a single unit small
  // batches spread over more workgroups (D = 64, against 2 tiles, 2 units, 2 workgroups): 200 tokens of 3 prompts, 8 / 4,
  // 16 us against 27, 16 decoding sequences at 2000 keys, 16 / 8, 25 against 31, 4096 tokens of one prompt, 8 / 4, 167 against
  // 211.  A third workgroup fits there only (registers): 167 us against 225 with two; four pieces per CU: 300 tokens at 6000
  // keys, 4 / 1, 37 us against 32.  fp16 is slower with pieces of one unit (512 tokens of one prompt, 32 / 8, D = 128, 25 us against
  // 23) and gains nothing from three workgroups (D = 64: 4 x 1000 tokens at up to 2000 keys, 16 / 8, 64 us against 62; D = 128
  // has registers for two).
  static constexpr int NT = D == 256 || sizeof(T) == 4 ? 1 : 2;
  static constexpr int MIN = sizeof(T) == 4 ? 1 : 2;
  static constexpr int AIM = D == 64 && sizeof(T) == 4 ? 3 : 2;
  static constexpr int TR = kWavesWg * 16 * NT;                        // rows per tile
  static constexpr int FEW = 16 * NT;                                  // rows up to which wavefronts deal the keys
  static constexpr int KS = D == 256 || sizeof(T) == 4 ? 32 : 64;  // keys per stage
  static constexpr int E = 16 / sizeof(T);                             // elements per 16-byte unit
  static constexpr int UPR = D / E;                                    // units per row
  static constexpr int SW = (UPR < 16 ? UPR : 16) - 1;                 // swizzle mask
  static constexpr int VEC = KS * UPR / kThreads;                      // units per thread, tensor and stage
  static constexpr bool kOwnBlocks = D <= 128;                         // see Wave::own_blocks
  static constexpr int STATE = D + 4;                                  // row stride of the states added up in LDS
  static constexpr int kStageBytes = 4 * KS * D * static_cast<int>(sizeof(T));
  // wavefronts with keys of their own in a tile of few rows
  static constexpr int kDealt = kOwnBlocks ? kWavesWg : (KS / kBlockKeys < kWavesWg ? KS / kBlockKeys : kWavesWg);
  static constexpr int kStateBytes = kDealt * FEW * (STATE + 2) * 4;
  static constexpr int kTail = kStageBytes > kStateBytes ? kStageBytes : kStateBytes;  // where the flags are
  static constexpr int kLdsBytes = kTail + 16 + TR * 4;
};

// ---- the cut -------------------------------------------------------------------------------------------------------
struct Seq {
  int c0, start, rows, tiles;  // first token, its position, rows per kv head, tiles
  int units;                   // of 128 keys, of the last tile
};
template <int TR>
__device__ __forceinline__ Seq load_seq(const ChunkArgs &a, int b) {
  Seq s{0, 0, 0, 0, 0};
  if (b < a.B) {
    s.c0 = min(max(a.cu[b], 0), a.tokens);
    const int c1 = min(max(a.cu[b + 1], s.c0), a.tokens);
    const int n = min(c1 - s.c0, a.max_q);
    s.start = a.start[b];
    const int64_t last = static_cast<int64_t>(s.start) + n;  // keys the last token sees
    s.units = (static_cast<int>(last < 0 ? 0 : (last > a.max_len ? a.max_len : last)) + 127) >> 7;
    s.rows = n * a.group;
    s.tiles = (s.rows + TR - 1) / TR;
  }
  return s;
}
// The last key that row r of a sequence sees, -1: none.
__device__ __forceinline__ int last_key(const ChunkArgs &a, int start, int r) {
  const int64_t p = static_cast<int64_t>(start) + r / a.group;
  return static_cast<int>(p < -1 ? -1 : (p > a.max_len - 1 ? a.max_len - 1 : p));
}
// Units per piece: the work of a kv head (every tile taken as long as its sequence's last) over the pieces aimed at.
template <typename C>
__device__ __forceinline__ int units_per_piece(const ChunkArgs &a, const Seq &first, int lane) {
  float work = 0.f;
  for (int j = 0; j < a.B; j += 64) {
    const Seq s = j == 0 ? first : load_seq<C::TR>(a, j + lane);
    work += group_sum<64>(static_cast<float>(s.tiles) * static_cast<float>(s.units));
  }
  const float q = ceilf(work * static_cast<float>(a.Hkv) / static_cast<float>(a.target));
  return __builtin_amdgcn_readfirstlane(max(C::MIN, static_cast<int>(fminf(q, 1.0e9f))));
}
// Pieces of every tile of a sequence.  One that has few rows only streams keys, each its own: shorter pieces spread such
// streams better over the device (32 sequences of up to 4000 keys, 16 / 8, 60 us, 65 us with whole pieces), while tiles of many
// rows that start together share their keys in the caches.  Pieces that are short anyway stay whole (1 sequence of 32000 keys,
// 16 / 8, pieces of 4 units 35 us, of 2 units 38 us).
template <typename C>
__device__ __forceinline__ int pieces_of(const Seq &s, int per) {
  const int p = C::kOwnBlocks && s.rows <= C::FEW && per >= 8 ? (per + 1) / 2 : per;
  return max(1, (s.units + p - 1) / p);
}

struct Piece {
  int b, tile, piece, pieces, slot, c0, start, rows;
};
// The `flat`-th piece (MERGE: the `flat`-th cut tile) of a kv head; false: there is none.  slot: number of the piece (MERGE: of
// the tile's first piece) among the pieces of cut tiles.
template <typename C, bool MERGE>
__device__ __forceinline__ bool find_piece(const ChunkArgs &a, int flat, int lane, Piece &p) {
  const Seq first = load_seq<C::TR>(a, lane);
  const int per = units_per_piece<C>(a, first, lane);
  int done = 0, slots = 0;
  for (int j = 0; j < a.B; j += 64) {
    const Seq s = j == 0 ? first : load_seq<C::TR>(a, j + lane);
    const int pieces = pieces_of<C>(s, per);
    const bool cut = pieces > 1;
    const int mine = MERGE ? (cut ? s.tiles : 0) : s.tiles * pieces;
    const int upto = done + wave_prefix_i32(mine);
    const int my_slots = cut ? s.tiles * pieces : 0;
    const int slots_upto = slots + wave_prefix_i32(my_slots);
    const uint64_t hit = __ballot(flat < upto);
    if (hit) {
      const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      auto at = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int rest = flat - at(upto - mine);
      if (static_cast<unsigned>(rest) >= static_cast<unsigned>(at(mine))) return false;  // (sums past 31 bits: cu falls and rises)
      p.b = j + l;
      p.c0 = at(s.c0);
      p.start = at(s.start);
      p.rows = at(s.rows);
      p.pieces = at(pieces);
      const int order = MERGE ? rest : rest / p.pieces;
      p.piece = MERGE ? 0 : rest - order * p.pieces;
      p.tile = at(s.tiles) - 1 - order;  // the tiles that see most keys first
      p.slot = at(slots_upto - my_slots) + p.tile * p.pieces + p.piece;
      return true;
    }
    done = __builtin_amdgcn_readlane(upto, 63);
    slots = __builtin_amdgcn_readlane(slots_upto, 63);
  }
  return false;
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

// One wavefront's part of a piece of a tile: its rows' queries, statistics and results, and the steps of a block of 32 keys.
template <typename T, int D>
struct Wave {
  using C = Cfg<T, D>;
  static constexpr bool kHalf = sizeof(T) == 2;
  using S = typename std::conditional<kHalf, _Float16, float>::type;
  using KFrag = typename std::conditional<kHalf, half8_t, float>::type;
  using Probs = typename std::conditional<kHalf, half8_t, float8_t>::type;
  using VFrag = Probs;  // of a d tile
  static constexpr int NT = C::NT, KS = C::KS, UPR = C::UPR, SW = C::SW, DT = D / 16;
  static constexpr int QF = kHalf ? D / 32 : D / 4;  // operand registers of a column tile (8 halves or 1 float each)
  static constexpr int kRow = D * static_cast<int>(sizeof(T)), kTensor = 2 * KS * kRow;  // bytes: a row, both stages of K
  // A row's 16-byte units lie XORed by these, so that the lanes of a read find 256 bytes of different banks: the same unit of 16
  // rows of K; a pair of units of 8 rows of V.  Linear in the row's bits.
  static constexpr __host__ __device__ int swz_k(int row) { return kHalf && D == 64 ? (row >> 1) & SW : row & SW; }
  static constexpr __host__ __device__ int swz_v(int row) { return !kHalf ? row & SW : (D == 64 ? row & 6 : (2 * row) & 14); }

  const ChunkArgs &a;
  const Piece &pc;
  int tid, wave, lane, c, g, hk;
  int row0, n_rows, wrow;            // the tile's first row, its rows, this wavefront's first
  int k0, k_end, mixed_from;         // keys of the piece; see clean()
  int wave_first, wave_last;         // last keys that the first and the last of the wavefront's rows see
  int pos[NT];                       // of this lane's rows
  int kaddr, vaddr;
  const T *kbase, *vbase;
  int64_t page_elems;
  // page numbers by scalar loads: a vector load would have to be waited for behind the stage on its way
  typedef const int32_t __attribute__((address_space(4))) *scalar_ptr;
  scalar_ptr table;
  lds_byte *smem;
  // flags[0]: some unit of V was cleaned; flags[1]: some result is a NaN that its row's sum does not explain; row_nan[r]: row r's
  // sum is a NaN
  int *flags, *row_nan;
  KFrag qf[NT][QF];
  float4_t o[NT][DT], lsum[NT];
  float m[NT];

  __device__ __forceinline__ Wave(const ChunkArgs &args, const Piece &piece, int head, bool few)
      : a(args), pc(piece), hk(head) {
    tid = threadIdx.x;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    lane = tid & 63;
    c = lane & 15;
    g = lane >> 4;
    smem = (lds_byte *)chunk_smem;
    flags = reinterpret_cast<int *>(chunk_smem + C::kTail);
    row_nan = flags + 4;
    row0 = pc.tile * C::TR;
    n_rows = min(pc.rows - row0, C::TR);
    // rows past the tile repeat its last one and are not stored
    wrow = few ? 0 : wave * 16 * NT;
#pragma unroll
    for (int t = 0; t < NT; ++t) pos[t] = position(min(wrow + t * 16 + c, n_rows - 1));
    wave_first = position(min(wrow, n_rows - 1));
    wave_last = position(min(wrow + 16 * NT, n_rows) - 1);
    const int tile_first = position(0), k_all = position(n_rows - 1) + 1;  // keys the tile sees: [0, k_all)
    const int units = (k_all + 127) >> 7;
    k0 = static_cast<int>(static_cast<int64_t>(units) * pc.piece / pc.pieces) << 7;
    k_end = min(static_cast<int>(static_cast<int64_t>(units) * (pc.piece + 1) / pc.pieces) << 7, k_all);
    mixed_from = tile_first < 0 ? 0 : (tile_first + 1) / KS * KS;
    table = (scalar_ptr)(a.page_table + static_cast<int64_t>(pc.b) * a.max_pages);
    page_elems = static_cast<int64_t>(a.Hkv) * kPageKeys * D;
    kbase = static_cast<const T *>(a.k) + static_cast<int64_t>(hk) * kPageKeys * D;
    vbase = static_cast<const T *>(a.v) + static_cast<int64_t>(hk) * kPageKeys * D;
    // Where this lane reads its operands, as byte offsets into a stage of K / V; the steps of the products flip or add constant
    // bits of them.  Made opaque where they are used, or the compiler keeps every one of the flipped offsets in registers.
    kaddr = c * kRow + (g ^ swz_k(c)) * 16;
    const int vkey = kHalf ? 4 * g + (c >> 2) : 4 * g;
    vaddr = vkey * kRow + (kHalf ? ((((c & 3) >> 1) ^ swz_v(vkey)) * 16 + (c & 1) * 8) : (c ^ swz_v(vkey)) * 16);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = kMasked;
      lsum[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[t][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
  }

  __device__ __forceinline__ int position(int r) const { return last_key(a, pc.start, row0 + r); }
  __device__ __forceinline__ int64_t row_at(int r) const {  // of q and out
    const int rr = row0 + r, i = rr / a.group;
    return (static_cast<int64_t>(pc.c0 + i) * a.Hq + hk * a.group + (rr - i * a.group)) * D;
  }
  __device__ __forceinline__ int page_of(int key) const { return table[min(key, k_end - 1) >> kPageShift]; }
  __device__ __forceinline__ int64_t key_at(int page, int key) const {  // a page number outside the pool is clamped into it
    return min(max(page, 0), a.n_pages - 1) * page_elems + static_cast<int64_t>(key & (kPageKeys - 1)) * D;
  }

  // Q as the right operand of the first product, for the whole piece.  fp32: product step 4 i + e takes d = 16 i + 4 g + e, so that a
  // lane's operands of four steps are one 16-byte unit, of Q as of K.
  __device__ __forceinline__ void load_q() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const S *qrow = static_cast<const S *>(a.q) + row_at(min(wrow + t * 16 + c, n_rows - 1));
#pragma unroll
      for (int i = 0; i < D * static_cast<int>(sizeof(T)) / 64; ++i) {
        if constexpr (kHalf) {
          qf[t][i] = *reinterpret_cast<const half8_t *>(qrow + i * 32 + g * 8);
        } else {
          const float4_t x = *reinterpret_cast<const float4_t *>(qrow + i * 16 + g * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[t][4 * i + e] = x[e];
        }
      }
    }
  }

  // Zero probability times infinity or NaN is NaN.  Where every row of the tile sees the key finish() sets that right; V must not
  // hold any where some row does not.
  // clean(): a 16-byte unit of V of key `key` in LDS becomes zeros behind the piece's last key, and loses its infinities and
  // NaN (true: it had some); finish() gives them at the end to the rows that see them.  Keys from mixed_from on, a multiple
  // of KS, are cleaned: every key that some row does not see is among them, and every key behind the last.
  __device__ __forceinline__ bool clean(lds_byte *place, int key) const {
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
  }

  __device__ __forceinline__ void read_k(int place, KFrag (&kf)[2][QF]) const {  // place: byte offset of the block's rows
    int ka = kaddr + place;
    asm volatile("" : "+v"(ka));
#pragma unroll
    for (int tk = 0; tk < 2; ++tk)
#pragma unroll
      for (int i = 0; i < kRow / 64; ++i) {
        if constexpr (kHalf) {
          kf[tk][i] = lds_at<KFrag>(smem, (ka ^ (i * 64)) + tk * 16 * kRow);
        } else {
          const float4_t x = lds_at<float4_t>(smem, (ka ^ (i * 64)) + tk * 16 * kRow);
#pragma unroll
          for (int e = 0; e < 4; ++e) kf[tk][4 * i + e] = x[e];
        }
      }
  }
  // V^T fragments of a block, d tile by d tile.  fp32: product step (tk, e) takes keys tk * 16 + 4 g + e, g = 0 .. 3, so that
  // a lane's score register e is its right operand; d tile 4 h + i holds d = 64 h + 4 c + i, so that a lane's operands of four
  // tiles are one 16-byte unit (single floats in their place: 3 x 819 tokens at up to 17600 keys, 2 / 1, D = 128, 332 us against 298).
  __device__ __forceinline__ void read_v(int place, VFrag (&vf)[DT]) const {
    int va = vaddr + place;
    asm volatile("" : "+v"(va));
    if constexpr (kHalf) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const half4_t lo = lds_tr(smem, va ^ (dt * 32)), hi = lds_tr(smem, (va ^ (dt * 32)) + 16 * kRow);
        vf[dt] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int h = 0; h < DT / 4; ++h) {
          const float4_t x = lds_at<float4_t>(smem, (va ^ ((j & 3) * 16)) + ((j >> 2) * 16 + (j & 3)) * kRow + h * 256);
#pragma unroll
          for (int i = 0; i < 4; ++i) vf[4 * h + i][j] = x[i];
        }
    }
  }
  // Four results of this lane that lie side by side in a row, and where: n counts them, n < DT.
  __device__ __forceinline__ float4_t four(int t, int n) const {
    if constexpr (kHalf) return o[t][n];
    else return float4_t{o[t][n & ~3][n & 3], o[t][(n & ~3) + 1][n & 3], o[t][(n & ~3) + 2][n & 3], o[t][(n & ~3) + 3][n & 3]};
  }
  __device__ __forceinline__ int four_at(int n) const { return kHalf ? n * 16 + 4 * g : (n >> 2) * 64 + 16 * g + 4 * (n & 3); }
  __device__ __forceinline__ void scores(const KFrag (&kf)[2][QF], float4_t (&sc)[NT][2]) const {
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
  }
  template <bool MASK>
  __device__ __forceinline__ float score(const float4_t (&sc)[NT][2], int kb, int t, int j) const {
    const float v = sc[t][j >> 2][j & 3];
    return MASK && kb + (j >> 2) * 16 + 4 * g + (j & 3) > pos[t] ? kMasked : v;
  }
  template <bool MASK>
  __device__ __forceinline__ void exps(const float4_t (&sc)[NT][2], int kb, float (&p)[NT][8]) const {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = score<MASK>(sc, kb, t, j);
        p[t][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.scale_log2e, -m[t]));
        if (MASK && x <= kMasked) p[t][j] = 0.f;
      }
  }
  // Probabilities against a level that follows the running maximum: it is moved, and everything rescaled, only when one of
  // them passes kTop (the first block of a row always does).  Until then a block needs no maximum over its row at all.
  // fp16: the level lies 2^kBelow under the maximum that set it, so that p is 2^10 at the maximum and 2^15 at most: below
  // 2^-24 of the largest weight of a row its others lose bits, below 2^-35 they are lost.  (Against the maximum itself those
  // under 2^-25 would be, and 65536 such keys hold 2^-9 of the sum.)
  // fp32: the level lies 2^8 above, so that p is at most 1 and a sum of weighted values ends where the sum of the values does.
  static constexpr float kBelow = kHalf ? 10.f : -8.f, kTop = kHalf ? 32768.f : 1.f;
  // Large scores: the level is a product rounded to fp32, taken a step or two low so that the largest score never lies under what it
  // was meant to be over.  Where a step is more than kTop leaves room for (levels past 2^23) p ends at kTop: scores within
  // 2^-22 of the largest then weigh the same, which is what the rounding of their own sums leaves of them.
  // MASK: some key of the block at kb is behind some row's position.
  template <bool MASK>
  __device__ __forceinline__ void softmax(const float4_t (&sc)[NT][2], int kb, Probs (&pf)[NT]) {
    float p[NT][8];
    exps<MASK>(sc, kb, p);
    float top = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, p[t][j]);
    if (__builtin_expect(__any(top > kTop), 0)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float mx = score<MASK>(sc, kb, t, 0);
#pragma unroll
        for (int j = 1; j < 8; ++j) mx = fmaxf(mx, score<MASK>(sc, kb, t, j));
        const float level = __builtin_fmaf(max_xor32(max_xor16(mx)), a.scale_log2e, -kBelow);
        const float mnew = fmaxf(m[t], level * (level > 0.f ? 1.f - 0x1p-23f : 1.f + 0x1p-23f));
        const float corr = __builtin_amdgcn_exp2f(m[t] - mnew);
        m[t] = mnew;
        lsum[t] *= corr;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[t][dt] *= corr;
      }
      exps<MASK>(sc, kb, p);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j) p[t][j] = p[t][j] > kTop ? kTop : p[t][j];  // (a NaN stays one)
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (kHalf) pf[t][j] = static_cast<_Float16>(p[t][j]);
        else pf[t][j] = p[t][j];
      }
  }
  __device__ __forceinline__ void add_values(const VFrag (&vf)[DT], const Probs (&pf)[NT]) {
    if constexpr (kHalf) {
      const half8_t ones = {1, 1, 1, 1, 1, 1, 1, 1};
      // the row sums as a product with ones: every register of the result holds the row's sum
#pragma unroll
      for (int t = 0; t < NT; ++t) lsum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[t], lsum[t], 0, 0, 0);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[dt], pf[t], o[t][dt], 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int t = 0; t < NT; ++t) lsum[t][0] += pf[t][j];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int t = 0; t < NT; ++t) o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[dt][j], pf[t][j], o[t][dt], 0, 0, 0);
      }
    }
  }
  template <bool MASK>
  __device__ __forceinline__ void block(int buf, int sub, int kb) {
    KFrag kf[2][QF];
    float4_t sc[NT][2];
    Probs pf[NT];
    const int place = (buf * KS + sub * kBlockKeys) * kRow;
    read_k(place, kf);
    scores(kf, sc);
    softmax<MASK>(sc, kb, pf);
    VFrag vf[DT];
    read_v(kTensor + place, vf);
    add_values(vf, pf);
  }

  // ---- the keys in stages that the workgroup shares -------------------------------------------------------------------------
  // K and V go from memory to LDS directly (16 bytes a lane; a wavefront fills 1 KiB in lane order, so the swizzle is made on
  // the side of memory: the lane of place u of a row fetches unit u ^ swz(row)).  Load p of a thread covers row
  // p kStep + tid / UPR of the stage; its offset within the page differs by constants from load 0's.
  static constexpr int kStep = kThreads / UPR;
  __device__ __forceinline__ void load_stage(int page, int key0, int buf) const {
    const int64_t base = key_at(page, key0);
    const unsigned place = buf * (KS * kRow) + wave * 1024;
    const unsigned koff = tid / UPR * kRow + ((tid % UPR) ^ swz_k(tid / UPR)) * 16;
    const unsigned voff = tid / UPR * kRow + ((tid % UPR) ^ swz_v(tid / UPR)) * 16;
#pragma unroll
    for (int p = 0; p < C::VEC; ++p) {
      load_lds16(kbase + base, (koff ^ (swz_k(p * kStep) * 16)) + p * kStep * kRow, smem + place + p * kThreads * 16);
      load_lds16(vbase + base, (voff ^ (swz_v(p * kStep) * 16)) + p * kStep * kRow, smem + kTensor + place + p * kThreads * 16);
    }
  }
  // The units that this thread has fetched are in LDS, and clean.  (The barrier behind this call makes them everybody's.)
  // NEXT: another stage's loads have been issued since, and stay under way.
  template <bool NEXT = false>
  __device__ __forceinline__ void stage_arrived(int key0, int buf) const {
    if constexpr (NEXT) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * C::VEC) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (key0 + KS > mixed_from) {  // uniform
      bool bad = false;
#pragma unroll 1
      for (int p = 0; p < C::VEC; ++p)
        bad |= clean(smem + kTensor + buf * (KS * kRow) + (p * kThreads + tid) * 16, key0 + p * kStep + tid / UPR);
      if (bad) flags[0] = 1;
    }
  }
  static __device__ __forceinline__ void products(bool on) {
    if (on) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
  }
  // At the top of stage s its keys are in buffer s & 1 for everybody and stage s + 1 is on its way into the other buffer.
  // few: the wavefronts have the same rows and deal the blocks of a stage.
  __device__ __forceinline__ void shared_stages(bool few) {
    const int n_stages = k_end > k0 ? (k_end - k0 + KS - 1) / KS : 0;
    const bool idle = wrow >= n_rows;  // a wavefront without rows only loads
    if (n_stages == 0) return;
    const int page0 = page_of(k0), page1 = page_of(k0 + KS);
    int s = 0, page = page_of(k0 + 2 * KS);
    load_q();
    asm volatile("" ::: "memory");  // the queries' loads are issued before the stages'
    load_stage(page0, k0, 0);
    lds_barrier();  // the flags are cleared
    if (n_stages > 1) {
      load_stage(page1, k0 + KS, 1);
      stage_arrived<true>(k0, 0);
    } else {
      stage_arrived(k0, 0);
    }
    lds_barrier();
    // Stages that every row of the tile sees whole run as a software pipeline: while one block's scores and values are
    // multiplied, the next operands come from LDS, so a wavefront never waits for an LDS read that it has just made.  The
    // barrier that ends a stage stands in the middle of its last block, behind that block's last LDS read.
    // Of the two or three wavefronts of a SIMD the one at its products goes first: they fall out of step, and one's products run
    // under another's exponentials (2048 tokens at 129024 keys, 16 / 8, 2130 -> 1995 us, 16 x 4096 tokens 1188 -> 1151 us).
    if constexpr (!kHalf || D <= 128) {  // (fp32, D = 128: 4 x 512 tokens, 16 / 8, 80 us, 82 us without; fp16, D = 256: spills)
      const int seen = position(0) + 1 - k0;  // keys of the piece that all rows see
      const int n_fast = few || seen <= 0 ? 0 : min(seen / KS, n_stages);
      if (n_fast > 0) {
        KFrag kf[2][QF];
        if (!idle) read_k(0, kf);
        for (; s < n_fast; ++s) {
          const int buf = s & 1, key0 = k0 + s * KS, place = buf * (KS * kRow);
          VFrag vf[DT];
          float4_t sc[NT][2];
          Probs pf[NT];
          if (!idle) {
#pragma unroll
            for (int sub = 0; sub + 1 < KS / kBlockKeys; ++sub) {
              products(true);
              scores(kf, sc);
              read_v(kTensor + place + sub * kBlockKeys * kRow, vf);
              read_k(place + (sub + 1) * kBlockKeys * kRow, kf);
              __builtin_amdgcn_sched_barrier(0);
              products(false);
              softmax<false>(sc, key0, pf);
              products(true);
              add_values(vf, pf);
              __builtin_amdgcn_sched_barrier(0);
            }
            products(true);
            scores(kf, sc);
            read_v(kTensor + place + (KS - kBlockKeys) * kRow, vf);
          }
          if (s + 1 < n_stages) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            stage_arrived(key0 + KS, buf ^ 1);
            lds_barrier();
            if (s + 2 < n_stages) load_stage(page, key0 + 2 * KS, buf);
            page = page_of(key0 + 3 * KS);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (!idle) {
            if (s + 1 < n_fast) read_k((buf ^ 1) * (KS * kRow), kf);
            products(false);
            softmax<false>(sc, key0, pf);
            products(true);
            add_values(vf, pf);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        products(false);
      }
    }
    for (; s < n_stages; ++s) {
      const int buf = s & 1, key0 = k0 + s * KS;
#pragma unroll
      for (int sub = 0; sub < KS / kBlockKeys; ++sub) {
        const int kb = key0 + sub * kBlockKeys;
        const bool mine = few ? sub == wave : !idle;
        if (mine && kb <= wave_last && kb < k_end) {  // wave-uniform
          if (kb + kBlockKeys - 1 > wave_first) block<true>(buf, sub, kb);
          else block<false>(buf, sub, kb);
        }
      }
      if (s + 1 < n_stages) {
        stage_arrived(key0 + KS, buf ^ 1);
        lds_barrier();
        if (s + 2 < n_stages) load_stage(page, key0 + 2 * KS, buf);
        page = page_of(key0 + 3 * KS);
      }
    }
  }

  // ---- few rows: every wavefront its own keys ---------------------------------------------------------------------------------
  // Bound by the stream of keys, so every wavefront takes blocks of its own (block i of the piece goes to wavefront i % 4) and
  // waits for nobody: K goes to registers in operand order (16 rows x 64 bytes a load), V through a strip of LDS of the
  // wavefront's own, both read once and therefore past the caches.
  static constexpr int kVBytes = kBlockKeys * kRow, kLoads = kVBytes / 1024;  // V of a block; loads of a lane for it, as many for K
  static constexpr int kStrips = kHalf ? 2 : 1;                               // of a wavefront
  __device__ __forceinline__ int strip_at(int buf) const { return (wave * kStrips + buf) * kVBytes; }
  __device__ __forceinline__ void fetch_own_v(int page, int kb, int buf) const {
    constexpr int kRowsALoad = 1024 / kRow;
    static_assert(!C::kOwnBlocks || kStrips * kWavesWg * kVBytes <= C::kStageBytes, "the strips fit the stages' LDS");
    const int64_t base = key_at(page, kb);
    int l = lane;
    asm volatile("" : "+v"(l));  // offsets are made here, not kept
    const unsigned v_row = static_cast<unsigned>(l) / UPR, v_off = v_row * kRow + ((l % UPR) ^ swz_v(v_row)) * 16;
#pragma unroll
    for (int p = 0; p < kLoads; ++p)
      load_lds16<T, 2>(vbase + base, (v_off ^ (swz_v(p * kRowsALoad) * 16)) + p * 1024, smem + strip_at(buf) + p * 1024);
  }
  __device__ __forceinline__ void fetch_own_k(int page, int kb, KFrag (&kf)[2][QF]) const {
    constexpr int E = C::E;
    const int64_t base = key_at(page, kb);
    int l = lane;
    asm volatile("" : "+v"(l));
    const T *rows = kbase + base + (l & 15) * D + (l >> 4) * E;
#pragma unroll
    for (int tk = 0; tk < 2; ++tk)
#pragma unroll
      for (int i = 0; i < kRow / 64; ++i) {
        const u32x4_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(rows + tk * 16 * D + i * 4 * E));
        if constexpr (kHalf) {
          kf[tk][i] = __builtin_bit_cast(half8_t, x);
        } else {
          const float4_t f = __builtin_bit_cast(float4_t, x);
#pragma unroll
          for (int e = 0; e < 4; ++e) kf[tk][4 * i + e] = f[e];
        }
      }
  }
  __device__ __forceinline__ void fetch_own(int page, int kb, int buf, KFrag (&kf)[2][QF]) const {
    fetch_own_v(page, kb, buf);
    fetch_own_k(page, kb, kf);
  }
  __device__ __forceinline__ void clean_own(int kb, int strip) const {
    if (kb + kBlockKeys > mixed_from) {
      bool bad = false;
#pragma unroll 1
      for (int p = 0; p < kLoads; ++p) bad |= clean(smem + strip + p * 1024 + lane * 16, kb + (p * 64 + lane) / UPR);
      if (bad) flags[0] = 1;
    }
  }
  __device__ __forceinline__ void use_own(int kb, int buf, const KFrag (&kf)[2][QF]) {
    float4_t sc[NT][2];
    Probs pf[NT];
    scores(kf, sc);
    __builtin_amdgcn_sched_barrier(0);
    clean_own(kb, strip_at(buf));
    softmax<true>(sc, kb, pf);
    __builtin_amdgcn_sched_barrier(0);
    VFrag vf[DT];
    read_v(strip_at(buf), vf);
    add_values(vf, pf);
  }
  __device__ __forceinline__ void own_blocks() {
    constexpr int kHop = kWavesWg * kBlockKeys;
    lds_barrier();  // the flags are cleared
    int kb = k0 + wave * kBlockKeys;
    if (kb >= k_end) return;
    const int page0 = page_of(kb);
    int page = page_of(kb + kHop);
    load_q();
    asm volatile("" ::: "memory");  // the queries' loads are issued before the keys'
    if constexpr (kHalf) own_two_ahead(kb, page0, page);
    else own_one(kb, page0, page);
  }
  // fp16: both a block ahead.
  __device__ __forceinline__ void own_two_ahead(int kb, int page0, int page) {
    constexpr int kHop = kWavesWg * kBlockKeys;
    KFrag now[2][QF], next[2][QF];
    fetch_own(page0, kb, 0, now);
#pragma unroll 1
    for (int buf = 0;; buf ^= 1) {
      // the block in use has arrived when no more than the next one's loads are under way (loads return in order)
      if (kb + kHop < k_end) {
        fetch_own(page, kb + kHop, buf ^ 1, next);
        page = page_of(kb + 2 * kHop);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kLoads) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      use_own(kb, buf, now);
      kb += kHop;
      if (kb >= k_end) break;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V of the block just used is in registers: its strip is free
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
#pragma unroll
        for (int kk = 0; kk < QF; ++kk) now[tk][kk] = next[tk][kk];
    }
  }
  // fp32: blocks are twice as large and products eight times as long.  The next keys are fetched into the registers of this block's as
  // soon as its scores are there, the next values into this block's strip as soon as they are in registers.
  __device__ __forceinline__ void own_one(int kb, int page0, int page) {
    constexpr int kHop = kWavesWg * kBlockKeys;
    KFrag kf[2][QF];
    fetch_own(page0, kb, 0, kf);
#pragma unroll 1
    for (bool more = true; more; kb += kHop) {
      more = kb + kHop < k_end;
      float4_t sc[NT][2];
      Probs pf[NT];
      VFrag vf[DT];
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      scores(kf, sc);
      __builtin_amdgcn_sched_barrier(0);
      if (more) fetch_own_k(page, kb + kHop, kf);
      clean_own(kb, strip_at(0));
      softmax<true>(sc, kb, pf);
      read_v(strip_at(0), vf);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) {
        fetch_own_v(page, kb + kHop, 0);
        page = page_of(kb + 2 * kHop);
      }
      __builtin_amdgcn_sched_barrier(0);
      add_values(vf, pf);
    }
  }

  // ---- the results ----------------------------------------------------------------------------------------------------------
  __device__ __forceinline__ void sum_lanes() {
    if constexpr (!kHalf) {
#pragma unroll
      for (int t = 0; t < NT; ++t) lsum[t][0] = sum_xor32(sum_xor16(lsum[t][0]));
    }
  }
  // no key seen: zeros; a NaN stays one
  static __device__ __forceinline__ float inverse(float l) { return l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l); }
  // rows of this wavefront, straight from its registers; `part` >= 0: to that row of the states instead
  __device__ __forceinline__ void store_rows(int64_t part) {
    sum_lanes();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = wrow + t * 16 + c;
      if (r >= n_rows) continue;
      const bool nan = lsum[t][0] != lsum[t][0];
      float all = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) all += (o[t][dt][0] + o[t][dt][1]) + (o[t][dt][2] + o[t][dt][3]);
      if (all != all && !nan) flags[1] = 1;  // (also infinities of both signs, which finish() leaves as they are)
      if (g == 0) row_nan[r] = nan;
      if (part >= 0) {
        float *po = a.part_o + (part + r) * D;
#pragma unroll
        for (int n = 0; n < DT; ++n) *reinterpret_cast<float4_t *>(po + four_at(n)) = four(t, n);
        if (g == 0) {
          a.part_ml[(part + r) * 2] = m[t];
          a.part_ml[(part + r) * 2 + 1] = lsum[t][0];
        }
      } else {
        const float inv = inverse(lsum[t][0]);
        S *orow = static_cast<S *>(a.out) + row_at(r);
#pragma unroll
        for (int n = 0; n < DT; ++n) {
          typedef S vec4 __attribute__((ext_vector_type(4)));
          const float4_t x = four(t, n);
          vec4 h;
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = static_cast<S>(x[e] * inv);
          *reinterpret_cast<vec4 *>(orow + four_at(n)) = h;
        }
      }
    }
  }
  // the wavefronts have the same rows: their states are added up through LDS (everybody has left it)
  __device__ __forceinline__ void store_sum(int64_t part) {
    sum_lanes();
    float *so = reinterpret_cast<float *>(chunk_smem);
    float *sml = so + C::kDealt * C::FEW * C::STATE;
    if (wave < C::kDealt) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int r = wave * C::FEW + t * 16 + c;
#pragma unroll
        for (int n = 0; n < DT; ++n) *reinterpret_cast<float4_t *>(so + r * C::STATE + four_at(n)) = four(t, n);
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
      if (acc != acc && l == l) flags[1] = 1;
      if (d == 0) row_nan[r] = l != l;
      if (part >= 0) {
        a.part_o[(part + r) * D + d] = acc;
        if (d == 0) {
          a.part_ml[(part + r) * 2] = mx;
          a.part_ml[(part + r) * 2 + 1] = l;
        }
      } else {
        stf(static_cast<T *>(a.out) + row_at(r) + d, acc * inverse(l));
      }
    }
  }
  // What the values that every row sees hold in element d: 1 infinities, 2 negative ones, 4 NaN.
  __device__ __forceinline__ void find_kinds(int *kinds) const {
    for (int d = tid; d < D; d += kThreads) kinds[d] = 0;
    __syncthreads();
    const int64_t n = static_cast<int64_t>(max(min(mixed_from, k_end) - k0, 0)) * UPR;
#pragma unroll 1
    for (int64_t x = tid; x < n; x += kThreads) {
      const int key = k0 + static_cast<int>(x / UPR), d = static_cast<int>(x % UPR) * C::E;
      const T *at = vbase + key_at(table[key >> kPageShift], key) + d;
      if (!unit_bad<T>(*reinterpret_cast<const u32x4_t *>(at))) continue;
#pragma unroll 1
      for (int e = 0; e < C::E; ++e) {
        const float v = ldf(at + e);
        if (!(fabsf(v) < __builtin_inff())) atomicOr(kinds + d + e, v != v ? 4 : (v > 0.f ? 1 : 2));
      }
    }
    __syncthreads();
  }
  // Infinities and NaN of V as every row that sees their key has them, whatever it weighs: those that were cleaned away are added, and
  // a NaN that comes from a weight that rounds to 0 becomes the infinity.  Rare, so through memory and without a thought for speed.
  // (Looking for such a NaN at the end of every piece: 16 x 4096 tokens, 16 / 8, 1142 -> 1150 us.)
  __device__ __forceinline__ void finish(int64_t part) {
    lds_barrier();
    const bool cleaned = flags[0] != 0, odd = flags[1] != 0;
    if (!cleaned && !odd) return;
    __threadfence_block();
    __syncthreads();
    int *kinds = reinterpret_cast<int *>(chunk_smem);
    if (odd) find_kinds(kinds);
    for (int x = tid; x < n_rows * D; x += kThreads) {
      const int r = x / D, d = x % D, last = position(r);
      float sum = 0.f;
      if (cleaned) {
        for (int key = max(k0, mixed_from); key < k_end && key <= last; ++key) {
          const float v = ldf(vbase + key_at(table[key >> kPageShift], key) + d);
          if (!(fabsf(v) < __builtin_inff())) sum += v;
        }
      }
      const int kind = odd && !row_nan[r] ? kinds[d] : 0;
      if (sum == 0.f && kind == 0) continue;
      T *out = static_cast<T *>(a.out) + row_at(r) + d;
      float v = part >= 0 ? a.part_o[(part + r) * D + d] : ldf(out);
      if (v != v && (kind == 1 || kind == 2)) v = kind == 1 ? __builtin_inff() : -__builtin_inff();
      if (part >= 0) a.part_o[(part + r) * D + d] = v + sum;
      else stf(out, v + sum);
    }
  }
};

template <typename T, int D>
__global__ __launch_bounds__(kThreads, (Cfg<T, D>::kLdsBytes <= 80 * 1024 ? 2 : 1)) void chunk_attn_kernel(ChunkArgs a) {
  using C = Cfg<T, D>;
  using W = Wave<T, D>;
  const int hk = blockIdx.x % a.Hkv;
  Piece pc;
  if (!find_piece<C, false>(a, blockIdx.x / a.Hkv, threadIdx.x & 63, pc)) return;
  const int n_rows = min(pc.rows - pc.tile * C::TR, C::TR);
  int64_t part = -1;
  if (pc.pieces > 1) {
    const int64_t slot = static_cast<int64_t>(pc.slot) * a.Hkv + hk;
    if (slot < 0 || slot >= a.slots || n_rows > a.slot_rows) return;  // (only where cu falls and rises: the cut is bounded by both)
    part = slot * a.slot_rows;
  }
  if (threadIdx.x < 2) reinterpret_cast<int *>(chunk_smem + C::kTail)[threadIdx.x] = 0;
  if (n_rows <= C::FEW) {
    W w(a, pc, hk, true);
    if constexpr (C::kOwnBlocks) w.own_blocks();
    else w.shared_stages(true);
    __syncthreads();
    w.store_sum(part);
    w.finish(part);
  } else {
    W w(a, pc, hk, false);
    w.shared_stages(false);
    __syncthreads();
    w.store_rows(part);
    w.finish(part);
  }
}

// Adds the pieces of a cut tile: out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M).  A workgroup takes up to 16 rows of the tile;
// where these are fewer, or the pieces many, several threads share an element and take every P-th piece each, and their sums
// are added up in a fixed tree through LDS (one token of 63 pieces, 16 / 8: 5.6 us, 8.4 us one after the other).  A thread has four pieces
// on their way at a time, and what bounds this kernel is the chain of such trips.
constexpr int kMergeRows = 16;
struct Sum {
  float m, l;
  float4_t o;
};
__device__ __forceinline__ void add_sum(Sum &a, const Sum &b) {
  const float top = fmaxf(a.m, b.m), fa = __builtin_amdgcn_exp2f(a.m - top), fb = __builtin_amdgcn_exp2f(b.m - top);
  a.m = top;
  a.l = a.l * fa + b.l * fb;
#pragma unroll
  for (int e = 0; e < 4; ++e) a.o[e] = add_weighted(add_weighted(0.f, fa, a.o[e]), fb, b.o[e]);
}
template <typename T, int D, int kMergeThreads>
__global__ __launch_bounds__(kMergeThreads) void chunk_merge_kernel(ChunkArgs a) {
  using C = Cfg<T, D>;
  const int hk = blockIdx.x % a.Hkv, tid = threadIdx.x;
  Piece pc;
  if (!find_piece<C, true>(a, blockIdx.x / a.Hkv, tid & 63, pc)) return;
  const int row0 = pc.tile * C::TR, n_rows = min(pc.rows - row0, C::TR);
  if (pc.slot < 0 || (static_cast<int64_t>(pc.slot) + pc.pieces - 1) * a.Hkv + hk >= a.slots || n_rows > a.slot_rows) return;
  constexpr int kAhead = 4;
  const int first = blockIdx.y * a.merge_rows, rows = min(a.merge_rows, n_rows - first);
  if (rows <= 0) return;
  const int64_t step = static_cast<int64_t>(a.Hkv) * a.slot_rows;  // between the pieces' states
  // threads of an element: a power of two, all of them with the same piece in neighbouring threads
  int log_rows = 0;
  while ((1 << log_rows) < rows) ++log_rows;
  const int items = (D / 4) << log_rows, parts = max(1, kMergeThreads / items);
  for (int at0 = 0; at0 < items; at0 += kMergeThreads) {  // (more than one pass only where parts is 1)
    const int item = (at0 + tid) % items, part = tid / items, r = first + item / (D / 4), d = item % (D / 4) * 4;
    const bool live = r < first + rows;
    Sum sum{kMasked, 0.f, float4_t{0.f, 0.f, 0.f, 0.f}};
    if (live) {
      const int64_t base = (static_cast<int64_t>(pc.slot) * a.Hkv + hk) * a.slot_rows + r;
      for (int s0 = part; s0 < pc.pieces; s0 += kAhead * parts) {
        Sum got[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int64_t at = base + min(s0 + i * parts, pc.pieces - 1) * step;
          got[i].m = a.part_ml[at * 2];
          got[i].l = a.part_ml[at * 2 + 1];
          got[i].o = *reinterpret_cast<const float4_t *>(a.part_o + at * D + d);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          if (s0 + i * parts < pc.pieces) add_sum(sum, got[i]);
      }
    }
    // (parts is a power of two, like all the sizes it is made from; one that had no piece adds nothing)
    __shared__ Sum sums[kMergeThreads];
    for (int half = parts / 2; half > 0; half /= 2) {
      if (part >= half && part < 2 * half) sums[tid] = sum;
      __syncthreads();
      if (part < half) add_sum(sum, sums[tid + half * items]);
    }
    if (part > 0 || !live) continue;
    const float inv = sum.l > 0.f ? 1.0f / sum.l : (sum.l == 0.f ? 0.f : sum.l);
    const int rr = row0 + r, i = rr / a.group;
    T *out = static_cast<T *>(a.out) + (static_cast<int64_t>(pc.c0 + i) * a.Hq + hk * a.group + (rr - i * a.group)) * D + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) stf(out + e, sum.o[e] * inv);
  }
}

struct Sizes {
  int64_t tiles;      // at most, per kv head
  int64_t grid;       // pieces at most, per kv head
  int64_t slots;      // pieces of cut tiles at most, over the kv heads
  int64_t cut_tiles;  // cut tiles at most, per kv head
  int slot_rows, target;
};
struct Tile {
  int rows, min_units, aim;
};
template <typename T>
Tile tile_for(int D) {
  if (D == 64) return {Cfg<T, 64>::TR, Cfg<T, 64>::MIN, Cfg<T, 64>::AIM};
  if (D == 128) return {Cfg<T, 128>::TR, Cfg<T, 128>::MIN, Cfg<T, 128>::AIM};
  return {Cfg<T, 256>::TR, Cfg<T, 256>::MIN, Cfg<T, 256>::AIM};
}
Tile tile_of(int dtype, int D) { return dtype == AXHIP_FLOAT32 ? tile_for<float>(D) : tile_for<__half>(D); }

// Bounds of the cut for any cu_tokens and start within tokens, B, max_q and max_len.  With q units per piece, q >= work / target
// and pieces = ceil(units / p) > 1 for a cut tile, p >= q / 2: its pieces are at most 2 units / p <= 4 units / q, all cut
// tiles' together at most 4 work / q <= 4 target.
Sizes sizes_for(Tile tile, int tokens, int B, int Hkv, int group, int max_q, int max_len) {
  Sizes z{};
  const int tile_rows = tile.rows;
  const int64_t rows = static_cast<int64_t>(tokens) * group;
  z.tiles = rows / tile_rows + B;
  const int64_t per_seq = (static_cast<int64_t>(max_q) * group + tile_rows - 1) / tile_rows;
  if (z.tiles > per_seq * B) z.tiles = per_seq * B;
  z.target = tile.aim * device_cu_count();
  const int64_t units = (static_cast<int64_t>(max_len) + 127) / 128;
  const int64_t most = (units + tile.min_units - 1) / tile.min_units;  // pieces of one tile
  const int64_t cut = 4 * static_cast<int64_t>(z.target) / Hkv + 1;    // pieces of cut tiles, per kv head
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
template <typename T, int D>
int launch(ChunkArgs a, const Sizes &z, hipStream_t st) {
  using C = Cfg<T, D>;
  static std::atomic<uint64_t> raised{0};
  const int rc = raise_dynamic_lds(reinterpret_cast<const void *>(&chunk_attn_kernel<T, D>), C::kLdsBytes, raised);
  if (rc != AXHIP_OK) return rc;
  hipLaunchKernelGGL((chunk_attn_kernel<T, D>), dim3(static_cast<unsigned>(z.grid * a.Hkv)), dim3(kThreads), C::kLdsBytes, st, a);
  if (z.cut_tiles > 0) {
    // 1024 threads where every tile has few rows or there are few tiles (1 token of 128000 keys, 16 / 1: 31 us, 41 us with 256), 256
    // where most workgroups find sixteen rows of few pieces or none (8 x 2000 tokens, 16 / 8: 195 us, 208 us with 1024).
    // Fewer rows a workgroup, and more threads an element, as long as that leaves a workgroup per CU (of 256 threads four): with 16
    // rows the 1 token of 128000 keys takes 123 us, 64 tokens at 16000 keys, 16 / 8, 38 us instead of 30, 512 tokens at
    // 8000 keys, 16 / 8, 55 instead of 54.
    const int cus = device_cu_count(), tiles = static_cast<int>(z.cut_tiles * a.Hkv);
    const auto groups = [&](int rows) { return (z.slot_rows + rows - 1) / rows; };
    const bool wide = groups(kMergeRows) == 1 || tiles * groups(kMergeRows) <= cus;
    const int most = wide ? cus : 4 * cus;
    a.merge_rows = kMergeRows;
    while (a.merge_rows > 1 && tiles * groups(a.merge_rows / 2) <= most) a.merge_rows /= 2;
    const dim3 grid(static_cast<unsigned>(tiles), groups(a.merge_rows));
    if (wide) hipLaunchKernelGGL((chunk_merge_kernel<T, D, 1024>), grid, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((chunk_merge_kernel<T, D, 256>), grid, dim3(256), 0, st, a);
  }
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
  const Sizes z = sizes_for(tile_of(dtype, D), tokens, B, Hkv, Hq / Hkv, max_q, max_len);
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
  const Sizes z = sizes_for(tile_of(dtype, D), tokens, B, Hkv, group, max_q, max_len);
  const size_t need = static_cast<size_t>(z.slots) * z.slot_rows * (D + 2) * sizeof(float);
  if (need && (!workspace || !aligned_to(workspace, 16))) return AXHIP_INVALID_PTR;
  if (workspace_bytes < need) return AXHIP_OUT_OF_MEMORY;
  if (z.grid * Hkv > kMostWorkgroups) return AXHIP_INVALID_ARGUMENT;
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
