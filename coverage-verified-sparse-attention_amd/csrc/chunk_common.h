// What the kernels of chunk attention share: the mathematics, the row tiles,
// the state of a wave's rows and its masks.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),  s_ij = scale q_i . k_j
//
// over the keys j of the sequence that token i sees, in one pass over the keys
// with a running reference m and sum l of each row.
//
// Rows.  The G query heads of a KV head share its keys, so a row is a (token,
// head of the group) pair and the rows of a sequence and KV head run over
// tokens, then heads: keys are read once for the whole group at any G, and a
// tile of rows spans few tokens, which wastes little of the causal mask's
// diagonal.  A wave has 32 rows (or 64).
//
// Products.  Both on 32x32x16 bf16 matrix instructions, transposed: S^T = K
// Q^T leaves lane l the scores of row l % 32 (16 of 32 keys, lane l ^ 32 the
// others), and its keys stand in the order in which O^T = V^T P^T takes them as
// the second operand: the weights go from one product to the next without
// leaving the lane.  V^T comes from the row-major tile through the transposing
// LDS read.  The weights are rounded to bf16 for the second product (as V is;
// at most half a step, 2^-8 of each weight); their sum l is taken in 32 bits
// before that.
//
// Keys go straight into LDS, 16 bytes a lane; the vectors of row r are permuted
// by swizzle(r), so that both the row reads of K and the transposing reads of V
// spread over all banks.
//
// Values that a row does not see.  A weight of zero does not remove an infinite
// or NaN value, so in tiles that some row sees in part such values are taken
// out of V; the first key of each kind is noted for each column, and rows that
// see that key get it back at the end.
#pragma once
#include "cvsa_common.h"

#include <type_traits>
#include <utility>

namespace cvsa {

// The sequences that bring min_rows to max_rows rows (tokens times G), their row
// tiles, and how their keys are spread over workgroups: many rows by splits of
// split_len keys, few rows by `splits` equal ranges of all their keys, sequence
// after sequence.  Parts of a row that several workgroups have are joined: of
// many rows part [split][token of the class * H_q + head], of few rows
// [2 * range + (the part starts its sequence)][KV head][row].
struct ChunkClass {
  int min_rows, max_rows;
  int tile_rows, tiles;
  int splits, split_len;
  int unit_log2;    // few rows: keys of a unit, 31: a unit has all of a sequence
  int tokens;       // of these sequences
  int only, only_first, only_len;  // many rows: the one such sequence, -1: several
  int same_len;     // what every sequence brings, 0: they differ
  float *part_o;    // [parts, D]: sums of weighted values
  float2 *part_ml;  // [parts]: reference (base 2), sum
};

struct ChunkArgs {
  const uint16_t *q;
  int64_t q_st, q_sh;
  const uint16_t *k_cache, *v_cache;
  int num_blocks;
  const int32_t *block_tables;
  int64_t bt_sb;
  int W;
  const int32_t *context_lens, *cu;
  int B, H_q, H_kv, G;
  int bs_log2;
  float c;  // scale * log2(e)
  int causal;
  uint16_t *out;  // [tokens, H_q, D]
  float *lse;     // [tokens, H_q] or null
};

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 chunk_bf16x8_t __attribute__((ext_vector_type(8)));
typedef short chunk_short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) chunk_short4_t chunk_lds_short4;

template <int N, class F, int... I>
__device__ __forceinline__ void unrolled(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void unrolled(F f) {
  unrolled<N>(f, std::make_integer_sequence<int, N>());
}

// Key and row ranges of a row tile.
struct ChunkTile {
  int seq, row0, rows;  // sequence, first row, rows of the sequence (and KV head)
  int first, part0;     // the sequence's first token, in all and in its class
  int pos0;             // position of that token
  int keys;             // keys that the tile's last row sees
};

__device__ __forceinline__ int chunk_tile_keys(const ChunkArgs &a, int pos0, int ctx, int rows,
                                               int row0, int tile_rows) {
  const int last = (min(row0 + tile_rows, rows) - 1) / a.G;
  const int seen = a.causal ? pos0 + last + 1 : ctx;
  return max(0, min(seen, a.W << a.bs_log2));
}

// Sequence b, without tokens if it is not of the class (or there is none); at
// least one unit if it has tokens.
struct ChunkSeq {
  int first, len, ctx, keys, units;
};
__device__ __forceinline__ ChunkSeq chunk_look(const ChunkArgs &a, const ChunkClass &c, int b) {
  ChunkSeq s = {0, 0, 0, 0, 0};
  if (b >= a.B) return s;
  s.first = c.same_len > 0 ? b * c.same_len : a.cu[b];
  s.len = c.same_len > 0 ? c.same_len : a.cu[b + 1] - s.first;
  s.ctx = a.context_lens[b];
  s.keys = max(0, min(s.ctx, a.W << a.bs_log2));
  if (s.len * a.G < c.min_rows || s.len * a.G > c.max_rows) s.len = 0;
  else s.units = (max(s.keys - 1, 0) >> c.unit_log2) + 1;
  return s;
}

// Tiles of a sequence (its units are nt) that see more than `keys` keys, keys >= 0.
template <int TR>
__device__ __forceinline__ int chunk_longer(const ChunkArgs &a, const ChunkSeq &s, int keys) {
  const int nt = (s.len * a.G + TR - 1) / TR;
  if (!a.causal) return s.keys > keys ? nt : 0;
  // Token x and later see more.
  const int x = keys - (max(s.ctx, 0) - s.len);
  if (x >= s.len || keys >= (a.W << a.bs_log2)) return 0;
  return x <= 0 ? nt : nt - x * a.G / TR;
}

// Row tile `id` of a class, of up to 64 sequences in the order of their keys (to
// 64), the longest first: tiles differ, by the causal mask and the contexts, and
// one that starts late should be short.  4 prompts of 1024 tokens, 32 heads on 8
// of 128: 51 us, in the order of the sequences 62.  Ragged prompts (64 to 163
// tokens after up to 2000): 64 of them in this order reach 714 TFLOP/s, 65 and 128
// in their own 679 and 700.
template <int TR>
__device__ __forceinline__ ChunkTile chunk_find_tile(const ChunkArgs &a, const ChunkClass &c,
                                                     int id) {
  const int lane = threadIdx.x & 63;
  ChunkTile t;
  int first, len, ctx, tile, part0 = 0;
  if (c.only >= 0) {
    t.seq = c.only;
    first = c.only_first;
    len = c.only_len;
    ctx = a.context_lens[t.seq];
    tile = c.tiles - 1 - id;
  } else {
    const ChunkSeq own = chunk_look(a, c, lane);
    auto look = [&](int b0) { return b0 == 0 ? own : chunk_look(a, c, b0 + lane); };
    // Tiles of more than 64 level + 63 keys; level -1: all.
    auto longer = [&](const ChunkSeq &s, int level) {
      return level < 0 ? (s.len * a.G + TR - 1) / TR : chunk_longer<TR>(a, s, 64 * level + 63);
    };
    // The lowest level that at most id tiles pass.  Past 64 sequences, where each
    // try would read all of them again, their own order does.
    const bool sorted = a.B <= kWave;
    int low = 0, high = 0, above = 0;  // tiles that pass level high
    if (sorted)
      high = __builtin_amdgcn_readfirstlane(wave_max_u32(own.len > 0 ? own.keys : 0)) >> 6;
    while (low < high) {
      const int mid = (low + high) >> 1;
      const int n = __builtin_amdgcn_readfirstlane(wave_sum_u32(longer(own, mid)));
      if (n <= id) {
        high = mid;
        above = n;
      } else {
        low = mid + 1;
      }
    }
    // Of the tiles between this level and the one below, by sequence.
    id -= above;
    t.seq = a.B - 1;
    first = len = ctx = tile = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWave) {
      const ChunkSeq s = look(b0);
      const int nt = longer(s, -1), over = sorted ? longer(s, low) : 0;
      const int n = (sorted ? longer(s, low - 1) : nt) - over;
      const int incl = (int)wave_incl_scan_u32((uint32_t)n);
      const int toks = (int)wave_incl_scan_u32((uint32_t)s.len);
      const int total = __builtin_amdgcn_readlane(incl, 63);
      if (id < total) {
        const int l = __popcll(__ballot(incl <= id));
        t.seq = b0 + l;
        first = __builtin_amdgcn_readlane(s.first, l);
        len = __builtin_amdgcn_readlane(s.len, l);
        ctx = __builtin_amdgcn_readlane(s.ctx, l);
        tile = __builtin_amdgcn_readlane(nt - over - 1 + incl - n, l) - id;
        part0 += __builtin_amdgcn_readlane(toks - s.len, l);
        break;
      }
      id -= total;
      part0 += __builtin_amdgcn_readlane(toks, 63);
    }
  }
  // Known to the compiler as the same in all lanes.
  t.seq = __builtin_amdgcn_readfirstlane(t.seq);
  len = __builtin_amdgcn_readfirstlane(len);
  ctx = __builtin_amdgcn_readfirstlane(ctx);
  tile = __builtin_amdgcn_readfirstlane(tile);
  t.first = __builtin_amdgcn_readfirstlane(first);
  t.part0 = __builtin_amdgcn_readfirstlane(part0);
  t.rows = len * a.G;
  t.row0 = tile * TR;
  t.pos0 = ctx - len;
  t.keys = chunk_tile_keys(a, t.pos0, ctx, t.rows, t.row0, TR);
  return t;
}

// The ranges of few rows' units (fewer than 2^31 in all): n, none of them empty,
// the first `more` one unit longer than the others.
struct ChunkRanges {
  uint32_t n, len, more;

  __device__ __forceinline__ ChunkRanges(const ChunkClass &c, uint32_t units) {
    n = min(units, (uint32_t)c.splits);
    len = units / max(n, 1u);
    more = units - len * n;
  }
  __device__ __forceinline__ uint32_t start(uint32_t r) const { return r * len + min(r, more); }
  __device__ __forceinline__ uint32_t of(uint32_t unit) const {
    const uint32_t longer = more * (len + 1);
    return unit < longer ? unit / (len + 1) : more + (unit - longer) / max(len, 1u);
  }
};

// A lane's row of a tile.
struct ChunkRow {
  bool ok;       // of the sequence
  int tok, head;
  int last_key;  // the last key that it sees, of those before k1
};

__device__ __forceinline__ ChunkRow chunk_row(const ChunkArgs &a, const ChunkTile &t, int h,
                                              int row, int k1) {
  ChunkRow r;
  r.ok = row < t.rows;
  const int at = r.ok ? row : t.row0;
  r.tok = at / a.G;
  r.head = h * a.G + at - r.tok * a.G;
  r.last_key = a.causal ? min(t.pos0 + r.tok, k1 - 1) : k1 - 1;
  return r;
}

// Q^T as the second operand: row l % 32, 8 columns from 16 ks + 8 (l / 32).
template <int D>
__device__ __forceinline__ void chunk_load_q(const ChunkArgs &a, const ChunkTile &t,
                                             const ChunkRow &r, chunk_bf16x8_t (&q)[D / 16]) {
  const uint16_t *p = a.q + (int64_t)(t.first + r.tok) * a.q_st + r.head * a.q_sh +
                      ((threadIdx.x >> 5) & 1) * 8;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
    q[ks] = *reinterpret_cast<const chunk_bf16x8_t *>(p + ks * 16);
}

// Place of 16-byte vector ch of row r of a tile: 16 rows (32 or 64 at D = 64
// and 32, whose rows share a sweep of the banks) read at one column, or 8 rows
// read at 4, fall on all banks evenly.
template <int D>
__device__ __forceinline__ int chunk_swizzle(int r, int ch) {
  constexpr int CPR = D / 8;
  if constexpr (CPR >= 16) return ch ^ (((r & 3) << 2) | ((r >> 2) & 3));
  else if constexpr (CPR == 8) return ch ^ (((r & 2) << 1) | ((r >> 2) & 3));
  else return ch ^ ((r >> 2) & 3);
}

// Bytes from a tile's start to what the lane reads of it: K of row l % 32 (and
// 32 rows on, 64 D bytes, the same), columns 16 ks + 8 (l / 32); and V of the
// transposing reads: lane l gets column 32 d + l % 32 of the keys 4 (l / 32) .. + 4
// (i = 0) or 8 on (i = 1), and 16 keys on, 32 D bytes, the same.
template <int D>
__device__ __forceinline__ uint32_t chunk_k_place(int ks) {
  const int l31 = threadIdx.x & 31, half = (threadIdx.x >> 5) & 1;
  return (l31 * D + chunk_swizzle<D>(l31, 2 * ks + half) * 8) * 2;
}
template <int D>
__device__ __forceinline__ uint32_t chunk_v_place(int d, int i) {
  const int lane = threadIdx.x & 63;
  const int r = 4 * (lane >> 5) + ((lane & 15) >> 2) + 8 * i;
  const int ch = d * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  return (r * D + chunk_swizzle<D>(r, ch) * 8 + (lane & 1) * 4) * 2;
}
__device__ __forceinline__ uint4 chunk_read_k(const char *at) {
  return *reinterpret_cast<const uint4 *>(at);
}
__device__ __forceinline__ uint4 chunk_read_v(char *lo, char *hi) {
  const uint2 x =
      __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((chunk_lds_short4 *)lo));
  const uint2 y =
      __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((chunk_lds_short4 *)hi));
  return make_uint4(x.x, x.y, y.x, y.y);
}

// The places of a lane's reads, from a tile's start.  At D = 256 the second half
// of the columns is 256 bytes on.
template <int D>
struct ChunkPlaces {
  static constexpr int KU = D == 256 ? 8 : D / 16, DU = D == 256 ? 4 : D / 32;
  uint32_t k[KU], v[DU][2];

  __device__ __forceinline__ void init(uint32_t tile) {
#pragma unroll
    for (int ks = 0; ks < KU; ++ks) k[ks] = tile + chunk_k_place<D>(ks);
#pragma unroll
    for (int d = 0; d < DU; ++d)
#pragma unroll
      for (int i = 0; i < 2; ++i) v[d][i] = tile + chunk_v_place<D>(d, i);
  }
  // As new values (in each step): the buffer's address then goes into the
  // instruction, where it would take registers of its own.
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int ks = 0; ks < KU; ++ks) asm volatile("" : "+v"(k[ks]));
#pragma unroll
    for (int d = 0; d < DU; ++d) asm volatile("" : "+v"(v[d][0]), "+v"(v[d][1]));
  }
  // Keys 32 kb .. + 32 of columns 16 ks .. + 16; columns 32 d .. + 32 of keys 16 j
  // .. + 16.
  __device__ __forceinline__ uint4 read_k(const char *tile, int kb, int ks) const {
    return chunk_read_k(tile + k[ks % KU] + (64 * kb * D + ks / KU * 256));
  }
  __device__ __forceinline__ uint4 read_v(char *tile, int j, int d) const {
    const int at = 32 * j * D + d / DU * 256;
    return chunk_read_v(tile + v[d % DU][0] + at, tile + v[d % DU][1] + at);
  }
};

__device__ __forceinline__ f32x16_t chunk_mfma(const uint4 &x, const uint4 &y, const f32x16_t &c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(chunk_bf16x8_t, x),
                                                 __builtin_bit_cast(chunk_bf16x8_t, y), c, 0, 0,
                                                 0);
}

__device__ __forceinline__ uint32_t chunk_cvt_bf16x2(float lo, float hi) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  f2 v;
  v.x = lo;
  v.y = hi;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// Infinite and NaN elements of a bf16 pair, as masks of their bits.
__device__ __forceinline__ uint32_t nonfinite_bf16x2(uint32_t w) {
  const uint32_t lo = (w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u;
  const uint32_t hi = (w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
  return lo | hi;
}

// Values taken out of V: the first key of +inf, -inf and NaN of each column
// (none: INT_MAX), and whether there is any.
template <int D>
struct ChunkTaken {
  int first[3][D];
  int any;

  __device__ __forceinline__ void clear(int threads) {
    for (int i = threadIdx.x; i < 3 * D; i += threads) (&first[0][0])[i] = 0x7fffffff;
    if (threadIdx.x == 0) any = 0;
  }
  // A vector of V in LDS, columns from col of key `key`: zeros where there is
  // no key, else its infinite and NaN values taken out.
  __device__ __forceinline__ void clean(uint4 *at, bool is_key, int key, int col) {
    const uint4 w = *at;
    const uint4 bad = make_uint4(nonfinite_bf16x2(w.x), nonfinite_bf16x2(w.y),
                                 nonfinite_bf16x2(w.z), nonfinite_bf16x2(w.w));
    if (!is_key) {
      *at = make_uint4(0, 0, 0, 0);
    } else if ((bad.x | bad.y | bad.z | bad.w) != 0) {
      *at = make_uint4(w.x & ~bad.x, w.y & ~bad.y, w.z & ~bad.z, w.w & ~bad.w);
      for (int i = 0; i < 8; ++i) {
        const uint32_t pair = i < 2 ? w.x : i < 4 ? w.y : i < 6 ? w.z : w.w;
        const uint32_t v = pair >> (16 * (i & 1)) & 0xffffu;
        if ((v & 0x7f80u) == 0x7f80u)
          atomicMin(&first[v == 0x7f80u ? 0 : v == 0xff80u ? 1 : 2][col + i], key);
      }
      any = 1;
    }
  }
  // Back to the rows that see them.
  __device__ __forceinline__ void restore(int last_key, f32x16_t (&o)[D / 32]) const {
    if (!any) return;
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      __builtin_amdgcn_sched_barrier(0);  // few reads at once: registers
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = d * 32 + 8 * (e / 4) + 4 * half + e % 4;
        if (first[0][col] <= last_key) o[d][e] += INFINITY;
        if (first[1][col] <= last_key) o[d][e] -= INFINITY;
        if (first[2][col] <= last_key) o[d][e] = __builtin_nanf("");
      }
    }
  }
};

// Scores S^T of KB * 32 keys from tile0 on (registers e of block kb hold key
// 32 kb + 8 (e / 4) + 4 (l / 32) + e % 4): -inf for keys whose bit is clear and
// those past the row's last.
template <int KB>
__device__ __forceinline__ void chunk_mask(f32x16_t (&st)[KB], uint64_t keys, int tile0,
                                           int last_key) {
  const int half = (threadIdx.x >> 5) & 1;
  const uint64_t mine = keys >> (4 * half);
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int key = kb * 32 + 8 * (e / 4) + e % 4;
      const bool see = ((mine >> key) & 1) && tile0 + key + 4 * half <= last_key;
      st[kb][e] = see ? st[kb][e] : -INFINITY;
    }
}

// State of a lane's row (its half of the columns and keys).
template <int D>
struct ChunkState {
  f32x16_t o[D / 32];  // O^T: registers e of block d, column 32 d + 8 (e / 4) + 4 (l / 32) + e % 4
  float m, neg_m;      // reference (base 2) and its negative, NaN while there is none
  float l;             // the lane's part of the sum

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    m = -INFINITY;
    neg_m = __builtin_nanf("");
    l = 0.f;
  }

  // exp2(c s - reference) of a step's scores as bf16 pairs; their sum.
  // before(j) precedes 16 keys' part.
  template <int KB, class F>
  static __device__ __forceinline__ float weigh(const f32x16_t (&st)[KB], float c, float neg_ref,
                                                uint4 (&pw)[2 * KB], F before) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 2 * KB; ++j) {
      before(j);
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(st[j / 2][8 * (j % 2) + e], c, neg_ref));
        sum[e % 4] += p[e];
      }
      pw[j] = make_uint4(chunk_cvt_bf16x2(p[0], p[1]), chunk_cvt_bf16x2(p[2], p[3]),
                         chunk_cvt_bf16x2(p[4], p[5]), chunk_cvt_bf16x2(p[6], p[7]));
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }

  // Weights of a step's scores.  The reference is the row's maximum when it was
  // set; it moves only when the weights of a step outgrow it (their sum in a
  // lane passes 2^20, or there is no reference yet: NaN), so that steps need no
  // maximum.  Weights of up to 2^20 have the same relative precision.
  template <int KB, class F>
  __device__ __forceinline__ void weights(const f32x16_t (&st)[KB], float c, uint4 (&pw)[2 * KB],
                                          F before) {
    settle(st, c, pw, weigh(st, c, neg_m, pw, before));
  }
  // The rest of weights(), given their sum for the present reference.
  template <int KB>
  __device__ __forceinline__ void settle(const f32x16_t (&st)[KB], float c, uint4 (&pw)[2 * KB],
                                         float sum) {
    if (__ballot(!(sum < 1048576.f)) != 0) {
      float top[4] = {st[0][0], st[0][1], st[0][2], st[0][3]};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) top[e % 4] = fmaxf(top[e % 4], st[kb][e]);
      float x, y;
      xchg32(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), x, y);
      const float nm = fmaxf(m, fmaxf(x, y) * c);
      const float alpha = nm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - nm);
      m = nm;
      neg_m = nm == -INFINITY ? __builtin_nanf("") : -nm;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
      sum = weigh(st, c, nm == -INFINITY ? 0.f : -nm, pw, [](int) {});
    }
    l += sum;
  }

  // The sum over both halves of the keys.
  __device__ __forceinline__ void finish() {
    float x, y;
    xchg32(l, x, y);
    l = x + y;
  }

  // The row's output.
  __device__ __forceinline__ void store(const ChunkArgs &a, const ChunkTile &t,
                                        const ChunkRow &r) const {
    const int half = (threadIdx.x >> 5) & 1;
    const int64_t at = (int64_t)(t.first + r.tok) * a.H_q + r.head;
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing is zero
    // The halves exchange columns, so that each has 8 in a row.
    uint16_t *po = a.out + at * D + 8 * half;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = chunk_cvt_bf16x2(o[d][4 * g + 2 * i] * inv, o[d][4 * g + 2 * i + 1] * inv);
        const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        if (r.ok)
          *reinterpret_cast<uint4 *>(po + d * 32 + 8 * g) = make_uint4(x[0], y[0], x[1], y[1]);
      }
    if (a.lse && r.ok && half == 0)
      a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
  // The row's state as part `at`, for a join.
  __device__ __forceinline__ void store_part(const ChunkClass &c, const ChunkRow &r,
                                             int64_t at) const {
    if (!r.ok) return;
    const int half = (threadIdx.x >> 5) & 1;
    float *po = c.part_o + at * D + 4 * half;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4 *>(po + d * 32 + 8 * g) =
            make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    if (half == 0) c.part_ml[at] = make_float2(m, l);
  }
};

// A load of 64 vectors of 16 bytes straight into LDS: from byte off (of each
// lane) + soff of block blk, to 1 KiB at lds.  readable: bytes of the block that
// may be read (0: none, nothing is fetched).
__device__ __forceinline__ void chunk_load_lds(const uint16_t *cache, uint32_t blk,
                                               uint32_t block_bytes, uint32_t readable,
                                               uint32_t off, uint32_t soff, uint16_t *lds) {
  const char *base = (const char *)cache + (uint64_t)blk * block_bytes;
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char *>(base), (short)0, (int)readable, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      rsrc, (__attribute__((address_space(3))) void *)lds, 16, (int)off, (int)soff, 0, 0);
}

}  // namespace cvsa
