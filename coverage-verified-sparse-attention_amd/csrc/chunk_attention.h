// Attention of a chunk of new tokens over the paged cache: kernel template.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),  s_ij = scale q_i . k_j
//
// over the keys j of the sequence that token i sees, in one pass over the
// keys with the running maximum m and sum l of each row.
//
// Rows.  The G query heads of a KV head share its keys, so a row is a (token,
// head of the group) pair and the rows of a sequence and KV head run over
// tokens, then heads: keys are read once for the whole group at any G, and a
// tile of rows spans few tokens, which wastes little of the causal mask's
// diagonal.  A workgroup takes RW * 32 rows; RW waves have 32 rows each.
//
// Products.  Both on 32x32x16 bf16 matrix instructions, transposed: S^T = K
// Q^T leaves lane l the scores of row l % 32 (16 of 32 keys, lane l ^ 32 the
// others), so the row's maximum and sum take one lane exchange, and its keys
// stand in the order in which O^T = V^T P^T takes them as the second operand:
// the weights go from one product to the next without leaving the lane.  V^T
// comes from the row-major tile through the transposing LDS read.  The weights
// are rounded to bf16 for the second product (as V is; at most half a step,
// 2^-8 of each weight); their sum l is taken in 32 bits before that.
//
// Keys.  Each step takes KW tiles of KT keys of K and V through LDS, loaded
// straight into it 16 bytes a lane; the vectors of row r are permuted by
// swizzle(r), so that both the row reads of K and the transposing reads of V
// spread over all banks.  Tile s + 1 is in flight while tile s is worked on.
// Block-table entries are read a step ahead of their use.  With eight row
// waves (many rows) half of the waves multiply while the other half makes
// weights: 8192 rows of 32 heads over 16384 keys, D = 128: 1357 us, 1225
// TFLOP/s, where all waves in step take 1760 (a large bf16 matrix product of
// the library: 1375 TFLOP/s).  With KW > 1 (few rows) each of KW groups of waves
// takes its own tile, and their states are joined at the end.  splits > 1
// spreads the keys over several workgroups, whose states a second kernel
// joins.
#pragma once
#include "cvsa_common.h"

#include <type_traits>
#include <utility>

namespace cvsa {

struct ChunkArgs {
  const uint16_t *q;
  int64_t q_st, q_sh;
  const uint16_t *k_cache, *v_cache;
  int num_blocks;
  const int32_t *block_tables;
  int64_t bt_sb;
  int W;
  const int32_t *context_lens, *cu;
  int B, H_q, H_kv, G, tokens;
  int bs_log2;
  float c;  // scale * log2(e)
  int causal;
  uint16_t *out;  // [tokens, H_q, D]
  float *lse;     // [tokens, H_q] or null
  int tiles;      // row tiles of all sequences
  int splits, split_len;
  float *part_o;   // [splits, tokens * H_q, D]: sum of weighted values
  float2 *part_ml; // [splits, tokens * H_q]: maximum (base 2), sum
};

// Keys of a wave's tile, and tiles of a workgroup (LDS: 2 stages of KW * KT
// rows of K and V).
template <int D>
constexpr int chunk_key_tiles(int RW) {
  return RW == 1 ? (D == 256 ? 2 : 4) : RW == 2 ? 2 : 1;
}
// Eight row waves: D = 64 and 128 only.
template <int D>
constexpr int chunk_keys(int RW) {
  return RW <= 2 || D == 256 ? 32 : 64;
}

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 chunk_bf16x8_t __attribute__((ext_vector_type(8)));
typedef short chunk_short4_t __attribute__((ext_vector_type(4)));

// Key and row ranges of a row tile.
struct ChunkTile {
  int seq, row0, rows;  // sequence, first row, rows of the sequence (and KV head)
  int first;            // the sequence's first token
  int pos0;             // position of that token
  int keys;             // keys that the tile's last row sees
};

__device__ __forceinline__ int chunk_tile_keys(const ChunkArgs &a, int pos0, int ctx, int rows,
                                               int row0, int tile_rows) {
  const int last = (min(row0 + tile_rows, rows) - 1) / a.G;
  const int seen = a.causal ? pos0 + last + 1 : ctx;
  return max(0, min(seen, a.W << a.bs_log2));
}

// The row tile `id` in the order of sequences.
__device__ __forceinline__ ChunkTile chunk_find_tile(const ChunkArgs &a, int id, int tile_rows) {
  const int lane = threadIdx.x & 63;
  ChunkTile t;
  int first = 0, len = 0, before = 0;
  t.seq = a.B - 1;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const int b = b0 + lane;
    const int lo = b < a.B ? a.cu[b] : 0;
    const int n = b < a.B ? a.cu[b + 1] - lo : 0;
    const int nt = (n * a.G + tile_rows - 1) / tile_rows;
    const int incl = (int)wave_incl_scan_u32((uint32_t)nt);
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (id < total) {
      const int l = __popcll(__ballot(incl <= id));
      t.seq = b0 + l;
      first = __builtin_amdgcn_readlane(lo, l);
      len = __builtin_amdgcn_readlane(n, l);
      before = __builtin_amdgcn_readlane(incl - nt, l);
      break;
    }
    id -= total;
  }
  const int ctx = a.context_lens[t.seq];
  t.first = first;
  t.rows = len * a.G;
  t.row0 = (id - before) * tile_rows;
  t.pos0 = ctx - len;
  t.keys = chunk_tile_keys(a, t.pos0, ctx, t.rows, t.row0, tile_rows);
  return t;
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

// First keys whose value in a column is +inf, -inf or NaN, of those taken out
// of V (none: INT_MAX): rows that see such a key get it back at the end.
constexpr int kNoKey = 0x7fffffff;

template <int N, class F, int... I>
__device__ __forceinline__ void unrolled(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void unrolled(F f) {
  unrolled<N>(f, std::make_integer_sequence<int, N>());
}

template <int D, int RW>
__global__ __launch_bounds__(RW *chunk_key_tiles<D>(RW) * 64, D == 256 ? 1 : 2) void
chunk_attention_kernel(const ChunkArgs a) {
  constexpr int KW = chunk_key_tiles<D>(RW), KT = chunk_keys<D>(RW);
  constexpr int NW = RW * KW, NT = NW * 64, TR = RW * 32;
  constexpr int CPR = D / 8, NR = KW * KT, NC = NR * CPR;
  constexpr int P = (NC + NT - 1) / NT;  // vectors of K and of V per thread and step
  constexpr int KB = KT / 32, KS = D / 16, DB = D / 32;
  static_assert(NC % NT == 0 || (P == 1 && NC % 64 == 0), "a step's vectors");
  static_assert((KW - 1) * RW <= 4 && (KW == 1 || NR * 2 >= 32 * 4), "room to join");
  constexpr int kStage = NR * D;  // elements of a step's K or V
  // Four arrays of their own: a load into one does not hold up reads of another.
  __shared__ __align__(16) uint16_t s_k0[kStage], s_k1[kStage], s_v0[kStage], s_v1[kStage];
  __shared__ float2 s_ml[KW > 1 ? (KW - 1) * RW * 32 : 1];
  __shared__ int s_first[3][D];  // keys of taken-out +inf, -inf, NaN
  __shared__ int s_taken;        // any

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave % RW, kw = wave / RW;
  const int l31 = lane & 31, half = lane >> 5;

  // KV heads vary fastest: workgroups go round the XCDs, so one XCD's cache
  // sees the keys of few heads.  Late row tiles, whose rows see most keys,
  // start first.
  int id = blockIdx.x;
  const int h = id % a.H_kv;
  id /= a.H_kv;
  const int split = id % a.splits;
  id = a.tiles - 1 - id / a.splits;
  const ChunkTile t = chunk_find_tile(a, id, TR);
  const int k0 = split * a.split_len;
  // The last split also takes keys past the plan's bound.
  const int k1 = split < a.splits - 1 ? min(t.keys, k0 + a.split_len) : t.keys;
  if (a.splits > 1 && k0 >= k1) return;
  const int steps = k1 > k0 ? (k1 - k0 + NR - 1) / NR : 0;

  const int row = t.row0 + wr * 32 + l31;
  const bool live = t.row0 + wr * 32 < t.rows;  // the wave has rows
  const bool row_ok = row < t.rows;
  const int tok = (row_ok ? row : t.row0) / a.G;
  const int head = h * a.G + (row_ok ? row : t.row0) - tok * a.G;
  // The last key that the row, and that the tile's first row, sees.
  const int last_key = a.causal ? min(t.pos0 + tok, k1 - 1) : k1 - 1;
  const int full_keys = a.causal ? min(t.pos0 + t.row0 / a.G + 1, k1) : k1;

  // Q^T as the second operand: row l % 32, 8 columns from 16 ks + 8 (l / 32).
  chunk_bf16x8_t q[KS];
  {
    const uint16_t *p = a.q + (int64_t)(t.first + tok) * a.q_st + head * a.q_sh + half * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      q[ks] = *reinterpret_cast<const chunk_bf16x8_t *>(p + ks * 16);
  }

  const int32_t *const bt = a.block_tables + t.seq * a.bt_sb;
  const int bs_mask = (1 << a.bs_log2) - 1;
  const int row_bytes = a.H_kv * D * 2;
  const uint32_t block_bytes = (uint32_t)row_bytes << a.bs_log2;

  for (int i = tid; i < 3 * D; i += NT) (&s_first[0][0])[i] = kNoKey;
  if (tid == 0) s_taken = 0;
  __syncthreads();

  // Block-table entries (-1: no key) of the thread's vectors in step s, and of
  // the keys of its wave's tile, a key per lane.
  auto entry = [&](int key) { return key < k1 ? bt[key >> a.bs_log2] : -1; };
  auto lookup = [&](int s, int (&blk)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) blk[p] = entry(k0 + s * NR + (tid + p * NT) / CPR);
  };
  auto lookup_tile = [&](int s) {
    return KT == 64 || lane < KT ? entry(k0 + s * NR + kw * KT + lane) : 0;
  };
  auto in_pool = [&](int blk) { return (uint32_t)blk < (uint32_t)a.num_blocks; };
  // Vectors of step s of K or V to LDS: vector c goes to place c, which holds
  // vector c % CPR (swizzled) of row c / CPR.  Where there is no block of the
  // pool, block 0 is read in its place.
  auto request = [&](const uint16_t *cache, int s, const int (&blk)[P], uint16_t *lds) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = tid + p * NT;
      if (NC % NT == 0 || p * NT + wave * 64 < NC) {
        const int r = c / CPR;
        const char *at = (const char *)cache + (h * D + chunk_swizzle<D>(r, c % CPR) * 8) * 2 +
                         (uint64_t)(uint32_t)(in_pool(blk[p]) ? blk[p] : 0) * block_bytes +
                         (uint32_t)(((k0 + s * NR + r) & bs_mask) * row_bytes);
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void *)at,
            (__attribute__((address_space(3))) void *)(lds + (p * NT + wave * 64) * 8), 16, 0, 0);
      }
    }
  };
  // V of a step that some row sees in part, or with keys that are none: zeros
  // where there is no key, and, as a weight of zero does not remove an infinite
  // or NaN value, such values are taken out and noted.  Each thread looks after
  // the vectors that it loaded.
  auto clean_v = [&](int s, const int (&blk)[P], uint16_t *lds) {
    bool none = false;
#pragma unroll
    for (int p = 0; p < P; ++p) none |= !in_pool(blk[p]);
    if (k0 + (s + 1) * NR <= full_keys && __ballot(none) == 0) return;
    unrolled<P>([&](auto pi) {
      constexpr int p = decltype(pi)::value;
      const int c = tid + p * NT;
      if (NC % NT == 0 || c < NC) {
        uint4 *const at = reinterpret_cast<uint4 *>(lds + c * 8);
        const uint4 w = *at;
        const uint4 bad = make_uint4(nonfinite_bf16x2(w.x), nonfinite_bf16x2(w.y),
                                     nonfinite_bf16x2(w.z), nonfinite_bf16x2(w.w));
        if (!in_pool(blk[p])) {
          *at = make_uint4(0, 0, 0, 0);
        } else if ((bad.x | bad.y | bad.z | bad.w) != 0) {
          *at = make_uint4(w.x & ~bad.x, w.y & ~bad.y, w.z & ~bad.z, w.w & ~bad.w);
          const int r = c / CPR, col = chunk_swizzle<D>(r, c % CPR) * 8;
          for (int i = 0; i < 8; ++i) {
            const uint32_t pair = i < 2 ? w.x : i < 4 ? w.y : i < 6 ? w.z : w.w;
            const uint32_t v = pair >> (16 * (i & 1)) & 0xffffu;
            if ((v & 0x7f80u) == 0x7f80u)
              atomicMin(&s_first[v == 0x7f80u ? 0 : v == 0xff80u ? 1 : 2][col + i],
                        k0 + s * NR + r);
          }
          s_taken = 1;
        }
      }
    });
  };

  f32x16_t o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = -INFINITY, neg_m = __builtin_nanf("");  // the rows' reference (base 2)
  float l = 0.f;                                    // the lane's part of their sum

  // S^T: registers e of block kb hold key 32 kb + 8 (e / 4) + 4 half + e % 4.
  auto scores = [&](const uint16_t *lds, f32x16_t (&st)[KB]) {
    const uint16_t *const kt = lds + kw * KT * D;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int r = kb * 32 + l31;
        const chunk_bf16x8_t k = *reinterpret_cast<const chunk_bf16x8_t *>(
            kt + r * D + chunk_swizzle<D>(r, 2 * ks + half) * 8);
        st[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[ks], ks ? st[kb] : f32x16_t{}, 0, 0,
                                                         0);
      }
  };
  // Keys that the row does not see leave step s's scores.
  auto mask = [&](int s, int blk, f32x16_t (&st)[KB]) {
    const int tile0 = k0 + s * NR + kw * KT;  // the wave's first key
    const uint64_t valid = __ballot(in_pool(blk));
    if (tile0 + KT > full_keys || ~valid != 0) {
      asm volatile("");  // a branch: not 64 selects in every step
      const uint64_t mine = valid >> (4 * half);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = kb * 32 + 8 * (e / 4) + e % 4;
          const bool see = ((mine >> key) & 1) && tile0 + key + 4 * half <= last_key;
          st[kb][e] = see ? st[kb][e] : -INFINITY;
        }
    }
  };
  // Weights of a step's scores.  The rows' reference is their maximum when it
  // was set; it moves only when the weights of a step outgrow it (their sum in
  // a lane passes 2^20, or there is no reference yet: NaN), so that steps need
  // no maximum.  Weights of up to 2^20 have the same relative precision.
  auto weigh = [&](const f32x16_t (&st)[KB], float neg_ref, uint4 (&pw)[2 * KB], auto before) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 2 * KB; ++j) {
      before(j);
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(st[j / 2][8 * (j % 2) + e], a.c, neg_ref));
        sum[e % 4] += p[e];
      }
      pw[j] = make_uint4(chunk_cvt_bf16x2(p[0], p[1]), chunk_cvt_bf16x2(p[2], p[3]),
                         chunk_cvt_bf16x2(p[4], p[5]), chunk_cvt_bf16x2(p[6], p[7]));
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
  };
  auto nothing = [](int) {};
  auto weights = [&](const f32x16_t (&st)[KB], uint4 (&pw)[2 * KB], auto before) {
    float sum = weigh(st, neg_m, pw, before);
    if (__ballot(!(sum < 1048576.f)) != 0) {
      float top[4] = {st[0][0], st[0][1], st[0][2], st[0][3]};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) top[e % 4] = fmaxf(top[e % 4], st[kb][e]);
      float x, y;
      xchg32(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), x, y);
      const float nm = fmaxf(m, fmaxf(x, y) * a.c);
      const float alpha = nm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - nm);
      m = nm;
      neg_m = nm == -INFINITY ? __builtin_nanf("") : -nm;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
      sum = weigh(st, nm == -INFINITY ? 0.f : -nm, pw, nothing);
    }
    l += sum;
  };
  // O^T += V^T P^T, 16 keys at a time: lane l has column 32 d + l % 32 of the
  // keys 4 half .. + 4 and 8 + 4 half .. + 4, a transposing read each.
  const int vrow = 4 * half + ((lane & 15) >> 2);
  const int vch = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  auto accumulate = [&](uint16_t *lds, const uint4 (&pw)[2 * KB]) {
    typedef __attribute__((address_space(3))) chunk_short4_t lds_short4;
    uint16_t *const vt = lds + kw * KT * D + (lane & 1) * 4;
#pragma unroll
    for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const int r0 = 16 * j + vrow, r1 = r0 + 8;
        const uint2 lo = __builtin_bit_cast(
            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (lds_short4 *)(vt + r0 * D + chunk_swizzle<D>(r0, d * 4 + vch) * 8)));
        const uint2 hi = __builtin_bit_cast(
            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (lds_short4 *)(vt + r1 * D + chunk_swizzle<D>(r1, d * 4 + vch) * 8)));
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(chunk_bf16x8_t, make_uint4(lo.x, lo.y, hi.x, hi.y)),
            __builtin_bit_cast(chunk_bf16x8_t, pw[j]), o[d], 0, 0, 0);
      }
  };
  if constexpr (RW < 8) {
    // Blocks of the thread's vectors of steps s and s + 1, and of the wave's
    // keys of step s.
    int b0[P], b1[P], tile_blk;
    // Step s, whose loads are under way into k_cur and v_cur: once they are
    // there, those of step s + 1 follow into k_next and v_next, whose readers
    // have passed the barrier.
    auto step = [&](int s, uint16_t *k_cur, uint16_t *v_cur,
                    uint16_t *k_next, uint16_t *v_next) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // every load of this wave has arrived
      clean_v(s, b0, v_cur);
      lds_barrier();
      if (s + 1 < steps) {
        request(a.k_cache, s + 1, b1, k_next);
        request(a.v_cache, s + 1, b1, v_next);
      }
      const int blk = tile_blk;
      tile_blk = lookup_tile(s + 1);
#pragma unroll
      for (int p = 0; p < P; ++p) b0[p] = b1[p];
      lookup(s + 2, b1);
      if (live) {
        f32x16_t st[KB];
        uint4 pw[2 * KB];
        scores(k_cur, st);
        mask(s, blk, st);
        weights(st, pw, nothing);
        accumulate(v_cur, pw);
      }
    };
    if (steps > 0) {
      lookup(0, b0);
      lookup(1, b1);
      tile_blk = lookup_tile(0);
      request(a.k_cache, 0, b0, s_k0);
      request(a.v_cache, 0, b0, s_v0);
      for (int s = 0; s < steps; s += 2) {
        step(s, s_k0, s_v0, s_k1, s_v1);
        if (s + 1 < steps) step(s + 1, s_k1, s_v1, s_k0, s_v0);
      }
    }
  } else {
    // Eight waves, two to a SIMD, the second four half a step behind: while
    // one multiplies (V of step s, K of step s + 1) the other makes weights,
    // with a barrier after each half.  In halves of the first four, step s
    // makes weights in half 2 s and multiplies in half 2 s + 1.  V of step s and K
    // of step s + 1 are free after half 2 s + 2, in half 2 s + 3 the loads that
    // take their place start, and they are waited for after half 2 s + 4.
    // Places in a buffer of the lane's vectors of K and V: a constant from one
    // block of keys, or 16 keys, to the next.
    typedef __attribute__((address_space(3))) chunk_short4_t lds_short4;
    uint32_t ka[KS], va[DB][2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      ka[ks] = (l31 * D + chunk_swizzle<D>(l31, 2 * ks + half) * 8) * 2;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = vrow + 8 * i;
        va[d][i] = (r * D + chunk_swizzle<D>(r, d * 4 + vch) * 8 + (lane & 1) * 4) * 2;
      }
    // V of one step, then K of the next.  The order is the source's: the LDS
    // reads run kAhead products ahead, and between(i) follows product i.
    auto multiply = [&](char *v, const char *k, const uint4 (&pw)[2 * KB], f32x16_t (&st)[KB],
                        auto between) {
      // The places as new values in each step: the buffer's address then goes
      // into the instruction, where it would take registers of its own.
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(ka[ks]));
#pragma unroll
      for (int d = 0; d < DB; ++d) asm volatile("" : "+v"(va[d][0]), "+v"(va[d][1]));
      constexpr int NV = 2 * KB * DB, N = NV + KB * KS, kAhead = 4;
      uint4 f[kAhead + 1];
      auto fetch = [&](auto at) {
        constexpr int i = decltype(at)::value;
        if constexpr (i < NV) {
          constexpr int j = i / DB, d = i % DB;
          const uint2 lo = __builtin_bit_cast(
              uint2,
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(v + va[d][0] + 32 * j * D)));
          const uint2 hi = __builtin_bit_cast(
              uint2,
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(v + va[d][1] + 32 * j * D)));
          f[i % (kAhead + 1)] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else if constexpr (i < N) {
          constexpr int ks = (i - NV) / KB, kb = (i - NV) % KB;
          f[i % (kAhead + 1)] = *reinterpret_cast<const uint4 *>(k + ka[ks] + 64 * kb * D);
        }
      };
      unrolled<kAhead>(fetch);
      __builtin_amdgcn_sched_barrier(0);
      unrolled<N>([&](auto at) {
        constexpr int i = decltype(at)::value;
        const chunk_bf16x8_t x = __builtin_bit_cast(chunk_bf16x8_t, f[i % (kAhead + 1)]);
        if constexpr (i < NV) {
          constexpr int j = i / DB, d = i % DB;
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              x, __builtin_bit_cast(chunk_bf16x8_t, pw[j]), o[d], 0, 0, 0);
        } else {
          constexpr int ks = (i - NV) / KB, kb = (i - NV) % KB;
          st[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, q[ks], ks ? st[kb] : f32x16_t{}, 0,
                                                           0, 0);
        }
        fetch(std::integral_constant<int, i + kAhead>());
        between(at);
        __builtin_amdgcn_sched_barrier(0);
      });
    };

    // Blocks.  Lane i looks up key i of a step for the whole wave, a step
    // ahead of the loads; where there is no key or no block of the pool, its
    // bit of the step's key mask is clear and block 0 is read in its place.
    // The rows of one load of the wave (4 at D = 128, 8 at D = 64) lie in one
    // block, the rows of a step at the same places of their blocks in every
    // step, or every other one (128-token pages: steps of 64 keys start at
    // multiples of 64).  So a load takes a block's address, the same in all
    // lanes, and a lane's constant offset.
    static_assert(NR == 64 && NC % NT == 0 && 64 / CPR <= 8, "a lane per key, a block per load");
    auto lookup_keys = [&](int s) { return bt[min(k0 + s * NR + lane, k1 - 1) >> a.bs_log2]; };
    uint32_t row_off[P];  // of the thread's vectors, in a block
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = tid + p * NT, r = c / CPR;
      row_off[p] = (r & bs_mask) * row_bytes + (h * D + chunk_swizzle<D>(r, c % CPR) * 8) * 2;
    }
    const uint32_t odd_off = a.bs_log2 == 7 ? 64 * row_bytes : 0;
    auto locate = [&](int s, int found, uint32_t (&blk)[P]) {
      const bool ok = k0 + s * NR + lane < k1 && in_pool(found);
      const int id = ok ? found : 0;
#pragma unroll
      for (int p = 0; p < P; ++p)
        blk[p] = __builtin_amdgcn_readlane(id, (p * NT + wave * 64) / CPR);
      return __ballot(ok);
    };
    auto load_one = [&](const uint16_t *cache, uint32_t blk, int odd, uint16_t *lds, int p) {
      const char *base = (const char *)cache + (uint64_t)blk * block_bytes;
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char *>(base), (short)0, (int)block_bytes, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void *)(lds + (p * NT + wave * 64) * 8), 16,
          (int)row_off[p], odd ? (int)odd_off : 0, 0, 0);
    };
    auto load = [&](const uint16_t *cache, const uint32_t (&blk)[P], int odd, uint16_t *lds) {
#pragma unroll
      for (int p = 0; p < P; ++p) load_one(cache, blk[p], odd, lds, p);
    };
    // clean_v and mask, for the steps that need them.
    auto clean = [&](int s, uint64_t keys, uint16_t *lds) {
      if (k0 + (s + 1) * NR <= full_keys && ~keys == 0) return;
      int none[P];
#pragma unroll
      for (int p = 0; p < P; ++p) none[p] = (int)(keys >> ((tid + p * NT) / CPR) & 1) - 1;
      clean_v(s, none, lds);
    };
    auto hide = [&](int s, uint64_t keys, f32x16_t (&st)[KB]) {
      if (k0 + (s + 1) * NR <= full_keys && ~keys == 0) return;
      mask(s, (int)(keys >> lane & 1) - 1, st);
    };
    // Barrier after the wave's LDS accesses, its loads left in flight.
    auto barrier = []() {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xc07f);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    // Every load of this wave has arrived.
    auto arrived = []() {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0f70);
      asm volatile("" ::: "memory");
    };

    // Eight waves, two to a SIMD, the second four half a step behind: while one
    // multiplies (V of step s, K of step s + 1) the other makes weights, with a
    // barrier after each half.  In halves of the first four, step s makes
    // weights in half 2 s and multiplies in half 2 s + 1.  Buffers of V of step
    // s - 1 and K of step s are free after half 2 s; in half 2 s + 1 both
    // groups start the loads of V of step s + 1 and K of step s + 2 into them,
    // each among what it computes then, and after half 2 s + 2 both have
    // waited for theirs.
    static_assert(P <= KB, "a load to 16 keys' weights");
    constexpr int kEvery = (2 * KB * DB + KB * KS) / (2 * P) < 5
                               ? (2 * KB * DB + KB * KS) / (2 * P) : 5;  // products to a load
    auto walk = [&](auto late_group) {
      constexpr bool LATE = decltype(late_group)::value;
      f32x16_t st[KB];
      uint32_t blk1[P], blk2[P];  // of steps s + 1 and s + 2
      uint64_t key0, key1, key2;  // keys of steps s to s + 2
      int found;                  // blocks of step s + 2
      auto step = [&](int s, auto parity, uint16_t *k_cur, uint16_t *k_next, uint16_t *v_cur,
                      uint16_t *v_next) {
        constexpr int A = decltype(parity)::value;
        // The i-th of the 2 P loads that step s starts.
        auto next_load = [&](int i) {
          if (i < P) load_one(a.v_cache, blk1[i], 1 - A, v_next, i);
          else if (i < 2 * P) load_one(a.k_cache, blk2[i - P], A, k_cur, i - P);
        };
        auto next_blocks = [&]() {
          key2 = locate(s + 2, found, blk2);
          found = lookup_keys(s + 3);
        };
        uint4 pw[2 * KB];
        if (LATE) next_blocks();
        if (live) {
          hide(s, key0, st);
          weights(st, pw, [&](int j) {
            if (LATE) {
              next_load(j);
              __builtin_amdgcn_sched_barrier(0);
            }
          });
        } else if (LATE) {
#pragma unroll
          for (int i = 0; i < 2 * P; ++i) next_load(i);
        }
        if (!LATE) {
          arrived();
          clean(s, key0, v_cur);
        }
        barrier();
        if (!LATE) next_blocks();
        if (live) {
          __builtin_amdgcn_s_setprio(1);
          multiply((char *)v_cur, (const char *)k_next, pw, st, [&](auto at) {
            constexpr int i = decltype(at)::value;
            if (!LATE && i % kEvery == kEvery / 2) next_load(i / kEvery);
          });
          __builtin_amdgcn_s_setprio(0);
        } else if (!LATE) {
#pragma unroll
          for (int i = 0; i < 2 * P; ++i) next_load(i);
        }
        if (LATE) {
          arrived();
          clean(s + 1, key1, v_next);
        }
        barrier();
#pragma unroll
        for (int p = 0; p < P; ++p) blk1[p] = blk2[p];
        key0 = key1;
        key1 = key2;
      };
      key0 = locate(0, lookup_keys(0), blk2);
      load(a.k_cache, blk2, 0, s_k0);
      load(a.v_cache, blk2, 0, s_v0);
      key1 = locate(1, lookup_keys(1), blk1);
      load(a.k_cache, blk1, 1, s_k1);
      found = lookup_keys(2);
      arrived();
      if (LATE) clean(0, key0, s_v0);
      barrier();
      if (live) scores(s_k0, st);
      if (LATE) barrier();
      for (int s = 0; s < steps; s += 2) {
        step(s, std::integral_constant<int, 0>(), s_k0, s_k1, s_v0, s_v1);
        if (s + 1 < steps)
          step(s + 1, std::integral_constant<int, 1>(), s_k1, s_k0, s_v1, s_v0);
      }
      if (!LATE) barrier();
      arrived();  // no load may outlive the workgroup's LDS
    };
    if (steps > 0) {
      if (wave >= 4) walk(std::true_type());
      else walk(std::false_type());
    }
  }

  float x, y;
  xchg32(l, x, y);
  l = x + y;

  if constexpr (KW > 1) {
    // The states of the groups of waves, joined in order by the first group:
    // an array of K or V for each wave, float4 i of row r at place i ^ (r % 8).
    auto room = [&](int w) {
      return reinterpret_cast<float4 *>(w == 0 ? s_k0 : w == 1 ? s_k1 : w == 2 ? s_v0 : s_v1);
    };
    auto at = [&](int d, int g) { return l31 * (D / 4) + ((8 * d + 2 * g + half) ^ (l31 & 7)); };
    __syncthreads();
    if (kw > 0) {
      const int w = (kw - 1) * RW + wr;
      float4 *const so = room(w);
      if (half == 0) s_ml[w * 32 + l31] = make_float2(m, l);
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          so[at(d, g)] =
              make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int i = 0; i < KW - 1; ++i) {
      const int w = i * RW + wr;
      const float4 *const so = room(w);
      const float2 ml = s_ml[w * 32 + l31];
      const float nm = fmaxf(m, ml.x);
      const float a0 = nm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - nm);
      const float a1 = nm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - nm);
      m = nm;
      l = l * a0 + ml.y * a1;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 v = so[at(d, g)];
          o[d][4 * g] = o[d][4 * g] * a0 + v.x * a1;
          o[d][4 * g + 1] = o[d][4 * g + 1] * a0 + v.y * a1;
          o[d][4 * g + 2] = o[d][4 * g + 2] * a0 + v.z * a1;
          o[d][4 * g + 3] = o[d][4 * g + 3] * a0 + v.w * a1;
        }
    }
  }

  if (s_taken) {
    // Infinite and NaN values back to the rows that see them.
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = d * 32 + 8 * (e / 4) + 4 * half + e % 4;
        if (s_first[0][col] <= last_key) o[d][e] += INFINITY;
        if (s_first[1][col] <= last_key) o[d][e] -= INFINITY;
        if (s_first[2][col] <= last_key) o[d][e] = __builtin_nanf("");
      }
  }

  if (!row_ok) return;
  const int64_t at = (int64_t)(t.first + tok) * a.H_q + head;
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.tokens * a.H_q;
    float *po = a.part_o + (split * rows + at) * D + 4 * half;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4 *>(po + d * 32 + 8 * g) =
            make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    if (half == 0) a.part_ml[split * rows + at] = make_float2(m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing is zero
  uint16_t *po = a.out + at * D + 4 * half;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2 *>(po + d * 32 + 8 * g) =
          make_uint2(chunk_cvt_bf16x2(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                     chunk_cvt_bf16x2(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
  if (a.lse && half == 0)
    a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace cvsa
