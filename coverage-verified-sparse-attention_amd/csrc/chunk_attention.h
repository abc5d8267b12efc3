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
// Keys.  The waves of the workgroup stage KW tiles of KT keys of K and V
// through LDS, 16 bytes at a time, the vectors of row r permuted by
// swizzle(r): both the row reads of K and the transposing reads of V then
// spread over all banks.  Tile t + 1 is in flight in registers while tile t
// is worked on.  Block-table entries are read one tile ahead of their use.
// With KW > 1 (few rows) each of KW groups of waves takes its own tile, and
// their states are joined at the end.  splits > 1 spreads the keys over
// several workgroups, whose states a second kernel joins.
#pragma once
#include "cvsa_common.h"

namespace cvsa {

struct ChunkArgs {
  const uint16_t *q;
  int64_t q_st, q_sh;
  const uint16_t *k_cache, *v_cache;
  int64_t num_blocks;
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

// A bf16 pair with infinities and NaN replaced by zero; `rest` the pair with
// all else replaced.
__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t w, uint32_t &rest) {
  const uint32_t lo = (w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u;
  const uint32_t hi = (w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
  rest = w & (lo | hi);
  return w & ~(lo | hi);
}

template <int D, int RW>
__global__ __launch_bounds__(RW *chunk_key_tiles<D>(RW) * 64, D == 256 ? 1 : 2) void
chunk_attention_kernel(const ChunkArgs a) {
  constexpr int KW = chunk_key_tiles<D>(RW), KT = chunk_keys<D>(RW);
  constexpr int NW = RW * KW, NT = NW * 64, TR = RW * 32;
  constexpr int CPR = D / 8, NR = KW * KT, NC = NR * CPR;
  constexpr int P = (NC + NT - 1) / NT;  // vectors of K and of V per thread and step
  constexpr int KB = KT / 32, KS = D / 16, DB = D / 32;
  constexpr int kMerge = KW > 1 ? (KW - 1) * RW * 32 * (D + 4) * 4 : 0;
  constexpr int kStage = NR * D;  // elements of a stage of K
  constexpr int kTiles = 2 * 2 * kStage * 2;
  __shared__ __align__(16) char s_mem[kTiles > kMerge ? kTiles : kMerge];
  __shared__ uint8_t s_valid[2][NR];
  __shared__ uint32_t s_nonfinite[2][NW];
  __shared__ float2 s_ml[KW > 1 ? (KW - 1) * RW * 32 : 1];
  uint16_t *const sk = reinterpret_cast<uint16_t *>(s_mem);
  uint16_t *const sv = sk + 2 * kStage;

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
  const int64_t row_elems = (int64_t)a.H_kv * D;

  // The physical row of the thread's p-th vector's key in step s, -1: no key.
  auto lookup = [&](int s, int (&blk)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int key = k0 + s * NR + (tid + p * NT) / CPR;
      blk[p] = -1;
      if (key < k1 && tid + p * NT < NC) blk[p] = bt[key >> a.bs_log2];
    }
  };
  uint4 kr[P], vr[P];
  bool ok[P];
  auto request = [&](int s, const int (&blk)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = tid + p * NT;
      const int key = k0 + s * NR + c / CPR;
      ok[p] = blk[p] >= 0 && blk[p] < a.num_blocks;
      kr[p] = vr[p] = make_uint4(0, 0, 0, 0);
      if (ok[p]) {
        const int64_t at = (((int64_t)blk[p] << a.bs_log2) + (key & bs_mask)) * row_elems +
                           h * D + (c % CPR) * 8;
        kr[p] = *reinterpret_cast<const uint4 *>(a.k_cache + at);
        vr[p] = *reinterpret_cast<const uint4 *>(a.v_cache + at);
      }
    }
  };
  // Vectors to LDS, zeros where there is no key; in steps that some row sees
  // in part, whether V holds an infinity or NaN.
  auto stage = [&](int s, int buf) {
    bool odd = false;
    const bool partial = k0 + (s + 1) * NR > full_keys;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = tid + p * NT;
      if (NC % NT == 0 || c < NC) {
        const int r = c / CPR, ch = c % CPR;
        const int at = buf * kStage + r * D + chunk_swizzle<D>(r, ch) * 8;
        *reinterpret_cast<uint4 *>(sk + at) = kr[p];
        *reinterpret_cast<uint4 *>(sv + at) = vr[p];
        if (ch == 0) s_valid[buf][r] = ok[p];
        if (partial) {
          uint32_t r0, r1, r2, r3;
          finite_bf16x2(vr[p].x, r0);
          finite_bf16x2(vr[p].y, r1);
          finite_bf16x2(vr[p].z, r2);
          finite_bf16x2(vr[p].w, r3);
          odd |= (r0 | r1 | r2 | r3) != 0;
        }
      }
    }
    const uint64_t any = __ballot(odd);
    if (lane == 0) s_nonfinite[buf][wave] = any != 0;
  };

  f32x16_t o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = -INFINITY, l = 0.f;  // running reference (base 2) and the lane's part of the sum

  int blk[P];
  lookup(0, blk);
  request(0, blk);
  lookup(1, blk);
  for (int s = 0; s < steps; ++s) {
    const int buf = s & 1;
    stage(s, buf);
    if (s + 1 < steps) {
      request(s + 1, blk);
      lookup(s + 2, blk);
    }
    lds_barrier();
    if (!live) continue;
    const uint16_t *const kt = sk + buf * kStage + kw * KT * D;
    const uint16_t *const vt = sv + buf * kStage + kw * KT * D;

    // S^T: registers e of block kb hold key 32 kb + 8 (e / 4) + 4 half + e % 4.
    f32x16_t st[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) st[kb][e] = 0.f;
      const int r = kb * 32 + l31;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const chunk_bf16x8_t k = *reinterpret_cast<const chunk_bf16x8_t *>(
            kt + r * D + chunk_swizzle<D>(r, 2 * ks + half) * 8);
        st[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[ks], st[kb], 0, 0, 0);
      }
    }

    const int tile0 = k0 + s * NR + kw * KT;  // the wave's first key
    const uint64_t valid = __ballot(lane < KT ? s_valid[buf][kw * KT + lane] != 0 : true);
    const bool partial = tile0 + KT > full_keys || ~valid != 0;
    if (partial) {
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

    // The reference moves only when a row's maximum passes it by 2^8: weights
    // stay below 2^8, at the same relative precision.
    float mx = st[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, st[kb][e]);
    float x, y;
    xchg32(mx, x, y);
    mx = fmaxf(x, y) * a.c;
    if (__ballot(mx > m + 8.f) != 0) {
      const float nm = fmaxf(m, mx);
      const float alpha = nm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - nm);
      m = nm;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    uint4 pw[2 * KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(fmaf(st[kb][8 * u + e], a.c, -ref));
          l += p[e];
        }
        pw[2 * kb + u] = make_uint4(chunk_cvt_bf16x2(p[0], p[1]), chunk_cvt_bf16x2(p[2], p[3]),
                                    chunk_cvt_bf16x2(p[4], p[5]), chunk_cvt_bf16x2(p[6], p[7]));
      }

    // O^T += V^T P^T, 16 keys at a time: lane l has column 32 d + l % 32 of the
    // keys 4 half .. + 4 and 8 + 4 half .. + 4, a transposing read each.
    typedef __attribute__((address_space(3))) chunk_short4_t lds_short4;
    const bool odd = partial && __ballot(lane < NW && s_nonfinite[buf][lane % NW] != 0) != 0;
    const int vrow = 4 * half + ((lane & 15) >> 2);
    const int vch = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    auto vread = [&](int j, int d) {
      const int r0 = 16 * j + vrow, r1 = r0 + 8;
      uint16_t *p0 = const_cast<uint16_t *>(vt) + r0 * D +
                     chunk_swizzle<D>(r0, d * 4 + vch) * 8 + (lane & 1) * 4;
      uint16_t *p1 = const_cast<uint16_t *>(vt) + r1 * D +
                     chunk_swizzle<D>(r1, d * 4 + vch) * 8 + (lane & 1) * 4;
      const uint2 lo = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)p0));
      const uint2 hi = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)p1));
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    };
    if (!odd) {
#pragma unroll
      for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
        for (int d = 0; d < DB; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(chunk_bf16x8_t, vread(j, d)),
              __builtin_bit_cast(chunk_bf16x8_t, pw[j]), o[d], 0, 0, 0);
    } else {
      // A value that some rows do not see is infinite or NaN, and a weight of
      // zero does not remove it: such values are left out of the product and
      // added key by key for the rows that see them.
#pragma unroll
      for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const uint4 v = vread(j, d);
          uint4 rest, fin;
          fin.x = finite_bf16x2(v.x, rest.x);
          fin.y = finite_bf16x2(v.y, rest.y);
          fin.z = finite_bf16x2(v.z, rest.z);
          fin.w = finite_bf16x2(v.w, rest.w);
          const chunk_bf16x8_t pj = __builtin_bit_cast(chunk_bf16x8_t, pw[j]);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(chunk_bf16x8_t, fin), pj, o[d], 0, 0, 0);
          if (__ballot((rest.x | rest.y | rest.z | rest.w) != 0) == 0) continue;
          for (int key = 0; key < 16; ++key) {
            // key 4 hk + i (+ 8) is element i (+ 4) of the lanes of half hk
            const int hk = (key >> 2) & 1, el = (key & 3) + 4 * (key >> 3);
            const uint32_t keep = el & 1 ? 0xffff0000u : 0xffffu;
            uint4 one;
            one.x = half == hk && (el >> 1) == 0 ? rest.x & keep : 0u;
            one.y = half == hk && (el >> 1) == 1 ? rest.y & keep : 0u;
            one.z = half == hk && (el >> 1) == 2 ? rest.z & keep : 0u;
            one.w = half == hk && (el >> 1) == 3 ? rest.w & keep : 0u;
            if (__ballot((one.x | one.y | one.z | one.w) != 0) == 0) continue;
            f32x16_t add;
#pragma unroll
            for (int e = 0; e < 16; ++e) add[e] = 0.f;
            add = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                __builtin_bit_cast(chunk_bf16x8_t, one), pj, add, 0, 0, 0);
            const bool see = tile0 + 16 * j + key <= last_key;
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] += see ? add[e] : 0.f;
          }
        }
    }
  }

  float x, y;
  xchg32(l, x, y);
  l = x + y;

  if constexpr (KW > 1) {
    // The states of the groups of waves, joined in order by the first group.
    constexpr int RS = D + 4;
    float *const so = reinterpret_cast<float *>(s_mem);
    __syncthreads();
    if (kw > 0) {
      const int base = ((kw - 1) * RW + wr) * 32 + l31;
      if (half == 0) s_ml[base] = make_float2(m, l);
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4 *>(so + base * RS + d * 32 + 8 * g + 4 * half) =
              make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int w = 0; w < KW - 1; ++w) {
      const int base = (w * RW + wr) * 32 + l31;
      const float2 ml = s_ml[base];
      const float nm = fmaxf(m, ml.x);
      const float a0 = nm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - nm);
      const float a1 = nm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - nm);
      m = nm;
      l = l * a0 + ml.y * a1;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 v =
              *reinterpret_cast<const float4 *>(so + base * RS + d * 32 + 8 * g + 4 * half);
          o[d][4 * g] = o[d][4 * g] * a0 + v.x * a1;
          o[d][4 * g + 1] = o[d][4 * g + 1] * a0 + v.y * a1;
          o[d][4 * g + 2] = o[d][4 * g + 2] * a0 + v.z * a1;
          o[d][4 * g + 3] = o[d][4 * g + 3] * a0 + v.w * a1;
        }
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
