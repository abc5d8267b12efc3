// The attention weight that a chunk's queries give to each key of the paged cache
// (cvsa_add_key_weights), by which a cache is cut:
//
//   w_j  <-  (j is new ? 0 : w_j) + sum over rows i that see j of exp(scale q_i . k_j - lse_i)
//
// for each sequence and KV head, a row being a (token, query head of the group) pair
// and lse_i its log-sum-exp, which the attention returns.  One product, on 32x32x16
// matrix instructions with the queries as first operand: a lane has 16 rows'
// scores of one key, adds their exponentials in registers, and the key's sum is
// complete after one exchange with the lane of the other 16 rows.  Nothing is
// added in an order that varies: no atomics.
//
// With c = scale log2(e) and lse2 = lse c / scale the exponent is one fma, c s -
// lse2, and the error of c (2^-24) scales with the exponent, not with lse: the keys
// that matter have small ones.
//
// Few rows (up to 32 of a sequence and KV head: single tokens, drafts): reading the
// keys bounds it.  A wave keeps all rows in registers and streams keys, 32 at a
// time, from memory straight into the operand's registers, the next 32 under way;
// no LDS, no barrier.  The keys of all sequences, end to end, are cut into equal
// ranges, one for each wave that fits the GPU.
//
// Many rows: the vector and matrix pipes bound it (32 exponentials of a wave, with a
// fused multiply and an addition each, to 16 products at D = 128), so the products
// of the next 32 rows stand between the exponentials of these.  A workgroup keeps a
// tile of 256 keys in registers, 64 a wave, and the rows that see any of them pass by
// through LDS, 128 at a time: a row is read once for 256 keys and an LDS read feeds
// two products.  The passes of all tiles, end to end, are cut into equal ranges, one
// for each workgroup, which so loads one or two tiles of keys; a tile that several
// ranges share is joined in order by a second kernel.
//
// Measured, heads of 128.  Few rows: a token of each of 32 sequences of 8 K keys at
// most, 32 heads on 8, 8 bits: 33 us for 147 MB, 4.4 TB/s (a copy reaches 5.1).  Many
// rows: 4096 tokens over themselves, 32 heads on 8, 8 bits: 82 us with 4 to join, 850
// TFLOP/s of the product (a large one of the library 1318); the vector pipe's 52
// instructions to 8 products, 16 of them exponentials, take 400 cycles of a SIMD where
// the products take 256, so 47 us at 2.2 GHz.  The last 64 of 2048 tokens over 32768
// keys of bf16: 31 and 5, where half of the time a workgroup waits for its two tiles of
// keys (a word of each line of the second one read ahead of time into the XCD's cache,
// whose 4 MB the first ones fill: 37 for 35).
#include "chunk_common.h"

#include <algorithm>
#include <cmath>

namespace cvsa {

struct WeighArgs {
  const uint16_t *q;
  int64_t q_st, q_sh;
  const float *lse;       // [tokens, H_q]
  const char *k_cache;
  const uint8_t *k_scales;
  int num_blocks;
  const int32_t *block_tables;
  int64_t bt_sb;
  int W;
  const int32_t *context_lens, *cu;
  int B, H_q, H_kv, G;
  int bs_log2;
  float c, lse_factor;    // scale * log2(e), c / scale
  int causal, window;     // window: tokens of a sequence that count, 0: all
  float *weights;         // [B, H_kv, S]
  int64_t S;
  float *parts;           // many rows: [range][H_kv][2][kWeighKeys] sums of shared tiles
};

constexpr int kWeighFewRows = 32;
constexpr int kWeighKeys = 256;  // of a tile of many rows

// A sequence's rows that count, 0 .. rows, from its token `skip` on.
struct WeighSeq {
  int first, pos0, keys, rows;  // first counting token of the batch, its position
  int before;                   // keys that the chunk did not bring
};

__device__ __forceinline__ WeighSeq weigh_look(const WeighArgs &a, int b, bool few) {
  WeighSeq s = {0, 0, 0, 0, 0};
  if (b >= a.B) return s;
  const int first = a.cu[b], len = a.cu[b + 1] - first, ctx = a.context_lens[b];
  const int count = a.window > 0 ? min(len, a.window) : len;
  s.first = first + len - count;
  s.pos0 = ctx - count;
  s.before = ctx - len;
  s.rows = count * a.G;
  if (len > 0 && (s.rows <= kWeighFewRows) == few)
    s.keys = max(0, min(ctx, a.W << a.bs_log2));
  else
    s.rows = 0;
  return s;
}

// Keys, 16 bytes at a time as they lie: of bf16 columns 16 ks + 8 (l / 32), of 8
// bits (WIDE, see chunk_load_q) 32 j + 16 (l / 32), which make two steps.
template <int D, bool F8>
struct WeighKeys {
  static constexpr int N = F8 ? D / 32 : D / 16;
  uint4 w[N];

  __device__ __forceinline__ void load(const char *row, int half) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      w[i] = *reinterpret_cast<const uint4 *>(row + 32 * i + 16 * half);
  }
  // The operand of step ks; 8 bits: times the scale, exactly, as the attention has them.
  __device__ __forceinline__ uint4 get(int ks, float scale) const {
    if constexpr (F8) {
      const uint4 &v = w[ks / 2];
      return chunk_from_8(ks % 2 ? make_uint2(v.z, v.w) : make_uint2(v.x, v.y), scale, scale);
    } else {
      return w[ks];
    }
  }
};

// The queries' operand of step ks, in the columns that the keys have: bytes from a
// tile's start to row l % 32.  At D = 256 the second half of the columns is 256
// bytes on.
template <int D, bool F8>
struct WeighPlaces {
  static constexpr int N = D == 256 ? 8 : D / 16;
  uint32_t at[N];

  __device__ __forceinline__ void init() {
    const int l31 = threadIdx.x & 31, half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int ks = 0; ks < N; ++ks) {
      const int ch = F8 ? ks / 2 * 4 + half * 2 + ks % 2 : 2 * ks + half;
      at[ks] = (l31 * D + chunk_swizzle<D>(l31, ch) * 8) * 2;
    }
  }
  __device__ __forceinline__ void renew() {  // see ChunkPlaces
#pragma unroll
    for (int ks = 0; ks < N; ++ks) asm volatile("" : "+v"(at[ks]));
  }
  __device__ __forceinline__ uint4 read(const char *tile, int ks) const {
    return chunk_read_k(tile + at[ks % N] + ks / N * 256);
  }
};

// Where key `key` of a sequence lies; block 0 if it is none (ok false).
struct WeighKeyAt {
  bool ok;
  int blk;
};
__device__ __forceinline__ WeighKeyAt weigh_key_at(const WeighArgs &a, int key, int keys,
                                                   int found) {
  const bool ok = key < keys && (uint32_t)found < (uint32_t)a.num_blocks;
  return {ok, ok ? found : 0};
}

template <int D, bool F8>
__device__ __forceinline__ const char *weigh_row(const WeighArgs &a, int blk, int key, int h) {
  const int64_t token = ((int64_t)blk << a.bs_log2) + (key & ((1 << a.bs_log2) - 1));
  return a.k_cache + (token * a.H_kv + h) * (D * (F8 ? 1 : 2));
}

// Sum of 16 values as a tree.
__device__ __forceinline__ float sum16(const float (&p)[16]) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = p[i] + p[i + 8];
  return ((s[0] + s[4]) + (s[1] + s[5])) + ((s[2] + s[6]) + (s[3] + s[7]));
}

// Workgroups of a CU, by registers.
template <int D, bool F8>
constexpr int weigh_few_fit() {
  return D == 256 ? (F8 ? 2 : 1) : D == 128 && !F8 ? 2 : 3;
}

template <int D, bool F8>
__global__ __launch_bounds__(256, (weigh_few_fit<D, F8>())) void weigh_few_kernel(
    const WeighArgs a) {
  constexpr int KS = D / 16;
  const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The heads of a range go to one XCD, where the workgroups of a head are a multiple of
  // 8 (powers of two of KV heads): see the chunk attention of few rows.
  const uint32_t n_wgs = gridDim.x / a.H_kv;
  const int h = blockIdx.x / n_wgs;
  const uint32_t range = blockIdx.x % n_wgs * 4 + wave, ranges = n_wgs * 4;

  // The wave's units of 32 keys.
  const WeighSeq own = weigh_look(a, lane, true);
  uint32_t total = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const WeighSeq s = b0 == 0 ? own : weigh_look(a, b0 + lane, true);
    total += __builtin_amdgcn_readfirstlane(wave_sum_u32((uint32_t)(s.keys + 31) / 32));
  }
  const uint32_t each = total / ranges, more = total - each * ranges;
  const uint32_t begin = range * each + min(range, more);
  const uint32_t end = begin + each + (range < more ? 1 : 0);

  uint32_t before = 0;
  for (int b0 = 0; b0 < a.B && before < end; b0 += kWave) {
    const WeighSeq mine = b0 == 0 ? own : weigh_look(a, b0 + lane, true);
    const uint32_t units = (uint32_t)(mine.keys + 31) / 32;
    const uint32_t incl = wave_incl_scan_u32(units), last = before + incl, start = last - units;
    uint64_t todo = __ballot(units > 0 && start < end && last > begin);
    while (todo != 0) {
      const int l = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int seq = b0 + l;
      const int first = __builtin_amdgcn_readlane(mine.first, l);
      const int pos0 = __builtin_amdgcn_readlane(mine.pos0, l);
      const int keys = __builtin_amdgcn_readlane(mine.keys, l);
      const int rows = __builtin_amdgcn_readlane(mine.rows, l);
      // Those of the table: the context may be longer.
      const int old = min(__builtin_amdgcn_readlane(mine.before, l), keys);
      const uint32_t from = __builtin_amdgcn_readlane(start, l);
      const int t0 = (int)(begin > from ? begin - from : 0);
      const int t1 = (int)min(end - from, (uint32_t)__builtin_amdgcn_readlane(units, l));
      const int32_t *const bt = a.block_tables + seq * a.bt_sb;
      float *const w = a.weights + ((int64_t)seq * a.H_kv + h) * a.S;

      // Queries: rows past the last are zeros and do not count.
      chunk_bf16x8_t q[KS];
      const int row = min(l31, rows - 1), tok = row / a.G;
      {
        const uint16_t *p = a.q + (int64_t)(first + tok) * a.q_st +
                            (int64_t)(h * a.G + row - tok * a.G) * a.q_sh + half * (F8 ? 16 : 8);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          q[ks] = *reinterpret_cast<const chunk_bf16x8_t *>(
              p + (F8 ? ks / 2 * 32 + ks % 2 * 8 : ks * 16));
      }
      const float my_lse = a.lse[(int64_t)(first + tok) * a.H_q + h * a.G + row - tok * a.G];
      float neg[16];  // of the lane's rows 8 (e / 4) + 4 (l / 32) + e % 4
      uint32_t live = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int r = 8 * (e / 4) + e % 4;
        const float x = __shfl(my_lse, r + 4 * half, 64);
        neg[e] = -x * a.lse_factor;
        if (r + 4 * half < rows && x != -INFINITY) live |= 1u << e;
      }

      auto lookup = [&](int t) { return bt[min((t * 32 + l31) >> a.bs_log2, a.W - 1)]; };
      struct Tile {
        WeighKeys<D, F8> k;
        bool ok;
        uint32_t scale;
        float w;
      };
      auto request = [&](int t, int found, Tile &x) {
        const int key = t * 32 + l31;
        const WeighKeyAt at = weigh_key_at(a, key, keys, found);
        x.ok = at.ok;
        x.k.load(weigh_row<D, F8>(a, at.blk, at.ok ? key : 0, h), half);
        x.scale = F8 ? a.k_scales[(int64_t)at.blk * a.H_kv + h] : 127u;
        x.w = key < old ? w[key] : 0.f;
      };
      auto add = [&](int t, const Tile &x) {
        f32x16_t s;
        const float scale = chunk_scale(x.scale);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          s = chunk_mfma(__builtin_bit_cast(uint4, q[ks]), x.k.get(ks, scale),
                         ks ? s : f32x16_t{});
        const int key = t * 32 + l31;
        // The first row that sees the key, and the lane's rows from there on.
        const int min_row = a.causal && key > pos0 ? min(key - pos0, 1 << 20) * a.G : 0;
        float p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = 8 * (e / 4) + e % 4;
          const bool see = (live >> e & 1) && r + 4 * half >= min_row;
          const float v = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, neg[e]));
          p[e] = see ? v : 0.f;
        }
        float u, v;
        xchg32(sum16(p), u, v);
        const float sum = x.ok ? u + v : 0.f;
        if (half == 0 && key < keys) w[key] = x.w + sum;
      };
      Tile even, odd;
      int found = lookup(t0 + 1);
      request(t0, lookup(t0), even);
      for (int t = t0; t < t1; t += 2) {
        request(t + 1, found, odd);
        found = lookup(t + 2);
        add(t, even);
        if (t + 1 >= t1) break;
        request(t + 2, found, even);
        found = lookup(t + 3);
        add(t + 1, odd);
      }
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
}

// Rows that pass by together.
template <int D>
constexpr int weigh_rows() {
  return D == 256 ? 64 : 128;
}

// Passes of a sequence's tiles: `full` of each of the tiles that all rows see in part
// at least, then `step` fewer from tile to tile.  (Rows come G to a token, so the
// rows before a tile's first token are a multiple of the rows of a pass.)
struct WeighPasses {
  int tiles, old;  // tiles, of which all rows see the first old ones
  uint32_t full, first, step;  // first: what tile 0 would have, were it of the latter

  __device__ __forceinline__ WeighPasses(const WeighArgs &a, const WeighSeq &s, int pass_rows) {
    tiles = s.rows > 0 ? (s.keys + kWeighKeys - 1) / kWeighKeys : 0;
    full = (uint32_t)(s.rows + pass_rows - 1) / pass_rows;
    old = a.causal ? min(tiles, s.pos0 < 0 ? 0 : s.pos0 / kWeighKeys + 1) : tiles;
    step = kWeighKeys / pass_rows * a.G;
    // (rows + pos0 G) / pass_rows rounded up, the sum not negative where it is used
    const int64_t seen = max((int64_t)0, s.rows + (int64_t)s.pos0 * a.G);
    first = (uint32_t)((seen + pass_rows - 1) / pass_rows);
  }
  __device__ __forceinline__ uint32_t of(int tile) const {
    return tile < old ? full : first - tile * step;
  }
  // Of the tiles before this one.
  __device__ __forceinline__ uint32_t before(int tile) const {
    const uint32_t a = min(tile, old), n = tile - a;
    // first - (a + i) step for i < n
    return a * full + n * (first - a * step) - (uint32_t)((uint64_t)n * (n - 1) / 2) * step;
  }
  __device__ __forceinline__ uint32_t all() const { return before(tiles); }
};

// The ranges of all passes of a head, the first `more` a pass longer.
struct WeighRanges {
  uint32_t n, len, more;

  __device__ __forceinline__ WeighRanges(uint32_t ranges, uint32_t passes) {
    n = ranges;
    len = passes / ranges;
    more = passes - len * ranges;
  }
  __device__ __forceinline__ uint32_t start(uint32_t r) const { return r * len + min(r, more); }
  __device__ __forceinline__ uint32_t of(uint32_t pass) const {
    const uint32_t longer = more * (len + 1);
    return pass < longer ? pass / (len + 1) : more + (pass - longer) / max(len, 1u);
  }
};

template <int D, bool F8>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void weigh_many_kernel(const WeighArgs a) {
  constexpr int KS = D / 16, CPR = D / 8, RB = weigh_rows<D>(), TILES = RB / 32;
  constexpr int NV = RB * CPR / 256;  // vectors of a thread, of a pass
  static_assert(NV >= 1, "a vector for each thread");
  // Two arrays: a load into one does not hold up reads of the other.
  __shared__ __align__(16) uint16_t s_q0[RB * D], s_q1[RB * D];
  __shared__ __align__(16) float s_lse[4][RB];
  __shared__ uint32_t s_low[4][TILES];  // which are -inf
  constexpr int kAhead = KS < 3 ? KS : 3;

  const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // KV heads vary fastest: workgroups go round the XCDs, so one XCD's cache sees the
  // keys and queries of few heads.
  const int h = blockIdx.x % a.H_kv;
  const uint32_t range = blockIdx.x / a.H_kv;
  const WeighSeq own = weigh_look(a, lane, false);
  uint32_t total = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const WeighPasses p(a, b0 == 0 ? own : weigh_look(a, b0 + lane, false), RB);
    total += __builtin_amdgcn_readfirstlane(wave_sum_u32(p.all()));
  }
  const WeighRanges ranges(gridDim.x / a.H_kv, total);
  const uint32_t begin = ranges.start(range), end = ranges.start(range + 1);

  // Of two workgroups of a CU the older one's waves go first and would end early, the
  // other one left alone (after 68 and 90 us); so the younger ones are favoured for half
  // of their passes (both after 80).
  uint32_t favoured = 2 * blockIdx.x >= gridDim.x ? (end - begin + 1) / 2 : 0;
  if (favoured > 0) __builtin_amdgcn_s_setprio(1);

  // Tokens and heads from a thread's first row to its others, and to the next pass.
  int step_tok[NV], step_g[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    step_tok[i] = i * 256 / CPR / a.G;
    step_g[i] = i * 256 / CPR - step_tok[i] * a.G;
  }
  // The wave's loads into LDS have arrived; a barrier alone does not wait for them.
  auto loaded = []() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" ::: "memory");
  };
  const int pass_tok = RB / a.G, pass_g = RB - pass_tok * a.G;

  // Passes pass0 .. pass1 of a tile's rows, which are those from its first key's on.
  auto walk = [&](int seq, const WeighSeq &s, int tile, int pass0, int pass1, bool shared)
      __attribute__((always_inline)) {
    const int key0 = tile * kWeighKeys;
    const int tile_tok = a.causal ? max(0, key0 - s.pos0) : 0;
    // Rows count from the tile's first; those of the range.
    const int all_rows = s.rows - tile_tok * a.G;
    const int row0 = pass0 * RB, row1 = min(pass1 * RB, all_rows);
    const int pos0 = s.pos0 + tile_tok;
    const int first_tok = row0 / a.G, first_g = row0 - first_tok * a.G;
    // What is waited for first is asked for first: where the wave's keys are, then the
    // rows, then the keys.
    const int32_t *const bt = a.block_tables + seq * a.bt_sb;
    float *const weights = a.weights + ((int64_t)seq * a.H_kv + h) * a.S;
    int found[2];
    float was[2];  // what is added to, of the lanes that write
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = key0 + wave * 64 + i * 32 + l31;
      found[i] = bt[min(key >> a.bs_log2, a.W - 1)];
      was[i] = !shared && half == 0 && key < min(s.keys, s.before) ? weights[key] : 0.f;
    }

    // Rows that pass by, straight into LDS: the thread's vectors, 16 bytes each,
    // whose places are permuted as chunk_swizzle has them; and, of pass p, log-sum-
    // exps for s_lse[p % 4].  The thread's first row lies `off` bytes from the pass's
    // first token, whose head base_g is the pass's first row; from pass to pass
    // without a division, in 32 bits.
    const char *base = (const char *)(a.q + (int64_t)(s.first + tile_tok + first_tok) * a.q_st +
                                      (int64_t)h * a.G * a.q_sh);
    int base_g = first_g;
    auto row_bytes = [&](int tok, int g) {
      return (uint32_t)tok * (uint32_t)a.q_st * 2 + (uint32_t)g * (uint32_t)a.q_sh * 2;
    };
    const uint32_t wrap = row_bytes(1, 0) - row_bytes(0, a.G);
    const int tid_tok = (first_g + tid / CPR) / a.G;
    int g = first_g + tid / CPR - tid_tok * a.G;
    uint32_t off = row_bytes(tid_tok, g);
    auto request = [&](int r0, uint16_t *buf) __attribute__((always_inline)) {
      unrolled<NV>([&](auto n) {
        constexpr int i = decltype(n)::value;
        const int r = (tid + i * 256) / CPR;
        uint32_t at = off + row_bytes(step_tok[i], step_g[i]);
        at += g + step_g[i] >= a.G ? wrap : 0u;
        at = r0 + r < row1 ? at : 0;  // past the last: the first
        const char *from = base + at + chunk_swizzle<D>(r, tid % CPR) * 16;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void *)from,
            (__attribute__((address_space(3))) void *)(buf + (i * 256 + wave * 64) * 8), 16, 0, 0);
      });
      base_g += pass_g;
      const bool next = base_g >= a.G;
      base_g -= next ? a.G : 0;
      base += (int64_t)(pass_tok + next) * a.q_st * 2;
      g += pass_g;
      off += row_bytes(0, pass_g) - (next ? row_bytes(1, 0) : 0u);
      if (g >= a.G) {
        g -= a.G;
        off += wrap;
      }
    };
    const int lse_tok = (first_g + tid % RB) / a.G;
    int lse_g = first_g + tid % RB - lse_tok * a.G;
    const float *lse_at = a.lse +
                          (int64_t)(s.first + tile_tok + first_tok + lse_tok) * a.H_q + h * a.G +
                          lse_g;
    auto request_lse = [&](int r0) __attribute__((always_inline)) {
      float x = -INFINITY;
      if (tid >= RB) return x;
      if (r0 + tid < row1) x = *lse_at;
      lse_at += (int64_t)pass_tok * a.H_q + pass_g;
      lse_g += pass_g;
      if (lse_g >= a.G) {
        lse_g -= a.G;
        lse_at += a.H_q - a.G;
      }
      return x;
    };
    auto store_lse = [&](int pass, float x) __attribute__((always_inline)) {
      if (tid >= RB) return;
      // A row that saw nothing gives nothing.
      const float term = x == -INFINITY ? -INFINITY : -x * a.lse_factor;
      s_lse[pass % 4][tid] = term;
      const uint64_t low = __ballot(term == -INFINITY);
      if (l31 == 0) s_low[pass % 4][tid / 32] = (uint32_t)(half ? low >> 32 : low);
    };
    // The buffers are free: nobody reads what the last tile left.
    const int passes = (row1 - row0 + RB - 1) / RB;
    request(row0, s_q0);
    const float lse0 = request_lse(row0);
    float lse1 = 0.f;
    if (passes > 1) {
      request(row0 + RB, s_q1);
      lse1 = request_lse(row0 + RB);
    }

    // The wave's keys, as the second operand.
    uint4 k[2][KS];
    bool ok[2];
    bool all_ok = true;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = key0 + wave * 64 + i * 32 + l31;
      const WeighKeyAt at = weigh_key_at(a, key, s.keys, found[i]);
      ok[i] = at.ok;
      all_ok = all_ok && at.ok;
      const char *p = weigh_row<D, F8>(a, at.blk, at.ok ? key : 0, h);
      if constexpr (F8) {
        WeighKeys<D, true> raw;
        raw.load(p, half);
        const float scale = chunk_scale(a.k_scales[(int64_t)at.blk * a.H_kv + h]);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) k[i][ks] = raw.get(ks, scale);
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          k[i][ks] = *reinterpret_cast<const uint4 *>(p + ks * 32 + half * 16);
      }
    }
    // The first row that sees the lane's first key (the second one is 32 tokens on), or
    // one before the tile's: the difference is cut there, its product could overflow.
    const int min_row =
        (a.causal ? max(key0 + wave * 64 + l31 - pos0, -kWeighKeys) : -kWeighKeys) * a.G;
    // Rows from here on see all of the wave's keys.
    const int last_key = key0 + wave * 64 + 63;
    const int full_row = a.causal && last_key > pos0 ? min(last_key - pos0, kWeighKeys) * a.G : 0;
    // Rows before see none of them.
    const int first_key = key0 + wave * 64;
    const int first_row =
        a.causal && first_key > pos0 ? min(first_key - pos0, kWeighKeys) * a.G : 0;
    const bool keys_ok = __ballot(!all_ok) == 0;

    store_lse(0, lse0);
    if (passes > 1) store_lse(1, lse1);

    float sum[2] = {0.f, 0.f};
    loaded();
    __syncthreads();
    WeighPlaces<D, F8> place;
    place.init();
    uint4 f[kAhead + 1];  // of the queries, read ahead of their products
    auto fetch = [&](const uint16_t *rows, auto n) {
      constexpr int ks = decltype(n)::value;
      if constexpr (ks < KS) f[ks % (kAhead + 1)] = place.read((const char *)rows, ks);
    };
    auto product = [&](f32x16_t (&st)[2], auto n) {
      constexpr int ks = decltype(n)::value;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        st[i] = chunk_mfma(f[ks % (kAhead + 1)], k[i][ks], ks ? st[i] : f32x16_t{});
    };
    // Exponentials of st, the scores of 32 rows, between the products of the next 32;
    // neg: the first of the rows' terms, and then of the next ones'.
    float4 neg;
    // MASK: of the scores that are not all seen, those that are count, but for rows past
    // the last and those that saw nothing, whose terms are -inf (none: bits).
    auto weigh = [&](const f32x16_t (&st)[2], int base, const float *lse, f32x16_t (&nxt)[2],
                     const uint16_t *rows, const float *next_lse, auto mask, uint32_t none)
        __attribute__((always_inline)) {
      constexpr bool MASK = decltype(mask)::value;
      unrolled<kAhead>([&](auto n) { fetch(rows, n); });
      // Eight scores, four rows of both of the lane's keys, at a time; each is added
      // one later: an addition right behind the exponential would wait.
      float part[2][4], last = 0.f;
      float4 next_neg;
      // Bits 8 g + x of the lane's rows that see its keys and count.
      uint32_t seen[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        seen[i] = ~0u << min(max(0, min_row + i * 32 * a.G - base - 4 * half), 31) &
                  ~(none >> 4 * half);
      auto add = [&](auto n, float p) {
        constexpr int m = decltype(n)::value, i = m % 8 / 4, x = m % 4;
        part[i][x] = m / 8 == 0 ? p : part[i][x] + p;
      };
      unrolled<32>([&](auto n) {
        constexpr int m = decltype(n)::value, g = m / 8, i = m % 8 / 4, x = m % 4;
        // The products end early, so that the next exponentials do not wait.
        constexpr int p0 = m < 28 ? m * KS / 28 : KS, p1 = m < 28 ? (m + 1) * KS / 28 : KS;
        if constexpr (m % 8 == 0)
          next_neg = *reinterpret_cast<const float4 *>(
              (g < 3 ? lse + 8 * (g + 1) : next_lse) + 4 * half);
        unrolled<p1 - p0>([&](auto o) {
          constexpr int ks = p0 + decltype(o)::value;
          product(nxt, std::integral_constant<int, ks>());
          fetch(rows, std::integral_constant<int, ks + kAhead>());
        });
        const float ref = x == 0 ? neg.x : x == 1 ? neg.y : x == 2 ? neg.z : neg.w;
        float p = __builtin_amdgcn_exp2f(fmaf(st[i][4 * g + x], a.c, ref));
        if constexpr (MASK) {
          int on;  // the builtin becomes a comparison and a selection: 6 us of 97
          asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(on) : "v"(seen[i]), "n"(8 * g + x));
          p = __int_as_float(__float_as_int(p) & on);
        }
        if constexpr (m > 0) add(std::integral_constant<int, m - 1>(), last);
        last = p;
        if constexpr (m % 8 == 7) neg = next_neg;
        __builtin_amdgcn_sched_barrier(0);
      });
      add(std::integral_constant<int, 31>(), last);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        sum[i] += (part[i][0] + part[i][1]) + (part[i][2] + part[i][3]);
    };
    auto rows32 = [&](const f32x16_t (&st)[2], int base, const float *lse, f32x16_t (&nxt)[2],
                      const uint16_t *rows, const float *next_lse, uint32_t none)
        __attribute__((always_inline)) {
      place.renew();
      if (keys_ok && none == 0 && base >= full_row) {
        weigh(st, base, lse, nxt, rows, next_lse, std::false_type(), none);
      } else if (base + 32 > first_row) {
        weigh(st, base, lse, nxt, rows, next_lse, std::true_type(), none);
      } else {  // none of them sees any of the wave's keys
        neg = *reinterpret_cast<const float4 *>(next_lse + 4 * half);
        if (base + 64 > first_row)
          unrolled<KS>([&](auto n) {
            fetch(rows, n);
            product(nxt, n);
          });
      }
    };
    // Pass p: the weights of 32 rows with the products of the next 32, at last of the
    // first ones of pass p + 1, whose rows arrive meanwhile; those of pass p + 2 take
    // the buffer of pass p.
    f32x16_t st0[2], st1[2];
    unrolled<KS>([&](auto n) {
      fetch(s_q0, n);
      product(st0, n);
    });
    neg = *reinterpret_cast<const float4 *>(s_lse[0] + 4 * half);
    auto pass = [&](int p, uint16_t *cur, uint16_t *next) __attribute__((always_inline)) {
      const int r0 = row0 + p * RB;
      const float *const lse = s_lse[p % 4];
      auto none = [&](int i) { return (uint32_t)__builtin_amdgcn_readfirstlane(s_low[p % 4][i]); };
      unrolled<TILES - 1>([&](auto n) __attribute__((always_inline)) {
        constexpr int i = decltype(n)::value;
        if constexpr (i % 2 == 0)
          rows32(st0, r0 + 32 * i, lse + 32 * i, st1, cur + 32 * (i + 1) * D, lse + 32 * (i + 1),
                 none(i));
        else
          rows32(st1, r0 + 32 * i, lse + 32 * i, st0, cur + 32 * (i + 1) * D, lse + 32 * (i + 1),
                 none(i));
      });
      loaded();
      __syncthreads();
      const bool more = p + 2 < passes;
      float next_lse = 0.f;
      if (more) {
        request(r0 + 2 * RB, cur);
        next_lse = request_lse(r0 + 2 * RB);
      }
      constexpr int i = TILES - 1;
      rows32(st1, r0 + 32 * i, lse + 32 * i, st0, next, s_lse[(p + 1) % 4], none(i));
      if (more) store_lse(p + 2, next_lse);
      if (favoured > 0 && --favoured == 0) __builtin_amdgcn_s_setprio(0);
    };
    static_assert(TILES % 2 == 0, "two sets of scores in turn");
    for (int p = 0; p < passes; p += 2) {
      pass(p, s_q0, s_q1);
      if (p + 1 < passes) pass(p + 1, s_q1, s_q0);
    }
    __syncthreads();  // the buffers are the next tile's
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float u, v;
      xchg32(sum[i], u, v);
      const int at = wave * 64 + i * 32 + l31, key = key0 + at;
      const float all = ok[i] ? u + v : 0.f;
      if (half != 0) continue;
      if (shared) {
        a.parts[(((int64_t)range * a.H_kv + h) * 2 + (pass0 == 0)) * kWeighKeys + at] = all;
      } else if (key < s.keys) {
        weights[key] = was[i] + all;
      }
    }
  };

  uint32_t before = 0;
  for (int b0 = 0; b0 < a.B && before < end; b0 += kWave) {
    const WeighSeq mine = b0 == 0 ? own : weigh_look(a, b0 + lane, false);
    const uint32_t passes = WeighPasses(a, mine, RB).all();
    const uint32_t incl = wave_incl_scan_u32(passes), last = before + incl, start = last - passes;
    uint64_t todo = __ballot(passes > 0 && start < end && last > begin);
    while (todo != 0) {
      const int l = __builtin_ctzll(todo);
      todo &= todo - 1;
      WeighSeq s;
      s.first = __builtin_amdgcn_readlane(mine.first, l);
      s.pos0 = __builtin_amdgcn_readlane(mine.pos0, l);
      s.keys = __builtin_amdgcn_readlane(mine.keys, l);
      s.rows = __builtin_amdgcn_readlane(mine.rows, l);
      s.before = __builtin_amdgcn_readlane(mine.before, l);
      const WeighPasses p(a, s, RB);
      const uint32_t from = __builtin_amdgcn_readlane(start, l);
      const uint32_t p0 = begin > from ? begin - from : 0, p1 = min(end - from, p.all());
      // The last tile that starts at p0 or before.
      int tile = last_that(p.tiles, [&](int n) { return p.before(n) <= p0; });
      for (; tile < p.tiles && p.before(tile) < p1; ++tile) {
        const uint32_t first = p.before(tile), n = p.of(tile);
        const uint32_t a0 = p0 > first ? p0 - first : 0, a1 = min(p1 - first, n);
        walk(b0 + l, s, tile, (int)a0, (int)a1, a0 > 0 || a1 < n);
      }
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
}

// The parts of tiles that several ranges share, in order.
template <int D>
__global__ __launch_bounds__(kWeighKeys) void weigh_join_kernel(const WeighArgs a, int n_ranges) {
  constexpr int RB = weigh_rows<D>();
  const int lane = threadIdx.x & 63, h = blockIdx.y;
  // Tiles of all sequences, end to end; their passes before them.
  uint32_t total = 0;
  int seq = -1, want = blockIdx.x;
  uint32_t first = 0;
  WeighSeq s = {};
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const WeighSeq mine = weigh_look(a, b0 + lane, false);
    const WeighPasses p(a, mine, RB);
    const uint32_t passes = p.all(), incl = wave_incl_scan_u32(passes);
    const uint32_t tiles = wave_incl_scan_u32((uint32_t)p.tiles);
    const int all_tiles = __builtin_amdgcn_readlane(tiles, 63);
    if (seq < 0 && want < all_tiles) {
      const int l = __popcll(__ballot((int)tiles <= want));
      seq = b0 + l;
      s.pos0 = __builtin_amdgcn_readlane(mine.pos0, l);
      s.keys = __builtin_amdgcn_readlane(mine.keys, l);
      s.rows = __builtin_amdgcn_readlane(mine.rows, l);
      s.before = __builtin_amdgcn_readlane(mine.before, l);
      first = total + __builtin_amdgcn_readlane(incl - passes, l);
      want -= __builtin_amdgcn_readlane(tiles - (uint32_t)p.tiles, l);
    } else if (seq < 0) {
      want -= all_tiles;
    }
    total += __builtin_amdgcn_readlane(incl, 63);
  }
  if (seq < 0) return;
  const WeighPasses p(a, s, RB);
  const WeighRanges ranges((uint32_t)n_ranges, total);
  first += p.before(want);
  const uint32_t r0 = ranges.of(first), r1 = ranges.of(first + p.of(want) - 1);
  const int key = want * kWeighKeys + threadIdx.x;
  if (r0 == r1 || key >= s.keys) return;
  float *const w = a.weights + ((int64_t)seq * a.H_kv + h) * a.S + key;
  const float was = key < s.before ? *w : 0.f;
  float sum = 0.f;
  auto part = [&](uint32_t r) {
    return a.parts + (((int64_t)r * a.H_kv + h) * 2 + (r == r0)) * kWeighKeys + threadIdx.x;
  };
  for (uint32_t r = r0; r <= r1; r += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r + i <= r1 ? *part(r + i) : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[i];
  }
  *w = was + sum;
}

struct WeighPlan {
  bool few, many;
  int ranges;       // of a head, many rows
  int64_t tiles;    // of all sequences of many rows, at most
  int64_t passes;   // likewise
  size_t bytes;
};

static WeighPlan plan_weigh(const int32_t *cu, int B, int G, int H_kv, int D, int window,
                            int64_t keys) {
  WeighPlan p = {};
  const int pass_rows = D == 256 ? weigh_rows<256>() : weigh_rows<128>();
  const int64_t tiles = (keys + kWeighKeys - 1) / kWeighKeys;
  for (int b = 0; b < B; ++b) {
    const int len = cu[b + 1] - cu[b];
    const int64_t rows = (int64_t)(window > 0 ? std::min(len, window) : len) * G;
    if (rows == 0) continue;
    if (rows <= kWeighFewRows) {
      p.few = true;
      continue;
    }
    p.many = true;
    p.tiles += tiles;
    p.passes += tiles * ((rows + pass_rows - 1) / pass_rows);
  }
  // A range for each workgroup that fits the GPU.
  p.ranges = std::max(1, 256 * (D == 256 ? 1 : 2) / H_kv);
  if (p.many) p.bytes = (size_t)p.ranges * H_kv * 2 * kWeighKeys * sizeof(float);
  return p;
}

template <int D, bool F8>
static void launch_weigh(const WeighArgs &a, const WeighPlan &p, hipStream_t s) {
  if (p.many) {
    hipLaunchKernelGGL((weigh_many_kernel<D, F8>), dim3((unsigned)(p.ranges * a.H_kv)), dim3(256),
                       0, s, a);
    hipLaunchKernelGGL(weigh_join_kernel<D>, dim3((unsigned)p.tiles, (unsigned)a.H_kv),
                       dim3(kWeighKeys), 0, s, a, p.ranges);
  }
  if (p.few) {
    const unsigned wgs =
        (unsigned)std::max(1, 256 * weigh_few_fit<D, F8>() / a.H_kv) * a.H_kv;
    hipLaunchKernelGGL((weigh_few_kernel<D, F8>), dim3(wgs), dim3(256), 0, s, a);
  }
}

template <bool F8>
static void launch_weigh_d(const WeighArgs &a, const WeighPlan &p, int D, hipStream_t s) {
  if (D == 32) launch_weigh<32, F8>(a, p, s);
  else if (D == 64) launch_weigh<64, F8>(a, p, s);
  else if (D == 128) launch_weigh<128, F8>(a, p, s);
  else launch_weigh<256, F8>(a, p, s);
}

static bool weigh_shape_ok(const int32_t *cu, int32_t B, int32_t H_q, int32_t H_kv, int64_t S,
                           int32_t window) {
  if (!cu || B <= 0 || B > 65535 || H_kv <= 0 || H_kv > 65535 || H_q <= 0 || H_q > 65536 ||
      H_q % H_kv || H_q / H_kv > 128 || S <= 0 || S > 0x7fffffff || window < 0 || cu[0] != 0)
    return false;
  for (int b = 0; b < B; ++b)
    if (cu[b + 1] < cu[b]) return false;
  return cu[B] <= (1 << 24) && (int64_t)cu[B] * (H_q / H_kv) < (1 << 30);
}

}  // namespace cvsa

using namespace cvsa;

extern "C" size_t cvsa_add_key_weights_workspace_bytes(const int32_t *cu_host, int32_t B,
                                                       int32_t H_q, int32_t H_kv, int32_t D,
                                                       int64_t S, int32_t window) {
  if (!weigh_shape_ok(cu_host, B, H_q, H_kv, S, window)) return 0;
  return plan_weigh(cu_host, B, H_q / H_kv, H_kv, D, window, S).bytes;
}

extern "C" int cvsa_add_key_weights(float *weights, int64_t S, const uint16_t *q,
                                    int64_t q_stride_t, int64_t q_stride_h, const float *lse,
                                    const void *k_cache, const uint8_t *k_scales,
                                    int64_t num_blocks, const int32_t *block_tables,
                                    int64_t bt_stride_b, const int32_t *context_lens,
                                    const int32_t *cu_seqlens, const int32_t *cu_host, int32_t B,
                                    int32_t H_q, int32_t H_kv, int32_t D, int32_t block_size,
                                    int32_t W, float scale, int32_t causal, int32_t window,
                                    void *workspace, size_t workspace_bytes, void *stream) {
  CVSA_REQUIRE(weights && q && lse && k_cache && block_tables && context_lens && cu_seqlens &&
                   cu_host,
               CVSA_ERR_INVALID, "add_key_weights: null pointer argument");
  CVSA_REQUIRE(head_dim_supported(D), CVSA_ERR_UNSUPPORTED,
               "add_key_weights: D=%d not in {32, 64, 128, 256}", D);
  CVSA_REQUIRE(block_size_supported(block_size), CVSA_ERR_UNSUPPORTED,
               "add_key_weights: block_size=%d not in {8, 16, 32, 64, 128}", block_size);
  CVSA_REQUIRE(H_kv > 0 && H_q > 0 && H_q % H_kv == 0, CVSA_ERR_INVALID,
               "add_key_weights: head counts H_q=%d H_kv=%d", H_q, H_kv);
  CVSA_REQUIRE(H_q / H_kv <= 128 && W <= kMaxPagesWide && B <= 65535 && H_kv <= 65535,
               CVSA_ERR_UNSUPPORTED,
               "add_key_weights: G=%d (at most 128), W=%d (at most %d) or B=%d (at most 65535) not "
               "supported", H_q / H_kv, W, kMaxPagesWide, B);
  CVSA_REQUIRE(weigh_shape_ok(cu_host, B, H_q, H_kv, S, window) && num_blocks > 0 && W > 0 &&
                   bt_stride_b >= W,
               CVSA_ERR_INVALID, "add_key_weights: bad sizes or chunk offsets (B=%d W=%d)", B, W);
  CVSA_REQUIRE(S >= (int64_t)W * block_size, CVSA_ERR_INVALID,
               "add_key_weights: weights of %lld keys for tables of %lld", (long long)S,
               (long long)W * block_size);
  CVSA_REQUIRE(scale > 0.f && scale < INFINITY && (causal == 0 || causal == 1), CVSA_ERR_INVALID,
               "add_key_weights: scale must be positive and finite, causal 0 or 1");
  CVSA_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache) & 15) == 0 && q_stride_t % 8 == 0 &&
                   q_stride_h % 8 == 0,
               CVSA_ERR_INVALID, "add_key_weights: rows must be 16-byte aligned");
  const WeighPlan p =
      plan_weigh(cu_host, B, H_q / H_kv, H_kv, D, window, (int64_t)W * block_size);
  if (!p.few && !p.many) return CVSA_OK;
  CVSA_REQUIRE(p.passes < (1LL << 31) && p.tiles < (1LL << 32) / kWeighKeys, CVSA_ERR_UNSUPPORTED,
               "add_key_weights: too many queries and keys");
  // Many rows: the bytes from the first token of a pass to any of its rows are counted
  // in 32 bits.  (Few rows have addresses of 64.)
  const int64_t G = H_q / H_kv;
  const int64_t pass_rows = D == 256 ? weigh_rows<256>() : weigh_rows<128>();
  CVSA_REQUIRE(q_stride_t >= 0 && q_stride_h >= 0, CVSA_ERR_INVALID,
               "add_key_weights: negative stride of the queries");
  CVSA_REQUIRE(!p.many || (q_stride_t < (1LL << 31) && (G == 1 || q_stride_h < (1LL << 31)) &&
                           (pass_rows + G - 2) / G * q_stride_t + (G - 1) * q_stride_h <
                               (1LL << 31)),
               CVSA_ERR_UNSUPPORTED, "add_key_weights: queries too far apart");
  CVSA_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes), CVSA_ERR_WORKSPACE,
               "add_key_weights: needs a workspace of %zu bytes", p.bytes);
  WeighArgs a = {};
  a.q = q; a.q_st = q_stride_t; a.q_sh = q_stride_h;
  a.lse = lse;
  a.k_cache = (const char *)k_cache; a.k_scales = k_scales;
  a.num_blocks = (int)std::min<int64_t>(num_blocks, INT32_MAX);
  a.block_tables = block_tables; a.bt_sb = bt_stride_b; a.W = W;
  a.context_lens = context_lens; a.cu = cu_seqlens;
  a.B = B; a.H_q = H_q; a.H_kv = H_kv; a.G = H_q / H_kv;
  a.bs_log2 = __builtin_ctz(block_size);
  a.c = (float)(scale * 1.4426950408889634);
  a.lse_factor = (float)((double)a.c / scale);
  a.causal = causal; a.window = window;
  a.weights = weights; a.S = S;
  a.parts = (float *)workspace;
  const hipStream_t s = (hipStream_t)stream;
  if (k_scales) launch_weigh_d<true>(a, p, D, s);
  else launch_weigh_d<false>(a, p, D, s);
  return cvsa_host::check_launch("add_key_weights");
}
