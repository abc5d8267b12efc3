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
// Many rows: the matrix and vector pipes bound it (32 exponentials of a wave to 16
// products at D = 128).  A workgroup keeps 256 keys in registers, 64 a wave, and the
// rows pass by through LDS, 64 at a time, so a row is read once for 256 keys and an
// LDS read feeds two products.  Rows are cut into segments, a (segment, 256 keys)
// pair is a job; jobs whose rows see none of their keys are left out.  If a
// sequence has several segments their sums are joined in order by a second kernel.
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
  // Sequences of few rows have at most few_rows of them, those of many more.
  int few_rows;
  // Many rows.
  int segment;            // rows
  int max_segments;       // of a sequence
  float *parts;           // [B, H_kv, max_segments, S] where max_segments > 1
};

constexpr int kWeighFewRows = 32;
constexpr int kWeighKeys = 256;      // of a job of many rows
constexpr int kWeighRows = 64;       // that pass by together
constexpr int kMaxSegments = 32;

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
  if (len > 0 && (s.rows <= a.few_rows) == few)
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
  // The operand of step ks.
  __device__ __forceinline__ uint4 get(int ks) const {
    if constexpr (F8) {
      const uint4 &v = w[ks / 2];
      return chunk_from_8(ks % 2 ? make_uint2(v.z, v.w) : make_uint2(v.x, v.y), 1.f, 1.f);
    } else {
      return w[ks];
    }
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
  const int h = blockIdx.x % a.H_kv;
  const uint32_t range = blockIdx.x / a.H_kv * 4 + wave, ranges = gridDim.x / a.H_kv * 4;

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
      const int old = __builtin_amdgcn_readlane(mine.before, l);
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
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          s = chunk_mfma(__builtin_bit_cast(uint4, q[ks]), x.k.get(ks), ks ? s : f32x16_t{});
        const int key = t * 32 + l31;
        // The first row that sees the key, and the lane's rows from there on.
        const int min_row = a.causal && key > pos0 ? min(key - pos0, 1 << 20) * a.G : 0;
        const float c = a.c * chunk_scale(x.scale);
        float p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = 8 * (e / 4) + e % 4;
          const bool see = (live >> e & 1) && r + 4 * half >= min_row;
          const float v = __builtin_amdgcn_exp2f(fmaf(s[e], c, neg[e]));
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

// Segment `seg` of a sequence of many rows: the keys that its last row sees.
__device__ __forceinline__ int weigh_segment_keys(const WeighArgs &a, int pos0, int keys, int rows,
                                                  int seg) {
  if (seg * a.segment >= rows) return 0;
  const int last = (min((seg + 1) * a.segment, rows) - 1) / a.G;
  return a.causal ? max(0, min(keys, pos0 + last + 1)) : keys;
}

template <int D, bool F8>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void weigh_many_kernel(const WeighArgs a) {
  constexpr int KS = D / 16, CPR = D / 8, RB = kWeighRows;
  constexpr int NV = RB * CPR / 256;  // vectors of a thread, of the rows that pass by
  static_assert(NV >= 1, "a vector for each thread");
  __shared__ __align__(16) uint16_t s_q[2][RB * D];
  __shared__ __align__(16) float s_lse[2][RB];

  const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const WeighSeq own = weigh_look(a, lane, false);
  auto jobs_of = [&](const WeighSeq &s) {
    uint32_t n = 0;
    for (int seg = 0; seg < a.max_segments; ++seg)
      n += (uint32_t)(weigh_segment_keys(a, s.pos0, s.keys, s.rows, seg) + kWeighKeys - 1) /
           kWeighKeys;
    return n;
  };
  const uint32_t own_jobs = jobs_of(own);

  for (uint32_t id = blockIdx.x;; id += gridDim.x) {
    const int h = id % a.H_kv;
    uint32_t job = id / a.H_kv;
    // The job's sequence, segment and keys.
    int seq = -1;
    WeighSeq s = {};
    for (int b0 = 0; b0 < a.B; b0 += kWave) {
      const WeighSeq look = b0 == 0 ? own : weigh_look(a, b0 + lane, false);
      const uint32_t n = b0 == 0 ? own_jobs : jobs_of(look);
      const uint32_t incl = wave_incl_scan_u32(n);
      const uint32_t all = __builtin_amdgcn_readlane(incl, 63);
      if (job < all) {
        const int l = __popcll(__ballot(incl <= job));
        seq = b0 + l;
        s.first = __builtin_amdgcn_readlane(look.first, l);
        s.pos0 = __builtin_amdgcn_readlane(look.pos0, l);
        s.keys = __builtin_amdgcn_readlane(look.keys, l);
        s.rows = __builtin_amdgcn_readlane(look.rows, l);
        s.before = __builtin_amdgcn_readlane(look.before, l);
        job -= __builtin_amdgcn_readlane(incl - n, l);
        break;
      }
      job -= all;
    }
    if (seq < 0) return;
    int seg, tile;
    {
      const uint32_t n = lane < a.max_segments
                             ? (uint32_t)(weigh_segment_keys(a, s.pos0, s.keys, s.rows, lane) +
                                          kWeighKeys - 1) / kWeighKeys
                             : 0u;
      const uint32_t incl = wave_incl_scan_u32(n);
      seg = __popcll(__ballot(incl <= job));
      tile = (int)(job - __builtin_amdgcn_readlane(incl - n, seg));
    }
    const int key0 = tile * kWeighKeys;
    const int row1 = min((seg + 1) * a.segment, s.rows);
    int row0 = seg * a.segment;
    // Rows before see none of the keys; whole passes of rows.
    if (a.causal && key0 > s.pos0)
      row0 = max(row0, (int)min((int64_t)(key0 - s.pos0) * a.G, (int64_t)row1 - 1) / RB * RB);
    const int32_t *const bt = a.block_tables + seq * a.bt_sb;

    // Rows that pass by: the thread's vectors and, of the first threads, a
    // log-sum-exp.
    uint4 next[NV];
    float next_lse = 0.f;
    auto at_row = [&](int r) {  // its token and head
      const int row = min(r, row1 - 1), tok = row / a.G;
      return make_int2(s.first + tok, h * a.G + row - tok * a.G);
    };
    auto request = [&](int r0) {
      unrolled<NV>([&](auto n) {
        constexpr int i = decltype(n)::value;
        const int c = tid + i * 256;
        const int2 at = at_row(r0 + c / CPR);
        next[i] = *reinterpret_cast<const uint4 *>(a.q + (int64_t)at.x * a.q_st +
                                                   (int64_t)at.y * a.q_sh + c % CPR * 8);
      });
      if (tid < RB) {
        const int2 at = at_row(r0 + tid);
        const float x = a.lse[(int64_t)at.x * a.H_q + at.y];
        // A row that saw nothing gives nothing.
        next_lse = x == -INFINITY ? -INFINITY : -x * a.lse_factor;
      }
    };
    auto store = [&](int buf) {
      unrolled<NV>([&](auto n) {
        constexpr int i = decltype(n)::value;
        const int c = tid + i * 256, r = c / CPR;
        *reinterpret_cast<uint4 *>(&s_q[buf][r * D + chunk_swizzle<D>(r, c % CPR) * 8]) = next[i];
      });
      if (tid < RB) s_lse[buf][tid] = next_lse;
    };
    request(row0);

    // The wave's keys, as the second operand: bf16, the scales apart.
    uint4 k[2][KS];
    float c[2];
    int min_row[2];
    bool ok[2];
    bool all_ok = true;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = key0 + wave * 64 + i * 32 + l31;
      const WeighKeyAt at =
          weigh_key_at(a, key, s.keys, bt[min(key >> a.bs_log2, a.W - 1)]);
      ok[i] = at.ok;
      all_ok = all_ok && at.ok;
      const char *p = weigh_row<D, F8>(a, at.blk, at.ok ? key : 0, h);
      if constexpr (F8) {
        // Columns as the bf16 rows of LDS have them.
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          k[i][ks] = chunk_from_8(*reinterpret_cast<const uint2 *>(p + ks * 16 + half * 8), 1.f,
                                  1.f);
        c[i] = a.c * chunk_scale(a.k_scales[(int64_t)at.blk * a.H_kv + h]);
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          k[i][ks] = *reinterpret_cast<const uint4 *>(p + ks * 32 + half * 16);
        c[i] = a.c;
      }
      min_row[i] = a.causal && key > s.pos0
                       ? (int)min((int64_t)(key - s.pos0) * a.G, (int64_t)0x7fffffff) : 0;
    }
    // Rows from here on see all of the wave's keys.
    const int last_key = key0 + wave * 64 + 63;
    const int full_row = a.causal && last_key > s.pos0
                             ? (int)min((int64_t)(last_key - s.pos0) * a.G, (int64_t)0x7fffffff)
                             : 0;
    const bool keys_ok = __ballot(!all_ok) == 0;

    float sum[2] = {0.f, 0.f};
    store(0);
    __syncthreads();
    int buf = 0;
    for (int r0 = row0; r0 < row1; r0 += RB, buf ^= 1) {
      if (r0 + RB < row1) request(r0 + RB);
#pragma unroll
      for (int rt = 0; rt < RB / 32; ++rt) {
        f32x16_t st[2];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint4 x = chunk_read_k((const char *)&s_q[buf][rt * 32 * D] + chunk_k_place<D>(ks));
#pragma unroll
          for (int i = 0; i < 2; ++i) st[i] = chunk_mfma(x, k[i][ks], ks ? st[i] : f32x16_t{});
        }
        float neg[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 v =
              *reinterpret_cast<const float4 *>(&s_lse[buf][rt * 32 + 8 * g + 4 * half]);
          neg[4 * g] = v.x; neg[4 * g + 1] = v.y; neg[4 * g + 2] = v.z; neg[4 * g + 3] = v.w;
        }
        const int base = r0 + rt * 32;
        const bool whole = keys_ok && base >= full_row && base + 32 <= row1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            p[e] = __builtin_amdgcn_exp2f(fmaf(st[i][e], c[i], neg[e]));
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int r = base + 8 * (e / 4) + 4 * half + e % 4;
              p[e] = r >= min_row[i] && r < row1 && neg[e] != -INFINITY ? p[e] : 0.f;
            }
          }
          sum[i] += sum16(p);
        }
      }
      if (r0 + RB < row1) store(buf ^ 1);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float u, v;
      xchg32(sum[i], u, v);
      const int key = key0 + wave * 64 + i * 32 + l31;
      const float total = ok[i] ? u + v : 0.f;
      if (half == 0 && key < s.keys) {
        const int64_t at = ((int64_t)seq * a.H_kv + h);
        if (s.rows > a.segment)
          a.parts[(at * a.max_segments + seg) * a.S + key] = total;
        else
          a.weights[at * a.S + key] = (key < s.before ? a.weights[at * a.S + key] : 0.f) + total;
      }
    }
  }
}

// The segments' sums, in order.
__global__ __launch_bounds__(256) void weigh_join_kernel(const WeighArgs a) {
  const int seq = blockIdx.z, h = blockIdx.y;
  const int first = a.cu[seq], len = a.cu[seq + 1] - first, ctx = a.context_lens[seq];
  const int count = a.window > 0 ? min(len, a.window) : len, rows = count * a.G;
  if (rows <= a.few_rows || rows <= a.segment) return;
  const int keys = max(0, min(ctx, a.W << a.bs_log2)), pos0 = ctx - count;
  const int segs = (rows + a.segment - 1) / a.segment;
  const int64_t at = (int64_t)seq * a.H_kv + h;
  for (int key = blockIdx.x * 256 + threadIdx.x; key < keys; key += gridDim.x * 256) {
    float sum = key < ctx - len ? a.weights[at * a.S + key] : 0.f;
    // Whole jobs of 256 keys were written.
    int seg = 0;
    while (seg < segs && (key & -kWeighKeys) >= weigh_segment_keys(a, pos0, keys, rows, seg)) ++seg;
    for (; seg < segs; ++seg) sum += a.parts[(at * a.max_segments + seg) * a.S + key];
    a.weights[at * a.S + key] = sum;
  }
}

struct WeighPlan {
  bool few, many;
  int segment, max_segments;
  size_t bytes;
};

static WeighPlan plan_weigh(const int32_t *cu, int B, int G, int H_kv, int window, int64_t S) {
  WeighPlan p = {};
  int64_t most = 0;
  for (int b = 0; b < B; ++b) {
    const int len = cu[b + 1] - cu[b];
    const int64_t rows = (int64_t)(window > 0 ? std::min(len, window) : len) * G;
    if (rows == 0) continue;
    if (rows <= kWeighFewRows) p.few = true;
    else p.many = true;
    most = std::max(most, rows);
  }
  // Segments of 512 rows, or as long as the most segments need.
  p.segment = (int)std::max<int64_t>(512, ((most + kMaxSegments - 1) / kMaxSegments + 63) / 64 * 64);
  p.max_segments = (int)std::max<int64_t>(1, (most + p.segment - 1) / p.segment);
  if (p.many && p.max_segments > 1)
    p.bytes = (size_t)B * H_kv * p.max_segments * (size_t)S * sizeof(float);
  return p;
}

template <int D, bool F8>
static void launch_weigh(const WeighArgs &a, const WeighPlan &p, hipStream_t s) {
  if (p.many) {
    const unsigned wgs = 256 * (D == 256 ? 1 : 2);
    hipLaunchKernelGGL((weigh_many_kernel<D, F8>), dim3(wgs), dim3(256), 0, s, a);
    if (p.max_segments > 1) {
      const unsigned x = (unsigned)std::min<int64_t>(64, (a.S + 255) / 256);
      hipLaunchKernelGGL(weigh_join_kernel, dim3(x, a.H_kv, a.B), dim3(256), 0, s, a);
    }
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
                                                       int32_t H_q, int32_t H_kv, int64_t S,
                                                       int32_t window) {
  if (!weigh_shape_ok(cu_host, B, H_q, H_kv, S, window)) return 0;
  return plan_weigh(cu_host, B, H_q / H_kv, H_kv, window, S).bytes;
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
  const WeighPlan p = plan_weigh(cu_host, B, H_q / H_kv, H_kv, window, S);
  if (!p.few && !p.many) return CVSA_OK;
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
  a.few_rows = kWeighFewRows;
  a.segment = p.segment; a.max_segments = p.max_segments;
  a.parts = (float *)workspace;
  const hipStream_t s = (hipStream_t)stream;
  if (k_scales) launch_weigh_d<true>(a, p, D, s);
  else launch_weigh_d<false>(a, p, D, s);
  return cvsa_host::check_launch("add_key_weights");
}
