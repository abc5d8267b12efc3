// Eviction from the paged cache by accumulated attention weight
// (cvsa_evict_tokens): of each sequence and KV head the first `sinks` tokens, the
// last `recent` and, of those between, the ones of the largest weights stay, `keep`
// in all; ties go to the lowest slot.
//
// Attention does not depend on the order of the keys, so what can stay in place
// does: slots below keep - recent whose token stays are not touched; the others of
// them take the kept tokens from behind, in order; the last `recent` go to the end,
// in order, so that the next call finds them there.  That moves the fewest rows: a
// token in the middle moves only if its slot is cut off.
//
// The m-th largest weight is found by its bits, 11, 11 and 10 at a time (histograms
// in LDS); then a walk over the slots in order writes down which old slot each new
// one gets.  Rows of up to 16384 slots (by the tables' width): one workgroup for each
// sequence and head has its weights in registers.  Longer ones: chunks of 8192 slots
// have a workgroup each, a launch for each histogram and one for the walk, in which
// every chunk adds up the others' counts (131072 slots, 8 heads: one workgroup each
// 167 us, so 30 before the rows are moved).
//
// A destination is a source itself only among slots keep - recent .. keep.  Where there
// are many sequences and heads, the workgroup that planned moves the rows too: those of
// the holes, then the window's in rounds, in order, each read before it is written.
// Else a wave for each 64 slots moves their arrivals in a launch of its own, in no
// order, and workgroups of the first launch copy the window's rows aside.
//
// Measured: 32 sequences of 8 heads, 4160 tokens to 4096, 256 of them recent, 8 bits: 26
// to 30 us in one launch for 51 MB (23 where the caches hold some of them, 39 where they
// hold none; 12 until the rows are known); a first cut of 131072 to 16384, 8 heads of
// bf16, 14600 rows a head: 7 + 7 + 7 + 10 and 28 to move 120 MB (41 from memory alone).
// Cut again at the same length, as a loop of calls does, the heaviest tokens are in
// front already: 8200 rows, then 5900, 4700 .., moved in 25 us to 12.  The plans are
// chains of short dependent steps, not bound by a rate.
//
// 8 bits: a page with arrivals gets the largest scale of its tokens' pages; payloads
// are shifted to it, which rounds only what becomes subnormal.
#include "cvsa_common.h"

#include "cache8.h"

#include <algorithm>

namespace cvsa {

struct EvictArgs {
  float *weights;  // [B, H_kv, S]
  int64_t S;
  char *k_cache, *v_cache;
  uint8_t *k_scales, *v_scales;
  int64_t num_blocks;
  const int32_t *block_tables;
  int64_t bt_sb;
  int W, bs_log2;
  const int32_t *context_lens;
  int B, H_kv, row_bytes;  // of a token and head
  int keep, sinks, recent;
  int32_t *kept;           // [B, H_kv, keep]
  int select_wgs;          // workgroups of a launch before those that copy aside
  // Workspace, each [B, H_kv, ...].  What slots keep - recent .. keep hold, and the
  // scales of the pages from the first of these slots' to the last's.
  char *aside;             // [2, recent, row_bytes]
  float *aside_weights;    // [recent]
  uint8_t *aside_scales;   // [2, aside_pages]
  int aside_pages;
  // Short rows.
  int32_t *pages;          // [1 + pages]: pages with arrivals, their number first
  // Long rows: of chunks.
  int chunks;              // of a row of the tables
  uint16_t *hist;          // [3, chunks, kBins]
  uint32_t *above;         // [chunks]: weights above the bins chosen so far
  uint32_t *state;         // [4]: bins and what is still wanted, after passes 1 and 2
  int32_t *tails;          // [keep]: kept slots from keep - recent on, the last first
  int32_t *n_holes;        // [1]
};

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / kWave;
constexpr int kBins = 2048, kCopies = 4;
constexpr int kChunk = 8 * kEvictThreads;       // slots
constexpr int kShortRow = 16 * kEvictThreads;

__device__ __forceinline__ int evict_context(const EvictArgs &a, int b) {
  return max(0, min(a.context_lens[b], a.W << a.bs_log2));
}
// Block of a slot, -1: none of the pool.
__device__ __forceinline__ int evict_block(const EvictArgs &a, int b, int slot) {
  const int blk = a.block_tables[b * a.bt_sb + (slot >> a.bs_log2)];
  return (uint32_t)blk < (uint64_t)a.num_blocks ? blk : -1;
}
// Row of a slot and head in the caches.
__device__ __forceinline__ int64_t evict_row(const EvictArgs &a, int blk, int slot, int h) {
  const int64_t token = ((int64_t)blk << a.bs_log2) + (slot & ((1 << a.bs_log2) - 1));
  return token * a.H_kv + h;
}

// Weights' order as unsigned numbers; NaN is above all, zeros are equal.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xffffffffu;
  return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}

// Bits that a pass looks at.
__host__ __device__ constexpr int pass_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__host__ __device__ constexpr int pass_bits(int pass) { return pass == 2 ? 10 : 11; }

// Sums over the workgroup: of the threads before this one, and of all.  s is used
// again only after another barrier.
struct EvictScan {
  uint32_t before, all;
};
__device__ __forceinline__ EvictScan evict_scan(uint32_t v, uint32_t *s) {
  const int wave = threadIdx.x >> 6;
  const uint32_t incl = wave_incl_scan_u32(v);
  if ((threadIdx.x & 63) == 63) s[wave] = incl;
  __syncthreads();
  EvictScan r = {incl - v, 0};
#pragma unroll
  for (int w = 0; w < kEvictWaves; ++w) {
    const uint32_t x = s[w];
    r.before += w < wave ? x : 0u;
    r.all += x;
  }
  return r;
}

// The bin that holds the want-th largest, and how many are above it, from the
// thread's two bins 2047 - 2 t (n0) and the one below (n1).
struct EvictBin {
  uint32_t bin, above;
};
struct EvictFind {  // LDS of one search
  uint32_t sum[kEvictWaves], bin, above;
};
__device__ __forceinline__ EvictBin evict_find(uint32_t n0, uint32_t n1, int bits, uint32_t want,
                                               EvictFind &f) {
  const EvictScan s = evict_scan(n0 + n1, f.sum);
  if (s.before < want && want <= s.before + n0 + n1) {
    const bool second = want > s.before + n0;
    f.bin = (uint32_t)((1 << bits) - 1 - 2 * (int)threadIdx.x - (second ? 1 : 0));
    f.above = s.before + (second ? n0 : 0u);
  }
  __syncthreads();
  return {f.bin, f.above};
}

// A thread's share of the slots: four together in each of N steps of the workgroup.
template <int N>
struct EvictKeys {
  uint32_t key[4 * N];

  static __device__ __forceinline__ int slot(int first, int i) {
    return first + i / 4 * 4 * kEvictThreads + 4 * (int)threadIdx.x + i % 4;
  }
  // Slots first .. of a row, those of begin .. end.
  __device__ __forceinline__ void load(const float *w, int first, int begin, int end) {
    float v[4 * N];
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
      const int j = slot(first, i);
      v[i] = j >= begin && j < end ? w[j] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) key[i] = weight_key(v[i]);
  }
  // Counts of those whose bits `known` are `prefix`, by the next ones, into hist.
  __device__ __forceinline__ void count(uint32_t *hist, int pass, uint32_t known, uint32_t prefix,
                                        int first, int begin, int end) const {
    const uint32_t mask = (1u << pass_bits(pass)) - 1;
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
      const int j = slot(first, i);
      if (j >= begin && j < end && (key[i] & known) == prefix)
        atomicAdd(&hist[key[i] >> pass_shift(pass) & mask], 1u);
    }
  }
};

// Clears n words (a multiple of 4) of LDS; the caller waits.
__device__ __forceinline__ void evict_clear(void *s, int n) {
  for (int i = threadIdx.x; i < n / 4; i += kEvictThreads)
    reinterpret_cast<uint4 *>(s)[i] = make_uint4(0, 0, 0, 0);
}
// A thread's two bins from the top, over the copies, which it leaves cleared.
template <int BITS>
__device__ __forceinline__ void evict_bins(uint32_t (*hist)[1 << BITS], uint32_t &n0,
                                           uint32_t &n1) {
  const int top = (1 << BITS) - 1 - 2 * (int)threadIdx.x;
  n0 = n1 = 0;
  if (top <= 0) return;
#pragma unroll
  for (int c = 0; c < kCopies; ++c) {
    uint2 &at = *reinterpret_cast<uint2 *>(&hist[c][top - 1]);
    const uint2 two = at;
    at = make_uint2(0, 0);
    n0 += two.y;
    n1 += two.x;
  }
}

__device__ __forceinline__ void evict_copy_aside(const EvictArgs &a) {
  // A thread for each 16 bytes of keys and of values, then one for each page.
  const int per_row = a.row_bytes / 16, front = a.keep - a.recent;
  const int64_t n_bh = (int64_t)a.B * a.H_kv, n_rows = n_bh * a.recent;
  int64_t i = (int64_t)((int)blockIdx.x - a.select_wgs) * kEvictThreads + threadIdx.x;
  if (i < n_rows * per_row) {
    const int64_t row = i / per_row, bh = row / a.recent;
    const int part = (int)(i - row * per_row), n = (int)(row - bh * a.recent);
    const int b = (int)(bh / a.H_kv), h = (int)(bh % a.H_kv);
    if (evict_context(a, b) <= a.keep) return;
    const int slot = front + n, blk = evict_block(a, b, slot);
    if (part == 0) a.aside_weights[row] = a.weights[bh * a.S + slot];
    if (blk < 0) return;
    const int64_t from = evict_row(a, blk, slot, h) * a.row_bytes + part * 16;
    char *const to = a.aside + ((bh * 2) * a.recent + n) * a.row_bytes + part * 16;
    *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(a.k_cache + from);
    *reinterpret_cast<uint4 *>(to + (int64_t)a.recent * a.row_bytes) =
        *reinterpret_cast<const uint4 *>(a.v_cache + from);
    return;
  }
  i -= n_rows * per_row;
  if (!a.k_scales || i >= n_bh * a.aside_pages) return;
  const int64_t bh = i / a.aside_pages;
  const int n = (int)(i - bh * a.aside_pages), b = (int)(bh / a.H_kv), h = (int)(bh % a.H_kv);
  if (evict_context(a, b) <= a.keep) return;
  const int blk = evict_block(a, b, ((front >> a.bs_log2) + n) << a.bs_log2);
  if (blk < 0) return;
  a.aside_scales[bh * 2 * a.aside_pages + n] = a.k_scales[(int64_t)blk * a.H_kv + h];
  a.aside_scales[(bh * 2 + 1) * a.aside_pages + n] = a.v_scales[(int64_t)blk * a.H_kv + h];
}

__device__ __forceinline__ int64_t shfl_i64(int64_t v, int lane) {
  const uint32_t lo = (uint32_t)__shfl((int)v, lane, 64);
  return (int64_t)__shfl((int)(v >> 32), lane, 64) << 32 | lo;
}
// Most of a lane's page: the largest of the 2^log2 lanes (64 at most) that have it.
__device__ __forceinline__ uint32_t page_max(uint32_t v, int log2) {
  for (int m = 1; m < 1 << min(log2, 6); m *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, m, 64));
  return v;
}

// What a lane's page gets: where its slots' rows come from.
struct EvictPage {
  int slot0, count, blk;        // its first slot, how many; blk -1: none of the pool
  int src[2], from[2];          // of the lane's slots: old slots (themselves: they stay), blocks
  int shift[2][2];              // of keys' and values' payloads
  int byte[2];                  // the page's scales, where they change (-1)
};

// The page's scales, and how far payloads are shifted: to the largest scale of the
// page's tokens.  were: of keys and values, those of pages up to last_page, which may
// have got others by now (null: none has).
__device__ __forceinline__ void evict_scales(const EvictArgs &a, int h, int row0,
                                             const uint8_t *were_k, const uint8_t *were_v,
                                             EvictPage &p) {
  const int last_page = (a.keep - 1) >> a.bs_log2;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const uint8_t *const scales = kv ? a.v_scales : a.k_scales;
    const uint8_t *const were = kv ? were_v : were_k;
    const int old = p.blk >= 0 ? scales[(int64_t)p.blk * a.H_kv + h] : 0;
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int r = row0 + 64 * n, of = p.src[n] >> a.bs_log2;
      p.shift[kv][n] = 0;
      if (r >= p.count || p.blk < 0) continue;
      p.shift[kv][n] = p.src[n] == p.slot0 + r   ? old
                       : p.from[n] < 0           ? 0
                       : were && of <= last_page ? were[of]
                                                 : scales[(int64_t)p.from[n] * a.H_kv + h];
      top = max(top, (uint32_t)p.shift[kv][n]);
    }
    const int byte = (int)page_max(top, a.bs_log2);
    p.byte[kv] = byte != old ? byte : -1;
#pragma unroll
    for (int n = 0; n < 2; ++n) p.shift[kv][n] -= byte;
  }
}
__device__ __forceinline__ void evict_put_scales(const EvictArgs &a, int h, int row0,
                                                 const EvictPage &p) {
  if (row0 != 0 || p.blk < 0) return;
  if (p.byte[0] >= 0) a.k_scales[(int64_t)p.blk * a.H_kv + h] = (uint8_t)p.byte[0];
  if (p.byte[1] >= 0) a.v_scales[(int64_t)p.blk * a.H_kv + h] = (uint8_t)p.byte[1];
}
// Whether the row of the lane's slot n is written: one that stays, only where its
// payload changes with the scale.
__device__ __forceinline__ bool evict_writes(const EvictPage &p, int row0, int n) {
  const int r = row0 + 64 * n;
  return r < p.count && p.blk >= 0 &&
         (p.src[n] != p.slot0 + r ? p.from[n] >= 0 : (p.shift[0][n] | p.shift[1][n]) != 0);
}

// Moves the rows that a wave's lanes have to write, each of its slots; four groups of
// both keys and values are read before they are written.  ASIDE: old slots front ..
// keep are read where they were copied to.
template <bool F8, bool ASIDE>
__device__ __forceinline__ void evict_move_rows(const EvictArgs &a, int h, int row0,
                                                const EvictPage &p, const char *aside,
                                                int front) {
  constexpr int kBatch = 4;
  const int lane = threadIdx.x & 63;
  const int per_row = a.row_bytes / 16, rows = 64 / per_row;  // lanes of a row, rows at once
  const int part = lane % per_row * 16, sub = lane / per_row;
  unrolled<2>([&](auto half) __attribute__((always_inline)) {
    constexpr int n = decltype(half)::value;
    if (n == 1 && a.bs_log2 <= 6) return;
    const int slot = p.slot0 + row0 + 64 * n;
    const bool write = evict_writes(p, row0, n);
    const uint64_t mask = __ballot(write);
    const int n_rows = __popcll(mask);
    // Their lanes first, in order.
    const int before = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                      __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    const int list = __builtin_amdgcn_ds_permute(
        (write ? before : n_rows + lane - before) * 4, lane);
    // Rows of the caches, or -1 - n: row n of those copied aside.
    const int64_t to = evict_row(a, p.blk, slot, h);
    int64_t at = evict_row(a, p.from[n], p.src[n], h);
    if (ASIDE && p.src[n] != slot && p.src[n] < a.keep) at = -1 - (int64_t)(p.src[n] - front);
    const int shifts = F8 ? (p.shift[0][n] + 256) | (p.shift[1][n] + 256) << 16 : 0;
    for (int t0 = 0; t0 < n_rows; t0 += rows * kBatch) {
      uint4 v[kBatch][2];
      int by[kBatch];
      int64_t to_row[kBatch];
      unrolled<kBatch>([&](auto group) __attribute__((always_inline)) {
        constexpr int g = decltype(group)::value;
        const int t = t0 + g * rows + sub, of = __shfl(list, min(t, 63), 64);
        int64_t row = shfl_i64(at, of);
        to_row[g] = shfl_i64(to, of);
        by[g] = F8 ? __shfl(shifts, of, 64) : 0;
        v[g][0] = v[g][1] = make_uint4(0, 0, 0, 0);
        if (t >= n_rows) return;
        const bool put_aside = ASIDE && row < 0;
        const char *const k = put_aside ? aside : a.k_cache;
        const char *const v_ = put_aside ? aside + (int64_t)a.recent * a.row_bytes : a.v_cache;
        row = (put_aside ? -1 - row : row) * a.row_bytes + part;
        v[g][0] = *reinterpret_cast<const uint4 *>(k + row);
        v[g][1] = *reinterpret_cast<const uint4 *>(v_ + row);
      });
      unrolled<kBatch>([&](auto group) __attribute__((always_inline)) {
        constexpr int g = decltype(group)::value;
        if (t0 + g * rows + sub >= n_rows) return;
        if constexpr (F8) {
          const int k = (by[g] & 0xffff) - 256, v_ = (by[g] >> 16) - 256;
          if (k != 0) v[g][0] = shifted_8_bits(v[g][0], k);
          if (v_ != 0) v[g][1] = shifted_8_bits(v[g][1], v_);
        }
        const int64_t row = to_row[g] * a.row_bytes + part;
        *reinterpret_cast<uint4 *>(a.k_cache + row) = v[g][0];
        *reinterpret_cast<uint4 *>(a.v_cache + row) = v[g][1];
      });
    }
  });
}

// Short rows: old slots of the new ones; N steps of 4096 slots.  Then the pages with
// arrivals (MOVE 0), or their rows are moved here (1, and 2: of 8 bits).
template <int N, int MOVE>
__global__ __launch_bounds__(kEvictThreads) void evict_plan_kernel(const EvictArgs a) {
  if (MOVE == 0 && (int)blockIdx.x >= a.select_wgs) {
    evict_copy_aside(a);
    return;
  }
  // Histograms, the passes' in turn, as each leaves its own cleared; after them, in
  // their place, the holes and the old slots.
  constexpr int kSlots = N * 4 * kEvictThreads, kPages = kSlots / 8;
  __shared__ __align__(16) union {
    uint32_t hist[2][kCopies][kBins];
    uint16_t slots[2][kSlots];
  } s;
  uint16_t *const holes = s.slots[0], *const src = s.slots[1];
  __shared__ __align__(16) uint8_t s_page[kPages];
  __shared__ EvictFind s_find[3];
  __shared__ uint32_t s_step[N][kEvictWaves], s_sum[2][kEvictWaves], s_stay;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / a.H_kv);
  float *const w = a.weights + bh * a.S;
  EvictKeys<N> keys;
  // Of all the tables' slots: the context's length is on its way yet.
  keys.load(w, 0, 0, a.W << a.bs_log2);
  const int ctx = evict_context(a, b);
  int32_t *const kept = a.kept + bh * a.keep;
  const int n_pages = (a.keep + (1 << a.bs_log2) - 1) >> a.bs_log2;
  int32_t *const pages = MOVE ? nullptr : a.pages + bh * (1 + n_pages);
  if (ctx <= a.keep) {  // nothing to cut
    for (int j = tid; j < a.keep; j += kEvictThreads) kept[j] = j < ctx ? j : -1;
    if (MOVE == 0 && tid == 0) pages[0] = 0;
    return;
  }
  const int front = a.keep - a.recent, back = ctx - a.recent;
  evict_clear(s.hist, 2 * kCopies * kBins);
  evict_clear(s_page, kPages / 4);
  __syncthreads();

  // The want-th largest of the middle: `threshold`, of whose equals the first `want`
  // stay.  None wanted: nothing is above this, and none of its equals stays.
  uint32_t want = (uint32_t)(front - a.sinks), threshold = 0xffffffffu;
  if (want > 0) {
    uint32_t known = 0;
    threshold = 0;
    unrolled<3>([&](auto n) __attribute__((always_inline)) {
      constexpr int pass = decltype(n)::value;
      constexpr int bits = pass_bits(pass);
      uint32_t(*const hist)[1 << bits] = reinterpret_cast<uint32_t(*)[1 << bits]>(
          &s.hist[pass % 2][0][0]);
      keys.count(hist[wave % kCopies], pass, known, threshold, 0, a.sinks, back);
      __syncthreads();
      uint32_t n0, n1;
      evict_bins<bits>(hist, n0, n1);
      const EvictBin at = evict_find(n0, n1, bits, want, s_find[pass]);
      threshold |= at.bin << pass_shift(pass);
      known |= ((1u << bits) - 1) << pass_shift(pass);
      want -= at.above;
    });
  }

  // The slots in order: the kept ones below `front` stay, the others are holes; the
  // kept ones behind fill them.  Counts of larger and (high half) equal weights.
  auto put = [&](int slot, int old) {
    kept[slot] = old;
    if (MOVE) src[slot] = (uint16_t)old;
  };
  for (int j = tid; j < a.sinks; j += kEvictThreads) put(j, j);
  for (int j = tid; j < a.recent; j += kEvictThreads) put(front + j, back + j);
  uint32_t count[N], incl[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    count[n] = 0;
#pragma unroll
    for (int i = 4 * n; i < 4 * n + 4; ++i) {
      const int j = keys.slot(0, i);
      if (j >= a.sinks && j < back)
        count[n] += keys.key[i] > threshold ? 1u : keys.key[i] == threshold ? 0x10000u : 0u;
    }
    incl[n] = wave_incl_scan_u32(count[n]);
    if ((tid & 63) == 63) s_step[n][wave] = incl[n];
  }
  __syncthreads();
  // Kept ones before each of the thread's slots, and below front.
  uint32_t above = 0, equal = 0, rank[4 * N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t gt = above, eq = equal;
#pragma unroll
    for (int v = 0; v < kEvictWaves; ++v) {
      const uint32_t x = s_step[n][v];
      gt += v < wave ? x & 0xffffu : 0u;
      eq += v < wave ? x >> 16 : 0u;
      above += x & 0xffffu;
      equal += x >> 16;
    }
    gt += (incl[n] - count[n]) & 0xffffu;
    eq += (incl[n] - count[n]) >> 16;
#pragma unroll
    for (int i = 4 * n; i < 4 * n + 4; ++i) {
      const int j = keys.slot(0, i);
      const bool in = j >= a.sinks && j < back, larger = in && keys.key[i] > threshold;
      const bool same = in && keys.key[i] == threshold;
      rank[i] = gt + min(eq, want);
      const bool keep = larger || (same && eq < want);
      if (j == front) s_stay = rank[i];  // the next slot after those that may stay
      if (in && j < front) {
        if (keep) {
          put(j, j);
        } else {
          holes[(uint32_t)(j - a.sinks) - rank[i]] = (uint16_t)j;
          s_page[j >> a.bs_log2] = 1;
        }
      }
      if (!keep || j < front) rank[i] = 0xffffffffu;
      gt += larger ? 1u : 0u;
      eq += same ? 1u : 0u;
    }
  }
  __syncthreads();
  const uint32_t stay = s_stay;
#pragma unroll
  for (int i = 0; i < 4 * N; ++i)
    if (rank[i] != 0xffffffffu) put(holes[rank[i] - stay], keys.slot(0, i));

  // Pages with arrivals: those of holes, and from front on all.
  const int window = front >> a.bs_log2;  // its first page
  __shared__ uint16_t s_list[MOVE ? kPages : 1];
  int listed = 0;
  for (int p0 = 0, turn = 0; p0 < n_pages; p0 += kEvictThreads, turn ^= 1) {
    const int p = p0 + tid;
    const bool any = p < n_pages && (MOVE ? p < window && s_page[p]
                                          : s_page[p] || (a.recent > 0 && p >= window));
    const EvictScan sum = evict_scan(any ? 1u : 0u, s_sum[turn]);
    if (any && MOVE) s_list[listed + sum.before] = (uint16_t)p;
    if (any && !MOVE) pages[1 + listed + sum.before] = p;
    listed += (int)sum.all;
  }
  if constexpr (MOVE == 0) {
    if (tid == 0) pages[0] = listed;
  } else {
    constexpr bool F8 = MOVE == 2;
    __syncthreads();
    const int h = (int)(bh % a.H_kv), lane = tid & 63, bs = 1 << a.bs_log2;
    const int at_once = 64 >> a.bs_log2;  // pages of a wave, of 64 slots at most
    const int mine = lane >> a.bs_log2, row0 = lane & (bs - 1);
    auto look = [&](bool there, int page) __attribute__((always_inline)) {
      EvictPage p = {page << a.bs_log2, 0, -1};
      if (there) {
        p.count = min(bs, a.keep - p.slot0);
        p.blk = evict_block(a, b, p.slot0);
      }
      const int slot = p.slot0 + row0;
      p.src[0] = row0 < p.count ? src[slot] : slot;
      p.from[0] = p.src[0] != slot ? evict_block(a, b, p.src[0]) : p.blk;
      p.src[1] = slot + 64;
      p.from[1] = -1;
      p.shift[0][0] = p.shift[1][0] = p.shift[0][1] = p.shift[1][1] = 0;
      return p;
    };
    // Those before the window's are no sources.
    for (int i = wave * at_once; i < listed; i += kEvictWaves * at_once) {
      const bool there = i + mine < listed;
      EvictPage p = look(there, s_list[there ? i + mine : 0]);
      const int slot = p.slot0 + row0;
      if (p.src[0] != slot) w[slot] = w[p.src[0]];
      if constexpr (F8) {
        evict_scales(a, h, row0, nullptr, nullptr, p);
        evict_put_scales(a, h, row0, p);
      }
      evict_move_rows<F8, false>(a, h, row0, p, nullptr, front);
    }
    __syncthreads();
    // The window's, in rounds, each read before it is written.  What a round reads lies
    // at the slots that it writes or behind them, so rounds before have not written it.
    const int per = min(at_once, max(1, (n_pages - window + kEvictWaves - 1) / kEvictWaves));
    const int per_row = a.row_bytes / 16, rows = 64 / per_row;  // lanes of a row, rows at once
    const int part = lane % per_row * 16, sub = lane / per_row;
    constexpr int kSteps = 16;  // rows of 256 bytes at most
    for (int q0 = window; q0 < n_pages; q0 += kEvictWaves * per) {
      const int page = q0 + wave * per + mine;
      EvictPage p = look(mine < per && page < n_pages, page);
      const int slot = p.slot0 + row0;
      const bool moves = p.src[0] != slot;
      const float weight = moves ? w[p.src[0]] : 0.f;
      if constexpr (F8) evict_scales(a, h, row0, nullptr, nullptr, p);
      const int write = evict_writes(p, row0, 0) ? 1 : 0;
      const int64_t at = evict_row(a, p.from[0], p.src[0], h), to = evict_row(a, p.blk, slot, h);
      const int slots = per << a.bs_log2;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        char *const cache = kv ? a.v_cache : a.k_cache;
        uint4 v[kSteps];
        unrolled<kSteps>([&](auto step) __attribute__((always_inline)) {
          constexpr int n = decltype(step)::value;
          v[n] = make_uint4(0, 0, 0, 0);
          if (n * rows >= slots) return;
          const int of = n * rows + sub;
          const int64_t row = shfl_i64(at, of);
          if (__shfl(write, of, 64))
            v[n] = *reinterpret_cast<const uint4 *>(cache + row * a.row_bytes + part);
        });
        __syncthreads();
        if (kv == 0) {
          if (moves) w[slot] = weight;
          if constexpr (F8) evict_put_scales(a, h, row0, p);
        }
        unrolled<kSteps>([&](auto step) __attribute__((always_inline)) {
          constexpr int n = decltype(step)::value;
          if (n * rows >= slots) return;
          const int of = n * rows + sub;
          const int64_t row = shfl_i64(to, of);
          const int by = F8 ? __shfl(p.shift[kv][0], of, 64) : 0;
          if (!__shfl(write, of, 64)) return;
          if (F8 && by != 0) v[n] = shifted_8_bits(v[n], by);
          *reinterpret_cast<uint4 *>(cache + row * a.row_bytes + part) = v[n];
        });
      }
    }
  }
}

// Long rows: the bins that pass `pass` chooses from the histograms of all chunks.
__device__ __forceinline__ EvictBin evict_choose(const EvictArgs &a, int64_t bh, int pass,
                                                 int chunks, uint32_t want, EvictFind &f) {
  const int top = (1 << pass_bits(pass)) - 1 - 2 * (int)threadIdx.x;
  uint32_t n0 = 0, n1 = 0;
  if (top > 0) {
    const uint16_t *const h = a.hist + (bh * 3 + pass) * (int64_t)a.chunks * kBins + top - 1;
    for (int c0 = 0; c0 < chunks; c0 += 16) {
      uint32_t two[16];
#pragma unroll
      for (int c = 0; c < 16; ++c)
        two[c] = *reinterpret_cast<const uint32_t *>(h + (int64_t)min(c0 + c, chunks - 1) * kBins);
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        if (c0 + c >= chunks) two[c] = 0;
        n0 += two[c] >> 16;
        n1 += two[c] & 0xffffu;
      }
    }
  }
  return evict_find(n0, n1, pass_bits(pass), want, f);
}

// A chunk's histogram of the bits of a pass, of the weights in the bins chosen before.
template <int PASS>
__global__ __launch_bounds__(kEvictThreads) void evict_count_kernel(const EvictArgs a) {
  if (PASS == 0 && (int)blockIdx.x >= a.select_wgs) {
    evict_copy_aside(a);
    return;
  }
  constexpr int kBits = pass_bits(PASS);
  __shared__ __align__(16) uint32_t s_hist[kCopies][1 << kBits];
  __shared__ EvictFind s_find;
  __shared__ uint32_t s_sum[kEvictWaves];
  const int64_t bh = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x % a.chunks), first = chunk * kChunk;
  const int ctx = evict_context(a, (int)(bh / a.H_kv));
  const int front = a.keep - a.recent, back = ctx - a.recent;
  if (ctx <= a.keep || first >= back || front == a.sinks) return;
  EvictKeys<2> keys;
  keys.load(a.weights + bh * a.S, first, a.sinks, back);
  evict_clear(s_hist, kCopies << kBits);
  uint32_t prefix = 0, known = 0;
  if constexpr (PASS > 0) {
    uint32_t *const state = a.state + bh * 4;
    uint32_t want = (uint32_t)(front - a.sinks);
    if constexpr (PASS == 2) {
      prefix = state[0] << pass_shift(0);
      known = ((1u << pass_bits(0)) - 1) << pass_shift(0);
      want = state[1];
    }
    const EvictBin at =
        evict_choose(a, bh, PASS - 1, (back + kChunk - 1) / kChunk, want, s_find);
    if (chunk == 0 && threadIdx.x == 0) {
      state[2 * PASS - 2] = at.bin;
      state[2 * PASS - 1] = want - at.above;
    }
    // The chunk's weights above that bin, of those in the bins before.
    const uint32_t mask = (1u << pass_bits(PASS - 1)) - 1;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = keys.slot(first, i);
      if (j >= a.sinks && j < back && (keys.key[i] & known) == prefix &&
          (keys.key[i] >> pass_shift(PASS - 1) & mask) > at.bin)
        ++n;
    }
    const uint32_t all = evict_scan(n, s_sum).all;
    uint32_t *const above = a.above + bh * a.chunks + chunk;
    if (threadIdx.x == 0) *above = PASS == 1 ? all : *above + all;
    prefix |= at.bin << pass_shift(PASS - 1);
    known |= mask << pass_shift(PASS - 1);
  }
  if (PASS == 0) __syncthreads();  // later ones have waited in the search
  keys.count(s_hist[(threadIdx.x >> 6) % kCopies], PASS, known, prefix, first, a.sinks, back);
  __syncthreads();
  uint32_t n0, n1;
  evict_bins<kBits>(s_hist, n0, n1);
  const int top = (1 << kBits) - 1 - 2 * (int)threadIdx.x;
  if (top > 0)  // of at most 8192 slots: 16 bits
    *reinterpret_cast<uint32_t *>(
        a.hist + ((bh * 3 + PASS) * (int64_t)a.chunks + chunk) * kBins + top - 1) = n0 << 16 | n1;
}

// A chunk's slots in order: where the kept ones are, holes and what fills them.  A
// hole n is -2 - n in kept.
__global__ __launch_bounds__(kEvictThreads) void evict_walk_kernel(const EvictArgs a) {
  __shared__ EvictFind s_find;
  __shared__ uint32_t s_sum[2][kEvictWaves], s_before[2][kEvictWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t bh = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x % a.chunks), first = chunk * kChunk;
  const int ctx = evict_context(a, (int)(bh / a.H_kv));
  const int front = a.keep - a.recent, back = ctx - a.recent;
  if (ctx <= a.keep || first >= back) return;
  EvictKeys<2> keys;
  keys.load(a.weights + bh * a.S, first, a.sinks, back);
  const uint32_t m = (uint32_t)(front - a.sinks);  // kept ones of the middle
  uint32_t threshold = 0xffffffffu, want = 0;
  uint32_t gt = 0, eq = 0;  // larger and equal ones in the chunks before
  if (m > 0) {
    const uint32_t *const state = a.state + bh * 4;
    want = state[3];
    const EvictBin at = evict_choose(a, bh, 2, (back + kChunk - 1) / kChunk, want, s_find);
    want -= at.above;
    threshold = state[0] << pass_shift(0) | state[2] << pass_shift(1) | at.bin;
    for (int c = wave; c < chunk; c += kEvictWaves) {
      const uint16_t *const h = a.hist + ((bh * 3 + 2) * (int64_t)a.chunks + c) * kBins;
      static_assert(1 << pass_bits(2) == 16 * kWave, "16 bins of a lane");
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int bin = (i * kWave + lane) * 8;
        const uint4 v = *reinterpret_cast<const uint4 *>(h + bin);
        const uint32_t two[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t n = two[k / 2] >> (k % 2 * 16) & 0xffffu;
          gt += (uint32_t)(bin + k) > at.bin ? n : 0u;
          eq += (uint32_t)(bin + k) == at.bin ? n : 0u;
        }
      }
      if (lane == 0) gt += a.above[bh * a.chunks + c];
    }
    gt = wave_sum_u32(gt);
    eq = wave_sum_u32(eq);
    if (lane == 0) {
      s_before[0][wave] = gt;
      s_before[1][wave] = eq;
    }
    __syncthreads();
    gt = eq = 0;
    for (int v = 0; v < kEvictWaves; ++v) {
      gt += s_before[0][v];
      eq += s_before[1][v];
    }
  }
  int32_t *const kept = a.kept + bh * a.keep, *const tails = a.tails + bh * a.keep;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    uint32_t count = 0;
#pragma unroll
    for (int i = 4 * n; i < 4 * n + 4; ++i) {
      const int j = keys.slot(first, i);
      if (j >= a.sinks && j < back)
        count += keys.key[i] > threshold ? 1u : keys.key[i] == threshold ? 0x10000u : 0u;
    }
    const EvictScan s = evict_scan(count, s_sum[n]);
    uint32_t g = gt + (s.before & 0xffffu), e = eq + (s.before >> 16);
#pragma unroll
    for (int i = 4 * n; i < 4 * n + 4; ++i) {
      const int j = keys.slot(first, i);
      if (j < a.sinks || j >= back) continue;
      const bool larger = keys.key[i] > threshold, same = keys.key[i] == threshold;
      const uint32_t rank = g + min(e, want);
      const bool keep = larger || (same && e < want);
      if (j == front) a.n_holes[bh] = (int32_t)(m - rank);
      if (j < front) {
        kept[j] = keep ? j : -2 - (int32_t)((uint32_t)(j - a.sinks) - rank);
      } else if (keep) {
        tails[m - 1 - rank] = j;
      }
      g += larger ? 1u : 0u;
      e += same ? 1u : 0u;
    }
    gt += s.all & 0xffffu;
    eq += s.all >> 16;
  }
}

// Rows of pages' arrivals and their weights, and in 8 bits the pages' scales and their
// other rows.  A wave for as many pages as have 64 slots together (one of 128): what
// leads to a row is four loads, each with what the last one brought (256 rows of 4096
// kept ones of 16 a page, 64 cut: 8 us where each page has a wave 15; 256 recent ones
// besides, 33 MB: 17 and 21).
template <bool F8, bool LONG>
__global__ __launch_bounds__(256) void evict_move_kernel(const EvictArgs a, int wgs_each) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Heads vary fastest: they move the same tokens often, whose rows lie side by side.
  const int h = (int)(blockIdx.x % a.H_kv), wg = (int)(blockIdx.x / a.H_kv % wgs_each);
  const int b = (int)(blockIdx.x / a.H_kv / wgs_each);
  const int64_t bh = (int64_t)b * a.H_kv + h;
  const int bs = 1 << a.bs_log2, n_pages = (a.keep + bs - 1) >> a.bs_log2;
  const int ctx = LONG ? evict_context(a, b) : 0, front = a.keep - a.recent;
  int32_t *const kept = a.kept + bh * a.keep;
  float *const w = a.weights + bh * a.S;
  const int32_t *const pages = LONG ? nullptr : a.pages + bh * (1 + n_pages);
  const int listed = LONG ? n_pages : pages[0];
  const char *const aside = a.aside + bh * 2 * a.recent * (int64_t)a.row_bytes;
  const int at_once = max(1, 64 >> a.bs_log2);  // pages
  const int mine = bs < 64 ? lane >> a.bs_log2 : 0, row0 = lane & (bs - 1);
  int i = (wg * 4 + wave) * at_once;
  const int step = wgs_each * 4 * at_once;
  // Looked up before it is known whether there is one: one wait for both.
  int next = LONG ? 0 : pages[1 + min(i + mine, n_pages - 1)];
  for (; i < listed; i += step) {
    const bool there = i + mine < listed;
    const int page = LONG ? i + mine : next, slot0 = page << a.bs_log2;
    if (!LONG) next = pages[1 + min(i + step + mine, n_pages - 1)];
    const int count = there ? min(bs, a.keep - slot0) : 0;
    const int blk = !there || (LONG && ctx <= a.keep) ? -1 : evict_block(a, b, slot0);
    // The lane's slots.
    EvictPage p = {slot0, count, blk};
    bool any = false;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int r = row0 + 64 * n, slot = slot0 + r;
      p.src[n] = slot;
      p.from[n] = blk;
      p.shift[0][n] = p.shift[1][n] = 0;
      if (r >= count) continue;
      if constexpr (LONG) {
        if (ctx <= a.keep) {
          kept[slot] = slot < ctx ? slot : -1;
          continue;
        }
        if (slot >= front) {
          p.src[n] = slot + ctx - a.keep;
        } else if (slot >= a.sinks) {
          const int at = kept[slot];
          p.src[n] = at >= 0 ? at : (a.tails + bh * a.keep)[a.n_holes[bh] - 1 - (-2 - at)];
        }
        if (slot < a.sinks || p.src[n] != slot) kept[slot] = p.src[n];
      } else {
        p.src[n] = kept[slot];
      }
      if (p.src[n] == slot) continue;
      any = true;
      p.from[n] = evict_block(a, b, p.src[n]);
      w[slot] = p.src[n] < a.keep ? a.aside_weights[bh * a.recent + p.src[n] - front] : w[p.src[n]];
    }
    if (__ballot(any && blk >= 0) == 0) continue;
    if constexpr (F8) {
      const uint8_t *const were = a.aside_scales + bh * 2 * a.aside_pages - (front >> a.bs_log2);
      evict_scales(a, h, row0, were, were + a.aside_pages, p);
      evict_put_scales(a, h, row0, p);
    }
    evict_move_rows<F8, true>(a, h, row0, p, aside, front);
  }
}

struct EvictPlan {
  bool long_rows, one_launch;
  int chunks, aside_pages;
  size_t aside, aside_weights, aside_scales, pages, hist, above, state, tails, n_holes;
  size_t bytes;
};

// keys: of a row of the tables.
static EvictPlan plan_evict(int64_t bh, int row_bytes, int bs, int64_t keys, int keep, int recent,
                            bool f8) {
  EvictPlan p = {};
  auto take = [&](size_t n) {
    const size_t at = p.bytes;
    p.bytes += (n + 255) / 256 * 256;
    return at;
  };
  // Tables that hold no more than is kept: nothing to cut or to move, and the plan
  // kernel alone says so.
  if (keep >= keys) {
    p.one_launch = true;
    return p;
  }
  p.long_rows = keys > kShortRow;
  // One launch where a workgroup for each sequence and head is one for each compute
  // unit, or has little to move (rows at most, of keys): 256 of them, 4160 tokens to
  // 4096, 8 bits, 22.9 us for 36.4, 128 20.9 for 27.3, 64 19.7 for 23.8, 8 19.0 for
  // 18.0; 16384 to 8192, 256 of them 96 for 133, 128 73 for 63, 16 51 for 30.
  const int64_t moved = recent + std::min<int64_t>(keep, std::max<int64_t>(0, keys - keep));
  p.one_launch = !p.long_rows && row_bytes <= 256 && bs <= 64 &&
                 (bh >= 256 || moved * row_bytes <= 1024 * bh);
  if (p.one_launch) return p;
  p.chunks = (int)((keys + kChunk - 1) / kChunk);
  p.aside_pages = std::max(0, (keep - 1) / bs - (keep - recent) / bs + 1);
  p.aside = take((size_t)bh * 2 * recent * row_bytes);
  p.aside_weights = take((size_t)bh * recent * 4);
  p.aside_scales = take(f8 ? (size_t)bh * 2 * p.aside_pages : 0);
  if (p.long_rows) {
    p.hist = take((size_t)bh * 3 * p.chunks * kBins * 2);
    p.above = take((size_t)bh * p.chunks * 4);
    p.state = take((size_t)bh * 16);
    p.tails = take((size_t)bh * keep * 4);
    p.n_holes = take((size_t)bh * 4);
  } else {
    p.pages = take((size_t)bh * (1 + (keep + bs - 1) / bs) * 4);
  }
  return p;
}

static bool evict_sizes_ok(int32_t B, int32_t H_kv, int32_t D, int32_t block_size, int32_t keep,
                           int32_t sinks, int32_t recent) {
  return B > 0 && H_kv > 0 && (int64_t)B * H_kv < (1 << 24) && head_dim_supported(D) &&
         block_size_supported(block_size) && keep > 0 && keep <= (1 << 26) && sinks >= 0 &&
         recent >= 0 && (int64_t)sinks + recent <= keep;
}

}  // namespace cvsa

using namespace cvsa;

extern "C" size_t cvsa_evict_tokens_workspace_bytes(int32_t B, int32_t H_kv, int32_t D,
                                                    int32_t block_size, int32_t W,
                                                    int32_t cache_bits, int32_t keep,
                                                    int32_t sinks, int32_t recent) {
  if (!evict_sizes_ok(B, H_kv, D, block_size, keep, sinks, recent) || W <= 0 ||
      W > kMaxPagesWide || (cache_bits != 8 && cache_bits != 16))
    return 0;
  return plan_evict((int64_t)B * H_kv, D * cache_bits / 8, block_size, (int64_t)W * block_size,
                    keep, recent, cache_bits == 8)
      .bytes;
}

extern "C" int cvsa_evict_tokens(float *weights, int64_t S, void *k_cache, void *v_cache,
                                 uint8_t *k_scales, uint8_t *v_scales, int64_t num_blocks,
                                 const int32_t *block_tables, int64_t bt_stride_b, int32_t W,
                                 const int32_t *context_lens, int32_t B, int32_t H_kv, int32_t D,
                                 int32_t block_size, int32_t keep, int32_t sinks, int32_t recent,
                                 int32_t *kept, void *workspace, size_t workspace_bytes,
                                 void *stream) {
  CVSA_REQUIRE(weights && k_cache && v_cache && block_tables && context_lens && kept,
               CVSA_ERR_INVALID, "evict_tokens: null pointer argument");
  CVSA_REQUIRE(!k_scales == !v_scales, CVSA_ERR_INVALID,
               "evict_tokens: scales of keys and values, or of neither");
  CVSA_REQUIRE(head_dim_supported(D), CVSA_ERR_UNSUPPORTED,
               "evict_tokens: D=%d not in {32, 64, 128, 256}", D);
  CVSA_REQUIRE(block_size_supported(block_size), CVSA_ERR_UNSUPPORTED,
               "evict_tokens: block_size=%d not in {8, 16, 32, 64, 128}", block_size);
  CVSA_REQUIRE(W > 0 && W <= kMaxPagesWide, CVSA_ERR_UNSUPPORTED,
               "evict_tokens: W=%d not supported (at most %d)", W, kMaxPagesWide);
  CVSA_REQUIRE(evict_sizes_ok(B, H_kv, D, block_size, keep, sinks, recent) && num_blocks > 0 &&
                   bt_stride_b >= W,
               CVSA_ERR_INVALID, "evict_tokens: bad sizes B=%d H_kv=%d keep=%d sinks=%d recent=%d",
               B, H_kv, keep, sinks, recent);
  CVSA_REQUIRE(S >= (int64_t)W * block_size, CVSA_ERR_INVALID,
               "evict_tokens: weights of %lld keys for tables of %lld", (long long)S,
               (long long)W * block_size);
  CVSA_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0, CVSA_ERR_INVALID,
               "evict_tokens: caches must be 16-byte aligned");
  CVSA_REQUIRE(k_cache != v_cache && (!k_scales || k_scales != v_scales), CVSA_ERR_INVALID,
               "evict_tokens: keys and values must have caches and scales of their own");
  const int64_t bh = (int64_t)B * H_kv;
  const int row_bytes = D * (k_scales ? 1 : 2);
  const int64_t keys = (int64_t)W * block_size;
  const EvictPlan p = plan_evict(bh, row_bytes, block_size, keys, keep, recent,
                                 k_scales != nullptr);
  CVSA_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes &&
                                ((uintptr_t)workspace & 255) == 0),
               CVSA_ERR_WORKSPACE,
               "evict_tokens: needs a 256-byte aligned workspace of %zu bytes", p.bytes);
  const int64_t aside = p.one_launch ? 0
                                     : bh * recent * (row_bytes / 16) +
                                           (k_scales ? bh * p.aside_pages : 0);
  const int64_t aside_wgs = (aside + kEvictThreads - 1) / kEvictThreads;
  const int64_t select_wgs = p.long_rows ? bh * p.chunks : bh;
  CVSA_REQUIRE(aside_wgs + select_wgs < (1LL << 32) / kEvictThreads, CVSA_ERR_UNSUPPORTED,
               "evict_tokens: too many sequences, heads or recent tokens");
  EvictArgs a = {};
  a.weights = weights; a.S = S;
  a.k_cache = (char *)k_cache; a.v_cache = (char *)v_cache;
  a.k_scales = k_scales; a.v_scales = v_scales;
  a.num_blocks = num_blocks;
  a.block_tables = block_tables; a.bt_sb = bt_stride_b; a.W = W;
  a.bs_log2 = __builtin_ctz(block_size);
  a.context_lens = context_lens;
  a.B = B; a.H_kv = H_kv; a.row_bytes = row_bytes;
  a.keep = keep; a.sinks = sinks; a.recent = recent;
  a.kept = kept;
  char *const ws = (char *)workspace;
  a.aside = ws + p.aside;
  a.aside_weights = (float *)(ws + p.aside_weights);
  a.aside_scales = (uint8_t *)(ws + p.aside_scales);
  a.aside_pages = p.aside_pages;
  a.pages = (int32_t *)(ws + p.pages);
  a.chunks = p.chunks;
  a.hist = (uint16_t *)(ws + p.hist);
  a.above = (uint32_t *)(ws + p.above);
  a.state = (uint32_t *)(ws + p.state);
  a.tails = (int32_t *)(ws + p.tails);
  a.n_holes = (int32_t *)(ws + p.n_holes);
  a.select_wgs = (int)select_wgs;
  const hipStream_t s = (hipStream_t)stream;
  const dim3 select((unsigned)select_wgs), first((unsigned)(select_wgs + aside_wgs));
  const dim3 threads(kEvictThreads);
  if (p.long_rows) {
    hipLaunchKernelGGL(evict_count_kernel<0>, first, threads, 0, s, a);
    hipLaunchKernelGGL(evict_count_kernel<1>, select, threads, 0, s, a);
    hipLaunchKernelGGL(evict_count_kernel<2>, select, threads, 0, s, a);
    hipLaunchKernelGGL(evict_walk_kernel, select, threads, 0, s, a);
  } else {
    auto plan = [&](auto move) {
      constexpr int MOVE = decltype(move)::value;
      if (keys <= 4 * kEvictThreads)
        hipLaunchKernelGGL((evict_plan_kernel<1, MOVE>), first, threads, 0, s, a);
      else if (keys <= 8 * kEvictThreads)
        hipLaunchKernelGGL((evict_plan_kernel<2, MOVE>), first, threads, 0, s, a);
      else
        hipLaunchKernelGGL((evict_plan_kernel<4, MOVE>), first, threads, 0, s, a);
    };
    if (!p.one_launch) {
      plan(std::integral_constant<int, 0>());
    } else {
      k_scales ? plan(std::integral_constant<int, 2>()) : plan(std::integral_constant<int, 1>());
      return cvsa_host::check_launch("evict_tokens");
    }
  }
  // Four waves in a workgroup, in turn past 8192 workgroups.
  const int64_t n_pages = (keep + block_size - 1) / block_size;
  const int64_t wave_pages = std::max(1, 64 / block_size);
  const int each = (int)std::max<int64_t>(
      1, std::min((n_pages + 4 * wave_pages - 1) / (4 * wave_pages), 8192 / bh));
  const dim3 grid((unsigned)(bh * each));
  auto move = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, each); };
  if (p.long_rows) k_scales ? move(evict_move_kernel<true, true>) : move(evict_move_kernel<false, true>);
  else k_scales ? move(evict_move_kernel<true, false>) : move(evict_move_kernel<false, false>);
  return cvsa_host::check_launch("evict_tokens");
}
