// Attention of a chunk of new tokens over the paged cache: the join of split
// keys, the launch plan and the entry points.  Sequences that bring few rows
// (chunk_stream.h) and many (chunk_prefill.h) get a launch each.
#include "chunk_launch.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace cvsa {

constexpr int kJoinThreads = 256;

// The parts of a row joined in the order of the keys: of few rows (RANGES) those
// of the ranges that its sequence spans, of many rows its splits.  D / 4 threads
// have a float4 of the row each; with few rows `groups` such groups share a
// row's parts, and their sums are joined in LDS.
template <int D, bool RANGES>
__global__ __launch_bounds__(kJoinThreads) void chunk_join_kernel(const ChunkArgs a,
                                                                  const ChunkClass c,
                                                                  int groups) {
  constexpr int L = D / 4, NG = kJoinThreads / L;
  __shared__ float4 s_o[NG][L];
  __shared__ float2 s_ml[NG];
  const int group = threadIdx.x / L, d = threadIdx.x % L * 4;
  const int per_wg = NG / groups, mine = group % groups;
  const uint32_t rows = (uint32_t)c.tokens * a.H_q;  // below 2^31
  const uint32_t want = blockIdx.x * per_wg + group / groups;
  const uint32_t row = min(want, rows - 1);
  // The row's token in its class: its sequence and place in it.  The rows of a
  // workgroup may be of several tokens; each lane looks for its own, a wave's
  // lanes over the same sequences.
  const int class_tok = (int)(row / a.H_q), head = (int)(row % a.H_q);
  int tok = 0, first = 0, len = 0, ctx = 0;
  uint32_t unit0 = 0, units = 0, total = 0;  // of the sequence, of all
  const int lane = threadIdx.x & 63;
  int base = 0;  // tokens of the class before b0
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const ChunkSeq s = chunk_look(a, c, b0 + lane);
    const int end = base + (int)wave_incl_scan_u32((uint32_t)s.len);
    const int unit_end = (int)wave_incl_scan_u32((uint32_t)s.units);
    const int last = __builtin_amdgcn_readlane(end, 63);
    // the first sequence that ends past the token, by bisection over lanes
    int l = 0;
#pragma unroll
    for (int step = 32; step > 0; step >>= 1)
      if (__shfl(end, l + step - 1, 64) <= class_tok) l += step;
    l &= 63;
    const int n = __shfl(s.len, l, 64), u = __shfl(s.units, l, 64);
    const int before = __shfl(end, l, 64) - n, u0 = __shfl(unit_end, l, 64) - u;
    const int f = __shfl(s.first, l, 64), x = __shfl(s.ctx, l, 64);
    if (class_tok >= base && class_tok < last) {
      first = f;
      len = n;
      ctx = x;
      tok = class_tok - before;
      unit0 = total + u0;
      units = u;
    }
    base = last;
    total += __builtin_amdgcn_readlane(unit_end, 63);
  }
  int parts;
  int64_t part0, stride;  // the row's first part, from its second to the next
  int64_t second;
  if (RANGES) {
    const ChunkRanges ranges(c, total);
    const int r0 = ranges.of(unit0 + c.extra_units), r1 = ranges.of(unit0 + units - 1);
    const int h = head / a.G, place = tok * a.G + head % a.G;
    parts = r1 - r0 + 1;
    part0 = ((int64_t)(2 * r0 + 1) * a.H_kv + h) * c.tile_rows + place;
    second = part0 + (int64_t)a.H_kv * c.tile_rows;
    stride = (int64_t)2 * a.H_kv * c.tile_rows;
  } else {
    const int row0 = (tok * a.G + head % a.G) / c.tile_rows * c.tile_rows;
    const int keys = chunk_tile_keys(a, ctx - len, ctx, len * a.G, row0, c.tile_rows);
    parts = min((keys + c.split_len - 1) / c.split_len, c.splits);
    part0 = row;
    second = (int64_t)rows + row;
    stride = rows;
  }
  auto part = [&](int s) { return s == 0 ? part0 : second + (s - 1) * stride; };
  const bool whole = parts == 1;  // complete already
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float w, float sum, const float4 &v) {
    l = fmaf(sum, w, l);
    o.x = fmaf(v.x, w, o.x);
    o.y = fmaf(v.y, w, o.y);
    o.z = fmaf(v.z, w, o.z);
    o.w = fmaf(v.w, w, o.w);
  };
  // Four parts at a time, all of their loads under way at once.
  for (int s0 = mine; s0 < parts && !whole; s0 += 4 * groups) {
    float2 ml[4];
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + i * groups;
      const int64_t at = part(s < parts ? s : s0);
      ml[i] = c.part_ml[at];
      v[i] = *reinterpret_cast<const float4 *>(c.part_o + at * D + d);
    }
    float nm = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) nm = fmaxf(nm, ml[i].x);
    const float ref = nm == -INFINITY ? 0.f : nm, alpha = __builtin_amdgcn_exp2f(m - ref);
    m = nm;
    l *= alpha;
    o.x *= alpha;
    o.y *= alpha;
    o.z *= alpha;
    o.w *= alpha;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (s0 + i * groups < parts) add(__builtin_amdgcn_exp2f(ml[i].x - ref), ml[i].y, v[i]);
  }
  if (groups > 1) {  // the same in every thread
    s_o[group][d / 4] = o;
    if (d == 0) s_ml[group] = make_float2(m, l);
    __syncthreads();
    if (mine > 0) return;
    for (int g = 1; g < groups; ++g) m = fmaxf(m, s_ml[group + g].x);
    const float top = m == -INFINITY ? 0.f : m;
    const float2 own = s_ml[group];
    const float4 have = o;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    add(__builtin_amdgcn_exp2f(own.x - top), own.y, have);
    for (int g = 1; g < groups; ++g) {
      const float2 ml = s_ml[group + g];
      add(__builtin_amdgcn_exp2f(ml.x - top), ml.y, s_o[group + g][d / 4]);
    }
  }
  if (want >= rows || whole) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t at = (int64_t)(first + tok) * a.H_q + head;
  *reinterpret_cast<uint2 *>(a.out + at * D + d) =
      make_uint2(chunk_cvt_bf16x2(o.x * inv, o.y * inv), chunk_cvt_bf16x2(o.z * inv, o.w * inv));
  if (a.lse && d == 0)
    a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Groups of threads that share a row: as many as keep the GPU's CUs busy when
// rows are few (one row of 64 parts: 64 loads in a row by one group, or 8 by
// eight).
template <int D, bool RANGES>
static void launch_join(const ChunkArgs &a, const ChunkClass &c, hipStream_t s) {
  constexpr int NG = kJoinThreads / (D / 4);
  const int64_t rows = (int64_t)c.tokens * a.H_q;
  const int parts = RANGES ? c.splits / c.tiles + 1 : c.splits;  // of a row, about
  int groups = 1;
  while (groups < NG && groups * 2 <= parts && rows * groups < 1024 * NG) groups *= 2;
  const int per_wg = NG / groups;
  hipLaunchKernelGGL((chunk_join_kernel<D, RANGES>), dim3((unsigned)((rows + per_wg - 1) / per_wg)),
                     dim3(kJoinThreads), 0, s, a, c, groups);
}

struct ChunkPlan {
  ChunkClass few, many;  // tiles 0: no such sequence
  bool join_few, join_many;
  size_t bytes;  // of the workspace
};

// Splits of many rows' keys: the number with the shortest estimate of rounds of
// workgroups, joined (rounds of the longest at one rate for all head sizes took
// 380 us for 215: 10 prompts of up to 4792 tokens, 8 heads on 2 of 64; 2460 for
// 1767: 5 of 2127 after 22 K keys, 32 on 16 of 32).  chunk: tokens of a chunk
// (its tiles' mean), whose tiles are taken to see from max_keys - chunk to
// max_keys keys.
template <int D>
static int plan_splits(const ChunkClass &c, int H_q, int H_kv, int64_t max_keys, double chunk) {
  // us for 64 keys of a tile on a full CU; workgroups that fill one (two of eight
  // waves fit at D = 64, but one alone is as fast), of which a single one has less
  // than its share of the time.
  const double step = D == 32 ? 0.52 : D == 256 ? 2.8 : D == 128 ? 1.45
                              : c.tile_rows == 256 ? 1.15 : 0.6;
  const int fit = D == 32 ? 3 : c.tile_rows == 128 && D == 64 ? 2 : 1;
  const double hi = (double)max_keys, lo = std::max(hi - chunk, 0.), mean = (lo + hi) / 2;
  const double items = (double)c.tiles * H_kv;
  double best = 1e30;
  int splits = 1;
  // 1 to 8, as many as fill one to four rounds, and the most: 256 keys each.
  const double most = std::max(1., std::min(64., std::floor(hi / 256)));
  for (int i = 1; i <= 14; ++i) {
    const double want = i <= 8 ? i : i <= 12 ? (i - 8) * 256 * fit / items : most / (i - 12);
    const int n = (int)std::max(1., std::min(most, want));
    const double len = hi / n;
    // Mean of ceil(keys / len) from lo to hi.
    auto area = [&](double x) {
      const double q = std::floor(x / len);
      return len * q * (q + 1) / 2 + (q + 1) * (x - q * len);
    };
    const double parts = n == 1 || hi - lo < 1 ? n : (area(hi) - area(lo)) / (hi - lo);
    const double wgs = items * parts;
    const double share = std::min<double>(fit, std::max((fit + 2) / 3., wgs / 256));
    // 8 us for a workgroup's start and end, 12 if it writes a part.  Alike ones
    // take whole rounds; of different ones the long start first and the short
    // fill up.
    const double ends = n == 1 ? 8 : 12, wg = mean / 64 * step * share / parts + ends;
    const double rounds = wgs / (256 * fit), whole = std::ceil(rounds - 1e-6);
    double us = std::max(len / 64 * step * share + ends,
                         wg * (whole - (whole - rounds) * (hi - lo) / hi));
    // The rows in several parts are written and read once more, at 3 TB/s.
    if (n > 1)
      us += 8 + std::min(parts, 2 * (parts - 1)) * c.tokens * H_q * D * 8 / 3e6;
    if (us < best * (splits == 1 ? 0.95 : 1)) {
      best = us;
      splits = n;
    }
  }
  return splits;
}

template <int D, bool F8>
static ChunkPlan plan_chunk(const int32_t *cu, int B, int H_q, int H_kv, int64_t max_keys) {
  const int G = H_q / H_kv;
  ChunkPlan p = {};
  p.few.min_rows = 1;
  p.few.max_rows = chunk_few_rows<D>();
  p.many.min_rows = p.few.max_rows + 1;
  p.many.max_rows = 0x7fffffff;
  int longest = 0;
  for (int b = 0; b < B; ++b) longest = std::max(longest, cu[b + 1] - cu[b]);
  // 4 or 8 waves: see the kernel.
  const bool start = max_keys <= 4096 && longest >= max_keys / 4;
  p.many.tile_rows = D == 128 || (D == 64 && !start) ? 256 : 128;
  int64_t most_few = 0;
  bool same = true;
  for (int b = 0; b < B; ++b) {
    const int64_t rows = (int64_t)(cu[b + 1] - cu[b]) * G;
    if (rows <= p.few.max_rows) most_few = std::max(most_few, rows);
    same = same && cu[b + 1] - cu[b] == cu[1];
  }
  p.few.tile_rows = most_few > 32 ? 64 : 32;
  p.few.same_len = p.many.same_len = same ? cu[1] : 0;
  p.many.only = -1;
  int sequences = 0;     // of many rows
  int64_t weighted = 0;  // tokens of a tile's chunk, over all tiles
  for (int b = 0; b < B; ++b) {
    const int n = cu[b + 1] - cu[b];
    ChunkClass &c = (int64_t)n * G <= p.few.max_rows ? p.few : p.many;
    c.tiles += (int)(((int64_t)n * G + c.tile_rows - 1) / c.tile_rows);
    c.tokens += n;
    if (&c != &p.many) continue;
    weighted += (int64_t)n * (((int64_t)n * G + c.tile_rows - 1) / c.tile_rows);
    if (++sequences == 1) {
      c.only = b;
      c.only_first = cu[b];
      c.only_len = n;
    }
  }
  if (sequences > 1) p.many.only = -1;
  // Few rows: a range for each workgroup that fits the GPU, of one unit at least;
  // up to 256 keys, a step or two of the waves, are not worth a join.
  constexpr int unit_log2 = chunk_stream_waves<D, F8>() == 2 ? 6 : 7;
  static_assert(chunk_stream_waves<D, F8>() * 32 == 1 << unit_log2, "a step of the waves");
  const bool whole = max_keys <= 256;
  p.few.unit_log2 = p.many.unit_log2 = whole ? 31 : unit_log2;
  // A sequence's start and end cost a workgroup about as much as 3 units of 128 keys of
  // 8 bits.  Counted so and not, 32 single tokens over up to 8 K keys, 32 heads on 8: at
  // D = 32 29.5 us and 33.3, 64 38.7 and 43.5, 128 68.5 and 73.8, 256 126 and 133; equal
  // sequences lose 1% (8 drafts of 5 tokens at 32 K keys, 28 heads on 4: 44 and 43, 55
  // and 54, 90 and 89, 210 and 209).
  p.few.extra_units = F8 && !whole ? 3 : 0;
  const int64_t units =
      (int64_t)p.few.tiles * (whole ? 1 : (max_keys + (1 << unit_log2) - 1) >> unit_log2);
  const int fit = most_few > 32 ? chunk_stream_fit<D, 2, F8>() : chunk_stream_fit<D, 1, F8>();
  p.few.splits = (int)std::max<int64_t>(1, std::min<int64_t>(256 * fit / H_kv, units));
  p.join_few = p.few.tiles > 0 && p.few.splits > 1 && !whole;
  int64_t splits = 1;
  if (p.many.tiles > 0)
    splits = plan_splits<D>(p.many, H_q, H_kv, max_keys, (double)weighted / p.many.tiles);
  p.many.split_len = (int)(((max_keys + splits - 1) / splits + 127) / 128 * 128);
  p.many.splits = (int)std::max<int64_t>(1, (max_keys + p.many.split_len - 1) / p.many.split_len);
  p.join_many = p.many.tiles > 0 && p.many.splits > 1;
  for (ChunkClass *c : {&p.few, &p.many}) {
    if (!(c == &p.few ? p.join_few : p.join_many)) continue;
    const size_t rows = c == &p.few ? (size_t)2 * c->splits * H_kv * c->tile_rows
                                    : (size_t)c->splits * c->tokens * H_q;
    c->part_ml = (float2 *)p.bytes;  // offsets until there is a workspace
    p.bytes += (rows * sizeof(float2) + 255) / 256 * 256;
    c->part_o = (float *)p.bytes;
    p.bytes += (rows * D * sizeof(float) + 255) / 256 * 256;
  }
  return p;
}

template <bool F8>
static ChunkPlan plan_chunk_d(const int32_t *cu, int B, int H_q, int H_kv, int D,
                              int64_t max_keys) {
  if (D == 32) return plan_chunk<32, F8>(cu, B, H_q, H_kv, max_keys);
  if (D == 64) return plan_chunk<64, F8>(cu, B, H_q, H_kv, max_keys);
  if (D == 128) return plan_chunk<128, F8>(cu, B, H_q, H_kv, max_keys);
  return plan_chunk<256, F8>(cu, B, H_q, H_kv, max_keys);
}

static int64_t chunk_grid(const ChunkClass &c, int H_kv) {
  return (int64_t)c.tiles * H_kv * c.splits;  // of many rows
}

template <int D>
static void launch_chunk(const ChunkArgs &a, const ChunkPlan &p, hipStream_t s) {
  const bool f8 = a.k_scales != nullptr;
  if (p.many.tiles > 0) {
    const unsigned grid = (unsigned)chunk_grid(p.many, a.H_kv);
    if (f8) launch_chunk_prefill<D, true>(a, p.many, grid, s);
    else launch_chunk_prefill<D, false>(a, p.many, grid, s);
    if (p.join_many) launch_join<D, false>(a, p.many, s);
  }
  if (p.few.tiles > 0) {
    if (f8) launch_chunk_stream<D, true>(a, p.few, s);
    else launch_chunk_stream<D, false>(a, p.few, s);
    if (p.join_few) launch_join<D, true>(a, p.few, s);
  }
}

static bool chunk_shape_ok(const int32_t *cu, int32_t B, int32_t H_q, int32_t H_kv, int32_t D,
                           int32_t block_size, int32_t W) {
  if (!cu || B <= 0 || B > (1 << 20) || H_kv <= 0 || H_q <= 0 || H_q % H_kv ||
      H_q / H_kv > 128 || H_q > 65536 || W <= 0 || W > kMaxPagesWide ||
      !head_dim_supported(D) || !block_size_supported(block_size) || cu[0] != 0)
    return false;
  for (int b = 0; b < B; ++b)
    if (cu[b + 1] < cu[b]) return false;
  return cu[B] <= (1 << 24) && (int64_t)cu[B] * (H_q / H_kv) < (1 << 30) &&
         (int64_t)cu[B] * H_q < (1LL << 31);
}

// Most keys of a sequence, as far as the host knows.  Contexts are on the device,
// so without the caller's bound the splits of many rows are cut for sequences that
// fill the table: in a table for 128 K keys, 32 heads on 8 of 128, 512 tokens at 4 K
// keys take 88 us and 100 at 8 K 159, with the bound 49 and 35.
static int64_t chunk_max_keys(int32_t W, int32_t block_size, int32_t max_context_len) {
  const int64_t all = (int64_t)W * block_size;
  return max_context_len > 0 ? std::min<int64_t>(all, max_context_len) : all;
}

}  // namespace cvsa

using namespace cvsa;

template <bool F8>
static size_t chunk_workspace_bytes(const int32_t *cu_host, int32_t B, int32_t H_q, int32_t H_kv,
                                    int32_t D, int32_t block_size, int32_t W,
                                    int32_t max_context_len) {
  if (!chunk_shape_ok(cu_host, B, H_q, H_kv, D, block_size, W) || cu_host[B] == 0) return 0;
  return plan_chunk_d<F8>(cu_host, B, H_q, H_kv, D,
                          chunk_max_keys(W, block_size, max_context_len))
      .bytes;
}

extern "C" size_t cvsa_chunk_attention_workspace_bytes(const int32_t *cu_host, int32_t B,
                                                       int32_t H_q, int32_t H_kv, int32_t D,
                                                       int32_t block_size, int32_t W,
                                                       int32_t max_context_len) {
  return chunk_workspace_bytes<false>(cu_host, B, H_q, H_kv, D, block_size, W, max_context_len);
}

extern "C" size_t cvsa_chunk_attention8_workspace_bytes(const int32_t *cu_host, int32_t B,
                                                        int32_t H_q, int32_t H_kv, int32_t D,
                                                        int32_t block_size, int32_t W,
                                                        int32_t max_context_len) {
  return chunk_workspace_bytes<true>(cu_host, B, H_q, H_kv, D, block_size, W, max_context_len);
}

// Over caches of bf16, or of 8 bits (with scales).
static int chunk_attention(const char *who, const uint16_t *q, int64_t q_stride_t,
                           int64_t q_stride_h, const void *k_cache, const void *v_cache,
                           const uint8_t *k_scales, const uint8_t *v_scales, int64_t num_blocks,
                           const int32_t *block_tables, int64_t bt_stride_b,
                           const int32_t *context_lens, const int32_t *cu_seqlens,
                           const int32_t *cu_host, int32_t B, int32_t H_q, int32_t H_kv, int32_t D,
                           int32_t block_size, int32_t W, int32_t max_context_len, float scale,
                           int32_t causal, uint16_t *out, float *lse, void *workspace,
                           size_t workspace_bytes, void *stream) {
  CVSA_REQUIRE(q && k_cache && v_cache && block_tables && context_lens && cu_seqlens && cu_host &&
                   out,
               CVSA_ERR_INVALID, "%s: null pointer argument", who);
  CVSA_REQUIRE(head_dim_supported(D), CVSA_ERR_UNSUPPORTED,
               "%s: D=%d not in {32, 64, 128, 256}", who, D);
  CVSA_REQUIRE(block_size_supported(block_size), CVSA_ERR_UNSUPPORTED,
               "%s: block_size=%d not in {8, 16, 32, 64, 128}", who, block_size);
  CVSA_REQUIRE(H_kv > 0 && H_q > 0 && H_q % H_kv == 0, CVSA_ERR_INVALID,
               "%s: head counts H_q=%d H_kv=%d", who, H_q, H_kv);
  CVSA_REQUIRE(H_q / H_kv <= 128 && W <= kMaxPagesWide, CVSA_ERR_UNSUPPORTED,
               "%s: G=%d (at most 128) or W=%d (at most %d) not supported", who,
               H_q / H_kv, W, kMaxPagesWide);
  CVSA_REQUIRE(chunk_shape_ok(cu_host, B, H_q, H_kv, D, block_size, W) && num_blocks > 0 &&
                   bt_stride_b >= W,
               CVSA_ERR_INVALID, "%s: bad sizes or chunk offsets (B=%d W=%d)", who, B, W);
  CVSA_REQUIRE((int64_t)block_size * H_kv * D < (1 << 30), CVSA_ERR_UNSUPPORTED,
               "%s: a block of %d tokens of %d heads is too large", who, block_size, H_kv);
  CVSA_REQUIRE(scale > 0.f && scale < INFINITY, CVSA_ERR_INVALID,
               "%s: scale must be positive and finite", who);
  CVSA_REQUIRE(max_context_len >= 0 && (causal == 0 || causal == 1), CVSA_ERR_INVALID,
               "%s: bad max_context_len=%d or causal=%d", who, max_context_len, causal);
  CVSA_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) ==
                       0 &&
                   q_stride_t % 8 == 0 && q_stride_h % 8 == 0,
               CVSA_ERR_INVALID, "%s: rows must be 16-byte aligned", who);
  const int32_t tokens = cu_host[B];
  if (tokens == 0) return CVSA_OK;
  const int64_t max_keys = chunk_max_keys(W, block_size, max_context_len);
  ChunkPlan p = k_scales ? plan_chunk_d<true>(cu_host, B, H_q, H_kv, D, max_keys)
                         : plan_chunk_d<false>(cu_host, B, H_q, H_kv, D, max_keys);
  CVSA_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes &&
                                ((uintptr_t)workspace & 255) == 0),
               CVSA_ERR_WORKSPACE,
               "%s: needs a 256-byte aligned workspace of %zu bytes", who, p.bytes);
  CVSA_REQUIRE(chunk_grid(p.many, H_kv) < (1LL << 31) &&
                   (int64_t)p.few.tiles * ((int64_t)W * block_size / 64 + 4) < (1LL << 31),
               CVSA_ERR_UNSUPPORTED, "%s: too many row tiles or keys", who);
  for (ChunkClass *c : {&p.few, &p.many}) {
    c->part_ml = (float2 *)((char *)workspace + (size_t)c->part_ml);
    c->part_o = (float *)((char *)workspace + (size_t)c->part_o);
  }
  ChunkArgs a = {};
  a.q = q; a.q_st = q_stride_t; a.q_sh = q_stride_h;
  a.k_cache = (const uint16_t *)k_cache; a.v_cache = (const uint16_t *)v_cache;
  a.k_scales = k_scales; a.v_scales = v_scales;
  a.num_blocks = (int)std::min<int64_t>(num_blocks, INT32_MAX);
  a.block_tables = block_tables; a.bt_sb = bt_stride_b; a.W = W;
  a.context_lens = context_lens; a.cu = cu_seqlens;
  a.B = B; a.H_q = H_q; a.H_kv = H_kv; a.G = H_q / H_kv;
  a.bs_log2 = __builtin_ctz(block_size);
  a.c = scale * 1.4426950408889634f;
  a.causal = causal;
  a.out = out; a.lse = lse;
  const hipStream_t s = (hipStream_t)stream;
  if (D == 32) launch_chunk<32>(a, p, s);
  else if (D == 64) launch_chunk<64>(a, p, s);
  else if (D == 128) launch_chunk<128>(a, p, s);
  else launch_chunk<256>(a, p, s);
  return cvsa_host::check_launch(who);
}

extern "C" int cvsa_chunk_attention(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h,
                                    const uint16_t *k_cache, const uint16_t *v_cache,
                                    int64_t num_blocks, const int32_t *block_tables,
                                    int64_t bt_stride_b, const int32_t *context_lens,
                                    const int32_t *cu_seqlens, const int32_t *cu_host, int32_t B,
                                    int32_t H_q, int32_t H_kv, int32_t D, int32_t block_size,
                                    int32_t W, int32_t max_context_len, float scale,
                                    int32_t causal, uint16_t *out, float *lse, void *workspace,
                                    size_t workspace_bytes, void *stream) {
  return chunk_attention("chunk_attention", q, q_stride_t, q_stride_h, k_cache, v_cache, nullptr,
                         nullptr, num_blocks, block_tables, bt_stride_b, context_lens, cu_seqlens,
                         cu_host, B, H_q, H_kv, D, block_size, W, max_context_len, scale, causal,
                         out, lse, workspace, workspace_bytes, stream);
}

extern "C" int cvsa_chunk_attention8(const uint16_t *q, int64_t q_stride_t, int64_t q_stride_h,
                                     const uint8_t *k_cache, const uint8_t *v_cache,
                                     const uint8_t *k_scales, const uint8_t *v_scales,
                                     int64_t num_blocks, const int32_t *block_tables,
                                     int64_t bt_stride_b, const int32_t *context_lens,
                                     const int32_t *cu_seqlens, const int32_t *cu_host, int32_t B,
                                     int32_t H_q, int32_t H_kv, int32_t D, int32_t block_size,
                                     int32_t W, int32_t max_context_len, float scale,
                                     int32_t causal, uint16_t *out, float *lse, void *workspace,
                                     size_t workspace_bytes, void *stream) {
  CVSA_REQUIRE(k_scales && v_scales, CVSA_ERR_INVALID,
               "chunk_attention8: null pointer argument");
  return chunk_attention("chunk_attention8", q, q_stride_t, q_stride_h, k_cache, v_cache, k_scales,
                         v_scales, num_blocks, block_tables, bt_stride_b, context_lens, cu_seqlens,
                         cu_host, B, H_q, H_kv, D, block_size, W, max_context_len, scale, causal,
                         out, lse, workspace, workspace_bytes, stream);
}
