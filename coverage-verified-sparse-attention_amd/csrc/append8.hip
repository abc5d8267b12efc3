// New tokens written to the 8-bit paged cache (cvsa_append_chunk_kv8): norms and
// rotation as for the bf16 cache, then e4m3 payloads with a power of two for each
// page and head.
//
// Of a page's new rows y (one head, keys or values): top = max |y| of the finite
// ones, e the smallest exponent with top <= 448 * 2^e, payload = y 2^-e rounded to
// nearest even (a relative half step of 2^-4; the scaling itself is exact).  Tokens
// that the page held before keep their exponent if it is as large; else they are
// brought to the new one, a shift of their exponents that rounds only what becomes
// subnormal.  Powers of two cost nothing: e4m3's relative step does not depend on
// where in its range a value lies, and with them payload * 2^e is a bf16 exactly,
// which the attention's conversions make in one instruction.  Infinite and NaN
// values become NaN and do not count for top.
//
// A page and head is a job of its own: a wave has up to four passes of 64 D / 16
// lanes over its rows (all of a 16-token page at D = 128 in two), larger pages take
// several waves of a workgroup, smaller ones share a wave with other heads.  Values
// wait in registers, in 32 bits, for the page's largest, so every element is read
// and written once, and the single rounding is that to 8 bits.
//
// Measured: 8191 tokens of 28 heads on 4 of 128, queries and keys normed and rotated, 31
// to 35 us for 147 MB, 4.2 to 4.7 TB/s (a copy reaches 5.1).  Single tokens are bound by
// latency: one of 32 heads on 8 4.7 us, 32 of them 5.6.
#include "cache8.h"
#include "rotary_common.h"

namespace cvsa {

struct Append8Args {
  uint8_t *k_cache, *v_cache, *k_scales, *v_scales;
  int bs_log2;
  int waves;       // of a page and head, 1 to 8
  int heads;       // of a wave
  int passes;      // of a wave, up to kAppendPasses
  int head_jobs;   // waves or groups of waves over the heads
  int64_t units;   // pages that the chunk may touch, see append8_kernel
  unsigned page_wgs;
};

constexpr int kAppendPasses = 4;
constexpr int kAppendThreads = 512;

// Pages: sequence b has the units from cu[b] / block_size + 2 b on: n tokens touch
// at most (n - 2) / block_size + 2 pages (rounded down; none if n = 0, one if n =
// 1), and the next sequence starts at least n / block_size + 2 units on.  What is
// behind a sequence's last page is empty.
template <class T, int D, bool PAIRS, bool ONCE>
__global__ __launch_bounds__(kAppendThreads) void append8_kernel(const RotaryArgs a,
                                                                 const Append8Args e) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wg_waves = blockDim.x >> 6;
  if (blockIdx.x >= e.page_wgs) {  // the queries' rows
    rotary_rows<T, D, PAIRS, true, ONCE, true>(
        a, (int64_t)(blockIdx.x - e.page_wgs) * wg_waves + wave);
    return;
  }
  constexpr int LR = D / 16, RW = 64 / LR, ES = Vec8<T>::kSize;
  __shared__ uint32_t s_top[kAppendThreads / kWave];
  const int lane = threadIdx.x & 63, j = lane % LR, sub = lane / LR;
  const int bs = 1 << e.bs_log2;

  // The job: unit, keys or values, heads; and this wave's part of its rows.
  int64_t job = (int64_t)blockIdx.x * (wg_waves / e.waves) + wave / e.waves;
  const int part = wave % e.waves;
  const int head0 = (int)(job % e.head_jobs) * e.heads;
  job /= e.head_jobs;
  const bool values = job & 1;
  const int64_t unit = job >> 1;
  const int head = head0 + (e.heads > 1 ? sub >> e.bs_log2 : 0);

  int b = 0, lo = 0, hi = 0, page = 0;  // rows lo .. hi of the page are new
  int blk = -1;
  int64_t token0 = 0;                   // of row 0
  if (unit < e.units) {
    b = last_that(a.B, [&](int b) {
      return (int64_t)(a.cu[b] >> e.bs_log2) + 2 * (int64_t)b <= unit;
    });
    const int first = a.cu[b], n = a.cu[b + 1] - first, ctx = a.context_lens[b];
    const int64_t before = (int64_t)ctx - n;
    const int64_t p = (before >> e.bs_log2) + (unit - ((first >> e.bs_log2) + 2 * (int64_t)b));
    const int64_t start = p << e.bs_log2;
    if (n > 0 && p >= 0 && p < a.W && start < ctx) {
      page = (int)p;
      blk = a.block_tables[b * a.bt_sb + page];
      lo = (int)max(before - start, (int64_t)0);
      hi = (int)min(ctx - start, (int64_t)bs);
      token0 = first + (start - before);
    }
  }
  const bool live = blk >= 0 && blk < a.num_blocks && hi > lo;
  if (!live) blk = lo = hi = 0;

  const RotaryPlace<D, PAIRS> at(a, j);
  auto row_of = [&](int u) { return e.heads > 1 ? sub & (bs - 1) : (part * e.passes + u) * RW + sub; };
  // Whether some row of pass u is new (the same in all lanes).
  auto pass_live = [&](int u) {
    const int r0 = e.heads > 1 ? 0 : (part * e.passes + u) * RW;
    return u < e.passes && r0 < hi && r0 + RW > lo;
  };
  const char *const src = (const char *)(values ? a.v : a.k);
  const int64_t st = values ? a.v_st : a.k_st, sh = values ? a.v_sh : a.k_sh;
  const int src_head = min(head, a.H_kv - 1);
  Vec8<T> x0[kAppendPasses], x1[kAppendPasses];
  unrolled<kAppendPasses>([&](auto pass) {
    constexpr int u = decltype(pass)::value;
    if (!pass_live(u)) return;  // lanes without a new row read the nearest one
    const int64_t t = token0 + min(max(row_of(u), lo), hi - 1);
    const char *p = src + (t * st + src_head * sh) * ES;
    x0[u].load(p + at.c0 * 8 * ES);
    x1[u].load(p + at.c1 * 8 * ES);
  });
  uint8_t *const scales = values ? e.v_scales : e.k_scales;
  const int64_t scale_at = (int64_t)blk * a.H_kv + src_head;
  const int old = live && lo > 0 ? scales[scale_at] : 0;

  float f0[kAppendPasses][8], f1[kAppendPasses][8];
  uint32_t top = 0;
  unrolled<kAppendPasses>([&](auto pass) {
    constexpr int u = decltype(pass)::value;
    if (!pass_live(u)) return;
    x0[u].get(f0[u]);
    x1[u].get(f1[u]);
    const int r = row_of(u);
    if (!values) {
      float cs[8], sn[8];
      at.angles(a, (int64_t)page * bs + r, cs, sn);
      at.norm(a, a.k_w, f0[u], f1[u]);
      if (a.table) at.turn(cs, sn, f0[u], f1[u]);
    }
    if (r >= lo && r < hi) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t m0 = __float_as_uint(f0[u][i]) & 0x7fffffffu;
        const uint32_t m1 = __float_as_uint(f1[u][i]) & 0x7fffffffu;
        top = max(top, finite_bits(m0) ? m0 : 0u);
        top = max(top, finite_bits(m1) ? m1 : 0u);
      }
    }
  });
  // The largest of the page and head: over the lanes of its rows, then the waves.
  // Values are not negative, so their bits are in their order.
  const int span = e.heads > 1 ? bs * LR : 64;
  top = max(top, dpp_u<kDppQuadXor1>(top));  // spans of 16 lanes at least
  top = max(top, dpp_u<kDppQuadXor2>(top));
  top = max(top, dpp_u<kDppRowHalfMirror>(top));
  top = max(top, dpp_u<kDppRowMirror>(top));
  if (span > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(top, top, false, false);
    top = max(r[0], r[1]);
  }
  if (span > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    top = max(r[0], r[1]);
  }
  if (e.waves > 1) {  // the same in all of the launch
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    for (int w = 0; w < e.waves; ++w) top = max(top, s_top[wave - part + w]);
  }
  if (!live || head >= a.H_kv) return;

  const int byte = max(scale_byte(top), old);
  const float inv = power_of_two(127 - byte);
  const bool clamp = byte - 127 >= kHighExponent;
  uint8_t *const rows = (values ? e.v_cache : e.k_cache) + ((int64_t)blk * bs * a.H_kv + head) * D;
  const int64_t row_bytes = (int64_t)a.H_kv * D;
  if (lo > 0 && byte != old) {  // earlier tokens, to the larger scale
    for (int u = 0; u < e.passes; ++u) {
      const int r = row_of(u);
      if (r >= lo) continue;
      uint8_t *const p = rows + r * row_bytes;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint2 *const w = reinterpret_cast<uint2 *>(p + (i ? at.c1 : at.c0) * 8);
        *w = shifted_8_bits(*w, old - byte);
      }
    }
  }
  unrolled<kAppendPasses>([&](auto pass) {
    constexpr int u = decltype(pass)::value;
    if (!pass_live(u)) return;
    const int r = row_of(u);
    if (r < lo || r >= hi) return;
    uint8_t *const p = rows + r * row_bytes;
    *reinterpret_cast<uint2 *>(p + at.c0 * 8) = to_8_bits(f0[u], inv, clamp);
    *reinterpret_cast<uint2 *>(p + at.c1 * 8) = to_8_bits(f1[u], inv, clamp);
  });
  // One lane of the page and head.
  if (part == 0 && (lane & (span - 1)) == 0 && byte != old)
    scales[scale_at] = (uint8_t)byte;
}

template <class T, int D>
static void launch_append8(const RotaryArgs &a, const Append8Args &e, bool pairs, bool once,
                           dim3 grid, dim3 block, hipStream_t s) {
  auto go = [&](auto p, auto o) {
    hipLaunchKernelGGL((append8_kernel<T, D, decltype(p)::value, decltype(o)::value>), grid, block,
                       0, s, a, e);
  };
  const std::true_type yes;
  const std::false_type no;
  if (pairs) once ? go(yes, yes) : go(yes, no);
  else once ? go(no, yes) : go(no, no);
}

template <class T>
static void launch_append8_d(const RotaryArgs &a, const Append8Args &e, int D, bool pairs,
                             bool once, dim3 grid, dim3 block, hipStream_t s) {
  if (D == 32) launch_append8<T, 32>(a, e, pairs, once, grid, block, s);
  else if (D == 64) launch_append8<T, 64>(a, e, pairs, once, grid, block, s);
  else if (D == 128) launch_append8<T, 128>(a, e, pairs, once, grid, block, s);
  else launch_append8<T, 256>(a, e, pairs, once, grid, block, s);
}

}  // namespace cvsa

using namespace cvsa;

extern "C" int cvsa_append_chunk_kv8(
    const void *k, int64_t k_stride_t, int64_t k_stride_h, const void *v, int64_t v_stride_t,
    int64_t v_stride_h, const void *q, int64_t q_stride_t, int64_t q_stride_h, int32_t dtype,
    uint8_t *k_cache, uint8_t *v_cache, uint8_t *k_scales, uint8_t *v_scales, int64_t num_blocks,
    const int32_t *block_tables, int64_t bt_stride_b, int32_t W, const int32_t *context_lens,
    const int32_t *cu_seqlens, int32_t B, int32_t tokens, const float *table, int64_t table_len,
    int32_t rot_dim, int32_t interleaved, const void *q_weight, const void *k_weight,
    int32_t weight_dtype, float eps, int32_t H_q, int32_t H_kv, int32_t D, int32_t block_size,
    void *q_out, void *stream) {
  CVSA_REQUIRE(k && v && k_cache && v_cache && k_scales && v_scales && block_tables &&
                   context_lens && cu_seqlens && (!q || q_out),
               CVSA_ERR_INVALID, "append_chunk_kv8: null pointer argument");
  CVSA_REQUIRE(B > 0 && W > 0 && num_blocks > 0 && bt_stride_b >= W, CVSA_ERR_INVALID,
               "append_chunk_kv8: bad sizes B=%d W=%d", B, W);
  CVSA_REQUIRE(block_size_supported(block_size), CVSA_ERR_UNSUPPORTED,
               "append_chunk_kv8: block_size=%d not in {8, 16, 32, 64, 128}", block_size);
  CVSA_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0, CVSA_ERR_INVALID,
               "append_chunk_kv8: caches must be 16-byte aligned");
  CVSA_REQUIRE(k_cache != v_cache && k_scales != v_scales, CVSA_ERR_INVALID,
               "append_chunk_kv8: keys and values must have caches and scales of their own");
  RotaryArgs a = {};
  a.k = k; a.k_st = k_stride_t; a.k_sh = k_stride_h;
  a.v = v; a.v_st = v_stride_t; a.v_sh = v_stride_h;
  if (q) {
    a.q = q; a.q_st = q_stride_t; a.q_sh = q_stride_h; a.q_out = q_out;
  }
  a.table = table; a.table_len = table_len; a.R = rot_dim;
  a.q_w = q ? q_weight : nullptr; a.k_w = k_weight; a.w_dtype = weight_dtype; a.eps = eps;
  a.tokens = tokens; a.H_q = H_q; a.H_kv = H_kv;
  a.num_blocks = num_blocks;
  a.block_tables = block_tables; a.bt_sb = bt_stride_b; a.W = W; a.block_size = block_size;
  a.B = B; a.context_lens = context_lens; a.cu = cu_seqlens;
  const int rc = check_rotary("append_chunk_kv8", a, dtype, D, interleaved);
  if (rc != CVSA_OK) return rc;

  Append8Args e = {};
  e.k_cache = k_cache; e.v_cache = v_cache;
  e.k_scales = k_scales; e.v_scales = v_scales;
  e.bs_log2 = __builtin_ctz(block_size);
  const int rows = 64 / (D / 16);  // of a pass
  const int passes = block_size > rows ? block_size / rows : 1;
  e.heads = rows > block_size ? rows / block_size : 1;
  e.passes = passes < kAppendPasses ? passes : kAppendPasses;
  e.waves = passes / e.passes;
  e.head_jobs = (H_kv + e.heads - 1) / e.heads;
  e.units = (int64_t)(tokens / block_size) + 2 * (int64_t)B;
  const int wg_waves = e.waves > 4 ? 8 : 4;
  const int64_t jobs = e.units * 2 * e.head_jobs, per_wg = wg_waves / e.waves;
  const int64_t page_wgs = (jobs + per_wg - 1) / per_wg;
  // The page jobs have the keys; the rows of a launch beside them are the queries'.
  RotaryArgs r = a;
  r.k = nullptr;
  bool once;
  const int64_t q_waves = q ? rotary_waves(r, D, true, once) : 0;
  if (!q) once = tokens >= 2048;
  a.groups = r.groups; a.per_wave = r.per_wave; a.segs = r.segs;
  const int64_t wgs = page_wgs + (q_waves + wg_waves - 1) / wg_waves;
  CVSA_REQUIRE(wgs < (1LL << 32) / (wg_waves * 64), CVSA_ERR_UNSUPPORTED,
               "append_chunk_kv8: too many tokens, sequences or heads");
  e.page_wgs = (unsigned)page_wgs;
  const dim3 grid((unsigned)wgs), block(wg_waves * 64);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == CVSA_DTYPE_BF16) launch_append8_d<Bf16>(a, e, D, interleaved, once, grid, block, s);
  else if (dtype == CVSA_DTYPE_FP16) launch_append8_d<Fp16>(a, e, D, interleaved, once, grid, block, s);
  else launch_append8_d<float>(a, e, D, interleaved, once, grid, block, s);
  return cvsa_host::check_launch("append_chunk_kv8");
}
