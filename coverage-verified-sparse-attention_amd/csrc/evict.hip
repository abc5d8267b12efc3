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
// First launch: a workgroup for each sequence and head finds the m-th largest
// weight by its bits, 11, 11 and 10 at a time (histograms in LDS), then walks the
// slots once in order and writes down which old slot each new one gets.  A
// destination is a source itself only among slots keep - recent .. keep; other
// workgroups of the launch copy these rows aside.  Second launch: a wave for each
// page with arrivals, keys and values apart, no order among them.
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
  // Workspace, each [B, H_kv, ...].
  int32_t *holes;          // [keep]
  float *moved_weights;    // [keep]
  uint8_t *moved_scales;   // [2, keep]: bytes of the scales of the sources' pages
  int32_t *pages;          // [1 + pages]: pages with arrivals, their number first
  char *aside;             // [2, recent, row_bytes]
  unsigned plan_wgs;       // workgroups before those that copy aside
};

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / kWave;
constexpr int kBins = 2048, kCopies = 4;
constexpr int kSlots = 4;  // of a thread and step

__device__ __forceinline__ int evict_context(const EvictArgs &a, int b) {
  return max(0, min(a.context_lens[b], a.W << a.bs_log2));
}
// Block of a slot, -1: none of the pool.
__device__ __forceinline__ int evict_block(const EvictArgs &a, int b, int slot) {
  const int blk = a.block_tables[b * a.bt_sb + (slot >> a.bs_log2)];
  return (uint32_t)blk < (uint64_t)a.num_blocks ? blk : -1;
}
__device__ __forceinline__ int64_t evict_row(const EvictArgs &a, int blk, int slot, int h) {
  const int64_t token = ((int64_t)blk << a.bs_log2) + (slot & ((1 << a.bs_log2) - 1));
  return (token * a.H_kv + h) * a.row_bytes;
}

// Weights' order as unsigned numbers; NaN is above all, zeros are equal.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xffffffffu;
  return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}

// Sums over the workgroup of each wave's total before this one, and in all.
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
  __syncthreads();
  return r;
}

__device__ __forceinline__ void evict_copy_aside(const EvictArgs &a) {
  // A thread for each 16 bytes of keys and of values.
  const int per_row = a.row_bytes / 16;
  const int64_t i = (int64_t)(blockIdx.x - a.plan_wgs) * kEvictThreads + threadIdx.x;
  const int64_t rows = i / per_row;
  const int part = (int)(i - rows * per_row) * 16;
  const int64_t bh = rows / a.recent;
  const int n = (int)(rows - bh * a.recent), b = (int)(bh / a.H_kv), h = (int)(bh % a.H_kv);
  if (b >= a.B || evict_context(a, b) <= a.keep) return;
  const int slot = a.keep - a.recent + n, blk = evict_block(a, b, slot);
  if (blk < 0) return;
  const int64_t from = evict_row(a, blk, slot, h) + part;
  char *const to = a.aside + ((bh * 2) * a.recent + n) * a.row_bytes + part;
  *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(a.k_cache + from);
  *reinterpret_cast<uint4 *>(to + (int64_t)a.recent * a.row_bytes) =
      *reinterpret_cast<const uint4 *>(a.v_cache + from);
}

__global__ __launch_bounds__(kEvictThreads) void evict_plan_kernel(const EvictArgs a) {
  if (blockIdx.x >= a.plan_wgs) {
    evict_copy_aside(a);
    return;
  }
  __shared__ uint32_t s_hist[kCopies][kBins];
  __shared__ uint32_t s_sum[kEvictWaves];
  __shared__ uint32_t s_bin, s_above;
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / a.H_kv), h = (int)(bh % a.H_kv);
  const int ctx = evict_context(a, b);
  float *const w = a.weights + bh * a.S;
  int32_t *const kept = a.kept + bh * a.keep, *const holes = a.holes + bh * a.keep;
  const int n_pages = (a.keep + (1 << a.bs_log2) - 1) >> a.bs_log2;
  int32_t *const pages = a.pages + bh * (1 + n_pages);
  if (ctx <= a.keep) {  // nothing to cut
    for (int j = tid; j < a.keep; j += kEvictThreads) kept[j] = j < ctx ? j : -1;
    if (tid == 0) pages[0] = 0;
    return;
  }
  const int front = a.keep - a.recent, back = ctx - a.recent;
  uint32_t want = (uint32_t)(front - a.sinks);  // of the middle, which has more

  // The want-th largest: `threshold`, of whose equals the first `want` stay.
  uint32_t threshold = 0xffffffffu, known = 0;
  if (want == 0) {
    // None of the middle: nothing is above this, and none of its equals stays.
  } else {
    threshold = 0;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kCopies * kBins; i += kEvictThreads) (&s_hist[0][0])[i] = 0;
      __syncthreads();
      uint32_t *const hist = s_hist[(tid >> 6) % kCopies];
      for (int j = a.sinks + tid; j < back; j += kEvictThreads) {
        const uint32_t k = weight_key(w[j]);
        if ((k & known) == threshold) atomicAdd(&hist[k >> shift & ((1u << bits) - 1)], 1u);
      }
      __syncthreads();
      // Bins from the largest on, two a thread.
      const int top = (1 << bits) - 1 - 2 * tid;
      uint32_t n0 = 0, n1 = 0;
      if (top > 0) {
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          n0 += s_hist[c][top];
          n1 += s_hist[c][top - 1];
        }
      }
      const EvictScan s = evict_scan(n0 + n1, s_sum);
      if (s.before < want && want <= s.before + n0 + n1) {
        const bool second = want > s.before + n0;
        s_bin = (uint32_t)(second ? top - 1 : top);
        s_above = s.before + (second ? n0 : 0u);
      }
      __syncthreads();
      threshold |= s_bin << shift;
      known |= ((1u << bits) - 1) << shift;
      want -= s_above;
      __syncthreads();
    }
  }

  // The slots in order: the kept ones below `front` stay, the others are holes; the
  // kept ones behind fill them.
  for (int j = tid; j < a.sinks; j += kEvictThreads) kept[j] = j;
  for (int j = tid; j < a.recent; j += kEvictThreads) kept[front + j] = back + j;
  uint32_t above = 0, equal = 0;  // before the step
  uint32_t stay = 0;              // kept ones below front
  auto walk = [&](int begin, int end, bool tail) {
    for (int j0 = begin; j0 < end; j0 += kEvictThreads * kSlots) {
      const int first = j0 + tid * kSlots;
      uint32_t key[kSlots];
      uint32_t count = 0;
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        key[i] = first + i < end ? weight_key(w[first + i]) : 0u;
        if (first + i < end)
          count += (key[i] > threshold ? 1u : 0u) + (key[i] == threshold ? 0x10000u : 0u);
      }
      const EvictScan s = evict_scan(count, s_sum);
      uint32_t gt = above + (s.before & 0xffffu), eq = equal + (s.before >> 16);
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        const int slot = first + i;
        if (slot >= end) break;
        const bool keep = key[i] > threshold || (key[i] == threshold && eq < want);
        const uint32_t rank = gt + min(eq, want);  // kept ones before
        if (!tail) {
          if (keep) kept[slot] = slot;
          else holes[(uint32_t)(slot - a.sinks) - rank] = slot;
        } else if (keep) {
          kept[holes[rank - stay]] = slot;
        }
        gt += key[i] > threshold ? 1u : 0u;
        eq += key[i] == threshold ? 1u : 0u;
      }
      above += s.all & 0xffffu;
      equal += s.all >> 16;
    }
  };
  walk(a.sinks, front, false);
  stay = above + min(equal, want);
  __syncthreads();
  walk(front, back, true);
  __syncthreads();

  // What moves: its weight and the scales of where it comes from.
  float *const moved = a.moved_weights + bh * a.keep;
  uint8_t *const scales = a.moved_scales + bh * 2 * a.keep;
  for (int j = tid; j < a.keep; j += kEvictThreads) {
    const int src = kept[j];
    if (src == j) continue;
    moved[j] = w[src];
    if (a.k_scales) {
      const int blk = evict_block(a, b, src);
      scales[j] = blk < 0 ? 0 : a.k_scales[(int64_t)blk * a.H_kv + h];
      scales[a.keep + j] = blk < 0 ? 0 : a.v_scales[(int64_t)blk * a.H_kv + h];
    }
  }
  __syncthreads();
  for (int j = tid; j < a.keep; j += kEvictThreads)
    if (kept[j] != j) w[j] = moved[j];
  // Pages with arrivals.
  int listed = 0;
  for (int p0 = 0; p0 < n_pages; p0 += kEvictThreads) {
    const int p = p0 + tid;
    bool any = false;
    if (p < n_pages) {
      const int end = min((p + 1) << a.bs_log2, a.keep);
      for (int j = p << a.bs_log2; j < end; ++j) any = any || kept[j] != j;
    }
    const EvictScan s = evict_scan(any ? 1u : 0u, s_sum);
    if (any) pages[1 + listed + s.before] = p;
    listed += (int)s.all;
  }
  if (tid == 0) pages[0] = listed;
}

// Rows of a page's arrivals, and in 8 bits the page's scale and its other rows.
// Keys by even waves, values by odd ones.
template <bool F8>
__global__ __launch_bounds__(256) void evict_move_kernel(const EvictArgs a, int wgs_each) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t bh = blockIdx.x / wgs_each;
  const int b = (int)(bh / a.H_kv), h = (int)(bh % a.H_kv);
  const bool values = wave & 1;
  const int bs = 1 << a.bs_log2, n_pages = (a.keep + bs - 1) >> a.bs_log2;
  const int32_t *const kept = a.kept + bh * a.keep;
  const int32_t *const pages = a.pages + bh * (1 + n_pages);
  const int listed = pages[0];
  char *const cache = values ? a.v_cache : a.k_cache;
  const char *const aside = a.aside + (bh * 2 + values) * a.recent * (int64_t)a.row_bytes;
  const int per_row = a.row_bytes / 16, rows = 64 / per_row;  // lanes of a row, rows at once
  const int part = lane % per_row * 16, sub = lane / per_row;
  for (int i = (int)(blockIdx.x % wgs_each) * 2 + wave / 2; i < listed; i += wgs_each * 2) {
    const int page = pages[1 + i], slot0 = page << a.bs_log2;
    const int blk = evict_block(a, b, slot0);
    if (blk < 0) continue;
    const int count = min(bs, a.keep - slot0);
    int byte = 0, old = 0;
    if constexpr (F8) {
      const uint8_t *const from = a.moved_scales + (bh * 2 + values) * a.keep;
      uint8_t *const at = (values ? a.v_scales : a.k_scales) + (int64_t)blk * a.H_kv + h;
      old = *at;
      uint32_t top = 0;
      for (int r = lane; r < count; r += 64)
        top = max(top, kept[slot0 + r] == slot0 + r ? (uint32_t)old : (uint32_t)from[slot0 + r]);
      byte = (int)wave_max_u32(top);
      if (lane == 0 && byte != old) *at = (uint8_t)byte;
    }
    // Up to four groups of rows are read before they are written.
    constexpr int kBatch = 4;
    for (int r0 = 0; r0 < count; r0 += rows * kBatch) {
      uint4 v[kBatch];
      int shift[kBatch];
      bool write[kBatch];
      unrolled<kBatch>([&](auto n) {
        constexpr int g = decltype(n)::value;
        const int r = r0 + g * rows + sub, slot = slot0 + r;
        v[g] = make_uint4(0, 0, 0, 0);
        write[g] = false;
        shift[g] = 0;
        if (r >= count) return;
        const int src = kept[slot];
        const char *p = nullptr;
        if (src == slot) {  // stays; its payload, where the scale has changed
          if (!F8 || byte == old) return;
          shift[g] = old - byte;
          p = cache + evict_row(a, blk, slot, h);
        } else {
          const int from = evict_block(a, b, src);
          if (from < 0) return;
          if constexpr (F8)
            shift[g] = a.moved_scales[(bh * 2 + values) * a.keep + slot] - byte;
          p = src < a.keep ? aside + (int64_t)(src - (a.keep - a.recent)) * a.row_bytes
                           : cache + evict_row(a, from, src, h);
        }
        v[g] = *reinterpret_cast<const uint4 *>(p + part);
        write[g] = true;
      });
      unrolled<kBatch>([&](auto n) {
        constexpr int g = decltype(n)::value;
        if (!write[g]) return;
        const int slot = slot0 + r0 + g * rows + sub;
        if constexpr (F8) {
          if (shift[g] != 0) v[g] = shifted_8_bits(v[g], shift[g]);
        }
        *reinterpret_cast<uint4 *>(cache + evict_row(a, blk, slot, h) + part) = v[g];
      });
    }
  }
}

struct EvictPlan {
  size_t holes, weights, scales, pages, aside, bytes;
};

static EvictPlan plan_evict(int64_t bh, int row_bytes, int bs, int keep, int recent, bool f8) {
  EvictPlan p = {};
  auto take = [&](size_t n) {
    const size_t at = p.bytes;
    p.bytes += (n + 255) / 256 * 256;
    return at;
  };
  p.holes = take((size_t)bh * keep * 4);
  p.weights = take((size_t)bh * keep * 4);
  p.scales = take(f8 ? (size_t)bh * keep * 2 : 0);
  p.pages = take((size_t)bh * (1 + (keep + bs - 1) / bs) * 4);
  p.aside = take((size_t)bh * 2 * recent * row_bytes);
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
                                                    int32_t block_size, int32_t cache_bits,
                                                    int32_t keep, int32_t sinks, int32_t recent) {
  if (!evict_sizes_ok(B, H_kv, D, block_size, keep, sinks, recent)) return 0;
  return plan_evict((int64_t)B * H_kv, D * cache_bits / 8, block_size, keep, recent,
                    cache_bits == 8)
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
  const int64_t bh = (int64_t)B * H_kv;
  const int row_bytes = D * (k_scales ? 1 : 2);
  const EvictPlan p = plan_evict(bh, row_bytes, block_size, keep, recent, k_scales != nullptr);
  CVSA_REQUIRE(workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 255) == 0,
               CVSA_ERR_WORKSPACE,
               "evict_tokens: needs a 256-byte aligned workspace of %zu bytes", p.bytes);
  const int64_t aside = bh * recent * (row_bytes / 16);
  CVSA_REQUIRE(aside / kEvictThreads + bh < (1LL << 31) - 1, CVSA_ERR_UNSUPPORTED,
               "evict_tokens: too many recent tokens");
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
  a.holes = (int32_t *)(ws + p.holes);
  a.moved_weights = (float *)(ws + p.weights);
  a.moved_scales = (uint8_t *)(ws + p.scales);
  a.pages = (int32_t *)(ws + p.pages);
  a.aside = ws + p.aside;
  a.plan_wgs = (unsigned)bh;
  const hipStream_t s = (hipStream_t)stream;
  const unsigned wgs = (unsigned)(bh + (aside + kEvictThreads - 1) / kEvictThreads);
  hipLaunchKernelGGL(evict_plan_kernel, dim3(wgs), dim3(kEvictThreads), 0, s, a);
  // Two pages at once in a workgroup; enough of them to fill the GPU, or one for
  // each two pages.
  const int n_pages = (keep + block_size - 1) / block_size;
  const int each = (int)std::max<int64_t>(1, std::min<int64_t>((n_pages + 1) / 2, 4096 / bh));
  const dim3 grid((unsigned)(bh * each));
  if (k_scales) hipLaunchKernelGGL(evict_move_kernel<true>, grid, dim3(256), 0, s, a, each);
  else hipLaunchKernelGGL(evict_move_kernel<false>, grid, dim3(256), 0, s, a, each);
  return cvsa_host::check_launch("evict_tokens");
}
