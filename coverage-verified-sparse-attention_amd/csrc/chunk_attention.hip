// Attention of a chunk of new tokens over the paged cache: the join of split
// keys, the launch plan and the entry points.  Kernel: chunk_attention.h.
#include "chunk_attention.h"

#include <algorithm>
#include <type_traits>

namespace cvsa {

constexpr int kJoinThreads = 256;

// The states of a row's splits joined in the order of the keys: a workgroup
// per token, D / 4 threads per row.
template <int D>
__global__ __launch_bounds__(kJoinThreads) void chunk_join_kernel(const ChunkArgs a,
                                                                  int tile_rows) {
  const int tok = blockIdx.x;
  const int lane = threadIdx.x & 63;
  int b = 0, n = a.B;
  while (n > 1) {  // the last sequence with cu[b] <= tok, 64 candidates a look
    const int step = (n + 63) / 64;
    const bool le = lane * step < n && a.cu[b + lane * step] <= tok;
    const int k = __popcll(__ballot(le)) - 1;
    b += k * step;
    n = min(step, n - k * step);
  }
  const int first = a.cu[b], len = a.cu[b + 1] - first, ctx = a.context_lens[b];
  const int64_t rows = (int64_t)a.tokens * a.H_q;
  for (int i = threadIdx.x; i < a.H_q * (D / 4); i += kJoinThreads) {
    const int head = i / (D / 4), d = i % (D / 4) * 4;
    const int row0 = ((tok - first) * a.G + head % a.G) / tile_rows * tile_rows;
    const int keys = chunk_tile_keys(a, ctx - len, ctx, len * a.G, row0, tile_rows);
    const int parts = min((keys + a.split_len - 1) / a.split_len, a.splits);
    const int64_t at = (int64_t)tok * a.H_q + head;
    float m = -INFINITY;
    for (int s = 0; s < parts; ++s) m = fmaxf(m, a.part_ml[s * rows + at].x);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < parts; ++s) {
      const float2 ml = a.part_ml[s * rows + at];
      const float w = __builtin_amdgcn_exp2f(ml.x - ref);
      const float4 v = *reinterpret_cast<const float4 *>(a.part_o + (s * rows + at) * D + d);
      l = fmaf(ml.y, w, l);
      o.x = fmaf(v.x, w, o.x);
      o.y = fmaf(v.y, w, o.y);
      o.z = fmaf(v.z, w, o.z);
      o.w = fmaf(v.w, w, o.w);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2 *>(a.out + at * D + d) =
        make_uint2(chunk_cvt_bf16x2(o.x * inv, o.y * inv), chunk_cvt_bf16x2(o.z * inv, o.w * inv));
    if (a.lse && d == 0)
      a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
}

template <int D>
static void launch_chunk(const ChunkArgs &a, int row_waves, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.tiles * a.H_kv * a.splits));
  auto go = [&](auto rw) {
    constexpr int RW = decltype(rw)::value;
    if constexpr (RW < 8 || D == 64 || D == 128)
      hipLaunchKernelGGL((chunk_attention_kernel<D, RW>), grid,
                         dim3(RW * chunk_key_tiles<D>(RW) * 64), 0, s, a);
  };
  if (row_waves == 1) go(std::integral_constant<int, 1>());
  else if (row_waves == 2) go(std::integral_constant<int, 2>());
  else if (row_waves == 4) go(std::integral_constant<int, 4>());
  else go(std::integral_constant<int, 8>());
  if (a.splits > 1)
    hipLaunchKernelGGL(chunk_join_kernel<D>, dim3(a.tokens), dim3(kJoinThreads), 0, s, a,
                       row_waves * 32);
}

struct ChunkPlan {
  int row_waves, tiles, splits, split_len;
};

// Row waves of a workgroup and splits of the keys, from the chunk lengths and
// the most keys a sequence can hold.
static ChunkPlan plan_chunk(const int32_t *cu, int B, int H_kv, int G, int D, int64_t max_keys) {
  ChunkPlan p;
  int64_t longest = 0;
  for (int b = 0; b < B; ++b) longest = std::max<int64_t>(longest, cu[b + 1] - cu[b]);
  const int64_t rows = longest * G;
  p.row_waves = rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 || D == 256 || D == 32 ? 4 : 8;
  const int64_t tile_rows = p.row_waves * 32;
  int64_t tiles = 0;
  for (int b = 0; b < B; ++b)
    tiles += ((int64_t)(cu[b + 1] - cu[b]) * G + tile_rows - 1) / tile_rows;
  p.tiles = (int)tiles;
  const int64_t items = std::max<int64_t>(1, tiles * H_kv);
  // Splits of at least 512 keys, enough of them for four workgroups per CU.
  const int64_t want = std::min<int64_t>((1024 + items - 1) / items, 64);
  int64_t len = std::max<int64_t>(512, (max_keys + want - 1) / want);
  len = (len + 127) / 128 * 128;
  p.split_len = (int)len;
  p.splits = items >= 512 ? 1 : (int)std::max<int64_t>(1, (max_keys + len - 1) / len);
  return p;
}

static size_t chunk_part_bytes(const ChunkPlan &p, int64_t rows, int D) {
  if (p.splits <= 1) return 0;
  const size_t ml = ((size_t)p.splits * rows * sizeof(float2) + 255) / 256 * 256;
  return ml + (size_t)p.splits * rows * D * sizeof(float);
}

static bool chunk_shape_ok(const int32_t *cu, int32_t B, int32_t H_q, int32_t H_kv, int32_t D,
                           int32_t block_size, int32_t W) {
  if (!cu || B <= 0 || B > (1 << 20) || H_kv <= 0 || H_q <= 0 || H_q % H_kv ||
      H_q / H_kv > 128 || H_q > 65536 || W <= 0 || W > kMaxPagesWide ||
      !head_dim_supported(D) || !block_size_supported(block_size) || cu[0] != 0)
    return false;
  for (int b = 0; b < B; ++b)
    if (cu[b + 1] < cu[b]) return false;
  return cu[B] <= (1 << 24) && (int64_t)cu[B] * (H_q / H_kv) < (1 << 30);
}

static int64_t chunk_max_keys(int32_t W, int32_t block_size, int32_t max_context_len) {
  const int64_t all = (int64_t)W * block_size;
  return max_context_len > 0 ? std::min<int64_t>(all, max_context_len) : all;
}

}  // namespace cvsa

using namespace cvsa;

extern "C" size_t cvsa_chunk_attention_workspace_bytes(const int32_t *cu_host, int32_t B,
                                                       int32_t H_q, int32_t H_kv, int32_t D,
                                                       int32_t block_size, int32_t W,
                                                       int32_t max_context_len) {
  if (!chunk_shape_ok(cu_host, B, H_q, H_kv, D, block_size, W) || cu_host[B] == 0) return 0;
  const ChunkPlan p = plan_chunk(cu_host, B, H_kv, H_q / H_kv, D,
                                 chunk_max_keys(W, block_size, max_context_len));
  return chunk_part_bytes(p, (int64_t)cu_host[B] * H_q, D);
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
  CVSA_REQUIRE(q && k_cache && v_cache && block_tables && context_lens && cu_seqlens && cu_host &&
                   out,
               CVSA_ERR_INVALID, "chunk_attention: null pointer argument");
  CVSA_REQUIRE(head_dim_supported(D), CVSA_ERR_UNSUPPORTED,
               "chunk_attention: D=%d not in {32, 64, 128, 256}", D);
  CVSA_REQUIRE(block_size_supported(block_size), CVSA_ERR_UNSUPPORTED,
               "chunk_attention: block_size=%d not in {8, 16, 32, 64, 128}", block_size);
  CVSA_REQUIRE(H_kv > 0 && H_q > 0 && H_q % H_kv == 0, CVSA_ERR_INVALID,
               "chunk_attention: head counts H_q=%d H_kv=%d", H_q, H_kv);
  CVSA_REQUIRE(H_q / H_kv <= 128 && W <= kMaxPagesWide, CVSA_ERR_UNSUPPORTED,
               "chunk_attention: G=%d (at most 128) or W=%d (at most %d) not supported",
               H_q / H_kv, W, kMaxPagesWide);
  CVSA_REQUIRE(chunk_shape_ok(cu_host, B, H_q, H_kv, D, block_size, W) && num_blocks > 0 &&
                   bt_stride_b >= W,
               CVSA_ERR_INVALID, "chunk_attention: bad sizes or chunk offsets (B=%d W=%d)", B, W);
  CVSA_REQUIRE((int64_t)block_size * H_kv * D < (1 << 30), CVSA_ERR_UNSUPPORTED,
               "chunk_attention: a block of %d tokens of %d heads is too large", block_size, H_kv);
  CVSA_REQUIRE(scale > 0.f && scale < INFINITY, CVSA_ERR_INVALID,
               "chunk_attention: scale must be positive and finite");
  CVSA_REQUIRE(max_context_len >= 0 && (causal == 0 || causal == 1), CVSA_ERR_INVALID,
               "chunk_attention: bad max_context_len=%d or causal=%d", max_context_len, causal);
  CVSA_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) ==
                       0 &&
                   q_stride_t % 8 == 0 && q_stride_h % 8 == 0,
               CVSA_ERR_INVALID, "chunk_attention: rows must be 16-byte aligned");
  const int32_t tokens = cu_host[B];
  if (tokens == 0) return CVSA_OK;
  const ChunkPlan p = plan_chunk(cu_host, B, H_kv, H_q / H_kv, D,
                                 chunk_max_keys(W, block_size, max_context_len));
  const int64_t rows = (int64_t)tokens * H_q;
  const size_t need = chunk_part_bytes(p, rows, D);
  CVSA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need &&
                             ((uintptr_t)workspace & 255) == 0),
               CVSA_ERR_WORKSPACE,
               "chunk_attention: needs a 256-byte aligned workspace of %zu bytes", need);
  CVSA_REQUIRE((int64_t)p.tiles * H_kv * p.splits < (1LL << 31), CVSA_ERR_UNSUPPORTED,
               "chunk_attention: too many row tiles");
  ChunkArgs a = {};
  a.q = q; a.q_st = q_stride_t; a.q_sh = q_stride_h;
  a.k_cache = k_cache; a.v_cache = v_cache; a.num_blocks = (int)std::min<int64_t>(num_blocks, INT32_MAX);
  a.block_tables = block_tables; a.bt_sb = bt_stride_b; a.W = W;
  a.context_lens = context_lens; a.cu = cu_seqlens;
  a.B = B; a.H_q = H_q; a.H_kv = H_kv; a.G = H_q / H_kv; a.tokens = tokens;
  a.bs_log2 = __builtin_ctz(block_size);
  a.c = scale * 1.4426950408889634f;
  a.causal = causal;
  a.out = out; a.lse = lse;
  a.tiles = p.tiles; a.splits = p.splits; a.split_len = p.split_len;
  if (p.splits > 1) {
    a.part_ml = (float2 *)workspace;
    a.part_o = (float *)((char *)workspace +
                         ((size_t)p.splits * rows * sizeof(float2) + 255) / 256 * 256);
  }
  const hipStream_t s = (hipStream_t)stream;
  if (D == 32) launch_chunk<32>(a, p.row_waves, s);
  else if (D == 64) launch_chunk<64>(a, p.row_waves, s);
  else if (D == 128) launch_chunk<128>(a, p.row_waves, s);
  else launch_chunk<256>(a, p.row_waves, s);
  return cvsa_host::check_launch("chunk_attention");
}
