// Norms of queries and keys for each head with the position rotation in the
// same pass, written out (cvsa_qk_norm_rope) or, for keys, straight into the
// paged cache with the values beside them (cvsa_append_chunk_kv); and the
// pages a chunk of new tokens takes from the allocator (cvsa_reserve_chunk).
//
// A row is one head of one token: y = x * rsqrt(mean(x^2) + eps) * w, then
// pairs (a, b) -> (a cos - b sin, b cos + a sin) with the cosines and sines
// of the token's position, from a table.  All of it in 32 bits, rounded once
// to the output's type.
//
// The work is bound by memory: every element is read and written once.  A
// lane holds two 16-byte vectors of 8 elements of a row, chosen so that both
// members of every rotated pair are in one lane: D/16 lanes make a row and
// sum its squares with DPP moves.  A wave takes the heads of one token, so
// the cosines and sines are read once for all of them; the rows of up to
// three passes are requested before the first is worked on.
#include "rotary_common.h"

namespace cvsa {

// The allocation rule of the one-token append for each of a chunk's tokens in
// turn: a token at a page's start whose page is not allocated yet takes the
// next block, sequence after sequence.  So sequence b takes the pages from
// max(pages_allocated, pages of its context) to the pages of its new context.
constexpr int kReserveThreads = 1024;

__global__ __launch_bounds__(kReserveThreads) void reserve_chunk_kernel(
    int32_t *__restrict__ block_tables, int64_t bt_sb, int W, int32_t *__restrict__ context_lens,
    int32_t *__restrict__ pages_allocated, const int32_t *__restrict__ cu, int B, int next_free,
    int64_t num_blocks, int block_size) {
  __shared__ int s_first[kReserveThreads], s_count[kReserveThreads], s_base[kReserveThreads];
  __shared__ uint32_t wsum[kReserveThreads / kWave];
  const int i = threadIdx.x, lane = i & 63, wave = i >> 6;
  int base = next_free;
  for (int b0 = 0; b0 < B; b0 += kReserveThreads) {
    const int b = b0 + i;
    int first = 0, count = 0;
    if (b < B) {
      const int n = cu[b + 1] - cu[b];
      const int ctx = context_lens[b], alloc = pages_allocated[b];
      first = max(alloc, (ctx + block_size - 1) / block_size);
      count = n > 0 ? max(0, (ctx + n + block_size - 1) / block_size - first) : 0;
      context_lens[b] = ctx + n;
      pages_allocated[b] = alloc + count;
    }
    const uint32_t incl = wave_incl_scan_u32((uint32_t)count);
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    uint32_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kReserveThreads / kWave; ++w) {
      before += w < wave ? wsum[w] : 0u;
      total += wsum[w];
    }
    s_first[i] = first;
    s_count[i] = count;
    s_base[i] = base + (int)(before + incl) - count;
    base += (int)total;
    __syncthreads();
    for (int s = wave; s < min(kReserveThreads, B - b0); s += kReserveThreads / kWave)
      for (int p = lane; p < s_count[s]; p += kWave)
        if (s_first[s] + p < W && s_base[s] + p < num_blocks)
          block_tables[(b0 + s) * bt_sb + s_first[s] + p] = s_base[s] + p;
    __syncthreads();
  }
}

template <class T, int D, bool PAIRS, bool APPEND, bool ONCE>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryArgs a) {
  rotary_rows<T, D, PAIRS, APPEND, ONCE>(
      a, (int64_t)blockIdx.x * (kRotaryThreads / kWave) + (threadIdx.x >> 6));
}

template <class T, int D, bool APPEND>
static void launch_rotary(const RotaryArgs &a, int pairs, bool once, int64_t waves,
                          hipStream_t s) {
  const dim3 grid((unsigned)((waves + 3) / 4)), block(kRotaryThreads);
  auto go = [&](auto p, auto o) {
    hipLaunchKernelGGL((rotary_kernel<T, D, decltype(p)::value, APPEND, decltype(o)::value>),
                       grid, block, 0, s, a);
  };
  const std::true_type yes;
  const std::false_type no;
  if (pairs) once ? go(yes, yes) : go(yes, no);
  else once ? go(no, yes) : go(no, no);
}

template <class T, bool APPEND>
static void launch_rotary_d(const RotaryArgs &a, int D, int pairs, bool once, int64_t waves,
                            hipStream_t s) {
  if (D == 32) launch_rotary<T, 32, APPEND>(a, pairs, once, waves, s);
  else if (D == 64) launch_rotary<T, 64, APPEND>(a, pairs, once, waves, s);
  else if (D == 128) launch_rotary<T, 128, APPEND>(a, pairs, once, waves, s);
  else launch_rotary<T, 256, APPEND>(a, pairs, once, waves, s);
}

// Passes of a token and how many a wave takes: all of them once the tokens
// alone make enough waves to fill the GPU (2048), one otherwise.  With so many
// tokens the outputs are also stored past the caches: 8191 tokens of 28 + 4 heads
// of 128 take 29.7 us, 35.6 with ordinary stores.  The rule looks at the tokens
// alone, not at the bytes.  2047 tokens (neither) and 2048 (both), heads of 128:
// 1 + 1 heads 10.3 and 10.1 us, 32 + 8 10.6 and 10.0, 128 + 16 27.2 and 27.1, and
// 64 + 8 heads of fp32, whose 75 MB in and 75 MB out fit the last-level cache from
// pass to pass, 26.0 and 32.4.
int64_t rotary_waves(RotaryArgs &a, int D, bool append, bool &once) {
  const int rows = 64 / (D / 16);
  a.groups = (a.q ? (a.H_q + rows - 1) / rows : 0) +
             (a.k ? (a.H_kv * (append ? 2 : 1) + rows - 1) / rows : 0);
  once = a.tokens >= 2048;
  a.per_wave = once ? a.groups : 1;
  a.segs = a.groups ? (a.groups + a.per_wave - 1) / a.per_wave : 0;
  return (int64_t)a.tokens * a.segs;
}

template <bool APPEND>
static void enqueue_rotary(RotaryArgs &a, int dtype, int D, int pairs, void *stream) {
  bool once;
  const int64_t waves = rotary_waves(a, D, APPEND, once);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == CVSA_DTYPE_BF16) launch_rotary_d<Bf16, APPEND>(a, D, pairs, once, waves, s);
  else if (dtype == CVSA_DTYPE_FP16) launch_rotary_d<Fp16, APPEND>(a, D, pairs, once, waves, s);
  else launch_rotary_d<float, APPEND>(a, D, pairs, once, waves, s);
}

static bool dtype_ok(int32_t t) {
  return t == CVSA_DTYPE_BF16 || t == CVSA_DTYPE_FP16 || t == CVSA_DTYPE_FP32;
}

int check_rotary(const char *who, const RotaryArgs &a, int32_t dtype, int32_t D,
                        int32_t interleaved) {
  CVSA_REQUIRE(dtype_ok(dtype), CVSA_ERR_INVALID, "%s: unknown dtype code %d", who, dtype);
  CVSA_REQUIRE(head_dim_supported(D), CVSA_ERR_UNSUPPORTED,
               "%s: D=%d not in {32, 64, 128, 256}", who, D);
  CVSA_REQUIRE(interleaved == 0 || interleaved == 1, CVSA_ERR_INVALID,
               "%s: interleaved must be 0 or 1", who);
  CVSA_REQUIRE(a.tokens > 0 && a.tokens <= (1 << 26) && (!a.q || (a.H_q > 0 && a.H_q <= 65536)) &&
                   (!a.k || (a.H_kv > 0 && a.H_kv <= 65536)),
               CVSA_ERR_INVALID, "%s: bad sizes tokens=%d H_q=%d H_kv=%d", who, a.tokens, a.H_q,
               a.H_kv);
  if (a.table) {
    CVSA_REQUIRE(a.R >= 16 && a.R <= D && a.R % 16 == 0, CVSA_ERR_UNSUPPORTED,
                 "%s: rotated dimensions %d must be a multiple of 16, at most D=%d", who, a.R, D);
    CVSA_REQUIRE(a.table_len > 0 && ((uintptr_t)a.table & 15) == 0, CVSA_ERR_INVALID,
                 "%s: the table must hold rows and be 16-byte aligned", who);
  }
  CVSA_REQUIRE((!a.q_w && !a.k_w) || dtype_ok(a.w_dtype), CVSA_ERR_INVALID,
               "%s: unknown weight dtype code %d", who, a.w_dtype);
  CVSA_REQUIRE((((uintptr_t)a.q_w | (uintptr_t)a.k_w) & 15) == 0, CVSA_ERR_INVALID,
               "%s: weights must be 16-byte aligned", who);
  const int64_t unit = dtype == CVSA_DTYPE_FP32 ? 4 : 8;  // elements of 16 bytes
  const uintptr_t ptrs = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out |
                         (uintptr_t)a.k_out;
  CVSA_REQUIRE((ptrs & 15) == 0 && a.q_st % unit == 0 && a.q_sh % unit == 0 &&
                   a.k_st % unit == 0 && a.k_sh % unit == 0 && a.v_st % unit == 0 &&
                   a.v_sh % unit == 0,
               CVSA_ERR_INVALID, "%s: rows must be 16-byte aligned", who);
  return CVSA_OK;
}

}  // namespace cvsa

using namespace cvsa;

extern "C" int cvsa_qk_norm_rope(const void *q, int64_t q_stride_t, int64_t q_stride_h,
                                 const void *k, int64_t k_stride_t, int64_t k_stride_h,
                                 int32_t dtype, const void *positions, int32_t positions_bytes,
                                 const float *table, int64_t table_len, int32_t rot_dim,
                                 int32_t interleaved, const void *q_weight, const void *k_weight,
                                 int32_t weight_dtype, float eps, int32_t tokens, int32_t H_q,
                                 int32_t H_kv, int32_t D, void *q_out, void *k_out,
                                 void *stream) {
  CVSA_REQUIRE(q && q_out && (!k || k_out) && (!table || positions), CVSA_ERR_INVALID,
               "qk_norm_rope: null pointer argument");
  CVSA_REQUIRE(!table || positions_bytes == 4 || positions_bytes == 8, CVSA_ERR_INVALID,
               "qk_norm_rope: positions of %d bytes, not 4 or 8", positions_bytes);
  RotaryArgs a = {};
  a.q = q; a.q_st = q_stride_t; a.q_sh = q_stride_h; a.q_out = q_out;
  if (k) {
    a.k = k; a.k_st = k_stride_t; a.k_sh = k_stride_h; a.k_out = k_out;
  }
  a.table = table; a.table_len = table_len; a.R = rot_dim;
  a.q_w = q_weight; a.k_w = k ? k_weight : nullptr; a.w_dtype = weight_dtype; a.eps = eps;
  a.tokens = tokens; a.H_q = H_q; a.H_kv = H_kv; a.positions = positions;
  a.wide = positions_bytes == 8;
  const int rc = check_rotary("qk_norm_rope", a, dtype, D, interleaved);
  if (rc != CVSA_OK) return rc;
  enqueue_rotary<false>(a, dtype, D, interleaved, stream);
  return cvsa_host::check_launch("qk_norm_rope");
}

extern "C" int cvsa_append_chunk_kv(
    const void *k, int64_t k_stride_t, int64_t k_stride_h, const void *v, int64_t v_stride_t,
    int64_t v_stride_h, const void *q, int64_t q_stride_t, int64_t q_stride_h, int32_t dtype,
    uint16_t *k_cache, uint16_t *v_cache, int64_t num_blocks, const int32_t *block_tables,
    int64_t bt_stride_b, int32_t W, const int32_t *context_lens, const int32_t *cu_seqlens,
    int32_t B, int32_t tokens, const float *table, int64_t table_len, int32_t rot_dim,
    int32_t interleaved, const void *q_weight, const void *k_weight, int32_t weight_dtype,
    float eps, int32_t H_q, int32_t H_kv, int32_t D, int32_t block_size, void *q_out,
    void *stream) {
  CVSA_REQUIRE(k && v && k_cache && v_cache && block_tables && context_lens && cu_seqlens &&
                   (!q || q_out),
               CVSA_ERR_INVALID, "append_chunk_kv: null pointer argument");
  CVSA_REQUIRE(B > 0 && W > 0 && num_blocks > 0 && bt_stride_b >= W, CVSA_ERR_INVALID,
               "append_chunk_kv: bad sizes B=%d W=%d", B, W);
  CVSA_REQUIRE(block_size_supported(block_size), CVSA_ERR_UNSUPPORTED,
               "append_chunk_kv: block_size=%d not in {8, 16, 32, 64, 128}", block_size);
  CVSA_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0, CVSA_ERR_INVALID,
               "append_chunk_kv: caches must be 16-byte aligned");
  RotaryArgs a = {};
  a.k = k; a.k_st = k_stride_t; a.k_sh = k_stride_h;
  a.v = v; a.v_st = v_stride_t; a.v_sh = v_stride_h;
  if (q) {
    a.q = q; a.q_st = q_stride_t; a.q_sh = q_stride_h; a.q_out = q_out;
  }
  a.table = table; a.table_len = table_len; a.R = rot_dim;
  a.q_w = q ? q_weight : nullptr; a.k_w = k_weight; a.w_dtype = weight_dtype; a.eps = eps;
  a.tokens = tokens; a.H_q = H_q; a.H_kv = H_kv;
  a.k_cache = k_cache; a.v_cache = v_cache; a.num_blocks = num_blocks;
  a.block_tables = block_tables; a.bt_sb = bt_stride_b; a.W = W; a.block_size = block_size;
  a.B = B; a.context_lens = context_lens; a.cu = cu_seqlens;
  const int rc = check_rotary("append_chunk_kv", a, dtype, D, interleaved);
  if (rc != CVSA_OK) return rc;
  enqueue_rotary<true>(a, dtype, D, interleaved, stream);
  return cvsa_host::check_launch("append_chunk_kv");
}

extern "C" int cvsa_reserve_chunk(int32_t *block_tables, int64_t bt_stride_b, int32_t W,
                                  int32_t *context_lens, int32_t *pages_allocated,
                                  const int32_t *cu_seqlens, int32_t B, int32_t next_free_block,
                                  int64_t num_blocks, int32_t block_size, void *stream) {
  CVSA_REQUIRE(block_tables && context_lens && pages_allocated && cu_seqlens, CVSA_ERR_INVALID,
               "reserve_chunk: null pointer argument");
  CVSA_REQUIRE(B > 0 && W > 0 && num_blocks > 0 && bt_stride_b >= W && next_free_block >= 0,
               CVSA_ERR_INVALID, "reserve_chunk: bad sizes B=%d W=%d", B, W);
  CVSA_REQUIRE(block_size_supported(block_size), CVSA_ERR_UNSUPPORTED,
               "reserve_chunk: block_size=%d not in {8, 16, 32, 64, 128}", block_size);
  hipLaunchKernelGGL(reserve_chunk_kernel, dim3(1), dim3(kReserveThreads), 0,
                     (hipStream_t)stream, block_tables, bt_stride_b, W, context_lens,
                     pages_allocated, cu_seqlens, B, next_free_block, num_blocks, block_size);
  return cvsa_host::check_launch("reserve_chunk");
}
