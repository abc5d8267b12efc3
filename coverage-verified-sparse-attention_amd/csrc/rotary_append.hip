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
#include "cvsa_common.h"

#include <type_traits>

namespace cvsa {

struct RotaryArgs {
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // token and head strides, in elements
  void *q_out, *k_out;                         // contiguous [tokens, heads, D]
  const float *table;                          // [table_len, R]: cosines, then sines
  int64_t table_len;
  int R;
  const void *q_w, *k_w;
  int w_dtype;
  float eps;
  int tokens, H_q, H_kv;
  int groups, per_wave, segs;  // passes of a token, of a wave, waves of a token
  const void *positions;       // without APPEND: int32 or, wide, int64
  bool wide;
  // APPEND
  uint16_t *k_cache, *v_cache;
  int64_t num_blocks;
  const int32_t *block_tables;
  int64_t bt_sb;
  int W, block_size, B;
  const int32_t *context_lens, *cu;
};

struct Bf16 {};
struct Fp16 {};

// 16 bytes stored; ONCE: not to be kept in the caches.
template <bool ONCE>
__device__ __forceinline__ void store16(char *p, const uint4 &w) {
  typedef unsigned v4u_t __attribute__((ext_vector_type(4)));
  const v4u_t v = {w.x, w.y, w.z, w.w};
  if constexpr (ONCE) __builtin_nontemporal_store(v, reinterpret_cast<v4u_t *>(p));
  else *reinterpret_cast<v4u_t *>(p) = v;
}

// 8 elements of a row as 32-bit floats, and back.
template <class T>
struct Vec8;

template <>
struct Vec8<Bf16> {
  static constexpr int kSize = 2;
  uint4 w;
  __device__ __forceinline__ void load(const char *p) { w = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = bf16_lo(w.x); f[1] = bf16_hi(w.x); f[2] = bf16_lo(w.y); f[3] = bf16_hi(w.y);
    f[4] = bf16_lo(w.z); f[5] = bf16_hi(w.z); f[6] = bf16_lo(w.w); f[7] = bf16_hi(w.w);
  }
  template <bool ONCE>
  static __device__ __forceinline__ void store(char *p, const float (&f)[8]) {
    store16<ONCE>(p, make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])));
  }
};

template <>
struct Vec8<Fp16> {
  static constexpr int kSize = 2;
  uint4 w;
  __device__ __forceinline__ void load(const char *p) { w = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const h8 h = __builtin_bit_cast(h8, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)h[e];
  }
  template <bool ONCE>
  static __device__ __forceinline__ void store(char *p, const float (&f)[8]) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    h8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (_Float16)f[e];
    store16<ONCE>(p, __builtin_bit_cast(uint4, h));
  }
};

template <>
struct Vec8<float> {
  static constexpr int kSize = 4;
  float4 a, b;
  __device__ __forceinline__ void load(const char *p) {
    a = reinterpret_cast<const float4 *>(p)[0];
    b = reinterpret_cast<const float4 *>(p)[1];
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  template <bool ONCE>
  static __device__ __forceinline__ void store(char *p, const float (&f)[8]) {
    store16<ONCE>(p, __builtin_bit_cast(uint4, make_float4(f[0], f[1], f[2], f[3])));
    store16<ONCE>(p + 16, __builtin_bit_cast(uint4, make_float4(f[4], f[5], f[6], f[7])));
  }
};

__device__ __forceinline__ void load_weights(const void *w, int dtype, int at, float (&f)[8]) {
  if (dtype == CVSA_DTYPE_FP32) {
    Vec8<float> v;
    v.load((const char *)w + at * 4);
    v.get(f);
  } else if (dtype == CVSA_DTYPE_FP16) {
    Vec8<Fp16> v;
    v.load((const char *)w + at * 2);
    v.get(f);
  } else {
    Vec8<Bf16> v;
    v.load((const char *)w + at * 2);
    v.get(f);
  }
}

constexpr int kRotaryThreads = 256;
constexpr int kRotaryBatch = 3;  // passes whose rows are requested together

template <class T, int D, bool PAIRS, bool APPEND, bool ONCE>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryArgs a) {
  constexpr int LR = D / 16;   // lanes of a row
  constexpr int RW = 64 / LR;  // rows of a pass
  constexpr int ES = Vec8<T>::kSize;
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * (kRotaryThreads / kWave) + (threadIdx.x >> 6);
  const int t = __builtin_amdgcn_readfirstlane((int)(w / a.segs));
  const int g0 = __builtin_amdgcn_readfirstlane((int)(w % a.segs)) * a.per_wave;
  if (t >= a.tokens) return;
  const int g_end = min(g0 + a.per_wave, a.groups);
  const int j = lane % LR, sub = lane / LR;
  // A token's rows: passes over the heads of q, then passes over those of k
  // and, with APPEND, v behind them.
  const int gq = a.q ? (a.H_q + RW - 1) / RW : 0;
  auto row_of = [&](int g, int &head) {  // 0: q, 1: k, 2: v, -1: none
    if (g < gq) {
      head = g * RW + sub;
      return head < a.H_q ? 0 : -1;
    }
    head = (g - gq) * RW + sub;
    if (head < a.H_kv) return 1;
    head -= a.H_kv;
    return APPEND && head < a.H_kv ? 2 : -1;
  };

  // The lane's two vectors of a row, and whether they are rotated.
  int c0, c1;
  bool r0, r1;
  if (PAIRS) {
    c0 = j;
    c1 = j + LR;
    r0 = c0 < a.R / 8;
    r1 = c1 < a.R / 8;
  } else {
    const int hc = a.R / 16;  // vectors of a rotated half
    r0 = r1 = j < hc;
    c0 = r0 ? j : 2 * j;      // past the rotated ones: 2 hc + 2 (j - hc)
    c1 = r0 ? j + hc : 2 * j + 1;
  }

  // Lanes without a row read the token's first.
  auto source = [&](int g) -> const char * {
    int head;
    const int kind = row_of(g, head);
    const bool q = g < gq, v = kind == 2;
    const int64_t st = q ? a.q_st : v ? a.v_st : a.k_st, sh = q ? a.q_sh : v ? a.v_sh : a.k_sh;
    return (const char *)(q ? a.q : v ? a.v : a.k) + (t * st + (kind < 0 ? 0 : head) * sh) * ES;
  };

  Vec8<T> x0[kRotaryBatch], x1[kRotaryBatch];
  auto request = [&](int gb) {
#pragma unroll
    for (int u = 0; u < kRotaryBatch; ++u) {
      if (gb + u < g_end) {
        const char *p = source(gb + u);
        x0[u].load(p + c0 * 8 * ES);
        x1[u].load(p + c1 * 8 * ES);
      }
    }
  };
  request(g0);

  int64_t pos;
  int64_t slot = -1;  // token's row in the cache, -1: not written
  if constexpr (APPEND) {
    // The sequence of token t: the last b with cu[b] <= t, 64 candidates a
    // look.
    int b = 0, n = a.B;
    while (n > 1) {
      const int step = (n + 63) / 64;
      const bool le = lane * step < n && a.cu[b + lane * step] <= t;
      const int k = __popcll(__ballot(le)) - 1;
      b += k * step;
      n = min(step, n - k * step);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    const int at = a.context_lens[b] - (a.cu[b + 1] - t);
    pos = at;
    if (at >= 0) {
      const int page = at / a.block_size;
      if (page < a.W) {
        const int blk = a.block_tables[b * a.bt_sb + page];
        if (blk >= 0 && blk < a.num_blocks)
          slot = (int64_t)blk * a.block_size + (at - page * a.block_size);
      }
    }
  } else {
    pos = !a.positions ? 0
          : a.wide     ? static_cast<const int64_t *>(a.positions)[t]
                       : static_cast<const int32_t *>(a.positions)[t];
  }

  // Cosines and sines of the lane's pairs; NaN at a position that the table
  // does not hold.
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) cs[e] = sn[e] = __builtin_nanf("");
  if (a.table && pos >= 0 && pos < a.table_len) {
    const float *row = a.table + pos * a.R;
    const int half = a.R / 2;
    if (PAIRS) {  // 4 pairs of each vector
      if (r0) {
        const float4 c = *reinterpret_cast<const float4 *>(row + 4 * c0);
        const float4 s = *reinterpret_cast<const float4 *>(row + half + 4 * c0);
        cs[0] = c.x; cs[1] = c.y; cs[2] = c.z; cs[3] = c.w;
        sn[0] = s.x; sn[1] = s.y; sn[2] = s.z; sn[3] = s.w;
      }
      if (r1) {
        const float4 c = *reinterpret_cast<const float4 *>(row + 4 * c1);
        const float4 s = *reinterpret_cast<const float4 *>(row + half + 4 * c1);
        cs[4] = c.x; cs[5] = c.y; cs[6] = c.z; cs[7] = c.w;
        sn[4] = s.x; sn[5] = s.y; sn[6] = s.z; sn[7] = s.w;
      }
    } else if (r0) {  // 8 pairs across the two vectors
      Vec8<float> c, s;
      c.load((const char *)(row + 8 * c0));
      s.load((const char *)(row + half + 8 * c0));
      c.get(cs);
      s.get(sn);
    }
  }
  if (!a.table) r0 = r1 = false;

  for (int gb = g0; gb < g_end; gb += kRotaryBatch) {
    if (gb != g0) request(gb);
#pragma unroll
    for (int u = 0; u < kRotaryBatch; ++u) {
      const int g = gb + u;
      if (g >= g_end) break;
      int head;
      const int kind = row_of(g, head);
      float f0[8], f1[8];
      x0[u].get(f0);
      x1[u].get(f1);
      if (kind != 2) {
        const void *wt = g < gq ? a.q_w : a.k_w;
        if (wt) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(f0[e], f0[e], ss);
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(f1[e], f1[e], ss);
          ss = group_sum<LR>(ss);
          const float inv = rsqrtf(ss * (1.f / D) + a.eps);
          float w0[8], w1[8];
          load_weights(wt, a.w_dtype, c0 * 8, w0);
          load_weights(wt, a.w_dtype, c1 * 8, w1);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f0[e] = f0[e] * inv * w0[e];
            f1[e] = f1[e] * inv * w1[e];
          }
        }
        if (PAIRS) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (r0) {
              const float x = f0[2 * e], y = f0[2 * e + 1];
              f0[2 * e] = x * cs[e] - y * sn[e];
              f0[2 * e + 1] = y * cs[e] + x * sn[e];
            }
            if (r1) {
              const float x = f1[2 * e], y = f1[2 * e + 1];
              f1[2 * e] = x * cs[4 + e] - y * sn[4 + e];
              f1[2 * e + 1] = y * cs[4 + e] + x * sn[4 + e];
            }
          }
        } else if (r0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = f0[e], y = f1[e];
            f0[e] = x * cs[e] - y * sn[e];
            f1[e] = y * cs[e] + x * sn[e];
          }
        }
      }
      if (kind < 0) continue;
      if (kind == 0 || !APPEND) {
        char *p = kind == 0 ? (char *)a.q_out + ((int64_t)t * a.H_q + head) * D * ES
                            : (char *)a.k_out + ((int64_t)t * a.H_kv + head) * D * ES;
        Vec8<T>::template store<ONCE>(p + c0 * 8 * ES, f0);
        Vec8<T>::template store<ONCE>(p + c1 * 8 * ES, f1);
      } else if (slot >= 0) {
        uint16_t *p = (kind == 1 ? a.k_cache : a.v_cache) + (slot * a.H_kv + head) * D;
        Vec8<Bf16>::store<ONCE>((char *)(p + c0 * 8), f0);
        Vec8<Bf16>::store<ONCE>((char *)(p + c1 * 8), f1);
      }
    }
  }
}

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

template <class T, int D, bool APPEND>
static void launch_rotary(const RotaryArgs &a, int pairs, bool once, hipStream_t s) {
  const int64_t waves = (int64_t)a.tokens * a.segs;
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
static void launch_rotary_d(const RotaryArgs &a, int D, int pairs, bool once, hipStream_t s) {
  if (D == 32) launch_rotary<T, 32, APPEND>(a, pairs, once, s);
  else if (D == 64) launch_rotary<T, 64, APPEND>(a, pairs, once, s);
  else if (D == 128) launch_rotary<T, 128, APPEND>(a, pairs, once, s);
  else launch_rotary<T, 256, APPEND>(a, pairs, once, s);
}

// Passes of a token and how many a wave takes: all of them once the tokens
// alone make enough waves to fill the GPU (2048), one otherwise.  With so many
// tokens the outputs are also stored past the caches: 8191 tokens of 28 + 4 heads
// of 128 take 29.7 us, 35.6 with ordinary stores.  The rule looks at the tokens
// alone, not at the bytes.  2047 tokens (neither) and 2048 (both), heads of 128:
// 1 + 1 heads 10.3 and 10.1 us, 32 + 8 10.6 and 10.0, 128 + 16 27.2 and 27.1, and
// 64 + 8 heads of fp32, whose 75 MB in and 75 MB out fit the last-level cache from
// pass to pass, 26.0 and 32.4.
template <bool APPEND>
static void enqueue_rotary(RotaryArgs &a, int dtype, int D, int pairs, void *stream) {
  const int rows = 64 / (D / 16);
  a.groups = (a.q ? (a.H_q + rows - 1) / rows : 0) +
             (a.k ? (a.H_kv * (APPEND ? 2 : 1) + rows - 1) / rows : 0);
  const bool once = a.tokens >= 2048;
  a.per_wave = once ? a.groups : 1;
  a.segs = (a.groups + a.per_wave - 1) / a.per_wave;
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == CVSA_DTYPE_BF16) launch_rotary_d<Bf16, APPEND>(a, D, pairs, once, s);
  else if (dtype == CVSA_DTYPE_FP16) launch_rotary_d<Fp16, APPEND>(a, D, pairs, once, s);
  else launch_rotary_d<float, APPEND>(a, D, pairs, once, s);
}

}  // namespace cvsa

using namespace cvsa;

static bool dtype_ok(int32_t t) {
  return t == CVSA_DTYPE_BF16 || t == CVSA_DTYPE_FP16 || t == CVSA_DTYPE_FP32;
}

// What both entry points ask of their rows, table and weights.
static int check_rotary(const char *who, const RotaryArgs &a, int32_t dtype, int32_t D,
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
