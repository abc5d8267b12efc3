// What the kernels that norm and rotate rows share: arguments, vectors, the norm
// and the rotation of a row, and the walk over the rows of tokens.
#pragma once
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

// The lane's two vectors of a row (lane j of the D / 16 that share it), both
// members of every rotated pair among them, and whether they are rotated.
template <int D, bool PAIRS>
struct RotaryPlace {
  int c0, c1;
  bool r0, r1;

  __device__ __forceinline__ RotaryPlace(const RotaryArgs &a, int j) {
    if (PAIRS) {
      c0 = j;
      c1 = j + D / 16;
      r0 = c0 < a.R / 8;
      r1 = c1 < a.R / 8;
    } else {
      const int hc = a.R / 16;  // vectors of a rotated half
      r0 = r1 = j < hc;
      c0 = r0 ? j : 2 * j;      // past the rotated ones: 2 hc + 2 (j - hc)
      c1 = r0 ? j + hc : 2 * j + 1;
    }
  }
  // Cosines and sines of the lane's pairs; NaN at a position that the table
  // does not hold.
  __device__ __forceinline__ void angles(const RotaryArgs &a, int64_t pos, float (&cs)[8],
                                         float (&sn)[8]) const {
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
  }
  // The norm of the row (weight null: none).
  __device__ __forceinline__ void norm(const RotaryArgs &a, const void *weight, float (&f0)[8],
                                       float (&f1)[8]) const {
    if (!weight) return;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(f0[e], f0[e], ss);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(f1[e], f1[e], ss);
    ss = group_sum<D / 16>(ss);
    const float inv = rsqrtf(ss * (1.f / D) + a.eps);
    float w0[8], w1[8];
    load_weights(weight, a.w_dtype, c0 * 8, w0);
    load_weights(weight, a.w_dtype, c1 * 8, w1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f0[e] = f0[e] * inv * w0[e];
      f1[e] = f1[e] * inv * w1[e];
    }
  }
  __device__ __forceinline__ void turn(const float (&cs)[8], const float (&sn)[8], float (&f0)[8],
                                       float (&f1)[8]) const {
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
};

// x or y, whose values are given: a choice by the lane among members of the arguments
// becomes a load from a chosen address, and all of them go into scratch memory for it
// (8 ragged prompts, 19 K tokens into a bf16 cache: 221 us for 84).
template <class T>
__device__ __forceinline__ T rotary_pick(bool first, T x, T y) {
  return first ? x : y;
}

constexpr int kRotaryThreads = 256;
constexpr int kRotaryBatch = 3;  // passes whose rows are requested together

// Wave w of a launch over rows; Q_ONLY: there are none but the queries'.
template <class T, int D, bool PAIRS, bool APPEND, bool ONCE, bool Q_ONLY = false>
__device__ __forceinline__ void rotary_rows(const RotaryArgs &a, int64_t w) {
  constexpr int LR = D / 16;   // lanes of a row
  constexpr int RW = 64 / LR;  // rows of a pass
  constexpr int ES = Vec8<T>::kSize;
  const int lane = threadIdx.x & 63;
  const int t = __builtin_amdgcn_readfirstlane((int)(w / a.segs));
  const int g0 = __builtin_amdgcn_readfirstlane((int)(w % a.segs)) * a.per_wave;
  if (t >= a.tokens) return;
  const int g_end = min(g0 + a.per_wave, a.groups);
  const int j = lane % LR, sub = lane / LR;
  // A token's rows: passes over the heads of q, then passes over those of k
  // and, with APPEND, v behind them.
  const int gq = a.q ? (a.H_q + RW - 1) / RW : 0;
  auto row_of = [&](int g, int &head) {  // 0: q, 1: k, 2: v, -1: none
    if (Q_ONLY || g < gq) {
      head = g * RW + sub;
      return head < a.H_q ? 0 : -1;
    }
    head = (g - gq) * RW + sub;
    if (head < a.H_kv) return 1;
    head -= a.H_kv;
    return APPEND && head < a.H_kv ? 2 : -1;
  };

  const RotaryPlace<D, PAIRS> at(a, j);

  // Lanes without a row read the token's first.
  auto source = [&](int g) -> const char * {
    int head;
    const int kind = row_of(g, head);
    const bool q = Q_ONLY || g < gq, v = kind == 2;
    const int64_t st = rotary_pick(q, a.q_st, rotary_pick(v, a.v_st, a.k_st));
    const int64_t sh = rotary_pick(q, a.q_sh, rotary_pick(v, a.v_sh, a.k_sh));
    return (const char *)rotary_pick(q, a.q, rotary_pick(v, a.v, a.k)) +
           (t * st + (kind < 0 ? 0 : head) * sh) * ES;
  };

  Vec8<T> x0[kRotaryBatch], x1[kRotaryBatch];
  auto request = [&](int gb) {
#pragma unroll
    for (int u = 0; u < kRotaryBatch; ++u) {
      if (gb + u < g_end) {
        const char *p = source(gb + u);
        x0[u].load(p + at.c0 * 8 * ES);
        x1[u].load(p + at.c1 * 8 * ES);
      }
    }
  };
  request(g0);

  int64_t pos;
  int64_t slot = -1;  // token's row in the cache, -1: not written
  if constexpr (APPEND) {
    const int b = last_that(a.B, [&](int b) { return a.cu[b] <= t; });
    const int place = a.context_lens[b] - (a.cu[b + 1] - t);
    pos = place;
    if (place >= 0) {
      const int page = place / a.block_size;
      if (page < a.W) {
        const int blk = a.block_tables[b * a.bt_sb + page];
        if (blk >= 0 && blk < a.num_blocks)
          slot = (int64_t)blk * a.block_size + (place - page * a.block_size);
      }
    }
  } else {
    pos = !a.positions ? 0
          : a.wide     ? static_cast<const int64_t *>(a.positions)[t]
                       : static_cast<const int32_t *>(a.positions)[t];
  }

  float cs[8], sn[8];
  at.angles(a, pos, cs, sn);

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
        at.norm(a, Q_ONLY || g < gq ? a.q_w : a.k_w, f0, f1);
        if (a.table) at.turn(cs, sn, f0, f1);
      }
      if (kind < 0) continue;
      if (Q_ONLY || kind == 0 || !APPEND) {
        char *p = Q_ONLY || kind == 0 ? (char *)a.q_out + ((int64_t)t * a.H_q + head) * D * ES
                            : (char *)a.k_out + ((int64_t)t * a.H_kv + head) * D * ES;
        Vec8<T>::template store<ONCE>(p + at.c0 * 8 * ES, f0);
        Vec8<T>::template store<ONCE>(p + at.c1 * 8 * ES, f1);
      } else if (slot >= 0) {
        uint16_t *p = rotary_pick(kind == 1, a.k_cache, a.v_cache) + (slot * a.H_kv + head) * D;
        Vec8<Bf16>::store<ONCE>((char *)(p + at.c0 * 8), f0);
        Vec8<Bf16>::store<ONCE>((char *)(p + at.c1 * 8), f1);
      }
    }
  }
}

// What the entry points ask of their rows, table and weights.
int check_rotary(const char *who, const RotaryArgs &a, int32_t dtype, int32_t D,
                 int32_t interleaved);
// Waves of a launch over the rows of a.tokens tokens; sets a.groups, a.per_wave and
// a.segs.  once: its outputs are stored past the caches.
int64_t rotary_waves(RotaryArgs &a, int D, bool append, bool &once);

}  // namespace cvsa
