// Chunk attention of many rows (more than 64 of a sequence and KV head): the
// products bound it.
//
// D = 64 and 128: a workgroup takes 256 rows, eight waves, two to a SIMD; steps
// of 64 keys.  With all waves in step both waves of a SIMD want the matrix pipe
// at once and then the vector pipe at once; so the second four run half a step
// behind the first, with a barrier after each half: while one wave multiplies (V
// of step s, K of step s + 1: 32 products of 32 cycles at D = 128) the other
// makes weights (about 110 vector instructions, 32 of them exponentials, and
// as long).  8192 rows of 32 heads over up to 16384 keys, D = 128: 1357 us,
// 1225 TFLOP/s, against 1758 us in step (a large bf16 matrix product of the
// library reaches 1375 TFLOP/s).  What keeps the halves short:
//  - LDS reads run four products ahead, in the source's order;
//  - the loads of the next keys stand between the products, one every fifth,
//    or between the weights: issued together they hold the wave up 350 cycles;
//  - a load takes the address of its rows' one block and a constant offset per
//    lane, no 64-bit arithmetic in lanes;
//  - no maximum in a step (see weights()).
//
// D = 32 and 256: a workgroup takes 128 rows, four waves in step, each its own
// overlap.  4096 tokens after as many, 32 heads on 8: 179 us at D = 32 (vector
// instructions active in 77% of the cycles, the matrix pipe in 26%) and 1028 at D =
// 256 (802 TFLOP/s; vector 43%, matrix 33%, LDS 17%: no pipe is full, the one wave
// of a SIMD takes them in turns).
//
// 128 rows also at D = 64 for prompts from near their start: smaller tiles waste
// less of the causal mask and end closer together, though a step takes longer:
// 2048 tokens from the start 34 us for 40, 16 prompts of up to 1000 after 2000 175
// for 189, but 4096 tokens after as many 243 for 231 (32 heads on 8).
//
// Over 8 bits: K and V come into registers, are made bf16 and written to the same
// places of LDS, a step ahead; the products are the same.  8192 tokens after as many,
// 32 heads on 8 of 128, 1395 us, 1191 TFLOP/s (bf16: 1357 above); 512 after 130560 922
// us and 8 to join, 1200.  (Bytes straight into LDS and made bf16 at each read: every
// wave would convert all of the workgroup's keys.)
#pragma once
#include "chunk_common.h"

namespace cvsa {

template <int D>
constexpr int chunk_step_keys() {
  return D == 256 ? 32 : 64;
}

// A thread's share of a step's 8-bit K or V: BYTES of them (8 or 16, of one row),
// loaded into registers and written to LDS as bf16.
template <int BYTES>
struct ChunkRaw {
  uint32_t w[BYTES / 4];
  uint32_t scale;  // its byte

  // From byte off of block blk; the block's scale of the head is `scales` on.
  __device__ __forceinline__ void load(const uint16_t *cache, const uint8_t *scales, int blk,
                                       uint32_t block_bytes, uint32_t off, int H_kv) {
    const char *p = (const char *)cache + (uint64_t)blk * block_bytes + off;
    if constexpr (BYTES == 16) {
      const uint4 v = *reinterpret_cast<const uint4 *>(p);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2 *>(p);
      w[0] = v.x; w[1] = v.y;
    }
    scale = scales[(int64_t)blk * H_kv];
  }
  // To columns col .. of row r of a bf16 tile.
  template <int D>
  __device__ __forceinline__ void store(uint16_t *tile, int r, int col) const {
    const float s = chunk_scale(scale);
#pragma unroll
    for (int i = 0; i < BYTES / 8; ++i)
      *reinterpret_cast<uint4 *>(tile + r * D + chunk_swizzle<D>(r, col / 8 + i) * 8) =
          chunk_from_8(make_uint2(w[2 * i], w[2 * i + 1]), s, s);
  }
};

// NW waves with 32 rows each.  F8: K and V are of 8 bits.  Nothing but their way
// into LDS differs: they pass through registers, where the matrix instructions'
// bf16 is made of them once for all rows of the workgroup (16 conversions and 4
// LDS writes a wave and step at D = 128), and are loaded a step earlier for it.
template <int D, int NW, bool F8>
__global__ __launch_bounds__(NW * 64, D == 256 ? 1 : D == 32 ? 3 : 2) void
chunk_prefill_kernel(const ChunkArgs a, const ChunkClass cl) {
  constexpr int NT = NW * 64, KT = chunk_step_keys<D>();
  constexpr int CPR = D / 8, NC = KT * CPR;
  constexpr int P = NC / NT;  // vectors of K and of V per thread and step
  // 8 bits: values of a load, threads of a row, loads per thread and step.
  constexpr int EV = KT * D / NT < 16 ? 8 : 16, TPR = D / EV, P8 = KT * D / NT / EV;
  constexpr int KB = KT / 32, KS = D / 16, DB = D / 32;
  static_assert(NC % NT == 0, "a step's vectors");
  constexpr int kStage = KT * D;  // elements of a step's K or V
  // Four arrays of their own: a load into one does not hold up reads of another.
  __shared__ __align__(16) uint16_t s_k0[kStage], s_k1[kStage], s_v0[kStage], s_v1[kStage];
  __shared__ ChunkTaken<D> s_taken;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // KV heads vary fastest: workgroups go round the XCDs, so one XCD's cache
  // sees the keys of few heads.
  int id = blockIdx.x;
  const int h = id % a.H_kv;
  id /= a.H_kv;
  const int split = id % cl.splits;
  const ChunkTile t = chunk_find_tile<NW * 32>(a, cl, id / cl.splits);
  const int k0 = split * cl.split_len;
  // The last split also takes keys past the plan's bound.
  const int k1 = split < cl.splits - 1 ? min(t.keys, k0 + cl.split_len) : t.keys;
  if (cl.splits > 1 && k0 >= k1) return;
  const int steps = k1 > k0 ? (k1 - k0 + KT - 1) / KT : 0;

  const int32_t *const bt = a.block_tables + t.seq * a.bt_sb;
  const int bs_mask = (1 << a.bs_log2) - 1;
  const int row_bytes = a.H_kv * D * (F8 ? 1 : 2);
  const uint32_t block_bytes = (uint32_t)row_bytes << a.bs_log2;

  // Blocks.  Lane i looks up key i of a step for the whole wave, a step ahead
  // of the loads; where there is no key or no block of the pool, its bit of the
  // step's key mask is clear and block 0 is read in its place.
  auto lookup_keys = [&](int s) {
    return bt[min((k0 + s * KT + (lane & (KT - 1))) >> a.bs_log2, a.W - 1)];
  };
  // All of the first lookups are under way before the first is waited for, and
  // before Q.
  const int found0 = lookup_keys(0), found1 = lookup_keys(1), found2 = lookup_keys(2);
  const int found3 = F8 && NW == 8 ? lookup_keys(3) : 0;

  const bool live = t.row0 + wave * 32 < t.rows;  // the wave has rows
  const ChunkRow row = chunk_row(a, t, h, t.row0 + wave * 32 + (lane & 31), k1);
  const int full_keys = a.causal ? min(t.pos0 + t.row0 / a.G + 1, k1) : k1;  // all rows see
  chunk_bf16x8_t q[KS];
  chunk_load_q<D>(a, t, row, q);

  // Barrier after the wave's LDS accesses, its loads left in flight.
  auto barrier = []() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  s_taken.clear(NT);
  barrier();

  ChunkState<D> state;
  state.init();

  auto in_pool = [&](int s, int found) {
    return k0 + s * KT + (lane & (KT - 1)) < k1 && (uint32_t)found < (uint32_t)a.num_blocks;
  };
  // V of a step that some row sees in part, or with keys that are none; each
  // thread looks after the vectors that it loaded.
  auto whole = [&](int s, uint64_t keys) { return k0 + (s + 1) * KT <= full_keys && ~keys == 0; };
  auto clean = [&](int s, uint64_t keys, uint16_t *lds) {
    if (whole(s, keys)) return;
    if constexpr (F8) {
      unrolled<P>([&](auto pi) {
        constexpr int i = decltype(pi)::value % (EV / 8);
        const int c = tid + decltype(pi)::value / (EV / 8) * NT, r = c / TPR;
        const int ch = c % TPR * (EV / 8) + i;
        s_taken.clean(reinterpret_cast<uint4 *>(lds + r * D + chunk_swizzle<D>(r, ch) * 8),
                      keys >> r & 1, k0 + s * KT + r, ch * 8);
      });
    } else {
      unrolled<P>([&](auto pi) {
        const int c = tid + decltype(pi)::value * NT, r = c / CPR;
        s_taken.clean(reinterpret_cast<uint4 *>(lds + c * 8), keys >> r & 1, k0 + s * KT + r,
                      chunk_swizzle<D>(r, c % CPR) * 8);
      });
    }
  };
  // Every load of this wave has arrived.
  auto arrived = []() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" ::: "memory");
  };
  ChunkPlaces<D> at;
  at.init(0);

  if constexpr (NW == 8) {
    // V of one step, then K of the next.  The order is the source's: the LDS
    // reads run kAhead products ahead, and between(i) follows product i.
    auto multiply = [&](char *v, const char *k, const uint4 (&pw)[2 * KB], f32x16_t (&st)[KB],
                        auto between) {
      at.renew();
      constexpr int NV = 2 * KB * DB, N = NV + KB * KS, kAhead = 4;
      uint4 f[kAhead + 1];
      auto fetch = [&](auto n) {
        constexpr int i = decltype(n)::value;
        if constexpr (i < NV) {
          constexpr int j = i / DB, d = i % DB;
          f[i % (kAhead + 1)] =
              at.read_v(v, j, d);
        } else if constexpr (i < N) {
          constexpr int ks = (i - NV) / KB, kb = (i - NV) % KB;
          f[i % (kAhead + 1)] = at.read_k(k, kb, ks);
        }
      };
      unrolled<kAhead>(fetch);
      __builtin_amdgcn_sched_barrier(0);
      unrolled<N>([&](auto at) {
        constexpr int i = decltype(at)::value;
        const uint4 x = f[i % (kAhead + 1)];
        if constexpr (i < NV) {
          constexpr int j = i / DB, d = i % DB;
          state.o[d] = chunk_mfma(x, pw[j], state.o[d]);
        } else {
          constexpr int ks = (i - NV) / KB, kb = (i - NV) % KB;
          st[kb] = chunk_mfma(x, __builtin_bit_cast(uint4, q[ks]), ks ? st[kb] : f32x16_t{});
        }
        fetch(std::integral_constant<int, i + kAhead>());
        between(at);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    auto first_scores = [&](const uint16_t *lds, f32x16_t (&st)[KB]) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          st[kb] = chunk_mfma(at.read_k((const char *)lds, kb, ks),
                              __builtin_bit_cast(uint4, q[ks]), ks ? st[kb] : f32x16_t{});
    };

    // The rows of one load of the wave (4 at D = 128, 8 at D = 64) lie in one
    // block, the rows of a step at the same places of their blocks in every
    // step, or every other one (128-token pages: steps of 64 keys start at
    // multiples of 64).
    static_assert(KT == 64 && 64 / CPR <= 8, "a lane per key, a block per load");
    uint32_t row_off[P];  // of the thread's vectors, in a block
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = tid + p * NT, r = c / CPR;
      row_off[p] = (r & bs_mask) * row_bytes + (h * D + chunk_swizzle<D>(r, c % CPR) * 8) * 2;
    }
    const uint32_t odd_off = a.bs_log2 == 7 ? 64 * row_bytes : 0;
    // 8 bits: eight threads of a row, so a wave's rows lie in one block too.
    static_assert(!F8 || (TPR == 8 && P8 == 1), "a block per load");
    const int r8 = tid / 8, c8 = tid % 8 * EV;
    const uint32_t off8 = (r8 & bs_mask) * row_bytes + h * D + c8;
    ChunkRaw<EV> raw_k, raw_v;
    auto load8 = [&](const uint16_t *cache, const uint8_t *scales, int blk, int odd) {
      ChunkRaw<EV> x;
      x.load(cache, scales + h, blk, block_bytes, off8 + (odd ? odd_off : 0), a.H_kv);
      return x;
    };
    auto locate8 = [&](int s, int found, int &blk) {
      const bool ok = in_pool(s, found);
      blk = __builtin_amdgcn_readlane(ok ? found : 0, wave * 8);
      return __ballot(ok);
    };
    auto locate = [&](int s, int found, uint32_t (&blk)[P]) {
      const bool ok = in_pool(s, found);
      const int at = ok ? found : 0;
#pragma unroll
      for (int p = 0; p < P; ++p)
        blk[p] = __builtin_amdgcn_readlane(at, (p * NT + wave * 64) / CPR);
      return __ballot(ok);
    };
    auto load = [&](const uint16_t *cache, uint32_t blk, int odd, uint16_t *lds, int p) {
      chunk_load_lds(cache, blk, block_bytes, block_bytes, row_off[p], odd ? odd_off : 0,
                     lds + (p * NT + wave * 64) * 8);
    };

    // In halves of the first four waves, step s makes weights in half 2 s and
    // multiplies in half 2 s + 1.  Buffers of V of step s - 1 and K of step s
    // are free after half 2 s; in half 2 s + 1 both groups start the loads of V
    // of step s + 1 and K of step s + 2 into them, each among what it computes
    // then, and after half 2 s + 2 both have waited for theirs.  Of 8-bit values
    // they write these into them then, loaded a step before, and start the loads of
    // the step after.
    static_assert(P <= KB, "a load to 16 keys' weights");
    constexpr int kEvery = (2 * KB * DB + KB * KS) / (2 * P) < 5
                               ? (2 * KB * DB + KB * KS) / (2 * P) : 5;  // products to a load
    auto walk = [&](auto late_group) {
      constexpr bool LATE = decltype(late_group)::value;
      f32x16_t st[KB];
      uint32_t blk1[P], blk2[P];  // of steps s + 1 and s + 2
      uint64_t key0, key1, key2;  // keys of steps s to s + 2
      int found;                  // blocks of step s + 2 (8 bits: s + 3)
      uint64_t key3 = 0;          // 8 bits: keys and blocks of steps s + 2 and s + 3
      int blk_v = 0, blk_k = 0;
      auto step = [&](int s, auto parity, uint16_t *k_cur, uint16_t *k_next, uint16_t *v_cur,
                      uint16_t *v_next) {
        constexpr int A = decltype(parity)::value;
        // The i-th of the 2 P loads that step s starts.
        auto next_load = [&](int i) {
          if constexpr (F8) {
            if (i == 0) {
              raw_v.template store<D>(v_next, r8, c8);
              raw_v = load8(a.v_cache, a.v_scales, blk_v, A);
            } else if (i == 1) {
              raw_k.template store<D>(k_cur, r8, c8);
              raw_k = load8(a.k_cache, a.k_scales, blk_k, 1 - A);
            }
          } else if (i < P) load(a.v_cache, blk1[i], 1 - A, v_next, i);
          else if (i < 2 * P) load(a.k_cache, blk2[i - P], A, k_cur, i - P);
        };
        auto next_blocks = [&]() {
          if constexpr (F8) {
            key3 = locate8(s + 3, found, blk_k);
            found = lookup_keys(s + 4);
          } else {
            key2 = locate(s + 2, found, blk2);
            found = lookup_keys(s + 3);
          }
        };
        uint4 pw[2 * KB];
        if (LATE) next_blocks();
        if (live) {
          if (!whole(s, key0)) chunk_mask(st, key0, k0 + s * KT, row.last_key);
          state.weights(st, a.c, pw, [&](int j) {
            if (LATE) {
              next_load(j);
              __builtin_amdgcn_sched_barrier(0);
            }
          });
        } else if (LATE) {
#pragma unroll
          for (int i = 0; i < 2 * P; ++i) next_load(i);
        }
        if (!LATE) {
          if (!F8) arrived();
          clean(s, key0, v_cur);
        }
        barrier();
        if (!LATE) next_blocks();
        if (live) {
          __builtin_amdgcn_s_setprio(1);
          multiply((char *)v_cur, (const char *)k_next, pw, st, [&](auto at) {
            constexpr int i = decltype(at)::value;
            if (!LATE && i % kEvery == kEvery / 2) next_load(i / kEvery);
          });
          __builtin_amdgcn_s_setprio(0);
        } else if (!LATE) {
#pragma unroll
          for (int i = 0; i < 2 * P; ++i) next_load(i);
        }
        if (LATE) {
          if (!F8) arrived();
          clean(s + 1, key1, v_next);
        }
        barrier();
#pragma unroll
        for (int p = 0; p < P; ++p) blk1[p] = blk2[p];
        key0 = key1;
        key1 = key2;
        if constexpr (F8) {
          key2 = key3;
          blk_v = blk_k;
        }
      };
      if constexpr (F8) {
        int b0, b1;
        key0 = locate8(0, found0, b0);
        key1 = locate8(1, found1, b1);
        key2 = locate8(2, found2, blk_v);
        raw_k = load8(a.k_cache, a.k_scales, b0, 0);
        const ChunkRaw<EV> v0 = load8(a.v_cache, a.v_scales, b0, 0);
        const ChunkRaw<EV> k1 = load8(a.k_cache, a.k_scales, b1, 1);
        raw_k.template store<D>(s_k0, r8, c8);
        raw_v = load8(a.v_cache, a.v_scales, b1, 1);
        raw_k = load8(a.k_cache, a.k_scales, blk_v, 0);
        v0.template store<D>(s_v0, r8, c8);
        k1.template store<D>(s_k1, r8, c8);
        found = found3;
      } else {
        key0 = locate(0, found0, blk2);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          load(a.k_cache, blk2[p], 0, s_k0, p);
          load(a.v_cache, blk2[p], 0, s_v0, p);
        }
        key1 = locate(1, found1, blk1);
#pragma unroll
        for (int p = 0; p < P; ++p) load(a.k_cache, blk1[p], 1, s_k1, p);
        found = found2;
        arrived();
      }
      if (LATE) clean(0, key0, s_v0);
      barrier();
      if (live) first_scores(s_k0, st);
      if (LATE) barrier();
      for (int s = 0; s < steps; s += 2) {
        step(s, std::integral_constant<int, 0>(), s_k0, s_k1, s_v0, s_v1);
        if (s + 1 < steps)
          step(s + 1, std::integral_constant<int, 1>(), s_k1, s_k0, s_v1, s_v0);
      }
      if (!LATE) barrier();
      if (!F8) arrived();  // no load may outlive the workgroup's LDS
    };
    if (steps > 0) {
      if (wave >= 4) walk(std::true_type());
      else walk(std::false_type());
    }
  } else {
    // One wave to a SIMD, so its own instructions have to fill both pipes: in
    // step s the products of K of step s + 1 stand between the exponentials of
    // step s; then V of step s is added.  K of step s + 2 and V of step s + 1
    // are under way meanwhile.  The rows of a load lie in one block, but for 16
    // rows of 8-token pages (D = 32), where lanes carry whole addresses.
    constexpr int RPL = 64 / CPR;
    uint32_t row_off[P];  // of the lane's vector of each load, in the block of the load's rows
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int r = (p * NT + tid) / CPR;
      row_off[p] = lane / CPR * row_bytes + (h * D + chunk_swizzle<D>(r, lane % CPR) * 8) * 2;
    }
    auto load_one = [&](const uint16_t *cache, int s, int at, uint16_t *lds, int p) {
      uint16_t *const to = lds + (p * NT + wave * 64) * 8;
      if constexpr (RPL <= 8) {
        const int r = (p * NT + wave * 64) / CPR;
        chunk_load_lds(cache, __builtin_amdgcn_readlane(at, r), block_bytes,
                       s < steps ? block_bytes : 0, row_off[p],
                       ((k0 + s * KT + r) & bs_mask) * row_bytes, to);
      } else {
        const int c = tid + p * NT, r = c / CPR;
        const uint32_t blk = __shfl(at, r, 64);
        const char *from = (const char *)cache + (uint64_t)blk * block_bytes +
                           (uint32_t)(((k0 + s * KT + r) & bs_mask) * row_bytes) +
                           (h * D + chunk_swizzle<D>(r, c % CPR) * 8) * 2;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                         (__attribute__((address_space(3))) void *)to, 16, 0, 0);
      }
    };
    auto load = [&](const uint16_t *cache, int s, int at, uint16_t *lds) {
#pragma unroll
      for (int p = 0; p < P; ++p) load_one(cache, s, at, lds, p);
    };
    // 8 bits: into registers in the step before the one that starts by writing
    // them to LDS.
    ChunkRaw<EV> raw_k[P8], raw_v[P8];
    auto load8 = [&](const uint16_t *cache, const uint8_t *scales, int s, int at,
                     ChunkRaw<EV> (&x)[P8]) {
#pragma unroll
      for (int p = 0; p < P8; ++p) {
        const int c = tid + p * NT, r = c / TPR;
        x[p].load(cache, scales + h, __shfl(at, r, 64), block_bytes,
                  ((k0 + s * KT + r) & bs_mask) * row_bytes + h * D + c % TPR * EV, a.H_kv);
      }
    };
    auto store8 = [&](const ChunkRaw<EV> (&x)[P8], uint16_t *lds) {
#pragma unroll
      for (int p = 0; p < P8; ++p) {
        const int c = tid + p * NT;
        x[p].template store<D>(lds, c / TPR, c % TPR * EV);
      }
    };
    constexpr int NK = KB * KS, NV = 2 * KB * DB, NE = 16 * KB, kAhead = 4;
    uint4 f[kAhead + 1];
    auto fetch_k = [&](const char *k, auto n) {
      constexpr int i = decltype(n)::value, ks = i / KB, kb = i % KB;
      if constexpr (i < NK) f[i % (kAhead + 1)] = at.read_k(k, kb, ks);
    };
    auto k_product = [&](auto at, f32x16_t (&st)[KB]) {
      constexpr int i = decltype(at)::value, ks = i / KB, kb = i % KB;
      st[kb] = chunk_mfma(f[i % (kAhead + 1)], __builtin_bit_cast(uint4, q[ks]),
                          ks ? st[kb] : f32x16_t{});
    };
    auto scores = [&](const uint16_t *k, f32x16_t (&st)[KB]) {
      unrolled<kAhead>([&](auto i) { fetch_k((const char *)k, i); });
      unrolled<NK>([&](auto at) {
        k_product(at, st);
        fetch_k((const char *)k, std::integral_constant<int, decltype(at)::value + kAhead>());
      });
    };
    // Weights of st between the products of the next scores.
    auto weights_and_scores = [&](const f32x16_t (&st)[KB], uint4 (&pw)[2 * KB], const char *k,
                                  f32x16_t (&nxt)[KB]) {
      unrolled<kAhead>([&](auto i) { fetch_k(k, i); });
      float sum[4] = {0.f, 0.f, 0.f, 0.f}, even = 0.f;
      uint32_t words[NE / 2];
      unrolled<NE>([&](auto at) {
        constexpr int e = decltype(at)::value;
        // products e NK / NE up to (e + 1) NK / NE
        constexpr int i0 = e * NK / NE, i1 = (e + 1) * NK / NE;
        unrolled<i1 - i0>([&](auto n) {
          constexpr int i = i0 + decltype(n)::value;
          k_product(std::integral_constant<int, i>(), nxt);
          fetch_k(k, std::integral_constant<int, i + kAhead>());
        });
        const float p = __builtin_amdgcn_exp2f(fmaf(st[e / 16][e % 16], a.c, state.neg_m));
        sum[e % 4] += p;
        if constexpr (e % 2 == 0) even = p;
        else words[e / 2] = chunk_cvt_bf16x2(even, p);
        __builtin_amdgcn_sched_barrier(0);
      });
#pragma unroll
      for (int j = 0; j < 2 * KB; ++j)
        pw[j] = make_uint4(words[4 * j], words[4 * j + 1], words[4 * j + 2], words[4 * j + 3]);
      state.settle(st, a.c, pw, (sum[0] + sum[1]) + (sum[2] + sum[3]));
    };
    auto accumulate = [&](char *v, const uint4 (&pw)[2 * KB]) {
      auto fetch = [&](auto n) {
        constexpr int i = decltype(n)::value, j = i / DB, d = i % DB;
        if constexpr (i < NV)
          f[i % (kAhead + 1)] =
              at.read_v(v, j, d);
      };
      unrolled<kAhead>(fetch);
      __builtin_amdgcn_sched_barrier(0);
      unrolled<NV>([&](auto at) {
        constexpr int i = decltype(at)::value, j = i / DB, d = i % DB;
        state.o[d] = chunk_mfma(f[i % (kAhead + 1)], pw[j], state.o[d]);
        fetch(std::integral_constant<int, i + kAhead>());
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    int at1, found;             // blocks of step s + 1; looked up of step s + 2
    uint64_t key0, key1, key2;  // keys of steps s to s + 2
    auto locate = [&](int s, int looked_up, int &at) {
      const bool ok = in_pool(s, looked_up);
      at = ok ? looked_up : 0;
      return __ballot(ok);
    };
    auto step = [&](int s, uint16_t *k_cur, uint16_t *k_next, uint16_t *v_cur, uint16_t *v_next,
                    f32x16_t (&cur)[KB], f32x16_t (&nxt)[KB]) {
      at.renew();
      if constexpr (F8) {
        store8(raw_v, v_cur);
        store8(raw_k, k_next);
      } else {
        arrived();
      }
      clean(s, key0, v_cur);
      barrier();
      int at2;
      key2 = locate(s + 2, found, at2);
      found = lookup_keys(s + 3);
      if constexpr (F8) {
        load8(a.v_cache, a.v_scales, s + 1, at1, raw_v);
        load8(a.k_cache, a.k_scales, s + 2, at2, raw_k);
      } else {
        load(a.v_cache, s + 1, at1, v_next);
        load(a.k_cache, s + 2, at2, k_cur);
      }
      at1 = at2;
      if (live) {
        if (!whole(s, key0)) chunk_mask(cur, key0, k0 + s * KT, row.last_key);
        uint4 pw[2 * KB];
        weights_and_scores(cur, pw, (const char *)k_next, nxt);
        accumulate((char *)v_cur, pw);
      }
      key0 = key1;
      key1 = key2;
    };
    if (steps > 0) {
      f32x16_t st0[KB], st1[KB];
      int at0;
      found = found2;
      key0 = locate(0, found0, at0);
      key1 = locate(1, found1, at1);
      if constexpr (F8) {
        load8(a.k_cache, a.k_scales, 0, at0, raw_k);
        load8(a.v_cache, a.v_scales, 0, at0, raw_v);
        store8(raw_k, s_k0);
        load8(a.k_cache, a.k_scales, 1, at1, raw_k);
      } else {
        load(a.k_cache, 0, at0, s_k0);
        load(a.v_cache, 0, at0, s_v0);
        if (steps > 1) load(a.k_cache, 1, at1, s_k1);
        arrived();
      }
      barrier();
      if (live) scores(s_k0, st0);
      for (int s = 0; s < steps; s += 2) {
        step(s, s_k0, s_k1, s_v0, s_v1, st0, st1);
        if (s + 1 < steps) step(s + 1, s_k1, s_k0, s_v1, s_v0, st1, st0);
      }
      if (!F8) arrived();  // no load may outlive the workgroup's LDS
    }
  }
  __syncthreads();  // the last note of a taken-out value

  state.finish();
  s_taken.restore(row.last_key, state.o);
  if (cl.splits > 1 && (k0 > 0 || k1 < t.keys))
    state.store_part(cl, row, ((int64_t)split * cl.tokens + t.part0 + row.tok) * a.H_q + row.head);
  else
    state.store(a, t, row);
}

}  // namespace cvsa
