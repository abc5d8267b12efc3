// Chunk attention of few rows (up to 64 of a sequence and KV head): single
// tokens, drafts, short chunks.  Reading K and V bounds it, so the kernel is
// made to keep loads in flight.
//
// Every wave of a workgroup has all the rows (RT tiles of 32) and takes its own
// tiles of 32 keys, in buffers of its own: two of K and two of V, no barrier
// in the walk.  K of tile s + 2 is requested once tile s has been multiplied, V
// likewise, so one to two tiles are under way at any time (64 to 128 KiB a CU
// at D = 128).  The waves' states are joined at the end.
//
// Sequences differ in length, so the keys of all of them are laid end to end (in
// units of 32 keys a wave, or of a sequence if none is longer) and cut into as
// many equal ranges as workgroups fit the GPU; a workgroup walks its range,
// sequence by sequence, for one KV head (the heads' workgroups read the same
// rows at about the same time).  Sequences that lie in one range are complete
// there; parts of the others are joined by a second kernel.  (Splits of equal
// length for each sequence, with rounds of workgroups, took 133 us where ranges
// take 113: 32 sequences of up to 8 K keys, 32 heads on 8 of 128.)
//
// Measured with the join, heads of 128: 32 sequences of 8 K keys, one token each,
// 193 us, 5.6 TB/s (a copy of 1 GB reaches 5.1); one sequence of 128 K keys 104 us,
// 5.2 TB/s; 8 drafts of 5 tokens at 32 K keys 112 us, 4.8 TB/s.  What is left is
// the kernel's start (6 us to the first products) and the join (5 to 7 us).  The
// decode kernels, which take single tokens only, need 88 us for the one sequence
// (14 for one of 8 K keys, 15 here), and keep the weights of the second product in
// two bf16 parts where these round them to one.
// Over 8 bits: a token each of 32 sequences of up to 8 K keys, 32 heads on 8, 63 us and
// 5 to join, 277 MB, 4.4 TB/s in the walk; 8 drafts of 5 tokens at 32 K keys, 28 heads
// on 4, 80 to 85 and 6, 269 MB.  The conversions to bf16 stand before each product there:
// with 35 rows they, the products and the loads' waits of a wave follow each other.  The
// weights are kept in two bf16 parts there too, as no decode kernel reads such caches:
// one part took 67.7 and 78 us with the join where two take 68.5 and 86 to 90 (the
// products of the second parts behind those of all the first, not between them: 91).
#pragma once
#include "chunk_common.h"

namespace cvsa {

template <int D, bool F8>
constexpr int chunk_stream_waves() {
  return D == 256 && !F8 ? 2 : 4;
}

// Over 8 bits each row tile has a workgroup of its own; those of the same keys run on
// one XCD, whose L2 the second reads, where the ranges and KV heads are a multiple of
// its 8 together.  (Both tiles in a wave: its registers are moved to and fro, and one
// wave to a SIMD takes its conversions, products and waits in turns: 8 drafts of 5
// tokens at 32 K keys, 28 heads on 4, with one part of the weights 77 us for 71.)
//
// Workgroups of a CU: by LDS one at D >= 128, two at 64; by registers at 32.  With
// two row tiles one at 64 as well, whose fewer parts gain more than twice the
// waves do: 61 us for 66 (8 drafts of 5 tokens at 32 K keys, 28 heads on 4).
template <int D, int RT, bool F8>
constexpr int chunk_stream_fit() {
  if (F8) return D == 256 ? 1 : 3 - RT;
  return D >= 128 ? 1 : D == 64 ? 3 - RT : 4 - RT;
}

template <int D, int RT, bool F8>
__global__ __launch_bounds__((chunk_stream_waves<D, F8>() * 64),
                             (chunk_stream_fit<D, RT, F8>())) void
chunk_stream_kernel(const ChunkArgs a, const ChunkClass cl) {
  constexpr int NW = chunk_stream_waves<D, F8>(), NT = NW * 64, KT = 32;
  static_assert(!F8 || RT == 1, "8 bits: a workgroup for each row tile");
  constexpr int DV = F8 ? D / 2 : D;           // a row's bytes are those of DV bf16 values
  constexpr int CPR = DV / 8, RPL = 64 / CPR;  // rows of a load
  constexpr int P = KT / RPL;                  // loads of a tile of K or V
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int kTile = KT * DV;
  __shared__ __align__(16) uint16_t s_k0[NW * kTile], s_k1[NW * kTile], s_v0[NW * kTile],
      s_v1[NW * kTile];
  __shared__ float2 s_ml[NW - 1][RT * 32];
  __shared__ ChunkTaken<D> s_taken;

  const int tid = threadIdx.x;
  // Over 8 bits the heads of a range go to one XCD: each of its rows has 128 bytes at
  // D = 128, and an XCD that reads all heads' draws on all of its L2's channels (plain
  // reads of such rows: 5.2 TB/s with an XCD for each head, 5.6 so).  This holds for
  // numbers of ranges that are multiples of the 8 XCDs, as powers of two of KV heads
  // give over many keys; with others (3 heads: 170) a range's heads are spread.
  const uint32_t n_ranges = gridDim.x / a.H_kv;
  const uint32_t range = F8 ? blockIdx.x % n_ranges : blockIdx.x / a.H_kv;
  const ChunkSeq first = chunk_look(a, cl, tid & 63);
  uint32_t total = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave)
    total += __builtin_amdgcn_readfirstlane(wave_sum_u32(
        (uint32_t)(b0 == 0 ? first : chunk_look(a, cl, b0 + (tid & 63))).units));
  const ChunkRanges ranges(cl, total);
  if (range >= ranges.n) return;
  const uint32_t begin = ranges.start(range), end = ranges.start(range + 1);

  // Units u0 .. u1 of a sequence.
  auto walk = [&](const ChunkTile &t, int u0, int u1, int units) {
    // New to the compiler for each sequence, or it keeps everything that
    // follows from the lane and the head over the loop, and spills.
    int id = tid, h = F8 ? blockIdx.x / n_ranges : blockIdx.x % a.H_kv;
    asm volatile("" : "+v"(id), "+s"(h));
    const int lane = id & 63, wave = __builtin_amdgcn_readfirstlane(id >> 6);
    const int l31 = lane & 31, half = lane >> 5;
    const int k0 = max(u0 - cl.extra_units, 0) << cl.unit_log2;
    const int k1 = u1 < units ? (u1 - cl.extra_units) << cl.unit_log2 : t.keys;

    const int bs_mask = (1 << a.bs_log2) - 1;
    const int row_bytes = a.H_kv * DV * 2;
    const uint32_t block_bytes = (uint32_t)row_bytes << a.bs_log2;
    uint32_t row_off[P];  // of the lane's vector of each load, in the block of the load's rows
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int r = p * RPL + lane / CPR;
      row_off[p] = lane / CPR * row_bytes + (h * DV + chunk_swizzle<DV>(r, lane % CPR) * 8) * 2;
    }
    std::conditional_t<F8, ChunkPlaces8<D>, ChunkPlaces<D>> place;
    place.init(wave * kTile * 2);

    ChunkRow row[RT];
    chunk_bf16x8_t q[RT][KS];
    ChunkState<D> state[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      row[r] = chunk_row(a, t, h, t.row0 + r * 32 + l31, k1);
      chunk_load_q<D, F8>(a, t, row[r], q[r]);
      state[r].init();
    }
    const int full_keys = a.causal ? min(t.pos0 + t.row0 / a.G + 1, k1) : k1;  // all rows see

    const int32_t *const bt = a.block_tables + t.seq * a.bt_sb;

    // The wave's s-th tile; lane i (mod 32) looks up its key i.
    auto first_key = [&](int s) { return k0 + (s * NW + wave) * KT; };
    const int mine = k1 - k0 - wave * KT;
    const int steps = mine > 0 ? (mine + NW * KT - 1) / (NW * KT) : 0;
    auto lookup = [&](int s) { return bt[min((first_key(s) + l31) >> a.bs_log2, a.W - 1)]; };

    // A tile's K or V: block 0 in place of keys that are none (`at` in the key's
    // lane).  The rows of a load lie in one block, but for 16 rows of 8-token
    // pages (D = 32).
    auto request = [&](const uint16_t *cache, int s, int at, uint16_t *lds) {
      const uint32_t readable = s < steps ? block_bytes : 0;  // past the last tile: no fetch
#pragma unroll
      for (int p = 0; p < P; ++p) {
        uint16_t *const to = lds + wave * kTile + p * 512;
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (RPL <= 8) {
          chunk_load_lds(cache, __builtin_amdgcn_readlane(at, p * RPL), block_bytes, readable,
                         row_off[p], ((first_key(s) + p * RPL) & bs_mask) * row_bytes, to);
        } else {
          const int r = p * RPL + lane / CPR;
          const uint32_t blk = __shfl(at, r, 64);
          const char *from = (const char *)cache + (uint64_t)blk * block_bytes +
                             (uint32_t)(((first_key(s) + r) & bs_mask) * row_bytes) +
                             (h * DV + chunk_swizzle<DV>(r, lane % CPR) * 8) * 2;
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                           (__attribute__((address_space(3))) void *)to, 16, 0, 0);
        }
      }
    };

    s_taken.clear(NT);
    __syncthreads();

    int at2;                    // blocks of tile s + 2
    uint64_t key0, key1, key2;  // keys of tiles s to s + 2
    int found;                  // looked up of tile s + 3
    // 8 bits: bytes of the scales of the lane's key in tiles s to s + 2.
    uint32_t ks0 = 0, ks1 = 0, ks2 = 0, vs0 = 0, vs1 = 0, vs2 = 0;
    auto scale_of = [&](const uint8_t *scales, int at) {
      return (uint32_t)scales[(int64_t)at * a.H_kv + h];
    };
    auto locate = [&](int s, int looked_up, int &at) {
      const bool ok = first_key(s) + l31 < k1 && (uint32_t)looked_up < (uint32_t)a.num_blocks;
      at = ok ? looked_up : 0;
      return __ballot(ok);
    };
    auto step = [&](int s, uint16_t *k_cur, uint16_t *v_cur) {
      place.renew();
      const int ahead = lookup(s + 3);
      f32x16_t st[RT][1];
      auto k_product = [&](const uint4 &k, int ks) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
          st[r][0] = chunk_mfma(k, __builtin_bit_cast(uint4, q[r][ks]), ks ? st[r][0] : f32x16_t{});
      };
      if constexpr (F8) {
        const float scale = chunk_scale(ks0);
#pragma unroll
        for (int j = 0; j < DB; ++j) {
          const uint4 w = chunk_read_k((const char *)k_cur + place.k[j]);
          k_product(chunk_from_8(make_uint2(w.x, w.y), scale, scale), 2 * j);
          k_product(chunk_from_8(make_uint2(w.z, w.w), scale, scale), 2 * j + 1);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) k_product(place.read_k((const char *)k_cur, 0, ks), ks);
      }
      __builtin_amdgcn_sched_barrier(0);  // K has been read
      key2 = locate(s + 2, found, at2);
      request(a.k_cache, s + 2, at2, k_cur);
      if constexpr (F8) {
        ks2 = scale_of(a.k_scales, at2);
        vs2 = scale_of(a.v_scales, at2);
      }
      found = ahead;
      bool whole = first_key(s) + KT <= full_keys && ~key0 == 0;
      uint64_t bad_scale = 0;
      if constexpr (F8) {
        bad_scale = __ballot(vs0 == 255u);
        whole = whole && bad_scale == 0;
      }
      if (!whole) {
        // A branch to the compiler: it would make selects of it for every tile.
        if constexpr (F8) asm volatile("");
#pragma unroll
        for (int r = 0; r < RT; ++r) chunk_mask(st[r], key0, first_key(s), row[r].last_key);
      }
      uint4 pw[RT][F8 ? 4 : 2];  // 8 bits: the weights in two parts
#pragma unroll
      for (int r = 0; r < RT; ++r) state[r].weights(st[r], a.c, pw[r], [](int) {});
      if (!whole) {
        // The wave's vectors of V, as they were loaded; they have arrived once
        // the first of them has been waited for here.
#pragma unroll 1
        for (int p = 0; p < P; ++p) {
          const int r = p * RPL + lane / CPR;
          uint4 *const at = reinterpret_cast<uint4 *>(v_cur + wave * kTile + p * 512 + lane * 8);
          if constexpr (F8)
            s_taken.clean8(at, key0 >> r & 1, bad_scale >> r & 1, first_key(s) + r,
                           chunk_swizzle<DV>(r, lane % CPR) * 16);
          else
            s_taken.clean(at, key0 >> r & 1, first_key(s) + r,
                          chunk_swizzle<D>(r, lane % CPR) * 8);
        }
      }
      // 8 bits: a scale for 8 keys, which lie in one page; of keys that are none,
      // and of pages whose scale is NaN, the values are zeros now.
      const uint32_t mine = (key0 >> l31 & 1) && vs0 != 255u ? vs0 : 127u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float scale[2];
        if constexpr (F8) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            scale[i] = chunk_scale(__builtin_amdgcn_readlane(mine, 16 * j + 8 * i));
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          uint4 v;
          if constexpr (F8) v = chunk_from_8(chunk_read_v8((char *)v_cur + place.v[d] + 16 * j * D),
                                             scale[0], scale[1]);
          else v = place.read_v((char *)v_cur, j, d);
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            state[r].o[d] = chunk_mfma(v, pw[r][j], state[r].o[d]);
            if constexpr (F8) state[r].o[d] = chunk_mfma(v, pw[r][2 + j], state[r].o[d]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // V has been read
      request(a.v_cache, s + 2, at2, v_cur);
      key0 = key1;
      key1 = key2;
      ks0 = ks1;
      ks1 = ks2;
      vs0 = vs1;
      vs1 = vs2;
    };
    if (steps > 0) {
      int at;
      const int f0 = lookup(0), f1 = lookup(1);
      found = lookup(2);
      key0 = locate(0, f0, at);
      request(a.k_cache, 0, at, s_k0);
      if constexpr (F8) {
        ks0 = scale_of(a.k_scales, at);
        vs0 = scale_of(a.v_scales, at);
      }
      request(a.v_cache, 0, at, s_v0);
      key1 = locate(1, f1, at);
      request(a.k_cache, 1, at, s_k1);
      if constexpr (F8) {
        ks1 = scale_of(a.k_scales, at);
        vs1 = scale_of(a.v_scales, at);
      }
      request(a.v_cache, 1, at, s_v1);
      for (int s = 0; s < steps; s += 2) {
        step(s, s_k0, s_v0);
        if (s + 1 < steps) step(s + 1, s_k1, s_v1);
      }
      // No load may reach the buffers once they are the join's.
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0f70);
      asm volatile("" ::: "memory");
    }

    // The waves' states, joined in order by the first: an array of K or V for
    // each other wave, float4 i of row r at place i ^ (r % 8).
    static_assert(NW <= 4 && NW * kTile * 2 >= RT * 32 * D * 4, "room to join");
    auto room = [&](int w) {
      return reinterpret_cast<float4 *>(w == 1 ? s_k1 : w == 2 ? s_v0 : s_v1);
    };
    auto spot = [&](int r, int d, int g) {
      return (r * 32 + l31) * (D / 4) + ((8 * d + 2 * g + half) ^ (l31 & 7));
    };
#pragma unroll
    for (int r = 0; r < RT; ++r) state[r].finish();
    __syncthreads();
    if (wave > 0) {
      float4 *const so = room(wave);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (half == 0) s_ml[wave - 1][r * 32 + l31] = make_float2(state[r].m, state[r].l);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            so[spot(r, d, g)] = make_float4(state[r].o[d][4 * g], state[r].o[d][4 * g + 1],
                                             state[r].o[d][4 * g + 2], state[r].o[d][4 * g + 3]);
      }
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        for (int w = 1; w < NW; ++w) {
          const float4 *const so = room(w);
          const float2 ml = s_ml[w - 1][r * 32 + l31];
          const float nm = fmaxf(state[r].m, ml.x);
          const float a0 = nm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(state[r].m - nm);
          const float a1 = nm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - nm);
          state[r].m = nm;
          state[r].l = state[r].l * a0 + ml.y * a1;
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            __builtin_amdgcn_sched_barrier(0);  // few reads at once: registers
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float4 v = so[spot(r, d, g)];
              state[r].o[d][4 * g] = state[r].o[d][4 * g] * a0 + v.x * a1;
              state[r].o[d][4 * g + 1] = state[r].o[d][4 * g + 1] * a0 + v.y * a1;
              state[r].o[d][4 * g + 2] = state[r].o[d][4 * g + 2] * a0 + v.z * a1;
              state[r].o[d][4 * g + 3] = state[r].o[d][4 * g + 3] * a0 + v.w * a1;
            }
          }
        }
        s_taken.restore(row[r].last_key, state[r].o);
        const int64_t part = (int64_t)(2 * (int)range + (k0 == 0)) * a.H_kv + h;
        if (k0 == 0 && u1 == units) state[r].store(a, t, row[r]);
        else state[r].store_part(cl, row[r], part * cl.tile_rows + t.row0 + r * 32 + l31);
      }
    }
    __syncthreads();  // the buffers and s_taken are the next sequence's
  };

  uint32_t before = 0;  // units
  for (int b0 = 0; b0 < a.B && before < end; b0 += kWave) {
    const ChunkSeq mine = b0 == 0 ? first : chunk_look(a, cl, b0 + (tid & 63));
    const uint32_t incl = wave_incl_scan_u32((uint32_t)mine.units);
    const uint32_t last = before + incl, start = last - mine.units;
    uint64_t todo = __ballot(mine.units > 0 && start < end && last > begin);
    while (todo != 0) {
      const int l = __builtin_ctzll(todo);
      todo &= todo - 1;
      ChunkTile t = {};
      t.seq = b0 + l;
      t.first = __builtin_amdgcn_readlane(mine.first, l);
      const int len = __builtin_amdgcn_readlane(mine.len, l);
      t.rows = len * a.G;
      t.pos0 = __builtin_amdgcn_readlane(mine.ctx, l) - len;
      t.keys = __builtin_amdgcn_readlane(mine.keys, l);
      const int units = __builtin_amdgcn_readlane(mine.units, l);
      const uint32_t from = before + __builtin_amdgcn_readlane(incl, l) - units;
      const int u1 = end < from + units ? (int)(end - from) : units;
      if (u1 <= cl.extra_units) continue;  // none of its keys
      if constexpr (F8) {
        t.row0 = blockIdx.y * 32;
        if (t.row0 >= t.rows) continue;
      }
      walk(t, (int)(begin > from ? begin - from : 0), u1, units);
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
}

}  // namespace cvsa
