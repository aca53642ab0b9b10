// Attention over the pages of a key/value cache: its kernels, how they split the work, and their launches. Compiled for the fp16
// cache (PagedCache, paged.hip) and for the one in 8 bits (PagedCache8, paged8.hip).
#pragma once
#include <algorithm>

#include "decode_split.h"
#include "flash.h"
#include "paged.h"
#include "paged_plan.h"
#include "row_overlap.h"

HI_EXPORT size_t hi_attn_paged_work_bytes(int M, int B, int Hq, int Hkv, int D, int ragged);

namespace {

// ------------------------------------------------------------------ attention
//
// o = sum_k w_k v_k, w_k = 2^(x_k - m) / l, x the logits times log2(e) / sqrt(D). Logits, m, l, O and the parts that splits
// exchange are fp32. The 2^(x_k - m) are rounded to fp16 for the product with V, as in the slot cache's kernels, for its matrix
// instructions take no fp32: 2^-11 of each weight at most (the error against 64 bits becomes 2.5e-4 to 2.9e-4 of the result, 2.1e-4
// with fp32 weights and the result rounded alone), and a weight under 2^-25 of the largest that its wave has seen becomes 0: in all at
// most 2^-25 sum |v| of the keys.
// An infinity or NaN in a V row reaches the rows that see its key and no other: as itself, or as NaN where its weight has become 0.
struct AttnArgs {
  const f16* q;
  int64_t ldq;
  f16* out;
  int64_t ldo;
  float* lse;  // [Hq][M] or null
  const int *start, *pos;
  int M, B, Hq, Hkv, shared;  // positions below `shared` are on the pages of table row 0
  int G;                      // Hq / Hkv, and what divides by it (plan_token)
  uint32_t magic;
  float scale_log2;
};

// ---- row runs (and the common part of a shared prefix)
//
// Block = (unit, kv head): 32 RG packed rows, i.e. the G query heads of a kv head in 32 RG / G tokens, against a range of
// keys, with the tile loop of the slot cache's prefill attention (prefill.hip, flash_tile.h): packing reads K and V once for the
// group's heads and fills the tile where a run has few tokens. What paging changes:
//  * 8 keys from a multiple of 8 lie on one page, and a DMA instruction covers 4 or 8 keys. So each instruction has a
//    buffer descriptor of its own for its 8 keys: base from the page id, range from the keys that are left (0 for no page: zeros).
//    A wave's entries of tile t + 3 are loaded, a lane each, while tile t is computed, made into offsets and lengths by
//    those lanes, and read out of them as scalars; lane offsets inside the 8 keys never change;
//  * page ids outside the cache: found in one pass over the block's entries before the loop; only a block that has some takes
//    the masked tile for all of its keys, and hides them there.
// Where the row tiles are fewer than the GPU's CUs, their keys are split (paged_plan.h). A split stores its unnormalised O, m
// and l in fp32, in the lanes' order; of each kFan splits of a tile the block that arrives last joins them, of each kFan such
// groups the last again, until one block has the tile. Nobody waits. A launch of its own for the joins, us: 7 prompt
// chunks of 1 to 411 rows 28.9 (here 26.3), and 3 more for every small batch.
// What bounds it: 2048 rows after 4096 positions (32/8 heads of 128) 178 us, 965 TFLOP/s (the slot cache's kernel 174); smaller
// batches a chain of about 12 us around their tiles: start and pos, the plan, the table, the first K tile (2 to 3 us), the
// parts' stores, arrival and join (5 us). Few rows: attn_rows_kernel.
struct FlashPlan {
  float *ml, *po;  // partial results: [slot][2][BQ] m and l, O [slot][RG][D / 8][64][4], a prefix's [slot][BQ][D]
  int slots;       // slots there are, each of all kv heads
  int cus, b1, b2; // > 0: split over that many; plan_budget's quotients
  int least, fan;  // key tiles that a split has at least, splits that a tile has at most (0: any)
  int splits;      // of the shared prefix
  int* counters;   // [slots * Hkv], arrivals of a tile's splits
};

// What a block works on; found by every wave by itself from start and pos.
struct FlashUnit {
  int b, row0, n, pos;   // sequence, its first row, rows, first position
  int tile, splits, split, slot;  // slot of split 0 (meaningful with splits > 1)
};

// Integer reductions over a whole wave in DPP moves (a __shfl_xor is an LDS round trip, and a plan has dozens).
template <int CTRL>
__device__ __forceinline__ int dpp_or(int old, int v) {  // lanes without a source get `old`
  return __builtin_amdgcn_update_dpp(old, v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ int wave_total(int v) {
  v += dpp_or<0xB1>(0, v);   // quad_perm [1,0,3,2]
  v += dpp_or<0x4E>(0, v);   // quad_perm [2,3,0,1]
  v += dpp_or<0x141>(0, v);  // row_half_mirror
  v += dpp_or<0x140>(0, v);  // row_mirror
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
         __builtin_amdgcn_readlane(v, 48);
}
__device__ __forceinline__ int wave_most(int v) {
  v = max(v, dpp_or<0xB1>(v, v));
  v = max(v, dpp_or<0x4E>(v, v));
  v = max(v, dpp_or<0x141>(v, v));
  v = max(v, dpp_or<0x140>(v, v));
  return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive sum
  v += dpp_or<0x111>(0, v);  // row_shr 1, 2, 4, 8
  v += dpp_or<0x112>(0, v);
  v += dpp_or<0x114>(0, v);
  v += dpp_or<0x118>(0, v);
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31), r2 = __builtin_amdgcn_readlane(v, 47);
  return v + (lane >= 16 ? r0 : 0) + (lane >= 32 ? r1 : 0) + (lane >= 48 ? r2 : 0);
}

// Unit `at` of the batch; false if there are not so many. Wave-uniform.
template <int BQ>
__device__ __forceinline__ bool flash_unit(const AttnArgs& a, int cap, const FlashPlan& f, int at, int lane, FlashUnit& u) {
  struct Seq { int row0, n, pos, tiles, te; };  // te: key tiles
  auto seq = [&](int b) {
    Seq s{0, 0, 0, 0, 0};
    if (b < a.B) {
      const int s0 = a.start[b], s1 = a.start[b + 1];
      s.pos = a.pos[b];
      s.row0 = plan_first(s0, a.M);
      s.n = plan_rows(s0, s1, a.M);
      s.tiles = plan_tiles(s.n, a.G, BQ);
      s.te = plan_key_tiles(plan_end(s.pos, s.n, cap));
    }
    return s;
  };
  int L = kPlanNoSplit;
  const Seq first = seq(lane);
  if (f.cus > 0) {
    int T = 0, longest = 0;
    uint32_t work = 0;  // in key tiles; under the budget's T < 2 cus it does not overflow
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const Seq s = b0 ? seq(b0 + lane) : first;
      T += s.tiles;
      work += (uint32_t)s.tiles * (uint32_t)s.te;
      if (s.tiles) longest = max(longest, s.te);
    }
    T = wave_total(T);
    const int budget = plan_budget(T, a.Hkv, f.cus, f.b1, f.b2);
    if (budget > 0) {
      longest = wave_most(longest);
      L = plan_length((uint32_t)wave_total((int)work), budget, f.least);
      if (f.fan > 0) L = max(L, plan_div(longest + f.fan - 1, f.fan));
      for (; L < longest; L = plan_longer(L)) {
        int units = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
          const Seq s = b0 ? seq(b0 + lane) : first;
          units += s.tiles * plan_splits(s.te, L);
        }
        if (wave_total(units) <= min(budget, f.slots)) break;
      }
    }
  }
  int before = 0, slot = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Seq s = b0 ? seq(b0 + lane) : first;
    const int splits = plan_splits(s.te, L);
    const int n = s.tiles * splits, own = splits > 1 ? n : 0;
    const int upto = wave_scan(n, lane);
    const uint64_t hit = __ballot(before + upto > at);
    const int slots = f.cus > 0 ? wave_scan(own, lane) : 0;
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto take = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      u.b = b0 + l;
      u.row0 = take(s.row0);
      u.n = take(s.n);
      u.pos = take(s.pos);
      u.splits = take(splits);
      const int tiles = take(s.tiles), i = at - before - (take(upto) - take(n));
      const int down = u.splits == 1 ? i : plan_div(i, u.splits);
      u.tile = tiles - 1 - down;  // the most keys first
      u.split = i - down * u.splits;
      u.slot = slot + take(slots) - take(own) + u.tile * u.splits;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    slot += __builtin_amdgcn_readlane(slots, 63);
  }
  return false;
}

constexpr int kFan = 8;  // splits that one block joins

// Partial results in 16-byte pieces (index i), past the L2s, which are not coherent with each other: sc1 (bit 4).
struct PartBuffer {
  __amdgpu_buffer_rsrc_t rs;
  __device__ __forceinline__ PartBuffer(float* p, size_t bytes)
      : rs(__builtin_amdgcn_make_buffer_rsrc(p, (short)0, (int)bytes, 0x00020000)) {}
  __device__ __forceinline__ void store(int64_t i, f32x4 v) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rs, (int)(i * 16), 0, 16);
  }
  __device__ __forceinline__ f32x4 load(int64_t i) const {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(i * 16), 0, 16));
  }
};

// The scale of kv head hk's V (or K) on page id, and one element's value.
template <bool V>
__device__ __forceinline__ float page_scale(const PagedCache&, int, int, int) { return 1.f; }
template <bool V>
__device__ __forceinline__ float page_scale(const PagedCache8& c, int id, int hk, int Hkv) {
  return exponent_scale((V ? c.vexp : c.kexp)[(int64_t)id * Hkv + hk]);
}
__device__ __forceinline__ float element(f16 v, float) { return (float)v; }
__device__ __forceinline__ float element(uint8_t v, float scale) {
  f16x2 lo{}, hi{};
  f8x4_to_f16(v, scale, lo, hi);
  return (float)lo[0];
}

// One block: kv head hk of unit `unit`, or with PREFIX split `unit` of row tile `tile` of the shared prefix.
template <int D, int RG, bool PREFIX, class C>
__device__ __forceinline__ void pages_block(const AttnArgs& a, const C& c, const FlashPlan& f, int hk, int unit, int tile) {
  constexpr int NW = 2 * RG, BQ = 32 * RG;
  constexpr int CPR = D / 8;                   // 16-byte chunks per key row
  constexpr int IPW = kFpBKV * CPR / 64 / NW;  // DMA instructions per wave per tile and operand
  constexpr int DT = D / 32;                   // 32-row output tiles of O^T
  constexpr int NQ = D / 16;                   // MFMAs of one 32-key block's logits
  constexpr int KPW = kFpBKV / NW;             // keys of a tile that a wave fetches
  constexpr int NG = KPW / 8;                  // in groups of 8, one page each
  constexpr int IPG = IPW / NG;                // DMA instructions per group
  static_assert(IPW * 64 * NW == kFpBKV * CPR && IPG * NG == IPW, "tile DMA split");
  using Sm = typename std::conditional<C::kF8, Fp8Smem<D, RG>, FpSmem<D, RG>>::type;
  extern __shared__ u32x4 fp_smem[];
  u32x4* const ks_ = fp_smem;                                // [2][kTile]: K stages
  u32x4* const vs_ = fp_smem + kFpStages * Sm::kTile;        // [2][kTile]: V stages
  f32x16* const mo = reinterpret_cast<f32x16*>(fp_smem);     // [RG][DT][64]: the merge
  float* const ml = reinterpret_cast<float*>(fp_smem + Sm::kMl);  // [2][RG][64]: the second waves' m and l
  int* const flag = reinterpret_cast<int*>(fp_smem + Sm::kFlag);  // [NW], before the loop

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wave % RG, kh = wave / RG;     // row group, key half
  const int fr = lane & 31, fk = lane >> 5;
  const int G = a.G, page = 1 << c.shift, cap = c.capacity();
  FlashUnit u;
  int end;     // keys that some row of the tile sees
  int kb, ke;  // the split's
  // of the next key tile to be located: this lane's group of 8 keys, and its page
  int key = wave * KPW + 8 * (lane & (NG - 1)), id, id1 = -1;  // (id1: of the tile after it, for the 8-bit cache's prologue)
  if constexpr (PREFIX) {
    u = FlashUnit{0, 0, a.M, 0, tile, f.splits, unit, 0};
    u.slot = u.tile * f.splits;
    plan_range(a.shared, u.splits, u.split, kb, ke);
    key += kb;
    id = key < ke ? c.entry(0, key >> c.shift) : -1;  // requested together with the positions
    int most = -1;  // the last position of any of the tile's rows
    for (int i = u.tile * BQ + lane; i < min((u.tile + 1) * BQ, u.n * G); i += 64) most = max(most, a.pos[plan_token(i, a.magic)]);
    end = max(min(wave_most(most), a.shared - 1), -1) + 1;
  } else {
    if (!flash_unit<BQ>(a, cap, f, unit, lane, u)) return;
    end = plan_tile_end(u.pos, u.n, u.tile, G, a.magic, BQ, cap);
    plan_range(end, u.splits, u.split, kb, ke);
    key += kb;
    id = key < ke ? c.entry(u.b, key >> c.shift) : -1;
    if constexpr (C::kF8) id1 = key + kFpBKV < ke ? c.entry(u.b, (key + kFpBKV) >> c.shift) : -1;
  }
  const int kv_end = min(ke, end);
  const int nt = kv_end > kb ? (kv_end - kb + kFpBKV - 1) / kFpBKV : 0;

  // this lane's row and the last key it sees
  const int pr = u.tile * BQ + rg * 32 + fr;
  const bool row = pr < u.n * G;
  const int token = row ? plan_token(pr, a.magic) : 0, h = hk * G + (row ? pr - token * G : 0);
  const int64_t qrow = u.row0 + token;
  int qpos = -1;
  if (row) qpos = PREFIX ? min(a.pos[token], a.shared - 1) : (int)min((int64_t)u.pos + token, (int64_t)cap - 1);

  float m_i = -__builtin_huge_valf(), l_i = 0.f;
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[dt][e] = 0.f;
  const int xaddr = (lane ^ 32) << 2;                          // lane l ^ 32, for ds_bpermute
  auto xor32 = [&](float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(xaddr, __builtin_bit_cast(int, v)));
  };
  if (nt > 0) {
    const float scale_log2 = a.scale_log2;
    // this lane's Q fragments: d = 16 ks + 8 fk + 0..7 (zero without a row)
    f16x8 qf[NQ];
#pragma unroll
    for (int ks = 0; ks < NQ; ks++) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (row) v = *reinterpret_cast<const u32x4*>(a.q + qrow * a.ldq + h * D + 16 * ks + 8 * fk);
      qf[ks] = __builtin_bit_cast(f16x8, v);
    }
    const int tb = PREFIX ? 0 : u.b;  // table row
    // the groups' byte offsets in kp / vp and readable bytes: of the next K tile, and of the next V tile (one before)
    constexpr int EB = sizeof(typename C::Elem);
    uint32_t klo[NG], khi[NG], vlo[NG], vhi[NG];
    int kn[NG], vn[NG];
    int ke = 0, ve = 0;  // F8: the exponents of the lane's group
    auto fetch = [&] { id = key < kv_end ? c.entry(tb, key >> c.shift) : -1; };
    auto take = [&] {
      const bool ok = c.has(id) && key < kv_end;
      const int64_t off = ok ? (id * c.stride + ((int64_t)hk * page + (key & (page - 1))) * D) * EB : 0;
      const int n = ok ? min(8, kv_end - key) * D * EB : 0;
      if constexpr (C::kF8) {
        const int64_t at = (ok ? (int64_t)id * a.Hkv : 0) + hk;
        ke = c.kexp[at];
        ve = c.vexp[at];
      }
#pragma unroll
      for (int g = 0; g < NG; g++) {
        klo[g] = __builtin_amdgcn_readlane((int)off, g);
        khi[g] = __builtin_amdgcn_readlane((int)(off >> 32), g);
        kn[g] = __builtin_amdgcn_readlane(n, g);
      }
      key += kFpBKV;
    };
    auto group = [](const typename C::Elem* base, uint32_t lo, uint32_t hi, int n) {
      return __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<typename C::Elem*>(base) + (((uint64_t)hi << 32) | lo), (short)0, n,
                                               0x00020000);
    };
    constexpr int kFeed = C::kF8 ? kFeedWiden : kFeedDma;
    int koff[IPW], voff[IPW];
    auto next = [&] {
#pragma unroll
      for (int g = 0; g < NG; g++) {
        vlo[g] = klo[g];
        vhi[g] = khi[g];
        vn[g] = kn[g];
      }
      take();
      fetch();
    };
    // F8: a wave's share of a tile comes as codes (a group of 8 keys is D / 2 lanes of DMA) and is made into fp16 by the wave itself,
    // one tile before the others read it: no barrier more, and no registers held from tile to tile. The codes' place in LDS is free
    // again as soon as they are read, and the next tile's are sent for. One chunk goes behind each MFMA of the last block's P.V
    // (2048 rows behind 4096 positions, Hq 32, Hkv 8, D 128: 190 to 195 us by card, with all of them after those MFMAs 3 % more on
    // one card; the fp16 cache 184).
    constexpr int RPW = KPW * D / 1024;  // 16-byte reads of a lane per wave and operand, 2 chunks each
    int vexps = 0;  // the exponents of the V tile that lies there as codes; the K tile's are ke
    u32x4* const own_k = fp_smem + 2 * kFpStages * Sm::kTile + wave * RPW * 64;
    u32x4* const own_v = own_k + Sm::kTile / 2;
    u32x4 wk[RPW], wv[RPW];  // a tile's codes
    auto codes_to = [&](const typename C::Elem* base, const uint32_t (&lo)[NG], const uint32_t (&hi)[NG], const int (&n)[NG], u32x4* to) {
      if constexpr (C::kF8) {
#pragma unroll
        for (int g = 0; g < NG; g++)
          if (D == 128 || lane < 32) lds_dma16(group(base, lo[g], hi[g], n[g]), to + g * (D / 2), lane * 16);
      }
    };
    auto read_codes = [&](const u32x4* from, u32x4 (&w)[RPW]) {
#pragma unroll
      for (int i = 0; i < RPW; i++) w[i] = from[i * 64 + lane];
    };
    // Where a lane's first chunk goes in a K and a V tile, in bytes. The others' places follow from it by constants: the second
    // chunk of a read in bit 4, and at D = 128 K's second group of keys in the swizzle's bit 3. The asm below keeps the compiler
    // from holding each place in a register of its own for the whole loop, where it then spilled 16 (100 rows behind 4000
    // positions, Hq 32, Hkv 8: 29.5 us with those, 28.0 without).
    const int key0 = wave * KPW + lane / (D / 16), piece0 = lane % (D / 16);
    const int k_put = 16 * (key0 * CPR + ((2 * piece0) ^ k_swz<D>(key0))), v_put = 16 * (key0 * CPR + ((2 * piece0) ^ v_swz<D>(key0)));
    static_assert(!C::kF8 || D == 64 || KPW % 16 == 0, "a wave's keys begin a period of the swizzle");
    auto widen = [&](int j, const u32x4 (&w)[RPW], int exps, u32x4* tile, int put, bool k) {  // chunk j of a lane's
      const int i = j / 2;
      float scale;
      if constexpr (D == 128) {
        scale = exponent_scale(__builtin_amdgcn_readlane(exps, i));
      } else {
        const int e0 = __builtin_amdgcn_readlane(exps, 2 * i), e1 = __builtin_amdgcn_readlane(exps, 2 * i + 1);
        scale = exponent_scale(lane < 32 ? e0 : e1);
      }
      asm("" : "+v"(put));
      const int at = (put ^ (16 * (j & 1)) ^ (k && D == 128 ? 128 * (i & 1) : 0)) + i * (1024 / D) * CPR * 16;
      const f16x8 x = j & 1 ? f8x8_to_f16(w[i][2], w[i][3], scale) : f8x8_to_f16(w[i][0], w[i][1], scale);
      *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(tile) + at) = __builtin_bit_cast(u32x4, x);
    };
    auto issue_k = [&](int i, int st) {
      if constexpr (C::kF8) widen(i, wk, ke, ks_ + st * Sm::kTile, k_put, true);
      else lds_dma16(group(c.kp, klo[i / IPG], khi[i / IPG], kn[i / IPG]), ks_ + st * Sm::kTile + (wave * IPW + i) * 64, koff[i]);
    };
    auto issue_v = [&](int i, int st) {
      if constexpr (C::kF8) widen(i, wv, vexps, vs_ + st * Sm::kTile, v_put, false);
      else lds_dma16(group(c.vp, vlo[i / IPG], vhi[i / IPG], vn[i / IPG]), vs_ + st * Sm::kTile + (wave * IPW + i) * 64, voff[i]);
    };
    auto codes_v = [&] {
      if constexpr (C::kF8) read_codes(own_v, wv);
    };
    auto refill = [&] {  // (the codes are read: their values have been used)
      if constexpr (C::kF8) {
        vexps = ve;
        asm volatile("" ::: "memory");
        next();
        codes_to(c.kp, klo, khi, kn, own_k);
        codes_to(c.vp, vlo, vhi, vn, own_v);
      }
    };
    auto advance = [&](int) {
      if constexpr (C::kF8) read_codes(own_k, wk);
      else next();
      __builtin_amdgcn_sched_barrier(0);
    };
    auto first_advance = [&] { advance(0); };
    if constexpr (C::kF8) {
      // K tiles 0 and 1 and V tile 0 at once (K tile 1's codes in the last V stage, which is free until tile 0 is computed), then K tile 2's
      // and V tile 1's codes on their way
      u32x4* const more_k = vs_ + Sm::kTile + wave * RPW * 64;
      take();
      id = id1;
      const int ke0 = ke, ve0 = ve;
      codes_to(c.kp, klo, khi, kn, own_k);
      codes_to(c.vp, klo, khi, kn, own_v);
      next();
      const int ke1 = ke, ve1 = ve;
      codes_to(c.kp, klo, khi, kn, more_k);
      wait_vmcnt<0>();
      asm volatile("" ::: "memory");
      u32x4 wm[RPW];
      read_codes(own_k, wk);
      read_codes(own_v, wv);
      read_codes(more_k, wm);
#pragma unroll
      for (int i = 0; i < IPW; i++) {
        widen(i, wk, ke0, ks_, k_put, true);
        widen(i, wv, ve0, vs_, v_put, false);
        widen(i, wm, ke1, ks_ + Sm::kTile, k_put, true);
      }
      ve = ve1;
      refill();
    } else {
      // DMA instruction i of this wave fills slots (wave IPW + i) * 64 + lane of a tile: slot s holds
      // key s / CPR, physical chunk s % CPR, i.e. logical chunk (s % CPR) ^ swz(key)
#pragma unroll
      for (int i = 0; i < IPW; i++) {
        const int s = (wave * IPW + i) * 64 + lane, r = s / CPR, p = s % CPR;
        koff[i] = ((r & 7) * D + 8 * (p ^ k_swz<D>(r))) * 2;
        voff[i] = ((r & 7) * D + 8 * (p ^ v_swz<D>(r))) * 2;
      }
      take();
      fetch();
    }
    // whether some key of the block lies on no page
    int hid[2], hi = (kb >> c.shift) + tid;
    const int h_last = (kv_end - 1) >> c.shift;
#pragma unroll
    for (int k = 0; k < 2; k++, hi += 128 * RG) hid[k] = hi <= h_last ? c.entry(tb, hi) : 0;
    // tiles at the front that all of this wave's rows see whole (none for a wave without rows), and the last key any sees
    int least = row ? min(qpos, kv_end - 1) : kv_end;
    least = -wave_most(-least);
    const int most = wave_most(qpos);
    bool holes = false;
    int n_full = most < 0 ? 0 : max(least + 1 - kb, 0) / kFpBKV;
    auto before_barrier = [&] {  // of the prologue
      bool hole = !c.has(hid[0]) || !c.has(hid[1]);
      for (; hi <= h_last; hi += 128 * RG) hole |= !c.has(c.entry(tb, hi));
      const bool some = __any(hole);
      if (lane == 0) flag[wave] = some;
      asm volatile("" ::: "memory");
      wait_lgkm0();
    };
    auto after_barrier = [&] {
#pragma unroll
      for (int w = 0; w < NW; w++) holes |= flag[w] != 0;
      holes = __builtin_amdgcn_readfirstlane(holes);
      if (holes) n_full = 0;
    };
    uint32_t seen = 0xff;  // which of the wave's 8 groups of a masked tile lie on pages
    auto enter_masked = [&](int t) {
      if (holes) {
        const int k = kb + t * kFpBKV + kFpKPW * kh + 8 * (lane & 7);
        seen = (uint32_t)__ballot(k < kv_end && c.has(c.entry(tb, k >> c.shift))) & 0xff;
      }
    };
    auto hidden = [&](int t, int kt, int e) {
      const int k = kb + t * kFpBKV + kFpKPW * kh + 32 * kt + 8 * (e >> 2) + 4 * fk + (e & 3);
      return k > qpos || !((seen >> (4 * kt + (e >> 2))) & 1);
    };
    auto live = [&](int t) {
      const int k0 = kb + t * kFpBKV + kFpKPW * kh;
      return k0 <= most && k0 < kv_end;
    };

    constexpr bool kGuard = true;
    int odd_tile = INT32_MAX;
#include "flash_tile.h"
    // the infinities and NaN of the masked tiles, key by key (rare: fp16 overflow in a V row)
#pragma unroll 1
    for (int ot = odd_tile; ot < nt; ot++) {
      const int k0 = kb + ot * kFpBKV + kFpKPW * kh;
#pragma unroll 1
      for (int k = k0; k < min(k0 + kFpKPW, kv_end); k++) {
        const int vid = c.entry(tb, k >> c.shift);
        if (!c.has(vid)) continue;
        const auto vrow = c.vp + vid * c.stride + ((int64_t)hk * page + (k & (page - 1))) * D + 4 * fk;
        const float vs = page_scale<true>(c, vid, hk, a.Hkv);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int g = 0; g < 4; g++) {
            typedef typename C::Elem x4 __attribute__((ext_vector_type(4)));
            const x4 x = *reinterpret_cast<const x4*>(vrow + dt * 32 + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float v = element(x[e], vs);
              if (k <= qpos && !(__builtin_fabsf(v) < __builtin_huge_valf())) o[dt][4 * g + e] += v;
            }
          }
      }
    }
  }

  // ---- merge the two key halves of each row group: the second wave hands (m, l, O) over
  wait_vmcnt<0>();
  __syncthreads();  // every wave is done with the stages, and no DMA is in flight
  const bool rg_empty = u.tile * BQ + rg * 32 >= u.n * G;  // a row group behind the run
  l_i += xor32(l_i);
  if (kh == 1) {
#pragma unroll
    for (int dt = 0; dt < DT; dt++) mo[(rg * DT + dt) * 64 + lane] = o[dt];
    ml[rg * 64 + lane] = m_i;
    ml[(RG + rg) * 64 + lane] = l_i;
  }
  __syncthreads();
  const bool parts = PREFIX || u.splits > 1;
  if (parts && u.slot + u.split >= f.slots) return;  // (not reached: the plan stays within the slots)
  const int64_t slot = (int64_t)(u.slot + u.split) * a.Hkv + hk;
  const PartBuffer po(f.po, (size_t)f.slots * a.Hkv * BQ * D * 4);
  if (kh == 0 && !rg_empty) {
    const float m1 = ml[rg * 64 + lane], l1 = ml[(RG + rg) * 64 + lane];
    const float m = fmaxf(m_i, m1), ref = m == -__builtin_huge_valf() ? 0.f : m;  // -inf: no key seen
    const float a0 = __builtin_amdgcn_exp2f(m_i - ref), a1 = __builtin_amdgcn_exp2f(m1 - ref);
    const float l = l_i * a0 + l1 * a1, inv = l == 0.f ? 0.f : 1.f / l;
    if (parts) {  // (lanes without a row store what their zero queries gave; nothing reads it)
      if (fk == 0) {
        st_coherent(f.ml + slot * 2 * BQ + rg * 32 + fr, m);
        st_coherent(f.ml + slot * 2 * BQ + BQ + rg * 32 + fr, l);
      }
    } else if (a.lse && row && fk == 0) {
      a.lse[(int64_t)h * a.M + qrow] = m + log2f(l);
    }
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
      const f32x16 o1 = mo[(rg * DT + dt) * 64 + lane];
#pragma unroll
      for (int g = 0; g < 4; g++) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = o[dt][4 * g + e] * a0 + o1[4 * g + e] * a1;
        // a prefix's rows are read whole by the next launch, a split's by the blocks of this one, in the lanes' order
        if (PREFIX) reinterpret_cast<f32x4*>(f.po)[(slot * BQ + rg * 32 + fr) * (D / 4) + fk + (dt * 4 + g) * 2] = v;
        else if (parts) po.store(((slot * RG + rg) * DT * 4 + dt * 4 + g) * 64 + lane, v);
        else if (row) {
          f16x4 w;
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = (f16)(v[e] * inv);
          *reinterpret_cast<f16x4*>(a.out + qrow * a.ldo + h * D + dt * 32 + 8 * g + 4 * fk) = w;
        }
      }
    }
  }
  if (PREFIX || !parts) return;

  // ---- joins: the block's waves share the row groups that have rows, and a group's waves its 8-dim chunks, CB of them requested
  // at once. Members of a group of splits stand `step` slots apart; the joined part goes to its first member's place, its
  // arrivals are counted at that slot's counter, one further on for every level.
  constexpr int NC = DT * 4, CB = 4;
  const int groups = min(RG, (u.n * G - u.tile * BQ + 31) / 32), jg = wave % groups, P = NW / groups, part = wave / groups;
  const int jr = jg * 32 + fr, jpr = u.tile * BQ + jr;  // the lane's row here
  const bool jrow = jpr < u.n * G;
  const int jtoken = jrow ? plan_token(jpr, a.magic) : 0, jh = hk * G + (jrow ? jpr - jtoken * G : 0);
  f16* const jout = a.out + (int64_t)(u.row0 + jtoken) * a.ldo + jh * D + 4 * fk;
  int n = u.splits, at = u.split, step = 1;
  for (int level = 0;; level++, at /= kFan, n = (n + kFan - 1) / kFan, step *= kFan) {
    const int first = at / kFan * kFan, size = min(kFan, n - first);
    if (size == 1) continue;  // in its place already (and a counter further on may be another tile's)
    const int64_t s0 = (int64_t)(u.slot + first * step) * a.Hkv + hk, ds = (int64_t)step * a.Hkv;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's stores are complete
    __syncthreads();
    if (tid == 0) {
      int* ctr = f.counters + s0 + (int64_t)level * a.Hkv;
      const bool last = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == size - 1;
      if (last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // ready for the next launch
      *flag = last;
    }
    __syncthreads();
    if (*flag == 0) return;
    const bool done = n <= kFan;
    float m = -__builtin_huge_valf(), l = 0.f;
    if (part < P) {
      float w[kFan], ls[kFan];
#pragma unroll
      for (int k = 0; k < kFan; k++) {
        const float* p = f.ml + (s0 + min(k, size - 1) * ds) * 2 * BQ + jr;
        w[k] = ld_coherent(p);
        ls[k] = ld_coherent(p + BQ);
      }
      f32x4 v[CB][kFan];
      auto request = [&](int c0) {
#pragma unroll
        for (int i = 0; i < CB; i++)
#pragma unroll
          for (int k = 0; k < kFan; k++)
            if (k < size) v[i][k] = po.load((((s0 + k * ds) * RG + jg) * NC + min(c0 + i * P, NC - 1)) * 64 + lane);
      };
      request(part);
#pragma unroll
      for (int k = 0; k < kFan; k++) m = fmaxf(m, w[k]);
      const float ref = m == -__builtin_huge_valf() ? 0.f : m;
#pragma unroll
      for (int k = 0; k < kFan; k++) {
        w[k] = exp2f(w[k] - ref);
        if (k < size) l = __builtin_fmaf(w[k], ls[k], l);
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      for (int c0 = part; c0 < NC; c0 += CB * P) {
        if (c0 != part) request(c0);
#pragma unroll
        for (int i = 0; i < CB; i++) {
          const int c8 = c0 + i * P;
          f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < kFan; k++)
            if (k < size)
#pragma unroll
              for (int e = 0; e < 4; e++) sum[e] = __builtin_fmaf(w[k], v[i][k][e], sum[e]);
          if (c8 < NC) {
            if (!done) {
              po.store(((s0 * RG + jg) * NC + c8) * 64 + lane, sum);
            } else if (jrow) {
              f16x4 y;
#pragma unroll
              for (int e = 0; e < 4; e++) y[e] = (f16)(sum[e] * inv);
              *reinterpret_cast<f16x4*>(jout + 8 * c8) = y;
            }
          }
        }
      }
    }
    // every wave of a row group has read the first member's m and l before the joined ones take their place (O's chunks are
    // each read and written by one wave)
    if (!done) __syncthreads();
    if (part == 0 && fk == 0) {
      if (!done) {
        st_coherent(f.ml + s0 * 2 * BQ + jr, m);
        st_coherent(f.ml + s0 * 2 * BQ + BQ + jr, l);
      } else if (a.lse && jrow) {
        a.lse[(int64_t)jh * a.M + u.row0 + jtoken] = m + log2f(l);
      }
    }
    if (done) return;
  }
}

// grid (Hkv, units): a kv head's blocks are on as few XCDs as there can be
template <int D, int RG, class C>
__global__ void __launch_bounds__(128 * RG) attn_pages_kernel(AttnArgs a, C c, FlashPlan f) {
  pages_block<D, RG, false>(a, c, f, blockIdx.x, blockIdx.y, 0);
}

// Joins N parts (m, l, O) to the running (M, L, O), which is relative to M (-inf: no key yet); parts from `count` on are
// left out.
template <int N>
__device__ __forceinline__ void join_parts(float& M, float& L, f32x4& O, const float (&ms)[N], const float (&ls)[N],
                                           const f32x4 (&os)[N], int count) {
  float most = M;
#pragma unroll
  for (int k = 0; k < N; k++)
    if (k < count) most = fmaxf(most, ms[k]);
  const float ref = most == -__builtin_huge_valf() ? 0.f : most, w0 = exp2f(M - ref);
  M = most;
  L *= w0;
#pragma unroll
  for (int e = 0; e < 4; e++) O[e] *= w0;
#pragma unroll
  for (int k = 0; k < N; k++) {
    if (k >= count) continue;
    const float w = exp2f(ms[k] - ref);
    L = __builtin_fmaf(w, ls[k], L);
#pragma unroll
    for (int e = 0; e < 4; e++) O[e] = __builtin_fmaf(w, os[k][e], O[e]);
  }
}

// What a lane of step_block and attn_rows_kernel holds of a 32-key tile: its K rows (keys 4 x + r % 4 of its group, k steps of 32
// dims; a lane's share of a step is free, as long as Q's is the same) and its 8 V rows of DL dims. Of the fp16 cache these are
// the operands themselves. Of the 8-bit one they are codes and their page's exponents, loaded in the same way and
// made into fp16 where they are used: one instruction per two values.
template <int D, class C>
struct PageFrags;
template <int D>
struct PageFrags<D, PagedCache> {
  static constexpr int kStep = 8;  // lane group fk's dims of step s: dim(s) + kStep fk on, 8 of them
  static constexpr int dim(int s) { return 32 * s; }
  typedef typename std::conditional<D == 128, u32x4, u32x2>::type VT;
  u32x4 kf[2][D / 32];
  VT vr[8];
  __device__ __forceinline__ void load_k(const PagedCache&, const f16* p, int, int, int) {
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int s = 0; s < D / 32; s++) kf[x][s] = *reinterpret_cast<const u32x4*>(p + 4 * x * D + 32 * s);
  }
  __device__ __forceinline__ void load_v(const PagedCache&, const f16* p, int, int, int) {
#pragma unroll
    for (int i = 0; i < 8; i++) vr[i] = *reinterpret_cast<const VT*>(p + i * D);
  }
  __device__ __forceinline__ float k_scale() const { return 1.f; }
  __device__ __forceinline__ f16x8 k(int x, int s, float) const { return __builtin_bit_cast(f16x8, kf[x][s]); }
  __device__ __forceinline__ void v(VT (&out)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; i++) out[i] = vr[i];
  }
  // V row i's dims 2 n and 2 n + 1 (of the lane's DL) as two fp16, and row i made zero
  __device__ __forceinline__ float v_scale() const { return 1.f; }
  __device__ __forceinline__ uint32_t v2(int i, int n, float) const { return vr[i][n]; }
  __device__ __forceinline__ void clear_v(int i) { vr[i] = VT{}; }
};
template <int D>
struct PageFrags<D, PagedCache8> {
  static constexpr int kStep = 16;  // 16 codes a load: two steps' shares
  static constexpr int dim(int s) { return 64 * (s >> 1) + 8 * (s & 1); }
  typedef typename std::conditional<D == 128, u32x4, u32x2>::type VT;
  typedef typename std::conditional<D == 128, u32x2, uint32_t>::type VR;
  u32x4 kr[2][D / 64];
  VR vr[8];
  int ke, ve;
  __device__ __forceinline__ void load_k(const PagedCache8& c, const uint8_t* p, int id, int hk, int Hkv) {
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int s = 0; s < D / 64; s++) kr[x][s] = *reinterpret_cast<const u32x4*>(p + 4 * x * D + 64 * s);
    ke = c.kexp[(c.has(id) ? (int64_t)id * Hkv : 0) + hk];
  }
  __device__ __forceinline__ void load_v(const PagedCache8& c, const uint8_t* p, int id, int hk, int Hkv) {
#pragma unroll
    for (int i = 0; i < 8; i++) vr[i] = *reinterpret_cast<const VR*>(p + i * D);
    ve = c.vexp[(c.has(id) ? (int64_t)id * Hkv : 0) + hk];
  }
  __device__ __forceinline__ float k_scale() const { return exponent_scale(ke); }
  __device__ __forceinline__ f16x8 k(int x, int s, float scale) const {
    const u32x4 w = kr[x][s >> 1];
    return s & 1 ? f8x8_to_f16(w[2], w[3], scale) : f8x8_to_f16(w[0], w[1], scale);
  }
  __device__ __forceinline__ float v_scale() const { return exponent_scale(ve); }
  __device__ __forceinline__ uint32_t v2(int i, int n, float scale) const {
    uint32_t w;
    if constexpr (D == 128) w = vr[i][n >> 1];
    else w = vr[i];
    return f8x2_to_f16(w, n & 1, scale);
  }
  __device__ __forceinline__ void clear_v(int i) { vr[i] = VR{}; }
  __device__ __forceinline__ void v(VT (&out)[8]) const {
    const float scale = exponent_scale(ve);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if constexpr (D == 128) {
        out[i] = __builtin_bit_cast(u32x4, f8x8_to_f16(vr[i][0], vr[i][1], scale));
      } else {
        f16x2 lo{}, hi{};
        f8x4_to_f16(vr[i], scale, lo, hi);
        out[i] = u32x2{as_u32(lo), as_u32(hi)};
      }
    }
  }
};
// ---- one row per sequence
//
// The slot cache's decode attention (decode.hip: a wave takes 32 keys, K Q^T and V^T P^T on 16x16x32 MFMAs with the group's
// heads as columns, K and V straight into operand registers, refilled as soon as they are used) with its splits
// (decode_split.h), over pages: the 8 keys that a lane's K rows, or its V rows, come from lie on one page, so a lane has
// one 64-bit address each for K and V per tile, from entries requested a tile ahead. What the slot kernel leaves to the
// buffer bounds is done in registers, in a wave's last tile and in tiles with an entry that is no page only: logits of
// keys that are not there become -inf, their V rows zeros.
// Measured: 64 sequences of 1000 keys, 32/8 heads of 128, 48.0 us (5.5 TB/s; slots 47.2), 48 of 100 to 2000 46.3 (4.5 TB/s;
// slots 43.5), one of 4001 10.3 (slots 9.4: the table is one more load in the chain from the position to K).
// OWN: the keys behind a shared prefix; a split leaves its part for join_block.
struct StepPlan {
  int S, S1;      // splits of a pair: the launch's, and those that give every CU a block (splits_used)
  int K;          // > 0: a split per K keys instead
  int* counters;  // [B * Hkv], arrivals of a pair's splits
  float *ml, *po; // partial results: [B][Hq][S][2] m and l, [B][Hq][S][D] O
};

// Keys from `base` on that sequence b's row sees.
__device__ __forceinline__ int step_keys(const AttnArgs& a, int cap, int b, int base) {
  return plan_end(a.pos[b], 1, cap) > base ? plan_end(a.pos[b], 1, cap) - base : 0;
}

template <int GC, int D, int NWV>
struct StepSmem {
  float wo[NWV][GC][D];
  float wm[NWV][GC], wl[NWV][GC];
  float sm[GC][kDecodeMaxSplits], sw[GC][kDecodeMaxSplits];
  float tm[GC], tl[GC];
  int is_last;
};

// Element d of head g over a block's waves.
template <int GC, int D, int NWV>
__device__ __forceinline__ void step_sum(const StepSmem<GC, D, NWV>& sh, int g, int d, float& M, float& L, float& O) {
  M = -__builtin_huge_valf();
#pragma unroll
  for (int w = 0; w < NWV; w++) M = fmaxf(M, sh.wm[w][g]);
  L = O = 0.f;
#pragma unroll
  for (int w = 0; w < NWV; w++) {
    const float e = sh.wm[w][g] == -__builtin_huge_valf() ? 0.f : exp2f(sh.wm[w][g] - M);
    L = __builtin_fmaf(sh.wl[w][g], e, L);
    O = __builtin_fmaf(sh.wo[w][g][d], e, O);
  }
}

// Splits that a run of len keys is cut into.
__device__ __forceinline__ int step_used(const StepPlan& f, int len) {
  return f.K > 0 ? plan_step_splits(len, f.K, f.S) : splits_used(len, f.S, f.S1);
}

// One block: split `split` of sequence b and kv head hk. With `keep` a sequence's only part is left in the waves' LDS (step_sum).
template <int GC, int D, int NWV, bool OWN, class C>
__device__ __forceinline__ void step_block(const AttnArgs& a, const C& c, const StepPlan& f,
                                           StepSmem<GC, D, NWV>& sh, int hk, int b, int split, bool keep = false) {
  constexpr int KS = D / 32;               // k steps of a logits product
  constexpr int DL = D / 16;               // V dims (and P.V products) per lane
  constexpr int BK = NWV * kDaTile;        // keys per block pass
  constexpr int NT = NWV * 64;
  typedef PageFrags<D, C> Fr;
  const int G = a.G, page = 1 << c.shift;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int len = step_keys(a, c.capacity(), b, OWN ? a.shared : 0);
  const int S_eff = step_used(f, len);
  if (split >= S_eff) return;
  // (the groups of 8 keys start on multiples of 8)
  const int chunk = ((len < kPlanDiv ? plan_div(len + S_eff - 1, S_eff) : (len + S_eff - 1) / S_eff) + 7) & ~7;
  const int base = OWN ? a.shared : 0;
  const int start = base + split * chunk, end = base + min(len, (split + 1) * chunk);

  const int r = lane & 15, fk = lane >> 4;
  // S^T = K Q^T (16x16x32): A row r of block x is the tile's key 8 (r / 4) + 4 x + r % 4, so lane group fk of the C layout
  // ends up with keys 8 fk .. 8 fk + 7 of head r: the B operand of the 32-key P.V product. V: lane (r, fk) loads dims
  // DL r .. of keys 8 fk + i.
  const int kg = 8 * (r >> 2), vg = 8 * fk;  // the lane's key groups in a tile
  const auto kl = c.kp + ((int64_t)hk * page + (r & 3)) * D + Fr::kStep * fk;
  const auto vl = c.vp + (int64_t)hk * page * D + DL * r;
  auto entry = [&](int key) { return key < end ? c.entry(!OWN && key < a.shared ? 0 : b, key >> c.shift) : -1; };
  // element offset of the group that starts at `key`; that of page 0 for keys that are not there
  auto place = [&](int id, int key) { return c.has(id) ? id * c.stride + (int64_t)(key & (page - 1)) * D : (int64_t)0; };
  Fr kv;
  auto load_k = [&](int id, int key) { kv.load_k(c, kl + place(id, key), id, hk, a.Hkv); };
  int vid_next = -1;  // the V group that is requested next
  int64_t va = 0;
  auto load_v = [&] { kv.load_v(c, vl + va, vid_next, hk, a.Hkv); };
  const int t_first = start + wave * kDaTile;
  const f16* qg = a.q + (int64_t)b * a.ldq + (hk * G + (r < G ? r : 0)) * D + Fr::kStep * fk;
  float m = -__builtin_huge_valf(), l = 0.f;  // of head r; l over this lane's keys only
  f32x4 o[DL];                                // O^T: dim DL (4 fk + i) + n of head r in o[n][i]
#pragma unroll
  for (int n = 0; n < DL; n++) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (t_first < end) {
    int kid = entry(t_first + kg), vid = entry(t_first + vg);
    bool there = c.has(vid);  // this lane's V group of the tile lies on a page
    bool whole = __all(there) && t_first + kDaTile <= end;
    va = place(vid, t_first + vg);
    vid_next = vid;
    load_k(kid, t_first + kg);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) qf[s] = *reinterpret_cast<const u32x4*>(qg + Fr::dim(s));
    load_v();
    kid = entry(t_first + BK + kg);
    vid = entry(t_first + BK + vg);
    // One tile; the next tile's K is requested as soon as this one's is used, and so is its V.
    auto tile = [&](int t0, auto maskc, auto lastc) {
      constexpr bool MASK = decltype(maskc)::value, LAST = decltype(lastc)::value;
      f32x4 sc[2];
      const float ks = kv.k_scale();
#pragma unroll
      for (int x = 0; x < 2; x++) {
        sc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; s++)
          sc[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv.k(x, s, ks), __builtin_bit_cast(f16x8, qf[s]), sc[x], 0, 0, 0);
      }
      const bool was = there;
      if constexpr (!LAST) {
        __builtin_amdgcn_sched_barrier(0);
        load_k(kid, t0 + BK + kg);
        there = c.has(vid);
        whole = __all(there) && t0 + BK + kDaTile <= end;
        va = place(vid, t0 + BK + vg);
        vid_next = vid;
        kid = entry(t0 + 2 * BK + kg);
        vid = entry(t0 + 2 * BK + vg);
        __builtin_amdgcn_sched_barrier(0);
      }
      float p[8];
      float mx = -__builtin_huge_valf();
#pragma unroll
      for (int k = 0; k < 8; k++) {
        p[k] = sc[k >> 2][k & 3] * a.scale_log2;
        if (MASK && !(was && t0 + vg + k < end)) p[k] = -__builtin_huge_valf();
        mx = fmaxf(mx, p[k]);
      }
      const float m_old = m;
      m = fmaxf(m, rows_reduce<true>(mx));
      // -inf while no key was there, or every logit so far is: their weights are 0
      const float mn = m == -__builtin_huge_valf() ? 0.f : m;
      const float alpha = exp2f(m_old - mn);  // 0 on the first tile (m = -inf)
      float ps = 0.f;
      f16x8 ph;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        p[k] = exp2f(p[k] - mn);
        ps += p[k];
        ph[k] = (f16)p[k];
      }
      l = __builtin_fmaf(l, alpha, ps);
#pragma unroll
      for (int n = 0; n < DL; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[n][i] *= alpha;
      if constexpr (MASK) {
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (!(was && t0 + vg + k < end)) kv.clear_v(k);
      }
      const float vs = kv.v_scale();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n2 = 0; n2 < DL / 2; n2++) {
        uint32_t v2[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v2[k] = kv.v2(k, n2, vs);
#pragma unroll
        for (int n = 2 * n2; n < 2 * n2 + 2; n++) {
          u32x4 w;
#pragma unroll
          for (int k = 0; k < 4; k++) w[k] = __builtin_amdgcn_perm(v2[2 * k + 1], v2[2 * k], n & 1 ? 0x07060302u : 0x05040100u);
          o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), ph, o[n], 0, 0, 0);
        }
      }
      if constexpr (!LAST) {
        __builtin_amdgcn_sched_barrier(0);
        load_v();
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const std::true_type yes{};
    const std::false_type no{};
    int t0 = t_first;
    for (; t0 + BK < end; t0 += BK) {
      if (whole) tile(t0, no, no);
      else tile(t0, yes, no);
    }
    tile(t0, yes, yes);
  }
  l = rows_reduce<false>(l);

  // ---- merge the block's waves (a wave without keys has m = -inf and weight 0)
  if (r < G) {
    if (fk == 0) {
      sh.wm[wave][r] = m;
      sh.wl[wave][r] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int n = 0; n < DL; n += 4)
        *reinterpret_cast<f32x4*>(&sh.wo[wave][r][DL * (4 * fk + i) + n]) =
            f32x4{o[n][i], o[n + 1][i], o[n + 2][i], o[n + 3][i]};
  }
  __syncthreads();
  const bool single = S_eff == 1;
  if (OWN && keep && single) return;
  const int64_t pair = (int64_t)b * a.Hq + hk * G;  // of head 0 of the group; its partials start at pair * S
  auto store = [&](int g, int d, float M, float L, float O) {
    a.out[(int64_t)b * a.ldo + (hk * G + g) * D + d] = (f16)(L == 0.f ? 0.f : O / L);
    if (a.lse && d == 0) a.lse[(int64_t)(hk * G + g) * a.M + b] = M + log2f(L);
  };
  for (int i = tid; i < G * D; i += NT) {
    const int g = i / D, d = i % D;
    float M, L, O;
    step_sum(sh, g, d, M, L, O);
    const int64_t at = (pair + g) * f.S + split;
    if (!OWN && single) {
      store(g, d, M, L, O);
    } else {
      st_coherent(f.po + at * D + d, O);
      if (d == 0) {
        st_coherent(f.ml + 2 * at, M);
        st_coherent(f.ml + 2 * at + 1, L);
      }
    }
  }
  if (OWN || single) return;
  constexpr int EPT = (GC * D + NT - 1) / NT;  // output elements per thread
  constexpr bool AHEAD = GC <= 8;      // (16 heads would not fit the registers)
  float v0[EPT][16];
  {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this thread's partial stores are complete
    __syncthreads();
    if (tid == 0) {
      int* ctr = f.counters + b * a.Hkv + hk;
      const int done = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      sh.is_last = done == S_eff - 1;
      if (sh.is_last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // ready for the next launch
    }
    __syncthreads();
    if (!sh.is_last) return;
    // ---- the last block merges the S_eff splits of every head of its group, in split order. The (m, l) pairs and the
    //      first 16 splits' partial outputs are requested in one round.
    if constexpr (AHEAD) {
#pragma unroll
      for (int e = 0; e < EPT; e++) {
        const int i = tid + e * NT;
        const int g = min(i / D, G - 1), d = i % D;
        const float* pp = f.po + (pair + g) * f.S * D + d;
#pragma unroll
        for (int k = 0; k < 16; k++) v0[e][k] = ld_coherent(pp + (int64_t)min(k, S_eff - 1) * D);
      }
    }
    {
      for (int i = tid; i < G * S_eff; i += NT) {
        const int g = i / S_eff, s = i - g * S_eff;
        const float* pp = f.ml + ((pair + g) * f.S + s) * 2;
        sh.sm[g][s] = ld_coherent(pp);
        sh.sw[g][s] = ld_coherent(pp + 1);
      }
      __syncthreads();
      for (int g = wave; g < G; g += NWV) {  // S_eff is at most a wave's lanes
        const float ms = lane < S_eff ? sh.sm[g][lane] : -__builtin_huge_valf(), ls = lane < S_eff ? sh.sw[g][lane] : 0.f;
        const float M = wave_max(ms);
        const float e = ms == -__builtin_huge_valf() ? 0.f : exp2f(ms - M);
        const float L = wave_sum(ls * e);
        if (lane < S_eff) sh.sw[g][lane] = e;
        if (lane == 0) {
          sh.tm[g] = M;
          sh.tl[g] = L;
        }
      }
      __syncthreads();
    }
  }
  // splits s0 .. s0 + 15 of element (g, d)
  auto sum16 = [&](int g, const float (&v)[16], int s0, float& O) {
#pragma unroll
    for (int k = 0; k < 16; k++) O = __builtin_fmaf(v[k], s0 + k < S_eff ? sh.sw[g][s0 + k] : 0.f, O);
  };
  auto load16 = [&](int g, int d, int s0, float (&v)[16]) {
    const float* pp = f.po + (pair + g) * f.S * D + d;
#pragma unroll
    for (int k = 0; k < 16; k++) v[k] = ld_coherent(pp + (int64_t)min(s0 + k, S_eff - 1) * D);
  };
  {
#pragma unroll
    for (int e = 0; e < EPT; e++) {
      const int i = tid + e * NT;
      if (i < G * D) {
        const int g = i / D, d = i % D;
        float O = 0.f;
        if constexpr (AHEAD) sum16(g, v0[e], 0, O);
        for (int s0 = AHEAD ? 16 : 0; s0 < S_eff; s0 += 16) {
          float v[16];
          load16(g, d, s0, v);
          sum16(g, v, s0, O);
        }
        store(g, d, sh.tm[g], sh.tl[g], O);
      }
    }
  }
}

// grid (Hkv, B, S): a pair's used splits come first in dispatch order
template <int GC, int D, int NWV, class C>
__global__ void __launch_bounds__(NWV * 64, 3) attn_step_kernel(AttnArgs a, C c, StepPlan f) {
  __shared__ StepSmem<GC, D, NWV> sh;
  step_block<GC, D, NWV, false>(a, c, f, sh, blockIdx.x, blockIdx.y, blockIdx.z);
}

// ---- few rows
//
// Runs of a few rows (decoding sequences, drafted tokens to verify, short chunks; row_columns): the step's products with packed
// rows (token, head of the group) as columns, NC blocks of 16, so that K and V fragments feed NC products each. The keys
// behind a row are hidden in the tiles that hold them, and infinities and NaN among their V rows go to the rows that see them
// as in flash_tile.h. Block = (row tile, kv head, split); of a tile's splits the block that arrives last joins all. Two
// blocks of 8 waves would not fit a CU's registers: there is a unit for every CU, by the plan of all lengths; many tiles
// have blocks of 4 waves and a step's splits, which need no plan.
// What bounds it: small batches the chain of a step (one row after 4000 11.9 us, a plan's 1 to 2 more than attn_step_kernel);
// 48 rows after 100 to 2000 45.5 us, 4.6 TB/s; 8 x 5 rows after 700 to 4000 21.1, 3.7 TB/s, its 256 blocks' first tiles
// (4 us) and the joins (4 us) around 12 us of keys.
template <int D, int NC, int NWV>
struct RowsSmem {
  float wo[NWV][16 * NC][D + 4];  // (+ 4: the 16 columns' stores on distinct banks)
  float wm[NWV][16 * NC], wl[NWV][16 * NC];
  int is_last;
};

// Unit `at` of the batch's row tiles, each of them as many units as its sequence's keys have splits: blocks without work come
// last, where they keep no other from a CU. u.slot is the tile's number. False if there are not so many.
template <int COLS>
__device__ __forceinline__ bool rows_unit(const AttnArgs& a, int cap, const StepPlan& f, int at, int lane, FlashUnit& u) {
  int before = 0, slot = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    int row0 = 0, rows = 0, pos = 0;
    if (b < a.B) {
      const int s0 = a.start[b], s1 = a.start[b + 1];
      pos = a.pos[b];
      row0 = plan_first(s0, a.M);
      rows = plan_rows(s0, s1, a.M);
    }
    const int tiles = plan_tiles(rows, a.G, COLS), splits = step_used(f, plan_end(pos, rows, cap)), n = tiles * splits;
    const int upto = wave_scan(n, lane), slots = wave_scan(tiles, lane);
    const uint64_t hit = __ballot(before + upto > at);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto take = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int i = at - before - (take(upto) - take(n));
      u = FlashUnit{b0 + l, take(row0), take(rows), take(pos), 0, take(splits), 0, 0};
      u.tile = u.splits == 1 ? i : plan_div(i, u.splits);
      u.split = i - u.tile * u.splits;
      u.slot = slot + take(slots) - take(tiles) + u.tile;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    slot += __builtin_amdgcn_readlane(slots, 63);
  }
  return false;
}

template <int D, int NC, int NWV, class C>
__global__ void __launch_bounds__(NWV * 64, NC == 1 ? 3 : 2) attn_rows_kernel(AttnArgs a, C c, StepPlan f, FlashPlan fp, int tiles) {
  constexpr int KS = D / 32;               // k steps of a logits product
  constexpr int DL = D / 16;               // V dims (and P.V products) per lane
  constexpr int BK = NWV * kDaTile;        // keys per block pass
  constexpr int NT = NWV * 64, COLS = 16 * NC, D4 = D / 4;
  typedef PageFrags<D, C> Fr;
  extern __shared__ u32x4 fp_smem[];
  auto& sh = *reinterpret_cast<RowsSmem<D, NC, NWV>*>(fp_smem);
  const int G = a.G, page = 1 << c.shift, cap = c.capacity();
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hk = blockIdx.x;
  FlashUnit u;
  int counter;
  if constexpr (NWV == 8) {
    if (!flash_unit<COLS>(a, cap, fp, blockIdx.y, lane, u)) return;
    if (u.splits > 1 && u.slot + u.split >= fp.slots) return;  // (not reached: the plan stays within the slots)
    counter = u.slot;
  } else {
    if (!rows_unit<COLS>(a, cap, f, blockIdx.y, lane, u)) return;
    // (a start that decreases may have more tiles, or units, than there are: such tiles are left out whole)
    if (u.slot >= tiles || (int)blockIdx.y - u.split + u.splits > (int)gridDim.y) return;
    counter = u.slot;
    u.slot *= f.S;
  }
  const int len = plan_tile_end(u.pos, u.n, u.tile, G, a.magic, COLS, cap);
  const int S_eff = u.splits, split = u.split;
  const int chunk = ((len < kPlanDiv ? plan_div(len + S_eff - 1, S_eff) : (len + S_eff - 1) / S_eff) + 7) & ~7;
  const int start = split * chunk, end = min(len, start + chunk);
  const int first = u.tile * COLS, cols = min(COLS, u.n * G - first);  // packed rows of the tile

  const int r = lane & 15, fk = lane >> 4;
  const int kg = 8 * (r >> 2), vg = 8 * fk;  // the lane's key groups in a tile (step_block)
  const auto kl = c.kp + ((int64_t)hk * page + (r & 3)) * D + Fr::kStep * fk;
  const auto vl = c.vp + (int64_t)hk * page * D + DL * r;
  auto entry = [&](int key) { return key < end ? c.entry(u.b, key >> c.shift) : -1; };
  auto place = [&](int id, int key) { return c.has(id) ? id * c.stride + (int64_t)(key & (page - 1)) * D : (int64_t)0; };
  // the last key that the lane's columns see (-1 without a row), and the keys that every row of the tile sees
  int qpos[NC];
  const f16* qg[NC];
#pragma unroll
  for (int x = 0; x < NC; x++) {
    const int pr = first + 16 * x + r, token = plan_token(min(pr, first + cols - 1), a.magic);
    qpos[x] = 16 * x + r < cols ? (int)min((int64_t)u.pos + token, (int64_t)cap - 1) : -1;
    qg[x] = a.q + (int64_t)(u.row0 + token) * a.ldq + (hk * G + min(pr, first + cols - 1) - token * G) * D + Fr::kStep * fk;
  }
  const int common = min(end, plan_end(u.pos, plan_token(first, a.magic) + 1, cap));
  Fr kv;
  auto load_k = [&](int id, int key) { kv.load_k(c, kl + place(id, key), id, hk, a.Hkv); };
  int vid_next = -1;  // the V group that is requested next
  int64_t va = 0;
  auto load_v = [&] { kv.load_v(c, vl + va, vid_next, hk, a.Hkv); };
  const int t_first = start + wave * kDaTile;
  float m[NC], l[NC];  // of the lane's columns; l over this lane's keys only
  f32x4 o[NC][DL];     // O^T: dim DL (4 fk + i) + n of column 16 x + r in o[x][n][i]
#pragma unroll
  for (int x = 0; x < NC; x++) {
    m[x] = -__builtin_huge_valf();
    l[x] = 0.f;
#pragma unroll
    for (int n = 0; n < DL; n++) o[x][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (t_first < end) {
    int kid = entry(t_first + kg), vid = entry(t_first + vg);
    bool there = c.has(vid);  // this lane's V group of the tile lies on a page
    bool whole = __all(there) && t_first + kDaTile <= common;
    va = place(vid, t_first + vg);
    vid_next = vid;
    load_k(kid, t_first + kg);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 qf[NC][KS];
#pragma unroll
    for (int x = 0; x < NC; x++)
#pragma unroll
      for (int s = 0; s < KS; s++) qf[x][s] = *reinterpret_cast<const u32x4*>(qg[x] + Fr::dim(s));
    load_v();
    kid = entry(t_first + BK + kg);
    vid = entry(t_first + BK + vg);
    int odd_tile = INT32_MAX;  // the first masked tile with infinities or NaN in V
    auto tile = [&](int t0, auto maskc, auto lastc) {
      constexpr bool MASK = decltype(maskc)::value, LAST = decltype(lastc)::value;
      f32x4 sc[NC][2];
      const float ks = kv.k_scale();
      if constexpr (C::kF8) {  // a fragment at a time: made once for all products
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
          for (int s = 0; s < KS; s++) {
            const f16x8 k = kv.k(y, s, ks);
#pragma unroll
            for (int x = 0; x < NC; x++)
              sc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, __builtin_bit_cast(f16x8, qf[x][s]),
                                                                s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[x][y], 0, 0, 0);
          }
      } else {
#pragma unroll
        for (int x = 0; x < NC; x++)
#pragma unroll
          for (int y = 0; y < 2; y++) {
            sc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; s++)
              sc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv.k(y, s, ks), __builtin_bit_cast(f16x8, qf[x][s]), sc[x][y], 0,
                                                                0, 0);
          }
      }
      const bool was = there;
      if constexpr (!LAST) {
        __builtin_amdgcn_sched_barrier(0);
        load_k(kid, t0 + BK + kg);
        there = c.has(vid);
        whole = __all(there) && t0 + BK + kDaTile <= common;
        va = place(vid, t0 + BK + vg);
        vid_next = vid;
        kid = entry(t0 + 2 * BK + kg);
        vid = entry(t0 + 2 * BK + vg);
        __builtin_amdgcn_sched_barrier(0);
      }
      f16x8 ph[NC];
#pragma unroll
      for (int x = 0; x < NC; x++) {
        float p[8];
        float mx = -__builtin_huge_valf();
#pragma unroll
        for (int k = 0; k < 8; k++) {
          p[k] = sc[x][k >> 2][k & 3] * a.scale_log2;
          if (MASK && !(was && t0 + vg + k < end && t0 + vg + k <= qpos[x])) p[k] = -__builtin_huge_valf();
          mx = fmaxf(mx, p[k]);
        }
        const float m_old = m[x];
        m[x] = fmaxf(m[x], rows_reduce<true>(mx));
        const float mn = m[x] == -__builtin_huge_valf() ? 0.f : m[x];  // no key seen: all weights are 0
        const float alpha = __builtin_amdgcn_exp2f(m_old - mn);
        float ps = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) {
          p[k] = __builtin_amdgcn_exp2f(p[k] - mn);
          ps += p[k];
          ph[x][k] = (f16)p[k];
        }
        l[x] = __builtin_fmaf(l[x], alpha, ps);
#pragma unroll
        for (int n = 0; n < DL; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[x][n][i] *= alpha;
      }
      typename Fr::VT vf[8];
      kv.v(vf);
      if constexpr (MASK) {
        // rows behind the end are zeros; infinities and NaN, which a row that does not see their key would turn to
        // NaN, are taken out and given to the rows that see them after the loop
        uint32_t odd = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
          if (!(was && t0 + vg + k < end)) vf[k] = typename Fr::VT{};
#pragma unroll
          for (int i = 0; i < DL / 2; i++) odd |= (vf[k][i] & 0x7fff7fffu) + 0x04000400u;  // an exponent of ones carries
        }
        if (__any((odd & 0x80008000u) != 0)) {
          odd_tile = min(odd_tile, t0);
#pragma unroll
          for (int k = 0; k < 8; k++)
#pragma unroll
            for (int i = 0; i < DL / 2; i++) {
              if ((vf[k][i] & 0x7c00u) == 0x7c00u) vf[k][i] &= 0xffff0000u;
              if ((vf[k][i] & 0x7c000000u) == 0x7c000000u) vf[k][i] &= 0x0000ffffu;
            }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < DL; n++) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; k++)
          w[k] = __builtin_amdgcn_perm(vf[2 * k + 1][n >> 1], vf[2 * k][n >> 1], n & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int x = 0; x < NC; x++)
          o[x][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), ph[x], o[x][n], 0, 0, 0);
      }
      if constexpr (!LAST) {
        __builtin_amdgcn_sched_barrier(0);
        load_v();
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const std::true_type yes{};
    const std::false_type no{};
    int t0 = t_first;
    for (; t0 + BK < end; t0 += BK) {
      if (whole) tile(t0, no, no);
      else tile(t0, yes, no);
    }
    tile(t0, yes, yes);
#pragma unroll 1
    for (int t = odd_tile; t < end; t += BK)
#pragma unroll 1
      for (int k = t; k < min(t + kDaTile, end); k++) {
        const int id = c.entry(u.b, k >> c.shift);
        if (!c.has(id)) continue;
        const auto vrow = c.vp + id * c.stride + ((int64_t)hk * page + (k & (page - 1))) * D + 4 * DL * fk;
        const float vs = page_scale<true>(c, id, hk, a.Hkv);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int n = 0; n < DL; n++) {
            const float v = element(vrow[DL * i + n], vs);
            if (!(__builtin_fabsf(v) < __builtin_huge_valf()))
#pragma unroll
              for (int x = 0; x < NC; x++)
                if (k <= qpos[x]) o[x][n][i] += v;
          }
      }
  }

  // ---- merge the block's waves (a wave without keys has m = -inf and weight 0)
#pragma unroll
  for (int x = 0; x < NC; x++) {
    l[x] = rows_reduce<false>(l[x]);
    if (16 * x + r >= cols) continue;
    if (fk == 0) {
      sh.wm[wave][16 * x + r] = m[x];
      sh.wl[wave][16 * x + r] = l[x];
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int n = 0; n < DL; n += 4)
        *reinterpret_cast<f32x4*>(&sh.wo[wave][16 * x + r][DL * (4 * fk + i) + n]) =
            f32x4{o[x][n][i], o[x][n + 1][i], o[x][n + 2][i], o[x][n + 3][i]};
  }
  __syncthreads();
  auto store = [&](int col, int d, float M, float L, f32x4 O) {
    const int token = plan_token(first + col, a.magic), h = hk * G + first + col - token * G;
    f16x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = (f16)(L == 0.f ? 0.f : O[e] / L);
    *reinterpret_cast<f16x4*>(a.out + (int64_t)(u.row0 + token) * a.ldo + h * D + d) = v;
    if (a.lse && d == 0) a.lse[(int64_t)h * a.M + u.row0 + token] = M + log2f(L);
  };
  const bool single = S_eff == 1;
  const int64_t part0 = (int64_t)u.slot * a.Hkv + hk;  // split 0's part; the others follow Hkv parts apart
  const PartBuffer po(f.po, (size_t)(NWV == 8 ? fp.slots : tiles * f.S) * a.Hkv * COLS * D * 4);
  for (int i = tid; i < cols * D4; i += NT) {
    const int col = i / D4, d = 4 * (i % D4);
    float M = -__builtin_huge_valf(), L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    float ms[NWV], ls[NWV];
    f32x4 os[NWV];
#pragma unroll
    for (int w = 0; w < NWV; w++) {
      ms[w] = sh.wm[w][col];
      ls[w] = sh.wl[w][col];
      os[w] = *reinterpret_cast<const f32x4*>(&sh.wo[w][col][d]);
    }
    join_parts(M, L, O, ms, ls, os, NWV);
    if (single) {
      store(col, d, M, L, O);
    } else {
      const int64_t part = part0 + (int64_t)split * a.Hkv;
      po.store(part * (COLS * D4) + i, O);
      if (d == 0) {
        st_coherent(f.ml + part * 2 * COLS + col, M);
        st_coherent(f.ml + part * 2 * COLS + COLS + col, L);
      }
    }
  }
  if (single) return;
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this thread's partial stores are complete
  __syncthreads();
  if (tid == 0) {
    int* ctr = f.counters + counter * a.Hkv + hk;
    sh.is_last = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == S_eff - 1;
    if (sh.is_last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // ready for the next launch
  }
  __syncthreads();
  if (!sh.is_last) return;
  // ---- the last block joins the splits, in their order, 8 requested at once
  for (int i = tid; i < cols * D4; i += NT) {
    const int col = i / D4, d = 4 * (i % D4);
    float M = -__builtin_huge_valf(), L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s0 = 0; s0 < S_eff; s0 += 8) {
      float ms[8], ls[8];
      f32x4 os[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int64_t part = part0 + (int64_t)min(s0 + k, S_eff - 1) * a.Hkv;
        ms[k] = ld_coherent(f.ml + part * 2 * COLS + col);
        ls[k] = ld_coherent(f.ml + part * 2 * COLS + COLS + col);
        os[k] = po.load(part * (COLS * D4) + i);
      }
      join_parts(M, L, O, ms, ls, os, S_eff - s0);
    }
    store(col, d, M, L, O);
  }
}

// ---- a shared prefix
//
// Its parts (pages_block) and the sequences' own keys (step_block) are computed apart and joined. Where the prefix leaves half
// of the GPU idle, both run in one launch, and a launch for the joins follows; else the own keys run in a second launch,
// whose blocks join.
constexpr int kPartThreads = 256;
struct PartSmem {
  float m[kPartThreads], l[kPartThreads];
  f32x4 o[kPartThreads];
};

// Joins the prefix's parts and the `own` parts of sequence b, kv head hk. A thread takes 4 dims of a head, and where there are
// more threads than those, every P-th part, 8 requested at once; the P threads' results are joined through LDS. SAME: the
// own parts come of this launch; an only one is asked of sum(g, d, M, L, O).
template <int D, bool SAME, typename Sum>
__device__ __forceinline__ void join_block(const AttnArgs& a, const FlashPlan& f, const StepPlan& st, int BQ, PartSmem& sh, int hk,
                                           int b, int own, Sum sum) {
  constexpr int D4 = D / 4, NT = kPartThreads;
  const int G = a.G, tid = threadIdx.x, S = f.splits;
  const int items = G * D4, P = items < NT ? NT / items : 1;
  const int64_t dm = (int64_t)a.Hkv * 2 * BQ, dn = (int64_t)a.Hkv * BQ * D;
#pragma unroll 1
  for (int i0 = 0; i0 < items; i0 += NT) {
    const int part = items < NT ? tid / items : 0, item = items < NT ? tid - part * items : i0 + tid;
    const bool active = part < P && item < items;
    const int g = item / D4, d = 4 * (item % D4);
    float M = -__builtin_huge_valf(), L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    if (active) {
      const int pr = b * G + g, tile = pr / BQ, at = pr - tile * BQ;
      const int64_t slot = (int64_t)tile * S * a.Hkv + hk, mine = ((int64_t)b * a.Hq + hk * G + g) * st.S;
      const float* ml = f.ml + slot * 2 * BQ + at;
      const float* po = f.po + (slot * BQ + at) * D + d;
      if (SAME && own == 1) {
        if (part == 0) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float v;
            sum(g, d + e, M, L, v);
            O[e] = v;
          }
        }
      } else {
#pragma unroll 1
        for (int s = part; s < own; s += P) {
          const float* p = st.ml + 2 * (mine + s);
          const float* q = st.po + (mine + s) * D + d;
          const float ms[1] = {SAME ? ld_coherent(p) : p[0]}, ls[1] = {SAME ? ld_coherent(p + 1) : p[1]};
          f32x4 os[1];
#pragma unroll
          for (int e = 0; e < 4; e++) os[0][e] = SAME ? ld_coherent(q + e) : q[e];
          join_parts(M, L, O, ms, ls, os, 1);
        }
      }
#pragma unroll 1
      for (int s0 = part; s0 < S; s0 += 8 * P) {
        float ms[8], ls[8];
        f32x4 os[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const int s = min(s0 + k * P, S - 1);
          ms[k] = ml[s * dm];
          ls[k] = ml[s * dm + BQ];
          os[k] = *reinterpret_cast<const f32x4*>(po + s * dn);
        }
        join_parts(M, L, O, ms, ls, os, (S - s0 + P - 1) / P);
      }
    }
    if (P > 1) {
      __syncthreads();
      sh.m[tid] = M;
      sh.l[tid] = L;
      sh.o[tid] = O;
      __syncthreads();
      if (active && part == 0)
        for (int p = 1; p < P; p++) {
          const float ms[1] = {sh.m[p * items + item]}, ls[1] = {sh.l[p * items + item]};
          const f32x4 os[1] = {sh.o[p * items + item]};
          join_parts(M, L, O, ms, ls, os, 1);
        }
    }
    if (active && part == 0) {
      f16x4 v;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = (f16)(L == 0.f ? 0.f : O[e] / L);
      *reinterpret_cast<f16x4*>(a.out + (int64_t)b * a.ldo + (hk * G + g) * D + d) = v;
      if (a.lse && d == 0) a.lse[(int64_t)(hk * G + g) * a.M + b] = M + log2f(L);
    }
  }
}

// grid (Hkv, prefix blocks + own blocks): the prefix's splits x tiles first, then (with both kinds in one launch) blocks
// that take the sequences' splits in turn, sequence by sequence and split by split.
template <int GC, int D, int RG>
__global__ void __launch_bounds__(128 * RG) attn_prefix_kernel(AttnArgs a, PagedCache c, FlashPlan f, StepPlan st, int tiles) {
  const int np = f.splits * tiles, y = blockIdx.y;
  if (y < np) {
    const int split = tiles == 1 ? y : y / tiles;
    pages_block<D, RG, true>(a, c, f, blockIdx.x, split, y - split * tiles);
    return;
  }
  extern __shared__ u32x4 fp_smem[];
  auto& sh = *reinterpret_cast<StepSmem<GC, D, 2 * RG>*>(fp_smem);
  const int step = gridDim.y - np;
  int b = y - np, split = 0;
  for (;; b += step) {
    while (b >= a.B) {
      b -= a.B;
      split++;
    }
    if (split >= st.S) break;
    // (turned by split: the same blocks would get the long sequences' splits again)
    const int turned = b + split * (a.B / 2 + 1) % a.B;
    step_block<GC, D, 2 * RG, true>(a, c, st, sh, blockIdx.x, turned < a.B ? turned : turned - a.B, split);
    __syncthreads();  // the block's LDS is used again
  }
}

// After it, where it took the sequences' splits too: grid (Hkv, B).
template <int D>
__global__ void __launch_bounds__(kPartThreads) attn_parts_kernel(AttnArgs a, int cap, FlashPlan f, StepPlan st, int BQ) {
  __shared__ PartSmem sh;
  join_block<D, false>(a, f, st, BQ, sh, blockIdx.x, blockIdx.y, step_used(st, step_keys(a, cap, blockIdx.y, a.shared)),
                       [](int, int, float&, float&, float&) {});
}

// Else: grid (Hkv, B, S).
template <int GC, int D>
__global__ void __launch_bounds__(kPartThreads, 3) attn_own_kernel(AttnArgs a, PagedCache c, FlashPlan f, StepPlan st, int BQ) {
  __shared__ StepSmem<GC, D, 4> sh;
  __shared__ PartSmem ps;
  const int hk = blockIdx.x, b = blockIdx.y, split = blockIdx.z;
  const int own = step_used(st, step_keys(a, c.capacity(), b, a.shared));
  if (split >= own) return;
  step_block<GC, D, 4, true>(a, c, st, sh, hk, b, split, true);
  if (own > 1) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this thread's partial stores are complete
    __syncthreads();
    if (threadIdx.x == 0) {
      int* ctr = st.counters + b * a.Hkv + hk;
      sh.is_last = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == own - 1;
      if (sh.is_last) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // ready for the next launch
    }
    __syncthreads();
    if (!sh.is_last) return;
  }
  join_block<D, true>(a, f, st, BQ, ps, hk, b, own,
                      [&](int g, int d, float& M, float& L, float& O) { step_sum(sh, g, d, M, L, O); });
}

// Row groups per block: 4 (128 packed rows), or 2 where a sequence has 64 packed rows or less on average.
int flash_row_groups(int M, int B, int G) { return (int64_t)M * G <= 64 * (int64_t)B ? 2 : 4; }

size_t flash_slot_bytes(int RG, int D) { return (size_t)32 * RG * (D + 2) * 4; }

// Slots (each of all kv heads) that M rows of B sequences can need: those of plan_budget's largest, none where even full
// tiles are too many to be split.
int flash_slots(int M, int G, int Hkv, int RG, int cus) {
  const int least = plan_tiles(M, G, 32 * RG);
  return plan_budget(least, Hkv, cus, cus / Hkv, 2 * cus / Hkv) ? max(2 * cus / Hkv, 1) : 0;
}

// Row tiles that the rows can make: every sequence with rows has at most one part-filled tile.
int64_t flash_tiles(int M, int B, int G, int RG) {
  return B == 1 ? plan_tiles(M, G, 32 * RG) : (int64_t)M * G / (32 * RG) + min(B, M);
}
size_t flash_bytes(int M, int G, int Hkv, int RG, int D, int cus) {
  return (size_t)flash_slots(M, G, Hkv, RG, cus) * Hkv * flash_slot_bytes(RG, D);
}

// The work buffer begins with the arrival counters, in every call: one buffer may serve calls of all forms. Pairs (sequence, kv
// head) with more than one split count there, or slots, two for each CU at most.
constexpr int kCounters = 4096;
constexpr size_t kWorkHead = kCounters * 4;

// Splits of a decode step's pairs. With at most an eighth as many pairs as CUs, blocks of 8 waves and the slot cache's rule
// (decode_split.h): the step is a chain of latencies. With more, blocks of 4 waves and a split per 256 keys (pairs for a
// quarter of the CUs), 320 (for one a CU) or 768: a batch of mixed lengths ends with its longest blocks, while every split
// costs its part's way through memory; equal lengths lose 1 to 3 %. Measured against that rule for all, us: 100 sequences of
// 50 to 2000 keys, 12/2 heads of 128, 35.7 -> 28.0; 31 of 1 to 300, 32/8 of 128, 11.4 -> 8.5; 120 of 1 to 700, 32/4 of 64, 15.3
// -> 12.3; 30 of 500 to 4000, 32/8 of 128, 65.3 -> 60.4; 48 of 100 to 2000 46.8 -> 46.8; 16 of 4097 52.3 -> 54.0. (192, 320
// or 352 keys for the first two and 704 or 1024 for the last: within 3 % over 17 batches, 288 and 12 splits worse.) From two
// pairs a CU on, a split per 4096 keys only, so that one long sequence does not hold up the batch: 64 of 1000 keys lose 12 %
// by a second split (beyond kCounters pairs, which have no counters, none). A sequence's splits depend on the batch's
// size, not on the other lengths.
void step_splits(int B, int Hkv, int G, int cus, StepPlan& f, bool& wide) {
  const int64_t pairs = (int64_t)B * Hkv;
  f.K = 0;
  wide = G <= 8 && decode_splits(B, Hkv, cus) >= kDaWideSplits;
  if (wide) {
    f.S = f.S1 = decode_splits_wide(B, Hkv, cus);
    return;
  }
  f.S1 = 1;
  f.S = pairs > kCounters ? 1 : (int)std::min((int64_t)8, 4 * kCounters / pairs);
  if (pairs < 2 * cus) f.S = max(f.S, decode_splits(B, Hkv, cus));
  f.K = 4 * pairs <= cus ? 256 : pairs <= cus ? 320 : pairs < 2 * cus ? 768 : 4096;
}
// Floats of the partial results' m and l, a multiple of 4 (O is read in 16-byte pieces).
size_t step_ml(const StepPlan& f, int B, int Hq) { return ((size_t)B * Hq * f.S * 2 + 3) & ~(size_t)3; }
size_t step_bytes(const StepPlan& f, int B, int Hq, int D) { return (step_ml(f, B, Hq) + (size_t)B * Hq * f.S * D) * 4; }

constexpr int kRowsMinSplit = 1;  // key tiles
constexpr int kRowsFan = 32;      // the block that arrives last joins all splits of a tile

// Column blocks of 16 packed rows of the kernel for few rows, or 0: the row tiles of pages_block. It has no stages to fill and
// one level of joins, but reads a run's keys once per 32 packed rows instead of 64 or 128. So it takes
//  * batches of a tile per sequence (on average, with no run of more than 384 packed rows while every sequence has a row):
//    pages / rows, us, 32/8 heads of 128: 1 row after 4000 18.0 / 11.9, 48 after 100 to 2000 57.4 / 45.5, 8 x 5 rows after 700
//    to 4000 23.4 / 21.1, 64 x 2 after 1000 60.1 / 49.7, 63 after 1000 and 65 after 16000 245 / 156, 31 after 500 and 97 (388
//    packed) after 8000 59.0 / 89.6;
//  * and where the tiles are at most half as many as CUs and can read 1536 keys for each CU in all, going by the table's
//    width, the one bound that the host has: 32 rows after 1000 21.3 / 14.0, after 8000 30.4 / 22.9, 100 after 4000 27.3 / 32.4,
//    64 after 16000 40.6 / 53.2, 32 after 32000 48.5 / 60.5; 12/2 heads of 128, 19 after 1881 22.7 / 14.5, 250 after 1000
//    22.8 / 18.1. In tables of 1, 8 and 32 times the width that they need, 32 rows after 1000 take 13.9, 13.9 and 21.1, 100 rows
//    17.4, 21.3 and 21.2.
int row_columns(int M, int B, int G, int Hkv, int64_t cap, int cus) {
  const int tiles = plan_tiles(M, G, 32);
  const bool one = (int64_t)M * G <= 32 * (int64_t)B && (int64_t)(M - min(B, M) + 1) * G <= 384;
  const bool few = 2 * (int64_t)max(min(B, M), tiles) * Hkv <= cus && tiles * Hkv * cap <= 1536 * (int64_t)cus;
  return !one && !few ? 0 : (int64_t)M * G <= 16 * (int64_t)B ? 1 : 2;
}
// Its row tiles (at most), and how they are split. Up to a tile for every second CU, blocks of 8 waves and flash_unit's plan
// (slots > 0), which knows all lengths; beyond, blocks of 4 waves and a step's splits.
int64_t rows_plan(int M, int B, int G, int Hkv, int NC, int cus, StepPlan& f, int& slots) {
  const int most = max(min(B, M), plan_tiles(M, G, 16 * NC));
  const int64_t tiles = B == 1 ? most : (int64_t)M * G / (16 * NC) + min(B, M);
  bool wide;
  step_splits(most, Hkv, 16, cus, f, wide);  // (16 heads: never blocks of 8 waves)
  if (tiles * Hkv > kCounters) f.S = 1;
  slots = 2 * (int64_t)most * Hkv <= cus ? 2 * cus / Hkv : 0;
  return tiles;
}
size_t rows_bytes(const StepPlan& f, int64_t tiles, int slots, int Hkv, int NC, int D) {
  return (slots ? slots : f.S == 1 ? 0 : (size_t)tiles * f.S) * Hkv * 16 * NC * (D + 2) * 4;
}

// Splits of a prefix of `shared` positions for T row tiles, and whether the own keys go into the same launch (`mixed`): where
// half of the CUs are through with the prefix in 12 key tiles, the other half takes the own keys; beyond that the prefix needs
// all of them, and the own keys are faster in small blocks after it. Apart / mixed, us, 32/8 heads of 128: 32 sequences
// after 8192 with 300 own keys 33.2 / 25.3, 8 after 8192 23.7 / 18.5, 32 after 16384 (8 tiles) with 30 32.0 / 29.2, 64 after
// 32768 (32 tiles) with 200 66.9 / 81.5, 8 after 32768 (16 tiles) with 300 42.4 / 44.1.
int prefix_splits(int T, int Hkv, int shared, int cus, bool& mixed) {
  const int te = plan_key_tiles(shared), half = max(1, cus / 2 / max(1, T * Hkv)), S = max(1, min(half, te / 4));
  mixed = 2 * T * Hkv <= cus && (te + S - 1) / S <= 12;
  return mixed ? S : max(1, min(cus / max(1, T * Hkv), (te + 1) / 2));
}

// Whether a decode step that reads the prefix again for every sequence is faster. Its re-reads mostly hit the caches, at 14
// TB/s; reading it once costs 5 us (a second launch, the parts' way through memory) and the prefix at 8 TB/s. Measured with 2
// to 64 sequences after prefixes of 512 to 32768, 20 or 300 keys of their own, in 32/8 and 12/2 heads of 128 and 32/4 of
// 64: 0.5 % above the faster of the two on average (us, once / again, 300 own keys, 32/8 of 128: 4 after 4096 16.6 / 14.1,
// after 16384 23.4 / 27.8; 8 after 2048 16.7 / 15.0, after 4096 17.4 / 19.9; 32 after 1024 22.8 / 25.1, after 4096 23.2 / 52.1).
bool prefix_reread(const AttnArgs& a, int D) {
  const double mb = 4e-6 * a.shared * a.Hkv * D;
  return a.B * mb / 14 < 5 + mb / 8;
}

// Largest grid's blocks and what a kernel's LDS limit needs; 0, or a negative code.
template <typename K>
int flash_fits(K kern, int threads, size_t lds, const char* who) {
  const int bpc = hi_blocks_per_cu(reinterpret_cast<const void*>(kern), threads, lds);  // lifts the LDS limit
  if (bpc < 0) return -2;
  if (bpc == 0) HI_FAIL("%s: the kernel does not fit on a CU", who);
  return 0;
}

template <int D, int RG, class C>
int flash_launch(const AttnArgs& a, const C& c, int cus, void* work, hipStream_t s, const char* who) {
  const int G = a.G, cap = c.W << c.shift;
  FlashPlan f{};
  const int slots = cap > kPlanMinSplit * kPlanTile ? flash_slots(a.M, G, a.Hkv, RG, cus) : 0;
  if (slots) {
    f.slots = slots;
    f.cus = cus;
    f.least = kPlanMinSplit;
    f.b1 = cus / a.Hkv;
    f.b2 = 2 * cus / a.Hkv;
    f.counters = (int*)work;
    f.ml = (float*)((char*)work + kWorkHead);
    f.po = f.ml + (size_t)slots * a.Hkv * 2 * 32 * RG;
  }
  const int64_t units = std::max(flash_tiles(a.M, a.B, G, RG), (int64_t)slots);
  // (the tiles of any start, also one that gives the same rows to every sequence, are counted in int)
  if (units > 65535 || (int64_t)a.B * plan_tiles(a.M, G, 32 * RG) > INT32_MAX)
    HI_FAIL("%s: %d rows of %d sequences are too many", who, a.M, a.B);
  const auto kern = attn_pages_kernel<D, RG, C>;
  const size_t lds = C::kF8 ? Fp8Smem<D, RG>::kBytes : FpSmem<D, RG>::kBytes;
  if (const int rc = flash_fits(kern, 128 * RG, lds, who)) return rc;
  hipLaunchKernelGGL(kern, dim3(a.Hkv, (unsigned)units), dim3(128 * RG), lds, s, a, c, f);
  HI_TRY(hipGetLastError());
  return 0;
}

template <int D, int NC, int NWV, class C>
int rows_launch(const AttnArgs& a, const C& c, const StepPlan& f, const FlashPlan& fp, int64_t tiles, int64_t units,
                hipStream_t s, const char* who) {
  if (units > 65535 || (int64_t)a.B * plan_tiles(a.M, a.G, 16 * NC) * f.S > INT32_MAX)  // as flash_launch
    HI_FAIL("%s: %d rows of %d sequences are too many", who, a.M, a.B);
  const auto kern = attn_rows_kernel<D, NC, NWV, C>;
  const size_t lds = sizeof(RowsSmem<D, NC, NWV>);
  if (const int rc = flash_fits(kern, NWV * 64, lds, who)) return rc;
  hipLaunchKernelGGL(kern, dim3(a.Hkv, (unsigned)units), dim3(NWV * 64), lds, s, a, c, f, fp, (int)tiles);
  HI_TRY(hipGetLastError());
  return 0;
}

template <int D, int NC, class C>
int rows_run(const AttnArgs& a, const C& c, int cus, void* work, hipStream_t s, const char* who) {
  StepPlan f;
  FlashPlan fp{};
  const int64_t tiles = rows_plan(a.M, a.B, a.G, a.Hkv, NC, cus, f, fp.slots);
  f.counters = (int*)work;
  f.ml = (float*)((char*)work + kWorkHead);
  f.po = f.ml + (fp.slots ? fp.slots : (size_t)tiles * f.S) * a.Hkv * 2 * 16 * NC;
  if (!fp.slots) return rows_launch<D, NC, 4>(a, c, f, fp, tiles, tiles * f.S, s, who);
  fp.cus = cus;
  fp.b1 = cus / a.Hkv;
  fp.b2 = 2 * cus / a.Hkv;
  fp.least = kRowsMinSplit;
  fp.fan = kRowsFan;
  return rows_launch<D, NC, 8>(a, c, f, fp, tiles, std::max(tiles, (int64_t)fp.slots), s, who);
}

template <int D, class C>
int step_run(const AttnArgs& a, const C& c, int cus, void* work, hipStream_t s, const char* who) {
  if (a.B > 65535) HI_FAIL("%s: %d sequences (at most 65535)", who, a.B);
  StepPlan f;
  bool wide;
  step_splits(a.B, a.Hkv, a.G, cus, f, wide);
  f.counters = (int*)work;
  f.ml = (float*)((char*)work + kWorkHead);
  f.po = f.ml + step_ml(f, a.B, a.Hq);
  const dim3 grid(a.Hkv, a.B, f.S);
  const int G = a.G;
  if (G > 8) hipLaunchKernelGGL((attn_step_kernel<16, D, 4, C>), grid, dim3(256), 0, s, a, c, f);
  else if (G > 4) {
    if (wide) hipLaunchKernelGGL((attn_step_kernel<8, D, 8, C>), grid, dim3(512), 0, s, a, c, f);
    else hipLaunchKernelGGL((attn_step_kernel<8, D, 4, C>), grid, dim3(256), 0, s, a, c, f);
  } else {
    if (wide) hipLaunchKernelGGL((attn_step_kernel<4, D, 8, C>), grid, dim3(512), 0, s, a, c, f);
    else hipLaunchKernelGGL((attn_step_kernel<4, D, 4, C>), grid, dim3(256), 0, s, a, c, f);
  }
  HI_TRY(hipGetLastError());
  return 0;
}

// Splits of the sequences' own keys behind a shared prefix. In the prefix's launch, one per 512 keys (256 in blocks of 4
// waves), up to 8; in their own, as any decode step in blocks of 4 waves.
void own_splits(int B, int Hkv, int RG, int cus, bool mixed, StepPlan& f) {
  bool wide;
  step_splits(B, Hkv, 16, cus, f, wide);  // (more than 8 heads a group: never blocks of 8 waves)
  if (!mixed) return;
  f.S = 8;
  f.K = RG == 2 ? 256 : 512;
}

size_t shared_bytes(int B, int Hq, int Hkv, int D, int cus) {
  size_t most = 0;
  StepPlan st;
  bool wide;
  step_splits(B, Hkv, Hq / Hkv, cus, st, wide);  // the prefix read again for every sequence
  most = step_bytes(st, B, Hq, D);
  const int RG = flash_row_groups(B, 1, Hq / Hkv), T = plan_tiles(B, Hq / Hkv, 32 * RG);
  for (const bool mixed : {false, true}) {
    own_splits(B, Hkv, RG, cus, mixed, st);
    // (std::max: the host's plain max is one of ints)
    most = std::max(most, step_bytes(st, B, Hq, D) + (size_t)T * max(1, cus / max(1, T * Hkv)) * Hkv * flash_slot_bytes(RG, D));
  }
  return most;
}

template <int D, int RG>
int shared_launch(const AttnArgs& a, const PagedCache& c, int cus, void* work, hipStream_t s, const char* who) {
  const int G = a.G, T = plan_tiles(a.M, G, 32 * RG), BQ = 32 * RG;
  if (a.B > 65535) HI_FAIL("%s: %d sequences (at most 65535)", who, a.B);
  bool mixed;
  FlashPlan f{};
  f.splits = prefix_splits(T, a.Hkv, a.shared, cus, mixed);
  f.slots = T * f.splits;
  StepPlan st;
  own_splits(a.B, a.Hkv, RG, cus, mixed, st);
  if (mixed) st.S = max(1, min(st.S, ((c.W << c.shift) - a.shared + st.K - 1) / st.K));
  st.counters = (int*)work;
  st.ml = (float*)((char*)work + kWorkHead);
  st.po = st.ml + step_ml(st, a.B, a.Hq);
  f.ml = st.po + (size_t)a.B * a.Hq * st.S * D;
  f.po = f.ml + (size_t)f.slots * a.Hkv * 2 * BQ;
  // twice the blocks that the prefix leaves room for (two blocks a CU at D = 64): fewer or more are slower
  const int room = (D == 64 ? 2 : 1) * cus - f.slots * a.Hkv, own = mixed ? max(1, min(a.B * st.S, 2 * room / a.Hkv)) : 0;
  const auto kern = G > 8 ? attn_prefix_kernel<16, D, RG> : G > 4 ? attn_prefix_kernel<8, D, RG> : attn_prefix_kernel<4, D, RG>;
  const size_t lds = FpSmem<D, RG>::kBytes;
  static_assert(sizeof(StepSmem<16, D, 2 * RG>) <= FpSmem<D, RG>::kBytes, "both kinds of blocks fit the LDS");
  if (const int rc = flash_fits(kern, 128 * RG, lds, who)) return rc;
  hipLaunchKernelGGL(kern, dim3(a.Hkv, f.slots + own), dim3(128 * RG), lds, s, a, c, f, st, T);
  HI_TRY(hipGetLastError());
  if (mixed) {
    hipLaunchKernelGGL((attn_parts_kernel<D>), dim3(a.Hkv, a.B), dim3(kPartThreads), 0, s, a, c.W << c.shift, f, st, BQ);
  } else {
    const dim3 grid(a.Hkv, a.B, st.S);
    if (G > 8) hipLaunchKernelGGL((attn_own_kernel<16, D>), grid, dim3(kPartThreads), 0, s, a, c, f, st, BQ);
    else if (G > 4) hipLaunchKernelGGL((attn_own_kernel<8, D>), grid, dim3(kPartThreads), 0, s, a, c, f, st, BQ);
    else hipLaunchKernelGGL((attn_own_kernel<4, D>), grid, dim3(kPartThreads), 0, s, a, c, f, st, BQ);
  }
  HI_TRY(hipGetLastError());
  return 0;
}

int attn_check(const char* who, const void* q, int ldq, const int* pos, const void* out, int ldo, const float* lse, int M,
               int Hq, int Hkv, int D) {
  if (M < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || Hq / Hkv > 16) HI_FAIL("%s: M %d, Hq %d, Hkv %d (Hq / Hkv in 1..16)", who, M, Hq, Hkv);
  if ((int64_t)M * Hq > (1 << 27)) HI_FAIL("%s: %d rows of %d heads", who, M, Hq);
  if (M == 0) return 0;
  if (!q || !pos || !out || ((uintptr_t)q & 15) || ldq % 8 || ldq < Hq * D || ((uintptr_t)pos & 3))
    HI_FAIL("%s: q must be 16-byte aligned with ldq %% 8 == 0 and ldq >= Hq * D, pos 4-byte aligned, none null", who);
  if (((uintptr_t)out & 7) || ldo % 4 || ldo < Hq * D) HI_FAIL("%s: out must be 8-byte aligned, ldo %% 4 == 0, ldo >= Hq * D", who);
  if ((uintptr_t)lse & 3) HI_FAIL("%s: lse must be 4-byte aligned", who);
  if (!in_place_or_apart(q, 2 * (int64_t)ldq, 2 * (int64_t)Hq * D, out, 2 * (int64_t)ldo, 2 * (int64_t)Hq * D, M))
    HI_FAIL("%s: out must be q (with its row stride) or apart from it", who);
  return 0;
}

template <class C>
int attn_run(const AttnArgs& a, const C& c, int D, int cus, void* work, hipStream_t s, const char* who) {
  const int G = a.G;
  if (a.start) {
    const int NC = row_columns(a.M, a.B, G, a.Hkv, (int64_t)c.W << c.shift, cus);
    if (NC == 1) return D == 64 ? rows_run<64, 1>(a, c, cus, work, s, who) : rows_run<128, 1>(a, c, cus, work, s, who);
    if (NC == 2) return D == 64 ? rows_run<64, 2>(a, c, cus, work, s, who) : rows_run<128, 2>(a, c, cus, work, s, who);
    const bool small = flash_row_groups(a.M, a.B, G) == 2;
    return D == 64 ? (small ? flash_launch<64, 2>(a, c, cus, work, s, who) : flash_launch<64, 4>(a, c, cus, work, s, who))
                   : (small ? flash_launch<128, 2>(a, c, cus, work, s, who) : flash_launch<128, 4>(a, c, cus, work, s, who));
  }
  if constexpr (!C::kF8)
    if (a.shared && !prefix_reread(a, D)) {
      const bool small = flash_row_groups(a.M, 1, G) == 2;
      return D == 64 ? (small ? shared_launch<64, 2>(a, c, cus, work, s, who) : shared_launch<64, 4>(a, c, cus, work, s, who))
                     : (small ? shared_launch<128, 2>(a, c, cus, work, s, who) : shared_launch<128, 4>(a, c, cus, work, s, who));
    }
  return D == 64 ? step_run<64>(a, c, cus, work, s, who) : step_run<128>(a, c, cus, work, s, who);
}

// What a call's parts need behind the counters. More rows or sequences may need less: the splits get fewer.
size_t paged_bytes(int M, int B, int Hq, int Hkv, int D, bool ragged, int cus) {
  StepPlan f;
  if (!ragged) {
    bool wide;
    step_splits(B, Hkv, Hq / Hkv, cus, f, wide);
    return step_bytes(f, B, Hq, D);
  }
  const int G = Hq / Hkv, NC = row_columns(M, B, G, Hkv, 1, cus);  // a wider table may take the other kernel
  size_t rows = 0;
  if (NC) {
    int slots;
    const int64_t tiles = rows_plan(M, B, G, Hkv, NC, cus, f, slots);
    rows = rows_bytes(f, tiles, slots, Hkv, NC, D);
  }
  return std::max(rows, flash_bytes(M, G, Hkv, flash_row_groups(M, B, G), D, cus));
}

// What any call of at most M rows of at most B sequences needs; ragged: with start or without. Beyond kCounters pairs a step has one
// split, its need grows with B. Row tiles need the same slots for any M that has some, of 4 row groups once a sequence can have over 64
// packed rows; so do the few rows' blocks of 8 waves, smaller ones. Their blocks of 4 waves have splits while tiles * Hkv <=
// kCounters: for every number of sequences with rows (more of them than rows are as many as rows) and NC, the most tiles of those.
size_t paged_most_bytes(int M, int B, int Hq, int Hkv, int D, bool ragged, int cus) {
  const int G = Hq / Hkv, few = kCounters / Hkv;
  const int steps = ragged ? min(M, B) : B;  // a step has as many rows as sequences
  size_t most = paged_bytes(steps, steps, Hq, Hkv, D, false, cus);
  for (int b = 1; b <= min(steps, few); b++) most = std::max(most, paged_bytes(b, b, Hq, Hkv, D, false, cus));
  if (!ragged) return most;
  most = std::max(most, flash_bytes(1, G, Hkv, (int64_t)M * G > 64 ? 4 : 2, D, cus));
  for (int b = 1; b <= min(steps, few); b++)
    for (const int NC : {1, 2}) {
      StepPlan f;
      bool wide;
      step_splits(b, Hkv, 16, cus, f, wide);  // as rows_plan
      const int64_t rows = std::min((int64_t)M, 16 * NC * (int64_t)b / G);
      const int64_t tiles = std::min(rows * G / (16 * NC) + b, (int64_t)few);
      most = std::max(most, rows_bytes(f, tiles, 0, Hkv, NC, D));
    }
  return most;
}

size_t shared_most_bytes(int B, int Hq, int Hkv, int D, int cus) {
  size_t most = shared_bytes(B, Hq, Hkv, D, cus);
  // beyond both, one split: the need grows with B
  const int64_t few = max(kCounters / Hkv, 128 * (cus / Hkv + 1) / (Hq / Hkv) + 1);
  for (int b = 1; b <= std::min((int64_t)B, few); b++) most = std::max(most, shared_bytes(b, Hq, Hkv, D, cus));
  return most;
}

// Sizes of a work buffer's call that the attention can take.
bool work_sizes(int M, int B, int Hq, int Hkv, int D) {
  return M >= 0 && B >= 0 && Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && Hq / Hkv <= 16 && (D == 64 || D == 128) &&
         (int64_t)max(M, B) * Hq <= (1 << 27);
}

// hi_attn_paged and hi_attn_paged8 behind the check of their cache.
template <class C>
int attn_paged_call(const char* who, const C& c, const void* q, int ldq, const int* start, const int* pos, void* out, int ldo, float* lse,
                    int M, int B, int Hq, int Hkv, int D, void* work, size_t work_bytes, hipStream_t s) {
  if (B == 0 && (M == 0 || start)) return 0;  // rows of no sequence
  if (attn_check(who, q, ldq, pos, out, ldo, lse, M, Hq, Hkv, D)) return -1;
  if (!start && M != B) HI_FAIL("%s: %d rows for %d sequences (one each without start)", who, M, B);
  if ((uintptr_t)start & 3) HI_FAIL("%s: start must be 4-byte aligned", who);
  if (M == 0) return 0;
  const size_t need = hi_attn_paged_work_bytes(M, B, Hq, Hkv, D, start != nullptr);
  if (!work || ((uintptr_t)work & 15) || work_bytes < need)
    HI_FAIL("%s: work of %zu bytes (at least %zu, 16-byte aligned)", who, work_bytes, need);
  const HiDevice* d = hi_device();
  if (!d) return -2;
  const AttnArgs a{(const f16*)q, ldq, (f16*)out, ldo, lse, start, pos, M, B, Hq, Hkv, 0, Hq / Hkv, plan_magic(Hq / Hkv),
                   1.4426950408889634f / sqrtf((float)D)};
  return attn_run(a, c, D, d->cus, work, s, who);
}

}  // namespace
