// Serving from a paged key/value cache: rotation and cache write of projected rows (hi_rope_cache_paged), attention over
// the pages (hi_attn_paged) and attention of a batch whose sequences share their first positions (hi_attn_shared).
// The cache and its table: paged.h.
#include "flash.h"
#include "paged.h"
#include "paged_plan.h"

namespace {

// ------------------------------------------------------------------ rotation and cache write
struct RopePagedArgs {
  f16* qkv;
  int64_t ldq;
  f16* qo;
  int64_t ldqo;
  int Hq, Hkv, D, rot, cs_rows, B;
  const void* cs;
  const int *seq, *pos;
};

// Where row m's k and v go: the first element of kv head 0's row on its page, or -1 if the row has no place (a negative
// position, one behind the table or the cs rows, a sequence outside the table, no page).
__device__ __forceinline__ int64_t rope_place(const RopePagedArgs& a, const PagedCache& c, int m, int& p) {
  p = a.pos[m];
  const int b = a.seq ? a.seq[m] : m;
  if ((unsigned)p >= (unsigned)min(c.capacity(), a.cs_rows) || (unsigned)b >= (unsigned)a.B) return -1;
  const int id = c.entry(b, p >> c.shift);
  if (!c.has(id)) return -1;
  return (int64_t)id * c.stride + (int64_t)(p & ((1 << c.shift) - 1)) * a.D;
}

// One rotated pair: products of fp16 numbers are exact in fp32, each result is rounded to fp16 once.
__device__ __forceinline__ void turn(f16& x, f16& y, float c, float s) {
  const float a = (float)x, b = (float)y;
  x = (f16)__builtin_fmaf(a, c, -(b * s));
  y = (f16)__builtin_fmaf(b, c, a * s);
}

// Any alignment and any even rot: block per row, a wave per head at a time, a lane per pair or element.
template <typename CS>
__global__ void __launch_bounds__(256) rope_paged_any_kernel(RopePagedArgs a, PagedCache c, bool inter) {
  const int m = blockIdx.x, lane = threadIdx.x & 63;
  int p;
  const int64_t at = rope_place(a, c, m, p);
  if (at < 0) return;
  const int half = a.rot / 2, D = a.D, page = 1 << c.shift;
  const CS* tab = (const CS*)a.cs + (int64_t)p * a.rot;
  for (int h = threadIdx.x >> 6; h < a.Hq + 2 * a.Hkv; h += 4) {
    const f16* src = a.qkv + (int64_t)m * a.ldq + (int64_t)h * D;
    f16* dst = h < a.Hq ? a.qo + (int64_t)m * a.ldqo + (int64_t)h * D
               : h < a.Hq + a.Hkv ? const_cast<f16*>(c.kp) + at + (int64_t)(h - a.Hq) * page * D
                                  : const_cast<f16*>(c.vp) + at + (int64_t)(h - a.Hq - a.Hkv) * page * D;
    const int rot = h < a.Hq + a.Hkv ? a.rot : 0;
    for (int j = lane; j < rot / 2; j += 64) {
      const int i0 = inter ? 2 * j : j, i1 = inter ? 2 * j + 1 : j + half;
      f16 x = src[i0], y = src[i1];
      turn(x, y, (float)tab[2 * j], (float)tab[2 * j + 1]);
      dst[i0] = x;
      dst[i1] = y;
    }
    if (src != dst)
      for (int j = rot + lane; j < D; j += 64) dst[j] = src[j];
  }
}

// ------------------------------------------------------------------ attention
struct AttnArgs {
  const f16* q;
  int64_t ldq;
  f16* out;
  int64_t ldo;
  float* lse;  // [Hq][M] or null
  const int *start, *pos;
  int M, B, Hq, Hkv, shared;  // positions below `shared` are on the pages of table row 0
  float scale_log2;
};

// One block per (row, query head): tiles of 256 keys, a key per thread for the logits, a dim per thread for P.V.
template <int D>
__global__ void __launch_bounds__(256) attn_paged_simple_kernel(AttnArgs a, PagedCache c) {
  __shared__ float sp[256], red[4], sq[D], so[256];
  __shared__ int sid[256];
  const int m = blockIdx.x, h = blockIdx.y, hk = h / (a.Hq / a.Hkv), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int b = m, t = 0;
  if (a.start) {
    for (b = 0; b < a.B; b++)
      if (a.start[b] <= m && m < a.start[b + 1]) break;
    if (b == a.B) return;
    t = m - a.start[b];
  }
  const int n = (int)min((int64_t)a.pos[b] + t + 1, (int64_t)c.capacity());
  if (tid < D) sq[tid] = (float)a.q[(int64_t)m * a.ldq + h * D + tid];
  float mx = -__builtin_huge_valf(), l = 0.f, o = 0.f;
  const int page = 1 << c.shift, d = tid % D, part = tid / D;
  for (int k0 = 0; k0 < n; k0 += 256) {
    __syncthreads();
    const int k = k0 + tid;
    const int id = k < n ? c.entry(k < a.shared ? 0 : b, k >> c.shift) : -1;
    float x = -__builtin_huge_valf();
    if (c.has(id)) {
      const f16* kr = c.kp + id * c.stride + ((int64_t)hk * page + (k & (page - 1))) * D;
      float s = 0.f;
      for (int i = 0; i < D; i++) s = __builtin_fmaf(sq[i], (float)kr[i], s);
      x = s * a.scale_log2;
    }
    const float wm = wave_max(x);
    if (lane == 0) red[wave] = wm;
    __syncthreads();
    const float mn = fmaxf(mx, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float ref = mn == -__builtin_huge_valf() ? 0.f : mn;
    const float alpha = exp2f(mx - ref), p = exp2f(x - ref);
    mx = mn;
    sp[tid] = p;
    sid[tid] = c.has(id) ? id : -1;
    l = l * alpha + p;
    o *= alpha;
    __syncthreads();
    for (int j = part; j < 256; j += 256 / D)
      if (sid[j] >= 0) o = __builtin_fmaf(sp[j], (float)c.vp[sid[j] * c.stride + ((int64_t)hk * page + ((k0 + j) & (page - 1))) * D + d], o);
  }
  l = wave_sum(l);
  __syncthreads();
  if (lane == 0) red[wave] = l;
  so[tid] = o;
  __syncthreads();
  l = (red[0] + red[1]) + (red[2] + red[3]);
  if (tid < D) {
    for (int j = 1; j < 256 / D; j++) o += so[tid + j * D];
    a.out[(int64_t)m * a.ldo + h * D + tid] = (f16)(l == 0.f ? 0.f : o / l);
  }
  if (a.lse && tid == 0) a.lse[(int64_t)h * a.M + m] = mx + log2f(l);
}

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
// Where the row tiles are fewer than the GPU's CUs, their keys are split (paged_plan.h); a split stores its
// unnormalised O, m and l in fp32, in the lanes' order, and attn_join_kernel joins them.
struct FlashPlan {
  float *ml, *po;  // partial results: [slot][2][BQ] m and l, [slot][RG][D / 8][64][4] O
  int slots;       // slots there are, each of all kv heads
  int cus;         // > 0: split over that many
  int splits;      // of the shared prefix
};

// What a block works on; found by every wave by itself from start and pos.
struct FlashUnit {
  int b, row0, n, pos;   // sequence, its first row, rows, first position
  int tile, splits, split, slot;  // slot of split 0 (meaningful with splits > 1)
};

__device__ __forceinline__ int wave_total(int v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}
__device__ __forceinline__ int64_t wave_total(int64_t v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}
__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, kWave);
    if (lane >= o) v += u;
  }
  return v;
}

// Unit `at` of the batch, or with TILES row tile `at` (split 0 of it); false if there are not so many. Wave-uniform.
template <int BQ, bool TILES>
__device__ __forceinline__ bool flash_unit(const AttnArgs& a, int cap, const FlashPlan& f, int at, int lane, FlashUnit& u) {
  const int G = a.Hq / a.Hkv;
  struct Seq { int row0, n, pos, tiles, end; };
  auto seq = [&](int b) {
    Seq s{0, 0, 0, 0, 0};
    if (b < a.B) {
      const int s0 = a.start[b], s1 = a.start[b + 1];
      s.pos = a.pos[b];
      s.row0 = plan_first(s0, a.M);
      s.n = plan_rows(s0, s1, a.M);
      s.tiles = plan_tiles(s.n, G, BQ);
      s.end = plan_end(s.pos, s.n, cap);
    }
    return s;
  };
  int L = kPlanNoSplit;
  const Seq first = seq(lane);
  if (f.cus > 0) {
    int T = 0, longest = 0;
    int64_t work = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const Seq s = b0 ? seq(b0 + lane) : first;
      T += s.tiles;
      work += (int64_t)s.tiles * s.end;
      if (s.tiles) longest = max(longest, s.end);
    }
    T = wave_total(T);
    const int budget = plan_budget(T, a.Hkv, f.cus);
    if (budget > 0) {
      work = wave_total(work);
      for (int o = 32; o > 0; o >>= 1) longest = max(longest, __shfl_xor(longest, o, kWave));
      for (L = plan_length(work, budget); L < longest; L = plan_longer(L)) {
        int units = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
          const Seq s = b0 ? seq(b0 + lane) : first;
          units += s.tiles * plan_splits(s.end, L);
        }
        if (wave_total(units) <= min(budget, f.slots)) break;
      }
    }
  }
  int before = 0, slot = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Seq s = b0 ? seq(b0 + lane) : first;
    const int splits = plan_splits(s.end, L);
    const int n = TILES ? s.tiles : s.tiles * splits, own = splits > 1 ? s.tiles * splits : 0;
    const int upto = wave_scan(n, lane), slots = wave_scan(own, lane);
    const uint64_t hit = __ballot(before + upto > at);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto take = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      u.b = b0 + l;
      u.row0 = take(s.row0);
      u.n = take(s.n);
      u.pos = take(s.pos);
      u.splits = take(splits);
      const int tiles = take(s.tiles), i = at - before - (take(upto) - take(n));
      u.tile = tiles - 1 - (TILES ? i : i / u.splits);  // the most keys first
      u.split = TILES ? 0 : i % u.splits;
      u.slot = slot + take(slots) - take(own) + u.tile * u.splits;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    slot += __builtin_amdgcn_readlane(slots, 63);
  }
  return false;
}

template <int D, int RG, bool PREFIX>
__global__ void __launch_bounds__(128 * RG) attn_pages_kernel(AttnArgs a, PagedCache c, FlashPlan f) {
  constexpr int NW = 2 * RG, BQ = 32 * RG;
  constexpr int CPR = D / 8;                   // 16-byte chunks per key row
  constexpr int IPW = kFpBKV * CPR / 64 / NW;  // DMA instructions per wave per tile and operand
  constexpr int DT = D / 32;                   // 32-row output tiles of O^T
  constexpr int NQ = D / 16;                   // MFMAs of one 32-key block's logits
  constexpr int KPW = kFpBKV / NW;             // keys of a tile that a wave fetches
  constexpr int NG = KPW / 8;                  // in groups of 8, one page each
  constexpr int IPG = IPW / NG;                // DMA instructions per group
  static_assert(IPW * 64 * NW == kFpBKV * CPR && IPG * NG == IPW, "tile DMA split");
  using Sm = FpSmem<D, RG>;
  extern __shared__ u32x4 fp_smem[];
  u32x4* const ks_ = fp_smem;                                // [2][kTile]: K stages
  u32x4* const vs_ = fp_smem + kFpStages * Sm::kTile;        // [2][kTile]: V stages
  f32x16* const mo = reinterpret_cast<f32x16*>(fp_smem);     // [RG][DT][64]: the merge
  float* const ml = reinterpret_cast<float*>(fp_smem + Sm::kMl);  // [2][RG][64]: the second waves' m and l
  int* const flag = reinterpret_cast<int*>(fp_smem + Sm::kMl);    // [NW], before the loop

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wave % RG, kh = wave / RG;     // row group, key half
  const int fr = lane & 31, fk = lane >> 5;
  const int G = a.Hq / a.Hkv, page = 1 << c.shift, cap = c.capacity();
  const int hk = blockIdx.x % a.Hkv;            // blocks of a kv head on as few XCDs as there can be
  FlashUnit u;
  int end;  // keys that some row of the tile sees
  if constexpr (PREFIX) {
    u = FlashUnit{0, 0, a.M, 0, (int)(blockIdx.x / a.Hkv) / f.splits, f.splits, (int)(blockIdx.x / a.Hkv) % f.splits, 0};
    u.slot = u.tile * f.splits;
    int most = -1;  // the last position of any of the tile's rows
    for (int i = u.tile * BQ + lane; i < min((u.tile + 1) * BQ, u.n * G); i += 64) most = max(most, a.pos[i / G]);
    for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, kWave));
    end = __builtin_amdgcn_readfirstlane(max(min(most, a.shared - 1), -1) + 1);
  } else {
    if (!flash_unit<BQ, false>(a, cap, f, blockIdx.x / a.Hkv, lane, u)) return;
    end = plan_tile_end(u.pos, u.n, u.tile, G, BQ, cap);
  }
  int kb, kv_end;
  plan_range(PREFIX ? a.shared : end, u.splits, u.split, kb, kv_end);
  kv_end = min(kv_end, end);
  const int nt = kv_end > kb ? (kv_end - kb + kFpBKV - 1) / kFpBKV : 0;

  // this lane's row and the last key it sees
  const int pr = u.tile * BQ + rg * 32 + fr;
  const bool row = pr < u.n * G;
  const int token = row ? pr / G : 0, h = hk * G + (row ? pr - token * G : 0);
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
    // whether some key of the block lies on no page
    const int tb = PREFIX ? 0 : u.b;  // table row
    bool hole = false;
    for (int i = (kb >> c.shift) + tid; i <= (kv_end - 1) >> c.shift; i += 128 * RG) hole |= !c.has(c.entry(tb, i));
    const bool any_hole = __any(hole);
    if (lane == 0) flag[wave] = any_hole;

    // DMA instruction i of this wave fills slots (wave IPW + i) * 64 + lane of a tile: slot s holds
    // key s / CPR, physical chunk s % CPR, i.e. logical chunk (s % CPR) ^ swz(key)
    int koff[IPW], voff[IPW];
#pragma unroll
    for (int i = 0; i < IPW; i++) {
      const int s = (wave * IPW + i) * 64 + lane, r = s / CPR, p = s % CPR;
      koff[i] = ((r & 7) * D + 8 * (p ^ k_swz<D>(r))) * 2;
      voff[i] = ((r & 7) * D + 8 * (p ^ v_swz<D>(r))) * 2;
    }
    // the groups' byte offsets in kp / vp and readable bytes: of the next K tile, and of the next V tile (one before)
    uint32_t klo[NG], khi[NG], vlo[NG], vhi[NG];
    int kn[NG], vn[NG];
    int key = kb + wave * KPW + 8 * (lane & (NG - 1)), id = -1;  // of the tile after: this lane's group and its page
    auto fetch = [&] { id = key < kv_end ? c.entry(tb, key >> c.shift) : -1; };
    auto take = [&] {
      const bool ok = c.has(id);
      const int64_t off = ok ? (id * c.stride + ((int64_t)hk * page + (key & (page - 1))) * D) * 2 : 0;
      const int n = ok ? min(8, kv_end - key) * D * 2 : 0;
#pragma unroll
      for (int g = 0; g < NG; g++) {
        klo[g] = __builtin_amdgcn_readlane((int)off, g);
        khi[g] = __builtin_amdgcn_readlane((int)(off >> 32), g);
        kn[g] = __builtin_amdgcn_readlane(n, g);
      }
      key += kFpBKV;
    };
    auto advance = [&] {
#pragma unroll
      for (int g = 0; g < NG; g++) {
        vlo[g] = klo[g];
        vhi[g] = khi[g];
        vn[g] = kn[g];
      }
      take();
      fetch();
      __builtin_amdgcn_sched_barrier(0);
    };
    auto group = [](const f16* base, uint32_t lo, uint32_t hi, int n) {
      return __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<f16*>(base) + (((uint64_t)hi << 32) | lo), (short)0, n,
                                               0x00020000);
    };
    auto issue_k = [&](int i, int st) {
      lds_dma16(group(c.kp, klo[i / IPG], khi[i / IPG], kn[i / IPG]), ks_ + st * Sm::kTile + (wave * IPW + i) * 64, koff[i]);
    };
    auto issue_v = [&](int i, int st) {
      lds_dma16(group(c.vp, vlo[i / IPG], vhi[i / IPG], vn[i / IPG]), vs_ + st * Sm::kTile + (wave * IPW + i) * 64, voff[i]);
    };
    fetch();
    take();
    fetch();

    __syncthreads();  // every wave's flag is written
    bool holes = false;
#pragma unroll
    for (int w = 0; w < NW; w++) holes |= flag[w] != 0;
    holes = __builtin_amdgcn_readfirstlane(holes);
    // tiles at the front that all of this wave's rows see whole (none for a wave without rows), and the last key any sees
    int least = row ? min(qpos, kv_end - 1) : kv_end, most = qpos;
    for (int x = 16; x > 0; x >>= 1) {
      least = min(least, __shfl_xor(least, x, kWave));
      most = max(most, __shfl_xor(most, x, kWave));
    }
    least = __builtin_amdgcn_readfirstlane(least);
    most = __builtin_amdgcn_readfirstlane(most);
    const int n_full = holes || most < 0 ? 0 : max(least + 1 - kb, 0) / kFpBKV;
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

#include "flash_tile.h"
  }

  // ---- merge the two key halves of each row group: the second wave hands (m, l, O) over
  wait_vmcnt<0>();
  __syncthreads();  // every wave is done with the stages, and no DMA is in flight
  l_i += xor32(l_i);
  if (kh == 1) {
#pragma unroll
    for (int dt = 0; dt < DT; dt++) mo[(rg * DT + dt) * 64 + lane] = o[dt];
    ml[rg * 64 + lane] = m_i;
    ml[(RG + rg) * 64 + lane] = l_i;
  }
  __syncthreads();
  if (kh == 1) return;
  const float m1 = ml[rg * 64 + lane], l1 = ml[(RG + rg) * 64 + lane];
  const float m = fmaxf(m_i, m1), ref = m == -__builtin_huge_valf() ? 0.f : m;  // -inf: no key seen
  const float a0 = __builtin_amdgcn_exp2f(m_i - ref), a1 = __builtin_amdgcn_exp2f(m1 - ref);
  const float l = l_i * a0 + l1 * a1;
  if (PREFIX || u.splits > 1) {  // rows behind the run hold what their zero queries gave; nothing reads them
    if (u.slot + u.split >= f.slots) return;
    const int64_t slot = (int64_t)(u.slot + u.split) * a.Hkv + hk;
    if (fk == 0) {
      f.ml[slot * 2 * BQ + rg * 32 + fr] = m;
      f.ml[slot * 2 * BQ + BQ + rg * 32 + fr] = l;
    }
    f32x4* po = reinterpret_cast<f32x4*>(f.po) + ((slot * RG + rg) * DT * 4) * 64 + lane;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
      const f32x16 o1 = mo[(rg * DT + dt) * 64 + lane];
#pragma unroll
      for (int g = 0; g < 4; g++) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = o[dt][4 * g + e] * a0 + o1[4 * g + e] * a1;
        po[(dt * 4 + g) * 64] = v;
      }
    }
    return;
  }
  if (!row) return;
  if (a.lse && fk == 0) a.lse[(int64_t)h * a.M + qrow] = m + log2f(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  f16* orow = a.out + qrow * a.ldo + h * D;
#pragma unroll
  for (int dt = 0; dt < DT; dt++) {
    const f32x16 o1 = mo[(rg * DT + dt) * 64 + lane];
#pragma unroll
    for (int g = 0; g < 4; g++) {
      f16x4 v;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = (f16)((o[dt][4 * g + e] * a0 + o1[4 * g + e] * a1) * inv);
      *reinterpret_cast<f16x4*>(orow + dt * 32 + 8 * g + 4 * fk) = v;
    }
  }
}

// Joins a tile's splits: block = (row tile, kv head, row group, 32 dims), wave = 8 of the dims, in the lanes' order of the
// partial results. m = max m_s, w_s = 2^(m_s - m), out = sum w_s O_s / sum w_s l_s.
template <int D, int RG>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a, int cap, FlashPlan f) {
  constexpr int BQ = 32 * RG, DT = D / 32;
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6, fr = lane & 31, fk = lane >> 5;
  int i = blockIdx.x;
  const int dt = i % DT, rg = i / DT % RG;
  i /= DT * RG;
  const int hk = i % a.Hkv, G = a.Hq / a.Hkv;
  FlashUnit u;
  if (!flash_unit<BQ, true>(a, cap, f, i / a.Hkv, lane, u) || u.splits == 1 || u.slot + u.splits > f.slots) return;
  const int pr = u.tile * BQ + rg * 32 + fr;
  if (pr >= u.n * G) return;
  const int token = pr / G, h = hk * G + pr - token * G;
  const float* ml = f.ml + ((int64_t)u.slot * a.Hkv + hk) * 2 * BQ + rg * 32 + fr;
  const f32x4* po = reinterpret_cast<const f32x4*>(f.po) + ((((int64_t)u.slot * a.Hkv + hk) * RG + rg) * DT * 4 + dt * 4 + g) * 64 + lane;
  const int64_t sm = (int64_t)a.Hkv * 2 * BQ, so = (int64_t)a.Hkv * RG * DT * 4 * 64;
  float m = -__builtin_huge_valf();
#pragma unroll 8
  for (int s = 0; s < u.splits; s++) m = fmaxf(m, ml[s * sm]);
  const float ref = m == -__builtin_huge_valf() ? 0.f : m;
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < u.splits; s++) {
    const float w = exp2f(ml[s * sm] - ref);
    const f32x4 v = po[s * so];
    l = __builtin_fmaf(w, ml[s * sm + BQ], l);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = __builtin_fmaf(w, v[e], o[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  f16x4 v;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = (f16)(o[e] * inv);
  *reinterpret_cast<f16x4*>(a.out + (int64_t)(u.row0 + token) * a.ldo + h * D + dt * 32 + 8 * g + 4 * fk) = v;
  if (a.lse && dt == 0 && g == 0 && fk == 0) a.lse[(int64_t)h * a.M + u.row0 + token] = m + log2f(l);
}

// Row groups per block: 4 (128 packed rows), or 2 where a sequence has 64 packed rows or less on average.
int flash_row_groups(int M, int B, int G) { return (int64_t)M * G <= 64 * (int64_t)B ? 2 : 4; }

size_t flash_slot_bytes(int RG, int D) { return (size_t)32 * RG * (D + 2) * 4; }

// Slots (each of all kv heads) that M rows of B sequences can need: those of plan_budget's largest, none where even full
// tiles are too many to be split.
int flash_slots(int M, int G, int Hkv, int RG, int cus) {
  const int least = plan_tiles(M, G, 32 * RG);
  return plan_budget(least, Hkv, cus) ? max(2 * cus / Hkv, 1) : 0;
}

template <int D, int RG>
int flash_launch(AttnArgs a, const PagedCache& c, int cus, void* work, hipStream_t s, const char* who) {
  const int G = a.Hq / a.Hkv, cap = c.W << c.shift;
  FlashPlan f{nullptr, nullptr, 0, 0, 1};
  const int slots = cap > kPlanMinSplit ? flash_slots(a.M, G, a.Hkv, RG, cus) : 0;
  if (slots) {
    f.slots = slots;
    f.cus = cus;
    f.ml = (float*)work;
    f.po = f.ml + (size_t)slots * a.Hkv * 2 * 32 * RG;
  }
  // every sequence with rows has at most one part-filled tile
  const int64_t tiles = a.B == 1 ? plan_tiles(a.M, G, 32 * RG) : (int64_t)a.M * G / (32 * RG) + min(a.B, a.M);
  const int64_t blocks = max(tiles, (int64_t)slots) * a.Hkv, join = tiles * a.Hkv * RG * (D / 32);
  // (the tiles of any start, also one that gives the same rows to every sequence, are counted in int)
  if (blocks > INT32_MAX || (slots && join > INT32_MAX) || (int64_t)a.B * plan_tiles(a.M, G, 32 * RG) > INT32_MAX) HI_FAIL("%s: %d rows are too many", who, a.M);
  const auto kern = attn_pages_kernel<D, RG, false>;
  const size_t lds = FpSmem<D, RG>::kBytes;
  const int bpc = hi_blocks_per_cu(reinterpret_cast<const void*>(kern), 128 * RG, lds);  // lifts the LDS limit
  if (bpc < 0) return -2;
  if (bpc == 0) HI_FAIL("%s: the kernel does not fit on a CU", who);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(128 * RG), lds, s, a, c, f);
  HI_TRY(hipGetLastError());
  if (slots) {
    hipLaunchKernelGGL((attn_join_kernel<D, RG>), dim3((unsigned)join), dim3(256), 0, s, a, cap, f);
    HI_TRY(hipGetLastError());
  }
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
  return 0;
}

int attn_run(const AttnArgs& a, const PagedCache& c, int D, int cus, void* work, hipStream_t s, const char* who) {
  if (a.start) {
    const bool small = flash_row_groups(a.M, a.B, a.Hq / a.Hkv) == 2;
    return D == 64 ? (small ? flash_launch<64, 2>(a, c, cus, work, s, who) : flash_launch<64, 4>(a, c, cus, work, s, who))
                   : (small ? flash_launch<128, 2>(a, c, cus, work, s, who) : flash_launch<128, 4>(a, c, cus, work, s, who));
  }
  const dim3 grid(a.M, a.Hq);
  if (D == 64) hipLaunchKernelGGL(attn_paged_simple_kernel<64>, grid, dim3(256), 0, s, a, c);
  else hipLaunchKernelGGL(attn_paged_simple_kernel<128>, grid, dim3(256), 0, s, a, c);
  HI_TRY(hipGetLastError());
  return 0;
}

}  // namespace

HI_EXPORT int hi_rope_cache_paged(void* qkv, int ldq, void* q_out, int ldqo, int M, int Hq, int Hkv, int D, const void* cs,
                                  int cs_rows, int cs_f32, int rot, int interleaved, const int* seq, const int* pos,
                                  void* kp, void* vp, long long page_stride, int pages, int page, const int* table, int ldt,
                                  int W, int B, void* stream) {
  const char* who = "hi_rope_cache_paged";
  PagedCache c;
  if (paged_cache(who, kp, vp, page_stride, pages, page, table, ldt, W, B, Hkv, D, c)) return -1;
  if (M < 0 || Hq < 1 || Hq > 4096 || rot < 0 || rot % 2 || rot > D || cs_rows < 1 || (!seq && M > B))
    HI_FAIL("%s: M %d, Hq %d, rot %d (even, at most D), cs rows %d, B %d (at least M without seq)", who, M, Hq, rot, cs_rows, B);
  if (M == 0) return 0;
  if (!qkv || !q_out || (rot && !cs) || !pos || ldq < (Hq + 2 * Hkv) * D || ldqo < Hq * D || ((uintptr_t)qkv & 1) ||
      ((uintptr_t)q_out & 1) || ((uintptr_t)cs & (cs_f32 ? 7 : 3)) || ((uintptr_t)pos & 3) || ((uintptr_t)seq & 3))
    HI_FAIL("%s: a null or misaligned pointer, ldq < (Hq + 2 Hkv) D or q_out's row stride < Hq D", who);
  if (!hi_device()) return -2;
  const RopePagedArgs a{(f16*)qkv, ldq, (f16*)q_out, ldqo, Hq, Hkv, D, rot, cs_rows, B, cs, seq, pos};
  if (cs_f32) hipLaunchKernelGGL(rope_paged_any_kernel<float>, dim3(M), dim3(256), 0, (hipStream_t)stream, a, c, interleaved != 0);
  else hipLaunchKernelGGL(rope_paged_any_kernel<f16>, dim3(M), dim3(256), 0, (hipStream_t)stream, a, c, interleaved != 0);
  HI_TRY(hipGetLastError());
  return 0;
}

HI_EXPORT size_t hi_attn_paged_work_bytes(int M, int B, int Hq, int Hkv, int D, int ragged) {
  const HiDevice* d = hi_device();
  if (!d || M < 0 || B < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || Hq / Hkv > 16 || (D != 64 && D != 128) || (int64_t)M * Hq > (1 << 27))
    return 0;
  if (!ragged) return 16;
  const int RG = flash_row_groups(M, B, Hq / Hkv);
  return 16 + (size_t)flash_slots(M, Hq / Hkv, Hkv, RG, d->cus) * Hkv * flash_slot_bytes(RG, D);
}

HI_EXPORT int hi_attn_paged(const void* q, int ldq, const void* kp, const void* vp, long long page_stride, int pages,
                            int page, const int* table, int ldt, int W, const int* start, const int* pos, void* out, int ldo,
                            float* lse, int M, int B, int Hq, int Hkv, int D, void* work, size_t work_bytes, void* stream) {
  const char* who = "hi_attn_paged";
  PagedCache c;
  if (paged_cache(who, kp, vp, page_stride, pages, page, table, ldt, W, B, Hkv, D, c)) return -1;
  if (attn_check(who, q, ldq, pos, out, ldo, lse, M, Hq, Hkv, D)) return -1;
  if (!start && M != B) HI_FAIL("%s: %d rows for %d sequences (one each without start)", who, M, B);
  if ((uintptr_t)start & 3) HI_FAIL("%s: start must be 4-byte aligned", who);
  if (M == 0 || B == 0) return 0;
  const size_t need = hi_attn_paged_work_bytes(M, B, Hq, Hkv, D, start != nullptr);
  if (!work || ((uintptr_t)work & 15) || work_bytes < need)
    HI_FAIL("%s: work of %zu bytes (at least %zu, 16-byte aligned)", who, work_bytes, need);
  const HiDevice* d = hi_device();
  if (!d) return -2;
  const AttnArgs a{(const f16*)q, ldq, (f16*)out, ldo, lse, start, pos, M, B, Hq, Hkv, 0, 1.4426950408889634f / sqrtf((float)D)};
  return attn_run(a, c, D, d->cus, work, (hipStream_t)stream, who);
}

HI_EXPORT size_t hi_attn_shared_work_bytes(int B, int Hq, int Hkv, int D) {
  (void)B, (void)Hq, (void)Hkv, (void)D;
  return 16;
}

HI_EXPORT int hi_attn_shared(const void* q, int ldq, const void* kp, const void* vp, long long page_stride, int pages,
                             int page, const int* table, int ldt, int W, int shared, const int* pos, void* out, int ldo,
                             float* lse, int B, int Hq, int Hkv, int D, void* work, size_t work_bytes, void* stream) {
  const char* who = "hi_attn_shared";
  PagedCache c;
  if (paged_cache(who, kp, vp, page_stride, pages, page, table, ldt, W, B, Hkv, D, c)) return -1;
  if (attn_check(who, q, ldq, pos, out, ldo, lse, B, Hq, Hkv, D)) return -1;
  if (shared < 0 || shared % page || shared > (int64_t)W * page)
    HI_FAIL("%s: %d shared positions (whole pages of %d, at most the table's %d)", who, shared, page, W);
  if (B == 0) return 0;
  const size_t need = hi_attn_shared_work_bytes(B, Hq, Hkv, D);
  if (!work || ((uintptr_t)work & 15) || work_bytes < need)
    HI_FAIL("%s: work of %zu bytes (at least %zu, 16-byte aligned)", who, work_bytes, need);
  const HiDevice* d = hi_device();
  if (!d) return -2;
  const AttnArgs a{(const f16*)q, ldq, (f16*)out, ldo, lse, nullptr, pos, B, B, Hq, Hkv, shared, 1.4426950408889634f / sqrtf((float)D)};
  return attn_run(a, c, D, d->cus, work, (hipStream_t)stream, who);
}
