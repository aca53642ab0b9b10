// Prefill kernels around the GEMM, behind the reference's C-ABI: the RoPE + KV-cache write that
// follows a QKV GEMM (hi_rope_cache; src/api.cu:579-586, kernels.cuh:1120-1158, ctypes
// scripts/hipinfer.py:164-168) and causal prefill attention over a cache slot (hi_flash_prefill,
// hi_flash_prefill_lse; api.cu:594-623, kernels.cuh:1160-1329, ctypes hipinfer.py:171-202).
//
// Flash prefill for gfx950 (D = 64 or 128):
//  * block = 32 RG query rows (RG 4, or 2 for small grids) of one query head and 2 RG waves: the waves of row group g (g and
//    g + RG) share its 32 rows and split every 128-key tile, keys 0..63 and 64..127, each with its
//    own online-softmax state; the pair merges (m, l, O) through LDS at the end. Two waves per
//    SIMD let one wave's softmax run beside the other's matrix work. The wave's Q rows stay in
//    registers as v_mfma_f32_32x32x16_f16 operands for the whole kernel;
//  * 128-key K/V tiles of the head's cache rows go straight from global memory into LDS by buffer
//    DMA (no register staging), two LDS stages each: K tile j + 2 and V tile j + 1 stream in while
//    tile j is computed, one barrier per tile. Both tiles keep the cache's row-major order with their
//    16-byte chunks XOR-swizzled by the key; the swizzle is applied to the DMA's per-lane source
//    address, since a DMA instruction writes 64 consecutive 16-byte LDS slots;
//  * the tiles are pipelined inside each wave: while the softmax of tile j runs on the vector units,
//    the matrix cores work on the logits of tile j + 1 and on tile j's P.V, interleaved instruction by
//    instruction. What bounds it: at T = 2048 after 4096 positions (Hq 32, Hkv 8, D 128) the MFMAs
//    alone take about half of the GPU's cycles and the clock drops to 1.8 GHz under the load; 204 ->
//    173 us (850 -> 1000 TFLOP/s) against back-to-back products, T = 1024 from 0 26.6 -> 22.1 us, 333
//    rows after 1500 36.8 -> 27.2, D = 64 T = 2048 after 2048 76.7 -> 68;
//  * S^T = K Q^T over the wave's 64 keys, in 32-key MFMA blocks: with the K fragment as first
//    operand each lane ends with 16 keys per block of ONE query row (split between lanes l and
//    l + 32), so the row max and sum of the online softmax are the lane's own values; lanes l and
//    l ^ 32 exchange them only where the reference max moves and at the end;
//  * logits are scaled by log2(e) / sqrt(D) and the softmax runs in base 2 (the reference's
//    log2-domain form, kernels.cuh:1236-1262); P is rounded to fp16 for P.V, the row sum l keeps
//    fp32 p, as the reference does. exp2 is the hardware's v_exp_f32, whose results below 2^-126
//    flush to zero: such p round to fp16 zero anyway and vanish against l >= 1 in fp32. A row's
//    reference max moves only when the row's max passes it by more than 2^8 (p <= 256), and O is
//    rescaled only then;
//  * O^T += V^T P^T: the P registers of a lane are already a B fragment of the next product once
//    the key order inside each 16-key step is permuted identically for P and V^T (lane half fk
//    takes keys 4 fk + 0..3 and 8 + 4 fk + 0..3), so P never goes through LDS. The V^T fragments
//    come from the row-major V tile through ds_read_tr16_b64, which transposes 4 keys x 16 d
//    blocks within each 16-lane group; O^T keeps the lane -> query row map, so the per-row
//    rescale by exp2(m_old - m_new) is per lane;
//  * causal mask on absolute positions (row t at p0 + t sees keys 0..p0+t): only the block's last
//    one or two tiles (and an odd one before them) carry the mask arithmetic, and a wave leaves out
//    the key halves wholly above its rows' diagonal; cache rows past the block's last key read as
//    zeros (the DMA's buffer range ends there);
//  * blocks run the longest query tiles (the most keys) first, across all heads.
#include "flash.h"

namespace {

template <int D, int RG>
__global__ void __launch_bounds__(128 * RG)
    flash_prefill_kernel(const f16* __restrict__ q, int64_t ldq, const f16* __restrict__ kc,
                         const f16* __restrict__ vc, int max_seq, f16* __restrict__ out, int64_t ldo, int T, int p0,
                         int Hq, int Hkv, float scale_log2, float* __restrict__ lse) {
  constexpr int NW = 2 * RG, BQ = 32 * RG;
  constexpr int CPR = D / 8;                   // 16-byte chunks per key row
  constexpr int IPW = kFpBKV * CPR / 64 / NW;  // DMA instructions per wave per tile and operand
  constexpr int DT = D / 32;                   // 32-row output tiles of O^T
  constexpr int NQ = D / 16;                   // MFMAs of one 32-key block's logits
  static_assert(IPW * 64 * NW == kFpBKV * CPR, "tile DMA split");
  static_assert(kFpStages == 2 && kFpKPW == 64, "the tile body is written for two stages and two key blocks");
  using Sm = FpSmem<D, RG>;
  extern __shared__ u32x4 fp_smem[];
  u32x4* const ks_ = fp_smem;                                // [2][kTile]: K stages
  u32x4* const vs_ = fp_smem + kFpStages * Sm::kTile;        // [2][kTile]: V stages
  f32x16* const mo = reinterpret_cast<f32x16*>(fp_smem);     // [RG][DT][64]: the merge
  float* const ml = reinterpret_cast<float*>(fp_smem + Sm::kMl);  // [2][RG][64]: the second waves' m and l

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wave % RG, kh = wave / RG;     // row group, key half
  const int fr = lane & 31, fk = lane >> 5;
  // grid (Hq, query tiles), dispatched x first: all heads' longest query tile first; block x runs
  // on XCD x % 8, which takes a contiguous range of query heads (those sharing a KV head)
  const int q0 = (gridDim.y - 1 - blockIdx.y) * BQ;
  const int h = Hq % 8 ? blockIdx.x : (blockIdx.x % 8) * (Hq / 8) + blockIdx.x / 8, hk = h / (Hq / Hkv);
  const int qw = q0 + rg * 32;                  // this wave's first query row
  const int qi = qw + fr;                       // this lane's query row
  const int qpos = p0 + qi;
  const int kv_end = p0 + min(q0 + BQ, T);      // keys any row of the block can see
  const int nt = (kv_end + kFpBKV - 1) / kFpBKV;  // key tiles; the first n_full hold no masked key
  const int n_full = (p0 + q0 + 1) / kFpBKV;

  // this lane's Q fragments: row qi, d = 16 ks + 8 fk + 0..7 (zero past T)
  f16x8 qf[NQ];
#pragma unroll
  for (int ks = 0; ks < NQ; ks++) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (qi < T) v = *reinterpret_cast<const u32x4*>(q + (int64_t)qi * ldq + h * D + 16 * ks + 8 * fk);
    qf[ks] = __builtin_bit_cast(f16x8, v);
  }

  // the head's cache rows 0..kv_end-1: loads past them return zeros
  const __amdgpu_buffer_rsrc_t k_rs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<f16*>(kc + (int64_t)hk * max_seq * D), (short)0, kv_end * D * 2, 0x00020000);
  const __amdgpu_buffer_rsrc_t v_rs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<f16*>(vc + (int64_t)hk * max_seq * D), (short)0, kv_end * D * 2, 0x00020000);
  // DMA instruction i of this wave fills slots (wave IPW + i) * 64 + lane of a tile: slot s holds
  // key s / CPR, physical chunk s % CPR, i.e. logical chunk (s % CPR) ^ swz(key)
  int koff[IPW], voff[IPW];
#pragma unroll
  for (int i = 0; i < IPW; i++) {
    const int s = (wave * IPW + i) * 64 + lane, r = s / CPR, p = s % CPR;
    koff[i] = (r * D + 8 * (p ^ k_swz<D>(r))) * 2;
    voff[i] = (r * D + 8 * (p ^ v_swz<D>(r))) * 2;
  }
  // issue instruction i of the next K (V) tile into stage st; koff / voff then point at the one after
  auto issue_k = [&](int i, int st) {
    lds_dma16(k_rs, ks_ + st * Sm::kTile + (wave * IPW + i) * 64, koff[i]);
    koff[i] += kFpBKV * D * 2;
    asm volatile("" : "+v"(koff[i]));  // one running offset, not a base and an induction variable
  };
  auto issue_v = [&](int i, int st) {
    lds_dma16(v_rs, vs_ + st * Sm::kTile + (wave * IPW + i) * 64, voff[i]);
    voff[i] += kFpBKV * D * 2;
    asm volatile("" : "+v"(voff[i]));
  };

  const int xaddr = (lane ^ 32) << 2;                          // lane l ^ 32, for ds_bpermute
  auto xor32 = [&](float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(xaddr, __builtin_bit_cast(int, v)));
  };

  // m_i: the row's reference max (the same in lanes l and l ^ 32); l_i: this lane's share of the
  // row's sum (its own keys; the two lanes' shares are added at the end)
  float m_i = -__builtin_huge_valf(), l_i = 0.f;
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[dt][e] = 0.f;

  auto hidden = [&](int t, int kt, int e) {
    return t * kFpBKV + kFpKPW * kh + 32 * kt + 8 * (e >> 2) + 4 * fk + (e & 3) > qpos;
  };
  auto enter_masked = [](int) {};
  constexpr bool kGuard = false;
  int odd_tile = 0;
  auto advance = [] {};
  auto before_barrier = [] {};
  auto after_barrier = [] {};
  auto live = [&](int t) {
    const int k0 = t * kFpBKV + kFpKPW * kh;
    return k0 <= p0 + qw + 31 && k0 < kv_end;
  };

#include "flash_tile.h"

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
  if (kh == 1 || qi >= T) return;
  const float m1 = ml[rg * 64 + lane], l1 = ml[(RG + rg) * 64 + lane];
  const float m = fmaxf(m_i, m1);  // finite: key 0 is visible to every row
  const float a0 = __builtin_amdgcn_exp2f(m_i - m), a1 = __builtin_amdgcn_exp2f(m1 - m);
  const float l = l_i * a0 + l1 * a1;
  if (lse && fk == 0) lse[(int64_t)h * T + qi] = m + log2f(l);
  const float inv = 1.f / l;
  f16* orow = out + (int64_t)qi * ldo + h * D;
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

// Any alignment (2-byte accesses only): block (row, head group), one wave per head of the row's
// Hq + 2 Hkv heads. A q head is rotated in place, a k head rotated into the cache, a v head copied
// into the cache; lane j takes the pairs (j, j + D/2), (j + 64, j + 64 + D/2), ... of its head.
// Each pair goes through rope_pair, as in the 16-byte kernel below, so both give the same bits.
constexpr int kRopeHeadsPerBlock = 4;

__global__ void __launch_bounds__(64 * kRopeHeadsPerBlock)
    rope_cache_heads_kernel(f16* qkv, int64_t ldq, int Hq, int Hkv, int D, const f16x2* __restrict__ cs,
                            const int* __restrict__ pos, int pos_base, int slot_base, f16* kc, f16* vc, int max_seq) {
  const int r = blockIdx.x, lane = threadIdx.x & 63;
  const int head = blockIdx.y * kRopeHeadsPerBlock + (threadIdx.x >> 6);
  if (head >= Hq + 2 * Hkv) return;
  const int at = pos ? pos[r] : pos_base + r;                  // position in the cache
  const int64_t cslot = pos ? (int64_t)slot_base + r : slot_base;
  f16* src = qkv + (int64_t)r * ldq + (int64_t)head * D;
  if (head >= Hq + Hkv) {
    f16* dst = vc + ((cslot * Hkv + (head - Hq - Hkv)) * max_seq + at) * D;
    for (int e = lane; e < D; e += 64) dst[e] = src[e];
    return;
  }
  f16* dst = head < Hq ? src : kc + ((cslot * Hkv + (head - Hq)) * max_seq + at) * D;
  const int half = D >> 1;
  const f16x2* tab = cs + (int64_t)at * half;
  for (int j = lane; j < half; j += 64) {
    f16 lo = src[j], hi = src[j + half];
    rope_pair(lo, hi, tab[j]);
    dst[j] = lo;
    dst[j + half] = hi;
  }
}

// The same with 16-byte accesses: a thread step rotates 8 pairs of one head (the 8 elements at d
// and the 8 at d + D/2, and their 8 table entries) or copies 8 elements of v. Used when D/2 is a
// multiple of 8 and every row, cache and the table are 16-byte aligned; each pair is rotated by
// rope_pair, as above, so the two kernels give the same bits.
__global__ void __launch_bounds__(256)
    rope_cache_v8_kernel(f16* qkv, int64_t ldq, int Hq, int Hkv, int D, const f16x2* __restrict__ cs,
                         const int* __restrict__ pos, int pos_base, int slot_base, f16* kc, f16* vc, int max_seq) {
  const int HD = D / 2, C = HD / 8, row = blockIdx.x;
  const int p = pos ? pos[row] : pos_base + row;
  const int slot = pos ? slot_base + row : slot_base;
  f16* base = qkv + (int64_t)row * ldq;
  const int nrot = (Hq + Hkv) * C, nv = Hkv * D / 8;
  for (int i = threadIdx.x; i < nrot + nv; i += blockDim.x) {
    if (i < nrot) {
      const int hh = i / C, d = (i - hh * C) * 8;
      f16* x = base + hh * D;
      f16x8 a = *reinterpret_cast<const f16x8*>(x + d), b = *reinterpret_cast<const f16x8*>(x + d + HD);
      const u32x4* tp = reinterpret_cast<const u32x4*>(cs + (int64_t)p * HD + d);
      const u32x4 c0 = tp[0], c1 = tp[1];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        f16 y1 = a[j], y2 = b[j];
        rope_pair(y1, y2, as_h2(j < 4 ? c0[j] : c1[j - 4]));
        a[j] = y1;
        b[j] = y2;
      }
      f16* dst = hh < Hq ? x : kc + (((int64_t)slot * Hkv + hh - Hq) * max_seq + p) * D;
      *reinterpret_cast<f16x8*>(dst + d) = a;
      *reinterpret_cast<f16x8*>(dst + d + HD) = b;
    } else {
      const int c = i - nrot, h = c / (D / 8), e = (c - h * (D / 8)) * 8;
      *reinterpret_cast<u32x4*>(vc + (((int64_t)slot * Hkv + h) * max_seq + p) * D + e) =
          *reinterpret_cast<const u32x4*>(base + (Hq + Hkv + h) * D + e);
    }
  }
}

bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int flash_prefill(const void* q, int ldq, const void* kc, const void* vc, int max_seq, void* out, int ldo, int T,
                  int p0, int Hq, int Hkv, int D, float* lse, void* stream, const char* who) {
  if (!hi_device()) return -2;
  if (D != 64 && D != 128) HI_FAIL("%s: head_dim %d not supported (64 or 128)", who, D);
  if (T < 0 || p0 < 0 || Hkv < 1 || Hq < Hkv || Hq % Hkv || max_seq < 1 || (int64_t)p0 + T > max_seq)
    HI_FAIL("%s: bad shape T=%d p0=%d Hq=%d Hkv=%d max_seq=%d", who, T, p0, Hq, Hkv, max_seq);
  if (T == 0) return 0;
  if ((int64_t)max_seq * D * 2 > INT32_MAX)  // a head's cache rows are addressed by 32-bit byte offsets
    HI_FAIL("%s: max_seq %d too long for 32-bit cache offsets (at most %d at D=%d)", who, max_seq,
            (int)(INT32_MAX / (2 * D)), D);
  if (!q || !kc || !vc || !out) HI_FAIL("%s: null tensor pointer", who);
  if (!aligned(q, 16) || ldq % 8 || ldq < Hq * D) HI_FAIL("%s: q must be 16-byte aligned, ldq %% 8 == 0, ldq >= Hq*D", who);
  if (!aligned(kc, 16) || !aligned(vc, 16)) HI_FAIL("%s: kc / vc must be 16-byte aligned", who);
  if (!aligned(out, 8) || ldo % 4 || ldo < Hq * D) HI_FAIL("%s: out must be 8-byte aligned, ldo %% 4 == 0, ldo >= Hq*D", who);
  const float scale_log2 = 1.4426950408889634f / sqrtf((float)D);
  const HiDevice* d = hi_device();
  if (!d) return -2;
  // Query rows per block: 128, or 64 while that grid is still resident at once. A CU takes a key tile
  // for 64 rows only 10-25 % faster than for 128, but the longest query tile is half as tall and a
  // small grid reaches twice the CUs: T = 512 from 0 (Hq 32, D 128) 14.4 -> 11.1 us, 64 rows after
  // 2000 28.4 -> 22.6, 777 rows of 12 heads 16.6 -> 12.7; past one round it loses (640 rows after 2048
  // 39.8 -> 48.9). At D = 64 two such blocks share a CU: that pays while most tiles are short of
  // the diagonal (777 rows from 0 12.3 -> 10.2 us), not after a long prefix (960 after 2048 34.5 -> 35.3).
  const int slots = D == 64 && p0 < T ? 2 * d->cus : d->cus;
  const bool small = (int64_t)Hq * ((T + 63) / 64) <= slots;
  const int rg = small ? 2 : kFpRG, bq = 32 * rg;
  if ((T + bq - 1) / bq > 65535) HI_FAIL("%s: T=%d exceeds %d query rows", who, T, 65535 * bq);
  const dim3 grid(Hq, (T + bq - 1) / bq);
  const hipStream_t s = (hipStream_t)stream;
  const auto kern = D == 128 ? (small ? flash_prefill_kernel<128, 2> : flash_prefill_kernel<128, kFpRG>)
                             : (small ? flash_prefill_kernel<64, 2> : flash_prefill_kernel<64, kFpRG>);
  const size_t lds = D == 128 ? (small ? FpSmem<128, 2>::kBytes : FpSmem<128, kFpRG>::kBytes)
                              : (small ? FpSmem<64, 2>::kBytes : FpSmem<64, kFpRG>::kBytes);
  const int bpc = hi_blocks_per_cu(reinterpret_cast<const void*>(kern), 64 * 2 * rg, lds);  // lifts the LDS limit
  if (bpc < 0) return -2;
  if (bpc == 0) HI_FAIL("%s: the kernel does not fit on a CU", who);
  hipLaunchKernelGGL(kern, grid, dim3(64 * 2 * rg), lds, s, (const f16*)q, (int64_t)ldq, (const f16*)kc,
                     (const f16*)vc, max_seq, (f16*)out, (int64_t)ldo, T, p0, Hq, Hkv, scale_log2, lse);
  HI_TRY(hipGetLastError());
  return 0;
}

}  // namespace

// RoPE + KV-cache write for M qkv rows [M, ldq] = [q (Hq*D) | k (Hkv*D) | v (Hkv*D)]: q rotated in
// place, rotated k and raw v to kc / vc [slots][Hkv][max_seq][D]. Row m sits at position pos[m] in
// slot slot_base + m (pos non-null: decode) or at pos_base + m in slot slot_base (prefill).
// cs: [max_seq][D/2] (cos, sin) fp16 pairs. Positions must lie in [0, max_seq).
HI_EXPORT int hi_rope_cache(void* qkv, int ldq, int M, int Hq, int Hkv, int D, const void* cs, const int* pos,
                            int pos_base, int slot_base, void* kc, void* vc, int max_seq, void* stream) {
  if (!hi_device()) return -2;
  if (M < 0 || Hq < 1 || Hkv < 1 || D < 2 || D % 2 || max_seq < 1 || slot_base < 0)
    HI_FAIL("hi_rope_cache: bad shape M=%d Hq=%d Hkv=%d D=%d max_seq=%d", M, Hq, Hkv, D, max_seq);
  if (M == 0) return 0;
  if (!qkv || !cs || !kc || !vc) HI_FAIL("hi_rope_cache: null tensor pointer");
  if (ldq < (Hq + 2 * Hkv) * D) HI_FAIL("hi_rope_cache: ldq %d < (Hq + 2 Hkv) D", ldq);
  if ((Hq + 2 * Hkv + kRopeHeadsPerBlock - 1) / kRopeHeadsPerBlock > 65535)
    HI_FAIL("hi_rope_cache: %d heads per row exceed the launch grid", Hq + 2 * Hkv);
  if (!pos && (pos_base < 0 || (int64_t)pos_base + M > max_seq))
    HI_FAIL("hi_rope_cache: positions %d..%d outside the cache (max_seq %d)", pos_base, pos_base + M - 1, max_seq);
  if (!aligned(cs, 4)) HI_FAIL("hi_rope_cache: cs must be 4-byte aligned");
  const bool v8 = D % 16 == 0 && ldq % 8 == 0 && aligned(qkv, 16) && aligned(cs, 16) && aligned(kc, 16) && aligned(vc, 16);
  if (v8)
    hipLaunchKernelGGL(rope_cache_v8_kernel, dim3(M), dim3(256), 0, (hipStream_t)stream, (f16*)qkv, (int64_t)ldq, Hq, Hkv,
                       D, (const f16x2*)cs, pos, pos_base, slot_base, (f16*)kc, (f16*)vc, max_seq);
  else
    hipLaunchKernelGGL(rope_cache_heads_kernel, dim3(M, (Hq + 2 * Hkv + kRopeHeadsPerBlock - 1) / kRopeHeadsPerBlock),
                       dim3(64 * kRopeHeadsPerBlock), 0, (hipStream_t)stream, (f16*)qkv, (int64_t)ldq, Hq, Hkv, D,
                       (const f16x2*)cs, pos, pos_base, slot_base, (f16*)kc, (f16*)vc, max_seq);
  HI_TRY(hipGetLastError());
  return 0;
}

// Causal prefill attention of T query rows (row t at position p0 + t; head h at columns h*D of
// q [T, ldq]) over one cache slot kc / vc [Hkv][max_seq][D], keys 0..p0+t; out [T, ldo].
HI_EXPORT int hi_flash_prefill(const void* q, int ldq, const void* kc, const void* vc, int max_seq, void* out, int ldo,
                               int T, int p0, int Hq, int Hkv, int D, void* stream) {
  return flash_prefill(q, ldq, kc, vc, max_seq, out, ldo, T, p0, Hq, Hkv, D, nullptr, stream, "hi_flash_prefill");
}

// The same, and each row's log2-domain log-sum-exp of the scaled logits into lse [Hq][T] fp32.
HI_EXPORT int hi_flash_prefill_lse(const void* q, int ldq, const void* kc, const void* vc, int max_seq, void* out,
                                   int ldo, int T, int p0, int Hq, int Hkv, int D, float* lse, void* stream) {
  if (!lse) HI_FAIL("hi_flash_prefill_lse: lse must not be null");
  return flash_prefill(q, ldq, kc, vc, max_seq, out, ldo, T, p0, Hq, Hkv, D, lse, stream, "hi_flash_prefill_lse");
}
