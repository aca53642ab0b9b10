// Serving from a paged key/value cache in 8 bits: rotation, rounding to 8 bits and cache write of projected rows
// (hi_rope_cache_paged8), and attention over the pages (hi_attn_paged8; the kernels are paged_attn.h's).
//
// An element's value is its e4m3 code times 2^k with one k per page and kv head, of K and of V apart. e4m3 has 4 significant bits at
// any magnitude, so an exponent as good as any other scale costs a byte a page, and a power of two makes both directions exact but
// for the one rounding to 4 bits. Where a page's k grows with later positions, codes move down by whole binary orders: exactly, but
// those that come below 2^-6 * 2^k (2^-13 of the page's largest value at most) become subnormal codes and are rounded again, to steps
// of 2^-9 * 2^k, at every growth, so that such small values depend on which rows came in one call. A stored value is off by less
// than 2^-4 of it + 2^-9 * 2^k in all: half steps of exponents that grow add up to less than twice the last one's.
//
// The attention kernels' fp16 operands are the stored values; those below 2^-21 are rounded to fp16's least steps, 2^-24.
#include "paged_attn.h"

namespace {

constexpr float kMost = 61440.f;             // 240 * 2^8: the largest value that is fp16 after rounding to 4 bits
constexpr int kExpMin = -32, kExpMax = 8;    // of the least (2^-24) and the largest page maximum

// The least k with most <= 448 * 2^k: 448 = 1.75 * 2^8.
__device__ __forceinline__ int exponent_of(float most) {
  const int b = __builtin_bit_cast(int, most);
  const int k = (b >> 23) - 127 - 8 + ((b & 0x7fffff) > 0x600000);
  return min(max(k, kExpMin), kExpMax);  // (0: -135)
}

// 4 values at 2^-k as codes; NaN stays NaN.
__device__ __forceinline__ uint32_t f8x4(float a, float b, float c, float d) {
  int w = 0;
#if defined(__HIP_DEVICE_COMPILE__)
  w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
#endif
  return (uint32_t)w;
}

// 4 codes times a power of two.
__device__ __forceinline__ uint32_t f8x4_scaled(uint32_t w, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  w = f8x4(lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale);
#endif
  return w;
}

struct Rope8Args {
  f16* qkv;
  int64_t ldq;
  f16* qo;
  int64_t ldqo;
  int M, B, Hq, Hkv, D, rot, cs_rows;
  const void* cs;
  const int *start, *pos;
  int8_t *kexp, *vexp;
  int units, inter;
};

// The positions [lo, hi) of sequence b's rows that have a place in a table, as numbers of rows, and its first row.
struct Run {
  int row0, n, pos, lo, hi;
};
__device__ __forceinline__ Run run_of(const Rope8Args& a, int cap, int b) {
  Run r{b, 1, 0, 0, 0};
  if (b >= a.B) {
    r.n = 0;
    return r;
  }
  r.pos = a.pos[b];
  if (a.start) {
    const int s0 = a.start[b], s1 = a.start[b + 1];
    r.row0 = plan_first(s0, a.M);
    r.n = plan_rows(s0, s1, a.M);
  } else if (b >= a.M) {
    r.n = 0;
  }
  r.lo = max(r.pos, 0);
  r.hi = plan_end(r.pos, r.n, cap);
  return r;
}

// n entries of a cs row, 16 bytes at a time.
template <typename CS, int n>
__device__ __forceinline__ void load_cs(const CS* tab, CS (&t)[n]) {
#pragma unroll
  for (int k = 0; k < (int)(n * sizeof(CS) / 16); k++) {
    const u32x4 w = reinterpret_cast<const u32x4*>(tab)[k];
    __builtin_memcpy((char*)t + 16 * k, &w, 16);
  }
}

// A K or V head's 8 elements from d on of a row, rotated for K: products of fp16 numbers are exact in fp32.
template <typename CS, bool WIDE>
__device__ __forceinline__ void head8(const Rope8Args& a, const f16* head, const CS* tab, int rot, int d, float (&y)[8]) {
  const int half = rot / 2;
  if constexpr (WIDE) {  // 16-byte accesses: 8 elements are all rotated or none, in one half
    const f16x8 x = *reinterpret_cast<const f16x8*>(head + d);
    if (d >= rot) {
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = (float)x[e];
    } else if (a.inter) {
      CS t[8];
      load_cs<CS, 8>(tab + d, t);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float u = (float)x[e], v = (float)x[e + 1], c = (float)t[e], s = (float)t[e + 1];
        y[e] = __builtin_fmaf(u, c, -(v * s));
        y[e + 1] = __builtin_fmaf(v, c, u * s);
      }
    } else {
      const bool low = d < half;
      const int j = low ? d : d - half;
      const f16x8 z = *reinterpret_cast<const f16x8*>(head + (low ? d + half : j));
      CS t[16];
      load_cs<CS, 16>(tab + 2 * j, t);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float own = (float)x[e], other = (float)z[e], c = (float)t[2 * e], s = (float)t[2 * e + 1];
        y[e] = low ? __builtin_fmaf(own, c, -(other * s)) : __builtin_fmaf(own, c, other * s);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int i = d + e;
      if (i >= rot) {
        y[e] = (float)head[i];
        continue;
      }
      const bool low = a.inter ? !(i & 1) : i < half;
      const int j = a.inter ? i >> 1 : low ? i : i - half, o = a.inter ? i ^ 1 : low ? i + half : j;
      const float own = (float)head[i], other = (float)head[o], c = (float)tab[2 * j], s = (float)tab[2 * j + 1];
      y[e] = low ? __builtin_fmaf(own, c, -(other * s)) : __builtin_fmaf(own, c, other * s);
    }
  }
}

// The q heads of row m, in pair steps that read all of what they write (in place too).
template <typename CS, bool WIDE>
__device__ __forceinline__ void rotate_q(const Rope8Args& a, const PagedCache8& c, int m) {
  const int lane = threadIdx.x & 63, cap = min(c.capacity(), a.cs_rows), half = a.rot / 2, D = a.D;
  const f16* const row = a.qkv + (int64_t)m * a.ldq;
  f16* const out = a.qo + (int64_t)m * a.ldqo;
  // steps of 8 pairs (or 4 interleaved ones: the same 8 elements), then of 8 elements that stay; the first two are requested before
  // the row's place is known
  const int turns = a.rot / (a.inter ? 8 : 16), per = turns + (D - a.rot) / 8, steps = WIDE ? a.Hq * per : 0;
  struct Step {
    f16x8 x, z;
  } ahead[2] = {};
  auto load = [&](int i, Step& s) {
    const int h = i / per, j = i - h * per, d = j < turns ? 8 * j : a.rot + 8 * (j - turns);
    s.x = *reinterpret_cast<const f16x8*>(row + h * D + d);
    if (!a.inter && j < turns) s.z = *reinterpret_cast<const f16x8*>(row + h * D + d + half);
  };
#pragma unroll
  for (int k = 0; k < 2; k++)
    if ((int)threadIdx.x + 256 * k < steps) load(threadIdx.x + 256 * k, ahead[k]);
  int b = -1, p = -1;
  if (a.start) {
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const Run r = run_of(a, cap, b0 + lane);
      const uint64_t hit = __ballot(m >= r.row0 && m < r.row0 + r.n);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        b = b0 + l;
        const int64_t at = (int64_t)__builtin_amdgcn_readlane(r.pos, l) + (m - __builtin_amdgcn_readlane(r.row0, l));
        p = at < 0 || at >= cap ? -1 : (int)at;
        break;
      }
    }
  } else {
    b = m;
    p = a.pos[m];
    if ((unsigned)p >= (unsigned)cap) p = -1;
  }
  if (p < 0 || !c.has(c.entry(b, p >> c.shift))) return;
  const CS* tab = (const CS*)a.cs + (int64_t)p * a.rot;
  if constexpr (WIDE) {
    auto finish = [&](int i, Step& s) {
      const int h = i / per, j = i - h * per, d = j < turns ? 8 * j : a.rot + 8 * (j - turns);
      f16* const dst = out + h * D + d;
      if (j < turns) {
        if (a.inter) {
          CS t[8];
          load_cs<CS, 8>(tab + d, t);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float u = (float)s.x[e], v = (float)s.x[e + 1], cc = (float)t[e], sn = (float)t[e + 1];
            s.x[e] = (f16)__builtin_fmaf(u, cc, -(v * sn));
            s.x[e + 1] = (f16)__builtin_fmaf(v, cc, u * sn);
          }
        } else {
          CS t[16];
          load_cs<CS, 16>(tab + 2 * d, t);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float u = (float)s.x[e], v = (float)s.z[e], cc = (float)t[2 * e], sn = (float)t[2 * e + 1];
            s.x[e] = (f16)__builtin_fmaf(u, cc, -(v * sn));
            s.z[e] = (f16)__builtin_fmaf(v, cc, u * sn);
          }
          *reinterpret_cast<f16x8*>(dst + half) = s.z;
        }
      }
      *reinterpret_cast<f16x8*>(dst) = s.x;
    };
#pragma unroll
    for (int k = 0; k < 2; k++)
      if ((int)threadIdx.x + 256 * k < steps) finish(threadIdx.x + 256 * k, ahead[k]);
    for (int i = threadIdx.x + 512; i < steps; i += 256) {
      Step s;
      load(i, s);
      finish(i, s);
    }
  } else {
    for (int i = threadIdx.x; i < a.Hq * (D - half); i += 256) {  // a pair or an element each
      const int h = i / (D - half), j = i - h * (D - half);
      const f16* src = row + (int64_t)h * D;
      f16* dst = out + (int64_t)h * D;
      if (j >= half) {
        dst[j + half] = src[j + half];
        continue;
      }
      const int i0 = a.inter ? 2 * j : j, i1 = a.inter ? 2 * j + 1 : j + half;
      const float u = (float)src[i0], v = (float)src[i1], cc = (float)tab[2 * j], s = (float)tab[2 * j + 1];
      dst[i0] = (f16)__builtin_fmaf(u, cc, -(v * s));
      dst[i1] = (f16)__builtin_fmaf(v, cc, u * s);
    }
  }
}

// Blocks 0 .. units * groups - 1: the new rows of one page of one sequence, for T threads per (kv head, K or V); then a block per
// row for q. Two passes over the rows: the largest value, then the codes; the first 4 rounds of rows stay in registers. T follows
// the page, so that 4 rounds are a page up to 64 positions (128 at D = 64); longer ones are read again for the codes.
// What bounds it: 2048 rows of 32/8 heads of 128 on pages of 64 take 11.5 us, 4.1 TB/s, memory and a launch's ends (q's blocks
// first 13.2: the pages' are the longer chains); 48 rows 3.4, the chain position -> page -> exponent -> stores.
constexpr int kHeld = 4;
template <typename CS, bool WIDE, int T>
__global__ void __launch_bounds__(256) rope_paged8_kernel(Rope8Args a, PagedCache8 c, int groups) {
  __shared__ float red[4];
  constexpr int PER = 256 / T;  // (kv head, K or V) pairs of a block
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = a.D, page = 1 << c.shift;
  if ((int)blockIdx.x >= a.units * groups) {
    rotate_q<CS, WIDE>(a, c, blockIdx.x - a.units * groups);
    return;
  }
  const int unit = blockIdx.x / groups, item = (blockIdx.x - unit * groups) * PER + tid / T, t = tid % T;
  // ---- the unit's sequence and page
  const int cap = min(c.capacity(), a.cs_rows);
  int b = -1, pg = 0;
  Run r{};
  if (!a.start) {
    r = run_of(a, cap, unit);
    if (r.hi <= r.lo) return;
    b = unit;
    pg = r.lo >> c.shift;
  } else {
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const Run x = run_of(a, cap, b0 + lane);
      const int n = x.hi > x.lo ? ((x.hi - 1) >> c.shift) - (x.lo >> c.shift) + 1 : 0;
      const int upto = wave_scan(n, lane);
      const uint64_t hit = __ballot(before + upto > unit);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
        b = b0 + l;
        r = Run{get(x.row0), get(x.n), get(x.pos), get(x.lo), get(x.hi)};
        pg = (r.lo >> c.shift) + unit - before - (get(upto) - get(n));
        break;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (b < 0) return;
  }
  const int id = c.entry(b, pg);
  if (!c.has(id)) return;
  const int first = max(r.lo, pg << c.shift), last = min(r.hi, (pg + 1) << c.shift);  // the page's new positions
  const int o0 = first & (page - 1), n = last - first, row0 = r.row0 + (first - r.pos);
  const bool active = item < 2 * a.Hkv;  // (all threads of a block meet at the barriers)
  const bool V = item >= a.Hkv;
  const int h = active ? V ? item - a.Hkv : item : 0, rot = V ? 0 : a.rot;
  const f16* const src = a.qkv + (int64_t)row0 * a.ldq + (int64_t)(a.Hq + (V ? a.Hkv : 0) + h) * D;
  uint8_t* const codes = const_cast<uint8_t*>(V ? c.vp : c.kp) + (int64_t)id * c.stride + (int64_t)h * page * D;
  int8_t* const exps = (V ? a.vexp : a.kexp) + (int64_t)id * a.Hkv + h;
  const int lanes = D / 8, tr = t / lanes, d = 8 * (t - tr * lanes), RPP = T / lanes;  // rows of a round
  const int old = active && o0 > 0 ? *exps : kExpMin;
  float most = 0.f;
  auto value = [&](int i, float (&y)[8]) {
    head8<CS, WIDE>(a, src + (int64_t)i * a.ldq, (const CS*)a.cs + (int64_t)(first + i) * a.rot, rot, d, y);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (__builtin_fabsf(y[e]) > kMost) y[e] = __builtin_copysignf(kMost, y[e]);
      most = fmaxf(most, __builtin_fabsf(y[e]));  // (a NaN is passed over)
    }
  };
  float y[kHeld][8];
#pragma unroll
  for (int k = 0; k < kHeld; k++)
    if (active && tr + k * RPP < n) value(tr + k * RPP, y[k]);
  for (int i = tr + kHeld * RPP; active && i < n; i += RPP) {
    float z[8];
    value(i, z);
  }
  most = wave_max(most);
  if constexpr (T > 64) {
    if (lane == 0) red[wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; w++) most = fmaxf(most, red[(wave & ~(T / 64 - 1)) + w]);
  }
  if (!active) return;
  const int now = max(exponent_of(most), o0 > 0 ? min(max(old, kExpMin), kExpMax) : kExpMin);
  const float scale = exponent_scale(-now);
  auto put = [&](int i, const float (&v)[8]) {
    const u32x2 w = {f8x4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale),
                     f8x4(v[4] * scale, v[5] * scale, v[6] * scale, v[7] * scale)};
    *reinterpret_cast<u32x2*>(codes + (int64_t)(o0 + i) * D + d) = w;
  };
#pragma unroll
  for (int k = 0; k < kHeld; k++)
    if (tr + k * RPP < n) put(tr + k * RPP, y[k]);
  for (int i = tr + kHeld * RPP; i < n; i += RPP) {
    float z[8];
    value(i, z);
    put(i, z);
  }
  if (t == 0) *exps = (int8_t)now;
  if (o0 > 0 && now != old) {  // earlier positions move to the page's new exponent
    const float change = exponent_scale(old - now);
    for (int i = tr; i < o0; i += RPP) {
      u32x2* const p = reinterpret_cast<u32x2*>(codes + (int64_t)i * D + d);
      const u32x2 w = *p;
      u32x2 v = {};
#pragma unroll
      for (int k = 0; k < 2; k++) v[k] = f8x4_scaled(w[k], change);
      *p = v;
    }
  }
}

int cache8(const char* who, const void* kexp, const void* vexp, PagedCache8& c) {
  if (!kexp || !vexp) HI_FAIL("%s: kexp and vexp must not be null", who);
  c.kexp = (const int8_t*)kexp;
  c.vexp = (const int8_t*)vexp;
  return 0;
}

}  // namespace

HI_EXPORT int hi_rope_cache_paged8(void* qkv, int ldq, void* q_out, int ldqo, int M, int Hq, int Hkv, int D, const void* cs, int cs_rows,
                                   int cs_f32, int rot, int interleaved, const int* start, const int* pos, void* kp, void* vp,
                                   void* kexp, void* vexp, long long page_stride, int pages, int page, const int* table, int ldt,
                                   int W, int B, void* stream) {
  const char* who = "hi_rope_cache_paged8";
  PagedCache8 c;
  if (paged_cache(who, kp, vp, page_stride, pages, page, table, ldt, W, B, Hkv, D, c) || cache8(who, kexp, vexp, c)) return -1;
  if (M < 0 || Hq < 1 || Hq > 4096 || rot < 0 || rot % 2 || rot > D || cs_rows < 1 || (!start && M != B))
    HI_FAIL("%s: M %d, Hq %d, rot %d (even, at most D), cs rows %d, B %d (M without start)", who, M, Hq, rot, cs_rows, B);
  if (M == 0 || B == 0) return 0;
  if (!qkv || !q_out || (rot && !cs) || !pos || ldq < (Hq + 2 * Hkv) * D || ldqo < Hq * D || ((uintptr_t)qkv & 1) ||
      ((uintptr_t)q_out & 1) || ((uintptr_t)cs & (cs_f32 ? 7 : 3)) || ((uintptr_t)pos & 3) || ((uintptr_t)start & 3))
    HI_FAIL("%s: a null or misaligned pointer, ldq < (Hq + 2 Hkv) D or q_out's row stride < Hq D", who);
  if (!in_place_or_apart(qkv, 2 * (int64_t)ldq, 2 * (int64_t)(Hq + 2 * Hkv) * D, q_out, 2 * (int64_t)ldqo, 2 * (int64_t)Hq * D, M))
    HI_FAIL("%s: q_out must be qkv (with its row stride) or apart from it", who);
  // pages that rows lie on: of a sequence's n rows at most (n - 2) / page + 2, or 1
  const int64_t units = start ? std::min((int64_t)M, (int64_t)M / page + 2 * (int64_t)std::min(B, M)) : M;
  const int T = page <= 16 ? 64 : page <= 32 ? 128 : 256, groups = (2 * Hkv * T + 255) / 256;
  if (units * groups + M > INT32_MAX) HI_FAIL("%s: %d rows of %d heads are too many", who, M, Hkv);
  if (!hi_device()) return -2;
  const Rope8Args a{(f16*)qkv, ldq, (f16*)q_out, ldqo, M, B, Hq, Hkv, D, rot, cs_rows, cs, start, pos, (int8_t*)kexp, (int8_t*)vexp,
                    (int)units, interleaved != 0};
  const hipStream_t s = (hipStream_t)stream;
  const bool wide = rot % (interleaved ? 8 : 16) == 0 && ldq % 8 == 0 && ldqo % 8 == 0 &&
                    (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)cs) & 15) == 0;
  const dim3 grid((unsigned)(units * groups + M));
  auto launch = [&](auto t) {
    constexpr int kT = decltype(t)::value;
    const auto kern = cs_f32 ? (wide ? rope_paged8_kernel<float, true, kT> : rope_paged8_kernel<float, false, kT>)
                             : (wide ? rope_paged8_kernel<f16, true, kT> : rope_paged8_kernel<f16, false, kT>);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a, c, groups);
  };
  if (T == 64) launch(std::integral_constant<int, 64>{});
  else if (T == 128) launch(std::integral_constant<int, 128>{});
  else launch(std::integral_constant<int, 256>{});
  HI_TRY(hipGetLastError());
  return 0;
}

HI_EXPORT int hi_attn_paged8(const void* q, int ldq, const void* kp, const void* vp, const void* kexp, const void* vexp,
                             long long page_stride, int pages, int page, const int* table, int ldt, int W, const int* start,
                             const int* pos, void* out, int ldo, float* lse, int M, int B, int Hq, int Hkv, int D, void* work,
                             size_t work_bytes, void* stream) {
  const char* who = "hi_attn_paged8";
  PagedCache8 c;
  if (paged_cache(who, kp, vp, page_stride, pages, page, table, ldt, W, B, Hkv, D, c) || cache8(who, kexp, vexp, c)) return -1;
  return attn_paged_call(who, c, q, ldq, start, pos, out, ldo, lse, M, B, Hq, Hkv, D, work, work_bytes, (hipStream_t)stream);
}
