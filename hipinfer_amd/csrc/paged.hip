// Serving from a paged key/value cache: rotation and cache write of projected rows (hi_rope_cache_paged), attention over
// the pages (hi_attn_paged) and attention of a batch whose sequences share their first positions (hi_attn_shared).
// The cache and its table: paged.h.
#include "paged_attn.h"

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

// 16-byte accesses: a step turns 8 pairs (the 8 elements at d and the 8 at d + rot / 2, or 8 interleaved ones: 4 pairs) or
// copies 8 elements; block per row, a thread per step up to 512. `per` steps a q or k head, `turns` of them rotate. The row is
// requested before its place is known (position, table entry and cs row are a chain of three loads). 2048 rows of 32/8 heads
// of 128 10.2 us, 5.0 TB/s, what a large copy reaches (the kernel above 15.5); one row 2.3 us, the chain (5.2).
template <typename CS, bool INTER>
__global__ void __launch_bounds__(512) rope_paged_kernel(RopePagedArgs a, PagedCache c, int per, int turns) {
  constexpr int NP = INTER ? 4 : 8;  // pairs of a step
  const int m = blockIdx.x, nrot = (a.Hq + a.Hkv) * per, n = nrot + a.Hkv * a.D / 8, half = a.rot / 2;
  const f16* row = a.qkv + (int64_t)m * a.ldq;
  int i = threadIdx.x, h, d;
  bool turning;
  f16x8 x, y;
  auto load = [&] {
    turning = false;
    if (i < nrot) {
      h = i / per;
      const int j = i - h * per;
      turning = j < turns;
      d = turning ? 8 * j : a.rot + 8 * (j - turns);
    } else {
      const int j = i - nrot, w = a.D / 8;
      h = j / w;
      d = 8 * (j - h * w);
      h += a.Hq + a.Hkv;
    }
    const f16* src = row + h * a.D + d;
    x = *reinterpret_cast<const f16x8*>(src);
    if (!INTER && turning) y = *reinterpret_cast<const f16x8*>(src + half);
  };
  if (i < n) load();
  int p;
  const int64_t at = rope_place(a, c, m, p);
  if (at < 0) return;
  const int page = 1 << c.shift;
  while (i < n) {
    f16* dst = h < a.Hq ? a.qo + (int64_t)m * a.ldqo + h * a.D
               : h < a.Hq + a.Hkv ? const_cast<f16*>(c.kp) + at + (int64_t)(h - a.Hq) * page * a.D
                                  : const_cast<f16*>(c.vp) + at + (int64_t)(h - a.Hq - a.Hkv) * page * a.D;
    if (turning) {
      const CS* tab = (const CS*)a.cs + (int64_t)p * a.rot + (INTER ? d : 2 * d);
      CS t[2 * NP];
#pragma unroll
      for (int k = 0; k < (int)(2 * NP * sizeof(CS) / 16); k++)
        reinterpret_cast<u32x4*>(t)[k] = reinterpret_cast<const u32x4*>(tab)[k];
#pragma unroll
      for (int k = 0; k < NP; k++) {
        f16 u = INTER ? x[2 * k] : x[k], v = INTER ? x[2 * k + 1] : y[k];
        turn(u, v, (float)t[2 * k], (float)t[2 * k + 1]);
        if constexpr (INTER) {
          x[2 * k] = u;
          x[2 * k + 1] = v;
        } else {
          x[k] = u;
          y[k] = v;
        }
      }
      if constexpr (!INTER) *reinterpret_cast<f16x8*>(dst + d + half) = y;
    }
    *reinterpret_cast<f16x8*>(dst + d) = x;
    i += blockDim.x;
    if (i < n) load();
  }
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
  if (!in_place_or_apart(qkv, 2 * (int64_t)ldq, 2 * (int64_t)(Hq + 2 * Hkv) * D, q_out, 2 * (int64_t)ldqo, 2 * (int64_t)Hq * D, M))
    HI_FAIL("%s: q_out must be qkv (with its row stride) or apart from it", who);
  if (!hi_device()) return -2;
  const RopePagedArgs a{(f16*)qkv, ldq, (f16*)q_out, ldqo, Hq, Hkv, D, rot, cs_rows, B, cs, seq, pos};
  const hipStream_t s = (hipStream_t)stream;
  const bool v8 = rot % (interleaved ? 8 : 16) == 0 && ldq % 8 == 0 && ldqo % 8 == 0 &&
                  (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)cs) & 15) == 0;
  if (v8) {
    const int turns = rot / (interleaved ? 8 : 16), per = turns + (D - rot) / 8;
    const int steps = (Hq + Hkv) * per + Hkv * D / 8;
    const dim3 block(min(512, (steps + 63) & ~63));
    const auto kern = cs_f32 ? (interleaved ? rope_paged_kernel<float, true> : rope_paged_kernel<float, false>)
                             : (interleaved ? rope_paged_kernel<f16, true> : rope_paged_kernel<f16, false>);
    hipLaunchKernelGGL(kern, dim3(M), block, 0, s, a, c, per, turns);
  } else {
    const auto kern = cs_f32 ? rope_paged_any_kernel<float> : rope_paged_any_kernel<f16>;
    hipLaunchKernelGGL(kern, dim3(M), dim3(256), 0, s, a, c, interleaved != 0);
  }
  HI_TRY(hipGetLastError());
  return 0;
}

HI_EXPORT size_t hi_attn_paged_work_bytes(int M, int B, int Hq, int Hkv, int D, int ragged) {
  const HiDevice* d = hi_device();
  if (!d || !work_sizes(M, B, Hq, Hkv, D)) return 0;
  return kWorkHead + (M == 0 || B == 0 ? 0 : paged_bytes(M, B, Hq, Hkv, D, ragged != 0, d->cus));
}

HI_EXPORT size_t hi_attn_paged_work_bytes_max(int M, int B, int Hq, int Hkv, int D, int ragged) {
  const HiDevice* d = hi_device();
  if (!d || !work_sizes(M, B, Hq, Hkv, D)) return 0;
  return kWorkHead + (M == 0 || B == 0 ? 0 : paged_most_bytes(M, B, Hq, Hkv, D, ragged != 0, d->cus));
}

HI_EXPORT int hi_attn_paged(const void* q, int ldq, const void* kp, const void* vp, long long page_stride, int pages,
                            int page, const int* table, int ldt, int W, const int* start, const int* pos, void* out, int ldo,
                            float* lse, int M, int B, int Hq, int Hkv, int D, void* work, size_t work_bytes, void* stream) {
  const char* who = "hi_attn_paged";
  PagedCache c;
  if (paged_cache(who, kp, vp, page_stride, pages, page, table, ldt, W, B, Hkv, D, c)) return -1;
  return attn_paged_call(who, c, q, ldq, start, pos, out, ldo, lse, M, B, Hq, Hkv, D, work, work_bytes, (hipStream_t)stream);
}

HI_EXPORT size_t hi_attn_shared_work_bytes(int B, int Hq, int Hkv, int D) {
  const HiDevice* d = hi_device();
  if (!d || !work_sizes(B, B, Hq, Hkv, D)) return 0;
  return kWorkHead + (B == 0 ? 0 : shared_bytes(B, Hq, Hkv, D, d->cus));
}

HI_EXPORT size_t hi_attn_shared_work_bytes_max(int B, int Hq, int Hkv, int D) {
  const HiDevice* d = hi_device();
  if (!d || !work_sizes(B, B, Hq, Hkv, D)) return 0;
  return kWorkHead + (B == 0 ? 0 : shared_most_bytes(B, Hq, Hkv, D, d->cus));
}

HI_EXPORT int hi_attn_shared(const void* q, int ldq, const void* kp, const void* vp, long long page_stride, int pages,
                             int page, const int* table, int ldt, int W, int shared, const int* pos, void* out, int ldo,
                             float* lse, int B, int Hq, int Hkv, int D, void* work, size_t work_bytes, void* stream) {
  const char* who = "hi_attn_shared";
  PagedCache c;
  if (paged_cache(who, kp, vp, page_stride, pages, page, table, ldt, W, B, Hkv, D, c)) return -1;
  if (B == 0) return 0;
  if (attn_check(who, q, ldq, pos, out, ldo, lse, B, Hq, Hkv, D)) return -1;
  if (shared < 0 || shared % page || shared > (int64_t)W * page)
    HI_FAIL("%s: %d shared positions (whole pages of %d, at most the table's %d)", who, shared, page, W);
  const size_t need = hi_attn_shared_work_bytes(B, Hq, Hkv, D);
  if (!work || ((uintptr_t)work & 15) || work_bytes < need)
    HI_FAIL("%s: work of %zu bytes (at least %zu, 16-byte aligned)", who, work_bytes, need);
  const HiDevice* d = hi_device();
  if (!d) return -2;
  const AttnArgs a{(const f16*)q, ldq, (f16*)out, ldo, lse, nullptr, pos, B, B, Hq, Hkv, shared, Hq / Hkv, plan_magic(Hq / Hkv),
                   1.4426950408889634f / sqrtf((float)D)};
  return attn_run(a, c, D, d->cus, work, (hipStream_t)stream, who);
}
