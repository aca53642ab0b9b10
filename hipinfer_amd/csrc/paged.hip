// Serving from a paged key/value cache: rotation and cache write of projected rows (hi_rope_cache_paged), attention over
// the pages (hi_attn_paged) and attention of a batch whose sequences share their first positions (hi_attn_shared).
// The cache and its table: paged.h.
#include "paged.h"

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

int attn_run(const AttnArgs& a, const PagedCache& c, int D, hipStream_t s) {
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
  (void)M, (void)B, (void)Hq, (void)Hkv, (void)D, (void)ragged;
  return 16;
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
  if (!hi_device()) return -2;
  const AttnArgs a{(const f16*)q, ldq, (f16*)out, ldo, lse, start, pos, M, B, Hq, Hkv, 0, 1.4426950408889634f / sqrtf((float)D)};
  return attn_run(a, c, D, (hipStream_t)stream);
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
  if (!hi_device()) return -2;
  const AttnArgs a{(const f16*)q, ldq, (f16*)out, ldo, lse, nullptr, pos, B, B, Hq, Hkv, shared, 1.4426950408889634f / sqrtf((float)D)};
  return attn_run(a, c, D, (hipStream_t)stream);
}
