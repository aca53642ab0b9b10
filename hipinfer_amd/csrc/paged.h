// The paged key/value cache as the kernels see it, and what its host entry points check alike.
#pragma once
#include "hi_common.h"

// kp / vp [pages][Hkv][page][D] fp16, pages `stride` halves apart (the same for both); position p of sequence b is
// row p % page of page table[b][p / page]. A page id outside [0, pages) is no page.
struct PagedCache {
  typedef f16 Elem;
  static constexpr bool kF8 = false;
  const f16 *kp, *vp;
  int64_t stride;
  int pages, shift;  // page = 1 << shift
  const int* table;
  int ldt, W;        // table row stride, entries per row

  __device__ __forceinline__ int capacity() const { return W << shift; }
  __device__ __forceinline__ bool has(int id) const { return (unsigned)id < (unsigned)pages; }
  // entry i of sequence b's table row; -1 behind its end
  __device__ __forceinline__ int entry(int b, int i) const { return (unsigned)i < (unsigned)W ? table[(int64_t)b * ldt + i] : -1; }
};

// The same in 8 bits: kp / vp [pages][Hkv][page][D] e4m3 codes, pages `stride` bytes apart, an element's value its code times 2 to the
// power of its page's and head's exponent, kexp / vexp [pages][Hkv], as fp16.
struct PagedCache8 {
  typedef uint8_t Elem;
  static constexpr bool kF8 = true;
  const uint8_t *kp, *vp;
  int64_t stride;
  int pages, shift;
  const int* table;
  int ldt, W;
  const int8_t *kexp, *vexp;

  __device__ __forceinline__ int capacity() const { return W << shift; }
  __device__ __forceinline__ bool has(int id) const { return (unsigned)id < (unsigned)pages; }
  __device__ __forceinline__ int entry(int b, int i) const { return (unsigned)i < (unsigned)W ? table[(int64_t)b * ldt + i] : -1; }
};

// 2^e as a float for a stored exponent (-128 and -127, which no float has: 2^-126).
__device__ __forceinline__ float exponent_scale(int e) { return __builtin_bit_cast(float, (max(e, -126) + 127) << 23); }
// 2 of 4 codes as fp16 values, the lower or the upper two.
__device__ __forceinline__ uint32_t f8x2_to_f16(uint32_t w, int upper, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
  return upper ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true))
               : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
#else
  return 0;
#endif
}
// 4 codes as fp16 values: the product of code and scale rounded once (exact unless it is subnormal or overflows).
__device__ __forceinline__ void f8x4_to_f16(uint32_t w, float scale, f16x2& lo, f16x2& hi) {
#if defined(__HIP_DEVICE_COMPILE__)
  lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
  hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true));
#endif
}
__device__ __forceinline__ f16x8 f8x8_to_f16(uint32_t a, uint32_t b, float scale) {
  f16x2 x[4] = {};
  f8x4_to_f16(a, scale, x[0], x[1]);
  f8x4_to_f16(b, scale, x[2], x[3]);
  return f16x8{x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
}

constexpr int kMinPage = 8;  // the attention kernels take keys in groups of 8 that lie on one page

// Checks a cache's arguments and fills `c`; 0, or -1 with the reason printed.
template <class C>
int paged_cache(const char* who, const void* kp, const void* vp, long long page_stride, int pages, int page, const int* table, int ldt,
                int W, int B, int Hkv, int D, C& c) {
  constexpr int kAlign = 16 / sizeof(typename C::Elem);  // elements of an access
  if (D != 64 && D != 128) HI_FAIL("%s: head dim %d (64 or 128)", who, D);
  if (page < kMinPage || (page & (page - 1))) HI_FAIL("%s: page of %d positions (a power of two >= %d)", who, page, kMinPage);
  if (Hkv < 1 || Hkv > 4096 || pages < 1 || W < 1 || B < 0 || ldt < W)
    HI_FAIL("%s: Hkv %d, pages %d, table [%d, %d] with row stride %d", who, Hkv, pages, B, W, ldt);
  if ((int64_t)W * page > (1 << 30)) HI_FAIL("%s: %d pages of %d positions (at most 2^30 positions a sequence)", who, W, page);
  if ((int64_t)Hkv * page * D * 2 > INT32_MAX) HI_FAIL("%s: a page of over 2 GiB", who);
  if (page_stride % kAlign || (pages > 1 && page_stride < (int64_t)Hkv * page * D))
    HI_FAIL("%s: page stride %lld (a multiple of %d, at least Hkv * page * D)", who, page_stride, kAlign);
  if (!kp || !vp || (!table && B > 0) || ((uintptr_t)kp & 15) || ((uintptr_t)vp & 15) || ((uintptr_t)table & 3))
    HI_FAIL("%s: kp and vp must be 16-byte aligned, table 4-byte aligned, none null", who);
  int shift = 0;
  while ((1 << shift) < page) shift++;
  c.kp = (const typename C::Elem*)kp;
  c.vp = (const typename C::Elem*)vp;
  c.stride = page_stride;
  c.pages = pages;
  c.shift = shift;
  c.table = table;
  c.ldt = ldt;
  c.W = W;
  return 0;
}
