// The paged key/value cache as the kernels see it, and what its host entry points check alike.
#pragma once
#include "hi_common.h"

// kp / vp [pages][Hkv][page][D] fp16, pages `stride` halves apart (the same for both); position p of sequence b is
// row p % page of page table[b][p / page]. A page id outside [0, pages) is no page.
struct PagedCache {
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

constexpr int kMinPage = 8;  // the attention kernels take keys in groups of 8 that lie on one page

// Checks the cache's arguments and fills `c`; 0, or -1 with the reason printed.
inline int paged_cache(const char* who, const void* kp, const void* vp, long long page_stride, int pages, int page,
                       const int* table, int ldt, int W, int B, int Hkv, int D, PagedCache& c) {
  if (D != 64 && D != 128) HI_FAIL("%s: head dim %d (64 or 128)", who, D);
  if (page < kMinPage || (page & (page - 1))) HI_FAIL("%s: page of %d positions (a power of two >= %d)", who, page, kMinPage);
  if (Hkv < 1 || Hkv > 4096 || pages < 1 || W < 1 || B < 0 || ldt < W)
    HI_FAIL("%s: Hkv %d, pages %d, table [%d, %d] with row stride %d", who, Hkv, pages, B, W, ldt);
  if ((int64_t)W * page > (1 << 30)) HI_FAIL("%s: %d pages of %d positions (at most 2^30 positions a sequence)", who, W, page);
  if ((int64_t)Hkv * page * D * 2 > INT32_MAX) HI_FAIL("%s: a page of over 2 GiB", who);
  if (page_stride % 8 || (pages > 1 && page_stride < (int64_t)Hkv * page * D))
    HI_FAIL("%s: page stride %lld (a multiple of 8, at least Hkv * page * D)", who, page_stride);
  if (!kp || !vp || (!table && B > 0) || ((uintptr_t)kp & 15) || ((uintptr_t)vp & 15) || ((uintptr_t)table & 3))
    HI_FAIL("%s: kp and vp must be 16-byte aligned, table 4-byte aligned, none null", who);
  int shift = 0;
  while ((1 << shift) < page) shift++;
  c = PagedCache{(const f16*)kp, (const f16*)vp, (int64_t)page_stride, pages, shift, table, ldt, W};
  return 0;
}
