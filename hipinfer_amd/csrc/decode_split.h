// What decode attention over slots (decode.hip) and over pages (paged.hip) have in common: how the keys of a (sequence, kv
// head) pair are split over blocks, and the exchange of the splits' results.
#pragma once
#include "hi_common.h"

namespace {

constexpr int kDecodeMaxSplits = 64;
constexpr int kDaTile = 32;  // keys per wave tile (one k step of P.V)

__device__ __forceinline__ float ld_coherent(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void st_coherent(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Maximum (or sum) over the four 16-lane rows of a wave, each lane with the lanes of its own column.
template <bool MAX>
__device__ __forceinline__ float rows_reduce(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = MAX ? fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])) : __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = MAX ? fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1])) : __uint_as_float(b[0]) + __uint_as_float(b[1]);
#endif
  return v;
}

// Splits in use for `len` keys when a launch has S per pair, S1 of them to give every CU its two blocks (one of
// 8 waves): of those, one per 256 keys, but down to 128 keys a split while there are at most
// 16 (what the merge requests in one round): shorter waves finish sooner, and more splits cost more
// in the merge (one sequence of 4001 keys, 32/8 heads: 16 splits 10.8 us, 32 splits 12.5; of 2500: 16
// 9.5, 10 9.9). Up to 256 keys one split, which has no partials and no merge (200 keys, two splits / one, us:
// one sequence 7.3 / 5.8, 8 of them 8.6 / 6.2, 24 10.5 / 6.9). Beyond S1, where the launch has them
// (decode_splits_max), only for runs over 1024 keys, which would end a ragged batch late.
__device__ __forceinline__ int splits_used(int len, int S, int S1) {
  if (len <= 256) return 1;
  return max(min(S1, max((len + 255) / 256, min(16, (len + 127) / 128))), min(S, (len + 1023) / 1024));
}

// Splits of a (sequence, kv head) pair that give every CU two blocks (as api.cu:643-646), at most the
// work buffer's 64.
int decode_splits(int B, int Hkv, int cus) { return min((2 * cus + B * Hkv - 1) / (B * Hkv), kDecodeMaxSplits); }

// Blocks of 8 waves where that is 16 or more (at most about an eighth as many pairs as CUs): a launch this
// small is a chain of latencies, and a block of 256 keys is then one tile per wave (one sequence of
// 2500 keys 9.45 -> 9.0 us, of 8000 14.8 -> 13.8, four of 700 to 800 at D = 64 8.1 -> 7.4); with more
// pairs 4 waves balance better (40 sequences of 300 to 2400, 12/2 heads: 19.5 against 25.5). A CU holds one
// such block at D = 128 (12 waves of 137 registers), so the launch has at most one for each: with two, the
// lengths that use more than half of them run a part-filled second round (32/8 heads of 128, two / one, us: one
// sequence of 12000 21.4 / 17.0, two of 6000 20.8 / 16.7, four of 2000 15.3 / 11.9, one of 32000 34.4 / 29.6; two
// of 6000, 32/4 heads of 64, 10.5 / 10.4, of 20000 18.5 / 15.3).
constexpr int kDaWideSplits = 16;
int decode_splits_wide(int B, int Hkv, int cus) { return min(max(cus / (B * Hkv), 1), kDecodeMaxSplits); }

// Splits per pair that a launch has for its long runs (splits_used): 2 S1, or S1 where more would be spread
// worse over the CUs. A batch may be uniform, all of its pairs then take S1 + 1 splits at once: S1 blocks
// a pair that are a whole number for every CU stay that, and so do those whose last layer over the CUs
// would be left emptier by more than a sixteenth of all layers. At S1 = 1 a second split also brings the
// partials and their merge, and a part-filled second round of blocks (a CU holds 3 at D = 128). Measured
// with 32/8 heads of 128, S1 alone / up to 2 S1, us: 64 x 1025 keys 49.6 / 55.1, 64 x 2000 94.1 / 100.5,
// 120 x 1025 91.6 / 101.8, 16 x 4097 52.8 / 57.1, 44 x 2049 70.9 / 76.7; 24 x 3073 66.0 / 60.6, 52 x 2049
// 89.5 / 85.8, 30 of 500 to 4000 70.0 / 66.0, 24 of 576 to 4608 68.8 / 54.5. It reads no lengths: a
// sequence's sums do not depend on its neighbours'.
int decode_splits_max(int B, int Hkv, int S1, int cus) {
  const int n0 = B * Hkv * S1, n1 = n0 + B * Hkv;  // blocks
  const int l0 = (n0 + cus - 1) / cus, l1 = (n1 + cus - 1) / cus;  // layers of one block a CU
  // n0 / (l0 cus) and n1 / (l1 cus) are the shares of the layers that are filled
  const bool worse = S1 == 1 || n0 % cus == 0 || 16 * ((int64_t)n0 * l1 - (int64_t)n1 * l0) > (int64_t)l0 * l1 * cus;
  return worse ? S1 : min(2 * S1, kDecodeMaxSplits);
}

}  // namespace
