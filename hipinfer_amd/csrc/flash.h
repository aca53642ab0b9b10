// What the causal attention kernels of prefill.hip (a cache slot) and paged.hip (pages) have in common: the LDS tiles and
// their swizzle, the DMA into them and the transpose read out of them. Their tile loop is flash_tile.h.
#pragma once
#include <type_traits>

#include "hi_common.h"

namespace {

constexpr int kFpRG = 4;              // 32-row groups per block (2 waves each); 2 for small grids
constexpr int kFpKPW = 64;            // keys per wave per tile (32-key MFMA blocks of the wave's half)
constexpr int kFpBKV = 2 * kFpKPW;    // keys per tile
constexpr int kFpStages = 2;          // LDS stages of K/V tiles
constexpr float kFpMaxLag = 8.f;      // log2 of how far a row's reference max may trail its max

// XOR term of key r's 16-byte chunks in the K tile: the 16 keys (D = 128) or 8 key pairs (D = 64)
// that one 128-bit fragment read serves per cycle land on distinct banks.
template <int D>
__device__ __forceinline__ int k_swz(int r) {
  if constexpr (D == 128) return r & 15;
  else return (r >> 1) & 7;
}
// XOR term of key r's chunks in the V tile. A transpose read covers keys r..r+3 (r % 4 == 0) at
// 4 consecutive chunks per 32 lanes and 2 per 16 lanes; the terms 0, 6, 12, 10 (D = 128) or 0, 6,
// 4, 2 (D = 64) for r % 4 = 0..3 move those chunks to distinct banks at either width.
template <int D>
__device__ __forceinline__ int v_swz(int r) {
  const int a = r & 3;
  return ((2 * a) ^ (4 * a)) & (D / 8 - 1);
}

// LDS of one block: two stages of K tiles and two of V tiles while the keys stream, then in the same
// bytes the O^T accumulators the second wave of each row group hands to the first; last, the second
// waves' m and l. It is dynamic LDS: reads of a __shared__ array that a DMA instruction also writes
// made the compiler wait for every DMA in flight (s_waitcnt vmcnt(0)) before the first of them, right
// after the next tile's DMA had been issued, so that no tile streamed in while another was computed.
template <int D, int RG>
struct FpSmem {
  static constexpr int kTile = kFpBKV * D / 8;                // 16-byte chunks of one K or V tile
  static constexpr int kMl = 2 * kFpStages * kTile;           // chunk index of m and l
  static constexpr size_t kBytes = kMl * 16 + 2 * RG * 64 * 4;
  static_assert(RG * (D / 32) * 64 * 64 <= kMl * 16, "merge fits the stages");
};

typedef short i16x4 __attribute__((ext_vector_type(4)));

// The two builtins below sit in the device pass only: in this kernel's host pass they made the
// compiler drop the kernel's launch stub without a diagnostic (an undefined symbol at load).
// 16-byte buffer DMA of each lane's chunk at byte offset voff into LDS slot lane of `lds`.
__device__ __forceinline__ void lds_dma16(__amdgpu_buffer_rsrc_t rs, void* lds, int voff) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)lds, 16, voff, 0, 0, 0);
#endif
}
// ds_read_tr16_b64 at LDS address p: within each 16-lane group, lane i receives element i % 4 of
// the 4 halves lane 4 e + i / 4 addresses, as its element e.
__device__ __forceinline__ f16x4 lds_read_tr16(const f16* __restrict__ p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)p));
#else
  return f16x4{};
#endif
}

}  // namespace
