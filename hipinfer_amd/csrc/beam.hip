// Beam search's selection (hi_beam_select): of the continuations of `beams` rows of logits by every token of the vocabulary, the n
// with the best scores, score(k, t) = scores[k] + x[k][t] - max - log(sum exp(x[k] - max)).
//
// The logits are read once, as a stream: that is the floor, 2 bytes a logit. Which of them can be among the n best is left open
// there: a wave notes the largest of every 512 consecutive logits (a segment), and the maximum and sum of exponentials of every 4
// segments. The n best candidates lie in the n best segments, segments ordered by their best candidate and then by place: a
// candidate outside them has n segments, so n candidates, before it. So a second kernel, a block per sequence, joins the sums,
// picks n segments, and reads those again: 512 n logits instead of beams * vocabulary.
//
// Exponentials and a lane's sum of 32 are fp32 (relative to the lane's own maximum), joined in 64 bits; scores are compared in 64
// bits, as keys of 64 bits: 40 bits of the distance d from the best (of 1 + d, 2^-35 of it), then the place, so that a key is unique
// and the lowest (beam, token) wins a tie.
#include "hi_common.h"

namespace {

constexpr int kSeg = 512;         // logits of a segment: a wave's 16-byte loads
constexpr int kSegs = 4;          // segments of a wave
constexpr int kMaxBeams = 64, kMaxBest = 64;
constexpr int kPick = 256;        // threads of the second kernel
constexpr int kList = 2048;       // candidates that are ranked in LDS
constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint64_t kNone = ~0ull;

// Work buffer: the segments' maxima [R][segs] fp16, the waves' maxima and sums [R][waves] fp32 pairs.
struct BeamWork {
  int segs, waves;
  size_t pairs, bytes;
  __host__ __device__ BeamWork(int R, int V) {
    segs = (V + kSeg - 1) / kSeg;
    waves = (segs + kSegs - 1) / kSegs;
    pairs = ((size_t)R * segs * 2 + 15) & ~(size_t)15;
    bytes = pairs + (size_t)R * waves * 8;
  }
};

// 8 logits from i on of a row of V; -inf behind its end.
template <bool WIDE>
__device__ __forceinline__ f16x8 load8(const f16* row, int V, int i) {
  if (WIDE && i + 8 <= V) return *reinterpret_cast<const f16x8*>(row + i);
  f16x8 x;
#pragma unroll
  for (int e = 0; e < 8; e++) x[e] = i + e < V ? row[i + e] : (f16)(-__builtin_huge_valf());
  return x;
}

// grid (ceil(waves / 4), R); WIDE: rows on 16-byte boundaries
template <bool WIDE>
__global__ void __launch_bounds__(256) beam_scan_kernel(const f16* __restrict__ logits, int64_t ldl, int V, int R, char* work) {
  const BeamWork w(R, V);
  const int r = blockIdx.y, wave = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (wave >= w.waves) return;
  const f16* row = logits + r * ldl;
  f16x8 x[kSegs];
#pragma unroll
  for (int s = 0; s < kSegs; s++) x[s] = load8<WIDE>(row, V, (wave * kSegs + s) * kSeg + lane * 8);
  // (a NaN is passed over by the maxima and makes the sum NaN)
  float most[kSegs], m = -__builtin_huge_valf();
#pragma unroll
  for (int s = 0; s < kSegs; s++) {
    float v = -__builtin_huge_valf();
#pragma unroll
    for (int e = 0; e < 8; e++) v = fmaxf(v, (float)x[s][e]);
    m = fmaxf(m, v);
    most[s] = wave_max(v);
  }
  const float ref = m == -__builtin_huge_valf() ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int s = 0; s < kSegs; s++)
#pragma unroll
    for (int e = 0; e < 8; e++) sum += __builtin_amdgcn_exp2f(((float)x[s][e] - ref) * kLog2e);
  float M = most[0];
#pragma unroll
  for (int s = 1; s < kSegs; s++) M = fmaxf(M, most[s]);
  const float Mref = M == -__builtin_huge_valf() ? 0.f : M;
  sum = wave_sum(sum * __builtin_amdgcn_exp2f((m - Mref) * kLog2e));
  if (lane < kSegs && wave * kSegs + lane < w.segs) {
    float v = most[0];
#pragma unroll
    for (int s = 1; s < kSegs; s++) v = lane == s ? most[s] : v;
    ((f16*)work)[(int64_t)r * w.segs + wave * kSegs + lane] = (f16)v;
  }
  if (lane == 0) {
    float* p = (float*)(work + w.pairs) + 2 * ((int64_t)r * w.waves + wave);
    p[0] = M;
    p[1] = sum;
  }
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

struct PickSmem {
  double base[kMaxBeams];   // scores[k] - log sum; NaN for a beam without candidates
  float top[kMaxBeams];     // the beam's largest logit
  uint64_t best[kPick];
  uint64_t list[kList];
  uint64_t out[kMaxBest];   // the n least keys in order
  uint64_t red[kPick / 64];
  uint64_t limit;
  int found;
};

// Key of distance d >= 0 from the best score and place `at` < 2^24; kNone from 2^31 on (and for NaN).
__device__ __forceinline__ uint64_t key_of(double d, uint32_t at) {
  if (!(d < 2147483648.0)) return kNone;
  const uint64_t b = (uint64_t)__builtin_bit_cast(int64_t, 1.0 + d) - 0x3ff0000000000000ull;
  return (b >> 17) << 24 | at;
}

// The n least of the block's keys, in order, into sh.out (kNone behind the last). each(f) calls f with every key of the thread, the
// same ones every time; keys are unique but for kNone.
template <typename Each>
__device__ __forceinline__ void least_keys(PickSmem& sh, int n, Each each) {
  const int tid = threadIdx.x;
  uint64_t mine = kNone;
  each([&](uint64_t k) { mine = k < mine ? k : mine; });
  sh.best[tid] = mine;
  if (tid < n) sh.out[tid] = kNone;
  if (tid == 0) {
    sh.limit = kNone - 1;  // with fewer than n threads that have any, all keys that are any
    sh.found = 0;
  }
  __syncthreads();
  // the n-th least of the threads' least keys bounds the n-th least of all
  int before = 0;
#pragma unroll 16
  for (int t = 0; t < kPick; t++) before += sh.best[t] < mine;
  if (before == n - 1 && mine != kNone) sh.limit = mine;
  __syncthreads();
  const uint64_t limit = sh.limit;
  if (mine <= limit)
    each([&](uint64_t k) {
      if (k <= limit) {
        const int at = atomicAdd(&sh.found, 1);
        if (at < kList) sh.list[at] = k;
      }
    });
  __syncthreads();
  const int found = sh.found;
  if (found <= kList) {
    for (int i = tid; i < found; i += kPick) {
      const uint64_t k = sh.list[i];
      int rank = 0;
      for (int j = 0; j < found; j++) rank += sh.list[j] < k;
      if (rank < n) sh.out[rank] = k;
    }
    __syncthreads();
    return;
  }
  // so many at or before the bound (thousands of equal logits): one after the other
  uint64_t last = 0;
  for (int j = 0; j < n; j++) {
    uint64_t k = kNone;
    each([&](uint64_t v) {
      if ((j == 0 || v > last) && v < k) k = v;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t v = __shfl_xor((unsigned long long)k, o, 64);
      k = v < k ? v : k;
    }
    if ((tid & 63) == 0) sh.red[tid >> 6] = k;
    __syncthreads();
    last = kNone;
#pragma unroll
    for (int q = 0; q < kPick / 64; q++) last = sh.red[q] < last ? sh.red[q] : last;
    if (tid == 0) sh.out[j] = last;
    __syncthreads();
  }
}

// One block per sequence.
template <bool WIDE>
__global__ void __launch_bounds__(kPick) beam_pick_kernel(const f16* __restrict__ logits, int64_t ldl, const float* __restrict__ scores,
                                                          int V, int R, int K, int n, const char* work, float* best, int* parent,
                                                          int* token) {
  __shared__ PickSmem sh;
  __shared__ uint32_t seg[kMaxBest];  // the places of the first logits of the picked segments
  const BeamWork w(R, V);
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const f16* const most = (const f16*)work + (int64_t)b * K * w.segs;
  const float* const pairs = (const float*)(work + w.pairs) + 2 * (int64_t)b * K * w.waves;
  // ---- the beams' log sums
  for (int k = wave; k < K; k += kPick / 64) {
    const float* p = pairs + 2 * (int64_t)k * w.waves;
    float M = -__builtin_huge_valf();
    for (int i = lane; i < w.waves; i += 64) M = fmaxf(M, p[2 * i]);
    M = wave_max(M);
    double sum = 0;
    for (int i = lane; i < w.waves; i += 64) sum += (double)p[2 * i + 1] * exp((double)p[2 * i] - (double)M);
    sum = wave_sum64(sum);
    if (lane == 0) {
      const double s = (double)scores[b * K + k];
      sh.top[k] = M;
      sh.base[k] = s - s == 0.0 && M - M == 0.f && sum - sum == 0.0 ? s - log(sum) : __builtin_nan("");  // none of them infinite
    }
  }
  __syncthreads();
  auto score = [&](int k, float x) { return ((double)x - (double)sh.top[k]) + sh.base[k]; };
  double top = -__builtin_huge_val();
  for (int k = 0; k < K; k++)
    if (sh.base[k] > top) top = sh.base[k];  // a beam's best candidate is its largest logit
  // ---- the n best segments
  least_keys(sh, n, [&](auto f) {
    for (int i = tid; i < K * w.segs; i += kPick) {
      const int k = i / w.segs;
      f(key_of(top - score(k, (float)most[i]), (uint32_t)(k * V + (i - k * w.segs) * kSeg)));
    }
  });
  if (tid < n) seg[tid] = sh.out[tid] == kNone ? ~0u : (uint32_t)sh.out[tid] & 0xffffff;
  __syncthreads();
  // ---- the n best candidates in them
  least_keys(sh, n, [&](auto f) {
    for (int i = tid; i < n * (kSeg / 8); i += kPick) {
      const uint32_t first = seg[i / (kSeg / 8)];
      if (first == ~0u) continue;
      const int k = first / V, t = first - k * V + i % (kSeg / 8) * 8;
      const f16x8 x = load8<WIDE>(logits + ((int64_t)b * K + k) * ldl, V, t);
#pragma unroll
      for (int e = 0; e < 8; e++) f(key_of(top - score(k, (float)x[e]), (uint32_t)(k * V + t + e)));
    }
  });
  if (tid < n) {
    const uint64_t key = sh.out[tid];
    float s = -__builtin_huge_valf();
    int k = -1, t = -1;
    if (key != kNone) {
      const int at = (int)(key & 0xffffff);
      k = at / V;
      t = at - k * V;
      s = (float)score(k, (float)logits[((int64_t)b * K + k) * ldl + t]);
      k += b * K;
    }
    best[b * n + tid] = s;
    parent[b * n + tid] = k;
    token[b * n + tid] = t;
  }
}

}  // namespace

HI_EXPORT size_t hi_beam_select_work_bytes(int B, int beams, int V, int n) {
  if (B < 0 || beams < 1 || beams > kMaxBeams || V < 1 || n < 1 || n > kMaxBest || (int64_t)beams * V > 1 << 24 ||
      (int64_t)B * beams > 65535) return 0;
  return BeamWork(B * beams, V).bytes + 16;
}

HI_EXPORT int hi_beam_select(const void* logits, long long ldl, const float* scores, int B, int beams, int V, int n, float* best,
                             int* parent, int* token, void* work, size_t work_bytes, void* stream) {
  const char* who = "hi_beam_select";
  if (B < 0 || beams < 1 || beams > kMaxBeams || V < 1 || n < 1 || n > kMaxBest || (int64_t)beams * V > 1 << 24)
    HI_FAIL("%s: B %d, %d beams (1 to %d), V %d (beams * V at most 2^24), n %d (1 to %d)", who, B, beams, kMaxBeams, V, n, kMaxBest);
  if ((int64_t)B * beams > 65535) HI_FAIL("%s: %d rows of logits (at most 65535)", who, B * beams);
  if (B == 0) return 0;
  if (!logits || !scores || !best || !parent || !token || ((uintptr_t)logits & 1) || ldl < V ||
      ((uintptr_t)scores | (uintptr_t)best | (uintptr_t)parent | (uintptr_t)token) & 3)
    HI_FAIL("%s: a null or misaligned pointer, or ldl < V", who);
  const BeamWork w(B * beams, V);
  if (!work || ((uintptr_t)work & 15) || work_bytes < w.bytes)
    HI_FAIL("%s: work of %zu bytes (at least %zu, 16-byte aligned)", who, work_bytes, w.bytes);
  if (!hi_device()) return -2;
  const hipStream_t s = (hipStream_t)stream;
  const f16* x = (const f16*)logits;
  const bool wide = ((uintptr_t)x & 15) == 0 && ldl % 8 == 0;
  const int R = B * beams;
  const dim3 grid((w.waves + 3) / 4, R);
  if (wide) {
    hipLaunchKernelGGL(beam_scan_kernel<true>, grid, dim3(256), 0, s, x, (int64_t)ldl, V, R, (char*)work);
    hipLaunchKernelGGL(beam_pick_kernel<true>, dim3(B), dim3(kPick), 0, s, x, (int64_t)ldl, scores, V, R, beams, n,
                       (const char*)work, best, parent, token);
  } else {
    hipLaunchKernelGGL(beam_scan_kernel<false>, grid, dim3(256), 0, s, x, (int64_t)ldl, V, R, (char*)work);
    hipLaunchKernelGGL(beam_pick_kernel<false>, dim3(B), dim3(kPick), 0, s, x, (int64_t)ldl, scores, V, R, beams, n,
                       (const char*)work, best, parent, token);
  }
  HI_TRY(hipGetLastError());
  return 0;
}
