// Beam search's selection (hi_beam_select): of the continuations of `beams` rows of logits by every token of the vocabulary, the n
// with the best scores, score(k, t) = scores[k] + x[k][t] - max - log(sum exp(x[k] - max)).
//
// The logits are read once, as a stream: that is the floor, 2 bytes a logit. Which of them can be among the n best is left open
// there: a wave notes the largest of every 512 consecutive logits (a segment), and the maximum and sum of exponentials of every 4
// segments. The n best candidates lie in the n best segments, segments ordered by their best candidate and then by place: a
// candidate outside them has n segments, so n candidates, before it. So a second kernel, a block per sequence, joins the sums,
// picks n segments, and reads those again: 512 n logits instead of beams * vocabulary.
//
// Exponentials are fp32, and so are their sums within a wave's 2048 logits (a lane's 32 relative to the lane's own maximum, then over
// the lanes); a row's waves are joined in 64 bits. That leaves a row's log sum off by 2^-17 at most, a small part of what the fp16
// logits are rounded by, and candidates of different rows that are nearer to each other may come in either order. Computed scores
// are compared by keys of 64 bits: 40 bits of the distance d from the best (of 1 + d, 2^-35 of it), then the place, so that a key is
// unique and the lowest (beam, token) wins a tie.
#include "hi_common.h"
#include "row_overlap.h"

namespace {

constexpr int kSeg = 512;         // logits of a segment: a wave's 16-byte loads
constexpr int kSegs = 4;          // segments of a wave
constexpr int kMaxBeams = 64, kMaxBest = 64;
constexpr int kPick = 1024;       // threads of the second kernel
constexpr int kGroups = 64;       // of them, for a bound on the n-th best segment: at least n
constexpr int kAhead = 4;         // segments that a thread has in registers
constexpr int kList = 2048;       // candidates that are ranked in LDS
constexpr float kSlack = 1 + 0x1p-19f;  // more than fp32 distances are off by
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

// grid (ceil(waves / 4), R); WIDE: rows on 16-byte boundaries. 256 rows of 128256 logits 13.7 us, 4.8 TB/s: a large copy's rate.
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
  double logsum[kMaxBeams];  // log sum exp(x - top); NaN for a beam without candidates
  double off[kMaxBeams];     // how far the beam's best candidate is from the best of all; infinite without candidates
  float score[kMaxBeams];    // scores[k]
  float top[kMaxBeams];      // the beam's largest logit
  float far[kMaxBeams];      // off as fp32
  float best[kGroups];
  uint64_t list[kList];
  uint64_t out[kMaxBest];   // the n least keys in order
  uint64_t red[kPick / 64];
  float limit;
  int found;
};

// Key of distance d >= 0 from the best score and place `at` < 2^24; kNone from 2^31 on (and for NaN).
__device__ __forceinline__ uint64_t key_of(double d, uint32_t at) {
  if (!(d < 2147483648.0)) return kNone;
  const uint64_t b = (uint64_t)__builtin_bit_cast(int64_t, 1.0 + d) - 0x3ff0000000000000ull;
  return (b >> 17) << 24 | at;
}
// No distance whose key is that of d or less exceeds this.
__device__ __forceinline__ float limit_of(uint64_t key) {
  const double d = __builtin_bit_cast(double, (int64_t)((((key >> 24) + 1) << 17) + 0x3ff0000000000000ull)) - 1.0;
  return (float)d * kSlack;
}

// The n least of the block's keys, in order, into sh.out (kNone behind the last); keys are unique but for kNone. push(f) calls f with
// a few keys of the thread, the n least of all among them; all(f) with every one. The few are ranked in LDS; where they are too many
// for it (thousands of equal logits), all are gone through n times.
template <typename Push, typename All>
__device__ __forceinline__ void least_keys(PickSmem& sh, int n, Push push, All all) {
  const int tid = threadIdx.x;
  if (tid < n) sh.out[tid] = kNone;
  if (tid == 0) sh.found = 0;
  __syncthreads();
  push([&](uint64_t k) {
    if (k == kNone) return;
    const int at = atomicAdd(&sh.found, 1);
    if (at < kList) sh.list[at] = k;
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
  uint64_t last = 0;
  for (int j = 0; j < n; j++) {
    uint64_t k = kNone;
    all([&](uint64_t v) {
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

// One block per sequence. What is compared for every segment and logit is the fp32 distance from the best, far[k] + (top[k] - x), off
// by 2^-22 of it at most; the keys of 64 bits are made for those alone that can be among the n best by it:
//  * of the segments, those up to the n-th least of 64 groups' least distances (at least n segments are that near);
//  * of their logits, those up to the n-th segment's best one (the segments' best ones are n that near).
// What bounds it: a chain of some ten waits (sums and segments from memory, exp and log in 64 bits, two rankings, the picked logits from
// memory): 7.5 us for 4 beams, 8.8 for 32 times 8 (with 64-bit keys for every segment and logit, in blocks of 256: 16.8 and 27.8).
template <bool WIDE>
__global__ void __launch_bounds__(kPick) beam_pick_kernel(const f16* __restrict__ logits, int64_t ldl, const float* __restrict__ scores,
                                                          int V, int R, int K, int n, const char* work, float* best, int* parent,
                                                          int* token) {
  __shared__ PickSmem sh;
  __shared__ int seg_beam[kMaxBest], seg_token[kMaxBest];  // the picked segments' first logits; -1
  const BeamWork w(R, V);
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = K * w.segs;
  const f16* const most = (const f16*)work + (int64_t)b * S;
  const float* const pairs = (const float*)(work + w.pairs) + 2 * (int64_t)b * K * w.waves;
  f16 x0[kAhead];  // the thread's first segments, requested ahead of the sums
#pragma unroll
  for (int j = 0; j < kAhead; j++) x0[j] = tid + j * kPick < S ? most[tid + j * kPick] : (f16)0.f;
  // ---- the beams' log sums
  for (int k = wave; k < K; k += kPick / 64) {
    const float* p = pairs + 2 * (int64_t)k * w.waves;
    const float s = scores[b * K + k];
    float M = -__builtin_huge_valf();
    for (int i = lane; i < w.waves; i += 64) M = fmaxf(M, p[2 * i]);
    M = wave_max(M);
    double sum = 0;
    for (int i = lane; i < w.waves; i += 64) sum += (double)p[2 * i + 1] * exp((double)p[2 * i] - (double)M);
    sum = wave_sum64(sum);
    if (lane == 0) {
      sh.score[k] = s;
      sh.top[k] = M;
      sh.logsum[k] = s - s == 0.f && M - M == 0.f && sum - sum == 0.0 ? log(sum) : __builtin_nan("");  // none of them infinite
    }
  }
  __syncthreads();
  // ---- how far the beams' best candidates (their largest logits) are from the best of all. Log sums and logits are added to
  // differences of scores, never to a score: beside one of 1e17 or the lowest float they would be rounded away, and candidates that
  // differ would be equal by their keys but not by `far`.
  static_assert(kMaxBeams <= 64, "a lane per beam");
  if (wave == 0) {
    const bool any = lane < K && sh.logsum[lane] == sh.logsum[lane];
    const float s = any ? sh.score[lane] : -__builtin_huge_valf(), most = wave_max(s);
    const double e = any ? ((double)s - (double)most) - sh.logsum[lane] : -__builtin_huge_val();
    double top = e;
    for (int o = 1; o < K; o <<= 1) top = fmax(top, __shfl_xor(top, o, 64));  // (of the 2^i >= K lanes that hold the beams)
    if (lane < K) {
      sh.off[lane] = any ? top - e : __builtin_huge_val();
      sh.far[lane] = (float)sh.off[lane];
    }
  }
  __syncthreads();
  auto key = [&](int k, float x, int t) { return key_of(sh.off[k] + ((double)sh.top[k] - (double)x), (uint32_t)(k * V + t)); };
  auto far = [&](int k, float x) { return sh.far[k] + (sh.top[k] - x); };
  // ---- the n best segments
  const float inv = 1.0f / (float)w.segs;
  auto beam_of = [&](int i) {  // i / segs, below 64: the product is off by less than one
    int k = (int)((float)i * inv);
    if (k * w.segs > i) k--;
    return i - k * w.segs >= w.segs ? k + 1 : k;
  };
  auto segments = [&](auto f) {  // f(beam, segment, its largest logit)
    auto one = [&](int i, float x) {
      const int k = beam_of(i);
      f(k, i - k * w.segs, x);
    };
#pragma unroll
    for (int j = 0; j < kAhead; j++)
      if (tid + j * kPick < S) one(tid + j * kPick, (float)x0[j]);
    for (int i = tid + kAhead * kPick; i < S; i += kPick) one(i, (float)most[i]);
  };
  float near = __builtin_huge_valf(), d0[kAhead];  // (d0: the first segments' distances)
#pragma unroll
  for (int j = 0; j < kAhead; j++) {
    const int i = tid + j * kPick;
    d0[j] = i < S ? far(beam_of(i), (float)x0[j]) : __builtin_huge_valf();
    near = fminf(near, d0[j]);
  }
  for (int i = tid + kAhead * kPick; i < S; i += kPick) near = fminf(near, far(beam_of(i), (float)most[i]));
  constexpr int kLanes = kPick / kGroups;  // of a group
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) near = fminf(near, __shfl_xor(near, o, 64));
  if ((tid & (kLanes - 1)) == 0) sh.best[tid / kLanes] = near;
  if (tid == 0) sh.limit = __builtin_huge_valf();
  __syncthreads();
  if (tid < kGroups) {
    const float mine = sh.best[tid];
    int before = 0;
#pragma unroll
    for (int g = 0; g < kGroups; g++) before += sh.best[g] < mine || (sh.best[g] == mine && g < tid);
    if (before == n - 1) sh.limit = mine * kSlack + 0x1p-34f;  // (infinite with fewer than n groups that have any)
  }
  __syncthreads();
  const float limit = sh.limit;
  least_keys(
      sh, n,
      [&](auto f) {
        auto one = [&](int i, float x) {
          const int k = beam_of(i);
          f(key(k, x, (i - k * w.segs) * kSeg));
        };
#pragma unroll
        for (int j = 0; j < kAhead; j++)
          if (d0[j] <= limit && tid + j * kPick < S) one(tid + j * kPick, (float)x0[j]);
        for (int i = tid + kAhead * kPick; i < S; i += kPick) {
          const float x = (float)most[i];
          if (far(beam_of(i), x) <= limit) one(i, x);
        }
      },
      [&](auto f) { segments([&](int k, int s, float x) { f(key(k, x, s * kSeg)); }); });
  if (tid < n) {
    const int at = sh.out[tid] == kNone ? -1 : (int)(sh.out[tid] & 0xffffff), k = at < 0 ? -1 : at / V;
    seg_beam[tid] = k;
    seg_token[tid] = at - k * V;
  }
  const uint64_t nth = sh.out[n - 1];
  const float cut = nth == kNone ? __builtin_huge_valf() : limit_of(nth);
  __syncthreads();
  // ---- the n best candidates in them
  auto chunks = [&](auto f) {  // f(beam, logit, token)
    for (int i = tid; i < n * (kSeg / 8); i += kPick) {
      const int k = seg_beam[i / (kSeg / 8)], t = seg_token[i / (kSeg / 8)] + i % (kSeg / 8) * 8;
      if (k < 0) continue;
      const f16x8 x = load8<WIDE>(logits + ((int64_t)b * K + k) * ldl, V, t);
#pragma unroll
      for (int e = 0; e < 8; e++) f(k, (float)x[e], t + e);
    }
  };
  least_keys(
      sh, n,
      [&](auto f) {
        chunks([&](int k, float x, int t) {
          if (far(k, x) <= cut) f(key(k, x, t));
        });
      },
      [&](auto f) { chunks([&](int k, float x, int t) { f(key(k, x, t)); }); });
  if (tid < n) {
    const uint64_t q = sh.out[tid];
    float s = -__builtin_huge_valf();
    int k = -1, t = -1;
    if (q != kNone) {
      const int at = (int)(q & 0xffffff);
      k = at / V;
      t = at - k * V;
      s = (float)(((double)logits[((int64_t)b * K + k) * ldl + t] - (double)sh.top[k]) + ((double)sh.score[k] - sh.logsum[k]));
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
  // a sequence's block has read its scores before it writes as many in their place; other places are other blocks'
  if (!in_place_or_apart(scores, 4 * (int64_t)beams, 4 * (int64_t)beams, best, 4 * (int64_t)n, 4 * (int64_t)n, B))
    HI_FAIL("%s: best must be scores (with n == beams) or apart from it", who);
  const BeamWork w(B * beams, V);
  if (!work || ((uintptr_t)work & 15) || work_bytes < w.bytes)
    HI_FAIL("%s: work of %zu bytes (at least %zu, 16-byte aligned)", who, work_bytes, w.bytes);
  const int64_t places = 4 * (int64_t)B * n;
  const CallRows rows[] = {{"logits", logits, 2 * (int64_t)ldl, 2 * (int64_t)V, B * beams, false},
                           call_flat("scores", scores, 4 * (int64_t)B * beams, false), call_flat("best", best, places, true, 1),
                           call_flat("parent", parent, places, true), call_flat("token", token, places, true),
                           call_flat("work", work, (int64_t)w.bytes, true)};
  const char *a0, *a1;
  if (call_rows_meet(rows, a0, a1)) HI_FAIL("%s: %s and %s must be apart", who, a0, a1);
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
