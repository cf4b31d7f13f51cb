// Choice of the largest of many 32-bit keys by one thread block, and where each chosen one stands among the others.
#pragma once
#include "common.cuh"

namespace swb {

// Order-preserving key of a float: a < b as numbers means key(a) < key(b); -0 and +0 are one key, every NaN lies above +inf.
__device__ __forceinline__ uint32_t float_key(float x) {
  if (x != x) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(x + 0.f);           // -0 + 0 = +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int SELECT_BINS = 2048;

// The `want`-th largest of the n keys (1 <= want <= n): keys above `key` are in, and of those equal to it the first `ties`.
struct Threshold {
  uint32_t key;
  int ties;
};

// Three rounds over the keys (11, 11 and 10 bits from the top): a histogram of the keys that agree with the digits found so far, then the bin
// in which the count from above reaches `want`. Counts are whole numbers, so the result does not depend on the order of the atomics. `hist` holds
// SELECT_BINS + 64 ints of shared memory; all THREADS threads call it, and the keys are written before it (it begins with a barrier).
template <int THREADS, typename Key>
__device__ Threshold select_threshold(const Key& key, int n, int want, int* hist) {
  constexpr int WARPS = THREADS / 32, PER = SELECT_BINS / THREADS;
  static_assert(SELECT_BINS % THREADS == 0 && WARPS <= 32, "bins are shared out evenly");
  int* totals = hist + SELECT_BINS;            // [32] of the warps, then {bin, left}
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t prefix = 0, mask = 0;
#pragma unroll 1
  for (int round = 0; round < 3; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, width = round == 2 ? 10 : 11;
    for (int i = tid; i < SELECT_BINS; i += THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
      const uint32_t k = key(i);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << width) - 1u)], 1);
    }
    __syncthreads();
    // thread t adds up bins from the top: 2047 - t PER down to 2047 - (t PER + PER - 1)
    int mine[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += mine[j] = hist[SELECT_BINS - 1 - (tid * PER + j)];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) totals[warp] = incl;
    __syncthreads();
    int before = incl - sum;
    for (int w = 0; w < warp; ++w) before += totals[w];
    if (before < want && want <= before + sum) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (before < want && want <= before + mine[j]) {
          totals[32] = SELECT_BINS - 1 - (tid * PER + j);
          totals[33] = want - before;
        }
        before += mine[j];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)totals[32] << shift;
    mask |= ((1u << width) - 1u) << shift;
    want = totals[33];
    // the next round's first barrier stands between these reads and the next writes of `totals`
  }
  return Threshold{prefix, want};
}

// Whether each key is in. Every warp owns a run of the indexes, `seg` long; `eq_before` is the number of keys equal to the threshold in front of this
// warp's run (exclusive sums over warps), so ties go to the lowest index. visit(i, in, before) is called by whole warps: `before` counts the chosen
// keys of the run in front of i.
template <typename Key, typename Visit>
__device__ __forceinline__ void for_each_choice(const Key& key, const Threshold& t, int first, int last, int eq_before, const Visit& visit) {
  const int lane = threadIdx.x & 31;
  const uint32_t below = (1u << lane) - 1u;
  int chosen = 0;
  for (int i0 = first; i0 < last; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t k = i < last ? key(i) : 0u;
    const uint32_t gt = __ballot_sync(0xffffffffu, i < last && k > t.key), eq = __ballot_sync(0xffffffffu, i < last && k == t.key);
    const bool is_eq = (eq >> lane) & 1u;
    const bool in = ((gt >> lane) & 1u) || (is_eq && eq_before + __popc(eq & below) < t.ties);
    const uint32_t ins = __ballot_sync(0xffffffffu, in);
    if (i < last) visit(i, in, chosen + __popc(ins & below));
    chosen += __popc(ins);
    eq_before += __popc(eq);
  }
}

// Exclusive sum of `v` (one value of each warp, given by all its lanes) over the warps in front; `slot` holds 32 ints. Begins and ends with a barrier.
template <int THREADS>
__device__ __forceinline__ int warps_before(int v, int* slot, int* total = nullptr) {
  const int warp = threadIdx.x >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slot[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w == warp) before = all;
    all += slot[w];
  }
  if (total) *total = all;
  __syncthreads();
  return before;
}

}  // namespace swb
