// Choice of the largest of many 32-bit keys by a team of warps, and where each chosen one stands among the others.
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
constexpr int SELECT_INTS = SELECT_BINS + 64;          // shared memory of a team

// The threads that share a choice: a whole number of warps with consecutive threads, the team's number within its block giving the barrier.
template <int SIZE>
struct Team {
  static constexpr int WARPS = SIZE / 32;
  int rank, id;
  __device__ __forceinline__ explicit Team(int tid) : rank(tid % SIZE), id(tid / SIZE) {}
  __device__ __forceinline__ int lane() const { return rank & 31; }
  __device__ __forceinline__ int warp() const { return rank >> 5; }
  __device__ __forceinline__ void sync() const {
    if constexpr (SIZE == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "n"(SIZE) : "memory");
  }
};

// The `want`-th largest of the n keys (1 <= want <= n): keys above `key` are in, and of those equal to it the first `ties`.
struct Threshold {
  uint32_t key;
  int ties;
};

// Three rounds over the keys (11, 11 and 10 bits from the top): a histogram of the keys that agree with the digits found so far, then the bin
// in which the count from above reaches `want`. Counts are whole numbers, so the result does not depend on the order of the atomics. The first digit is
// a sign, an exponent and two bits more: numbers of one spread fall into some twenty bins, so that few lanes of a warp meet in one. `hist` holds SELECT_INTS ints
// of shared memory of 16-byte alignment; the whole team calls it (it begins with a barrier, behind which the keys are read).
template <int SIZE, typename Key>
__device__ Threshold select_threshold(const Team<SIZE>& team, const Key& key, int n, int want, int* hist) {
  constexpr int PER = SELECT_BINS / SIZE;
  static_assert(SELECT_BINS % SIZE == 0 && PER >= 2 && SIZE <= 1024, "bins are shared out evenly");
  int* totals = hist + SELECT_BINS;            // [32] of the warps, then {bin, left}
  const int lane = team.lane();
  uint32_t prefix = 0, mask = 0;
#pragma unroll 1
  for (int round = 0; round < 3; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, width = round == 2 ? 10 : 11;
    for (int i = team.rank; i < SELECT_BINS / 4; i += SIZE) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
    team.sync();
    for (int i = team.rank; i < n; i += SIZE) {
      const uint32_t k = key(i);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << width) - 1u)], 1);
    }
    team.sync();
    // the thread of rank r holds the r-th run of PER bins from the top
    const int* run = hist + SELECT_BINS - (team.rank + 1) * PER;
    int mine[PER], sum = 0;
    if constexpr (PER % 4 == 0) {
#pragma unroll
      for (int j = 0; j < PER; j += 4) *reinterpret_cast<int4*>(mine + j) = *reinterpret_cast<const int4*>(run + j);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) mine[j] = run[j];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += mine[j];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) totals[team.warp()] = incl;
    team.sync();
    int before = incl - sum;
    for (int w = 0; w < team.warp(); ++w) before += totals[w];
    if (before < want && want <= before + sum) {
#pragma unroll
      for (int j = PER - 1; j >= 0; --j) {
        if (before < want && want <= before + mine[j]) {
          totals[32] = SELECT_BINS - (team.rank + 1) * PER + j;
          totals[33] = want - before;
        }
        before += mine[j];
      }
    }
    team.sync();
    prefix |= (uint32_t)totals[32] << shift;
    mask |= ((1u << width) - 1u) << shift;
    want = totals[33];
    // the next round's first barrier stands between these reads and the next writes of `totals`
  }
  return Threshold{prefix, want};
}

// The keys first..last - 1 of one warp's run, 32 neighbours at a time, by whole warps: visit(i, in, ins) with whether key i is chosen and the lanes whose keys are
// (i may lie behind the run: then it is not). eq_before: keys equal to the threshold in front of the run, so ties go to the lowest index.
template <typename Key, typename Visit>
__device__ __forceinline__ void for_each_choice(const Key& key, const Threshold& t, int first, int last, int eq_before, const Visit& visit) {
  const int lane = threadIdx.x & 31;
  const uint32_t below = (1u << lane) - 1u;
  for (int i0 = first; i0 < last; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t k = i < last ? key(i) : 0u;
    const uint32_t eq = __ballot_sync(0xffffffffu, i < last && k == t.key);
    const bool in = i < last && (k > t.key || (k == t.key && eq_before + __popc(eq & below) < t.ties));
    visit(i, in, __ballot_sync(0xffffffffu, in));
    eq_before += __popc(eq);
  }
}

// Exclusive sum of `v` (one value of each warp, given by all its lanes) over the team's warps in front; `slot` holds 32 ints. Begins and ends with a barrier.
template <int SIZE>
__device__ __forceinline__ int warps_before(const Team<SIZE>& team, int v, int* slot, int* total = nullptr) {
  team.sync();
  if (team.lane() == 0) slot[team.warp()] = v;
  team.sync();
  int before = 0, all = 0;
  for (int w = 0; w < Team<SIZE>::WARPS; ++w) {
    if (w == team.warp()) before = all;
    all += slot[w];
  }
  if (total) *total = all;
  team.sync();
  return before;
}

}  // namespace swb
