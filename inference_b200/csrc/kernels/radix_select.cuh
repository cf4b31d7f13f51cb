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

// The `want`-th largest of n keys (1 <= want <= n): keys above `key` are in, and of those equal to it the first `ties`.
struct Threshold {
  uint32_t key;
  int ties;
};

// Histogram of the first digit, 11 bits from the top: a sign, an exponent and two bits more, so numbers of one spread fall into some twenty bins and few lanes
// of a warp meet in one. The caller clears the bins, adds every key once, and puts the team's barrier behind each of both. `hist`: SELECT_INTS ints of shared
// memory with 16-byte alignment.
template <int SIZE>
__device__ __forceinline__ void clear_bins(const Team<SIZE>& team, int* hist) {
  for (int i = team.rank; i < SELECT_BINS / 4; i += SIZE) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
}
__device__ __forceinline__ void count_key(int* hist, uint32_t key) { atomicAdd(&hist[key >> 21], 1); }

// The bin in which the count from the top reaches `want`, in totals[32..]: {bin, what is left to find in it, its count, 0, 0}. Ends with a barrier.
template <int SIZE>
__device__ __forceinline__ void find_bin(const Team<SIZE>& team, const int* hist, int want, int* totals) {
  constexpr int PER = SELECT_BINS / SIZE;
  static_assert(SELECT_BINS % SIZE == 0 && PER >= 2 && PER <= 32, "bins are shared out evenly, a thread's among a warp");
  // the thread of rank r adds up the r-th run of PER bins from the top, from a place of its own on so that neighbours meet in no bank
  const int* run = hist + SELECT_BINS - (team.rank + 1) * PER;
  int sum = 0;
  if constexpr (PER % 4 == 0) {
#pragma unroll
    for (int j = 0; j < PER / 4; ++j) {
      const int4 x = reinterpret_cast<const int4*>(run)[(j + team.lane() * PER / 32) & (PER / 4 - 1)];
      sum += (x.x + x.y) + (x.z + x.w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += run[j];
  }
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (team.lane() >= o) incl += v;
  }
  if (team.lane() == 31) totals[team.warp()] = incl;
  team.sync();
  int before = incl - sum;
  for (int w = 0; w < team.warp(); ++w) before += totals[w];
  // one thread's run holds the place: its warp looks at the bins, a lane each, or it does so itself where they are few
  const bool here = before < want && want <= before + sum;
  if constexpr (PER >= 16) {
    const uint32_t owner = __ballot_sync(0xffffffffu, here);
    if (owner) {
      const int lane = __ffs(owner) - 1, start = __shfl_sync(0xffffffffu, before, lane);
      const int bin = SELECT_BINS - (team.warp() * 32 + lane) * PER - 1 - team.lane();
      const int mine = team.lane() < PER ? hist[bin] : 0;
      int to = mine;
#pragma unroll
      for (int o = 1; o < PER; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, to, o);
        if (team.lane() >= o) to += v;
      }
      if (team.lane() < PER && start + to - mine < want && want <= start + to)
        totals[32] = bin, totals[33] = want - start - to + mine, totals[34] = mine, totals[35] = totals[36] = 0;
    }
  } else if (here) {
    for (int j = PER - 1; j >= 0; --j) {
      const int mine = run[j];
      if (before < want && want <= before + mine)
        totals[32] = SELECT_BINS - (team.rank + 1) * PER + j, totals[33] = want - before, totals[34] = mine, totals[35] = totals[36] = 0;
      before += mine;
    }
  }
  team.sync();
}

// From the first digit's histogram on. A bin with no more keys than the team has threads is gathered and every thread counts what lies above its key; a fuller
// one is taken apart by its other 21 bits. Counts are whole numbers, so the result does not depend on the order of the atomics. The bins' memory is
// free afterwards (behind a barrier of the team).
template <int SIZE, typename Key>
__device__ Threshold select_threshold(const Team<SIZE>& team, const Key& key, int n, int want, int* hist) {
  int* totals = hist + SELECT_BINS;            // [32] of the warps, find_bin's five, {key, ties}
  find_bin(team, hist, want, totals);
  const uint32_t bin = (uint32_t)totals[32];
  const int left = totals[33], m = totals[34];
  if (m <= SIZE) {
    uint32_t* list = reinterpret_cast<uint32_t*>(hist);
#pragma unroll 4
    for (int i = team.rank; i < n; i += SIZE) {
      const uint32_t k = key(i);
      if ((k >> 21) == bin) list[atomicAdd(&totals[35], 1)] = k;
    }
    team.sync();
    if (team.rank < m) {
      const uint32_t mine = list[team.rank];
      int above = 0, same = 0;
      for (int j = 0; j < m; ++j) above += list[j] > mine, same += list[j] == mine;
      if (above < left && left <= above + same) totals[37] = (int)mine, totals[38] = left - above;      // one key fits: its owners write the same
    }
    team.sync();
    return Threshold{(uint32_t)totals[37], totals[38]};
  }
  uint32_t prefix = bin << 21, mask = 0x7ffu << 21;
  want = left;
#pragma unroll 1
  for (int round = 0; round < 2; ++round) {
    const int shift = round == 0 ? 10 : 0;
    const uint32_t digit = round == 0 ? 0x7ffu : 0x3ffu;
    clear_bins(team, hist);                    // every thread is past its reads of the bins: find_bin ended with a barrier
    team.sync();
    for (int i = team.rank; i < n; i += SIZE) {
      const uint32_t k = key(i);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digit], 1);
    }
    team.sync();
    find_bin(team, hist, want, totals);
    prefix |= (uint32_t)totals[32] << shift;
    mask |= digit << shift;
    want = totals[33];
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

// Exclusive sums of `v` (one pair of each warp, given by all its lanes) over the team's warps in front, and those of all. `slot` holds 32 pairs that nobody reads or
// writes around the call; a barrier stands within.
struct PairSums {
  int2 before, all;
};
template <int SIZE>
__device__ __forceinline__ PairSums sum_over_warps(const Team<SIZE>& team, int2 v, int2* slot) {
  if (team.lane() == 0) slot[team.warp()] = v;
  team.sync();
  PairSums s{make_int2(0, 0), make_int2(0, 0)};
  for (int w = 0; w < Team<SIZE>::WARPS; ++w) {
    if (w == team.warp()) s.before = s.all;
    const int2 x = slot[w];
    s.all.x += x.x, s.all.y += x.y;
  }
  return s;
}

// How many keys of a warp's run lie above the threshold, and how many are equal to it.
template <typename Key>
__device__ __forceinline__ int2 count_run(const Key& key, const Threshold& t, int first, int last) {
  int above = 0, same = 0;
#pragma unroll 4
  for (int i = first + (int)(threadIdx.x & 31); i < last; i += 32) {
    const uint32_t k = key(i);
    above += k > t.key, same += k == t.key;
  }
  return make_int2(__reduce_add_sync(0xffffffffu, above), __reduce_add_sync(0xffffffffu, same));
}

// A first digit of float_keys in proportion to the numbers between zero and the largest, for choices of few among many of one spread: a bin at the choice's border
// holds a thousandth of them where one of exponent and two bits holds a tenth. Numbers below zero fall into the lowest bin. Where the largest is not a positive
// finite number that can be divided by, the key's own digits serve.
struct LinearDigit {
  float scale;                                 // 0: the key's own digits
  __device__ __forceinline__ explicit LinearDigit(uint32_t largest) {
    const float top = __uint_as_float(largest & 0x7fffffffu);
    scale = (largest & 0x80000000u) && top > 1e-30f && top < INFINITY ? (float)(SELECT_BINS - 1) / top : 0.f;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t key) const {
    if (scale == 0.f) return key >> 21;
    return (key & 0x80000000u) ? min((uint32_t)(__uint_as_float(key & 0x7fffffffu) * scale), (uint32_t)SELECT_BINS - 1u) : 0u;
  }
};

// The indexes of the `want` largest of n keys in ascending order, put(place, index), ties to the lowest index. keys: shared memory of 16-byte alignment, read in fours (up to
// three behind the last are read and not used); largest: the largest of them. Where a team has a thread for each key in the border's bin and for each chosen one, or
// for every other, one pass gathers both and two counts put them into order. The caller clears the bins; the whole team calls it, and the keys are written before it (it begins with a barrier).
template <int SIZE, typename Put>
__device__ __forceinline__ void choose_in_order(const Team<SIZE>& team, const uint32_t* keys, int n, int want, uint32_t largest, int* hist, const Put& put) {
  int* totals = hist + SELECT_BINS;
  const LinearDigit digit(largest);
  const auto each = [&](const auto& visit) {
    for (int i = team.rank * 4; i < n; i += SIZE * 4) {
      const uint4 k = *reinterpret_cast<const uint4*>(keys + i);
      visit(i, k.x);
      if (i + 1 < n) visit(i + 1, k.y);
      if (i + 2 < n) visit(i + 2, k.z);
      if (i + 3 < n) visit(i + 3, k.w);
    }
  };
  team.sync();
  constexpr int MOST = SIZE < 256 ? 2 * SIZE : SIZE;      // of few threads each puts two in order (with 256 that costs registers, and 8 % of 64 sequences' selections)
  if (want <= MOST) {
    each([&](int, uint32_t k) { atomicAdd(&hist[digit(k)], 1); });
    team.sync();
    find_bin(team, hist, want, totals);
    const uint32_t bin = (uint32_t)totals[32];
    const int left = totals[33], m = totals[34];
    if (m <= SIZE) {
      uint32_t* border = reinterpret_cast<uint32_t*>(hist);      // keys of the border's bin, their indexes, and what is chosen
      int *border_at = hist + SIZE, *chosen = hist + 2 * SIZE;
      each([&](int i, uint32_t k) {
        const uint32_t d = digit(k);
        if (d < bin) return;
        if (d > bin) {
          chosen[atomicAdd(&totals[36], 1)] = i;
        } else {
          const int j = atomicAdd(&totals[35], 1);
          border[j] = k, border_at[j] = i;
        }
      });
      team.sync();
      if (team.rank < m) {
        const uint32_t mine = border[team.rank];
        const int at = border_at[team.rank];
        int above = 0;
#pragma unroll 4
        for (int j = 0; j < m; ++j) above += border[j] > mine || (border[j] == mine && border_at[j] < at);
        if (above < left) chosen[want - left + above] = at;
      }
      team.sync();
#pragma unroll 1
      for (int i = team.rank; i < want; i += SIZE) {
        const int at = chosen[i];
        int place = 0, j = 0;
        for (; j + 4 <= want; j += 4) {
          const int4 x = *reinterpret_cast<const int4*>(chosen + j);
          place += (x.x < at) + (x.y < at) + (x.z < at) + (x.w < at);
        }
        for (; j < want; ++j) place += chosen[j] < at;
        put(place, at);
        if constexpr (MOST == SIZE) break;
      }
      return;
    }
    clear_bins(team, hist);
    team.sync();
  }
  each([&](int, uint32_t k) { count_key(hist, k); });
  team.sync();
  const auto key = [&](int i) { return keys[i]; };
  const Threshold t = select_threshold(team, key, n, want, hist);
  const int seg = ((n + SIZE - 1) / SIZE) * 32, lo = min(team.warp() * seg, n), hi = min(lo + seg, n);
  const PairSums sums = sum_over_warps(team, count_run(key, t, lo, hi), reinterpret_cast<int2*>(hist));
  int at = sums.before.x + min(sums.before.y, t.ties);
  for_each_choice(key, t, lo, hi, sums.before.y, [&](int i, bool in, uint32_t ins) {
    if (in) put(at + __popc(ins & ((1u << team.lane()) - 1u)), i);
    at += __popc(ins);
  });
}

}  // namespace swb
