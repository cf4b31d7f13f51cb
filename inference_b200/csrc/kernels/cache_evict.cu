// Eviction from a paged cache by accumulated attention weight.
//
// Of a sequence's L cached tokens each key/value head keeps `keep`: those whose position is below `first` or among the last `recent`, and of the others the ones
// of largest weight (ties: the lowest index). Kept entries behind index `keep` move, in order, into the holes that the others leave in front of it, so
// sources and targets never meet and the copies run in any order. Attention does not depend on the order of its keys; what an entry's position
// was is recorded from then on (entries without a record stand in order in front of the next position).
#include "common.cuh"
#include "radix_select.cuh"

#include <climits>

namespace swb {
namespace {

struct EvictParams {
  char* k;                   // [blocks, Hkv, bs, k_bytes]
  char* v;
  int k_bytes, v_bytes;      // of a row
  const int* table;
  long long table_stride;
  int max_blocks, num_blocks, bs, Hkv;
  const int* kv_lens;
  int* new_lens;
  const int* next;           // position of each sequence's next token
  float* weights;            // [num_seqs, Hkv, .], inner stride 1
  long long w_seq, w_head;
  int* positions;
  long long p_seq, p_head;
  int capacity;              // entries of a row of weights and positions
  int keep, recent, first;
  int* moves;                // per (sequence, head): holes [max_moves], then sources [max_moves]
  int max_moves;
};

constexpr int EVICT_THREADS = 512, EVICT_WARPS = EVICT_THREADS / 32, EVICT_CLUSTER = 8;
constexpr int EVICT_CACHED = 16384;            // keys that a block holds in shared memory; with more it computes them again in every pass
constexpr int EVICT_LISTED = 1024;             // keys in the border's bin that one block can take apart alone

__device__ __forceinline__ int entry_position(const int* pos, int i, int len, int next) {
  const int x = pos[i];
  return x >= 0 ? x : next - (len - i);
}

// Shared memory of the cluster's first block, or of another one.
__device__ __forceinline__ uint32_t in_block(const void* at, int rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(at)), "r"(rank));
  return remote;
}
__device__ __forceinline__ int load_from(const int* at, int rank) {
  int x;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(in_block(at, rank)) : "memory");
  return x;
}
__device__ __forceinline__ void store_to(const void* at, int rank, uint32_t x) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(in_block(at, rank)), "r"(x) : "memory");
}
__device__ __forceinline__ int4 load4_from(const int* at, int rank) {
  int4 x;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(in_block(at, rank)) : "memory");
  return x;
}
__device__ __forceinline__ int add_to(const int* at, int rank, int x) {
  int old;
  asm volatile("atom.shared::cluster.add.s32 %0, [%1], %2;" : "=r"(old) : "r"(in_block(at, rank)), "r"(x) : "memory");
  return old;
}

// `blocks` blocks, a cluster, share a (sequence, head): each has an equal run of the entries in front of `keep` and one of those behind. The first one's histogram
// takes the others' in, and it finds the threshold for all; what is kept in front of a run follows from the keys above and equal to the threshold
// there, so every block knows the places of its holes (not kept, in front of `keep`) and sources (kept, behind it) in the list of moves. The moves are
// then shared out evenly. Counts are whole numbers: nothing depends on the order of the atomics.
// What bounds it is the chain of steps that wait for one another (16 384 keys fit a block, so a pass over them is short): 64 sequences of up to 4608 keys to 4096, 8
// heads, of which a quarter has anything to lose: 30 us, a third of them for the moves (4 TB/s while they last, of rows of 256 bytes in random places); 2 sequences of
// 30 000 keys to 4000 with 8 blocks a head: 36 us. Two launches, a plan by one block a head and moves by many, took 56 and 93 us.
template <typename W>
__global__ void __launch_bounds__(EVICT_THREADS, 2) evict_kernel(const EvictParams p, int blocks) {
  pdl_launch_dependents();
  extern __shared__ uint32_t evict_keys[];
  __shared__ __align__(16) int hist[SELECT_INTS];
  __shared__ uint32_t s_list[EVICT_LISTED];
  __shared__ int s_listed, s_count[4];         // length of the list; keys above and equal to the threshold, in front of and behind `keep`
  const Team<EVICT_THREADS> team(threadIdx.x);
  const int rank = blockIdx.x % blocks, h = blockIdx.x / blocks, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t below = (1u << lane) - 1u;
  int* totals = hist + SELECT_BINS;
  const auto meet = [&]() {
    if (blocks > 1) {
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
      __syncthreads();
    }
  };
  clear_bins(team, hist);
  pdl_wait();
  const int len = min(p.kv_lens[seq], min(p.max_blocks * p.bs, p.capacity)), keep = p.keep;
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[seq] = min(p.kv_lens[seq], keep);
  if (len <= keep) return;                     // the whole cluster
  int* moves = p.moves + ((size_t)seq * p.Hkv + h) * 2 * (size_t)p.max_moves;      // holes, then sources
  float* w = p.weights + seq * p.w_seq + h * p.w_head;
  int* pos = p.positions + seq * p.p_seq + h * p.p_head;
  const int next = p.next[seq];
  const auto cut = [&](int n, int r) { return (int)((long long)n * r / blocks); };
  const int a0 = cut(keep, rank), na = cut(keep, rank + 1) - a0, b0 = keep + cut(len - keep, rank), nb = keep + cut(len - keep, rank + 1) - b0;
  const auto entry = [&](int i) { return i < na ? a0 + i : b0 + i - na; };          // of this block's i-th key
  const auto fresh_key = [&](int i) -> uint32_t {
    const int e = entry(i), at = entry_position(pos, e, len, next);
    return at < p.first || at >= next - p.recent ? 0xffffffffu : float_key(w[e]);
  };
  const bool cached = na + nb <= EVICT_CACHED;
  const auto key = [&](int i) -> uint32_t { return cached ? evict_keys[i] : fresh_key(i); };
  // histograms of `digit` of the keys that agree with prefix under mask, gathered in the first block; bin and rest in its totals
  const auto find = [&](uint32_t prefix, uint32_t mask, int shift, uint32_t digit, int want) {
#pragma unroll 8
    for (int i = tid; i < na + nb; i += EVICT_THREADS) {
      const uint32_t k = mask ? key(i) : fresh_key(i);
      if (!mask && cached) evict_keys[i] = k;
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digit], 1);
    }
    meet();
    if (rank == 0 && blocks > 1) {             // four bins to a thread, of all blocks at once
      static_assert(SELECT_BINS == 4 * EVICT_THREADS, "bins are shared out evenly");
      int4 x[EVICT_CLUSTER];
#pragma unroll
      for (int r = 1; r < EVICT_CLUSTER; ++r) x[r] = r < blocks ? load4_from(hist + tid * 4, r) : make_int4(0, 0, 0, 0);
      int4 sum = reinterpret_cast<int4*>(hist)[tid];
#pragma unroll
      for (int r = 1; r < EVICT_CLUSTER; ++r) sum.x += x[r].x, sum.y += x[r].y, sum.z += x[r].z, sum.w += x[r].w;
      reinterpret_cast<int4*>(hist)[tid] = sum;
      __syncthreads();
    }
    if (rank == 0) find_bin(team, hist, want, totals);
    meet();
  };
  meet();                                      // all blocks run and their bins are clear
  find(0u, 0u, 21, 0x7ffu, keep);
  uint32_t prefix = (uint32_t)load_from(&totals[32], 0), mask = 0x7ffu;
  int want = load_from(&totals[33], 0);
  const int m = load_from(&totals[34], 0);
  Threshold th;
  if (m <= EVICT_LISTED) {
    // Every block gathers its own and asks for room in the first one's list once (an addition to another block's memory with an answer takes some 100 cycles,
    // one behind the other). The first block then chooses by the other 21 bits.
    if (tid == 0) s_listed = 0;
    meet();                                    // everybody has read the totals
#pragma unroll 4
    for (int i = tid; i < na + nb; i += EVICT_THREADS) {
      const uint32_t k = key(i);
      if ((k >> 21) == prefix) s_list[atomicAdd(&s_listed, 1)] = k;
    }
    if (rank == 0) clear_bins(team, hist);
    meet();                                    // the first block's list has its own keys and their number
    if (rank > 0) {
      const int own = s_listed;
      __syncthreads();
      if (tid == 0 && own) s_listed = add_to(&s_listed, 0, own);
      __syncthreads();
      for (int i = tid; i < own; i += EVICT_THREADS) store_to(&s_list[s_listed + i], 0, s_list[i]);
    }
    if (blocks > 1) meet();
    if (rank == 0) {
      const auto rest = [&](int i) { return s_list[i] << 11; };
      for (int i = tid; i < m; i += EVICT_THREADS) count_key(hist, rest(i));
      __syncthreads();
      const Threshold t = select_threshold(team, rest, m, want, hist);
      if (tid == 0) totals[39] = (int)(prefix << 21 | t.key >> 11), totals[40] = t.ties;
    }
    meet();
    th = Threshold{(uint32_t)load_from(&totals[39], 0), load_from(&totals[40], 0)};
  } else {
    prefix <<= 21, mask <<= 21;
#pragma unroll 1
    for (int round = 0; round < 2; ++round) {
      const int shift = round == 0 ? 10 : 0;
      const uint32_t digit = round == 0 ? 0x7ffu : 0x3ffu;
      meet();                                  // everybody has read the totals
      clear_bins(team, hist);
      meet();
      find(prefix, mask, shift, digit, want);
      prefix |= (uint32_t)load_from(&totals[32], 0) << shift;
      mask |= digit << shift;
      want = load_from(&totals[33], 0);
    }
    th = Threshold{prefix, want};
  }
  // runs of this block's warps, and what lies in front of them
  const auto run = [&](int n) { return ((n + EVICT_THREADS - 1) / EVICT_THREADS) * 32; };
  const int lo_a = min(warp * run(na), na), hi_a = min(lo_a + run(na), na), lo_b = na + min(warp * run(nb), nb), hi_b = min(lo_b + run(nb), na + nb);
  meet();                                      // the totals are read: their neighbours are written again
  int2* slots = reinterpret_cast<int2*>(hist);
  const PairSums a = sum_over_warps(team, count_run(key, th, lo_a, hi_a), slots);
  const PairSums b = sum_over_warps(team, count_run(key, th, lo_b, hi_b), slots + 32);
  if (tid == 0) s_count[0] = a.all.x, s_count[1] = a.all.y, s_count[2] = b.all.x, s_count[3] = b.all.y;
  meet();
  // lane r has block r's counts
  int4 mine = make_int4(0, 0, 0, 0);
  if (lane < blocks) mine = make_int4(load_from(&s_count[0], lane), load_from(&s_count[1], lane), load_from(&s_count[2], lane), load_from(&s_count[3], lane));
  const auto all_of = [&](int x) { return __reduce_add_sync(0xffffffffu, x); };
  const auto before = [&](int x) { return __reduce_add_sync(0xffffffffu, lane < rank ? x : 0); };
  const int all_above = all_of(mine.x), all_same = all_of(mine.y);
  const int above_a = a.before.x + before(mine.x), same_a = a.before.y + before(mine.y), above_b = b.before.x + before(mine.z), same_b = b.before.y + before(mine.w);
  const int kept_a = all_above + min(all_same, th.ties), total = keep - kept_a;
  int hole_at = a0 + lo_a - (above_a + min(same_a, th.ties));
  for_each_choice(key, th, lo_a, hi_a, same_a, [&](int i, bool in, uint32_t) {
    const bool hole = i < hi_a && !in;
    const uint32_t holes = __ballot_sync(0xffffffffu, hole);
    if (hole) moves[hole_at + __popc(holes & below)] = entry(i);
    hole_at += __popc(holes);
  });
  int source_at = all_above + above_b + min(all_same + same_b, th.ties) - kept_a;
  for_each_choice(key, th, lo_b, hi_b, all_same + same_b, [&](int i, bool in, uint32_t ins) {
    if (in) moves[p.max_moves + source_at + __popc(ins & below)] = entry(i);
    source_at += __popc(ins);
  });
  __syncthreads();                             // no key of this block is computed any more
  for (int i = tid; i < na; i += EVICT_THREADS)          // what stays has a record from now on
    if (pos[a0 + i] < 0) pos[a0 + i] = next - (len - (a0 + i));
  meet();                                      // the list is complete

  // Up to 32 moves to a warp: its lanes look one up each, all at once, then it copies their rows, eight moves on their way together.
  const int* table = p.table + seq * p.table_stride;
  const int k_words = p.k_bytes / (int)sizeof(W), words = k_words + p.v_bytes / (int)sizeof(W);
  W* kc = reinterpret_cast<W*>(p.k);
  W* vc = reinterpret_cast<W*>(p.v);
  const int stride = EVICT_WARPS * blocks;
  for (int m0 = warp * blocks + rank; m0 < total; m0 += 32 * stride) {
    const int m = m0 + lane * stride, n = min(32, (total - m0 + stride - 1) / stride);
    long long to = -1, from = -1;              // rows, -1: none
    float weight = 0.f;
    int place = 0, target = -1;
    if (m < total) {
      const int hole = moves[m], source = moves[p.max_moves + m];
      const int to_block = table[hole / p.bs], from_block = table[source / p.bs];
      weight = w[source], place = entry_position(pos, source, len, next), target = hole;
      if ((unsigned)to_block < (unsigned)p.num_blocks && (unsigned)from_block < (unsigned)p.num_blocks) {
        to = ((long long)to_block * p.Hkv + h) * p.bs + hole % p.bs;
        from = ((long long)from_block * p.Hkv + h) * p.bs + source % p.bs;
      }
    }
    for (int i0 = 0; i0 < words; i0 += 32) {
      const int i = i0 + lane;
      W* base = i < k_words ? kc + i : vc + (i - k_words);
      const int row = i < k_words ? k_words : words - k_words;
      for (int j0 = 0; j0 < n; j0 += 8) {
        W x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const long long f = __shfl_sync(0xffffffffu, from, j0 + j);
          if (f >= 0 && i < words) x[j] = base[f * row];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const long long t = __shfl_sync(0xffffffffu, to, j0 + j);
          if (t >= 0 && i < words) base[t * row] = x[j];
        }
      }
    }
    if (target >= 0) w[target] = weight, pos[target] = place;
  }
  meet();                                      // what moved is read
  for (int i = b0 + tid; i < b0 + nb; i += EVICT_THREADS) w[i] = 0.f;
  const int c0 = keep + cut(p.capacity - keep, rank), c1 = keep + cut(p.capacity - keep, rank + 1);
  for (int i = c0 + tid; i < c1; i += EVICT_THREADS) pos[i] = -1;
}

}  // namespace
}  // namespace swb

extern "C" {

// See EvictParams. dims: host int[11] = num_seqs, Hkv, table width, blocks, block_size, k row bytes, v row bytes, capacity, keep, recent, first;
// sizes: host long long[5] = strides of weights (sequence and head) and positions, ints that `moves` has room for: two for each of the entries that can move, min(keep,
// capacity - keep), per (sequence, head).
int swb_evict(const int* dims, const long long* sizes, void* k, void* v, const int* table, long long table_stride, const int* kv_lens, int* new_lens, const int* next,
              float* weights, int* positions, int* moves, void* stream) {
  using namespace swb;
  const int seqs = dims[0], Hkv = dims[1], max_blocks = dims[2], blocks = dims[3], bs = dims[4], kb = dims[5], vb = dims[6], capacity = dims[7];
  const int keep = dims[8], recent = dims[9], first = dims[10];
  if (seqs <= 0) return 0;
  const int most = capacity > keep ? (capacity - keep < keep ? capacity - keep : keep) : 0;
  if (seqs > 65535 || Hkv < 1 || Hkv > 65535 || bs < 1 || kb < 2 || vb < 2 || ((kb | vb) & 1) || keep < 1 || recent < 0 || first < 0 || first > keep - recent || blocks < 1 ||
      max_blocks < 1 || (long long)max_blocks * bs > INT_MAX || !k || !v || !table || !kv_lens || !new_lens || !next || !weights || !positions || (most && !moves) || sizes[4] < 2ll * seqs * Hkv * most)
    return -3;
  const EvictParams p{reinterpret_cast<char*>(k), reinterpret_cast<char*>(v), kb, vb, table, table_stride, max_blocks, blocks, bs, Hkv, kv_lens, new_lens, next, weights,
                      sizes[0], sizes[1], positions, sizes[2], sizes[3], capacity, keep, recent, first, moves, most};
  // a block for every 2048 entries where that fills the chip no further than one round (with up to four rounds, 64 sequences take as long)
  int share = 1;
  while (share < EVICT_CLUSTER && share * 2048 < capacity && (long long)share * 2 * Hkv * seqs <= 2 * 148) share *= 2;
  const int cached = capacity / share + 2;
  const size_t smem = 4 * (size_t)(cached < EVICT_CACHED ? cached : EVICT_CACHED);
  const bool wide = ((kb | vb) & 15) == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  auto kernel = wide ? evict_kernel<uint4> : evict_kernel<uint16_t>;
  if (smem > 32 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -(int)e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(Hkv * share, seqs), cfg.blockDim = dim3(EVICT_THREADS), cfg.dynamicSmemBytes = smem, cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = share, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, share);
  return e == cudaSuccess ? 0 : -(int)e;
}

}  // extern "C"
