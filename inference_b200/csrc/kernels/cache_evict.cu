// Eviction from a paged cache by accumulated attention weight.
//
// Of a sequence's L cached tokens each key/value head keeps `keep`: those whose position is below `first` or among the last `recent`, and of the others the ones
// of largest weight (ties: the lowest index). Kept entries behind index `keep` move, in order, into the holes that the others leave in front of it, so
// sources and targets never meet and the copies run in any order. Attention does not depend on the order of its keys; what an entry's position
// was is recorded from then on (entries without a record stand in order in front of the next position).
#include "common.cuh"
#include "radix_select.cuh"

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
  int* moves;                // per (sequence, head): count, then holes [max_moves], then sources [max_moves]
  int max_moves;
};

constexpr int EVICT_THREADS = 512;
constexpr int EVICT_CACHED = 40960;            // keys held in shared memory; longer rows are read again in every pass

__device__ __forceinline__ int entry_position(const int* pos, int i, int len, int next) {
  const int x = pos[i];
  return x >= 0 ? x : next - (len - i);
}

__global__ void __launch_bounds__(EVICT_THREADS, 2) evict_plan_kernel(const EvictParams p) {
  pdl_launch_dependents();
  extern __shared__ uint32_t evict_keys[];
  __shared__ __align__(16) int hist[SELECT_INTS];
  const Team<EVICT_THREADS> team(threadIdx.x);
  const int h = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const int len = min(p.kv_lens[seq], min(p.max_blocks * p.bs, p.capacity)), keep = p.keep;
  int* moves = p.moves + ((size_t)seq * p.Hkv + h) * (1 + 2 * (size_t)p.max_moves);
  if (h == 0 && tid == 0) p.new_lens[seq] = min(p.kv_lens[seq], keep);
  if (len <= keep) {
    if (tid == 0) moves[0] = 0;
    return;
  }
  float* w = p.weights + seq * p.w_seq + h * p.w_head;
  int* pos = p.positions + seq * p.p_seq + h * p.p_head;
  const int next = p.next[seq];
  const auto fresh_key = [&](int i) -> uint32_t {
    const int at = entry_position(pos, i, len, next);
    return at < p.first || at >= next - p.recent ? 0xffffffffu : float_key(w[i]);
  };
  const bool cached = len <= EVICT_CACHED;
  clear_bins(team, hist);
  __syncthreads();
  for (int i = tid; i < len; i += EVICT_THREADS) {
    const uint32_t k = fresh_key(i);
    if (cached) evict_keys[i] = k;
    count_key(hist, k);
  }
  const auto key = [&](int i) -> uint32_t { return cached ? evict_keys[i] : fresh_key(i); };
  __syncthreads();
  const Threshold th = select_threshold(team, key, len, keep, hist);
  // Every warp has a run of the entries in front of `keep` and one of those behind. What is kept in front of a run follows from the keys above and equal
  // to the threshold there, and holes are what is not kept in front of `keep`, sources what is kept behind.
  const auto run = [&](int n) { return ((n + EVICT_THREADS - 1) / EVICT_THREADS) * 32; };
  const int lo_a = min(warp * run(keep), keep), hi_a = min(lo_a + run(keep), keep);
  const int lo_b = min(keep + warp * run(len - keep), len), hi_b = min(lo_b + run(len - keep), len);
  const PairSums a = sum_over_warps(team, count_run(key, th, lo_a, hi_a), reinterpret_cast<int2*>(hist));
  const PairSums b = sum_over_warps(team, count_run(key, th, lo_b, hi_b), reinterpret_cast<int2*>(hist) + 32);
  const int kept_a = a.all.x + min(a.all.y, th.ties), total = keep - kept_a;
  int hole_at = lo_a - (a.before.x + min(a.before.y, th.ties));
  for_each_choice(key, th, lo_a, hi_a, a.before.y, [&](int i, bool in, uint32_t) {
    const bool hole = i < hi_a && !in;
    const uint32_t holes = __ballot_sync(0xffffffffu, hole);
    if (hole) moves[1 + hole_at + __popc(holes & ((1u << lane) - 1u))] = i;
    hole_at += __popc(holes);
  });
  int source_at = a.all.x + b.before.x + min(a.all.y + b.before.y, th.ties) - kept_a;
  for_each_choice(key, th, lo_b, hi_b, a.all.y + b.before.y, [&](int i, bool in, uint32_t ins) {
    if (in) moves[1 + p.max_moves + source_at + __popc(ins & ((1u << lane) - 1u))] = i;
    source_at += __popc(ins);
  });
  if (tid == 0) moves[0] = total;
  __syncthreads();
  // weights and positions: records for what stays, then the moves, then the tail is cleared
  for (int i = tid; i < keep; i += EVICT_THREADS)
    if (pos[i] < 0) pos[i] = next - (len - i);
  __syncthreads();
  for (int m = tid; m < total; m += EVICT_THREADS) {
    const int hole = moves[1 + m], from = moves[1 + p.max_moves + m];
    w[hole] = w[from];
    pos[hole] = entry_position(pos, from, len, next);
  }
  __syncthreads();
  for (int i = keep + tid; i < len; i += EVICT_THREADS) w[i] = 0.f;
  for (int i = keep + tid; i < p.capacity; i += EVICT_THREADS) pos[i] = -1;
}

constexpr int MOVE_WARPS = 8;

// A warp per entry: its key row, then its value row, in words of type W.
template <typename W>
__global__ void __launch_bounds__(MOVE_WARPS * 32) evict_move_kernel(const EvictParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, seq = blockIdx.z, lane = threadIdx.x & 31;
  const int* moves = p.moves + ((size_t)seq * p.Hkv + h) * (1 + 2 * (size_t)p.max_moves);
  const int m = blockIdx.x * MOVE_WARPS + (threadIdx.x >> 5);
  if (m >= moves[0]) return;
  const int hole = moves[1 + m], from = moves[1 + p.max_moves + m];
  const int* table = p.table + seq * p.table_stride;
  const int to_block = table[hole / p.bs], from_block = table[from / p.bs];
  if ((unsigned)to_block >= (unsigned)p.num_blocks || (unsigned)from_block >= (unsigned)p.num_blocks) return;
  const size_t to = ((size_t)to_block * p.Hkv + h) * p.bs + hole % p.bs, fr = ((size_t)from_block * p.Hkv + h) * p.bs + from % p.bs;
  const auto copy = [&](char* base, int bytes) {
    const W* src = reinterpret_cast<const W*>(base + fr * bytes);
    W* dst = reinterpret_cast<W*>(base + to * bytes);
    for (int i = lane; i < bytes / (int)sizeof(W); i += 32) dst[i] = src[i];
  };
  copy(p.k, p.k_bytes);
  copy(p.v, p.v_bytes);
}

}  // namespace
}  // namespace swb

extern "C" {

// Ints of the list of moves: per (sequence, head) a count and two indexes for each of the entries that can move.
long long swb_evict_moves(int num_seqs, int Hkv, int capacity, int keep) {
  const long long most = capacity > keep ? (capacity - keep < keep ? capacity - keep : keep) : 0;
  return (long long)num_seqs * Hkv * (1 + 2 * most);
}

// See EvictParams. dims: host int[11] = num_seqs, Hkv, table width, blocks, block_size, k row bytes, v row bytes, capacity, keep, recent, first;
// strides: host long long[4] = weights sequence and head, positions sequence and head. moves: swb_evict_moves ints.
int swb_evict(const int* dims, const long long* strides, void* k, void* v, const int* table, long long table_stride, const int* kv_lens, int* new_lens, const int* next,
              float* weights, int* positions, int* moves, void* stream) {
  using namespace swb;
  const int seqs = dims[0], Hkv = dims[1], max_blocks = dims[2], blocks = dims[3], bs = dims[4], kb = dims[5], vb = dims[6], capacity = dims[7];
  const int keep = dims[8], recent = dims[9], first = dims[10];
  if (seqs <= 0) return 0;
  if (seqs > 65535 || Hkv < 1 || Hkv > 65535 || bs < 1 || kb < 2 || vb < 2 || ((kb | vb) & 1) || keep < 1 || recent < 0 || first < 0 || first > keep - recent || blocks < 1 ||
      max_blocks < 1 || !k || !v || !table || !kv_lens || !new_lens || !next || !weights || !positions || !moves)
    return -3;
  const int most = capacity > keep ? (capacity - keep < keep ? capacity - keep : keep) : 0;
  const EvictParams p{reinterpret_cast<char*>(k), reinterpret_cast<char*>(v), kb, vb, table, table_stride, max_blocks, blocks, bs, Hkv, kv_lens, new_lens, next, weights,
                      strides[0], strides[1], positions, strides[2], strides[3], capacity, keep, recent, first, moves, most};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const size_t smem = 4 * (size_t)(capacity < EVICT_CACHED ? capacity : EVICT_CACHED);
  if (smem > 32 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(evict_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -(int)e;
  }
  int rc = launch_kernel(evict_plan_kernel, dim3(Hkv, seqs), dim3(EVICT_THREADS), smem, s, p);
  if (rc || most == 0) return rc;
  const dim3 grid((most + MOVE_WARPS - 1) / MOVE_WARPS, Hkv, seqs), block(MOVE_WARPS * 32);
  const bool wide = ((kb | vb) & 15) == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  return wide ? launch_kernel(evict_move_kernel<uint4>, grid, block, 0, s, p) : launch_kernel(evict_move_kernel<uint16_t>, grid, block, 0, s, p);
}

}  // extern "C"
