// What drafted trees and beams do to a paged cache: what a token of a tree sees, the path of a tree that the model agrees with and the moves that close its cache entries up, and
// copies of pages.
//
// Caches are tensors [blocks, ...], one or two a layer, whose pages have one number in all of them: a list of bases and row sizes goes to the kernels by value, so that a
// launch takes every layer and nothing is uploaded in front of it.
#include "common.cuh"
#include "gemm_tcgen05.cuh"

#include <climits>
#include <cstring>

namespace swb {

SWB_REGISTER_STATUS_UNIT(branch_ops);

namespace {

constexpr int MAX_TENSORS = 96, MAX_PAIRS = 256;          // of a launch
constexpr size_t MAX_ARGUMENTS = 32764;                    // bytes that a kernel's arguments may take (CUDA 12.1 and later, from compute capability 7.0 on)

struct Tensors {
  char* base[MAX_TENSORS];
  long long page_bytes[MAX_TENSORS];
  int heads[MAX_TENSORS];                                  // a page is [heads, block_size, row]
  int start[MAX_TENSORS], cols[MAX_TENSORS];               // of the acceptance: columns of the tensors in front of this one, and of one of its rows
  int n;
};

// ---- what a tree's tokens see -----------------------------------------------------------------------------------------------------------------------
// A thread follows its token's parents to the root: they come in descending order, so that each word of the row is finished before the next one is begun.
__global__ void __launch_bounds__(128) plan_tree_kernel(const int* __restrict__ parents, const int* __restrict__ cu_q, int num_seqs, int uniform_q, int tokens, int words, unsigned* mask,
                                                        int* depths) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x * 128 + threadIdx.x;
  if (t >= tokens || (cu_q && (t < cu_q[0] || t >= cu_q[num_seqs]))) return;
  const int seq = seq_of_token(cu_q, num_seqs, uniform_q, t), q0 = cu_q ? cu_q[seq] : seq * uniform_q;
  if (q0 < 0) return;
  unsigned* row = mask + (long long)t * words;
  int i = t - q0, depth = 0, word = words;
  unsigned bits = 0;
  for (;;) {
    const int w = i >> 5;
    if (w < word) {
      if (word < words) row[word] = bits;
      for (int z = min(word, words) - 1; z > w; --z) row[z] = 0;
      word = w, bits = 0;
    }
    if (w < words) bits |= 1u << (i & 31);
    const int up = parents[q0 + i];
    if (up < 0 || up >= i) break;                          // the root, or no token in front of this one
    i = up, ++depth;
  }
  if (word < words) row[word] = bits;
  for (int z = min(word, words) - 1; z >= 0; --z) row[z] = 0;
  depths[t] = depth;
}

// ---- the path that the model agrees with --------------------------------------------------------------------------------------------------------------
struct AcceptParams {
  const long long* picks;
  const long long* tokens;
  const int* parents;
  const int* cu_q;
  const int* kv_lens;
  const int* table;
  long long table_stride;
  int num_seqs, uniform_q, total, max_blocks, num_blocks, bs, width, units;      // units: 16-byte (or smaller) columns of all tensors
  int* path;                 // [num_seqs, width]
  int* counts;
  long long* next;
  int* lens;
};

constexpr int ACCEPT_THREADS = 256, ACCEPT_BLOCKS = 4, MOVES = 8;         // ACCEPT_BLOCKS of them to an SM: 64 registers a thread

struct Move {
  int from_page, from_row, to_page, to_row;                // to_page < 0: nothing to move
};

// Block x of sequence y finds the sequence's path, then each of its threads takes columns of rows of all tensors along the path: entry path[d] goes to d. path[d] >= d and both
// ascend, so that an entry which is written has been read before, by the same thread, and none is read after it was written.
//
// The path: each token asks whether it is its parent's pick, all at once, and a parent keeps the first child that is (a minimum of whole numbers: in any order the same); the walk
// from the root is then one shared read a step. (A warp that looked for each step's child among the tokens waited for memory at every step: 12.2 us for one tree of 25 tokens, 41.7 us
// for 64 trees of 48.) What is left of a small call is the latency of three dependent loads, the walk and one round of moves.
template <typename V>
__global__ void __launch_bounds__(ACCEPT_THREADS, ACCEPT_BLOCKS) accept_tree_kernel(const __grid_constant__ Tensors pages, const AcceptParams p) {
  pdl_launch_dependents();
  __shared__ int s_count;
  __shared__ Move s_move[ACCEPT_THREADS];
  extern __shared__ int s_path[];                          // [width]: first each token's accepted child, then the path
  const int seq = blockIdx.y, tid = threadIdx.x;
  pdl_wait();
  const int q0 = p.cu_q ? p.cu_q[seq] : seq * p.uniform_q, q1 = p.cu_q ? p.cu_q[seq + 1] : q0 + p.uniform_q;
  const int n = q0 < 0 ? 0 : min(min(min(q1, p.total) - q0, p.uniform_q), p.width), len = max(min(p.kv_lens[seq], p.max_blocks * p.bs), 0), base = len - (q1 - q0);
  for (int i = tid; i < n; i += ACCEPT_THREADS) s_path[i] = n;
  __syncthreads();
  for (int i = 1 + tid; i < n; i += ACCEPT_THREADS) {
    const int up = p.parents[q0 + i];
    const long long token = p.tokens[q0 + i];
    if (up >= 0 && up < i && p.picks[q0 + up] == token) atomicMin(s_path + up, i);
  }
  __syncthreads();
  if (tid == 0) {
    int count = 0;
    for (int node = 0; node < n;) {                        // nodes ascend: count <= node, and what stands below node is not read again
      const int next = s_path[node];
      s_path[count++] = node;
      node = next;
    }
    s_count = count;
  }
  __syncthreads();
  const int count = s_count;
  if (blockIdx.x == 0) {
    for (int d = tid; d < p.width; d += ACCEPT_THREADS) p.path[(long long)seq * p.width + d] = d < count ? s_path[d] : -1;
    if (tid == 0) {
      p.counts[seq] = count;
      p.next[seq] = count > 0 ? p.picks[q0 + s_path[count - 1]] : -1;
      p.lens[seq] = max(base + count, 0);
    }
  }
  const int* table = p.table + seq * p.table_stride;
  for (int first = 1; first < count; first += ACCEPT_THREADS) {
    const int d = first + tid;
    Move mine = {0, 0, -1, 0};
    if (d < count && s_path[d] != d && base + d >= 0) {
      const int from = base + s_path[d], to = base + d, block = table[from / p.bs], there = table[to / p.bs];
      if ((unsigned)block < (unsigned)p.num_blocks && (unsigned)there < (unsigned)p.num_blocks) mine = {block, from % p.bs, there, to % p.bs};
    }
    __syncthreads();                                       // the moves before these have been read
    s_move[tid] = mine;
    __syncthreads();
    const int moves = min(count - first, ACCEPT_THREADS);
    for (int u = blockIdx.x * ACCEPT_THREADS + tid; u < p.units; u += gridDim.x * ACCEPT_THREADS) {
      int lo = 0, hi = pages.n;                            // the tensor whose columns u is among
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pages.start[mid] <= u) lo = mid; else hi = mid;
      }
      const int cols = pages.cols[lo], at = u - pages.start[lo], head = at / cols;
      const long long row_bytes = (long long)cols * sizeof(V), page_bytes = pages.page_bytes[lo];
      char* column = pages.base[lo] + head * p.bs * row_bytes + (at - head * cols) * (long long)sizeof(V);
      for (int d0 = 0; d0 < moves; d0 += MOVES) {
        V x[MOVES];
#pragma unroll
        for (int i = 0; i < MOVES; ++i)
          if (d0 + i < moves && s_move[d0 + i].to_page >= 0)
            x[i] = *reinterpret_cast<const V*>(column + s_move[d0 + i].from_page * page_bytes + s_move[d0 + i].from_row * row_bytes);
#pragma unroll
        for (int i = 0; i < MOVES; ++i)
          if (d0 + i < moves && s_move[d0 + i].to_page >= 0)
            *reinterpret_cast<V*>(column + s_move[d0 + i].to_page * page_bytes + s_move[d0 + i].to_row * row_bytes) = x[i];
      }
    }
  }
}

// ---- copies of pages ------------------------------------------------------------------------------------------------------------------------------------
struct Pairs {
  int src[MAX_PAIRS], dst[MAX_PAIRS];
};
static_assert(sizeof(Tensors) + sizeof(Pairs) + 64 <= MAX_ARGUMENTS && sizeof(Tensors) + sizeof(AcceptParams) <= MAX_ARGUMENTS, "arguments of a launch");
constexpr int COPY_THREADS = 256, COPY_UNROLL = 8;

// Block (pair, piece of the page, tensor). from / to: the pairs on the device, where they are not among the arguments.
template <typename V>
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(const __grid_constant__ Tensors pages, const __grid_constant__ Pairs pairs, const int* from, const int* to, int num_blocks,
                                                                  int pieces) {
  pdl_launch_dependents();
  const int pair = blockIdx.x / pieces, piece = blockIdx.x % pieces, t = blockIdx.y;
  pdl_wait();
  const int src = from ? from[pair] : pairs.src[pair], dst = from ? to[pair] : pairs.dst[pair];
  if ((unsigned)src >= (unsigned)num_blocks || (unsigned)dst >= (unsigned)num_blocks || src == dst) return;
  const long long bytes = pages.page_bytes[t], n = bytes / sizeof(V);
  const V* a = reinterpret_cast<const V*>(pages.base[t] + src * bytes);
  V* b = reinterpret_cast<V*>(pages.base[t] + dst * bytes);
  for (long long i0 = (long long)piece * COPY_THREADS * COPY_UNROLL + threadIdx.x; i0 < n; i0 += (long long)pieces * COPY_THREADS * COPY_UNROLL) {
    V x[COPY_UNROLL];
#pragma unroll
    for (int i = 0; i < COPY_UNROLL; ++i)
      if (i0 + i * COPY_THREADS < n) x[i] = a[i0 + i * COPY_THREADS];
#pragma unroll
    for (int i = 0; i < COPY_UNROLL; ++i)
      if (i0 + i * COPY_THREADS < n) b[i0 + i * COPY_THREADS] = x[i];
  }
}

// Tensors first .. first + MAX_TENSORS - 1 of the list; the widest access that all their rows start on. step > 0: tensor i is like the first one and begins i * step behind it.
struct TensorList {
  const long long* base;
  const long long* page_bytes;
  const int* heads;
  int n;
  long long step;
};
Tensors part_of(const TensorList& list, int first) {
  Tensors t;
  t.n = list.n - first < MAX_TENSORS ? list.n - first : MAX_TENSORS;
  for (int i = 0; i < t.n; ++i) {
    const int at = list.step > 0 ? 0 : first + i;
    t.base[i] = reinterpret_cast<char*>(list.base[at]) + (list.step > 0 ? (first + i) * list.step : 0);
    t.page_bytes[i] = list.page_bytes[at];
    t.heads[i] = list.heads ? list.heads[at] : 1;
  }
  return t;
}
int access_bytes(const Tensors& t, int rows_of_page) {
  long long all = 16;
  for (int i = 0; i < t.n; ++i) all |= reinterpret_cast<long long>(t.base[i]) | (t.page_bytes[i] / ((long long)t.heads[i] * rows_of_page));
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
}

template <typename V>
int launch_accept(Tensors& t, AcceptParams p, cudaStream_t s) {
  long long units = 0;
  for (int i = 0; i < t.n; ++i) {
    const long long cols = t.page_bytes[i] / t.heads[i] / p.bs / (long long)sizeof(V);
    if (units + cols * t.heads[i] > INT_MAX / 2) return -3;
    t.start[i] = (int)units, t.cols[i] = (int)cols;
    units += cols * t.heads[i];
  }
  p.units = (int)units;
  // as many columns to a thread as it takes for all blocks to be on the SMs at once: each of them finds the path by itself
  const long long most = (units + ACCEPT_THREADS - 1) / ACCEPT_THREADS, each = (most * p.num_seqs + device_sm_count() * ACCEPT_BLOCKS - 1) / (device_sm_count() * ACCEPT_BLOCKS);
  const unsigned blocks = (unsigned)(units ? (most + each - 1) / each : 1);
  return launch_kernel(accept_tree_kernel<V>, dim3(blocks, p.num_seqs), dim3(ACCEPT_THREADS), (size_t)p.width * 4, s, t, p);
}

template <typename V>
int launch_copy(const Tensors& t, const Pairs& pairs, const int* from, const int* to, int n, int num_blocks, cudaStream_t s) {
  long long most = 0;
  for (int i = 0; i < t.n; ++i) most = t.page_bytes[i] > most ? t.page_bytes[i] : most;
  const long long step = (long long)COPY_THREADS * COPY_UNROLL * sizeof(V);
  long long pieces = (most + step - 1) / step;
  if (pieces > 64) pieces = 64;
  return launch_kernel(copy_pages_kernel<V>, dim3((unsigned)(n * pieces), t.n), dim3(COPY_THREADS), 0, s, t, pairs, from, to, num_blocks, (int)pieces);
}

}  // namespace
}  // namespace swb

extern "C" {

// mask [tokens, words] and depths [tokens] of a step's trees. parents [tokens]: places within the sequence, below the token's own (others: none).
int swb_plan_tree(const int* parents, const int* cu_q, int num_seqs, int uniform_q, int tokens, int words, void* mask, int* depths, void* stream) {
  using namespace swb;
  if (tokens <= 0 || num_seqs <= 0) return 0;
  if (!parents || !mask || !depths || uniform_q < 1 || words < 1 || tokens > INT_MAX - 128) return -3;
  return launch_kernel(plan_tree_kernel, dim3((tokens + 127) / 128), dim3(128), 0, reinterpret_cast<cudaStream_t>(stream), parents, cu_q, num_seqs, uniform_q, tokens, words,
                       reinterpret_cast<unsigned*>(mask), depths);
}

// dims: host int[8] = num_seqs, tokens of each sequence (with cu_q: at most), tokens, table width, blocks, block_size, width of path, tensors. base, page_bytes, heads: host lists
// of the tensors [blocks, heads, block_size, row]; with step > 0 lists of one, all tensors are alike and begin step bytes apart.
int swb_accept_tree(const int* dims, const void* picks, const void* tokens, const int* parents, const long long* base, const long long* page_bytes, const int* heads, long long step, const int* table,
                    long long table_stride, const int* cu_q, const int* kv_lens, int* path, int* counts, void* next, int* lens, void* stream) {
  using namespace swb;
  AcceptParams p = {};
  p.num_seqs = dims[0], p.uniform_q = dims[1], p.total = dims[2], p.max_blocks = dims[3], p.num_blocks = dims[4], p.bs = dims[5], p.width = dims[6];
  const int n = dims[7];
  if (p.num_seqs <= 0) return 0;
  if (p.num_seqs > 65535 || p.uniform_q < 1 || p.total < 0 || p.max_blocks < 1 || p.bs < 1 || p.width < 1 || p.width > 8192 || n < 0 || (n > 0 && (!base || !page_bytes || !heads || p.num_blocks < 1)) ||
      !table || !kv_lens || !path || !counts || !next || !lens || (p.total > 0 && (!picks || !tokens || !parents)) || (long long)p.max_blocks * p.bs > INT_MAX)
    return -3;
  p.picks = reinterpret_cast<const long long*>(picks), p.tokens = reinterpret_cast<const long long*>(tokens), p.parents = parents, p.cu_q = cu_q, p.kv_lens = kv_lens, p.table = table;
  p.table_stride = table_stride, p.path = path, p.counts = counts, p.next = reinterpret_cast<long long*>(next), p.lens = lens;
  for (int i = 0; i < (step > 0 && n > 1 ? 1 : n); ++i)
    if (heads[i] < 1 || page_bytes[i] < 1 || page_bytes[i] % ((long long)heads[i] * p.bs)) return -3;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int first = 0;
  do {
    Tensors t = part_of({base, page_bytes, heads, n, step}, first);
    int rc;
    switch (access_bytes(t, p.bs)) {
      case 16: rc = launch_accept<uint4>(t, p, s); break;
      case 8: rc = launch_accept<uint2>(t, p, s); break;
      case 4: rc = launch_accept<uint32_t>(t, p, s); break;
      case 2: rc = launch_accept<uint16_t>(t, p, s); break;
      default: rc = launch_accept<uint8_t>(t, p, s);
    }
    if (rc) return rc;
    first += MAX_TENSORS;
  } while (first < n);
  return 0;
}

// base, page_bytes and step as above. src and dst: n pairs, on the device or (on_host) lists of the host. Pairs whose numbers are not pages of the tensors are passed over.
int swb_copy_pages(const long long* base, const long long* page_bytes, long long step, int tensors, int num_blocks, const int* src, const int* dst, int n, int on_host, void* stream) {
  using namespace swb;
  if (n <= 0 || tensors <= 0) return 0;
  if (!base || !page_bytes || !src || !dst || num_blocks < 1 || n > INT_MAX / 64) return -3;
  for (int i = 0; i < (step > 0 ? 1 : tensors); ++i)
    if (page_bytes[i] < 1) return -3;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  for (int first = 0; first < tensors; first += MAX_TENSORS) {
    const Tensors t = part_of({base, page_bytes, nullptr, tensors, step}, first);
    const int access = access_bytes(t, 1);
    for (int at = 0; at < n;) {
      Pairs pairs;
      const int take = on_host ? (n - at < MAX_PAIRS ? n - at : MAX_PAIRS) : n;
      if (on_host) memcpy(pairs.src, src + at, sizeof(int) * take), memcpy(pairs.dst, dst + at, sizeof(int) * take);
      const int *from = on_host ? nullptr : src, *to = on_host ? nullptr : dst;
      int rc;
      switch (access) {
        case 16: rc = launch_copy<uint4>(t, pairs, from, to, take, num_blocks, s); break;
        case 8: rc = launch_copy<uint2>(t, pairs, from, to, take, num_blocks, s); break;
        case 4: rc = launch_copy<uint32_t>(t, pairs, from, to, take, num_blocks, s); break;
        case 2: rc = launch_copy<uint16_t>(t, pairs, from, to, take, num_blocks, s); break;
        default: rc = launch_copy<uint8_t>(t, pairs, from, to, take, num_blocks, s);
      }
      if (rc) return rc;
      at += take;
    }
  }
  return 0;
}

}  // extern "C"
