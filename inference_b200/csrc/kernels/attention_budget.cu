// Attention of new tokens over a paged cache, each on its own: over the pages that were selected for it, or over the whole cache with the weight that
// every key receives added up.
//
// A problem is one query token, one key/value head and up to 16 of the query heads that share it; its keys are dealt out to `num_splits` blocks in tiles. A block
// goes over its keys once with the running maximum and sum of the softmax in 32 bits, and leaves an un-normalised sum of values with both; the blocks of a
// problem are joined by a second launch (none where a problem has one block and no weights are kept). Weights need the maximum and sum over all
// keys, which are known at the end only: the scores are kept (4 bytes a key and query head, beside the keys' and values' 2 (D + Dv) a key), and the
// second launch turns them into weights and adds up those of a key over heads and tokens, in a fixed order and without atomics.
//
// Masked keys (behind what a token sees, on pages that are not there) take no part: their scores are -inf whatever the products were, and
// their values are not multiplied at all, so that what the memory holds there does not matter.
#include "attention_common.cuh"

#include <climits>

namespace swb {
using namespace attn;

namespace {

constexpr int ROWS = 16;                     // query heads of a problem

struct BudgetParams {
  const void* q;
  long long q_stride_tok, q_stride_head;
  void* out;
  long long out_stride_tok;
  const void* k;
  const void* v;
  const int* table;
  long long table_stride;
  int max_blocks, num_blocks, bs;
  const int* cu_q;
  const int* kv_lens;
  int num_seqs, uniform_q, tokens, Hkv, G, head_tiles, D, Dv;
  float scale, softcap;
  const int* pages;          // [tokens, Hkv, width]: the problem's pages by their place in the sequence; null: all pages
  const int* counts;         // [tokens, Hkv]
  int width;
  int num_splits;
  float* part_o;             // [problems, num_splits, ROWS, Dv]
  float* part_ml;            // [problems, num_splits, ROWS, 2]
  float* scores;             // [tokens, Hq, capacity] in log2 units, where weights are kept
  long long capacity;
  float* weights;            // [num_seqs, Hkv, .], inner stride 1
  long long w_seq, w_head;
};

// What a query token is: its sequence and the keys it sees.
struct Token {
  int seq, q0, q_len, seen;
};
__device__ __forceinline__ Token token_of(const BudgetParams& p, int t) {
  Token x;
  x.seq = seq_of_token(p.cu_q, p.num_seqs, p.uniform_q, t);
  x.q0 = p.cu_q ? p.cu_q[x.seq] : x.seq * p.uniform_q;
  x.q_len = p.cu_q ? p.cu_q[x.seq + 1] - x.q0 : p.uniform_q;
  x.seen = max(min(p.kv_lens[x.seq] - (x.q_len - 1 - (t - x.q0)), p.max_blocks * p.bs), 0);
  return x;
}

__device__ __forceinline__ void store_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_out(bf16* p, float x) { *p = __float2bfloat16(x); }

// ---- any types and widths: 32-bit arithmetic on ordinary cores --------------------------------------------------------------------------------------
constexpr int PLAIN_TILE = 32, PLAIN_THREADS = 128;

template <typename E, int COLS>       // COLS * 128 >= Dv
__global__ void __launch_bounds__(PLAIN_THREADS) attn_budget_plain_kernel(const BudgetParams p) {
  pdl_launch_dependents();
  extern __shared__ float plain_smem[];
  const int ldk = p.D + 1;
  float* sq = plain_smem;                          // [ROWS][D]
  float* sk = sq + ROWS * p.D;                     // [PLAIN_TILE][D + 1]
  float* sp = sk + PLAIN_TILE * ldk;               // [PLAIN_TILE][ROWS]
  __shared__ long long s_row[PLAIN_TILE];          // first row of the key's page + its place, -1: masked
  __shared__ float s_m[ROWS], s_l[ROWS], s_alpha[ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.x % p.num_splits, y = blockIdx.x / p.num_splits, hy = y % (p.Hkv * p.head_tiles), t = y / (p.Hkv * p.head_tiles);
  const int h = hy / p.head_tiles, ht = hy % p.head_tiles, g0 = ht * ROWS, rows = min(ROWS, p.G - g0);
  pdl_wait();
  if (p.cu_q && t >= p.cu_q[p.num_seqs]) return;
  const Token tok = token_of(p, t);
  const size_t list = (size_t)t * p.Hkv + h;
  const int count = p.pages ? min(max(p.counts[list], 0), p.width) : 0;
  const int total = p.pages ? count * p.bs : tok.seen;
  const int tiles = (total + PLAIN_TILE - 1) / PLAIN_TILE, per = (tiles + p.num_splits - 1) / p.num_splits;
  const int t_lo = split * per, t_hi = min(tiles, t_lo + per);
  const E* q = reinterpret_cast<const E*>(p.q) + t * p.q_stride_tok + (size_t)(h * p.G + g0) * p.q_stride_head;
  for (int i = tid; i < rows * p.D; i += PLAIN_THREADS) sq[i] = to_f(q[(i / p.D) * p.q_stride_head + i % p.D]);
  if (tid < ROWS) s_m[tid] = -INFINITY, s_l[tid] = 0.f;
  float o[COLS][ROWS];
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) o[c][r] = 0.f;
  const E* kc = reinterpret_cast<const E*>(p.k);
  const E* vc = reinterpret_cast<const E*>(p.v);
  for (int tile = t_lo; tile < t_hi; ++tile) {
    __syncthreads();
    if (tid < PLAIN_TILE) {
      const int j = tile * PLAIN_TILE + tid;
      long long row = -1;
      if (j < total) {
        const int page = p.pages ? p.pages[list * p.width + j / p.bs] : j / p.bs;
        const long long key = (long long)page * p.bs + j % p.bs;
        if (page >= 0 && key < tok.seen) {
          const int block = p.table[tok.seq * p.table_stride + page];
          if ((unsigned)block < (unsigned)p.num_blocks) row = ((long long)block * p.Hkv + h) * p.bs + j % p.bs;
        }
      }
      s_row[tid] = row;
    }
    __syncthreads();
    for (int i = tid; i < PLAIN_TILE * p.D; i += PLAIN_THREADS) {
      const int key = i / p.D, d = i % p.D;
      sk[key * ldk + d] = s_row[key] >= 0 ? to_f(kc[s_row[key] * p.D + d]) : 0.f;
    }
    __syncthreads();
    // lane = key, a warp every fourth row
    for (int r = warp; r < rows; r += PLAIN_THREADS / 32) {
      float s = 0.f;
      for (int d = 0; d < p.D; ++d) s = fmaf(sq[r * p.D + d], sk[lane * ldk + d], s);
      const bool live = s_row[lane] >= 0;
      s = live ? score_transform(s, p.scale, p.softcap) : -INFINITY;
      const int j = tile * PLAIN_TILE + lane;
      if (p.scores && j < total) p.scores[((size_t)t * p.Hkv * p.G + h * p.G + g0 + r) * p.capacity + j] = s;
      const float m0 = s_m[r], m1 = fmaxf(m0, warp_max(s)), base = m1 == -INFINITY ? 0.f : m1;
      const float e = exp2f(s - base), sum = warp_sum(e);
      sp[lane * ROWS + r] = live ? e : 0.f;
      __syncwarp();                                // s_m is read by all lanes before lane 0 writes it
      if (lane == 0) {
        const float alpha = exp2f(m0 - base);
        s_alpha[r] = alpha, s_m[r] = m1, s_l[r] = s_l[r] * alpha + sum;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < rows) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) o[c][r] *= s_alpha[r];
      }
    for (int key = 0; key < PLAIN_TILE; ++key) {
      if (s_row[key] < 0) continue;
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const int d = c * PLAIN_THREADS + tid;
        const float x = d < p.Dv ? to_f(vc[s_row[key] * p.Dv + d]) : 0.f;
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (r < rows) o[c][r] = fmaf(sp[key * ROWS + r], x, o[c][r]);
      }
    }
  }
  __syncthreads();
  const size_t problem = ((size_t)t * p.Hkv + h) * p.head_tiles + ht;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (r >= rows) break;
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const int d = c * PLAIN_THREADS + tid;
      if (d >= p.Dv) continue;
      if (p.part_o) p.part_o[((problem * p.num_splits + split) * ROWS + r) * p.Dv + d] = o[c][r];
      else store_out(reinterpret_cast<E*>(p.out) + t * p.out_stride_tok + (size_t)(h * p.G + g0 + r) * p.Dv + d, s_l[r] == 0.f ? 0.f : o[c][r] / s_l[r]);
    }
  }
  if (p.part_o && tid < rows) {
    float* ml = p.part_ml + ((problem * p.num_splits + split) * ROWS + tid) * 2;
    ml[0] = s_m[tid], ml[1] = s_l[tid];
  }
}

// ---- joining ------------------------------------------------------------------------------------------------------------------------------------------
constexpr int JOIN_THREADS = 128, MAX_SPLITS = 64;

// A block per problem: the parts of each row, weighed by their distance to the common maximum.
template <typename E>
__global__ void __launch_bounds__(JOIN_THREADS) attn_budget_join_kernel(const BudgetParams p) {
  pdl_launch_dependents();
  __shared__ float s_w[ROWS][MAX_SPLITS];
  const int tid = threadIdx.x, hy = blockIdx.x % (p.Hkv * p.head_tiles), t = blockIdx.x / (p.Hkv * p.head_tiles);
  const int h = hy / p.head_tiles, ht = hy % p.head_tiles, g0 = ht * ROWS, rows = min(ROWS, p.G - g0), S = p.num_splits;
  pdl_wait();
  if (p.cu_q && t >= p.cu_q[p.num_seqs]) return;
  const size_t problem = ((size_t)t * p.Hkv + h) * p.head_tiles + ht;
  if (tid < rows) {
    const float* ml = p.part_ml + (problem * S * ROWS + tid) * 2;
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < S; ++s) M = fmaxf(M, ml[(size_t)s * ROWS * 2]);
    const float base = M == -INFINITY ? 0.f : M;
    for (int s = 0; s < S; ++s) L += (s_w[tid][s] = exp2f(ml[(size_t)s * ROWS * 2] - base)) * ml[(size_t)s * ROWS * 2 + 1];
    const float inv = L == 0.f ? 0.f : 1.f / L;
    for (int s = 0; s < S; ++s) s_w[tid][s] *= inv;
  }
  __syncthreads();
  for (int i = tid; i < rows * p.Dv; i += JOIN_THREADS) {
    const int r = i / p.Dv, d = i % p.Dv;
    const float* o = p.part_o + (problem * S * ROWS + r) * p.Dv + d;
    float x = 0.f;
    for (int s = 0; s < S; ++s)
      if (s_w[r][s] != 0.f) x = fmaf(s_w[r][s], o[(size_t)s * ROWS * p.Dv], x);
    store_out(reinterpret_cast<E*>(p.out) + t * p.out_stride_tok + (size_t)(h * p.G + g0 + r) * p.Dv + d, x);
  }
}

constexpr int WEIGH_THREADS = 256, MAX_GROUP = 128;

// A block per (run of keys, key/value head, sequence): the weights of the sequence's new tokens, added up token by token and head by head.
__global__ void __launch_bounds__(WEIGH_THREADS) attn_budget_weigh_kernel(const BudgetParams p) {
  pdl_launch_dependents();
  __shared__ float s_m[MAX_GROUP], s_inv[MAX_GROUP];
  const int tid = threadIdx.x, h = blockIdx.y, seq = blockIdx.z, S = p.num_splits;
  const long long j = (long long)blockIdx.x * WEIGH_THREADS + tid;
  pdl_wait();
  const int q0 = p.cu_q ? p.cu_q[seq] : seq * p.uniform_q, q1 = p.cu_q ? p.cu_q[seq + 1] : q0 + p.uniform_q;
  const int len = min(p.kv_lens[seq], p.max_blocks * p.bs);
  if ((long long)blockIdx.x * WEIGH_THREADS >= len) return;
  float sum = 0.f;
  for (int t = q0; t < q1; ++t) {
    const int seen = p.kv_lens[seq] - (q1 - 1 - t);
    __syncthreads();
    for (int g = tid; g < p.G; g += WEIGH_THREADS) {
      const size_t problem = ((size_t)t * p.Hkv + h) * p.head_tiles + g / ROWS;
      const float* ml = p.part_ml + (problem * S * ROWS + g % ROWS) * 2;
      float M = -INFINITY, L = 0.f;
      for (int s = 0; s < S; ++s) M = fmaxf(M, ml[(size_t)s * ROWS * 2]);
      const float base = M == -INFINITY ? 0.f : M;
      for (int s = 0; s < S; ++s) L += exp2f(ml[(size_t)s * ROWS * 2] - base) * ml[(size_t)s * ROWS * 2 + 1];
      s_m[g] = base, s_inv[g] = L == 0.f ? 0.f : 1.f / L;
    }
    __syncthreads();
    if (j < seen && j < len) {
      const float* s = p.scores + ((size_t)t * p.Hkv + h) * p.G * p.capacity + j;
      for (int g = 0; g < p.G; ++g) sum = fmaf(exp2f(s[g * p.capacity] - s_m[g]), s_inv[g], sum);
    }
  }
  if (j < len) p.weights[seq * p.w_seq + h * p.w_head + j] += sum;
}

template <typename E>
int launch_plain(const BudgetParams& p, cudaStream_t s) {
  const size_t smem = 4 * ((size_t)ROWS * p.D + (size_t)PLAIN_TILE * (p.D + 1) + PLAIN_TILE * ROWS);
  auto kernel = p.Dv <= 128 ? attn_budget_plain_kernel<E, 1> : attn_budget_plain_kernel<E, 2>;
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -(int)e;
  }
  return launch_kernel(kernel, dim3(p.num_splits * p.Hkv * p.head_tiles * p.tokens), dim3(PLAIN_THREADS), smem, s, p);
}

int heads_in_tiles(int G) { return (G + ROWS - 1) / ROWS; }

}  // namespace
}  // namespace swb

extern "C" {

// Bytes of the workspace: the parts of the problems, and the scores where weights are kept (scores = 1; capacity: keys of the widest table row).
long long swb_attn_budget_workspace(int tokens, int Hkv, int G, int Dv, int num_splits, long long capacity, int scores) {
  const long long parts = num_splits > 1 || scores ? (long long)tokens * Hkv * swb::heads_in_tiles(G) * num_splits * swb::ROWS * (Dv + 2) * 4 : 0;
  return parts + (scores ? (long long)tokens * Hkv * G * capacity * 4 : 0);
}

// See BudgetParams. dims: host int[16] = tokens, num_seqs, tokens of each sequence (without cu_q), table width, blocks, block_size, Hkv, G, D, Dv,
// width of the page lists, splits, fp32, 0, 0, 0; strides: host long long[8] = q token and head, out token, table, weights sequence and head, 0, 0.
// pages and counts, or weights, or neither.
int swb_attn_budget(const int* dims, const long long* strides, const void* q, void* out, const void* k, const void* v, const int* table, const int* cu_q,
                    const int* kv_lens, const int* pages, const int* counts, float* weights, float scale, float softcap, void* workspace, long long workspace_bytes,
                    void* stream) {
  using namespace swb;
  BudgetParams p = {};
  p.tokens = dims[0], p.num_seqs = dims[1], p.uniform_q = dims[2], p.max_blocks = dims[3], p.num_blocks = dims[4], p.bs = dims[5];
  p.Hkv = dims[6], p.G = dims[7], p.D = dims[8], p.Dv = dims[9], p.width = dims[10], p.num_splits = dims[11];
  const int fp32 = dims[12];
  if (p.tokens <= 0 || p.num_seqs <= 0) return 0;
  if (p.num_seqs > 65535 || p.Hkv > 65535 || p.max_blocks < 1 || p.num_blocks < 1 || p.bs < 1 || p.Hkv < 1 || p.G < 1 || p.G > MAX_GROUP || p.D < 1 || p.D > 256 ||
      p.Dv < 1 || p.Dv > 256 || p.num_splits < 1 || p.num_splits > MAX_SPLITS || (!cu_q && p.uniform_q < 1) || (pages && (!counts || p.width < 1 || weights)) || !q || !out ||
      !k || !v || !table || !kv_lens)
    return -3;
  p.head_tiles = heads_in_tiles(p.G);
  if ((long long)p.tokens * p.Hkv * p.head_tiles * p.num_splits > INT_MAX) return -3;
  p.q = q, p.out = out, p.k = k, p.v = v, p.table = table, p.cu_q = cu_q, p.kv_lens = kv_lens, p.pages = pages, p.counts = counts, p.weights = weights;
  p.q_stride_tok = strides[0], p.q_stride_head = strides[1], p.out_stride_tok = strides[2], p.table_stride = strides[3], p.w_seq = strides[4], p.w_head = strides[5];
  p.scale = scale, p.softcap = softcap, p.capacity = (long long)p.max_blocks * p.bs;
  if (swb_attn_budget_workspace(p.tokens, p.Hkv, p.G, p.Dv, p.num_splits, p.capacity, weights != nullptr) > workspace_bytes) return -3;
  if (p.num_splits > 1 || weights) {
    const size_t rows = (size_t)p.tokens * p.Hkv * p.head_tiles * p.num_splits * ROWS;
    p.part_o = reinterpret_cast<float*>(workspace);
    p.part_ml = p.part_o + rows * p.Dv;
    if (weights) p.scores = p.part_ml + rows * 2;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int rc = fp32 ? launch_plain<float>(p, s) : launch_plain<bf16>(p, s);
  if (rc || !p.part_o) return rc;
  const dim3 grid(p.Hkv * p.head_tiles * p.tokens);
  rc = fp32 ? launch_kernel(attn_budget_join_kernel<float>, grid, dim3(JOIN_THREADS), 0, s, p)
            : launch_kernel(attn_budget_join_kernel<bf16>, grid, dim3(JOIN_THREADS), 0, s, p);
  if (rc || !weights) return rc;
  return launch_kernel(attn_budget_weigh_kernel, dim3((unsigned)((p.capacity + WEIGH_THREADS - 1) / WEIGH_THREADS), p.Hkv, p.num_seqs), dim3(WEIGH_THREADS), 0, s, p);
}

}  // extern "C"
