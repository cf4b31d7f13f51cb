// Attention of a tree of new tokens behind a paged cache: token i of a sequence sees every key in front of the step's tokens, and of these the ones whose bit in
// its row of the mask is set (itself and what it continues).
//
// A problem is a tile of rows of one sequence and key/value head; row r is token r / G and query head r % G of the group, so that the heads of a group share the keys that
// are read for them. Keys are dealt out to `num_splits` blocks a problem, which leave un-normalised sums of values with their maximum and sum for a second launch; one split
// finishes its rows itself. Scores, maxima and sums are 32-bit numbers; every sum has one order and there are no atomics.
//
// Keys that no row of the tile sees (behind the cache's end, on pages that are not there) and those that single rows do not see take no part: their scores are -inf whatever
// the products were, and their values are not multiplied, so that infinities and NaN there do not spread.
#include "attention_common.cuh"
#include "gemm_tcgen05.cuh"

#include <climits>

namespace swb {
using namespace attn;

SWB_REGISTER_STATUS_UNIT(attn_tree);

namespace {

constexpr int MAX_SPLITS = 64, MAX_GROUP = 128;

struct TreeParams {
  const void* q;
  long long q_tok, q_head;
  void* out;
  long long out_tok;
  const void* k;
  const void* v;
  const int* table;
  long long table_stride;
  int max_blocks, num_blocks, bs;
  const int* cu_q;
  const int* kv_lens;
  const unsigned* mask;      // [tokens, words], rows mask_tok apart
  long long mask_tok;
  int words;
  int num_seqs, uniform_q, tokens, Hkv, G, D, Dv;
  float scale, softcap;
  int tiles, num_splits;     // row tiles of a sequence, splits of a tile's keys
  float* part_o;             // [split][tokens][Hq][Dv]; null: one split
  float2* part_ml;           // [split][tokens][Hq]: maximum (log2 units) and sum
};

// A sequence's part of the step.
struct Span {
  int q0, n;                 // its first row of q and its tokens
  int len, base;             // cached tokens with the new ones, and without (below zero where the table has no room for all new ones)
};
__device__ __forceinline__ Span span_of(const TreeParams& p, int seq) {
  Span s;
  s.q0 = p.cu_q ? p.cu_q[seq] : seq * p.uniform_q;
  s.n = p.cu_q ? p.cu_q[seq + 1] - s.q0 : p.uniform_q;
  s.len = max(min(p.kv_lens[seq], p.max_blocks * p.bs), 0);
  s.base = s.len - s.n;
  return s;
}

__device__ __forceinline__ bool sees(const unsigned* row, int words, int rel) {
  return rel < 0 || ((rel >> 5) < words && (row[rel >> 5] >> (rel & 31) & 1u));
}

__device__ __forceinline__ void store_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_out(bf16* p, float x) { *p = __float2bfloat16(x); }

// ---- any types and widths: 32-bit arithmetic on ordinary cores --------------------------------------------------------------------------------------
constexpr int PR = 32, PK = 32, PLAIN_THREADS = 128;          // rows and keys of a tile

__device__ __forceinline__ int padded4(int d) { return (d + 3) / 4 * 4; }

// One row of `width` numbers as 32-bit numbers, zeros behind its end: a warp.
template <typename E, bool VEC>
__device__ __forceinline__ void fetch_row(float* to, const E* from, int width, int lane) {
  if constexpr (VEC) {
    for (int d = lane * 4; d < width; d += 128) *reinterpret_cast<float4*>(to + d) = load_row4(from + d);
  } else {
    for (int d = lane; d < padded4(width); d += 32) to[d] = d < width ? to_f(from[d]) : 0.f;
  }
}

// COLS * 64 >= Dv. VEC: rows of the caches start on four numbers and are a multiple of four long.
template <typename E, int COLS, bool VEC>
__global__ void __launch_bounds__(PLAIN_THREADS) attn_tree_plain_kernel(const TreeParams p) {
  pdl_launch_dependents();
  extern __shared__ __align__(16) float tree_smem[];
  const int ldk = padded4(p.D) + 4, ldv = padded4(p.Dv);       // lanes with neighbouring keys meet in no bank
  float* sq = tree_smem;                           // [PR][ldk]
  float* sk = sq + PR * ldk;                       // [PK][ldk]
  float* sv = sk + PK * ldk;                       // [PK][ldv]
  float* sp = sv + PK * ldv;                       // [PK][PR + 4]
  constexpr int LDP = PR + 4;
  __shared__ long long s_row[PK];                  // first row of the key's page + its place, -1: no such key
  __shared__ float s_alpha[PR], s_m[PR], s_l[PR];
  __shared__ unsigned s_seen[PR];                  // keys of the tile that a row sees
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.x % p.num_splits, y = blockIdx.x / p.num_splits, h = y % p.Hkv, z = y / p.Hkv, tile = z % p.tiles, seq = z / p.tiles;
  pdl_wait();
  const Span s = span_of(p, seq);
  const int r0 = tile * PR, rows = min(PR, min(s.n, p.uniform_q) * p.G - r0);
  if (rows <= 0) return;
  const E* q = reinterpret_cast<const E*>(p.q);
  for (int r = warp; r < PR; r += PLAIN_THREADS / 32) {
    const int t = s.q0 + (r0 + r) / p.G, g = (r0 + r) % p.G;
    const bool live = r < rows && (unsigned)t < (unsigned)p.tokens;
    const E* from = q + (live ? t * p.q_tok + (long long)(h * p.G + g) * p.q_head : 0);
    for (int d = lane; d < ldk - 4; d += 32) sq[r * ldk + d] = live && d < p.D ? to_f(from[d]) : 0.f;
  }
  if (tid < PR) s_m[tid] = -INFINITY, s_l[tid] = 0.f;
  float o[COLS][16];                               // rows 16 (tid / 64) .. + 15 of columns tid % 64 + 64 c
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[c][r] = 0.f;
  const int col = tid % 64, half = tid / 64;
  const int kt = (s.len + PK - 1) / PK, per = (kt + p.num_splits - 1) / p.num_splits;
  const int lo = min(split * per, kt), hi = min(kt, lo + per);
  for (int it = lo; it < hi; ++it) {
    const int j0 = it * PK;
    __syncthreads();
    if (tid < PK) {
      long long row = -1;
      const int j = j0 + tid;
      if (j < s.len) {
        const int block = p.table[seq * p.table_stride + j / p.bs];
        if ((unsigned)block < (unsigned)p.num_blocks) row = ((long long)block * p.Hkv + h) * p.bs + j % p.bs;
      }
      s_row[tid] = row;
      const unsigned there = __ballot_sync(0xffffffffu, row >= 0);
      unsigned seen = 0;                           // lane = row
      const int t = s.q0 + (r0 + tid) / p.G;
      if (tid < rows && (unsigned)t < (unsigned)p.tokens) {
        if (j0 + PK <= s.base) {
          seen = 0xffffffffu;
        } else {
          for (int i = 0; i < PK; ++i) seen |= (unsigned)sees(p.mask + t * p.mask_tok, p.words, j0 + i - s.base) << i;
        }
      }
      s_seen[tid] = seen & there;
    }
    __syncthreads();
    for (int i = warp; i < PK; i += PLAIN_THREADS / 32) {
      const long long row = s_row[i];
      if (row >= 0) {
        fetch_row<E, VEC>(sk + i * ldk, reinterpret_cast<const E*>(p.k) + row * p.D, p.D, lane);
        fetch_row<E, VEC>(sv + i * ldv, reinterpret_cast<const E*>(p.v) + row * p.Dv, p.Dv, lane);
      } else {
        for (int d = lane; d < ldk; d += 32) sk[i * ldk + d] = 0.f;
        for (int d = lane; d < ldv; d += 32) sv[i * ldv + d] = 0.f;
      }
    }
    __syncthreads();
    // scores: a thread has 8 rows of one key
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    for (int d = 0; d < ldk - 4; d += 4) {
      const float4 k = *reinterpret_cast<const float4*>(sk + lane * ldk + d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 a = *reinterpret_cast<const float4*>(sq + (warp * 8 + i) * ldk + d);
        x[i] = fmaf(a.x, k.x, x[i]), x[i] = fmaf(a.y, k.y, x[i]), x[i] = fmaf(a.z, k.z, x[i]), x[i] = fmaf(a.w, k.w, x[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = warp * 8 + i;
      const bool live = s_seen[r] >> lane & 1u;
      const float sc = live ? score_transform(x[i], p.scale, p.softcap) : -INFINITY;
      const float m0 = s_m[r], m1 = fmaxf(m0, warp_max(sc)), base = m1 == -INFINITY ? 0.f : m1;
      const float e = exp2f(sc - base), sum = warp_sum(e);
      sp[lane * LDP + r] = live ? e : 0.f;
      __syncwarp();                                // s_m is read by all lanes before lane 0 writes it
      if (lane == 0) {
        const float alpha = exp2f(m0 - base);
        s_alpha[r] = alpha, s_m[r] = m1, s_l[r] = s_l[r] * alpha + sum;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float alpha = s_alpha[half * 16 + r];
#pragma unroll
      for (int c = 0; c < COLS; ++c) o[c][r] *= alpha;
    }
    const bool whole = j0 + PK <= s.base;          // all rows see all keys, or none does (then its value is a zero)
    for (int key = 0; key < PK; ++key) {
      float w[16];
#pragma unroll
      for (int r = 0; r < 16; r += 4) *reinterpret_cast<float4*>(w + r) = *reinterpret_cast<const float4*>(sp + key * LDP + half * 16 + r);
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const int d = c * 64 + col;
        const float val = d < p.Dv ? sv[key * ldv + d] : 0.f;
        if (whole || isfinite(val)) {
#pragma unroll
          for (int r = 0; r < 16; ++r) o[c][r] = fmaf(w[r], val, o[c][r]);
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (s_seen[half * 16 + r] >> key & 1u) o[c][r] = fmaf(w[r], val, o[c][r]);
        }
      }
    }
  }
  __syncthreads();
  const int Hq = p.Hkv * p.G;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = half * 16 + r, t = s.q0 + (r0 + row) / p.G, head = h * p.G + (r0 + row) % p.G;
    if (row >= rows || (unsigned)t >= (unsigned)p.tokens) continue;
    const float l = s_l[row];
    const long long at = ((long long)split * p.tokens + t) * Hq + head;
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const int d = c * 64 + col;
      if (d >= p.Dv) continue;
      if (p.part_o) p.part_o[at * p.Dv + d] = o[c][r];
      else store_out(reinterpret_cast<E*>(p.out) + t * p.out_tok + (long long)head * p.Dv + d, l == 0.f ? 0.f : o[c][r] / l);
    }
    if (p.part_o && col == 0) p.part_ml[at] = make_float2(s_m[row], l);
  }
}

// ---- sum of the splits --------------------------------------------------------------------------------------------------------------------------------
// A warp to a row and head, weighed by the distance of its splits' maxima to the common one.
constexpr int JOIN_THREADS = 128;

template <typename E>
__global__ void __launch_bounds__(JOIN_THREADS) attn_tree_join_kernel(const TreeParams p) {
  pdl_launch_dependents();
  const int Hq = p.Hkv * p.G, lane = threadIdx.x & 31, S = p.num_splits;
  const long long i = (long long)blockIdx.x * (JOIN_THREADS / 32) + (threadIdx.x >> 5), rows = (long long)p.tokens * Hq;
  pdl_wait();
  if (i >= rows) return;
  const int t = (int)(i / Hq), head = (int)(i % Hq);
  if (p.cu_q) {
    if (t < p.cu_q[0] || t >= p.cu_q[p.num_seqs]) return;
    const int seq = seq_of_token(p.cu_q, p.num_seqs, p.uniform_q, t);
    if (t - p.cu_q[seq] >= p.uniform_q) return;              // more tokens than the call was told of: not computed
  }
  float2 a = make_float2(-INFINITY, 0.f), b = a;
  if (lane < S) a = p.part_ml[lane * rows + i];
  if (lane + 32 < S) b = p.part_ml[(lane + 32) * rows + i];
  const float top = warp_max(fmaxf(a.x, b.x)), base = top == -INFINITY ? 0.f : top;
  const float fa = exp2f(a.x - base), fb = exp2f(b.x - base);
  const float sum = warp_sum(fmaf(fa, a.y, fb * b.y)), inv = sum == 0.f ? 0.f : 1.f / sum;
  E* out = reinterpret_cast<E*>(p.out) + t * p.out_tok + (long long)head * p.Dv;
  for (int d0 = 0; d0 < p.Dv; d0 += 32) {
    const int d = d0 + lane;
    float x = 0.f;
    for (int s = 0; s < S; ++s) {                            // all lanes: each has the factors of two splits
      const float f = __shfl_sync(0xffffffffu, s < 32 ? fa : fb, s & 31);
      if (d < p.Dv) x = fmaf(f, p.part_o[(s * rows + i) * p.Dv + d], x);
    }
    if (d < p.Dv) store_out(out + d, x * inv);
  }
}

template <typename E, int COLS, bool VEC>
int launch_plain(const TreeParams& p, cudaStream_t s) {
  const int ldk = (p.D + 3) / 4 * 4 + 4, ldv = (p.Dv + 3) / 4 * 4;
  const size_t smem = 4 * ((size_t)(PR + PK) * ldk + (size_t)PK * ldv + PK * (PR + 4));
  auto kernel = attn_tree_plain_kernel<E, COLS, VEC>;
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -(int)e;
  }
  return launch_kernel(kernel, dim3((unsigned)((long long)p.num_splits * p.Hkv * p.tiles * p.num_seqs)), dim3(PLAIN_THREADS), smem, s, p);
}

template <typename E>
int launch_plain(const TreeParams& p, cudaStream_t s) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
  const bool vec = (p.D | p.Dv) % 4 == 0 && at % (4 * sizeof(E)) == 0;
  if (p.Dv <= 64) return vec ? launch_plain<E, 1, true>(p, s) : launch_plain<E, 1, false>(p, s);
  if (p.Dv <= 128) return vec ? launch_plain<E, 2, true>(p, s) : launch_plain<E, 2, false>(p, s);
  return vec ? launch_plain<E, 4, true>(p, s) : launch_plain<E, 4, false>(p, s);
}

}  // namespace
}  // namespace swb

extern "C" {

// See TreeParams. dims: host int[16] = tokens, num_seqs, tokens of each sequence (with cu_q: at most), table width, blocks, block_size, Hkv, G, D, Dv, words of a mask row, splits,
// fp32, 0, 0, 0; strides: host long long[8] = q token and head, out token, table, mask token, 0, 0, 0. workspace (16-byte aligned), with more
// than one split: 4 splits tokens Hq (Dv + 2) bytes.
int swb_attn_tree(const int* dims, const long long* strides, const void* q, void* out, const void* k, const void* v, const int* table, const int* cu_q, const int* kv_lens,
                  const void* mask, float scale, float softcap, void* workspace, long long workspace_bytes, void* stream) {
  using namespace swb;
  TreeParams p = {};
  p.tokens = dims[0], p.num_seqs = dims[1], p.uniform_q = dims[2], p.max_blocks = dims[3], p.num_blocks = dims[4], p.bs = dims[5];
  p.Hkv = dims[6], p.G = dims[7], p.D = dims[8], p.Dv = dims[9], p.words = dims[10], p.num_splits = dims[11];
  const int fp32 = dims[12];
  if (p.tokens <= 0 || p.num_seqs <= 0) return 0;
  if (p.num_seqs > 65535 || p.max_blocks < 1 || p.num_blocks < 1 || p.bs < 1 || p.Hkv < 1 || p.G < 1 || p.G > MAX_GROUP || p.D < 1 || p.D > 256 || p.Dv < 1 || p.Dv > 256 ||
      p.num_splits < 1 || p.num_splits > MAX_SPLITS || p.uniform_q < 1 || p.words < 1 || !q || !out || !k || !v || !table || !kv_lens || !mask)
    return -3;
  if ((long long)p.max_blocks * p.bs > INT_MAX || (long long)p.uniform_q * p.G > INT_MAX - PR) return -3;
  p.tiles = (p.uniform_q * p.G + PR - 1) / PR;
  if ((long long)p.tiles * p.num_seqs * p.Hkv > INT_MAX / p.num_splits || (long long)p.tokens * p.Hkv * p.G > INT_MAX) return -3;
  p.q = q, p.out = out, p.k = k, p.v = v, p.table = table, p.cu_q = cu_q, p.kv_lens = kv_lens, p.mask = reinterpret_cast<const unsigned*>(mask);
  p.q_tok = strides[0], p.q_head = strides[1], p.out_tok = strides[2], p.table_stride = strides[3], p.mask_tok = strides[4];
  p.scale = scale, p.softcap = softcap;
  const long long rows = (long long)p.tokens * p.Hkv * p.G;
  if (p.num_splits > 1) {
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || 4 * rows * p.num_splits * (p.Dv + 2) > workspace_bytes) return -3;
    p.part_ml = reinterpret_cast<float2*>(workspace);
    p.part_o = reinterpret_cast<float*>(workspace) + rows * p.num_splits * 2;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int rc = fp32 ? launch_plain<float>(p, s) : launch_plain<bf16>(p, s);
  if (rc || p.num_splits == 1) return rc;
  const dim3 grid((unsigned)((rows + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32)));
  return fp32 ? launch_kernel(attn_tree_join_kernel<float>, grid, dim3(JOIN_THREADS), 0, s, p) : launch_kernel(attn_tree_join_kernel<bf16>, grid, dim3(JOIN_THREADS), 0, s, p);
}

}  // extern "C"
