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
#include "attention_tc.cuh"
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
  int q_vec, out_vec;        // rows of q and of out start on what a load and a store take: 16 bytes, four numbers in the plain kernel and the sum of the splits
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
// 32 x 32 tiles, as rows are few: two trees of 21 tokens x 16 heads behind 900 keys are 24 problems of 29 tiles, 34 us with the sum of the splits (53 with a row of keys fetched at a time, single
// multiply-adds and a long epilogue). A block alone takes 5 to 6 us a tile, three on an SM 10: shared reads (9 for 16 paired multiply-adds of the scores, 6 for 16 of the values) and
// multiply-adds wait for one another, at a quarter to a half of the issue slots.
constexpr int PR = 32, PK = 32, PLAIN_THREADS = 128, ROUND = PLAIN_THREADS / PK;          // rows and keys of a tile; tiles whose keys are looked up at once

__device__ __forceinline__ int padded4(int d) { return (d + 3) / 4 * 4; }

// N rows of `width` numbers as 32-bit numbers, zeros behind their ends and for those without a place (from[i] null): a warp, with all of a round's loads in flight before the first of them
// is kept (a row at a time each waited for memory: 11 of 53 us of two trees of 21 tokens x 16 heads behind 900 keys).
template <typename E, bool VEC, int N>
__device__ __forceinline__ void fetch_rows(float* to, int ld, const E* const (&from)[N], int width, int lane) {
  constexpr int W = VEC ? 4 : 1;
  const int end = VEC ? width : padded4(width);
  for (int d = lane * W; d < end; d += 32 * W) {
    float4 x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if constexpr (VEC) {
        if (from[i]) x[i] = load_row4(from[i] + d);
      } else {
        if (from[i] && d < width) x[i].x = to_f(from[i][d]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (VEC) *reinterpret_cast<float4*>(to + i * ld + d) = x[i];
      else to[i * ld + d] = x[i].x;
    }
  }
}

// Word i of a token's row of the mask.
__device__ __forceinline__ unsigned mask_word(const unsigned* row, int words, int i) { return i < words ? row[i] : 0u; }

// Which of the 32 keys from `rel` places behind the cache's end on (in front of it: rel < 0) a token sees.
__device__ __forceinline__ unsigned sees32(const unsigned* row, int words, int rel) {
  if (rel <= -32) return 0xffffffffu;
  if (rel < 0) return ((1u << -rel) - 1u) | (mask_word(row, words, 0) << -rel);
  return __funnelshift_r(mask_word(row, words, rel >> 5), mask_word(row, words, (rel >> 5) + 1), rel & 31);
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
  constexpr int LDP = PR + 4, MINE = PR / (PLAIN_THREADS / 32);        // rows, and keys of a tile, of a warp
  static_assert(PR == 32 && PK == 32);
  __shared__ long long s_row[ROUND * PK];          // of a round of tiles: first row of the key's page + its place, -1: no such key
  __shared__ __align__(8) float s_alpha[PR];
  __shared__ long long s_dst[PR], s_ml[PR];
  __shared__ float s_m[PR], s_l[PR];               // at the end: a warp has its rows' in registers
  __shared__ unsigned s_seen[PR];                  // keys of the tile that a row sees
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.x % p.num_splits, y = blockIdx.x / p.num_splits, h = y % p.Hkv, z = y / p.Hkv, tile = z % p.tiles, seq = z / p.tiles;
  pdl_wait();
  const Span s = span_of(p, seq);
  const int r0 = tile * PR, rows = min(PR, min(s.n, p.uniform_q) * p.G - r0);
  if (rows <= 0) return;
  const E* q = reinterpret_cast<const E*>(p.q);
  // lane = row: its token, and where its results go (-1: there is no such row)
  const int Hq = p.Hkv * p.G, token = s.q0 + (r0 + lane) / p.G, head = h * p.G + (r0 + lane) % p.G;
  const bool live = lane < rows && (unsigned)token < (unsigned)p.tokens;
  if (warp == 0) {
    const long long at = ((long long)split * p.tokens + token) * Hq + head;
    s_dst[lane] = !live ? -1 : p.part_o ? at * p.Dv : token * p.out_tok + (long long)head * p.Dv;
    s_ml[lane] = at;
  }
  {
    const long long mine = live ? token * p.q_tok + head * p.q_head : -1;
    const E* from[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const long long at = __shfl_sync(0xffffffffu, mine, warp * MINE + i);
      from[i] = at >= 0 ? q + at : nullptr;
    }
    // four numbers at a time in bf16, where a load then takes 8 bytes of a lane and not 2 (8 trees of 20 tokens, heads of 256, 1500 keys: 241 us, a number at a time 264); one in fp32 (the two
    // trees above: 35.1 us, four at a time 35.9)
    if (VEC && sizeof(E) == 2 && p.q_vec) fetch_rows<E, VEC>(sq + warp * MINE * ldk, ldk, from, p.D, lane);
    else fetch_rows<E, false>(sq + warp * MINE * ldk, ldk, from, p.D, lane);
  }
  float m[MINE], l[MINE];                          // of rows warp * MINE + i: maximum (log2 units) and sum, the same in all lanes
#pragma unroll
  for (int i = 0; i < MINE; ++i) m[i] = -INFINITY, l[i] = 0.f;
  unsigned long long o[COLS][8];                   // rows 16 (tid / 64) .. + 15, two in a place, of columns tid % 64 + 64 c
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int r = 0; r < 8; ++r) o[c][r] = 0;
  const int col = tid % 64, half = tid / 64;
  const int kt = (s.len + PK - 1) / PK, per = (kt + p.num_splits - 1) / p.num_splits;
  const int lo = min(split * per, kt), hi = min(kt, lo + per);
  for (int it = lo; it < hi; ++it) {
    const int j0 = it * PK, at = (it - lo) % ROUND * PK;
    __syncthreads();
    if (at == 0) {                                 // where the keys of the next tiles lie: a thread to a key
      long long row = -1;
      const int j = j0 + tid;
      if (j < s.len) {
        const int block = p.table[seq * p.table_stride + j / p.bs];
        if ((unsigned)block < (unsigned)p.num_blocks) row = ((long long)block * p.Hkv + h) * p.bs + j % p.bs;
      }
      s_row[tid] = row;
      __syncthreads();
    }
    if (warp == 0) {
      const unsigned there = __ballot_sync(0xffffffffu, s_row[at + lane] >= 0);
      s_seen[lane] = live ? sees32(p.mask + token * p.mask_tok, p.words, j0 - s.base) & there : 0u;
    }
    {
      const E *k[MINE], *v[MINE];
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const long long row = s_row[at + warp * MINE + i];
        k[i] = row >= 0 ? reinterpret_cast<const E*>(p.k) + row * p.D : nullptr;
        v[i] = row >= 0 ? reinterpret_cast<const E*>(p.v) + row * p.Dv : nullptr;
      }
      fetch_rows<E, VEC>(sk + warp * MINE * ldk, ldk, k, p.D, lane);
      fetch_rows<E, VEC>(sv + warp * MINE * ldv, ldv, v, p.Dv, lane);
    }
    __syncthreads();
    // where rows differ in what they see: whether all values are numbers (else a product with a weight of zero would be none)
    bool odd = false;
    if (j0 + PK > s.base) {
      for (int i = tid; i < PK * ldv; i += PLAIN_THREADS) odd |= !isfinite(sv[i]);
      odd = __syncthreads_or(odd);
    }
    // scores: a thread has 8 rows of one key, sums of the even and the odd numbers
    unsigned long long xx[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) xx[i] = 0;
#pragma unroll 2
    for (int d = 0; d < ldk - 4; d += 4) {
      const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(sk + lane * ldk + d);
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(sq + (warp * MINE + i) * ldk + d);
        xx[i] = fma2(a.y, k.y, fma2(a.x, k.x, xx[i]));
      }
    }
    float x[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      float even, other;
      unpack2(xx[i], even, other);
      x[i] = even + other;
    }
    float top[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      x[i] = s_seen[warp * MINE + i] >> lane & 1u ? score_transform(x[i], p.scale, p.softcap) : -INFINITY;
      top[i] = x[i];
    }
#pragma unroll
    for (int step = 16; step; step >>= 1) {        // the rows' reductions side by side
#pragma unroll
      for (int i = 0; i < MINE; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], step));
    }
    float sum[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int r = warp * MINE + i;
      const float m1 = fmaxf(m[i], top[i]), base = m1 == -INFINITY ? 0.f : m1, alpha = exp2f(m[i] - base);
      sum[i] = exp2f(x[i] - base);
      sp[lane * LDP + r] = s_seen[r] >> lane & 1u ? sum[i] : 0.f;
      if (lane == 0) s_alpha[r] = alpha;
      l[i] *= alpha, m[i] = m1;
    }
#pragma unroll
    for (int step = 16; step; step >>= 1) {
#pragma unroll
      for (int i = 0; i < MINE; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], step);
    }
#pragma unroll
    for (int i = 0; i < MINE; ++i) l[i] += sum[i];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const unsigned long long alpha = *reinterpret_cast<const unsigned long long*>(s_alpha + half * 16 + 2 * r);
#pragma unroll
      for (int c = 0; c < COLS; ++c) o[c][r] = fma2(o[c][r], alpha, 0ull);
    }
    if (!odd) {
#pragma unroll 4
      for (int key = 0; key < PK; ++key) {
        unsigned long long w[8];
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
          const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(sp + key * LDP + half * 16 + 2 * r);
          w[r] = two.x, w[r + 1] = two.y;
        }
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          const int d = c * 64 + col;
          const float val = d < p.Dv ? sv[key * ldv + d] : 0.f;
          const unsigned long long both = pack2(val, val);
#pragma unroll
          for (int r = 0; r < 8; ++r) o[c][r] = fma2(w[r], both, o[c][r]);
        }
      }
    } else {
#pragma unroll 1
      for (int key = 0; key < PK; ++key) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          const int d = c * 64 + col;
          const float val = d < p.Dv ? sv[key * ldv + d] : 0.f;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int row = half * 16 + 2 * r;
            float lower, upper;
            unpack2(o[c][r], lower, upper);
            if (s_seen[row] >> key & 1u) lower = fmaf(sp[key * LDP + row], val, lower);
            if (s_seen[row + 1] >> key & 1u) upper = fmaf(sp[key * LDP + row + 1], val, upper);
            o[c][r] = pack2(lower, upper);
          }
        }
      }
    }
  }
  // one row after another in little code: what a block runs once, it waits for from the instruction memory (all 16 rows unrolled, with their divisions: 10 us for a step without keys, now 5)
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) s_m[warp * MINE + i] = m[i], s_l[warp * MINE + i] = p.part_o ? l[i] : l[i] == 0.f ? 0.f : 1.f / l[i];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = half * 16 + r;
    const long long at = s_dst[row];
    if (at < 0) continue;
    const float factor = p.part_o ? 1.f : s_l[row];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const int d = c * 64 + col;
      float even, other;
      unpack2(o[c][r / 2], even, other);
      const float sum = (r % 2 ? other : even) * factor;
      if (d >= p.Dv) continue;
      if (p.part_o) p.part_o[at + d] = sum;
      else store_out(reinterpret_cast<E*>(p.out) + at + d, sum);
    }
  }
  if (p.part_o && tid < PR && s_dst[tid] >= 0) p.part_ml[s_ml[tid]] = make_float2(s_m[tid], s_l[tid]);
}

// ---- bf16, widths up to 128, pages of 16-key groups: products on the tensor memory's matrix instructions -----------------------------------------------------
//
// A block has up to 256 rows of a problem and walks its keys in tiles of 128. It works on two things at once ("slots"), so that the products of one run beside the softmax of the other:
// with more than 128 rows on their two halves, which share the tiles, else on the even and the odd tiles, whose results it joins at its end.
//   warp 16      producer: a box of 16 keys x 64 columns to a lane, so that a tile of K or V is one instruction of the warp; groups of keys that are not there are fetched from
//                behind the cache, which fills zeros in
//   warps 17, 18 matrix instructions, one warp a slot: S = Q K^T, then O += P V with P in tensor memory, where it takes the place of S, and V as it lies (its rows are the product's
//                inner dimension); the scores of the next tile follow the product that frees their place
//   (warp 19 makes the last four a group that hands registers on)
//   warps 0-15   softmax, eight to a slot, two threads to a row with 64 of a tile's keys each; in tiles of the tree they apply the mask and see to it that V holds numbers
// Tensor memory of a slot: S (128 columns; P in the first half of each thread's own 64), O (128). Shared memory has seven buffers of a tile: Q, three of K, and two of V with Q's second half
// or three of V.
// 64 tokens x 32 heads (8 key/value heads) behind 100 000 keys, blocks of 256 rows and 44 tiles: 121 us with the sum of the splits, 0.87 PFLOP/s; some 95 without any softmax. (One slot a block and
// two blocks to an SM, each tile asked for when the one before it was used: 155.) A tile takes a slot some 3400 cycles: 1850 from its scores to its weights, of them 1000 for the exponentials, which
// the special-function units alone would need 1024 for at least (1190 in fact), and 1570 from there to the next scores, of them 1024 for the products; those of both slots together keep the tensor
// cores busy for 2048. Maxima of three numbers and one vote in place of two were 3 % of it. What did not help: tiles of 64 keys with two of scores a slot, references a tile old in place of a row's own maximum (its steps cost more
// than the exchange), Q in tensor memory beside tiles of 64 keys (152: the softmax's steps come twice as often), P handed over in two
// halves (147: one more wait for the stores and one more signal a tile), copies of 16 keys x 128 columns, which take two thirds of the time of two of 64 columns (5 % more here, 3 % less for 48 trees
// of up to 48 tokens behind 4100 keys), tiles asked for in the second-level cache four ahead (147), first tiles, Q and tensor memory asked for beside one another in front of the first barrier (no change).
constexpr int TC_ROWS = 128, TC_KEYS = 128, TC_THREADS = 640, TMA_WARP = 16, MMA_WARP = 17, K_STAGES = 3, V_STAGES = 3, SOFT_REGS = 112, ROLE_REGS = 32;
constexpr uint32_t TC_COLS = 512;
constexpr float TC_RESCALE = 8.f;          // O is rescaled when a maximum has grown by more than 2^8

// What a block works on. It lies in shared memory: the softmax has all of its registers full of scores, and reads what it needs of it where it needs it.
struct Block {
  Span s;
  int seq, h, r0, rows, split, t_lo, n_tiles;
  int tail;                // first tile that has keys of the tree, or behind it
  int two;                 // the slots are halves of the rows
};

struct TcBars {
  uint64_t q_full, k_full[K_STAGES], k_empty[K_STAGES], v_full[V_STAGES], v_empty[V_STAGES], v_clean[V_STAGES], s_full[2], p_full[2], o_final;
  uint32_t tmem_base;
  int abort;
  int odd;                 // some new token's value is no number
  unsigned dead[16];       // groups of a tile's keys that are not there
  Block block;
};
static_assert(sizeof(TcBars) <= 512, "room in front of the exchange");
template <int DA, int VA>
struct TcCfg {
  static constexpr uint32_t KT = DA * TC_ATOM_BYTES, VT = VA * TC_ATOM_BYTES, LAST = KT > VT ? KT : VT;      // the last buffer is Q's or V's
  static constexpr uint32_t Q = 0, K = KT, V = K + K_STAGES * KT, X = V + 2 * VT, BARS = X + LAST, EXCHANGE = BARS + 512;
  static constexpr size_t BYTES = EXCHANGE + 2 * 2 * TC_ROWS * 4;          // [slot][half][row]
};

__device__ __forceinline__ Block load_block(TcBars* bars) {
  static_assert(sizeof(Block) % 4 == 0, "words");
  Block b;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(Block) / 4); ++i) reinterpret_cast<int*>(&b)[i] = reinterpret_cast<volatile int*>(&bars->block)[i];
  return b;
}

// A place in a ring of stages, and how often it has been gone round (its lowest bit).
struct Ring {
  int at, round;
  __device__ __forceinline__ void advance(int by, int stages) {
    at += by;
    if (at >= stages) at -= stages, round ^= 1;
  }
};

// Which of the 64 keys from key0 on a row sees.
__device__ __forceinline__ unsigned long long seen_keys(const unsigned* row, int words, int key0, int base, int len, unsigned dead) {
  const int rel = key0 - base;
  unsigned long long seen = ~0ull;
  if (rel > -64) {
    const int from = max(rel, 0), w = from >> 5, sh = from & 31;
    const unsigned a = w < words ? row[w] : 0u, b = w + 1 < words ? row[w + 1] : 0u, c = w + 2 < words ? row[w + 2] : 0u;
    seen = (unsigned long long)__funnelshift_r(b, c, sh) << 32 | __funnelshift_r(a, b, sh);
    if (rel < 0) seen = seen << -rel | ((1ull << -rel) - 1);
  }
  const int left = len - key0;
  if (left < 64) seen &= left > 0 ? (1ull << left) - 1 : 0ull;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    if (dead >> g & 1u) seen &= ~(0xffffull << 16 * g);
  return seen;
}


__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}

// 2^x on the multiply-add pipes, for x below 100: x = n + f, |f| <= 1/2, the polynomial of `ex2_fma2` in f times 2^n. Below -126.5 it is zero; what is not a number stays so.
__device__ __forceinline__ float ex2_fma(float x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-127.f));
  const float t = x + 12582912.f, f = x - (t - 12582912.f);
  float r = fmaf(f, EXP_5, EXP_4);
  r = fmaf(r, f, EXP_3), r = fmaf(r, f, EXP_2), r = fmaf(r, f, EXP_1), r = fmaf(r, f, EXP_0);
  return r * __int_as_float((__float_as_int(t) << 23) + 0x3f800000);
}

// A row's columns in tensor memory times f: whole warp.
template <int COLS>
__device__ __forceinline__ void scale_columns(uint32_t at, float f) {
#pragma unroll
  for (int c = 0; c < COLS / 16; ++c) {                                     // narrow pieces: scores stay in registers meanwhile
    float o[16];
    tmem_ld_32x32b_x16(at + c * 16, o);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] *= f;
    tmem_st_x16(at + c * 16, o);
  }
}

// Q of a slot: rows of 16-byte chunks in 128-byte swizzle atoms of 64 columns; the slots share the work where there is one half of the rows only.
template <int DA, int VA>
__device__ __forceinline__ void fetch_queries(const TreeParams& p, uint8_t* smem, const Block& b, int slot, int tid) {
  using C = TcCfg<DA, VA>;
  constexpr int CH = DA * 8, STEP = 256 / CH, N = TC_ROWS / STEP;           // a thread has chunk c of every STEP-th row
  const Span s = b.s;
  const int r0 = b.r0 + (b.two ? slot * TC_ROWS : 0), rows = b.rows - (b.two ? slot * TC_ROWS : 0), c = tid % CH, first = tid / CH;
  uint8_t* to = smem + (b.two && slot ? C::X : C::Q) + (c >> 3) * TC_ATOM_BYTES;
  uint4 x[N / 2];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    if (!b.two && part != slot) continue;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const int r = first + (part * (N / 2) + i) * STEP, tr = s.q0 + (r0 + r) / p.G;
      x[i] = make_uint4(0, 0, 0, 0);
      if (r < rows && (unsigned)tr < (unsigned)p.tokens && c * 8 < p.D) {
        const bf16* from = reinterpret_cast<const bf16*>(p.q) + tr * p.q_tok + (long long)(b.h * p.G + (r0 + r) % p.G) * p.q_head + c * 8;
        if (p.q_vec) {
          x[i] = *reinterpret_cast<const uint4*>(from);
        } else {
          const uint16_t* w = reinterpret_cast<const uint16_t*>(from);
          x[i] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const int r = first + (part * (N / 2) + i) * STEP;
      *reinterpret_cast<uint4*>(to + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x[i];
    }
  }
}

template <int DA, int VA, bool CAP>
__device__ __forceinline__ void tree_softmax(const TreeParams& p, TcBars* bars, uint8_t* smem, uint32_t tmem) {
  using C = TcCfg<DA, VA>;
  constexpr int OUT = VA * 32;                                              // output columns of a thread
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = warp >> 3, half = (warp >> 2) & 1, w4 = warp & 3, tid = threadIdx.x & 255, row = w4 * 32 + lane;
  const uint32_t t_s = tmem + ((uint32_t)(w4 * 32) << 16) + slot * 256 + half * 64, t_o = t_s - half * 64 + 128 + half * OUT;
  float* word = reinterpret_cast<float*>(smem + C::EXCHANGE) + slot * (2 * TC_ROWS) + row;
  int steps, by, j, tail;                                                   // tiles of this slot, from one to the next, the first one, the first of the tree
  {
    const Block b = load_block(bars);
    fetch_queries<DA, VA>(p, smem, b, slot, tid);
    steps = b.two ? b.n_tiles : (b.n_tiles - slot + 1) >> 1, by = b.two ? 1 : 2, j = b.two ? 0 : slot, tail = b.tail;
  }
  // token of this thread's row, and whether it is one of the step's
  const auto token_of = [&](const Block& b, bool& mine) {
    const int r = row + (b.two ? slot * TC_ROWS : 0), t = b.s.q0 + (b.r0 + r) / p.G;
    mine = r < b.rows && (unsigned)t < (unsigned)p.tokens;
    return t;
  };
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(&bars->q_full);

  float scale_log2 = p.scale * 1.4426950408889634f, to_cap = 0.f;           // the capped score is cap (1 - 2 / (2^(to_cap s) + 1))
  if constexpr (CAP) to_cap = 2.f * scale_log2 / p.softcap, scale_log2 = 1.4426950408889634f;
  // Handed over instead of a maximum when a wait ran out. A maximum is a number or infinite also where all scores are NaN: -inf is among what it is taken of.
  const float STOP = __int_as_float(0x7fffffff);
  float m = -INFINITY, l = 0.f;
  bool ok = true, whole = true;                                             // whole: no wait inside a tile has run out
  for (int i = 0; i < steps; ++i, j += by) {
    ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[slot], i & 1, &bars->abort, 30 + slot));
    uint32_t x[64];
    float mx = STOP;
    if (ok) {
      tc_fence_after_sync();
      tmem_ld_x32(t_s, x);
      tmem_ld_x32(t_s + 32, x + 32);
      tmem_ld_wait();
      if constexpr (CAP) {
#pragma unroll
        for (int e = 0; e < 64; ++e) x[e] = __float_as_uint(fmaf(-2.f * p.softcap, rcp_approx(ex2(__uint_as_float(x[e]) * to_cap) + 1.f), p.softcap));
      }
      const unsigned dead = bars->dead[j & 15];
      if (j >= tail || dead) {
        const Block b = load_block(bars);
        bool mine;
        const int t = token_of(b, mine);
        const unsigned long long seen = seen_keys(p.mask + (mine ? t : 0) * p.mask_tok, p.words, (b.t_lo + j) * TC_KEYS + half * 64, b.s.base, b.s.len, dead >> half * 4);
#pragma unroll
        for (int e = 0; e < 64; ++e)
          if (!(seen >> e & 1ull)) x[e] = __float_as_uint(-INFINITY);
      }
      float m0 = __uint_as_float(x[0]), m1 = __uint_as_float(x[1]), m2 = __uint_as_float(x[2]), m3 = __uint_as_float(x[3]);
#pragma unroll
      for (int e = 4; e + 7 < 64; e += 8)
        m0 = max3(m0, x[e], x[e + 1]), m1 = max3(m1, x[e + 2], x[e + 3]), m2 = max3(m2, x[e + 4], x[e + 5]), m3 = max3(m3, x[e + 6], x[e + 7]);
      m0 = max3(m0, x[60], x[61]), m1 = max3(m1, x[62], x[63]);
      mx = fmaxf(fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)), -INFINITY);
    }
    // (Its word of the tile before is read by then: this tile's scores wait for that one's weights.)
    word[half * TC_ROWS] = mx;
    pair_sync(1 + slot * 4 + w4);
    const float theirs = word[(half ^ 1) * TC_ROWS];
    const float m_new = fmaxf(fmaxf(mx, theirs), m);
    // Both halves vote on the same two words, so that they leave at the same tile.
    const bool stop = __float_as_int(mx) == 0x7fffffff || __float_as_int(theirs) == 0x7fffffff;
    const bool grow = (m_new - m) * scale_log2 > TC_RESCALE;                // on the first tile with a key that the row sees (m = -inf)
    if (__any_sync(0xffffffffu, grow || stop)) {
      ok = !__any_sync(0xffffffffu, stop);
      if (!ok) {
        pair_sync(1 + slot * 4 + w4);                                       // both have read the words that are written next
        break;
      }
      const float f = grow ? ex2((m - m_new) * scale_log2) : 1.f;
      if (grow) l *= f, m = m_new;
      if (i > 0) scale_columns<OUT>(t_o, f);                                // the product before this one is done: the scores came behind it
    }
    const float neg_m = m == -INFINITY ? 0.f : -m * scale_log2;
    const unsigned long long sc2 = pack2(scale_log2, scale_log2), nm2 = pack2(neg_m, neg_m);
    unsigned long long l0 = 0ull, l1 = 0ull;
#pragma unroll
    // Packed P overwrites the row in place. Weights are rounded to bf16, half a step each, as the product with bf16 values takes both operands in one type: results are off by 0.0023 of their size in place of
    // the 0.0017 that their own rounding to bf16 costs. Two parts of each weight would double that product. Their sum l is of the 32-bit numbers.
    for (int e = 0; e < 64; e += 4) {
      float v0, v1, v2, v3;
      unpack2(fma2(pack2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), sc2, nm2), v0, v1);
      unpack2(fma2(pack2(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])), sc2, nm2), v2, v3);
      v0 = ex2(v0), v1 = ex2(v1), v2 = ex2(v2), v3 = e % 8 == 4 ? ex2_fma(v3) : ex2(v3);        // one in eight beside the special-function unit: 122 us, 115 (one in four 122, in sixteen 117)
      l0 = add2(l0, pack2(v0, v1)), l1 = add2(l1, pack2(v2, v3));
      x[e >> 1] = pack_bf16x2(v0, v1), x[(e >> 1) + 1] = pack_bf16x2(v2, v3);
    }
    float x0, x1;
    unpack2(add2(l0, l1), x0, x1);
    l += x0 + x1;
    tmem_st_x32(t_s, x);
    tmem_st_wait();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->p_full[slot]);
    if (j >= tail && !(by == 1 && slot)) {
      // Values behind the sequence's end are anything, and those of new tokens are not for every row: what is no number becomes a zero in front of the products, and is added
      // to the rows that see it at the end.
      const Block b = load_block(bars);
      const int stages = b.two ? 2 : 3, at_stage = j % stages, tile0 = (b.t_lo + j) * TC_KEYS;
      if (!__all_sync(0xffffffffu, mbar_wait(&bars->v_full[at_stage], (j / stages) & 1, &bars->abort, 35))) {
        whole = false;
        continue;                                                           // the next tile's wait runs out too
      }
      for (int e = tid; e < TC_KEYS * VA * 8; e += 256) {
        const int r = e / (VA * 8), c = e % (VA * 8);
        if (tile0 + r < b.s.base) continue;
        uint4* at = reinterpret_cast<uint4*>(smem + C::V + at_stage * C::VT + (c >> 3) * TC_ATOM_BYTES + r * 128 + ((c & 7) << 4));      // any chunk of the row
        if (tile0 + r >= b.s.len) {
          *at = make_uint4(0, 0, 0, 0);
          continue;
        }
        uint4 v = *at;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
        bool odd = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if ((w[k] & 0x7f80u) == 0x7f80u) w[k] &= 0xffff0000u, odd = true;
          if ((w[k] & 0x7f800000u) == 0x7f800000u) w[k] &= 0xffffu, odd = true;
        }
        if (odd) *at = v, bars->odd = 1;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->v_clean[at_stage]);
    }
  }
  ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_final, 0, &bars->abort, 32 + slot)) && ok && whole;
  word[half * TC_ROWS] = ok ? l : -1.f;                                     // a sum is not below zero, but may be no number
  pair_sync(1 + slot * 4 + w4);
  const float other = word[(half ^ 1) * TC_ROWS], m_used = m;
  ok = ok && __all_sync(0xffffffffu, other != -1.f);
  const Block b = load_block(bars);
  const Span s = b.s;
  bool mine;
  const int t = token_of(b, mine), r0 = b.r0 + (b.two ? slot * TC_ROWS : 0), rows = b.rows - (b.two ? slot * TC_ROWS : 0), head = b.h * p.G + (r0 + row) % p.G;
  tc_fence_after_sync();
  float sum = half ? other + l : l + other, f = 1.f;
  const bool both = !b.two && b.n_tiles > 1;                                // two parts of the same rows
  float4* hand = reinterpret_cast<float4*>(smem + C::V) + tid;              // two idle V tiles: chunk c of a thread at 256 c
  float* hand_ml = reinterpret_cast<float*>(smem + C::BARS - 1024) + row;   // and the end of the last one: of both threads of a row, which have the same
  if (both) {
    if (slot) {
      if (ok) {
#pragma unroll
        for (int c = 0; c < OUT / 16; ++c) {
          float o[16];
          tmem_ld_32x32b_x16(t_o + c * 16, o);
#pragma unroll
          for (int e = 0; e < 4; ++e) hand[(c * 4 + e) * 256] = make_float4(o[e * 4], o[e * 4 + 1], o[e * 4 + 2], o[e * 4 + 3]);
        }
      }
      hand_ml[0] = ok ? m_used : STOP, hand_ml[TC_ROWS] = sum;
    }
    asm volatile("bar.sync 9, 512;" ::: "memory");
    if (slot) return;
    const float m1 = hand_ml[0], l1 = hand_ml[TC_ROWS];
    ok = ok && __all_sync(0xffffffffu, __float_as_int(m1) != 0x7fffffff);
    if (ok) {
      const float top = fmaxf(m_used, m1), base = top == -INFINITY ? 0.f : top;
      f = ex2((m_used - base) * scale_log2);
      const float f1 = ex2((m1 - base) * scale_log2);
      sum = fmaf(f, sum, f1 * l1);
      m = top;
#pragma unroll
      for (int c = 0; c < OUT / 16; ++c) {
        float o[16];
        tmem_ld_32x32b_x16(t_o + c * 16, o);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 y = hand[(c * 4 + e) * 256];
          o[e * 4] = fmaf(f, o[e * 4], f1 * y.x), o[e * 4 + 1] = fmaf(f, o[e * 4 + 1], f1 * y.y);
          o[e * 4 + 2] = fmaf(f, o[e * 4 + 2], f1 * y.z), o[e * 4 + 3] = fmaf(f, o[e * 4 + 3], f1 * y.w);
        }
        tmem_st_x16(t_o + c * 16, o);
      }
      tmem_st_wait();
    }
  } else if (steps == 0) {
    return;
  }
  if (!ok) return;
  const bool odd = bars->odd != 0;
  // values that are no numbers, of new tokens among this block's keys that the row sees: columns from d0 on
  const auto add_odd = [&](uint32_t* o, int d0) {
    const int* table = p.table + b.seq * p.table_stride;
    for (int key = max(b.t_lo * TC_KEYS, max(s.base, 0)); key < min(s.len, (b.t_lo + b.n_tiles) * TC_KEYS); ++key) {
      const int block = table[key / p.bs];
      if (!mine || (unsigned)block >= (unsigned)p.num_blocks || !sees(p.mask + t * p.mask_tok, p.words, key - s.base)) continue;
      const bf16* v = reinterpret_cast<const bf16*>(p.v) + (((long long)block * p.Hkv + b.h) * p.bs + key % p.bs) * p.Dv + d0;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float y = d0 + e < p.Dv ? __bfloat162float(v[e]) : 0.f;
        if (!isfinite(y)) o[e] = __float_as_uint(__uint_as_float(o[e]) + y);
      }
    }
    __syncwarp();
  };
  if (p.part_o) {
    const long long at = ((long long)b.split * p.tokens + t) * (p.Hkv * p.G) + head;
#pragma unroll
    for (int c = 0; c < OUT / 32; ++c) {
      uint32_t o[32];
      tmem_ld_x32(t_o + c * 32, o);
      tmem_ld_wait();
      const int d0 = half * OUT + c * 32;
      if (odd) add_odd(o, d0);
      if (mine) {
        float* to = p.part_o + at * p.Dv + d0;
#pragma unroll
        for (int v = 0; v < 8; ++v)
          if (d0 + v * 4 < p.Dv)
            reinterpret_cast<float4*>(to)[v] = make_float4(__uint_as_float(o[v * 4]), __uint_as_float(o[v * 4 + 1]), __uint_as_float(o[v * 4 + 2]), __uint_as_float(o[v * 4 + 3]));
      }
    }
    if (half == 0 && mine) p.part_ml[at] = make_float2(m == -INFINITY ? -INFINITY : m * scale_log2, sum);
    return;
  }
  // through the idle Q tile (and K's behind it), so that rows are written in runs: 16-byte chunk c of row r lies at c ^ (r & (chunks - 1))
  constexpr int BYTES = OUT * 2, CHUNKS = BYTES / 16;
  static_assert(8 * 32 * BYTES <= C::LAST && 8 * 32 * BYTES <= 4 * C::KT, "a slot's rows fit in front of what the other reads");
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint8_t* slab = smem + (slot ? C::X : C::Q) + (warp & 7) * (32 * BYTES);
#pragma unroll
  for (int c = 0; c < OUT / 32; ++c) {
    uint32_t o[32];
    tmem_ld_x32(t_o + c * 32, o);
    tmem_ld_wait();
    if (odd) add_odd(o, half * OUT + c * 32);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      uint4 u;
      u.x = pack_bf16x2(__uint_as_float(o[v * 8]) * inv, __uint_as_float(o[v * 8 + 1]) * inv);
      u.y = pack_bf16x2(__uint_as_float(o[v * 8 + 2]) * inv, __uint_as_float(o[v * 8 + 3]) * inv);
      u.z = pack_bf16x2(__uint_as_float(o[v * 8 + 4]) * inv, __uint_as_float(o[v * 8 + 5]) * inv);
      u.w = pack_bf16x2(__uint_as_float(o[v * 8 + 6]) * inv, __uint_as_float(o[v * 8 + 7]) * inv);
      *reinterpret_cast<uint4*>(slab + lane * BYTES + (((c * 4 + v) ^ (lane & (CHUNKS - 1))) << 4)) = u;
    }
  }
  __syncwarp();
  bf16* out = reinterpret_cast<bf16*>(p.out);
#pragma unroll
  for (int it = 0; it < CHUNKS; ++it) {                                     // CHUNKS lanes write one row's part
    const int r = (32 / CHUNKS) * it + lane / CHUNKS, ch = lane % CHUNKS, rr = r0 + w4 * 32 + r, to_t = s.q0 + rr / p.G, d = half * OUT + ch * 8;
    if (w4 * 32 + r >= rows || (unsigned)to_t >= (unsigned)p.tokens || d >= p.Dv) continue;
    const uint4 u = *reinterpret_cast<const uint4*>(slab + r * BYTES + ((ch ^ (r & (CHUNKS - 1))) << 4));
    bf16* to = out + to_t * p.out_tok + (long long)(b.h * p.G + rr % p.G) * p.Dv + d;
    if (p.out_vec) {
      *reinterpret_cast<uint4*>(to) = u;
    } else {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = __ushort_as_bfloat16((unsigned short)(w[e >> 1] >> (e & 1) * 16));
    }
  }
}

template <int DA, int VA, bool CAP>
__global__ void __launch_bounds__(TC_THREADS, 1) attn_tree_tc_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const TreeParams p) {
  using C = TcCfg<DA, VA>;
  extern __shared__ __align__(1024) uint8_t smem[];
  TcBars* bars = reinterpret_cast<TcBars*>(smem + C::BARS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  pdl_launch_dependents();
  pdl_wait(TL_ATTN_DECODE);
  // row tiles of a problem are neighbours: they run together and find one another's keys in the second-level cache
  Block b;
  const int tile = blockIdx.x % p.tiles, y = blockIdx.x / p.tiles, z = y / p.num_splits;
  b.split = y % p.num_splits, b.h = z % p.Hkv, b.seq = z / p.Hkv;
  b.s = span_of(p, b.seq);
  b.r0 = tile * 2 * TC_ROWS, b.rows = min(2 * TC_ROWS, min(b.s.n, p.uniform_q) * p.G - b.r0);
  if (b.rows <= 0) return;                                 // uniform, like the next one, in front of all barriers
  b.two = b.rows > TC_ROWS;
  const int all = (b.s.len + TC_KEYS - 1) / TC_KEYS, per = (all + p.num_splits - 1) / p.num_splits;
  b.t_lo = min(b.split * per, all), b.n_tiles = min(all, b.t_lo + per) - b.t_lo, b.tail = max(max(b.s.base, 0) / TC_KEYS - b.t_lo, 0);
  if (b.n_tiles <= 0) {                                    // fewer tiles than splits, or nothing in the cache
    for (int r = threadIdx.x; r < b.rows; r += TC_THREADS) {
      const int t = b.s.q0 + (b.r0 + r) / p.G, head = b.h * p.G + (b.r0 + r) % p.G;
      if ((unsigned)t >= (unsigned)p.tokens) continue;
      if (p.part_o) p.part_ml[((long long)b.split * p.tokens + t) * (p.Hkv * p.G) + head] = make_float2(-INFINITY, 0.f);
      else
        for (int d = 0; d < p.Dv; ++d) reinterpret_cast<bf16*>(p.out)[t * p.out_tok + (long long)head * p.Dv + d] = __float2bfloat16(0.f);
    }
    return;
  }
  static_assert(16 * SOFT_REGS + 4 * ROLE_REGS <= 20 * 96, "registers that the block was launched with");
  const int users = b.two ? 2 : 1, v_stages = b.two ? 2 : 3;
  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 16);
    for (int i = 0; i < K_STAGES; ++i) mbar_init(&bars->k_full[i], 1), mbar_init(&bars->k_empty[i], users);
    for (int i = 0; i < V_STAGES; ++i) mbar_init(&bars->v_full[i], 1), mbar_init(&bars->v_empty[i], users), mbar_init(&bars->v_clean[i], 8);
    for (int i = 0; i < 2; ++i) mbar_init(&bars->s_full[i], 1), mbar_init(&bars->p_full[i], 8);
    mbar_init(&bars->o_final, 2);
    bars->abort = 0, bars->odd = 0, bars->block = b;
    mbar_fence_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&bars->tmem_base, TC_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  if (warp >= TMA_WARP) {
    // Scores and weights of a thread's 64 keys take more registers than a 640th of the SM's: what the other warps do not need goes to the softmax's, 20 * 96 = 16 * SOFT_REGS + 4 * ROLE_REGS at most.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(ROLE_REGS));
    if (warp == TMA_WARP) {
      // lane = group of 16 keys + 8 * swizzle atom of a copy; looked up 32 groups ahead of it, one to a lane
      const int* table = p.table + b.seq * p.table_stride;
      const int g = lane & 7, atom = lane >> 3, none = p.num_blocks * p.Hkv * p.bs;
      const auto look_up = [&](int j) {
        const int key = (b.t_lo + j) * TC_KEYS + lane * 16;
        int row = none;
        if (key < b.s.len) {
          const int block = table[key / p.bs];
          if ((unsigned)block < (unsigned)p.num_blocks) row = (block * p.Hkv + b.h) * p.bs + key % p.bs;
        }
        return row;
      };
      bool ok = true;
      int issued_k = 0, issued_v = 0, rows = 0, ahead = look_up(0);
      Ring k{0, 0}, v{0, 0};
      for (int j = 0; j < b.n_tiles && ok; ++j) {
        if ((j & 3) == 0) rows = ahead, ahead = look_up(j + 4);
        const int row = __shfl_sync(0xffffffffu, rows, (j & 3) * 8 + g);
        const unsigned dead = __ballot_sync(0xffffffffu, row == none) & 0xffu;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->k_empty[k.at], k.round ^ 1, &bars->abort, 10));
        if (!ok) break;
        if (lane == 0) {
          bars->dead[j & 15] = dead;
          mbar_arrive_expect_tx(&bars->k_full[k.at], C::KT);
        }
        __syncwarp();
        if (atom < DA) tma_load_2d(smem + C::K + k.at * C::KT + atom * TC_ATOM_BYTES + g * 2048, &tmap_k, &bars->k_full[k.at], atom * 64, row);
        issued_k = j + 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_empty[v.at], v.round ^ 1, &bars->abort, 11));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&bars->v_full[v.at], C::VT);
        __syncwarp();
        if (atom < VA) tma_load_2d(smem + C::V + v.at * C::VT + atom * TC_ATOM_BYTES + g * 2048, &tmap_v, &bars->v_full[v.at], atom * 64, row);
        issued_v = j + 1;
        k.advance(1, K_STAGES);
        v.advance(1, v_stages);
      }
      if (!ok) {                                             // copies in flight land before the block's memory is released
        volatile int never = 0;
        for (int j = max(0, issued_k - K_STAGES); j < issued_k; ++j) mbar_wait(&bars->k_full[j % K_STAGES], (j / K_STAGES) & 1, &never, 13);
        for (int j = max(0, issued_v - v_stages); j < issued_v; ++j) mbar_wait(&bars->v_full[j % v_stages], (j / v_stages) & 1, &never, 14);
      }
    } else if (warp <= MMA_WARP + 1) {
      constexpr uint32_t IDESC_QK = umma_idesc_bf16_f32(TC_ROWS, TC_KEYS), IDESC_PV = umma_idesc_bf16_f32(TC_ROWS, VA * 64) | (1u << 16);      // V is MN-major
      const int slot = warp - MMA_WARP, steps = b.two ? b.n_tiles : (b.n_tiles - slot + 1) >> 1, by = b.two ? 1 : 2, first = b.two ? 0 : slot;
      const uint64_t qd = umma_desc_kmajor_sw128(smem_u32(smem + (b.two && slot ? C::X : C::Q))), kd = umma_desc_kmajor_sw128(smem_u32(smem + C::K)), vd = umma_desc_mnmajor_sw128(smem_u32(smem + C::V));
      const uint32_t t_s = tmem + slot * 256, t_o = t_s + 128;
      const auto wait = [&](uint64_t* bar, uint32_t parity, int where) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, &bars->abort, where)) != 0; };
      Ring k{first, 0}, v{first, 0};
      const auto scores = [&]() {                            // one lane
#pragma unroll
        for (int e = 0; e < DA * 4; ++e) {
          const uint32_t off = ((e >> 2) * TC_ATOM_BYTES + (e & 3) * 32) >> 4;
          umma_f16_ss(t_s, qd + off, kd + k.at * (C::KT >> 4) + off, IDESC_QK, e > 0);
        }
        umma_commit(&bars->s_full[slot]);
        umma_commit(&bars->k_empty[k.at]);
      };
      bool ok = wait(&bars->q_full, 0, 20);
      if (ok && steps > 0) {
        ok = wait(&bars->k_full[k.at], k.round, 21);
        if (ok) {
          tc_fence_after_sync();
          if (elect_one()) scores();
          __syncwarp();
          k.advance(by, K_STAGES);
        }
      }
      for (int i = 0; i < steps && ok; ++i) {
        const int j = first + i * by;
        const bool more = i + 1 < steps;
        ok = j < b.tail ? wait(&bars->v_full[v.at], v.round, 23) : wait(&bars->v_clean[v.at], (j - b.tail) / v_stages & 1, 23);
        if (ok && more) ok = wait(&bars->k_full[k.at], k.round, 21);
        if (ok) ok = wait(&bars->p_full[slot], i & 1, 24 + slot);
        if (!ok) break;
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int e = 0; e < TC_KEYS / 16; ++e)
            umma_f16_ts(t_o, t_s + (e >> 2) * 64 + (e & 3) * 8, vd + v.at * (C::VT >> 4) + e * (2048 >> 4), IDESC_PV, i > 0 || e > 0);
          umma_commit(&bars->v_empty[v.at]);
          if (more) scores();
        }
        __syncwarp();
        v.advance(by, v_stages);
        k.advance(by, K_STAGES);
      }
      if (elect_one()) umma_commit(&bars->o_final);          // also where a wait ran out: it tracks what has been issued
      __syncwarp();
      if (!ok) {
        volatile int never = 0;
        mbar_wait(&bars->o_final, 0, &never, 27);
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFT_REGS));
    tree_softmax<DA, VA, CAP>(p, bars, smem, tmem);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, TC_COLS);
  }
}

// ---- sum of the splits --------------------------------------------------------------------------------------------------------------------------------
// A warp to a row and head, weighed by the distance of its splits' maxima to the common one; the parts of eight splits are on their way together. VEC: four columns to a lane.
constexpr int JOIN_THREADS = 128, JOIN_AHEAD = 8;

template <typename E, bool VEC>
__global__ void __launch_bounds__(JOIN_THREADS) attn_tree_join_kernel(const TreeParams p) {
  pdl_launch_dependents();
  constexpr int W = VEC ? 4 : 1;
  const int Hq = p.Hkv * p.G, lane = threadIdx.x & 31, S = p.num_splits;
  const long long i = (long long)blockIdx.x * (JOIN_THREADS / 32) + (threadIdx.x >> 5), rows = (long long)p.tokens * Hq;
  pdl_wait(TL_ATTN_MERGE);
  if (i >= rows) return;
  const int t = (int)(i / Hq), head = (int)(i % Hq);
  if (p.cu_q) {
    if (t < p.cu_q[0] || t >= p.cu_q[p.num_seqs]) return;
    const int seq = seq_of_token(p.cu_q, p.num_seqs, p.uniform_q, t);
    if (t - p.cu_q[seq] >= p.uniform_q) return;              // more tokens than the call was told of: not computed
  }
  float2 a = make_float2(-INFINITY, 0.f), b = a;
  if (lane < S) a = __ldcg(p.part_ml + lane * rows + i);
  if (lane + 32 < S) b = __ldcg(p.part_ml + (lane + 32) * rows + i);
  const float top = warp_max(fmaxf(a.x, b.x)), base = top == -INFINITY ? 0.f : top;
  float fa = exp2f(a.x - base), fb = exp2f(b.x - base);
  const float sum = warp_sum(fmaf(fa, a.y, fb * b.y)), inv = sum == 0.f ? 0.f : 1.f / sum;
  fa *= inv, fb *= inv;
  E* out = reinterpret_cast<E*>(p.out) + t * p.out_tok + (long long)head * p.Dv;
  for (int d0 = 0; d0 < p.Dv; d0 += 32 * W) {
    const int d = d0 + lane * W;
    const float* part = p.part_o + i * p.Dv + d;
    float x[W];
#pragma unroll
    for (int k = 0; k < W; ++k) x[k] = 0.f;
    for (int s0 = 0; s0 < S; s0 += JOIN_AHEAD) {
      float y[JOIN_AHEAD][W], f[JOIN_AHEAD];
#pragma unroll
      for (int u = 0; u < JOIN_AHEAD; ++u) {                 // all lanes: each has the factors of two splits
        const int s = s0 + u;
        f[u] = __shfl_sync(0xffffffffu, s < 32 ? fa : fb, s & 31);
        const bool take = s < S && d < p.Dv && f[u] != 0.f;  // of a split without keys nothing was written
        if constexpr (VEC) {
          const float4 v = take ? __ldcg(reinterpret_cast<const float4*>(part + s * rows * p.Dv)) : make_float4(0.f, 0.f, 0.f, 0.f);
          y[u][0] = v.x, y[u][W > 1] = v.y, y[u][W / 2] = v.z, y[u][W - 1] = v.w;
        } else {
          y[u][0] = take ? __ldcg(part + s * rows * p.Dv) : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < JOIN_AHEAD; ++u)
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (f[u] != 0.f) x[k] = fmaf(f[u], y[u][k], x[k]);
    }
    if (d >= p.Dv) continue;
    if (VEC && p.out_vec) {
      store_row4(out + d, make_float4(x[0], x[W > 1], x[W / 2], x[W - 1]));
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k) store_out(out + d + k, x[k]);
    }
  }
}

template <typename E>
int launch_join(TreeParams p, cudaStream_t s) {
  const long long rows = (long long)p.tokens * p.Hkv * p.G;
  p.out_vec = (reinterpret_cast<uintptr_t>(p.out) & (4 * sizeof(E) - 1)) == 0 && p.out_tok % 4 == 0;
  return launch_kernel(p.Dv % 4 == 0 ? attn_tree_join_kernel<E, true> : attn_tree_join_kernel<E, false>, dim3((unsigned)((rows + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32))),
                       dim3(JOIN_THREADS), 0, s, p);
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
int launch_plain(TreeParams p, cudaStream_t s) {
  p.q_vec = reinterpret_cast<uintptr_t>(p.q) % (4 * sizeof(E)) == 0 && p.q_tok % 4 == 0 && p.q_head % 4 == 0;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
  const bool vec = (p.D | p.Dv) % 4 == 0 && at % (4 * sizeof(E)) == 0;
  if (p.Dv <= 64) return vec ? launch_plain<E, 1, true>(p, s) : launch_plain<E, 1, false>(p, s);
  if (p.Dv <= 128) return vec ? launch_plain<E, 2, true>(p, s) : launch_plain<E, 2, false>(p, s);
  return vec ? launch_plain<E, 4, true>(p, s) : launch_plain<E, 4, false>(p, s);
}

template <int DA, int VA, bool CAP>
int launch_tc(const CUtensorMap& k, const CUtensorMap& v, const TreeParams& p, cudaStream_t s) {
  auto kernel = attn_tree_tc_kernel<DA, VA, CAP>;
  constexpr size_t smem = TcCfg<DA, VA>::BYTES;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return -(int)e;
  return launch_kernel(kernel, dim3((unsigned)((long long)p.tiles * p.num_splits * p.Hkv * p.num_seqs)), dim3(TC_THREADS), smem, s, k, v, p);
}

template <bool CAP>
int launch_tc(TreeParams p, cudaStream_t s) {
  p.q_vec = (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && p.q_tok % 8 == 0 && p.q_head % 8 == 0;
  p.out_vec = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.out_tok % 8 == 0;
  CUtensorMap k, v;
  const int rows = p.num_blocks * p.Hkv * p.bs;
  int rc = make_tmap_bf16_2d(&k, p.k, rows, p.D, p.D, 16);
  if (!rc) rc = make_tmap_bf16_2d(&v, p.v, rows, p.Dv, p.Dv, 16);
  if (rc) return rc;
  if (p.D <= 64) return p.Dv <= 64 ? launch_tc<1, 1, CAP>(k, v, p, s) : launch_tc<1, 2, CAP>(k, v, p, s);
  return p.Dv <= 64 ? launch_tc<2, 1, CAP>(k, v, p, s) : launch_tc<2, 2, CAP>(k, v, p, s);
}

// The matrix instructions take widths of whole 16-byte chunks, the copies pages of whole groups of 16 keys; a maximum of products is one of scores where these grow with them.
bool tc_fits(const TreeParams& p, int fp32) {
  return !fp32 && p.D % 8 == 0 && p.Dv % 8 == 0 && p.D <= 128 && p.Dv <= 128 && p.bs % 16 == 0 && p.scale > 0.f && (long long)p.num_blocks * p.Hkv * p.bs < INT_MAX &&
         ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15) == 0;
}

}  // namespace
}  // namespace swb

extern "C" {

// See TreeParams. dims: host int[16] = tokens, num_seqs, tokens of each sequence (with cu_q: at most), table width, blocks, block_size, Hkv, G, D, Dv, words of a mask row, splits,
// fp32, 0, 0, 0; strides: host long long[8] = q token and head, out token, table, mask token, 0, 0, 0. workspace (16-byte aligned), with more
// than one split: 4 splits tokens Hq (Dv + 2) + 16 bytes.
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
  // tiles and the pages that are looked up ahead of them reach up to 1007 keys behind a sequence's end
  if ((long long)p.max_blocks * p.bs > INT_MAX - 1024 || (long long)p.uniform_q * p.G > INT_MAX - 2 * TC_ROWS) return -3;
  p.scale = scale, p.softcap = softcap, p.k = k, p.v = v;
  const bool fast = tc_fits(p, fp32);
  const int tile = fast ? 2 * TC_ROWS : PR;
  p.tiles = (p.uniform_q * p.G + tile - 1) / tile;
  if ((long long)p.tiles * p.num_seqs * p.Hkv > INT_MAX / p.num_splits || (long long)p.tokens * p.Hkv * p.G > INT_MAX) return -3;
  p.q = q, p.out = out, p.table = table, p.cu_q = cu_q, p.kv_lens = kv_lens, p.mask = reinterpret_cast<const unsigned*>(mask);
  p.q_tok = strides[0], p.q_head = strides[1], p.out_tok = strides[2], p.table_stride = strides[3], p.mask_tok = strides[4];
  const long long rows = (long long)p.tokens * p.Hkv * p.G;
  if (p.num_splits > 1) {
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || 4 * rows * p.num_splits * (p.Dv + 2) + 16 > workspace_bytes) return -3;
    p.part_ml = reinterpret_cast<float2*>(workspace);
    p.part_o = reinterpret_cast<float*>(workspace) + (rows * p.num_splits * 2 + 3) / 4 * 4;      // on 16 bytes again
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int rc = fast ? (softcap > 0.f ? launch_tc<true>(p, s) : launch_tc<false>(p, s)) : fp32 ? launch_plain<float>(p, s) : launch_plain<bf16>(p, s);
  if (rc || p.num_splits == 1) return rc;
  return fp32 ? launch_join<float>(p, s) : launch_join<bf16>(p, s);
}

}  // extern "C"
