// Attention of new tokens over a paged cache, each on its own: over the pages that were selected for it, or over the whole cache with the weight that
// every key receives added up.
//
// A problem is up to 16 rows of queries with one key/value head: query heads that share it, of one token, or where tokens of a sequence read the same keys and the
// heads are few, of several tokens. Its keys are dealt out to `num_splits` blocks. A block goes over its keys once with the running maximum and sum of the softmax in
// 32 bits, and is left with an un-normalised sum of values and both. Up to 8 blocks of a problem, where all problems' are 296 at most, are a cluster and join their parts from one
// another's shared memory; otherwise they leave them in the workspace for a second launch. Weights need the maximum and sum over all keys, which are known at
// the end only: the scores are kept (4 bytes a key and query head, beside the keys' and values' 2 (D + Dv) a key) and turned into weights there. With one token a sequence, up to 16
// heads a group and one block or a cluster a problem, the blocks do so themselves; in every other case the second launch does, which adds up those of a key token by token
// and head by head. Every sum has one order, and there are no atomics.
//
// Masked keys (behind what a token sees, on pages that are not there) take no part: their scores are -inf whatever the products were, and
// their values are not multiplied at all, so that what the memory holds there does not matter.
#include "attention_common.cuh"
#include "gemm_tcgen05.cuh"

#include <climits>

namespace swb {
using namespace attn;

SWB_REGISTER_STATUS_UNIT(attn_budget);

namespace {

constexpr int ROWS = 16;                     // of queries in a problem
constexpr int MAX_SPLITS = 64, MAX_CLUSTER = 8, MAX_GROUP = 128;

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
  const int* pages;          // [tokens, Hkv, width]: the problem's pages by their place in the sequence; null: all pages, with weights
  const int* counts;         // [tokens, Hkv]
  int width;
  int num_splits;
  int run;                   // tokens of a problem (more than one only without page lists)
  int cluster;               // the splits of a problem are a cluster
  int weigh_here;            // blocks add their weights themselves
  float* part_o;             // [tokens, Hq, num_splits, Dv], null where blocks or clusters finish the output
  float* part_ml;            // [tokens, Hq, num_splits, 2]: maximum (log2 units) and sum; null where no second launch reads them
  float* scores;             // [tokens, Hq, capacity] in log2 units, where weights are kept
  long long capacity;
  float* weights;            // [num_seqs, Hkv, .], inner stride 1
  long long w_seq, w_head;
  int q_vec, out_vec;        // rows of q are 16-byte aligned, those of out 8-byte
  int whole_rows;            // a TMA box holds whole rows (widths are multiples of 64), else 64 columns
};

// Cached tokens of a sequence; a length that the table has no pages for is the table's end, and the last new token's place is there.
__device__ __forceinline__ int length_of(const BudgetParams& p, int seq) { return min(p.kv_lens[seq], p.max_blocks * p.bs); }

// Rows of q in front of the first sequence's and behind the last one's.
__device__ __forceinline__ bool of_no_sequence(const BudgetParams& p, int t) { return p.cu_q && (t < p.cu_q[0] || t >= p.cu_q[p.num_seqs]); }

// What a query token is: its sequence and the keys it sees.
struct Token {
  int seq, q0, q_len, seen;
};
__device__ __forceinline__ Token token_of(const BudgetParams& p, int t) {
  Token x;
  x.seq = seq_of_token(p.cu_q, p.num_seqs, p.uniform_q, t);
  x.q0 = p.cu_q ? p.cu_q[x.seq] : x.seq * p.uniform_q;
  x.q_len = p.cu_q ? p.cu_q[x.seq + 1] - x.q0 : p.uniform_q;
  x.seen = max(length_of(p, x.seq) - (x.q_len - 1 - (t - x.q0)), 0);
  return x;
}

__device__ __forceinline__ size_t part_at(const BudgetParams& p, int t, int head, int split) { return ((size_t)t * p.Hkv * p.G + head) * p.num_splits + split; }

__device__ __forceinline__ void store_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_out(bf16* p, float x) { *p = __float2bfloat16(x); }

// ---- any types and widths: 32-bit arithmetic on ordinary cores --------------------------------------------------------------------------------------
constexpr int PLAIN_TILE = 32, PLAIN_THREADS = 128, PLAIN_WARPS = PLAIN_THREADS / 32;

__device__ __forceinline__ int plain_ldk(int D) { return (D + 3) / 4 * 4 + 4; }      // lanes with neighbouring keys meet in no bank

// One tile of rows of `width` numbers into shared memory as 32-bit numbers, rows ld apart (a warp a row at a time, eight rows on their way), zeros where a key is masked and
// behind the row's end. VEC: four numbers at a time.
template <typename E, bool VEC>
__device__ __forceinline__ void plain_fetch(float* to, int ld, const E* from, int width, const long long* rows) {
  constexpr int STEP = VEC ? 4 : 1, KEYS = PLAIN_TILE / PLAIN_WARPS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, padded = (width + 3) / 4 * 4;
  for (int d = lane * STEP; d < padded; d += 32 * STEP) {
    float4 x[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const long long row = rows[warp + i * PLAIN_WARPS];
      x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row >= 0 && d < width) {
        if constexpr (VEC) x[i] = load_row4(from + row * width + d);
        else x[i].x = to_f(from[row * width + d]);
      }
    }
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      float* at = to + (warp + i * PLAIN_WARPS) * ld + d;
      if constexpr (VEC) *reinterpret_cast<float4*>(at) = x[i];
      else *at = x[i].x;
    }
  }
}

// R: rows that a problem can have, 4, 8 or 16. COLS * 128 >= Dv.
template <typename E, int COLS, int R, bool VEC>
__global__ void __launch_bounds__(PLAIN_THREADS) attn_budget_plain_kernel(const BudgetParams p) {
  pdl_launch_dependents();
  extern __shared__ __align__(16) float plain_smem[];
  const int ldk = plain_ldk(p.D), D4 = ldk - 4, ldv = (p.Dv + 3) / 4 * 4;
  float* sq = plain_smem;                          // [R][D4], zeros behind a row's end
  float* sk = sq + R * D4;                         // [PLAIN_TILE][ldk]
  float* sv = sk + PLAIN_TILE * ldk;               // [PLAIN_TILE][ldv]
  float* sp = sv + PLAIN_TILE * ldv;               // [PLAIN_TILE][R]
  __shared__ long long s_row[PLAIN_TILE];          // first row of the key's page + its place, -1: masked
  __shared__ float s_m[ROWS], s_l[ROWS], s_alpha[ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.x % p.num_splits, y = blockIdx.x / p.num_splits, hy = y % (p.Hkv * p.head_tiles), t = y / (p.Hkv * p.head_tiles);
  const int h = hy / p.head_tiles, ht = hy % p.head_tiles, g0 = ht * ROWS, rows = min(R, p.G - g0);
  pdl_wait();
  if (of_no_sequence(p, t)) return;
  const Token tok = token_of(p, t);
  const size_t list = (size_t)t * p.Hkv + h;
  const int count = p.pages ? min(max(p.counts[list], 0), p.width) : 0;
  const int total = p.pages ? count * p.bs : tok.seen;
  const int tiles = (total + PLAIN_TILE - 1) / PLAIN_TILE, per = (tiles + p.num_splits - 1) / p.num_splits;
  const int t_lo = split * per, t_hi = min(tiles, t_lo + per);
  const E* q = reinterpret_cast<const E*>(p.q) + t * p.q_stride_tok + (size_t)(h * p.G + g0) * p.q_stride_head;
  for (int r = warp; r < R; r += PLAIN_WARPS)
    for (int d = lane; d < D4; d += 32) sq[r * D4 + d] = r < rows && d < p.D ? to_f(q[r * p.q_stride_head + d]) : 0.f;
  if (tid < ROWS) s_m[tid] = -INFINITY, s_l[tid] = 0.f, s_alpha[tid] = 1.f;
  float o[COLS][R];
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int r = 0; r < R; ++r) o[c][r] = 0.f;
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
    plain_fetch<E, VEC>(sk, ldk, reinterpret_cast<const E*>(p.k), p.D, s_row);
    plain_fetch<E, VEC>(sv, ldv, reinterpret_cast<const E*>(p.v), p.Dv, s_row);
    __syncthreads();
    // lane = key, a warp every fourth row
    constexpr int MINE = R / PLAIN_WARPS;
    float s[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) s[i] = 0.f;
    for (int d = 0; d < D4; d += 4) {
      const float4 k = *reinterpret_cast<const float4*>(sk + lane * ldk + d);
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(sq + (warp + i * PLAIN_WARPS) * D4 + d);
        s[i] = fmaf(x.x, k.x, s[i]), s[i] = fmaf(x.y, k.y, s[i]), s[i] = fmaf(x.z, k.z, s[i]), s[i] = fmaf(x.w, k.w, s[i]);
      }
    }
    const bool live = s_row[lane] >= 0;
    const int j = tile * PLAIN_TILE + lane;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int r = warp + i * PLAIN_WARPS;
      if (r >= rows) {
        sp[lane * R + r] = 0.f;
        continue;
      }
      const float x = live ? score_transform(s[i], p.scale, p.softcap) : -INFINITY;
      if (p.scores && j < total) p.scores[((size_t)t * p.Hkv * p.G + h * p.G + g0 + r) * p.capacity + j] = x;
      const float m0 = s_m[r], m1 = fmaxf(m0, warp_max(x)), base = m1 == -INFINITY ? 0.f : m1;
      const float e = exp2f(x - base), sum = warp_sum(e);
      sp[lane * R + r] = live ? e : 0.f;
      __syncwarp();                                // s_m is read by all lanes before lane 0 writes it
      if (lane == 0) {
        const float alpha = exp2f(m0 - base);
        s_alpha[r] = alpha, s_m[r] = m1, s_l[r] = s_l[r] * alpha + sum;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float alpha = s_alpha[r];
#pragma unroll
      for (int c = 0; c < COLS; ++c) o[c][r] *= alpha;
    }
#pragma unroll 4
    for (int key = 0; key < PLAIN_TILE; ++key) {   // masked keys have zeros in both
      float w[R];
#pragma unroll
      for (int r = 0; r < R; r += 4) *reinterpret_cast<float4*>(w + r) = *reinterpret_cast<const float4*>(sp + key * R + r);
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const int d = c * PLAIN_THREADS + tid;
        const float x = d < p.Dv ? sv[key * ldv + d] : 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) o[c][r] = fmaf(w[r], x, o[c][r]);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rows) break;
    const int head = h * p.G + g0 + r;
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const int d = c * PLAIN_THREADS + tid;
      if (d >= p.Dv) continue;
      if (p.part_o) p.part_o[part_at(p, t, head, split) * p.Dv + d] = o[c][r];
      else store_out(reinterpret_cast<E*>(p.out) + t * p.out_stride_tok + (size_t)head * p.Dv + d, s_l[r] == 0.f ? 0.f : o[c][r] / s_l[r]);
    }
  }
  if (p.part_ml && tid < rows) *reinterpret_cast<float2*>(p.part_ml + part_at(p, t, h * p.G + g0 + tid, split) * 2) = make_float2(s_m[tid], s_l[tid]);
}

// ---- bf16, widths up to 128, pages of 16-key groups: matrix instructions fed by TMA ------------------------------------------------------------------------
//
// Every warp runs on its own: it has a ring of groups of 16 keys (K and V, at most 4 KB each) that it fills with TMA boxes and empties itself, so that no
// warp waits for another before the end. Group i of a block goes to warp i % 4. With queries as rows of 16, S = Q K^T leaves the weights of a head and pairs of
// neighbouring keys in a thread, which is what the second operand of O^T = V^T P^T wants: nothing is moved in between, and heads
// are the 8 columns of that product, so a group of up to 8 query heads wastes none of it.
// A group is some 1300 cycles of a warp's steps behind one another (products 270 and 200, weights 350, the next copies 260); a chain of loads and products whose
// length is not known when compiled took 500 cycles more (selected pages of 500 tokens: 120 us, and 97 with it known), a soft cap's branch at every score 130.
// What a block costs before its first group and behind its last (some 4 us: look-ups that wait for one another, the joining of its warps) is hidden by the other
// blocks of its SM. Rings of three groups leave room for two blocks, rings of two for three; the bytes on their way are the same. Two groups where blocks are many and
// short (500 tokens with 4 key/value heads and 64 pages each: 90 us, 11.7 TB/s through the second-level cache; before the steps were shortened 126, and 165 with two
// blocks), three where they are few (512 blocks of 128 pages: 87 us, 6.2 TB/s, 95 % of what a copy gets; with three blocks the last 68 of them run alone, 96 us). Many are
// nine to an SM: 1600 blocks of 32, 64 and 128 pages take 73, 128 and 241 us with two groups, 77, 134 and 247 with three. Which is the better one in between hangs on how the last
// round of blocks comes out: 512 of 64 pages take 54 and 50 us, 1120 take 93 and 98. 48 sequences of up
// to 8191 keys, 8 key/value heads, in 8 splits: 192 us, 6.4 TB/s, and 17 for their weights. Warps that take equal runs of all problems' keys one behind the other, and fill
// their rings across problems, took 112 us where these took 94: SMs differ in what they get of a busy memory, and nothing evens that out then.
constexpr int FW = 4;                               // warps
constexpr int HALF_BYTES = 2048, GROUP_BYTES = 4 * HALF_BYTES;      // 16 rows of 64 columns; K low, K high, V low, V high
constexpr int SQ_BYTES = ROWS * 256, LDO = 132;
constexpr int fast_smem_bytes(int FS) { return 1024 + FW * FS * GROUP_BYTES + SQ_BYTES + 256; }
constexpr int FINISH_FLOATS = FW * ROWS * LDO + FW * ROWS * 2 + ROWS * 2 + ROWS * 2 + ROWS * MAX_CLUSTER + ROWS * FW;
static_assert(FINISH_FLOATS * 4 <= FW * 2 * GROUP_BYTES, "the warps' results fit where the ring was");

// 16-byte chunk c (0..15) of row r (0..15) of a K or V group: two boxes of 64 columns with the 128-byte swizzle
__device__ __forceinline__ uint32_t group_off(int r, int c) { return (uint32_t)(((c >> 3) << 11) + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }
__device__ __forceinline__ uint32_t q_off(int r, int c) { return (uint32_t)(r * 256 + ((c ^ (r & 7)) << 4)); }

// Values behind the first `live` rows of a group are not multiplied: whole warp.
__device__ __forceinline__ void zero_values(uint8_t* group, int live, int halves, int lane) {
  for (int j = lane; j < (16 - live) * 8 * halves; j += 32) {
    const int half = j / ((16 - live) * 8), at = j % ((16 - live) * 8);
    *reinterpret_cast<uint4*>(group + (2 + half) * HALF_BYTES + live * 128 + at * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();                         // the next copy into the group comes behind these writes
  __syncwarp();
}

// Whether all values of rows from..to - 1 of a group are finite: whole warp.
__device__ __forceinline__ bool finite_values(const uint8_t* group, int from, int to, int halves, int lane) {
  bool finite = true;
  for (int half = 0; half < halves; ++half)
    for (int j = lane; j < (to - from) * 8; j += 32) {
      const uint4 x = *reinterpret_cast<const uint4*>(group + (2 + half) * HALF_BYTES + from * 128 + j * 16);
#pragma unroll
      for (const uint32_t w : {x.x, x.y, x.z, x.w}) finite = finite && (w & 0x7f80u) != 0x7f80u && (w & 0x7f800000u) != 0x7f800000u;
    }
  return __all_sync(0xffffffffu, finite);
}

// 2^x for x <= 0 within 2 ulp, as exp2f, which took 1 to 4 % longer; weights below 2^-126 of the largest are zeros.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cluster(uint32_t at, int rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(rank));
  return remote;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t at) {
  float2 x;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t at) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
  return x;
}

// NT: eights of rows, 1 or 2; FS: groups in a warp's ring, 3 or 2; WIDE: keys and values are 128 wide, so that all steps of a product are known and its loads run ahead
template <int NT, int FS, bool WIDE>
__global__ void __launch_bounds__(FW * 32, FS == 2 && NT == 1 ? 3 : 2) attn_budget_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const BudgetParams p) {
  pdl_launch_dependents();
  extern __shared__ uint8_t fast_smem[];
  uint8_t* smem = fast_smem + ((1024u - (smem_u32(fast_smem) & 1023u)) & 1023u);
  uint8_t* sQ = smem + FW * FS * GROUP_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sQ + SQ_BYTES);
  volatile int* s_abort = reinterpret_cast<volatile int*>(bars + FW * FS);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* ring = smem + warp * FS * GROUP_BYTES;
  uint64_t* full = bars + warp * FS;
  if (tid == 0) {
    for (int i = 0; i < FW * FS; ++i) mbar_init(&bars[i], 1);
    *s_abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  __syncthreads();
  pdl_wait(TL_ATTN_DECODE);
  const int S = p.num_splits, split = blockIdx.x % S, y = blockIdx.x / S, per_token = p.Hkv * p.head_tiles, hy = y % per_token;
  const int h = hy / p.head_tiles, g0 = hy % p.head_tiles * ROWS, heads = min(ROWS, p.G - g0);      // heads of a token
  int t = y / per_token, tokens = 1;                // first token, and how many
  Token tok;
  if (p.run == 1) {
    if (of_no_sequence(p, t)) return;
    tok = token_of(p, t);
  } else {
    const int runs = (p.uniform_q - 1) / p.run + 1;
    tok.seq = t / runs;
    const int q0 = p.cu_q ? p.cu_q[tok.seq] : tok.seq * p.uniform_q, q1 = p.cu_q ? p.cu_q[tok.seq + 1] : q0 + p.uniform_q;
    t = q0 + t % runs * p.run;
    tokens = min(p.run, min(q1, p.tokens) - t);
    if (tokens <= 0 || t < 0) return;
    tok.seen = max(length_of(p, tok.seq) - (q1 - t - tokens), 0);            // of the last token
  }
  const int rows = heads * tokens;                  // row r: token r / heads, head r % heads
  const int sub = p.bs >> 4;                        // groups of a page
  const size_t list = (size_t)t * p.Hkv + h;
  const int* pages = p.pages ? p.pages + list * p.width : nullptr;
  const int groups = p.pages ? min(max(p.counts[list], 0), p.width) * sub : (tok.seen + 15) >> 4;
  const int per = (groups + S - 1) / S, lo = min(split * per, groups), n = min(groups, lo + per) - lo;
  const int mine = n > warp ? (n - warp + FW - 1) / FW : 0;
  const int k_halves = (p.D + 63) >> 6, v_halves = (p.Dv + 63) >> 6, boxes = k_halves + v_halves;
  const int* table = p.table + tok.seq * p.table_stride;

  // Rows of this warp's groups i0..i0 + 31, one to a lane, and how many keys from the group's first on the last token sees (what it sees behind the group counts
  // up to 16: a row of a token before it sees less).
  int row_l = 0, live_l = 0;
  const auto locate = [&](int i0) {
    const int i = i0 + lane;
    live_l = 0;
    if (i < mine) {
      const int g = lo + warp + i * FW, page = pages ? pages[g / sub] : g / sub, off = (g % sub) * 16;
      if (page >= 0 && page < p.max_blocks) {
        const int block = table[page];
        live_l = (unsigned)block < (unsigned)p.num_blocks ? max(0, min(16 + ROWS, tok.seen - (page * p.bs + off))) : 0;
        row_l = (block * p.Hkv + h) * p.bs + off;
      }
    }
  };
  int live_st = 0;                                  // lane s: live keys of the group in stage s
  const auto issue = [&](int i, int stage) {
    if (i >= mine) return;
    if ((i & 31) == 0) locate(i);
    const int row = __shfl_sync(0xffffffffu, row_l, i & 31), live = __shfl_sync(0xffffffffu, live_l, i & 31);
    if (lane == stage) live_st = live;
    if (live == 0) return;                          // nothing is read of a group without live keys
    if (lane == 0) mbar_arrive_expect_tx(&full[stage], (uint32_t)boxes * HALF_BYTES);
    if (p.whole_rows) {
      if (lane == 0) {
        tma_load_3d(ring + stage * GROUP_BYTES, &tmap_k, &full[stage], 0, row, 0);
        tma_load_3d(ring + stage * GROUP_BYTES + 2 * HALF_BYTES, &tmap_v, &full[stage], 0, row, 0);
      }
      return;
    }
    __syncwarp();
    if (lane < boxes) {
      const bool is_k = lane < k_halves;
      const int half = is_k ? lane : lane - k_halves;
      tma_load_2d(ring + stage * GROUP_BYTES + (is_k ? 0 : 2 * HALF_BYTES) + half * HALF_BYTES, is_k ? &tmap_k : &tmap_v, &full[stage], half * 64, row);
    }
  };
#pragma unroll
  for (int i = 0; i < FS; ++i) issue(i, i);

  const bf16* q = reinterpret_cast<const bf16*>(p.q) + t * p.q_stride_tok + (size_t)(h * p.G + g0) * p.q_stride_head;
  for (int i = tid; i < ROWS * 16; i += FW * 32) {
    const int r = i >> 4, c = i & 15;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (r < rows && c * 8 < p.D) {
      const bf16* from = q + r / heads * p.q_stride_tok + r % heads * p.q_stride_head + c * 8;
      if (p.q_vec) {
        x = *reinterpret_cast<const uint4*>(from);
      } else {
        const uint16_t* w = reinterpret_cast<const uint16_t*>(from);
        x = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
      }
    }
    *reinterpret_cast<uint4*>(sQ + q_off(r, c)) = x;
  }
  __syncthreads();
  const int gr = lane >> 2, t4 = lane & 3, mi = lane >> 3;
  uint32_t qf[8][4];
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    ldsm_x4(smem_u32(sQ) + q_off((mi & 1) * 8 + (lane & 7), kk * 2 + (mi >> 1)), qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
    if (NT == 1) qf[kk][1] = qf[kk][3] = 0u;        // rows 8..15 are no heads
  }
  const int k_steps = WIDE ? 8 : (p.D + 15) >> 4, v_steps = WIDE ? 8 : (p.Dv + 15) >> 4;

  float o[NT][8][4], m[NT], l[NT];
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    m[x] = -INFINITY, l[x] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[x][i][0] = o[x][i][1] = o[x][i][2] = o[x][i][3] = 0.f;
  }
  float* score[NT];                                 // of this lane's rows, at the block's first key
  int behind[NT];                                   // keys that the problem's last token sees and this lane's row does not
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    const int r = gr + 8 * x;
    score[x] = p.scores && r < rows ? p.scores + ((size_t)(t + r / heads) * p.Hkv * p.G + h * p.G + g0 + r % heads) * p.capacity + (size_t)lo * 16 : nullptr;
    behind[x] = r < rows ? tokens - 1 - r / heads : 0;
  }
  uint32_t phases = 0;
  int stage = 0;
  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    const int live = __shfl_sync(0xffffffffu, live_st, stage);
    if (live > 0) {
      if (!mbar_wait(&full[stage], (phases >> stage) & 1u, s_abort, 700 + stage)) {
        ok = false;
        break;
      }
      phases ^= 1u << stage;
      if (lane == stage) live_st = 0;               // nothing in flight there
      const uint32_t sK = smem_u32(ring + stage * GROUP_BYTES), sV = sK + 2 * HALF_BYTES;
      if (live < 16) zero_values(ring + stage * GROUP_BYTES, live, v_halves, lane);
      float s[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        if (kk >= k_steps) break;
        uint32_t b0, b1, b2, b3;
        ldsm_x4(sK + group_off((mi >> 1) * 8 + (lane & 7), kk * 2 + (mi & 1)), b0, b1, b2, b3);
        mma_16816(s[0], qf[kk], b0, b1);
        mma_16816(s[1], qf[kk], b2, b3);
      }
      uint32_t pf[NT][2];
      float v[NT][4], base[NT];                     // keys 2 t4, 2 t4 + 1, 8 + 2 t4, 9 + 2 t4 of head gr + 8 x
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[x][e] = s[e >> 1][2 * x + (e & 1)];
      if (p.softcap > 0.f) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[x][e] = score_transform(v[x][e], p.scale, p.softcap);
      } else {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[x][e] = score_transform(v[x][e], p.scale, 0.f);
      }
      if (live - (tokens - 1) < 16) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((e >> 1) * 8 + t4 * 2 + (e & 1) >= live - behind[x]) v[x][e] = -INFINITY;
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        if (score[x]) {
          float* to = score[x] + (size_t)(warp + i * FW) * 16 + t4 * 2;
          *reinterpret_cast<float2*>(to) = make_float2(v[x][0], v[x][1]);
          *reinterpret_cast<float2*>(to + 8) = make_float2(v[x][2], v[x][3]);
        }
        base[x] = fmaxf(fmaxf(v[x][0], v[x][1]), fmaxf(v[x][2], v[x][3]));
      }
      bool more = false;
#pragma unroll
      for (int x = 0; x < NT; ++x) base[x] = fmaxf(base[x], __shfl_xor_sync(0xffffffffu, base[x], 1));
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        base[x] = fmaxf(m[x], fmaxf(base[x], __shfl_xor_sync(0xffffffffu, base[x], 2)));
        more = more || base[x] > m[x];
      }
      if (__any_sync(0xffffffffu, more)) {          // otherwise every factor is one
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          const float alpha = exp2f(m[x] - (base[x] == -INFINITY ? 0.f : base[x]));
          m[x] = base[x];
          l[x] *= alpha;
          const float a0 = __shfl_sync(0xffffffffu, alpha, t4 * 8), a1 = __shfl_sync(0xffffffffu, alpha, t4 * 8 + 4);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[x][j][0] *= a0, o[x][j][1] *= a1, o[x][j][2] *= a0, o[x][j][3] *= a1;
        }
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        if (base[x] == -INFINITY) base[x] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[x][e] = exp2_fast(v[x][e] - base[x]);
        l[x] += (v[x][0] + v[x][1]) + (v[x][2] + v[x][3]);
        // The product takes its weights in bf16 (half a step, 2^-8 of each at most): bf16 cases come within 2.1e-3 of the result in 64 bits, and within 1.65e-3, the rounding of the
        // result alone, with weights in 32 bits, which the matrix instructions have no form for beside bf16 values. The sum that divides them keeps its 32 bits, so that it is the
        // one of the weights that are handed out.
        pf[x][0] = pack_bf16(v[x][0], v[x][1]), pf[x][1] = pack_bf16(v[x][2], v[x][3]);
      }
      // Keys that some of the tokens do not see weigh nothing for those, which is enough where their values are numbers.
      if (live - (tokens - 1) >= 16 || tokens == 1 || finite_values(ring + stage * GROUP_BYTES, max(live - (tokens - 1), 0), min(live, 16), v_halves, lane)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= v_steps) break;
          uint32_t a[4];
          ldsm_x4_trans(sV + group_off((mi >> 1) * 8 + (lane & 7), j * 2 + (mi & 1)), a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int x = 0; x < NT; ++x) mma_16816(o[x][j], a, pf[x][0], pf[x][1]);
        }
      } else {
        // Each token has a product of its own, behind which the values that only later ones see are zeros, and takes its own columns from it.
        for (int i = tokens - 1; i >= 0; --i) {
          const int own = max(live - (tokens - 1 - i), 0);
          if (own < 16) zero_values(ring + stage * GROUP_BYTES, own, v_halves, lane);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j >= v_steps) break;
            uint32_t a[4];
            ldsm_x4_trans(sV + group_off((mi >> 1) * 8 + (lane & 7), j * 2 + (mi & 1)), a[0], a[1], a[2], a[3]);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              mma_16816(c, a, pf[x][0], pf[x][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((8 * x + t4 * 2 + (e & 1)) / heads == i) o[x][j][e] += c[e];
            }
          }
          __syncwarp();
        }
      }
      __syncwarp();                                 // every lane has read the stage
    } else {
#pragma unroll
      for (int x = 0; x < NT; ++x)
        if (score[x]) {                             // a page that is not there: its keys weigh nothing
          float* to = score[x] + (size_t)(warp + i * FW) * 16 + t4 * 2;
          *reinterpret_cast<float2*>(to) = *reinterpret_cast<float2*>(to + 8) = make_float2(-INFINITY, -INFINITY);
        }
    }
    issue(i + FS, stage);
    if (++stage == FS) stage = 0;
  }
  if (!ok) {                                        // a wait ran out: let the copies in flight land before the memory goes away
    for (int s = 0; s < FS; ++s)
      for (int it = 0; __shfl_sync(0xffffffffu, live_st, s) > 0 && it < (1 << 20); ++it)
        if (mbar_try_wait(&full[s], (phases >> s) & 1u)) break;
  }
  __syncthreads();                                  // the rings are free
  float* sO = reinterpret_cast<float*>(smem);       // [FW][ROWS][LDO]
  float* sM = sO + FW * ROWS * LDO;                 // [FW][ROWS][2]
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    float sum = l[x];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (t4 == 0) *reinterpret_cast<float2*>(sM + (warp * ROWS + gr + 8 * x) * 2) = make_float2(m[x], sum);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sO[(warp * ROWS + 8 * x + t4 * 2 + (e & 1)) * LDO + j * 16 + gr + (e >> 1) * 8] = o[x][j][e];
  }
  __syncthreads();
  float* sPart = sM + FW * ROWS * 2;                // [ROWS][2]: the block's maximum and sum
  float* sAll = sPart + ROWS * 2;                   // [ROWS][2]: the problem's maximum, 1 / sum
  float* sFactor = sAll + ROWS * 2;                 // [ROWS][MAX_CLUSTER]
  float* sWarps = sFactor + ROWS * MAX_CLUSTER;     // [ROWS][FW]
  const auto token_at = [&](int r) { return t + r / heads; };
  const auto head_at = [&](int r) { return h * p.G + g0 + r % heads; };
  const bool parts = p.part_o != nullptr;
  bf16* out = reinterpret_cast<bf16*>(p.out);
  if (tid < rows) {                                 // a row's warps, weighed by their distance to the common maximum
    float m_of[FW], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < FW; ++w) M = fmaxf(M, m_of[w] = sM[(w * ROWS + tid) * 2]);
    const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < FW; ++w) L = fmaf(m_of[w] = exp2f(m_of[w] - base), sM[(w * ROWS + tid) * 2 + 1], L);
    const float inv = L == 0.f ? 0.f : 1.f / L, f = !parts && S == 1 ? inv : 1.f;
    *reinterpret_cast<float4*>(sWarps + tid * 4) = make_float4(m_of[0] * f, m_of[1] * f, m_of[2] * f, m_of[3] * f);
    sPart[tid * 2] = M, sPart[tid * 2 + 1] = L;
    sAll[tid * 2] = base, sAll[tid * 2 + 1] = inv;
    if (p.part_ml) *reinterpret_cast<float2*>(p.part_ml + part_at(p, token_at(tid), head_at(tid), split) * 2) = make_float2(M, L);
  }
  __syncthreads();
  const int d = lane * 4;                           // a row to a warp, four columns to a lane
  const auto store = [&](int r, float4 x) {
    bf16* to = out + token_at(r) * p.out_stride_tok + (size_t)head_at(r) * p.Dv + d;
    if (p.out_vec) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
    else to[0] = __float2bfloat16(x.x), to[1] = __float2bfloat16(x.y), to[2] = __float2bfloat16(x.z), to[3] = __float2bfloat16(x.w);
  };
#pragma unroll 4
  for (int r = warp; r < rows; r += FW) {
    if (d >= p.Dv) break;
    const float4 f = *reinterpret_cast<const float4*>(sWarps + r * 4);
    float4* at = reinterpret_cast<float4*>(sO + r * LDO + d);
    const float4 x0 = at[0], x1 = at[ROWS * LDO / 4], x2 = at[2 * ROWS * LDO / 4], x3 = at[3 * ROWS * LDO / 4];
    const auto sum = [&](float a, float b, float c, float e) { return fmaf(f.x, a, f.y * b) + fmaf(f.z, c, f.w * e); };
    const float4 x = make_float4(sum(x0.x, x1.x, x2.x, x3.x), sum(x0.y, x1.y, x2.y, x3.y), sum(x0.z, x1.z, x2.z, x3.z), sum(x0.w, x1.w, x2.w, x3.w));
    if (parts) {
      float2* to = reinterpret_cast<float2*>(p.part_o + part_at(p, token_at(r), head_at(r), split) * p.Dv + d);
      to[0] = make_float2(x.x, x.y), to[1] = make_float2(x.z, x.w);
    } else if (S == 1) {
      store(r, x);
    } else {
      at[0] = x;                                    // warp 0's, which this thread alone reads
    }
  }
  if (parts) return;
  if (S > 1) {
    cluster_barrier();
    if (tid < rows) {
      float m_of[MAX_CLUSTER], l_of[MAX_CLUSTER], M = -INFINITY, L = 0.f;
#pragma unroll
      for (int s = 0; s < MAX_CLUSTER; ++s) {
        m_of[s] = -INFINITY, l_of[s] = 0.f;
        if (s < S) {
          const uint32_t at = in_cluster(smem_u32(sPart + tid * 2), s);
          const float2 x = ld_cluster2(at);
          m_of[s] = x.x, l_of[s] = x.y;
        }
        M = fmaxf(M, m_of[s]);
      }
      const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int s = 0; s < MAX_CLUSTER; ++s) L = fmaf(m_of[s] = exp2f(m_of[s] - base), l_of[s], L);
      const float inv = L == 0.f ? 0.f : 1.f / L;
      sAll[tid * 2] = base, sAll[tid * 2 + 1] = inv;
#pragma unroll
      for (int s = 0; s < MAX_CLUSTER; ++s) sFactor[tid * MAX_CLUSTER + s] = m_of[s] * inv;
    }
    __syncthreads();
#pragma unroll 2
    for (int r = split + S * warp; r < rows; r += S * FW) {
      if (d >= p.Dv) break;
      const uint32_t at = smem_u32(sO + r * LDO + d);
      float4 o_of[MAX_CLUSTER], x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < MAX_CLUSTER; ++s) o_of[s] = s < S ? ld_cluster4(in_cluster(at, s)) : x;
#pragma unroll
      for (int s = 0; s < MAX_CLUSTER; ++s) {
        const float f = sFactor[r * MAX_CLUSTER + s];
        x.x = fmaf(f, o_of[s].x, x.x), x.y = fmaf(f, o_of[s].y, x.y), x.z = fmaf(f, o_of[s].z, x.z), x.w = fmaf(f, o_of[s].w, x.w);
      }
      store(r, x);
    }
  }
  if (p.weigh_here) {                               // one token: row r is head r, and the block's scores are its own writes
    float* w = p.weights + tok.seq * p.w_seq + h * p.w_head;
    const float* from = p.scores + ((size_t)t * p.Hkv * p.G + h * p.G) * p.capacity;
    const int end = min((lo + n) * 16, tok.seen);
    for (int j0 = lo * 16 + tid; j0 < end; j0 += 4 * FW * 32) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
      for (int r = 0; r < rows; ++r) {
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = j0 + k * FW * 32 < end ? from[r * p.capacity + j0 + k * FW * 32] : -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (x[k] != -INFINITY) sum[k] = fmaf(exp2_fast(x[k] - sAll[r * 2]), sAll[r * 2 + 1], sum[k]);      // a key that is not there gets nothing of the row, whatever its sum is
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (j0 + k * FW * 32 < end) w[j0 + k * FW * 32] += sum[k];
    }
  }
  if (S > 1) cluster_barrier();                     // nobody's shared memory goes away while another block reads it
}

bool fast_fits(const BudgetParams& p, int fp32) {
  return !fp32 && p.D % 8 == 0 && p.Dv % 8 == 0 && p.D <= 128 && p.Dv <= 128 && p.bs % 16 == 0 && (long long)p.num_blocks * p.Hkv * p.bs <= INT_MAX &&
         ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15) == 0;
}

int launch_fast(BudgetParams p, cudaStream_t s) {
  p.out_vec = (reinterpret_cast<uintptr_t>(p.out) & 7) == 0 && p.out_stride_tok % 4 == 0;
  p.q_vec = (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && p.q_stride_tok % 8 == 0 && p.q_stride_head % 8 == 0;
  CUtensorMap tk, tv;
  const int rows = p.num_blocks * p.Hkv * p.bs;
  p.whole_rows = (p.D | p.Dv) % 64 == 0;
  const auto make_tmap = p.whole_rows ? make_tmap_bf16_blocks : make_tmap_bf16_2d;
  int rc = make_tmap(&tk, p.k, rows, p.D, p.D, 16);
  if (rc) return rc;
  rc = make_tmap(&tv, p.v, rows, p.Dv, p.Dv, 16);
  if (rc) return rc;
  const bool one = p.G * p.run <= 8, wide = p.D == 128 && p.Dv == 128;
  const int problems = (p.run > 1 ? p.num_seqs * ((p.uniform_q - 1) / p.run + 1) : p.tokens) * p.Hkv * p.head_tiles;
  const bool many = one && (long long)problems * p.num_splits >= 9 * 148;      // measured at the kernel
  const int smem = fast_smem_bytes(many ? 2 : 3), which = (many ? 2 : one) + 3 * wide;
  using Kernel = decltype(&attn_budget_kernel<1, 2, true>);
  static constexpr Kernel kernels[6] = {attn_budget_kernel<2, 3, false>, attn_budget_kernel<1, 3, false>, attn_budget_kernel<1, 2, false>,
                                        attn_budget_kernel<2, 3, true>, attn_budget_kernel<1, 3, true>, attn_budget_kernel<1, 2, true>};
  const Kernel kernel = kernels[which];
  static bool configured[6][64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[which][dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return -(int)e;
    if (dev >= 0 && dev < 64) configured[which][dev] = true;
  }
  const dim3 grid(p.num_splits * problems), block(FW * 32);
  if (!p.cluster) return launch_kernel(kernel, grid, block, smem, s, tk, tv, p);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.num_splits, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tk, tv, p);
  return e == cudaSuccess ? 0 : -(int)e;
}

// ---- joining ------------------------------------------------------------------------------------------------------------------------------------------
constexpr int JOIN_THREADS = 128;
static_assert(MAX_GROUP <= JOIN_THREADS, "a block weighs a row to a thread");

// {maximum, sum} of a row in each of its splits -> factors of the splits' values, exp2(max - common) / sum; by one warp.
__device__ __forceinline__ void split_factors(const float* ml, int S, int lane, float* factor) {
  float m[2], l[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = lane + 32 * i;
    const float2 x = s < S ? __ldcg(reinterpret_cast<const float2*>(ml) + s) : make_float2(-INFINITY, 0.f);
    m[i] = x.x, l[i] = x.y;
  }
  const float M = warp_max(fmaxf(m[0], m[1])), base = M == -INFINITY ? 0.f : M;
  const float e0 = exp2f(m[0] - base), e1 = exp2f(m[1] - base);
  const float L = warp_sum(fmaf(e0, l[0], e1 * l[1])), inv = L == 0.f ? 0.f : 1.f / L;
  if (lane < S) factor[lane] = e0 * inv;
  if (lane + 32 < S) factor[lane + 32] = e1 * inv;
}

// The first `join_blocks` blocks join the parts of one row each; the others weigh keys of one (sequence, key/value head) each, V neighbouring ones to a lane. SPLIT: the
// block's warps share 32 V keys and each takes a part of the rows, whose sums are added up in one order (16 tokens, 4 heads of a group, 6001 keys: 20 us with a key to a
// lane and all 64 rows one behind the other, 7 so); else each warp has keys of its own. Rows are then few and blocks many and short: an SM holds 16 of them, so that
// their look-ups hide one another (48 sequences of up to 8191 keys, 8 key/value heads of 4 heads: 21 us with 8 blocks, 17 with 16).
template <typename E, int V, bool SPLIT>
__global__ void __launch_bounds__(JOIN_THREADS, SPLIT ? 1 : 16) attn_budget_finish_kernel(const BudgetParams p, int join_blocks) {
  pdl_launch_dependents();
  constexpr int WARPS = JOIN_THREADS / 32, RUN = 32 * V * (SPLIT ? 1 : WARPS), U = V == 1 ? 16 : SPLIT ? 8 : 2;      // U: rows whose scores are on their way together
  __shared__ float s_factor[MAX_SPLITS];
  __shared__ __align__(8) float s_all[MAX_GROUP * 2];
  __shared__ size_t s_row[MAX_GROUP];
  __shared__ int s_seen[MAX_GROUP];
  __shared__ float s_sum[WARPS][32 * V];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, S = p.num_splits, Hq = p.Hkv * p.G;
  pdl_wait();
  if ((int)blockIdx.x < join_blocks) {
    const int t = blockIdx.x / Hq, head = blockIdx.x % Hq;
    if (of_no_sequence(p, t)) return;
    if (warp == 0) split_factors(p.part_ml + part_at(p, t, head, 0) * 2, S, lane, s_factor);
    __syncthreads();
    for (int d = tid; d < p.Dv; d += JOIN_THREADS) {
      const float* o = p.part_o + part_at(p, t, head, 0) * p.Dv + d;
      float x = 0.f;
#pragma unroll 16
      for (int s = 0; s < S; ++s) x = fmaf(s_factor[s], __ldcg(o + (size_t)s * p.Dv), x);
      store_out(reinterpret_cast<E*>(p.out) + t * p.out_stride_tok + (size_t)head * p.Dv + d, x);
    }
    return;
  }
  const int blocks = (int)((p.capacity + RUN - 1) / RUN), i = blockIdx.x - join_blocks;
  const int h = i / blocks % p.Hkv, seq = i / blocks / p.Hkv;
  const int first = i % blocks * RUN, at = ((SPLIT ? 0 : warp * 32) + lane) * V;      // of the block, and of this lane behind it
  const int q0 = max(p.cu_q ? p.cu_q[seq] : seq * p.uniform_q, 0), q1 = p.cu_q ? p.cu_q[seq + 1] : q0 + p.uniform_q;
  const int q_end = q0 + min(min(q1, p.tokens) - q0, p.uniform_q);      // tokens whose scores are there
  const int len = length_of(p, seq);
  if (first >= len) return;
  const int room = len - first - at;
  const size_t j0 = (size_t)first + at;
  float* w = p.weights + seq * p.w_seq + h * p.w_head + j0;
  const bool whole = V == 4 && room >= 4 && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  float sum[V], old[V];
#pragma unroll
  for (int k = 0; k < V; ++k) sum[k] = 0.f, old[k] = 0.f;
  if (!SPLIT || warp == 0) {
    if (whole) {
      const float4 x = *reinterpret_cast<const float4*>(w);
      old[0] = x.x, old[V > 1] = x.y, old[V / 2] = x.z, old[V - 1] = x.w;
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) old[k] = k < room ? w[k] : 0.f;
    }
  }
  constexpr int STEP = SPLIT ? WARPS : 1;
  const int batch = MAX_GROUP / p.G;             // tokens whose rows a block has room for
  for (int t0 = q0; t0 < q_end; t0 += batch) {
    const int pairs = min(batch, q_end - t0) * p.G;
    __syncthreads();
    if (tid < pairs) {                           // MAX_GROUP <= JOIN_THREADS: a row to a thread
      const int tok = tid / p.G;
      s_row[tid] = ((size_t)(t0 + tok) * Hq + h * p.G + tid % p.G) * p.capacity;
      s_seen[tid] = len - (q1 - 1 - t0 - tok);
    }
    __syncthreads();
    float x[U][V];
    const auto load = [&](int r0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = min(r0 + u * STEP, pairs - 1), left = r0 + u * STEP < pairs ? s_seen[r] - first - at : 0;      // keys that the row sees; behind them nothing is written
        if constexpr (V == 4) {
          const float4 y = left > 0 ? __ldcg(reinterpret_cast<const float4*>(p.scores + s_row[r] + j0)) : make_float4(0.f, 0.f, 0.f, 0.f);
          x[u][0] = left > 0 ? y.x : -INFINITY, x[u][1] = left > 1 ? y.y : -INFINITY, x[u][2] = left > 2 ? y.z : -INFINITY, x[u][3] = left > 3 ? y.w : -INFINITY;
        } else {
          x[u][0] = left > 0 ? __ldcg(p.scores + s_row[r] + j0) : -INFINITY;
        }
      }
    };
    int r0 = SPLIT ? warp : 0;
    if constexpr (SPLIT) load(r0);               // on their way while the rows' sums are
    if (tid < pairs) {
      const int tok = tid / p.G;
      const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + part_at(p, t0 + tok, h * p.G + tid % p.G, 0);
      float M = -INFINITY, L = 0.f;
      for (int s0 = 0; s0 < S; s0 += 8) {
        float2 y[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) y[s] = s0 + s < S ? __ldcg(ml + s0 + s) : make_float2(-INFINITY, 0.f);
        float top = M;
#pragma unroll
        for (int s = 0; s < 8; ++s) top = fmaxf(top, y[s].x);
        const float base = top == -INFINITY ? 0.f : top;
        L *= exp2f(M - base);
#pragma unroll
        for (int s = 0; s < 8; ++s) L = fmaf(exp2f(y[s].x - base), y[s].y, L);
        M = top;
      }
      s_all[tid * 2] = M == -INFINITY ? 0.f : M, s_all[tid * 2 + 1] = L == 0.f ? 0.f : 1.f / L;
    }
    __syncthreads();
    if constexpr (!SPLIT) load(r0);
    while (r0 < pairs) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float2 all = *reinterpret_cast<const float2*>(s_all + min(r0 + u * STEP, pairs - 1) * 2);
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (x[u][k] != -INFINITY) sum[k] = fmaf(exp2_fast(x[u][k] - all.x), all.y, sum[k]);      // keys that a row does not see get nothing of it, whatever its sum is
      }
      r0 += U * STEP;
      if (r0 < pairs) load(r0);
    }
  }
  if constexpr (SPLIT) {
#pragma unroll
    for (int k = 0; k < V; ++k) s_sum[warp][k * 32 + lane] = sum[k];
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int o = 1; o < WARPS; ++o) sum[k] += s_sum[o][k * 32 + lane];
  }
  if (whole) {
    *reinterpret_cast<float4*>(w) = make_float4(old[0] + sum[0], old[V > 1] + sum[V > 1], old[V / 2] + sum[V / 2], old[V - 1] + sum[V - 1]);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < room) w[k] = old[k] + sum[k];
  }
}

template <typename E>
int launch_finish(const BudgetParams& p, bool join, bool weigh, cudaStream_t s) {
  const bool four = p.capacity % 4 == 0;         // rows of scores start on 16 bytes
  const bool split = p.uniform_q * (long long)p.G >= 16;
  const int join_blocks = join ? p.tokens * p.Hkv * p.G : 0, run = 32 * (four ? 4 : 1) * (split ? 1 : JOIN_THREADS / 32);
  const long long blocks = join_blocks + (weigh ? (p.capacity + run - 1) / run * p.Hkv * p.num_seqs : 0);
  if (blocks > INT_MAX) return -3;
  auto kernel = four ? (split ? attn_budget_finish_kernel<E, 4, true> : attn_budget_finish_kernel<E, 4, false>)
                     : (split ? attn_budget_finish_kernel<E, 1, true> : attn_budget_finish_kernel<E, 1, false>);
  return launch_kernel(kernel, dim3((unsigned)blocks), dim3(JOIN_THREADS), 0, s, p, join_blocks);
}

template <typename E, int R, bool VEC>
int launch_plain(const BudgetParams& p, cudaStream_t s) {
  const int ldk = (p.D + 3) / 4 * 4 + 4, ldv = (p.Dv + 3) / 4 * 4;
  const size_t smem = 4 * ((size_t)R * (ldk - 4) + (size_t)PLAIN_TILE * (ldk + ldv + R));
  auto kernel = p.Dv <= 128 ? attn_budget_plain_kernel<E, 1, R, VEC> : attn_budget_plain_kernel<E, 2, R, VEC>;
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -(int)e;
  }
  return launch_kernel(kernel, dim3(p.num_splits * p.Hkv * p.head_tiles * p.tokens), dim3(PLAIN_THREADS), smem, s, p);
}

template <typename E, bool VEC>
int launch_plain(const BudgetParams& p, cudaStream_t s) {
  return p.G <= 4 ? launch_plain<E, 4, VEC>(p, s) : p.G <= 8 ? launch_plain<E, 8, VEC>(p, s) : launch_plain<E, 16, VEC>(p, s);
}

template <typename E>
int launch_plain(const BudgetParams& p, cudaStream_t s) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
  return (p.D | p.Dv) % 4 == 0 && at % (4 * sizeof(E)) == 0 ? launch_plain<E, true>(p, s) : launch_plain<E, false>(p, s);
}

int heads_in_tiles(int G) { return (G + ROWS - 1) / ROWS; }

}  // namespace
}  // namespace swb

extern "C" {

// See BudgetParams. dims: host int[16] = tokens, num_seqs, tokens of each sequence (with cu_q: at most), table width, blocks, block_size, Hkv, G, D, Dv,
// width of the page lists, splits, fp32, 0, 0, 0; strides: host long long[8] = q token and head, out token, table, weights sequence and head, 0, 0.
// pages and counts, or weights. workspace (16-byte aligned), where results are joined by a second launch or weights are kept: 4 tokens Hq (splits (Dv + 2) +
// keys of the table, with weights) + 16 bytes.
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
      p.Dv < 1 || p.Dv > 256 || p.num_splits < 1 || p.num_splits > MAX_SPLITS || p.uniform_q < 1 || !pages == !weights || (pages && (!counts || p.width < 1)) || !q || !out ||
      !k || !v || !table || !kv_lens)
    return -3;
  p.head_tiles = heads_in_tiles(p.G);
  if ((long long)p.tokens * p.Hkv * p.head_tiles * p.num_splits > INT_MAX || (long long)p.max_blocks * p.bs > INT_MAX || (long long)p.width * p.bs > INT_MAX) return -3;
  p.q = q, p.out = out, p.k = k, p.v = v, p.table = table, p.cu_q = cu_q, p.kv_lens = kv_lens, p.pages = pages, p.counts = counts, p.weights = weights;
  p.q_stride_tok = strides[0], p.q_stride_head = strides[1], p.out_stride_tok = strides[2], p.table_stride = strides[3], p.w_seq = strides[4], p.w_head = strides[5];
  p.scale = scale, p.softcap = softcap, p.capacity = (long long)p.max_blocks * p.bs;
  const bool fast = fast_fits(p, fp32);
  // tokens of one sequence read the same keys: as many as rows allow share a problem
  p.run = 1;
  while (fast && !pages && p.run * 2 * p.G <= ROWS && p.run < p.uniform_q) p.run *= 2;
  const long long problems = (p.run > 1 ? (long long)p.num_seqs * ((p.uniform_q - 1) / p.run + 1) : p.tokens) * p.Hkv * p.head_tiles;
  if (problems > INT_MAX / p.num_splits) return -3;
  // Blocks of a cluster start together and wait for one another, which costs nothing while all of them fit the chip at once; behind that a second launch is cheaper
  // (48 sequences of up to 8191 keys, 8 key/value heads, 4 splits: 305 us as clusters, 213 with a second launch)
  const bool own_weights = fast && p.uniform_q == 1 && p.head_tiles == 1;       // else there is a second launch in any case
  p.cluster = fast && p.num_splits > 1 && p.num_splits <= MAX_CLUSTER && problems * p.num_splits <= 2 * 148 && (!weights || own_weights);
  p.weigh_here = weights && own_weights && (p.cluster || p.num_splits == 1);
  const bool join = p.num_splits > 1 && !p.cluster, weigh = weights && !p.weigh_here;
  if (join || weights) {
    // workspace: the parts of the rows, and the scores where weights are kept, in front of them
    const size_t rows = (size_t)p.tokens * p.Hkv * p.G, parts = rows * p.num_splits;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || (long long)(4 * (parts * (p.Dv + 2) + (weights ? rows * p.capacity : 0)) + 16) > workspace_bytes) return -3;
    float* ws = reinterpret_cast<float*>(workspace);
    if (weights) p.scores = ws, ws += rows * p.capacity;
    ws += (4 - (rows * p.capacity * (weights != nullptr)) % 4) % 4;
    if (join || weigh) p.part_ml = ws;
    if (join) p.part_o = ws + parts * 2;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int rc = fast ? launch_fast(p, s) : fp32 ? launch_plain<float>(p, s) : launch_plain<bf16>(p, s);
  if (rc || !(join || weigh)) return rc;
  return fp32 ? launch_finish<float>(p, join, weigh, s) : launch_finish<bf16>(p, join, weigh, s);
}

}  // extern "C"
