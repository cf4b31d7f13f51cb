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
  int q_vec, out_vec;        // rows of q and of out start on 16 bytes
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

// ---- bf16, widths up to 128, pages of 16-key groups: products on the tensor memory's matrix instructions -----------------------------------------------------
//
// A block has 128 rows and walks its keys in tiles of 128.
//   warp 8      producer: a box of 16 keys x 64 columns to a lane, so that a tile of K or V is one instruction of the warp; groups of keys that are not there are fetched
//               from behind the cache, which fills zeros in
//   warp 9      matrix instructions: S = Q K^T, then O += P V with P in tensor memory, where it takes the place of S, and V as it lies (its rows are the product's inner dimension)
//   warps 0-7   softmax, two threads to a row with 64 of a tile's keys each; in tiles of the tree they apply the mask and see to it that V holds numbers
// One tile of K and one of V fit beside Q where two blocks share an SM: the products of one run beside the softmax of the other.
constexpr int TC_ROWS = 128, TC_KEYS = 128, TC_THREADS = 320, TMA_WARP = 8, MMA_WARP = 9;
constexpr uint32_t TC_COLS = 256, COL_S = 0, COL_O = 128;
constexpr float TC_RESCALE = 8.f;          // O is rescaled when a maximum has grown by more than 2^8

struct TcBars {
  uint64_t q_full, k_full, k_empty, v_full, v_empty, s_full, p_full, o_final;
  uint32_t tmem_base;
  int abort;
  int odd;                 // some new token's value is no number
  unsigned dead[2];        // groups of a tile's keys that are not there
};
template <int DA, int VA>
struct TcCfg {
  static constexpr uint32_t Q = 0, K = DA * TC_ATOM_BYTES, V = 2 * DA * TC_ATOM_BYTES, BARS = V + VA * TC_ATOM_BYTES, EXCHANGE = BARS + 256;
  static constexpr size_t BYTES = EXCHANGE + 2 * 2 * TC_ROWS * 4 + 1024;
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

template <int DA, int VA, bool CAP>
__device__ __forceinline__ void tree_softmax(const TreeParams& p, TcBars* bars, uint8_t* smem, uint32_t tmem, const Span& s, int seq, int h, int r0, int rows, int split, int t_lo, int n_tiles) {
  using C = TcCfg<DA, VA>;
  constexpr int OUT = VA * 32;                                              // output columns of a thread
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = warp >> 2, w4 = warp & 3, row = w4 * 32 + lane;
  const uint32_t lane_base = (uint32_t)(w4 * 32) << 16, t_s = tmem + lane_base + COL_S, t_o = tmem + lane_base + COL_O + half * OUT;
  float* exchange = reinterpret_cast<float*>(smem + C::EXCHANGE) + row;
  const int t = s.q0 + (r0 + row) / p.G, head = h * p.G + (r0 + row) % p.G;
  const bool mine = row < rows && (unsigned)t < (unsigned)p.tokens;
  const unsigned* mask = p.mask + (mine ? t : 0) * p.mask_tok;
  // Q: rows of 16-byte chunks in 128-byte swizzle atoms of 64 columns
  for (int i = tid; i < TC_ROWS * DA * 8; i += 256) {
    const int r = i / (DA * 8), c = i % (DA * 8), tr = s.q0 + (r0 + r) / p.G;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (r < rows && (unsigned)tr < (unsigned)p.tokens && c * 8 < p.D) {
      const bf16* from = reinterpret_cast<const bf16*>(p.q) + tr * p.q_tok + (long long)(h * p.G + (r0 + r) % p.G) * p.q_head + c * 8;
      if (p.q_vec) {
        x = *reinterpret_cast<const uint4*>(from);
      } else {
        const uint16_t* w = reinterpret_cast<const uint16_t*>(from);
        x = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
      }
    }
    *reinterpret_cast<uint4*>(smem + C::Q + (c >> 3) * TC_ATOM_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x;
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(&bars->q_full);

  float scale_log2 = p.scale * 1.4426950408889634f, to_cap = 0.f;           // the capped score is cap (1 - 2 / (2^(to_cap s) + 1))
  if constexpr (CAP) to_cap = 2.f * scale_log2 / p.softcap, scale_log2 = 1.4426950408889634f;
  const float STOP = __int_as_float(0x7fffffff);                            // handed over instead of a maximum when a wait ran out
  float m_used = -INFINITY, l = 0.f;
  bool ok = true, values_ok = true;
  for (int j = 0; j < n_tiles; ++j) {
    ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full, j & 1, &bars->abort, 30));
    const int tile0 = (t_lo + j) * TC_KEYS, key0 = tile0 + half * 64;
    const bool tail = tile0 + TC_KEYS > s.base;
    uint32_t x[64];
    float mx = STOP;
    if (ok) {
      tc_fence_after_sync();
      tmem_ld_x32(t_s + half * 64, x);
      tmem_ld_x32(t_s + half * 64 + 32, x + 32);
      tmem_ld_wait();
      if constexpr (CAP) {
#pragma unroll
        for (int i = 0; i < 64; ++i) x[i] = __float_as_uint(fmaf(-2.f * p.softcap, rcp_approx(ex2(__uint_as_float(x[i]) * to_cap) + 1.f), p.softcap));
      }
      const unsigned dead = bars->dead[j & 1];
      if (tail || dead) {
        const unsigned long long seen = seen_keys(mask, p.words, key0, s.base, s.len, dead >> half * 4);
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (!(seen >> i & 1ull)) x[i] = __float_as_uint(-INFINITY);
      }
      float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        m0 = fmaxf(m0, __uint_as_float(x[i])), m1 = fmaxf(m1, __uint_as_float(x[i + 1]));
        m2 = fmaxf(m2, __uint_as_float(x[i + 2])), m3 = fmaxf(m3, __uint_as_float(x[i + 3]));
      }
      mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
    }
    float* slot = exchange + (j & 1) * (2 * TC_ROWS);
    slot[half * TC_ROWS] = mx;
    pair_sync(1 + w4);
    const float other = slot[(half ^ 1) * TC_ROWS];
    ok = ok && __all_sync(0xffffffffu, __float_as_int(other) != 0x7fffffff);
    if (!ok) break;                                                         // both halves leave at the same tile
    const float m_new = fmaxf(fmaxf(mx, other), m_used);
    const bool grow = (m_new - m_used) * scale_log2 > TC_RESCALE;           // true on the first tile with a key that the row sees (m_used = -inf)
    if (__any_sync(0xffffffffu, grow)) {
      const float f = grow ? ex2((m_used - m_new) * scale_log2) : 1.f;
      if (grow) l *= f, m_used = m_new;
      if (j > 0) {
#pragma unroll
        for (int c = 0; c < OUT / 16; ++c) {
          float o[16];
          tmem_ld_32x32b_x16(t_o + c * 16, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= f;
          tmem_st_x16(t_o + c * 16, o);
        }
      }
    }
    const float neg_m = m_used == -INFINITY ? 0.f : -m_used * scale_log2;
    const unsigned long long sc2 = pack2(scale_log2, scale_log2), nm2 = pack2(neg_m, neg_m);
    unsigned long long l0 = 0ull, l1 = 0ull;
#pragma unroll
    for (int i = 0; i < 64; i += 4) {       // packed P overwrites the row in place
      float a, b, c, d;
      unpack2(fma2(pack2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sc2, nm2), a, b);
      unpack2(fma2(pack2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), sc2, nm2), c, d);
      a = ex2(a), b = ex2(b), c = ex2(c), d = ex2(d);
      l0 = add2(l0, pack2(a, b)), l1 = add2(l1, pack2(c, d));
      x[i >> 1] = pack_bf16x2(a, b), x[(i >> 1) + 1] = pack_bf16x2(c, d);
    }
    float x0, x1;
    unpack2(add2(l0, l1), x0, x1);
    l += x0 + x1;
    tmem_st_x32(t_s + half * 32, x);
    tmem_st_wait();
    tc_fence_before_sync();
    if (tail) {
      // Values behind the sequence's end are anything, and those of new tokens are not for every row: what is no number becomes a zero in front of the product, and is added
      // to the rows that see it at the end.
      values_ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_full, j & 1, &bars->abort, 31));
      if (!values_ok) continue;             // the next wait runs out too
      for (int i = tid; i < TC_KEYS * VA * 8; i += 256) {
        const int r = i / (VA * 8), c = i % (VA * 8);
        if (tile0 + r < s.base) continue;
        uint4* at = reinterpret_cast<uint4*>(smem + C::V + (c >> 3) * TC_ATOM_BYTES + r * 128 + ((c & 7) << 4));      // any chunk of the row
        uint4 v = *at;
        if (tile0 + r >= s.len) {
          *at = make_uint4(0, 0, 0, 0);
          continue;
        }
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u, odd = true;
          if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu, odd = true;
        }
        if (odd) *at = v, bars->odd = 1;
      }
      fence_proxy_async_smem();
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->p_full);
  }
  if (!ok) return;
  ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_final, 0, &bars->abort, 32)) && values_ok;
  float* slot = exchange + (n_tiles & 1) * (2 * TC_ROWS);
  slot[half * TC_ROWS] = ok ? l : STOP;
  pair_sync(1 + w4);
  const float other = slot[(half ^ 1) * TC_ROWS];
  if (!ok) return;
  tc_fence_after_sync();
  const float sum = half ? other + l : l + other;
  const bool odd = bars->odd != 0;
  // values that are no numbers, of new tokens among this block's keys that the row sees: columns from d0 on
  const auto add_odd = [&](uint32_t* o, int d0) {
    const int* table = p.table + seq * p.table_stride;
    for (int key = max(t_lo * TC_KEYS, max(s.base, 0)); key < min(s.len, (t_lo + n_tiles) * TC_KEYS); ++key) {
      const int block = table[key / p.bs];
      if (!mine || (unsigned)block >= (unsigned)p.num_blocks || !sees(mask, p.words, key - s.base)) continue;
      const bf16* v = reinterpret_cast<const bf16*>(p.v) + (((long long)block * p.Hkv + h) * p.bs + key % p.bs) * p.Dv + d0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float y = d0 + i < p.Dv ? __bfloat162float(v[i]) : 0.f;
        if (!isfinite(y)) o[i] = __float_as_uint(__uint_as_float(o[i]) + y);
      }
    }
  };
  if (p.part_o) {
    const long long at = ((long long)split * p.tokens + t) * (p.Hkv * p.G) + head;
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
    if (half == 0 && mine) p.part_ml[at] = make_float2(m_used == -INFINITY ? -INFINITY : m_used * scale_log2, sum);
    return;
  }
  // through the idle Q and K tiles, so that rows are written in runs: 16-byte chunk c of row r lies at c ^ (r & (chunks - 1))
  constexpr int BYTES = OUT * 2, CHUNKS = BYTES / 16;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint8_t* slab = smem + C::Q + warp * (32 * BYTES);
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
    bf16* to = out + to_t * p.out_tok + (long long)(h * p.G + rr % p.G) * p.Dv + d;
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
__global__ void __launch_bounds__(TC_THREADS, 2) attn_tree_tc_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const TreeParams p) {
  using C = TcCfg<DA, VA>;
  extern __shared__ uint8_t tc_smem[];
  uint8_t* smem = tc_smem + ((1024u - (smem_u32(tc_smem) & 1023u)) & 1023u);
  TcBars* bars = reinterpret_cast<TcBars*>(smem + C::BARS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // row tiles of a problem are neighbours: they run together and find one another's keys in the second-level cache
  const int tile = blockIdx.x % p.tiles, y = blockIdx.x / p.tiles, split = y % p.num_splits, z = y / p.num_splits, h = z % p.Hkv, seq = z / p.Hkv;
  pdl_launch_dependents();
  pdl_wait(TL_ATTN_DECODE);
  const Span s = span_of(p, seq);
  const int r0 = tile * TC_ROWS, rows = min(TC_ROWS, min(s.n, p.uniform_q) * p.G - r0);
  if (rows <= 0) return;                                   // uniform, like the next one, in front of all barriers
  const int all = (s.len + TC_KEYS - 1) / TC_KEYS, per = (all + p.num_splits - 1) / p.num_splits, t_lo = min(split * per, all), n_tiles = min(all, t_lo + per) - t_lo;
  if (n_tiles <= 0) {                                      // fewer tiles than splits, or nothing in the cache
    for (int r = threadIdx.x; r < rows; r += TC_THREADS) {
      const int t = s.q0 + (r0 + r) / p.G, head = h * p.G + (r0 + r) % p.G;
      if ((unsigned)t >= (unsigned)p.tokens) continue;
      if (p.part_o) p.part_ml[((long long)split * p.tokens + t) * (p.Hkv * p.G) + head] = make_float2(-INFINITY, 0.f);
      else
        for (int d = 0; d < p.Dv; ++d) reinterpret_cast<bf16*>(p.out)[t * p.out_tok + (long long)head * p.Dv + d] = __float2bfloat16(0.f);
    }
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 8);
    mbar_init(&bars->k_full, 1);
    mbar_init(&bars->k_empty, 1);
    mbar_init(&bars->v_full, 1);
    mbar_init(&bars->v_empty, 1);
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->p_full, 8);
    mbar_init(&bars->o_final, 1);
    bars->abort = 0, bars->odd = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&bars->tmem_base, TC_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  if (warp == TMA_WARP) {
    // lane = group of 16 keys + 8 * swizzle atom
    const int* table = p.table + seq * p.table_stride;
    const int g = lane & 7, atom = lane >> 3, none = p.num_blocks * p.Hkv * p.bs;
    bool ok = true;
    int issued_k = 0, issued_v = 0;
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int key = (t_lo + j) * TC_KEYS + g * 16;
      int row = none;
      if (key < s.len) {
        const int block = table[key / p.bs];
        if ((unsigned)block < (unsigned)p.num_blocks) row = (block * p.Hkv + h) * p.bs + key % p.bs;
      }
      const unsigned dead = __ballot_sync(0xffffffffu, row == none) & 0xffu;
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->k_empty, (j & 1) ^ 1, &bars->abort, 10));
      if (!ok) break;
      if (lane == 0) {
        bars->dead[j & 1] = dead;
        mbar_arrive_expect_tx(&bars->k_full, DA * TC_ATOM_BYTES);
      }
      __syncwarp();
      if (atom < DA) tma_load_2d(smem + C::K + atom * TC_ATOM_BYTES + g * 2048, &tmap_k, &bars->k_full, atom * 64, row);
      issued_k = j + 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_empty, (j & 1) ^ 1, &bars->abort, 11));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&bars->v_full, VA * TC_ATOM_BYTES);
      __syncwarp();
      if (atom < VA) tma_load_2d(smem + C::V + atom * TC_ATOM_BYTES + g * 2048, &tmap_v, &bars->v_full, atom * 64, row);
      issued_v = j + 1;
    }
    if (!ok) {                                             // copies in flight land before the block's memory is released
      volatile int never = 0;
      if (issued_k) mbar_wait(&bars->k_full, (issued_k - 1) & 1, &never, 13);
      if (issued_v) mbar_wait(&bars->v_full, (issued_v - 1) & 1, &never, 14);
    }
  } else if (warp == MMA_WARP) {
    constexpr uint32_t IDESC_QK = umma_idesc_bf16_f32(TC_ROWS, TC_KEYS), IDESC_PV = umma_idesc_bf16_f32(TC_ROWS, VA * 64) | (1u << 16);      // V is MN-major
    const uint64_t qd = umma_desc_kmajor_sw128(smem_u32(smem + C::Q)), kd = umma_desc_kmajor_sw128(smem_u32(smem + C::K)), vd = umma_desc_mnmajor_sw128(smem_u32(smem + C::V));
    const auto wait = [&](uint64_t* bar, uint32_t parity, int where) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, &bars->abort, where)) != 0; };
    bool ok = wait(&bars->q_full, 0, 20);
    for (int j = 0; j <= n_tiles && ok; ++j) {
      if (j > 0) {                                         // O += P V of the tile before
        ok = wait(&bars->p_full, (j - 1) & 1, 22) && wait(&bars->v_full, (j - 1) & 1, 23);
        if (!ok) break;
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < TC_KEYS / 16; ++k) umma_f16_ts(tmem + COL_O, tmem + COL_S + k * 8, vd + k * (2048 >> 4), IDESC_PV, j > 1 || k > 0);
          umma_commit(&bars->v_empty);
        }
        __syncwarp();
      }
      if (j < n_tiles) {
        ok = wait(&bars->k_full, j & 1, 21);
        if (!ok) break;
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < DA * 4; ++k) {
            const uint32_t off = ((k >> 2) * TC_ATOM_BYTES + (k & 3) * 32) >> 4;
            umma_f16_ss(tmem + COL_S, qd + off, kd + off, IDESC_QK, k > 0);
          }
          umma_commit(&bars->s_full);
          umma_commit(&bars->k_empty);
        }
        __syncwarp();
      }
    }
    if (elect_one()) umma_commit(&bars->o_final);          // also where a wait ran out: it tracks what has been issued
    __syncwarp();
    if (!ok) {
      volatile int never = 0;
      mbar_wait(&bars->o_final, 0, &never, 27);
      __syncwarp();
    }
  } else {
    tree_softmax<DA, VA, CAP>(p, bars, smem, tmem, s, seq, h, r0, rows, split, t_lo, n_tiles);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, TC_COLS);
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
      if (d < p.Dv && f != 0.f) x = fmaf(f, p.part_o[(s * rows + i) * p.Dv + d], x);      // of a split without keys nothing was written
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
  if ((long long)p.max_blocks * p.bs > INT_MAX || (long long)p.uniform_q * p.G > INT_MAX - TC_ROWS) return -3;
  p.scale = scale, p.softcap = softcap, p.k = k, p.v = v;
  const bool fast = tc_fits(p, fp32);
  const int tile = fast ? TC_ROWS : PR;
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
  const dim3 grid((unsigned)((rows + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32)));
  return fp32 ? launch_kernel(attn_tree_join_kernel<float>, grid, dim3(JOIN_THREADS), 0, s, p) : launch_kernel(attn_tree_join_kernel<bf16>, grid, dim3(JOIN_THREADS), 0, s, p);
}

}  // extern "C"
