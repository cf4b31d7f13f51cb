// Summaries of cache pages and the choice of pages by them.
//
// Summary of a page of one key/value head: s = the sum of its keys, a = max |s| over the columns, codes rint(127 s / a) in 8 bits and the scale
// a / (127 block_size), so that code * scale is the mean key to within half a step. Sums and the quotient in front of the rounding are 64-bit numbers: which of two
// neighbouring codes a column gets does not hang on the order of a sum.
//
// Score of a page for a query token and a key/value head: the group's queries as 8-bit codes of one common step, scale * max over the group of
// the codes' dot product. The dot products are whole numbers and the scale multiplies once, so a score has one value whatever computes it, and ties go to
// the lowest page.
#include "common.cuh"
#include "radix_select.cuh"

#include <climits>

namespace swb {
namespace {

struct SummaryParams {
  const void* k;             // [blocks, Hkv, bs, D]
  int8_t* codes;             // [blocks, Hkv, D]
  float* scales;             // [blocks, Hkv]
  const int* table;          // [num_seqs, table_stride]
  long long table_stride;
  int max_blocks, num_blocks, bs, Hkv, D;
  const int* cu_q;
  const int* kv_lens;
  int num_seqs, uniform_q;
};

constexpr int SUMMARY_WARPS = 4;

// rint(127 s / a), where step = 127 / a in 32 bits. The product of 32-bit numbers is off by less than 4 2^-24 127: only where it comes that near a half are the 64-bit
// numbers divided.
__device__ __forceinline__ int8_t summary_code(double s, double a, float step) {
  const float r = (float)s * step, q = rintf(r);
  if (fabsf(fabsf(r - q) - 0.5f) > 1e-4f && step < 1e30f && step > 1e-30f) return (int8_t)(int)q;
  return (int8_t)(int)rint(127.0 * s / a);
}

// The page of a warp: its place, or -1.
__device__ __forceinline__ long long summary_place(const SummaryParams& p, int h) {
  const int seq = blockIdx.z;
  const int q_len = p.cu_q ? p.cu_q[seq + 1] - p.cu_q[seq] : p.uniform_q;
  const int len = min(p.kv_lens[seq], p.max_blocks * p.bs);
  if (len <= 0 || q_len <= 0) return -1;
  const unsigned page = (unsigned)(max(len - q_len, 0) / p.bs) + blockIdx.x;      // the first page that the new tokens can complete, and on
  if (page >= (unsigned)(len / p.bs)) return -1;
  const int block = p.table[seq * p.table_stride + page];
  return (unsigned)block < (unsigned)p.num_blocks ? (long long)block * p.Hkv + h : -1;
}

// Two bf16 numbers as 64-bit ones of 2^-896 times their size: sign, exponent and fraction moved to their places, the exponent's bias left as it is. Zeros and numbers
// below the normal range come out right as well; infinities and NaN come out as numbers and are looked for apart.
__device__ __forceinline__ double scaled_low(uint32_t w) { return __hiloint2double(((int)(w << 16) >> 3) & (int)0x8fffe000u, 0); }
__device__ __forceinline__ double scaled_high(uint32_t w) { return __hiloint2double(((int)w >> 3) & (int)0x8fffe000u, 0); }

// bf16 pages up to 128 wide, widths of a multiple of four: a lane has four columns, 16 rows of a page on their way at once. A change of type to 64 bits
// runs at a sixteenth of the rate, and one for each number bounds the kernel: 81 us for 120 000 tokens of 8 heads. Sums of four rows in 32 bits with what each addition leaves
// out beside them took 14 instructions a number, 61 us. Moving the bits takes three and the addition in 64 bits, at half the rate, one: 49 us, 5.0 TB/s. (Two pages of a
// warp at once: 59; eight of them one behind the other: 83.)
// BS16: pages of 16 keys, whose rows need no question each (14 us for one prompt of 15 000 tokens with them, 9.6 without).
template <bool BS16>
__global__ void __launch_bounds__(SUMMARY_WARPS * 32) page_summary_quads_kernel(const SummaryParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, h = blockIdx.y * SUMMARY_WARPS + (threadIdx.x >> 5), bs = BS16 ? 16 : p.bs;
  if (h >= p.Hkv) return;
  const long long at = summary_place(p, h);
  if (at < 0) return;
  const bool live = lane * 4 < p.D;
  const uint2* k = reinterpret_cast<const uint2*>(reinterpret_cast<const bf16*>(p.k) + at * bs * p.D) + (live ? lane : 0);
  const int row = p.D / 4;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  __nv_bfloat162 size = __float2bfloat162_rn(0.f);       // the largest of both, NaN where there is one
  for (int t0 = 0; t0 < bs; t0 += 16) {
    uint2 x[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) x[t] = BS16 || t0 + t < bs ? __ldg(k + (size_t)(t0 + t) * row) : make_uint2(0u, 0u);
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      s[0] += scaled_low(x[t].x), s[1] += scaled_high(x[t].x), s[2] += scaled_low(x[t].y), s[3] += scaled_high(x[t].y);
      size = __hmax2_nan(size, __habs2(reinterpret_cast<const __nv_bfloat162&>(x[t].x)));
      size = __hmax2_nan(size, __habs2(reinterpret_cast<const __nv_bfloat162&>(x[t].y)));
    }
  }
  double a = 0.0;
  const bool bad = __any_sync(0xffffffffu, !(__low2float(size) < INFINITY && __high2float(size) < INFINITY));
#pragma unroll
  for (int c = 0; c < 4; ++c) a = fmax(a, fabs(s[c] *= 0x1p896));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmax(a, __shfl_xor_sync(0xffffffffu, a, o));
  uint32_t codes = 0u;
  const float step = __fdiv_rn(127.f, (float)a);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (!bad && a > 0.0) codes |= (uint32_t)(uint8_t)summary_code(s[c], a, step) << (8 * c);
  if (live) reinterpret_cast<uint32_t*>(p.codes + at * p.D)[lane] = codes;
  if (lane == 0) p.scales[at] = bad ? NAN : (float)(a / (127.0 * bs));
}

// Any other: a warp per (page, head); lane l holds columns l, l + 32, ... of up to COLS * 32.
template <typename E, int COLS>
__global__ void __launch_bounds__(SUMMARY_WARPS * 32) page_summary_kernel(const SummaryParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, h = blockIdx.y * SUMMARY_WARPS + (threadIdx.x >> 5);
  if (h >= p.Hkv) return;
  const long long at = summary_place(p, h);
  if (at < 0) return;
  const E* k = reinterpret_cast<const E*>(p.k) + at * p.bs * p.D;
  double s[COLS];
#pragma unroll
  for (int c = 0; c < COLS; ++c) s[c] = 0.0;
  for (int t = 0; t < p.bs; ++t) {
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const int d = c * 32 + lane;
      if (d < p.D) s[c] += (double)to_f(k[(size_t)t * p.D + d]);
    }
  }
  double a = 0.0;
  bool bad = false;
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    a = fmax(a, fabs(s[c]));
    bad |= !(fabs(s[c]) < INFINITY);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmax(a, __shfl_xor_sync(0xffffffffu, a, o));
  bad = __any_sync(0xffffffffu, bad);
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    const int d = c * 32 + lane;
    if (d < p.D) p.codes[at * p.D + d] = bad || a == 0.0 ? (int8_t)0 : summary_code(s[c], a, __fdiv_rn(127.f, (float)a));
  }
  if (lane == 0) p.scales[at] = bad ? NAN : (float)(a / (127.0 * p.bs));
}

// codes * scales as 32-bit numbers, four at a time where rows allow.
__global__ void __launch_bounds__(256) page_values_kernel(const int8_t* codes, const float* scales, float* out, long long n, int D, int four) {
  pdl_launch_dependents();
  pdl_wait();
  const long long step = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (four ? n / 4 : n); i += step) {
    if (four) {
      const char4 c = reinterpret_cast<const char4*>(codes)[i];
      const float s = scales[n <= 0xffffffffll ? (uint32_t)i / (uint32_t)(D / 4) : i / (D / 4)];
      reinterpret_cast<float4*>(out)[i] = make_float4(c.x * s, c.y * s, c.z * s, c.w * s);
    } else {
      out[i] = codes[i] * scales[i / D];
    }
  }
}

struct SelectParams {
  const void* q;
  long long q_stride_tok, q_stride_head;
  const int8_t* codes;
  const float* scales;
  const int* table;
  long long table_stride;
  int max_blocks, num_blocks, bs, Hkv, G, D;
  const int* cu_q;
  const int* kv_lens;
  int num_seqs, uniform_q, tokens;
  int first, top, last;
  int* pages;                // [tokens, Hkv, first + top + last]
  int* counts;               // [tokens, Hkv]
  int fp32;                  // type of q
  int q_vec;                 // bf16 rows of 16-byte alignment
  int share;                 // blocks of a problem
};

constexpr int SELECT_THREADS = 256, SELECT_WARPS = SELECT_THREADS / 32;

__device__ __forceinline__ void mma_s8(int* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Sixteen codes of a row from column d on, zeros behind its end. FULL: rows are 32 KS codes, 16-byte aligned.
template <bool FULL>
__device__ __forceinline__ uint4 load_codes(const int8_t* row, int d, int D, bool vec) {
  if (FULL) return __ldg(reinterpret_cast<const uint4*>(row + d));
  if (d >= D) return make_uint4(0, 0, 0, 0);
  if (vec) return __ldg(reinterpret_cast<const uint4*>(row + d));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (d + i < D) w[i >> 2] |= (uint32_t)(uint8_t)row[d + i] << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float load_query(const SelectParams& p, long long at) {
  return p.fp32 ? reinterpret_cast<const float*>(p.q)[at] : __bfloat162float(reinterpret_cast<const bf16*>(p.q)[at]);
}

// rint(127 x / a), |x| <= a. Where both are bf16, 127 x has 15 bits and the quotient, a fraction over a's 8 bits and powers of two, is either a
// half exactly or further from one than 2^-16 of itself: its rounding to 32 bits moves nothing across. Other numbers are divided in 64 bits.
// (Near the end of the 32-bit range both are made smaller first, by a power of two.)
__device__ __forceinline__ int8_t query_code(float x, float a, bool fp32) {
  if (fp32) return (int8_t)(int)rint(127.0 * (double)x / (double)a);
  const float s = a > 0x1p100f ? 0x1p-64f : 1.f;
  return (int8_t)(int)rintf(__fdiv_rn(127.f * (x * s), a * s));
}

// A block per (run of TT tokens of a sequence, head). The dot products are 8-bit matrix products: 16 rows are pages, 8 columns the tokens' query heads (a token's heads
// are filled up to a power of two, with copies of its first, which change no maximum; GP is that power where it is known), so that a head's neighbours are a thread's own or a shuffle away and
// every thread ends with one page's score for one token. A page's row is fetched 16 codes at a time (8 at a time took 8 % longer
// over a prompt): the lane of page g and quarter t holds columns 64 j + 16 t and on, for two steps, and the queries' codes are read in the same order, so the order of the columns within a step is another than the instruction's and the sum the same.
// Then the tokens are shared out among teams of warps, each of which chooses among its token's scores.
// CL: p.share blocks, a cluster, score a part of the pages each into the first one's memory, and that one chooses (few problems over long caches).
// Shared memory: the teams' histograms, codes of the queries [TT, G, 32 KS], keys [TT, pages].
// 64 sequences of up to 1025 pages, 8 heads: 20 us (54 MB: 2.7 TB/s), most of it latency, of the look-ups and the first rows (half) and of the choice's steps (a quarter).
// 1000 tokens of a prompt over 1063 pages: 90 us, of which scores and choice have about the same part; 2 instructions a cycle, 250 MB through the second-level cache. Registers are
// what is short: 100 spilled bytes in the loop over pages cost 15 us, and two blocks an SM with none 10.
template <int TT, int KS, bool FULL, int GP, bool CL>
__global__ void __launch_bounds__(SELECT_THREADS, KS == 8 ? 2 : TT == 1 && !CL ? 4 : 3) page_select_kernel(const SelectParams p) {
  constexpr int TEAM = SELECT_THREADS / TT, LD = 32 * KS;
  pdl_launch_dependents();
  extern __shared__ __align__(16) uint8_t select_smem[];
  __shared__ float s_amax[SELECT_WARPS];
  __shared__ uint32_t s_largest[TT];
  __shared__ int s_bad[TT], s_cand[TT];           // s_cand: pages to choose among
  const Team<TEAM> team(threadIdx.x);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* hist = reinterpret_cast<int*>(select_smem) + team.id * SELECT_INTS;
  int8_t* qc = reinterpret_cast<int8_t*>(select_smem + TT * SELECT_INTS * 4);
  uint32_t* keys = reinterpret_cast<uint32_t*>(qc + TT * p.G * LD);
  const int ldkeys = (p.max_blocks + 3) & ~3;
  // blocks that run together share what they read: the tokens of a prompt a head's codes, the heads of a decode step a page's memory
  const int runs = (p.uniform_q + TT - 1) / TT, all_runs = runs * p.num_seqs;
  const int share = CL ? p.share : 1, rank = CL ? blockIdx.x % share : 0, x = CL ? blockIdx.x / share : blockIdx.x;
  const int h = TT > 1 ? x / all_runs : x % p.Hkv, run = TT > 1 ? x % all_runs : x / p.Hkv, seq = run / runs;
  if (tid < TT) s_bad[tid] = 0, s_largest[tid] = 0u;
  pdl_wait();
  const int q0 = p.cu_q ? p.cu_q[seq] : seq * p.uniform_q, q1 = p.cu_q ? p.cu_q[seq + 1] : q0 + p.uniform_q;
  const int t0 = q0 + (run % runs) * TT;
  if (t0 < 0 || t0 >= min(q1, p.tokens)) return;
  const int len = min(p.kv_lens[seq], p.max_blocks * p.bs), width = p.first + p.top + p.last;
  const auto pages_of = [&](int t) {               // pages that token t sees
    const int seen = len - (q1 - 1 - t);
    return seen > 0 ? (seen + p.bs - 1) / p.bs : 0;
  };
  // this team's token: what needs no scores
  const int t = t0 + team.id, n = t < min(q1, p.tokens) ? pages_of(t) : 0;
  int* out = p.pages + ((size_t)t * p.Hkv + h) * width;
  if (team.rank == 0) s_cand[team.id] = n > width ? n - p.first - p.last : 0;
  if (rank == 0 && t < min(q1, p.tokens)) {
    if (team.rank == 0) p.counts[(size_t)t * p.Hkv + h] = min(n, width);
    if (n <= width) {
      for (int i = team.rank; i < width; i += TEAM) out[i] = i < n ? i : -1;
    } else {
      for (int i = team.rank; i < p.first; i += TEAM) out[i] = i;
      for (int i = team.rank; i < p.last; i += TEAM) out[p.first + p.top + i] = n - p.last + i;
    }
  }
  const int most = pages_of(min(min(t0 + TT, q1), p.tokens) - 1), cand = most - p.first - p.last;      // the last token sees most
  if (p.top == 0 || most <= width) return;
  clear_bins(team, hist);
  __syncthreads();                                 // s_bad is set, the bins are clear
  // the token's queries as codes of one step
  if (n > width) {
    const long long q = t * p.q_stride_tok + (long long)h * p.G * p.q_stride_head;
    int8_t* to = qc + team.id * p.G * LD;
    float a = 0.f;
    bool bad = false;
    const auto look = [&](float x) {
      a = fmaxf(a, fabsf(x));
      bad |= !(fabsf(x) < INFINITY);
    };
    const auto known = [&]() {                       // the largest size of all, and whether every number is finite
      a = warp_max(a);
      if (lane == 0) s_amax[warp] = a;
      if (bad) s_bad[team.id] = 1;
      team.sync();
      a = 0.f;
      for (int w = 0; w < Team<TEAM>::WARPS; ++w) a = fmaxf(a, s_amax[team.id * Team<TEAM>::WARPS + w]);
      bad = s_bad[team.id] != 0 || a == 0.f;
    };
    if (FULL && p.q_vec) {                           // eight bf16 numbers at a time
      const bf16* from = reinterpret_cast<const bf16*>(p.q) + q;
      float x[8];
      for (int i = team.rank; i < p.G * 16; i += TEAM) {
        load_row8(from + (i >> 4) * p.q_stride_head + (i & 15) * 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) look(x[e]);
      }
      known();
      for (int i = team.rank; i < p.G * 16; i += TEAM) {
        load_row8(from + (i >> 4) * p.q_stride_head + (i & 15) * 8, x);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!bad) w[e >> 2] |= (uint32_t)(uint8_t)query_code(x[e], a, 0) << (8 * (e & 3));
        *reinterpret_cast<uint2*>(to + i * 8) = make_uint2(w[0], w[1]);
      }
    } else {
#pragma unroll 4
      for (int i = team.rank; i < p.G * p.D; i += TEAM) look(load_query(p, q + (i / p.D) * p.q_stride_head + i % p.D));
      known();
#pragma unroll 4
      for (int i = team.rank; i < p.G * LD; i += TEAM) {
        const int g = i / LD, d = i % LD;
        const float x = d < p.D ? load_query(p, q + g * p.q_stride_head + d) : 0.f;
        to[i] = bad ? (int8_t)0 : query_code(x, a, p.fp32);
      }
    }
  }
  __syncthreads();

  constexpr int NT = TT == 4 ? 2 : 1;              // products beside each other: TT Gp <= 8 NT, or one token in turns of 8 heads
  static_assert(TT == 1 || TT * GP <= 8 * NT, "every token of a block has columns");
  const int gr = lane >> 2, t4 = lane & 3;
  int Gp = GP ? GP : 1;
  while (!GP && Gp < p.G && Gp < 8) Gp <<= 1;
  const int turns = TT == 1 && !GP ? (p.G + 7) / 8 : 1;
  uint2 b[NT][KS];
  const auto load_heads = [&](int turn) {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int c = x * 8 + gr, tok = min(c / Gp, TT - 1), g = turn * 8 + c % Gp;
      const uint4* from = reinterpret_cast<const uint4*>(qc + (tok * p.G + (g < p.G ? g : 0)) * LD);
#pragma unroll
      for (int s = 0; s < KS; s += 2) {
        const uint4 y = from[s * 2 + t4];
        b[x][s] = make_uint2(y.x, y.y), b[x][s + 1] = make_uint2(y.z, y.w);
      }
    }
  };
  if (turns == 1) load_heads(0);
  const bool vec = (p.D & 15) == 0 && (reinterpret_cast<uintptr_t>(p.codes) & 15) == 0;
  const int* table = p.table + seq * p.table_stride + p.first;
  const auto locate = [&](int i) {
    const int block = i < cand ? table[i] : -1;
    return (unsigned)block < (unsigned)p.num_blocks ? block : -1;
  };
  uint32_t first_keys = 0;                         // of the cluster's first block
  if (CL) {
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first_keys) : "r"(smem_u32(keys)));
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");        // it runs
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  // keeps the score of candidate i for a token, which has `most` of them
  const auto keep = [&](int tok, int most, int i, int best, float scale, bool there) -> uint32_t {
    if (i >= most) return 0u;
    const uint32_t k = float_key(there ? __fmul_rn((float)best, scale) : -INFINITY);
    if (CL) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(first_keys + 4u * i), "r"(k) : "memory");
    else keys[tok * ldkeys + i] = k;
    return k;
  };
  // the largest key of each token, where a thread keeps keys of several
  const auto note = [&](int tok, uint32_t k) {
    if (k) atomicMax(&s_largest[tok], k);
  };
  // with four heads and more a thread ends with one score in each product: page gr or gr + 8, and this token
  const int odd_quarter = t4 & 1, tok0 = Gp == 4 ? t4 >> 1 : 0;
  int most_of[NT];
  uint32_t largest[NT];                            // of the keys that this thread keeps for that token
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    largest[x] = 0u;
    const int tok = x * (8 / Gp) + tok0;
    most_of[x] = tok < TT && (Gp == 4 || t4 < 2) ? s_cand[tok] : 0;
  }
  // rows gr and gr + 8 of the u-th 16 of a warp's 32 pages
  const auto fetch = [&](uint32_t (*a)[4], int blocks, int u) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int mine = __shfl_sync(0xffffffffu, blocks, u * 16 + half * 8 + gr);
      const int8_t* row = p.codes + ((size_t)max(mine, 0) * p.Hkv + h) * p.D;        // a page that is not there: any row, its score is not used
#pragma unroll
      for (int s = 0; s < KS; s += 2) {
        const uint4 x = load_codes<FULL>(row, s * 32 + t4 * 16, p.D, vec);
        a[s][half] = x.x, a[s][2 + half] = x.y, a[s + 1][half] = x.z, a[s + 1][2 + half] = x.w;
      }
    }
  };
  const auto score = [&](const uint32_t (*a)[4], int i0, int u, float scale, uint32_t there) {
    int c[NT][4];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      c[x][0] = c[x][1] = c[x][2] = c[x][3] = 0;
      if (turns == 1) {
#pragma unroll
        for (int s = 0; s < KS; ++s) mma_s8(c[x], a[s], b[x][s].x, b[x][s].y);
      }
    }
    if (turns > 1) {
      int best[4] = {INT_MIN, INT_MIN, INT_MIN, INT_MIN};
      for (int turn = 0; turn < turns; ++turn) {
        load_heads(turn);
        int d[4] = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) mma_s8(d, a[s], b[0][s].x, b[0][s].y);
#pragma unroll
        for (int e = 0; e < 4; ++e) best[e] = max(best[e], d[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) c[0][e] = best[e];
    }
    // c: pages gr and gr + 8, columns 2 t4 and 2 t4 + 1
    const int mine = u * 16 + gr + 8 * odd_quarter;
    const float sc = __shfl_sync(0xffffffffu, scale, mine);
    const bool here = (there >> mine) & 1u;
    if (GP || Gp >= 4) {
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        int lo = max(c[x][0], c[x][1]), hi = max(c[x][2], c[x][3]);
        lo = max(lo, __shfl_xor_sync(0xffffffffu, lo, 1)), hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
        if (Gp == 8) lo = max(lo, __shfl_xor_sync(0xffffffffu, lo, 2)), hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, 2));
        largest[x] = max(largest[x], keep(x * (8 / Gp) + tok0, most_of[x], i0 + mine, odd_quarter ? hi : lo, sc, here));
      }
    } else {
      const float other = __shfl_sync(0xffffffffu, scale, mine ^ 8), sc_lo = odd_quarter ? other : sc, sc_hi = odd_quarter ? sc : other;
      const int lo_page = u * 16 + gr, hi_page = lo_page + 8;
      const bool lo_here = (there >> lo_page) & 1u, hi_here = (there >> hi_page) & 1u;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        if (Gp == 2) {
          const int tok = x * 4 + t4, most = tok < TT ? s_cand[tok] : 0;
          note(tok, keep(tok, most, i0 + lo_page, max(c[x][0], c[x][1]), sc_lo, lo_here));
          note(tok, keep(tok, most, i0 + hi_page, max(c[x][2], c[x][3]), sc_hi, hi_here));
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int tok = x * 8 + t4 * 2 + e, most = tok < TT ? s_cand[tok] : 0;
            note(tok, keep(tok, most, i0 + lo_page, c[x][e], sc_lo, lo_here));
            note(tok, keep(tok, most, i0 + hi_page, c[x][2 + e], sc_hi, hi_here));
          }
        }
      }
    }
  };
  // while 16 pages are scored the next 16 are on their way, and the blocks of the 32 behind them
  uint32_t even[KS][4], odd[KS][4];
  const auto scales_of = [&](int block) { return block >= 0 ? p.scales[(size_t)block * p.Hkv + h] : 0.f; };
  const int step = SELECT_THREADS * share;
  int i0 = rank * SELECT_THREADS + warp * 32, block = locate(i0 + lane), next = locate(i0 + step + lane);
  float scale = scales_of(block);
  if (i0 < cand) fetch(even, block, 0);
  for (; i0 < cand; i0 += step) {
    const uint32_t there = __ballot_sync(0xffffffffu, block >= 0);
    fetch(odd, block, 1);
    score(even, i0, 0, scale, there);
    const float here = scale;
    block = next;
    next = locate(i0 + 2 * step + lane);
    scale = scales_of(block);
    if (i0 + step < cand) fetch(even, block, 0);
    score(odd, i0, 1, here, there);
  }
#pragma unroll
  for (int x = 0; x < NT; ++x)
    if (most_of[x] > 0 && largest[x]) atomicMax(&s_largest[x * (8 / Gp) + tok0], largest[x]);
  __syncthreads();
  if (CL) {
    if (rank > 0 && tid == 0) {
      uint32_t to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(s_largest)));
      asm volatile("red.shared::cluster.max.u32 [%0], %1;" ::"r"(to), "r"(s_largest[0]) : "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank > 0) return;
  }
  // The team's and its token's numbers once more: kept over the scores, where registers are short, they are spilled.
  int self;
  asm volatile("mov.u32 %0, %%tid.x;" : "=r"(self));
  __builtin_assume(self >= 0 && self < SELECT_THREADS);
  const Team<TEAM> choosing(self);
  const int of = s_cand[choosing.id];              // this token's candidates
  if (of == 0) return;                             // whole teams leave
  int* to = p.pages + ((size_t)(t0 + choosing.id) * p.Hkv + h) * (p.first + p.top + p.last) + p.first;
  choose_in_order(choosing, keys + choosing.id * ldkeys, of, p.top, s_largest[choosing.id], reinterpret_cast<int*>(select_smem) + choosing.id * SELECT_INTS,
                  [&](int place, int i) { to[place] = p.first + i; });
}

// Tokens of a block: as many as the 16 columns of two products hold (4 at most), where sequences have them, as long as the scores leave room for two blocks on an SM.
int select_tokens(int uniform, int G, int pages) {
  int Gp = 1, TT = 1;
  while (Gp < G) Gp <<= 1;
  while (TT < 4 && TT * 2 * Gp <= (TT == 1 ? 8 : 16) && TT < uniform && (long long)TT * 2 * pages * 4 <= 64 * 1024) TT *= 2;
  return TT;
}

template <int TT, int KS, bool FULL, int GP, bool CL = false>
int launch_select(const SelectParams& p, cudaStream_t s) {
  const size_t smem = TT * ((size_t)SELECT_INTS * 4 + (size_t)p.G * 32 * KS + 4 * (size_t)((p.max_blocks + 3) & ~3));
  auto kernel = page_select_kernel<TT, KS, FULL, GP, CL>;
  if (smem > 47 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -(int)e;
  }
  const dim3 grid((unsigned)(p.num_seqs * ((p.uniform_q + TT - 1) / TT) * p.Hkv * (CL ? p.share : 1)));
  if (!CL) return launch_kernel(kernel, grid, dim3(SELECT_THREADS), smem, s, p);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = dim3(SELECT_THREADS), cfg.dynamicSmemBytes = smem, cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.share, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess ? 0 : -(int)e;
}

template <int KS, bool FULL, int GP>
int launch_select(SelectParams p, cudaStream_t s) {
  // few problems over many pages: up to 8 blocks each, of 256 pages and more
  const long long problems = (long long)p.num_seqs * p.uniform_q * p.Hkv;
  p.share = 1;
  while (p.share < 8 && p.share * 512 <= p.max_blocks && problems * p.share * 2 <= 2 * 148) p.share *= 2;
  if (p.share > 1) return launch_select<1, KS, FULL, GP, true>(p, s);
  const int TT = select_tokens(p.uniform_q, p.G, p.max_blocks);
  if constexpr (GP != 8) {                         // eight heads fill a product's columns with one token
    if (TT == 4) return launch_select<4, KS, FULL, GP>(p, s);
    if (TT == 2) return launch_select<2, KS, FULL, GP>(p, s);
  }
  return launch_select<1, KS, FULL, GP>(p, s);
}

// Groups of 3 or 4 and of 5 to 8 heads of 128 columns have kernels of their own: without the choice of the reduction and the ends of rows in the loop they
// issue fewer instructions a page.
int launch_select(const SelectParams& p, cudaStream_t s) {
  if (p.D == 128 && (reinterpret_cast<uintptr_t>(p.codes) & 15) == 0 && p.G > 2 && p.G <= 8) return p.G <= 4 ? launch_select<4, true, 4>(p, s) : launch_select<4, true, 8>(p, s);
  return p.D <= 128 ? launch_select<4, false, 0>(p, s) : launch_select<8, false, 0>(p, s);
}

}  // namespace
}  // namespace swb

extern "C" {

// See SummaryParams. dims: host int[9] = num_seqs, max new tokens of a sequence, table width, blocks, block_size, Hkv, D, fp32, 0.
int swb_page_summaries(const int* dims, const void* k, void* codes, void* scales, const int* table, long long table_stride, const int* cu_q,
                       const int* kv_lens, void* stream) {
  using namespace swb;
  const int seqs = dims[0], max_q = dims[1], max_blocks = dims[2], blocks = dims[3], bs = dims[4], Hkv = dims[5], D = dims[6], fp32 = dims[7];
  if (seqs <= 0 || max_q <= 0 || max_blocks <= 0) return 0;
  if (bs < 1 || Hkv < 1 || D < 1 || D > 256 || blocks < 1 || seqs > 65535 || (long long)max_blocks * bs > INT_MAX || !k || !codes || !scales || !table || !kv_lens) return -3;
  const SummaryParams p{k, reinterpret_cast<int8_t*>(codes), reinterpret_cast<float*>(scales), table, table_stride, max_blocks, blocks, bs, Hkv, D, cu_q, kv_lens, seqs, max_q};
  // n new tokens complete at most (n + bs - 1) / bs pages
  const dim3 grid((max_q - 1) / bs + 1, (Hkv + SUMMARY_WARPS - 1) / SUMMARY_WARPS, seqs);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 block(SUMMARY_WARPS * 32);
  if (!fp32 && D <= 128 && D % 4 == 0 && ((reinterpret_cast<uintptr_t>(k) & 7) | (reinterpret_cast<uintptr_t>(codes) & 3)) == 0)
    return bs == 16 ? launch_kernel(page_summary_quads_kernel<true>, grid, block, 0, s, p) : launch_kernel(page_summary_quads_kernel<false>, grid, block, 0, s, p);
  if (D <= 128) return fp32 ? launch_kernel(page_summary_kernel<float, 4>, grid, block, 0, s, p) : launch_kernel(page_summary_kernel<bf16, 4>, grid, block, 0, s, p);
  return fp32 ? launch_kernel(page_summary_kernel<float, 8>, grid, block, 0, s, p) : launch_kernel(page_summary_kernel<bf16, 8>, grid, block, 0, s, p);
}

// out [rows, D] = codes [rows, D] * scales [rows].
int swb_page_values(const void* codes, const void* scales, float* out, long long rows, int D, void* stream) {
  using namespace swb;
  if (rows <= 0) return 0;
  if (D < 1 || !codes || !scales || !out) return -3;
  const long long n = rows * D;
  const int four = D % 4 == 0 && (reinterpret_cast<uintptr_t>(codes) & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const long long want = (n / (four ? 4 : 1) + 255) / 256, blocks = want < 8 * 148 ? want : 8 * 148;
  return launch_kernel(page_values_kernel, dim3((unsigned)(blocks < 1 ? 1 : blocks)), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), reinterpret_cast<const int8_t*>(codes),
                       reinterpret_cast<const float*>(scales), out, n, D, four);
}

// See SelectParams. dims: host int[14] = tokens, num_seqs, tokens of each sequence (with cu_q: at most), table width, blocks, block_size, Hkv, G, D, first,
// top, last, fp32, 0.
int swb_page_select(const int* dims, const void* q, long long q_stride_tok, long long q_stride_head, const void* codes, const void* scales, const int* table,
                    long long table_stride, const int* cu_q, const int* kv_lens, int* pages, int* counts, void* stream) {
  using namespace swb;
  const int T = dims[0], seqs = dims[1], uniform = dims[2], max_blocks = dims[3], blocks = dims[4], bs = dims[5], Hkv = dims[6], G = dims[7], D = dims[8];
  const int first = dims[9], top = dims[10], last = dims[11], fp32 = dims[12];
  if (T <= 0 || seqs <= 0) return 0;
  if ((long long)seqs * uniform * Hkv > INT_MAX / 8 || bs < 1 || Hkv < 1 || G < 1 || D < 1 || blocks < 1 || max_blocks < 1 || first < 0 || top < 0 || last < 1 || (long long)first + top + last > INT_MAX || uniform < 1 || D > 256 || (long long)max_blocks * bs > INT_MAX || !q || !codes ||
      !scales || !table || !kv_lens || !pages || !counts)
    return -3;
  // a token's histogram, codes and scores in one block's shared memory
  if (4ll * SELECT_INTS + (long long)G * (D <= 128 ? 128 : 256) + 4ll * ((max_blocks + 3) & ~3) > 200 * 1024) return -3;
  const SelectParams p{q, q_stride_tok, q_stride_head, reinterpret_cast<const int8_t*>(codes), reinterpret_cast<const float*>(scales), table, table_stride,
                       max_blocks, blocks, bs, Hkv, G, D, cu_q, kv_lens, seqs, uniform, T, first, top, last, pages, counts, fp32,
                       !fp32 && (reinterpret_cast<uintptr_t>(q) & 15) == 0 && (q_stride_tok | q_stride_head) % 8 == 0, 1};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return launch_select(p, s);
}

}  // extern "C"
