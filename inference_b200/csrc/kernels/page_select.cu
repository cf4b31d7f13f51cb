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

// A warp per (page, head); lane l holds columns l, l + 32, ... of up to COLS * 32.
template <typename E, int COLS>
__global__ void __launch_bounds__(SUMMARY_WARPS * 32) page_summary_kernel(const SummaryParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int h = blockIdx.y * SUMMARY_WARPS + (threadIdx.x >> 5), seq = blockIdx.z;
  if (h >= p.Hkv) return;
  const int q_len = p.cu_q ? p.cu_q[seq + 1] - p.cu_q[seq] : p.uniform_q;
  const int len = min(p.kv_lens[seq], p.max_blocks * p.bs);
  const int page = max(len - q_len, 0) / p.bs + blockIdx.x;      // the first page that the new tokens can complete, and on
  if ((page + 1) * p.bs > len || q_len <= 0) return;
  const int block = p.table[seq * p.table_stride + page];
  if ((unsigned)block >= (unsigned)p.num_blocks) return;
  const size_t at = (size_t)block * p.Hkv + h;
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
    if (d < p.D) p.codes[at * p.D + d] = bad || a == 0.0 ? (int8_t)0 : (int8_t)(int)rint(127.0 * s[c] / a);
  }
  if (lane == 0) p.scales[at] = bad ? NAN : (float)(a / (127.0 * p.bs));
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
};

constexpr int SELECT_THREADS = 256;

// A block per (token, head). Shared memory: keys [pages], codes of the group's queries [G, D rounded up to 16].
template <typename E>
__global__ void __launch_bounds__(SELECT_THREADS) page_select_kernel(const SelectParams p) {
  pdl_launch_dependents();
  extern __shared__ uint4 select_smem[];
  __shared__ int hist[SELECT_BINS + 64];
  __shared__ float s_amax[SELECT_THREADS / 32];
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.x % p.Hkv, t = blockIdx.x / p.Hkv;
  const int Dp = (p.D + 15) & ~15;
  int8_t* qc = reinterpret_cast<int8_t*>(select_smem);
  uint32_t* keys = reinterpret_cast<uint32_t*>(qc + p.G * Dp);
  if (tid == 0) s_bad = 0;
  pdl_wait();
  if (p.cu_q && t >= p.cu_q[p.num_seqs]) return;          // behind the last sequence
  const int seq = seq_of_token(p.cu_q, p.num_seqs, p.uniform_q, t);
  const int q0 = p.cu_q ? p.cu_q[seq] : seq * p.uniform_q, q_len = p.cu_q ? p.cu_q[seq + 1] - q0 : p.uniform_q;
  const int seen = min(p.kv_lens[seq] - (q_len - 1 - (t - q0)), p.max_blocks * p.bs);
  const int n = seen > 0 ? (seen + p.bs - 1) / p.bs : 0;
  const int width = p.first + p.top + p.last;
  int* out = p.pages + ((size_t)t * p.Hkv + h) * width;
  if (tid == 0) p.counts[(size_t)t * p.Hkv + h] = min(n, width);
  if (n <= width) {
    for (int i = tid; i < width; i += SELECT_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  for (int i = tid; i < p.first; i += SELECT_THREADS) out[i] = i;
  for (int i = tid; i < p.last; i += SELECT_THREADS) out[p.first + p.top + i] = n - p.last + i;
  if (p.top == 0) return;
  __syncthreads();                                         // s_bad is set
  // the group's queries as codes of one step
  const E* q = reinterpret_cast<const E*>(p.q) + t * p.q_stride_tok + (size_t)h * p.G * p.q_stride_head;
  float a = 0.f;
  bool bad = false;
  for (int i = tid; i < p.G * p.D; i += SELECT_THREADS) {
    const float x = fabsf(to_f(q[(i / p.D) * p.q_stride_head + i % p.D]));
    a = fmaxf(a, x);
    bad |= !(x < INFINITY);
  }
  a = warp_max(a);
  if (lane == 0) s_amax[warp] = a;
  if (bad) s_bad = 1;
  __syncthreads();
  a = 0.f;
#pragma unroll
  for (int w = 0; w < SELECT_THREADS / 32; ++w) a = fmaxf(a, s_amax[w]);
  bad = s_bad != 0;
  for (int i = tid; i < p.G * Dp; i += SELECT_THREADS) {
    const int g = i / Dp, d = i % Dp;
    const float x = d < p.D ? to_f(q[g * p.q_stride_head + d]) : 0.f;
    qc[i] = bad || a == 0.f ? (int8_t)0 : (int8_t)(int)rint(127.0 * (double)x / (double)a);
  }
  __syncthreads();
  const int cand = n - p.first - p.last;
  for (int i = tid; i < cand; i += SELECT_THREADS) {
    const int block = p.table[seq * p.table_stride + p.first + i];
    float score = -INFINITY;                               // a page that is not there ranks last
    if ((unsigned)block < (unsigned)p.num_blocks) {
      const size_t at = (size_t)block * p.Hkv + h;
      const int8_t* c = p.codes + at * p.D;
      int best = INT_MIN;
      for (int g = 0; g < p.G; ++g) {
        int dot = 0;
        for (int d = 0; d < p.D; ++d) dot += (int)c[d] * (int)qc[g * Dp + d];
        best = max(best, dot);
      }
      score = __fmul_rn((float)best, p.scales[at]);
    }
    keys[i] = float_key(score);
  }
  const auto key = [&](int i) { return keys[i]; };
  __syncthreads();
  const Threshold th = select_threshold<SELECT_THREADS>(key, cand, p.top, hist);
  const int seg = ((cand + SELECT_THREADS - 1) / SELECT_THREADS) * 32;
  const int lo = min(warp * seg, cand), hi = min(lo + seg, cand);
  int gt = 0, eq = 0;
  for (int i = lo + lane; i < hi; i += 32) gt += keys[i] > th.key, eq += keys[i] == th.key;
  gt = __reduce_add_sync(0xffffffffu, gt), eq = __reduce_add_sync(0xffffffffu, eq);
  const int eq_before = warps_before<SELECT_THREADS>(eq, hist), gt_before = warps_before<SELECT_THREADS>(gt, hist);
  int* to = out + p.first + gt_before + min(eq_before, th.ties);
  for_each_choice(key, th, lo, hi, eq_before, [&](int i, bool in, int before) {
    if (in) to[before] = p.first + i;
  });
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
  if (bs < 1 || Hkv < 1 || D < 1 || D > 256 || blocks < 1 || seqs > 65535 || !k || !codes || !scales || !table || !kv_lens) return -3;
  const SummaryParams p{k, reinterpret_cast<int8_t*>(codes), reinterpret_cast<float*>(scales), table, table_stride, max_blocks, blocks, bs, Hkv, D, cu_q, kv_lens, seqs, max_q};
  // n new tokens complete at most (n + bs - 1) / bs pages
  const dim3 grid((max_q + bs - 1) / bs, (Hkv + SUMMARY_WARPS - 1) / SUMMARY_WARPS, seqs);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 block(SUMMARY_WARPS * 32);
  if (D <= 128) return fp32 ? launch_kernel(page_summary_kernel<float, 4>, grid, block, 0, s, p) : launch_kernel(page_summary_kernel<bf16, 4>, grid, block, 0, s, p);
  return fp32 ? launch_kernel(page_summary_kernel<float, 8>, grid, block, 0, s, p) : launch_kernel(page_summary_kernel<bf16, 8>, grid, block, 0, s, p);
}

// Bytes of shared memory that a selection over `pages` pages needs; above the limit of a block it is refused.
long long swb_page_select_smem(int pages, int G, int D) { return (long long)G * ((D + 15) & ~15) + 4ll * pages; }

// See SelectParams. dims: host int[14] = tokens, num_seqs, tokens of each sequence (without cu_q), table width, blocks, block_size, Hkv, G, D, first,
// top, last, fp32, 0.
int swb_page_select(const int* dims, const void* q, long long q_stride_tok, long long q_stride_head, const void* codes, const void* scales, const int* table,
                    long long table_stride, const int* cu_q, const int* kv_lens, int* pages, int* counts, void* stream) {
  using namespace swb;
  const int T = dims[0], seqs = dims[1], uniform = dims[2], max_blocks = dims[3], blocks = dims[4], bs = dims[5], Hkv = dims[6], G = dims[7], D = dims[8];
  const int first = dims[9], top = dims[10], last = dims[11], fp32 = dims[12];
  if (T <= 0 || seqs <= 0) return 0;
  if ((long long)T * Hkv > INT_MAX || bs < 1 || Hkv < 1 || G < 1 || D < 1 || blocks < 1 || max_blocks < 1 || first < 0 || top < 0 || last < 1 || (!cu_q && uniform < 1) || !q || !codes ||
      !scales || !table || !kv_lens || !pages || !counts)
    return -3;
  const long long smem = swb_page_select_smem(max_blocks, G, D);
  if (smem > 200 * 1024) return -3;
  const SelectParams p{q, q_stride_tok, q_stride_head, reinterpret_cast<const int8_t*>(codes), reinterpret_cast<const float*>(scales), table, table_stride,
                       max_blocks, blocks, bs, Hkv, G, D, cu_q, kv_lens, seqs, uniform, T, first, top, last, pages, counts};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto kernel = fp32 ? page_select_kernel<float> : page_select_kernel<bf16>;
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return -(int)e;
  }
  return launch_kernel(kernel, dim3(Hkv * T), dim3(SELECT_THREADS), (size_t)smem, s, p);
}

}  // extern "C"
