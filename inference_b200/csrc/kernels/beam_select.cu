// The best continuations of several beams: of all pairs (beam k, token v) of a prompt the `count` of largest score s_k + x_kv - log sum_u exp x_ku, equal ones in the order of
// beam and token.
//
// Two scores may differ in the last bits of 32-bit numbers only, and which of them is the better one decides which beam lives. So sums of exponentials, logarithms and scores are
// 64-bit numbers, rounded once when they are handed out. Within a beam the order is that of the logits, which takes none of them.
//
// The first launch reads every logit once: a block holds a piece of a row in registers, takes its maximum, its sum of exponentials and its `count` largest logits. A bound for these
// comes from the threads' own maxima: `count` threads have one at least as large as the count-th largest of them, so that no smaller logit is among the `count` largest, and few others are
// as large. The second launch joins the pieces, one block a prompt. Rows of beams that are not alive (scores that are not finite) are not read.
#include "common.cuh"

#include <climits>

namespace swb {

SWB_REGISTER_STATUS_UNIT(beam_select);

namespace {

constexpr int MAX_COUNT = 128, MAX_BEAMS = 256, CHUNK_THREADS = 256, ROOM = 1024;

struct Entry {
  float x;
  int token;                 // -1: none
};
struct Piece {
  double sum;                // of exp(x - top)
  double top;                // -inf: no logit is allowed; +inf: one of them is no number
};

struct BeamParams {
  const void* logits;
  long long stride;
  const float* scores;       // [batch, beams]
  int batch, beams, vocab, count, pieces;
  Piece* piece;              // [rows, pieces]
  Entry* best;               // [rows, pieces, count], in order
  float* out_scores;         // [batch, count]
  int* out_beams;
  long long* out_tokens;
};

__device__ __forceinline__ bool alive(float score) { return isfinite(score); }

__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// V numbers of 16 bytes
template <typename E>
__device__ __forceinline__ void load16(const E* p, float* x) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(E) == 4) x[i] = __uint_as_float(w[i]);
    else x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <typename E, int EPT>
__global__ void __launch_bounds__(CHUNK_THREADS) beam_chunk_kernel(const BeamParams p) {
  pdl_launch_dependents();
  constexpr int W = 16 / sizeof(E), VECS = EPT / W, WARPS = CHUNK_THREADS / 32;
  __shared__ __align__(16) float s_max[CHUNK_THREADS];
  __shared__ Entry s_found[ROOM];
  __shared__ double s_sum[WARPS];
  __shared__ float s_bound;
  __shared__ int s_count, s_tally[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.y, n = p.count;
  pdl_wait();
  if (!alive(p.scores[row])) return;
  const E* from = reinterpret_cast<const E*>(p.logits) + row * p.stride;
  const int ahead = (int)((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(E));       // numbers of the row's first 16 bytes that are not its own
  const int first = blockIdx.x * CHUNK_THREADS * EPT - ahead;
  float x[EPT];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int at = first + (i * CHUNK_THREADS + tid) * W;
    if (at >= 0 && at + W <= p.vocab) {
      load16(from + at, x + i * W);
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) x[i * W + j] = at + j >= 0 && at + j < p.vocab ? to_f(from[at + j]) : -INFINITY;
    }
  }
  const auto token_of = [&](int e) { return first + ((e / W) * CHUNK_THREADS + tid) * W + e % W; };
  float mine = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < EPT; ++e) bad = bad || !(x[e] < INFINITY), mine = fmaxf(mine, x[e]);
  s_max[tid] = mine;
  if (tid == 0) s_count = 0, s_bound = -INFINITY;
  if (tid < 2) s_tally[tid] = 0;
  bad = __syncthreads_or(bad);
  // rank of the thread's maximum among all threads'
  int rank = 0;
  float top = -INFINITY;
  for (int j = 0; j < CHUNK_THREADS; j += 4) {
    const float4 y = *reinterpret_cast<const float4*>(s_max + j);
    rank += (y.x > mine || (y.x == mine && j < tid)) + (y.y > mine || (y.y == mine && j + 1 < tid)) + (y.z > mine || (y.z == mine && j + 2 < tid)) +
            (y.w > mine || (y.w == mine && j + 3 < tid));
    top = fmaxf(top, fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
  }
  if (rank == n - 1) s_bound = mine;
  double sum = 0.0;
  if (top > -INFINITY && !bad) {
#pragma unroll
    for (int e = 0; e < EPT; ++e) sum += exp((double)x[e] - (double)top);
  }
  sum = warp_sum64(sum);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  const long long at = (long long)row * p.pieces + blockIdx.x;
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w) sum += s_sum[w];
    p.piece[at] = Piece{sum, bad ? (double)INFINITY : (double)top};
  }
  if (bad) return;                                         // the row offers nothing
  const float bound = s_bound;
#pragma unroll
  for (int e = 0; e < EPT; ++e)
    if (x[e] >= bound && x[e] > -INFINITY) {
      const int i = atomicAdd(&s_count, 1);
      if (i < ROOM) s_found[i] = Entry{x[e], token_of(e)};
    }
  __syncthreads();
  int found = s_count;
  if (found > ROOM) {
    // Many logits as large as the bound (ties): the count-th largest by halving the range of the logits' bit patterns, and of equal ones the first tokens.
    int turn = 0;
    const auto tally = [&](auto test) {
      int c = 0;
#pragma unroll
      for (int e = 0; e < EPT; ++e) c += x[e] > -INFINITY && test(e);
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) atomicAdd(&s_tally[turn], c);
      __syncthreads();
      c = s_tally[turn];
      turn ^= 1;
      if (tid == 0) s_tally[turn] = 0;                     // of the round before, which all have read
      __syncthreads();
      return c;
    };
    unsigned key = 0;
    for (int b = 31; b >= 0; --b) {
      const unsigned next = key | 1u << b;
      if (tally([&](int e) { return order_of(x[e]) >= next; }) >= n) key = next;
    }
    const int need = n - tally([&](int e) { return order_of(x[e]) > key; });
    int limit = 0;                                         // the last of them is at this place
    for (int b = 30; b >= 0; --b) {
      const int next = limit | 1 << b;
      if (tally([&](int e) { return order_of(x[e]) == key && token_of(e) < next; }) < need) limit = next;
    }
    if (tid == 0) s_count = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EPT; ++e)
      if (x[e] > -INFINITY && (order_of(x[e]) > key || (order_of(x[e]) == key && token_of(e) <= limit))) s_found[atomicAdd(&s_count, 1)] = Entry{x[e], token_of(e)};
    __syncthreads();
    found = s_count;
  }
  Entry* out = p.best + at * n;
  for (int i = tid; i < found; i += CHUNK_THREADS) {
    const Entry me = s_found[i];
    int before = 0;
    for (int j = 0; j < found; ++j) {
      const Entry e = s_found[j];
      before += e.x > me.x || (e.x == me.x && e.token < me.token);
    }
    if (before < n) out[before] = me;
  }
  for (int i = found + tid; i < n; i += CHUNK_THREADS) out[i] = Entry{-INFINITY, -1};
}

// ---- one block a prompt -----------------------------------------------------------------------------------------------------------------------------
constexpr int JOIN_THREADS = 512;

struct Choice {
  double s;
  long long at;              // beam * vocab + token
};
__device__ __forceinline__ bool better(double s, long long at, const Choice& c) { return s > c.s || (s == c.s && at < c.at); }

__global__ void __launch_bounds__(JOIN_THREADS) beam_join_kernel(const BeamParams p) {
  pdl_launch_dependents();
  __shared__ double s_log[MAX_BEAMS];                      // of a beam's sum of exponentials; NaN: it offers nothing
  __shared__ double s_max[JOIN_THREADS];
  __shared__ Choice s_found[ROOM];
  __shared__ Choice s_warp[JOIN_THREADS / 32];
  __shared__ double s_bound;
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x, n = p.count, K = p.beams;
  pdl_wait();
  const float* score = p.scores + (long long)b * K;
  if (tid == 0) s_count = 0, s_bound = -INFINITY;
  for (int k = warp; k < K; k += JOIN_THREADS / 32) {
    const Piece* piece = p.piece + ((long long)b * K + k) * p.pieces;
    double top = -INFINITY, sum = 0.0;
    if (alive(score[k])) {
      for (int i = lane; i < p.pieces; i += 32) top = fmax(top, piece[i].top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (isfinite(top))
        for (int i = lane; i < p.pieces; i += 32) sum += piece[i].top > -INFINITY ? piece[i].sum * exp(piece[i].top - top) : 0.0;
      sum = warp_sum64(sum);
    }
    if (lane == 0) s_log[k] = isfinite(top) ? top + log(sum) : (double)NAN;
  }
  __syncthreads();
  const int per_beam = p.pieces * n, total = K * per_beam;
  const Entry* best = p.best + (long long)b * total;
  // the i-th candidate; s = -inf: none
  const auto candidate = [&](int i) {
    const int k = i / per_beam;
    Choice c{-INFINITY, LLONG_MAX};
    const double log_sum = s_log[k];
    if (log_sum != log_sum) return c;
    const Entry e = best[i];
    if (e.token < 0) return c;
    c.s = (double)score[k] + ((double)e.x - log_sum);
    c.at = (long long)k * p.vocab + e.token;
    return c;
  };
  double mine = -INFINITY;
  for (int i = tid; i < total; i += JOIN_THREADS) mine = fmax(mine, candidate(i).s);
  s_max[tid] = mine;
  __syncthreads();
  int rank = 0;
  for (int j = 0; j < JOIN_THREADS; ++j) rank += s_max[j] > mine || (s_max[j] == mine && j < tid);
  if (rank == n - 1) s_bound = mine;
  __syncthreads();
  const double bound = s_bound;
  for (int i = tid; i < total; i += JOIN_THREADS) {
    const Choice c = candidate(i);
    if (c.s >= bound && c.s > -INFINITY) {
      const int at = atomicAdd(&s_count, 1);
      if (at < ROOM) s_found[at] = c;
    }
  }
  __syncthreads();
  const int found = s_count;
  const auto store = [&](int at, const Choice& c) {
    const long long to = (long long)b * n + at;
    const bool none = !(c.s > -INFINITY);
    p.out_scores[to] = (float)c.s;
    p.out_beams[to] = none ? -1 : (int)(c.at / p.vocab);
    p.out_tokens[to] = none ? -1 : c.at % p.vocab;
  };
  if (found <= ROOM) {
    for (int i = tid; i < found; i += JOIN_THREADS) {
      const Choice me = s_found[i];
      int before = 0;
      for (int j = 0; j < found; ++j) before += better(s_found[j].s, s_found[j].at, me);
      if (before < n) store(before, me);
    }
    for (int i = found + tid; i < n; i += JOIN_THREADS) store(i, Choice{-INFINITY, LLONG_MAX});
    return;
  }
  // more ties than there is room for: one after the other
  Choice last{INFINITY, -1};
  for (int r = 0; r < n; ++r) {
    Choice c{-INFINITY, LLONG_MAX};
    for (int i = tid; i < total; i += JOIN_THREADS) {
      const Choice x = candidate(i);
      if ((x.s < last.s || (x.s == last.s && x.at > last.at)) && better(x.s, x.at, c)) c = x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Choice y{__shfl_xor_sync(0xffffffffu, c.s, o), __shfl_xor_sync(0xffffffffu, c.at, o)};
      if (better(y.s, y.at, c)) c = y;
    }
    if (lane == 0) s_warp[warp] = c;
    __syncthreads();
    for (int w = 0; w < JOIN_THREADS / 32; ++w)
      if (better(s_warp[w].s, s_warp[w].at, c)) c = s_warp[w];
    if (tid == 0) store(r, c);
    last = c;
    __syncthreads();
  }
}

constexpr int EPT = 32;

}  // namespace
}  // namespace swb

extern "C" {

// Pieces that a row of `vocab` logits is read in, and bytes of workspace a row and piece of it needs.
int swb_beam_pieces(int vocab, int count, long long* bytes) {
  using namespace swb;
  const long long step = CHUNK_THREADS * EPT;
  *bytes = (long long)sizeof(Piece) + (long long)sizeof(Entry) * count;
  return (int)((vocab + 7ll + step - 1) / step);
}

// logits [batch * beams, vocab], rows `stride` numbers apart; scores [batch, beams]. workspace (16-byte aligned): batch beams pieces bytes of swb_beam_pieces.
int swb_beam_select(const void* logits, long long stride, int fp32, const float* scores, int batch, int beams, int vocab, int count, float* out_scores, int* out_beams, void* out_tokens,
                    void* workspace, long long workspace_bytes, void* stream) {
  using namespace swb;
  if (batch <= 0) return 0;
  BeamParams p = {};
  long long bytes = 0;
  if (!logits || !scores || !out_scores || !out_beams || !out_tokens || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || beams < 1 || beams > MAX_BEAMS || vocab < 1 ||
      vocab > INT_MAX - 65536 || count < 1 || count > MAX_COUNT || (long long)batch * beams > 65535)
    return -3;
  p.pieces = swb_beam_pieces(vocab, count, &bytes);
  const long long rows = (long long)batch * beams;
  if (rows * p.pieces * bytes > workspace_bytes || (long long)beams * p.pieces * count > INT_MAX) return -3;
  p.logits = logits, p.stride = stride, p.scores = scores, p.batch = batch, p.beams = beams, p.vocab = vocab, p.count = count;
  p.piece = reinterpret_cast<Piece*>(workspace), p.best = reinterpret_cast<Entry*>(p.piece + rows * p.pieces);
  p.out_scores = out_scores, p.out_beams = out_beams, p.out_tokens = reinterpret_cast<long long*>(out_tokens);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(p.pieces, (unsigned)rows);
  const int rc = fp32 ? launch_kernel(beam_chunk_kernel<float, EPT>, grid, dim3(CHUNK_THREADS), 0, s, p) : launch_kernel(beam_chunk_kernel<bf16, EPT>, grid, dim3(CHUNK_THREADS), 0, s, p);
  if (rc) return rc;
  return launch_kernel(beam_join_kernel, dim3(batch), dim3(JOIN_THREADS), 0, s, p);
}

}  // extern "C"
