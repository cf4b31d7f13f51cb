// The best continuations of several beams: of all pairs (beam k, token v) of a prompt the `count` of largest score s_k + x_kv - log sum_u exp x_ku, equal ones in the order of
// beam and token.
//
// Two scores may differ in the last bits of 32-bit numbers only, and which of them is the better one decides which beam lives. So logarithms and scores are 64-bit numbers, rounded once when
// they are handed out, and an exponential, and a sum of however many, is within 2^-28.5 of its value. Within a beam the order is that of the logits, which takes none of them.
//
// The first launch reads every logit once: a block walks over a piece of a row, 16 logits a thread at a time with the next ones on their way, adds up their exponentials and keeps a note of the
// sixteens whose largest may be among its `count` largest; their logits are looked at in the end, when the bound for these is tight. It comes from the threads' own maxima so far: each of
// the eight warps gives its (count / 8)-th largest, and the smallest of these has `count` logits at least as large as itself, of different threads, and not many more; it is raised behind 1, 2, 4, 8..
// steps. The second launch joins the pieces, one block a prompt, with a bound from their ordered lists. Rows of beams that are not alive (scores that are not finite) are not read.
//
// Measured on the device: 32 prompts of 8 beams over 128 256 tokens (131 MB) 59 us (bf16, half the bytes: 55), of them some 12 the join; the pieces alone would take 27 without exponentials, at 18 to 19
// instructions a logit. A warp there waits 12 cycles between two instructions: 2.6 for logits, 2.1 for results of the multiply-adds, 1.5 each for the table's numbers and for its turn, 1.2 each for barriers and
// for a pipe that is busy; 41 % of the issue slots are used, with 3.5 blocks to an SM of the four that it holds. 4 beams of one prompt 16 us, of them 7 the pieces; 50 beams of 3 prompts, 100 continuations, 60 to
// 65 us. With exponentials and sums in 64 bits throughout it took 178, 22 and 135 us, with the candidates looked up as they came and ranked one by one 75, 22 and 150.
//
// Where more than 1024 sixteens, or logits, of a piece are as large as its bound (ties of a finite number in place of tokens that are not allowed, logits that rise with the token's number), the piece is gone
// through some 65 times: 4 beams over 128 256 tokens 90 us where logits rise, 122 where all are alike, 96 with five tokens allowed and -1e9 for the others, 14 with -inf for them.
//
// Exponentials run on the multiply-add pipes, two at a time, by the table method of Tang (1989): x = k ln2 / 32 + r, where k times the first part of ln2 / 32 leaves x without a rounding, and e^x = 2^(k / 32) (1 +
// e^r - 1) with 2^(k mod 32 / 32) from a table of two numbers each; the top's whole power of two leaves the exponent, so that nothing is larger than two. What a sum rounds off is added up beside it:
// the sum starts at two, and no part is larger, so that one subtraction gives what was really added, and the rest of a part is a small number. (Adding up e^r - 1 beside the table's numbers took an operation
// less; with hundreds of equal logits a thread its roundings all went one way, 6e-8 of the sum.)
#include "attention_tc.cuh"

#include <cfloat>
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
  double sum;                // of e^(x - top)
  double top;                // -inf: no logit is allowed; +inf: one of them is no number
};

struct BeamParams {
  const void* logits;
  long long stride;
  const float* scores;       // [batch, beams]
  int batch, beams, vocab, count;
  int pieces, steps;         // of a row; of a piece
  Piece* piece;              // [rows, pieces]
  Entry* best;               // [rows, pieces, count], in order
  float* out_scores;         // [batch, count]
  int* out_beams;
  long long* out_tokens;
};

__device__ __forceinline__ bool alive(float score) { return isfinite(score); }

__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __float_as_uint(x + 0.f);             // zeros of both signs are one number
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float of_order(unsigned u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 16 bytes of numbers
template <typename E>
__device__ __forceinline__ void load16(const E* p, float* x) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(E) == 4) x[i] = __uint_as_float(w[i]);
    else x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// 2^(i / 32): a 32-bit number, and what is missing as a share of it
__constant__ float2 POWERS[32] = {
    {1.f, 0.f}, {1.0218972f, -4.70845762e-08f}, {1.04427373f, 4.62854715e-08f}, {1.06714046f, -5.56042252e-08f}, {1.09050775f, -1.19921575e-08f}, {1.1143868f, -4.87760623e-08f},
    {1.13878858f, 4.72978243e-08f}, {1.1637249f, -3.48144269e-08f}, {1.18920708f, 3.19341815e-08f}, {1.21524739f, -2.68866653e-08f}, {1.24185777f, 3.62105723e-08f}, {1.26905096f, 1.11842102e-09f},
    {1.29683959f, -3.09907193e-08f}, {1.32523668f, -2.63830096e-08f}, {1.35425556f, -7.47521334e-09f}, {1.38390994f, -4.24563567e-08f}, {1.41421354f, 1.71142709e-08f}, {1.44518077f, 2.30019666e-08f},
    {1.47682619f, -3.04768335e-08f}, {1.50916445f, -1.65385377e-08f}, {1.54221082f, 5.23333421e-09f}, {1.5759809f, -3.5920646e-08f}, {1.61049032f, 6.10759177e-09f}, {1.64575553f, -3.11405444e-08f},
    {1.68179286f, -1.47196051e-08f}, {1.71861935f, -2.82181016e-08f}, {1.75625217f, -5.25879518e-09f}, {1.79470909f, -6.36038733e-09f}, {1.8340081f, -6.12825968e-09f}, {1.87416768f, -2.48804088e-08f},
    {1.91520655f, 5.14060927e-09f}, {1.95714414f, -8.69726691e-09f}};
constexpr float PER_STEP = 46.1662407f, STEP_HIGH = 0.0216598511f, STEP_LOW = 9.98318228e-07f;      // 32 / ln 2; ln 2 / 32 in two parts, the first of 12 bits
constexpr float MAGIC = 12582912.f;                        // x + MAGIC has x rounded to a whole number in its low bits
constexpr float LEAST = 80.f;                              // what lies further below the top counts as that far: 2^-115 of it
constexpr float FAR = 30000.f;                             // |x| 32 / ln 2 is below 2^22

// large += e^x for two logits, at least e^least, over the power of two 2^((MAGIC - magic) / 32); small += what large rounds off
__device__ __forceinline__ void add_exponentials(float x0, float x1, float least, float magic, const float2* powers, unsigned long long& large, unsigned long long& small) {
  const unsigned long long x = pack2(fmaxf(x0, least), fmaxf(x1, least)), neg = pack2(-1.f, -1.f);
  const unsigned long long t = fma2(x, pack2(PER_STEP, PER_STEP), pack2(magic, magic)), k = add2(t, pack2(-magic, -magic));
  const unsigned long long r = fma2(k, pack2(-STEP_LOW, -STEP_LOW), fma2(k, pack2(-STEP_HIGH, -STEP_HIGH), x));      // |r| < 0.0115
  float t0, t1;
  unpack2(t, t0, t1);
  const int n0 = __float_as_int(t0), n1 = __float_as_int(t1);      // their low bits are k less the power of two's
  const float2 w0 = powers[n0 & 31], w1 = powers[n1 & 31];
  const unsigned long long q = fma2(fma2(fma2(r, pack2(1.f / 6.f, 1.f / 6.f), pack2(0.5f, 0.5f)), r, pack2(1.f, 1.f)), r, pack2(w0.y, w1.y));      // e^r - 1 and the table's share
  const unsigned long long v = pack2(__int_as_float((n0 & ~31) * (1 << 18) + __float_as_int(w0.x)), __int_as_float((n1 & ~31) * (1 << 18) + __float_as_int(w1.x)));
  const unsigned long long sum = add2(large, fma2(v, q, v)), less = fma2(sum, neg, large);      // less: what was added, exactly, with the other sign
  small = add2(small, fma2(v, q, add2(v, less)));                                                // and what of v + v q was not
  large = sum;
}

// A warp's numbers in descending order.
__device__ __forceinline__ float sort_warp(float v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, step);
      const bool down = (lane & size) == 0 || size == 32, first = (lane & step) == 0;
      v = down == first ? fmaxf(v, o) : fminf(v, o);
    }
  return v;
}

// The `nth` largest (from 1 on) of a warp's numbers, in every lane.
__device__ __forceinline__ float nth_largest(float v, int nth, int lane) {
  if (nth > 8) return __shfl_sync(0xffffffffu, sort_warp(v, lane), nth - 1);
  unsigned key = order_of(v), best = 0;                    // one after the other
  for (int i = 0; i < nth; ++i) {
    best = __reduce_max_sync(0xffffffffu, key);
    const unsigned there = __ballot_sync(0xffffffffu, key == best);
    if (lane == __ffs(there) - 1) key = 0;                 // below all numbers
  }
  return best ? of_order(best) : -INFINITY;
}

// The nth largest of the numbers of a block of eight warps: each warp sorts its own, and a number's rank is its place there and how many of each other warp's are before it (equal ones: the lower
// warp's first). sorted: 256 words of shared memory, which are not read any more when this begins.
__device__ __forceinline__ float nth_of_block(float v, int nth, float* sorted, float* result) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  v = sort_warp(v, lane);
  sorted[tid] = v;
  __syncthreads();
  int rank = lane;
#pragma unroll
  for (int d = 1; d < 8; ++d) {
    const int w = (warp + d) & 7;
    int at = 0;                                            // numbers of warp w that are before this one
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) {
      const float x = sorted[w * 32 + at + step - 1];
      at += x > v || (x == v && w < warp) ? step : 0;
    }
    const float x = sorted[w * 32 + at];
    rank += at + (x > v || (x == v && w < warp));
  }
  if (rank == nth - 1) *result = v;
  __syncthreads();
  return *result;
}

// A number that `nth` of the block's are at least as large as. For few of them the smallest of the warps' nth / 8-th largest, with some three times as many above it, which costs less than to rank those; for
// many the nth largest itself.
__device__ __forceinline__ float bound_of_block(float v, int nth, float* sorted, float* result) {
  if (nth > 32) return nth_of_block(v, nth, sorted, result);
  const float mine = nth_largest(v, (nth + 7) / 8, threadIdx.x & 31);
  __syncthreads();                                         // sorted is read no more
  if ((threadIdx.x & 31) == 0) sorted[threadIdx.x >> 5] = mine;
  __syncthreads();
  float x = sorted[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) x = fminf(x, sorted[w]);
  return x;
}

// Stores each of `found` entries of shared memory at its rank, where that is below n. Few entries are shared by all threads, which then count a part of the others each.
template <int THREADS, typename T, typename Before, typename Store>
__device__ __forceinline__ void store_ranked(const T* entries, int found, int n, int* ranks, Before before, Store store) {
  const int tid = threadIdx.x;
  if (found > THREADS / 2) {
    for (int i = tid; i < found; i += THREADS) {
      const T me = entries[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < found; ++j) rank += before(entries[j], me);
      if (rank < n) store(rank, me);
    }
    return;
  }
  if (tid < found) ranks[tid] = 0;
  __syncthreads();
  if (found > 0) {
    const int parts = THREADS / found, each = (found + parts - 1) / parts, i = tid % found, part = tid / found;
    if (part < parts) {
      const T me = entries[i];
      int rank = 0;
      for (int j = part * each; j < min(found, (part + 1) * each); ++j) rank += before(entries[j], me);
      if (rank) atomicAdd(&ranks[i], rank);
    }
  }
  __syncthreads();
  if (tid < found && ranks[tid] < n) store(ranks[tid], entries[tid]);
}

template <typename E, int EPT>
__global__ void __launch_bounds__(CHUNK_THREADS, 4) beam_chunk_kernel(const BeamParams p) {
  pdl_launch_dependents();
  constexpr int W = 16 / sizeof(E), VECS = EPT / W, WARPS = CHUNK_THREADS / 32, STEP = CHUNK_THREADS * EPT;
  __shared__ Entry s_found[ROOM];
  __shared__ float2 s_powers[32];
  __shared__ double s_sum[WARPS], s_whole[WARPS];
  __shared__ float s_bound[2][WARPS];
  __shared__ int s_rank[CHUNK_THREADS];
  __shared__ float s_sorted[CHUNK_THREADS], s_nth;
  __shared__ Entry s_note[ROOM];                           // the largest of a thread's logits of a step, and which they are
  __shared__ int s_count, s_notes, s_tally[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.y, n = p.count;
  if (tid < 32) s_powers[tid] = POWERS[tid];
  if (tid == 0) s_count = 0, s_notes = 0;
  if (tid < 2) s_tally[tid] = 0;
  pdl_wait();
  if (!alive(p.scores[row])) return;
  const E* from = reinterpret_cast<const E*>(p.logits) + row * p.stride;
  const int ahead = (int)((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(E));       // numbers of the row's first 16 bytes that are not its own
  const int steps = min(p.steps, (p.vocab + ahead + STEP - 1) / STEP - (int)blockIdx.x * p.steps);
  const long long at = (long long)row * p.pieces + blockIdx.x;
  Entry* out = p.best + at * n;
  if (steps <= 0) {                                        // behind the row's end, as rows start at different places
    if (tid == 0) p.piece[at] = Piece{0.0, -INFINITY};
    for (int i = tid; i < n; i += CHUNK_THREADS) out[i] = Entry{-INFINITY, -1};
    return;
  }
  const int first = blockIdx.x * p.steps * STEP - ahead;
  const auto token_of = [&](int step, int e) { return first + step * STEP + ((e / W) * CHUNK_THREADS + tid) * W + e % W; };
  const auto load = [&](int step, float* x) {
    const int start = first + step * STEP;
    if (start >= 0 && start + STEP <= p.vocab) {
#pragma unroll
      for (int i = 0; i < VECS; ++i) load16(from + start + (i * CHUNK_THREADS + tid) * W, x + i * W);
    } else {
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        const int t = start + (i * CHUNK_THREADS + tid) * W;
        if (t >= 0 && t + W <= p.vocab) {
          load16(from + t, x + i * W);
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) x[i * W + j] = t + j >= 0 && t + j < p.vocab ? to_f(from[t + j]) : -INFINITY;
        }
      }
    }
  };
  // once more, from the caches: what is rare takes no registers
  const auto logit_of = [&](int step, int e) {
    const int token = token_of(step, e);
    return token >= 0 && token < p.vocab ? to_f(from[token]) : -INFINITY;
  };
  float seen = -INFINITY, bound = -FLT_MAX;                // the thread's largest logit so far, NaN if there is one; -inf: not allowed
  unsigned long long large = pack2(2.f, 2.f), small = 0ull;
  float warp_top = -INFINITY, limit = -INFINITY, magic = MAGIC;
  double sum = 0.0;                                        // over 2^(power / 32)
  int power = 0;                                           // a multiple of 32
  const auto flush = [&]() {
    float a, b, c, d;
    unpack2(large, a, b);
    unpack2(small, c, d);
    sum += ((double)a - 2.0) + ((double)b - 2.0) + ((double)c + (double)d);
    large = pack2(2.f, 2.f), small = 0ull;
  };
  const auto process = [&](int step, const float* x) {
    float mine = x[0];
#pragma unroll
    for (int e = 1; e < EPT; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(mine) : "f"(x[e]));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(seen) : "f"(mine));
    if ((step & (step + 1)) == 0) {
      const float bound_w = nth_largest(seen, (n + WARPS - 1) / WARPS, lane);
      const int turn = __popc(step) & 1;                   // steps 0, 1, 3, 7..: read in one round what the next but one writes
      if (lane == 0) s_bound[turn][warp] = bound_w;
      __syncthreads();
      float b = s_bound[turn][0];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) b = fminf(b, s_bound[turn][w]);
      bound = fmaxf(bound, b);
    }
    if (mine >= bound) {
      const int i = atomicAdd(&s_notes, 1);
      if (i < ROOM) s_note[i] = Entry{mine, step * CHUNK_THREADS + tid};
    }
    if (__any_sync(0xffffffffu, mine > limit) || step % 64 == 63) {      // the warp's top has a new power of two, or small has grown
      const float top = fmaxf(warp_max(mine), warp_top);
      flush();
      if (fabsf(top) <= FAR) {
        const int next = (__float_as_int(fmaf(top, PER_STEP, MAGIC)) & ~31) - 0x4b400000;
        if (warp_top > -INFINITY) sum = ldexp(sum, max(min(power - next, 0) / 32, -2000));
        power = next, magic = MAGIC - (float)power;
        limit = (float)(power + 31) * (STEP_HIGH + STEP_LOW);       // up to it k stays below the next power of two
      }
      warp_top = fmaxf(warp_top, top);
    }
    if (fabsf(warp_top) <= FAR) {
      const float least = fmaxf(warp_top - LEAST, -FAR);
#pragma unroll
      for (int e = 0; e < EPT; e += 2) add_exponentials(x[e], x[e + 1], least, magic, s_powers, large, small);
    }
  };
  float x[EPT], y[EPT];
  load(0, x);
  for (int step = 0; step < steps; step += 2) {
    if (step + 1 < steps) load(step + 1, y);
    process(step, x);
    if (step + 1 == steps) break;
    if (step + 2 < steps) load(step + 2, x);
    process(step + 1, y);
  }
  flush();
  // The two parts of ln 2 / 32 are 5.1e-14 short of it. k of them are taken off a logit, k up to 1.4e6, and so the sum is one over e^(power * parts) to within the few thousand by which k differs from power.
  double whole = (double)power * ((double)STEP_HIGH + (double)STEP_LOW);
  if (!(fabsf(warp_top) <= FAR)) {                         // no logit is allowed, or the largest is out of the rounding's reach
    sum = 0.0, whole = (double)warp_top;
    if (warp_top > -INFINITY) {
#pragma unroll 1
      for (int step = 0; step < steps; ++step)
#pragma unroll 1
        for (int e = 0; e < EPT; ++e) sum += exp((double)logit_of(step, e) - whole);
    }
  }
  sum = warp_sum64(sum);
  if (lane == 0) s_sum[warp] = sum, s_whole[warp] = whole;
  const bool bad = __syncthreads_or(!(seen < INFINITY));
  if (bad) {                                               // the row offers nothing
    if (tid == 0) p.piece[at] = Piece{0.0, (double)INFINITY};
    return;
  }
  if (warp == WARPS - 1) {
    const double t = lane < WARPS ? s_whole[lane] : -INFINITY, v = lane < WARPS ? s_sum[lane] : 0.0;
    double all = t;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = fmax(all, __shfl_xor_sync(0xffffffffu, all, o));
    const double total = warp_sum64(t > -INFINITY ? v * exp(t - all) : 0.0);
    if (lane == 0) p.piece[at] = Piece{total, all};
  }
  int found = s_notes;
  if (found <= ROOM) {
    bound = fmaxf(bound, bound_of_block(seen, n, s_sorted, &s_nth));
    const int of = lane / EPT, e = lane % EPT;             // 32 / EPT notes to a warp, a logit to a lane
    for (int i = warp * (32 / EPT) + of; i < found; i += WARPS * (32 / EPT)) {
      const Entry note = s_note[i];
      if (note.x < bound) continue;
      const int token = first + note.token / CHUNK_THREADS * STEP + (e / W * CHUNK_THREADS + note.token % CHUNK_THREADS) * W + e % W;
      const float y = token >= 0 && token < p.vocab ? to_f(from[token]) : -INFINITY;
      if (y >= bound) {
        const int to = atomicAdd(&s_count, 1);
        if (to < ROOM) s_found[to] = Entry{y, token};
      }
    }
    __syncthreads();
    found = s_count;
  }
  if (found > ROOM) {
    // Many logits as large as the bound (ties): the count-th largest by halving the range of the logits' bit patterns, and of equal ones the first tokens.
    int turn = 0;
    const auto tally = [&](auto test) {
      int c = 0;
#pragma unroll 1
      for (int step = 0; step < steps; ++step)
#pragma unroll 4
        for (int e = 0; e < EPT; ++e) {
          const float y = logit_of(step, e);
          c += y > -INFINITY && test(y, token_of(step, e));
        }
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
      if (tally([&](float y, int) { return order_of(y) >= next; }) >= n) key = next;
    }
    const int need = n - tally([&](float y, int) { return order_of(y) > key; });
    int last = 0;                                          // the last of them is at this place
    for (int b = 30; b >= 0; --b) {
      const int next = last | 1 << b;
      if (tally([&](float y, int token) { return order_of(y) == key && token < next; }) < need) last = next;
    }
    if (tid == 0) s_count = 0;
    __syncthreads();
#pragma unroll 1
    for (int step = 0; step < steps; ++step)
#pragma unroll 1
      for (int e = 0; e < EPT; ++e) {
        const float y = logit_of(step, e);
        if (y > -INFINITY && (order_of(y) > key || (order_of(y) == key && token_of(step, e) <= last))) s_found[atomicAdd(&s_count, 1)] = Entry{y, token_of(step, e)};
      }
    __syncthreads();
    found = s_count;
  }
  store_ranked<CHUNK_THREADS>(s_found, found, n, s_rank, [](const Entry& a, const Entry& b) { return (int)(a.x > b.x) | ((int)(a.x == b.x) & (int)(a.token < b.token)); },
                              [&](int rank, const Entry& e) { out[rank] = e; });
  for (int i = found + tid; i < n; i += CHUNK_THREADS) out[i] = Entry{-INFINITY, -1};
}

// ---- one block a prompt -----------------------------------------------------------------------------------------------------------------------------
constexpr int JOIN_THREADS = 256, JOIN_WARPS = JOIN_THREADS / 32, HELD = 2048, MAX_LISTS = 1536;

struct Choice {
  double s;
  long long at;              // beam, and token in the low 32 bits
};
__device__ __forceinline__ bool better(double s, long long at, const Choice& c) { return (int)(s > c.s) | ((int)(s == c.s) & (int)(at < c.at)); }

__global__ void __launch_bounds__(JOIN_THREADS) beam_join_kernel(const BeamParams p) {
  pdl_launch_dependents();
  __shared__ Entry s_held[HELD];
  __shared__ double s_log[MAX_BEAMS];                      // of a beam's sum of exponentials; NaN: it offers nothing
  __shared__ Choice s_found[ROOM];
  __shared__ Choice s_warp[JOIN_WARPS];
  __shared__ int s_rank[JOIN_THREADS], s_live[MAX_LISTS], s_lives;
  __shared__ float s_sorted[JOIN_THREADS], s_nth;
  __shared__ int s_count, s_tally[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x, n = p.count, K = p.beams;
  pdl_wait();
  const float* score = p.scores + (long long)b * K;
  const int per_beam = p.pieces * n, total = K * per_beam;
  const Entry* best = p.best + (long long)b * total;
  const bool few = total <= HELD;
  if (few) {                                               // on their way beside the sums
    Entry e[HELD / JOIN_THREADS];
#pragma unroll
    for (int u = 0; u < HELD / JOIN_THREADS; ++u)
      if (u * JOIN_THREADS + tid < total) e[u] = best[u * JOIN_THREADS + tid];
#pragma unroll
    for (int u = 0; u < HELD / JOIN_THREADS; ++u) s_held[u * JOIN_THREADS + tid] = e[u];
  }
  if (tid == 0) s_count = 0, s_lives = 0;
  // as many lanes to a beam as it has pieces, 32 at most
  int group = 1;
  while (group < p.pieces && group < 32) group *= 2;
  const int in = lane & (group - 1);
  for (int k0 = 0; k0 < K; k0 += JOIN_THREADS / group) {
    const int k = k0 + tid / group;
    const bool mine = k < K && alive(score[k]);
    const Piece* piece = p.piece + ((long long)b * K + k) * p.pieces;
    const auto load = [&](int i) { return mine && i < p.pieces ? piece[i] : Piece{0.0, -INFINITY}; };
    const Piece own = load(in), next = load(in + group);   // most rows have no more
    double top = fmax(own.top, next.top), sum = 0.0;
    for (int i = in + 2 * group; i < p.pieces; i += group) top = fmax(top, load(i).top);
    for (int o = group >> 1; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (isfinite(top)) {
      const auto part = [&](const Piece& x) { return x.top > -INFINITY ? x.sum * exp(x.top - top) : 0.0; };
      sum = part(own) + part(next);
      for (int i = in + 2 * group; i < p.pieces; i += group) sum += part(load(i));
    }
    for (int o = group >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (k < K && in == 0) s_log[k] = isfinite(top) ? top + log(sum) : (double)NAN;
  }
  __syncthreads();
  // the i-th candidate; s = -inf: none
  const float share = 1.f / (float)per_beam;
  const auto choice = [&](int i, const Entry& e) {
    int k = (int)((float)i * share);                       // i / per_beam, or one beside it
    k += (k + 1) * per_beam <= i ? 1 : k * per_beam > i ? -1 : 0;
    const double log_sum = s_log[k];
    Choice c{-INFINITY, LLONG_MAX};
    if (log_sum != log_sum || e.token < 0) return c;
    c.s = (double)score[k] + ((double)e.x - log_sum);
    c.at = (long long)k << 32 | e.token;
    return c;
  };
  const auto candidate = [&](int i) { return choice(i, best[i]); };
  // (The block runs once over all of this: code that is not there need not be fetched, so that loops are left as they are.)
  // A bound as in the pieces: over all entries where there is room for their scores. Else from the lists, which are in order: where m of them have an entry d of some score, m (d + 1) entries are as
  // good, and the best of the bounds of d = 0, 1, 3, 7.. is taken, as one beam may have most of the best or all of them a few.
  const int lists = K * p.pieces;
  // (Neighbours go to different warps, so that each has its share of every beam's.)
  const int place = lane * JOIN_WARPS + warp;
  float bound = -INFINITY;
  if (few) {
    double mine = -INFINITY;
#pragma unroll 1
    for (int i = place; i < total; i += JOIN_THREADS) mine = fmax(mine, choice(i, s_held[i]).s);
    bound = bound_of_block(__double2float_rd(mine), n, s_sorted, &s_nth);       // (rounded down: a bound is no exact number)
  } else {
#pragma unroll 1
    for (int d = 0; d < n; d = 2 * d + 1) {
      float mine = -INFINITY;
#pragma unroll 2
      for (int i = place; i < lists; i += JOIN_THREADS) mine = fmaxf(mine, __double2float_rd(candidate(i * n + d).s));
      bound = fmaxf(bound, bound_of_block(mine, (n + d) / (d + 1), s_sorted, &s_nth));
    }
  }
  const auto take = [&](const Choice& c) {
    const bool good = c.s >= (double)bound && c.s > -INFINITY;
    if (good) {
      const int at = atomicAdd(&s_count, 1);
      if (at < ROOM) s_found[at] = c;
    }
    return good;
  };
  const auto collect = [&]() {
    if (few) {
#pragma unroll 1
      for (int i = place; i < total; i += JOIN_THREADS)
        take(choice(i, s_held[i]));
    } else {
      // lists whose first entry is good enough, each a warp's, four of them on their way together
      for (int i = place; i < lists; i += JOIN_THREADS) {
        const Choice c = candidate(i * n);
        if (c.s >= (double)bound && c.s > -INFINITY) s_live[atomicAdd(&s_lives, 1)] = i;
      }
      __syncthreads();
      const int lives = s_lives;
      for (int i0 = warp * 4; i0 < lives; i0 += JOIN_WARPS * 4) {
        Choice c[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) c[u] = i0 + u < lives && lane < n ? candidate(s_live[i0 + u] * n + lane) : Choice{-INFINITY, LLONG_MAX};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          bool more = __all_sync(0xffffffffu, take(c[u]));
          for (int e = 32; more && e < n; e += 32) more = __all_sync(0xffffffffu, e + lane < n && take(candidate(s_live[i0 + u] * n + e + lane)));
        }
      }
    }
    __syncthreads();
    return s_count;
  };
  int found = collect();
  if (found > ROOM) {
    // A few beams have most of the best: the bound is put where between `count` and ROOM are left, by halving the range of its bit patterns and counting in the ordered lists.
    unsigned low = order_of(bound), high = 0xff800001u;    // too many, and none
    int turn = 0;
    while (high - low > 1 && !(found >= n && found <= ROOM)) {
      const unsigned mid = low + (high - low) / 2;
      const double at = (double)of_order(mid);
      if (tid < 2) s_tally[tid] = tid == turn ? 0 : s_tally[tid];
      __syncthreads();
      int mine_too = 0;
      for (int i = tid; i < lists; i += JOIN_THREADS) {
        int a = 0, z = n;                                  // the first entry below it is in a..z
        while (a < z) {
          const int m = (a + z) >> 1;
          if (candidate(i * n + m).s >= at) a = m + 1;
          else z = m;
        }
        mine_too += a;
      }
      mine_too = __reduce_add_sync(0xffffffffu, mine_too);
      if (lane == 0) atomicAdd(&s_tally[turn], mine_too);
      __syncthreads();
      found = s_tally[turn];
      turn ^= 1;
      if (found < n) high = mid;
      else low = mid;
    }
    if (found >= n && found <= ROOM) {
      bound = of_order(low);
      if (tid == 0) s_count = 0, s_lives = 0;
      __syncthreads();
      found = collect();
    } else {
      found = ROOM + 1;
    }
  }
  const auto store = [&](int at, const Choice& c) {
    const long long to = (long long)b * n + at;
    const bool none = !(c.s > -INFINITY);
    p.out_scores[to] = (float)c.s;
    p.out_beams[to] = none ? -1 : (int)(c.at >> 32);
    p.out_tokens[to] = none ? -1 : c.at & 0x7fffffff;
  };
  if (found <= ROOM) {
    store_ranked<JOIN_THREADS>(s_found, found, n, s_rank, [](const Choice& a, const Choice& b) { return better(a.s, a.at, b); }, store);
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
    for (int w = 0; w < JOIN_WARPS; ++w)
      if (better(s_warp[w].s, s_warp[w].at, c)) c = s_warp[w];
    if (tid == 0) store(r, c);
    last = c;
    __syncthreads();
  }
}

// A row's pieces: steps of 4096 logits, of 2048 where those are too few for the SMs, in as many pieces as the SMs hold blocks.
struct Pieces {
  int per_thread, steps, n;
};
Pieces pieces_of(long long rows, int vocab) {
  Pieces p;
  const auto steps = [&](int e) { return (vocab + 7ll + CHUNK_THREADS * e - 1) / (CHUNK_THREADS * e); };      // a row may start anywhere within 16 bytes
  p.per_thread = rows * steps(16) < 148 ? 8 : 16;
  const long long all = steps(p.per_thread), want = rows < 4 * 148 ? 4 * 148 / rows : 1;
  p.steps = (int)((all + want - 1) / want);
  p.n = (int)((all + p.steps - 1) / p.steps);
  return p;
}

template <typename E>
int launch_chunks(const BeamParams& p, cudaStream_t s) {
  const long long rows = (long long)p.batch * p.beams;
  const dim3 grid(p.pieces, (unsigned)rows);
  return pieces_of(rows, p.vocab).per_thread == 16 ? launch_kernel(beam_chunk_kernel<E, 16>, grid, dim3(CHUNK_THREADS), 0, s, p)
                                                   : launch_kernel(beam_chunk_kernel<E, 8>, grid, dim3(CHUNK_THREADS), 0, s, p);
}

}  // namespace
}  // namespace swb

extern "C" {

// Bytes of workspace.
long long swb_beam_workspace_bytes(int batch, int beams, int vocab, int count) {
  using namespace swb;
  const long long rows = (long long)batch * beams;
  return rows < 1 || vocab < 1 ? 0 : rows * pieces_of(rows, vocab).n * ((long long)sizeof(Piece) + (long long)sizeof(Entry) * count);
}

// logits [batch * beams, vocab], rows `stride` numbers apart; scores [batch, beams]. workspace: 16-byte aligned.
int swb_beam_select(const void* logits, long long stride, int fp32, const float* scores, int batch, int beams, int vocab, int count, float* out_scores, int* out_beams, void* out_tokens,
                    void* workspace, long long workspace_bytes, void* stream) {
  using namespace swb;
  if (batch <= 0) return 0;
  BeamParams p = {};
  if (!logits || !scores || !out_scores || !out_beams || !out_tokens || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || beams < 1 || beams > MAX_BEAMS || vocab < 1 ||
      vocab > INT_MAX - 65536 || count < 1 || count > MAX_COUNT || (long long)batch * beams > 65535)
    return -3;
  const long long rows = (long long)batch * beams;
  const Pieces pieces = pieces_of(rows, vocab);
  p.pieces = pieces.n, p.steps = pieces.steps;
  if (swb_beam_workspace_bytes(batch, beams, vocab, count) > workspace_bytes || beams * p.pieces > MAX_LISTS) return -3;
  p.logits = logits, p.stride = stride, p.scores = scores, p.batch = batch, p.beams = beams, p.vocab = vocab, p.count = count;
  p.piece = reinterpret_cast<Piece*>(workspace), p.best = reinterpret_cast<Entry*>(p.piece + rows * p.pieces);
  p.out_scores = out_scores, p.out_beams = out_beams, p.out_tokens = reinterpret_cast<long long*>(out_tokens);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int rc = fp32 ? launch_chunks<float>(p, s) : launch_chunks<bf16>(p, s);
  if (rc) return rc;
  return launch_kernel(beam_join_kernel, dim3(batch), dim3(JOIN_THREADS), 0, s, p);
}

}  // extern "C"
