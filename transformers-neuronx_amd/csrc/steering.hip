// What is done to a decode step's logits before a token is chosen from them, and what is said of it afterwards:
// penalties for repeated tokens, biases and masks of allowed tokens (`adjust_logits`), and log-probabilities with the
// best alternatives (`log_probs`).
#include "common.h"

TNX_DEFINE_ERROR_API

// A row's rules, as the host writes them (LogitRules, 8 words a row).
struct RowRules {
  int slot;                 // whose history; below zero: none is kept
  float repetition, presence, frequency;
  int bias_begin, bias_end; // its biases among the batch's
  int mask_row;             // its mask among the masks; below zero: every token is allowed
  int unused;
};

// ---------------------------------------------------------------- histories

// A history is the list of a sequence's distinct tokens, in the order of their first appearance, as pairs {token, twice the times
// it was chosen + 1 if the prompt has it}: it is as long as it must be, read in one go, and a step appends at most one entry.
// heads[i] = {slot, first pair, pairs}: the slot's history becomes these pairs, and the token it waits for none.
__global__ void __launch_bounds__(256)
start_history_kernel(const int* __restrict__ heads, const int2* __restrict__ pairs, int2* __restrict__ entries, int* __restrict__ used,
                     int* __restrict__ last, int capacity) {
  const int* h = heads + 3 * (size_t)blockIdx.x;
  int2* mine = entries + (size_t)h[0] * capacity;
  for (int i = threadIdx.x; i < h[2]; i += 256) mine[i] = pairs[h[1] + i];
  if (threadIdx.x == 0) {
    used[h[0]] = h[2];
    if (last) last[h[0]] = -1;
  }
}

// The host has checked every slot and every length against the history's sizes.
extern "C" int tnx_start_history(const int* heads, int num, const int* pairs, int* entries, int* used, int* last, int slots, int capacity,
                                 hipStream_t stream) {
  TNX_REQUIRE(num >= 0 && slots > 0 && capacity > 0, "start_history: bad sizes num=%d slots=%d capacity=%d", num, slots, capacity);
  if (num == 0) return 0;
  start_history_kernel<<<num, 256, 0, stream>>>(heads, (const int2*)pairs, (int2*)entries, used, last, capacity);
  TNX_CHECK_LAUNCH("start_history");
  return 0;
}

// ---------------------------------------------------------------- adjusting logits

__device__ __forceinline__ bool is_allowed(const unsigned* mask, int token) {
  return mask == nullptr || ((mask[token >> 5] >> (token & 31)) & 1u);
}

// x / rho where x > 0, x * rho elsewhere; then frequency * times and, if it was chosen at all, presence less
__device__ __forceinline__ float penalised(float x, const RowRules& r, int info) {
  const int times = info >> 1;
  x = x > 0.f ? x / r.repetition : x * r.repetition;
  return x - (r.frequency * (float)times + (times > 0 ? r.presence : 0.f));
}

// One block a row. Every logit is written by one thread at a time: history entries name distinct tokens, so do a row's
// biases, a barrier lies between the two, and tokens that the mask bars are left to the last loop, which writes nothing else.
__global__ void __launch_bounds__(256)
adjust_logits_kernel(float* __restrict__ logits, const RowRules* __restrict__ rules, const int* __restrict__ bias_tokens,
                     const float* __restrict__ bias_values, int2* __restrict__ entries, int* __restrict__ used, int capacity,
                     const int* __restrict__ last, const unsigned* __restrict__ masks, int words, int vocab) {
  const RowRules r = rules[blockIdx.x];
  float* row = logits + (size_t)blockIdx.x * vocab;
  const unsigned* mask = r.mask_row >= 0 ? masks + (size_t)r.mask_row * words : nullptr;
  __shared__ int found;
  if (r.slot >= 0) {
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    int2* mine = entries + (size_t)r.slot * capacity;
    const int n = max(0, min(used[r.slot], capacity)), token = last[r.slot];
    for (int i = threadIdx.x; i < n; i += 256) {
      int2 e = mine[i];
      if (e.x == token) {
        e.y += 2;
        mine[i].y = e.y;
        found = 1;
      }
      if (e.x >= 0 && e.x < vocab && is_allowed(mask, e.x)) row[e.x] = penalised(row[e.x], r, e.y);
    }
    __syncthreads();
    if (threadIdx.x == 0 && !found && token >= 0 && token < vocab && n < capacity) {
      mine[n] = make_int2(token, 2);
      used[r.slot] = n + 1;
      if (is_allowed(mask, token)) row[token] = penalised(row[token], r, 2);
    }
    __syncthreads();
  }
  for (int i = r.bias_begin + threadIdx.x; i < r.bias_end; i += 256) {
    const int t = bias_tokens[i];
    const float b = bias_values[i];
    if (is_allowed(mask, t)) row[t] = b == -INFINITY ? b : row[t] + b;
  }
  if (mask != nullptr)
    for (int i = threadIdx.x; i < vocab; i += 256)
      if (!is_allowed(mask, i)) row[i] = -INFINITY;
}

// The host has checked the rows' slots, masks and bias tokens against the sizes given here.
extern "C" int tnx_adjust_logits(float* logits, const int* rules, const int* bias_tokens, const float* bias_values, int* entries, int* used,
                                 int capacity, const int* last, const int* masks, int rows, int vocab, hipStream_t stream) {
  TNX_REQUIRE(rows >= 0 && vocab > 0 && capacity >= 0, "adjust_logits: bad sizes rows=%d vocab=%d capacity=%d", rows, vocab, capacity);
  if (rows == 0) return 0;
  adjust_logits_kernel<<<rows, 256, 0, stream>>>(logits, (const RowRules*)rules, bias_tokens, bias_values, (int2*)entries, used, capacity,
                                                 last, (const unsigned*)masks, (vocab + 31) / 32, vocab);
  TNX_CHECK_LAUNCH("adjust_logits");
  return 0;
}

// ---------------------------------------------------------------- log-probabilities

// With m the largest logit and l the sum of exp(x - m): the log-probability of a token is x - m - log l. A NaN counts as -inf, as
// it does where a token is chosen. Of a row of nothing but -inf every log-probability is -inf; where m is +inf, the tokens that have
// it share the whole, and l is their number.
__device__ __forceinline__ float log_prob_of(float x, float m, float log_l) {
  if (!(x > -INFINITY)) return -INFINITY;          // and a NaN
  return (x == m ? 0.f : x - m) - log_l;
}

__device__ __forceinline__ unsigned long long order_key(float x, int idx) {
  if (x != x) x = -INFINITY;
  if (x == 0.f) x = 0.f;       // -0 and +0 are one value: the lower token id decides between them
  unsigned u = __float_as_uint(x);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (unsigned)(~(unsigned)idx);
}

// exp(d) for d <= 0 by the hardware's power of two; log2(e) in two parts, so that only the roundings of d and of the power's argument
// are left: 2^-24 of |d| each, and what is far below the largest adds little.
__device__ __forceinline__ float exp_of(float d) {
  const float hi = 1.44269502162933349609375f, lo = 1.92596299112661746887e-8f;
  return __builtin_amdgcn_exp2f(fmaf(d, hi, d * lo));
}

// A row read four logits at a time from the boundary of 16 bytes at or before it: quad q holds elements 4 q - lead to 4 q - lead + 3;
// what lies outside the row reads as -inf. A NaN reads as -inf as well.
struct Quads {
  const float* row;
  int vocab, lead, count;
  __device__ __forceinline__ Quads(const float* r, int v)
      : row(r), vocab(v), lead((int)(((uintptr_t)r >> 2) & 3)), count((v + (int)(((uintptr_t)r >> 2) & 3) + 3) / 4) {}
  __device__ __forceinline__ int first(int q) const { return 4 * q - lead; }
  __device__ __forceinline__ f32x4 operator()(int q) const {
    const int i = 4 * q - lead;
    f32x4 x;
    if (q < count && i >= 0 && i + 3 < vocab) {
      x = *(const f32x4*)(row + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = q < count && i + e >= 0 && i + e < vocab ? row[i + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = fmaxf(x[e], -INFINITY);
    return x;
  }
};

#define SCORE_GROUPS 256       // groups of threads whose largest logits are ranked against one another
#define SCORE_GATHER 1024      // the most logits that are gathered for the alternatives
#define SCORE_MOST_TOP 32
#define SCORE_WIDE_ROWS 512

// One block of THREADS a row, one pass over it with a running maximum and sum.
//
// The alternatives come from the same pass: a thread notes its largest logit, and as many groups of threads as alternatives are
// wanted, those with the largest logits, hold all of them (of the others each group's best is already beaten by so many). Only
// the logits of these groups are looked at again, and those of them that are no smaller than the last group's best, hardly more than
// the alternatives themselves, are ranked in LDS. Should they be more than fit (the best of a long row all in a few threads' places),
// the alternatives are found one by one, each with a pass of its own.
template <int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS)
log_probs_kernel(const float* __restrict__ logits, const int* __restrict__ tokens, float* __restrict__ out, int* __restrict__ top_tokens,
                 float* __restrict__ top_out, int top, int vocab) {
  constexpr int WAVES = THREADS / 64, PER_GROUP = THREADS / SCORE_GROUPS;
  __shared__ float scratch[WAVES], sums[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Quads quads(logits + (size_t)blockIdx.x * vocab, vocab);
  const float* row = quads.row;

  float m = -INFINITY, s = 0.f;
  int at = tid;                       // the quads among which the thread's largest logit came first
  for (int q0 = tid; q0 < quads.count; q0 += 4 * THREADS) {
    f32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = quads(q0 + k * THREADS);
    float here = v[0][0];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) here = fmaxf(here, v[k][e]);
    if (here > m) {
      s *= m > -INFINITY ? exp_of(m - here) : 0.f;
      m = here;
      at = q0;
    }
    const float base = fmaxf(m, -3.402823466e38f);       // -inf less -inf would be no number
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) s += exp_of(v[k][e] - base);
  }
  const float mine = m;
  m = wave_max(m);
  if (lane == 0) scratch[wave] = m;
  __syncthreads();
  m = scratch[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) m = fmaxf(m, scratch[w]);
  if (m < INFINITY) {
    s = mine > -INFINITY ? s * exp_of(mine - m) : 0.f;
  } else {                            // those at +inf are counted
    s = 0.f;
    for (int q = tid; q < quads.count; q += THREADS) {
      const f32x4 x = quads(q);
#pragma unroll
      for (int e = 0; e < 4; ++e) s += x[e] == INFINITY ? 1.f : 0.f;
    }
  }
  const float log_l = logf(block_sum<WAVES>(s, sums));
  if (tid == 0) {
    const int t = tokens[blockIdx.x];
    out[blockIdx.x] = t >= 0 && t < vocab ? log_prob_of(row[t], m, log_l) : -INFINITY;
  }
  if constexpr (TOP) {
    __shared__ unsigned long long best[SCORE_GROUPS], gathered[SCORE_GATHER], one[WAVES];
    __shared__ int winners[SCORE_MOST_TOP], num_winners, num_gathered;
    __shared__ unsigned long long least;
    // the thread's best as a key (its logit, then the lower token id), and its group's
    unsigned long long key = 0;
    if (tid < quads.count) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4 x = quads(at + k * THREADS);
        const int i = quads.first(at + k * THREADS);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + e >= 0 && i + e < vocab) {
            const unsigned long long other = order_key(x[e], i + e);
            key = other > key ? other : key;
          }
      }
    }
#pragma unroll
    for (int o = 1; o < PER_GROUP; o <<= 1) {
      const unsigned long long other = __shfl_xor(key, o, 64);
      key = other > key ? other : key;
    }
    if (tid % PER_GROUP == 0) best[tid / PER_GROUP] = key;
    if (tid == 0) {
      num_winners = num_gathered = 0;
      least = 0;
    }
    __syncthreads();
    if (tid < SCORE_GROUPS && best[tid] != 0) {          // (0: a group without logits)
      const unsigned long long b = best[tid];
      int rank = 0;
      for (int j = 0; j < SCORE_GROUPS; ++j) rank += best[j] > b ? 1 : 0;
      if (rank < top) {
        winners[rank] = tid;
        atomicAdd(&num_winners, 1);
      }
      if (rank == top - 1) least = b;                    // (fewer groups than alternatives: everything is gathered)
    }
    __syncthreads();
    // group g's quads are those of its threads: k * THREADS + PER_GROUP * g + j
    const int rounds = (quads.count + THREADS - 1) / THREADS * PER_GROUP;
    const unsigned long long floor_key = least;
    for (int w = wave; w < num_winners; w += WAVES)
      for (int n = lane; n < rounds; n += 64) {
        const int q = n / PER_GROUP * THREADS + PER_GROUP * winners[w] + n % PER_GROUP;
        const f32x4 x = quads(q);
        const int i = quads.first(q);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (q < quads.count && i + e >= 0 && i + e < vocab) {
            const unsigned long long k = order_key(x[e], i + e);
            if (k >= floor_key) {
              const int to = atomicAdd(&num_gathered, 1);
              if (to < SCORE_GATHER) gathered[to] = k;
            }
          }
      }
    __syncthreads();
    const int n = num_gathered;
    int* ids = top_tokens + (size_t)blockIdx.x * top;
    float* values = top_out + (size_t)blockIdx.x * top;
    if (n <= SCORE_GATHER) {
      for (int c = tid; c < n; c += THREADS) {
        const unsigned long long k = gathered[c];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += gathered[j] > k ? 1 : 0;
        if (rank < top) {
          const int t = (int)(~(unsigned)k);
          ids[rank] = t;
          values[rank] = log_prob_of(row[t], m, log_l);
        }
      }
    } else {
      unsigned long long below = ~0ull;
      for (int r = 0; r < top; ++r) {
        unsigned long long b = 0;
        for (int i = tid; i < vocab; i += THREADS) {
          const unsigned long long k = order_key(row[i], i);
          if (k < below && k > b) b = k;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
          const unsigned long long other = __shfl_xor(b, o, 64);
          b = other > b ? other : b;
        }
        __syncthreads();
        if (lane == 0) one[wave] = b;
        __syncthreads();
        for (int w = 0; w < WAVES; ++w) b = one[w] > b ? one[w] : b;
        below = b;
        if (tid == 0) {
          const int t = (int)(~(unsigned)b);
          ids[r] = t;
          values[r] = log_prob_of(row[t], m, log_l);
        }
      }
    }
  }
}

template <int THREADS>
static void launch_log_probs(const float* logits, const int* tokens, float* out, int* top_tokens, float* top_out, int top, int rows, int vocab,
                             hipStream_t stream) {
  if (top) log_probs_kernel<THREADS, true><<<rows, THREADS, 0, stream>>>(logits, tokens, out, top_tokens, top_out, top, vocab);
  else log_probs_kernel<THREADS, false><<<rows, THREADS, 0, stream>>>(logits, tokens, out, top_tokens, top_out, top, vocab);
}

extern "C" int tnx_log_probs(const float* logits, const int* tokens, float* out, int* top_tokens, float* top_out, int top, int rows,
                             int vocab, hipStream_t stream) {
  TNX_REQUIRE(rows >= 0 && vocab > 0 && vocab < (1 << 30) && top >= 0 && top <= SCORE_MOST_TOP && top <= vocab,
              "log_probs: bad sizes rows=%d vocab=%d top=%d", rows, vocab, top);
  if (rows == 0) return 0;
  if (rows <= SCORE_WIDE_ROWS) launch_log_probs<1024>(logits, tokens, out, top_tokens, top_out, top, rows, vocab, stream);
  else launch_log_probs<256>(logits, tokens, out, top_tokens, top_out, top, rows, vocab, stream);
  TNX_CHECK_LAUNCH("log_probs");
  return 0;
}
