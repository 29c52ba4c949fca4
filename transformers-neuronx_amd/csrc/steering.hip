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

#define SCORE_THREADS 256

__global__ void __launch_bounds__(SCORE_THREADS)
log_probs_kernel(const float* __restrict__ logits, const int* __restrict__ tokens, float* __restrict__ out, int* __restrict__ top_tokens,
                 float* __restrict__ top_out, int top, int vocab) {
  __shared__ float scratch[SCORE_THREADS / 64];
  __shared__ unsigned long long best[SCORE_THREADS / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* row = logits + (size_t)blockIdx.x * vocab;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < vocab; i += SCORE_THREADS) m = fmaxf(m, row[i]);
  m = wave_max(m);
  if (lane == 0) scratch[wave] = m;
  __syncthreads();
  for (int w = 0; w < SCORE_THREADS / 64; ++w) m = fmaxf(m, scratch[w]);
  float s = 0.f;
  for (int i = threadIdx.x; i < vocab; i += SCORE_THREADS) {
    const float x = row[i];
    s += x == m ? 1.f : x > -INFINITY ? expf(x - m) : 0.f;
  }
  const float log_l = logf(block_sum<SCORE_THREADS / 64>(s, scratch));
  if (threadIdx.x == 0) {
    const int t = tokens[blockIdx.x];
    out[blockIdx.x] = t >= 0 && t < vocab ? log_prob_of(row[t], m, log_l) : -INFINITY;
  }
  unsigned long long below = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long b = 0;
    for (int i = threadIdx.x; i < vocab; i += SCORE_THREADS) {
      const unsigned long long key = order_key(row[i], i);
      if (key < below && key > b) b = key;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor(b, o, 64);
      b = other > b ? other : b;
    }
    __syncthreads();
    if (lane == 0) best[wave] = b;
    __syncthreads();
    for (int w = 0; w < SCORE_THREADS / 64; ++w) b = best[w] > b ? best[w] : b;
    below = b;
    if (threadIdx.x == 0) {
      const int t = (int)(~(unsigned)b);
      top_tokens[(size_t)blockIdx.x * top + k] = t;
      top_out[(size_t)blockIdx.x * top + k] = log_prob_of(row[t], m, log_l);
    }
  }
}

extern "C" int tnx_log_probs(const float* logits, const int* tokens, float* out, int* top_tokens, float* top_out, int top, int rows,
                             int vocab, hipStream_t stream) {
  TNX_REQUIRE(rows >= 0 && vocab > 0 && top >= 0 && top <= 32 && top <= vocab, "log_probs: bad sizes rows=%d vocab=%d top=%d", rows, vocab,
              top);
  if (rows == 0) return 0;
  log_probs_kernel<<<rows, SCORE_THREADS, 0, stream>>>(logits, tokens, out, top_tokens, top_out, top, vocab);
  TNX_CHECK_LAUNCH("log_probs");
  return 0;
}
