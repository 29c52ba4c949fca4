// What is done to a decode step's logits before a token is chosen from them, and what is said of it afterwards:
// penalties for repeated tokens, biases and masks of allowed tokens (`adjust_logits`), and log-probabilities with the
// best alternatives (`log_probs`).
#include "common.h"
#include "token_order.h"

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

#define ADJUST_THREADS 1024
#define ADJUST_AHEAD 4         // history entries of a thread that are on their way together
#define ADJUST_BARRED 16       // logits that a thread may have to bar

// Block 0 of a row does what names single tokens, its history and its biases; the others write -inf where the mask bars a token,
// ADJUST_THREADS * ADJUST_BARRED logits each. A logit is written by one thread at a time: history entries name distinct tokens,
// so do a row's biases, a barrier lies between the two, and barred tokens are left to the other blocks, which write nothing else.
//
// Of a row's logits only those named are read, and only those barred written: what bounds a batch is the way from the rules to the
// history's entries, to the logits and back, and to the biases' logits and back, trips to memory one behind the other, not their bytes.
// One row with 120 entries 2.2 us, 64 rows of 50,272 with 1,500 entries and 300 biases 6.7, with half of the tokens barred as well 9.2;
// half of the tokens barred alone 6.6 (one logit a lane, so that a wave's stores lie side by side; four a lane 10.4).
__global__ void __launch_bounds__(ADJUST_THREADS)
adjust_logits_kernel(float* __restrict__ logits, const RowRules* __restrict__ rules, const int* __restrict__ bias_tokens,
                     const float* __restrict__ bias_values, int2* __restrict__ entries, int* __restrict__ used, int capacity,
                     const int* __restrict__ last, const unsigned* __restrict__ masks, int words, int vocab) {
  const RowRules r = rules[blockIdx.y];
  float* row = logits + (size_t)blockIdx.y * vocab;
  const unsigned* mask = r.mask_row >= 0 ? masks + (size_t)r.mask_row * words : nullptr;
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    if (mask == nullptr) return;
    const int i0 = (int)(blockIdx.x - 1) * (ADJUST_THREADS * ADJUST_BARRED) + tid;
    unsigned word[ADJUST_BARRED];
#pragma unroll
    for (int k = 0; k < ADJUST_BARRED; ++k) word[k] = mask[min(i0 + k * ADJUST_THREADS, vocab - 1) >> 5];
#pragma unroll
    for (int k = 0; k < ADJUST_BARRED; ++k) {
      const int i = i0 + k * ADJUST_THREADS;
      if (i < vocab && !((word[k] >> (i & 31)) & 1u)) row[i] = -INFINITY;
    }
    return;
  }
  // the first of the biases are asked for now, to be there when the history is done
  int bias_at = r.bias_begin + tid, bias_token = 0;
  float bias = 0.f;
  if (bias_at < r.bias_end) {
    bias_token = bias_tokens[bias_at];
    bias = bias_values[bias_at];
  }
  if (r.slot >= 0) {
    __shared__ int found;
    if (tid == 0) found = 0;
    int2* mine = entries + (size_t)r.slot * capacity;
    const int n = max(0, min(used[r.slot], capacity)), token = last[r.slot];
    __syncthreads();
    for (int i0 = tid; i0 < n; i0 += ADJUST_THREADS * ADJUST_AHEAD) {
      int2 e[ADJUST_AHEAD];
      float x[ADJUST_AHEAD];
      bool on[ADJUST_AHEAD];
#pragma unroll
      for (int k = 0; k < ADJUST_AHEAD; ++k) {
        const int i = i0 + k * ADJUST_THREADS;
        e[k] = i < n ? mine[i] : make_int2(-1, 0);
      }
#pragma unroll
      for (int k = 0; k < ADJUST_AHEAD; ++k) {
        const bool there = e[k].x >= 0 && e[k].x < vocab;
        x[k] = there ? row[e[k].x] : 0.f;
        on[k] = there && is_allowed(mask, e[k].x);
      }
#pragma unroll
      for (int k = 0; k < ADJUST_AHEAD; ++k) {
        const int i = i0 + k * ADJUST_THREADS;
        if (i < n && e[k].x == token) {
          e[k].y += 2;
          mine[i].y = e[k].y;
          found = 1;
        }
        if (on[k]) row[e[k].x] = penalised(x[k], r, e[k].y);
      }
    }
    __syncthreads();
    if (tid == 0 && !found && token >= 0 && token < vocab && n < capacity) {
      mine[n] = make_int2(token, 2);
      used[r.slot] = n + 1;
      if (is_allowed(mask, token)) row[token] = penalised(row[token], r, 2);
    }
    __syncthreads();
  }
  while (bias_at < r.bias_end) {
    if (is_allowed(mask, bias_token)) row[bias_token] = bias == -INFINITY ? bias : row[bias_token] + bias;
    bias_at += ADJUST_THREADS;
    if (bias_at < r.bias_end) {
      bias_token = bias_tokens[bias_at];
      bias = bias_values[bias_at];
    }
  }
}

// The host has checked the rows' slots, masks and bias tokens against the sizes given here.
extern "C" int tnx_adjust_logits(float* logits, const int* rules, const int* bias_tokens, const float* bias_values, int* entries, int* used,
                                 int capacity, const int* last, const int* masks, int rows, int vocab, hipStream_t stream) {
  TNX_REQUIRE(rows >= 0 && rows <= 65535 && vocab > 0 && vocab < (1 << 30) && capacity >= 0,
              "adjust_logits: bad sizes rows=%d vocab=%d capacity=%d", rows, vocab, capacity);
  if (rows == 0) return 0;
  const int per_block = ADJUST_THREADS * ADJUST_BARRED;
  const int blocks = 1 + (masks ? (vocab + per_block - 1) / per_block : 0);
  adjust_logits_kernel<<<dim3(blocks, rows), ADJUST_THREADS, 0, stream>>>(logits, (const RowRules*)rules, bias_tokens, bias_values,
                                                                          (int2*)entries, used, capacity, last, (const unsigned*)masks,
                                                                          (vocab + 31) / 32, vocab);
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

// log2(e) in two parts, of which the second is what the first lacks
#define LOG2E_HI 1.44269502162933349609375f
#define LOG2E_LO 1.92596299112661746887e-8f
// exp(d) for d <= 0 by the hardware's power of two: the roundings of d and of the power's argument are left, 2^-24 of |d| each.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(fmaf(d, LOG2E_HI, d * LOG2E_LO)); }

// exp(x - r) for many x and one r is 2^(x log2(e) - r log2(e)): one multiply-add and the power an element, with the product of r
// rounded, and what the rounding lost put back behind the sum. Left is the rounding of the power's argument, and 1.3e-8 of x - r for
// what the constant lacks.
struct PowersBelow {
  float r, shift, lost;
  __device__ __forceinline__ void at(float reference) {
    r = reference;
    shift = -(r * LOG2E_HI);
    lost = fmaf(-r, LOG2E_HI, -shift);
  }
  __device__ __forceinline__ float operator()(float x) const { return __builtin_amdgcn_exp2f(fmaf(x, LOG2E_HI, shift)); }
  __device__ __forceinline__ float back() const { return __builtin_amdgcn_exp2f(lost); }
};
// `lost` is up to half a unit in the last place of r log2(e): 8 where |r| is just below this, from about 1.4e9 on beyond what the
// hardware's powers hold (2^-126 to 2^128, and less than that is 0). Rows whose maximum lies further out are summed again with care.
#define SCORE_FAR 1e8f

// A row read four logits at a time from the boundary of 16 bytes at or before it: quad q holds elements 4 q - lead to 4 q - lead + 3;
// what lies outside the row reads as -inf.
struct Quads {
  const float* row;
  int vocab, lead, count;
  __device__ __forceinline__ Quads(const float* r, int v)
      : row(r), vocab(v), lead((int)(((uintptr_t)r >> 2) & 3)), count((v + (int)(((uintptr_t)r >> 2) & 3) + 3) / 4) {}
  __device__ __forceinline__ int first(int q) const { return 4 * q - lead; }
  __device__ __forceinline__ bool whole(int q) const { return 4 * q - lead >= 0 && 4 * q - lead + 3 < vocab; }
  template <bool ONCE>
  __device__ __forceinline__ f32x4 inside(int q) const {
    const f32x4* p = (const f32x4*)(row + 4 * q - lead);
    return ONCE ? __builtin_nontemporal_load(p) : *p;
  }
  __device__ __forceinline__ f32x4 operator()(int q) const {
    if (whole(q)) return inside<false>(q);
    const int i = 4 * q - lead;
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = i + e >= 0 && i + e < vocab ? row[i + e] : -INFINITY;
    return x;
  }
};

#define SCORE_GROUPS 128       // groups of threads whose largest logits are ranked against one another
#define SCORE_GATHER 1024      // the most logits that are gathered for the alternatives
#define SCORE_MOST_TOP 32

// One block of THREADS a row, one pass over it with a running maximum and sum.
//
// The alternatives come from the same pass: a thread notes its largest logit, and as many groups of threads as alternatives are
// wanted, those with the largest logits, hold all of them (of the others each group's best is already beaten by so many). Only
// the logits of these groups are looked at again, and those of them that are no smaller than the last group's best, hardly more than
// the alternatives themselves, are ranked in LDS. Should they be more than fit (the best of a long row all in a few threads' places),
// the alternatives are found one by one, each with a pass of its own.
//
// Many rows are bound by memory. A few are bound by what one compute unit can do: a row of 50,272 takes 5.7 us without and 9.4 with
// alternatives, of which 2.6 are those of any launch, about 3 the powers and maxima, and the rest five barriers with a trip through
// LDS or memory each. (Rows held in registers, all asked for at once: 7.3 and 17. Groups of 128 for 256, 2 keys a read: 4 us of 6.)
template <int THREADS, bool TOP, bool ONCE>
__global__ void __launch_bounds__(THREADS)
log_probs_kernel(const float* __restrict__ logits, const int* __restrict__ tokens, float* __restrict__ out, int* __restrict__ top_tokens,
                 float* __restrict__ top_out, int top, int vocab) {
  constexpr int WAVES = THREADS / 64, PER_GROUP = THREADS / SCORE_GROUPS;
  __shared__ float scratch[WAVES], sums[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Quads quads(logits + (size_t)blockIdx.x * vocab, vocab);
  const float* row = quads.row;

  float m = -INFINITY, s = 0.f;
  int at = max(quads.first(tid), 0);          // where the thread's largest logit came first
  PowersBelow power;
  power.at(-SCORE_FAR);
  auto take = [&](const f32x4 (&v)[4], int q0) __attribute__((always_inline)) {
    float here = v[0][0];                     // (the larger of a number and a NaN is the number)
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) here = fmaxf(here, v[k][e]);
    if (here > m) {
      PowersBelow next;
      next.at(fmaxf(here, -SCORE_FAR));
      s *= __builtin_amdgcn_exp2f(fmaf(power.r - next.r, LOG2E_HI, power.lost - next.lost));
      power = next;
      m = here;
      if constexpr (TOP) {
#pragma unroll
        for (int k = 3; k >= 0; --k)
#pragma unroll
          for (int e = 3; e >= 0; --e) at = v[k][e] == here ? quads.first(q0 + k * THREADS) + e : at;
      }
    }
    float part[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[e & 1] += power(v[k][e]);
    s += part[0] + part[1];
  };
  for (int b = 0; b < quads.count; b += 4 * THREADS) {
    f32x4 v[4];
    if (quads.whole(b) && quads.whole(b + 4 * THREADS - 1)) {         // the same for all threads
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = quads.template inside<ONCE>(b + tid + k * THREADS);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = quads(b + tid + k * THREADS);
    }
    take(v, b + tid);
  }
  const float mine = m;
  m = wave_max(m);
  if (lane == 0) scratch[wave] = m;
  __syncthreads();
  m = scratch[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) m = fmaxf(m, scratch[w]);
  s = block_sum<WAVES>(s * power.back() * exp_of(power.r - m), sums);
  if (!(s >= 0.5f && s < INFINITY) || !(fabsf(m) < SCORE_FAR)) {
    // with a NaN somewhere, or a maximum that is far out or none: one by one (the maximum itself is 1 of any sum that is right)
    float exact = 0.f;
    for (int q = tid; q < quads.count; q += THREADS) {
      const f32x4 x = quads(q);
#pragma unroll
      for (int e = 0; e < 4; ++e) exact += x[e] > -INFINITY ? (x[e] == m ? 1.f : exp_of(x[e] - m)) : 0.f;
    }
    s = block_sum<WAVES>(exact, sums);
  }
  const float log_l = logf(s);
  if (tid == 0) {
    const int t = tokens[blockIdx.x];
    out[blockIdx.x] = t >= 0 && t < vocab ? log_prob_of(row[t], m, log_l) : -INFINITY;
  }
  if constexpr (TOP) {
    __shared__ __align__(16) unsigned long long best[SCORE_GROUPS];
    __shared__ unsigned long long gathered[SCORE_GATHER], one[WAVES];
    __shared__ int winners[SCORE_MOST_TOP], num_gathered;
    __shared__ unsigned long long least;
    // the thread's best as a key (its logit, then the lower token id), and its group's
    unsigned long long key = tid < quads.count ? order_key(mine, at) : 0;
#pragma unroll
    for (int o = 1; o < PER_GROUP; o <<= 1) {
      const unsigned long long other = __shfl_xor(key, o, 64);
      key = other > key ? other : key;
    }
    if (tid % PER_GROUP == 0) best[tid / PER_GROUP] = key;
    if (tid == 0) {
      num_gathered = 0;
      least = 0;
    }
    __syncthreads();
    const int groups = (min(quads.count, THREADS) + PER_GROUP - 1) / PER_GROUP;      // that have logits; the others' keys are 0
    if (tid < groups) {
      const unsigned long long b = best[tid];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < SCORE_GROUPS; j += 2) {
        const ulonglong2 two = *(const ulonglong2*)&best[j];
        rank += (two.x > b ? 1 : 0) + (two.y > b ? 1 : 0);
      }
      if (rank < top) winners[rank] = tid;
      if (rank == top - 1) least = b;                    // (fewer groups than alternatives: everything is gathered)
    }
    __syncthreads();
    // group g's quads are those of its threads: k * THREADS + PER_GROUP * g + j
    const int rounds = (quads.count + THREADS - 1) / THREADS * PER_GROUP;
    const unsigned long long floor_key = least;
    // a wave takes 64 of them at a time
    const int parts = (rounds + 63) / 64;
    for (int item = wave; item < min(top, groups) * parts; item += WAVES) {
      const int n = item % parts * 64 + lane;
      if (n < rounds) {
        const int q = n / PER_GROUP * THREADS + PER_GROUP * winners[item / parts] + n % PER_GROUP;
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
          values[rank] = log_prob_of(key_value(k), m, log_l);
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
          values[r] = log_prob_of(key_value(b), m, log_l);
        }
      }
    }
  }
}

template <int THREADS, bool ONCE>
static void launch_log_probs(const float* logits, const int* tokens, float* out, int* top_tokens, float* top_out, int top, int rows, int vocab,
                             hipStream_t stream) {
  if (top) log_probs_kernel<THREADS, true, ONCE><<<rows, THREADS, 0, stream>>>(logits, tokens, out, top_tokens, top_out, top, vocab);
  else log_probs_kernel<THREADS, false, ONCE><<<rows, THREADS, 0, stream>>>(logits, tokens, out, top_tokens, top_out, top, vocab);
}

extern "C" int tnx_log_probs(const float* logits, const int* tokens, float* out, int* top_tokens, float* top_out, int top, int rows,
                             int vocab, hipStream_t stream) {
  TNX_REQUIRE(rows >= 0 && vocab > 0 && vocab < (1 << 30) && top >= 0 && top <= SCORE_MOST_TOP && top <= vocab,
              "log_probs: bad sizes rows=%d vocab=%d top=%d", rows, vocab, top);
  if (rows == 0) return 0;
  // 1,024 threads where each has a whole round of 16 logits and the rows are no more than the blocks that run at once, 512 otherwise.
  // In us, 1,024 / 512: 64 rows of 50,272 with 20 alternatives 11.9 / 14.0, 512 rows 25.0 / 26.4, 777 rows 40.9 / 40.2; 64 rows of
  // 32,001 with 5 9.5 / 10.3, of 12,000 7.1 / 7.2, of 5,000 7.0 / 6.4, 2,048 rows of 5,000 29.3 / 18.7.
  // Rows that the caches cannot hold are marked as read once: 2,048 rows of 50,272 without alternatives 62.3 us (6.6 TB/s), 70.9 plain,
  // 2,048 of 32,001 41.8 and 46.6; but 777 of 32,001 (99 MB) with 20 28.6 and 27.5, 64 of 50,272 16.9 and 14.0.
  const bool once = (long long)rows * vocab * 4 >= (128ll << 20);
  if (rows <= 512 && vocab >= 16 * 1024) launch_log_probs<1024, false>(logits, tokens, out, top_tokens, top_out, top, rows, vocab, stream);
  else if (once) launch_log_probs<512, true>(logits, tokens, out, top_tokens, top_out, top, rows, vocab, stream);
  else launch_log_probs<512, false>(logits, tokens, out, top_tokens, top_out, top, rows, vocab, stream);
  TNX_CHECK_LAUNCH("log_probs");
  return 0;
}

// The log-probabilities, those of the alternatives and their tokens, one behind the other in pinned host memory.
__global__ void send_log_probs_kernel(const int* __restrict__ out, const int* __restrict__ best, const int* __restrict__ ids, int rows,
                                      int top, int* __restrict__ landing) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x, n = rows * top;
  if (i < rows) landing[i] = out[i];
  else if (i < rows + n) landing[i] = best[i - rows];
  else if (i < rows + 2 * n) landing[i] = ids[i - rows - n];
}

extern "C" int tnx_send_log_probs(const float* out, const float* best, const int* ids, int rows, int top, int* landing, hipStream_t stream) {
  TNX_REQUIRE(rows >= 0 && rows < (1 << 24) && top >= 0 && top <= SCORE_MOST_TOP && landing, "send_log_probs: bad sizes rows=%d top=%d", rows,
              top);
  if (rows == 0) return 0;
  send_log_probs_kernel<<<(rows * (1 + 2 * top) + 255) / 256, 256, 0, stream>>>((const int*)out, (const int*)best, ids, rows, top, landing);
  TNX_CHECK_LAUNCH("send_log_probs");
  return 0;
}
