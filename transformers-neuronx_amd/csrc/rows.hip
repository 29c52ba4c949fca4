// Rows of several tensors copied to other rows of them: the pages of a cache (every layer's keys and values) and
// the per-request state beside them, when a request is forked, a pool compacted, or its size changed.
//
//   target[o][p][:] = source[o][p][:]   for every o, and every place p < tokens
//
// A row is `outer` runs of places, one behind the other; a place is `inner` bytes. Keys [heads, page, size] are
// `heads` runs of places of a token's values; values [heads, size, page], turned inside a page, are heads * size runs
// of places of one number. Only the places that hold tokens are moved; what lies behind them in the target stays.
#include "common.h"

TNX_DEFINE_ERROR_API

// One tensor of a set, as the host writes it (64-bit words).
struct RowTensor {
  const char* from;         // where its rows are read
  char* to;                 // and where they are written: the same tensor, or its successor of another size
  long long from_stride;    // bytes from one row to the next
  long long to_stride;
  long long run;            // bytes of a run: places * inner
  long long inner;          // bytes of a place; 0: the tensor counts no tokens, its rows are copied whole
  long long outer;          // runs in a row
  long long grain;          // 16 where every run of both sides begins on 16 bytes; 4, 2 or 1 otherwise
};

#define ROW_THREADS 256

template <typename V>
__device__ __forceinline__ void copy_runs(const char* from, char* to, long long stride, unsigned length, unsigned runs) {
  // `length` bytes of each of `runs` runs that lie `stride` bytes apart; the last unit of a run may be a part of one
  const unsigned per_run = (length + sizeof(V) - 1) / sizeof(V), units = per_run * runs;
  for (unsigned u = blockIdx.x * ROW_THREADS + threadIdx.x; u < units; u += gridDim.x * ROW_THREADS) {
    const unsigned o = u / per_run, at = (u - o * per_run) * (unsigned)sizeof(V);
    const char* s = from + o * stride + at;
    char* d = to + o * stride + at;
    if (at + sizeof(V) <= length) {
      *(V*)d = *(const V*)s;
    } else {
      for (unsigned b = 0; b < length - at; ++b) d[b] = s[b];
    }
  }
}

// pairs[i] = {source row, target row, tokens}; tokens below zero: the whole row.
__global__ void __launch_bounds__(ROW_THREADS)
copy_rows_kernel(const RowTensor* __restrict__ tensors, const int* __restrict__ pairs) {
  const RowTensor t = tensors[blockIdx.y];
  const int* p = pairs + 3 * (size_t)blockIdx.z;
  const char* from = t.from + p[0] * t.from_stride;
  char* to = t.to + p[1] * t.to_stride;
  unsigned length = (unsigned)t.run, runs = (unsigned)t.outer;
  if (p[2] >= 0 && t.inner > 0) length = (unsigned)min(t.run, p[2] * t.inner);
  if (length == t.run) {       // whole runs lie one behind the other
    length *= runs;
    runs = 1;
  }
  if (t.grain == 16) copy_runs<tnx_u32x4>(from, to, t.run, length, runs);
  else if (t.grain == 4) copy_runs<unsigned>(from, to, t.run, length, runs);
  else if (t.grain == 2) copy_runs<unsigned short>(from, to, t.run, length, runs);
  else copy_runs<unsigned char>(from, to, t.run, length, runs);
}

// `largest`: the bytes of the set's largest row (below 2^31).
extern "C" int tnx_copy_rows(const void* tensors, int num_tensors, const int* pairs, int num_pairs, long long largest,
                             hipStream_t stream) {
  TNX_REQUIRE(num_tensors > 0 && num_tensors <= 65535 && num_pairs >= 0 && largest > 0 && largest < (1ll << 31),
              "copy_rows: bad sizes tensors=%d pairs=%d largest row=%lld", num_tensors, num_pairs, largest);
  const unsigned blocks = (unsigned)((largest + ROW_THREADS * 64 - 1) / (ROW_THREADS * 64));
  for (int first = 0; first < num_pairs; first += 65535) {
    const unsigned n = (unsigned)(num_pairs - first < 65535 ? num_pairs - first : 65535);
    copy_rows_kernel<<<dim3(blocks, num_tensors, n), ROW_THREADS, 0, stream>>>((const RowTensor*)tensors, pairs + 3 * (size_t)first);
    TNX_CHECK_LAUNCH("copy_rows");
  }
  return 0;
}
