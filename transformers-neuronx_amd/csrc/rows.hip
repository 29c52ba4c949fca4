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
  long long grain;          // 16 where every run of both sides begins on 16 bytes; else 4, 2 or 1, of which a place has a whole number
};

#define ROW_THREADS 256
#define ROW_UNITS 4           // units of a thread that are asked for together, before any is stored

// The first `bytes` (below 16) of a unit, by pieces of the sizes that make them up.
__device__ __forceinline__ void store_part(char* d, tnx_u32x4 v, unsigned bytes) {
  unsigned long long w[2] = {((unsigned long long)v[1] << 32) | v[0], ((unsigned long long)v[3] << 32) | v[2]};
  unsigned long long x = w[0];
  if (bytes & 8) {
    *(unsigned long long*)d = x;
    d += 8;
    x = w[1];
  }
  if (bytes & 4) {
    *(unsigned*)d = (unsigned)x;
    d += 4;
    x >>= 32;
  }
  if (bytes & 2) {
    *(unsigned short*)d = (unsigned short)x;
    d += 2;
    x >>= 16;
  }
  if (bytes & 1) *d = (char)x;
}
template <typename V>
__device__ __forceinline__ void store_part(char*, V, unsigned) {}

// `length` bytes of each of `runs` runs that lie `stride` bytes apart, to every target. A unit is a V; the last of a run may be a
// part of one where V is 16 bytes (runs there are whole units long, so all of it can be read), and never is for smaller V, of which
// a place holds a whole number.
template <typename V>
__device__ __forceinline__ void copy_runs(const char* from, char* to, long long to_stride, const int* targets, int num_targets,
                                          long long stride, unsigned length, unsigned runs) {
  constexpr unsigned SIZE = sizeof(V);
  const unsigned per_run = (length + SIZE - 1) / SIZE, units = per_run * runs;
  for (unsigned u0 = blockIdx.x * (ROW_THREADS * ROW_UNITS) + threadIdx.x; u0 < units; u0 += gridDim.x * (ROW_THREADS * ROW_UNITS)) {
    V v[ROW_UNITS];
    long long at[ROW_UNITS];
    unsigned left[ROW_UNITS];
#pragma unroll
    for (int k = 0; k < ROW_UNITS; ++k) {
      const unsigned u = min(u0 + k * ROW_THREADS, units - 1);
      const unsigned o = u / per_run, in = (u - o * per_run) * SIZE;
      at[k] = o * stride + in;
      left[k] = u0 + k * ROW_THREADS < units ? min(length - in, SIZE) : 0;
      v[k] = *(const V*)(from + at[k]);
    }
    for (int i = 0; i < num_targets; ++i) {
      char* d = to + targets[i] * to_stride;
#pragma unroll
      for (int k = 0; k < ROW_UNITS; ++k) {
        if (left[k] == SIZE) *(V*)(d + at[k]) = v[k];
        else if (left[k]) store_part(d + at[k], v[k], left[k]);
      }
    }
  }
}

// groups[i] = {source row, tokens, first target, targets}: a source that several rows become is read once. Tokens below zero: the
// whole row.
__global__ void __launch_bounds__(ROW_THREADS)
copy_rows_kernel(const RowTensor* __restrict__ tensors, const int4* __restrict__ groups, const int* __restrict__ targets) {
  const RowTensor t = tensors[blockIdx.y];
  const int4 g = groups[blockIdx.z];
  const char* from = t.from + g.x * t.from_stride;
  unsigned length = (unsigned)t.run, runs = (unsigned)t.outer;
  if (g.y >= 0 && t.inner > 0) length = (unsigned)min(t.run, g.y * t.inner);
  if (length == 0) return;
  if (length == t.run) {       // whole runs lie one behind the other
    length *= runs;
    runs = 1;
  }
  const int* to = targets + g.z;
  if (t.grain == 16) copy_runs<tnx_u32x4>(from, t.to, t.to_stride, to, g.w, t.run, length, runs);
  else if (t.grain == 4) copy_runs<unsigned>(from, t.to, t.to_stride, to, g.w, t.run, length, runs);
  else if (t.grain == 2) copy_runs<unsigned short>(from, t.to, t.to_stride, to, g.w, t.run, length, runs);
  else copy_runs<unsigned char>(from, t.to, t.to_stride, to, g.w, t.run, length, runs);
}

// `units`: of 16 bytes or less, in what is copied of the set's largest row (below 2^31).
extern "C" int tnx_copy_rows(const void* tensors, int num_tensors, const int* groups, int num_groups, const int* targets, long long units,
                             hipStream_t stream) {
  TNX_REQUIRE(num_tensors > 0 && num_tensors <= 65535 && num_groups >= 0 && units > 0 && units < (1ll << 31),
              "copy_rows: bad sizes tensors=%d groups=%d units=%lld", num_tensors, num_groups, units);
  const unsigned blocks = (unsigned)((units + ROW_THREADS * ROW_UNITS - 1) / (ROW_THREADS * ROW_UNITS));
  for (int first = 0; first < num_groups; first += 65535) {
    const unsigned n = (unsigned)(num_groups - first < 65535 ? num_groups - first : 65535);
    copy_rows_kernel<<<dim3(blocks, num_tensors, n), ROW_THREADS, 0, stream>>>((const RowTensor*)tensors, (const int4*)groups + first,
                                                                               targets);
    TNX_CHECK_LAUNCH("copy_rows");
  }
  return 0;
}
