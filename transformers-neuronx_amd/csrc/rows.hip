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

#define ROW_LINE 128          // bytes that memory is read by; a half of it is what it is written by at least

// The first `bytes` (0 to 16) of `v`, and the rest of `w`.
__device__ __forceinline__ tnx_u32x4 joined(tnx_u32x4 v, tnx_u32x4 w, unsigned bytes) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int here = min(max((int)bytes - 4 * j, 0), 4);
    const unsigned mask = here == 4 ? ~0u : (1u << (8 * here)) - 1u;
    w[j] = (v[j] & mask) | (w[j] & ~mask);
  }
  return w;
}

// The first `bytes` (0 to 15) of a unit stored, by pieces of the sizes that make them up.
__device__ __forceinline__ void store_part(char* d, tnx_u32x4 v, unsigned bytes) {
  unsigned long long x = ((unsigned long long)v[1] << 32) | v[0];
  if (bytes & 8) {
    *(unsigned long long*)d = x;
    d += 8;
    x = ((unsigned long long)v[3] << 32) | v[2];
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

// `length` bytes of each of `runs` runs that lie `stride` bytes apart, to every target, by units of a V. A run may end inside a unit
// where V is 16 bytes (it can be read whole: runs are whole units long); of a smaller V a place holds a whole number.
//
// FILL: what a run's last line lacks is filled up with what the target has there. Values turned inside a page are runs of 128 bytes,
// of which a page that is not full moves a part; memory then reads, changes and writes back what it is given a part of. Values of 32
// layers of 32 heads of 128, page 64, 8 pages to 24, in us: whole pages 77; 40 tokens (80 bytes of 128) parts 226, filled up 147; 32
// tokens (64 bytes) parts 57, filled up 145; 20 tokens 106 and 151. So lines are filled up where more than half of one is moved.
//
// What bounds it is memory: stores are marked as not read again soon, which leaves the caches to the sources, a thread moves one unit,
// and the blocks that run side by side are those of one tensor, whose rows lie nearest to one another. 20 whole pages of OPT-6.7b to 20
// others, 0.67 GB read and as much written: 220 us, 6.1 TB/s (a large copy by the runtime 4.9); four units a thread 252, tensors side by
// side 254, both 270; with plain stores 4.7 TB/s.
template <typename V, bool FILL>
__device__ __forceinline__ void copy_runs(const char* from, char* to, long long to_stride, const int* targets, int num_targets,
                                          long long stride, unsigned length, unsigned runs) {
  constexpr unsigned SIZE = sizeof(V);
  const unsigned wide = FILL ? (unsigned)min((long long)(length + ROW_LINE - 1) / ROW_LINE * ROW_LINE, stride) : length;
  const unsigned per_run = (wide + SIZE - 1) / SIZE, units = per_run * runs;
  for (unsigned u = blockIdx.x * ROW_THREADS + threadIdx.x; u < units; u += gridDim.x * ROW_THREADS) {
    const unsigned o = u / per_run, in = (u - o * per_run) * SIZE;
    const unsigned mine = in < length ? min(length - in, SIZE) : 0;        // bytes of the unit that are the source's
    const long long at = o * stride + in;
    const V v = *(const V*)(from + at);
    for (int i = 0; i < num_targets; ++i) {
      V* d = (V*)(to + targets[i] * to_stride + at);
      if constexpr (FILL) {
        V w = v;
        if (mine < SIZE) w = __builtin_nontemporal_load(d);
        __builtin_nontemporal_store(joined(v, w, mine), d);      // (one store for what a wave has of a line)
      } else if (mine == SIZE) {
        __builtin_nontemporal_store(v, d);
      } else if constexpr (SIZE == 16) {
        store_part((char*)d, v, mine);
      }
    }
  }
}

// A list of rows, as the host writes it: for every group of rows that one source becomes {source row, tokens, first target, targets}
// (tokens below zero: the whole row), then the targets of all groups. A short one goes along with the launch, which saves a copy of its
// own and the wait for it: 24 layers of OPT-350m, 1 page to 3, 21 -> 9 us a call.
#define ROW_WORDS 256
struct RowList {
  int words[ROW_WORDS];
};

// A source that several rows become is read once.
template <bool HERE>
__global__ void __launch_bounds__(ROW_THREADS)
copy_rows_kernel(const RowTensor* __restrict__ tensors, const RowList list, const int* __restrict__ far, int first_group, int num_groups) {
  const RowTensor t = tensors[blockIdx.z];
  const int* words = HERE ? list.words : far;
  const int at = 4 * (first_group + (int)blockIdx.y);
  const int4 g = make_int4(words[at], words[at + 1], words[at + 2], words[at + 3]);
  const char* from = t.from + g.x * t.from_stride;
  unsigned length = (unsigned)t.run, runs = (unsigned)t.outer;
  if (g.y >= 0 && t.inner > 0) length = (unsigned)min(t.run, g.y * t.inner);
  if (length == 0) return;
  if (length == t.run) {       // whole runs lie one behind the other
    length *= runs;
    runs = 1;
  }
  const int* to = words + 4 * num_groups + g.z;
  const bool fill = runs > 1 && length % ROW_LINE > ROW_LINE / 2;
  if (t.grain == 16 && fill) copy_runs<tnx_u32x4, true>(from, t.to, t.to_stride, to, g.w, t.run, length, runs);
  else if (t.grain == 16) copy_runs<tnx_u32x4, false>(from, t.to, t.to_stride, to, g.w, t.run, length, runs);
  else if (t.grain == 4) copy_runs<unsigned, false>(from, t.to, t.to_stride, to, g.w, t.run, length, runs);
  else if (t.grain == 2) copy_runs<unsigned short, false>(from, t.to, t.to_stride, to, g.w, t.run, length, runs);
  else copy_runs<unsigned char, false>(from, t.to, t.to_stride, to, g.w, t.run, length, runs);
}

// The list lies in `host` where it has at most ROW_WORDS words, else in `far` (device memory). `units`: of 16 bytes or less, in what
// is copied of the set's largest row (below 2^31).
extern "C" int tnx_copy_rows(const void* tensors, int num_tensors, const int* host, int num_words, const int* far, int num_groups,
                             long long units, hipStream_t stream) {
  TNX_REQUIRE(num_tensors > 0 && num_tensors <= 65535 && num_groups > 0 && num_words > 4 * num_groups && units > 0 && units < (1ll << 31),
              "copy_rows: bad sizes tensors=%d groups=%d words=%d units=%lld", num_tensors, num_groups, num_words, units);
  TNX_REQUIRE(num_words <= ROW_WORDS ? host != nullptr : far != nullptr, "copy_rows: a list of %d words is missing", num_words);
  const unsigned blocks = (unsigned)((units + ROW_THREADS - 1) / ROW_THREADS);
  RowList list;
  if (num_words <= ROW_WORDS) {
    for (int i = 0; i < num_words; ++i) list.words[i] = host[i];
    for (int i = num_words; i < ROW_WORDS; ++i) list.words[i] = 0;
  }
  for (int first = 0; first < num_groups; first += 65535) {
    const dim3 grid(blocks, (unsigned)(num_groups - first < 65535 ? num_groups - first : 65535), num_tensors);
    if (num_words <= ROW_WORDS)
      copy_rows_kernel<true><<<grid, ROW_THREADS, 0, stream>>>((const RowTensor*)tensors, list, nullptr, first, num_groups);
    else
      copy_rows_kernel<false><<<grid, ROW_THREADS, 0, stream>>>((const RowTensor*)tensors, RowList{}, far, first, num_groups);
    TNX_CHECK_LAUNCH("copy_rows");
  }
  return 0;
}
