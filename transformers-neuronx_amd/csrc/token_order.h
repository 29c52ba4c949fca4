// The order among a row's tokens, one for the choice of a token and for the alternatives that are told beside it: by logit, ties to the
// lower token id, a NaN as -inf.
#pragma once
#include "common.h"

// ordered logit bits above the inverted token id: the larger key comes first
__device__ __forceinline__ uint64_t order_key(float x, int idx) {
  if (x != x) x = -INFINITY;  // NaN orders last
  if (x == 0.f) x = 0.f;      // -0 and +0 are one value: the lower token id decides between them
  uint32_t u = __float_as_uint(x);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)(~(uint32_t)idx);
}

// the logit of a key
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u);
}
