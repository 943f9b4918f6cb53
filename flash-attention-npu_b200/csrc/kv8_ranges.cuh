// Rows and keys of a sequence over an 8-bit KV cache, as arithmetic that the kernels (kv8.cuh) and a host test share: offsets,
// lengths and windows come from the caller's tensors and are never trusted.
#pragma once

#ifdef __CUDACC__
#define FA_KV8_HD __host__ __device__ __forceinline__
#else
#define FA_KV8_HD inline
#endif

#include <stdint.h>

namespace fa {

// Query rows [row0, row0 + len) of a packed sequence from its two offsets, cut to the `total` rows there are; false: they had to be.
FA_KV8_HD bool kv8_query_rows(int from, int upto, int total, int& row0, int& len) {
  row0 = from < 0 ? 0 : from > total ? total : from;
  const int end = upto < row0 ? row0 : upto > total ? total : upto;
  len = end - row0;
  return row0 == from && end == upto;
}

struct Kv8Mask {
  int wl, wr;  // taken literally where `local`: a side below -1 ends in front of (or starts behind) the diagonal
  bool causal, local;
};

// Keys [lo, hi) of the k_len that the query tokens i_lo .. i_hi of a sequence see; none: an empty range within them.  (A range behind
// the last key had the page table read there, and the scales of blocks that nobody has written.)  Within 32 bits: the planner holds keys and
// rows to 2^30, and the sides of a window to [-2^30, 2^30).
FA_KV8_HD void kv8_key_range(const Kv8Mask& m, int k_len, int koff, int i_lo, int i_hi, int& lo, int& hi) {
  lo = 0;
  hi = k_len;
  if (m.causal && i_hi + koff + 1 < hi) hi = i_hi + koff + 1;
  if (m.local) {
    const int first = i_lo + koff - m.wl, behind = i_hi + koff + m.wr + 1;
    lo = first < 0 ? 0 : first > k_len ? k_len : first;
    hi = behind > k_len ? k_len : behind;
  }
  if (hi < lo) hi = lo;
}

}  // namespace fa
