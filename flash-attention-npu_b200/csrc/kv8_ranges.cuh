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

}  // namespace fa
