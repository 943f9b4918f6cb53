// New keys and values -> codes and scales of an 8-bit KV cache.
//
// The scale of a (token block, kv head) is the smallest power of two, 2^-40 at least, that brings the largest finite element
// into the codes' range (448 for e4m3, 127 for int8).  A power of two makes dividing by it, and expressing held codes in a larger one,
// exact up to the one rounding to a code.  It costs nothing in e4m3 (a floating-point code keeps its relative precision) and up to one
// bit in int8: codes of normal elements, blocks of 128 tokens of 128, are off by 1.40 % of the elements' size (2-norm) where amax / 127 as the
// scale gives 0.94 %.  A run is the new tokens that fall into one block: if rows are there in front of it, the block keeps its scale where that is larger,
// and otherwise its codes are rewritten in the new one; a run that starts at the block's first row starts the block afresh, so a
// recycled page needs no clearing.  Rows behind the run are left alone.  Runs own their blocks: no atomics, no order to depend on.
//
// HBM-bound: 2 bytes an element in, 1 out.  A run's elements stay in registers between the maximum and the rounding, eight 16-byte chunks a
// thread, so they are read once: a warp by itself writes a run of up to 256 chunks (16 tokens of head dim 128, and every
// decoding token), the CTA's eight warps together one of up to 2048; what a longer run has beyond that is read twice.
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"

namespace fa {

constexpr int kLeastScaleExp = 127 - 40;
constexpr int kAppendThreads = 256, kAppendWarps = kAppendThreads / 32;
constexpr int kBatch = 8, kWarpRun = 32 * kBatch;

// Bit pattern of the power of two above, from the largest |finite element| as an fp32 value.
template <int CODE>
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) & 255;
  const uint32_t m = u & 0x7fffffu;
  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  const int s = CODE == FA_CODE_E4M3 ? e - 8 + (m > 0x600000u) : e - 6 + (m > 0x7e0000u);
  return __uint_as_float((uint32_t)max(s, kLeastScaleExp) << 23);
}

// Two values in units of the scale -> two codes.  Round to nearest even; infinities saturate; NaN stays NaN (e4m3) or is 0 (int8).
template <int CODE>
__device__ __forceinline__ uint32_t encode2(float a, float b) {
  if (CODE == FA_CODE_E4M3) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(b), "f"(a));
    return r;
  }
  const int x = min(max(__float2int_rn(a), -127), 127), y = min(max(__float2int_rn(b), -127), 127);
  return (uint32_t)(x & 255) | ((uint32_t)(y & 255) << 8);
}

template <typename T>
__device__ __forceinline__ void unpack_pair(uint32_t w, float& a, float& b) {
  if (std::is_same<T, __nv_bfloat16>::value) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x;
    b = f.y;
  }
}
// Running maximum of |element| per half word: NaN when one is (NAN_TOO), or as if none were.
template <typename T, bool NAN_TOO>
__device__ __forceinline__ uint32_t abs_max2(uint32_t mx, uint32_t w) {
  w &= 0x7fff7fffu;
  uint32_t r;
  if (std::is_same<T, __nv_bfloat16>::value) {
    if (NAN_TOO) asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(mx), "r"(w));
    else asm("max.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(mx), "r"(w));
  } else {
    if (NAN_TOO) asm("max.NaN.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(mx), "r"(w));
    else asm("max.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(mx), "r"(w));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t abs_max8(uint32_t mx, const uint4& x) {
  return abs_max2<T, true>(abs_max2<T, true>(abs_max2<T, true>(abs_max2<T, true>(mx, x.x), x.y), x.z), x.w);
}
// A pair with its infinities taken out.
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  constexpr uint32_t inf = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  return ((w & 0x7fffu) == inf ? 0u : w & 0xffffu) | (((w >> 16) & 0x7fffu) == inf ? 0u : w & 0xffff0000u);
}

// How GROUP threads share a run's 16-byte chunks: each has one column of every step-th row (what is left over idles).
struct Share {
  int col, row, step;
  __device__ __forceinline__ Share(int t, int group, int chunks) {
    step = group / chunks;
    row = t / chunks;
    col = t - row * chunks;
    if (row >= step) row = 1 << 30;
  }
};

// One run: `rows` tokens into block rows first .. first + rows - 1.  GROUP threads work together (a warp, or the whole CTA), t is
// the thread among them; load(r): its column of new token r; dst: of the
// block's first row.
// BATCH: chunks of a thread that stay in registers; 1 is a short piece of code for runs of a token (a decoding step is over before the
// instructions of the long one have arrived: 64 tokens 15.3 us with it alone).
template <typename T, int CODE, int GROUP, int BATCH, typename Load>
__device__ __forceinline__ void write_run(Load load, uint8_t* dst, int64_t row_stride, int first, int rows, const Share& my, float* scale, int t,
                                          float* s_red) {
  const float old = *scale;
  uint4 keep[BATCH];
  uint32_t mx = 0;
  auto fetch = [&](int r0) {
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      keep[k] = make_uint4(0, 0, 0, 0);
      if (r0 + k * my.step < rows) keep[k] = load(r0 + k * my.step);
    }
  };
  const int more = BATCH * my.step;
  for (int r0 = my.row + more; r0 < rows; r0 += more) {  // (the first batch last: it stays)
    fetch(r0);
#pragma unroll
    for (int k = 0; k < BATCH; ++k) mx = abs_max8<T>(mx, keep[k]);
  }
  fetch(my.row);
#pragma unroll
  for (int k = 0; k < BATCH; ++k) mx = abs_max8<T>(mx, keep[k]);
  float lo, hi;
  unpack_pair<T>(mx, lo, hi);
  const bool finite = lo < INFINITY && hi < INFINITY;
  if (!finite) {  // rare: the maximum without infinities and NaN
    mx = 0;
#pragma unroll 1
    for (int r = my.row; r < rows; r += my.step) {
      const uint4 x = load(r);
      mx = abs_max2<T, false>(abs_max2<T, false>(mx, finite2<T>(x.x)), finite2<T>(x.y));
      mx = abs_max2<T, false>(abs_max2<T, false>(mx, finite2<T>(x.z)), finite2<T>(x.w));
    }
    unpack_pair<T>(mx, lo, hi);
  }
  float amax = fmaxf(lo, hi);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (GROUP > 32) {
    __syncthreads();  // the run before this one has read s_red
    if ((t & 31) == 0) s_red[t >> 5] = amax;
    __syncthreads();  // (everybody has read the old scale)
#pragma unroll
    for (int w = 0; w < GROUP / 32; ++w) amax = fmaxf(amax, s_red[w]);
  } else {
    __syncwarp();
  }
  const float need = pow2_scale<CODE>(amax);
  const float now = first == 0 ? need : fmaxf(old, need);
  if (t == 0) *scale = now;
  if (first > 0 && now != old) {  // the block's scale has grown: its codes are written again
    const float ratio = __fdiv_rn(old, now);
#pragma unroll 1
    for (int r = my.row; r < first; r += my.step) {
      uint2* at = reinterpret_cast<uint2*>(dst + (int64_t)r * row_stride);
      uint2 w = *at;
      uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t l2, h2;
        decode4<CODE>(ww[e], l2, h2);
        const float2 f0 = __half22float2(*reinterpret_cast<__half2*>(&l2)), f1 = __half22float2(*reinterpret_cast<__half2*>(&h2));
        ww[e] = encode2<CODE>(__fmul_rn(f0.x, ratio), __fmul_rn(f0.y, ratio)) |
                (encode2<CODE>(__fmul_rn(f1.x, ratio), __fmul_rn(f1.y, ratio)) << 16);
      }
      *at = w;
    }
  }
  dst += (int64_t)first * row_stride;
  auto put = [&](int r, const uint4& x, auto by) {  // by(x): x / now, correctly rounded
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t half[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a, b;
      unpack_pair<T>(w[e], a, b);
      half[e] = encode2<CODE>(by(a), by(b));
    }
    *reinterpret_cast<uint2*>(dst + (int64_t)r * row_stride) = make_uint2(half[0] | (half[1] << 16), half[2] | (half[3] << 16));
  };
  const uint32_t bits = __float_as_uint(now), exponent = bits >> 23;
  if ((bits & 0x7fffffu) == 0 && exponent >= 1 && exponent <= 253) {  // a power of two: its reciprocal is exact
    const float inv = __uint_as_float((254u - exponent) << 23);
    auto by = [&](float v) { return __fmul_rn(v, inv); };
    auto all = [&](auto one) {
      for (int r0 = my.row;;) {
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
          if (r0 + k * my.step < rows) one(r0 + k * my.step, keep[k]);
        r0 += more;
        if (r0 >= rows) break;
        fetch(r0);
      }
    };
    // Two fp16 elements at a time, where none is special and the reciprocal is a normal fp16: the product is exact (or so small that its code
    // is 0 either way).  x / now + 1536 is rounded to a whole number, whose low byte is the code.  7300 tokens of seven prompts, 8 heads of
    // 128, int8: 17.3 us one element after the other, 19 instructions each, 15.6 with this and the prefetch.
    if (BATCH > 1 && std::is_same<T, __half>::value && finite && exponent >= 112 && exponent <= 141) {
      const uint32_t inv2 = pack2<__half>(inv, inv);
      all([&](int r, const uint4& x) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        uint32_t c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (CODE == FA_CODE_E4M3) {
            uint32_t y;
            uint16_t z;
            asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(y) : "r"(w[e]), "r"(inv2));
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;\n" : "=h"(z) : "r"(y));
            c[e] = z;
          } else {
            asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(c[e]) : "r"(w[e]), "r"(inv2), "r"(0x66006600u));
          }
        }
        constexpr uint32_t sel = CODE == FA_CODE_E4M3 ? 0x5410 : 0x6420;
        *reinterpret_cast<uint2*>(dst + (int64_t)r * row_stride) = make_uint2(__byte_perm(c[0], c[1], sel), __byte_perm(c[2], c[3], sel));
      });
    } else {
      all([&](int r, const uint4& x) { put(r, x, by); });
    }
  } else {  // a scale that somebody else has chosen: rare, and kept short
#pragma unroll 1
    for (int r = my.row; r < rows; r += my.step) put(r, load(r), [&](float v) { return __fdiv_rn(v, now); });
  }
}

// ---- packed tokens with a slot each ----
// grid (windows of tokens, groups of (kv head, K or V) pairs).  A CTA lists the runs that start in its window and writes them for
// its pairs: short ones a warp each, side by side, then the long ones together.
constexpr int kMaxWindow = 256;

template <typename T, int CODE>
__global__ void __launch_bounds__(kAppendThreads, 4) kv8_append_kernel(const __grid_constant__ fa_kv8_append_params p, int window, int32_t* status) {
  __shared__ float s_red[kAppendWarps];
  __shared__ int s_runs, s_tok[kMaxWindow], s_len[kMaxWindow];
  __shared__ uint32_t s_slot[kMaxWindow];
  grid_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t t0 = (int64_t)blockIdx.x * window;
  const uint32_t sb = (uint32_t)p.c.scale_block, blocks = (uint32_t)p.rows / sb;
  const int64_t slots = (int64_t)p.kv_outer * p.rows;  // below 2^31
  if (tid == 0) s_runs = 0;
  // The window's elements are wanted whatever its slots say: on their way to L2 while those are looked up.
  const int pairs = 2 * p.h_k;
  const int mine = (pairs - blockIdx.y + gridDim.y - 1) / gridDim.y;  // every gridDim.y-th pair
  if (window > 1 && mine > 1) {
    const int lines = ceil_div(p.d, 64), here = (int)min((int64_t)window, p.total - t0);
    for (int i = tid; i < here * mine * lines; i += kAppendThreads) {
      const int line = i % lines, m = i / lines % mine, tok = i / lines / mine, pair = blockIdx.y + m * gridDim.y;
      const bool is_v = pair & 1;
      const T* x = reinterpret_cast<const T*>(is_v ? p.v : p.k) + (int64_t)(pair >> 1) * (is_v ? p.v_head_stride : p.k_head_stride) +
                   (t0 + tok) * (is_v ? p.v_tok_stride : p.k_tok_stride) + line * 64;
      asm volatile("prefetch.global.L2 [%0];\n" ::"l"(x));
    }
  }
  __syncthreads();
  if (tid < window && t0 + tid < p.total) {
    const int64_t s = p.slots[t0 + tid], before = t0 + tid > 0 ? p.slots[t0 + tid - 1] : -1;
    if (s >= slots) raise_bad_index(status);  // nowhere to write: skipped, like padding
    if (s >= 0 && s < slots && (before != s - 1 || (uint32_t)s % sb == 0)) {  // a run starts
      const int r = atomicAdd(&s_runs, 1);  // (in any order: runs do not know of one another)
      s_tok[r] = tid;
      s_slot[r] = (uint32_t)s;
    }
  }
  __syncthreads();
  const int runs = s_runs;
  for (int r = warp; r < runs; r += kAppendWarps) {  // it goes on while the slots follow one another within the block
    const int64_t t = t0 + s_tok[r], s = s_slot[r];
    const int most = (int)min((int64_t)(sb - (uint32_t)s % sb), p.total - t);
    int len = 0, more = 0;
    do {
      bool on[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = len + 32 * k + lane;
        on[k] = i < most && p.slots[t + i] == s + i;
      }
      more = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned off = ~__ballot_sync(0xffffffffu, on[k]);
        if (more == 32 * k) more += off ? __ffs(off) - 1 : 32;
      }
      len += more;
    } while (more == 128);
    if (lane == 0) s_len[r] = len;
  }
  __syncthreads();
  const int chunks = p.d >> 3;
  const Share alone(lane, 32, chunks), together(tid, kAppendThreads, chunks);
  auto run = [&](auto group, auto batch, int r, int pair, int t) {
    const int hk = pair >> 1;
    const bool is_v = pair & 1;
    const uint32_t s = s_slot[r], blk = s / sb, outer = blk / blocks, in = blk - outer * blocks;
    const int64_t tok = is_v ? p.v_tok_stride : p.k_tok_stride, row_stride = is_v ? p.vc_row_stride : p.kc_row_stride;
    const T* x = reinterpret_cast<const T*>(is_v ? p.v : p.k) + (int64_t)hk * (is_v ? p.v_head_stride : p.k_head_stride) + (t0 + s_tok[r]) * tok;
    uint8_t* codes = reinterpret_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + (int64_t)hk * (is_v ? p.vc_head_stride : p.kc_head_stride) +
                     outer * (is_v ? p.vc_outer_stride : p.kc_outer_stride) + (int64_t)(in * sb) * row_stride;
    float* scale = is_v ? p.c.v_scale + hk * p.c.vs_head_stride + outer * p.c.vs_outer_stride + in * p.c.vs_block_stride
                        : p.c.k_scale + hk * p.c.ks_head_stride + outer * p.c.ks_outer_stride + in * p.c.ks_block_stride;
    const Share& my = decltype(group)::value == 32 ? alone : together;
    x += my.col * 8;
    auto load = [&](int row) { return *reinterpret_cast<const uint4*>(x + (int64_t)row * tok); };
    write_run<T, CODE, decltype(group)::value, decltype(batch)::value>(load, codes + my.col * 8, row_stride, (int)(s % sb), s_len[r], my, scale, t, s_red);
  };
  using std::integral_constant;
  for (int i = warp; i < runs * mine; i += kAppendWarps) {
    const int m = i / runs, r = i - m * runs, pair = blockIdx.y + m * gridDim.y, n = s_len[r] * chunks;
    if (n <= 32) run(integral_constant<int, 32>(), integral_constant<int, 1>(), r, pair, lane);
    else if (n <= kWarpRun) run(integral_constant<int, 32>(), integral_constant<int, kBatch>(), r, pair, lane);
  }
  for (int r = 0; r < runs; ++r) {
    if (s_len[r] * chunks <= kWarpRun) continue;
    for (int pair = blockIdx.y; pair < pairs; pair += gridDim.y)
      run(integral_constant<int, kAppendThreads>(), integral_constant<int, kBatch>(), r, pair, tid);
  }
}

// ---- new tokens of an attention call: (b, s_new, h_k, d) behind cache_seqlens, k rotated when rotary tables are given ----
// Units (touched block of a sequence, kv head, K or V), GROUP threads each; BATCH as above.
template <typename T, int CODE, int GROUP, int BATCH>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_dense_kernel(const __grid_constant__ Kv8Params p, int touched, int units) {
  __shared__ float s_red[kAppendWarps];
  grid_wait();
  const int tid = threadIdx.x;
  const int unit = GROUP == 32 ? blockIdx.x * kAppendWarps + (tid >> 5) : blockIdx.x;
  if (unit >= units) return;
  const int pairs = 2 * p.a.h_k, seq = unit / pairs, pair = unit - seq * pairs, hk = pair >> 1;
  const int bi = seq / touched, nth = seq - bi * touched;
  const bool is_v = pair & 1;
  const int len = cache_len(p.a, bi, p.status), sb = p.c.scale_block;
  const int blk = len / sb + nth;  // of the sequence
  const int lo = max(len, blk * sb), hi = min(len + p.a.seqlen_new, (blk + 1) * sb);
  if (hi <= lo) return;
  int row = blk * sb, outer = bi;
  if (p.a.block_table) {
    const int pg = row / p.a.page_size;
    row -= pg * p.a.page_size;
    outer = p.a.block_table[(int64_t)bi * p.a.block_table_batch_stride + pg];
    // a page that is not there gets nothing: clamping would write into somebody else's
    if ((unsigned)outer >= (unsigned)p.a.kv_outer) {
      raise_bad_index(p.status);
      return;
    }
  } else if (p.a.cache_batch_idx) {
    outer = p.a.cache_batch_idx[bi];
    if ((unsigned)outer >= (unsigned)p.a.kv_outer) {
      raise_bad_index(p.status);
      return;
    }
  }
  const T* x = is_v ? reinterpret_cast<const T*>(p.a.v_new) + (int64_t)bi * p.a.vnew_batch_stride + (int64_t)hk * p.a.vnew_head_stride
                    : reinterpret_cast<const T*>(p.a.k_new) + (int64_t)bi * p.a.knew_batch_stride + (int64_t)hk * p.a.knew_head_stride;
  const int64_t tok = is_v ? p.a.vnew_row_stride : p.a.knew_row_stride, row_stride = is_v ? p.a.v_row_stride : p.a.k_row_stride;
  uint8_t* codes = const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(is_v ? p.a.v : p.a.k)) +
                   (int64_t)outer * (is_v ? p.a.v_batch_stride : p.a.k_batch_stride) + (int64_t)hk * (is_v ? p.a.v_head_stride : p.a.k_head_stride) +
                   (int64_t)row * row_stride;
  float* scale = is_v ? p.c.v_scale + outer * p.c.vs_outer_stride + (int64_t)(row / sb) * p.c.vs_block_stride + hk * p.c.vs_head_stride
                      : p.c.k_scale + outer * p.c.ks_outer_stride + (int64_t)(row / sb) * p.c.ks_block_stride + hk * p.c.ks_head_stride;
  const bool rotate = !is_v && p.a.rotary_cos != nullptr;
  const Share my(GROUP == 32 ? (tid & 31) : tid, GROUP, p.a.d >> 3);
  const int c = my.col;
  auto load = [&](int r) {
    const T* xr = x + (int64_t)(lo - len + r) * tok;
    uint4 v = *reinterpret_cast<const uint4*>(xr + c * 8);
    if (rotate) {
      const int pos = min(lo + r, p.a.rotary_seqlen - 1);
      const T* cosr = reinterpret_cast<const T*>(p.a.rotary_cos) + (int64_t)pos * (p.a.rotary_dim >> 1);
      const T* sinr = reinterpret_cast<const T*>(p.a.rotary_sin) + (int64_t)pos * (p.a.rotary_dim >> 1);
      v = rotary_chunk<T>(v, xr, c * 8, cosr, sinr, p.a.rotary_dim, p.a.rotary_interleaved != 0);
    }
    return v;
  };
  write_run<T, CODE, GROUP, BATCH>(load, codes + c * 8, row_stride, lo - blk * sb, hi - lo, my, scale, GROUP == 32 ? (tid & 31) : tid, s_red);
}

template <typename T, int CODE>
static cudaError_t append_t(const fa_kv8_append_params& p, int num_sm, int32_t* status, cudaStream_t st) {
  // A window has as many tokens as leave every SM eight CTAs, up to a scale block, in which one run of a prompt starts: one for a
  // decoding step, whose runs then lie side by side.  A CTA has eight pairs for warps that write alone and one for long runs; where runs may
  // be long but the tokens are few, as many (up to four) as bring the CTAs into one wave, since they may be a decoding batch as well as a
  // prompt (blocks of 128 tokens, 8 heads, one or as many pairs as the rule says: 64 requests 5.8 and 3.5 us, a prompt of 64 tokens 5.1
  // and 5.4; 128 requests 10.2 and 3.7, a prompt 7.3 and 9.2).
  const int pairs = 2 * p.h_k, sb = p.c.scale_block;
  const bool maybe_long = std::min<int64_t>(p.total, sb) * (p.d / 8) > kWarpRun;
  const int64_t waves = (p.total * pairs + 4LL * num_sm - 1) / (4LL * num_sm);
  const int each = !maybe_long ? kAppendWarps : waves > 4 ? 1 : (int)waves, groups = (pairs + each - 1) / each;
  const int most = std::min(kMaxWindow, sb);
  const int window = (int)std::min<int64_t>(most, std::max<int64_t>(1, p.total * groups / (8LL * num_sm)));
  const dim3 grid((unsigned)((p.total + window - 1) / window), (unsigned)groups);
  return launch_dependent(kv8_append_kernel<T, CODE>, grid, kAppendThreads, 0, st, p, window, status);
}
cudaError_t launch_kv8_append(const fa_kv8_append_params& p, int num_sm, int32_t* status, cudaStream_t st) {
  if (p.dtype == FA_BF16)
    return p.c.code == FA_CODE_E4M3 ? append_t<__nv_bfloat16, FA_CODE_E4M3>(p, num_sm, status, st)
                                    : append_t<__nv_bfloat16, FA_CODE_INT8>(p, num_sm, status, st);
  return p.c.code == FA_CODE_E4M3 ? append_t<__half, FA_CODE_E4M3>(p, num_sm, status, st) : append_t<__half, FA_CODE_INT8>(p, num_sm, status, st);
}

template <typename T, int CODE>
static cudaError_t append_dense_t(const Kv8Params& p, cudaStream_t st) {
  const int sb = p.c.scale_block, touched = (p.a.seqlen_new + sb - 2) / sb + 1, units = touched * p.a.b * 2 * p.a.h_k;
  const int n = std::min(sb, p.a.seqlen_new) * (p.a.d / 8);
  const dim3 one((unsigned)units), eight((unsigned)ceil_div(units, kAppendWarps));  // units a CTA
  if (n <= 32) return launch_dependent(kv8_append_dense_kernel<T, CODE, 32, 1>, eight, kAppendThreads, 0, st, p, touched, units);
  if (n <= kWarpRun) return launch_dependent(kv8_append_dense_kernel<T, CODE, 32, kBatch>, eight, kAppendThreads, 0, st, p, touched, units);
  return launch_dependent(kv8_append_dense_kernel<T, CODE, kAppendThreads, kBatch>, one, kAppendThreads, 0, st, p, touched, units);
}
cudaError_t launch_kv8_append_dense(const Kv8Params& p, cudaStream_t st) {
  if (p.a.dtype == FA_BF16)
    return p.c.code == FA_CODE_E4M3 ? append_dense_t<__nv_bfloat16, FA_CODE_E4M3>(p, st) : append_dense_t<__nv_bfloat16, FA_CODE_INT8>(p, st);
  return p.c.code == FA_CODE_E4M3 ? append_dense_t<__half, FA_CODE_E4M3>(p, st) : append_dense_t<__half, FA_CODE_INT8>(p, st);
}

}  // namespace fa
