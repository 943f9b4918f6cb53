// New keys and values -> codes and scales of an 8-bit KV cache.
//
// The scale of a (token block, kv head) is the smallest power of two, 2^-40 at least, that brings the largest finite element
// into the codes' range (448 for e4m3, 127 for int8).  A power of two costs nothing in e4m3 (a floating-point code keeps its
// relative precision) and makes dividing by it, and expressing held codes in a larger one, exact up to the one rounding to a
// code.  A run is the new tokens that fall into one block: if rows are there in front of it, the block keeps its scale where that is larger,
// and otherwise its codes are rewritten in the new one; a run that starts at the block's first row starts the block afresh, so a
// recycled page needs no clearing.  Rows behind the run are left alone.  Runs own their blocks: no atomics, no order to depend on.
//
// HBM-bound: 2 bytes an element in, 1 out.  A run's elements stay in registers between the maximum and the rounding (up to
// kKeep 16-byte chunks a thread, the rest is read again), so everything is read once.
#include <type_traits>

#include "kv8.cuh"

namespace fa {

constexpr int kLeastScaleExp = 127 - 40;
constexpr int kAppendThreads = 256;

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

// x / s, correctly rounded: by the reciprocal where that is exact.
struct Divide {
  float s, inv;
  bool pow2;
  __device__ __forceinline__ explicit Divide(float scale) : s(scale) {
    const uint32_t u = __float_as_uint(scale);
    pow2 = (u & 0x7fffffu) == 0 && (u >> 23) >= 1 && (u >> 23) <= 253;
    inv = pow2 ? __uint_as_float((254u - (u >> 23)) << 23) : 0.f;
  }
  __device__ __forceinline__ float operator()(float x) const { return pow2 ? __fmul_rn(x, inv) : __fdiv_rn(x, s); }
};

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
// Largest |element| bits of a pair among the finite ones, per half word.
template <typename T>
__device__ __forceinline__ uint32_t finite_abs2(uint32_t w) {
  constexpr uint32_t inf = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u;
  const uint32_t a = w & 0x7fff7fffu;
  return a & __vcmpltu2(a, inf);
}

// One run: `rows` tokens of `chunks` 16-byte chunks each into block rows first .. first + rows - 1.  GROUP threads work together
// (a warp, or the whole CTA); `load(row, chunk)` gives a chunk of the source.
template <typename T, int CODE, int GROUP, typename Load>
__device__ __forceinline__ void write_run(Load load, uint8_t* block, int64_t row_stride, int first, int rows, int chunks, float* scale,
                                          int t, float* s_red) {
  constexpr int kKeep = 8;
  const int n = rows * chunks;
  uint4 keep[kKeep];
  uint32_t mx = 0;
#pragma unroll
  for (int k = 0; k < kKeep; ++k) {
    const int c = t + k * GROUP;
    keep[k] = make_uint4(0, 0, 0, 0);
    if (c < n) keep[k] = load(c / chunks, c % chunks);
  }
#pragma unroll
  for (int k = 0; k < kKeep; ++k)
    mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(finite_abs2<T>(keep[k].x), finite_abs2<T>(keep[k].y)),
                               __vmaxu2(finite_abs2<T>(keep[k].z), finite_abs2<T>(keep[k].w))));
  for (int c = t + kKeep * GROUP; c < n; c += GROUP) {
    const uint4 x = load(c / chunks, c % chunks);
    mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(finite_abs2<T>(x.x), finite_abs2<T>(x.y)), __vmaxu2(finite_abs2<T>(x.z), finite_abs2<T>(x.w))));
  }
  float lo, hi;
  unpack_pair<T>(mx, lo, hi);
  float amax = fmaxf(lo, hi);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (GROUP > 32) {
    __syncthreads();  // the run before this one has read s_red and the scale
    if ((t & 31) == 0) s_red[t >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < GROUP / 32; ++w) amax = fmaxf(amax, s_red[w]);
  }
  const float need = pow2_scale<CODE>(amax), old = *scale;
  const float now = first == 0 ? need : fmaxf(old, need);
  if (GROUP > 32) __syncthreads();
  else __syncwarp();
  if (t == 0) *scale = now;
  if (first > 0 && now != old) {  // the block's scale has grown: its codes are written again
    const float ratio = __fdiv_rn(old, now);
    const int held = first * chunks;
    for (int c = t; c < held; c += GROUP) {
      uint2* at = reinterpret_cast<uint2*>(block + (int64_t)(c / chunks) * row_stride + (c % chunks) * 8);
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
  const Divide by(now);
  auto store = [&](int c, const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t half[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a, b;
      unpack_pair<T>(w[e], a, b);
      half[e] = encode2<CODE>(by(a), by(b));
    }
    *reinterpret_cast<uint2*>(block + (int64_t)(first + c / chunks) * row_stride + (c % chunks) * 8) =
        make_uint2(half[0] | (half[1] << 16), half[2] | (half[3] << 16));
  };
#pragma unroll
  for (int k = 0; k < kKeep; ++k)
    if (t + k * GROUP < n) store(t + k * GROUP, keep[k]);
  for (int c = t + kKeep * GROUP; c < n; c += GROUP) store(c, load(c / chunks, c % chunks));
}

// ---- packed tokens with a slot each ----
// grid (token windows, kv heads, 2: K or V).  A CTA writes the runs that start in its window: those of up to kShortRun tokens a
// warp each (a decoding step's tokens are runs of one), longer ones together.
constexpr int kShortRun = 8, kMaxWindow = 32;

template <typename T, int CODE>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const __grid_constant__ fa_kv8_append_params p, int window, int32_t* status) {
  __shared__ float s_red[kAppendThreads / 32];
  __shared__ int s_first[kMaxWindow], s_len[kMaxWindow];
  __shared__ int64_t s_block[kMaxWindow];
  grid_wait();
  const int tid = threadIdx.x, hk = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const int64_t t0 = (int64_t)blockIdx.x * window;
  const int sb = p.c.scale_block, chunks = p.d >> 3;
  const int64_t slots = (int64_t)p.kv_outer * p.rows;
  if (tid < window) {
    const int64_t t = t0 + tid;
    int len = 0;
    int64_t blk = -1;
    int row = 0;
    if (t < p.total) {
      const int64_t s = p.slots[t];
      if (s >= slots) raise_bad_index(status);  // nowhere to write: skipped, like padding
      if (s >= 0 && s < slots) {
        blk = s / sb;
        row = (int)(s - blk * sb);
        // a run goes on while the slots follow one another within the block
        const int64_t before = t > 0 ? p.slots[t - 1] : -1;
        len = row == 0 || before != s - 1;
      }
    }
    s_first[tid] = row;
    s_len[tid] = len;
    s_block[tid] = blk;
  }
  __syncthreads();
  for (int w = tid >> 5; w < window; w += kAppendThreads / 32) {  // lengths of the runs that start here, 32 tokens at a time
    if (s_len[w] == 0) continue;
    const int64_t t = t0 + w, s = s_block[w] * sb + s_first[w];
    const int most = (int)min((int64_t)(sb - s_first[w]), p.total - t), lane = tid & 31;
    int len = 0;
    for (;;) {
      const int i = len + lane;
      const unsigned off = __ballot_sync(0xffffffffu, i >= most || p.slots[t + i] != s + i);
      if (off) {
        len += __ffs(off) - 1;
        break;
      }
      len += 32;
    }
    __syncwarp();
    if (lane == 0) s_len[w] = len;
  }
  __syncthreads();
  const T* src = reinterpret_cast<const T*>(is_v ? p.v : p.k) + (int64_t)hk * (is_v ? p.v_head_stride : p.k_head_stride);
  const int64_t tok_stride = is_v ? p.v_tok_stride : p.k_tok_stride;
  uint8_t* codes = reinterpret_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + (int64_t)hk * (is_v ? p.vc_head_stride : p.kc_head_stride);
  const int64_t outer_stride = is_v ? p.vc_outer_stride : p.kc_outer_stride, row_stride = is_v ? p.vc_row_stride : p.kc_row_stride;
  float* scale = (is_v ? p.c.v_scale : p.c.k_scale) + (int64_t)hk * (is_v ? p.c.vs_head_stride : p.c.ks_head_stride);
  const int64_t so = is_v ? p.c.vs_outer_stride : p.c.ks_outer_stride, sbs = is_v ? p.c.vs_block_stride : p.c.ks_block_stride;
  const int blocks = p.rows / sb;
  auto run = [&](auto group, int w, int t) {
    constexpr int GROUP = decltype(group)::value;
    const int64_t blk = s_block[w], outer = blk / blocks;
    const int in = (int)(blk - outer * blocks);
    const T* x = src + (t0 + w) * tok_stride;
    auto load = [&](int r, int c) { return *reinterpret_cast<const uint4*>(x + (int64_t)r * tok_stride + c * 8); };
    write_run<T, CODE, GROUP>(load, codes + outer * outer_stride + (int64_t)in * sb * row_stride, row_stride, s_first[w], s_len[w], chunks,
                              scale + outer * so + (int64_t)in * sbs, t, s_red);
  };
  for (int w = tid >> 5; w < window; w += kAppendThreads / 32)
    if (s_len[w] > 0 && s_len[w] <= kShortRun) run(std::integral_constant<int, 32>(), w, tid & 31);
  for (int w = 0; w < window; ++w)
    if (s_len[w] > kShortRun) run(std::integral_constant<int, kAppendThreads>(), w, tid);
}

// ---- new tokens of an attention call: (b, s_new, h_k, d) behind cache_seqlens, k rotated when rotary tables are given ----
// grid (blocks that a sequence can touch x b, kv heads, 2).
template <typename T, int CODE, int GROUP>
__global__ void __launch_bounds__(GROUP) kv8_append_dense_kernel(const __grid_constant__ Kv8Params p, int touched) {
  __shared__ float s_red[GROUP / 32];
  grid_wait();
  const int bi = blockIdx.x / touched, nth = blockIdx.x - bi * touched, hk = blockIdx.y, tid = threadIdx.x;
  const bool is_v = blockIdx.z != 0;
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
  auto load = [&](int r, int c) {
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
  write_run<T, CODE, GROUP>(load, codes, row_stride, lo - blk * sb, hi - lo, p.a.d >> 3, scale, tid, s_red);
}

template <typename T, int CODE>
static cudaError_t append_t(const fa_kv8_append_params& p, int num_sm, int32_t* status, cudaStream_t st) {
  // Windows of as many tokens as leave every SM eight CTAs: a window of one token finds a decoding step's runs side by side, a
  // longer one spares the CTAs in which no run of a prompt starts.
  int64_t w = p.total * p.h_k * 2 / (8LL * num_sm);
  const int window = (int)(w < 1 ? 1 : w > kMaxWindow ? kMaxWindow : w);
  const dim3 grid((unsigned)((p.total + window - 1) / window), (unsigned)p.h_k, 2);
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
  const int sb = p.c.scale_block, touched = (p.a.seqlen_new + sb - 2) / sb + 1;
  const dim3 grid((unsigned)(touched * p.a.b), (unsigned)p.a.h_k, 2);
  if (p.a.seqlen_new <= kShortRun) return launch_dependent(kv8_append_dense_kernel<T, CODE, 32>, grid, 32, 0, st, p, touched);
  return launch_dependent(kv8_append_dense_kernel<T, CODE, kAppendThreads>, grid, kAppendThreads, 0, st, p, touched);
}
cudaError_t launch_kv8_append_dense(const Kv8Params& p, cudaStream_t st) {
  if (p.a.dtype == FA_BF16)
    return p.c.code == FA_CODE_E4M3 ? append_dense_t<__nv_bfloat16, FA_CODE_E4M3>(p, st) : append_dense_t<__nv_bfloat16, FA_CODE_INT8>(p, st);
  return p.c.code == FA_CODE_E4M3 ? append_dense_t<__half, FA_CODE_E4M3>(p, st) : append_dense_t<__half, FA_CODE_INT8>(p, st);
}

}  // namespace fa
