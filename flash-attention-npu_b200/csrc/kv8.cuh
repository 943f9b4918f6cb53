// KV caches held in 8 bits: what their kernels share.
//
// A cache holds codes, one byte per element, and one fp32 scale for every (block of scale_block tokens, kv head) of K and of V;
// an element stands for code * scale.  Codes are e4m3 floating point or int8.  Every code is a value of fp16, so the matrix
// products run in fp16 on the codes themselves and the scales stay outside of them, in fp32.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "kv8_ranges.cuh"
#include "tc5_ptx.cuh"

namespace fa {

constexpr int kScaleGranule = 16;  // scale blocks are multiples of this: sixteen keys that start at a multiple have one scale

struct Kv8Params {
  fa_fwd_params a;  // k / v: codes, strides in elements = bytes
  fa_kv8_cache c;
  int32_t wl, wr, wl_on_device;  // normalised window; wl_on_device: the left rule is finished from the lengths on the device
  int32_t group;                 // query heads of a kv head: they share a tile, row = token * group + head
  int32_t m_blocks;              // row tiles of the longest sequence
  int32_t box_rows;              // rows of one TMA box: a page, or the part of it that fits a stage
  int32_t num_splits, blocks_per_split;
  int32_t persistent;  // resident CTAs share all key blocks equally; num_splits = partial slots of a unit
  float* o_partial;    // [split][lse_index][d] fp32
  float* lse_partial;  // [split][lse_index]
  int64_t lse_elems;
  int32_t* status;
};

// A scale of V as the kernels use it.  Scales are positive, or zero for blocks of zeros: zero, or too small to have a reciprocal, counts as 2^-64;
// NaN stays NaN.  (K's enter the scores as they are; the tile kernel looks for the maximum before it multiplies by them.)
__device__ __forceinline__ float usable_scale(float s) { return s < 0x1p-64f ? 0x1p-64f : s; }

// Four codes of a 32-bit word -> two fp16 pairs (bytes 0, 1 and bytes 2, 3); exact.
template <int CODE>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (CODE == FA_CODE_E4M3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // byte + 128 as the low mantissa bits of 1024: 1152 + code, then minus 1152
    const uint32_t u = w ^ 0x80808080u;
    asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(lo) : "r"(__byte_perm(u, 0x64646464u, 0x4140)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(hi) : "r"(__byte_perm(u, 0x64646464u, 0x4342)), "r"(0x64806480u));
  }
}

// What a kernel needs of a sequence.
struct Kv8Seq {
  int q_row0, q_len, k_len, koff;  // koff: key that query row 0's diagonal falls on
  int key_lo, key_hi;              // keys that some query row sees
  int batch_row;                   // contiguous cache
  const int32_t* pages;            // paged cache
};

// What the caller's tensors say of a sequence, cut to what there is; fine: nothing had to be cut, and its rows are no more than the caller's
// longest run, for which there are tiles.
struct Kv8Lens {
  int q_row0, q_len, k_len;
  bool fine;
};
__device__ __forceinline__ Kv8Lens kv8_lens(const Kv8Params& p, int bi) {
  int from = 0, upto = 0, held = 0;  // (all on their way before the first is looked at)
  if (p.a.cu_seqlens_q) from = p.a.cu_seqlens_q[bi], upto = p.a.cu_seqlens_q[bi + 1];
  if (p.a.seqused_k) held = p.a.seqused_k[bi];
  Kv8Lens n{0, p.a.seqlen_q, p.a.seqlen_k + p.a.seqlen_new, true};
  if (p.a.cu_seqlens_q) n.fine = kv8_query_rows(from, upto, p.a.total_q, n.q_row0, n.q_len) && n.q_len <= p.a.seqlen_q;
  if (p.a.seqused_k) {
    const int fits = min(max(held, 0), max(p.a.seqlen_k - p.a.seqlen_new, 0));
    n.fine &= fits == held;
    n.k_len = fits + p.a.seqlen_new;
  }
  return n;
}

// The left-window rule needs the longest sequence; warp-collective.
__device__ __forceinline__ Kv8Mask kv8_mask(const Kv8Params& p, int lane) {
  Kv8Mask m{p.wl, p.wr, false, false};
  if (p.wl_on_device) {
    int mx = 0;
    for (int i = lane; i < p.a.b; i += 32) mx = max(mx, kv8_lens(p, i).k_len);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (mx > 0 && m.wl >= mx - 1) m.wl = -1;
  }
  m.causal = m.wl < 0 && m.wr == 0;
  m.local = (m.wl >= 0 || m.wr >= 0) && !m.causal;
  return m;
}

// block_m: rows of a tile
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Params& p, const Kv8Mask& m, int bi, int mb, int block_m) {
  Kv8Seq s;
  const Kv8Lens n = kv8_lens(p, bi);
  if (!n.fine) raise_bad_index(p.status);  // (here alone: every sequence comes by)
  s.q_row0 = n.q_row0;
  s.q_len = n.q_len;
  s.k_len = n.k_len;
  s.koff = s.k_len - s.q_len;
  const int i_lo = mb * block_m / p.group, i_hi = min(s.q_len, (mb * block_m + block_m - 1) / p.group + 1) - 1;
  kv8_key_range(m, s.k_len, s.koff, i_lo, i_hi, s.key_lo, s.key_hi);
  s.pages = nullptr;
  s.batch_row = bi;
  if (p.a.block_table) s.pages = p.a.block_table + (int64_t)bi * p.a.block_table_batch_stride;
  else if (p.a.cache_batch_idx) s.batch_row = outer_index(p.a, p.a.cache_batch_idx[bi], p.status);
  return s;
}

// ---- the work list of a CTA ----
// A unit is a row tile of one (sequence, kv head).  One unit (or one of its key splits) per CTA, or resident CTAs with equal
// shares of all units' key blocks: gridDim.x / h_k CTAs a kv head, head fastest, so that the heads of a token, which are neighbours in memory,
// are read at the same time (8 sequences of 131072 keys, 8 heads of 128 bytes, calls in a CUDA graph: 313 us, 402 with one unit after
// the other).  A head's units are
// laid end to end, each as its key blocks (one, fully masked, when it sees no key, so that its rows are written) behind OVH
// virtual blocks that stand for its fixed cost; CTA c of the head takes virtual blocks [c * quota, (c + 1) * quota).  A unit that
// CTA boundaries cut leaves one partial per CTA in consecutive slots.  Producer and consumer warps walk the list independently of one
// another.
struct Kv8Seg {
  int bi, hk, mb;
  int lo, cnt;          // key blocks [lo, lo + cnt)
  int slot, fill_from;  // partial slot; the unit's first CTA marks slots fill_from .. as empty
  int masked;           // the one block stands in for no visible key
  int valid;            // 0: no more work; 1: run; 2: nothing to run here, take the next
};

template <int BM, int BN, int OVH>
struct Kv8Walk {
  int bi, nb_lo, nb_hi, n_b, quota, cur, g1, ustart;

  __device__ __forceinline__ static void blocks(const Kv8Params& p, const Kv8Mask& m, int bi, int mb, int& nb_lo, int& nb_hi) {
    const Kv8Lens n = kv8_lens(p, bi);
    const int i_lo = mb * BM / p.group, i_hi = min(n.q_len, (mb * BM + BM - 1) / p.group + 1) - 1;
    int lo, hi;
    kv8_key_range(m, n.k_len, n.k_len - n.q_len, i_lo, i_hi, lo, hi);
    if (i_hi < i_lo) hi = lo;
    nb_lo = lo / BN;
    nb_hi = hi > lo ? ceil_div(hi, BN) : nb_lo;
  }

  __device__ __forceinline__ void next(const Kv8Params& p, const Kv8Mask& m, Kv8Seg& sg) {
    if (!p.persistent || cur >= g1 || bi >= p.a.b) {
      sg.valid = 0;
      return;
    }
    const int seg_lo = cur - ustart, seg_hi = min(n_b, g1 - ustart);
    const int lo = max(seg_lo - OVH, 0), hi = max(seg_hi - OVH, 0);
    const int first_cta = (ustart + OVH) / quota;  // the CTA (of this head's) that holds the first real block
    const bool first = lo == 0 && hi > 0;
    sg = Kv8Seg{bi, (int)blockIdx.x % p.a.h_k, 0, nb_lo + lo, hi - lo, (int)blockIdx.x / p.a.h_k - first_cta,
                first ? (ustart + n_b - 1) / quota - first_cta + 1 : p.num_splits, nb_hi <= nb_lo, hi > lo ? 1 : 2};
    cur = ustart + seg_hi;
    if (seg_hi == n_b) {
      ustart += n_b;
      if (++bi < p.a.b) {
        blocks(p, m, bi, 0, nb_lo, nb_hi);
        n_b = max(1, nb_hi - nb_lo) + OVH;
      }
    }
  }

  // warp-collective: the first segment of this CTA
  __device__ __forceinline__ void first(const Kv8Params& p, const Kv8Mask& m, int lane, Kv8Seg& sg) {
    const int nbat = p.a.b;
    bi = nb_lo = nb_hi = cur = g1 = ustart = 0;
    n_b = quota = 1;
    if (!p.persistent) {  // kv head fastest, then row tile, split, sequence
      int idx = blockIdx.x;
      const int h = idx % p.a.h_k;
      idx /= p.a.h_k;
      const int mb = p.m_blocks - 1 - idx % p.m_blocks;  // the last rows see most keys
      idx /= p.m_blocks;
      const int split = idx % p.num_splits, b = idx / p.num_splits;
      int lo, hi;
      blocks(p, m, b, mb, lo, hi);
      if (p.num_splits > 1) {
        lo += split * p.blocks_per_split;
        hi = min(hi, lo + p.blocks_per_split);
      }
      sg = Kv8Seg{b, h, mb, lo, max(0, hi - lo), split, p.num_splits, 0, 1};
      return;
    }
    int total = 0, n_max = 1;
    for (int b0 = 0; b0 < nbat; b0 += 32) {
      int n = 0;
      if (b0 + lane < nbat) {
        int lo, hi;
        blocks(p, m, b0 + lane, 0, lo, hi);
        n = max(1, hi - lo) + OVH;
      }
      int mx = n, sm = n;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        sm += __shfl_xor_sync(0xffffffffu, sm, o);
      }
      n_max = max(n_max, mx);
      total += sm;
    }
    quota = max(ceil_div(total, (int)gridDim.x / p.a.h_k), ceil_div(n_max - OVH, p.num_splits - 1));
    cur = (int)blockIdx.x / p.a.h_k * quota;
    g1 = min(total, cur + quota);
    bi = nbat;
    if (cur < g1) {
      for (int b0 = 0; b0 < nbat && bi == nbat; b0 += 32) {
        int lo = 0, hi = 0, n = 0;
        if (b0 + lane < nbat) {
          blocks(p, m, b0 + lane, 0, lo, hi);
          n = max(1, hi - lo) + OVH;
        }
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, b0 + lane < nbat && ustart + incl > cur);
        if (hit) {
          const int src = __ffs(hit) - 1;
          bi = b0 + src;
          ustart += __shfl_sync(0xffffffffu, incl - n, src);
          nb_lo = __shfl_sync(0xffffffffu, lo, src);
          nb_hi = __shfl_sync(0xffffffffu, hi, src);
          n_b = __shfl_sync(0xffffffffu, n, src);
        } else {
          ustart += __shfl_sync(0xffffffffu, incl, 31);
        }
      }
    }
    next(p, m, sg);
  }
};

// One row's query chunk of 8 elements, rotated when rotary tables are given.
template <typename T>
__device__ __forceinline__ uint4 kv8_q_chunk(const Kv8Params& p, const T* qrow, int c8, int k_len, int i, bool rot_per_token) {
  uint4 q4 = *reinterpret_cast<const uint4*>(qrow + c8);
  if (p.a.rotary_cos) {
    const int pos = min(k_len - p.a.seqlen_new + (rot_per_token ? i : 0), p.a.rotary_seqlen - 1);
    const T* cosr = reinterpret_cast<const T*>(p.a.rotary_cos) + (int64_t)pos * (p.a.rotary_dim >> 1);
    const T* sinr = reinterpret_cast<const T*>(p.a.rotary_sin) + (int64_t)pos * (p.a.rotary_dim >> 1);
    q4 = rotary_chunk<T>(q4, qrow, c8, cosr, sinr, p.a.rotary_dim, p.a.rotary_interleaved != 0);
  }
  return q4;
}

// fp16 queries take part as they are.  bf16 queries become fp16 times a power of two of their row, the one that brings the row's
// largest element to [2^14, 2^15): exact for every element above 2^-31 of that, and at most 2^-39 of it off below.  Returns the factor that takes the
// products back; `amax_bits`: the row's largest |element| as a bf16 bit pattern.
__device__ __forceinline__ float bf16_row_factor(uint32_t amax_bits, float& up) {
  int e = (int)(amax_bits >> 7);  // biased exponent
  if (e == 255 || e == 0) e = 127 + 14;  // infinities and NaN stay what they are; an empty row has nothing to bring up
  e = max(e, 127 - 98);
  up = __int_as_float((127 + (127 + 14 - e)) << 23);
  return __int_as_float((127 - (127 + 14 - e)) << 23);
}

}  // namespace fa
