// Attention over an 8-bit KV cache for many query rows: tcgen05 products with accumulators in TMEM, fp16 operands.
//
// A CTA has a tile of packed query rows (row = token * group + head; all heads of a kv head's group, so a key is turned into fp16
// once for all of them) against a range of key blocks.  Tiles that are few share the key blocks of the whole launch out equally
// among resident CTAs, as the decode kernel does (Kv8Walk).
// Arithmetic as in kv8_decode_kernel.cuh: V's scale in the exponent, P' in fp16, scales never in a product.  The reference m of
// the exponent is the running maximum, moved only when that has grown by more than 2^8: P' = 2^(x - m + 7) stays below 2^15, far from
// fp16's end, and below 2^7 it has as many bits as a 16-bit output shows (subnormals: off by 2^-32 of the largest at most); so O is rescaled in TMEM a few times a tile and
// not at every block.
//
// Warps: 4 per sub-tile  softmax, one thread per row (P, rescale of O, epilogue); each loads its rows of Q
//        4               converters: two turn K's codes into fp16 tiles in the swizzled operand layout, two V's
//        1 per sub-tile  MMA issue
//        1               scout: pages and scales, some blocks ahead (and one or two warps fill up the warpgroup)
// Two sub-tiles of 128 rows against the same keys, or (DUAL: no more than 128 rows) the same rows against even and odd key blocks, merged
// in the epilogue: with one chain of score, softmax and product a CTA of 128 rows idles between its steps (two such CTAs an SM: 55 us for
// drafts of 3 - 16 tokens, 8 heads a group, over 3001 - 20000 keys; DUAL 43.5).  256 columns: one sub-tile, O fills TMEM.
// Blocks of 64 keys, two S buffers per sub-tile: S of block j + 1 is there when the softmax of block j ends, so its threads wait for no
// product.  A thread keeps its 64 scores in registers, and P' goes back into the columns it read, as the TMEM operand of P.V: no
// shared-memory traffic and no proxy fence for P.  S of block j + 2 lands on P of block j; the same thread issues both products, in
// this order.  TMEM: per sub-tile S 2 x 64, O 128 columns.
// TMA cannot convert, so the codes pass through registers: copied ahead into shared memory as they are, read back by the thread that asked
// for them, turned and stored again.
//
// Bound: four chunks of 301 - 2048 tokens against 1777 - 8192 keys, 32 / 8 heads of 128: 490 us in a CUDA graph, 870 TFLOP/s of what the masks leave.  Per 64
// keys and 256 rows a CTA takes 2400 cycles; the products take 1024 of them on the tensor pipe, the exponentials 1024 on the special-function
// unit, shared memory is busy for 750.  What is left is the chain of one softmax warp (poll, TMEM load, maximum, exponentials, TMEM store,
// fence) with two such warps a scheduler, as many as registers allow: without any exponential it still takes 1950.  Tried against 485 us
// and without gain: a quarter of the exponentials as polynomials (485), a look at the next block's barriers ahead of time (515 - 535), blocks of 128 keys
// with P through shared memory (636).
#pragma once

#include <type_traits>

#include "kv8.cuh"

namespace fa {

template <int HD_, int NSUB_, bool DUAL_>
struct Kv8TileTraits {
  static constexpr int HD = HD_, NSUB = NSUB_;  // sub-tiles: 128 rows each, or (DUAL) the same 128 rows against even and odd key blocks
  static constexpr bool DUAL = DUAL_;
  static_assert(NSUB == 1 || HD <= 128, "256 columns of O and two S buffers leave TMEM room for one sub-tile");
  static_assert(!DUAL || NSUB == 2, "two streams");
  static constexpr int ROW_TILES = DUAL ? 1 : NSUB, BM = 128 * ROW_TILES, BN = 64;
  static constexpr int AHEAD = DUAL ? 4 : 2;  // blocks whose Q.K^T is issued before a block's P.V: two of each stream
  static constexpr int GROUPS = BN / kScaleGranule;
  static constexpr int HALVES = HD / 64;                 // 64-column halves of Q, K, V
  static constexpr int KV_HALF = BN * 128, SLOT_BYTES = HALVES * KV_HALF;
  static constexpr int Q_HALF = 128 * 128, Q_BYTES = HALVES * Q_HALF;  // per 128 rows
  static constexpr int RESIDENT = 1;
  static constexpr int RING = HD == 256 ? 3 : HD == 128 && !DUAL ? 6 : 8;
  // Codes on their way: FETCH parts of K's tiles and as many of V's, UNITS parts a tile.
  static constexpr int UNITS = HD == 256 ? 2 : 1, FETCH = HD == 64 ? 4 : HD == 128 ? 2 : 3;
  static constexpr int RING_OFF = ROW_TILES * Q_BYTES, CODE_OFF = RING_OFF + RING * SLOT_BYTES, CODE_BYTES = BN / UNITS * HD;
  static constexpr int SMEM_BYTES = 1024 + CODE_OFF + 2 * FETCH * CODE_BYTES;
  static_assert(SMEM_BYTES + 4400 <= 232448, "more than an SM has");
  static constexpr int SOFTMAX_WARPS = 4 * NSUB, CONV_WARPS = 4, NTHREADS = 32 * (SOFTMAX_WARPS + CONV_WARPS + 4);
  // Registers by warpgroup (setmaxnreg; one sub-tile of 256 columns has enough as it is): shares of the 128 a thread that a CTA is launched
  // with and never more.
  static constexpr bool SPLIT = NSUB == 2;
  static constexpr int SOFTMAX_REGS = 176, CONV_REGS = 80, ISSUE_REGS = 48;
  static_assert(!SPLIT || 2 * SOFTMAX_REGS + CONV_REGS + ISSUE_REGS <= 4 * 120, "more registers than a CTA is launched with");
  static constexpr int TMEM = 512, O_COL = 256, SUB_STEP = 128;  // columns: S of sub-tile t at t * SUB_STEP + buffer * BN, O at O_COL + t * SUB_STEP
  static constexpr int SCR = 8;   // blocks that the scout may be ahead
  static constexpr int OVH = 4;   // a unit's fixed cost in blocks (Kv8Walk)
  // Does sub-tile t work on block n of the CTA's, and as its how manieth?
  __device__ __forceinline__ static bool mine(int n, int t) { return !DUAL || (n & 1) == t; }
  __device__ __forceinline__ static int local(int n) { return DUAL ? n >> 1 : n; }
};

struct Kv8TileShared {
  uint64_t q_full[2], kv_full[8], kv_empty[8];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];  // [sub-tile][buffer]
  uint64_t sc_full[8], sc_empty[8];
  uint64_t other_done;  // DUAL: sub-tile 1's reference, sum and O of the segment are there
  float2 ml[128];       // ... the first two; before that, the factor of the row's query
  uint64_t half_way;    // sub-tile 0 is at its first exponentials
  float4 sc[8][3];      // of a block: score factor, log2 of V's scale, its reciprocal, per 16 keys
  int64_t at[8][2][4];  // ... and where K's and V's codes of 16 keys start, from the head's first; -1: zeros
  uint32_t tmem_base;
  int abort_flag;
};

// Bounded wait for two barriers at once: a poll takes some 160 cycles even where there is nothing to wait for.
__device__ __forceinline__ bool kv8_wait2(uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1, volatile int* abort_flag, int id) {
  for (uint32_t i = 0; i < tc5::kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
        "and.pred p, p, q;\n\tselp.b32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(b0), "r"(p0), "r"(b1), "r"(p1)
        : "memory");
    if (ok) return true;
    if ((i & 255u) == 255u && *abort_flag) return false;
  }
  if (*abort_flag == 0) *abort_flag = id;
  return false;
}

// Ring positions in the order the products need the tiles: K_0 .. K_(AHEAD-1) | V_0 K_AHEAD | V_1 ... | V_last.
__device__ __forceinline__ uint32_t kv8_ring_at(bool is_v, int it, int cnt, int ahead) {
  const int head = min(cnt, ahead);
  return is_v ? head + it + min(it, cnt - head) : it < head ? it : 2 * it - head + 1;
}
template <int SLOTS>
struct Kv8Ring {
  uint32_t at = 0, phase = 0;
  __device__ __forceinline__ void next(uint32_t& slot, uint32_t& par) {
    slot = at;
    par = phase;
    if (++at == SLOTS) { at = 0; phase ^= 1; }
  }
};

// ---------------- scout: where a block's keys are, and its scales ----------------
// One warp, up to SCR blocks ahead: pages and scales are two dependent loads that the converters need not wait for.  Four blocks are looked
// up at once, and the next four before these are handed over: one after the other, a block took the two loads' latency.
template <class Tr>
__device__ __forceinline__ bool kv8_scout(const Kv8Params& p, const Kv8Seq sq, const Kv8Seg sg, Kv8TileShared* sh, float mul, int base, int lane) {
  volatile int* abort_flag = &sh->abort_flag;
  constexpr int LANES = 2 * Tr::GROUPS, BATCH = 32 / LANES;  // of a block: K of its 16-key groups, then V of them
  const int sub = lane / LANES, grp = lane % Tr::GROUPS;
  const bool is_v = lane % LANES >= Tr::GROUPS;
  const float* scale = is_v ? p.c.v_scale + sg.hk * p.c.vs_head_stride : p.c.k_scale + sg.hk * p.c.ks_head_stride;
  const int64_t s_outer = is_v ? p.c.vs_outer_stride : p.c.ks_outer_stride, s_block = is_v ? p.c.vs_block_stride : p.c.ks_block_stride;
  const int64_t c_outer = is_v ? p.a.v_batch_stride : p.a.k_batch_stride, c_row = is_v ? p.a.v_row_stride : p.a.k_row_stride;
  auto look_up = [&](int it, int64_t& at, float& s) {
    const int t = (sg.lo + it) * Tr::BN + grp * kScaleGranule;
    at = -1;  // nothing there: zeros
    s = 0.f;
    if (it < sg.cnt && t < sq.key_hi && t + kScaleGranule > sq.key_lo) {  // some row sees a key of the group: its page is a live one
      int outer = sq.batch_row, row = t;
      bool there = true;
      if (sq.pages) {
        const int pg = t / p.a.page_size, id = __ldg(sq.pages + pg);
        row = t - pg * p.a.page_size;
        outer = outer_index(p.a, id, p.status);
        there = outer == id;
      }
      if (there) {
        at = outer * c_outer + row * c_row;
        s = __ldg(scale + outer * s_outer + (row / p.c.scale_block) * s_block);
      }
    }
  };
  int64_t at, at_next;
  float s, s_next;
  look_up(sub, at, s);
  for (int it0 = 0; it0 < sg.cnt; it0 += BATCH) {
    look_up(it0 + BATCH + sub, at_next, s_next);
    for (int k = 0; k < BATCH && it0 + k < sg.cnt; ++k) {
      const int n = base + it0 + k, e = n % Tr::SCR;
      if (n >= Tr::SCR && !tc5::mbar_wait(tc5::smem_addr(&sh->sc_empty[e]), (n / Tr::SCR - 1) & 1, abort_flag, 72)) return false;
      if (k == sub) {
        sh->at[e][is_v][grp] = at;
        if (!is_v) {
          reinterpret_cast<float*>(&sh->sc[e][0])[grp] = s * mul;
        } else {
          const float v = usable_scale(s);
          reinterpret_cast<float*>(&sh->sc[e][1])[grp] = log2f(v);
          reinterpret_cast<float*>(&sh->sc[e][2])[grp] = 1.f / v;
        }
      }
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(tc5::smem_addr(&sh->sc_full[e]));
    }
    at = at_next;
    s = s_next;
  }
  return true;
}

// ---------------- converters ----------------
// Two warps turn K's tiles, two V's.  A thread has the 16-code chunks of column tid % 4 in every 64-column half, of rows tid / 4 + 16 k (two
// rows of a quarter warp meet eight different banks); it copies the codes of FETCH tiles ahead into places of its own, so that nobody but
// itself waits for them.  (With the codes in registers instead, three tiles ahead, a block took 2700 cycles, mostly in loads that a
// warp's few scoreboards do not tell apart.)
template <class Tr, int CODE>
__device__ __forceinline__ bool kv8_convert(const Kv8Params& p, const Kv8Seq sq, const Kv8Seg sg, Kv8TileShared* sh, uint32_t smem, int first, int tid) {
  constexpr int GROUPS = Tr::GROUPS / Tr::UNITS;
  volatile int* abort_flag = &sh->abort_flag;
  const bool is_v = tid >= 64;
  const int lane = tid & 31, c4 = tid & 3, row0 = (tid & 63) >> 2;
  const uint8_t* base = (is_v ? reinterpret_cast<const uint8_t*>(p.a.v) + (int64_t)sg.hk * p.a.v_head_stride + row0 * p.a.v_row_stride
                              : reinterpret_cast<const uint8_t*>(p.a.k) + (int64_t)sg.hk * p.a.k_head_stride + row0 * p.a.k_row_stride) + c4 * 16;
  const int cols_left = p.a.d - c4 * 16;  // halves h with 64 h < cols_left hold columns of the head
  const uint32_t codes = smem + Tr::CODE_OFF + is_v * Tr::FETCH * Tr::CODE_BYTES + (tid & 63) * 16;
  const uint32_t tiles = smem + Tr::RING_OFF + row0 * 128, lo = ((c4 * 2) ^ (row0 & 7)) << 4, hi = ((c4 * 2 + 1) ^ (row0 & 7)) << 4;

  auto fetch = [&](int j) {
    const int it = j / Tr::UNITS, part = j % Tr::UNITS, n = first + it, e = n % Tr::SCR;
    if (it < sg.cnt) {
      const uint32_t to = codes + j % Tr::FETCH * Tr::CODE_BYTES;
      int64_t from[GROUPS];
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) from[k] = sh->at[e][is_v][part * GROUPS + k];
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) {
        const int64_t at = from[k];
        const int t = (sg.lo + it) * Tr::BN + (part * GROUPS + k) * kScaleGranule + row0;
        const bool on = at >= 0 && t >= sq.key_lo && t < sq.key_hi;
        const uint8_t* src = on ? base + at : reinterpret_cast<const uint8_t*>(p.a.k);
#pragma unroll
        for (int h = 0; h < Tr::HALVES; ++h) {  // zeros where nothing is
          const bool there = on && h * 64 < cols_left;
          cp_async_16(to + (k * Tr::HALVES + h) * 1024, there ? src + h * 64 : src, there);
        }
      }
      if (part == Tr::UNITS - 1) {
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(tc5::smem_addr(&sh->sc_empty[e]));
      }
    }
    cp_async_commit();
  };
  constexpr int TILES = (Tr::FETCH + Tr::UNITS - 1) / Tr::UNITS;  // (begun) tiles ahead
  for (int j = 0; j < Tr::FETCH; ++j) {
    const int n = first + j / Tr::UNITS;
    if (n < first + sg.cnt && !tc5::mbar_wait(tc5::smem_addr(&sh->sc_full[n % Tr::SCR]), (n / Tr::SCR) & 1, abort_flag, 70)) return false;
    fetch(j);
  }
  for (int it = 0; it < sg.cnt; ++it) {
    const uint32_t pos = 2 * first + kv8_ring_at(is_v, it, sg.cnt, Tr::AHEAD), slot = pos % Tr::RING;
    const uint32_t empty = tc5::smem_addr(&sh->kv_empty[slot]), empty_par = (pos / Tr::RING & 1) ^ 1;
    const int n = first + it + TILES;
    const bool more = it + TILES < sg.cnt;
    if (!kv8_wait2(empty, empty_par, more ? tc5::smem_addr(&sh->sc_full[n % Tr::SCR]) : empty, more ? (n / Tr::SCR) & 1 : empty_par, abort_flag, 71))
      return false;
#pragma unroll
    for (int part = 0; part < Tr::UNITS; ++part) {
      const int j = it * Tr::UNITS + part;
      cp_async_wait<Tr::FETCH - 1>();
      const uint32_t from = codes + j % Tr::FETCH * Tr::CODE_BYTES, tile = tiles + slot * Tr::SLOT_BYTES + part * GROUPS * (16 * 128);
      constexpr int NC = GROUPS * Tr::HALVES;
      uint32_t x[NC][4];
#pragma unroll
      for (int i = 0; i < NC; ++i)
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n"
                     : "=r"(x[i][0]), "=r"(x[i][1]), "=r"(x[i][2]), "=r"(x[i][3])
                     : "r"(from + i * 1024)
                     : "memory");
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const uint32_t at = tile + (i % Tr::HALVES) * Tr::KV_HALF + (i / Tr::HALVES) * (16 * 128);
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) decode4<CODE>(x[i][k], h[2 * k], h[2 * k + 1]);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(at + lo), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(at + hi), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
      }
      if (part == Tr::UNITS - 1) {
        tc5::fence_proxy_async();  // generic-proxy stores -> visible to the MMA
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(tc5::smem_addr(&sh->kv_full[slot]));
      }
      fetch(j + Tr::FETCH);
    }
  }
  return true;
}

// ---------------- MMA issue, sub-tile t ----------------
template <class Tr>
__device__ __forceinline__ bool kv8_issue(Kv8TileShared* sh, uint32_t smem, uint32_t tmem, Kv8Ring<Tr::RING>& ring, int first, int seg, int t, int cnt) {
  volatile int* abort_flag = &sh->abort_flag;
  constexpr uint32_t idesc_qk = tc5::make_idesc(0, 128, Tr::BN, 0), idesc_pv = tc5::make_idesc(0, 128, Tr::HD, 1);
  const uint64_t q_desc = tc5::make_smem_desc(smem + (Tr::DUAL ? 0 : t * Tr::Q_BYTES), 16, 1024);
  const uint64_t k_desc0 = tc5::make_smem_desc(smem + Tr::RING_OFF, 16, 1024);            // K-major
  const uint64_t v_desc0 = tc5::make_smem_desc(smem + Tr::RING_OFF, Tr::KV_HALF, 1024);   // N-contiguous
  constexpr uint64_t kSlot = Tr::SLOT_BYTES >> 4;
  // 16 columns per k-step = 32 bytes inside the 128-byte swizzle span
  auto off = [](int ks, int half) { return (uint64_t)(((ks >> 2) * half + (ks & 3) * 32) >> 4); };
  const uint32_t s_tmem0 = tmem + t * Tr::SUB_STEP, o_tmem = tmem + Tr::O_COL + t * Tr::SUB_STEP;
  if (!tc5::mbar_wait(tc5::smem_addr(&sh->q_full[Tr::DUAL ? 0 : t]), seg & 1, abort_flag, 73)) return false;
  // a ring slot is free when the products of every sub-tile that has rows have read it
  auto release = [&](uint32_t slot) { tc5::mma_commit(tc5::smem_addr(&sh->kv_empty[slot])); };
  // The buffer's last P has been read by the product of this thread in front of this one, its scores before that P was written.
  auto qk = [&](int it) {
    uint32_t slot, par;
    ring.next(slot, par);
    if (!Tr::mine(first + it, t)) return true;
    const int n = Tr::local(first + it);
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->kv_full[slot]), par, abort_flag, 74)) return false;
    tc5::tc_fence_after();
    const uint64_t k_desc = k_desc0 + slot * kSlot;
    const uint32_t s_tmem = s_tmem0 + (n & 1) * Tr::BN;
    if (tc5::elect_one()) {
      tc5::mma_ss_c<false>(s_tmem, q_desc, k_desc, idesc_qk);
#pragma unroll
      for (int ks = 1; ks < Tr::HD / 16; ++ks) tc5::mma_ss_c<true>(s_tmem, q_desc + off(ks, Tr::Q_HALF), k_desc + off(ks, Tr::KV_HALF), idesc_qk);
      tc5::mma_commit(tc5::smem_addr(&sh->s_full[t][n & 1]));
      release(slot);
    }
    __syncwarp();
    return true;
  };
  auto pv = [&](int it) {
    uint32_t slot, par;
    ring.next(slot, par);
    if (!Tr::mine(first + it, t)) return true;
    const int n = Tr::local(first + it);
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->kv_full[slot]), par, abort_flag, 76)) return false;
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->p_full[t][n & 1]), (n >> 1) & 1, abort_flag, 77)) return false;
    tc5::tc_fence_after();
    const uint64_t v_desc = v_desc0 + slot * kSlot;
    const uint32_t p_tmem = s_tmem0 + (n & 1) * Tr::BN;
    if (tc5::elect_one()) {
      if (it < (Tr::DUAL ? 2 : 1)) tc5::mma_ts_c<false>(o_tmem, p_tmem, v_desc, idesc_pv);
      else tc5::mma_ts_c<true>(o_tmem, p_tmem, v_desc, idesc_pv);
#pragma unroll
      for (int ks = 1; ks < Tr::BN / 16; ++ks) tc5::mma_ts_c<true>(o_tmem, p_tmem + ks * 8, v_desc + (uint64_t)(ks * (2048 >> 4)), idesc_pv);
      tc5::mma_commit(tc5::smem_addr(&sh->pv_done[t][n & 1]));
      release(slot);
    }
    __syncwarp();
    return true;
  };
  for (int it = 0; it < min(cnt, Tr::AHEAD); ++it)
    if (!qk(it)) return false;
  for (int it = 0; it < cnt; ++it)
    if (!pv(it) || (it + Tr::AHEAD < cnt && !qk(it + Tr::AHEAD))) return false;
  return true;
}

// ---------------- softmax, one thread per row ----------------
template <class Tr, typename T, bool CAP>
__device__ __forceinline__ bool kv8_softmax(const Kv8Params& p, const Kv8Mask& mask, const Kv8Seq& sq, const Kv8Seg& sg, Kv8TileShared* sh,
                                            uint32_t smem, uint32_t tmem, int first, int seg, int t, int lane_row) {
  volatile int* abort_flag = &sh->abort_flag;
  const int lane = lane_row & 31, warp = lane_row >> 5;
  const int rr = sg.mb * Tr::BM + (Tr::DUAL ? 0 : t * 128) + lane_row, rows_total = sq.q_len * p.group;
  const bool live = rr < rows_total;
  const int i = rr / p.group, head = sg.hk * p.group + (rr - i * p.group);
  // ---- Q: fp16, negated for a negative scale (scores then grow with the products), bf16 rows brought into fp16's range ----
  // A warp loads the rows of its threads, whole rows at a time (a thread with a row of its own: 12000 cycles for 256 rows of 256 bytes).
  float back = 1.f;
  if (sg.cnt > 0) {
    if (!Tr::DUAL || t == 0) {
      constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
      constexpr int LANES = Tr::HD / 8, ROWS = 32 / LANES;  // of a row; rows at a time
      const int ch = lane % LANES, sub = lane / LANES;
      const bool rot = mask.causal || mask.local;
      const float sign = p.a.softmax_scale < 0.f ? -1.f : 1.f;
      const T* qhead = reinterpret_cast<const T*>(p.a.q) + (int64_t)sg.bi * p.a.q_batch_stride + (int64_t)sg.hk * p.group * p.a.q_head_stride + ch * 8;
      const uint32_t q_smem = smem + (Tr::DUAL ? 0 : t * Tr::Q_BYTES) + (ch >> 3) * Tr::Q_HALF;
      const int rr0 = rr - lane, row0 = lane_row - lane;
#pragma unroll 1
      for (int k0 = 0; k0 < 32 / ROWS; k0 += 8) {
        uint4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int qr = rr0 + (k0 + k) * ROWS + sub, qi = qr / p.group;
          x[k] = make_uint4(0, 0, 0, 0);
          if (qr < rows_total && ch * 8 < p.a.d) {
            const T* q = qhead + (int64_t)(sq.q_row0 + qi) * p.a.q_row_stride + (int64_t)(qr - qi * p.group) * p.a.q_head_stride;
            x[k] = *reinterpret_cast<const uint4*>(q);
          }
        }
        if (p.a.rotary_cos) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int qr = rr0 + (k0 + k) * ROWS + sub, qi = qr / p.group;
            if (qr < rows_total && ch * 8 < p.a.d) {
              const T* q = qhead + (int64_t)(sq.q_row0 + qi) * p.a.q_row_stride + (int64_t)(qr - qi * p.group) * p.a.q_head_stride;
              x[k] = kv8_q_chunk<T>(p, q - ch * 8, ch * 8, sq.k_len, qi, rot);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
          if (BF) {
            uint32_t mx = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = max(mx, max(w[e] & 0x7fffu, w[e] >> 16 & 0x7fffu));
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            float up;
            const float down = bf16_row_factor(mx, up), mine = __shfl_sync(0xffffffffu, down, lane % ROWS * LANES);
            if (lane / ROWS == k0 + k) back = mine;
            up *= sign;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack2<__half>(__uint_as_float(w[e] << 16) * up, __uint_as_float(w[e] & 0xffff0000u) * up);
          } else if (sign < 0.f) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] ^= 0x80008000u;
          }
          const int row = row0 + (k0 + k) * ROWS + sub;
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(q_smem + row * 128 + (((ch & 7) ^ (row & 7)) << 4)), "r"(w[0]), "r"(w[1]),
                       "r"(w[2]), "r"(w[3])
                       : "memory");
        }
      }
      if (Tr::DUAL) sh->ml[lane_row].x = back;
      tc5::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(tc5::smem_addr(&sh->q_full[t]));
    } else {  // (behind it the segment before is through: sub-tile 0 has read what this one left of it)
      if (!tc5::mbar_wait(tc5::smem_addr(&sh->q_full[0]), seg & 1, abort_flag, 75)) return false;
      back = sh->ml[lane_row].x;
    }
  }
  // ---- what the row sees ----
  int row_lo = 0, row_hi = sq.k_len - 1;
  if (mask.causal) row_hi = min(row_hi, i + sq.koff);
  if (mask.local) {
    row_hi = min(row_hi, i + sq.koff + mask.wr);
    row_lo = max(0, i + sq.koff - mask.wl);
  }
  if (!live) row_hi = -1;
  // ... and every row of the warp: keys [all_lo, all_hi)
  const int all_lo = __reduce_max_sync(0xffffffffu, live ? row_lo : 0), all_hi = __reduce_min_sync(0xffffffffu, live ? row_hi + 1 : 0x7fffffff);
  const bool any_live = __any_sync(0xffffffffu, live);
  const float cap_l2 = p.a.softcap * kLog2e;
  const uint32_t lane_base = (uint32_t)warp << 21;  // 32 TMEM lanes a warp
  const uint32_t o_tmem = tmem + Tr::O_COL + t * Tr::SUB_STEP + lane_base;
  float m_ref = -INFINITY, l = 0.f;
  auto capped = [&](float z) { return cap_l2 * (1.f - __fdividef(2.f, __expf(2.f * z) + 1.f)); };  // z: score / cap

  const int cnt = sg.cnt, lo = sg.lo;
  // Sub-tile 1 starts half a block behind: one computes exponentials while the other loads scores and looks for the maximum, else both wait
  // for the special-function unit and then leave it idle, and stay in step to the end.
  bool start = Tr::NSUB == 2 && cnt > 0 && (Tr::DUAL || seg == 0);
  if (start && t == 1 && !tc5::mbar_wait(tc5::smem_addr(&sh->half_way), seg & 1, abort_flag, 83)) return false;
  auto pass = [&] {
    if (start && t == 0 && lane == 0) tc5::mbar_arrive(tc5::smem_addr(&sh->half_way));
    start = false;
  };
  for (int it = 0; it < cnt; ++it) {
    if (!Tr::mine(first + it, t)) continue;
    const int n = Tr::local(first + it), b = n & 1, e = (first + it) % Tr::SCR, t0 = (lo + it) * Tr::BN;
    const uint32_t s_tmem = tmem + t * Tr::SUB_STEP + b * Tr::BN + lane_base;
    // (P.V of two blocks before is over when S of this one is there.  Where this thread waits for the one of a block, the next on that
    // buffer cannot be over, so that a barrier is never two phases on.)
    if (!kv8_wait2(tc5::smem_addr(&sh->s_full[t][b]), (n >> 1) & 1, tc5::smem_addr(&sh->sc_full[e]), ((first + it) / Tr::SCR) & 1, abort_flag, 79))
      return false;
    tc5::tc_fence_after();
    uint32_t r[2][32];
    if (any_live) {  // (rows of the products do not mix: what a warp without rows leaves in P is its own)
      tc5::tmem_ld32(s_tmem, r[0]);
      tc5::tmem_ld32(s_tmem + 32, r[1]);
      const float4 f4 = sh->sc[e][0], l4 = sh->sc[e][1], i4 = sh->sc[e][2];
      const float c1[4] = {f4.x * back, f4.y * back, f4.z * back, f4.w * back}, lv[4] = {l4.x, l4.y, l4.z, l4.w}, inv[4] = {i4.x, i4.y, i4.z, i4.w};
      tc5::tmem_wait_ld();
      const bool edge = t0 < all_lo || t0 + Tr::BN > all_hi;
      if (edge) {  // some row does not see all: its other scores become -inf, where no bit is set
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int from = row_lo - (t0 + c * 32), upto = row_hi - (t0 + c * 32);
          const uint32_t below = upto < 0 ? 0u : upto >= 31 ? 0xffffffffu : (2u << upto) - 1u;
          const uint32_t bits = below & (from <= 0 ? 0xffffffffu : from >= 32 ? 0u : 0xffffffffu << from);
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (!(bits >> k & 1)) r[c][k] = 0xff800000u;
        }
      }
      // ---- maximum ----
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float x = -INFINITY;
#pragma unroll
        for (int k = (g & 1) * 16; k < (g & 1) * 16 + 16; k += 2)
          x = fmaxf(x, fmaxf(__uint_as_float(r[g >> 1][k]), __uint_as_float(r[g >> 1][k + 1])));
        // a group without a key: -inf, whatever its factors
        mx = fmaxf(mx, x == -INFINITY ? -INFINITY : CAP ? capped(x * c1[g]) + lv[g] : fmaf(x, c1[g], lv[g]));
      }
      const bool move = mx > m_ref + 8.f;  // (also from -inf)
      if (__any_sync(0xffffffffu, move)) {
        const float f = move && m_ref != -INFINITY ? fast_exp2(m_ref - mx) : 1.f;
        if (move) m_ref = mx;
        l *= f;
        if (it >= (Tr::DUAL ? 2 : 1) && __any_sync(0xffffffffu, f != 1.f)) {  // O up to the block before
          if (!tc5::mbar_wait(tc5::smem_addr(&sh->pv_done[t][b ^ 1]), ((n - 1) >> 1) & 1, abort_flag, 81)) return false;
          tc5::tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < Tr::HD / 8; ++c) {
            uint32_t o[8];
            tc5::tmem_ld8(o_tmem + c * 8, o);
            tc5::tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tc5::tmem_st8(o_tmem + c * 8, o);
          }
        }
      }
      pass();
      // ---- P' ----
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref - 7.f;
      uint32_t w[32];
      auto make_p = [&](auto masked) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float d = lv[g] - m_use;
          const uint64_t c12 = tc5::pack_f32x2(c1[g], c1[g]), d2 = tc5::pack_f32x2(d, d);
          uint64_t sum2 = tc5::pack_f32x2(0.f, 0.f);
#pragma unroll
          for (int k = (g & 1) * 16; k < (g & 1) * 16 + 16; k += 2) {
            const float s0 = __uint_as_float(r[g >> 1][k]), s1 = __uint_as_float(r[g >> 1][k + 1]);
            float x0, x1;
            if (CAP) {
              x0 = capped(s0 * c1[g]) + d;
              x1 = capped(s1 * c1[g]) + d;
            } else {
              tc5::unpack_f32x2(tc5::fma_f32x2(tc5::pack_f32x2(s0, s1), c12, d2), x0, x1);
            }
            if (decltype(masked)::value) {  // hidden is hidden, whatever the factors (-cap, or NaN of -inf * 0)
              x0 = s0 == -INFINITY ? s0 : x0;
              x1 = s1 == -INFINITY ? s1 : x1;
            }
            x0 = fast_exp2(x0);
            x1 = fast_exp2(x1);
            sum2 = tc5::add_f32x2(sum2, tc5::pack_f32x2(x0, x1));
            w[g * 8 + (k & 15) / 2] = pack2<__half>(x0, x1);
          }
          float sum0, sum1;
          tc5::unpack_f32x2(sum2, sum0, sum1);
          l = fmaf(sum0 + sum1, inv[g], l);
        }
      };
      if (edge) make_p(std::true_type());
      else make_p(std::false_type());
      tc5::tmem_st32(s_tmem, w);
      tc5::tmem_wait_st();  // (and O's)
    }
    pass();
    tc5::tc_fence_before();
    __syncwarp();
    if (lane == 0) {
      tc5::mbar_arrive(tc5::smem_addr(&sh->p_full[t][b]));
      tc5::mbar_arrive(tc5::smem_addr(&sh->sc_empty[e]));
    }
  }
  pass();
  // ---- output ----
  const int last = Tr::DUAL ? (((first + cnt - 1) & 1) == t ? cnt - 1 : cnt - 2) : cnt - 1;  // this sub-tile's last block
  if (last >= 0) {
    const int n = Tr::local(first + last);
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->pv_done[t][n & 1]), (n >> 1) & 1, abort_flag, 82)) return false;
    tc5::tc_fence_after();
  }
  float f = 0.f, f1 = 0.f;  // factors of this sub-tile's O, and (DUAL) of sub-tile 1's, which lies in the same TMEM lanes
  if (Tr::DUAL && cnt > 0) {
    if (t == 1) {
      sh->ml[lane_row] = make_float2(m_ref, l);
      tc5::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(tc5::smem_addr(&sh->other_done));
      return true;
    }
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->other_done), seg & 1, abort_flag, 84)) return false;
    tc5::tc_fence_after();
    const float2 o = sh->ml[lane_row];
    const float m = fmaxf(m_ref, o.x);
    f = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - m);
    f1 = o.x == -INFINITY ? 0.f : fast_exp2(o.x - m);
    l = l * f + o.y * f1;
    m_ref = m;
  } else if (Tr::DUAL && t == 1) {
    return true;
  } else {
    f = 1.f;
  }
  if (!any_live) return true;
  const bool dead = l == 0.f;  // (a NaN is none)
  const float scale = dead ? 0.f : 1.f / l;
  f *= scale;
  f1 *= scale;
  const float lse = dead ? -INFINITY : (m_ref - 7.f + log2f(l)) * kLn2;
  const bool to_partial = p.persistent || p.num_splits > 1;
  const int64_t lse_idx = (int64_t)sg.bi * p.a.lse_batch_stride + (int64_t)head * p.a.lse_head_stride + sq.q_row0 + i;
  if (live) {
    if (to_partial) {
      p.lse_partial[(int64_t)sg.slot * p.lse_elems + lse_idx] = lse;
      for (int sl = sg.fill_from; sl < p.num_splits; ++sl) p.lse_partial[(int64_t)sl * p.lse_elems + lse_idx] = -INFINITY;
    } else {
      p.a.lse[lse_idx] = dead ? INFINITY : lse;
    }
  }
  T* orow = reinterpret_cast<T*>(p.a.o) + (int64_t)sg.bi * p.a.o_batch_stride + (int64_t)(sq.q_row0 + i) * p.a.o_row_stride +
            (int64_t)head * p.a.o_head_stride;
  float* prow = to_partial ? p.o_partial + ((int64_t)sg.slot * p.lse_elems + lse_idx) * p.a.d : nullptr;
#pragma unroll 1
  for (int c = 0; c < Tr::HD / 16; ++c) {
    uint32_t r[16], r1[16];
    if (cnt > 0) {
      tc5::tmem_ld16(o_tmem + c * 16, r);
      if (Tr::DUAL) tc5::tmem_ld16(o_tmem + Tr::SUB_STEP + c * 16, r1);
      tc5::tmem_wait_ld();
    }
    if (live && !(dead && to_partial)) {
#pragma unroll
      for (int k = 0; k < 16; k += 8) {
        if (c * 16 + k < p.a.d) {
          float x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {  // (a factor of 0: that O may be anything)
            x[u] = f == 0.f ? 0.f : __uint_as_float(r[k + u]) * f;
            if (Tr::DUAL) x[u] += f1 == 0.f ? 0.f : __uint_as_float(r1[k + u]) * f1;
          }
          if (to_partial) {
            *reinterpret_cast<float4*>(prow + c * 16 + k) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(prow + c * 16 + k + 4) = make_float4(x[4], x[5], x[6], x[7]);
          } else {
            *reinterpret_cast<uint4*>(orow + c * 16 + k) =
                make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
          }
        }
      }
    }
    __syncwarp();  // the next columns are loaded by all lanes together
  }
  return true;
}

template <class Tr, int CODE>
__global__ void __launch_bounds__(Tr::NTHREADS, Tr::RESIDENT) kv8_tile_kernel(const __grid_constant__ Kv8Params p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ Kv8TileShared sh;
  grid_wait();
  grid_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  if (tid == 0) {
    for (int s = 0; s < Tr::RING; ++s) {
      tc5::mbar_init(tc5::smem_addr(&sh.kv_full[s]), Tr::CONV_WARPS / 2);
      tc5::mbar_init(tc5::smem_addr(&sh.kv_empty[s]), Tr::ROW_TILES);
    }
    for (int s = 0; s < Tr::SCR; ++s) {
      tc5::mbar_init(tc5::smem_addr(&sh.sc_full[s]), 1);
      tc5::mbar_init(tc5::smem_addr(&sh.sc_empty[s]), 4 * Tr::ROW_TILES + Tr::CONV_WARPS);
    }
    for (int t = 0; t < 2; ++t) {
      tc5::mbar_init(tc5::smem_addr(&sh.q_full[t]), 4);
      for (int b = 0; b < 2; ++b) {
        tc5::mbar_init(tc5::smem_addr(&sh.s_full[t][b]), 1);
        tc5::mbar_init(tc5::smem_addr(&sh.p_full[t][b]), 4);
        tc5::mbar_init(tc5::smem_addr(&sh.pv_done[t][b]), 1);
      }
    }
    tc5::mbar_init(tc5::smem_addr(&sh.other_done), 4);
    tc5::mbar_init(tc5::smem_addr(&sh.half_way), 4);
    sh.abort_flag = 0;
    tc5::fence_barrier_init();
  }
  if (warp == 0) {
    tc5::tmem_alloc(tc5::smem_addr(&sh.tmem_base), Tr::TMEM);
    tc5::tmem_relinquish();
  }
  tc5::tc_fence_before();
  __syncthreads();
  tc5::tc_fence_after();
  const uint32_t tmem = sh.tmem_base;

  // Every warp walks the CTA's segments by itself: run(segment, its sequence, key blocks and segments with key blocks before it).
  // (All barriers run on from segment to segment.  Q, S and O of the next one are written when the softmax warps have read O, which is
  // behind the last product.)
  // What outlasts a block lives in shared memory, a copy a warp: registers are for the scores.
  struct WarpState {
    Kv8Walk<Tr::BM, Tr::BN, Tr::OVH> walk;
    Kv8Mask mask;
    Kv8Seg sg;
    Kv8Seq sq;
  };
  __shared__ WarpState s_state[Tr::NTHREADS / 32];
  WarpState& st = s_state[warp];
  auto walk = [&](auto run) {
    {
      Kv8Walk<Tr::BM, Tr::BN, Tr::OVH> w;
      Kv8Seg sg;
      const Kv8Mask mask = kv8_mask(p, lane);
      w.first(p, mask, lane, sg);
      if (lane == 0) {
        st.mask = mask;
        st.walk = w;
        st.sg = sg;
      }
    }
    int blocks = 0, segs = 0;
    for (;;) {
      __syncwarp();
      const int valid = st.sg.valid;
      if (!valid) return;
      if (valid == 1) {
        if (lane == 0) st.sq = kv8_seq(p, st.mask, st.sg.bi, st.sg.mb, Tr::BM);
        __syncwarp();
        if (st.sg.mb * Tr::BM < st.sq.q_len * p.group) {
          if (!run(st.sq, st.sg, blocks, segs)) return;
          blocks += st.sg.cnt;
          segs += st.sg.cnt > 0;
        }
      }
      __syncwarp();
      if (lane == 0) st.walk.next(p, st.mask, st.sg);
    }
  };
  if (warp < Tr::SOFTMAX_WARPS) {
    if (Tr::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(Tr::SOFTMAX_REGS));
    const int t = warp >> 2, row = tid - t * 128;
    auto softmax = [&](auto type, auto cap) {
      walk([&](const Kv8Seq& sq, const Kv8Seg& sg, int blocks, int segs) {
        return kv8_softmax<Tr, decltype(type), decltype(cap)::value>(p, st.mask, sq, sg, &sh, smem, tmem, blocks, segs, t, row);
      });
    };
    const bool cap = p.a.softcap > 0.f;
    if (p.a.dtype == FA_BF16) {
      if (cap) softmax(__nv_bfloat16(), std::true_type());
      else softmax(__nv_bfloat16(), std::false_type());
    } else {
      if (cap) softmax(__half(), std::true_type());
      else softmax(__half(), std::false_type());
    }
  } else if (warp < Tr::SOFTMAX_WARPS + Tr::CONV_WARPS) {
    if (Tr::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(Tr::CONV_REGS));
    walk([&](const Kv8Seq& sq, const Kv8Seg& sg, int blocks, int) {
      return kv8_convert<Tr, CODE>(p, sq, sg, &sh, smem, blocks, tid - 32 * Tr::SOFTMAX_WARPS);
    });
    cp_async_wait<0>();  // (something is left only when a wait has given up)
  } else {
    if (Tr::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(Tr::ISSUE_REGS));
    const int t = warp - Tr::SOFTMAX_WARPS - Tr::CONV_WARPS;
    const float s = fabsf(p.a.softmax_scale), mul = p.a.softcap > 0.f ? s / p.a.softcap : s * kLog2e;
    if (t == 2) {
      walk([&](const Kv8Seq& sq, const Kv8Seg& sg, int blocks, int) { return kv8_scout<Tr>(p, sq, sg, &sh, mul, blocks, lane); });
    } else if (t < Tr::NSUB) {
      Kv8Ring<Tr::RING> ring;
      walk([&](const Kv8Seq&, const Kv8Seg& sg, int blocks, int segs) {
        return sg.cnt == 0 || kv8_issue<Tr>(&sh, smem, tmem, ring, blocks, segs, t, sg.cnt);
      });
    }
  }

  __syncwarp();
  tc5::tc_fence_before();
  __syncthreads();
  if (sh.abort_flag) {
    for (int k = 0; k < 64; ++k) __nanosleep(2000);  // let products in flight end before TMEM goes
    if (tid == 0 && p.status) atomicExch(p.status, (sh.abort_flag << 16) | ((int)blockIdx.x % 0xffff + 1));
  }
  if (warp == 0) {
    tc5::tc_fence_after();
    tc5::tmem_dealloc(tmem, Tr::TMEM);
  }
}

}  // namespace fa
