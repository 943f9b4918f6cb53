// Attention over an 8-bit KV cache for many query rows: tcgen05 products with accumulators in TMEM, fp16 operands.
//
// A CTA has a tile of packed query rows (row = token * group + head; all heads of a kv head's group, so a key is turned into fp16
// once for all of them) against a range of key blocks.  Tiles that are few share the key blocks of the whole launch out equally
// among resident CTAs, as the decode kernel does (Kv8Walk).
// Arithmetic as in kv8_decode_kernel.cuh: V's scale in the exponent, P' in fp16, scales never in a product.  The reference m of
// the exponent is the running maximum, moved only when that has grown by more than 2^8: P' = 2^(x - m + 7) stays below 2^15, far from
// fp16's end, and below 2^7 it has as many bits as a 16-bit output shows; so O is rescaled in TMEM a few times a tile and
// not at every block.
//
// Warps: 4 per sub-tile of 128 rows  softmax, one thread per row (Q load, P, rescale of O, epilogue)
//        4                           converters: codes -> fp16 tiles in the swizzled operand layout; global loads of a tile in flight
//                                    while the one before is turned
//        1 per sub-tile              MMA issue
//        1                           scout: pages and scales, some blocks ahead (and one or two warps fill up the warpgroup)
// Blocks of 64 keys, two S buffers per sub-tile: S of block j + 1 is there when the softmax of block j ends, so its threads wait for no
// product.  A thread keeps its 64 scores in registers, and P' goes back into the columns it read, as the TMEM operand of P.V: no
// shared-memory traffic and no proxy fence for P.  S of block j + 2 lands on P of block j; the same thread issues both products, in
// this order.  TMEM: per sub-tile S 2 x 64, O 128 columns; one sub-tile with 256 columns of O for head dims above 128.
// (Before, 128 keys at a time, P through shared memory, S read twice from TMEM: 636 us for four chunks of 301 - 2048 tokens against
// 1777 - 8192 keys, 32 / 8 heads, of which a third was waiting for products and fences.)
//
// Bound: per 128 keys and 256 rows of head dim 128 the products take 2048 cycles of an SM's tensor pipe, the exponentials 2048 of its
// special-function unit, 320 KB through shared memory 2560, turning the codes about 1000 of 8192 issue slots.  TMA cannot convert,
// so the codes pass through registers.
#pragma once

#include <type_traits>

#include "kv8.cuh"

namespace fa {

template <int HD_, int NSUB_>
struct Kv8TileTraits {
  static constexpr int HD = HD_, NSUB = NSUB_;  // sub-tiles of 128 rows
  static_assert(NSUB == 1 || HD <= 128, "256 columns of O and two S buffers leave TMEM room for one sub-tile");
  static constexpr int BM = 128 * NSUB, BN = 64;
  static constexpr int GROUPS = BN / kScaleGranule;
  static constexpr int HALVES = HD / 64;                 // 64-column halves of Q, K, V
  static constexpr int KV_HALF = BN * 128, SLOT_BYTES = HALVES * KV_HALF;
  static constexpr int Q_HALF = 128 * 128, Q_BYTES = HALVES * Q_HALF;  // per sub-tile
  static constexpr int RESIDENT = NSUB == 1 && HD <= 128 ? 2 : 1;      // CTAs of an SM
  static constexpr int RING = HD == 256 || RESIDENT == 2 ? 4 : 8;
  static constexpr int RING_OFF = NSUB * Q_BYTES;
  static constexpr int SMEM_BYTES = 1024 + RING_OFF + RING * SLOT_BYTES;
  static constexpr int SOFTMAX_WARPS = 4 * NSUB, CONV_WARPS = 4, NTHREADS = 32 * (SOFTMAX_WARPS + CONV_WARPS + 4);
  // Registers by warpgroup (setmaxnreg; one sub-tile of 256 columns has enough as it is): shares of what a CTA is launched with
  // (128 a thread, 80 where two are resident) and never more.
  static constexpr bool SPLIT = HD <= 128;
  static constexpr int LAUNCH_REGS = NSUB == 2 ? 120 : 80, SOFTMAX_REGS = NSUB == 2 ? 160 : 128, CONV_REGS = NSUB == 2 ? 112 : 64, ISSUE_REGS = NSUB == 2 ? 48 : 40;
  static_assert(NSUB * SOFTMAX_REGS + CONV_REGS + ISSUE_REGS <= (NSUB + 2) * LAUNCH_REGS && RESIDENT * NTHREADS * LAUNCH_REGS <= 65536 || !SPLIT,
                "more registers than a CTA is launched with");
  static constexpr int CHUNKS = BN * HD / 16 / 128;  // 16-code chunks of a converter thread in a tile
  // TMEM columns: S of sub-tile t at t * SUB_STEP + buffer * BN, O at O_COL + t * SUB_STEP
  static constexpr int TMEM = RESIDENT == 2 ? 256 : 512, O_COL = RESIDENT == 2 ? 128 : 256, SUB_STEP = 128;
  static constexpr int SCR = 8;   // blocks that the scout may be ahead
  static constexpr int OVH = 4;   // a unit's fixed cost in blocks (Kv8Walk)
};

struct Kv8TileShared {
  uint64_t q_full[2], kv_full[8], kv_empty[8];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];  // [sub-tile][buffer]
  uint64_t sc_full[8], sc_empty[8];
  float4 sc[8][3];      // of a block: score factor, log2 of V's scale, its reciprocal, per 16 keys
  int64_t at[8][2][4];  // ... and where K's and V's codes of 16 keys start, from the head's first; -1: zeros
  uint32_t tmem_base;
  int abort_flag;
};

// Bounded wait for three barriers at once: a poll takes some 160 cycles even where there is nothing to wait for, and three in a row are
// a sixth of a block's softmax.
__device__ __forceinline__ bool kv8_wait3(uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1, uint32_t b2, uint32_t p2, volatile int* abort_flag, int id) {
  for (uint32_t i = 0; i < tc5::kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q, r;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n\t"
        "and.pred p, p, q;\n\tand.pred p, p, r;\n\tselp.b32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(b0), "r"(p0), "r"(b1), "r"(p1), "r"(b2), "r"(p2)
        : "memory");
    if (ok) return true;
    if ((i & 255u) == 255u && *abort_flag) return false;
  }
  if (*abort_flag == 0) *abort_flag = id;
  return false;
}

// Ring positions in the order the products need the tiles: K_0 | K_1 V_0 | K_2 V_1 | ... | V_last.
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
// One warp, up to SCR blocks ahead: pages and scales are two dependent loads that the converters need not wait for.
template <class Tr>
__device__ __forceinline__ bool kv8_scout(const Kv8Params& p, const Kv8Seq sq, const Kv8Seg sg, Kv8TileShared* sh, float mul, int base, int lane) {
  volatile int* abort_flag = &sh->abort_flag;
  const bool is_v = lane >= Tr::GROUPS, on = lane < 2 * Tr::GROUPS;  // lanes 0 .. GROUPS - 1: K of 16-key group `lane`, then V
  const int grp = lane % Tr::GROUPS;
  const float* scale = is_v ? p.c.v_scale + sg.hk * p.c.vs_head_stride : p.c.k_scale + sg.hk * p.c.ks_head_stride;
  const int64_t s_outer = is_v ? p.c.vs_outer_stride : p.c.ks_outer_stride, s_block = is_v ? p.c.vs_block_stride : p.c.ks_block_stride;
  const int64_t c_outer = is_v ? p.a.v_batch_stride : p.a.k_batch_stride, c_row = is_v ? p.a.v_row_stride : p.a.k_row_stride;
  for (int it = 0; it < sg.cnt; ++it) {
    const int n = base + it, e = n % Tr::SCR, t = (sg.lo + it) * Tr::BN + grp * kScaleGranule;
    int64_t at = -1;  // nothing there: zeros
    float s = 0.f;
    if (on && t < sq.key_hi && t + kScaleGranule > sq.key_lo) {  // some row sees a key of the group: its page is a live one
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
    if (n >= Tr::SCR && !tc5::mbar_wait(tc5::smem_addr(&sh->sc_empty[e]), (n / Tr::SCR - 1) & 1, abort_flag, 72)) return false;
    if (on) {
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
  return true;
}

// ---------------- converters ----------------
// A thread turns 16-code chunks of column tid % 4 in every 64-column half, of rows tid / 4 + 32 k: two rows of a quarter warp meet eight
// different banks.
template <class Tr, int CODE>
__device__ __forceinline__ bool kv8_convert(const Kv8Params& p, const Kv8Seq sq, const Kv8Seg sg, Kv8TileShared* sh, uint32_t ring_smem,
                                            Kv8Ring<Tr::RING>& ring, int first, int tid) {
  constexpr int NC = Tr::CHUNKS, ROWS = NC / Tr::HALVES;
  volatile int* abort_flag = &sh->abort_flag;
  const int lane = tid & 31, c4 = tid & 3, row0 = tid >> 2, in_grp = row0 % kScaleGranule;
  const int64_t k_rs = p.a.k_row_stride, v_rs = p.a.v_row_stride;
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(p.a.k) + (int64_t)sg.hk * p.a.k_head_stride + c4 * 16 + in_grp * k_rs;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(p.a.v) + (int64_t)sg.hk * p.a.v_head_stride + c4 * 16 + in_grp * v_rs;
  const int cols_left = p.a.d - c4 * 16;  // halves h with 64 h < cols_left hold columns of the head

  auto fetch = [&](uint4 (&x)[NC], int it, bool is_v) {
    const int e = (first + it) % Tr::SCR, t0 = (sg.lo + it) * Tr::BN;
    const uint8_t* base = is_v ? vb : kb;
    const bool whole = t0 >= sq.key_lo && t0 + Tr::BN <= sq.key_hi;
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int row = row0 + 32 * k;
      const int64_t at = sh->at[e][is_v][row / kScaleGranule];
      const bool on = at >= 0 && (whole || (t0 + row >= sq.key_lo && t0 + row < sq.key_hi));
#pragma unroll
      for (int h = 0; h < Tr::HALVES; ++h) {
        uint4& y = x[k * Tr::HALVES + h];
        y = make_uint4(0, 0, 0, 0);
        if (on && h * 64 < cols_left) y = __ldg(reinterpret_cast<const uint4*>(base + at + h * 64));
      }
    }
  };
  auto put = [&](const uint4 (&x)[NC]) {
    uint32_t slot, par;
    ring.next(slot, par);
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->kv_empty[slot]), par ^ 1, abort_flag, 71)) return false;
    const uint32_t tile = ring_smem + slot * Tr::SLOT_BYTES + row0 * 128;
    const uint32_t lo = ((c4 * 2) ^ (row0 & 7)) << 4, hi = ((c4 * 2 + 1) ^ (row0 & 7)) << 4;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const uint32_t at = tile + (i % Tr::HALVES) * Tr::KV_HALF + (i / Tr::HALVES) * (32 * 128);
      uint32_t h[8];
      decode4<CODE>(x[i].x, h[0], h[1]);
      decode4<CODE>(x[i].y, h[2], h[3]);
      decode4<CODE>(x[i].z, h[4], h[5]);
      decode4<CODE>(x[i].w, h[6], h[7]);
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(at + lo), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(at + hi), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
    }
    tc5::fence_proxy_async();  // generic-proxy stores -> visible to the MMA
    __syncwarp();
    if (lane == 0) tc5::mbar_arrive(tc5::smem_addr(&sh->kv_full[slot]));
    return true;
  };

  // tiles in ring order, one ahead in registers
  int kq = 0, vq = 0;
  bool ok = true;
  auto load = [&](uint4 (&x)[NC]) {
    if (kq < sg.cnt && kq <= vq + 1) {
      const int n = first + kq;
      if (!tc5::mbar_wait(tc5::smem_addr(&sh->sc_full[n % Tr::SCR]), (n / Tr::SCR) & 1, abort_flag, 70)) return ok = false;
      fetch(x, kq, false);
      ++kq;
    } else {
      if (vq == sg.cnt) return false;
      fetch(x, vq, true);
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(tc5::smem_addr(&sh->sc_empty[(first + vq) % Tr::SCR]));
      ++vq;
    }
    return true;
  };
  uint4 xa[NC], xb[NC];
  bool more = load(xa);
  while (more) {
    more = load(xb);
    if (!put(xa)) return false;
    if (!more) break;
    more = load(xa);
    if (!put(xb)) return false;
  }
  return ok;
}

// ---------------- MMA issue, sub-tile t ----------------
template <class Tr>
__device__ __forceinline__ bool kv8_issue(Kv8TileShared* sh, uint32_t smem, uint32_t tmem, Kv8Ring<Tr::RING>& ring, int first, int seg, int t, int cnt) {
  volatile int* abort_flag = &sh->abort_flag;
  constexpr uint32_t idesc_qk = tc5::make_idesc(0, 128, Tr::BN, 0), idesc_pv = tc5::make_idesc(0, 128, Tr::HD, 1);
  const uint64_t q_desc = tc5::make_smem_desc(smem + t * Tr::Q_BYTES, 16, 1024);
  const uint64_t k_desc0 = tc5::make_smem_desc(smem + Tr::RING_OFF, 16, 1024);            // K-major
  const uint64_t v_desc0 = tc5::make_smem_desc(smem + Tr::RING_OFF, Tr::KV_HALF, 1024);   // N-contiguous
  constexpr uint64_t kSlot = Tr::SLOT_BYTES >> 4;
  // 16 columns per k-step = 32 bytes inside the 128-byte swizzle span
  auto off = [](int ks, int half) { return (uint64_t)(((ks >> 2) * half + (ks & 3) * 32) >> 4); };
  const uint32_t s_tmem0 = tmem + t * Tr::SUB_STEP, o_tmem = tmem + Tr::O_COL + t * Tr::SUB_STEP;
  if (!tc5::mbar_wait(tc5::smem_addr(&sh->q_full[t]), seg & 1, abort_flag, 73)) return false;
  // a ring slot is free when the products of every sub-tile that has rows have read it
  auto release = [&](uint32_t slot) { tc5::mma_commit(tc5::smem_addr(&sh->kv_empty[slot])); };
  // The buffer's last P has been read by the product of this thread in front of this one, its scores before that P was written.
  auto qk = [&](int it) {
    uint32_t slot, par;
    ring.next(slot, par);
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->kv_full[slot]), par, abort_flag, 74)) return false;
    tc5::tc_fence_after();
    const uint64_t k_desc = k_desc0 + slot * kSlot;
    const int n = first + it;
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
    const int n = first + it;
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->kv_full[slot]), par, abort_flag, 76)) return false;
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->p_full[t][n & 1]), (n >> 1) & 1, abort_flag, 77)) return false;
    tc5::tc_fence_after();
    const uint64_t v_desc = v_desc0 + slot * kSlot;
    const uint32_t p_tmem = s_tmem0 + (n & 1) * Tr::BN;
    if (tc5::elect_one()) {
      if (it == 0) tc5::mma_ts_c<false>(o_tmem, p_tmem, v_desc, idesc_pv);
      else tc5::mma_ts_c<true>(o_tmem, p_tmem, v_desc, idesc_pv);
#pragma unroll
      for (int ks = 1; ks < Tr::BN / 16; ++ks) tc5::mma_ts_c<true>(o_tmem, p_tmem + ks * 8, v_desc + (uint64_t)(ks * (2048 >> 4)), idesc_pv);
      tc5::mma_commit(tc5::smem_addr(&sh->pv_done[t][n & 1]));
      release(slot);
    }
    __syncwarp();
    return true;
  };
  if (!qk(0) || (cnt > 1 && !qk(1))) return false;
  for (int it = 0; it < cnt; ++it)
    if (!pv(it) || (it + 2 < cnt && !qk(it + 2))) return false;
  return true;
}

// ---------------- softmax, one thread per row ----------------
template <class Tr, typename T, bool CAP>
__device__ __forceinline__ bool kv8_softmax(const Kv8Params& p, const Kv8Mask& mask, const Kv8Seq& sq, const Kv8Seg& sg, Kv8TileShared* sh,
                                            uint32_t smem, uint32_t tmem, int first, int t, int lane_row) {
  volatile int* abort_flag = &sh->abort_flag;
  const int lane = lane_row & 31, warp = lane_row >> 5;
  const int rr = sg.mb * Tr::BM + t * 128 + lane_row, rows_total = sq.q_len * p.group;
  const bool live = rr < rows_total;
  const int i = rr / p.group, head = sg.hk * p.group + (rr - i * p.group);
  // ---- Q: fp16, negated for a negative scale (scores then grow with the products), bf16 rows brought into fp16's range ----
  float back = 1.f;
  if (sg.cnt > 0) {
    const uint32_t q_smem = smem + t * Tr::Q_BYTES + lane_row * 128;
    const T* qrow = reinterpret_cast<const T*>(p.a.q) + (int64_t)sg.bi * p.a.q_batch_stride + (int64_t)(sq.q_row0 + i) * p.a.q_row_stride +
                    (int64_t)head * p.a.q_head_stride;
    const bool rot = mask.causal || mask.local;
    float up = 1.f;
    if (std::is_same<T, __nv_bfloat16>::value) {
      uint32_t mx = 0;
      if (live) {
#pragma unroll 4
        for (int c8 = 0; c8 < p.a.d; c8 += 8) {
          const uint4 x = kv8_q_chunk<T>(p, qrow, c8, sq.k_len, i, rot);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w = e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w;
            mx = max(mx, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
          }
        }
      }
      back = bf16_row_factor(mx, up);
    }
    const float sign = p.a.softmax_scale < 0.f ? -1.f : 1.f;
    up *= sign;
#pragma unroll 2
    for (int ch = 0; ch < Tr::HD / 8; ++ch) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (live && ch * 8 < p.a.d) x = kv8_q_chunk<T>(p, qrow, ch * 8, sq.k_len, i, rot);
      uint32_t w[4] = {x.x, x.y, x.z, x.w};
      if (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = pack2<__half>(__uint_as_float(w[e] << 16) * up, __uint_as_float(w[e] & 0xffff0000u) * up);
      } else if (sign < 0.f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] ^= 0x80008000u;
      }
      const uint32_t at = q_smem + (ch >> 3) * Tr::Q_HALF + (((ch & 7) ^ (lane_row & 7)) << 4);
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
    tc5::fence_proxy_async();
    __syncwarp();
    if (lane == 0) tc5::mbar_arrive(tc5::smem_addr(&sh->q_full[t]));
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
  for (int it = 0; it < cnt; ++it) {
    const int n = first + it, b = n & 1, e = n % Tr::SCR, t0 = (lo + it) * Tr::BN;
    const uint32_t s_tmem = tmem + t * Tr::SUB_STEP + b * Tr::BN + lane_base;
    // (P.V of two blocks before is over when S of this one is there, but no phase of a barrier may be missed.  In front of the first two
    // blocks there was none: the phase before a barrier's first counts as over.)
    if (!kv8_wait3(tc5::smem_addr(&sh->s_full[t][b]), (n >> 1) & 1, tc5::smem_addr(&sh->sc_full[e]), (n / Tr::SCR) & 1,
                   tc5::smem_addr(&sh->pv_done[t][b]), ((n >> 1) + 1) & 1, abort_flag, 79))
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
        if (it > 0 && __any_sync(0xffffffffu, f != 1.f)) {  // O up to the block before
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
    tc5::tc_fence_before();
    __syncwarp();
    if (lane == 0) {
      tc5::mbar_arrive(tc5::smem_addr(&sh->p_full[t][b]));
      tc5::mbar_arrive(tc5::smem_addr(&sh->sc_empty[e]));
    }
  }
  // ---- output ----
  if (sg.cnt > 0) {
    const int last = first + sg.cnt - 1;
    if (!tc5::mbar_wait(tc5::smem_addr(&sh->pv_done[t][last & 1]), (last >> 1) & 1, abort_flag, 82)) return false;
    tc5::tc_fence_after();
  }
  if (!any_live) return true;
  const bool dead = l == 0.f;  // (a NaN is none)
  const float f = dead ? 0.f : 1.f / l;
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
#pragma unroll
  for (int c = 0; c < Tr::HD / 32; ++c) {
    uint32_t r[32];
    if (sg.cnt > 0) {
      tc5::tmem_ld32(o_tmem + c * 32, r);
      tc5::tmem_wait_ld();
    }
    if (live && !(dead && to_partial)) {
#pragma unroll
      for (int k = 0; k < 32; k += 8) {
        if (c * 32 + k < p.a.d) {
          float x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) x[u] = dead ? 0.f : __uint_as_float(r[k + u]) * f;
          if (to_partial) {
            *reinterpret_cast<float4*>(prow + c * 32 + k) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(prow + c * 32 + k + 4) = make_float4(x[4], x[5], x[6], x[7]);
          } else {
            *reinterpret_cast<uint4*>(orow + c * 32 + k) =
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
      tc5::mbar_init(tc5::smem_addr(&sh.kv_full[s]), Tr::CONV_WARPS);
      tc5::mbar_init(tc5::smem_addr(&sh.kv_empty[s]), Tr::NSUB);
    }
    for (int s = 0; s < Tr::SCR; ++s) {
      tc5::mbar_init(tc5::smem_addr(&sh.sc_full[s]), 1);
      tc5::mbar_init(tc5::smem_addr(&sh.sc_empty[s]), Tr::SOFTMAX_WARPS + Tr::CONV_WARPS);
    }
    for (int t = 0; t < 2; ++t) {
      tc5::mbar_init(tc5::smem_addr(&sh.q_full[t]), 4);
      for (int b = 0; b < 2; ++b) {
        tc5::mbar_init(tc5::smem_addr(&sh.s_full[t][b]), 1);
        tc5::mbar_init(tc5::smem_addr(&sh.p_full[t][b]), 4);
        tc5::mbar_init(tc5::smem_addr(&sh.pv_done[t][b]), 1);
      }
    }
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
      walk([&](const Kv8Seq& sq, const Kv8Seg& sg, int blocks, int) {
        return kv8_softmax<Tr, decltype(type), decltype(cap)::value>(p, st.mask, sq, sg, &sh, smem, tmem, blocks, t, row);
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
    Kv8Ring<Tr::RING> ring;
    walk([&](const Kv8Seq& sq, const Kv8Seg& sg, int blocks, int) {
      return sg.cnt == 0 || kv8_convert<Tr, CODE>(p, sq, sg, &sh, smem + Tr::RING_OFF, ring, blocks, tid - 32 * Tr::SOFTMAX_WARPS);
    });
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
