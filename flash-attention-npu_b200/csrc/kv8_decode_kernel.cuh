// Attention over an 8-bit KV cache for few query rows: the rows of a kv head's query group share a tile of 8, 16 or 32, the whole of a
// sequence's.
//
// HBM-bound: K and V of the visible range are read once, at one byte per element.  A producer warp moves stages of BN keys
// (K and V) with tiled TMA loads into a ring, and the stage's scales with 4-byte asynchronous copies; consumer warps own 8 or 16 query
// rows and a slice of the stage's keys each, turn codes into fp16 in registers and multiply with mma.sync (the tile kernel on such calls:
// 2.2 times as long for 8 rows, 7 % longer for 32; its 128-row tensor instruction waits for the turning of codes all the same).
// Calls in a CUDA graph: 8 sequences of 131072 keys, 64 / 8 heads of 128, 315 us, 6.8 TB/s (by themselves, between other kernels' writes, 341 -
// 371).  64 ragged ones of up to 8191 keys with a token appended: 108 us, 5.6 TB/s.  32 sequences with a window of 4096 keys and 4 tokens,
// 64 / 8 heads: 123 us of 40 that HBM would take -- at 32 rows a warp scheduler holds three warps of 168 registers, and what they wait for is
// one another's products and the instruction cache, not memory (ncu: issue 37 %, mma 25 %).  Eight key slices of 32 rows each, with every code
// turned once, spill and took 205 us; the forms here spill too: 204 bytes a thread at 32 rows of 128 columns and 156 at 16 (168 registers), 280 at
// 32 rows of 64 (two CTAs, 96 registers), 220 - 360 at 256 columns.
//
// Arithmetic.  K = ck * sk(block), V = cv * sv(block).  With the running maximum over x_j = scale * log2e * sk * (q . ck_j) + log2 sv,
//   P'_j = 2^(x_j - m + 15),   O = sum_j P'_j cv_j / l,   l = sum_j P'_j / sv_j,   LSE = ln2 (m - 15) + ln l:
// V's scale rides in the exponent, so that no product is scaled and P' spans all of fp16 (up to 2^15) where what it is multiplied
// with is largest.  P' is rounded to fp16 (2^-12) for the second product, which is what a 16-bit output can show; below 2^-14 (2^-29 of the
// largest) it is a subnormal, off by 2^-25 at most, that is by 2^-40 of the row's largest weight times scale for each code.  The codes
// are fp16 values, sums and statistics are fp32.
//
// Both products are transposed, S^T = K Q^T and O^T = V^T P^T: query rows are the narrow side of mma m16n8k16, so that the eight rows
// of a usual query group fill it (rows on the wide side: 8 % faster at 32 rows, half of every product padding at 8; one short sequence 13.5 us against 11.3).  P^T comes out of S^T by a transposition
// of 8 x 8 tiles within the warp (movmatrix).
// Fragments straight from the codes.  A contraction may run over its index in any order, and output columns may be numbered in
// any order, as long as both operands agree: lane (g8, t4) takes LB consecutive bytes of key rows g8 and g8 + 8 as the K elements of
// its k-steps (four a step), and for V VB consecutive bytes of four key rows as columns g8 and g8 + 8 of VB / 2 tiles, two
// rows' bytes interleaved by a byte permutation.  So every shared-memory access is a wide one, free of bank conflicts under the TMA
// swizzle, and each code is turned once: per 16 keys of head dim 128 and 8 rows a warp issues 8 loads, 64 conversions, 16 permutations
// and 16 mma (32 cycles of an SM's mma.sync rate, against 178 cycles in which HBM delivers the bytes).
#pragma once

#include <type_traits>

#include "kv8.cuh"

namespace fa {

template <int HD_, int WM_, int NQ_>
struct Kv8Traits {
  static constexpr int HD = HD_, WM = WM_, NQ = NQ_, WN = HD == 128 && WM == 2 ? 5 : 4, NCW = WM * WN;  // NQ: 8-row tiles of a warp; WM warps' rows, WN warps' keys
  static_assert(HD == 64 || HD == 128 || HD == 256, "tile widths; a head dim below the width leaves zero columns (TMA fill)");
  static constexpr int BM = 8 * NQ * WM;
  static constexpr int BN = HD == 256 ? 64 : 32 * WN;
  static constexpr int NTHREADS = 32 * (NCW + 1);
  static constexpr int NW = BN / WN;   // keys of a consumer warp in a stage
  static constexpr int NG = NW / kScaleGranule;  // 16-key groups of them
  static constexpr int KS = HD / 16;
  static constexpr int ROWB = HD < 128 ? HD : 128;  // bytes of a key row in one TMA box (the swizzle's span)
  static constexpr int HALVES = HD / ROWB;
  static constexpr int LB = ROWB / 4;  // bytes of a key row that a lane owns in K, per half
  static constexpr int VB = ROWB / 8;  // and in V
  static constexpr int HALF_BYTES = BN * ROWB;
  static constexpr int KV_BYTES = HALVES * HALF_BYTES;
  static constexpr int STAGE_BYTES = 2 * KV_BYTES;
  // up to 16 rows: two resident CTAs of 96 KiB rings (64 columns: 80 KiB); 32 rows: one CTA with all of it (64 columns: two).
  // 32 rows of 128 columns: five key slices, since ten consumer warps and the producer fill the warp schedulers' registers (four: 128 us against 124
  // in the case above).
  static constexpr int RESIDENT = WM == 1 || HD == 64 ? 2 : 1;
  static constexpr int ST = HD == 64 ? 5 : WM == 1 ? 3 : 5;
  static constexpr int GROUPS = BN / kScaleGranule;
  static constexpr int SLAB_LD = ROWB + 4;
  static constexpr int PIPE_BYTES = ST * STAGE_BYTES;
  // Q fragments, and when the keys are done the merged rows (fp32), 128 columns at a time
  static constexpr int Q_BYTES = BM * HD * 2, SLAB_BYTES = BM * SLAB_LD * 4;
  static constexpr int TILE_BYTES = Q_BYTES > SLAB_BYTES ? Q_BYTES : SLAB_BYTES;
  static constexpr int ML_BYTES = WN * BM * 8;
  static constexpr int SC_BYTES = ST * 2 * GROUPS * 4;
  static constexpr int BAR_BYTES = 2 * ST * 8;
  // [ring | Q or rows | (m, l) | scales | row factors | barriers], the ring at a 1024-byte aligned base
  static constexpr int SMEM_BYTES = 1024 + PIPE_BYTES + TILE_BYTES + ML_BYTES + SC_BYTES + BM * 4 + BAR_BYTES;
  static constexpr bool Q_IN_REGS = HD * NQ <= 256;
  static_assert(SMEM_BYTES * RESIDENT <= 227 * 1024 - 2048 * RESIDENT, "shared memory");
};

// Byte address of 16-byte chunk `ch` of row `row` in a tile laid out by TMA boxes of ROWB columns with the swizzle of that span.
template <class Tr>
__device__ __forceinline__ uint32_t code_addr(uint32_t tile, int row, int ch) {
  if (Tr::ROWB == 128) return tile + (ch >> 3) * Tr::HALF_BYTES + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
  return tile + row * 64 + ((ch ^ ((row >> 1) & 3)) << 4);
}
__device__ __forceinline__ void lds128(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <int N>
__device__ __forceinline__ void lds64(uint32_t (&r)[N], uint32_t addr) {
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];\n" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
}
__device__ __forceinline__ float lds32f(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(addr));
  return v;
}

// The stages of one segment.
template <class Tr>
__device__ __forceinline__ bool kv8_producer(const Kv8Params& p, const Kv8Seq& sq, const Kv8Seg& sg, const CUtensorMap* tm_k,
                                             const CUtensorMap* tm_v, uint32_t pipe, uint32_t scales, uint32_t full0, uint32_t empty0,
                                             uint32_t it_base, int lane, volatile int* abort_flag) {
  const int box = p.box_rows, n_box = Tr::BN / box;
  const int outer_none = p.a.kv_outer > 0 ? p.a.kv_outer : p.a.b;  // a TMA coordinate beyond the pool: zeros arrive
  for (int it = 0; it < sg.cnt; ++it) {
    const uint32_t git = it_base + (uint32_t)it;
    const int stage = (int)(git % Tr::ST);
    const int t0 = (sg.lo + it) * Tr::BN;
    // pages are looked up where some row sees a key of theirs, and only there: others may be stale
    int row = 0, outer = outer_none;
    const int tb = t0 + lane * box;
    if (lane < n_box && tb < sq.key_hi && tb + box > sq.key_lo) {
      row = tb;
      outer = sq.batch_row;
      if (sq.pages) {
        const int pg = tb / p.a.page_size;
        row = tb - pg * p.a.page_size;
        outer = __ldg(sq.pages + pg);
        check_outer_index(p.a, outer, p.status);
      }
    }
    const float* src = nullptr;
    const int kv = lane / Tr::GROUPS, grp = lane % Tr::GROUPS, tg = t0 + grp * kScaleGranule;
    if (lane < 2 * Tr::GROUPS && tg < sq.key_hi && tg + kScaleGranule > sq.key_lo) {
      int o = sq.batch_row, r = tg;
      bool there = true;
      if (sq.pages) {
        const int pg = tg / p.a.page_size, id = __ldg(sq.pages + pg);
        r = tg - pg * p.a.page_size;
        o = outer_index(p.a, id, p.status);
        there = o == id;  // else its codes arrive as zeros, and the scale of another page is none of theirs
      }
      const int blk = r / p.c.scale_block;
      if (there)
        src = kv == 0 ? p.c.k_scale + o * p.c.ks_outer_stride + blk * p.c.ks_block_stride + sg.hk * p.c.ks_head_stride
                      : p.c.v_scale + o * p.c.vs_outer_stride + blk * p.c.vs_block_stride + sg.hk * p.c.vs_head_stride;
    }
    if (git >= (uint32_t)Tr::ST && !tc5::mbar_wait(empty0 + stage * 8, ((git / Tr::ST) - 1) & 1, abort_flag)) return false;
    const uint32_t k_base = pipe + stage * Tr::STAGE_BYTES, v_base = k_base + Tr::KV_BYTES, full = full0 + stage * 8;
    if (lane == 0) tc5::mbar_arrive_expect_tx(full, Tr::STAGE_BYTES);
    __syncwarp();
    if (lane < n_box) {
      const uint32_t at = lane * box * Tr::ROWB;
#pragma unroll
      for (int hf = 0; hf < Tr::HALVES; ++hf) {
        tc5::tma_load_4d(k_base + hf * Tr::HALF_BYTES + at, tm_k, full, 128 * hf, sg.hk, row, outer);
        tc5::tma_load_4d(v_base + hf * Tr::HALF_BYTES + at, tm_v, full, 128 * hf, sg.hk, row, outer);
      }
    }
    if (lane < 2 * Tr::GROUPS) {  // nothing to read: zero
      const uint32_t dst = scales + (stage * 2 * Tr::GROUPS + lane) * 4;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src ? src : p.c.k_scale), "r"(src ? 4 : 0) : "memory");
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(full) : "memory");
  }
  return true;
}

// Q rows -> fp16 fragments in shared memory, [8-row tile][k-step][lane][2 registers], and the factor of each row.
template <class Tr, typename T>
__device__ __forceinline__ void kv8_load_q(const Kv8Params& p, const Kv8Seq& sq, const Kv8Seg& sg, uint32_t q_base, float* factor,
                                           bool rot_per_token, int warp, int lane) {
  constexpr int LPR = Tr::HD / 8, RPW = 32 / LPR;  // lanes of a row, rows of a warp
  const int rows_total = sq.q_len * p.group, sub = lane / LPR, c8 = (lane % LPR) * 8;
  for (int r0 = warp * RPW; r0 < Tr::BM; r0 += Tr::NCW * RPW) {
    const int row = r0 + sub;
    Vec16 x;
    x.u = make_uint4(0, 0, 0, 0);
    if (row < rows_total && c8 < p.a.d) {
      const int i = row / p.group, head = sg.hk * p.group + (row - i * p.group);
      const T* qrow = reinterpret_cast<const T*>(p.a.q) + (int64_t)sg.bi * p.a.q_batch_stride +
                      (int64_t)(sq.q_row0 + i) * p.a.q_row_stride + (int64_t)head * p.a.q_head_stride;
      x.u = kv8_q_chunk<T>(p, qrow, c8, sq.k_len, i, rot_per_token);
    }
    uint32_t w[4] = {x.u.x, x.u.y, x.u.z, x.u.w};
    float back = 1.f;
    if (std::is_same<T, __nv_bfloat16>::value) {
      uint32_t mx = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = max(mx, max(w[e] & 0x7fffu, (w[e] >> 16) & 0x7fffu));
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      float up;
      back = bf16_row_factor(mx, up);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = pack2<__half>(__uint_as_float(w[e] << 16) * up, __uint_as_float(w[e] & 0xffff0000u) * up);
    }
    if (c8 == 0) factor[row] = back;
    // elements c8 .. c8 + 7 are two k-steps' four of lane (row % 8, t4)
    const int half = c8 / (4 * Tr::LB), col = c8 % (4 * Tr::LB), t4 = col / Tr::LB;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int ks = half * (Tr::LB / 4) + (col % Tr::LB) / 4 + st;
      const uint32_t at = q_base + (((row >> 3) * Tr::KS + ks) * 32 + (row & 7) * 4 + t4) * 8;
      asm volatile("st.shared.v2.b32 [%0], {%1,%2};\n" ::"r"(at), "r"(w[2 * st]), "r"(w[2 * st + 1]) : "memory");
    }
  }
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}

template <class Tr, int CODE>
__global__ void __launch_bounds__(Tr::NTHREADS, Tr::RESIDENT)
kv8_decode_kernel(const __grid_constant__ Kv8Params p, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  constexpr int NG = Tr::NG, NQ = Tr::NQ, KS = Tr::KS, BN = Tr::BN, BM = Tr::BM, ST = Tr::ST, WN = Tr::WN, NCW = Tr::NCW, NCT = NCW * 32;
  constexpr int DT = Tr::HD / 16;  // 16-column tiles of the output
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_lse[BM];
  __shared__ int s_abort;
  __shared__ Kv8Seg s_seg;

  grid_wait();
  grid_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g8 = lane >> 2, t4 = lane & 3;

  const uint32_t raw = smem_u32(smem);
  const uint32_t pipe = (raw + 1023u) & ~1023u;
  uint8_t* smem_al = smem + (pipe - raw);
  float* slab = reinterpret_cast<float*>(smem_al + Tr::PIPE_BYTES);
  const uint32_t q_base = pipe + Tr::PIPE_BYTES;
  float2* ml = reinterpret_cast<float2*>(smem_al + Tr::PIPE_BYTES + Tr::TILE_BYTES);
  const uint32_t scales = q_base + Tr::TILE_BYTES + Tr::ML_BYTES;
  float* factor = reinterpret_cast<float*>(smem_al + Tr::PIPE_BYTES + Tr::TILE_BYTES + Tr::ML_BYTES + Tr::SC_BYTES);
  const uint32_t full0 = scales + Tr::SC_BYTES + BM * 4, empty0 = full0 + ST * 8;
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      tc5::mbar_init(full0 + s * 8, 33);    // the byte count's arrival, and every producer lane's when its scale has landed
      tc5::mbar_init(empty0 + s * 8, NCW);  // one arrival per consumer warp
    }
    s_abort = 0;
    tc5::fence_barrier_init();
  }
  if (warp == NCW && lane == 0) { tc5::tma_prefetch_desc(&tm_k); tc5::tma_prefetch_desc(&tm_v); }
  __syncthreads();

  const Kv8Mask mask = kv8_mask(p, lane);
  using Walk = Kv8Walk<BM, BN, 512 / BN>;  // a unit's fixed cost (Q load, merge of the warps, store) is worth about 512 keys
  if (warp == NCW) {
    // ================= producer warp =================
    Walk w;
    Kv8Seg sg;
    w.first(p, mask, lane, sg);
    uint32_t it_base = 0;
    while (sg.valid) {
      if (sg.valid == 1) {
        const Kv8Seq sq = kv8_seq(p, mask, sg.bi, 0, BM);
        if (sq.q_len > 0) {
          if (!kv8_producer<Tr>(p, sq, sg, &tm_k, &tm_v, pipe, scales, full0, empty0, it_base, lane, &s_abort)) break;
          it_base += (uint32_t)sg.cnt;
        }
      }
      w.next(p, mask, sg);
    }
  } else {
    // ================= consumer warps =================
    Walk w;
    if (warp == 0) {
      Kv8Seg sg;
      w.first(p, mask, lane, sg);
      if (lane == 0) s_seg = sg;
    }
    const int wm = warp / WN, wn = warp % WN;
    const uint32_t q_frag = q_base + wm * (NQ * KS * 256) + lane * 8;
    const bool to_partial = p.persistent || p.num_splits > 1, has_softcap = p.a.softcap > 0.f;
    const float sc_mul = has_softcap ? p.a.softmax_scale / p.a.softcap : p.a.softmax_scale * kLog2e;
    const float cap_l2 = p.a.softcap * kLog2e;
    uint32_t it_base = 0;
    for (;;) {
      asm volatile("bar.sync 1, %0;\n" ::"n"(NCT));  // the segment is published
      const Kv8Seg sg = s_seg;
      asm volatile("bar.sync 1, %0;\n" ::"n"(NCT));  // ... and read by everybody
      if (!sg.valid) break;
      const Kv8Seq sq = kv8_seq(p, mask, sg.bi, 0, BM);
      const int rows = min(BM, sq.q_len * p.group);  // (one tile holds all that a sequence may have)
      if (sg.valid == 1 && rows > 0) {
        const bool per_token = mask.causal || mask.local;
        if (p.a.dtype == FA_BF16) kv8_load_q<Tr, __nv_bfloat16>(p, sq, sg, q_base, factor, per_token, warp, lane);
        else kv8_load_q<Tr, __half>(p, sq, sg, q_base, factor, per_token, warp, lane);
        asm volatile("bar.sync 1, %0;\n" ::"n"(NCT));

        // lane (g8, t4): query rows 8 nq + 2 t4 + u (u = 0, 1) of this warp's, keys g8 and g8 + 8 of every 16
        float o_acc[DT][NQ][4], m_run[NQ][2], l_run[NQ][2], mul[NQ][2];
        int row_lo[NQ][2], row_hi[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_acc[dt][nq][e] = 0.f;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int r = (wm * NQ + nq) * 8 + 2 * t4 + u, i = r / p.group;
            int lo = 0, hi = sq.k_len - 1;
            if (mask.causal) hi = min(hi, i + sq.koff);
            if (mask.local) {
              hi = min(hi, i + sq.koff + mask.wr);
              lo = max(0, i + sq.koff - mask.wl);
            }
            row_lo[nq][u] = lo;
            row_hi[nq][u] = r < rows ? hi : -1;
            mul[nq][u] = factor[r] * sc_mul;
            m_run[nq][u] = -INFINITY;
            l_run[nq][u] = 0.f;
          }
        }
        uint32_t qf[Tr::Q_IN_REGS ? KS : 1][NQ][2];
        if (Tr::Q_IN_REGS) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) lds64(qf[ks][nq], q_frag + (nq * KS + ks) * 256);
        }
        // every row of the tile sees keys [all_lo, all_hi)
        const int i_last = (rows - 1) / p.group;
        int all_lo = 0, all_hi = sq.k_len;
        if (mask.causal) all_hi = min(all_hi, sq.koff + 1);
        if (mask.local) {
          all_hi = min(all_hi, sq.koff + mask.wr + 1);
          all_lo = max(0, i_last + sq.koff - mask.wl);
        }

        for (int it = 0; it < sg.cnt; ++it) {
          const uint32_t git = it_base + (uint32_t)it;
          const int stage = (int)(git % ST);
          if (!tc5::mbar_wait(full0 + stage * 8, (git / ST) & 1, &s_abort)) break;
          const uint32_t k_base = pipe + stage * Tr::STAGE_BYTES, v_base = k_base + Tr::KV_BYTES;
          const uint32_t sc = scales + stage * (2 * Tr::GROUPS * 4) + (wn * Tr::NW / kScaleGranule) * 4;
          const int t0 = (sg.lo + it) * BN, col0 = t0 + wn * Tr::NW;

          // [2 h + u]: key g8 + 8 h, row u.  At least four sums side by side: one product waits 30 cycles for the one before it.
          constexpr int PARTS = NG * NQ >= 4 ? 1 : 4 / (NG * NQ);
          float s_part[PARTS][NG][NQ][4], (&s_acc)[NG][NQ][4] = s_part[0];
#pragma unroll
          for (int pt = 0; pt < PARTS; ++pt)
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                for (int e = 0; e < 4; ++e) s_part[pt][g][nq][e] = 0.f;
#pragma unroll
          for (int cj = 0; cj < KS / 4; ++cj) {  // 16 bytes of a key row: four k-steps
            const int ch = Tr::ROWB == 128 ? (cj >> 1) * 8 + 2 * t4 + (cj & 1) : t4;
            uint32_t q2[4][NQ][2];
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq) {
                if (Tr::Q_IN_REGS) {
                  q2[s][nq][0] = qf[cj * 4 + s][nq][0];
                  q2[s][nq][1] = qf[cj * 4 + s][nq][1];
                } else {
                  lds64(q2[s][nq], q_frag + (nq * KS + cj * 4 + s) * 256);
                }
              }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              uint32_t ka[4], kb[4];
              lds128(ka, code_addr<Tr>(k_base, wn * Tr::NW + g * 16 + g8, ch));
              lds128(kb, code_addr<Tr>(k_base, wn * Tr::NW + g * 16 + 8 + g8, ch));
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                uint32_t a[4];
                decode4<CODE>(ka[s], a[0], a[2]);
                decode4<CODE>(kb[s], a[1], a[3]);
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) mma_16816<__half>(s_part[s % PARTS][g][nq], a, q2[s][nq][0], q2[s][nq][1]);
              }
            }
          }

#pragma unroll
          for (int pt = 1; pt < PARTS; ++pt)
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                for (int e = 0; e < 4; ++e) s_acc[g][nq][e] += s_part[pt][g][nq][e];

          // scores -> x (above), maximum, P'
          // (rows behind the tile's last one have Q = 0 and are never stored)
          const bool edge = t0 < all_lo || t0 + BN > all_hi || sg.masked;
          float inv[NG];
          float mx[NQ][2];
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) mx[nq][0] = mx[nq][1] = -INFINITY;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float ks_ = lds32f(sc + g * 4), vs = usable_scale(lds32f(sc + (Tr::GROUPS + g) * 4));
            const float lv = log2f(vs);
            inv[g] = 1.f / vs;
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int u = e & 1;
                float x = s_acc[g][nq][e];
                if (has_softcap) {
                  const float ex = __expf(2.f * (x * (ks_ * mul[nq][u])));
                  x = cap_l2 * (1.f - __fdividef(2.f, ex + 1.f)) + lv;
                } else {
                  x = fmaf(x, ks_ * mul[nq][u], lv);
                }
                if (edge) {
                  const int j = col0 + g * 16 + 8 * (e >> 1) + g8;
                  if (j < row_lo[nq][u] || j > row_hi[nq][u]) x = -INFINITY;
                }
                s_acc[g][nq][e] = x;
                mx[nq][u] = fmaxf(mx[nq][u], x);
              }
          }
          bool any_moved = false;
          float corr[NQ][2];
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float m = mx[nq][u];
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
              m = fmaxf(m_run[nq][u], m);
              const float m_use = m == -INFINITY ? 0.f : m - 15.f;
              const bool moved = m_run[nq][u] != m && m_run[nq][u] != -INFINITY;
              corr[nq][u] = moved ? fast_exp2(m_run[nq][u] - m) : 1.f;
              any_moved |= moved;
              m_run[nq][u] = m;
              float l = l_run[nq][u] * corr[nq][u];
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                const float p0 = fast_exp2(s_acc[g][nq][u] - m_use), p1 = fast_exp2(s_acc[g][nq][2 + u] - m_use);
                s_acc[g][nq][u] = p0;
                s_acc[g][nq][2 + u] = p1;
                l = fmaf(p0 + p1, inv[g], l);
              }
              l_run[nq][u] = l;
            }
          if (any_moved) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                for (int e = 0; e < 4; ++e) o_acc[dt][nq][e] *= corr[nq][e & 1];
          }

          // codes of keys that no row of the tile sees may be anything; 0 * NaN is NaN
          const bool cut = t0 < sq.key_lo || t0 + BN > sq.key_hi;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            uint32_t b[NQ][2];
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
              b[nq][0] = transpose_8x8(pack2<__half>(s_acc[g][nq][0], s_acc[g][nq][1]));
              b[nq][1] = transpose_8x8(pack2<__half>(s_acc[g][nq][2], s_acc[g][nq][3]));
            }
#pragma unroll
            for (int half = 0; half < Tr::HALVES; ++half) {
              uint32_t vw[4][4];  // key rows 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int row = wn * Tr::NW + g * 16 + 2 * t4 + (r & 1) + 8 * (r >> 1);
                if (Tr::ROWB == 128) lds128(vw[r], code_addr<Tr>(v_base, row, half * 8 + g8));
                else lds64(vw[r], code_addr<Tr>(v_base, row, g8 >> 1) + (g8 & 1) * 8);
                if (cut) {
                  const int j = t0 + row;
                  if (j < sq.key_lo || j >= sq.key_hi) {
#pragma unroll
                    for (int e = 0; e < Tr::VB / 4; ++e) vw[r][e] = 0;
                  }
                }
              }
#pragma unroll
              for (int e = 0; e < Tr::VB / 4; ++e) {
#pragma unroll
                for (int pr = 0; pr < 2; ++pr) {  // columns 4 e + 2 pr (tile row g8) and the next (tile row g8 + 8)
                  const uint32_t sel = pr == 0 ? 0x5140u : 0x7362u;
                  uint32_t a[4];
                  decode4<CODE>(__byte_perm(vw[0][e], vw[1][e], sel), a[0], a[1]);
                  decode4<CODE>(__byte_perm(vw[2][e], vw[3][e], sel), a[2], a[3]);
#pragma unroll
                  for (int nq = 0; nq < NQ; ++nq) mma_16816<__half>(o_acc[half * (Tr::VB / 2) + e * 2 + pr][nq], a, b[nq][0], b[nq][1]);
                }
              }
            }
          }
          __syncwarp();
          if (lane == 0) tc5::mbar_arrive(empty0 + stage * 8);
        }
        it_base += (uint32_t)sg.cnt;

        // ---- merge of the WN key slices and output ----
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float l = l_run[nq][u];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (g8 == 0) ml[wn * BM + (wm * NQ + nq) * 8 + 2 * t4 + u] = make_float2(m_run[nq][u], l);
          }
        asm volatile("bar.sync 1, %0;\n" ::"n"(NCT));
        float f_row[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int trow = (wm * NQ + nq) * 8 + 2 * t4 + u;
            float m_all = -INFINITY;
#pragma unroll
            for (int k = 0; k < WN; ++k) m_all = fmaxf(m_all, ml[k * BM + trow].x);
            const float m_use = m_all == -INFINITY ? 0.f : m_all;
            float l_all = 0.f;
#pragma unroll
            for (int k = 0; k < WN; ++k) {
              const float2 x = ml[k * BM + trow];
              l_all += x.y * fast_exp2(x.x - m_use);
            }
            // only a sum of exactly 0 means that the row saw no key: a NaN stays one
            f_row[nq][u] = l_all == 0.f ? 0.f : fast_exp2(m_run[nq][u] - m_use) / l_all;
            if (wn == 0 && g8 == 0) s_lse[trow] = l_all == 0.f ? -INFINITY : (m_use - 15.f + log2f(l_all)) * kLn2;
          }
        // Slice 0 stores, the others add in turn: a fixed order.  Tile dt of a half holds columns 2 dt and 2 dt + 1 of every lane group's VB.
#pragma unroll
        for (int half = 0; half < Tr::HALVES; ++half) {
#pragma unroll 1
          for (int turn = 0; turn < WN; ++turn) {
            if (wn == turn) {
#pragma unroll
              for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  float* dst = slab + ((wm * NQ + nq) * 8 + 2 * t4 + u) * Tr::SLAB_LD + g8 * Tr::VB;
                  const float f = f_row[nq][u];
#pragma unroll
                  for (int e4 = 0; e4 < Tr::VB / 4; ++e4) {
                    float4* q4 = reinterpret_cast<float4*>(dst + e4 * 4);
                    const int dt = half * (Tr::VB / 2) + e4 * 2;
                    float4 v = make_float4(o_acc[dt][nq][u] * f, o_acc[dt][nq][2 + u] * f, o_acc[dt + 1][nq][u] * f, o_acc[dt + 1][nq][2 + u] * f);
                    if (turn > 0) {
                      const float4 old = *q4;
                      v.x += old.x; v.y += old.y; v.z += old.z; v.w += old.w;
                    }
                    *q4 = v;
                  }
                }
            }
            asm volatile("bar.sync 1, %0;\n" ::"n"(NCT));
          }
          for (int c = tid; c < BM * (Tr::ROWB / 4); c += NCT) {
            const int trow = c / (Tr::ROWB / 4), s4 = (c % (Tr::ROWB / 4)) * 4, c4 = half * Tr::ROWB + s4;
            if (trow >= rows) continue;
            const int i = trow / p.group, head = sg.hk * p.group + (trow - i * p.group);
            const int64_t lse_idx = (int64_t)sg.bi * p.a.lse_batch_stride + (int64_t)head * p.a.lse_head_stride + sq.q_row0 + i;
            const float lse_row = s_lse[trow];
            const bool dead = lse_row == -INFINITY;
            if (c4 == 0) {
              if (to_partial) {
                p.lse_partial[(int64_t)sg.slot * p.lse_elems + lse_idx] = lse_row;
                for (int sl = sg.fill_from; sl < p.num_splits; ++sl) p.lse_partial[(int64_t)sl * p.lse_elems + lse_idx] = -INFINITY;
              } else {
                p.a.lse[lse_idx] = dead ? INFINITY : lse_row;
              }
            }
            if (c4 >= p.a.d || (dead && to_partial)) continue;
            const float4 acc = *reinterpret_cast<const float4*>(slab + trow * Tr::SLAB_LD + s4);
            if (to_partial) {
              *reinterpret_cast<float4*>(p.o_partial + ((int64_t)sg.slot * p.lse_elems + lse_idx) * p.a.d + c4) = acc;
            } else {
              uint2 w2;
              if (p.a.dtype == FA_BF16) {
                w2.x = pack2<__nv_bfloat16>(acc.x, acc.y);
                w2.y = pack2<__nv_bfloat16>(acc.z, acc.w);
              } else {
                w2.x = pack2<__half>(acc.x, acc.y);
                w2.y = pack2<__half>(acc.z, acc.w);
              }
              const int64_t off = (int64_t)sg.bi * p.a.o_batch_stride + (int64_t)(sq.q_row0 + i) * p.a.o_row_stride +
                                  (int64_t)head * p.a.o_head_stride + c4;
              *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.a.o) + off) = w2;
            }
          }
          if (half + 1 < Tr::HALVES) asm volatile("bar.sync 1, %0;\n" ::"n"(NCT));  // the rows are read: the next columns may come
        }
      }
      if (!p.persistent) break;
      if (warp == 0) {
        Kv8Seg nx;
        w.next(p, mask, nx);
        if (s_abort) nx.valid = 0;  // decided here, for all warps
        if (lane == 0) s_seg = nx;
      }
    }
  }

  __syncthreads();
  if (s_abort) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);  // let copies in flight land before the CTA retires
    if (tid == 0 && p.status) atomicExch(p.status, 0x40000000 | (int)blockIdx.x);
  }
}

}  // namespace fa
