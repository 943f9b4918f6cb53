// Host side of the 8-bit KV cache's entry points: validation, planning, launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <string>

#include "kv8_api.cuh"
#include "tc5_api.cuh"

namespace fa {

// api.cu
int fail_bwd(int code, const std::string& msg);
void count_launches(int n);
int merge_partials(const fa_combine_params& c, const int32_t* rows_end, cudaStream_t st);
void window_rule(int seqlen_q, int max_k, bool causal, int& wl, int& wr, bool& is_causal, bool& is_local);
int sm_count();
void clear_error();

static int fail(int code, const std::string& msg) { return fail_bwd(code, msg); }
static int cuda_fail(const char* what, cudaError_t e) { return fail(FA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e)); }

static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int check_cache(const fa_kv8_cache& c, int rows, int d) {
  if (!c.k_scale || !c.v_scale) return fail(FA_ERR_INVALID, "an 8-bit KV cache needs the scales of K and of V");
  if (c.code != FA_CODE_E4M3 && c.code != FA_CODE_INT8) return fail(FA_ERR_INVALID, "an 8-bit KV cache holds e4m3 or int8 codes");
  if (d <= 0 || d > 256 || d % 16 != 0)
    return fail(FA_ERR_INVALID, "an 8-bit KV cache needs a head dimension that is a multiple of 16 and at most 256");
  if (c.scale_block <= 0 || c.scale_block % kScaleGranule != 0)
    return fail(FA_ERR_INVALID, "the tokens of a scale block must be a multiple of 16");
  if (rows % c.scale_block != 0) return fail(FA_ERR_INVALID, "scale blocks must divide the rows of a page or of a cache row");
  return FA_OK;
}

// New tokens are written by many warps at once, each its block and head: scales that several of them share (expanded tensors), or that K and V
// share, would be read and written at the same time.  Reading such a cache is fine.
static int check_written(const fa_kv8_cache& c, const void* k, const void* v, int64_t outer, int rows, int h_k) {
  auto shared = [&](int64_t by_outer, int64_t by_block, int64_t by_head) {
    return (outer > 1 && by_outer == 0) || (rows > c.scale_block && by_block == 0) || (h_k > 1 && by_head == 0);
  };
  if (k == v || c.k_scale == c.v_scale || shared(c.ks_outer_stride, c.ks_block_stride, c.ks_head_stride) ||
      shared(c.vs_outer_stride, c.vs_block_stride, c.vs_head_stride))
    return fail(FA_ERR_INVALID, "new tokens need a KV cache in which each of K, V and the scales has memory of its own");
  return FA_OK;
}

struct Kv8Plan {
  Kv8Params p;
  Kv8TileInfo tile;
  int hd, grid;
  bool tiled;
  size_t lse_bytes, workspace_bytes;
};

static int make_kv8_plan(const fa_fwd_params& a_in, const fa_kv8_cache& c, Kv8Plan* out) {
  std::memset(out, 0, sizeof(*out));
  fa_fwd_params a = a_in;
  if (a.b <= 0) return fail(FA_ERR_INVALID, "batch size must be positive");
  if (a.dtype != FA_FP16 && a.dtype != FA_BF16) return fail(FA_ERR_INVALID, "FlashAttention only supports FP16 and BF16 data types");
  if (a.h <= 0 || a.h_k <= 0 || a.h % a.h_k != 0)
    return fail(FA_ERR_INVALID, "Number of heads in key/value must divide number of heads in query");
  if (a.seqlen_q < 0 || a.seqlen_k < 0) return fail(FA_ERR_INVALID, "negative sequence length");
  if (a.softcap < 0.f) return fail(FA_ERR_INVALID, "softcap must be non-negative (0.0 disables softcap)");
  if (a.num_splits < 0) return fail(FA_ERR_INVALID, "num_splits must be >= 0");
  if (a.cu_seqlens_k || a.alibi_slopes || a.kv_total || a.kv_pos_offset || a.partial_out)
    return fail(FA_ERR_UNSUPPORTED, "an 8-bit KV cache takes no cu_seqlens_k, alibi_slopes, sharded positions or partial output");
  if (a.block_table && a.page_size <= 0) return fail(FA_ERR_INVALID, "paged KV cache needs page_size > 0");
  if (a.block_table && !a.seqused_k) return fail(FA_ERR_INVALID, "paged KV cache needs the per-sequence key lengths");
  if (a.block_table && a.kv_outer <= 0) return fail(FA_ERR_INVALID, "paged KV cache needs kv_outer = the number of pages");
  if (a.cache_batch_idx && (a.block_table || a.kv_outer <= 0))
    return fail(FA_ERR_INVALID, "cache_batch_idx needs a contiguous cache and kv_outer = the number of cache rows");
  if (a.kv_outer < 0) return fail(FA_ERR_INVALID, "negative kv_outer");
  if (!a.block_table && !a.cache_batch_idx && a.kv_outer > 0 && a.kv_outer < a.b)
    return fail(FA_ERR_INVALID, "a contiguous KV cache needs one row per sequence, or cache_batch_idx");
  if ((a.k_new != nullptr) != (a.v_new != nullptr)) return fail(FA_ERR_INVALID, "k and v must be passed together");
  if (a.k_new && a.seqlen_new <= 0) return fail(FA_ERR_INVALID, "seqlen_new must be positive when k, v are given");
  if (!a.k_new && a.seqlen_new != 0) return fail(FA_ERR_INVALID, "seqlen_new given without k, v");
  if (a.k_new && !a.seqused_k) return fail(FA_ERR_INVALID, "appending k, v needs cache_seqlens");
  if ((2LL * a.seqlen_new / kScaleGranule + 4) * a.b * a.h_k > 0x3fffffffLL) return fail(FA_ERR_UNSUPPORTED, "too many new tokens in one call");
  if (a.seqlen_new > a.seqlen_k) return fail(FA_ERR_INVALID, "the new tokens do not fit into the KV cache");
  if ((a.rotary_cos != nullptr) != (a.rotary_sin != nullptr)) return fail(FA_ERR_INVALID, "rotary_cos and rotary_sin must be passed together");
  if (a.rotary_cos) {
    if (!a.k_new) return fail(FA_ERR_INVALID, "rotary embedding is only applied together with new k, v");
    if (a.rotary_dim <= 0 || a.rotary_dim % 16 != 0 || a.rotary_dim > a.d)
      return fail(FA_ERR_INVALID, "rotary_dim must be divisible by 16 and at most the head dimension");
    if (a.rotary_seqlen < a.seqlen_k) return fail(FA_ERR_INVALID, "rotary_cos / rotary_sin must have a row for every position of the cache");
  }
  // Rows, keys and window sides: sums and differences of two of them stay within 32 bits (kv8_ranges.cuh).
  const int64_t all_rows = (int64_t)std::max(a.seqlen_q, a.cu_seqlens_q ? a.total_q : 0) * (a.h / a.h_k);
  if (all_rows > 0x3fffffff) return fail(FA_ERR_UNSUPPORTED, "too many query rows in one call");
  if (a.seqlen_k > 1 << 30) return fail(FA_ERR_UNSUPPORTED, "too many tokens in a sequence's part of the KV cache");
  const int rows = a.block_table ? a.page_size : a.seqlen_k;
  const int64_t outer = a.kv_outer > 0 ? a.kv_outer : a.b;
  if (int rc = check_cache(c, rows, a.d); rc != FA_OK) return rc;
  if (a.h_k == 1) a.k_head_stride = a.v_head_stride = a.d;  // (the stride of a dimension of one element may be anything)
  if (outer == 1) a.k_batch_stride = (int64_t)rows * a.k_row_stride, a.v_batch_stride = (int64_t)rows * a.v_row_stride;
  auto ok16 = [&](int64_t s) { return s > 0 && s % 16 == 0; };
  if (!ok16(a.k_head_stride) || !ok16(a.k_row_stride) || !ok16(a.k_batch_stride) || !ok16(a.v_head_stride) || !ok16(a.v_row_stride) ||
      !ok16(a.v_batch_stride) || !al16(a.k) || !al16(a.v))
    return fail(FA_ERR_UNSUPPORTED, "the codes of an 8-bit KV cache must start at 16-byte boundaries, with strides that are multiples of 16");
  auto ok8 = [](int64_t s) { return s % 8 == 0; };
  if (!al16(a.q) || !ok8(a.q_row_stride) || !ok8(a.q_head_stride) || !ok8(a.q_batch_stride) || !al16(a.k_new) || !al16(a.v_new) ||
      !ok8(a.knew_row_stride) || !ok8(a.knew_head_stride) || !ok8(a.knew_batch_stride) || !ok8(a.vnew_row_stride) ||
      !ok8(a.vnew_head_stride) || !ok8(a.vnew_batch_stride) || !al16(a.o) || !ok8(a.o_row_stride) || !ok8(a.o_head_stride) || !ok8(a.o_batch_stride))
    return fail(FA_ERR_UNSUPPORTED, "q, o and the new k, v must start at 16-byte boundaries, with strides that are multiples of 8");

  if (a.k_new)
    if (int rc = check_written(c, a.k, a.v, outer, rows, a.h_k); rc != FA_OK) return rc;

  Kv8Params& p = out->p;
  p.a = a;
  p.c = c;
  p.group = a.h / a.h_k;
  // ---- window ----
  int wl = a.window_left, wr = a.window_right, max_k = -1;
  if (!a.seqused_k) max_k = a.seqlen_k;
  else if (a.max_seqlen_k_known >= 0) max_k = a.max_seqlen_k_known + a.seqlen_new;
  if (max_k < 0) {
    if (wl >= 0 && wl >= a.seqlen_k - 1) max_k = a.seqlen_k;  // covers the longest sequence there can be
    else if (wl >= 0) p.wl_on_device = 1;
    if (max_k < 0) max_k = 0;
  }
  bool is_causal = false, is_local = false;
  window_rule(a.seqlen_q, max_k, a.causal != 0, wl, wr, is_causal, is_local);
  p.wl = std::clamp(wl, -(1 << 30), (1 << 30) - 1);  // (which is as wide as any)
  p.wr = std::clamp(wr, -(1 << 30), (1 << 30) - 1);

  // ---- tile and key splits ----
  const int rows_max = a.seqlen_q * p.group;
  out->hd = a.d <= 64 ? 64 : a.d <= 128 ? 128 : 256;
  out->tiled = rows_max > 32;  // (both sides measured: kv8_decode_kernel.cuh)
  out->tile = out->tiled ? kv8_tile_info(out->hd, rows_max > 128 && out->hd <= 128 ? 256 : 128) : kv8_decode_info(out->hd, rows_max <= 8 ? 8 : rows_max <= 16 ? 16 : 32);
  const Kv8TileInfo& t = out->tile;
  p.m_blocks = std::max(1, ceil_div(rows_max, t.block_m));
  p.box_rows = t.block_n;
  if (a.block_table && a.page_size % p.box_rows != 0) {
    p.box_rows &= -p.box_rows;  // a power of two divides the stage ...
    while (a.page_size % p.box_rows != 0) p.box_rows >>= 1;  // ... and the page (16 does)
  }
  long long range = a.seqlen_k;
  if (is_local && wl >= 0) range = std::min<long long>(range, (long long)wl + std::max(wr, 0) + ceil_div(t.block_m, p.group) + 1);
  const int max_blocks = std::max(1, std::min(ceil_div((int)range, t.block_n) + 1, ceil_div(a.seqlen_k, t.block_n)));
  const int num_sm = a.num_sm > 0 ? a.num_sm : sm_count();
  if (num_sm <= 0) return fail(FA_ERR_CUDA, "cannot query the SM count of the current device");
  const long long units = (long long)a.b * a.h_k * p.m_blocks, slots = (long long)num_sm * t.resident;
  if (units * max_blocks > 0x3fffffffLL) return fail(FA_ERR_UNSUPPORTED, "too many key blocks in one call");
  int ns = 1;
  if (a.num_splits >= 1) {
    ns = std::min(a.num_splits, max_blocks);
  } else if (p.m_blocks > 1) {
    // as many key ranges as fill the chip, of at least eight blocks each
    if (units < slots) ns = (int)std::max<long long>(1, std::min<long long>(slots / units, max_blocks / 8));
  } else if (max_blocks >= 4) {
    p.persistent = 1;
    // Partial slots of a unit.  They bound how finely the longest sequence is cut: with a slot for every CTA that an average unit gets, two
    // thirds of the chip waited for a sequence twice as long as the others.
    ns = (int)std::max<long long>(4, std::min<long long>(2 * slots / units + 3, max_blocks / 2 + 1));
  }
  if (!p.persistent) {
    p.blocks_per_split = ceil_div(max_blocks, ns);
    ns = ceil_div(max_blocks, p.blocks_per_split);
  }
  p.num_splits = ns;
  out->grid = (int)(p.persistent ? std::max(1LL, slots / a.h_k) * a.h_k : units * ns);
  const bool varlen = a.cu_seqlens_q != nullptr;
  p.lse_elems = varlen ? (int64_t)a.h * a.total_q : (int64_t)a.b * a.h * a.seqlen_q;
  if (p.lse_elems > 0 && (varlen ? a.lse_head_stride != a.total_q : (a.lse_head_stride != a.seqlen_q || a.lse_batch_stride != (int64_t)a.h * a.seqlen_q)))
    return fail(FA_ERR_INVALID, "lse must be contiguous");
  if (ns > 1) {
    out->lse_bytes = ((size_t)ns * p.lse_elems * sizeof(float) + 15) & ~(size_t)15;
    out->workspace_bytes = out->lse_bytes + (size_t)ns * p.lse_elems * a.d * sizeof(float);
  }
  return FA_OK;
}

static int run_kv8_fwd(const fa_fwd_params& a_in, const fa_kv8_cache& c, void* ws, size_t ws_bytes, void* (*alloc)(size_t, void*), void* ctx,
                       cudaStream_t st) {
  const bool no_rows = a_in.total_q == 0 || a_in.seqlen_q == 0;  // (new tokens are appended all the same)
  if (!a_in.k || !a_in.v || (!no_rows && (!a_in.q || !a_in.o || !a_in.lse))) return fail(FA_ERR_INVALID, "q, k, v, o and lse must be non-null");
  Kv8Plan P;
  if (int rc = make_kv8_plan(a_in, c, &P); rc != FA_OK) return rc;
  Kv8Params& p = P.p;
  const fa_fwd_params& a = p.a;
  if (P.workspace_bytes && !no_rows) {
    if (!ws && alloc) {
      ws = alloc(P.workspace_bytes, ctx);
      ws_bytes = ws ? P.workspace_bytes : 0;
    }
    if (!ws || ws_bytes < P.workspace_bytes) return fail(FA_ERR_WORKSPACE, "workspace missing or too small");
    if (!al16(ws)) return fail(FA_ERR_WORKSPACE, "workspace must be 16-byte aligned");
    p.lse_partial = static_cast<float*>(ws);
    p.o_partial = reinterpret_cast<float*>(static_cast<char*>(ws) + P.lse_bytes);
  }
  p.status = device_status_word();
  if (!p.status) return fail(FA_ERR_CUDA, "cannot look up the device status word");
  if (a.k_new) {
    const cudaError_t e = launch_kv8_append_dense(p, st);
    if (e != cudaSuccess) return cuda_fail("append launch", e);
    count_launches(1);
  }
  if (no_rows) return FA_OK;
  cudaError_t e;
  if (P.tiled) {
    const bool small = P.tile.block_m == 128;
    auto* launch = P.hd == 64    ? (small ? launch_kv8_tile_64_128 : launch_kv8_tile_64_256)
                   : P.hd == 128 ? (small ? launch_kv8_tile_128_128 : launch_kv8_tile_128_256)
                                 : launch_kv8_tile_256_128;
    e = launch(p, P.grid, st);
  } else {
    CUtensorMap tm_k, tm_v;
    const int64_t rows = a.block_table ? a.page_size : a.seqlen_k, outer = a.kv_outer > 0 ? a.kv_outer : a.b;
    const int box_cols = P.hd == 64 ? 64 : 128;
    if (!kv8_encode_map(&tm_k, a.k, a.d, a.h_k, rows, outer, a.k_head_stride, a.k_row_stride, a.k_batch_stride, box_cols, p.box_rows) ||
        !kv8_encode_map(&tm_v, a.v, a.d, a.h_k, rows, outer, a.v_head_stride, a.v_row_stride, a.v_batch_stride, box_cols, p.box_rows))
      return fail(FA_ERR_CUDA, "cuTensorMapEncodeTiled failed for the KV cache");
    const bool e4m3 = c.code == FA_CODE_E4M3;
    auto* launch = P.hd == 64    ? (e4m3 ? launch_kv8_decode_64_e4m3 : launch_kv8_decode_64_int8)
                   : P.hd == 128 ? (e4m3 ? launch_kv8_decode_128_e4m3 : launch_kv8_decode_128_int8)
                                 : (e4m3 ? launch_kv8_decode_256_e4m3 : launch_kv8_decode_256_int8);
    e = launch(P.tile.block_m, p, tm_k, tm_v, P.grid, st);
  }
  if (e != cudaSuccess) return cuda_fail("attention kernel launch", e);
  count_launches(1);
  if (p.num_splits == 1) return FA_OK;
  const bool varlen = a.cu_seqlens_q != nullptr;
  fa_combine_params m;
  std::memset(&m, 0, sizeof(m));
  m.o_partial = p.o_partial;
  m.lse_partial = p.lse_partial;
  m.o = a.o;
  m.lse = a.lse;
  m.num_splits = p.num_splits;
  m.b = varlen ? 1 : a.b;
  m.s = varlen ? a.total_q : a.seqlen_q;
  m.h = a.h;
  m.d = a.d;
  m.lp_split_stride = p.lse_elems;
  m.lp_batch_stride = m.lse_batch_stride = a.lse_batch_stride;
  m.lp_row_stride = m.lse_row_stride = 1;
  m.lp_head_stride = m.lse_head_stride = a.lse_head_stride;
  m.op_split_stride = p.lse_elems * a.d;
  m.op_batch_stride = a.lse_batch_stride * a.d;
  m.op_row_stride = a.d;
  m.op_head_stride = a.lse_head_stride * a.d;
  m.o_batch_stride = varlen ? 0 : a.o_batch_stride;
  m.o_row_stride = a.o_row_stride;
  m.o_head_stride = a.o_head_stride;
  m.out_dtype = a.dtype;
  return merge_partials(m, varlen ? a.cu_seqlens_q + a.b : nullptr, st);
}

static int run_kv8_append(const fa_kv8_append_params& p_in, cudaStream_t st) {
  fa_kv8_append_params p = p_in;
  if (p.total < 0 || p.h_k <= 0 || p.kv_outer <= 0 || p.rows <= 0) return fail(FA_ERR_INVALID, "bad sizes of the KV cache or the new tokens");
  if (p.dtype != FA_FP16 && p.dtype != FA_BF16) return fail(FA_ERR_INVALID, "FlashAttention only supports FP16 and BF16 data types");
  if (int rc = check_cache(p.c, p.rows, p.d); rc != FA_OK) return rc;
  if (p.total == 0) return FA_OK;
  if (!p.k || !p.v || !p.k_cache || !p.v_cache || !p.slots) return fail(FA_ERR_INVALID, "k, v, the caches and the slots must be non-null");
  if (p.h_k == 1) p.k_head_stride = p.v_head_stride = p.kc_head_stride = p.vc_head_stride = p.d;
  if (p.total == 1) p.k_tok_stride = p.v_tok_stride = 0;
  auto ok8 = [](int64_t s) { return s % 8 == 0; };
  if (!al16(p.k) || !al16(p.v) || !ok8(p.k_tok_stride) || !ok8(p.k_head_stride) || !ok8(p.v_tok_stride) || !ok8(p.v_head_stride))
    return fail(FA_ERR_UNSUPPORTED, "the new k, v must start at 16-byte boundaries, with strides that are multiples of 8");
  if (p.kv_outer == 1) p.kc_outer_stride = (int64_t)p.rows * p.kc_row_stride, p.vc_outer_stride = (int64_t)p.rows * p.vc_row_stride;
  auto ok16 = [](int64_t s) { return s > 0 && s % 16 == 0; };
  if (!al16(p.k_cache) || !al16(p.v_cache) || !ok16(p.kc_outer_stride) || !ok16(p.kc_row_stride) || !ok16(p.kc_head_stride) ||
      !ok16(p.vc_outer_stride) || !ok16(p.vc_row_stride) || !ok16(p.vc_head_stride))
    return fail(FA_ERR_UNSUPPORTED, "the codes of an 8-bit KV cache must start at 16-byte boundaries, with strides that are multiples of 16");
  if (p.total > 0x7fffffffLL || p.h_k > 32767) return fail(FA_ERR_UNSUPPORTED, "too many new tokens or heads in one call");
  if ((int64_t)p.kv_outer * p.rows > 0x7fffffffLL) return fail(FA_ERR_UNSUPPORTED, "too many tokens in the KV cache");
  if (int rc = check_written(p.c, p.k_cache, p.v_cache, p.kv_outer, p.rows, p.h_k); rc != FA_OK) return rc;
  const int num_sm = p.num_sm > 0 ? p.num_sm : sm_count();
  int32_t* status = device_status_word();
  if (!status || num_sm <= 0) return fail(FA_ERR_CUDA, "cannot query the current device");
  const cudaError_t e = launch_kv8_append(p, num_sm, status, st);
  if (e != cudaSuccess) return cuda_fail("append launch", e);
  count_launches(1);
  return FA_OK;
}

static int run_kvcache_plan(const fa_kvcache_plan_params& p, cudaStream_t st) {
  if (p.b <= 0) return fail(FA_ERR_INVALID, "batch size must be positive");
  if (p.b > FA_B200_PLAN_MAX_REQUESTS)
    return fail(FA_ERR_UNSUPPORTED, "a step has at most " + std::to_string(FA_B200_PLAN_MAX_REQUESTS) + " requests");
  if (p.page_size <= 0 || p.cols < 0 || p.n_free < 0 || p.total < 0 || p.total >= 0x7fffffffLL)
    return fail(FA_ERR_INVALID, "bad sizes of the page table, the free list or the packed batch");
  if ((int64_t)p.cols * p.page_size > 0x7fffffffLL) return fail(FA_ERR_UNSUPPORTED, "a row of the page table covers too many tokens");
  if (!p.have || !p.add || (!p.table && p.cols) || (!p.free_pages && p.n_free) || ((!p.slots || !p.positions) && p.total) || !p.cu_new || !p.after ||
      !p.pages_taken)
    return fail(FA_ERR_INVALID, "an input or output of the plan is null");
  if (p.b > 1 && p.table_stride < p.cols) return fail(FA_ERR_INVALID, "the rows of the page table must not overlap");
  const int num_sm = p.num_sm > 0 ? p.num_sm : sm_count();
  int32_t* status = device_status_word();
  if (!status || num_sm <= 0) return fail(FA_ERR_CUDA, "cannot query the current device");
  const cudaError_t e = launch_kvcache_plan(p, num_sm, status, st);
  if (e != cudaSuccess) return cuda_fail("plan launch", e);
  count_launches(1);
  return FA_OK;
}

}  // namespace fa

extern "C" {

int fa_b200_kv8_fwd(const fa_fwd_params* p, const fa_kv8_cache* c, void* workspace, size_t workspace_bytes, void* stream) {
  if (!p || !c) return fa::fail(FA_ERR_INVALID, "null params");
  fa::clear_error();
  return fa::run_kv8_fwd(*p, *c, workspace, workspace_bytes, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

size_t fa_b200_kv8_fwd_workspace(const fa_fwd_params* p, const fa_kv8_cache* c) {
  if (!p || !c) return 0;
  fa::clear_error();
  fa::Kv8Plan P;
  return fa::make_kv8_plan(*p, *c, &P) == FA_OK ? P.workspace_bytes : 0;
}

int fa_b200_kv8_fwd_alloc(const fa_fwd_params* p, const fa_kv8_cache* c, void* (*alloc)(size_t, void*), void* ctx, void* stream) {
  if (!p || !c || !alloc) return fa::fail(FA_ERR_INVALID, "null params");
  fa::clear_error();
  return fa::run_kv8_fwd(*p, *c, nullptr, 0, alloc, ctx, static_cast<cudaStream_t>(stream));
}

int fa_b200_kv8_append(const fa_kv8_append_params* p, void* stream) {
  if (!p) return fa::fail(FA_ERR_INVALID, "null params");
  fa::clear_error();
  return fa::run_kv8_append(*p, static_cast<cudaStream_t>(stream));
}

int fa_b200_kvcache_plan(const fa_kvcache_plan_params* p, void* stream) {
  if (!p) return fa::fail(FA_ERR_INVALID, "null params");
  fa::clear_error();
  return fa::run_kvcache_plan(*p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
