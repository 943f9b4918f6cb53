"""CPU: refusals at the edges of the contract of the operators around an 8-bit KV cache, and the index arithmetic that keeps their kernels
within their tensors.  Nothing is launched."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

import flash_attn_npu_v3 as fa3
from flash_b200 import kv8
from flash_b200 import lib as L
from test_kv8_cpu import _fwd, _message

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-npu_b200", "csrc")


def _append(**change):
    """A call that nothing is wrong with (K and V, codes and scales in memory of their own), but for the changes."""
    p = L.Kv8AppendParams()
    p.k = p.v = p.slots = 256
    p.k_cache, p.v_cache = 1 << 20, 2 << 20
    p.k_tok_stride = p.v_tok_stride = 1024
    p.k_head_stride = p.v_head_stride = 128
    p.kc_outer_stride = p.vc_outer_stride = 128 * 1024
    p.kc_row_stride = p.vc_row_stride = 1024
    p.kc_head_stride = p.vc_head_stride = 128
    p.total, p.kv_outer, p.rows, p.h_k, p.d, p.dtype, p.num_sm = 10, 4, 128, 8, 128, L.FA_BF16, 148
    c = L.Kv8Cache()
    c.k_scale, c.v_scale = 3 << 20, 4 << 20
    c.ks_outer_stride = c.vs_outer_stride = 16
    c.ks_block_stride = c.vs_block_stride = 8
    c.ks_head_stride = c.vs_head_stride = 1
    c.scale_block, c.code = 64, L.CODE_E4M3
    for k, v in change.items():
        setattr(c if hasattr(c, k) else p, k, v)
    p.c = c
    return p


OVERLAPS = [dict(ks_outer_stride=0), dict(vs_outer_stride=0), dict(ks_block_stride=0), dict(vs_block_stride=0), dict(ks_head_stride=0),
            dict(vs_head_stride=0), dict(ks_outer_stride=0, ks_block_stride=0, ks_head_stride=0)]


@pytest.mark.parametrize("change", OVERLAPS + [dict(v_cache=1 << 20), dict(v_scale=3 << 20)])
def test_append_refuses_what_shares_memory(change):
    """Scales of several blocks or heads, or of K and of V, in one place: many would read and write it at once."""
    p = _append(**change)
    assert "of its own" in _message(L.load().fa_b200_kv8_append(C.byref(p), None))


@pytest.mark.parametrize("change", [dict(kc_outer_stride=0), dict(kc_row_stride=0), dict(vc_head_stride=0), dict(vc_row_stride=1032),
                                    dict(kc_head_stride=136), dict(kc_outer_stride=128 * 1024 + 8)])
def test_append_takes_the_strides_that_its_header_says(change):
    p = _append(**change)
    assert "multiples of 16" in _message(L.load().fa_b200_kv8_append(C.byref(p), None))


def _no_device(rc):
    """Every check has passed: what is missing is the GPU (this test launches nothing where there is one)."""
    return "device" in _message(rc)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch")
@pytest.mark.parametrize("change", [
    {}, dict(h_k=1, ks_head_stride=0, vs_head_stride=0, kc_head_stride=0), dict(kv_outer=1, ks_outer_stride=0, kc_outer_stride=0, vc_outer_stride=0),
    dict(scale_block=128, ks_block_stride=0, vs_block_stride=0)])
def test_append_strides_of_one_element_may_be_anything(change):
    assert _no_device(L.load().fa_b200_kv8_append(C.byref(_append(**change)), None))


def _fwd_new(**change):
    return _fwd(**{**dict(k=1 << 30, v=2 << 30, k_scale=3 << 20, v_scale=4 << 20, k_new=256, v_new=256, seqlen_new=1,
                          knew_batch_stride=1024, knew_row_stride=1024, knew_head_stride=128, vnew_batch_stride=1024, vnew_row_stride=1024,
                          vnew_head_stride=128, num_splits=1), **change})


@pytest.mark.parametrize("change", OVERLAPS + [dict(v=1 << 30), dict(v_scale=3 << 20)])
def test_new_tokens_refuse_what_shares_memory(change):
    p, c = _fwd_new(**change)
    assert "of its own" in _message(L.load().fa_b200_kv8_fwd(C.byref(p), C.byref(c), None, 0, None))


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch")
@pytest.mark.parametrize("change", OVERLAPS + [dict(v=256, k=256), dict(v_scale=256, k_scale=256)])
def test_expanded_scales_may_be_read(change):
    """A call without new tokens takes one scale for all blocks and heads, and one cache for K and V."""
    p, c = _fwd(num_splits=1, **change)
    assert _no_device(L.load().fa_b200_kv8_fwd(C.byref(p), C.byref(c), None, 0, None))


@pytest.mark.parametrize("change,said", [
    (dict(seqlen_q=1 << 30, lse_batch_stride=32 << 30, lse_head_stride=1 << 30), "too many query rows"),
    (dict(cu_seqlens_q=256, total_q=1 << 29, lse_head_stride=1 << 29), "too many query rows"),
    (dict(seqlen_k=(1 << 31) - 128, k_batch_stride=1 << 41, v_batch_stride=1 << 41, b=1, h=1, h_k=1, total_q=1), "too many tokens")])
def test_sizes_beyond_the_index_arithmetic_are_refused(change, said):
    p, c = _fwd(**change)
    assert said in _message(L.load().fa_b200_kv8_fwd(C.byref(p), C.byref(c), None, 0, None))


def test_caches_and_tables_that_are_too_small_are_refused():
    """A contiguous cache of fewer rows than sequences, a page table whose rows run into one another."""
    lib = L.load()
    for new in ({}, dict(k_new=256, v_new=256, seqlen_new=1)):
        p, c = _fwd(kv_outer=1, **new)
        assert "one row per sequence" in _message(lib.fa_b200_kv8_fwd(C.byref(p), C.byref(c), None, 0, None))
    p = L.KvcachePlanParams()
    for n in ("have", "add", "table", "free_pages", "slots", "cu_new", "after", "positions", "pages_taken"):
        setattr(p, n, 256)
    p.total, p.b, p.cols, p.page_size, p.n_free, p.num_sm = 4, 4, 16, 16, 8, 148
    for stride in (0, 15, -16):
        p.table_stride = stride
        assert "overlap" in _message(lib.fa_b200_kvcache_plan(C.byref(p), None))


def test_differentiable_calls_refuse_codes():
    q, kc, s = torch.zeros(2, 32, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 32, 2, 64, dtype=torch.int8), torch.ones(2, 1, 2)
    with pytest.raises(RuntimeError, match="does not support descale"):
        fa3.flash_attn_func(q, kc, kc, k_descale=s, v_descale=s)
    cu = torch.tensor([0, 32, 64], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="does not support descale"):
        fa3.flash_attn_varlen_func(q.flatten(0, 1), kc.flatten(0, 1), kc.flatten(0, 1), cu, cu, 32, 32, k_descale=s, v_descale=s)


def test_odd_strides_of_dimensions_of_one_element_are_put_right():
    base = torch.arange(4096, dtype=torch.float32).to(torch.bfloat16)
    for shape, strides in (((1, 1, 4, 64), (1001, 333, 64, 1)), ((2, 1, 1, 64), (128, 7, 3, 1)), ((1, 4, 64), (5, 64, 1))):
        t = torch.as_strided(base, shape, strides)
        a = kv8._aligned(t)
        assert torch.equal(a, t) and all(s % 8 == 0 for s in a.stride()[:-1]) and a.data_ptr() % 16 == 0
    t = base[:512].view(2, 4, 64)
    assert kv8._aligned(t) is t


RANDOM = r"""
#include <cstdio>
#include <initializer_list>
#include <limits>
#include <random>
#include "kv8_ranges.cuh"
std::mt19937 rng(5);
int any() {
  const int top = std::numeric_limits<int>::max(), low = std::numeric_limits<int>::min();
  switch (rng() % 6) {
    case 0: return 0;
    case 1: return top - (int)(rng() % 3);
    case 2: return low + (int)(rng() % 3);
    case 3: return (int)(rng() % 200);
    case 4: return -(int)(rng() % 200);
    default: return (int)rng();
  }
}
int held(int side) { return side < -(1 << 30) ? -(1 << 30) : side > (1 << 30) - 1 ? (1 << 30) - 1 : side; }
int some() { return any() & std::numeric_limits<int>::max(); }
"""


def _run(tmp_path, source):
    src, exe = tmp_path / "ranges.cpp", tmp_path / "ranges"
    src.write_text(RANDOM + source)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    subprocess.run([str(exe)], check=True)


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_query_rows_are_among_the_rows_there_are(tmp_path):
    """Whatever the offsets hold; and as given wherever that is possible."""
    _run(tmp_path, r"""
int main() {
  for (int round = 0; round < 400000; ++round) {
    const int total = round % 3 ? (int)(rng() % 100) : some(), from = any(), upto = any();
    int row0, len;
    const bool as_given = fa::kv8_query_rows(from, upto, total, row0, len), fine = from >= 0 && upto >= from && upto <= total;
    if (row0 < 0 || len < 0 || (long long)row0 + len > total || as_given != fine || (fine && (row0 != from || len != upto - from))) {
      std::printf("rows %d %d of %d: %d %d %d\n", from, upto, total, row0, len, (int)as_given);
      return 1;
    }
  }
  return 0;
}
""")


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_visible_keys_are_among_the_keys_there_are(tmp_path):
    """Whatever the window; and every key that a row sees is among them, counted one by one."""
    _run(tmp_path, r"""
int main() {
  for (int round = 0; round < 400000; ++round) {
    const bool wild = round % 2;
    const int k_len = wild ? some() / 2 : (int)(rng() % 40), q_len = wild ? 1 + some() / 4 : 1 + (int)(rng() % 12);
    fa::Kv8Mask m{};
    const int kind = (int)(rng() % 3);
    m.causal = kind == 1;
    m.local = kind == 2;
    m.wl = wild ? held(any()) : (int)(rng() % 24) - 6;
    m.wr = m.causal ? 0 : wild ? held(any()) : (int)(rng() % 24) - 6;
    const int i_lo = (int)(rng() % q_len), i_hi = i_lo + (int)(rng() % (q_len - i_lo)), koff = k_len - q_len;
    int lo, hi;
    fa::kv8_key_range(m, k_len, koff, i_lo, i_hi, lo, hi);
    if (lo < 0 || hi < lo || hi > k_len) {
      std::printf("keys %d, rows %d, window %d %d: [%d, %d)\n", k_len, q_len, m.wl, m.wr, lo, hi);
      return 1;
    }
    for (int i = i_lo; !wild && i <= i_hi; ++i)
      for (int j = 0; j < k_len; ++j) {
        const bool seen = m.causal ? j <= i + koff : m.local ? j >= i + koff - m.wl && j <= i + koff + m.wr : true;
        if (seen && (j < lo || j >= hi)) {
          std::printf("keys %d, rows %d, window %d %d: row %d key %d outside [%d, %d)\n", k_len, q_len, m.wl, m.wr, i, j, lo, hi);
          return 1;
        }
      }
  }
  return 0;
}
""")
