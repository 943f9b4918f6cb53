"""CPU: the operators around a KV cache held in 8 bits -- struct layout, refusals, plans and traced shapes.  Nothing is launched."""
import ctypes as C

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import flash_attn_npu_v3 as fa3
import kv8_util as U
from flash_b200 import lib as L


def test_struct_layout_matches_header():
    # sizes produced by gcc for include/fa_b200.h (x86-64 LP64)
    assert C.sizeof(L.Kv8Cache) == 72
    assert C.sizeof(L.Kv8AppendParams) == 224
    assert C.sizeof(L.KvcachePlanParams) == 120


def _fwd(**kw):
    p = L.FwdParams()
    p.q = p.k = p.v = p.o = p.lse = 256
    p.b, p.seqlen_q, p.seqlen_k, p.h, p.h_k, p.d = 2, 1, 4096, 32, 8, 128
    p.total_q = 2
    p.q_head_stride = p.o_head_stride = 128
    p.q_row_stride = p.o_row_stride = p.q_batch_stride = p.o_batch_stride = 32 * 128
    p.k_head_stride = p.v_head_stride = 128
    p.k_row_stride = p.v_row_stride = 8 * 128
    p.k_batch_stride = p.v_batch_stride = 4096 * 8 * 128
    p.lse_batch_stride, p.lse_head_stride = 32, 1
    p.seqused_k = 256
    p.dtype, p.num_sm, p.softmax_scale = L.FA_BF16, 148, 0.088
    p.max_seqlen_k_known = p.window_left = p.window_right = -1
    c = L.Kv8Cache()
    c.k_scale = c.v_scale = 256
    c.ks_outer_stride = c.vs_outer_stride = 32 * 8
    c.ks_block_stride = c.vs_block_stride = 8
    c.ks_head_stride = c.vs_head_stride = 1
    c.scale_block, c.code = 128, L.CODE_E4M3
    for k, v in kw.items():
        setattr(c if hasattr(c, k) else p, k, v)
    return p, c


def _message(rc):
    assert rc < 0
    return L.load().fa_b200_last_error().decode()


@pytest.mark.parametrize("change,said", [
    (dict(d=72), "multiple of 16"), (dict(d=272), "at most 256"), (dict(scale_block=24), "multiple of 16"),
    (dict(scale_block=0), "multiple of 16"), (dict(scale_block=96), "divide"), (dict(code=2), "e4m3 or int8"),
    (dict(k_scale=0), "scales"), (dict(h=12), "divide"), (dict(alibi_slopes=256), "alibi"), (dict(cu_seqlens_k=256), "cu_seqlens_k"),
    (dict(k_row_stride=1032), "16"), (dict(k=264), "16-byte"), (dict(q_row_stride=4100), "multiples of 8"),
    (dict(block_table=256, page_size=128), "kv_outer"), (dict(k_new=256, seqlen_new=1), "passed together"),
    (dict(k_new=256, v_new=256, seqlen_new=5000), "fit"), (dict(k_new=256, v_new=256, seqlen_new=1 << 30, seqlen_k=1 << 30), "too many new tokens"),
    (dict(rotary_cos=256, rotary_sin=256), "together with new"),
    (dict(k_new=256, v_new=256, seqlen_new=1, rotary_cos=256, rotary_sin=256, rotary_dim=128, rotary_seqlen=4095), "every position"),
    (dict(softcap=-1.0), "softcap"), (dict(partial_out=1), "partial"), (dict(lse_head_stride=2), "contiguous"), (dict(dtype=2), "FP16 and BF16")])
def test_attention_refusals(change, said):
    p, c = _fwd(**change)
    assert said in _message(L.load().fa_b200_kv8_fwd(C.byref(p), C.byref(c), None, 0, None))


def test_workspace_holds_the_partials():
    lib = L.load()
    p, c = _fwd(num_splits=4)
    assert lib.fa_b200_kv8_fwd_workspace(C.byref(p), C.byref(c)) == 4 * 2 * 32 * (128 + 1) * 4
    p, c = _fwd(num_splits=1)
    assert lib.fa_b200_kv8_fwd_workspace(C.byref(p), C.byref(c)) == 0
    p, c = _fwd(num_splits=4)
    assert "workspace" in _message(lib.fa_b200_kv8_fwd(C.byref(p), C.byref(c), None, 0, None))


@pytest.mark.parametrize("change,said", [
    (dict(d=24), "multiple of 16"), (dict(rows=100), "divide"), (dict(k=8), "16-byte"), (dict(k_tok_stride=100), "multiples of 8"),
    (dict(kc_row_stride=1028), "16"), (dict(dtype=5), "FP16 and BF16"), (dict(slots=0), "non-null"), (dict(total=-1), "sizes"),
    (dict(kv_outer=0), "sizes"), (dict(h_k=32768), "too many new tokens or heads"), (dict(kv_outer=1 << 25), "too many tokens in the KV cache")])
def test_append_refusals(change, said):
    p = L.Kv8AppendParams()
    p.k = p.v = p.k_cache = p.v_cache = p.slots = 256
    p.k_tok_stride = p.v_tok_stride = 1024
    p.k_head_stride = p.v_head_stride = 128
    p.kc_outer_stride = p.vc_outer_stride = 128 * 1024
    p.kc_row_stride = p.vc_row_stride = 1024
    p.kc_head_stride = p.vc_head_stride = 128
    p.total, p.kv_outer, p.rows, p.h_k, p.d, p.dtype, p.num_sm = 10, 4, 128, 8, 128, L.FA_BF16, 148
    _, p.c = _fwd()
    for k, v in change.items():
        setattr(p, k, v)
    assert said in _message(L.load().fa_b200_kv8_append(C.byref(p), None))


@pytest.mark.parametrize("change,said", [
    (dict(b=0), "positive"), (dict(b=L.PLAN_MAX_REQUESTS + 1), "16384"), (dict(page_size=0), "sizes"), (dict(total=-1), "sizes"),
    (dict(cols=1 << 20, page_size=1 << 12), "too many"), (dict(have=0), "null"), (dict(free_pages=0), "null")])
def test_plan_refusals(change, said):
    p = L.KvcachePlanParams()
    for n in ("have", "add", "table", "free_pages", "slots", "cu_new", "after", "positions", "pages_taken"):
        setattr(p, n, 256)
    p.table_stride, p.total, p.b, p.cols, p.page_size, p.n_free, p.num_sm = 16, 4, 4, 16, 16, 8, 148
    for k, v in change.items():
        setattr(p, k, v)
    assert said in _message(L.load().fa_b200_kvcache_plan(C.byref(p), None))


def test_host_tensors_are_refused():
    kc, s = torch.zeros(2, 32, 2, 64, dtype=torch.int8), torch.ones(2, 1, 2)
    q, k = torch.zeros(2, 1, 4, 64, dtype=U.BF), torch.zeros(3, 2, 64, dtype=U.BF)
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fa3.flash_attn_with_kvcache(q, kc, kc, cache_seqlens=i32, k_descale=s, v_descale=s)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fa3.quantized_kvcache_append(k, k, kc, kc, s, s, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fa3.paged_kvcache_plan(i32, i32, torch.zeros(2, 4, dtype=torch.int32), i32, 16, 3)


def test_traced_shapes():
    """The registered operators say their results' shapes without running."""
    with FakeTensorMode():
        new = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
        kc, s = new((9, 32, 2, 64), U.E4M3), new((9, 2, 2), torch.float32)
        lens, table = new((3,), torch.int32), new((3, 5), torch.int32)
        q, k = new((3, 2, 8, 64), U.BF), new((3, 2, 2, 64), U.BF)
        for new_tokens in (None, k):
            out, lse, *_ = fa3.flash_attn_with_kvcache(q, kc, kc, new_tokens, new_tokens, cache_seqlens=lens, page_table=table, k_descale=s,
                                                       v_descale=s, return_softmax_lse=True)
            assert out.shape == q.shape and out.dtype == U.BF and lse.shape == (3, 8, 2)
        slots, cu, after, pos, taken = fa3.paged_kvcache_plan(lens, lens, table, new((40,), torch.int32), 32, 17)
        assert slots.shape == pos.shape == (17,) and slots.dtype == torch.int64
        assert cu.shape == (4,) and after.shape == (3,) and taken.shape == (1,)
        assert fa3.quantized_kvcache_append(new((17, 2, 64), U.BF), new((17, 2, 64), U.BF), kc, kc, s, s, slots) is None


def test_plain_forms():
    """The oracle's own pieces, at values worked out by hand."""
    assert U.scale_for(448.0, U.E4M3) == 1.0 and U.scale_for(448.5, U.E4M3) == 2.0 and U.scale_for(0.0, U.E4M3) == 2.0 ** -40
    assert U.scale_for(127.0, U.INT8) == 1.0 and U.scale_for(63.6, U.INT8) == 1.0 and U.scale_for(63.5, U.INT8) == 0.5
    x = torch.tensor([17.0, 19.0, 500.0, -0.0009765625, 0.0029296875, float("nan")], dtype=torch.float64)
    got = U.values_of(U.nearest(x, U.E4M3))
    assert got[:5].tolist() == [16.0, 20.0, 448.0, 0.0, 0.00390625] and bool(got[5].isnan())
    assert U.nearest(torch.tensor([0.5, 1.5, -2.5, 300.0, float("nan")], dtype=torch.float64), U.INT8).tolist() == [0, 2, -2, 127, 0]
    table = [[7, 0, 0], [5, 6, 0]]
    slots, cu, after, pos, taken = U.plan([4, 7], [3, 2], table, [9, 8], 4, 6)
    assert table == [[7, 9, 0], [5, 6, 8]] and slots == [36, 37, 38, 27, 32, -1] and cu == [0, 3, 5] and after == [7, 9]
    assert pos == [4, 5, 6, 7, 8, 0] and taken == [2]
