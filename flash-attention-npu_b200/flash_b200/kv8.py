"""Torch-facing launchers of the operators around a KV cache held in 8 bits (fa_b200_kv8_*, fa_b200_kvcache_plan).

A cache holds codes (``torch.float8_e4m3fn`` or ``torch.int8``) and fp32 scales, one for every (block of tokens, kv head) of K
and of V: an element stands for code * scale.  As in ``ops``, PyTorch is plumbing and there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import lib as L
from . import ops

INT32_MAX = 2 ** 31 - 1
CODES = {torch.float8_e4m3fn: L.CODE_E4M3, torch.int8: L.CODE_INT8}


def holds_codes(*caches) -> bool:
    return any(isinstance(t, torch.Tensor) and t.dtype in CODES for t in caches)


def _cache_block(k_cache, v_cache, k_descale, v_descale, like: Optional[torch.Tensor]) -> L.Kv8Cache:
    """Checks a cache and its scales; ``like``: the tensor whose device everything has to be on."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not t.is_cuda:
            raise RuntimeError("flash_b200 runs on CUDA tensors only (there is no CPU implementation)")
        if t.dtype not in CODES:
            raise RuntimeError(f"{name} must hold 8-bit codes (torch.float8_e4m3fn or torch.int8)")
        if t.dim() != 4 or t.stride(-1) != 1:
            raise RuntimeError(f"{name} must be (pages or rows, tokens, nheads_k, headdim) with a contiguous last dimension")
    if v_cache.dtype != k_cache.dtype or v_cache.shape != k_cache.shape:
        raise RuntimeError("k_cache and v_cache must have the same dtype and shape")
    outer, rows, h_k, _ = k_cache.shape
    for name, t in (("k_descale", k_descale), ("v_descale", v_descale)):
        if t is None:
            raise RuntimeError("an 8-bit KV cache needs k_descale and v_descale")
        if t.dtype != torch.float32 or not t.is_cuda or t.dim() != 3 or t.shape[0] != outer or t.shape[2] != h_k or t.shape[1] == 0:
            raise RuntimeError(f"{name} must be an fp32 tensor of shape (pages or rows, blocks of tokens, nheads_k)")
        if rows % t.shape[1] != 0 or (rows // t.shape[1]) % 16 != 0:
            raise RuntimeError(f"{name} must divide the cache's tokens into equal blocks of a multiple of 16")
    if k_descale.shape != v_descale.shape:
        raise RuntimeError("k_descale and v_descale must have the same shape")
    for t in (v_cache, k_descale, v_descale, like):
        if t is not None and t.device != k_cache.device:
            raise RuntimeError("the KV cache, its scales and the inputs must be on the same device")
    c = L.Kv8Cache()
    c.k_scale, c.v_scale = k_descale.data_ptr(), v_descale.data_ptr()
    c.ks_outer_stride, c.ks_block_stride, c.ks_head_stride = k_descale.stride()
    c.vs_outer_stride, c.vs_block_stride, c.vs_head_stride = v_descale.stride()
    c.scale_block, c.code = rows // k_descale.shape[1], CODES[k_cache.dtype]
    return c


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """The kernels read 16 bytes at a time; strides count for dimensions of one element too."""
    if t is None or (t.data_ptr() % 16 == 0 and t.stride(-1) == 1 and all(s % 8 == 0 for s in t.stride()[:-1])):
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def attention_forward_kv8(q, k_cache, v_cache, k_descale, v_descale, *, k_new=None, v_new=None, cu_seqlens_q=None, max_seqlen_q=None,
                          seqused_k=None, cache_batch_idx=None, block_table=None, rotary_cos=None, rotary_sin=None,
                          rotary_interleaved=True, softmax_scale=None, causal=False, window_left=-1, window_right=-1, softcap=0.0,
                          num_splits=0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of q over an 8-bit cache on the current stream: (out, lse) as ``ops.attention_forward`` returns them.
    k_new / v_new (b, s_new, h_k, d) are first appended (``append_kv8`` says how); the cache, the scales then change in place."""
    lib = L.load()
    if not q.is_cuda:
        raise RuntimeError("flash_b200 runs on CUDA tensors only (there is no CPU implementation)")
    ops._dtype_code(q)
    if q.dim() != (4 if cu_seqlens_q is None else 3):
        raise RuntimeError("q must be (batch, seqlen_q, nheads, headdim), or (total_q, nheads, headdim) with cu_seqlens_q")
    c = _cache_block(k_cache, v_cache, k_descale, v_descale, q)
    if q.shape[-1] != k_cache.shape[-1]:
        raise RuntimeError("query and KV cache must have the same head dimension")
    for name, t in (("cu_seqlens_q", cu_seqlens_q), ("cache_seqlens", seqused_k), ("cache_batch_idx", cache_batch_idx),
                    ("page_table", block_table)):
        ops._check_i32(t, name)
        if t is not None and t.device != q.device:
            raise RuntimeError(f"{name} must be on the device of q")
    b = q.shape[0] if cu_seqlens_q is None else cu_seqlens_q.numel() - 1
    for name, t in (("cache_seqlens", seqused_k), ("cache_batch_idx", cache_batch_idx)):
        if t is not None and (t.dim() != 1 or t.numel() != b or not t.is_contiguous()):
            raise RuntimeError(f"{name} must be a contiguous int32 tensor of shape (batch_size,)")
    if block_table is not None and (block_table.dim() != 2 or block_table.shape[0] != b):
        raise RuntimeError("page_table must have shape (batch_size, max_num_pages_per_seq)")
    if cu_seqlens_q is not None and max_seqlen_q is not None and int(max_seqlen_q) > INT32_MAX:
        raise RuntimeError("too many query rows in one call")
    if block_table is not None and block_table.shape[1] * k_cache.shape[1] > INT32_MAX:
        raise RuntimeError("too many tokens in a sequence's part of the KV cache")
    if block_table is None and cache_batch_idx is None and k_cache.shape[0] != b:
        raise RuntimeError("a contiguous KV cache needs one row per sequence, or cache_batch_idx")
    if (k_new is None) != (v_new is None):
        raise RuntimeError("k and v must be passed together")
    for name, t in (("k", k_new), ("v", v_new)):
        if t is not None and (t.dtype != q.dtype or t.device != q.device or t.dim() != 4 or t.shape[0] != b or
                              t.shape[1] != k_new.shape[1] or t.shape[2:] != k_cache.shape[2:]):
            raise RuntimeError(f"{name} must be (batch_size, seqlen_new, nheads_k, headdim) with the dtype and device of q")
    for name, t in (("rotary_cos", rotary_cos), ("rotary_sin", rotary_sin)):
        if t is not None and (t.dtype != q.dtype or t.device != q.device or t.dim() != 2 or not t.is_contiguous()):
            raise RuntimeError(f"{name} must be a contiguous 2-D tensor with the dtype and device of q")
    if rotary_cos is not None and rotary_sin is not None and rotary_cos.shape != rotary_sin.shape:
        raise RuntimeError("rotary_cos and rotary_sin must have the same shape")
    # Python's numbers, in the 32 bits that they go into: a window beyond is as wide as one can be
    window_left, window_right, num_splits = (max(-INT32_MAX, min(INT32_MAX, int(x))) for x in (window_left, window_right, num_splits))
    q, k_new, v_new = _aligned(q), _aligned(k_new), _aligned(v_new)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(ops._lse_shape(q, cu_seqlens_q is not None), dtype=torch.float32, device=q.device)
    with torch.cuda.device(q.device):
        p = ops.build_params(q, k_cache, v_cache, out, lse, k_new=k_new, v_new=v_new, cu_seqlens_q=cu_seqlens_q,
                             max_seqlen_q=max_seqlen_q, seqused_k=seqused_k, cache_batch_idx=cache_batch_idx,
                             block_table=block_table, rotary_cos=rotary_cos, rotary_sin=rotary_sin,
                             rotary_interleaved=rotary_interleaved,
                             softmax_scale=q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale, causal=causal,
                             window_left=window_left, window_right=window_right, softcap=softcap, num_splits=num_splits,
                             num_sm=ops._num_sm(q.device))
        nbytes = lib.fa_b200_kv8_fwd_workspace(C.byref(p), C.byref(c))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        L.check(lib.fa_b200_kv8_fwd(C.byref(p), C.byref(c), ops._ptr(ws), nbytes, torch.cuda.current_stream(q.device).cuda_stream))
    return out, lse


def append_kv8(k, v, k_cache, v_cache, k_descale, v_descale, slot_mapping) -> None:
    """k, v (total, h_k, d) -> codes at ``slot_mapping`` (total,) int64 of an 8-bit cache, and the scales of the blocks they
    fall into, in place (fa_b200_kv8_append)."""
    lib = L.load()
    if not k.is_cuda:
        raise RuntimeError("flash_b200 runs on CUDA tensors only (there is no CPU implementation)")
    p = L.Kv8AppendParams()
    p.dtype = ops._dtype_code(k)
    p.c = _cache_block(k_cache, v_cache, k_descale, v_descale, k)
    if k.dim() != 3 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device or k.shape[1:] != k_cache.shape[2:]:
        raise RuntimeError("k and v must be (total, nheads_k, headdim), of one dtype and on the device of the cache")
    if (slot_mapping.dtype != torch.int64 or slot_mapping.device != k.device or slot_mapping.dim() != 1 or
            slot_mapping.numel() != k.shape[0] or not slot_mapping.is_contiguous()):
        raise RuntimeError("slot_mapping must be a contiguous int64 tensor of shape (total,) on the device of k")
    k, v = _aligned(k), _aligned(v)
    p.k, p.v, p.k_cache, p.v_cache, p.slots = (t.data_ptr() for t in (k, v, k_cache, v_cache, slot_mapping))
    p.k_tok_stride, p.k_head_stride, _ = k.stride()
    p.v_tok_stride, p.v_head_stride, _ = v.stride()
    p.kc_outer_stride, p.kc_row_stride, p.kc_head_stride, _ = k_cache.stride()
    p.vc_outer_stride, p.vc_row_stride, p.vc_head_stride, _ = v_cache.stride()
    p.total, p.h_k, p.d = k.shape
    p.kv_outer, p.rows = k_cache.shape[:2]
    p.num_sm = ops._num_sm(k.device)
    with torch.cuda.device(k.device):
        L.check(lib.fa_b200_kv8_append(C.byref(p), torch.cuda.current_stream(k.device).cuda_stream))


def kvcache_plan(cache_seqlens, new_seqlens, page_table, free_pages, page_size, total_new, num_free=None):
    """One step's pages, slots, offsets and positions (fa_b200_kvcache_plan); ``page_table`` changes in place.
    Returns (slot_mapping, cu_seqlens_new, cache_seqlens afterwards, positions, pages taken)."""
    lib = L.load()
    if not page_table.is_cuda:
        raise RuntimeError("flash_b200 runs on CUDA tensors only (there is no CPU implementation)")
    dev, b = page_table.device, cache_seqlens.numel()
    for name, t in (("cache_seqlens", cache_seqlens), ("new_seqlens", new_seqlens), ("free_pages", free_pages), ("num_free", num_free)):
        if t is not None and (t.dtype != torch.int32 or t.device != dev or not t.is_contiguous() or t.dim() != 1):
            raise RuntimeError(f"{name} must be a contiguous 1-D int32 tensor on the device of page_table")
    if new_seqlens.numel() != b or (num_free is not None and num_free.numel() != 1):
        raise RuntimeError("new_seqlens must have shape (batch_size,) and num_free shape (1,)")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != b or page_table.stride(1) != 1 or (
            b > 1 and page_table.stride(0) < page_table.shape[1]):
        raise RuntimeError("page_table must be an int32 tensor of shape (batch_size, max_num_pages_per_seq) whose rows do not overlap")
    total, page_size = int(total_new), int(page_size)
    if total < 0:
        raise RuntimeError("total_new must not be negative")
    if not 0 < page_size <= INT32_MAX or total > INT32_MAX:
        raise RuntimeError("bad sizes of the page table, the free list or the packed batch")
    i32 = dict(dtype=torch.int32, device=dev)
    slots, positions = torch.empty(total, dtype=torch.int64, device=dev), torch.empty(total, **i32)
    cu, after, taken = torch.empty(b + 1, **i32), torch.empty(b, **i32), torch.empty(1, **i32)
    p = L.KvcachePlanParams()
    p.have, p.add, p.table, p.free_pages = (t.data_ptr() for t in (cache_seqlens, new_seqlens, page_table, free_pages))
    p.num_free = ops._ptr(num_free)
    p.slots, p.cu_new, p.after, p.positions, p.pages_taken = (t.data_ptr() for t in (slots, cu, after, positions, taken))
    p.table_stride, p.total = page_table.stride(0), total
    p.b, p.cols, p.page_size, p.n_free = b, page_table.shape[1], page_size, free_pages.numel()
    p.num_sm = ops._num_sm(dev)
    with torch.cuda.device(dev):
        L.check(lib.fa_b200_kvcache_plan(C.byref(p), torch.cuda.current_stream(dev).cuda_stream))
    return slots, cu, after, positions, taken
