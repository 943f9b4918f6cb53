"""GPU: serving from a KV cache held in 8 bits -- step plan, quantising append, attention -- against plain forms in 64 bits."""
import ctypes as C
import math

import pytest
import torch

import flash_attn_npu_v3 as fa3
import kv8_util as U
from flash_b200 import kv8
from flash_b200 import lib as L
from flash_b200 import ops
from kv8_util import BF, E4M3, FP, INT8

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _raw(t):
    return t.contiguous().view(torch.uint8)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _status():
    L.check(L.load().fa_b200_check_status(torch.cuda.current_stream().cuda_stream))


# ---------------------------------------------------------------- plan
PLANS = [  # have, new, columns, free pages, page, rows of padding
    ([0], [1], 1, [3], 16, 0),
    ([5, 0, 16, 31], [1, 0, 1, 40], 8, list(range(20, 40)), 16, 3),
    ([0, 0, 0], [0, 0, 0], 2, [1, 2], 16, 0),                        # nobody brings anything
    ([0, 0, 0], [0, 0, 0], 2, [], 16, 2),                            # an empty free list that nobody needs
    ([100, 3, 60, 10], [200, 200, 4, 6], 8, [9, 8, 7, 6], 64, 1),     # the second request runs the list out
    ([15, 30, 7], [1, 40, 9], 4, list(range(9)), 16, 0),              # the second does not fit its row of the table
    ([1, 2, 3], [7, 1, 1], 3, [4, 5, 6, 7], 1, 0),                    # a page of one token
]


@pytest.mark.parametrize("have,new,cols,free,page,pad", PLANS)
def test_plan(have, new, cols, free, page, pad):
    total = sum(new) + pad
    wide = torch.full((len(have), cols + 3), -7, dtype=torch.int32)  # a table that is a view of a wider one
    wide[:, :cols] = torch.arange(len(have) * cols, dtype=torch.int32).view(-1, cols) + 100
    rows = wide[:, :cols].tolist()
    table = wide.cuda()
    got = fa3.paged_kvcache_plan(_i32(have), _i32(new), table[:, :cols], _i32(free), page, total)
    want = U.plan(have, new, rows, free, page, total)
    for g, w in zip(got, want):
        assert g.tolist() == w
    assert table[:, :cols].tolist() == rows and bool((table[:, cols:] == -7).all())
    _status()


@pytest.mark.parametrize("b,most", [(1, 3000), (257, 40), (3000, 7), (16384, 3)])
def test_plan_many(b, most):
    g = _gen(b)
    have = torch.randint(0, 500, (b,), generator=g)
    new = torch.randint(0, most, (b,), generator=g)
    cols, page = -(-(500 + most) // 32), 32
    rows = torch.arange(b * cols).view(b, cols).tolist()
    need = sum(-(-(a + n) // page) - -(-a // page) for a, n in zip(have.tolist(), new.tolist()))
    free = list(range(10 ** 6, 10 ** 6 + need + 5))
    total = int(new.sum()) + 11
    table = _i32(rows)
    # as many as are needed, or the last few too few: the count lives on the device
    for count in (need, need - 2):
        want_rows = [list(r) for r in rows]
        want = U.plan(have.tolist(), new.tolist(), want_rows, free[:count], page, total)
        table.copy_(_i32(rows))
        got = fa3.paged_kvcache_plan(_i32(have.tolist()), _i32(new.tolist()), table, _i32(free), page, total, _i32([count]))
        for g_, w in zip(got, want):
            assert g_.tolist() == w
        assert table.tolist() == want_rows


# ---------------------------------------------------------------- append
def _random_cache(g, outer, rows, h_k, d, blocks, dtype):
    code = torch.randint(0, 256, (outer, rows, h_k, d), generator=g, dtype=torch.uint8)
    if dtype == E4M3:
        code[(code & 127) == 127] = 60  # no NaN codes among the tokens that are there
    else:
        code[code == 128] = 0
    return code.view(dtype), torch.exp2(torch.randint(-6, 3, (outer, blocks, h_k), generator=g).float())


APPENDS = [  # tokens there and new ones of each sequence, page, scale block, h_k, d, type, codes
    ([0], [1], 16, 16, 1, 16, BF, E4M3),
    ([5, 0, 31], [1, 1, 1], 32, 16, 2, 64, BF, E4M3),
    ([5, 0, 31, 64], [9, 70, 1, 17], 64, 32, 3, 80, FP, INT8),
    ([100, 0], [300, 129], 128, 128, 2, 128, BF, INT8),
    ([3, 250], [40, 259], 256, 256, 1, 256, FP, E4M3),
    ([7] * 33, [2] * 33, 48, 48, 2, 96, BF, E4M3),
]


def _layout(have, new, page, g):
    """Pages of every sequence, and the slots of the new tokens in packed order."""
    per = [-(-(a + n) // page) for a, n in zip(have, new)]
    ids = torch.randperm(sum(per) + 2, generator=g).tolist()
    table, slots = [], []
    for n_pages, a, n in zip(per, have, new):
        mine, ids = ids[:n_pages], ids[n_pages:]
        table.append(mine)
        slots += [mine[t // page] * page + t % page for t in range(a, a + n)]
    return table, slots, sum(per) + 2


@pytest.mark.parametrize("have,new,page,sb,h_k,d,dtype,codes", APPENDS)
@pytest.mark.parametrize("odd", [False, True])
def test_append(have, new, page, sb, h_k, d, dtype, codes, odd):
    g = _gen(sum(have) + d)
    table, slots, pages = _layout(have, new, page, g)
    total = len(slots)
    want, scales = [], []
    x = [torch.randn((total, h_k, d), generator=g) * torch.exp2(torch.randint(-4, 9, (total, 1, 1), generator=g).float()) for _ in range(2)]
    if odd:  # values that have no code, none at all, next to none, and the largest
        x[0][0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 1.0])
        x[1][-1] = 0.0
        x[0][-1, -1] = 1e-30 if dtype == BF else 6e-8
        x[1][0, 0, 0] = 3e38 if dtype == BF else 65504.0
        x[1][total // 2, :, 3] = -math.inf
    x = [t.to(dtype) for t in x]
    kc, ks = _random_cache(g, pages, page, h_k, d, page // sb, codes)
    vc, vs = _random_cache(g, pages, page, h_k, d, page // sb, codes)
    # heads, pages and scales with strides of their own
    def strided(t, pad):
        big = torch.full(t.shape[:-2] + (t.shape[-2] + 1, t.shape[-1] + pad), 99, dtype=torch.uint8 if t.element_size() == 1 else t.dtype, device="cuda")
        v = big.view(t.dtype)[..., :t.shape[-2], :t.shape[-1]]
        v.copy_(t)
        return v, big
    (kcd, kbig), (vcd, _), (ksd, _), (vsd, _) = strided(kc, 16), strided(vc, 16), strided(ks, 1), strided(vs, 1)
    (kd, _), (vd, _) = strided(x[0], 8), strided(x[1], 8)
    before = kbig.clone()
    slots_pad = slots[:total // 2] + [-1, -1] + slots[total // 2:]
    def padded(t):  # rows of padding hold anything
        junk = torch.full((2,) + t.shape[1:], math.nan, dtype=t.dtype, device="cuda")
        return torch.cat([t[:total // 2], junk, t[total // 2:]])
    # (padding inside a block's run would cut it in two: only where the sequences meet)
    bounds = [sum(new[:r]) for r in range(len(new) + 1)]
    if total // 2 in bounds:
        fa3.quantized_kvcache_append(padded(kd), padded(vd), kcd, vcd, ksd, vsd, torch.tensor(slots_pad, device="cuda"))
    else:
        fa3.quantized_kvcache_append(kd, vd, kcd, vcd, ksd, vsd, torch.tensor(slots, device="cuda"))
    U.append(x[0], kc, ks, slots)
    U.append(x[1], vc, vs, slots)
    for got, want in ((ksd, ks), (vsd, vs)):
        assert torch.equal(got.cpu(), want)
    for got, want in ((kcd, kc), (vcd, vc)):
        a, b = U.values_of(got.cpu()), U.values_of(want)
        assert torch.equal(a.nan_to_num(1e9), b.nan_to_num(1e9)), int((a != b).sum())
    outside = torch.ones_like(kbig, dtype=torch.bool)
    outside[..., :h_k, :d] = False
    assert torch.equal(kbig[outside], before[outside])
    _status()


def test_append_nothing_and_only_padding():
    kc, ks = _random_cache(_gen(1), 3, 32, 2, 64, 2, E4M3)
    kd, sd = kc.cuda(), ks.cuda()
    for n in (0, 5):
        x = torch.ones((n, 2, 64), dtype=BF, device="cuda")
        fa3.quantized_kvcache_append(x, x, kd, kd.clone(), sd, sd.clone(), torch.full((n,), -1, dtype=torch.int64, device="cuda"))
    assert torch.equal(_raw(kd).cpu(), _raw(kc)) and torch.equal(sd.cpu(), ks)


# ---------------------------------------------------------------- attention
def _cache_for(g, lens, page, sb, h_k, d, codes, pow2=True, poison=True):
    """A cache with `lens` tokens in it: (codes, scales, table or None) on the host, what nobody owns full of NaN codes and
    NaN scales (int8: of the largest codes), and the 64-bit values of every sequence."""
    room = max(max(lens), 1)
    unit = page or sb
    per = -(-room // unit) * unit // unit
    outer = len(lens) * per + 1 if page else len(lens)
    rows = page or per * sb
    code = torch.full((outer, rows, h_k, d), 127, dtype=torch.uint8)
    scale = torch.full((outer, rows // sb, h_k), math.nan)
    table = torch.randperm(outer, generator=g)[:len(lens) * per].view(len(lens), per) if page else None
    values = []
    for r, n in enumerate(lens):
        x = torch.randn((n, h_k, d), generator=g, dtype=torch.float64) * torch.exp(torch.randn((1, h_k, 1), generator=g, dtype=torch.float64))
        got = torch.zeros((n, h_k, d), dtype=torch.float64)
        for b0 in range(0, n, sb):
            b1 = min(n, b0 + sb)
            o, i = (int(table[r, b0 // page]), b0 % page // sb) if page else (r, b0 // sb)
            x[b0:b1] *= 2.0 ** float(torch.randn((), generator=g))
            for h in range(h_k):
                amax = float(x[b0:b1, h].abs().max())
                s = torch.tensor(U.scale_for(amax, codes) if pow2 else amax / U.MOST[codes], dtype=torch.float32)
                c = U.nearest(x[b0:b1, h] / s.double(), codes)
                code[o, i * sb:i * sb + b1 - b0, h] = c.view(torch.uint8)
                scale[o, i, h] = s
                got[b0:b1, h] = U.values_of(c) * s.double()
        values.append(got)
    return code.view(codes), scale, (table.int() if table is not None else None), values


ATTEND = [  # s_q, keys of the sequences, h, h_k, d, page, sb, type, codes, mask
    (1, [1], 1, 1, 16, 16, 16, BF, E4M3, {}),
    (1, [0, 1, 17, 300], 4, 4, 64, 32, 16, FP, E4M3, dict(causal=True)),          # a sequence without keys
    (1, [2000, 5], 32, 8, 128, 128, 128, BF, E4M3, dict(causal=True)),
    (1, [129, 640, 64], 8, 1, 128, 0, 64, BF, INT8, {}),                           # contiguous, MQA
    (4, [3, 500, 130], 16, 2, 128, 64, 64, FP, INT8, dict(causal=True)),           # rows that see nothing
    (2, [700, 90], 12, 4, 96, 48, 48, BF, E4M3, dict(causal=True, softcap=20.0)),
    (1, [513, 31], 5, 1, 256, 16, 16, BF, E4M3, dict(causal=True)),
    (3, [400, 77], 8, 2, 192, 0, 32, FP, E4M3, dict(causal=True, window=(100, -1))),
    (2, [1500, 260], 64, 8, 128, 256, 64, BF, E4M3, dict(causal=True, window=(257, 0))),
    (5, [100, 33], 6, 2, 64, 32, 32, BF, INT8, dict(window=(40, 8))),
    (40, [40, 300], 4, 2, 64, 64, 16, FP, E4M3, dict(causal=True)),
    (129, [129, 1000], 8, 8, 128, 128, 64, BF, E4M3, dict(causal=True)),
    (200, [777, 200, 150], 6, 2, 80, 16, 16, FP, INT8, dict(causal=True)),         # the last has fewer keys than rows
    (300, [301], 2, 1, 256, 32, 32, BF, E4M3, {}),
    (130, [600], 16, 2, 128, 0, 128, BF, INT8, dict(causal=True, window=(64, -1), softcap=30.0)),
    (257, [1030], 7, 1, 64, 64, 64, BF, E4M3, dict(causal=True)),
]


@pytest.mark.parametrize("pow2", [True, False])
@pytest.mark.parametrize("s_q,lens,h,h_k,d,page,sb,dtype,codes,mask", ATTEND)
def test_attention(s_q, lens, h, h_k, d, page, sb, dtype, codes, mask, pow2):
    g = _gen(s_q * 1000 + d)
    kc, ks, table, kv = _cache_for(g, lens, page, sb, h_k, d, codes, pow2)
    vc, vs = kc.clone(), ks.clone()
    b = len(lens)
    vcode, vscale, _, vv = _cache_for(_gen(d + 7), lens, 0, sb, h_k, d, codes, pow2)  # values of their own, through the same table
    for r, n in enumerate(lens):
        for b0 in range(0, n, sb):
            b1 = min(n, b0 + sb)
            o, i = (int(table[r, b0 // page]), b0 % page // sb) if page else (r, b0 // sb)
            vc[o, i * sb:i * sb + b1 - b0] = vcode[r, b0:b1]
            vs[o, i] = vscale[r, b0 // sb]
    q = torch.randn((b, s_q, h, d), generator=g).to(dtype)
    scale = d ** -0.5
    out, lse, *_ = fa3.flash_attn_with_kvcache(
        q.cuda(), kc.cuda(), vc.cuda(), cache_seqlens=_i32(lens), page_table=table.cuda() if page else None, k_descale=ks.cuda(),
        v_descale=vs.cuda(), return_softmax_lse=True, causal=mask.get("causal", False), window_size=mask.get("window", (-1, -1)),
        softcap=mask.get("softcap", 0.0))
    is_causal, is_local, wl, wr = L.normalize_window(s_q, max(lens), mask.get("causal", False), *mask.get("window", (-1, -1)))
    for r, n in enumerate(lens):
        want = U.attend(q[r], kv[r], vv[r], scale, is_causal, (wl, wr) if is_local else None, mask.get("softcap", 0.0))
        U.check_attention(out[r], lse[r], want, mask.get("softcap", 0.0), f"sequence {r}")
    _status()


@pytest.mark.parametrize("q_lens,lens,h,h_k,d,dtype,codes", [
    ([1, 1, 1], [300, 1, 40], 8, 2, 128, BF, E4M3), ([3, 0, 16, 1], [900, 44, 16, 513], 16, 2, 64, FP, E4M3),
    ([1, 200, 37, 0, 90], [700, 333, 37, 12, 1200], 8, 2, 128, BF, INT8), ([300], [300], 4, 1, 256, FP, E4M3)])
def test_packed_queries(q_lens, lens, h, h_k, d, dtype, codes):
    g = _gen(sum(q_lens))
    kc, ks, table, kv = _cache_for(g, lens, 64, 32, h_k, d, codes)
    q = torch.randn((sum(q_lens), h, d), generator=g).to(dtype)
    cu = [sum(q_lens[:i]) for i in range(len(q_lens) + 1)]
    wide = torch.zeros((q.shape[0], h + 1, d + 8), dtype=dtype, device="cuda")  # rows and heads with strides of their own
    wide[:, :h, :d] = q
    out, lse, *_ = fa3.flash_attn_with_kvcache(
        wide[:, :h, :d], kc.cuda(), kc.cuda(), cache_seqlens=_i32(lens), page_table=table.cuda(), cu_seqlens_q=_i32(cu),
        max_seqlen_q=max(q_lens), k_descale=ks.cuda(), v_descale=ks.cuda(), causal=True, return_softmax_lse=True)
    assert out.shape == q.shape and lse.shape == (h, q.shape[0])
    for r, n in enumerate(lens):
        rows = slice(cu[r], cu[r + 1])
        U.check_attention(out[rows], lse[:, rows], U.attend(q[rows], kv[r], kv[r], d ** -0.5, True), tag=f"sequence {r}")


@pytest.mark.parametrize("splits", [1, 2, 5])
def test_key_splits_give_the_same(splits):
    g = _gen(9)
    kc, ks, table, kv = _cache_for(g, [1200, 100], 128, 128, 2, 128, E4M3)
    q = torch.randn((2, 1, 8, 128), generator=g).to(BF)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), kc.cuda(), cache_seqlens=_i32([1200, 100]), page_table=table.cuda(),
                                               k_descale=ks.cuda(), v_descale=ks.cuda(), num_splits=splits, return_softmax_lse=True)
    for r in range(2):
        U.check_attention(out[r], lse[r], U.attend(q[r], kv[r], kv[r], 128 ** -0.5), tag=f"{splits} splits")


def test_small_and_large_numbers():
    """Queries whose elements span bf16's range take part exactly; scales from 2^-40 to 2^30 within one sequence, zero scales
    and blocks of zeros among them; scores in the hundreds."""
    g = _gen(3)
    n, d = 512, 64
    kc, ks, table, _ = _cache_for(g, [n], 0, 16, 1, d, E4M3)
    vs = torch.exp2(torch.linspace(-40, 30, n // 16).round())[None, :, None]
    vs[0, 5] = 0.0
    vc = torch.randn((1, n, 1, d), generator=g).clamp(-3, 3).to(E4M3)
    vc[0, 48:64] = 0.0
    k64 = U.values_of(kc[0]) * ks[0].double().repeat_interleave(16, 0)[:, :, None]
    v64 = U.values_of(vc[0]) * vs[0].double().repeat_interleave(16, 0)[:, :, None]
    for up in (1.0, 2.0 ** 60, 2.0 ** -70):
        q = torch.randn((1, 1, 8, d), generator=g)
        q[0, 0, :, :8] *= 2.0 ** -12
        q = (q * up).to(BF)
        out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), vc.cuda(), cache_seqlens=_i32([n]), k_descale=ks.cuda(),
                                                   v_descale=vs.cuda(), softmax_scale=1.5 / up, return_softmax_lse=True)
        U.check_attention(out[0], lse[0], U.attend(q[0], k64, v64, 1.5 / up), tag=f"queries times {up}")


def test_nan_and_infinity():
    """A NaN among the keys or values reaches the rows that see it and no others; infinite queries make NaN."""
    g = _gen(4)
    kc, ks, table, kv = _cache_for(g, [200, 200, 200], 32, 32, 1, 64, E4M3)
    vc = kc.clone()
    kc.view(torch.uint8)[int(table[0, 1]), 3, 0, 5] = 127
    vc.view(torch.uint8)[int(table[1, 2]), 9, 0, 7] = 127
    q = torch.randn((3, 1, 4, 64), generator=g).to(BF)
    q[2, 0, 1, 0] = math.inf
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), vc.cuda(), cache_seqlens=_i32([200, 200, 200]), page_table=table.cuda(),
                                               k_descale=ks.cuda(), v_descale=ks.cuda(), return_softmax_lse=True)
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    gone = out[1].isnan()
    assert bool(gone[..., 7].all()) and int(gone.sum()) == 4 and bool(lse[1].isfinite().all())
    assert bool(out[2, :, 1].isnan().all()) and bool(out[2, :, [0, 2, 3]].isfinite().all())
    # behind a window they are not read: the same tokens, out of sight
    out, lse, *_ = fa3.flash_attn_with_kvcache(q[:2].cuda(), kc.cuda(), vc.cuda(), cache_seqlens=_i32([200, 200]), page_table=table[:2].cuda(),
                                               k_descale=ks.cuda(), v_descale=ks.cuda(), causal=True, window_size=(100, 0), return_softmax_lse=True)
    for r in range(2):
        U.check_attention(out[r], lse[r], U.attend(q[r], kv[r], kv[r], 64 ** -0.5, window=(100, 0)), tag=f"window, sequence {r}")


@pytest.mark.parametrize("s_new,lens,d,page,sb,dtype,codes,interleaved", [
    (1, [0, 15, 16, 100], 64, 32, 16, BF, E4M3, False), (3, [30, 0, 126], 128, 0, 64, FP, INT8, True),
    (200, [5, 90], 128, 64, 32, BF, E4M3, False), (2, [77], 256, 48, 16, FP, E4M3, True)])
def test_new_tokens(s_new, lens, d, page, sb, dtype, codes, interleaved):
    """k / v of the call: appended (k rotated first) as the append writes them, then attended to as the cache holds them."""
    g = _gen(s_new + d)
    b, h, h_k, rot = len(lens), 8, 2, d // 2
    after = [n + s_new for n in lens]
    kc, ks, table, _ = _cache_for(g, after, page, sb, h_k, d, codes)
    vc, vs = kc.clone(), ks.clone()
    room = (table.shape[1] * page) if page else kc.shape[1]
    angle = torch.rand((room, rot // 2), generator=g) * 6
    cos, sin = torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)
    q = torch.randn((b, s_new, h, d), generator=g).to(dtype)
    kn, vn = (torch.randn((b, s_new, h_k, d), generator=g).to(dtype) * 3 for _ in range(2))

    def rotate(x, pos):  # fp32 products rounded one by one, then to the type
        x = x.float()
        c, s = (t[pos].float()[:, None] for t in (cos, sin))
        r = x[..., :rot]
        x1, x2 = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
        y1, y2 = x1 * c - x2 * s, x1 * s + x2 * c
        y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
        return torch.cat([y, x[..., rot:]], -1).to(dtype)

    kcd, vcd, ksd, vsd = kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda()
    out, lse, *_ = fa3.flash_attn_with_kvcache(
        q.cuda(), kcd, vcd, kn.cuda(), vn.cuda(), cache_seqlens=_i32(lens), page_table=table.cuda() if page else None,
        rotary_cos=cos.cuda(), rotary_sin=sin.cuda(), rotary_interleaved=interleaved, k_descale=ksd, v_descale=vsd, causal=True,
        return_softmax_lse=True)
    for r, n in enumerate(lens):
        pos = list(range(n, n + s_new))
        slots = [int(table[r, t // page]) * page + t % page if page else r * kc.shape[1] + t for t in pos]
        U.append(rotate(kn[r], pos), kc, ks, slots)
        U.append(vn[r], vc, vs, slots)
    for got, want in ((kcd, kc), (vcd, vc)):
        a, w = U.values_of(got.cpu()), U.values_of(want)
        assert torch.equal(a.nan_to_num(1e9), w.nan_to_num(1e9))
    assert torch.equal(ksd.cpu().nan_to_num(9), ks.nan_to_num(9)) and torch.equal(vsd.cpu().nan_to_num(9), vs.nan_to_num(9))
    for r, n in enumerate(after):
        k64, v64 = (torch.stack([U.values_of(c[o, i]) * s[o, i // sb].double()[:, None] for o, i in (
            (int(table[r, t // page]), t % page) if page else (r, t) for t in range(n))]) for c, s in ((kc, ks), (vc, vs)))
        want = U.attend(rotate(q[r], list(range(n - s_new, n))), k64, v64, d ** -0.5, True)
        U.check_attention(out[r], lse[r], want, tag=f"sequence {r}")


def test_cache_rows_by_index():
    g = _gen(6)
    lens = [90, 200, 33]
    kc, ks, _, kv = _cache_for(g, [200, 33, 90, 10], 0, 32, 2, 64, E4M3)
    q = torch.randn((3, 1, 4, 64), generator=g).to(FP)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), kc.cuda(), cache_seqlens=_i32(lens), cache_batch_idx=_i32([2, 0, 1]),
                                               k_descale=ks.cuda(), v_descale=ks.cuda(), return_softmax_lse=True)
    for r, row in enumerate([2, 0, 1]):
        U.check_attention(out[r], lse[r], U.attend(q[r], kv[row], kv[row], 0.125), tag=f"row {row}")


def test_cache_beyond_32_bit_offsets():
    """A pool of more than 4 GB: its last pages are written and read at their own places."""
    page, h_k, d = 128, 8, 128
    pages = (5 << 30) // (page * h_k * d)
    kc = torch.zeros((pages, page, h_k, d), dtype=torch.uint8, device="cuda").view(E4M3)
    vc = torch.zeros((pages, page, h_k, d), dtype=torch.uint8, device="cuda").view(E4M3)
    ks, vs = (torch.zeros((pages, 1, h_k), dtype=torch.float32, device="cuda") for _ in range(2))
    g = _gen(8)
    n = 200
    mine = [pages - 1, pages - 3]
    x = [torch.randn((n, h_k, d), generator=g).to(BF) for _ in range(2)]
    slots = [mine[t // page] * page + t % page for t in range(n)]
    fa3.quantized_kvcache_append(x[0].cuda(), x[1].cuda(), kc, vc, ks, vs, torch.tensor(slots, device="cuda"))
    q = torch.randn((1, 1, 32, d), generator=g).to(BF)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc, vc, cache_seqlens=_i32([n]), page_table=_i32([mine]), k_descale=ks,
                                               v_descale=vs, return_softmax_lse=True)
    small = [torch.zeros((2, page, h_k, d), dtype=torch.uint8).view(E4M3) for _ in range(2)]
    sc = [torch.zeros((2, 1, h_k)) for _ in range(2)]
    v64 = []
    for i in range(2):
        U.append(x[i], small[i], sc[i], list(range(n)))
        v64.append((U.values_of(small[i]) * sc[i].double()[..., None]).flatten(0, 1)[:n])
    U.check_attention(out[0], lse[0], U.attend(q[0], v64[0], v64[1], d ** -0.5))
    assert int(_raw(kc[:pages - 3]).max()) == 0 and float(ks[:pages - 3].max()) == 0.0


# ---------------------------------------------------------------- together
class Server:
    """What a serving program keeps: pool, free list, table, lengths; and the same tokens in 64 bits on the host."""

    def __init__(self, b, pages, page, sb, h, h_k, d, dtype, codes, cols):
        self.page, self.h, self.h_k, self.d, self.dtype = page, h, h_k, d, dtype
        self.kc, self.vc = (torch.full((pages, page, h_k, d), 127, dtype=torch.uint8, device="cuda").view(codes) for _ in range(2))
        self.ks, self.vs = (torch.full((pages, page // sb, h_k), math.nan, device="cuda") for _ in range(2))
        self.table = torch.full((b, cols), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(b, dtype=torch.int32, device="cuda")
        self.free = torch.arange(pages, dtype=torch.int32).flip(0).contiguous().cuda()

    def step(self, q, k, v, new, most):
        """All on the device: no length is looked at here."""
        slots, cu, after, _, taken = fa3.paged_kvcache_plan(self.lens, new, self.table, self.free, self.page, k.shape[0])
        fa3.quantized_kvcache_append(k, v, self.kc, self.vc, self.ks, self.vs, slots)
        out, lse, *_ = fa3.flash_attn_with_kvcache(q, self.kc, self.vc, cache_seqlens=after, page_table=self.table, cu_seqlens_q=cu,
                                                   max_seqlen_q=most, k_descale=self.ks, v_descale=self.vs, causal=True, return_softmax_lse=True)
        return out, lse, after, taken


@pytest.mark.parametrize("dtype,codes,page,sb,d", [(BF, E4M3, 32, 32, 128), (FP, INT8, 64, 16, 64)])
def test_serving_steps(dtype, codes, page, sb, d):
    """Prompts of several lengths, then steps that mix decoding and a late prompt, against 64-bit attention over 64-bit copies of the
    tokens: what is off beyond the attention's own rounding is the codes' (each off by half a step of its code)."""
    g = _gen(d)
    b, h, h_k = 4, 8, 2
    srv = Server(b, 40, page, sb, h, h_k, d, dtype, codes, 12)
    host = [(torch.zeros((0, h_k, d), dtype=torch.float64), torch.zeros((0, h_k, d), dtype=torch.float64)) for _ in range(b)]
    table = [[-1] * 12 for _ in range(b)]
    kc, vc = srv.kc.cpu(), srv.vc.cpu()
    ks, vs = srv.ks.cpu(), srv.vs.cpu()
    lens, free = [0] * b, srv.free.tolist()
    for new in ([70, 5, 0, 200], [1, 1, 0, 1], [1, 1, 90, 1], [1, 1, 1, 1]):
        total = sum(new)
        q = torch.randn((total, h, d), generator=g).to(dtype)
        k, v = (torch.randn((total, h_k, d), generator=g).to(dtype) for _ in range(2))
        out, lse, after, taken = srv.step(q.cuda(), k.cuda(), v.cuda(), _i32(new), max(new))
        slots, cu, lens_after, _, n = U.plan(lens, new, table, free, page, total)
        U.append(k, kc, ks, slots)
        U.append(v, vc, vs, slots)
        assert after.tolist() == lens_after and taken.tolist() == n
        free, lens = free[n[0]:], lens_after
        srv.free, srv.lens = srv.free[n[0]:].contiguous(), after
        for r in range(b):
            rows = slice(cu[r], cu[r + 1])
            if new[r] == 0:
                continue
            pages = [(table[r][t // page], t % page) for t in range(lens[r])]
            k64, v64 = (torch.stack([U.values_of(c[o, i]) * s[o, i // sb].double()[:, None] for o, i in pages]) for c, s in ((kc, ks), (vc, vs)))
            U.check_attention(out[rows], lse[:, rows], U.attend(q[rows], k64, v64, d ** -0.5, True), tag=f"{new}, sequence {r}")
    assert torch.equal(U.values_of(srv.kc.cpu()).nan_to_num(1e9), U.values_of(kc).nan_to_num(1e9))
    _status()


def test_step_in_a_graph():
    """One captured step replayed with other lengths, tokens and tables gives what an eager one gives; another stream too."""
    g = _gen(12)
    b, h, h_k, d, page = 3, 8, 2, 128, 32
    most, total = 40, 64
    def fresh():
        srv = Server(b, 30, page, 32, h, h_k, d, BF, E4M3, 8)
        srv.kc.view(torch.uint8).zero_(), srv.vc.view(torch.uint8).zero_(), srv.ks.fill_(1.0), srv.vs.fill_(1.0)
        return srv
    q = torch.zeros((total, h, d), dtype=BF, device="cuda")
    k, v = (torch.zeros((total, h_k, d), dtype=BF, device="cuda") for _ in range(2))
    new = torch.zeros(b, dtype=torch.int32, device="cuda")
    srv = fresh()
    srv.step(q, k, v, new, most)  # loads everything
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse, after, taken = srv.step(q, k, v, new, most)
    eager = fresh()
    for step, lens_new in enumerate(([40, 3, 11], [1, 1, 1], [0, 30, 1], [1, 1, 1])):
        n = sum(lens_new)
        q.copy_(torch.randn((total, h, d), generator=g))
        k.copy_(torch.randn((total, h_k, d), generator=g))
        v.copy_(torch.randn((total, h_k, d), generator=g))
        new.copy_(_i32(lens_new))
        graph.replay()
        o2, l2, a2, t2 = eager.step(q, k, v, new, most)
        assert torch.equal(after, a2) and torch.equal(taken, t2) and torch.equal(srv.table, eager.table)
        assert torch.equal(out[:n], o2[:n]) and torch.equal(lse[:, :n], l2[:, :n])
        assert torch.equal(_raw(srv.kc), _raw(eager.kc)) and torch.equal(srv.ks, eager.ks) and torch.equal(srv.vs, eager.vs)
        for s, a in ((srv, after), (eager, a2)):
            s.lens.copy_(a)
            s.free.copy_(torch.roll(s.free, -int(t2)))


def test_streams_and_calls_at_once():
    """Two calls in flight on two streams, tensors made on a third: each is what it is alone, and again when repeated."""
    g = _gen(13)
    kc, ks, table, kv = _cache_for(g, [4000, 3000], 128, 64, 2, 128, E4M3)
    args = (kc.cuda(), kc.cuda())
    qs = [torch.randn((2, 1, 8, 128), generator=g).to(BF).cuda() for _ in range(2)]
    kw = dict(cache_seqlens=_i32([4000, 3000]), page_table=table.cuda(), k_descale=ks.cuda(), v_descale=ks.cuda(), return_softmax_lse=True)
    alone = [fa3.flash_attn_with_kvcache(q, *args, **kw)[:2] for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for st, q in zip(streams, qs):
            with torch.cuda.stream(st):
                got.append(fa3.flash_attn_with_kvcache(q, *args, **kw)[:2])
        torch.cuda.synchronize()
        for (o, l), (o1, l1) in zip(got, alone):
            assert torch.equal(o, o1) and torch.equal(l, l1)


@pytest.mark.parametrize("s_q,h,h_k,d,dtype,codes,mask", [
    (5, 16, 2, 64, BF, E4M3, dict(causal=True)), (16, 8, 1, 128, FP, INT8, {}), (6, 12, 2, 96, BF, INT8, dict(causal=True, window=(90, 0))),
    (9, 8, 2, 64, FP, E4M3, dict(softcap=15.0)), (33, 4, 2, 128, BF, E4M3, dict(window=(70, 20)))])
@pytest.mark.parametrize("b,most", [(3, 900), (110, 330)])
def test_between_decode_and_prompt(s_q, h, h_k, d, dtype, codes, mask, b, most):
    """33 to 128 rows of a kv head: key blocks of 64 in two streams.  Few long sequences, which CTAs share, and many short ones, several a
    CTA: one block, an odd number, none at all, a first block that falls to either stream."""
    g = _gen(s_q * 100 + b)
    lens = [0, 1, 64, 65, 129, 200][:b] + torch.randint(0, most, (max(0, b - 6),), generator=g).tolist()
    if b == 3:
        lens = [most, 0, most // 2 + 1]
    kc, ks, table, kv = _cache_for(g, lens, 32, 16, h_k, d, codes)
    q = torch.randn((b, s_q, h, d), generator=g).to(dtype)
    causal, window, cap = mask.get("causal", False), mask.get("window", (-1, -1)), mask.get("softcap", 0.0)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), kc.cuda(), cache_seqlens=_i32(lens), page_table=table.cuda(), k_descale=ks.cuda(),
                                               v_descale=ks.cuda(), causal=causal, window_size=window, softcap=cap, return_softmax_lse=True)
    is_causal, is_local, wl, wr = L.normalize_window(s_q, max(lens), causal, *window)
    for r in range(b):
        want = U.attend(q[r], kv[r], kv[r], d ** -0.5, is_causal, (wl, wr) if is_local else None, cap)
        U.check_attention(out[r], lse[r], want, cap, f"sequence {r} of {lens[r]}")
    _status()


@pytest.mark.parametrize("page,sb", [(160, 32), (48, 16), (320, 160), (64, 64), (16, 16), (0, 16)])
def test_pages_that_do_not_divide_a_stage(page, sb):
    """32 rows of 128 columns take stages of 160 keys: boxes of a page, of a part of it, of a whole stage."""
    g = _gen(page + 1)
    lens = [960, 481, 160, 1]
    kc, ks, table, kv = _cache_for(g, lens, page, sb, 2, 128, E4M3)
    q = torch.randn((4, 4, 16, 128), generator=g).to(BF)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), kc.cuda(), cache_seqlens=_i32(lens), page_table=table.cuda() if page else None,
                                               k_descale=ks.cuda(), v_descale=ks.cuda(), causal=True, return_softmax_lse=True)
    for r in range(4):
        U.check_attention(out[r], lse[r], U.attend(q[r], kv[r], kv[r], 128 ** -0.5, True), tag=f"sequence {r}")
    _status()


@pytest.mark.parametrize("s_q,h,where", [(8, 16, "k"), (8, 16, "v"), (40, 16, "k"), (40, 16, "v")])
@pytest.mark.parametrize("token", [3, 70, 299])
def test_nan_among_many_rows(s_q, h, where, token):
    """One NaN code, in a block of either stream: a key's reaches every row that sees it and no other; a value's the one column of every row
    that sees it -- and of others, where its weight is 0 and 0 * NaN is NaN, as in the formula."""
    g = _gen(token)
    kc, ks, table, kv = _cache_for(g, [300], 32, 32, 2, 64, E4M3)
    vc = kc.clone()
    (kc if where == "k" else vc).view(torch.uint8)[int(table[0, token // 32]), token % 32, 0, 5] = 127
    q = torch.randn((1, s_q, h, 64), generator=g).to(BF)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), vc.cuda(), cache_seqlens=_i32([300]), page_table=table.cuda(), causal=True,
                                               k_descale=ks.cuda(), v_descale=ks.cuda(), return_softmax_lse=True)
    sees = torch.arange(s_q) + 300 - s_q >= token
    gone = out[0].isnan().cpu()
    assert not bool(gone[:, h // 2:].any())
    if where == "k":
        assert not bool(gone[~sees].any()) and bool(gone[sees][:, :h // 2].all()) and bool(lse[0, :h // 2].cpu()[:, sees].isnan().all())
    else:
        assert bool(gone[sees][:, :h // 2, 5].all()) and int(gone.sum()) == int(gone[..., 5].sum())
        assert bool(lse.isfinite().all())
    rest = slice(h // 2, h)  # of the other kv head
    U.check_attention(out[0, :, rest], lse[0, rest], U.attend(q[0, :, rest], kv[0][:, 1:], kv[0][:, 1:], 64 ** -0.5, True))


@pytest.mark.parametrize("q_lens,h,splits", [([1, 0, 3], 8, 0), ([16, 3, 0], 16, 0), ([16, 3, 0], 16, 3), ([130, 5, 60], 8, 0), ([130, 5, 60], 8, 2)])
def test_rows_behind_the_last_sequence(q_lens, h, splits):
    """A padded batch: rows that belong to no sequence are left as they were, whatever is merged."""
    g = _gen(sum(q_lens))
    lens, d, pad = [700, 400, 90], 64, 5
    kc, ks, table, kv = _cache_for(g, lens, 64, 32, 2, d, E4M3)
    kc, ks, table = kc.cuda(), ks.cuda(), table.cuda()
    n = sum(q_lens)
    q = torch.randn((n + pad, h, d), generator=g).to(BF).cuda()
    cu = [sum(q_lens[:i]) for i in range(4)]
    out, lse = torch.full_like(q, 7.0), torch.full((h, n + pad), 7.0, device="cuda")
    c = kv8._cache_block(kc, kc, ks, ks, q)
    cu_t, lens_t = _i32(cu), _i32(lens)
    p = ops.build_params(q, kc, kc, out, lse, cu_seqlens_q=cu_t, max_seqlen_q=max(q_lens), seqused_k=lens_t, block_table=table, softmax_scale=d ** -0.5,
                         causal=True, window_left=-1, window_right=-1, softcap=0.0, num_splits=splits)
    lib = L.load()
    nbytes = lib.fa_b200_kv8_fwd_workspace(C.byref(p), C.byref(c))
    ws = torch.full((max(nbytes, 16),), 255, dtype=torch.uint8, device="cuda")  # (NaN wherever nothing is written)
    L.check(lib.fa_b200_kv8_fwd(C.byref(p), C.byref(c), ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream))
    assert bool((out[n:] == 7).all()) and bool((lse[:, n:] == 7).all())
    for r in range(3):
        rows = slice(cu[r], cu[r + 1])
        U.check_attention(out[rows], lse[:, rows], U.attend(q[rows].cpu(), kv[r], kv[r], d ** -0.5, True), tag=f"sequence {r}")


def test_new_tokens_without_queries():
    """A call with no query row still appends."""
    g = _gen(21)
    kc, ks, table, _ = _cache_for(g, [40, 70], 32, 32, 2, 64, E4M3)
    x = torch.randn((2, 3, 2, 64), generator=g).to(BF).cuda()
    table, lens = table.cuda(), _i32([37, 67])
    slots = torch.tensor([int(table[r, t // 32]) * 32 + t % 32 for r, n in enumerate((37, 67)) for t in range(n, n + 3)], device="cuda")
    state = [[kc.cuda(), kc.cuda(), ks.cuda(), ks.cuda()] for _ in range(2)]
    out = fa3.flash_attn_with_kvcache(torch.empty((2, 0, 4, 64), dtype=BF, device="cuda"), *state[0][:2], x, x, cache_seqlens=lens, page_table=table,
                                      k_descale=state[0][2], v_descale=state[0][3])
    fa3.quantized_kvcache_append(x.flatten(0, 1), x.flatten(0, 1), *state[1], slots)
    assert out.shape == (2, 0, 4, 64)
    for a, b in zip(*state):
        assert torch.equal(_raw(a), _raw(b))


@pytest.mark.parametrize("blocks", [1, 8])
@pytest.mark.parametrize("codes", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_append_of_special_values(dtype, codes, blocks):
    """Long and short runs whose elements are infinite, NaN, zero, subnormal or halfway between codes, next to ones that are not."""
    g = _gen(31)
    n, d = 200, 64
    for first in (0, 5):
        kc, ks = _random_cache(g, 3, 128, 2, d, blocks, codes)
        x = torch.randn((n, 2, d), generator=g) * 3
        x[10, 0, 3], x[20, 0, 4], x[30, 0, 5] = math.inf, -math.inf, math.nan
        x[40:60] = 0.0
        x[60:80] *= 2.0 ** -24 if dtype == FP else 2.0 ** -130
        x[80:100] = torch.randint(-254, 255, (20, 2, d), generator=g) / 2.0  # halves of an int8 code at scale 1
        x = x.to(dtype)
        want_c, want_s = kc.clone(), ks.clone()
        slots = list(range(128 + first, 128 + first + 100)) + list(range(first, first + 100))
        U.append(x, want_c, want_s, slots)
        got = [kc.cuda(), kc.cuda(), ks.cuda(), ks.cuda()]
        fa3.quantized_kvcache_append(x.cuda(), x.cuda(), *got, torch.tensor(slots, device="cuda"))
        for c, s in (got[0::2], got[1::2]):
            assert torch.equal(s.cpu(), want_s)
            a, b = U.values_of(c.cpu()), U.values_of(want_c)
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def test_under_torch_compile():
    g = _gen(14)
    kc, ks, table, _ = _cache_for(g, [100, 60], 32, 32, 2, 64, E4M3)
    q = torch.randn((2, 1, 4, 64), generator=g).to(BF).cuda()
    kn = torch.randn((2, 1, 2, 64), generator=g).to(BF).cuda()
    lens, table = _i32([90, 50]), table.cuda()

    def step(q, kn, kc, vc, ks, vs):
        out, lse, *_ = fa3.flash_attn_with_kvcache(q, kc, vc, kn, kn, cache_seqlens=lens, page_table=table, k_descale=ks, v_descale=vs,
                                                   causal=True, return_softmax_lse=True)
        return out * 2, lse

    state = [[kc.cuda(), kc.cuda(), ks.cuda(), ks.cuda()] for _ in range(2)]
    a = step(q, kn, *state[0])
    c = torch.compile(step, fullgraph=True, backend="aot_eager")(q, kn, *state[1])
    for x, y in zip(a, c):
        assert torch.equal(x, y)
    for x, y in zip(*state):
        assert torch.equal(_raw(x), _raw(y))


def test_refusals_with_tensors():
    g = _gen(15)
    kc, ks, table, _ = _cache_for(g, [64, 64], 32, 32, 2, 64, E4M3)
    kc, ks, table, lens = kc.cuda(), ks.cuda(), table.cuda(), _i32([64, 64])
    q = torch.zeros((2, 1, 4, 64), dtype=BF, device="cuda")
    call = lambda **kw: fa3.flash_attn_with_kvcache(**{**dict(  # noqa: E731
        q=q, k_cache=kc, v_cache=kc, cache_seqlens=lens, page_table=table, k_descale=ks, v_descale=ks), **kw})
    call()
    for kw, said in [
            (dict(k_descale=None), "k_descale"), (dict(k_descale=ks.half()), "fp32"), (dict(k_descale=ks[:, :, :1]), "shape"),
            (dict(v_descale=ks.cpu()), "fp32"), (dict(v_cache=kc.view(INT8)), "same dtype"), (dict(v_cache=kc.to(BF)), "8-bit codes"),
            (dict(q=q.float()), "FP16 and BF16"), (dict(q=q[..., :32].contiguous()), "head dimension"), (dict(q_descale=ks), "q_descale"),
            (dict(scheduler_metadata=torch.zeros(192, dtype=torch.uint8, device="cuda")), "scheduler_metadata"),
            (dict(page_table=table.long()), "int32"), (dict(cache_seqlens=lens.long()), "int32"), (dict(cache_seqlens=None), "lengths"),
            (dict(page_table=None), "one row per sequence"), (dict(k=q[:, :, :2]), "together"), (dict(attention_chunk=2), "attention_chunk"),
            (dict(qv=q), "qv"), (dict(cache_leftpad=lens), "leftpad")]:
        with pytest.raises(RuntimeError, match=said):
            call(**kw)
    with pytest.raises(RuntimeError, match="descale"):  # a 16-bit cache has no scales
        call(k_cache=kc.to(BF), v_cache=kc.to(BF))
    x, slots = torch.zeros((3, 2, 64), dtype=BF, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for args, said in [((x, x, kc, kc, ks, ks, slots.int()), "int64"), ((x, x[:2], kc, kc, ks, ks, slots), "one dtype"),
                       ((x, x, kc.to(BF), kc, ks, ks, slots), "8-bit codes"), ((x.float(), x, kc, kc, ks, ks, slots), "FP16 and BF16")]:
        with pytest.raises(RuntimeError, match=said):
            fa3.quantized_kvcache_append(*args)
    for args, said in [((lens.long(), lens, table, lens, 32, 4), "int32"), ((lens, lens[:1], table, lens, 32, 4), "new_seqlens"),
                       ((lens, lens, table.t(), lens, 32, 4), "page_table"), ((lens, lens, table, lens, 0, 4), "sizes")]:
        with pytest.raises(RuntimeError, match=said):
            fa3.paged_kvcache_plan(*args)
