"""GPU: what the operators around an 8-bit KV cache do at the edges of their contract -- indices and lengths out of range, more tokens than rows,
numbers of every size in both attention kernels, negative softmax scales, windows as long as the longest sequence."""
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
from test_kv8_gpu import _cache_for, _gen, _i32, _random_cache, _raw, _status

pytestmark = pytest.mark.gpu


def _reported():
    """Whether the device status word told of an index out of range (and clears it)."""
    torch.cuda.synchronize()
    rc = L.load().fa_b200_check_status(torch.cuda.current_stream().cuda_stream)
    assert rc == 0 or "out of range" in L.load().fa_b200_last_error().decode()
    return rc != 0


def _values(table, page, n, codes, scale, gone=()):
    """64-bit values of a sequence's first n tokens; pages in `gone` hold nothing (zeros)."""
    sb = page // scale.shape[1]
    rows = []
    for t in range(n):
        o, i = int(table[t // page]), t % page
        rows.append(torch.zeros(codes.shape[2:], dtype=torch.float64) if t // page in gone else
                    U.values_of(codes[o, i]) * scale[o, i // sb].double()[:, None])
    return torch.stack(rows)


# ---------------------------------------------------------------- plan
@pytest.mark.parametrize("have,new,total,after,cu,real", [
    ([5, 0, 16], [4, 10, 3], 12, [9, 0, 16], [0, 4, 12, 12], 4),             # the second is cut, the third has no row at all
    ([5, 0, 16], [4, 8, 0], 12, [9, 8, 16], [0, 4, 12, 12], 12),             # just as many tokens as rows
    ([5, 0, 16], [4, 8, 1], 12, [9, 8, 16], [0, 4, 12, 12], 12),
    ([1, 2], [1, 1], 0, [1, 2], [0, 0, 0], 0),
    ([0, 0, 5], [2 ** 31 - 1, 2 ** 31 - 1, 3], 6, [0, 0, 5], [0, 6, 6, 6], 0),  # sums beyond 32 bits
    ([7, 0, 3], [2, 2 ** 31 - 1, 1], 6, [9, 0, 3], [0, 2, 6, 6], 2)])
def test_plan_of_more_tokens_than_rows(have, new, total, after, cu, real):
    """A request whose tokens end behind the packed batch is left as it was and reported; offsets stay within the batch."""
    page, cols, free = 16, 4, [30, 31, 32, 33, 34]
    rows = torch.arange(len(have) * cols).view(-1, cols) + 100
    table = _i32(rows.tolist())
    slots, cu_got, after_got, positions, taken = fa3.paged_kvcache_plan(_i32(have), _i32(new), table, _i32(free), page, total)
    assert _reported() == (sum(new) > total)
    assert after_got.tolist() == after and cu_got.tolist() == cu
    want_rows, used, want_slots = rows.tolist(), 0, []
    for r, (a, b) in enumerate(zip(have, after)):
        for col in range(-(-a // page), -(-b // page)):
            want_rows[r][col], used = free[used], used + 1
        want_slots += [want_rows[r][t // page] * page + t % page for t in range(a, b)]
    assert taken.tolist() == [used] and table.tolist() == want_rows
    assert len(want_slots) == real and slots.tolist() == want_slots + [-1] * (total - real)


@pytest.mark.parametrize("have,new", [([-1, 4], [3, 2]), ([4, 4], [-3, 2])])
def test_plan_of_negative_lengths(have, new):
    table = torch.full((2, 3), 7, dtype=torch.int32, device="cuda")
    slots, cu, after, _, taken = fa3.paged_kvcache_plan(_i32(have), _i32(new), table, _i32([9, 8]), 4, 6)
    assert _reported()
    assert after.tolist() == [have[0], 6] and taken.tolist() == [1] and table.tolist() == [[7, 7, 7], [7, 9, 7]]
    at = max(new[0], 0)
    assert cu.tolist() == [0, at, at + 2] and slots.tolist() == ([-1] * at + [36, 37] + [-1] * 6)[:6]


def test_sizes_beyond_32_bits_are_refused():
    table, lens = torch.zeros((2, 4), dtype=torch.int32, device="cuda"), _i32([1, 1])
    for page in (2 ** 32 + 16, -2 ** 32 + 16):
        with pytest.raises(RuntimeError, match="sizes"):
            fa3.paged_kvcache_plan(lens, lens, table, lens, page, 4)
    with pytest.raises(RuntimeError, match="sizes"):
        fa3.paged_kvcache_plan(lens, lens, table, lens, 16, 2 ** 31)
    codes, scales = torch.zeros((4, 16, 1, 16), dtype=torch.int8, device="cuda"), torch.ones((4, 1, 1), device="cuda")
    for most in (2 ** 32 + 1, -1, 2 ** 30):
        with pytest.raises(RuntimeError, match="sequence length|query rows"):
            fa3.flash_attn_with_kvcache(torch.zeros((40, 2, 16), dtype=BF, device="cuda"), codes, codes, cache_seqlens=lens, page_table=table,
                                        cu_seqlens_q=_i32([0, 20, 40]), max_seqlen_q=most, k_descale=scales, v_descale=scales)
    # a page table whose columns cover 2^32 + 2^14 tokens
    kc = torch.zeros((2, 1 << 14, 1, 16), dtype=torch.int8, device="cuda")
    ks = torch.ones((2, 1, 1), device="cuda")
    table = torch.zeros((1, (1 << 18) + 1), dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="too many tokens"):
        fa3.flash_attn_with_kvcache(torch.zeros((1, 1, 1, 16), dtype=BF, device="cuda"), kc, kc, cache_seqlens=_i32([40]), page_table=table,
                                    k_descale=ks, v_descale=ks)


# ---------------------------------------------------------------- append
def test_append_to_slots_that_are_not_there():
    """Slots at and behind the cache's end are skipped and reported; what is around stays as it was."""
    g = _gen(41)
    kc, ks = _random_cache(g, 3, 32, 2, 64, 2, E4M3)
    x = torch.randn((6, 2, 64), generator=g).to(BF)
    slots = [95, 96, 97, 2 ** 40, 10, 2 ** 63 - 1]
    got = [kc.cuda(), kc.cuda(), ks.cuda(), ks.cuda()]
    fa3.quantized_kvcache_append(x.cuda(), x.cuda(), *got, torch.tensor(slots, device="cuda"))
    assert _reported()
    U.append(x, kc, ks, [s if s < 96 else -1 for s in slots])
    for c, s in (got[0::2], got[1::2]):
        assert torch.equal(s.cpu(), ks) and torch.equal(U.values_of(c.cpu()), U.values_of(kc))


@pytest.mark.parametrize("s_q", [2, 40])
@pytest.mark.parametrize("bad", [6, -1, 2 ** 30, -2 ** 31])
def test_new_tokens_on_pages_that_are_not_there(bad, s_q):
    """A sequence whose last page's number is out of range: nothing is written for it, the others get theirs."""
    g = _gen(42)
    kc, ks = _random_cache(g, 6, 32, 2, 64, 2, E4M3)
    table = torch.tensor([[0, 1], [2, bad], [4, 5]], dtype=torch.int32)
    lens = [30, 33, 40]
    x = torch.randn((3, 3, 2, 64), generator=g).to(BF)
    q = torch.randn((3, s_q, 4, 64), generator=g).to(BF)
    got = [kc.cuda(), kc.cuda(), ks.cuda(), ks.cuda()]
    scale = 2.0 ** -14  # (the codes are any)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), *got[:2], x.cuda(), x.cuda(), cache_seqlens=_i32(lens), page_table=table.cuda(),
                                               k_descale=got[2], v_descale=got[3], softmax_scale=scale, causal=True, return_softmax_lse=True)
    assert _reported()
    for r in (0, 2):
        U.append(x[r], kc, ks, [int(table[r, t // 32]) * 32 + t % 32 for t in range(lens[r], lens[r] + 3)])
    for c, s in (got[0::2], got[1::2]):
        assert torch.equal(s.cpu(), ks) and torch.equal(U.values_of(c.cpu()), U.values_of(kc))
    for r in range(3):
        kv = _values(table[r], 32, lens[r] + 3, kc, ks, (1,) if r == 1 else ())
        U.check_attention(out[r], lse[r], U.attend(q[r], kv, kv, scale, True), tag=f"sequence {r}")


@pytest.mark.parametrize("s_q", [1, 40])
def test_expanded_scales_are_read_and_never_written(s_q):
    """One scale for a whole cache, expanded to its blocks and heads, serves attention; calls that append refuse it and leave all as it was."""
    g = _gen(52)
    kc, _ = _random_cache(g, 5, 32, 2, 64, 2, INT8)
    table, lens = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32), [60, 33]
    one = torch.full((1,), 0.015625, device="cuda")
    ks = one.expand(5, 2, 2)
    kd, vd = kc.cuda(), kc.cuda()
    q = torch.randn((2, s_q, 4, 64), generator=g).to(BF)
    kw = dict(cache_seqlens=_i32(lens), page_table=table.cuda(), k_descale=ks, v_descale=ks, causal=True, return_softmax_lse=True)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kd, kd, **kw)
    for r, n in enumerate(lens):
        kv = _values(table[r], 32, n, kc, ks.cpu())
        U.check_attention(out[r], lse[r], U.attend(q[r], kv, kv, 0.125, True), tag=f"sequence {r}")
    x, slots = torch.randn((2, 1, 2, 64), generator=g).to(BF).cuda(), torch.tensor([60, 97], device="cuda")
    own = [torch.full((5, 2, 2), 0.015625, device="cuda") for _ in range(2)]
    for c, s in (((kd, vd), (ks, own[1])), ((kd, vd), (own[0], ks)), ((kd, vd), (own[0], own[0])), ((kd, kd), own),
                 ((kd, vd), (own[0][:1].expand(5, 2, 2), own[1])), ((kd, vd), (own[0][:, :1].expand(5, 2, 2), own[1]))):
        with pytest.raises(RuntimeError, match="of its own"):
            fa3.quantized_kvcache_append(x[:, 0], x[:, 0], *c, *s, slots)
        with pytest.raises(RuntimeError, match="of its own"):
            fa3.flash_attn_with_kvcache(q.cuda(), *c, x, x, **{**kw, "k_descale": s[0], "v_descale": s[1]})
    for t in (kd, vd):
        assert torch.equal(t.cpu(), kc)
    assert all(bool((t == 0.015625).all()) for t in own + [one])
    _status()


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("s_q", [1, 12, 40, 200])
@pytest.mark.parametrize("bad", [9, -1])
def test_a_page_that_is_not_there_holds_nothing(bad, s_q):
    """Its keys and values are zeros, whatever stands on the page that the number would be clamped to."""
    g = _gen(43)
    code = torch.randint(0, 100, (9, 32, 2, 64), generator=g, dtype=torch.uint8)
    code[0], code[8] = 127, 127
    scale = torch.exp2(torch.randint(-3, 2, (9, 2, 2), generator=g).float())
    scale[0], scale[8] = math.nan, math.nan
    table = torch.tensor([[1, 2, 3, bad, 4, 5, 6], [7, 3, 5, 1, 2, 6, 4]], dtype=torch.int32)
    q = torch.randn((2, s_q, 4, 64), generator=g).to(BF)
    kd, sd = code.view(E4M3).cuda(), scale.cuda()
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kd, kd, cache_seqlens=_i32([200, 130]), page_table=table.cuda(), k_descale=sd, v_descale=sd,
                                               softmax_scale=2.0 ** -12, return_softmax_lse=True)
    assert _reported()
    for r, n in enumerate([200, 130]):
        kv = _values(table[r], 32, n, code.view(E4M3), scale, (3,) if r == 0 else ())
        U.check_attention(out[r], lse[r], U.attend(q[r], kv, kv, 2.0 ** -12), tag=f"sequence {r}")


@pytest.mark.parametrize("s_q", [1, 40])
@pytest.mark.parametrize("bad", [4, -1, 2 ** 31 - 1])
def test_cache_rows_out_of_range(bad, s_q):
    """A sequence whose cache row is not there gets no token and is reported; the others are what they are without it."""
    g = _gen(55)
    kc, ks = _random_cache(g, 4, 96, 2, 64, 3, INT8)
    rows, lens = [2, bad, 1], [60, 33, 95]
    x, q = torch.randn((3, 1, 2, 64), generator=g).to(FP), torch.randn((3, s_q, 4, 64), generator=g).to(FP)
    got, scale = [kc.cuda(), kc.cuda(), ks.cuda(), ks.cuda()], 2.0 ** -12  # (the codes are any)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), *got[:2], x.cuda(), x.cuda(), cache_seqlens=_i32(lens), cache_batch_idx=_i32(rows),
                                               k_descale=got[2], v_descale=got[3], softmax_scale=scale, causal=True, return_softmax_lse=True)
    assert _reported()
    for r in (0, 2):
        U.append(x[r], kc, ks, [rows[r] * 96 + lens[r]])
    for c, s in (got[0::2], got[1::2]):
        assert torch.equal(s.cpu(), ks) and torch.equal(c.cpu(), kc)
    for r in (0, 2):
        kv = torch.stack([U.values_of(kc[rows[r], t]) * ks[rows[r], t // 32].double()[:, None] for t in range(lens[r] + 1)])
        U.check_attention(out[r], lse[r], U.attend(q[r], kv, kv, scale, True), tag=f"sequence {r}")


@pytest.mark.parametrize("s_q", [1, 40, 200])
def test_lengths_out_of_range(s_q):
    """A length beyond the cache counts as all of it, a negative one as none; both are reported."""
    g = _gen(44)
    kc, ks, table, kv = _cache_for(g, [96, 96, 96], 32, 16, 2, 64, INT8)
    q = torch.randn((3, s_q, 4, 64), generator=g).to(FP)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), kc.cuda(), cache_seqlens=_i32([97, -3, 2 ** 31 - 1]), page_table=table.cuda(),
                                               k_descale=ks.cuda(), v_descale=ks.cuda(), causal=True, return_softmax_lse=True)
    assert _reported()
    for r, n in enumerate([96, 0, 96]):
        U.check_attention(out[r], lse[r], U.attend(q[r], kv[r][:n], kv[r][:n], 0.125, True), tag=f"sequence {r}")


@pytest.mark.parametrize("cu,most,rows", [
    ([0, 3, 50], 4, [(0, 3), (3, 10)]), ([0, 3, 2 ** 31 - 1], 7, [(0, 3), (3, 10)]), ([-4, 3, 10], 7, [(0, 3), (3, 10)]),
    ([0, 7, 2], 40, [(0, 7), (7, 7)]), ([20, 30, 10], 4, [(10, 10), (10, 10)]), ([0, 300, 10], 200, [(0, 10), (10, 10)])])
@pytest.mark.parametrize("splits", [0, 3])
def test_offsets_out_of_range(cu, most, rows, splits):
    """Offsets of packed queries beyond the rows there are: the rows of the sequence end where the queries do, nothing behind them is touched, and the
    call is reported.  Sequences whose run is longer than the longest that the caller gave have just that many rows computed."""
    g = _gen(51)
    lens, total, pad, h, d = [300, 120], 10, 64, 8, 64
    kc, ks, table, kv = _cache_for(g, lens, 64, 32, 2, d, E4M3)
    kc, ks, table = kc.cuda(), ks.cuda(), table.cuda()
    big = torch.full((total + 2 * pad, h, d), math.nan, dtype=BF, device="cuda")  # rows in front of and behind the queries
    q = big[pad:pad + total]
    q.copy_(torch.randn((total, h, d), generator=g))
    o_big, l_big = torch.full_like(big, 7.0), torch.full((pad + h * total + pad,), 7.0, device="cuda")
    out, lse = o_big[pad:pad + total], l_big[pad:pad + h * total].view(h, total)
    c = kv8._cache_block(kc, kc, ks, ks, q)
    cu_t, lens_t = _i32(cu), _i32(lens)
    p = ops.build_params(q, kc, kc, out, lse, cu_seqlens_q=cu_t, max_seqlen_q=most, seqused_k=lens_t, block_table=table, softmax_scale=0.125,
                         causal=True, num_splits=splits)
    lib = L.load()
    nbytes = lib.fa_b200_kv8_fwd_workspace(C.byref(p), C.byref(c))
    ws = torch.full((max(nbytes, 16) + 256,), 255, dtype=torch.uint8, device="cuda")
    L.check(lib.fa_b200_kv8_fwd(C.byref(p), C.byref(c), ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream))
    assert _reported()
    for t in (o_big[:pad], o_big[pad + total:], l_big[:pad], l_big[pad + h * total:]):
        assert bool((t == 7).all())
    assert bool((ws[nbytes:] == 255).all())
    for r, (a, b) in enumerate(rows):
        if b > a and b - a <= most:
            upto = min(b, cu[-1]) - a  # (rows behind the last offset belong to no sequence)
            want = U.attend(q[a:b].cpu(), kv[r], kv[r], 0.125, True)
            U.check_attention(out[a:a + upto], lse[:, a:a + upto], (want[0][:upto], want[1][:, :upto], want[2][:upto]), tag=f"sequence {r}")


@pytest.mark.parametrize("s_q", [1, 4, 8, 33])
@pytest.mark.parametrize("form", ["none", "int"])
def test_lengths_by_default_and_as_a_number(form, s_q):
    g = _gen(45)
    kc, ks, _, kv = _cache_for(g, [96, 96], 0, 16, 2, 64, E4M3)
    q = torch.randn((2, s_q, 8, 64), generator=g).to(BF)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), kc.cuda(), cache_seqlens=None if form == "none" else 77, k_descale=ks.cuda(),
                                               v_descale=ks.cuda(), causal=True, return_softmax_lse=True)
    n = 96 if form == "none" else 77
    for r in range(2):
        U.check_attention(out[r], lse[r], U.attend(q[r], kv[r][:n], kv[r][:n], 0.125, True), tag=f"sequence {r}")
    _status()


@pytest.mark.parametrize("s_q", [1, 5, 20, 40, 150])
@pytest.mark.parametrize("up", [1.0, 2.0 ** 60, 2.0 ** -70, -1.0])
def test_numbers_of_every_size(s_q, up):
    """Queries whose elements span bf16's range, scales from 2^-40 to 2^30 within one sequence with zero scales and blocks of zeros among them, scores in
    the hundreds, negative softmax scales, for every number of rows.

    Allowed, beside the output's half step and P's rounding to fp16 (2^-11 of every p |v|):
    scores: sums over four steps of 16 products, each step off by at most 2^-22 of the sum S of all |q k| (fp32, truncated), so by 2^-20 S, which a
    weight is off by twice (itself and the sum) and the LSE once;
    small P': P' has fp16's subnormals below, off by at most 2^-25 of a unit in which the largest P' is 2^7 at least, so by 2^-32 of the largest p * scale for
    each code."""
    g = _gen(int(s_q))
    n, d = 512, 64
    kc, ks, _, _ = _cache_for(g, [n], 0, 16, 1, d, E4M3)
    vs = torch.exp2(torch.linspace(-40, 30, n // 16).round())[None, :, None]
    vs[0, 5] = 0.0
    vc = torch.randn((1, n, 1, d), generator=g).clamp(-3, 3).to(E4M3)
    vc[0, 48:64] = 0.0
    k64 = U.values_of(kc[0]) * ks[0].double().repeat_interleave(16, 0)[:, :, None]
    each = vs[0].double().repeat_interleave(16, 0)  # (n, 1)
    c64 = U.values_of(vc[0])
    q = torch.randn((1, s_q, 8, d), generator=g)
    q[..., :8] *= 2.0 ** -12
    q = (q * abs(up)).to(BF)
    scale = 1.5 / up
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), vc.cuda(), cache_seqlens=_i32([n]), k_descale=ks.cuda(), v_descale=vs.cuda(),
                                               softmax_scale=scale, causal=True, return_softmax_lse=True)
    o64, l64, size = U.attend(q[0], k64, c64 * each[:, :, None], scale, True)
    seen = torch.arange(n)[None] <= torch.arange(s_q)[:, None] + n - s_q
    q64, half = q[0].double(), torch.finfo(BF).eps / 2
    for h in range(8):
        x = torch.where(seen, q64[:, h] @ k64[:, 0].T * scale, -math.inf)
        small = 2.0 ** -32 * (torch.softmax(x, -1) * each[:, 0]).amax(-1, keepdim=True) * c64[:, 0].abs().sum(0)
        score = 2.0 ** -20 * (q64[:, h].abs() @ k64[:, 0].abs().T * abs(scale)).amax(-1, keepdim=True)
        off = (out[0, :, h].double().cpu() - o64[:, h]).abs()
        allowed = half * o64[:, h].abs() + ((2.0 ** -11 + 2 * score) * size[:, h] + small) * (1 + half) + 2.0 ** -24
        assert bool((off <= allowed).all()), (h, float((off / allowed).max()))
        off = (lse[0, h].double().cpu() - l64[h]).abs()
        assert bool((off <= 2.0 ** -16 + 2.0 ** -22 * l64[h].abs() + score[:, 0]).all()), (h, float(off.max()))
    _status()


@pytest.mark.parametrize("s_q", [1, 4, 8, 33])
@pytest.mark.parametrize("softcap", [0.0, 25.0])
def test_negative_softmax_scale(s_q, softcap):
    g = _gen(46)
    kc, ks, table, kv = _cache_for(g, [300, 41], 32, 32, 2, 128, INT8, pow2=False)
    q = torch.randn((2, s_q, 16, 128), generator=g).to(FP)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), kc.cuda(), cache_seqlens=_i32([300, 41]), page_table=table.cuda(), k_descale=ks.cuda(),
                                               v_descale=ks.cuda(), softmax_scale=-0.1, softcap=softcap, causal=True, return_softmax_lse=True)
    for r in range(2):
        U.check_attention(out[r], lse[r], U.attend(q[r], kv[r], kv[r], -0.1, True, softcap=softcap), softcap, f"sequence {r}")
    _status()


@pytest.mark.parametrize("s_q,h", [(1, 4), (7, 8), (20, 8), (150, 4)])
@pytest.mark.parametrize("left,right", [(299, -1), (300, -1), (298, -1), (298, 0), (299, 0), (-5, 3), (-3, 3), (-40, 3), (2, -2)])
def test_windows_about_the_longest_sequence(s_q, h, left, right):
    """A left side that reaches over the longest sequence is none, also where only the device knows its length; sides below -1 are taken literally."""
    g = _gen(47)
    lens = [64, 300, 150]
    kc, ks, table, kv = _cache_for(g, lens, 64, 32, 2, 64, E4M3)
    q = torch.randn((3, s_q, h, 64), generator=g).to(BF)
    table = torch.cat([table, torch.zeros((3, 9), dtype=torch.int32)], 1)
    for r, n in enumerate(lens):
        table[r, -(-n // 64):] = 2 ** 30  # (room beyond the lengths, whose pages nobody may look up)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), kc.cuda(), cache_seqlens=_i32(lens), page_table=table.cuda(), k_descale=ks.cuda(),
                                               v_descale=ks.cuda(), window_size=(left, right), return_softmax_lse=True)
    is_causal, is_local, wl, wr = L.normalize_window(s_q, max(lens), False, left, right)
    for r in range(3):
        U.check_attention(out[r], lse[r], U.attend(q[r], kv[r], kv[r], 0.125, is_causal, (wl, wr) if is_local else None), tag=f"sequence {r}")
    _status()


@pytest.mark.parametrize("s_q,h", [(8, 4), (40, 4)])
@pytest.mark.parametrize("left,right,sees", [(2 ** 32, 0, "causal"), (2 ** 63 - 1, 0, "causal"), (2 ** 32 + 5, 2 ** 40, "all"), (-2 ** 32, -2 ** 40 - 1, "all"),
                                             (-2 ** 31, 3, "nothing"), (-2 ** 32 + 4, 3, "nothing"), (4, -2 ** 31, "nothing"), (4, -2 ** 33 + 4, "nothing")])
def test_windows_at_and_beyond_32_bits(left, right, sees, s_q, h):
    """Numbers that 32 bits cannot hold mean what they say, and so do sums of positions with those that are just held."""
    g = _gen(54)
    kc, ks, table, kv = _cache_for(g, [100], 64, 32, 2, 64, E4M3)
    table = torch.cat([table, torch.full((1, 14), 2 ** 30, dtype=torch.int32)], 1)
    q = torch.randn((1, s_q, h, 64), generator=g).to(BF)
    out, lse, *_ = fa3.flash_attn_with_kvcache(q.cuda(), kc.cuda(), kc.cuda(), cache_seqlens=_i32([100]), page_table=table.cuda(), k_descale=ks.cuda(),
                                               v_descale=ks.cuda(), window_size=(left, right), return_softmax_lse=True)
    U.check_attention(out[0], lse[0], U.attend(q[0], kv[0], kv[0], 0.125, sees == "causal", (-200, -200) if sees == "nothing" else None))
    _status()


@pytest.mark.parametrize("s_q,h,d", [(1, 8, 128), (4, 16, 128), (4, 16, 64), (16, 8, 64), (150, 8, 128), (40, 8, 256), (1, 8, 256)])
def test_a_call_repeats_itself(s_q, h, d):
    """Bit for bit, with another call of other inputs in between."""
    g = _gen(48)
    kc, ks, table, _ = _cache_for(g, [900, 77, 300], 32, 16, 2, d, E4M3)
    kd, sd = kc.cuda(), ks.cuda()
    qs = [torch.randn((3, s_q, h, d), generator=g).to(BF).cuda() for _ in range(2)]
    call = lambda i: fa3.flash_attn_with_kvcache(qs[i], kd, kd, cache_seqlens=_i32([900, 77, 300]), page_table=table.cuda(), k_descale=sd,  # noqa: E731
                                                 v_descale=sd, causal=True, return_softmax_lse=True)[:2]
    first, _, again = call(0), call(1), call(0)
    for a, b in zip(first, again):
        assert torch.equal(_raw(a), _raw(b))


def test_odd_strides_of_dimensions_of_one_element():
    """... are put right on the way, as rows of a wider tensor are."""
    g = _gen(53)
    kc, ks, _, kv = _cache_for(g, [100], 0, 32, 2, 64, E4M3)
    big = torch.randn(3000, generator=g).to(BF)
    q, kn = torch.as_strided(big, (1, 1, 8, 64), (1001, 333, 64, 1)), torch.as_strided(big, (1, 1, 2, 64), (77, 5, 72, 1), 1024)
    dev = big.cuda()
    qd, knd = torch.as_strided(dev, (1, 1, 8, 64), (1001, 333, 64, 1)), torch.as_strided(dev, (1, 1, 2, 64), (77, 5, 72, 1), 1024)
    got = [kc.cuda(), kc.cuda(), ks.cuda(), ks.cuda()]
    out, lse, *_ = fa3.flash_attn_with_kvcache(qd, *got[:2], knd, knd, cache_seqlens=_i32([64]), k_descale=got[2], v_descale=got[3], causal=True,
                                               return_softmax_lse=True)
    U.append(kn[0], kc, ks, [64])
    x = torch.stack([U.values_of(kc[0, t]) * ks[0, t // 32].double()[:, None] for t in range(65)])
    U.check_attention(out[0], lse[0], U.attend(q[0], x, x, 0.125, True))
    for c, s in (got[0::2], got[1::2]):
        assert torch.equal(s.cpu()[0, :3], ks[0, :3]) and torch.equal(U.values_of(c.cpu()[0, :65]), U.values_of(kc[0, :65]))


# ---------------------------------------------------------------- other calls
def test_codes_are_for_kv_cache_calls_only():
    """The differentiable calls refuse codes with and without scales, also where a gradient is wanted."""
    kc, s = torch.zeros((2, 32, 2, 64), dtype=INT8, device="cuda"), torch.ones((2, 1, 2), device="cuda")
    cu = _i32([0, 32, 64])
    for grad in (False, True):
        q = torch.zeros((2, 32, 4, 64), dtype=BF, device="cuda", requires_grad=grad)
        with pytest.raises(RuntimeError, match="does not support descale"):
            fa3.flash_attn_func(q, kc, kc, k_descale=s, v_descale=s)
        with pytest.raises(RuntimeError, match="same dtype"):
            fa3.flash_attn_func(q, kc, kc)
        with pytest.raises(RuntimeError, match="does not support descale"):
            fa3.flash_attn_varlen_func(q.flatten(0, 1), kc.flatten(0, 1), kc.flatten(0, 1), cu, cu, 32, 32, k_descale=s, v_descale=s)


def test_a_16_bit_call_asks_nothing_of_an_8_bit_one(monkeypatch):
    """The native path is tried before anything is asked about codes."""
    x = torch.randn((2, 64, 2, 64), generator=_gen(49)).to(BF).cuda()
    q = torch.randn((2, 1, 4, 64), generator=_gen(50)).to(BF).cuda()
    want = fa3.flash_attn_with_kvcache(q, x, x, cache_seqlens=_i32([60, 33]))
    monkeypatch.setattr(kv8, "holds_codes", None)
    assert torch.equal(fa3.flash_attn_with_kvcache(q, x, x, cache_seqlens=_i32([60, 33])), want)
