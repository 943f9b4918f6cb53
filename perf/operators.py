"""Serving from a paged key / value cache held in 8 bits: one step's operators, as cases that a timing program can draw, prepare and run.

A case is a dict of plain values.  ``op`` says which operator it runs:

  plan    request lengths -> pages from the free list into the page table, slot of every new token, packed offsets, positions
  append  new keys and values -> 8-bit codes in the pages, one scale for each (block of tokens, head)
  attend  attention of one or many query rows per sequence over such a cache; with ``append`` the call brings new tokens too

The definitions, for a page table of ``page`` tokens a page, scale blocks of ``sb`` tokens, and codes that stand for code * scale:

  plan    request r holds ceil(have / page) pages and needs ceil((have + new) / page); the missing ones come off the free list in
          request order; a request that the list or its row of the table has no room for is left as it was, its slots are -1
  append  scale = the smallest power of two, 2^-40 at least, with amax(finite values) <= 448 * scale (e4m3) or 127 * scale (int8);
          a block whose first rows are already there keeps its scale where that is larger, else its codes are expressed in the new
          scale; rows behind the new ones are left alone.  Codes are rounded to nearest even; infinities saturate
  attend  softmax(scale * q K^T, capped, masked) V and the log of the sum; rows without a visible key give 0 and +inf

With ``own`` false each runs in elementary operations, else through this repository's package.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MOST = {"e4m3": 448.0, "int8": 127.0}
LEAST_SCALE = 2.0 ** -40


def _plan(b, lo, hi, new_lo, new_hi, page, cols, **more):
    return dict(dict(op="plan", b=b, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi, page=page, cols=cols, pad=0), **more)


def _append(b, lo, hi, new_lo, new_hi, page, sb, hk, d, dtype="bf16", codes="e4m3", **more):
    return dict(dict(op="append", b=b, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi, page=page, sb=sb, hk=hk, d=d, dtype=dtype,
                     codes=codes, pad=0), **more)


def _attend(b, sq, sk, sk_lo, h, hk, d, page, sb, dtype="bf16", codes="e4m3", **more):
    """sq / sk: query rows and keys of the longest sequence, sq_lo / sk_lo of the shortest.  page 0: a contiguous cache.  packed:
    queries as (total, h, d) with their offsets.  window: keys visible to the left, -1 for all."""
    return dict(dict(op="attend", b=b, sq=sq, sq_lo=sq, sk=sk, sk_lo=sk_lo, h=h, hk=hk, d=d, page=page, sb=sb, dtype=dtype,
                     codes=codes, causal=True, window=-1, softcap=0.0, packed=False, append=False, scales="pow2"), **more)


def listed():
    return [
        # a decoding step of a small batch: one token each, nothing but latency
        dict(_plan(8, 100, 4000, 1, 1, 64, 64), name="plan_b8"),
        # a step of a large server: decoding requests and prompts together, some rows of padding for a captured graph
        dict(_plan(1024, 1, 8000, 1, 64, 16, 640, pad=333), name="plan_b1024_mixed"),
        # the tokens of one decoding step
        dict(_append(64, 1024, 8191, 1, 1, 128, 128, 8, 128), name="append_decode_b64"),
        # prompts of several requests in one packed step, blocks of 16 tokens, the other types
        dict(_append(7, 0, 300, 37, 2048, 64, 16, 8, 128, "fp16", "int8", pad=61), name="append_prompts_fp16_int8"),
        # long prompts, one scale for each page
        dict(_append(8, 0, 40, 2048, 2048, 128, 128, 8, 128), name="append_prompts_8x2048"),
        # one user's decoding step on a short context: too few heads to fill the chip by themselves
        dict(_attend(1, 1, 2048, 2048, 32, 8, 128, 128, 128), name="attend_single_L2048"),
        # a serving batch of ragged lengths, contiguous cache, the new tokens appended by the call
        dict(_attend(64, 1, 8191, 1024, 32, 8, 128, 0, 64, append=True), name="attend_b64_append"),
        # speculative decoding on a paged cache with a sliding window
        dict(_attend(32, 4, 32768, 512, 64, 8, 128, 256, 128, window=4096, scales="any"), name="attend_b32_paged_window"),
        # long context: 2.1 GB of codes for 8 query rows
        dict(_attend(8, 1, 131072, 131072, 64, 8, 128, 128, 128), name="attend_long_L131072"),
        # wide heads, small pages, capped scores, the other types
        dict(_attend(16, 1, 4099, 300, 32, 8, 256, 32, 16, "fp16", "int8", softcap=50.0), name="attend_paged_d256_int8"),
        # one step of chunked prefill: ragged chunks of several requests against their paged caches
        dict(_attend(4, 2048, 8192, 1777, 32, 8, 128, 128, 64, sq_lo=301, packed=True), name="attend_chunks_paged"),
        # drafts of 16 tokens to be checked in one pass over long caches: many rows for a decode, few for a prefill
        dict(_attend(6, 16, 20000, 3001, 32, 4, 64, 64, 32, "fp16", "e4m3", sq_lo=3, packed=True), name="attend_drafts_d64"),
    ]


HEADS = ((4, 4), (8, 8), (16, 16), (32, 32), (8, 1), (16, 4), (16, 8), (32, 8), (64, 8), (12, 4), (5, 1), (48, 8))
MOST_CODES = 2.2e9   # of one cache pair: the long context
MOST_FLOPS = 2.0e11  # of one call: the chunks


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "append", "append", "attend", "attend", "attend", "attend"))
    page = rng.choice((16, 32, 64, 128, 256))
    sb = rng.choice([n for n in (16, 32, 64, 128, 256) if n <= page])
    dtype, codes = rng.choice(("bf16", "bf16", "fp16")), rng.choice(("e4m3", "e4m3", "int8"))
    d = rng.choice((64, 80, 96, 128, 128, 128, 192, 256))
    h, hk = rng.choice(HEADS)
    if op == "plan":
        b, hi = _log(rng, 1, 1024), _log(rng, 10, 8000)
        most = _log(rng, 1, 64)
        return _plan(b, rng.randint(0, hi), hi, rng.choice((0, 1)), most, page, -(-(hi + most) // page) + rng.randint(0, 9), pad=rng.choice((0, 5, 333)))
    if op == "append":
        most = _log(rng, 1, 2048)
        b = min(_log(rng, 1, 64), max(1, 16384 * 1024 // (most * hk * d)))
        hi = _log(rng, 1, 1000)
        return _append(b, rng.randint(0, hi), hi, max(1, most // rng.choice((1, 1, 7))), most, page, sb, hk, d, dtype, codes, pad=rng.choice((0, 61)))
    b, sk = _log(rng, 1, 64), _log(rng, 17, 131072)
    sq = rng.choice((1, 1, 1, 2, 4, _log(rng, 5, 64), _log(rng, 64, 2048)))
    sk = max(sk, sq)
    c = _attend(b, sq, sk, 0, h, hk, d, page, sb, dtype, codes)
    c["page"] = rng.choice((0, page, page))
    c["causal"] = rng.random() < 0.8
    c["window"] = rng.choice((-1, -1, -1, 1000, 4096))
    c["softcap"] = rng.choice((0.0, 0.0, 0.0, 30.0))
    c["append"] = sq <= 4 and rng.random() < 0.3
    c["packed"] = not c["append"] and rng.random() < 0.5
    c["scales"] = rng.choice(("pow2", "any")) if not c["append"] else "pow2"
    c["causal"] = c["causal"] or c["window"] >= 0
    while c["b"] > 1 and (2.0 * c["b"] * c["sk"] * hk * d > MOST_CODES or 4.0 * c["b"] * c["sq"] * c["sk"] * h * d > MOST_FLOPS):
        c["b"] -= 1
    while 4.0 * c["sq"] * c["sk"] * h * d > MOST_FLOPS and c["sq"] > 1:
        c["sq"] //= 2
    c["sq_lo"] = max(1, c["sq"] // rng.choice((1, 3, 20))) if c["packed"] else c["sq"]
    c["sk_lo"] = max(c["sq"], c["sk"] // rng.choice((1, 2, 8, 32)))
    return c


# ---- sizes ----
def _spread(lo, hi, n):
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(c):
    """(query rows, keys) of every sequence of an attend case, appended ones included, in a fixed mixed order."""
    more = c["sq"] if c["append"] else 0
    got = list(zip(_spread(c["sq_lo"], c["sq"], c["b"]), [n + more for n in _spread(c["sk_lo"], c["sk"], c["b"])]))
    np.random.RandomState(c["b"]).shuffle(got)
    return got


def _held(c):
    """(tokens held, new tokens) of every request of a plan or append case."""
    got = list(zip(_spread(c["lo"], c["hi"], c["b"]), _spread(c["new_lo"], c["new_hi"], c["b"])[::-1]))
    np.random.RandomState(c["b"]).shuffle(got)
    return got


def _room(c):
    """Tokens that a sequence's part of the cache has room for: whole pages, or whole scale blocks of a contiguous cache."""
    unit = c["page"] or c["sb"]
    most = max(k for _, k in _lengths(c)) if c["op"] == "attend" else max(a + n for a, n in _held(c))
    return -(-most // unit) * unit


def _pairs(c):
    """Visible (query, key) pairs of every sequence."""
    got = []
    for nq, nk in _lengths(c):
        i = np.arange(nq, dtype=np.int64)
        last = np.minimum(i + nk - nq, nk - 1) if c["causal"] else np.full(nq, nk - 1, dtype=np.int64)
        first = np.maximum(0, i + nk - nq - c["window"]) if c["window"] >= 0 else 0
        got.append(float(np.maximum(0, last + 1 - first).sum()))
    return got


def work(case):
    c = case
    if c["op"] == "plan":
        total = sum(n for _, n in _held(c)) + c["pad"]
        fresh = sum(-(-(a + n) // c["page"]) - -(-a // c["page"]) for a, n in _held(c))
        # lengths in; offsets, lengths, slots, positions out; the pages taken are read, and written into the table
        return {"bytes": 4.0 * (2 * c["b"] + 2 * c["b"] + 1 + 2 * fresh) + 12.0 * total, "flops": float(total)}
    if c["op"] == "append":
        total = sum(n for _, n in _held(c))
        blocks = sum(-(-(a + n) // c["sb"]) - a // c["sb"] for a, n in _held(c) if n)
        return {"bytes": 2.0 * total * c["hk"] * c["d"] * 3 + 2.0 * 4 * blocks * c["hk"] + 8.0 * (total + c["pad"]),
                "flops": 4.0 * total * c["hk"] * c["d"]}
    nq = sum(a for a, _ in _lengths(c))
    seen = sum(min(k, c["window"] + q) if c["window"] >= 0 else k for q, k in _lengths(c))
    more = 2.0 * 3 * nq * c["hk"] * c["d"] if c["append"] else 0.0
    return {"bytes": 4.0 * nq * c["h"] * c["d"] + 4.0 * nq * c["h"] + 2.0 * seen * c["hk"] * (c["d"] + 4.0 / c["sb"]) + more,
            "flops": 4.0 * c["d"] * c["h"] * sum(_pairs(c))}


# ---- inputs ----
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pow2_scale(amax, codes):
    """The smallest power of two, LEAST_SCALE at least, with amax <= MOST * scale."""
    m, e = torch.frexp(amax)
    top, shift = (0.875, 9) if codes == "e4m3" else (0.9921875, 7)
    return torch.ldexp(torch.ones_like(m), e - shift + (m > top).to(e.dtype)).clamp(min=LEAST_SCALE)


def _encode(x, codes):
    """x: values in units of their scale."""
    if codes == "e4m3":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).clamp(-127.0, 127.0).round().to(torch.int8)


def _filled(gen, outer, room, sb, hk, d, codes, scales):
    """A cache that tokens were written into: codes (outer, room, hk, d) and scales (outer, room / sb, hk)."""
    # a row of the cache at a time: normal values whose size differs from block to block and head to head
    got = torch.empty((outer, room, hk, d), dtype=CODES[codes], device="cuda")
    scale = torch.empty((outer, room // sb, hk), dtype=torch.float32, device="cuda")
    rows = max(1, (1 << 28) // (room * hk * d))
    for i in range(0, outer, rows):
        n = min(rows, outer - i)
        x = torch.randn((n, room // sb, sb, hk, d), generator=gen, device="cuda")
        x *= torch.exp(0.4 * torch.randn((n, room // sb, 1, hk, 1), generator=gen, device="cuda"))
        amax = x.abs().amax(dim=(2, 4))
        s = _pow2_scale(amax, codes) if scales == "pow2" else amax / MOST[codes]
        got[i:i + n] = _encode(x / s[:, :, None, :, None], codes).view(n, room, hk, d)
        scale[i:i + n] = s
    return got, scale


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    host = np.random.RandomState(int(seed) % (1 << 31))
    if c["op"] == "attend":
        return _prepare_attend(c, gen, host)
    held = _held(c)
    host.shuffle(held)
    s = dict(c, total=sum(n for _, n in held) + c["pad"], lens=_i32([a for a, _ in held]), new=_i32([n for _, n in held]))
    cols = c["cols"] if c["op"] == "plan" else _room(c) // c["page"]
    # a cache has just the pages that an append case uses; a plan case has pages for every column of its table and a few more
    pages = host.permutation(c["b"] * cols + 8 if c["op"] == "plan" else sum(-(-(a + n) // c["page"]) for a, n in held))
    table = np.zeros((c["b"], cols), dtype=np.int64)
    used = 0
    for r, (a, _) in enumerate(held):
        n = -(-a // c["page"])
        table[r, :n] = pages[used:used + n]
        used += n
    if c["op"] == "plan":
        s["table"], s["free"] = _i32(table.tolist()), _i32(pages[used:].tolist())
        return s
    slots = []
    for r, (a, n) in enumerate(held):
        n0 = -(-a // c["page"])
        n1 = -(-(a + n) // c["page"])
        table[r, n0:n1] = pages[used:used + n1 - n0]
        used += n1 - n0
        at = np.arange(a, a + n)
        slots.append(table[r, at // c["page"]] * c["page"] + at % c["page"])
    slots.append(np.full(c["pad"], -1))
    s["slots"] = torch.from_numpy(np.concatenate(slots).astype(np.int64)).cuda()
    shape = (s["total"], c["hk"], c["d"])
    for n in ("k", "v"):
        # now and then a token or a channel much larger than the others
        x = torch.randn(shape, generator=gen, device="cuda")
        x *= 1.0 + 6.0 * (torch.rand(shape[:2] + (1,), generator=gen, device="cuda") < 0.02)
        s[n] = x.to(TYPES[c["dtype"]])
        s[n + "_cache"], s[n + "_scale"] = _filled(gen, used, c["page"], c["sb"], c["hk"], c["d"], c["codes"], "pow2")
    return s


def _prepare_attend(c, gen, host):
    lengths = _lengths(c)
    host.shuffle(lengths)
    dt, b, hk, d = TYPES[c["dtype"]], c["b"], c["hk"], c["d"]
    new = c["sq"] if c["append"] else 0
    s = dict(c, lens=_i32([k - new for _, k in lengths]), scale=d ** -0.5, cu=None, table=None, k_new=None, v_new=None)
    room, outer, rows = _room(c), b, _room(c)
    if c["page"]:
        cols = room // c["page"]
        outer, rows = b * cols, c["page"]
        s["table"] = _i32(host.permutation(outer).reshape(b, cols).tolist())
    for n in ("k", "v"):
        s[n + "_cache"], s[n + "_scale"] = _filled(gen, outer, rows, c["sb"], hk, d, c["codes"], c["scales"])
        if new:
            s[n + "_new"] = torch.randn((b, new, hk, d), generator=gen, device="cuda").to(dt)
    if c["packed"]:
        s["cu"] = _i32([0] + np.cumsum([a for a, _ in lengths]).tolist())
        s["q"] = torch.randn((sum(a for a, _ in lengths), c["h"], d), generator=gen, device="cuda").to(dt)
    else:
        s["q"] = torch.randn((b, c["sq"], c["h"], d), generator=gen, device="cuda").to(dt)
    return s


# ---- one pass ----
def _package():
    path = os.path.abspath("flash-attention-npu_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_attn_npu_v3
    return flash_attn_npu_v3


def run(s):
    if s["op"] == "plan":
        if own:
            return (*_package().paged_kvcache_plan(s["lens"], s["new"], s["table"], s["free"], s["page"], s["total"]), s["table"])
        return _plain_plan(s)
    if s["op"] == "append":
        if own:
            _package().quantized_kvcache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"])
        else:
            for n in ("k", "v"):
                _plain_append(s[n], s[n + "_cache"], s[n + "_scale"], s["slots"], s["codes"])
        return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    state = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]) if s["append"] else ()
    if own:
        got = _package().flash_attn_with_kvcache(
            s["q"], s["k_cache"], s["v_cache"], s["k_new"], s["v_new"], cache_seqlens=s["lens"], page_table=s["table"],
            cu_seqlens_q=s["cu"], max_seqlen_q=s["sq"] if s["packed"] else None, k_descale=s["k_scale"], v_descale=s["v_scale"],
            softmax_scale=s["scale"], causal=s["causal"], window_size=(s["window"], -1), softcap=s["softcap"],
            return_softmax_lse=True)
        return (got[0], got[1]) + state
    return _plain_attend(s) + state


def _plain_plan(s):
    have, new, page, free, table = s["lens"].long(), s["new"].long(), s["page"], s["free"].long(), s["table"]
    cols = table.shape[1]
    had, need_to = (have + page - 1) // page, (have + new + page - 1) // page
    fits = need_to <= cols
    need = torch.where(fits, need_to - had, 0)
    upto = need.cumsum(0)
    granted = fits & (upto <= free.numel())
    after = torch.where(granted, have + new, have)
    cu = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    col = torch.arange(cols, device=table.device)
    fresh = (col >= had[:, None]) & (col < need_to[:, None]) & granted[:, None]
    taken = (upto - need - had)[:, None] + col
    table.copy_(torch.where(fresh, free[taken.clamp(0, free.numel() - 1)], table.long()))
    t = torch.arange(s["total"], device=table.device)
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=have.numel() - 1)
    real = t < cu[-1]
    pos = torch.where(real, have[r] + t - cu[r], 0)
    slot = table[r, (pos // page).clamp(max=cols - 1)].long() * page + pos % page
    slot = torch.where(real & granted[r], slot, -1)
    pages = torch.where(granted, need, 0).sum().reshape(1)
    return slot, cu.int(), after.int(), pos.int(), pages.int(), table


def _plain_append(x, cache, scale, slots, codes):
    outer, room, hk, d = cache.shape
    sb, n = room // scale.shape[1], outer * scale.shape[1]
    keep = slots >= 0
    at, x = slots[keep], x[keep].float()
    blk, row = at // sb, at % sb
    sizes = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    amax = torch.zeros((n, hk), device=x.device).scatter_reduce(0, blk[:, None].expand(-1, hk), sizes, "amax")
    first = torch.full((n,), sb, device=x.device).scatter_reduce(0, blk, row, "amin")
    old, need = scale.view(n, hk), _pow2_scale(amax, codes)
    fresh = torch.where((first == 0)[:, None], need, torch.maximum(old, need))
    now = torch.where((first < sb)[:, None], fresh, old)
    flat = cache.view(n, sb, hk, d)
    again = _encode(flat.float() * (old / now)[:, None, :, None], codes)
    held = (torch.arange(sb, device=x.device) < first[:, None])[:, :, None] & ((first < sb)[:, None] & (now != old))[:, None, :]
    bytes_ = torch.where(held[..., None], again.view(torch.uint8), flat.view(torch.uint8)).view(n * sb, hk, d)
    bytes_[at] = _encode(x / now[blk][:, :, None], codes).view(torch.uint8)
    cache.copy_(bytes_.view(cache.dtype).view(cache.shape))
    scale.copy_(now.view(scale.shape))


def _plain_attend(s):
    b, h, hk, d = s["b"], s["h"], s["hk"], s["d"]
    kc, vc, lens = s["k_cache"], s["v_cache"], s["lens"].long()
    dev, sb = kc.device, s["sb"]
    if s["k_new"] is not None:
        pos = lens[:, None] + torch.arange(s["sq"], device=dev)
        if s["table"] is not None:
            slots = s["table"].gather(1, pos // s["page"]).long() * s["page"] + pos % s["page"]
        else:
            slots = torch.arange(b, device=dev)[:, None] * kc.shape[1] + pos
        for n in ("k", "v"):
            _plain_append(s[n + "_new"].flatten(0, 1), s[n + "_cache"], s[n + "_scale"], slots.flatten(), s["codes"])
        lens = lens + s["sq"]

    def values(cache, scale):  # (b, hk, keys, d)
        if s["table"] is not None:
            table = s["table"].long()
            cache, scale = cache.view(torch.uint8)[table].view(cache.dtype).flatten(1, 2), scale[table].flatten(1, 2)
        x = cache.float().view(b, -1, sb, hk, d) * scale[:, :, None, :, None]
        return x.flatten(1, 2).transpose(1, 2)

    if s["cu"] is not None:  # packed rows -> (b, sq, h, d)
        cu = s["cu"].long()
        rows = cu[1:] - cu[:-1]
        at = cu[:-1, None] + torch.arange(s["sq"], device=dev)
        q = s["q"][at.clamp(max=s["q"].shape[0] - 1)].float()
    else:
        rows = torch.full((b,), s["sq"], device=dev)
        q = s["q"].float()
    q = q.view(b, -1, hk, h // hk, d).permute(0, 2, 3, 1, 4).flatten(2, 3)  # (b, hk, group * sq, d)
    score = torch.matmul(q, values(kc, s["k_scale"]).transpose(2, 3)) * s["scale"]
    if s["softcap"] > 0:
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    i, j = torch.arange(s["sq"], device=dev), torch.arange(score.shape[-1], device=dev)
    seen = (j < lens[:, None]).view(b, 1, -1)
    edge = i[None, :, None] + (lens - rows)[:, None, None]
    if s["causal"]:
        seen = seen & (j <= edge)
    if s["window"] >= 0:
        seen = seen & (j >= edge - s["window"])
    seen = seen.expand(b, s["sq"], -1)[:, None, None]
    score = torch.where(seen, score.view(b, hk, h // hk, s["sq"], -1), -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), values(vc, s["v_scale"])).view(b, hk, h // hk, s["sq"], d) / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, top + torch.log(total), math.inf)[..., 0]
    out = out.permute(0, 3, 1, 2, 4).reshape(b, s["sq"], h, d).to(s["q"].dtype)
    lse = lse.reshape(b, h, s["sq"])
    if s["cu"] is not None:
        real = i < rows[:, None]
        out, lse = out[real], lse.transpose(1, 2)[real].t().contiguous()
    return out, lse


# ---- in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "plan":
        return None
    if s["op"] == "append":
        got = [_exact_append(s[n].double(), s[n + "_cache"], s[n + "_scale"], s["slots"].tolist(), s["codes"]) for n in ("k", "v")]
        return got[0][0], got[1][0], got[0][1], got[1][1]
    lens = s["lens"].tolist()
    new = s["sq"] if s["k_new"] is not None else 0
    state = ()
    if new:
        slots = [(int(s["table"][r, (n + i) // s["page"]]) * s["page"] + (n + i) % s["page"]) if s["page"] else r * s["k_cache"].shape[1] + n + i
                 for r, n in enumerate(lens) for i in range(new)]
        for n in ("k", "v"):
            _exact_append(s[n + "_new"].flatten(0, 1).double(), s[n + "_cache"], s[n + "_scale"], slots, s["codes"], write=True)
        state = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    packed = s["cu"] is not None
    lse = torch.full((s["h"], out.shape[0]) if packed else (s["b"], s["h"], s["sq"]), math.inf, dtype=torch.float64, device="cuda")
    cu = s["cu"].tolist() if packed else None
    group = s["h"] // s["hk"]
    for r in range(s["b"]):
        n = lens[r] + new
        q = (s["q"][cu[r]:cu[r + 1]] if packed else s["q"][r]).double()
        o_r, l_r = (out[cu[r]:cu[r + 1]], lse[:, cu[r]:cu[r + 1]]) if packed else (out[r], lse[r])
        i = torch.arange(q.shape[0], device="cuda")[:, None] + n - q.shape[0]
        first = max(0, n - q.shape[0] - s["window"]) if s["window"] >= 0 else 0
        j = torch.arange(first, n, device="cuda")[None]
        hidden = torch.zeros(i.shape[0], n - first, dtype=torch.bool, device="cuda")
        if s["causal"]:
            hidden |= j > i
        if s["window"] >= 0:
            hidden |= j < i - s["window"]
        for g in range(s["hk"]):
            kv = []
            for m in ("k", "v"):
                codes, scale = s[m + "_cache"], s[m + "_scale"]
                if s["page"]:
                    ids = s["table"][r, :-(-n // s["page"])].tolist()
                    codes = torch.cat([codes[p, :, g].view(torch.uint8) for p in ids]).view(codes.dtype)
                    scale = torch.cat([scale[p, :, g] for p in ids])
                else:
                    codes, scale = codes[r, :, g], scale[r, :, g]
                kv.append(codes[first:n].to(torch.float64) * scale.double().repeat_interleave(s["sb"])[first:n, None])
            x = torch.einsum("igd,jd->gij", q[:, g * group:(g + 1) * group], kv[0]) * s["scale"]
            if s["softcap"] > 0:
                x = torch.tanh(x / s["softcap"]) * s["softcap"]
            x.masked_fill_(hidden, -math.inf)
            l = torch.logsumexp(x, dim=-1)
            some = torch.isfinite(l)
            p = torch.where(some[..., None], torch.exp(x - torch.where(some, l, 0.0)[..., None]), 0.0)
            o_r[:, g * group:(g + 1) * group] = torch.einsum("gij,jd->igd", p, kv[1])
            l_r[g * group:(g + 1) * group] = torch.where(some, l, math.inf)
    return (out, lse) + state


def _exact_append(x, cache, scale, slots, codes, write=False):
    """Block by block, in 64 bits: (values of the codes, scales)."""
    outer, room, hk, d = cache.shape
    sb, most = room // scale.shape[1], MOST[codes]
    code = cache.to(torch.float64).view(-1, sb, hk, d)
    s64 = scale.double().view(-1, hk)
    tokens = {}
    for t, slot in enumerate(slots):
        if slot >= 0:
            tokens.setdefault(slot // sb, []).append((slot % sb, t))

    def near(v):  # to the nearest code, ties to the even one
        v = v.clamp(-most, most)
        if codes == "int8":
            return torch.round(v)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(v / step) * step

    for blk, rows in tokens.items():
        first = min(r for r, _ in rows)
        at, t = [r for r, _ in rows], [k for _, k in rows]
        amax = x[t].abs().amax(dim=(0, 2))
        need = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=1e-300) / most)))
        need = torch.where(amax <= most * need / 2, need / 2, need).clamp(min=LEAST_SCALE)  # a logarithm next to a whole number
        now = need if first == 0 else torch.maximum(need, s64[blk])
        if first:
            grown = near(code[blk, :first] * (s64[blk] / now)[None, :, None])
            code[blk, :first] = torch.where((now != s64[blk])[None, :, None], grown, code[blk, :first])
        code[blk, at] = near(x[t] / now[None, :, None])
        s64[blk] = now
    code = code.view(cache.shape)
    if write:
        cache.copy_(code.float().to(cache.dtype))
        scale.copy_(s64.view(scale.shape).float())
    return (code if codes == "e4m3" else None), s64.view(scale.shape)
