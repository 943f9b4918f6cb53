"""Plain forms of the operators around a KV cache held in 8 bits, in 64 bits (and Python integers) on the host, for their tests."""
import math

import torch

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF, FP = torch.bfloat16, torch.float16


def values_of(codes):
    """Codes as 64-bit values (also of NaN codes)."""
    return codes.to(torch.float32).double()


def nearest(x, dtype):
    """64-bit values in units of their scale -> codes: to the nearest, ties to even, saturating; NaN -> NaN, or 0 in int8."""
    most = MOST[dtype]
    y = x.clamp(-most, most)
    if dtype == INT8:
        return torch.round(torch.nan_to_num(y, nan=0.0)).to(INT8)
    mant, exp = torch.frexp(y.abs())  # y = mant * 2^exp, mant in [0.5, 1)
    step = torch.ldexp(torch.ones_like(y), (exp - 4).clamp(min=-9))  # four significant bits, subnormal step 2^-9
    return torch.where(torch.isnan(y), y, torch.round(y / step) * step).to(torch.float32).to(E4M3)


def scale_for(amax, dtype):
    """amax: a Python float."""
    s = 2.0 ** -40
    while amax > MOST[dtype] * s:
        s *= 2
    return s


def append(x, cache, scale, slots):
    """x (total, h_k, d) into cache (outer, rows, h_k, d) / scale (outer, blocks, h_k), all on the host and in place."""
    outer, rows, h_k, d = cache.shape
    sb = rows // scale.shape[1]
    x64 = x.double()
    runs = {}
    for t, s in enumerate(slots):
        if s >= 0:
            runs.setdefault(s // sb, []).append((s % sb, t))
    for blk, run in runs.items():
        o, i = divmod(blk, rows // sb)
        first, lines, toks = run[0][0], [r for r, _ in run], [t for _, t in run]
        for h in range(h_k):
            v = x64[toks, h]
            fin = v[torch.isfinite(v)].abs()
            need = scale_for(float(fin.max()) if fin.numel() else 0.0, cache.dtype)
            old = float(scale[o, i, h])
            now = need if first == 0 else max(old, need)
            at = i * sb
            if first > 0 and now != old:
                cache[o, at:at + first, h] = nearest(values_of(cache[o, at:at + first, h]) * (old / now), cache.dtype)
            cache[o, [at + r for r in lines], h] = nearest(v / now, cache.dtype)
            scale[o, i, h] = now


def plan(have, new, table, free, page, total):
    """Lists of Python integers; table: list of rows, changed in place."""
    cu, after, taken, at, slots, positions, ok = [0], [], 0, 0, [], [], []
    for r, (a, n) in enumerate(zip(have, new)):
        had, needed = -(-a // page), -(-(a + n) // page)
        fits = needed <= len(table[r])
        need = needed - had if fits else 0
        granted = fits and at + need <= len(free)
        if need == 0:
            granted = fits
        if granted and need:
            table[r][had:needed] = free[at:at + need]
            taken = at + need
        at += need
        after.append(a + n if granted else a)
        cu.append(cu[-1] + n)
        for i in range(n):
            positions.append(a + i)
            slots.append(table[r][(a + i) // page] * page + (a + i) % page if granted else -1)
    slots, positions = slots[:total], positions[:total]
    pad = total - len(slots)
    return slots + [-1] * pad, cu, after, positions + [0] * pad, [taken]


def attend(q, k, v, scale, causal=False, window=None, softcap=0.0):
    """One sequence: q (s_q, h, d), k / v (s_k, h_k, d) in 64 bits -> (out, lse, sum of p |v|).  window: the (left, right) of a call that
    is local after the window rule (oracle/golden.py), taken literally as there: a right side of -1 ends a key before the diagonal."""
    s_q, h, d = q.shape
    s_k, h_k, _ = k.shape
    i = torch.arange(s_q)[:, None] + s_k - s_q
    j = torch.arange(s_k)[None]
    seen = torch.ones(s_q, s_k, dtype=torch.bool)
    if causal:
        seen &= j <= i
    if window is not None:
        seen &= (j >= i - window[0]) & (j <= i + window[1])
    out, size = torch.zeros(s_q, h, d, dtype=torch.float64), torch.zeros(s_q, h, d, dtype=torch.float64)
    lse = torch.full((h, s_q), math.inf, dtype=torch.float64)
    alive = seen.any(1)
    for g in range(h):
        x = q[:, g].double() @ k[:, g // (h // h_k)].T * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        x = torch.where(seen, x, -math.inf)[alive]
        if not x.numel():
            continue
        p = torch.softmax(x, -1)
        vv = v[:, g // (h // h_k)]
        out[alive, g] = p @ vv
        size[alive, g] = p @ vv.abs()
        lse[g, alive] = torch.logsumexp(x, -1)
    return out, lse, size


def check_attention(out, lse, want, softcap=0.0, tag=""):
    """Rounding errors, each at most half a step: the output's (eps / 2 of its value, 2^-25 among fp16's subnormals) and P's to fp16
    (2^-11 of every p |v|).  Scores are sums in fp32 under an exponential of relative error 2^-22: 2^-14 covers scores of up to
    some hundreds; a capped score is off by up to cap * 2^-20 more (an exponential with error 2^-20, divided once).  LSE: the
    same relative errors of the sum, absolute here, and half a step of fp32."""
    o64, l64, size = want
    if not o64.numel():
        return
    half = torch.finfo(out.dtype).eps / 2
    cap = softcap * 2.0 ** -20
    o, l = out.double().cpu(), lse.double().cpu()
    allowed = half * o64.abs() + (2.0 ** -11 + 2.0 ** -14 + 2 * cap) * size * (1 + half) + 2.0 ** -24
    off = (o - o64).abs() - allowed
    assert torch.isfinite(o).all(), tag
    assert float(off.max()) <= 0, (tag, float(off.max()), float((o - o64).abs().max()))
    dead = torch.isinf(l64)
    assert torch.equal(torch.isposinf(l), dead), tag
    off_l = (l - l64)[~dead].abs() - (2.0 ** -16 + cap + 2.0 ** -22 * l64[~dead].abs())
    assert not off_l.numel() or float(off_l.max()) <= 0, (tag, float(off_l.max()))
