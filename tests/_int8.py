"""Plain 64-bit forms of the int8 cache for the tests: written from the definition, token by token."""
import math

import torch


def near(x):
    """Nearest whole number, halves to the even one."""
    low = torch.floor(x)
    rest = x - low
    return low + ((rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2.0) == 1.0))).to(x.dtype)


def make_cache(pages, Hkv, P, D, device, seed=0, zero=False):
    g = torch.Generator().manual_seed(seed)
    k = torch.randint(-127, 128, (pages, Hkv, P, D), generator=g).to(torch.int8)
    v = torch.randint(-127, 128, (pages, Hkv, P // 16, D, 16), generator=g).to(torch.int8)
    ka = (torch.rand(pages, Hkv, generator=g) * 2 + 0.5).bfloat16().float()
    va = (torch.rand(pages, Hkv, generator=g) * 2 + 0.5).bfloat16().float()
    if zero:
        for t in (k, v, ka, va):
            t.zero_()
    return [t.to(device) for t in (k, v, ka, va)]


def v_rows(v):
    """[pages, Hkv, P / 16, D, 16] -> [pages, Hkv, P, D]"""
    p, h, n, d, s = v.shape
    return v.transpose(-1, -2).reshape(p, h, n * s, d)


def write(rows, amax, x, table, starts, cu):
    """One of K and V: ``rows`` [pages, Hkv, P, D] and ``amax`` in 64 bits, changed and returned."""
    P = rows.shape[2]
    for b, start in enumerate(starts):
        n = cu[b + 1] - cu[b]
        at = 0
        while at < n:
            page, lo = table[b][(start + at) // P], (start + at) % P
            c = min(P - lo, n - at)
            new = x[cu[b] + at:cu[b] + at + c].double().transpose(0, 1)
            old = amax[page].clone() if lo else torch.zeros_like(amax[page])
            top = torch.maximum(old, new.abs().amax((1, 2)))
            one = torch.where(top > 0, top, torch.ones_like(top))[:, None, None]
            if lo:
                grew = (top > old)[:, None, None]
                rows[page, :, :lo] = torch.where(grew, near(rows[page, :, :lo] * old[:, None, None] / one), rows[page, :, :lo])
            rows[page, :, lo:lo + c] = near(127 * new / one)
            amax[page] = top
            at += c
    return rows, amax


def attention(q, k_rows, v_rows_, ka, va, table, ctx, scale):
    """Result in 64 bits, and how far a kernel may be off it (before its rounding to bf16): scores summed in fp32 over
    products of fp16 values, weights rounded to fp16."""
    B, Hq, D = q.shape
    Hkv, P = k_rows.shape[1], k_rows.shape[2]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(out)
    for b, n in enumerate(ctx):
        if n == 0:
            continue
        pg = torch.tensor(table[b][:(n + P - 1) // P], device=q.device)
        k = (k_rows[pg].double() * ka[pg].double()[:, :, None, None] / 127).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
        v = (v_rows_[pg].double() * va[pg].double()[:, :, None, None] / 127).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
        qq = q[b].double().view(Hkv, -1, D)
        s = torch.einsum("hgd,hnd->hgn", qq, k) * scale
        w = torch.softmax(s, -1)
        out[b] = torch.einsum("hgn,hnd->hgd", w, v).reshape(Hq, D)
        # a score: at most 16 + D / 16 additions that each lose up to 2^-22 of the sum of |products|, four factors of 2^-24, and q's
        # small elements kept to 2^-24 of the row's largest; half again for the maximum that all scores are compared with
        mag = torch.einsum("hgd,hnd->hgn", qq.abs(), k.abs()).amax(-1)
        tiny = qq.abs().amax(-1) * k.abs().sum(-1).amax(-1, keepdim=True)
        ds = 2 * scale * ((16 + D / 16) * 2.0 ** -22 * mag + 4 * 2.0 ** -24 * mag + 2.0 ** -24 * tiny)
        # a weight: fp16's half step 2^-11, exp2's 2^-21, fp32 sums of them.  Below 2^-14 fp16 keeps 2^-25; the weight is stored times
        # its page's V magnitude over the largest page's, at least 1/8, and the largest weight is at least one: 8 * 2^-25 of that
        ew = 2 * ds + 2.0 ** -11 + 2.0 ** -20
        av = torch.einsum("hgn,hnd->hgd", w, v.abs())
        top = torch.exp(s.amax(-1) - torch.logsumexp(s, -1))
        off[b] = (ew[..., None] * av + (8 * 2.0 ** -25 * top)[..., None] * v.abs().sum(1)[:, None, :] + 2.0 ** -20 * av).reshape(Hq, D)
    return out, off


def default_scale(D):
    return 1.0 / math.sqrt(D)
