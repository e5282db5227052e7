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
        ds = 2 * abs(scale) * ((16 + D / 16) * 2.0 ** -22 * mag + 4 * 2.0 ** -24 * mag + 2.0 ** -24 * tiny)
        # a weight: fp16's half step 2^-11, exp2's 2^-21, fp32 sums of them.  Below 2^-14 fp16 keeps 2^-25; the weight is stored times
        # its page's V magnitude over the largest page's, at least 1/8, and the largest weight is at least one: 8 * 2^-25 of that
        ew = 2 * ds + 2.0 ** -11 + 2.0 ** -20
        av = torch.einsum("hgn,hnd->hgd", w, v.abs())
        top = torch.exp(s.amax(-1) - torch.logsumexp(s, -1))
        off[b] = (ew[..., None] * av + (8 * 2.0 ** -25 * top)[..., None] * v.abs().sum(1)[:, None, :] + 2.0 ** -20 * av).reshape(Hq, D)
    return out, off


def default_scale(D):
    return 1.0 / math.sqrt(D)


class Recorder:
    """Records every int8 operator call of a run, inputs and outputs, and checks each against the definition in 64 bits.
    (Whole models are not compared with unquantised ones: a rounding of one percent of a score of eighty is a factor of two in
    its weight, so nothing bounds that distance.)"""

    def __init__(self, monkeypatch):
        from axonml_b200.ops import int8, paged
        self.calls = []
        for mod, name in ((int8, "rms_norm_int8"), (int8, "swiglu_int8"), (int8, "quantize_int8"), (int8, "int8_linear"),
                          (paged, "kv_write_int8"), (paged, "decode_attention_int8")):
            monkeypatch.setattr(mod, name, self._wrap(name, getattr(mod, name)))

    def _wrap(self, name, fn):
        def call(*args, **kw):
            copy = [a.clone() if torch.is_tensor(a) else a for a in args]
            got = fn(*args, **kw)
            after = [a.clone() for a in args[2:6]] if name == "kv_write_int8" else got
            self.calls.append((name, copy, dict(kw), after))
            return got
        return call

    def names(self):
        return [c[0] for c in self.calls]

    def check(self):
        for name, a, kw, got in self.calls:
            getattr(self, "_" + name)(a, kw, got)

    @staticmethod
    def _rows(q, s, y, off):
        # half a step, and what the value itself and its scale are off: `off` of the row's largest value
        assert ((q.double() * s.double()[..., None] - y).abs() <= s.double()[..., None] * (0.5 + 127 * 2 * off)).all()
        assert ((s.double() - y.abs().amax(-1) / 127).abs() <= off * s.double()).all()

    def _rms_norm_int8(self, a, kw, got):
        x, w, eps = a[0], a[1], a[2]
        h = x if kw.get("residual") is None else x + kw["residual"]
        if kw.get("residual") is not None:
            assert torch.equal(got[2], h)
        d = h.double()
        # the sum of squares: at most D / 256 + 12 roundings in any order, halved by the root; eight more elsewhere
        off = (d.shape[-1] / 512 + 14) * 2.0 ** -24
        self._rows(got[0], got[1], d * torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + eps) * w.double(), off)

    def _swiglu_int8(self, a, kw, got):
        g, u = a[0].double().chunk(2, -1)
        # exp's two steps and its argument's rounding (below 2^5 here, times log2(e)), reciprocal's two, two products
        self._rows(got[0], got[1], g * torch.sigmoid(g) * u, (2 * 2 + 32 * 1.45 + 2 * 2 + 4) * 2.0 ** -24)

    def _quantize_int8(self, a, kw, got):
        self._rows(got[0], got[1], a[0].double(), 2 * 2.0 ** -24)

    def _int8_linear(self, a, kw, got):
        want = (a[0].double() @ a[2].double().t()) * a[1].double()[:, None] * a[3].double()
        assert got.dtype == torch.bfloat16 and ((got.double() - want).abs() <= (2.0 ** -8 + 4 * 2.0 ** -24) * want.abs()).all()

    def _kv_write_int8(self, a, kw, got):
        k, v, kc, vc, ka, va, table, starts = a[:8]
        n = k.shape[0] // table.shape[0]
        cu = [n * i for i in range(table.shape[0] + 1)]
        for x, rows, amax, c, m in ((k, kc, ka, got[0], got[2]), (v, v_rows(vc), va, v_rows(got[1]), got[3])):
            want = write(rows.double(), amax.double(), x, table.tolist(), starts.tolist(), cu)
            assert torch.equal(c.double(), want[0]) and torch.equal(m.double(), want[1])

    def _decode_attention_int8(self, a, kw, got):
        q, kc, vc, ka, va, table, ctx = a[:7]
        want, off = attention(q, kc, v_rows(vc), ka, va, table.tolist(), ctx.tolist(), default_scale(q.shape[-1]))
        assert ((got.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all()


def far_below(n, ctx, device):
    """A cache whose keys are all alike, a query that scores each -1.1e32, and what attention gives: the mean of the values."""
    B, D, P = len(ctx), 128, 16
    per = (n + P - 1) // P
    kc, vc, ka, va = make_cache(B * per, 1, P, D, device, seed=5)
    kc.fill_(127)
    ka.fill_(1e31)
    table = torch.arange(B * per, dtype=torch.int32, device=device).view(B, per)
    q = torch.full((B, 2, D), -1.0, dtype=torch.bfloat16, device=device)
    rows = v_rows(vc).double() * (va.double() / 127)[..., None, None]
    want = torch.stack([rows[table[b].long(), 0].reshape(-1, D)[:c].mean(0).expand(2, D) for b, c in enumerate(ctx)])
    return [kc, vc, ka, va], q, table, want


def far_below_off(want, dtype):
    """Equal scores: weights of one and a sum that is exact; the weights times a page's magnitude ratio are rounded to fp16
    (2^-11 of the values, whose mean of magnitudes is below 8 here), the result to its type."""
    return 2.0 ** -11 * 8 + torch.finfo(dtype).eps / 2 * (want.abs() + 2.0 ** -8)
