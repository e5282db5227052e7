"""The 8-bit serving operators: what is measured, and their plain forms.

Four operators that a decoder served in 8 bits is made of, as ``axonml_b200.ops`` offers them:

* ``norm``: root-mean-square norm of ``x + residual`` to int8 rows with one scale a row,
* ``swiglu``: ``silu(gate) * up`` to int8 rows with one scale a row,
* ``linear``: int8 rows times an int8 matrix, a scale for each row and each output channel,
* ``write`` / ``attention``: a paged K/V cache of int8 with one magnitude for each page and head -
  new tokens written to it, and one query token per sequence attending over it.

``run`` takes the plain form (elementary torch operations) where ``own`` is false and the
framework's operators where it is true.  What is held in 8 bits is returned as the values it stands
for, in bf16."""
import math

import torch

own = False

BF, F32, I32, I8 = torch.bfloat16, torch.float32, torch.int32, torch.int8


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token through the norm of an 8B-sized decoder: a decode step of a single user
        {"name": "norm 1x4096", "op": "norm", "rows": 1, "dim": 4096, "residual": True, "dtype": "bf16"},
        # a prefill of 8192 tokens, the residual stream updated on the way
        {"name": "norm 8192x4096", "op": "norm", "rows": 8192, "dim": 4096, "residual": True, "dtype": "bf16"},
        # an fp32 stream of an odd width, no residual: an embedding's first norm
        {"name": "norm 1021x5125 fp32", "op": "norm", "rows": 1021, "dim": 5125, "residual": False, "dtype": "fp32"},
        # the feed-forward gate of a full decode batch
        {"name": "swiglu 64x14336", "op": "swiglu", "rows": 64, "dim": 14336, "dtype": "bf16"},
        # the same for a prefill, with the 7B model's width
        {"name": "swiglu 4096x11008", "op": "swiglu", "rows": 4096, "dim": 11008, "dtype": "bf16"},
        # the q|k|v product of one decoded token: nothing but the weights' bytes
        {"name": "linear 1x6144x4096", "op": "linear", "rows": 1, "out": 6144, "in": 4096, "bias": False, "dtype": "bf16"},
        # the gate|up product of a decode batch of 64
        {"name": "linear 64x28672x4096", "op": "linear", "rows": 64, "out": 28672, "in": 4096, "bias": False, "dtype": "bf16"},
        # the gate|up product of a prefill: bound by the tensor cores
        {"name": "linear 8192x28672x4096", "op": "linear", "rows": 8192, "out": 28672, "in": 4096, "bias": False, "dtype": "bf16"},
        # a prefill of several prompts of different lengths into the cache, behind what they hold already
        {"name": "write 8192 in 7", "op": "write", "tokens": 8192, "seqs": 7, "kv": 8, "dim": 128, "page": 16, "start": 40},
        # a decode batch: one token each, somewhere inside a page
        {"name": "write 64 in 64", "op": "write", "tokens": 64, "seqs": 64, "kv": 8, "dim": 128, "page": 16, "start": 60},
        # one user with a short context: latency
        {"name": "attention 1 x 777", "op": "attention", "seqs": 1, "ctx": 777, "heads": 32, "kv": 8, "dim": 128, "page": 16, "spread": 0.0},
        # a full batch with ragged contexts: the cache's bytes
        {"name": "attention 64 x 8192", "op": "attention", "seqs": 64, "ctx": 8192, "heads": 32, "kv": 8, "dim": 128, "page": 16, "spread": 0.7},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "swiglu", "linear", "write", "attention"])
    if op in ("norm", "swiglu"):
        dim = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            dim = max(16, dim // 16 * 16)
        rows = _log(rng, 1, max(1, min(16384, 8192 * 4096 // dim)))
        case = {"op": op, "rows": rows, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "fp32"])}
        if op == "norm":
            case["residual"] = rng.random() < 0.6
        return case
    if op == "linear":
        k, n = _log(rng, 64, 16384), _log(rng, 16, 32768)
        if rng.random() < 0.6:
            k, n = max(32, k // 32 * 32), max(32, n // 32 * 32)
        most = 8192 * 28672 * 4096 // (n * k)
        return {"op": op, "rows": _log(rng, 1, max(1, min(8192, most))), "out": n, "in": k,
                "bias": rng.random() < 0.3, "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    dim, kv, page = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 5, 8, 16]), rng.choice([16, 16, 32, 64])
    if op == "write":
        seqs = _log(rng, 1, 64)
        tokens = seqs if rng.random() < 0.4 else _log(rng, seqs, max(seqs, 8192 * 8 * 128 // (kv * dim)))
        return {"op": op, "tokens": min(tokens, 16384), "seqs": seqs, "kv": kv, "dim": dim, "page": page, "start": _log(rng, 1, 200)}
    seqs, group = _log(rng, 1, 128), rng.choice([1, 2, 4, 5, 7, 8, 16])
    most = 64 * 8192 * 8 * 128 // 2
    ctx = _log(rng, 1, max(1, min(65536, most // (seqs * kv * dim * max(1, group // 4)))))
    return {"op": op, "seqs": seqs, "ctx": ctx, "heads": kv * group, "kv": kv, "dim": dim, "page": page,
            "spread": rng.choice([0.0, 0.5, 1.0])}


# ----------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F32).to(dtype)


def _rows16(n, k):
    """An int8 matrix whose rows start on 16-byte boundaries, as the framework's quantisers lay them out."""
    return torch.empty(n, (k + 15) // 16 * 16, dtype=I8, device="cuda")[:, :k]


def _lengths(g, n, total):
    """`n` lengths of at least one that add up to `total`."""
    if n == total:
        return [1] * n
    cuts = torch.rand(n, generator=g, device="cuda").cumsum(0)
    cuts = [0] + [int(c) for c in (cuts / cuts[-1] * (total - n)).round().long().tolist()]
    cuts[-1] = total - n
    return [1 + max(0, cuts[i + 1] - cuts[i]) for i in range(n)]


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = {"op": op, "case": dict(case)}
    if op in ("norm", "swiglu"):
        dt = BF if case["dtype"] == "bf16" else F32
        rows, dim = case["rows"], case["dim"]
        if op == "norm":
            # a residual stream: some channels are far larger than the others
            big = 1.0 + 20.0 * (torch.rand(dim, generator=g, device="cuda") < 0.01).float()
            s["x"] = (_randn(g, rows, dim) * big).to(dt)
            s["residual"] = _randn(g, rows, dim, dtype=dt) if case["residual"] else None
            s["weight"] = (1.0 + 0.2 * _randn(g, dim)).to(dt)
        else:
            s["x"] = _randn(g, rows, 2 * dim, dtype=dt)
        return s
    if op == "linear":
        m, n, k = case["rows"], case["out"], case["in"]
        s["q"], s["w"] = _rows16(m, k), _rows16(n, k)
        for t in (s["q"], s["w"]):      # rows quantised from a bell curve whose largest value sits near three sigma and a half
            for a in range(0, t.shape[0], 4096):
                t[a:a + 4096] = (_randn(g, *t[a:a + 4096].shape) * 36.0).round_().clamp_(-127, 127).to(I8)
        s["q_scale"] = torch.rand(m, generator=g, device="cuda") * 0.03 + 0.01
        s["w_scale"] = torch.rand(n, generator=g, device="cuda") * 4e-4 + 2e-4
        s["bias"] = _randn(g, n, dtype=F32) if case["bias"] else None
        s["dtype"] = BF if case["dtype"] == "bf16" else F32
        return s
    kv, dim, page = case["kv"], case["dim"], case["page"]
    if op == "write":
        n, t = case["seqs"], case["tokens"]
        shape = _gen(n * 100003 + t)      # lengths go by the case: the cache of another seed has as many pages
        lens = _lengths(shape, n, t)
        start = (torch.rand(n, generator=shape, device="cuda") * (case["start"] + 1)).long().tolist()
        need = [(a + b + page - 1) // page for a, b in zip(start, lens)]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device="cuda").tolist()
        table = torch.zeros(n, max(need), dtype=I32)
        for i, c in enumerate(need):
            table[i, :c] = torch.tensor(order[:c], dtype=I32)
            order = order[c:]
        s["table"], s["starts"] = table.cuda(), torch.tensor(start, dtype=I32).cuda()
        s["cu"] = torch.tensor([0] + lens, dtype=I32).cumsum(0).to(I32).cuda()
        s["tokens"] = t
        # keys have a few strong channels, values none
        strong = 1.0 + 6.0 * (torch.rand(kv, dim, generator=g, device="cuda") < 0.05).float()
        s["k"], s["v"] = (_randn(g, t, kv, dim) * strong).to(BF), _randn(g, t, kv, dim, dtype=BF)
    else:
        n, most = case["seqs"], case["ctx"]
        ctx = (most * (1.0 - case["spread"] * torch.rand(n, generator=g, device="cuda"))).round().long().clamp(0, most)
        ctx[0] = most
        need = ((ctx + page - 1) // page).tolist()
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(I32)
        table, at = torch.zeros(n, max(need), dtype=I32, device="cuda"), 0
        for i, c in enumerate(need):
            table[i, :c] = order[at:at + c]
            at += c
        s["table"], s["ctx"] = table, ctx.to(I32)
        s["q"] = _randn(g, n, case["heads"], dim, dtype=BF)
    s["k_cache"] = torch.randint(-127, 128, (pages, kv, page, dim), generator=g, device="cuda", dtype=I8)
    s["v_cache"] = torch.randint(-127, 128, (pages, kv, page // 16, dim, 16), generator=g, device="cuda", dtype=I8)
    s["k_amax"] = torch.rand(pages, kv, generator=g, device="cuda") * 2.0 + (1.0 if op == "attention" else 2.0)
    s["v_amax"] = torch.rand(pages, kv, generator=g, device="cuda") * 2.0 + 1.0
    if op == "write":                   # magnitudes that earlier bf16 tokens left: bf16 values themselves
        s["k_amax"], s["v_amax"] = s["k_amax"].to(BF).float(), s["v_amax"].to(BF).float()
    return s


# ------------------------------------------------------------------------------------ plain forms
def _values(q, scale):
    """What int8 stands for, in bf16."""
    return torch.mul(q, scale, out=torch.empty(q.shape, dtype=BF, device=q.device))


def _to_int8(t, amax):
    """round(127 t / amax), ties to even; nothing where the magnitude is nothing.  The quotient of
    two exact numbers rounds once, so a value next to a border stays on its side of it."""
    return torch.where(amax > 0, (t * 127.0 / amax).round(), torch.zeros_like(t)).to(I8)


def _plain_norm(s):
    x, r = s["x"], s["residual"]
    h = x if r is None else x + r
    hf = h.float()
    t = hf * s["weight"].float()
    amax = t.abs().amax(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(hf.square().mean(-1, keepdim=True) + 1e-5)
    q, scale = _to_int8(t, amax), amax * rstd / 127.0
    out = {"values": _values(q, scale), "scale": scale.squeeze(-1)}
    if r is not None:
        out["stream"] = h
    return out


def _plain_swiglu(s):
    g, u = s["x"].float().chunk(2, dim=-1)
    y = g / (1.0 + torch.exp(-g)) * u
    amax = y.abs().amax(-1, keepdim=True)
    scale = amax / 127.0
    return {"values": _values(_to_int8(y, amax), scale), "scale": scale.squeeze(-1)}


def _plain_linear(s):
    y = s["q"].float() @ s["w"].float().t()
    y = y * s["q_scale"][:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["dtype"])


def _write_one(x, cache, amax, table_page, slot, first, touched, transposed):
    """The new rows of one of K and V into its pages: the page's magnitude grows to the largest it
    holds, what it held before the first new slot is scaled to it, the new rows are rounded to it."""
    pages, kv = amax.shape
    new = torch.zeros_like(amax).scatter_reduce_(0, table_page[:, None].expand(-1, kv), x.float().abs().amax(-1), "amax")
    old = torch.where((first == 0)[:, None], torch.zeros_like(amax), amax)       # a page begun anew forgets
    grown = torch.where(touched[:, None], torch.maximum(old, new), amax)
    rows = cache.permute(0, 2, 4, 1, 3).reshape(pages, -1, kv, x.shape[-1]) if transposed else cache.transpose(1, 2)
    ratio = rows.float() * old[:, None, :, None] / torch.where(grown > 0, grown, torch.ones_like(grown))[:, None, :, None]
    scaled = ratio.round().to(I8)
    held = torch.arange(rows.shape[1], device=x.device)[None, :] < first[:, None]
    again = (held & touched[:, None])[:, :, None, None] & (grown > old)[:, None, :, None]
    rows = torch.where(again, scaled, rows)
    rows[table_page, slot] = _to_int8(x.float(), grown[table_page][:, :, None])
    if transposed:
        cache.copy_(rows.view(pages, -1, 16, kv, x.shape[-1]).permute(0, 3, 1, 4, 2))
    else:
        cache.copy_(rows.transpose(1, 2))
    amax.copy_(grown)


def _plain_write(s):
    page = s["case"]["page"]
    token = torch.arange(s["tokens"], device="cuda", dtype=I32)
    row = torch.searchsorted(s["cu"][1:], token, right=True)
    pos = (s["starts"][row] + token - s["cu"][row]).long()
    at, slot = s["table"][row, pos // page].long(), pos % page
    first = torch.full((s["k_amax"].shape[0],), page, device="cuda").scatter_reduce_(0, at, slot, "amin")
    touched = first < page
    _write_one(s["k"], s["k_cache"], s["k_amax"], at, slot, first, touched, False)
    _write_one(s["v"], s["v_cache"], s["v_amax"], at, slot, first, touched, True)


def _plain_attention(s):
    q, table, ctx = s["q"].float(), s["table"].long(), s["ctx"]
    b, hq, d = q.shape
    kv = s["k_amax"].shape[1]
    length = table.shape[1] * s["case"]["page"]
    k = s["k_cache"][table].float() * (s["k_amax"][table] / 127.0)[..., None, None]            # [B, pages, kv, page, D]
    k = k.transpose(1, 2).reshape(b, kv, length, d)
    score = torch.matmul(q.view(b, kv, hq // kv, d), k.transpose(2, 3)) / math.sqrt(d)
    del k
    seen = (torch.arange(length, device="cuda")[None, :] < ctx[:, None])[:, None, None, :]
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = s["v_cache"][table].float() * (s["v_amax"][table] / 127.0)[..., None, None, None]      # [B, pages, kv, page/16, D, 16]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(b, kv, length, d)
    out = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return out.view(b, hq, d).to(BF)


# -------------------------------------------------------------------------------------------- run
def _held(s):
    return {"k": _values(s["k_cache"], (s["k_amax"] / 127.0)[:, :, None, None]), "k_amax": s["k_amax"],
            "v": _values(s["v_cache"], (s["v_amax"] / 127.0)[:, :, None, None, None]), "v_amax": s["v_amax"]}


def run(s):
    op = s["op"]
    if own:
        from axonml_b200.ops import int8, paged
        if op == "norm":
            got = int8.rms_norm_int8(s["x"], s["weight"], 1e-5, residual=s["residual"])
            out = {"values": _values(got[0], got[1][:, None]), "scale": got[1]}
            if s["residual"] is not None:
                out["stream"] = got[2]
            return out
        if op == "swiglu":
            q, scale = int8.swiglu_int8(s["x"])
            return {"values": _values(q, scale[:, None]), "scale": scale}
        if op == "linear":
            return int8.int8_linear(s["q"], s["q_scale"], s["w"], s["w_scale"], bias=s["bias"], out_dtype=s["dtype"])
        if op == "write":
            paged.kv_write_int8(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_amax"], s["v_amax"], s["table"], s["starts"],
                                cu_seqlens=s["cu"])
            return _held(s)
        return paged.decode_attention_int8(s["q"], s["k_cache"], s["v_cache"], s["k_amax"], s["v_amax"], s["table"], s["ctx"])
    if op == "norm":
        return _plain_norm(s)
    if op == "swiglu":
        return _plain_swiglu(s)
    if op == "linear":
        return _plain_linear(s)
    if op == "write":
        _plain_write(s)
        return _held(s)
    return _plain_attention(s)


# ---------------------------------------------------------------------------------- 64-bit answers
def _near(x):
    """Nearest whole number, halves to the even one."""
    low = torch.floor(x)
    rest = x - low
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2.0) == 1.0))
    return low + up


def _steps(t, top):
    return torch.where(top > 0, _near(127.0 * t / torch.where(top > 0, top, torch.ones_like(top))), torch.zeros_like(t))


def _exact_rows(t, norm):
    top = t.abs().max(-1, keepdim=True).values
    scale = top * norm / 127.0
    return {"values": _steps(t, top) * scale, "scale": scale[:, 0]}


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "norm":
        h = s["x"] if s["residual"] is None else s["x"] + s["residual"]       # the stream keeps its type's rounding
        d = h.double()
        out = _exact_rows(d * s["weight"].double(), (d.pow(2).sum(-1, keepdim=True) / d.shape[-1] + 1e-5).pow(-0.5))
        if s["residual"] is not None:
            out["stream"] = s["x"].double() + s["residual"].double()
        return out
    if op == "swiglu":
        n = case["dim"]
        d = s["x"].double()
        return _exact_rows(d[:, :n] * torch.special.expit(d[:, :n]) * d[:, n:], 1.0)
    if op == "linear":
        if 2.0 * case["rows"] * case["out"] * case["in"] > 2.5e12:
            return None
        w = s["w"].double().t() * s["w_scale"].double()
        y = torch.cat([(s["q"][a:a + 1024].double() * s["q_scale"][a:a + 1024, None].double()) @ w
                       for a in range(0, case["rows"], 1024)])
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "write":
        page, out = case["page"], {}
        cu, starts, table = s["cu"].tolist(), s["starts"].tolist(), s["table"].tolist()
        for name in ("k", "v"):
            rows = s[name + "_cache"].double()
            if name == "v":
                rows = rows.transpose(-1, -2).reshape(rows.shape[0], rows.shape[1], page, -1)
            amax, x = s[name + "_amax"].double().clone(), s[name].double()
            for i in range(len(starts)):
                at, end = starts[i], starts[i] + cu[i + 1] - cu[i]
                src = cu[i]
                while at < end:                                   # page by page, as a sequence fills them
                    p, lo = table[i][at // page], at % page
                    n = min(page - lo, end - at)
                    new = x[src:src + n].transpose(0, 1)          # [kv, n, D]
                    before = amax[p] if lo else torch.zeros_like(amax[p])
                    top = torch.maximum(before, new.abs().amax((1, 2)))
                    if lo:
                        t = top[:, None, None]
                        kept = _near(rows[p, :, :lo] * before[:, None, None] / torch.where(t > 0, t, torch.ones_like(t)))
                        rows[p, :, :lo] = torch.where((top > before)[:, None, None], kept, rows[p, :, :lo])
                    rows[p, :, lo:lo + n] = _steps(new, top[:, None, None].expand_as(new))
                    amax[p] = top
                    at, src = at + n, src + n
            out[name + "_amax"] = amax
            held = rows * (amax / 127.0)[:, :, None, None]
            if name == "v":
                held = held.view(rows.shape[0], rows.shape[1], page // 16, 16, -1).transpose(-1, -2).contiguous()
            out[name] = held
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    kv, page, d = case["kv"], case["page"], case["dim"]
    for i, n in enumerate(s["ctx"].tolist()):
        if n == 0:
            continue
        pg = s["table"][i, :(n + page - 1) // page].long()
        k = (s["k_cache"][pg].double() * s["k_amax"][pg].double()[:, :, None, None] / 127).permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :n]
        v = (s["v_cache"][pg].double() * s["v_amax"][pg].double()[:, :, None, None, None] / 127)
        v = v.permute(1, 0, 2, 4, 3).reshape(kv, -1, d)[:, :n]
        w = torch.softmax(torch.einsum("hgd,hnd->hgn", s["q"][i].double().view(kv, -1, d), k) / math.sqrt(d), -1)
        out[i] = torch.einsum("hgn,hnd->hgd", w, v).reshape(-1, d)
    return out


# ------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op in ("norm", "swiglu"):
        n, width = case["rows"] * case["dim"], 2 if case["dtype"] == "bf16" else 4
        if op == "norm":
            moved = n * width * (3 if case["residual"] else 1) + case["dim"] * width
        else:
            moved = 2 * n * width
        return {"bytes": moved + 2 * n + 4 * case["rows"], "flops": n * (6 if op == "norm" else 8)}
    if op == "linear":
        m, n, k = case["rows"], case["out"], case["in"]
        return {"bytes": m * k + n * k + m * n * (2 if case["dtype"] == "bf16" else 4) + 4 * (m + n + (n if case["bias"] else 0)),
                "flops": 2 * m * n * k}
    if op == "write":
        n = case["tokens"] * case["kv"] * case["dim"] * 2
        return {"bytes": n * (2 + 2) + 8 * case["kv"] * -(-case["tokens"] // case["page"]), "flops": 3 * n}
    tokens = case["ctx"] + (case["seqs"] - 1) * case["ctx"] * (1.0 - case["spread"] / 2)
    return {"bytes": tokens * case["kv"] * (2 * case["dim"] + 8 / case["page"]) + 4 * case["seqs"] * case["heads"] * case["dim"],
            "flops": 4 * tokens * case["heads"] * case["dim"]}
