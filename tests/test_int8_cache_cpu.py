"""int8 paged cache on the CPU path: writes against the definition in 64 bits, attention, refusals."""
import pytest
import torch

import _int8 as R
from axonml_b200.ops import paged


def _case(B, lens, starts, Hkv, P, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    need = [(s + n + P - 1) // P for s, n in zip(starts, lens)]
    perm = torch.randperm(sum(need) + 2, generator=g).tolist()
    table, at = torch.zeros(B, max(need + [1]), dtype=torch.int32), 0
    for b, c in enumerate(need):
        table[b, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
        at += c
    T = sum(lens)
    k, v = torch.randn(T, Hkv, D, generator=g).bfloat16(), torch.randn(T, Hkv, D, generator=g).bfloat16()
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    return k, v, table, torch.tensor(starts, dtype=torch.int32), cu, sum(need) + 2


@pytest.mark.parametrize("lens,starts", [([1, 1, 1], [0, 15, 16]), ([40, 0, 3, 17], [0, 5, 30, 31]), ([5], [12])])
@pytest.mark.parametrize("P", [16, 32])
def test_writes_follow_the_definition(lens, starts, P):
    k, v, table, st, cu, pages = _case(len(lens), lens, starts, 2, P, 16)
    kc, vc, ka, va = R.make_cache(pages, 2, P, 16, "cpu")
    want_k = R.write(kc.double(), ka.double(), k, table.tolist(), starts, cu.tolist())
    want_v = R.write(R.v_rows(vc).double(), va.double(), v, table.tolist(), starts, cu.tolist())
    for _ in range(2):                                    # the same rows again change nothing
        paged.kv_write_int8(k, v, kc, vc, ka, va, table, st, cu)
        assert torch.equal(kc.double(), want_k[0]) and torch.equal(ka.double(), want_k[1])
        assert torch.equal(R.v_rows(vc).double(), want_v[0]) and torch.equal(va.double(), want_v[1])


def test_tokens_one_by_one_stay_near_the_values():
    """A page filled token by token is rounded again whenever it grows: still within a step per growth."""
    D, P = 16, 16
    kc, vc, ka, va = R.make_cache(1, 1, P, D, "cpu", zero=True)
    x = torch.randn(P, 1, D).bfloat16()
    table, grows = torch.zeros(1, 1, dtype=torch.int32), 0
    for t in range(P):
        before = ka.clone()
        paged.kv_write_int8(x[t:t + 1], x[t:t + 1], kc, vc, ka, va, table, torch.tensor([t], dtype=torch.int32))
        grows += int((ka > before).any())
    step = ka.item() / 127
    assert ka.item() == x.float().abs().max().item()
    assert (kc[0, 0].float() * step - x[:, 0].float()).abs().max().item() <= 0.5 * step * (grows + 1) * 1.0001
    assert torch.equal(R.v_rows(vc), kc)


def test_attention_over_what_was_written():
    Hkv, G, P, D = 2, 3, 16, 32
    lens, starts = [35, 1, 20], [0, 0, 0]
    k, v, table, st, cu, pages = _case(3, lens, starts, Hkv, P, D)
    kc, vc, ka, va = R.make_cache(pages, Hkv, P, D, "cpu", zero=True)
    paged.kv_write_int8(k, v, kc, vc, ka, va, table, st, cu)
    q = torch.randn(3, Hkv * G, D)
    ctx = torch.tensor([35, 0, 20], dtype=torch.int32)
    got = paged.decode_attention_int8(q, kc, vc, ka, va, table, ctx)
    want, _ = R.attention(q, kc, R.v_rows(vc), ka, va, table.tolist(), ctx.tolist(), R.default_scale(D))
    assert torch.allclose(got.double(), want, rtol=1e-5, atol=1e-6) and got[1].eq(0).all()
    dense_k, dense_v = k[:35].float(), v[:35].float()
    s = torch.einsum("hgd,nhd->hgn", q[0].view(Hkv, G, D), dense_k) / D ** 0.5
    ref = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), dense_v).reshape(-1, D)
    # a step of a page is at most max|x| / 127 and a value half a step off; scores move by that times sum|q|
    ds = 0.5 * dense_k.abs().max() / 127 * q[0].abs().sum(-1).max() / D ** 0.5
    assert (got[0] - ref).abs().max() <= 0.5 * dense_v.abs().max() / 127 + (torch.exp(2 * ds) - 1) * dense_v.abs().max()


def _good():
    k, v, table, st, cu, pages = _case(2, [3, 2], [0, 4], 2, 16, 16)
    c = R.make_cache(pages, 2, 16, 16, "cpu")
    return dict(k=k, v=v, k_cache=c[0], v_cache=c[1], k_amax=c[2], v_amax=c[3], block_table=table, starts=st, cu_seqlens=cu)


@pytest.mark.parametrize("change,err", [
    (dict(k=lambda t: t[:, :1]), ValueError), (dict(v=lambda t: t.float()), ValueError), (dict(k_cache=lambda t: t.float()), TypeError),
    (dict(v_cache=lambda t: R.v_rows(t)), ValueError), (dict(k_amax=lambda t: t[:, :1]), ValueError), (dict(v_amax=lambda t: t.double()), TypeError),
    (dict(block_table=lambda t: t.long()), TypeError), (dict(starts=lambda t: t[:1]), ValueError), (dict(starts=lambda t: t.long()), ValueError),
    (dict(cu_seqlens=lambda t: t[:2]), ValueError), (dict(cu_seqlens=lambda t: None), ValueError), (dict(starts=lambda t: t - 1), ValueError),
    (dict(starts=lambda t: t + 100), ValueError), (dict(block_table=lambda t: t + 100), ValueError), (dict(block_table=lambda t: t - 100), ValueError),
    (dict(cu_seqlens=lambda t: t + 9), ValueError), (dict(k_cache=lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)), ValueError),
    (dict(k_cache=lambda t: t[:, :, :8]), ValueError),
])
def test_write_refusals(change, err):
    a = _good()
    for name, f in change.items():
        a[name] = f(a[name])
    with pytest.raises(err):
        paged.kv_write_int8(**a)


@pytest.mark.parametrize("change,err", [
    (dict(q=lambda t: t[:1]), ValueError), (dict(q=lambda t: t[:, :3]), ValueError), (dict(q=lambda t: t[..., :8]), ValueError),
    (dict(ctx_lens=lambda t: t.long()), ValueError), (dict(ctx_lens=lambda t: t + 1000), ValueError), (dict(ctx_lens=lambda t: t - 50), ValueError),
    (dict(block_table=lambda t: t + 100), ValueError), (dict(v_amax=lambda t: t[:1]), ValueError),
])
def test_attention_refusals(change, err):
    g = _good()
    a = dict(q=torch.randn(2, 4, 16), ctx_lens=torch.tensor([3, 6], dtype=torch.int32),
             **{n: g[n] for n in ("k_cache", "v_cache", "k_amax", "v_amax", "block_table")})
    for name, f in change.items():
        a[name] = f(a[name])
    with pytest.raises(err):
        paged.decode_attention_int8(**a)


def test_no_gradients_and_no_heads():
    a = _good()
    with pytest.raises(RuntimeError):
        paged.kv_write_int8(**{**a, "k": a["k"].float().requires_grad_(), "v": a["v"].float()})
    caches = {n: a[n] for n in ("k_cache", "v_cache", "k_amax", "v_amax", "block_table")}
    q, cl = torch.randn(2, 4, 16, requires_grad=True), torch.tensor([3, 6], dtype=torch.int32)
    with pytest.raises(RuntimeError):
        paged.decode_attention_int8(q, **caches, ctx_lens=cl)
    with torch.no_grad():
        paged.decode_attention_int8(q, **caches, ctx_lens=cl)
    none = R.make_cache(2, 0, 16, 16, "cpu")
    with pytest.raises(ValueError):
        paged.decode_attention_int8(q.detach(), *none, a["block_table"], cl)


@pytest.mark.parametrize("n,ctx", [(1, [1]), (40, [40, 17])])
def test_attention_of_scores_far_below_zero(n, ctx):
    """Scores near -1e32: the weights are those of the differences."""
    c, q, table, want = R.far_below(n, ctx, "cpu")
    got = paged.decode_attention_int8(q, *c, table, torch.tensor(ctx, dtype=torch.int32))
    assert ((got.double() - want).abs() <= R.far_below_off(want, q.dtype)).all()
