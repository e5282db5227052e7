"""Rounding to int8 steps at the ends of fp32's range: quotients on the border between two steps go to the even one."""
import pytest
import torch

import _int8 as R
from axonml_b200.ops import int8 as I
from axonml_b200.ops import paged

pytestmark = pytest.mark.gpu


def _rows():
    """Rows x * (254, k, -k, ...) with odd k, so that 127 t / max|t| = k / 2 exactly, for x of a few bits at every exponent."""
    k = torch.arange(1, 254, 2, dtype=torch.float64)
    unit = torch.cat([torch.tensor([254.0], dtype=torch.float64), k, -k])          # 255 values
    x = torch.tensor([m * 2.0 ** e for e in range(-126, 120) for m in (1, 3, 5, 7, 11, 13)], dtype=torch.float64)
    x = x[(254 * x >= I.TINY) & (254 * x < 2.0 ** 128)]
    return x[:, None] * unit, torch.cat([torch.tensor([127.0], dtype=torch.float64), R.near(k / 2), R.near(-k / 2)])


@pytest.mark.parametrize("pad", [0, 1])                   # rows on the 16-byte grid, and off it
def test_rows_on_borders(pad, kernel_status):
    t, want = _rows()
    t = torch.cat([t, torch.zeros(len(t), 1 + pad, dtype=torch.float64)], 1)
    x = t.float().cuda()
    assert torch.equal(x.double().cpu(), t)
    q, s = I.quantize_int8(x)
    wrong = (q[:, :255].double().cpu() != want).any(-1)
    assert not wrong.any(), t[wrong][:, 0].tolist()[:10]
    a = t[:, 0] / 127
    assert ((s.double().cpu() - a).abs() <= 2.0 ** -23 * a).all()
    q, s = I.rms_norm_int8(x, torch.ones(x.shape[1], device="cuda"))
    wrong = (q[:, :255].double().cpu() != want).any(-1)
    assert not wrong.any(), t[wrong][:, 0].tolist()[:10]


@pytest.mark.parametrize("P,D", [(16, 64), (32, 128)])
def test_cache_rows_on_borders(P, D, kernel_status):
    """New rows as above, and what a page held: q a_old / a_new on borders."""
    t, want = _rows()
    n = len(t)
    unit = torch.zeros(n, 256, dtype=torch.float64)
    unit[:, :255] = t
    k = unit.view(n, 256 // D, D).float().cuda()                       # a sequence of 256 / D tokens in one head
    T = 256 // D
    for held in (0, 5):                                                # tokens that the page holds already
        kc, vc, ka, va = R.make_cache(n, 1, P, D, "cuda", seed=held)
        top = t[:, 0].float().cuda()
        old = (3 * top.double() / 14).float()                            # below the new magnitude: 3 q / 14 lies on a border for q = 7, 21, ...
        exact = (old.double() * 14 == 3 * top.double()) & (old.double() >= I.TINY)
        ka[:, 0], va[:, 0] = old, old
        kc[:, :, 0], vc[..., 0] = 7, 21
        before = [x.clone() for x in (kc, vc)]
        st = torch.full((n,), held, dtype=torch.int32, device="cuda")
        table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None]
        paged.kv_write_int8(k.reshape(n * T, 1, D), k.reshape(n * T, 1, D), kc, vc, ka, va, table, st)
        for rows, b in ((kc, before[0]), (R.v_rows(vc), R.v_rows(before[1]))):
            got = rows[:, 0, held:held + T].reshape(n, 256)[:, :255].double().cpu()
            wrong = (got != want).any(-1)
            assert not wrong.any(), t[wrong][:, 0].tolist()[:10]
            if held:
                kept = R.near(b[:, 0, :held].double() * old.double()[:, None, None] / top.double()[:, None, None])
                wrong = (rows[:, 0, :held].double() != kept).flatten(1).any(-1) & exact
                assert not wrong.any(), top[wrong].tolist()[:10]
        assert torch.equal(ka[:, 0], top) and torch.equal(va[:, 0], top)
