"""RMS norm to int8 rows of very large and very small values on the GPU."""
import pytest
import torch

import _int8_norm_range as C
from axonml_b200.ops import int8 as I

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [8, 60, 1000, 4096, 5125, 16384, 20001])       # rows in one warp, in registers, walked twice, off the 16-byte grid
@pytest.mark.parametrize("size,wsize,eps", C.CASES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("res", [False, True])
def test_norm_of_rows_at_the_ends_of_the_range(D, size, wsize, eps, dt, res, kernel_status):
    x, r, w = (None if t is None else t.cuda() for t in C.inputs(size, wsize, D, dt, res))
    C.check(I.rms_norm_int8(x, w, eps, residual=r), x, r, w, eps, D)


@pytest.mark.parametrize("D", [64, 2048, 4096])
def test_far_rows_among_many(D, kernel_status):
    """Blocks that take many rows each: the far ones are done again, the others keep their bits."""
    x = torch.randn(3000, D, device="cuda")
    w = 1 + 0.1 * torch.randn(D, device="cuda")
    q, s = I.rms_norm_int8(x, w)
    far = torch.rand(3000, device="cuda") < 0.3
    y = torch.where(far[:, None], x * 2.0 ** 80, x)
    q2, s2 = I.rms_norm_int8(y, w)
    assert torch.equal(q2, q) and torch.equal(s2[~far], s[~far])
    # without an eps beside the squares, and summed in another order: 81 / 2 + 8 roundings each
    want = x.double().mul(w.double()).abs().amax(-1) * torch.rsqrt(x.double().pow(2).mean(-1)) / 127
    assert ((s2.double() - want)[far].abs() <= 50 * 2.0 ** -24 * want[far]).all()


def test_values_that_are_not_finite_give_scales_that_are_not(kernel_status):
    for D in (64, 100, 9000):
        x = torch.randn(400, D, device="cuda")
        bad = torch.arange(400, device="cuda") % 7 == 3
        x[bad, 5] = float("inf")
        x[3, 5] = float("nan")
        q, s, h = I.rms_norm_int8(x, torch.ones(D, device="cuda"), residual=torch.zeros_like(x))
        assert torch.equal(s.isfinite(), ~bad) and torch.equal(h.isfinite().all(-1), ~bad)
