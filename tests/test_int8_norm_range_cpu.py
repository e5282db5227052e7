"""RMS norm to int8 rows of very large and very small values, on the CPU path."""
import pytest
import torch

import _int8_norm_range as C
from axonml_b200.ops import int8 as I


@pytest.mark.parametrize("size,wsize,eps", C.CASES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("res", [False, True])
def test_norm_of_rows_at_the_ends_of_the_range(size, wsize, eps, dt, res):
    x, r, w = C.inputs(size, wsize, 60, dt, res)
    C.check(I.rms_norm_int8(x, w, eps, residual=r), x, r, w, eps, 60)


def test_values_that_are_not_finite_give_scales_that_are_not():
    x = torch.randn(4, 8)
    x[1, 3], x[2, 2] = float("inf"), float("nan")
    q, s = I.rms_norm_int8(x, torch.ones(8))
    assert s.isfinite().tolist() == [True, False, False, True]


def test_an_eps_below_the_normal_numbers_is_refused():
    x = torch.full((1, 4), 1e-22)
    with pytest.raises(ValueError):
        I.rms_norm_int8(x, torch.ones(4), 1e-43)
    I.rms_norm_int8(x, torch.ones(4), 0.0)
