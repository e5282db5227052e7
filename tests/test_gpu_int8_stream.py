"""The residual stream that the int8 norm writes is x + residual to the last bit, subnormal values too."""
import pytest
import torch

from axonml_b200.ops import int8 as I

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 1000, 5125, 20001])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_stream_of_subnormal_values(D, dt, kernel_status):
    g = torch.Generator().manual_seed(D)
    size = torch.tensor([1.0, 1e-36, 1e-38, 1e-39, 1e-40])[:, None]
    x, r = ((torch.randn(5, D, generator=g) * size).to(dt) for _ in range(2))
    want = x + r
    assert (want.float().abs() < 2.0 ** -126).logical_and(want != 0).any()
    h = I.rms_norm_int8(x.cuda(), torch.ones(D, dtype=dt, device="cuda"), residual=r.cuda())[2]
    bits = torch.int32 if dt == torch.float32 else torch.int16
    assert torch.equal(h.cpu().view(bits), want.view(bits))
