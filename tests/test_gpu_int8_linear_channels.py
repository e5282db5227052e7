"""int8 product with half a billion channels: every channel is written, with its own value."""
import pytest
import torch

from axonml_b200.ops import int8 as I

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,Nn", [(1, 2 ** 29), (2, 2 ** 29 + 136)])
def test_half_a_billion_channels(M, Nn, kernel_status):
    K = 16
    w = torch.empty(Nn, K, dtype=torch.int8, device="cuda").random_(-127, 128)
    q = torch.randint(-127, 128, (M, K), dtype=torch.int8, device="cuda")
    ws = torch.ones(Nn, device="cuda")
    s = torch.full((M,), 0.5, device="cuda")
    y = I.int8_linear(q, s, w, ws)
    assert y.shape == (M, Nn)
    for a in range(0, Nn, 1 << 26):                       # sums of at most 16 * 127^2, halved: exact in fp32, one rounding to bf16
        want = (w[a:a + (1 << 26)].float() @ q.float().t()).mul_(0.5).bfloat16()
        assert torch.equal(y[:, a:a + (1 << 26)], want.t())
