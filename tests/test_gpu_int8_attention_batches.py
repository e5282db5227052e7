"""int8 decode attention over tables with more room than one launch can number."""
import pytest
import torch

import _int8 as R
from axonml_b200.ops import paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hkv,width", [(1030, 16, 2048), (5, 8, 1 << 20)])
def test_tables_with_more_tiles_than_a_launch_numbers(B, Hkv, width, kernel_status):
    """Wide tables (pages that several sequences share): the same as with narrow ones."""
    G, P, D, pages = 2, 1024, 64, 5
    c = R.make_cache(pages, Hkv, P, D, "cuda", seed=8)
    g = torch.Generator().manual_seed(B)
    narrow = torch.randint(0, pages, (B, 2), generator=g).int().cuda()
    ctx = torch.randint(0, 2 * P + 1, (B,), generator=g).int().cuda()
    q = torch.randn(B, Hkv * G, D, device="cuda").bfloat16()
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = narrow
    assert B * Hkv * width * (P // 16) > 2 ** 31 - 1
    got = paged.decode_attention_int8(q, *c, table, ctx)
    assert got[ctx == 0].eq(0).all()
    for b in {0, B // 2, B - 1}:
        want, off = R.attention(q[b:b + 1], c[0], R.v_rows(c[1]), c[2], c[3], narrow[b:b + 1].tolist(), [int(ctx[b])], R.default_scale(D))
        assert ((got[b:b + 1].double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all()


def test_a_table_that_no_launch_takes_is_refused():
    c = R.make_cache(1, 64, 1024, 64, "cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda").expand(1, 1 << 20)
    with pytest.raises(ValueError, match="pages"):
        paged.decode_attention_int8(torch.zeros(1, 64, 64, device="cuda").bfloat16(), *c, table, torch.ones(1, dtype=torch.int32, device="cuda"))
