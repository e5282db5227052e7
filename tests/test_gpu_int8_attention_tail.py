"""int8 decode attention with one strong token in front of a long flat tail, against 64 bits."""
import pytest
import torch

import _int8 as R
from axonml_b200.ops import paged

pytestmark = pytest.mark.gpu

# Weights are rounded to fp16: 2^-11 of a weight down to 2^-21 of the largest, 2^-32 of the largest below; a page's V magnitude relative to
# the largest one met (1/4 here) scales a weight before that.  The rest, relative: the strong token's exponent of at most 28 after four
# roundings 28 * 4 * 2^-24 * ln 2 = 4.6e-6; products summed in fp32, at most 27 tiles of a worker, 2^-22 each: 6.4e-6; a lane's share of
# the weights' sum, 27 additions of 2^-24: 1.6e-6; exp2 and the merge 1e-6: together below 2^-16.
STEP, FLOOR, REST = 2.0 ** -11, 4 * 2.0 ** -32, 2.0 ** -16


def _case(B, Hkv, G, D, n, down, ratio):
    """Token 0 of every sequence has a score `down` above all others (log2 of the weights) and, with `ratio` 1, no value."""
    P, per = 16, (n + 15) // 16
    pages = B * per
    kc, vc, ka, va = R.make_cache(pages, Hkv, P, D, "cuda", seed=n)
    vc.copy_((vc.int().abs() // 2 + 60).to(torch.int8))           # values of one sign
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).int().view(B, per).cuda()
    first = table[:, 0].long()
    kc.zero_()
    kc[first, :, 0, 0] = 127                                      # the strong token: q and k agree in one dim
    ka.fill_(1.0)
    va.fill_(1.0 if ratio == 1 else 0.25)
    va[first] = 1.0
    if ratio == 1:
        vc[first, :, 0, :, 0] = 0
    q = torch.zeros(B, Hkv * G, D, device="cuda").bfloat16()
    q[:, :, 0] = 1.0
    return q, kc, vc, ka, va, table, down / 1.4426950408889634     # score of token 0 is q k scale = scale


@pytest.mark.parametrize("down", [14, 20, 24, 26, 28])
@pytest.mark.parametrize("ratio", [1, 4])
@pytest.mark.parametrize("B,Hkv,G,D,n,spare", [(1, 1, 4, 128, 2047, 0), (1, 1, 4, 64, 60000, 0), (1, 2, 12, 128, 5000, 9000), (700, 1, 1, 64, 640, 0),
                                               (40, 8, 4, 128, 3001, 0), (6, 2, 2, 256, 1000, 3000)])
def test_a_long_tail_is_summed(B, Hkv, G, D, n, spare, ratio, down, kernel_status):
    q, kc, vc, ka, va, table, scale = _case(B, Hkv, G, D, n, down, ratio)
    wide = torch.cat([table, torch.zeros(B, spare, dtype=torch.int32, device="cuda")], 1)
    got = paged.decode_attention_int8(q, kc, vc, ka, va, wide, torch.full((B,), n, dtype=torch.int32, device="cuda"), scale).double()
    for b in {0, B // 2, B - 1}:
        pg = table[b].long()
        v = (R.v_rows(vc[pg]).double() * (va[pg].double() / 127)[..., None, None]).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
        w = torch.full((n,), 1.0, dtype=torch.float64, device="cuda")
        w[0] = 2.0 ** down
        w = w / w.sum()
        want = torch.einsum("n,hnd->hd", w, v).repeat_interleave(G, 0)
        off = ((STEP + REST) * w[:, None] + FLOOR * w[0]).mul(v.abs()).sum(1).repeat_interleave(G, 0)
        assert ((got[b] - want).abs() <= off + 2.0 ** -8 * (want + off)).all()
