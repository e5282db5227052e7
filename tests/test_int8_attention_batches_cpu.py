"""How a batch is split over launches of the int8 decode attention."""
import pytest

from axonml_b200.ops import paged


@pytest.mark.parametrize("B", [1, 7, 1024, 1025, 2500, 8000])
@pytest.mark.parametrize("G,Hkv,width,P", [(4, 8, 64, 16), (1, 1, 0, 16), (37, 8, 2048, 48), (4, 16, 131072, 16), (16, 32, 2048, 1024), (4, 8, 1 << 21, 64)])
def test_launches_stay_within_what_the_kernel_numbers(B, G, Hkv, width, P):
    each = paged._int8_sequences(B, G, Hkv, width, P)
    blocks = 1 if G <= 8 else -(-G // 16)
    assert 1 <= each <= min(B, 1024) and each * Hkv * blocks * (width * P // 16) <= 0x7f000000
    launches = -(-B // each)
    assert launches * each - B < launches                # even shares
    if B <= 1024 and B * Hkv * blocks * (width * P // 16) <= 0x7f000000:
        assert each == B


def test_an_empty_batch_and_a_table_that_no_launch_takes():
    assert paged._int8_sequences(0, 4, 8, 64, 16) == 1
    with pytest.raises(ValueError, match="pages"):
        paged._int8_sequences(1, 4, 128, 1 << 24, 16)
