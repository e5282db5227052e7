"""int8 rows and their product on the CPU path: the rounding rule, the scales, the refusals."""
import pytest
import torch

from axonml_b200.ops import int8 as I


def test_quantised_rows_round_to_the_nearest_step():
    x = torch.randn(7, 33)
    q, s = I.quantize_int8(x)
    a = x.double().abs().amax(-1, keepdim=True)
    # one rounding of 127 x, one of the quotient: 127 * 2 * 2^-24 of a step beside the half
    assert ((q.double() - 127 * x.double() / a).abs() <= 0.5 + 127 * 2 * 2.0 ** -24).all()
    assert torch.allclose(s.double(), a[:, 0] / 127, rtol=2 ** -23, atol=0)
    assert q.abs().amax(-1).eq(127).all()


def test_ties_go_to_the_even_step_and_zero_rows_stay_zero():
    x = torch.tensor([[254.0, 127.0, 1.0, 3.0, -5.0], [0.0, 0.0, 0.0, 0.0, 0.0]])
    q, s = I.quantize_int8(x)                      # 127 x / 254 = 127, 63.5, 0.5, 1.5, -2.5
    assert q.tolist() == [[127, 64, 0, 2, -2], [0, 0, 0, 0, 0]] and s.tolist() == [2.0, 0.0]


def test_norm_with_a_residual_returns_the_rounded_stream():
    x, r, w = torch.randn(2, 3, 40).bfloat16(), torch.randn(2, 3, 40).bfloat16(), torch.rand(40).bfloat16() + 0.5
    q, s, h = I.rms_norm_int8(x, w, 1e-5, residual=r)
    assert torch.equal(h, x + r) and q.shape == (2, 3, 40) and s.shape == (2, 3)
    hd = h.double()
    y = hd * torch.rsqrt(hd.pow(2).mean(-1, keepdim=True) + 1e-5) * w.double()
    assert ((q.double() * s.double()[..., None] - y).abs() <= s.double()[..., None] * 0.5001).all()
    q2, s2 = I.rms_norm_int8(h, w)
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_swiglu_rows_and_the_int8_weight():
    gu = torch.randn(5, 24)
    q, s = I.swiglu_int8(gu)
    g, u = gu.double().split(12, -1)
    y = g * torch.sigmoid(g) * u
    assert ((q.double() * s.double()[:, None] - y).abs() <= s.double()[:, None] * 0.5001).all()
    W = I.Int8Weight.from_dense(torch.randn(9, 12))
    assert W.shape == [9, 12] and W.size_bytes() == 9 * 16
    y = I.int8_linear(q, s, W.q, W.scale, out_dtype=torch.float32)
    ref = (q.double() * s.double()[:, None]) @ W.dequantize(torch.float64).t()
    assert torch.allclose(y.double(), ref, rtol=1e-6, atol=1e-6)
    assert W.linear(torch.randn(2, 3, 12)).shape == (2, 3, 9)


def test_linear_sums_are_exact_where_fp32_would_not_be():
    K = 100000
    q = torch.full((1, K), 127, dtype=torch.int8)
    w = torch.full((2, K), 127, dtype=torch.int8)
    w[1, 0] = 126
    y = I.int8_linear(q, torch.ones(1), w, torch.ones(2), out_dtype=torch.float32)
    assert y.tolist() == [[float(torch.tensor(127 * 127 * K, dtype=torch.float32)),
                           float(torch.tensor(127 * 127 * K - 127, dtype=torch.float32))]]


@pytest.mark.parametrize("call,err", [
    (lambda q, s, w, ws: I.int8_linear(q.float(), s, w, ws), TypeError),
    (lambda q, s, w, ws: I.int8_linear(q, s, w.float(), ws), TypeError),
    (lambda q, s, w, ws: I.int8_linear(q, s.double(), w, ws), TypeError),
    (lambda q, s, w, ws: I.int8_linear(q, s, w, ws, out_dtype=torch.float16), TypeError),
    (lambda q, s, w, ws: I.int8_linear(q[:, :5], s, w, ws), ValueError),
    (lambda q, s, w, ws: I.int8_linear(q, s[:1], w, ws), ValueError),
    (lambda q, s, w, ws: I.int8_linear(q, s, w, ws[:2]), ValueError),
    (lambda q, s, w, ws: I.int8_linear(q, s, w, ws, bias=torch.zeros(2)), ValueError),
    (lambda q, s, w, ws: I.int8_linear(torch.zeros(1, I.MAX_K + 1, dtype=torch.int8), torch.ones(1),
                                       torch.zeros(1, I.MAX_K + 1, dtype=torch.int8), torch.ones(1)), ValueError),
    (lambda q, s, w, ws: I.rms_norm_int8(torch.randn(2, 8), torch.ones(7)), ValueError),
    (lambda q, s, w, ws: I.rms_norm_int8(torch.randn(2, 8), torch.ones(8), residual=torch.randn(2, 8).bfloat16()), ValueError),
    (lambda q, s, w, ws: I.rms_norm_int8(torch.randn(2, 8), torch.ones(8, requires_grad=True)), RuntimeError),
    (lambda q, s, w, ws: I.swiglu_int8(torch.randn(2, 7)), ValueError),
    (lambda q, s, w, ws: I.quantize_int8(torch.randn(8)), ValueError),
    (lambda q, s, w, ws: I.quantize_int8(torch.zeros(2, 8, dtype=torch.int32)), TypeError),
])
def test_refusals(call, err):
    q, s = I.quantize_int8(torch.randn(2, 8))
    w, ws = I.quantize_int8(torch.randn(3, 8))
    with pytest.raises(err):
        call(q, s, w, ws)


def test_empty_batches():
    q, s = I.quantize_int8(torch.randn(0, 8))
    w, ws = I.quantize_int8(torch.randn(3, 8))
    assert q.shape == (0, 8) and s.shape == (0,)
    assert I.int8_linear(q, s, w, ws).shape == (0, 3)
