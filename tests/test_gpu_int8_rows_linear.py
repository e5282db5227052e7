"""int8 rows and their product on the GPU against the same in 64 bits."""
import pytest
import torch

from axonml_b200.ops import int8 as I

pytestmark = pytest.mark.gpu
U = 2.0 ** -24                                       # half a step of fp32, relative


def _check_rows(q, s, t, norm, off, scale_off):
    """``t`` [rows, D] in 64 bits.  ``off``: how far a kernel's t / max|t| may be from the real one, relative."""
    a = t.abs().amax(-1, keepdim=True)
    quot = torch.where(a > 0, 127 * t / torch.where(a > 0, a, torch.ones_like(a)), torch.zeros_like(t))
    assert ((q.double() - quot).abs() <= 0.5 + 127 * off).all()
    want = (a * norm)[:, 0] / 127
    assert ((s.double() - want).abs() <= scale_off * want).all()


@pytest.mark.parametrize("rows,D", [(1, 8), (1, 1), (3, 7), (5, 16), (1, 4096), (700, 4096), (64, 14336), (9, 16384), (3, 5125),
                                    (400, 2056), (2, 32768), (2, 40001), (3, 70000), (1000, 100)])
@pytest.mark.parametrize("dt,wdt", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("res", [False, True])
def test_rms_norm_rows(rows, D, dt, wdt, res, kernel_status):
    x = torch.randn(rows, D, device="cuda").to(dt)
    r = torch.randn(rows, D, device="cuda").to(dt) if res else None
    w = (1 + 0.2 * torch.randn(D, device="cuda")).to(wdt)
    got = I.rms_norm_int8(x, w, 1e-5, residual=r)
    h = x if r is None else x + r
    if res:
        assert torch.equal(got[2], h)
    hd = h.double()
    # t = h w is exact for two bf16 factors; else one rounding of t, one of max|t|, one of 127 t; one of the quotient
    off = U if dt == wdt == torch.bfloat16 else 4 * U
    # sum of squares: at most 70 sequential additions and squares in a thread, 10 in the tree, halved by the root; 5 more roundings
    _check_rows(got[0], got[1], hd * w.double(), torch.rsqrt(hd.pow(2).mean(-1, keepdim=True) + 1e-5), off, (81 / 2 + 6) * U)


@pytest.mark.parametrize("rows,F", [(1, 16), (2, 5), (64, 14336), (300, 11008), (3, 1021), (1, 40000), (900, 256), (300, 4096), (297, 16384)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_swiglu_and_plain_rows(rows, F, dt, kernel_status):
    gu = torch.randn(rows, 2 * F, device="cuda").to(dt)
    g, u = gu.double().split(F, -1)
    y = g * torch.sigmoid(g) * u
    # exp: two steps and the rounding of an argument of at most 6.5 log2(e); reciprocal: two steps; two products; for t and its maximum
    off = 2 * (2 * 2 + 6.5 * 1.45 * 2 + 2 * 2 + 4) * U + 3 * U
    q, s = I.swiglu_int8(gu)
    _check_rows(q, s, y, 1.0, off, off)
    q, s = I.quantize_int8(gu)
    _check_rows(q, s, gu.double(), 1.0, 2 * U, 2 * U)


def test_rows_of_strided_inputs_and_special_values(kernel_status):
    base = torch.randn(6, 3, 200, device="cuda").bfloat16()
    x = base[::2, :, 8:136]                                       # gaps between rows, a start off the 16-byte grid
    q, s = I.quantize_int8(x)
    q2, s2 = I.quantize_int8(x.contiguous())
    assert q.shape == (3, 3, 128) and torch.equal(q, q2) and torch.equal(s, s2)
    q3, _ = I.quantize_int8(base[..., 1:])                        # 2-byte aligned rows
    assert torch.equal(q3, I.quantize_int8(base[..., 1:].contiguous())[0])
    t = torch.randn(4, 64, device="cuda")
    t[0] = 0.0
    t[1, 5] = float("inf")
    t[2, 7] = float("nan")
    t[3, :3] = torch.tensor([254.0, 127.0, -3.0], device="cuda")
    q, s = I.quantize_int8(t)
    assert q[0].eq(0).all() and s[0] == 0 and torch.isinf(s[1]) and torch.isnan(s[2])
    assert q[3, :3].tolist() == [127, 64, -2] and s[3] == 2.0     # halves to the even step


def test_rows_do_not_write_outside_their_outputs(kernel_status):
    from axonml_b200 import _native as N
    for D in (24, 31, 16384 + 5):
        rows = 5
        x = torch.randn(rows, D, device="cuda").bfloat16()
        pad = (D + 15) // 16 * 16 + 16
        buf = torch.full((rows + 2, pad), 99, dtype=torch.int8, device="cuda")
        sc = torch.full((rows + 2,), -1.0, device="cuda")
        N.launch("ax_int8_rows", x.device.index, 0, 1, 1, x.data_ptr(), D, 0, 0, 0, 0.0, 0, 0, buf[1:].data_ptr(), pad, sc[1:].data_ptr(), rows, D)
        assert buf[0].eq(99).all() and buf[-1].eq(99).all() and buf[1:-1, D:].eq(99).all()
        assert sc[0] == -1 and sc[-1] == -1


def _product(q, s, w, ws, b):
    y = (q.double() @ w.double().t()) * s.double()[:, None] * ws.double()
    return (y, y) if b is None else (y + b.double(), y)


@pytest.mark.parametrize("M,Nn,K", [(1, 1, 1), (1, 128, 128), (1, 6144, 4096), (3, 1000, 77), (16, 257, 1024), (17, 300, 4096), (33, 4096, 2048),
                                    (64, 640, 512), (100, 4096, 4096), (128, 128, 16384), (129, 512, 640), (300, 1000, 1000), (1024, 2048, 4096),
                                    (257, 333, 129), (513, 64, 96), (2, 33000, 64), (700, 8200, 320), (5, 16, 131071)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bias", [False, True])
def test_int8_linear(M, Nn, K, dt, bias, kernel_status):
    q, s = I._aligned_rows(M, K, "cuda"), torch.rand(M, device="cuda") + 0.1
    w, ws = I._aligned_rows(Nn, K, "cuda"), torch.rand(Nn, device="cuda") + 0.1
    q.random_(-127, 128)
    w.random_(-127, 128)
    b = torch.randn(Nn, device="cuda") * 100 if bias else None
    y = I.int8_linear(q, s, w, ws, b, dt)
    want, prod = _product(q, s, w, ws, b)
    # the exact sum rounds to fp32, two scales and the bias round once each, then the type's own rounding
    tol = 3 * U * prod.abs() + U * want.abs() * 2
    if dt == torch.bfloat16:
        tol = tol + torch.finfo(dt).eps / 2 * (want.abs() + tol)
    assert y.dtype == dt and ((y.double() - want).abs() <= tol).all()


def test_int8_linear_largest_sum(kernel_status):
    """-128 times -128 over the largest K: the int32 sum just fits."""
    K = I.MAX_K
    q, w = I._aligned_rows(1, K, "cuda").fill_(-128), I._aligned_rows(130, K, "cuda").fill_(-128)
    y = I.int8_linear(q, torch.ones(1, device="cuda"), w, torch.ones(130, device="cuda"), out_dtype=torch.float32)
    assert (y.double() == float(torch.tensor(16384 * K, dtype=torch.float32))).all()
    q2, w2 = q.expand(200, K), w
    y = I.int8_linear(q2, torch.ones(200, device="cuda"), w2, torch.ones(130, device="cuda"), out_dtype=torch.float32)
    assert (y.double() == float(torch.tensor(16384 * K, dtype=torch.float32))).all()


def test_int8_linear_strides_and_shapes(kernel_status):
    x = torch.randn(2, 5, 96, device="cuda").bfloat16()
    q, s = I.quantize_int8(x)
    w, ws = I.quantize_int8(torch.randn(50, 96, device="cuda"))
    y = I.int8_linear(q, s, w, ws)
    assert y.shape == (2, 5, 50)
    wide = torch.zeros(50, 131, dtype=torch.int8, device="cuda")
    wide[:, 3:99] = w                                             # rows off the 16-byte grid are copied
    assert torch.equal(I.int8_linear(q, s, wide[:, 3:99], ws), y)
    assert torch.equal(I.int8_linear(q.transpose(0, 1), s.transpose(0, 1), w, ws), y.transpose(0, 1))
    assert torch.equal(I.int8_linear(q[0, 0], s[0, 0], w, ws), y[0, 0])
    assert I.int8_linear(q[:0], s[:0], w, ws).shape == (0, 5, 50)


def test_int8_operators_in_a_graph_and_on_another_stream(kernel_status):
    x = torch.randn(4, 256, device="cuda").bfloat16()
    w = torch.ones(256, device="cuda").bfloat16()
    W = I.Int8Weight.from_dense(torch.randn(512, 256, device="cuda"))

    def step():
        q, s, h = I.rms_norm_int8(x, w, residual=x)
        y = I.int8_linear(q, s, W.q, W.scale)
        q, s = I.swiglu_int8(y)
        return y, q, s, h
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    x.copy_(torch.randn(4, 256, device="cuda"))
    g.replay()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        want = step()
    side.synchronize()
    for a, b in zip(out, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("call,err", [
    (lambda: I.quantize_int8(torch.zeros(2, 8, device="cuda", dtype=torch.float16)), TypeError),
    (lambda: I.int8_linear(torch.zeros(2, 8, dtype=torch.int8, device="cuda"), torch.ones(2), torch.zeros(3, 8, dtype=torch.int8, device="cuda"),
                           torch.ones(3, device="cuda")), ValueError),
    (lambda: I.rms_norm_int8(torch.zeros(2, 8, device="cuda"), torch.ones(8)), ValueError),
])
def test_gpu_refusals(call, err):
    with pytest.raises(err):
        call()


def test_int8_linear_of_very_many_rows(kernel_status):
    """More row blocks than a grid's second dimension holds."""
    M, K, Nn = 8_400_000, 4096, 16
    q = torch.randint(-127, 128, (1, K), dtype=torch.int8, device="cuda")
    w = torch.randint(-127, 128, (Nn, K), dtype=torch.int8, device="cuda")
    s, ws = torch.ones(M, device="cuda"), torch.ones(Nn, device="cuda")
    y = I.int8_linear(q.expand(M, K), s, w, ws, out_dtype=torch.float32)
    assert y.eq((q.double() @ w.double().t()).float()).all()


def test_more_rows_than_the_kernels_take_are_refused():
    x = torch.zeros(1, 16, device="cuda").expand(I.MAX_ROWS + 1, 16)
    with pytest.raises(ValueError):
        I.quantize_int8(x)
    q = torch.zeros(1, 16, dtype=torch.int8, device="cuda").expand(I.MAX_ROWS + 1, 16)
    one = torch.ones(1, device="cuda")
    with pytest.raises(ValueError):
        I.int8_linear(q, one.expand(I.MAX_ROWS + 1), q[:1], one)


def test_more_than_2_to_the_31_elements(kernel_status):
    """Rows and products whose offsets pass 32 bits, against the same rows by themselves."""
    M, K, Nn = 530_000, 4096, 4104
    x = torch.empty(M, K, dtype=torch.bfloat16, device="cuda").normal_()
    w = torch.ones(K, device="cuda").bfloat16()
    last = slice(M - 300, M)
    q, s = I.quantize_int8(x)
    q1, s1 = I.quantize_int8(x[last].clone())
    assert torch.equal(q[last], q1) and torch.equal(s[last], s1)
    n = I.rms_norm_int8(x, w, residual=x)
    n1 = I.rms_norm_int8(x[last].clone(), w, residual=x[last].clone())
    assert all(torch.equal(a[last], b) for a, b in zip(n, n1))
    del n, n1
    g, g1 = I.swiglu_int8(x), I.swiglu_int8(x[last].clone())
    assert torch.equal(g[0][last], g1[0])
    del g, g1, x
    W = I.Int8Weight.from_dense(torch.randn(Nn, K, device="cuda"))
    y = I.int8_linear(q, s, W.q, W.scale)
    assert y.numel() > 2 ** 31 and torch.equal(y[last], I.int8_linear(q1, s1, W.q, W.scale))
