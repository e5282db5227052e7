"""RMS norm to int8 rows at the ends of fp32's range, checked against 64 bits."""
import torch

# magnitudes of a row's values, its weights' and eps: squares that overflow, t = h w that does, squares that vanish without an eps
CASES = [(1e20, 1.0, 1e-5), (2e38, 1.0, 1e-5), (1e30, 1e-20, 1e-5), (1e25, 1e20, 1e-5), (1e-24, 1.0, 0.0), (3e-33, 1.0, 0.0), (1e-17, 1.0, 1e-36),
         (1.0, 1.0, 0.0), (1e17, 1.0, 1e-5), (1.0, 1.0, 1e-5)]


def inputs(size, wsize, D, dt, res, g=None):
    """Three rows of the size under test among ordinary ones."""
    x = torch.rand(5, D, generator=g) * 2 - 1
    x[1:4] *= size
    x[0, 0] = x[4, -1] = 0.5
    x[1:4, 0] = size                                      # (no row is close to nothing)
    x = x.to(dt)
    r = (torch.rand(5, D, generator=g) - 0.5).to(dt) * (x.abs() / 4) if res else None
    return x, r, (wsize * (0.75 + 0.5 * torch.rand(D, generator=g))).to(dt)


def check(got, x, r, w, eps, D):
    h = x if r is None else x + r
    if r is not None:
        assert torch.equal(got[2], h)
    d, u = h.double(), 2.0 ** -24
    t = d * w.double()
    a = t.abs().amax(-1, keepdim=True)
    norm = torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + eps)
    # roundings of t, of max|t|, of 127 t and of the quotient
    assert ((got[0].double() - 127 * t / a).abs() <= 0.5 + 127 * 4 * u).all()
    # sum of squares: at most 70 sequential additions in a thread and 10 in the tree, halved by the root; eight roundings more
    want = (a * norm)[:, 0] / 127
    assert ((got[1].double() - want).abs() <= (81 / 2 + 8) * u * want).all()
