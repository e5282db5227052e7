"""int8 activations and weights: rows with one scale each, and the product of such rows with an
int8 matrix (``csrc/kernels/int8_rows.cu``, ``int8_gemm.cu``).

A value is ``q * scale`` with ``q`` in [-127, 127] and one fp32 scale per row (a token of the
activations, an output channel of a weight).  The producers round as the real numbers would:
``q = rint(127 y / max|y|)``, ties to even (of SwiGLU's ``y`` as fp32 holds it: its exponential is approximate, so a step
next to a border may be its neighbour); a row below ``TINY`` everywhere counts as zero, one with
a value that is not finite gets a scale that is not.  For inference; nothing here has a gradient.  CPU tensors
take the same maths in torch."""
from __future__ import annotations

import dataclasses

import torch

from .. import _native as N

MAX_K = 131071          # 2^14 K < 2^31: the int32 sum cannot overflow
MAX_ROWS = 1 << 30      # rows, columns and channels are 32-bit numbers on a GPU


def _aligned_rows(rows: int, cols: int, device) -> torch.Tensor:
    """int8 ``[rows, cols]`` whose rows start on 16-byte boundaries (the product's loads need that)."""
    return torch.empty_strided((rows, cols), (cols + -cols % 16, 1), dtype=torch.int8, device=device)


def _rows2d(t: torch.Tensor) -> torch.Tensor:
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _no_gradient() -> None:
    if torch.is_grad_enabled():
        raise RuntimeError("the int8 operators have no gradient: call them under torch.no_grad()")


TINY = 2.0 ** -118      # a group whose largest magnitude is below this counts as zero (its scale would not be a normal number)


def _steps(t: torch.Tensor, amax: torch.Tensor) -> torch.Tensor:
    one = torch.where(amax > 0, amax, torch.ones_like(amax))
    q = (t.double() * 127.0 / one.double()).round()
    return torch.where(amax > 0, q, torch.zeros_like(q)).nan_to_num_(0.0).to(torch.int8)


def _ref_rows(t: torch.Tensor, norm=None):
    amax = t.abs().amax(-1, keepdim=True) if t.shape[-1] else t.new_zeros(t.shape[:-1] + (1,))
    amax = torch.where(amax < TINY, torch.zeros_like(amax), amax)
    scale = (amax if norm is None else amax * norm) / 127.0
    return _steps(t, amax), scale.squeeze(-1).float()


def _ref_norm_rows(h: torch.Tensor, w: torch.Tensor, eps: float):
    mean = h.square().mean(-1, keepdim=True) + eps
    top = h.abs().amax(-1, keepdim=True)
    # sums outside fp32's range: values scaled by a power of two, which cancels
    out = ~((mean >= 2.0 ** -100) & mean.isfinite() & (h * w).isfinite().all(-1, keepdim=True)) & top.isfinite()
    f = torch.where(out, torch.ldexp(torch.ones_like(top), (1 - top.frexp().exponent).clamp(-126, 100)), torch.ones_like(top))
    h = h * f
    return _ref_rows(h * w, torch.rsqrt(h.square().mean(-1, keepdim=True) + eps * f * f))


_I8, _F32 = torch.int8, torch.float32
_KINDS = {torch.bfloat16: 1, torch.float32: 0}


def _kind(dtype: torch.dtype, what: str) -> int:
    k = _KINDS.get(dtype)
    if k is None:
        raise TypeError(f"{what} must be bf16 or fp32 on a GPU, not {dtype}")
    return k


def _launch_rows(mode: int, x: torch.Tensor, D: int, res=None, weight=None, eps: float = 0.0):
    flat = x.dim() == 2
    strides = x.stride() if flat else (0, 0)
    if strides[1] == 1:
        x2 = x
    else:
        x2 = _rows2d(x)
        strides = x2.stride()
    rows, dtype, index = x2.shape[0], x.dtype, x.get_device()
    if rows > MAX_ROWS or D > MAX_ROWS:
        raise ValueError(f"{rows} rows of {D} are more than the kernel takes ({MAX_ROWS})")
    wk = kind = _kind(dtype, "x")
    if D % 16 == 0 and mode != 2 and strides[0] == D:
        q = torch.empty_like(x2, dtype=_I8)
    else:
        q = _aligned_rows(rows, D, x.device)
    scale = x2.new_empty(rows, dtype=_F32)
    h, rp, rs, hp, wp = None, 0, 0, 0, 0
    if weight is not None:
        wt = weight.dtype
        if wt is not _F32 and wt is not dtype:
            weight, wt = weight.float(), _F32
        if not weight.is_contiguous():
            weight = weight.contiguous()
        wp, wk = weight.data_ptr(), _KINDS[wt]
    if res is not None:
        r2 = res if flat and res.stride(1) == 1 else _rows2d(res)
        h = torch.empty_like(x2) if strides[0] == D else torch.empty((rows, D), dtype=dtype, device=x.device)
        rp, rs, hp = r2.data_ptr(), r2.stride(0), h.data_ptr()
    if rows:
        N.launch("ax_int8_rows", index, mode, kind, wk, x2.data_ptr(), strides[0], rp, rs, wp, eps, hp, D, q.data_ptr(), q.stride(0),
                 scale.data_ptr(), rows, D)
    if not flat:
        lead = x.shape[:-1]
        q, scale = q.unflatten(0, lead), scale.view(lead)
        h = h.view(x.shape) if h is not None else None
    return q, scale, h


def _check_rows(x: torch.Tensor) -> None:
    if x.dim() < 2 or x.shape[-1] == 0:
        raise ValueError(f"rows [..., D] with D > 0 are needed, not {tuple(x.shape)}")
    if not x.is_floating_point():
        raise TypeError(f"x must be a floating tensor, not {x.dtype}")
    if x.requires_grad:
        _no_gradient()


def quantize_int8(x: torch.Tensor):
    """``x[..., K]`` to int8 rows: ``(q [..., K], scale [...])``.  For a weight ``[N, K]`` these are its
    channels.  Rows of ``q`` start on 16-byte boundaries."""
    _check_rows(x)
    if not x.is_cuda:
        return _ref_rows(x.float())
    return _launch_rows(0, x, x.shape[-1])[:2]


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: torch.Tensor | None = None):
    """RMSNorm over the last dim, to int8 rows: ``(q, scale)``.  With ``residual`` the norm is of
    ``h = x + residual`` (rounded to ``x``'s type) and the result is ``(q, scale, h)``.  Rows whose squares leave
    fp32's range (values above about 1e19; tiny ones with an ``eps`` of nothing) are scaled by a power of two first."""
    _check_rows(x)
    D, dev = x.shape[-1], x.get_device()                   # (-1: not on a GPU)
    if weight.dim() != 1 or weight.shape[0] != D:
        raise ValueError(f"weight {tuple(weight.shape)} does not fit rows of {D}")
    if weight.get_device() != dev:
        raise ValueError(f"weight is on {weight.device}, x on {x.device}")
    if 0 < abs(eps) < 2.0 ** -126:
        raise ValueError(f"eps must be 0 or a normal fp32 number, not {eps}")
    if weight.requires_grad:
        _no_gradient()
    if residual is not None:
        if residual.shape != x.shape or residual.dtype is not x.dtype or residual.get_device() != dev:
            raise ValueError("residual must have x's shape, type and device")
        if residual.requires_grad:
            _no_gradient()
    if x.is_cuda:
        q, scale, h = _launch_rows(1, x, D, residual, weight, eps)
    else:
        h = x if residual is None else x + residual
        q, scale = _ref_norm_rows(h.float(), weight.float(), eps)
    return (q, scale, h) if residual is not None else (q, scale)


def swiglu_int8(gate_up: torch.Tensor):
    """``silu(gate) * up`` of a fused ``[..., 2F]`` tensor laid out gate|up, to int8 rows ``(q, scale)``."""
    _check_rows(gate_up)
    F, odd = divmod(gate_up.shape[-1], 2)
    if odd:
        raise ValueError("gate|up needs an even last dim")
    if gate_up.is_cuda:
        return _launch_rows(2, gate_up, F)[:2]
    g, u = gate_up.float().split(F, dim=-1)
    return _ref_rows(torch.nn.functional.silu(g) * u)


def int8_linear(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``y = (q * scale) (weight * weight_scale)^T + bias``: ``q`` int8 ``[..., K]`` with ``scale`` ``[...]``,
    ``weight`` int8 ``[N, K]`` with ``weight_scale`` ``[N]``.  The integer sum is exact, the scales
    and the bias are applied in fp32, and the result is rounded to ``out_dtype`` (bf16 or fp32).  K is at most 131071.  Operands whose rows do not start
    on 16-byte boundaries are copied first; ``quantize_int8`` and the fused producers lay them out so."""
    if q.dtype is not _I8 or weight.dtype is not _I8:
        raise TypeError("q and weight must be int8")
    flat = q.dim() == 2
    if weight.dim() != 2 or q.dim() < 1 or q.shape[-1] != weight.shape[1]:
        raise ValueError(f"q {tuple(q.shape)} does not fit a weight {tuple(weight.shape)}")
    Nn, K = weight.shape
    if not 0 < K <= MAX_K:
        raise ValueError(f"K must be in 1..{MAX_K}, not {K}")
    q2 = q if flat else q.reshape(-1, K)
    M = q2.shape[0]
    fits = scale.dim() == 1 and scale.shape[0] == M if flat else scale.shape == q.shape[:-1]
    if not fits or weight_scale.dim() != 1 or weight_scale.shape[0] != Nn:
        raise ValueError(f"scales {tuple(scale.shape)}, {tuple(weight_scale.shape)} do not fit {tuple(q.shape)}, {tuple(weight.shape)}")
    if scale.dtype is not _F32 or weight_scale.dtype is not _F32:
        raise TypeError("scales must be fp32")
    kind = _KINDS.get(out_dtype)
    if kind is None:
        raise TypeError(f"out_dtype must be bf16 or fp32, not {out_dtype}")
    index = q.get_device()                                 # (-1: not on a GPU)
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != Nn or bias.get_device() != index:
            raise ValueError(f"bias {tuple(bias.shape)} on {bias.device} does not fit {Nn} channels on {q.device}")
        if bias.requires_grad:
            _no_gradient()
    if scale.get_device() != index or weight.get_device() != index or weight_scale.get_device() != index:
        raise ValueError(f"q is on {q.device}, its scale on {scale.device}, the weight on {weight.device}, its scale on {weight_scale.device}")
    if scale.requires_grad or weight_scale.requires_grad:
        _no_gradient()
    if index < 0:
        y = (q2.double() @ weight.double().t()).float() * scale.reshape(-1, 1) * weight_scale
        y = y if bias is None else y + bias.float()
        return y.to(out_dtype).view(*q.shape[:-1], Nn)
    if M > MAX_ROWS or Nn > MAX_ROWS:
        raise ValueError(f"{M} rows and {Nn} channels are more than the kernel takes ({MAX_ROWS})")
    out = torch.empty_strided((M, Nn), (Nn, 1), dtype=out_dtype, device=q.device)
    if M and Nn:
        qs, q1 = q2.stride()
        ws, w1 = weight.stride()
        qp, wp = q2.data_ptr(), weight.data_ptr()
        if q1 != 1 or qs % 16 or qp % 16:
            q2 = _aligned_rows(M, K, q.device).copy_(q2)
            qs, qp = q2.stride(0), q2.data_ptr()
        if w1 != 1 or ws % 16 or wp % 16:
            weight = _aligned_rows(Nn, K, q.device).copy_(weight)
            ws, wp = weight.stride(0), weight.data_ptr()
        if not scale.is_contiguous():
            scale = scale.contiguous()
        if not weight_scale.is_contiguous():
            weight_scale = weight_scale.contiguous()
        b = 0
        if bias is not None:
            bias = bias.float().contiguous()
            b = bias.data_ptr()
        N.launch("ax_int8_gemm", index, qp, qs, scale.data_ptr(), wp, ws, weight_scale.data_ptr(), b, out.data_ptr(), Nn, kind, M, Nn, K,
                 N.status_ptr(index))
    return out if flat else out.view(*q.shape[:-1], Nn)


@dataclasses.dataclass
class Int8Weight:
    """A linear layer's weight in int8 with one scale per output channel."""
    q: torch.Tensor
    scale: torch.Tensor

    @classmethod
    def from_dense(cls, w: torch.Tensor) -> "Int8Weight":
        with torch.no_grad():
            return cls(*quantize_int8(w))

    @property
    def shape(self): return list(self.q.shape)

    def size_bytes(self) -> int: return self.q.shape[0] * (self.q.shape[1] + 4)

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        return (self.q.float() * self.scale[:, None]).to(dtype)

    def linear(self, x: torch.Tensor, bias=None, out_dtype=torch.bfloat16) -> torch.Tensor:
        """``x[..., K]`` in bf16 or fp32, its rows quantised on the way."""
        q, s = quantize_int8(x)
        return int8_linear(q, s, self.q, self.scale, bias, out_dtype)
