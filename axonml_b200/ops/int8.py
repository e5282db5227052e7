"""int8 activations and weights: rows with one scale each, and the product of such rows with an
int8 matrix (``csrc/kernels/int8_rows.cu``, ``int8_gemm.cu``).

A value is ``q * scale`` with ``q`` in [-127, 127] and one fp32 scale per row (a token of the
activations, an output channel of a weight).  The producers round as the real numbers would:
``q = rint(127 y / max|y|)``, ties to even.  For inference; nothing here has a gradient.  CPU tensors
take the same maths in torch."""
from __future__ import annotations

import dataclasses

import torch

from .. import _native as N

MAX_K = 131071          # 2^14 K < 2^31: the int32 sum cannot overflow


def _aligned_rows(rows: int, cols: int, device) -> torch.Tensor:
    """int8 ``[rows, cols]`` whose rows start on 16-byte boundaries (the product's loads need that)."""
    pad = -cols % 16
    t = torch.empty((rows, cols + pad), dtype=torch.int8, device=device)
    return t[:, :cols] if pad else t


def _rows2d(t: torch.Tensor) -> torch.Tensor:
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _no_grad(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the int8 operators have no gradient: call them under torch.no_grad()")


def _same_device(x: torch.Tensor, **others) -> None:
    for name, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, the input on {x.device}")


def _steps(t: torch.Tensor, amax: torch.Tensor) -> torch.Tensor:
    one = torch.where(amax > 0, amax, torch.ones_like(amax))
    return torch.where(amax > 0, (t * 127.0 / one).round(), torch.zeros_like(t)).nan_to_num_(0.0).to(torch.int8)


def _ref_rows(t: torch.Tensor, norm=None):
    amax = t.abs().amax(-1, keepdim=True) if t.shape[-1] else t.new_zeros(t.shape[:-1] + (1,))
    scale = (amax if norm is None else amax * norm) / 127.0
    return _steps(t, amax), scale.squeeze(-1).float()


def _kind(t: torch.Tensor, what: str) -> int:
    if t.dtype == torch.bfloat16:
        return 1
    if t.dtype == torch.float32:
        return 0
    raise TypeError(f"{what} must be bf16 or fp32 on a GPU, not {t.dtype}")


def _launch_rows(mode: int, x: torch.Tensor, D: int, res=None, weight=None, eps: float = 0.0):
    x2 = _rows2d(x)
    rows, shape, dev = x2.shape[0], x.shape[:-1], x.device
    kind = _kind(x, "x")
    q = _aligned_rows(rows, D, dev)
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    h, rp, rs, hp, wp, wk = None, 0, 0, 0, 0, kind
    if weight is not None:
        if weight.dtype != torch.float32 and weight.dtype != x.dtype:
            weight = weight.float()
        weight = weight.contiguous()
        wp, wk = weight.data_ptr(), _kind(weight, "weight")
    if res is not None:
        r2 = _rows2d(res)
        h = torch.empty((rows, D), dtype=x.dtype, device=dev)
        rp, rs, hp = r2.data_ptr(), r2.stride(0), h.data_ptr()
    if rows:
        N.launch("ax_int8_rows", dev, mode, kind, wk, x2.data_ptr(), x2.stride(0), rp, rs, wp, eps, hp, D, q.data_ptr(), q.stride(0),
                 scale.data_ptr(), rows, D)
    if x.dim() != 2:
        q, scale = q.unflatten(0, shape), scale.view(shape)
        h = h.view(x.shape) if h is not None else None
    return q, scale, h


def _check_rows(x: torch.Tensor) -> None:
    if x.dim() < 2 or x.shape[-1] == 0:
        raise ValueError(f"rows [..., D] with D > 0 are needed, not {tuple(x.shape)}")
    if not x.is_floating_point():
        raise TypeError(f"x must be a floating tensor, not {x.dtype}")


def quantize_int8(x: torch.Tensor):
    """``x[..., K]`` to int8 rows: ``(q [..., K], scale [...])``.  For a weight ``[N, K]`` these are its
    channels.  Rows of ``q`` start on 16-byte boundaries."""
    _check_rows(x)
    _no_grad(x)
    if not x.is_cuda:
        return _ref_rows(x.float())
    return _launch_rows(0, x, x.shape[-1])[:2]


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: torch.Tensor | None = None):
    """RMSNorm over the last dim, to int8 rows: ``(q, scale)``.  With ``residual`` the norm is of
    ``h = x + residual`` (rounded to ``x``'s type) and the result is ``(q, scale, h)``."""
    _check_rows(x)
    _no_grad(x, weight, residual)
    _same_device(x, weight=weight, residual=residual)
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"weight {tuple(weight.shape)} does not fit rows of {x.shape[-1]}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have x's shape and type")
    if x.is_cuda:
        q, scale, h = _launch_rows(1, x, x.shape[-1], residual, weight, eps)
    else:
        h = x if residual is None else x + residual
        hf = h.float()
        q, scale = _ref_rows(hf * weight.float(), torch.rsqrt(hf.square().mean(-1, keepdim=True) + eps))
    return (q, scale, h) if residual is not None else (q, scale)


def swiglu_int8(gate_up: torch.Tensor):
    """``silu(gate) * up`` of a fused ``[..., 2F]`` tensor laid out gate|up, to int8 rows ``(q, scale)``."""
    _check_rows(gate_up)
    _no_grad(gate_up)
    if gate_up.shape[-1] % 2:
        raise ValueError("gate|up needs an even last dim")
    F = gate_up.shape[-1] // 2
    if gate_up.is_cuda:
        return _launch_rows(2, gate_up, F)[:2]
    g, u = gate_up.float().split(F, dim=-1)
    return _ref_rows(torch.nn.functional.silu(g) * u)


def _gemm_rows(t: torch.Tensor) -> torch.Tensor:
    if t.stride(1) == 1 and t.stride(0) % 16 == 0 and t.data_ptr() % 16 == 0:
        return t
    return _aligned_rows(t.shape[0], t.shape[1], t.device).copy_(t)


def int8_linear(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``y = (q * scale) (weight * weight_scale)^T + bias``: ``q`` int8 ``[..., K]`` with ``scale`` ``[...]``,
    ``weight`` int8 ``[N, K]`` with ``weight_scale`` ``[N]``.  The integer sum is exact; the result is
    rounded once, to ``out_dtype`` (bf16 or fp32).  K is at most 131071.  Operands whose rows do not start
    on 16-byte boundaries are copied first; ``quantize_int8`` and the fused producers lay them out so."""
    if q.dtype != torch.int8 or weight.dtype != torch.int8:
        raise TypeError("q and weight must be int8")
    if weight.dim() != 2 or q.dim() < 1 or q.shape[-1] != weight.shape[1]:
        raise ValueError(f"q {tuple(q.shape)} does not fit a weight {tuple(weight.shape)}")
    Nn, K = weight.shape
    if not 0 < K <= MAX_K:
        raise ValueError(f"K must be in 1..{MAX_K}, not {K}")
    if scale.shape != q.shape[:-1] or weight_scale.shape != (Nn,):
        raise ValueError(f"scales {tuple(scale.shape)}, {tuple(weight_scale.shape)} do not fit {tuple(q.shape)}, {tuple(weight.shape)}")
    if scale.dtype != torch.float32 or weight_scale.dtype != torch.float32:
        raise TypeError("scales must be fp32")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"out_dtype must be bf16 or fp32, not {out_dtype}")
    if bias is not None and bias.shape != (Nn,):
        raise ValueError(f"bias {tuple(bias.shape)} does not fit {Nn} channels")
    _same_device(q, scale=scale, weight=weight, weight_scale=weight_scale, bias=bias)
    _no_grad(scale, weight_scale, bias)
    lead = q.shape[:-1]
    q2 = q.reshape(-1, K) if q.dim() != 2 else q
    if not q.is_cuda:
        y = (q2.double() @ weight.double().t()).float() * scale.reshape(-1, 1) * weight_scale
        y = y if bias is None else y + bias.float()
        return y.to(out_dtype).view(*lead, Nn)
    M = q2.shape[0]
    out = torch.empty((M, Nn), dtype=out_dtype, device=q.device)
    if M and Nn:
        q2, w2 = _gemm_rows(q2), _gemm_rows(weight)
        s, ws = scale.contiguous(), weight_scale.contiguous()
        b = bias.float().contiguous() if bias is not None else None
        N.launch("ax_int8_gemm", q.device, q2.data_ptr(), q2.stride(0), s.data_ptr(), w2.data_ptr(), w2.stride(0), ws.data_ptr(),
                 b.data_ptr() if b is not None else 0, out.data_ptr(), Nn, int(out_dtype == torch.bfloat16), M, Nn, K,
                 N.status_ptr(q.device))
    return out if q.dim() == 2 else out.view(*lead, Nn)


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
