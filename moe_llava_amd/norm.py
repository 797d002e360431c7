"""Residual addition + root-mean-square norm, the step in front of every MLP of the RMS-norm model families
(qwen/modeling_qwen.py RMSNorm, and the LLaMA-form decoders), with 16-bit output, or 8-bit output for ``fp8`` experts.

    s = round(x + residual);  y = s / sqrt(mean(s^2) + eps) * weight

Everything between the two roundings is fp32 (the reference's modules round ``s * rstd`` to 16 bits before the weight;
here only y is rounded).  ``add_rms_norm`` is differentiable in x, residual and weight; both operators take rows of any
stride, bf16 or fp16, with a weight of the rows' type or fp32.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from . import _lib, ops
from .fp8 import Fp8Rows, _empty_rows, _gpu, _half_rows, _lead, _lead_scale, _stream
from .sharded_moe import module_has_hooks

MAX_M = 65536

_FORWARDS = {nn.RMSNorm.forward}     # forwards that are ``rms_norm(x, self.weight, self.eps)``


def _weight_code(w: Tensor, x: Tensor) -> int:
    if w.dtype == torch.float32:
        return ops.WG_F32
    if w.dtype == x.dtype:
        return ops.WG_BF16 if w.dtype == torch.bfloat16 else ops.WG_F16
    raise TypeError(f"weight: expected fp32 or the rows' type ({x.dtype}), got {w.dtype}")


def _check(x: Tensor, residual: Optional[Tensor], weight: Tensor):
    x2 = _half_rows(x, "x")
    _gpu(weight, "weight")
    M, dev = x2.shape[1], x2.device
    if not 1 <= M <= MAX_M:
        raise ValueError(f"x: row length {M} must be between 1 and {MAX_M}")
    if weight.dim() != 1 or weight.shape[0] != M or weight.device != dev:
        raise ValueError(f"weight {tuple(weight.shape)} on {weight.device} does not match x {tuple(x.shape)} on {dev}")
    if not weight.is_contiguous():
        weight = weight.contiguous()
    r2 = None
    if residual is not None:
        if not isinstance(residual, Tensor) or residual.shape != x.shape or residual.dtype != x.dtype or residual.device != dev:
            raise ValueError("residual must match x in shape, type and device")
        r2 = _half_rows(residual, "residual")
    return x2, r2, weight, _weight_code(weight, x2)


def _as(t: Tensor, x: Tensor) -> Tensor:
    return t if x.dim() == 2 else t.reshape(x.shape)


def _launch(x: Tensor, r: Optional[Tensor], w: Tensor, code: int, eps: float, want_y: bool, want_q: bool, want_rstd: bool):
    S, M = x.shape
    dev = x.device
    new = torch.empty_like if x.is_contiguous() else lambda t: torch.empty((S, M), dtype=t.dtype, device=dev)   # 1.2 us, 1.7
    y = new(x) if want_y else None
    s = new(x) if r is not None else None
    rstd = torch.empty((S,), dtype=torch.float32, device=dev) if want_rstd else None
    rows = _empty_rows(S, M, dev) if want_q else None
    if not S:
        return y, s, rstd, rows
    rp = ldr = sp = qp = qs = ldq = None
    if r is not None:
        rp, ldr, sp = r.data_ptr(), _lead(r, M), s.data_ptr()
    if want_q:
        q, sc = rows
        qp, qs, ldq = q.data_ptr(), sc.data_ptr(), _lead_scale(sc)
    with ops._on(dev):
        rc = _lib.load().moe_add_rms_norm_fwd(
            x.data_ptr(), _lead(x, M), rp, ldr or 0, w.data_ptr(), code, eps, S, M, y.data_ptr() if want_y else None, M, sp, M,
            rstd.data_ptr() if want_rstd else None, qp, M, qs, ldq or 0, ops._dt(x), _stream(dev.index))
    if rc:
        _lib.check(rc, "moe_add_rms_norm_fwd")
    return y, s, rstd, rows


class _AddRmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, residual: Optional[Tensor], weight: Tensor, eps: float):
        x2, r2, w, code = _check(x, residual, weight)
        y, s, rstd, _ = _launch(x2, r2, w, code, eps, True, False, True)
        out_s = _as(s, x) if s is not None else None
        ctx.save_for_backward(out_s if out_s is not None else x, weight, rstd)
        ctx.has_res = residual is not None
        ctx.set_materialize_grads(False)
        return (_as(y, x), out_s) if s is not None else _as(y, x)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy: Optional[Tensor], ds: Optional[Tensor] = None):
        s, weight, rstd = ctx.saved_tensors
        if dy is None and ds is None:
            return None, None, None, None
        s2 = _half_rows(s, "sum")
        S, M = s2.shape
        w = weight.contiguous()
        code = _weight_code(w, s2)
        if dy is None and not ctx.needs_input_grad[2]:
            return ds, ds if ctx.has_res else None, None, None
        dx = torch.empty((S, M), dtype=s2.dtype, device=s2.device)
        dw = torch.zeros((M,), dtype=w.dtype, device=w.device) if S == 0 else torch.empty((M,), dtype=w.dtype, device=w.device)
        if S:
            d2 = _half_rows(dy, "dy") if dy is not None else None
            e2 = _half_rows(ds, "dsum") if ds is not None else None
            lib = _lib.load()
            nws = lib.moe_add_rms_norm_bwd_workspace_bytes(S, M)
            ws = torch.empty((nws,), dtype=torch.uint8, device=s2.device)
            with ops._on(s2.device):
                rc = lib.moe_add_rms_norm_bwd(
                    d2.data_ptr() if d2 is not None else None, _lead(d2, M) if d2 is not None else 0,
                    e2.data_ptr() if e2 is not None else None, _lead(e2, M) if e2 is not None else 0, s2.data_ptr(),
                    _lead(s2, M), w.data_ptr(), code, rstd.data_ptr(), S, M, dx.data_ptr(), M, dw.data_ptr(), ws.data_ptr(),
                    nws, ops._dt(s2), _stream(s2.device.index))
            _lib.check(rc, "moe_add_rms_norm_bwd")
        dx = _as(dx, s)
        return dx, dx if ctx.has_res else None, dw, None


def add_rms_norm(x: Tensor, residual: Tensor, weight: Tensor, eps: float = 1e-6) -> Tuple[Tensor, Tensor]:
    """(y, s): the normed rows and the new residual stream, of x's shape and type.  Differentiable."""
    if residual is None:
        raise ValueError("residual is missing: rms_norm has the form without one")
    if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad or weight.requires_grad):
        return _AddRmsNormFn.apply(x, residual, weight, float(eps))
    x2, r2, w, code = _check(x, residual, weight)
    y, s, _, _ = _launch(x2, r2, w, code, float(eps), True, False, False)
    return _as(y, x), _as(s, x)


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6) -> Tensor:
    """The norm alone.  Differentiable."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _AddRmsNormFn.apply(x, None, weight, float(eps))
    x2, _, w, code = _check(x, None, weight)
    return _launch(x2, None, w, code, float(eps), True, False, False)[0].reshape(x.shape)


def add_rms_norm_fp8(x: Tensor, residual: Optional[Tensor], weight: Tensor, eps: float = 1e-6,
                     want_y: bool = True) -> Tuple[Fp8Rows, Optional[Tensor], Tensor]:
    """(rows, y, s): the normed rows in 8 bits ([S, M], quantised from the unrounded fp32 values), the same in 16 bits
    (``want_y``; the router reads them) and the new residual stream.  Row length a multiple of 16.  Inference only."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        raise NotImplementedError("8-bit output has no gradient: use add_rms_norm for training, or torch.no_grad()")
    x2, r2, w, code = _check(x, residual, weight)
    if x2.shape[1] % 16:
        raise ValueError(f"x: row length {x2.shape[1]} must be a multiple of 16 for 8-bit output")
    y, s, _, rows = _launch(x2, r2, w, code, float(eps), want_y, True, False)
    return rows, (_as(y, x) if want_y else None), (_as(s, x) if s is not None else x)


def register_rms_norm(cls):
    """Declare that ``cls.forward(x)`` is ``rms_norm(x, self.weight, self.eps)`` (or ``self.variance_epsilon``), up to the
    roundings in between, so that ``MoE.forward_normed`` may run the kernel in its place.  Returns ``cls``."""
    _FORWARDS.add(cls.forward)
    return cls


def weight_and_eps(module: nn.Module):
    """(weight, eps) of a norm module whose call is known to be ``rms_norm`` of them, else None: a forward that is not declared
    (it may scale by 1 + weight), hooks, no weight, or an eps that the module leaves to torch."""
    if getattr(type(module), "forward", None) not in _FORWARDS:
        return None
    d = module.__dict__                       # plain dict access where it finds something: nn.Module.__getattr__ is slow
    if "forward" in d or module_has_hooks(module):
        return None
    weight = d["_parameters"].get("weight")
    if weight is None:
        weight = getattr(module, "weight", None)
    eps = d.get("eps")
    if eps is None:
        eps = getattr(module, "eps", None)
    if eps is None:
        eps = getattr(module, "variance_epsilon", None)
    if not isinstance(weight, Tensor) or weight.dim() != 1 or eps is None:
        return None
    return weight, eps


@register_rms_norm
class RMSNorm(nn.Module):
    """``weight`` and ``eps`` of a root-mean-square norm (the attribute names of the reference's RMSNorm modules are
    ``weight`` and ``eps`` / ``variance_epsilon``); ``forward(x)`` or ``forward(x, residual)`` -> y or (y, s)."""

    def __init__(self, dim: int, eps: float = 1e-6, dtype=None, device=None):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim, dtype=dtype, device=device))
        self.eps = eps

    def forward(self, x: Tensor, residual: Optional[Tensor] = None):
        return rms_norm(x, self.weight, self.eps) if residual is None else add_rms_norm(x, residual, self.weight, self.eps)
