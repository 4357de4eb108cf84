"""RMS norm with its backward pass, on the device.

The norms of a decoder layer (``x / sqrt(mean(x^2) + eps) * weight`` over the
last dimension), with the residual addition in front of them fused:
:func:`rms_norm` is differentiable; :func:`rms_norm_forward` and
:func:`rms_norm_backward` are its two passes for a caller that sequences them
itself, as :class:`usaf_b200.engine.MoEBlock` does.  Sums and products run in
fp32 and every output is rounded once; the weight's gradient is summed in a
fixed order, so results repeat bit for bit.

Rows may be strided views as long as the last dimension is contiguous and the
leading ones fold into one stride (others are copied).  Types: fp32, bf16 or
fp16 rows; the weight has the rows' type or fp32.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call_on, differentiated, ptr

MAX_WIDTH = 32768


def _rows(t: torch.Tensor, H: int) -> Tuple[torch.Tensor, int]:
    """``t`` (or a copy) as rows of its last dimension, and their stride."""
    if t.is_contiguous():
        return t, H
    if t.stride(-1) == 1:
        try:
            v = t.view(-1, H)
            return v, v.stride(0)
        except RuntimeError:      # the leading dimensions do not fold into one stride
            pass
    return t.contiguous(), H


def _check(x: torch.Tensor, weight: torch.Tensor) -> Tuple[int, int, int, int]:
    """Width of the rows, their device and the types' codes."""
    shape = x.shape
    H = shape[-1] if shape else 0
    if H < 1 or weight.dim() != 1 or weight.numel() != H:
        raise ValueError(f"weight: expected shape ({H or '?'},), got {tuple(weight.shape)}")
    if H > MAX_WIDTH:
        raise ValueError(f"rows of {H} values; at most {MAX_WIDTH} are handled")
    dt, wdt, dev = x.dtype, weight.dtype, x.get_device()
    if wdt is not dt and wdt is not torch.float32:
        raise TypeError(f"weight: expected {dt} or torch.float32, got {wdt}")
    if weight.get_device() != dev:
        raise ValueError("weight: expected on the device of the rows")
    if not weight.is_contiguous():
        raise ValueError("weight: must be contiguous")
    code = _lib.dtype_code(dt)
    return H, dev, code, code if wdt is dt else _lib.F32


def _check_like(name: str, t: torch.Tensor, x: torch.Tensor) -> None:
    if not t.is_same_size(x):
        raise ValueError(f"{name}: expected shape {tuple(x.shape)}, got {tuple(t.shape)}")
    if t.dtype is not x.dtype:
        raise TypeError(f"{name}: expected dtype {x.dtype}, got {t.dtype}")
    if t.get_device() != x.get_device():
        raise ValueError(f"{name}: expected on {x.device}, got {t.device}")


def _dense_like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def rms_norm_forward(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                     residual: Optional[torch.Tensor] = None, want_rstd: bool = True):
    """``(y, rstd, total)``: ``total`` is ``x + residual`` rounded to the rows'
    type (``x`` itself without a residual), ``y`` its norm, ``rstd`` the fp32
    1/sqrt(mean + eps) of every row for :func:`rms_norm_backward` (None unless
    wanted)."""
    H, dev, code, wcode = _check(x, weight)
    if not eps >= 0:
        raise ValueError(f"eps: expected >= 0, got {eps}")
    n = x.numel() // H
    xr, ldx = _rows(x, H)
    at = ptr(xr)                  # on a CUDA device, and so are the others
    y = _dense_like(x)
    rstd = x.new_empty(n, dtype=torch.float32) if want_rstd else None
    total, res_at, ldr, total_at = x, None, 0, None
    if residual is not None:
        _check_like("residual", residual, x)
        residual, ldr = _rows(residual, H)
        total = _dense_like(x)
        res_at, total_at = residual.data_ptr(), total.data_ptr()
    call_on(dev, "usaf_rms_norm_fwd", at, ldx, res_at, ldr, weight.data_ptr(), code, wcode, n, H, float(eps), total_at,
            y.data_ptr(), rstd.data_ptr() if want_rstd else None)
    return y, rstd, total


def rms_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                      dsum: Optional[torch.Tensor] = None, want_dw: bool = True):
    """``(dx, dw)`` from the gradient ``dy`` of ``y``; ``x`` is the ``total`` of
    :func:`rms_norm_forward`.  ``dsum``, the gradient of ``total`` where it is
    used further, is added to ``dx``, which is then the gradient of ``x`` and of
    ``residual`` alike.  ``dw`` has the weight's type (None unless wanted)."""
    H, dev, code, wcode = _check(x, weight)
    n = x.numel() // H
    _check_like("dy", dy, x)
    if rstd.numel() != n or rstd.dtype is not torch.float32 or rstd.get_device() != dev or not rstd.is_contiguous():
        raise ValueError(f"rstd: expected {n} contiguous fp32 values on {x.device}")
    xr, ldx = _rows(x, H)
    at = ptr(xr)                  # on a CUDA device, and so are the others
    dyr, lddy = _rows(dy, H)
    ds_at, ldds = None, 0
    if dsum is not None:
        _check_like("dsum", dsum, x)
        dsum, ldds = _rows(dsum, H)
        ds_at = dsum.data_ptr()
    dx = _dense_like(x)
    dw = dw_at = ws_at = None
    if want_dw:
        dw = torch.empty_like(weight)
        ws = x.new_empty(_lib.LIB.usaf_rms_norm_workspace_bytes(n, H), dtype=torch.uint8)
        dw_at, ws_at = dw.data_ptr(), ws.data_ptr()
    call_on(dev, "usaf_rms_norm_bwd", dyr.data_ptr(), lddy, at, ldx, weight.data_ptr(), rstd.data_ptr(), ds_at, ldds,
            code, wcode, n, H, dx.data_ptr(), dw_at, ws_at)
    return dx, dw


class _RmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        y, rstd, total = rms_norm_forward(x, weight, eps, residual)
        ctx.save_for_backward(total, weight, rstd)
        ctx.has_residual = residual is not None
        ctx.set_materialize_grads(False)      # an unused output has no gradient to read
        return (y, total) if ctx.has_residual else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        total, weight, rstd = ctx.saved_tensors
        want_dw = ctx.needs_input_grad[1]
        if dy is None:
            dx, dw = dsum, (torch.zeros_like(weight) if want_dw else None)
        else:
            dx, dw = rms_norm_backward(dy, total, weight, rstd, dsum, want_dw=want_dw)
        return dx, dw, None, dx if ctx.has_residual else None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """``y``, the RMS norm of ``x`` over its last dimension; with ``residual``
    the pair ``(y, total)`` of the norm of ``x + residual`` and that sum.
    Differentiable in ``x``, ``weight`` and ``residual``, once and backward;
    forward mode is refused."""
    if differentiated(x, weight, residual):
        return _RmsNormFn.apply(x, weight, eps, residual)
    y, _, total = rms_norm_forward(x, weight, eps, residual, want_rstd=False)
    return y if residual is None else (y, total)
