"""Residual addition and root-mean-square norm, with FP8 or plain output, and
its backward (HIP, gfx950; no reference counterpart).

The norm stands in front of the linear layers of a decoder.
:func:`rms_norm_quantize` writes what the block-scaled GEMMs read -- E4M3
codes and block scales, as ``kernels.block_quantize_fp8`` makes them -- in the
pass that computes the norm, so the normalised activations never reach memory
in a wider type.  :func:`rms_norm` writes them plainly (the last norm in front
of an unquantised head), and :func:`rms_norm_backward` is the gradient of both:
the quantisation passes gradients through, as in the TCFP layers.

Every op runs on the tensors' GPU and current stream; there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _hip
from .kernels import _scale_format

__all__ = ["rms_norm", "rms_norm_quantize", "rms_norm_backward"]


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    out_dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``y = s * rstd * weight`` with ``s = x + residual`` and ``rstd = 1 /
    sqrt(mean(s^2) + eps)`` over the last axis.

    ``x`` and ``residual`` (one shape, fp32 or bf16 each; rows of 2-D tensors
    may be apart), ``weight`` [D] fp32 or bf16.  Sums and products are fp32.
    Returns ``(y, h, rstd)``: ``y`` in ``out_dtype`` (``x``'s by default),
    ``h`` = s in the residual's dtype (``x`` itself without a residual), and
    the fp32 ``rstd`` of every row, which the backward takes.  ``y`` is formed
    from s before its rounding to ``h``.
    """
    return _hip.host().rms_norm(x, weight, residual, float(eps),
                                x.dtype if out_dtype is None else out_dtype)


def rms_norm_quantize(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    block_size: int = 64,
    fp8_dtype: torch.dtype = torch.float8_e4m3fn,
    scale_format: str = "exponent",
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`rms_norm` whose output is FP8 codes and block scales.

    Returns ``(q, scales, h, rstd)``: ``q`` (shape of ``x``) and ``scales``
    [D // block_size, rows] as ``kernels.block_quantize_fp8`` returns them for
    the fp32 ``y`` -- int8 exponents, or fp32 multipliers with
    ``scale_format="fp32"``.  ``block_size`` 32, 64 or 128 divides D.
    """
    return _hip.host().rms_norm_quantize(x, weight, residual, float(eps), int(block_size),
                                         fp8_dtype, _scale_format(scale_format))


def rms_norm_backward(
    grad_y: torch.Tensor,
    h: torch.Tensor,
    rstd: torch.Tensor,
    weight: torch.Tensor,
    grad_h: torch.Tensor | None = None,
    *,
    need_weight_grad: bool = True,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Gradients of :func:`rms_norm` / :func:`rms_norm_quantize`.

    ``h`` and ``rstd`` are what the forward returned, ``grad_y`` (fp32 or
    bf16) the gradient of the normalised output and ``grad_h`` (``h``'s
    dtype) that of ``h``, when the residual stream is used further on.
    Returns ``(grad_x, grad_weight)``: ``grad_x`` in ``h``'s dtype, the
    gradient of ``x`` and of the residual alike, and the fp32 weight gradient
    (None with ``need_weight_grad=False``), summed over the rows in an order
    that depends on the sizes alone.
    """
    return _hip.host().rms_norm_backward(grad_y, h, rstd, weight, grad_h, bool(need_weight_grad))
