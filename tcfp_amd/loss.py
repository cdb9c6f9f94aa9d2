"""Softmax cross entropy of a linear head over a large vocabulary, with its
gradients, without storing the logits (HIP, gfx950; no reference counterpart).

The head of a language model multiplies the last hidden states with a weight of
one row a class; its logits, tokens x classes, are the largest matrix of a
training step.  Here the product's own epilogue reduces them to each token's
maximum and sum of exponentials.  The gradients of a sum or mean are made in the
same call, from exponentials in 16 bits that take at most 1 GiB of workspace while it
runs; where they would take more, and for gradients of every token's loss, the
backward pass forms the logits again, a run of classes at a time (256 MiB for the
run's gradients, or 512 bytes a token if that is more, and fp32 sums of the hidden states').  Memory beside the inputs and
gradients stays bounded either way.

Every op runs on the tensors' GPU and current stream; there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _hip

__all__ = ["linear_cross_entropy", "linear_cross_entropy_forward", "linear_cross_entropy_backward"]


def linear_cross_entropy(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.Tensor,
    *,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> torch.Tensor:
    """Cross entropy of ``hidden @ weight.T`` with ``targets``, fp32.

    ``hidden`` [..., D] and ``weight`` [classes, D] are bf16 (a head kept in fp32 is
    cast where it is used: ``weight.bfloat16()``), D a multiple of 8, rows of 2-D
    tensors may be apart; ``targets`` [...] int64.  Tokens whose target is
    ``ignore_index`` are left out: their loss is 0, their hidden state gets a zero
    gradient, and the mean is over the others (NaN if there are none).  A target that
    is neither that nor a class gives NaN.  Products and sums are fp32 (the
    reduction's fp64).

    ``reduction`` is ``"mean"``, ``"sum"`` or ``"none"`` (a loss for every token).
    Differentiable in ``hidden`` and ``weight``, once; gradients are bf16.  Those of a sum
    or mean are multiplied with the loss's own gradient once they are made, which rounds
    them a second time unless that is a power of two, and leave out classes less than
    2^-39 as likely as the likeliest of their 128 or 256 neighbours.  The hidden
    states of tokens left out are read all the same: a value there that is not
    finite reaches the weight's gradient.
    """
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    return _hip.host().linear_cross_entropy(hidden, weight, targets, int(ignore_index),
                                            reduction != "none", reduction == "mean")


def linear_cross_entropy_forward(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.Tensor,
    *,
    ignore_index: int = -100,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(losses, lse)`` of every token, fp32: :func:`linear_cross_entropy` without
    autograd or reduction, and the log sum of exponentials of its logits, which
    :func:`linear_cross_entropy_backward` takes."""
    return _hip.host().linear_cross_entropy_forward(hidden, weight, targets, int(ignore_index),
                                                    False, False)[:2]


def linear_cross_entropy_backward(
    grad: torch.Tensor,
    hidden: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.Tensor,
    lse: torch.Tensor,
    *,
    losses: torch.Tensor | None = None,
    count: torch.Tensor | None = None,
    ignore_index: int = -100,
    need_hidden_grad: bool = True,
    need_weight_grad: bool = True,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """``(grad_hidden, grad_weight)`` in bf16 (None where not asked for) of
    :func:`linear_cross_entropy`.

    ``grad`` (fp32) is the gradient of every token's loss, or one value for all of
    them, which ``count`` (one fp32 value on the device: the tokens of a mean)
    divides; ``lse`` and ``losses`` are what :func:`linear_cross_entropy_forward` returned.
    Without ``losses`` the gradient of a target's logit comes from ``lse``, whose rounding
    (2^-24 of it) is then in it: much, where a target's class is almost certain.
    """
    return _hip.host().linear_cross_entropy_backward(grad, hidden, weight, targets, lse, losses,
                                                     count, int(ignore_index),
                                                     bool(need_hidden_grad), bool(need_weight_grad))
