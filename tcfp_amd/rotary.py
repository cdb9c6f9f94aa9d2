"""Rotary positions of queries and keys (HIP, gfx950; no reference counterpart).

:func:`rotary_embedding` turns pairs of columns of every head by angles that
grow with the token's position, in training (it has a gradient) and in front of
``attention.kv_cache_write`` and ``attention.paged_attention`` when serving;
:func:`rotary_frequencies` makes the angles a position, stretched for contexts
longer than the trained one if asked.

Every op runs on the tensors' GPU and current stream; there is no CPU path.
"""
from __future__ import annotations

import math

import torch

from . import _hip

__all__ = ["rotary_frequencies", "rotary_embedding"]


def rotary_frequencies(
    dim: int,
    *,
    base: float = 10000.0,
    factor: float = 1.0,
    trained_length: int | None = None,
    slow_turns: float = 1.0,
    fast_turns: float = 32.0,
    device: torch.device | str | None = None,
) -> torch.Tensor:
    """Radians a position of each of the ``dim / 2`` pairs, ``base ** (-2 i /
    dim)``, float64.

    ``factor`` > 1 stretches them for a context that many times longer.  Without
    ``trained_length`` every pair is slowed down by it.  With it, pairs that turn
    fewer than ``slow_turns`` times within the trained length are slowed down,
    pairs that turn more than ``fast_turns`` times keep their pace (they tell
    neighbours apart, and have turned through every angle in training), and
    those between are blended linearly in their number of turns.
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and at least 2, got {dim}")
    if not (base > 0 and math.isfinite(base) and factor >= 1 and math.isfinite(factor)):
        raise ValueError(f"base must be positive and factor at least 1, got {base} and {factor}")
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if trained_length is None:
        f = f / factor
    else:
        if trained_length < 1 or not 0 <= slow_turns < fast_turns:
            raise ValueError("trained_length must be positive and slow_turns below fast_turns, got "
                             f"{trained_length}, {slow_turns} and {fast_turns}")
        turns = trained_length * f / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    return f if device is None else f.to(device)


def rotary_embedding(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    freqs: torch.Tensor,
    *,
    interleaved: bool = False,
    amplitude: float = 1.0,
    inverse: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``q`` [tokens, heads, dim] and ``k`` [tokens, kv_heads, dim] (fp32 or bf16;
    slices of a QKV projection's output are taken as they are; ``k`` may be None)
    with their first ``2 * len(freqs)`` columns turned.

    Pair i of a token's heads, ``(a, b)``, becomes ``amplitude * (a cos - b sin, a
    sin + b cos)`` of the angle ``positions[token] * freqs[i]`` (``positions``
    int64 [tokens], ``freqs`` float64, at most 2048 of them), the other columns stay
    as they are.  The pair's columns are ``i`` and ``len(freqs) + i``, or with
    ``interleaved`` ``2 i`` and ``2 i + 1``.  ``inverse`` turns the other way.
    Angles are formed in fp64, products in fp32, results rounded once, in new
    tensors.

    Differentiable in ``q`` and ``k``, any number of times: the gradient is turned the
    other way.
    """
    return _hip.host().rotary_embedding(q, k, positions, freqs, bool(interleaved),
                                        float(amplitude), bool(inverse))
