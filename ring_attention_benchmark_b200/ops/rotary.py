"""Rotary positions on q and k (sm_100a), with their gradient.

A pair (x1, x2) of token t is turned by ``positions[t] * inv_freq[p]``:
``(x1 cos - x2 sin, x2 cos + x1 sin) * scale``.  Two layouts: *half* pairs
element p with p + rotary_dim / 2, *interleaved* pairs 2p with 2p + 1; elements
behind ``rotary_dim = 2 * inv_freq.numel()`` pass through.  Positions are whole
numbers of any size: the kernel keeps the angle as a 64-bit fraction of a turn,
so far positions lose nothing.

Tensors are ``[tokens, heads, dim]`` in bf16, fp16 or fp32, with any strides
between tokens and heads (slices of one projection need no copy); sines,
products and sums are fp32 and each element is rounded once.

    inv_freq, scale = rotary_frequencies(128, base=500000.0, scaling="yarn", factor=8.0,
                                         original_length=8192, device="cuda")
    q, k = apply_rotary(q, k, positions, inv_freq, scale=scale)

`Rotary` holds the frequencies and the layout; `RingAttention(rotary=...)`
applies it to every call's q and k at this rank's global positions.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .._ext import load

SCALINGS = ("none", "linear", "ntk", "yarn", "bands")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none",
                       factor: float = 1.0, original_length: Optional[int] = None,
                       fast: float = 32.0, slow: float = 1.0, device=None
                       ) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, scale)``: float64 frequencies of the pairs (radians per
    position) and the factor on the rotated elements.

    ``scaling`` stretches the positions for contexts ``factor`` times as long as
    the ``original_length`` tokens the weights were trained with:

    * ``"none"``: ``base ** (-2 p / rotary_dim)``
    * ``"linear"``: every frequency divided by ``factor``
    * ``"ntk"``: the base grows by ``factor ** (rotary_dim / (rotary_dim - 2))``,
      so the slowest pair is divided by ``factor`` and the fastest kept
    * ``"yarn"``: pairs that turn more than ``fast`` times within
      ``original_length`` are kept, those below ``slow`` turns divided by
      ``factor``, a linear ramp over the pair index between the two; the scale is
      ``0.1 ln(factor) + 1``
    * ``"bands"``: as yarn, but the ramp runs linearly in the number of turns,
      and the scale stays 1
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError(f"base must be over 1, got {base}")
    if not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError(f"factor must be 1 or more, got {factor}")
    n = rotary_dim // 2
    p = torch.arange(n, dtype=torch.float64)
    scale = 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs rotary_dim over 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv = base ** (-2.0 * p / rotary_dim)
    if scaling == "linear":
        inv = inv / factor
    elif scaling in ("yarn", "bands"):
        if original_length is None or original_length < 1:
            raise ValueError(f"{scaling} scaling needs original_length")
        if not fast > slow > 0:
            raise ValueError("yarn and bands scaling need fast > slow > 0")
        if scaling == "yarn":
            # the pair index at which a pair turns `t` times within the original length
            def index(t):
                return rotary_dim * math.log(original_length / (2 * math.pi * t)) / (2 * math.log(base))

            lo = max(0.0, math.floor(index(fast)))
            # may lie behind the last pair: then no pair is divided by the whole factor
            hi = min(float(rotary_dim - 1), math.ceil(index(slow)))
            keep = 1.0 - ((p - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
            scale = 0.1 * math.log(factor) + 1.0
        else:
            turns = original_length * inv / (2 * math.pi)
            keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        inv = inv * keep + inv / factor * (1.0 - keep)
    return inv.to(device) if device is not None else inv, scale


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 inv_freq: torch.Tensor, *, interleaved: bool = False, scale: float = 1.0,
                 inverse: bool = False,
                 out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None):
    """Rotate ``q`` (and ``k``) to ``positions`` (int64 or int32, one per token).

    Returns ``(q', k')``, or ``q'`` alone when ``k`` is None.  ``inverse`` turns
    the other way.  ``out=(q_out, k_out)`` takes the results; passing the inputs
    themselves rotates in place (not where a gradient is needed).  What it writes
    counts as changed in place: a backward pass that saved it raises.

    The gradient is for backward passes, and for theirs; forward-mode tangents are refused.
    Forward and backward can be captured into a CUDA graph together.  As with
    every autograd operation, no eager graph that reaches the same leaves may be
    alive then: torch would wait for the eager graph's stream inside the capture
    and end it with an error.
    """
    if out is not None and torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (q, k, *out)):
        raise ValueError("apply_rotary: out= is not offered where a gradient is needed")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        qo, ko = load().rotary_autograd(q, k, positions, inv_freq, interleaved, scale, inverse)
        return qo if k is None else (qo, ko)
    if out is None:
        qo, ko = load().rotary(q, k, positions, inv_freq, interleaved, scale, inverse)
    else:
        qo, ko = load().rotary(q, k, positions, inv_freq, interleaved, scale, inverse, out[0],
                               out[1])
    return qo if k is None else (qo, ko)


class Rotary:
    """Frequencies and layout of a model's rotary positions, on one device.

        rotary = Rotary(head_dim, base=500000.0, interleaved=True, device="cuda")
        q, k = rotary(q, k, positions)
    """

    def __init__(self, rotary_dim: int, base: float = 10000.0, interleaved: bool = False,
                 scaling: str = "none", factor: float = 1.0,
                 original_length: Optional[int] = None, fast: float = 32.0, slow: float = 1.0,
                 device="cuda"):
        self.interleaved = bool(interleaved)
        self.rotary_dim = rotary_dim
        self.inv_freq, self.scale = rotary_frequencies(
            rotary_dim, base, scaling, factor, original_length, fast, slow, device)

    def to(self, device) -> "Rotary":
        """The same rotation with its frequencies on another device."""
        other = object.__new__(Rotary)
        other.__dict__.update(self.__dict__, inv_freq=self.inv_freq.to(device))
        return other

    def __call__(self, q, k, positions, out=None):
        return apply_rotary(q, k, positions, self.inv_freq, interleaved=self.interleaved,
                            scale=self.scale, out=out)
