"""Rotary positions with several axes.

``rotary(q, positions, freqs)`` turns pairs of every head's elements by angles
that are linear in the token's position:

    angle[t, p] = sum_a positions[t, a] * freqs[p, a]
    (x, y) -> (x cos - y sin, y cos + x sin)

so the product of two turned features depends on the difference of their
positions.  The axes may be row and column of an image, time, height and width
of a clip, or the coordinates of a keypoint; a row of ``freqs`` with one
non-zero entry gives a pair to one axis (:func:`rotary_freqs` builds such
tables), a full row mixes the axes.  Queries and keys with different numbers
of heads are turned in one launch; a single token is an ordinary call.  The
reference has no such operator.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch
import torch.nn as nn

from . import ops


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freqs, interleaved: bool, inverse: bool):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, freqs)
        ctx.flags = (interleaved, inverse)
        return ops.rotary_raw(q, k, positions, freqs, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        need = ctx.needs_input_grad
        if not need[0]:
            dq = None
        if not need[1]:
            dk = None
        if dq is None and dk is None:
            return (None,) * 6
        positions, freqs = ctx.saved_tensors
        interleaved, inverse = ctx.flags
        # the turn is orthogonal: its backward is the turn by -angle
        turn = _RotaryFn.apply if torch.is_grad_enabled() else ops.rotary_raw
        dq, dk = turn(dq, dk, positions, freqs, interleaved, not inverse)
        return dq, dk, None, None, None, None


def _check_heads(x: torch.Tensor, name: str) -> None:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError(f"dot_b200: {name} must be a CUDA tensor (dot_b200 runs on NVIDIA GPUs only)")
    if x.dim() < 3:
        raise ValueError(f"{name} must be [..., tokens, heads, head_dim]")
    if x.dtype not in ops._FEATURE_DTYPES:
        raise NotImplementedError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")


def _as_4d(x: torch.Tensor) -> torch.Tensor:
    if x.dim() == 3:
        return x.unsqueeze(0)
    return x.reshape(math.prod(x.shape[:-3]), *x.shape[-3:])


def rotary(q: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, k: Optional[torch.Tensor] = None,
           interleaved: bool = False):
    """``q`` [*, L, Hq, D] (and ``k`` [*, L, Hk, D]) with every head turned by its token's angles.

    ``positions``: [*, L, A] with q's leading axes, or [L, A] for all of them;
    int32, int64 or float32, any strides.  ``freqs``: float32 [P, A],
    2 P <= D; elements from 2 P on pass through.  Pair p is (x_p, x_{P+p}), or
    (x_2p, x_2p+1) with ``interleaved``.  q and k may be slices of wider rows
    (a fused projection); the results are dense.  Returns q', or (q', k') when
    k is given.  Differentiable in q and k, not in positions or freqs.
    """
    _check_heads(q, "q")
    shape = q.shape
    lead = shape[:-2]
    grad = q.requires_grad
    if k is not None:
        _check_heads(k, "k")
        if k.shape[:-2] != lead or k.size(-1) != shape[-1]:
            raise ValueError("k must have q's shape except for the number of heads")
        if k.dtype != q.dtype or k.get_device() != q.get_device():
            raise ValueError("k must have q's dtype and device")
        grad = grad or k.requires_grad
    if freqs.dim() != 2 or freqs.dtype != torch.float32:
        raise ValueError("freqs must be float32 [P, A]")
    if positions.dtype not in ops._POSITION_DTYPES:
        raise ValueError("positions must be int32, int64 or float32")
    if positions.get_device() != q.get_device() or freqs.get_device() != q.get_device():
        raise ValueError("positions and freqs must be on q's device")
    if positions.requires_grad or freqs.requires_grad:
        raise ValueError("positions and freqs are not differentiable here: detach them")
    P, A = freqs.shape
    if not 1 <= A <= 4:
        raise ValueError("freqs must have 1 to 4 axes")
    if 2 * P > shape[-1]:
        raise ValueError("freqs must hold at most D/2 pairs")
    if positions.shape != (*lead, A):
        if positions.shape != (lead[-1], A):
            raise ValueError("positions must be [*, L, A] with q's leading axes, or [L, A]")
        positions = positions.unsqueeze(0)
    elif len(lead) != 2:
        positions = positions.reshape(math.prod(lead[:-1]), lead[-1], A)
    if not freqs.is_contiguous():
        freqs = freqs.contiguous()
    q4, k4 = (q, k) if len(lead) == 2 else (_as_4d(q), None if k is None else _as_4d(k))
    if grad and torch.is_grad_enabled():
        q4, k4 = _RotaryFn.apply(q4, k4, positions, freqs, bool(interleaved), False)
    else:
        q4, k4 = ops.rotary_raw(q4, k4, positions, freqs, bool(interleaved))
    if len(lead) != 2:
        q4 = q4.view(shape)
        k4 = None if k is None else k4.view(k.shape)
    return q4 if k is None else (q4, k4)


def rotary_freqs(sections: Sequence[int], theta: float = 10000.0, shared_band: bool = False,
                 device=None) -> torch.Tensor:
    """Frequencies [P, A] that give ``sections[a]`` pairs to axis a, in order (P = sum(sections)).

    Each axis has its own band, theta ** (-j / sections[a]); with
    ``shared_band`` all pairs share one, theta ** (-p / P), cut into sections.
    """
    sections = [int(n) for n in sections]
    if not 1 <= len(sections) <= 4 or any(n < 0 for n in sections):
        raise ValueError("sections must be 1 to 4 numbers of pairs >= 0")
    if not theta > 0:
        raise ValueError("theta must be > 0")
    P = sum(sections)
    table = torch.zeros((P, len(sections)), dtype=torch.float64)
    at = 0
    for a, n in enumerate(sections):
        exponent = torch.arange(at, at + n, dtype=torch.float64) / P if shared_band and n else \
            torch.arange(n, dtype=torch.float64) / max(n, 1)
        table[at:at + n, a] = float(theta) ** -exponent
        at += n
    return table.to(device=device, dtype=torch.float32)


class Rotary(nn.Module):
    """``nn.Module`` of :func:`rotary` that holds its frequencies (a buffer, always float32)."""

    def __init__(self, sections: Sequence[int], theta: float = 10000.0, shared_band: bool = False,
                 interleaved: bool = False, device=None):
        super().__init__()
        self.sections = tuple(int(n) for n in sections)
        self.interleaved = interleaved
        self.register_buffer("freqs", rotary_freqs(sections, theta, shared_band, device), persistent=False)

    def _apply(self, fn, recurse=True):
        # a cast of the module to 16 bits moves the table but does not round it
        freqs = self.freqs
        super()._apply(fn, recurse)
        if self.freqs.dtype != torch.float32:
            self.freqs = freqs.to(self.freqs.device)
        return self

    def forward(self, q: torch.Tensor, positions: torch.Tensor, k: Optional[torch.Tensor] = None):
        return rotary(q, positions, self.freqs, k=k, interleaved=self.interleaved)

    def extra_repr(self) -> str:
        return f"sections={self.sections}, interleaved={self.interleaved}"
