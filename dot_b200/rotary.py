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
of heads are turned in one launch; a single token is an ordinary call.  Checks,
allocation and autograd are in ``csrc/torch_features.cpp``;
:func:`dot_b200.ops.rotary_raw` is a single call of the C-ABI.  The reference
has no such operator.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch
import torch.nn as nn

from . import _lib


def rotary(q: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, k: Optional[torch.Tensor] = None,
           interleaved: bool = False):
    """``q`` [*, L, Hq, D] (and ``k`` [*, L, Hk, D]) with every head turned by its token's angles.

    ``positions``: [*, L, A] with q's leading axes, or [L, A] for all of them;
    int32, int64 or float32, any strides.  ``freqs``: float32 [P, A],
    2 P <= D; elements from 2 P on pass through.  Pair p is (x_p, x_{P+p}), or
    (x_2p, x_2p+1) with ``interleaved``.  q and k may be slices of wider rows
    (a fused projection); the results are dense.  Returns q', or (q', k') when
    k is given.  Differentiable in q and k, not in positions or freqs;
    forward-mode tangents and ``torch.jit.trace`` raise NotImplementedError.
    """
    q, turned_k = _lib.torch_binding().rotary(q, positions, freqs, k, interleaved)
    return q if k is None else (q, turned_k)


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
