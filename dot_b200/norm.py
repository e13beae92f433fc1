"""Group normalisation with an activation on channels-last features.

``group_norm_act(x, num_groups, weight, bias)`` normalises x [N, *S, C] (any
number of position axes, channels last) over each sample's positions and
groups of C / num_groups consecutive channels, applies the channels' weight
and bias and an activation, in one operator with its backward:

    z = (x - mean) / sqrt(var + eps) * weight + bias,    y = act(z)

It stands between the layers that produce the features of a matching; a
position's features stay one row, as the score product and ``rotary`` read
them.  A tensor in torch's channels-last memory format [N, C, H, W] enters as
the view ``x.permute(0, 2, 3, 1)``, without a copy.  ``lengths`` holds each
sample's number of valid positions in padded sets (the same convention as
``bidirectional_softmax``'s): what lies beyond is neither read nor counted,
and its outputs and gradients are 0.  float32, bfloat16 and float16 are read
in place and computed in float32.  Checks, allocation and autograd are in
``csrc/torch_features.cpp``; :func:`dot_b200.ops.group_norm_forward_raw` and
``group_norm_backward_raw`` are single calls of the C-ABI.  The reference has
no such operator.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _lib

_ACTIVATION_CODES = {name: code for code, name in enumerate(_lib.ACTIVATIONS)}


def _activation_code(activation: str) -> int:
    code = _ACTIVATION_CODES.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {', '.join(_lib.ACTIVATIONS)}, got {activation!r}")
    return code


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, activation: str = "silu",
                   lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Group norm and activation of ``x`` [N, *S, C]; returns a dense tensor of x's shape and dtype.

    ``num_groups``: divides C, at most 28544.
    ``activation``: "silu", "gelu" (the erf form), "relu" or "none".
    ``weight``, ``bias``: [C], float32 or a 16-bit type.  ``lengths``: int32
    [N], valid positions of each sample in the flattened position axes.
    Gradients for x, weight and bias (once differentiable, in reverse mode);
    forward-mode tangents and ``torch.jit.trace`` raise NotImplementedError.
    """
    return _lib.torch_binding().group_norm_act(x, num_groups, weight, bias, eps, _activation_code(activation), lengths)


class GroupNormAct(nn.Module):
    """``nn.Module`` of :func:`group_norm_act` with weight 1 and bias 0 to start from."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str = "silu", device=None, dtype=None):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups != 0:
            raise ValueError("num_groups must be >= 1 and divide num_channels")
        _activation_code(activation)
        self.num_groups = num_groups
        self.num_channels = num_channels
        self.eps = eps
        self.activation = activation
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels, device=device, dtype=dtype))
            self.bias = nn.Parameter(torch.zeros(num_channels, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        if x.size(-1) != self.num_channels:
            raise ValueError(f"x must have {self.num_channels} channels last")
        return group_norm_act(x, self.num_groups, self.weight, self.bias, eps=self.eps, activation=self.activation,
                              lengths=lengths)

    def extra_repr(self) -> str:
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, activation={self.activation!r}"
