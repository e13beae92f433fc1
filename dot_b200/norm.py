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
in place and computed in float32.  The reference has no such operator.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib, ops


class _GroupNormActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, lengths, num_groups: int, eps: float, activation: int):
        y, stats = ops.group_norm_forward_raw(x, num_groups, weight, bias, eps, activation, lengths)
        ctx.save_for_backward(x, weight, bias, lengths, stats)
        ctx.groups_act = (num_groups, activation)
        return y

    @staticmethod
    def _grads(ctx, dy):
        x, weight, bias, lengths, stats = ctx.saved_tensors
        num_groups, activation = ctx.groups_act
        dx, dw, db = ops.group_norm_backward_raw(x, dy, num_groups, weight, bias, activation, stats, lengths,
                                                 *ctx.needs_input_grad[:3])
        return dx, dw, db, None, None, None, None

    _grads_once = staticmethod(once_differentiable(_grads.__func__))

    @staticmethod
    def backward(ctx, dy):
        # the wrapper that refuses a second differentiation is needed where one is recorded
        if torch.is_grad_enabled():
            return _GroupNormActFn._grads_once(ctx, dy)
        return _GroupNormActFn._grads(ctx, dy)


_ACTIVATION_CODES = {name: code for code, name in enumerate(_lib.ACTIVATIONS)}


def _activation_code(activation: str) -> int:
    code = _ACTIVATION_CODES.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {', '.join(_lib.ACTIVATIONS)}, got {activation!r}")
    return code


def _check_param(p: torch.Tensor, C: int, name: str, x: torch.Tensor) -> torch.Tensor:
    if p.dim() != 1 or p.size(0) != C:
        raise ValueError(f"{name} must have shape [{C}]")
    if p.get_device() != x.get_device():
        raise ValueError(f"{name} must be on {x.device}")
    return p if p.is_contiguous() else p.contiguous()


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, activation: str = "silu",
                   lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Group norm and activation of ``x`` [N, *S, C]; returns a dense tensor of x's shape and dtype.

    ``activation``: "silu", "gelu" (the erf form), "relu" or "none".
    ``weight``, ``bias``: [C], float32 or a 16-bit type.  ``lengths``: int32
    [N], valid positions of each sample in the flattened position axes.
    Gradients for x, weight and bias (once differentiable).
    """
    if not x.is_cuda:
        raise RuntimeError("dot_b200: x must be a CUDA tensor (dot_b200 runs on NVIDIA GPUs only)")
    if x.dim() < 2:
        raise ValueError("x must be [N, ..., C]")
    if x.dtype not in ops._FEATURE_DTYPES:
        raise NotImplementedError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    C = x.size(-1)
    if num_groups < 1 or C % num_groups != 0:
        raise ValueError(f"num_groups ({num_groups}) must be >= 1 and divide the channels ({C})")
    if not eps >= 0:
        raise ValueError("eps must be >= 0")
    act = _activation_code(activation)
    grad = x.requires_grad
    if weight is not None:
        weight = _check_param(weight, C, "weight", x)
        grad = grad or weight.requires_grad
    if bias is not None:
        bias = _check_param(bias, C, "bias", x)
        grad = grad or bias.requires_grad
    dt = x.dtype if weight is None else weight.dtype
    if dt not in ops._FEATURE_DTYPES or (bias is not None and bias.dtype != dt):
        # the kernels read both parameters as one type
        weight = None if weight is None else weight.to(torch.float32)
        bias = None if bias is None else bias.to(torch.float32)
    if lengths is not None:
        if lengths.dim() != 1 or lengths.size(0) != x.size(0):
            raise ValueError("lengths must be [N]")
        if lengths.dtype != torch.int32:
            raise ValueError("lengths must be int32")
        lengths = lengths.to(x.device).contiguous()
    if grad and torch.is_grad_enabled():
        return _GroupNormActFn.apply(x, weight, bias, lengths, num_groups, eps, act)
    return ops.group_norm_forward_raw(x, num_groups, weight, bias, eps, act, lengths)[0]


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
