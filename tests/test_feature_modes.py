"""Ways of calling the feature operators that their torch binding cannot serve:
a tangent of forward-mode differentiation and a trace are refused, not passed
by.  The refusals come before the device is looked at, so most need no GPU."""

import pytest
import torch
import torch.autograd.forward_ad as fw

import dot

FREQS = torch.ones(4, 2)
POS = torch.zeros(3, 2)


def calls(device):
    """Each input that may carry a tangent, with the call that takes it."""
    x, c, q = torch.rand(2, 3, 8, device=device), torch.rand(8, device=device), torch.rand(1, 3, 2, 8, device=device)
    pos, freqs = POS.to(device), FREQS.to(device)
    return [
        (x, lambda t: dot.group_norm_act(t, 2)),
        (c, lambda t: dot.group_norm_act(x, 2, t)),
        (c, lambda t: dot.group_norm_act(x, 2, None, t)),
        (q, lambda t: dot.rotary(t, pos, freqs)),
        (q, lambda t: dot.rotary(q, pos, freqs, k=t)),
        (pos, lambda t: dot.rotary(q, t, freqs)),
        (freqs, lambda t: dot.rotary(q, pos, t)),
    ]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("i", range(7))
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(device, i, grad):
    t, call = calls(device)[i]
    with fw.dual_level():
        dual = fw.make_dual(t.requires_grad_(grad), torch.ones_like(t))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        with pytest.raises(NotImplementedError, match="forward-mode"), torch.no_grad():
            call(dual)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("i", range(7))
def test_traces_are_refused(device, i):
    t, call = calls(device)[i]
    with pytest.raises(NotImplementedError, match="torch.jit.trace"):
        torch.jit.trace(call, (t,), check_trace=False)


@pytest.mark.gpu
def test_tangents_of_upstream_gradients_are_refused():
    x = torch.rand(2, 3, 8, device="cuda", requires_grad=True)
    q = torch.rand(1, 3, 2, 8, device="cuda", requires_grad=True)
    for leaf, y in ((x, dot.group_norm_act(x, 2)), (q, dot.rotary(q, POS.cuda(), FREQS.cuda()))):
        with fw.dual_level():
            up = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
            for create in (False, True):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    torch.autograd.grad(y, leaf, up, retain_graph=True, create_graph=create)
        (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y))   # and without one the gradient is there
        assert g.shape == leaf.shape
