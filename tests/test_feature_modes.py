"""Tensors and ways of calling that a binding working on memory could pass by: a
tangent of forward-mode differentiation and a trace are refused (before the device
is looked at, so most of it needs no GPU), a view that torch negates when it is read
counts as what it stands for, one without memory is refused."""

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


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(7))
def test_negated_views(i):
    t, call = calls("cuda")[i]
    view = torch._neg_view(t)
    assert view.is_neg() and torch.equal(call(view)[0], call(-t)[0])


@pytest.mark.gpu
def test_negated_views_of_complex_numbers():
    """Imaginary parts of conjugates, as positions in place and as the single channel of an input."""
    z = torch.randn(3, 2, 2, device="cuda")
    z = torch.view_as_complex(z).conj()
    q = torch.rand(1, 3, 2, 8, device="cuda")
    assert z.imag.is_neg()
    assert torch.equal(dot.rotary(q, z.imag, FREQS.cuda()), dot.rotary(q, z.imag.clone(), FREQS.cuda()))
    x = z.imag[..., None]
    assert torch.equal(dot.group_norm_act(x, 1), dot.group_norm_act(x.clone(), 1))


@pytest.mark.gpu
def test_negated_upstream_gradients():
    x = torch.rand(2, 3, 8, device="cuda", requires_grad=True)
    q = torch.rand(1, 3, 2, 8, device="cuda", requires_grad=True)
    for leaf, y in ((x, dot.group_norm_act(x, 2)), (q, dot.rotary(q, POS.cuda(), FREQS.cuda()))):
        dy = torch.rand_like(y)
        got, want = (torch.autograd.grad(y, leaf, g, retain_graph=True)[0] for g in (torch._neg_view(dy), -dy))
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(7))
def test_tensors_without_memory_are_refused(i):
    t, call = calls("cuda")[i]
    with pytest.raises(ValueError):
        call(torch._efficientzerotensor(tuple(t.shape), device="cuda"))
