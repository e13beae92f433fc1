"""Host side of the feature operators (group norm with an activation, rotary
positions): refusals of the Python API and of the C-ABI, frequency tables,
row layouts.  Nothing here needs a GPU."""

import ctypes

import pytest
import torch

import dot
from dot_b200 import _lib, ops

PTR = ctypes.c_void_p(16)   # never read: the checks come first


def test_cpu_tensors_are_rejected():
    with pytest.raises(RuntimeError, match="CUDA"):
        dot.group_norm_act(torch.rand(2, 4, 8), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        dot.rotary(torch.rand(1, 2, 8), torch.zeros(1, 1), torch.zeros(4, 1))


def test_module_arguments():
    with pytest.raises(ValueError, match="num_groups"):
        dot.GroupNormAct(3, 16)
    with pytest.raises(ValueError, match="activation"):
        dot.GroupNormAct(4, 16, activation="tanh")
    m = dot.GroupNormAct(4, 16, affine=False)
    assert m.weight is None and not list(m.parameters())
    with pytest.raises(ValueError, match="16 channels"):
        m(torch.rand(2, 3, 8))
    assert sum(p.numel() for p in dot.GroupNormAct(4, 16).parameters()) == 32


def test_frequency_tables():
    t = dot.rotary_freqs((2, 4), theta=100.0)
    assert t.shape == (6, 2) and t.dtype == torch.float32
    assert torch.allclose(t[:2, 0], torch.tensor([1.0, 0.1])) and (t[:2, 1] == 0).all()
    assert torch.allclose(t[2:, 1], torch.tensor([100.0 ** (-j / 4) for j in range(4)])) and (t[2:, 0] == 0).all()
    t = dot.rotary_freqs((1, 0, 3), theta=16.0, shared_band=True)
    assert torch.allclose(t.sum(1), torch.tensor([16.0 ** (-p / 4) for p in range(4)]))
    assert (t[:, 1] == 0).all() and t[0, 0] == 1 and (t[1:, 2] > 0).all()
    for bad in [(), (1, 2, 3, 4, 5), (-1,)]:
        with pytest.raises(ValueError):
            dot.rotary_freqs(bad)
    with pytest.raises(ValueError):
        dot.rotary_freqs((2,), theta=0.0)


def test_row_layouts_are_read_in_place_where_they_can_be():
    x = torch.rand(3, 4, 5, 8)
    same = lambda t, *want: (t.data_ptr(), *want)  # noqa: E731

    def look(t):
        y, N, S, C, xb, xp = ops._rows(t)
        assert (N, S, C) == (t.size(0), t[0, ..., 0].numel(), t.size(-1))
        flat = y.as_strided((N, S, C), (xb, xp, 1))
        assert torch.equal(flat, t.reshape(N, S, C))
        return y.data_ptr(), xb, xp

    assert look(x) == same(x, 160, 8)
    assert look(x[..., 2:6]) == same(x[..., 2:6], 160, 8)             # a slice of the channels
    assert look(x[:, 1:3]) == same(x[:, 1:3], 160, 8)
    assert look(x[:, :, ::2])[0] != x.data_ptr()                       # positions at two strides: copied
    assert look(x[:, 0, ::2]) == same(x, 160, 16)
    assert look(x.transpose(2, 3))[0] != x.data_ptr()
    assert look(x.transpose(1, 2))[0] != x.data_ptr()
    nchw = torch.rand(2, 8, 4, 5).contiguous(memory_format=torch.channels_last)
    assert look(nchw.permute(0, 2, 3, 1)) == same(nchw, 160, 8)
    assert look(x[:1].expand(3, 4, 5, 8)) == same(x, 0, 8)
    assert look(x[:, :1, :1])[0] == x.data_ptr()


def norm_fwd(**kw):
    a = dict(x=PTR, dtype=0, xb=0, xp=0, w=None, b=None, pdt=0, ln=None, N=1, S=4, C=8, G=2, eps=1e-5, act=1, y=PTR,
             stats=PTR, ws=PTR, nb=1 << 20)
    a.update(kw)
    return _lib.load().dot_group_norm_fwd(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(N=-1), -1, "negative"), (dict(G=0), -1, "num_groups"), (dict(G=3), -1, "num_groups"),
    (dict(G=-2), -1, "num_groups"), (dict(dtype=3), -4, "dtype"), (dict(pdt=9), -4, "dtype"),
    (dict(act=4), -1, "activation"), (dict(act=-1), -1, "activation"), (dict(eps=-1.0), -1, "eps"),
    (dict(eps=float("nan")), -1, "eps"), (dict(eps=float("inf")), -1, "eps"), (dict(x=None), -1, "null"),
    (dict(y=None), -1, "null"), (dict(stats=None), -1, "null"), (dict(S=1 << 31), -4, "large"),
    (dict(ws=None, S=1 << 20), -3, "workspace"), (dict(nb=8, S=1 << 20), -3, "workspace")])
def test_norm_forward_boundary(kw, code, text):
    assert norm_fwd(**kw) == code
    assert text in _lib.load().dot_last_error().decode()


def test_norm_backward_boundary():
    lib = _lib.load()

    def call(x=PTR, dy=PTR, stats=PTR, N=1, S=4, C=8, G=2, ws=PTR, nb=1 << 20, dx=PTR):
        return lib.dot_group_norm_bwd(x, 0, 0, 0, dy, 0, 0, None, None, 0, None, N, S, C, G, 1, stats, dx, None, None,
                                      ws, nb, None)

    assert call(dy=None) == -1 and call(stats=None) == -1 and call(G=3) == -1
    assert call(ws=None, S=1 << 20) == -3
    assert call(dx=None) == 0            # nothing asked for
    assert lib.dot_group_norm_bwd_workspace_bytes(0, 4, 8, 2) == 0
    assert lib.dot_group_norm_fwd_workspace_bytes(4, 0, 8, 2) == 0
    assert norm_fwd(N=0) == 0 and norm_fwd(S=0) == 0 and norm_fwd(C=0) == 0


def rotary(**kw):
    s = (ctypes.c_int64 * 3)(64, 16, 8)
    a = dict(q=PTR, qs=s, hq=2, k=None, ks=None, hk=0, dtype=0, pos=PTR, pdt=4, ps=s, freqs=PTR, B=1, L=4, D=8, P=4,
             A=2, il=0, inv=0, qo=PTR, ko=None)
    a.update(kw)
    return _lib.load().dot_rotary(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(B=-1), -1, "negative"), (dict(P=5), -1, "pairs"), (dict(A=0), -1, "axes"), (dict(A=5), -1, "axes"),
    (dict(dtype=4), -4, "dtype"), (dict(pdt=1), -4, "positions"), (dict(q=None), -1, "null"),
    (dict(qo=None), -1, "null"), (dict(qs=None), -1, "null"), (dict(hk=1), -1, "null"), (dict(pos=None), -1, "null"),
    (dict(freqs=None), -1, "null"), (dict(D=8194, P=4097), -4, "4096"), (dict(L=1 << 31), -4, "large")])
def test_rotary_boundary(kw, code, text):
    assert rotary(**kw) == code
    assert text in _lib.load().dot_last_error().decode()


def test_rotary_of_nothing():
    assert rotary(B=0) == 0 and rotary(L=0) == 0 and rotary(hq=0) == 0


def test_all_kernel_classes_are_reported():
    _lib.prof_begin(False)
    res = _lib.prof_end()
    assert {"norm_fwd", "norm_bwd", "rotary"} <= set(res)
    lib = _lib.load()
    assert lib.dot_prof_end_n(None, None, 12) == -1 and lib.dot_prof_end_n(None, None, -1) == -1
