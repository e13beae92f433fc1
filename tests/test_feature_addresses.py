"""Addresses that the feature operators' kernels could not read: the C-ABI refuses
them before any launch (no GPU needed), and so do the raw calls."""

import ctypes

import pytest
import torch

from dot_b200 import _lib, ops

GOOD = 64   # never read: the checks come first


def text():
    return _lib.load().dot_last_error().decode()


def norm_fwd(dtype=0, pdt=0, **at):
    p = {k: ctypes.c_void_p(at.get(k, GOOD)) for k in ("x", "w", "b", "ln", "y", "stats", "ws")}
    return _lib.load().dot_group_norm_fwd(p["x"], dtype, 32, 8, p["w"], p["b"], pdt, p["ln"], 1, 4, 8, 2, 1e-5, 1,
                                          p["y"], p["stats"], p["ws"], 1 << 20, None)


def norm_bwd(dtype=0, pdt=0, **at):
    p = {k: ctypes.c_void_p(at.get(k, GOOD)) for k in ("x", "dy", "w", "b", "ln", "stats", "dx", "dw", "db", "ws")}
    return _lib.load().dot_group_norm_bwd(p["x"], dtype, 32, 8, p["dy"], 32, 8, p["w"], p["b"], pdt, p["ln"], 1, 4, 8,
                                          2, 1, p["stats"], p["dx"], p["dw"], p["db"], p["ws"], 1 << 20, None)


@pytest.mark.parametrize("call", [norm_fwd, norm_bwd])
@pytest.mark.parametrize("which", ["stats", "ws"])
@pytest.mark.parametrize("off", [1, 2, 4, 7])
def test_statistics_and_workspace_are_read_in_pairs(call, which, off):
    assert call(**{which: GOOD + off}) == -1
    assert "8-byte aligned" in text()


@pytest.mark.parametrize("dtype,pdt,off", [(0, 1, 2), (1, 0, 1), (2, 2, 1)])
def test_norm_tensors_start_at_an_element(dtype, pdt, off):
    for call, names in ((norm_fwd, ("x", "y")), (norm_bwd, ("x", "dy", "dx"))):
        for name in names:
            assert call(dtype=dtype, pdt=pdt, **{name: GOOD + off}) == -1 and "elements" in text()
    for call, names in ((norm_fwd, ("w", "b")), (norm_bwd, ("w", "b", "dw", "db"))):
        for name in names:
            assert call(dtype=dtype, pdt=pdt, **{name: GOOD + (2 if pdt == 0 else 1)}) == -1 and "elements" in text()
    assert norm_fwd(ln=GOOD + 2) == -1 and norm_bwd(ln=GOOD + 2) == -1


def rotary(dtype=0, pdt=4, **at):
    s = (ctypes.c_int64 * 3)(64, 16, 8)
    p = {k: ctypes.c_void_p(at.get(k, GOOD)) for k in ("q", "k", "pos", "freqs", "qo", "ko")}
    return _lib.load().dot_rotary(p["q"], s, 2, p["k"], s, 2, dtype, p["pos"], pdt, s, p["freqs"], 1, 4, 8, 4, 2, 0, 0,
                                  p["qo"], p["ko"], None)


@pytest.mark.parametrize("name", ["q", "k", "qo", "ko"])
@pytest.mark.parametrize("dtype,off", [(0, 2), (1, 1), (2, 1)])
def test_rotary_tensors_start_at_an_element(name, dtype, off):
    assert rotary(dtype=dtype, **{name: GOOD + off}) == -1 and "elements" in text()


@pytest.mark.parametrize("pdt,off", [(0, 2), (3, 2), (4, 4)])
def test_positions_start_at_an_element(pdt, off):
    assert rotary(pdt=pdt, pos=GOOD + off) == -1 and "elements" in text()
    assert rotary(freqs=GOOD + 2) == -1 and "elements" in text()


@pytest.mark.gpu
def test_raw_statistics():
    x = torch.randn(2, 10, 32, device="cuda")
    y, stats = ops.group_norm_forward_raw(x, 4, None, None, 1e-5, 1)
    odd = torch.zeros(stats.numel() + 1, device="cuda")[1:]
    for bad in (stats.cpu(), odd):
        with pytest.raises(ValueError):
            ops.group_norm_backward_raw(x, y, 4, None, None, 1, bad)
