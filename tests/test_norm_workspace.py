"""Workspace of group norm calls: no more than the form that runs can use."""

import pytest
import torch

from dot_b200 import _lib

SMS = 148


def backward_bytes(N, S, C, G):
    return _lib.load().dot_group_norm_bwd_workspace_bytes(N, S, C, G)


@pytest.mark.parametrize("N,S,C,G", [(262144, 1, 1024, 32), (8192, 1, 4096, 32), (100000, 25, 128, 8),
                                     (149, 7, 64, 4), (4096, 64, 64, 8)])
def test_many_samples_keep_one_row_of_sums_each(N, S, C, G):
    """More samples than SMs: one block a sample, (sum dz, sum dz xh) of its channels and groups."""
    assert backward_bytes(N, S, C, G) <= N * (C + G) * 8 + 1024


@pytest.mark.parametrize("N", [1, 2, 3, 7, 16, 17, 18, 19, 37, 49, 74, 75, 147, 148])
@pytest.mark.parametrize("S", [1, 2, 5, 8, 33, 257, 100000])
def test_what_the_forms_use_fits(N, S):
    """A row of sums for each block of the sweeps, and for each chunk that the resident form may take."""
    C, G = 64, 8
    rows = -(-S // max(1, min(SMS // N, -(-S // 32))))
    sweeps = -(-S // rows)
    resident = max(K for K in range(1, 9) if K == 1 or (N * K <= SMS and K <= S))
    row = (C + G) * 8
    assert N * max(sweeps, resident) * row <= backward_bytes(N, S, C, G) <= N * max(sweeps, resident) * row + 1024


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 16, 18, 37, 74, 148, 149, 1000])
@pytest.mark.parametrize("S", [1, 3, 8, 40])
def test_nothing_is_written_beyond_it(N, S):
    """A backward call in a workspace of exactly that size leaves what follows as it was."""
    lib, C, G = _lib.load(), 48, 6
    gen = torch.Generator("cuda").manual_seed(N + S)
    x, dy = (torch.randn(N, S, C, generator=gen, device="cuda") for _ in range(2))
    y, dx = torch.empty_like(x), torch.empty_like(x)
    w, b = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    dw, db = torch.empty_like(w), torch.empty_like(b)
    stats = torch.empty(N, G, 2, device="cuda")
    fwd, bwd = lib.dot_group_norm_fwd_workspace_bytes(N, S, C, G), backward_bytes(N, S, C, G)
    ws = torch.full((max(fwd, bwd) + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    stream = _lib.raw_stream(0)
    assert lib.dot_group_norm_fwd(x.data_ptr(), 0, S * C, C, w.data_ptr(), b.data_ptr(), 0, None, N, S, C, G, 1e-5, 1,
                                  y.data_ptr(), stats.data_ptr(), ws.data_ptr(), fwd, stream) == 0
    assert (ws[fwd:] == 0xA5).all()
    ws.fill_(0xA5)
    assert lib.dot_group_norm_bwd(x.data_ptr(), 0, S * C, C, dy.data_ptr(), S * C, C, w.data_ptr(), b.data_ptr(), 0,
                                  None, N, S, C, G, 1, stats.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                  ws.data_ptr(), bwd, stream) == 0
    assert (ws[bwd:] == 0xA5).all()
