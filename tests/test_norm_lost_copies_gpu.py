"""A ring copy of the fused group norm that never arrives: the bounded wait runs
out, the kernel returns and every output that depends on the copy is NaN, in all
channels; what does not is as it was."""

import ctypes
import os
import subprocess

import pytest
import torch

import dot
from dot_b200 import build, ops
from tests import util as U

pytestmark = pytest.mark.gpu
DEV = "cuda"
SMS, C = 148, 64
ROWS = 2048           # positions of a block: 8 stages of 256 forwards, 16 of 128 backwards, 5 in the ring
S = SMS * ROWS


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("lost") / "lost_copies.so")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lost_copies.cu")
    subprocess.run([build._nvcc(), build.ARCH, "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-Xcompiler",
                    "-fvisibility=hidden", "--expt-relaxed-constexpr", "-cudart", "static", src, "-o", so], check=True)
    handle = ctypes.CDLL(so)
    handle.norm_workspace.restype = ctypes.c_size_t
    handle.norm_workspace.argtypes = [ctypes.c_int64] * 4
    handle.norm_losing.argtypes = [ctypes.c_int] * 3 + [ctypes.c_void_p] * 10 + [ctypes.c_int64] * 4
    return handle


@pytest.fixture(params=[8, 4], ids=["group_of_8", "group_of_4"])
def case(request):
    """Inputs and what the library computes from them; groups of whole vectors and of half ones."""
    G = C // request.param
    x, dy = (torch.randn(1, S, C, generator=torch.Generator(DEV).manual_seed(k), device=DEV).half() for k in (1, 2))
    w, b = (torch.randn(C, generator=U.gen(k)).to(DEV) for k in (3, 4))
    y, stats = ops.group_norm_forward_raw(x, G, w, b, 1e-5, 1)
    dx, dw, db = ops.group_norm_backward_raw(x, dy, G, w, b, 1, stats)
    return G, x, dy, w, b, stats, y, dx, dw, db


def run(lib, case, stage, back, backward):
    G, x, dy, w, b, stats = case[:6]
    y, dx, dw, db = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    st = stats[:2 * G].clone() if backward else torch.zeros(2 * G, device=DEV)
    ws = torch.empty(lib.norm_workspace(1, S, C, G), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    pointers = (t.data_ptr() for t in (x, dy, w, b, y, dx, dw, db, st, ws))
    rc = lib.norm_losing(stage, back, backward, *pointers, 1, S, C, G)
    assert rc == 0, rc
    return (dx, dw, db) if backward else (y, st)


def test_nothing_lost(lib, case):
    y, st = run(lib, case, -1, 0, 0)
    assert torch.equal(y, case[6]) and torch.equal(st, case[5][:st.numel()])
    for got, want in zip(run(lib, case, -1, 0, 1), case[7:]):
        assert torch.equal(got, want)


@pytest.mark.parametrize("stage", [3, 6])
def test_lost_on_the_way_in(lib, case, stage):
    """Stages of the first filling and of the second; every block loses one, so every sum does."""
    y, st = run(lib, case, stage, 0, 0)
    assert y.isnan().all() and st.isnan().all()
    for t in run(lib, case, stage, 0, 1):
        assert t.isnan().all()
    assert torch.equal(run(lib, case, -1, 0, 0)[0], case[6])   # the device is as usable as before


def test_lost_on_the_way_back(lib, case):
    """The last stage of the walk: its rows are NaN, everything else is there."""
    y, st = run(lib, case, 0, 1, 0)
    rows, want = y.view(SMS, ROWS, C), case[6].view(SMS, ROWS, C)
    assert rows[:, :256].isnan().all() and torch.equal(rows[:, 256:], want[:, 256:])
    assert torch.equal(st, case[5][:st.numel()])
    dx, dw, db = run(lib, case, 0, 1, 1)
    rows, want = dx.view(SMS, ROWS, C), case[7].view(SMS, ROWS, C)
    assert rows[:, :128].isnan().all() and torch.equal(rows[:, 128:], want[:, 128:])
    assert torch.equal(dw, case[8]) and torch.equal(db, case[9])


def test_lost_amid_the_way_back(lib, case):
    """No thread trusts a stage after it: its rows and those of the stages below are NaN."""
    y, _ = run(lib, case, 2, 1, 0)
    rows, want = y.view(SMS, ROWS, C), case[6].view(SMS, ROWS, C)
    assert rows[:, :3 * 256].isnan().all() and torch.equal(rows[:, 3 * 256:], want[:, 3 * 256:])
