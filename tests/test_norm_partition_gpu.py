"""A cooperative launch whose blocks cannot all run at once is told apart from a
failure, before anything ran, so that the forms without a grid barrier can take
the call (as in a context with a part of the device's SMs)."""

import ctypes

import pytest
import torch

import dot
from tests.test_norm_lost_copies_gpu import lib  # noqa: F401

pytestmark = pytest.mark.gpu
C, G = 64, 8


def test_too_many_blocks_for_one_launch(lib):  # noqa: F811
    lib.launch_together.argtypes = [ctypes.c_int] + [ctypes.c_void_p] * 4 + [ctypes.c_int64] * 2

    def call(blocks):
        x = torch.randn(blocks, 1, C, device="cuda").half()
        y, stats = torch.zeros_like(x), torch.zeros(blocks, G, 2, device="cuda")
        ws = torch.empty(max(256, lib.norm_workspace(blocks, 1, C, G)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        rc = lib.launch_together(blocks, x.data_ptr(), y.data_ptr(), stats.data_ptr(), ws.data_ptr(), C, G)
        return rc, x, y

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    rc, x, y = call(2 * sms)       # one block fills an SM's shared memory
    assert rc == 1 and (y == 0).all()
    rc, x, y = call(sms)           # and the next launch is as good as any
    assert rc == 0 and torch.equal(y, dot.group_norm_act(x, G))
