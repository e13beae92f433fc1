"""Group norm with thousands of groups: beyond the resident form's slabs and the
fused form's 1024, at the sizes where a block's shared memory passes what it
has without asking (44 KB beside the merges) and up to the most it can have.
Tolerances as in test_norm_gpu.py."""

import pytest
import torch

import dot
from tests.test_norm_gpu import check, inputs

pytestmark = pytest.mark.gpu
MOST = 28544   # (227 KB - 4 KB) / 8


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G", [2816, 2817, 3071, 5632, 5633, 6144, 6145, 14272, 14273, 24448, 24449, MOST])
def test_many_groups(G, dtype):
    """Forward and backward take the same numbers of groups."""
    x, dy, w, b = inputs(2, 40, G, dtype, torch.float32, G)
    check(x, dy, G, w, b, "silu")


@pytest.mark.parametrize("G,per", [(2817, 8), (5633, 3), (24449, 8)])
def test_many_groups_of_several_channels(G, per):
    x, dy, w, b = inputs(1, 23, G * per, torch.float16, torch.float16, G)
    check(x, dy, G, w, b, "none")


def test_padded_sets_of_many_groups():
    x, dy, w, b = inputs(3, 40, 5640, torch.float32, torch.float32, 1)
    check(x, dy, 5640, w, b, "silu", lengths=[40, 0, 17])


@pytest.mark.parametrize("grad", [False, True])
def test_more_groups_are_refused_by_the_forward(grad):
    x = torch.randn(1, 4, MOST + 1, device="cuda", requires_grad=grad)
    with pytest.raises(NotImplementedError, match="28544 groups"):
        dot.group_norm_act(x, MOST + 1)
