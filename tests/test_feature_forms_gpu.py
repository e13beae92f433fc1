"""The kernels' forms for large calls against the definition in fp64: rotary's runs
of heads, and group norm's walks (one launch, and two for strided rows) with every
activation and type.  Tolerances as in test_rotary_gpu.py and test_norm_gpu.py."""

import pytest
import torch

import dot
from tests import util as U
from tests.test_norm_gpu import check, inputs, norm64, strided_rows
from tests.test_rotary_gpu import near, rand, table

pytestmark = pytest.mark.gpu
DEV = "cuda"


# More than 148 * 2048 vectors of pairs: a thread takes four heads in turn, the
# last run of q's or k's heads fewer.
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,L,Hq,Hk,D,P,A", [
    (2, 4001, 5, 3, 80, 32, 3),      # part of a head is turned
    (1, 12007, 12, 3, 80, 32, 2),
    (1, 5003, 1, 9, 128, 64, 1),
    (3, 2501, 6, 7, 48, 20, 2),      # vectors of four in every type
    (1, 9001, 4, 3, 20, 10, 2),      # vectors of two
    (3, 5003, 5, 3, 6, 3, 2),        # single elements
    (1, 9001, 4, 4, 34, 5, 1),       # and a long copied tail
])
def test_runs_of_heads(B, L, Hq, Hk, D, P, A, interleaved, dtype):
    esz = torch.empty(0, dtype=dtype).element_size()
    vp = max(v for v in (1, 2, 4, 16 // esz) if P % v == 0 and D % v == 0)
    slots = P // vp + -(-(-(-(D - 2 * P) // vp)) // 2)
    assert B * L * slots * (Hq + Hk) > 148 * 2048
    q, k = rand(B, L, Hq, D, seed=1, dtype=dtype), rand(B, L, Hk, D, seed=2, dtype=dtype)
    dq, dk = rand(B, L, Hq, D, seed=4, dtype=dtype), rand(B, L, Hk, D, seed=5, dtype=dtype)
    pos, freqs = torch.randint(0, 50000, (B, L, A), generator=U.gen(3)).to(DEV), table(P, A)
    q.requires_grad_(True), k.requires_grad_(True)
    q2, k2 = dot.rotary(q, pos, freqs, k=k, interleaved=interleaved)
    near(q2.detach(), q.detach(), pos, freqs, interleaved)
    near(k2.detach(), k.detach(), pos, freqs, interleaved)
    gq, gk = torch.autograd.grad((q2, k2), (q, k), (dq, dk))
    near(gq, dq, pos, freqs, interleaved, -1.0)
    near(gk, dk, pos, freqs, interleaved, -1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_runs_of_heads_cut_from_wider_rows(dtype):
    """Queries and keys inside a fused projection, and queries alone."""
    wide = rand(1, 7001, 13, 64, seed=1, dtype=dtype)
    pos, freqs = torch.randint(0, 90, (7001, 2), generator=U.gen(3)).to(DEV), table(32, 2)
    q, k = wide[:, :, 1:7], wide[:, :, 7:12]
    q2, k2 = dot.rotary(q, pos, freqs, k=k)
    near(q2, q, pos, freqs)
    near(k2, k, pos, freqs)
    assert torch.equal(dot.rotary(q, pos, freqs), q2)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "relu"])
@pytest.mark.parametrize("C,G", [(64, 8), (48, 24)])      # a vector in one group, and across groups
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
def test_walks(act, C, G, dtype, wdtype, strided):
    N, S = 2, 40001
    x, dy, w, b = inputs(N, S, C, dtype, wdtype, C)
    if act == "relu":   # keep |z| off the kink, where rounding decides the slope
        z = norm64(x.double(), G, w.double(), b.double(), 1e-5, "none")
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    if strided:
        x, dy = strided_rows(x), strided_rows(dy)
    check(x, dy, G, w, b, act)


@pytest.mark.parametrize("act", ["gelu", "relu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_more_samples_than_blocks(act, dtype):
    """One block a sample forwards, two sweeps backwards."""
    x, dy, w, b = inputs(170, 65, 64, dtype, dtype, 3)
    if act == "relu":
        z = norm64(x.double(), 8, w.double(), b.double(), 1e-5, "none")
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    check(x, dy, 8, w, b, act, lengths=[65 - (11 * n) % 66 for n in range(170)])
