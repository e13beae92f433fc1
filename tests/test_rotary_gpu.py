"""Rotary positions on the GPU, against the definition in fp64.

Tolerances.  An angle is exact to fp64 and rounded to fp32 within one turn:
2 pi 2^-25 = 1.9e-7; sine and cosine add 1 ulp each, the two products and the
sum three roundings of 6e-8: below 1e-6 (|x| + |y|) for a pair, plus one
rounding of the result for 16-bit types.
"""

import pytest
import torch

import dot
from tests import util as U

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # unit roundoffs
TOL = 1e-6


def turn64(x, positions, freqs, interleaved=False, sign=1.0):
    """The definition in fp64 on x [..., H, D]; also |x| + |y| of each element's pair."""
    x = x.double()
    P = freqs.size(0)
    angle = sign * (positions.double()[..., None, :] * freqs.double()).sum(-1)[..., None, :]
    c, s = torch.cos(angle), torch.sin(angle)
    head, rest = x[..., :2 * P], x[..., 2 * P:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :P], head[..., P:])
    u, v, w = a * c - b * s, b * c + a * s, a.abs() + b.abs()
    if interleaved:
        u, w = torch.stack((u, v), -1).flatten(-2), torch.stack((w, w), -1).flatten(-2)
    else:
        u, w = torch.cat((u, v), -1), torch.cat((w, w), -1)
    return torch.cat((u, rest), -1), torch.cat((w, torch.zeros_like(rest)), -1)


def near(got, x, positions, freqs, interleaved=False, sign=1.0):
    want, size = turn64(x, positions, freqs, interleaved, sign)
    bound = TOL * size + UNIT[got.dtype] * want.abs() + 2.0 ** -25 * (got.dtype == torch.float16)
    err = (got.double() - want).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-30)).max())


def table(P, A, seed=0, mixed=False):
    if mixed:
        return torch.randn(P, A, generator=U.gen(seed)).to(DEV)
    share = [P // A + (a < P % A) for a in range(A)]
    return dot.rotary_freqs(share, device=DEV)


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=U.gen(seed)).to(DEV).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,Hq,Hk,D,P,A", [
    (1, 1, 1, 1, 2, 1, 1),
    (8, 1, 32, 8, 128, 64, 3),     # one new token a stream
    (2, 37, 4, 4, 64, 32, 2),
    (1, 301, 12, 3, 80, 32, 3),    # part of a head is turned
    (3, 5, 2, 1, 6, 3, 2),         # vectors of one element
    (2, 11, 3, 3, 20, 10, 4),      # vectors of two
    (1, 9, 5, 2, 24, 4, 1),
    (1, 4, 1, 1, 2048, 1024, 2),   # whole features as one head
    (1, 3, 1, 2, 1030, 257, 1),
    (2, 6, 2, 2, 16, 0, 1),        # nothing turned: a copy
    (70, 33, 1, 1, 32, 16, 2),
])
def test_matches_definition(B, L, Hq, Hk, D, P, A, interleaved, dtype):
    q, k = rand(B, L, Hq, D, seed=1, dtype=dtype), rand(B, L, Hk, D, seed=2, dtype=dtype)
    pos = torch.randint(0, 500, (B, L, A), generator=U.gen(3)).to(DEV)
    freqs = table(P, A) if P else torch.zeros(0, A, device=DEV)
    dq, dk = rand(B, L, Hq, D, seed=4, dtype=dtype), rand(B, L, Hk, D, seed=5, dtype=dtype)
    q.requires_grad_(True), k.requires_grad_(True)
    q2, k2 = dot.rotary(q, pos, freqs, k=k, interleaved=interleaved)
    assert q2.dtype == dtype and q2.shape == q.shape and k2.shape == k.shape and q2.is_contiguous()
    near(q2.detach(), q.detach(), pos, freqs, interleaved)
    near(k2.detach(), k.detach(), pos, freqs, interleaved)
    gq, gk = torch.autograd.grad((q2, k2), (q, k), (dq, dk))
    near(gq, dq, pos, freqs, interleaved, -1.0)
    near(gk, dk, pos, freqs, interleaved, -1.0)


@pytest.mark.parametrize("pdt", [torch.int32, torch.int64, torch.float32])
def test_position_types(pdt):
    q, freqs = rand(2, 50, 3, 32), table(16, 3, mixed=True)
    pos = (torch.rand(2, 50, 3, generator=U.gen(1)) * 90 - 30).to(DEV)
    pos = pos.to(pdt)
    near(dot.rotary(q, pos, freqs), q, pos, freqs)


@pytest.mark.parametrize("first", [10 ** 5, 2 ** 24 + 1, 2 ** 30 + 3])
def test_long_positions_keep_their_angles(first):
    """Integer positions beyond fp32's 24 bits: the fp64 angle is off by 2^30 2^-53 turns at most."""
    q, freqs = rand(1, 64, 2, 64), table(32, 1)
    pos = (first + torch.arange(64, device=DEV))[None, :, None]
    near(dot.rotary(q, pos, freqs), q, pos, freqs)


def test_products_depend_on_differences():
    """q_i . k_j is the same after all positions move together (1e-6 of |q||k| per factor, D/2 pairs)."""
    q, k, freqs = rand(1, 20, 1, 64, seed=1), rand(1, 20, 1, 64, seed=2), table(32, 2)
    pos = torch.randint(0, 40, (1, 20, 2), generator=U.gen(3)).to(DEV)
    scores = []
    for shift in (0, 1234):
        a, b = dot.rotary(q, pos + shift, freqs, k=k)
        scores.append(a[0, :, 0].double() @ b[0, :, 0].double().T)
    size = q[0, :, 0].norm(dim=1)[:, None] * k[0, :, 0].norm(dim=1)[None, :]
    assert ((scores[0] - scores[1]).abs() <= 1e-5 * size).all()


def test_position_layouts():
    q, freqs = rand(3, 40, 2, 32), table(16, 3)
    pos = torch.randint(0, 99, (3, 3, 40), generator=U.gen(4)).to(DEV)
    want = dot.rotary(q, pos.permute(1, 2, 0).contiguous(), freqs)
    assert torch.equal(dot.rotary(q, pos.permute(1, 2, 0), freqs), want)       # axes outermost in memory
    shared = pos[:, 0].T.contiguous()
    want = dot.rotary(q, shared.expand(3, 40, 3).contiguous(), freqs)
    assert torch.equal(dot.rotary(q, shared, freqs), want)                     # [L, A] for every sample
    assert torch.equal(dot.rotary(q, shared.expand(3, 40, 3), freqs), want)
    assert torch.equal(dot.rotary(q[0], shared, freqs), want[0])               # [L, H, D]
    five = q.view(3, 1, 40, 2, 32)
    assert torch.equal(dot.rotary(five, shared, freqs), want.view(3, 1, 40, 2, 32))
    assert torch.equal(dot.rotary(five, shared.expand(3, 1, 40, 3), freqs), want.view(3, 1, 40, 2, 32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["fused", "heads_first", "odd_offset", "last_axis_strided", "every_other"])
def test_layouts(kind, dtype):
    B, L, H, D, P = 2, 45, 4, 48, 20
    q = rand(B, L, H, D, seed=1, dtype=dtype)
    if kind == "fused":
        wide = rand(B, L, 3 * H, D, seed=9, dtype=dtype)
        wide[:, :, H:2 * H] = q
        src = wide[:, :, H:2 * H]
    elif kind == "heads_first":
        src = q.transpose(1, 2).contiguous().transpose(1, 2)
    elif kind == "odd_offset":
        flat = rand(q.numel() + 1, dtype=dtype)
        flat[1:] = q.reshape(-1)
        src = flat[1:].view(B, L, H, D)
    elif kind == "last_axis_strided":
        src = q.transpose(2, 3).contiguous().transpose(2, 3)
    else:
        wide = rand(B, 2 * L, H, D, dtype=dtype)
        wide[:, ::2] = q
        src = wide[:, ::2]
    assert torch.equal(src, q)
    pos, freqs = torch.randint(0, 60, (B, L, 2), generator=U.gen(2)).to(DEV), table(P, 2)
    assert torch.equal(dot.rotary(src, pos, freqs), dot.rotary(q, pos, freqs))
    leaf = q.detach().requires_grad_(True)
    out = dot.rotary(leaf, pos, freqs)
    (g1,) = torch.autograd.grad(out, leaf, src, retain_graph=True)
    (g2,) = torch.autograd.grad(out, leaf, q)
    assert torch.equal(g1, g2)


def test_gradient_of_an_expanded_scalar_and_of_one_output():
    q, k, freqs = rand(2, 30, 4, 32, seed=1), rand(2, 30, 2, 32, seed=2), table(16, 2)
    pos = torch.randint(0, 60, (2, 30, 2), generator=U.gen(2)).to(DEV)
    q.requires_grad_(True), k.requires_grad_(True)
    q2, k2 = dot.rotary(q, pos, freqs, k=k)
    gq, gk = torch.autograd.grad(q2.sum(), (q, k), allow_unused=True, retain_graph=True)
    near(gq, torch.ones_like(q), pos, freqs, sign=-1.0)
    assert gk is None or (gk == 0).all()
    (gk,) = torch.autograd.grad(k2.sum(), k)
    near(gk, torch.ones_like(k), pos, freqs, sign=-1.0)
    only_k = dot.rotary(q.detach(), pos, freqs, k=k)[1]
    (gk2,) = torch.autograd.grad(only_k.sum(), k)
    assert torch.equal(gk, gk2)


def test_gradient_against_differences_and_second_order():
    """The map is linear in q, so differences carry rounding only: u32 |f| sqrt(n) / h."""
    q, freqs = rand(2, 12, 3, 20, seed=1), table(8, 2)
    pos = torch.randint(0, 30, (2, 12, 2), generator=U.gen(2)).to(DEV)
    dy, d = rand(2, 12, 3, 20, seed=3), rand(2, 12, 3, 20, seed=4)
    leaf = q.detach().requires_grad_(True)
    (grad,) = torch.autograd.grad(dot.rotary(leaf, pos, freqs), leaf, dy)
    up, down = (float((dot.rotary(q + s * d, pos, freqs).double() * dy.double()).sum()) for s in (1.0, -1.0))
    want = float((grad.double() * d.double()).sum())
    assert abs((up - down) / 2 - want) <= 1e-5 * float(dy.norm() * (q.norm() + d.norm()))
    # differentiating the gradient in its upstream turns forward again
    g = dy.detach().requires_grad_(True)
    (first,) = torch.autograd.grad(dot.rotary(leaf, pos, freqs), leaf, g, create_graph=True)
    (second,) = torch.autograd.grad(first, g, d)
    near(second, d, pos, freqs)


def test_turning_back_restores():
    q, freqs = rand(2, 30, 4, 32), table(16, 2)
    pos = torch.randint(0, 60, (2, 30, 2), generator=U.gen(2)).to(DEV)
    back = dot.rotary(dot.rotary(q, pos, freqs), -pos, freqs)
    assert (back - q).abs().max() <= 4e-6 * q.abs().max()


def test_nonfinite_values_stay_in_their_pair():
    q, freqs = rand(1, 4, 2, 16), table(6, 2)
    pos = torch.randint(1, 60, (1, 4, 2), generator=U.gen(2)).to(DEV)
    good = dot.rotary(q, pos, freqs)
    q[0, 1, 0, 2] = float("nan")
    q[0, 2, 1, 13] = float("inf")       # beyond the pairs: copied
    got = dot.rotary(q, pos, freqs)
    bad = torch.isnan(got)
    assert bad.sum() == 2 and bad[0, 1, 0, 2] and bad[0, 1, 0, 8]
    assert got[0, 2, 1, 13] == float("inf")
    same = ~bad
    same[0, 2, 1, 13] = False
    assert torch.equal(got[same], good[same])
    # a masked token's position may hold anything: only that token suffers
    fpos = pos.float()
    fpos[0, 3] = float("nan")
    assert torch.equal(dot.rotary(q, fpos, freqs)[0, :3].nan_to_num(), got[0, :3].nan_to_num())


def test_empty_tensors():
    freqs = table(8, 2)
    pos = torch.zeros(0, 2, dtype=torch.int64, device=DEV)
    assert dot.rotary(torch.zeros(0, 3, 16, device=DEV), pos, freqs).shape == (0, 3, 16)
    q = torch.zeros(2, 0, 3, 16, device=DEV, requires_grad=True)
    out = dot.rotary(q, pos, freqs)
    assert torch.autograd.grad(out.sum(), q)[0].shape == q.shape
    none = dot.rotary(torch.zeros(2, 5, 0, 16, device=DEV), torch.zeros(5, 2, device=DEV), freqs)
    assert none.shape == (2, 5, 0, 16)


def test_streams_graphs_and_repeats():
    q, freqs = rand(4, 500, 6, 64), table(32, 2)
    pos = torch.randint(0, 60, (4, 500, 2), generator=U.gen(2)).to(DEV)
    want = dot.rotary(q, pos, freqs)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = dot.rotary(q.clone(), pos, freqs)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dot.rotary(q, pos, freqs)
    pos.add_(7)
    graph.replay()
    assert torch.equal(y, dot.rotary(q, pos, freqs))


def test_offsets_beyond_32_bits():
    L = 600_000
    wide = torch.empty(L, 4096, device=DEV, dtype=torch.bfloat16)   # 2.46e9 elements, 4.9 GB
    q = wide[:, 4032:].unflatten(1, (2, 32))
    q.copy_(torch.randn(L, 2, 32, device=DEV))
    pos, freqs = torch.arange(L, device=DEV)[:, None], table(16, 1)
    got = dot.rotary(q, pos, freqs)
    assert torch.equal(got, dot.rotary(q.contiguous(), pos, freqs))
    del wide, q
    torch.cuda.empty_cache()


def test_module():
    m = dot.Rotary((8, 8), interleaved=True).to(DEV)
    assert m.half().freqs.dtype == torch.float32 and m.freqs.is_cuda
    q, k = rand(2, 30, 4, 32), rand(2, 30, 1, 32, seed=1)
    pos = torch.randint(0, 60, (30, 2), generator=U.gen(2)).to(DEV)
    got, want = m(q, pos, k), dot.rotary(q, pos, m.freqs, k=k, interleaved=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    q, freqs = rand(2, 10, 4, 32), table(16, 2)
    pos = torch.zeros(2, 10, 2, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="D/2"):
        dot.rotary(q, pos, table(17, 2))
    with pytest.raises(ValueError, match="positions"):
        dot.rotary(q, pos[:, :9], freqs)
    with pytest.raises(ValueError, match="positions"):
        dot.rotary(q, pos[..., :1], freqs)
    with pytest.raises(ValueError, match="int32, int64 or float32"):
        dot.rotary(q, pos.double(), freqs)
    with pytest.raises(ValueError, match="device"):
        dot.rotary(q, pos.cpu(), freqs)
    with pytest.raises(ValueError, match="float32"):
        dot.rotary(q, pos, freqs.double())
    with pytest.raises(ValueError, match="axes"):
        dot.rotary(q, torch.zeros(2, 10, 5, device=DEV), torch.zeros(16, 5, device=DEV))
    with pytest.raises(ValueError, match="differentiable"):
        dot.rotary(q, pos, freqs.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="k must have q's shape"):
        dot.rotary(q, pos, freqs, k=rand(2, 10, 4, 30))
    with pytest.raises(ValueError, match="dtype"):
        dot.rotary(q, pos, freqs, k=rand(2, 10, 4, 32, dtype=torch.float16))
    with pytest.raises(NotImplementedError):
        dot.rotary(q.double(), pos, freqs)
    with pytest.raises(ValueError, match="tokens"):
        dot.rotary(q[0, 0], pos, freqs)
    with pytest.raises(NotImplementedError, match="4096"):
        dot.rotary(torch.zeros(1, 1, 8194, device=DEV), torch.zeros(1, 1, device=DEV),
                   torch.zeros(4097, 1, device=DEV))


def test_single_calls_of_the_c_abi():
    """dot_b200.ops.rotary_raw and the public operator are the same call."""
    from dot_b200 import ops

    q, k, freqs = rand(2, 30, 4, 40, seed=1), rand(2, 30, 2, 40, seed=2), table(16, 2)
    pos = torch.randint(0, 60, (30, 2), generator=U.gen(2)).to(DEV)
    want = dot.rotary(q, pos, freqs, k=k)
    got = ops.rotary_raw(q, k, pos.unsqueeze(0), freqs, False)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(ops.rotary_raw(None, k, pos.unsqueeze(0), freqs, False)[1], want[1])


def test_raw_refusals():
    from dot_b200 import ops

    q, pos, freqs = rand(2, 10, 4, 32), torch.zeros(2, 10, 2, device=DEV), table(16, 2)
    for bad in (lambda: ops.rotary_raw(None, None, pos, freqs, False),
                lambda: ops.rotary_raw(q[0], None, pos, freqs, False),
                lambda: ops.rotary_raw(q, q[:, :5], pos, freqs, False),
                lambda: ops.rotary_raw(q, q.half(), pos, freqs, False),
                lambda: ops.rotary_raw(q, None, pos[:, :9], freqs, False),
                lambda: ops.rotary_raw(q, None, pos.double(), freqs, False),
                lambda: ops.rotary_raw(q, None, pos, freqs[:, :1], False),
                lambda: ops.rotary_raw(q, None, pos, table(17, 2), False)):
        with pytest.raises(ValueError):
            bad()
