"""The matcher of examples/dense_matching.py: the feature operators, the scores
and the bidirectional softmax together, forward, backward and trained."""

import importlib.util
import os

import pytest
import torch

import dot

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("dense_matching", os.path.join(ROOT, "examples", "dense_matching.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def plain_encode(m, x, pos, lengths):
    """The encoder from torch operations in fp64."""
    def norm(v, mod, act):
        out = torch.zeros_like(v)
        for n, k in enumerate(lengths.tolist()):
            g = v[n, :k].reshape(k, mod.num_groups, -1)
            mean, var = g.mean(dim=(0, 2), keepdim=True), g.var(dim=(0, 2), keepdim=True, correction=0)
            z = ((g - mean) / torch.sqrt(var + mod.eps)).reshape(k, -1) * mod.weight.double() + mod.bias.double()
            out[n, :k] = torch.nn.functional.silu(z) if act else z
        return out

    lin = lambda v, mod: v @ mod.weight.double().T + mod.bias.double()  # noqa: E731
    v = norm(lin(norm(lin(x.double(), m.inp), m.norm1, True), m.out), m.norm2, False)
    angle = pos.double() @ m.turn.freqs.double().T
    a, b = v.chunk(2, dim=-1)
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), dim=-1)


def test_features_match_fp64():
    ex = example()
    torch.manual_seed(1)
    m = ex.Encoder(32).cuda()
    (d0, p0), _, _, lengths = ex.pairs(4, 64, 32, torch.Generator(device="cuda").manual_seed(2))
    torch.backends.cuda.matmul.allow_tf32 = False
    got, want = m(d0, p0, lengths), plain_encode(m, d0, p0, lengths)
    # two norms and two linear layers in fp32, each a few 1e-6 of its largest value
    assert float((got.double() - want).abs().max()) <= 2e-5 * float(want.abs().max())


def test_padding_does_not_matter():
    ex = example()
    torch.manual_seed(1)
    m = ex.Encoder(32).cuda()
    (d0, p0), (d1, p1), _, lengths = ex.pairs(4, 64, 32, torch.Generator(device="cuda").manual_seed(2))
    P = ex.matching(m(d0, p0, lengths), m(d1, p1, lengths), lengths)
    pad = torch.arange(64, device="cuda") >= lengths[:, None]
    d0, p0 = d0.clone(), p0.clone()
    d0[pad], p0[pad] = 1e4, 777.0
    assert torch.equal(P, ex.matching(m(d0, p0, lengths), m(d1, p1, lengths), lengths))
    assert (P[pad] == 0).all()


def test_it_learns():
    """Descriptors as noisy as they differ, positions shifted: the encoder has to learn both."""
    losses = example().train(steps=240, seed=3)
    assert sum(losses[-10:]) / 10 < 0.6 * sum(losses[:3]) / 3


def test_counted_launches():
    from dot_b200 import _lib

    ex = example()
    m = ex.Encoder(32).cuda()
    (d0, p0), _, _, lengths = ex.pairs(2, 64, 32, torch.Generator(device="cuda").manual_seed(2))
    _lib.prof_begin(False)
    m(d0, p0, lengths).sum().backward()
    n = _lib.prof_end()
    assert n["norm_fwd"]["launches"] == 2 and n["rotary"]["launches"] == 2 and n["norm_bwd"]["launches"] >= 2
    assert dot.rotary is not None
