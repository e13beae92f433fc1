"""Group norm with an activation on the GPU, against the definition in fp64.

Tolerances.  u is a type's unit roundoff (2^-24, 2^-8, 2^-11 for float32,
bfloat16, float16).  A forward value is a subtraction, a product, an fma and
the activation on statistics whose own error is a few tens of u32 (merges of
up to ~30 levels), the exponential adding 1e-6: 5e-6 of the sample's largest
value, plus one rounding u of the value itself for 16-bit outputs.  dx adds
two group sums of the same kind.  A parameter's gradient is a sum of n terms,
at most ~100 in one thread and then trees: 1e-5 of the sum of the terms'
magnitudes, plus one rounding.  A sigmoid or a normal density below float32's
smallest normal number 2^-126 becomes 0, and z times it with it: 300 * 2^-126
for the largest |z| here.
"""

import pytest
import torch

import dot
from tests import util as U

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {dt: torch.finfo(dt).eps / 2 for dt in (torch.float32, torch.bfloat16, torch.float16)}
FWD = 5e-6
SUM = 1e-5


def act64(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z.relu() if act == "relu" else z


def norm64(x, G, w, b, eps, act, lengths=None):
    """The definition in fp64 on x [N, S, C], sample by sample, group by group."""
    N, S, C = x.shape
    rows = []
    for n in range(N):
        k = S if lengths is None else int(lengths[n])
        if k == 0:
            rows.append(0 * torch.zeros(S, C, dtype=torch.float64, device=x.device) * (1 if w is None else w + b)
                        + 0 * x[n, :0].sum())
            continue
        v = x[n, :k].reshape(k, G, C // G)
        mean = v.mean(dim=(0, 2), keepdim=True)
        var = ((v - mean) ** 2).mean(dim=(0, 2), keepdim=True)
        z = ((v - mean) / torch.sqrt(var + eps)).reshape(k, C)
        if w is not None:
            z = z * w
        if b is not None:
            z = z + b
        rows.append(torch.nn.functional.pad(act64(z, act), (0, 0, 0, S - k)))
    return torch.stack(rows)


def near(actual, expected, scale, rtol, what):
    """|actual - expected| <= rtol * scale + one rounding of the expected value in actual's type."""
    u = UNIT[actual.dtype] if actual.dtype != torch.float32 else 0.0
    bound = rtol * scale + u * expected.abs() + 2.0 ** -25 * (actual.dtype == torch.float16) + 300 * 2.0 ** -126
    bad = ~((actual.double() - expected).abs() <= bound)
    assert not bad.any(), (what, float(((actual.double() - expected).abs() / bound).max()), int(bad.sum()))


def inputs(N, S, C, dtype, wdtype, seed, affine=True, offset=1.0):
    g = U.gen(seed)
    x = torch.randn(N, S, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + offset * torch.randn(C, generator=g)
    dy = torch.randn(N, S, C, generator=g)
    w = (1 + 0.3 * torch.randn(C, generator=g)) if affine else None
    b = 0.3 * torch.randn(C, generator=g) if affine else None
    put = lambda t, d: None if t is None else t.to(DEV).to(d)  # noqa: E731
    return put(x, dtype), put(dy, dtype), put(w, wdtype), put(b, wdtype)


def check(x, dy, G, w, b, act, lengths=None, eps=1e-5, fwd=FWD):
    """Forward and all gradients of one call against fp64."""
    leaf = lambda t: None if t is None else t.detach().requires_grad_(True)  # noqa: E731
    xs, ws, bs = leaf(x), leaf(w), leaf(b)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    y = dot.group_norm_act(xs, G, ws, bs, eps=eps, activation=act, lengths=ln)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(y, dot.group_norm_act(xs, G, ws, bs, eps=eps, activation=act, lengths=ln))
    wanted = [t for t in (xs, ws, bs) if t is not None]
    grads = torch.autograd.grad(y, wanted, dy)

    x64, w64, b64 = (None if t is None else t.detach().double().requires_grad_(True) for t in (x, w, b))
    y64 = norm64(x64, G, w64, b64, eps, act, lengths)
    grads64 = torch.autograd.grad(y64, [t for t in (x64, w64, b64) if t is not None], dy.double())
    top = lambda t: t.detach().abs().amax(dim=(1, 2), keepdim=True)  # noqa: E731
    near(y.detach(), y64.detach(), top(y64), fwd, "y")
    near(grads[0], grads64[0], top(grads64[0]), 2 * fwd, "dx")
    if w is not None:
        # terms of the parameters' sums, from the same chain with weight and bias per element
        ones = torch.ones_like(x64)
        we, be = (ones * w64.detach()).requires_grad_(True), (ones * b64.detach()).requires_grad_(True)
        te = torch.autograd.grad(norm64_elementwise(x64.detach(), G, we, be, eps, act, lengths), (we, be), dy.double())
        near(grads[1], grads64[1], te[0].abs().sum(dim=(0, 1)), SUM, "dweight")
        near(grads[2], grads64[2], te[1].abs().sum(dim=(0, 1)), SUM, "dbias")
        assert grads[1].dtype == w.dtype and grads[2].dtype == b.dtype
    if lengths is not None:
        for n, k in enumerate(lengths):
            assert (y[n, k:] == 0).all() and (grads[0][n, k:] == 0).all()
    return y, grads


def norm64_elementwise(x, G, w, b, eps, act, lengths):
    """norm64 with a weight and a bias for every element."""
    xh = norm64(x, G, None, None, eps, "none", lengths)
    y = act64(xh * w + b, act)
    if lengths is None:
        return y
    valid = torch.arange(x.size(1), device=x.device)[None, :] < torch.tensor(lengths, device=x.device)[:, None]
    return y * valid[..., None]


@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("N,S,C,G", [
    (1, 1, 1, 1),           # one value: its own mean
    (2, 1, 64, 8),          # one position
    (3, 7, 30, 10),         # three channels a group, narrow vectors
    (1, 257, 15, 5),        # single elements
    (2, 1961, 90, 6),       # groups across vectors
    (1, 4800, 256, 32),
    (5, 333, 24, 1),        # one group over all channels
    (2, 100, 40, 40),       # a channel a group
    (1, 9, 2056, 4),        # more channel vectors than a block has threads in float32
    (2, 65, 4112, 2),       # a group wider than a block's tile
    (40, 33, 16, 2),
])
def test_matches_definition(N, S, C, G, dtype, wdtype):
    x, dy, w, b = inputs(N, S, C, dtype, wdtype, N * 1000 + S + C)
    check(x, dy, G, w, b, "silu")


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "relu"])
@pytest.mark.parametrize("C,G", [(64, 8), (27, 9)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_activations(act, C, G, dtype):
    x, dy, w, b = inputs(2, 311, C, dtype, torch.float32, 5)
    if act == "relu":   # keep |z| off the kink, where rounding decides the slope
        z = norm64(x.double(), G, w.double(), b.double(), 1e-5, "none")
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    check(x, dy, G, w, b, act)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "none"])
def test_activation_extremes(act):
    """Far out on either side the activations keep their limits and stay finite."""
    z = torch.tensor([-300.0, -100.0, -89.0, -20.0, -5.0, 0.0, 5.0, 20.0, 89.0, 100.0, 300.0, 0.0], device=DEV)
    x = torch.stack([torch.ones(12, device=DEV), -torch.ones(12, device=DEV)]).reshape(1, 2, 12)   # xh = +-1
    w, b = torch.zeros(12, device=DEV), z.clone()
    check(x, torch.ones_like(x), 1, w, b, act, eps=0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("C,G", [(256, 32), (90, 6), (36, 4)])
def test_lengths(C, G, dtype):
    """Padded samples: an empty one, a single position, lengths around a chunk's ends; whatever the padding
    holds is not read."""
    S = 1024
    lengths = [1024, 0, 1, 31, 32, 33, 500, 1023]
    x, dy, w, b = inputs(len(lengths), S, C, dtype, torch.float32, 9)
    junk = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min], device=DEV).to(dtype)
    clean = check(x, dy, G, w, b, "silu", lengths)
    for n, k in enumerate(lengths):
        if k < S:
            fill = junk[torch.arange((S - k) * C, device=DEV) % 4].reshape(S - k, C)
            x[n, k:], dy[n, k:] = fill, fill.flip(0)
    ln = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    xs, ws, bs = x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = dot.group_norm_act(xs, G, ws, bs, lengths=ln)
    grads = torch.autograd.grad(y, (xs, ws, bs), dy)
    assert torch.equal(y, clean[0])
    for got, want in zip(grads, clean[1]):
        assert torch.equal(got, want)


def test_lengths_are_clamped():
    x, dy, w, b = inputs(3, 50, 32, torch.float32, torch.float32, 2)
    y = dot.group_norm_act(x, 4, w, b, lengths=torch.tensor([60, -3, 50], dtype=torch.int32, device=DEV))
    want = dot.group_norm_act(x, 4, w, b, lengths=torch.tensor([50, 0, 50], dtype=torch.int32, device=DEV))
    assert torch.equal(y, want)


def test_all_samples_empty():
    x, dy, w, b = inputs(3, 50, 32, torch.float32, torch.float32, 2)
    check(x, dy, 4, w, b, "silu", lengths=[0, 0, 0])


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
def test_without_parameters(weight, bias):
    x, dy, w, b = inputs(2, 77, 48, torch.float32, torch.float32, 3)
    xs = x.requires_grad_(True)
    y = dot.group_norm_act(xs, 6, w if weight else None, b if bias else None)
    (dx,) = torch.autograd.grad(y, xs, dy)
    x64 = x.detach().double().requires_grad_(True)
    y64 = norm64(x64, 6, w.double() if weight else None, b.double() if bias else None, 1e-5, "silu")
    (dx64,) = torch.autograd.grad(y64, x64, dy.double())
    U.assert_normwise(y, y64.detach().cpu(), FWD, "y")
    U.assert_normwise(dx, dx64.cpu(), 2 * FWD, "dx")


def test_gradients_on_their_own():
    """Only what is asked for is computed, with the same values."""
    x, dy, w, b = inputs(2, 500, 64, torch.float32, torch.float32, 4)
    full = check(x, dy, 8, w, b, "silu")[1]
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == k) for k, t in enumerate((x, w, b))]
        y = dot.group_norm_act(leaves[0], 8, leaves[1], leaves[2])
        (got,) = torch.autograd.grad(y, leaves[i], dy)
        assert torch.equal(got, full[i])


def test_mean_far_from_zero():
    """x around 4096 with a spread of 1: the stored fp32 mean is off by up to 4096 u32 = 2.4e-4 of the spread."""
    g = U.gen(1)
    x = (4096 + torch.randn(2, 3000, 64, generator=g)).to(DEV)
    y = dot.group_norm_act(x, 8, activation="none")
    want = norm64(x.double(), 8, None, None, 1e-5, "none")
    assert float((y.double() - want).abs().max()) <= 2.5e-4 + 5e-6 * float(want.abs().max())


def test_constant_group():
    """Variance zero: z is the bias, the gradient finite."""
    x = torch.full((2, 100, 32), 3.25, device=DEV)
    b = torch.linspace(-1, 1, 32, device=DEV)
    y = dot.group_norm_act(x, 4, torch.ones(32, device=DEV), b, activation="none")
    assert torch.allclose(y, b.expand_as(y), atol=1e-6)


def test_nonfinite_values_stay_in_their_group():
    x, dy, w, b = inputs(2, 200, 32, torch.float32, torch.float32, 6)
    good = dot.group_norm_act(x, 4, w, b)
    x[1, 50, 9] = float("inf")
    x[0, 10, 31] = float("nan")
    y = dot.group_norm_act(x, 4, w, b)
    assert torch.isnan(y[1, :, 8:16]).all() and torch.isnan(y[0, :, 24:]).all()
    assert torch.equal(y[1, :, :8], good[1, :, :8]) and torch.equal(y[1, :, 16:], good[1, :, 16:])
    assert torch.equal(y[0, :, :24], good[0, :, :24])


def strided(kind, x):
    """The same values in another memory layout."""
    N, S, C = x.shape
    if kind == "channel_slice":
        wide = torch.full((N, S, 2 * C + 8), 7.0, device=DEV, dtype=x.dtype)
        wide[..., 8:8 + C] = x
        return wide[..., 8:8 + C]
    if kind == "every_other_position":
        wide = torch.full((N, 2 * S, C), 7.0, device=DEV, dtype=x.dtype)
        wide[:, ::2] = x
        return wide[:, ::2]
    if kind == "odd_offset":
        flat = torch.full((x.numel() + 1,), 7.0, device=DEV, dtype=x.dtype)
        flat[1:] = x.reshape(-1)
        return flat[1:].view(N, S, C)
    if kind == "channels_first":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if kind == "batch_inside":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    assert kind == "flipped_memory"
    return x.permute(2, 1, 0).contiguous().permute(2, 1, 0)


@pytest.mark.parametrize("kind", ["channel_slice", "every_other_position", "odd_offset", "channels_first",
                                  "batch_inside", "flipped_memory"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(kind, dtype):
    x, dy, w, b = inputs(3, 130, 40, dtype, torch.float32, 8)
    xs, gs = strided(kind, x), strided(kind, dy)
    assert torch.equal(xs, x)
    check(xs, gs, 5, w, b, "silu")


def test_image_views_and_more_axes():
    """[N, C, H, W] in channels-last memory as a view; [N, T, H, W, C]; a gradient that is an expanded scalar."""
    g = U.gen(3)
    img = torch.randn(2, 32, 9, 11, generator=g).to(DEV).contiguous(memory_format=torch.channels_last)
    y = dot.group_norm_act(img.permute(0, 2, 3, 1), 4, activation="silu")
    want = norm64(img.permute(0, 2, 3, 1).reshape(2, 99, 32).double(), 4, None, None, 1e-5, "silu")
    U.assert_normwise(y.reshape(2, 99, 32), want.cpu(), FWD, "image")
    clip = torch.randn(2, 3, 5, 7, 16, generator=g).to(DEV).requires_grad_(True)
    y = dot.group_norm_act(clip, 2)
    y.sum().backward()
    c64 = clip.detach().double().reshape(2, 105, 16).requires_grad_(True)
    norm64(c64, 2, None, None, 1e-5, "silu").sum().backward()
    U.assert_normwise(clip.grad.reshape(2, 105, 16), c64.grad.cpu(), 2 * FWD, "clip")
    sliced = torch.randn(2, 6, 8, 16, generator=g).to(DEV)[:, 1:5, 2:7]   # positions at two strides: copied
    y = dot.group_norm_act(sliced, 2)
    assert torch.equal(y, dot.group_norm_act(sliced.contiguous(), 2))
    assert dot.group_norm_act(torch.randn(4, 16, device=DEV), 2).shape == (4, 16)


def test_empty_tensors():
    w = torch.ones(16, device=DEV, requires_grad=True)
    for shape in [(0, 5, 16), (3, 0, 16), (2, 0, 4, 16)]:
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        y = dot.group_norm_act(x, 4, w, torch.zeros(16, device=DEV))
        assert y.shape == shape
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == shape and (dw == 0).all()
    assert dot.group_norm_act(torch.zeros(2, 3, 0, device=DEV), 1).shape == (2, 3, 0)


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
def test_gradient_against_differences(which):
    """Central differences of the kernel's own forward along random directions.  Step h: truncation
    h^2 |f'''| / 6 is below 2e-3 of the slope's scale, rounding sqrt(n) u32 |f| / h below 1e-3 of it."""
    x, dy, w, b = inputs(2, 40, 24, torch.float32, torch.float32, 12)
    vals = {"x": x, "weight": w, "bias": b}
    leaves = {k: v.detach().requires_grad_(True) for k, v in vals.items()}
    call = lambda v: dot.group_norm_act(v["x"], 3, v["weight"], v["bias"], activation="gelu")  # noqa: E731
    grad = torch.autograd.grad(call(leaves), leaves[which], dy)[0].double()
    h = 0.02
    for seed in range(3):
        d = torch.randn(vals[which].shape, generator=U.gen(seed)).to(DEV)
        d = d / d.abs().max()
        loss = []
        for sign in (1.0, -1.0):
            v = dict(vals, **{which: vals[which] + sign * h * d})
            loss.append(float((call(v).double() * dy.double()).sum()))
        slope, want = (loss[0] - loss[1]) / (2 * h), float((grad * d.double()).sum())
        scale = float(grad.norm() * d.double().norm())
        assert abs(slope - want) <= 3e-3 * scale, (slope, want, scale)


def test_repeats_bit_for_bit():
    x, dy, w, b = inputs(3, 5000, 96, torch.bfloat16, torch.float32, 13)
    outs = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = dot.group_norm_act(leaves[0], 8, leaves[1], leaves[2])
        outs.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_on_a_side_stream():
    x, dy, w, b = inputs(2, 3000, 64, torch.float32, torch.float32, 14)
    want = dot.group_norm_act(x, 8, w, b)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x2 = x.clone()
        got = dot.group_norm_act(x2, 8, w, b)
    s.synchronize()
    assert torch.equal(got, want)


def test_in_a_graph():
    x, dy, w, b = inputs(2, 700, 64, torch.float32, torch.float32, 15)
    dot.group_norm_act(x, 8, w, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dot.group_norm_act(x, 8, w, b)
    x.mul_(1.5).add_(0.25)
    graph.replay()
    assert torch.equal(y, dot.group_norm_act(x, 8, w, b))


def test_module_matches_function():
    m = dot.GroupNormAct(4, 32, activation="gelu").to(DEV)
    with torch.no_grad():
        m.weight.uniform_(0.5, 1.5)
        m.bias.uniform_(-1, 1)
    x = torch.randn(2, 60, 32, device=DEV)
    m(x).square().sum().backward()
    assert m.weight.grad is not None and m.bias.grad is not None
    assert torch.equal(m(x), dot.group_norm_act(x, 4, m.weight, m.bias, activation="gelu"))
    ln = torch.tensor([60, 7], dtype=torch.int32, device=DEV)
    assert torch.equal(m(x, ln), dot.group_norm_act(x, 4, m.weight, m.bias, activation="gelu", lengths=ln))
    assert dot.GroupNormAct(4, 32, affine=False)(x).shape == x.shape


def test_offsets_beyond_32_bits():
    """A sample whose rows lie 2^31 elements apart in memory is read and written at 64-bit addresses."""
    rows = 600_000
    wide = torch.empty(rows, 4096, device=DEV, dtype=torch.bfloat16)   # 2.46e9 elements, 4.9 GB
    x = wide[:, 4064:]
    x.copy_(torch.randn(rows, 32, device=DEV))
    got = dot.group_norm_act(x.unsqueeze(0), 4)
    want = dot.group_norm_act(x.contiguous().unsqueeze(0), 4)
    assert torch.equal(got, want)
    del wide, x
    torch.cuda.empty_cache()


def test_refusals():
    x = torch.randn(2, 10, 32, device=DEV)
    w = torch.ones(32, device=DEV)
    with pytest.raises(ValueError, match="num_groups"):
        dot.group_norm_act(x, 5)
    with pytest.raises(ValueError, match="num_groups"):
        dot.group_norm_act(x, 0)
    with pytest.raises(ValueError, match="weight"):
        dot.group_norm_act(x, 4, w[:16])
    with pytest.raises(ValueError, match="bias must be on"):
        dot.group_norm_act(x, 4, w, w.cpu())
    with pytest.raises(ValueError, match="eps"):
        dot.group_norm_act(x, 4, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        dot.group_norm_act(x, 4, eps=float("nan"))
    with pytest.raises(ValueError, match="activation"):
        dot.group_norm_act(x, 4, activation="swish")
    with pytest.raises(ValueError, match="lengths must be int32"):
        dot.group_norm_act(x, 4, lengths=torch.tensor([1, 2], device=DEV))
    with pytest.raises(ValueError, match="lengths"):
        dot.group_norm_act(x, 4, lengths=torch.tensor([1], dtype=torch.int32, device=DEV))
    with pytest.raises(NotImplementedError):
        dot.group_norm_act(x.double(), 4)
    with pytest.raises(ValueError):
        dot.group_norm_act(x[0, 0], 4)
    with pytest.raises(RuntimeError):   # once differentiable
        y = dot.group_norm_act(x.requires_grad_(True), 4)
        (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("shape,expand", [((2, 5, 1, 16), (2, 5, 7, 16)), ((2, 1, 7, 16), (2, 5, 7, 16)),
                                          ((1, 5, 7, 16), (2, 5, 7, 16)), ((2, 1, 1, 16), (2, 5, 7, 16)),
                                          ((2, 5, 7, 1), (2, 5, 7, 16))])
def test_expanded_axes(shape, expand):
    """Inputs and gradients repeated along some axes (strides of 0) give what their copies give."""
    x, g = (torch.randn(shape, generator=U.gen(k)).to(DEV).expand(expand) for k in (1, 2))
    outs = []
    for a, b in ((x, g), (x.contiguous(), g.contiguous())):
        leaf = a.detach().requires_grad_(True)
        y = dot.group_norm_act(leaf, 4)
        outs.append((y.detach(), torch.autograd.grad(y, leaf, b)[0]))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("shape", [(2, 5000, 64), (1, 30, 24), (2, 4, 9, 15)])
def test_single_calls_of_the_c_abi(shape):
    """dot_b200.ops' raw functions and the public operator are the same calls."""
    from dot_b200 import ops

    x, dy = (torch.randn(shape, generator=U.gen(k)).to(DEV) for k in (1, 2))
    w, b = (torch.randn(shape[-1], generator=U.gen(k)).to(DEV) for k in (3, 4))
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = dot.group_norm_act(leaves[0], 1, leaves[1], leaves[2], activation="gelu")
    grads = torch.autograd.grad(y, leaves, dy)
    y2, stats = ops.group_norm_forward_raw(x, 1, w, b, 1e-5, 2)
    assert torch.equal(y, y2)
    for got, want in zip(ops.group_norm_backward_raw(x, dy, 1, w, b, 2, stats), grads):
        assert torch.equal(got, want)


def test_a_recorded_backward_is_not_differentiated_again():
    x = torch.randn(2, 10, 16, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(dot.group_norm_act(x, 4).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once differentiable"):
        (g.sum() + x.sum()).backward()


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,S,C,G,lengths", [
    (2, 40000, 64, 8, None),               # a vector in one group
    (1, 60001, 48, 24, None),              # groups across vectors, an odd end
    (3, 30011, 64, 4, [30011, 0, 17]),     # empty and nearly empty chunks
    (5, 17000, 40, 5, [1, 16999, 4096, 0, 8000]),
    (200, 65, 128, 32, None),              # more samples than SMs
    (149, 1, 512, 2, None),
    (1, 9000, 1024, 8, None),
    (160, 40, 24, 3, [40 - (7 * n) % 41 for n in range(160)]),
])
def test_beyond_one_cluster(N, S, C, G, lengths, dtype, strided):
    """Sizes that no cluster's registers hold, rows one after another and rows cut from wider ones."""
    x, dy, w, b = inputs(N, S, C, dtype, torch.float32, N + S)
    if strided:
        x, dy = strided_rows(x), strided_rows(dy)
    y, grads = check(x, dy, G, w, b, "silu", lengths)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    again = dot.group_norm_act(leaves[0], G, leaves[1], leaves[2], lengths=ln)
    assert torch.equal(again, y)
    for got, want in zip(torch.autograd.grad(again, leaves, dy), grads):
        assert torch.equal(got, want)


def strided_rows(x):
    wide = torch.full((*x.shape[:2], x.size(2) + 16), 7.0, device=DEV, dtype=x.dtype)
    wide[..., 8:8 + x.size(2)] = x
    return wide[..., 8:8 + x.size(2)]


def test_a_large_call_in_a_graph():
    x, dy, w, b = inputs(2, 30000, 64, torch.bfloat16, torch.float32, 15)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    torch.autograd.grad(dot.group_norm_act(leaves[0], 8, leaves[1], leaves[2]), leaves, dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dot.group_norm_act(leaves[0], 8, leaves[1], leaves[2])
        grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        x.mul_(1.5).add_(0.25)
    for _ in range(2):
        graph.replay()
    want = dot.group_norm_act(leaves[0], 8, leaves[1], leaves[2])
    assert torch.equal(y, want)
    for got, ref in zip(grads, torch.autograd.grad(want, leaves, dy)):
        assert torch.equal(got, ref)


def test_large_calls_on_two_streams():
    """Calls whose blocks wait for one another, at the same time on two streams."""
    x, dy, w, b = inputs(2, 30000, 64, torch.bfloat16, torch.float32, 16)
    want = dot.group_norm_act(x, 8, w, b)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(dot.group_norm_act(x, 8, w, b))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for o in outs for t in o)


def test_nearly_constant_groups_without_eps():
    """Variances down to a few roundings of the values, eps 0: finite, and within the values' own rounding."""
    for spread in (1e-3, 1e-5, 1e-6):
        x = (3.0 + spread * torch.randn(2, 5000, 32, generator=U.gen(7))).to(DEV)
        y = dot.group_norm_act(x, 4, eps=0.0, activation="none")
        want = norm64(x.double(), 4, None, None, 0.0, "none")
        assert torch.isfinite(y).all()
        # the stored mean is off by up to 3 * 2^-23 of the smallest standard deviation
        std = float(x.double().reshape(2, 5000, 4, 8).std(dim=(1, 3)).min())
        assert float((y.double() - want).abs().max()) <= 2.0 ** -22 / std + 1e-4 * float(want.abs().max())


def test_raw_refusals():
    from dot_b200 import ops

    x, w = torch.randn(2, 10, 32, device=DEV), torch.ones(32, device=DEV)
    y, stats = ops.group_norm_forward_raw(x, 4, w, None, 1e-5, 1)
    for bad in (lambda: ops.group_norm_forward_raw(x, 5, w, None, 1e-5, 1),
                lambda: ops.group_norm_forward_raw(x, 4, w[:16], None, 1e-5, 1),
                lambda: ops.group_norm_forward_raw(x, 4, w, w.half(), 1e-5, 1),
                lambda: ops.group_norm_forward_raw(x, 4, w, None, 1e-5, 1, torch.ones(2, device=DEV)),
                lambda: ops.group_norm_backward_raw(x, y.half(), 4, w, None, 1, stats),
                lambda: ops.group_norm_backward_raw(x, y[:1], 4, w, None, 1, stats),
                lambda: ops.group_norm_backward_raw(x, y, 4, w, None, 1, stats[:4])):
        with pytest.raises(ValueError):
            bad()
