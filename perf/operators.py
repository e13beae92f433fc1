"""Cases of the feature operators that stand before the matching layers.

Two operators prepare dense features for a soft matching (bidirectional
softmax or Sinkhorn): group normalisation with an activation on channels-last
maps, and rotary positions with several axes.  Each case is one call as a
matcher makes it: an inference call returns the outputs, a training call the
outputs and all gradients.  With ``own`` false the operators are computed from
elementary torch operations in 32 bits, with ``own`` true by dot_b200.

    group norm   z = (x - mean) * rsqrt(var + eps) * weight + bias,  y = act(z);
                 mean and var over a sample's valid positions and a group's
                 channels; positions beyond a sample's length give 0.
    rotary       angle[t, p] = sum_a positions[t, a] * freqs[p, a];  pair p of
                 every head of token t is turned by that angle, what lies
                 beyond the pairs passes through.
"""

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-5


# ---- cases ---------------------------------------------------------------------

def _gn(name, n, dims, c, g, dtype, act, train=False, ragged=False, wtype="f32"):
    case = {"op": "group_norm_act", "n": n, "s": math.prod(dims), "c": c, "g": g, "dtype": dtype, "act": act,
            "train": train, "ragged": ragged, "wtype": wtype}
    return dict(case, name=name) if name else case


def _rot(name, b, dims, hq, hk, d, pairs, axes, dtype, positions="grid", interleaved=False, train=False, offset=0):
    case = {"op": "rotary", "b": b, "l": math.prod(dims), "width": dims[-1], "hq": hq, "hk": hk, "d": d,
            "pairs": pairs, "axes": axes, "dtype": dtype, "positions": positions, "interleaved": interleaved,
            "train": train, "offset": offset}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one small patch's features at inference: the call's latency
        _gn("norm_patch_bf16", 1, (8, 8), 64, 8, "bf16", "silu"),
        # 1/8-resolution maps of a batch of 480 x 640 images at inference
        _gn("norm_coarse_bf16", 8, (60, 80), 256, 32, "bf16", "silu"),
        # 1/2-resolution maps of a batch of images at inference: beyond the L2 cache
        _gn("norm_stem_bf16", 16, (240, 320), 64, 16, "bf16", "relu"),
        # 1/4-resolution maps of an image pair, trained in float32
        _gn("norm_mid_train_f32", 2, (120, 160), 128, 32, "f32", "gelu", train=True),
        # ragged sets of 1024 keypoint descriptors, padded, one set empty: training
        _gn("norm_points_train_bf16", 16, (1024,), 256, 32, "bf16", "silu", train=True, ragged=True),
        # an odd crop with channel groups that fill no vector: training
        _gn("norm_crop_train_f16", 3, (37, 53), 90, 6, "f16", "silu", train=True, wtype="f16"),
        # clips normalised over time, height and width: the largest training call
        _gn("norm_clip_train_bf16", 2, (16, 60, 80), 256, 32, "bf16", "silu", train=True, wtype="bf16"),
        # one new token for each of eight streams
        _rot("rotary_token_bf16", 8, (1,), 32, 8, 128, 64, 3, "bf16", positions="each", offset=40000),
        # queries and keys of a clip, cut out of a fused projection
        _rot("rotary_clip_bf16", 1, (16, 30, 40), 16, 4, 128, 64, 3, "bf16"),
        # ragged keypoint sets with continuous coordinates
        _rot("rotary_points_f16", 16, (1024,), 4, 4, 64, 32, 2, "f16", positions="points"),
        # an odd crop's queries and keys, neighbouring pairs, trained in float32
        _rot("rotary_crop_train_f32", 4, (37, 53), 8, 8, 64, 32, 2, "f32", interleaved=True, train=True),
        # packed sequences of text and frames, part of each head turned: training
        _rot("rotary_packed_train_bf16", 1, (33333,), 12, 3, 80, 32, 3, "bf16", positions="each", train=True,
             offset=20000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_BYTES = 3.2e8   # below the largest listed case's


def draw(rng):
    while True:
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        train = rng.random() < 0.5
        if rng.random() < 0.5:
            cg = rng.choice((2, 3, 4, 5, 8, 8, 10, 15, 16, 24))
            g = rng.choice((1, 4, 6, 8, 16, 32, 32))
            case = _gn("", _log(rng, 1, 16), (_log(rng, 64, 76800),), cg * g, g, dtype,
                       rng.choice(("silu", "silu", "gelu", "none") if train else ("silu", "relu", "gelu")), train=train,
                       ragged=rng.random() < 0.3,
                       wtype=rng.choice(("f32", dtype)))
            sizes = (case["n"], case["s"], case["c"])
        else:
            hk = rng.choice((1, 2, 3, 4, 8, 12))
            hq = hk * rng.choice((1, 1, 2, 4))
            d = 2 * rng.choice((16, 20, 24, 32, 32, 40, 48, 64, 64, 128))
            axes = rng.choice((1, 2, 3))
            pairs = d // 2 if rng.random() < 0.7 else max(axes, d // 4 + rng.choice((0, 1, 2)))
            b, l = _log(rng, 1, 16), _log(rng, 1, 33333)
            positions = rng.choice(("grid", "points", "each"))
            case = _rot("", b, (l, min(l, rng.choice((16, 20, 40, 53)))), hq, hk, d, pairs, axes, dtype,
                        positions=positions, interleaved=rng.random() < 0.3, train=train,
                        offset=0 if dtype == "f32" or positions != "each" else _log(rng, 1, 40000))
            case["l"] = l
            sizes = (b, l, hq, hk, d, hq * d, hk * d, pairs, hq + 2 * hk, (hq + 2 * hk) * d)
        if work(case)["bytes"] <= _MOST_BYTES and 3072 not in sizes:
            return case


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    passes = 4 if case["train"] else 2          # x, y; and dy, dx where it trains
    if case["op"] == "group_norm_act":
        n, s, c = case["n"], case["s"], case["c"]
        valid = sum(_lengths(n, s)) if case["ragged"] else n * s
        elements = (passes // 2) * (valid + n * s) * c      # padding is written, not read
        wsize = 4 if case["wtype"] == "f32" else 2
        flops = (30 if case["train"] else 12) * valid * c
        return {"bytes": elements * size + passes * c * wsize, "flops": flops}
    tokens = case["b"] * case["l"]
    turned = tokens * (case["hq"] + case["hk"]) * case["d"]
    rows = tokens if case["positions"] != "grid" else case["l"]
    table = rows * case["axes"] * (4 if case["positions"] == "points" else 8) + case["pairs"] * case["axes"] * 4
    angles = tokens * case["pairs"] * (2 * case["axes"] + 20)
    return {"bytes": passes * turned * size + table, "flops": passes // 2 * (3 * turned + angles)}


# ---- inputs ----------------------------------------------------------------------

def _lengths(n, s):
    """Valid positions of each padded sample: a full one, then an empty one, then part-filled ones."""
    return [s if i == 0 else 0 if i == 1 and n > 2 else 1 + (s - 1) * ((7 * i) % n) // n for i in range(n)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    st = dict(case)
    if case["op"] == "group_norm_act":
        n, s, c = case["n"], case["s"], case["c"]
        wtype = _TYPES[case["wtype"]]
        # features keep an offset and a spread of their own in each channel
        st["x"] = (normal(n, s, c).mul_(0.5 + normal(c).abs()).add_(normal(c))).to(dtype)
        st["weight"] = (1 + 0.2 * normal(c)).to(wtype)
        st["bias"] = (0.2 * normal(c)).to(wtype)
        st["lengths"] = None
        if case["ragged"]:
            order = torch.randperm(n, generator=gen, device="cuda")
            st["lengths"] = torch.tensor(_lengths(n, s), dtype=torch.int32, device="cuda")[order].contiguous()
        if case["train"]:
            st["dy"] = normal(n, s, c).to(dtype)
            for name in ("x", "weight", "bias"):
                st[name].requires_grad_(True)
        return st
    b, l, hq, hk, d, axes = (case[k] for k in ("b", "l", "hq", "hk", "d", "axes"))
    if case["train"]:
        for name, h in (("q", hq), ("k", hk)):
            st[name] = normal(b, l, h, d).to(dtype).requires_grad_(True)
            st["d" + name] = normal(b, l, h, d).to(dtype)
    else:
        st["qkv"] = normal(b, l, hq + 2 * hk, d).to(dtype)   # a fused projection; the values stay where they are
    t = torch.arange(l, device="cuda")
    if case["positions"] == "points":       # continuous image coordinates
        st["positions"] = torch.rand(b, l, axes, generator=gen, device="cuda") * 64
    elif case["positions"] == "grid":       # frame, row and column of a token, the same for the batch
        w = max(1, case["width"])
        rows = (t // (w * w), (t // w) % w, t % w)
        st["positions"] = torch.stack(rows[3 - axes:], dim=-1)
    else:                                   # each token's own position along every axis
        first = torch.randint(0, case["offset"] + 1, (b, 1, 1), generator=gen, device="cuda")
        st["positions"] = (first + torch.randint(0, 64, (b, l, axes), generator=gen, device="cuda")).contiguous()
    # every axis has its own band of frequencies
    pairs = case["pairs"]
    share = [pairs // axes + (a < pairs % axes) for a in range(axes)]
    freqs = torch.zeros(pairs, axes, dtype=torch.float64)
    at = 0
    for a, n in enumerate(share):
        freqs[at:at + n, a] = 10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
        at += n
    st["freqs"] = freqs.float().cuda()
    return st


# ---- plain forms -----------------------------------------------------------------

def _act(z, act):
    """act(z) and its derivative."""
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return z * sg, sg * (1 + z * (1 - sg))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    return z, torch.ones_like(z)


def _plain_norm(st):
    n, s, c, g = st["n"], st["s"], st["c"], st["g"]
    x = st["x"].detach()
    w, b = (st[k].detach().float() for k in ("weight", "bias"))
    xf = x.float().view(n, s, g, c // g)
    if st["lengths"] is not None:
        valid = (torch.arange(s, device=x.device) < st["lengths"][:, None])[:, :, None, None]
        count = (st["lengths"].float() * (c // g)).clamp(min=1)[:, None, None, None]
    else:
        valid, count = None, float(s * (c // g))

    def keep(v):
        return v if valid is None else torch.where(valid, v, torch.zeros((), device=v.device))

    mean = keep(xf).sum(dim=(1, 3), keepdim=True) / count
    dev = keep(xf - mean)
    rstd = torch.rsqrt(dev.square().sum(dim=(1, 3), keepdim=True) / count + _EPS)
    xhat = dev * rstd
    wv, bv = w.view(g, c // g), b.view(g, c // g)
    y, slope = _act(xhat * wv + bv, st["act"])
    out = {"y": keep(y).reshape(n, s, c).to(x.dtype)}
    if st["train"]:
        dz = keep(st["dy"].float().view(n, s, g, c // g) * slope)
        out["dbias"] = dz.sum(dim=(0, 1)).reshape(c).to(st["bias"].dtype)
        out["dweight"] = (dz * xhat).sum(dim=(0, 1)).reshape(c).to(st["weight"].dtype)
        dxhat = dz * wv
        m1 = dxhat.sum(dim=(1, 3), keepdim=True) / count
        m2 = (dxhat * xhat).sum(dim=(1, 3), keepdim=True) / count
        out["dx"] = keep((dxhat - m1 - xhat * m2) * rstd).reshape(n, s, c).to(x.dtype)
    return out


def _turn(x, cos, sin, pairs, interleaved):
    xf = x.float()
    head, rest = xf[..., :2 * pairs], xf[..., 2 * pairs:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
    else:
        a, b = head[..., :pairs], head[..., pairs:]
    u, v = a * cos - b * sin, b * cos + a * sin
    head = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    return torch.cat((head, rest), dim=-1).to(x.dtype)


def _split(st):
    if st["train"]:
        return st["q"].detach(), st["k"].detach()
    return st["qkv"][:, :, :st["hq"]], st["qkv"][:, :, st["hq"]:st["hq"] + st["hk"]]


def _plain_rotary(st):
    angle = (st["positions"].float()[..., None, :] * st["freqs"]).sum(dim=-1)
    cos, sin = torch.cos(angle)[..., None, :], torch.sin(angle)[..., None, :]
    pairs, il = st["pairs"], st["interleaved"]
    q, k = _split(st)
    out = {"q": _turn(q, cos, sin, pairs, il), "k": _turn(k, cos, sin, pairs, il)}
    if st["train"]:
        out["dq"] = _turn(st["dq"], cos, -sin, pairs, il)
        out["dk"] = _turn(st["dk"], cos, -sin, pairs, il)
    return out


# ---- one pass --------------------------------------------------------------------

def run(st):
    if not own:
        return _plain_norm(st) if st["op"] == "group_norm_act" else _plain_rotary(st)
    import dot_b200

    if st["op"] == "group_norm_act":
        y = dot_b200.group_norm_act(st["x"], st["g"], st["weight"], st["bias"], eps=_EPS, activation=st["act"],
                                    lengths=st["lengths"])
        if not st["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if not st["train"]:
        q, k = _split(st)
        q, k = dot_b200.rotary(q, st["positions"], st["freqs"], k=k, interleaved=st["interleaved"])
        return {"q": q, "k": k}
    q, k = dot_b200.rotary(st["q"], st["positions"], st["freqs"], k=st["k"], interleaved=st["interleaved"])
    dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


# ---- 64 bits ---------------------------------------------------------------------

def _exact_norm(st):
    """Sample by sample, the gradients from differentiating the definition."""
    n, s, c, g = st["n"], st["s"], st["c"], st["g"]
    w, b = (st[k].detach().double().requires_grad_(st["train"]) for k in ("weight", "bias"))
    lengths = [s] * n if st["lengths"] is None else st["lengths"].tolist()
    y = torch.zeros(n, s, c, dtype=torch.float64, device="cuda")
    dx = torch.zeros_like(y) if st["train"] else None
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for i, length in enumerate(lengths):
        if length == 0:
            continue
        x = st["x"][i, :length].detach().double().requires_grad_(st["train"])
        by_group = x.reshape(length, g, c // g).transpose(0, 1).reshape(g, -1)
        var, mean = torch.var_mean(by_group, dim=1, correction=0, keepdim=True)
        z = ((by_group - mean) / torch.sqrt(var + _EPS)).reshape(g, length, c // g).transpose(0, 1).reshape(length, c)
        z = z * w + b
        if st["act"] == "silu":
            out = z * torch.sigmoid(z)
        elif st["act"] == "gelu":
            out = z * torch.special.ndtr(z)
        else:
            out = z.clamp(min=0) if st["act"] == "relu" else z
        y[i, :length] = out.detach()
        if st["train"]:
            grads = torch.autograd.grad(out, (x, w, b), st["dy"][i, :length].double())
            dx[i, :length] = grads[0]
            dw, db = dw + grads[1], db + grads[2]
    if not st["train"]:
        return {"y": y}
    return {"y": y, "dx": dx, "dweight": dw.detach(), "dbias": db.detach()}


def _exact_turn(x, rot, interleaved):
    """Pairs as complex numbers, multiplied by exp(i angle)."""
    pairs = rot.shape[-1]
    out = x.double().clone()
    head = out[..., :2 * pairs]
    shape = (*head.shape[:-1], pairs, 2) if interleaved else (*head.shape[:-1], 2, pairs)
    both = head.reshape(shape) if interleaved else head.reshape(shape).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(both.contiguous()) * rot)
    out[..., :2 * pairs] = (turned if interleaved else turned.transpose(-1, -2)).reshape(head.shape)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "group_norm_act":
        return _exact_norm(st)
    angle = torch.einsum("...a,pa->...p", st["positions"].double(), st["freqs"].double())[..., None, :]
    rot = torch.polar(torch.ones_like(angle), angle)
    q, k = _split(st)
    out = {"q": _exact_turn(q, rot, case["interleaved"]), "k": _exact_turn(k, rot, case["interleaved"])}
    if case["train"]:
        out["dq"] = _exact_turn(st["dq"], rot.conj(), case["interleaved"])
        out["dk"] = _exact_turn(st["dk"], rot.conj(), case["interleaved"])
    return out
