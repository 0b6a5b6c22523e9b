"""Activations kept in 8 bits between the forward and the backward pass: the work whose speed is tracked.

Values are kept in groups of 128 columns of a row (the last group of a row may be shorter): codes of 8 bits (``e4m3``: floating
point of 4 exponent and 3 mantissa bits, largest 448; ``int8``: -127 to 127) and one fp32 scale a group.  For ``int8`` it is the
group's largest magnitude over 127; for ``e4m3``, which has exponents of its own, the smallest power of two that brings the largest
magnitude to 448 or below.  What is kept is returned as the values it stands for, in the type of the tensor it was made from.

Operators:

* ``pack``: a tensor is kept and restored: a layer's input under activation checkpointing.
* ``norm``: residual addition and RMSNorm, the normalised row (without the weight) kept; backward from what was kept, and the
  norm's output restored for the weight gradient of the projection behind it.
* ``swiglu``: silu(gate) * up, gate and up kept; the product restored for the weight gradient of the down projection, and the
  backward.
* ``linear``: a projection whose input is kept in 8 bits: product, input gradient, weight gradient from the restored input.

Lengths, widths and types are those of the presets in ``config.py``, of ``bench.py`` and the tests.
"""
import math

import torch

own = False

GROUP = 128
LARGEST = {"e4m3": 448.0, "int8": 127.0}
EPS = 1e-5


def _case(name, op, fmt, tokens, width, out=0):
    c = {"name": name, "op": op, "fmt": fmt, "tokens": tokens, "width": width}
    if op == "linear":
        c["out"] = out
    return c


def listed():
    return [
        # inputs of the smallest test model's layers: nothing but launches
        _case("pack_128x256_int8", "pack", "int8", 128, 256),
        # gate|up width of the test models, which ends inside a group, at a length that is no multiple of any tile
        _case("pack_4001x688_e4m3", "pack", "e4m3", 4001, 688),
        # layer inputs of a 7B model at 128K tokens on one GPU: 1 GB of bf16
        _case("pack_131072x4096_e4m3", "pack", "e4m3", 131072, 4096),
        # one block of a short prompt in the small test model
        _case("norm_37x1024_e4m3", "norm", "e4m3", 37, 1024),
        # a rank's share of a long sequence: 2K tokens of a 7B or 8B model
        _case("norm_2048x4096_int8", "norm", "int8", 2048, 4096),
        # 64K tokens of the same model on one GPU
        _case("norm_65536x4096_e4m3", "norm", "e4m3", 65536, 4096),
        # MLP of the tiny preset
        _case("swiglu_128x688_e4m3", "swiglu", "e4m3", 128, 688),
        # MLP of the small preset, ragged length
        _case("swiglu_2047x2816_int8", "swiglu", "int8", 2047, 2816),
        # MLP of a 7B model at 16K tokens
        _case("swiglu_16384x11008_e4m3", "swiglu", "e4m3", 16384, 11008),
        # q|k|v projection of the tiny preset
        _case("linear_128x256x768_e4m3", "linear", "e4m3", 128, 256, 768),
        # gate|up projection of the small preset, ragged length
        _case("linear_1531x1024x5632_int8", "linear", "int8", 1531, 1024, 5632),
        # q|k|v projection of an 8B model with grouped keys, the weak-scaling benchmark's 8K tokens per GPU
        _case("linear_8192x4096x6144_e4m3", "linear", "e4m3", 8192, 4096, 6144),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op, fmt = rng.choice(["pack", "norm", "swiglu", "linear"]), rng.choice(["e4m3", "int8"])
    # widths are multiples of 8, as the kernels of this framework want them; most of these end inside a group
    width = 8 * _log(rng, 8, {"pack": 1792, "norm": 1024, "swiglu": 1792, "linear": 512}[op])
    most = {"pack": 131072 * 4096, "norm": 65536 * 4096, "swiglu": 16384 * 11008, "linear": 8192 * 4096}[op] // width
    c = {"op": op, "fmt": fmt, "tokens": _log(rng, 1, min(most, 8192 if op == "linear" else 131072)), "width": width}
    if op == "linear":
        c["out"] = 8 * _log(rng, 8, 768)
    return c


# ----------------------------------------------------------------------------- inputs


def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def _stream(g, tokens, width):
    """A residual stream: rows of different size, and a few channels far larger than the others, as trained models have them."""
    x = torch.randn(tokens, width, generator=g, device="cuda")
    x *= 0.5 + torch.rand(tokens, 1, generator=g, device="cuda")
    x *= torch.where(torch.rand(width, generator=g, device="cuda") < 0.005, 30.0, 1.0)
    return x.to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, n = case["tokens"], case["width"]
    s = dict(case)
    if case["op"] == "pack":
        s["x"] = _stream(g, T, n)
    elif case["op"] == "norm":
        s["x"], s["delta"] = _stream(g, T, n).requires_grad_(), _normal(g, T, n, scale=0.3)
        s["w"] = (1.0 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(torch.bfloat16).requires_grad_()
        s["dy"], s["ds"] = _normal(g, T, n, scale=0.02), _normal(g, T, n, scale=0.01)
    elif case["op"] == "swiglu":
        s["gu"] = _normal(g, T, 2 * n, scale=1.5).requires_grad_()
        s["dh"] = _normal(g, T, n, scale=0.02)
    else:
        s["x"] = _normal(g, T, n).requires_grad_()
        s["w"] = _normal(g, case["out"], n, scale=0.02).requires_grad_()
        s["dy"] = _normal(g, T, case["out"], scale=0.02)
    return s


# ----------------------------------------------------------------------------- plain forms


def _groups(x):
    """[T, n] -> [T, groups, 128], the last group filled up with zeros."""
    pad = -x.shape[1] % GROUP
    return torch.nn.functional.pad(x, (0, pad)).view(x.shape[0], -1, GROUP)


def _keep(x, fmt):
    """(codes as fp32 values, scales) of fp32 rows [T, n], both by groups."""
    v = _groups(x)
    top = v.abs().amax(-1, keepdim=True)
    some = top >= 2.0 ** -100
    if fmt == "e4m3":
        m, e = torch.frexp(top)                                                 # 448 = 0.875 * 2^9
        k = e - 9 + (m > 0.875).int()
        scale, inverse = torch.ldexp(some.float(), k), torch.ldexp(some.float(), -k)
        return (v * inverse).to(torch.float8_e4m3fn).float(), scale
    q = LARGEST[fmt]
    return torch.round(v * torch.where(some, q / top, 0.0)).clamp(-q, q), torch.where(some, top / q, 0.0)


def _kept(x, fmt, factor=None):
    """The fp32 values that stand for the rows of ``x``, each row's scales times ``factor`` [T, 1]."""
    c, scale = _keep(x, fmt)
    if factor is not None:
        scale = scale * factor.unsqueeze(-1)
    return (c * scale).view(x.shape[0], -1)[:, :x.shape[1]]


def _plain(s):
    op, fmt = s["op"], s["fmt"]
    if op == "pack":
        return _kept(s["x"].float(), fmt).to(torch.bfloat16)
    if op == "norm":
        w, dy = s["w"].float(), s["dy"].float()
        total = (s["x"].float() + s["delta"].float()).to(torch.bfloat16)        # the stream is stored in its type
        v = total.float()
        r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
        y = v * r * w
        xh = _kept(v, fmt, r)
        gw = dy * w
        dx = r * (gw - xh * (gw * xh).mean(-1, keepdim=True)) + s["ds"].float()
        dw = (dy * xh).sum(0)
        return [total] + [t.to(torch.bfloat16) for t in (y, xh * w, dx, dw)]
    if op == "swiglu":
        n = s["width"]
        g, u, dh = s["gu"][:, :n].float(), s["gu"][:, n:].float(), s["dh"].float()
        h = g / (1.0 + torch.exp(-g)) * u
        g, u = _kept(g, fmt), _kept(u, fmt)
        sig = 1.0 / (1.0 + torch.exp(-g))
        dgu = torch.cat([dh * u * sig * (1.0 + g * (1.0 - sig)), dh * g * sig], 1)
        return [t.to(torch.bfloat16) for t in (h, g * sig * u, dgu)]
    x, w, dy = s["x"].float(), s["w"].float(), s["dy"].float()
    back = _kept(x, fmt).to(torch.bfloat16).float()                             # restored in the input's type
    return [t.to(torch.bfloat16) for t in (x @ w.t(), dy @ w, dy.t() @ back)]


def _own(s):
    from odysseus_transformer_b200.ops import functional as F
    op, fmt = s["op"], s["fmt"]
    if op == "pack":
        return F.unpack8(F.pack8(s["x"], fmt))
    if op == "norm":
        total, y, kept = F.add_rmsnorm8(s["x"], s["delta"], s["w"], EPS, fmt)
        back = kept.restore()
        dx, dw = torch.autograd.grad((total, y), (s["x"], s["w"]), (s["ds"], s["dy"]))
        return [total.detach(), y.detach(), back, dx, dw]
    if op == "swiglu":
        h, kept = F.swiglu8(s["gu"], fmt)
        back = kept.restore()
        (dgu,) = torch.autograd.grad(h, s["gu"], s["dh"])
        return [h.detach(), back, dgu]
    y = F.linear(s["x"], s["w"], kept=F.pack8(s["x"].detach(), fmt))
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return [y.detach(), dx, dw]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ----------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    T, n = case["tokens"], case["width"]
    kept = T * (n + 4 * -(-n // GROUP))
    if case["op"] == "pack":          # read, keep, read what was kept, write
        return {"bytes": 4 * T * n + 2 * kept, "flops": 5 * T * n}
    if case["op"] == "norm":          # x, delta, s, y, dy, ds, dx and the restored output; kept once, read once
        return {"bytes": 16 * T * n + 2 * kept + 4 * n, "flops": 25 * T * n}
    if case["op"] == "swiglu":        # gate|up, product, its gradient, restored product, gradient of gate|up
        return {"bytes": 14 * T * n + 4 * kept, "flops": 40 * T * n}
    m = case["out"]                   # input and its gradient, weight and its gradient, output and its gradient
    return {"bytes": 4 * (T * n + n * m + T * m) + 2 * kept, "flops": 6 * T * n * m}


# ----------------------------------------------------------------------------- the definition in 64 bits


def _nearest(v, fmt):
    """The nearest value of the format to each |v| <= its largest, ties to the even one."""
    if fmt == "int8":
        return torch.round(v)
    _, e = torch.frexp(v)                                   # v = m * 2^e, 0.5 <= |m| < 1
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _stands_for(x, fmt):
    """What rows of doubles are kept as, group by group."""
    q = LARGEST[fmt]
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], GROUP):
        v = x[:, c:c + GROUP]
        top = v.abs().amax(1, keepdim=True)
        scale = top / q
        if fmt == "e4m3":
            m, e = torch.frexp(scale)                                                 # up to the next power of two
            scale = torch.ldexp(torch.ones_like(scale), torch.where(m == 0.5, e - 1, e))
        near = _nearest(v / scale, fmt) * scale
        out[:, c:c + GROUP] = torch.where(top < 2.0 ** -100, torch.zeros_like(v), near)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        op, fmt, d = case["op"], case["fmt"], torch.float64
        if op == "pack":
            return _stands_for(s["x"].to(d), fmt)
        if op == "norm":
            total = s["x"].to(d) + s["delta"].to(d)
            v = total.to(torch.bfloat16).to(d)
            w, dy = s["w"].to(d), s["dy"].to(d)
            r = (v.square().mean(1, keepdim=True) + EPS) ** -0.5
            y = v * r * w
            xh = _stands_for(v, fmt) * r
            back = xh * w
            c = (dy * back).mean(1, keepdim=True)
            dx = (dy * w - xh * c) * r + s["ds"].to(d)
            return [total, y, back, dx, (dy * xh).sum(0)]
        if op == "swiglu":
            n = case["width"]
            g, u, dh = s["gu"][:, :n].to(d), s["gu"][:, n:].to(d), s["dh"].to(d)
            h = u * g * torch.sigmoid(g)
            g, u = _stands_for(g, fmt), _stands_for(u, fmt)
            p = torch.sigmoid(g)
            return [h, u * g * p, torch.cat([dh * u * (p + g * p * torch.sigmoid(-g)), dh * g * p], 1)]
        x, w, dy = s["x"].to(d), s["w"].to(d), s["dy"].to(d)
        back = _stands_for(x, fmt).to(torch.bfloat16).to(d)
        return [x @ w.t(), dy @ w, dy.t() @ back]
