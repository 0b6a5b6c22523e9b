"""What activations kept in 8 bits stand for, in 64 bits and from the definition (no code of the package)."""
import math

import torch

LARGEST = {"e4m3": 448.0, "int8": 127.0}


def nearest(v, fmt):
    """The format's value nearest to each v, ties to the even one."""
    if fmt == "int8":
        return torch.round(v)
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)       # 3 mantissa bits; below 2^-6 the spacing stays
    return torch.round(v / step) * step


def keep(x, fmt):
    """(codes, scales of every value) of rows x [T, n], in 64 bits."""
    x = x.double()
    codes, scales = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.shape[0]):
        for c in range(0, x.shape[1], 128):
            v = x[t, c:c + 128]
            top = float("nan") if not torch.isfinite(v).all() else v.abs().max().item()
            if math.isnan(top):
                scales[t, c:c + 128] = top
            elif top >= 2.0 ** -100:
                s = top / LARGEST[fmt] if fmt == "int8" else 2.0 ** math.ceil(math.log2(top) - math.log2(448.0) - 1e-9)
                if fmt == "e4m3":
                    assert top / s <= 448 < 2 * top / s
                    s = min(s, 2.0 ** 119)                                   # nothing reads back as infinity
                codes[t, c:c + 128], scales[t, c:c + 128] = nearest(v / s, fmt).clamp(-LARGEST[fmt], LARGEST[fmt]), s
    return codes, scales


def spread(scale, n):
    """Scales [T, ceil(n / 128)] as one for every value [T, n], in 64 bits."""
    return scale.double().repeat_interleave(128, 1)[:, :n]


def norm(s, w, eps):
    """(s r w, s r, r) of rows s in 64 bits."""
    s = s.double()
    r = (s.square().mean(1, keepdim=True) + eps) ** -0.5
    return s * r * w.double(), s * r, r


def norm_grad(dy, xh, w, r, ds=None):
    """(dx, dw) of a norm whose normalised rows are xh, in 64 bits."""
    dy, xh = dy.double(), xh.double()
    g = dy * w.double()
    dx = r.double() * (g - xh * (g * xh).mean(1, keepdim=True))
    return dx if ds is None else dx + ds.double(), (dy * xh).sum(0)


def swiglu(g, u):
    return g.double() * torch.sigmoid(g.double()) * u.double()


def swiglu_grad(dh, g, u):
    dh, g, u = dh.double(), g.double(), u.double()
    p = torch.sigmoid(g)
    return torch.cat([dh * u * (p + g * p * torch.sigmoid(-g)), dh * g * p], 1)


def borders():
    """(x, codes) [T, 128]: bf16 values next to and on the borders of int8's codes, with every mantissa M for a group's largest and
    every other mantissa 2^0 to 2^-10 below it; the codes by whole numbers, nearest(127 X / (M 2^s)) with ties to the even one."""
    M = torch.arange(128, 256).view(-1, 1, 1, 1)
    s = torch.arange(11).view(1, -1, 1, 1)
    X = torch.stack([torch.arange(129, 256), torch.arange(128, 255)]).view(1, 1, 2, -1).expand(128, 11, 2, 127)
    X = torch.where((s > 0) | (X <= M), X, 0)
    X = torch.cat([(M << s).expand(128, 11, 2, 1), X], 3)                   # the group's largest first
    num, den = 2 * 127 * X, 2 * (M << s)
    q = (num + den // 2) // den
    q = q - ((num + den // 2) % den == 0).long() * (q % 2)
    sign = torch.where(torch.arange(128) % 3 == 0, -1, 1)
    x = torch.ldexp(X.double(), -s)
    return (x * sign).reshape(-1, 128), (q * sign).reshape(-1, 128)
